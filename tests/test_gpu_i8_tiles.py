"""Every LDS tile of the int8 product, whole K and split, on shapes that do not fill it: bit for bit."""
import re

import pytest
import torch

import libr3d_amd as R
from tests.test_gpu_i8 import run_gemm

SHAPES = [(15, 77, 128), (17, 37, 528), (10, 42, 3328), (18, 27, 2784), (19, 4567, 1024),
          (20, 4617, 1072), (52, 525, 6272), (90, 392, 6224), (71, 1679, 256), (61, 2592, 192),
          (18, 435, 4608), (18, 1374, 2720), (41, 8979, 256), (66, 5942, 176), (35, 2753, 5248),
          (751, 82, 5824), (434, 2314, 384), (130, 6566, 160), (71, 2735, 6400), (72, 2911, 5200),
          (404, 4773, 384), (456, 4728, 144), (66, 8545, 4864), (65, 5496, 6064), (965, 6207, 256),
          (987, 6657, 176), (341, 2746, 5888), (97, 8843, 5952), (1026, 4287, 128), (539, 7309, 160),
          (959, 6700, 1792), (2000, 8100, 1024), (2000, 8100, 1040)]
# (weight rows, tokens, K split, rows that begin inside lines): what those shapes have to reach between them
TILES = {(32, 16, 0, 0), (32, 16, 0, 1), (32, 16, 1, 0), (32, 16, 1, 1), (32, 32, 0, 0),
         (32, 32, 0, 1), (32, 32, 1, 0), (32, 32, 1, 1), (64, 32, 0, 0), (64, 32, 0, 1),
         (64, 32, 1, 0), (64, 32, 1, 1), (64, 64, 0, 0), (64, 64, 0, 1), (64, 64, 1, 0),
         (64, 64, 1, 1), (128, 64, 0, 0), (128, 64, 0, 1), (128, 64, 1, 0), (128, 64, 1, 1),
         (128, 96, 0, 0), (128, 96, 0, 1), (128, 96, 1, 0), (128, 96, 1, 1), (128, 128, 0, 0),
         (128, 128, 0, 1), (128, 128, 1, 0), (128, 128, 1, 1), (128, 192, 0, 0), (128, 192, 0, 1),
         (128, 256, 0, 0), (256, 256, 0, 0), (256, 256, 0, 1)}


def test_shapes_reach_every_tile():
    got = set()
    for M, N, K in SHAPES:
        i8, one = torch.zeros(K + 128, dtype=torch.int8), torch.ones(1)
        i8 = i8[-i8.data_ptr() % 128:][:K].view(1, K)
        y = torch.zeros(M, N, dtype=torch.bfloat16)
        ops = R.GemmOperands(i8.expand(M, K), one.expand(M), i8.expand(N, K), one.expand(N), y, dtype="i8a8", N=N, K=K, M=M)
        ops._t[0].stride[0] = ops._t[2].stride[0] = K           # described only: dense rows
        need = R.row_scratch_bytes("gemm_nt_q_i8a8", ops)
        if need:
            ops.set_scratch(y, need)                 # an aligned address is all it takes
            ops.args.scratch = (ops.args.scratch + 15) // 16 * 16
        text = R.describe("gemm_nt_q_i8a8", ops)[1]
        bn, bm, kc = (int(v) for v in re.search(r"bn=(\d+) bm=(\d+) .*kc=(\d+)", text).groups())
        got.add((bn, bm, int(kc > 1), int(K % 128 > 0)))
    assert TILES <= got, TILES - got


@pytest.mark.gpu
@pytest.mark.parametrize("M,N,K", SHAPES)
def test_tile(gpu, M, N, K):
    run_gemm(gpu, M, N, K)
    run_gemm(gpu, M, N, K, pitch=(K + 112, K + 48, N + 5), seed=1)
