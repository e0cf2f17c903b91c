"""Every LDS tile of the int8 product, whole K and split, on shapes that do not fill it: bit for bit."""
import re

import pytest
import torch

import libr3d_amd as R
from tests.test_gpu_i8 import run_gemm

SHAPES = [(33, 48, 224), (9, 41, 6256), (34, 3186, 672), (104, 308, 4432), (57, 2079, 256),
          (19, 563, 5856), (43, 8615, 160), (34, 3135, 5104), (100, 8905, 336), (68, 2818, 6112),
          (290, 6890, 176), (68, 5509, 5536), (894, 3592, 272), (98, 8247, 4560), (627, 5067, 160),
          (750, 8280, 560), (2000, 8100, 1040)]
# (weight rows, tokens, K split): what those shapes have to reach between them
TILES = {(32, 16, 0), (32, 16, 1), (32, 32, 0), (32, 32, 1), (64, 32, 0), (64, 32, 1), (64, 64, 0), (64, 64, 1),
         (128, 64, 0), (128, 64, 1), (128, 96, 0), (128, 96, 1), (128, 128, 0), (128, 128, 1), (128, 192, 0),
         (128, 256, 0), (256, 256, 0)}


def test_shapes_reach_every_tile():
    got = set()
    for M, N, K in SHAPES:
        i8, one = torch.zeros(1, K, dtype=torch.int8), torch.ones(1)
        y = torch.zeros(M, N, dtype=torch.bfloat16)
        ops = R.GemmOperands(i8.expand(M, K), one.expand(M), i8.expand(N, K), one.expand(N), y, dtype="i8a8", N=N, K=K, M=M)
        need = R.row_scratch_bytes("gemm_nt_q_i8a8", ops)
        if need:
            ops.set_scratch(y, need)                 # described only: an aligned address is all it takes
            ops.args.scratch = (ops.args.scratch + 15) // 16 * 16
        text = R.describe("gemm_nt_q_i8a8", ops)[1]
        bn, bm, kc = (int(v) for v in re.search(r"bn=(\d+) bm=(\d+) .*kc=(\d+)", text).groups())
        got.add((bn, bm, int(kc > 1)))
    assert TILES <= got, TILES - got


@pytest.mark.gpu
@pytest.mark.parametrize("M,N,K", SHAPES)
def test_tile(gpu, M, N, K):
    run_gemm(gpu, M, N, K)
    run_gemm(gpu, M, N, K, pitch=(K + 112, K + 48, N + 5), seed=1)
