"""Every LDS tile of the int8 product, whole K and split, on shapes that do not fill it: bit for bit."""
import re

import pytest
import torch

import libr3d_amd as R
from tests.test_gpu_i8 import run_gemm

pytestmark = pytest.mark.gpu

# (weight rows, tokens) of the tile, K split or not, a shape that the plan gives to it
TILES = [((64, 32), False, (35, 49, 816)), ((64, 32), True, (11, 65, 4880)),
         ((64, 64), False, (97, 4593, 176)), ((64, 64), True, (926, 133, 3616)),
         ((128, 64), False, (225, 4191, 272)), ((128, 64), True, (111, 2839, 5728)),
         ((128, 96), False, (919, 2256, 288)), ((128, 96), True, (717, 713, 5456)), ((128, 96), False, (500, 5300, 640)),
         ((128, 128), False, (777, 4020, 288)), ((128, 128), True, (196, 5055, 4112)),
         ((128, 192), False, (897, 4863, 128)), ((128, 192), False, (1001, 5376, 656)),
         ((128, 256), False, (898, 6608, 560)), ((256, 256), False, (2000, 8100, 1040))]


@pytest.mark.parametrize("tile,split,shape", TILES)
def test_tile(gpu, tile, split, shape):
    M, N, K = shape
    i8, one = torch.zeros(1, K, dtype=torch.int8), torch.ones(1)
    y = torch.zeros(M, N, dtype=torch.bfloat16)
    ops = R.GemmOperands(i8.expand(M, K), one.expand(M), i8.expand(N, K), one.expand(N), y, dtype="i8a8", N=N, K=K, M=M)
    need = R.row_scratch_bytes("gemm_nt_q_i8a8", ops)
    if need:
        ops.set_scratch(y, need)                     # described only: an aligned address is all it takes
        ops.args.scratch = (ops.args.scratch + 15) // 16 * 16
    text = R.describe("gemm_nt_q_i8a8", ops)[1]
    bn, bm, kc = (int(v) for v in re.search(r"bn=(\d+) bm=(\d+) .*kc=(\d+)", text).groups())
    assert (bn, bm) == tile and (kc > 1) == split, text
    run_gemm(gpu, M, N, K)
    run_gemm(gpu, M, N, K, pitch=(K + 112, K + 48, N + 5), seed=1)
