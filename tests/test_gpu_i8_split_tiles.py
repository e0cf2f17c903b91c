"""K split over planes on the int8 product's largest tiles: 256 x 256, whose planes are written from its own
32 x 32 results, 128 x 192 and 128 x 256 (weight rows x tokens), on shapes that do not fill them.  Bit for bit."""
import re

import pytest

import libr3d_amd as R
from tests.test_gpu_i8 import run_gemm
from tests.test_i8_scratch_hook import call

SHAPES = [(135, 5583, 11392), (131, 6291, 13328), (198, 5417, 20992), (205, 8339, 13312), (323, 5389, 17280),
          (1493, 2705, 7312), (1483, 1306, 17152), (1042, 3883, 7184)]
# (weight rows, tokens, rows that begin inside lines) of a split launch
FORMS = {(128, 192, 0), (128, 192, 1), (128, 256, 0), (256, 256, 0), (256, 256, 1)}


def test_shapes_reach_every_form():
    got, chunks = set(), set()
    for M, N, K in SHAPES:
        ops = call(M, N, K, K, 0)
        ops.args.scratch, ops.args.scratch_bytes = 1 << 20, R.row_scratch_bytes("gemm_nt_q_i8a8", ops)
        text = R.describe("gemm_nt_q_i8a8", ops)[1]
        bn, bm, kc = (int(v) for v in re.search(r"bn=(\d+) bm=(\d+) .*kc=(\d+)", text).groups())
        assert kc > 1, text
        got.add((bn, bm, int(K % 128 > 0)))
        chunks.add(kc)
    assert got == FORMS and {3, 5, 6} <= chunks, (got, chunks)


@pytest.mark.gpu
@pytest.mark.parametrize("M,N,K", SHAPES)
def test_split_tile(gpu, M, N, K):
    run_gemm(gpu, M, N, K)
    run_gemm(gpu, M, N, K, pitch=(K + 128, K + 256, N + 5), seed=1)
