"""The int8 GEMV at every token count it takes, whole K and over 2, 4 and 8 waves, bit for bit."""
import re

import pytest
import torch

import libr3d_amd as R
from tests.test_gpu_i8 import run_gemm

SHAPES = [(12901, 5376), (333, 656), (333, 1360), (130, 5104)]      # K in 1, 2, 4, 8 chunks


def _plan(M, N, K):
    i8, one = torch.zeros(1, K, dtype=torch.int8), torch.ones(1)
    ops = R.GemmOperands(i8.expand(M, K), one.expand(M), i8.expand(N, K), one.expand(N),
                         torch.zeros(M, N, dtype=torch.bfloat16), dtype="i8a8", N=N, K=K, M=M)
    return R.describe("gemm_nt_q_i8a8_decode", ops)[1]


def test_shapes_take_the_gemv():
    got = set()
    for M in range(1, 9):
        for N, K in SHAPES:
            m = re.search(r"arm=gemv .*kc=(\d+)", _plan(M, N, K))
            got |= {("tokens", M), ("chunks", int(m.group(1)))} if m else set()
    assert got == {("tokens", M) for M in range(1, 9)} | {("chunks", kc) for kc in (1, 2, 4, 8)}


@pytest.mark.gpu
@pytest.mark.parametrize("M", range(1, 9))
def test_gemv(gpu, M):
    for N, K in SHAPES:
        run_gemm(gpu, M, N, K, row="gemm_nt_q_i8a8_decode")
        run_gemm(gpu, M, N, K, pitch=(K + 48, K + 16, N + 3), row="gemm_nt_q_i8a8_decode", seed=1)
