"""The int8 product's scratch hook asks for the planes of the launch that the call takes: by its operands'
own alignment and pitches, and for none where the kernel for any alignment runs."""
import re

import pytest
import torch

import libr3d_amd as R
from tests.test_gpu_i8 import run_gemm

ROW = "gemm_nt_q_i8a8"


def call(M, N, K, pitch, off):
    """Operands whose rows are `pitch` bytes apart and `off` past a line; planned only, so they lie on each other."""
    i8 = torch.zeros(K + 512, dtype=torch.int8)
    at = -i8.data_ptr() % 128 + off
    row, one = i8[at:at + K].view(1, K), torch.ones(1)
    ops = R.GemmOperands(row.expand(M, K), one.expand(M), row.expand(N, K), one.expand(N),
                         torch.zeros(M, N, dtype=torch.bfloat16), dtype="i8a8", N=N, K=K, M=M)
    ops._t[0].stride[0] = ops._t[2].stride[0] = pitch
    return ops


def wanted(ops, M, N):
    """Bytes of the planes that the launch takes when it may have all it wants."""
    ops.args.scratch, ops.args.scratch_bytes = 1 << 20, 1 << 28          # an address; nothing is launched
    text = R.describe(ROW, ops)[1]
    ops.args.scratch, ops.args.scratch_bytes = None, 0
    kc = int(re.search(r" kc=(\d+)", text).group(1))
    return 4 * kc * M * N if "arm=tile" in text and kc > 1 else 0


# (off, pitch - K): rows on lines; a base, a pitch or both inside lines; off 16 bytes
PLACES = [(0, 0), (16, 0), (0, 16), (32, 48), (1, 0), (0, 3), (5, 7)]


@pytest.mark.parametrize("M,N,K", [(61, 4074, 7552), (264, 2832, 9600), (149, 192, 7040), (89, 3023, 9216), (3, 300, 5376),
                                   (40, 1500, 5360)])
def test_bytes_are_the_launch_s(M, N, K):
    got = {}
    for off, more in PLACES:
        ops = call(M, N, K, K + more, off)
        got[off, more] = R.row_scratch_bytes(ROW, ops)
        assert got[off, more] == wanted(ops, M, N), (off, more)
    assert got[1, 0] == got[0, 3] == got[5, 7] == 0


def test_some_of_the_shapes_split_only_inside_lines():
    for M, N, K in ((61, 4074, 7552), (264, 2832, 9600)):
        assert R.row_scratch_bytes(ROW, call(M, N, K, K, 0)) == 0 < R.row_scratch_bytes(ROW, call(M, N, K, K, 16))


def test_without_operands_as_dense_ones():
    M, N, K = 149, 192, 7040
    ops = call(M, N, K, K, 0)
    whole = R.row_scratch_bytes(ROW, ops)
    for i in range(5):
        ops._t[i].data = None                            # M by the parameter from here on
        assert R.row_scratch_bytes(ROW, ops) == whole > 0


@pytest.mark.gpu
@pytest.mark.parametrize("M,N,K", [(61, 4074, 7552), (264, 2832, 9600)])
def test_split_products_of_rows_inside_lines(gpu, M, N, K):
    run_gemm(gpu, M, N, K, offs=(16, 32, 0))
    run_gemm(gpu, M, N, K, pitch=(K + 16, K + 48, N + 3), seed=1)
