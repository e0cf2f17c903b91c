"""What a launch of the int8 rows can hold, on the CPU: the plans stay within a grid, or refuse."""
import re

import torch

import libr3d_amd as R


def gemm(M, N, K):
    """A call of any size over one row's memory: the rows of an operand may lie on each other."""
    i8 = torch.zeros(1, K, dtype=torch.int8)
    one = torch.ones(1)
    return R.GemmOperands(i8.expand(M, K), one.expand(M), i8.expand(N, K), one.expand(N),
                          torch.zeros(M, N, dtype=torch.bfloat16), dtype="i8a8", N=N, K=K, M=M)


def test_tall_products_keep_k_in_one_chunk():
    """The planes of a K split are joined a row a workgroup of the grid's second axis: 65535 at most."""
    for M, N, K in ((65535, 48, 8192), (65536, 48, 8192), (70000, 16, 16384), (200000, 8, 65536)):
        ops = gemm(M, N, K)
        need = R.row_scratch_bytes("gemm_nt_q_i8a8", ops)
        if need:
            ops.set_scratch(torch.empty(16, dtype=torch.uint8), need)
            ops.args.scratch = (ops.args.scratch + 15) // 16 * 16         # an address; nothing is launched
        rc, text = R.describe("gemm_nt_q_i8a8", ops)
        assert rc == R.RAD_OK
        kc = int(re.search(r" kc=(\d+)", text).group(1))
        assert kc == 1 or M <= 65535, text
        assert (need > 0) == (kc > 1)


def test_rows_past_a_grid_are_refused():
    ops = gemm(4, 8, 33)                              # K off 16: the kernel for any alignment
    for M, want in ((65535 * 32, R.RAD_OK), (65535 * 32 + 1, R.RAD_E_UNSUPPORTED)):
        ops._t[0].shape[0] = ops._t[1].shape[0] = ops._t[4].shape[0] = M
        assert R.describe("gemm_nt_q_i8a8", ops)[0] == want
    x = torch.zeros(3, 4000, dtype=torch.bfloat16)
    ops = R.QuantActI8Operands(x, torch.zeros(3, 4000, dtype=torch.int8), torch.zeros(3), n=4000)
    for M, want in ((1 << 22, R.RAD_OK), (1 << 24, R.RAD_E_UNSUPPORTED)):
        for t in range(3):
            ops._t[t].shape[0] = M
        assert R.describe("quant_act_i8", ops)[0] == want
