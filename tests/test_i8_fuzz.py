"""Seeded fuzz of the host side of the int8 rows and the sampler, the way tests/test_plan_fuzz.py treats
the others: describe, the scratch hooks and (without a GPU) the entries over mutated operand metadata
return a status each, and describe and the entry refuse the same calls."""
import random

import pytest
import torch

import libr3d_amd as R
from tests.test_plan_fuzz import CODES, _mutate, _no_gpu

GEMM = ["gemm_nt_q_i8a8", "gemm_nt_q_i8a8_decode"]


def _build(kind, rng):
    M, n = rng.choice([1, 2, 4, 16, 17, 64]), rng.choice([1, 4, 33, 128, 1000])
    i8 = lambda *s: torch.zeros(*s, dtype=torch.int8)  # noqa: E731
    bf = lambda *s: torch.zeros(*s, dtype=torch.bfloat16)  # noqa: E731
    if kind == "gemm":
        N, K = rng.choice([1, 17, 130, 256]), rng.choice([1, 16, 77, 384])
        keep = (i8(M, K), torch.ones(M), i8(N, K), torch.ones(N), bf(M, N))
        return rng.choice(GEMM), R.GemmOperands(*keep, dtype="i8a8", N=N, K=K, M=M), keep
    if kind == "quant":
        keep = (bf(M, n), i8(M, n), torch.ones(M))
        return "quant_act_i8", R.QuantActI8Operands(*keep, n=n), keep
    if kind == "gated":
        keep = (bf(M, 2 * n), i8(M, n), torch.ones(M), bf(M, n))
        return "gated_quant_i8", R.GatedQuantI8Operands(*keep, n=n), keep
    if kind == "norm":
        keep = (bf(M, n), bf(M, n), bf(n), i8(M, n), torch.ones(M), bf(M, n))
        return "rmsnorm_quant_i8", R.RmsNormQuantI8Operands(*keep, n=n, residual_out=bf(M, n)), keep
    keep = (torch.zeros(M, n), torch.zeros(M), torch.zeros(M, dtype=torch.int32), torch.zeros(M))
    one = torch.ones(M)
    return "sample_logits", R.SampleOperands(*keep, n_vocab=n, temperature=one, top_p=one), keep + (one,)


@pytest.mark.parametrize("seed", [1, 2, 3])
def test_plans_survive_mutated_operands(seed):
    rng = random.Random(seed)
    for _ in range(500):
        row, ops, keep = _build(rng.choice(["gemm", "quant", "gated", "norm", "sample"]), rng)
        _mutate(ops.args, rng)
        rc = R.describe(row, ops)[0]
        assert rc in CODES and R.row_scratch_bytes(row, ops) >= 0
        if _no_gpu():
            got = R.launch_row(row, ops)
            assert got == (rc if rc != R.RAD_OK else R.RAD_E_UNSUPPORTED)    # the chip gate
        del keep
