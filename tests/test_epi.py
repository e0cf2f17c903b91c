"""The gemm_nt_epi rows on the host: the table, the resolver, what the plan takes and what it refuses."""
import json
import os
import random
import subprocess
import sys

import pytest
import torch

import libr3d_amd as R
from tests.test_plan_fuzz import CODES, _mutate, _no_gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
ROWS = {"bf16": "gemm_nt_epi_bf16", "i8a8": "gemm_nt_epi_i8a8"}
bf = lambda *s: torch.zeros(*s, dtype=torch.bfloat16)  # noqa: E731
i8 = lambda *s: torch.zeros(*s, dtype=torch.int8)  # noqa: E731


def call(dtype="bf16", M=4, N=48, K=64, **kw):
    z = bf if dtype == "bf16" else i8
    t = dict(a=z(M, K), b=z(N, K), y=bf(M, N), a_scale=None, b_scale=None, bias=None, residual=None)
    if dtype == "i8a8":
        t.update(a_scale=torch.ones(M), b_scale=torch.ones(N, 1))
    par = dict(dtype=dtype, N=N, K=K)
    for k, v in kw.items():
        (t if k in t else par)[k] = v
    return R.GemmEpiOperands(t.pop("a"), t.pop("b"), t.pop("y"), **t, **par)


def rc(ops, dtype="bf16"):
    return R.describe(ROWS[dtype], ops)[0]


def test_table_and_resolution():
    rows = {r["name"]: r for r in R.ext_rows()}
    assert set(ROWS.values()) <= set(rows) and "gemm_nt_epi" in [s["op"] for s in R.ext_schemas()]
    for d, name in ROWS.items():
        assert R.resolve("gemm_nt_epi", dict(dtype=d, M=3, N=5, K=7))["name"] == name
    assert R.resolve("gemm_nt_epi", dict(dtype="fp8a8", M=3, N=5, K=7)) is None


def test_kill_switch():
    script = ("import sys, json; sys.path.insert(0, %r); import libr3d_amd as R; "
              "print(json.dumps([r['name'] for r in R.ext_rows()]))" % ROOT)
    out = subprocess.run([sys.executable, "-c", script], env=dict(os.environ, R3D_NO_EPI="1"), capture_output=True,
                         text=True, timeout=120, check=True)
    assert set(json.loads(out.stdout)) == {r["name"] for r in R.ext_rows()} - set(ROWS.values())


@pytest.mark.parametrize("dtype", ["bf16", "i8a8"])
def test_accepts(dtype):
    z = bf if dtype == "bf16" else i8
    ok = lambda **kw: rc(call(dtype, **kw), dtype) == R.RAD_OK  # noqa: E731
    assert ok() and ok(M=1, N=1, K=1) and ok(M=1000)
    for act in ("none", "relu", "silu", "sigmoid", "gelu", "gelu_tanh"):
        assert ok(act=act)
    assert ok(bias=torch.zeros(48)) and ok(bias=bf(48)) and ok(bias=bf(1).expand(48)) and ok(bias=torch.zeros(96)[::2])
    assert ok(residual=bf(4, 48)) and ok(residual=torch.zeros(4, 60)[:, :48]) and ok(residual=bf(1, 48).expand(4, 48))
    assert ok(y=torch.zeros(4, 48)) and ok(y=bf(4, 100)[:, :48]) and ok(y=bf(2, 2, 48))
    assert ok(a=z(4, 99)[:, :64], b=z(48, 99)[:, :64])
    y = bf(4, 48)
    assert ok(y=y, residual=y)                                        # in place
    both = bf(4, 96)
    assert ok(y=both[:, :48], residual=both[:, 48:]) and ok(y=both[:, 48:], residual=both[:, :48])


@pytest.mark.parametrize("dtype", ["bf16", "i8a8"])
def test_refuses(dtype):
    z = bf if dtype == "bf16" else i8
    got = lambda **kw: rc(call(dtype, **kw), dtype)  # noqa: E731
    for k in ("a", "b", "y"):
        ops = call(dtype)
        ops._t[{"a": 0, "b": 2, "y": 6}[k]].data = None
        assert rc(ops, dtype) == R.RAD_E_INVAL
    if dtype == "bf16":
        assert got(a_scale=torch.ones(4)) == got(b_scale=torch.ones(48)) == R.RAD_E_INVAL
        assert got(a=i8(4, 64)) == got(b=i8(48, 64)) == R.RAD_E_DTYPE
        assert got(K=(1 << 20) + 1, a=bf(1, 1).expand(4, (1 << 20) + 1)) == R.RAD_E_UNSUPPORTED
    else:
        assert got(a_scale=None) == got(b_scale=None) == R.RAD_E_INVAL
        assert got(a_scale=torch.ones(3)) == got(b_scale=torch.ones(48, 2)) == R.RAD_E_SHAPE
        assert got(a_scale=bf(4)) == got(b=bf(48, 64)) == R.RAD_E_DTYPE
        assert got(K=131072) == R.RAD_E_UNSUPPORTED
    assert rc(call(dtype, act="tanh"), dtype) == R.RAD_E_UNSUPPORTED
    other = {"bf16": "i8a8", "i8a8": "bf16"}[dtype]
    assert rc(call(dtype), other) in (R.RAD_E_INVAL, R.RAD_E_UNSUPPORTED)
    assert got(y=torch.zeros(4, 48, dtype=torch.float16)) == R.RAD_E_DTYPE
    assert got(bias=torch.zeros(48, dtype=torch.float16)) == got(residual=torch.zeros(4, 48, dtype=torch.int32)) == R.RAD_E_DTYPE
    assert got(bias=torch.zeros(47)) == got(bias=torch.zeros(1, 48)) == got(residual=bf(3, 48)) == R.RAD_E_SHAPE
    assert got(y=bf(4, 49)) == got(y=bf(4, 47)) == got(a=z(4, 63)) == got(b=z(47, 64)) == R.RAD_E_SHAPE
    assert got(K=0) == got(N=0) == got(M=0) == R.RAD_E_INVAL          # nothing of an operand is there
    assert got(a=z(4, 128)[:, ::2]) == got(y=bf(48, 4).T) == R.RAD_E_STRIDE
    assert got(y=bf(1, 48).expand(4, 48)) == R.RAD_E_STRIDE           # rows that overlap
    flat = bf(8 * 48)
    assert got(y=flat[:192].view(4, 48), residual=flat[8:200].view(4, 48)) == R.RAD_E_INVAL
    shared = torch.zeros(4, 48)
    assert got(y=shared.view(torch.bfloat16)[:, :48], residual=shared) == R.RAD_E_INVAL   # the same memory, other types


@pytest.mark.parametrize("dtype", ["bf16", "i8a8"])
def test_refuses_a_result_over_its_operands(dtype):
    """Workgroups read a and b while others write y."""
    got = lambda **kw: rc(call(dtype, **kw), dtype)  # noqa: E731
    mem = bf(4, 96)
    of = (lambda t: t) if dtype == "bf16" else (lambda t: t.view(torch.int8)[:, :64])
    assert got(y=mem[:, :48], a=of(mem[:, :64])) == R.RAD_E_INVAL
    big = bf(48, 64)
    assert got(y=big[:4, :48], b=of(big)) == R.RAD_E_INVAL
    assert got(y=mem[:, 32:80], bias=mem[1, 40:88]) == R.RAD_E_INVAL
    if dtype == "bf16":
        assert got(y=mem[:, :48], a=bf(4, 64)) == R.RAD_OK
    else:
        f = torch.zeros(4, 96)
        assert got(y=f[:, :48], a_scale=f[:, 5]) == got(y=f[:, :48], b_scale=f[1, :48]) == R.RAD_E_INVAL


def test_python_calls_refuse_host_tensors():
    with pytest.raises(ValueError):
        R.gemm_nt_epi(bf(2, 8), bf(3, 8), bf(2, 3), dtype="bf16", N=3, K=8)


@pytest.mark.parametrize("dtype", ["bf16", "i8a8"])
def test_scratch_hook(dtype):
    e = 2 if dtype == "bf16" else 1
    need = lambda M, N, K: R.row_scratch_bytes(ROWS[dtype], call(dtype, M=M, N=N, K=K // e))  # noqa: E731
    assert need(1, 64, 1024) == 0
    deep = need(13, 512, 21504)
    assert deep > 0 and deep % (13 * 512 * 4) == 0
    assert need(2048, 512, 21504) <= 1 << 28


@pytest.mark.parametrize("seed", [1, 2, 3])
def test_plans_survive_mutated_operands(seed):
    rng = random.Random(seed)
    for _ in range(400):
        dtype = rng.choice(["bf16", "i8a8"])
        M, N, K = rng.choice([1, 4, 17, 64]), rng.choice([1, 17, 130, 256]), rng.choice([1, 16, 77, 384])
        keep = dict(bias=torch.zeros(N), residual=bf(M, N), y=bf(M, N))
        ops = call(dtype, M=M, N=N, K=K, **keep)
        _mutate(ops.args, rng)
        got = rc(ops, dtype)
        assert got in CODES and R.row_scratch_bytes(ROWS[dtype], ops) >= 0
        if _no_gpu():
            assert R.launch_row(ROWS[dtype], ops) == (got if got != R.RAD_OK else R.RAD_E_UNSUPPORTED)
