"""The rmsnorm_block row on the host: table, resolver, what the plan takes and what it refuses."""
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
ROW = "rmsnorm_block"
bf = lambda *s: torch.zeros(*s, dtype=torch.bfloat16)  # noqa: E731


def call(M=4, n=64, **kw):
    t = dict(x=bf(M, n), residual=bf(M, n), w_post=bf(n), gate=bf(n), w_pre=bf(n), residual_out=bf(M, n), out=bf(M, n),
             q=None, scale=None)
    par = dict(n=n)
    for k, v in kw.items():
        (t if k in t else par)[k] = v
    return R.RmsNormBlockOperands(t.pop("x"), **t, **par)


def rc(**kw):
    return R.describe(ROW, call(**kw))[0]


def test_table_resolution_and_switch():
    assert ROW in {r["name"] for r in R.ext_rows()} and ROW in [s["op"] for s in R.ext_schemas()]
    assert R.resolve(ROW, dict(M=1, n=7, eps=1e-6, dtype="f32"))["name"] == ROW
    assert R.resolve(ROW, dict(M=1, n=0, eps=1e-6, dtype="f32")) is None
    script = ("import sys, json; sys.path.insert(0, %r); import libr3d_amd as R; "
              "print(json.dumps([r['name'] for r in R.ext_rows()]))" % ROOT)
    out = subprocess.run([sys.executable, "-c", script], env=dict(os.environ, R3D_NO_BLOCK_NORM="1"), capture_output=True,
                         text=True, timeout=120, check=True)
    assert set(json.loads(out.stdout)) == {r["name"] for r in R.ext_rows()} - {ROW}


def test_accepts():
    ok = lambda **kw: rc(**kw) == R.RAD_OK  # noqa: E731
    assert ok() and ok(M=1, n=1, gate=None) and ok(n=32768) and ok(x=torch.zeros(4, 64))
    assert ok(residual=None) and ok(w_post=None) and ok(gate=None) and ok(residual_out=None)
    assert ok(w_pre=None, out=None)
    assert ok(gate=bf(4, 1)) and ok(gate=bf(4, 64)) and ok(gate=bf(1, 64).expand(4, 64)) and ok(gate=bf(1, 1).expand(4, 1))
    f = torch.zeros
    assert ok(w_post=f(64), gate=f(4, 1), w_pre=f(64)) and ok(out=f(4, 64))
    assert ok(q=torch.zeros(4, 64, dtype=torch.int8), scale=f(4)) and ok(q=torch.zeros(4, 64, dtype=torch.uint8), scale=f(4, 1))
    assert ok(n=130, q=torch.zeros(4, 130, dtype=torch.uint8), scale=f(4, 2), out=None)
    x, r = bf(4, 64), bf(4, 64)
    assert ok(residual=r, residual_out=r) and ok(x=x, residual_out=x) and ok(x=x, residual=r, residual_out=r, out=x)
    wide = bf(4, 192)
    assert ok(x=wide[:, :64], residual=wide[:, 64:128], residual_out=wide[:, 64:128], out=wide[:, 128:])
    assert ok(group=64) and ok(q=torch.zeros(4, 64, dtype=torch.uint8), scale=f(4, 1), group=128)


def test_refuses():
    f = torch.zeros
    q8, u8 = torch.zeros(4, 64, dtype=torch.int8), torch.zeros(4, 64, dtype=torch.uint8)
    assert rc(q=q8) == rc(scale=f(4)) == R.RAD_E_INVAL
    assert rc(residual_out=None, out=None) == rc(w_pre=None) == rc(out=None) == R.RAD_E_INVAL
    assert rc(x=f(4, 64, dtype=torch.float16)) == rc(residual=f(4, 64)) == rc(residual_out=f(4, 64)) == R.RAD_E_DTYPE
    assert rc(w_post=f(64)) == rc(gate=f(64)) == rc(q=q8, scale=bf(4)) == rc(out=q8) == R.RAD_E_DTYPE
    assert rc(q=torch.zeros(4, 64, dtype=torch.int32), scale=f(4)) == R.RAD_E_DTYPE
    assert rc(n=32769) == R.RAD_E_UNSUPPORTED
    assert rc(group=32) == rc(q=u8, scale=f(4, 1), group=64) == R.RAD_E_UNSUPPORTED
    assert rc(x=bf(4, 63)) == rc(residual=bf(3, 64)) == rc(w_post=bf(63)) == rc(gate=bf(63)) == rc(gate=bf(3, 1)) == R.RAD_E_SHAPE
    assert rc(gate=bf(3, 64)) == rc(out=bf(4, 65)) == rc(q=q8, scale=f(3)) == R.RAD_E_SHAPE
    assert rc(n=130, q=torch.zeros(4, 130, dtype=torch.uint8), scale=f(4, 1)) == R.RAD_E_SHAPE
    assert rc(x=bf(4, 128)[:, ::2]) == rc(w_pre=bf(128)[::2]) == rc(gate=bf(128)[::2]) == R.RAD_E_STRIDE
    assert rc(residual_out=bf(1, 64).expand(4, 64)) == rc(out=bf(1, 64).expand(4, 64)) == R.RAD_E_STRIDE
    assert rc(q=q8, scale=f(1).expand(4)) == R.RAD_E_STRIDE
    assert rc(eps=-1.0) == rc(eps=float("nan")) == R.RAD_E_INVAL
    flat = bf(600)
    a, b = flat[:256].view(4, 64), flat[8:264].view(4, 64)
    assert rc(x=a, residual_out=b) == rc(residual=a, residual_out=b) == rc(residual=a, out=b) == R.RAD_E_INVAL
    assert rc(gate=a, out=b) == rc(residual_out=a, out=a) == rc(residual_out=a, out=b) == R.RAD_E_INVAL
    assert rc(w_pre=flat[:64], residual_out=a) == rc(w_post=flat[:64], out=a) == R.RAD_E_INVAL
    assert rc(x=f(4, 64), out=None, w_pre=None, residual_out=f(4, 64).view(torch.bfloat16)[:, :64]) == R.RAD_OK
    x = f(4, 64)
    assert rc(x=x, residual_out=x.view(torch.bfloat16)[:, :64]) == R.RAD_E_INVAL          # the same memory, another type


def test_python_call_refuses_host_tensors():
    with pytest.raises(ValueError):
        R.rmsnorm_block(bf(2, 8), n=8, w_pre=bf(8), out=bf(2, 8))


@pytest.mark.parametrize("seed", [1, 2, 3])
def test_plans_survive_mutated_operands(seed):
    rng = random.Random(seed)
    for _ in range(500):
        M, n = rng.choice([1, 2, 4, 17]), rng.choice([1, 4, 33, 128, 1000])
        kw = dict(gate=rng.choice([None, bf(n), bf(M, 1), bf(M, n)]))
        if rng.random() < 0.5:
            kw.update(q=torch.zeros(M, n, dtype=torch.int8), scale=torch.ones(M))
        ops = call(M=M, n=n, **kw)
        _mutate(ops.args, rng)
        got = R.describe(ROW, ops)[0]
        assert got in CODES and R.row_scratch_bytes(ROW, ops) == 0
        if _no_gpu():
            assert R.launch_row(ROW, ops) == (got if got != R.RAD_OK else R.RAD_E_UNSUPPORTED)
