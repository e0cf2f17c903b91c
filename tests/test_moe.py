"""The moe_layer row on the host: table, resolver, what the plan takes and what it refuses."""
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
ROW = "moe_layer"
bf = lambda *s: torch.zeros(*s, dtype=torch.bfloat16)  # noqa: E731


def aligned(shape, dtype):
    """Zeros on a 16-byte boundary."""
    n = 1
    for s in shape:
        n *= s
    size = torch.empty(0, dtype=dtype).element_size()
    buf = torch.zeros(n * size + 16, dtype=torch.uint8)
    return buf[-buf.data_ptr() % 16:][:n * size].view(dtype).view(shape)


def call(dtype="bf16", M=4, n=64, f=96, E=8, top_k=2, scratch=True, **kw):
    code = {"bf16": torch.bfloat16, "i8": torch.int8, "mxfp4": torch.uint8}[dtype]
    half = 2 if dtype == "mxfp4" else 1
    t = dict(x=aligned((M, n), torch.bfloat16), logits=torch.zeros(M, E), gate_up=aligned((E, 2 * f, n // half), code),
             down=aligned((E, n, f // half), code), y=bf(M, n), gate_up_scale=None, down_scale=None, ids=None, weights=None)
    if dtype == "i8":
        t.update(gate_up_scale=torch.ones(E, 2 * f), down_scale=torch.ones(E, n))
    if dtype == "mxfp4":
        t.update(gate_up_scale=torch.zeros(E, 2 * f, n // 32, dtype=torch.uint8),
                 down_scale=torch.zeros(E, n, f // 32, dtype=torch.uint8))
    par = dict(dtype=dtype, n=n, f=f, E=E, top_k=top_k)
    for k, v in kw.items():
        (t if k in t else par)[k] = v
    ops = R.MoeLayerOperands(t.pop("x"), t.pop("logits"), t.pop("gate_up"), t.pop("down"), t.pop("y"), **t, **par)
    if scratch:
        ops.args.scratch, ops.args.scratch_bytes = 1 << 20, R.row_scratch_bytes(ROW, ops)
    return ops


def rc(*a, **kw):
    return R.describe(ROW, call(*a, **kw))[0]


def test_table_resolution_and_switch():
    assert ROW in {r["name"] for r in R.ext_rows()} and ROW in [s["op"] for s in R.ext_schemas()]
    for d in ("bf16", "i8", "mxfp4"):
        assert R.resolve(ROW, dict(dtype=d, M=64))["name"] == ROW
    assert R.resolve(ROW, dict(dtype="i8", M=65)) is None and R.resolve(ROW, dict(dtype="fp8", M=1)) is None
    script = ("import sys, json; sys.path.insert(0, %r); import libr3d_amd as R; "
              "print(json.dumps([r['name'] for r in R.ext_rows()]))" % ROOT)
    out = subprocess.run([sys.executable, "-c", script], env=dict(os.environ, R3D_NO_MOE="1"), capture_output=True,
                         text=True, timeout=120, check=True)
    assert set(json.loads(out.stdout)) == {r["name"] for r in R.ext_rows()} - {ROW}


@pytest.mark.parametrize("dtype", ["bf16", "i8", "mxfp4"])
def test_accepts(dtype):
    ok = lambda **kw: rc(dtype, **kw) == R.RAD_OK  # noqa: E731
    i32 = torch.zeros(4, 2, dtype=torch.int32)
    assert ok() and ok(M=64) and ok(M=1, E=1, top_k=1, n=32, f=32) and ok(E=512, top_k=16)
    assert ok(y=torch.zeros(4, 64)) and ok(logits=bf(4, 8)) and ok(logits=torch.zeros(4, 20)[:, :8])
    assert ok(ids=i32, weights=torch.zeros(4, 2)) and ok(ids=torch.zeros(4, 5, dtype=torch.int32)[:, :2])
    for a in ("silu", "gelu", "gelu_tanh", "relu", "sigmoid", "none"):
        assert ok(act=a)
    assert ok(score="sigmoid", renorm=0, weight_scale=2.5)
    assert ok(x=aligned((4, 128), torch.bfloat16)[:, :64]) and ok(x=aligned((1, 64), torch.bfloat16).expand(4, 64))
    assert ok(y=bf(4, 100)[:, :64]) and ok(y=bf(2, 2, 64))
    if dtype == "i8":
        assert ok(gate_up_scale=torch.ones(8, 192, 1), down_scale=torch.ones(1, 64).expand(8, 64))


@pytest.mark.parametrize("dtype", ["bf16", "i8", "mxfp4"])
def test_refuses(dtype):
    got = lambda **kw: rc(dtype, **kw)  # noqa: E731
    code = {"bf16": torch.bfloat16, "i8": torch.int8, "mxfp4": torch.uint8}[dtype]
    half = 2 if dtype == "mxfp4" else 1
    wide = aligned((8, 192, 128 // half), code)
    assert R.describe(ROW, call(dtype, gate_up=wide[:, :, :64 // half]))[0] == R.RAD_OK
    assert got(scratch=False) == R.RAD_E_UNSUPPORTED
    ops = call(dtype)
    ops.args.scratch_bytes -= 1
    assert R.describe(ROW, ops)[0] == R.RAD_E_UNSUPPORTED
    ops = call(dtype)
    ops.args.scratch += 8
    assert R.describe(ROW, ops)[0] == R.RAD_E_UNSUPPORTED
    for i in (0, 1, 2, 4, 6):
        ops = call(dtype)
        ops._t[i].data = None
        assert R.describe(ROW, ops)[0] == R.RAD_E_INVAL
    assert got(M=65) == got(E=513, top_k=1) == got(E=40, top_k=17) == R.RAD_E_UNSUPPORTED
    assert got(act="tanh") == got(score="topk") == R.RAD_E_UNSUPPORTED
    assert got(top_k=9) == got(top_k=0) == got(logits=torch.zeros(4, 7)) == got(logits=torch.zeros(3, 8)) == R.RAD_E_SHAPE
    assert got(x=aligned((3, 64), torch.bfloat16)) == got(y=bf(4, 63)) == R.RAD_E_SHAPE
    assert got(gate_up=aligned((8, 96, 64 // half), code)) == got(down=aligned((7, 64, 96 // half), code)) == R.RAD_E_SHAPE
    assert got(ids=torch.zeros(4, 1, dtype=torch.int32)) == got(weights=torch.zeros(3, 2)) == R.RAD_E_SHAPE
    odd = {"bf16": 68, "i8": 72, "mxfp4": 80}[dtype]
    assert got(n=odd) == got(f=odd) == R.RAD_E_UNSUPPORTED
    assert got(x=torch.zeros(4, 64)) == got(y=torch.zeros(4, 64, dtype=torch.float16)) == R.RAD_E_DTYPE
    assert got(ids=torch.zeros(4, 2, dtype=torch.int64)) == got(logits=torch.zeros(4, 8, dtype=torch.int32)) == R.RAD_E_DTYPE
    assert got(x=aligned((4, 72), torch.bfloat16)[:, 4:68]) == got(x=aligned((4, 68), torch.bfloat16)[:, :64]) == R.RAD_E_UNSUPPORTED
    assert got(y=bf(1, 64).expand(4, 64)) == got(weights=torch.zeros(1, 2).expand(4, 2)) == R.RAD_E_STRIDE
    flat = aligned((8, 192, 68 // half), code)
    assert got(gate_up=flat[:, :, 4 // half:]) == R.RAD_E_UNSUPPORTED               # off 16 bytes
    pairs = torch.zeros(4, 2)
    assert got(ids=pairs.view(torch.int32), weights=pairs) == R.RAD_E_INVAL
    lg = torch.zeros(4, 8)
    assert got(logits=lg, weights=lg[:, :2]) == R.RAD_E_INVAL
    if dtype == "bf16":
        assert got(gate_up_scale=torch.ones(8, 192)) == R.RAD_E_INVAL
        assert got(gate_up=aligned((8, 192, 64), torch.int8)) == R.RAD_E_DTYPE
    else:
        assert got(gate_up_scale=None) == got(down_scale=None) == R.RAD_E_INVAL
        assert got(down_scale=bf(8, 64)) == R.RAD_E_DTYPE
        assert got(gate_up_scale=call(dtype)._tensors[3][:7]) == R.RAD_E_SHAPE


def test_scale_rows_lie_apart():
    """A plane of one row's scales for all rows may be shorter than the four that a load takes."""
    for name, rows, K in (("gate_up_scale", 192, 64), ("down_scale", 64, 96)):
        one = torch.zeros(8, 1, K // 32, dtype=torch.uint8)
        assert rc("mxfp4", **{name: one.expand(8, rows, K // 32)}) == R.RAD_E_STRIDE
        near = torch.zeros(8 * rows * (K // 32), dtype=torch.uint8).as_strided((8, rows, K // 32), (rows, K // 32 - 1, 1))
        assert rc("mxfp4", **{name: near}) == R.RAD_E_STRIDE
        flat = torch.zeros(1, rows, K // 32, dtype=torch.uint8)
        assert rc("mxfp4", **{name: flat.expand(8, rows, K // 32)}) == R.RAD_OK        # one plane for all experts
    assert rc("i8", down_scale=torch.ones(1, 1).expand(8, 64)) == R.RAD_E_STRIDE
    assert rc("i8", down_scale=torch.ones(1, 64).expand(8, 64)) == R.RAD_OK


@pytest.mark.parametrize("dtype", ["bf16", "i8", "mxfp4"])
def test_refuses_results_over_the_experts(dtype):
    gu = call(dtype)._tensors[2]
    assert rc(dtype, gate_up=gu, y=gu.view(-1).view(torch.bfloat16)[-256:].view(4, 64)) == R.RAD_E_INVAL
    assert rc(dtype, gate_up=gu, ids=gu.view(-1).view(torch.int32)[:8].view(4, 2)) == R.RAD_E_INVAL
    dn = call(dtype)._tensors[4]
    assert rc(dtype, down=dn, weights=dn.view(-1).view(torch.float32)[64:72].view(4, 2)) == R.RAD_E_INVAL


def test_scratch_hook():
    assert R.row_scratch_bytes(ROW, call(M=4, f=96, top_k=2)) == 12304 + 4 * 2 * (96 * 2 * 2 + 64 * 4)
    assert R.row_scratch_bytes(ROW, call(M=4, f=96, top_k=2, y=torch.zeros(4, 64))) == 12304 + 4 * 2 * (96 * 2 * 3 + 64 * 4)


def test_python_call_refuses_host_tensors():
    with pytest.raises(ValueError):
        R.moe_layer(bf(2, 8), torch.zeros(2, 2), bf(2, 16, 8), bf(2, 8, 8), bf(2, 8), dtype="bf16", n=8, f=8, E=2, top_k=1)


@pytest.mark.parametrize("seed", [1, 2, 3])
def test_plans_survive_mutated_operands(seed):
    rng = random.Random(seed)
    for _ in range(400):
        M, E = rng.choice([1, 4, 17, 64]), rng.choice([1, 8, 70])
        k = min(E, rng.choice([1, 2, 8]))
        ops = call(rng.choice(["bf16", "i8", "mxfp4"]), M=M, E=E, top_k=k, n=rng.choice([32, 64, 128]),
                   f=rng.choice([32, 96]), ids=torch.zeros(M, k, dtype=torch.int32), weights=torch.zeros(M, k))
        _mutate(ops.args, rng)
        got = R.describe(ROW, ops)[0]
        assert got in CODES and R.row_scratch_bytes(ROW, ops) >= 0
        if _no_gpu():
            assert R.launch_row(ROW, ops) == (got if got != R.RAD_OK else R.RAD_E_UNSUPPORTED)
