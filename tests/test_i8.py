"""The int8 rows on the CPU: the second row table, resolution, and every refusal that the plans
make, through describe (which launches nothing) over host tensors."""
import json
import os
import subprocess
import sys

import pytest
import torch

import libr3d_amd as R

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
INT8 = {"gemm_nt_q_i8a8", "gemm_nt_q_i8a8_decode", "quant_act_i8", "gated_quant_i8",
        "rmsnorm_quant_i8"}


def gemm(M=4, N=48, K=64, **kw):
    t = dict(a=torch.zeros(M, K, dtype=torch.int8), a_scale=torch.ones(M),
             b=torch.zeros(N, K, dtype=torch.int8), b_scale=torch.ones(N, 1),
             y=torch.zeros(M, N, dtype=torch.bfloat16))
    par = dict(dtype="i8a8", N=N, K=K, M=M)
    for k, v in kw.items():
        (t if k in t else par)[k] = v
    return R.GemmOperands(t["a"], t["a_scale"], t["b"], t["b_scale"], t["y"], **par)


def rc(row, ops):
    return R.describe(row, ops)[0]


def test_table_and_resolution():
    rows = {r["name"]: r for r in R.ext_rows()}
    assert INT8 <= set(rows)
    assert not set(rows) & {r["name"] for r in R.rows()}
    ops = [s["op"] for s in R.ext_schemas()]
    assert {"quant_act_i8", "gated_quant_i8", "rmsnorm_quant_i8"} <= set(ops)
    assert not set(ops) & {s["op"] for s in R.schemas()}
    known = set(ops) | {s["op"] for s in R.schemas()}
    assert all(r["op"] in known and r["launch"] for r in rows.values())
    q = lambda **kw: (R.resolve("gemm_nt_q", dict(dict(dtype="i8a8", N=64, K=64, group=64), **kw)) or {}).get("name")
    assert q(M=1) == q(M=16) == "gemm_nt_q_i8a8_decode"
    assert q(M=17) == "gemm_nt_q_i8a8"
    assert q(M=4, K=77, group=77) == "gemm_nt_q_i8a8_decode"
    assert R.resolve("rmsnorm_quant_i8", dict(M=1, n=7, eps=1e-6, dtype="bf16"))["name"] == "rmsnorm_quant_i8"
    assert R.resolve("rmsnorm_quant_i8", dict(M=1, n=7, eps=1e-6, dtype="f32")) is None
    assert R.resolve("quant_act_i8", dict(M=1, n=7, dtype="f32"))["name"] == "quant_act_i8"
    assert R.resolve("gated_quant_i8", dict(M=1, n=0, dtype="f32")) is None


@pytest.mark.parametrize("env,gone", [("R3D_NO_I8", INT8), ("R3D_NO_I8_DEC", {"gemm_nt_q_i8a8_decode"})])
def test_kill_switches_hide_rows(env, gone):
    script = ("import sys, json; sys.path.insert(0, %r); import libr3d_amd as R; "
              "print(json.dumps([[r['name'] for r in R.ext_rows()], len(R.rows())]))" % ROOT)
    out = subprocess.run([sys.executable, "-c", script], env=dict(os.environ, **{env: "1"}),
                         capture_output=True, text=True, timeout=120, check=True)
    names, n = json.loads(out.stdout)
    assert n == len(R.rows()) and set(names) == {r["name"] for r in R.ext_rows()} - gone


def test_gemm_accepts():
    for row in ("gemm_nt_q_i8a8", "gemm_nt_q_i8a8_decode"):
        assert rc(row, gemm()) == R.RAD_OK
        assert rc(row, gemm(M=1, N=1, K=1)) == R.RAD_OK
        assert rc(row, gemm(a_scale=torch.ones(4, 1), b_scale=torch.ones(48))) == R.RAD_OK
        assert rc(row, gemm(a_scale=torch.ones(1).expand(4), b_scale=torch.ones(1, 1).expand(48, 1))) == R.RAD_OK
        assert rc(row, gemm(a=torch.zeros(4, 99, dtype=torch.int8)[:, :64])) == R.RAD_OK
        assert rc(row, gemm(y=torch.zeros(2, 2, 48, dtype=torch.bfloat16))) == R.RAD_OK
    assert rc("gemm_nt_q_i8a8", gemm(M=17)) == R.RAD_OK


def test_gemm_refuses():
    row = "gemm_nt_q_i8a8"
    i8 = lambda *s: torch.zeros(*s, dtype=torch.int8)  # noqa: E731
    assert rc("gemm_nt_q_i8a8_decode", gemm(M=17)) == R.RAD_E_UNSUPPORTED
    assert rc(row, gemm(a=None)) == R.RAD_E_UNSUPPORTED
    assert rc(row, gemm(a_scale=None)) == R.RAD_E_UNSUPPORTED
    assert rc(row, gemm(a_sum=torch.ones(4))) == R.RAD_E_UNSUPPORTED
    assert rc(row, gemm(b_ref=torch.ones(4, dtype=torch.bfloat16))) == R.RAD_E_UNSUPPORTED
    for dtype in ("fp8a8", "mxfp4a8"):
        ops = gemm()
        ops._p[0].sval = dtype.encode()
        assert rc(row, ops) == R.RAD_E_UNSUPPORTED
    assert rc(row, gemm(extra_params=[("pb1", 1)])) == R.RAD_E_UNSUPPORTED
    for i, dt in ((0, "U8"), (1, "BF16"), (2, "F8E4M3"), (3, "F16"), (4, "F32")):
        ops = gemm()
        ops._t[i].dtype = R.DT[dt]
        assert rc(row, ops) == R.RAD_E_UNSUPPORTED, i
    assert rc(row, gemm(group=32)) == R.RAD_E_SHAPE
    for i, v in ((1, 0), (1, -48), (2, 0), (2, -1), (1, 1 << 40)):
        ops = gemm()
        ops._p[i].ival = v
        assert rc(row, ops) == R.RAD_E_SHAPE
    assert rc(row, gemm(K=131072, a=i8(4, 131072), b=i8(1, 131072).expand(48, -1))) == R.RAD_E_UNSUPPORTED
    assert rc(row, gemm(y=torch.zeros(4, 47, dtype=torch.bfloat16))) == R.RAD_E_SHAPE
    assert rc(row, gemm(y=torch.zeros(0, 48, dtype=torch.bfloat16))) != R.RAD_OK
    assert rc(row, gemm(a=i8(3, 64))) == R.RAD_E_SHAPE
    assert rc(row, gemm(a=i8(4, 63))) == R.RAD_E_SHAPE
    assert rc(row, gemm(b=i8(47, 64))) == R.RAD_E_SHAPE
    assert rc(row, gemm(a_scale=torch.ones(3))) == R.RAD_E_SHAPE
    assert rc(row, gemm(a_scale=torch.ones(4, 2))) == R.RAD_E_SHAPE
    assert rc(row, gemm(b_scale=torch.ones(1, 48))) == R.RAD_E_SHAPE
    assert rc(row, gemm(a=i8(64, 4).T)) == R.RAD_E_STRIDE
    assert rc(row, gemm(y=torch.zeros(48, 4, dtype=torch.bfloat16).T)) == R.RAD_E_STRIDE
    assert rc(row, gemm(y=torch.zeros(48, dtype=torch.bfloat16).expand(4, 48))) == R.RAD_E_STRIDE
    ops = gemm()
    ops._t[2].stride[0] = 1 << 27                     # 16 rows past 32-bit offsets
    assert rc(row, ops) == R.RAD_E_UNSUPPORTED
    ops._t[2].stride[0] = -64
    assert rc(row, ops) == R.RAD_E_STRIDE
    ops = gemm()
    ops._t[4].rank = 9
    assert rc(row, ops) == R.RAD_E_UNSUPPORTED


def band(op, M=3, n=20, **kw):
    bf = lambda *s: torch.zeros(*s, dtype=torch.bfloat16)  # noqa: E731
    t = dict(x=bf(M, 2 * n if op == "gated" else n), q=torch.zeros(M, n, dtype=torch.int8),
             scale=torch.zeros(M), out=None, residual=None, residual_out=None, w=bf(n))
    par = dict(n=n, M=M)
    for k, v in kw.items():
        (t if k in t else par)[k] = v
    if op == "quant":
        return "quant_act_i8", R.QuantActI8Operands(t["x"], t["q"], t["scale"], **par)
    if op == "gated":
        return "gated_quant_i8", R.GatedQuantI8Operands(t["x"], t["q"], t["scale"], t["out"], **par)
    return "rmsnorm_quant_i8", R.RmsNormQuantI8Operands(
        t["x"], t["residual"], t["w"], t["q"], t["scale"], t["out"], residual_out=t["residual_out"], **par)


@pytest.mark.parametrize("op", ["quant", "gated", "norm"])
def test_band_refusals(op):
    bf = lambda *s: torch.zeros(*s, dtype=torch.bfloat16)  # noqa: E731
    w = 2 if op == "gated" else 1
    ok = lambda **kw: rc(*band(op, **kw))  # noqa: E731
    assert ok() == ok(M=1, n=1) == ok(scale=torch.zeros(3, 1)) == R.RAD_OK
    assert ok(x=bf(3, 99)[:, :20 * w]) == R.RAD_OK
    assert ok(x=torch.zeros(3, 20 * w)) == (R.RAD_E_DTYPE if op == "norm" else R.RAD_OK)
    assert ok(q=bf(3, 20)) == ok(scale=bf(3)) == R.RAD_E_DTYPE
    row, ops = band(op)
    ops._t[3 if op == "norm" else 1].dtype = R.DT["U8"]
    assert rc(row, ops) == R.RAD_E_DTYPE
    row, ops = band(op)
    ops._t[4 if op == "norm" else 2].dtype = R.DT["BF16"]
    assert rc(row, ops) == R.RAD_E_DTYPE
    for v in (0, -1, 19, 1 << 40):
        row, ops = band(op)
        ops._p[0].ival = v
        assert rc(row, ops) == R.RAD_E_SHAPE
    assert ok(x=bf(0, 20 * w)) != R.RAD_OK
    assert ok(q=torch.zeros(2, 20, dtype=torch.int8)) == R.RAD_E_SHAPE
    assert ok(q=torch.zeros(20, 3, dtype=torch.int8).T) == R.RAD_E_STRIDE
    assert ok(q=torch.zeros(20, dtype=torch.int8).expand(3, 20)) == R.RAD_E_STRIDE
    assert ok(scale=torch.zeros(2)) == R.RAD_E_SHAPE
    assert ok(scale=torch.zeros(3, 2)) == R.RAD_E_SHAPE
    assert ok(scale=torch.zeros(1).expand(3)) == R.RAD_E_STRIDE
    assert ok(x=bf(20 * w, 3).T) == R.RAD_E_STRIDE
    row, ops = band(op)
    ops._t[0].data += 1                               # an odd address of bf16
    assert rc(row, ops) == R.RAD_E_STRIDE
    if op == "gated":
        assert ok(act="silu") == ok(act="sigmoid") == R.RAD_OK
        assert ok(act="gelu") == R.RAD_E_UNSUPPORTED
        assert ok(out=bf(3, 20)) == ok(out=torch.zeros(3, 20)) == R.RAD_OK
        assert ok(out=bf(3, 19)) == R.RAD_E_SHAPE
    if op == "norm":
        assert ok(residual=bf(3, 20)) == ok(residual=bf(3, 20), residual_out=bf(3, 20)) == R.RAD_OK
        assert ok(residual_out=bf(3, 20)) == R.RAD_E_INVAL            # nothing to add
        assert ok(residual=torch.zeros(3, 21, dtype=torch.bfloat16)) == R.RAD_E_SHAPE
        assert ok(w=bf(21)) == ok(w=bf(1, 20)) == R.RAD_E_SHAPE
        assert ok(w=torch.zeros(20)) == R.RAD_OK
        assert ok(eps=-1.0) == ok(eps=float("nan")) == R.RAD_E_INVAL
        row, ops = band(op, residual=bf(3, 20))
        ops._t[6].data = None
        assert rc(row, ops) == R.RAD_E_INVAL


def test_entries_match_describe_without_a_gpu():
    """The launch pointers refuse what describe refuses, and stop at the chip gate otherwise."""
    if torch.cuda.is_available():
        pytest.skip("host tensors must not reach a kernel")
    assert R.launch_row("gemm_nt_q_i8a8", gemm(group=32)) == R.RAD_E_SHAPE
    assert R.launch_row("gemm_nt_q_i8a8", gemm()) == R.RAD_E_UNSUPPORTED
    row, ops = band("quant")
    ops._p[0].ival = 0
    assert R.launch_row(row, ops) == R.RAD_E_SHAPE
    assert R.launch_row(*band("norm")) == R.RAD_E_UNSUPPORTED
