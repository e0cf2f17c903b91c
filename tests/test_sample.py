"""The sample_logits row on the CPU: its registration, its scratch hook, and what its plan refuses
(through describe, which launches nothing, over host tensors)."""
import os
import subprocess
import sys

import pytest
import torch

import libr3d_amd as R

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
ROW = "sample_logits"


def ops(M=3, V=50, **kw):
    t = dict(logits=torch.zeros(M, V), u=torch.zeros(M), token=torch.zeros(M, dtype=torch.int32), prob=None,
             temperature=None, top_k=None, top_p=None, min_p=None)
    par = dict(n_vocab=V, M=M)
    for k, v in kw.items():
        (t if k in t else par)[k] = v
    return R.SampleOperands(t["logits"], t["u"], t["token"], t["prob"], temperature=t["temperature"],
                            top_k=t["top_k"], top_p=t["top_p"], min_p=t["min_p"], **par)


def rc(**kw):
    return R.describe(ROW, ops(**kw))[0]


def test_registered():
    row = {r["name"]: r for r in R.ext_rows()}[ROW]
    assert row["op"] == ROW and row["launch"] and row["scratch"]
    assert R.resolve(ROW, dict(M=1, n_vocab=10, dtype="bf16"))["name"] == ROW
    assert R.resolve(ROW, dict(M=1, n_vocab=10, dtype="f16")) is None
    s = {s["op"]: s for s in R.ext_schemas()}[ROW]
    assert [o[0] for o in s["operands"]] == ["logits", "u", "temperature", "top_k", "top_p", "min_p", "token", "prob"]
    out = subprocess.run([sys.executable, "-c", "import sys; sys.path.insert(0, %r); import libr3d_amd as R; "
                          "print([r['name'] for r in R.ext_rows()])" % ROOT],
                         env=dict(os.environ, R3D_NO_SAMPLE="1"), capture_output=True, text=True, timeout=120, check=True)
    assert ROW not in out.stdout and "quant_act_i8" in out.stdout


def test_accepts():
    f, i = torch.ones(3), torch.ones(3, dtype=torch.int32)
    assert rc() == rc(M=1, V=1) == R.RAD_OK
    assert rc(logits=torch.zeros(3, 50, dtype=torch.bfloat16)) == R.RAD_OK
    assert rc(logits=torch.zeros(3, 99)[:, :50]) == rc(logits=torch.zeros(50).expand(3, 50)) == R.RAD_OK
    assert rc(temperature=f, top_k=i, top_p=f[:, None], min_p=f, prob=f) == R.RAD_OK
    assert rc(temperature=torch.ones(1).expand(3), u=torch.ones(1, 1).expand(3, 1)) == R.RAD_OK
    assert rc(token=torch.zeros(3, 2, dtype=torch.int32)[:, 0]) == R.RAD_OK


def test_refuses():
    f, i = torch.ones(3), torch.ones(3, dtype=torch.int32)
    for name in ("logits", "u", "token"):
        o = ops()
        o._t[{"logits": 0, "u": 1, "token": 6}[name]].data = None
        assert R.describe(ROW, o)[0] == R.RAD_E_INVAL
    for at, dt in ((0, "F16"), (1, "BF16"), (2, "BF16"), (3, "I64"), (4, "F16"), (5, "I32"), (6, "I64"), (7, "BF16")):
        o = ops(temperature=f, top_k=i, top_p=f, min_p=f, prob=f)
        o._t[at].dtype = R.DT[dt]
        assert R.describe(ROW, o)[0] == R.RAD_E_DTYPE, at
    assert rc(token=torch.zeros(3, dtype=torch.int64)) == rc(top_k=f) == R.RAD_E_DTYPE
    for v in (0, -1, 49, (1 << 22) + 1, 1 << 40):
        o = ops()
        o._p[0].ival = v
        assert R.describe(ROW, o)[0] == R.RAD_E_SHAPE
    assert rc(logits=torch.zeros(1).expand(65536, 1), V=1, u=torch.zeros(1).expand(65536),
              token=torch.zeros(65536, dtype=torch.int32)) == R.RAD_E_SHAPE
    for name in ("u", "temperature", "top_p", "min_p", "prob"):
        assert rc(**{name: torch.ones(2)}) == rc(**{name: torch.ones(3, 2)}) == R.RAD_E_SHAPE
    assert rc(top_k=i[:2]) == rc(token=i[:2]) == R.RAD_E_SHAPE
    assert rc(token=torch.zeros(1, dtype=torch.int32).expand(3)) == rc(prob=torch.zeros(1).expand(3)) == R.RAD_E_STRIDE
    assert rc(logits=torch.zeros(50, 3).T) == R.RAD_E_STRIDE
    o = ops()
    o._t[0].data += 2
    assert R.describe(ROW, o)[0] == R.RAD_E_STRIDE
    o = ops()
    o._p[1].sval = b"bf16"                          # contradicts the operand
    assert R.describe(ROW, o)[0] == R.RAD_E_DTYPE


def test_scratch_hook():
    one = R.row_scratch_bytes(ROW, ops(M=1, V=4096))
    assert one > 0 and one % 8 == 0
    assert R.row_scratch_bytes(ROW, ops(M=7, V=4096)) == 7 * one
    assert R.row_scratch_bytes(ROW, ops(M=1, V=4097)) == one + 8 + 64 + 256
    o = ops()
    o._p[0].ival = 1 << 40
    assert R.row_scratch_bytes(ROW, o) == 0
    if torch.cuda.is_available():
        pytest.skip("host tensors must not reach a kernel")
    o = ops()
    assert R.launch_row(ROW, o) == R.RAD_E_UNSUPPORTED          # no scratch
