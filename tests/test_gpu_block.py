"""rmsnorm_block on the GPU against 64 bits, element by element, in guarded memory."""
import pytest
import torch

import libr3d_amd as R
from tests import block_util as B
from tests.test_gpu_i8 import Box

pytestmark = pytest.mark.gpu
KIND = {"bf16": torch.bfloat16, "f32": torch.float32}


def inputs(M, n, x="bf16", w="bf16", gate="channel", post=True, residual=True, seed=0):
    g = torch.Generator().manual_seed(seed * 1000003 + M * 7919 + n)
    r = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    shape = {"channel": (n,), "token": (M, 1), "full": (M, n), "none": None}[gate]
    return dict(x=(r(M, n) * torch.exp(r(M, 1))).to(KIND[x]), residual=(3 * r(M, n)).bfloat16() if residual else None,
                w_post=(1 + 0.2 * r(n)).to(KIND[w]) if post else None,
                gate=None if shape is None else (0.6 + 0.3 * r(*shape)).to(KIND[w]), w_pre=(1 + 0.2 * r(n)).to(KIND[w]))


def run(dev, M, n, out="bf16", codes=None, offs=(0,) * 6, pad=(0,) * 6, pre=True, res_out=True, wadd=None, res_scale=None,
        eps=1e-6, data=None, **kw):
    t = data or inputs(M, n, **kw)
    if not pre:
        t["w_pre"] = None
    on = lambda v: None if v is None else v.to(dev)  # noqa: E731
    X = Box(t["x"], dev, offs[0], n + pad[0])
    Rs = None if t["residual"] is None else Box(t["residual"], dev, offs[1], n + pad[1])
    gate = t["gate"]
    G = None if gate is None or gate.shape != (M, n) else Box(gate, dev, offs[2], n + pad[2])
    new = lambda kind, i, cols=n: Box(torch.full((M, cols), -7, dtype=kind), dev, offs[i], cols + pad[i])  # noqa: E731
    H = new(torch.bfloat16, 3) if res_out else None
    O = new(KIND[out], 4) if out and pre else None
    Q = S = None
    if codes and pre:
        Q = new(torch.int8 if codes == "i8" else torch.uint8, 5) if codes == "i8" else Box(
            torch.full((M, n), 7, dtype=torch.uint8), dev, offs[5], n + pad[5])
        S = Box(torch.full((M, 1 if codes == "i8" else (n + 127) // 128), -7.0), dev, 0, (1 if codes == "i8" else (n + 127) // 128) + 1)
    of = lambda b: None if b is None else b.t  # noqa: E731
    ops = R.RmsNormBlockOperands(X.t, n=n, residual=of(Rs), w_post=on(t["w_post"]), gate=G.t if G else on(gate),
                                 w_pre=on(t["w_pre"]), residual_out=of(H), out=of(O), q=of(Q), scale=of(S), eps=eps, wadd=wadd,
                                 res_scale=res_scale)
    print(R.describe("rmsnorm_block", ops)[1], offs, pad, flush=True)
    assert R.launch_row("rmsnorm_block", ops, torch.cuda.current_stream().cuda_stream) == R.RAD_OK
    torch.cuda.synchronize()
    d = {k: on(v) for k, v in t.items()}
    h, eh, v, ev = B.exact(**d, eps=eps, wadd=wadd or 0.0, res_scale=1.0 if res_scale is None else res_scale)
    if H:
        B.check("residual_out", H.t, h, eh)
    if O:
        B.check("out", O.t, v, ev)
    if Q:
        (B.check_i8 if codes == "i8" else B.check_e4m3)(Q.t, S.t, v, ev)
    assert all(b.around() for b in (X, Rs, G, H, O, Q, S) if b)


@pytest.mark.parametrize("n", [1, 2, 7, 8, 9, 63, 64, 100, 127, 128, 129, 511, 512, 1000, 2047, 2560, 4097, 5376, 6151, 8192,
                               12295, 16384, 21504, 30001, 32768])
def test_widths(gpu, n):
    for codes, out in ((None, "bf16"), ("i8", None), ("e4m3", "f32")):
        run(gpu, 3, n, out=out, codes=codes)


@pytest.mark.parametrize("M,n", [(1, 5376), (2, 5376), (333, 5376), (2048, 5376), (1030, 2305), (5000, 256), (700, 16384),
                                 (300, 32768), (400, 21504), (20000, 40)])
def test_rows(gpu, M, n):
    run(gpu, M, n, codes="i8")
    run(gpu, M, n, x="f32", w="f32", gate="token", codes="e4m3", out=None)


@pytest.mark.parametrize("x", ["bf16", "f32"])
@pytest.mark.parametrize("w", ["bf16", "f32"])
@pytest.mark.parametrize("gate", ["none", "channel", "token", "full"])
def test_operands(gpu, x, w, gate):
    for post in (True, False):
        for residual in (True, False):
            run(gpu, 5, 1000, x=x, w=w, gate=gate, post=post, residual=residual, out="f32", codes="i8")
            run(gpu, 3, 777, x=x, w=w, gate=gate, post=post, residual=residual, res_out=False, codes="e4m3", out=None)
    run(gpu, 4, 1000, x=x, w=w, gate=gate, pre=False)


def test_parameters(gpu):
    run(gpu, 6, 1000, wadd=1.0, res_scale=0.875, eps=1e-5, codes="i8")
    run(gpu, 6, 1000, wadd=0.3, res_scale=-1.7, eps=0.0)
    run(gpu, 6, 1000, res_scale=0.0, gate="full", codes="e4m3")


@pytest.mark.parametrize("offs,pad", [((1, 0, 0, 0, 0, 0), (0,) * 6), ((0, 1, 3, 5, 7, 1), (3, 1, 5, 7, 1, 9)),
                                      ((3, 2, 1, 1, 2, 3), (8, 16, 24, 8, 16, 8)), ((8, 8, 8, 8, 8, 16), (1, 1, 1, 1, 1, 1))])
def test_alignment(gpu, offs, pad):
    for n in (512, 1001, 5376):
        run(gpu, 4, n, gate="full", offs=offs, pad=pad, codes="i8", out="bf16")
        run(gpu, 4, n, gate="full", offs=offs, pad=pad, codes="e4m3", out="f32", x="f32", w="f32")


def test_in_place(gpu):
    """residual_out over the residual, x or a full gate, and out over x: each as with memory of its own."""
    for M, n in ((1, 5376), (300, 2001), (7, 21504)):
        t = {k: v.to(gpu) for k, v in inputs(M, n, gate="full").items()}
        want = [torch.empty(M, n, dtype=torch.bfloat16, device=gpu) for _ in range(2)]
        assert R.rmsnorm_block(n=n, residual_out=want[0], out=want[1], **t) == R.RAD_OK
        for ro, o in (("residual", None), ("x", None), ("gate", None), ("residual", "x"), ("x", "gate"), (None, "residual")):
            u = {k: v.clone() for k, v in t.items()}
            h = u[ro] if ro else torch.empty_like(want[0])
            v = u[o] if o else torch.empty_like(want[0])
            assert R.rmsnorm_block(n=n, residual_out=h, out=v, **u) == R.RAD_OK
            torch.cuda.synchronize()
            assert torch.equal(h, want[0]) and torch.equal(v, want[1])


def test_broadcast_rows(gpu):
    M, n = 40, 700
    t = inputs(M, n, gate="full")
    t["gate"], t["residual"] = t["gate"][:1].expand(M, n), t["residual"][:1].expand(M, n)
    d = {k: v.to(gpu) for k, v in t.items()}
    d["gate"], d["residual"] = t["gate"][:1].to(gpu).expand(M, n), t["residual"][:1].to(gpu).expand(M, n)
    o = torch.empty(M, n, device=gpu)
    assert R.rmsnorm_block(n=n, out=o, **d) == R.RAD_OK
    _, _, v, ev = B.exact(**t)
    B.check("out", o.cpu(), v, ev)


def test_rows_of_zeros_infinities_and_nans(gpu):
    """They stay in their rows; a row of zeros has zeros, scale 1."""
    M, n = 6, 1000
    t = inputs(M, n)
    t["x"][0], t["residual"][0] = 0, 0
    t["x"][2, 5], t["x"][3, 999], t["residual"][4, 0] = float("inf"), float("nan"), float("-inf")
    d = {k: v.to(gpu) for k, v in t.items()}
    h, o = (torch.empty(M, n, dtype=torch.bfloat16, device=gpu) for _ in range(2))
    q8, s8 = torch.empty(M, n, dtype=torch.int8, device=gpu), torch.empty(M, device=gpu)
    qf, sf = torch.empty(M, n, dtype=torch.uint8, device=gpu), torch.empty(M, 8, device=gpu)
    assert R.rmsnorm_block(n=n, residual_out=h, out=o, q=q8, scale=s8, **d) == R.RAD_OK
    assert R.rmsnorm_block(n=n, q=qf, scale=sf, residual_out=h, out=o, **d) == R.RAD_OK
    torch.cuda.synchronize()
    h, o, q8, s8, qf, sf = (v.cpu() for v in (h, o, q8, s8, qf, sf))
    assert not h[0].any() and not o[0].any() and not q8[0].any() and s8[0] == 1 and not qf[0].any() and (sf[0] == 1).all()
    want, _, v, ev = B.exact(**t)
    good = [1, 5]
    B.check("out", o[good], v[good], ev[good])
    B.check_i8(q8[good], s8[good], v[good], ev[good])
    B.check_e4m3(qf[good], sf[good], v[good], ev[good])
    assert torch.equal(h.isnan(), want.isnan()) and torch.equal(h.isinf(), want.isinf())
    assert torch.equal(o[2:5].isnan(), v[2:5].isnan())
    for i in (2, 3, 4):
        assert not s8[i].isfinite() and not q8[i].any()


@pytest.mark.parametrize("size", [1e-39, 1e-37, 3e-36, 1e-30])
def test_weights_near_the_end_of_the_range(gpu, size):
    """Scales of values that f32 has few numbers below, zeros among them."""
    M, n = 3, 640
    t = inputs(M, n, w="f32")
    t["w_pre"] *= size
    t["w_pre"][::7] = 0
    for codes in ("i8", "e4m3"):
        run(gpu, M, n, out="f32", codes=codes, data=dict(t))


def test_streams_and_graph(gpu):
    M, n = 9, 5376
    t = inputs(M, n)
    d = {k: v.to(gpu) for k, v in t.items()}
    h, q, s = torch.zeros(M, n, dtype=torch.bfloat16, device=gpu), torch.zeros(M, n, dtype=torch.int8, device=gpu), torch.zeros(M, device=gpu)
    ops = R.RmsNormBlockOperands(n=n, residual_out=h, q=q, scale=s, **d)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    assert R.launch_row("rmsnorm_block", ops, side.cuda_stream) == R.RAD_OK
    torch.cuda.synchronize()
    _, _, v, ev = B.exact(**t)
    B.check_i8(q.cpu(), s.cpu(), v, ev)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        assert R.launch_row("rmsnorm_block", ops, torch.cuda.current_stream().cuda_stream) == R.RAD_OK
    for seed in (1, 2, 3):
        u = inputs(M, n, seed=seed)
        for k in u:
            d[k].copy_(u[k])
        graph.replay()
        torch.cuda.synchronize()
        hw, eh, v, ev = B.exact(**u)
        B.check("residual_out", h.cpu(), hw, eh)
        B.check_i8(q.cpu(), s.cpu(), v, ev)
