"""moe_layer on the GPU against 64 bits: choices equal, weights and every element of y within bounds that count the
roundings.  Operands lie in guarded memory, and what lies around every output has to be left as it was."""
import math

import pytest
import torch

import libr3d_amd as R
from tests import moe_util as U
from tests.test_gpu_i8 import Box

pytestmark = pytest.mark.gpu
KIND = {"bf16": torch.bfloat16, "f32": torch.float32}


def experts(g, dtype, E, rows, K):
    if dtype == "bf16":
        return (torch.randn(E, rows, K, generator=g) * K ** -0.5).bfloat16(), None
    if dtype == "i8":
        w = torch.randint(-128, 128, (E, rows, K), generator=g, dtype=torch.int32).to(torch.int8)
        return w, (0.5 + torch.rand(E, rows, generator=g)) * K ** -0.5 / 74
    mid = 127 + round(math.log2(K ** -0.5 / 2.9))
    w = torch.randint(0, 256, (E, rows, K // 2), generator=g, dtype=torch.int32).to(torch.uint8)
    return w, torch.randint(mid - 1, mid + 2, (E, rows, K // 32), generator=g, dtype=torch.int32).to(torch.uint8)


def inputs(dtype, M, n, f, E, seed=0, logits=None):
    g = torch.Generator().manual_seed(seed * 1000003 + M * 7919 + n * 31 + f * 7 + E)
    gu, gus = experts(g, dtype, E, 2 * f, n)
    dn, dns = experts(g, dtype, E, n, f)
    lg = 1.5 * torch.randn(M, E, generator=g) if logits is None else logits
    return dict(x=torch.randn(M, n, generator=g).bfloat16(), logits=lg, gate_up=gu, down=dn, gate_up_scale=gus, down_scale=dns)


def padded(t, dev, extra):
    """t on the device, its rows `extra` elements apart from each other (16-byte multiples) and its planes further."""
    if t is None or not extra:
        return None if t is None else t.to(dev)
    E, rows, K = t.shape
    big = torch.zeros(E, rows + 1, K + extra, dtype=t.dtype, device=dev)
    big[:, :rows, :K] = t.to(dev)
    return big[:, :rows, :K]


def run(dev, dtype, M, n, f, E, k, y="bf16", seed=0, logits=None, extra=0, pad=0, data=None, **par):
    t = data or inputs(dtype, M, n, f, E, seed, logits)
    X = Box(t["x"], dev, 0, n + 8 * bool(extra))
    Y = Box(torch.full((M, n), -7.0, dtype=KIND[y]), dev, pad, n + pad)
    I = Box(torch.full((M, k), -9, dtype=torch.int32), dev, pad, k + pad)
    W = Box(torch.full((M, k), -9.0), dev, 0, k + 2 * pad)
    L = Box(t["logits"], dev, pad, E + pad)
    d = {m: padded(t[m], dev, extra) for m in ("gate_up", "down")}
    s = {m: padded(t[m], dev, 3 * bool(extra)) if dtype == "mxfp4" else None if t[m] is None else t[m].to(dev)
         for m in ("gate_up_scale", "down_scale")}
    ops = R.MoeLayerOperands(X.t, L.t, d["gate_up"], d["down"], Y.t, **s, ids=I.t, weights=W.t, dtype=dtype, n=n, f=f, E=E,
                             top_k=k, **par)
    need = R.row_scratch_bytes("moe_layer", ops)
    S = Box(torch.full((1, need), 0xFF, dtype=torch.uint8), dev)
    ops.set_scratch(S.t, need)
    print(R.describe("moe_layer", ops)[1], extra, pad, flush=True)
    assert R.launch_row("moe_layer", ops, torch.cuda.current_stream().cuda_stream) == R.RAD_OK
    torch.cuda.synchronize()
    on = {m: None if v is None else v.to(dev) for m, v in t.items()}
    want = U.exact(**on, dtype=dtype, f=f, top_k=k, parts=3 if y == "f32" else 2, **par)
    use = U.check((Y.t, I.t, W.t), want)
    assert all(b.around() for b in (X, Y, I, W, L, S))
    return use


DTYPES = ["bf16", "i8", "mxfp4"]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("M", [1, 2, 3, 7, 8, 9, 16, 17, 33, 63, 64])
def test_tokens(gpu, dtype, M):
    run(gpu, dtype, M, 288, 160, 12, 3)
    run(gpu, dtype, M, 288, 160, 12, 3, y="f32")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,f", [(32, 32), (32, 512), (512, 32), (64, 96), (96, 64), (256, 256), (544, 1056), (2048, 768), (1120, 2080)])
def test_sizes(gpu, dtype, n, f):
    for M, y in ((1, "f32"), (5, "bf16"), (20, "f32")):
        run(gpu, dtype, M, n, f, 6, 2, y=y)


@pytest.mark.parametrize("dtype,step", [("bf16", 8), ("i8", 16)])
def test_odd_sizes(gpu, dtype, step):
    for n, f in ((step, step), (3 * step, 5 * step), (37 * step, 21 * step), (130 * step, 67 * step)):
        for M in (1, 11):
            run(gpu, dtype, M, n, f, 5, 2, y="f32")


@pytest.mark.parametrize("E,k", [(1, 1), (2, 2), (3, 1), (16, 16), (63, 5), (64, 8), (65, 8), (128, 8), (130, 4), (256, 16),
                                 (257, 9), (300, 1), (512, 16)])
def test_experts(gpu, E, k):
    for M in (1, 6, 64):
        run(gpu, "mxfp4", M, 64, 64, E, k, y="f32")
    run(gpu, "i8", 30, 64, 48, E, k, score="sigmoid", renorm=0)


@pytest.mark.parametrize("dtype", DTYPES)
def test_crowded_expert(gpu, dtype):
    """Every token chooses the same experts: jobs of all widths, and more than one an expert."""
    for M in (9, 16, 17, 32, 33, 64):
        for E, k in ((2, 1), (40, 2), (200, 3)):
            lg = torch.zeros(M, E)
            lg[:, E // 2] = 4.0
            lg[: M // 2, 0] = 2.0
            for y in ("bf16", "f32"):
                run(gpu, dtype, M, 160, 96, E, k, y=y, logits=lg)


@pytest.mark.parametrize("act", ["silu", "gelu", "gelu_tanh", "relu", "sigmoid", "none"])
def test_activations(gpu, act):
    run(gpu, "bf16", 5, 256, 128, 8, 2, y="f32", act=act)
    run(gpu, "mxfp4", 12, 256, 128, 8, 2, act=act)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renorm", [0, 1])
def test_scores(gpu, score, renorm):
    g = torch.Generator().manual_seed(3)
    for E, k in ((8, 3), (100, 8), (400, 16)):
        for spread, shift in ((0.1, 0), (6, 0), (3, -60), (3, 60), (2, -200), (20, 0)):
            lg = spread * torch.randn(10, E, generator=g) + shift
            run(gpu, "i8", 10, 64, 48, E, k, y="f32", logits=lg, score=score, renorm=renorm, weight_scale=2.5)
            run(gpu, "i8", 10, 64, 48, E, k, y="f32", logits=lg.bfloat16(), score=score, renorm=renorm)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renorm", [0, 1])
def test_masks(gpu, score, renorm):
    """Rows with nothing, with fewer than top_k, ties, infinities, NaN and the type's lowest value."""
    inf, nan, low = float("inf"), float("nan"), torch.finfo(torch.float32).min
    E, k = 70, 4
    g = torch.Generator().manual_seed(4)
    lg = torch.randn(14, E, generator=g)
    lg[0] = -inf
    lg[1] = nan
    lg[2], lg[2, 69] = -inf, 0.5
    lg[3], lg[3, 3], lg[3, 68] = -inf, 0.25, 0.25
    lg[4] = 1.0                                   # all equal
    lg[5], lg[5, ::2] = -0.0, 0.0                 # zeros of both signs are equal
    lg[6, 10], lg[6, 60] = inf, inf
    lg[7] = low
    lg[8], lg[8, 5], lg[8, 40] = low, 1.0, 2.0
    lg[9, ::3] = nan
    lg[10] = inf
    lg[11, 64:] = 9.0
    lg[13] = -inf
    for dtype, y in (("bf16", "f32"), ("mxfp4", "bf16")):
        run(gpu, dtype, 14, 96, 64, E, k, y=y, logits=lg, score=score, renorm=renorm)
    none = torch.full((3, E), -inf)
    run(gpu, "bf16", 3, 96, 64, E, k, logits=none, score=score, renorm=renorm)


@pytest.mark.parametrize("dtype", DTYPES)
def test_strides(gpu, dtype):
    for M, pad in ((1, 0), (4, 1), (20, 3)):
        for y in ("bf16", "f32"):
            run(gpu, dtype, M, 288, 160, 7, 2, y=y, extra=32, pad=pad)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("M,n,f,E,k", [(1, 5376, 1344, 32, 8), (4, 2048, 768, 64, 4), (13, 2048, 1408, 32, 4), (64, 1024, 1344, 128, 8)])
def test_larger(gpu, dtype, M, n, f, E, k):
    run(gpu, dtype, M, n, f, E, k)
    run(gpu, dtype, M, n, f, E, k, y="f32")


def test_scales_at_their_ends(gpu):
    """E8M0 0 (2^-127), 255 (NaN) and what leaves bf16's range belong to their rows alone; int8 scales 0, inf and NaN."""
    t = inputs("mxfp4", 3, 64, 32, 2)
    t["logits"] = torch.tensor([[9.0, 0.0]]).expand(3, 2).contiguous()
    t["down_scale"][0, 5], t["down_scale"][0, 6], t["down_scale"][0, 7] = 0, 255, 254
    on = {m: None if v is None else v.to(gpu) for m, v in t.items()}
    y = torch.empty(3, 64, device=gpu)
    assert R.moe_layer(y=y, dtype="mxfp4", n=64, f=32, E=2, top_k=1, **on) == R.RAD_OK
    _, _, _, want, err = U.exact(**on, dtype="mxfp4", f=32, top_k=1, parts=3)
    rest = [i for i in range(64) if i not in (6, 7)]
    U.E.check(y[:, rest], want[:, rest], err[:, rest])
    assert y[:, 6].isnan().all() and not y[:, 7].isfinite().any()
    t = inputs("i8", 3, 64, 32, 2)
    t["logits"] = torch.tensor([[9.0, 0.0]]).expand(3, 2).contiguous()
    t["down_scale"][0, 5], t["down_scale"][0, 6], t["down_scale"][0, 7] = 0.0, float("nan"), float("inf")
    on = {m: None if v is None else v.to(gpu) for m, v in t.items()}
    assert R.moe_layer(y=y, dtype="i8", n=64, f=32, E=2, top_k=1, **on) == R.RAD_OK
    _, _, _, want, err = U.exact(**on, dtype="i8", f=32, top_k=1, parts=3)
    U.E.check(y[:, rest], want[:, rest], err[:, rest])
    assert y[:, 6].isnan().all() and not y[:, 7].isfinite().any()


def test_tokens_do_not_meet(gpu):
    """NaN and inf in one token's activation, or in an expert that it alone chose, reach its row alone."""
    M, n, f, E = 9, 256, 96, 6
    t = inputs("bf16", M, n, f, E)
    t["logits"] = torch.full((M, E), -1.0)
    t["logits"][:, 1], t["logits"][:, 2] = 3.0, 2.0
    t["logits"][4, 5] = 8.0
    t["x"][7, 100], t["x"][2, 255] = float("nan"), float("inf")
    t["gate_up"][5, 3, 9], t["down"][5, 200, 0] = float("nan"), float("inf")
    on = {m: None if v is None else v.to(gpu) for m, v in t.items()}
    for kind, parts in ((torch.float32, 3), (torch.bfloat16, 2)):
        y = torch.empty(M, n, dtype=kind, device=gpu)
        assert R.moe_layer(y=y, dtype="bf16", n=n, f=f, E=E, top_k=2, **on) == R.RAD_OK
        rows = [m for m in range(M) if m not in (2, 4, 7)]
        _, _, _, want, err = U.exact(**on, dtype="bf16", f=f, top_k=2, parts=parts)
        U.E.check(y[rows], want[rows], err[rows])
        assert y[7].isnan().all() and not y[2].isfinite().any() and not y[4].isfinite().any()


@pytest.mark.parametrize("M", [1, 5, 9, 64])
def test_result_over_the_inputs(gpu, M):
    """y in the memory of x, and (f32) of the logits."""
    n, f, E, k = 64, 96, 64, 4
    t = inputs("i8", M, n, f, E)
    on = {m: None if v is None else v.to(gpu) for m, v in t.items()}
    want = U.exact(**on, dtype="i8", f=f, top_k=k, parts=2), U.exact(**on, dtype="i8", f=f, top_k=k, parts=3)
    for name, w in zip(("x", "logits"), want):
        d = dict(on, x=on["x"].clone(), logits=on["logits"].clone())
        ids, ws = torch.zeros(M, k, dtype=torch.int32, device=gpu), torch.zeros(M, k, device=gpu)
        assert R.moe_layer(y=d[name], ids=ids, weights=ws, dtype="i8", n=n, f=f, E=E, top_k=k, **d) == R.RAD_OK
        torch.cuda.synchronize()
        U.check((d[name], ids, ws), w)


def test_streams_and_graph(gpu):
    """Two streams at once with their scratch each, and a captured call replayed over new tokens, bit for bit as called."""
    for dtype, M in (("bf16", 3), ("i8", 40), ("mxfp4", 64)):
        n, f, E, k = 320, 160, 20, 3
        t = inputs(dtype, M, n, f, E)
        on = {m: None if v is None else v.to(gpu) for m, v in t.items()}

        def bound():
            y = torch.zeros(M, n, device=gpu)
            ids, w = torch.zeros(M, k, dtype=torch.int32, device=gpu), torch.zeros(M, k, device=gpu)
            ops = R.MoeLayerOperands(y=y, ids=ids, weights=w, dtype=dtype, n=n, f=f, E=E, top_k=k, **on)
            ops.set_scratch(torch.full((R.row_scratch_bytes("moe_layer", ops),), 0xA5, dtype=torch.uint8, device=gpu))
            return y, ids, w, ops
        want = U.exact(**on, dtype=dtype, f=f, top_k=k, parts=3)
        two = [(torch.cuda.Stream(), bound()) for _ in range(2)]
        torch.cuda.synchronize()
        for s, b in two:
            assert R.launch_row("moe_layer", b[3], s.cuda_stream) == R.RAD_OK
        torch.cuda.synchronize()
        for s, b in two:
            U.check(b[:3], want)
        y, ids, w, ops = bound()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            assert R.launch_row("moe_layer", ops, torch.cuda.current_stream().cuda_stream) == R.RAD_OK
        for i in range(3):
            u = inputs(dtype, M, n, f, E, seed=i + 1)
            on["x"].copy_(u["x"])
            on["logits"].copy_(u["logits"])
            y.fill_(-1)
            graph.replay()
            torch.cuda.synchronize()
            U.check((y, ids, w), U.exact(**on, dtype=dtype, f=f, top_k=k, parts=3))
            again = torch.zeros_like(y)
            assert R.moe_layer(y=again, dtype=dtype, n=n, f=f, E=E, top_k=k, **on) == R.RAD_OK
            torch.cuda.synchronize()
            assert torch.equal(y, again)
