"""moe_layer where a workgroup's run of units takes several passes, where LDS holds few tokens' rows, and where a row of h takes several
steps of three spans: each case is shown on the host to be one of these, then run against 64 bits."""
import pytest
import torch

import libr3d_amd as R
from tests import moe_util as U
from tests.moe_passes import launch, passes
from tests.test_gpu_moe import DTYPES, inputs, run

pytestmark = pytest.mark.gpu
CAP = 128                                              # units whose int8 scales lie in LDS at a time


def crowd(M, E, k, each, seed=0):
    """Logits by which `each` tokens beside each other choose the same experts, the next ones others."""
    g = torch.Generator().manual_seed(seed)
    lg = torch.randn(M, E, generator=g)
    for m in range(M):
        lg[m, [(m // each * k + i) % E for i in range(k)]] = 9.0 - torch.arange(k) / 8
    return lg


def case(dtype, M, n, f, E, k, logits):
    """(the launch, each product's passes) of a call with these choices."""
    t = {m: None if v is None else v[:1].expand(E, *v.shape[1:]) for m, v in inputs(dtype, 1, n, f, 1).items()
         if m not in ("x", "logits")}
    ops = R.MoeLayerOperands(torch.empty(M, n, dtype=torch.bfloat16), logits, t["gate_up"], t["down"], torch.empty(M, n),
                             gate_up_scale=t["gate_up_scale"], down_scale=t["down_scale"], dtype=dtype, n=n, f=f, E=E, top_k=k)
    g = launch(ops)
    ids = U.choose(logits, k)[0].flatten()
    tokens = torch.bincount(ids[ids >= 0], minlength=E).tolist()
    cap = CAP if dtype == "i8" else 1 << 30
    return g, passes(tokens, f // 8, g["up_width"], g["up_rows"], cap, g["blocks"]), \
        passes(tokens, (n + 15) // 16, g["down_width"], g["down_rows"], cap, g["blocks"])


# jobs of one, two and three tokens a read of the down planes, of one and two of the up planes
WIDTHS = [("down", 1, 32, 14336), ("down", 2, 32, 10752), ("down", 3, 32, 7680), ("up", 1, 40960, 32), ("up", 2, 30720, 64)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("which,width,n,f", WIDTHS)
def test_narrow_jobs(gpu, dtype, which, width, n, f):
    for M in (1, 7, 20):
        logits = crowd(M, 3, 2, 100)
        g, _, _ = case(dtype, M, n, f, 3, 2, logits)
        assert g[which + "_width"] == min(width, 2 * M) and g["parts"] == 1
        for y in ("bf16", "f32"):
            run(gpu, dtype, M, n, f, 3, 2, y=y, logits=logits)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,f,M,E,k", [(512, 14336, 64, 2, 2), (2048, 9 * 512 + 32, 64, 2, 1), (64, 28672, 1, 2, 1), (64, 28672, 9, 2, 1),
                                       (32, 65536, 3, 1, 1), (1056, 7712, 40, 3, 3)])
def test_rows_of_h_in_parts(gpu, dtype, n, f, M, E, k):
    """Launches over a part of h's columns each, the last one shorter, that add to the sums of the ones before."""
    logits = crowd(M, E, k, 100)
    g, _, _ = case(dtype, M, n, f, E, k, logits)
    assert g["parts"] > 1
    for y in ("bf16", "f32"):
        run(gpu, dtype, M, n, f, E, k, y=y, logits=logits)


@pytest.mark.parametrize("dtype", DTYPES)
def test_up_passes(gpu, dtype):
    """Rows of n = 30720 leave LDS two tokens', and a run has jobs of more."""
    M, n, f, E, k = 64, 30720, 32, 15, 15
    logits = torch.randn(M, E, generator=torch.Generator().manual_seed(2))
    g, up, _ = case(dtype, M, n, f, E, k, logits)
    assert g["up_rows"] == 2 and up[0] >= 3
    run(gpu, dtype, M, n, f, E, k, y="f32", logits=logits)


@pytest.mark.parametrize("dtype", DTYPES)
def test_down_passes(gpu, dtype):
    """Rows of h of f = 7680 leave LDS few tokens', a job of 32 rows of y is two units, and a run has more jobs than LDS holds."""
    M, n, f, E, k = 60, 32, 7680, 64, 16
    logits = crowd(M, E, k, 1)
    g, _, down = case(dtype, M, n, f, E, k, logits)
    assert down[0] >= 2 and g["down_rows"] <= 6
    for y in ("bf16", "f32"):
        run(gpu, dtype, M, n, f, E, k, y=y, logits=logits)


@pytest.mark.parametrize("n,f,which", [(32, 2560, 1), (4096, 32, 2), (736, 2560, 1)])
def test_int8_scales_in_parts(gpu, n, f, which):
    """More than 128 units a run: the scales' LDS is filled again, in the middle of a job."""
    M, E, k = 64, 256, 8
    logits = crowd(M, E, k, 2)
    got = case("i8", M, n, f, E, k, logits)
    assert got[which][0] >= 2 and got[which][1] and got[which][2]
    run(gpu, "i8", M, n, f, E, k, y="f32", logits=logits)
    run(gpu, "i8", M, n, f, E, k, y="bf16", logits=torch.randn(M, E, generator=torch.Generator().manual_seed(1)))


@pytest.mark.parametrize("f", [4128, 4352, 4608, 7200, 7680])
def test_steps_of_three_spans(gpu, f):
    """e2m1 rows of h of 9 and 15 spans, whole ones and some that end inside a span."""
    assert -(-f // 512) in (9, 15)
    for M, n in ((1, 64), (6, 96), (30, 48 * 32)):
        for y in ("bf16", "f32"):
            run(gpu, "mxfp4", M, n, f, 5, 2, y=y)


@pytest.mark.parametrize("dtype", DTYPES)
def test_parts_of_padded_planes(gpu, dtype):
    """Rows and planes of the experts further apart than their columns, and h in parts."""
    M, n, f, E, k = 60, 2048, 9 * 512 + 32, 2, 1
    logits = crowd(M, E, k, 100)
    assert case(dtype, M, n, f, E, k, logits)[0]["parts"] > 1
    run(gpu, dtype, M, n, f, E, k, y="f32", logits=logits, extra=32, pad=3)


@pytest.mark.parametrize("dtype", DTYPES)
def test_parts_captured(gpu, dtype):
    """A call of several down launches, captured once and replayed over new tokens with other work between, bit for bit as called."""
    M, n, f, E, k = 64, 512, 14336, 2, 2
    assert case(dtype, M, n, f, E, k, crowd(M, E, k, 100))[0]["parts"] > 1
    t = inputs(dtype, M, n, f, E)
    on = {m: None if v is None else v.to(gpu) for m, v in t.items()}
    y = torch.zeros(M, n, device=gpu)
    ops = R.MoeLayerOperands(y=y, dtype=dtype, n=n, f=f, E=E, top_k=k, **on)
    ops.set_scratch(torch.full((R.row_scratch_bytes("moe_layer", ops),), 0xA5, dtype=torch.uint8, device=gpu))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        assert R.launch_row("moe_layer", ops, torch.cuda.current_stream().cuda_stream) == R.RAD_OK
    for i in range(3):
        g = torch.Generator().manual_seed(i)
        on["x"].copy_(torch.randn(M, n, generator=g).bfloat16())
        on["logits"].copy_(torch.randn(M, E, generator=g))
        y.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        _, _, _, want, err = U.exact(**on, dtype=dtype, f=f, top_k=k, parts=3)
        U.E.check(y, want, err)
        again = torch.zeros_like(y)
        assert R.moe_layer(y=again, dtype=dtype, n=n, f=f, E=E, top_k=k, **on) == R.RAD_OK
        torch.cuda.synchronize()
        assert torch.equal(y, again)
