"""The activations of gemm_nt_epi and moe_layer against 64 bits, relative to their own size down to where f32's normal numbers end,
on every kernel that has them: products are made so that an activation's argument is the f32 number it is meant to be.

Bounds, in U = 2^-24 of the value (an ulp is 2 U at most), and 2^-126 where hardware may round a result under the normal range to 0:
  sigmoid    3 ulp
  silu       that and a product
  gelu       v erfc(z) / 2: z = -v / sqrt 2 by a rounded constant and a product is off by 2 U, which erfc takes by its
             condition z erfc'(z) / erfc(z); erfc itself is good to 16 ulp; one product more
  gelu_tanh  v sigmoid(x), x = v (c1 + c2 v^2): v^2 and c2 round by 3.5 U, the sum, c1 and the product by less than 2.5 U; 1.25 U
             more from x log2 e and its constant, all taken by |x| (1 - sigmoid(x)); exp2 and the reciprocal an ulp each, the
             sum and the last product half of one"""
import pytest
import torch

import libr3d_amd as R
from tests import epi_util as E

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def values():
    mag = torch.cat((torch.logspace(-6, 2, 700, dtype=torch.float64), torch.linspace(0.5, 20, 300, dtype=torch.float64),
                     torch.tensor([20.0, 25.0, 60.0, 85.0, 87.0, 88.5, 104.0]))).float()
    return torch.cat((mag, -mag, torch.zeros(1)))


def want(name, v):
    """(activation, bound) in 64 bits of f32 arguments."""
    x = v.double()
    y = E.act(name, x)
    if name in ("none", "relu"):
        return y, torch.zeros_like(y)
    if name == "sigmoid":
        return y, 6 * U * y.abs() + 2.0 ** -126
    if name == "silu":
        rel = torch.full_like(y, 7.0)
    elif name == "gelu":
        z = -x * 0.5 ** 0.5
        rel = 2 * (z * 2 / torch.pi ** 0.5 / torch.special.erfcx(z)).abs() + 33       # e^(-z z) / erfc z = 1 / erfcx z
        rel = torch.where(z < -5, torch.full_like(rel, 33.0), rel)                    # erfc is 2 there, and erfcx no number
    else:
        a = 2 * (2 / torch.pi) ** 0.5 * (x + 0.044715 * x ** 3)
        rel = 7.25 * a.abs() * (1 - torch.sigmoid(a)) + 7
    return y, rel * U * y.abs() + 2.0 ** -126 * (1 + x.abs())


def hold(name, got, v):
    y, tol = want(name, v)
    tol = tol + E.HALF[got.dtype] * (y.abs() + tol) * (got.dtype != torch.float32)    # f32 results are the values
    off = (got.double() - y).abs()
    bad = ~(off <= tol)
    assert not bad.any(), (name, int(bad.sum()), float((off / tol.clamp_min(1e-300))[bad].max()), v.expand_as(got)[bad][:4].tolist())


SPECIAL = torch.tensor([float("inf"), float("-inf"), float("nan"), 3.4e38, -3.4e38, 1e30, -1e30])
INF, NAN = float("inf"), float("nan")
LIMITS = {"none": [INF, -INF, NAN, 3.4e38, -3.4e38, 1e30, -1e30], "relu": [INF, 0, NAN, 3.4e38, 0, 1e30, 0],
          "sigmoid": [1, 0, NAN, 1, 0, 1, 0], "silu": [INF, NAN, NAN, 3.4e38, 0, 1e30, 0],
          "gelu": [INF, NAN, NAN, 3.4e38, 0, 1e30, 0], "gelu_tanh": [INF, NAN, NAN, 3.4e38, 0, 1e30, 0]}


def product(dev, dtype, M, K, v, act, y, arm="", planes=False, special=False):
    """act(v) in every row: int8 ones, v in b's scales; or three bf16 ones a row against v cut in three."""
    N = len(v)
    one = 1 if dtype == "i8a8" else 3
    kind = torch.int8 if dtype == "i8a8" else torch.bfloat16
    a, b = torch.zeros(M, K, dtype=kind), torch.zeros(N, K, dtype=kind)
    at = [0, K // 2, K - 1][:one]
    a[:, at] = 1
    kw = {}
    if dtype == "i8a8":
        b[:, 0] = 1
        kw = dict(a_scale=torch.ones(M, device=dev), b_scale=v.to(dev))
    else:
        left = v.clone()
        for c in at:
            b[:, c] = left.view(torch.int32).bitwise_and(-65536).view(torch.float32).bfloat16()
            left = left - b[:, c].float()
    Y = torch.empty(M, N, dtype=y, device=dev)
    A, B = a.to(dev), b.to(dev)
    ops = R.GemmEpiOperands(A, B, Y, dtype=dtype, N=N, K=K, act=act, **kw)
    text = R.describe("gemm_nt_epi_" + dtype, ops)[1]
    assert arm in text and (R.row_scratch_bytes("gemm_nt_epi_" + dtype, ops) > 0) == planes, text
    assert R.gemm_nt_epi(A, B, Y, dtype=dtype, N=N, K=K, act=act, **kw) == R.RAD_OK
    assert torch.equal(Y.nan_to_num(7.0), Y[:1].nan_to_num(7.0).expand(M, N))
    got = Y[0].cpu()
    if special:
        lim = torch.tensor(LIMITS[act]).to(y)
        assert torch.equal(got.isnan(), lim.isnan()) and torch.equal(got[~lim.isnan()], lim[~lim.isnan()])
    else:
        hold(act, got, v)


# the GEMV, a small and the widest tile, K in planes, any alignment (K in bytes)
ARMS = [(1, 2048, "arm=gemv"), (40, 1024, "arm=tile"), (8000, 1024, "bn=256 bm=256"), (12, 43008, "arm=tile"), (5, 1026, "arm=any"),
        (30, 1026, "arm=any")]


@pytest.mark.parametrize("act", E.ACTS)
@pytest.mark.parametrize("dtype", ["i8a8", "bf16"])
@pytest.mark.parametrize("M,K,arm", ARMS)
def test_products(gpu, dtype, act, M, K, arm):
    v = values()
    for y in (torch.float32, torch.bfloat16):
        product(gpu, dtype, M, K // (1 if dtype == "i8a8" else 2), v, act, y, arm, planes=K > 40000)


@pytest.mark.parametrize("act", E.ACTS)
def test_limits(gpu, act):
    for M, K, _ in ARMS:
        if M < 8000:
            product(gpu, "i8a8", M, K, SPECIAL, act, torch.float32, planes=K > 40000, special=True)


@pytest.mark.parametrize("act", E.ACTS)
@pytest.mark.parametrize("M", [1, 9])
def test_experts(gpu, act, M):
    """One expert whose gate rows' scales are the arguments, up rows 1, and the identity behind them."""
    v = values()
    f = -(-len(v) // 16) * 16
    v = torch.cat((v, torch.ones(f - len(v))))
    x = torch.zeros(M, 32)
    x[:, 0] = 1
    gu = torch.zeros(1, 2 * f, 32, dtype=torch.int8)
    gu[..., 0] = 1
    scale = torch.cat((v, torch.ones(f)))[None]
    down = torch.zeros(1, 32, f, dtype=torch.int8)
    for c in range(0, f, 32):                          # 32 rows of the identity at a time
        down.zero_()
        i = torch.arange(min(32, f - c))
        down[0, i, c + i] = 1
        y = torch.empty(M, 32, device=gpu)
        assert R.moe_layer(x.bfloat16().to(gpu), torch.zeros(M, 1, device=gpu), gu.to(gpu), down.to(gpu), y, dtype="i8", n=32, f=f,
                           E=1, top_k=1, gate_up_scale=scale.to(gpu), down_scale=torch.ones(1, 32, device=gpu), act=act) == R.RAD_OK
        hold(act, y[:, :len(i)].cpu(), v[c:c + 32])
