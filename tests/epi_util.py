"""gemm_nt_epi in 64 bits, and how far a 32-bit kernel may be from it."""
import torch

HALF = {torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}     # half a step, relative to the value
ACTS = ["none", "relu", "silu", "sigmoid", "gelu", "gelu_tanh"]


def act(name, v):
    if name == "relu":
        return torch.where(v < 0, torch.zeros_like(v), v)
    if name == "silu":
        return v * torch.sigmoid(v)
    if name == "sigmoid":
        return torch.sigmoid(v)
    if name == "gelu":
        return 0.5 * v * torch.special.erfc(-v * 0.5 ** 0.5)
    if name == "gelu_tanh":
        return v * torch.sigmoid(2 * (2 / torch.pi) ** 0.5 * (v + 0.044715 * v ** 3))
    return v


def exact(a, b, sa=None, sb=None, bias=None, residual=None, name="none"):
    """(y, the tolerance without y's own rounding) in f64, on the operands' device.

    v = S sum + bias.  At bf16 the products are exact in f32 and summed 32 at a time along a chain of K / 32
    results (and up to 32 planes): with a whole step (2^-23) for each of K / 32 + 64 roundings of a sum that is
    never over sum |a b|.  At i8a8 the sum is exact; its conversion and two products round once each.  The sum
    with the bias, the activation and the residual's sum round once each; no activation's slope is over 1.13, and
    each is good to 16 half steps of |v| (sigmoid 3 ulp, the argument's roundings, which the slope damps)."""
    A, B = a.double(), b.double()
    v = A @ B.T
    if sa is None:
        err = (a.shape[1] / 32 + 64) * 2.0 ** -23 * (A.abs() @ B.abs().T)
    else:
        v = v * sa.double().reshape(-1, 1) * sb.double().reshape(1, -1)
        err = 3 * 2.0 ** -24 * v.abs()
    if bias is not None:
        v = v + bias.double()
        err = err + 2.0 ** -24 * v.abs()
    y = act(name, v)
    if name != "none":
        err = 1.13 * err + 16 * 2.0 ** -24 * v.abs().clamp_min(1.0 if name == "sigmoid" else 0.0)
    if residual is not None:
        y = y + residual.double()
        err = err + 2.0 ** -24 * y.abs()
    return y, err


def check(got, want, err):
    """got within err and its own type's rounding of want."""
    w = want.abs()
    tol = err + HALF[got.dtype] * (w + err) + 2.0 ** -133
    off = (got.double() - want).abs()
    bad = ~(off <= tol)
    assert not bad.any(), (int(bad.sum()), float((off / tol)[bad].max()), bad.nonzero()[:4].tolist())
    return float((off / tol).max())
