"""rmsnorm_block in 64 bits, and how far a 32-bit kernel may be from it."""
import torch

HALF = {torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}     # half a step, relative to the value
U = 2.0 ** -24


def exact(x, residual=None, w_post=None, gate=None, w_pre=None, eps=1e-6, wadd=0.0, res_scale=1.0):
    """(h, its tolerance, v, its tolerance) in f64 before anything is rounded to an output's type.

    t = (x rs) (w + wadd): four roundings (rs, two products, the weight's sum; the sum of squares is in f64), one
    more with the gate, one for res_scale's own rounding, one of the last sum: h is off by at most
    7 U (|gate t| + |res_scale residual|).  rs of h changes by what the errors of h change its sum of squares; v
    takes that, h's own error and four more roundings."""
    d = lambda t: t.double()  # noqa: E731
    h = d(x)
    if w_post is not None:
        h = h / torch.sqrt((h * h).mean(1, keepdim=True) + eps) * (d(w_post) + wadd)
    if gate is not None:
        h = h * d(gate)
    size = h.abs()
    if residual is not None:
        r = res_scale * d(residual)
        h, size = h + r, size + r.abs()
    eh = 7 * U * size
    if w_pre is None:
        return h, eh, None, None
    n = h.shape[1]
    total = (h * h).sum(1, keepdim=True) + n * eps
    rs = torch.sqrt(n / total)
    w = d(w_pre) + wadd
    v = h * rs * w
    rel = (h.abs() * eh).sum(1, keepdim=True) / total * 1.01
    ev = (rs * w).abs() * eh * 1.01 + v.abs() * (rel + 4 * U)
    return h, eh, v, ev


def check(name, got, want, err):
    tol = err + HALF[got.dtype] * (want.abs() + err) + 2.0 ** -133
    off = (got.double() - want).abs()
    bad = ~(off <= tol)
    assert not bad.any(), (name, int(bad.sum()), float((off / tol)[bad].max()), bad.nonzero()[:4].tolist())


def check_i8(q, scale, v, ev):
    s = scale.double().reshape(-1, 1)
    amax = v.abs().amax(1, keepdim=True)
    want = torch.where(amax > 0, (amax / 127).clamp_min(2.0 ** -126), torch.ones_like(amax))
    near = ev.amax(1, keepdim=True) / 127 + 3 * U * want
    assert ((s - want).abs() <= near).all()
    # the code's own rounding; v * (1 / s) takes two more of at most 127 codes
    assert ((q.double() * s - v).abs() <= s * (0.5 + 127 * 3 * U) + ev).all()
    assert (q.abs().amax(1) <= 127).all()


def check_e4m3(q, scale, v, ev):
    n = v.shape[1]
    pad = lambda t: torch.nn.functional.pad(t, (0, -n % 128)).unflatten(1, (-1, 128))  # noqa: E731
    amax = pad(v).abs().amax(2)
    want = torch.where(amax > 0, (amax / 448).clamp_min(2.0 ** -126), torch.ones_like(amax))
    assert ((scale.double() - want).abs() <= pad(ev).amax(2) / 448 + 3 * U * want).all()
    s = scale.double().repeat_interleave(128, 1)[:, :n]
    got = q.view(torch.float8_e4m3fn).double() * s
    # half a step of e4m3: 2^-4 of the value, 2^-10 of the scale under 2^-6 of it
    assert ((got - v).abs() <= (2.0 ** -4 * v.abs()).maximum(2.0 ** -10 * s) * (1 + 4 * U) + 1.07 * ev).all()
