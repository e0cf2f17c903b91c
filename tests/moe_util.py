"""moe_layer in 64 bits, and how far a 32-bit kernel may be from it."""
import math

import torch

from tests import epi_util as E

U = 2.0 ** -24
E2M1 = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, -0.0, -0.5, -1.0, -1.5, -2.0, -3.0, -4.0, -6.0]


def plane(w, s, dtype):
    """f64 weights of one expert's codes."""
    if dtype == "bf16":
        return w.double()
    if dtype == "i8":
        return w.double() * s.double().reshape(-1, 1)
    v = torch.tensor(E2M1, dtype=torch.float64, device=w.device)[torch.stack((w & 15, w >> 4), -1).flatten(-2).long()]
    return v * torch.exp2(s.double() - 127).repeat_interleave(32, -1)


def choose(logits, top_k, score="softmax", renorm=1, weight_scale=1.0):
    """(ids, weights in f64, their relative tolerance) a token, in plain Python."""
    M = len(logits)
    ids = torch.full((M, top_k), -1, dtype=torch.int32)
    weights, tol = torch.zeros(M, top_k, dtype=torch.float64), torch.zeros(M, 1, dtype=torch.float64)
    for m, row in enumerate(logits.double().tolist()):
        there = [(-v, e) for e, v in enumerate(row) if v > -math.inf]
        chosen = sorted(there)[:top_k]
        if not chosen:
            continue
        top = -chosen[0][0]
        ex = lambda v: 1.0 if v == top else math.exp(v - top)  # noqa: E731
        sig = lambda v: 1.0 / (1.0 + math.exp(-v)) if v > -700 else math.exp(v)  # noqa: E731
        if score == "softmax":
            s = [ex(-v) for v, _ in chosen]
            total = math.fsum(s) if renorm else math.fsum(ex(-v) for v, _ in there)
        else:
            s = [sig(-v) for v, _ in chosen]
            total = math.fsum(s) if renorm else 1.0
            if total == 0.0:
                s = [ex(-v) for v, _ in chosen]
                total = math.fsum(s)
        for i, (_, e) in enumerate(chosen):
            ids[m, i], weights[m, i] = e, s[i] / total * weight_scale
        far = [top + v for v, _ in chosen if top + v < math.inf]
        # exp of a rounded difference d is off by d U, exp and a division by 4 half steps each, twice (the sum's too)
        tol[m] = (2 * max(far + [0.0]) + 24) * U
    return ids, weights, tol


def exact(x, logits, gate_up, down, dtype, f, top_k, gate_up_scale=None, down_scale=None, act="silu", score="softmax",
          renorm=1, weight_scale=1.0, parts=2):
    """(ids, weights, weights' relative tolerance, y, y's tolerance but for its own rounding).

    Sums of exact products as in epi_util.exact: K / 32 + 64 roundings of at most a step of sum |w x|.  h = act(g) u w
    passes the errors of its three factors on and takes three roundings.  Then it is kept as the sum of two bf16
    numbers (2^-16 of it) where y is bf16, of three (2^-24) where y is f32.  y is the sum over the choices of sums of
    parts * f / 32 results."""
    dev = x.device
    ids, weights, rel = choose(logits.cpu(), top_k, score, renorm, weight_scale)
    y = torch.zeros(x.shape, dtype=torch.float64, device=dev)
    err, size = torch.zeros_like(y), torch.zeros_like(y)
    X, n = x.double(), x.shape[1]
    for e in sorted(set(ids.flatten().tolist()) - {-1}):
        m, i = torch.nonzero(ids == e, as_tuple=True)
        w = weights[m, i].to(dev)[:, None]
        ew = (rel[m, 0].to(dev)[:, None] * w).abs() + 2.0 ** -126
        m = m.to(dev)
        W = plane(gate_up[e], None if gate_up_scale is None else gate_up_scale[e], dtype)
        gu = X[m] @ W.T
        eu = (n / 32 + 64) * 2.0 ** -23 * (X[m].abs() @ W.abs().T) + 2 * U * gu.abs()
        g, u = gu[:, :f], gu[:, f:]
        a = E.act(act, g)
        ea = 1.13 * eu[:, :f] + 16 * U * g.abs().clamp_min(1.0 if act == "sigmoid" else 0.0)
        h = a * u * w
        eh = ((u * w).abs() * ea + (a * w).abs() * eu[:, f:] + (a * u).abs() * ew) * 1.01 + 4 * U * h.abs()
        eh = eh + 2.0 ** (-8 * parts) * h.abs() + 2.0 ** -133
        D = plane(down[e], None if down_scale is None else down_scale[e], dtype)
        y.index_add_(0, m, h @ D.T)
        err.index_add_(0, m, eh @ D.abs().T)
        size.index_add_(0, m, h.abs() @ D.abs().T)
    err = err + (parts * f / 32 + 64 + top_k) * 2.0 ** -23 * size
    return ids, weights, rel, y, err


def check(got, want):
    y, ids, weights = got
    wi, ww, rel, wy, err = want
    assert torch.equal(ids.cpu(), wi), (ids.cpu()[(ids.cpu() != wi).any(1)][:3], wi[(ids.cpu() != wi).any(1)][:3])
    off = (weights.cpu().double() - ww).abs()
    assert (off <= rel * ww.abs() + 2.0 ** -126).all(), float((off / (rel * ww.abs() + 2.0 ** -126)).max())
    return E.check(y, wy, err)
