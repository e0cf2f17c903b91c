"""Checks of captured int8 and sampler launches for tests/replay_dump.py, in float64 from the PRE
state: the product's sums are exact integers and its epilogue three f32 roundings, so its elements are
compared bit for bit; a producer's scale may be off by 2^-20 of itself (the roundings of h, 1/127 and
their products), a code by 1/2 + 127 * 2^-20 from h / s, an output by 2^-20 and its own rounding, plus,
for a gate past the least normal sigmoid, 2^-126 (1 + |gate|) |up|; the norm's residual_out is one f32 addition
and one rounding, compared bit for bit; tokens have to be equal.  A probability is off by its f32 rounding and,
as the kept mass is at least 1 and made of V numbers of unit 2^-s at most, by V 2^-(s + 1) of itself, s = min(62 -
ceil(log2 V), 51); both doubled, and 2^-126 for a share that f32 has no normal number for."""
import numpy as np

F32, BF16, I8, I32 = 0, 1, 8, 10


def _span(c, i, state):
    t = c.tensors[i]
    np_t = {F32: np.float32, BF16: np.uint16, I8: np.int8, I32: np.int32}[t["dt"]]
    return t, np.asarray((c.pre if state == "pre" else c.post)[i], np.uint8).view(np_t)


def _rows(c, i, rows, cols, state):
    """[rows, cols] of an operand; bf16 as float32."""
    t, v = _span(c, i, state)
    pitch = t["stride"][t["rank"] - 2] if t["rank"] >= 2 else 0
    v = np.stack([v[r * pitch:r * pitch + cols] for r in range(rows)])
    return (v.astype(np.uint32) << 16).view(np.float32) if t["dt"] == BF16 else v


def _column(c, i, rows, state, default=None):
    """One number a row, [rows] or [rows, 1]; `default` where the operand is absent."""
    if not c.present(i):
        return [default] * rows
    t, v = _span(c, i, state)
    return [v[r * t["stride"][0]].item() for r in range(rows)]


def _numel(t):
    return int(np.prod(t["shape"][:t["rank"]], dtype=np.int64))


def _bf16(v):
    """float32 to the nearest bf16, ties to even, as float32."""
    u = np.asarray(v, np.float32).view(np.uint32).astype(np.uint64)
    r = (((u + 0x7FFF + (u >> 16 & 1)) >> 16) << 16).astype(np.uint32).view(np.float32)
    return np.where(np.isnan(v), v, r)


def _same(got, want):
    return bool(np.all((got == want) | (np.isnan(got) & np.isnan(want))))


def check_gemm(c):
    N, K = c.geti("N"), c.geti("K")
    M = _numel(c.tensors[4]) // N
    a, b = _rows(c, 0, M, K, "pre").astype(np.float64), _rows(c, 2, N, K, "pre").astype(np.float64)
    sa, sb = (np.asarray(_column(c, i, r, "pre"), np.float32) for i, r in ((1, M), (3, N)))
    y = (a @ b.T).astype(np.float32) * sa[:, None] * sb[None, :]
    ok = _same(_rows(c, 4, M, N, "post"), _bf16(y))
    return ok, "M=%d N=%d K=%d elements %s" % (M, N, K, "bit-exact" if ok else "DIFFER")


def check_band(c):
    n = c.geti("n")
    norm, gated = c.row == "rmsnorm_quant_i8", c.row == "gated_quant_i8"
    rows = _numel(c.tensors[0]) // (2 * n if gated else n)
    x = _rows(c, 0, rows, 2 * n if gated else n, "pre").astype(np.float64)
    flush, ok = 0.0, True
    with np.errstate(all="ignore"):
        if norm:
            if c.present(1):
                s = _bf16(x.astype(np.float32) + _rows(c, 1, rows, n, "pre"))
                x = _rows(c, 6, rows, n, "post").astype(np.float64)
                ok = _same(x, s)
            w = _rows(c, 2, 1, n, "pre").astype(np.float64) + c.getf("wadd", 0.0)
            h = x / np.sqrt((x * x).mean(1, keepdims=True) + c.getf("eps", 1e-6)) * w
        elif gated:
            g, up = x[:, :n], x[:, n:]
            sg = 1.0 / (1.0 + np.exp(-g))
            h = (sg if c.gets("act") == "sigmoid" else g * sg) * up
            flush = 2.0 ** -126 * (1 + np.abs(g)) * np.abs(up)
        else:
            h = x
    iq = 3 if norm else 1
    q = _rows(c, iq, rows, n, "post").astype(np.float64)
    s = np.asarray(_column(c, iq + 1, rows, "post"), np.float64)
    fin = np.isfinite(h).all(1)
    amax = np.abs(h).max(1)
    want = np.where(amax > 0, np.maximum(amax / 127, 2.0 ** -126), 1.0)
    tol = np.max(flush * np.ones_like(h), 1) / 127 if gated else 0.0
    ok = ok and bool(np.all((np.abs(s - want) <= 2.0 ** -20 * want + tol)[fin])) and not np.isfinite(s[~fin]).any()
    lim = 0.5 + 127 * 2.0 ** -20 + flush / s[:, None] * 2
    with np.errstate(all="ignore"):
        ok = ok and bool(np.all((np.abs(h / s[:, None] - q) <= lim)[fin])) and not q[~fin].any()
    if not c.row.startswith("quant") and c.present(iq + 2):
        out = _rows(c, iq + 2, rows, n, "post")
        r = 2.0 ** -20 + (2.0 ** -8 if c.tensors[iq + 2]["dt"] == BF16 else 0.0)
        ok = ok and bool(np.all((np.abs(out - h) <= r * np.abs(h) + flush + 2.0 ** -133)[fin]))
    return ok, "rows=%d n=%d codes and scales %s" % (rows, n, "within the bound" if ok else "DIFFER")


def _token(x, u, T, k, p, m):
    """The token, and its share of the kept mass."""
    x = x.astype(np.float64)
    there = x > -np.inf
    if not there.any():
        return -1, 0.0
    x = np.where(there, x, -np.inf)
    if not T > 0:
        return int(np.argmax(x)), 1.0
    with np.errstate(all="ignore"):
        w = np.nan_to_num(np.where(x == x.max(), 1.0, np.exp((x - x.max()) / T)), nan=0.0)
    order = np.lexsort((np.arange(len(x)), -x))
    order = order[there[order]]
    order = order[:k] if k > 0 else order
    if p < 1:
        cum = np.cumsum(w[order])
        order = order[:max(int(np.sum(cum - w[order] < p * cum[-1])), 1)]
    order = order[w[order] >= min(m, 1.0)] if m > 0 else order
    kept = np.sort(order)
    cum = np.cumsum(w[kept])
    i = min(int(np.searchsorted(cum, max(u, 0.0) * cum[-1], side="right")), len(kept) - 1)
    while w[kept[i]] == 0:
        i -= 1
    return int(kept[i]), float(w[kept[i]] / cum[-1])


def check_sample(c):
    V = c.geti("n_vocab")
    M = _numel(c.tensors[0]) // V
    x = _rows(c, 0, M, V, "pre")
    col = [_column(c, i, M, "pre", d) for i, d in ((1, 0.0), (2, 1.0), (3, 0), (4, 1.0), (5, 0.0))]
    got, prob = _column(c, 6, M, "post"), _column(c, 7, M, "post")
    want = [_token(x[r], *[v[r] for v in col]) for r in range(M)]
    bits = max(V - 1, 0).bit_length()
    rel = 2.0 ** -23 + V * 2.0 ** -min(62 - bits, 51)
    bad = [r for r in range(M) if got[r] != want[r][0]]
    off = [r for r in range(M) if prob[r] is not None and not abs(prob[r] - want[r][1]) <= rel * want[r][1] + 2.0 ** -126]
    return not bad and not off, "M=%d V=%d tokens %s%s" % (
        M, V, "equal" if not bad else "differ in rows %s" % bad[:8],
        "" if not off else ", probabilities in rows %s" % off[:8])


def check(c):
    if c.row == "sample_logits":
        return check_sample(c)
    return check_gemm(c) if c.row.startswith("gemm") else check_band(c)
