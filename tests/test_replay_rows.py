"""The host replay of captured int8 and sampler launches tells a wrong output from a right one: captures made
here, on the CPU, with one output changed by the least that it can be."""
import numpy as np
import pytest

from tests import replay_rows as RR
from tests.replay_dump import Capture
from tests.test_gpu_sample import plain


def bf16(v):
    """Bits of float32 values, to nearest even."""
    u = np.asarray(v, np.float32).view(np.uint32).astype(np.uint64)
    return np.where(np.isnan(v), 0x7FC0, (u + 0x7FFF + (u >> 16 & 1)) >> 16).astype(np.uint16)


def wide(bits):
    return (np.asarray(bits, np.uint16).astype(np.uint32) << 16).view(np.float32)


DT = {np.dtype(np.float32): 0, np.dtype(np.uint16): 1, np.dtype(np.int8): 8, np.dtype(np.int32): 10}


def capture(row, params, pre, post):
    """A capture of dense operands; `post` {index: array} differs from `pre`; None is an absent operand."""
    c = Capture.__new__(Capture)
    c.row, c.rc, c.tunables, c.scratch = row, 0, [], None
    c.params = {k: (0, v, 0, "", 0.0) if isinstance(v, int) else (1, 0, 0, v, 0.0) if isinstance(v, str)
                else (2, 0, 0, "", v) for k, v in params.items()}
    c.tensors, c.pre, c.post = [], [], []
    for i, t in enumerate(pre):
        if t is None:
            c.tensors.append(dict(dt=0, rank=0, shape=[], stride=[], bytes=0, trunc=0, null=1))
            c.pre.append(np.zeros(0, np.uint8)), c.post.append(np.zeros(0, np.uint8))
            continue
        t = np.ascontiguousarray(t)
        stride = [int(np.prod(t.shape[j + 1:], dtype=np.int64)) for j in range(t.ndim)]
        c.tensors.append(dict(dt=DT[t.dtype], rank=t.ndim, shape=list(t.shape), stride=stride, bytes=t.nbytes, trunc=0,
                              null=0))
        c.pre.append(t.view(np.uint8).ravel().copy())
        c.post.append(np.ascontiguousarray(post.get(i, t)).view(np.uint8).ravel().copy())
    return c


def norm(change=None, special=False):
    rng = np.random.default_rng(3)
    M, n, eps = 3, 40, 1e-6
    x, r = bf16(rng.standard_normal((M, n))), bf16(4 * rng.standard_normal((M, n)))
    if special:
        x[0, 5] = 0x7F80                                       # an infinity in the first row
    w = bf16(1 + 0.1 * rng.standard_normal(n))
    added = bf16(wide(x) + wide(r))
    out = added.copy()
    if change:
        change(out, wide(x) + wide(r))
    v = wide(out).astype(np.float64)
    with np.errstate(all="ignore"):
        h = v / np.sqrt((v * v).mean(1, keepdims=True) + eps) * wide(w)
        s = (np.abs(h).max(1) / 127).astype(np.float32)
        q = np.where(np.isfinite(s)[:, None], np.rint(h / s[:, None]), 0).astype(np.int8)
    zero = [np.zeros((M, n), np.int8), np.zeros(M, np.float32), None, np.zeros((M, n), np.uint16)]
    return capture("rmsnorm_quant_i8", dict(n=n, M=M, eps=eps, dtype="bf16"), [x, r, w] + zero, {3: q, 4: s, 6: out})


def one_step(out, exact):
    out[1, 7] += 1


def cut(out, exact):
    """Cut off instead of rounded."""
    out[1:] = (exact[1:].view(np.uint32) >> 16).astype(np.uint16)


@pytest.mark.parametrize("special", [False, True])
def test_residual_out(special):
    ok, text = RR.check(norm(special=special))
    assert ok, text
    for change in (one_step, cut):
        assert not RR.check(norm(change, special))[0], change.__name__


def sample(factor=1.0, prob=True):
    rng = np.random.default_rng(4)
    M, V = 5, 300
    x, u = (2 * rng.standard_normal((M, V))).astype(np.float32), rng.random(M).astype(np.float32)
    x[4] = -np.inf
    T, k = np.array([1, 0.7, 0, 2, 1], np.float32), np.array([0, 40, 0, 7, 0], np.int32)
    p = np.array([1, 0.9, 1, 0.5, 0.5], np.float32)
    want = [plain(x[i], float(u[i]), float(T[i]), int(k[i]), float(p[i])) for i in range(M)]
    post = {6: np.array([t for t, _ in want], np.int32)}
    share = np.array([s for _, s in want], np.float32)
    share[1] *= np.float32(factor)
    if prob:
        post[7] = share
    return capture("sample_logits", dict(n_vocab=V, M=M, dtype="f32"),
                   [x, u, T, k, p, None, np.zeros(M, np.int32), np.zeros(M, np.float32) if prob else None], post)


def test_probability():
    for prob in (True, False):
        ok, text = RR.check(sample(prob=prob))
        assert ok, text
    for factor in (1 + 2.0 ** -20, 0.0, float("nan"), -1.0):
        assert not RR.check(sample(factor))[0], factor
    c = sample()
    c.post[6].view(np.int32)[0] += 1
    assert not RR.check(c)[0]
