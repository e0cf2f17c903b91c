"""The sample_logits row on the GPU against a plain float64 sampler on the CPU: the tokens have to
be equal, the probability within two f32 roundings and the masses' 2^-44.  The row's masses are off
by at most 2^-44 a token, so a token could only differ where u falls within about 2^-35 of a border;
no case here lies there (uniform numbers have 24 bits and the borders are exact or generic)."""
import numpy as np
import pytest
import torch

import libr3d_amd as R

pytestmark = pytest.mark.gpu


def plain(x, u, T=1.0, k=0, p=1.0, m=0.0):
    """(token, probability, runner-up margin) of one row of float32 logits."""
    x = np.asarray(x, np.float64)
    there = x > -np.inf
    if not there.any():
        return -1, 0.0
    x = np.where(there, x, -np.inf)
    top = x.max()
    if not T > 0:
        return int(np.argmax(x)), 1.0
    with np.errstate(all="ignore"):
        w = np.where(x == top, 1.0, np.exp((x - top) / T))
    w = np.where(there & ~np.isnan(w), w, 0.0)
    order = np.lexsort((np.arange(len(x)), -x))
    order = order[there[order]]
    if k > 0:
        order = order[:k]
    if p < 1:
        c = np.cumsum(w[order])
        before = c - w[order]
        n = int(np.sum(before < p * c[-1]))
        order = order[:max(n, 1)]
    if m > 0:
        order = order[w[order] >= min(m, 1.0)]
    kept = np.sort(order)
    c = np.cumsum(w[kept])
    i = min(int(np.searchsorted(c, (u if u > 0 else 0.0) * c[-1], side="right")), len(kept) - 1)
    while w[kept[i]] == 0:                      # u = 1: the last token with any mass
        i -= 1
    return int(kept[i]), float(w[kept[i]] / c[-1])


def check(dev, x, u, T=None, k=None, p=None, m=None, pitch=None, off=0, stream=None, label=""):
    M, V = x.shape
    if pitch:
        buf = torch.full((off + M * pitch,), 1e30, dtype=x.dtype, device=dev)   # what must not be read
        xd = buf[off:].as_strided((M, V), (pitch, 1))
        xd.copy_(x)
    else:
        xd = x.to(dev)
    d = lambda t, dt: None if t is None else torch.as_tensor(t, dtype=dt).to(dev)  # noqa: E731
    token = torch.full((M + 2,), -77, dtype=torch.int32, device=dev)
    prob = torch.full((M + 2, 1), -5.0, device=dev)
    print("sample", M, V, x.dtype, label, flush=True)
    rc = R.sample_logits(xd, d(u, torch.float32), token[1:M + 1], prob[1:M + 1], n_vocab=V,
                         temperature=d(T, torch.float32), top_k=d(k, torch.int32), top_p=d(p, torch.float32),
                         min_p=d(m, torch.float32), stream=stream)
    assert rc == R.RAD_OK
    torch.cuda.synchronize()
    f = lambda t, i, dflt: dflt if t is None else float(torch.as_tensor(t, dtype=torch.float32).reshape(-1)[i])  # noqa: E731
    want = [plain(x[i].float().numpy(), f(u, i, 0), f(T, i, 1.0), int(f(k, i, 0)), f(p, i, 1.0), f(m, i, 0.0))
            for i in range(M)]
    got = token.cpu().tolist()
    assert got[0] == got[-1] == -77
    bad = [(i, got[i + 1], want[i]) for i in range(M) if got[i + 1] != want[i][0]]
    assert not bad, bad[:5]
    pr = prob.cpu().double()[:, 0]
    assert pr[0] == pr[-1] == -5.0
    w = torch.tensor([t[1] for t in want], dtype=torch.float64)
    assert ((pr[1:-1] - w).abs() <= 2.0 ** -22 * w + 2.0 ** -40).all()


def settings(g, M):
    pick = lambda v: torch.tensor(v)[torch.randint(0, len(v), (M,), generator=g)]  # noqa: E731
    return dict(T=pick([0.0, 0.3, 0.7, 1.0, 1.0, 2.0, -1.0]), k=pick([0, 0, -3, 1, 2, 7, 50, 1000, 10 ** 6]).int(),
                p=pick([1.0, 1.0, 2.0, 0.99, 0.9, 0.5, 0.01, 0.0]), m=pick([0.0, 0.0, -1.0, 0.01, 0.2, 1.0, 3.0]))


@pytest.mark.parametrize("V", [1, 2, 3, 7, 64, 100, 1000, 4095, 4096, 4097, 8193, 32000, 50257, 131075])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_settings(gpu, V, dtype):
    g = torch.Generator().manual_seed(V)
    M = 40
    x = (3 * torch.randn(M, V, generator=g)).to(dtype)
    u = torch.rand(M, generator=g)
    u[0], u[1], u[2], u[3] = 0.0, 1.0, 1 - 2.0 ** -24, -1.0
    check(gpu, x, u, **settings(g, M))
    check(gpu, x, u, **settings(g, M), pitch=V + 3, off=1)
    check(gpu, x, u)


def test_each_cut_alone(gpu):
    g = torch.Generator().manual_seed(2)
    M, V = 24, 10000
    x, u = 2 * torch.randn(M, V, generator=g), torch.rand(M, generator=g)
    check(gpu, x, u, T=torch.linspace(0.05, 30, M))
    check(gpu, x, u, k=torch.arange(1, M + 1) ** 3)
    check(gpu, x, u, p=torch.linspace(0.0, 1.0, M))
    check(gpu, x, u, m=torch.linspace(0.0, 1.1, M))
    check(gpu, x, u, k=torch.full((M,), 300), p=torch.linspace(0.02, 0.999, M))
    check(gpu, x, u, T=torch.full((M,), 5.0), k=torch.full((M,), 9000), p=torch.linspace(0.02, 0.999, M))
    check(gpu, x, u, p=torch.full((M,), 0.9), m=torch.linspace(0.0, 0.5, M))


def test_every_token_in_turn(gpu):
    """Eight equal logits: u = i / 8 is the border itself, and belongs to token i."""
    x = torch.full((8, 40), float("-inf"))
    x[:, 3:40:5] = 1.5
    u = torch.arange(8) / 8.0
    check(gpu, x, u)
    token = torch.empty(8, dtype=torch.int32, device=gpu)
    assert R.sample_logits(x.to(gpu), u.to(gpu), token, n_vocab=40) == R.RAD_OK
    assert token.cpu().tolist() == list(range(3, 40, 5))
    check(gpu, x, u, k=torch.full((8,), 4))                      # ties: the lowest indices
    check(gpu, x, u, p=torch.full((8,), 0.5))
    check(gpu, x, u, p=torch.full((8,), 0.51))


@pytest.mark.parametrize("V", [9000, 70001])
def test_many_equal_logits(gpu, V):
    """More tokens in a border bin than the list holds: equal ones, two levels of them, and bf16
    values in clusters; the cuts land inside the ties."""
    g = torch.Generator().manual_seed(V)
    M = 12
    u = torch.rand(M, generator=g)
    flat = torch.zeros(M, V)
    two = torch.where(torch.rand(M, V, generator=g) < 0.3, 0.0, -0.7)
    few = torch.randint(-3, 3, (M, V), generator=g) * 0.125
    far = 1e-4 * torch.randn(M, V, generator=g)                   # one cluster, and one token far below
    far[:, 5] = -30.0
    for label, x in (("flat", flat), ("two", two), ("few", few), ("far", far), ("zeros", -0.0 * two.sign())):
        check(gpu, x, u, label=label)
        check(gpu, x, u, k=torch.linspace(1, V - 1, M).int(), label=label)
        check(gpu, x, u, p=torch.linspace(0.01, 0.99, M), label=label)
        check(gpu, x, u, k=torch.linspace(V // 2, V - 1, M).int(), p=torch.linspace(0.05, 0.99, M),
              m=torch.tensor([0.0, 0.6] * 6), label=label)
        check(gpu, x.bfloat16(), u, k=torch.linspace(1, V - 1, M).int(), p=torch.linspace(0.99, 0.05, M), label=label)


def test_masked_rows(gpu):
    """Rows with nothing, one token, NaN, infinities, and the lowest number of the type as a mask."""
    V = 5000
    inf = float("inf")
    x = torch.full((10, V), -inf)
    x[1, 4321] = -1e30
    x[2, 7], x[2, 8] = float("nan"), 0.25
    x[3] = float("nan")
    x[4, 100], x[4, 200], x[4, 300] = inf, inf, 5.0
    x[5] = torch.finfo(torch.float32).min
    x[5, 77] = 0.0
    x[6] = torch.finfo(torch.float32).min
    x[7, :2] = torch.tensor([3e38, -3e38])
    x[8, 10:20] = 1e-42                                          # subnormal differences
    x[8, 15] = 3e-42
    x[9, 4999] = 2.0
    u = torch.linspace(0, 0.99, 10)
    for kw in ({}, dict(k=[3] * 10), dict(p=[0.7] * 10), dict(k=[2] * 10, p=[0.7] * 10, m=[0.1] * 10), dict(T=[0.0] * 10),
               dict(T=[1e-30] * 10, k=[5] * 10), dict(T=[inf] * 10, k=[5] * 10, p=[0.5] * 10), dict(T=[float("nan")] * 10)):
        check(gpu, x, u, label=str(kw), **kw)


def test_one_setting_for_all_rows_and_streams(gpu):
    g = torch.Generator().manual_seed(11)
    M, V = 6, 20000
    x, u = 3 * torch.randn(M, V, generator=g), torch.rand(M, generator=g)
    xd, ud = x.to(gpu), u.to(gpu)
    T = torch.tensor([0.8], device=gpu).expand(M)
    k = torch.tensor([[40]], dtype=torch.int32, device=gpu).expand(M, 1)
    torch.cuda.synchronize()
    outs = []
    for s in (torch.cuda.Stream(), torch.cuda.Stream()):          # two calls at once
        token = torch.zeros(M, dtype=torch.int32, device=gpu)
        torch.cuda.synchronize()
        assert R.sample_logits(xd, ud, token, n_vocab=V, temperature=T, top_k=k, stream=s.cuda_stream) == R.RAD_OK
        outs.append(token)
    torch.cuda.synchronize()
    want = [plain(x[i].numpy(), float(u[i]), float(np.float32(0.8)), 40)[0] for i in range(M)]
    assert outs[0].cpu().tolist() == outs[1].cpu().tolist() == want


def test_captured_and_repeated(gpu):
    """A captured launch replayed over new logits and numbers, on dirty scratch, and the same bits
    from every run."""
    g = torch.Generator().manual_seed(12)
    M, V = 5, 30000
    x, u = torch.zeros(M, V, device=gpu), torch.zeros(M, device=gpu)
    p, k = torch.full((M,), 0.8, device=gpu), torch.full((M,), 200, dtype=torch.int32, device=gpu)
    token, prob = torch.zeros(M, dtype=torch.int32, device=gpu), torch.zeros(M, device=gpu)
    ops = R.SampleOperands(x, u, token, prob, n_vocab=V, top_p=p, top_k=k)
    scratch = torch.full((R.row_scratch_bytes("sample_logits", ops),), 0xA5, dtype=torch.uint8, device=gpu)
    ops.set_scratch(scratch)
    x.copy_(2 * torch.randn(M, V, generator=g))
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        assert R.launch_row("sample_logits", ops, torch.cuda.current_stream().cuda_stream) == R.RAD_OK
    for i in range(4):
        xc, uc = 2 * torch.randn(M, V, generator=g), torch.rand(M, generator=g)
        x.copy_(xc), u.copy_(uc)
        scratch.fill_(0xA5 + i)
        seen = set()
        for _ in range(3):
            graph.replay()
            torch.cuda.synchronize()
            seen.add((tuple(token.cpu().tolist()), tuple(prob.cpu().tolist())))
        assert len(seen) == 1
        want = [plain(xc[j].numpy(), float(uc[j]), 1.0, 200, float(np.float32(0.8)))[0] for j in range(M)]
        assert list(seen.pop()[0]) == want


def test_short_or_missing_scratch_is_refused(gpu):
    x, u = torch.zeros(2, 100, device=gpu), torch.zeros(2, device=gpu)
    token = torch.full((2,), -7, dtype=torch.int32, device=gpu)
    ops = R.SampleOperands(x, u, token, n_vocab=100)
    assert R.launch_row("sample_logits", ops) == R.RAD_E_UNSUPPORTED
    need = R.row_scratch_bytes("sample_logits", ops)
    buf = torch.empty(need + 16, dtype=torch.uint8, device=gpu)
    ops.set_scratch(buf, need - 1)
    assert R.launch_row("sample_logits", ops) == R.RAD_E_UNSUPPORTED
    ops.set_scratch(buf[8:], need)
    assert R.launch_row("sample_logits", ops) == R.RAD_E_UNSUPPORTED
    torch.cuda.synchronize()
    assert token.cpu().tolist() == [-7, -7]


def test_frequencies(gpu):
    """4096 numbers spread evenly over one row: every kept token as often as its share, within one."""
    V, M = 600, 4096
    g = torch.Generator().manual_seed(1)
    row = 1.5 * torch.randn(V, generator=g)
    x = row.to(gpu).expand(M, V)
    u = (torch.arange(M) + 0.5) / M
    token = torch.empty(M, dtype=torch.int32, device=gpu)
    k = torch.tensor([30], dtype=torch.int32, device=gpu).expand(M)
    assert R.sample_logits(x, u.to(gpu), token, n_vocab=V, top_k=k) == R.RAD_OK
    n = torch.bincount(token.cpu().long(), minlength=V).double()
    w = torch.exp(row.double())
    w[row.argsort(descending=True)[30:]] = 0
    assert ((n - M * w / w.sum()).abs() <= 1.0 + 1e-6).all()
