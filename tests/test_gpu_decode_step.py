"""The int8 layer and the sampler as a decode step uses them: norm -> gate and up product -> gated
producer -> down product -> norm with the residual -> lm_head -> token.  Each stage is held against
64 bits on the inputs that it got (codes, sums and tokens of the stage before are compared there), and
the captured step against the eager one bit for bit.

Bounds: h of the norm is off by the roundings of rs, of two products and of the weight's own use,
4 * 2^-24 < 2^-21 relative; of the gated producer by 2^-21 (its sigmoid within 3 ulp and two products).
A scale adds the roundings of 1/127 and of its product, a code those of 1/s and of h * (1/s): a code lies
within 1/2 + 127 * 2^-20 of h / s.  An element of a product over K e4m3 codes with one scale a block of
128 is off by no more than K + K / 128 + 2 roundings of partial sums that stay below the sum of magnitudes."""
import numpy as np
import pytest
import torch

import libr3d_amd as R

pytestmark = pytest.mark.gpu


def plain_token(x, u, T, k, p, m):
    """The token of one row of float32 logits, in float64."""
    x = np.asarray(x, np.float64)
    if not T > 0:
        return int(np.argmax(x))
    w = np.exp((x - x.max()) / T)
    order = np.lexsort((np.arange(len(x)), -x))
    if k > 0:
        order = order[:k]
    if p < 1:
        c = np.cumsum(w[order])
        order = order[:max(int(np.sum(c - w[order] < p * c[-1])), 1)]
    order = order[w[order] >= m]
    kept = np.sort(order)
    c = np.cumsum(w[kept])
    return int(kept[min(int(np.searchsorted(c, u * c[-1], side="right")), len(kept) - 1)])


class Step:
    def __init__(self, dev, M, E, F, V, seed):
        g = torch.Generator().manual_seed(seed)
        self.M, self.E, self.F, self.V, self.dev = M, E, F, V, dev
        code = lambda *s: torch.randint(-127, 128, s, generator=g, dtype=torch.int32).to(torch.int8)  # noqa: E731
        self.gu, self.gu_s = code(2 * F, E), torch.rand(2 * F, generator=g) * 2e-3 + 1e-4
        self.dn, self.dn_s = code(E, F), torch.rand(E, generator=g) * 2e-3 + 1e-4
        self.w1, self.w2 = (1 + 0.1 * torch.randn(2, E, generator=g)).bfloat16()
        rng = np.random.default_rng(seed)
        self.head = rng.integers(0, 256, (V, E), dtype=np.uint8)
        self.head[(self.head & 127) == 127] = 0                      # no NaN
        self.head_s = (2e-4 + 4e-4 * torch.rand(V, E // 128, generator=g)).bfloat16()
        self.blob = torch.from_numpy(R.join_head(self.head, self.head_s.view(torch.int16).numpy().view(np.uint16)))
        for n in ("gu", "gu_s", "dn", "dn_s", "w1", "w2", "blob"):
            setattr(self, n + "_d", getattr(self, n).to(dev))
        self.T = torch.tensor([1.0, 0.7, 0.0, 1.3, 1.0])[torch.arange(M) % 5].clone()
        self.k = torch.tensor([0, 40, 0, 7, 300], dtype=torch.int32)[torch.arange(M) % 5].clone()
        self.p = torch.tensor([1.0, 0.9, 1.0, 0.5, 0.95, 0.8])[torch.arange(M) % 6].clone()
        self.m = torch.tensor([0.0, 0.0, 0.05])[torch.arange(M) % 3].clone()
        z = lambda *s, dt=torch.float32: torch.zeros(*s, dtype=dt, device=dev)  # noqa: E731
        b16, i8 = torch.bfloat16, torch.int8
        self.x, self.r = z(M, E, dt=b16), z(M, E, dt=b16)
        self.q1, self.s1 = z(M, E, dt=i8), z(M)
        self.y1, self.q2, self.s2 = z(M, 2 * F, dt=b16), z(M, F, dt=i8), z(M)
        self.y2, self.r2 = z(M, E, dt=b16), z(M, E, dt=b16)
        self.q3, self.s3, self.h3 = z(M, E, dt=i8), z(M), z(M, E, dt=b16)
        self.logits, self.u = z(M, V), z(M)
        self.token, self.prob = z(M, dt=torch.int32), z(M)
        self.set_d = [t.to(dev) for t in (self.T, self.k, self.p, self.m)]
        self.g = g

    def inputs(self):
        self.x.copy_(torch.randn(self.M, self.E, generator=self.g))
        self.r.copy_(3 * torch.randn(self.M, self.E, generator=self.g))
        self.u.copy_(torch.rand(self.M, generator=self.g))

    OUT = ("q1", "s1", "y1", "q2", "s2", "y2", "r2", "q3", "s3", "h3", "logits", "token", "prob")

    def clear(self):
        for n in self.OUT:
            getattr(self, n).zero_()

    def run(self):
        E, F, V = self.E, self.F, self.V
        assert R.rmsnorm_quant_i8(self.x, None, self.w1_d, self.q1, self.s1, n=E) == R.RAD_OK
        assert R.gemm_nt_q(self.q1, self.s1, self.gu_d, self.gu_s_d, self.y1, dtype="i8a8", N=2 * F, K=E)[0] == R.RAD_OK
        assert R.gated_quant_i8(self.y1, self.q2, self.s2, n=F) == R.RAD_OK
        assert R.gemm_nt_q(self.q2, self.s2, self.dn_d, self.dn_s_d, self.y2, dtype="i8a8", N=E, K=F)[0] == R.RAD_OK
        assert R.rmsnorm_quant_i8(self.y2, self.r, self.w2_d, self.q3, self.s3, self.h3, n=E,
                                  residual_out=self.r2) == R.RAD_OK
        assert R.logits_gemm(self.h3, self.blob_d, self.logits, n_vocab=V, n_embd=E) == R.RAD_OK
        T, k, p, m = self.set_d
        assert R.sample_logits(self.logits, self.u, self.token, self.prob, n_vocab=V, temperature=T, top_k=k,
                               top_p=p, min_p=m) == R.RAD_OK

    def outputs(self):
        torch.cuda.synchronize()
        return [getattr(self, n).cpu().clone() for n in self.OUT]


def check_codes(h, q, s):
    """Codes and scales of rows h (float64)."""
    want = h.abs().amax(1) / 127
    assert ((s.double() - want).abs() <= 2.0 ** -20 * want).all()
    assert ((h / s.double()[:, None] - q.double()).abs() <= 0.5 + 127 * 2.0 ** -20).all()


def check_product(a, sa, b, sb, y):
    s = (a.double() @ b.double().T).numpy().astype(np.int64).astype(np.float32)
    want = torch.from_numpy((s * sa.numpy()[:, None]).astype(np.float32) * sb.numpy()[None, :]).bfloat16()
    assert torch.equal(y.view(torch.int16), want.view(torch.int16))


def normed(r, w, eps=1e-6):
    r = r.double()
    return r / torch.sqrt((r * r).mean(1, keepdim=True) + eps) * w.double()


@pytest.mark.parametrize("M,E,F,V", [(1, 512, 1376, 5000), (5, 1024, 1000, 3001), (24, 512, 2704, 9000)])
def test_step(gpu, M, E, F, V):
    st = Step(gpu, M, E, F, V, seed=M)
    st.inputs()
    st.run()
    q1, s1, y1, q2, s2, y2, r2, q3, s3, h3, logits, token, prob = st.outputs()
    check_codes(normed(st.x.cpu(), st.w1), q1, s1)
    check_product(q1, s1, st.gu, st.gu_s, y1)
    gate, up = y1.double()[:, :F], y1.double()[:, F:]
    check_codes(gate * torch.sigmoid(gate) * up, q2, s2)
    check_product(q2, s2, st.dn, st.dn_s, y2)
    r = (y2.float() + st.r.cpu().float()).bfloat16()
    assert torch.equal(r, r2)
    h = normed(r, st.w2)
    check_codes(h, q3, s3)
    assert ((h3.double() - h).abs() <= h.abs() * (2.0 ** -8 + 2.0 ** -20)).all()
    c = torch.from_numpy(st.head).view(torch.float8_e4m3fn).double() * st.head_s.double().repeat_interleave(128, 1)
    lim = h3.double().abs() @ c.abs().T * ((E + E // 128 + 2) * 2.0 ** -24)
    assert ((logits.double() - h3.double() @ c.T).abs() <= lim).all()
    for i in range(M):
        want = plain_token(logits[i].numpy(), float(st.u[i]), float(st.T[i]), int(st.k[i]), float(st.p[i]), float(st.m[i]))
        assert int(token[i]) == want, i


def test_captured_step(gpu):
    """Two graphs of two steps of different sizes, each with a pool of its own, replayed in turn over new
    inputs with eager steps between; bit for bit."""
    steps = [Step(gpu, 3, 512, 1376, 5000, seed=11), Step(gpu, 17, 512, 1376, 5000, seed=12)]
    graphs = []
    for st in steps:
        st.inputs()
        st.run()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            st.run()
        graphs.append(graph)
    for turn in range(3):
        for st in steps:
            st.inputs()
            st.clear()
        for graph in graphs:
            graph.replay()
        got = [st.outputs() for st in steps]
        for st, outs in zip(steps, got):
            st.clear()
            st.run()
            for name, a, b in zip(st.OUT, outs, st.outputs()):
                assert torch.equal(a, b), (turn, name)
