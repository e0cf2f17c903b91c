"""The norms between blocks, the router's product, the expert layer and a quantised projection as a decoder layer runs
them: one stream, one workspace, each step held against 64 bits of what the step before it wrote, and the whole
captured and replayed."""
import pytest
import torch

import libr3d_amd as R
from tests import block_util as B
from tests import epi_util as E
from tests import moe_util as U
from tests.test_gpu_moe import experts

pytestmark = pytest.mark.gpu


class Layer:
    """The half of a decoder layer behind its attention, and the next one's first projection; `scratch` may be shared."""

    def __init__(self, dev, M, n, f, E_, k, dtype, act="silu", score="softmax", seed=0):
        g = torch.Generator().manual_seed(seed)
        r = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
        self.M, self.n, self.f, self.E, self.k, self.dtype, self.act, self.score, self.dev = M, n, f, E_, k, dtype, act, score, dev
        on = lambda t: None if t is None else t.to(dev)  # noqa: E731
        self.w_attn, self.w_ffn, self.w_out, self.w_next = ((1 + 0.1 * r(n)).bfloat16().to(dev) for _ in range(4))
        self.gate = (0.7 + 0.2 * r(n)).bfloat16().to(dev)
        self.router, self.router_bias = (2 * r(E_, n) * n ** -0.5).bfloat16().to(dev), (0.1 * r(E_)).to(dev)
        self.gu, self.gus = map(on, experts(g, dtype, E_, 2 * f, n))
        self.dn, self.dns = map(on, experts(g, dtype, E_, n, f))
        self.N = n + 40
        self.proj = torch.randint(-127, 128, (self.N, n), generator=g, dtype=torch.int32).to(torch.int8).to(dev)
        self.proj_scale = ((0.5 + torch.rand(self.N, generator=g)) * n ** -0.5 / 74).to(dev)
        self.proj_bias = r(self.N).bfloat16().to(dev)
        new = lambda *s, t=torch.bfloat16: torch.zeros(*s, dtype=t, device=dev)  # noqa: E731
        self.attn, self.res, self.h1, self.x, self.y, self.h2 = (new(M, n) for _ in range(6))
        self.logits, self.ids, self.weights = new(M, E_, t=torch.float32), new(M, k, t=torch.int32), new(M, k, t=torch.float32)
        self.q, self.qs, self.out = new(M, n, t=torch.int8), new(M, t=torch.float32), new(M, self.N)
        self.steps = [
            ("rmsnorm_block", R.RmsNormBlockOperands(self.attn, n=n, residual=self.res, w_post=self.w_attn, w_pre=self.w_ffn,
                                                     residual_out=self.h1, out=self.x)),
            ("gemm_nt_epi", R.GemmEpiOperands(self.x, self.router, self.logits, bias=self.router_bias, dtype="bf16", N=E_, K=n)),
            ("moe_layer", R.MoeLayerOperands(self.x, self.logits, self.gu, self.dn, self.y, gate_up_scale=self.gus,
                                             down_scale=self.dns, ids=self.ids, weights=self.weights, act=act, score=score,
                                             dtype=dtype, n=n, f=f, E=E_, top_k=k)),
            ("rmsnorm_block", R.RmsNormBlockOperands(self.y, n=n, residual=self.h1, w_post=self.w_out, gate=self.gate,
                                                     w_pre=self.w_next, residual_out=self.h2, q=self.q, scale=self.qs)),
            ("gemm_nt_epi", R.GemmEpiOperands(self.q, self.proj, self.out, a_scale=self.qs, b_scale=self.proj_scale,
                                              bias=self.proj_bias, dtype="i8a8", N=self.N, K=n))]
        self.rows = [R.resolve(op, {"M": M, "N": E_ if i == 1 else self.N, "K": n, "n": n, "dtype": (None, "bf16", dtype,
                                    None, "i8a8")[i] or "bf16"})["name"] for i, (op, _) in enumerate(self.steps)]
        self.need = max(R.row_scratch_bytes(row, ops) for row, (_, ops) in zip(self.rows, self.steps))

    def share(self, scratch):
        for _, ops in self.steps:
            ops.set_scratch(scratch)

    def inputs(self, seed):
        g = torch.Generator().manual_seed(1000 + seed)
        self.attn.copy_(torch.randn(self.M, self.n, generator=g))
        self.res.copy_(2 * torch.randn(self.M, self.n, generator=g))

    def run(self):
        s = torch.cuda.current_stream().cuda_stream
        for row, (_, ops) in zip(self.rows, self.steps):
            assert R.launch_row(row, ops, s) == R.RAD_OK, row

    def outputs(self):
        return [t.clone() for t in (self.h1, self.x, self.logits, self.ids, self.weights, self.y, self.h2, self.q, self.qs, self.out)]

    def check(self):
        h, eh, v, ev = B.exact(self.attn, self.res, self.w_attn, None, self.w_ffn)
        B.check("h1", self.h1, h, eh)
        B.check("x", self.x, v, ev)
        E.check(self.logits, *E.exact(self.x, self.router, bias=self.router_bias))
        U.check((self.y, self.ids, self.weights),
                U.exact(self.x, self.logits, self.gu, self.dn, self.dtype, self.f, self.k, self.gus, self.dns, self.act, self.score))
        h, eh, v, ev = B.exact(self.y, self.h1, self.w_out, self.gate, self.w_next)
        B.check("h2", self.h2, h, eh)
        B.check_i8(self.q, self.qs, v, ev)
        E.check(self.out, *E.exact(self.q, self.proj, self.qs, self.proj_scale, self.proj_bias))


SIZES = [(1, 1344, 320, 40, 4, "mxfp4"), (4, 512, 256, 16, 2, "i8"), (13, 640, 352, 32, 4, "bf16"), (64, 512, 224, 32, 8, "mxfp4")]


@pytest.mark.parametrize("M,n,f,experts_,k,dtype", SIZES)
def test_layer(gpu, M, n, f, experts_, k, dtype):
    """Eager, with one workspace for every step, then captured: each replay gives what the eager run gave, bit for bit,
    with eager work of the same operators between the replays."""
    L = Layer(gpu, M, n, f, experts_, k, dtype)
    L.share(torch.full((L.need,), 0xFF, dtype=torch.uint8, device=gpu))
    eager = []
    for seed in range(3):
        L.inputs(seed)
        L.run()
        torch.cuda.synchronize()
        L.check()
        eager.append(L.outputs())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        L.run()
    other = Layer(gpu, M, n, f, experts_, k, dtype, seed=5)
    other.share(torch.full((other.need,), 0x11, dtype=torch.uint8, device=gpu))
    for seed in (1, 0, 2, 1):
        L.inputs(seed)
        for t in (L.h1, L.x, L.logits, L.y, L.h2, L.out):
            t.fill_(-3)
        L.ids.fill_(-5)
        graph.replay()
        got = L.outputs()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, eager[seed]))
        other.inputs(seed)
        other.run()
        torch.cuda.synchronize()
        other.check()


def test_two_graphs_share_a_workspace(gpu):
    """Two layers captured with one workspace, replayed by turns on one stream."""
    one, two = (Layer(gpu, 13, 512, 160, 24, 4, "mxfp4", score="sigmoid", seed=s) for s in (1, 2))
    scratch = torch.full((max(one.need, two.need),), 0x77, dtype=torch.uint8, device=gpu)
    graphs = []
    for L in (one, two):
        L.share(scratch)
        L.inputs(9)
        L.run()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            L.run()
        graphs.append(graph)
    for seed in range(3):
        for L in (one, two):
            L.inputs(seed)
        for graph in graphs + graphs[::-1]:
            graph.replay()
        torch.cuda.synchronize()
        one.check()
        two.check()


@pytest.mark.parametrize("M", [2, 20])
def test_padded_batch(gpu, M):
    """Rows behind the last sequence, whose logits a mask holds at -inf, have no experts: their y is 0, and memory behind
    the batch is left as it was."""
    n, f, E_, k = 256, 96, 12, 3
    L = Layer(gpu, M, n, f, E_, k, "bf16")
    L.share(torch.zeros(L.need, dtype=torch.uint8, device=gpu))
    L.inputs(0)
    L.run()
    L.logits[M // 2:] = float("-inf")
    L.y.fill_(7)
    assert R.launch_row("moe_layer", L.steps[2][1], torch.cuda.current_stream().cuda_stream) == R.RAD_OK
    torch.cuda.synchronize()
    assert (L.y[M // 2:] == 0).all() and (L.ids[M // 2:] == -1).all() and (L.weights[M // 2:] == 0).all()
    U.check((L.y, L.ids, L.weights), U.exact(L.x, L.logits, L.gu, L.dn, "bf16", f, k))
