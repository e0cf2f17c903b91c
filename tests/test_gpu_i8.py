"""The int8 rows on the GPU.  The product sums exactly in i32 and its epilogue is three f32
roundings, so every element is compared bit for bit with 64-bit integers and the same roundings;
the quantiser's codes and scales likewise.  Operands lie in guarded memory at the alignments and
pitches named, and what lies around every output has to be left as it was."""
import numpy as np
import pytest
import torch

import libr3d_amd as R

pytestmark = pytest.mark.gpu
GUARD = 512


class Box:
    """A [rows, cols] tensor inside guarded memory: `off` elements past an aligned address, rows
    `pitch` elements apart."""

    def __init__(self, host, dev, off=0, pitch=None):
        host = torch.as_tensor(host)
        flat = host.reshape(-1, host.shape[-1])
        rows, cols = flat.shape
        self.pitch, self.off, self.rows, self.cols = pitch or cols, off, rows, cols
        size = host.element_size()
        self.buf = torch.full(((2 * GUARD + off + rows * self.pitch) * size,), 0x5A, dtype=torch.uint8,
                              device=dev).view(host.dtype)
        self.t = self.buf[GUARD + off:].as_strided((rows, cols), (self.pitch, 1))
        self.t.copy_(flat)

    def around(self):
        """True when nothing but the rows' own elements has changed."""
        b = self.buf.clone()
        b[GUARD + self.off:].as_strided((self.rows, self.cols), (self.pitch, 1)).fill_(0)
        want = torch.full((b.numel() * b.element_size(),), 0x5A, dtype=torch.uint8, device=b.device).view(b.dtype)
        want[GUARD + self.off:].as_strided((self.rows, self.cols), (self.pitch, 1)).fill_(0)
        return bool(torch.equal(b.view(torch.uint8), want.view(torch.uint8)))


def codes(g, *shape):
    return torch.randint(-128, 128, shape, generator=g, dtype=torch.int32).to(torch.int8)


def scales(g, n):
    return torch.exp(2 * torch.randn(n, generator=g))


def product(a, sa, b, sb):
    """bf16 bits of (f32(sum) * sa) * sb: sums below 2^53 are exact in f64."""
    s = (a.double() @ b.double().T).numpy().astype(np.int64).astype(np.float32)
    y = (s * sa.numpy()[:, None]).astype(np.float32) * sb.numpy()[None, :]
    return torch.from_numpy(y.astype(np.float32)).bfloat16()


def run_gemm(dev, M, N, K, seed=0, offs=(0, 0, 0), pitch=(None, None, None), scratch=True, row=None,
             a=None, b=None, stream=None):
    g = torch.Generator().manual_seed(seed * 1000003 + M * 7919 + N * 31 + K)
    a = codes(g, M, K) if a is None else a
    b = codes(g, N, K) if b is None else b
    sa, sb = scales(g, M), scales(g, N)
    A, B = Box(a, dev, offs[0], pitch[0]), Box(b, dev, offs[1], pitch[1])
    Y = Box(torch.full((M, N), -7.0, dtype=torch.bfloat16), dev, offs[2], pitch[2])
    ops = R.GemmOperands(A.t, sa.to(dev), B.t, sb[:, None].to(dev), Y.t, dtype="i8a8", N=N, K=K, M=M)
    if row is None:
        row = R.resolve("gemm_nt_q", {"dtype": "i8a8", "M": M, "N": N, "K": K, "group": K})["name"]
    need = R.row_scratch_bytes(row, ops)
    if need and scratch:
        S = Box(torch.full((1, need), 0x5A, dtype=torch.uint8), dev)
        ops.set_scratch(S.t, need)
    print("i8a8", M, N, K, offs, pitch, R.describe(row, ops)[1], flush=True)
    assert R.launch_row(row, ops, stream or torch.cuda.current_stream().cuda_stream) == R.RAD_OK
    torch.cuda.synchronize()
    want = product(a, sa, b, sb)
    got = Y.t.cpu()
    assert torch.equal(got.view(torch.int16), want.view(torch.int16)), (got - want).abs().max()
    assert A.around() and B.around() and Y.around()
    if need and scratch:
        assert S.around()


@pytest.mark.parametrize("M", [1, 2, 3, 7, 8, 9, 13, 16, 17, 31, 33, 64, 65, 130, 257, 300])
def test_gemm_rows(gpu, M):
    run_gemm(gpu, M, 130, 1360)
    run_gemm(gpu, M, 1, 128)


@pytest.mark.parametrize("K", [1, 3, 15, 16, 17, 48, 63, 64, 112, 127, 128, 144, 1000, 1008, 2049])
def test_gemm_depth(gpu, K):
    for M in (1, 9, 40, 150):
        run_gemm(gpu, M, 77, K)


@pytest.mark.parametrize("N", [1, 2, 5, 15, 17, 63, 65, 129, 255, 257, 600])
def test_gemm_columns(gpu, N):
    for M in (1, 12, 70, 270):
        run_gemm(gpu, M, N, 256)


@pytest.mark.parametrize("offs,pitch", [((1, 0, 0), (None,) * 3), ((0, 3, 0), (None,) * 3), ((0, 0, 1), (None,) * 3),
                                        ((16, 48, 3), (288, 272, 301)), ((0, 0, 0), (257, 300, 299)),
                                        ((5, 7, 1), (259, 261, 293))])
def test_gemm_alignment(gpu, offs, pitch):
    for M in (1, 6, 15, 33, 140):
        run_gemm(gpu, M, 290, 256, offs=offs, pitch=pitch)


@pytest.mark.parametrize("M,N,K", [(1, 2048, 5376), (4, 640, 21504), (16, 5376, 4096), (16, 1000, 21504),
                                   (40, 1500, 5376), (100, 700, 8192), (129, 5120, 1024), (600, 1100, 5360),
                                   (1030, 2060, 2048)])
def test_gemm_larger(gpu, M, N, K):
    run_gemm(gpu, M, N, K)
    run_gemm(gpu, M, N, K, scratch=False)


def test_gemm_extreme_sums(gpu):
    """The largest sum that i32 holds, of both signs, through every kernel's width."""
    K = 131071
    for M in (1, 16, 40, 140):
        a = torch.full((M, K), -128, dtype=torch.int8)
        b = torch.full((20, K), -128, dtype=torch.int8)
        b[1::2] = 127
        run_gemm(gpu, M, 20, K, a=a, b=b)
        run_gemm(gpu, M, 20, K - 15, a=a[:, 15:].contiguous(), b=b[:, 15:].contiguous())


def test_gemm_scales_at_their_ends(gpu):
    """Scale stride 0, and scales of 0, inf and NaN, which belong to their rows alone."""
    g = torch.Generator().manual_seed(5)
    for M in (3, 30, 200):
        N, K = 40, 512
        a, b = codes(g, M, K), codes(g, N, K)
        sa, sb = torch.full((M,), 0.5), scales(g, N)
        sb[3], sb[4], sb[5] = 0.0, float("inf"), float("nan")
        y = torch.empty(M, N, dtype=torch.bfloat16, device=gpu)
        sa_d = torch.tensor([0.5], device=gpu).expand(M)
        rc, _ = R.gemm_nt_q(a.to(gpu), sa_d, b.to(gpu), sb.to(gpu), y, dtype="i8a8", N=N, K=K)
        assert rc == R.RAD_OK
        want = product(a, sa, b, sb)
        assert torch.equal(torch.nan_to_num(y.cpu(), 9.0), torch.nan_to_num(want, 9.0))
        assert torch.equal(y.cpu().isnan(), want.isnan())


def test_gemm_streams_and_graph(gpu):
    """Another stream, two streams at once, and a captured launch replayed over new inputs."""
    g = torch.Generator().manual_seed(8)
    for M in (5, 48, 400):
        N, K = 700, 1536
        a, b, sa, sb = codes(g, M, K), codes(g, N, K), scales(g, M), scales(g, N)
        A, B, SA, SB = a.to(gpu), b.to(gpu), sa.to(gpu), sb.to(gpu)
        row = R.resolve("gemm_nt_q", {"dtype": "i8a8", "M": M, "N": N, "K": K})["name"]

        def bound():
            y = torch.zeros(M, N, dtype=torch.bfloat16, device=gpu)
            ops = R.GemmOperands(A, SA, B, SB, y, dtype="i8a8", N=N, K=K, M=M)
            need = R.row_scratch_bytes(row, ops)
            if need:
                ops.set_scratch(torch.empty(need, dtype=torch.uint8, device=gpu))
            return y, ops
        torch.cuda.synchronize()
        two = [(torch.cuda.Stream(), *bound()) for _ in range(2)]
        torch.cuda.synchronize()
        for s, _, ops in two:
            assert R.launch_row(row, ops, s.cuda_stream) == R.RAD_OK
        torch.cuda.synchronize()
        want = product(a, sa, b, sb)
        for _, y, _ in two:
            assert torch.equal(y.cpu(), want)
        y, ops = bound()
        graph = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph):
            assert R.launch_row(row, ops, torch.cuda.current_stream().cuda_stream) == R.RAD_OK
        for k in range(3):
            a = codes(g, M, K)
            A.copy_(a)
            y.zero_()
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(y.cpu(), product(a, sa, b, sb)), k


# ------------------------------------------------------------------------------- the producers

def quantise(h):
    """Scales and codes of f32 rows, in the definition's own roundings (numpy f32)."""
    h = h.numpy().astype(np.float32)
    with np.errstate(all="ignore"):
        amax = np.abs(h).max(1)
        s = np.where(amax > 0, np.maximum(amax * np.float32(1 / 127), np.float32(2.0 ** -126)), np.float32(1))
        s = np.where(np.isnan(amax), np.float32("nan"), s).astype(np.float32)
        q = np.rint(h * (np.float32(1) / s)[:, None])
    q = np.where(np.isfinite(s)[:, None], q, 0)
    return torch.from_numpy(q.astype(np.int8)), torch.from_numpy(s)


def same(x, y):
    return torch.equal(torch.nan_to_num(x, 3.25), torch.nan_to_num(y, 3.25)) and torch.equal(x.isnan(), y.isnan())


def activation(g, M, n, dtype=torch.bfloat16):
    return (torch.randn(M, n, generator=g) * torch.exp(torch.randn(M, 1, generator=g))).to(dtype)


SIZES = [(1, 1), (1, 7), (3, 8), (5, 9), (2, 63), (4, 512), (3, 513), (600, 520), (2, 4096), (7, 5376), (530, 5376),
         (3, 8191), (2, 16392), (2, 24576), (2, 24577), (1, 32768), (2, 32775), (513, 2056), (1, 70001)]


@pytest.mark.parametrize("M,n", SIZES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_quant(gpu, M, n, dtype):
    g = torch.Generator().manual_seed(M * 131 + n)
    x = activation(g, M, n, dtype)
    for off, pad in ((0, 0), (1, 3)):
        X, Q = Box(x, gpu, off, n + pad), Box(torch.full((M, n), 99, dtype=torch.int8), gpu, off, n + pad)
        S = Box(torch.full((M, 1), -1.0), gpu, off)
        print("quant", M, n, dtype, off, flush=True)
        assert R.quant_act_i8(X.t, Q.t, S.t, n=n) == R.RAD_OK
        q, s = quantise(x.float())
        assert torch.equal(Q.t.cpu(), q) and torch.equal(S.t.cpu()[:, 0], s)
        assert X.around() and Q.around() and S.around()


def test_quant_special_rows(gpu):
    """Rows of zeros, of subnormals, of the largest numbers, with an infinity, with a NaN."""
    for n in (9, 640, 40000):
        x = torch.zeros(9, n)
        x[1] = 1e-40
        x[2, 0], x[2, -1] = 3e38, -1e38
        x[3, n // 2] = float("inf")
        x[4, n - 1] = float("-inf")
        x[5, 0] = float("nan")
        x[6, 0], x[6, 1] = float("nan"), float("inf")
        x[7] = -2.0
        x[8, 3] = 2.0 ** -126
        for t in (x, x.bfloat16()):
            q = torch.full((9, n), 99, dtype=torch.int8, device=gpu)
            s = torch.zeros(9, device=gpu)
            assert R.quant_act_i8(t.to(gpu), q, s, n=n) == R.RAD_OK
            wq, ws = quantise(t.float())
            assert torch.equal(q.cpu(), wq) and same(s.cpu(), ws)
            assert (q.cpu()[3:7] == 0).all() and not torch.isfinite(s.cpu()[3:7]).any()


@pytest.mark.parametrize("M,n", SIZES)
@pytest.mark.parametrize("res,wdt,wadd", [(False, torch.float32, None), (True, torch.bfloat16, None),
                                          (True, torch.float32, 1.0)])
def test_norm(gpu, M, n, res, wdt, wadd):
    g = torch.Generator().manual_seed(M * 131 + n + 1)
    x, r = activation(g, M, n), activation(g, M, n)
    w = (1 + 0.2 * torch.randn(n, generator=g)).to(wdt)
    eps = 1e-5
    f = (x.float() + r.float()).bfloat16() if res else x
    v = f.float().numpy()
    rs = (1.0 / np.sqrt((v.astype(np.float64) ** 2).sum(1) / n + eps)).astype(np.float32)
    wf = w.float().numpy() + np.float32(wadd or 0)
    h = torch.from_numpy((v * rs[:, None]).astype(np.float32) * wf.astype(np.float32))
    q, s = quantise(h)
    for off, pad, place in ((0, 0, "apart"), (1, 5, "apart"), (0, 0, "residual"), (1, 1, "x")):
        if not res and place != "apart":
            continue
        X, Q = Box(x, gpu, off, n + pad), Box(torch.full((M, n), 99, dtype=torch.int8), gpu, off, n + pad)
        Rs = Box(r, gpu, off, n + pad) if res else None
        Ro = {"apart": Box(torch.zeros_like(x), gpu, off, n + pad), "residual": Rs, "x": X}[place] if res else None
        S, W = Box(torch.full((M, 1), -1.0), gpu, off), Box(w[None], gpu, off)
        odt = torch.float32 if wdt == torch.float32 else torch.bfloat16
        O = Box(torch.zeros(M, n, dtype=odt), gpu, off, n + pad) if place == "apart" else None
        print("norm", M, n, res, wdt, off, place, flush=True)
        rc = R.rmsnorm_quant_i8(X.t, Rs.t if res else None, W.t[0], Q.t, S.t, O.t if O else None, n=n,
                                residual_out=Ro.t if res else None, eps=eps, wadd=wadd)
        assert rc == R.RAD_OK
        assert torch.equal(Q.t.cpu(), q) and torch.equal(S.t.cpu()[:, 0], s)
        if res:
            assert torch.equal(Ro.t.cpu(), f)
        if O:
            assert torch.equal(O.t.cpu(), h.to(odt))
        for b in (X, Q, Rs, Ro, S, W, O):
            assert b is None or b.around()


def test_norm_special_rows(gpu):
    """Rows of zeros with and without eps; an infinity or a NaN, and a sum of squares past f32,
    stay in their own row."""
    for n in (16, 700, 33000):
        x = torch.ones(6, n, dtype=torch.bfloat16)
        x[0] = 0
        x[1, 3] = float("inf")
        x[2, n - 1] = float("nan")
        x[3] = 1e38
        x[4] = 1e-38
        w = torch.ones(n, dtype=torch.bfloat16, device=gpu)
        q, s = torch.empty(6, n, dtype=torch.int8, device=gpu), torch.empty(6, device=gpu)
        assert R.rmsnorm_quant_i8(x.to(gpu), None, w, q, s, n=n) == R.RAD_OK
        qc, sc = q.cpu(), s.cpu()
        assert (qc[0] == 0).all() and sc[0] == 1.0
        assert sc[1].isnan() and sc[2].isnan() and (qc[1:3] == 0).all()
        assert (qc[3] == 127).all() and abs(float(sc[3]) * 127 - 1) < 1e-6    # 4 roundings of 2^-24
        assert (qc[5] == 127).all() and (qc[4] == 127).all()
        assert R.rmsnorm_quant_i8(x[:1].to(gpu), None, w, q[:1], s[:1], n=n, eps=0.0) == R.RAD_OK
        assert s.cpu()[0].isnan()                         # 0 * (1 / 0)


@pytest.mark.parametrize("M,n", SIZES)
@pytest.mark.parametrize("act", ["silu", "sigmoid"])
def test_gated(gpu, M, n, act):
    """Against 64 bits.  sigmoid is within 3 f32 steps (2^-22 relative for the two roundings of
    the exp and one of the quotient), the two products round once each: |h - h64| <= 2^-21 |h64|.
    Where the sigmoid is below 2^-126 (gates under -87) f32 has no normal number for it: it is off
    by up to 2^-126, which the factors gate and up multiply.
    The codes' value is then within half a scale and that; the scale within 2^-21 and its own two
    roundings, 2^-20 in all."""
    g = torch.Generator().manual_seed(M * 131 + n + 2)
    for dtype in (torch.bfloat16, torch.float32):
        x = (3 * activation(g, M, 2 * n, dtype).float()).to(dtype)
        d = x.double()
        sg = torch.sigmoid(d[:, :n])
        h = (d[:, :n] * sg if act == "silu" else sg) * d[:, n:]
        for off, pad in ((0, 0), (1, 3)):
            X, Q = Box(x, gpu, off, 2 * n + pad), Box(torch.full((M, n), 99, dtype=torch.int8), gpu, off, n + pad)
            S, O = Box(torch.full((M, 1), -1.0), gpu, off), Box(torch.zeros(M, n), gpu, off, n + pad)
            print("gated", M, n, act, dtype, off, flush=True)
            assert R.gated_quant_i8(X.t, Q.t, S.t, O.t, n=n, act=act) == R.RAD_OK
            s = S.t.cpu().double()
            amax = h.abs().amax(1, keepdim=True)
            want = torch.where(amax > 0, (amax / 127).clamp_min(2.0 ** -126), 1.0)
            assert ((s - want).abs() <= 2.0 ** -20 * want).all()
            out = O.t.cpu().double()
            flush = 2.0 ** -126 * (1 + (d[:, n:] * (d[:, :n] if act == "silu" else 1)).abs())
            bad = ((out - h).abs() > 2.0 ** -21 * h.abs() + flush).nonzero()
            assert not len(bad), [(float(d[i, j]), float(d[i, n + j]), float(h[i, j]), float(out[i, j]))
                                  for i, j in bad[:5]]
            assert ((Q.t.cpu().double() * s - out).abs() <= s * (0.5 + 2.0 ** -14)).all()
            assert X.around() and Q.around() and S.around() and O.around()


def test_gated_far_gates(gpu):
    """Gates where exp leaves f32, infinities and NaN: sigmoid 0 or 1, and a row's own NaN."""
    gate = torch.tensor([[-1e30, -200.0, -104.0, -89.0, -88.0, 0.0, 40.0, 1e30]])
    up = torch.full((1, 8), 2.0)
    for act in ("silu", "sigmoid"):
        q, s = torch.empty(3, 8, dtype=torch.int8, device=gpu), torch.empty(3, device=gpu)
        o = torch.empty(3, 8, device=gpu)
        x = torch.cat([gate, up], 1).repeat(3, 1)
        x[1, 2] = float("nan")
        x[2, 7] = float("inf")
        assert R.gated_quant_i8(x.to(gpu), q, s, o, n=8, act=act) == R.RAD_OK
        d = gate.double()
        sg = torch.sigmoid(d)
        h = (d * sg if act == "silu" else sg) * 2
        # a sigmoid under 2^-126 is 0: off by less than that, times gate and up (= 2) as above; at
        # 104 and past it the product itself is under 2^-126
        flush = 2.0 ** -126 * (1 + 2 * d.abs().clamp_max(104))
        assert ((o[0].cpu().double() - h).abs() <= 2.0 ** -21 * h.abs() + flush).all()
        assert s.cpu()[1].isnan() and (q.cpu()[1] == 0).all()
        if act == "silu":
            assert s.cpu()[2] == float("inf") and (q.cpu()[2] == 0).all()


def test_producers_in_a_graph(gpu):
    """The three producers captured one after the other, replayed over new inputs."""
    g = torch.Generator().manual_seed(4)
    M, n = 6, 2000
    x = activation(g, M, 2 * n).to(gpu)
    r, w = activation(g, M, n).to(gpu), torch.ones(n, dtype=torch.bfloat16, device=gpu)
    out = [[torch.zeros(M, n, dtype=torch.int8, device=gpu), torch.zeros(M, device=gpu)] for _ in range(3)]
    ro = torch.zeros_like(r)

    def all3():
        s = torch.cuda.current_stream().cuda_stream
        assert R.quant_act_i8(x[:, :n], *out[0], n=n, stream=s) == R.RAD_OK
        assert R.gated_quant_i8(x, *out[1], n=n, stream=s) == R.RAD_OK
        assert R.rmsnorm_quant_i8(x[:, n:], r, w, *out[2], n=n, residual_out=ro, stream=s) == R.RAD_OK
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        all3()
    for k in range(3):
        x.copy_(activation(g, M, 2 * n))
        graph.replay()
        torch.cuda.synchronize()
        got = [[t.clone() for t in o] for o in out] + [[ro.clone()]]
        for o in out:
            o[0].zero_(), o[1].zero_()
        all3()
        torch.cuda.synchronize()
        assert all(torch.equal(t, u) for p, o in zip(got, out + [[ro]]) for t, u in zip(p, o)), k
