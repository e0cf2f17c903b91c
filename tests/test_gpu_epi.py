"""gemm_nt_epi on the GPU against 64 bits, element by element; operands lie in guarded memory at the alignments
and pitches named, and what lies around the output has to be left as it was."""
import pytest
import torch

import libr3d_amd as R
from tests import epi_util as E
from tests.test_gpu_i8 import Box
from tests.test_gpu_i8_tiles import SHAPES

pytestmark = pytest.mark.gpu


def operands(dtype, M, N, K, seed=0):
    g = torch.Generator().manual_seed(seed * 1000003 + M * 7919 + N * 31 + K)
    if dtype == "bf16":
        return torch.randn(M, K, generator=g).bfloat16(), torch.randn(N, K, generator=g).bfloat16() * K ** -0.5, None, None, g
    code = lambda *s: torch.randint(-128, 128, s, generator=g, dtype=torch.int32).to(torch.int8)  # noqa: E731
    return code(M, K), code(N, K), torch.rand(M, generator=g) * 0.02, torch.rand(N, generator=g) * K ** -0.5 * 0.05, g


def run(dev, dtype, M, N, K, act="none", bias="f32", residual="bf16", y="bf16", offs=(0, 0, 0), pitch=(None,) * 3,
        scratch=True, seed=0, inplace=False, want_arm=None, a=None, b=None):
    a0, b0, sa, sb, g = operands(dtype, M, N, K, seed)
    a, b = a0 if a is None else a, b0 if b is None else b
    kinds = {"bf16": torch.bfloat16, "f32": torch.float32}
    C = None if bias is None else torch.randn(N, generator=g).to(kinds[bias])
    res = None if residual is None else (2 * torch.randn(M, N, generator=g)).to(kinds[residual])
    A, B = Box(a, dev, offs[0], pitch[0]), Box(b, dev, offs[1], pitch[1])
    Y = Box(res.to(kinds[y]) if inplace else torch.full((M, N), -7.0, dtype=kinds[y]), dev, offs[2], pitch[2])
    if inplace:
        res = res.to(kinds[y])
    Rs = None if res is None else Y if inplace else Box(res, dev, 1, N + 3)
    on = lambda t: None if t is None else t.to(dev)  # noqa: E731
    ops = R.GemmEpiOperands(A.t, B.t, Y.t, a_scale=on(sa), b_scale=on(sb), bias=on(C), residual=None if Rs is None else Rs.t,
                            act=act, dtype=dtype, N=N, K=K)
    row = R.resolve("gemm_nt_epi", {"dtype": dtype, "M": M, "N": N, "K": K})["name"]
    need = R.row_scratch_bytes(row, ops)
    if need and scratch:
        S = Box(torch.full((1, need), 0x5A, dtype=torch.uint8), dev)
        ops.set_scratch(S.t, need)
    text = R.describe(row, ops)[1]
    print(text, offs, pitch, flush=True)
    if want_arm:
        assert want_arm in text
    assert R.launch_row(row, ops, torch.cuda.current_stream().cuda_stream) == R.RAD_OK
    torch.cuda.synchronize()
    want, err = E.exact(a.to(dev), b.to(dev), on(sa), on(sb), on(C), on(res), act)
    use = E.check(Y.t, want, err)
    assert A.around() and B.around() and Y.around() and (Rs is None or Rs.around())
    if need and scratch:
        assert S.around()
    return use


@pytest.mark.parametrize("dtype", ["bf16", "i8a8"])
@pytest.mark.parametrize("M", [1, 2, 3, 7, 8, 9, 16, 17, 33, 64, 65, 130, 257])
def test_rows(gpu, dtype, M):
    run(gpu, dtype, M, 130, 1360)
    run(gpu, dtype, M, 1, 128, residual=None)


@pytest.mark.parametrize("dtype", ["bf16", "i8a8"])
@pytest.mark.parametrize("K", [1, 3, 8, 15, 16, 24, 40, 63, 64, 72, 120, 128, 136, 1000, 1016, 2049])
def test_depth(gpu, dtype, K):
    for M in (1, 9, 40, 150):
        run(gpu, dtype, M, 77, K, act="silu")


@pytest.mark.parametrize("dtype", ["bf16", "i8a8"])
@pytest.mark.parametrize("N", [1, 2, 5, 15, 17, 63, 65, 129, 255, 600])
def test_columns(gpu, dtype, N):
    for M, y in ((1, "bf16"), (12, "f32"), (70, "bf16"), (270, "f32")):
        run(gpu, dtype, M, N, 256, y=y, act="gelu_tanh")


@pytest.mark.parametrize("dtype", ["bf16", "i8a8"])
@pytest.mark.parametrize("act", E.ACTS)
def test_activations(gpu, dtype, act):
    for M, bias, res, y in ((3, "f32", None, "f32"), (3, None, "f32", "bf16"), (50, "bf16", "bf16", "f32"),
                            (200, "f32", "f32", "bf16")):
        run(gpu, dtype, M, 300, 520, act, bias, res, y)
        run(gpu, dtype, M, 50, 133, act, bias, res, y)                # K off 16 bytes


@pytest.mark.parametrize("dtype", ["bf16", "i8a8"])
@pytest.mark.parametrize("offs,pitch", [((1, 0, 0), (None,) * 3), ((0, 3, 0), (None,) * 3), ((0, 0, 1), (None,) * 3),
                                        ((16, 48, 3), (288, 272, 301)), ((0, 0, 0), (257, 300, 299)),
                                        ((5, 7, 1), (259, 261, 293))])
def test_alignment(gpu, dtype, offs, pitch):
    for M, y in ((1, "f32"), (6, "bf16"), (33, "f32"), (140, "bf16")):
        run(gpu, dtype, M, 290, 256, offs=offs, pitch=pitch, y=y, act="relu")


@pytest.mark.parametrize("dtype", ["bf16", "i8a8"])
@pytest.mark.parametrize("M,N,K", SHAPES)
def test_tiles(gpu, dtype, M, N, K):
    """The shapes that reach every LDS tile, whole and split, on rows that begin on lines and inside them (K in
    bytes)."""
    e = 2 if dtype == "bf16" else 1
    run(gpu, dtype, M, N, K // e, act="gelu", want_arm="arm=tile")
    run(gpu, dtype, M, N, K // e, y="f32", pitch=((K + 112) // e, (K + 48) // e, N + 5), seed=1)


@pytest.mark.parametrize("dtype", ["bf16", "i8a8"])
@pytest.mark.parametrize("M,N,K", [(1, 2048, 5376), (4, 128, 5376), (13, 5376, 4096), (16, 1000, 10752), (333, 1187, 5360),
                                   (1030, 2060, 2048)])
def test_larger(gpu, dtype, M, N, K):
    run(gpu, dtype, M, N, K, act="gelu_tanh")
    run(gpu, dtype, M, N, K, scratch=False, y="f32")


@pytest.mark.parametrize("dtype", ["bf16", "i8a8"])
def test_in_place(gpu, dtype):
    for M, N, K in ((2, 700, 512), (2, 700, 511), (40, 300, 5376), (300, 700, 1024), (2048, 2560, 512)):
        for y in ("bf16", "f32"):
            run(gpu, dtype, M, N, K, inplace=True, y=y, act="silu")


@pytest.mark.parametrize("dtype", ["bf16", "i8a8"])
def test_broadcast_bias_and_residual(gpu, dtype):
    for M, N, K in ((3, 100, 256), (3, 100, 255), (90, 200, 512), (20, 256, 8192)):
        a, b, sa, sb, g = operands(dtype, M, N, K)
        on = lambda t: None if t is None else t.to(gpu)  # noqa: E731
        bias, res = torch.randn(2 * N, generator=g), torch.randn(1, N, generator=g).bfloat16()
        y = torch.empty(M, N, device=gpu)
        for c in (bias[::2], bias[:1].expand(N)):
            cd = c.to(gpu) if c.stride(0) == 0 else bias.to(gpu)[::2]
            cd = bias[:1].to(gpu).expand(N) if c.stride(0) == 0 else cd
            assert R.gemm_nt_epi(on(a), on(b), y, a_scale=on(sa), b_scale=on(sb), bias=cd,
                                 residual=res.to(gpu).expand(M, N), dtype=dtype, N=N, K=K) == R.RAD_OK
            want, err = E.exact(a, b, sa, sb, c, res.expand(M, N))
            E.check(y.cpu(), want, err)


def test_infinities_stay_in_their_rows(gpu):
    """inf and NaN among the operands: the row's, the column's or the element's result alone, and an infinite
    product is infinite, also where K, a chunk or a split ends inside a line."""
    for M, N, K in ((1, 40, 1000), (5, 40, 4104), (5, 40, 77), (20, 200, 5000), (20, 64, 77), (150, 300, 1032)):
        a, b, _, _, g = operands("bf16", M, N, K)
        a = a.abs() + 0.125
        b = b.abs() + 0.125
        a[M - 1, K - 1] = float("inf")
        b[3, K // 2] = float("nan")
        b[7, 0] = float("-inf")
        y = torch.empty(M, N, dtype=torch.bfloat16, device=gpu)
        res = torch.zeros(M, N)
        res[0, 11] = float("nan")
        # what follows the operands in memory is NaN
        A = torch.full((M * K + 64,), float("nan"), dtype=torch.bfloat16, device=gpu)
        B = torch.full((N * K + 64,), float("nan"), dtype=torch.bfloat16, device=gpu)
        A[:M * K], B[:N * K] = a.flatten().to(gpu), b.flatten().to(gpu)
        assert R.gemm_nt_epi(A[:M * K].view(M, K), B[:N * K].view(N, K), y, residual=res.to(gpu), dtype="bf16", N=N, K=K) == R.RAD_OK
        want = a.double() @ b.double().T + res.double()
        got = y.cpu().double()
        assert torch.equal(got.isnan(), want.isnan()), (M, N, K)
        inf = want.isinf()
        assert torch.equal(got[inf], want[inf]) and not got[~inf].isinf().any()


@pytest.mark.parametrize("dtype", ["bf16", "i8a8"])
def test_streams_and_graph(gpu, dtype):
    """Another stream, two streams at once, and a captured launch replayed over new inputs."""
    for M, N, K in ((5, 700, 1536), (48, 700, 4096), (400, 700, 1536)):
        a, b, sa, sb, g = operands(dtype, M, N, K)
        on = lambda t: None if t is None else t.to(gpu)  # noqa: E731
        A, B, SA, SB = on(a), on(b), on(sa), on(sb)
        bias = torch.randn(N, generator=g)
        C = bias.to(gpu)
        row = R.resolve("gemm_nt_epi", {"dtype": dtype, "M": M, "N": N, "K": K})["name"]

        def bound():
            y = torch.zeros(M, N, dtype=torch.bfloat16, device=gpu)
            ops = R.GemmEpiOperands(A, B, y, a_scale=SA, b_scale=SB, bias=C, act="gelu", dtype=dtype, N=N, K=K)
            need = R.row_scratch_bytes(row, ops)
            if need:
                ops.set_scratch(torch.empty(need, dtype=torch.uint8, device=gpu))
            return y, ops
        want, err = E.exact(a, b, sa, sb, bias, None, "gelu")
        two = [(torch.cuda.Stream(), *bound()) for _ in range(2)]
        torch.cuda.synchronize()
        for s, y, ops in two:
            assert R.launch_row(row, ops, s.cuda_stream) == R.RAD_OK
        torch.cuda.synchronize()
        for s, y, ops in two:
            E.check(y.cpu(), want, err)
        y, ops = bound()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            assert R.launch_row(row, ops, torch.cuda.current_stream().cuda_stream) == R.RAD_OK
        for i in range(3):
            a2 = operands(dtype, M, N, K, seed=20 + i)[0]
            A.copy_(a2)
            y.fill_(-1)
            graph.replay()
            torch.cuda.synchronize()
            want, err = E.exact(a2, b, sa, sb, bias, None, "gelu")
            E.check(y.cpu(), want, err)
            again = torch.zeros_like(y)
            assert R.gemm_nt_epi(A, B, again, a_scale=SA, b_scale=SB, bias=C, act="gelu", dtype=dtype, N=N, K=K) == R.RAD_OK
            torch.cuda.synchronize()
            assert torch.equal(y, again)                              # bit for bit
