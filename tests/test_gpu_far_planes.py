"""gemm_nt_epi, rmsnorm_block and moe_layer with rows and experts whose byte offsets pass 2^31 and 2^32.  The memory
between the rows is never touched."""
import pytest
import torch

import libr3d_amd as R
from tests import epi_util as E
from tests import moe_util as U
from tests.test_gpu_block import inputs as block_inputs
from tests.test_gpu_epi import operands
from tests.test_gpu_far_rows import far
from tests.test_gpu_moe import inputs as moe_inputs

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["bf16", "i8a8"])
@pytest.mark.parametrize("M,N,K,pa,pb", [(4, 1100, 384, 0, 1 << 22), (13, 1100, 384, 0, 1 << 22), (1100, 300, 384, 1 << 22, 0),
                                         (40, 1100, 384, 0, (1 << 22) + 16), (1100, 40, 77, (1 << 22) + 2, 0)])
def test_product_operands(gpu, dtype, M, N, K, pa, pb):
    """Pitches in bytes; 2^22 is the fast kernels' largest."""
    a, b, sa, sb, g = operands(dtype, M, N, K)
    size = a.element_size()
    on = lambda t: None if t is None else t.to(gpu)  # noqa: E731
    put = lambda t, p: far(t, gpu, p // size) if p else t.to(gpu)  # noqa: E731
    bias = torch.randn(N, generator=g)
    y = torch.empty(M, N, dtype=torch.bfloat16, device=gpu)
    assert R.gemm_nt_epi(put(a, pa), put(b, pb), y, a_scale=on(sa), b_scale=on(sb), bias=on(bias), act="silu", dtype=dtype,
                         N=N, K=K) == R.RAD_OK
    torch.cuda.synchronize()
    E.check(y, *E.exact(on(a), on(b), on(sa), on(sb), on(bias), None, "silu"))


@pytest.mark.parametrize("dtype", ["bf16", "i8a8"])
@pytest.mark.parametrize("M", [3, 20, 300])
def test_product_rows_out(gpu, dtype, M):
    N, K = 260, 512
    pitch = (1 << 32) // (2 * (M - 1)) + 24
    a, b, sa, sb, g = operands(dtype, M, N, K)
    on = lambda t: None if t is None else t.to(gpu)  # noqa: E731
    res = torch.randn(M, N, generator=g).bfloat16()
    y, r = far(torch.zeros(M, N, dtype=torch.bfloat16), gpu, pitch), far(res, gpu, pitch)
    assert R.gemm_nt_epi(on(a), on(b), y, a_scale=on(sa), b_scale=on(sb), residual=r, dtype=dtype, N=N, K=K) == R.RAD_OK
    torch.cuda.synchronize()
    E.check(y.contiguous(), *E.exact(on(a), on(b), on(sa), on(sb), None, on(res)))


def test_block(gpu):
    """The rows far apart give what the same rows give side by side."""
    M, n, pitch = 4, 1000, (1 << 31) // 3 + 7
    t = block_inputs(M, n, gate="full")
    on = {k: v.to(gpu) for k, v in t.items()}
    away = {k: far(v, gpu, pitch) if v.dim() == 2 else v.to(gpu) for k, v in t.items()}
    got = []
    for d, new in ((on, lambda kind: torch.zeros(M, n, dtype=kind, device=gpu)),
                   (away, lambda kind: far(torch.zeros(M, n, dtype=kind), gpu, pitch * (1 if kind == torch.bfloat16 else 2)))):
        o = dict(residual_out=new(torch.bfloat16), out=new(torch.bfloat16), q=new(torch.int8),
                 scale=torch.zeros(M, device=gpu))
        assert R.rmsnorm_block(n=n, **d, **o) == R.RAD_OK
        torch.cuda.synchronize()
        got.append(o)
    assert all(torch.equal(got[0][k], got[1][k]) for k in got[0])


@pytest.mark.parametrize("dtype", ["bf16", "i8", "mxfp4"])
def test_experts(gpu, dtype):
    """Five experts' planes more than 2^32 bytes from the first to the last, and far rows of y and of the logits."""
    M, n, f, E_, k = 5, 256, 160, 5, 3
    t = moe_inputs(dtype, M, n, f, E_)
    on = {m: None if v is None else v.to(gpu) for m, v in t.items()}
    apart = dict(on)
    for m in ("gate_up", "down"):
        w = t[m]
        step = ((1 << 32) // w.element_size() // (E_ - 1) + 4096) // 16 * 16
        buf = torch.empty((E_ - 1) * step + w[0].numel(), dtype=w.dtype, device=gpu)
        apart[m] = buf.as_strided(w.shape, (step, w.shape[2], 1))
        apart[m].copy_(w)
    apart["logits"] = far(t["logits"], gpu, (1 << 30) // 4)
    y = far(torch.zeros(M, n, dtype=torch.bfloat16), gpu, (1 << 32) // 2 // (M - 1) + 8)
    ids, w = torch.zeros(M, k, dtype=torch.int32, device=gpu), torch.zeros(M, k, device=gpu)
    assert R.moe_layer(y=y, ids=ids, weights=w, dtype=dtype, n=n, f=f, E=E_, top_k=k, **apart) == R.RAD_OK
    torch.cuda.synchronize()
    U.check((y.contiguous(), ids, w), U.exact(**on, dtype=dtype, f=f, top_k=k))


@pytest.mark.parametrize("dtype", ["bf16", "i8", "mxfp4"])
def test_expert_rows(gpu, dtype):
    """Rows of an expert's plane as far apart as the row takes them, under 2^31 bytes from the first to the last."""
    M, n, f, E_, k = 3, 64, 32, 2, 1
    t = moe_inputs(dtype, M, n, f, E_)
    on = {m: None if v is None else v.to(gpu) for m, v in t.items()}
    apart = dict(on)
    for m in ("gate_up", "down"):
        w = t[m]
        pitch = ((1 << 31) // w.shape[1] - 32) // 16 * 16 // w.element_size()
        buf = torch.empty(E_ * w.shape[1] * pitch, dtype=w.dtype, device=gpu)
        apart[m] = buf.as_strided(w.shape, (w.shape[1] * pitch, pitch, 1))
        apart[m].copy_(w)
    y = torch.zeros(M, n, device=gpu)
    ids, w = torch.zeros(M, k, dtype=torch.int32, device=gpu), torch.zeros(M, k, device=gpu)
    assert R.moe_layer(y=y, ids=ids, weights=w, dtype=dtype, n=n, f=f, E=E_, top_k=k, **apart) == R.RAD_OK
    torch.cuda.synchronize()
    U.check((y, ids, w), U.exact(**on, dtype=dtype, f=f, top_k=k, parts=3))
