"""Rows whose byte offsets pass 2^31 and 2^32: the int8 product's operands and output, the producers' and the
sampler's rows.  The memory between the rows is never touched."""
import numpy as np
import pytest
import torch

import libr3d_amd as R
from tests.test_gpu_i8 import codes, product, scales
from tests.test_gpu_sample import plain

pytestmark = pytest.mark.gpu


def far(t, dev, pitch):
    """t's rows `pitch` elements apart in fresh memory."""
    buf = torch.empty((t.shape[0] - 1) * pitch + t.shape[1], dtype=t.dtype, device=dev)
    v = buf.as_strided(t.shape, (pitch, 1))
    v.copy_(t)
    return v


# 2^22 bytes is the largest pitch of the fast kernels; past it, and off 16, the kernel for any alignment runs
@pytest.mark.parametrize("M,N,K,pa,pb", [(4, 1100, 384, 384, 1 << 22), (300, 1100, 384, 384, 1 << 22),
                                         (1100, 300, 384, 1 << 22, 400), (40, 1100, 384, 400, (1 << 22) + 16),
                                         (1100, 40, 77, (1 << 22) + 1, 77)])
def test_product(gpu, M, N, K, pa, pb):
    g = torch.Generator().manual_seed(M)
    a, b, sa, sb = codes(g, M, K), codes(g, N, K), scales(g, M), scales(g, N)
    y = torch.empty(M, N, dtype=torch.bfloat16, device=gpu)
    rc, row = R.gemm_nt_q(far(a, gpu, pa), sa.to(gpu), far(b, gpu, pb), sb.to(gpu), y, dtype="i8a8", N=N, K=K)
    assert rc == R.RAD_OK
    torch.cuda.synchronize()
    assert torch.equal(y.cpu().view(torch.int16), product(a, sa, b, sb).view(torch.int16))


@pytest.mark.parametrize("M", [3, 20])
def test_product_rows_out(gpu, M):
    g = torch.Generator().manual_seed(M)
    N, K, pitch = 260, 512, (1 << 32) // (2 * (M - 1)) + 24
    a, b, sa, sb = codes(g, M, K), codes(g, N, K), scales(g, M), scales(g, N)
    y = far(torch.zeros(M, N, dtype=torch.bfloat16), gpu, pitch)
    assert R.gemm_nt_q(a.to(gpu), sa.to(gpu), b.to(gpu), sb.to(gpu), y, dtype="i8a8", N=N, K=K)[0] == R.RAD_OK
    torch.cuda.synchronize()
    assert torch.equal(y.cpu().view(torch.int16), product(a, sa, b, sb).view(torch.int16))


def test_producers(gpu):
    """The rows far apart give what the same rows give side by side."""
    g = torch.Generator().manual_seed(3)
    M, n = 4, 1000
    x, r = (torch.randn(M, 2 * n, generator=g).bfloat16() for _ in range(2))
    w = torch.randn(n, generator=g).bfloat16().to(gpu)
    pitch = (1 << 31) // 3 + 7
    near = [torch.zeros(M, n, dtype=torch.int8, device=gpu), torch.zeros(M, device=gpu)]
    away = [far(torch.zeros(M, n, dtype=torch.int8), gpu, 2 * pitch), torch.zeros(M, device=gpu)]
    xd, rd, xf = x.to(gpu), r.to(gpu), far(x, gpu, pitch)
    rn, rf = rd[:, :n].contiguous(), far(r[:, :n], gpu, pitch)
    for f in (lambda x_, r_, o: R.quant_act_i8(x_[:, :n], *o, n=n), lambda x_, r_, o: R.gated_quant_i8(x_, *o, n=n),
              lambda x_, r_, o: R.rmsnorm_quant_i8(x_[:, :n], r_, w, *o, n=n, residual_out=r_)):
        assert f(xd, rn, near) == f(xf, rf, away) == R.RAD_OK
        torch.cuda.synchronize()
        assert all(torch.equal(a.cpu(), b.cpu()) for a, b in zip(near, away))
    assert torch.equal(rn.cpu(), rf.cpu())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_sampler(gpu, dtype):
    g = torch.Generator().manual_seed(4)
    M, V = 4, 9000
    x, u = (2 * torch.randn(M, V, generator=g)).to(dtype), torch.rand(M, generator=g)
    k, p = [0, 40, 0, 5000], [1.0, 0.9, 0.8, 0.95]
    token = torch.zeros(M, dtype=torch.int32, device=gpu)
    assert R.sample_logits(far(x, gpu, (1 << 30) + 3), u.to(gpu), token, n_vocab=V,
                           top_k=torch.tensor(k, dtype=torch.int32, device=gpu),
                           top_p=torch.tensor(p, device=gpu)) == R.RAD_OK
    want = [plain(x[i].float().numpy(), float(u[i]), 1.0, k[i], float(np.float32(p[i])))[0] for i in range(M)]
    assert token.cpu().tolist() == want
