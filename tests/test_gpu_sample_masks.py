"""sample_logits over rows masked with a finite number, as programs mask that have no infinity: the lowest of
the type, or -1e4.  With fewer tokens allowed than a top-k asks for, the cut lies among the masked ones, which
are equal and more than the kernel lists; their weight is 0, or, at high temperatures, is not."""
import pytest
import torch

from tests.test_gpu_sample import check

pytestmark = pytest.mark.gpu
F32, BF16 = torch.float32, torch.bfloat16
LOWEST = {t: torch.finfo(t).min for t in (F32, BF16)}


def masked(g, M, V, allowed, mask, dtype):
    x = torch.full((M, V), float(mask), dtype=dtype)
    for i in range(M):
        n = allowed[i % len(allowed)]
        x[i, torch.randperm(V, generator=g)[:n]] = (2 * torch.randn(n, generator=g)).to(dtype)
    return x


@pytest.mark.parametrize("V", [8193, 20000, 262144])
@pytest.mark.parametrize("mask,dtype", [(LOWEST[F32], F32), (-1e4, F32), (LOWEST[BF16], BF16), (-1e4, BF16)])
def test_more_asked_for_than_allowed(gpu, V, mask, dtype):
    g = torch.Generator().manual_seed(V)
    M = 12
    x, u = masked(g, M, V, [1, 20, 49, 50, 51, 1300], mask, dtype), torch.rand(M, generator=g)
    k = [50] * M
    check(gpu, x, u, k=k, label="k")
    check(gpu, x, u, k=k, p=torch.linspace(0.05, 0.999, M), label="k p")
    check(gpu, x, u, k=k, m=[0.0, 0.05, 1.0] * 4, label="k m")
    check(gpu, x, u, k=[2000, 2048, 1, 30] * 3, p=[0.9, 1.0] * 6, m=[0.0, 0.01, 0.0] * 4, T=[0.2, 1.0, 3.0] * 4, label="all")
    check(gpu, x, u, p=torch.linspace(0.05, 0.999, M), label="p")
    check(gpu, x, u, k=[V // 2] * M, p=[0.7, 1.0] * 6, label="half")
    check(gpu, x, u, m=[1e-30, 0.01, 0.5] * 4, label="m")


@pytest.mark.parametrize("V", [8193, 50257])
def test_masks_that_keep_a_weight(gpu, V):
    """At these temperatures a masked token weighs from e^-700 to nearly as much as an allowed one."""
    g = torch.Generator().manual_seed(V)
    M = 12
    x, u = masked(g, M, V, [3, 60, 400], -1e4, F32), torch.rand(M, generator=g)
    T = [14.5, 20.0, 100.0, 400.0, 1000.0, 1500.0, 2500.0, 5e3, 1e4, 1e5, 1e6, 1e8]
    check(gpu, x, u, T=T, label="T")
    check(gpu, x, u, T=T, k=[50] * M, label="k")
    check(gpu, x, u, T=T, k=[500] * M, p=torch.linspace(0.05, 0.999, M), label="k p")
    check(gpu, x, u, T=T, p=torch.linspace(0.999, 0.05, M), label="p")
    check(gpu, x, u, T=T, m=[1e-4, 0.3, 0.9] * 4, label="m")
