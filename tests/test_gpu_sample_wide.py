"""sample_logits at its limits: the widest vocabulary, more rows than workgroups, top-k's around every size
at which the kernel changes how it orders a list, rows that hold about k tokens.  Against the same float64
sampler; at 2^22 tokens a mass is off by up to 2^-41, a border by some 2^-29 of the mass, and the uniform
numbers (24 bits, generic) do not lie within that of one."""
import numpy as np
import pytest
import torch

from tests.test_gpu_sample import check

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("V,dtype", [(4194304, torch.float32), (4194301, torch.bfloat16)])
def test_widest_vocabulary(gpu, V, dtype):
    g = torch.Generator().manual_seed(V)
    M = 8
    x = torch.randn(M, V, generator=g).to(dtype)
    check(gpu, x, torch.rand(M, generator=g), T=[1.0, 0.5, 1.0, 0.2, 1.0, 1.0, 0.3, 0.0],
          k=[0, 50, 1000, 0, 5000, 2048, 0, 0], p=[1.0, 0.9, 1.0, 0.9, 0.95, 0.6, 1.0, 0.5],
          m=[0.0, 0.0, 0.02, 0.0, 0.0, 0.0, 0.3, 0.0])


@pytest.mark.parametrize("M,V", [(700, 5000), (300, 40000), (1100, 200), (257, 4097)])
def test_more_rows_than_workgroups(gpu, M, V):
    """Every row needs bins; then every other one."""
    g = torch.Generator().manual_seed(M)
    x, u = 2 * torch.randn(M, V, generator=g), torch.rand(M, generator=g)
    check(gpu, x, u, p=torch.linspace(0.02, 0.98, M))
    check(gpu, x, u, p=torch.where(torch.arange(M) % 2 == 0, 1.0, 0.7), k=torch.arange(M) % 5 * 7)


def test_list_sizes(gpu):
    """Top-k's around the sizes at which a list is ordered another way."""
    g = torch.Generator().manual_seed(7)
    ks = [n + d for n in (1, 64, 128, 256, 512, 1024, 2048) for d in (-1, 0, 1)]
    M, V = len(ks), 200000
    x, u = 2 * torch.randn(M, V, generator=g), torch.rand(M, generator=g)
    check(gpu, x, u, k=ks)
    check(gpu, x, u, k=ks, p=torch.linspace(0.1, 0.999, M))
    check(gpu, x, u, k=ks, p=torch.linspace(0.999, 0.1, M), m=[0.0, 0.02, 0.1] * 7)
    check(gpu, (x * 8).round() / 8, u, k=ks, p=torch.linspace(0.3, 0.999, M))       # ties across every cut
    check(gpu, x, u, p=torch.linspace(0.001, 0.2, M), m=[0.0, 0.02, 0.1] * 7)


def test_about_k_tokens_present(gpu):
    """A mask that leaves 60 tokens of 20000, and k just below, at and above that."""
    g = torch.Generator().manual_seed(8)
    M, V = 12, 20000
    x = torch.full((M, V), float("-inf"))
    for i in range(M):
        x[i, torch.randperm(V, generator=g)[:60]] = torch.randn(60, generator=g)
    u = torch.rand(M, generator=g)
    k = [59, 60, 61] * 4
    check(gpu, x, u, k=k)
    check(gpu, x, u, k=k, p=[0.999999, 0.5, 0.9] * 4)
    check(gpu, x, u, k=[60, 5000, 4999] * 4, p=[0.999999, 0.5, 0.9, 1.0] * 3)


def test_min_p_of_one_at_high_temperatures(gpu, monkeypatch):
    """A weight that rounds to 1 in float64 is not below min_p = 1, however far its logit lies below the
    largest.  numpy's exp is off by one in the last place there (exp(-4.7e-17) is 1 - 4.7e-17, nearer to 1
    than to 1 - 2^-53 = 1 - 1.11e-16, and comes out as the latter), so under 2^-30 the sampler it is held
    against takes 1 + z, which z^2 / 2 < 2^-61 moves by less than 2^-8 of a last place."""
    exp = np.exp
    monkeypatch.setattr(np, "exp", lambda z: np.where(np.abs(z) < 2.0 ** -30, 1.0 + z, exp(z)))
    g = torch.Generator().manual_seed(9)
    M, V = 8, 9000
    x, u = 3 * torch.randn(M, V, generator=g), torch.rand(M, generator=g)
    T = [1e20, 1e17, 1e30, 3e38, 1.0, 1e4, 1e8, float("inf")]
    for m in (1.0, 2.0, 1 - 2.0 ** -24, 0.5):
        check(gpu, x, u, T=T, m=[m] * M)
        check(gpu, x, u, T=T, m=[m] * M, k=[300, 9000, 1, 0] * 2)
        check(gpu, x, u, T=T, m=[m] * M, p=[0.9] * M)


@pytest.mark.parametrize("V", [8192, 8193, 20000, 300000])
def test_min_p_that_keeps_more_than_a_list(gpu, V):
    g = torch.Generator().manual_seed(V)
    M = 6
    x, u = 0.1 * torch.randn(M, V, generator=g), torch.rand(M, generator=g)
    check(gpu, x, u, m=[0.3, 0.5, 0.7, 0.8, 0.05, 1e-30])
    check(gpu, x, u, m=[1e-30] * M, T=[0.01, 0.1, 1.0, 10.0, 0.02, 0.003])
    check(gpu, torch.zeros(M, V), u, m=[0.3, 0.5, 0.7, 1.0, 0.05, 1e-30])
