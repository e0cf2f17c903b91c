"""Launch scratch that gemm_nt_epi's and moe_layer's Python calls take belongs to the stream that the launch goes to."""
import pytest
import torch

import libr3d_amd as R
from tests import test_scratch_stream as S


def epi_call(dev, stream):
    """A product whose K is split over planes in scratch."""
    M, N, K = 13, 256, 4096
    t = [torch.zeros(s, K, dtype=torch.bfloat16, device=dev) for s in (M, N)]
    y = torch.zeros(M, N, dtype=torch.bfloat16, device=dev)
    S.written(dev)
    return R.gemm_nt_epi(*t, y, dtype="bf16", N=N, K=K, stream=stream)


def moe_call(dev, stream):
    M, n, f, E = 3, 64, 32, 4
    bf = lambda *s: torch.zeros(*s, dtype=torch.bfloat16, device=dev)  # noqa: E731
    t = [bf(M, n), torch.zeros(M, E, device=dev), bf(E, 2 * f, n), bf(E, n, f), bf(M, n)]
    S.written(dev)
    return R.moe_layer(*t, dtype="bf16", n=n, f=f, E=E, top_k=2, stream=stream)


CALLS = [epi_call, moe_call]


@pytest.mark.parametrize("call", CALLS)
@pytest.mark.parametrize("stream,want", [(0, "default"), (0x1230, "raw 4656")])
def test_scratch_is_of_the_launch_s_stream(monkeypatch, call, stream, want):
    streams = S.Streams(monkeypatch)
    assert call("cpu", stream) == R.RAD_OK
    assert streams.at == [want] and streams.now == "current"


@pytest.mark.gpu
@pytest.mark.parametrize("call", CALLS)
def test_scratch_on_the_gpu(gpu, monkeypatch, call):
    S.test_scratch_on_the_gpu(gpu, monkeypatch, call)
