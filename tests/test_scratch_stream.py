"""Launch scratch that a Python call takes belongs to the stream that its launch goes to: it is freed when the
call returns, so memory of another stream's pool could be handed out while the kernels still write to it."""
import contextlib

import pytest
import torch

import libr3d_amd as R


def written(dev):
    """Operands made on the current stream are there for the launch's."""
    if dev != "cpu":
        torch.cuda.synchronize()


def i8_call(dev, stream):
    """A product whose K is split over planes in scratch."""
    M, N, K = 13, 256, 4096
    t = [torch.zeros(M, K, dtype=torch.int8, device=dev), torch.ones(M, device=dev),
         torch.zeros(N, K, dtype=torch.int8, device=dev), torch.ones(N, device=dev),
         torch.zeros(M, N, dtype=torch.bfloat16, device=dev)]
    written(dev)
    return R.gemm_nt_q(*t, dtype="i8a8", N=N, K=K, stream=stream)[0]


def mx_call(dev, stream):
    """The e2m1 tile row over its split's planes."""
    M, N, K = 40, 1000, 2048
    u8 = lambda *s: torch.zeros(*s, dtype=torch.uint8, device=dev)  # noqa: E731
    t = [u8(M, K), torch.ones(M, K // 128, device=dev), u8(N, K // 2), u8(N, K // 32),
         torch.zeros(M, N, dtype=torch.bfloat16, device=dev)]
    written(dev)
    return R.gemm_nt_q(*t, dtype="mxfp4a8", N=N, K=K, stream=stream)[0]


def sample_call(dev, stream):
    t = [torch.zeros(2, 100, device=dev), torch.zeros(2, device=dev), torch.zeros(2, dtype=torch.int32, device=dev)]
    written(dev)
    return R.sample_logits(*t, n_vocab=100, stream=stream)


CALLS = [i8_call, mx_call, sample_call]


class Streams:
    """torch's streams without a GPU: a stream is a name, and `at` holds the one that each allocation of bytes
    was made on."""

    def __init__(self, monkeypatch):
        self.now, self.at = "current", []
        empty = torch.empty

        @contextlib.contextmanager
        def on(s):
            was, self.now = self.now, self.now if s is None else s
            yield
            self.now = was

        def bytes_of(*shape, **kw):
            self.at.append(self.now)
            return empty(*shape, **dict(kw, device="cpu"))
        cuda = torch.cuda
        monkeypatch.setattr(cuda, "stream", on)
        monkeypatch.setattr(cuda, "device", lambda d: contextlib.nullcontext())
        monkeypatch.setattr(cuda, "current_device", lambda: 0)
        monkeypatch.setattr(cuda, "default_stream", lambda device=None: "default")
        # of a null pointer torch makes a stream of its own
        monkeypatch.setattr(cuda, "ExternalStream", lambda p, device=None: "raw %d" % p if p else "another")
        monkeypatch.setattr(torch, "empty", bytes_of)
        monkeypatch.setattr(R, "_one_gpu", lambda *t: torch.device("cuda:0"))
        monkeypatch.setattr(R, "launch_row", lambda row, ops, stream=0: R.RAD_OK)


@pytest.mark.parametrize("call", CALLS)
@pytest.mark.parametrize("stream,want", [(0, "default"), (0x1230, "raw 4656")])
def test_scratch_is_of_the_launch_s_stream(monkeypatch, call, stream, want):
    streams = Streams(monkeypatch)
    assert call("cpu", stream) == R.RAD_OK
    assert streams.at == [want] and streams.now == "current"


@pytest.mark.gpu
@pytest.mark.parametrize("call", CALLS)
def test_scratch_on_the_gpu(gpu, monkeypatch, call):
    empty, at = torch.empty, []

    def bytes_of(*shape, **kw):
        at.append(torch.cuda.current_stream().cuda_stream)
        return empty(*shape, **kw)
    other = torch.cuda.Stream()
    torch.cuda.synchronize()
    monkeypatch.setattr(torch, "empty", bytes_of)
    for current, stream, want in ((None, 0, 0), (other, 0, 0), (None, other.cuda_stream, other.cuda_stream),
                                  (other, None, other.cuda_stream), (None, None, 0)):
        at.clear()
        torch.cuda.synchronize()
        with torch.cuda.stream(current):
            assert call(gpu, stream) == R.RAD_OK
        torch.cuda.synchronize()
        assert at == [want], (stream, want)
