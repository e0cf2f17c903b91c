"""h of moe_layer holds the 24 bits of f32 whatever y's type is."""
import pytest
import torch

import libr3d_amd as R

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["bf16", "i8", "mxfp4"])
@pytest.mark.parametrize("y", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("M", [1, 9])
def test_h_keeps_its_bits(gpu, dtype, y, M):
    """x's columns are 1, 2^-1 .. 2^-23 and the weights 0 and 1, so that h of the rows 2 i and 2 i + 1 are a random 24-bit
    number and its first nine bits: y[i], their difference, is what stands behind these.  Every product and every sum
    of some of them is a multiple of 2^-23 under 2, which f32 holds: nothing is rounded but y."""
    n, f = 64, 128
    g = torch.Generator().manual_seed(7)
    bits = torch.zeros(f, n, dtype=torch.int64)
    bits[::2, :24] = torch.randint(0, 2, (f // 2, 24), generator=g)
    bits[::2, 0] = 1
    bits[1::2, :9] = bits[::2, :9]
    gate = torch.zeros(f, n, dtype=torch.int64)
    gate[:, 0] = 1
    down = torch.zeros(n, f, dtype=torch.int64)
    i = torch.arange(f // 2)
    down[i, 2 * i], down[i, 2 * i + 1] = 1, -1
    planes = [torch.cat((gate, bits))[None], down[None]]
    scales = [None, None]
    if dtype == "bf16":
        planes = [p.bfloat16() for p in planes]
    elif dtype == "i8":
        planes, scales = [p.to(torch.int8) for p in planes], [torch.ones(1, p.shape[1]) for p in planes]
    else:                                     # e2m1: 2 is 1, 10 is -1
        nib = [torch.where(p < 0, 10, 2 * p).to(torch.uint8) for p in planes]
        planes = [p[..., ::2] | p[..., 1::2] << 4 for p in nib]
        scales = [torch.full((1, p.shape[1], p.shape[2] // 32), 127, dtype=torch.uint8) for p in nib]
    x = torch.zeros(M, n)
    x[:, :24] = 2.0 ** -torch.arange(24)
    on = lambda t: None if t is None else t.to(gpu)  # noqa: E731
    got = torch.empty(M, n, dtype=y, device=gpu)
    assert R.moe_layer(x.bfloat16().to(gpu), torch.zeros(M, 1, device=gpu), on(planes[0]), on(planes[1]), got,
                       gate_up_scale=on(scales[0]), down_scale=on(scales[1]), dtype=dtype, n=n, f=f, E=1, top_k=1,
                       act="none") == R.RAD_OK
    h = bits.double() @ (2.0 ** -torch.arange(n).double())
    want = (h[::2] - h[1::2]).to(y).expand(M, f // 2)
    assert torch.equal(got[:, :f // 2].cpu(), want)
