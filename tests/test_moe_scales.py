"""moe_layer refuses results in the memory of the experts' scales: ids and weights are written while other workgroups read them."""
import pytest
import torch

import libr3d_amd as R
from tests.test_moe import ROW, aligned, bf, call, rc

NAMES = ["gate_up_scale", "down_scale"]


def over(dtype, name, at):
    """The call's own scales in memory that begins `at` bytes before room for results, and views of that room."""
    own = call(dtype)._tensors[{"gate_up_scale": 3, "down_scale": 5}[name]]
    mem = aligned((own.numel() * own.element_size() + 4096,), torch.uint8)
    size = own.numel() * own.element_size()
    s = mem[:size].view(own.dtype).view(own.shape)
    s.copy_(own)
    room = mem[size + at:size + at + 1024]
    return s, dict(y=room[:512].view(torch.bfloat16).view(4, 64), ids=room[:32].view(torch.int32).view(4, 2),
                   weights=room[:32].view(torch.float32).view(4, 2))


@pytest.mark.parametrize("dtype", ["i8", "mxfp4"])
@pytest.mark.parametrize("name", NAMES)
@pytest.mark.parametrize("result", ["y", "ids", "weights"])
def test_refuses_results_over_the_scales(dtype, name, result):
    for at, want in ((-512, R.RAD_E_INVAL), (-4, R.RAD_E_INVAL), (0, R.RAD_OK), (64, R.RAD_OK)):
        s, of = over(dtype, name, at)
        assert rc(dtype, **{name: s, result: of[result]}) == want, at


@pytest.mark.parametrize("name,rows,K", [("gate_up_scale", 192, 64), ("down_scale", 64, 96)])
def test_planes_apart(name, rows, K):
    """What lies between experts' scales, or behind one plane for all of them, is not theirs but for the span's sake."""
    mem = aligned((1 << 16,), torch.uint8)
    one = mem[:rows * (K // 32)].view(1, rows, K // 32).expand(8, rows, K // 32)
    behind = mem[rows * (K // 32):][:512].view(torch.bfloat16).view(4, 64)
    assert rc("mxfp4", **{name: one, "y": behind}) == R.RAD_OK
    assert rc("mxfp4", **{name: one, "y": mem[:512].view(torch.bfloat16).view(4, 64)}) == R.RAD_E_INVAL
    wide = mem.view(torch.float32).as_strided((8, rows), (1024, 1))
    last = mem[7 * 4096 + 4 * rows - 4:][:32].view(torch.int32).view(4, 2)
    past = mem[7 * 4096 + 4 * rows:][:32].view(torch.int32).view(4, 2)
    assert rc("i8", **{name: wide, "ids": last}) == R.RAD_E_INVAL
    assert rc("i8", **{name: wide, "ids": past}) == R.RAD_OK


def test_other_results_stand():
    assert R.describe(ROW, call("i8", y=bf(4, 64), weights=torch.zeros(4, 2)))[0] == R.RAD_OK
