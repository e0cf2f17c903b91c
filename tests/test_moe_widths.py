"""moe_layer's launches on the host: tokens that share one read of an expert's planes, in each of the two products."""
import pytest

from tests.moe_passes import launch, passes
from tests.test_moe import call


def sizes(dtype, M, n, f, E, top_k):
    """A call's launch; the planes are never touched, so that one expert's memory serves all."""
    one = call(dtype, M=M, n=n, f=f, E=1, top_k=1)
    more = {k: one._tensors[i].expand(E, *one._tensors[i].shape[1:]) for i, k in
            ((2, "gate_up"), (3, "gate_up_scale"), (4, "down"), (5, "down_scale")) if one._tensors[i] is not None}
    return launch(call(dtype, M=M, n=n, f=f, E=E, top_k=top_k, **more))


@pytest.mark.parametrize("dtype", ["bf16", "i8", "mxfp4"])
def test_wide_experts_are_read_once_for_eight_tokens(dtype):
    """LDS holds one token's h of f = 14336, and more than eight of the tokens' 4096 columns."""
    g = sizes(dtype, 64, 4096, 14336, 8, 2)
    assert g["up_width"] == 8 and g["down_width"] >= 8 and g["parts"] > 1
    g = sizes(dtype, 1, 4096, 14336, 8, 2)                # a token an expert: nothing to share
    assert g["parts"] == 1
    g = sizes(dtype, 64, 30720, 1024, 8, 2)
    assert g["up_width"] == 2 and g["down_width"] >= 8 and g["parts"] == 1


@pytest.mark.parametrize("dtype", ["bf16", "i8", "mxfp4"])
def test_limits(dtype):
    """One token's columns of x in LDS; rows of h of any length up to f's limit."""
    from tests.test_moe import R, rc
    n = {"bf16": 66560, "i8": 62464, "mxfp4": 66560}[dtype]
    assert sizes(dtype, 1, n, 32, 1, 1)["up_width"] == 1
    assert rc(dtype, M=1, n=n + 32, f=32, E=1, top_k=1) == R.RAD_E_UNSUPPORTED
    assert sizes(dtype, 1, 32, 65536, 1, 1)["parts"] >= 3
    assert rc(dtype, M=1, n=32, f=65568, E=1, top_k=1) == R.RAD_E_UNSUPPORTED


def test_widths_are_bound_by_rows_and_columns():
    for M, n, f, E, k in ((1, 64, 96, 8, 1), (64, 64, 96, 8, 2), (13, 4096, 7168, 8, 2), (64, 2048, 768, 64, 8)):
        g = sizes("mxfp4", M, n, f, E, k)
        for p in ("up", "down"):
            assert 1 <= g[p + "_width"] <= min(8 * g[p + "_ct"], g[p + "_rows"]) and g[p + "_rows"] <= min(64, M * k)


def test_passes():
    assert passes([3], 4, 8, 8) == (1, False, False)
    assert passes([8] * 64, 32, 8, 8) == (1, False, False)
    assert passes([8] * 256, 4, 8, 8)[0] == 1 and passes([8] * 512, 4, 8, 8)[0] == 2
    assert passes([1] * 64, 2048, 8, 8, cap=128) == (4, True, True)        # 512 units of two jobs, 128 at a time
