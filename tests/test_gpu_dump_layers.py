"""R3D_DUMP over gemm_nt_epi, rmsnorm_block and moe_layer: a child process launches a layer of them, the captures replay
on the host and, byte for byte, on the device, and a capture with a mistake in it is told from a good one."""
import os
import subprocess
import sys

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

_CHILD = r"""
import sys
sys.path.insert(0, %r)
import torch
from tests.test_gpu_expert_block import Layer
dev = torch.device("cuda:0")
for M, dtype in ((3, "i8"), (20, "mxfp4"), (9, "bf16")):
    L = Layer(dev, M, 320, 128, 12, 3, dtype, seed=M)
    L.share(torch.zeros(L.need, dtype=torch.uint8, device=dev))
    L.inputs(M)
    L.run()
torch.cuda.synchronize()
print("LAUNCHED")
"""


def test_capture_and_replay(gpu, tmp_path):
    env = dict(os.environ, R3D_DUMP=str(tmp_path), R3D_DUMP_MAX="3")
    p = subprocess.run([sys.executable, "-c", _CHILD % ROOT], env=env, capture_output=True, text=True, timeout=300)
    assert p.returncode == 0 and "LAUNCHED" in p.stdout, p.stdout[-2000:] + p.stderr[-2000:]
    caps, got = sorted(os.listdir(tmp_path)), {}
    for d in caps:
        row = d.split("_", 1)[1]
        got[row] = got.get(row, 0) + 1
    assert got == {"gemm_nt_epi_bf16": 3, "gemm_nt_epi_i8a8": 3, "rmsnorm_block": 3, "moe_layer": 3}, caps
    from tests import replay_dump as RD
    for d in caps:
        c = RD.Capture(str(tmp_path / d))
        ok, msg = RD.replay_oracle(c)
        assert ok, (d, msg)
        out = [i for i in (5, 6, 7) if c.present(i)] if c.row == "rmsnorm_block" else [6]
        for i in out:
            good, c.post[i] = c.post[i], np.array(c.post[i])
            c.post[i][3] ^= 0x55                       # the exponent of the first float, or the second bf16 value's
            assert not RD.replay_oracle(c)[0], (d, i)
            c.post[i] = good
    p = subprocess.run([sys.executable, os.path.join(ROOT, "tests", "replay_dump.py"), str(tmp_path), "--device"],
                       capture_output=True, text=True, timeout=300)
    assert p.returncode == 0, p.stdout[-3000:] + p.stderr[-2000:]
    assert "%d capture(s), 0 divergent" % len(caps) in p.stdout, p.stdout[-3000:]
