"""R3D_DUMP over the int8 rows and the sampler: a child process launches each, the captures replay on
the host and, byte for byte, on the device, and a capture with a mistake in it is told from a good one."""
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
from tests.test_gpu_decode_step import Step
dev = torch.device("cuda:0")
for M in (3, 20):
    st = Step(dev, M, 512, 704, 4500, seed=M)
    st.inputs()
    st.run()
import libr3d_amd as R
assert R.quant_act_i8(st.x, st.q1, st.s1, n=512) == 0
torch.cuda.synchronize()
print("LAUNCHED")
"""

ROWS = {"gemm_nt_q_i8a8_decode": 2, "gemm_nt_q_i8a8": 2, "quant_act_i8": 1, "gated_quant_i8": 2,
        "rmsnorm_quant_i8": 2, "logits_gemm_e4m3": 2, "sample_logits": 2}


def test_capture_and_replay(gpu, tmp_path):
    env = dict(os.environ, R3D_DUMP=str(tmp_path), R3D_DUMP_MAX="2")
    p = subprocess.run([sys.executable, "-c", _CHILD % ROOT], env=env, capture_output=True, text=True, timeout=300)
    assert p.returncode == 0 and "LAUNCHED" in p.stdout, p.stdout[-2000:] + p.stderr[-2000:]
    caps, got = sorted(os.listdir(tmp_path)), {}
    for d in caps:
        row = d.split("_", 1)[1]
        got[row] = got.get(row, 0) + 1
    assert got == ROWS, caps
    from tests import replay_dump as RD
    out = {"gemm": 4, "quan": 1, "gate": 1, "rmsn": 3, "samp": 6}
    for d in caps:
        c = RD.Capture(str(tmp_path / d))
        ok, msg = RD.replay_oracle(c)
        assert ok, (d, msg)
        if c.row != "logits_gemm_e4m3":
            i = out[c.row[:4]]
            c.post[i] = np.array(c.post[i])
            c.post[i][1] ^= 0x55                       # the second byte of the output
            assert not RD.replay_oracle(c)[0], d
    p = subprocess.run([sys.executable, os.path.join(ROOT, "tests", "replay_dump.py"), str(tmp_path), "--device"],
                       capture_output=True, text=True, timeout=300)
    assert p.returncode == 0, p.stdout[-3000:] + p.stderr[-2000:]
    assert "%d capture(s), 0 divergent" % len(caps) in p.stdout, p.stdout[-3000:]
