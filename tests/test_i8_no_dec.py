"""R3D_NO_I8_DEC turns the int8 GEMV off, not only its row: up to 8 tokens the any-M row takes its tiles, with
the same bits.  In child processes, which read the switch."""
import json
import os
import subprocess
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
SHAPES = [(1, 5000, 5376), (2, 333, 1360), (3, 500, 2320), (4, 1201, 2048), (6, 333, 1360), (7, 1001, 1536), (8, 700, 1040)]

_PLANS = r"""
import sys, json
sys.path.insert(0, %r)
import torch
import libr3d_amd as R
out = []
for M, N, K in %r:
    i8, one = torch.zeros(1, K, dtype=torch.int8), torch.ones(1)
    ops = R.GemmOperands(i8.expand(M, K), one.expand(M), i8.expand(N, K), one.expand(N),
                         torch.zeros(M, N, dtype=torch.bfloat16), dtype="i8a8", N=N, K=K, M=M)
    out.append(R.describe("gemm_nt_q_i8a8", ops)[1].split()[0])
print(json.dumps(out))
"""

_RUN = r"""
import sys
sys.path.insert(0, %r)
import torch
from tests.test_gpu_i8 import run_gemm
dev = torch.device("cuda:0")
for M, N, K in %r:
    run_gemm(dev, M, N, K)
    run_gemm(dev, M, N, K, pitch=(K + 48, K + 16, N + 3), seed=1)
print("RAN")
"""


def child(script, env, timeout=120):
    p = subprocess.run([sys.executable, "-c", script % (ROOT, SHAPES)], env=dict(os.environ, **env), capture_output=True,
                       text=True, timeout=timeout)
    assert p.returncode == 0, p.stdout[-2000:] + p.stderr[-2000:]
    return p.stdout


def test_no_call_takes_the_gemv():
    assert json.loads(child(_PLANS, {})) == ["arm=gemv"] * len(SHAPES)
    assert json.loads(child(_PLANS, {"R3D_NO_I8_DEC": "1"})) == ["arm=tile"] * len(SHAPES)


@pytest.mark.gpu
def test_tiles_of_few_tokens(gpu):
    out = child(_RUN, {"R3D_NO_I8_DEC": "1"}, timeout=110)
    assert "RAN" in out and "arm=gemv" not in out and out.count("arm=tile") == 2 * len(SHAPES), out[-2000:]
