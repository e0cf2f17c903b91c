"""Checks of captured gemm_nt_epi, rmsnorm_block and moe_layer launches for tests/replay_dump.py: the outputs from the
PRE state in float64, within the bounds that the rows' own tests count (epi_util, block_util, moe_util)."""
import numpy as np
import torch

from tests import block_util as B
from tests import epi_util as E
from tests import moe_util as U

TYPES = {0: torch.float32, 1: torch.bfloat16, 3: torch.uint8, 5: torch.uint8, 6: torch.uint8, 7: torch.uint8, 8: torch.int8,
         10: torch.int32}
FP4 = 5


def tensor(c, i, state="pre"):
    """Operand i, None where it is absent; two e2m1 codes a byte."""
    if not c.present(i):
        return None
    t = c.tensors[i]
    v = torch.from_numpy(np.array((c.pre if state == "pre" else c.post)[i], np.uint8)).view(TYPES[t["dt"]])
    shape, stride = t["shape"][:t["rank"]], t["stride"][:t["rank"]]
    if t["dt"] == FP4:
        shape, stride = shape[:-1] + [shape[-1] // 2], [s // 2 for s in stride[:-1]] + [1]
    return v.as_strided(shape, stride)


def rows(t, cols):
    return None if t is None else t.reshape(-1, cols)


def check_epi(c):
    N, K = c.geti("N"), c.geti("K")
    a, sa, b, sb, bias, res = (tensor(c, i) for i in range(6))
    y = rows(tensor(c, 6, "post"), N)
    want, err = E.exact(rows(a, K), b, sa, sb, bias, rows(res, N), c.gets("act") or "none")
    E.check(y, want, err)
    return "M=%d N=%d K=%d" % (len(y), N, K)


def check_block(c):
    n = c.geti("n")
    x, res, w_post, gate, w_pre = (tensor(c, i) for i in range(5))
    h, eh, v, ev = B.exact(rows(x, n), rows(res, n), w_post, gate if gate is None or gate.dim() == 1 else rows(gate, gate.shape[-1]),
                           w_pre, c.getf("eps", 1e-6), c.getf("wadd", 0.0), c.getf("res_scale", 1.0))
    for i, want, err in ((5, h, eh), (6, v, ev)):
        if c.present(i):
            B.check("operand %d" % i, rows(tensor(c, i, "post"), n), want, err)
    if c.present(7):
        codes = B.check_i8 if c.tensors[7]["dt"] == 8 else B.check_e4m3
        codes(rows(tensor(c, 7, "post"), n), tensor(c, 8, "post"), v, ev)
    return "rows=%d n=%d" % (len(h), n)


def check_moe(c):
    n, f, k = c.geti("n"), c.geti("f"), c.geti("top_k")
    x, logits, gu, gus, dn, dns = (tensor(c, i) for i in range(6))
    y, ids, w = (tensor(c, i, "post") for i in (6, 7, 8))
    y = rows(y, n)
    want = U.exact(rows(x, n), rows(logits, c.geti("E")), gu, dn, c.gets("dtype"), f, k, gus, dns, c.gets("act") or "silu",
                   c.gets("score") or "softmax", c.geti("renorm", 1), c.getf("weight_scale", 1.0),
                   3 if y.dtype == torch.float32 else 2)
    U.check((y, want[0] if ids is None else rows(ids, k), want[1] if w is None else rows(w, k)), want)
    return "M=%d n=%d f=%d experts=%d" % (len(y), n, f, c.geti("E"))


CHECKS = {"gemm_nt_epi_bf16": check_epi, "gemm_nt_epi_i8a8": check_epi, "rmsnorm_block": check_block, "moe_layer": check_moe}


def check(c):
    try:
        return True, CHECKS[c.row](c) + " within the bounds"
    except AssertionError as e:
        return False, "DIFFER %s" % (e,)
