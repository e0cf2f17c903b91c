"""Workloads of the operators around the quantised linear layer, as a serving program calls them:
operands, outputs and launch scratch bound once, then one row launch a pass.

Every case names one operator and its sizes:

  epi   gemm_nt_epi: Y = act(A . W^T [* a_scale * b_scale] + bias) + residual, rounded once, in bf16 or
        in int8 codes with one f32 scale a token and one an output channel
  norm  rmsnorm_block: what lies between two blocks, the norm after one, its gate, the residual's
        scale and addition, and the norm before the next: bf16, or int8 or e4m3 codes of it
  moe   moe_layer: a mixture-of-experts layer for a few tokens: the choice of top_k experts from the
        router's logits, their gated MLPs, and the weighted sum; weights in bf16, int8 or mxfp4

Codes come back as the bf16 values that they and their scales stand for.  The sizes are those of the
27B-class model that bench.py and the tests use (hidden 5376, MLP 21504, q/k/v joined 8192, attention
output 4096; its MLP cut into experts of 1344), or generic ones.

`own` False computes the plain forms in elementary torch operations; True calls the library.
"""
import math

import torch

own = False

HIDDEN, MLP, QKV, ATTN = 5376, 21504, 8192, 4096
EPS = 1e-6
TINY = 2.0 ** -126                   # the least int8 scale: the smallest normal f32
WEIGHT_BYTES = {"bf16": 2.0, "i8": 1.0, "mxfp4": 0.5 + 1 / 32}


def listed():
    return [
        # the router of 128 experts over four decoding sequences: latency alone
        dict(name="epi_router_m4", op="epi", dtype="bf16", M=4, N=128, K=HIDDEN, bias=True, residual=False, act="none", y="f32"),
        # one sequence's attention output projected and added to its residual stream
        dict(name="epi_out_m1", op="epi", dtype="i8a8", M=1, N=HIDDEN, K=ATTN, bias=False, residual=True, act="none", y="bf16"),
        # an odd batch of decoding sequences through an MLP's first matrix
        dict(name="epi_up_m13", op="epi", dtype="bf16", M=13, N=MLP, K=HIDDEN, bias=True, residual=False, act="gelu_tanh", y="bf16"),
        # a prompt of no round length through a joined q/k/v plane that a shard cut unevenly, with its bias
        dict(name="epi_qkv_m333", op="epi", dtype="bf16", M=333, N=QKV - 5, K=HIDDEN - 16, bias=True, residual=False, act="none", y="bf16"),
        # a full prefill chunk through an MLP's first matrix: the largest product
        dict(name="epi_up_m2048", op="epi", dtype="i8a8", M=2048, N=MLP, K=HIDDEN, bias=True, residual=False, act="gelu_tanh", y="bf16"),
        # one sequence between its attention and its MLP: launch and latency
        dict(name="norm_m1", op="norm", M=1, n=HIDDEN, post=True, gate="channel", residual=True, out="bf16"),
        # an odd prompt on its way into an int8 projection, with a gate a token
        dict(name="norm_m333", op="norm", M=333, n=HIDDEN, post=True, gate="token", residual=True, out="i8"),
        # a full prefill chunk
        dict(name="norm_m2048", op="norm", M=2048, n=HIDDEN, post=True, gate="none", residual=True, out="bf16"),
        # one sequence decoding: eight of 128 experts
        dict(name="moe_m1", op="moe", dtype="mxfp4", M=1, n=HIDDEN, f=1344, E=128, top_k=8, score="softmax", renorm=1, act="silu", y="bf16"),
        # a small batch over int8 experts of a smaller model, sums left in f32 for what adds to them
        dict(name="moe_m4", op="moe", dtype="i8", M=4, n=2048, f=768, E=64, top_k=4, score="sigmoid", renorm=1, act="silu", y="f32"),
        # an odd batch with padded rows over bf16 experts, weights not renormalised
        dict(name="moe_m13", op="moe", dtype="bf16", M=13, n=2048, f=1408, E=32, top_k=4, score="softmax", renorm=0, act="gelu_tanh", y="bf16"),
        # the largest decode batch: nearly every expert is read
        dict(name="moe_m64", op="moe", dtype="mxfp4", M=64, n=HIDDEN, f=1344, E=128, top_k=8, score="softmax", renorm=1, act="silu", y="bf16"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["epi", "norm", "moe"])
    if op == "epi":
        dtype = rng.choice(["bf16", "i8a8"])
        lo, hi = rng.choice([(1, 16), (17, 128), (129, 2048)])
        most = MLP * HIDDEN
        while True:
            M, N, K = _log_int(rng, lo, hi), _log_int(rng, 60, MLP), 8 * _log_int(rng, 32, MLP // 8)
            if dtype == "i8a8":
                K = K // 16 * 16
            if 1 << 19 <= N * K <= most and M * N * K * (2 if dtype == "bf16" else 1) <= 2048 * most:
                break
        return dict(op=op, dtype=dtype, M=M, N=N, K=K, bias=rng.random() < 0.6, residual=rng.random() < 0.5,
                    act=rng.choice(["none", "none", "relu", "silu", "gelu", "gelu_tanh", "sigmoid"]),
                    y=rng.choice(["bf16", "bf16", "f32"]))
    if op == "norm":
        n = _log_int(rng, 100, 16384)
        if rng.random() < 0.7:
            n = (n + 7) // 8 * 8
        while True:
            M = _log_int(rng, 1, 4096)
            if M * n <= 2048 * HIDDEN:
                break
        return dict(op=op, M=M, n=n, post=rng.random() < 0.8, gate=rng.choice(["none", "channel", "token", "full"]),
                    residual=rng.random() < 0.85, out=rng.choice(["bf16", "bf16", "i8", "e4m3"]))
    dtype = rng.choice(["bf16", "i8", "mxfp4"])
    while True:
        E, M = _log_int(rng, 4, 256), _log_int(rng, 1, 64)
        n, f = 32 * _log_int(rng, 8, HIDDEN // 32), 32 * _log_int(rng, 6, 80)
        top_k = min(E, rng.choice([1, 2, 4, 6, 8]))
        if 1 << 24 <= E * 3 * n * f * WEIGHT_BYTES[dtype] <= 128 * 3 * HIDDEN * 1344 * WEIGHT_BYTES["mxfp4"]:
            break
    return dict(op=op, dtype=dtype, M=M, n=n, f=f, E=E, top_k=top_k, score=rng.choice(["softmax", "softmax", "sigmoid"]),
                renorm=rng.choice([0, 1, 1]), act=rng.choice(["silu", "silu", "gelu_tanh"]), y=rng.choice(["bf16", "bf16", "f32"]))


# ------------------------------------------------------------------------------- inputs

def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def _rand(g, *shape):
    return torch.rand(*shape, generator=g, device="cuda")


def _bytes(g, lo, hi, *shape, dtype=torch.uint8):
    return torch.randint(lo, hi, shape, generator=g, device="cuda", dtype=dtype)


def _codes(g, rows, K):
    """int8 codes of normal rows on their largest magnitude, and scales like those of
    activations or weights."""
    x = _randn(g, rows, K)
    s = x.abs().amax(1) / 127.0
    return torch.round(x / s[:, None]).to(torch.int8), s


def _activation(g, M, n):
    """bf16 rows of an activation: rows of different sizes, a few channels far above the rest."""
    x = _randn(g, M, n) * torch.exp(0.5 * _randn(g, M, 1))
    at = torch.randint(0, n, (max(1, n // 512),), generator=g, device="cuda")
    x[:, at] *= 5.0
    return x.bfloat16()


def _experts(g, dtype, E, rows, K):
    """One plane an expert, and its scales: weights of about 1 / sqrt(K)."""
    if dtype == "bf16":
        w = torch.empty(E, rows, K, dtype=torch.bfloat16, device="cuda")
        return w.normal_(0.0, K ** -0.5, generator=g), None
    if dtype == "i8":
        return _bytes(g, -127, 128, E, rows, K, dtype=torch.int8), (0.5 + _rand(g, E, rows)) * (K ** -0.5 / 73.0)
    # nibbles of all sixteen values (their spread is 2.9), scales around 2^-9 over sqrt(K) of 1024
    mid = 127 + round(math.log2(K ** -0.5 / 2.9))
    return _bytes(g, 0, 256, E, rows, K // 2), _bytes(g, mid - 1, mid + 2, E, rows, K // 32)


def prepare(case, seed):
    g = _gen(seed)
    op, M = case["op"], case["M"]
    t = dict(case)
    if op == "epi":
        N, K = case["N"], case["K"]
        t["a_scale"] = t["b_scale"] = None
        if case["dtype"] == "i8a8":
            t["a"], t["a_scale"] = _codes(g, M, K)
            t["b"], sb = _codes(g, N, K)
            t["b_scale"] = K ** -0.5 * sb
        else:
            t["a"], t["b"] = _activation(g, M, K), (K ** -0.5 * _randn(g, N, K)).bfloat16()
        t["bias"] = 0.5 * _randn(g, N) if case["bias"] else None
        t["residual"] = (4 * _randn(g, M, N)).bfloat16() if case["residual"] else None
    elif op == "norm":
        n = case["n"]
        t["x"] = _activation(g, M, n)
        t["residual"] = (4 * _randn(g, M, n)).bfloat16() if case["residual"] else None
        t["w_post"] = (1 + 0.1 * _randn(g, n)).bfloat16() if case["post"] else None
        t["w_pre"] = (1 + 0.1 * _randn(g, n)).bfloat16()
        shape = {"none": None, "channel": (n,), "token": (M, 1), "full": (M, n)}[case["gate"]]
        t["gate"] = None if shape is None else (0.7 + 0.3 * _randn(g, *shape)).bfloat16()
        t["res_scale"] = 1.0 if case["gate"] == "none" else 0.875
    else:
        n, f, E = case["n"], case["f"], case["E"]
        t["x"] = _activation(g, M, n)
        t["logits"] = 1.5 * _randn(g, M, E)
        if M >= 8:
            t["logits"][M - M // 8:] = -math.inf          # rows that pad the batch
        t["gate_up"], t["gate_up_scale"] = _experts(g, case["dtype"], E, 2 * f, n)
        t["down"], t["down_scale"] = _experts(g, case["dtype"], E, n, f)
    return t


# ------------------------------------------------------------------------------ the calls

def run(state):
    return _library(state) if own else _plain[state["op"]](state)


def _library(t):
    if "call" not in t:                       # bound once, as a program keeps its launches
        t["call"] = _bind(t)
    launch, ops, stream, result = t["call"]
    rc = launch(ops, stream)
    if rc:
        raise RuntimeError("the row refused the launch: %d" % rc)
    if t["op"] == "norm" and t["out"] != "bf16":
        h, q, scale, value = result
        M, n = q.shape
        if t["out"] == "i8":
            torch.mul(q, scale, out=value)
        else:                                 # a scale a group of 128
            each = scale.repeat_interleave(128, 1)[:, :n]
            torch.mul(q.view(torch.float8_e4m3fn).float(), each, out=value)
        return h, value
    return result


def _bind(t):
    import libr3d_amd as R
    empty = lambda shape, dtype: torch.empty(shape, dtype=dtype, device="cuda")  # noqa: E731
    kind = {"bf16": torch.bfloat16, "f32": torch.float32}
    op, M = t["op"], t["M"]
    if op == "epi":
        N, K = t["N"], t["K"]
        y = empty((M, N), kind[t["y"]])
        ops = R.GemmEpiOperands(t["a"], t["b"], y, a_scale=t["a_scale"], b_scale=t["b_scale"], bias=t["bias"],
                                residual=t["residual"], act=t["act"], dtype=t["dtype"], N=N, K=K, M=M)
        row = R.resolve("gemm_nt_epi", {"dtype": t["dtype"], "M": M, "N": N, "K": K})["name"]
        result = y
    elif op == "norm":
        n = t["n"]
        h, out, q, scale = empty((M, n), torch.bfloat16), None, None, None
        if t["out"] == "bf16":
            out = empty((M, n), torch.bfloat16)
            result = (h, out)
        else:
            q = empty((M, n), torch.int8 if t["out"] == "i8" else torch.uint8)
            scale = empty((M, 1 if t["out"] == "i8" else (n + 127) // 128), torch.float32)
            result = (h, q, scale, empty((M, n), torch.bfloat16))
        ops = R.RmsNormBlockOperands(t["x"], residual=t["residual"], w_post=t["w_post"], gate=t["gate"], w_pre=t["w_pre"],
                                     residual_out=h, out=out, q=q, scale=scale, n=n, eps=EPS, res_scale=t["res_scale"], M=M)
        row = "rmsnorm_block"
    else:
        n, k = t["n"], t["top_k"]
        y = empty((M, n), kind[t["y"]])
        ids, weights = empty((M, k), torch.int32), empty((M, k), torch.float32)
        result = (y, ids, weights)
        ops = R.MoeLayerOperands(t["x"], t["logits"], t["gate_up"], t["down"], y, gate_up_scale=t["gate_up_scale"],
                                 down_scale=t["down_scale"], ids=ids, weights=weights, dtype=t["dtype"], n=n, f=t["f"],
                                 E=t["E"], top_k=k, act=t["act"], score=t["score"], renorm=t["renorm"], M=M)
        row = "moe_layer"
    need = R.row_scratch_bytes(row, ops)
    if need > 0:
        ops.set_scratch(empty((need,), torch.uint8), need)
    return R.row_launcher(row), ops, torch.cuda.current_stream().cuda_stream, result


# -------------------------------------------------------------------------- the plain forms

def _sigmoid(v):
    return 1.0 / (1.0 + torch.exp(-v))


_act = {
    "none": lambda v: v,
    "relu": lambda v: v.clamp_min(0.0),
    "silu": lambda v: v * _sigmoid(v),
    "sigmoid": _sigmoid,
    "gelu": lambda v: 0.5 * v * (1.0 + torch.erf(v * 0.5 ** 0.5)),
    "gelu_tanh": lambda v: v * _sigmoid(2.0 * (2.0 / math.pi) ** 0.5 * (v + 0.044715 * v * v * v)),
}
_store = {"bf16": torch.Tensor.bfloat16, "f32": torch.Tensor.float}


def _epi(t):
    v = t["a"].float() @ t["b"].float().T
    if t["a_scale"] is not None:
        v = v * t["a_scale"][:, None] * t["b_scale"]
    if t["bias"] is not None:
        v = v + t["bias"]
    v = _act[t["act"]](v)
    if t["residual"] is not None:
        v = v + t["residual"].float()
    return _store[t["y"]](v)


def _rms(v, w):
    return v * (1.0 / torch.sqrt(v.double().square().mean(1, keepdim=True) + EPS)).float() * w.float()


def _norm(t):
    h = t["x"].float()
    if t["w_post"] is not None:
        h = _rms(h, t["w_post"])
    if t["gate"] is not None:
        h = h * t["gate"].float()
    if t["residual"] is not None:
        h = t["residual"].float() * t["res_scale"] + h
    v = _rms(h, t["w_pre"])
    if t["out"] == "i8":                      # amax on 127, to nearest even
        amax = v.abs().amax(1, keepdim=True)
        s = torch.where(amax > 0, (amax * (1.0 / 127.0)).clamp_min(TINY), 1.0)
        v = torch.round(v * (1.0 / s)).clamp(-127, 127) * s
    elif t["out"] == "e4m3":                  # amax of 128 on 448
        M, n = v.shape
        g = torch.nn.functional.pad(v, (0, -n % 128)).view(M, -1, 128)
        amax = g.abs().amax(2, keepdim=True)
        s = torch.where(amax > 0, amax * (1.0 / 448.0), 1.0)
        g = (g * (1.0 / s)).clamp(-448, 448).to(torch.float8_e4m3fn).float() * s
        v = g.view(M, -1)[:, :n]
    return h.bfloat16(), v.bfloat16()


_E2M1 = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, -0.0, -0.5, -1.0, -1.5, -2.0, -3.0, -4.0, -6.0]


def _weights(w, scale, dtype):
    """f32 weights of [..., rows, K] codes."""
    if dtype == "bf16":
        return w.float()
    if dtype == "i8":
        return w.float() * scale[..., None]
    pair = torch.stack((w & 15, w >> 4), -1).flatten(-2)              # the low nibble is the even column
    v = torch.tensor(_E2M1, device=w.device)[pair.int()]
    return (v.unflatten(-1, (-1, 32)) * torch.exp2(scale.float() - 127.0)[..., None]).flatten(-2)


def _route(t):
    """ids [M, k] (-1: none) and f32 weights [M, k], by falling logit, ties by index."""
    x = t["logits"].float()
    value, at = torch.sort(x, dim=1, descending=True, stable=True)
    value, at = value[:, :t["top_k"]], at[:, :t["top_k"]]
    there = value > -math.inf
    top = torch.where(there[:, :1], value[:, :1], 0.0)
    if t["score"] == "softmax":
        w = torch.exp(value - top)
        total = w.sum(1, keepdim=True) if t["renorm"] else torch.exp(x - top).sum(1, keepdim=True)
        w = w / torch.where(there[:, :1], total, 1.0)
    else:
        w = _sigmoid(value)
        if t["renorm"]:
            w = w / torch.where(there[:, :1], w.sum(1, keepdim=True), 1.0)
    return torch.where(there, at, -1).int(), w * there


def _moe(t):
    ids, weights = _route(t)
    M, E, k, dtype = t["M"], t["E"], t["top_k"], t["dtype"]
    x = t["x"].float()
    pick = ids.clamp_min(0).long()
    if M * k < E:                             # the chosen experts' planes, one product a choice
        at = pick.flatten()
        scales = [None if t[s] is None else t[s][at] for s in ("gate_up_scale", "down_scale")]
        gu = _weights(t["gate_up"][at], scales[0], dtype) @ x.repeat_interleave(k, 0)[:, :, None]
        gate, up = gu[:, :, 0].chunk(2, 1)
        h = _act[t["act"]](gate) * up * weights.reshape(-1, 1)
        y = (_weights(t["down"][at], scales[1], dtype) @ h[:, :, None]).view(M, k, -1).sum(1)
    else:                                     # every expert over every token, weight 0 where not chosen
        dense = torch.zeros(M, E, device=x.device).scatter_add_(1, pick, weights)
        gu = torch.matmul(_weights(t["gate_up"], t["gate_up_scale"], dtype), x.T.contiguous())
        gate, up = gu.chunk(2, 1)             # [E, f, M]
        h = _act[t["act"]](gate) * up * dense.T[:, None, :]
        y = torch.matmul(_weights(t["down"], t["down_scale"], dtype), h).sum(0).T
    return _store[t["y"]](y.contiguous()), ids, weights


_plain = dict(epi=_epi, norm=_norm, moe=_moe)


# ------------------------------------------------------------------- what a pass must do

def work(case):
    op, M = case["op"], case["M"]
    size = {"bf16": 2, "f32": 4}
    if op == "epi":
        N, K = case["N"], case["K"]
        e = 2 if case["dtype"] == "bf16" else 1
        b = e * (N * K + M * K) + size[case["y"]] * M * N + (4 * N if case["bias"] else 0)
        b += (2 * M * N if case["residual"] else 0) + (4 * (M + N) if e == 1 else 0)
        return {"bytes": b, "flops": 2 * M * N * K}
    if op == "norm":
        n = case["n"]
        b = M * n * (2 + 2 + (2 if case["residual"] else 0) + (2 if case["out"] == "bf16" else 1))
        b += {"none": 0, "channel": 2 * n, "token": 2 * M, "full": 2 * M * n}[case["gate"]] + 2 * n * (1 + case["post"])
        return {"bytes": b, "flops": 0}
    n, f, E, k = case["n"], case["f"], case["E"], case["top_k"]
    rows = M - M // 8 if M >= 8 else M        # padded rows choose no expert
    read = E * (1.0 - (1.0 - k / E) ** rows)  # experts that someone chose
    b = read * 3 * n * f * WEIGHT_BYTES[case["dtype"]] + (read * 4 * (2 * f + n) if case["dtype"] == "i8" else 0)
    return {"bytes": int(b) + M * (2 * n + 4 * E + 8 * k + size[case["y"]] * n), "flops": 6 * rows * k * n * f}


# ------------------------------------------------------------------ the same in 64 bits

def _exact_act(name, v):
    if name == "relu":
        return torch.where(v > 0, v, torch.zeros_like(v))
    if name == "silu":
        return v * torch.sigmoid(v)
    if name == "sigmoid":
        return torch.sigmoid(v)
    if name == "gelu":
        return v * 0.5 * torch.erfc(-v / math.sqrt(2.0))
    if name == "gelu_tanh":
        return 0.5 * v * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (v + 0.044715 * v.pow(3))))
    return v


def _exact_epi(t):
    a = t["a"].double()
    if t["a_scale"] is not None:
        a = a * t["a_scale"].double()[:, None]
    out = []
    for n in range(0, t["N"], 4096):          # some weight rows at a time
        b = t["b"][n:n + 4096].double()
        if t["b_scale"] is not None:
            b = b * t["b_scale"][n:n + 4096].double()[:, None]
        v = torch.mm(a, b.T)
        if t["bias"] is not None:
            v += t["bias"][n:n + 4096].double()
        v = _exact_act(t["act"], v)
        if t["residual"] is not None:
            v = t["residual"][:, n:n + 4096].double() + v
        out.append(v)
    return torch.cat(out, 1)


def _unit_rms(v):
    return v * torch.rsqrt(v.pow(2).mean(1, keepdim=True) + EPS)


def _to_e4m3(v):
    """The nearest of sign, four exponent and three fraction bits, within 448."""
    step = torch.exp2(torch.floor(torch.log2(v.abs().clamp_min(2.0 ** -6))) - 3)
    return (torch.round(v / step) * step).clamp(-448, 448)


def _exact_norm(t):
    h = t["x"].double()
    if t["w_post"] is not None:
        h = t["w_post"].double() * _unit_rms(h)
    if t["gate"] is not None:
        h = t["gate"].double() * h
    if t["residual"] is not None:
        h = h + t["res_scale"] * t["residual"].double()
    v = t["w_pre"].double() * _unit_rms(h)
    if t["out"] == "i8":
        s = v.abs().amax(1, keepdim=True) / 127.0
        v = torch.round(v / s) * s
    elif t["out"] == "e4m3":
        parts = []
        for k in range(0, t["n"], 128):
            part = v[:, k:k + 128]
            s = part.abs().amax(1, keepdim=True) / 448.0
            parts.append(_to_e4m3(part / s) * s)
        v = torch.cat(parts, 1)
    return h, v


def _exact_plane(w, scale, dtype):
    """One expert's plane in 64 bits."""
    if dtype == "bf16":
        return w.double()
    if dtype == "i8":
        return w.double() * scale.double()[:, None]
    v = torch.empty(w.shape[0], 2 * w.shape[1], dtype=torch.float64, device=w.device)
    for nibble, part in ((0, w % 16), (1, w // 16)):
        size = part % 8
        e, odd = (size // 2).double(), (size % 2).double()
        mag = torch.where(size < 2, odd * 0.5, (1.0 + 0.5 * odd) * torch.exp2(e - 1.0))
        v[:, nibble::2] = torch.where(part >= 8, -mag, mag)
    return v * torch.exp2(scale.double() - 127.0).repeat_interleave(32, 1)


def _exact_moe(t):
    M, E, k, dtype = t["M"], t["E"], t["top_k"], t["dtype"]
    logits = t["logits"].double()
    ids = torch.full((M, k), -1, dtype=torch.int32)
    weights = torch.zeros(M, k, dtype=torch.float64)
    for m in range(M):                        # a token at a time, over the logits that are there
        row = [(-v, e) for e, v in enumerate(logits[m].tolist()) if v > -math.inf]
        chosen = sorted(row)[:k]
        if not chosen:
            continue
        if t["score"] == "softmax":
            top = -chosen[0][0]
            s = [math.exp(-v - top) for v, _ in chosen]
            total = sum(s) if t["renorm"] else math.fsum(math.exp(-v - top) for v, _ in row)
        else:
            s = [1.0 / (1.0 + math.exp(v)) for v, _ in chosen]
            total = sum(s) if t["renorm"] else 1.0
        for i, (_, e) in enumerate(chosen):
            ids[m, i], weights[m, i] = e, s[i] / total
    x = t["x"].double()
    y = torch.zeros(M, t["n"], dtype=torch.float64, device=x.device)
    scale = lambda name, e: None if t[name] is None else t[name][e]  # noqa: E731
    for e in range(E):
        m, i = torch.nonzero(ids == e, as_tuple=True)
        if not len(m):
            continue
        m, w = m.to(x.device), weights[m, i].to(x.device)
        gu = torch.mm(x[m], _exact_plane(t["gate_up"][e], scale("gate_up_scale", e), dtype).T)
        h = _exact_act(t["act"], gu[:, :t["f"]]) * gu[:, t["f"]:] * w[:, None]
        y.index_add_(0, m, torch.mm(h, _exact_plane(t["down"][e], scale("down_scale", e), dtype).T))
    return y, ids, weights


def exact(case, seed):
    return {"epi": _exact_epi, "norm": _exact_norm, "moe": _exact_moe}[case["op"]](prepare(case, seed))
