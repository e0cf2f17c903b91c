"""Workloads of the int8 linear layer and of the sampler that follows the lm_head, as a serving
program calls them: operands, outputs and launch scratch bound once, then one row launch a pass.

Every case names one operator and its sizes:

  gemm    gemm_nt_q at i8a8: Y[M, N] = (A[M, K] . W[N, K]^T) * a_scale[m] * b_scale[n], int8 codes,
          one f32 scale a token and one an output channel, bf16 Y
  norm    rmsnorm_quant_i8: residual + x in bf16, its RMS norm, int8 codes with one scale a token
  quant   quant_act_i8: the same codes and scales of a bf16 activation
  gated   gated_quant_i8: the same of silu(gate) * up, gate_up [M, 2n]
  sample  sample_logits: one token a row from given uniform numbers, after the row's own
          temperature, top-k, top-p and min-p

Codes come back as the bf16 values that they and their scale stand for.  The sizes are those of
the 27B-class model that bench.py and the tests use: hidden 5376, MLP 21504, q/k/v joined 8192,
attention output 4096, vocabulary 262144.

`own` False computes the plain forms in elementary torch operations; True calls the library.
"""
import math

import torch

own = False

HIDDEN, MLP, QKV, ATTN, VOCAB = 5376, 21504, 8192, 4096, 262144
EPS = 1e-6
TINY = 2.0 ** -126                   # the least scale: the smallest normal f32


def listed():
    return [
        # one sequence decoding: a gate or up projection, the weights read once
        dict(name="gemm_gate_m1", op="gemm", M=1, N=MLP, K=HIDDEN),
        # an odd batch of decoding sequences: the down projection (long K, few rows)
        dict(name="gemm_down_m13", op="gemm", M=13, N=HIDDEN, K=MLP),
        # a prompt of no round length through a joined q/k/v plane that a shard cut unevenly
        dict(name="gemm_qkv_m333", op="gemm", M=333, N=QKV - 5, K=HIDDEN - 16),
        # a full prefill chunk through a gate or up projection: the largest product
        dict(name="gemm_gate_m2048", op="gemm", M=2048, N=MLP, K=HIDDEN),
        # a decode step's norm: launch and latency
        dict(name="norm_m4", op="norm", M=4, n=HIDDEN),
        # the same norm over one prefill chunk
        dict(name="norm_m2048", op="norm", M=2048, n=HIDDEN),
        # a decode step's attention output, before its projection
        dict(name="quant_m4", op="quant", M=4, n=ATTN),
        # the same over one prefill chunk
        dict(name="quant_m2048", op="quant", M=2048, n=ATTN),
        # a decode step's MLP: the joined gate_up row of four sequences
        dict(name="gated_m4", op="gated", M=4, n=MLP),
        # the same over one prefill chunk: the widest rows there are
        dict(name="gated_m2048", op="gated", M=2048, n=MLP),
        # one sequence decoding: its next token
        dict(name="sample_m1", op="sample", M=1, V=VOCAB, dtype="f32"),
        # a decode batch whose rows each have settings of their own, greedy ones among them
        dict(name="sample_m128", op="sample", M=128, V=VOCAB, dtype="f32"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["gemm", "gemm", "gemm", "norm", "quant", "gated", "sample", "sample"])
    if op == "gemm":
        lo, hi = rng.choice([(1, 16), (17, 128), (129, 2048)])
        while True:
            M, N, K = _log_int(rng, lo, hi), _log_int(rng, 500, MLP), 16 * _log_int(rng, 32, MLP // 16)
            if N * K >= 1 << 20 and N * K <= MLP * HIDDEN:
                return dict(op=op, M=M, N=N, K=K)
    if op == "sample":
        while True:
            M, V = _log_int(rng, 1, 256), _log_int(rng, 1000, VOCAB)
            if M * V <= 128 * VOCAB:
                return dict(op=op, M=M, V=V, dtype=rng.choice(["f32", "bf16"]))
    n = _log_int(rng, 500, MLP if op == "gated" else 8192)
    if rng.random() < 0.7:
        n = n // 8 * 8
    while True:
        M = _log_int(rng, 1, 4096)
        if M * n <= 2048 * {"norm": HIDDEN, "quant": ATTN, "gated": MLP}[op]:
            return dict(op=op, M=M, n=n)


# ------------------------------------------------------------------------------- inputs

def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def _rand(g, *shape):
    return torch.rand(*shape, generator=g, device="cuda")


def _pick(g, values, n):
    at = torch.randint(0, len(values), (n,), generator=g, device="cuda")
    return torch.tensor(values, device="cuda")[at]


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


def _logits(g, M, V, dtype):
    """Rows with a head of likely tokens over a broad tail; about one in eight rows has most of
    its tokens masked out, as a grammar does."""
    x = 2.5 * _randn(g, M, V)
    at = torch.randint(0, V, (M, 48), generator=g, device="cuda")
    x.scatter_(1, at, 8.0 + 2.0 * _randn(g, M, 48))
    strict = _rand(g, M, 1) < 0.125
    masked = _rand(g, M, V) < torch.where(strict, 0.995, 0.01)
    masked[:, 0] = False                      # something is always allowed
    x = x.masked_fill_(masked, -math.inf)
    return x.bfloat16() if dtype == "bf16" else x


def prepare(case, seed):
    g = _gen(seed)
    op, M = case["op"], case["M"]
    if op == "gemm":
        a, sa = _codes(g, M, case["K"])
        b, sb = _codes(g, case["N"], case["K"])
        return dict(op=op, a=a, a_scale=sa, b=b, b_scale=0.02 * sb)
    if op == "norm":
        n = case["n"]
        return dict(op=op, x=_activation(g, M, n), residual=(4 * _randn(g, M, n)).bfloat16(),
                    w=(1 + 0.1 * _randn(g, n)).bfloat16())
    if op == "quant":
        return dict(op=op, x=_activation(g, M, case["n"]))
    if op == "gated":
        return dict(op=op, x=_activation(g, M, 2 * case["n"]))
    return dict(op=op, logits=_logits(g, M, case["V"], case["dtype"]),
                temperature=_pick(g, [0.0, 0.6, 0.8, 1.0, 1.0, 1.3], M),
                top_k=_pick(g, [0, 0, 20, 50, 200, 1000], M).to(torch.int32),
                top_p=_pick(g, [1.0, 1.0, 0.95, 0.9, 0.5], M),
                min_p=_pick(g, [0.0, 0.0, 0.02, 0.1], M), u=_rand(g, M))


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
    if t["op"] in ("norm", "quant", "gated"):
        q, scale, value = result[0], result[1], result[2]
        torch.mul(q, scale, out=value)
        return (value,) + result[3:]
    return result


def _bind(t):
    import libr3d_amd as R
    empty = lambda shape, dtype: torch.empty(shape, dtype=dtype, device="cuda")  # noqa: E731
    op = t["op"]
    if op == "gemm":
        (M, K), N = t["a"].shape, len(t["b"])
        y = empty((M, N), torch.bfloat16)
        ops = R.GemmOperands(t["a"], t["a_scale"], t["b"], t["b_scale"], y, dtype="i8a8", N=N, K=K, M=M)
        row = R.resolve("gemm_nt_q", {"dtype": "i8a8", "M": M, "N": N, "K": K, "group": K})["name"]
        result = y
    elif op == "sample":
        M, V = t["logits"].shape
        token, prob = empty((M,), torch.int32), empty((M,), torch.float32)
        ops = R.SampleOperands(t["logits"], t["u"], token, prob, temperature=t["temperature"],
                               top_k=t["top_k"], top_p=t["top_p"], min_p=t["min_p"], n_vocab=V, M=M)
        row = "sample_logits"
        result = (token, prob)
    else:
        M, n = t["x"].shape
        n = n // 2 if op == "gated" else n
        q, scale = empty((M, n), torch.int8), empty((M, 1), torch.float32)
        result = (q, scale, empty((M, n), torch.bfloat16))
        if op == "norm":
            added = empty((M, n), torch.bfloat16)
            ops = R.RmsNormQuantI8Operands(t["x"], t["residual"], t["w"], q, scale, residual_out=added,
                                           n=n, eps=EPS, M=M)
            row = "rmsnorm_quant_i8"
            result += (added,)
        elif op == "quant":
            ops = R.QuantActI8Operands(t["x"], q, scale, n=n, M=M)
            row = "quant_act_i8"
        else:
            ops = R.GatedQuantI8Operands(t["x"], q, scale, n=n, act="silu", M=M)
            row = "gated_quant_i8"
    need = R.row_scratch_bytes(row, ops)
    if need > 0:
        ops.set_scratch(empty((need,), torch.uint8), need)
    return R.row_launcher(row), ops, torch.cuda.current_stream().cuda_stream, result


# -------------------------------------------------------------------------- the plain forms

def _gemm(t):
    y = t["a"].float() @ t["b"].float().T
    return (y * t["a_scale"][:, None] * t["b_scale"]).bfloat16()


def _quantised(h):
    """The values of h's int8 codes, one scale a row: amax on 127, to nearest even."""
    amax = h.abs().amax(1, keepdim=True)
    s = torch.where(amax > 0, (amax * (1.0 / 127.0)).clamp_min(TINY), 1.0)
    q = torch.round(h * (1.0 / s)).clamp(-127, 127)
    return (q * s).bfloat16()


def _norm(t):
    r = (t["residual"].float() + t["x"].float()).bfloat16()
    f = r.float()
    rs = (1.0 / torch.sqrt(f.double().square().mean(1, keepdim=True) + EPS)).float()
    return _quantised((f * rs) * t["w"].float()), r


def _quant(t):
    return (_quantised(t["x"].float()),)


def _gated(t):
    gate, up = t["x"].float().chunk(2, 1)
    return (_quantised(gate * (1.0 / (1.0 + torch.exp(-gate))) * up),)


def _sample(t):
    # in 64 bits throughout: a token's border is where a long sum passes a number
    x = t["logits"].double()
    M, V = x.shape
    top = x.amax(1, keepdim=True)
    greedy = t["temperature"][:, None] <= 0
    w = torch.exp((x - top) / torch.where(greedy, 1.0, t["temperature"][:, None]).double())
    value, at = torch.sort(x, dim=1, descending=True, stable=True)
    ws = w.gather(1, at)
    k = t["top_k"][:, None]
    k = torch.where(greedy, 1, torch.where(k > 0, k, V))
    keep = torch.arange(V, device="cuda") < k
    ws = ws * keep
    c = torch.cumsum(ws, 1)
    keep &= (c - ws < t["top_p"][:, None].double() * c[:, -1:]) | (t["top_p"][:, None] >= 1)
    keep &= ws >= t["min_p"][:, None].double()
    w = w * torch.zeros_like(keep).scatter_(1, at, keep)
    c = torch.cumsum(w, 1)
    total = c[:, -1:]
    token = (c <= t["u"][:, None].double() * total).sum(1, keepdim=True)
    last = (w > 0).long().mul(torch.arange(V, device="cuda")).amax(1, keepdim=True)
    token = torch.minimum(token, last)
    return token[:, 0].int(), (w.gather(1, token) / total)[:, 0].float()


_plain = dict(gemm=_gemm, norm=_norm, quant=_quant, gated=_gated, sample=_sample)


# ------------------------------------------------------------------- what a pass must do

def work(case):
    op, M = case["op"], case["M"]
    if op == "gemm":
        N, K = case["N"], case["K"]
        return {"bytes": N * K + M * K + 4 * (M + N) + 2 * M * N, "flops": 2 * M * N * K}
    if op == "sample":
        return {"bytes": M * case["V"] * (2 if case["dtype"] == "bf16" else 4) + 28 * M, "flops": 0}
    n = case["n"]
    if op == "norm":
        return {"bytes": M * n * (2 + 2 + 2 + 1) + 4 * M + 2 * n, "flops": 0}
    return {"bytes": M * n * (3 if op == "quant" else 5) + 4 * M, "flops": 0}


# ------------------------------------------------------------------ the same in 64 bits

def _on_127(h):
    s = h.abs().amax(1, keepdim=True) / 127.0
    return torch.round(h / s) * s


def exact(case, seed):
    t = prepare(case, seed)
    op = case["op"]
    if op == "gemm":
        a = t["a"].double() * t["a_scale"].double()[:, None]
        out = []
        for n in range(0, case["N"], 4096):   # some weight rows at a time
            b = t["b"][n:n + 4096].double() * t["b_scale"][n:n + 4096].double()[:, None]
            out.append(torch.mm(a, b.T))
        return torch.cat(out, 1)
    if op == "norm":
        r = t["x"].double() + t["residual"].double()
        h = r.bfloat16().double()             # the row that the norm is defined over
        h = h * torch.rsqrt(h.pow(2).mean(1, keepdim=True) + EPS) * t["w"].double()
        return _on_127(h), r
    if op == "quant":
        return (_on_127(t["x"].double()),)
    if op == "gated":
        n = case["n"]
        out = []
        for m in range(0, case["M"], 256):
            h = t["x"][m:m + 256].double()
            out.append(_on_127(h[:, :n] * torch.sigmoid(h[:, :n]) * h[:, n:]))
        return (torch.cat(out),)
    tokens, probs = [], []
    for m in range(case["M"]):                # a row at a time, over its kept tokens only
        x = t["logits"][m].double()
        T, k = float(t["temperature"][m]), int(t["top_k"][m])
        p, floor = float(t["top_p"][m]), float(t["min_p"][m])
        if T <= 0:
            tokens.append(int(torch.nonzero(x == x.max())[0]))
            probs.append(1.0)
            continue
        order = torch.argsort(-x, stable=True)
        if k > 0:
            order = order[:k]
        w = torch.exp((x[order] - x.max()) / T)
        kept = len(order)
        if p < 1:
            kept = 1 + int(torch.searchsorted(torch.cumsum(w, 0), p * w.sum()))
        kept = min(kept, int((w >= floor).sum()))
        order, back = torch.sort(order[:kept])
        w = w[:kept][back]
        c = torch.cumsum(w, 0)
        i = min(int(torch.searchsorted(c, t["u"][m].double() * c[-1], right=True)), kept - 1)
        tokens.append(int(order[i]))
        probs.append(float(w[i] / c[-1]))
    return (torch.tensor(tokens, dtype=torch.int32), torch.tensor(probs, dtype=torch.float64))
