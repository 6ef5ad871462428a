"""The 8-bit integer operators of this package as cases that can be timed and checked one by one.

Weights are int8 with one scale per output channel, activations are quantised to int8 with one scale per token.

Kinds of case (`"kind"`):
  quant    rows of 16-bit activations (a view of a wider buffer, or whole) -> int8 codes and a scale per row
  linear   codes and scales of the tokens, times int8 weights, to 16 bits; `dynamic`: straight from 16-bit activations
  mlp      residual add + RMSNorm + quantisation, gate_up linear, SiLU * mul + quantisation, down linear: half a decoder layer
  moe      from router logits to the weighted sum of the chosen experts' outputs
"""
import math
import os
import sys

import torch

own = False

DEV = "cuda"
EPS = 1e-6
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


def listed():
    return [
        # one token's hidden state in front of a projection: nothing but latency
        {"name": "quant_m1", "kind": "quant", "M": 1, "K": 5120, "pitch": 5120, "dtype": "bf16"},
        # a prompt's attention output, a slice of a wider buffer, of odd length
        {"name": "quant_m2047", "kind": "quant", "M": 2047, "K": 8192, "pitch": 10240, "dtype": "fp16"},
        # a small model's projection for one token, activations still in 16 bits
        {"name": "linear_m1_small", "kind": "linear", "M": 1, "N": 2048, "K": 2048, "dtype": "bf16", "bias": True, "dynamic": True},
        # a wide projection for a small decode batch
        {"name": "linear_m8", "kind": "linear", "M": 8, "N": 27648, "K": 5120, "dtype": "bf16", "bias": False, "dynamic": False},
        # an odd decode batch
        {"name": "linear_m27", "kind": "linear", "M": 27, "N": 17408, "K": 5120, "dtype": "bf16", "bias": False, "dynamic": False},
        # a prompt of odd length
        {"name": "linear_m4001", "kind": "linear", "M": 4001, "N": 17408, "K": 5120, "dtype": "bf16", "bias": False, "dynamic": False},
        # half a decoder layer for three tokens
        {"name": "mlp_m3", "kind": "mlp", "M": 3, "H": 5120, "I": 13824, "dtype": "fp16"},
        # half a 70B-class decoder layer for a prompt's chunk
        {"name": "mlp_m2048", "kind": "mlp", "M": 2048, "H": 8192, "I": 28672, "dtype": "bf16"},
        # a mixture of 128 small experts: one user's stream, a small batch, a prompt's chunk
        {"name": "moe_t1", "kind": "moe", "T": 1, "E": 128, "k": 8, "H": 2048, "I": 768, "dtype": "bf16"},
        {"name": "moe_t16", "kind": "moe", "T": 16, "E": 128, "k": 8, "H": 2048, "I": 768, "dtype": "bf16"},
        {"name": "moe_t4096", "kind": "moe", "T": 4096, "E": 128, "k": 8, "H": 2048, "I": 768, "dtype": "bf16"},
        # a mixture of few wide experts, three tokens
        {"name": "moe_t3_wide", "kind": "moe", "T": 3, "E": 8, "k": 2, "H": 4096, "I": 14336, "dtype": "fp16"},
    ]


def _log(rng, lo, hi, step=1):
    v = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi))) / step)) * step
    v = max(lo, min(hi, v))
    return v + step if v == 3072 else v


def draw(rng):
    kind = rng.choice(["quant", "linear", "linear", "linear", "mlp", "moe", "moe", "moe"])
    dtype = rng.choice(["bf16", "fp16"])
    if kind == "quant":
        K = _log(rng, 256, 28672, rng.choice([1, 8, 128]))
        M = _log(rng, 1, min(8192, 2047 * 8192 * 2 // K))
        pitch = K + rng.choice([0, 0, 8, 2048])
        return {"kind": kind, "M": M, "K": K, "pitch": pitch + 8 if pitch == 3072 else pitch, "dtype": dtype}
    if kind == "linear":
        while True:
            c = {"kind": kind, "M": _log(rng, 1, 4096), "N": _log(rng, 128, 28672, rng.choice([1, 8, 128])), "K": _log(rng, 256, 16384, rng.choice([16, 128])),
                 "dtype": dtype, "bias": rng.random() < 0.5, "dynamic": rng.random() < 0.5}
            if c["M"] * c["N"] * c["K"] <= 4001 * 17408 * 5120:
                return c
    if kind == "mlp":
        while True:
            c = {"kind": kind, "M": _log(rng, 1, 2048), "H": _log(rng, 1024, 8192, 128), "I": _log(rng, 2048, 28672, 128), "dtype": dtype}
            if c["M"] * c["H"] * c["I"] <= 1 << 37:
                return c
    while True:
        E = rng.choice([8, 16, 60, 64, 128])
        c = {"kind": kind, "T": _log(rng, 1, 32) if rng.random() < 0.6 else _log(rng, 33, 4096), "E": E, "k": rng.randint(1, 8),
             "H": _log(rng, 1024, 4096, 128), "I": _log(rng, 512, 4096, 128), "dtype": dtype}
        if c["k"] <= E and E * c["H"] * c["I"] <= 1 << 28 and c["T"] * c["k"] * c["H"] * c["I"] <= 4096 * 8 * 2048 * 768:
            return c


# ---------------------------------------------------------------------------------------------------------------- inputs
def _hidden(g, M, K):
    """Activations as a decoder layer has them: mostly normal, a few channels much larger, and in a batch one row of padding."""
    x = torch.randn(M, K, generator=g, device=DEV)
    x *= 1 + 19 * (torch.rand(K, generator=g, device=DEV) < 0.002).float()
    if M >= 8:
        x[M // 2].zero_()
    return x


def _weights(g, *shape):
    """Codes and scales as a per-channel quantiser leaves them: normal weights, the largest of a row at 127."""
    w = torch.randint(-127, 128, shape, generator=g, device=DEV, dtype=torch.int8)
    s = (0.5 + torch.rand(shape[:-1], generator=g, device=DEV)) * (0.02 / math.sqrt(shape[-1]))
    return w, s


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    dt = DTYPES[case["dtype"]]
    s = dict(case)
    kind = case["kind"]
    if kind == "quant":
        wide = _hidden(g, case["M"], case["pitch"]).to(dt)
        s["x"] = wide[:, :case["K"]]
    elif kind == "linear":
        M, N, K = case["M"], case["N"], case["K"]
        s["w"], s["ws"] = _weights(g, N, K)
        s["b"] = torch.randn(N, generator=g, device=DEV).to(dt) if case["bias"] else None
        if case["dynamic"]:
            s["x"] = _hidden(g, M, K).to(dt)
        else:
            s["q"] = (torch.randn(M, K, generator=g, device=DEV) * 32).clamp_(-127, 127).to(torch.int8)
            s["qs"] = 0.01 + 0.05 * torch.rand(M, generator=g, device=DEV)
    elif kind == "mlp":
        M, H, I = case["M"], case["H"], case["I"]
        s["hidden"] = _hidden(g, M, H).to(dt)
        s["residual"] = torch.randn(M, H, generator=g, device=DEV).to(dt)
        s["residual_out"] = torch.empty_like(s["residual"])
        s["norm"] = (1 + 0.1 * torch.randn(H, generator=g, device=DEV)).to(dt)
        s["w13"], s["s13"] = _weights(g, 2 * I, H)
        s["w2"], s["s2"] = _weights(g, H, I)
    else:
        T, E, H, I = case["T"], case["E"], case["H"], case["I"]
        s["x"] = _hidden(g, T, H).to(dt)
        s["logits"] = torch.randn(T, E, generator=g, device=DEV)
        s["w13"], s["s13"] = _weights(g, E, 2 * I, H)
        s["w2"], s["s2"] = _weights(g, E, H, I)
    return s


# ---------------------------------------------------------------------------------------------------------- the package's
_package = None


def _ops():
    global _package
    if _package is None:
        path = os.path.join(os.getcwd(), "llm-scaler_b200")
        if path not in sys.path:
            sys.path.insert(0, path)
        import custom_esimd_kernels_vllm as package
        package.set_overlap_mode(2)      # weights stay as they are while requests run
        _package = package
    return _package


def _run_own(s):
    p = _ops()
    kind, dt = s["kind"], DTYPES[s["dtype"]]
    if kind == "quant":
        return p.quantize_int8(s["x"])
    if kind == "linear":
        if s["dynamic"]:
            return p.linear_int8_dynamic(s["x"], s["w"], s["ws"], s["b"])
        return p.linear_int8(s["q"], s["qs"], s["w"], s["ws"], s["b"], dt)
    if kind == "mlp":
        q, qs = p.resadd_rmsnorm_quantize_int8(s["hidden"], s["residual"], s["norm"], EPS, s["residual_out"])
        gate_up = p.linear_int8(q, qs, s["w13"], s["s13"], None, dt)
        q, qs = p.silu_mul_quantize_int8(gate_up)
        return p.linear_int8(q, qs, s["w2"], s["s2"], None, dt), s["residual_out"]
    return p.moe_forward_int8(s["x"], s["logits"], s["w13"], s["s13"], s["w2"], s["s2"], s["k"])


# -------------------------------------------------------------------------------------------------------- the plain forms
def _quantize(x):
    """Codes (as fp32) and scales of fp32 rows.  127 x is exact for 16-bit x and the division rounds once, so codes are the
    definition's."""
    a = x.abs().amax(-1, keepdim=True).clamp(min=1e-12)
    return torch.round(127.0 * x / a), a[..., 0] / torch.full_like(a[..., 0], 127.0)


def _linear(q, qs, w, ws, b=None):
    out = (q @ w.float().t()) * qs[:, None] * ws[None, :]
    return out if b is None else out + b.float()


def _silu_mul(gate_up):
    g, u = gate_up.chunk(2, dim=-1)
    return g / (1.0 + torch.exp(-g)) * u


def _experts(q, qs, w13, s13, w2, s2):
    """q [G, R, H], qs [G, R], weights [G, ., .]: each group's rows through its expert, fp32."""
    h = torch.bmm(q, w13.float().transpose(1, 2)) * qs[..., None] * s13[:, None, :]
    q, qs = _quantize(_silu_mul(h))
    return torch.bmm(q, w2.float().transpose(1, 2)) * qs[..., None] * s2[:, None, :]


def _moe(s):
    T, E, k = s["T"], s["E"], s["k"]
    logits = s["logits"].float()
    top, ids = torch.sort(logits, dim=1, descending=True, stable=True)      # equal logits: the lowest index first
    top, ids = top[:, :k], ids[:, :k]
    w = torch.exp(top - top[:, :1])
    w = w / w.sum(1, keepdim=True)
    q, qs = _quantize(s["x"].float())
    flat = ids.reshape(-1)
    token = torch.arange(T * k, device=DEV) // k
    if T * k <= E:      # an expert's matrices for every pair
        y = _experts(q[token][:, None], qs[token][:, None], s["w13"][flat], s["s13"][flat], s["w2"][flat], s["s2"][flat])[:, 0]
    else:               # each expert's pairs behind one another, padded to the fullest expert
        order = torch.sort(flat, stable=True).indices
        counts = torch.bincount(flat, minlength=E)
        rank = torch.empty_like(order)
        rank[order] = torch.arange(T * k, device=DEV) - (counts.cumsum(0) - counts)[flat[order]]
        cap = int(counts.max())
        slot = flat * cap + rank
        rows = torch.zeros(E * cap, s["H"], device=DEV)
        scales = torch.zeros(E * cap, device=DEV)
        rows[slot], scales[slot] = q[token], qs[token]
        y = _experts(rows.view(E, cap, -1), scales.view(E, cap), s["w13"], s["s13"], s["w2"], s["s2"]).view(E * cap, -1)[slot]
    return (y.view(T, k, -1) * w[..., None]).sum(1)


def _run_plain(s):
    kind, dt = s["kind"], DTYPES[s["dtype"]]
    if kind == "quant":
        q, qs = _quantize(s["x"].float())
        return q.to(torch.int8), qs
    if kind == "linear":
        q, qs = _quantize(s["x"].float()) if s["dynamic"] else (s["q"].float(), s["qs"])
        return _linear(q, qs, s["w"], s["ws"], s["b"]).to(dt)
    if kind == "mlp":
        v = s["hidden"].float() + s["residual"].float()
        n = v * torch.rsqrt((v * v).mean(1, keepdim=True) + EPS) * s["norm"].float()
        gate_up = _linear(*_quantize(n), s["w13"], s["s13"]).to(dt)
        return _linear(*_quantize(_silu_mul(gate_up.float())), s["w2"], s["s2"]).to(dt), v.to(dt)
    return _moe(s).to(dt)


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ------------------------------------------------------------------------------------------------------------------- work
def work(case):
    kind = case["kind"]
    if kind == "quant":
        M, K = case["M"], case["K"]
        return {"bytes": 3 * M * K + 4 * M, "flops": 2 * M * K}
    if kind == "linear":
        M, N, K = case["M"], case["N"], case["K"]
        x = 2 * M * K if case["dynamic"] else M * K + 4 * M
        return {"bytes": x + N * K + 4 * N + 2 * M * N + (2 * N if case["bias"] else 0), "flops": 2 * M * N * K}
    if kind == "mlp":
        M, H, I = case["M"], case["H"], case["I"]
        return {"bytes": 3 * H * I + 4 * (2 * I + H) + 2 * H + 8 * M * H, "flops": 6 * M * H * I}
    T, E, k, H, I = (case[n] for n in ("T", "E", "k", "H", "I"))
    touched = E * (1 - (1 - k / E) ** T)      # experts that T tokens choose on average, each choosing k of E
    return {"bytes": touched * (3 * H * I + 4 * (2 * I + H)) + 4 * T * H + 4 * T * E, "flops": 6 * T * k * H * I}


# ----------------------------------------------------------------------------------------------------- the same in 64 bits
def _codes64(x):
    a = torch.clamp(torch.max(torch.abs(x), dim=-1).values, min=1e-12)
    return torch.round((127 * x) / a.unsqueeze(-1)), a / 127


def _matmul64(codes, scales, weight, weight_scale):
    return torch.matmul(codes, weight.double().T) * torch.outer(scales, weight_scale.double())


def _gated64(z):
    half = z.shape[-1] // 2
    return z[..., :half] * torch.sigmoid(z[..., :half]) * z[..., half:]


def exact(case, seed):
    s = prepare(case, seed)
    kind, dt = case["kind"], DTYPES[case["dtype"]]
    if kind == "quant":
        codes, scales = _codes64(s["x"].double())
        return codes.to(torch.int8), scales
    if kind == "linear":
        codes, scales = _codes64(s["x"].double()) if case["dynamic"] else (s["q"].double(), s["qs"].double())
        out = _matmul64(codes, scales, s["w"], s["ws"])
        return out if s["b"] is None else out + s["b"].double()
    if kind == "mlp":
        v = s["hidden"].double() + s["residual"].double()
        n = v / torch.sqrt(torch.mean(v ** 2, dim=1, keepdim=True) + EPS) * s["norm"].double()
        z = _matmul64(*_codes64(n), s["w13"], s["s13"]).to(dt).double()      # the first linear's output is one of 16 bits
        return _matmul64(*_codes64(_gated64(z)), s["w2"], s["s2"]), v
    T, k = case["T"], case["k"]
    out = torch.zeros(T, case["H"], dtype=torch.float64, device=DEV)
    order = torch.argsort(s["logits"].double(), dim=1, descending=True, stable=True)[:, :k]
    p = torch.softmax(s["logits"].double().gather(1, order), dim=1)
    codes, scales = _codes64(s["x"].double())
    for e in range(case["E"]):
        t, slot = torch.nonzero(order == e, as_tuple=True)
        if len(t):
            z = _matmul64(codes[t], scales[t], s["w13"][e], s["s13"][e])
            y = _matmul64(*_codes64(_gated64(z)), s["w2"][e], s["s2"][e])
            out.index_add_(0, t, y * p[t, slot].unsqueeze(1))
    return out
