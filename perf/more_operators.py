"""Expert routing and layers of 4-bit group-quantised weights as cases that can be timed and checked one by one.

A weight is a 4-bit code q with a scale s and a zero point z for each group of 32, 64 or 128 values along k: w = (q - z) * s, z = 8 where there
are no zero points.  Activations, scales and outputs have 16 bits.

Kinds of case (`"kind"`):
  route    router logits -> the chosen experts of every token and their weights
  linear   16-bit activations (whole, or a slice of a wider buffer) times a 4-bit weight, with or without a bias
  moe      an expert layer for given experts and weights: up, gate, SiLU * mul, down, weighted sum
"""
import math
import os
import sys

import torch

own = False

DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def listed():
    return [
        # one token of a mixture of 256 experts in groups, chosen with a bias for balance: nothing but latency
        {"name": "route_t1", "kind": "route", "T": 1, "E": 256, "k": 8, "scoring": "sigmoid", "bias": True, "groups": 8, "top_groups": 4, "group_score": "top2", "dtype": "fp32"},
        # a prompt of odd length through the same router
        {"name": "route_t4093", "kind": "route", "T": 4093, "E": 256, "k": 8, "scoring": "sigmoid", "bias": True, "groups": 8, "top_groups": 4, "group_score": "top2", "dtype": "fp32"},
        # a large prefill batch, softmax over 128 experts
        {"name": "route_t16384", "kind": "route", "T": 16384, "E": 128, "k": 8, "scoring": "softmax", "bias": False, "groups": 1, "top_groups": 1, "group_score": "max", "dtype": "bf16"},
        # a small model's projection for one token
        {"name": "linear_m1_small", "kind": "linear", "M": 1, "N": 2048, "K": 2048, "pitch": 2048, "G": 128, "zero": True, "bias": True, "dtype": "bf16"},
        # a 70B-class up projection for one token
        {"name": "linear_m1", "kind": "linear", "M": 1, "N": 28672, "K": 8192, "pitch": 8192, "G": 128, "zero": True, "bias": False, "dtype": "fp16"},
        # a down projection for an odd decode batch, finer groups
        {"name": "linear_m7", "kind": "linear", "M": 7, "N": 5120, "K": 13824, "pitch": 13824, "G": 64, "zero": True, "bias": False, "dtype": "bf16"},
        # a larger decode batch, finest groups, no zero points; the activations are a slice of a wider buffer
        {"name": "linear_m33", "kind": "linear", "M": 33, "N": 17408, "K": 5120, "pitch": 10240, "G": 32, "zero": False, "bias": False, "dtype": "bf16"},
        # a prompt of odd length
        {"name": "linear_m4001", "kind": "linear", "M": 4001, "N": 17408, "K": 5120, "pitch": 5120, "G": 128, "zero": True, "bias": False, "dtype": "bf16"},
        # a mixture of 128 small experts: one user's stream, a small batch, a prompt's chunk
        {"name": "moe_t1", "kind": "moe", "T": 1, "E": 128, "k": 8, "H": 2048, "I": 768, "G": 128, "zero": True, "pad": 0, "dtype": "bf16"},
        {"name": "moe_t16", "kind": "moe", "T": 16, "E": 128, "k": 8, "H": 2048, "I": 768, "G": 64, "zero": True, "pad": 0, "dtype": "fp16"},
        # a batch of odd size with padding at its end, whose tokens go to no expert
        {"name": "moe_t311", "kind": "moe", "T": 311, "E": 64, "k": 6, "H": 2048, "I": 1408, "G": 32, "zero": False, "pad": 9, "dtype": "bf16"},
        {"name": "moe_t4096", "kind": "moe", "T": 4096, "E": 128, "k": 8, "H": 2048, "I": 768, "G": 128, "zero": True, "pad": 0, "dtype": "bf16"},
    ]


def _log(rng, lo, hi, step=1):
    v = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi))) / step)) * step
    return max((lo + step - 1) // step * step, min(hi // step * step, v))


def draw(rng):
    kind = rng.choice(["route", "route", "linear", "linear", "linear", "linear", "moe", "moe", "moe", "moe"])
    if kind == "route":
        E, groups = rng.choice([(8, 1), (16, 4), (60, 1), (64, 8), (96, 6), (128, 1), (160, 8), (256, 8), (384, 1), (512, 1), (512, 16)])
        bias = rng.random() < 0.5
        top_groups = rng.randint(1, groups)
        return {"kind": kind, "T": _log(rng, 1, min(16384, (1 << 21) // E)), "E": E, "k": rng.randint(1, min(10, E // groups * top_groups)),
                "scoring": rng.choice(["sigmoid", "softmax"]), "bias": bias, "groups": groups, "top_groups": top_groups,
                "group_score": rng.choice(["max", "top2"]), "dtype": rng.choice(["fp32", "bf16", "fp16"])}
    dtype, zero, G = rng.choice(["bf16", "fp16"]), rng.random() < 0.7, rng.choice([32, 64, 128, 128])
    while kind == "linear":
        M = _log(rng, 1, 16) if rng.random() < 0.5 else _log(rng, 17, 4096)
        K = _log(rng, 256, 28672, G)
        c = {"kind": kind, "M": M, "N": _log(rng, 128, 28672, rng.choice([1, 8, 128])), "K": K, "pitch": K + rng.choice([0, 0, 1, 512]), "G": G, "zero": zero,
             "bias": rng.random() < 0.5, "dtype": dtype}
        if c["N"] * c["K"] <= 28672 * 8192 and c["M"] * c["N"] * c["K"] <= 4001 * 17408 * 5120:
            return c
    while True:
        E = rng.choice([8, 16, 60, 64, 128])
        c = {"kind": kind, "T": _log(rng, 1, 32) if rng.random() < 0.6 else _log(rng, 33, 4096), "E": E, "k": rng.randint(1, 8),
             "H": _log(rng, 1024, 4096, 128), "I": _log(rng, 512, 4096, G), "G": G, "zero": zero, "pad": 0, "dtype": dtype}
        c["pad"] = rng.choice([0, c["T"] // 10])
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


def _weight(g, N, K, G, zero, dt, experts=()):
    """Codes, scales and zero points as a quantiser of near-normal weights leaves them: codes uint8 [.., N, K / 2], two to a byte with the even k in
    the lower half; scales and zero points [.., K / G, N]."""
    z = torch.randint(6, 11, (*experts, K // G, N), generator=g, device=DEV, dtype=torch.uint8) if zero else None
    s = ((0.5 + torch.rand(*experts, K // G, N, generator=g, device=DEV)) * (0.25 / math.sqrt(K))).to(dt)
    q = torch.randn(*experts, N, K // G, G, generator=g, device=DEV, dtype=torch.float16).mul_(2.6)
    q += z.transpose(-1, -2).unsqueeze(-1).half() if zero else 8
    q = q.round_().clamp_(0, 15).to(torch.uint8).view(*experts, N, K // 2, 2)
    return {"w": q[..., 0] | (q[..., 1] << 4), "s": s, "z": z}


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    s = dict(case)
    dt = DTYPES[case["dtype"]]
    if case["kind"] == "route":
        T, E = case["T"], case["E"]
        s["logits"] = (1.5 * torch.randn(T, E, generator=g, device=DEV)).to(dt)
        if T >= 8:
            s["logits"][T // 2].zero_()      # a row of padding: all experts alike
        s["b"] = 0.1 * torch.randn(E, generator=g, device=DEV) if case["bias"] else None
    elif case["kind"] == "linear":
        M, N, K = case["M"], case["N"], case["K"]
        s["x"] = _hidden(g, M, case["pitch"]).to(dt)[:, :K]
        s["weight"] = _weight(g, N, K, case["G"], case["zero"], dt)
        s["b"] = torch.randn(N, generator=g, device=DEV).to(dt) if case["bias"] else None
    else:
        T, E, k, H, I = (case[n] for n in ("T", "E", "k", "H", "I"))
        s["x"] = _hidden(g, T, H).to(dt)
        s["up"] = _weight(g, 2 * I, H, case["G"], case["zero"], dt, (E,))
        s["down"] = _weight(g, H, I, case["G"], case["zero"], dt, (E,))
        p, ids = torch.softmax(torch.randn(T, E, generator=g, device=DEV), 1).topk(k, 1)
        s["topk_weights"], s["topk_ids"] = (p / p.sum(1, keepdim=True)).contiguous(), ids.to(torch.int32)
        if case["pad"]:
            s["topk_ids"][-case["pad"]:], s["topk_weights"][-case["pad"]:] = -1, 0
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
    if s["kind"] == "route":
        return p.route_experts(s["logits"], s["k"], scoring=s["scoring"], bias=s["b"], num_groups=s["groups"], top_groups=s["top_groups"], group_score=s["group_score"])
    if s["kind"] == "linear":
        w = s["weight"]
        return p.linear_w4(s["x"], w["w"], w["s"], w["z"], s["b"])
    u, d = s["up"], s["down"]
    return p.moe_forward_w4(s["x"], s["topk_weights"], s["topk_ids"], u["w"], u["s"], d["w"], d["s"], u["z"], d["z"])


# -------------------------------------------------------------------------------------------------------- the plain forms
def _route(s):
    """Choices go by 64 bits, so that no rounding decides between two experts; the weights are computed in 32."""
    logits, k = s["logits"].double(), s["k"]

    def scores(l):
        if s["scoring"] == "sigmoid":
            return 1 / (1 + torch.exp(-l))
        e = torch.exp(l - l.amax(1, keepdim=True))
        return e / e.sum(1, keepdim=True)

    key = logits if s["b"] is None else scores(logits) + s["b"].double()
    if s["groups"] > 1:
        parts = (len(logits), s["groups"], -1)
        if s["group_score"] == "max":
            of_group = key.view(parts).amax(-1)
        else:
            best = scores(logits) if s["b"] is None else key
            of_group = torch.sort(best.view(parts), dim=-1, descending=True).values[..., :2].sum(-1)
        groups = torch.sort(of_group, dim=1, descending=True, stable=True).indices[:, :s["top_groups"]]
        out = torch.ones_like(of_group, dtype=torch.bool).scatter_(1, groups, False)
        key = key.view(parts).masked_fill(out[..., None], -math.inf).view(len(logits), -1)
    ids = torch.sort(key, dim=1, descending=True, stable=True).indices[:, :k]      # equal keys: the lowest index first
    w = scores(s["logits"].float()).gather(1, ids)
    return w / w.sum(1, keepdim=True), ids.to(torch.int32)


def _dequant(weight, dtype=torch.float32):
    """fp32 [.., N, K]"""
    w, s, z = weight["w"], weight["s"], weight["z"]
    q = torch.stack((w & 15, w >> 4), -1).to(dtype)
    *e, N, half, _ = q.shape
    q = q.view(*e, N, s.shape[-2], -1)
    q = q - (8 if z is None else z.to(dtype).transpose(-1, -2).unsqueeze(-1))
    return (q * s.to(dtype).transpose(-1, -2).unsqueeze(-1)).view(*e, N, 2 * half)


def _of(weight, experts):
    return {n: None if t is None else t[experts] for n, t in weight.items()}


def _experts(x, up, down):
    """x [G, R, H]: each group's rows through its expert, fp32."""
    g, u = torch.bmm(x, _dequant(up).transpose(1, 2)).chunk(2, -1)
    return torch.bmm(g / (1 + torch.exp(-g)) * u, _dequant(down).transpose(1, 2))


def _moe(s):
    T, E, k = s["T"], s["E"], s["k"]
    x, flat = s["x"].float(), s["topk_ids"].long().view(-1)
    token = torch.arange(T * k, device=DEV) // k
    if T * k <= E:      # an expert's matrices for every pair
        some = flat.clamp(min=0)
        y = _experts(x[token][:, None], _of(s["up"], some), _of(s["down"], some))[:, 0]
    else:               # each expert's pairs behind one another, padded to the fullest expert; pairs of no expert come last
        flat = torch.where(flat < 0, E, flat)
        order = torch.sort(flat, stable=True).indices
        counts = torch.bincount(flat, minlength=E + 1)
        rank = torch.empty_like(order)
        rank[order] = torch.arange(T * k, device=DEV) - (counts.cumsum(0) - counts)[flat[order]]
        cap = max(1, int(counts[:E].max()))
        slot = torch.where(flat < E, flat * cap + rank, E * cap)
        rows = torch.zeros(E * cap + 1, s["H"], device=DEV)
        rows[slot] = x[token]
        y = rows.clone()
        y[:-1] = _experts(rows[:-1].view(E, cap, -1), s["up"], s["down"]).view(E * cap, -1)
        y = y[slot]
    w = torch.where(s["topk_ids"] < 0, 0, s["topk_weights"])
    return (y.view(T, k, -1) * w[..., None]).sum(1)


def _run_plain(s):
    if s["kind"] == "route":
        return _route(s)
    dt = DTYPES[s["dtype"]]
    if s["kind"] == "linear":
        out = s["x"].float() @ _dequant(s["weight"]).t()
        return (out if s["b"] is None else out + s["b"].float()).to(dt)
    return _moe(s).to(dt)


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ------------------------------------------------------------------------------------------------------------------- work
def work(case):
    if case["kind"] == "route":
        T, E, k = case["T"], case["E"], case["k"]
        return {"bytes": T * E * (4 if case["dtype"] == "fp32" else 2) + 8 * T * k + (4 * E if case["bias"] else 0), "flops": 8 * T * E}
    per = 0.5 + (3 if case["zero"] else 2) / case["G"]      # bytes of a weight with its share of scale and zero point
    if case["kind"] == "linear":
        M, N, K = case["M"], case["N"], case["K"]
        return {"bytes": 2 * M * K + N * K * per + 2 * M * N + (2 * N if case["bias"] else 0), "flops": 2 * M * N * K}
    E, k, H, I = (case[n] for n in ("E", "k", "H", "I"))
    T = case["T"] - case["pad"]
    touched = E * (1 - (1 - k / E) ** T)      # experts that T tokens choose on average, each choosing k of E
    return {"bytes": touched * 3 * H * I * per + 4 * case["T"] * H + 8 * case["T"] * k, "flops": 6 * T * k * H * I}


# ----------------------------------------------------------------------------------------------------- the same in 64 bits
def _full64(p):
    low, high = torch.bitwise_and(p["w"], 0x0F), torch.bitwise_right_shift(p["w"], 4)
    codes = torch.empty(*low.shape[:-1], 2 * low.shape[-1], dtype=torch.float64, device=DEV)
    codes[..., ::2], codes[..., 1::2] = low, high
    per = codes.shape[-1] // p["s"].shape[-2]
    zero = 8.0 if p["z"] is None else torch.repeat_interleave(p["z"].double().mT, per, dim=-1)
    return codes.sub_(zero).mul_(torch.repeat_interleave(p["s"].double().mT, per, dim=-1))


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "route":
        l, k, n = s["logits"].double(), case["k"], case["groups"]
        p = torch.sigmoid(l) if case["scoring"] == "sigmoid" else torch.softmax(l, dim=1)
        choice = l if s["b"] is None else p + s["b"].double()
        if n > 1:
            of = (p if s["b"] is None and case["group_score"] == "top2" else choice).reshape(-1, n, case["E"] // n)
            best = of.topk(min(2, of.shape[2]) if case["group_score"] == "top2" else 1, dim=2).values.sum(2)
            keep = torch.argsort(best, dim=1, descending=True, stable=True)[:, :case["top_groups"]]
            member = torch.arange(case["E"], device=DEV) // (case["E"] // n)
            choice = torch.where((member[None, :, None] == keep[:, None, :]).any(2), choice, -math.inf)
        ids = torch.argsort(choice, dim=1, descending=True, stable=True)[:, :k]
        chosen = torch.take_along_dim(p, ids, 1)
        return chosen / torch.sum(chosen, 1, keepdim=True), ids.to(torch.int32)
    if case["kind"] == "linear":
        out = torch.matmul(s["x"].double(), _full64(s["weight"]).T)
        return out if s["b"] is None else out + s["b"].double()
    out = torch.zeros(case["T"], case["H"], dtype=torch.float64, device=DEV)
    for e in range(case["E"]):
        t, slot = torch.nonzero(s["topk_ids"] == e, as_tuple=True)
        if len(t):
            z = s["x"][t].double() @ _full64(_of(s["up"], e)).T
            gate, up = z[:, :case["I"]], z[:, case["I"]:]
            y = (gate * torch.sigmoid(gate) * up) @ _full64(_of(s["down"], e)).T
            out.index_add_(0, t, y * s["topk_weights"][t, slot].double().unsqueeze(1))
    return out
