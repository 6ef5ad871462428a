"""Expert routing and the layers of 4-bit group-quantised weights in 64 bits.  They have no counterpart in the reference."""
import math

import torch


def route(logits, top_k, scoring="softmax", bias=None, num_groups=1, top_groups=1, group_score="max", renormalize=True, scale=1.0):
    """Weights [T, k] (64 bits) and ids [T, k], token by token and expert by expert."""
    T, E = logits.shape
    weights, ids = torch.zeros(T, top_k, dtype=torch.float64), torch.full((T, top_k), -1, dtype=torch.int32)
    size = E // num_groups
    for t in range(T):
        l = logits[t].double()
        if bool((l != l).any()) or bool((l == math.inf).any()) or bool((l == -math.inf).all()):
            continue
        p = torch.sigmoid(l) if scoring == "sigmoid" else torch.softmax(l, 0)
        key = l.clone() if bias is None else p + bias.double()
        with_bias = p if bias is None else key.clone()
        dead = (l == -math.inf) | ~(key > -math.inf)
        key[dead], with_bias = -math.inf, torch.where(dead, torch.tensor(-math.inf, dtype=torch.float64), with_bias)
        if num_groups > 1:
            of = []
            for g in range(num_groups):
                best = sorted((with_bias if group_score == "top2" else key)[g * size:(g + 1) * size].tolist(), reverse=True)
                left = [b for b in best[:2 if group_score == "top2" else 1] if b > -math.inf]      # what is out of the choice does not count
                of.append(sum(left) if left else -math.inf)
            keep = sorted(range(num_groups), key=lambda g: (-of[g], g))[:top_groups]
            for g in range(num_groups):
                if g not in keep:
                    key[g * size:(g + 1) * size] = -math.inf
        order = sorted(range(E), key=lambda e: (-float(key[e]), e))[:top_k]
        order = [e for e in order if float(key[e]) > -math.inf]
        if not order:
            continue
        chosen = l[order]
        if renormalize:      # relative to the largest, so that nothing underflows
            log_p = torch.nn.functional.logsigmoid(chosen) if scoring == "sigmoid" else chosen
            w = torch.softmax(log_p, 0)
        else:
            w = p[order]
        weights[t, :len(order)], ids[t, :len(order)] = w * scale, torch.tensor(order, dtype=torch.int32)
    return weights, ids


def pack(q):
    """Codes [.., K] -> uint8 [.., K / 2], the even k in the low half."""
    return (q[..., 0::2] | (q[..., 1::2] << 4)).to(torch.uint8)


def quantize(weight, group, symmetric=False, dtype=torch.bfloat16):
    """Codes uint8 [.., N, K], scales [.., K / group, N] in `dtype`, zero points uint8 or None, of a float weight [.., N, K]: a group's range on 15 steps."""
    *lead, N, K = weight.shape
    w = weight.double().reshape(*lead, N, K // group, group)
    if symmetric:
        s = (w.abs().amax(-1) / 7).clamp(min=1e-8).to(dtype)
        z = torch.full_like(s, 8, dtype=torch.float64)
    else:
        lo, hi = w.amin(-1).clamp(max=0), w.amax(-1).clamp(min=0)
        s = ((hi - lo) / 15).clamp(min=1e-8).to(dtype)
        z = (-lo / s.double()).round().clamp(0, 15)
    q = ((w / s.double()[..., None]).round() + z[..., None]).clamp(0, 15).to(torch.uint8).reshape(*lead, N, K)
    turn = lambda a: a.transpose(-1, -2).contiguous()      # noqa: E731
    return q, turn(s), None if symmetric else turn(z.to(torch.uint8))


def dequant(packed, scale, zero=None):
    """(q - z) s in 64 bits, [.., N, K]."""
    b = packed.view(torch.uint8)
    q = torch.stack((b & 15, b >> 4), -1).flatten(-2).double()
    group = q.shape[-1] // scale.shape[-2]
    wide = lambda a: a.double().transpose(-1, -2).repeat_interleave(group, -1)      # noqa: E731
    return (q - (8.0 if zero is None else wide(zero))) * wide(scale)


def linear(x, packed, scale, zero=None, bias=None):
    out = x.double() @ dequant(packed, scale, zero).t()
    return out if bias is None else out + bias.double()


def expert(x, w13, w2):
    """One expert's output in 64 bits, of dequantised matrices."""
    g, u = (x.double() @ w13.t()).chunk(2, -1)
    return (g * torch.sigmoid(g) * u) @ w2.t()


def moe(x, weights, ids, w13, s13, w2, s2, z13=None, z2=None):
    """(out [T, H], size [T]): size^2 is the sum of the squares of what is added up, the scale of a row's rounding errors."""
    E = w13.shape[0]
    out, size = torch.zeros(x.shape[0], w2.shape[1], dtype=torch.float64), torch.zeros(x.shape[0], dtype=torch.float64)
    one = lambda t, e: None if t is None else t[e]      # noqa: E731
    for e in range(E):
        t, slot = torch.nonzero(ids == e, as_tuple=True)
        if len(t):
            y = expert(x[t], dequant(w13[e], s13[e], one(z13, e)), dequant(w2[e], s2[e], one(z2, e))) * weights[t, slot, None].double()
            out.index_add_(0, t, y)
            size.index_add_(0, t, (y * y).sum(1))
    return out, size.sqrt()
