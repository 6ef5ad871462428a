"""The 8-bit integer operators in 64 bits: one scale per row of codes, sums of integers exact.  They have no counterpart in the reference."""
import torch

MIN_AMAX = 1e-12


def quantize_rows(x: torch.Tensor):
    """Codes (int8), the unrounded 127 x / a they come from, and a / 127, of any float rows; a row that is not finite: zeros, NaN."""
    v = x.double()
    a = v.abs().amax(-1, keepdim=True).clamp(min=MIN_AMAX)
    finite = torch.isfinite(v).all(-1, keepdim=True)
    t = torch.where(finite, 127 * v / a, torch.zeros_like(v))
    scale = torch.where(finite, a / 127, torch.full_like(a, float("nan")))
    return t.round().to(torch.int8), t, scale[..., 0]


def silu_mul(gate_up: torch.Tensor):
    g, u = gate_up.double().chunk(2, -1)
    return g * torch.sigmoid(g) * u


def resadd_rmsnorm(hidden, residual, weight, eps):
    """(v, rmsnorm(v) * weight) of v = hidden + residual."""
    v = hidden.double() + residual.double()
    return v, v / torch.sqrt((v * v).mean(-1, keepdim=True) + eps) * weight.double()


def linear(codes, scale, weight, weight_scale, bias=None):
    """The products add up exactly: each is below 2^14, and there are fewer than 2^17."""
    out = (codes.double() @ weight.double().t()) * scale.double()[:, None] * weight_scale.double()[None, :]
    return out if bias is None else out + bias.double()


def route(logits, top_k, renormalize=True):
    """Chosen experts and weights; the lowest index first among equal logits."""
    l = logits.double()
    ids = torch.sort(l, dim=1, descending=True, stable=True).indices[:, :top_k]
    w = torch.softmax(l, 1).gather(1, ids)
    return ids, w / w.sum(1, keepdim=True) if renormalize else w


def moe(x, logits, w13, s13, w2, s2, top_k, renormalize=True):
    ids, w = route(logits, top_k, renormalize)
    codes, _, scale = quantize_rows(x)
    out = torch.zeros(x.shape[0], w2.shape[1], dtype=torch.float64)
    for e in ids.unique().tolist():
        t, slot = torch.nonzero(ids == e, as_tuple=True)
        h = silu_mul(linear(codes[t], scale[t], w13[e], s13[e]))
        q, _, r = quantize_rows(h)
        out.index_add_(0, t, linear(q, r, w2[e], s2[e]) * w[t, slot, None])
    return out
