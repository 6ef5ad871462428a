"""Inputs and tolerances of the tests of expert routing and the 4-bit group-quantised layers."""
import torch

from oracle import w4

DT = {"bf16": torch.bfloat16, "fp16": torch.float16}


def half_step(dtype):
    """What one rounding to `dtype` is off by at most, relative to the value."""
    return torch.finfo(dtype).eps / 2


def weight(g, N, K, group, dtype, zero=True, experts=()):
    """Codes over the whole range, zero points from 0 to 15, scales of either sign of about 1 / sqrt(K)."""
    q = torch.randint(0, 16, (*experts, N, K), generator=g, dtype=torch.uint8)
    s = ((torch.rand(*experts, K // group, N, generator=g) + 0.5) * 0.3 / K ** 0.5 * (1 - 2 * (torch.rand(*experts, K // group, N, generator=g) < 0.1).float())).to(dtype)
    z = torch.randint(0, 16, (*experts, K // group, N), generator=g, dtype=torch.uint8) if zero else None
    return w4.pack(q), s, z


def check_linear(out, x, packed, scale, zero=None, bias=None, what=""):
    """Three roundings to 16 bits at most: of a weight (many tokens), of the output, none of the sums, which are fp32.

    Per output: half a step of itself, half a step of every product, and K roundings of 2^-24 of the sums' terms, where q and z may be summed apart.
    Over all outputs: a weight's roundings are independent, so their share is half a step of the root of the sum of the products' squares."""
    u = half_step(x.dtype)
    w, v = w4.dequant(packed, scale, zero), x.double()
    ref = w4.linear(x, packed, scale, zero, bias)
    b = packed.view(torch.uint8)
    top = torch.stack((b & 15, b >> 4), -1).flatten(-2).double()
    group = top.shape[-1] // scale.shape[-2]
    wide = lambda a: a.double().transpose(-1, -2).repeat_interleave(group, -1)      # noqa: E731
    top = (top + (8.0 if zero is None else wide(zero))) * wide(scale).abs()
    terms, apart = v.abs() @ w.abs().t(), v.abs() @ top.t()
    d = (out.double().cpu() - ref).abs()
    tiny = torch.finfo(x.dtype).smallest_normal * torch.finfo(x.dtype).eps / 2
    bound = u * (ref.abs() + terms) + (v.shape[1] + 64) * 2.0 ** -24 * apart + tiny
    # the largest finite value and half a step is where `dtype` rounds to infinity: outputs surely beyond it are infinite, those that may be either may be either
    edge = torch.finfo(x.dtype).max * (1 + u / 2)
    got = out.double().cpu()
    beyond = ref.abs() - bound > edge
    assert bool((got[beyond] == torch.sign(ref[beyond]) * float("inf")).all()), what
    held = ref.abs() + bound < edge
    d, bound = torch.where(held, d, torch.zeros_like(d)), torch.where(held, bound, torch.ones_like(bound))
    assert bool((d <= bound).all()), "%s: %.3g of the bound" % (what, float((d / bound).max()))
    spread = ((v * v) @ (w * w).t()).sum().sqrt()
    norm = float(d.norm())
    most = float(u * (ref.norm() + spread) + 16 * 2.0 ** -24 * apart.norm() + tiny * d.numel() ** 0.5)
    assert norm <= most, "%s: error %.3g of %.3g allowed" % (what, norm, most)


def check_moe(out, ref, size, dtype, what=""):
    """Six roundings on the way: the up and gate weights, h, the down weights, each expert's output, the sum.  Independent and of half a step each, they add up to
    sqrt(6) half steps of what is summed; a row of few values may be off by more than the mean, so four."""
    d = out.double().cpu() - ref
    most = 4 * half_step(dtype) * (size + ref.norm(dim=1)) / 2 + 1e-30
    assert bool((d.norm(dim=1) <= most).all()), "%s: %.3g of the bound" % (what, float((d.norm(dim=1) / most).max()))


def check_moe_by_terms(out, a, what=""):
    """As check_moe, for weights whose products cancel: the roundings' shares of the outputs one by one, to first order.

    With zero points far from the codes' middle the values of a group are alike, an output is the difference of few large sums, and an error of half a step of every product can be many
    half steps of it: 260 tokens of bf16, with nothing but the weights rounded to 16 bits in an otherwise exact computation, are 1.76 of check_moe's bound off, and 1.80 with h,
    the experts' outputs and their sum rounded as well.  Each error is at most u of its value and they are independent, so that the mean square of all is at most
    the sum of u^2 times the squares below.  The root is exceeded by a row of few terms by less than twice: a rounding's mean square is u^2 / 6 of its value's, not u^2."""
    x, w, ids, w13, s13, w2, s2, z13, z2 = a
    u, square = half_step(x.dtype), torch.zeros(x.shape[0], dtype=torch.float64)
    ref, _ = w4.moe(*a)
    for i in range(w13.shape[0]):
        t, slot = torch.nonzero(ids == i, as_tuple=True)
        if not len(t):
            continue
        up, down = w4.dequant(w13[i], s13[i], None if z13 is None else z13[i]), w4.dequant(w2[i], s2[i], None if z2 is None else z2[i])
        gate, lin = (x[t].double() @ up.t()).chunk(2, -1)
        d_gate, d_lin = (x[t].double() ** 2 @ (up * up).t()).chunk(2, -1)
        p = torch.sigmoid(gate)
        h = gate * p * lin
        d_h = (p * (1 + gate * (1 - p)) * lin) ** 2 * d_gate + (gate * p) ** 2 * d_lin + h * h
        y, scale = h @ down.t(), w[t, slot].double() ** 2
        square.index_add_(0, t, scale * (((d_h + h * h) @ (down * down).t()).sum(1) + (y * y).sum(1)))
    most = 2 * u * (square + (ref * ref).sum(1)).sqrt() + 1e-30
    d = (out.double().cpu() - ref).norm(dim=1)
    assert bool((d <= most).all()), "%s: %.3g of the bound" % (what, float((d / most).max()))
