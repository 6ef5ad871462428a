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
