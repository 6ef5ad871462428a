"""Int8 expert layers of more than 2^19 expert outputs, each held in 16 bits in front of the weighted sum: an output that 16 bits cannot hold still
enters the sum with its value, as it does in smaller calls."""
import pytest
import torch

from oracle import int8
from test_gpu_int8_moe import experts_interval, make, on_gpu, ops  # noqa: F401

pytestmark = pytest.mark.gpu


def held(v, dt):
    """As a 16-bit number, or as it is where that would be infinite."""
    r = v.to(dt).double()
    return torch.where(torch.isinf(r), v, r)


@pytest.mark.parametrize("T,E,k,H,I", [(600, 8, 2, 512, 64), (65, 16, 8, 1024, 272), (2100, 4, 4, 64, 48)])
@pytest.mark.parametrize("sdt", [torch.float32, torch.bfloat16])
def test_an_output_beyond_fp16_does_not_make_the_sum_infinite(ops, T, E, k, H, I, sdt):  # noqa: F811
    assert T * k * H > 1 << 19
    x, logits, w13, s13, w2, s2 = make(T, E, H, I, torch.float16, T, sdt)
    logits = logits / 4
    ids, w = int8.route(logits, k)
    codes, _, scale = int8.quantize_rows(x)
    pairs = [(e, *torch.nonzero(ids == e, as_tuple=True)) for e in range(E)]
    h = [int8.silu_mul(int8.linear(codes[t], scale[t], w13[e], s13[e])) for e, t, _ in pairs]
    # experts' scales that put the largest outputs at four times the largest fp16 number
    y = [int8.linear(*(lambda q, _, r: (q, r))(*int8.quantize_rows(h[e])), w2[e], s2[e]) for e, _, _ in pairs]
    s2 = (s2.float() * (4 * 65504 / max(v.abs().max().item() for v in y))).to(sdt)
    lo, hi = torch.zeros(2, T, H, dtype=torch.float64)
    beyond = torch.zeros(T, H, dtype=torch.bool)
    for e, t, slot in pairs:
        a, b = experts_interval(h[e], w2[e], s2[e], torch.float16, True)
        beyond[t] |= (a > 65520) | (b < -65520)
        a, b = held(a, torch.float16), held(b, torch.float16)
        slack = 2.0 ** -19 * w[t, slot, None] * torch.maximum(a.abs(), b.abs())
        lo.index_add_(0, t, w[t, slot, None] * a - slack)
        hi.index_add_(0, t, w[t, slot, None] * b + slack)
    lo, hi = lo.half().double(), hi.half().double()
    fits = beyond & torch.isfinite(lo) & torch.isfinite(hi)
    assert fits.sum() > 20
    o = ops.moe_forward_int8(*on_gpu((x, logits, w13, s13, w2, s2)), k).cpu().double()
    bad = (o < lo) | (o > hi) | torch.isnan(o)
    assert not bad.any(), (int(bad.sum()), int((bad & beyond).sum()), bad.numel())


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
def test_tokens_that_are_not_finite_stay_so(ops, dt):  # noqa: F811
    T, k, H = 600, 2, 512
    a = list(make(T, 8, H, 64, dt, 5))
    good = ops.moe_forward_int8(*on_gpu(a), k)
    a[0][7, 3], a[0][300, 0] = float("inf"), float("nan")
    out = ops.moe_forward_int8(*on_gpu(a), k)
    assert torch.isnan(out[[7, 300]]).all()
    keep = [i for i in range(T) if i not in (7, 300)]
    assert torch.equal(out[keep], good[keep])
    # a scale that is infinite makes its column infinite, or NaN, and no other
    a = list(make(T, 8, H, 64, dt, 5))
    a[5][:, 9] = float("inf")
    out = ops.moe_forward_int8(*on_gpu(a), k)
    assert not torch.isfinite(out[:, 9]).any()
    keep = [i for i in range(H) if i != 9]
    assert torch.equal(out[:, keep], good[:, keep])
