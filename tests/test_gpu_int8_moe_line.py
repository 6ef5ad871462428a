"""The line between the int8 expert layer's two forms has two conditions: little that every CTA has to fetch, and room for a CTA's sums and scales of
all pairs (24 KB each).  A layer that meets the first and not the second goes through grouped GEMMs."""
import pytest
import torch

from oracle import int8
from test_gpu_int8_moe import experts_interval, make, on_gpu, ops  # noqa: F401

pytestmark = pytest.mark.gpu


def one_kernel(T, k, H, I):
    return T <= 16 and T * (4 * k * I + H) <= 40960 and T * k * -(-H // min(H, 148)) * 4 <= 24 * 1024


def check(out, a, k, exact):
    """The interval of a layer's outputs; exact: experts' outputs stay in fp32, which one kernel's always do."""
    x, logits, w13, s13, w2, s2 = a
    ids, w = int8.route(logits, k)
    codes, _, scale = int8.quantize_rows(x)
    lo, hi = torch.zeros(2, *out.shape, dtype=torch.float64)
    for e in ids.unique().tolist():
        t, slot = torch.nonzero(ids == e, as_tuple=True)
        h = int8.silu_mul(int8.linear(codes[t], scale[t], w13[e], s13[e]))
        y = experts_interval(h, w2[e], s2[e], x.dtype, exact)
        slack = 2.0 ** -19 * w[t, slot, None] * torch.maximum(y[0].abs(), y[1].abs())
        lo.index_add_(0, t, w[t, slot, None] * y[0] - slack)
        hi.index_add_(0, t, w[t, slot, None] * y[1] + slack)
    lo, hi, o = lo.to(x.dtype).double(), hi.to(x.dtype).double(), out.cpu().double()
    bad = (o < lo) | (o > hi)
    assert not bad.any(), (int(bad.sum()), bad.numel())
    assert (hi - lo).norm() <= 0.1 * o.norm()


@pytest.mark.parametrize("T,E,k,H,I,fits", [(1, 32, 32, 32768, 16, False), (1, 27, 27, 32768, 16, True), (1, 28, 28, 32768, 16, False), (2, 24, 24, 18368, 16, True), (2, 26, 26, 18368, 16, False),
                                            (2, 20, 20, 11264, 32, True)])
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
def test_layers_of_many_pairs_and_wide_rows(ops, T, E, k, H, I, fits, dt):  # noqa: F811
    assert T * (4 * k * I + H) <= 40960 and one_kernel(T, k, H, I) == fits
    a = make(T, E, H, I, dt, T + k)
    before = ops.launch_count()
    out = ops.moe_forward_int8(*on_gpu(a), k)
    assert (ops.last_kernel() == "moe_i8") == fits and ops.launch_count() - before == (1 if fits else 6)
    check(out, a, k, fits or T * k * H <= 1 << 19)
