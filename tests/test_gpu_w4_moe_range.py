"""The 4-bit expert layer where one expert's weighted output is beyond what 16 bits hold and the sum is not."""
import pytest
import torch

import custom_esimd_kernels_vllm as e
from custom_esimd_kernels_vllm import _lib as L
from oracle import w4
from test_gpu_w4 import dev, moe_inputs
from w4_util import check_moe

pytestmark = pytest.mark.gpu


def large(T, k, dt, zero, seed=0, shape=(256, 160), groups=(64, 32)):
    """The largest expert output is 0.9 of the largest finite value; pairs of slots have the same expert with weights of 3 and -2."""
    H, I = shape
    a = list(moe_inputs(T, 6, k, H, I, *groups, dt, zero, seed))
    a[2][:, 1::2] = a[2][:, 0::2]
    a[1][:, 0::2], a[1][:, 1::2] = 3.0, -2.0
    top = torch.finfo(a[0].dtype).max
    y = max(float(w4.moe(a[0], torch.ones(T, 1), torch.full((T, 1), i), *a[3:])[0].abs().max()) for i in range(6))
    a[6] = (a[6].double() * (0.9 * top / (k // 2) / y)).to(a[0].dtype)
    return a


@pytest.mark.parametrize("T", [1, 5, 40, 300])
@pytest.mark.parametrize("zero", [True, False])
@pytest.mark.parametrize("force", [0, 2])
def test_outputs_beyond_fp16_enter_the_sum(T, zero, force):
    """Whatever the number of tokens: the weighted outputs reach 2.7 times 65504, their sums 0.9 of it."""
    for k, shape, groups in ((2, (256, 160), (64, 32)), (4, (128, 128), (128, 64)), (2, (512, 384), (32, 128))):
        a = large(T, k, "fp16", zero, k, shape, groups)
        ref, size = w4.moe(*a)
        assert float(size.max()) > 65504 > float(ref.abs().max())
        L.set_force_kernel(force)
        try:
            out = e.moe_forward_w4(*dev(*a))
        finally:
            L.set_force_kernel(0)
        assert bool(torch.isfinite(out).all())
        check_moe(out, ref, size, a[0].dtype, "%d tokens, k %d" % (T, k))


@pytest.mark.parametrize("T", [3, 300])
def test_sums_beyond_fp16_are_infinite(T):
    a = large(T, 2, "fp16", True)
    a[1][:, 1] = 0
    ref, _ = w4.moe(*a)
    out = e.moe_forward_w4(*dev(*a)).double().cpu()
    over = ref.abs() > 65520 * (1 + 2.0 ** -6)
    assert bool(over.any()) and bool((out[over] == torch.sign(ref[over]) * float("inf")).all()) and bool(torch.isfinite(out[ref.abs() < 65520 * (1 - 2.0 ** -6)]).all())
