"""4-bit layers whose activations and scales are at opposite ends of bf16's range, and whose outputs are ordinary."""
import pytest
import torch

import custom_esimd_kernels_vllm as e
from oracle import w4
from test_gpu_w4 import dev, gen, moe_inputs
from w4_util import check_linear, check_moe, weight

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


@pytest.mark.parametrize("M", [1, 5, 8, 16, 40, 300])
@pytest.mark.parametrize("exponent", [-118, -100, -60, 60, 100, 118])
def test_linear(M, exponent):
    """Powers of two alone: x 2^exponent and scales 2^-exponent, which leaves the outputs and the roundings what they were."""
    N, K = 200, 512
    x, (w, s, z) = torch.randn(M, K, generator=gen(M)).to(BF), weight(gen(1), N, K, 64, BF)
    plain = e.linear_w4(*dev(x, w, s, z))
    x, s = (x.double() * 2.0 ** exponent).to(BF), (s.double() * 2.0 ** -exponent).to(BF)
    out = e.linear_w4(*dev(x, w, s, z))
    check_linear(out, x, w, s, z)
    if abs(exponent) <= 100:
        assert torch.equal(out, plain)


@pytest.mark.parametrize("T", [1, 6, 100])
@pytest.mark.parametrize("exponent", [-110, 110])
def test_expert_layer(T, exponent):
    a = list(moe_inputs(T, 8, 2, 256, 128, 64, 32, "bf16"))
    a[0], a[4] = (a[0].double() * 2.0 ** exponent).to(BF), (a[4].double() * 2.0 ** -exponent).to(BF)
    check_moe(e.moe_forward_w4(*dev(*a)), *w4.moe(*a), BF)
