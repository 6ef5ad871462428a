"""What a row's codes and scale depend on: nothing but the row, whatever kernel the number of rows chooses; only the last bits of the norm's scale may
follow the order in which squares add up."""
import pytest
import torch

from gpu_util import DEV
from test_gpu_int8 import ops  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("K", [768, 1024, 2056, 8192, 16384, 28672])
def test_a_row_by_itself_and_among_others(ops, dt, K):  # noqa: F811
    g = torch.Generator().manual_seed(K)
    x, y = (torch.randn(300, K, generator=g).to(dt).to(DEV) for _ in range(2))
    two = torch.cat([x, y], 1)
    w = (1 + 0.2 * torch.randn(K, generator=g)).to(dt).to(DEV)
    plain, silu, norm = ops.quantize_int8(x), ops.silu_mul_quantize_int8(two), ops.resadd_rmsnorm_quantize_int8(x, y, w, 1e-6, torch.empty_like(x))
    for n in (1, 140, 200):
        for many, few in ((plain, ops.quantize_int8(x[:n])), (silu, ops.silu_mul_quantize_int8(two[:n]))):
            assert torch.equal(many[0][:n], few[0]) and torch.equal(many[1][:n], few[1])
        few = ops.resadd_rmsnorm_quantize_int8(x[:n], y[:n].clone(), w, 1e-6)
        assert torch.equal(norm[0][:n], few[0])
        # K squares in any order: sums of at most 1024 threads' 32 each, half of that in the root
        assert ((norm[1][:n].double() - few[1].double()).abs() <= 64 * 2.0 ** -24 * few[1].double()).all()
    odd = torch.empty(300 * K + 1, dtype=dt, device=DEV)[1:].view(300, K).copy_(x)      # element by element
    assert all(torch.equal(a, b) for a, b in zip(plain, ops.quantize_int8(odd)))
