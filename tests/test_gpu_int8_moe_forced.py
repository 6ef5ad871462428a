"""The int8 expert layer of a few tokens without a cooperative launch, for GPUs that cannot hold all of one kernel's CTAs at a time:
set_force_kernel(2) takes the grouped GEMMs, with the same bits."""
import pytest
import torch

from test_gpu_int8_moe import make, on_gpu, one_kernel, ops  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("T,E,k,H,I", [(1, 8, 2, 64, 32), (1, 128, 8, 2048, 768), (2, 8, 2, 1344, 1024), (3, 8, 2, 4096, 1024), (5, 6, 3, 1328, 144), (16, 512, 10, 256, 48), (16, 3, 2, 2048, 64)])
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
def test_grouped_on_request(ops, T, E, k, H, I, dt):  # noqa: F811
    assert one_kernel(T, k, H, I)
    a = on_gpu(make(T, E, H, I, dt, T * E + k))
    ref = ops.moe_forward_int8(*a, k)
    assert ops.last_kernel() == "moe_i8"
    ops.set_force_kernel(2)
    try:
        before = ops.launch_count()
        out = ops.moe_forward_int8(*a, k)
        assert ops.last_kernel() == "moe_i8_sum" and ops.launch_count() - before == 6
    finally:
        ops.set_force_kernel(0)
    assert torch.equal(out, ref)
