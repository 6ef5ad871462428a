"""One-kernel int8 expert layers whose CTAs own nine to fifteen rows of the down matrices: a stage of the ring holds just those rows, and no lane reads
a sixteenth (tests/test_int8_moe_sizes.py has the sizes)."""
import pytest
import torch

from test_gpu_int8_moe import check, make, on_gpu, one_kernel, ops  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("T,E,k,H,I", [(1, 8, 2, 1280, 2048), (1, 8, 4, 1408, 2048), (2, 8, 2, 1344, 1024), (3, 8, 1, 1504, 1024), (3, 8, 2, 1200, 512), (2, 4, 2, 1760, 688),
                                       (1, 6, 1, 1936, 1776), (2, 40, 4, 2080, 320), (1, 4, 2, 2208, 64), (5, 6, 3, 1328, 144)])
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
def test_nine_to_fifteen_rows(ops, T, E, k, H, I, dt):  # noqa: F811
    a = make(T, E, H, I, dt, T * E + k)
    assert one_kernel(T, k, H, I) and 9 <= -(-H // 148) <= 15
    g = on_gpu(a)
    for _ in range(3):
        out = ops.moe_forward_int8(*g, k)
        assert ops.last_kernel() == "moe_i8"
    check(out, a, k)
