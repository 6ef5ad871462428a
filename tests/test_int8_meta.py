"""Shapes and types of the 8-bit integer operators without data: fake tensors (torch.compile, export) and the meta device.  No GPU needed."""
import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

BF, F16, F32, I8 = torch.bfloat16, torch.float16, torch.float32, torch.int8


def _describe(out):
    out = out if isinstance(out, (tuple, list)) else (out,)
    return [(tuple(t.shape), t.dtype) for t in out]


def _calls(e, new):
    """(operator call, what it returns): empty and odd sizes among them."""
    return [
        (lambda: e.quantize_int8(new((5, 77), F32)), [((5, 77), I8), ((5,), F32)]),
        (lambda: e.quantize_int8(new((0, 64), BF)), [((0, 64), I8), ((0,), F32)]),
        (lambda: e.silu_mul_quantize_int8(new((3, 128), F16)), [((3, 64), I8), ((3,), F32)]),
        (lambda: e.resadd_rmsnorm_quantize_int8(new((4, 48), BF), new((4, 48), BF), new((48,), BF), 1e-6), [((4, 48), I8), ((4,), F32)]),
        (lambda: e.resadd_rmsnorm_quantize_int8(new((4, 48), BF), new((4, 48), BF), new((48,), BF), 1e-6, new((4, 48), BF)), [((4, 48), I8), ((4,), F32)]),
        (lambda: e.linear_int8(new((7, 64), I8), new((7,), F32), new((30, 64), I8), new((30,), F32)), [((7, 30), BF)]),
        (lambda: e.linear_int8(new((7, 64), I8), new((7,), F32), new((30, 64), I8), new((30,), F32), new((30,), F16), F16), [((7, 30), F16)]),
        (lambda: e.linear_int8_dynamic(new((7, 64), F16), new((30, 64), I8), new((30,), BF)), [((7, 30), F16)]),
        (lambda: e.moe_forward_int8(new((6, 64), BF), new((6, 8), F32), new((8, 96, 64), I8), new((8, 96), F32), new((8, 64, 48), I8), new((8, 64), F32), 2), [((6, 64), BF)]),
    ]


@pytest.mark.parametrize("device", ["meta", "fake cuda"])
@pytest.mark.parametrize("i", range(9))
def test_outputs_without_data(lib_built, device, i):
    import custom_esimd_kernels_vllm as e
    if device == "meta":
        call, want = _calls(e, lambda s, dt: torch.empty(s, dtype=dt, device="meta"))[i]
        assert _describe(call()) == want
    else:
        with FakeTensorMode():
            call, want = _calls(e, lambda s, dt: torch.empty(s, dtype=dt, device="cuda"))[i]
            out = call()
            assert _describe(out) == want and all(t.device.type == "cuda" for t in (out if isinstance(out, (tuple, list)) else (out,)))


def test_shapes_that_do_not_fit_are_refused_without_data_too(lib_built):
    import custom_esimd_kernels_vllm as e
    new = lambda s, dt: torch.empty(s, dtype=dt, device="meta")
    for call in (lambda: e.quantize_int8(new((5,), F32)), lambda: e.silu_mul_quantize_int8(new((3, 127), F16)),
                 lambda: e.linear_int8(new((7, 64), I8), new((7,), F32), new((30, 48), I8), new((30,), F32)),
                 lambda: e.linear_int8(new((7, 64), I8), new((7,), F32), new((30, 64), I8), new((30,), F32), None, F32),
                 lambda: e.linear_int8_dynamic(new((7, 64), F32), new((30, 64), I8), new((30,), BF)),
                 lambda: e.moe_forward_int8(new((6, 64), BF), new((5, 8), F32), new((8, 96, 64), I8), new((8, 96), F32), new((8, 64, 48), I8), new((8, 64), F32), 2)):
        with pytest.raises(RuntimeError):
            call()
