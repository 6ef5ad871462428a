"""Outputs without data of expert routing and the 4-bit layers: a call that the operators refuse for its types or sizes is refused while it is traced.  No GPU needed."""
import pytest
import torch

BF, F16, F32, F64, U8, I8, I32, I64 = torch.bfloat16, torch.float16, torch.float32, torch.float64, torch.uint8, torch.int8, torch.int32, torch.int64
LINEAR = dict(x=((5, 256), BF), weight=((30, 128), U8), scale=((4, 30), BF), zero=((4, 30), U8), bias=((30,), BF))
MOE = dict(x=((6, 128), F16), topk_weights=((6, 2), F32), topk_ids=((6, 2), I32), gate_up_weight=((8, 128, 64), U8), gate_up_scale=((8, 2, 128), F16), down_weight=((8, 128, 32), U8),
           down_scale=((8, 2, 128), F16), gate_up_zero=((8, 2, 128), U8), down_zero=((8, 2, 128), U8))


@pytest.fixture(scope="module")
def e(lib_built):
    import custom_esimd_kernels_vllm
    return custom_esimd_kernels_vllm


def call(f, arguments, **changed):
    return f(**{n: torch.empty(v[0], dtype=v[1], device="meta") if isinstance(v, tuple) else v for n, v in {**arguments, **changed}.items() if v is not None})


def test_calls_that_are_taken(e):
    assert call(e.linear_w4, LINEAR).shape == (5, 30) and call(e.linear_w4, LINEAR, weight=((30, 32), I32), zero=None, bias=None).shape == (5, 30)
    assert call(e.moe_forward_w4, MOE).shape == (6, 128) and call(e.moe_forward_w4, MOE, gate_up_zero=None, down_weight=((8, 128, 8), I32)).shape == (6, 128)


@pytest.mark.parametrize("changed", [dict(x=((5,), BF)), dict(x=((5, 256), F32)), dict(x=((5, 128), BF)), dict(weight=((30, 128), I8)), dict(weight=((1, 30, 128), U8)), dict(weight=((31, 128), U8)),
                                     dict(weight=((30, 0), U8)), dict(scale=((4, 30), F16)), dict(scale=((4, 31), BF)), dict(scale=((0, 30), BF)), dict(scale=((3, 30), BF)), dict(scale=((16, 30), BF)),
                                     dict(scale=((1, 30), BF)), dict(scale=((30,), BF)), dict(zero=((4, 30), I8)), dict(zero=((2, 30), U8)), dict(zero=((120,), U8)), dict(bias=((31,), BF)),
                                     dict(bias=((1, 30), BF)), dict(bias=((30,), F32))])
def test_linears_that_are_refused(e, changed):
    with pytest.raises(RuntimeError):
        call(e.linear_w4, LINEAR, **changed)


@pytest.mark.parametrize("changed", [dict(x=((6, 128), F32)), dict(x=((6, 256), F16)), dict(x=((5, 128), F16)), dict(x=((6, 128), BF)), dict(topk_ids=((6, 2), I64)), dict(topk_ids=((5, 2), I32)),
                                     dict(topk_ids=((6, 3), I32)), dict(topk_ids=((6, 0), I32), topk_weights=((6, 0), F32)), dict(topk_ids=((12,), I32)), dict(topk_weights=((6, 2), F16)),
                                     dict(topk_weights=((6, 1), F32)), dict(topk_weights=((5, 2), F32)), dict(gate_up_weight=((128, 64), U8)), dict(gate_up_weight=((7, 128, 64), U8)),
                                     dict(gate_up_weight=((8, 126, 64), U8)), dict(gate_up_weight=((8, 128, 32), U8)), dict(gate_up_weight=((8, 128, 64), F16)), dict(gate_up_scale=((7, 2, 128), F16)),
                                     dict(gate_up_scale=((8, 3, 128), F16)), dict(gate_up_scale=((8, 8, 128), F16), gate_up_zero=None), dict(gate_up_scale=((8, 2, 128), BF)), dict(down_weight=((8, 128, 64), U8)),
                                     dict(down_weight=((8, 64, 32), U8)), dict(down_weight=((7, 128, 32), U8)), dict(down_scale=((8, 2, 64), F16)), dict(down_scale=((8, 4, 128), F16), down_zero=None),
                                     dict(down_scale=((2, 128), F16)), dict(gate_up_zero=((8, 2, 128), F16)), dict(gate_up_zero=((8, 1, 128), U8)), dict(down_zero=((2, 128), U8))])
def test_expert_layers_that_are_refused(e, changed):
    with pytest.raises(RuntimeError):
        call(e.moe_forward_w4, MOE, **changed)


@pytest.mark.parametrize("changed", [dict(top_k=0), dict(top_k=9), dict(top_k=5), dict(num_groups=0), dict(num_groups=3), dict(num_groups=-2), dict(top_groups=0), dict(top_groups=5),
                                     dict(bias=((7,), F32)), dict(bias=((1, 8), F32)), dict(bias=((8,), F64)), dict(logits=((4, 0), F32)), dict(logits=((8,), F32)), dict(logits=((4, 8), F64))])
def test_routes_that_are_refused(e, changed):
    arguments = dict(logits=((4, 8), F32), top_k=4, num_groups=4, top_groups=2, bias=((8,), BF))
    assert call(e.route_experts, arguments)[0].shape == (4, 4)
    with pytest.raises(RuntimeError):
        call(e.route_experts, arguments, **changed)
