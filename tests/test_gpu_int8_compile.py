"""The 8-bit integer operators under torch.compile's tracing (no code generation), and torch's own check of their schemas and fake implementations."""
import pytest
import torch

from gpu_util import DEV
from test_gpu_int8 import ops  # noqa: F401
from test_gpu_int8_moe import make, on_gpu

pytestmark = pytest.mark.gpu


def _weights(n, k, seed):
    g = torch.Generator().manual_seed(seed)
    return torch.randint(-127, 128, (n, k), generator=g, dtype=torch.int8).to(DEV), (torch.rand(n, generator=g) * 1e-2 + 1e-3).to(DEV)


def test_schemas_and_fake_implementations(ops):  # noqa: F811
    n = torch.ops.b2q_int8
    x, y = (torch.randn(6, 128, device=DEV).bfloat16() for _ in range(2))
    w, ws = _weights(48, 128, 0)
    q, s = ops.quantize_int8(x)
    a = on_gpu(make(6, 8, 128, 64, torch.bfloat16, 1))
    tests = ("test_schema", "test_faketensor")
    for op, args in [(n.quantize, (x,)), (n.silu_mul_quantize, (x,)), (n.resadd_rmsnorm_quantize, (x, y, x[0].clone(), 1e-6, torch.empty_like(x))),
                     (n.linear, (q, s, w, ws, None, torch.float16)), (n.linear_dynamic, (x, w, ws, ws[:48].bfloat16())), (n.moe_forward, (*a, 2, True))]:
        torch.library.opcheck(op.default, args, test_utils=tests)


@pytest.mark.parametrize("dynamic", [False, True])
def test_a_traced_layer_equals_an_eager_one(ops, dynamic):  # noqa: F811
    w1, s1 = _weights(512, 256, 1)
    w2, s2 = _weights(256, 256, 2)
    norm = torch.ones(256, dtype=torch.bfloat16, device=DEV)
    experts = on_gpu(make(1, 8, 256, 64, torch.bfloat16, 3))[2:]

    def layer(x, residual, logits):
        gate_up = ops.linear_int8(*ops.resadd_rmsnorm_quantize_int8(x, residual, norm, 1e-6), w1, s1)
        x = ops.linear_int8(*ops.silu_mul_quantize_int8(gate_up), w2, s2)
        return ops.moe_forward_int8(x, logits, *experts, 2) + ops.linear_int8_dynamic(x, w2, s2)

    torch._dynamo.reset()
    traced = torch.compile(layer, backend="aot_eager", fullgraph=True, dynamic=dynamic)
    for M in (3, 40, 7):
        x, r, l = torch.randn(M, 256, device=DEV).bfloat16(), torch.randn(M, 256, device=DEV).bfloat16(), torch.randn(M, 8, device=DEV)
        ra, rb = r.clone(), r.clone()
        want, got = layer(x, ra, l), traced(x, rb, l)
        assert torch.equal(want, got) and torch.equal(ra, rb) and not torch.equal(ra, r)
