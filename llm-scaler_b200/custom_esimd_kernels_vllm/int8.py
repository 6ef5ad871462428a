"""8-bit integer operators: int8 weights with one scale per output channel, activations quantised to int8 with one scale per token.

The reference has no such format, so these have names of their own and the torch namespace `b2q_int8` (csrc/torch_int8.cpp ->
libb2q_int8.so, over the C ABI of include/b2q.h).  All of them run on torch's current stream and may be captured in a CUDA graph.
"""
import os

import torch

from . import _lib as L

_PATH = os.path.join(os.path.dirname(os.path.abspath(__file__)), "libb2q_int8.so")
_MISSING = None if os.path.exists(_PATH) else "b2q: %s is missing; build it with `python llm-scaler_b200/build.py`" % _PATH
_CHECK_STATUS = os.environ.get("B2Q_CHECK_STATUS") == "1"
if _MISSING and os.environ.get("B2Q_PYTHON_DISPATCH") != "1" and not _CHECK_STATUS:
    raise ImportError(_MISSING)      # under these two the other ops do without a C++ layer, so that only the operators here fail
if not _MISSING:
    torch.ops.load_library(_PATH)


def _fakes():
    """Outputs without data, for tracing: the sizes are checked as the ops check them, pointers and strides are not."""
    fake, check, f32 = torch.library.register_fake, torch._check, torch.float32
    half = (torch.bfloat16, torch.float16)

    def codes(x, columns):
        return x.new_empty((x.shape[0], columns), dtype=torch.int8), x.new_empty((x.shape[0],), dtype=f32)

    @fake("b2q_int8::quantize")
    def _(x):
        check(x.dim() == 2 and x.dtype in half + (f32,), lambda: "x must be 2-D bf16, fp16 or fp32")
        return codes(x, x.shape[1])

    @fake("b2q_int8::silu_mul_quantize")
    def _(gate_up):
        check(gate_up.dim() == 2 and gate_up.dtype in half and gate_up.shape[1] % 2 == 0, lambda: "gate_up must be 2-D bf16 or fp16 with an even number of columns")
        return codes(gate_up, gate_up.shape[1] // 2)

    @fake("b2q_int8::resadd_rmsnorm_quantize")
    def _(hidden, residual, norm_weight, eps, residual_out):
        check(hidden.dim() == 2 and hidden.dtype in half and residual.shape == hidden.shape, lambda: "hidden and residual must be 2-D bf16 / fp16 of the same shape")
        check(norm_weight.dim() == 1 and norm_weight.shape[0] == hidden.shape[1], lambda: "norm_weight must have K elements")
        return codes(hidden, hidden.shape[1])

    def linear(x, weight, weight_scale, dtype):
        check(x.dim() == 2 and weight.dim() == 2 and weight.dtype == torch.int8 and weight.shape[1] == x.shape[1], lambda: "weight must be int8 [N, K]")
        check(weight_scale.numel() == weight.shape[0], lambda: "weight_scale must have N elements")
        check(dtype in half, lambda: "outputs are bf16 or fp16")
        return x.new_empty((x.shape[0], weight.shape[0]), dtype=dtype)

    @fake("b2q_int8::linear")
    def _(codes, scale, weight, weight_scale, bias, out_dtype):
        check(codes.dtype == torch.int8 and scale.numel() == codes.shape[0], lambda: "codes must be int8 and scale have M elements")
        return linear(codes, weight, weight_scale, out_dtype)

    @fake("b2q_int8::linear_dynamic")
    def _(x, weight, weight_scale, bias):
        return linear(x, weight, weight_scale, x.dtype)

    @fake("b2q_int8::moe_forward")
    def _(x, router_logits, gate_up_weight, gate_up_scale, down_weight, down_scale, top_k, renormalize):
        check(x.dim() == 2 and x.dtype in half, lambda: "x must be a bf16 / fp16 [T, H] tensor")
        check(router_logits.dim() == 2 and router_logits.shape[0] == x.shape[0], lambda: "router_logits must be a [T, E] tensor")
        check(down_weight.dim() == 3 and down_weight.shape[1] == x.shape[1], lambda: "down_weight must be an int8 [E, H, I] tensor")
        return x.new_empty(x.shape)


if not _MISSING:
    _fakes()


class _Ops:
    """The ops' only overloads, looked up once: a call is worth a few microseconds."""

    def __init__(self):
        for name in ("quantize", "silu_mul_quantize", "resadd_rmsnorm_quantize", "linear", "linear_dynamic", "moe_forward"):
            setattr(self, name, getattr(torch.ops.b2q_int8, name).default)


class _NoOps:
    def __getattr__(self, name):
        raise ImportError(_MISSING)


_ops = _NoOps() if _MISSING else _Ops()

if _CHECK_STATUS and not _MISSING:
    # debugging, as for the other ops: every call synchronises and raises if a bounded device-side wait has expired
    class _Checked:
        def __getattr__(self, name):
            op = getattr(torch.ops.b2q_int8, name)

            def run(*args):
                out = op(*args)
                code = L.device_status()
                if code:
                    raise RuntimeError("b2q: b2q_int8::%s: a bounded device-side wait expired (code %d); results are not valid" % (name, code))
                return out
            return run

    _ops = _Checked()


def quantize_int8(x):
    """Rows of x (bf16, fp16 or fp32 [M, K], rows contiguous) -> codes int8 [M, K], scale fp32 [M].

    scale = max(amax, 1e-12) / 127, codes = rint(127 x / amax), halves to even, decided exactly.  A row with an infinity or a NaN gets
    the scale NaN and zero codes.  Tokens, or at load time the rows of a weight."""
    return _ops.quantize(x)


def silu_mul_quantize_int8(gate_up):
    """quantize_int8 of silu(gate) * up, gate_up bf16 / fp16 [M, 2K]; the product is not rounded to 16 bits in between.  Its codes are within half a
    step and the product's own fp32 error."""
    return _ops.silu_mul_quantize(gate_up)


def resadd_rmsnorm_quantize_int8(hidden, residual, norm_weight, eps, residual_out=None):
    """v = hidden + residual; residual_out (residual itself by default) <- v; returns quantize_int8 of rmsnorm(v) * norm_weight, with codes within half a
    step and the fp32 error.  The last bits of a scale may depend on the number of rows."""
    return _ops.resadd_rmsnorm_quantize(hidden, residual, norm_weight, eps, residual_out)


def linear_int8(codes, scale, weight, weight_scale, bias=None, out_dtype=torch.bfloat16):
    """out[m, n] = scale[m] * weight_scale[n] * (codes[m] . weight[n]) (+ bias[n]); codes int8 [M, K], weight int8 [N, K], K % 16 == 0."""
    return _ops.linear(codes, scale, weight, weight_scale, bias, out_dtype)


def linear_int8_dynamic(x, weight, weight_scale, bias=None):
    """linear_int8(*quantize_int8(x), ...) in x's type; for a few tokens one launch."""
    return _ops.linear_dynamic(x, weight, weight_scale, bias)


def moe_forward_int8(x, router_logits, gate_up_weight, gate_up_scale, down_weight, down_scale, top_k, renormalize=True):
    """A whole expert layer: top_k of router_logits [T, E], silu(x W_gate) * (x W_up), down projection, weighted sum -> [T, H] in x's type.

    gate_up_weight int8 [E, 2I, H] (gate rows, then up), gate_up_scale [E, 2I], down_weight int8 [E, H, I], down_scale [E, H]; x and the
    intermediate rows are quantised to int8 per row.  Weights of the chosen experts are their softmax, renormalised over the chosen or
    not.  A few tokens take one kernel."""
    return _ops.moe_forward(x, router_logits, gate_up_weight, gate_up_scale, down_weight, down_scale, top_k, renormalize)
