"""Expert routing, and layers of 4-bit weights with a scale and a zero point per group of 32, 64 or 128 values along k (GPTQ and AWQ checkpoints).

The reference has group 128 without zero points and the softmax top-k alone, so these have names of their own and the torch namespace `b2q_w4`
(csrc/torch_w4.cpp -> libb2q_w4.so, over the C ABI of include/b2q.h).  All of them run on torch's current stream and may be captured in a CUDA
graph.
"""
import os

import torch

from . import _lib as L

_PATH = os.path.join(os.path.dirname(os.path.abspath(__file__)), "libb2q_w4.so")
_MISSING = None if os.path.exists(_PATH) else "b2q: %s is missing; build it with `python llm-scaler_b200/build.py`" % _PATH
_CHECK_STATUS = os.environ.get("B2Q_CHECK_STATUS") == "1"
if _MISSING and os.environ.get("B2Q_PYTHON_DISPATCH") != "1" and not _CHECK_STATUS:
    raise ImportError(_MISSING)      # under these two the other ops do without a C++ layer, so that only the operators here fail
if not _MISSING:
    torch.ops.load_library(_PATH)


def _fakes():
    """Outputs without data, for tracing: types and sizes are checked as csrc/torch_w4.cpp checks them; pointers, strides and the C functions' limits are not."""
    fake, check = torch.library.register_fake, torch._check
    half = (torch.bfloat16, torch.float16)

    def refuse(condition, message):
        check(condition, lambda: message)

    def weight(name, x, w, s, z, experts=()):
        """(N, K) of a weight, [N, K / 2] behind `experts`."""
        d = len(experts)
        refuse(w.dtype in (torch.uint8, torch.int32), name + " weight must be uint8 (two codes to a byte) or int32 (eight)")
        refuse(w.dim() == 2 + d and s.dim() == 2 + d, name + " weight must be [.., N, K / 2] (int32: K / 8), its scale [.., K / group, N]")
        N, K, groups = w.shape[d], w.shape[d + 1] * (2 if w.dtype == torch.uint8 else 8), s.shape[d]
        refuse(s.dtype == x.dtype, name + " scale must have the activations' type")
        refuse(s.shape[d + 1] == N, name + " scale must be [.., K / group, N]")
        refuse(groups > 0, name + " scale has no groups")
        refuse(K > 0 and K % groups == 0, name + " scale has a number of groups that does not divide K")
        refuse(K // groups in (32, 64, 128), name + " groups must have 32, 64 or 128 values")
        if experts:
            refuse(w.shape[0] == experts[0] and s.shape[0] == experts[0], name + " weight and scale must have the same number of experts")
        if z is not None:
            refuse(z.dtype == torch.uint8 and z.dim() == s.dim() and all(i == j for i, j in zip(z.shape, s.shape)), name + " zero must be uint8 of the scale's shape")
        return N, K

    @fake("b2q_w4::route_experts")
    def _(logits, top_k, scoring, bias, num_groups, top_groups, group_score, renormalize, scale):
        refuse(logits.dim() == 2 and logits.dtype in half + (torch.float32,), "logits must be 2-D bf16, fp16 or fp32")
        T, E = logits.shape
        refuse(scoring in (0, 1) and group_score in (0, 1), "scoring must be 0 (softmax) or 1 (sigmoid), group_score 0 (max) or 1 (top2)")
        refuse(num_groups > 0, "num_groups must divide the number of experts")
        refuse(E > 0 and E % num_groups == 0, "num_groups must divide the number of experts")
        refuse(0 < top_groups and top_groups <= num_groups, "top_groups must be between 1 and num_groups")
        refuse(0 < top_k and top_k <= E // num_groups * top_groups, "top_k must be between 1 and the number of experts in top_groups groups")
        if bias is not None:
            refuse(bias.dim() == 1 and bias.shape[0] == E and bias.dtype in half + (torch.float32,), "bias must be a bf16, fp16 or fp32 [E] tensor")
        return logits.new_empty((T, top_k), dtype=torch.float32), logits.new_empty((T, top_k), dtype=torch.int32)

    @fake("b2q_w4::linear")
    def _(x, w, scale, zero, bias):
        refuse(x.dim() == 2 and x.dtype in half, "x must be 2-D bf16 or fp16")
        N, K = weight("the", x, w, scale, zero)
        refuse(x.shape[1] == K, "weight has another K than x")
        if bias is not None:
            refuse(bias.dim() == 1 and bias.shape[0] == N and bias.dtype == x.dtype, "bias must be an [N] tensor of x's type")
        return x.new_empty((x.shape[0], N))

    @fake("b2q_w4::moe_forward")
    def _(x, topk_weights, topk_ids, gate_up_weight, gate_up_scale, down_weight, down_scale, gate_up_zero, down_zero):
        refuse(x.dim() == 2 and x.dtype in half, "x must be a bf16 / fp16 [T, H] tensor")
        refuse(topk_ids.dim() == 2 and topk_ids.shape[0] == x.shape[0] and topk_ids.shape[1] > 0 and topk_ids.dtype == torch.int32, "topk_ids must be an int32 [T, top_k] tensor")
        refuse(topk_weights.dim() == 2 and topk_weights.shape[0] == topk_ids.shape[0] and topk_weights.shape[1] == topk_ids.shape[1] and topk_weights.dtype == torch.float32,
               "topk_weights must be an fp32 tensor of the shape of topk_ids")
        refuse(gate_up_weight.dim() == 3 and gate_up_weight.shape[0] > 0, "the gate_up weight must be of [E, 2I, H], with experts")
        E, H = gate_up_weight.shape[0], x.shape[1]
        two_i, k_up = weight("the gate_up", x, gate_up_weight, gate_up_scale, gate_up_zero, (E,))
        n_down, k_down = weight("the down", x, down_weight, down_scale, down_zero, (E,))
        refuse(k_up == H and two_i % 2 == 0, "the gate_up weight must be of [E, 2I, H]")
        refuse(n_down == H and 2 * k_down == two_i, "the down weight must be of [E, H, I]")
        return x.new_empty(x.shape)


class _Ops:
    """The ops' only overloads, looked up once: a call is worth a few microseconds."""

    def __init__(self):
        for name in ("route_experts", "linear", "moe_forward"):
            setattr(self, name, getattr(torch.ops.b2q_w4, name).default)


class _NoOps:
    def __getattr__(self, name):
        raise ImportError(_MISSING)


class _Checked:
    """Debugging, as for the other ops: every call synchronises and raises if a bounded device-side wait has expired."""

    def __getattr__(self, name):
        op = getattr(torch.ops.b2q_w4, name)

        def run(*args):
            out = op(*args)
            code = L.device_status()
            if code:
                raise RuntimeError("b2q: b2q_w4::%s: a bounded device-side wait expired (code %d); results are not valid" % (name, code))
            return out
        return run


if _MISSING:
    _ops = _NoOps()
else:
    _fakes()
    _ops = _Checked() if _CHECK_STATUS else _Ops()


_SCORING, _GROUP_SCORE = {"softmax": 0, "sigmoid": 1}, {"max": 0, "top2": 1}      # B2Q_SCORE_*, B2Q_GROUP_*


def route_experts(logits, top_k, scoring="softmax", bias=None, num_groups=1, top_groups=1, group_score="max", renormalize=True, scale=1.0):
    """Router logits [T, E] -> weights fp32 [T, top_k], ids int32 [T, top_k], the best expert first, the lowest index first among equals.

    Scores are the softmax or the sigmoid of the logits; `bias` [E] is added to them for the choice only.  With num_groups > 1 only the experts of the
    top_groups best groups can be chosen; a group counts by its best expert ("max") or the sum of its two best ("top2").  Weights are the chosen scores,
    divided by their sum if `renormalize`, times `scale`.  Choices are exact.  Where no expert is left (masked by -inf, or the token's logits hold a
    NaN or +inf) the id is -1 and the weight 0."""
    try:
        return _ops.route_experts(logits, top_k, _SCORING[scoring], bias, num_groups, top_groups, _GROUP_SCORE[group_score], renormalize, scale)
    except KeyError as unknown:
        raise RuntimeError("b2q: scoring is \"softmax\" or \"sigmoid\" and group_score \"max\" or \"top2\", not %s" % unknown) from None


def linear_w4(x, weight, scale, zero=None, bias=None):
    """x [M, K] (bf16 or fp16, rows contiguous) times a 4-bit weight -> [M, N] in x's type: out = x @ ((q - zero) * scale).T (+ bias).

    weight: codes q, uint8 [N, K / 2] with the even k in the low half of a byte, or int32 [N, K / 8], lowest nibble first; scale [K / group, N] in x's type,
    group 32, 64 or 128; zero uint8 [K / group, N], 8 everywhere if None; bias [N] in x's type."""
    return _ops.linear(x, weight, scale, zero, bias)


def moe_forward_w4(x, topk_weights, topk_ids, gate_up_weight, gate_up_scale, down_weight, down_scale, gate_up_zero=None, down_zero=None):
    """A whole expert layer for given routes (route_experts' outputs): silu(x W_gate) * (x W_up), down projection, weighted sum -> [T, H] in x's type.

    gate_up_weight of [E, 2I, H] (gate rows, then up) and down_weight of [E, H, I] in linear_w4's forms, scales and zeros [E, groups, rows].  ids
    outside [0, E) contribute nothing."""
    return _ops.moe_forward(x, topk_weights, topk_ids, gate_up_weight, gate_up_scale, down_weight, down_scale, gate_up_zero, down_zero)
