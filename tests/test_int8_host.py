"""Host side of the 8-bit integer operators: what the C entry points refuse before any launch, scratch sizes, and what the sources of their
kernels have to keep to.  No GPU needed."""
import os
import re

import pytest
import torch

from oracle import int8
from test_warp_waits import _per_lane_waits

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "llm-scaler_b200", "csrc")
P = 1 << 20      # an address that nothing reads: every call below is refused before a launch


@pytest.fixture(scope="module")
def L(lib_built):
    from custom_esimd_kernels_vllm import _lib
    return _lib


def refused(L, code, rc):
    assert rc == code
    assert L.launch_count() == refused.before


def test_quantisers_refuse(L):
    refused.before = L.launch_count()
    f = L.lib.b2q_quantize_int8
    refused(L, -1, f(None, 0, 64, P, P, 1, 64, None))
    refused(L, -1, f(P, 0, 64, None, P, 1, 64, None))
    refused(L, -3, f(P, 3, 64, P, P, 1, 64, None))
    refused(L, -2, f(P, 0, 63, P, P, 1, 64, None))
    refused(L, -2, f(P, 0, 64, P, P, 1, 0, None))
    refused(L, -2, f(P, 0, 64, P, P, -1, 64, None))
    refused(L, -4, f(P + 1, 0, 64, P, P, 1, 64, None))
    refused(L, -4, f(P + 2, 2, 64, P, P, 1, 64, None))
    refused(L, -4, f(P, 0, 64, P, P + 2, 1, 64, None))
    refused(L, -10, f(P, 0, 1 << 31, P, P, 1, 1 << 31, None))
    refused(L, 0, f(P, 0, 64, P, P, 0, 64, None))
    g = L.lib.b2q_silu_mul_quantize_int8
    refused(L, -2, g(P, 0, 127, P, P, 1, 64, None))
    refused(L, -3, g(P, 2, 128, P, P, 1, 64, None))
    refused(L, 0, g(P, 0, 128, P, P, 0, 64, None))
    h = L.lib.b2q_resadd_rmsnorm_quantize_int8
    refused(L, -1, h(P, P, None, P, 0, 1e-6, P, P, 1, 64, None))
    refused(L, -3, h(P, P, P, P, 2, 1e-6, P, P, 1, 64, None))
    refused(L, -4, h(P, P + 1, P, P, 0, 1e-6, P, P, 1, 64, None))
    refused(L, 0, h(P, P, P, P, 0, 1e-6, P, P, 0, 64, None))


def linear(L, q=P, ldq=64, s=P, w=P, ws=P, wst=2, b=None, out=P, ot=0, ldo=32, M=4, N=32, K=64):
    return L.lib.b2q_linear_int8(q, ldq, s, w, ws, wst, b, out, ot, ldo, M, N, K, None)


@pytest.mark.parametrize("code,args", [(-1, dict(q=None)), (-1, dict(s=None)), (-1, dict(w=None)), (-1, dict(ws=None)), (-1, dict(out=None)), (-3, dict(ot=2)), (-3, dict(wst=3)),
                                       (-2, dict(K=72, ldq=80)), (-2, dict(K=0)), (-2, dict(ldo=31)), (-2, dict(ldq=48)), (-2, dict(M=-1)), (-4, dict(q=P + 8)), (-4, dict(ldq=72)),
                                       (-4, dict(w=P + 4)), (-4, dict(out=P + 1)), (-4, dict(s=P + 2)), (-4, dict(ws=P + 2)), (-4, dict(b=P + 1)),
                                       (-10, dict(K=131072, ldq=131072)), (-10, dict(M=1 << 31)), (0, dict(M=0)), (0, dict(N=0, ldo=0))])
def test_linear_refuses(L, code, args):
    refused.before = L.launch_count()
    refused(L, code, linear(L, **args))


def test_dynamic_linear_refuses(L):
    refused.before = L.launch_count()
    f = lambda x=P, t=0, ldx=4096, K=4096, M=64, ws=None, wsb=0: L.lib.b2q_linear_int8_dynamic(x, t, ldx, P, P, 2, None, P, 64, M, 64, K, ws, wsb, None)
    need = L.lib.b2q_linear_int8_dynamic_workspace_bytes(64, 64, 4096)
    assert need >= 64 * 4096 + 64 * 4
    refused(L, -1, f(x=None))
    refused(L, -3, f(t=2))
    refused(L, -2, f(ldx=4095))
    refused(L, -4, f(x=P + 1))
    refused(L, -1, f())
    refused(L, -4, f(ws=P + 8, wsb=need))
    refused(L, -8, f(ws=P, wsb=need - 1))
    refused(L, 0, f(M=0))
    # one launch, no scratch
    assert L.lib.b2q_linear_int8_dynamic_workspace_bytes(1, 2048, 2048) == 0
    assert L.lib.b2q_linear_int8_dynamic_workspace_bytes(0, 2048, 2048) == 0
    assert L.lib.b2q_linear_int8_dynamic_workspace_bytes(1, 1 << 20, 2048) > 0


def layer(L, **change):
    a = L.MoeInt8(T=3, E=8, top_k=2, H=64, I=32, act_dtype=0, logits_dtype=2, s13_dtype=2, s2_dtype=2, renormalize=1)
    for i, n in enumerate(("x", "logits", "w13", "s13", "w2", "s2", "out")):
        setattr(a, n, P + (i << 12))
    ws, wsb = change.pop("ws", P), change.pop("wsb", 1 << 30)
    for k, v in change.items():
        setattr(a, k, v)
    return L.lib.b2q_moe_forward_int8(a, ws, wsb, None)


@pytest.mark.parametrize("code,args", [(-1, {n: None}) for n in ("x", "logits", "w13", "s13", "w2", "s2", "out", "ws")] + [(-4, {n: P + 8}) for n in ("x", "w13", "w2", "out", "ws")] + [
    (-4, dict(logits=P + 2)), (-4, dict(s13=P + 2)), (-4, dict(s2=P + 1)), (-3, dict(act_dtype=2)), (-3, dict(logits_dtype=3)), (-3, dict(s13_dtype=-1)), (-3, dict(s2_dtype=5)),
    (-2, dict(top_k=9)), (-2, dict(top_k=0)), (-2, dict(E=0)), (-2, dict(H=72)), (-2, dict(I=40)), (-2, dict(T=-1)), (-10, dict(E=1025)), (-10, dict(E=64, top_k=33)),
    (-10, dict(H=32784)), (-10, dict(I=131072)), (-8, dict(wsb=100)), (0, dict(T=0))])
def test_expert_layer_refuses(L, code, args):
    refused.before = L.launch_count()
    refused(L, code, layer(L, **args))


@pytest.mark.parametrize("T,E,k,H,I", [(1, 8, 2, 64, 32), (16, 128, 8, 2048, 768), (17, 128, 8, 2048, 768), (4096, 128, 8, 2048, 768), (16, 4, 2, 8192, 64)])
def test_expert_layer_scratch(L, T, E, k, H, I):
    """Two buffers of h at least: fp32 and codes; with more tokens also each pair's codes of x and output."""
    rows, got = T * k, L.lib.b2q_moe_forward_int8_workspace_bytes(T, E, k, H, I)
    few = T <= 16 and T * (4 * k * I + H) <= 40960
    least = rows * 5 * I + (0 if few else rows * H * (5 if rows * H <= 1 << 19 else 3))
    assert least <= got <= least + 64 * rows + 300 * E + 8192


def test_no_scratch_for_what_is_refused(L):
    f = L.lib.b2q_moe_forward_int8_workspace_bytes
    assert f(0, 8, 2, 64, 32) == f(4, 0, 2, 64, 32) == f(4, 8, 0, 64, 32) == f(4, 2000, 2, 64, 32) == f(4, 64, 33, 64, 32) == 0


def test_ops_are_registered_and_refuse_cpu_tensors(L):
    import custom_esimd_kernels_vllm as e
    x = torch.zeros(2, 64, dtype=torch.float16)
    for call in (lambda: e.quantize_int8(x), lambda: e.silu_mul_quantize_int8(x), lambda: e.resadd_rmsnorm_quantize_int8(x, x, x[0], 1e-6),
                 lambda: e.linear_int8(x.char(), x[:, 0].float(), x.char(), x[:, 0].float()), lambda: e.linear_int8_dynamic(x, x.char(), x[:, 0].float()),
                 lambda: e.moe_forward_int8(x, x, x.char()[None], x, x.char()[None], x, 1)):
        with pytest.raises((RuntimeError, NotImplementedError)):
            call()


# ------------------------------------------------------------------------------------------------------------- the oracle
def test_oracle_halves_go_to_even_and_rows_that_are_not_finite_are_nan():
    q, t, s = int8.quantize_rows(torch.tensor([[127.0, 0.5, 1.5, -2.5, 63.5], [float("inf"), 1, 2, 3, 4], [0, 0, 0, 0, 0]]))
    assert q.tolist() == [[127, 0, 2, -2, 64], [0] * 5, [0] * 5]
    assert s[0] == 1 and torch.isnan(s[1]) and 0 < s[2] < 1e-13


def test_oracle_layer_of_one_expert_is_two_linears():
    g = torch.Generator().manual_seed(0)
    x = torch.randn(3, 32, generator=g)
    w13, w2 = (torch.randint(-127, 128, s, generator=g, dtype=torch.int8) for s in ((1, 32, 32), (1, 32, 16)))
    s13, s2 = torch.rand(1, 32, generator=g), torch.rand(1, 32, generator=g)
    c, _, s = int8.quantize_rows(x)
    q, _, r = int8.quantize_rows(int8.silu_mul(int8.linear(c, s, w13[0], s13[0])))
    assert torch.equal(int8.moe(x, torch.zeros(3, 1), w13, s13, w2, s2, 1), int8.linear(q, r, w2[0], s2[0]))
    ids, w = int8.route(torch.tensor([[1.0, 2.0, 2.0, 0.0]]), 2)
    assert ids.tolist() == [[1, 2]] and w.tolist() == [[0.5, 0.5]]


# ------------------------------------------------------------------------------------------------------------ the sources
def _source(name):
    with open(os.path.join(CSRC, name)) as f:
        return f.read()


def test_expert_layer_waits_together_and_for_its_copies():
    text = _source("moe_i8.cu")
    assert _per_lane_waits(text) == []
    kernel = text.split("__global__ ")[1]
    # the weights' thread, and the warps that fetch the codes of their own stages
    assert kernel.count("drain_issued(") == 2
    code = re.sub(r"//[^\n]*", "", text)
    # every stage is read by ordinary loads and released behind them
    assert len(re.findall(r"\bmbar_arrive_read\(empty \+", code)) == 2 and not re.search(r"\bmbar_arrive\(empty \+", code)


@pytest.mark.parametrize("name", ["i8_quant.cu", "i8_stream.cu", "moe_i8_many.cu", "i8.cuh"])
def test_kernels_that_start_early_read_their_inputs_by_ordinary_loads(name):
    """No read-only path (__ldg, const __restrict__) but for weights, which nobody writes while requests run."""
    code = re.sub(r"//[^\n]*", "", _source(name))
    assert "__ldg(" not in code and "__restrict__" not in code
    assert len(re.findall(r"ld\.global\.nc", code)) == (1 if name == "i8.cuh" else 0)


def test_status_codes_are_distinct():
    seen = {}
    for f in sorted(os.listdir(CSRC)):
        if f.endswith((".cu", ".cuh")):
            for m in re.finditer(r"\bST_\w+ = (\d+)", _source(f)):
                seen.setdefault(m.group(1), set()).add(f)
    assert all(len(v) == 1 for k, v in seen.items() if k[0] in "89"), seen
