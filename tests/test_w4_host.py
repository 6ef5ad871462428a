"""Host side of expert routing and the layers of 4-bit group-quantised weights: what the C entry points refuse before any launch, scratch sizes, outputs
without data, the package without their library, and the oracle.  No GPU needed."""
import math
import os
import shutil
import subprocess
import sys

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

from oracle import w4

PKG = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "llm-scaler_b200", "custom_esimd_kernels_vllm")
P = 1 << 20      # an address that nothing reads: every call below is refused before a launch
BF, F16, F32, U8, I32 = torch.bfloat16, torch.float16, torch.float32, torch.uint8, torch.int32


@pytest.fixture(scope="module")
def L(lib_built):
    from custom_esimd_kernels_vllm import _lib
    return _lib


def route(L, logits=P, lt=2, ldl=64, bias=None, bt=2, w=P, ids=P, T=3, E=64, k=4, scoring=0, groups=1, top=1, score=0, renorm=1, scale=1.0):
    return L.lib.b2q_route_experts(logits, lt, ldl, bias, bt, w, ids, T, E, k, scoring, groups, top, score, renorm, scale, None)


@pytest.mark.parametrize("code,args", [(-1, dict(logits=None)), (-1, dict(w=None)), (-1, dict(ids=None)), (-3, dict(lt=3)), (-3, dict(lt=-1)), (-3, dict(bias=P, bt=7)), (-5, dict(scoring=2)),
                                       (-5, dict(score=-1)), (-2, dict(T=-1)), (-2, dict(E=0)), (-2, dict(k=0)), (-2, dict(ldl=63)), (-2, dict(E=16, k=17)), (-2, dict(groups=0)),
                                       (-2, dict(groups=7)), (-2, dict(groups=8, top=9)), (-2, dict(groups=8, top=0)), (-2, dict(groups=32, top=2, k=5)), (-10, dict(E=1025, ldl=1025)),
                                       (-10, dict(k=33)), (-10, dict(groups=64, top=64)), (-10, dict(T=1 << 31)), (-4, dict(logits=P + 2)), (-4, dict(logits=P + 1, lt=0)),
                                       (-4, dict(bias=P + 1, bt=1)), (-4, dict(bias=P + 2)), (-4, dict(w=P + 2)), (-4, dict(ids=P + 1)), (0, dict(T=0))])
def test_routing_refuses(L, code, args):
    before = L.launch_count()
    assert route(L, **args) == code and L.launch_count() == before


def linear(L, x=P, t=0, ldx=256, w=P, s=P, z=P, b=P, out=P, ldo=32, M=4, N=32, K=256, G=64, ws=P, wsb=1 << 30):
    return L.lib.b2q_linear_w4(x, t, ldx, w, s, z, b, out, ldo, M, N, K, G, ws, wsb, None)


@pytest.mark.parametrize("code,args", [(-1, dict(x=None)), (-1, dict(w=None)), (-1, dict(s=None)), (-1, dict(out=None)), (-1, dict(M=200, K=4096, ldx=4097, ws=None)), (-3, dict(t=2)),
                                       (-2, dict(M=-1)), (-2, dict(N=-1)), (-2, dict(K=0)), (-2, dict(G=16)), (-2, dict(G=256)), (-2, dict(G=0)), (-2, dict(K=96)), (-2, dict(ldx=255)),
                                       (-2, dict(ldo=31)), (-10, dict(M=1 << 31)), (-10, dict(N=1 << 31, ldo=1 << 31)), (-10, dict(K=1 << 21, ldx=1 << 21)),
                                       (-10, dict(N=1 << 20, ldo=1 << 20, K=1 << 18, ldx=1 << 18, G=32)), (-4, dict(x=P + 1)), (-4, dict(w=P + 8)), (-4, dict(s=P + 1)), (-4, dict(b=P + 1)),
                                       (-4, dict(out=P + 1)), (-4, dict(M=200, ldx=257, ws=P + 128)), (-8, dict(M=200, ldx=257, wsb=100)), (0, dict(M=0)), (0, dict(N=0, ldo=0))])
def test_linear_refuses(L, code, args):
    before = L.launch_count()
    assert linear(L, **args) == code and L.launch_count() == before


def layer(L, **change):
    a = L.MoeW4(T=3, E=8, top_k=2, H=128, I=64, group13=64, group2=32, act_dtype=0)
    for i, n in enumerate(("x", "weights", "ids", "w13", "s13", "z13", "w2", "s2", "z2", "out")):
        setattr(a, n, P + (i << 12))
    ws, wsb = change.pop("ws", P), change.pop("wsb", 1 << 30)
    for k, v in change.items():
        setattr(a, k, v)
    return L.lib.b2q_moe_forward_w4(a, ws, wsb, None)


@pytest.mark.parametrize("code,args", [(-1, {n: None}) for n in ("x", "weights", "ids", "w13", "s13", "w2", "s2", "out", "ws")] + [(-4, {n: P + 8}) for n in ("x", "w13", "w2", "out", "ws")] + [
    (-4, {n: P + 2}) for n in ("weights", "ids")] + [(-4, {n: P + 1}) for n in ("s13", "s2")] + [
    (-3, dict(act_dtype=2)), (-2, dict(T=-1)), (-2, dict(E=0)), (-2, dict(top_k=0)), (-2, dict(H=0)), (-2, dict(H=96)), (-2, dict(I=48)), (-2, dict(group13=16)), (-2, dict(group2=256)),
    (-10, dict(E=1025)), (-10, dict(top_k=33)), (-10, dict(T=1 << 27)), (-10, dict(H=1 << 21)), (-10, dict(I=1 << 21)), (-10, dict(E=1024, I=1 << 20)), (-10, dict(E=1, H=1 << 18, I=1 << 19)),
    (-10, dict(T=1 << 25, top_k=32, H=1 << 16)), (-8, dict(wsb=100)), (0, dict(T=0))])
def test_expert_layer_refuses(L, code, args):
    before = L.launch_count()
    assert layer(L, **args) == code and L.launch_count() == before


def test_no_layer(L):
    assert L.lib.b2q_moe_forward_w4(None, P, 1 << 30, None) == -1


@pytest.mark.parametrize("T,E,k,H,I", [(1, 8, 2, 64, 32), (16, 128, 8, 2048, 768), (48, 128, 8, 2048, 768), (4096, 128, 8, 2048, 768), (1, 1, 1, 1 << 20, 32)])
def test_expert_layer_scratch(L, T, E, k, H, I):
    """Each pair's h and output, and of many tokens its row of x; the form of few has its outputs in 32 bits, and a maximum of 32 bits for 16 values of h."""
    rows, got = T * k, L.lib.b2q_moe_forward_w4_workspace_bytes(T, E, k, H, I)
    least = rows * (2 * I + 4 * H)
    assert least <= got <= least + rows * (I // 4 + 64) + 300 * E + 8192


def test_linear_scratch(L):
    f = L.lib.b2q_linear_w4_workspace_bytes
    assert f(1, 2048, 2048, 128) == 0 and f(0, 64, 128, 128) == 0 and f(4, 64, 130, 128) == 0 and f(4, 64, 128, 100) == 0 and f(1 << 31, 64, 128, 128) == 0
    # tokens whose rows may have to be copied; sums of parts of k
    assert f(4000, 4096, 4096, 128) >= 4000 * 4096 * 2
    for M in (17, 40, 100):
        assert M * 4096 * 2 <= f(M, 512, 4096, 64) <= M * 4096 * 2 + 8 * 4 * (M + 128) * 512 + 65536
    g = L.lib.b2q_moe_forward_w4_workspace_bytes
    assert g(0, 8, 2, 64, 32) == g(4, 0, 2, 64, 32) == g(4, 8, 0, 64, 32) == g(4, 2000, 2, 64, 32) == g(4, 64, 33, 64, 32) == g(4, 8, 2, 1 << 21, 32) == g(1 << 27, 8, 2, 64, 32) == 0


# ----------------------------------------------------------------------------------------------------------- torch ops
def _arguments(new):
    moe = (new((6, 128), F16), new((6, 2), F32), new((6, 2), I32), new((8, 128, 64), U8), new((8, 2, 128), F16), new((8, 128, 32), U8), new((8, 2, 128), F16))
    return [("route_experts", (new((6, 64), BF), 4), dict(scoring="sigmoid", bias=new((64,), F32), num_groups=8, top_groups=4, group_score="top2"), [((6, 4), F32), ((6, 4), I32)]),
            ("route_experts", (new((0, 8), F32), 2), {}, [((0, 2), F32), ((0, 2), I32)]),
            ("linear_w4", (new((5, 128), BF), new((30, 64), U8), new((1, 30), BF)), {}, [((5, 30), BF)]),
            ("linear_w4", (new((0, 256), F16), new((30, 32), I32), new((8, 30), F16), new((8, 30), U8), new((30,), F16)), {}, [((0, 30), F16)]),
            ("moe_forward_w4", moe, {}, [((6, 128), F16)]),
            ("moe_forward_w4", moe, dict(gate_up_zero=new((8, 2, 128), U8), down_zero=new((8, 2, 128), U8)), [((6, 128), F16)])]


@pytest.mark.parametrize("device", ["meta", "fake cuda", "cpu"])
@pytest.mark.parametrize("i", range(6))
def test_outputs_without_data_and_no_cpu_path(L, device, i):
    import custom_esimd_kernels_vllm as e
    if device == "fake cuda":
        with FakeTensorMode():
            name, args, kw, want = _arguments(lambda s, dt: torch.empty(s, dtype=dt, device="cuda"))[i]
            out = getattr(e, name)(*args, **kw)
    else:
        name, args, kw, want = _arguments(lambda s, dt: torch.empty(s, dtype=dt, device=device))[i]
        if device == "cpu":
            with pytest.raises((RuntimeError, NotImplementedError)):
                getattr(e, name)(*args, **kw)
            return
        out = getattr(e, name)(*args, **kw)
    out = out if isinstance(out, tuple) else (out,)
    assert [(tuple(t.shape), t.dtype) for t in out] == want


def test_fakes_refuse_what_the_operators_refuse(L):
    import custom_esimd_kernels_vllm as e
    new = lambda s, dt: torch.empty(s, dtype=dt, device="meta")      # noqa: E731
    for call in (lambda: e.linear_w4(new((5, 128), F32), new((30, 64), U8), new((1, 30), F32)), lambda: e.linear_w4(new((5, 128), BF), new((30, 32), U8), new((1, 30), BF)),
                 lambda: e.linear_w4(new((5, 128), BF), new((30, 64), torch.int8), new((1, 30), BF)), lambda: e.linear_w4(new((5, 128), BF), new((30, 64), U8), new((1, 31), BF)),
                 lambda: e.moe_forward_w4(new((6, 128), BF), new((6, 2), F32), new((5, 2), I32), *(new((8, 128, 64), U8), new((8, 2, 128), BF)) * 2),
                 lambda: e.route_experts(new((4,), F32), 2), lambda: e.route_experts(new((4, 8), torch.float64), 2),
                 lambda: e.route_experts(new((4, 8), F32), 2, scoring="softplus"), lambda: e.route_experts(new((4, 8), F32), 2, group_score="sum")):
        with pytest.raises(RuntimeError):
            call()


CALL = """
import custom_esimd_kernels_vllm as e
print("imported", e._lib.lib.b2q_version() >= 100)
try:
    e.linear_w4(None, None, None)
except ImportError as x:
    print("refused", "libb2q_w4.so" in str(x))
"""


@pytest.mark.parametrize("switch", ["B2Q_PYTHON_DISPATCH", "B2Q_CHECK_STATUS", None])
def test_without_the_library(L, tmp_path, switch):
    """The switches that keep the other ops on their Python implementation do without it until one of these operators is called; otherwise the import is refused."""
    shutil.copytree(PKG, tmp_path / "custom_esimd_kernels_vllm", ignore=shutil.ignore_patterns("__pycache__", "libb2q_w4.so"))
    r = subprocess.run([sys.executable, "-c", CALL], cwd=tmp_path, env=dict(os.environ, PYTHONPATH=str(tmp_path), **({switch: "1"} if switch else {})), capture_output=True, text=True)
    if switch:
        assert r.returncode == 0 and r.stdout.split("\n")[:2] == ["imported True", "refused True"], r.stderr[-500:]
    else:
        assert r.returncode != 0 and "llm-scaler_b200/build.py" in r.stderr


# ---------------------------------------------------------------------------------------------------------- the oracle
def test_oracle_routes():
    w, ids = w4.route(torch.tensor([[1.0, 3.0, 3.0, 0.0], [-math.inf, 2.0, -math.inf, -math.inf], [0.0, math.nan, 0.0, 0.0], [-math.inf] * 4]), 2)
    assert ids.tolist() == [[1, 2], [1, -1], [-1, -1], [-1, -1]] and w.tolist() == [[0.5, 0.5], [1.0, 0.0], [0.0, 0.0], [0.0, 0.0]]
    # groups (0, 1), (2, 3): the first by its best, the second by the sum of two; the bias moves choices and no weight
    l = torch.tensor([[2.0, -9.0, 1.0, 1.0]])
    assert w4.route(l, 1, num_groups=2, group_score="max")[1].tolist() == [[0]]
    assert w4.route(l, 1, "sigmoid", num_groups=2, group_score="top2")[1].tolist() == [[2]]
    w, ids = w4.route(l, 1, "sigmoid", bias=torch.tensor([0.0, 5.0, 0.0, 0.0]), renormalize=False, scale=2.0)
    assert ids.tolist() == [[1]] and float(w) == pytest.approx(2 / (1 + math.exp(9)))


def test_oracle_weights():
    g = torch.Generator().manual_seed(0)
    w = torch.randn(6, 128, generator=g)
    for symmetric in (True, False):
        q, s, z = w4.quantize(w, 32, symmetric, torch.float16)
        packed = w4.pack(q)
        assert packed.shape == (6, 64) and s.shape == (4, 6) and (z is None) == symmetric
        assert torch.equal(packed.view(torch.int32)[:, 0] >> 4 & 15, q[:, 1].int())
        back = w4.dequant(packed, s, z)
        # half a step of a group, and half of one more at its ends, where codes are cut off or the zero point was rounded
        assert bool(((back - w).abs() <= 1.01 * s.double().t().repeat_interleave(32, 1)).all())
        x = torch.randn(3, 128, generator=g)
        assert torch.equal(w4.linear(x, packed, s, z), x.double() @ back.t())
        assert torch.equal(w4.dequant(packed.view(torch.int32), s, z), back)


def test_oracle_layer_is_the_sum_of_its_experts():
    g = torch.Generator().manual_seed(0)
    x = torch.randn(2, 64, generator=g)
    w13, s13, _ = w4.quantize(torch.randn(3, 64, 64, generator=g), 32, True)
    w2, s2, _ = w4.quantize(torch.randn(3, 64, 32, generator=g), 32, True)
    out, size = w4.moe(x, torch.tensor([[0.5, 2.0], [1.0, 1.0]]), torch.tensor([[1, 2], [7, -1]]), w4.pack(w13), s13, w4.pack(w2), s2)
    y = [w4.expert(x[:1], w4.dequant(w4.pack(w13[i]), s13[i]), w4.dequant(w4.pack(w2[i]), s2[i])) for i in range(3)]
    assert torch.allclose(out[:1], 0.5 * y[1] + 2 * y[2], rtol=1e-12, atol=1e-12) and not bool(out[1].any()) and float(size[1]) == 0
