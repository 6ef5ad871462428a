"""Expert routing and the 4-bit group-quantised layers as a program uses them: which form serves, scratch and graphs, rows and weights that are not finite,
offsets beyond 32 bits, refusals, tracing."""
import ctypes as C
import math
import os
import subprocess
import sys

import pytest
import torch

import custom_esimd_kernels_vllm as e
from custom_esimd_kernels_vllm import _lib as L
from gpu_util import DEV
from oracle import w4
from test_gpu_w4 import check_route, dev, gen, moe_inputs, run_linear, run_moe
from w4_util import DT, check_linear, check_moe, check_moe_by_terms, weight

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


@pytest.fixture
def tensor_cores():
    L.set_force_kernel(2)
    yield
    L.set_force_kernel(0)


# -------------------------------------------------------------------------------------------------- which form serves
@pytest.mark.parametrize("M,N,K,group", [(1, 1, 32, 32), (1, 300, 2048, 128), (3, 129, 160, 32), (8, 1024, 4096, 64), (16, 2000, 1024, 128)])
@pytest.mark.parametrize("dt", ["bf16", "fp16"])
def test_few_tokens_on_tensor_cores_on_request(tensor_cores, M, N, K, group, dt):
    run_linear(M, N, K, group, dt, True, True)
    assert L.last_kernel() == "umma_g4"


@pytest.mark.parametrize("T,E,k,H,I,g13,g2", [(1, 8, 2, 256, 128, 64, 32), (5, 3, 3, 128, 96, 32, 32), (16, 64, 6, 384, 704, 64, 64), (1, 128, 8, 512, 256, 128, 128)])
def test_expert_layer_of_few_tokens_as_grouped_products_on_request(tensor_cores, T, E, k, H, I, g13, g2):
    for dt in DT:
        run_moe(moe_inputs(T, E, k, H, I, g13, g2, dt))
        assert L.last_kernel() == "g4_sum"


def test_which_kernels_serve():
    w, s, z = dev(*weight(gen(0), 512, 1024, 128, BF))
    for M, name in ((1, "g4_stream"), (8, "g4_stream"), (40, "umma_g4"), (500, "umma_g4")):
        e.linear_w4(torch.zeros(M, 1024, dtype=BF, device=DEV), w, s, z)
        assert L.last_kernel() == name
    for T, name in ((1, "g4_pairs_sum"), (20, "g4_pairs_sum"), (300, "g4_sum")):
        e.moe_forward_w4(*dev(*moe_inputs(T, 16, 2, 128, 64, 32, 32, "bf16")))
        assert L.last_kernel() == name


@pytest.mark.parametrize("M", [1, 12, 40, 300])
def test_overlap_modes_agree(M):
    w, s, z = dev(*weight(gen(0), 512, 512, 128, BF))
    a = dev(*moe_inputs(M, 8, 2, 512, 256, 128, 64, "bf16"))
    outs = []
    try:
        for mode in (0, 1, 2):
            L.set_overlap_mode(mode)
            x = a[0]
            for _ in range(3):
                x = e.moe_forward_w4(e.linear_w4(x, w, s, z), *a[1:])
            outs.append(x)
    finally:
        L.set_overlap_mode(1)
    assert torch.equal(outs[0], outs[1]) and torch.equal(outs[0], outs[2])


# -------------------------------------------------------------------------------------------- scratch, pitches, graphs
def guarded(shape, dtype, fill):
    """A tensor of `shape` with a row's worth of `fill` on either side, and a function that says whether those still stand."""
    n, pad = math.prod(shape), 512
    t = torch.full((n + 2 * pad,), fill, dtype=dtype, device=DEV)
    return t[pad:pad + n].view(shape), lambda: bool((t[:pad] == fill).all()) and bool((t[pad + n:] == fill).all())


@pytest.mark.parametrize("M", [1, 7, 12, 40, 100, 300])
@pytest.mark.parametrize("garbage", [0, 255])
def test_linear_within_its_scratch_and_pitch(M, garbage):
    N, K, G, ldo = 200, 4096, 64, 211
    x, (w, s, z) = torch.randn(M, K, generator=gen(M)).bfloat16(), weight(gen(1), N, K, G, BF)
    need = L.lib.b2q_linear_w4_workspace_bytes(M, N, K, G)
    ws, ws_ok = guarded((max(need, 1),), torch.uint8, garbage)
    out, out_ok = guarded((M, ldo), BF, 3.0)
    d = dev(x, w, s, z)
    for _ in range(3):
        rc = L.lib.b2q_linear_w4(d[0].data_ptr(), 0, K, d[1].data_ptr(), d[2].data_ptr(), d[3].data_ptr(), None, out.data_ptr(), ldo, M, N, K, G, ws.data_ptr(), need,
                                 torch.cuda.current_stream().cuda_stream)
        assert rc == 0
        check_linear(out[:, :N], x, w, s, z)
    assert ws_ok() and out_ok() and bool((out[:, N:] == 3).all())


@pytest.mark.parametrize("T", [1, 20, 200])
@pytest.mark.parametrize("garbage", [0, 255])
def test_expert_layer_within_its_scratch(T, garbage):
    E, k, H, I = 8, 2, 160, 96
    a = moe_inputs(T, E, k, H, I, 32, 32, "bf16")
    need = L.lib.b2q_moe_forward_w4_workspace_bytes(T, E, k, H, I)
    ws, ws_ok = guarded((need,), torch.uint8, garbage)
    out, out_ok = guarded((T, H), BF, 3.0)
    d = dev(*a)
    m = L.MoeW4(T=T, E=E, top_k=k, H=H, I=I, group13=32, group2=32, act_dtype=0, out=out.data_ptr())
    for name, t in zip(("x", "weights", "ids", "w13", "s13", "w2", "s2", "z13", "z2"), d):
        setattr(m, name, t.data_ptr())
    for _ in range(3):
        assert L.lib.b2q_moe_forward_w4(C.byref(m), ws.data_ptr(), need, torch.cuda.current_stream().cuda_stream) == 0
        check_moe(out, *w4.moe(*a), BF)
    assert ws_ok() and out_ok()


def test_routing_writes_its_rows_alone():
    l = torch.randn(37, 96, generator=gen(0))
    (w, w_ok), (ids, ids_ok) = guarded((37, 5), torch.float32, 3.0), guarded((37, 5), torch.int32, 7)
    d = l.to(DEV)
    assert L.lib.b2q_route_experts(d.data_ptr(), 2, 96, None, 0, w.data_ptr(), ids.data_ptr(), 37, 96, 5, 0, 1, 1, 0, 1, 1.0, torch.cuda.current_stream().cuda_stream) == 0
    assert torch.equal(ids.cpu(), w4.route(l, 5)[1]) and w_ok() and ids_ok()


def captured(f, pool=None):
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        f()
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, pool=pool):
        out = f()
    return g, out


@pytest.mark.parametrize("M", [1, 40, 100])
def test_two_graphs_of_one_memory_pool(M):
    """The second's scratch lies where the first's was; they are replayed in turn.  40 and 100 tokens have their sums over k in parts."""
    a, b = torch.randn(M, 4096, device=DEV).to(BF), torch.randn(M, 4096, device=DEV).to(BF)
    w, s, z = dev(*weight(gen(2), 256, 4096, 128, BF))
    m = dev(*moe_inputs(M, 8, 2, 256, 128, 64, 32, "bf16"))[1:]
    run = lambda x: e.moe_forward_w4(e.linear_w4(x, w, s, z), *m)      # noqa: E731
    want = run(a), run(b)
    g, first = captured(lambda: run(a))
    h, second = captured(lambda: run(b), g.pool())
    for _ in range(4):
        g.replay()
        got = first.clone()
        h.replay()
        assert torch.equal(got, want[0]) and torch.equal(second, want[1])


# ------------------------------------------------------------------------------------------------- values at the edges
@pytest.mark.parametrize("M", [1, 16, 40, 300])
@pytest.mark.parametrize("dt", ["bf16", "fp16"])
def test_a_scale_that_is_not_finite_spoils_its_own_output_alone(M, dt):
    x, (w, s, z) = torch.randn(M, 512, generator=gen(M)).to(DT[dt]), weight(gen(1), 96, 512, 64, DT[dt])
    want = e.linear_w4(*dev(x, w, s, z))
    s[3, 5], s[0, 40] = math.nan, math.inf
    got = e.linear_w4(*dev(x, w, s, z))
    keep = [n for n in range(96) if n not in (5, 40)]
    assert torch.equal(got[:, keep], want[:, keep]) and not bool(torch.isfinite(got[:, [5, 40]]).any())


@pytest.mark.parametrize("T", [3, 24, 200])
@pytest.mark.parametrize("dt", ["bf16", "fp16"])
def test_a_token_that_is_not_finite_spoils_its_own_output_alone(T, dt):
    a = list(moe_inputs(T, 8, 2, 256, 128, 64, 32, dt))
    want = e.moe_forward_w4(*dev(*a))
    a[0][0, 7], a[0][T // 2, 100], a[1][T - 1, 1] = math.inf, math.nan, math.nan
    got = e.moe_forward_w4(*dev(*a))
    bad = sorted({0, T // 2, T - 1})
    keep = [t for t in range(T) if t not in bad]
    assert torch.equal(got[keep], want[keep])
    assert bool(torch.isnan(got[T // 2]).all()) and bool(torch.isnan(got[T - 1]).all()) and not bool(torch.isfinite(got[0]).all())


@pytest.mark.parametrize("T", [2, 30, 260])
@pytest.mark.parametrize("dt", ["bf16", "fp16"])
def test_expert_layer_with_any_zero_point_and_scales_apart(T, dt):
    """Zero points over all of uint8; the outputs' scales from 1 / 8 to 8 times the usual."""
    a = list(moe_inputs(T, 6, 2, 256, 128, 64, 32, dt))
    g = gen(5)
    for zero, scale in ((7, 4), (8, 6)):
        a[zero] = torch.randint(0, 256, a[zero].shape, generator=g, dtype=torch.uint8)
        a[scale] = (a[scale].float() / 16 * 2.0 ** torch.randint(-3, 4, (a[scale].shape[-1],), generator=g)).to(a[0].dtype)
    check_moe_by_terms(e.moe_forward_w4(*dev(*a)), a, "any zero")


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("bt", [torch.float32, BF, torch.float16])
def test_route_bias_at_the_edges(scoring, bt):
    """A bias of -inf or NaN takes an expert out, in groups too; very large ones hide the scores behind them, so that the lowest index decides."""
    l = torch.randn(9, 32, generator=gen(0))
    bias = torch.randn(32, generator=gen(1)).to(bt)
    bias[3], bias[17] = -math.inf, math.nan
    bias[8:16] = -math.inf
    for kw in ({}, dict(num_groups=4, top_groups=2), dict(num_groups=4, top_groups=3, group_score="top2"), dict(num_groups=4, top_groups=4)):
        check_route(l, 6, scoring=scoring, bias=bias, **kw)
    check_route(l, 4, scoring=scoring, bias=torch.full((32,), -math.inf).to(bt))
    check_route(l, 5, scoring=scoring, bias=(bias.nan_to_num(0, 0, 0) * 3e4).round().to(bt), renormalize=False, scale=-2.5)


def test_route_of_one_expert():
    for dt in (torch.float32, BF, torch.float16):
        check_route(torch.randn(5, 1, generator=gen(0)).to(dt), 1)
        check_route(torch.randn(5, 1, generator=gen(0)).to(dt), 1, scoring="sigmoid", renormalize=False)


@pytest.mark.parametrize("T,E", [(150, 128), (700, 4), (1500, 3)])
def test_a_token_comes_out_the_same_wherever_it_stands(T, E):
    """The rows of an expert are collected by atomics: their order, and so the tile a row is in, changes from call to call, its bits do not."""
    a = dev(*moe_inputs(T, E, 2, 256, 288, 64, 32, "bf16"))
    want = e.moe_forward_w4(*a)
    for seed in range(6):
        order = torch.randperm(T, generator=gen(seed)).to(DEV)
        assert torch.equal(e.moe_forward_w4(*(t[order] for t in a[:3]), *a[3:]), want[order])


def test_route_of_equal_and_of_many_near_experts():
    """More than a warp's lanes of candidates, and choices that only 64 bits tell apart among them."""
    g = gen(3)
    l = torch.zeros(12, 256)
    l[1] = 1 + torch.arange(256) % 3 * 2.0 ** -23
    l[2, 100:] = -1
    l[3] = torch.arange(256) // 8 * 0.5
    l[4] = torch.randint(0, 2, (256,), generator=g) * 1.0
    l[5:] = 0.5 + torch.randint(0, 4, (7, 256), generator=g) * 2.0 ** -24
    bias = torch.randint(0, 3, (256,), generator=g) * 2.0 ** -24
    for kw in ({}, dict(scoring="sigmoid"), dict(scoring="sigmoid", bias=bias), dict(bias=bias), dict(num_groups=8, top_groups=3), dict(num_groups=8, top_groups=3, group_score="top2"),
               dict(scoring="sigmoid", bias=bias, num_groups=8, top_groups=4, group_score="top2"), dict(num_groups=16, top_groups=5, group_score="top2", bias=bias)):
        for k in (1, 8, 32):
            check_route(l, k, **kw)
            check_route(l[:, :192].contiguous(), min(k, 24), **{n: v[:192].contiguous() if torch.is_tensor(v) else v for n, v in kw.items()})


# ------------------------------------------------------------------------------------------- offsets beyond 32 bits
def test_linear_weight_beyond_two_gib():
    N, K, G = 70000, 65536, 128
    w = torch.randint(0, 256, (N, K // 2), dtype=torch.uint8, device=DEV)
    s = (torch.rand(K // G, N, device=DEV) * 0.01 + 0.001).to(BF)
    z = torch.randint(0, 16, (K // G, N), dtype=torch.uint8, device=DEV)
    rows = torch.tensor([0, 1, 40000, 65535, 65536, 65600, N - 2, N - 1])
    part = w[rows.to(DEV)].cpu(), s[:, rows.to(DEV)].cpu(), z[:, rows.to(DEV)].cpu()
    for M in (1, 12, 40, 200):
        x = torch.randn(M, K, generator=gen(M)).to(BF)
        check_linear(e.linear_w4(x.to(DEV), w, s, z)[:, rows.to(DEV)], x, *part, what="%d tokens" % M)


def test_linear_output_beyond_two_to_the_31():
    M, N, K = 40003, 60001, 128
    w, s, z = dev(*weight(gen(0), N, K, 128, BF))
    x = torch.randn(M, K, device=DEV).to(BF)
    out = e.linear_w4(x, w, s, z)
    rows, cols = torch.tensor([0, 1, 35800, M - 2, M - 1], device=DEV), torch.tensor([0, 7, 30000, N - 2, N - 1], device=DEV)
    check_linear(out[rows][:, cols], x[rows].cpu(), w[cols].cpu(), s[:, cols].cpu(), z[:, cols].cpu())


@pytest.mark.parametrize("T", [2, 400])
def test_experts_beyond_two_gib(T):
    E, H, I = 300, 4096, 2048
    new = lambda *shape: torch.randint(0, 256, shape, dtype=torch.uint8, device=DEV)      # noqa: E731
    w13, w2 = new(E, 2 * I, H // 2), new(E, H, I // 2)
    s13, s2 = ((torch.rand(E, k // 128, n, device=DEV) * 0.004 + 0.001).to(BF) for k, n in ((H, 2 * I), (I, H)))
    x, w = torch.randn(T, H, generator=gen(0)).to(BF), torch.rand(T, 2, generator=gen(1)) + 0.1
    ids = torch.randint(0, E, (T, 2), generator=gen(2), dtype=torch.int32)
    ids[0], ids[-1] = torch.tensor([E - 1, E - 2]), torch.tensor([E - 2, 0])
    out = e.moe_forward_w4(*dev(x, w, ids), w13, s13, w2, s2)
    few = torch.tensor([E - 2, E - 1, 0])
    local = torch.full((E,), -1, dtype=torch.int32)
    local[few.long()] = torch.arange(3, dtype=torch.int32)
    part = [t[few.to(DEV)].cpu() for t in (w13, s13, w2, s2)]
    rows = [0, T - 1]
    check_moe(out[rows], *w4.moe(x[rows], w[rows], local[ids[rows].long()], *part), BF)


def test_pairs_beyond_two_to_the_31():
    T, E, k, H, I = 70001, 8, 8, 4096, 32
    w13, s13, z13 = weight(gen(0), 2 * I, H, 128, BF, True, (E,))
    w2, s2, z2 = weight(gen(1), H, I, 32, BF, True, (E,))
    x = torch.randn(T, H, device=DEV).to(BF)
    w, ids = e.route_experts(torch.randn(T, E, device=DEV), k)
    out = e.moe_forward_w4(x, w, ids, *dev(w13, s13, w2, s2, z13, z2))
    rows = [0, 1, 65535, 65536, T - 2, T - 1]
    check_moe(out[rows], *w4.moe(*(t[rows].cpu() for t in (x, w, ids)), w13, s13, w2, s2, z13, z2), BF)


def test_logits_beyond_two_to_the_31():
    T = (1 << 21) + 5
    l = torch.empty(T, 1024, dtype=BF, device=DEV).normal_()
    w, ids = e.route_experts(l, 8)
    rows = [0, 1, T // 2, T - 6, T - 1]
    ref_w, ref_ids = w4.route(l[rows].cpu(), 8)
    assert torch.equal(ids[rows].cpu(), ref_ids) and bool(((w[rows].cpu().double() - ref_w).abs() <= 80 * 2.0 ** -24 * ref_w).all())


# ------------------------------------------------------------------------------------------------------------- refusals
def test_refusals():
    x = torch.randn(4, 128, device=DEV).to(BF)
    w, s, z = dev(*weight(gen(0), 32, 128, 64, BF))
    b = torch.zeros(32, dtype=BF, device=DEV)
    a = dev(*moe_inputs(4, 4, 2, 128, 64, 64, 32, "bf16"))
    l = torch.randn(4, 16, device=DEV)

    def other(i, t):
        return lambda: e.moe_forward_w4(*a[:i], t, *a[i + 1:])

    calls = [lambda: e.linear_w4(x.float(), w, s, z), lambda: e.linear_w4(x[0], w, s, z), lambda: e.linear_w4(x.t(), w, s, z), lambda: e.linear_w4(x[:1].expand(4, 128), w, s, z),
             lambda: e.linear_w4(x[:, :64], w, s, z), lambda: e.linear_w4(x, w[:, ::2], s, z), lambda: e.linear_w4(x, w.float(), s, z), lambda: e.linear_w4(x, w, s.half(), z),
             lambda: e.linear_w4(x, w, s.t(), z), lambda: e.linear_w4(x, w, s[:, :16], z), lambda: e.linear_w4(x, w, s[:0], z), lambda: e.linear_w4(x, w, s.repeat(4, 1)),
             lambda: e.linear_w4(x, w, s, z.float()), lambda: e.linear_w4(x, w, s, z[:1]), lambda: e.linear_w4(x, w, s, z, b.float()), lambda: e.linear_w4(x, w, s, z, b[:16]),
             lambda: e.linear_w4(x, w.cpu(), s, z), lambda: e.linear_w4(x, w, s, z.cpu()), lambda: e.linear_w4(x.cpu(), w, s, z), lambda: e.linear_w4(x, w, s, z, b.cpu()),
             lambda: e.linear_w4(x, torch.empty(32 * 64 + 8, dtype=torch.uint8, device=DEV)[8:].view(32, 64), s, z),
             other(0, a[0].float()), other(0, a[0][:, :64]), other(0, torch.cat((a[0], a[0]), 1)[:, :128]), other(1, a[1].half()), other(1, a[1][:, :1]), other(2, a[2].long()),
             other(2, a[2][:3]), other(3, a[3][:2]), other(3, a[3][:, :-1].contiguous()), other(4, a[4].half()), other(5, a[5][:, :64].contiguous()), other(6, a[6][:, :1]), other(7, a[7].int()),
             other(8, a[8].cpu()), other(2, a[2][:, :0]),
             lambda: e.route_experts(l, 0), lambda: e.route_experts(l, 17), lambda: e.route_experts(l.double(), 2), lambda: e.route_experts(l[0], 2), lambda: e.route_experts(l.t(), 2),
             lambda: e.route_experts(l, 2, num_groups=3), lambda: e.route_experts(l, 2, num_groups=4, top_groups=5), lambda: e.route_experts(l, 5, num_groups=4, top_groups=1),
             lambda: e.route_experts(l, 2, bias=l[0, :8]), lambda: e.route_experts(l, 2, bias=l[0].cpu()), lambda: e.route_experts(l, 2, bias=l[0].double()),
             lambda: e.route_experts(torch.zeros(2, 2000, device=DEV), 2), lambda: e.route_experts(torch.zeros(2, 128, device=DEV), 64), lambda: e.route_experts(l, 2, scoring="top")]
    before = L.launch_count()
    for i, call in enumerate(calls):
        with pytest.raises((RuntimeError, NotImplementedError)):
            call()
            pytest.fail("call %d" % i)
    assert L.launch_count() == before
    torch.cuda.synchronize()


# -------------------------------------------------------------------------------------------------------------- tracing
def test_schemas_and_fake_implementations():
    n = torch.ops.b2q_w4
    a = dev(*moe_inputs(6, 8, 2, 128, 64, 64, 32, "bf16"))
    w, s, z = dev(*weight(gen(0), 32, 128, 64, BF))
    for op, args in [(n.route_experts, (torch.randn(6, 8, device=DEV), 2, 1, torch.zeros(8, device=DEV), 2, 1, 1, True, 1.0)), (n.linear, (a[0], w, s, z, None)), (n.moe_forward, tuple(a))]:
        torch.library.opcheck(op.default, args, test_utils=("test_schema", "test_faketensor"))


@pytest.mark.parametrize("dynamic", [False, True])
def test_a_traced_layer_equals_an_eager_one(dynamic):
    weights = dev(*moe_inputs(1, 8, 2, 128, 64, 64, 32, "bf16"))[3:]
    gate = torch.randn(8, 128, device=DEV).to(BF)
    w, s, z = dev(*weight(gen(0), 128, 128, 64, BF))

    def layer(x):
        x = e.linear_w4(x, w, s, z)
        tw, ids = e.route_experts(x @ gate.t(), 2, "sigmoid", num_groups=2)
        return e.moe_forward_w4(x, tw, ids, *weights)

    torch._dynamo.reset()
    traced = torch.compile(layer, backend="aot_eager", fullgraph=True, dynamic=dynamic)
    for M in (3, 40, 7):
        x = torch.randn(M, 128, device=DEV).to(BF)
        assert torch.equal(traced(x), layer(x))


def test_checked_calls():
    """With B2Q_CHECK_STATUS=1 every call synchronises and looks at the device's status."""
    code = ("import torch, custom_esimd_kernels_vllm as e\n"
            "x = torch.randn(40, 128, device='cuda').bfloat16(); w = torch.full((64, 64), 0x98, dtype=torch.uint8, device='cuda'); s = torch.ones(1, 64, device='cuda').bfloat16()\n"
            "out = e.linear_w4(x, w, s)\n"
            "w, i = e.route_experts(x, 2)\n"
            "print(torch.allclose(out.float(), x[:, 1::2].float().sum(1, keepdim=True).expand(40, 64), rtol=8e-3, atol=1e-3), i.shape)\n")
    path = os.path.dirname(os.path.dirname(e.__file__))
    r = subprocess.run([sys.executable, "-c", code], env=dict(os.environ, PYTHONPATH=path, B2Q_CHECK_STATUS="1"), capture_output=True, text=True)
    assert r.returncode == 0 and r.stdout.split() == ["True", "torch.Size([40,", "2])"], r.stdout + r.stderr[-500:]
