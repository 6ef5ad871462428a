"""Expert routing, linears and expert layers of 4-bit group-quantised weights against 64 bits."""
import math

import pytest
import torch

import custom_esimd_kernels_vllm as e
from gpu_util import DEV
from oracle import w4
from w4_util import DT, check_linear, check_moe, half_step, weight

pytestmark = pytest.mark.gpu


def gen(seed):
    return torch.Generator().manual_seed(seed)


def dev(*ts):
    return [None if t is None else t.to(DEV) for t in ts]


# ------------------------------------------------------------------------------------------------------------- routing
def check_route(logits, k, **kw):
    got_w, got_ids = e.route_experts(logits.to(DEV), k, **{n: v.to(DEV) if torch.is_tensor(v) else v for n, v in kw.items()})
    ref_w, ref_ids = w4.route(logits, k, **kw)
    assert got_ids.dtype == torch.int32 and got_w.dtype == torch.float32
    assert torch.equal(got_ids.cpu(), ref_ids)
    # some sixteen roundings (two exponentials, sums, quotients), and that of l - max, half a step of up to 64
    assert bool(((got_w.double().cpu() - ref_w).abs() <= (16 + 64) * 2.0 ** -24 * ref_w.abs() + 1e-37).all())


@pytest.mark.parametrize("T,E,k,groups,top_groups", [(1, 256, 8, 8, 4), (7, 8, 2, 1, 1), (33, 64, 6, 1, 1), (5, 160, 6, 8, 3), (4, 1024, 32, 32, 5), (3, 60, 4, 1, 1),
                                                     (2, 512, 10, 1, 1), (9, 16, 4, 16, 7), (1, 1, 1, 1, 1), (6, 96, 1, 6, 1), (130, 128, 8, 1, 1), (3, 250, 5, 5, 2)])
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("biased", [False, True])
def test_route(T, E, k, groups, top_groups, scoring, biased):
    g = gen(T * E + k)
    for dt, group_score, renormalize, scale in ((torch.float32, "max", True, 1.0), (torch.bfloat16, "top2", False, 2.5), (torch.float16, "top2", True, 0.5)):
        logits = (2 * torch.randn(T, E, generator=g)).to(dt)
        bias = 0.2 * torch.randn(E, generator=g) if biased else None
        check_route(logits, k, scoring=scoring, bias=bias, num_groups=groups, top_groups=top_groups, group_score=group_score, renormalize=renormalize, scale=scale)


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
def test_route_ties_masks_and_bad_rows(scoring):
    g = gen(5)
    inf = math.inf
    logits = torch.randint(-2, 3, (24, 64), generator=g).float()      # ties everywhere
    logits[1] = 0
    logits[2] = -inf
    logits[3, 5:] = -inf
    logits[4, 7] = math.nan
    logits[5, 9] = inf
    logits[6, ::2] = -inf
    logits[7] = -0.0
    logits[7, ::3] = 0.0
    logits[8, :32] = -inf
    logits[9] = torch.finfo(torch.float32).min
    logits[10] = -300 + torch.arange(64) / 64.0      # scores that underflow
    logits[11] = 40 + torch.arange(64) % 3           # sigmoids that 64 bits round to 1
    bias = torch.randint(-1, 2, (64,), generator=g).float() / 4
    bias[3], bias[40] = -inf, math.nan
    for b in (None, bias):
        for groups, top_groups, score in ((1, 1, "max"), (8, 3, "max"), (8, 3, "top2")):
            check_route(logits, 6, scoring=scoring, bias=b, num_groups=groups, top_groups=top_groups, group_score=score)
            if scoring == "softmax" or b is not None:
                check_route(logits, 6, scoring=scoring, bias=b, num_groups=groups, top_groups=top_groups, group_score=score, renormalize=False)


def test_route_decides_between_neighbours():
    """Logits one unit in the last place apart, whose scores fp32 cannot tell apart, and biases that all but cancel the difference of two scores."""
    base = torch.tensor([9.0, 12.0, 3.5, 14.0])
    steps = torch.arange(64, dtype=torch.int32) * 5 % 64
    logits = torch.stack([(torch.full((64,), float(b)).view(torch.int32) + steps).view(torch.float32) for b in base])
    for scoring in ("sigmoid", "softmax"):
        for bias in (None, torch.zeros(64), torch.linspace(0, 1e-8, 64)):
            check_route(logits, 8, scoring=scoring, bias=bias)
            check_route(logits, 8, scoring=scoring, bias=bias, num_groups=8, top_groups=4, group_score="top2")
    l = torch.randn(40, 32, generator=gen(1))
    for t in range(40):
        p = torch.sigmoid(l[t].double())
        check_route(l[t:t + 1], 8, scoring="sigmoid", bias=(1.5 - p).float())


def test_route_strided_rows_and_streams():
    wide = torch.randn(17, 100, generator=gen(3)).to(DEV)
    a = e.route_experts(wide[:, 3:67], 4)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        b = e.route_experts(wide[:, 3:67].contiguous(), 4)
    s.synchronize()
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    assert e.route_experts(wide[:0, :64], 4)[1].shape == (0, 4)


# ------------------------------------------------------------------------------------------------------------- linear
def run_linear(M, N, K, group, dt, zero, bias, seed=0, pitch=None, as_int32=False):
    g = gen(seed + M * 7 + N + K)
    dtype = DT[dt]
    x = torch.randn(M, pitch or K, generator=g).to(dtype)
    if M > 2:
        x[M // 2] = 0
    packed, s, z = weight(g, N, K, group, dtype, zero)
    b = torch.randn(N, generator=g).to(dtype) if bias else None
    w = packed.view(torch.int32) if as_int32 else packed
    out = e.linear_w4(x.to(DEV)[:, :K], *dev(w, s, z, b))
    assert out.dtype == dtype and out.shape == (M, N)
    check_linear(out, x[:, :K], packed, s, z, b, "%dx%dx%d g%d %s" % (M, N, K, group, dt))


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("dt", ["bf16", "fp16"])
@pytest.mark.parametrize("M", [1, 2, 5, 8, 9, 16, 17, 33, 64, 65, 128, 200, 300])
def test_linear_tokens(M, dt, group):
    run_linear(M, 264, 768, group, dt, True, M % 2 == 0)


@pytest.mark.parametrize("M,N,K,group,zero", [(1, 1, 128, 128, True), (1, 7, 32, 32, False), (3, 129, 160, 32, True), (4, 2048, 2048, 128, True), (1, 5000, 4096, 64, False),
                                              (8, 2065, 6144, 128, True), (16, 512, 14336, 64, True), (1, 300, 28672, 128, True), (33, 515, 1088, 64, False), (70, 1000, 2048, 128, True),
                                              (257, 130, 2048, 32, True), (520, 1032, 1024, 128, True), (1000, 384, 4096, 64, True), (129, 4096, 512, 128, False), (40, 33, 96, 32, True),
                                              (2, 20000, 256, 64, True), (12, 640, 128, 128, False), (24, 3000, 5120, 32, True), (2049, 257, 256, 128, True)])
def test_linear_shapes(M, N, K, group, zero):
    for i, dt in enumerate(DT):
        run_linear(M, N, K, group, dt, zero, i == 0, as_int32=i == 1)


@pytest.mark.parametrize("M", [1, 6, 40, 150])
@pytest.mark.parametrize("extra", [1, 3, 8, 640])
def test_linear_takes_slices(M, extra):
    run_linear(M, 200, 512, 128, "bf16", True, False, pitch=512 + extra)


@pytest.mark.parametrize("M", [1, 9, 50, 300])
@pytest.mark.parametrize("dt", ["bf16", "fp16"])
def test_linear_range(M, dt):
    """Rows of huge and of tiny values, outliers, zero points beyond 15, scales at the ends of what the weights can hold, and rows that are not finite, which
    no other row sees."""
    g = gen(M)
    dtype, N, K = DT[dt], 96, 384
    x = torch.randn(M, K, generator=g)
    big, small = (1e30, 1e-30) if dt == "bf16" else (3e3, 1e-4)
    x[0] *= small
    x[M // 2] *= big
    x[M - 1, ::37] *= 300
    x = x.to(dtype)
    packed, s, z = weight(g, N, K, 64, dtype)
    s = (s.float() * torch.logspace(-2, 1, N)).to(dtype)
    z[:, ::5] = 16
    z[:, 1::7] = 255
    out = e.linear_w4(*dev(x, packed, s, z))
    for m in sorted({0, M // 2, M - 1}):
        check_linear(out[m:m + 1], x[m:m + 1], packed, s, z, None, "row %d" % m)
    if M > 1:
        bad = x.clone()
        bad[0, 5], bad[M // 2, 17] = math.inf, math.nan
        got = e.linear_w4(*dev(bad, packed, s, z))
        keep = [m for m in range(M) if m not in (0, M // 2)]
        assert torch.equal(got[keep], out[keep])
        assert not bool(torch.isfinite(got[0]).any()) and bool(torch.isnan(got[M // 2]).all())


def test_linear_empty():
    x, (w, s, z) = torch.zeros(0, 128, dtype=torch.bfloat16), weight(gen(0), 16, 128, 128, torch.bfloat16)
    assert e.linear_w4(*dev(x, w, s, z)).shape == (0, 16)
    assert e.linear_w4(*dev(torch.zeros(3, 128, dtype=torch.bfloat16), w[:0], s[:, :0].contiguous(), z[:, :0].contiguous())).shape == (3, 0)


# --------------------------------------------------------------------------------------------------------- expert layer
def moe_inputs(T, E, k, H, I, g13, g2, dt, zero=True, seed=0):
    g = gen(seed + T + E + H)
    dtype = DT[dt]
    x = torch.randn(T, H, generator=g).to(dtype)
    ids = torch.stack([torch.randperm(E, generator=g)[:k] for _ in range(T)]).to(torch.int32)
    w = torch.rand(T, k, generator=g) + 0.1
    w13, s13, z13 = weight(g, 2 * I, H, g13, dtype, zero, (E,))
    w2, s2, z2 = weight(g, H, I, g2, dtype, zero, (E,))
    return x, w, ids, w13, s13, w2, s2, z13, z2


def run_moe(a, what=""):
    out = e.moe_forward_w4(*dev(*a))
    check_moe(out, *w4.moe(*a), a[0].dtype, what)
    return out


@pytest.mark.parametrize("T", [1, 2, 3, 8, 16, 17, 40, 130, 600])
@pytest.mark.parametrize("dt", ["bf16", "fp16"])
def test_moe_tokens(T, dt):
    run_moe(moe_inputs(T, 8, 2, 256, 128, 64, 32, dt))


@pytest.mark.parametrize("T,E,k,H,I,g13,g2,zero", [(1, 128, 8, 512, 256, 128, 128, True), (5, 3, 3, 128, 96, 32, 32, False), (16, 64, 6, 384, 704, 64, 64, True), (33, 16, 1, 256, 384, 128, 128, True),
                                                   (300, 5, 4, 640, 160, 128, 32, False), (1, 1, 1, 128, 32, 32, 32, True), (64, 200, 8, 256, 128, 64, 128, True), (7, 12, 12, 1024, 512, 128, 64, True),
                                                   (1000, 4, 2, 256, 256, 64, 64, True), (3, 8, 2, 2048, 1408, 128, 64, True)])
def test_moe_shapes(T, E, k, H, I, g13, g2, zero):
    for dt in DT:
        run_moe(moe_inputs(T, E, k, H, I, g13, g2, dt, zero))


@pytest.mark.parametrize("T", [1, 6, 50, 400])
def test_moe_routes(T):
    """Ids of no expert here, an expert named twice, all tokens at one expert, weights of zero and below."""
    a = list(moe_inputs(T, 6, 3, 256, 160, 64, 32, "bf16", seed=1))
    ids, w = a[2], a[1]
    ids[::2, 0] = -1
    ids[1::3, 1] = 6
    ids[:, 2] = 4
    w[::4, 2] = 0
    w[1::4, 2] = -1.5
    run_moe(a, "mixed")
    ids[:] = 3
    run_moe(a, "all at one, three times")
    ids[:, 0], ids[:, 1], ids[:, 2] = -1, 1 << 30, -(1 << 31)
    assert not bool(e.moe_forward_w4(*dev(*a)).any())


def test_moe_of_routed_tokens():
    """Routing and expert layer together, with padding rows that go nowhere."""
    for T in (1, 24, 210):
        x, _, _, *weights = moe_inputs(T, 16, 4, 256, 128, 128, 64, "bf16")
        logits = torch.randn(T, 16, generator=gen(T))
        if T > 2:
            logits[-2:] = -math.inf
        bias = 0.1 * torch.randn(16, generator=gen(1))
        kw = dict(scoring="sigmoid", num_groups=4, top_groups=2, group_score="top2", scale=1.5)
        w, ids = e.route_experts(logits.to(DEV), 4, bias=bias.to(DEV), **kw)
        out = e.moe_forward_w4(x.to(DEV), w, ids, *dev(*weights))
        rw, rids = w4.route(logits, 4, bias=bias, **kw)
        check_moe(out, *w4.moe(x, rw, rids, *weights), x.dtype)
        if T > 2:
            assert not bool(out[-2:].any())


def test_moe_empty():
    a = moe_inputs(2, 4, 2, 128, 64, 64, 32, "bf16")
    assert e.moe_forward_w4(*dev(*(t[:0] for t in a[:3]), *a[3:])).shape == (0, 128)


@pytest.mark.parametrize("T", [1, 20, 300])
def test_graph_replays_and_repeats(T):
    """Captured once and replayed on new inputs; the same bits every time, and those of a call outside the graph."""
    x, w, ids, *weights = dev(*moe_inputs(T, 8, 2, 256, 128, 64, 32, "bf16"))
    lw, ls, lz = dev(*weight(gen(2), 520, 256, 64, torch.bfloat16))
    logits = torch.randn(T, 8, generator=gen(9)).to(DEV)

    def step():
        tw, ti = e.route_experts(logits, 2)
        return e.linear_w4(e.moe_forward_w4(x, tw, ti, *weights), lw, ls, lz)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for seed in range(3):
        x.copy_(torch.randn(x.shape, generator=gen(seed)).to(x.dtype))
        logits.copy_(torch.randn(logits.shape, generator=gen(seed + 10)))
        graph.replay()
        first = out.clone()
        for _ in range(5):
            graph.replay()
            assert torch.equal(out, first)
        assert torch.equal(step(), first)


def test_two_streams_at_once():
    a, b = dev(*moe_inputs(40, 8, 2, 256, 128, 64, 32, "bf16")), dev(*moe_inputs(3, 8, 2, 256, 128, 64, 32, "bf16", seed=4))
    lw, ls, lz = dev(*weight(gen(2), 520, 256, 64, torch.bfloat16))
    want = [e.moe_forward_w4(*a), e.moe_forward_w4(*b), e.linear_w4(a[0], lw, ls, lz)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    for _ in range(10):
        got = []
        for s, f in zip(streams, (lambda: e.moe_forward_w4(*a), lambda: e.moe_forward_w4(*b), lambda: e.linear_w4(a[0], lw, ls, lz))):
            with torch.cuda.stream(s):
                got.append(f())
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(got, want))
