"""The int8 expert layer against its definition in 64 bits (oracle/int8.py).

No tolerance on the output: an interval that holds it is followed through the layer.  h is known to 2^-17 (SiLU's exponential is good to 10
units of 2^-23 for |gate| <= 7, each fp32 step to 2^-24), routing weights to 2^-19.  Rounding is monotone, so the ends of h's interval, rounded
as the layer rounds them, give the ends of its row's scale and of every code; nearly all codes have equal ends.  What the others can differ
by, times |w2|, is the interval of an expert's output, which the remaining steps (rounded to 16 bits before the weighted sum, where there are
more than 2^19 of them) map to the result's."""
import math

import pytest
import torch

from gpu_util import DEV
from oracle import int8

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops(lib_built):
    import custom_esimd_kernels_vllm as e
    yield e
    e.set_overlap_mode(1)
    assert e._lib.device_status() == 0


def make(T, E, H, I, dt, seed, sdt=torch.float32, ldt=torch.float32):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(T, H, generator=g).to(dt)
    logits = torch.randn(T, E, generator=g).to(ldt)
    w13 = torch.randint(-127, 128, (E, 2 * I, H), generator=g, dtype=torch.int8)
    w2 = torch.randint(-127, 128, (E, H, I), generator=g, dtype=torch.int8)
    s13 = ((0.5 + torch.rand(E, 2 * I, generator=g)) * 0.02 / math.sqrt(H)).to(sdt)
    s2 = ((0.5 + torch.rand(E, H, generator=g)) * 0.02 / math.sqrt(I)).to(sdt)
    return x, logits, w13, s13, w2, s2


def on_gpu(a):
    return [t.to(DEV) for t in a]


def one_kernel(T, k, H, I):
    """Whether the layer takes one kernel: little that every CTA has to fetch."""
    return T <= 16 and T * (4 * k * I + H) <= 40960


def experts_interval(h, w2, s2, dt, exact):
    """Ends of an expert's output for rows h (64 bits, good to 2^-17)."""
    lo, hi = h.abs() * (1 - 2.0 ** -17), h.abs() * (1 + 2.0 ** -17)
    a_lo, a_hi = [v.amax(1, keepdim=True).clamp(min=int8.MIN_AMAX) for v in (lo, hi)]
    q_lo, q_hi = (127 * lo / a_hi).round(), (127 * hi / a_lo).clamp(max=127).round()
    mid, off = h.sign() * (q_lo + q_hi) / 2, (q_hi - q_lo) / 2
    scale, spread = (a_lo + a_hi) / 254, (a_hi - a_lo) / 254
    y = scale * (mid @ w2.double().t()) * s2.double()
    err = (scale + spread) * (off @ w2.double().abs().t()) * s2.double() + y.abs() * (spread / scale + 2.0 ** -21)
    if exact:
        return y - err, y + err
    return (y - err).to(dt).double(), (y + err).to(dt).double()


def check(out, a, k, renorm=True):
    x, logits, w13, s13, w2, s2 = a
    exact, dt = k * x.numel() <= 1 << 19, x.dtype
    ids, w = int8.route(logits, k, renorm)
    codes, _, scale = int8.quantize_rows(x)
    lo, hi = torch.zeros(2, *out.shape, dtype=torch.float64)
    for e in ids.unique().tolist():
        t, slot = torch.nonzero(ids == e, as_tuple=True)
        h = int8.silu_mul(int8.linear(codes[t], scale[t], w13[e], s13[e]))
        y = experts_interval(h, w2[e], s2[e], dt, exact)
        slack = 2.0 ** -19 * w[t, slot, None] * torch.maximum(y[0].abs(), y[1].abs())
        lo.index_add_(0, t, w[t, slot, None] * y[0] - slack)
        hi.index_add_(0, t, w[t, slot, None] * y[1] + slack)
    lo, hi, o = lo.to(dt).double(), hi.to(dt).double(), out.cpu().double()
    bad = (o < lo) | (o > hi)
    assert not bad.any(), (int(bad.sum()), bad.numel(), torch.nonzero(bad)[:4].tolist())
    # and the interval is no wider than what it stands for
    assert ((hi - lo).norm() <= 0.1 * o.norm())


SHAPES = [(1, 8, 2, 64, 32), (1, 128, 8, 2048, 768), (2, 16, 1, 128, 48), (3, 8, 2, 4096, 1024), (5, 60, 4, 1008, 176), (7, 4, 4, 144, 400), (8, 256, 8, 512, 256), (13, 128, 8, 1040, 528),
          (16, 128, 8, 2048, 768), (16, 3, 2, 6400, 64), (16, 512, 10, 256, 128), (4, 1024, 32, 64, 64), (16, 8, 2, 5120, 128),
          (16, 512, 10, 256, 48), (16, 128, 1, 2048, 128), (13, 128, 2, 1040, 240), (7, 4, 4, 144, 80), (8, 256, 8, 512, 128), (1, 3, 2, 512, 5040), (1, 2, 1, 4096, 9216),
          (1, 40, 4, 24576, 96), (16, 3, 2, 2048, 64), (15, 40, 1, 2448, 64), (16, 4, 4, 512, 112), (2, 40, 32, 4480, 16), (2, 4, 2, 512, 14336),
          (17, 128, 8, 512, 256), (33, 8, 2, 272, 144), (64, 16, 4, 1024, 512), (100, 60, 4, 512, 400), (300, 8, 2, 512, 1040), (257, 300, 6, 128, 64), (700, 4, 1, 256, 128), (64, 16, 8, 1024, 64), (65, 16, 8, 1024, 64)]


@pytest.mark.parametrize("T,E,k,H,I", SHAPES)
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
def test_expert_layer(ops, T, E, k, H, I, dt):
    sdt = [torch.float32, torch.bfloat16, torch.float16][(T + E) % 3]
    a = make(T, E, H, I, dt, T * E + k, sdt)
    out = ops.moe_forward_int8(*on_gpu(a), k)
    assert out.shape == (T, H) and out.dtype == dt
    assert (ops.last_kernel() == "moe_i8") == one_kernel(T, k, H, I)
    check(out, a, k)


@pytest.mark.parametrize("T", [1, 6, 16, 40])
def test_weights_that_are_not_renormalised(ops, T):
    a = make(T, 16, 256, 128, torch.bfloat16, T)
    check(ops.moe_forward_int8(*on_gpu(a), 3, False), a, 3, False)


@pytest.mark.parametrize("T", [4, 16, 24])
@pytest.mark.parametrize("ldt", [torch.bfloat16, torch.float16, torch.float32])
def test_equal_logits_go_to_the_lowest_index(ops, T, ldt):
    a = list(make(T, 40, 128, 64, torch.float16, T))
    l = torch.randint(-2, 3, (T, 40), generator=torch.Generator().manual_seed(T)).float()
    l[0] = 0
    l[1, ::2] = -0.0
    l[1, 1::2] = 0.0
    l[2, 5:] = -float("inf")
    a[1] = l.to(ldt)
    check(ops.moe_forward_int8(*on_gpu(a), 6), a, 6)


@pytest.mark.parametrize("T", [1, 16, 48])
def test_all_tokens_to_the_same_experts(ops, T):
    a = list(make(T, 32, 256, 160, torch.bfloat16, T))
    a[1] = torch.zeros(T, 32)
    a[1][:, 30:] = 4.0
    check(ops.moe_forward_int8(*on_gpu(a), 2), a, 2)


@pytest.mark.parametrize("T", [5, 40])
def test_a_token_without_logits_and_tokens_that_are_not_finite(ops, T):
    a = list(make(T, 8, 128, 64, torch.bfloat16, 3))
    good = ops.moe_forward_int8(*on_gpu(a), 2)
    a[1][1, 3] = float("nan")
    a[0][2, 5] = float("inf")
    out = ops.moe_forward_int8(*on_gpu(a), 2)
    assert (out[1] == 0).all() and torch.isnan(out[2]).all()
    keep = [i for i in range(T) if i not in (1, 2)]
    assert torch.equal(out[keep], good[keep])


@pytest.mark.parametrize("T,I,fewer", [(16, 64, (1, 3, 9)), (60, 272, (1, 2, 17, 20, 33, 59)), (16, 272, (1, 3, 9))])
def test_a_layer_is_repeatable_and_a_token_does_not_see_the_others(ops, T, I, fewer):
    """Integer sums, slots added in order: the same bits whatever shares the batch, in one kernel or several."""
    a = on_gpu(make(T, 64, 512, I, torch.bfloat16, 11))
    out = ops.moe_forward_int8(*a, 6)
    for _ in range(20):
        assert torch.equal(ops.moe_forward_int8(*a, 6), out)
    for n in fewer:
        assert torch.equal(ops.moe_forward_int8(a[0][:n].contiguous(), a[1][:n].contiguous(), *a[2:], 6), out[:n])


def test_few_tokens_take_one_kernel(ops):
    a = on_gpu(make(16, 128, 256, 64, torch.bfloat16, 1))
    before = ops.launch_count()
    ops.moe_forward_int8(*a, 8)
    assert ops.launch_count() - before == 1 and ops.last_kernel() == "moe_i8"


@pytest.mark.parametrize("T", [2, 40])
def test_weights_of_more_than_4_gb(ops, T):
    E, H, I, used = 520, 2048, 2048, [3, 519]
    a = make(T, 2, H, I, torch.bfloat16, T)
    assert one_kernel(T, 2, H, I) == (T == 2)
    whole = []
    for t in a[2:]:
        v = torch.zeros(E, *t.shape[1:], dtype=t.dtype, device=DEV)
        v[used] = t.to(DEV)
        whole.append(v)
    assert whole[0].numel() > 2 ** 32
    logits = torch.full((T, E), -50.0)
    logits[:, used] = a[1]
    check(ops.moe_forward_int8(a[0].to(DEV), logits.to(DEV), *whole, 2), a, 2)


@pytest.mark.parametrize("mode", [0, 1])
@pytest.mark.parametrize("T", [2, 16, 60, 300])
def test_weights_written_right_before_the_layer(ops, T, mode):
    """Only overlap mode 2 declares weights static: before it, a layer sees what the kernel in front of it has written."""
    sets = [on_gpu(make(T, 16, 512, 256, torch.bfloat16, seed)) for seed in (7, 8)]
    x, logits = sets[0][:2]
    ops.set_overlap_mode(0)
    refs = [ops.moe_forward_int8(x, logits, *a[2:], 4) for a in sets]
    assert not torch.equal(*refs)
    ops.set_overlap_mode(mode)
    now = [t.clone() for t in sets[0][2:]]
    for i in range(30):
        for t, v in zip(now, sets[i % 2][2:]):
            t.copy_(v)
        assert torch.equal(ops.moe_forward_int8(x, logits, *now, 4), refs[i % 2])
    ops.set_overlap_mode(1)


@pytest.mark.parametrize("mode", [0, 1, 2])
@pytest.mark.parametrize("T", [1, 16, 60])
def test_layers_behind_one_another(ops, T, mode):
    """x and the logits of a layer come from the kernel right in front of it; eager, on another stream, and replayed."""
    a = on_gpu(make(T, 32, 256, 192, torch.bfloat16, 5))
    wr = torch.randint(-127, 128, (32, 256), dtype=torch.int8, device=DEV)
    sr = torch.full((32,), 2e-3, device=DEV)

    def chain():
        x = a[0]
        for _ in range(5):
            x = ops.moe_forward_int8(x, ops.linear_int8_dynamic(x, wr, sr), *a[2:], 4)
            x = (x.float() / x.float().abs().amax(1, keepdim=True).clamp(min=1e-6)).to(x.dtype)
            x = ops.moe_forward_int8(x, ops.linear_int8_dynamic(x, wr, sr), *a[2:], 4)
        return x

    torch.cuda.synchronize()
    ops.set_overlap_mode(0)
    ref = chain()
    torch.cuda.synchronize()
    ops.set_overlap_mode(mode)
    st = torch.cuda.Stream()
    with torch.cuda.stream(st):
        for _ in range(10):
            assert torch.equal(chain(), ref)
    st.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y = chain()
    for _ in range(5):
        y.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, ref)
    ops.set_overlap_mode(1)


def test_scratch_may_hold_anything(ops):
    """A workspace full of any byte, and of what an earlier layer of other sizes left there."""
    L = ops._lib
    a = on_gpu(make(9, 24, 256, 128, torch.float16, 2))
    x, logits, w13, s13, w2, s2 = a
    ref = ops.moe_forward_int8(*a, 3)
    need = L.lib.b2q_moe_forward_int8_workspace_bytes(9, 24, 3, 256, 128)
    ws = torch.empty(need + 256, dtype=torch.uint8, device=DEV)
    base = (ws.data_ptr() + 255) // 256 * 256
    for fill in (0, 255, 1, None):
        if fill is not None:
            ws.fill_(fill)
        out = torch.zeros_like(ref)
        m = L.MoeInt8(x=x.data_ptr(), logits=logits.data_ptr(), w13=w13.data_ptr(), s13=s13.data_ptr(), w2=w2.data_ptr(), s2=s2.data_ptr(), out=out.data_ptr(),
                      T=9, E=24, top_k=3, H=256, I=128, act_dtype=L.F16, logits_dtype=L.F32, s13_dtype=L.F32, s2_dtype=L.F32, renormalize=1)
        assert L.lib.b2q_moe_forward_int8(m, base, need, L.stream(x)) == 0
        assert torch.equal(out, ref)


def test_refusals(ops):
    x, logits, w13, s13, w2, s2 = a = on_gpu(make(4, 8, 64, 32, torch.bfloat16, 0))
    before = ops.launch_count()
    for i, bad in [(0, x.float()), (0, x[:3]), (0, x[0]), (1, logits[:, :7].contiguous()), (1, logits.double()), (2, w13.float()), (2, w13[:, :, :32]), (2, w13[:, :63].contiguous()),
                   (3, s13[:7]), (4, w2.transpose(1, 2)), (4, w2[:7].contiguous()), (5, s2[:, :3].contiguous()), (5, s2.double()), (0, x.cpu())]:
        args = list(a)
        args[i] = bad
        with pytest.raises(RuntimeError):
            ops.moe_forward_int8(*args, 2)
    for k in (0, 9, -1):
        with pytest.raises(RuntimeError):
            ops.moe_forward_int8(*a, k)
    odd = on_gpu(make(4, 8, 72, 32, torch.bfloat16, 0))
    with pytest.raises(RuntimeError):
        ops.moe_forward_int8(*odd, 2)
    assert ops.launch_count() == before
    assert ops.moe_forward_int8(x[:0], logits[:0], w13, s13, w2, s2, 2).shape == (0, 64)
