"""8-bit integer operators against their definition in 64 bits (oracle/int8.py).

Tolerances.  Codes of stored values are exact.  A linear's output is an exact integer times two fp32 scales, each product rounded once, plus
a bias: within 2^-21 of the addends.  Rounding is monotone, so the 16-bit output lies between the rounded ends of that interval.
Codes of computed rows (SiLU * mul, RMSNorm) are within half a step and the fp32 error of the value in front of the rounding: SiLU's
exponential is good to 21 units of 2^-23 for |gate| <= 16, the norm's sum of squares to 60 of 2^-24."""
import pytest
import torch

from gpu_util import DEV
from oracle import int8

pytestmark = pytest.mark.gpu

DTS = [torch.bfloat16, torch.float16]


@pytest.fixture(scope="module")
def ops(lib_built):
    import custom_esimd_kernels_vllm as e
    yield e
    e.set_overlap_mode(1)
    assert e._lib.device_status() == 0


def check_linear(out, codes, scale, w, ws, bias=None):
    prod = int8.linear(codes, scale, w, ws)
    b = torch.zeros(w.shape[0], dtype=torch.float64) if bias is None else bias.double()
    ref = prod + b
    tol = 2.0 ** -21 * (prod.abs() + b.abs())
    lo, hi = (ref - tol).to(out.dtype).double(), (ref + tol).to(out.dtype).double()
    bad = (out.cpu().double() < lo) | (out.cpu().double() > hi)
    assert not bad.any(), (int(bad.sum()), bad.numel(), torch.nonzero(bad)[:4].tolist())


def make_linear(M, N, K, seed, full=False):
    g = torch.Generator().manual_seed(seed)
    lo, hi = (-128, 128) if full else (-127, 128)
    codes = torch.randint(lo, hi, (M, K), generator=g, dtype=torch.int8)
    w = torch.randint(lo, hi, (N, K), generator=g, dtype=torch.int8)
    return codes, torch.rand(M, generator=g) * 0.05 + 0.001, w, torch.rand(N, generator=g) * 0.002 + 1e-4, torch.randn(N, generator=g)


# ------------------------------------------------------------------------------------------------------------ quantiser
@pytest.mark.parametrize("dt", DTS + [torch.float32])
@pytest.mark.parametrize("M,K,pitch", [(1, 1, 1), (1, 7, 7), (3, 8, 8), (1, 5120, 5120), (5, 333, 340), (4, 1000, 1000), (300, 256, 264), (200, 512, 512), (160, 1000, 1008),
                                       (149, 2056, 2056), (7, 8192, 10240), (150, 8192, 8200), (2, 28672, 28672), (149, 28672, 28672), (2, 32776, 32776), (3, 4099, 4099)])
def test_rows_to_codes_are_exact(ops, dt, M, K, pitch):
    g = torch.Generator().manual_seed(K + M)
    x = torch.randn(M, pitch, generator=g).to(dt)
    x[:, 0] = x[:, 0] * 8
    if M > 2:
        x[1] = 0
    wide = x.to(DEV)
    q, s = ops.quantize_int8(wide[:, :K])
    rq, _, rs = int8.quantize_rows(x[:, :K])
    assert q.shape == (M, K) and q.dtype == torch.int8 and s.dtype == torch.float32
    assert torch.equal(q.cpu(), rq)
    a = x[:, :K].float().abs().amax(1).clamp(min=int8.MIN_AMAX)
    assert torch.equal(s.cpu(), a / torch.full_like(a, 127.0))


@pytest.mark.parametrize("dt", DTS + [torch.float32])
def test_halves_go_to_even(ops, dt):
    """amax 127 * 2^e: every x = (k + 1/2) 2^e is an exact half, and half of the largest value is one whatever the largest is."""
    k = torch.arange(-127, 127, dtype=torch.float32) + 0.5
    for e in (-20, -6, 0, 6):
        row = torch.cat([torch.tensor([127.0]), k]) * 2.0 ** (0 if dt == torch.float16 and e == -20 else e)
        q, _ = ops.quantize_int8(row.to(dt)[None].to(DEV))
        assert torch.equal(q.cpu(), int8.quantize_rows(row.to(dt)[None])[0])
    top = torch.linspace(0.5, 3.0, 997).to(dt)
    rows = torch.stack([top, top / 2, -top / 2, top * 0.25], 1)
    rows = torch.nn.functional.pad(rows, (0, 4))
    for r in (rows, rows[:, :4].contiguous()):
        q, _ = ops.quantize_int8(r.to(DEV))
        assert torch.equal(q.cpu(), int8.quantize_rows(r)[0])
    assert set(q.cpu()[:, 1].tolist()) == {64}


@pytest.mark.parametrize("K", [64, 67])
def test_extreme_rows(ops, K):
    x = torch.randn(8, K, dtype=torch.float32)
    x[0] *= 1e30; x[1] *= 1e-30; x[2, 3] = 3.3e38; x[3] = 1e-12; x[4, 1] = float("inf"); x[5, 2] = float("nan"); x[6] = 0; x[7, 5] = -float("inf")
    x = x.bfloat16()
    q, s = ops.quantize_int8(x.to(DEV))
    rq, _, rs = int8.quantize_rows(x)
    assert torch.equal(q.cpu(), rq)
    assert torch.equal(torch.isnan(s.cpu()), torch.isnan(rs)) and torch.isnan(rs).tolist() == [i in (4, 5, 7) for i in range(8)]
    ok = ~torch.isnan(rs)
    assert ((s.cpu().double() - rs).abs()[ok] <= 2.0 ** -23 * rs[ok]).all()
    # and whatever is made from such a row is NaN
    if K % 16 == 0:
        w = torch.ones(8, K, dtype=torch.int8, device=DEV)
        out = ops.linear_int8(q, s, w, torch.ones(8, device=DEV))
        assert torch.isnan(out).all(1).cpu().tolist() == [i in (4, 5, 7) for i in range(8)]
        out = ops.linear_int8_dynamic(x.to(DEV), w, torch.ones(8, device=DEV))
        assert torch.isnan(out).all(1).cpu().tolist() == [i in (4, 5, 7) for i in range(8)]


def near(q, s, value, code_tol, scale_tol):
    _, t, rs = int8.quantize_rows(value)
    assert ((q.cpu().double() - t).abs() <= 0.5 + code_tol).all()
    assert ((s.cpu().double() - rs).abs() <= scale_tol * rs).all()


@pytest.mark.parametrize("dt", DTS)
@pytest.mark.parametrize("M,K,extra", [(1, 8, 0), (3, 13824, 0), (5, 129, 3), (160, 768, 0), (149, 1536, 16), (150, 28672, 0), (2, 40000, 0), (1, 16384, 0)])
def test_silu_mul_quantize(ops, dt, M, K, extra):
    g = torch.Generator().manual_seed(K)
    x = (torch.randn(M, 2 * K + extra, generator=g) * 3).clamp(-16, 16).to(dt)
    gu = x.to(DEV)[:, :2 * K]
    q, s = ops.silu_mul_quantize_int8(gu)
    near(q, s, int8.silu_mul(x[:, :2 * K]), 127 * 2 * 25 * 2.0 ** -23, 25 * 2.0 ** -23)


@pytest.mark.parametrize("dt", DTS)
@pytest.mark.parametrize("in_place", [True, False])
@pytest.mark.parametrize("M,K", [(1, 16), (3, 5120), (2, 77), (200, 1024), (2048, 512), (149, 8192), (151, 28672), (1, 32776)])
def test_resadd_rmsnorm_quantize(ops, dt, in_place, M, K):
    g = torch.Generator().manual_seed(K)
    h, r = torch.randn(M, K, generator=g).to(dt), torch.randn(M, K, generator=g).to(dt)
    w = (1 + 0.2 * torch.randn(K, generator=g)).to(dt)
    rd = r.to(DEV)
    ro = rd if in_place else torch.empty_like(rd)
    q, s = ops.resadd_rmsnorm_quantize_int8(h.to(DEV), rd, w.to(DEV), 1e-5, None if in_place else ro)
    v, n = int8.resadd_rmsnorm(h, r, w, 1e-5)
    near(q, s, n, 127 * 8 * 2.0 ** -24, 64 * 2.0 ** -24)
    assert torch.equal(ro.cpu(), (h.float() + r.float()).to(dt))
    if not in_place:
        assert torch.equal(rd.cpu(), r)


def test_a_row_of_zeros_and_a_row_of_nothing_finite(ops):
    h = torch.zeros(3, 64, dtype=torch.bfloat16)
    h[1, 4] = float("nan")
    h[2] = 1
    q, s = ops.resadd_rmsnorm_quantize_int8(h.to(DEV), torch.zeros_like(h).to(DEV), torch.ones(64, dtype=torch.bfloat16, device=DEV), 1e-6)
    assert q[0].abs().max() == 0 and q[1].abs().max() == 0 and (q[2] == 127).all()
    assert torch.isnan(s).tolist() == [False, True, False]
    gu = torch.zeros(2, 128, dtype=torch.float16)
    gu[1, 70] = float("inf"); gu[1, 6] = 1.0
    q, s = ops.silu_mul_quantize_int8(gu.to(DEV))
    assert q.abs().max() == 0 and torch.isnan(s).tolist() == [False, True]


# --------------------------------------------------------------------------------------------------------------- linear
SHAPES = [(1, 1, 16), (1, 2048, 2048), (2, 7, 48), (3, 300, 272), (8, 5000, 512), (9, 129, 1040), (15, 2368, 4096), (16, 1000, 144), (16, 296, 28672), (1, 9473, 64),
          (17, 1, 16), (17, 129, 272), (27, 4352, 1280), (32, 100, 4096), (33, 2048, 2048), (64, 513, 640), (65, 1000, 1040), (100, 4096, 128), (128, 255, 9216),
          (129, 777, 528), (200, 2304, 384), (256, 256, 4096), (257, 2600, 256), (300, 9000, 144), (513, 5121, 400), (1025, 4100, 272), (700, 16, 2048)]


@pytest.mark.parametrize("M,N,K", SHAPES)
@pytest.mark.parametrize("dt", DTS)
def test_linear(ops, M, N, K, dt):
    codes, s, w, ws, b = make_linear(M, N, K, M + N + K, full=True)
    b = b.to(dt)
    if (M + N) % 3 == 0:
        b = None
    sdt = [torch.float32, torch.bfloat16, torch.float16][(M + K // 16) % 3]
    ws = ws.to(sdt)
    out = ops.linear_int8(codes.to(DEV), s.to(DEV), w.to(DEV), ws.to(DEV), None if b is None else b.to(DEV), dt)
    assert out.shape == (M, N) and out.dtype == dt
    check_linear(out, codes, s, w, ws, b)


@pytest.mark.parametrize("M,N,K", SHAPES)
def test_dynamic_is_quantise_and_linear(ops, M, N, K):
    g = torch.Generator().manual_seed(M * N)
    dt = DTS[M % 2]
    x = torch.randn(M, K, generator=g).to(dt)
    if M > 4:
        x[3] = 0
    _, _, w, ws, b = make_linear(1, N, K, K)
    args = (w.to(DEV), ws.to(DEV), b.to(dt).to(DEV))
    out = ops.linear_int8_dynamic(x.to(DEV), *args)
    q, s = ops.quantize_int8(x.to(DEV))
    assert torch.equal(out, ops.linear_int8(q, s, *args, dt))
    rq, _, rs = int8.quantize_rows(x)
    check_linear(out, rq, rs, w, ws, b.to(dt))


@pytest.mark.parametrize("M", [5, 40, 600])
def test_strided_inputs_and_outputs_of_every_form(ops, M):
    N, K = 300, 256
    codes, s, w, ws, _ = make_linear(M, N, K + 64, M)
    wide = codes.to(DEV)
    wk = w[:, :K].contiguous()
    out = ops.linear_int8(wide[:, 32:32 + K], s.to(DEV), wk.to(DEV), ws.to(DEV))
    check_linear(out, codes[:, 32:32 + K], s, wk, ws)
    x = torch.randn(M, K + 9).half()
    d = ops.linear_int8_dynamic(x.to(DEV)[:, 3:3 + K], wk.to(DEV), ws.to(DEV))      # rows that are not 16-byte aligned
    q, _, r = int8.quantize_rows(x[:, 3:3 + K])
    check_linear(d, q, r, wk, ws)


@pytest.mark.parametrize("M", [1, 16, 17, 64, 300])
def test_largest_sums_do_not_overflow(ops, M):
    K, N = 131056, 40
    codes = torch.full((M, K), -128, dtype=torch.int8)
    w = torch.full((N, K), -128, dtype=torch.int8)
    s, ws = torch.full((M,), 1e-5), torch.full((N,), 1e-5)
    out = ops.linear_int8(codes.to(DEV), s.to(DEV), w.to(DEV), ws.to(DEV))
    check_linear(out, codes, s, w, ws)


@pytest.mark.parametrize("mode", [0, 1, 2])
def test_overlap_modes_streams_and_graphs(ops, mode):
    """A chain of all three operators, its codes made right in front of the linear that reads them, on a stream of its own and replayed."""
    ops.set_overlap_mode(mode)
    for M in (3, 40, 300):
        x = torch.randn(M, 1024).bfloat16().to(DEV)
        w = torch.randint(-127, 128, (2048, 1024), dtype=torch.int8, device=DEV)
        w2 = torch.randint(-127, 128, (1024, 1024), dtype=torch.int8, device=DEV)
        ws, ws2 = torch.full((2048,), 1e-3, device=DEV), torch.full((1024,), 1e-3, device=DEV)

        def chain():
            y = x
            for _ in range(4):
                q, s = ops.silu_mul_quantize_int8(ops.linear_int8_dynamic(y, w, ws))
                y = ops.linear_int8(q, s, w2, ws2)
            return y

        torch.cuda.synchronize()
        ops.set_overlap_mode(0)
        ref = chain()
        ops.set_overlap_mode(mode)
        torch.cuda.synchronize()
        st = torch.cuda.Stream()
        with torch.cuda.stream(st):
            for _ in range(10):
                assert torch.equal(chain(), ref)
        g = torch.cuda.CUDAGraph()
        st.synchronize()
        with torch.cuda.graph(g):
            y = chain()
        for _ in range(5):
            y.zero_()
            g.replay()
            torch.cuda.synchronize()
            assert torch.equal(y, ref)
    ops.set_overlap_mode(1)


def test_empty_batches(ops):
    w, ws = torch.zeros(32, 64, dtype=torch.int8, device=DEV), torch.ones(32, device=DEV)
    q, s = ops.quantize_int8(torch.empty(0, 64, dtype=torch.float16, device=DEV))
    assert q.shape == (0, 64) and s.shape == (0,)
    assert ops.linear_int8(q, s, w, ws).shape == (0, 32)
    assert ops.linear_int8_dynamic(torch.empty(0, 64, dtype=torch.float16, device=DEV), w, ws).shape == (0, 32)
    assert ops.silu_mul_quantize_int8(torch.empty(0, 64, dtype=torch.float16, device=DEV))[0].shape == (0, 32)


def test_offsets_beyond_32_bits(ops):
    """Rows and outputs of more than 2^31 elements: every block of rows like the first."""
    g = torch.Generator().manual_seed(2)
    x = torch.randn(1000, 32768, generator=g).bfloat16().to(DEV)
    q, s = ops.quantize_int8(x)
    many_q, many_s = ops.quantize_int8(x.repeat(70, 1))
    assert many_q.numel() > 2 ** 31
    assert (many_q.view(70, 1000, -1) == q).all() and (many_s.view(70, 1000) == s).all()
    del many_q, many_s
    many_q, many_s = ops.silu_mul_quantize_int8(x.repeat(135, 1))
    q, s = ops.silu_mul_quantize_int8(x)
    assert many_q.numel() > 2 ** 31 and (many_q.view(135, 1000, -1) == q).all() and (many_s.view(135, 1000) == s).all()
    del many_q, many_s
    codes, scale, w, ws, _ = [t.to(DEV) for t in make_linear(1000, 16384, 64, 3)]
    out = ops.linear_int8(codes, scale, w, ws)
    many = ops.linear_int8(codes.repeat(140, 1), scale.repeat(140), w, ws)
    assert many.numel() > 2 ** 31 and (many.view(140, 1000, -1) == out).all()


def test_refusals(ops):
    q, s = torch.zeros(4, 64, dtype=torch.int8, device=DEV), torch.ones(4, device=DEV)
    w, ws = torch.zeros(32, 64, dtype=torch.int8, device=DEV), torch.ones(32, device=DEV)
    x = torch.zeros(4, 64, dtype=torch.float16, device=DEV)
    before = ops.launch_count()
    for args in [(q.float(), s, w, ws), (q, s[:3], w, ws), (q, s.half(), w, ws), (q, s, w.float(), ws), (q, s, w.t(), ws), (q, s, w[:, :32], ws),
                 (q, s, w, ws[:5]), (q, s, w, ws.double()), (q[:, :40], s, w[:, :40].contiguous(), ws), (q, s, w, ws, ws), (q, s, w, ws, None, torch.float32),
                 (q.t(), s, w, ws), (q.cpu(), s, w, ws), (q[0], s, w, ws)]:
        with pytest.raises(RuntimeError):
            ops.linear_int8(*args)
    for args in [(x.float(), w, ws), (x, w, ws[:3]), (x[0], w, ws), (x, w.cpu(), ws), (x, w, ws, torch.zeros(32, device=DEV))]:
        with pytest.raises(RuntimeError):
            ops.linear_int8_dynamic(*args)
    for bad in (x.double(), x[0], x.t(), x.cpu(), x[:, :0]):
        with pytest.raises((RuntimeError, NotImplementedError)):
            ops.quantize_int8(bad)
    with pytest.raises(RuntimeError):
        ops.silu_mul_quantize_int8(x[:, :7])
    with pytest.raises(RuntimeError):
        ops.resadd_rmsnorm_quantize_int8(x, x[:3], x[0].contiguous(), 1e-6)
    with pytest.raises(RuntimeError):
        ops.resadd_rmsnorm_quantize_int8(x, x, x[0, :8].contiguous(), 1e-6)
    assert ops.launch_count() == before
