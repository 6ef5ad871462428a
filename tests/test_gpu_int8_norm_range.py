"""The residual-norm quantiser on finite rows whose sum of squares fp32 does not hold: the same scale and codes as of any other row."""
import pytest
import torch

from gpu_util import DEV
from oracle import int8
from test_gpu_int8 import near, ops  # noqa: F401

pytestmark = pytest.mark.gpu

FORMS = [(200, 64), (200, 1024), (3, 5120), (149, 8192), (300, 2048), (2, 16384), (1, 32768), (2, 77), (1, 32776)]      # a warp or a CTA per row; element by element


@pytest.mark.parametrize("M,K", FORMS)
@pytest.mark.parametrize("scale", [1e15, 1e18, 2e19, 1e25, 1e30, 1e37])
def test_huge_rows(ops, M, K, scale):  # noqa: F811
    g = torch.Generator().manual_seed(K)
    h, r = ((torch.randn(M, K, generator=g) * scale).bfloat16() for _ in range(2))
    w = (1 + 0.2 * torch.randn(K, generator=g)).bfloat16()
    rd = r.to(DEV)
    q, s = ops.resadd_rmsnorm_quantize_int8(h.to(DEV), rd, w.to(DEV), 1e-5)
    near(q, s, int8.resadd_rmsnorm(h, r, w, 1e-5)[1], 127 * 8 * 2.0 ** -24, 64 * 2.0 ** -24)
    assert torch.equal(rd.cpu(), (h.float() + r.float()).bfloat16())


@pytest.mark.parametrize("M,K", FORMS)
def test_rows_of_all_sizes_beside_one_another(ops, M, K):  # noqa: F811
    """Ordinary rows keep their bits whatever stands beside them; in the others a few values are huge, or each of another size."""
    g = torch.Generator().manual_seed(K + 1)
    h, r = torch.randn(M, K, generator=g).bfloat16(), torch.randn(M, K, generator=g).bfloat16()
    w = (1 + 0.2 * torch.randn(K, generator=g)).bfloat16()
    plain = [t.cpu() for t in ops.resadd_rmsnorm_quantize_int8(h.to(DEV), r.to(DEV), w.to(DEV), 1e-5)]
    h[0::4, K // 3] = 3e38
    h[0::4, K - 1] = -2e30
    h[1::4] = (h[1::4].float() * 10 ** torch.linspace(-30, 36, K)).bfloat16()
    h[2::4, 5] = float("inf")
    r[0::4, K // 3] = 0
    q, s = ops.resadd_rmsnorm_quantize_int8(h.to(DEV), r.to(DEV), w.clamp(max=1).to(DEV), 1e-5)
    n = int8.resadd_rmsnorm(h, r, w.clamp(max=1), 1e-5)[1]
    keep = [i for i in range(M) if i % 4 < 2]
    near(q[keep], s[keep], n[keep], 127 * 8 * 2.0 ** -24, 64 * 2.0 ** -24)
    assert torch.isnan(s[2::4]).all() and (q[2::4] == 0).all()
    q, s = ops.resadd_rmsnorm_quantize_int8(h.to(DEV), r.to(DEV), w.to(DEV), 1e-5)
    assert torch.equal(q[3::4].cpu(), plain[0][3::4]) and torch.equal(s[3::4].cpu(), plain[1][3::4])


@pytest.mark.parametrize("M,K", FORMS)
def test_huge_rows_under_weights_of_zero(ops, M, K):  # noqa: F811
    """Where the weight is 0, v enters the sum of squares as residual_out has it, in 16 bits; everything else in fp32."""
    g = torch.Generator().manual_seed(K + 2)
    h, r = ((torch.randn(M, K, generator=g) * 1e25).bfloat16() for _ in range(2))
    w = (1 + 0.2 * torch.randn(K, generator=g)).bfloat16()
    w[torch.randperm(K, generator=g)[:K // 3]] = 0
    v = h.double() + r.double()
    if K % 8 == 0 and K <= 32768:                            # the others are read twice, and exact
        v = torch.where(w == 0, (h.float() + r.float()).bfloat16().double(), v)
    n = v / torch.sqrt((v * v).mean(1, keepdim=True) + 1e-5) * w.double()
    q, s = ops.resadd_rmsnorm_quantize_int8(h.to(DEV), r.to(DEV), w.to(DEV), 1e-5)
    near(q, s, n, 127 * 8 * 2.0 ** -24, 64 * 2.0 ** -24)


def test_the_values_written_are_read_back_behind_the_writes():
    """What a thread reads back there goes by volatile loads, which the compiler orders among themselves only."""
    import os
    import re
    src = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "llm-scaler_b200", "csrc", "i8_quant.cu")
    with open(src) as f:
        body = re.sub(r"//[^\n]*", "", f.read()).split("if (!(sum < INFINITY)) {")[1].split("residual_out")[0]
    assert "__syncwarp();" in body
