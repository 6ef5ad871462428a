"""Sizes next to 2^31: the quantisers' columns are counted in steps of 512, the linears' rows in tiles, and neither count may pass the largest
int.  Refused before any launch; no GPU needed."""
import re
import os

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "llm-scaler_b200", "csrc")
P = 1 << 20      # an address that nothing reads
TOP = (1 << 31) - 1


@pytest.fixture(scope="module")
def L(lib_built):
    from custom_esimd_kernels_vllm import _lib
    return _lib


@pytest.mark.parametrize("K", [TOP, TOP - 511])
def test_quantisers_refuse_columns_whose_count_would_overflow(L, K):
    with open(os.path.join(CSRC, "i8_quant.cu")) as f:
        steps = set(re.findall(r"for \(int c = threadIdx\.x; c < p\.K; c \+= (\d+)\)", f.read()))
    assert steps == {"512"}                                   # K - 1 + 512 is the last value of such a count
    before = L.launch_count()
    assert L.lib.b2q_quantize_int8(P, 0, K, P, P, 1, K, None) == -10
    assert L.lib.b2q_resadd_rmsnorm_quantize_int8(P, P, P, P, 0, 1e-6, P, P, 1, K, None) == -10
    assert L.launch_count() == before


@pytest.mark.parametrize("size", [dict(M=TOP), dict(M=TOP - 4094), dict(N=TOP, ldo=TOP), dict(N=TOP - 4094, ldo=TOP)])
def test_linears_refuse_rows_whose_tiles_would_overflow(L, size):
    a = dict(M=1, N=32, K=32, ldo=32)
    a.update(size)
    before = L.launch_count()
    assert L.lib.b2q_linear_int8(P, a["K"], P, P, P, 2, None, P, 0, a["ldo"], a["M"], a["N"], a["K"], None) == -10
    assert L.lib.b2q_linear_int8_dynamic(P, 0, a["K"], P, P, 2, None, P, a["ldo"], a["M"], a["N"], a["K"], P, 1 << 50, None) == -10
    assert L.launch_count() == before
