"""Scratch of the int8 expert layer on both sides of the second condition of its one-kernel form (24 KB of a CTA's sums).  No GPU needed: the library
assumes 148 SMs where it sees none."""
import os
import re

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.mark.parametrize("k,few", [(27, True), (28, False), (32, False)])
def test_scratch_follows_both_conditions(lib_built, k, few):
    from custom_esimd_kernels_vllm import _lib as L
    T, H, I = 1, 32768, 16
    assert T * (4 * k * I + H) <= 40960 and (T * k * 222 * 4 <= 24 * 1024) == few
    got = L.lib.b2q_moe_forward_int8_workspace_bytes(T, 32, k, H, I)
    assert (got < k * H) == few                                # the grouped form keeps codes of x for every pair


def test_the_header_states_both():
    with open(os.path.join(ROOT, "include", "b2q.h")) as f:
        text = " ".join(re.sub(r"\n \*", "\n", f.read()).split())
    assert "T (4 top_k I + H) <= 40960 and T top_k ceil(H / SMs) <= 6144" in text


def test_scratch_of_the_grouped_form_on_request(lib_built):
    from custom_esimd_kernels_vllm import _lib as L
    f = L.lib.b2q_moe_forward_int8_workspace_bytes
    shape = (1, 128, 8, 2048, 768)
    few = f(*shape)
    L.lib.b2q_set_force_kernel(2)
    try:
        assert f(*shape) >= few + 8 * 2048
    finally:
        L.lib.b2q_set_force_kernel(0)
    assert f(*shape) == few
