"""How much scratch the 4-bit expert layer asks for.  No GPU needed."""
import pytest


@pytest.mark.parametrize("T,E,k,H,I", [(49, 8, 8, 256, 4096), (400, 1024, 1, 128, 2048), (41, 8, 1, 512, 8192), (4096, 128, 8, 2048, 768), (8192, 64, 8, 4096, 14336), (300, 5, 4, 640, 160)])
def test_many_tokens_ask_for_nothing_of_the_form_of_few(lib_built, T, E, k, H, I):
    """More than 384 pairs, or than five per expert: a row of x, of h and of the outputs in 16 bits for each pair, its place and weight, and the lists of experts and tiles."""
    from custom_esimd_kernels_vllm import _lib as L
    pairs = T * k
    assert pairs > min(384, 5 * E)
    got = L.lib.b2q_moe_forward_w4_workspace_bytes(T, E, k, H, I)
    least = pairs * (2 * H + 2 * I + 2 * H)
    assert least <= got <= least + 13 * pairs + 300 * E + 8192


@pytest.mark.parametrize("T,E,k,H,I", [(48, 128, 8, 2048, 768), (40, 8, 1, 512, 8192), (1, 8, 2, 256, 128)])
def test_few_tokens_may_be_served_by_either_form(lib_built, T, E, k, H, I):
    from custom_esimd_kernels_vllm import _lib as L
    pairs = T * k
    got = L.lib.b2q_moe_forward_w4_workspace_bytes(T, E, k, H, I)
    assert got >= max(pairs * (2 * I + I // 4 + 4 * H), pairs * (2 * I + 4 * H))
