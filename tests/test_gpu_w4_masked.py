"""Expert routing where experts are masked: groups with one expert left or none, by logits and by the bias, at every width of the kernel."""
import math

import pytest
import torch

from test_gpu_w4 import check_route, gen
from w4_util import DT

pytestmark = pytest.mark.gpu
INF = math.inf
# groups of 32 at each width of the kernel (up to 64, 128, 256, 512, 1024 experts), full and not, and of other sizes
WIDTHS = [(64, 2), (96, 3), (128, 4), (160, 5), (256, 8), (384, 12), (512, 16), (1024, 32), (8, 4), (60, 4), (96, 6), (250, 5), (512, 32), (18, 9)]


def some_left(E, groups):
    """Rows of normal logits: each group with one expert left; the first alone with one, the best of all, or the worst; every second with one; two groups of one expert each and no
    others; one expert in all; two left in each; nothing masked."""
    size, g = E // groups, gen(E + groups)
    l = 1.5 * torch.randn(9, E, generator=g)
    of = torch.arange(E) // size
    one = torch.arange(E) % size == (of * 7 + 1) % size      # one expert of each group
    l[0, ~one] = -INF
    l[1:3, (of == 0) & ~one] = -INF
    l[1, (of == 0) & one], l[2, (of == 0) & one] = 8.0, -8.0
    l[3, (of % 2 == 1) & ~one] = -INF
    l[4, ~(one & (of >= groups - 2))] = -INF
    l[5, ~(one & (of == groups // 2))] = -INF
    l[6, ~(one | one.roll(1))] = -INF
    l[7, (of > 0) & ~one] = -INF
    return l


@pytest.mark.parametrize("E,groups", WIDTHS)
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("dt", list(DT) + ["fp32"])
def test_groups_with_one_expert_left(E, groups, scoring, dt):
    l, bias = some_left(E, groups).to({**DT, "fp32": torch.float32}[dt]), 0.3 * torch.randn(E, generator=gen(E))
    out = bias.clone()      # the bias leaves one in the second group, none in the third
    of = torch.arange(E) // (E // groups)
    out[(of == 1) & (torch.arange(E) % (E // groups) != 0)] = -INF
    out[of == 2] = math.nan
    for b in (None, bias, out):
        for top in sorted({1, groups // 2, groups - 1, groups}):
            for score in ("top2", "max"):
                check_route(l, min(8, top * (E // groups)), scoring=scoring, bias=b, num_groups=groups, top_groups=top, group_score=score)


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("bt", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("E,groups", [(16, 4), (128, 4), (60, 6)])
def test_biases_of_the_types_lowest_value(E, groups, scoring, bt):
    """They put an expert behind all others but do not take it out, two in a group neither, whose sum fp32 does not hold."""
    size, low = E // groups, torch.finfo(bt).min
    l = torch.randn(5, E, generator=gen(1))
    for left in range(groups):      # groups whose biases are ordinary
        bias = torch.full((E,), low, dtype=bt)
        bias[:left * size] = (0.2 * torch.randn(left * size, generator=gen(2))).to(bt)
        bias[-size:-1] = -INF       # and one expert of the last group
        for top in range(1, groups + 1):
            for score in ("top2", "max"):
                check_route(l, min(6, top * size), scoring=scoring, bias=bias, num_groups=groups, top_groups=top, group_score=score)


def test_sigmoids_that_are_not_renormalised():
    """Without a bias, at the edges: masked rows, scores that underflow and scores that round to one."""
    l = torch.randn(10, 64, generator=gen(7))
    l[1, 3:] = -INF
    l[2] = -INF
    l[3] = -300 + torch.arange(64) / 64.0
    l[4] = 40 + torch.arange(64) % 3
    l[5] = torch.finfo(torch.float32).min
    l[6] = torch.finfo(torch.float32).max
    l[7] = -80 - torch.arange(64) / 8.0
    l[8, 1], l[9, 1] = math.nan, INF
    for kw in ({}, dict(num_groups=8, top_groups=3), dict(num_groups=8, top_groups=3, group_score="top2"), dict(num_groups=2, top_groups=1, group_score="top2")):
        check_route(l, 6, scoring="sigmoid", renormalize=False, scale=2.0, **kw)
