"""The oracle's choice of groups with masked experts, worked out by hand.  No GPU needed."""
import math

import pytest
import torch

from oracle import w4

OUT = -math.inf


@pytest.mark.parametrize("logits,bias,k,top,want", [
    # groups of two by their sums: one expert left counts for itself, sigmoid(5) = 0.993 < 2 sigmoid(0) = 1
    ([5, OUT, 0, 0, OUT, OUT, OUT, OUT], None, 2, 2, [0, 2]), ([5, OUT, 0, 0, OUT, OUT, OUT, OUT], None, 3, 2, [0, 2, 3]), ([5, OUT, 0, 0, OUT, OUT, OUT, OUT], None, 2, 1, [2, 3]),
    # 0.95, 0.54, 0.50, 0.24
    ([3, OUT, -1, -1, -1.2, -1, -2, -2], None, 2, 2, [0, 2]),
    ([1, OUT, 2, OUT, 0.5, OUT, 3, OUT], None, 2, 2, [6, 2]), ([1, OUT, 2, OUT, 0.5, OUT, 3, OUT], None, 4, 4, [6, 2, 0, 4]), ([1, OUT, 2, OUT, 0.5, OUT, 3, OUT], None, 3, 2, [6, 2, -1]),
    # taken out by the bias, and out by its logit: an expert's bias goes with it
    ([0, 0, 0, 0], [0.1, OUT, -0.3, -0.4], 1, 1, [0]), ([0, 0, 0, 0], [0.1, math.nan, -0.1, -0.1], 1, 1, [2]), ([0, OUT, 0, 0], [0.1, 9, -0.1, -0.1], 1, 1, [2]),
    ([0, OUT, 0, 0], [0.1, -9, -0.3, -0.3], 1, 1, [0])])
def test_a_group_counts_by_what_is_left_in_it(logits, bias, k, top, want):
    l, b = torch.tensor([logits], dtype=torch.float32), None if bias is None else torch.tensor(bias)
    assert w4.route(l, k, "sigmoid", bias=b, num_groups=len(logits) // 2, top_groups=top, group_score="top2")[1].tolist() == [want]
