"""The widest rows that layer normalisation takes: kernels count columns, and two sums for each, in 32 bits."""
import pytest
import torch

from tensornet_b200.ops import functional as F


@pytest.mark.parametrize("columns", [2 ** 30 + 1, 2 ** 31 - 1024, 2 ** 31 - 66, 2 ** 31])
def test_wider_rows_are_refused(columns):
    with pytest.raises(ValueError, match="columns"):
        F.layer_norm(torch.empty((1, columns), device="meta"))


def test_the_widest_are_taken():
    assert F.layer_norm(torch.empty((1, 2 ** 30), device="meta")).shape == (1, 2 ** 30)


def test_sums_over_a_block_lie_where_two_are_read_at_a_time():
    """``block_sum`` reads its shared memory in pairs: what is handed to it has to be declared in pairs, which is what aligns it."""
    import os
    import re

    import tensornet_b200

    with open(os.path.join(os.path.dirname(tensornet_b200.__file__), "csrc", "layer_norm.cu")) as f:
        text = f.read()
    assert re.search(r"void block_sum\(.*float2\* s,", text)
    assert len(re.findall(r"block_sum<\d>\(", text)) == 6
    assert set(re.findall(r"block_sum<\d>\(\w+, \w+, (\w+),", text)) == {"s_sum"}
    assert set(re.findall(r"__shared__ (\w+) s_sum\[", text)) == {"float2"}
