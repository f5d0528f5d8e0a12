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
