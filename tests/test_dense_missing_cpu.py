"""Operands that are missing: refused, not read as another operator's call."""
import pytest
import torch


def test_gated_linear_without_its_second_weight():
    from nano_ktrans_b200 import gated_linear

    x = torch.zeros(2, 8, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="up_weight is missing"):
        gated_linear(x, x, None)
