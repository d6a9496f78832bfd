"""Shapes of gate, scale and shift of the gated residual step, on the CPU."""

from __future__ import annotations

import pytest
import torch

from avgen_amd import layers


@pytest.mark.parametrize("modulation", ["gate", "scale", "shift"])
def test_one_row_without_leading_sizes(modulation):
    """A modulation of the shape of a single row reaches the op's own checks."""
    x = torch.zeros(8)
    assert all(t is None or t.shape == (8,) for t in layers._one_modulation(x.shape, None, x, x))
    with pytest.raises(RuntimeError, match="no CPU path"):
        layers.gated_add_rms_norm(x, x, **{modulation: x})


@pytest.mark.parametrize("shape", [(2, 8), (1, 1, 8)])
def test_more_sizes_than_the_row_are_refused(shape):
    with pytest.raises(ValueError, match="broadcast"):
        layers.gated_add_rms_norm(torch.zeros(8), torch.zeros(8), gate=torch.zeros(shape))
