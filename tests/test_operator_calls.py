"""CPU: checks of the training-step operators' Python entries that need no GPU: counts past 32 bits, options of an optimiser's groups, models that
take no group norm."""
import pytest
import torch

from openpcdet_amd import _lib, backbones_2d, focal, optim, unet


# ---- counts ----------------------------------------------------------------------------------------------------------------
def test_counts_past_32_bits():
    _lib.check_counts("op", 0, 1, 2 ** 31 - 1)
    for big in (2 ** 31, 2 ** 32 + 5):
        with pytest.raises(ValueError, match="op: a count of %d is past 32 bits" % big):
            _lib.check_counts("op", 3, big, 1)
