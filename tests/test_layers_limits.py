"""Limits of the layer operators, without a GPU."""
import pytest

from sdc_b200 import capi
from sdc_b200.layers import AdapterBatch


def test_adapter_batches_end_before_their_look_ahead_passes_32_bits():
    """The weights' gradients look tokens up as much as 18 tiles of 32 slots ahead."""
    with pytest.raises(ValueError, match="fewer than"):
        AdapterBatch([2 ** 31 - 1024], [0], 1, device="cpu")
    lib, fake = capi.lib(), 1 << 20  # never dereferenced: validation fails first
    for tokens in (2 ** 31 - 1024, 2 ** 31 - 500, 2 ** 31 - 1):
        assert lib.sdc_adapter_outer(1, fake, 64, tokens, fake, None, 2, fake, 4, 8, 64, 0, fake, None) == capi.SDC_ERR_INVALID
        assert "fewer than" in capi.last_error()
    assert lib.sdc_adapter_outer(1, fake, 64, 2 ** 31 - 1025, fake, None, 2, fake, 4, 8, 64, 0, fake, None) == capi.SDC_ERR_INVALID
    assert "null" in capi.last_error()
