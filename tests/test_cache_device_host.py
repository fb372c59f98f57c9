"""A streaming cache's device, however the caller names it."""
import pytest
import torch

from nsn_amd.errors import IntegrityError
from nsn_amd.stream_cache import StreamingKVCache


@pytest.mark.parametrize("name", ["cpu", "cpu:0", torch.device("cpu"), torch.device("cpu", 0)])
def test_one_device_has_one_name(name):
    """Copies between caches compare devices, and a ragged compression asks the device's type."""
    a = StreamingKVCache(1, 2, 2, 256, max_append=64, device=name)
    b = StreamingKVCache(1, 2, 2, 256, max_append=64, device=torch.device("cpu"))
    assert a.device == b.device == a.side(0, "K").tail.device
    for x, y in ((a, b), (b, a)):
        with pytest.raises(IntegrityError, match="GPU"):     # (not: the caches differ)
            x.copy_from(y, [0, 1])
    assert a.device.type == "cpu"
