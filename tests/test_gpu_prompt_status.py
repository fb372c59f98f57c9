"""Flags of StreamingKVCache.prompt: raised by the call, left in the caller's word, or
(check=False, no word given) in the cache's own, which check_status reads."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def test_flags_of_an_unchecked_prompt_reach_check_status():
    from nsn_amd import _lib
    from nsn_amd.errors import NumericalFailure
    from nsn_amd.stream_cache import StreamingKVCache
    g = torch.Generator(device="cuda").manual_seed(1)
    q, k, v = (torch.randn((90, h, 128), generator=g, device="cuda").half() for h in (4, 2, 2))
    lens = [40, 50]

    def fresh():
        return StreamingKVCache(1, 2, 2, 512, max_append=256)
    c = fresh()
    c.prompt(0, q, k, v, lens, check=False)
    c.check_status()
    v[30, 1, 7] = float("inf")
    c = fresh()
    c.prompt(0, q, k, v, lens, check=False)
    assert c.seq_length == [lens]
    with pytest.raises(NumericalFailure, match="prompt"):
        c.check_status()
    # a word of the caller's keeps them to itself
    c, st = fresh(), torch.zeros(1, dtype=torch.int32, device="cuda")
    c.prompt(0, q, k, v, lens, check=False, status=st)
    assert int(st.item()) == _lib.ST_NONFINITE_OUTPUT
    c.check_status()
    # and a checked call raises and leaves the cache as it was
    c = fresh()
    with pytest.raises(NumericalFailure):
        c.prompt(0, q, k, v, lens)
    assert c.seq_length == [[0, 0]]
    c.check_status()
