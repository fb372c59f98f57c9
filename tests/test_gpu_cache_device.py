"""A streaming cache on "cuda" works like one on "cuda:0", and copies between them."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def test_a_cache_on_the_current_device():
    from nsn_amd.stream_cache import StreamingKVCache
    g = torch.Generator(device="cuda").manual_seed(2)
    k, v = (torch.randn((2, 2, 300, 128), generator=g, device="cuda").half() for _ in "kv")
    q = torch.randn((2, 8, 128), generator=g, device="cuda").bfloat16()
    got = []
    for name in ("cuda", torch.device("cuda"), None):
        c = StreamingKVCache(1, 2, 2, 512, max_append=384, device=name)
        c.append(0, k, v, counts=[300, 140])
        c.post_prefill()                       # ragged: the block counts are uploaded
        assert c.seq_compressed == [[192, 64]]
        other = StreamingKVCache(1, 2, 2, 512, max_append=384, device="cuda:0")
        other.copy_from(c, [1, 0])
        got.append((c.decode(0, q, kernel="fast")[0], other.decode(0, q.flip(0).contiguous(), kernel="fast")[0].flip(0)))
    for a, b in got:
        assert torch.equal(a, got[0][0]) and torch.equal(b, got[0][0])
