"""The streaming cache's device lengths under a HIP graph's capture (no device needed:
the capture is pretended): what the capture makes is not kept for eager calls, what
a graph reads is not dropped, and no upload is recorded."""
import torch

from nsn_amd import _dev
from nsn_amd.stream_cache import StreamingKVCache


def test_lengths_under_a_capture(monkeypatch):
    c = StreamingKVCache(1, 3, 2, 256, max_append=64, device=torch.device("cpu"))
    there = c.length_tensor([7, 7, 9])
    c._gpu = True
    with monkeypatch.context() as m:
        m.setattr(_dev, "capturing", lambda: True)
        m.setattr(torch, "tensor", lambda *a, **k: (_ for _ in ()).throw(AssertionError("a recorded upload")))
        for L in (8, [8, 9, 9], [1, 2, 1]):
            t = c.length_tensor(L)
            assert t.tolist() == (L if isinstance(L, list) else [L] * 3) and t.dtype == torch.int32
        assert c._offsets([4, 0, 5]).tolist() == [0, 4, 4, 9] and c._offsets([0, 0, 0]).tolist() == [0] * 4
        assert list(c._len_dev) == [(7, 7, 9)]
        assert c.length_tensor([7, 7, 9]) is there
    c._gpu = False
    for n in range(1000, 1600):                 # (the oldest entries are dropped)
        c.length_tensor(n)
    assert len(c._len_dev) <= 256 and c.length_tensor(1599).tolist() == [1599] * 3
    assert any(t is there for t in c._len_captured.values()) and there.tolist() == [7, 7, 9]
