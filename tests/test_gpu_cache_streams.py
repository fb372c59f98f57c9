"""A streaming cache's calls from two streams: a stream does not read lengths that
another one has yet to write."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("lens", [[300, 300, 300], [300, 70, 190]])
@pytest.mark.parametrize("branch", [False, True])
def test_two_streams_decode_at_the_same_lengths(lens, branch):
    from nsn_amd.stream_cache import StreamingKVCache
    g = torch.Generator(device="cuda").manual_seed(1)
    k, v = (torch.randn((3, 2, 300, 128), generator=g, device="cuda").half() for _ in "kv")
    q = torch.randn((3, 8, 128), generator=g, device="cuda").bfloat16()

    def make():
        c = StreamingKVCache(1, 3, 2, 1024, max_append=512)
        c.append(0, k, v, counts=lens)
        c.post_prefill()
        return c.branch(1, 256) if branch else c
    want = make().decode(0, q, kernel="fast")[0].clone()
    c = make()
    st = [torch.zeros(1, dtype=torch.int32, device="cuda") for _ in range(2)]
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(a):
        torch.cuda._sleep(200_000_000)          # the first stream writes its lengths long after the second one's call
        first = c.decode(0, q, kernel="fast", check=False, status=st[0])[0]
    with torch.cuda.stream(b):
        second = c.decode(0, q, kernel="fast", check=False, status=st[1])[0]
    b.synchronize()
    assert torch.equal(second, want)
    torch.cuda.synchronize()
    assert torch.equal(first, want) and int(st[0].item()) == int(st[1].item()) == 0
