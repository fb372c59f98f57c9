"""Calls of a streaming cache captured into a HIP graph, with lengths that are on the
device before the capture or not: replays, and eager calls before, between and after
them, agree."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def filled(lens, slots=1, seed=1):
    from nsn_amd.stream_cache import StreamingKVCache
    g = torch.Generator(device="cuda").manual_seed(seed)
    c = StreamingKVCache(slots, len(lens), 2, 1024, max_append=512)
    for s in range(slots):
        k, v = (torch.randn((len(lens), 2, max(lens), 128), generator=g, device="cuda").half() for _ in "kv")
        c.append(s, k, v, counts=lens)
    c.post_prefill()
    return c, torch.randn((len(lens), 8, 128), generator=g, device="cuda").bfloat16()


@pytest.mark.parametrize("lens", [[300, 300], [300, 70]])
@pytest.mark.parametrize("branch", [False, True])
@pytest.mark.parametrize("called_before", [False, True])
def test_a_captured_decode(lens, branch, called_before):
    c, q = filled(lens)
    other, _ = filled(lens)
    if branch:
        c, other, q = c.branch(2, 256), other.branch(2, 256), q.repeat_interleave(2, 0).contiguous()
    want = other.decode(0, q, kernel="fast")[0].clone()
    if called_before:
        assert torch.equal(c.decode(0, q, kernel="fast")[0], want)
    st = torch.zeros(1, dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = c.decode(0, q, kernel="fast", check=False, status=st)[0]
    for i in range(3):
        if i:
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, want) and int(st.item()) == 0
            out.zero_()
        assert torch.equal(c.decode(0, q, kernel="fast")[0], want)      # (i = 0: before the first replay)
        # other lengths, more than are kept, and work in their memory between the replays
        for n in range(1000 + 300 * i, 1300 + 300 * i):
            c.length_tensor(n)
        torch.full((1 << 16,), -1, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("called_before", [False, True])
def test_a_captured_prefill(called_before):
    c, _ = filled([200, 130])
    other, _ = filled([200, 130])
    g = torch.Generator(device="cuda").manual_seed(3)
    q, k, v = (torch.randn((2, h, 30, 128), generator=g, device="cuda").half() for h in (8, 2, 2))
    want = other.prefill(0, q, k, v).clone()
    if called_before:
        assert torch.equal(c.prefill(0, q, k, v), want)
    st = torch.zeros(1, dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = c.prefill(0, q, k, v, check=False, status=st)
    assert torch.equal(c.prefill(0, q, k, v), want)
    for _ in range(3):
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(c.prefill(0, q, k, v), want) and int(st.item()) == 0


@pytest.mark.parametrize("lens", [[40, 0, 60, 130], [50, 50, 50, 50]])
def test_a_captured_prompt(lens):
    """Every replay attends the prompts and writes the tails from the rows as they are by then."""
    from nsn_amd import kernels
    from nsn_amd.stream_cache import StreamingKVCache
    g = torch.Generator(device="cuda").manual_seed(4)
    n = sum(lens)
    q, k, v = (torch.randn((n, h, 128), generator=g, device="cuda").half() for h in (8, 2, 2))
    cu = torch.tensor([0] + [sum(lens[:i + 1]) for i in range(4)], dtype=torch.int32, device="cuda")
    c = StreamingKVCache(1, 4, 2, 512, max_append=256)
    st = torch.zeros(1, dtype=torch.int32, device="cuda")
    kernels.prompt_attention(q, k, v, cu)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = c.prompt(0, q, k, v, lens, check=False, status=st)
    assert c.seq_length == [lens]
    for i in range(3):
        k.normal_(generator=g), v.normal_(generator=g)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, kernels.prompt_attention(q, k, v, cu)) and int(st.item()) == 0
        at = 0
        for b, m in enumerate(lens):
            for name, t in (("K", k), ("V", v)):
                assert torch.equal(c.side(0, name).tail[b, :, :m], t[at:at + m].transpose(0, 1))
            at += m
