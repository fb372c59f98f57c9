"""Beam search over the packed cache, byte for byte: after transformers' generate with
several beams every row of every slot holds what a cache holds that was given that
row's tokens alone, one step after the other (a row's arithmetic does not depend on
the other rows of its batch)."""
import pytest
import torch

pytest.importorskip("transformers")
from nsn_amd import adapter  # noqa: E402
from tests.test_gpu_adapter import model  # noqa: E402

pytestmark = pytest.mark.gpu


def same_rows(a, b):
    """Lengths, and every valid byte of both sides, equal."""
    assert a.seq_length == b.seq_length and a.seq_compressed == b.seq_compressed
    for name in ("K", "V"):
        x, y = a.storage(name), b.storage(name)
        assert torch.equal(x["blocks"], y["blocks"])
        for s in range(a.slots):
            nb, rest = a.seq_compressed[s][0] // 64, a.seq_length[s][0] - a.seq_compressed[s][0]
            for k in ("codes", "norm", "min", "scale", "factor", "headers", "tail"):
                n = rest if k == "tail" else nb
                p, q = (t[k][s, :, :, :n].contiguous().view(torch.uint8) for t in (x, y))
                assert torch.equal(p, q), (name, s, k)


@pytest.mark.parametrize("prompt,new", [(20, 40), (100, 60)])      # (the second one packs a block on the way)
def test_generate_with_beams_moves_every_slot(prompt, new):
    m, cfg, ids = model()
    m.generation_config.eos_token_id = None
    m.generation_config.pad_token_id = 0
    ids, beams = ids[:, :prompt], 3
    rows = ids.shape[0] * beams
    history = [[] for _ in range(rows)]
    orders = []

    class Recorded(adapter.PackedKVCache):
        def reorder_cache(self, beam_idx):
            order = beam_idx.tolist()
            orders.append(order)
            history[:] = [list(history[i]) for i in order]
            super().reorder_cache(beam_idx)

    def record(module, args):
        for row, tokens in zip(history, args[0].tolist()):
            row.extend(tokens)

    def cache(kind):
        return kind(cfg, rows, 512, max_prefill=128, auto_policy=True)
    restore = adapter.install(m)
    try:
        with torch.no_grad():
            got = cache(Recorded)
            hook = m.model.embed_tokens.register_forward_pre_hook(record)
            out = m.generate(ids, past_key_values=got, max_new_tokens=new, do_sample=False, num_beams=beams)
            hook.remove()
            alone = cache(adapter.PackedKVCache)
            tokens = torch.tensor(history, device=ids.device)
            m(input_ids=tokens[:, :prompt], past_key_values=alone, use_cache=True)
            for i in range(prompt, tokens.shape[1]):
                m(input_ids=tokens[:, i:i + 1], past_key_values=alone, use_cache=True)
    finally:
        restore()
    assert out.shape == (ids.shape[0], prompt + new)
    assert len(orders) >= new - 1 and any(o != list(range(rows)) for o in orders)
    assert all(i // beams == p // beams for o in orders for i, p in enumerate(o))
    assert got.store.length == [tokens.shape[1]] * got.store.slots
    same_rows(got.store, alone.store)


def test_a_reorder_is_a_copy_of_rows():
    """Two caches with the same prompts: one reordered, the other not, given each other's next tokens."""
    m, cfg, ids = model()
    order = [1, 1]
    restore = adapter.install(m)
    try:
        with torch.no_grad():
            caches = []
            for nxt in ([[5], [9]], [[7], [5]], [[7], [9]]):
                c = adapter.PackedKVCache(cfg, 2, 512, arm="PACKED_KV_FUSED", max_prefill=256)
                m(input_ids=ids, past_key_values=c, use_cache=True)
                c.post_prefill()
                if not caches:
                    c.reorder_cache(torch.tensor(order, device="cuda"))
                caches.append((c, m(input_ids=torch.tensor(nxt, device="cuda"), past_key_values=c, use_cache=True).logits))
    finally:
        restore()
    (moved, a), (_, b), (_, d) = caches
    assert torch.equal(a[0], b[1]) and torch.equal(a[1], d[1])
    assert moved.store.seq_length == [[151, 151]] * moved.store.slots
