"""GPU-resident streaming packed K/V cache (the reference's PackedCache, rebuilt).

The reference keeps, per slot (layer x loop) and side, a growing dict of
packed block groups joined with ``torch.cat`` on every compression and an
fp16/bf16 tail cut with ``clone`` (experiments/ac08/source/
loop_kv_pk01_cache.py:76-132).  Here every slot owns preallocated storage:

- packed blocks ``[B, Hkv, cap, ...]`` (codes, norm, min, scale, decode
  factors, 12-byte headers), written in place by one encoder launch per
  compression (``nsn_encode_blocks`` with a block offset);
- a tail buffer of ``tail_cap`` tokens, re-based after each compression
  (one device copy of the surviving tokens).

The policy is the reference's:

- ``post_prefill``: compress to ``max(0, ((L - 64) // 64) * 64)``
  (``loop_kv_pk01_cache.py:122-123``);
- ``post_decode``: once ``L - compressed >= 128``, compress one more block
  (``:124-127``);

so after either call the tail holds 64..127 tokens (fewer only for short
sequences).  Headers carry the token offset of each block ('<QHBB', as
``encode_group`` writes them, ``:31-37``).

Sequences of a batch may have different lengths (the ragged decode batch of
the C2 workload): every sequence has its own length and compressed prefix,
the policy applies per sequence, and appends may carry a per-sequence token
count.  Lengths are host integers, so nothing here synchronises with the
device; while every sequence of a slot has the same state, each operation is
one launch for the whole batch, otherwise one per sequence that changes.
"""
from __future__ import annotations

import weakref
from dataclasses import dataclass
from itertools import accumulate

import torch

from . import _dev, _lib
from .errors import IntegrityError, NumericalFailure, require
from .kernels import BLOCK, DIM, PackedKV

MIN_TAIL = 64


def prefill_target(length: int) -> int:
    """Compressed-token target after the prefill (loop_kv_pk01_cache.py:122-123)."""
    return max(0, ((length - MIN_TAIL) // BLOCK) * BLOCK)


def decode_target(length: int, compressed: int) -> int:
    """Compressed-token target after a decode step (loop_kv_pk01_cache.py:124-127)."""
    return compressed + BLOCK if length - compressed >= 2 * BLOCK else compressed


@dataclass
class _Side:
    kv: PackedKV
    headers: torch.Tensor   # u8 [B, H, cap, 12]


class StreamingKVCache:
    """Packed K/V of ``slots`` attention slots for ``batch`` sequences x ``heads`` kv-heads.

    max_tokens bounds the sequence length (block capacity = max_tokens // 64);
    max_append bounds the tokens appended between two compressions (a
    prefill chunk, or 1 per decode step).  ``dtype`` is the tail's dtype
    (fp16 or bf16; both kernels read either); appended K/V of another dtype
    are converted to it.

    ``seq_length[slot]`` / ``seq_compressed[slot]`` hold each sequence's token
    count and packed prefix; ``length[slot]`` / ``compressed[slot]`` are the
    longest sequence's length and the shortest packed prefix (the common
    values when the batch is uniform).
    """

    def __init__(self, slots, batch, heads, max_tokens, *, bits=3, dtype=torch.float16, max_append=512,
                 device=None):
        device = torch.empty(0, device=device or torch.device("cuda:0")).device   # (with its index, however named)
        require(bits in (3, 4, 5), "Bits")
        require(dtype in (torch.float16, torch.bfloat16), "Tail dtype")
        self.slots, self.batch, self.heads, self.bits, self.dtype = slots, batch, heads, bits, dtype
        self.block_cap = max(1, max_tokens // BLOCK)
        self.tail_cap = 2 * BLOCK + max_append
        self.device = device
        self._gpu = device.type == "cuda"
        nbytes = BLOCK * DIM * bits // 8
        # one allocation per array for all slots ([slots, batch, heads, ...]):
        # sequences are copied over every slot by one launch
        lead = (slots, batch, heads, self.block_cap)
        # the packed-block counts, [slots, K and V, batch]: a slot's are set by
        # one launch (or one upload) per compression
        counts = torch.zeros((slots, 2, batch), dtype=torch.int32, device=device)
        self._blocks = list(counts.unbind(0))
        self._storage, self._sides = {}, {}
        for i, name in enumerate(("K", "V")):
            w = dict(codes=torch.empty(lead + (nbytes,), dtype=torch.uint8, device=device),
                     norm=torch.empty(lead + (BLOCK,), dtype=torch.float16, device=device),
                     min=torch.empty(lead + (DIM,), dtype=torch.float16, device=device),
                     scale=torch.empty(lead + (DIM,), dtype=torch.float16, device=device),
                     factor=torch.empty(lead + (BLOCK,), dtype=torch.float32, device=device),
                     blocks=counts[:, i],
                     tail=torch.zeros((slots, batch, heads, self.tail_cap, DIM), dtype=dtype, device=device),
                     headers=torch.zeros(lead + (12,), dtype=torch.uint8, device=device))
            self._storage[name] = w
            for s in range(slots):
                kv = PackedKV(**{k: w[k][s] for k in ("codes", "norm", "min", "scale", "factor", "blocks", "tail")},
                              bits=bits)
                self._sides[(s, name)] = _Side(kv, w["headers"][s])
        self.seq_length = [[0] * batch for _ in range(slots)]       # tokens held per slot and sequence
        self.seq_compressed = [[0] * batch for _ in range(slots)]   # of which packed
        self._len_dev = {}               # cached int32 length tensors: {lengths: {stream: tensor}}
        self._len_captured = {}          # of which HIP graphs read
        self.status = _dev.new_status(device)
        self.encoded_blocks = [0] * slots
        self._side = None                # second stream of the compressions
        # a branch (see branch()): the cache whose packed blocks its sequences
        # continue, those blocks per slot, and the tokens they hold per sequence
        self.prefix, self._prefix_sides = None, None
        self.prefix_tokens = [[0] * batch for _ in range(slots)]
        self._branches = weakref.WeakSet()   # live branches: they read this cache's blocks
        self._c_store = None             # the storage as nsn_cache_copy takes it

    # ------------------------------------------------------------------ views
    def side(self, slot, name) -> PackedKV:
        return self._sides[(slot, name)].kv

    def headers(self, slot, name) -> torch.Tensor:
        return self._sides[(slot, name)].headers

    def storage(self, name) -> dict:
        """Every array of side ``name`` over all slots ([slots, batch, heads, ...];
        ``blocks`` [slots, batch]): ``side(slot, name)`` and ``headers`` are views of it."""
        return self._storage[name]

    @property
    def length(self):
        """Per slot: the longest sequence's token count."""
        return [max(x) for x in self.seq_length]

    @property
    def compressed(self):
        """Per slot: the shortest packed prefix."""
        return [min(x) for x in self.seq_compressed]

    def uniform(self, slot) -> bool:
        """Every sequence of the slot holds the same tokens and packed prefix."""
        L, C = self.seq_length[slot], self.seq_compressed[slot]
        return min(L) == max(L) and min(C) == max(C)

    def lengths(self, slot) -> torch.Tensor:
        """int32 [B] device tensor of the slot's per-sequence lengths."""
        return self.length_tensor(self.seq_length[slot])

    def length_tensor(self, L) -> torch.Tensor:
        """int32 [B] device tensor of the lengths L (an int for every sequence, or
        one per sequence), made once per distinct value and stream and kept (for
        good, once a HIP graph reads it): another stream could read it before it
        is written.  What a capture makes itself is the graph's alone: unset until
        a replay, it must not answer an eager call."""
        key = tuple(L) if isinstance(L, (list, tuple)) else (int(L),) * self.batch
        kept = self._len_dev.get(key)
        if self._gpu and _dev.capturing():
            if not kept:
                return self._upload(key)
            t = self._len_captured[key] = next(iter(kept.values()))
            return t
        stream = _dev.stream() if self._gpu else 0
        t = kept.get(stream) if kept else None
        if t is None:
            t = self._upload(key)
            # the oldest lengths are dropped (a dropped tensor's memory is
            # reused only by later work on its stream)
            if kept is None and len(self._len_dev) >= 256:
                self._len_dev.pop(next(iter(self._len_dev)))
            self._len_dev.setdefault(key, {})[stream] = t
        return t

    def _upload(self, values):
        """int32 device tensor of host integers.  Uploaded from pinned memory
        without a host wait: a pageable copy would drain the stream first, so
        every new length (each chunk, each decode step) would leave the GPU idle
        while the host issues the next launches.  One value for all -- each decode
        step of a uniform batch brings a new one -- is a single fill on the device
        instead, and so is each run of equal values under a capture: a recorded
        copy would read host memory that is gone by the replay."""
        if min(values) == max(values):
            return torch.full((len(values),), values[0], dtype=torch.int32, device=self.device)
        if not (self._gpu and _dev.capturing()):
            t = torch.tensor(values, dtype=torch.int32, pin_memory=self._gpu)
            return t.to(self.device, non_blocking=self._gpu)
        t = torch.empty(len(values), dtype=torch.int32, device=self.device)
        cuts = [i for i in range(len(values)) if i == 0 or values[i] != values[i - 1]]
        for i, end in zip(cuts, cuts[1:] + [len(values)]):
            t[i:end].fill_(values[i])
        return t

    def tail_len(self, slot):
        """Tail tokens of the slot (the batch must be uniform)."""
        if not self.uniform(slot):
            raise IntegrityError("Ragged slot: use seq_tail_len")
        return self.seq_length[slot][0] - self.seq_compressed[slot][0]

    def seq_tail_len(self, slot, b):
        return self.seq_length[slot][b] - self.seq_compressed[slot][b]

    def advance(self, slot, n=1):
        """Count n more tokens in every sequence of the slot: the host side of
        an append its caller made on the device (a device-position tail
        append, replayed from a HIP graph)."""
        L = self.seq_length[slot]
        for b in range(self.batch):
            L[b] += n

    def reset(self, slot):
        """Empty the slot for a new batch of sequences (its storage is kept;
        nothing past a sequence's length is ever read).  A branch keeps its
        prefix; a cache with branches stays as it is."""
        self._require_no_branch()
        for b in range(self.batch):
            self.seq_length[slot][b] = 0
            self.seq_compressed[slot][b] = 0
        self._blocks[slot].zero_()
        self.encoded_blocks[slot] = 0

    # ------------------------------------------------------------------ updates
    def append(self, slot, k, v, counts=None):
        """Append k, v [B, H, n, 128] to the slot's tails (converted to the tail
        dtype if needed).  ``counts`` (one int per sequence, each <= n) appends
        only sequence b's first counts[b] tokens; default n for every sequence."""
        require(k.shape == v.shape and k.ndim == 4 and tuple(k.shape[:2]) == (self.batch, self.heads)
                and k.shape[3] == DIM, "Append shape")
        n = k.shape[2]
        L, C = self.seq_length[slot], self.seq_compressed[slot]
        # (every sequence alike, a uniform batch's append: checked once, not per sequence)
        same = counts is None and self.uniform(slot)
        counts = [n] * self.batch if counts is None else [int(c) for c in counts]
        require(len(counts) == self.batch and all(0 <= c <= n for c in counts), "Append counts")
        for b in range(1 if same else self.batch):
            if L[b] - C[b] + counts[b] > self.tail_cap:
                raise IntegrityError("Tail overflow: compress before appending more tokens")
            if L[b] + counts[b] > self.block_cap * BLOCK + self.tail_cap:
                raise IntegrityError("Cache capacity exceeded")
        require(k.dtype in (torch.float16, torch.bfloat16, torch.float32) and v.dtype == k.dtype, "Append dtype")
        k, v = k.contiguous(), v.contiguous()
        # another dtype converts inside the append kernel (no separate pass);
        # an fp32 tail takes the converted copy
        cast = k.dtype != self.dtype and self.dtype in (torch.float16, torch.bfloat16)
        if k.dtype != self.dtype and not cast:
            k, v = k.to(self.dtype), v.to(self.dtype)
        kt, vt = self._sides[(slot, "K")].kv.tail, self._sides[(slot, "V")].kv.tail
        lib = _lib.lib()
        dt = _dev.dtype_code(self.dtype)
        offs = [L[0] - C[0]] if same else [L[b] - C[b] for b in range(self.batch)]
        sdt = _dev.dtype_code(k.dtype)

        def launch(kp, vp, ktp, vtp, rows, cnt, off):
            if cast:
                rc = lib.nsn_tail_append_cast(kp, vp, sdt, rows, cnt, n, ktp, vtp, self.tail_cap, off, dt,
                                              _dev.stream())
                _lib.check(rc, "nsn_tail_append_cast")
            else:
                rc = lib.nsn_tail_append(kp, vp, rows, cnt, n, ktp, vtp, self.tail_cap, off, dt, _dev.stream())
                _lib.check(rc, "nsn_tail_append")
        if same or (len(set(offs)) == 1 and len(set(counts)) == 1):
            if counts[0]:
                launch(k.data_ptr(), v.data_ptr(), kt.data_ptr(), vt.data_ptr(), self.batch * self.heads, counts[0],
                       offs[0])
        else:
            for b in range(self.batch):   # one launch per sequence: its own offset and count
                if counts[b]:
                    launch(k[b].data_ptr(), v[b].data_ptr(), kt[b].data_ptr(), vt[b].data_ptr(), self.heads,
                           counts[b], offs[b])
        for b in range(self.batch):
            L[b] += counts[b]

    def compress_to(self, slot, target):
        """Encode tail tokens up to absolute position `target` (a multiple of
        64; an int for every sequence or one per sequence) into packed
        blocks, in place; the tails keep the rest."""
        targets = [int(target)] * self.batch if not isinstance(target, (list, tuple)) else [int(t) for t in target]
        require(len(targets) == self.batch, "Compress targets")
        L, C = self.seq_length[slot], self.seq_compressed[slot]
        for b in range(self.batch):
            start, tgt = C[b], targets[b]
            if not (tgt >= start and (tgt - start) % BLOCK == 0):
                raise IntegrityError("Block overlap/ordering")
            if tgt == start:
                continue
            if L[b] < tgt + BLOCK:
                raise IntegrityError("Tail/compressed divergence")
            if tgt // BLOCK > self.block_cap:
                raise IntegrityError("Cache capacity exceeded")
        moving = [b for b in range(self.batch) if targets[b] != C[b]]
        if not moving:
            return
        if (len(moving) == self.batch and len(set(C)) == 1 and len(set(targets)) == 1 and len(set(L)) == 1
                and len(set(self.prefix_tokens[slot])) == 1):
            self._encode_rows(slot, None, C[0], targets[0], L[0])   # the whole batch in one launch per side
        else:
            for b in moving:
                self._encode_rows(slot, b, C[b], targets[b], L[b])
        # blocks added per sequence (the most any sequence gained in this call)
        self.encoded_blocks[slot] += max((targets[b] - C[b]) // BLOCK for b in moving)
        for b in moving:
            C[b] = targets[b]
        nblocks = [c // BLOCK for c in C]
        if len(set(nblocks)) == 1:
            self._blocks[slot].fill_(nblocks[0])
        else:   # from pinned memory without a host wait, like the lengths
            gpu = self.device.type == "cuda"
            self._blocks[slot].copy_(torch.tensor([nblocks, nblocks], dtype=torch.int32, pin_memory=gpu),
                                     non_blocking=gpu)

    def _encode_rows(self, slot, b, start, target, length):
        """Encode tokens [start, target) of sequence b (or of every sequence,
        b None) from the tail into blocks start/64 .., then re-base the tail."""
        lib = _lib.lib()
        n = target - start
        nb = n // BLOCK
        rest = length - target
        rows = self.heads if b is not None else self.batch * self.heads
        sel = (lambda t: t[b]) if b is not None else (lambda t: t)

        def encode(name, stream):
            sd = self._sides[(slot, name)]
            kv = sd.kv
            rc = lib.nsn_encode_blocks(
                sel(kv.tail).data_ptr(), _dev.dtype_code(self.dtype), rows, nb,
                self.tail_cap * DIM, 0, self.bits, _lib.NORM_LANES8, 1,
                sel(kv.codes).data_ptr(), sel(kv.norm).data_ptr(), sel(kv.min).data_ptr(),
                sel(kv.scale).data_ptr(), sel(sd.headers).data_ptr(), sel(kv.factor).data_ptr(), self.block_cap,
                start // BLOCK, start + self.prefix_tokens[slot][b or 0], None, self.status.data_ptr(), stream)
            _lib.check(rc, "nsn_encode_blocks")
        # K and V are encoded side by side: V on a second stream forked from
        # and joined back into the current one (each launch alone is too
        # small to fill the GPU)
        cur = torch.cuda.current_stream(self.device)
        if self._side is None:
            self._side = torch.cuda.Stream(device=self.device)
        self._side.wait_stream(cur)
        encode("K", cur.cuda_stream)
        encode("V", self._side.cuda_stream)
        cur.wait_stream(self._side)
        # re-base the surviving tail tokens [n, n + rest) of every row to [0, rest)
        if rest <= 0:
            return
        kt, vt = sel(self._sides[(slot, "K")].kv.tail), sel(self._sides[(slot, "V")].kv.tail)
        if rest <= n:   # disjoint: one copy launch for both sides
            step = n * DIM * kt.element_size()
            rc = lib.nsn_tail_append(kt.data_ptr() + step, vt.data_ptr() + step, rows, rest, self.tail_cap,
                                     kt.data_ptr(), vt.data_ptr(), self.tail_cap, 0, _dev.dtype_code(self.dtype),
                                     _dev.stream())
            _lib.check(rc, "nsn_tail_append")
        else:           # overlapping rows: through a copy of the source
            for tail in (kt, vt):
                tail[..., :rest, :] = tail[..., n:n + rest, :].clone()

    def post_prefill(self):
        for s in range(self.slots):
            self.compress_to(s, [prefill_target(L) for L in self.seq_length[s]])

    def post_decode(self):
        for s in range(self.slots):
            if max(self.seq_length[s]) - min(self.seq_compressed[s]) < 2 * BLOCK:
                continue   # (no sequence of the slot has a target past its packed prefix)
            self.compress_to(s, [decode_target(L, C) for L, C in zip(self.seq_length[s], self.seq_compressed[s])])

    def check_status(self):
        """Raise if any compression flagged nonfinite input or fp16 metadata trouble, or
        a prompt that was given no status word a nonfinite output (syncs)."""
        s = _dev.read_status(self.status)
        if s:
            from .primitives import _encode_raise
            _encode_raise(s)
            if s & _lib.ST_CAPACITY:
                raise IntegrityError("Prompt offsets or tail capacity")
            if s & _lib.ST_NONFINITE_OUTPUT:
                raise NumericalFailure("Nonfinite prompt attention output")

    def prompt(self, slot, q, k, v, lengths, **kw):
        """Causal attention over whole prompts of different lengths laid end to end,
        and the append of their tokens: q [N, Hq, 128], k, v [N, heads, 128] (fp16 or
        bf16, rows of any stride), sequence b the next ``lengths[b]`` rows (one int
        per sequence, their sum N; 0 for a sequence that takes no part).  A prompt
        sees no context: its sequence must be empty, and it must fit the tail
        (compress afterwards, with ``post_prefill``).  Returns out [N, Hq, 128];
        ``kw`` as ``kernels.prompt_attention`` takes them (``check=False`` without a
        ``status``: ``check_status`` reports the flags)."""
        lengths = [int(n) for n in lengths]
        require(self.prefix is None, "A branch decodes only: prompts go to the cache it branches from")
        require(len(lengths) == self.batch and all(n >= 0 for n in lengths) and sum(lengths) == q.shape[0],
                "Prompt lengths")
        require(k.ndim == 3 and k.shape[1] == self.heads, "Prompt K/V shape/type")
        for n, L in zip(lengths, self.seq_length[slot]):
            require(n == 0 or L == 0, "A prompt's sequence must be empty")
            if n > self.tail_cap or n > self.block_cap * BLOCK + self.tail_cap:
                raise IntegrityError("Tail overflow: compress before appending more tokens")
        cu = self._offsets(lengths)
        st = kw.get("status")
        if st is None and not kw.get("check", True):
            st = kw["status"] = self.status
        out = _attn().prompt_attention(q, k, v, cu, **kw)
        kt, vt = self._sides[(slot, "K")].kv.tail, self._sides[(slot, "V")].kv.tail
        rc = _lib.lib().nsn_prompt_append(
            k.data_ptr(), v.data_ptr(), _dev.dtype_code(k.dtype), k.shape[0], self.heads, *_attn()._row_strides(k),
            *_attn()._row_strides(v), cu.data_ptr(), self.batch, kt.data_ptr(), vt.data_ptr(), self.tail_cap,
            _dev.dtype_code(self.dtype), (self.status if st is None else st).data_ptr(), _dev.stream())
        _lib.check(rc, "nsn_prompt_append")
        for b, n in enumerate(lengths):
            self.seq_length[slot][b] += n
        return out

    def _offsets(self, lengths):
        """Device offsets of sequences of these lengths laid end to end."""
        return self._upload([0, *accumulate(lengths)])

    # ------------------------------------------------------------------ sequences
    def _require_no_branch(self):
        require(not len(self._branches), "The cache's packed blocks are read by its branches")

    def branch(self, fan, max_tokens, *, max_append=512):
        """A cache of ``fan`` sequences for each of this one's, which continue it
        behind its packed blocks: those are shared, not copied (``decode`` reads them
        once for all the sequences that continue them), only the tail's tokens are,
        into each branch's own tail.  ``max_tokens`` bounds a branch's own tokens,
        those of the tail included.  Row p * fan + i of the branch continues row p.

        ``seq_length`` of a branch counts its own tokens, ``prefix_tokens`` the shared
        ones.  It appends, compresses and decodes (fast kernel) like any cache, and
        forks among the rows of one prefix (a row emptied there keeps the prefix);
        prompts and prefill are refused.  Its decode holds the prefix's directions and
        weights in fp16 (the bounds of ``kernels.shared_prefix_attention``), where
        ``decode`` over a whole cache keeps them exact or as fp16 hi + lo.  While a
        branch lives this cache may grow, but not be reset, forked or copied into
        (its packed blocks must stay)."""
        require(fan >= 1, "Sequences per prefix")
        require(self.prefix is None, "A branch has no branches of its own")
        require(self.bits in (3, 5), "Branches need 3- or 5-bit codes")
        child = StreamingKVCache(self.slots, self.batch * fan, self.heads, max_tokens, bits=self.bits, dtype=self.dtype,
                                 max_append=max_append, device=self.device)
        runs = [(begin, end, [(L - C, 0) for L, C in per]) for begin, end, per in self._runs()]
        if max(L for _, _, per in runs for L, _ in per) > child.tail_cap:
            raise IntegrityError("Tail overflow: compress before branching")
        child._move_rows(self, [(p, p * fan + i) for p in range(self.batch) for i in range(fan)], runs)
        # (the counts of now: this cache may compress more)
        counts = [x.clone() for x in self._blocks]
        child._prefix_sides = {}
        for s in range(self.slots):
            for i, name in enumerate(("K", "V")):
                kv = self._sides[(s, name)].kv
                child._prefix_sides[(s, name)] = PackedKV(kv.codes, kv.norm, kv.min, kv.scale, kv.factor, counts[s][i],
                                                          None, self.bits)
            held = list(zip(self.seq_length[s], self.seq_compressed[s]))
            child.seq_length[s] = [L - C for L, C in held for _ in range(fan)]
            child.prefix_tokens[s] = [C for _, C in held for _ in range(fan)]
        child.prefix = self
        self._branches.add(child)
        return child

    def fork(self, parents):
        """Row i of every slot becomes a copy of row ``parents[i]`` (-1: it is
        emptied): packed blocks, headers, tail and length -- several samples of
        one prompt, a beam search's surviving rows, finished rows freed.  One int
        per row; rows named by themselves stay untouched.  In place and in one
        launch for all slots (per run of slots with equal lengths), whatever the
        mapping; work enqueued before on the current stream is seen."""
        parents = [int(p) for p in parents]
        require(len(parents) == self.batch and all(-1 <= p < self.batch for p in parents), "Fork rows")
        self._require_no_branch()
        if self.prefix is not None:
            fan = self.batch // self.prefix.batch
            require(all(p < 0 or p // fan == i // fan for i, p in enumerate(parents)), "A branch forks within its prefix")
        self._copy_rows(self, parents, _in_place_moves(parents))

    def copy_from(self, source, rows):
        """Row i of every slot becomes a copy of row ``rows[i]`` of ``source``
        (-1: it is emptied): running sequences move to a cache of another batch or
        capacity.  The caches agree in slots, heads, bits and tail dtype; every
        copied row must fit this cache."""
        rows = [int(r) for r in rows]
        require(source is not self, "Fork rows in place with fork()")
        require(self.prefix is None and source.prefix is None, "Rows of a branch stay with their prefix")
        self._require_no_branch()
        require(len(rows) == self.batch and all(-1 <= r < source.batch for r in rows), "Copied rows")
        require((source.slots, source.heads, source.bits, source.dtype) ==
                (self.slots, self.heads, self.bits, self.dtype) and source.device == self.device,
                "Caches differ in slots, heads, bits, dtype or device")
        # (sorted: the moves of one source follow each other and read it once)
        self._copy_rows(source, rows, sorted((r, i) for i, r in enumerate(rows)))

    def _copy_rows(self, source, rows, moves):
        """Carry out ``moves`` ((source row, row) pairs, -1 as source: emptied) and
        take over the lengths: row i's are those of row rows[i] of ``source``."""
        runs = source._runs()
        for _, _, per in runs:
            for n, c in (per[r] for r in rows if r >= 0):   # (refused here, before anything is written)
                if c // BLOCK > self.block_cap or n - c > self.tail_cap:
                    raise IntegrityError("Cache capacity exceeded")
        self._move_rows(source, moves, runs)
        for begin, end, per in runs:
            L = [per[r][0] if r >= 0 else 0 for r in rows]
            C = [per[r][1] if r >= 0 else 0 for r in rows]
            self.seq_length[begin:end] = [L[:] for _ in range(begin, end)]
            self.seq_compressed[begin:end] = [C[:] for _ in range(begin, end)]

    def _runs(self):
        """Runs of slots with equal lengths (all of them, as a rule): (first, end, (length,
        packed) per row)."""
        L, C, n = self.seq_length, self.seq_compressed, self.slots
        if n and L.count(L[0]) == n and C.count(C[0]) == n:
            return [(0, n, list(zip(L[0], C[0])))]
        cuts = [s for s in range(n) if s == 0 or L[s] != L[s - 1] or C[s] != C[s - 1]]
        return [(s, end, list(zip(L[s], C[s]))) for s, end in zip(cuts, cuts[1:] + [n])]

    def _move_rows(self, source, moves, runs):
        """Launch ``moves`` from ``source``'s rows over its ``_runs`` (first, end, lengths)."""
        _dev.require_current(self._blocks[0])
        lib, stream = _lib.lib(), _dev.stream()
        parts = _launches(moves)
        for begin, end, per in runs:
            for part in parts:
                table, held = [], None
                for src, dst in part:
                    if dst == _lib.CACHE_HELD:
                        held = src
                    L, C = (0, 0) if src == _lib.CACHE_NONE else per[held if src == _lib.CACHE_HELD else src]
                    table.append((src, dst, C // BLOCK, L - C))
                rc = lib.nsn_cache_copy(source._store(), self._store(), self.heads, self.bits, begin, end,
                                        (_lib.CacheMove * len(table))(*table), len(table), stream)
                _lib.check(rc, "nsn_cache_copy")

    def _store(self):
        if self._c_store is None:
            sides = []
            for name in ("K", "V"):
                w = self._storage[name]
                sides.append(_lib.CacheSide(*(w[k].data_ptr() for k in ("codes", "norm", "min", "scale", "factor",
                                                                        "headers", "tail", "blocks"))))
            self._c_store = _lib.CacheStore(*sides, self.batch, self.block_cap, self.tail_cap, 2 * self.batch)
        return self._c_store

    # ------------------------------------------------------------------ attention
    def decode(self, slot, q, **kw):
        """Decode attention of q [B, Hq, 128] over the slot (packed blocks + tail;
        each sequence over its own length): (out, ctx).  A branch's sequences
        attend their prefix too, read once for all that share it
        (``shared_prefix_attention``; ctx is None)."""
        L = max(self.seq_length[slot])
        if self.prefix is not None:
            require(kw.pop("kernel", "fast") == "fast", "A branch decodes on the fast kernel")
            kw.setdefault("max_prefix_blocks", max(self.prefix_tokens[slot]) // BLOCK)
            out = _attn().shared_prefix_attention(q, self._prefix_sides[(slot, "K")], self._prefix_sides[(slot, "V")],
                                                  self.side(slot, "K"), self.side(slot, "V"), self.lengths(slot),
                                                  max_seq_len=L, **kw)
            return out, None
        return _attn().decode_attention(q, self.side(slot, "K"), self.side(slot, "V"), self.lengths(slot),
                                        max_seq_len=L, **kw)

    def prefill(self, slot, q, k_chunk, v_chunk, append=False, **kw):
        """Chunked-prefill attention of q [B, Hq, n, 128] over the slot's
        context plus the chunk's own K/V (not yet appended).  ``append=True``
        also appends the chunk to every sequence's tail in the same launch
        (k_chunk / v_chunk in the compute dtype; the tail rows get them
        rounded to the tail dtype, as ``append`` would).  bf16 chunks carry
        their softmax weights as bf16 hi + lo (``precise_weights``) while some
        sequence of the slot has less than one block of context: its first
        queries attend a handful of tokens."""
        require(self.prefix is None, "A branch decodes only: prefill the cache it branches from")
        kw.setdefault("precise_weights", min(self.seq_length[slot]) < BLOCK)
        kw.setdefault("max_ctx_len", max(self.seq_length[slot]))
        if append:
            n = k_chunk.shape[2]
            L, C = self.seq_length[slot], self.seq_compressed[slot]
            for b in range(self.batch):
                if L[b] - C[b] + n > self.tail_cap:
                    raise IntegrityError("Tail overflow: compress before appending more tokens")
                if L[b] + n > self.block_cap * BLOCK + self.tail_cap:
                    raise IntegrityError("Cache capacity exceeded")
            out = _attn().prefill_attention(q, self.side(slot, "K"), self.side(slot, "V"), self.lengths(slot),
                                            k_chunk, v_chunk, append=True, **kw)
            for b in range(self.batch):
                L[b] += n
            return out
        has_ctx = max(self.seq_length[slot]) > 0
        return _attn().prefill_attention(q, self.side(slot, "K") if has_ctx else None,
                                         self.side(slot, "V") if has_ctx else None, self.lengths(slot),
                                         k_chunk, v_chunk, **kw)


def _in_place_moves(parents):
    """(source, row) moves that make row i a copy of row parents[i] (-1:
    emptied), ordered so that every row is read before it is written and the
    moves of one source follow each other.  A cycle's first row is held
    (CACHE_HELD) until its last row takes it."""
    children = {}
    for i, p in enumerate(parents):
        if p >= 0 and p != i:
            children.setdefault(p, []).append(i)
    moves, cyclic = [], [False] * len(parents)
    state = [0] * len(parents)   # 1: on the present walk, 2: done
    cycles = []
    for i in range(len(parents)):
        walk = []
        while i >= 0 and state[i] == 0 and parents[i] != i:
            state[i] = 1
            walk.append(i)
            i = parents[i]
        if i >= 0 and state[i] == 1 and parents[i] != i:
            cycles.append(walk[walk.index(i):])
            for j in cycles[-1]:
                cyclic[j] = True
        for j in walk:
            state[j] = 2
    # the rows that hang off others, leaves first
    todo = [i for i, p in enumerate(parents) if p == i or p < 0 or cyclic[i]]
    order = []
    while todo:
        i = todo.pop()
        order.append(i)
        todo.extend(c for c in children.get(i, ()) if not cyclic[c])
    for i in reversed(order):
        moves.extend((i, c) for c in children.get(i, ()) if not cyclic[c])
    for c in cycles:   # row c[k] becomes row c[k + 1], the last one the first
        moves.append((c[0], _lib.CACHE_HELD))
        moves.extend((c[k + 1], c[k]) for k in range(len(c) - 1))
        moves.append((_lib.CACHE_HELD, c[-1]))
    return moves + [(-1, i) for i, p in enumerate(parents) if p < 0]


def _launches(moves):
    """Moves cut into launches' worth; a cycle stays whole.  Source -1 becomes
    CACHE_NONE."""
    out, part, cycle = [], [], []
    for src, dst in moves:
        held = src == _lib.CACHE_HELD and bool(cycle)
        m = (src if held or src >= 0 else _lib.CACHE_NONE, dst)
        if dst == _lib.CACHE_HELD or cycle:
            cycle.append(m)
            if not held:
                continue
            unit, cycle = cycle, []
        else:
            unit = [m]
        require(len(unit) <= _lib.CACHE_MAX_MOVES, f"A cycle of more than {_lib.CACHE_MAX_MOVES - 2} rows")
        if len(part) + len(unit) > _lib.CACHE_MAX_MOVES:
            out.append(part)
            part = []
        part = part + unit
    return out + [part] if part else out


def _attn():
    from . import kernels
    return kernels
