"""Sequences of different lengths: how they are packed into one row of tokens
(``PackedSequences``), and the paged key/value cache they are decoded over
(``PagedKV``). No counterpart in the reference, whose models take padded batches
and whose cache grows by concatenation
(oslo/models/gptj/modeling_gptj.py:205-233)."""

import numpy as np
import torch

from .fused_kernels_utils import FusedPackedAttention, FusedPagedDecodeAttention, FusedPagedKV

PACKED_BLOCK = 128  # positions of a sequence one block of the attention kernels takes
CUS = 256  # of an MI355X


class PackedSequences(object):
    """Sequences of ``lengths`` tokens (host integers, zero allowed) laid one
    behind the other along one row. Made once per batch, before any capture,
    and shared by every layer and by the backward: it holds, on ``device``, the
    list of 128-position blocks the attention kernels take their work from
    (``blocks``: int32 [2, n, 4]; the blocks with most keys first, then those
    with most queries left first), each token's position in its own sequence
    (``positions``) and the sequence it belongs to (``sequence``), both int32 [total]."""

    def __init__(self, lengths, device):
        lengths = [int(n) for n in lengths]
        if any(n < 0 for n in lengths):
            raise ValueError("PackedSequences: lengths must not be negative")
        self.lengths = tuple(lengths)
        self.total = sum(lengths)
        self.max_length = max(lengths, default=0)
        if self.total >= 2 ** 31:
            raise ValueError("PackedSequences: more than 2^31 - 1 tokens")
        n = np.asarray(lengths, dtype=np.int64)
        starts = np.concatenate([[0], np.cumsum(n)[:-1]]).astype(np.int64) if len(n) else n
        counts = -(-n // PACKED_BLOCK)
        owner = np.repeat(np.arange(len(n)), counts)
        block = np.arange(len(owner)) - np.repeat(np.cumsum(counts) - counts, counts)
        entries = np.zeros((len(owner), 4), dtype=np.int32)
        entries[:, 0], entries[:, 1], entries[:, 2] = starts[owner], n[owner], block
        keys = np.minimum((block + 1) * PACKED_BLOCK, n[owner])
        queries = n[owner] - block * PACKED_BLOCK
        order = [np.argsort(-keys, kind="stable"), np.argsort(-queries, kind="stable")]
        positions = np.arange(self.total, dtype=np.int32)
        positions -= np.repeat(starts.astype(np.int32), n)
        parts = [entries[np.concatenate(order)].ravel(), positions, np.repeat(np.arange(len(n), dtype=np.int32), n),
                 (starts + n - 1).astype(np.int32)]
        # (one copy, here: inside a capture, or on whatever stream asks first, none could be made)
        held = torch.from_numpy(np.concatenate(parts)).to(device).split([len(p) for p in parts])
        self.blocks = held[0].view(2, len(owner), 4)
        self.positions, self.sequence, self._last = held[1:]
        self._queries = queries[order[1]]  # of the blocks with most queries first: how many are left
        self._shared = {}
        self.kept = {}  # what the models look up for these sequences (rotary tables), for as long as they live

    @property
    def device(self):
        return self.blocks.device

    def shared_blocks(self, heads, kv_heads, head_dim, window=0):
        """(split, parts) for the gradients of keys and values: the first ``split``
        blocks of the list are worked on by ``parts`` kernel blocks each, which take
        the query heads of a group between them, because one alone would go on
        when the rest of the card has finished. Host arithmetic only."""
        key = (heads, kv_heads, head_dim, window)
        found = self._shared.get(key)
        if found is None:
            found = self._shared[key] = self._share(heads // kv_heads, kv_heads, 2 if head_dim == 64 else 1, window)
        return found

    def _share(self, group, kv_heads, blocks_per_cu, window):
        if group == 1 or not len(self._queries):
            return 0, 1
        # tiles of 32 queries a block walks per head, and two for its start and end
        tiles = -(-np.minimum(self._queries, window + PACKED_BLOCK - 1 if window else self._queries) // 32) + 2
        work = tiles * group
        average = work.sum() * kv_heads / (CUS * blocks_per_cu)  # a CU's, if it were spread evenly
        limit = 0.75 * average
        # (below a tenth more than the average the last blocks hide in the others' unevenness; the sums of a
        # shared block cost about 32 tiles of time)
        if work[0] <= max(1.1 * average, work[0] / group + 32):
            return 0, 1
        parts = next(p for p in range(2, group + 1) if group % p == 0 and (work[0] / p <= max(limit, 32) or p == group))
        return int((work > max(limit, 32)).sum()), parts

    def last_tokens(self):
        """int64 [sequences] on the device: the row of each sequence's last token
        (sequences must not be empty)."""
        if any(n == 0 for n in self.lengths):
            raise ValueError("PackedSequences: an empty sequence has no last token")
        return self._last.to(torch.int64)


class PagedKV(object):
    """One layer's key/value cache in pages: ``key_pages`` and ``value_pages``
    [num_pages, key/value heads, page_size, head_dim], and ``table`` int32
    [sequences, max_pages], the page that holds positions [i * page_size, (i + 1)
    * page_size) of each sequence. fp16 or bf16; or 8-bit (``float8_e4m3fn``) with
    ``key_scales`` and ``value_scales`` uint8 [num_pages, heads, page_size]: the
    power-of-two scale of each slot's vector, as its exponent + 127."""

    def __init__(self, key_pages, value_pages, table, key_scales=None, value_scales=None):
        if key_pages.dim() != 4 or key_pages.shape != value_pages.shape or key_pages.dtype != value_pages.dtype:
            raise ValueError("PagedKV: pages must be two [pages, heads, page_size, head_dim] tensors alike")
        if not (key_pages.is_contiguous() and value_pages.is_contiguous()):
            raise ValueError("PagedKV: pages must be contiguous")
        if table.dim() != 2 or table.dtype != torch.int32 or not table.is_contiguous():
            raise ValueError("PagedKV: the table must be a contiguous int32 [sequences, max_pages] tensor")
        self.quantized = key_pages.dtype == torch.float8_e4m3fn
        if not self.quantized and key_pages.dtype not in (torch.float16, torch.bfloat16):
            raise ValueError(f"PagedKV: pages of fp16, bf16 or float8_e4m3fn, not {key_pages.dtype}")
        scales = (key_scales, value_scales)
        if self.quantized:
            if not all(isinstance(s, torch.Tensor) and s.dtype == torch.uint8 and s.shape == key_pages.shape[:3]
                       and s.is_contiguous() for s in scales):
                raise ValueError("PagedKV: 8-bit pages need contiguous uint8 [pages, heads, page_size] scales")
        elif any(s is not None for s in scales):
            raise ValueError("PagedKV: scales go with 8-bit pages")
        tensors = [value_pages, table] + [s for s in scales if s is not None]
        if any(t.device != key_pages.device for t in tensors):
            raise ValueError("PagedKV: pages, table and scales must be on one device")
        self.key_pages, self.value_pages, self.table = key_pages, value_pages, table
        self.key_scales, self.value_scales = scales

    @property
    def page_size(self):
        return self.key_pages.shape[2]

    @classmethod
    def allocate(cls, table, num_pages, kv_heads, page_size, head_dim, dtype, device, quantized=False):
        """An empty cache of ``num_pages`` pages under ``table`` (layers that grow
        together share one table)."""
        shape = (num_pages, kv_heads, page_size, head_dim)
        if not quantized:
            return cls(torch.zeros(shape, dtype=dtype, device=device), torch.zeros(shape, dtype=dtype, device=device),
                       table)
        pages = [torch.zeros(shape, dtype=torch.uint8, device=device).view(torch.float8_e4m3fn) for _ in range(2)]
        scales = [torch.full(shape[:3], 127, dtype=torch.uint8, device=device) for _ in range(2)]
        return cls(*pages, table, *scales)


class SequenceLayer(object):
    """What a fused attention module is handed as ``layer_past`` when its tokens
    [1, T] belong to sequences of different lengths: ``attend`` takes query
    [T, H, D], key and value [T, Hkv, D] and returns [T, H, D]; ``positions``
    (int32 on the device) are the tokens' positions in their sequences, all
    below ``max_position``; ``shared`` holds what the layers of one forward
    work out once, ``kept`` what stays for the next one."""

    positions = max_position = shared = kept = None

    def row_positions(self, tokens):
        """``positions`` for a row of ``tokens``: 0 behind the last sequence (such
        rows are computed and seen by nobody)."""
        extra = tokens - self.positions.numel()
        if extra < 0:
            raise ValueError(f"{self.positions.numel()} tokens of sequences in a row of {tokens}")
        return torch.cat([self.positions, self.positions.new_zeros(extra)]) if extra else self.positions

    def attend(self, query, key, value, scale, window=None):
        raise NotImplementedError


class PackedLayer(SequenceLayer):
    """Whole sequences packed into the row (prompts or training documents);
    with ``cache`` their keys and values also go into that layer's ``PagedKV``."""

    def __init__(self, packed, cache, shared):
        self.packed, self.cache, self.shared, self.kept = packed, cache, shared, packed.kept
        self.positions, self.max_position = packed.positions, packed.max_length

    def attend(self, query, key, value, scale, window=None):
        if self.cache is not None:
            n = self.packed.total
            FusedPagedKV.write(self.cache, key[:n], value[:n], self.packed.sequence, self.packed.positions)
        return FusedPackedAttention.apply(query, key, value, self.packed, scale, window)


class PagedState(object):
    """The layers' paged caches while one token per sequence is decoded at a
    time, under one table, with pages for ``capacity`` positions of each sequence.
    ``lengths`` (int32 [sequences] on the device) is the position of the token being
    fed: the number of positions written, or the last position of a sequence that is
    full, which its next tokens overwrite. Nothing in a step depends
    on the host, so a step can be captured into a graph and replayed."""

    def __init__(self, lengths, capacity, layers, kv_heads, head_dim, dtype, device, page_size=64, quantized=False):
        self.capacity = int(capacity)
        if self.capacity < 1 or any(not 0 <= n <= self.capacity for n in lengths):
            raise ValueError("PagedState: lengths from zero to a capacity of at least one position")
        each = -(-self.capacity // page_size)
        num_pages = len(lengths) * each
        self.table = torch.arange(num_pages, dtype=torch.int32, device=device).view(len(lengths), each)
        # (a sequence that is full feeds its next token to its last position, like one that gets there by steps)
        self.lengths = torch.tensor([min(int(n), self.capacity - 1) for n in lengths], dtype=torch.int32, device=device)
        self.visible = self.lengths + 1
        self.rows = torch.arange(len(lengths), dtype=torch.int32, device=device)
        self.step_values = {}  # what layers share within one step
        self.kept = {}  # what outlives a step: the rotary tables, which a captured step reads
        self.caches = [PagedKV.allocate(self.table, num_pages, kv_heads, page_size, head_dim, dtype, device, quantized)
                       for _ in range(layers)]

    def prompt_layers(self, packed):
        """``layer_past`` of every layer for the prompts, packed into one row."""
        if len(packed.lengths) > self.table.shape[0] or packed.max_length > self.capacity:
            raise ValueError(f"PagedState: {len(packed.lengths)} prompts of up to {packed.max_length} tokens, places for "
                             f"{self.table.shape[0]} of up to {self.capacity}")
        shared = {}
        return [PackedLayer(packed, cache, shared) for cache in self.caches]

    def begin_step(self):
        """``layer_past`` of every layer for the next tokens, [1, sequences]."""
        self.step_values.clear()
        torch.add(self.lengths, 1, out=self.visible)
        return [PagedLayer(self, cache) for cache in self.caches]

    def end_step(self):
        """The tokens are in the cache."""
        self.lengths.add_(1).clamp_(max=self.capacity - 1)


class PagedLayer(SequenceLayer):
    """One new token per sequence over a layer's paged cache."""

    def __init__(self, state, cache):
        self.state, self.cache, self.shared, self.kept = state, cache, state.step_values, state.kept
        self.positions, self.max_position = state.lengths, state.capacity

    def attend(self, query, key, value, scale, window=None):
        FusedPagedKV.write(self.cache, key, value, self.state.rows, self.state.lengths)
        return FusedPagedDecodeAttention.apply(query, self.cache, self.state.visible, scale, window)


def sequence_layers(packed, layers):
    """``layer_past`` of every layer for tokens packed into one row."""
    shared = {}
    return [PackedLayer(packed, None, shared) for _ in range(layers)]


def packed_labels(labels, packed):
    """Targets of a packed row: the next token of the same sequence; -100 (no
    target) at a sequence's last token and behind the last sequence."""
    targets = torch.full_like(labels, -100)
    if packed.total > 1:
        first = packed.positions[1:] == 0
        targets[..., :packed.total - 1] = labels[..., 1:packed.total].masked_fill(first, -100)
    return targets
