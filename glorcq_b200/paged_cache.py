"""Paged key/value cache held in 8 bits, with a length of its own for every sequence.

The reference decodes over transformers' static fp16 cache with one position for the whole batch
(inference/graph_wrapper.py:41-47, 84-127; ``decoder.StaticKVCache`` here).  This cache takes half of its bytes, hands memory out in
pages, and lets the sequences of a batch have lengths of their own:

    q = paged_append(q, k, v, cos, sin, *cache, start)      # norms, rotation, keys and values into the pages
    y = paged_attention(q, *cache, start)                   # causal attention over the pages
    k, v = paged_read(*cache, first, row_start, n_rows)     # rows back as fp16

``cache`` is (k_pages, v_pages, k_scale, v_scale, page_table): codes (pages, kv heads, tokens, channels) in ``torch.int8`` or
``torch.float8_e4m3fn``, one fp32 scale for each (page, kv head), and the (B, pages) int32 table of each sequence's pages.
``PagedKVCache`` owns these for all layers of a model, and is a ``past_key_values`` of ``GLoRCQDecoder`` and
``GLoRCQGraphWrapper``.  The definitions (positions, block scales, what happens to invalid pages) are those of glq_paged_append,
glq_paged_attention and glq_paged_read in include/glorcq_b200.h.
"""

from __future__ import annotations

import ctypes

import torch

from . import _lib

DTYPES = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}
PAGE_SIZES, HEAD_SIZES = (16, 32, 64, 128), (32, 64, 128, 256)


def paged_append(q, k, v, cos, sin, k_pages, v_pages, k_scale, v_scale, page_table, start, q_start=None, q_norm=None, k_norm=None,
                 eps=1e-6, q_out=None):
    """Write the new keys and values k, v (N, kv heads, D) fp16 into the pages and return the rotated queries (N, heads, D) fp16.

    Sequence b holds ``start[b]`` tokens ((B,) or (1,) int64, on the device) and gets rows ``q_start[b] .. q_start[b + 1]`` ((B + 1,)
    int32; None: N / B each).  ``cos`` / ``sin`` ((positions, D / 2) fp32) may be None (no rotation), ``q_norm`` / ``k_norm`` ((D,) fp16) are the
    weights of per-head RMS norms, ``q`` may be None (returns None), ``q_out`` may be q itself.  Rows of no sequence are not written.  A page that
    the call writes belongs to one sequence."""
    return _lib.native().paged_append(q, k, v, cos, sin, k_pages, v_pages, k_scale, v_scale, page_table, start, q_start, q_norm, k_norm,
                                      eps, q_out)


def paged_attention(q, k_pages, v_pages, k_scale, v_scale, page_table, start, q_start=None, max_new=None, scale=None, out=None):
    """Causal attention of the rows q (N, heads, D) fp16, already rotated and in the cache, over keys 0 .. the row's own position.

    ``max_new``: at least the most rows of one sequence, known to the host (None: N); with ``q_start`` it chooses the kernel.  ``scale``: of the scores
    (None: D ** -0.5).  Returns (N, heads, D) fp16; rows of no sequence are not written."""
    return _lib.native().paged_attention(q, k_pages, v_pages, k_scale, v_scale, page_table, start, q_start,
                                         -1 if max_new is None else max_new, q.shape[-1] ** -0.5 if scale is None else scale, out)


def paged_read(k_pages, v_pages, k_scale, v_scale, page_table, start, q_start, rows):
    """Keys and values (rows, kv heads, D) fp16 of positions ``start[b] ..`` of every sequence: rows ``q_start[b] .. q_start[b + 1]``
    are sequence b's (None: rows / B each); rows of no sequence are not written."""
    return _lib.native().paged_read(k_pages, v_pages, k_scale, v_scale, page_table, start, q_start, rows)


def rope_tables(head_dim, positions, theta, device):
    """(cos, sin), each (positions, head_dim / 2) fp32; angles in 64 bits, so that far positions keep theirs."""
    freq = float(theta) ** (-torch.arange(0, head_dim, 2, device=device, dtype=torch.float64) / head_dim)
    angle = torch.outer(torch.arange(positions, device=device, dtype=torch.float64), freq)
    return angle.cos().float(), angle.sin().float()


class PagedKVCache:
    """Pages of all layers of a model, and who has which.

    ``dtype``: "int8" or "e4m3".  The error of a value, by the scale s of its block (one head's tokens of a page): below s with "int8", at most
    s / 2 where one call wrote the whole block; at most 2^-4 of the value and 2^-9 s with "e4m3".  s is the block's largest magnitude / 127 (448) where one call
    wrote it, and below twice that where tokens came one by one and its scale was doubled on the way.
    ``num_pages`` None: pages for every sequence's ``max_cache_len`` tokens, handed out at once; otherwise that many for all,
    and ``reserve`` / ``release`` hand them out and take them back.  The page table is device memory that captured calls read when they
    run."""

    def __init__(self, config, max_batch_size, max_cache_len, device, dtype="int8", page_size=64, num_pages=None):
        if dtype not in DTYPES:
            raise RuntimeError(f"paged cache: dtype must be one of {', '.join(DTYPES)}, got {dtype}")
        if page_size not in PAGE_SIZES:
            raise RuntimeError(f"paged cache: pages hold 16, 32, 64 or 128 tokens, got {page_size}")
        c = config
        if c.head_dim not in HEAD_SIZES:
            raise RuntimeError(f"paged cache: head sizes are 32, 64, 128 and 256, got {c.head_dim}")
        self.max_batch_size, self.max_cache_len, self.page_size = max_batch_size, max_cache_len, page_size
        self.max_pages = -(-max_cache_len // page_size)
        self.device = torch.device(device)
        n = max_batch_size * self.max_pages if num_pages is None else num_pages
        pages = (c.num_hidden_layers, n, c.num_key_value_heads, page_size, c.head_dim)
        self.k, self.v = (torch.zeros(pages, dtype=torch.uint8, device=device).view(DTYPES[dtype]) for _ in range(2))
        self.k_scale, self.v_scale = (torch.zeros(pages[:3], dtype=torch.float32, device=device) for _ in range(2))
        self.page_table = torch.full((max_batch_size, self.max_pages), -1, dtype=torch.int32, device=device)
        self.cos, self.sin = rope_tables(c.head_dim, self.max_pages * page_size, c.rope_theta, device)
        self._free = list(range(n - 1, -1, -1))
        self._owned = [[] for _ in range(max_batch_size)]
        self._layers = {}
        if num_pages is None:
            for b in range(max_batch_size):
                self.reserve(b, max_cache_len)

    def reserve(self, sequence, length):
        """Give the sequence the pages that ``length`` tokens need."""
        have = self._owned[sequence]
        want = -(-length // self.page_size) - len(have)
        if want <= 0:
            return
        if length > self.max_pages * self.page_size:
            raise RuntimeError(f"paged cache: {length} tokens of a sequence are more than {self.max_pages * self.page_size}")
        if want > len(self._free):
            raise RuntimeError(f"paged cache: {want} pages are wanted and {len(self._free)} are free")
        new = [self._free.pop() for _ in range(want)]
        self.page_table[sequence, len(have):len(have) + want] = torch.tensor(new, dtype=torch.int32).to(self.device)
        have.extend(new)

    def release(self, sequence):
        """Take the sequence's pages back."""
        self.page_table[sequence].fill_(-1)
        self._free.extend(reversed(self._owned[sequence]))
        self._owned[sequence] = []

    def reset(self):
        """Forget all tokens; the sequences keep their pages (a block whose first slot is written starts anew)."""
        self.k_scale.zero_()
        self.v_scale.zero_()

    def layer(self, layer, batch):
        """(k_pages, v_pages, k_scale, v_scale, page_table) of one layer for the first ``batch`` sequences."""
        got = self._layers.get((layer, batch))
        if got is None:
            if batch > self.max_batch_size:
                raise RuntimeError(f"paged cache: {batch} sequences are more than {self.max_batch_size}")
            got = self._layers[layer, batch] = (self.k[layer], self.v[layer], self.k_scale[layer], self.v_scale[layer], self.page_table[:batch])
        return got

    def append(self, layer, q, k, v, start, batch, q_start=None, q_norm=None, k_norm=None, eps=1e-6):
        return paged_append(q, k, v, self.cos, self.sin, *self.layer(layer, batch), start, q_start, q_norm, k_norm, eps)

    def attend(self, layer, q, start, batch, q_start=None, max_new=None):
        return paged_attention(q, *self.layer(layer, batch), start, q_start, max_new)

    def read(self, layer, sequence, first, count):
        """Keys and values (count, kv heads, D) fp16 of ``count`` tokens of one sequence from position ``first`` on."""
        pages = self.layer(layer, self.max_batch_size)
        return paged_read(*pages[:4], self.page_table[sequence:sequence + 1], torch.tensor([first], dtype=torch.int64, device=self.device),
                          None, count)

    def snapshot(self, n):
        """What the first ``n`` positions of every sequence hold, for ``restore``."""
        ids = self.page_table[:, : -(-n // self.page_size)].reshape(-1).long()
        ids = ids[(ids >= 0) & (ids < self.k.shape[1])]       # (what is no page is nobody's)
        return ids, [t[:, ids].clone() for t in self._tensors()]

    def restore(self, kept):
        ids, values = kept
        for t, x in zip(self._tensors(), values):
            t[:, ids] = x

    def raise_on_error(self):
        """To be called where the host synchronises anyway (``GLoRCQGraphWrapper.generate`` does): raises where a wait in one of the cache's kernels
        on this device has run out since the last look, which left rows of its call incomplete."""
        word = (ctypes.c_ulonglong * 4)()
        with torch.cuda.device(self.device):
            _lib.check(_lib.lib().glq_paged_error(word, 1), "paged_error")
        if word[0]:
            raise RuntimeError(f"paged cache: a wait ran out (code {word[0]}, thread {word[3] & 0xffffffff} of block {word[3] >> 32}); results since the last look may be incomplete")

    def _tensors(self):
        return self.k.view(torch.uint8), self.v.view(torch.uint8), self.k_scale, self.v_scale
