"""Exact attention over the hot pool for a batch whose sequences share
prefixes (``weaver_prefix_*``): personas behind one system prompt, candidates
of one question, drafts of one context.

The sequences are grouped; each group's prefix pages are read once for 256 rows
(queries x query heads of a kv head) of the group's queries together, and by a
sequence with 512 rows or more for itself.  Lengths are in tokens and live on the device, so one
plan (and one captured graph) serves a batch while its sequences grow within
their pages.  One token per sequence, draft batches and prompt chunks may be
mixed in one call::

    plan = PrefixPlan(engine, q_heads=32, kv_heads=8, head_dim=128, scale=128 ** -0.5,
                      q_indptr=[0, 1, 2, 10], suffix_indptr=[0, 4, 8, 12],    # 3 sequences, 1 + 1 + 8 queries
                      group_indptr=[0, 3], prefix_indptr=[0, 2048])           # one group, a prefix of 2048 pages
    plan.run(q=q_out, hot_k=hot_k, hot_v=hot_v, prefix_refs=prefix_refs, suffix_refs=suffix_refs,
             prefix_lens=prefix_lens, suffix_lens=suffix_lens, out=out)

With ``partials=True`` the run writes (m, l, o) instead, to be merged
(``merge_partials``) with those of a ``WeaverPlan`` over the cold blocks of the
same queries.
"""
from __future__ import annotations

import ctypes
import struct

import numpy as np

from . import _native as N
from .types import BLOCK_SIZE
from .weaver import WeaverEngine, raw_stream

_VIEWS = struct.Struct("=12Q").pack  # weaver_prefix_views
assert struct.calcsize("=12Q") == ctypes.sizeof(N.PrefixViewsC)


def _indptr(name, x) -> np.ndarray:
    a = np.asarray(x)
    if a.ndim != 1 or a.size < 2 or not np.issubdtype(a.dtype, np.integer):
        raise ValueError(f"{name} must be a list of at least two whole numbers")
    if int(a.min()) < 0 or int(a.max()) >= 1 << 32:
        raise ValueError(f"{name} has entries outside 0 .. 2^32 - 1")
    return np.ascontiguousarray(a, dtype=np.uint32)


class PrefixPlan:
    """A plan over groups of sequences (``weaver_prefix_plan_create``).
    ``q_indptr`` (queries) and ``suffix_indptr`` (own pages) have one entry per
    sequence and one more; ``group_indptr`` (sequences) and ``prefix_indptr``
    (prefix pages) one per group and one more.  Without groups every sequence
    is on its own and has no prefix.  Query j of a sequence's nq sees its whole
    prefix and, with ``causal``, the first ``suffix_len - nq + 1 + j`` of its
    own tokens, else all of them."""

    def __init__(self, engine: WeaverEngine, *, q_heads: int, kv_heads: int, head_dim: int, scale: float, q_indptr,
                 suffix_indptr, group_indptr=None, prefix_indptr=None, causal: bool = True, partials: bool = False):
        qi, si = _indptr("q_indptr", q_indptr), _indptr("suffix_indptr", suffix_indptr)
        B = qi.size - 1
        if si.size != B + 1:
            raise ValueError("q_indptr and suffix_indptr differ in length")
        if (group_indptr is None) != (prefix_indptr is None):
            raise ValueError("group_indptr and prefix_indptr come together")
        gi = _indptr("group_indptr", np.array([0, B]) if group_indptr is None else group_indptr)
        pi = _indptr("prefix_indptr", np.array([0, 0]) if prefix_indptr is None else prefix_indptr)
        if gi.size != pi.size:
            raise ValueError("group_indptr and prefix_indptr differ in length")
        flags = (N.FLAG_CAUSAL if causal else 0) | (N.FLAG_PARTIALS if partials else 0)
        self.shape = N.PrefixShapeC(gi.size - 1, B, q_heads, kv_heads, head_dim, float(scale), flags)
        h = ctypes.c_void_p()
        N.check(N.lib().weaver_prefix_plan_create(engine.handle, ctypes.byref(self.shape), qi.ctypes.data,
                                                  gi.ctypes.data, pi.ctypes.data, si.ctypes.data, ctypes.byref(h)))
        self._h = h
        self.device, self.partials = engine.device, partials
        self.n_tokens, self.n_prefix_pages, self.n_suffix_pages = int(qi[-1]), int(pi[-1]), int(si[-1])
        import torch
        self._f16, self._f32, self._words = (torch.float16,), (torch.float32,), (torch.int32, torch.uint32)
        self.n_groups, self.n_seqs = gi.size - 1, B
        self._heads, self._page = (q_heads, head_dim), (BLOCK_SIZE, kv_heads, head_dim)
        self._rows, self._values = self.n_tokens * q_heads, self.n_tokens * q_heads * head_dim

    def close(self) -> None:
        if getattr(self, "_h", None):
            N.lib().weaver_prefix_plan_destroy(self._h)
            self._h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    @property
    def kernel_count(self) -> int:
        return N.lib().weaver_prefix_plan_kernel_count(self._h)

    def _ptr(self, name, t, dtypes, numel, tail=None):
        if t is None or isinstance(t, int):
            return t or 0
        if t.get_device() != self.device:
            raise ValueError(f"{name} must be a CUDA tensor on device {self.device}")
        if t.dtype not in dtypes:
            raise ValueError(f"{name} is {t.dtype}")
        if not t.is_contiguous():
            raise ValueError(f"{name} must be contiguous")
        if tail is not None and t.shape[1:] != tail:
            raise ValueError(f"{name} has shape {tuple(t.shape)}, expected [..., {', '.join(map(str, tail))}]")
        if t.numel() < numel:
            raise ValueError(f"{name} has {t.numel()} elements, the plan needs {numel}")
        return t.data_ptr()

    def views(self, *, q, hot_k, hot_v, prefix_refs=None, suffix_refs=None, prefix_lens=None, suffix_lens=None, out=None,
              part_m=None, part_l=None, part_o=None, hot_pool_blocks=None) -> bytes:
        """The C views (``weaver_prefix_views``) of CUDA tensors, kept for
        repeated runs (raw addresses: the tensors have to live until the last run
        with them is over): ``q`` / ``out [tokens, Hq, d]`` f16, ``hot_k`` / ``hot_v
        [blocks, 16, Hkv, d]`` f16 (or raw pointers with ``hot_pool_blocks``),
        refs and lengths int32 or uint32, partials fp32."""
        if hot_pool_blocks is None:
            if isinstance(hot_k, int):
                raise ValueError("raw pool pointers need hot_pool_blocks")
            hot_pool_blocks = 0 if hot_k is None else hot_k.shape[0]
        for name, pool in (("hot_k", hot_k), ("hot_v", hot_v)):
            if hasattr(pool, "shape") and pool.shape[0] < hot_pool_blocks:
                raise ValueError(f"{name} has fewer than {hot_pool_blocks} blocks")
        ptr, n = self._ptr, self._rows
        return _VIEWS(ptr("q", q, self._f16, self._values, self._heads), ptr("hot_k", hot_k, self._f16, 0, self._page),
                      ptr("hot_v", hot_v, self._f16, 0, self._page), hot_pool_blocks,
                      ptr("prefix_refs", prefix_refs, self._words, self.n_prefix_pages),
                      ptr("suffix_refs", suffix_refs, self._words, self.n_suffix_pages),
                      ptr("prefix_lens", prefix_lens, self._words, self.n_groups),
                      ptr("suffix_lens", suffix_lens, self._words, self.n_seqs),
                      ptr("out", out, self._f16, self._values, self._heads), ptr("part_m", part_m, self._f32, n),
                      ptr("part_l", part_l, self._f32, n), ptr("part_o", part_o, self._f32, self._values))

    def run_views(self, views: bytes, stream=None) -> None:
        N.check(N.lib().weaver_prefix_run(self._h, views, raw_stream(stream, self.device)))

    def run(self, stream=None, **tensors) -> None:
        """One attention over the batch on ``stream`` (default: torch's current
        stream).  Only one run of a plan may be in flight at a time."""
        self.run_views(self.views(**tensors), stream)

    def status(self) -> None:
        """Wait for the device's work, replayed graphs included, and raise
        ``WeaverError`` if a run met a block reference beyond the pool or a
        length beyond its pages."""
        N.check(N.lib().weaver_prefix_plan_status(self._h))


__all__ = ["PrefixPlan"]
