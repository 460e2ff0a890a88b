"""Position rotation of query and key heads and the append into the paged hot
pool (``weaver_rope_*``).

The hot pool holds rotated keys.  :meth:`Rope.append` makes them where they are
needed: in one kernel it rotates (and, with weights, first RMS-norms) the
query and key heads of a batch of new tokens, writes K and V into the tokens'
slots of the hot pool and q where the attention of the same stream reads it
(``WeaverPlan.run``, ``PrefixPlan.run``).  :meth:`Rope.rotate` is the same
without the pool, for keys that live in a flat cache
(``WeaverEngine.multihead_attention``).

A decode step of a batch::

    rope = Rope(engine, head_dim=128, theta=500000.0)
    slots = token_slots(refs, indptr, lens, q_indptr)          # host; or kept on the device
    rope.append(q, k, v, positions, slots, hot_k, hot_v, q_out, bad_flag)
    plan.run(q=q_out, hot_k=hot_k, hot_v=hot_v, ...)

The reference's rotation is ``ops.metal:107-160``, its append to a flat cache
``inference.rs:504-562``.
"""
from __future__ import annotations

import ctypes
import math
import struct

import numpy as np

from . import _native as N
from .types import BLOCK_SIZE, REF_MASK
from .weaver import raw_stream

LAYOUTS = {"half": N.ROPE_HALF, "interleaved": N.ROPE_INTERLEAVED}
# weaver_rope_views as bytes in one go: a call made every layer spends its time in the host
_VIEWS = struct.Struct("=4I3Q6Q3QfI2Q4Q4QQ").pack
assert struct.calcsize("=4I3Q6Q3QfI2Q4Q4QQ") == ctypes.sizeof(N.RopeViewsC)


def rope_frequencies(rot_dim: int, theta: float = 10000.0, scaling: dict | None = None) -> tuple[np.ndarray, float]:
    """(radians per position of every pair, factor on cosines and sines) in
    64 bits.  ``scaling`` stretches the rotation for contexts beyond the
    trained one, ``{"type": ..., "factor": s, ...}``:

    * ``linear``: every frequency / s;
    * ``ntk``: theta * s^(r / (r - 2)), so the slowest pair is scaled by s and
      the fastest not at all;
    * ``yarn`` (Peng et al. 2023; ``original_length``, ``beta_fast`` = 32,
      ``beta_slow`` = 1): pairs that turn more than beta_fast times over the
      original length keep their frequency, those below beta_slow times take
      f / s, a linear ramp over the pair index between; cosines and sines
      times ``attention_factor`` (default 0.1 ln s + 1);
    * ``bands`` (``original_length``, ``low`` = 1, ``high`` = 4): f / s where
      the wavelength exceeds original_length / low, f where it is below
      original_length / high, between them interpolated in the number of
      turns."""
    if rot_dim < 0 or rot_dim % 2:
        raise ValueError(f"rot_dim {rot_dim}")
    if not (math.isfinite(theta) and theta > 0):
        raise ValueError(f"theta {theta}")
    i = np.arange(rot_dim // 2, dtype=np.float64)
    f = float(theta) ** (-2.0 * i / max(rot_dim, 1))
    if not scaling:
        return f, 1.0
    kind = scaling.get("type")
    known = {"linear": set(), "ntk": set(), "yarn": {"original_length", "beta_fast", "beta_slow", "attention_factor"},
             "bands": {"original_length", "low", "high"}}
    if kind not in known:
        raise ValueError(f"unknown rope scaling {kind!r}")
    extra = set(scaling) - known[kind] - {"type", "factor"}
    if extra:
        raise ValueError(f"rope scaling {kind!r} does not take {sorted(extra)}")

    def positive(name, default=None):
        x = scaling.get(name, default)
        if x is None:
            raise ValueError(f"rope scaling {kind!r} needs {name}")
        x = float(x)
        if not (math.isfinite(x) and x > 0):
            raise ValueError(f"rope scaling {name} {x}")
        return x

    s = positive("factor")
    if kind == "linear":
        return f / s, 1.0
    if kind == "ntk":
        if rot_dim <= 2:
            raise ValueError("ntk scaling needs rot_dim > 2")
        return (float(theta) * s ** (rot_dim / (rot_dim - 2.0))) ** (-2.0 * i / rot_dim), 1.0
    length = positive("original_length")
    turns = length * f / (2.0 * math.pi)  # of each pair over the original length
    if kind == "yarn":
        if theta == 1.0:
            raise ValueError("yarn scaling needs theta != 1")
        fast, slow = positive("beta_fast", 32.0), positive("beta_slow", 1.0)

        def pair_of(n):  # the (fractional) pair that turns n times
            return rot_dim * math.log(length / (n * 2.0 * math.pi)) / (2.0 * math.log(theta))
        # the ramp may end behind the last pair (the method bounds its end by rot_dim - 1): the last pairs
        # then still turn more than `slow` times and are mixed, not scaled whole
        low, high = max(math.floor(pair_of(fast)), 0), min(math.ceil(pair_of(slow)), rot_dim - 1)
        ramp = np.clip((i - low) / max(high - low, 1e-3), 0.0, 1.0)
        factor = scaling.get("attention_factor")
        return f * (1.0 - ramp) + f / s * ramp, (0.1 * math.log(s) + 1.0) if factor is None else float(factor)
    lo, hi = float(scaling.get("low", 1.0)), float(scaling.get("high", 4.0))
    if not hi > lo:
        raise ValueError("bands scaling needs high > low")
    keep = np.clip((turns - lo) / (hi - lo), 0.0, 1.0)
    return f * keep + f / s * (1.0 - keep), 1.0


def token_slots(refs, indptr, lens, q_indptr) -> np.ndarray:
    """Pool slots of the batch's new tokens (host arrays in, int64 out): the
    queries ``q_indptr[b] .. q_indptr[b+1]`` of sequence b are the tokens that
    follow its first ``lens[b]``, in the pages ``refs[indptr[b]:indptr[b+1]]``."""
    refs = np.asarray(refs, np.uint32) & np.uint32(REF_MASK)
    B = len(lens)
    for name, x in (("indptr", np.asarray(indptr)[:B + 1]), ("q_indptr", np.asarray(q_indptr))):
        if x.shape != (B + 1,) or x[0] < 0 or (x[1:] < x[:-1]).any():
            raise ValueError(f"{name} is not a non-decreasing list of an entry per sequence and one more")
    if int(q_indptr[0]) or any(int(n) < 0 for n in lens):
        raise ValueError("q_indptr[0] is not 0, or a length is negative")
    out = np.empty(int(q_indptr[-1]), np.int64)
    for b in range(len(lens)):
        n = int(q_indptr[b + 1]) - int(q_indptr[b])
        idx = int(lens[b]) + np.arange(n, dtype=np.int64)
        pages = refs[int(indptr[b]):int(indptr[b + 1])]
        if n and int(idx[-1]) >= len(pages) * BLOCK_SIZE:
            raise ValueError(f"sequence {b} needs {int(idx[-1]) // BLOCK_SIZE + 1} pages and has {len(pages)}")
        out[int(q_indptr[b]):int(q_indptr[b + 1])] = pages[idx // BLOCK_SIZE].astype(np.int64) * BLOCK_SIZE + \
            idx % BLOCK_SIZE
    return out


class Rope:
    """The rotation of one head geometry (see :func:`rope_frequencies` for
    ``theta`` and ``scaling``; ``inv_freq`` gives the frequencies directly).
    ``layout`` pairs element i with i + rot_dim/2 (``"half"``) or 2i with 2i+1
    (``"interleaved"``); elements from ``rot_dim`` on are not rotated."""

    def __init__(self, engine, *, head_dim: int, rot_dim: int | None = None, theta: float = 10000.0,
                 layout: str = "half", scaling: dict | None = None, inv_freq=None, amplitude: float | None = None):
        import torch
        rot_dim = head_dim if rot_dim is None else int(rot_dim)
        if layout not in LAYOUTS:
            raise ValueError(f"layout {layout!r}, not one of {sorted(LAYOUTS)}")
        if inv_freq is None:
            f, amp = rope_frequencies(rot_dim, theta, scaling)
        elif scaling is not None:
            raise ValueError("inv_freq and scaling exclude each other")
        else:
            f, amp = np.asarray(inv_freq, np.float64), 1.0
        f = np.ascontiguousarray(f, dtype=np.float64)
        if f.shape != (rot_dim // 2,):
            raise ValueError(f"inv_freq needs rot_dim / 2 = {rot_dim // 2} values")
        self.inv_freq, self.amplitude = f, amp if amplitude is None else float(amplitude)
        self.head_dim, self.rot_dim, self.layout, self.device = int(head_dim), rot_dim, layout, engine.device
        c = N.RopeConfigC(self.head_dim, rot_dim, LAYOUTS[layout], self.amplitude, f.ctypes.data)
        h = ctypes.c_void_p()
        N.check(N.lib().weaver_rope_create(engine.handle, ctypes.byref(c), ctypes.byref(h)))
        self._h = h
        self._types = {torch.float16: N.F16, torch.bfloat16: N.BF16}
        self._f16, self._i32, self._i64 = torch.float16, torch.int32, torch.int64

    def close(self) -> None:
        if getattr(self, "_h", None):
            N.lib().weaver_rope_destroy(self._h)
            self._h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def _refuse(self, name, t, shape, dtype):
        """Says what is wrong with a tensor that failed its check."""
        if t is None:
            raise ValueError(f"{name} is missing")
        if not t.is_cuda or t.get_device() != self.device:
            raise ValueError(f"{name} must be a CUDA tensor on device {self.device}")
        if t.dtype != dtype:
            raise ValueError(f"{name} is {t.dtype}, not {dtype}")
        if tuple(t.shape) != tuple(shape):
            raise ValueError(f"{name} has shape {tuple(t.shape)}, not {tuple(shape)}")
        raise ValueError(f"the last dimension of {name} must be contiguous")

    def _heads(self, name, t, shape, dtype):
        """(pointer, token stride, head stride) of a [tokens, heads, head_dim] tensor."""
        if t is None:
            self._refuse(name, t, shape, dtype)
        st = t.stride() if t.dim() == 3 else (0, 0, 0)
        if t.shape != shape or t.dtype != dtype or t.get_device() != self.device or st[2] != 1:
            self._refuse(name, t, shape, dtype)
        return t.data_ptr(), st[0], st[1]

    def _flat(self, name, t, n, dtype):
        if t is None or t.shape != (n,) or t.dtype != dtype or t.get_device() != self.device or (n > 1 and t.stride(0) != 1):
            self._refuse(name, t, (n,), dtype)
        return t.data_ptr()

    def _inputs(self, q, k, positions, q_weight, k_weight, q_out, out_dtype):
        """Tokens, heads, type code, and the views of q, k, positions, the weights and q_out."""
        lead = q if q is not None else k
        if lead is None:
            raise ValueError("neither q nor k given")
        if lead.dim() != 3:
            raise ValueError("heads are [tokens, heads, head_dim] tensors")
        dt, T, d = lead.dtype, lead.shape[0], self.head_dim
        if dt not in self._types:
            raise ValueError(f"heads are {dt}, not float16 or bfloat16")
        hq, qv, qo = 0, (0, 0, 0), (0, 0, 0)
        if q is not None:
            hq = q.shape[1]
            qv = self._heads("q", q, (T, hq, d), dt)
            qo = self._heads("q_out", q_out, (T, hq, d), out_dtype or dt)
        hkv, kv = 0, (0, 0, 0)
        if k is not None:
            if k.dim() != 3:
                raise ValueError("heads are [tokens, heads, head_dim] tensors")
            hkv = k.shape[1]
            kv = self._heads("k", k, (T, hkv, d), dt)
        return (T, hq, hkv, dt, qv, kv, qo, self._flat("positions", positions, T, self._i32),
                0 if q_weight is None else self._flat("q_weight", q_weight, d, dt),
                0 if k_weight is None else self._flat("k_weight", k_weight, d, dt))

    def rotate(self, q, k, positions, q_out, k_out=None, *, q_weight=None, k_weight=None, eps: float = 1e-6,
               stream=None) -> None:
        """``q_out`` / ``k_out`` = the rotated (with a weight: normed, then
        rotated) ``q [T, Hq, d]`` / ``k [T, Hkv, d]`` (float16 or bfloat16, any
        token and head strides; outputs of the inputs' type, the input itself
        included, but no memory of another argument).  ``q`` or ``k`` may be
        None.  ``positions [T]`` int32."""
        T, hq, hkv, dt, qv, kv, qo, pos, qw, kw = self._inputs(q, k, positions, q_weight, k_weight, q_out, None)
        ko = (0, 0, 0) if k is None else self._heads("k_out", k_out, (T, hkv, self.head_dim), dt)
        raw = _VIEWS(T, hq, hkv, self._types[dt], qv[0], kv[0], 0, qv[1], qv[2], kv[1], kv[2], 0, 0, pos, qw, kw, eps, 0,
                     qo[0], ko[0], qo[1], qo[2], ko[1], ko[2], 0, 0, 0, 0, 0)
        N.check(N.lib().weaver_rope_rotate(self._h, raw, raw_stream(stream, self.device)))

    def append(self, q, k, v, positions, slots, hot_k, hot_v, q_out, bad_flag, *, q_weight=None, k_weight=None,
               eps: float = 1e-6, hot_pool_blocks: int | None = None, stream=None) -> None:
        """Rotates ``q [T, Hq, d]`` into ``q_out`` (float16) and ``k [T, Hkv,
        d]`` into row ``slots[t]`` (int64: block * 16 + row; negative: padding,
        skipped) of ``hot_k [blocks, 16, Hkv, d]``, and copies ``v`` into
        ``hot_v``.  ``q`` (with ``q_out``) and ``v`` (with ``hot_v``) may be
        None.  ``hot_k`` / ``hot_v`` may be raw device pointers (a
        ``DeviceFabric`` layer's) with ``hot_pool_blocks``.  ``bad_flag`` (one
        int32) gets 1 OR-ed in for a slot beyond the pool, whose token is
        skipped.  The slots of one call must be distinct.  ``q_out`` (``q``
        itself excepted), the pools and ``bad_flag`` share no memory with another
        argument."""
        if k is None:
            raise ValueError("append needs k")
        T, hq, hkv, dt, qv, kv, qo, pos, qw, kw = self._inputs(q, k, positions, q_weight, k_weight, q_out, self._f16)
        if (v is None) != (hot_v is None):
            raise ValueError("v and hot_v come together")
        vv = (0, 0, 0) if v is None else self._heads("v", v, (T, hkv, self.head_dim), dt)
        blocks, pools = hot_pool_blocks, [0, 0]
        for i, pool in enumerate((hot_k, hot_v)):
            if pool is None or isinstance(pool, int):
                pools[i] = pool or 0
                continue
            name, n = ("hot_k", "hot_v")[i], pool.shape[0]
            if pool.shape != (n, BLOCK_SIZE, hkv, self.head_dim) or pool.dtype != self._f16 or \
                    pool.get_device() != self.device:
                self._refuse(name, pool, (n, BLOCK_SIZE, hkv, self.head_dim), self._f16)
            if not pool.is_contiguous():
                raise ValueError(f"{name} must be contiguous")
            if blocks is None:
                blocks = n
            if n < blocks:
                raise ValueError(f"{name} has fewer than {blocks} blocks")
            pools[i] = pool.data_ptr()
        if blocks is None:
            raise ValueError("raw pool pointers need hot_pool_blocks")
        if bad_flag is None or bad_flag.dtype != self._i32 or bad_flag.numel() < 1 or bad_flag.get_device() != self.device:
            raise ValueError(f"bad_flag must be an int32 CUDA tensor on device {self.device}")
        raw = _VIEWS(T, hq, hkv, self._types[dt], qv[0], kv[0], vv[0], qv[1], qv[2], kv[1], kv[2], vv[1], vv[2], pos, qw, kw,
                     eps, 0, qo[0], 0, qo[1], qo[2], 0, 0, self._flat("slots", slots, T, self._i64), pools[0], pools[1],
                     blocks, bad_flag.data_ptr())
        N.check(N.lib().weaver_rope_append(self._h, raw, raw_stream(stream, self.device)))


__all__ = ["Rope", "rope_frequencies", "token_slots"]
