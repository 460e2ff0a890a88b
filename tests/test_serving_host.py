"""Host side of the rotation, the append and the shared-prefix attention,
without a GPU: frequencies, slots, and every refusal that the C entries make
before they touch the device."""
import ctypes
import math

import numpy as np
import pytest

import aether_nexus_b200 as W
from aether_nexus_b200 import _native as N
from aether_nexus_b200.prefix import _indptr

INVALID, UNSUPPORTED, MISALIGNED, CAPACITY = 1, 2, 3, 8


def test_frequencies_plain_and_linear():
    f, amp = W.rope_frequencies(128, 500000.0)
    assert f.dtype == np.float64 and f.shape == (64,) and amp == 1.0
    assert f[0] == 1.0 and math.isclose(f[63], 500000.0 ** (-126 / 128), rel_tol=1e-14)
    g, amp = W.rope_frequencies(128, 500000.0, {"type": "linear", "factor": 4.0})
    assert np.array_equal(g, f / 4.0) and amp == 1.0


def test_frequencies_ntk_scales_the_slowest_pair_by_the_factor():
    f, _ = W.rope_frequencies(64, 10000.0)
    g, _ = W.rope_frequencies(64, 10000.0, {"type": "ntk", "factor": 8.0})
    assert g[0] == 1.0 and math.isclose(g[-1], f[-1] / 8.0, rel_tol=1e-12)
    assert (np.diff(g) < 0).all()


def test_frequencies_yarn_and_bands_keep_fast_pairs_and_scale_slow_ones():
    f, _ = W.rope_frequencies(128, 10000.0)
    g, amp = W.rope_frequencies(128, 10000.0, {"type": "yarn", "factor": 16.0, "original_length": 4096})
    turns = 4096 * f / (2 * math.pi)
    assert np.allclose(g[turns > 34], f[turns > 34], rtol=1e-14) and np.allclose(g[turns < 0.9], f[turns < 0.9] / 16)
    assert math.isclose(amp, 0.1 * math.log(16.0) + 1.0)
    assert W.rope_frequencies(128, 10000.0, {"type": "yarn", "factor": 16.0, "original_length": 4096,
                                             "attention_factor": 1.5})[1] == 1.5
    h, amp = W.rope_frequencies(128, 10000.0, {"type": "bands", "factor": 8.0, "original_length": 8192, "low": 1,
                                               "high": 4})
    turns = 8192 * f / (2 * math.pi)
    assert np.array_equal(h[turns >= 4], f[turns >= 4]) and np.allclose(h[turns <= 1], f[turns <= 1] / 8.0, rtol=1e-15)
    mid = (turns > 1) & (turns < 4)
    assert ((h[mid] < f[mid]) & (h[mid] > f[mid] / 8.0)).all() and amp == 1.0


@pytest.mark.parametrize("rot_dim,theta,length,factor", [
    (128, 10000.0, 131072, 16.0), (128, 10000.0, 65536, 16.0), (16, 10000.0, 32768, 16.0), (64, 10000.0, 1 << 20, 4.0),
    (128, 500000.0, 65536, 16.0)])
def test_frequencies_yarn_ramp_may_end_behind_the_last_pair(rot_dim, theta, length, factor):
    """The ramp between the pairs that turn 32 times and once over the original
    length, written out pair by pair (Peng et al. 2023: its upper index is
    bounded by rot_dim - 1, not by the last pair): a pair that still turns more
    than once is mixed, never scaled whole."""
    got, _ = W.rope_frequencies(rot_dim, theta, {"type": "yarn", "factor": factor, "original_length": length})

    def index(turns):
        return rot_dim / 2 * math.log(length / (2 * math.pi * turns)) / math.log(theta)
    low, high = max(math.floor(index(32)), 0), min(math.ceil(index(1)), rot_dim - 1)
    for i in range(rot_dim // 2):
        f = theta ** (-2 * i / rot_dim)
        inside = min(max((i - low) / (high - low), 0.0), 1.0)  # 0: keeps f, 1: f / factor
        assert math.isclose(got[i], (1 - inside) * f + inside * f / factor, rel_tol=1e-12), i
        if length * f / (2 * math.pi) > 1.0:
            assert got[i] > f / factor * (1 + 1e-9), i


@pytest.mark.parametrize("kw", [dict(rot_dim=7), dict(theta=-1.0), dict(theta=float("nan")),
                                dict(scaling={"type": "other", "factor": 2.0}),
                                dict(scaling={"type": "linear", "factor": 0.0}),
                                dict(scaling={"type": "linear", "factor": 2.0, "low": 1}),
                                dict(scaling={"type": "bands", "factor": 2.0, "original_length": 10, "low": 4, "high": 4})])
def test_frequencies_refuse(kw):
    with pytest.raises(ValueError):
        W.rope_frequencies(**{"rot_dim": 64, **kw})


def test_token_slots():
    refs = np.array([5, 0x80000002, 9, 1], np.uint32)
    got = W.token_slots(refs, [0, 2, 2, 4], [15, 0, 17], [0, 3, 3, 5])
    assert got.tolist() == [5 * 16 + 15, 2 * 16, 2 * 16 + 1, 1 * 16 + 1, 1 * 16 + 2]
    with pytest.raises(ValueError):
        W.token_slots(refs, [0, 2], [31], [0, 2])


@pytest.fixture
def engine_memory():
    """Zeroed memory in an engine's place: device 0, read only after the checks."""
    return ctypes.create_string_buffer(1 << 16)


def _rope(engine, **kw):
    f = np.linspace(1.0, 0.1, 64)
    c = N.RopeConfigC(**{**dict(head_dim=128, rot_dim=128, layout=0, amplitude=1.0, inv_freq=f.ctypes.data), **kw})
    h = ctypes.c_void_p()
    return N.lib().weaver_rope_create(engine, ctypes.byref(c), ctypes.byref(h)), h


@pytest.mark.parametrize("kw,status", [
    (dict(head_dim=96), UNSUPPORTED), (dict(rot_dim=24), UNSUPPORTED), (dict(rot_dim=144), UNSUPPORTED),
    (dict(head_dim=64), UNSUPPORTED), (dict(layout=2), INVALID), (dict(inv_freq=None), INVALID),
    (dict(amplitude=float("inf")), INVALID)])
def test_rope_create_refuses(engine_memory, kw, status):
    rc, h = _rope(engine_memory, **kw)
    assert rc == status and not h.value


def test_rope_create_refuses_nan_frequency(engine_memory):
    f = np.full(64, np.nan)
    assert _rope(engine_memory, inv_freq=f.ctypes.data)[0] == INVALID
    assert N.lib().weaver_rope_create(None, None, None) == INVALID


def _rope_views(**kw):
    d = dict(n_tokens=4, q_heads=8, kv_heads=2, dtype=0, q=1 << 20, k=2 << 20, v=3 << 20, q_token_stride=1024,
             q_head_stride=128, k_token_stride=256, k_head_stride=128, v_token_stride=256, v_head_stride=128,
             positions=4 << 20, eps=1e-6, q_out=5 << 20, k_out=6 << 20, q_out_token_stride=1024,
             q_out_head_stride=128, k_out_token_stride=256, k_out_head_stride=128, slots=7 << 20, hot_k=8 << 20,
             hot_v=9 << 20, hot_pool_blocks=4, bad_flag=10 << 20)
    d.update(kw)
    return N.RopeViewsC(**d)


BOTH = [
    (dict(dtype=2), UNSUPPORTED), (dict(q_heads=0, kv_heads=0), INVALID), (dict(q_heads=70000), CAPACITY),
    (dict(positions=None), INVALID), (dict(positions=(4 << 20) + 2), INVALID),
    (dict(q_weight=11 << 20, eps=-1.0), INVALID), (dict(k_weight=11 << 20, eps=float("nan")), INVALID),
    (dict(q_weight=(11 << 20) + 8), MISALIGNED), (dict(q=None), INVALID), (dict(q_out=None), INVALID),
    (dict(q=(1 << 20) + 2), MISALIGNED), (dict(q_token_stride=1020), MISALIGNED),
    (dict(q_out_token_stride=512), INVALID), (dict(q_out_head_stride=0), INVALID),
    (dict(q_out=(1 << 20) + 128), INVALID),                              # half a head further on: overlaps q
    (dict(q_out=1 << 20, q_out_token_stride=2048), INVALID),             # q itself, with other strides
]


@pytest.mark.parametrize("kw,status", BOTH + [
    (dict(k=None), INVALID), (dict(k_out=None), INVALID), (dict(k_out_head_stride=64), INVALID),
    (dict(k_out=(6 << 20) + 4), MISALIGNED)])
def test_rotate_refuses(engine_memory, kw, status):
    rc, h = _rope(engine_memory)
    assert rc == 0
    assert N.lib().weaver_rope_rotate(h, ctypes.byref(_rope_views(**kw)), None) == status, N.lib().weaver_last_error()
    N.lib().weaver_rope_destroy(h)


@pytest.mark.parametrize("kw,status", BOTH + [
    (dict(k=None), INVALID), (dict(kv_heads=0), INVALID), (dict(slots=None), INVALID), (dict(bad_flag=None), INVALID),
    (dict(hot_k=None), INVALID), (dict(hot_v=None), INVALID), (dict(v=None), INVALID), (dict(hot_v=8 << 20), INVALID),
    (dict(hot_pool_blocks=0), INVALID), (dict(hot_k=(8 << 20) + 8), MISALIGNED), (dict(v_token_stride=252), MISALIGNED),
    (dict(slots=(7 << 20) + 4), MISALIGNED), (dict(hot_v=(8 << 20) + 4096), INVALID)])
def test_append_refuses(engine_memory, kw, status):
    rc, h = _rope(engine_memory)
    assert rc == 0
    assert N.lib().weaver_rope_append(h, ctypes.byref(_rope_views(**kw)), None) == status, N.lib().weaver_last_error()
    N.lib().weaver_rope_destroy(h)


# q covers 8192 bytes from 1 << 20, k and v 2048 each from 2 << 20 and 3 << 20 (two heads of 256 bytes a token)
OVERLAPS = [
    dict(q_out=2 << 20, q_heads=2, q_token_stride=256, q_out_token_stride=256),   # k itself
    dict(q_out=(2 << 20) - 8192 + 256),                                           # its last head: k's first
    dict(q_out=(4 << 20) - 4096), dict(q_out=(11 << 20) - 4096, q_weight=11 << 20), dict(q_out=11 << 20, k_weight=11 << 20),
]


@pytest.mark.parametrize("kw", OVERLAPS + [
    dict(k_out=1 << 20), dict(k_out=(1 << 20) + 8192 - 256), dict(k_out=4 << 20), dict(k_out=5 << 20),
    dict(k_out=(5 << 20) + 1024, k_out_token_stride=1024),                        # two of the heads of q_out
    dict(k=5 << 20, k_out=5 << 20), dict(k=1 << 20, q_out=1 << 20)])              # in place over what another one reads
def test_rotate_refuses_outputs_over_other_arguments(engine_memory, kw):
    rc, h = _rope(engine_memory)
    assert rc == 0
    assert N.lib().weaver_rope_rotate(h, ctypes.byref(_rope_views(**kw)), None) == INVALID, N.lib().weaver_last_error()
    assert b"overlap" in N.lib().weaver_last_error()
    N.lib().weaver_rope_destroy(h)


# the pools cover 32768 bytes from 8 << 20 and 9 << 20
@pytest.mark.parametrize("kw", OVERLAPS + [
    dict(q_out=3 << 20), dict(q_out=8 << 20), dict(q_out=(9 << 20) + 32768 - 256), dict(q_out=(8 << 20) - 4096),
    dict(q_out=7 << 20), dict(q_out=(10 << 20) - 4096),
    dict(q=8 << 20), dict(k=8 << 20), dict(k=(8 << 20) + 32768 - 256), dict(v=9 << 20), dict(v=8 << 20), dict(k=9 << 20),
    dict(slots=(8 << 20) + 32768 - 8), dict(positions=9 << 20), dict(bad_flag=9 << 20), dict(k_weight=8 << 20),
    dict(bad_flag=(7 << 20) + 8), dict(bad_flag=4 << 20), dict(bad_flag=(1 << 20) + 4)])
def test_append_refuses_outputs_over_other_arguments(engine_memory, kw):
    rc, h = _rope(engine_memory)
    assert rc == 0
    assert N.lib().weaver_rope_append(h, ctypes.byref(_rope_views(**kw)), None) == INVALID, N.lib().weaver_last_error()
    assert b"overlap" in N.lib().weaver_last_error()
    N.lib().weaver_rope_destroy(h)


def test_no_tokens_is_no_launch(engine_memory):
    rc, h = _rope(engine_memory)
    empty = N.RopeViewsC()
    assert N.lib().weaver_rope_rotate(h, ctypes.byref(empty), None) == 0
    assert N.lib().weaver_rope_append(h, ctypes.byref(empty), None) == 0
    assert N.lib().weaver_rope_rotate(None, ctypes.byref(empty), None) == INVALID
    N.lib().weaver_rope_destroy(h)
    N.lib().weaver_rope_destroy(None)


def _prefix_create(engine, q=(0, 1, 3), g=(0, 2), p=(0, 4), s=(0, 1, 2), **kw):
    shape = N.PrefixShapeC(**{**dict(num_groups=len(g) - 1, num_seqs=len(q) - 1, q_heads=8, kv_heads=2, head_dim=128,
                                     scale=0.1, flags=1), **kw})
    arr = [np.array(x, np.uint32) for x in (q, g, p, s)]
    h = ctypes.c_void_p()
    return N.lib().weaver_prefix_plan_create(engine, ctypes.byref(shape), *[a.ctypes.data for a in arr], ctypes.byref(h))


@pytest.mark.parametrize("kw,status", [
    (dict(head_dim=96), UNSUPPORTED), (dict(kv_heads=3), INVALID), (dict(q_heads=0), INVALID),
    (dict(flags=2), UNSUPPORTED), (dict(scale=float("nan")), INVALID), (dict(q=(0, 3, 1)), INVALID),
    (dict(q=(1, 2, 3)), INVALID), (dict(g=(0, 1)), INVALID), (dict(g=(0, 2, 1), p=(0, 1, 2)), INVALID),
    (dict(p=(4, 0)), INVALID), (dict(s=(0, 2, 1)), INVALID), (dict(q=(0, 1, 1 << 30)), CAPACITY),
    (dict(p=(0, 1 << 27)), CAPACITY), (dict(num_groups=0), INVALID)])
def test_prefix_plan_refuses(engine_memory, kw, status):
    assert _prefix_create(engine_memory, **kw) == status, N.lib().weaver_last_error()


def test_prefix_null_arguments():
    assert N.lib().weaver_prefix_plan_create(None, None, None, None, None, None, None) == INVALID
    assert N.lib().weaver_prefix_run(None, None, None) == INVALID
    assert N.lib().weaver_prefix_plan_status(None) == INVALID
    assert N.lib().weaver_prefix_plan_kernel_count(None) == 0
    N.lib().weaver_prefix_plan_destroy(None)


@pytest.mark.parametrize("bad", [[0], [0.0, 1.0], [[0, 1]], [0, -1], [0, 1 << 32]])
def test_indptr_refuses(bad):
    with pytest.raises(ValueError):
        _indptr("q_indptr", bad)


@pytest.mark.parametrize("scaling", [
    {"type": "linear"}, {"type": "yarn", "factor": 4.0}, {"type": "bands", "factor": 4.0}, {"factor": 2.0},
    {"type": "yarn", "factor": 4.0, "original_length": 0}, {"type": "bands", "factor": 4.0, "original_length": math.nan},
    {"type": "yarn", "factor": 4.0, "original_length": 4096, "beta_slow": 0},
    {"type": "yarn", "factor": 4.0, "original_length": 4096, "beta_fast": -1},
    {"type": "yarn", "factor": 4.0, "original_length": math.inf}])
def test_frequencies_refuse_incomplete_scalings(scaling):
    with pytest.raises(ValueError):
        W.rope_frequencies(64, 10000.0, scaling)


class _CpuEngine:
    """An engine whose device is torch's number for the CPU: calls get as far as their last check of arguments."""
    device = -1

    def __init__(self, memory):
        self.handle = ctypes.cast(memory, ctypes.c_void_p)


@pytest.mark.parametrize("missing", ["k_out", "q_out", "positions"])
def test_rotate_names_a_missing_argument(engine_memory, missing):
    import torch
    rope = W.Rope(_CpuEngine(engine_memory), head_dim=64)
    a = dict(q=torch.zeros(2, 4, 64, dtype=torch.float16), k=torch.zeros(2, 1, 64, dtype=torch.float16),
             positions=torch.zeros(2, dtype=torch.int32), q_out=torch.zeros(2, 4, 64, dtype=torch.float16),
             k_out=torch.zeros(2, 1, 64, dtype=torch.float16))
    a[missing] = None
    with pytest.raises(ValueError, match=missing):
        rope.rotate(**a)


@pytest.mark.parametrize("missing", ["k", "q_out", "positions", "slots", "bad_flag"])
def test_append_names_a_missing_argument(engine_memory, missing):
    import torch
    rope = W.Rope(_CpuEngine(engine_memory), head_dim=64)
    a = dict(q=torch.zeros(2, 4, 64, dtype=torch.float16), k=torch.zeros(2, 1, 64, dtype=torch.float16), v=None,
             positions=torch.zeros(2, dtype=torch.int32), slots=torch.zeros(2, dtype=torch.int64),
             hot_k=torch.zeros(1, 16, 1, 64, dtype=torch.float16), hot_v=None,
             q_out=torch.zeros(2, 4, 64, dtype=torch.float16), bad_flag=torch.zeros(1, dtype=torch.int32))
    a[missing] = None
    with pytest.raises(ValueError, match=missing):
        rope.append(**a)


@pytest.mark.parametrize("args", [
    ([5, 6], [0, 2], [-3], [0, 2]),          # would count pages from the list's end
    ([5, 6], [0, 2], [1], [1, 3]),           # token 0 belongs to no sequence
    ([5, 6, 7], [0, 2], [1], [0, 2, 4]),     # more sequences of queries than lengths
    ([5, 6], [0, 2], [1, 2], [0, 1, 2]),     # more lengths than page lists
    ([5, 6], [0, 1, 2], [1, 2], [0, 2, 1]), ([5, 6], [0, 2, 1], [1, 2], [0, 1, 2]), ([5, 6], [-2, 2], [1], [0, 1])])
def test_token_slots_refuse_what_leaves_a_slot_unset(args):
    with pytest.raises(ValueError):
        W.token_slots(*args)


def test_token_slots_without_tokens():
    assert W.token_slots([], [0, 0], [0], [0, 0]).shape == (0,)
