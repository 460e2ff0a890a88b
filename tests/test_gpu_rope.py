"""Position rotation, head norms and the append into the hot pool on the GPU
against the formulas in 64 bits.  Needs a B200.

Tolerance of an element y = a c - b s (and the like) stored in type t: the
store rounds by at most eps(t)/2 |y| (half a step, at least half the smallest
subnormal); before it the fp32 work is off by at most 2^-19 (|a| + |b|): the
angle by 2^-25 turns = 2^-22.3, sincospif, the norm's factor (rsqrt, a sum of
d squares in a tree of 2^-24 relative steps), its two products, and the two
products and one sum of the rotation by a few 2^-24 each."""
import math

import pytest

pytestmark = pytest.mark.gpu

import numpy as np  # noqa: E402

import aether_nexus_b200 as W  # noqa: E402


@pytest.fixture(scope="module")
def engine():
    import torch
    if not torch.cuda.is_available():
        pytest.fail("no CUDA device: GPU tests need a B200")
    e = W.WeaverEngine(0)
    yield e
    e.close()


def reference(x, pos, inv_freq, amp, rot, layout, weight=None, eps=1e-6):
    """(y, |a| + |b| of every element's pair) in 64 bits."""
    import torch
    x = x.double()
    if weight is not None:
        x = x / (x.square().mean(-1, keepdim=True) + eps).sqrt() * weight.double()
    y, mag = x.clone(), x.abs()
    ang = pos.double()[:, None] * torch.as_tensor(inv_freq, dtype=torch.float64, device=x.device)
    c, s = ang.cos()[:, None] * amp, ang.sin()[:, None] * amp
    if layout == "half":
        ia, ib = slice(0, rot // 2), slice(rot // 2, rot)
    else:
        ia, ib = slice(0, rot, 2), slice(1, rot, 2)
    a, b = x[..., ia], x[..., ib]
    y[..., ia], y[..., ib] = a * c - b * s, b * c + a * s
    mag[..., ia] = mag[..., ib] = (a.abs() + b.abs()) * max(abs(amp), 1.0)
    return y, mag


def check(got, y, mag, what=""):
    import torch
    info = torch.finfo(got.dtype)
    tol = y.abs() * (info.eps / 2) + mag * 2.0 ** -19 + info.smallest_normal * info.eps / 2
    err = (got.double() - y).abs()
    assert (err <= tol).all(), f"{what}: {int((err > tol).sum())} of {err.numel()} off, worst {float((err / tol).max()):.2f}"


def heads(T, H, d, dtype, seed, fused=0):
    """[T, H, d] rows, a slice of a wider buffer where fused > 0."""
    import torch
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(T, H + fused, d, generator=g, device="cuda").mul_(2).to(dtype)[:, fused // 2:fused // 2 + H]


@pytest.mark.parametrize("T,Hq,Hkv,d,rot,layout,dtype,norm,far", [
    (1, 32, 8, 128, 128, "half", "float16", False, 0),
    (1, 14, 2, 64, 64, "interleaved", "bfloat16", True, 1000000),
    (5, 1, 1, 128, 16, "interleaved", "float16", True, 7),
    (3, 64, 8, 128, 96, "half", "bfloat16", False, -40),
    (17, 14, 2, 64, 16, "half", "float16", True, 131071),
    (33, 3, 3, 64, 48, "interleaved", "float16", False, 2147483600),
    (700, 12, 2, 128, 128, "interleaved", "bfloat16", True, 4000000),
    (257, 32, 8, 64, 64, "half", "float16", True, 0),
    (2, 5, 1, 128, 0, "half", "float16", True, 3),  # norm only
])
def test_rotate(engine, T, Hq, Hkv, d, rot, layout, dtype, norm, far):
    import torch
    dt = getattr(torch, dtype)
    q, k = heads(T, Hq, d, dt, 1, fused=4), heads(T, Hkv, d, dt, 2, fused=6)
    pos = far + torch.arange(T, device="cuda", dtype=torch.int32) % 37
    qw, kw = ((1 + 0.3 * heads(1, 1, d, torch.float32, s)[0, 0]).to(dt) if norm else None for s in (3, 4))
    rope = W.Rope(engine, head_dim=d, rot_dim=rot, theta=50000.0, layout=layout, amplitude=1.25)
    qo = torch.full(q.shape, math.nan, dtype=dt, device="cuda")
    ko = torch.full(k.shape, math.nan, dtype=dt, device="cuda")
    rope.rotate(q, k, pos, qo, ko, q_weight=qw, k_weight=kw, eps=1e-5)
    for got, x, w in ((qo, q, qw), (ko, k, kw)):
        check(got, *reference(x, pos, rope.inv_freq, 1.25, rot, layout, w, 1e-5))
    # one of the two alone, in place, in a buffer laid out [heads, tokens, d]: the same values
    qt = q.transpose(0, 1).contiguous().transpose(0, 1)
    rope.rotate(qt, None, pos, qt, q_weight=qw, eps=1e-5)
    assert torch.equal(qt, qo)
    rope.rotate(None, k, pos, None, k, k_weight=kw, eps=1e-5)
    assert torch.equal(k, ko)


def test_only_one_of_two_weights(engine):
    import torch
    q, k = heads(9, 4, 64, torch.float16, 5), heads(9, 2, 64, torch.float16, 6)
    w = (1 + 0.1 * heads(1, 1, 64, torch.float32, 7)[0, 0]).half()
    pos = torch.arange(9, device="cuda", dtype=torch.int32)
    rope = W.Rope(engine, head_dim=64)
    qo, ko = torch.empty_like(q), torch.empty_like(k)
    rope.rotate(q, k, pos, qo, ko, k_weight=w)
    check(qo, *reference(q, pos, rope.inv_freq, 1.0, 64, "half"))
    check(ko, *reference(k, pos, rope.inv_freq, 1.0, 64, "half", w))


def test_zero_and_special_rows(engine):
    """A zero head stays zero under the norm; an infinite element spoils its own head only."""
    import torch
    q = heads(2, 3, 128, torch.float16, 8)
    q[0, 1] = 0
    q[1, 2, 5] = math.inf
    w = torch.ones(128, dtype=torch.float16, device="cuda")
    pos = torch.tensor([3, 4], device="cuda", dtype=torch.int32)
    rope = W.Rope(engine, head_dim=128)
    out = torch.empty_like(q)
    rope.rotate(q, None, pos, out, q_weight=w)
    assert (out[0, 1] == 0).all() and not torch.isfinite(out[1, 2]).all()
    ok = torch.ones(2, 3, dtype=torch.bool, device="cuda")
    ok[1, 2] = False
    y, mag = reference(q, pos, rope.inv_freq, 1.0, 128, "half", w)
    check(out[ok], y[ok], mag[ok])


@pytest.mark.parametrize("scaling", [None, dict(type="yarn", factor=16.0, original_length=65536),
                                     dict(type="bands", factor=8.0, original_length=8192, low=1.0, high=4.0)])
def test_far_positions_keep_relative_angles(engine, scaling):
    """q.k depends on the distance only: rotated at p and p + 9 for p near 2^30 as near 0."""
    import torch
    rope = W.Rope(engine, head_dim=128, theta=500000.0, scaling=scaling)
    x = heads(1, 2, 128, torch.float16, 9)
    dots = []
    for base in (0, 1 << 20, (1 << 30) + 12345):
        rows = []
        for p in (base, base + 9):
            out = torch.empty_like(x)
            rope.rotate(x, None, torch.tensor([p], device="cuda", dtype=torch.int32), out)
            rows.append(out.double())
        dots.append(float((rows[0] * rows[1]).sum()))
    # each rotated element is off by 2^-11 of its size (f16), two factors per product
    bound = 2 * 2.0 ** -11 * 2 * float(x.double().square().sum()) * rope.amplitude ** 2
    assert max(dots) - min(dots) <= bound


@pytest.mark.parametrize("T,pad,Hq,Hkv,d,dtype,layout,norm", [
    (1, 0, 32, 8, 128, "float16", "half", False),
    (64, 5, 12, 2, 128, "bfloat16", "half", True),
    (333, 100, 14, 2, 64, "float16", "interleaved", True),
    (40, 40, 8, 8, 64, "bfloat16", "half", False),  # padding only
    (2000, 1, 64, 8, 128, "float16", "half", False),
])
def test_append(engine, T, pad, Hq, Hkv, d, dtype, layout, norm):
    import torch
    dt, live = getattr(torch, dtype), T - pad
    q, k, v = heads(T, Hq, d, dt, 1, 8), heads(T, Hkv, d, dt, 2, 2), heads(T, Hkv, d, dt, 3)
    w = (1 + 0.3 * heads(1, 1, d, torch.float32, 4)[0, 0]).to(dt) if norm else None
    pos = torch.arange(T, device="cuda", dtype=torch.int32) + 1000
    blocks = live // 16 + 4
    gen = torch.Generator().manual_seed(5)
    slots = torch.full((T,), -1, dtype=torch.int64)
    slots[:live] = torch.randperm(blocks * 16, generator=gen)[:live]
    pool = [heads(blocks * 16, Hkv, d, torch.float16, 10 + i).reshape(blocks, 16, Hkv, d) for i in range(2)]
    before = [p.clone() for p in pool]
    qo = torch.full((T, Hq, d), 7.0, dtype=torch.float16, device="cuda")
    bad = torch.zeros(1, dtype=torch.int32, device="cuda")
    rope = W.Rope(engine, head_dim=d, theta=10000.0, layout=layout, rot_dim=d // 2)
    rope.append(q, k, v, pos, slots.cuda(), pool[0], pool[1], qo, bad, q_weight=w, k_weight=w)
    assert int(bad) == 0
    args = (pos, rope.inv_freq, 1.0, d // 2, layout, w)
    check(qo[:live], *(x[:live] for x in reference(q, *args)), what="q")
    assert (qo[live:] == 7.0).all()  # padding rows are left alone
    rows = [p.view(-1, Hkv, d) for p in pool]
    at = slots[:live].cuda()
    check(rows[0][at], *(x[:live] for x in reference(k, *args)), what="k")
    assert torch.equal(rows[1][at], v[:live].half())
    untouched = torch.ones(blocks * 16, dtype=torch.bool, device="cuda")
    untouched[at] = False
    for r, b in zip(rows, before):
        assert torch.equal(r[untouched], b.view(-1, Hkv, d)[untouched])


def test_append_skips_and_reports_slots_beyond_the_pool(engine):
    import torch
    q, k = heads(4, 4, 64, torch.float16, 1), heads(4, 2, 64, torch.float16, 2)
    pos = torch.arange(4, device="cuda", dtype=torch.int32)
    guard = torch.zeros(4, 16, 2, 64, dtype=torch.float16, device="cuda")  # the pool is its first 2 blocks
    bad = torch.zeros(1, dtype=torch.int32, device="cuda")
    qo = torch.zeros_like(q)
    rope = W.Rope(engine, head_dim=64)
    slots = torch.tensor([31, 32, 1 << 40, -(1 << 50)], device="cuda")
    rope.append(q, k, None, pos, slots, guard[:2], None, qo, bad)
    assert int(bad) == 1
    assert (guard.view(64, 2, 64)[31] != 0).any() and (guard.view(64, 2, 64)[:31] == 0).all() and (guard[2:] == 0).all()
    assert (qo[0] != 0).any() and (qo[1:] == 0).all()


def test_append_keys_only_without_queries(engine):
    import torch
    k, v = heads(20, 2, 128, torch.bfloat16, 1), heads(20, 2, 128, torch.bfloat16, 2)
    pos = torch.arange(20, device="cuda", dtype=torch.int32)
    pool = torch.zeros(2, 2, 16, 2, 128, dtype=torch.float16, device="cuda")
    bad = torch.zeros(1, dtype=torch.int32, device="cuda")
    rope = W.Rope(engine, head_dim=128)
    rope.append(None, k, v, pos, torch.arange(20, device="cuda"), pool[0], pool[1], None, bad)
    check(pool[0].view(-1, 2, 128)[:20], *reference(k, pos, rope.inv_freq, 1.0, 128, "half"))
    assert torch.equal(pool[1].view(-1, 2, 128)[:20], v.half()) and int(bad) == 0


def test_append_replayed_from_a_graph_on_its_own_stream(engine):
    """Captured once, replayed with other inputs in the same buffers."""
    import torch
    q, k, v = heads(6, 8, 128, torch.float16, 1), heads(6, 2, 128, torch.float16, 2), heads(6, 2, 128, torch.float16, 3)
    pos = torch.arange(6, device="cuda", dtype=torch.int32)
    slots = torch.arange(6, device="cuda")
    pool = torch.zeros(2, 3, 16, 2, 128, dtype=torch.float16, device="cuda")
    bad = torch.zeros(1, dtype=torch.int32, device="cuda")
    qo = torch.zeros_like(q)
    rope = W.Rope(engine, head_dim=128)
    torch.cuda.synchronize()
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.graph(graph, stream=side):
        rope.append(q, k, v, pos, slots, pool[0], pool[1], qo, bad)
    rope.close()  # the launch holds the frequencies itself
    pos += 100
    slots += 16
    k.copy_(heads(6, 2, 128, torch.float16, 12))
    graph.replay()
    torch.cuda.synchronize()
    check(pool[0].view(-1, 2, 128)[16:22], *reference(k, pos, rope.inv_freq, 1.0, 128, "half"))
    assert (pool[0].view(-1, 2, 128)[:16] == 0).all() and torch.equal(pool[1].view(-1, 2, 128)[16:22], v)


@pytest.mark.parametrize("change", ["dtype", "shape", "stride", "positions", "device", "slots", "pool"])
def test_python_refusals(engine, change):
    import torch
    a = dict(q=heads(4, 8, 64, torch.float16, 1), k=heads(4, 2, 64, torch.float16, 2),
             v=heads(4, 2, 64, torch.float16, 3), positions=torch.zeros(4, dtype=torch.int32, device="cuda"),
             slots=torch.arange(4, device="cuda"), pool=torch.zeros(2, 1, 16, 2, 64, dtype=torch.float16, device="cuda"))
    if change == "dtype":
        a["k"] = a["k"].bfloat16()
    elif change == "shape":
        a["k"] = a["k"][:3]
    elif change == "stride":
        a["q"] = heads(4, 8, 128, torch.float16, 1)[..., ::2]
    elif change == "positions":
        a["positions"] = a["positions"].long()
    elif change == "device":
        a["positions"] = a["positions"].cpu()
    elif change == "slots":
        a["slots"] = a["slots"].int()
    elif change == "pool":
        a["pool"] = a["pool"].transpose(2, 3).contiguous().transpose(2, 3)
    rope = W.Rope(engine, head_dim=64)
    bad = torch.zeros(1, dtype=torch.int32, device="cuda")
    qo = torch.zeros(4, 8, 64, dtype=torch.float16, device="cuda")
    with pytest.raises(ValueError):
        rope.append(a["q"], a["k"], a["v"], a["positions"], a["slots"], a["pool"][0], a["pool"][1], qo, bad)


def test_one_token_of_any_stride(engine):
    """With one token its stride does not matter (a slice whose stride is odd)."""
    import torch
    wide = torch.zeros(2, 8 * 64 + 3, dtype=torch.float16, device="cuda")
    q = wide[:1, :512].view(1, 8, 64)
    q.copy_(heads(1, 8, 64, torch.float16, 1))
    out = torch.empty(1, 8, 64, dtype=torch.float16, device="cuda")
    pos = torch.tensor([5], dtype=torch.int32, device="cuda")
    rope = W.Rope(engine, head_dim=64)
    rope.rotate(q, None, pos, out)
    check(out, *reference(q, pos, rope.inv_freq, 1.0, 64, "half"))


def test_broadcast_heads_as_input(engine):
    """One key head given to four by a stride of zero."""
    import torch
    k = heads(6, 1, 128, torch.bfloat16, 2).expand(6, 4, 128)
    out = torch.empty(6, 4, 128, dtype=torch.bfloat16, device="cuda")
    pos = torch.arange(6, device="cuda", dtype=torch.int32)
    rope = W.Rope(engine, head_dim=128)
    rope.rotate(None, k, pos, None, out)
    check(out, *reference(k, pos, rope.inv_freq, 1.0, 128, "half"))


def test_no_tokens(engine):
    import torch
    e = torch.empty(0, 4, 64, dtype=torch.float16, device="cuda")
    pool = torch.zeros(1, 16, 4, 64, dtype=torch.float16, device="cuda")
    rope = W.Rope(engine, head_dim=64)
    none = torch.empty(0, dtype=torch.int32, device="cuda")
    rope.rotate(e, e, none, e, e)
    rope.append(e, e, None, none, none.long(), pool, None, e, torch.zeros(1, dtype=torch.int32, device="cuda"))


@pytest.mark.parametrize("layout", ["tokens", "heads", "pairs"])
def test_slices_of_one_buffer_lie_next_to_each_other(engine, layout):
    """Inputs and outputs that share a buffer and no element of it: the same results as from buffers of their own."""
    import torch
    T, H, d = 37, 4, 64
    pos = torch.arange(T, device="cuda", dtype=torch.int32) + 11
    rope = W.Rope(engine, head_dim=d)
    data = [heads(T, H, d, torch.float16, 50 + i) for i in range(4)]
    if layout == "tokens":    # [T][q k q_out k_out][H][d]
        buf = torch.zeros(T, 4, H, d, dtype=torch.float16, device="cuda")
        part = [buf[:, i] for i in range(4)]
    elif layout == "heads":   # [q k q_out k_out][H][T][d], one after the other
        buf = torch.zeros(4, H, T, d, dtype=torch.float16, device="cuda")
        part = [buf[i].transpose(0, 1) for i in range(4)]
    else:                     # [T][H][q k q_out k_out][d]
        buf = torch.zeros(T, H, 4, d, dtype=torch.float16, device="cuda")
        part = [buf[:, :, i] for i in range(4)]
    for p, x in zip(part, data):
        p.copy_(x)
    rope.rotate(part[0], part[1], pos, part[2], part[3])
    for i in range(2):
        assert torch.equal(part[i], data[i])
        check(part[2 + i], *reference(data[i], pos, rope.inv_freq, 1.0, d, "half"))
    before = buf.clone()
    for args in ((part[0], part[1], part[1], part[3]), (part[0], part[1], part[2], part[2]),
                 (part[0], part[1], part[2], part[0])):
        with pytest.raises(W.WeaverError) as e:
            rope.rotate(args[0], args[1], pos, args[2], args[3])
        assert e.value.status == 1
    assert torch.equal(buf, before)
