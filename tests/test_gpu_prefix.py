"""Attention for a batch that shares prefixes on the GPU against the formula in
64 bits.  Needs a B200.

Tolerance of an output y = sum p v / sum p (p = e^(s - max)): y is rounded to
f16 by at most 2^-11 |y|; each probability is rounded to f16 before the product
with V (2^-11 relative, or 2^-25 absolute where it is subnormal, against a sum
of at least 1); a score of d products is off by at most ds = (d + 4) 2^-24
scale sum |q||k| in fp32, which changes p by ds, in the product and in the
sum; the exponentials and the sums of fp32 add less than 2^-17.  With W = sum
p |v| / sum p that is 2^-11 |y| + W (2^-11 + 2 ds + 2^-17) + n 2^-25 max|v| /
sum p + 2^-25 (half the smallest subnormal of the output)."""
import math
import random

import pytest

pytestmark = pytest.mark.gpu

import aether_nexus_b200 as W  # noqa: E402


@pytest.fixture(scope="module")
def engine():
    import torch
    if not torch.cuda.is_available():
        pytest.fail("no CUDA device: GPU tests need a B200")
    e = W.WeaverEngine(0)
    yield e
    e.close()


class Batch:
    """Groups [(prefix tokens, [(queries, own tokens), ...]), ...] over a
    shuffled pool whose every other row is `junk`."""

    def __init__(self, groups, Hq, Hkv, d, seed=0, junk=math.nan, spare_pages=0, qscale=2.0):
        import torch
        rng, g = random.Random(seed), torch.Generator(device="cuda").manual_seed(seed)
        self.groups, self.Hq, self.Hkv, self.d = groups, Hq, Hkv, d
        self.seqs = [s for _, ss in groups for s in ss]
        pages = lambda n: (n + 15) // 16 + spare_pages  # noqa: E731
        total = sum(pages(p) for p, _ in groups) + sum(pages(s) for _, s in self.seqs) + 3
        ids = list(range(total))
        rng.shuffle(ids)
        self.blocks = total
        self.hot_k = torch.full((total, 16, Hkv, d), junk, dtype=torch.float16, device="cuda")
        self.hot_v = torch.full_like(self.hot_k, junk)
        self.q_indptr, self.group_indptr, self.prefix_indptr, self.suffix_indptr = [0], [0], [0], [0]
        self.prefix_refs, self.suffix_refs = [], []
        self.rows = []  # every list's (pool rows)

        def take(n, refs, ptr):
            mine = [ids.pop() for _ in range(pages(n))]
            refs += [i | (1 << 31 if rng.random() < 0.5 else 0) for i in mine]
            ptr.append(len(refs))
            rows = torch.tensor([i * 16 + r for i in mine for r in range(16)][:n], dtype=torch.int64, device="cuda")
            for pool in (self.hot_k, self.hot_v):
                pool.view(-1, Hkv, d)[rows] = torch.randn(n, Hkv, d, generator=g, device="cuda").half()
            return rows
        self.prefix_rows = [take(p, self.prefix_refs, self.prefix_indptr) for p, _ in groups]
        self.suffix_rows = [take(s, self.suffix_refs, self.suffix_indptr) for _, s in self.seqs]
        for _, ss in groups:
            self.group_indptr.append(self.group_indptr[-1] + len(ss))
        for nq, _ in self.seqs:
            self.q_indptr.append(self.q_indptr[-1] + nq)
        self.T = self.q_indptr[-1]
        self.q = (qscale * torch.randn(self.T, Hq, d, generator=g, device="cuda")).half()
        self.prefix_lens = self.words([p for p, _ in groups])
        self.suffix_lens = self.words([s for _, s in self.seqs])
        self.out = torch.full(self.q.shape, math.nan, dtype=torch.float16, device="cuda")

    @staticmethod
    def words(x):
        import numpy as np
        import torch
        return torch.from_numpy(np.array(list(x) or [0], np.uint32).view(np.int32)).cuda()

    def plan(self, engine, **kw):
        return W.PrefixPlan(engine, **{**dict(q_heads=self.Hq, kv_heads=self.Hkv, head_dim=self.d, scale=self.d ** -0.5,
                                              q_indptr=self.q_indptr, group_indptr=self.group_indptr,
                                              prefix_indptr=self.prefix_indptr, suffix_indptr=self.suffix_indptr), **kw})

    def views(self, **kw):
        return {**dict(q=self.q, hot_k=self.hot_k, hot_v=self.hot_v, prefix_refs=self.words(self.prefix_refs),
                       suffix_refs=self.words(self.suffix_refs), prefix_lens=self.prefix_lens,
                       suffix_lens=self.suffix_lens, out=self.out), **kw}

    def reference(self, causal=True):
        """(y, tolerance) in 64 bits."""
        import torch
        y = torch.zeros(self.q.shape, dtype=torch.float64, device="cuda")
        tol = torch.full_like(y, 2.0 ** -25)
        G, b = self.Hq // self.Hkv, 0
        for gi, (_, ss) in enumerate(self.groups):
            for nq, n in ss:
                rows = torch.cat([self.prefix_rows[gi], self.suffix_rows[b]])
                P = len(self.prefix_rows[gi])
                k = self.hot_k.view(-1, self.Hkv, self.d)[rows].double().repeat_interleave(G, 1).transpose(0, 1)
                v = self.hot_v.view(-1, self.Hkv, self.d)[rows].double().repeat_interleave(G, 1).transpose(0, 1)
                t = slice(self.q_indptr[b], self.q_indptr[b + 1])
                b += 1
                if not nq or not len(rows):
                    continue
                q = self.q[t].double().transpose(0, 1)
                s = q @ k.transpose(1, 2) * self.d ** -0.5
                ds = (self.d + 4) * 2.0 ** -24 * self.d ** -0.5 * (q.abs() @ k.abs().transpose(1, 2)).amax(-1, keepdim=True)
                if causal:
                    pos = torch.arange(len(rows), device="cuda") - P
                    lim = torch.arange(nq, device="cuda") + (n - nq + 1)
                    s = s.masked_fill(pos[None, :] >= lim.clamp(min=0)[:, None], -math.inf)
                m = s.amax(-1, keepdim=True)
                p = torch.where(s > -math.inf, torch.exp(s - m.clamp(min=-1e300)), 0.0)
                l = p.sum(-1, keepdim=True)
                seen = l > 0
                l = torch.where(seen, l, 1.0)
                out = p @ v / l
                Wv = p @ v.abs() / l
                bound = out.abs() * 2.0 ** -11 + Wv * (2.0 ** -11 + 2 * ds + 2.0 ** -17) + \
                    len(rows) * 2.0 ** -25 * v.abs().amax() / l
                y[t], tol[t] = out.transpose(0, 1), tol[t] + torch.where(seen, bound, 0.0).transpose(0, 1)
        return y, tol

    def check(self, got=None, causal=True):
        got = self.out if got is None else got
        y, tol = self.reference(causal)
        err = (got.double() - y).abs()
        assert (err <= tol).all(), f"{int((~(err <= tol)).sum())} of {err.numel()} off, worst {float((err / tol).max()):.2f}"


GEOMETRY = [(32, 8, 128), (14, 2, 64), (12, 2, 128), (8, 8, 64), (64, 8, 128), (16, 1, 128), (40, 1, 64)]

SHAPES = {
    "one_token": [(0, [(1, 1)])],
    "one_page": [(16, [(1, 16)])],
    "prefix_only": [(37, [(1, 0), (1, 0)])],
    "no_prefix": [(0, [(1, 5), (1, 100), (3, 3)])],
    "nothing_to_see": [(0, [(2, 0), (1, 4)]), (0, [(1, 0)])],
    "queries_without_tokens": [(9, [(4, 2), (3, 0)]), (0, [(5, 2)])],  # limits below zero
    "odd_groups": [(131, [(1, 17), (2, 33), (1, 1)]), (0, [(1, 40)]), (16, [(7, 129)]), (257, [(1, 0), (0, 9), (1, 2)])],
    "empty_group": [(50, []), (50, [(1, 3)])],
    "drafts": [(1000, [(8, 8 + i) for i in range(9)])],
    "many_sequences": [(300, [(1, 1 + 7 * i % 45) for i in range(70)])],
    "long_prefix": [(20011, [(1, 20)])],
    "long_suffix": [(3, [(2, 9001)])],
    "prompts": [(513, [(200, 200), (77, 190), (1, 31)])],
    "prompt_alone": [(0, [(300, 300)])],
    "prompts_long": [(1500, [(260, 1000), (129, 129)]), (0, [(140, 700)])],
}


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("geometry", GEOMETRY[:3], ids=lambda g: "x".join(map(str, g)))
@pytest.mark.parametrize("shape", sorted(SHAPES))
def test_against_the_formula(engine, shape, geometry, causal):
    b = Batch(SHAPES[shape], *geometry, seed=len(shape))
    plan = b.plan(engine, causal=causal)
    plan.run(**b.views())
    plan.status()
    b.check(causal=causal)
    first = b.out.clone()
    b.out.fill_(math.nan)
    plan.run(**b.views())
    plan.status()
    assert first.equal(b.out)  # the same sums in the same order


@pytest.mark.parametrize("geometry", GEOMETRY[3:], ids=lambda g: "x".join(map(str, g)))
@pytest.mark.parametrize("shape", ["odd_groups", "drafts", "prompts"])
def test_head_layouts(engine, shape, geometry):
    b = Batch(SHAPES[shape], *geometry, seed=3)
    plan = b.plan(engine)
    plan.run(**b.views())
    plan.status()
    b.check()


@pytest.mark.parametrize("rows", [1, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 255, 256, 257, 300])
@pytest.mark.parametrize("tokens", [15, 127, 129, 700])
def test_row_and_page_edges(engine, rows, tokens):
    """Query rows and lengths around every tile edge, one kv head."""
    b = Batch([(tokens, [(1, 0)] * rows)], 1, 1, 128, seed=rows + tokens)
    plan = b.plan(engine)
    plan.run(**b.views())
    plan.status()
    b.check()


@pytest.mark.parametrize("qscale", [0.0, 40.0])
@pytest.mark.parametrize("shape", ["drafts", "prompts_long"])
def test_flat_and_peaked_scores(engine, shape, qscale):
    """Equal scores, and scores so far apart that single tokens win."""
    b = Batch(SHAPES[shape], 8, 2, 128, seed=5, qscale=qscale)
    plan = b.plan(engine)
    plan.run(**b.views())
    plan.status()
    b.check()


@pytest.mark.parametrize("shape", ["drafts", "prompts_long", "long_suffix"])
def test_growing_scores(engine, shape):
    """Scores that rise all along the pages, so the running maximum moves at every tile."""
    import torch
    b = Batch(SHAPES[shape], 4, 2, 64, seed=6)
    b.q.fill_(0.5)
    for rows in b.prefix_rows + b.suffix_rows:
        ramp = torch.linspace(-6, 6, max(len(rows), 1), device="cuda").half()[:, None, None]
        b.hot_k.view(-1, 2, 64)[rows] = ramp.expand(-1, 2, 64)[:len(rows)]
    plan = b.plan(engine)
    plan.run(**b.views())
    plan.status()
    b.check()


def test_lengths_change_under_one_plan_and_graph(engine):
    """One capture serves every length up to the pages' capacity."""
    import torch
    groups = [(100, [(1, 30), (4, 50)]), (333, [(1, 1)])]
    b = Batch(groups, 12, 2, 128, seed=7, spare_pages=2)
    plan = b.plan(engine)
    views = b.views()
    plan.run(**views)
    plan.status()
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.graph(graph, stream=side):
        plan.run(**views)
    for pre, suf in (([100, 333], [30, 50, 1]), ([0, 333], [30, 0, 1]), ([99, 1], [16, 3, 0]), ([100, 17], [5, 50, 1])):
        full_p, full_s = b.prefix_rows, b.suffix_rows
        b.prefix_lens.copy_(Batch.words(pre))
        b.suffix_lens.copy_(Batch.words(suf))
        b.out.fill_(math.nan)
        graph.replay()
        torch.cuda.synchronize()
        b.prefix_rows = [r[:n] for r, n in zip(full_p, pre)]
        b.suffix_rows = [r[:n] for r, n in zip(full_s, suf)]
        groups_now = [(pre[0], [(1, suf[0]), (4, suf[1])]), (pre[1], [(1, suf[2])])]
        b.groups = groups_now
        b.check()
        b.prefix_rows, b.suffix_rows, b.groups = full_p, full_s, groups
    plan.status()


def test_full_pages_without_lengths(engine):
    b = Batch([(64, [(1, 32), (1, 16)])], 8, 2, 64, seed=8)
    plan = b.plan(engine)
    plan.run(**b.views(prefix_lens=None, suffix_lens=None))
    plan.status()
    b.check()


@pytest.mark.parametrize("rows", [1, 40])
def test_bad_refs_are_skipped_and_reported(engine, rows):
    """A reference beyond the pool: its tokens are left out, the status says so once."""
    import torch
    b = Batch([(300, [(rows, 200)])], 4, 1, 128, seed=9, junk=0.0)
    refs = list(b.prefix_refs)
    refs[3], refs[7], refs[-1] = b.blocks, 0x7FFFFFFF, 0xFFFFFFFF
    plan = b.plan(engine)
    plan.run(**b.views(prefix_refs=Batch.words(refs)))
    with pytest.raises(W.WeaverError) as e:
        plan.status()
    assert e.value.status == 4
    plan.status()  # read and cleared
    keep = torch.ones(300, dtype=torch.bool, device="cuda")
    keep[48:64] = keep[112:128] = keep[288:] = False
    b.prefix_rows = [b.prefix_rows[0][keep]]
    b.check()


@pytest.mark.parametrize("rows", [2, 40])
def test_bad_refs_far_into_a_long_prefix(engine, rows):
    """Many token tiles an item: single bad references at its start, middle and end."""
    import torch
    n = 40000
    b = Batch([(n, [(rows, 20)])], 8, 8, 128, seed=19, junk=0.0)
    refs, keep = list(b.prefix_refs), torch.ones(n, dtype=torch.bool, device="cuda")
    for page in (0, 77, 1203, 1250, 2001, len(refs) - 1):
        refs[page] = b.blocks + page
        keep[page * 16:page * 16 + 16] = False
    plan = b.plan(engine)
    plan.run(**b.views(prefix_refs=Batch.words(refs)))
    with pytest.raises(W.WeaverError) as e:
        plan.status()
    assert e.value.status == 4
    b.prefix_rows = [b.prefix_rows[0][keep]]
    b.check()


@pytest.mark.parametrize("geometry", [(32, 8, 128), (14, 2, 64)], ids=lambda g: "x".join(map(str, g)))
def test_own_lists_of_very_different_lengths(engine, geometry):
    """Few rows a list, 1 to 6000 own tokens: items of many lengths, cut anywhere."""
    b = Batch([(90, [(1, 1 + (i * 977) % 401 * (15 if i % 5 == 0 else 1)) for i in range(45)])], *geometry, seed=23)
    plan = b.plan(engine)
    plan.run(**b.views())
    plan.status()
    b.check()


def test_more_lists_than_the_item_search_looks_at(engine):
    """Thousands of short lists beside one long one."""
    b = Batch([(40, [(1, 1 + i % 37) for i in range(470)] + [(1, 5000)])], 8, 8, 64, seed=29)
    plan = b.plan(engine)
    plan.run(**b.views())
    plan.status()
    b.check()


def test_lengths_beyond_the_pages_are_cut_and_reported(engine):
    b = Batch([(32, [(1, 16)])], 4, 1, 64, seed=10)
    plan = b.plan(engine)
    plan.run(**b.views(prefix_lens=Batch.words([1000]), suffix_lens=Batch.words([0xFFFFFFFF])))
    with pytest.raises(W.WeaverError) as e:
        plan.status()
    assert e.value.status == 4
    b.check()


def test_infinite_keys_behind_the_causal_limit(engine):
    """A key of +inf that only the last query sees leaves the earlier queries alone."""
    import torch
    b = Batch([(40, [(6, 70)])], 4, 1, 64, seed=11)
    y, tol = b.reference()
    b.hot_k.view(-1, 1, 64)[b.suffix_rows[0][-1]] = math.inf
    plan = b.plan(engine)
    plan.run(**b.views())
    plan.status()
    err = (b.out.double() - y).abs()[:5]
    assert (err <= tol[:5]).all()
    assert not torch.isfinite(b.out[5]).all()


@pytest.mark.parametrize("shape", ["odd_groups", "prompts", "nothing_to_see"])
def test_partials(engine, shape):
    """(m, l, o): o / l is the output, m + log l the log-sum-exp."""
    import torch
    b = Batch(SHAPES[shape], 12, 2, 128, seed=12)
    plan = b.plan(engine, partials=True)
    n = b.T * b.Hq
    m, l = (torch.full((n,), math.nan, device="cuda") for _ in range(2))
    o = torch.full((n, b.d), math.nan, device="cuda")
    plan.run(**b.views(out=None, part_m=m, part_l=l, part_o=o))
    plan.status()
    out = torch.empty(n, b.d, dtype=torch.float16, device="cuda")
    W.merge_partials(m.view(1, n), l.view(1, n), o.view(1, n, b.d), out)
    b.check(out.view(b.T, b.Hq, b.d))
    assert torch.equal(m == -math.inf, l == 0)


def test_two_plans_on_two_streams(engine):
    import torch
    bs = [Batch(SHAPES[s], 8, 2, 128, seed=13 + i) for i, s in enumerate(("drafts", "prompts"))]
    plans, streams = [b.plan(engine) for b in bs], [torch.cuda.Stream() for _ in bs]
    views = [p.views(**b.views()) for p, b in zip(plans, bs)]
    keep = [b.views() for b in bs]
    views = [p.views(**k) for p, k in zip(plans, keep)]
    torch.cuda.synchronize()
    for _ in range(5):
        for p, v, s in zip(plans, views, streams):
            p.run_views(v, s)
    for p, b in zip(plans, bs):
        p.status()
        b.check()


@pytest.mark.parametrize("change", ["q_dtype", "q_short", "out_strides", "refs", "pool", "lens_device", "lens_dtype"])
def test_python_refusals(engine, change):
    import torch
    b = Batch([(32, [(1, 16)])], 4, 1, 64, seed=14)
    plan = b.plan(engine)
    v = b.views()
    if change == "q_dtype":
        v["q"] = v["q"].bfloat16()
    elif change == "q_short":
        v["q"] = v["q"][:0]
    elif change == "out_strides":
        v["out"] = torch.zeros(1, 64, 4, dtype=torch.float16, device="cuda").transpose(1, 2)
    elif change == "refs":
        v["prefix_refs"] = v["prefix_refs"][:1]
    elif change == "pool":
        v["hot_v"] = v["hot_v"][:2]
    elif change == "lens_device":
        v["prefix_lens"] = v["prefix_lens"].cpu()
    elif change == "lens_dtype":
        v["suffix_lens"] = v["suffix_lens"].long()
    with pytest.raises(ValueError):
        plan.run(**v)


def test_null_views_are_refused(engine):
    b = Batch([(32, [(1, 16)])], 4, 1, 64, seed=15)
    plan = b.plan(engine)
    for name in ("q", "hot_k", "hot_v", "prefix_refs", "suffix_refs", "out"):
        with pytest.raises((W.WeaverError, ValueError)):
            plan.run(**b.views(**{name: None}))
    for name in ("q", "out"):
        with pytest.raises(W.WeaverError) as e:
            plan.run(**b.views(**{name: getattr(b, name).data_ptr() + 2}))
        assert e.value.status == 3


def test_out_over_q_is_refused(engine):
    b = Batch([(32, [(2, 16)])], 4, 1, 64, seed=16)
    plan = b.plan(engine)
    with pytest.raises(W.WeaverError) as e:
        plan.run(**b.views(out=b.q))
    assert e.value.status == 1


@pytest.mark.parametrize("shape", ["drafts", "prompts", "many_sequences"])
def test_rows_behind_the_last_query_are_left_alone(engine, shape):
    """A batch padded behind its last query: the padding of out keeps what it held."""
    import torch
    b = Batch(SHAPES[shape], 8, 2, 128, seed=17)
    pad = torch.full((9,) + tuple(b.q.shape[1:]), math.nan, dtype=torch.float16, device="cuda")
    out = torch.full((b.T + 9,) + tuple(b.q.shape[1:]), 3.0, dtype=torch.float16, device="cuda")
    plan = b.plan(engine)
    plan.run(**b.views(q=torch.cat([b.q, pad]), out=out))
    plan.status()
    b.check(out[:b.T])
    assert (out[b.T:] == 3.0).all()


def test_negative_and_zero_scale(engine):
    """scale < 0 turns the order of the scores round, 0 weighs every token alike."""
    b = Batch(SHAPES["prompts"], 8, 2, 64, seed=18)
    q = b.q.clone()
    for scale, factor in ((-b.d ** -0.5, -1.0), (0.0, 0.0)):
        plan = b.plan(engine, scale=scale)
        b.q = q
        plan.run(**b.views())
        plan.status()
        b.q = q * factor  # the formula with scale d^-1/2 and the queries turned round
        b.check()
    b.q = q
    small = Batch([(40, [(1, 9)])], 4, 1, 128, seed=19)  # the 16-row tiles too
    plan = small.plan(engine, scale=-small.d ** -0.5)
    plan.run(**small.views())
    plan.status()
    small.q = -small.q
    small.check()


@pytest.mark.parametrize("over", ["q", "q_last_row", "hot_k", "hot_v_last_page", "prefix_refs", "suffix_refs", "prefix_lens",
                                  "suffix_lens"])
@pytest.mark.parametrize("partials", [False, True])
def test_outputs_over_inputs_are_refused(engine, over, partials):
    """Every output over every input, by whole buffers and by a last row; nothing is written."""
    import torch
    b = Batch([(32, [(2, 16), (1, 3)])], 4, 1, 64, seed=21, junk=0.0)
    plan = b.plan(engine, partials=partials)
    views = b.views()
    for name in ("q", "hot_k", "hot_v", "prefix_refs", "suffix_refs", "prefix_lens", "suffix_lens"):
        # behind each input as much room as the largest output takes
        t = views[name]
        room = torch.zeros(t.numel() * t.element_size() + 16384, dtype=torch.uint8, device="cuda")
        views[name] = room[:t.numel() * t.element_size()].view(t.dtype).view(t.shape)
        views[name].copy_(t)
    name = over.split("_last")[0]
    t = views[name]
    at = t.data_ptr() + (t.numel() * t.element_size() - 16 if "_last" in over else 0)
    assert at % 16 == 0
    n = b.T * b.Hq
    own = dict(part_m=torch.zeros(n, device="cuda"), part_l=torch.zeros(n, device="cuda"),
               part_o=torch.zeros(n, b.d, device="cuda"), out=None) if partials else dict(out=b.out)
    held = t.clone()
    for output in [x for x, y in own.items() if y is not None]:
        with pytest.raises(W.WeaverError) as e:
            plan.run(**{**views, **own, output: at})
        assert e.value.status == 1 and "overlaps " + name in str(e.value)
    assert torch.equal(t, held)
    plan.run(**{**views, **own})
    plan.status()


def test_partial_outputs_over_each_other_are_refused(engine):
    import torch
    b = Batch([(32, [(2, 16), (1, 3)])], 4, 1, 64, seed=22)
    plan = b.plan(engine, partials=True)
    n = b.T * b.Hq
    room = torch.zeros(n * (b.d + 2), device="cuda")
    m, l, o = room[n * b.d:n * b.d + n], room[n * b.d + n:], room[:n * b.d]
    plan.run(**b.views(out=None, part_m=m, part_l=l, part_o=o))  # neighbours
    plan.status()
    for args in ((m, m, o), (m, o[-n:], o), (o[:n], l, o), (room[n * b.d - 1:][:n], l, o), (m, room[n * b.d + n - 1:][:n], o)):
        with pytest.raises(W.WeaverError) as e:
            plan.run(**b.views(out=None, part_m=args[0], part_l=args[1], part_o=args[2]))
        assert e.value.status == 1


def one_list(kind, n, logits_of, sink=False):
    """Lists of n tokens that share nine pages, so that the formula is a sum over
    their 144 rows by how often they come: "prompt" is one sequence of 2048
    queries (8192 rows a kv head), "single_tokens" 300 of one query; either way an
    item walks through as much of a list as a plan gives it.  Only the first
    dimension of q and K counts.  Returns (plan's arguments, tensors, out, the
    rows' scores, their counts, v) with the last three in 64 bits."""
    import torch
    Hq, Hkv, d, kinds = 32, 8, 128, 9
    g = torch.Generator(device="cuda").manual_seed(31)
    logits = logits_of(torch.randn(kinds, 16, generator=g, device="cuda"))
    hot_k = torch.zeros(kinds, 16, Hkv, d, dtype=torch.float16, device="cuda")
    hot_v = torch.rand(kinds, 16, 1, d, generator=g, device="cuda").add_(0.5).half().repeat(1, 1, Hkv, 1)
    if sink:
        logits[0, 0] = 0.0
        hot_v[0, 0] = 0.0
    hot_k[..., 0] = (logits / (8.0 * d ** -0.5)).half()[..., None]
    pages = [0] + [1 + i % (kinds - 1) for i in range(n // 16 - 1)]
    seqs = 1 if kind == "prompt" else 300
    nq = 2048 if kind == "prompt" else 1
    q = torch.zeros(seqs * nq, Hq, d, dtype=torch.float16, device="cuda")
    q[..., 0] = 8.0
    out = torch.full_like(q, math.nan)
    geometry = dict(q_heads=Hq, kv_heads=Hkv, head_dim=d, scale=d ** -0.5, q_indptr=[nq * b for b in range(seqs + 1)],
                    suffix_indptr=[len(pages) * b for b in range(seqs + 1)], causal=False)
    tensors = dict(q=q, hot_k=hot_k, hot_v=hot_v, suffix_refs=Batch.words(pages * seqs), out=out)
    count = torch.bincount(torch.tensor(pages, device="cuda"), minlength=kinds).double()[:, None]
    return geometry, tensors, out, hot_k[:, :, 0, 0].double() * 8.0 * d ** -0.5, count, hot_v[:, :, 0].double()


@pytest.mark.parametrize("kind,n", [("prompt", 1 << 19), ("single_tokens", 1 << 20)])
def test_long_sums_do_not_drift(engine, kind, n):
    """Flat scores over a very long list.

    The tensor cores add 16 tokens a step to the accumulator in two sums that are
    cut, not rounded: at most 2 * 2^-23 of it a step, so 2^-23 a step of the final
    sum while it grows evenly, 2^-12 over the 2048 steps of the longest run.  The
    fp32 sum of the probabilities is off by 2^-24 for each of the run's additions,
    512 of a token tile or 2048 of a page: 2^-13.  Both times W, beside the
    module's bound."""
    import torch
    geometry, tensors, out, s, count, v = one_list(kind, n, lambda x: x)
    plan = W.PrefixPlan(engine, **geometry)
    plan.run(**tensors)
    plan.status()
    p = torch.exp(s - s.max()) * count
    l = p.sum()
    y = (p[..., None] * v).sum((0, 1)) / l  # v > 0: also W
    ds = (128 + 4) * 2.0 ** -24 * s.abs().amax()
    tol = y * (2.0 ** -11 + 2.0 ** -11 + 2 * ds + 2.0 ** -17 + 2.0 ** -12 + 2.0 ** -13) + n * 2.0 ** -25 * v.amax() / l + \
        2.0 ** -25
    err = (out.double() - y).abs()
    assert (err <= tol).all(), f"worst {float((err / tol).max()):.2f}, {float((err / y).max()):.5f} of the value"


@pytest.mark.parametrize("tail,spread", [(-14.0, 1.0), (-17.5, 0.0), (-20.0, 1.0)])
@pytest.mark.parametrize("kind,n", [("prompt", 1 << 18), ("single_tokens", 1 << 14)])
def test_one_dominant_token_leaves_the_tail_its_weight(engine, kind, n, tail, spread):
    """A first token that takes nearly all of the softmax and has V = 0 (an
    attention sink) before a long tail `tail` nats below it: the output is the
    tail's share.

    The probabilities are held in f16 times a power of two, at least 2^7 for the
    largest, so one below f16's normal numbers is off by at most 2^-25 against a
    sum of 2^7: n 2^-32 max|v| in all.  Beside it the relative terms of the
    module's bound and of long sums (test_long_sums_do_not_drift), times W, here
    the tail's own share."""
    import torch
    geometry, tensors, out, s, count, v = one_list(kind, n, lambda x: tail + spread * x, sink=True)
    plan = W.PrefixPlan(engine, **geometry)
    plan.run(**tensors)
    plan.status()
    p = torch.exp(s) * count
    l = p.sum()
    y = (p[..., None] * v).sum((0, 1)) / l
    ds = (128 + 4) * 2.0 ** -24 * s.abs().amax()
    tol = y * (2.0 ** -11 + 2.0 ** -11 + 2 * ds + 2.0 ** -17 + 2.0 ** -12 + 2.0 ** -13) + n * 2.0 ** -32 * v.amax() / l + \
        2.0 ** -25
    assert (tol < 0.25 * y).all()  # the bound says something about the tail
    err = (out.double() - y).abs()
    assert (err <= tol).all(), f"worst {float((err / tol).max()):.2f}, {float((err / y).max()):.3f} of the value"


def test_status_waits_for_a_replay_on_another_stream(engine):
    """A captured run replayed behind other work, not on the stream it was
    captured on: the status that follows at once is that run's, and it is cleared
    for the next."""
    import torch
    b = Batch([(300, [(2, 20)])], 4, 1, 128, seed=33, junk=0.0)
    refs, good = Batch.words(b.prefix_refs), Batch.words(b.prefix_refs)
    plan = b.plan(engine)
    views = b.views(prefix_refs=refs)
    torch.cuda.synchronize()
    graph, side, other = torch.cuda.CUDAGraph(), torch.cuda.Stream(), torch.cuda.Stream()
    with torch.cuda.graph(graph, stream=side):
        plan.run(**views)
    for bad in (True, False, True):
        refs.copy_(good)
        if bad:
            refs[3] = b.blocks
        torch.cuda.synchronize()
        with torch.cuda.stream(other):
            torch.cuda._sleep(20_000_000)  # about 10 ms
            graph.replay()
        if bad:
            with pytest.raises(W.WeaverError) as e:
                plan.status()
            assert e.value.status == 4
        else:
            plan.status()
            b.check()
        assert other.query()


def test_a_plan_is_ready_when_it_is_made(engine):
    """Plans of different batches made, run at once on a stream of their own and
    dropped, one after the other in the memory that the last one left."""
    import torch
    bs = [Batch(SHAPES[s], 8, 2, 128, seed=34 + i) for i, s in enumerate(("drafts", "prompts", "many_sequences"))]
    views = [b.views(out=None) for b in bs]
    want = []
    for b in bs:
        plan = b.plan(engine)
        plan.run(**b.views())
        plan.status()
        b.check()
        want.append(b.out.clone())
    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    for i in range(30):
        b = bs[i % 3]
        out = torch.empty_like(b.out)
        torch.cuda.synchronize()
        plan = b.plan(engine)
        plan.run(stream, **{**views[i % 3], "out": out})
        stream.synchronize()
        assert torch.equal(out, want[i % 3])
        plan.close()
