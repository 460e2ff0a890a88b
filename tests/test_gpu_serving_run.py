"""The serving operators together, as a decode loop uses them: append into the
hot pool, attention behind a shared prefix, the step over cold codes merged in,
the flat-cache path, a DeviceFabric's pools.  Needs a B200.

Attention outputs are held to the path's parity bar (conftest.assert_close:
2e-3 + 1e-2 |reference|), the references computed in 64 bits from what the pool
holds."""
import math

import numpy as np
import pytest

from conftest import assert_close

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


def normal(shape, seed, dtype="float16", scale=1.0):
    import torch
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (scale * torch.randn(*shape, generator=g, device="cuda")).to(getattr(torch, dtype))


def words(x):
    import torch
    return torch.from_numpy(np.asarray(x, np.uint32).view(np.int32)).cuda()


def attend(q, k, v, scale):
    """softmax(scale q.K) V in 64 bits: q [n, Hq, d], k / v [t, Hkv, d], every token seen."""
    import torch
    G = q.shape[1] // k.shape[1]
    k, v = (x.double().repeat_interleave(G, 1).transpose(0, 1) for x in (k, v))
    return (torch.softmax(q.double().transpose(0, 1) @ k.transpose(1, 2) * scale, -1) @ v).transpose(0, 1)


@pytest.mark.parametrize("Hq,Hkv,d,dtype", [(32, 8, 128, "float16"), (14, 2, 64, "bfloat16")])
def test_a_batch_grows_behind_a_shared_prompt(engine, Hq, Hkv, d, dtype):
    """A prompt is appended once; then every step of one captured graph appends
    one token to each of five sequences and attends, over page boundaries."""
    import torch
    B, prompt, steps = 5, 203, 20
    scale = d ** -0.5
    pages = (prompt + 15) // 16
    own = (steps + 15) // 16
    blocks = pages + B * own + 2
    order = np.random.default_rng(1).permutation(blocks).astype(np.uint32)
    prefix_refs, suffix_refs = order[:pages], order[pages:pages + B * own]
    hot_k = torch.full((blocks, 16, Hkv, d), math.nan, dtype=torch.float16, device="cuda")
    hot_v = torch.full_like(hot_k, math.nan)
    rope = W.Rope(engine, head_dim=d, theta=500000.0)
    bad = torch.zeros(1, dtype=torch.int32, device="cuda")
    weight = (1 + 0.1 * normal((d,), 2, "float32")).to(getattr(torch, dtype))

    # the prompt: keys, values and the prompt's own attention (one sequence, causal)
    q, k, v = (normal((prompt, h, d), 3 + i, dtype) for i, h in enumerate((Hq, Hkv, Hkv)))
    qo = torch.empty((prompt, Hq, d), dtype=torch.float16, device="cuda")
    pos = torch.arange(prompt, device="cuda", dtype=torch.int32)
    slots = torch.from_numpy(W.token_slots(prefix_refs, [0, pages], [0], [0, prompt])).cuda()
    rope.append(q, k, v, pos, slots, hot_k, hot_v, qo, bad, q_weight=weight, k_weight=weight)
    alone = W.PrefixPlan(engine, q_heads=Hq, kv_heads=Hkv, head_dim=d, scale=scale, q_indptr=[0, prompt],
                         suffix_indptr=[0, pages])
    out = torch.empty_like(qo)
    alone.run(q=qo, hot_k=hot_k, hot_v=hot_v, suffix_refs=words(prefix_refs), suffix_lens=words([prompt]), out=out)
    alone.status()
    rows_k, rows_v = (p.view(-1, Hkv, d) for p in (hot_k, hot_v))
    for t in (0, 1, 15, 16, prompt - 1):
        ref = attend(qo[t:t + 1], rows_k[slots[:t + 1]], rows_v[slots[:t + 1]], scale)
        assert_close(out[t:t + 1].cpu(), ref.cpu(), what=f"prompt token {t}")

    # the steps, captured
    plan = W.PrefixPlan(engine, q_heads=Hq, kv_heads=Hkv, head_dim=d, scale=scale, q_indptr=range(B + 1),
                        suffix_indptr=[own * b for b in range(B + 1)], group_indptr=[0, B], prefix_indptr=[0, pages])
    q, k, v = (normal((B, h, d), 13 + i, dtype) for i, h in enumerate((Hq, Hkv, Hkv)))
    qo, out = (torch.empty((B, Hq, d), dtype=torch.float16, device="cuda") for _ in range(2))
    pos = torch.full((B,), prompt - 1, dtype=torch.int32, device="cuda")
    lens = torch.zeros(B, dtype=torch.int32, device="cuda")
    step_slots = torch.empty(B, dtype=torch.int64, device="cuda")
    tensors = dict(q=qo, hot_k=hot_k, hot_v=hot_v, prefix_refs=words(prefix_refs), suffix_refs=words(suffix_refs),
                   prefix_lens=words([prompt]), suffix_lens=lens, out=out)
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=side):
        rope.append(q, k, v, pos, step_slots, hot_k, hot_v, qo, bad, q_weight=weight, k_weight=weight)
        plan.run(**tensors)
    mine = [[] for _ in range(B)]
    for s in range(steps):
        new = W.token_slots(suffix_refs, [own * b for b in range(B + 1)], [s] * B, range(B + 1))
        step_slots.copy_(torch.from_numpy(new))
        pos += 1
        lens += 1
        for x, seed in ((q, 100), (k, 200), (v, 300)):
            x.copy_(normal(x.shape, seed + s, dtype))
        graph.replay()
        torch.cuda.synchronize()
        for b in range(B):
            mine[b].append(int(new[b]))
            at = torch.cat([slots, torch.tensor(mine[b], device="cuda")])
            assert_close(out[b:b + 1].cpu(), attend(qo[b:b + 1], rows_k[at], rows_v[at], scale).cpu(), what=f"step {s}")
    plan.status()
    assert int(bad) == 0


def test_hot_tokens_and_cold_codes_merge(engine, oracle_mod):
    """The hot part through PrefixPlan, the cold part through WeaverPlan, joined
    by merge_partials: the oracle's softmax over both."""
    import torch
    from aether_nexus_b200 import synth
    w = synth.make_workload("c1", seed=5, flag_refs=True, num_seqs=3, q_heads=16, kv_heads=4, head_dim=128,
                            hot_tokens=160, cold_tokens=1024, dict_size=512, shuffle_pages=True)
    dw = synth.to_device(w)
    B, nq, Hq, d = w["q"].shape
    rows = B * nq * Hq
    m, l, o = (torch.empty((2, rows) + t, dtype=torch.float32, device="cuda") for t in ((), (), (d,)))
    hot = W.PrefixPlan(engine, q_heads=Hq, kv_heads=4, head_dim=d, scale=w["scale"], q_indptr=range(B + 1),
                       suffix_indptr=w["hot_indptr"], partials=True)
    hot.run(q=dw["q"].view(-1, Hq, d), hot_k=dw["hot_k"], hot_v=dw["hot_v"], suffix_refs=dw["hot_refs"], part_m=m[0],
            part_l=l[0], part_o=o[0])
    cold = W.WeaverPlan(engine, num_seqs=B, num_queries=nq, q_heads=Hq, kv_heads=4, head_dim=d, dict_size=w["dict_size"],
                        scale=w["scale"], hot_indptr=[0] * (B + 1), cold_indptr=w["cold_indptr"], partials=True)
    cold.run(q=dw["q"], hot_k=None, hot_v=None, hot_refs=None, hot_pool_blocks=0, cold_k=dw["k_codes"],
             cold_v=dw["v_codes"], cold_refs=dw["cold_refs"], k_dict=dw["k_dict"], v_dict=dw["v_dict"], part_m=m[1],
             part_l=l[1], part_o=o[1])
    hot.status()
    cold.status()
    out = torch.empty((rows, d), dtype=torch.float16, device="cuda")
    W.merge_partials(m, l, o, out)
    torch.cuda.synchronize()
    assert_close(out.cpu(), oracle_mod.config_decode(w, precision="f64").reshape(rows, d), what="hot + cold")


def test_the_decode_step_reads_what_append_wrote(engine):
    """Full pages: WeaverPlan over the same pool and PrefixPlan agree with the formula."""
    import torch
    Hq, Hkv, d, blocks = 32, 8, 128, 6
    n = blocks * 16
    hot_k, hot_v = (torch.zeros((blocks, 16, Hkv, d), dtype=torch.float16, device="cuda") for _ in range(2))
    refs = np.array([3, 0, 5, 1, 4, 2], np.uint32)
    rope = W.Rope(engine, head_dim=d, layout="interleaved", rot_dim=64)
    q, k, v = (normal((n, h, d), 21 + i) for i, h in enumerate((Hq, Hkv, Hkv)))
    qo = torch.empty_like(q)
    bad = torch.zeros(1, dtype=torch.int32, device="cuda")
    slots = torch.from_numpy(W.token_slots(refs, [0, blocks], [0], [0, n])).cuda()
    rope.append(q, k, v, torch.arange(n, device="cuda", dtype=torch.int32), slots, hot_k, hot_v, qo, bad)
    last = qo[-1:].contiguous()
    ref = attend(last, hot_k.view(-1, Hkv, d)[slots], hot_v.view(-1, Hkv, d)[slots], d ** -0.5).cpu()
    step, pre = torch.empty_like(last), torch.empty_like(last)
    plan = W.WeaverPlan(engine, num_seqs=1, num_queries=1, q_heads=Hq, kv_heads=Hkv, head_dim=d, dict_size=512,
                        scale=d ** -0.5, hot_indptr=[0, blocks], cold_indptr=[0, 0])
    plan.run(q=last, hot_k=hot_k, hot_v=hot_v, hot_refs=words(refs), cold_k=None, cold_v=None, cold_refs=None,
             cold_pool_blocks=0, k_dict=None, v_dict=None, out=step)
    pp = W.PrefixPlan(engine, q_heads=Hq, kv_heads=Hkv, head_dim=d, scale=d ** -0.5, q_indptr=[0, 1],
                      suffix_indptr=[0, blocks])
    pp.run(q=last, hot_k=hot_k, hot_v=hot_v, suffix_refs=words(refs), out=pre)
    plan.status()
    pp.status()
    assert_close(step.cpu(), ref, what="WeaverPlan")
    assert_close(pre.cpu(), ref, what="PrefixPlan")


def test_rotated_heads_in_a_flat_cache(engine):
    import torch
    T, Hq, Hkv, d = 77, 12, 2, 128
    q, k, v = (normal((T, h, d), 31 + i) for i, h in enumerate((Hq, Hkv, Hkv)))
    rope = W.Rope(engine, head_dim=d, scaling=dict(type="linear", factor=2.0))
    rope.rotate(q, k, torch.arange(T, device="cuda", dtype=torch.int32), q, k)  # in place
    out = torch.empty((1, Hq, d), dtype=torch.float16, device="cuda")
    engine.multihead_attention(q[-1:].contiguous(), k, v, out, T)
    torch.cuda.synchronize()
    assert_close(out.cpu(), attend(q[-1:], k, v, d ** -0.5).cpu())


def test_pools_of_a_device_fabric(engine):
    """Raw pointers of a layer: append, then attend; the two layers stay apart."""
    import torch
    from aether_nexus_b200.fabric import DeviceFabric
    Hq, Hkv, d = 8, 2, 64
    fab = DeviceFabric(layers=2, kv_heads=Hkv, head_dim=d, dict_size=64, hot_blocks=4, cold_blocks=1, separate_v=True,
                       max_block_refs=4)
    rope = W.Rope(engine, head_dim=d)
    n = 20
    slots = torch.arange(16, 16 + n, device="cuda")
    plan = W.PrefixPlan(engine, q_heads=Hq, kv_heads=Hkv, head_dim=d, scale=d ** -0.5, q_indptr=[0, n],
                        suffix_indptr=[0, 2], causal=False)
    bad = torch.zeros(1, dtype=torch.int32, device="cuda")
    pos = torch.arange(n, device="cuda", dtype=torch.int32)
    outs, refs = [], []
    for layer in range(2):
        lv = fab.layer_views(layer)
        q, k, v = (normal((n, h, d), 41 + 10 * layer + i) for i, h in enumerate((Hq, Hkv, Hkv)))
        qo, ko = torch.empty_like(q), torch.empty_like(k)
        rope.append(q, k, v, pos, slots, lv["hot_k"], lv["hot_v"], qo, bad, hot_pool_blocks=lv["hot_pool_blocks"])
        rope.rotate(None, k, pos, None, ko)
        refs.append((qo, ko, v))
    for layer in range(2):
        lv = fab.layer_views(layer)
        qo, ko, v = refs[layer]
        out = torch.empty_like(qo)
        plan.run(q=qo, hot_k=lv["hot_k"], hot_v=lv["hot_v"], hot_pool_blocks=lv["hot_pool_blocks"],
                 suffix_refs=words([1, 2]), suffix_lens=words([n]), out=out)
        plan.status()
        assert_close(out.cpu(), attend(qo, ko, v, d ** -0.5).cpu(), what=f"layer {layer}")
    assert int(bad) == 0
    fab.close()
