"""The serving operators around the decode step: position rotation with
per-head norms, the append into the paged hot pool, and attention for a batch
whose sequences share a prefix.

``run`` computes a case either in its plain form (elementary torch operations
in 32 bits, angles in 64) or, where ``own`` is true, through the package's
entry points.  ``exact`` is the definition in 64 bits.
"""
import math
import random

import torch

own = False

BLOCK = 16
# (query heads, key/value heads, head size) of the framework's presets and of its 70B workload
HEADS = {"8b": (32, 8, 128), "2b": (32, 8, 64), "half_b": (14, 2, 64), "1_5b": (12, 2, 128), "70b": (64, 8, 128)}
DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16}
EPS = 1e-6
THETA = 500000.0


# ---- cases ------------------------------------------------------------------

def listed():
    rot = dict(op="rotate", dtype="f16", layout="half", rot=128, norm=False, scaling="none", far=0, spread=1)
    app = dict(op="append", dtype="f16", layout="half", rot=128, norm=False, scaling="none", far=0, pad=0, spread=1)
    att = dict(op="prefix", groups=1, nq=1, ragged=True, spread=1)
    return [
        # one token of one sequence: launch latency
        dict(rot, name="rotate_one_token", heads="8b", tokens=1),
        # an odd prompt chunk of a small model: normed heads, half of each head rotated, neighbouring pairs
        dict(rot, name="rotate_chunk_norm", heads="half_b", tokens=1777, dtype="bf16", layout="interleaved", rot=32,
             norm=True),
        # a long prompt of a 70B layer far into a scaled context
        dict(rot, name="rotate_long_far", heads="70b", tokens=8192, scaling="yarn", far=900000, norm=True),
        # one decode step of a small batch
        dict(app, name="append_step", heads="8b", tokens=16),
        # a verify batch of 64 sequences x 8 drafts, the batch padded at its end, normed heads
        dict(app, name="append_verify", heads="1_5b", tokens=512, dtype="bf16", norm=True, pad=37, far=30000),
        # an odd chunk of a small model, interleaved pairs, part of the head, linearly scaled
        dict(app, name="append_chunk", heads="half_b", tokens=4099, layout="interleaved", rot=32, scaling="linear"),
        # a long prompt of an 8B layer
        dict(app, name="append_prompt", heads="8b", tokens=16384),
        # four short continuations of one short prompt: latency
        dict(att, name="prefix_small", heads="half_b", seqs=4, prefix=200, suffix=40),
        # a serving batch behind one long system prompt
        dict(att, name="prefix_decode", heads="8b", seqs=64, prefix=32768, suffix=300),
        # a speculative-verify batch: 16 sequences x 8 drafts
        dict(att, name="prefix_verify", heads="8b", seqs=16, nq=8, prefix=8191, suffix=500),
        # prompt chunks behind a shared prefix
        dict(att, name="prefix_prompt", heads="8b", seqs=4, nq=1024, prefix=4096, suffix=1100),
        # six groups with prefixes of their own (one without), a 70B layer
        dict(att, name="prefix_groups", heads="70b", groups=6, seqs=40, prefix=20000, suffix=900),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["rotate", "append", "prefix"])
    heads = rng.choice(sorted(HEADS))
    d = HEADS[heads][2]
    case = dict(op=op, heads=heads, spread=rng.randrange(1 << 30))
    if op == "prefix":
        form = rng.choice(["decode", "verify", "prompt"])
        case["groups"] = rng.choice([1, 1, 2, 5])
        case["ragged"] = rng.random() < 0.8
        if form == "prompt":
            case["nq"] = _log(rng, 16, 1000)
            case["seqs"] = rng.randint(1, 4)
            case["prefix"] = _log(rng, 1, 4000)
            case["suffix"] = case["nq"] + _log(rng, 1, 200)
        else:
            case["nq"] = 1 if form == "decode" else rng.randint(2, 8)
            case["seqs"] = _log(rng, 1, 64)
            case["prefix"] = _log(rng, 1, 30000)
            case["suffix"] = case["nq"] + _log(rng, 1, 600)
        case["groups"] = min(case["groups"], case["seqs"])
        return case
    case["tokens"] = _log(rng, 1, 8000)
    case["dtype"] = rng.choice(["f16", "bf16"])
    case["layout"] = rng.choice(["half", "interleaved"])
    case["rot"] = rng.choice([d, d, d // 2, d // 4])
    case["norm"] = rng.random() < 0.5
    case["scaling"] = rng.choice(["none", "linear", "yarn"])
    case["far"] = rng.choice([0, _log(rng, 1, 1000000)])
    if op == "append":
        case["pad"] = rng.choice([0, rng.randrange(case["tokens"])])
    return case


def _lengths(case):
    """Per group (sequences, prefix tokens), per sequence (queries, suffix tokens); from the case alone."""
    rng = random.Random(case["spread"])
    n_groups, n_seqs = case["groups"], case["seqs"]
    cuts = sorted(rng.sample(range(1, n_seqs), n_groups - 1)) if n_groups > 1 else []
    bounds = [0] + cuts + [n_seqs]
    groups = []
    for g in range(n_groups):
        pre = case["prefix"]
        if n_groups > 1:
            pre = 0 if g == 1 else max(1, int(pre * rng.uniform(0.2, 1.0)))
        groups.append((bounds[g + 1] - bounds[g], pre))
    seqs = []
    for b in range(n_seqs):
        nq, suf = case["nq"], case["suffix"]
        if case["ragged"]:
            nq = max(1, int(nq * rng.uniform(0.6, 1.0)))
            suf = nq + int((suf - nq) * rng.uniform(0.0, 1.0))
        seqs.append((nq, suf))
    return groups, seqs


def work(case):
    hq, hkv, d = HEADS[case["heads"]]
    if case["op"] == "rotate":
        n = case["tokens"] * (hq + hkv) * d
        return {"bytes": 4 * n + 4 * case["tokens"], "flops": n * (6 + (4 if case["norm"] else 0))}
    if case["op"] == "append":
        t = case["tokens"] - case["pad"]
        return {"bytes": 4 * t * (hq + 2 * hkv) * d + 12 * case["tokens"],
                "flops": t * (hq + hkv) * d * (6 + (4 if case["norm"] else 0))}
    groups, seqs = _lengths(case)
    kv = sum(p for _, p in groups) + sum(s for _, s in seqs)
    pairs, b = 0, 0
    for n, pre in groups:
        for nq, suf in seqs[b:b + n]:
            pairs += nq * pre + sum(suf - nq + 1 + j for j in range(nq))
        b += n
    tokens = sum(nq for nq, _ in seqs)
    return {"bytes": kv * hkv * d * 4 + tokens * hq * d * 4, "flops": 4 * d * hq * pairs}


# ---- inputs -------------------------------------------------------------------

def _randn(gen, shape, dtype, scale=1.0):
    return (torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32) * scale).to(dtype)


def _heads_inputs(case, seed):
    """q, k, v as slices of one projection's output, positions, slots, pools, weights."""
    hq, hkv, d = HEADS[case["heads"]]
    t, dt = case["tokens"], DTYPES[case["dtype"]]
    gen = torch.Generator(device="cuda").manual_seed(seed)
    rng = random.Random(seed)
    s = {}
    if case["heads"] == "2b":  # three projections of their own
        s["q"], s["k"], s["v"] = (_randn(gen, (t, h, d), dt, 1.5) for h in (hq, hkv, hkv))
    else:  # one fused projection
        fused = _randn(gen, (t, hq + 2 * hkv, d), dt, 1.5)
        s["q"], s["k"], s["v"] = fused[:, :hq], fused[:, hq:hq + hkv], fused[:, hq + hkv:]
    first = case["far"]
    s["positions"] = torch.arange(first, first + t, device="cuda", dtype=torch.int32)
    s["qw"] = s["kw"] = None
    if case["norm"]:
        s["qw"] = (1.0 + 0.2 * torch.randn(d, generator=gen, device="cuda")).to(dt)
        s["kw"] = (1.0 + 0.2 * torch.randn(d, generator=gen, device="cuda")).to(dt)
    if case["op"] == "append":
        live = t - case["pad"]
        n_blocks = (live + BLOCK - 1) // BLOCK + 5
        order = list(range(n_blocks))
        rng.shuffle(order)
        start = rng.randrange(BLOCK)
        idx = torch.arange(start, start + live, device="cuda")
        refs = torch.tensor(order, device="cuda", dtype=torch.int64)
        slots = torch.full((t,), -1, device="cuda", dtype=torch.int64)
        slots[:live] = refs[idx // BLOCK] * BLOCK + idx % BLOCK
        s["slots"] = slots
        s["hot_k"] = _randn(gen, (n_blocks, BLOCK, hkv, d), torch.float16)
        s["hot_v"] = _randn(gen, (n_blocks, BLOCK, hkv, d), torch.float16)
    return s


def _pages(rng, counts, first):
    """Shuffled pool blocks for each count of tokens; the flag bit of a reference is set at random."""
    n = [(c + BLOCK - 1) // BLOCK for c in counts]
    ids = first[:sum(n)]
    del first[:sum(n)]
    ptr = [0]
    for c in n:
        ptr.append(ptr[-1] + c)
    refs = [i | (0x80000000 if rng.random() < 0.3 else 0) for i in ids]
    return refs, ptr


def _u32(values):
    return torch.tensor([v - (1 << 32) if v >= 1 << 31 else v for v in values] or [0], device="cuda",
                        dtype=torch.int32)


def _prefix_inputs(case, seed):
    hq, hkv, d = HEADS[case["heads"]]
    groups, seqs = _lengths(case)
    gen = torch.Generator(device="cuda").manual_seed(seed)
    rng = random.Random(seed)
    need = sum((p + BLOCK - 1) // BLOCK for _, p in groups) + sum((x + BLOCK - 1) // BLOCK for _, x in seqs)
    n_blocks = need + 7
    order = list(range(n_blocks))
    rng.shuffle(order)
    s = {"groups": groups, "seqs": seqs}
    s["prefix_refs_host"], s["prefix_indptr"] = _pages(rng, [p for _, p in groups], order)
    s["suffix_refs_host"], s["suffix_indptr"] = _pages(rng, [x for _, x in seqs], order)
    s["prefix_refs"], s["suffix_refs"] = _u32(s["prefix_refs_host"]), _u32(s["suffix_refs_host"])
    s["prefix_lens"] = _u32([p for _, p in groups])
    s["suffix_lens"] = _u32([x for _, x in seqs])
    s["group_indptr"], s["q_indptr"] = [0], [0]
    for n, _ in groups:
        s["group_indptr"].append(s["group_indptr"][-1] + n)
    for nq, _ in seqs:
        s["q_indptr"].append(s["q_indptr"][-1] + nq)
    # normal rows, so logits spread by about 2; a key stands out here and there, as in trained heads
    s["q"] = _randn(gen, (s["q_indptr"][-1], hq, d), torch.float16, 2.0)
    s["hot_k"] = _randn(gen, (n_blocks, BLOCK, hkv, d), torch.float16)
    s["hot_k"][torch.rand(n_blocks, BLOCK, generator=gen, device="cuda") < 0.004] *= 2.5
    s["hot_v"] = _randn(gen, (n_blocks, BLOCK, hkv, d), torch.float16)
    return s


# ---- the rotation's frequencies ------------------------------------------------

YARN = dict(factor=16.0, original_length=65536, beta_fast=32.0, beta_slow=1.0)
LINEAR = dict(factor=4.0)


def _frequencies(case):
    """(inverse frequencies, factor on cos and sin) in 64 bits."""
    r = case["rot"]
    i = torch.arange(r // 2, dtype=torch.float64)
    f = THETA ** (-2.0 * i / r)
    if case["scaling"] == "linear":
        return f / LINEAR["factor"], 1.0
    if case["scaling"] == "yarn":
        def pair_of(turns):  # the pair that makes `turns` turns over the original length
            return r * math.log(YARN["original_length"] / (turns * 2.0 * math.pi)) / (2.0 * math.log(THETA))
        low = max(math.floor(pair_of(YARN["beta_fast"])), 0)
        high = min(math.ceil(pair_of(YARN["beta_slow"])), r // 2 - 1)
        ramp = ((i - low) / max(high - low, 1e-3)).clamp(0.0, 1.0)
        return f * (1.0 - ramp) + f / YARN["factor"] * ramp, 0.1 * math.log(YARN["factor"]) + 1.0
    return f, 1.0


# ---- prepare and run -------------------------------------------------------------

def prepare(case, seed):
    hq, hkv, d = HEADS[case["heads"]]
    s = _prefix_inputs(case, seed) if case["op"] == "prefix" else _heads_inputs(case, seed)
    s["case"] = case
    if case["op"] == "prefix":
        s["out"] = torch.zeros_like(s["q"])
    else:
        f, af = _frequencies(case)
        s["freq"], s["factor"] = f.cuda(), af
        odt = torch.float16 if case["op"] == "append" else s["q"].dtype
        s["q_out"] = torch.zeros(s["q"].shape, device="cuda", dtype=odt)
        s["k_out"] = torch.zeros(s["k"].shape, device="cuda", dtype=odt) if case["op"] == "rotate" else None
    if own:
        from aether_nexus_b200 import PrefixPlan, Rope, WeaverEngine
        s["engine"] = WeaverEngine(torch.cuda.current_device())
        if case["op"] == "prefix":
            s["plan"] = PrefixPlan(s["engine"], q_heads=hq, kv_heads=hkv, head_dim=d, scale=1.0 / math.sqrt(d),
                                   q_indptr=s["q_indptr"], group_indptr=s["group_indptr"],
                                   prefix_indptr=s["prefix_indptr"], suffix_indptr=s["suffix_indptr"], causal=True)
        else:
            scaling = {"none": None, "linear": dict(type="linear", **LINEAR), "yarn": dict(type="yarn", **YARN)}
            s["rope"] = Rope(s["engine"], head_dim=d, rot_dim=case["rot"], theta=THETA, layout=case["layout"],
                             scaling=scaling[case["scaling"]])
            s["bad"] = torch.zeros(1, device="cuda", dtype=torch.int32)
    return s


def run(state):
    op = state["case"]["op"]
    if own:
        return {"rotate": _own_rotate, "append": _own_append, "prefix": _own_prefix}[op](state)
    return {"rotate": _plain_rotate, "append": _plain_append, "prefix": _plain_prefix}[op](state)


def _own_rotate(s):
    s["rope"].rotate(s["q"], s["k"], s["positions"], s["q_out"], s["k_out"], q_weight=s["qw"], k_weight=s["kw"],
                     eps=EPS)
    return s["q_out"], s["k_out"]


def _own_append(s):
    s["rope"].append(s["q"], s["k"], s["v"], s["positions"], s["slots"], s["hot_k"], s["hot_v"], s["q_out"], s["bad"],
                     q_weight=s["qw"], k_weight=s["kw"], eps=EPS)
    return s["q_out"], s["hot_k"], s["hot_v"]


def _own_prefix(s):
    s["plan"].run(q=s["q"], hot_k=s["hot_k"], hot_v=s["hot_v"], prefix_refs=s["prefix_refs"],
                  suffix_refs=s["suffix_refs"], prefix_lens=s["prefix_lens"], suffix_lens=s["suffix_lens"],
                  out=s["out"])
    return s["out"]


def _plain_turn(x, weight, s):
    """Norm and rotation of [tokens, heads, d] in 32 bits."""
    case, x = s["case"], x.float()
    if weight is not None:
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * weight.float()
    r = case["rot"]
    angle = s["positions"].double()[:, None] * s["freq"][None, :]
    cos = (torch.cos(angle) * s["factor"]).float()[:, None, :]
    sin = (torch.sin(angle) * s["factor"]).float()[:, None, :]
    if case["layout"] == "half":
        a, b = x[..., :r // 2], x[..., r // 2:r]
        y = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    else:
        a, b = x[..., 0:r:2], x[..., 1:r:2]
        y = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    return torch.cat([y, x[..., r:]], -1)


def _plain_rotate(s):
    s["q_out"].copy_(_plain_turn(s["q"], s["qw"], s))
    s["k_out"].copy_(_plain_turn(s["k"], s["kw"], s))
    return s["q_out"], s["k_out"]


def _plain_append(s):
    live = s["case"]["tokens"] - s["case"]["pad"]
    hkv, d = s["k"].shape[1:]
    slots = s["slots"][:live]
    s["q_out"][:live] = _plain_turn(s["q"], s["qw"], s)[:live].half()
    s["hot_k"].view(-1, hkv, d)[slots] = _plain_turn(s["k"], s["kw"], s)[:live].half()
    s["hot_v"].view(-1, hkv, d)[slots] = s["v"][:live].half()
    return s["q_out"], s["hot_k"], s["hot_v"]


def _plain_rows(pool, refs, ptr, i, n):
    """The first n rows of page list i of a pool: [heads, n, d] in 32 bits."""
    blocks = (refs[ptr[i]:ptr[i + 1]] & 0x7FFFFFFF).long()
    return pool[blocks].flatten(0, 1)[:n].float().transpose(0, 1)


def _plain_prefix(s):
    q, out = s["q"], s["out"]
    hkv, d = s["hot_k"].shape[2:]
    g = q.shape[1] // hkv
    scale = 1.0 / math.sqrt(d)
    b = 0
    for gi, (n, pre) in enumerate(s["groups"]):
        t0, t1 = s["q_indptr"][b], s["q_indptr"][b + n]
        # [kv heads, tokens * group, d]: one product per kv head for every query of the group
        rows = q[t0:t1].float().view(t1 - t0, hkv, g, d).permute(1, 0, 2, 3).reshape(hkv, -1, d)
        m = torch.full(rows.shape[:2], -math.inf, device=q.device)
        l = torch.zeros_like(m)
        acc = torch.zeros_like(rows)
        if pre:
            k = _plain_rows(s["hot_k"], s["prefix_refs"], s["prefix_indptr"], gi, pre)
            v = _plain_rows(s["hot_v"], s["prefix_refs"], s["prefix_indptr"], gi, pre)
            p = torch.matmul(rows, k.transpose(1, 2)).mul_(scale)
            m = p.amax(-1)
            p = p.sub_(m[..., None]).exp_()
            l = p.sum(-1)
            acc = torch.matmul(p, v)
            del p
        for j in range(b, b + n):
            nq, suf = s["seqs"][j]
            r0, r1 = (s["q_indptr"][j] - t0) * g, (s["q_indptr"][j + 1] - t0) * g
            k = _plain_rows(s["hot_k"], s["suffix_refs"], s["suffix_indptr"], j, suf)
            v = _plain_rows(s["hot_v"], s["suffix_refs"], s["suffix_indptr"], j, suf)
            p = torch.matmul(rows[:, r0:r1], k.transpose(1, 2)) * scale
            limit = torch.arange(r1 - r0, device=q.device) // g + (suf - nq + 1)
            p = p.masked_fill(torch.arange(suf, device=q.device)[None, :] >= limit[:, None], -math.inf)
            m2 = torch.maximum(m[:, r0:r1], p.amax(-1))
            p = torch.exp(p - m2[..., None])
            old = torch.exp(m[:, r0:r1] - m2)
            o = acc[:, r0:r1] * old[..., None] + torch.matmul(p, v)
            o = o / (l[:, r0:r1] * old + p.sum(-1))[..., None]
            out[s["q_indptr"][j]:s["q_indptr"][j + 1]] = \
                o.view(hkv, nq, g, d).permute(1, 0, 2, 3).reshape(nq, hkv * g, d).half()
        b += n
    return out


# ---- the definitions in 64 bits ----------------------------------------------------

def exact(case, seed):
    if case["op"] == "prefix":
        return _exact_prefix(_prefix_inputs(case, seed), HEADS[case["heads"]])
    s = _heads_inputs(case, seed)
    q, k = _exact_turn(case, s, "q", "qw"), _exact_turn(case, s, "k", "kw")
    if case["op"] == "rotate":
        return q, k
    pools = [s["hot_k"].double(), s["hot_v"].double()]
    keep = s["slots"] >= 0
    where = s["slots"][keep]
    for pool, new in zip(pools, (k, s["v"].double())):
        pool[where // BLOCK, where % BLOCK] = new[keep]
    q[~keep] = 0.0  # padding: the zeros that the output held
    return q, pools[0], pools[1]


def _exact_turn(case, s, name, wname):
    x, r = s[name].double(), case["rot"]
    if s[wname] is not None:
        x = x / (x.square().sum(-1, keepdim=True) / x.shape[-1] + EPS).sqrt() * s[wname].double()
    freq, factor = _frequencies(case)
    out = x.clone()
    for i in range(r // 2):
        ia, ib = (i, i + r // 2) if case["layout"] == "half" else (2 * i, 2 * i + 1)
        turn = torch.polar(torch.full(s["positions"].shape, factor, device="cuda", dtype=torch.float64),
                           s["positions"].double() * float(freq[i]))
        z = torch.complex(x[..., ia], x[..., ib]) * turn[:, None]
        out[..., ia], out[..., ib] = z.real, z.imag
    return out


def _exact_prefix(s, geometry):
    hq, hkv, d = geometry
    out = torch.zeros(s["q"].shape, device="cuda", dtype=torch.float64)
    cells = torch.arange(BLOCK, device="cuda")
    b = 0
    for gi, (n, pre) in enumerate(s["groups"]):
        for j in range(b, b + n):
            nq, suf = s["seqs"][j]
            pages = s["prefix_refs_host"][s["prefix_indptr"][gi]:s["prefix_indptr"][gi + 1]]
            mine = s["suffix_refs_host"][s["suffix_indptr"][j]:s["suffix_indptr"][j + 1]]
            where = [(torch.tensor([p % (1 << 31) for p in part], device="cuda", dtype=torch.int64)[:, None] * BLOCK
                      + cells).flatten()[:count] for part, count in ((pages, pre), (mine, suf))]
            where = torch.cat(where)
            q = s["q"][s["q_indptr"][j]:s["q_indptr"][j + 1]].double()
            seen = torch.arange(nq, device="cuda")[:, None] + (pre + suf - nq) >= torch.arange(pre + suf, device="cuda")
            for h in range(hkv):
                keys = s["hot_k"].view(-1, hkv, d)[where, h].double()
                values = s["hot_v"].view(-1, hkv, d)[where, h].double()
                for c in range(h * (hq // hkv), (h + 1) * (hq // hkv)):
                    logits = (q[:, c] @ keys.T / math.sqrt(d)).masked_fill(~seen, -math.inf)
                    out[s["q_indptr"][j]:s["q_indptr"][j + 1], c] = torch.softmax(logits, -1) @ values
        b += n
    return out
