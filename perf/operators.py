"""The paged KV-cache operators as cases to measure, with their plain forms.

Four operators that a serving program runs one after the other on one layer of
a cache kept in pages:

  rope    rotary positions of q and k and the append of k and v to the pages
  attend  attention of a chunk of new tokens over the pages (one token: decode)
  mass    the attention weight each cached key received, accumulated
  evict   the choice of the keys to keep by that weight, and their compaction

run() computes them in elementary torch operations, or, with `own` set,
through jetsonfabric_b200.paged. Sequences are ragged: the rows of sequence b
are q_start[b]..q_start[b + 1] - 1 and its keys the slots 0..kv_len[b] - 1 of
its row of the page table; its new tokens hold the last slots.
"""
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


# ---- cases -----------------------------------------------------------------------

def listed():
    return [
        # one new token of one short conversation, 12/2 heads: the latency of a decode step
        dict(name="rope_decode_one", op="rope", heads=12, kv_heads=2, head_dim=128, dtype="f16", source="f32",
             page_size=16, seqs=1, q_lo=1, q_hi=1, kv_lo=777, kv_hi=777, pad=0, rope_dims=128, interleaved=False,
             scaling="none"),
        # a prompt's chunk at 28/4 heads with positions scaled beyond the trained context
        dict(name="rope_chunk_scaled", op="rope", heads=28, kv_heads=4, head_dim=128, dtype="bf16", source="bf16",
             page_size=64, seqs=2, q_lo=8000, q_hi=8192, kv_lo=40000, kv_hi=65536, pad=0, rope_dims=128,
             interleaved=False, scaling="yarn"),
        # ragged prompts, rotation of half the head in the interleaved layout, f32 projections
        dict(name="rope_partial_ragged", op="rope", heads=40, kv_heads=8, head_dim=128, dtype="f16", source="f32",
             page_size=16, seqs=9, q_lo=37, q_hi=411, kv_lo=500, kv_hi=2100, pad=5, rope_dims=64, interleaved=True,
             scaling="linear"),
        # decode of one short conversation
        dict(name="attend_decode_one", op="attend", heads=12, kv_heads=2, head_dim=128, dtype="f16", page_size=16,
             seqs=1, q_lo=1, q_hi=1, kv_lo=777, kv_hi=777, pad=0, window=0),
        # 64 sequences decoding together after prompts of 1024 tokens, 28/4 heads
        dict(name="attend_decode_batch", op="attend", heads=28, kv_heads=4, head_dim=128, dtype="bf16", page_size=16,
             seqs=64, q_lo=1, q_hi=1, kv_lo=1025, kv_hi=1280, pad=0, window=0),
        # few sequences with very long contexts: the cache is the work
        dict(name="attend_decode_long", op="attend", heads=28, kv_heads=4, head_dim=128, dtype="f16", page_size=64,
             seqs=6, q_lo=1, q_hi=1, kv_lo=9001, kv_hi=65001, pad=0, window=0),
        # chunks of several prompts over what is cached, with a sliding window, 40/8 heads, padded batch
        dict(name="attend_chunk_ragged", op="attend", heads=40, kv_heads=8, head_dim=128, dtype="f16", page_size=16,
             seqs=5, q_lo=65, q_hi=519, kv_lo=1500, kv_hi=6011, pad=3, window=2048),
        # a whole prompt at once: the matrix products are the work
        dict(name="attend_prompt", op="attend", heads=28, kv_heads=4, head_dim=128, dtype="bf16", page_size=64,
             seqs=1, q_lo=8192, q_hi=8192, kv_lo=8192, kv_hi=8192, pad=0, window=0),
        # the weights of one decode step of 64 sequences
        dict(name="mass_decode_batch", op="mass", heads=28, kv_heads=4, head_dim=128, dtype="bf16", page_size=16,
             seqs=64, q_lo=1, q_hi=1, kv_lo=1025, kv_hi=1280, pad=0, window=0),
        # the weights of prompt chunks
        dict(name="mass_chunk", op="mass", heads=16, kv_heads=2, head_dim=128, dtype="f16", page_size=64,
             seqs=3, q_lo=700, q_hi=2048, kv_lo=2048, kv_hi=8000, pad=0, window=0),
        # one conversation grown past a small budget
        dict(name="evict_one", op="evict", heads=12, kv_heads=2, head_dim=128, dtype="f16", page_size=16, seqs=1,
             kv_lo=700, kv_hi=700, budget=512, recent=64),
        # a batch of long conversations cut to half a budget's worth, a few still below it
        dict(name="evict_batch", op="evict", heads=28, kv_heads=4, head_dim=128, dtype="bf16", page_size=64, seqs=32,
             kv_lo=1500, kv_hi=8192, budget=2048, recent=256),
    ]


def _between(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["rope", "attend", "attend", "attend", "mass", "evict"])
    heads, kv_heads = rng.choice([(12, 2), (16, 2), (28, 4), (40, 8), (8, 8), (14, 2), (6, 1)])
    case = dict(op=op, heads=heads, kv_heads=kv_heads, head_dim=rng.choice([64, 128, 128, 128, 96]),
                dtype=rng.choice(["f16", "bf16"]), page_size=rng.choice([16, 32, 64, 128]))
    if op == "evict":
        hi = _between(rng, 40, 8192)
        budget = _between(rng, 16, 2048)
        case.update(seqs=_between(rng, 1, 24), kv_lo=max(1, int(hi * rng.uniform(0.2, 1))), kv_hi=hi, budget=budget,
                    recent=int(budget * rng.uniform(0, 1)))
        return case
    if op == "rope":
        rows = _between(rng, 1, 8000)
        seqs = min(rows, _between(rng, 1, 40))
        q_hi = max(1, rows // seqs)
        kv_hi = q_hi + _between(rng, 1, 60000 // seqs)
        dims = [d for d in (32, 64, 96, 128) if d <= case["head_dim"]]
        case.update(source=rng.choice(["f32", case["dtype"]]), seqs=seqs, q_lo=max(1, int(q_hi * rng.uniform(0.3, 1))),
                    q_hi=q_hi, kv_lo=max(q_hi, int(kv_hi * rng.uniform(0.5, 1))), kv_hi=kv_hi, pad=rng.randrange(4),
                    rope_dims=rng.choice(dims), interleaved=rng.random() < 0.5,
                    scaling=rng.choice(["none", "linear", "yarn"]))
        return case
    if rng.random() < 0.5:  # single tokens
        seqs = _between(rng, 1, 64)
        kv_hi = _between(rng, 2, min(65000, 100000 // seqs))
        q_lo = q_hi = 1
    else:
        seqs = _between(rng, 1, 8)
        q_hi = _between(rng, 2, 6000 // seqs)
        q_lo = max(1, int(q_hi * rng.uniform(0.1, 1)))
        kv_hi = q_hi + _between(rng, 1, 12000 // seqs)
        if heads * q_hi * kv_hi * seqs > 28 * 8192 * 4096:
            kv_hi = max(q_hi, 28 * 8192 * 4096 // (heads * q_hi * seqs))
    case.update(seqs=seqs, q_lo=q_lo, q_hi=q_hi, kv_lo=max(q_hi, int(kv_hi * rng.uniform(0.4, 1))), kv_hi=kv_hi,
                pad=rng.randrange(4), window=rng.choice([0, 0, _between(rng, 8, 4096)]))
    return case


def _spread(lo, hi, n):
    """n lengths from lo to hi in a fixed mixed order, a function of the case alone."""
    if n == 1:
        return [hi]
    order = sorted(range(n), key=lambda b: (b * 7919 + 13) % 104729)
    return [lo + (hi - lo) * order[b] // (n - 1) for b in range(n)]


def _lengths(case):
    kv = _spread(case["kv_lo"], case["kv_hi"], case["seqs"])
    if case["op"] == "evict":
        return [0] * case["seqs"], kv
    new = _spread(case["q_lo"], case["q_hi"], case["seqs"])
    return new, [max(k, n) for k, n in zip(kv, new)]


def _pairs(new, kv, window):
    """(row, key) pairs that attend, and the keys that any row attends."""
    window = window or max(kv)
    pairs = sum(sum(min(window, k - n + i + 1) for i in range(n)) for n, k in zip(new, kv))
    return pairs, sum(min(k, n + window - 1) for n, k in zip(new, kv))


def work(case):
    new, kv = _lengths(case)
    kvh, hd = case["kv_heads"], case["head_dim"]
    if case["op"] == "evict":
        kept = sum(min(k, case["budget"]) for k in kv) * kvh
        return {"bytes": 4 * kvh * sum(kv) + kept * (4 + 4 + 2 * 2 * 2 * hd), "flops": 0}
    rows, h = sum(new), case["heads"]
    if case["op"] == "rope":
        src = 4 if case["source"] == "f32" else 2
        return {"bytes": rows * hd * (h + 2 * kvh) * (src + 2) + 4 * rows, "flops": 3 * rows * case["rope_dims"] * (h + kvh)}
    pairs, keys = _pairs(new, kv, case["window"])
    if case["op"] == "attend":
        return {"bytes": rows * h * (hd * 2 * 2 + 4) + keys * kvh * hd * 2 * 2, "flops": 4 * hd * h * pairs}
    return {"bytes": rows * h * (hd * 2 + 4) + keys * kvh * hd * 2 + 8 * kvh * sum(kv), "flops": 2 * hd * h * pairs}


# ---- inputs ----------------------------------------------------------------------

def _frequencies(rope_dims, scaling):
    """Radians per position of each pair, and the factor on cos and sin."""
    inv = [1e6 ** (-2 * i / rope_dims) for i in range(rope_dims // 2)]
    if scaling == "linear":
        return [f / 4 for f in inv], 1.0
    if scaling == "yarn":  # four times a trained context of 32768: low frequencies are interpolated
        def edge(turns):
            return rope_dims * math.log(32768 / (turns * 2 * math.pi)) / (2 * math.log(1e6))
        low, high = max(math.floor(edge(32)), 0), min(math.ceil(edge(1)), rope_dims - 1)
        high = high + 1e-3 if high == low else high
        keep = [1 - min(max((i - low) / (high - low), 0), 1) for i in range(rope_dims // 2)]
        return [f * k + f / 4 * (1 - k) for f, k in zip(inv, keep)], 0.1 * math.log(4) + 1
    return inv, 1.0


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    host = torch.Generator().manual_seed(seed)
    new, kv = _lengths(case)
    seqs, ps, kvh, hd, h = case["seqs"], case["page_size"], case["kv_heads"], case["head_dim"], case["heads"]
    dt = DTYPES[case["dtype"]]
    width = max(-(-k // ps) for k in kv)
    kept = -(-case["budget"] // ps) if case["op"] == "evict" else 0
    pages = seqs * (width + kept) + 3

    def normal(*shape, std=1.0, dtype=dt):
        return (torch.randn(*shape, device="cuda", generator=g) * std).to(dtype)

    # the pages of a cache in use lie in no order; the rest of the pool is other conversations' keys
    k_pool, v_pool = normal(pages, ps, kvh, hd), normal(pages, ps, kvh, hd)
    order = torch.randperm(pages, generator=host).to(torch.int32)
    table = order[:seqs * width].view(seqs, width).cuda()
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    rows = starts[-1] + case.get("pad", 0)
    s = dict(case=case, k_pool=k_pool, v_pool=v_pool, table=table, max_kv=max(kv), max_q=max(new), n=starts[-1],
             q_start=torch.tensor(starts, dtype=torch.int32).cuda(), kv_len=torch.tensor(kv, dtype=torch.int32).cuda(),
             scale=hd ** -0.5)
    if case["op"] == "rope":
        src = DTYPES[case["source"]]
        s.update(q=normal(rows, h, hd, dtype=src), k=normal(rows, kvh, hd, dtype=src), v=normal(rows, kvh, hd, dtype=src),
                 q_out=torch.zeros(rows, h, hd, dtype=dt, device="cuda"))
        freq, factor = _frequencies(case["rope_dims"], case["scaling"])
        s.update(freq=torch.tensor(freq, dtype=torch.float64).cuda(), factor=factor)
        first = torch.tensor([k - n for k, n in zip(kv, new)])  # positions follow the slots
        seq = torch.repeat_interleave(torch.arange(seqs), torch.tensor(new))
        pos = torch.zeros(rows, dtype=torch.int32)
        pos[:s["n"]] = (torch.arange(s["n"]) - torch.tensor(starts)[seq] + first[seq]).to(torch.int32)
        s.update(pos=pos.cuda())
    elif case["op"] == "evict":
        # few keys gather most of the weight and a window leaves some with none at all
        mass = torch.rand(seqs, kvh, width * ps, device="cuda", generator=g).pow(-1.5) - 1
        mass = mass * (torch.rand(seqs, kvh, width * ps, device="cuda", generator=g) > 0.05)
        s.update(mass=mass, new_table=order[seqs * width:seqs * (width + kept)].view(seqs, kept).cuda(),
                 keep=torch.empty(seqs, kvh, case["budget"], dtype=torch.int32, device="cuda"),
                 new_len=torch.empty(seqs, dtype=torch.int32, device="cuda"),
                 new_mass=torch.zeros(seqs, kvh, case["budget"], device="cuda"))
    else:
        s.update(q=normal(rows, h, hd, std=1.5), out=torch.zeros(rows, h, hd, dtype=dt, device="cuda"),
                 lse=torch.zeros(rows, h, device="cuda"))
        if case["op"] == "mass":
            _attend(s)
            s.update(mass=torch.rand(seqs, kvh, width * ps, device="cuda", generator=g) * 4,
                     new_mass=torch.zeros(seqs, kvh, width * ps, device="cuda"))
    if own:
        from jetsonfabric_b200 import paged
        s["cache"] = paged.PagedCache(k_pool, v_pool)
        s["batch"] = paged.PagedBatch(s["q_start"], s["kv_len"], table)
        if case["op"] == "rope":
            s["rope"] = paged.Rope(s["freq"], interleaved=case["interleaved"], factor=s["factor"])
        if case["op"] == "attend":
            s["workspace"] = paged.attention_workspace()
    return s


# ---- plain forms -----------------------------------------------------------------

def _rows(s):
    """Sequence and place in it of every row."""
    r = torch.arange(s["n"], device="cuda")
    seq = torch.searchsorted(s["q_start"].long(), r, right=True) - 1
    return seq, r - s["q_start"].long()[seq]


def _gathered(s, pool):
    """[sequences, kv_heads, keys, head_dim] in 32 bits."""
    x = pool[s["table"].long()]
    return x.flatten(1, 2)[:, :s["max_kv"]].transpose(1, 2).float()


def _scores(s):
    """[sequences, kv_heads, rows, group, keys]: scaled scores, the lowest where a key is masked, and the mask."""
    case = s["case"]
    seqs, kvh, group = case["seqs"], case["kv_heads"], case["heads"] // case["kv_heads"]
    seq, at = _rows(s)
    q = torch.zeros(seqs, s["max_q"], case["heads"], case["head_dim"], device="cuda")
    q[seq, at] = s["q"][:s["n"]].float()
    q = q.view(seqs, s["max_q"], kvh, group, -1).permute(0, 2, 1, 3, 4).flatten(2, 3)
    x = torch.matmul(q, _gathered(s, s["k_pool"]).transpose(2, 3)) * s["scale"]
    x = x.view(seqs, kvh, s["max_q"], group, s["max_kv"])
    count = (s["q_start"][1:] - s["q_start"][:-1])[:, None]
    pos = (s["kv_len"][:, None] - count + torch.arange(s["max_q"], device="cuda"))[:, None, :, None, None]
    key = torch.arange(s["max_kv"], device="cuda")
    seen = (key <= pos) & (torch.arange(s["max_q"], device="cuda") < count)[:, None, :, None, None]
    if case["window"]:
        seen = seen & (key > pos - case["window"])
    return x.masked_fill_(~seen, -math.inf), seen, seq, at


def _attend(s):
    case = s["case"]
    x, seen, seq, at = _scores(s)
    top = x.amax(-1, keepdim=True).clamp_min(-1e30)
    p = x.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    out = torch.matmul(p.flatten(2, 3), _gathered(s, s["v_pool"])).view(*p.shape[:-1], -1) / total.clamp_min(1e-30)
    out = out.permute(0, 2, 1, 3, 4).flatten(2, 3)
    lse = (top + total.log()).squeeze(-1).permute(0, 2, 1, 3).flatten(2, 3)
    s["out"][:s["n"]] = out[seq, at].to(s["out"].dtype)
    s["lse"][:s["n"]] = lse[seq, at]
    return {"out": s["out"], "lse": s["lse"]}


def _mass(s):
    case = s["case"]
    x, seen, seq, at = _scores(s)
    lse = torch.zeros(case["seqs"], s["max_q"], case["heads"], device="cuda")
    lse[seq, at] = s["lse"][:s["n"]]
    lse = lse.view(case["seqs"], s["max_q"], case["kv_heads"], -1).permute(0, 2, 1, 3)[..., None]
    added = x.sub_(lse).exp_().sum((2, 3))
    key = torch.arange(s["max_kv"], device="cuda")
    kv = s["kv_len"][:, None, None]
    old = kv - (s["q_start"][1:] - s["q_start"][:-1])[:, None, None]
    before = torch.where(key < old, s["mass"][..., :s["max_kv"]], 0.0)
    s["new_mass"][..., :s["max_kv"]] = torch.where(key < kv, before + added, s["new_mass"][..., :s["max_kv"]])
    return {"mass": s["new_mass"]}


def _slots(s, table, slot):
    """(page, place) of slots [sequences, ...] through a page table."""
    ps = s["case"]["page_size"]
    page = torch.gather(table.long(), 1, (slot // ps).flatten(1)).view_as(slot)
    return page, slot % ps


def _rope(s):
    case = s["case"]
    dims, n = case["rope_dims"], s["n"]
    angle = s["pos"][:n, None].double() * s["freq"]
    cos, sin = ((f(angle) * s["factor"]).float()[:, None] for f in (torch.cos, torch.sin))

    def turned(x):
        x = x[:n].float()
        part, rest = x[..., :dims], x[..., dims:]
        if case["interleaved"]:
            a, b = part[..., 0::2], part[..., 1::2]
            part = torch.stack((a * cos - b * sin, a * sin + b * cos), -1).flatten(-2)
        else:
            a, b = part[..., :dims // 2], part[..., dims // 2:]
            part = torch.cat((a * cos - b * sin, a * sin + b * cos), -1)
        return torch.cat((part, rest), -1)

    s["q_out"][:n] = turned(s["q"]).to(s["q_out"].dtype)
    seq, at = _rows(s)
    slot = (s["kv_len"] - (s["q_start"][1:] - s["q_start"][:-1])).long()[seq] + at
    page, place = s["table"].long()[seq, slot // case["page_size"]], slot % case["page_size"]
    s["k_pool"][page, place] = turned(s["k"]).to(s["k_pool"].dtype)
    s["v_pool"][page, place] = s["v"][:n].to(s["v_pool"].dtype)
    return {"q": s["q_out"], "k": s["k_pool"], "v": s["v_pool"]}


def _evict(s):
    case = s["case"]
    budget, recent, kvh = case["budget"], case["recent"], case["kv_heads"]
    mass = s["mass"][..., :s["max_kv"]]
    key = torch.arange(s["max_kv"], device="cuda")
    kv = s["kv_len"][:, None, None]
    rank = torch.where(key >= kv - recent, math.inf, mass)
    rank = torch.where(key < kv, rank, -math.inf)
    best = torch.sort(rank, dim=-1, descending=True, stable=True).indices[..., :budget]
    room = budget - best.shape[-1]
    valid = torch.arange(best.shape[-1], device="cuda") < kv
    best = torch.sort(torch.where(valid, best, s["max_kv"]), dim=-1).values
    keep = torch.where(valid, best, -1)
    s["keep"].copy_(torch.cat((keep, keep.new_full((*keep.shape[:-1], room), -1)), -1))
    s["new_len"].copy_(s["kv_len"].clamp_max(budget))
    source = torch.where(valid, best, 0)
    seq, head, i = torch.nonzero(valid.expand_as(best), as_tuple=True)
    page, place = _slots(s, s["table"], source)
    page, place = page[seq, head, i], place[seq, head, i]
    to_page, to_place = s["new_table"].long()[seq, i // case["page_size"]], i % case["page_size"]
    for_k, for_v = s["k_pool"][page, place, head], s["v_pool"][page, place, head]
    s["k_pool"][to_page, to_place, head] = for_k
    s["v_pool"][to_page, to_place, head] = for_v
    s["new_mass"][seq, head, i] = mass[seq, head, source[seq, head, i]]
    return {"keep": s["keep"], "kv_len": s["new_len"], "k": s["k_pool"], "v": s["v_pool"], "mass": s["new_mass"]}


def run(state):
    s, op = state, state["case"]["op"]
    if own:
        from jetsonfabric_b200 import paged
        if op == "rope":
            paged.rope_append(s["q"], s["k"], s["v"], s["pos"], s["rope"], s["cache"], s["batch"], s["q_out"])
            return {"q": s["q_out"], "k": s["k_pool"], "v": s["v_pool"]}
        if op == "attend":
            paged.attention(s["q"], s["cache"], s["batch"], s["out"], s["workspace"], scale=s["scale"],
                            window=s["case"]["window"], lse=s["lse"])
            return {"out": s["out"], "lse": s["lse"]}
        if op == "mass":
            paged.attention_mass(s["q"], s["lse"], s["cache"], s["batch"], s["new_mass"], mass_in=s["mass"],
                                 scale=s["scale"], window=s["case"]["window"])
            return {"mass": s["new_mass"]}
        paged.evict(s["mass"], s["cache"], s["batch"], s["keep"], s["new_len"], recent=s["case"]["recent"],
                    mass_out=s["new_mass"], page_table_out=s["new_table"])
        return {"keep": s["keep"], "kv_len": s["new_len"], "k": s["k_pool"], "v": s["v_pool"], "mass": s["new_mass"]}
    return {"rope": _rope, "attend": _attend, "mass": _mass, "evict": _evict}[op](s)


# ---- the definitions in 64 bits, sequence by sequence -----------------------------

def exact(case, seed):
    s = prepare(case, seed)
    new, kv = _lengths(case)
    ps, kvh, hd = case["page_size"], case["kv_heads"], case["head_dim"]
    table = s["table"].tolist()

    def flat(pool, b):
        return torch.cat([pool[p] for p in table[b]])[:kv[b]].double()

    def evicted():
        budget, ps = case["budget"], case["page_size"]
        keep = torch.full((case["seqs"], case["kv_heads"], budget), -1, dtype=torch.int32)
        new_len = torch.tensor([min(n, budget) for n in kv], dtype=torch.int32)
        k_pool, v_pool, mass = s["k_pool"].double(), s["v_pool"].double(), s["new_mass"].double()
        weights = s["mass"].cpu().numpy()
        for b, n in enumerate(kv):
            k_old, v_old = flat(s["k_pool"], b), flat(s["v_pool"], b)
            m = min(n, budget)
            to = torch.arange(m, device="cuda")
            page = s["new_table"][b].long()[to // ps]
            for head in range(case["kv_heads"]):
                w = weights[b, head, :n].tolist()
                late = range(max(0, n - case["recent"]), n) if n > budget else range(n)
                early = sorted(range(n - len(late)), key=lambda j: (-w[j], j))[:m - len(late)]
                chosen = torch.tensor(sorted([*early, *late]), dtype=torch.long)
                keep[b, head, :m] = chosen.to(torch.int32)
                at = chosen.cuda()
                k_pool[page, to % ps, head] = k_old[at, head]
                v_pool[page, to % ps, head] = v_old[at, head]
                mass[b, head, :m] = s["mass"][b, head, at].double()
        return {"keep": keep.cuda(), "kv_len": new_len.cuda(), "k": k_pool, "v": v_pool, "mass": mass}

    if case["op"] == "evict":
        return evicted()
    starts = s["q_start"].tolist()
    if case["op"] == "rope":
        q_out, k_pool, v_pool = s["q_out"].double(), s["k_pool"].double(), s["v_pool"].double()
        dims = case["rope_dims"]
        half = dims // 2
        pairs = [(2 * i, 2 * i + 1) if case["interleaved"] else (i, i + half) for i in range(half)]
        lo, hi = (torch.tensor(p, device="cuda") for p in zip(*pairs))
        for b in range(case["seqs"]):
            r = slice(starts[b], starts[b + 1])
            turn = torch.polar(torch.full_like(s["freq"], s["factor"]), torch.zeros_like(s["freq"]))
            turn = turn * torch.exp(1j * s["pos"][r, None, None].double() * s["freq"])
            done = {}
            for name in ("q", "k"):
                x = s[name][r].double().clone()
                z = torch.complex(x[..., lo], x[..., hi]) * turn
                x[..., lo], x[..., hi] = z.real, z.imag
                done[name] = x
            q_out[r] = done["q"]
            slots = torch.arange(kv[b] - new[b], kv[b], device="cuda")
            page = s["table"][b].long()[slots // ps]
            k_pool[page, slots % ps] = done["k"]
            v_pool[page, slots % ps] = s["v"][r].double()
        return {"q": q_out, "k": k_pool, "v": v_pool}
    group = case["heads"] // kvh
    if case["op"] == "attend":
        out, lse = s["out"].double(), s["lse"].double()
    else:
        mass = s["new_mass"].double()
    for b in range(case["seqs"]):
        r = slice(starts[b], starts[b + 1])
        keys = flat(s["k_pool"], b)
        values = flat(s["v_pool"], b) if case["op"] == "attend" else None
        distance = torch.arange(kv[b] - new[b], kv[b], device="cuda")[:, None] - torch.arange(kv[b], device="cuda")
        hidden = distance < 0
        if case["window"]:
            hidden |= distance >= case["window"]
        if case["op"] == "mass":
            mass[b, :, :kv[b] - new[b]] = s["mass"][b, :, :kv[b] - new[b]].double()
            mass[b, :, kv[b] - new[b]:kv[b]] = 0
        for head in range(case["heads"]):
            x = s["q"][r, head].double() @ keys[:, head // group].T * s["scale"]
            x[hidden] = -math.inf
            if case["op"] == "attend":
                lse[r, head] = torch.logsumexp(x, -1)
                out[r, head] = torch.softmax(x, -1) @ values[:, head // group]
            else:
                mass[b, head // group, :kv[b]] += torch.exp(x - s["lse"][r, head, None].double()).sum(0)
    return {"out": out, "lse": lse} if case["op"] == "attend" else {"mass": mass}
