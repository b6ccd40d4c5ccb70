"""Performance cases of the paged cache: what a serving program calls while the keys and values of its
requests are still uncompressed.

A step starts with the requests' lengths: the block tables grow by the pages the new tokens need and
every new token gets its slot (``build_block_tables``).  In every layer the queries and keys are rotated
by their positions (one axis for text, several for images and video; ``rope_axes``), the keys and values
are written to their pages (``append_kv`` does both), and the chunk of new tokens attends over the pages
of its request (``paged_attention``), over all of them or over a sliding window and the first few.

Shapes are those of the repository's configurations: 8 KV heads (fewer on a rank of a sharded model, other
numbers for the odd case) with 4 or 8 query heads each, head_dim 128, contexts up to 131072.  The lengths of a
case's requests follow from its fields (``shape`` seeds them); which pages a request owns, and all values,
come from the seed.

``run`` has each operator twice: as the framework's call (``own``) and in its plain form, elementary torch
operations in 32 bits (the angles of the rotation in 64) rounded once at the end.
"""
import math
import random

import torch

own = False

D = 128
DEV = "cuda"
DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
MOST_SCORES = 1 << 30     # scores of a drawn attention case: sequences x longest chunk x longest context x query heads


# ── the cases ────────────────────────────────────────────────────────────────

def listed():
    return [
        # Block tables of a decode step of 16 requests: the smallest call, once per token.
        dict(name="tables_step_16", op="tables", requests=16, new=1, ctx=8192, page=16, pad=0, short=False, shape=1),
        # Block tables of a full batch: chunked prefills between decoding requests, a padded batch.
        dict(name="tables_mixed_512", op="tables", requests=512, new=257, ctx=32768, page=64, pad=37, short=False, shape=2),
        # Rotation of a few speculated tokens of one request.
        dict(name="rope_5", op="rope", tokens=5, heads=8, gqa=4, axes=1, far=131072, dtype="fp16", shape=3),
        # Rotation of a prompt with images: three axes (time, height, width).
        dict(name="rope_axes_6k", op="rope", tokens=6007, heads=8, gqa=4, axes=3, far=4096, dtype="bf16", shape=4),
        # Rotation and cache write of a decode step of 32 requests.
        dict(name="append_32", op="append", tokens=32, heads=8, gqa=4, axes=1, far=32768, page=64, pad=3, dtype="bf16", shape=5),
        # Rotation and cache write of a chunk of 8192 prompt tokens with images.
        dict(name="append_axes_8k", op="append", tokens=8192, heads=8, gqa=8, axes=3, far=8192, page=16, pad=0, dtype="bf16", shape=6),
        # One token of one request: latency is all there is.
        dict(name="attn_1x1061", op="attn", requests=1, new=1, ctx=1060, heads=8, gqa=4, page=64, window=0, sinks=0,
             holes=False, dtype="fp16", shape=7),
        # A decode step of 64 requests of different lengths.
        dict(name="attn_decode_64", op="attn", requests=64, new=1, ctx=8192, heads=8, gqa=4, page=16, window=0, sinks=0,
             holes=False, dtype="bf16", shape=8),
        # A chunk of 2048 prompt tokens behind a long context.
        dict(name="attn_2k_at_30k", op="attn", requests=1, new=2048, ctx=30000, heads=8, gqa=4, page=64, window=0, sinks=0,
             holes=False, dtype="bf16", shape=9),
        # Chunks of up to 509 tokens of seven requests.
        dict(name="attn_7_chunks", op="attn", requests=7, new=509, ctx=6000, heads=8, gqa=8, page=32, window=0, sinks=0,
             holes=False, dtype="fp16", shape=10),
        # A chunk under a sliding window with four sink tokens.
        dict(name="window_4k", op="attn", requests=1, new=4000, ctx=8000, heads=8, gqa=4, page=16, window=1024, sinks=4,
             holes=False, dtype="bf16", shape=11),
        # A decode step of 24 long requests under a sliding window with 64 sink tokens.
        dict(name="window_decode_24", op="attn", requests=24, new=1, ctx=32768, heads=8, gqa=4, page=64, window=4096, sinks=64,
             holes=False, dtype="bf16", shape=12),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["tables", "rope", "append", "attn", "attn", "attn", "window", "window"])
    shape = rng.randrange(1 << 20)
    page = rng.choice([16, 32, 64, 128])
    if op == "tables":
        requests = _log_int(rng, 1, 2048)
        return dict(op=op, requests=requests, new=rng.choice([1, _log_int(rng, 2, max(3, 65536 // requests))]), ctx=_log_int(rng, 64, 131072),
                    page=page, pad=rng.choice([0, rng.randint(1, 300)]), short=rng.random() < 0.15, shape=shape)
    heads, gqa = rng.choice([8, 8, 4, 2, 1, 3]), rng.choice([4, 4, 8, 8, 1, 2, 5, 7, 16])
    dtype = rng.choice(["fp16", "bf16"])
    if op in ("rope", "append"):
        case = dict(op=op, tokens=_log_int(rng, 1, 8192), heads=heads, gqa=gqa, axes=rng.choice([1, 1, 2, 3, 3, 4]), far=_log_int(rng, 1024, 1 << 20),
                    dtype=rng.choice([dtype, dtype, "fp32"]) if op == "rope" else dtype, shape=shape)
        if op == "append":
            case.update(page=page, pad=rng.choice([0, rng.randint(0, case["tokens"] - 1)]))
        return case
    H_q = heads * gqa
    new = rng.choice([1, 1, rng.randint(2, 8), _log_int(rng, 9, 2048)])
    ctx = _log_int(rng, 1, 65536)
    new = max(1, min(new, MOST_SCORES // (H_q * (ctx + new))))
    most = MOST_SCORES // (H_q * new * (ctx + new))
    pages = (1 << 21) // (heads * (ctx + new))              # (a few GB of keys and values at most)
    requests = _log_int(rng, 1, max(1, min(most, pages, 256)))
    return dict(op="attn", requests=requests, new=new, ctx=ctx, heads=heads, gqa=gqa, page=page,
                window=_log_int(rng, 1, 8192) if op == "window" else 0, sinks=rng.choice([0, 1, 4, 64, 200]) if op == "window" else 0,
                holes=rng.random() < 0.15, dtype=dtype, shape=shape)


# ── inputs ───────────────────────────────────────────────────────────────────

def _lengths(case):
    """(tokens in the cache, new tokens) per request.  A request that decodes has one new token; chunks differ,
    and the first request has the longest chunk behind the longest context."""
    rng = random.Random(case["shape"])
    n, ctx, new = case["requests"], case["ctx"], case["new"]
    old = [ctx] + [rng.choice([rng.randint(0, ctx), rng.randint(ctx // 2, ctx)]) for _ in range(n - 1)]
    fresh = [new] + [rng.choice([1, rng.randint(0, new), rng.randint(1, new)]) for _ in range(n - 1)]
    return old, fresh


def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def _positions(case, gen):
    """[axes, tokens] int32.  Text has one position; an image's tokens share a time and count their rows and
    columns from it."""
    rng = random.Random(case["shape"])
    tokens, axes = case["tokens"], case["axes"]
    start = rng.randint(0, max(0, case["far"] - tokens))
    t = torch.arange(tokens, device=DEV)
    if axes == 1:
        return (start + t).to(torch.int32)[None]
    width = rng.randint(5, 40)
    rows = [start + t // (width * width), start + t // width % width, start + t % width, start + t // 7]
    at = torch.stack(rows[:axes])
    text = (t // 100) % 2 == 0                              # runs of text between the images
    at = torch.where(text[None], (start + t)[None], at)
    return (at + torch.randint(0, 2, at.shape, generator=gen, device=DEV)).to(torch.int32)


def _sections(case):
    """How many of the 64 rotation frequencies each axis owns."""
    rng = random.Random(case["shape"] + 1)
    axes = case["axes"]
    cuts = [0] + sorted(rng.sample(range(4, 61), axes - 1)) + [64]
    return [b - a for a, b in zip(cuts, cuts[1:])]


def _pages(n, heads, page, dtype, gen):
    return tuple(torch.randn(n, heads, page, D, generator=gen, device=DEV, dtype=torch.float32).to(dtype) for _ in range(2))


def prepare(case, seed):
    op, gen = case["op"], _gen(seed)
    s = dict(op=op)
    if op == "tables":
        old, fresh = _lengths(case)
        page = case["page"]
        held = [-(-c // page) for c in old]
        need = [-(-(c + n) // page) - h for c, n, h in zip(old, fresh, held)]
        width = max(h + n for h, n in zip(held, need)) + 2
        total = sum(held) + sum(need)
        order = torch.randperm(total + 8, generator=gen, device=DEV).to(torch.int32)
        edge = torch.cumsum(_ints([0] + held), 0)
        e = torch.arange(width, device=DEV)
        mine = e[None] < _ints(held)[:, None]
        s["tables"] = torch.where(mine, order[(edge[:-1, None] + e[None]).clamp(max=total)], -1).to(torch.int32)
        s["free"] = order[sum(held):].contiguous()
        if case["short"]:                                   # fewer free pages than the step needs
            s["free"] = s["free"][: max(1, sum(need) // 2)].contiguous()
        s.update(ctx=_ints(old), new=_ints(fresh), page=page, n_tokens=sum(fresh) + case["pad"], start=_ints([0]))
        return s
    heads, gqa, dtype = case["heads"], case["gqa"], DTYPES[case["dtype"]]
    if op in ("rope", "append"):
        T = case["tokens"]
        s["q"], s["k"], s["v"] = (torch.randn(T, h, D, generator=gen, device=DEV).to(dtype) for h in (heads * gqa, heads, heads))
        s["positions"] = _positions(case, gen)
        s["sections"] = _sections(case)
        s["inv_freq"] = (5e5 ** (-torch.arange(D // 2, device=DEV, dtype=torch.float64) / (D // 2))).float()
        if op == "append":
            page, live = case["page"], T - case["pad"]
            n = -(-live // page) + 3
            s["k_pages"], s["v_pages"] = _pages(n, heads, page, dtype, gen)
            order = torch.randperm(n, generator=gen, device=DEV)
            t = torch.arange(T, device=DEV)
            s["slots"] = torch.where(t < live, order[(t // page).clamp(max=n - 1)] * page + t % page, -1)
        return s
    old, fresh = _lengths(case)
    page, n = case["page"], case["requests"]
    lens = [c + f for c, f in zip(old, fresh)]
    blocks = [-(-x // page) for x in lens]
    width, total = max(blocks) + 1, sum(blocks)
    s["k_pages"], s["v_pages"] = _pages(total + 1, heads, page, dtype, gen)
    order = torch.randperm(total + 1, generator=gen, device=DEV).to(torch.int32)
    edge = torch.cumsum(_ints([0] + blocks), 0)
    e = torch.arange(width, device=DEV)
    table = torch.where(e[None] < _ints(blocks)[:, None], order[(edge[:-1, None] + e[None]).clamp(max=total)], -1).to(torch.int32)
    if case["holes"]:                                       # pages that were dropped from the middle of a cache
        table = torch.where(torch.rand(table.shape, generator=gen, device=DEV) < 0.2, -1, table)
    T = sum(fresh)
    s.update(tables=table, q=(torch.randn(T, heads * gqa, D, generator=gen, device=DEV) * 1.5).to(dtype),
             q_start=torch.cat([_ints([0]), torch.cumsum(_ints(fresh), 0).to(torch.int32)]), lens=_ints(lens), max_new=max(fresh),
             window=case["window"], sinks=case["sinks"], scale=D ** -0.5)
    return s


# ── the operators ────────────────────────────────────────────────────────────

def _tables(s):
    if own:
        from rdkv_b200.paged import build_block_tables
        p = build_block_tables(s["ctx"], s["new"], s["tables"], s["free"], s["page"], s["n_tokens"], free_start=s["start"])
        return dict(tables=s["tables"], slot_map=p.slot_map, positions=p.positions, q_start=p.q_start, kv_lens=p.kv_lens,
                    free_next=p.free_next, missing=p.missing)
    ctx, new, table, free, page, T = s["ctx"].long(), s["new"].long(), s["tables"], s["free"], s["page"], s["n_tokens"]
    width, F = table.shape[1], free.shape[0]
    held = (ctx + page - 1) // page
    full = (ctx + new + page - 1) // page
    need = (full.clamp(max=width) - held).clamp(min=0)
    end = torch.cumsum(need, 0) + s["start"].long()
    base = end - need
    e = torch.arange(width, device=table.device)
    at = base[:, None] + e[None] - held[:, None]
    fresh = (e[None] >= held[:, None]) & (e[None] < (held + need)[:, None])
    got = torch.where(at < F, free[at.clamp(0, F - 1)], -1)
    table.copy_(torch.where(fresh, got, table))
    q_end = torch.cumsum(new, 0)
    t = torch.arange(T, device=table.device)
    i = torch.searchsorted(q_end, t, right=True)
    live = i < ctx.shape[0]
    i = i.clamp(max=ctx.shape[0] - 1)
    pos = ctx[i] + t - (q_end - new)[i]
    block = pos // page
    page_id = torch.where(block < width, table[i, block.clamp(max=width - 1)].long(), -1)
    lost = (full - torch.maximum(held, full.clamp(max=width))).clamp(min=0).sum() + (end[-1:] - F).clamp(min=0)
    return dict(tables=table, slot_map=torch.where(live & (page_id >= 0), page_id * page + pos % page, -1),
                positions=torch.where(live, pos, 0).int(), q_start=torch.cat([torch.zeros_like(q_end[:1]), q_end]).int(),
                kv_lens=(ctx + new).int(), free_next=end[-1:].clamp(max=F).int(), missing=lost.int())


def _rotated(x, positions, inv_freq, sections):
    axis = torch.repeat_interleave(torch.arange(len(sections), device=x.device), torch.tensor(sections, device=x.device), output_size=64)
    angle = positions.double()[axis].t() * inv_freq.double()[None]        # [tokens, 64]
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]
    a, b = x.float().split(D // 2, dim=2)
    return torch.cat([a * cos - b * sin, b * cos + a * sin], dim=2).to(x.dtype)


def _rope(s):
    if own:
        from rdkv_b200.rope import rope_axes
        q, k = rope_axes(s["q"], s["k"], s["positions"], s["inv_freq"], sections=s["sections"])
        return dict(q=q, k=k)
    return dict(q=_rotated(s["q"], s["positions"], s["inv_freq"], s["sections"]),
                k=_rotated(s["k"], s["positions"], s["inv_freq"], s["sections"]))


def _append(s):
    if own:
        from rdkv_b200.paged import append_kv
        q = append_kv(s["k"], s["v"], s["k_pages"], s["v_pages"], s["slots"], q=s["q"], positions=s["positions"], inv_freq=s["inv_freq"],
                      sections=s["sections"])
        return dict(q=q, k_pages=s["k_pages"], v_pages=s["v_pages"])
    page = s["k_pages"].shape[2]
    q = _rotated(s["q"], s["positions"], s["inv_freq"], s["sections"])
    k = _rotated(s["k"], s["positions"], s["inv_freq"], s["sections"])
    live = s["slots"] >= 0
    t = torch.where(live, torch.arange(live.shape[0], device=live.device), live.int().argmax())   # (padding: the first live token again)
    slot = s["slots"][t]
    s["k_pages"][slot // page, :, slot % page] = k[t]
    s["v_pages"][slot // page, :, slot % page] = s["v"][t]
    return dict(q=q, k_pages=s["k_pages"], v_pages=s["v_pages"])


def _attention(s):
    q, tables, q_start, lens = s["q"], s["tables"], s["q_start"], s["lens"]
    if own:
        from rdkv_b200.paged import paged_attention
        return dict(out=paged_attention(q, s["k_pages"], s["v_pages"], tables, q_start, lens, max_new=s["max_new"], window=s["window"],
                                        sinks=s["sinks"], scale=s["scale"]))
    n, width = tables.shape
    heads, page = s["k_pages"].shape[1:3]
    T, H_q, L = q.shape[0], q.shape[1], width * page
    gqa, longest = H_q // heads, s["max_new"]
    at = tables.long().clamp(min=0)
    keys, values = (p[at].float().permute(0, 2, 1, 3, 4).reshape(n, heads, 1, L, D) for p in (s["k_pages"], s["v_pages"]))
    new = (q_start[1:] - q_start[:-1]).long()
    j = torch.arange(longest, device=q.device)
    rows = (q_start[:-1].long()[:, None] + j[None]).clamp(max=T - 1)
    queries = q[rows].float().reshape(n, longest, heads, gqa, D).permute(0, 2, 3, 1, 4)
    scores = torch.matmul(queries, keys.transpose(3, 4)).mul_(s["scale"])
    pos = ((lens.long() - new)[:, None] + j[None])[:, :, None]             # [n, longest, 1]
    key = torch.arange(L, device=q.device)[None, None]
    seen = (key <= pos) & (key < lens.long()[:, None, None])
    if s["window"] > 0:
        seen &= (key > pos - s["window"]) | (key < s["sinks"])
    seen &= (tables >= 0).repeat_interleave(page, dim=1)[:, None]
    scores.masked_fill_(~seen[:, None, None], -math.inf)
    top = scores.amax(dim=4, keepdim=True)
    weights = scores.sub_(torch.where(top == -math.inf, 0.0, top)).exp_()
    total = weights.sum(dim=4, keepdim=True)
    out = torch.matmul(weights, values) / torch.where(total == 0, 1.0, total)
    t = torch.arange(T, device=q.device)
    i = torch.searchsorted(q_start[1:].long(), t, right=True).clamp(max=n - 1)
    return dict(out=out[i, :, :, (t - q_start.long()[i]).clamp(max=longest - 1)].reshape(T, H_q, D).to(q.dtype))


def run(state):
    return {"tables": _tables, "rope": _rope, "append": _append, "attn": _attention}[state["op"]](state)


def work(case):
    op = case["op"]
    if op == "tables":
        old, fresh = _lengths(case)
        pages = sum(-(-(c + f) // case["page"]) - -(-c // case["page"]) for c, f in zip(old, fresh))
        tokens = sum(fresh) + case["pad"]
        return {"bytes": 16 * case["requests"] + 8 * pages + 12 * tokens, "flops": tokens}
    heads, gqa, size = case["heads"], case["gqa"], 4 if case["dtype"] == "fp32" else 2
    if op in ("rope", "append"):
        T = case["tokens"]
        q, k = T * heads * gqa * D * size, T * heads * D * size
        moved = 2 * (q + k) if op == "rope" else 2 * q + 4 * (T - case["pad"]) * heads * D * size + 8 * T
        return {"bytes": moved + 4 * T * case["axes"], "flops": 3 * T * heads * (gqa + 1) * D}
    old, fresh = _lengths(case)
    window, sinks = case["window"], case["sinks"]
    keys = pairs = 0
    for c, f in zip(old, fresh):
        if f == 0:
            continue
        lo = max(0, c - window + 1) if window > 0 else 0                   # the first key of the first token's window
        keys += c + f - lo + min(sinks if window > 0 else 0, lo)
        if window > 0:
            for p in range(c, c + f):
                first = max(0, p - window + 1)
                pairs += p + 1 - first + min(sinks, first)
        else:
            pairs += f * c + f * (f + 1) // 2
    kept = 0.8 if case["holes"] else 1.0
    return {"bytes": int(4 * kept * keys * heads * D) + 4 * sum(fresh) * heads * gqa * D, "flops": int(4 * kept * pairs * heads * gqa * D)}


# ── the definitions in 64 bits ───────────────────────────────────────────────

def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "tables":
        return None                                         # whole numbers
    if op in ("rope", "append"):
        turn = torch.empty(case["tokens"], 64, dtype=torch.float64, device=DEV)
        first = 0
        for axis, n in enumerate(s["sections"]):
            turn[:, first:first + n] = s["positions"][axis].double()[:, None] * s["inv_freq"][first:first + n].double()
            first += n
        unit = torch.polar(torch.ones_like(turn), turn)[:, None]
        both = {}
        for name in ("q", "k"):
            x = s[name].double()
            z = torch.complex(x[..., :64].contiguous(), x[..., 64:].contiguous()) * unit
            both[name] = torch.cat([z.real, z.imag], dim=2)
        if op == "rope":
            return both
        pages = {"k_pages": s["k_pages"].double(), "v_pages": s["v_pages"].double()}
        page = case["page"]
        slots = s["slots"][: case["tokens"] - case["pad"]]
        for name, rows in (("k_pages", both["k"]), ("v_pages", s["v"].double())):
            pages[name][slots // page, :, slots % page] = rows[: slots.shape[0]]
        return dict(q=both["q"], **pages)
    old, fresh = _lengths(case)
    heads, gqa, page = case["heads"], case["gqa"], case["page"]
    out = torch.zeros(sum(fresh), heads * gqa, D, dtype=torch.float64, device=DEV)
    row = 0
    for i, (c, f) in enumerate(zip(old, fresh)):
        if f == 0:
            continue
        L = c + f
        ids = s["tables"][i, : -(-L // page)].long()
        there = (ids >= 0).repeat_interleave(page)[:L]
        kept = torch.arange(L, device=DEV)[there]
        pos = torch.arange(c, L, device=DEV)[:, None]
        hidden = kept[None] > pos
        if case["window"] > 0:
            hidden |= (kept[None] <= pos - case["window"]) & (kept[None] >= case["sinks"])
        nothing = hidden.all(dim=1)
        for h in range(heads):
            k, v = (p[ids.clamp(min=0), h].reshape(-1, D)[:L][there].double() for p in (s["k_pages"], s["v_pages"]))
            for g in range(gqa):
                a = s["q"][row:row + f, h * gqa + g].double() @ k.t() * s["scale"]
                a.masked_fill_(hidden, -math.inf)
                w = torch.softmax(a, dim=1)
                w[nothing] = 0
                out[row:row + f, h * gqa + g] = w @ v
        row += f
    return dict(out=out)
