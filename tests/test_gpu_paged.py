"""The paged cache's operators on the GPU against their definitions in 64 bits."""
import random

import pytest
import torch

import paged_reference as R

pytestmark = pytest.mark.gpu

F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def starts(new):
    return ints([sum(new[:i]) for i in range(len(new) + 1)])


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def randn(*shape, seed, dtype):
    return torch.randn(*shape, generator=gen(seed), device="cuda").to(dtype)


# ── block tables ─────────────────────────────────────────────────────────────

@pytest.mark.parametrize("requests,page,ctx_most,new_most,pad,short,narrow", [
    (0, 16, 0, 0, 5, False, False), (1, 16, 0, 1, 0, False, False), (1, 64, 63, 1, 3, False, False), (7, 16, 40, 40, 0, False, False),
    (7, 16, 40, 40, 9, True, False), (33, 32, 500, 3, 1, False, True), (513, 128, 1000, 9, 70, True, True), (3000, 16, 300, 4, 0, False, False),
    (5, 48, 1000, 2000, 0, False, False), (16384, 16, 64, 2, 10, False, False)])
def test_block_tables(requests, page, ctx_most, new_most, pad, short, narrow):
    from rdkv_b200.paged import build_block_tables
    rng = random.Random(requests * page + pad)
    ctx = [rng.choice([0, rng.randint(-3, ctx_most), ctx_most]) for _ in range(requests)]
    new = [rng.choice([0, 1, rng.randint(-2, new_most), new_most]) for _ in range(requests)]
    pages = [-(-(max(c, 0) + max(n, 0)) // page) for c, n in zip(ctx, new)]
    held = [-(-max(c, 0) // page) for c in ctx]
    width = max([2] + pages) - (1 if narrow else -1)
    table = [[rng.choice([-1, rng.randint(0, 10 ** 6)]) if e < h else -7 for e in range(width)] for h in held]
    need = sum(p - h for p, h in zip(pages, held))
    free = rng.sample(range(10 ** 6), max(0, need // 2 if short else need + 3))
    total = sum(max(n, 0) for n in new)
    start = rng.choice([0, 2])
    want = R.tables(ctx, new, table, free, page, total + pad, start)
    wide = torch.full((max(requests, 1), width + 5), -9, dtype=torch.int32, device="cuda")     # (rows of a wider tensor)
    dev = wide[:requests, :width]
    if requests:
        dev.copy_(ints(table))
    plan = build_block_tables(ints(ctx), ints(new), dev, ints(free), page, total + pad, free_start=ints([start]) if start else None)
    assert dev.tolist() == want["tables"] and (wide[:, width:] == -9).all()
    for name in ("slot_map", "positions", "q_start", "kv_lens", "free_next", "missing"):
        assert getattr(plan, name).tolist() == want[name], name
    # the same step again into the same plan: nothing it wrote is read as something else
    again = build_block_tables(ints(ctx), ints(new), dev, ints(free), page, total + pad, free_start=ints([start]), out=plan)
    assert again is plan and dev.tolist() == want["tables"] and plan.slot_map.tolist() == want["slot_map"]


def test_block_tables_fewer_token_places_than_tokens():
    from rdkv_b200.paged import build_block_tables
    table = torch.full((2, 4), -1, dtype=torch.int32, device="cuda")
    plan = build_block_tables(ints([0, 0]), ints([20, 30]), table, ints([5, 6, 7, 8]), 16, 25)
    assert plan.slot_map.tolist() == [5 * 16 + p for p in range(16)] + [6 * 16 + p for p in range(4)] + [7 * 16 + p for p in range(5)]
    assert plan.q_start.tolist() == [0, 20, 50] and plan.free_next.tolist() == [4] and plan.missing.tolist() == [0]


def test_block_tables_lengths_at_the_end_of_32_bits():
    """Lengths whose sums pass 32 bits neither wrap into the table nor into the slots."""
    from rdkv_b200.paged import build_block_tables
    big = 2 ** 31 - 1
    table = torch.full((2, 3), 4, dtype=torch.int32, device="cuda")
    plan = build_block_tables(ints([big, 0]), ints([big, 1]), table, ints([9]), 16, 4)
    assert (plan.slot_map == -1).all() and plan.kv_lens.tolist() == [big, 1] and plan.q_start.tolist() == [0, big, big]
    assert table.tolist() == [[4, 4, 4], [9, 4, 4]]


# ── rotation and cache write ─────────────────────────────────────────────────

def near(got, want, src, dtype, what=""):
    """A rotated value: rounded once (u of its size), sine and cosine within 2^-21."""
    other = torch.cat([src[..., 64:], src[..., :64]], dim=-1).double().abs() + src.double().abs()
    tol = (torch.finfo(dtype).eps / 2) * want.abs() * (1 + 2.0 ** -10) + 2.0 ** -20 * other + 2.0 ** -25
    bad = (got.double() - want).abs() > tol
    assert not bad.any(), f"{what}: {int(bad.sum())} values off, worst {float(((got.double() - want).abs() - tol).max()):.3g}"


INV = lambda: (5e5 ** (-torch.arange(64, device="cuda", dtype=torch.float64) / 64)).float()


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("T,H_q,H_kv,sections,pos64", [
    (1, 32, 8, (64,), False), (5, 7, 1, (16, 24, 24), True), (130, 3, 3, (0, 64), False), (1000, 8, 2, (10, 20, 30, 4), True), (0, 4, 4, (64,), False)])
def test_rope_axes(dtype, T, H_q, H_kv, sections, pos64):
    from rdkv_b200.rope import rope_axes
    q, k = randn(T, H_q, 128, seed=1, dtype=dtype), randn(T, H_kv, 128, seed=2, dtype=dtype)
    pos = torch.randint(0, 2 ** 24, (len(sections), T), generator=gen(3), device="cuda", dtype=torch.int64 if pos64 else torch.int32)
    pos[:, ::3] %= 100
    kept = q.clone(), k.clone()
    q2, k2 = rope_axes(q, k, pos if len(sections) > 1 else pos[0], INV(), sections=sections)
    assert torch.equal(q, kept[0]) and torch.equal(k, kept[1])
    for got, x, name in ((q2, q, "q"), (k2, k, "k")):
        near(got, R.rotate(x, pos, INV(), sections), x, dtype, name)
    # in place, and views of one fused projection (strided heads; a width that no 16-byte load fits)
    for extra in (8, 3):
        wide = torch.zeros(T, (H_q + H_kv), 128 + extra, dtype=dtype, device="cuda")
        wide[:, :H_q, :128], wide[:, H_q:, :128] = q, k
        a, b = wide[:, :H_q, :128], wide[:, H_q:, :128]
        rope_axes(a, b, pos, INV(), sections=sections, q_out=a, k_out=b)
        assert torch.equal(a, q2) and torch.equal(b, k2) and (wide[..., 128:] == 0).all()


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("layout", ["heads first", "rows first", "odd"])
@pytest.mark.parametrize("T,page", [(1, 16), (77, 16), (300, 48)])
def test_append(dtype, layout, T, page):
    from rdkv_b200.paged import append_kv
    from rdkv_b200.rope import rope_axes
    H_q, H_kv, n = 6, 3, T // page + 4
    sections = (20, 20, 24)
    q, k, v = (randn(T, h, 128, seed=s, dtype=dtype) for s, h in ((1, H_q), (2, H_kv), (3, H_kv)))
    pos = torch.randint(0, 5000, (3, T), generator=gen(4), device="cuda", dtype=torch.int32)

    def pages(seed):
        if layout == "heads first":
            return randn(n, H_kv, page, 128, seed=seed, dtype=dtype)
        if layout == "rows first":
            return randn(n, page, H_kv, 128, seed=seed, dtype=dtype).permute(0, 2, 1, 3)
        return randn(n, H_kv, page, 131, seed=seed, dtype=dtype)[..., :128]
    kp, vp = pages(5), pages(6)
    slots = torch.randperm(n * page, generator=gen(7), device="cuda")[:T]
    slots[T // 2] = -1
    if T > 10:
        slots[3], slots[4] = n * page, -(2 ** 40)
    want_k, want_v = kp.clone(), vp.clone()
    live = ((slots >= 0) & (slots < n * page)).nonzero()[:, 0]
    q_rot, k_rot = rope_axes(q, k, pos, INV(), sections=sections)
    for rotated in (True, False):
        want_k[slots[live] // page, :, slots[live] % page] = (k_rot if rotated else k)[live]
        want_v[slots[live] // page, :, slots[live] % page] = v[live]
        if rotated:
            assert torch.equal(append_kv(k, v, kp, vp, slots, q=q, positions=pos, inv_freq=INV(), sections=sections), q_rot)
        else:
            assert append_kv(k, v, kp, vp, slots) is None
        assert torch.equal(kp, want_k) and torch.equal(vp, want_v)      # what no slot names is left as it was
    q2 = q.clone()
    assert append_kv(k, v, kp, vp, slots, q=q2, positions=pos, inv_freq=INV(), sections=sections, q_out=q2) is q2 and torch.equal(q2, q_rot)


# ── attention ────────────────────────────────────────────────────────────────

def check(got, want, what=""):
    out, tol = want
    off = (got.double() - out).abs() - tol
    assert torch.isfinite(got).all(), f"{what}: not finite"
    assert not (off > 0).any(), f"{what}: {int((off > 0).sum())} values off, worst by {float(off.max()):.3g}"


def run(lens, new, H_kv, g, page, dtype, seed=0, window=0, sinks=0, pad=0, max_new="true", hole=0.0, **kw):
    from rdkv_b200.paged import paged_attention
    k, v, table = R.build_cache(lens, H_kv, page, dtype, seed=seed)
    if hole:
        table = torch.where(torch.rand(table.shape, generator=gen(seed + 5), device="cuda") < hole, 12345678, table)
    T = sum(new) + pad
    q = randn(T, H_kv * g, 128, seed=seed + 1, dtype=dtype) * 1.5
    most = max(new, default=0) if max_new == "true" else max_new
    got = paged_attention(q, k, v, table, starts(new), ints(lens), max_new=most, window=window, sinks=sinks, check_status=True, **kw)
    check(got, R.attention(q, k, v, table, starts(new), ints(lens), window, sinks, kw.get("scale")), f"{lens} {new}")
    return q, k, v, table, got


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("page", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("H_kv,g", [(2, 4), (1, 1), (1, 16), (3, 5)])
def test_decode(dtype, page, H_kv, g):
    """One new token a request, lengths around the edges of pages and tiles."""
    lens = [1, 2, 15, 16, 17, 63, 64, 65, 127, 128, 129, 200, 513, 1000]
    run(lens, [1] * len(lens), H_kv, g, page, dtype, seed=page + g)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("page", [16, 64, 128, 512])
@pytest.mark.parametrize("H_kv,g", [(2, 4), (1, 1), (1, 16), (2, 7), (1, 8)])
def test_chunks(dtype, page, H_kv, g):
    """Chunks of every kind in one batch: the whole prompt, behind a context, single tokens, none."""
    lens = [1, 130, 300, 129, 700, 40, 64, 257, 0, 5]
    new = [1, 130, 7, 128, 333, 0, 64, 1, 0, 2]
    run(lens, new, H_kv, g, page, dtype, seed=page + g, pad=3)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (16, 4), (100, 0), (128, 64), (500, 200), (10000, 5), (33, 10000), (2 ** 40, 2 ** 40)])
@pytest.mark.parametrize("g,page", [(4, 16), (3, 128)])
def test_window_and_sinks(dtype, window, sinks, g, page):
    lens = [1, 17, 900, 600, 1301, 300]
    run(lens, [1] * len(lens), 2, g, page, dtype, seed=window, window=window, sinks=sinks)
    run(lens, [1, 17, 250, 1, 130, 300], 2, g, page, dtype, seed=window + 1, window=window, sinks=sinks)


@pytest.mark.parametrize("new", [[1, 1, 1], [200, 1, 77]])
def test_rows_that_see_nothing(new):
    """Lengths of zero, more new tokens than the cache holds, and pages that are gone."""
    from rdkv_b200.paged import paged_attention
    k, v, table = R.build_cache([300, 300, 300], 2, 16, BF16, seed=3)
    table[2] = -1
    q = randn(sum(new), 8, 128, seed=4, dtype=BF16)
    lens = ints([0, 0 if new[0] == 1 else 1, 300])
    got = paged_attention(q, k, v, table, starts(new), lens, max_new=max(new))
    check(got, R.attention(q, k, v, table, starts(new), lens))
    assert (got[:new[0]] == 0).all() and (got[-new[2]:] == 0).all()
    lens = ints([min(n, 300) // 2 for n in new])                        # negative positions in front
    got = paged_attention(q, k, v, table, starts(new), lens, max_new=max(new))
    check(got, R.attention(q, k, v, table, starts(new), lens))


@pytest.mark.parametrize("new", [[1, 1, 1, 1], [150, 3, 1, 64]])
@pytest.mark.parametrize("window,sinks", [(0, 0), (90, 20)])
def test_missing_pages_are_not_seen(new, window, sinks):
    run([400, 333, 1000, 64], new, 2, 4, 16, F16, seed=8, window=window, sinks=sinks, hole=0.3)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("new", [[1, 1, 1], [150, 2, 64]])
@pytest.mark.parametrize("window,sinks", [(0, 0), (50, 10)])
def test_what_stands_in_masked_places_does_not_matter(dtype, new, window, sinks):
    """NaN and infinities behind a request's end, in pages that nobody owns and outside the window."""
    from rdkv_b200.paged import paged_attention
    lens = [300, 131, 64]
    k, v, table = R.build_cache(lens, 2, 32, dtype, seed=5)
    q = randn(sum(new), 8, 128, seed=6, dtype=dtype)
    args = (table, starts(new), ints(lens))
    want = R.attention(q, k, v, *args, window, sinks)
    clean = paged_attention(q, k, v, *args, max_new=max(new), window=window, sinks=sinks)
    check(clean, want)
    seen = torch.zeros(k.shape[0], 32, dtype=torch.bool, device="cuda")
    for i, (n, f) in enumerate(zip(lens, new)):
        for s in range(n):
            if window == 0 or s < sinks or s > n - f - window:
                seen[table[i, s // 32], s % 32] = True
    for bad in (float("nan"), float("inf"), -float("inf")):
        k2, v2 = (torch.where(seen[:, None, :, None], x, torch.tensor(bad, dtype=dtype, device="cuda")) for x in (k, v))
        got = paged_attention(q, k2, v2, *args, max_new=max(new), window=window, sinks=sinks)
        assert torch.equal(got, clean)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("g", [1, 4])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_a_bad_value_reaches_the_tokens_that_see_it_and_no_others(dtype, g, bad):
    """A value row that is not finite inside a chunk: tokens in front of it, whose mask it is behind, stay clean, and
    where it is in one channel the other channels do."""
    from rdkv_b200.paged import paged_attention
    lens, new = [700, 200], [500, 200]
    k, v, table = R.build_cache(lens, 1, 16, dtype, seed=15)
    q = randn(sum(new), g, 128, seed=16, dtype=dtype)
    args = (table, starts(new), ints(lens))
    clean = paged_attention(q, k, v, *args, max_new=500)
    at = 437                                                            # of request 0: its chunk starts at 200
    v[table[0, at // 16], 0, at % 16, 5] = bad
    got = paged_attention(q, k, v, *args, max_new=500)
    row = at - 200
    assert torch.equal(got[:row], clean[:row]) or (got[:row].float() - clean[:row].float()).abs().max() < 2 * torch.finfo(dtype).eps * 4
    assert not torch.isfinite(got[row:500, :, 5]).any()
    others = [c for c in range(128) if c != 5]
    want = R.attention(q, k, torch.nan_to_num(v, nan=0.0, posinf=0.0), *args)
    check(got[:, :, others], (want[0][:, :, others], want[1][:, :, others]))
    check(got[:row], (want[0][:row], want[1][:row]))
    check(got[500:], (want[0][500:], want[1][500:]))


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("new", [[1, 1], [3, 2], [300, 100]])
def test_a_bad_key_reaches_the_tokens_that_see_it_and_no_others(dtype, new):
    from rdkv_b200.paged import paged_attention
    lens = [400, 150]
    k, v, table = R.build_cache(lens, 2, 16, dtype, seed=18)
    q = randn(sum(new), 8, 128, seed=19, dtype=dtype)
    args = (table, starts(new), ints(lens))
    want = R.attention(q, k, v, *args)
    at = 398 if new[0] <= 3 else 250                                    # of request 0, in its KV head 1
    k[table[0, at // 16], 1, at % 16, 7] = float("nan")
    got = paged_attention(q, k, v, *args, max_new=max(new))
    first = max(0, at - (400 - new[0]))
    assert torch.isnan(got[first:new[0], 4:]).all()
    check(got[:, :4], (want[0][:, :4], want[1][:, :4]))
    check(got[:first], (want[0][:first], want[1][:first]))
    check(got[new[0]:], (want[0][new[0]:], want[1][new[0]:]))


@pytest.mark.parametrize("new", [[1, 1], [100, 3]])
def test_lengths_past_what_the_table_holds(new):
    """A length behind the table's last page, up to the end of 32 bits: the tokens there are, are seen."""
    from rdkv_b200.paged import paged_attention
    k, v, table = R.build_cache([320, 64], 2, 64, BF16, seed=28, width_extra=0)
    q = randn(sum(new), 4, 128, seed=29, dtype=BF16)
    for lens in ([5000, 300], [2 ** 31 - 1, 2 ** 31 - 1]):
        got = paged_attention(q, k, v, table, starts(new), ints(lens), max_new=max(new))
        check(got, R.attention(q, k, v, table, starts(new), ints([6000, 6000])))      # (every token is in front of the new ones)


@pytest.mark.parametrize("max_new", [None, 1, 3, 10 ** 6])
def test_max_new_is_only_a_hint(max_new):
    run([40, 300, 77], [9, 30, 1], 2, 4, 16, BF16, seed=2, max_new=max_new)
    run([40, 300, 77], [1, 1, 1], 2, 4, 16, BF16, seed=2, max_new=max_new)


def test_many_requests_and_few():
    rng = random.Random(4)
    lens = [rng.choice([1, rng.randint(1, 400)]) for _ in range(700)]
    run(lens, [1] * 700, 1, 4, 16, BF16, seed=21)
    new = [rng.choice([0, 1, 2, rng.randint(0, n)]) for n in lens]
    run(lens[:300], [min(a, b) for a, b in zip(new, lens)][:300], 1, 2, 16, F16, seed=22)
    run(lens, [min(a, b) for a, b in zip(new, lens)], 2, 8, 16, BF16, seed=26)
    run(lens[:18], [1] * 18, 1, 4, 16, F16, seed=27)                     # (clusters of 12 CTAs; of 8)
    run(lens[:31], [1] * 31, 1, 4, 16, F16, seed=28)
    run([5000], [1], 1, 8, 64, F16, seed=23)
    run([5000], [1], 8, 1, 64, BF16, seed=24, window=3000, sinks=4)
    run([3000], [700], 1, 4, 64, BF16, seed=25)


@pytest.mark.parametrize("sinks", [0, 1, 64, 65, 128, 129, 192, 193, 600])
@pytest.mark.parametrize("window", [1, 63, 64, 65, 300])
def test_windows_and_sinks_that_begin_and_end_in_either_half_of_a_tile(window, sinks):
    """Half tiles that none of an item's rows see are left out, and nothing else is."""
    for lead in (0, 31, 32, 63, 64, 65, 96, 127):
        run([700 + lead, 1500], [200 + lead, 130], 1, 4, 32, BF16, seed=80 + lead, window=window, sinks=sinks)


@pytest.mark.parametrize("every", [0, 1, 7, 25])
def test_chunks_that_see_nothing_one_after_another(every):
    """Runs of items without a tile, longer than what the warps of a CTA may be apart, between items with some."""
    from rdkv_b200.paged import paged_attention
    lens = [300 if every and i % every == 0 else 0 for i in range(50)]
    k, v, table = R.build_cache([300] * 50, 2, 32, BF16, seed=91)
    new = [(130, 64, 17, 200)[i % 4] for i in range(50)]
    q = randn(sum(new), 8, 128, seed=92, dtype=BF16)
    for kw in ({}, dict(window=40, sinks=3)):
        got = paged_attention(q, k, v, table, starts(new), ints(lens), max_new=200, check_status=True, **kw)
        check(got, R.attention(q, k, v, table, starts(new), ints(lens), **kw))
        rec = torch.full((q.shape[0] * 8, 132), 7.0, device="cuda")
        paged_attention(q, k, v, table, starts(new), ints(lens), max_new=200, out_partial=rec, check_status=True, **kw)
        assert torch.isfinite(rec[:, 1]).all() and ((rec[:, 1] == 0) == (rec[:, 0] == float("-inf"))).all()


@pytest.mark.parametrize("new", [[1, 1], [150, 70]])
def test_broadcast_views(new):
    """Queries are taken as they are; pages and results are refused."""
    from rdkv_b200.paged import append_kv, paged_attention
    from rdkv_b200.rope import rope_axes
    lens, T = [300, 111], sum(new)
    k, v, table = R.build_cache(lens, 2, 32, BF16, seed=71)
    args = (table, starts(new), ints(lens))
    q = randn(T, 8, 128, seed=72, dtype=BF16)
    for x in (q[:1].expand(T, 8, 128), q[:, :1].expand(T, 8, 128)):
        check(paged_attention(x, k, v, *args, max_new=max(new)), R.attention(x, k, v, *args))
    for x, y in ((k[:, :1].expand_as(k), v[:, :1].expand_as(v)), (k[:1].expand_as(k), v[:1].expand_as(v))):
        for pages in ((x, v), (k, y)):
            with pytest.raises(ValueError, match="broadcast"):
                paged_attention(q, *pages, *args, max_new=max(new))
    rows = randn(T, 2, 128, seed=73, dtype=BF16)
    slots, pos = torch.arange(T, device="cuda"), torch.arange(T, device="cuda")
    many = torch.empty(T, 1, 128, device="cuda", dtype=BF16).expand(T, 8, 128)
    for call in (lambda: paged_attention(q, k, v, *args, out=many), lambda: rope_axes(q, rows, pos, INV(), q_out=many),
                 lambda: rope_axes(q, rows, pos, INV(), k_out=many[:, :2]), lambda: append_kv(rows, rows, k[:1].expand_as(k), v, slots),
                 lambda: append_kv(rows, rows, k, v[:, :1].expand_as(v), slots),
                 lambda: append_kv(rows, rows, k, v, slots, q=q, positions=pos, inv_freq=INV(), q_out=many)):
        with pytest.raises(ValueError, match="broadcast"):
            call()


@pytest.mark.parametrize("max_new", [1, 200])
@pytest.mark.parametrize("start", [[3, 4, 9], [0, 0, 300], [2, 150, 200], [-7, 3, 8]])
def test_rows_in_front_and_starts_outside(start, max_new):
    """Query rows in front of the first request's are padding too, and rows outside the tensor are not touched.  A length below zero counts as none."""
    from rdkv_b200.paged import paged_attention
    k, v, table = R.build_cache([400, 333], 2, 32, BF16, seed=61)
    T = 203
    q = randn(T, 8, 128, seed=62, dtype=BF16)
    clamped = [min(max(x, 0), T) for x in start]
    for lens in ([400, 333], [-5, 300]):
        got = paged_attention(q, k, v, table, ints(start), ints(lens), max_new=max_new, check_status=True)
        check(got, R.attention(q, k, v, table, ints(clamped), ints([max(n, 0) for n in lens])))
        assert (got[:max(min(clamped), 0)] == 0).all() and (got[max(clamped):] == 0).all()


@pytest.mark.parametrize("S,H_kv,max_new", [(2, 2, 1), (2, 2, 200), (30, 1, 1), (60, 2, 1), (600, 1, 1), (600, 1, 200)])
def test_starts_that_fall_are_refused(S, H_kv, max_new):
    """Requests would share query rows.  The kernels compute nothing and say so, wherever the fall stands."""
    from rdkv_b200.paged import paged_attention
    k, v, table = R.build_cache([40] * S, H_kv, 32, BF16, seed=63)
    q = randn(S + 9, 4 * H_kv, 128, seed=64, dtype=BF16)
    for at in sorted({1, S // 2 + 1, S}):                     # q_start[at] < q_start[at - 1]
        start = [i + 3 if i < at else i for i in range(S + 1)]
        out = torch.full_like(q, 7.0)
        with pytest.raises(ValueError, match="q_start must not fall"):
            paged_attention(q, k, v, table, ints(start), ints([40] * S), max_new=max_new, out=out, check_status=True)
        assert (out == 7.0).all()


@pytest.mark.parametrize("new", [[1, 1], [100, 37]])
def test_layouts_and_buffers(new):
    """Pages whose rows come before their heads, query rows out of a fused projection (also with a stride no 16-byte
    load fits), a given result buffer whose padding is left as it was, scales."""
    from rdkv_b200.paged import paged_attention
    lens, pad = [300, 111], 5
    T = sum(new) + pad
    k, v, table = R.build_cache(lens, 2, 64, BF16, seed=31)
    args = (table, starts(new), ints(lens))
    k2, v2 = (x.permute(0, 2, 1, 3).contiguous().permute(0, 2, 1, 3) for x in (k, v))
    both = torch.cat([k, v], dim=3)
    for extra in (8, 3):
        q = torch.randn(T, 12, 128 + extra, device="cuda", generator=gen(1)).to(BF16)[:, 2:10, :128]
        want = paged_attention(q.contiguous(), k, v, *args, max_new=max(new), scale=0.2)
        check(want, R.attention(q, k, v, *args, scale=0.2))
        assert (want[-pad:] == 0).all()
        out = torch.full((T, 12, 136), 7.0, device="cuda", dtype=BF16)
        for pages in ((k2, v2), (both[..., :128], both[..., 128:])):
            got = paged_attention(q, *pages, *args, max_new=max(new), scale=0.2, out=out[:, 2:10, :128])
            assert torch.equal(got[:-pad], want[:-pad])
            assert (got[-pad:] == 7).all() and (out[:, :2] == 7).all() and (out[:, 10:] == 7).all() and (out[..., 128:] == 7).all()


def test_no_tokens_no_requests():
    from rdkv_b200.paged import paged_attention
    k, v, table = R.build_cache([64], 2, 16, F16, seed=1)
    assert paged_attention(randn(0, 8, 128, seed=1, dtype=F16), k, v, table, ints([0, 0]), ints([64])).shape == (0, 8, 128)
    q = randn(3, 8, 128, seed=1, dtype=F16)
    assert (paged_attention(q, k, v, table[:0], ints([0]), ints([])) == 0).all()
    assert (paged_attention(q, k[:0], v[:0], table, ints([0, 3]), ints([64])) == 0).all()
    assert (paged_attention(q, k, v, table[:, :0], ints([0, 3]), ints([64])) == 0).all()


@pytest.mark.parametrize("new", [[1, 1, 1], [130, 5, 0]])
@pytest.mark.parametrize("window", [0, 64])
def test_records_merge(new, window):
    """Records of the old tokens' pages and of the rest, merged, are the whole result."""
    from rdkv_b200.decode import lse_combine
    from rdkv_b200.paged import paged_attention
    lens = [400, 70, 9]
    q, k, v, table, whole = run(lens, new, 2, 4, 16, BF16, seed=41, window=window, sinks=5 if window else 0)
    T = sum(new)
    front, back = table.clone(), table.clone()
    front[:, 3:], back[:, :3] = -1, -1
    rec = torch.empty(2, T * 8, 132, device="cuda")
    for part, r in zip((front, back), rec):
        assert paged_attention(q, k, v, part, starts(new), ints(lens), max_new=max(new), window=window, sinks=5 if window else 0,
                               out_partial=r) is r
    got = lse_combine(rec.permute(1, 0, 2)).reshape(T, 8, 128)
    check(got, R.attention(q, k, v, table, starts(new), ints(lens), window, 5 if window else 0))
    one = torch.empty(T * 8, 1, 132, device="cuda")
    paged_attention(q, k, v, table, starts(new), ints(lens), max_new=max(new), window=window, sinks=5 if window else 0, out_partial=one)
    # the combine divides by the total, the kernel multiplies by its reciprocal: both are within 3 * 2^-24 of the quotient,
    # so they round to the same value or to neighbours, one step (eps) apart at most
    got = lse_combine(one).reshape(T, 8, 128)
    step = (got.to(BF16).double() - whole.double()).abs() <= torch.finfo(BF16).eps * got.double().abs()
    assert bool(step.all())


def test_offsets_past_32_bits():
    """Pages that lie more than 2^31 elements into their tensor."""
    from rdkv_b200.paged import append_kv, paged_attention
    n, page, H = 2 ** 31 // (8 * 64 * 128) + 40, 64, 8
    k = torch.empty(n, H, page, 128, dtype=BF16, device="cuda")
    v = torch.empty(n, H, page, 128, dtype=BF16, device="cuda")
    ids = [n - 1, 3, n - 20]
    rows = randn(180, H, 128, seed=1, dtype=BF16), randn(180, H, 128, seed=2, dtype=BF16)
    slots = torch.tensor([ids[p // page] * page + p % page for p in range(180)], device="cuda")
    append_kv(*rows, k, v, slots)
    small = [torch.zeros(3, H, page, 128, dtype=BF16, device="cuda") for _ in range(2)]
    append_kv(*rows, *small, torch.arange(180, device="cuda"))
    for new in (1, 100):
        q = randn(new, 32, 128, seed=3, dtype=BF16)
        got = paged_attention(q, k, v, ints([ids]), ints([0, new]), ints([180]))
        assert torch.equal(got, paged_attention(q, *small, ints([[0, 1, 2]]), ints([0, new]), ints([180])))


@pytest.mark.parametrize("new", [[1] * 6, [90, 1, 40, 3, 128, 17]])
@pytest.mark.parametrize("g", [4, 5, 7])
def test_results_repeat(new, g):
    """The same call again, beside others on another stream and after one with large queries (7 query heads a KV head
    leave rows of a tile without a token): the same bits."""
    from rdkv_b200.paged import paged_attention
    lens = [700, 64, 999, 300, 2000, 17]
    q, k, v, table, want = run(lens, new, 2, g, 16, BF16, seed=51)
    for size in (100.0, 1e-3):
        paged_attention(q * size, k, v, table, starts(new), ints(lens), max_new=max(new))
        assert torch.equal(paged_attention(q, k, v, table, starts(new), ints(lens), max_new=max(new)), want)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    mine, others = [], []
    for _ in range(20):
        mine.append(paged_attention(q, k, v, table, starts(new), ints(lens), max_new=max(new)))
        with torch.cuda.stream(side):
            others.append(paged_attention(q, k, v, table, starts(new), ints(lens), max_new=max(new)))
    torch.cuda.synchronize()
    assert all(torch.equal(x, want) for x in mine + others)


# ── together ─────────────────────────────────────────────────────────────────

def test_a_step_captured_and_replayed_with_other_lengths():
    """Tables, rotation, write and attention of a batch in one graph; two such graphs replayed side by side."""
    from rdkv_b200.paged import append_kv, build_block_tables, paged_attention
    S, page, H_kv, g, width = 3, 16, 2, 4, 30
    graphs = []
    for seed in (1, 2):
        st = dict(ctx=ints([0] * S), new=ints([0] * S), table=torch.full((S, width), -1, dtype=torch.int32, device="cuda"),
                  free=torch.randperm(S * width, generator=gen(seed), device="cuda").int(), start=ints([0]),
                  q=randn(64, H_kv * g, 128, seed=seed, dtype=BF16), k=randn(64, H_kv, 128, seed=seed + 5, dtype=BF16),
                  v=randn(64, H_kv, 128, seed=seed + 9, dtype=BF16), kp=torch.zeros(S * width, H_kv, page, 128, dtype=BF16, device="cuda"),
                  vp=torch.zeros(S * width, H_kv, page, 128, dtype=BF16, device="cuda"))

        def step(st=st):
            plan = build_block_tables(st["ctx"], st["new"], st["table"], st["free"], page, 64, free_start=st["start"])
            q = append_kv(st["k"], st["v"], st["kp"], st["vp"], plan.slot_map, q=st["q"], positions=plan.positions, inv_freq=INV())
            return plan, q, paged_attention(q, st["kp"], st["vp"], st["table"], plan.q_start, plan.kv_lens, max_new=64)
        step()
        graph, stream = torch.cuda.CUDAGraph(), torch.cuda.Stream()
        with torch.cuda.graph(graph):
            st["plan"], st["q_rot"], st["out"] = step()
        st["start"].zero_(); st["table"].fill_(-1)
        graphs.append((st, graph, stream))
    torch.cuda.synchronize()
    for new in ([33, 1, 20], [1, 1, 1], [0, 40, 3], [1, 0, 63]):
        for st, graph, stream in graphs:
            stream.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(stream):
                st["new"].copy_(ints(new))
                graph.replay()
        torch.cuda.synchronize()
        for st, graph, stream in graphs:
            lens = [a + b for a, b in zip(st["ctx"].tolist(), new)]
            assert st["plan"].kv_lens.tolist() == lens and st["plan"].missing.item() == 0
            want = R.attention(st["q_rot"], st["kp"], st["vp"], st["table"], starts(new), ints(lens))
            check(st["out"], want)
            st["ctx"].copy_(ints(lens)); st["start"].copy_(st["plan"].free_next)


def test_from_chunked_prefill_to_a_packed_cache():
    """A prompt prefilled in chunks is the prompt prefilled at once; its pages are packed, and the packed layer and the
    pages of the tokens after it answer one decode step through merged records."""
    from rdkv_b200 import synth
    from rdkv_b200.decode import DecodeTable, lse_combine, packed_decode_attention
    from rdkv_b200.packing import pack_kv
    from rdkv_b200.paged import append_kv, build_block_tables, paged_attention
    N, H_kv, g, page = 500, 2, 4, 16
    q, k, v = (randn(N, h, 128, seed=s, dtype=F16) for s, h in ((1, H_kv * g), (2, H_kv), (3, H_kv)))

    def prefill(chunks):
        table = torch.full((1, 40), -1, dtype=torch.int32, device="cuda")
        kp, vp = (torch.zeros(40, H_kv, page, 128, dtype=F16, device="cuda") for _ in range(2))
        start, free, at, outs = None, torch.randperm(40, generator=gen(9), device="cuda").int(), 0, []
        for n in chunks:
            plan = build_block_tables(ints([at]), ints([n]), table, free, page, n, free_start=start)
            rot = append_kv(k[at:at + n], v[at:at + n], kp, vp, plan.slot_map, q=q[at:at + n], positions=plan.positions, inv_freq=INV())
            outs.append(paged_attention(rot, kp, vp, table, plan.q_start, plan.kv_lens, max_new=n))
            start, at = plan.free_next, at + n
        return table, kp, vp, rot, torch.cat(outs)
    table, kp, vp, rot, once = prefill([N])
    table2, kp2, vp2, _, chunked = prefill([1, 130, 255, 64, 50])
    assert torch.equal(table, table2) and torch.equal(kp, kp2) and torch.equal(vp, vp2)
    want = R.attention(rot, kp, vp, table, ints([0, N]), ints([N]))
    check(once, want); check(chunked, want)
    # the first 480 tokens are packed; the last 20 stay in their pages
    P = 480
    dense = [x[table[0, :P // page].long()].permute(1, 0, 2, 3).reshape(1, H_kv, P, 128) for x in (kp, vp)]
    vb, kb = synth.make_v_bits(H_kv, P, 400, seed=3).cuda(), synth.make_k_bits(H_kv, seed=3).cuda()
    layer, v16 = pack_kv(dense[0].contiguous(), dense[1].contiguous(), vb, kb, g)
    dt = DecodeTable([layer], [v16], H_kv * g)
    rec = torch.empty(2, H_kv * g, 132, device="cuda")
    packed_decode_attention(rot[-1:], dt, out_partial=rec[0])
    rest = table.clone()
    rest[:, :P // page] = -1
    paged_attention(rot[-1:], kp, vp, rest, ints([0, 1]), ints([N]), max_new=1, out_partial=rec[1])
    got = lse_combine(rec.permute(1, 0, 2))
    tail = [x[table[0, P // page:32].long()].permute(1, 0, 2, 3).reshape(1, H_kv, -1, 128).contiguous() for x in (kp, vp)]
    one = packed_decode_attention(rot[-1:], dt, new_k=tail[0], new_v=tail[1], n_new=N - P)[0]
    assert torch.allclose(got, one, rtol=1e-2, atol=2e-3)


# ── refusals ─────────────────────────────────────────────────────────────────

def test_refusals():
    from rdkv_b200.paged import append_kv, build_block_tables, paged_attention
    from rdkv_b200.rope import rope_axes
    k, v, table = R.build_cache([64, 64], 2, 16, F16, seed=1)
    q = randn(2, 8, 128, seed=1, dtype=F16)
    good = dict(q=q, k_pages=k, v_pages=v, block_tables=table, q_start=ints([0, 1, 2]), kv_lens=ints([64, 64]))
    for change in (dict(q=q.float()), dict(q=q.to(BF16)), dict(q=q[:, :7]), dict(q=q[..., :64]), dict(q=q[0]), dict(v_pages=v[1:]), dict(v_pages=v.to(BF16)),
                   dict(k_pages=k[:, :, :8], v_pages=v[:, :, :8]), dict(block_tables=table.long()), dict(block_tables=table[:1]),
                   dict(q_start=ints([0, 2])), dict(kv_lens=ints([64])), dict(kv_lens=ints([64, 64]).long()), dict(window=-1), dict(sinks=3), dict(max_new=-1), dict(scale=0.0), dict(scale=-1.0), dict(scale=float("inf")), dict(scale=1e-50),
                   dict(out=torch.empty_like(q).float()), dict(out=torch.empty(2, 8, 129, dtype=F16, device="cuda")[..., 1:]),
                   dict(out_partial=torch.empty(16, 131, device="cuda")), dict(out=torch.empty_like(q), out_partial=torch.empty(16, 132, device="cuda")),
                   dict(k_pages=torch.empty(10, 2, 16, 132, dtype=F16, device="cuda")[..., :128], v_pages=torch.empty(10, 2, 16, 128, dtype=F16, device="cuda")),
                   dict(k_pages=k[:, :, :, ::2], v_pages=v[:, :, :, ::2])):
        with pytest.raises(ValueError):
            paged_attention(**{**good, **change})
    with pytest.raises(RuntimeError, match="CUDA"):
        paged_attention(**{**good, "q": q.cpu()})
    rows, slots = randn(2, 2, 128, seed=2, dtype=F16), torch.zeros(2, dtype=torch.int64, device="cuda")
    for args, kw in (((rows, rows[:1], k, v, slots), {}), ((rows.float(), rows.float(), k, v, slots), {}), ((rows, rows, k, v, slots.int()), {}),
                     ((rows, rows, k, v, slots[:1]), {}), ((rows, rows, k, v, slots), dict(q=q)), ((rows, rows, k, v, slots), dict(positions=ints([0, 1]))),
                     ((rows, rows, k, v, slots), dict(q=q, positions=ints([0]), inv_freq=INV())),
                     ((rows, rows, k, v, slots), dict(q=q.to(BF16), positions=ints([0, 1]), inv_freq=INV())),
                     ((rows, rows, k, v, slots), dict(q_out=q, positions=ints([0, 1]), inv_freq=INV()))):
        with pytest.raises(ValueError):
            append_kv(*args, **kw)
    pos = torch.zeros(3, 2, dtype=torch.int32, device="cuda")
    for p, f, sec in ((pos, INV(), None), (pos, INV(), (32, 32)), (pos, INV(), (30, 30, 5)), (pos, INV(), (70, -3, -3)), (pos.float(), INV(), (20, 20, 24)),
                      (pos[:, :1], INV(), (20, 20, 24)), (pos, INV().double(), (20, 20, 24)), (pos, INV()[:32], (20, 20, 24)),
                      (pos.repeat(2, 1), INV(), (10, 10, 10, 10, 10, 14))):
        with pytest.raises(ValueError):
            rope_axes(q, rows, p, f, sections=sec)
    with pytest.raises(ValueError):
        rope_axes(q, rows.to(BF16), pos[0], INV())
    base = (ints([3, 4]), ints([1, 1]), table, ints([5, 6]), 16, 2)
    for i, bad in ((0, ints([3])), (0, ints([3, 4]).long()), (2, table[:1]), (2, table.long()), (3, ints([[5]])), (4, 0), (5, -1)):
        with pytest.raises(ValueError):
            build_block_tables(*[bad if j == i else x for j, x in enumerate(base)])
    plan = build_block_tables(*base)
    with pytest.raises(ValueError):
        build_block_tables(*base, free_start=plan.free_next, out=plan)
    with pytest.raises(ValueError):
        build_block_tables(plan.kv_lens, *base[1:], out=plan)
    with pytest.raises(ValueError):
        paged_attention(**{**good, "out": q})
    with pytest.raises(ValueError):
        build_block_tables(*base[:5], 3, out=plan)
    n = 16385
    with pytest.raises(ValueError):
        build_block_tables(ints([0] * n), ints([0] * n), torch.zeros(n, 1, dtype=torch.int32, device="cuda"), ints([1]), 16, 1)
