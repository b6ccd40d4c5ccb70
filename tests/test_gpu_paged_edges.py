"""The paged cache on the GPU: calls at the edge of what its documentation allows."""
import random
from fractions import Fraction

import pytest
import torch

import paged_reference as R
from test_gpu_paged import BF16, F16, INV, check, gen, ints, near, randn, starts

pytestmark = pytest.mark.gpu


def test_records_off_16_bytes_are_refused():
    from rdkv_b200.paged import paged_attention
    k, v, table = R.build_cache([64], 2, 16, F16, seed=1)
    q = randn(1, 8, 128, seed=2, dtype=F16)
    flat = torch.zeros(8 * 132 + 4, device="cuda")
    for shift in (1, 2, 3):
        with pytest.raises(ValueError, match="16 bytes"):
            paged_attention(q, k, v, table, ints([0, 1]), ints([64]), out_partial=flat[shift:shift + 8 * 132].view(8, 132))
    paged_attention(q, k, v, table, ints([0, 1]), ints([64]), out_partial=flat[4:].view(8, 132))
    assert (flat[:4] == 0).all() and (flat[5::132] > 0).all()


# ── starts behind the last row ───────────────────────────────────────────────

def wanted(q, k, v, table, start, lens, T):
    """The reference with the rows' own positions: row t of request i stands at lens[i] - (start[i+1] - t), whether the
    rows up to start[i+1] are all there or not."""
    clamped = [min(max(x, 0), T) for x in start]
    own = [max(0, n - max(0, start[i + 1] - T)) for i, n in enumerate(lens)]
    return R.attention(q, k, v, table, ints(clamped), ints(own))


@pytest.mark.parametrize("max_new", [1, 300])
@pytest.mark.parametrize("start,T", [([0, 0, 300], 203), ([0, 40, 2 ** 31 - 1], 60), ([0, 300, 333], 7), ([-5, 3, 400], 399)])
def test_starts_behind_the_last_row_keep_positions(start, T, max_new):
    """Rows that the tensor does not have are not computed; those it has stand where they stood."""
    from rdkv_b200.paged import paged_attention
    k, v, table = R.build_cache([500, 450], 2, 32, BF16, seed=61)
    q = randn(T, 8, 128, seed=62, dtype=BF16)
    for lens in ([500, 450], [310, 400], [4, 0]):
        got = paged_attention(q, k, v, table, ints(start), ints(lens), max_new=max_new, check_status=True)
        check(got, wanted(q, k, v, table, start, lens, T), f"{lens}")


def test_a_step_with_fewer_token_places_than_tokens():
    """Tables, write and attention of such a step agree on where its rows stand."""
    from rdkv_b200.paged import append_kv, build_block_tables, paged_attention
    table = torch.full((2, 4), -1, dtype=torch.int32, device="cuda")
    kp, vp = (torch.full((9, 2, 16, 128), float("nan"), dtype=BF16, device="cuda") for _ in range(2))     # (what was never written shows)
    plan = build_block_tables(ints([0, 0]), ints([20, 30]), table, ints([5, 6, 7, 8]), 16, 25)
    q, k, v = (randn(25, h, 128, seed=h, dtype=BF16) for h in (8, 2, 2))
    rot = append_kv(k, v, kp, vp, plan.slot_map, q=q, positions=plan.positions, inv_freq=INV())
    got = paged_attention(rot, kp, vp, table, plan.q_start, plan.kv_lens, check_status=True)
    kp, vp = kp.nan_to_num(), vp.nan_to_num()
    check(got, R.attention(rot, kp, vp, table, ints([0, 20, 25]), ints([20, 5])))


# ── what a call remembers ────────────────────────────────────────────────────

@pytest.mark.parametrize("new", [[1, 1], [40, 30]])
def test_numbers_in_tensors_are_read_at_every_call(new):
    """window, sinks, scale and max_new may be tensors of one element: their values count, not their identity."""
    from rdkv_b200.paged import paged_attention
    lens = [300, 111]
    k, v, table = R.build_cache(lens, 2, 32, BF16, seed=31)
    q = randn(sum(new), 8, 128, seed=32, dtype=BF16)
    args = (q, k, v, table, starts(new), ints(lens))
    window, sinks, scale, most = (torch.tensor(x) for x in (200, 3, 0.08, 1))
    for w, s, c in ((200, 3, 0.08), (17, 0, 0.3), (64, 40, 0.01)):
        window.fill_(w); sinks.fill_(s); scale.fill_(c); most.fill_(max(new))
        got = paged_attention(*args, max_new=most, window=window, sinks=sinks, scale=scale)
        assert torch.equal(got, paged_attention(*args, max_new=max(new), window=w, sinks=s, scale=float(scale)))


def test_sections_in_tensors_are_read_at_every_call():
    from rdkv_b200.paged import append_kv
    from rdkv_b200.rope import rope_axes
    T = 9
    q, k = randn(T, 4, 128, seed=1, dtype=BF16), randn(T, 2, 128, seed=2, dtype=BF16)
    pos = torch.randint(0, 5000, (2, T), generator=gen(3), device="cuda", dtype=torch.int32)
    kp, vp = (torch.zeros(1, 2, 16, 128, dtype=BF16, device="cuda") for _ in range(2))
    sections = [torch.tensor(64), torch.tensor(0)]
    for n in (64, 20, 0):
        sections[0].fill_(n); sections[1].fill_(64 - n)
        want = rope_axes(q, k, pos, INV(), sections=(n, 64 - n))
        for x, y in zip(rope_axes(q, k, pos, INV(), sections=sections), want):
            assert torch.equal(x, y)
        got = append_kv(k, k, kp, vp, torch.arange(T, device="cuda"), q=q, positions=pos, inv_freq=INV(), sections=sections)
        assert torch.equal(got, want[0]) and torch.equal(kp[0, :, :T].transpose(0, 1), want[1])


# ── starts that fall ─────────────────────────────────────────────────────────

@pytest.mark.parametrize("S,H_kv,max_new", [(2, 2, 1), (2, 2, 200), (60, 2, 1), (600, 1, 200)])
def test_starts_that_fall_leave_zeros_in_a_result_of_the_call(S, H_kv, max_new):
    """Without check_status nobody is told; what comes back is not what memory happened to hold."""
    from rdkv_b200.paged import paged_attention
    k, v, table = R.build_cache([40] * S, H_kv, 32, BF16, seed=63)
    q = randn(S + 9, 4 * H_kv, 128, seed=64, dtype=BF16)
    for at in sorted({1, S // 2 + 1, S}):
        start = [i + 3 if i < at else i for i in range(S + 1)]
        held = torch.full_like(q, 7.0)
        del held                                                        # (the allocator hands out this memory next)
        out = paged_attention(q, k, v, table, ints(start), ints([40] * S), max_new=max_new)
        assert (out == 0).all()


# ── values that are not finite ───────────────────────────────────────────────

def bits(x):
    return x.contiguous().view(torch.int16)


def spoil(k, v, table, lens, at, seed, dtype):
    """A copy of v with NaN and infinities in some channels of the tokens ``at`` = [(request, token)], and where they are."""
    rng = random.Random(seed)
    v, where = v.clone(), []
    page = k.shape[2]
    for i, s in at:
        for h in range(k.shape[1]):
            channels = rng.sample(range(128), rng.choice([1, 1, 3, 128]))
            kind = torch.tensor([rng.choice([float("nan"), float("inf"), -float("inf")]) for _ in channels], dtype=dtype, device="cuda")
            v[table[i, s // page], h, s % page, channels] = kind
            where.append((i, s, h, channels))
    return v, where


def touched(T, H_q, H_kv, start, lens, where, window, sinks):
    """Which results see one of these values."""
    out = torch.zeros(T, H_q, 128, dtype=torch.bool)
    g = H_q // H_kv
    for i, s, h, channels in where:
        p = torch.arange(start[i], start[i + 1]) + lens[i] - start[i + 1]
        sees = (s <= p) & ((s > p - window) if window > 0 and s >= sinks else torch.ones_like(p, dtype=torch.bool))
        for c in channels:
            out[start[i]:start[i + 1], h * g:(h + 1) * g, c] |= sees[:, None]
    return out.cuda()


def spoiled(lens, new, H_kv, g, page, dtype, at, seed=0, window=0, sinks=0, max_new=None):
    """Results that see such a value are not finite, all others are those of the same call with clean values, bit for bit;
    and so in records."""
    from rdkv_b200.paged import paged_attention
    k, v, table = R.build_cache(lens, H_kv, page, dtype, seed=seed)
    T, H_q = sum(new), H_kv * g
    q = randn(T, H_q, 128, seed=seed + 1, dtype=dtype)
    args = (table, starts(new), ints(lens))
    kw = dict(max_new=max(new) if max_new is None else max_new, window=window, sinks=sinks, check_status=True)
    bad, where = spoil(k, v, table, lens, at, seed, dtype)
    seen = touched(T, H_q, H_kv, starts(new).tolist(), lens, where, window, sinks)
    clean = paged_attention(q, k, v, *args, **kw)
    check(clean, R.attention(q, k, v, *args, window, sinks))
    got = paged_attention(q, k, bad, *args, **kw)
    assert not torch.isfinite(got[seen]).any()
    assert torch.equal(bits(got[~seen]), bits(clean[~seen]))
    recs = [torch.zeros(T * H_q, 132, device="cuda") for _ in range(2)]
    for x, r in zip((v, bad), recs):
        paged_attention(q, k, x, *args, out_partial=r, **kw)
    assert torch.equal(recs[0][:, :2], recs[1][:, :2])
    o, o_bad = (r[:, 4:].reshape(T, H_q, 128) for r in recs)
    assert not torch.isfinite(o_bad[seen]).any() and torch.equal(o_bad[~seen], o[~seen])
    return q, k, bad, args, kw, got


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("g", [1, 4, 5])
@pytest.mark.parametrize("window,sinks", [(0, 0), (1, 0), (3, 2), (40, 20), (150, 70), (300, 0)])
@pytest.mark.parametrize("new", [[3, 2, 1], [260, 130, 1]])
def test_bad_values_reach_the_results_that_see_them(dtype, g, window, sinks, new):
    """In the chunk, at either end of the window, at the last sink, in front of everything, at a page's first and last row."""
    lens = [700, 333, 64]
    at = [(0, s) for s in (0, 1, 19, 20, 69, 70, 300, 399, 400, 438, 439, 440, 441, 511, 512, 550, 600, 697, 698, 699)]
    at += [(1, s) for s in (2, 31, 200, 203, 300, 331, 332)] + [(2, 62), (2, 63)]
    spoiled(lens, new, 2, g, 32, dtype, at, seed=g + window, window=window, sinks=sinks)
    spoiled(lens, new, 2, g, 32, dtype, [(0, sum(lens) % 97 + 600)], seed=g, window=window, sinks=sinks)
    spoiled([5 * n for n in new], new, 1, g, 16, dtype, [(0, 4 * new[0] + 1), (1, 5 * new[1] - 1)], seed=g, window=window, sinks=sinks)   # (clusters)


@pytest.mark.parametrize("new,max_new", [([700, 700, 690], 700), ([16] * 9, 16), ([4] * 60, 4)])
def test_bad_values_behind_a_long_context_among_other_requests(new, max_new):
    """One bad value in the first request's chunk behind 20000 tokens, CTAs with several segments: the others' results are
    there, and no wait runs out (check_status)."""
    lens = [20000 + n for n in new[:1]] + [3000 + 400 * (i % 5) + n for i, n in enumerate(new[1:])]
    spoiled(lens, new, 2, 4, 64, BF16, [(0, 20000 + new[0] // 2)], seed=5, max_new=max_new)


def test_results_repeat_with_bad_values():
    """A value in a tile that only the second half of an item sees: the first half's results are the same every time."""
    from rdkv_b200.paged import paged_attention
    lens, new = [992 + 64, 608 + 64], [64, 64]               # (4 query heads: an item is two halves of 32 tokens; tiles of 128 keys)
    for at in ([(0, 1024 + 20)], [(0, 1024 + 31), (1, 640 + 5)]):
        q, k, bad, args, kw, got = spoiled(lens, new, 2, 4, 32, F16, at, seed=17)
        for _ in range(30):
            assert torch.equal(bits(paged_attention(q, k, bad, *args, **kw)), bits(got))


# ── waits that run out ───────────────────────────────────────────────────────

@pytest.mark.parametrize("requests,new,H_kv,window", [(30, 1, 1, 0), (30, 4, 1, 9000), (200, 1, 2, 0), (200, 4, 2, 1300), (160, 20, 1, 0), (160, 300, 1, 0), (160, 300, 1, 200)])
def test_a_wait_that_runs_out_is_reported(requests, new, H_kv, window):
    """With no time to wait, a CTA gives up at its first wait that the first try (about 1 us) does not see the end of, and with all of them after cold
    memory some do: in clusters, on the line of units, in chunks of one half and of several items.  The call ends, its status
    words say so, and the next call is right."""
    import ctypes as C
    from rdkv_b200 import paged
    from rdkv_b200._lib import PagedAttentionArgs, lib, raw_stream
    lens = [20000 if requests < 100 else 1500] * requests
    k, v, table = R.build_cache(lens, H_kv, 64, BF16, seed=3)
    other = torch.empty(1 << 26, dtype=torch.int32, device="cuda")       # (twice what L2 holds)
    q = randn(requests * new, 4 * H_kv, 128, seed=4, dtype=BF16)
    start, tokens = starts([new] * requests), ints(lens)
    want = paged.paged_attention(q, k, v, table, start, tokens, max_new=new, window=window, check_status=True)
    _, direct, n_ws, index, fields, _ = paged._attention_check(q, k, v, table, start, tokens, new, window, 0, None)
    assert direct
    words = lib().rdkv_paged_attention_status_words()
    args = PagedAttentionArgs.from_buffer_copy(fields)
    for wait_us, expected in ((0, 1), (2000000, 0)):
        out, ws = torch.zeros_like(q), torch.zeros(n_ws, dtype=torch.int32, device="cuda")
        seen = set()
        for _ in range(10):
            other.fill_(1)
            assert lib().rdkv_paged_attention_within(C.addressof(args), q.data_ptr(), k.data_ptr(), v.data_ptr(), table.data_ptr(), start.data_ptr(),
                                                     tokens.data_ptr(), out.data_ptr(), out.stride(0), out.stride(1), 0, None, ws.data_ptr(), 4 * n_ws,
                                                     wait_us, raw_stream(index)) == 0
            seen.add(int(ws[:words].max()))
        assert expected in seen and seen <= {0, expected}
    assert torch.equal(out, want)
    assert torch.equal(paged.paged_attention(q, k, v, table, start, tokens, max_new=new, window=window, check_status=True), want)


# ── far positions ────────────────────────────────────────────────────────────

TWO_PI = Fraction(6283185307179586476925286766559005768394, 10 ** 39)     # 2 pi to 40 digits


@pytest.mark.parametrize("far", [2 ** 24, 2 ** 29, 2 ** 31 - 1, 2 ** 40, 2 ** 53])
def test_far_positions_lose_nothing(far):
    """Angles from exact arithmetic: position * inv_freq as a fraction, its whole turns taken off with 2 pi to 40 digits
    (an error of far * 1e-40 turns), sine and cosine of what is left in 64 bits."""
    from rdkv_b200.rope import rope_axes
    rng = random.Random(far)
    positions = [far, far - 1] + [rng.randint(far // 2, far) for _ in range(10)]
    inv = INV()
    rest = [[float((p * Fraction(f)) % TWO_PI) for f in inv.tolist()] for p in positions]
    q = randn(len(positions), 3, 128, seed=5, dtype=torch.float32)
    pos = torch.tensor(positions, device="cuda", dtype=torch.int64 if far > 2 ** 31 - 1 else torch.int32)
    angle = torch.tensor(rest, dtype=torch.float64, device="cuda")[:, None]
    a, b = q.double()[..., :64], q.double()[..., 64:]
    want = torch.cat([a * angle.cos() - b * angle.sin(), b * angle.cos() + a * angle.sin()], dim=2)
    for got in rope_axes(q, q[:, :1], pos, inv):
        near(got, want[:, :got.shape[1]], q[:, :got.shape[1]], torch.float32)


# ── results that share memory with what is read ──────────────────────────────

@pytest.mark.parametrize("new", [[1, 1], [40, 3]])
def test_a_result_that_shares_rows_with_the_queries_is_refused(new):
    from rdkv_b200.paged import paged_attention
    lens, T = [300, 111], sum(new)
    k, v, table = R.build_cache(lens, 2, 32, BF16, seed=71)
    args = (k, v, table, starts(new), ints(lens))
    buf = randn(2 * T, 12, 128, seed=72, dtype=BF16)
    for q, out in ((buf[:T, :8], buf[1:T + 1, :8]), (buf[1:T + 1, :8], buf[:T, :8]), (buf[:T, :8], buf[:T, 1:9]), (buf[:T, :8], buf[:T, 4:12]),
                   (buf[:T, :8], buf[:T, :8]), (buf[:2 * T:2, :8], buf[:T, 4:12])):
        kept = buf.clone()
        with pytest.raises(ValueError, match="share memory"):
            paged_attention(q, *args, out=out)
        assert torch.equal(buf, kept)
    wide = randn(2 * T, 16, 128, seed=73, dtype=BF16)
    for q, out in ((wide[:T, :8], wide[:T, 8:]), (wide[:T, :8], wide[T:, :8]), (wide[::2, :8], wide[1::2, :8]), (wide[:T, :8], wide[1:T + 1, 8:])):
        want = paged_attention(q.contiguous(), *args)
        assert torch.equal(paged_attention(q, *args, out=out), want)


def test_rotated_rows_that_share_memory_are_refused():
    from rdkv_b200.paged import append_kv
    from rdkv_b200.rope import rope_axes
    T = 20
    pos, slots = torch.arange(T, device="cuda"), torch.arange(T, device="cuda")
    kp, vp = (torch.zeros(4, 2, 16, 128, dtype=BF16, device="cuda") for _ in range(2))
    buf = randn(2 * T, 16, 128, seed=74, dtype=BF16)
    q, k, v = buf[:T, :8], buf[:T, 8:10], buf[:T, 10:12]
    kept = buf.clone()
    for kw in (dict(q_out=buf[1:T + 1, :8]), dict(q_out=buf[:T, 1:9]), dict(q_out=buf[:T, 4:12]), dict(k_out=buf[1:T + 1, 8:10]), dict(k_out=buf[:T, 7:9]),
               dict(q_out=q, k_out=buf[:T, 6:8]), dict(q_out=buf[T:, :8], k_out=buf[T:, 7:9]), dict(q_out=buf[:2 * T:2, :8]),
               dict(q_out=buf.view(-1, 8, 128)[:T]), dict(k_out=buf[:T, :2])):
        with pytest.raises(ValueError, match="memory"):
            rope_axes(q, k, pos, INV(), **kw)
        if "k_out" not in kw:
            with pytest.raises(ValueError, match="memory"):
                append_kv(k, v, kp, vp, slots, q=q, positions=pos, inv_freq=INV(), **kw)
    with pytest.raises(ValueError, match="memory"):
        append_kv(k, v, kp, vp, slots, q=q, positions=pos, inv_freq=INV(), q_out=buf[:T, 3:11])
    with pytest.raises(ValueError, match="memory"):
        append_kv(k, v, kp, vp, slots, q=q, positions=pos, inv_freq=INV(), q_out=buf[:T, 8:])
    with pytest.raises(ValueError, match="memory"):
        append_kv(k, v, kp, kp, slots)
    assert torch.equal(buf, kept) and (kp == 0).all() and (vp == 0).all()
    want = rope_axes(q.contiguous(), k.contiguous(), pos, INV())
    for kw in (dict(q_out=buf[T:, :8], k_out=buf[T:, 8:10]), dict(q_out=buf[T:, 4:12]), dict(k_out=buf[:T, 14:]), dict(q_out=q, k_out=k)):
        buf.copy_(kept)
        got = rope_axes(q, k, pos, INV(), **kw)
        assert all(torch.equal(x, y) for x, y in zip(got, want)) and all(got[("q_out", "k_out").index(n)] is x for n, x in kw.items())
    for out in (buf[T:, :8], q):
        buf.copy_(kept)
        assert torch.equal(append_kv(k, v, kp, vp, slots, q=q, positions=pos, inv_freq=INV(), q_out=out), want[0])
        assert torch.equal(kp.transpose(1, 2).reshape(-1, 2, 128)[:T], want[1])


def test_a_plan_whose_tensors_share_memory_is_refused():
    from rdkv_b200.paged import build_block_tables
    table = torch.full((3, 4), -1, dtype=torch.int32, device="cuda")
    args = (ints([0, 5, 9]), ints([20, 1, 4]), table, ints([5, 6, 7, 8]), 16, 25)
    plan = build_block_tables(*args)
    ring = torch.zeros(64, dtype=torch.int32, device="cuda")
    for bad in (dict(kv_lens=plan.q_start[1:]), dict(free_next=plan.missing), dict(kv_lens=plan.positions[5:8]), dict(positions=plan.slot_map.view(torch.int32)[:25]),
                dict(q_start=ring[:4], positions=ring[3:28]), dict(kv_lens=args[0]), dict(free_next=table[1, 2:3])):
        with pytest.raises(ValueError, match="shares memory"):
            build_block_tables(*args, out=plan._replace(**bad))
    table.fill_(-1)
    again = build_block_tables(*args, out=plan._replace(q_start=ring[:4], positions=ring[4:29], kv_lens=ring[30:33]))
    table.fill_(-1)
    for x, y in zip(again, build_block_tables(*args)):
        assert torch.equal(x, y)


def test_results_whose_rows_overlap_are_refused():
    from rdkv_b200.paged import append_kv, paged_attention
    from rdkv_b200.rope import rope_axes
    lens, T = [300, 111], 3
    k, v, table = R.build_cache(lens, 2, 32, BF16, seed=71)
    q, rows = randn(T, 8, 128, seed=72, dtype=BF16), randn(T, 2, 128, seed=73, dtype=BF16)
    pos, slots, flat = torch.arange(T, device="cuda"), torch.arange(T, device="cuda"), torch.zeros(1 << 20, dtype=BF16, device="cuda")
    many, few = flat.as_strided((T, 8, 128), (512, 128, 1)), flat.as_strided((T, 2, 128), (128, 64, 1))
    pages = flat.as_strided(k.shape, (32 * 128, 32 * 128, 128, 1))
    for call in (lambda: paged_attention(q, k, v, table, ints([0, 1, 3]), ints(lens), out=many), lambda: rope_axes(q, rows, pos, INV(), q_out=many),
                 lambda: rope_axes(q, rows, pos, INV(), k_out=few), lambda: append_kv(rows, rows, pages, v, slots), lambda: append_kv(rows, rows, k, pages, slots),
                 lambda: append_kv(rows, rows, k, v, slots, q=q, positions=pos, inv_freq=INV(), q_out=many)):
        with pytest.raises(ValueError, match="overlap"):
            call()
    args = (table.clamp(max=1), ints([0, 1, 3]), ints(lens))             # read, such pages are pages
    assert torch.equal(paged_attention(q, pages, v, *args), paged_attention(q, pages.contiguous(), v, *args))


# ── shapes ───────────────────────────────────────────────────────────────────

def test_tensors_without_dimensions_are_refused():
    from rdkv_b200.paged import append_kv, build_block_tables, paged_attention
    from rdkv_b200.rope import rope_axes
    k, v, table = R.build_cache([64], 2, 16, F16, seed=1)
    rows, q, none, slots, pos = randn(2, 2, 128, seed=2, dtype=F16), randn(2, 8, 128, seed=3, dtype=F16), torch.zeros((), device="cuda"), torch.zeros(2, dtype=torch.int64, device="cuda"), ints([0, 1])
    half, number = none.half(), none.int()
    for call in (lambda: append_kv(half, half, k, v, slots), lambda: append_kv(rows, half, k, v, slots), lambda: append_kv(rows, rows, half, half, slots),
                 lambda: append_kv(rows, rows, k, v, none.long()), lambda: append_kv(rows, rows, k, v, slots, q=half, positions=pos, inv_freq=INV()),
                 lambda: append_kv(rows, rows, k, v, slots, q=q, positions=number, inv_freq=INV()), lambda: rope_axes(q, rows, number, INV()),
                 lambda: append_kv(rows, rows, k, v, slots, q=q, positions=pos, inv_freq=none), lambda: rope_axes(half, half, pos, INV()),
                 lambda: rope_axes(q, rows, pos, INV(), q_out=half), lambda: paged_attention(half, k, v, table, ints([0, 2]), ints([64])),
                 lambda: paged_attention(q, half, half, table, ints([0, 2]), ints([64])), lambda: paged_attention(q, k, v, number, ints([0, 2]), ints([64])),
                 lambda: paged_attention(q, k, v, table, number, ints([64])), lambda: paged_attention(q, k, v, table, ints([0, 2]), number),
                 lambda: paged_attention(q, k, v, table, ints([0, 2]), ints([64]), out=half), lambda: build_block_tables(number, number, table, number, 16, 2),
                 lambda: build_block_tables(ints([0]), ints([1]), number, ints([1]), 16, 2)):
        with pytest.raises(ValueError):
            call()


def test_extents_past_32_bits_are_refused():
    """2^32 + 4 tokens are not four."""
    from rdkv_b200.paged import append_kv, build_block_tables
    many = 2 ** 32 + 4
    k, v, table = R.build_cache([64], 2, 16, F16, seed=1)
    kept = k.clone(), v.clone()
    rows = randn(1, 2, 128, seed=2, dtype=F16).expand(many, 2, 128)
    slots = torch.empty(many, dtype=torch.int64, device="cuda")
    slots[:4] = torch.arange(4, device="cuda")
    with pytest.raises(ValueError, match="2\\^31"):
        append_kv(rows, rows, k, v, slots)
    del slots
    with pytest.raises(ValueError, match="2\\^31"):
        build_block_tables(ints([0]), ints([1]), table[:1], ints([1]), 2 ** 32 + 16, 4)
    with pytest.raises(ValueError, match="2\\^31"):
        build_block_tables(ints([0]), ints([1]), table[:1], ints([1]), 16, many)
    assert torch.equal(k, kept[0]) and torch.equal(v, kept[1])


# ── captures ─────────────────────────────────────────────────────────────────

FIRST_CALLS = '''
import sys
sys.path[:0] = [{root!r}, {tests!r}]
import torch
import paged_reference as R
from test_gpu_paged import BF16, F16, INV, check, ints, randn, starts
from rdkv_b200.paged import append_kv, build_block_tables, paged_attention
torch.zeros(1, device="cuda")
lens, new, window = {case!r}
S, T, dtype = len(lens), sum(new), {dtype}
table = torch.arange(S * 8, device="cuda", dtype=torch.int32).view(S, 8)
kp, vp = (randn(S * 8, 2, 64, 128, seed=s, dtype=dtype) for s in (1, 2))
q, k, v = (randn(T, h, 128, seed=h, dtype=dtype) for h in (8, 2, 2))
ctx, fresh, free, inv = ints([a - b for a, b in zip(lens, new)]), ints(new), ints([0]), INV()
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    plan = build_block_tables(ctx, fresh, table, free, 64, T)
    rot = append_kv(k, v, kp, vp, plan.slot_map, q=q, positions=plan.positions, inv_freq=inv)
    out = paged_attention(rot, kp, vp, table, plan.q_start, plan.kv_lens, max_new=max(new), window=window)
table.copy_(torch.arange(S * 8, device="cuda", dtype=torch.int32).view(S, 8))
for _ in range(2):
    graph.replay()
    torch.cuda.synchronize()
check(out, R.attention(rot, kp, vp, table, starts(new), ints(lens), window))
check(paged_attention(rot, kp, vp, table, plan.q_start, plan.kv_lens, max_new=max(new), window=window), R.attention(rot, kp, vp, table, starts(new), ints(lens), window))
print("as wanted")
'''


@pytest.mark.parametrize("case,dtype", [(([400, 77], [1, 1], 0), "BF16"), (([400] * 40, [1] * 40, 0), "F16"), (([400, 77], [100, 60], 0), "BF16"), (([400, 77], [100, 60], 64), "F16")])
def test_the_first_calls_of_a_process_are_captured(case, dtype):
    """Nothing has been loaded, asked for or set when a capture begins."""
    import os
    import subprocess
    import sys
    tests = os.path.dirname(os.path.abspath(__file__))
    code = FIRST_CALLS.format(root=os.path.dirname(tests), tests=tests, case=case, dtype=dtype)
    done = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300)
    assert done.returncode == 0 and "as wanted" in done.stdout, done.stderr[-2000:]


@pytest.mark.parametrize("new", [[1] * 3, [1] * 40, [90, 40, 7]])
def test_two_graphs_of_one_pool_and_threads_side_by_side(new):
    """Graphs that share a memory pool, replayed one after the other, and calls of several host threads on streams of their own."""
    import threading
    from rdkv_b200.paged import paged_attention
    lens = [300 + 7 * i for i in range(len(new))]
    k, v, table = R.build_cache(lens, 2, 32, BF16, seed=31)
    qs = [randn(sum(new), 8, 128, seed=s, dtype=BF16) for s in range(4)]
    args = (k, v, table, starts(new), ints(lens))
    want = [paged_attention(q, *args, max_new=max(new)) for q in qs]
    graphs = []
    for q in qs[:2]:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, pool=graphs[0][0].pool() if graphs else None):
            out = paged_attention(q, *args, max_new=max(new))
        graphs.append((graph, out))
    for _ in range(5):
        for (graph, out), x in zip(graphs, want):
            graph.replay()
            assert torch.equal(out, x)
    got = [[] for _ in qs]

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(20):
                got[i].append(paged_attention(qs[i], *args, max_new=max(new)))
            torch.cuda.current_stream().synchronize()
    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    torch.cuda.synchronize()
    [t.start() for t in threads]; [t.join() for t in threads]
    assert all(len(g) == 20 and all(torch.equal(x, w) for x in g) for g, w in zip(got, want))
