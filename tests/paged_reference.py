"""The paged-cache operators from their definitions, in 64 bits and plain loops over requests."""
import math

import torch


def tables(ctx, new, table, free, page, n_tokens, start=0):
    """Python lists in, the new table and the step's lists out."""
    table = [list(r) for r in table]
    width = len(table[0]) if table else 0
    ctx, new = [max(c, 0) for c in ctx], [max(n, 0) for n in new]
    at, missing = start, 0
    for i, (c, n) in enumerate(zip(ctx, new)):
        for e in range(-(-c // page), -(-(c + n) // page)):
            if e >= width:
                missing += 1
                continue
            table[i][e] = free[at] if at < len(free) else -1
            missing += at >= len(free)
            at += 1
    slots, positions, q_start = [], [], [0]
    for i, (c, n) in enumerate(zip(ctx, new)):
        for p in range(c, c + n):
            e = p // page
            pid = table[i][e] if e < width else -1
            slots.append(pid * page + p % page if pid >= 0 else -1)
            positions.append(p)
        q_start.append(len(slots))
    pad = n_tokens - len(slots)
    return dict(tables=table, slot_map=(slots + [-1] * pad)[:n_tokens], positions=(positions + [0] * pad)[:n_tokens], q_start=q_start,
                kv_lens=[c + n for c, n in zip(ctx, new)], free_next=[min(at, len(free))], missing=[missing])


def rotate(x, positions, inv_freq, sections):
    """x [T,H,128], positions [axes,T] -> the rotated rows in 64 bits."""
    angle, first = torch.empty(x.shape[0], 64, dtype=torch.float64, device=x.device), 0
    for axis, n in enumerate(sections):
        angle[:, first:first + n] = positions[axis].double()[:, None] * inv_freq[first:first + n].double()[None]
        first += n
    c, s = angle.cos()[:, None], angle.sin()[:, None]
    a, b = x.double()[..., :64], x.double()[..., 64:]
    return torch.cat([a * c - b * s, b * c + a * s], dim=2)


def attention(q, k_pages, v_pages, table, q_start, kv_lens, window=0, sinks=0, scale=None):
    """(out [T,H_q,128] float64, tolerance of the same shape): zeros where a token sees nothing or belongs to no
    request.  The tolerance counts what a kernel for 16-bit types rounds: a softmax weight to 16 bits (half a step
    of its own size: u), the result to 16 bits (u of its size), and scores summed in 32 bits, whose error is a
    relative one of the weights (128 products, 2^-23 of the sum of their sizes each; twice, for weights and total)."""
    scale = 128 ** -0.5 if scale is None else scale
    u = torch.finfo(q.dtype).eps / 2
    T, H_q, D = q.shape
    n_pages, H_kv, page, _ = k_pages.shape
    g = H_q // H_kv
    out = torch.zeros(T, H_q, D, dtype=torch.float64, device=q.device)
    tol = torch.zeros_like(out)
    starts, lens, rows = q_start.tolist(), kv_lens.tolist(), table.tolist()
    for i, L in enumerate(lens):
        t0, t1 = starts[i], starts[i + 1]
        L_in = min(L, len(rows[i]) * page)
        if t1 <= t0 or L_in <= 0:
            continue
        key = torch.tensor([s for s in range(L_in) if 0 <= rows[i][s // page] < n_pages], device=q.device, dtype=torch.int64)
        if key.numel() == 0:
            continue
        ids = torch.tensor(rows[i], device=q.device)[key // page].long()
        pos = torch.arange(L - (t1 - t0), L, device=q.device)[:, None]
        seen = key[None] <= pos
        if window > 0:
            seen &= (key[None] > pos - window) | (key[None] < sinks)
        for h in range(H_kv):
            k, v = k_pages[ids, h, key % page].double(), v_pages[ids, h, key % page].double()
            for hq in range(h * g, h * g + g):
                x = q[t0:t1, hq].double()
                s = torch.where(seen, x @ torch.nan_to_num(k).t() * scale, -math.inf)
                top = s.amax(dim=1, keepdim=True)
                w = (s - torch.where(top == -math.inf, 0.0, top)).exp()
                w = w / w.sum(dim=1, keepdim=True).clamp(min=1e-300)
                v0 = torch.nan_to_num(v, nan=0.0, posinf=0.0, neginf=0.0)
                o = w @ v0
                size = torch.where(seen, x.abs() @ torch.nan_to_num(k, posinf=0.0, neginf=0.0).abs().t() * scale, 0.0).amax(dim=1, keepdim=True)
                delta = size * 128 * 2.0 ** -23 + 2.0 ** -18
                out[t0:t1, hq] = o
                tol[t0:t1, hq] = u * o.abs() + (u + 2 * delta) * (w @ v0.abs()) * (1 + u) + torch.finfo(q.dtype).smallest_normal * u * 2
    return out, tol


def build_cache(lens, H_kv, page, dtype, *, seed, device="cuda", spare=2, width_extra=1):
    """Random pages, and block tables that scatter the requests' pages over them."""
    g = torch.Generator(device=device).manual_seed(seed)
    blocks = [-(-n // page) for n in lens]
    n = sum(blocks) + spare
    k, v = (torch.randn(n, H_kv, page, 128, generator=g, device=device).to(dtype) for _ in range(2))
    order = torch.randperm(n, generator=g, device=device).tolist()
    width = max(blocks, default=0) + width_extra
    table, at = [], 0
    for b in blocks:
        table.append(order[at:at + b] + [-1] * (width - b))
        at += b
    return k, v, torch.tensor(table, dtype=torch.int32, device=device).reshape(len(lens), width)
