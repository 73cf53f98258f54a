"""Plain models of the paged key/value cache's operators, on the CPU: what the kernels are compared with."""

import math

import torch

E4M3 = torch.float8_e4m3fn


def rope_table(rot, rows, theta=10000.0):
    inv = theta ** (-torch.arange(0, rot, 2, dtype=torch.float64) / rot)
    a = torch.arange(rows, dtype=torch.float64)[:, None] * inv
    return torch.stack([a.cos(), a.sin()], -1).float()


def rotate(x, positions, table, interleaved):
    """fp32 rotation of `x [T, H, D]`, one rounding per operation; tokens outside the table pass."""
    half = table.shape[1]
    inside = (positions >= 0) & (positions < table.shape[0])
    f = table[positions.clamp(0, table.shape[0] - 1).long()]
    c, s = f[:, None, :, 0], f[:, None, :, 1]
    x = x.float()
    y = x.clone()
    if interleaved:
        a, b = x[..., 0:2 * half:2], x[..., 1:2 * half:2]
        y[..., 0:2 * half:2], y[..., 1:2 * half:2] = a * c - b * s, a * s + b * c
    else:
        a, b = x[..., :half], x[..., half:2 * half]
        y[..., :half], y[..., half:2 * half] = a * c - b * s, a * s + b * c
    return torch.where(inside[:, None, None], y, x)


def scale_of(amax):
    """Smallest power of two that brings amax to at most 448 (of nothing: the smallest normal number)."""
    if amax == 0:
        return 2.0 ** -126
    m, e = math.frexp(amax)
    return max(2.0 ** (e - 9 if m <= 0.875 else e - 8), 2.0 ** -126)


def append(x, cache, scale, table, lens, cu):
    """`x` (fp32 [T, H, 128]) into `cache [pages, page, H, 128]`, token by token and page by page."""
    pages, page = cache.shape[:2]
    width = table.shape[1]
    for b in range(table.shape[0]):
        n = int(cu[b + 1] - cu[b])
        first = int(lens[b]) - n
        by_page = {}
        for i in range(n):
            pos = first + i
            if pos < 0 or pos >= width * page or not 0 <= int(table[b, pos // page]) < pages:
                continue
            by_page.setdefault(pos // page, []).append((pos % page, int(cu[b]) + i))
        for at, rows in by_page.items():
            pid = int(table[b, at])
            slots, toks = [r[0] for r in rows], [r[1] for r in rows]
            new = x[toks]
            if scale is None:
                cache[pid, slots] = new.to(cache.dtype)
                continue
            held = max(first - at * page, 0)
            for h in range(cache.shape[2]):
                s = scale_of(float(new[:, h].abs().max()))
                if held:
                    s = max(s, float(scale[pid, h]))
                    old = cache[pid, :held, h].float() * (float(scale[pid, h]) / s)
                    cache[pid, :held, h] = old.to(E4M3)
                scale[pid, h] = s
                cache[pid, slots, h] = (new[:, h] / s).to(E4M3)


def gathered(cache, scale, table_row, length):
    """fp64 [length, H, 128] of one sequence and which of its keys lie in pages that exist."""
    pages, page = cache.shape[:2]
    out = torch.zeros(length, cache.shape[2], cache.shape[3], dtype=torch.float64)
    there = torch.zeros(length, dtype=torch.bool)
    for at in range(-(-length // page)):
        pid = int(table_row[at])
        if not 0 <= pid < pages:
            continue
        n = min(page, length - at * page)
        x = cache[pid, :n].double()
        if scale is not None:
            x = x * scale[pid].double()[None, :, None]
        out[at * page:at * page + n] = x
        there[at * page:at * page + n] = True
    return out, there


def attend(q, k_cache, v_cache, k_scale, v_scale, table, lens, cu, scale, causal):
    """(out, lse, weight): fp64 by definition; `weight` is softmax applied to |v|, what errors of the probabilities scale with."""
    T, Hq, D = q.shape
    H = k_cache.shape[2]
    group = Hq // H
    out = torch.zeros(T, Hq, D, dtype=torch.float64)
    mag = torch.zeros(T, Hq, D, dtype=torch.float64)
    lse = torch.full((Hq, T), -math.inf, dtype=torch.float64)
    page, width = k_cache.shape[1], table.shape[1]
    for b in range(table.shape[0]):
        lo, hi = int(cu[b]), int(cu[b + 1])
        n, length = hi - lo, min(max(int(lens[b]), 0), page * width)
        if n == 0:
            continue
        k, there = gathered(k_cache, k_scale, table[b], length)
        v, _ = gathered(v_cache, v_scale, table[b], length)
        j = torch.arange(length)
        visible = there[None, :].expand(n, length).clone()
        if causal:
            visible &= j[None, :] <= (int(lens[b]) - n + torch.arange(n))[:, None]
        for h in range(Hq):
            if length == 0:
                continue
            s = (q[lo:hi, h].double() @ k[:, h // group].T) * scale
            s = s.masked_fill(~visible, -math.inf)
            top = s.amax(-1, keepdim=True)
            p = torch.exp(s - top.masked_fill(top == -math.inf, 0.0))
            total = p.sum(-1, keepdim=True)
            w = p / total.clamp(min=1e-300)
            out[lo:hi, h] = w @ v[:, h // group]
            mag[lo:hi, h] = w @ v[:, h // group].abs()
            lse[h, lo:hi] = (top + total.log())[:, 0]
    return out, lse, mag


def make_cache(gen, pages, page, heads, dtype, eight, heads_first=True):
    """A pool with something everywhere, slots that no sequence owns included."""
    shape = (pages, heads, page, 128) if heads_first else (pages, page, heads, 128)
    x = torch.randn(shape, generator=gen)
    if not eight:
        pool, scale = x.to(dtype), None
    else:
        scale = torch.exp2(torch.randint(-9, -5, (pages, heads), generator=gen).float())
        x = x / (scale[:, :, None, None] if heads_first else scale[:, None, :, None])
        pool = x.clamp(-448, 448).to(E4M3)
    return (pool.transpose(1, 2) if heads_first else pool), scale


def make_tables(gen, lens, page, pages, width=None):
    """Pages of a random order, none used twice; entries that no token needs name no page."""
    used = [-(-max(n, 0) // page) for n in lens]
    width = max(max(used), 1) if width is None else width
    order = torch.randperm(pages, generator=gen).int()
    table = torch.full((len(lens), width), -1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(used):
        table[b, :n] = order[at:at + n]
        at += n
    assert at <= pages
    return table
