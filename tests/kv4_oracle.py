"""Plain float64 restatement of the 4-bit cache's calls, element by element position.

Independent of the kernels' code: numpy on the CPU, one formula per element.
"""
from __future__ import annotations

import numpy as np

BLOCK = 32
GROUP = 64


def _half(x, up):
    """The FP16 neighbour of float64 values not below (up) / not above them."""
    h = np.asarray(x, np.float64).astype(np.float16)
    off = h.astype(np.float64) < x if up else h.astype(np.float64) > x
    return np.where(off, np.nextafter(h, np.float16(np.inf if up else -np.inf)), h).astype(np.float64)


def quantise(x):
    """(codes, step, minimum) of rows x [..., d] in float64: codes [..., d], scales [..., d / 64]."""
    x = np.asarray(x, np.float64)
    g = x.reshape(*x.shape[:-1], x.shape[-1] // GROUP, GROUP)
    bad = ~np.isfinite(g).all(-1)
    g = np.clip(np.where(bad[..., None], 0.0, g), -65504.0, 65504.0)
    low = _half(g.min(-1), up=False)
    step = _half((g.max(-1) - low) / 15, up=True)
    codes = np.where(step[..., None] > 0,
                     np.rint((g - low[..., None]) / np.where(step > 0, step, 1.0)[..., None]), 0.0)
    step, low = np.where(bad, np.nan, step), np.where(bad, np.nan, low)
    return np.where(bad[..., None], 0.0, codes).reshape(x.shape), step, low


def values(x):
    """What the cache holds for rows x."""
    codes, step, low = quantise(x)
    c = codes.reshape(*step.shape, GROUP)
    return (c * step[..., None] + low[..., None]).reshape(codes.shape)


def positions(d):
    """Byte and shift of every element's key and value code, and byte of its scales: each [32, d]."""
    r, c = np.meshgrid(np.arange(BLOCK), np.arange(d), indexing="ij")
    g, e, ng = c // GROUP, c % GROUP, d // GROUP
    key = r * (d // 2) + 8 * ng * (e // 16) + 8 * g + (e % 16) // 2
    value = (16 * d + (r // 2) * d + 8 * ng * (e // 8) + 8 * g + 4 * ((e % 8) // 4) + 2 * (r % 2)
             + (e % 4) // 2)
    key_scale = 32 * d + 4 * ((g * 8 + r % 8) * 4 + r // 8)
    value_scale = 34 * d + 64 * g + 2 * ((r % 8) // 2 * 8 + r // 16 * 4 + (r % 16) // 8 * 2 + r % 2)
    return key, value, 4 * (c % 2), key_scale, value_scale


def entry_of(k, v):
    """The entry [36 d] of a block's keys and values [32, d]."""
    d = k.shape[-1]
    entry = np.zeros(36 * d, np.uint8)
    key, value, shift, key_scale, value_scale = positions(d)
    halves = entry.view(np.float16)
    for x, at, scale, low_at in ((k, key, key_scale, 2), (v, value, value_scale, d)):
        codes, step, low = quantise(x)
        np.bitwise_or.at(entry, at, (codes.astype(np.uint8) << shift).astype(np.uint8))
        with np.errstate(invalid="ignore"):
            halves[scale // 2] = np.repeat(step, GROUP, -1).astype(np.float16)
            halves[(scale + low_at) // 2] = np.repeat(low, GROUP, -1).astype(np.float16)
    return entry


def read_entry(entry):
    """(keys, values, |key| bounds, |value| bounds) [32, d] in float64 of an entry [36 d]."""
    d = entry.shape[-1] // 36
    key, value, shift, key_scale, value_scale = positions(d)
    halves = np.ascontiguousarray(entry).view(np.float16).astype(np.float64)
    kc = (entry[key] >> shift) & 15
    vc = (entry[value] >> shift) & 15
    ks, km = halves[key_scale // 2], halves[key_scale // 2 + 1]
    vs, vm = halves[value_scale // 2], halves[(value_scale + d) // 2]
    with np.errstate(invalid="ignore", over="ignore"):
        return ks * kc + km, vs * vc + vm, ks * kc + np.abs(km), vs * 15 + np.abs(vm)


def plan(add, lens, table, free, top, max_tokens):
    """One step, request by request: (slots, positions, cu, lens, table, free, top, refused)."""
    lens, table, free = lens.copy(), table.copy(), free.copy()
    n, width = table.shape
    slots, where = np.full(max_tokens, -1, np.int64), np.zeros(max_tokens, np.int64)
    cu, refused, taken, wanted, back = [0], [], 0, 0, []
    for b in range(n):
        grow = max(int(add[b]), 0)
        after = max(int(lens[b]) + int(add[b]), 0)
        held, want = -(-int(lens[b]) // BLOCK), -(-after // BLOCK)
        why = "table" if want > width else "slots" if grow and cu[-1] + grow > max_tokens else None
        if why is None:
            need = max(want - held, 0)
            wanted += need
            if need and wanted > top:
                why = "pool"
        if why is None:
            for j in range(held, want):
                table[b, j] = free[top - 1 - taken]
                taken += 1
            back += [int(table[b, j]) for j in range(want, held)]
        refused.append(why)
        for i in range(min(grow, max_tokens)):
            at, p = cu[-1] + i, int(lens[b]) + i
            if at < max_tokens:
                where[at] = p
                if why is None:
                    slots[at] = int(table[b, p // BLOCK]) * BLOCK + p % BLOCK
        if why is None:
            lens[b] = after
        cu.append(cu[-1] + grow)
    base = top - taken
    for r, block in enumerate(back):
        free[base + len(back) - 1 - r] = block
    return slots, where, np.array(cu), lens, table, free, base + len(back), refused


def attention(q, pool, table, lens, scale, selected=None, counts=None):
    """float64 (out, lse, tolerance parts) of q [B, T, QH, D]; pool uint8 [P, KH, 36 D].

    The third and fourth results are, per row, the largest sum of |q| |k| * scale over
    the tokens it sees (the size of what a logit is summed from) and the largest |v| part.
    """
    n, new, qh, d = q.shape
    kh = pool.shape[1]
    out = np.zeros(q.shape)
    lse = np.full(q.shape[:-1], -np.inf)
    logit, size = np.zeros(q.shape[:-1]), np.zeros(q.shape[:-1])
    for b in range(n):
        length = int(lens[b])
        blocks = -(-length // BLOCK)
        if blocks == 0 or length < 0 or blocks > table.shape[1]:
            continue
        for h in range(kh):
            ids = list(range(blocks))
            if selected is not None:
                group = h // (kh // selected.shape[1])
                ids = [int(x) for x in selected[b, group, :int(counts[b, group])]] + [blocks - 1]
            ids = [i for i in ids if 0 <= table[b, i] < pool.shape[0]]
            if not ids:
                continue
            parts = [read_entry(pool[table[b, i], h]) for i in ids]
            k, v, ka, va = (np.concatenate([p[j] for p in parts]) for j in range(4))
            where = (np.array(ids)[:, None] * BLOCK + np.arange(BLOCK)).reshape(-1)
            for i in range(new):
                sees = where <= length - new + i
                if not sees.any():
                    continue
                for a in range(h * (qh // kh), (h + 1) * (qh // kh)):
                    row = q[b, i, a].astype(np.float64)
                    x = scale * (k[sees] @ row)
                    top = x.max()
                    p = np.exp(x - top)
                    out[b, i, a] = p @ v[sees] / p.sum()
                    lse[b, i, a] = top + np.log(p.sum())
                    logit[b, i, a] = abs(scale) * (ka[sees] @ np.abs(row)).max()
                    size[b, i, a] = va[sees].max()
    return out, lse, logit, size
