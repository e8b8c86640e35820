"""The paged 8-bit KV cache in plain 64-bit numpy: what lfm25_kv8_plan, lfm25_kv8_append and lfm25_kv8_attention are
held to. Written from the definitions, position by position and page by page."""

from __future__ import annotations

import numpy as np
import torch

MOST = {torch.int8: 127.0, torch.float8_e4m3fn: 448.0}
LARGEST = 1.875 * 2.0 ** 127


def plan(past, counts, table, ring, cursor, rows, page):
    """(table, ring, row_starts, slots, cursor, status) after the call; requests one after another."""
    table, ring = table.copy(), ring.copy()
    width, taken, given = table.shape[1], int(cursor[0]), int(cursor[1])
    sound = taken >= 0 and 0 <= given - taken <= len(ring)
    free = given - taken if sound else 0
    took = gave = asked = offered = 0
    old = ring.copy()
    starts, slots, status = [0], np.full(rows, -1, np.int64), []
    for b, (p, c) in enumerate(zip(past.tolist(), counts.tolist())):
        at = starts[-1]
        starts.append(at + max(c, 0))
        held = -(-p // page)
        if p < 0 or held > width:
            status.append(1)
        elif c < 0:
            offered += held
            if held and (not sound or free + offered > len(ring)):
                status.append(4)
                continue
            for j in range(held):
                ring[(given + gave) % len(ring)] = table[b, j]
                gave += 1
            status.append(0)
        else:
            after = -(-(p + c) // page)
            if after > width:
                status.append(2)
                continue
            if c and starts[-1] > rows:
                status.append(8)
                continue
            asked += after - held
            if after > held and asked > free:
                status.append(4)
                continue
            for j in range(held, after):
                table[b, j] = old[(taken + took) % len(ring)]
                took += 1
            for i in range(c):
                slots[at + i] = table[b, (p + i) // page] * page + (p + i) % page
            status.append(0)
    slots[slots < 0] = -1
    return table, ring, np.minimum(np.array(starts), 2 ** 31 - 1), slots, np.array([taken + took, given + gave]), np.array(status)


def round_codes(v, dtype):
    if dtype == torch.int8:
        return np.clip(np.rint(v), -127, 127)
    a = np.abs(v)
    e = np.floor(np.log2(np.where(a > 0, a, 1.0)))
    step = np.exp2(np.maximum(e, -6) - 3)
    return np.copysign(np.minimum(np.rint(a / step) * step, 448.0), v)


def scale_for(largest, dtype):
    e = -120
    while largest > MOST[dtype] * 2.0 ** e:
        e += 1
    return 2.0 ** e


def append(x, slots, codes, scales, dtype):
    """codes float64 [pages, kv, page, dim], scales float64 [pages, kv] after rows x float64 [rows, kv, dim]; in place."""
    pages, kv, page, dim = codes.shape
    r = 0
    while r < len(slots):
        slot = int(slots[r])
        if not 0 <= slot < pages * page:
            r += 1
            continue
        n = 1
        while r + n < len(slots) and slots[r + n] == slot + n and (slot + n) % page:
            n += 1
        p, off = slot // page, slot % page
        for h in range(kv):
            new = x[r: r + n, h]
            old = scales[p, h] if off else 0.0
            if not np.isfinite(new).all() or np.isnan(old):
                scales[p, h] = np.nan
                codes[p, h, off: off + n] = 0
                continue
            s = max(old, scale_for(np.abs(new).max(), dtype))
            if off and s > old:
                codes[p, h, :off] = round_codes(codes[p, h, :off] * (old / s), dtype)
            codes[p, h, off: off + n] = round_codes(np.clip(new, -LARGEST, LARGEST) / s, dtype)
            scales[p, h] = s
        r += n


def attention(q, keys, values, ks, vs, table, past, starts, scale):
    """(out, reach) float64 [rows, heads, dim] and the bound of the kernels' error; NaN in rows behind the last request's.
    keys, values float64 codes [pages, kv, page, dim], ks, vs their scales.

    The bound, with p the normalized probabilities, eps = 2^-24 the half step of FP32 and L positions: a score is a sum of
    dim exact products in FP32 (each partial sum off by 2 eps of the sum of magnitudes A, an adder that truncates included)
    and four more roundings, so log2(p) is off by (2 dim + 8) eps A log2(e) and p, with the exponential's own 2 eps, by
    r = (2 dim + 8) eps A + 2 eps of itself; numerator and denominator are sums of at most L such terms in FP32 (2 L eps).
    p is rounded to BF16, each by its own d with |d| <= 2^-8, in the numerator and in the sum alike, which is off by the mean
    m = sum p d: (sum p (1 + d) v) / (1 + m) - o = sum p d (v - o) / (1 + m), at most 2^-8 (A_v + |o|) / (1 - 2^-8) with A_v =
    sum p |v| (the 1.01 has the divisor). The factor that takes a value scale out of the sum again is rounded too (2^-8 |o|,
    and |o| <= A_v) where it is no power of two (`exact_scales` has them all powers); the result is rounded to BF16 once more.
    What falls below FP32's smallest normal number, 2^-126, may become 0: a probability (before the division by their sum,
    which is 1 or more, since the largest is 1), its product with a value, the result. That is at most 2^-126 (|v| + 1) for
    each position and 2^-126 once."""
    rows, heads, dim = q.shape
    kv, page = keys.shape[1], keys.shape[2]
    group = heads // kv
    out, reach = np.full(q.shape, np.nan), np.zeros(q.shape)
    exact_scales = all((np.frexp(s[np.isfinite(s) & (s > 0)])[0] == 0.5).all() for s in (ks, vs))
    eps = 2.0 ** -24
    for b, p0 in enumerate(np.asarray(past).tolist()):
        r0, r1 = int(starts[b]), int(starts[b + 1])
        for r in range(r0, r1):
            length = p0 + (r - r0) + 1
            if length <= 0:
                out[r] = 0.0
                continue
            ids = table[b, : -(-length // page)]
            for h in range(kv):
                k = (keys[ids, h] * ks[ids, h][:, None, None]).reshape(-1, dim)[:length]
                v = (values[ids, h] * vs[ids, h][:, None, None]).reshape(-1, dim)[:length]
                x = q[r, h * group: (h + 1) * group]
                s = x @ k.T * scale
                size = np.abs(x) @ np.abs(k).T * scale
                e = np.exp(s - s.max(1, keepdims=True))
                p = e / e.sum(1, keepdims=True)
                o, a = p @ v, p @ np.abs(v)
                rel = (2 * dim + 8) * eps * size.max(1, keepdims=True) + 2 * eps + 2 * length * eps
                out[r, h * group: (h + 1) * group] = o
                step = 2.0 ** -8 * (1 if exact_scales else 2)
                reach[r, h * group: (h + 1) * group] = ((step + 2 * rel) * a + 2.0 ** -8 * np.abs(o)) * 1.01 + \
                    2.0 ** -8 * (np.abs(o) + step * a) + 2.0 ** -126 * (1 + length * (1 + np.abs(v).max()))
    return out, reach
