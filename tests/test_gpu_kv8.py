"""The paged 8-bit KV cache on the GPU against its plain 64-bit forms: pages, slots and codes exactly, the attention within
the bound that kv8_plain.attention derives."""

from __future__ import annotations

import numpy as np
import pytest
import torch

import kv8_plain as plain

pytestmark = pytest.mark.gpu
FORMATS = [torch.int8, torch.float8_e4m3fn]
NAN_CODE = {torch.int8: -128, torch.float8_e4m3fn: 0x7f}


def ints(v, dtype=torch.int32):
    return torch.tensor(np.asarray(v).astype(np.int64), dtype=dtype, device="cuda")


def host(t):
    return t.cpu().numpy().astype(np.int64)


# ---------------------------------------------------------------- plan

def run_plan(ops, past, counts, table, ring, cursor, rows, page, in_place=False):
    n = len(past)
    t, f, c = ints(table), ints(ring), ints(cursor, torch.int64)
    starts, slots, status = ints(np.full(n + 1, -7)), ints(np.full(rows, -7)), ints(np.full(n, -7))
    following = c if in_place else ints([-7, -7], torch.int64)
    ops.kv8_plan(ints(past), ints(counts), t, f, c, starts, slots, following, status, page=page)
    if not in_place:
        assert host(c).tolist() == list(cursor)
    return [host(x) for x in (t, f, starts, slots, following, status)]


def random_plan(seed, n, page, width, longest, spare, ended=0.1, bad=0.0):
    rng = np.random.default_rng(seed)
    past = rng.integers(0, longest + 1, n)
    counts = np.where(rng.random(n) < 0.5, 1, rng.integers(0, 4 * page, n))
    counts[rng.random(n) < ended] = -1
    past[rng.random(n) < bad] = -rng.integers(1, 9)
    counts[rng.random(n) < bad] = width * page + 5
    held = np.minimum(-(-np.maximum(past, 0) // page), width)
    total = int(held.sum()) + spare
    order = rng.permutation(total)
    table, k = np.full((n, width), -1), 0
    for b, h in enumerate(held):
        table[b, :h] = order[k: k + h]
        k += h
    taken = int(rng.integers(0, 10 ** 11))
    ring = np.full(total, -5)
    ring[(taken + np.arange(spare)) % total] = order[k:]
    return past, counts, table, ring, np.array([taken, taken + spare])


@pytest.mark.parametrize("seed,n,page,width,longest,spare,slack", [
    (0, 1, 64, 4, 150, 9, 0), (1, 1, 16, 1, 0, 1, 3), (2, 16, 64, 17, 900, 40, 0), (3, 300, 16, 40, 300, 900, 11),
    (4, 1000, 32, 70, 2000, 4000, 5000), (5, 1025, 128, 9, 900, 2000, 1), (6, 4096, 16, 12, 100, 9000, 77),
    (7, 50, 256, 3, 500, 0, 0), (8, 64, 32, 20, 500, 30, 0), (9, 333, 16, 30, 400, 200, 0)])
@pytest.mark.parametrize("in_place", [False, True])
def test_plan(gpu, lab, seed, n, page, width, longest, spare, slack, in_place):
    """Ragged lengths, pools that run short (the last three), rings that have gone round, requests that end."""
    past, counts, table, ring, cursor = random_plan(seed, n, page, width, longest, spare)
    rows = max(1, int(np.maximum(counts, 0).sum()) + slack)
    want = plain.plan(past, counts, table, ring, cursor, rows, page)
    got = run_plan(lab.ops, past, counts, table, ring, cursor, rows, page, in_place)
    for g, w in zip(got, want):
        assert np.array_equal(g, w)
    assert (got[5] == 4).any() == (seed >= 7)


@pytest.mark.parametrize("seed", range(4))
def test_plan_refuses_single_requests(gpu, lab, seed):
    """Negative and overlong lengths, rows past the end: each refused with its reason, the others served."""
    past, counts, table, ring, cursor = random_plan(20 + seed, 200, 32, 8, 220, 500, bad=0.1)
    counts[counts > 8 * 32] = np.where(np.arange((counts > 8 * 32).sum()) % 2, 2 ** 31 - 1, 8 * 32)
    past[3], counts[3] = 8 * 32 + 1, -1
    past[4], counts[4] = 2 ** 31 - 1, 2 ** 31 - 1
    rows = 700
    want = plain.plan(past, counts, table, ring, cursor, rows, 32)
    for g, w in zip(run_plan(lab.ops, past, counts, table, ring, cursor, rows, 32), want):
        assert np.array_equal(g, w)
    assert {0, 1, 2} <= set(want[5].tolist())


def test_plan_reports_rows_past_the_end(gpu, lab):
    past, counts = np.zeros(3, int), np.array([4, 5, 0])
    args = (past, counts, np.full((3, 1), -1), np.arange(5), np.array([0, 5]), 8, 16)
    got = run_plan(lab.ops, *args)
    assert got[5].tolist() == [0, 8, 0] and got[3].tolist() == [0, 1, 2, 3, -1, -1, -1, -1] and got[4].tolist() == [1, 5]
    for g, w in zip(got, plain.plan(*args)):
        assert np.array_equal(g, w)


@pytest.mark.parametrize("cursor", [[5, 4], [-1, 2], [0, 7], [-3, -1]])
def test_plan_takes_a_false_cursor_for_an_empty_pool(gpu, lab, cursor):
    args = (np.array([16, 16, 3]), np.array([1, -1, 1]), np.array([[0], [1], [2]]), np.arange(6), np.array(cursor), 3, 16)
    args[2].resize(3, 1)
    table = np.concatenate([args[2], np.full((3, 1), -1)], 1)
    args = args[:2] + (table,) + args[3:]
    got = run_plan(lab.ops, *args)
    assert got[5].tolist() == [4, 4, 0] and got[4].tolist() == cursor and got[3].tolist() == [-1, 2 * 16 + 3, -1]
    for g, w in zip(got, plain.plan(*args)):
        assert np.array_equal(g, w)


# ---------------------------------------------------------------- append

def empty_cache(pages, kv, page, dim, dtype, fill=None):
    """A pool whose bytes and scales are garbage: NaN scales, and NaN codes where the format has them."""
    code = NAN_CODE[dtype] if fill is None else fill
    k = torch.full((pages, kv, page, dim), code, dtype=torch.int8, device="cuda")
    v = torch.full((pages, kv, dim, page), code, dtype=torch.int8, device="cuda")
    s = torch.full((2, pages, kv), float("nan"), device="cuda")
    return [k.view(dtype), v.view(dtype), s[0], s[1]]


def host_cache(cache):
    """float64 codes [pages, kv, page, dim] and scales of keys and of values."""
    k, v, ks, vs = cache
    return [k.float().cpu().numpy().astype(np.float64), v.float().cpu().numpy().astype(np.float64).transpose(0, 1, 3, 2).copy(),
            ks.cpu().numpy().astype(np.float64), vs.cpu().numpy().astype(np.float64)]


def bf16(v):
    return torch.tensor(v, dtype=torch.float32).to(torch.bfloat16)


def check_append(ops, cache, keys, values, slots):
    want = host_cache(cache)
    dtype = cache[0].dtype
    ops.kv8_append(keys, values, slots, *cache)
    s = slots.cpu().numpy()
    plain.append(keys.double().cpu().numpy(), s, want[0], want[2], dtype)
    plain.append(values.double().cpu().numpy(), s, want[1], want[3], dtype)
    for g, w in zip(host_cache(cache), want):
        assert np.array_equal(g, w, equal_nan=True)


def rows_of(rng, rows, kv, dim, spread, apart=0):
    """Keys and values as slices of one wider product, of sizes that differ by row."""
    size = np.exp2(rng.integers(-spread, spread + 1, (rows, 1)))
    x = bf16(rng.normal(size=(rows, 2 * kv * dim + apart)) * size).cuda()
    return x[:, apart: apart + kv * dim].view(rows, kv, dim), x[:, apart + kv * dim:].view(rows, kv, dim)


@pytest.mark.parametrize("dtype", FORMATS)
@pytest.mark.parametrize("page,kv,dim", [(16, 1, 64), (32, 3, 64), (64, 8, 64), (64, 2, 128), (128, 2, 64), (256, 1, 128), (16, 5, 128)])
def test_append(gpu, lab, dtype, page, kv, dim):
    """Passes of one row, a few, and many onto requests that grow: scales that rise over what a page holds, runs that begin
    and end inside pages and segments, pages of no order, rows without a slot between."""
    rng = np.random.default_rng(page + kv + dim)
    pages = 40
    order = rng.permutation(pages)
    cache = empty_cache(pages, kv, page, dim, dtype)
    held = [0, 0, 0, 0]
    free = 0
    table = [[] for _ in held]
    for counts in ([1, 0, 7, page], [1, 3, 1, 1], [9, page + 1, 0, 1], [1, 1, 1, 2], [0, 0, 0, 0], [2 * page + 5, 8, 17, 1], [1, 1, 1, 1]):
        slots = []
        for b, c in enumerate(counts):
            for pos in range(held[b], held[b] + c):
                if pos // page == len(table[b]):
                    table[b].append(order[free])
                    free += 1
                slots.append(table[b][pos // page] * page + pos % page)
            held[b] += c
            slots += [-1] * (b % 2)
        slots += [pages * page, 2 ** 31 - 1, -2 ** 31]
        k, v = rows_of(rng, len(slots), kv, dim, 3, apart=8)
        check_append(lab.ops, cache, k, v, ints(slots))


@pytest.mark.parametrize("dtype", FORMATS)
@pytest.mark.parametrize("rows", [1, 7, 8, 511, 513, 1500])
def test_append_row_counts(gpu, lab, dtype, rows):
    """Both groupings of rows into blocks, and runs that begin in one block's rows and end in another's."""
    rng = np.random.default_rng(rows)
    cache = empty_cache(rows // 64 + 2, 2, 64, 64, dtype)
    k, v = rows_of(rng, rows, 2, 64, 1)
    check_append(lab.ops, cache, k.contiguous(), v.contiguous(), ints(3 + np.arange(rows)))


def test_append_decode_batch(gpu, lab):
    rng = np.random.default_rng(5)
    cache = empty_cache(300, 8, 64, 64, torch.int8, fill=3)
    cache[2].fill_(2.0 ** -6), cache[3].fill_(2.0 ** -3)
    k, v = rows_of(rng, 300, 8, 64, 2)
    slots = rng.permutation(300) * 64 + rng.integers(0, 64, 300)
    check_append(lab.ops, cache, k, v, ints(slots))


@pytest.mark.parametrize("dtype", FORMATS)
def test_append_values_at_the_edges(gpu, lab, dtype):
    """Zeros, subnormals, the largest BF16, powers of two at the codes' border, ties."""
    most = 3.3895313892515355e38
    rows = [np.zeros(64), np.full(64, 2.0 ** -133), np.full(64, -2.0 ** -126), np.full(64, most), np.linspace(-127, 127, 64),
            np.linspace(-448, 448, 64), np.full(64, 127.5), np.full(64, 449.0), np.arange(64) + 0.5, np.exp2(np.arange(64) - 40.0),
            np.r_[most, np.ones(63)], -np.arange(64) / 8]
    x = bf16(np.array(rows)[:, None, :]).cuda()
    for i in range(len(rows)):  # each alone on a page's beginning, then all pairs after one another
        check_append(lab.ops, empty_cache(1, 1, 16, 64, dtype), x[i: i + 1], -x[i: i + 1], ints([0]))
        for j in range(len(rows)):
            cache = empty_cache(1, 1, 16, 64, dtype)
            check_append(lab.ops, cache, x[i: i + 1], x[j: j + 1], ints([0]))
            check_append(lab.ops, cache, x[j: j + 1], x[i: i + 1], ints([1]))


@pytest.mark.parametrize("dtype", FORMATS)
@pytest.mark.parametrize("what", [float("nan"), float("inf"), -float("inf")])
def test_append_of_what_is_not_finite(gpu, lab, dtype, what):
    """The page's scale for that head is NaN until the page begins anew; other heads, pages and the other cache keep theirs."""
    rng = np.random.default_rng(2)
    cache = empty_cache(3, 2, 32, 64, dtype)
    k, v = rows_of(rng, 40, 2, 64, 1)
    check_append(lab.ops, cache, k, v, ints(np.arange(40)))
    k, v = k.clone(), v.clone()
    k[2, 1, 63] = what
    check_append(lab.ops, cache, k[:5], v[:5], ints(40 + np.arange(5)))
    assert cache[2][1, 1].isnan() and cache[2][:2].isnan().sum() == 1 and not cache[3][:2].isnan().any()
    check_append(lab.ops, cache, k[5:6], v[5:6], ints([45]))
    assert cache[2][1, 1].isnan()
    check_append(lab.ops, cache, k[6:8], v[6:8], ints([32, 33]))
    assert not cache[2][1, 1].isnan()


@pytest.mark.parametrize("dtype", FORMATS)
def test_append_in_steps_keeps_within_a_step(gpu, lab, dtype):
    """A page filled one position at a time, values rising so that its scale grows again and again: every value within one
    int8 step of the final scale (half a step, a quarter, an eighth, ... at the moves between scales), or FP8's half step and,
    below its normal range, as much of the subnormal step."""
    rng = np.random.default_rng(3)
    cache = empty_cache(1, 2, 64, 64, dtype)
    x = bf16(rng.normal(size=(64, 2, 64)) * np.exp2(np.arange(64) / 6.0)[:, None, None]).cuda()
    for r in range(64):
        lab.ops.kv8_append(x[r: r + 1], x[r: r + 1], ints([r]), *cache)
    k, v, ks, vs = host_cache(cache)
    assert np.array_equal(k, v) and np.array_equal(ks, vs)
    got, true = k[0] * ks[0][:, None, None], x.double().cpu().numpy().transpose(1, 0, 2)
    step = ks[0][:, None, None] * (1.0 if dtype == torch.int8 else 2.0 ** -9)
    allowed = step if dtype == torch.int8 else np.maximum(step, 2.0 ** -4 * np.abs(true) * (1 + 2.0 ** -4) + step)
    assert (np.abs(got - true) <= allowed).all()


# ---------------------------------------------------------------- attention

def make_case(seed, past, counts, kv, group, dim, page, dtype, spare=2, pad=0, stretch=1.0, width=None, powers=True):
    """A cache that holds every request's positions (garbage elsewhere), the pass's tensors, and host copies."""
    rng = np.random.default_rng(seed)
    past, counts = np.asarray(past), np.asarray(counts)
    n, heads = len(past), kv * group
    held = np.maximum(-(-(past + counts) // page), 0)
    pages = int(held.sum()) + spare
    order = rng.permutation(pages)
    width = int(held.max()) + 1 if width is None else width
    table, k = rng.choice([-1, 2 ** 30, pages], (n, width)), 0  # what is not held is no page
    codes = [np.full((pages, kv, page, dim), NAN_CODE[dtype], np.int64) for _ in range(2)]
    scales = [np.full((pages, kv), np.nan) for _ in range(2)]
    for b in range(n):
        table[b, : held[b]] = order[k: k + held[b]]
        for j, p in enumerate(order[k: k + held[b]]):
            live = min(page, past[b] + counts[b] - j * page)
            for c in codes:
                c[p, :, :live] = rng.integers(-127, 128, (kv, live, dim)) if dtype == torch.int8 else rng.choice(
                    np.r_[0:0x7f, 0x80:0xff], (kv, live, dim))
            for i, s in enumerate(scales):
                s[p] = np.exp2(rng.integers(-7, -4, kv) - (0 if dtype == torch.int8 else 2)) * (1 if powers else rng.uniform(0.6, 1, kv))
        k += held[b]
    as8 = lambda c: torch.tensor(c.astype(np.uint8) if dtype != torch.int8 else c.astype(np.int8), device="cuda").view(dtype)  # noqa: E731
    cache = [as8(codes[0]), as8(codes[1].transpose(0, 1, 3, 2).copy()), torch.tensor(scales[0], dtype=torch.float32, device="cuda"),
             torch.tensor(scales[1], dtype=torch.float32, device="cuda")]
    starts = np.r_[0, np.cumsum(counts)]
    rows = int(starts[-1]) + pad
    q = bf16(rng.normal(size=(rows, heads * dim + 24)) * stretch).cuda()[:, 16: 16 + heads * dim].view(rows, heads, dim)
    return dict(cache=cache, table=ints(table), past=ints(past), starts=ints(starts), q=q, max_rows=max(1, int(counts.max())),
                page=page, dim=dim, rows=rows, heads=heads)


def attend(ops, c, status=None, out=None, **change):
    c = c | change
    if out is None:
        out = torch.full((c["rows"], c["heads"], c["dim"]), 7.0, dtype=torch.bfloat16, device="cuda")
    ops.kv8_attention(c["q"], *c["cache"], c["table"], c["past"], c["starts"], out, max_rows=c["max_rows"], status=status,
                      **({"scale": c["scale"]} if "scale" in c else {}))
    return out


def check_attention(ops, c, **change):
    c = c | change
    status = ints([0])
    got = attend(ops, c, status).double().cpu().numpy()
    k, v, ks, vs = host_cache(c["cache"])
    want, reach = plain.attention(c["q"].double().cpu().numpy(), k, v, ks, vs, host(c["table"]), host(c["past"]), host(c["starts"]),
                                  c.get("scale", c["dim"] ** -0.5))
    behind = np.isnan(want)
    assert (got[behind] == 7.0).all()
    far = np.abs(got - want)[~behind] > reach[~behind]
    assert not np.isnan(got).any() and not far.any(), (far.mean(), np.abs(got - want)[~behind].max(), reach[~behind].max())
    assert host(status)[0] == 0
    return got


@pytest.mark.parametrize("dtype", FORMATS)
@pytest.mark.parametrize("page,kv,group,dim", [(64, 8, 2, 64), (16, 2, 1, 64), (32, 1, 16, 64), (128, 2, 3, 64), (256, 4, 5, 64),
                                               (64, 2, 4, 128), (16, 3, 8, 128), (32, 1, 2, 128), (256, 1, 7, 128)])
def test_attention_of_single_tokens(gpu, lab, dtype, page, kv, group, dim):
    past = [0, 1, 15, 16, 17, 31, 32, 63, 64, 65, 255, 256, 257, 700, 1023, 1500]
    check_attention(lab.ops, make_case(page, past, [1] * len(past), kv, group, dim, page, dtype, pad=3))


@pytest.mark.parametrize("dtype", FORMATS)
@pytest.mark.parametrize("page,kv,group,dim", [(64, 2, 2, 64), (16, 1, 1, 64), (32, 1, 16, 64), (256, 2, 3, 64), (64, 1, 4, 128), (16, 1, 5, 128)])
def test_attention_of_few_rows(gpu, lab, dtype, page, kv, group, dim):
    """Rows x query heads up to and past the 16 columns of the single-token form, none, and first positions."""
    most = 16 // group
    past = [0, 0, 5, 62, 63, 64, 130, 200, 300, 7]
    counts = [1, most, most + 1, 1, most, most + 1, 0, 2, 2 * most + 3, 1]
    check_attention(lab.ops, make_case(group, past, counts, kv, group, dim, page, dtype, pad=2))


@pytest.mark.parametrize("dtype", FORMATS)
@pytest.mark.parametrize("page,kv,group,dim", [(64, 2, 2, 64), (16, 1, 1, 64), (128, 1, 3, 64), (32, 2, 4, 128), (64, 1, 16, 128), (256, 1, 1, 128)])
def test_attention_of_prompts(gpu, lab, dtype, page, kv, group, dim):
    check_attention(lab.ops, make_case(9, [0, 0, 33, 129, 0, 400], [200, 65, 64, 127, 0, 131], kv, group, dim, page, dtype, pad=4))


@pytest.mark.parametrize("dtype", FORMATS)
def test_attention_of_single_tokens_beside_a_prompt(gpu, lab, dtype):
    past = [300, 40, 0, 555, 17, 1000]
    check_attention(lab.ops, make_case(4, past, [1, 1, 150, 1, 1, 90], 4, 2, 64, 16, dtype))


@pytest.mark.parametrize("dtype", FORMATS)
@pytest.mark.parametrize("counts,dim,group", [([1, 3], 64, 2), ([2, 1], 128, 5), ([40, 1], 64, 2), ([33, 17], 128, 4)])
def test_attention_over_long_contexts(gpu, lab, dtype, counts, dim, group):
    """Divided over many blocks: more parts than the shorter request has units, and a table wider than either needs."""
    check_attention(lab.ops, make_case(1, [9000, 130], counts, 1, group, dim, 128, dtype, width=600))


@pytest.mark.parametrize("n,kv,dim", [(3, 2, 64), (64, 1, 64), (65, 1, 64), (200, 1, 64), (256, 1, 128), (257, 1, 64), (130, 2, 128)])
def test_attention_of_batches_of_uneven_lengths(gpu, lab, n, kv, dim):
    """One long context, short ones, requests that rest and one past its table, in parts found on the device."""
    rng = np.random.default_rng(n)
    past = rng.integers(0, 90, n)
    past[[0, n // 2, n - 1]] = [4000, 700, 2300]
    counts = rng.integers(1, 3, n)
    counts[1::7] = 0
    c = make_case(n, past, counts, kv, 2, dim, 32, torch.float8_e4m3fn, width=130)
    check_attention(lab.ops, c)
    k, v, ks, vs = host_cache(c["cache"])
    want, reach = plain.attention(c["q"].double().cpu().numpy(), k, v, ks, vs, host(c["table"]), past, host(c["starts"]), dim ** -0.5)
    starts, moved = host(c["starts"]), past.copy()
    moved[n // 2] = 5000  # past the table: NaN there, the others as before
    status = ints([0])
    got = attend(lab.ops, c, status, past=ints(moved)).double().cpu().numpy()
    mine = slice(starts[n // 2], starts[n // 2 + 1])
    assert np.isnan(got[mine]).all() and host(status)[0] == (lab.ops.KV8_BAD_PAGE if counts[n // 2] else 0)
    keep = np.ones(len(got), bool)
    keep[mine] = False
    assert (np.abs(got - want)[keep] <= reach[keep]).all()


def test_attention_of_long_contexts_beside_prompts(gpu, lab):
    for dim, n in ((64, 20), (128, 5), (64, 70), (128, 66)):
        past, counts = [60 * b for b in range(n)], [1] * n
        past[3], counts[1], counts[2], counts[n - 1] = 7000, 150, 0, 40
        check_attention(lab.ops, make_case(n, past, counts, 2, 2, dim, 64, torch.int8))


@pytest.mark.parametrize("counts", [[1, 1], [30, 30]])
def test_attention_of_peaked_and_flat_scores(gpu, lab, counts):
    for stretch, scale in ((40.0, 0.125), (1.0, 0.0), (1e-3, 1.0), (3e4, 2.0)):
        c = make_case(6, [500, 77], counts, 2, 2, 64, 64, torch.int8, stretch=stretch)
        check_attention(lab.ops, c, scale=scale)


@pytest.mark.parametrize("dtype", FORMATS)
@pytest.mark.parametrize("counts", [[1, 2, 1], [100, 1, 20]])
def test_attention_with_scales_of_any_value(gpu, lab, dtype, counts):
    check_attention(lab.ops, make_case(8, [200, 100, 0], counts, 2, 2, 64, 32, dtype, powers=False))


@pytest.mark.parametrize("counts,width", [([5, 1, 3], None), ([90, 50, 3], None), ([5, 1, 3], 200), ([90, 50, 3], 200)])
def test_attention_of_rows_that_see_nothing(gpu, lab, counts, width):
    """Positions before the first give zeros, those after it attend as ever."""
    c = make_case(3, [-2, -1, -7], counts, 2, 2, 64, 16, torch.int8, width=width)
    got = check_attention(lab.ops, c)
    assert (got[:2] == 0).all() and (got[counts[0]] == 0).all() and (got[-3:] == 0).all() and (got[2] != 0).any()


def nan_rows(c, bad):
    """Rows of output that must be NaN: those of request b that see position `bad[b]` or later."""
    past, starts = host(c["past"]), host(c["starts"])
    want = np.zeros(c["rows"], bool)
    for b, first in bad.items():
        for r in range(starts[b], starts[b + 1]):
            want[r] = past[b] + r - starts[b] >= first
    return want


@pytest.mark.parametrize("dtype", FORMATS)
@pytest.mark.parametrize("counts,width", [([3, 1, 1], None), ([80, 70, 1], None), ([3, 1, 1], 300), ([80, 70, 1], 300)])
@pytest.mark.parametrize("number", [-1, 9999, -2 ** 31, 2 ** 31 - 1])
def test_attention_with_a_page_outside_the_pool(gpu, lab, dtype, counts, width, number):
    """NaN for the rows that attend to it and no others, and a status bit."""
    c = make_case(5, [62, 20, 300], counts, 2, 2, 64, 64, dtype, width=width)
    c["table"][0, 1] = number
    status = ints([4])
    got = attend(lab.ops, c, status).float().isnan().cpu().numpy()
    assert host(status)[0] == 4 | 1
    want = nan_rows(c, {0: 64})
    assert (got.all((1, 2)) == want).all() and (got.any((1, 2)) == want).all()


@pytest.mark.parametrize("dtype", FORMATS)
@pytest.mark.parametrize("which", [2, 3])
@pytest.mark.parametrize("counts", [[3, 1], [90, 30]])
def test_attention_of_a_lost_page(gpu, lab, dtype, which, counts):
    """A NaN scale (what kv8_append leaves of a value that is not finite) reaches the rows that attend to its page in its
    head, and only those."""
    c = make_case(5, [30, 10], counts, 2, 2, 64, 32, dtype)
    c["cache"][which][host(c["table"])[0, 1], 1] = float("nan")
    got = attend(lab.ops, c).float().isnan().cpu().numpy()
    want = nan_rows(c, {0: 32})
    assert (got[:, 2:].all((1, 2)) == want).all() and (got[:, 2:].any((1, 2)) == want).all() and not got[:, :2].any()


@pytest.mark.parametrize("counts,width", [([6, 2], 2), ([100, 2], 2)])
def test_attention_past_the_table(gpu, lab, counts, width):
    c = make_case(5, [60, 3], counts, 2, 2, 64, 32, torch.int8)
    c["table"] = c["table"][:, :width].contiguous()
    status = ints([0])
    got = attend(lab.ops, c, status).float().isnan().cpu().numpy()
    want = nan_rows(c, {0: 64})
    assert (got.all((1, 2)) == want).all() and (got.any((1, 2)) == want).all() and host(status)[0] == 1


@pytest.mark.parametrize("starts,rows_left", [([0, 9, 12], [0]), ([0, 3, 40], [1]), ([5, 3, 6], [0]), ([-4, 2, 4], [0]), ([0, 12, 12], [0])])
def test_attention_refuses_rows_it_cannot_place(gpu, lab, starts, rows_left):
    """More than max_rows rows, offsets outside the rows or out of order: the request's rows are left, the others served."""
    c = make_case(5, [60, 300], [6, 6], 2, 2, 64, 64, torch.int8)
    status = ints([0])
    got = attend(lab.ops, c, status, starts=ints(starts), max_rows=8)
    assert host(status)[0] == 2
    for b in (0, 1):
        r0, r1 = max(starts[b], 0), min(starts[b + 1], 12)
        if b in rows_left:
            others = set(range(max(starts[1 - b], 0), min(starts[2 - b], 12)))
            assert all((got[r] == 7.0).all() for r in range(r0, r1) if r not in others)
        else:
            assert all((got[r] != 7.0).any() for r in range(r0, r1))


def test_attention_leaves_rows_behind_the_last(gpu, lab):
    c = make_case(5, [60, 300], [6, 60], 2, 2, 64, 64, torch.int8, pad=100)
    got = attend(lab.ops, c)
    assert (got[66:] == 7.0).all() and (got[:66] != 7.0).any((1, 2)).all()


@pytest.mark.parametrize("counts", [[1] * 5, [70, 1, 1, 33, 1]])
def test_attention_gives_the_same_bits_again(gpu, lab, counts):
    c = make_case(5, [600, 30, 4000, 0, 77], counts, 4, 2, 64, 64, torch.float8_e4m3fn)
    first = attend(lab.ops, c)
    for _ in range(3):
        assert torch.equal(attend(lab.ops, c), first)


@pytest.mark.parametrize("counts", [[1, 1], [64, 3]])
def test_cache_past_four_gigabytes(gpu, lab, counts):
    """Pages whose bytes lie past 2^32 in either cache."""
    pages, kv, page, dim = (1 << 32) // (8 * 64 * 64) + 40, 8, 64, 64
    cache = [torch.zeros(pages, kv, page, dim, dtype=torch.int8, device="cuda"), torch.zeros(pages, kv, dim, page, dtype=torch.int8, device="cuda"),
             torch.full((pages, kv), float("nan"), device="cuda"), torch.full((pages, kv), float("nan"), device="cuda")]
    rng = np.random.default_rng(0)
    far = pages - 1 - rng.permutation(30)
    past = np.array([640, 100])
    table = np.full((2, 16), -1)
    table[0], table[1, :3] = far[:16], far[16:19]
    total = past + counts
    slots = np.concatenate([table[b, np.arange(t) // page] * page + np.arange(t) % page for b, t in enumerate(total)])
    k, v = rows_of(rng, len(slots), kv, dim, 0)
    lab.ops.kv8_append(k, v, ints(slots), *cache)
    near = [torch.stack([t[int(p)] for p in far]) for t in cache]  # the same pages, as a small pool
    small = np.where(table >= 0, np.argsort(far)[np.searchsorted(np.sort(far), np.maximum(table, far.min()))], -1)
    q = bf16(rng.normal(size=(int(np.sum(counts)), 16, dim))).cuda()
    c = dict(cache=cache, table=ints(table), past=ints(past), starts=ints(np.r_[0, np.cumsum(counts)]), q=q, max_rows=max(counts),
             page=page, dim=dim, rows=len(q), heads=16)
    got = attend(lab.ops, c)
    c |= dict(cache=near, table=ints(small))
    assert torch.equal(got, attend(lab.ops, c))
    check_attention(lab.ops, c)
    assert not cache[0][: pages - 30].any() and cache[2][: pages - 30].isnan().all()


# ---------------------------------------------------------------- together

class Serving:
    """A small pool and its requests, driven by the three calls; the host keeps every key and value."""

    def __init__(self, ops, requests, width, pages, page, kv, group, dim, dtype, seed):
        self.ops, self.page, self.kv, self.group, self.dim, self.dtype = ops, page, kv, group, dim, dtype
        self.rng = np.random.default_rng(seed)
        self.cache = empty_cache(pages, kv, page, dim, dtype)
        self.table = ints(np.full((requests, width), -1))
        self.ring = ints(self.rng.permutation(pages))
        self.cursor = ints([0, pages], torch.int64)
        self.past, self.n = np.zeros(requests, np.int64), requests
        self.model = host_cache(self.cache)

    def step(self, counts, pad=0):
        counts = np.asarray(counts)
        rows = int(np.maximum(counts, 0).sum()) + pad
        past, c = ints(self.past), ints(counts)
        starts, slots, status = ints(np.zeros(self.n + 1)), ints(np.zeros(rows)), ints(np.zeros(self.n))
        self.ops.kv8_plan(past, c, self.table, self.ring, self.cursor, starts, slots, self.cursor, status, page=self.page)
        k, v = rows_of(self.rng, rows, self.kv, self.dim, 1)
        q = bf16(self.rng.normal(size=(rows, self.kv * self.group, self.dim))).cuda()
        out = torch.full((rows, self.kv * self.group, self.dim), 7.0, dtype=torch.bfloat16, device="cuda")
        self.ops.kv8_append(k, v, slots, *self.cache)
        self.ops.kv8_attention(q, *self.cache, self.table, past, starts, out, max_rows=max(1, int(counts.max())))
        assert not host(status).any()
        s = host(slots)
        plain.append(k.double().cpu().numpy(), s, self.model[0], self.model[2], self.dtype)
        plain.append(v.double().cpu().numpy(), s, self.model[1], self.model[3], self.dtype)
        want, reach = plain.attention(q.double().cpu().numpy(), *self.model, host(self.table), self.past, host(starts), self.dim ** -0.5)
        got = out.double().cpu().numpy()
        behind = np.isnan(want)
        assert (np.abs(got - want)[~behind] <= reach[~behind]).all() and (got[behind] == 7.0).all()
        for g, w in zip(host_cache(self.cache), self.model):
            assert np.array_equal(g, w, equal_nan=True)
        self.past = np.where(counts < 0, 0, self.past + counts)


@pytest.mark.parametrize("dtype", FORMATS)
@pytest.mark.parametrize("page,kv,group,dim", [(32, 2, 2, 64), (16, 1, 4, 128)])
def test_serving(gpu, lab, dtype, page, kv, group, dim):
    """Requests come, grow by prompts and single tokens, end, and others take their pages: against 64 bits at every step."""
    s = Serving(lab.ops, 4, 12, 24, page, kv, group, dim, dtype, seed=page)
    s.step([40, 0, 5, 0])
    s.step([1, 70, 1, 0], pad=3)
    for _ in range(3):
        s.step([1, 1, 1, 0])
    s.step([-1, 1, 30, 100])
    s.step([50, -1, 1, 1])
    s.step([1, 33, 1, 1])
    held = -(-s.past // page)
    c = host(s.cursor)
    assert c[1] - c[0] == 24 - held.sum()
    free = host(s.ring)[np.arange(c[0], c[1]) % 24].tolist()
    used = [int(p) for b in range(4) for p in host(s.table)[b, : held[b]]]
    assert sorted(free + used) == list(range(24))


def test_ops_refuse_gpu_tensors_of_other_shapes(gpu, lab):
    ops = lab.ops
    c = make_case(0, [30], [2], 2, 2, 64, 16, torch.int8)
    out = torch.zeros(2, 4, 64, dtype=torch.bfloat16, device="cuda")
    good = dict(query=c["q"], key_cache=c["cache"][0], value_cache=c["cache"][1], key_scales=c["cache"][2], value_scales=c["cache"][3],
                block_table=c["table"], past=c["past"], row_starts=c["starts"], output=out)
    ops.kv8_attention(**good, max_rows=2)
    for name, other in (("query", c["q"][:1]), ("query", c["q"].float()), ("query", c["q"].transpose(0, 1)), ("output", out[:, :3].contiguous()),
                        ("output", out[:, :, :32]), ("value_cache", c["cache"][0]), ("key_scales", c["cache"][2][:1]),
                        ("key_scales", c["cache"][2].double()), ("block_table", c["table"][0]), ("row_starts", c["starts"][:1]),
                        ("past", c["past"].long()), ("key_cache", c["cache"][0].float())):
        with pytest.raises(ValueError):
            ops.kv8_attention(**(good | {name: other}), max_rows=2)
    for change in (dict(max_rows=0), dict(max_rows=2, scale=-1.0), dict(max_rows=2, scale=float("nan")), dict(max_rows=2, status=c["past"].float())):
        with pytest.raises(ValueError):
            ops.kv8_attention(**good, **change)
    k = torch.zeros(4, 2, 64, dtype=torch.bfloat16, device="cuda")
    slots = ints(np.arange(4))
    odd = torch.zeros(2 * 4 * 132, dtype=torch.bfloat16, device="cuda").as_strided((4, 2, 64), (132, 64, 1))
    for keys, values, s in ((k[:3], k, slots), (k, k[:, :1], slots), (k, k.half(), slots), (k, k, slots.long()), (odd, k, slots), (k.transpose(1, 2), k, slots)):
        with pytest.raises(ValueError):
            ops.kv8_append(keys, values, s, *c["cache"])
    ops.kv8_append(k[:0], k[:0], slots[:0], *c["cache"])
    one = ints([0])
    two = ints([0, 0], torch.int64)
    for bad in ("counts", "cursor", "row_starts", "status", "slots", "block_table"):
        args = dict(past=one, counts=one, block_table=ints([[0]]), free_pages=one, cursor=two, row_starts=ints([0, 0]), slots=one, next_cursor=two, status=one)
        args[bad] = args[bad][:0]
        with pytest.raises(ValueError):
            ops.kv8_plan(**args, page=16)
