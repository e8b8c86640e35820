"""Pages of the 8-bit cache that several requests have, and lengths that go back: kv8_plan with `shared` and `held` against the
plain form, and a server's life cycle in which no page may be lost or have two owners."""

from __future__ import annotations

import numpy as np
import pytest
import torch

import kv8_plain as cells
import test_kv8_pages as plain
from test_gpu_kv8 import FORMATS, bf16, check_attention, empty_cache, host, host_cache, ints, random_plan

pytestmark = pytest.mark.gpu


def run_plan(ops, past, counts, table, ring, cursor, rows, page, in_place=False, **pages):
    n = len(past)
    t, f, c = ints(table), ints(ring), ints(cursor, torch.int64)
    starts, slots, status = ints(np.full(n + 1, -7)), ints(np.full(rows, -7)), ints(np.full(n, -7))
    following = c if in_place else ints([-7, -7], torch.int64)
    extra = {k: ints(v) for k, v in pages.items()}
    ops.kv8_plan(ints(past), ints(counts), t, f, c, starts, slots, following, status, page=page, **extra)
    return [host(x) for x in (t, f, starts, slots, following, status)], {k: host(v) for k, v in extra.items()}


SIZES = [(0, 1, 64, 4, 150, 9, 0), (2, 16, 64, 17, 900, 40, 0), (3, 300, 16, 40, 300, 900, 11), (4, 1000, 32, 70, 2000, 4000, 5000),
         (5, 1025, 128, 9, 900, 2000, 1), (6, 4096, 16, 12, 100, 9000, 77), (8, 64, 32, 20, 500, 30, 0), (9, 333, 16, 30, 400, 200, 0)]


@pytest.mark.parametrize("seed,n,page,width,longest,spare,slack", SIZES)
@pytest.mark.parametrize("in_place", [False, True])
def test_plan_with_shared_pages(gpu, lab, seed, n, page, width, longest, spare, slack, in_place):
    past, counts, table, ring, cursor = random_plan(seed, n, page, width, longest, spare, ended=0.3)
    rng = np.random.default_rng(seed)
    shared = np.where(rng.random(n) < 0.5, rng.integers(-1, width + 2, n), 0)
    rows = max(1, int(np.maximum(counts, 0).sum()) + slack)
    args = past, counts, table, ring, cursor, rows, page
    for g, w in zip(run_plan(lab.ops, *args, in_place=in_place, shared=shared)[0], plain.plan(*args, shared=shared)):
        assert np.array_equal(g, w)
    for g, w in zip(run_plan(lab.ops, *args, in_place=in_place, shared=np.zeros(n, int))[0], plain.plan(*args)):
        assert np.array_equal(g, w)


@pytest.mark.parametrize("seed,n,page,width,longest,spare,slack", SIZES)
@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("both", [False, True])
def test_plan_with_held_pages(gpu, lab, seed, n, page, width, longest, spare, slack, in_place, both):
    past, counts, table, ring, cursor = random_plan(seed, n, page, width, longest, spare, ended=0.3)
    rng = np.random.default_rng(seed)
    held = np.minimum(-(-past // page), width)
    past = np.where(rng.random(n) < 0.5, rng.integers(0, past + 1), past)  # lengths that have gone back
    held = np.where(rng.random(n) < 0.05, rng.integers(-1, width + 2, n), held)
    shared = {"shared": np.where(rng.random(n) < 0.3, rng.integers(0, 3, n), 0)} if both else {}
    ring = np.concatenate([ring, np.full(n * width, -9)])  # (as many as could come back)
    cursor = np.array([3, 3 + spare])
    ring[3: 3 + spare] = rng.permutation(spare) + 10 ** 6
    rows = max(1, int(np.maximum(counts, 0).sum()) + slack)
    args = past, counts, table, ring, cursor, rows, page
    (got, pages), want = run_plan(lab.ops, *args, in_place=in_place, **shared, held=held), plain.plan(*args, **shared, held=held)
    for g, w in zip(got + [pages["held"]], want):
        assert np.array_equal(g, w)


class Server:
    """A pool with one sequence of plan calls on it; every page is in the ring or one request's own at all times."""

    def __init__(self, ops, requests, width, pages, page):
        self.ops, self.page, self.pages, self.n = ops, page, pages, requests
        self.table, self.ring = ints(np.full((requests, width), -1)), ints(np.random.default_rng(0).permutation(pages))
        self.cursor = ints([0, pages], torch.int64)
        self.past, self.extra = np.zeros(requests, np.int64), {"shared": ints(np.zeros(requests)), "held": ints(np.zeros(requests))}

    def step(self, counts, kept=None):
        """One pass; of a request's new rows, `kept` stay."""
        counts = np.asarray(counts)
        rows = max(1, int(np.maximum(counts, 0).sum()))
        starts, slots, status = ints(np.zeros(self.n + 1)), ints(np.zeros(rows)), ints(np.zeros(self.n))
        past = ints(self.past)
        self.ops.kv8_plan(past, ints(counts), self.table, self.ring, self.cursor, starts, slots, self.cursor, status, page=self.page, **self.extra)
        assert not host(status).any()
        self.past = np.where(counts < 0, 0, self.past + (counts if kept is None else np.asarray(kept)))
        self.pass_ = past, starts, slots, rows
        self.check()

    def owned(self):
        shared, held = host(self.extra["shared"]), host(self.extra["held"])
        assert (held >= -(-self.past // self.page)).all()
        return [int(p) for b in range(self.n) for p in host(self.table)[b, shared[b]: max(shared[b], held[b])]]

    def check(self):
        c = host(self.cursor)
        free = host(self.ring)[np.arange(c[0], c[1]) % self.pages].tolist()
        assert sorted(free + self.owned()) == list(range(self.pages))

    def fork(self, to, of, pages):
        """Request `to` begins with the first pages of request `of`."""
        self.table[to, :pages] = self.table[of, :pages]
        self.extra["shared"][to] = self.extra["held"][to] = pages
        self.past[to] = pages * self.page


def test_a_shared_beginning(gpu, lab):
    """One request's pages as the beginning of three others, which grow and end in any order, and whose rows others take: no
    page goes to the ring before its owner ends, none twice."""
    s = Server(lab.ops, 5, 12, 40, 16)
    s.step([70, 5, 0, 0, 0])
    s.fork(2, 0, 4)
    s.fork(3, 0, 2)
    s.step([1, 1, 30, 1, 0])
    s.fork(4, 0, 4)
    s.step([0, -1, 1, 50, 2])
    s.step([0, 20, -1, 1, 1])
    s.extra["shared"][2] = 0
    s.step([1, 1, 33, -1, 1])
    s.extra["shared"][3] = 0
    first = host(s.table)[0, :4].tolist()
    for _ in range(3):
        s.step([0, 1, 1, 9, 17])
        assert host(s.table)[4, :4].tolist() == first
    s.step([0, 1, 1, 1, -1])
    s.step([-1, 1, 1, 1, 0])
    s.extra["shared"][4] = 0
    s.step([-1, -1, -1, -1, -1])
    assert not s.owned() and host(s.cursor)[1] - host(s.cursor)[0] == 40


def test_rejected_drafts(gpu, lab):
    """Passes of a few rows of which some are kept, across page borders, beside a prompt and requests that end: no page is lost."""
    s = Server(lab.ops, 4, 6, 17, 16)
    s.step([15, 31, 0, 5])
    rng = np.random.default_rng(1)
    for _ in range(12):
        s.step([3, 4, 0, 1], kept=[int(rng.integers(0, 3)), int(rng.integers(0, 3)), 0, 1])
    assert len(s.owned()) <= 10
    s.step([1, -1, 80, 1])
    s.step([5, 20, 1, -1], kept=[0, 20, 1, 0])
    s.past[2] = 0  # all the way back
    s.step([1, 1, 0, 33])
    s.step([0, 1, 70, 1])
    s.step([-1, -1, -1, -1])
    assert not s.owned()


@pytest.mark.parametrize("dtype", FORMATS)
def test_attention_over_a_shared_beginning(gpu, lab, dtype):
    """A second request goes on from the first's pages after a third has ended and its pages have gone round: it reads what
    the first wrote."""
    page, kv, dim, rng = 16, 2, 64, np.random.default_rng(3)
    s = Server(lab.ops, 3, 8, 14, page)
    cache = empty_cache(14, kv, page, dim, dtype)

    def one(counts):
        s.step(counts)
        past, starts, slots, rows = s.pass_
        k, v = (bf16(rng.normal(size=(rows, kv, dim))).cuda() for _ in range(2))
        lab.ops.kv8_append(k, v, slots, *cache)
        return dict(cache=cache, table=s.table, past=past, starts=starts, q=bf16(rng.normal(size=(rows, 2 * kv, dim))).cuda(), rows=rows,
                    heads=2 * kv, dim=dim, page=page, max_rows=max(1, max(counts)))

    one([35, 0, 20])
    s.fork(1, 0, 2)
    check_attention(lab.ops, one([1, 20, 1]))
    one([0, -1, -1])
    s.extra["shared"][1] = 0
    check_attention(lab.ops, one([1, 60, 0]))
    s.fork(2, 0, 2)
    check_attention(lab.ops, one([1, 1, 18]))
    check_attention(lab.ops, one([1, 1, 1]))


@pytest.mark.parametrize("dtype", FORMATS)
def test_attention_after_rejected_drafts(gpu, lab, dtype):
    """What was rejected is written over: each pass reads what was kept and its own rows, in pages that stay the request's."""
    page, kv, dim, rng = 16, 2, 64, np.random.default_rng(4)
    s = Server(lab.ops, 2, 8, 9, page)
    cache = empty_cache(9, kv, page, dim, dtype)
    model = [np.zeros((9, kv, page, dim)), np.zeros((9, kv, page, dim)), np.zeros((9, kv)), np.zeros((9, kv))]
    for counts, kept in (([14, 30], [14, 30]), ([4, 3], [1, 0]), ([4, 3], [1, 3]), ([4, 3], [4, 1]), ([1, 5], [0, 0]), ([3, 2], [3, 2])):
        s.step(counts, kept)
        past, starts, slots, rows = s.pass_
        k, v = (bf16(rng.normal(size=(rows, kv, dim)) * np.exp2(rng.integers(-2, 3, (rows, 1, 1)))).cuda() for _ in range(2))
        lab.ops.kv8_append(k, v, slots, *cache)
        cells.append(k.double().cpu().numpy(), host(slots), model[0], model[2], dtype)
        cells.append(v.double().cpu().numpy(), host(slots), model[1], model[3], dtype)
        for got, want in zip(host_cache(cache), model):  # of the positions that have been written
            used = np.isfinite(got) & (want != 0)
            assert np.array_equal(got[used], want[used])
        check_attention(lab.ops, dict(cache=cache, table=s.table, past=past, starts=starts, q=bf16(rng.normal(size=(rows, 2 * kv, dim))).cuda(),
                                      rows=rows, heads=2 * kv, dim=dim, page=page, max_rows=max(counts)))


def test_plan_refuses_other_shared(gpu, lab):
    args = (np.zeros(3, int), np.ones(3, int), np.full((3, 2), -1), np.arange(6), np.array([0, 6]), 3, 16)
    for bad in (np.zeros(2), np.zeros(4)):
        for name in ("shared", "held"):
            with pytest.raises(ValueError, match=name):
                run_plan(lab.ops, *args, **{name: bad})
    with pytest.raises(ValueError, match="shared"):
        lab.ops.kv8_plan(*[ints(a) for a in args[:4]], ints(args[4], torch.int64), ints(np.zeros(4)), ints(np.zeros(3)),
                         ints([0, 0], torch.int64), ints(np.zeros(3)), page=16, shared=torch.zeros(3, dtype=torch.int32))


@pytest.mark.parametrize("n", [64, 65, 256, 257, 600, 1024, 1025, 2000, 4096])
@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("seed", [1, 2])
def test_plan_refuses_single_requests_of_large_batches(gpu, lab, n, in_place, seed):
    """Every reason among requests that a thread has several of: bad lengths, past the table, past the rows, a short pool."""
    past, counts, table, ring, cursor = random_plan(seed, n, 32, 8, 220, 2 * n, ended=0.2, bad=0.2)
    rng = np.random.default_rng(seed)
    past = np.where(rng.random(n) < 0.1, 8 * 32 + rng.integers(1, 9, n), past)
    counts = np.where(rng.random(n) < 0.1, 0, counts)
    wanted = np.maximum(counts, 0).sum()
    for rows in (max(1, int(wanted) - 3 * n), int(wanted) + 5):
        args = past, counts, table, ring, cursor, rows, 32
        for g, w in zip(run_plan(lab.ops, *args, in_place=in_place)[0], plain.plan(*args)):
            assert np.array_equal(g, w)
