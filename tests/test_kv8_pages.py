"""Whose the pages of the paged 8-bit cache are: the plain form of kv8_plan with shared pages, and its refusals on the host."""

from __future__ import annotations

import ctypes

import numpy as np
import pytest

import kv8_plain as plain
from test_kv8 import ODD, P, plan_args


class Pages(ctypes.Structure):  # include/lfm25_hip.h
    _fields_ = [("shared", ctypes.c_void_p), ("held", ctypes.c_void_p)]


def plan(past, counts, table, ring, cursor, rows, page, shared=None, held=None):
    """(table, ring, row_starts, slots, cursor, status, held) after the call: requests one after another, each page of each by
    itself. Apart from kv8_plain.plan, which it has to agree with where nothing is shared and no length has gone back."""
    table, ring, old = table.copy(), ring.copy(), ring.copy()
    n, width = table.shape
    shared = np.zeros(n, int) if shared is None else shared
    sound = cursor[0] >= 0 and 0 <= cursor[1] - cursor[0] <= len(ring)
    free = [old[i % len(ring)] for i in range(cursor[0], cursor[1])] if sound else []
    room = len(ring) - len(free) if sound else -1  # what may be given back
    taken = given = 0
    short = full = False  # the first that the pool cannot serve leaves all behind it without pages
    starts, slots, status, kept = [0], [], [], []
    for b in range(n):
        p, c, first = int(past[b]), int(counts[b]), int(shared[b])
        own = -(-p // page) if held is None else int(held[b])
        new = max(c, 0)
        kept.append(own)
        starts.append(starts[-1] + new)
        mine = [-1] * new
        if p < 0 or not -(-p // page) <= own <= width or not 0 <= first <= width or (c > 0 and p < first * page):
            status.append(1)
        elif c < 0:
            pages = [table[b, j] for j in range(first, own)]
            full = full or (len(pages) > 0 and given + len(pages) > room)
            if full and pages:
                status.append(4)
            else:
                for q in pages:
                    ring[(cursor[1] + given) % len(ring)] = q
                    given += 1
                kept[-1] = 0
                status.append(0)
        elif -(-(p + c) // page) > width:
            status.append(2)
        elif c and starts[-1] > rows:
            status.append(8)
        else:
            need = max(-(-(p + c) // page) - own, 0)
            short = short or need > len(free) - taken
            if need and short:
                status.append(4)
            else:
                for j in range(need):
                    table[b, own + j] = free[taken]
                    taken += 1
                kept[-1] += need
                mine = [table[b, q // page] * page + q % page for q in range(p, p + c)]
                status.append(0)
        slots += mine
    slots = np.array((slots + [-1] * rows)[:rows], np.int64)
    slots[slots < 0] = -1
    return (table, ring, np.minimum(np.array(starts), 2 ** 31 - 1), slots, np.array([cursor[0] + taken, cursor[1] + given]),
            np.array(status), np.array(kept))


@pytest.mark.parametrize("seed", range(30))
def test_plain_forms_agree_where_nothing_is_shared(seed):
    rng = np.random.default_rng(seed)
    n, width, page, pages = 9, 7, 16, 40
    past, counts = rng.integers(-1, 100, n), rng.integers(-1, 40, n)
    table, ring = rng.integers(0, 99, (n, width)), rng.integers(0, 99, pages)
    taken = int(rng.integers(0, 1000))
    cursor = np.array([taken, taken + rng.integers(0, pages + 1)])
    args = past, counts, table, ring, cursor, int(rng.integers(1, 200)), page
    for a, b in zip(plan(*args), plain.plan(*args)):
        assert np.array_equal(a, b)


def test_plain_shared_pages_by_hand():
    """Two requests with a page of the first's: the second ends, then the first, and every page is in the ring once."""
    table = np.array([[7, 1, -1], [7, 2, -1], [-1, -1, -1]])
    ring, cursor, shared = np.array([3, 4, 5, 6, 0, 8, 9, 10]), np.array([0, 2]), np.array([0, 1, 0])
    out = plan(np.array([20, 20, 0]), np.array([1, -1, 0]), table, ring, cursor, 1, 16, shared)
    assert out[1].tolist() == [3, 4, 2, 6, 0, 8, 9, 10] and out[4].tolist() == [0, 3] and out[5].tolist() == [0, 0, 0]
    out = plan(np.array([21, 0, 0]), np.array([-1, 0, 0]), out[0], out[1], out[4], 1, 16, shared)
    assert out[1][:5].tolist() == [3, 4, 2, 7, 1] and out[4].tolist() == [0, 5]
    out = plan(np.array([20, 15, 0]), np.array([0, 1, 1]), table, ring, cursor, 9, 16, np.array([3, 1, 4]))
    assert out[5].tolist() == [0, 1, 1] and (out[3] == -1).all()  # a new row among shared pages; more of them than the row holds


def test_plain_lengths_that_go_back_by_hand():
    """Drafts of three rows of which some are kept: the second page is taken once and given back once."""
    table, ring, cursor, held, past = np.array([[0, -1, -1, -1]]), np.array([1, 2, 3, 4, 5]), np.array([0, 4]), np.array([1]), 15
    for kept in (1, 0, 1, 1, 3):
        out = plan(np.array([past]), np.array([3]), table, ring, cursor, 3, 16, held=held)
        table, ring, cursor, held, past = out[0], out[1], out[4], out[6], past + kept
        assert table.tolist() == [[0, 1, -1, -1]] and cursor.tolist() == [1, 4] and held.tolist() == [2] and out[5].tolist() == [0]
    out = plan(np.array([past]), np.array([-1]), table, ring, cursor, 1, 16, held=held)
    assert out[1].tolist() == [1, 2, 3, 4, 0] and out[4].tolist() == [1, 6] and out[5].tolist() == [0] and out[6].tolist() == [0]
    out = plan(np.array([17]), np.array([1]), table, ring, cursor, 1, 16, held=np.array([1]))
    assert out[5].tolist() == [1] and out[6].tolist() == [1]  # less than the length takes


def test_plan_with_refuses(lab):
    lib = lab.load_library()
    call, stream = plan_args()
    assert lab.ops._PLAN_PAGES.size == ctypes.sizeof(Pages)
    for pages, message in ((None, b"null"), (bytes(Pages(shared=ODD)), b"misaligned"), (bytes(Pages(held=ODD)), b"misaligned")):
        assert lib.lfm25_kv8_plan_with(call, pages, stream) == lab._lib.LFM25_EINVAL
        assert message in lib.lfm25_last_error()
    assert lib.lfm25_kv8_plan_with(None, bytes(Pages()), stream) == lab._lib.LFM25_EINVAL and b"null" in lib.lfm25_last_error()
    assert lib.lfm25_kv8_plan_with(plan_args(page=48)[0], bytes(Pages(shared=P)), stream) == lab._lib.LFM25_EINVAL
    assert b"page" in lib.lfm25_last_error()
