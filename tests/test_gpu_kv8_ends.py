"""The paged 8-bit cache's attention at the ends of what it takes: the longest contexts, the most requests and KV heads."""

from __future__ import annotations

import numpy as np
import pytest
import torch

import kv8_plain as plain
from test_gpu_kv8 import FORMATS, attend, bf16, check_append, check_attention, empty_cache, host, host_cache, ints, make_case, rows_of

pytestmark = pytest.mark.gpu
MOST = 2 ** 31 - 65536  # positions that are attended to


@pytest.mark.parametrize("rows,first", [(4, MOST - 2), (4, 2 ** 31 - 300), (20, MOST - 18)])
def test_attention_over_the_longest_table(gpu, lab, rows, first):
    """A row of the table that stands for nearly 2^31 positions. All but the last pages that count are one page whose scores
    are about -760 (e^-760 is 0 in FP32): rows up to the last position attend to the others, those behind it are NaN and
    reported."""
    page, dim, kv = 256, 64, 1
    width, last = 2 ** 31 // page - 1, MOST // page - 2
    rng = np.random.default_rng(1)
    c = make_case(1, [0], [2 * page], kv, 1, dim, page, torch.int8)
    cache = [t[torch.from_numpy(host(c["table"])[0, :2]).cuda()].contiguous() for t in c["cache"]]
    cache[0][0] = -127
    cache[2][0] = 1.0
    table = torch.zeros(1, width, dtype=torch.int32, device="cuda")
    table[0, last:] = 1
    q = bf16(rng.uniform(0.5, 1.0, size=(rows, kv, dim))).cuda()
    status = ints([0])
    got = attend(lab.ops, c, status, cache=cache, table=table, past=ints([first]), starts=ints([0, rows]), q=q, rows=rows, heads=kv,
                 max_rows=rows).double().cpu().numpy()
    counted = max(0, min(rows, MOST - first))
    assert host(status)[0] == lab.ops.KV8_BAD_PAGE and np.isnan(got[counted:]).all() and not np.isnan(got[:counted]).any()
    k, v, ks, vs = host_cache(cache)
    want, reach = plain.attention(q[:counted].double().cpu().numpy(), k, v, ks, vs, np.array([[1, 1]]), [first - last * page], [0, counted],
                                  dim ** -0.5)
    assert (np.abs(got[:counted] - want) <= reach).all()


@pytest.mark.parametrize("n,prompts,width", [(1000, 0, None), (4096, 0, None), (1000, 3, None), (4096, 40, 60)])
def test_attention_of_many_requests(gpu, lab, n, prompts, width):
    """Up to the most requests, single tokens or prompts among them, and requests that rest."""
    rng = np.random.default_rng(n + prompts)
    past, counts = rng.integers(0, 40, n), rng.integers(0, 3, n)
    past[[0, n // 3, n - 1]] = 500, 900, 200
    counts[rng.permutation(n)[:prompts]] = rng.integers(9, 60, prompts)
    check_attention(lab.ops, make_case(n, past, counts, 1, 2, 64, 16, FORMATS[prompts % 2], width=width, pad=3))


@pytest.mark.parametrize("kv,group,dim,page", [(256, 1, 64, 16), (256, 1, 128, 16), (96, 16, 64, 16), (7, 13, 128, 32)])
@pytest.mark.parametrize("counts,width", [([1, 2], None), ([1, 30], None), ([2, 1], 200), ([20, 1], 200)])
def test_attention_of_many_heads(gpu, lab, kv, group, dim, page, counts, width):
    check_attention(lab.ops, make_case(kv, [33, 70], counts, kv, group, dim, page, FORMATS[group % 2], width=width))


@pytest.mark.parametrize("n,width", [(1, 3), (1, 600), (5, 3), (5, 600), (100, 3), (100, 600), (300, 600)])
@pytest.mark.parametrize("max_rows", [1, 64])
def test_attention_of_requests_that_all_rest(gpu, lab, n, width, max_rows):
    """No request has new rows: everything is left as it was."""
    c = make_case(1, [40] * n, [0] * n, 2, 2, 64, 16, torch.int8, width=width, pad=70)
    status = ints([0])
    assert (attend(lab.ops, c, status, max_rows=max_rows) == 7.0).all() and host(status)[0] == 0


@pytest.mark.parametrize("dtype", FORMATS)
@pytest.mark.parametrize("kv,dim,page,rows", [(256, 128, 256, 300), (256, 64, 16, 40), (1, 64, 16, 9000)])
def test_append_of_many_heads_and_rows(gpu, lab, dtype, kv, dim, page, rows):
    rng = np.random.default_rng(rows)
    cache = empty_cache(rows // page + 3, kv, page, dim, dtype)
    k, v = rows_of(rng, rows, kv, dim, 2)
    check_append(lab.ops, cache, k, v, ints(5 + np.arange(rows)))
    check_append(lab.ops, cache, k[:3] * 16, v[:3] * 16, ints(5 + rows + np.arange(3)))
