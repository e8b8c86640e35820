"""The paged 8-bit cache's attention at the ends of what it takes: the longest contexts, the most requests and KV heads."""

from __future__ import annotations

import numpy as np
import pytest
import torch

import kv8_plain as plain
from test_gpu_kv8 import FORMATS, attend, bf16, check_attention, host, host_cache, ints, make_case

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
