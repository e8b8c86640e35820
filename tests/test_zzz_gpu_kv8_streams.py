"""The 8-bit paged cache in a captured graph, on another stream and on two at once.

In a file of its own, after all others: once two streams beside the default one have run anything (an addition of torch's
will do), the persistent decode of the same process finds its blocks off the XCDs that it relies on, reports that and stops.
"""

import numpy as np
import pytest
import torch

from test_gpu_kv8 import FORMATS, attend, empty_cache, ints, make_case

pytestmark = pytest.mark.gpu


def test_two_streams(gpu, lab):
    """Calls on two streams at once, each with tensors of its own, give what they give alone."""
    cases = [make_case(s, past, counts, 4, 2, 64, 64, f) for s, f in ((1, FORMATS[0]), (2, FORMATS[1]))
             for past, counts in (([2000, 900], [60, 1]), ([3000, 5, 70], [1, 2, 1]))]
    alone = [attend(lab.ops, c) for c in cases]
    streams = [torch.cuda.current_stream(), torch.cuda.Stream()]
    outs = [torch.full_like(a, 7.0) for a in alone]
    torch.cuda.synchronize()
    for _ in range(5):
        for i, (c, o) in enumerate(zip(cases, outs)):
            with torch.cuda.stream(streams[i // 2]):
                attend(lab.ops, c, out=o)
    torch.cuda.synchronize()
    for a, o in zip(alone, outs):
        assert torch.equal(a, o)


def test_a_pass_on_another_stream(gpu, lab):
    """A pass on a stream that is not the default one: what it gives on the default one."""
    ops, n, page, kv, dim = lab.ops, 3, 32, 2, 64
    g = torch.Generator(device="cuda").manual_seed(3)
    x = torch.randn(90, 8 * dim, generator=g, device="cuda").to(torch.bfloat16)

    def one():
        cache = empty_cache(20, kv, page, dim, torch.int8)
        table, ring, cursor = ints([[-1] * 6] * n), ints(range(20)), ints([0, 20], torch.int64)
        past, starts, slots, status = ints([0] * n), ints([0] * (n + 1)), ints([0] * 90), ints([0] * n)
        out = torch.full((90, 4, dim), 7.0, dtype=torch.bfloat16, device="cuda")
        ops.kv8_plan(past, ints([40, 1, 45]), table, ring, cursor, starts, slots, cursor, status, page=page)
        q, k, v = x.split([4 * dim, 2 * dim, 2 * dim], dim=1)
        ops.kv8_append(k.view(90, kv, dim), v.view(90, kv, dim), slots, *cache)
        ops.kv8_attention(q.view(90, 4, dim), *cache, table, past, starts, out, max_rows=45)
        return out, table, slots, cache[0]

    want = one()
    torch.cuda.synchronize()
    with torch.cuda.stream(torch.cuda.Stream()):
        got = one()
    torch.cuda.synchronize()
    assert not bool((want[0][:86] == 7.0).all()) and bool((want[0][86:] == 7.0).all())
    for a, b in zip(want, got):
        assert torch.equal(a, b)


def test_a_captured_pass(gpu, lab):
    """Plan, append and attention in one graph, replayed as the lengths go on: every replay against the eager calls on a
    second pool, with other work between."""
    ops, page, kv, dim, n = lab.ops, 16, 2, 64, 3
    pools = []
    for _ in range(2):
        pools.append(dict(cache=empty_cache(30, kv, page, dim, torch.int8), table=ints(np.full((n, 9), -1)), ring=ints(np.arange(30)),
                          cursor=ints([0, 30], torch.int64), past=ints(np.zeros(n)), counts=ints([1] * n), starts=ints(np.zeros(n + 1)),
                          slots=ints(np.zeros(40)), status=ints(np.zeros(n)), qkv=torch.zeros(40, 8 * dim, dtype=torch.bfloat16, device="cuda"),
                          out=torch.zeros(40, 4, dim, dtype=torch.bfloat16, device="cuda")))

    def one(p):
        ops.kv8_plan(p["past"], p["counts"], p["table"], p["ring"], p["cursor"], p["starts"], p["slots"], p["cursor"], p["status"], page=page)
        q, k, v = p["qkv"].split([4 * dim, 2 * dim, 2 * dim], dim=1)
        ops.kv8_append(k.view(40, kv, dim), v.view(40, kv, dim), p["slots"], *p["cache"])
        ops.kv8_attention(q.view(40, 4, dim), *p["cache"], p["table"], p["past"], p["starts"], p["out"], max_rows=40)

    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        one(pools[0])
    g = torch.Generator(device="cuda").manual_seed(1)
    for counts in ([30, 1, 0], [1, 1, 9], [1, 20, 1], [1, 1, 1], [0, 0, 3], [11, 1, 1]):
        qkv = torch.randn(40, 8 * dim, generator=g, device="cuda").to(torch.bfloat16)
        for p in pools:
            p["qkv"].copy_(qkv), p["counts"].copy_(ints(counts)), p["out"].fill_(7.0)
        graph.replay()
        one(pools[1])
        torch.cuda.synchronize()
        for name in ("out", "table", "slots", "starts", "cursor", "status", "ring"):
            assert torch.equal(pools[0][name], pools[1][name]), name
        for a, b in zip(pools[0]["cache"], pools[1]["cache"]):
            assert torch.equal(a.view(torch.int8) if a.dtype == torch.int8 else a.nan_to_num(-1), b.view(torch.int8) if b.dtype == torch.int8 else b.nan_to_num(-1))
        for p in pools:
            p["past"].add_(p["counts"])
