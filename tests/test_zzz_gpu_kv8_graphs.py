"""The 8-bit paged cache in captured graphs that hold a workspace, the combination of parts and the second launch for slots.

Runs among the last files, as test_zzz_gpu_kv8_streams.py does and for its reason: a capture works on a stream of its own."""

import numpy as np
import pytest
import torch

from test_gpu_kv8 import FORMATS, empty_cache, ints

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", FORMATS)
@pytest.mark.parametrize("rows,width,group,steps", [
    (50, 700, 2, ([40, 1, 0], [1, 1, 40], [30, 15, 5], [1, 1, 1], [0, 0, 50])),            # tiles and single tokens in parts
    (3, 700, 4, ([3, 0, 0], [1, 1, 1], [0, 2, 1], [1, 1, 1])),                             # single tokens only, in parts
    (8300, 700, 2, ([8190, 1, 0], [1, 1, 30], [1, 1, 1], [100, 50, 8000]))])               # slots in a launch of their own
def test_a_captured_pass_over_a_wide_table(gpu, lab, dtype, rows, width, group, steps):
    ops, page, kv, dim, n, pages = lab.ops, 32, 1, 64, 3, 700
    assert lab.load_library().lfm25_kv8_attention_workspace_bytes(rows, kv * group, kv, dim, n, rows, width, page) > 0
    heads = kv * group
    pools = []
    for _ in range(2):
        pools.append(dict(cache=empty_cache(pages, kv, page, dim, dtype), table=ints(np.full((n, width), -1)), ring=ints(np.arange(pages)),
                          cursor=ints([0, pages], torch.int64), past=ints(np.zeros(n)), counts=ints([0] * n), starts=ints(np.zeros(n + 1)),
                          slots=ints(np.zeros(rows)), status=ints(np.zeros(n)), held=ints(np.zeros(n)), bits=ints([0]),
                          qkv=torch.zeros(rows, (heads + 2 * kv) * dim, dtype=torch.bfloat16, device="cuda"),
                          out=torch.zeros(rows, heads, dim, dtype=torch.bfloat16, device="cuda")))

    def one(p):
        ops.kv8_plan(p["past"], p["counts"], p["table"], p["ring"], p["cursor"], p["starts"], p["slots"], p["cursor"], p["status"], page=page,
                     held=p["held"])
        q, k, v = p["qkv"].split([heads * dim, kv * dim, kv * dim], dim=1)
        ops.kv8_append(k.view(rows, kv, dim), v.view(rows, kv, dim), p["slots"], *p["cache"])
        ops.kv8_attention(q.view(rows, heads, dim), *p["cache"], p["table"], p["past"], p["starts"], p["out"], max_rows=rows, status=p["bits"])

    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        one(pools[0])
    g = torch.Generator(device="cuda").manual_seed(rows)
    for counts in steps:
        qkv = torch.randn(rows, (heads + 2 * kv) * dim, generator=g, device="cuda").to(torch.bfloat16)
        for p in pools:
            p["qkv"].copy_(qkv), p["counts"].copy_(ints(counts)), p["out"].fill_(7.0)
        graph.replay()
        one(pools[1])
        torch.cuda.synchronize()
        total = sum(counts)
        assert not pools[0]["status"].any() and not pools[0]["bits"].any()
        assert (pools[0]["out"][total:] == 7.0).all() and not (pools[0]["out"][:total] == 7.0).all(2).any()
        for name in ("out", "table", "slots", "starts", "cursor", "ring", "held"):
            assert torch.equal(pools[0][name], pools[1][name]), name
        for a, b in zip(pools[0]["cache"], pools[1]["cache"]):
            assert torch.equal(a.view(torch.int8) if a.element_size() == 1 else a.nan_to_num(-1), b.view(torch.int8) if b.element_size() == 1 else b.nan_to_num(-1))
        for p in pools:
            p["past"].add_(p["counts"])


def test_two_graphs_of_one_memory_pool(gpu, lab):
    """Two passes captured into graphs that share their memory, workspaces included, replayed in turn: each gives what its calls
    give eagerly."""
    from test_gpu_kv8 import attend, make_case
    cases = [make_case(s, past, counts, 2, 2, 64, 64, f, width=400)
             for s, past, counts, f in ((1, [3000, 900], [60, 1], FORMATS[0]), (2, [2500, 5, 700], [1, 2, 1], FORMATS[1]))]
    want = [attend(lab.ops, c) for c in cases]
    outs, graphs = [torch.full_like(w, 7.0) for w in want], [torch.cuda.CUDAGraph() for _ in cases]
    for i, (c, o) in enumerate(zip(cases, outs)):
        with torch.cuda.graph(graphs[i], pool=graphs[0].pool() if i else None):
            attend(lab.ops, c, out=o)
    for _ in range(4):
        for i in (0, 1, 1, 0):
            outs[i].fill_(7.0)
            graphs[i].replay()
            assert torch.equal(outs[i], want[i])
        assert torch.equal(attend(lab.ops, cases[0]), want[0])
