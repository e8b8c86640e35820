"""Value scales of the paged 8-bit KV cache that are far apart or no powers of two: what the attention makes of them."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from test_gpu_kv8 import FORMATS, attend, host, make_case

pytestmark = pytest.mark.gpu


def uniform_case(scale, past, counts, page, dtype, width=None, dim=64):
    """Scores that are all 0. A request's first page has value scale 1 and codes 0, the others `scale` and codes that rise with
    the dimension, the same at every position. With (the outputs in 64 bits, those too near a rounding border to be told)."""
    c = make_case(1, past, counts, 2, 2, dim, page, dtype, width=width)
    c["q"] = torch.zeros(c["rows"], c["heads"], dim, dtype=torch.bfloat16, device="cuda")
    codes = (torch.arange(dim, device="cuda") * 127 // dim + 1).float() if dtype == torch.int8 else torch.exp2(torch.arange(dim, device="cuda") / 8).to(dtype).float()
    table, starts = host(c["table"]), host(c["starts"])
    value, scales = c["cache"][1], c["cache"][3]
    want = np.zeros((c["rows"], c["heads"], dim))
    for b, p in enumerate(past):
        pages = -(-(p + counts[b]) // page)
        for j in range(pages):
            fill = codes * (j > 0)
            value[int(table[b, j])] = fill[None, :, None].expand(2, dim, page).to(dtype)
            scales[int(table[b, j])] = scale if j else 1.0
        for i in range(counts[b]):
            seen = p + i + 1
            want[starts[b] + i] = codes.double().cpu().numpy() * scale * max(seen - page, 0) / seen
    longest = max(p + n for p, n in zip(past, counts))
    # The scaled probability is a BF16 number (the scale is), so it is not rounded. Left are FP32's roundings: sums of `longest`
    # terms above and below, and a dozen factors, exponentials and logarithms, each off by 2^-23 at most.
    margin = (2 * longest + 12) * 2.0 ** -23
    low, high = (torch.tensor(want * (1 + s * margin)).to(torch.bfloat16) for s in (-1, 1))
    return c, low, high


@pytest.mark.parametrize("dtype", FORMATS)
@pytest.mark.parametrize("scale", [230 / 256, 255 / 256, 198 / 256, 240 / 1024])
@pytest.mark.parametrize("past,counts,page,width", [([200, 130], [1, 1], 64, None), ([300, 0], [40, 300], 64, None),
                                                    ([150, 20], [2, 1], 16, None), ([100, 30], [90, 70], 16, None),
                                                    ([900, 200], [1, 1], 64, 400), ([700, 30], [60, 1], 32, 200)])
def test_the_sum_takes_a_value_scale_out_in_fp32(gpu, lab, dtype, scale, past, counts, page, width):
    """A scale whose reciprocal is no BF16 number: the outputs are the rounded exact ones."""
    c, low, high = uniform_case(scale, past, counts, page, dtype, width)
    got = attend(lab.ops, c).cpu()
    sure = low == high
    assert int(sure.sum()) > sure.numel() // 2 and int((got != low)[sure].sum()) == 0
