"""Value scales of the paged 8-bit KV cache that are far apart or no powers of two: what the attention makes of them."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from test_gpu_kv8 import FORMATS, attend, check_attention, host, make_case

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


def set_scales(c, past, counts, exponent, rng=None):
    """Value scales 2^exponent(j, pages, head) of each request's page j (0 where that is None)."""
    table, scales = host(c["table"]), c["cache"][3].cpu()
    for b, p in enumerate(past):
        pages = max(0, -(-(p + counts[b]) // c["page"]))
        for j in range(pages):
            for h in range(scales.shape[1]):
                e = exponent(j, pages, h)
                scales[table[b, j], h] = 0.0 if e is None else 2.0 ** e * (1 if rng is None else rng.uniform(0.5, 1))
    c["cache"][3].copy_(scales)


@pytest.mark.parametrize("dtype", FORMATS)
@pytest.mark.parametrize("counts,width", [([2], None), ([100], None), ([2], 600), ([100], 600)])
def test_a_later_positions_scale_leaves_earlier_rows(gpu, lab, dtype, counts, width):
    """Rows up to position 15 see one page of scale 2^-100, those after it one of scale 1 too."""
    c = make_case(2, [15], counts, 2, 2, 64, 16, dtype, width=width)
    set_scales(c, [15], counts, lambda j, n, h: -100 if j == 0 else 0)
    got = check_attention(lab.ops, c)
    assert 0 < np.abs(got[0]).max() < 2.0 ** -90


PROFILES = {
    "rising": lambda j, n, h: -60 + 80 * j // n,
    "falling": lambda j, n, h: 20 - 80 * j // n,
    "in turn": lambda j, n, h: (-90, 30, 0, -40)[(j + h) % 4],
    "one large": lambda j, n, h: 25 if j == n // 2 else -70,
    "one small": lambda j, n, h: -120 if j == n // 2 else 20,
    "one zero": lambda j, n, h: None if j == n // 2 else 2,
    "all but one zero": lambda j, n, h: 2 if j == n // 2 else None,
    "all zero": lambda j, n, h: None,
    "subnormal": lambda j, n, h: -130 - j % 19,
    "subnormal beside others": lambda j, n, h: (-140, -60, 0)[j % 3],
    "largest": lambda j, n, h: (110, -120)[j % 2],
    "steps past a unit": lambda j, n, h: -66 * (j % 3) + 12,
}


@pytest.mark.parametrize("dtype,page,dim", [(FORMATS[0], 16, 64), (FORMATS[1], 64, 64), (FORMATS[1], 32, 128), (FORMATS[0], 128, 128)])
@pytest.mark.parametrize("past,counts,width", [([200, 130, 7], [1, 1, 2], None), ([900, 40], [3, 1], 400), ([300, 0], [40, 300], None),
                                               ([700, 30], [60, 1], 200), ([1500], [45], 300)])
@pytest.mark.parametrize("profile", PROFILES)
def test_attention_with_value_scales_far_apart(gpu, lab, dtype, page, dim, past, counts, width, profile):
    """Single tokens and tiles, whole and in parts: what each row sees counts by its own scale, however far apart they are."""
    c = make_case(11, past, counts, 2, 2, dim, page, dtype, width=width, stretch=2.0)
    set_scales(c, past, counts, PROFILES[profile])
    got = check_attention(lab.ops, c)
    assert profile == "all zero" or profile == "subnormal" or np.abs(got).max() > 0


@pytest.mark.parametrize("dtype", FORMATS)
@pytest.mark.parametrize("counts,width", [([1, 2, 1], None), ([100, 1, 20], None), ([1, 2, 1], 500), ([100, 1, 20], 500)])
@pytest.mark.parametrize("stretch", [0.0, 1.0, 300.0])
def test_attention_with_scales_far_apart_and_of_any_value(gpu, lab, dtype, counts, width, stretch):
    """No powers of two, and scores so far apart that a page of small scale outweighs one of large scale, or the other way."""
    past = [400, 100, 0]
    c = make_case(8, past, counts, 2, 2, 64, 16, dtype, stretch=stretch, width=width)
    set_scales(c, past, counts, lambda j, n, h: (-100, 10, -30, -75, 0)[(j + h) % 5], np.random.default_rng(1))
    check_attention(lab.ops, c)
