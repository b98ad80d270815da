"""Every chunk of positions counts once: calls whose work is cut into parts that are joined.

All keys are alike, so every position that a row sees has the same weight.  Value channel j of a position is 1 where the position lies in
chunk j of `chunk` positions (modulo the channels), else 0, so that a channel of the result is the share of its chunks' positions among those
that the row sees.  A chunk that is left out, or taken twice, changes its channel by far more than the tolerance: weights of 1 and values
of 0 and 1 are exact (l = 0, s = half(1 / 15) makes 15 s = 0.99976), sums are whole numbers in FP32 but for the factor 15 s, the
parts' maxima are equal up to the rounding of scores, and the result is rounded once."""
import numpy as np
import pytest
import torch

import ternary_llm_b200 as tl
from tests.test_cache4_ways_cpu import record, workspace
from tests.test_gpu_cache4 import HALF_STEP, TYPES, layout
from ternary_llm_b200 import cache4_ops as ops

pytestmark = pytest.mark.gpu

ONE = float(np.float16(1 / 15)) * 15


def marked(batch, kv_heads, rows, dim, chunk):
    """Channel j is ONE in the chunks j, j + dim, ..; a head's channels are turned by its number, a sequence's by 5 times its own."""
    c = ops.Cache4.empty(batch, kv_heads, rows, dim)
    c.k_codes.fill_(0x77)
    for p in (c.k_params, c.v_params):
        p[..., 0], p[..., 1] = float(np.float16(1 / 15)), 0.0
    x = torch.zeros(batch, kv_heads, rows, dim, dtype=torch.uint8)
    p = torch.arange(rows)
    for b in range(batch):
        for g in range(kv_heads):
            x[b, g, p, (p // chunk + g + 5 * b) % dim] = 15
    w = x.view(batch, kv_heads, rows, dim // 8, 8)
    low = w[..., 0::2]                                                    # value 2 i in nibble i, value 2 i + 1 in nibble i + 4
    high = w[..., 1::2]
    word = torch.cat((low[..., 0::2] | low[..., 1::2] << 4, high[..., 0::2] | high[..., 1::2] << 4), -1)
    c.v_codes.copy_(word.reshape(batch, kv_heads, rows, dim // 2))
    return c


def check_marks(out, before, new, heads, kv_heads, dim, chunk, dtype):
    per, at = heads // kv_heads, 0
    y = out.double().cpu().numpy()
    for b, (a, n) in enumerate(zip(before, new)):
        if not n:
            continue
        m = np.arange(a + 1, a + n + 1)                                    # positions that each row sees
        counts = np.zeros((n, dim))
        for j in range((a + n + chunk - 1) // chunk):
            counts[:, (j + 5 * b) % dim] += np.clip(m - j * chunk, 0, chunk)
        for g in range(kv_heads):
            want = ONE * np.roll(counts, g, axis=1) / m[:, None]
            got = y[at:at + n, g * per:(g + 1) * per]
            # weights are 1 as FP16, times s exact to 2^-11; the sum of weights and the division FP32; scores of equal keys differ by nothing
            bound = (HALF_STEP[dtype] + 2.0 ** -11 + 2.0 ** -18) * want + (2.0 ** -25 if dtype == torch.float16 else 1e-38) + 8 * 2.0 ** -18 * ONE / 15
            err = np.abs(got - want[:, None])
            assert (err <= bound[:, None]).all(), (b, g, float((err / bound[:, None]).max()), np.unravel_index(np.argmax(err / bound[:, None]), err.shape))
            # a chunk more or less changes this much
            assert (bound.max(1) < ONE * chunk / m / 2)[m >= chunk].all()
        at += n


def run(before, new, heads, kv_heads, dim, dtype, way, size, most=None, chunk=32):
    gen = torch.Generator(device="cuda").manual_seed(sum(before) + sum(new))
    lens = [a + n for a, n in zip(before, new)]
    most = max(new) if most is None else most
    first, lens_dev, tokens = layout(before, new)
    rows = max(lens)
    assert workspace(len(new), kv_heads, rows, dim, tokens, heads, most, rows) == (record(*way, dim) if way else 0)
    c = marked(len(new), kv_heads, rows, dim, chunk)
    q = (size * torch.randn(tokens, heads, dim, generator=gen, device="cuda")).to(dtype)
    out = torch.full_like(q, 7.0)
    ops.attention(c, q, out, first, lens_dev, max_new=most, max_len=rows)
    tl.check_device_errors()
    check_marks(out, before, new, heads, kv_heads, dim, chunk, dtype)


FOUR, EIGHT, SIXTEEN, TILES, PAIRS = (296, 4), (296, 8), (148, 16), (148, 128), (148, 256)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("before,new,heads,kv_heads,dim,way", [
    ([20000], [1], 4, 1, 64, FOUR), ([9999, 0, 5001], [1, 1, 1], 32, 8, 128, FOUR), ([2600, 40], [1, 1], 3, 1, 64, FOUR), ([1600 + 97 * i for i in range(30)], [1] * 30, 6, 6, 128, FOUR),
    ([131000], [1], 8, 2, 128, FOUR), ([0, 30000, 31, 32, 33, 12345], [1] * 6, 8, 2, 64, FOUR),
    ([20000], [1], 8, 1, 64, EIGHT), ([2600, 40, 7000], [2, 1, 2], 32, 8, 128, EIGHT), ([5000 + 311 * i for i in range(12)], [1] * 12, 35, 5, 64, EIGHT),
    ([20000], [1], 16, 1, 64, SIXTEEN), ([1300, 2900, 1777], [5, 3, 1], 32, 8, 128, SIXTEEN), ([4001, 17, 9000], [4, 2, 3], 12, 4, 64, SIXTEEN),
    ([3000], [32], 2, 2, 128, SIXTEEN), ([2990, 0], [31, 32], 1, 1, 64, SIXTEEN),
    ([300], [1], 32, 8, 128, None), ([31 * i for i in range(40)], [1 + i % 2 for i in range(40)], 16, 8, 64, None), ([700], [32], 3, 3, 128, None)])
@pytest.mark.parametrize("size", [0.0, 1.0])
def test_few_rows(dtype, before, new, heads, kv_heads, dim, way, size):
    run(before, new, heads, kv_heads, dim, dtype, way, size)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("before,new,heads,kv_heads,dim,way", [
    ([2100], [79], 32, 8, 128, TILES), ([4000, 900], [65, 40], 32, 8, 64, TILES), ([2500], [300], 6, 2, 128, TILES),
    ([9000], [500], 16, 4, 128, PAIRS), ([16000], [512], 32, 8, 128, PAIRS), ([6000, 100, 0], [600, 1, 31], 32, 8, 64, PAIRS), ([0] + [300] * 20, [2000] + [1] * 20, 32, 8, 128, PAIRS),
    ([500], [79], 32, 8, 128, None), ([0, 77], [300, 250], 8, 2, 64, None), ([0], [2000], 32, 8, 128, None), ([5, 900, 70], [701, 33, 300], 32, 8, 64, None)])
@pytest.mark.parametrize("size", [0.0, 1.0])
def test_prompts(dtype, before, new, heads, kv_heads, dim, way, size):
    run(before, new, heads, kv_heads, dim, dtype, way, size)
