"""Calls of the 4-bit cache at the edges of what they are told: sequences that share rows, hints, parts of the work."""
import numpy as np
import pytest
import torch

import ternary_llm_b200 as tl
from tests.test_gpu_cache4 import TYPES, check_attention, ints, layout, new_cache, random_cache
from ternary_llm_b200 import cache4_ops as ops

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("first,lens,rows,heads,kv_heads,dim", [
    ((0, 300, 200, 600), (300, 0, 400), 600, 8, 2, 64),            # whole tiles of 128 rows
    ((0, 1200, 900, 2000), (1200, 0, 1100), 1200, 32, 8, 64),      # of 256
    ((0, 300, 200, 600), (6000, 0, 6000), 6000, 8, 2, 128),        # cut
    ((0, 1200, 900, 1800), (9000, 0, 9000), 9000, 32, 8, 128),
    ((0, 2, 1, 4), (300, 0, 300), 300, 8, 2, 64),                  # few rows, in one CTA and cut
    ((0, 2, 1, 4), (5000, 0, 5000), 5000, 8, 2, 64),
    (tuple(range(700)) + (600, 710), (40,) * 701, 40, 4, 4, 64)])
def test_sequences_that_share_rows(first, lens, rows, heads, kv_heads, dim):
    """Attention writes nothing and says so."""
    c = new_cache(len(lens), kv_heads, rows, dim)
    for p in (c.k_params, c.v_params):
        p.fill_(0.5)
    q = torch.randn(first[-1], heads, dim, device="cuda").half()
    new = max(max(b - a, 1) for a, b in zip(first, first[1:]))
    for most in (new, 0, first[-1]):
        out = torch.full_like(q, 7.0)
        ops.attention(c, q, out, ints(*first), ints(*lens), max_new=most)
        with pytest.raises(tl.TllmError, match="outside its tensors"):
            tl.check_device_errors()
        assert (out == 7).all()


@pytest.mark.parametrize("before,new,heads,kv_heads,dim", [
    ([7 * i % 3000 for i in range(32)], [1] * 32, 32, 8, 128),                             # single tokens
    ([i % 61 for i in range(4096)], [1] * 4096, 8, 2, 64),
    ([0] + [11 * i % 900 for i in range(40)], [500] + [1] * 40, 8, 2, 128),                # a prompt beside them
    ([0] + [300] * 20, [1500] + [1] * 20, 32, 8, 64),
    ([0] + [100] * 15, [1] + [20] * 15, 16, 4, 64), ([5, 900, 70], [701, 0, 300], 32, 8, 64), ([0] * 9 + [3], [0] * 9 + [130], 16, 8, 64)])
def test_lengths_that_nobody_names(before, new, heads, kv_heads, dim):
    """Without a number of new rows, and with the right one."""
    gen = torch.Generator(device="cuda").manual_seed(len(new))
    lens = [a + n for a, n in zip(before, new)]
    c = random_cache(gen, len(new), kv_heads, max(lens), dim, lens)
    first, lens_dev, tokens = layout(before, new)
    some = {0, 1, 2, len(new) // 2, len(new) - 2, len(new) - 1}
    for dtype in TYPES:
        q = torch.randn(tokens, heads, dim, generator=gen, device="cuda").to(dtype)
        for most in (0, max(new)):
            out = torch.full_like(q, 7.0)
            ops.attention(c, q, out, first, lens_dev, max_new=most)
            tl.check_device_errors()
            check_attention(c, q, out, before, new, heads, dtype, dim ** -0.5, some)


def test_a_long_prompt_named_as_single_tokens():
    """Its units of few rows do not fit 31 bits: the call is taken as without the hint, and not refused."""
    gen = torch.Generator(device="cuda").manual_seed(1)
    n, heads, kv_heads, dim = 62000, 32, 8, 64
    c = random_cache(gen, 1, kv_heads, 131072, dim, [n])
    q = torch.randn(n, heads, dim, generator=gen, device="cuda").half()
    outs = [torch.full_like(q, 7.0) for _ in range(2)]
    for most, out in zip((0, 1), outs):
        ops.attention(c, q, out, ints(0, n), ints(n), max_new=most)
    tl.check_device_errors()
    assert torch.equal(*outs)
    for i in (0, 127, 128, 30001, n - 1):                                  # rows of the prompt, each as one token behind i
        check_attention(c, q[i:i + 1], outs[1][i:i + 1], [i], [1], heads, torch.float16, dim ** -0.5)
