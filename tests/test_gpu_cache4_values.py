"""Attention over 4-bit caches that a caller filled: scales of either sign, and of sizes far apart."""
import numpy as np
import pytest
import torch

import ternary_llm_b200 as tl
from tests.test_gpu_cache4 import TYPES, check_attention, ints, new_cache
from ternary_llm_b200 import cache4_ops as ops

pytestmark = pytest.mark.gpu


def filled(gen, batch, kv_heads, rows, dim, k_scale, v_scale):
    """Random codes with params (s, l) that put a value's middle near 0: l = noise - 7.5 s; k_scale and v_scale are [rows, dim / 64] or numbers."""
    c = new_cache(batch, kv_heads, rows, dim)
    for codes, params, scale in ((c.k_codes, c.k_params, k_scale), (c.v_codes, c.v_params, v_scale)):
        codes.copy_(torch.randint(0, 256, codes.shape, generator=gen, device="cuda"))
        s = torch.as_tensor(scale, device="cuda", dtype=torch.float32).expand(batch, kv_heads, rows, dim // 64)
        params[..., 0] = s.half()
        params[..., 1] = (s * (torch.rand(s.shape, generator=gen, device="cuda") - 7.5)).half()
    return c


def attend(c, before, new, heads, dtype, gen, scale=None, q=None):
    q = torch.randn(new, heads, c.dim, generator=gen, device="cuda").to(dtype) if q is None else q
    out = torch.empty_like(q)
    ops.attention(c, q, out, ints(0, new), ints(before + new), scale=scale, max_new=new)
    tl.check_device_errors()
    check_attention(c, q, out, [before], [new], heads, dtype, c.dim ** -0.5 if scale is None else scale)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("new,heads,kv_heads", [(1, 8, 2), (2, 8, 2), (3, 10, 2), (90, 8, 2), (400, 8, 2)])
def test_scales_of_values_below_zero(dtype, dim, new, heads, kv_heads):
    """All negative; one negative among positive ones, far larger; keys' too."""
    gen = torch.Generator(device="cuda").manual_seed(dim + new)
    before, rows = 300, 300 + new
    attend(filled(gen, 1, kv_heads, rows, dim, 0.2, -0.3), before, new, heads, dtype, gen)
    attend(filled(gen, 1, kv_heads, rows, dim, -0.2, -0.3), before, new, heads, dtype, gen)
    for at in (0, 40, before - 1):
        v = torch.full((rows, dim // 64), 0.01)
        v[at] = -100.0
        attend(filled(gen, 1, kv_heads, rows, dim, -0.1, v), before, new, heads, dtype, gen)
    v = torch.where(torch.arange(rows)[:, None] % 3 == 0, -0.5, 0.25).expand(rows, dim // 64)
    attend(filled(gen, 1, kv_heads, rows, dim, 0.1, v), before, new, heads, dtype, gen)
