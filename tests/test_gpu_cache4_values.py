"""Attention over 4-bit caches that a caller filled: scales of either sign, and of sizes far apart."""
import numpy as np
import pytest
import torch

import ternary_llm_b200 as tl
from tests._cache4_few import check_few
from tests.test_gpu_cache4 import HALF_STEP, TINY, TYPES, check_attention, ints, new_cache
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


def sharp(gen, dim, n, small, large, at, dtype):
    """Keys that the query -u of one head gives a score of -45 at position `at` and some 0 elsewhere; values of size `large` there, `small` elsewhere."""
    u = torch.where(torch.rand(2, dim, generator=gen, device="cuda") < 0.5, -1.0, 1.0)
    size = torch.full((n, 1, 1), 0.02, device="cuda")
    size[at] = 45.0 / dim ** 0.5
    k = size * u + 0.01 * torch.randn(n, 2, dim, generator=gen, device="cuda")
    v = torch.randn(n, 2, dim, generator=gen, device="cuda") * torch.where(torch.arange(n, device="cuda") == at, large, small)[:, None, None]
    return u, k.to(dtype), v.to(dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("per", [1, 4, 7, 16])
@pytest.mark.parametrize("small,large", [(0.01, 100.0), (1e-3, 3e4), (2e-5, 3e4)])
def test_a_large_value_without_weight(dtype, dim, per, small, large):
    """Before, among and behind the positions that have the weight."""
    n = 400
    for at in (0, 17, 200, n - 2):
        gen = torch.Generator(device="cuda").manual_seed(at + per)
        u, k, v = sharp(gen, dim, n, small, large, at, dtype)
        c = new_cache(1, 2, n, dim)
        ops.append(c, None, k, v, ints(0, n), ints(n))
        q = (-u[:, None] * (1 + 0.1 * torch.rand(2, per, 1, generator=gen, device="cuda"))).reshape(1, 2 * per, dim).to(dtype)
        out = torch.empty_like(q)
        ops.attention(c, q, out, ints(0, 1), ints(n), max_new=1)
        tl.check_device_errors()
        check_few(c, q, out, [n - 1], [1], 2 * per, HALF_STEP[dtype], TINY[dtype], dim ** -0.5)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("new,heads,dim", [(2, 4, 64), (4, 4, 128), (3, 8, 64), (8, 8, 128)])
def test_values_behind_a_row_do_not_move_it(dtype, new, heads, dim):
    """The last token's value, a million times the others': rows before it repeat, bit for bit, and keep their bound."""
    gen = torch.Generator(device="cuda").manual_seed(new)
    n = 300 + new
    x = torch.randn(2, n, 2, dim, generator=gen, device="cuda").mul(0.01).to(dtype)
    q = torch.randn(new, heads, dim, generator=gen, device="cuda").to(dtype)
    outs = []
    for large in (False, True):
        y = x[1].clone()
        if large:
            y[-1] *= 1e6
        c = new_cache(1, 2, n, dim)
        ops.append(c, None, x[0], y, ints(0, n), ints(n))
        out = torch.empty_like(q)
        ops.attention(c, q, out, ints(0, new), ints(n), max_new=new)
        tl.check_device_errors()
        check_few(c, q, out, [n - new], [new], heads, HALF_STEP[dtype], TINY[dtype], dim ** -0.5)
        outs.append(out)
    assert torch.equal(outs[0][:-1], outs[1][:-1]) and not torch.equal(outs[0][-1], outs[1][-1])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("before,new,heads,kv_heads,dim", [
    ([0], [1], 4, 1, 64), ([300], [1], 32, 8, 128), ([127, 0, 1000], [1, 1, 1], 12, 4, 64), ([20000], [1], 8, 1, 64), ([5000], [1], 8, 2, 128), ([100, 2000], [5, 3], 8, 2, 128),
    ([2600, 40], [2, 1], 4, 1, 64), ([1300], [8], 8, 2, 128), ([700, 3], [8, 2], 6, 2, 64), ([2047], [4], 8, 1, 128)])
def test_few_rows_hold_their_bound(dtype, before, new, heads, kv_heads, dim):
    """Scores of few rows are sums of whole numbers: nothing is rounded to 11 bits before the weights."""
    gen = torch.Generator(device="cuda").manual_seed(sum(before) + dim)
    lens = [a + n for a, n in zip(before, new)]
    first = ints(*np.concatenate([[0], np.cumsum(new)]).tolist())
    c = new_cache(len(new), kv_heads, max(lens), dim)
    full = ints(*np.concatenate([[0], np.cumsum(lens)]).tolist())
    x = torch.randn(2, sum(lens), kv_heads, dim, generator=gen, device="cuda")
    x[0] = 3 * x[0] + 2 * torch.randn(kv_heads, dim, generator=gen, device="cuda")
    ops.append(c, None, x[0].half(), x[1].half(), full, ints(*lens))
    q = torch.randn(sum(new), heads, dim, generator=gen, device="cuda").to(dtype)
    out = torch.empty_like(q)
    ops.attention(c, q, out, first, ints(*lens), max_new=max(new), max_len=max(lens))
    tl.check_device_errors()
    check_few(c, q, out, before, new, heads, HALF_STEP[dtype], TINY[dtype], dim ** -0.5)
