"""The operators of the 4-bit cache against 64 bits."""
import numpy as np
import pytest
import torch

import ternary_llm_b200 as tl
from tests import _cache4 as ref
from ternary_llm_b200 import cache4_ops as ops

pytestmark = pytest.mark.gpu

HALF_STEP = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}
TINY = {torch.float16: 2.0 ** -25, torch.bfloat16: 1e-38, torch.float32: 1e-38}       # half of the smallest step


def f64(t):
    return t.double().cpu().numpy()


def ints(*v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def rounded(x, dtype):
    return f64(torch.from_numpy(x).to(dtype))


# ---- rotary ------------------------------------------------------------------------------
def rotary_case(dtype, tokens, heads, kv_heads, dim, rot, half, start, amplitude=1.0, wide=0, inverse=False, in_place=False):
    gen = torch.Generator(device="cuda").manual_seed(tokens + dim + rot)
    table = ops.RotaryTable(rot, 500000.0, half=half, amplitude=amplitude)
    both = torch.randn(tokens, (heads + kv_heads) * dim + wide, generator=gen, device="cuda").to(dtype)
    q, k = both[:, :heads * dim].view(tokens, heads, dim), both[:, heads * dim:(heads + kv_heads) * dim].view(tokens, kv_heads, dim)
    position = start + torch.arange(tokens, device="cuda", dtype=torch.int32) * 3
    x = [f64(q), f64(k)]
    rest = both[:, (heads + kv_heads) * dim:].clone()
    out = (q, k) if in_place else (torch.full((tokens, heads, dim), 7.0, device="cuda", dtype=dtype), torch.full((tokens, kv_heads, dim), 7.0, device="cuda", dtype=dtype))
    ops.rotary(q, k if kv_heads else None, position, table, None if in_place else out[0], None if in_place or not kv_heads else out[1], inverse=inverse)
    assert torch.equal(both[:, (heads + kv_heads) * dim:], rest)
    for y, v in zip(out, x):
        want = ref.rotate(v, position.cpu().numpy().astype(np.int64) * (-1 if inverse else 1), table.frequencies, amplitude, half)
        size = np.abs(want)
        pairs = np.abs(v).max(initial=0.0) * 2 * amplitude
        # the angle to 2^-25 of half a turn at most and what sincospi rounds (2 units in the last place), products and the sum, the result
        bound = HALF_STEP[dtype] * size + pairs * (np.pi * 2.0 ** -24 + 4 * 2.0 ** -23) + TINY[dtype]
        assert (np.abs(f64(y) - want) <= bound).all()
        assert (f64(y)[..., rot:] == v[..., rot:]).all()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("tokens,heads,kv_heads,dim,rot,start", [
    (1, 32, 8, 64, 64, 1500), (5, 3, 1, 128, 128, 2 ** 31 - 100), (7, 4, 4, 80, 32, 0), (3, 2, 0, 8, 2, 5), (33, 5, 2, 96, 24, 100000), (2, 1, 1, 256, 256, -4),
    (9, 7, 3, 72, 72, 999999), (4, 40, 8, 512, 130, 77), (257, 2, 2, 64, 16, 31)])
def test_rotary(dtype, half, tokens, heads, kv_heads, dim, rot, start):
    rotary_case(dtype, tokens, heads, kv_heads, dim, rot, half, start)
    rotary_case(dtype, tokens, heads, kv_heads, dim, rot, half, start, amplitude=1.25, wide=16, in_place=True)


@pytest.mark.parametrize("half", [False, True])
def test_rotary_back_is_the_gradient(half):
    """Turning back after turning gives the input; the gradient of a product with the turned vector is the other vector turned back."""
    rotary_case(torch.float32, 6, 3, 2, 64, 48, half, 12345, inverse=True)
    gen = torch.Generator(device="cuda").manual_seed(1)
    table, position = ops.RotaryTable(48, 1e4, half=half), ints(0, 5, 1000, 70000)
    x, g = torch.randn(2, 4, 3, 64, generator=gen, device="cuda")
    y, back, turned_back = torch.empty_like(x), torch.empty_like(x), torch.empty_like(x)
    ops.rotary(x, None, position, table, y)
    ops.rotary(y, None, position, table, back, inverse=True)
    assert (back - x).abs().max() <= 16 * 2.0 ** -24 * float(x.abs().max()) * 2
    ops.rotary(g, None, position, table, turned_back, inverse=True)
    e = torch.randn(x.shape, generator=gen, device="cuda")
    there, here = torch.empty_like(x), torch.empty_like(x)
    ops.rotary(x + e, None, position, table, there)
    ops.rotary(x - e, None, position, table, here)
    difference, gradient = ((there - here).double() / 2 * g.double()).sum(), (e.double() * turned_back.double()).sum()
    # each factor is off by at most 16 units in the last place of a pair
    assert abs(difference - gradient) <= 4 * 16 * 2.0 ** -24 * float((e.abs().double().max() + x.abs().double().max()) * g.abs().double().sum())


def test_rotary_of_nothing():
    t = ops.RotaryTable(64)
    x = torch.empty(0, 4, 64, device="cuda")
    ops.rotary(x, x, torch.empty(0, dtype=torch.int32, device="cuda"), t)


# ---- append and read -----------------------------------------------------------------------
def new_cache(batch, kv_heads, rows, dim):
    c = ops.Cache4.empty(batch, kv_heads, rows, dim)
    for p in (c.k_params, c.v_params):
        p.fill_(float("nan"))
    c.k_codes.fill_(0xa5)
    c.v_codes.fill_(0x5a)
    return c


def contents(c):
    return [t.clone() for t in (c.k_codes, c.k_params, c.v_codes, c.v_params)]


def layout(before, new):
    first = np.concatenate([[0], np.cumsum(new)])
    return ints(*first.tolist()), ints(*[a + n for a, n in zip(before, new)]), int(first[-1])


def append_case(dtype, before, new, heads, kv_heads, dim, half=True, rot=None, rows=None, wide=0, spread=1.0, table=True, in_place=False, tail=0):
    gen = torch.Generator(device="cuda").manual_seed(sum(new) + dim)
    batch = len(new)
    rows = rows or max(a + n for a, n in zip(before, new)) + 3
    c = new_cache(batch, kv_heads, rows, dim)
    was = contents(c)
    first, lens, tokens = layout(before, new)
    width = (heads + 2 * kv_heads) * dim + wide
    packed = (spread * torch.randn(tokens + tail, width, generator=gen, device="cuda")).to(dtype)
    q, k, v = (t.unflatten(1, (-1, dim)) for t in packed[:, :width - wide].split([heads * dim, kv_heads * dim, kv_heads * dim], 1))
    kept = packed.clone()
    t = ops.RotaryTable(rot or dim, 1e4, half=half) if table else None
    q_out = None if in_place else torch.full((tokens + tail, heads, dim), 7.0, dtype=dtype, device="cuda")
    ops.append(c, q if heads else None, k, v, first, lens, t, q_out if heads else None)
    back = [torch.full((tokens + tail, kv_heads, dim), 7.0, dtype=torch.float32, device="cuda") for _ in range(2)]
    ops.read(c, *back, first, lens)
    tl.check_device_errors()
    assert torch.equal(packed[:, heads * dim:], kept[:, heads * dim:])                          # k and v are only read
    qo = q if in_place else q_out
    assert in_place or torch.equal(packed, kept)
    assert torch.equal(qo[tokens:], kept[tokens:, :heads * dim].view(-1, heads, dim)) if in_place else bool((qo[tokens:] == 7).all())
    # the same rows by the operator that turns alone: the rounded activations that are held
    position = torch.cat([torch.arange(a, a + n, dtype=torch.int32, device="cuda") for a, n in zip(before, new)] + [ints(*[0] * tail)])
    kt, qt = kept[:, heads * dim:(heads + kv_heads) * dim].unflatten(1, (-1, dim)).contiguous(), kept[:, :heads * dim].unflatten(1, (-1, dim)).contiguous()
    if table:
        ops.rotary(kt, qt if heads else None, position, t)
    assert torch.equal(qo[:tokens], qt[:tokens])
    at = 0
    now = contents(c)
    for b, (a, n) in enumerate(zip(before, new)):
        for side, x in ((0, kt), (2, v)):
            codes, params = ref.quantise(f64(x[at:at + n]).swapaxes(0, 1))
            assert (ref.unpack(now[side][b, :, a:a + n].cpu().numpy()) == codes).all()
            assert (now[side + 1][b, :, a:a + n].cpu().numpy() == params).all()
            want = ref.values(codes, params).swapaxes(0, 1)
            assert (np.abs(f64(back[side // 2][at:at + n]) - want) <= 2.0 ** -24 * np.abs(want) + 1e-38).all()
        for i in range(4):                                                                    # the other rows are as they were
            other = torch.ones(rows, dtype=torch.bool, device="cuda")
            other[a:a + n] = False
            assert torch.equal(now[i][b][:, other].view(torch.uint8), was[i][b][:, other].view(torch.uint8))
        at += n
    for t in back:
        assert (t[tokens:] == 7).all()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("before,new,heads,kv_heads,dim", [
    ([0], [1], 1, 1, 64), ([300, 0, 7999], [1, 1, 1], 32, 8, 128), ([0, 5, 64, 9], [130, 0, 3, 1], 6, 2, 64), ([63], [66], 5, 5, 128), ([0], [700], 40, 8, 64),
    ([2] * 37, [1] * 37, 4, 1, 128), ([10] * 70, [1, 0] * 35, 2, 2, 64)])
def test_append_and_read(dtype, before, new, heads, kv_heads, dim):
    append_case(dtype, before, new, heads, kv_heads, dim)
    append_case(dtype, before, new, heads, kv_heads, dim, half=False, rot=dim // 2, wide=8, in_place=True, tail=2)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("spread", [1e-7, 1e-4, 1000.0, 3e4])
def test_append_of_small_and_large_values(dtype, spread):
    append_case(dtype, [3, 0], [5, 9], 0, 3, 128, spread=spread, table=False)
    append_case(dtype, [3, 0], [5, 9], 2, 3, 64, spread=min(spread, 8000.0), rot=10)          # a turned pair stays inside FP16


def test_append_values_at_the_borders():
    """Equal values, ties, infinities, values beyond the limit; a NaN marks its position and leaves the values finite."""
    c = new_cache(1, 2, 16, 64)
    x = torch.zeros(6, 2, 64, dtype=torch.bfloat16, device="cuda")
    x[0] = 0.37
    x[1, :, :31] = torch.arange(31, device="cuda") / 2
    x[1, :, 31:] = 15
    x[2, :, 0], x[2, :, 1], x[2, :, 2] = float("inf"), float("-inf"), 1e30
    x[3] = 1e38
    x[4, 0, 5] = float("nan")
    y = x.clone()
    y[4], y[5, 1, 63] = 1.5, float("nan")
    first, lens = ints(0, 6), ints(6)
    ops.append(c, None, x, y, first, lens)
    k, v = torch.empty(2, 6, 2, 64, dtype=torch.float32, device="cuda")
    ops.read(c, k, v, first, lens)
    tl.check_device_errors()
    assert (k[0] == float(torch.tensor(0.37).bfloat16())).all()
    assert torch.equal(k[1, 0, :31], torch.arange(31, device="cuda").div(2).round())         # ties go to even codes
    assert (k[2, :, 0] == 61440).all() and (k[2, :, 1] == -61440).all() and (k[2, :, 2] == 61440).all() and (k[3] == 61440).all()
    assert k[4, 0].isnan().all() and not k[4, 1].isnan().any() and k[5, 1].isnan().all() and not k[5, 0].isnan().any()
    assert v.isfinite().all() and (v[5, 1] == 0).all()


def test_padding_and_sequences_outside_the_tensors():
    c = new_cache(3, 1, 8, 64)
    was = contents(c)
    x = torch.randn(7, 1, 64, device="cuda").half()
    # the first sequence is longer than its positions: its first row is padding; the second takes no part
    q, out = x.clone(), torch.full((7, 1, 64), 7.0, dtype=torch.float16, device="cuda")
    first, lens = ints(1, 4, 4, 6), ints(2, 0, 2)
    ops.append(c, q, x, x, first, lens)
    assert torch.equal(q, x)                                       # no table: nothing turns
    k = torch.full((7, 1, 64), 7.0, device="cuda")
    ops.read(c, k, None, first, lens)
    ops.attention(c, x, out, first, lens)
    tl.check_device_errors()
    assert (k[[0, 6]] == 7).all() and (k[1] == 0).all() and (k[2:6] != 7).all()
    assert (out[[0, 6]] == 7).all() and (out[1] == 0).all() and out.isfinite().all()
    assert torch.equal(contents(c)[0][1], was[0][1]) and torch.equal(contents(c)[0][:, :, 2:], was[0][:, :, 2:])
    for first, lens in ((ints(0, 3, 2, 6), ints(3, 3, 4)), (ints(0, 2, 4, 8), ints(2, 2, 4)), (ints(-1, 2, 4, 6), ints(3, 2, 2)), (ints(0, 2, 4, 6), ints(2, 9, 2)),
                        (ints(0, 2, 4, 6), ints(2, -1, 2))):
        for call in (lambda: ops.append(c, None, x, x, first, lens), lambda: ops.read(c, k, None, first, lens), lambda: ops.attention(c, x, out, first, lens)):
            call()
            with pytest.raises(tl.TllmError, match="outside its tensors"):
                tl.check_device_errors()
            tl.check_device_errors()


@pytest.mark.parametrize("new", [1, 9, 300])
def test_sequences_above_the_limit_of_a_call(new):
    c = new_cache(1, 2, 1200, 64)
    x = torch.randn(1000, 2, 64, device="cuda").half()
    ops.append(c, None, x, x, ints(0, 1000), ints(1000))
    q, out = torch.randn(new, 4, 64, device="cuda").half(), torch.empty(new, 4, 64, device="cuda", dtype=torch.float16)
    ops.attention(c, q, out, ints(0, new), ints(1000), max_new=new, max_len=1000)
    tl.check_device_errors()
    check_attention(c, q, out, [1000 - new], [new], 4, torch.float16, 0.125)
    ops.attention(c, q, out, ints(0, new), ints(1000), max_new=new, max_len=900)
    with pytest.raises(tl.TllmError, match="outside its tensors"):
        tl.check_device_errors()
    check_attention(c, q, out, [900 - new], [new], 4, torch.float16, 0.125)          # as a sequence of 900 positions


def test_nothing_to_do():
    for batch, tokens in ((0, 0), (2, 0), (0, 3)):
        c = ops.Cache4.empty(batch, 2, 8, 64)
        first, lens = ints(*[0] * (batch + 1)), ints(*[3] * batch)
        x = torch.full((tokens, 2, 64), 7.0, dtype=torch.float16, device="cuda")
        y = x.clone()
        ops.append(c, x, x, x, first, lens)
        ops.read(c, y, y.clone(), first, lens)
        ops.attention(c, x, y, first, lens)
        assert (y == 7).all()
    tl.check_device_errors()


# ---- attention -------------------------------------------------------------------------------
def random_cache(gen, batch, kv_heads, rows, dim, lens, spread=1.0):
    """Codes and params as append writes them; behind each sequence's length anything, NaN among it."""
    c = new_cache(batch, kv_heads, rows, dim)
    first, lens_dev, tokens = layout([0] * batch, lens)
    x = (spread * torch.randn(2, tokens, kv_heads, dim, generator=gen, device="cuda") + torch.randn(kv_heads, dim, generator=gen, device="cuda")).half()
    ops.append(c, None, x[0], x[1], first, lens_dev)
    return c


def check_attention(c, q, out, before, new, heads, dtype, scale, sequences=None):
    """Every row of the call against 64 bits."""
    kc, kp, vc, vp = (t.cpu().numpy() for t in (c.k_codes, c.k_params, c.v_codes, c.v_params))
    per, at = heads // c.kv_heads, 0
    x, y = f64(q), f64(out)
    for b, (a, n) in enumerate(zip(before, new)):
        m = a + n
        for g in range(c.kv_heads if n and (sequences is None or b in sequences) else 0):
            k, v = (ref.values(ref.unpack(codes[b, g, :m]), params[b, g, :m]) for codes, params in ((kc, kp), (vc, vp)))
            rows = x[at:at + n, g * per:(g + 1) * per].reshape(n * per, c.dim)
            middle = ref.values(np.full((m, c.dim), 8), vp[b, g, :m])
            want, size, reach = ref.attention(rows, k, v, np.repeat(np.arange(a, m), per), scale, np.maximum(np.abs(v), np.abs(v - middle)))
            # weights and values may enter as 11 bits (half a step each), keys too: a score moves by 2^-11 of the sum of its terms' sizes, a
            # weight and the sum of the weights by that; scores and sums in FP32.  Where v enters as s (c - 8) and l + 8 s, the rounded weight
            # meets the first part, |v - (l + 8 s)|, and the second is FP32
            bound = (2 * 2.0 ** -11 + 2 * (2.0 ** -11 + (c.dim + m) * 2.0 ** -24) * reach[:, None]) * size + HALF_STEP[dtype] * np.abs(want) + TINY[dtype]
            err = np.abs(y[at:at + n, g * per:(g + 1) * per].reshape(n * per, c.dim) - want)
            assert (err <= bound).all(), (b, g, float((err / bound).max()))
        at += n


def attention_case(dtype, before, new, heads, kv_heads, dim, scale=None, hints=True, rows=None, wide=0, spread=1.0, sequences=None):
    gen = torch.Generator(device="cuda").manual_seed(sum(before) + 7 * sum(new) + dim)
    lens = [a + n for a, n in zip(before, new)]
    first, lens_dev, tokens = layout(before, new)
    c = random_cache(gen, len(new), kv_heads, rows or max(lens) + 5, dim, lens, spread)
    q = torch.randn(tokens + 1, heads * dim + wide, generator=gen, device="cuda").to(dtype)[:, :heads * dim].unflatten(1, (heads, dim))
    out = torch.full((tokens + 1, heads * dim + wide), 7.0, dtype=dtype, device="cuda")
    o = out[:, :heads * dim].unflatten(1, (heads, dim))
    ops.attention(c, q, o, first, lens_dev, scale=scale, max_new=max(new) if hints else 0, max_len=max(lens) if hints else 0)
    tl.check_device_errors()
    assert (out[tokens:] == 7).all() and (out[:, heads * dim:] == 7).all()
    check_attention(c, q, o, before, new, heads, dtype, dim ** -0.5 if scale is None else scale, sequences)
    return c, q, o


TYPES = [torch.float16, torch.bfloat16]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("before,heads,kv_heads,dim", [
    ([0], 1, 1, 64), ([0], 32, 8, 128), ([1], 4, 4, 128), ([14, 15, 16], 8, 2, 64), ([31], 16, 1, 128), ([63, 64, 65], 8, 8, 64), ([300], 32, 8, 64),
    ([127, 0, 1000], 12, 4, 128), ([2047], 40, 8, 64), ([5000], 32, 8, 128), ([20000], 8, 1, 64), ([17] * 40, 6, 2, 128), ([0, 3000] * 9, 32, 8, 64),
    ([255], 20, 1, 64), ([600, 5], 33, 1, 128), ([40], 64, 1, 64)])
def test_one_token(dtype, before, heads, kv_heads, dim):
    attention_case(dtype, before, [1] * len(before), heads, kv_heads, dim)
    attention_case(dtype, before, [1] * len(before), heads, kv_heads, dim, scale=0.3, hints=False, wide=24)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("before,new,heads,kv_heads,dim", [
    ([0], [2], 1, 1, 64), ([100, 0, 2000], [5, 2, 3], 32, 8, 128), ([15], [3], 16, 1, 128), ([0], [16], 4, 4, 64), ([700, 3], [8, 0], 6, 2, 64),
    ([30, 31, 32, 33], [4, 3, 2, 1], 8, 4, 128), ([3000], [7], 40, 8, 64), ([126], [9], 12, 4, 128), ([0], [33], 1, 1, 128), ([64], [64], 2, 1, 64),
    ([1000, 0], [31, 1], 5, 5, 64)])
def test_few_tokens(dtype, before, new, heads, kv_heads, dim):
    attention_case(dtype, before, new, heads, kv_heads, dim)
    attention_case(dtype, before, new, heads, kv_heads, dim, hints=False, wide=8)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("before,new,heads,kv_heads,dim", [
    ([0], [127], 4, 1, 64), ([0], [128], 4, 4, 128), ([0], [129], 8, 2, 64), ([1], [300], 6, 2, 128), ([500], [257], 5, 1, 64), ([0, 77, 3, 0], [200, 1, 0, 90], 8, 2, 128),
    ([128], [128], 32, 8, 64), ([2000], [64], 32, 8, 128), ([900, 0], [40, 600], 3, 3, 64), ([0], [1000], 40, 8, 64), ([5000], [130], 16, 2, 128)])
def test_prompts(dtype, before, new, heads, kv_heads, dim):
    attention_case(dtype, before, new, heads, kv_heads, dim)


@pytest.mark.parametrize("before,new,heads,kv_heads,dim", [
    ([1249], [1], 8, 2, 128), ([1250], [1], 8, 2, 128), ([2499], [1], 4, 1, 64), ([2500], [1], 4, 1, 64),                  # one CTA a head, or several
    ([2600, 40], [1, 1], 8, 1, 128), ([2600, 40], [1, 1], 16, 1, 64), ([2600, 40], [2, 1], 4, 1, 64),                      # tiles of 4, 8 and 16 rows, cut
    ([1300], [8], 8, 2, 128), ([1300], [9], 8, 2, 128), ([0] * 25, [33] * 25, 6, 6, 64), ([0] * 24, [33] * 24, 6, 6, 64),  # few rows and many
    ([900], [140], 4, 1, 64), ([1800], [140], 4, 1, 64), ([1800], [300], 5, 1, 128), ([4000, 5], [129, 200], 2, 2, 64)])   # prompts whole and cut
def test_both_sides_of_the_lines_between_ways(before, new, heads, kv_heads, dim):
    for dtype in TYPES:
        attention_case(dtype, before, new, heads, kv_heads, dim)


@pytest.mark.parametrize("new", [1, 7, 150])
@pytest.mark.parametrize("scale", [0.0, -0.3, 1e-30])
def test_scales_that_are_not_positive(new, scale):
    attention_case(torch.float16, [90], [new], 8, 2, 64, scale=scale)
    attention_case(torch.bfloat16, [2000], [new], 4, 1, 128, scale=scale)


@pytest.mark.parametrize("new", [1, 40])
def test_the_native_call_and_the_other_way_agree(new):
    """A scale that is no plain float takes the checks in Python and ctypes."""
    c, q, out = attention_case(torch.float16, [3000], [new], 8, 2, 128, scale=1.0)
    other = torch.full_like(q[:new], 7.0)
    ops.attention(c, q[:new], other, ints(0, new), ints(3000 + new), scale=1, max_new=new, max_len=3000 + new)
    assert torch.equal(other, out[:new])
    table, x = ops.RotaryTable(128), q[:new].contiguous()
    position, y, z = torch.arange(new, dtype=torch.int32, device="cuda"), torch.empty_like(x), torch.empty_like(x)
    ops.rotary(x, None, position, table, y)
    ops.rotary(x, None, position, table, z, inverse=0)
    assert torch.equal(y, z)


@pytest.mark.parametrize("new", [[1, 1], [3, 40], [200, 130]])
@pytest.mark.parametrize("new_hint,len_hint", [(0, 0), (1, 2700), (5, 0), (1000, 100000), (90, 2700), (1, 0)])
def test_hints_do_not_matter(new, new_hint, len_hint):
    """Wrong numbers of rows choose another way of the work, not another result; so do loose limits of positions."""
    gen = torch.Generator(device="cuda").manual_seed(5)
    before, lens = [400, 2500], [400 + new[0], 2500 + new[1]]
    c = random_cache(gen, 2, 2, 3000, 128, lens)
    first, lens_dev, tokens = layout(before, new)
    q = torch.randn(tokens, 8, 128, generator=gen, device="cuda").half()
    out = torch.empty_like(q)
    ops.attention(c, q, out, first, lens_dev, max_new=new_hint, max_len=len_hint)
    tl.check_device_errors()
    check_attention(c, q, out, before, new, 8, torch.float16, 128 ** -0.5)


@pytest.mark.parametrize("new", [1, 6, 150])
@pytest.mark.parametrize("spread,size", [(1.0, 60.0), (3000.0, 1e-3), (1e-5, 1.0), (0.0, 1.0)])
def test_sharp_flat_large_and_small(new, spread, size):
    """One position takes nearly all weight; keys and values far from 1; all keys alike."""
    for dtype in TYPES:
        gen = torch.Generator(device="cuda").manual_seed(new)
        c = random_cache(gen, 1, 2, 900, 64, [700 + new], spread)
        q = (size * torch.randn(new, 8, 64, generator=gen, device="cuda")).to(dtype)
        out = torch.empty_like(q)
        ops.attention(c, q, out, ints(0, new), ints(700 + new), max_new=new)
        check_attention(c, q, out, [700], [new], 8, dtype, 64 ** -0.5)


@pytest.mark.parametrize("new", [1, 5, 200])
def test_scales_of_values_that_differ(new):
    """Values of neighbouring positions whose scales lie 2^20 apart, in both orders."""
    gen = torch.Generator(device="cuda").manual_seed(new)
    for up in (True, False):
        c = random_cache(gen, 1, 1, 600, 128, [400 + new])
        n = 400 + new
        size = torch.logspace(-4, 2, n, device="cuda")
        size = size if up else size.flip(0)
        v = (size[:, None, None] * torch.randn(n, 1, 128, generator=gen, device="cuda")).half()
        k = torch.randn(n, 1, 128, generator=gen, device="cuda").half()
        ops.append(c, None, k, v, ints(0, n), ints(n))
        q = torch.randn(new, 4, 128, generator=gen, device="cuda").half()
        out = torch.empty_like(q)
        ops.attention(c, q, out, ints(0, new), ints(n), max_new=new)
        check_attention(c, q, out, [400], [new], 4, torch.float16, 128 ** -0.5)


@pytest.mark.parametrize("new", [3, 40, 300])
def test_a_nan_reaches_the_rows_that_see_it(new):
    """A position marked by append: rows before it are as without it, rows from it on are NaN, other heads are not touched."""
    gen = torch.Generator(device="cuda").manual_seed(new)
    before, bad = 200, 200 + new // 2
    n = before + new
    x = torch.randn(2, n, 2, 128, generator=gen, device="cuda").half()
    q = torch.randn(new, 8, 128, generator=gen, device="cuda").half()
    outs = []
    for mark in (False, True):
        c = new_cache(1, 2, n + 40, 128)
        y = x.clone()
        if mark:
            y[1, bad, 0, 100] = float("nan")
        ops.append(c, None, y[0], y[1], ints(0, n), ints(n))
        out = torch.empty_like(q)
        ops.attention(c, q, out, ints(0, new), ints(n), max_new=new)
        outs.append(out)
    tl.check_device_errors()
    sees = bad - before
    assert torch.equal(outs[0][:sees], outs[1][:sees]) and torch.equal(outs[0][:, 4:], outs[1][:, 4:])
    assert outs[1][sees:, :4].isnan().all() and outs[0].isfinite().all()


@pytest.mark.parametrize("new", [2, 140])
def test_a_query_that_is_not_finite_stays_alone(new):
    c, q, out = attention_case(torch.float16, [300], [new], 8, 2, 64)
    q = q[:new].clone()
    q[new // 2, 3, 7], q[0, 5, 0] = float("nan"), float("inf")
    again = torch.empty_like(q)
    ops.attention(c, q, again, ints(0, new), ints(300 + new), max_new=new)
    other = torch.ones(new, 8, dtype=torch.bool, device="cuda")
    other[new // 2, 3], other[0, 5] = False, False
    assert torch.equal(again[other], out[:new].contiguous()[other]) and again[new // 2, 3].isnan().all()


def test_same_result_every_time_and_on_two_streams():
    """Bit for bit: two runs, two streams at once, a captured graph replayed while another runs."""
    gen = torch.Generator(device="cuda").manual_seed(3)
    calls = []
    for before, new in (([9000, 100], [1, 1]), ([300], [700]), ([4000, 3], [4, 2]), ([6000], [200])):
        lens = [a + n for a, n in zip(before, new)]
        c = random_cache(gen, len(new), 2, max(lens), 128, lens)
        first, lens_dev, tokens = layout(before, new)
        q = torch.randn(tokens, 8, 128, generator=gen, device="cuda").half()
        calls.append((c, q, first, lens_dev, max(new), max(lens)))

    def run(outs):
        for (c, q, first, lens, n, m), o in zip(calls, outs):
            ops.attention(c, q, o, first, lens, max_new=n, max_len=m)

    def fresh():
        return [torch.full_like(c[1], 7.0) for c in calls]

    one = fresh()
    run(one)
    torch.cuda.synchronize()
    streams, sides = [torch.cuda.Stream() for _ in range(2)], [[fresh() for _ in range(4)] for _ in range(2)]
    torch.cuda.synchronize()
    for i in range(4):
        for s, outs in zip(streams, sides):
            with torch.cuda.stream(s):
                run(outs[i])
    torch.cuda.synchronize()
    graphs = []
    for s in streams:
        outs, g = fresh(), torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            run(outs)
        graphs.append((g, outs))
    for _ in range(3):
        for s, (g, _) in zip(streams, graphs):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    tl.check_device_errors()
    for outs in [o for side in sides for o in side] + [g[1] for g in graphs]:
        assert all(torch.equal(a, b) for a, b in zip(one, outs))


def test_a_graph_follows_lengths_on_the_device():
    """A captured step: lens grow on the device between replays."""
    gen = torch.Generator(device="cuda").manual_seed(8)
    batch, kv_heads, dim = 3, 2, 64
    lens = ints(5, 200, 0)
    c = random_cache(gen, batch, kv_heads, 400, dim, lens.tolist())
    first, table = ints(0, 1, 2, 3), ops.RotaryTable(dim, 1e4)
    q, k, v = torch.randn(3, batch, 2 * kv_heads, dim, generator=gen, device="cuda").half(), None, None
    q, k, v = q[0], q[1, :, :kv_heads].contiguous(), q[2, :, :kv_heads].contiguous()
    qo, out = torch.empty_like(q), torch.empty_like(q)

    def step():
        lens.add_(1)
        ops.append(c, q, k, v, first, lens, table, qo)
        ops.attention(c, qo, out, first, lens, max_new=1, max_len=400)

    step()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        step()
    for _ in range(70):
        g.replay()
    torch.cuda.synchronize()
    tl.check_device_errors()
    assert lens.tolist() == [76, 271, 71]
    check_attention(c, qo, out, [75, 270, 70], [1, 1, 1], 2 * kv_heads, torch.float16, dim ** -0.5)


def test_long_offsets():
    """A cache of more than 2^31 bytes of codes: the last sequence's rows lie behind that."""
    rows, kv_heads, dim = 70000, 8, 128
    batch = 2 ** 31 // (rows * kv_heads * dim // 2) + 2
    c = ops.Cache4.empty(batch, kv_heads, rows, dim)
    gen = torch.Generator(device="cuda").manual_seed(2)
    new = [0] * (batch - 1) + [3]
    n = 1200
    x = torch.randn(2, n, kv_heads, dim, generator=gen, device="cuda").half()
    lens = ints(*[0] * (batch - 1), n)
    ops.append(c, None, x[0], x[1], ints(*[0] * batch, n), lens)
    k, v = torch.empty(2, n, kv_heads, dim, dtype=torch.float32, device="cuda")
    ops.read(c, k, v, ints(*[0] * batch, n), lens)
    codes, params = ref.quantise(f64(x[1]))
    assert (np.abs(f64(v) - ref.values(codes, params)) <= 2.0 ** -24 * 10).all()
    q = torch.randn(3, 16, dim, generator=gen, device="cuda").half()
    out = torch.empty_like(q)
    ops.attention(c, q, out, ints(*[0] * batch, 3), lens, max_new=3, max_len=n)
    tl.check_device_errors()
    one = ops.Cache4(*(t[-1:] for t in (c.k_codes, c.k_params, c.v_codes, c.v_params)))
    check_attention(one, q, out, [n - 3], [3], 16, torch.float16, dim ** -0.5)


def test_prompt_then_steps_together():
    """The operators as a layer uses them: a ragged prompt, then steps, against exact attention over the keys and values that were appended."""
    gen = torch.Generator(device="cuda").manual_seed(11)
    batch, heads, kv_heads, dim, dtype = 3, 8, 2, 128, torch.bfloat16
    table = ops.RotaryTable(dim, 1e4, scaling=dict(type="llama3", factor=8, original=64))
    c = new_cache(batch, kv_heads, 400, dim)
    before = [0] * batch
    for new in ([200, 1, 77], [1, 1, 1], [1, 0, 1], [3, 90, 0], [1, 1, 1]):
        first, lens, tokens = layout(before, new)
        packed = torch.randn(tokens, (heads + 2 * kv_heads) * dim, generator=gen, device="cuda").to(dtype)
        q, k, v = (t.unflatten(1, (-1, dim)) for t in packed.split([heads * dim, kv_heads * dim, kv_heads * dim], 1))
        out = torch.empty(tokens, heads, dim, dtype=dtype, device="cuda")
        ops.append(c, q, k, v, first, lens, table)
        ops.attention(c, q, out, first, lens, max_new=max(new))
        tl.check_device_errors()
        check_attention(c, q, out, before, new, heads, dtype, dim ** -0.5)
        before = [a + n for a, n in zip(before, new)]


def test_refusals_on_the_device():
    c, x = ops.Cache4.empty(2, 2, 16, 64), torch.zeros(3, 2, 64, dtype=torch.float16, device="cuda")
    first, lens, out = ints(0, 1, 3), ints(1, 2), torch.zeros_like(x)
    with pytest.raises(ValueError, match="entries"):
        ops.append(c, None, x, x, first[:2], lens)
    with pytest.raises(ValueError, match="lens"):
        ops.attention(c, x, out, first, ints(1, 2, 3))
    with pytest.raises(TypeError):
        ops.attention(c, x, out, first.long(), lens)
    with pytest.raises(TypeError):
        ops.attention(c, x.float(), out.float(), first, lens)
    with pytest.raises(TypeError):
        ops.attention(c, x, out.bfloat16(), first, lens)
    with pytest.raises(ValueError):
        ops.attention(c, x, out[:2], first, lens)
    with pytest.raises(tl.TllmError, match="overlaps"):
        ops.attention(c, x, x, first, lens)
    with pytest.raises(tl.TllmError, match="query heads"):
        ops.attention(ops.Cache4.empty(2, 2, 16, 64), torch.zeros(3, 3, 64, dtype=torch.float16, device="cuda"),
                      torch.zeros(3, 3, 64, dtype=torch.float16, device="cuda"), first, lens)
    with pytest.raises(ValueError):
        ops.append(c, None, x[:, :1], x, first, lens)
    with pytest.raises(tl.TllmError, match="apart"):
        ops.append(c, None, x[:1].expand(3, 2, 64), x, first, lens)
    with pytest.raises(ValueError, match="contiguous"):
        ops.attention(ops.Cache4(*(t[:, :, ::2] for t in (c.k_codes, c.k_params, c.v_codes, c.v_params))), x, out, first, lens)
    with pytest.raises(ValueError, match="positions"):
        ops.rotary(x, None, ints(1, 2), ops.RotaryTable(64))
    with pytest.raises(tl.TllmError, match="16-byte"):
        ops.rotary(torch.zeros(3 * 128 + 1, dtype=torch.float16, device="cuda")[1:].view(3, 2, 64), None, ints(1, 2, 3), ops.RotaryTable(64))


def test_very_many_short_sequences():
    n = 32768
    attention_case(torch.float16, [i % 4 for i in range(n)], [1] * n, 1, 1, 64, rows=64, sequences={0, 1, 2, 3, 31, 32, 1000, n - 1})


@pytest.mark.parametrize("heads,new", [(8, 1), (64, 1), (64, 2)])
def test_more_tiles_than_ctas(heads, new):
    """A CTA takes several tiles, of different sequences."""
    n = 90
    attention_case(torch.bfloat16, [(7 * i) % 93 * (i % 5 > 0) for i in range(n)], [new * (i % 7 != 2) for i in range(n)], heads, 8, 64, sequences=set(range(0, n, 5)))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("before,new,heads,kv_heads,dim", [
    ([0], [79], 32, 8, 128), ([700], [150], 24, 24, 64), ([2100], [79], 32, 8, 128), ([5000, 40], [33, 100], 16, 4, 64), ([9000], [129], 16, 2, 128), ([3000], [500], 8, 4, 128),
    ([130] * 5, [200, 0, 128, 1, 65], 8, 2, 64), ([6000], [600], 32, 8, 64)])
def test_prompts_with_an_sm_for_each_tile(dtype, before, new, heads, kv_heads, dim):
    attention_case(dtype, before, new, heads, kv_heads, dim, sequences={0, 1, 4})
    attention_case(dtype, before, new, heads, kv_heads, dim, scale=-0.2, hints=False, wide=24, sequences={0, 3})


def test_a_copy_of_a_cache_is_its_own():
    import copy
    c = new_cache(1, 1, 8, 64)
    d = copy.deepcopy(c)
    was = contents(c)
    x = torch.randn(4, 1, 64, device="cuda").half()
    ops.append(d, None, x, x, ints(0, 4), ints(4))
    k = torch.empty_like(x)
    ops.read(d, k, None, ints(0, 4), ints(4))
    tl.check_device_errors()
    assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(contents(c), was)) and (k.float() - x.float()).abs().max() < 0.5
