"""Rotary positions against 64 bits with the bound that 64-bit angles give, at any position."""
import numpy as np
import pytest
import torch

from tests import _cache4 as ref
from tests.test_gpu_cache4 import HALF_STEP, TINY, f64
from ternary_llm_b200 import cache4_ops as ops

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", list(HALF_STEP))
@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("dim,rot,tokens", [(64, 64, 5), (128, 128, 700), (80, 32, 6), (96, 24, 7), (72, 36, 3)])
@pytest.mark.parametrize("start,inverse", [(0, False), (120000, False), (2 ** 31 - 1, False), (-2 ** 31, False), (2 ** 30 + 12345, True)])
def test_angles_are_64_bits(dtype, half, dim, rot, tokens, start, inverse):
    """A cosine or sine times the amplitude is one rounding, products and their sum are one each; 2^-30 of the pair covers the turns of a
    position, 2^-65 each of up to 2^31, and the 64-bit numbers that this computes with."""
    gen = torch.Generator(device="cuda").manual_seed(dim + tokens)
    table = ops.RotaryTable(rot, 500000.0, half=half, scaling=dict(type="yarn", factor=4.0, original=4096))
    x = torch.randn(tokens, 3, dim, generator=gen, device="cuda").to(dtype)
    way = -1 if start > 2 ** 30 else 1
    position = torch.tensor([start + way * 3 * i for i in range(tokens)], dtype=torch.int32, device="cuda")
    y = torch.empty_like(x)
    ops.rotary(x, None, position, table, y, inverse=inverse)
    at = position.cpu().numpy().astype(np.int64) * (-1 if inverse else 1)
    v = f64(x)
    want = ref.rotate(v, at, table.frequencies, table.amplitude, half)
    f = np.asarray(table.frequencies, np.longdouble)
    angle = at.astype(np.longdouble)[:, None] * f
    c, s = (np.abs(fn(angle).astype(np.float64))[:, None] * table.amplitude for fn in (np.cos, np.sin))
    one, two = (slice(0, rot // 2), slice(rot // 2, rot)) if half else (slice(0, rot, 2), slice(1, rot, 2))
    size, pair = np.zeros_like(v), np.zeros_like(v)
    a, b = np.abs(v[..., one]), np.abs(v[..., two])
    size[..., one], size[..., two] = a * c + b * s, b * c + a * s
    pair[..., one] = pair[..., two] = (a + b) * table.amplitude
    inner = 3.01 * 2.0 ** -24 * size + 2.0 ** -30 * pair
    bound = inner + HALF_STEP[dtype] * (np.abs(want) + inner) + TINY[dtype]
    err = np.abs(f64(y) - want)
    assert (err[..., :rot] <= bound[..., :rot]).all(), float((err / bound)[..., :rot].max())
    assert (f64(y)[..., rot:] == v[..., rot:]).all()


@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("rot", [2, 4])
@pytest.mark.parametrize("tokens,heads", [(1, 1), (5, 33), (700, 40)])
def test_the_smallest_head(half, rot, tokens, heads):
    """16 bytes: four FP32 numbers."""
    gen = torch.Generator(device="cuda").manual_seed(rot)
    table = ops.RotaryTable(rot, 1e4, half=half)
    x = torch.randn(tokens, heads, 4, generator=gen, device="cuda")
    position, y = torch.arange(tokens, dtype=torch.int32, device="cuda"), torch.empty_like(x)
    ops.rotary(x, None, position, table, y)
    v = f64(x)
    want = ref.rotate(v, np.arange(tokens), table.frequencies, 1.0, half)
    assert (np.abs(f64(y) - want) <= 2.0 ** -24 * np.abs(want) + 3.01 * 2.0 ** -24 * 2 * np.abs(v).max(-1, keepdims=True)).all()
