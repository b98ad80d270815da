"""The operators of the 4-bit cache in 64 bits, from their definitions, with numpy."""
import numpy as np

GROUP, LIMIT = 64, 61440.0
NIBBLE = [0, 4, 1, 5, 2, 6, 3, 7]        # of value i of eight


def pack(codes):
    """uint8 [.., dim / 2] of codes [.., dim]."""
    c = codes.astype(np.uint32).reshape(*codes.shape[:-1], codes.shape[-1] // 8, 8)
    word = sum(c[..., i] << np.uint32(4 * NIBBLE[i]) for i in range(8)).astype("<u4")
    return word.view(np.uint8).reshape(*codes.shape[:-1], codes.shape[-1] // 2)


def unpack(data):
    w = np.ascontiguousarray(data).view("<u4")
    return np.stack([(w >> np.uint32(4 * n)) & 15 for n in NIBBLE], -1).reshape(*data.shape[:-1], 2 * data.shape[-1])


def quantise(x):
    """(codes [.., dim], params float16 [.., dim / 64, 2]) of rounded activations x, given as float64; NaN counts as 0."""
    x = np.clip(np.nan_to_num(x, nan=0.0, posinf=LIMIT, neginf=-LIMIT), -LIMIT, LIMIT).reshape(*x.shape[:-1], x.shape[-1] // GROUP, GROUP)
    low = x.min(-1).astype(np.float16)
    d = (x - low.astype(np.float64)[..., None]).astype(np.float32)             # a difference and a quotient are FP32 operations
    s = ((x.max(-1) - low.astype(np.float64)).astype(np.float32) / np.float32(15)).astype(np.float16)
    with np.errstate(divide="ignore", invalid="ignore"):
        c = np.clip(np.rint(d / s.astype(np.float32)[..., None]), 0, 15)
    c = np.where(s[..., None] > 0, c, 0)
    return c.reshape(*x.shape[:-2], x.shape[-2] * GROUP).astype(np.uint8), np.stack([s, low], -1)


def values(codes, params):
    """float64 [.., dim] of codes [.., dim]."""
    p = np.repeat(params.astype(np.float64), GROUP, axis=-2)
    return codes * p[..., 0] + p[..., 1]


def rotate(x, positions, frequencies, amplitude, half):
    """x float64 [tokens, heads, dim]."""
    f = np.asarray(frequencies, np.longdouble)
    angle = np.asarray(positions, np.longdouble)[:, None] * f
    c, s = (np.asarray(fn(angle), np.float64)[:, None] * amplitude for fn in (np.cos, np.sin))
    rot, y = 2 * len(f), x.copy()
    one, two = (slice(0, rot // 2), slice(rot // 2, rot)) if half else (slice(0, rot, 2), slice(1, rot, 2))
    y[..., one], y[..., two] = x[..., one] * c - x[..., two] * s, x[..., two] * c + x[..., one] * s
    return y


def attention(q, k, v, position, scale, v_size):
    """One head: q [n, dim] at `position` [n], k and v [m, dim].  (result, sum of weights times v_size, largest sum of |q k scale|): a
    score is a sum of dim terms of these sizes, whatever the sign of the scale, and roundings are in proportion to them."""
    s = q @ k.T * scale
    sees = np.arange(len(k))[None] <= position[:, None]
    reach = np.where(sees, np.abs(q) @ np.abs(k).T * abs(scale), 0).max(-1, initial=0.0)
    s = np.where(sees, s, -np.inf)
    top = s.max(-1, initial=-np.inf, keepdims=True)
    p = np.where(sees, np.exp(s - np.where(np.isfinite(top), top, 0)), 0)
    total = p.sum(-1, keepdims=True)
    p = p / np.where(total > 0, total, 1)
    return p @ v, p @ v_size, reach
