"""Attention of few rows over the 4-bit cache against 64 bits, with the bound that its arithmetic gives.

Per group of 64 channels a query is x u with whole x, |x| <= 32512, and u = top / 32512, top its largest entry: half a unit and two FP32
roundings of a product of that size, below top / 64500.  Scores are then sums of whole numbers, met by the FP32 numbers s, l and u: ten
roundings of 2^-24, relative to |q| (s c + |l|), up to the argument of the exponential, which is good to 2^-22.  A weight meets s (c - 8) as 11
bits of weight * s, half a step of which is 2^-11, or where it is below FP16's normal numbers 2^-25 in a unit that is a 64th of the
largest weight * |s| that the row sees; it meets l + 8 s in FP32.  Sums: at most one rounding of 2^-23 for each eight positions, and some 40.
"""
import numpy as np

from tests import _cache4 as ref


def check_few(c, q, out, before, new, heads, half_step, tiny, scale, sequences=None):
    kc, kp, vc, vp = (t.cpu().numpy() for t in (c.k_codes, c.k_params, c.v_codes, c.v_params))
    per, dim, at = heads // c.kv_heads, c.dim, 0
    x, y = (t.double().cpu().numpy() for t in (q, out))
    for b, (a, n) in enumerate(zip(before, new)):
        m = a + n
        for g in range(c.kv_heads if n and (sequences is None or b in sequences) else 0):
            pk, pv = (np.repeat(p[b, g, :m].astype(np.float64), 64, axis=-2) for p in (kp, vp))
            k, v = ref.unpack(kc[b, g, :m]) * pk[..., 0] + pk[..., 1], ref.unpack(vc[b, g, :m]) * pv[..., 0] + pv[..., 1]
            rows = x[at:at + n, g * per:(g + 1) * per].reshape(n * per, dim)
            sees = np.arange(m)[None] <= np.repeat(np.arange(a, m), per)[:, None]
            score = np.where(sees, rows @ k.T * scale, -np.inf)
            w = np.exp(score - score.max(-1, keepdims=True))
            w /= w.sum(-1, keepdims=True)
            groups = range(dim // 64)
            top = [np.abs(rows[:, 64 * i:64 * i + 64]).max(-1, keepdims=True) for i in groups]
            digit = sum(t / 64500 @ np.abs(k[:, 64 * i:64 * i + 64]).sum(-1)[None] for i, t in zip(groups, top)) * abs(scale)
            terms = np.abs(rows) @ (np.abs(k - pk[..., 1]) + np.abs(pk[..., 1])).T * abs(scale)
            e = digit + 10 * 2.0 ** -24 * np.where(sees, terms, 0).max(-1, keepdims=True)
            e = 1.02 * w * (e + 2.0 ** -22)
            mid = pv[..., 1] + 8 * pv[..., 0]
            want = w @ v
            size = np.abs(v - mid) + np.abs(mid)
            floor = m * 2.0 ** -28 * np.repeat((w[:, :, None] * np.abs(vp[b, g, :m, :, 0].astype(np.float64))[None]).max(1), 64, axis=-1)
            bound = e @ np.abs(v) + np.abs(want) * e.sum(-1, keepdims=True) + 2.0 ** -11 * (w @ np.abs(v - mid)) + (m / 8 + 40) * 2.0 ** -23 * (w @ size) + floor
            bound = bound + half_step * (np.abs(want) + bound) + tiny
            err = np.abs(y[at:at + n, g * per:(g + 1) * per].reshape(n * per, dim) - want)
            assert (err <= bound).all(), (b, g, float((err / bound).max()))
        at += n
