"""Host side of the 4-bit cache: frequencies and turns of rotary positions against exact arithmetic, the layout's helpers, refusals that need
no GPU."""
import copy
import ctypes
import math
from fractions import Fraction

import numpy as np
import pytest
import torch

import ternary_llm_b200 as tl
from tests import _cache4 as ref
from ternary_llm_b200 import _lib, cache4_ops as ops

# 1 / (2 pi) to 60 digits
TURN = Fraction(159154943091895335768883763372514362034459645740456448747667, 10 ** 60)


@pytest.mark.parametrize("rot,base", [(2, 10000.0), (64, 500000.0), (128, 10000.0), (80, 1000000.0)])
def test_plain_frequencies(rot, base):
    f, a = ops.rotary_frequencies(rot, base)
    assert a == 1.0 and len(f) == rot // 2
    np.testing.assert_allclose(f, base ** (-2 * np.arange(rot // 2) / rot), rtol=4e-16 * math.log(base) * 4)


def test_scaled_frequencies():
    rot, base, factor, length = 128, 10000.0, 16.0, 4096
    plain = np.array(ops.rotary_frequencies(rot, base)[0])
    f, a = ops.rotary_frequencies(rot, base, dict(type="linear", factor=factor))
    assert a == 1.0 and np.allclose(f, plain / factor, rtol=1e-15)
    f, a = ops.rotary_frequencies(rot, base, dict(type="ntk", factor=factor))
    assert a == 1.0 and f[0] == 1.0 and np.isclose(f[-1], plain[-1] / factor, rtol=1e-12)      # the slowest pair by the whole factor
    f, a = ops.rotary_frequencies(rot, base, dict(type="yarn", factor=factor, original=length))
    f, turns = np.array(f), length * plain / (2 * math.pi)
    assert a == pytest.approx(0.1 * math.log(factor) + 1, rel=1e-7)
    assert (f[turns > 33] == plain[turns > 33]).all() and np.allclose(f[turns < 0.95], plain[turns < 0.95] / factor, rtol=1e-15)
    assert (np.diff(f) < 0).all() and (f <= plain).all() and (f >= plain / factor * (1 - 1e-15)).all()
    f, a = ops.rotary_frequencies(rot, base, dict(type="llama3", factor=factor, original=length))
    f = np.array(f)
    assert a == 1.0
    assert (f[turns >= 4] == plain[turns >= 4]).all() and np.allclose(f[turns <= 1], plain[turns <= 1] / factor, rtol=1e-15)
    between = (turns > 1) & (turns < 4)
    mix = (turns[between] - 1) / 3
    assert between.any() and np.allclose(f[between], (1 - mix) * plain[between] / factor + mix * plain[between], rtol=1e-13)


def test_turns_are_exact():
    f = ops.rotary_frequencies(128, 500000.0)[0] + [1.0, 0.0, 2 * math.pi, 3.5, -0.25]
    for x, t in zip(f, ops.rotary_turns(f)):
        want = Fraction(x) * TURN * 2 ** 64
        off = (Fraction(t) - want) % 2 ** 64
        off = min(off, 2 ** 64 - off)
        assert off <= 1 + 2 * Fraction(x.__abs__()), x          # a rounding in 64 bits of at most a turn, one to a unit


@pytest.mark.parametrize("args,word", [
    ((0, 10000.0), "rot_dim"), ((63, 10000.0), "rot_dim"), ((514, 1e4), "rot_dim"), ((64, 1.0), "base"), ((64, float("nan")), "base"),
    ((64, 1e4, dict(type="linear", factor=0.5)), "factor"), ((64, 1e4, dict(type="linear", factor=float("inf"))), "factor"),
    ((64, 1e4, dict(type="yarn", factor=4, original=0)), "original"), ((64, 1e4, dict(type="llama3", factor=4, original=10, low=4, high=4)), "low"),
    ((2, 1e4, dict(type="ntk", factor=4)), "rot_dim")])
def test_frequencies_refused(args, word):
    with pytest.raises(tl.TllmError, match=word):
        ops.rotary_frequencies(*args)


def test_scalings_refused_in_python():
    for scaling in (dict(type="none"), dict(factor=3.0), dict(type="linear", factor=2, beta=1), dict(type="yarn", factor=2)):
        with pytest.raises(ValueError):
            ops.rotary_frequencies(64, 1e4, scaling)
    with pytest.raises(ValueError):
        ops.RotaryTable(64, frequencies=[1.0], device="cpu")
    with pytest.raises(tl.TllmError):
        ops.rotary_turns([float("inf")])
    t = ops.RotaryTable(4, frequencies=[1.0, 0.5], amplitude=2.0, device="cpu")
    assert t.amplitude == 2.0 and t.turns.dtype == torch.int64 and (t.turns.numpy().view(np.uint64) == np.array(ops.rotary_turns([1.0, 0.5]), np.uint64)).all()


def test_layout_of_the_checks():
    c = np.random.default_rng(0).integers(0, 16, (3, 128))
    assert (ref.unpack(ref.pack(c)) == c).all()
    assert ref.pack(np.arange(8)[None]).tolist() == [[0x20, 0x64, 0x31, 0x75]]
    x = np.array([np.linspace(-1, 2, 64), np.full(64, 0.5), np.r_[np.zeros(63), 1e6]])
    codes, params = ref.quantise(x)
    got = ref.values(codes, params)
    assert np.abs(got[0] - x[0]).max() <= 0.1 + 2 ** -9 and (got[1] == 0.5).all() and (got[2, :63] == 0).all() and abs(got[2, 63] - ref.LIMIT) <= 64


P = 0x10000          # an address that is never followed: every call below is refused first


def cache(**kw):
    d = dict(k_codes=P, k_params=P, v_codes=P, v_params=P, batch=2, kv_heads=2, rows=256, dim=64)
    d.update(kw)
    return _lib.Cache4Desc(*d.values())


def heads(p=P, ld=128):
    return ctypes.byref(_lib.HeadsDesc(p, ld))


def table(turns=P, rot=64, amplitude=1.0):
    return ctypes.byref(_lib.RotaryTableDesc(turns, rot, 1, amplitude))


def refused(status, call, *args):
    assert call(*args, None) == status, tl.lib().tllm_b200_last_error()


NULL, ALIGN, SHAPE, SIZE = -1, -2, -3, -9


def test_rotary_refusals():
    f = tl.lib().tllm_b200_rotary

    def call(status, type=0, table_=None, pos=P, tokens=3, q=None, qo=None, nh=2, k=None, ko=None, nk=0, dim=64):
        refused(status, f, type, table() if table_ is None else table_, pos, tokens, heads() if q is None else q, heads(P * 16) if qo is None else qo, nh,
                k, ko, nk, dim, 0)

    call(SHAPE, type=3)
    call(SHAPE, type=-1)
    call(NULL, pos=None)
    call(NULL, q=heads(None))
    call(NULL, table_=table(None))
    call(SHAPE, table_=table(rot=66))
    call(SHAPE, table_=table(rot=63))
    call(SHAPE, table_=table(rot=0))
    call(SHAPE, table_=table(amplitude=float("inf")))
    call(ALIGN, table_=table(P + 4))
    call(SHAPE, tokens=-1)
    call(SHAPE, nh=0)
    call(SHAPE, dim=60)
    call(SHAPE, dim=520)
    call(NULL, nk=2)
    call(NULL, k=heads(), nk=2)
    call(ALIGN, q=heads(P + 8))
    call(ALIGN, q=heads(P, 132))
    call(SHAPE, q=heads(P, 127))
    call(ALIGN, pos=P + 2)
    call(SHAPE, q=heads(P), qo=heads(P + 16))                    # overlaps, and is not the same
    call(SHAPE, q=heads(P, 256), qo=heads(P + 256, 264))
    call(SHAPE, q=heads(P, 128), qo=heads(P, 256))


def test_cache_refusals():
    h = tl.lib()
    good = dict(c=cache(), type=0, first=P, lens=P, tokens=3)

    def append(status, table_=None, q=heads(), qo=heads(), nh=2, k=heads(), v=heads(), **kw):
        a = dict(good, **kw)
        refused(status, h.tllm_b200_cache4_append, ctypes.byref(a["c"]), a["type"], table_, a["first"], a["lens"], a["tokens"], q, qo, nh, k, v)

    def read(status, k=heads(), v=heads(), **kw):
        a = dict(good, **kw)
        refused(status, h.tllm_b200_cache4_read, ctypes.byref(a["c"]), a["type"], a["first"], a["lens"], a["tokens"], k, v)

    def attend(status, q=heads(P, 256), out=heads(P * 16, 256), nh=4, scale=1.0, new=0, most=0, ws=P, size=1 << 40, **kw):
        a = dict(good, **kw)
        refused(status, h.tllm_b200_cache4_attention, ctypes.byref(a["c"]), a["type"], a["first"], a["lens"], a["tokens"], q, out, nh, scale, new, most,
                ws, size)

    for f in (append, read, attend):
        f(NULL, c=cache(k_codes=None))
        f(NULL, c=cache(v_params=None))
        f(ALIGN, c=cache(v_codes=P + 8))
        f(SHAPE, c=cache(dim=96))
        f(SHAPE, c=cache(rows=0))
        f(SHAPE, c=cache(batch=-1))
        f(SHAPE, c=cache(kv_heads=0))
        f(NULL, first=None)
        f(NULL, lens=None)
        f(ALIGN, lens=P + 1)
        f(SHAPE, tokens=-1)
        f(SHAPE, type=7)
    append(SHAPE, type=2)
    attend(SHAPE, type=2)
    append(NULL, k=heads(None))
    append(NULL, v=None)
    append(NULL, q=None)
    append(NULL, qo=None)
    append(SHAPE, nh=-1)
    append(SHAPE, table_=table(rot=128))
    append(ALIGN, v=heads(P + 2))
    append(SHAPE, q=heads(), qo=heads(P + 32))
    read(NULL, k=None, v=None)
    read(SHAPE, v=heads(P, 120))
    attend(SHAPE, nh=3)
    attend(SHAPE, nh=0)
    attend(SHAPE, scale=float("nan"))
    attend(SHAPE, new=-1)
    attend(SHAPE, most=-1)
    attend(SHAPE, out=heads(P, 256))
    attend(SHAPE, out=heads(P + 512, 264))
    attend(ALIGN, out=heads(P * 16 + 8, 256))
    n = ctypes.c_size_t()
    assert h.tllm_b200_cache4_workspace(ctypes.byref(cache()), 3, 3, 0, 0, ctypes.byref(n)) == SHAPE
    assert h.tllm_b200_cache4_workspace(ctypes.byref(cache()), 3, 4, 0, 0, None) == NULL
    assert h.tllm_b200_cache4_workspace(ctypes.byref(cache()), -1, 4, 0, 0, ctypes.byref(n)) == SHAPE


def test_shapes_refused_in_python():
    kc, kp = torch.zeros(2, 2, 32, 32, dtype=torch.uint8), torch.zeros(2, 2, 32, 1, 2, dtype=torch.float16)
    c = ops.Cache4(kc, kp, kc, kp)
    assert (c.batch, c.kv_heads, c.rows, c.dim) == (2, 2, 32, 64)
    for bad in ((kc[0], kp, kc, kp), (kc, kp[..., 0], kc, kp), (kc, kp, kc[:1], kp), (kc[..., :16], kp, kc[..., :16], kp)):
        with pytest.raises(ValueError):
            ops.Cache4(*bad)
    with pytest.raises(ValueError, match="CUDA"):               # no CPU path
        c._desc()
    x = torch.zeros(3, 2, 64, dtype=torch.float16)
    t = ops.RotaryTable(64, device="cpu")
    with pytest.raises(TypeError):
        ops.rotary(x.double(), None, torch.zeros(3, dtype=torch.int32), t)
    with pytest.raises(ValueError):
        ops.rotary(x[0], None, torch.zeros(3, dtype=torch.int32), t)
    with pytest.raises(ValueError, match="k_out"):
        ops.rotary(x, None, torch.zeros(3, dtype=torch.int32), t, k_out=x)
    with pytest.raises(ValueError, match="behind one another"):
        ops._rows(x.transpose(0, 1), torch.float16, "q", 2, 3, 64)


def test_outputs_may_not_lie_over_other_inputs():
    h = tl.lib()
    three = ctypes.byref(_lib.RotaryTableDesc(P, 64, 1, 1.0))

    def rotary(q, qo, k, ko):
        refused(SHAPE, h.tllm_b200_rotary, 0, three, P, 3, q, qo, 2, k, ko, 1, 64, 0)

    rotary(heads(P), heads(P * 2), heads(P * 2), heads(P * 2))                     # q_out over k
    rotary(heads(P), heads(P), heads(P * 2, 64), heads(P, 64))                     # k_out over q
    rotary(heads(P), heads(P * 2), heads(P * 4, 64), heads(P * 2 + 256, 64))       # k_out over q_out
    rotary(heads(P, 192), heads(P, 192), heads(P + 128, 192), heads(P + 128, 192))  # rows of 192, keys begin inside the queries' 256 bytes
    c = cache()
    refused(SHAPE, h.tllm_b200_cache4_append, ctypes.byref(c), 0, None, P, P, 3, heads(P), heads(P * 2), 2, heads(P * 2), heads(P * 4))
    refused(SHAPE, h.tllm_b200_cache4_append, ctypes.byref(c), 0, None, P, P, 3, heads(P), heads(P * 2), 2, heads(P * 4), heads(P * 2 + 16))
    refused(SHAPE, h.tllm_b200_cache4_read, ctypes.byref(c), 0, P, P, 3, heads(P), heads(P + 16))
    refused(SHAPE, h.tllm_b200_rotary, 0, three, P, 2 ** 31 - 1, heads(), heads(), 2, None, None, 0, 64, 0)


def test_tensors_of_a_cache_and_a_table_are_set_once():
    kc, kp = torch.zeros(1, 1, 8, 32, dtype=torch.uint8), torch.zeros(1, 1, 8, 1, 2, dtype=torch.float16)
    c, t = ops.Cache4(kc, kp, kc.clone(), kp.clone()), ops.RotaryTable(64, 500000.0, half=False, scaling=dict(type="linear", factor=2.0), amplitude=1.5, device="cpu")
    for o, name, value in ((c, "k_codes", kc.clone()), (c, "rows", 4), (t, "turns", t.turns.clone()), (t, "amplitude", 1.0)):
        with pytest.raises(AttributeError, match="make another"):
            setattr(o, name, value)
    d, u = copy.deepcopy(c), copy.deepcopy(t)
    assert d.k_codes.data_ptr() != c.k_codes.data_ptr() and torch.equal(d.k_codes, c.k_codes) and d.rows == 8
    assert u.turns.data_ptr() != t.turns.data_ptr() and torch.equal(u.turns, t.turns)
    assert (u.rot_dim, u.half, u.amplitude, u.frequencies) == (64, False, 1.5, t.frequencies)
    assert copy.copy(c).k_codes is c.k_codes
