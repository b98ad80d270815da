"""A key/value cache held in 4 bits (include/tllm_b200_cache4.h) on torch tensors: rotary positions,
append, read back and attention for sequences of different lengths in one call.

    cache = Cache4.empty(batch, kv_heads, max_seq, dim)
    table = RotaryTable(dim, 500000.0, scaling=dict(type="llama3", factor=32, original=8192))
    append(cache, q, k, v, first, lens, table)           # q turned in place, k and v into the cache
    attention(cache, q, out, first, lens, max_new=1)

Activations are [tokens, heads, dim] (rows may lie apart, as parts of a wider tensor do); sequence b has the
rows first[b] .. first[b + 1] - 1, at the last of its lens[b] positions; both are int32 CUDA tensors.  Checks
of types, shapes and devices, then one call of the C ABI on torch's current stream; nothing here computes with
torch operations.  A cache and a table stand for the memory that they were made of: a call is refused once one of their
tensors is at other memory, or its storage has another size.
"""
from __future__ import annotations

import ctypes
import operator

import torch

from . import _lib
from .ops import _chk, _stream

GROUP = 64
TYPES = {torch.float16: 0, torch.bfloat16: 1, torch.float32: 2}
SCALINGS = {"linear": 1, "ntk": 2, "yarn": 3, "llama3": 4}


def _int(v) -> int:
    """A whole number as an int of C holds it: the largest for one above, -1 for a negative one."""
    return max(-1, min(operator.index(v), 2 ** 31 - 1))


def _frequencies(rot_dim: int, base: float, scaling: dict | None):
    """(C array, factor of the result)."""
    s = dict(scaling or {})
    kind = s.pop("type", None)
    if scaling is not None and kind not in SCALINGS:
        raise ValueError(f"scaling type {kind!r}: one of {', '.join(SCALINGS)}")
    d = _lib.RotaryScaling(SCALINGS.get(kind, 0), float(s.pop("factor", 1.0)))
    if kind in ("yarn", "llama3"):
        if "original" not in s:
            raise ValueError(f"scaling {kind!r} needs the original length")
        d.original = float(s.pop("original"))
        d.low, d.high = (float(s.pop("beta_slow", 1.0)), float(s.pop("beta_fast", 32.0))) if kind == "yarn" else \
            (float(s.pop("low", 1.0)), float(s.pop("high", 4.0)))
    if s:
        raise ValueError(f"scaling: unknown {', '.join(map(repr, s))}")
    rot_dim = _int(rot_dim)
    f, amplitude = (ctypes.c_double * max(1, min(rot_dim, 512) // 2))(), ctypes.c_float()          # the library writes no more than 256
    _lib.check(_lib.lib().tllm_b200_rotary_frequencies(rot_dim, base, ctypes.byref(d), f, ctypes.byref(amplitude)))
    return f, amplitude.value


def _turns(frequencies, n: int):
    out = (ctypes.c_uint64 * max(1, n))()
    _lib.check(_lib.lib().tllm_b200_rotary_turns(frequencies, n, out))
    return out


def rotary_frequencies(rot_dim: int, base: float, scaling: dict | None = None):
    """(angles a position of the rot_dim / 2 pairs, factor of the result).  scaling: type "linear" or "ntk"
    (factor), "yarn" (factor, original length, beta_fast, beta_slow) or "llama3" (factor, original, low, high)."""
    f, amplitude = _frequencies(rot_dim, base, scaling)
    return list(f), amplitude


def rotary_turns(frequencies):
    """The frequencies in turns a position, as 64-bit fractions."""
    n = len(frequencies)
    return list(_turns((ctypes.c_double * max(1, n))(*frequencies), n))[:n]


class _Fixed:
    """A C struct that begins with the addresses of tensors, set once.  The tensors are asked in each call whether they are still at that memory."""
    _native = None

    def _keep(self, struct, *tensors):
        """Native calls take the struct as it is here; any device or layout that they cannot take goes through _desc, which says what is wrong."""
        for t in tensors:
            if t.numel() and (t.storage_offset() + t.numel()) * t.element_size() > t.untyped_storage().nbytes():
                raise ValueError(f"a tensor of {tuple(t.shape)} whose storage holds {t.untyped_storage().nbytes()} bytes")
        parts = (part for t in tensors for s in (t.untyped_storage(),) for part in (t, s, s.nbytes()))
        device = tensors[0].get_device() if all(t.is_cuda and t.is_contiguous() and t.device == tensors[0].device for t in tensors) else -1
        self._native = bytes(struct), device, *parts

    def _same(self, struct, *names):
        """The struct, which names the tensors' present addresses, where these are what the handle was made of."""
        parts = self._native[2:]
        for i, name in enumerate(names):
            t, s, n = parts[3 * i:3 * i + 3]
            if s.nbytes() != n or bytes(struct)[8 * i:8 * i + 8] != self._native[0][8 * i:8 * i + 8]:
                raise ValueError(f"the memory of {name} is not what it was: make another {type(self).__name__}")
        return struct

    def __setattr__(self, name, value):
        if self._native is not None:
            raise AttributeError(f"{type(self).__name__}.{name} cannot be changed: make another {type(self).__name__}")
        object.__setattr__(self, name, value)


class RotaryTable(_Fixed):
    """Rotary positions of the first rot_dim entries of a head.  half: pairs (i, i + rot_dim / 2), else (2 i, 2 i + 1).
    frequencies: angles a position, instead of base and scaling; amplitude: factor of the result (default: the scaling's)."""

    def __init__(self, rot_dim: int, base: float = 10000.0, half: bool = True, scaling: dict | None = None, frequencies=None,
                 amplitude: float | None = None, device=None):
        if frequencies is None:
            f, own = _frequencies(rot_dim, base, scaling)
        else:
            f, own = (ctypes.c_double * max(1, len(frequencies)))(*frequencies), 1.0
            if 2 * len(frequencies) != rot_dim:
                raise ValueError(f"{len(frequencies)} frequencies for {rot_dim} entries")
        self.rot_dim, self.half, self._f = rot_dim, bool(half), f
        self.amplitude = own if amplitude is None else float(amplitude)
        turns = torch.frombuffer(_turns(f, rot_dim // 2), dtype=torch.int64, count=rot_dim // 2)
        self.turns = turns.clone() if device is not None and torch.device(device).type == "cpu" else turns.to("cuda" if device is None else device)
        self._keep(_lib.RotaryTableDesc(self.turns.data_ptr(), rot_dim, int(self.half), self.amplitude), self.turns)

    def __reduce__(self):
        return RotaryTable, (self.rot_dim, 0.0, self.half, None, self.frequencies, self.amplitude, str(self.turns.device))

    @property
    def frequencies(self):
        return list(self._f)[:self.rot_dim // 2]

    def _desc(self):
        return self._same(_lib.RotaryTableDesc(_chk(self.turns, torch.int64, "turns", self.rot_dim // 2), self.rot_dim, int(self.half), self.amplitude), "turns")


class Cache4(_Fixed):
    """Codes uint8 [batch, kv_heads, rows, dim / 2] and params float16 [batch, kv_heads, rows, dim / 64, 2] of keys and values.
    Params that append did not write: finite, of either sign, and s c + l of every code within FP16's range."""

    def __init__(self, k_codes, k_params, v_codes, v_params):
        if k_codes.dim() != 4:
            raise ValueError(f"k_codes must be [batch, kv_heads, rows, dim / 2], got {tuple(k_codes.shape)}")
        self.batch, self.kv_heads, self.rows, self.dim = *k_codes.shape[:3], 2 * k_codes.shape[3]
        if self.dim not in (64, 128):
            raise ValueError(f"head size {self.dim}: 64 or 128")
        for name, t, shape in (("k_codes", k_codes, k_codes.shape), ("v_codes", v_codes, k_codes.shape),
                               ("k_params", k_params, (*k_codes.shape[:3], self.dim // GROUP, 2)),
                               ("v_params", v_params, (*k_codes.shape[:3], self.dim // GROUP, 2))):
            if tuple(t.shape) != tuple(shape):
                raise ValueError(f"{name} must be {tuple(shape)}, got {tuple(t.shape)}")
        self.k_codes, self.k_params, self.v_codes, self.v_params = k_codes, k_params, v_codes, v_params
        all4 = (k_codes, k_params, v_codes, v_params)
        types = tuple(t.dtype for t in all4) == (torch.uint8, torch.float16) * 2
        self._keep(_lib.Cache4Desc(*(t.data_ptr() if types else None for t in all4), self.batch, self.kv_heads, self.rows, self.dim), *all4)

    def __reduce__(self):
        return Cache4, (self.k_codes, self.k_params, self.v_codes, self.v_params)

    @classmethod
    def empty(cls, batch: int, kv_heads: int, rows: int, dim: int, device=None):
        """A cache whose contents are not set."""
        device = "cuda" if device is None else device
        return cls(*(torch.empty(batch, kv_heads, rows, *last, dtype=t, device=device)
                     for last, t in (((dim // 2,), torch.uint8), ((dim // GROUP, 2), torch.float16)) * 2))

    def _desc(self):
        return self._same(_lib.Cache4Desc(_chk(self.k_codes, torch.uint8, "k_codes"), _chk(self.k_params, torch.float16, "k_params"),
                                          _chk(self.v_codes, torch.uint8, "v_codes"), _chk(self.v_params, torch.float16, "v_params"),
                                          self.batch, self.kv_heads, self.rows, self.dim), "k_codes", "k_params", "v_codes", "v_params")


def _rows(t, dtype, name: str, tokens: int, heads: int, dim: int):
    """[tokens, heads, dim] whose rows may lie apart."""
    if tuple(t.shape) != (tokens, heads, dim):
        raise ValueError(f"{name} must be {(tokens, heads, dim)}, got {tuple(t.shape)}")
    if heads and tokens and not t.is_contiguous() and (t.stride(2) != 1 or (heads > 1 and t.stride(1) != dim)):
        raise ValueError(f"{name}: the heads of a row must lie behind one another")
    p = _chk(t if t.is_contiguous() else t.as_strided((1,), (1,)), dtype, name)
    return _lib.HeadsDesc(p, t.stride(0) if tokens > 1 else heads * dim)


def _type(t, name: str, allowed) -> int:
    if t.dtype not in allowed:
        raise TypeError(f"{name} must be {' or '.join(str(a) for a in allowed)}, got {t.dtype}")
    if t.dim() != 3:
        raise ValueError(f"{name} must be [tokens, heads, dim], got {tuple(t.shape)}")
    return TYPES[t.dtype]


def _seqs(cache, first, lens):
    for name, t, n in (("first", first, cache.batch + 1), ("lens", lens, cache.batch)):
        if t.numel() != n:
            raise ValueError(f"{name} holds {t.numel()} entries, the cache's {cache.batch} sequences need {n}")
    return _chk(first, torch.int32, "first"), _chk(lens, torch.int32, "lens")


def _ref(d):
    return None if d is None else ctypes.byref(d)


def rotary(q, k, positions, table: RotaryTable, q_out=None, k_out=None, inverse: bool = False) -> None:
    """Turns q [tokens, heads, dim] and k [tokens, kv_heads, dim] (or None) by positions int32 [tokens], in place where no
    output is given; inverse turns back (the gradient).  FP16, BF16 or FP32."""
    st = _lib.host().rotary(table._native, q, k, positions, q_out, k_out, inverse)
    if st is not None:
        return _lib.check(st)
    kind = _type(q, "q", tuple(TYPES))
    tokens, heads, dim = q.shape
    if k is None and k_out is not None:
        raise ValueError("k_out without k")
    kv_heads = 0 if k is None else k.shape[1] if k.dim() == 3 else -1
    rows = [None if t is None else _rows(t, q.dtype, name, tokens, n, dim) for name, t, n in
            (("q", q, heads), ("q_out", q if q_out is None else q_out, heads), ("k", k, kv_heads), ("k_out", k if k_out is None else k_out, kv_heads))]
    _lib.check(_lib.lib().tllm_b200_rotary(
        kind, ctypes.byref(table._desc()), _chk(positions, torch.int32, "positions", tokens), tokens, _ref(rows[0]), _ref(rows[1]), heads,
        _ref(rows[2]), _ref(rows[3]), kv_heads, dim, int(bool(inverse)), _stream()))


def append(cache: Cache4, q, k, v, first, lens, table: RotaryTable | None = None, q_out=None) -> None:
    """Turns q (or None) into q_out (default: in place) and k, and writes k and v to the cache.  FP16 or BF16."""
    st = _lib.host().cache4_append(cache._native, None if table is None else table._native, q, k, v, first, lens, q_out)
    if st is not None:
        return _lib.check(st)
    kind = _type(k, "k", (torch.float16, torch.bfloat16))
    tokens, d = k.shape[0], cache._desc()
    if q is None and q_out is not None:
        raise ValueError("q_out without q")
    heads = 0 if q is None else q.shape[1] if q.dim() == 3 else -1
    rows = [None if t is None else _rows(t, k.dtype, name, tokens, n, cache.dim) for name, t, n in
            (("q", q, heads), ("q_out", q if q_out is None else q_out, heads), ("k", k, cache.kv_heads), ("v", v, cache.kv_heads))]
    f, n = _seqs(cache, first, lens)
    _lib.check(_lib.lib().tllm_b200_cache4_append(
        ctypes.byref(d), kind, _ref(None if table is None else table._desc()), f, n, tokens, _ref(rows[0]), _ref(rows[1]), heads, _ref(rows[2]),
        _ref(rows[3]), _stream()))


def read(cache: Cache4, k, v, first, lens) -> None:
    """Writes the keys and values at the rows' positions, as the cache holds them, to k and v [tokens, kv_heads, dim] (one of
    them may be None).  FP16, BF16 or FP32."""
    st = _lib.host().cache4_read(cache._native, k, v, first, lens)
    if st is not None:
        return _lib.check(st)
    some = v if k is None else k
    if some is None:
        raise ValueError("neither k nor v")
    kind, d = _type(some, "v" if k is None else "k", tuple(TYPES)), cache._desc()
    tokens = some.shape[0]
    rows = [None if t is None else _rows(t, some.dtype, name, tokens, cache.kv_heads, cache.dim) for name, t in (("k", k), ("v", v))]
    f, n = _seqs(cache, first, lens)
    _lib.check(_lib.lib().tllm_b200_cache4_read(ctypes.byref(d), kind, f, n, tokens, _ref(rows[0]), _ref(rows[1]), _stream()))


def attention(cache: Cache4, q, out, first, lens, scale: float | None = None, max_new: int = 0, max_len: int = 0) -> None:
    """out = softmax(scale q k') v over the positions up to each row's own (scale: dim ** -0.5).  max_new: about the most rows
    of a sequence, 0 where the caller does not know (then their average); it chooses the way of the work, and ways differ in
    the order of sums and in what they round to 11 bits.  max_len: no sequence holds more positions (0: the cache's rows);
    workspaces are as large as that needs.  FP16 or BF16."""
    if scale is None:
        scale = cache.dim ** -0.5
    st = _lib.host().cache4_attention(cache._native, q, out, first, lens, scale, max_new, max_len)
    if st is not None:
        return _lib.check(st)
    max_new, max_len = _int(max_new), _int(max_len)
    kind, d = _type(q, "q", (torch.float16, torch.bfloat16)), cache._desc()
    tokens, heads = q.shape[:2]
    x, y = _rows(q, q.dtype, "q", tokens, heads, cache.dim), _rows(out, q.dtype, "out", tokens, heads, cache.dim)
    f, n = _seqs(cache, first, lens)
    h, need = _lib.lib(), ctypes.c_size_t()
    _lib.check(h.tllm_b200_cache4_workspace(ctypes.byref(d), tokens, heads, max_new, max_len, ctypes.byref(need)))
    ws = torch.empty(need.value, dtype=torch.uint8, device=q.device) if need.value else None
    _lib.check(h.tllm_b200_cache4_attention(
        ctypes.byref(d), kind, f, n, tokens, ctypes.byref(x), ctypes.byref(y), heads, scale, max_new, max_len,
        None if ws is None else ws.data_ptr(), need.value, _stream()))
