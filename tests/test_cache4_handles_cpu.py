"""What a call of the 4-bit cache hands to the library after the tensors behind a handle changed: the native module with tensors that say they
are on a GPU, and functions that write down what they are given in the place of the library's."""
import ctypes

import pytest
import torch

from ternary_llm_b200 import _lib, cache4_ops as ops

VP, INT = ctypes.c_void_p, ctypes.c_int


class OnDevice(torch.Tensor):
    """A CPU tensor that says it is on device 0."""
    is_cuda = property(lambda self: True)

    def get_device(self):
        return 0


def on_device(*shape, dtype):
    return torch.zeros(*shape, dtype=dtype).as_subclass(OnDevice)


@pytest.fixture
def seen():
    """(structs that calls were given, the native module)."""
    host = _lib.host()                                   # builds nothing on the device
    from ternary_llm_b200 import _hostcall
    calls = []

    def cache(p):
        return _lib.Cache4Desc.from_buffer_copy(ctypes.string_at(p, ctypes.sizeof(_lib.Cache4Desc)))

    def table(p):
        return _lib.RotaryTableDesc.from_buffer_copy(ctypes.string_at(p, ctypes.sizeof(_lib.RotaryTableDesc)))

    rotary = ctypes.CFUNCTYPE(INT, INT, VP, VP, INT, VP, VP, INT, VP, VP, INT, INT, INT, VP)(lambda *a: calls.append(table(a[1])) or 0)
    append = ctypes.CFUNCTYPE(INT, VP, INT, VP, VP, VP, INT, VP, VP, INT, VP, VP, VP)(lambda *a: calls.append((cache(a[0]), table(a[2]) if a[2] else None)) or 0)
    read = ctypes.CFUNCTYPE(INT, VP, INT, VP, VP, INT, VP, VP, VP)(lambda *a: calls.append(cache(a[0])) or 0)
    attention = ctypes.CFUNCTYPE(INT, VP, INT, VP, VP, INT, VP, VP, INT, ctypes.c_float, INT, INT, VP, ctypes.c_size_t, VP)(
        lambda *a: calls.append(cache(a[0])) or 0)
    workspace = ctypes.CFUNCTYPE(INT, VP, INT, INT, INT, INT, VP)(lambda *a: 0)
    kept = [rotary, append, read, attention, workspace]
    real = [ctypes.cast(getattr(_lib.lib(), n), VP).value for n in ("tllm_b200_gemv_packed", "tllm_b200_gemv_int8_packed", "tllm_b200_gemm_packed")]
    _hostcall.bind(*real, lambda: 0, lambda d: 0, torch.float16, torch.int8, torch.uint8)
    _hostcall.bind_cache4(*(ctypes.cast(f, VP).value for f in kept), torch.bfloat16, torch.float32, torch.int32)
    yield calls, host
    _lib._host = None
    _lib.host()


def make():
    c = ops.Cache4(*(on_device(2, 2, 16, *last, dtype=t) for last, t in (((32,), torch.uint8), ((1, 2), torch.float16)) * 2))
    t = ops.RotaryTable(64, device="cpu")
    object.__setattr__(t, "turns", t.turns.as_subclass(OnDevice))
    object.__setattr__(t, "_native", None)
    t._keep(_lib.RotaryTableDesc(t.turns.data_ptr(), 64, 1, 1.0), t.turns)
    x = on_device(3, 2, 64, dtype=torch.float16)
    first, lens = on_device(3, dtype=torch.int32), on_device(2, dtype=torch.int32)

    def run():
        ops.append(c, x, x, x, first, lens, t)
        ops.read(c, x, None, first, lens)
        ops.attention(c, x, on_device(3, 2, 64, dtype=torch.float16), first, lens)
        ops.rotary(x, None, on_device(3, dtype=torch.int32), t)

    return c, t, run


NAMES = ("k_codes", "k_params", "v_codes", "v_params")


def addresses(c):
    return [getattr(c, n).data_ptr() for n in NAMES]


def given(d):
    return [getattr(d, n) for n in NAMES]


def test_calls_name_the_memory_of_the_tensors(seen):
    calls, _ = seen
    c, t, run = make()
    run()
    assert given(calls[0][0]) == given(calls[1]) == given(calls[2]) == addresses(c) and calls[0][1].turns == calls[3].turns == t.turns.data_ptr()
    assert (calls[2].batch, calls[2].kv_heads, calls[2].rows, calls[2].dim, calls[3].rot_dim) == (2, 2, 16, 64, 64)


def emptied(x):
    x.untyped_storage().resize_(0)


CHANGES = {
    "other": lambda x: setattr(x, "data", torch.zeros_like(x).as_subclass(OnDevice)),
    "larger": lambda x: x.resize_(2, *x.shape),
    "set": lambda x: x.set_(torch.zeros(4, dtype=x.dtype)),
    "emptied": emptied,
    "cut": lambda x: x.untyped_storage().resize_(x.numel() * x.element_size() - 1),
    "type": lambda x: setattr(x, "data", torch.zeros(x.shape, dtype=torch.int8 if x.element_size() > 1 else torch.int16)),
    "strides": lambda x: setattr(x, "data", torch.zeros(*x.shape[:-1], 2 * x.shape[-1], dtype=x.dtype)[..., ::2]),
}


@pytest.mark.parametrize("change", list(CHANGES))
@pytest.mark.parametrize("name", [*NAMES, "turns"])
def test_a_tensor_at_other_memory_is_refused(seen, name, change):
    calls, host = seen
    c, t, _ = make()
    x = on_device(3, 2, 64, dtype=torch.float16)
    first, lens = on_device(3, dtype=torch.int32), on_device(2, dtype=torch.int32)
    CHANGES[change](t.turns if name == "turns" else getattr(c, name))
    if name == "turns":
        assert host.rotary(t._native, x, None, lens.new_zeros(3).as_subclass(OnDevice), None, None, False) is None
        assert host.cache4_append(c._native, t._native, x, x, x, first, lens, None) is None
    else:
        assert host.cache4_append(c._native, None, x, x, x, first, lens, None) is None
        assert host.cache4_read(c._native, x, None, first, lens) is None
        assert host.cache4_attention(c._native, x, x, first, lens, 1.0, 0, 0) is None
    assert not calls


def test_a_part_of_a_storage_that_was_emptied(seen):
    """A slice whose storage went keeps an offset, which is no address."""
    calls, host = seen
    whole = [torch.zeros(3, 2, 16, *last, dtype=t) for last, t in (((32,), torch.uint8), ((1, 2), torch.float16)) * 2]
    c = ops.Cache4(*(t[1:].as_subclass(OnDevice) for t in whole))
    x = on_device(3, 2, 64, dtype=torch.float16)
    first, lens = on_device(3, dtype=torch.int32), on_device(2, dtype=torch.int32)
    assert host.cache4_read(c._native, x, None, first, lens) == 0 and given(calls[0]) == addresses(c)
    whole[2].untyped_storage().resize_(0)
    assert host.cache4_read(c._native, x, None, first, lens) is None and len(calls) == 1


@pytest.mark.parametrize("change", list(CHANGES))
def test_the_other_way_says_what_is_wrong(monkeypatch, change):
    monkeypatch.setattr(torch.cuda, "current_device", lambda: None)          # the device index of a CPU tensor
    c, t, _ = make()
    c._desc(), t._desc()
    CHANGES[change](c.v_params)
    with pytest.raises((ValueError, TypeError), match="v_params"):
        c._desc()
    CHANGES[change](t.turns)
    with pytest.raises((ValueError, TypeError), match="turns"):
        t._desc()


def test_memory_that_went_and_came_back_smaller(seen):
    """The address may be the old one then."""
    calls, host = seen
    c, _, _ = make()
    x, first, lens = on_device(3, 2, 64, dtype=torch.float16), on_device(3, dtype=torch.int32), on_device(2, dtype=torch.int32)
    storage = c.k_codes.untyped_storage()
    n = storage.nbytes()
    storage.resize_(0)
    storage.resize_(n - 64)
    assert host.cache4_read(c._native, x, None, first, lens) is None and not calls


def test_a_handle_of_tensors_without_memory():
    t = [torch.zeros(2, 2, 16, *last, dtype=t) for last, t in (((32,), torch.uint8), ((1, 2), torch.float16)) * 2]
    t[3].untyped_storage().resize_(16)
    with pytest.raises(ValueError, match="storage"):
        ops.Cache4(*t)


class Library:
    """Functions of the C ABI that write down their whole numbers, converted as the ABI has them."""

    def __init__(self):
        self.calls = []
        signatures = _lib.SIGNATURES
        for name in ("tllm_b200_cache4_workspace", "tllm_b200_cache4_attention", "tllm_b200_rotary"):
            types = signatures[name][1]
            setattr(self, name, ctypes.CFUNCTYPE(INT, *types)(lambda *a, name=name: self.calls.append((name, a)) or 0))


@pytest.mark.parametrize("max_new,max_len,want", [
    (1, 2 ** 32 + 5, (1, 2 ** 31 - 1)), (2 ** 32 + 1, 7, (2 ** 31 - 1, 7)), (2 ** 31, 2 ** 40, (2 ** 31 - 1, 2 ** 31 - 1)), (3, 4, (3, 4)), (-2 ** 32, 0, (-1, 0)),
    (0, -2 ** 32 + 9, (0, -1)), (True, 4, (1, 4))])
def test_hints_beyond_32_bits(seen, monkeypatch, max_new, max_len, want):
    """A limit that no int holds is none, and a negative one stays what the library refuses."""
    c, _, _ = make()
    x, first, lens = on_device(3, 2, 64, dtype=torch.float16), on_device(3, dtype=torch.int32), on_device(2, dtype=torch.int32)
    library = Library()
    monkeypatch.setattr(torch.cuda, "current_device", lambda: None)
    monkeypatch.setattr(ops, "_stream", lambda: None)
    monkeypatch.setattr(ops._lib, "lib", lambda: library)
    ops.attention(c, x, x.clone().as_subclass(OnDevice), first, lens, scale=1, max_new=max_new, max_len=max_len)      # a scale that is no float goes the other way
    (_, w), (_, a) = library.calls
    assert w[3:5] == a[9:11] == want
    with pytest.raises(TypeError):
        ops.attention(c, x, x.clone().as_subclass(OnDevice), first, lens, max_len=7.5)


@pytest.mark.parametrize("rot", [-2 ** 32 + 64, 2 ** 31])
def test_head_parts_beyond_32_bits(rot):
    with pytest.raises(_lib.TllmError, match="rot_dim"):
        ops.rotary_frequencies(rot, 1e4)
    with pytest.raises(_lib.TllmError, match="rot_dim"):
        ops.RotaryTable(rot, 1e4, device="cpu")


def test_layout_and_direction_are_truth_values(seen, monkeypatch):
    _, t, _ = make()
    library = Library()
    x = on_device(3, 2, 64, dtype=torch.float16)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: None)
    monkeypatch.setattr(ops, "_stream", lambda: None)
    monkeypatch.setattr(ops._lib, "lib", lambda: library)
    for inverse in (2 ** 32, 1, 0):
        ops.rotary(x, None, on_device(3, dtype=torch.int32), t, inverse=inverse)
    assert [a[11] for _, a in library.calls] == [1, 1, 0]
    monkeypatch.undo()
    assert _lib.RotaryTableDesc.from_buffer_copy(ops.RotaryTable(64, half=2 ** 32, device="cpu")._native[0]).half_layout == 1
