"""Which way a call of attention over the 4-bit cache takes, by the workspace that it asks for."""
import ctypes

import pytest

import ternary_llm_b200 as tl
from ternary_llm_b200 import _lib

P = 0x10000          # an address that is never followed


def workspace(batch, kv_heads, rows, dim, tokens, heads, max_new=0, max_len=0):
    n = ctypes.c_size_t()
    c = _lib.Cache4Desc(P, P, P, P, batch, kv_heads, rows, dim)
    assert tl.lib().tllm_b200_cache4_workspace(ctypes.byref(c), tokens, heads, max_new, max_len, ctypes.byref(n)) == 0
    return n.value


def record(ctas, rows, dim):
    """An entry of 32 bytes and two records of `rows` maxima, sums and outputs for each CTA."""
    return ctas * (32 + 2 * rows * (dim + 2) * 4)


@pytest.mark.parametrize("batch,kv_heads,rows,dim,heads", [(9, 8, 8192, 128, 32), (32, 8, 8192, 128, 32), (200, 8, 4096, 64, 32), (4096, 8, 64, 128, 32), (1, 8, 40000, 128, 32)])
def test_single_tokens_without_a_hint(batch, kv_heads, rows, dim, heads):
    """As with it: 4 rows of a head, in parts that are joined or in one CTA."""
    want = 0 if rows * dim <= 160000 else record(296, 4, dim)
    assert workspace(batch, kv_heads, rows, dim, batch, heads, 1) == want
    assert workspace(batch, kv_heads, rows, dim, batch, heads) == want


def test_prompts_beside_many_short_sequences_are_cut():
    """Whole tiles would take a CTA for each tile that any of the sequences might have."""
    assert workspace(64, 8, 4008, 128, 4063, 32, 4000) == workspace(64, 8, 4008, 128, 4063, 32) == record(148, 256, 128)
    assert workspace(1000, 8, 2008, 128, 2999, 32, 2000) == record(148, 256, 128)
    assert workspace(4, 8, 2008, 128, 2003, 32, 2000) == 0                   # few CTAs find nothing
    assert workspace(1, 8, 2008, 128, 2000, 32) == 0


def test_more_units_than_31_bits_hold():
    """Few rows by the hint, but far more of them: prompts of unknown length, as without the hint."""
    assert workspace(1, 8, 131072, 64, 60000, 32, 1) == record(296, 4, 64)
    assert workspace(1, 8, 131072, 64, 70000, 32, 1) == workspace(1, 8, 131072, 64, 70000, 32) != record(296, 4, 64)
    # and where parts of prompts are too many, whole tiles
    assert workspace(1, 1, 1 << 30, 64, 1000000, 1, 1000000) == 0 < workspace(1, 1, 1 << 30, 64, 1000, 1, 1000)


@pytest.mark.parametrize("type,dim,fits", [(2, 4, True), (2, 8, True), (2, 2, False), (0, 4, False), (1, 4, False), (0, 8, True), (2, 512, True), (2, 516, False)])
def test_head_sizes_of_rotary(type, dim, fits):
    """A multiple of 8, of 4 for FP32, up to 512; what is refused is refused before the device is looked for."""
    x, t = ctypes.byref(_lib.HeadsDesc(P, 2 * dim)), ctypes.byref(_lib.RotaryTableDesc(P, 2, 1, 1.0))
    status = tl.lib().tllm_b200_rotary(type, t, P, 0, x, x, 2, None, None, 0, dim, 0, None)
    assert (status != -3) == fits, tl.lib().tllm_b200_last_error()


def test_many_tiles_of_few_rows_stay_in_one_cta():
    """33 rows of a head and more are prompts where a tile of 16 would be cut."""
    assert workspace(1, 8, 1250, 128, 40, 32, 40) == 0 == workspace(1, 8, 2500, 64, 64, 32, 64)
    assert workspace(1, 8, 2541, 128, 40, 32, 40) == record(148, 128, 128) and workspace(1, 8, 6000, 64, 64, 32, 64) == record(148, 128, 64)
    assert workspace(1, 8, 2541, 128, 8, 32, 8) == record(148, 16, 128)
