"""What the operators around an e4m3 KV cache refuse, and the rotary frequencies' formulas: without a device."""

import ctypes
import math
import re

import pytest
import torch

from conftest import ROOT
from kvx import _lib, ops

BF16, FP8 = torch.bfloat16, torch.float8_e4m3fn


def cache(nb=2, bs=32, heads=2, hd=64, groups=2):
    codes = [torch.zeros((nb, bs, heads, hd), dtype=torch.uint8).view(FP8) for _ in range(2)]
    return (*codes, *(torch.ones((nb, groups, heads, 1)) for _ in range(2)))


def rows(n=3, heads=2, hd=64, dtype=BF16):
    return torch.zeros((n, heads, hd), dtype=dtype)


SLOTS = torch.zeros(3, dtype=torch.int32)
TABLES, LENS = torch.zeros((3, 1), dtype=torch.int32), torch.ones(3, dtype=torch.int32)


def test_structs_match_the_header():
    text = (ROOT / "include" / "kvx.h").read_text()
    for name, struct in (("kvx_fp8_cache", _lib.Fp8Cache), ("kvx_paged_batch", _lib.PagedBatch)):
        body = text[text.index(f"typedef struct {name} {{"):text.index(f"}} {name};")]
        fields = re.findall(r"(?:const )?(void\*|float\*|int32_t\*|int32_t|int64_t) (\w+);", body)
        sizes = {"int32_t": 4, "int64_t": 8}
        assert [(n, sizes.get(t, 8)) for t, n in fields] == [(n, ctypes.sizeof(t)) for n, t in struct._fields_]


def test_cpu_tensors_are_refused():
    c = cache()
    with pytest.raises(ValueError, match="ROCm device"):
        ops.store_kvcache_fp8(rows(), rows(), *c, SLOTS)
    with pytest.raises(ValueError, match="ROCm device"):
        ops.attention_fp8(rows(), *c, TABLES, LENS)
    with pytest.raises(ValueError, match="ROCm device"):
        ops.attention_weights_fp8(rows(), torch.zeros((3, 2)), c[0], c[2], TABLES, LENS)
    with pytest.raises(ValueError, match="ROCm device"):
        ops.rotary_embed(rows(), rows(), torch.zeros(3, dtype=torch.int64), ops.rotary_frequencies(64, device="cpu")[0])
    with pytest.raises(ValueError, match="ROCm device"):
        ops.select_tokens(torch.zeros((3, 2, 9)), LENS, 2)
    with pytest.raises(ValueError, match="ROCm device"):
        ops.compact_kvcache_fp8(*c, TABLES, torch.zeros((3, 2, 4), dtype=torch.int32), LENS, TABLES)


@pytest.mark.parametrize("change,error,match", [
    (dict(key=rows(dtype=torch.float64), value=rows(dtype=torch.float64)), NotImplementedError, "bfloat16"),
    (dict(value=rows(dtype=torch.float16)), TypeError, "dtype"),
    (dict(value=rows(2)), ValueError, "shapes"),
    (dict(key=rows(hd=48), value=rows(hd=48)), ValueError, "head_dim"),
    (dict(key=rows().transpose(1, 2), value=rows().transpose(1, 2)), ValueError, "packed"),
    (dict(slot_mapping=SLOTS.long()), TypeError, "int32"),
    (dict(slot_mapping=SLOTS[:2]), TypeError, "slot_mapping"),
    (dict(k_cache=cache()[0].view(torch.uint8)), ValueError, "float8_e4m3fn"),
    (dict(v_cache=cache(nb=3)[0]), ValueError, "equally sized"),
    (dict(k_scale=torch.ones((2, 2, 2, 1), dtype=BF16)), ValueError, "float32"),
    (dict(v_scale=torch.ones((2, 1, 2, 1))), ValueError, "scales"),
    (dict(k_scale=torch.ones((2, 3, 2, 1)), v_scale=torch.ones((2, 3, 2, 1))), ValueError, "divide"),
    (dict(k_scale=torch.ones((2, 2, 2))), ValueError, "scales")])
def test_stores_refused(change, error, match):
    args = dict(zip(("k_cache", "v_cache", "k_scale", "v_scale"), cache()), key=rows(), value=rows(), slot_mapping=SLOTS)
    with pytest.raises(error, match=match):
        ops.store_kvcache_fp8(**{**args, **change})


@pytest.mark.parametrize("change,error,match", [
    (dict(query=rows(dtype=torch.float32)), NotImplementedError, "bfloat16 or float16"),
    (dict(query=rows(heads=3)), ValueError, "multiple"),
    (dict(query=rows(hd=32)), ValueError, "head_dim"),
    (dict(block_tables=TABLES.long()), TypeError, "block_tables"),
    (dict(block_tables=torch.zeros((1, 3), dtype=torch.int32).expand(3, 3).t()), TypeError, "contiguous rows"),
    (dict(context_lens=LENS[:2]), TypeError, "context_lens"),
    (dict(cu_seqlens=LENS), TypeError, "cu_seqlens"),
    (dict(max_seqlen=2), ValueError, "max_seqlen"),
    (dict(out=rows(dtype=torch.float16)), ValueError, "out"),
    (dict(out=torch.zeros((3, 4, 64), dtype=BF16)[:, ::2]), ValueError, "out")])
def test_attention_refused(change, error, match):
    args = dict(zip(("k_cache", "v_cache", "k_scale", "v_scale"), cache()), query=rows(), block_tables=TABLES, context_lens=LENS)
    with pytest.raises(error, match=match):
        ops.attention_fp8(**{**args, **change})


@pytest.mark.parametrize("change,match", [
    (dict(lse=torch.zeros((3, 1))), "lse"), (dict(lse=torch.zeros((3, 2), dtype=BF16)), "lse"),
    (dict(weights=torch.zeros((3, 1, 9))), "weights"), (dict(weights=torch.zeros((3, 2, 9)), out=torch.zeros((3, 2, 8))), "weights"),
    (dict(out=torch.zeros((3, 2, 9), dtype=BF16)), "weights")])
def test_weights_refused(change, match):
    c = cache()
    args = dict(query=rows(), lse=torch.zeros((3, 2)), k_cache=c[0], k_scale=c[2], block_tables=TABLES, context_lens=LENS)
    with pytest.raises((TypeError, ValueError), match=match):
        ops.attention_weights_fp8(**{**args, **change})


@pytest.mark.parametrize("change,match", [
    (dict(positions=torch.zeros(3)), "positions"), (dict(positions=torch.zeros(2, dtype=torch.int64)), "positions"),
    (dict(frequencies=torch.zeros(16)), "float64"), (dict(key=rows(2)), "tokens"), (dict(key=rows(hd=32)), "head_dim"),
    (dict(key=rows(dtype=torch.float16)), "dtype"), (dict(query_out=rows(heads=3)), "shape"),
    (dict(query=torch.zeros((3, 64, 2), dtype=BF16).transpose(1, 2)), "packed")])
def test_rotary_refused(change, match):
    args = dict(query=rows(), key=rows(), positions=torch.zeros(3, dtype=torch.int64), frequencies=torch.zeros(16, dtype=torch.float64))
    with pytest.raises((TypeError, ValueError), match=match):
        ops.rotary_embed(**{**args, **change})


def test_selection_and_compaction_refused():
    with pytest.raises(ValueError, match="non-negative"):
        ops.select_tokens(torch.zeros((3, 2, 9)), LENS, -1)
    with pytest.raises(TypeError, match="weights"):
        ops.select_tokens(torch.zeros((3, 9)), LENS, 1)
    with pytest.raises(TypeError, match="context_lens"):
        ops.select_tokens(torch.zeros((2, 2, 9)), LENS, 1)
    indices = torch.zeros((3, 2, 4), dtype=torch.int32)
    with pytest.raises(TypeError, match="indices"):
        ops.compact_kvcache_fp8(*cache(), TABLES, indices[:2], LENS, TABLES)
    with pytest.raises(ValueError, match="row for each"):
        ops.compact_kvcache_fp8(*cache(), TABLES, indices, LENS, TABLES[:2])


# The C functions, with addresses that are never touched: every check comes before any device work.

def c_cache(**change):
    fields = dict(k_codes=4096, v_codes=4096, k_scales=4096, v_scales=4096, num_blocks=2, block_size=32, group_size=16,
                  num_heads=2, head_dim=64)
    return _lib.Fp8Cache(**{**fields, **change})


def c_batch(**change):
    fields = dict(block_tables=4096, context_lens=4096, cu_seqlens=None, table_stride=1, table_width=1, num_seqs=3,
                  max_seqlen=1, num_tokens=3)
    return _lib.PagedBatch(**{**fields, **change})


def attend(cache, batch, query=4096, stride=256, heads=4, dtype=_lib.DTYPE_BF16, out=4096, workspace=None, size=0, scale=1.0):
    _lib.check(_lib.lib().kvx_attention_fp8(ctypes.byref(cache), ctypes.byref(batch), query, stride, heads, dtype, scale, out,
                                            None, workspace, size, None))


@pytest.mark.parametrize("change,error,match", [
    (dict(group_size=8), NotImplementedError, "multiples of 16"), (dict(group_size=24), ValueError, "divide"),
    (dict(block_size=2048, group_size=2048), NotImplementedError, "multiples of 16"),
    (dict(head_dim=72), NotImplementedError, "head_dim"), (dict(head_dim=272), NotImplementedError, "head_dim"),
    (dict(num_heads=0), ValueError, "positive"), (dict(k_codes=None), ValueError, "NULL"), (dict(v_scales=None), ValueError, "NULL"),
    (dict(k_codes=4104), ValueError, "16 bytes"), (dict(num_blocks=2 ** 31 - 1, block_size=1024), NotImplementedError, "2\\^40")])
def test_c_caches_refused(change, error, match):
    with pytest.raises(error, match=match):
        attend(c_cache(**change), c_batch())


@pytest.mark.parametrize("change,error,match", [
    (dict(batch=dict(num_seqs=2)), ValueError, "one query row"), (dict(batch=dict(context_lens=None)), ValueError, "NULL"),
    (dict(batch=dict(num_seqs=-1)), ValueError, "non-negative"), (dict(batch=dict(table_width=2 ** 31 - 1)), NotImplementedError, "2\\^31"),
    (dict(batch=dict(num_seqs=70000, num_tokens=70000)), NotImplementedError, "65535"),
    (dict(heads=3), ValueError, "multiple"), (dict(dtype=_lib.DTYPE_FP32), NotImplementedError, "bf16 or fp16"), (dict(dtype=9), ValueError, "type"),
    (dict(query=4100), ValueError, "16 bytes"), (dict(stride=260), ValueError, "16 bytes"), (dict(out=None), ValueError, "out"),
    (dict(out=4098), ValueError, "16 bytes"), (dict(query=None), ValueError, "NULL"),
    (dict(scale=0.0), ValueError, "positive"), (dict(scale=-1.0), ValueError, "positive"), (dict(scale=math.inf), ValueError, "positive"),
    (dict(scale=math.nan), ValueError, "positive"), (dict(batch=dict(table_width=4000)), ValueError, "workspace")])
def test_c_attention_refused(change, error, match):
    change = dict(change)
    batch = c_batch(**change.pop("batch", {}))
    with pytest.raises(error, match=match):
        attend(c_cache(), batch, **change)


def test_other_c_calls_refused():
    handle, c, b = _lib.lib(), ctypes.byref(c_cache()), ctypes.byref(c_batch())
    with pytest.raises(ValueError, match="rotary_dim"):
        _lib.check(handle.kvx_rotary_embed(4096, 64, 4096, 64, 4096, 64, 4096, 64, 4096, 8, 4096, 1, 1, 1, 64, 66, 0, 1.0, 0, None))
    with pytest.raises(ValueError, match="positions"):
        _lib.check(handle.kvx_rotary_embed(4096, 64, 4096, 64, 4096, 64, 4096, 64, 4096, 2, 4096, 1, 1, 1, 64, 64, 0, 1.0, 0, None))
    with pytest.raises(NotImplementedError, match="too many tokens"):
        _lib.check(handle.kvx_store_kvcache_fp8(c, 4096, 128, 4096, 128, 0, 4096, 1 << 30, None))
    with pytest.raises(ValueError, match="rows must start"):
        _lib.check(handle.kvx_store_kvcache_fp8(c, 4096, 128, 4098, 128, 0, 4096, 3, None))
    with pytest.raises(ValueError, match="NULL"):
        _lib.check(handle.kvx_attention_weights_fp8(c, b, 4096, 256, 4, 0, 1.0, None, None, 4096, 32, None))
    with pytest.raises(ValueError, match="NULL"):
        _lib.check(handle.kvx_select_tokens(4096, 4096, 1, 1, 8, 4, 0, 4096, None, 4096, None))
    with pytest.raises(IndexError, match="do not hold"):
        _lib.check(handle.kvx_compact_kvcache_fp8(c, b, 4096, 4096, 33, 4096, 1, 1, None))


def test_calls_without_work_queue_nothing():
    handle, c = _lib.lib(), ctypes.byref(c_cache())
    none = ctypes.byref(c_batch(num_seqs=0, num_tokens=0, max_seqlen=0))
    assert handle.kvx_store_kvcache_fp8(c, None, 0, None, 0, 0, None, 0, None) == 0
    assert handle.kvx_attention_fp8(c, none, None, 0, 4, 0, 1.0, None, None, None, 0, None) == 0
    assert handle.kvx_attention_weights_fp8(c, none, None, 0, 4, 0, 1.0, None, None, None, 0, None) == 0
    assert handle.kvx_select_tokens(None, None, 0, 1, 0, 0, 0, None, None, None, None) == 0
    assert handle.kvx_compact_kvcache_fp8(c, none, None, None, 0, None, 0, 0, None) == 0
    assert handle.kvx_rotary_embed(None, 0, None, 0, None, 0, None, 0, None, 8, None, 0, 1, 1, 64, 64, 0, 1.0, 0, None) == 0


# Rotary frequencies

def test_frequencies_are_powers_of_the_base():
    f, magnitude = ops.rotary_frequencies(8, 10000.0, device="cpu")
    assert magnitude == 1.0 and f.dtype == torch.float64
    assert torch.allclose(f, torch.tensor([1.0, 0.1, 0.01, 0.001], dtype=torch.float64), rtol=1e-14, atol=0)


def test_scaled_frequencies():
    plain, _ = ops.rotary_frequencies(64, 10000.0, device="cpu")
    assert torch.allclose(ops.rotary_frequencies(64, 10000.0, "linear", 4.0, device="cpu")[0], plain / 4, rtol=1e-14, atol=0)
    grown, _ = ops.rotary_frequencies(64, 10000.0, "base", 4.0, device="cpu")
    assert grown[0] == 1.0 and math.isclose(grown[-1], plain[-1] / 4, rel_tol=1e-12)
    assert ((grown[1:] < plain[1:]) & (grown[1:] >= plain[1:] / 4 * (1 - 1e-12))).all()
    parts, magnitude = ops.rotary_frequencies(64, 10000.0, "by_parts", 4.0, 4096, device="cpu")
    assert math.isclose(magnitude, 0.1 * math.log(4.0) + 1.0)
    turns = plain * 4096 / (2 * math.pi)
    # The blend runs between the indices at which a pair turns 32 times and once, rounded outwards.
    stays, divided = (turns > 32 * (plain[0] / plain[1])), (turns < 1 / (plain[0] / plain[1]))
    assert stays.any() and divided.any()
    assert torch.equal(parts[stays], plain[stays]) and torch.allclose(parts[divided], plain[divided] / 4, rtol=1e-14, atol=0)
    assert (parts <= plain).all() and (parts >= plain / 4 * (1 - 1e-12)).all()
    assert torch.equal(ops.rotary_frequencies(64, 10000.0, "linear", 1.0, device="cpu")[0], plain)


@pytest.mark.parametrize("args,match", [
    ((7,), "even"), ((0,), "positive"), ((8, -1.0), "base"), ((8, 1e4, "linear", 0.5), "factor"), ((8, 1e4, "other"), "unknown"),
    ((8, 1e4, "by_parts", 4.0), "original_length"), ((8, 1e4, "by_parts", 4.0, 128, 1.0, 2.0), "fast")])
def test_frequencies_refused(args, match):
    with pytest.raises(ValueError, match=match):
        ops.rotary_frequencies(*args, device="cpu")


def test_numbers_past_32_bits_are_not_cut_to_them():
    with pytest.raises(NotImplementedError, match="at most"):
        ops.select_tokens(torch.zeros((3, 2, 9)), LENS, 2 ** 32 + 1)
    cu = torch.tensor([0, 1, 2, 5], dtype=torch.int32)
    assert ops._paged_batch(TABLES, LENS, cu, 2 ** 32 + 2, 5).max_seqlen == 5  # a hint: no sequence has more than all rows
    with pytest.raises(NotImplementedError, match="rows in one call"):
        ops._paged_batch(TABLES, LENS, cu, None, 2 ** 32 + 1)
