"""Calls around an e4m3 cache that are allowed and rare, against the definitions in 64 bits."""

import pytest
import torch

import fp8_cache_reference as ref
from kvx import ops
from test_gpu_fp8_cache import Setup, fp8, int32

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("per_kv", [1, 4, 130])  # 130 heads of a KV head: the kernel of many query rows
@pytest.mark.parametrize("native", [True, False])
def test_no_rows_for_sequences_that_have_tokens(gpu, monkeypatch, native, per_kv):
    """A decode step of no rows, without cu_seqlens: nothing attends, and no weight changes."""
    from kvx import _lib

    monkeypatch.setattr(_lib, "_bind", _lib.load_bind() if native else _lib._NoBind)
    s = Setup(gpu, [30, 300], None, 2, per_kv, 64, 32, 16)
    empty = s.q[:0].to(gpu)
    where, _ = s.batch()
    out, lse = ops.attention_fp8(empty, *s.caches(), *where, return_lse=True)
    assert out.shape == (0, 2 * per_kv, 64) and lse.shape == (0, 2 * per_kv)
    before = torch.rand((2, 2, s.tables.shape[1] * 32), device=gpu)
    args = (empty, lse, fp8(s.k, gpu), s.ks.to(gpu), *where)
    got = ops.attention_weights_fp8(*args, weights=before, out=torch.full_like(before, -1.0))
    assert torch.equal(got, before)
    mine = before.clone()
    assert torch.equal(ops.attention_weights_fp8(*args, weights=mine), before)
    assert (ops.attention_weights_fp8(*args) == 0).all()
