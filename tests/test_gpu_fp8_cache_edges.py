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


# ---------------------------------------------------------------------------
# Scales that are no powers of two: a user's own, which a group that goes on keeps.

def nearest(x):
    """float64 -> e4m3 codes by one rounding, ties to even: steps of 1/8 of the leading bit, 2^-9 below 2^-6."""
    x = x.clamp(-448.0, 448.0)
    step = torch.exp2(torch.floor(torch.log2(x.abs().clamp_min(2.0 ** -20))).clamp_min(-6.0) - 3)
    return (torch.round(x / step) * step).float().to(ref.FP8).view(torch.uint8)


def borders():
    """The 126 values halfway between neighbouring finite codes, as float64."""
    values = ref.decode(torch.arange(0x7F, dtype=torch.uint8))
    return (values[1:] + values[:-1]) / 2


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("hd,group", [(128, 16), (64, 64), (256, 128)])
def test_codes_are_nearest_under_a_kept_scale_of_any_value(gpu, hd, group, dtype):
    """The quotients of fp32 rows fall on the borders between codes and next to them, where x times 1 / s, and a quotient
    rounded to fp32 before it is rounded to a code, come out on the wrong side."""
    heads, blocks = 2, 6
    g = torch.Generator().manual_seed(group)
    codes, _ = ref.random_cache(blocks, group, group, heads, hd, 1)
    scales = ((torch.rand((blocks, 1, heads, 1), generator=g) + 0.5)
              * torch.randint(-30, 30, (blocks, 1, heads, 1), generator=g).float().exp2())
    n = 15  # tokens 1 .. 15 of each block's first group
    pick = borders()[torch.randint(0, 126, (blocks, n, heads, hd), generator=g)]
    x = (pick * scales.double()).float()
    up = torch.nextafter(x, torch.full_like(x, torch.inf))
    down = torch.nextafter(x, torch.zeros_like(x))
    x = torch.stack([x, up, down])[torch.randint(0, 3, (1, *x.shape), generator=g), torch.arange(blocks)[:, None, None, None],
                                   torch.arange(n)[:, None, None], torch.arange(heads)[:, None], torch.arange(hd)][0]
    x = x * (torch.randint(0, 2, x.shape, generator=g) * 2 - 1)
    limit = 448.0 * torch.exp2(torch.floor(torch.log2(scales)))  # up to here no larger power of two is asked for
    x = x.clamp(-limit, limit).to(dtype)
    slots = (torch.arange(blocks)[:, None] * group + torch.arange(1, n + 1)).flatten()
    want = codes.clone()
    want[:, 1:n + 1] = nearest(x.double() / scales.double())
    kc, vc, ks, vs = fp8(codes, gpu), fp8(codes, gpu), scales.to(gpu), scales.clone().to(gpu)
    rows = x.flatten(0, 1).to(gpu)
    ops.store_kvcache_fp8(rows, -rows, kc, vc, ks, vs, slots.int().to(gpu))
    assert torch.equal(ks.cpu(), scales) and torch.equal(vs.cpu(), scales)
    assert torch.equal(kc.view(torch.uint8).cpu(), want)
    want[:, 1:n + 1] = nearest(-x.double() / scales.double())
    assert torch.equal(vc.view(torch.uint8).cpu(), want)


@pytest.mark.parametrize("hd,group", [(128, 16), (64, 64)])
def test_codes_are_nearest_where_a_scale_of_any_value_grows(gpu, hd, group):
    """Old codes under a kept scale that makes some of them fall next to the border between two new ones."""
    heads, blocks = 2, 40
    g = torch.Generator().manual_seed(5)
    codes, _ = ref.random_cache(blocks, group, group, heads, hd, 1)
    aim = borders()[torch.randint(40, 110, (blocks, 1, heads, 1), generator=g)]
    held = ref.decode(torch.randint(60, 0x7F, aim.shape, generator=g, dtype=torch.uint8))
    scales = (aim / held).float()  # held * scale is nearly a border under a scale of 1
    while (scales >= 1).any():
        scales = torch.where(scales >= 1, scales / 2, scales)
    scales = torch.stack([scales, torch.nextafter(scales, scales * 2)])[torch.randint(0, 2, (1,), generator=g)][0]
    x = torch.full((blocks, heads, hd), 300.0, dtype=torch.bfloat16)  # asks for a scale of 1
    slots = torch.arange(blocks) * group + 3
    want = nearest(ref.decode(codes) * scales.double())
    want[:, 3] = nearest(x.double())
    kc, vc, ks, vs = fp8(codes, gpu), fp8(codes, gpu), scales.to(gpu), scales.clone().to(gpu)
    ops.store_kvcache_fp8(x.to(gpu), x.to(gpu), kc, vc, ks, vs, slots.int().to(gpu))
    assert (ks == 1).all() and (vs == 1).all()
    assert torch.equal(kc.view(torch.uint8).cpu(), want) and torch.equal(vc.view(torch.uint8).cpu(), want)


def compacted(gpu, codes, scales, block):
    """Blocks 0 .. n - 1 moved whole to n .. 2n - 1, in the order of the last row of each block first: codes and scales."""
    n, heads = codes.shape[0], codes.shape[2]
    twice = [torch.cat([t, torch.zeros_like(t)]) for t in (codes, scales)]
    kc, vc, ks, vs = fp8(twice[0], gpu), fp8(twice[0], gpu), twice[1].to(gpu), twice[1].clone().to(gpu)
    tables = torch.arange(n, dtype=torch.int32)[:, None]
    order = torch.arange(block - 1, -1, -1, dtype=torch.int32).repeat(n, heads, 1)
    ops.compact_kvcache_fp8(kc, vc, ks, vs, tables.to(gpu), order.to(gpu), int32([block] * n, gpu), (tables + n).to(gpu))
    assert torch.equal(kc.view(torch.uint8), vc.view(torch.uint8)) and torch.equal(ks, vs)
    return kc[n:].view(torch.uint8).cpu(), ks[n:].cpu()


@pytest.mark.parametrize("hd,group", [(128, 16), (64, 64), (256, 128)])
def test_compacted_codes_are_nearest_under_scales_of_any_value(gpu, hd, group):
    heads, blocks, block = 2, 20, 2 * group
    g = torch.Generator().manual_seed(5)
    codes, _ = ref.random_cache(blocks, block, group, heads, hd, 1)
    shape = (blocks, 2, heads, 1)
    aim = borders()[torch.randint(40, 110, shape, generator=g)]
    held = ref.decode(torch.randint(60, 0x7F, shape, generator=g, dtype=torch.uint8))
    scales = (aim / held).float()  # held * scale is nearly a border under each power of two
    # Codes whose value is the most that a scale holds, nearly: 448 s, and s a little more or less than a power of two.
    codes[::3, :group, 0, 3] = 0x7E
    scales[::3, 0, 0, 0] = torch.nextafter(torch.tensor(1.0), torch.tensor([2.0, 0.0])[torch.randint(0, 2, (7,), generator=g)])
    value = (ref.decode(codes) * scales.double().repeat_interleave(group, 1)).flip(1)
    want_scale = torch.tensor([[[[ref.least_scale(float(value[b, i * group:(i + 1) * group, h].abs().max()))]
                                 for h in range(heads)] for i in range(2)] for b in range(blocks)])
    got, got_scale = compacted(gpu, codes, scales, block)
    assert torch.equal(got_scale.double(), want_scale.double())
    assert torch.equal(got, nearest(value / want_scale.double().repeat_interleave(group, 1)))


def test_the_largest_values_are_compacted(gpu):
    """Codes of 256 and more under a scale of 2^120, as the largest bf16 values are stored, stand for more than fp32 holds."""
    block, heads, hd = 16, 2, 64
    codes, _ = ref.random_cache(4, block, 16, heads, hd, 1)
    codes[0, 3, 0, 5], codes[1, 9, 1, 7], codes[2] = 0x78, 0xFE, codes[2] & 0x77
    scales = torch.tensor([2.0 ** 120, 2.0 ** 120, 2.0 ** 120, 2.0 ** -100]).view(4, 1, 1, 1).repeat(1, 1, heads, 1)
    tables, indices = torch.arange(4)[:, None].int(), torch.arange(block).repeat(4, heads, 1).int()
    twice = [torch.cat([t, torch.zeros_like(t)]) for t in (codes, scales)]
    want, want_scale = ref.compact(*twice, tables, indices.flip(2), torch.tensor([block] * 4), tables + 4)
    got, got_scale = compacted(gpu, codes, scales, block)
    assert torch.equal(got_scale, want_scale[4:]) and torch.equal(got, want[4:])


# ---------------------------------------------------------------------------
# The second product's weights, in 16 bits

BITS_16 = 2.0 ** -16  # two roundings to bf16, the second of the first one's remainder: half a step, 2^-8, of 2^-8


@pytest.mark.parametrize("hd,per_kv,q_lens,dtype", [
    (128, 4, None, torch.bfloat16), (64, 8, [1, 4, 4, 3], torch.bfloat16), (256, 2, [2, 20, 7, 1], torch.bfloat16),
    (128, 4, [1, 40, 33, 8], torch.bfloat16), (64, 2, [1, 70, 33, 8], torch.bfloat16), (112, 3, [1, 40, 33, 8], torch.bfloat16),
    (128, 4, None, torch.float16), (128, 4, [1, 40, 33, 8], torch.float16), (64, 2, [1, 70, 33, 8], torch.float16)])
@pytest.mark.parametrize("powers", [True, False])
def test_the_weights_of_the_values_keep_16_bits(gpu, hd, per_kv, q_lens, dtype, powers):
    """Few rows and chunks, in both types, under any scales: outputs near 0, where the values cancel out, show it."""
    Setup(gpu, [33, 90, 300, 2100], q_lens, 2, per_kv, hd, 64, 32, dtype, powers=powers).check(p_step=BITS_16)


def test_rows_do_not_change_their_precision_with_the_hint(gpu):
    s = Setup(gpu, [200, 300], [150, 33], 1, 4, 64, 32, 32)
    for most in (1, 8, 16, 150, 183):  # the first two by the kernel of few rows, whose sequences may be longer
        s.check(p_step=BITS_16, max_seqlen=most)


@pytest.mark.parametrize("native", [True, False])
@pytest.mark.parametrize("recent", [5, 9, 2 ** 31, 2 ** 32 + 1])
def test_more_recent_tokens_than_are_kept(gpu, monkeypatch, native, recent):
    from kvx import _lib

    monkeypatch.setattr(_lib, "_bind", _lib.load_bind() if native else _lib._NoBind)
    weights = torch.rand((2, 2, 40), generator=torch.Generator().manual_seed(1))
    got = ops.select_tokens(weights.to(gpu), int32([40, 7], gpu), 5, recent)
    for a, b in zip(got, ref.select(weights, [40, 7], 5, recent)):
        assert torch.equal(a.cpu(), b)


def test_many_sequences_of_one_row_without_a_hint(gpu):
    """max_seqlen defaults to all rows, 4,100 of them for each of as many sequences."""
    n, heads, hd = 4100, 8, 144
    k, ks = ref.random_cache(300, 16, 16, heads, hd, 1)
    v, vs = ref.random_cache(300, 16, 16, heads, hd, 2)
    g = torch.Generator().manual_seed(3)
    tables = torch.randint(0, 300, (n, 1), generator=g, dtype=torch.int32).to(gpu)
    lens = torch.randint(0, 17, (n,), generator=g, dtype=torch.int32).to(gpu)
    q = torch.randn((n, heads, hd), generator=g).to(torch.bfloat16).to(gpu)
    args = (q, fp8(k, gpu), fp8(v, gpu), ks.to(gpu), vs.to(gpu), tables, lens)
    want = ops.attention_fp8(*args, return_lse=True)
    got = ops.attention_fp8(*args, return_lse=True, cu_seqlens=torch.arange(n + 1, dtype=torch.int32, device=gpu))
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_many_rows_and_heads_without_a_hint(gpu):
    n, rows, heads, hd = 1000, 70, 256, 16
    k, ks = ref.random_cache(50, 80, 16, 1, hd, 1)
    v, vs = ref.random_cache(50, 80, 16, 1, hd, 2)
    g = torch.Generator().manual_seed(3)
    tables = torch.randint(0, 50, (n, 1), generator=g, dtype=torch.int32).to(gpu)
    lens = torch.randint(60, 81, (n,), generator=g, dtype=torch.int32).to(gpu)
    q = torch.randn((n * rows, heads, hd), device=gpu).to(torch.bfloat16)
    args = (q, fp8(k, gpu), fp8(v, gpu), ks.to(gpu), vs.to(gpu), tables, lens)
    cu = torch.arange(n + 1, dtype=torch.int32, device=gpu) * rows
    want = ops.attention_fp8(*args, return_lse=True, cu_seqlens=cu, max_seqlen=rows)
    got = ops.attention_fp8(*args, return_lse=True, cu_seqlens=cu)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("rows", [1, 5, 40])
def test_a_captured_step_of_all_operators_replays(gpu, rows):
    """Rotary positions, write, attention, weights, choice and compaction in one graph, replayed as a context grows, with
    eager work between the replays; each against the same calls made one by one on tensors of their own."""
    heads, per_kv, hd, block, group, keep, width = 2, 4, 64, 64, 16, 20, 256
    g = torch.Generator().manual_seed(rows)

    def state():
        codes = torch.zeros((2, 12, block, heads, hd), dtype=torch.uint8, device=gpu).view(torch.float8_e4m3fn)
        return (codes, torch.ones((2, 12, block // group, heads, 1), device=gpu), torch.zeros((2, heads, width), device=gpu))

    tables, new = int32([[3, 1, 4, 0], [5, 9, 2, 6]], gpu), int32([[7], [8]], gpu)
    frequencies, magnitude = ops.rotary_frequencies(hd)
    qkv = torch.zeros((2 * rows, heads * (per_kv + 2), hd), dtype=torch.bfloat16, device=gpu)
    positions = torch.zeros(2 * rows, dtype=torch.int64, device=gpu)
    slots, lens, cu = (torch.zeros(n, dtype=torch.int32, device=gpu) for n in (2 * rows, 2, 3))

    def step(codes, scales, weights):
        q, k = ops.rotary_embed(qkv[:, :heads * per_kv], qkv[:, heads * per_kv:-heads], positions, frequencies, magnitude=magnitude)
        cache = (codes[0], codes[1], scales[0], scales[1])
        ops.store_kvcache_fp8(k, qkv[:, -heads:], *cache, slots)
        how = {} if rows == 1 else dict(cu_seqlens=cu, max_seqlen=rows)
        out, lse = ops.attention_fp8(q, *cache, tables, lens, return_lse=True, **how)
        ops.attention_weights_fp8(q, lse, codes[0], scales[0], tables, lens, weights=weights, **how)
        chosen = ops.select_tokens(weights, lens, keep, 4)
        ops.compact_kvcache_fp8(*cache, tables, chosen[0], chosen[1], new)
        return (out, lse, *chosen)

    def bits(outputs, kept):
        return [t.view(torch.uint8) if t.dtype == torch.float8_e4m3fn else t for t in (*outputs, *kept)]

    mine, eager = state(), state()
    slots.fill_(-1)
    step(*state())  # the library is loaded
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outputs = step(*mine)
    length = 0
    for _ in range(5):
        n = rows if length else max(1, rows - 3)  # the first step's last rows are none: slots of -1, and they see what is there
        length += n
        qkv.copy_(torch.randn(qkv.shape, generator=g))
        at = torch.full((2, rows), -1, dtype=torch.int64)
        at[:, :n] = torch.arange(length - n, length)
        positions.copy_(at.clamp_min(0).flatten())
        cpu = tables.cpu().long()
        slot = torch.where(at >= 0, cpu.gather(1, at.clamp_min(0) // block) * block + at % block, -1)
        slots.copy_(slot.flatten())
        lens.fill_(length)
        cu.copy_(torch.tensor([0, rows, 2 * rows]))
        graph.replay()
        torch.cuda.synchronize()
        want = step(*eager)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(bits(outputs, mine), bits(want, eager)))
        assert not want[0].isnan().any()
