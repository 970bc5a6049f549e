"""The operators around an e4m3 KV cache against their definitions in 64 bits (tests/fp8_cache_reference.py).

Tolerances. Products with e4m3 values are exact in the matrix cores' fp32, so a score is off by its sums alone, at most
(hd + 8) half steps of fp32 (2^-24) relative to sum |q k|, and a softmax weight by that plus a few half steps for the
exponential and the sums over the keys. P is rounded to bf16 for the second product: half a step (2^-8) of its value
at most with one operand, 2^-16 with two. The output is rounded once more to its type."""

import math

import pytest
import torch

import fp8_cache_reference as ref
from kvx import ops

pytestmark = pytest.mark.gpu
HALF_STEP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
NAN = 0x7F


def fp8(codes, gpu):
    return codes.to(gpu).view(torch.float8_e4m3fn)


def int32(values, gpu):
    return torch.tensor(values, dtype=torch.int32, device=gpu)


def tables_for(lens, block, seed, spare=3):
    """([B, width] int32 tables over shuffled blocks, blocks of the pool); -1 past each sequence's blocks."""
    need = [-(-max(0, n) // block) for n in lens]
    width = max(1, max(need, default=1))
    order = torch.randperm(sum(need) + spare, generator=torch.Generator().manual_seed(seed)).tolist()
    tables, at = torch.full((len(lens), width), -1, dtype=torch.int32), 0
    for b, n in enumerate(need):
        tables[b, :n] = torch.tensor(order[at:at + n], dtype=torch.int32)
        at += n
    return tables, sum(need) + spare


def query(n, heads, hd, dtype, seed):
    return torch.randn((n, heads, hd), generator=torch.Generator().manual_seed(seed)).to(dtype)


def check_attention(out, lse, want, want_lse, bound, dtype, hd, p_step):
    out, lse = out.cpu().double(), lse.cpu().double()
    for (row, head), (reach, score, keys) in bound.items():
        off = 2 * ((hd + 8) * 2.0 ** -24 * score + (keys + 16) * 2.0 ** -23)
        tol = HALF_STEP[dtype] * want[row, head].abs() * 1.01 + reach * (p_step + off) * 1.01 + 2.0 ** -24
        assert ((out[row, head] - want[row, head]).abs() <= tol).all(), (row, head)
        assert abs(lse[row, head] - want_lse[row, head]) <= off + abs(want_lse[row, head]) * 2.0 ** -22, (row, head)
    blind = (want_lse == -math.inf)
    assert (out[blind] == 0).all() and (lse[blind] == -math.inf).all()


class Setup:
    """A pool, tables and queries; ranges: rows of each sequence."""

    def __init__(self, gpu, lens, q_lens=None, heads=2, per_kv=4, hd=128, block=64, group=32, dtype=torch.bfloat16,
                 seed=0, powers=True, unused=None):
        self.gpu, self.lens, self.dtype, self.hd, self.block = gpu, lens, dtype, hd, block
        self.tables, blocks = tables_for(lens, block, seed)
        self.k, self.ks = ref.random_cache(blocks, block, group, heads, hd, seed + 1, powers)
        self.v, self.vs = ref.random_cache(blocks, block, group, heads, hd, seed + 2, powers)
        if unused is not None:  # every slot that holds no token
            used = torch.zeros(blocks * block, dtype=torch.bool)
            for b, n in enumerate(lens):
                used[ref.slots_of(self.tables[b], n, block)] = True
            self.k.flatten(0, 1)[~used] = unused
            self.v.flatten(0, 1)[~used] = unused
        counts = [1] * len(lens) if q_lens is None else q_lens
        ends = [sum(counts[:i + 1]) for i in range(len(counts))]
        self.ranges = [(e - c, e) for e, c in zip(ends, counts)]
        self.cu = None if q_lens is None else [0, *ends]
        self.q = query(ends[-1], heads * per_kv, hd, dtype, seed + 3)
        self.scale = hd ** -0.5

    def caches(self):
        return (fp8(self.k, self.gpu), fp8(self.v, self.gpu), self.ks.to(self.gpu), self.vs.to(self.gpu))

    def batch(self):
        cu = None if self.cu is None else int32(self.cu, self.gpu)
        most = None if self.cu is None else max(b - a for a, b in self.ranges)
        return (self.tables.to(self.gpu), int32(self.lens, self.gpu)), dict(cu_seqlens=cu, max_seqlen=most)

    def run(self, **more):
        where, how = self.batch()
        return ops.attention_fp8(self.q.to(self.gpu), *self.caches(), *where, self.scale, return_lse=True,
                                 **{**how, **more})

    def want(self):
        return ref.attention(self.q, self.k, self.v, self.ks, self.vs, self.tables, self.lens, self.ranges, self.scale)

    def check(self, p_step=2.0 ** -8, **more):
        check_attention(*self.run(**more), *self.want(), self.dtype, self.hd, p_step)


LENGTHS = [0, 1, 15, 16, 17, 31, 32, 33, 129, 300]


@pytest.mark.parametrize("heads,per_kv,hd,block,group,dtype", [
    (2, 4, 128, 64, 32, torch.bfloat16), (1, 1, 64, 16, 16, torch.bfloat16), (3, 7, 80, 48, 16, torch.bfloat16),
    (2, 16, 128, 256, 64, torch.float16), (1, 4, 256, 32, 32, torch.bfloat16), (2, 2, 16, 16, 16, torch.float16),
    (1, 8, 192, 128, 128, torch.bfloat16), (1, 20, 112, 256, 256, torch.bfloat16), (2, 33, 48, 16, 16, torch.float16),
    (4, 5, 96, 64, 16, torch.bfloat16), (1, 1, 240, 16, 16, torch.bfloat16)])
def test_single_tokens(gpu, heads, per_kv, hd, block, group, dtype):
    Setup(gpu, LENGTHS, None, heads, per_kv, hd, block, group, dtype, powers=hd != 80).check()


@pytest.mark.parametrize("per_kv", [1, 4])
@pytest.mark.parametrize("length", [2047, 4097])
def test_single_tokens_of_one_long_context(gpu, length, per_kv):
    Setup(gpu, [length], None, 2, per_kv, 128, 256, 64).check()


@pytest.mark.parametrize("heads,per_kv,hd,block,group,dtype", [
    (2, 4, 128, 64, 32, torch.bfloat16), (1, 1, 64, 16, 16, torch.bfloat16), (2, 3, 96, 32, 16, torch.float16),
    (1, 2, 256, 256, 64, torch.bfloat16), (1, 5, 192, 64, 64, torch.float16), (1, 8, 128, 128, 128, torch.bfloat16)])
def test_chunks(gpu, heads, per_kv, hd, block, group, dtype):
    # Whole prompts, a chunk behind a prefix, no rows, one row, more rows than tokens (the first see nothing).
    lens, rows = [67, 190, 40, 55, 3, 0], [67, 70, 0, 1, 9, 2]
    Setup(gpu, lens, rows, heads, per_kv, hd, block, group, dtype).check()


@pytest.mark.parametrize("rows", [2, 3, 4, 8, 17])
def test_a_few_proposed_tokens(gpu, rows):
    lens = [rows, 100, 257, 700]
    Setup(gpu, lens, [rows] * 4, 2, 4, 128, 64, 32).check()


@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("rows", [4, 8, 9, 40])
def test_few_and_many_rows_behind_long_contexts(gpu, rows, hd):
    # 16, 32, 36 and 160 rows a KV head, over several splits of the keys; some splits lie past a context.
    Setup(gpu, [3000, 2047, 10, 0], [rows, rows, min(rows, 10), 0], 1, 4, hd, 64, 32, unused=NAN).check()


def test_chunks_under_scales_that_are_no_powers_of_two(gpu):
    # V is rounded to bf16 once more there: half a step besides P's.
    for hd in (64, 128):
        Setup(gpu, [300, 50], [60, 50], 1, 2, hd, 64, 32, powers=False).check(p_step=2.0 ** -7)


@pytest.mark.parametrize("most", [1, 16, 300])
def test_max_seqlen_is_only_a_hint(gpu, most):
    s = Setup(gpu, [200, 300], [150, 33], 1, 4, 64, 32, 32)
    s.check(max_seqlen=most)
    s.check(max_seqlen=None)


def test_long_chunks_of_one_sequence(gpu):
    Setup(gpu, [700], [600], 1, 2, 128, 64, 32).check()


@pytest.mark.parametrize("code", [NAN, 0xFF, 0x7E])
@pytest.mark.parametrize("q_lens", [None, [1, 5, 30, 2], [1, 15, 16, 17]])
def test_slots_without_tokens_do_not_matter(gpu, code, q_lens):
    Setup(gpu, [1, 15, 47, 290], q_lens, 2, 4, 128, 64, 32, unused=code).check()


@pytest.mark.parametrize("hd,rows", [(64, 40), (128, 40), (256, 40), (128, 3)])
def test_codes_that_are_no_numbers_reach_only_rows_that_see_them(gpu, hd, rows):
    s = Setup(gpu, [77], [rows], 1, 2, hd, 16, 16, unused=NAN)
    token = 77 - rows + 1  # seen by all rows but the first
    slot = ref.slots_of(s.tables[0], 77, 16)[token]
    s.v.flatten(0, 1)[slot, 0, 5] = NAN
    out, lse = s.run()
    want, want_lse, bound = s.want()
    out = out.cpu().double()
    assert out[1:, :, 5].isnan().all() and not out[0].isnan().any()
    out[1:, :, 5] = want[1:, :, 5] = 0.0
    bound = {k: (reach.nan_to_num(0.0), score, keys) for k, (reach, score, keys) in bound.items()}
    check_attention(out, lse, want, want_lse, bound, s.dtype, hd, 2.0 ** -8)
    s.k.flatten(0, 1)[slot, 0, 7] = 0xFF
    out = s.run()[0].cpu()
    assert out[1:].isnan().all() and not out[0].isnan().any()


def test_every_code_comes_back_exactly(gpu):
    s = Setup(gpu, [1], None, 1, 1, 256, 16, 16)
    slot = int(s.tables[0, 0]) * 16
    s.v.flatten(0, 1)[slot, 0] = torch.arange(256, dtype=torch.uint8)
    out = s.run()[0].cpu().double().flatten()
    want = ref.values(s.v, s.vs)[slot, 0]
    assert torch.equal(out.isnan(), want.isnan()) and torch.equal(out.nan_to_num(9.0), want.nan_to_num(9.0))


@pytest.mark.parametrize("q_lens", [None, [3, 40]])
def test_blocks_outside_the_pool_hold_nothing_and_lengths_end_with_the_table(gpu, q_lens):
    s = Setup(gpu, [130, 200], q_lens, 1, 4, 64, 32, 16)
    s.tables[0, 1], s.tables[1, 0], s.tables[1, 3] = -1, 10 ** 6, -7
    s.lens = [130, 5000]
    s.check()


@pytest.mark.parametrize("q_lens", [None, [30, 25]])
def test_strided_queries_and_tables(gpu, q_lens):
    s = Setup(gpu, [40, 90], q_lens, 2, 2, 64, 16, 16)
    n = s.q.shape[0]
    fused = torch.randn((n, 8, 64), device=gpu).to(torch.bfloat16)
    fused[:, 1:5] = s.q.to(gpu)
    wide = torch.full((2, s.tables.shape[1] + 5), 10 ** 6, dtype=torch.int32, device=gpu)
    wide[:, 2:2 + s.tables.shape[1]] = s.tables.to(gpu)
    where, how = s.batch()
    got = ops.attention_fp8(fused[:, 1:5], *s.caches(), wide[:, 2:2 + s.tables.shape[1]], where[1], s.scale,
                            return_lse=True, **how)
    check_attention(*got, *s.want(), s.dtype, s.hd, 2.0 ** -8)


def test_rows_behind_the_last_sequence_are_left_as_they_were(gpu):
    s = Setup(gpu, [30, 40], [7, 20], 1, 2, 64, 16, 16)
    q = torch.cat([s.q, torch.randn((6, 2, 64)).to(s.dtype)]).to(gpu)
    out = torch.full(q.shape, 3.0, dtype=s.dtype, device=gpu)
    where, how = s.batch()
    got, lse = ops.attention_fp8(q, *s.caches(), *where, s.scale, out=out, return_lse=True, **how)
    assert got is out and (out[27:] == 3.0).all()
    check_attention(out[:27], lse[:27], *s.want(), s.dtype, s.hd, 2.0 ** -8)


def test_no_sequences_and_no_rows(gpu):
    s = Setup(gpu, [30], None, 1, 2, 64, 16, 16)
    empty = torch.empty((0, 2, 64), dtype=s.dtype, device=gpu)
    tables, lens = s.tables.to(gpu), int32([30], gpu)
    out, lse = ops.attention_fp8(empty, *s.caches(), tables[:0], lens[:0], return_lse=True)
    assert out.shape == (0, 2, 64) and lse.shape == (0, 2)
    ops.attention_fp8(empty, *s.caches(), tables, lens, cu_seqlens=int32([0, 0], gpu))
    weights = torch.rand((1, 1, 40), device=gpu)
    same = ops.attention_weights_fp8(empty, lse, *s.caches()[0::2], tables, lens, cu_seqlens=int32([0, 0], gpu),
                                     weights=weights, out=torch.empty_like(weights))
    assert torch.equal(same, weights)


@pytest.mark.parametrize("q_lens", [[0, 3, 0], [40, 0, 0], [0, 0, 70]])
def test_sequences_without_rows(gpu, q_lens):
    s = Setup(gpu, [50, 90, 300], q_lens, 2, 2, 64, 16, 16)
    s.check()
    where, how = s.batch()
    _, lse = s.run()
    before = torch.rand((3, 2, s.tables.shape[1] * 16), device=gpu)
    got = ops.attention_weights_fp8(s.q.to(gpu), lse, fp8(s.k, gpu), s.ks.to(gpu), *where, s.scale, weights=before,
                                    out=torch.empty_like(before), **how)
    for b, n in enumerate(q_lens):
        assert n or torch.equal(got[b], before[b])


@pytest.mark.parametrize("rows", [1, 50])
def test_a_cache_without_blocks(gpu, rows):
    q = query(rows, 4, 64, torch.bfloat16, 1).to(gpu)
    codes = torch.empty((0, 256, 2, 64), dtype=torch.uint8, device=gpu).view(torch.float8_e4m3fn)
    scales = torch.empty((0, 4, 2, 1), device=gpu)
    tables, lens = torch.zeros((1, 40), dtype=torch.int32, device=gpu), int32([9000], gpu)
    how = dict(cu_seqlens=int32([0, rows], gpu), max_seqlen=rows)
    out, lse = ops.attention_fp8(q, codes, codes, scales, scales, tables, lens, return_lse=True, **how)
    assert (out == 0).all() and (lse == -math.inf).all()
    weights = torch.rand((1, 2, 500), device=gpu)
    got = ops.attention_weights_fp8(q, lse, codes, scales, tables, lens, weights=weights, out=torch.empty_like(weights), **how)
    assert torch.equal(got, weights)
    ops.store_kvcache_fp8(q[:, :2], q[:, 2:], codes, codes, scales, scales, int32([0] * rows, gpu))


def test_large_scores_and_scales(gpu):
    s = Setup(gpu, [100, 50], None, 1, 4, 64, 32, 32)
    s.q *= 300.0  # scores of hundreds: one token takes nearly all
    s.vs *= 2.0 ** 90
    s.check()
    s.vs *= 2.0 ** -180
    out, lse = s.run()
    want, want_lse, bound = s.want()
    check_attention(out.cpu().double() * 2.0 ** 90, lse, want * 2.0 ** 90, want_lse,
                    {k: (r * 2.0 ** 90, a, n) for k, (r, a, n) in bound.items()}, s.dtype, 64, 2.0 ** -8)


def test_offsets_past_32_bits(gpu):
    # 9,000 blocks of 256 x 8 x 128 codes: 2.4 GB each of K and V; the sequence lies at the far end.
    blocks, block, heads, hd = 9000, 256, 8, 128
    s = Setup(gpu, [300, 513], None, heads, 4, hd, block, 64)
    far = torch.randperm(5, generator=torch.Generator().manual_seed(1)) + blocks - 5
    tables = torch.full((2, 3), -1, dtype=torch.int32)
    tables[0, :2], tables[1] = far[:2].int(), far[2:].int()
    caches = []
    for codes, dtype in ((s.k, torch.uint8), (s.v, torch.uint8), (s.ks, torch.float32), (s.vs, torch.float32)):
        big = torch.empty((blocks, *codes.shape[1:]), dtype=dtype, device=gpu)
        for b in range(2):
            for i in range(-(-s.lens[b] // block)):
                big[tables[b, i]] = codes[s.tables[b, i]].to(gpu)
        caches.append(big.view(torch.float8_e4m3fn) if dtype == torch.uint8 else big)
    got = ops.attention_fp8(s.q.to(gpu), *caches, tables.to(gpu), int32(s.lens, gpu), s.scale, return_lse=True)
    check_attention(*got, *s.want(), s.dtype, hd, 2.0 ** -8)
    # The cache write and compaction at the same place.
    x = torch.randn((70, heads, hd), generator=torch.Generator().manual_seed(5)).to(torch.bfloat16)
    base = int(far[0])
    slots = torch.arange(70) + base * block + 10
    before = [(c[base:base + 1].view(torch.uint8) if c.dtype == torch.float8_e4m3fn else c[base:base + 1]).cpu() for c in caches]
    ops.store_kvcache_fp8(x.to(gpu), x.to(gpu), *caches, slots.to(torch.int32).to(gpu))
    for codes, scale, c, sc in ((before[0], before[2], caches[0], caches[2]), (before[1], before[3], caches[1], caches[3])):
        want, want_scale = ref.store(x, codes, scale, (slots - base * block).tolist())
        assert torch.equal(c[base:base + 1].view(torch.uint8).cpu(), want)
        assert torch.equal(sc[base:base + 1].cpu(), want_scale)
    indices = torch.arange(100, dtype=torch.int32, device=gpu).repeat(1, heads, 1)
    ops.compact_kvcache_fp8(*caches, int32([[base]], gpu), indices, int32([100], gpu), int32([[1]], gpu))
    moved = caches[0][1, :100].float() * caches[2][1].repeat_interleave(64, 0)[:100]
    origin = caches[0][base, :100].float() * caches[2][base].repeat_interleave(64, 0)[:100]
    # Requantised under a scale at most as large: only e4m3 values below 2^-6 of the scale can round.
    assert ((moved - origin).abs() <= 2.0 ** -10 * caches[2][1].repeat_interleave(64, 0)[:100]).all()


def test_captured_calls_follow_the_lengths_and_do_not_share_workspaces(gpu):
    s = Setup(gpu, [1000, 1900], None, 1, 4, 128, 256, 64)
    tables, caches = s.tables.to(gpu), s.caches()
    q = [s.q.to(gpu), query(2, 4, 128, s.dtype, 9).to(gpu)]
    lens = int32([1, 1], gpu)
    graphs, outs = [], []
    for i in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(ops.attention_fp8(q[i], *caches, tables, lens, return_lse=True))
        graphs.append(graph)
    for now in ([1000, 1900], [5, 700], [0, 1899], [999, 64]):
        lens.copy_(int32(now, gpu))
        for graph in graphs:
            graph.replay()
        for i in range(2):
            again = ops.attention_fp8(q[i], *caches, tables, lens, return_lse=True)
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(outs[i], again))
    s.q, s.lens = q[1].cpu(), [999, 64]
    check_attention(*outs[1], *s.want(), s.dtype, 128, 2.0 ** -8)


def test_calls_on_two_streams_at_once(gpu):
    setups = [Setup(gpu, [1500 + i], None, 2, 4, 128, 256, 64, seed=10 * i) for i in range(2)]
    args = [(s.q.to(gpu), *s.caches(), *s.batch()[0]) for s in setups]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream(gpu) for _ in setups], [[], []]
    for _ in range(10):
        for i, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                got[i].append(ops.attention_fp8(*args[i], return_lse=True))
    torch.cuda.synchronize()
    for s, results in zip(setups, got):
        want = s.want()
        check_attention(*results[0], *want, s.dtype, 128, 2.0 ** -8)
        assert all(torch.equal(a, b) for r in results[1:] for a, b in zip(r, results[0]))


# ---------------------------------------------------------------------------
# Weights

@pytest.mark.parametrize("lens,q_lens,heads,per_kv,hd,block,group,dtype", [
    (LENGTHS, None, 2, 4, 128, 64, 32, torch.bfloat16), (LENGTHS, None, 1, 20, 80, 16, 16, torch.float16),
    ([67, 190, 40, 55, 3, 0], [67, 70, 0, 1, 9, 2], 2, 3, 64, 32, 16, torch.bfloat16),
    ([300, 77], [300, 5], 1, 2, 256, 256, 64, torch.bfloat16), ([520], [64], 1, 8, 128, 64, 64, torch.bfloat16),
    ([200, 33], [100, 33], 2, 3, 112, 64, 16, torch.float16), ([700, 9], [8, 9], 1, 4, 128, 64, 32, torch.bfloat16)])
def test_weights(gpu, lens, q_lens, heads, per_kv, hd, block, group, dtype):
    s = Setup(gpu, lens, q_lens, heads, per_kv, hd, block, group, dtype, unused=NAN)
    _, lse, bound = s.want()
    where, how = s.batch()
    room = s.tables.shape[1] * block
    for width in (room, room - 9, room + 40):
        want = ref.weights(s.q, lse.float(), s.k, s.ks, s.tables, s.lens, s.ranges, s.scale, width)
        args = (s.q.to(gpu), lse.float().to(gpu), fp8(s.k, gpu), s.ks.to(gpu), *where, s.scale)
        before = torch.rand((len(lens), heads, width), device=gpu)
        fresh = ops.attention_weights_fp8(*args, **how, out=torch.empty_like(before))
        added = ops.attention_weights_fp8(*args, **how, weights=before, out=torch.empty_like(before))
        mine = before.clone()
        assert ops.attention_weights_fp8(*args, **how, weights=mine) is mine
        assert torch.equal(added, mine) and torch.equal(added, before + fresh)
        # An exponential's error is that of its score and of the lse's float32; a sum's, a half step a term.
        score = max((b[1] for b in bound.values()), default=0.0)
        top = float(lse[lse.isfinite()].abs().max()) if lse.isfinite().any() else 0.0
        terms = max((b - a for a, b in s.ranges), default=0) * per_kv
        off = 2 * ((hd + 8) * 2.0 ** -24 * score + (top + score) * 2.0 ** -22 + (terms + 8) * 2.0 ** -24)
        assert ((fresh.cpu().double() - want).abs() <= want * off + 2.0 ** -100).all()
    if q_lens is None:
        assert ops.attention_weights_fp8(*args, **how).shape == (len(lens), heads, room)


# ---------------------------------------------------------------------------
# The cache write

def check_store(gpu, k, v, caches, slots, want=None):
    """Stores into copies of the caches (codes, scales, for K and V) and compares with the definition."""
    on = [(fp8(c, gpu), s.to(gpu)) for c, s in caches]
    (kc, ks), (vc, vs) = on
    ops.store_kvcache_fp8(k.to(gpu), v.to(gpu), kc, vc, ks, vs, int32(slots, gpu))
    result = []
    for x, (codes, scales), (got, got_scale) in zip((k, v), caches, on):
        want, want_scale = ref.store(x.cpu(), codes, scales, slots)
        assert torch.equal(got_scale.cpu().nan_to_num(-1.0), want_scale.nan_to_num(-1.0))
        got = got.view(torch.uint8).cpu()
        same = (got == want) | (ref.decode(got).isnan() & ref.decode(want).isnan())
        assert same.all()
        result.append((got, got_scale.cpu()))
    return result


def rows(n, heads, hd, dtype, seed, spread=3.0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn((n, heads, hd), generator=g) * (torch.randn((n, heads, 1), generator=g) * spread).exp()
    return x.to(dtype)


def pool(blocks, block, group, heads, hd, seed=0):
    return [ref.random_cache(blocks, block, group, heads, hd, seed + i) for i in range(2)]


@pytest.mark.parametrize("heads,hd,block,group,dtype", [
    (2, 128, 64, 32, torch.bfloat16), (1, 64, 16, 16, torch.float16), (3, 80, 48, 16, torch.float32),
    (2, 256, 64, 64, torch.bfloat16), (1, 16, 32, 32, torch.bfloat16), (8, 128, 256, 256, torch.bfloat16),
    (1, 128, 1024, 1024, torch.float16), (5, 192, 32, 16, torch.float32),
    (1, 64, 512, 16, torch.bfloat16)])
def test_prompts_are_stored(gpu, heads, hd, block, group, dtype):
    lens = [1, block, 2 * block + 5, group + 1, 3]
    tables, blocks = tables_for(lens, block, 3)
    slots = [s for b, n in enumerate(lens) for s in ref.slots_of(tables[b], n, block)]
    n = len(slots)
    check_store(gpu, rows(n, heads, hd, dtype, 1), rows(n, heads, hd, dtype, 2), pool(blocks, block, group, heads, hd), slots)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_tokens_are_appended_and_scales_grow(gpu, dtype):
    heads, hd, block, group = 2, 64, 32, 16
    caches = pool(4, block, group, heads, hd)
    g = torch.Generator().manual_seed(4)
    for t in range(40):  # token by token over two blocks, each value range its own
        slots = [2 * block + t if t < block else t - block, -1]
        x = rows(2, heads, hd, dtype, 100 + t) * float(torch.randn(1, generator=g).mul(2).exp())
        caches = check_store(gpu, x.to(dtype), rows(2, heads, hd, dtype, 200 + t), caches, slots)


def test_slots_in_any_order_within_a_group_and_outside_the_cache(gpu):
    caches = pool(3, 32, 16, 2, 64)
    slots = [5, 3, 4, -1, 96, 2 ** 31 - 1, -2 ** 31, 40, 33, 47, 95, 80, 70, 64, 71]
    check_store(gpu, rows(15, 2, 64, torch.bfloat16, 1), rows(15, 2, 64, torch.bfloat16, 2), caches, slots)
    check_store(gpu, rows(3, 2, 64, torch.bfloat16, 1), rows(3, 2, 64, torch.bfloat16, 2), caches, [-1, -1, 96])


@pytest.mark.parametrize("gap", [1, 15, 70, 300, 1100])
def test_skipped_tokens_do_not_interrupt_a_group(gpu, gap):
    caches = pool(3, 32, 16, 1, 64)
    slots = [3, 4] + [-1] * gap + [5, 10 ** 6, 6, 16] + [-1] * gap + [17, 40, -1, 41]
    n = len(slots)
    check_store(gpu, rows(n, 1, 64, torch.bfloat16, 1), rows(n, 1, 64, torch.bfloat16, 2), caches, slots)


def test_the_later_of_two_tokens_with_one_slot_is_stored(gpu):
    caches = pool(2, 32, 16, 1, 64)
    slots = [17] * 300 + [16, 18, 17, 16]
    check_store(gpu, rows(304, 1, 64, torch.bfloat16, 1), rows(304, 1, 64, torch.bfloat16, 2), caches, slots)


def test_values_that_are_no_numbers_and_extremes(gpu):
    caches = pool(2, 32, 16, 1, 64)
    x = rows(8, 1, 64, torch.bfloat16, 1)
    x[0, 0, 3], x[1, 0, 4], x[2, 0, 5] = math.nan, math.inf, -math.inf
    x[3] = 0.0
    for slots in ([0, 1, 2, 3, 4, 5, 6, 7], [3, 4, 5, 6, 7, 8, 9, 10]):
        check_store(gpu, x, -x, caches, slots)
    zeros = torch.zeros((3, 1, 64), dtype=torch.bfloat16)
    check_store(gpu, zeros, zeros + math.nan, caches, [16, 17, 18])
    check_store(gpu, zeros + math.inf, zeros + 2.0 ** -130, caches, [16, 17, 18])
    huge = torch.full((3, 1, 64), 2.0 ** 127, dtype=torch.bfloat16)
    check_store(gpu, huge, huge * 2.0 ** -100, caches, [16, 17, 18])
    for amax in (448.0, 450.0, 224.0, 0.875, 0.87890625, 7.0, 7.03125):  # about the border to the next scale
        edge = torch.full((1, 1, 64), amax, dtype=torch.bfloat16)
        check_store(gpu, edge, -edge / 2, caches, [0])
    bad = [(c, s.clone()) for c, s in caches]  # a scale that is none counts as a group that holds nothing
    bad[0][1].fill_(math.nan)
    bad[1][1].fill_(0.0)
    check_store(gpu, x, x, bad, list(range(3, 11)))


def test_rows_of_a_fused_projection_are_stored(gpu):
    caches = pool(3, 32, 16, 2, 64)
    fused = torch.randn((50, 3 * 2 + 2, 64), generator=torch.Generator().manual_seed(3)).to(torch.bfloat16).to(gpu)
    check_store(gpu, fused[:, 4:6], fused[:, 6:8], caches, list(range(20, 70)))


def test_a_captured_store_replays(gpu):
    caches = pool(3, 32, 16, 2, 64)
    (kc, ks), (vc, vs) = [(fp8(c, gpu), s.to(gpu)) for c, s in caches]
    k, v = torch.zeros((4, 2, 64), dtype=torch.bfloat16, device=gpu), torch.zeros((4, 2, 64), dtype=torch.bfloat16, device=gpu)
    slots = int32([-1] * 4, gpu)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.store_kvcache_fp8(k, v, kc, vc, ks, vs, slots)
    for i, at in enumerate(([0, 1, 2, 3], [4, 5, 40, 41], [-1, 6, -1, 42])):
        new = [rows(4, 2, 64, torch.bfloat16, 20 + i), rows(4, 2, 64, torch.bfloat16, 30 + i)]
        k.copy_(new[0])
        v.copy_(new[1])
        slots.copy_(int32(at, gpu))
        graph.replay()
        torch.cuda.synchronize()
        caches = [ref.store(x, *c, at) for x, c in zip(new, caches)]
        assert torch.equal(kc.view(torch.uint8).cpu(), caches[0][0]) and torch.equal(ks.cpu(), caches[0][1])
        assert torch.equal(vc.view(torch.uint8).cpu(), caches[1][0]) and torch.equal(vs.cpu(), caches[1][1])


# ---------------------------------------------------------------------------
# Rotary positions

@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("n,q_heads,k_heads,hd,rotary", [
    (5, 4, 1, 128, 128), (1, 3, 2, 64, 32), (33, 2, 2, 80, 20), (7, 1, 0, 96, 96), (3, 2, 1, 33, 12), (3, 0, 5, 256, 64), (4, 2, 1, 50, 2),
    (2, 8, 8, 192, 192), (700, 1, 1, 16, 16)])
def test_rotary(gpu, n, q_heads, k_heads, hd, rotary, interleaved, dtype):
    g = torch.Generator().manual_seed(n)
    fused = torch.randn((n, q_heads + k_heads + 1, hd), generator=g).to(dtype)
    q, k = fused[:, :q_heads], fused[:, q_heads:q_heads + k_heads]
    positions = torch.randint(0, 2 ** 31, (n,), generator=g)
    positions[0] = 0
    if n > 2:
        positions[1], positions[2] = 2 ** 31 - 1, -5
    frequencies, _ = ops.rotary_frequencies(rotary, 1e6, device="cpu")
    magnitude = 1.25
    angle = positions.double()[:, None, None] * frequencies
    for at in (positions, positions.to(torch.int32)):
        got = ops.rotary_embed(q.to(gpu), k.to(gpu), at.to(gpu), frequencies.to(gpu), interleaved, magnitude)
        for x, y in zip((q.double(), k.double()), got):
            pairs = x[..., :rotary].unflatten(-1, (-1, 2) if interleaved else (2, -1))
            a, b = pairs.unbind(-1 if interleaved else -2)
            turned = torch.stack([a * angle.cos() - b * angle.sin(), b * angle.cos() + a * angle.sin()],
                                 -1 if interleaved else -2).flatten(-2) * magnitude
            reach = (a.abs() + b.abs()) * magnitude
            reach = torch.stack([reach, reach], -1 if interleaved else -2).flatten(-2)
            # Sine and cosine within 2 steps of fp32 and the fraction of a turn within half a one (pi 2^-25 rad at
            # most); three products and a sum; the angle itself within 2^-51 of up to 2^31 rad. Then the rounding.
            tol = HALF_STEP[dtype] * turned.abs() * 1.01 + reach * (10 * 2.0 ** -24 + 2.0 ** -20) + 2.0 ** -24
            y = y.cpu().double()
            assert ((y[..., :rotary] - turned).abs() <= tol).all()
            assert torch.equal(y[..., rotary:], x[..., rotary:])


@pytest.mark.parametrize("hd,rotary", [(128, 64), (50, 20), (35, 10)])
def test_rotary_in_place_and_into_views(gpu, hd, rotary):
    x = torch.randn((9, 6, hd), device=gpu).to(torch.bfloat16)
    positions, (frequencies, _) = torch.arange(9, device=gpu), ops.rotary_frequencies(rotary)
    want = ops.rotary_embed(x[:, :4], x[:, 4:5], positions, frequencies)
    into = torch.zeros((9, 8, hd), dtype=torch.bfloat16, device=gpu)
    got = ops.rotary_embed(x[:, :4], x[:, 4:5], positions, frequencies, query_out=into[:, 2:6], key_out=into[:, 7:])
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    assert (into[:, :2] == 0).all() and (into[:, 6] == 0).all()
    mine = x.clone()
    ops.rotary_embed(mine[:, :4], mine[:, 4:5], positions, frequencies, query_out=mine[:, :4], key_out=mine[:, 4:5])
    assert torch.equal(mine[:, :4], want[0]) and torch.equal(mine[:, 4:5], want[1]) and torch.equal(mine[:, 5:], x[:, 5:])


def test_rotary_of_no_tokens(gpu):
    x = torch.empty((0, 2, 64), dtype=torch.bfloat16, device=gpu)
    out = ops.rotary_embed(x, x, torch.empty(0, dtype=torch.int64, device=gpu), ops.rotary_frequencies(64)[0])
    assert out[0].shape == (0, 2, 64)


# ---------------------------------------------------------------------------
# The tokens to keep, and compaction

@pytest.mark.parametrize("kind", ["random", "few", "equal", "odd"])
@pytest.mark.parametrize("width,keep,recent", [(1, 1, 0), (40, 7, 3), (1024, 1024, 5), (1025, 1, 0), (3001, 700, 700),
                                               (5000, 1234, 0), (5000, 33, 90), (200, 500, 10), (70, 0, 0)])
def test_selected_tokens(gpu, kind, width, keep, recent):
    g = torch.Generator().manual_seed(width + keep)
    weights = torch.rand((4, 2, width), generator=g)
    if kind == "few":
        weights = torch.randint(0, 3, weights.shape, generator=g).float() / 7
    elif kind == "equal":
        weights.fill_(0.25)
    elif kind == "odd":
        special = torch.tensor([math.nan, math.inf, -math.inf, 0.0, -0.0, -1.0, 1e-42, -1e-42])
        weights = torch.where(weights < 0.5, special[torch.randint(0, 8, weights.shape, generator=g)], weights)
    lens = [width, width // 2, 0, 2 * width]
    got = ops.select_tokens(weights.to(gpu), int32(lens, gpu), keep, recent)
    for x, y in zip(got, ref.select(weights, lens, keep, recent)):
        assert torch.equal(x.cpu().nan_to_num(-7.0) if x.is_floating_point() else x.cpu(),
                           y.nan_to_num(-7.0) if y.is_floating_point() else y)


@pytest.mark.parametrize("pool", [3, 70, 5000])
def test_weights_that_are_no_numbers_come_last(gpu, pool):
    weights = torch.full((1, 1, pool), math.nan)
    weights[0, 0, pool // 2] = 5.0
    for keep in (1, 2, pool - 1):
        got = ops.select_tokens(weights.to(gpu), int32([pool], gpu), keep)
        want = ref.select(weights, [pool], keep, 0)
        assert torch.equal(got[0].cpu(), want[0]) and torch.equal(got[2].cpu().nan_to_num(-7.0), want[2].nan_to_num(-7.0))


@pytest.mark.parametrize("kind", ["random", "few", "equal"])
@pytest.mark.parametrize("width", [32768, 32769])
def test_selected_tokens_about_the_longest_held_row(gpu, width, kind):
    weights = torch.rand((1, 1, width), generator=torch.Generator().manual_seed(2))
    weights = (weights * 3).floor() if kind == "few" else weights * 0 if kind == "equal" else weights
    for keep, recent in ((width - 1, 0), (17, 3), (20000, 1)):
        got = ops.select_tokens(weights.to(gpu), int32([width], gpu), keep, recent)
        for x, y in zip(got, ref.select(weights, [width], keep, recent)):
            assert torch.equal(x.cpu(), y)


def test_selected_tokens_of_a_long_context(gpu):
    weights = (torch.rand((1, 2, 70001), generator=torch.Generator().manual_seed(2)) * 500).round() / 500
    got = ops.select_tokens(weights.to(gpu), int32([69999], gpu), 9001, 1000)
    for x, y in zip(got, ref.select(weights, [69999], 9001, 1000)):
        assert torch.equal(x.cpu(), y)


@pytest.mark.parametrize("heads,hd,block,group", [(2, 128, 64, 32), (1, 80, 16, 16), (3, 256, 128, 128), (1, 16, 48, 16)])
@pytest.mark.parametrize("given_lens", [False, True])
def test_compaction(gpu, heads, hd, block, group, given_lens):
    lens, keep = [5, 3 * block + 7, 0, 2 * block], block + group + 3
    tables, blocks = tables_for(lens, block, 1)
    new, more = tables_for([min(n, keep) for n in lens], block, 2, spare=0)
    new = torch.where(new >= 0, new + blocks, -1).int()
    caches = pool(blocks + more, block, group, heads, hd)
    g = torch.Generator().manual_seed(3)
    counts = torch.tensor([min(n, keep) for n in lens], dtype=torch.int32)
    indices = torch.full((4, heads, keep), -1, dtype=torch.int32)
    for b, n in enumerate(lens):
        for h in range(heads):
            indices[b, h, :counts[b]] = torch.randperm(n, generator=g)[:counts[b]].sort().values.int()
    indices[1, 0, 3], indices[1, heads - 1, 4] = -5, 10 ** 6  # no tokens: zeros
    caches[0][0].flatten(0, 1)[int(tables[0, 0]) * block, 0, 1] = NAN
    on = [(fp8(c, gpu), s.to(gpu)) for c, s in caches]
    (kc, ks), (vc, vs) = on
    ops.compact_kvcache_fp8(kc, vc, ks, vs, tables.to(gpu), indices.to(gpu), counts.to(gpu), new.to(gpu),
                            int32(lens, gpu) if given_lens else None)
    for (codes, scales), (got, got_scale) in zip(caches, on):
        want, want_scale = ref.compact(codes, scales, tables, indices, counts, new, lens if given_lens else None)
        assert torch.equal(got_scale.cpu(), want_scale)
        got = got.view(torch.uint8).cpu()
        assert ((got == want) | (ref.decode(got).isnan() & ref.decode(want).isnan())).all()


# ---------------------------------------------------------------------------
# Together, as a model runner calls them

def test_a_sequence_from_prompt_to_eviction(gpu):
    """Prompt, decode steps, the blocks saved and restored elsewhere, eviction and a step behind it, on two layers."""
    layers, nb, bs, group, heads, per_kv, hd = 2, 12, 64, 32, 2, 4, 64
    g = torch.Generator(device=gpu).manual_seed(0)
    codes = torch.zeros((2, layers, nb, bs, heads, hd), dtype=torch.uint8, device=gpu).view(torch.float8_e4m3fn)
    scales = torch.zeros((2, layers, nb, bs // group, heads, 1), device=gpu)
    frequencies, magnitude = ops.rotary_frequencies(hd, 1e4, "by_parts", 4.0, 128)
    table, length = [7, 2, 9, 4], 0
    history = [[] for _ in range(layers)]  # float32 (k, v) as stored
    weights = torch.zeros((layers, 1, heads, nb * bs), device=gpu)

    def step(n, positions):
        nonlocal length
        slots = int32([table[t // bs] * bs + t % bs for t in range(length, length + n)], gpu)
        length += n
        tables, lens = int32([table], gpu), int32([length], gpu)
        for layer in range(layers):
            qkv = torch.randn((n, heads * (per_kv + 2), hd), generator=g, device=gpu).to(torch.bfloat16)
            q, k = ops.rotary_embed(qkv[:, :heads * per_kv], qkv[:, heads * per_kv:-heads], positions, frequencies,
                                    magnitude=magnitude)
            cache = (codes[0, layer], codes[1, layer], scales[0, layer], scales[1, layer])
            ops.store_kvcache_fp8(k, qkv[:, -heads:], *cache, slots)
            how = {} if n == 1 else dict(cu_seqlens=int32([0, n], gpu), max_seqlen=n)
            out, lse = ops.attention_fp8(q, *cache, tables, lens, return_lse=True, **how)
            ops.attention_weights_fp8(q, lse, cache[0], cache[2], tables, lens, weights=weights[layer], **how)
            want, want_lse, bound = ref.attention(q.cpu(), cache[0].view(torch.uint8).cpu(), cache[1].view(torch.uint8).cpu(),
                                                  cache[2].cpu(), cache[3].cpu(), tables.cpu(), [length], [(0, n)], hd ** -0.5)
            check_attention(out, lse, want, want_lse, bound, torch.bfloat16, hd, 2.0 ** -8)
            history[layer].append((k.float(), qkv[:, -heads:].float()))

    step(150, torch.arange(150, device=gpu))
    for t in range(150, 153):
        step(1, torch.tensor([t], device=gpu))
    for layer in range(layers):
        total = weights[layer, 0, :, :length].sum(-1).cpu().double()
        # Each row's softmax sums to 1 for each query head; 153 tokens, each sum within some steps of fp32.
        assert ((total - 153 * per_kv).abs() <= 153 * per_kv * 2.0 ** -17).all()
        # What is stored is within half a step of e4m3 (2^-4 of the value, or 2^-10 of the scale below 2^-6 of it), a
        # growing scale's second rounding included.
        for half in range(2):
            x = torch.cat([h[half] for h in history[layer]])
            slots = torch.tensor(ref.slots_of(table, length, bs), device=gpu)
            s = scales[half, layer].repeat_interleave(group, 1).flatten(0, 1)[slots]
            y = codes[half, layer].flatten(0, 1).view(torch.uint8)[slots].view(torch.float8_e4m3fn).float() * s
            assert ((y - x).abs() <= 2 * torch.maximum(2.0 ** -4 * x.abs(), 2.0 ** -10 * s)).all()
    # Blocks of both pools leave and come back into other blocks: nothing that is read changes.
    q = torch.randn((1, heads * per_kv, hd), generator=g, device=gpu).to(torch.bfloat16)

    def look(layer, table):
        return ops.attention_fp8(q, codes[0, layer], codes[1, layer], scales[0, layer], scales[1, layer],
                                 int32([table], gpu), int32([length], gpu))

    before = [look(layer, table) for layer in range(layers)]
    moved = [1, 3, 5, 8]
    for pool in (codes.view(torch.uint8), scales):
        _, _, stride = ops.entry_layout(ops.pool_layout(pool), ops.FORMAT_RAW)
        host = torch.empty(4 * stride, dtype=torch.uint8, pin_memory=True)
        entries = [host.data_ptr() + i * stride for i in range(4)]
        ops.save_blocks(pool, table, entries, ops.FORMAT_RAW)
        torch.cuda.synchronize()
        device_copy = host.to(gpu)
        entries = [device_copy.data_ptr() + i * stride for i in range(4)]
        ops.restore_blocks(pool, moved, entries, ops.FORMAT_RAW)
    assert all(torch.equal(look(layer, moved), b) for layer, b in enumerate(before))
    # Eviction to 70 tokens, 20 of them the last ones, into blocks 0 and 6.
    table, keep = moved, 70
    lens = int32([length], gpu)
    for layer in range(layers):
        cache = (codes[0, layer], codes[1, layer], scales[0, layer], scales[1, layer])
        indices, counts, kept = ops.select_tokens(weights[layer], lens, keep, 20)
        for a, b in zip((indices, counts, kept), ref.select(weights[layer].cpu(), [length], keep, 20)):
            assert torch.equal(a.cpu(), b)
        assert (indices[0, :, -20:].cpu() == torch.arange(length - 20, length)).all()
        old = [(codes[i, layer].view(torch.uint8).cpu(), scales[i, layer].cpu()) for i in range(2)]
        ops.compact_kvcache_fp8(*cache, int32([table], gpu), indices, counts, int32([[0, 6]], gpu))
        for i, (c, s) in enumerate(old):
            want, want_scale = ref.compact(c, s, torch.tensor([table]), indices.cpu(), counts.cpu(), torch.tensor([[0, 6]]))
            assert torch.equal(codes[i, layer].view(torch.uint8).cpu(), want)
            assert torch.equal(scales[i, layer].cpu(), want_scale)
        weights[layer].zero_()
        weights[layer, :, :, :keep] = kept
    table, length = [0, 6], keep
    step(1, torch.tensor([153], device=gpu))


def test_calls_give_the_same_with_and_without_the_native_binding(gpu, monkeypatch):
    from kvx import _lib

    s = Setup(gpu, [70, 5, 130], [20, 5, 7], 2, 3, 64, 32, 16)
    decode = Setup(gpu, [70, 5, 130], None, 2, 3, 64, 32, 16)
    where, how = s.batch()
    k, v = rows(6, 2, 64, torch.bfloat16, 1).to(gpu), rows(6, 2, 64, torch.bfloat16, 2).to(gpu)
    positions, (frequencies, _) = torch.arange(32, device=gpu), ops.rotary_frequencies(64)
    results = []
    for binding in (_lib.load_bind(), _lib._NoBind):
        monkeypatch.setattr(_lib, "_bind", binding)
        cache = s.caches()
        out, lse = ops.attention_fp8(s.q.to(gpu), *cache, *where, return_lse=True, **how)
        alone = ops.attention_fp8(s.q.to(gpu), *cache, *where, s.scale, cu_seqlens=how["cu_seqlens"])
        single = ops.attention_fp8(decode.q.to(gpu), *decode.caches(), *decode.batch()[0], out=torch.empty_like(decode.q, device=gpu))
        weights = ops.attention_weights_fp8(s.q.to(gpu), lse, cache[0], cache[2], *where, **how)
        ops.attention_weights_fp8(s.q.to(gpu), lse, cache[0], cache[2], *where, s.scale, weights=weights, **how)
        indices, counts, kept = ops.select_tokens(weights, where[1], 9, 3)
        ops.store_kvcache_fp8(k, v, *cache, int32([3, 4, 5, -1, 40, 41], gpu))
        turned = ops.rotary_embed(s.q.to(gpu), s.q[:, :2].to(gpu), positions, frequencies, True, 2.0)
        inplace = s.q.to(gpu)
        assert ops.rotary_embed(inplace, inplace[:, :0], positions, frequencies, query_out=inplace)[0] is inplace
        new = int32([[int(s.tables.max()) + 1] * 1] * 3, gpu)
        ops.compact_kvcache_fp8(*cache, where[0], indices[:1].repeat(3, 1, 1), counts.clamp_max(0), new, where[1])
        results.append([out, lse, alone, single, weights, indices, counts, kept, *turned, inplace,
                        *(c.view(torch.uint8) for c in cache)])
    for a, b in zip(*results):
        assert a.shape == b.shape and a.dtype == b.dtype and torch.equal(a, b)
    assert torch.equal(results[0][0], results[0][2])


@pytest.mark.parametrize("layers,block,group,heads,hd", [(3, 64, 16, 2, 128), (2, 32, 32, 1, 80), (1, 256, 64, 8, 64)])
def test_blocks_of_codes_and_scales_are_saved_and_restored(gpu, layers, block, group, heads, hd):
    caches = [ref.random_cache(7 * layers, block, group, heads, hd, i) for i in range(2)]
    codes = torch.stack([c for c, _ in caches]).view(2, layers, 7, block, heads, hd).to(gpu).view(torch.float8_e4m3fn)
    scales = torch.stack([s for _, s in caches]).view(2, layers, 7, block // group, heads, 1).to(gpu)
    for plane in (codes, scales):
        want = plane.view(torch.uint8).cpu().clone()
        stride = ops.entry_layout(ops.pool_layout(plane), ops.FORMAT_RAW)[2]
        entries = torch.empty((3, stride), dtype=torch.uint8, pin_memory=True)
        at = [entries[i].data_ptr() for i in range(3)]
        ops.save_blocks(plane, [5, 0, 2], at, ops.FORMAT_RAW)
        plane.view(torch.uint8).fill_(0x55)
        ops.restore_blocks(plane, [1, 6, 3], at, ops.FORMAT_RAW)
        got = plane.view(torch.uint8).cpu()
        for was, now in zip([5, 0, 2], [1, 6, 3]):
            assert torch.equal(got[:, :, now], want[:, :, was])
        for other in (0, 2, 4, 5):
            assert (got[:, :, other] == 0x55).all()


@pytest.mark.parametrize("rows", [33, 64, 127, 128, 129])
def test_weights_about_the_border_between_the_kernels(gpu, rows):
    test_weights(gpu, [190, 300, 5, 0], [rows, 8, 5, 1], 2, 1, 128, 64, 16, torch.bfloat16)


@pytest.mark.parametrize("lens", [[255, 256], [257, 511], [513, 1025], [2048, 1000]])
def test_chunks_about_the_borders_of_splits(gpu, lens):
    Setup(gpu, lens, [40, 3], 1, 4, 128, 256, 16, unused=NAN).check()


@pytest.mark.parametrize("heads,hd,group", [(8, 128, 16), (8, 128, 32), (4, 256, 64), (16, 64, 16)])
def test_tokens_appended_to_many_groups_at_once(gpu, heads, hd, group):
    # More than one workgroup for each: a workgroup's tokens continue, start and skip groups of their own.
    n, block = 500, 64
    g = torch.Generator().manual_seed(5)
    groups = torch.randperm(n + 7, generator=g)[:n]
    slots = groups * group + torch.randint(0, group, (n,), generator=g)
    slots[::9], slots[4::50] = groups[::9] * group, -1
    caches = pool(-(-(n + 7) * group // block), block, group, heads, hd)
    check_store(gpu, rows(n, heads, hd, torch.bfloat16, 1, 30.0), rows(n, heads, hd, torch.bfloat16, 2), caches, slots.tolist())
