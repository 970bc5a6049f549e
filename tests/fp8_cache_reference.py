"""The operators around an e4m3 KV cache by their definitions, in 64 bits on the CPU, one row at a time."""

import math

import torch

FP8 = torch.float8_e4m3fn
FLOOR = 2.0 ** -100


def least_scale(amax: float) -> float:
    """The least power of two s >= 2^-100 with amax <= 448 s."""
    s = FLOOR
    while amax > 448.0 * s:
        s *= 2.0
    return s


def encode(x: torch.Tensor, scale: float) -> torch.Tensor:
    """float64 values -> e4m3 codes (uint8) of x / scale. Exact quotients (scale is a power of two) rounded once: those
    of bf16, fp16 and fp32 inputs are fp32 values, and torch's conversion from fp32 rounds to nearest even."""
    return (x / scale).clamp(-448.0, 448.0).float().to(FP8).view(torch.uint8)


def decode(codes: torch.Tensor) -> torch.Tensor:
    return codes.view(FP8).double()


def finite_amax(x: torch.Tensor) -> float:
    x = x.abs()[x.isfinite()]
    return float(x.max()) if x.numel() else 0.0


def random_cache(blocks, block, group, heads, hd, seed, powers=True):
    """(codes uint8 [NB, BS, H, hd], scales float32 [NB, BS / G, H, 1]) of any finite codes, on the CPU."""
    g = torch.Generator().manual_seed(seed)
    codes = torch.randint(0, 256, (blocks, block, heads, hd), generator=g, dtype=torch.uint8)
    codes[(codes & 0x7F) == 0x7F] = 0x30
    scales = torch.randint(-9, -6, (blocks, block // group, heads, 1), generator=g).float().exp2()
    if not powers:
        scales *= torch.rand(scales.shape, generator=g) + 0.5
    return codes, scales


def values(codes, scales):
    """float64 [slots, H, hd]."""
    group = codes.shape[1] // scales.shape[1]
    return (decode(codes) * scales.double().repeat_interleave(group, 1)).flatten(0, 1)


def slots_of(table, context, block):
    """The slots of a sequence's cached tokens; None where the table names no block."""
    context = max(0, min(context, len(table) * block))
    return [int(table[t // block]) * block + t % block for t in range(context)]


def attention(q, k_codes, v_codes, k_scale, v_scale, tables, lens, ranges, softmax_scale):
    """(out, lse, bound): float64 [N, Hq, hd], [N, Hq], and {(row, head): (sum p |v|, largest sum |q k|, keys)}.

    Rows that are no sequence's stay NaN."""
    n, heads, hd = q.shape
    block, kv_heads, blocks = k_codes.shape[1], k_codes.shape[2], k_codes.shape[0]
    k, v, q = values(k_codes, k_scale), values(v_codes, v_scale), q.double()
    out = torch.full((n, heads, hd), math.nan, dtype=torch.float64)
    lse = torch.full((n, heads), math.nan, dtype=torch.float64)
    bound = {}
    for b, (first, end) in enumerate(ranges):
        slots = slots_of(tables[b], int(lens[b]), block)
        for row in range(first, end):
            seen = slots[:max(0, len(slots) - (end - first) + (row - first) + 1)]
            seen = torch.tensor([s for s in seen if 0 <= s // block < blocks], dtype=torch.long)
            for h in range(heads):
                kv = h // (heads // kv_heads)
                if not len(seen):
                    out[row, h], lse[row, h] = 0.0, -math.inf
                    continue
                s = k[seen, kv] @ q[row, h] * softmax_scale
                p = torch.softmax(s, 0)
                out[row, h] = (p[:, None] * v[seen, kv]).sum(0)
                lse[row, h] = torch.logsumexp(s, 0)
                bound[row, h] = ((p[:, None] * v[seen, kv].abs()).sum(0),
                                 float((k[seen, kv].abs() @ q[row, h].abs()).max()) * abs(softmax_scale), len(seen))
    return out, lse, bound


def weights(q, lse, k_codes, k_scale, tables, lens, ranges, softmax_scale, width):
    """float64 [B, H, width]: what each cached token received."""
    block, kv_heads, blocks = k_codes.shape[1], k_codes.shape[2], k_codes.shape[0]
    k, q, lse = values(k_codes, k_scale), q.double(), lse.double()
    heads = q.shape[1]
    total = torch.zeros((len(ranges), kv_heads, width), dtype=torch.float64)
    for b, (first, end) in enumerate(ranges):
        slots = slots_of(tables[b], int(lens[b]), block)
        for row in range(first, end):
            seen = [(t, s) for t, s in enumerate(slots[:max(0, len(slots) - (end - first) + (row - first) + 1)])
                    if 0 <= s // block < blocks and t < width]
            if not seen:
                continue
            t, s = (torch.tensor(x) for x in zip(*seen))
            for h in range(heads):
                kv = h // (heads // kv_heads)
                if lse[row, h] > -math.inf:
                    total[b, kv, t] += torch.exp(k[s, kv] @ q[row, h] * softmax_scale - lse[row, h])
    return total


def store(x, codes, scales, slots):
    """One of K and V written into copies of (codes, scales)."""
    codes, scales = codes.clone(), scales.clone()
    group = codes.shape[1] // scales.shape[1]
    flat, flat_scale = codes.flatten(0, 1), scales.view(-1, scales.shape[2])
    tokens = {}
    for i, s in enumerate(slots):
        if 0 <= s < flat.shape[0]:
            tokens.setdefault(s // group, {})[s % group] = i  # the later of two stays
    for g, rows in tokens.items():
        for h in range(codes.shape[2]):
            new = {r: x[i, h].double() for r, i in rows.items()}
            fit = least_scale(max(finite_amax(v) for v in new.values()))
            held = float(flat_scale[g, h])
            if 0 not in rows and 0 < held < math.inf:
                if held > fit:
                    fit = held
                elif fit > held:
                    at = slice(g * group, (g + 1) * group)
                    flat[at, h] = encode(decode(flat[at, h]) * held, fit)
            flat_scale[g, h] = fit
            for r, v in new.items():
                flat[g * group + r, h] = encode(v, fit)
    return codes, scales


def select(weights, lens, keep, recent):
    """(indices, counts, kept) by sorting."""
    b, heads, width = weights.shape
    indices = torch.full((b, heads, keep), -1, dtype=torch.int32)
    kept = torch.zeros((b, heads, keep))
    counts = torch.tensor([min(keep, max(0, min(int(n), width))) for n in lens], dtype=torch.int32)
    for i in range(b):
        n = max(0, min(int(lens[i]), width))
        last = min(recent, int(counts[i]))
        for h in range(heads):
            w = weights[i, h, :n - last].tolist()
            order = sorted(range(len(w)), key=lambda t: (math.isnan(w[t]), 0.0 if math.isnan(w[t]) else -w[t], t))
            picked = sorted(order[:int(counts[i]) - last]) + list(range(n - last, n))
            indices[i, h, :len(picked)] = torch.tensor(picked, dtype=torch.int32)
            kept[i, h, :len(picked)] = weights[i, h, picked]
    return indices, counts, kept


def compact(codes, scales, tables, indices, counts, new_tables, lens=None):
    """One of K and V with its kept tokens moved, in copies of (codes, scales)."""
    block, heads = codes.shape[1:3]
    group = block // scales.shape[1]
    x = values(codes, scales)
    codes, scales = codes.clone(), scales.clone()
    flat, flat_scale = codes.flatten(0, 1), scales.view(-1, heads)
    for b, n in enumerate(counts.tolist()):
        limit = tables.shape[1] * block if lens is None else min(int(lens[b]), tables.shape[1] * block)
        for h in range(heads):
            for first in range(0, n, group):
                rows = []
                for j in range(first, min(first + group, n)):
                    t = int(indices[b, h, j])
                    there = 0 <= t < limit and 0 <= int(tables[b, t // block]) < codes.shape[0]
                    rows.append(x[int(tables[b, t // block]) * block + t % block, h] if there
                                else torch.zeros(codes.shape[3], dtype=torch.float64))
                to = int(new_tables[b, first // block])
                if not 0 <= to < codes.shape[0]:
                    continue
                fit = least_scale(max(finite_amax(r) for r in rows))
                slot = to * block + first % block
                flat_scale[slot // group, h] = fit
                for j, r in enumerate(rows):
                    flat[slot + j, h] = encode(r, fit)
    return codes, scales
