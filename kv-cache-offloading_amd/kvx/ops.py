"""Operator API of the KV-block copy path, backed by libkvx's HIP kernels.

These functions keep the reference's names, argument meaning and out-param
style (nanovllm/layers/attention.py:33-40, nanovllm/engine/cpu_prefix_cache.py:20-28)
and accept the same tensors. Work is queued on torch's current HIP stream of
the tensors' device. Tensors must live on a ROCm device: there is no CPU or
torch-op fallback, so a missing or unloadable libkvx raises.
"""

import ctypes
import threading
from math import ceil, floor, log, pi, prod

import numpy as np
import torch

from kvx import _lib
from kvx._lib import BlockLayout, check, int32_array, lib, uint64_array
from kvx._lib import bind as _bind

FORMAT_RAW, FORMAT_FP8 = _lib.FORMAT_RAW, _lib.FORMAT_FP8
SCALE_DTYPES = {torch.bfloat16: _lib.SCALE_BF16, torch.float32: _lib.SCALE_FP32}

_INT32_MAX = 2 ** 31 - 1  # what ctypes would cut larger numbers to, without an error

# Largest finite float8_e4m3fn magnitude (the codec's clamp bound).
FP8_MAX = 448.0


def _require_device(*tensors: torch.Tensor) -> torch.device:
    device = tensors[0].device
    for t in tensors:
        if t.device.type != "cuda":
            raise ValueError("kvx operators need tensors on a ROCm device (got %s)" % t.device)
        if t.device != device:
            raise ValueError("kvx operators need all tensors on one device")
    return device


def _stream(device: torch.device, stream=None) -> int:
    if stream is None:
        stream = torch.cuda.current_stream(device)
    return stream.cuda_stream if hasattr(stream, "cuda_stream") else int(stream)


# A valid call goes to libkvx straight from the native binding (_lib.bind); one that the binding declines comes back as
# None and is checked, refused or carried out by the Python below it.

def store_kvcache(key: torch.Tensor, value: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                  slot_mapping: torch.Tensor):
    """Slot-mapped paged KV write (nanovllm/layers/attention.py:33-40).

    key/value: [N, num_heads, head_dim] with contiguous rows (the row stride
    may differ, e.g. V is a view of a fused QKV output). k_cache/v_cache:
    contiguous [num_blocks, block_size, num_heads, head_dim] layer views of
    the pool. slot_mapping: int32 [N]; -1 (graph padding) skips a token, and
    so does any slot outside the cache. Capturable in a HIP graph.

    Every call makes the reference's four asserts and checks shapes, dtypes
    and devices.
    """
    rc = _bind().store(key, value, k_cache, v_cache, slot_mapping)
    if rc is not None:
        if rc:
            check(rc, "store_kvcache")
        return
    N, num_heads, head_dim = key.shape
    D = num_heads * head_dim
    assert key.stride(-1) == 1 and value.stride(-1) == 1
    assert key.stride(1) == head_dim and value.stride(1) == head_dim
    assert k_cache.stride(1) == D and v_cache.stride(1) == D
    assert slot_mapping.numel() == N
    dtype = key.dtype
    if not (k_cache.dtype == v_cache.dtype == dtype):
        raise TypeError("key, value and caches must share one dtype")
    if not (k_cache.is_contiguous() and v_cache.is_contiguous()) or k_cache.numel() != v_cache.numel():
        raise ValueError("k_cache and v_cache must be equally sized contiguous slot arrays")
    index = _require_device(k_cache, v_cache).index
    if value.shape != key.shape:
        raise ValueError("key and value shapes differ")
    if value.dtype != dtype:
        raise TypeError("key, value and caches must share one dtype")
    if slot_mapping.dtype != torch.int32 or not slot_mapping.is_contiguous():
        raise TypeError("slot_mapping must be a contiguous int32 tensor")
    if key.get_device() != index or value.get_device() != index or slot_mapping.get_device() != index:
        _require_device(k_cache, key, value, slot_mapping)
        raise ValueError("kvx operators need all tensors on one device")
    if N == 0:
        return
    check(lib().kvx_store_kvcache(key.data_ptr(), key.stride(0), value.data_ptr(), value.stride(0), k_cache.data_ptr(),
                                  v_cache.data_ptr(), slot_mapping.data_ptr(), N, num_heads, head_dim,
                                  key.element_size(), k_cache.numel() // D,
                                  torch._C._cuda_getCurrentRawStream(index)), "store_kvcache")


# ---------------------------------------------------------------------------
# Views as [planes][plane_rows][head_dim]

def _plane_views(t: torch.Tensor):
    """Yields (tensor, planes, plane_rows, plane_stride) covering `t` in row-major order.

    The rows (last dim) must be contiguous. A view whose leading dims do not
    collapse into one uniformly strided plane dimension is split along its
    first dim.
    """
    if t.stride(-1) != 1 and t.shape[-1] > 1:
        raise ValueError("the last dim (head_dim) must be contiguous")
    hd = t.shape[-1]
    sizes, strides = list(t.shape[:-1]), list(t.stride()[:-1])
    dims = [(s, st) for s, st in zip(sizes, strides) if s != 1]
    # Longest suffix of dims whose rows are packed back to back.
    rows, expect, k = 1, hd, len(dims)
    while k > 0 and dims[k - 1][1] == expect:
        rows *= dims[k - 1][0]
        expect *= dims[k - 1][0]
        k -= 1
    lead = dims[:k]
    collapsible = all(lead[i][1] == lead[i + 1][1] * lead[i + 1][0] for i in range(len(lead) - 1))
    if collapsible:
        planes = prod(s for s, _ in lead) if lead else 1
        plane_stride = lead[-1][1] if lead else rows * hd
        yield t, planes, rows, plane_stride
        return
    for i in range(t.shape[0]):
        yield from _plane_views(t[i])


def _check_codec(values: torch.Tensor, payload: torch.Tensor, scale: torch.Tensor):
    if values.dtype != torch.bfloat16:
        raise NotImplementedError("the FP8 codec supports bfloat16 KV values")
    if payload.dtype != torch.float8_e4m3fn or payload.shape != values.shape or not payload.is_contiguous():
        raise ValueError("payload must be a contiguous float8_e4m3fn tensor shaped like the values")
    if scale.dtype not in SCALE_DTYPES or not scale.is_contiguous() or \
            tuple(scale.shape) != (*values.shape[:-1], 1):
        raise ValueError("scale must be a contiguous bfloat16/float32 tensor shaped [..., 1]")


def _codec(save: bool, values: torch.Tensor, payload: torch.Tensor, scale: torch.Tensor):
    rc = _bind().codec(save, values, payload, scale)
    if rc is not None:
        check(rc, "fp8_quantize" if save else "fp8_dequantize")
        return
    _check_codec(values, payload, scale)
    device = _require_device(values, payload, scale)
    if values.numel() == 0:
        return
    hd = values.shape[-1]
    stream = _stream(device)
    scale_bytes = scale.element_size()
    row = 0
    fn = lib().kvx_save_blocks if save else lib().kvx_restore_blocks
    for view, planes, rows, plane_stride in _plane_views(values):
        layout = BlockLayout(plane_stride, 0, planes, rows, hd, 1, 2, SCALE_DTYPES[scale.dtype])
        entry = payload.data_ptr() + row * hd
        scale_offset = scale.data_ptr() + row * scale_bytes - entry
        check(fn(view.data_ptr(), ctypes.byref(layout), FORMAT_FP8, int32_array([0]), uint64_array([entry]), 1,
                 scale_offset, stream), "fp8_quantize" if save else "fp8_dequantize")
        row += planes * rows


def fp8_quantize(source: torch.Tensor, payload: torch.Tensor, scale: torch.Tensor):
    """float8_e4m3fn payload with one scale (scale's dtype) per vector along the last dim.

    Same contract as nanovllm/engine/cpu_prefix_cache.py:20-24:
    scale = max(fp32(amax|x|) / 448, 1e-30) in scale's dtype, then
    payload = e4m3(clamp(fp32(x) / fp32(scale), -448, 448)). `source` may be a
    strided view (e.g. pool[:, :, block]); payload and scale are contiguous.
    """
    _codec(True, source, payload, scale)


def fp8_dequantize(payload: torch.Tensor, scale: torch.Tensor, target: torch.Tensor):
    """target = bf16(fp32(payload) * fp32(scale)) (nanovllm/engine/cpu_prefix_cache.py:27-28)."""
    _codec(False, target, payload, scale)


# ---------------------------------------------------------------------------
# Pool block lists

def pool_layout(pool: torch.Tensor, scale_dtype: torch.dtype | None = None) -> BlockLayout:
    """kvx_block_layout of a contiguous [2, L, NB, BS, H, hd] pool (model_runner.py:120)."""
    if pool.ndim != 6 or pool.shape[0] != 2 or not pool.is_contiguous():
        raise ValueError("pool must be a contiguous [2, layers, blocks, block_size, heads, head_dim] tensor")
    _, layers, nb, bs, heads, hd = pool.shape
    if scale_dtype is not None and scale_dtype not in SCALE_DTYPES:
        raise ValueError(f"FP8 scales must be bfloat16 or float32, not {scale_dtype}")
    # Without an explicit scale dtype, scales follow the pool dtype (the reference's default); pools of other
    # dtypes only use RAW entries, which carry no scales.
    scale = SCALE_DTYPES.get(scale_dtype if scale_dtype is not None else pool.dtype, _lib.SCALE_BF16)
    return BlockLayout(nb * bs * heads * hd, bs * heads * hd, 2 * layers, bs * heads, hd, nb,
                       pool.element_size(), scale)


def entry_layout(layout: BlockLayout, fmt: int) -> tuple[int, int, int]:
    """(logical bytes, scale offset, entry stride) of one host entry."""
    logical, offset, stride = ctypes.c_int64(), ctypes.c_int64(), ctypes.c_int64()
    check(lib().kvx_entry_layout(ctypes.byref(layout), fmt, ctypes.byref(logical), ctypes.byref(offset),
                                 ctypes.byref(stride)), "entry_layout")
    return logical.value, offset.value, stride.value


def save_blocks(pool: torch.Tensor, block_ids, entries, fmt: int, scale_dtype: torch.dtype | None = None,
                stream=None):
    """Queues save (gather [+ FP8 quantise]) of pool blocks into entry addresses."""
    if stream is None:
        rc = _bind().blocks(True, pool, block_ids, entries, fmt, scale_dtype)
        if rc is not None:
            check(rc, "save_blocks")
            return
    layout = pool_layout(pool, scale_dtype)
    _, offset, _ = entry_layout(layout, fmt)
    ids, entries = list(block_ids), list(entries)
    if len(ids) != len(entries):
        raise ValueError("one entry per block")
    device = _require_device(pool)
    check(lib().kvx_save_blocks(pool.data_ptr(), ctypes.byref(layout), fmt, int32_array(ids),
                                uint64_array(entries), len(ids), offset, _stream(device, stream)), "save_blocks")


def restore_blocks(pool: torch.Tensor, block_ids, entries, fmt: int, scale_dtype: torch.dtype | None = None,
                   stream=None):
    """Queues restore ([FP8 dequantise +] scatter) of entry addresses into pool blocks."""
    if stream is None:
        rc = _bind().blocks(False, pool, block_ids, entries, fmt, scale_dtype)
        if rc is not None:
            check(rc, "restore_blocks")
            return
    layout = pool_layout(pool, scale_dtype)
    _, offset, _ = entry_layout(layout, fmt)
    ids, entries = list(block_ids), list(entries)
    if len(ids) != len(entries):
        raise ValueError("one entry per block")
    device = _require_device(pool)
    check(lib().kvx_restore_blocks(pool.data_ptr(), ctypes.byref(layout), fmt, int32_array(ids),
                                   uint64_array(entries), len(ids), offset, _stream(device, stream)),
          "restore_blocks")


# ---------------------------------------------------------------------------
# Step inputs: host-to-device uploads read by a kernel

class _PinnedRing:
    """Pinned host buffers that kvx_upload kernels read, used in turn.

    A buffer is rewritten only after the kernel that last read it has run
    (an event per buffer; the host waits only if the stream is that far
    behind). A buffer grows, to a power of two, when an array does not fit.
    """

    def __init__(self, count: int = 16):
        self.buffers: list[torch.Tensor | None] = [None] * count
        self.events: list[torch.cuda.Event | None] = [None] * count
        self.next = 0

    def stage(self, host: np.ndarray) -> tuple[torch.Tensor, int]:
        """(a pinned uint8 buffer holding `host`'s bytes, its slot); pass the slot to read_by after the launch."""
        i = self.next
        self.next = (i + 1) % len(self.buffers)
        if self.events[i] is not None:
            self.events[i].synchronize()
        nbytes = host.nbytes
        buf = self.buffers[i]
        if buf is None or buf.numel() < nbytes:
            buf = torch.empty(max(256, 1 << (nbytes - 1).bit_length()), dtype=torch.uint8, pin_memory=True)
            self.buffers[i] = buf
        buf[:nbytes].numpy()[:] = host.reshape(-1).view(np.uint8)
        return buf, i

    def read_by(self, i: int, stream: torch.cuda.Stream):
        event = self.events[i] or torch.cuda.Event()
        event.record(stream)
        self.events[i] = event


_rings: dict[int, _PinnedRing] = {}
_rings_lock = threading.Lock()


def upload(values: np.ndarray, device: torch.device, stream=None, out: torch.Tensor | None = None) -> torch.Tensor:
    """A device copy of a host array, read from pinned memory by a kernel on the current stream (kvx_upload).

    Replaces the pinned non-blocking copies of a step's inputs
    (nanovllm/engine/model_runner.py:169-173, 187-190): a DMA copy on the
    compute stream queues behind every host-to-device DMA already queued on
    the device, a restore stream's included, while the kernel does not. The
    host does not wait for the GPU, except when 16 uploads are still queued.
    `out` (a contiguous device tensor of the array's dtype and size, e.g. a
    captured graph's static input) receives the copy instead of a new tensor.
    `stream` is a torch.cuda.Stream of the device (default: its current stream).
    Eager only: later uploads rewrite the ring's buffers, so a captured graph
    would replay whatever they hold by then. Inside a graph, call kvx_upload
    with a pinned source the caller owns and rewrites between replays.
    """
    host = np.ascontiguousarray(values)
    device = torch.device(device)
    if device.type != "cuda":
        raise ValueError(f"upload needs a ROCm device (got {device})")
    index = device.index if device.index is not None else torch.cuda.current_device()
    device = torch.device("cuda", index)
    dtype = torch.from_numpy(host[:0]).dtype
    if out is None:
        out = torch.empty(host.shape, dtype=dtype, device=device)
    elif out.device != device or out.dtype != dtype or out.numel() != host.size or not out.is_contiguous():
        raise ValueError(f"out must be a contiguous {dtype} tensor of {host.size} elements on {device}")
    if host.nbytes == 0:
        return out
    if host.nbytes > _lib.UPLOAD_MAX_BYTES:
        raise ValueError(f"upload of {host.nbytes} bytes exceeds {_lib.UPLOAD_MAX_BYTES}")
    if stream is not None and not isinstance(stream, torch.cuda.Stream):
        raise TypeError("stream must be a torch.cuda.Stream")
    with _rings_lock:
        ring = _rings.get(index)
        if ring is None:
            ring = _rings[index] = _PinnedRing()
        buf, slot = ring.stage(host)
        s = torch.cuda.current_stream(device) if stream is None else stream
        check(lib().kvx_upload(out.data_ptr(), buf.data_ptr(), host.nbytes, _stream(device, s)), "upload")
        ring.read_by(slot, s)
    return out


# ---------------------------------------------------------------------------
# A serving step around an e4m3 KV cache: rotary positions, the cache write, attention, eviction
#
# Such a cache is a float8_e4m3fn pool [2, L, NB, BS, H, hd] and its scales, a float32 pool [2, L, NB, BS / G, H, 1]:
# one scale for each group of G tokens of a block and each KV head. The operators take a layer's views of both, e.g.
# pool[0, layer], pool[1, layer], scales[0, layer], scales[1, layer]; save_blocks and restore_blocks (FORMAT_RAW) move
# the blocks of either pool.

_DTYPES = {torch.bfloat16: _lib.DTYPE_BF16, torch.float16: _lib.DTYPE_FP16, torch.float32: _lib.DTYPE_FP32}


def rotary_frequencies(rotary_dim: int, base: float = 10000.0, scaling: str | None = None, factor: float = 1.0,
                       original_length: int | None = None, fast: float = 32.0, slow: float = 1.0,
                       device=None) -> tuple[torch.Tensor, float]:
    """(frequencies, magnitude) for rotary_embed: rotary_dim / 2 float64 radians a position, and the outputs' factor.

    Pair i turns by base ** (-2 i / rotary_dim) a position. For contexts `factor` times as long as the trained one:
    - "linear": all positions are divided by `factor`;
    - "base": the base grows so that the slowest pair turns `factor` times slower and the fastest as before;
    - "by_parts": pairs that turn `fast` times or more over original_length positions stay, those that turn `slow`
      times or less are divided by `factor`, those between are blended linearly in their index, and outputs grow by
      0.1 ln(factor) + 1.
    """
    if rotary_dim <= 0 or rotary_dim % 2:
        raise ValueError(f"rotary_dim must be positive and even (got {rotary_dim})")
    if base <= 0 or factor < 1:
        raise ValueError(f"base must be positive and factor at least 1 (got {base} and {factor})")
    device = torch.device("cuda", torch.cuda.current_device()) if device is None else torch.device(device)
    if scaling not in (None, "linear", "base", "by_parts"):
        raise ValueError(f"unknown scaling {scaling!r}")
    if scaling == "base" and rotary_dim > 2:
        base = base * factor ** (rotary_dim / (rotary_dim - 2))
    index = torch.arange(rotary_dim // 2, dtype=torch.float64)
    frequencies = base ** (-2.0 * index / rotary_dim)
    magnitude = 1.0
    if scaling == "linear":
        frequencies = frequencies / factor
    elif scaling == "by_parts":
        if original_length is None or original_length <= 0 or fast <= slow or slow <= 0 or base <= 1:
            raise ValueError("by_parts needs a positive original_length, fast > slow > 0 and base > 1")

        def pair_turning(times: float) -> float:
            return rotary_dim * log(original_length / (times * 2 * pi)) / (2 * log(base))

        low, high = floor(pair_turning(fast)), ceil(pair_turning(slow))
        blend = ((index - low) / max(high - low, 1)).clamp(0.0, 1.0)  # 0: stays, 1: divided
        frequencies = frequencies * (1 - blend) + frequencies / factor * blend
        magnitude = 0.1 * log(factor) + 1.0
    return frequencies.to(device), magnitude


def _heads_of(t: torch.Tensor, name: str) -> tuple[int, int, int]:
    if t.ndim != 3 or (t.numel() and (t.stride(2) != 1 or t.stride(1) != t.shape[2])):
        raise ValueError(f"{name} must be [tokens, heads, head_dim] with packed heads")
    return t.shape


def _made(done, what: str):
    """What the native binding returned in place of outputs it made: those, or the status that kept it from them."""
    if type(done) is int:
        check(done, what)
    return done


def rotary_embed(query: torch.Tensor, key: torch.Tensor, positions: torch.Tensor, frequencies: torch.Tensor,
                 interleaved: bool = False, magnitude: float = 1.0, query_out: torch.Tensor | None = None,
                 key_out: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """Queries and keys rotated by their positions: (query_out, key_out), new tensors unless given.

    query, key: [N, heads, head_dim], bfloat16, float16 or float32, with packed heads (the token stride may differ,
    e.g. views of a fused QKV output). positions: int32 or int64 [N]. frequencies: float64 [rotary_dim / 2], radians
    a position (rotary_frequencies). The first rotary_dim elements of each head are rotated in pairs
    (i, i + rotary_dim / 2), or (2i, 2i + 1) if interleaved, and multiplied by magnitude; the rest is copied. An output
    may be its input (in place) but may not overlap it otherwise. Angles are taken in float64. Capturable.
    """
    done = _bind().rotary(query, key, positions, frequencies, interleaved, magnitude, query_out, key_out)
    if done is not None:
        return _made(done, "rotary_embed")
    n, q_heads, hd = _heads_of(query, "query")
    kn, k_heads, khd = _heads_of(key, "key")
    if kn != n or khd != hd:
        raise ValueError("query and key differ in tokens or head_dim")
    dtype = query.dtype
    if dtype not in _DTYPES:
        raise NotImplementedError(f"rotary_embed takes bfloat16, float16 or float32 tensors, not {dtype}")
    query_out = torch.empty((n, q_heads, hd), dtype=dtype, device=query.device) if query_out is None else query_out
    key_out = torch.empty((n, k_heads, hd), dtype=dtype, device=key.device) if key_out is None else key_out
    if _heads_of(query_out, "query_out") != query.shape or _heads_of(key_out, "key_out") != key.shape:
        raise ValueError("an output's shape differs from its input's")
    if not (key.dtype == query_out.dtype == key_out.dtype == dtype):
        raise TypeError("query, key and their outputs must share one dtype")
    if positions.dtype not in (torch.int32, torch.int64) or not positions.is_contiguous() or positions.shape != (n,):
        raise TypeError("positions must be a contiguous int32 or int64 tensor, one for each token")
    if frequencies.dtype != torch.float64 or not frequencies.is_contiguous() or frequencies.ndim != 1:
        raise TypeError("frequencies must be a contiguous float64 vector")
    device = _require_device(query, key, query_out, key_out, positions, frequencies)
    check(lib().kvx_rotary_embed(query.data_ptr(), query.stride(0), key.data_ptr(), key.stride(0),
                                 query_out.data_ptr(), query_out.stride(0), key_out.data_ptr(), key_out.stride(0),
                                 positions.data_ptr(), positions.element_size(), frequencies.data_ptr(), n, q_heads,
                                 k_heads, hd, 2 * frequencies.numel(), int(interleaved), magnitude, _DTYPES[dtype],
                                 _stream(device)), "rotary_embed")
    return query_out, key_out


def _fp8_cache(k_cache: torch.Tensor, k_scale: torch.Tensor, v_cache: torch.Tensor | None = None,
               v_scale: torch.Tensor | None = None) -> _lib.Fp8Cache:
    """kvx_fp8_cache of a layer's codes [NB, BS, H, hd] and scales [NB, BS / G, H, 1] (v_cache None: keys only)."""
    nb, bs, heads, hd = k_cache.shape if k_cache.ndim == 4 else (0, 0, 0, 0)
    groups = k_scale.shape[1] if k_scale.ndim == 4 else 0
    for cache, scale in ((k_cache, k_scale), (v_cache, v_scale)):
        if cache is None:
            continue
        if cache.dtype != torch.float8_e4m3fn or cache.shape != (nb, bs, heads, hd) or not cache.is_contiguous():
            raise ValueError("k_cache and v_cache must be equally sized contiguous float8_e4m3fn "
                             "[blocks, block_size, heads, head_dim] tensors")
        if scale.dtype != torch.float32 or scale.shape != (nb, groups, heads, 1) or not scale.is_contiguous():
            raise ValueError("scales must be contiguous float32 [blocks, groups, heads, 1] tensors")
    if groups <= 0 or bs % groups:
        raise ValueError(f"{groups} groups do not divide blocks of {bs} tokens")
    return _lib.Fp8Cache(k_cache.data_ptr(), 0 if v_cache is None else v_cache.data_ptr(), k_scale.data_ptr(),
                         0 if v_scale is None else v_scale.data_ptr(), nb, bs, bs // groups, heads, hd)


def _paged_batch(block_tables: torch.Tensor, context_lens: torch.Tensor, cu_seqlens: torch.Tensor | None = None,
                 max_seqlen: int | None = None, num_tokens: int = 0) -> _lib.PagedBatch:
    if block_tables.dtype != torch.int32 or block_tables.ndim != 2 or \
            (block_tables.numel() and block_tables.stride(1) != 1 and block_tables.shape[1] > 1):
        raise TypeError("block_tables must be an int32 [sequences, blocks] tensor with contiguous rows")
    seqs, width = block_tables.shape
    if max(seqs, width, num_tokens) > _INT32_MAX:
        raise NotImplementedError("more than 2^31 sequences, blocks or query rows in one call")
    if context_lens.dtype != torch.int32 or context_lens.shape != (seqs,) or not context_lens.is_contiguous():
        raise TypeError("context_lens must be a contiguous int32 tensor, one for each sequence")
    if cu_seqlens is not None:
        if cu_seqlens.dtype != torch.int32 or cu_seqlens.shape != (seqs + 1,) or not cu_seqlens.is_contiguous():
            raise TypeError("cu_seqlens must be a contiguous int32 tensor of sequences + 1")
        max_seqlen = num_tokens if max_seqlen is None else min(max_seqlen, num_tokens)
    else:
        if max_seqlen not in (None, 1):
            raise ValueError("without cu_seqlens each sequence has one query row: max_seqlen is 1")
        max_seqlen = min(1, num_tokens)
    return _lib.PagedBatch(block_tables.data_ptr(), context_lens.data_ptr(),
                           0 if cu_seqlens is None else cu_seqlens.data_ptr(), block_tables.stride(0), width, seqs,
                           max_seqlen, num_tokens)


def _present(*tensors):
    return [t for t in tensors if t is not None]


def store_kvcache_fp8(key: torch.Tensor, value: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                      k_scale: torch.Tensor, v_scale: torch.Tensor, slot_mapping: torch.Tensor):
    """store_kvcache into an e4m3 cache with one scale for each (group of tokens, KV head).

    key/value: [N, num_heads, head_dim], bfloat16, float16 or float32, packed heads, rows on 16 bytes (the token
    stride may differ). k_cache/v_cache: contiguous float8_e4m3fn [blocks, block_size, num_heads, head_dim] layer
    views, k_scale/v_scale: contiguous float32 [blocks, groups, num_heads, 1]; a group is block_size / groups tokens, a
    multiple of 16. slot_mapping: int32 [N], -1 and slots outside the cache skip a token; the tokens of one group
    stand together in it, as those of a sequence do, with none of another group between them.

    A group's scale becomes the least power of two s with |x| <= 448 s for what the call writes there (s >= 2^-100;
    infinities saturate, NaN stays NaN). A call that does not write a group's first slot continues it: the scale is
    the larger of the old and the new one, and rows already there are encoded anew where it grew. One that does starts
    the group over, whatever it held. Capturable in a HIP graph.
    """
    rc = _bind().store_fp8(key, value, k_cache, v_cache, k_scale, v_scale, slot_mapping)
    if rc is not None:
        if rc:
            check(rc, "store_kvcache_fp8")
        return
    n, heads, hd = _heads_of(key, "key")
    if _heads_of(value, "value") != key.shape:
        raise ValueError("key and value shapes differ")
    if key.dtype not in _DTYPES:
        raise NotImplementedError(f"store_kvcache_fp8 takes bfloat16, float16 or float32 rows, not {key.dtype}")
    if value.dtype != key.dtype:
        raise TypeError("key and value must share one dtype")
    cache = _fp8_cache(k_cache, k_scale, v_cache, v_scale)
    if (cache.num_heads, cache.head_dim) != (heads, hd):
        raise ValueError("rows and cache differ in heads or head_dim")
    if slot_mapping.dtype != torch.int32 or slot_mapping.shape != (n,) or not slot_mapping.is_contiguous():
        raise TypeError("slot_mapping must be a contiguous int32 tensor, one for each token")
    device = _require_device(k_cache, key, value, v_cache, k_scale, v_scale, slot_mapping)
    check(lib().kvx_store_kvcache_fp8(ctypes.byref(cache), key.data_ptr(), key.stride(0), value.data_ptr(),
                                      value.stride(0), _DTYPES[key.dtype], slot_mapping.data_ptr(), n,
                                      _stream(device)), "store_kvcache_fp8")


def _check_queries(query: torch.Tensor, cache: _lib.Fp8Cache):
    n, heads, hd = _heads_of(query, "query")
    if query.dtype not in (torch.bfloat16, torch.float16):
        raise NotImplementedError(f"queries of an e4m3 cache are bfloat16 or float16, not {query.dtype}")
    if hd != cache.head_dim or heads % max(1, cache.num_heads):
        raise ValueError("query heads must be a multiple of the cache's, with its head_dim")
    return n, heads, hd


def attention_fp8(query: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, k_scale: torch.Tensor,
                  v_scale: torch.Tensor, block_tables: torch.Tensor, context_lens: torch.Tensor,
                  softmax_scale: float | None = None, cu_seqlens: torch.Tensor | None = None,
                  max_seqlen: int | None = None, out: torch.Tensor | None = None, return_lse: bool = False):
    """Causal attention of each sequence's last tokens over its e4m3 cache: out, or (out, lse) with return_lse.

    query: [N, q_heads, head_dim], bfloat16 or float16, packed heads, rows on 16 bytes; q_heads a multiple of the
    cache's heads (grouped heads). Caches and scales as store_kvcache_fp8's, which has written this call's tokens
    already. block_tables: int32 [B, width]; context_lens: int32 [B], all cached tokens of a sequence; entries past
    a sequence's blocks are not read, ids outside the pool count as blocks without tokens.

    Decode: N == B, row b is sequence b's newest token. Chunks: cu_seqlens, int32 [B + 1], row range of each sequence
    (row i of n sees the tokens up to context - n + i) and max_seqlen, the most rows of one: a hint that sizes the
    launch and changes no result by more than its rounding. It defaults to N, which costs time where many sequences
    have few rows each (64 of 3 rows over 4,096 tokens of 8 heads: 310 us, with the hint 130); the width of
    block_tables sizes the launch likewise (one row over 2,048 tokens of 8 heads: 10 us, in tables of 131,072 tokens
    24). Rows of no sequence are left as they are; rows that see no token become 0. out: contiguous
    [N, q_heads, head_dim] of the query's type; lse: float32 [N, q_heads], log of the sum of exp(scores), -inf for
    rows that see no token. softmax_scale, positive, defaults to head_dim ** -0.5. Capturable in a HIP graph.
    """
    done = _bind().attention(query, k_cache, v_cache, k_scale, v_scale, block_tables, context_lens, softmax_scale,
                             cu_seqlens, max_seqlen, out, return_lse)
    if done is not None:
        return _made(done, "attention_fp8")
    cache = _fp8_cache(k_cache, k_scale, v_cache, v_scale)
    n, heads, hd = _check_queries(query, cache)
    batch = _paged_batch(block_tables, context_lens, cu_seqlens, max_seqlen, n)
    if out is None:
        out = torch.empty((n, heads, hd), dtype=query.dtype, device=query.device)
    elif out.shape != query.shape or out.dtype != query.dtype or not out.is_contiguous():
        raise ValueError("out must be a contiguous tensor of the query's shape and dtype")
    device = _require_device(k_cache, query, out, v_cache, k_scale, v_scale, block_tables, context_lens,
                             *_present(cu_seqlens))
    lse = torch.empty((n, heads), dtype=torch.float32, device=device) if return_lse else None
    need = ctypes.c_int64()
    check(lib().kvx_attention_fp8_workspace(ctypes.byref(cache), ctypes.byref(batch), heads, ctypes.byref(need)),
          "attention_fp8")
    workspace = torch.empty(need.value, dtype=torch.uint8, device=device) if need.value else None
    check(lib().kvx_attention_fp8(ctypes.byref(cache), ctypes.byref(batch), query.data_ptr(), query.stride(0), heads,
                                  _DTYPES[query.dtype], hd ** -0.5 if softmax_scale is None else softmax_scale,
                                  out.data_ptr(), None if lse is None else lse.data_ptr(),
                                  None if workspace is None else workspace.data_ptr(), need.value, _stream(device)),
          "attention_fp8")
    return (out, lse) if return_lse else out


def attention_weights_fp8(query: torch.Tensor, lse: torch.Tensor, k_cache: torch.Tensor, k_scale: torch.Tensor,
                          block_tables: torch.Tensor, context_lens: torch.Tensor, softmax_scale: float | None = None,
                          cu_seqlens: torch.Tensor | None = None, max_seqlen: int | None = None,
                          weights: torch.Tensor | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """Adds up the attention that each cached token received from a call of attention_fp8: what eviction goes by.

    out[b, h, t] = weights[b, h, t] + the sum of the softmax weights of token t over sequence b's rows and the query
    heads of KV head h. Arguments as attention_fp8's, with the lse that it returned. weights: contiguous float32
    [B, heads, width] (None: zeros, with width the tables' tokens); out: likewise, may be weights itself; default
    weights, in place, or a new tensor where weights is None. Tokens at or past width are dropped, and entries past a
    sequence's context keep their weights. Deterministic. Capturable in a HIP graph.
    """
    into = weights if out is None else out
    if into is not None:
        rc = _bind().attention_weights(query, lse, k_cache, k_scale, block_tables, context_lens, softmax_scale,
                                       cu_seqlens, max_seqlen, weights, into)
        if rc is not None:
            if rc:
                check(rc, "attention_weights_fp8")
            return into
    cache = _fp8_cache(k_cache, k_scale)
    n, heads, hd = _check_queries(query, cache)
    batch = _paged_batch(block_tables, context_lens, cu_seqlens, max_seqlen, n)
    if lse.dtype != torch.float32 or lse.shape != (n, heads) or not lse.is_contiguous():
        raise TypeError("lse must be a contiguous float32 [tokens, q_heads] tensor")
    if out is None:
        out = weights if weights is not None else torch.empty(
            (batch.num_seqs, cache.num_heads, batch.table_width * cache.block_size), dtype=torch.float32,
            device=query.device)
    for t in _present(weights, out):
        if t.dtype != torch.float32 or t.ndim != 3 or t.shape[:2] != (batch.num_seqs, cache.num_heads) or \
                t.shape != out.shape or not t.is_contiguous():
            raise ValueError("weights and out must be contiguous float32 [sequences, heads, width] tensors")
    device = _require_device(k_cache, query, lse, k_scale, block_tables, context_lens,
                             *_present(cu_seqlens, weights, out))
    check(lib().kvx_attention_weights_fp8(ctypes.byref(cache), ctypes.byref(batch), query.data_ptr(), query.stride(0),
                                          heads, _DTYPES[query.dtype],
                                          hd ** -0.5 if softmax_scale is None else softmax_scale, lse.data_ptr(),
                                          None if weights is None else weights.data_ptr(), out.data_ptr(),
                                          out.shape[2], _stream(device)), "attention_weights_fp8")
    return out


def select_tokens(weights: torch.Tensor, context_lens: torch.Tensor, keep: int,
                  recent: int = 0) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """The tokens of each (sequence, KV head) to keep, by their accumulated weight: (indices, counts, kept).

    weights: contiguous float32 [B, heads, width]; context_lens: int32 [B] (lengths beyond width count as width). A
    context of at most `keep` tokens is kept whole. Of a longer one, the last `recent` (at most keep) are kept and, of
    the others, the keep - recent with the largest weights: of equal ones the earliest, NaN below all. indices: int32
    [B, heads, keep], ascending, then -1; counts: int32 [B], the kept tokens of each sequence (its context_lens after
    compact_kvcache_fp8); kept: float32 [B, heads, keep], their weights, then 0. Capturable in a HIP graph.
    """
    done = _bind().select(weights, context_lens, keep, recent)
    if done is not None:
        return _made(done, "select_tokens")
    if weights.dtype != torch.float32 or weights.ndim != 3 or not weights.is_contiguous():
        raise TypeError("weights must be a contiguous float32 [sequences, heads, width] tensor")
    seqs, heads, width = weights.shape
    if context_lens.dtype != torch.int32 or context_lens.shape != (seqs,) or not context_lens.is_contiguous():
        raise TypeError("context_lens must be a contiguous int32 tensor, one for each sequence")
    if keep < 0 or recent < 0 or heads == 0:
        raise ValueError("keep and recent must be non-negative, and heads at least 1")
    if keep > _INT32_MAX:
        raise NotImplementedError(f"select_tokens keeps at most {_INT32_MAX} tokens (got {keep})")
    recent = min(recent, keep)
    device = _require_device(weights, context_lens)
    indices = torch.empty((seqs, heads, keep), dtype=torch.int32, device=device)
    counts = torch.empty((seqs,), dtype=torch.int32, device=device)
    kept = torch.empty((seqs, heads, keep), dtype=torch.float32, device=device)
    check(lib().kvx_select_tokens(weights.data_ptr(), context_lens.data_ptr(), seqs, heads, width, keep, recent,
                                  indices.data_ptr(), counts.data_ptr(), kept.data_ptr(), _stream(device)),
          "select_tokens")
    return indices, counts, kept


def compact_kvcache_fp8(k_cache: torch.Tensor, v_cache: torch.Tensor, k_scale: torch.Tensor, v_scale: torch.Tensor,
                        block_tables: torch.Tensor, indices: torch.Tensor, counts: torch.Tensor,
                        new_block_tables: torch.Tensor, context_lens: torch.Tensor | None = None):
    """Moves the kept tokens of each KV head to the front of other blocks: position j of sequence b in the blocks
    new_block_tables[b] becomes its token indices[b, h, j] in the blocks block_tables[b], for j < counts[b].

    Caches, scales and tables as store_kvcache_fp8's and attention_fp8's; indices and counts as select_tokens gives
    them (an index that is no token of the sequence gives zeros). New blocks may be no block that a table of the call
    names as a source, nor be named twice: shared prefixes stay as they are for their other users. Each group written
    gets the scale that store_kvcache_fp8 would give its values. context_lens: int32 [B], where indices may reach past
    a sequence (default: the tables' tokens). Capturable in a HIP graph.
    """
    rc = _bind().compact(k_cache, v_cache, k_scale, v_scale, block_tables, indices, counts, new_block_tables, context_lens)
    if rc is not None:
        if rc:
            check(rc, "compact_kvcache_fp8")
        return
    cache = _fp8_cache(k_cache, k_scale, v_cache, v_scale)
    seqs = block_tables.shape[0] if block_tables.ndim == 2 else 0
    if indices.dtype != torch.int32 or indices.ndim != 3 or indices.shape[:2] != (seqs, cache.num_heads) or \
            not indices.is_contiguous():
        raise TypeError("indices must be a contiguous int32 [sequences, heads, keep] tensor")
    if new_block_tables.ndim != 2 or new_block_tables.shape[0] != seqs:
        raise ValueError("new_block_tables must have a row for each sequence")
    lens = counts if context_lens is None else context_lens
    batch = _paged_batch(block_tables, lens)
    new = _paged_batch(new_block_tables, counts)
    if context_lens is None:
        batch.context_lens = None
    device = _require_device(k_cache, v_cache, k_scale, v_scale, block_tables, indices, counts, new_block_tables, lens)
    check(lib().kvx_compact_kvcache_fp8(ctypes.byref(cache), ctypes.byref(batch), indices.data_ptr(),
                                        counts.data_ptr(), indices.shape[2], new_block_tables.data_ptr(),
                                        new.table_stride, new.table_width, _stream(device)), "compact_kvcache_fp8")


# ---------------------------------------------------------------------------
# Test hooks

def sleep(microseconds: int, stream=None, device=None):
    """Queues a bounded busy wait on `stream` (torch's current stream by default)."""
    device = torch.device("cuda", torch.cuda.current_device()) if device is None else torch.device(device)
    check(lib().kvx_sleep(_stream(device, stream), int(microseconds)), "sleep")


SELFTEST_FIELDS = ("e4m3_encode_mismatch", "bf16_round_mismatch", "nan_not_preserved", "division_mismatch",
                   "e4m3_decode_mismatch", "encode_inputs_2p20", "division_pairs_2p20", "decode_sweeps")


def selftest(device=None) -> dict[str, int]:
    """Runs libkvx's exhaustive device self-test; returns its counters by name."""
    device = torch.device("cuda", torch.cuda.current_device()) if device is None else torch.device(device)
    counters = torch.zeros(8, dtype=torch.int64, device=device)
    check(lib().kvx_selftest(counters.data_ptr(), _stream(device)), "selftest")
    return dict(zip(SELFTEST_FIELDS, counters.cpu().tolist()))


# ---------------------------------------------------------------------------
# Token-granular copies (KV handoff)

def _plane_range(pool: torch.Tensor, layout: BlockLayout, planes) -> tuple[int, BlockLayout, tuple]:
    """(pool address, layout, leading dense dims) of the pool's (K/V, layer) planes [first, end).

    Plane p is K/V half p // L, layer p % L; None means all 2L planes, whose
    dense buffers keep the [2, L, ...] shape. A plane range is the same
    layout with fewer planes, starting at the first one's address.
    """
    if planes is None:
        return pool.data_ptr(), layout, (2, pool.shape[1])
    first, end = planes
    if not 0 <= first < end <= layout.planes:
        raise ValueError(f"plane range [{first}, {end}) is not within the pool's {layout.planes} planes")
    sub = BlockLayout(*(getattr(layout, name) for name, _ in BlockLayout._fields_))
    sub.planes = end - first
    return pool.data_ptr() + first * layout.plane_stride * layout.elem_bytes, sub, (end - first,)


def _token_copy(gather: bool, pool: torch.Tensor, block_table, num_tokens: int, dense: torch.Tensor, stream=None,
                planes=None):
    if pool.ndim != 6:
        raise ValueError("pool must be [2, layers, blocks, block_size, heads, head_dim]")
    address, layout, lead = _plane_range(pool, pool_layout(pool), planes)
    expected = (*lead, num_tokens, *pool.shape[-2:])
    if tuple(dense.shape) != expected or dense.dtype != pool.dtype or not dense.is_contiguous():
        raise ValueError(f"dense buffer must be a contiguous {pool.dtype} tensor of shape {expected}")
    if dense.device.type == "cuda":
        _require_device(pool, dense)
    elif not dense.is_pinned():
        raise ValueError("a host buffer must be pinned (device-accessible)")
    device = _require_device(pool)
    table = list(block_table)
    fn = lib().kvx_gather_tokens if gather else lib().kvx_scatter_tokens
    check(fn(address, ctypes.byref(layout), int32_array(table), len(table), num_tokens * pool.shape[4],
             dense.data_ptr(), _stream(device, stream)),
          "gather_tokens" if gather else "scatter_tokens")


def gather_tokens(pool: torch.Tensor, block_table, num_tokens: int, out: torch.Tensor, stream=None, planes=None):
    """out[:, :, t] = pool[:, :, block_table[t // BS], t % BS] for t < num_tokens.

    `out` is [2, L, num_tokens, H, hd] (kv_handoff.py:46-55's packed payload),
    on the pool's device or in pinned host memory. With planes=(first, end),
    only those (K/V, layer) planes (plane p = K/V p // L, layer p % L) are
    copied, into an `out` of shape [end - first, num_tokens, H, hd].
    """
    _token_copy(True, pool, block_table, num_tokens, out, stream, planes)


def scatter_tokens(pool: torch.Tensor, block_table, num_tokens: int, src: torch.Tensor, stream=None, planes=None):
    """pool[:, :, block_table[t // BS], t % BS] = src[:, :, t] for t < num_tokens (kv_handoff.py:112-118).

    planes=(first, end) as for gather_tokens."""
    _token_copy(False, pool, block_table, num_tokens, src, stream, planes)


def _token_fp8(gather: bool, pool: torch.Tensor, block_table, num_tokens: int, payload: torch.Tensor,
               scale: torch.Tensor, stream=None, planes=None):
    if pool.ndim != 6 or pool.dtype != torch.bfloat16:
        raise ValueError("pool must be a bfloat16 [2, layers, blocks, block_size, heads, head_dim] tensor")
    if scale.dtype not in SCALE_DTYPES:
        raise ValueError("scale must be a bfloat16 or float32 tensor")
    address, layout, lead = _plane_range(pool, pool_layout(pool, scale.dtype), planes)
    shape = (*lead, num_tokens, *pool.shape[-2:])
    if tuple(payload.shape) != shape or payload.dtype != torch.float8_e4m3fn or not payload.is_contiguous():
        raise ValueError(f"payload must be a contiguous float8_e4m3fn tensor of shape {shape}")
    if (tuple(scale.shape) != (*shape[:-1], 1) or scale.dtype not in SCALE_DTYPES
            or not scale.is_contiguous()):
        raise ValueError(f"scale must be a contiguous bfloat16/float32 tensor of shape {(*shape[:-1], 1)}")
    for t in (payload, scale):
        if t.device.type == "cuda":
            _require_device(pool, t)
        elif not (gather and t.is_pinned()):
            raise ValueError("an FP8 gather may write pinned host memory; a scatter reads device memory")
    device = _require_device(pool)
    table = list(block_table)
    fn = lib().kvx_gather_tokens_fp8 if gather else lib().kvx_scatter_tokens_fp8
    check(fn(address, ctypes.byref(layout), int32_array(table), len(table), num_tokens * pool.shape[4],
             payload.data_ptr(), scale.data_ptr(), _stream(device, stream)),
          "gather_tokens_fp8" if gather else "scatter_tokens_fp8")


def gather_tokens_fp8(pool: torch.Tensor, block_table, num_tokens: int, payload: torch.Tensor, scale: torch.Tensor,
                      stream=None, planes=None):
    """fp8_quantize of gather_tokens' [2, L, num_tokens, H, hd] payload, without the BF16 intermediate.

    payload: float8_e4m3fn [2, L, num_tokens, H, hd]; scale: [2, L, num_tokens, H, 1] in bfloat16 or float32,
    both on the pool's device or in pinned host memory. planes=(first, end) as for gather_tokens: payload
    [end - first, num_tokens, H, hd] and scale [end - first, num_tokens, H, 1].
    """
    _token_fp8(True, pool, block_table, num_tokens, payload, scale, stream, planes)


def scatter_tokens_fp8(pool: torch.Tensor, block_table, num_tokens: int, payload: torch.Tensor, scale: torch.Tensor,
                       stream=None, planes=None):
    """pool[:, :, block_table[t // BS], t % BS] = fp8_dequantize(payload, scale)[:, :, t] (device tensors).

    planes=(first, end) as for gather_tokens_fp8."""
    _token_fp8(False, pool, block_table, num_tokens, payload, scale, stream, planes)
