// Kernels that stream, for the operators around an e4m3 KV cache: rotary
// positions, the cache write, the choice of tokens to keep, and compaction.
// Bound by HBM bandwidth, or at a decode step's sizes by latency.
#include "kvx_step.h"

namespace kvx {
namespace {

constexpr int kThreads = 256;

// ---------------------------------------------------------------------------
// Elements as fp32: eight of them are one or two 16-byte pieces.

template <int kType>
struct Elem;
template <>
struct Elem<KVX_DTYPE_BF16> {
  using T = __bf16;
};
template <>
struct Elem<KVX_DTYPE_FP16> {
  using T = _Float16;
};
template <>
struct Elem<KVX_DTYPE_FP32> {
  using T = float;
};

template <typename T>
struct alignas(16) Piece {  // 16 bytes
  static constexpr int kCount = 16 / sizeof(T);
  T x[kCount];
};

// ---------------------------------------------------------------------------
// Rotary positions: (a, b) -> (a cos - b sin, b cos + a sin) * magnitude with
// the angle position * frequency, on pairs (i, i + rotary_dim / 2) or
// (2i, 2i + 1) of the head's first rotary_dim elements.
//
// The angle is taken in fp64 and reduced to a fraction of a turn there, so that
// positions of millions keep fp32's precision; one workgroup computes a token's
// rotary_dim / 2 sines and cosines once, into LDS, and applies them to all its
// heads. A table of them would be read for every token, and end at some position.

template <typename T, int kVec>
__device__ __forceinline__ void load_vec(const T* p, float* out) {
  if constexpr (kVec * sizeof(T) >= 16) {
    constexpr int kPer = Piece<T>::kCount;
#pragma unroll
    for (int i = 0; i < kVec / kPer; ++i) {
      const Piece<T> piece = reinterpret_cast<const Piece<T>*>(p)[i];
#pragma unroll
      for (int j = 0; j < kPer; ++j) out[i * kPer + j] = (float)piece.x[j];
    }
  } else {
#pragma unroll
    for (int i = 0; i < kVec; ++i) out[i] = (float)p[i];
  }
}
template <typename T, int kVec>
__device__ __forceinline__ void store_vec(T* p, const float* in) {
  if constexpr (kVec * sizeof(T) >= 16) {
    constexpr int kPer = Piece<T>::kCount;
#pragma unroll
    for (int i = 0; i < kVec / kPer; ++i) {
      Piece<T> piece;
#pragma unroll
      for (int j = 0; j < kPer; ++j) piece.x[j] = (T)in[i * kPer + j];
      reinterpret_cast<Piece<T>*>(p)[i] = piece;
    }
  } else {
#pragma unroll
    for (int i = 0; i < kVec; ++i) p[i] = (T)in[i];
  }
}

// kVec elements of each half (or 2 * kVec adjacent ones) a thread and step.
template <typename T, int kVec, bool kInterleaved>
__global__ __launch_bounds__(kThreads) void rotary_kernel(RotaryArgs a) {
  extern __shared__ float2 turns[];  // (cos, sin) * magnitude
  const int64_t token = blockIdx.x;
  const int pairs = a.rotary_dim / 2;
  const int64_t position = a.long_positions ? reinterpret_cast<const int64_t*>(a.positions)[token]
                                            : reinterpret_cast<const int32_t*>(a.positions)[token];
  for (int i = threadIdx.x; i < pairs; i += kThreads) {
    const double angle = (double)position * a.frequencies[i] * 0.15915494309189533577;  // in turns
    const float rest = (float)(angle - rint(angle));
    float s, c;
    sincospif(2.0f * rest, &s, &c);
    turns[i] = make_float2(c * a.magnitude, s * a.magnitude);
  }
  __syncthreads();
  const int heads = a.q_heads + a.k_heads;
  const int per_head = pairs / kVec;
  for (int i = threadIdx.x; i < heads * per_head; i += kThreads) {
    const int head = i / per_head, at = (i - head * per_head) * kVec;
    const bool is_key = head >= a.q_heads;
    const int h = is_key ? head - a.q_heads : head;
    const T* x = (is_key ? (const T*)a.key + token * a.k_stride : (const T*)a.query + token * a.q_stride) +
                 (int64_t)h * a.head_dim;
    T* y = (is_key ? (T*)a.key_out + token * a.k_out_stride : (T*)a.query_out + token * a.q_out_stride) +
           (int64_t)h * a.head_dim;
    float u[2 * kVec], w[2 * kVec];
    if (kInterleaved) {
      load_vec<T, 2 * kVec>(x + 2 * at, u);
    } else {
      load_vec<T, kVec>(x + at, u);
      load_vec<T, kVec>(x + at + pairs, u + kVec);
    }
#pragma unroll
    for (int j = 0; j < kVec; ++j) {
      const float2 t = turns[at + j];
      const int first = kInterleaved ? 2 * j : j, second = kInterleaved ? 2 * j + 1 : kVec + j;
      w[first] = u[first] * t.x - u[second] * t.y;
      w[second] = u[second] * t.x + u[first] * t.y;
    }
    if (kInterleaved) {
      store_vec<T, 2 * kVec>(y + 2 * at, w);
    } else {
      store_vec<T, kVec>(y + at, w);
      store_vec<T, kVec>(y + at + pairs, w + kVec);
    }
  }
  // The rest of each head is copied, unless the call is in place.
  const int rest = a.head_dim - a.rotary_dim;
  if (rest == 0) return;
  const bool q_moves = a.query != a.query_out, k_moves = a.key != a.key_out;
  if (!q_moves && !k_moves) return;
  const int vecs = rest / kVec;  // kVec divides it (launch_rotary)
  for (int i = threadIdx.x; i < heads * vecs; i += kThreads) {
    const int head = i / vecs, at = a.rotary_dim + (i - head * vecs) * kVec;
    const bool is_key = head >= a.q_heads;
    if (!(is_key ? k_moves : q_moves)) continue;
    const int64_t h = is_key ? head - a.q_heads : head;
    const T* x = is_key ? (const T*)a.key + token * a.k_stride : (const T*)a.query + token * a.q_stride;
    T* y = is_key ? (T*)a.key_out + token * a.k_out_stride : (T*)a.query_out + token * a.q_out_stride;
    x += h * a.head_dim + at;
    y += h * a.head_dim + at;
    if constexpr (kVec * sizeof(T) >= 16) {
#pragma unroll
      for (int j = 0; j < (int)(kVec * sizeof(T) / 16); ++j)
        reinterpret_cast<u32x4*>(y)[j] = reinterpret_cast<const u32x4*>(x)[j];
    } else {
#pragma unroll
      for (int j = 0; j < kVec; ++j) y[j] = x[j];
    }
  }
}

// ---------------------------------------------------------------------------
// The cache write. A workgroup holds the tokens of one group that stand
// together in the call, for one head of K or V: their largest magnitude gives
// the group's scale, under which their rows are encoded. A group that the call
// enters behind its first slot keeps its rows and the larger of both scales;
// where that grew, the rows that the call does not write are encoded anew.

template <typename T>
__global__ __launch_bounds__(kThreads) void store_fp8_kernel(Fp8Cache c, const T* __restrict__ key, int64_t key_stride,
                                                             const T* __restrict__ value, int64_t value_stride,
                                                             const int32_t* __restrict__ slots, int32_t num_tokens) {
  __shared__ int owner[kMaxGroup];  // the call's token for each of the group's rows; the last one that names it
  __shared__ int run_end;
  __shared__ float wave_amax[kThreads / kWave];
  const int token0 = blockIdx.x;
  const int head = blockIdx.y % c.heads;
  const bool is_v = blockIdx.y >= c.heads;
  const int64_t cache_slots = (int64_t)c.num_blocks * c.block_size;
  const int slot0 = slots[token0];
  if (slot0 < 0 || slot0 >= cache_slots) return;
  const int group = c.group_of(slot0);
  if (token0 > 0) {
    const int before = slots[token0 - 1];
    if (before >= 0 && c.group_of(before) == group) return;  // the group's run began earlier
  }
  for (int i = threadIdx.x; i < c.group; i += kThreads) owner[i] = -1;
  if (threadIdx.x == 0) run_end = num_tokens;
  __syncthreads();
  const int slot_base = group * c.group;
  for (int at = token0;; at += kThreads) {
    const int i = at + threadIdx.x;
    if (i < num_tokens) {
      const int s = slots[i];
      if (s < slot_base || s - slot_base >= c.group) atomicMin(&run_end, i);
    }
    __syncthreads();
    const int end = run_end;
    __syncthreads();
    if (i < end && i < num_tokens) atomicMax(&owner[slots[i] - slot_base], i);
    if (end < at + kThreads || at + kThreads >= num_tokens) break;
  }
  __syncthreads();

  const T* src = (is_v ? value : key) + (int64_t)head * c.head_dim;
  const int64_t src_stride = is_v ? value_stride : key_stride;
  uint8_t* codes = (is_v ? c.v : c.k) + ((int64_t)slot_base * c.heads + head) * c.head_dim;
  const int64_t row_bytes = (int64_t)c.heads * c.head_dim;
  float* scale = (is_v ? c.v_scale : c.k_scale) + (int64_t)group * c.heads + head;
  const int pieces = c.head_dim / 8;  // a thread's step: 8 elements of a row
  float amax = 0.0f;
  for (int i = threadIdx.x; i < c.group * pieces; i += kThreads) {
    const int row = i / pieces, at = (i - row * pieces) * 8, token = owner[row];
    if (token < 0) continue;
    float x[8];
    load_vec<T, 8>(src + token * src_stride + at, x);
#pragma unroll
    for (int j = 0; j < 8; ++j) amax = fmaxf(amax, finite_abs(x[j]));
  }
  amax = wave_max(amax);
  if (threadIdx.x % kWave == 0) wave_amax[threadIdx.x / kWave] = amax;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kThreads / kWave; ++i) amax = fmaxf(amax, wave_amax[i]);
  float held = 0.0f;
  if (owner[0] < 0) {
    const float before = *scale;
    if (before > 0.0f && before < INFINITY) held = before;
  }
  const float fit = fmaxf(scale_for(amax), held);
  const float inverse = 1.0f / fit;
  const bool grew = held > 0.0f && fit > held;
  const float shrink = held / fit;
  __syncthreads();  // every thread has read the scale
  if (threadIdx.x == 0) *scale = fit;
  for (int i = threadIdx.x; i < c.group * pieces; i += kThreads) {
    const int row = i / pieces, at = (i - row * pieces) * 8, token = owner[row];
    uint8_t* dst = codes + row * row_bytes + at;
    u32x2 out;
    if (token >= 0) {
      float x[8];
      load_vec<T, 8>(src + token * src_stride + at, x);
#pragma unroll
      for (int j = 0; j < 8; ++j) x[j] *= inverse;
      out.x = encode4(x[0], x[1], x[2], x[3]);
      out.y = encode4(x[4], x[5], x[6], x[7]);
    } else if (grew) {
      const u32x2 old = *reinterpret_cast<const u32x2*>(dst);
      float x[8];
      decode4(old.x, x);
      decode4(old.y, x + 4);
#pragma unroll
      for (int j = 0; j < 8; ++j) x[j] *= shrink;
      out.x = encode4(x[0], x[1], x[2], x[3]);
      out.y = encode4(x[4], x[5], x[6], x[7]);
    } else {
      continue;
    }
    *reinterpret_cast<u32x2*>(dst) = out;
  }
}

// ---------------------------------------------------------------------------
// The tokens to keep: for one (sequence, KV head), the last `recent` and the
// (keep - recent) of the earlier ones with the largest weight. A radix select
// finds the smallest weight that is kept, 8 bits of its ordered pattern a
// pass; the kept tokens are then written in order of their position, equal
// weights by the lowest.

constexpr int kSelectThreads = 1024;
constexpr int kSelectWaves = kSelectThreads / kWave;

// Orders as the weights do: -0 as +0, NaN below everything.
__device__ __forceinline__ uint32_t rank_of(float w) {
  if (w != w) return 0;
  const uint32_t u = w == 0.0f ? 0 : __float_as_uint(w);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

__global__ __launch_bounds__(kSelectThreads) void select_kernel(const float* __restrict__ weights, int32_t heads,
                                                                int32_t width, const int32_t* __restrict__ lens,
                                                                int32_t keep, int32_t recent,
                                                                int32_t* __restrict__ indices,
                                                                int32_t* __restrict__ counts,
                                                                float* __restrict__ kept) {
  __shared__ uint32_t bins[256];
  __shared__ uint32_t chosen, above;
  __shared__ uint32_t wave_over[kSelectWaves], wave_tied[kSelectWaves];
  const int64_t row = blockIdx.x;
  const int seq = (int)(row / heads), tid = threadIdx.x, wave = tid / kWave, lane = tid % kWave;
  const float* w = weights + row * width;
  int32_t* out = indices + row * keep;
  float* out_w = kept + row * keep;
  int n = lens[seq];
  n = n < 0 ? 0 : n > width ? width : n;
  const int count = n < keep ? n : keep;
  if (tid == 0 && row % heads == 0) counts[seq] = count;
  for (int i = count + tid; i < keep; i += kSelectThreads) {
    out[i] = -1;
    out_w[i] = 0.0f;
  }
  const int last = recent < count ? recent : count;  // kept at the end whatever they weigh
  const int pool = n - last, want = count - last;    // of the first `pool`, `want` are kept
  uint32_t prefix = 0, need = (uint32_t)want;
  if (want > 0 && want < pool) {
    for (int shift = 24; shift >= 0; shift -= 8) {
      if (tid < 256) bins[tid] = 0;
      __syncthreads();
      const uint32_t mask = shift == 24 ? 0 : ~0u << (shift + 8);
      for (int i = tid; i < pool; i += kSelectThreads) {
        const uint32_t r = rank_of(w[i]);
        if ((r & mask) == prefix) atomicAdd(&bins[(r >> shift) & 255], 1u);
      }
      __syncthreads();
      if (wave == 0) {
        // Lane l sums bins 255 - 4 l .. 252 - 4 l; a scan over the lanes finds the bin that holds the need-th largest.
        uint32_t b[4], total = 0;
        for (int j = 0; j < 4; ++j) total += b[j] = bins[255 - (lane * 4 + j)];
        uint32_t before = total;
        for (int d = 1; d < kWave; d <<= 1) {
          const uint32_t other = __shfl_up(before, d);
          if (lane >= d) before += other;
        }
        before -= total;
        if (before < need && need <= before + total) {
          for (int j = 0; j < 4; ++j) {
            if (before < need && need <= before + b[j]) {
              chosen = (uint32_t)(255 - (lane * 4 + j));
              above = before;
            }
            before += b[j];
          }
        }
      }
      __syncthreads();
      prefix |= chosen << shift;
      need -= above;
    }
  }
  // Over the threshold, or tied with it and among the first `need`.
  const bool all = want >= pool;
  uint32_t placed = 0, tied = 0;
  if (want > 0) {
    for (int base = 0; base < pool; base += kSelectThreads) {
      const int i = base + tid;
      const float x = i < pool ? w[i] : 0.0f;
      const uint32_t r = rank_of(x);
      const bool over = i < pool && (all || r > prefix), tie = i < pool && !all && r == prefix;
      const uint64_t over_mask = __ballot(over), tie_mask = __ballot(tie);
      if (lane == 0) {
        wave_over[wave] = __popcll(over_mask);
        wave_tied[wave] = __popcll(tie_mask);
      }
      __syncthreads();
      const uint64_t below = (uint64_t{1} << lane) - 1;
      uint32_t overs = __popcll(over_mask & below), ties = __popcll(tie_mask & below), all_over = 0, all_tied = 0;
      for (int j = 0; j < kSelectWaves; ++j) {
        const uint32_t o = wave_over[j], t = wave_tied[j];
        if (j < wave) {
          overs += o;
          ties += t;
        }
        all_over += o;
        all_tied += t;
      }
      const uint32_t tie_rank = tied + ties;
      if (over || (tie && tie_rank < need)) {
        const uint32_t at = placed + overs + (tie_rank < need ? tie_rank : need) - (tied < need ? tied : need);
        out[at] = i;
        out_w[at] = x;
      }
      const uint32_t taken_before = tied < need ? tied : need;
      tied += all_tied;
      placed += all_over + (tied < need ? tied : need) - taken_before;
      __syncthreads();
    }
  }
  for (int i = tid; i < last; i += kSelectThreads) {
    out[want + i] = pool + i;
    out_w[want + i] = w[pool + i];
  }
}

// ---------------------------------------------------------------------------
// Compaction: a workgroup gathers the rows of one group of the new blocks, for
// one head of K or V, and encodes them under a scale of their own.

__global__ __launch_bounds__(kThreads) void compact_kernel(Fp8Cache c, PagedBatch from,
                                                           const int32_t* __restrict__ indices,
                                                           const int32_t* __restrict__ counts, int32_t keep,
                                                           const int32_t* __restrict__ to_tables, int64_t to_stride,
                                                           int32_t to_width) {
  __shared__ float wave_amax[kThreads / kWave];
  __shared__ int64_t source[kMaxGroup];  // slot of each row, or -1
  const int head = blockIdx.y % c.heads, seq = blockIdx.z;
  const bool is_v = blockIdx.y >= c.heads;
  int count = counts[seq];
  count = count < 0 ? 0 : count > keep ? keep : count;
  const int first = blockIdx.x * c.group;
  if (first >= count) return;
  const int rows = count - first < c.group ? count - first : c.group;
  const int to_block = c.block_of(first);
  if (to_block >= to_width) return;
  const int target = to_tables[seq * to_stride + to_block];
  if (target < 0 || target >= c.num_blocks) return;
  const int64_t to_slot = (int64_t)target * c.block_size + (first - to_block * c.block_size);
  const int32_t* mine = indices + ((int64_t)seq * c.heads + head) * keep + first;
  const int context = context_of(from, seq, c.block_size);
  for (int i = threadIdx.x; i < rows; i += kThreads) {
    const int t = mine[i];
    int64_t slot = -1;
    if (t >= 0 && t < context) {
      const int b = c.block_of(t);
      const int id = from.tables[seq * from.table_stride + b];
      if (id >= 0 && id < c.num_blocks) slot = (int64_t)id * c.block_size + (t - b * c.block_size);
    }
    source[i] = slot;
  }
  __syncthreads();
  uint8_t* codes = is_v ? c.v : c.k;
  float* scales = is_v ? c.v_scale : c.k_scale;
  const int pieces = c.head_dim / 8;
  float amax = 0.0f;
  for (int i = threadIdx.x; i < rows * pieces; i += kThreads) {
    const int row = i / pieces, at = (i - row * pieces) * 8;
    const int64_t slot = source[row];
    if (slot < 0) continue;
    const float s = scales[(slot / c.group) * c.heads + head];
    const u32x2 w = *reinterpret_cast<const u32x2*>(codes + (slot * c.heads + head) * c.head_dim + at);
    float x[8];
    decode4(w.x, x);
    decode4(w.y, x + 4);
#pragma unroll
    for (int j = 0; j < 8; ++j) amax = fmaxf(amax, finite_abs(x[j] * s));
  }
  amax = wave_max(amax);
  if (threadIdx.x % kWave == 0) wave_amax[threadIdx.x / kWave] = amax;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kThreads / kWave; ++i) amax = fmaxf(amax, wave_amax[i]);
  const float fit = scale_for(amax), inverse = 1.0f / fit;
  if (threadIdx.x == 0) scales[(to_slot / c.group) * c.heads + head] = fit;
  for (int i = threadIdx.x; i < rows * pieces; i += kThreads) {
    const int row = i / pieces, at = (i - row * pieces) * 8;
    const int64_t slot = source[row];
    u32x2 out = {0, 0};
    if (slot >= 0) {
      const float s = scales[(slot / c.group) * c.heads + head];
      const u32x2 w = *reinterpret_cast<const u32x2*>(codes + (slot * c.heads + head) * c.head_dim + at);
      float x[8];
      decode4(w.x, x);
      decode4(w.y, x + 4);
#pragma unroll
      for (int j = 0; j < 8; ++j) x[j] = x[j] * s * inverse;
      out.x = encode4(x[0], x[1], x[2], x[3]);
      out.y = encode4(x[4], x[5], x[6], x[7]);
    }
    *reinterpret_cast<u32x2*>(codes + ((to_slot + row) * c.heads + head) * c.head_dim + at) = out;
  }
}

bool aligned16(const void* p) { return (uintptr_t)p % 16 == 0; }

template <typename T>
hipError_t rotary_of(const RotaryArgs& a, hipStream_t stream) {
  constexpr int kPer = 16 / sizeof(T);  // elements of a 16-byte piece
  const int64_t strides[] = {a.q_stride, a.k_stride, a.q_out_stride, a.k_out_stride};
  bool wide = aligned16(a.query) && aligned16(a.query_out) && aligned16(a.key) && aligned16(a.key_out) &&
              a.head_dim % kPer == 0 && a.rotary_dim % (2 * kPer) == 0;
  for (int64_t s : strides) wide = wide && s % kPer == 0;
  const size_t lds = (size_t)a.rotary_dim / 2 * sizeof(float2);
  const dim3 grid((unsigned)a.num_tokens), block(kThreads);
  if (wide && a.interleaved) rotary_kernel<T, kPer, true><<<grid, block, lds, stream>>>(a);
  else if (wide) rotary_kernel<T, kPer, false><<<grid, block, lds, stream>>>(a);
  else if (a.interleaved) rotary_kernel<T, 1, true><<<grid, block, lds, stream>>>(a);
  else rotary_kernel<T, 1, false><<<grid, block, lds, stream>>>(a);
  return hipGetLastError();
}

template <typename T>
hipError_t store_of(const Fp8Cache& c, const void* key, int64_t key_stride, const void* value, int64_t value_stride,
                    const int32_t* slots, int32_t num_tokens, hipStream_t stream) {
  store_fp8_kernel<T><<<dim3((unsigned)num_tokens, (unsigned)(2 * c.heads)), dim3(kThreads), 0, stream>>>(
      c, (const T*)key, key_stride, (const T*)value, value_stride, slots, num_tokens);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_rotary(const RotaryArgs& a, int32_t dtype, hipStream_t stream) {
  if (dtype == KVX_DTYPE_BF16) return rotary_of<__bf16>(a, stream);
  if (dtype == KVX_DTYPE_FP16) return rotary_of<_Float16>(a, stream);
  return rotary_of<float>(a, stream);
}

hipError_t launch_store_fp8(const Fp8Cache& c, const void* key, int64_t key_stride, const void* value,
                            int64_t value_stride, int32_t dtype, const int32_t* slots, int32_t num_tokens,
                            hipStream_t stream) {
  if (dtype == KVX_DTYPE_BF16) return store_of<__bf16>(c, key, key_stride, value, value_stride, slots, num_tokens, stream);
  if (dtype == KVX_DTYPE_FP16)
    return store_of<_Float16>(c, key, key_stride, value, value_stride, slots, num_tokens, stream);
  return store_of<float>(c, key, key_stride, value, value_stride, slots, num_tokens, stream);
}

hipError_t launch_select(const float* weights, int32_t rows, int32_t heads, int32_t width, const int32_t* context_lens,
                         int32_t keep, int32_t recent, int32_t* indices, int32_t* counts, float* kept,
                         hipStream_t stream) {
  select_kernel<<<dim3((unsigned)rows), dim3(kSelectThreads), 0, stream>>>(weights, heads, width, context_lens, keep,
                                                                         recent, indices, counts, kept);
  return hipGetLastError();
}

hipError_t launch_compact(const Fp8Cache& c, const PagedBatch& from, const int32_t* indices, const int32_t* counts,
                          int32_t keep, const int32_t* to_tables, int64_t to_stride, int32_t to_width,
                          hipStream_t stream) {
  const dim3 grid((unsigned)((keep + c.group - 1) / c.group), (unsigned)(2 * c.heads), (unsigned)from.num_seqs);
  compact_kernel<<<grid, dim3(kThreads), 0, stream>>>(c, from, indices, counts, keep, to_tables, to_stride, to_width);
  return hipGetLastError();
}

}  // namespace kvx
