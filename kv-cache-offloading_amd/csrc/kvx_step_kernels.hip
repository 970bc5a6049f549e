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

template <typename T, int kCount>
struct alignas(sizeof(T) * kCount) Piece {  // read and written at once; 16 bytes at most
  T x[kCount];
};
template <typename T, int kVec>
constexpr int kPieceOf = kVec * sizeof(T) > 16 ? 16 / sizeof(T) : kVec;

// ---------------------------------------------------------------------------
// Rotary positions: (a, b) -> (a cos - b sin, b cos + a sin) * magnitude with
// the angle position * frequency, on pairs (i, i + rotary_dim / 2) or
// (2i, 2i + 1) of the head's first rotary_dim elements.
//
// The angle is taken in fp64 and reduced to a fraction of a turn there, so that
// positions of millions keep fp32's precision; one workgroup computes a token's
// rotary_dim / 2 sines and cosines once, into LDS, and applies them to all its
// heads. A table of them would be read for every token, and end at some position.
// Bound by HBM: 16,381 tokens, 335 MB read and written, 62 us or 5.4 TB/s; at a
// decode step's sizes by latency, 64 tokens 3.0 us.

template <typename T, int kVec>
__device__ __forceinline__ void load_vec(const T* p, float* out) {
  constexpr int kPer = kPieceOf<T, kVec>;
#pragma unroll
  for (int i = 0; i < kVec / kPer; ++i) {
    const Piece<T, kPer> piece = reinterpret_cast<const Piece<T, kPer>*>(p)[i];
#pragma unroll
    for (int j = 0; j < kPer; ++j) out[i * kPer + j] = (float)piece.x[j];
  }
}
template <typename T, int kVec>
__device__ __forceinline__ void store_vec(T* p, const float* in) {
  constexpr int kPer = kPieceOf<T, kVec>;
#pragma unroll
  for (int i = 0; i < kVec / kPer; ++i) {
    Piece<T, kPer> piece;
#pragma unroll
    for (int j = 0; j < kPer; ++j) piece.x[j] = (T)in[i * kPer + j];
    reinterpret_cast<Piece<T, kPer>*>(p)[i] = piece;
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
      load_vec<T, kVec>(x + 2 * at, u);
      load_vec<T, kVec>(x + 2 * at + kVec, u + kVec);
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
      store_vec<T, kVec>(y + 2 * at, w);
      store_vec<T, kVec>(y + 2 * at + kVec, w + kVec);
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
    *reinterpret_cast<Piece<T, kVec>*>(y) = *reinterpret_cast<const Piece<T, kVec>*>(x);
  }
}

// ---------------------------------------------------------------------------
// The cache write. A workgroup holds the tokens of one group that stand
// together in the call, for one head of K or V: their largest magnitude gives
// the group's scale, under which their rows are encoded. A group that the call
// enters behind its first slot keeps its rows and the larger of both scales;
// where that grew, the rows that the call does not write are encoded anew.
// Rows are read once: a thread keeps its pieces of 8 elements of up to kHold
// rows in registers from the maximum to the encoding.
//
// Bound by HBM and by the wait for a group's maximum between its reads and its
// writes: 16,381 tokens of 8 heads of 128, 100 MB in groups of 64, 31 us or 3.3
// TB/s; 64 appended tokens 5.8 us, a chain of loads.
//
// Which tokens begin a group is known on the device only. A workgroup looks at
// `chunk` tokens and takes the groups that begin among them one after another.

constexpr int kStoreHold = 4;

template <typename T>
struct Eight {  // elements, as loaded
  u32x4 w[sizeof(T) / 2];
};
template <typename T>
__device__ __forceinline__ void expand(const Eight<T>& e, float* out) {
  const T* x = reinterpret_cast<const T*>(e.w);
#pragma unroll
  for (int j = 0; j < 8; ++j) out[j] = (float)x[j];
}
__device__ __forceinline__ u32x2 encode8(const float* x, float times) {
  u32x2 out;
  out.x = encode4(x[0] * times, x[1] * times, x[2] * times, x[3] * times);
  out.y = encode4(x[4] * times, x[5] * times, x[6] * times, x[7] * times);
  return out;
}

template <typename T, int kThreads>
__global__ __launch_bounds__(kThreads) void store_fp8_kernel(Fp8Cache c, const T* __restrict__ key, int64_t key_stride,
                                                             const T* __restrict__ value, int64_t value_stride,
                                                             const int32_t* __restrict__ slots, int32_t num_tokens,
                                                             int32_t chunk, int32_t lane_bits) {
  constexpr int kHold = kStoreHold;
  __shared__ int owner[kMaxGroup];  // the call's token for each of the group's rows; the last one that names it
  __shared__ int wave_end[kThreads / kWave];
  __shared__ float wave_amax[kThreads / kWave];
  const int tid = threadIdx.x, lane = tid % kWave, wave = tid / kWave;
  const Slice slice = slice_of(blockIdx.x, 2 * c.heads);
  const bool is_v = slice.head >= c.heads;
  const int head = is_v ? slice.head - c.heads : slice.head;
  const int64_t cache_slots = (int64_t)c.num_blocks * c.block_size;
  const int first = slice.unit * chunk;
  if (first >= num_tokens) return;
  auto group_at = [&](int token) {  // -1 where the token is skipped or none
    if (token < 0 || token >= num_tokens) return -1;
    const int s = slots[token];
    return s < 0 || s >= cache_slots ? -1 : c.group_of(s);
  };
  // Skipped tokens do not interrupt a group's: a token begins one if the last before it that is stored is not of it. The
  // one before the chunk's first is looked for 64 tokens at once: one by one, a gap of 16 K took 2,317 us,
  // and takes 60.
  const int mine = lane < chunk ? group_at(first + lane) : -1;
  const uint64_t stored = __ballot(mine >= 0);
  int outside = -1;  // the group of the last token before the chunk that is stored
  for (int from = first - kWave; stored && from > -kWave; from -= kWave) {
    const int group = group_at(from + lane);
    const uint64_t there = __ballot(group >= 0);
    if (there) {
      outside = __shfl(group, 63 - __clzll((long long)there));
      break;
    }
  }
  const uint64_t earlier = stored & ((uint64_t{1} << lane) - 1);
  const int inside = __shfl(mine, earlier ? 63 - __clzll((long long)earlier) : 0);
  const int before = earlier ? inside : outside;
  uint64_t begins = __ballot(mine >= 0 && mine != before);

  const T* src = (is_v ? value : key) + (int64_t)head * c.head_dim;
  const int64_t src_stride = is_v ? value_stride : key_stride;
  const int64_t row_bytes = (int64_t)c.heads * c.head_dim;
  const int at = (tid & ((1 << lane_bits) - 1)) * 8, row0 = tid >> lane_bits, row_step = kThreads >> lane_bits;
  const bool in_row = at < c.head_dim;
  for (; begins; begins &= begins - 1) {
    const int nth = __ffsll((unsigned long long)begins) - 1;
    const int token0 = first + nth, group = __shfl(mine, nth);
    float* scale = (is_v ? c.v_scale : c.k_scale) + (int64_t)group * c.heads + head;
    const float scale_before = *scale;
    const int slot_base = group * c.group;
    for (int i = tid; i < c.group; i += kThreads) owner[i] = -1;
    for (int from = token0;; from += kThreads) {
      const int i = from + tid;
      const int s = i < num_tokens ? slots[i] : -1;
      const bool in_group = s >= slot_base && s - slot_base < c.group;
      const uint64_t out = __ballot(i >= num_tokens || (!in_group && s >= 0 && s < cache_slots));
      if (lane == 0) wave_end[wave] = out ? wave * kWave + __ffsll((unsigned long long)out) - 1 : kThreads;
      __syncthreads();
      int end = kThreads;
#pragma unroll
      for (int w = kThreads / kWave - 1; w >= 0; --w)
        if (wave_end[w] < (w + 1) * kWave) end = wave_end[w];
      if (tid < end && in_group) atomicMax(&owner[s - slot_base], i);
      __syncthreads();
      if (end < kThreads) break;
    }

    Eight<T> held[kHold];
    float amax = 0.0f;
#pragma unroll
    for (int p = 0; p < kHold; ++p) {
      const int row = row0 + p * row_step, token = row < c.group && in_row ? owner[row] : -1;
      if (token < 0) continue;
      held[p] = *reinterpret_cast<const Eight<T>*>(src + token * src_stride + at);
    }
#pragma unroll
    for (int p = 0; p < kHold; ++p) {
      const int row = row0 + p * row_step, token = row < c.group && in_row ? owner[row] : -1;
      if (token < 0) continue;
      float x[8];
      expand<T>(held[p], x);
#pragma unroll
      for (int j = 0; j < 8; ++j) amax = fmaxf(amax, finite_abs(x[j]));
    }
    for (int row = row0 + kHold * row_step; row < c.group; row += row_step) {
      const int token = in_row ? owner[row] : -1;
      if (token < 0) continue;
      float x[8];
      expand<T>(*reinterpret_cast<const Eight<T>*>(src + token * src_stride + at), x);
#pragma unroll
      for (int j = 0; j < 8; ++j) amax = fmaxf(amax, finite_abs(x[j]));
    }
    amax = wave_max(amax);
    if (lane == 0) wave_amax[wave] = amax;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kThreads / kWave; ++w) amax = fmaxf(amax, wave_amax[w]);
    const float kept = owner[0] < 0 && scale_before > 0.0f && scale_before < INFINITY ? scale_before : 0.0f;
    const float fit = fmaxf(scale_for(amax), kept), inverse = 1.0f / fit, shrink = kept / fit;
    const bool grew = kept > 0.0f && fit > kept, power = is_power_of_two(fit);
    if (tid == 0) *scale = fit;
    uint8_t* codes = (is_v ? c.v : c.k) + ((int64_t)slot_base * c.heads + head) * c.head_dim + at;
    auto write = [&](int row, const Eight<T>* held_row) {
      const int token = row < c.group && in_row ? owner[row] : -1;
      u32x2* dst = reinterpret_cast<u32x2*>(codes + row * row_bytes);
      float x[8];
      if (token >= 0) {
        expand<T>(held_row ? *held_row : *reinterpret_cast<const Eight<T>*>(src + token * src_stride + at), x);
        if (!power) {
#pragma unroll
          for (int j = 0; j < 8; ++j) x[j] = quotient_odd(x[j], fit);
        }
        *dst = encode8(x, power ? inverse : 1.0f);
      } else if (grew && row < c.group && in_row) {
        decode4(dst->x, x);
        decode4(dst->y, x + 4);
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] = product_odd(x[j], shrink);
        *dst = encode8(x, 1.0f);
      }
    };
#pragma unroll
    for (int p = 0; p < kHold; ++p) write(row0 + p * row_step, &held[p]);
    for (int row = row0 + kHold * row_step; row < c.group; row += row_step) write(row, nullptr);
    __syncthreads();  // before the next group's owners
  }
}

// ---------------------------------------------------------------------------
// The tokens to keep: for one (sequence, KV head), the last `recent` and the
// (keep - recent) of the earlier ones with the largest weight. The smallest
// weight that is kept is found two bits at a time of the weights' ordered patterns: the
// greatest pattern that at least as many reach as are wanted. The kept tokens
// are then written in order of their position, of equal weights the first.
// A workgroup takes a row, and a wave a contiguous part of it. kHeld: up to 32
// weights a lane stay in registers throughout, so that two bits cost three
// comparisons and scalar bit counts for each 64 weights and one barrier (bit by
// bit, the barriers made it 18.6 and 33.1 us for rows of 8,192 and 32,767); rows
// of more than 32,768 are read again for each two (32,768: 33 us, 32,769: 91, 102,400: 308). The search ends early where exactly as
// many are reached as wanted, and leaves out bits that all patterns share. (A
// radix select by histograms in LDS took 21 and 46 us for rows of 8,192 and
// 32,767: weights crowd in few bins, and additions to one address take turns.)

constexpr int kSelectThreads = 1024;
constexpr int kSelectWaves = kSelectThreads / kWave;
constexpr int kSelectHeld = 32;

// Orders as the weights do: -0 as +0, NaN below everything.
__device__ __forceinline__ uint32_t rank_of(float w) {
  if (w != w) return 0;
  const uint32_t u = w == 0.0f ? 0 : __float_as_uint(w);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

__device__ __forceinline__ float weight_of(uint32_t rank) {
  return rank == 0 ? NAN : __uint_as_float(rank & 0x80000000u ? rank ^ 0x80000000u : ~rank);
}

template <bool kHeld>
__global__ __launch_bounds__(kSelectThreads) void select_kernel(const float* __restrict__ weights, int32_t heads,
                                                                int32_t width, const int32_t* __restrict__ lens,
                                                                int32_t keep, int32_t recent,
                                                                int32_t* __restrict__ indices,
                                                                int32_t* __restrict__ counts,
                                                                float* __restrict__ kept) {
  __shared__ uint32_t reached[16][3], varying[2];
  __shared__ uint32_t wave_a[kSelectWaves], wave_b[kSelectWaves];
  const int64_t row = blockIdx.x;
  const int seq = (int)(row / heads), tid = threadIdx.x, lane = tid % kWave;
  const int wave = __builtin_amdgcn_readfirstlane(tid / kWave);
  const float* w = weights + row * width;
  int32_t* out = indices + row * keep;
  float* out_w = kept + row * keep;
  int n = lens[seq];
  n = n < 0 ? 0 : n > width ? width : n;
  const int count = n < keep ? n : keep;
  const int last = recent < count ? recent : count;  // kept at the end whatever they weigh
  const int pool = n - last, want = count - last;    // of the first `pool`, `want` are kept
  if (tid == 0 && row % heads == 0) counts[seq] = count;
  for (int i = count + tid; i < keep; i += kSelectThreads) {
    out[i] = -1;
    out_w[i] = 0.0f;
  }
  for (int i = tid; i < last; i += kSelectThreads) {
    out[want + i] = pool + i;
    out_w[want + i] = w[pool + i];
  }
  if (want == pool) {
    for (int i = tid; i < pool; i += kSelectThreads) {
      out[i] = i;
      out_w[i] = w[i];
    }
    return;
  }
  if (want == 0) return;

  // The wave's part: [first, first + 64 per), as far as it lies within the pool. Past that, patterns are 0: no candidate
  // is reached by them, and of equal ones they come last (those of j >= per are left out).
  const int per = (pool + kSelectThreads - 1) / kSelectThreads, first = wave * per * kWave;
  auto read = [&](int j) {
    const int i = first + j * kWave + lane;
    return i < pool ? rank_of(w[i]) : 0u;
  };
  uint32_t held[kHeld ? kSelectHeld : 1];
  uint32_t set = 0, clear = 0;  // bits that are set, and clear, in some pattern
  if constexpr (kHeld) {
    // Whole loads first, from places within the row: behind a condition each would be waited for in turn.
#pragma unroll
    for (int j = 0; j < kSelectHeld; ++j) {
      const int i = first + j * kWave + lane;
      held[j] = __float_as_uint(w[i < pool ? i : pool - 1]);
    }
#pragma unroll
    for (int j = 0; j < kSelectHeld; ++j) {
      const bool in = j < per && first + j * kWave + lane < pool;
      held[j] = in ? rank_of(__uint_as_float(held[j])) : 0u;
      set |= held[j];
      clear |= in ? ~held[j] : 0u;
    }
  } else {
    for (int j = 0; j < per; ++j) {
      const uint32_t r = read(j);
      set |= r;
      clear |= first + j * kWave + lane < pool ? ~r : 0u;
    }
  }
  // body(j, pattern) for each j < per, and perhaps some more whose patterns are 0.
  auto each = [&](auto body) {
    if constexpr (kHeld) {
#pragma unroll
      for (int j = 0; j < kSelectHeld; j += 8) {
        if (j >= per) break;
#pragma unroll
        for (int k = 0; k < 8; ++k) body(j + k, held[j + k]);
      }
    } else {
      for (int j = 0; j < per; ++j) body(j, read(j));
    }
  };
  if (tid < 48) reached[tid / 3][tid % 3] = 0;
  if (tid < 2) varying[tid] = 0;
  __syncthreads();
#pragma unroll
  for (int d = 1; d < kWave; d <<= 1) {
    set |= __shfl_xor(set, d);
    clear |= __shfl_xor(clear, d);
  }
  if (lane == 0) {
    atomicOr(&varying[0], set);
    atomicOr(&varying[1], clear);
  }
  __syncthreads();
  uint32_t always = varying[0] & ~varying[1], open = varying[0] & varying[1];
  uint32_t prefix = 0, found = (uint32_t)pool;  // as many reach `prefix`
  for (int low = 30; low >= 0 && found != (uint32_t)want; low -= 2) {
    if (!(open >> low & 3)) {
      prefix |= always & 3u << low;
      continue;
    }
    uint32_t mine[3] = {0, 0, 0};
    each([&](int, uint32_t r) {
#pragma unroll
      for (uint32_t i = 0; i < 3; ++i) mine[i] += (uint32_t)__popcll(__ballot(r >= (prefix | (i + 1) << low)));
    });
    if (lane < 3) atomicAdd(&reached[low / 2][lane], lane == 0 ? mine[0] : lane == 1 ? mine[1] : mine[2]);
    __syncthreads();
    uint32_t digit = 0;
#pragma unroll
    for (uint32_t i = 0; i < 3; ++i) {
      const uint32_t all = reached[low / 2][i];
      if (all >= (uint32_t)want) {
        digit = i + 1;
        found = all;
      }
    }
    prefix |= digit << low;
  }
  // Kept: all that reach it, where those are as many as wanted; else what is above it, and of those equal to it, the
  // smallest weight that is kept, the first ones.
  const bool exact = found == (uint32_t)want;
  if (exact) --prefix;  // `above it` then, and none equal; it is not 0, which all reach
  uint32_t my_overs = 0, my_ties = 0;
  each([&](int j, uint32_t r) {
    my_overs += (uint32_t)__popcll(__ballot(r > prefix));
    my_ties += (uint32_t)__popcll(__ballot(j < per && r == prefix));
  });
  if (lane == 0) {
    wave_a[wave] = my_overs;
    wave_b[wave] = my_ties;
  }
  __syncthreads();
  uint32_t over_at = 0, tie_at = 0, need = (uint32_t)want;
  for (int i = 0; i < kSelectWaves; ++i) {
    if (i < wave) {
      over_at += wave_a[i];
      tie_at += wave_b[i];
    }
    need -= wave_a[i];
  }
  const uint64_t below = (uint64_t{1} << lane) - 1;
  each([&](int j, uint32_t r) {
    const bool over = r > prefix, tie = j < per && r == prefix;
    const uint64_t over_mask = __ballot(over), tie_mask = __ballot(tie);
    const uint32_t tie_rank = tie_at + (uint32_t)__popcll(tie_mask & below);
    if (over || (tie && tie_rank < need)) {
      const uint32_t at = over_at + (uint32_t)__popcll(over_mask & below) + (tie_rank < need ? tie_rank : need);
      out[at] = first + j * kWave + lane;
      out_w[at] = weight_of(r);  // loaded again, it would be waited for in each turn: 17.1 and 35.1 us
    }
    over_at += (uint32_t)__popcll(over_mask);
    tie_at += (uint32_t)__popcll(tie_mask);
  });
}

// ---------------------------------------------------------------------------
// Compaction: a workgroup gathers the rows of one group of the new blocks, for
// one head of K or V, and encodes them under a scale of their own. As in the
// cache write, a thread keeps the pieces that it read, of 16 codes here. Bound by
// reads of single rows of a head, 128 bytes from anywhere: 67 MB read and written
// for 8 contexts of 8 heads cut to 2,048 tokens in 20 us.

constexpr int kCompactHold = 2;
template <int kThreads>
__global__ __launch_bounds__(kThreads) void compact_kernel(Fp8Cache c, PagedBatch from,
                                                           const int32_t* __restrict__ indices,
                                                           const int32_t* __restrict__ counts, int32_t keep,
                                                           const int32_t* __restrict__ to_tables, int64_t to_stride,
                                                           int32_t to_width, int32_t lane_bits) {
  constexpr int kHold = kCompactHold;
  __shared__ float wave_amax[kThreads / kWave];
  constexpr int kRows = kThreads < 4 * kWave ? kHold * kThreads : kMaxGroup;  // fewer waves hold the group (launch_compact)
  __shared__ int64_t source[kRows], source_scale[kRows];  // each row's slot, or -1, and its scale's element
  const int tid = threadIdx.x;
  const Slice slice = slice_of(blockIdx.x, 2 * c.heads);
  const int seq = slice.unit % from.num_seqs;
  const bool is_v = slice.head >= c.heads;
  const int head = is_v ? slice.head - c.heads : slice.head;
  int count = counts[seq];
  count = count < 0 ? 0 : count > keep ? keep : count;
  const int first = slice.unit / from.num_seqs * c.group;
  if (first >= count) return;
  const int rows = count - first < c.group ? count - first : c.group;
  const int to_block = c.block_of(first);
  if (to_block >= to_width) return;
  const int target = to_tables[seq * to_stride + to_block];
  if (target < 0 || target >= c.num_blocks) return;
  uint8_t* codes = is_v ? c.v : c.k;
  float* scales = is_v ? c.v_scale : c.k_scale;
  const int64_t to_slot = (int64_t)target * c.block_size + (first - to_block * c.block_size);
  const int32_t* mine = indices + ((int64_t)seq * c.heads + head) * keep + first;
  const int context = context_of(c, from, seq);
  for (int i = tid; i < rows; i += kThreads) {
    const int t = mine[i];
    int64_t slot = -1, scale = 0;
    if (t >= 0 && t < context) {
      const int b = c.block_of(t), in = t - b * c.block_size;
      const int id = from.tables[seq * from.table_stride + b];
      if (id >= 0 && id < c.num_blocks) {
        slot = (int64_t)id * c.block_size + in;
        scale = ((int64_t)id * (c.block_size / c.group) + c.group_of(in)) * c.heads + head;
      }
    }
    source[i] = slot;
    source_scale[i] = scale;
  }
  __syncthreads();
  const int at = (tid & ((1 << lane_bits) - 1)) * 16, row0 = tid >> lane_bits, row_step = kThreads >> lane_bits;
  const bool in_row = at < c.head_dim;
  // A row's piece and its scale.
  struct Row {
    u32x4 codes;
    float scale;
  };
  auto read = [&](int row) {
    Row r = {u32x4{0, 0, 0, 0}, 0.0f};
    if (row < rows && in_row && source[row] >= 0) {
      r.codes = *reinterpret_cast<const u32x4*>(codes + (source[row] * c.heads + head) * c.head_dim + at);
      r.scale = scales[source_scale[row]];
    }
    return r;
  };
  // The largest finite code's value, over 2^10: the value itself may exceed fp32 (256 under a scale of 2^120, which a bf16
  // value of nearly 2^128 is stored as). Rounded to odd, so that it lies on its own side of the border between two scales.
  auto amax_of = [&](const Row& r) {
    float x[16], most = 0.0f;
#pragma unroll
    for (int i = 0; i < 4; ++i) decode4(r.codes[i], x + 4 * i);
#pragma unroll
    for (int i = 0; i < 16; ++i) most = fmaxf(most, finite_abs(x[i]));
    return finite_abs(product_odd(most * 0x1p-10f, r.scale));
  };
  Row held[kHold];
  float amax = 0.0f;
#pragma unroll
  for (int p = 0; p < kHold; ++p) held[p] = read(row0 + p * row_step);
#pragma unroll
  for (int p = 0; p < kHold; ++p) amax = fmaxf(amax, amax_of(held[p]));
  for (int row = row0 + kHold * row_step; row < rows; row += row_step) amax = fmaxf(amax, amax_of(read(row)));
  amax = wave_max(amax);
  if (tid % kWave == 0) wave_amax[tid / kWave] = amax;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kThreads / kWave; ++w) amax = fmaxf(amax, wave_amax[w]);
  const float fit = scale_for<10>(amax), inverse = 1.0f / fit;
  if (tid == 0)
    scales[((int64_t)target * (c.block_size / c.group) + c.group_of(first - to_block * c.block_size)) * c.heads + head] = fit;
  auto write = [&](const Row& r, int row) {
    if (row >= rows || !in_row) return;
    float x[16];
    const float times = r.scale * inverse;
#pragma unroll
    for (int i = 0; i < 4; ++i) decode4(r.codes[i], x + 4 * i);
    if (is_power_of_two(r.scale)) {
#pragma unroll
      for (int i = 0; i < 16; ++i) x[i] *= times;
    } else {
#pragma unroll
      for (int i = 0; i < 16; ++i) x[i] = product_odd(x[i], times);
    }
    const u32x2 lo = encode8(x, 1.0f), hi = encode8(x + 8, 1.0f);
    *reinterpret_cast<u32x4*>(codes + ((to_slot + row) * c.heads + head) * c.head_dim + at) = u32x4{lo.x, lo.y, hi.x, hi.y};
  };
#pragma unroll
  for (int p = 0; p < kHold; ++p) write(held[p], row0 + p * row_step);
  for (int row = row0 + kHold * row_step; row < rows; row += row_step) write(read(row), row);
}

template <typename T, int kVec>
hipError_t rotary_by(const RotaryArgs& a, hipStream_t stream) {
  const size_t lds = (size_t)a.rotary_dim / 2 * sizeof(float2);
  const dim3 grid((unsigned)a.num_tokens), block(kThreads);
  if (a.interleaved) rotary_kernel<T, kVec, true><<<grid, block, lds, stream>>>(a);
  else rotary_kernel<T, kVec, false><<<grid, block, lds, stream>>>(a);
  return hipGetLastError();
}

// By 16 bytes where everything lies on 16 bytes, halves of the rotated part among it; by two elements likewise (a head_dim
// of 80 with 20 rotated); else one by one.
template <typename T>
hipError_t rotary_of(const RotaryArgs& a, hipStream_t stream) {
  auto lies_on = [&](int count) {
    const int64_t elements[] = {a.q_stride, a.k_stride, a.q_out_stride, a.k_out_stride, a.head_dim, a.rotary_dim / 2};
    const void* pointers[] = {a.query, a.key, a.query_out, a.key_out};
    bool fits = true;
    for (int64_t e : elements) fits = fits && e % count == 0;
    for (const void* p : pointers) fits = fits && (uintptr_t)p % (count * sizeof(T)) == 0;
    return fits;
  };
  constexpr int kWide = 16 / sizeof(T);
  if (lies_on(kWide)) return rotary_by<T, kWide>(a, stream);
  if (lies_on(2)) return rotary_by<T, 2>(a, stream);
  return rotary_by<T, 1>(a, stream);
}

// Workgroups have one or two waves where their lanes can hold a group, else four: 16,384 tokens of 8 heads of 128 in groups
// of 16 take 27 us by one wave and 52 by four, in groups of 32 28.5 by two and 34.5 by four.
// Each looks at as many tokens as leave so many workgroups, and at most at a group's, so that most of a prompt's find one
// group that begins. A decode step's tokens begin a group each, which then wait for one another: with 2,048 / 4,096 / 8,192
// workgroups of one wave 1,024 appended tokens of 8 heads take 21.1 / 14.3 / 14.7 us, as many of a prompt 6.7 / 8.6 / 13.1
// (512: 12.3 / 9.1 / 10.0 and 6.6 / 8.3 / 9.8; 2,048: 38.9 / 24.3 / 24.4 and 6.9 / 8.7 / 13.6); with 1,024 / 2,048 / 4,096
// of four, in groups of 64, 43 / 42 / 42 and 8.3 / 13.2 / 15.1 (4,096 tokens: 162 / 156 / 148 and 8.9 / 15.0 / 25.2).
constexpr int kStoreFull = 4096, kStoreFullWide = 2048;

template <typename T, int kThreads>
hipError_t store_by(const Fp8Cache& c, const void* key, int64_t key_stride, const void* value, int64_t value_stride,
                    const int32_t* slots, int32_t num_tokens, int lane_bits, hipStream_t stream) {
  const int most = c.group < kWave ? c.group : kWave;
  int chunk = 1;
  constexpr int kFull = kThreads == kWave ? kStoreFull : kStoreFullWide;
  while (chunk < most && (int64_t)num_tokens * 2 * c.heads > (int64_t)chunk * kFull) chunk *= 2;
  if (chunk > most) chunk = most;
  const dim3 grid((unsigned)slices_grid((num_tokens + chunk - 1) / chunk, 2 * c.heads));
  store_fp8_kernel<T, kThreads><<<grid, dim3(kThreads), 0, stream>>>(
      c, (const T*)key, key_stride, (const T*)value, value_stride, slots, num_tokens, chunk, lane_bits);
  return hipGetLastError();
}
template <typename T>
hipError_t store_of(const Fp8Cache& c, const void* key, int64_t key_stride, const void* value, int64_t value_stride,
                    const int32_t* slots, int32_t num_tokens, hipStream_t stream) {
  int lane_bits = 1;
  while ((8 << lane_bits) < c.head_dim) ++lane_bits;
  const int pieces = c.group << lane_bits;
  if (pieces <= kStoreHold * kWave)
    return store_by<T, kWave>(c, key, key_stride, value, value_stride, slots, num_tokens, lane_bits, stream);
  if (pieces <= kStoreHold * 2 * kWave)
    return store_by<T, 2 * kWave>(c, key, key_stride, value, value_stride, slots, num_tokens, lane_bits, stream);
  return store_by<T, kThreads>(c, key, key_stride, value, value_stride, slots, num_tokens, lane_bits, stream);
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
  const dim3 grid((unsigned)rows), block(kSelectThreads);
  if (width <= kSelectThreads * kSelectHeld)
    select_kernel<true><<<grid, block, 0, stream>>>(weights, heads, width, context_lens, keep, recent, indices, counts, kept);
  else
    select_kernel<false><<<grid, block, 0, stream>>>(weights, heads, width, context_lens, keep, recent, indices, counts, kept);
  return hipGetLastError();
}

hipError_t launch_compact(const Fp8Cache& c, const PagedBatch& from, const int32_t* indices, const int32_t* counts,
                          int32_t keep, const int32_t* to_tables, int64_t to_stride, int32_t to_width,
                          hipStream_t stream) {
  const dim3 grid((unsigned)slices_grid((int64_t)((keep + c.group - 1) / c.group) * from.num_seqs, 2 * c.heads));
  int lane_bits = 0;
  while ((16 << lane_bits) < c.head_dim) ++lane_bits;
  // Waves as many as hold a group, up to four (8 contexts of 8 heads cut to 2,048 tokens in groups of 16 20 us, 41 by four).
  auto launch = [&](auto kernel, int threads) {
    kernel<<<grid, dim3(threads), 0, stream>>>(c, from, indices, counts, keep, to_tables, to_stride, to_width, lane_bits);
  };
  const int pieces = c.group << lane_bits;
  if (pieces <= kCompactHold * kWave) launch(compact_kernel<kWave>, kWave);
  else if (pieces <= kCompactHold * 2 * kWave) launch(compact_kernel<2 * kWave>, 2 * kWave);
  else launch(compact_kernel<kThreads>, kThreads);
  return hipGetLastError();
}

}  // namespace kvx
