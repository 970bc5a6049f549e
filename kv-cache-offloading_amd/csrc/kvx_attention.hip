// Attention over a paged e4m3 KV cache, and the weight that each cached token
// received, on CDNA4's matrix cores.
//
// Layout of a wave's work: 32 keys a step against 16 * kTiles query rows (a
// row is a query token and one of the query heads that share the KV head).
// Both products keep the query rows in the lanes:
//   S^T = K Q^T   mfma 16x16x32: A = 16 keys, B = 16 query rows; lane (c, g),
//                 c = lane % 16, g = lane / 16, gets row c's scores of keys 4 g + i
//   O^T = V^T P^T mfma 16x16x32 over the step's 32 keys: lane (c, g)'s P values
//                 are, without a move, the B operand, if the contraction takes
//                 the keys in the order 4 g + i of the first 16, then of the
//                 second. V^T's operand then needs, for one column of the
//                 head, the codes of those 8 keys: each lane loads them for
//                 head_dim / 16 adjacent columns and transposes bytes in registers.
// So neither K, V, S nor P passes through LDS. The codes become bf16 (or fp16)
// values in registers, which hold every e4m3 value exactly; K's scale is
// applied to the scores and V's to P, in fp32.
//
// Softmax statistics, sums and outputs are fp32 until the last rounding. P is
// rounded to bf16 for the second product, and the rounding's remainder added as
// a second bf16 operand, which leaves P with 16 bits in every kernel: outputs are
// as far from the formula's as their type's rounding alone leaves them, 0.0017.
// (By one operand, 8 bits, two chunks of 3,549 rows of 32 heads take 476 us in
// place of 590, and are 0.0023 off.)
#include <algorithm>
#include <type_traits>

#include "kvx_step.h"

namespace kvx {
namespace {

constexpr int kWaves = 4;
constexpr int kThreads = kWaves * kWave;
constexpr int kStep = 32;  // keys

template <int kType>
struct Query;
template <>
struct Query<KVX_DTYPE_BF16> {
  using T = __bf16;
  using Vec = bf16x8;
  static __device__ __forceinline__ f32x4 mfma(Vec a, Vec b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
  }
  static __device__ __forceinline__ uint32_t pair(uint32_t codes, bool high) {
    return high ? __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(codes, 1.0f, true))
                : __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(codes, 1.0f, false));
  }
};
template <>
struct Query<KVX_DTYPE_FP16> {
  using T = _Float16;
  using Vec = f16x8;
  static __device__ __forceinline__ f32x4 mfma(Vec a, Vec b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
  }
  static __device__ __forceinline__ uint32_t pair(uint32_t codes, bool high) {
    return high ? __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(codes, 1.0f, true))
                : __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(codes, 1.0f, false));
  }
};

// Eight codes (two words) as an operand of the query's type.
template <typename Q>
__device__ __forceinline__ typename Q::Vec decode8(uint32_t lo, uint32_t hi) {
  const u32x4 w = {Q::pair(lo, false), Q::pair(lo, true), Q::pair(hi, false), Q::pair(hi, true)};
  return __builtin_bit_cast(typename Q::Vec, w);
}

__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  const f32x2 v = {lo, hi};
  return __builtin_bit_cast(uint32_t, __builtin_convertvector(v, bf16x2));
}

// The largest (sum) of the values of the four lanes that hold one query row.
__device__ __forceinline__ float rows_max(float x) {
  x = fmaxf(x, __shfl_xor(x, 16));
  return fmaxf(x, __shfl_xor(x, 32));
}
__device__ __forceinline__ float rows_sum(float x) {
  x += __shfl_xor(x, 16);
  return x + __shfl_xor(x, 32);
}

// Rows x[0..3] of four bytes each -> their columns.
__device__ __forceinline__ void transpose4(const uint32_t* x, uint32_t* out) {
  const uint32_t a = __builtin_amdgcn_perm(x[1], x[0], 0x05010400u);  // bytes 0, 0', 1, 1'
  const uint32_t b = __builtin_amdgcn_perm(x[1], x[0], 0x07030602u);  // bytes 2, 2', 3, 3'
  const uint32_t c = __builtin_amdgcn_perm(x[3], x[2], 0x05010400u);
  const uint32_t d = __builtin_amdgcn_perm(x[3], x[2], 0x07030602u);
  out[0] = __builtin_amdgcn_perm(c, a, 0x05040100u);
  out[1] = __builtin_amdgcn_perm(c, a, 0x07060302u);
  out[2] = __builtin_amdgcn_perm(d, b, 0x05040100u);
  out[3] = __builtin_amdgcn_perm(d, b, 0x07060302u);
}

// A value that all lanes have, in a scalar register.
__device__ __forceinline__ int64_t scalar(int64_t x) {
  const uint32_t lo = __builtin_amdgcn_readfirstlane((int)(uint32_t)x);
  const uint32_t hi = __builtin_amdgcn_readfirstlane((int)(uint32_t)(x >> 32));
  return (int64_t)((uint64_t)hi << 32 | lo);
}
__device__ __forceinline__ float scalar(float x) {
  return __uint_as_float(__builtin_amdgcn_readfirstlane(__float_as_int(x)));
}
// A lane's value, in a scalar register.
__device__ __forceinline__ int64_t lane_value(int64_t x, int lane) {
  const uint32_t lo = __builtin_amdgcn_readlane((int)(uint32_t)x, lane);
  const uint32_t hi = __builtin_amdgcn_readlane((int)(uint32_t)(x >> 32), lane);
  return (int64_t)((uint64_t)hi << 32 | lo);
}
__device__ __forceinline__ float lane_value(float x, int lane) {
  return __uint_as_float(__builtin_amdgcn_readlane(__float_as_int(x), lane));
}

__device__ __forceinline__ uint32_t nan_bytes(uint32_t codes) {  // 0x80 in each byte that is a NaN code
  return ((codes & 0x7F7F7F7Fu) + 0x01010101u) & 0x80808080u;
}

// Four columns of a query row's weighted sum `y` over one split's keys, taken relative to 2^base and with the weights'
// sum: the output where there is one split, else a part of it.
template <typename T>
__device__ __forceinline__ void write_rows(const AttentionArgs& a, int split, int64_t row, int col, float base,
                                           float sum, f32x4 y) {
  if (a.splits > 1) {
    const int64_t rows = (int64_t)a.batch.num_tokens * a.q_heads, at = split * rows + row;
    *reinterpret_cast<f32x4*>(a.partial + at * a.cache.head_dim + col) = y;
    if (col == 0)
      *reinterpret_cast<f32x2*>(a.partial + a.splits * rows * a.cache.head_dim + at * 2) = f32x2{base, sum};
    return;
  }
  const float inverse = sum == 0.0f ? 0.0f : 1.0f / sum;
  alignas(8) T out[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) out[j] = (T)(sum == 0.0f ? 0.0f : y[j] * inverse);
  *reinterpret_cast<u32x2*>((T*)a.out + row * a.cache.head_dim + col) = *reinterpret_cast<const u32x2*>(out);
  if (a.lse && col == 0) a.lse[row] = sum == 0.0f ? -INFINITY : (base + log2f(sum)) * 0.69314718055994531f;
}

// Few query rows: single tokens, proposed ones, short chunks. Bound by the
// bytes of the codes; the four waves of a workgroup take its split's steps in
// turn and join their parts in LDS, and the splits of a context are joined by a
// second launch. A wave looks up 32 steps' blocks and scales at once, a lane
// for each 16-key tile, and loads a step's codes while it uses those of the one
// before. 64 sequences of 300 to 8,192 tokens on 8 heads of 128 take 96-100 us, 4.5
// TB/s; of even lengths 5.0-5.4.
// kHd: head_dim rounded up to 64, 128 or 256; the columns past head_dim are
// zeros. kTiles query tiles of 16 rows.
template <int kType, int kHd, int kTiles>
__global__ __launch_bounds__(kThreads, kHd * kTiles <= 128 ? 2 : 1) void few_rows_kernel(AttentionArgs a) {
  using Q = Query<kType>;
  using B = Query<KVX_DTYPE_BF16>;
  using T = typename Q::T;
  using Vec = typename Q::Vec;
  constexpr int kChunks = kHd / 64;    // 64 columns of K: one 16-byte load a lane
  constexpr int kCols = kHd / 16;      // columns of V a lane loads, transposes and accumulates
  constexpr int kRows = 16 * kTiles;
  __shared__ float parts[kWaves][16][kHd + 4];
  __shared__ float part_base[kWaves][kRows], part_sum[kWaves][kRows];
  const Fp8Cache& cache = a.cache;
  const int lane = threadIdx.x % kWave, c = lane % 16, g = lane / 16;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);

  const Slice slice = slice_of(blockIdx.x, cache.heads);
  const int seq = slice.unit % a.batch.num_seqs, rest = slice.unit / a.batch.num_seqs, head = slice.head;
  const int tile = rest % a.row_tiles, split = rest / a.row_tiles;
  if (split >= a.splits) return;
  const int context = context_of(cache, a.batch, seq);
  const int first_step = split * a.split_steps;
  // The first split also writes the rows that see nothing.
  if (first_step * kStep >= context && split > 0) return;
  const QueryRows rows = query_rows(a.batch, seq);
  const int num_rows = rows.count * a.per_kv;
  const int32_t* table = a.batch.tables + seq * a.batch.table_stride;
  const int64_t row_bytes = (int64_t)cache.heads * cache.head_dim;
  // A lane's places in a tile of K, 64 columns apart, and in one of V, a row apart. Columns past head_dim are read as
  // others before it: the query is 0 there, and the output is not written.
  uint32_t k_lane[kChunks];
#pragma unroll
  for (int k = 0; k < kChunks; ++k) k_lane[k] = c * (uint32_t)row_bytes + min(k * 64 + g * 16, cache.head_dim - 16);
  const uint32_t v_lane = 4 * g * (uint32_t)row_bytes + min(c * kCols, cache.head_dim - kCols);

  // A launch covers max_seqlen queries a sequence; longer ones wrap around.
  for (int tile_row = tile * kRows; tile_row < num_rows; tile_row += a.row_tiles * kRows) {
    // Query rows and the last key each may see.
    Vec q[kTiles][2 * kChunks];
    int last[kTiles];
#pragma unroll
    for (int n = 0; n < kTiles; ++n) {
      const int r = tile_row + n * 16 + c;
      const bool real = r < num_rows;
      const int nth = a.per_kv_of(r), sub = r - nth * a.per_kv;
      last[n] = real ? context - rows.count + nth : -1;
      const T* src = (const T*)a.query + (int64_t)(rows.first + nth) * a.q_stride +
                     (int64_t)(head * a.per_kv + sub) * cache.head_dim;
#pragma unroll
      for (int k = 0; k < kChunks; ++k) {
        const int at = k * 64 + g * 16;
        u32x4 lo = {0, 0, 0, 0}, hi = {0, 0, 0, 0};
        if (real && at < cache.head_dim) {
          lo = *reinterpret_cast<const u32x4*>(src + at);
          hi = *reinterpret_cast<const u32x4*>(src + at + 8);
        }
        q[n][2 * k] = __builtin_bit_cast(Vec, lo);
        q[n][2 * k + 1] = __builtin_bit_cast(Vec, hi);
      }
    }
    const int tile_last = min(tile_row + kRows, num_rows) - 1;
    const int most = context - rows.count + (int)a.per_kv_of(tile_last);
    // Every key up to here is seen by all of the tile's rows.
    const int least = context - rows.count + (int)a.per_kv_of(tile_row);

    f32x4 o[kTiles][kCols];
    float top[kTiles], base[kTiles], sum[kTiles];
#pragma unroll
    for (int n = 0; n < kTiles; ++n) {
      top[n] = -INFINITY;
      base[n] = sum[n] = 0.0f;
#pragma unroll
      for (int d = 0; d < kCols; ++d) o[n][d] = f32x4{0, 0, 0, 0};
    }
    const int end_step = most < 0 ? 0 : min(first_step + a.split_steps, most / kStep + 1);
    const int my_first = first_step + wave;
    const int my_steps = my_first < end_step ? (end_step - my_first + kWaves - 1) / kWaves : 0;

    u32x4 k_codes[2][kChunks];
    uint32_t v_codes[8][kCols / 4];
    int64_t info_row = -1;  // of tile lane % 2 of the batch's step lane / 2
    float info_k = 0.0f, info_v = 0.0f;  // as loaded: used at once, they would hold up the codes' loads
    auto look_up = [&](int nth) {
      const int step = my_first + (nth + lane / 2) * kWaves, key = step * kStep + lane % 2 * 16;
      info_row = -1;
      info_k = info_v = 0.0f;
      if (step < end_step && key < context) {
        const int block = cache.block_of(key), in = key - block * cache.block_size;
        const int id = table[block];
        if (id >= 0 && id < cache.num_blocks) {
          info_row = ((int64_t)id * cache.block_size + in) * cache.heads + head;
          const int64_t at = ((int64_t)id * (cache.block_size / cache.group) + cache.group_of(in)) * cache.heads + head;
          info_k = cache.k_scale[at];
          info_v = cache.v_scale[at];
        }
      }
    };
    auto row_of = [&](int nth, int t) { return lane_value(info_row, nth % 32 * 2 + t); };
    // Loads without a condition (tiles that are not there read as the pool's first one, and count for nothing): behind
    // one, the compiler would wait for all loads under way before it uses any.
    // K: lane (c, g) takes columns 16 g .. 16 g + 15 of each 64 of key c's row.
    auto load_k = [&](int nth) {
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const int64_t row = row_of(nth, t);
        const uint8_t* tile = cache.k + (row < 0 ? 0 : row) * cache.head_dim;
#pragma unroll
        for (int k = 0; k < kChunks; ++k) k_codes[t][k] = *reinterpret_cast<const u32x4*>(tile + k_lane[k]);
      }
    };
    // V: columns kCols c .. of keys 4 g + i.
    auto load_v = [&](int nth) {
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const int64_t row = row_of(nth, t);
        const uint8_t* tile = cache.v + (row < 0 ? 0 : row) * cache.head_dim;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint8_t* p = tile + i * row_bytes + v_lane;
          uint32_t(&v)[kCols / 4] = v_codes[4 * t + i];
          if constexpr (kCols == 4) {
            v[0] = *reinterpret_cast<const uint32_t*>(p);
          } else if constexpr (kCols == 8) {
            const u32x2 w = *reinterpret_cast<const u32x2*>(p);
            v[0] = w.x;
            v[1] = w.y;
          } else {
            const u32x4 w = *reinterpret_cast<const u32x4*>(p);
            v[0] = w.x;
            v[1] = w.y;
            v[2] = w.z;
            v[3] = w.w;
          }
        }
      }
    };
    auto use = [&](int nth) {
      const int key0 = (my_first + nth * kWaves) * kStep;
      bool there[2];
      float ks[2], vs[2];
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const int at = nth % 32 * 2 + t;
        there[t] = row_of(nth, t) >= 0;
        ks[t] = lane_value(info_k, at) * a.scale;
        vs[t] = lane_value(info_v, at);
      }
      f32x4 s[kTiles][2];
#pragma unroll
      for (int t = 0; t < 2; ++t) {
#pragma unroll
        for (int n = 0; n < kTiles; ++n) s[n][t] = f32x4{0, 0, 0, 0};
#pragma unroll
        for (int k = 0; k < kChunks; ++k) {
          const u32x4 w = k_codes[t][k];
          const Vec lo = decode8<Q>(w.x, w.y), hi = decode8<Q>(w.z, w.w);
#pragma unroll
          for (int n = 0; n < kTiles; ++n) {
            s[n][t] = Q::mfma(lo, q[n][2 * k], s[n][t]);
            s[n][t] = Q::mfma(hi, q[n][2 * k + 1], s[n][t]);
          }
        }
      }
      load_k(nth + 1);
      // Keys that some row may not see, and codes in their places that are no numbers.
      const bool partial = key0 + kStep - 1 > least || !there[0] || !there[1];
      bool mend = false;
      if (partial) {
        uint32_t nan = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j)
#pragma unroll
          for (int k = 0; k < kCols / 4; ++k) nan |= nan_bytes(v_codes[j][k]);
        mend = __any(nan != 0);
      }
      u32x4 p_hi[kTiles], p_lo[kTiles];
      uint32_t seen[kTiles];  // bit j: this lane's row sees its key j
#pragma unroll
      for (int n = 0; n < kTiles; ++n) {
        float x[8];
        seen[n] = 0xFF;
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] = s[n][j / 4][j % 4] * ks[j / 4];
        if (partial) {
          seen[n] = 0;
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const bool see = key0 + (j / 4) * 16 + 4 * g + j % 4 <= last[n] && there[j / 4];
            x[j] = see ? x[j] : -INFINITY;
            seen[n] |= see ? 1u << j : 0u;
          }
        }
        float high = x[0];
#pragma unroll
        for (int j = 1; j < 8; ++j) high = fmaxf(high, x[j]);
        if (__any(high > top[n] + 8.0f)) {  // see the chunks' kernel
          top[n] = fmaxf(rows_max(high), top[n]);
          const float now = top[n] == -INFINITY ? base[n] : ceilf(top[n]);
          // The base only rises, but for the first time, from 0, to a row's scores that may all lie below -128: nothing
          // has been summed then, and infinity times it would be NaN.
          const float fade = __builtin_amdgcn_exp2f(fminf(base[n] - now, 0.0f));
          base[n] = now;
          sum[n] *= fade;
#pragma unroll
          for (int d = 0; d < kCols; ++d) o[n][d] *= fade;
        }
        float p[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          p[j] = __builtin_amdgcn_exp2f(x[j] - base[n]);
          sum[n] += p[j];
        }
        uint32_t hi[4], lo[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float y0 = p[2 * j] * vs[j / 2], y1 = p[2 * j + 1] * vs[j / 2];
          hi[j] = pack_bf16(y0, y1);
          lo[j] = pack_bf16(y0 - __uint_as_float(hi[j] << 16), y1 - __uint_as_float(hi[j] & 0xFFFF0000u));
        }
        p_hi[n] = u32x4{hi[0], hi[1], hi[2], hi[3]};
        p_lo[n] = u32x4{lo[0], lo[1], lo[2], lo[3]};
      }
      if (mend) {
        // A key that is masked for a row adds nothing to it, though its code be NaN: NaN codes count as zeros, and rows
        // that see one become NaN.
#pragma unroll
        for (int k = 0; k < kCols / 4; ++k) {
          uint32_t in[8], lo[4], hi[4];
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            in[j] = nan_bytes(v_codes[j][k]) >> 7;
            v_codes[j][k] &= ~(in[j] * 0xFFu);
            in[j] *= 0x38u;  // 1.0
          }
          transpose4(in, lo);
          transpose4(in + 4, hi);
#pragma unroll
          for (int d = 0; d < 4; ++d) {
            const bf16x8 is_nan = decode8<B>(lo[d], hi[d]);
#pragma unroll
            for (int n = 0; n < kTiles; ++n) {
              u32x4 w;
#pragma unroll
              for (int j = 0; j < 4; ++j)
                w[j] = ((seen[n] >> (2 * j)) & 1u ? 0x3F80u : 0u) | ((seen[n] >> (2 * j + 1)) & 1u ? 0x3F800000u : 0u);
              const f32x4 hit = B::mfma(is_nan, __builtin_bit_cast(bf16x8, w), f32x4{0, 0, 0, 0});
#pragma unroll
              for (int i = 0; i < 4; ++i) o[n][4 * k + d][i] += hit[i] > 0.0f ? NAN : 0.0f;
            }
          }
        }
      }
#pragma unroll
      for (int k = 0; k < kCols / 4; ++k) {
        uint32_t in[8], lo[4], hi[4];
#pragma unroll
        for (int j = 0; j < 8; ++j) in[j] = v_codes[j][k];
        transpose4(in, lo);
        transpose4(in + 4, hi);
#pragma unroll
        for (int d = 0; d < 4; ++d) {
          const bf16x8 w = decode8<B>(lo[d], hi[d]);
#pragma unroll
          for (int n = 0; n < kTiles; ++n) {
            o[n][4 * k + d] = B::mfma(w, __builtin_bit_cast(bf16x8, p_hi[n]), o[n][4 * k + d]);
            o[n][4 * k + d] = B::mfma(w, __builtin_bit_cast(bf16x8, p_lo[n]), o[n][4 * k + d]);
          }
        }
      }
    };
    // K's registers are loaded for the next step once the scores are taken, V's once the outputs are; behind the last
    // step, from some tile of the batch, for nothing.
    for (int batch = 0; batch < my_steps; batch += 32) {
      look_up(batch);
      const int batch_end = min(batch + 32, my_steps);
      load_k(batch);
      load_v(batch);
      for (int nth = batch; nth < batch_end; ++nth) {
        use(nth);
        load_v(nth + 1);
      }
    }
#pragma unroll
    for (int n = 0; n < kTiles; ++n) {
      sum[n] = rows_sum(sum[n]);
      if (g == 0) {
        part_base[wave][n * 16 + c] = top[n] == -INFINITY ? -INFINITY : base[n];
        part_sum[wave][n * 16 + c] = sum[n];
      }
    }
    // The waves' parts, 16 rows at a time; threads take 4 columns of a row.
#pragma unroll
    for (int n = 0; n < kTiles; ++n) {
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int d = 0; d < kCols; d += 4)
          *reinterpret_cast<f32x4*>(&parts[wave][c][(4 * g + i) * kCols + d]) =
              f32x4{o[n][d][i], o[n][d + 1][i], o[n][d + 2][i], o[n][d + 3][i]};
      __syncthreads();
#pragma unroll
      for (int piece = threadIdx.x; piece < 16 * kHd / 4; piece += kThreads) {
        const int row = piece / (kHd / 4), col = piece % (kHd / 4) * 4, r = tile_row + n * 16 + row;
        if (r >= num_rows || col >= cache.head_dim) continue;
        float all = -INFINITY, total = 0.0f;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) all = fmaxf(all, part_base[w][n * 16 + row]);
        f32x4 y = {0, 0, 0, 0};
#pragma unroll
        for (int w = 0; w < kWaves; ++w) {
          const float fade = __builtin_amdgcn_exp2f(part_base[w][n * 16 + row] - all);
          const float part = part_sum[w][n * 16 + row];
          if (part == 0.0f) continue;  // also where nothing was seen, and `all` is no number to compare with
          total += part * fade;
          y += *reinterpret_cast<const f32x4*>(&parts[w][row][col]) * fade;
        }
        const int nth = a.per_kv_of(r), sub = r - nth * a.per_kv;
        const int64_t out_row = (int64_t)(rows.first + nth) * a.q_heads + head * a.per_kv + sub;
        write_rows<T>(a, split, out_row, col, all, total, y);
      }
      __syncthreads();
    }
  }
}

// ---------------------------------------------------------------------------
// Chunks of prompts: many query rows, bound by the matrix cores and the
// softmax's VALU work beside them.
//
// A workgroup takes 32 query rows a wave of one (sequence, KV head) and passes
// over the keys kKeys at a time. The waves convert the codes
// to bf16 (K: the query's type) into LDS once for all of them: K's rows as they
// are, V transposed, with the exponent of its scale applied by the converting
// instruction (what a user's own scale is besides, P takes: rounded into V, it
// would leave V 8 bits). LDS is double-buffered, the codes of the next keys are
// loaded into registers while the present ones are used, and their blocks are
// looked up one pass before that.
// As above, S^T = K Q^T and O^T = V^T P^T, now by mfma 32x32x16: lane (n, h), n =
// lane % 32, h = lane / 32, gets query row n's scores of keys 8 (i / 4) + 4 h + i % 4;
// V^T's rows in LDS hold the keys in the order in which P lies in the lanes.
// A wave's step is 32 keys: the scores of the next step are computed under the
// exponentials of this one, and the other wave of the SIMD fills what is left.
// The maximum that exponents are taken from moves only when a score exceeds it
// by 2^8: P <= 2^8 costs bf16 and fp32 no precision, and most steps need neither
// a reduction over lanes nor a pass over the outputs.
// Two chunks (3,549 rows of 32 heads of 128) behind 6-8 K tokens take 592 us, 627
// TFLOP/s; the matrix cores are busy for 52% of the time, with three products for
// each two that count, and arithmetic takes 60% of the issue cycles.

typedef float f32x16 __attribute__((ext_vector_type(16)));

template <int kType>
__device__ __forceinline__ f32x16 mfma32(typename Query<kType>::Vec a, typename Query<kType>::Vec b, f32x16 c) {
  if constexpr (kType == KVX_DTYPE_BF16) return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
  else return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}

// Two codes as bf16, times 2^exponent of `scale`.
__device__ __forceinline__ uint32_t pair_scaled(uint32_t codes, float scale, bool high) {
  return high ? __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(codes, scale, true))
              : __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(codes, scale, false));
}

// A scale over its power of two, within [1, 2).
__device__ __forceinline__ float rest_of(float scale) {
  return __uint_as_float((__float_as_uint(scale) & 0x007FFFFFu) | 0x3F800000u);
}

// What a pass needs to know of its keys' 16-key tiles.
template <int kTiles16>
struct KeyInfo {
  int64_t row[kTiles16];  // slot * heads + head of the first key, or -1
  float k_scale[kTiles16], v_scale[kTiles16];
};

// `x`, which the compiler cannot tell from a new value: what is derived from it is computed where it is used, where it
// would otherwise be kept in registers over whole loops that have none to spare.
template <int kThreads>
__device__ __forceinline__ unsigned recomputed(unsigned x) {
  asm volatile("" : "+v"(x));
  return x % kThreads;
}

template <int kType, int kHd, int kWaves, int kKeys>
__global__ __launch_bounds__(kWaves* kWave) void chunk_kernel(AttentionArgs a) {
  using Q = Query<kType>;
  using T = typename Q::T;
  using Vec = typename Q::Vec;
  constexpr int kThreads = kWaves * kWave;
  constexpr int kRows = 32;                   // of a wave
  constexpr int kSteps = kKeys / 32;
  constexpr int kTiles16 = kKeys / 16;
  constexpr int kDots = kHd / 16;             // mfmas over the head for 32 keys
  constexpr int kOuts = kHd / 32;             // tiles of 32 output columns
  constexpr int kKRow = kHd * 2 + 16;         // bytes between rows in LDS: 16 more, so that 8 lanes' pieces meet no bank twice
  constexpr int kVRow = kKeys * 2 + 16;
  constexpr int kKLoads = kKeys * kHd / 16 / kThreads;  // 16-byte pieces of K a thread
  constexpr int kVCols = 4;                             // adjacent columns of V that a thread transposes
  constexpr int kVThreads = kHd / kVCols;               // for a group of 8 keys
  constexpr int kVLoads = kKeys / 8 * kVThreads / kThreads;
  static_assert(kKLoads * kThreads * 16 == kKeys * kHd && kVLoads * kThreads == kKeys / 8 * kVThreads, "whole pieces");
  __shared__ alignas(16) uint8_t k_lds[2][kKeys * kKRow];
  __shared__ alignas(16) uint8_t v_lds[2][kHd * kVRow];
  __shared__ KeyInfo<kTiles16> info[4];
  __shared__ uint32_t nan_steps[4];           // steps of the pass whose V holds NaN codes, zeros in LDS
  const Fp8Cache& cache = a.cache;
  const int tid = threadIdx.x, lane = tid % kWave, n32 = lane % 32, h = lane / 32;
  const int wave = __builtin_amdgcn_readfirstlane(tid / kWave);
  const int pairs = a.batch.num_seqs * cache.heads;
  const int pair = blockIdx.x % pairs, rest = blockIdx.x / pairs;
  const int tile = a.row_tiles - 1 - rest % a.row_tiles, split = rest / a.row_tiles;  // the longest first
  const int seq = pair / cache.heads, head = pair % cache.heads;
  const int context = context_of(cache, a.batch, seq);
  const int split_passes = a.split_steps * kStep / kKeys, first_pass = split * split_passes;
  if (first_pass * kKeys >= context && split > 0) return;  // the first split also writes the rows that see nothing
  const QueryRows rows = query_rows(a.batch, seq);
  const int num_rows = rows.count * a.per_kv;
  const int32_t* table = a.batch.tables + seq * a.batch.table_stride;
  const int64_t row_bytes = (int64_t)cache.heads * cache.head_dim;

  for (int group_row = tile * kWaves * kRows; group_row < num_rows; group_row += a.row_tiles * kWaves * kRows) {
    const int first_row = group_row + wave * kRows;
    const int group_last = min(group_row + kWaves * kRows, num_rows) - 1;
    const int group_most = context - rows.count + (int)a.per_kv_of(group_last);  // last key that a row of the group sees
    const int group_least = context - rows.count + (int)a.per_kv_of(group_row);
    const int passes = group_most < 0 ? first_pass : min(first_pass + split_passes, group_most / kKeys + 1);
    const int wave_last = min(first_row + kRows, num_rows) - 1;
    const int most = wave_last < first_row ? -1 : context - rows.count + (int)a.per_kv_of(wave_last);
    const int least = context - rows.count + (int)a.per_kv_of(first_row);

    Vec q[kDots];
    const int r = first_row + n32;
    const bool real = r < num_rows;
    const int nth = a.per_kv_of(r), sub = r - nth * a.per_kv;
    const int last = real ? context - rows.count + nth : -1;
    const int out_row = real ? (rows.first + nth) * a.q_heads + head * a.per_kv + sub : -1;
    {
      const unsigned h = recomputed<kThreads>(threadIdx.x) % kWave / 32;
      const T* src = (const T*)a.query + (int64_t)(rows.first + nth) * a.q_stride +
                     (int64_t)(head * a.per_kv + sub) * cache.head_dim;
#pragma unroll
      for (int d = 0; d < kDots; ++d) {
        const int at = d * 16 + h * 8;
        u32x4 w = {0, 0, 0, 0};
        if (real && at < cache.head_dim) w = *reinterpret_cast<const u32x4*>(src + at);
        q[d] = __builtin_bit_cast(Vec, w);
      }
    }
    f32x16 o[kOuts];
#pragma unroll
    for (int d = 0; d < kOuts; ++d)
#pragma unroll
      for (int i = 0; i < 16; ++i) o[d][i] = 0.0f;
    float top = -INFINITY, base = 0.0f, sum = 0.0f;

    // The lookup of a pass's tiles by the first lanes: its blocks two passes before they are needed in LDS, their scales
    // one, so that neither load is waited for.
    int block_id = -1;
    int64_t found_row = -1;
    float found_k = 1.0f, found_v = 1.0f;
    auto find_block = [&](int pass) {
      const unsigned tid = recomputed<kThreads>(threadIdx.x);
      const int key = pass * kKeys + (int)tid * 16;
      block_id = tid < kTiles16 && key < context ? table[cache.block_of(key)] : -1;
    };
    auto find_scales = [&](int pass) {
      const unsigned tid = recomputed<kThreads>(threadIdx.x);
      const int key = pass * kKeys + (int)tid * 16;
      found_row = -1;
      found_k = found_v = 1.0f;
      if (block_id >= 0 && block_id < cache.num_blocks) {
        const int in = key - cache.block_of(key) * cache.block_size;
        const int64_t at = ((int64_t)block_id * (cache.block_size / cache.group) + cache.group_of(in)) * cache.heads + head;
        found_row = ((int64_t)block_id * cache.block_size + in) * cache.heads + head;
        found_k = cache.k_scale[at];
        found_v = cache.v_scale[at];
      }
    };
    auto put_info = [&](int pass) {
      const unsigned tid = recomputed<kThreads>(threadIdx.x);
      if (tid == 0) nan_steps[pass & 3] = 0;
      if (tid < kTiles16) {
        info[pass & 3].row[tid] = found_row;
        info[pass & 3].k_scale[tid] = found_row < 0 ? 1.0f : found_k * a.scale;
        info[pass & 3].v_scale[tid] = found_v;
      }
    };
    u32x4 k_raw[kKLoads];
    uint32_t v_raw[kVLoads][8];
    // Where a wave's lanes all read one 16-key tile, its address and scale are scalars.
    constexpr int kPieces = kHd / 16;  // of a key's row
    static_assert(kWave / kPieces <= 16 && 16 % (kWave / kPieces) == 0, "a wave's pieces of K lie in one tile");
    constexpr bool kVUniform = kVThreads * 2 >= kWave;
    auto load = [&](int pass) {
      const KeyInfo<kTiles16>& from = info[pass & 3];
      const unsigned lane = recomputed<kThreads>(threadIdx.x) % kWave;
#pragma unroll
      for (int i = 0; i < kKLoads; ++i) {
        const int key = (i * kThreads + wave * kWave) / kPieces;  // the wave's first
        const unsigned at = lane % kPieces * 16;
        const int64_t row = scalar(from.row[key / 16]);
        const uint8_t* tile = cache.k + row * cache.head_dim + key % 16 * row_bytes;
        k_raw[i] = u32x4{0, 0, 0, 0};
        if (row >= 0 && (int)at < cache.head_dim)
          k_raw[i] = *reinterpret_cast<const u32x4*>(tile + (lane / kPieces * (unsigned)row_bytes + at));
      }
#pragma unroll
      for (int i = 0; i < kVLoads; ++i) {
        const unsigned group = (i * kThreads + wave * kWave + lane) / kVThreads, at = lane % kVThreads * kVCols;
        const int64_t row = kVUniform ? scalar(from.row[(i * kThreads + wave * kWave) / kVThreads / 2]) : from.row[group / 2];
        const bool there = row >= 0 && (int)at < cache.head_dim;
        const uint8_t* tile = cache.v + row * cache.head_dim;
        const unsigned in_tile = group % 2 * 4 * (unsigned)row_bytes + at;
#pragma unroll
        for (int j = 0; j < 8; ++j) {  // keys 4 h + 0..3, then 8 + 4 h + 0..3
          v_raw[i][j] = 0;
          if (there) v_raw[i][j] = *reinterpret_cast<const uint32_t*>(tile + (j < 4 ? j : j + 4) * row_bytes + in_tile);
        }
      }
    };
    auto convert = [&](int pass) {
      const KeyInfo<kTiles16>& from = info[pass & 3];
      const unsigned lane = recomputed<kThreads>(threadIdx.x) % kWave;
      uint8_t* k_to = k_lds[pass & 1];
      uint8_t* v_to = v_lds[pass & 1];
#pragma unroll
      for (int i = 0; i < kKLoads; ++i) {
        const int key = (i * kThreads + wave * kWave) / kPieces;
        u32x4* to = reinterpret_cast<u32x4*>(k_to + key * kKRow + (lane / kPieces * kKRow + lane % kPieces * 32));
        to[0] = __builtin_bit_cast(u32x4, decode8<Q>(k_raw[i].x, k_raw[i].y));
        to[1] = __builtin_bit_cast(u32x4, decode8<Q>(k_raw[i].z, k_raw[i].w));
      }
      const bool masked = pass * kKeys + kKeys - 1 > group_least;  // some row does not see some key
#pragma unroll
      for (int i = 0; i < kVLoads; ++i) {
        const unsigned group = (i * kThreads + wave * kWave + lane) / kVThreads, col = lane % kVThreads * kVCols;
        const float scale = kVUniform ? scalar(from.v_scale[(i * kThreads + wave * kWave) / kVThreads / 2]) : from.v_scale[group / 2];
        if (masked) {
          uint32_t nan = 0;
#pragma unroll
          for (int j = 0; j < 8; ++j) nan |= nan_bytes(v_raw[i][j]);
          if (nan) {
            atomicOr(&nan_steps[pass & 3], 1u << (group / 4));
#pragma unroll
            for (int j = 0; j < 8; ++j) v_raw[i][j] &= ~((nan_bytes(v_raw[i][j]) >> 7) * 0xFFu);
          }
        }
        uint32_t lo[4], hi[4];
        transpose4(v_raw[i], lo);
        transpose4(v_raw[i] + 4, hi);
        // Column col + d is row col + d of V^T; as col is a multiple of 4, all four have the same row / 16. The XOR spreads
        // neighbouring threads' columns, 4 rows apart, over the banks, and leaves 16 lanes that read adjacent rows on
        // banks of their own.
        uint8_t* to = v_to + col * kVRow + ((group ^ (col / 16 % 4)) * 16);
#pragma unroll
        for (int d = 0; d < 4; ++d) {
          *reinterpret_cast<u32x4*>(to + d * kVRow) = u32x4{pair_scaled(lo[d], scale, false), pair_scaled(lo[d], scale, true),
                                                            pair_scaled(hi[d], scale, false), pair_scaled(hi[d], scale, true)};
        }
      }
    };
    // S^T of a step's 32 keys: K's operand for columns 16 d .. is at k_at(step)[d * 32].
    const int k_lane = n32 * kKRow + h * 16;
    auto k_at = [&](int buffer, int step) { return k_lds[buffer] + step * 32 * kKRow + k_lane; };
    // O^T += V^T P^T. A lane's row d * 32 + n32 holds, of a step's four groups of 8 keys, group 2 i + h in place
    // (2 i + h) ^ (row / 16 % 4).
    const int v_lane = n32 * kVRow + (h ^ (n32 / 16)) * 16;
    auto v_at = [&](int buffer, int step, int i, int d) {
      return v_lds[buffer] + v_lane + step * 64 + (i ^ (d % 2)) * 32 + d * 32 * kVRow;
    };
    // One step: the maximum, this step's P beside the scores of the next (kMore), which replace `x`, and this step's
    // output. Operands are read kAhead products ahead. The scheduling barriers keep it so: left alone, the compiler
    // waits for each operand right before its product.
    float tile_scale = 0.0f;   // lane l: of the pass's tile l
    bool own_scales = false;   // some of V's in the pass are no powers of two
    uint32_t tiles_there = 0;  // bit l: whether tile l is in a block
    constexpr int kAhead = 2;
    Vec k_next[kAhead + 1];
    auto read_k = [&](int buffer, int step, int t) {
      k_next[t % (kAhead + 1)] = *reinterpret_cast<const Vec*>(k_at(buffer, step) + t * 32);
    };
    auto work = [&](auto more, int pass, int step, f32x16& x) {
      constexpr bool kMore = decltype(more)::value;
      constexpr int kTurns = kDots, kEach = 8 / kTurns;
      static_assert(kTurns == 2 * kOuts && kEach * kTurns == 8, "as many products in both");
      const int buffer = pass & 1, key0 = pass * kKeys + step * 32;
      const float scale[2] = {lane_value(tile_scale, step * 2), lane_value(tile_scale, step * 2 + 1)};
      const bool there[2] = {(tiles_there >> (step * 2) & 1) != 0, (tiles_there >> (step * 2 + 1) & 1) != 0};
      if (key0 + 31 > least || !there[0] || !there[1]) {
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const bool see = key0 + 8 * (i / 4) + 4 * h + i % 4 <= last && there[i / 8];
          x[i] = see ? x[i] : -INFINITY;
        }
      }
      float low = x[0], high = x[8];
#pragma unroll
      for (int i = 1; i < 8; ++i) {
        low = fmaxf(low, x[i]);
        high = fmaxf(high, x[8 + i]);
      }
      high = fmaxf(low * scale[0], high * scale[1]);
      if (__any(high > top + 8.0f)) {
        top = fmaxf(top, fmaxf(high, __shfl_xor(high, 32)));
        // A whole number, so that `fade` is a power of two and nothing is rounded. The base only rises, but for the first
        // time, from 0, when nothing has been summed (as above).
        const float now_base = top == -INFINITY ? base : ceilf(top);
        const float fade = __builtin_amdgcn_exp2f(fminf(base - now_base, 0.0f));
        base = now_base;
        sum *= fade;
#pragma unroll
        for (int d = 0; d < kOuts; ++d) o[d] *= fade;
      }
      f32x16 next;
      if (kMore) {
#pragma unroll
        for (int i = 0; i < 16; ++i) next[i] = 0.0f;
      }
      bf16x8 v_next[kAhead + 1];
      auto read_v = [&](int t) {
        v_next[t % (kAhead + 1)] = *reinterpret_cast<const bf16x8*>(v_at(buffer, step, t / kOuts, t % kOuts));
      };
      // P takes what is left of V's scales through its exponents, and its sum goes without.
      float from[2] = {-base, -base}, over[2] = {1.0f, 1.0f}, part[2] = {0.0f, 0.0f};
      if (own_scales) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const float rest = rest_of(scalar(info[pass & 3].v_scale[step * 2 + i]));
          from[i] += __builtin_amdgcn_logf(rest);
          over[i] = __builtin_amdgcn_rcpf(rest);
        }
      }
      u32x4 p[2][2];  // P to bf16, and what the rounding left
      // The wave that has scores and exponentials to issue goes first, so that the SIMD's two waves fall out of step and
      // one's outputs run under the other's exponentials: 551 us in place of 599 for two chunks behind 6-8 K tokens.
      __builtin_amdgcn_s_setprio(1);
#pragma unroll
      for (int t = 0; t < kTurns; ++t) {
        if (kMore) {
          if (t + kAhead < kTurns) read_k(buffer, step + 1, t + kAhead);
          else read_v(t + kAhead - kTurns);
          __builtin_amdgcn_sched_barrier(0);
          next = mfma32<kType>(k_next[t % (kAhead + 1)], q[t], next);
        }
#pragma unroll
        for (int i = t * kEach; i < (t + 1) * kEach; ++i) {
          const float e0 = __builtin_amdgcn_exp2f(__builtin_fmaf(x[2 * i], scale[i / 4], from[i / 4]));
          const float e1 = __builtin_amdgcn_exp2f(__builtin_fmaf(x[2 * i + 1], scale[i / 4], from[i / 4]));
          part[i / 4] += e0 + e1;
          const uint32_t hi = pack_bf16(e0, e1);
          p[0][i / 4][i % 4] = hi;
          p[1][i / 4][i % 4] = pack_bf16(e0 - __uint_as_float(hi << 16), e1 - __uint_as_float(hi & 0xFFFF0000u));
        }
        if (kMore) __builtin_amdgcn_sched_barrier(0);
      }
#pragma unroll
      for (int i = 0; i < 2; ++i) sum = __builtin_fmaf(part[i], over[i], sum);
      if (!kMore) {
#pragma unroll
        for (int t = 0; t < kAhead; ++t) read_v(t);
      }
      __builtin_amdgcn_s_setprio(0);
#pragma unroll
      for (int t = 0; t < kTurns; ++t) {
        if (t + kAhead < kTurns) read_v(t + kAhead);
        else if (kMore) read_k(buffer, step + 2 < kSteps ? step + 2 : step, t + kAhead - kTurns);  // for the step after, if any
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int k = 0; k < 2; ++k)
          o[t % kOuts] = mfma32<KVX_DTYPE_BF16>(v_next[t % (kAhead + 1)], __builtin_bit_cast(bf16x8, p[k][t / kOuts]),
                                               o[t % kOuts]);
      }
      if (kMore) x = next;
    };

    if (passes > first_pass) {
      find_block(first_pass);
      find_scales(first_pass);
      put_info(first_pass);
      find_block(first_pass + 1);
      find_scales(first_pass + 1);
      put_info(first_pass + 1);
      find_block(first_pass + 2);
      __syncthreads();
      load(first_pass);
      convert(first_pass);
    }
    __syncthreads();
    for (int pass = first_pass; pass < passes; ++pass) {
      const int buffer = pass & 1;
      const KeyInfo<kTiles16>& now = info[pass & 3];
      find_scales(pass + 2);
      find_block(pass + 3);
      if (pass + 1 < passes) load(pass + 1);
      const int steps = most < pass * kKeys ? 0 : min(kSteps, (most - pass * kKeys) / 32 + 1);
      if (steps > 0) {
        f32x16 x;
#pragma unroll
        for (int i = 0; i < 16; ++i) x[i] = 0.0f;
#pragma unroll
        for (int d = 0; d < kDots; ++d) x = mfma32<kType>(*reinterpret_cast<const Vec*>(k_at(buffer, 0) + d * 32), q[d], x);
        tile_scale = now.k_scale[lane % kTiles16];
        own_scales = __any(rest_of(now.v_scale[lane % kTiles16]) != 1.0f);
        tiles_there = (uint32_t)__ballot(now.row[lane % kTiles16] >= 0);
#pragma unroll
        for (int t = 0; t < kAhead; ++t) read_k(buffer, 1, t);
#pragma unroll 1
        for (int step = 0; step < steps - 1; ++step) work(std::true_type{}, pass, step, x);
        work(std::false_type{}, pass, steps - 1, x);
        const uint32_t nan = nan_steps[pass & 3];
        if (nan) {
          // Rows that see a NaN code in a pass that is masked for others: its columns become NaN.
          const unsigned lane = recomputed<kThreads>(threadIdx.x) % kWave, n32 = lane % 32, h = lane / 32;
#pragma unroll 1
          for (int step = 0; step < steps; ++step) {
            if (!(nan >> step & 1)) continue;
#pragma unroll 1
            for (int i = 0; i < 2; ++i) {
              const int64_t row = now.row[step * 2 + i];
              if (row < 0) continue;
              u32x4 seen;
#pragma unroll
              for (int j = 0; j < 4; ++j) {
                const int key = pass * kKeys + step * 32 + i * 16 + 4 * h + (j < 2 ? 2 * j : 4 + 2 * j);
                seen[j] = (key <= last ? 0x3F80u : 0u) | (key + 1 <= last ? 0x3F800000u : 0u);
              }
#pragma unroll
              for (int d = 0; d < kOuts; ++d) {
                const int col = d * 32 + n32;
                u32x4 is_nan = {0, 0, 0, 0};
                if (col < cache.head_dim) {
#pragma unroll
                  for (int j = 0; j < 8; ++j) {
                    const int key = 4 * h + (j < 4 ? j : j + 4);
                    const uint8_t code = cache.v[row * cache.head_dim + key * row_bytes + col];
                    is_nan[j / 2] |= (code & 0x7F) == 0x7F ? (j % 2 ? 0x3F800000u : 0x3F80u) : 0u;
                  }
                }
                f32x16 hit;
#pragma unroll
                for (int j = 0; j < 16; ++j) hit[j] = 0.0f;
                hit = mfma32<KVX_DTYPE_BF16>(__builtin_bit_cast(bf16x8, is_nan), __builtin_bit_cast(bf16x8, seen), hit);
#pragma unroll
                for (int j = 0; j < 16; ++j) o[d][j] += hit[j] > 0.0f ? NAN : 0.0f;
              }
            }
          }
        }
      }
      if (pass + 1 < passes) convert(pass + 1);
      put_info(pass + 2);
      __syncthreads();
    }

    const float total = sum + __shfl_xor(sum, 32);
    if (out_row >= 0) {
      const unsigned h = recomputed<kThreads>(threadIdx.x) % kWave / 32;
#pragma unroll
      for (int d = 0; d < kOuts; ++d)
#pragma unroll
        for (int i = 0; i < 16; i += 4) {
          const int col = d * 32 + 8 * (i / 4) + 4 * h;
          if (col < cache.head_dim)
            write_rows<T>(a, split, out_row, col, top == -INFINITY ? -INFINITY : base, total,
                          f32x4{o[d][i], o[d][i + 1], o[d][i + 2], o[d][i + 3]});
        }
    }
    __syncthreads();  // before the next rows' passes write to LDS
  }
}

// Joins the splits: a workgroup per query row, its threads over 4 columns of one split after another. All parts are
// asked for at once, with the sums that weigh them: waited for by turns, 128 splits took 10 us.
constexpr int kMaxSplits = 128;
template <typename T, int kJoinThreads>
__global__ __launch_bounds__(kJoinThreads) void join_kernel(AttentionArgs a) {
  constexpr int kHeld = 4, kJoinWaves = kJoinThreads / kWave;
  __shared__ float fades[kMaxSplits];
  __shared__ float wave_top[kJoinWaves], wave_sum[kJoinWaves];
  __shared__ f32x4 parts[kJoinThreads];
  const int tid = threadIdx.x, seq = blockIdx.y, hd = a.cache.head_dim;
  const QueryRows rows = query_rows(a.batch, seq);
  const int context = context_of(a.cache, a.batch, seq);
  const int steps = (context + kStep - 1) / kStep, used = steps <= a.split_steps ? 1 : (steps - 1) / a.split_steps + 1;
  const int64_t total_rows = (int64_t)a.batch.num_tokens * a.q_heads;
  const float* stats = a.partial + a.splits * total_rows * hd;
  const int columns = hd <= 64 ? 16 : hd <= 128 ? 32 : 64, groups = kJoinThreads / columns;  // threads of 4 columns
  const int col = min(tid % columns * 4, hd - 4), group = tid / columns;
  for (int r = blockIdx.x; r < rows.count * a.q_heads; r += gridDim.x) {
    const int64_t row = (int64_t)rows.first * a.q_heads + r;
    const float* from = a.partial + row * hd + col;
    const f32x2 mine = *reinterpret_cast<const f32x2*>(stats + ((tid < used ? tid : 0) * total_rows + row) * 2);
    f32x4 part[kHeld];
#pragma unroll
    for (int i = 0; i < kHeld; ++i) {
      const int s = group + i * groups;
      part[i] = *reinterpret_cast<const f32x4*>(from + (s < used ? s : 0) * total_rows * hd);
    }
    const float my_sum = tid < used ? mine.y : 0.0f;
    float top = tid < used ? mine.x : -INFINITY;
#pragma unroll
    for (int d = 1; d < kWave; d <<= 1) top = fmaxf(top, __shfl_xor(top, d));
    if (tid % kWave == 0) wave_top[tid / kWave] = top;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kJoinWaves; ++w) top = fmaxf(top, wave_top[w]);
    const float fade = my_sum == 0.0f ? 0.0f : __builtin_amdgcn_exp2f(mine.x - top);
    float sum = my_sum == 0.0f ? 0.0f : my_sum * fade;
    if (tid < used) fades[tid] = fade;
#pragma unroll
    for (int d = 1; d < kWave; d <<= 1) sum += __shfl_xor(sum, d);
    if (tid % kWave == 0) wave_sum[tid / kWave] = sum;
    __syncthreads();
    sum = 0.0f;
#pragma unroll
    for (int w = 0; w < kJoinWaves; ++w) sum += wave_sum[w];
    f32x4 y = {0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < kHeld; ++i) {
      const int s = group + i * groups;
      const float times = s < used ? fades[s] : 0.0f;
      if (times != 0.0f) y += part[i] * times;  // a part of sum 0 may hold anything
    }
    for (int s = group + kHeld * groups; s < used; s += groups) {
      const f32x4 more = *reinterpret_cast<const f32x4*>(from + s * total_rows * hd);
      if (fades[s] != 0.0f) y += more * fades[s];
    }
    parts[tid] = y;
    __syncthreads();
    if (group == 0 && tid % columns * 4 < hd) {
      for (int i = 1; i < groups && i < used; ++i) y += parts[i * columns + tid];
      const float inverse = sum == 0.0f ? 0.0f : 1.0f / sum;
      alignas(8) T out[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) out[j] = (T)(sum == 0.0f ? 0.0f : y[j] * inverse);
      *reinterpret_cast<u32x2*>((T*)a.out + row * hd + col) = *reinterpret_cast<const u32x2*>(out);
      if (a.lse && col == 0) a.lse[row] = sum == 0.0f ? -INFINITY : (top + log2f(sum)) * 0.69314718055994531f;
    }
    __syncthreads();
  }
}

// ---------------------------------------------------------------------------
// The weight of each cached token: out = weights + the sum over the query rows
// that see it of exp(score - lse). A key belongs to one wave, which passes over
// all query rows in order: no atomics, one order of the sums.

// The query row r of a (sequence, KV head): its address, its last key, and its lse over log(2); infinity, which makes
// every weight 0, where there is no such row or it sees nothing.
template <typename T>
struct WeightRow {
  const T* query;
  float lse;
  int last;
};
template <typename T>
__device__ __forceinline__ WeightRow<T> weight_row(const WeightsArgs& a, const QueryRows& rows, int context, int head,
                                                   int r) {
  const bool real = r < rows.count * a.per_kv;
  const int nth = real ? (int)a.per_kv_of(r) : 0, q_head = head * a.per_kv + (real ? r - nth * a.per_kv : 0);
  WeightRow<T> row;
  row.query = (const T*)a.query + (int64_t)(rows.first + nth) * a.q_stride + (int64_t)q_head * a.cache.head_dim;
  row.last = real ? context - rows.count + nth : -1;
  row.lse = a.lse[real ? (int64_t)(rows.first + nth) * a.q_heads + q_head : 0];
  if (!real) row.lse = -INFINITY;
  row.lse = row.lse == -INFINITY ? INFINITY : row.lse * 1.4426950408889634f;
  return row;
}

// 16 adjacent keys' lookup, a lane for each.
struct KeyTile {
  int64_t row;  // slot * heads + head of the first key, or -1
  float scale;  // as loaded: multiplied at once, it would hold up K's loads
};
__device__ __forceinline__ KeyTile key_tile(const WeightsArgs& a, const int32_t* table, int context, int head, int key) {
  const Fp8Cache& cache = a.cache;
  KeyTile t = {-1, 0.0f};
  if (key < context) {
    const int block = cache.block_of(key), in = key - block * cache.block_size;
    const int id = table[block];
    if (id >= 0 && id < cache.num_blocks) {
      t.row = ((int64_t)id * cache.block_size + in) * cache.heads + head;
      t.scale = cache.k_scale[((int64_t)id * (cache.block_size / cache.group) + cache.group_of(in)) * cache.heads + head];
    }
  }
  return t;
}
// The sum over the 16 lanes of a row, in all of them.
__device__ __forceinline__ float sum16(float x) {
  x += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), 0x128, 0xF, 0xF, false));  // row_ror:8
  x += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), 0x124, 0xF, 0xF, false));
  x += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), 0x122, 0xF, 0xF, false));
  return x + __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), 0x121, 0xF, 0xF, false));
}

// Few query rows: bound by the bytes of K. A wave asks for kTiles * 16 keys at
// once; its query rows come straight from memory, 16 at a time. (Several turns
// of so many keys, each turn's asked for during the one before, took 32 us in
// place of 27 for 16 contexts of 2-8 K tokens, whose waves are few, and 142 in
// place of 144 for 64 of 32 K tokens on 2 heads.)
__device__ __forceinline__ void copy_weights(const WeightsArgs& a, int64_t at, int count, int lane) {  // nothing is added
  if (a.weights == a.out) return;
  for (int i = lane; i < count; i += kWave) a.out[at + i] = a.weights ? a.weights[at + i] : 0.0f;
}

template <int kType, int kHd, int kTiles>
__global__ __launch_bounds__(kThreads) void weights_few_kernel(WeightsArgs a) {
  using Q = Query<kType>;
  using T = typename Q::T;
  using Vec = typename Q::Vec;
  constexpr int kChunks = kHd / 64;
  const Fp8Cache& cache = a.cache;
  const int lane = threadIdx.x % kWave, c = lane % 16, g = lane / 16;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const Slice slice = slice_of(blockIdx.x, cache.heads);
  const int seq = slice.unit % a.batch.num_seqs, head = slice.head, pair = seq * cache.heads + head;
  const int key0 = (slice.unit / a.batch.num_seqs * kWaves + wave) * kTiles * 16;
  if (key0 >= a.width) return;
  const int context = context_of(cache, a.batch, seq);
  const int64_t base = (int64_t)pair * a.width;
  if (key0 >= context) return copy_weights(a, base + key0, min(kTiles * 16, a.width - key0), lane);
  const QueryRows rows = query_rows(a.batch, seq);
  const int num_rows = rows.count * a.per_kv;
  if (num_rows == 0) return copy_weights(a, base + key0, min(kTiles * 16, a.width - key0), lane);
  WeightRow<T> row = weight_row<T>(a, rows, context, head, c);
  const KeyTile mine = key_tile(a, a.batch.tables + seq * a.batch.table_stride, lane < kTiles ? context : 0, head,
                                key0 + lane * 16);
  const int32_t k_lane = c * cache.heads * cache.head_dim + g * 16;
  u32x4 k[kTiles][kChunks];
  float scale[kTiles];
#pragma unroll
  for (int t = 0; t < kTiles; ++t) {
    const int64_t at = lane_value(mine.row, t);
    scale[t] = lane_value(mine.scale, t) * a.scale;
#pragma unroll
    for (int i = 0; i < kChunks; ++i) {
      k[t][i] = u32x4{0, 0, 0, 0};
      if (at >= 0 && i * 64 + g * 16 < cache.head_dim)
        k[t][i] = *reinterpret_cast<const u32x4*>(cache.k + at * cache.head_dim + (k_lane + i * 64));
    }
  }
  // Lane (c, g) writes keys 4 g + i of tile c.
  float before[4] = {0, 0, 0, 0}, total[kTiles][4];
  const int my_key = key0 + c * 16 + 4 * g;
  if (a.weights && c < kTiles) {
#pragma unroll
    for (int i = 0; i < 4; ++i) before[i] = a.weights[base + (my_key + i < a.width ? my_key + i : 0)];
  }
#pragma unroll
  for (int t = 0; t < kTiles; ++t)
#pragma unroll
    for (int i = 0; i < 4; ++i) total[t][i] = 0.0f;
  for (int row0 = 0; row0 < num_rows; row0 += 16) {
    if (row0 > 0) row = weight_row<T>(a, rows, context, head, row0 + c);
    Vec q[2 * kChunks];
#pragma unroll
    for (int i = 0; i < kChunks; ++i) {
      const int at = i * 64 + g * 16;
      u32x4 lo = {0, 0, 0, 0}, hi = {0, 0, 0, 0};
      if (at < cache.head_dim) {
        lo = *reinterpret_cast<const u32x4*>(row.query + at);
        hi = *reinterpret_cast<const u32x4*>(row.query + at + 8);
      }
      q[2 * i] = __builtin_bit_cast(Vec, lo);
      q[2 * i + 1] = __builtin_bit_cast(Vec, hi);
    }
#pragma unroll
    for (int t = 0; t < kTiles; ++t) {
      f32x4 s = {0, 0, 0, 0};
#pragma unroll
      for (int i = 0; i < kChunks; ++i) {
        s = Q::mfma(decode8<Q>(k[t][i].x, k[t][i].y), q[2 * i], s);
        s = Q::mfma(decode8<Q>(k[t][i].z, k[t][i].w), q[2 * i + 1], s);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float p = __builtin_amdgcn_exp2f(s[i] * scale[t] - row.lse);
        total[t][i] += key0 + t * 16 + 4 * g + i <= row.last ? p : 0.0f;
      }
    }
  }
  float added[4] = {0, 0, 0, 0};
#pragma unroll
  for (int t = 0; t < kTiles; ++t) {
    const bool there = lane_value(mine.row, t) >= 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float sum = sum16(total[t][i]);
      added[i] = there && c == t ? sum : added[i];
    }
  }
  if (c < kTiles) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (my_key + i < a.width) a.out[base + my_key + i] = before[i] + added[i];
  }
}

// Many query rows: bound by the exponentials and the matrix cores. A wave keeps
// 32 keys' K as operands; the workgroup's waves share the query rows, 64 at a
// time, through LDS, and a wave computes the scores of the next 32 of them under
// the exponentials of these. 1,023 rows of 32 heads of 128 over 8 K tokens: 102 us.
template <int kType, int kHd>
__global__ __launch_bounds__(kThreads, kHd < 256 ? 3 : 2) void weights_many_kernel(WeightsArgs a) {
  using Q = Query<kType>;
  using T = typename Q::T;
  using Vec = typename Q::Vec;
  constexpr int kDots = kHd / 16;
  constexpr int kRowsHeld = 64;
  constexpr int kPitch = kHd * 2 + 16;
  constexpr int kLoads = kRowsHeld * kHd / 8 / kThreads;  // 16-byte pieces of the rows a thread
  __shared__ alignas(16) uint8_t q_lds[2][kRowsHeld * kPitch];
  __shared__ float lse_lds[2][kRowsHeld];
  __shared__ int last_lds[2][kRowsHeld];
  const Fp8Cache& cache = a.cache;
  const int tid = threadIdx.x, lane = tid % kWave, n32 = lane % 32, h = lane / 32;
  const int wave = __builtin_amdgcn_readfirstlane(tid / kWave);
  const int pairs = a.batch.num_seqs * cache.heads;
  const int pair = blockIdx.x % pairs, seq = pair / cache.heads, head = pair % cache.heads;
  const int group0 = (blockIdx.x / pairs) * kWaves * 32, key0 = group0 + wave * 32;
  const int context = context_of(cache, a.batch, seq);
  const int64_t base = (int64_t)pair * a.width;
  const QueryRows rows = query_rows(a.batch, seq);
  const int num_rows = group0 < context ? rows.count * a.per_kv : 0;

  const KeyTile mine = key_tile(a, a.batch.tables + seq * a.batch.table_stride, lane < 2 ? context : 0, head,
                                key0 + lane * 16);
  const bool there[2] = {lane_value(mine.row, 0) >= 0, lane_value(mine.row, 1) >= 0};
  const float scale[2] = {lane_value(mine.scale, 0) * a.scale, lane_value(mine.scale, 1) * a.scale};
  // K: lane (n, h) holds columns 16 d + 8 h .. of key n.
  Vec k[kDots];
  {
    const int64_t row = n32 < 16 ? lane_value(mine.row, 0) : lane_value(mine.row, 1);
    const uint8_t* src = cache.k + (row + (int64_t)(n32 % 16) * cache.heads) * cache.head_dim + h * 8;
    u32x2 raw[kDots];
#pragma unroll
    for (int d = 0; d < kDots; ++d) {
      raw[d] = u32x2{0, 0};
      if (row >= 0 && d * 16 < cache.head_dim) raw[d] = *reinterpret_cast<const u32x2*>(src + d * 16);
    }
#pragma unroll
    for (int d = 0; d < kDots; ++d) k[d] = decode8<Q>(raw[d].x, raw[d].y);
  }
  float total[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) total[i] = 0.0f;

  // Rows before the first that sees a key of the workgroup are left out.
  const int first_query = num_rows > 0 ? group0 - (context - rows.count) : 0;
  const int first_row = first_query > 0 ? first_query * a.per_kv / kRowsHeld * kRowsHeld : 0;
  u32x4 piece[kLoads];
  float lse = 0.0f;
  int last = -1;
  auto load = [&](int row0) {
    constexpr int kPieces = kHd / 8;
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      const int r = row0 + (i * kThreads + tid) / kPieces, at = (i * kThreads + tid) % kPieces * 8;
      const bool real = r < num_rows && at < cache.head_dim;
      const int nth = real ? (int)a.per_kv_of(r) : 0, sub = real ? r - nth * a.per_kv : 0;
      piece[i] = u32x4{0, 0, 0, 0};
      if (real)
        piece[i] = *reinterpret_cast<const u32x4*>((const T*)a.query + (int64_t)(rows.first + nth) * a.q_stride +
                                                   (int64_t)(head * a.per_kv + sub) * cache.head_dim + at);
    }
    if (tid < kRowsHeld) {
      const WeightRow<T> row = weight_row<T>(a, rows, context, head, row0 + tid < num_rows ? row0 + tid : INT32_MAX);
      lse = row.lse;
      last = row.last;
    }
  };
  auto put = [&](int buffer) {
    constexpr int kPieces = kHd / 8;
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      const int r = (i * kThreads + tid) / kPieces, at = (i * kThreads + tid) % kPieces * 16;
      *reinterpret_cast<u32x4*>(q_lds[buffer] + r * kPitch + at) = piece[i];
    }
    if (tid < kRowsHeld) {
      lse_lds[buffer][tid] = lse;
      last_lds[buffer][tid] = last;
    }
  };
  auto scores = [&](int buffer, int half) {
    const uint8_t* from = q_lds[buffer] + (half * 32 + n32) * kPitch + h * 16;
    f32x16 s;
#pragma unroll
    for (int i = 0; i < 16; ++i) s[i] = 0.0f;
#pragma unroll
    for (int d = 0; d < kDots; ++d) s = mfma32<kType>(k[d], *reinterpret_cast<const Vec*>(from + d * 32), s);
    return s;
  };
  auto add = [&](float row_lse, int row_last, const f32x16& s) {
    if (__any(key0 + 31 > row_last)) {
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(s[i], scale[i / 8], -row_lse));
        total[i] += key0 + 8 * (i / 4) + 4 * h + i % 4 <= row_last ? p : 0.0f;
      }
    } else {
#pragma unroll
      for (int i = 0; i < 16; ++i) total[i] += __builtin_amdgcn_exp2f(__builtin_fmaf(s[i], scale[i / 8], -row_lse));
    }
  };
  if (first_row < num_rows) {
    load(first_row);
    put(0);
    __syncthreads();
    int buffer = 0;
    f32x16 s = scores(0, 0);
    for (int row0 = first_row; row0 < num_rows; row0 += kRowsHeld, buffer ^= 1) {
      const bool more = row0 + kRowsHeld < num_rows;
      if (more) load(row0 + kRowsHeld);
      const f32x16 second = scores(buffer, 1);
      add(lse_lds[buffer][n32], last_lds[buffer][n32], s);
      if (more) put(buffer ^ 1);
      // Read before the barrier, behind which the next turn's rows but one may replace them.
      const float second_lse = lse_lds[buffer][32 + n32];
      const int second_last = last_lds[buffer][32 + n32];
      __syncthreads();
      if (more) s = scores(buffer ^ 1, 0);
      add(second_lse, second_last, second);
    }
  }
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    float sum = sum16(total[i]);
    sum += __shfl_xor(sum, 16);
    const int key = key0 + 8 * (i / 4) + 4 * h + i % 4;
    if (n32 == i && key < a.width)
      a.out[base + key] = (a.weights ? a.weights[base + key] : 0.0f) + (there[i / 8] && key < context ? sum : 0.0f);
  }
}

int padded_head(int head_dim) { return head_dim <= 64 ? 64 : head_dim <= 128 ? 128 : 256; }

// Query rows of one (sequence, KV head) up to which the few-rows kernel runs (16 contexts of 4 K tokens on 8 heads, 32
// rows: 65 us, the chunk kernel 83; 48 rows: 150 and 87).
constexpr int kFewRows = 32;
int few_tiles(int64_t rows, int padded) { return rows <= 16 || padded == 256 ? 1 : 2; }
constexpr int kChunkWaves = 8;
constexpr int chunk_keys(int padded) { return 16384 / padded; }

template <int kType, int kHd, int kTiles>
hipError_t few_rows_of(const AttentionArgs& a, hipStream_t stream) {
  const int64_t grid = slices_grid((int64_t)a.batch.num_seqs * a.splits * a.row_tiles, a.cache.heads);
  few_rows_kernel<kType, kHd, kTiles><<<dim3((unsigned)grid), dim3(kThreads), 0, stream>>>(a);
  return hipGetLastError();
}

template <int kType, int kHd>
hipError_t attention_typed(const AttentionArgs& a, hipStream_t stream) {
  using T = typename Query<kType>::T;
  const int64_t rows = (int64_t)a.batch.max_seqlen * a.per_kv;
  hipError_t err;
  bool few = rows <= kFewRows;
  if constexpr (kHd == 256) few = true;
  if (few) {
    if (few_tiles(rows, kHd) == 1) err = few_rows_of<kType, kHd, 1>(a, stream);
    else if constexpr (kHd < 256) err = few_rows_of<kType, kHd, 2>(a, stream);
    else err = hipErrorInvalidValue;
  } else {
    if constexpr (kHd < 256) {
      const int64_t grid = (int64_t)a.batch.num_seqs * a.cache.heads * a.splits * a.row_tiles;
      chunk_kernel<kType, kHd, kChunkWaves, chunk_keys(kHd)>
          <<<dim3((unsigned)grid), dim3(kChunkWaves * kWave), 0, stream>>>(a);
      err = hipGetLastError();
    } else {
      err = hipErrorInvalidValue;
    }
  }
  if (err != hipSuccess || a.splits == 1) return err;
  const int64_t rows_joined = std::min<int64_t>((int64_t)a.batch.max_seqlen * a.q_heads, 1 << 20);  // others follow these
  const dim3 grid((unsigned)rows_joined, (unsigned)a.batch.num_seqs);
  if (a.splits <= 16) join_kernel<T, 256><<<grid, dim3(256), 0, stream>>>(a);
  else join_kernel<T, 1024><<<grid, dim3(1024), 0, stream>>>(a);
  return hipGetLastError();
}

template <int kType>
hipError_t attention_sized(const AttentionArgs& a, hipStream_t stream) {
  switch (padded_head(a.cache.head_dim)) {
    case 64: return attention_typed<kType, 64>(a, stream);
    case 128: return attention_typed<kType, 128>(a, stream);
    default: return attention_typed<kType, 256>(a, stream);
  }
}

// Query rows of one (sequence, KV head) up to which the few-rows kernel takes the weights (16 contexts of 4 K tokens on 8
// heads, 128 rows: 47 us, the other 52; 256 rows: 76 and 67; on one head 9.6 and 10.1; 14.7 and 13.3).
constexpr int kFewWeightRows = 128;
template <int kType, int kHd>
hipError_t weights_typed(const WeightsArgs& a, hipStream_t stream) {
  const int64_t pairs = (int64_t)a.batch.num_seqs * a.cache.heads;
  if ((int64_t)a.batch.max_seqlen * a.per_kv <= kFewWeightRows) {
    constexpr int kTiles = kHd == 256 ? 2 : 4, kKeys = kWaves * kTiles * 16;
    const dim3 grid((unsigned)slices_grid((int64_t)a.batch.num_seqs * ((a.width + kKeys - 1) / kKeys), a.cache.heads));
    weights_few_kernel<kType, kHd, kTiles><<<grid, dim3(kThreads), 0, stream>>>(a);
  } else {
    constexpr int kKeys = kWaves * 32;
    const dim3 grid((unsigned)(pairs * ((a.width + kKeys - 1) / kKeys)));
    weights_many_kernel<kType, kHd><<<grid, dim3(kThreads), 0, stream>>>(a);
  }
  return hipGetLastError();
}

template <int kType>
hipError_t weights_sized(const WeightsArgs& a, hipStream_t stream) {
  switch (padded_head(a.cache.head_dim)) {
    case 64: return weights_typed<kType, 64>(a, stream);
    case 128: return weights_typed<kType, 128>(a, stream);
    default: return weights_typed<kType, 256>(a, stream);
  }
}

}  // namespace

constexpr int64_t kMostTiles = 1 << 18;
AttentionPlan attention_plan(const Fp8Cache& c, const PagedBatch& b, int32_t q_heads) {
  const int64_t rows = (int64_t)b.max_seqlen * (q_heads / c.heads);
  const bool few = rows <= kFewRows || padded_head(c.head_dim) == 256;
  const int64_t tile_rows = few ? 16 * few_tiles(rows, padded_head(c.head_dim)) : 32 * kChunkWaves;
  AttentionPlan plan;
  // As many tiles of rows as the longest sequence may have, but no more workgroups than keep 256 CUs busy for a thousand
  // rounds: max_seqlen may be all rows of a call of many short sequences, and workgroups take the tiles behind theirs.
  const int64_t room = std::max<int64_t>(kMostTiles / ((int64_t)b.num_seqs * c.heads), 1);
  plan.row_tiles = (int32_t)std::min((rows + tile_rows - 1) / tile_rows, room);
  const int64_t groups = (int64_t)b.num_seqs * c.heads * plan.row_tiles;
  const int64_t steps = ((int64_t)b.table_width * c.block_size + kStep - 1) / kStep;
  // Split the keys while there are too few workgroups to fill the chip, each keeping 256 keys or more (1,024: 16 chunks of
  // 6 tokens and 8 query heads over 4 K 40 us, now 20). Chunks: up to one workgroup a CU, which is what one has LDS
  // for (up to two, 256 of a chunk of 2,048 tokens over 8 K took 472 us, now 360; 160 of 1,280 over 4 K 204 and 162).
  // Few rows: with few (sequence, KV head) pairs, one workgroup a CU, as the join takes its time for each split (8 pairs of
  // 32 K tokens in 128 / 64 / 32 / 16 splits 23.7 / 21.6 / 19.8 / 25.7 us); with many, so many that contexts of unlike
  // lengths even out (61 of 300 to 8,192 tokens on 8 heads in 4 / 8 splits 114 / 105; 2,048 pairs of 2 K in 2 / 1 219 /
  // 193). About the borders, with contexts all of one length and 256 / 1,024 / 4,096 workgroups: 15 pairs of 8 K 13.3 / 14.5
  // / 14.5 us, 16 13.4 / 14.6 / 14.6, 32 18.6 / 23.7 / 23.6, 192 94 / 79 / 85, 240 97 / 100 / 103, 320 131 / 129 / 130;
  // 1,920 pairs of 2 K 185 / 186 / 206, 2,560 240 in each. Where all are as long, fewer splits would mostly do.
  const int64_t want = !few || groups < 16 ? 256 : groups < 256 ? 1024 : groups < 2048 ? 4096 : groups;
  const int64_t unit = few ? 8 : chunk_keys(padded_head(c.head_dim)) / kStep, least = 8;
  int64_t splits = want / groups;
  if (splits > steps / least) splits = steps / least;
  splits = splits < 1 ? 1 : splits > kMaxSplits ? kMaxSplits : splits;
  int64_t per = (steps + splits - 1) / splits;
  per = (per + unit - 1) / unit * unit;
  if (per < unit) per = unit;
  plan.split_steps = (int32_t)per;
  plan.splits = steps == 0 ? 1 : (int32_t)((steps + per - 1) / per);
  return plan;
}

int64_t attention_workspace(int32_t splits, int64_t num_tokens, int32_t q_heads, int32_t head_dim) {
  return splits <= 1 ? 0 : (int64_t)splits * num_tokens * q_heads * (head_dim + 2) * (int64_t)sizeof(float);
}

hipError_t launch_attention(const AttentionArgs& a, int32_t dtype, hipStream_t stream) {
  return dtype == KVX_DTYPE_BF16 ? attention_sized<KVX_DTYPE_BF16>(a, stream)
                                 : attention_sized<KVX_DTYPE_FP16>(a, stream);
}

hipError_t launch_attention_weights(const WeightsArgs& a, int32_t dtype, hipStream_t stream) {
  return dtype == KVX_DTYPE_BF16 ? weights_sized<KVX_DTYPE_BF16>(a, stream) : weights_sized<KVX_DTYPE_FP16>(a, stream);
}

}  // namespace kvx
