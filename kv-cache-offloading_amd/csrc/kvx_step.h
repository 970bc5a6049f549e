// Internal declarations of the operators around an e4m3 KV cache: what the C
// ABI layer (kvx_step_capi.hip) hands to the kernels, checked.
#pragma once

#include "kvx_internal.h"

namespace kvx {

typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));
typedef unsigned int u32x2 __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

constexpr int kMaxGroup = 1024;    // tokens under one scale
constexpr int kMaxHeadDim = 256;
constexpr int kWave = 64;

// A layer's e4m3 cache: slot s of head h is the row codes + (s * heads + h) *
// head_dim, its scale the element (s / group) * heads + h.
struct Fp8Cache {
  uint8_t* k;
  uint8_t* v;
  float* k_scale;
  float* v_scale;
  int32_t num_blocks, block_size, group, heads, head_dim;
  FastDiv block_of, group_of;  // position -> block of a sequence; slot or offset in a block -> group
};

// The sequences of a call: their blocks, their lengths, and which of the
// call's rows are whose queries (row b is sequence b's where cu_seqlens is NULL).
struct PagedBatch {
  const int32_t* tables;
  const int32_t* context_lens;
  const int32_t* cu_seqlens;
  int64_t table_stride;
  int32_t table_width, num_seqs, max_seqlen;
  int32_t num_tokens;
};

struct RotaryArgs {
  const void *query, *key;
  void *query_out, *key_out;
  int64_t q_stride, k_stride, q_out_stride, k_out_stride;  // elements between tokens
  const void* positions;
  const double* frequencies;
  int64_t num_tokens;
  int32_t q_heads, k_heads, head_dim, rotary_dim;
  int32_t long_positions, interleaved;
  float magnitude;
};

struct AttentionArgs {
  Fp8Cache cache;
  PagedBatch batch;
  const void* query;
  int64_t q_stride;  // elements between tokens
  int32_t q_heads, per_kv;  // query heads, and those of one KV head
  FastDiv per_kv_of;
  float scale;  // softmax scale * log2(e)
  void* out;
  float* lse;       // may be NULL
  float* partial;   // workspace (splits > 1): [splits][num_tokens * q_heads][head_dim], then the maxima and sums
  int32_t splits, split_steps;  // of the keys, and steps of 32 keys of each
  int32_t row_tiles;            // a launch's, of a sequence's query rows
};

// How a call is cut into workgroups, by its sizes alone.
struct AttentionPlan {
  int32_t splits, split_steps, row_tiles;
};

struct WeightsArgs {
  Fp8Cache cache;
  PagedBatch batch;
  const void* query;
  int64_t q_stride;
  int32_t q_heads, per_kv;
  FastDiv per_kv_of;
  float scale;
  const float* lse;
  const float* weights;  // may be NULL (zeros)
  float* out;
  int32_t width;         // weights of one (sequence, KV head)
};

hipError_t launch_rotary(const RotaryArgs& a, int32_t dtype, hipStream_t stream);
hipError_t launch_store_fp8(const Fp8Cache& c, const void* key, int64_t key_stride, const void* value,
                            int64_t value_stride, int32_t dtype, const int32_t* slots, int32_t num_tokens,
                            hipStream_t stream);
// What launch_attention takes in its arguments, and the workspace bytes that so many splits need (0 for one).
AttentionPlan attention_plan(const Fp8Cache& c, const PagedBatch& b, int32_t q_heads);
int64_t attention_workspace(int32_t splits, int64_t num_tokens, int32_t q_heads, int32_t head_dim);
hipError_t launch_attention(const AttentionArgs& a, int32_t dtype, hipStream_t stream);
hipError_t launch_attention_weights(const WeightsArgs& a, int32_t dtype, hipStream_t stream);
hipError_t launch_select(const float* weights, int32_t rows, int32_t heads, int32_t width, const int32_t* context_lens,
                         int32_t keep, int32_t recent, int32_t* indices, int32_t* counts, float* kept,
                         hipStream_t stream);
hipError_t launch_compact(const Fp8Cache& c, const PagedBatch& from, const int32_t* indices, const int32_t* counts,
                          int32_t keep, const int32_t* to_tables, int64_t to_stride, int32_t to_width,
                          hipStream_t stream);

// ---------------------------------------------------------------------------
// Device helpers

// The least power of two s >= 2^-100 with 2^kUp amax / s <= 448 = 0.875 * 2^9, for a
// finite amax >= 0. A power of two costs e4m3, itself a floating format, no
// precision, makes x / s and the requantisation of codes exact but for e4m3's
// own rounding, and lets no order of writes change a group's scale.
template <int kUp = 0>
__device__ __forceinline__ float scale_for(float amax) {
  const uint32_t u = __float_as_uint(amax);
  int e = (int)(u >> 23) - 127 - 8 + kUp + ((u & 0x7FFFFFu) > 0x600000u ? 1 : 0);
  e = e < -100 ? -100 : e;
  if (kUp > 0 && e > 127) e = 127;
  return __uint_as_float((uint32_t)(e + 127) << 23);
}

__device__ __forceinline__ bool is_power_of_two(float s) { return (__float_as_uint(s) & 0x7FFFFFu) == 0; }  // for s >= 2^-126

// For the fp32 number q nearest to q + rest: a neighbour of q + rest whose last bit is set, where rest is not 0. Rounded to
// the 4 bits of a code, that gives what q + rest itself gives; q, which may have become halfway between two codes, does not.
__device__ __forceinline__ float to_odd(float q, float rest) {
  const uint32_t u = __float_as_uint(q);
  if (!(rest < 0.0f || rest > 0.0f) || (u & 1) || q == 0.0f) return q;
  return __uint_as_float((rest > 0.0f) == (q > 0.0f) ? u + 1 : u - 1);
}

// x / s, and code * times, to odd. Scales are a user's own where they are no powers of two.
__device__ __forceinline__ float quotient_odd(float x, float s) {
  // Both within range of one another, so that the remainder is exact where x / s is no code of 0.
  const int e = (int)(__float_as_uint(s) >> 23) - 127;
  const float y = __builtin_amdgcn_ldexpf(x, -e), m = __builtin_amdgcn_ldexpf(s, -e), q = y / m;
  return to_odd(q, __builtin_fmaf(-q, m, y));
}
__device__ __forceinline__ float product_odd(float code, float times) {
  const float q = code * times;
  return to_odd(q, __builtin_fmaf(code, times, -q));
}

// Four fp32 -> four e4m3 codes, to nearest even. Infinities saturate at +-448, NaN stays NaN.
__device__ __forceinline__ float clamp448(float x) { return x > 448.0f ? 448.0f : x < -448.0f ? -448.0f : x; }
__device__ __forceinline__ uint32_t encode4(float a, float b, float c, float d) {
  const uint32_t w = __builtin_amdgcn_cvt_pk_fp8_f32(clamp448(a), clamp448(b), 0, false);
  return __builtin_amdgcn_cvt_pk_fp8_f32(clamp448(c), clamp448(d), w, true);
}

__device__ __forceinline__ void decode4(uint32_t w, float* out) {
  const f32x2 a = __builtin_amdgcn_cvt_pk_f32_fp8(w, false), b = __builtin_amdgcn_cvt_pk_f32_fp8(w, true);
  out[0] = a.x;
  out[1] = a.y;
  out[2] = b.x;
  out[3] = b.y;
}

// |x|, or 0 where x is not finite: what a scale is made for.
__device__ __forceinline__ float finite_abs(float x) {
  const uint32_t u = __float_as_uint(x) & 0x7FFFFFFFu;
  return u < 0x7F800000u ? __uint_as_float(u) : 0.0f;
}

// The largest of a wave's non-negative values, in every lane.
__device__ __forceinline__ float wave_max(float x) {
#pragma unroll
  for (int d = 1; d < kWave; d <<= 1) x = fmaxf(x, __shfl_xor(x, d));
  return x;
}

// Workgroup -> a unit of work and one of the `heads` slices of it that heads are. Workgroups go round-robin over the 8
// XCDs; a unit's slices follow each other on one of them. A cache's rows hold their heads side by side, 128 bytes each at
// head_dim 128: with one head's slices of all units on an XCD, it would read every eighth line of the pool, which meets a
// quarter of its L2's channels (decode of 64 sequences 116 us, 16,381 tokens stored 44).
struct Slice {
  int unit, head;
};
__device__ __forceinline__ Slice slice_of(unsigned bid, int heads) {
  const int nth = (int)(bid >> 3), round = nth / heads;
  return {round * 8 + (int)(bid & 7), nth - round * heads};
}
__host__ inline int64_t slices_grid(int64_t units, int64_t heads) { return (units + 7) / 8 * 8 * heads; }

// Tokens of sequence b that are cached, as its table can hold them; none in a cache without blocks.
__device__ __forceinline__ int context_of(const Fp8Cache& c, const PagedBatch& b, int seq) {
  const int64_t room = c.num_blocks > 0 ? (int64_t)b.table_width * c.block_size : 0;
  if (!b.context_lens) return (int)room;
  const int n = b.context_lens[seq];
  return n < 0 ? 0 : n > room ? (int)room : n;
}

// [first, first + count): the call's rows that are sequence b's queries.
struct QueryRows {
  int first, count;
};
__device__ __forceinline__ QueryRows query_rows(const PagedBatch& b, int seq) {
  if (!b.cu_seqlens) return {seq, seq < b.num_tokens ? 1 : 0};  // a call may have no rows at all
  int lo = b.cu_seqlens[seq], hi = b.cu_seqlens[seq + 1];
  lo = lo < 0 ? 0 : lo > b.num_tokens ? b.num_tokens : lo;
  hi = hi < lo ? lo : hi > b.num_tokens ? b.num_tokens : hi;
  return {lo, hi - lo};
}

}  // namespace kvx
