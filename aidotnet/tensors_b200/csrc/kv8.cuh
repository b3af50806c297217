// A paged key / value pool held in 8 bits: parameter blocks of its kernels, addressing, and the E4M3 codes.
#pragma once

#include "common.cuh"

namespace aidn {
namespace kv8 {

constexpr float kLargestCode = 448.f;
// Rows (queries x query heads of a group) of a sequence up to which the kernel for few queries is the faster one in all of these.  Us of the one and the other, L2
// flushed, 8 KV heads, with 32, 40, 64 and 96 rows (where the sides meet beyond 32 depends on how many sequences there are, and how long):
//   heads of 128   24 sequences of 2048 to 4096 keys   99 / 115   128 / 115   160 / 117   222 / 117
//                  2 sequences of 2048 to 4096 keys    35 / 50     40 / 50     44 / 50     52 / 52
//                  64 sequences of 350 to 700 keys     66 / 130    87 / 130   105 / 134   140 / 134
//   heads of 64    24                                  81 / 95    103 / 97    128 / 95    173 / 97
//                  2                                   31 / 42     35 / 42     40 / 42     46 / 42
//                  64                                  58 / 103    74 / 103    89 / 103   113 / 105
constexpr int kFewRows = 32;

constexpr int kLeastExponent = -100, kMostExponent = 119;   // of a scale: 448 * 2^119 is below the largest float

struct Pool {
  uint8_t* k;
  uint8_t* v;
  float* k_scale;   // [num_blocks, kv_heads]
  float* v_scale;
  const int32_t* table;
  int64_t table_stride;
  int64_t stride[3];   // bytes for (block, token, head)
  int32_t num_blocks, block_size, kv_heads, head_dim;
  int32_t block_shift;   // log2(block_size), or -1
};

struct Append {
  Pool c;
  const void* q;
  const void* k;
  const void* v;
  void* q_out;
  int64_t qs[2], ks[2], vs[2], os[2];   // elements for (token, head)
  const float* cosine;
  const float* sine;
  const int32_t* start;
  const int32_t* token_starts;   // or null: `each` tokens a sequence
  const int32_t* positions;
  int64_t tokens, max_position, each;
  int32_t batch, heads, dtype, rope;
};

struct Attend {
  Pool c;
  const void* q;
  void* out;
  float* lse;        // [queries, Hq] or null
  int64_t qs[3], os[3];
  const int32_t* kv_len;
  const int32_t* query_starts;
  const void* mask;
  int64_t mask_stride[4];
  int64_t queries;   // with query_starts: of all sequences
  int64_t seq_q, seq_kv;
  int64_t causal_offset;
  int32_t batch, num_q_heads, group;
  int64_t rows_above, rows_upto;   // with query_starts: sequences of no more, or more rows (queries x query heads of a group) are left out
  int32_t kv_begin, kv_count;   // KV heads of the handle's shard
  int32_t dtype, out_f32, mask_kind, causal, bottom_right;
  float scale, softcap;
  int32_t* status;
};

// ---- addressing -----------------------------------------------------------------------------------------------------

__device__ __forceinline__ int block_of(const Pool& c, int key) {
  return c.block_shift >= 0 ? key >> c.block_shift : (int)((uint32_t)key / (uint32_t)c.block_size);
}
// The table's entry, -1 for one outside the pool (and `bad` set).
__device__ __forceinline__ int checked_block(const Pool& c, int entry, bool& bad) {
  const bool out = entry < 0 || (c.num_blocks > 0 && entry >= c.num_blocks);
  bad = bad || out;
  return out ? -1 : entry;
}

// Queries of sequence b: the row of its first one, and how many.
struct Rows {
  int64_t first;
  int count;
};
__device__ __forceinline__ Rows rows_of(const Attend& p, int b) {
  if (!p.query_starts) return {(int64_t)b * p.seq_q, (int)p.seq_q};
  const int64_t first = p.query_starts[b], last = p.query_starts[b + 1];
  // (what the host cannot see: no row outside [0, queries) is touched whatever the starts are)
  int64_t n = (last < p.queries ? last : p.queries) - first;
  if (first < 0 || n < 0) n = 0;
  if (n * p.group <= p.rows_above || n * p.group > p.rows_upto) n = 0;   // another launch's
  if (n > p.seq_q) n = p.seq_q;
  return {first, (int)n};
}
__device__ __forceinline__ int keys_of(const Attend& p, int b) {
  int n = (int)p.seq_kv;
  if (p.kv_len) {
    const int l = p.kv_len[b];
    n = l < 0 ? 0 : (l < n ? l : n);
  }
  return n;
}
// Query i of n sees the keys below this.
__device__ __forceinline__ int visible(const Attend& p, int keys, int n, int i) {
  if (!p.causal) return keys;
  const int64_t end = (p.bottom_right ? (int64_t)keys - n : p.causal_offset) + i + 1;
  return end < 0 ? 0 : (end < keys ? (int)end : keys);
}
// Offsets of query i of sequence b, head h, in q and in out.
__device__ __forceinline__ int64_t query_at(const Attend& p, const int64_t* stride, const Rows& r, int b, int h, int i) {
  return (p.query_starts ? (r.first + i) * stride[2] : b * stride[0] + i * stride[2]) + h * stride[1];
}
__device__ __forceinline__ float* lse_at(const Attend& p, const Rows& r, int h, int i) {
  return p.lse + (r.first + i) * p.num_q_heads + h;
}

// ---- codes ----------------------------------------------------------------------------------------------------------

// Two codes (the low 16 bits of x) as two fp16 values, exact.
__device__ __forceinline__ uint32_t codes_to_f16(uint32_t x) {
  uint32_t r;
  asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, l;\n\t}" : "=r"(r) : "r"(x));
  return r;
}
__device__ __forceinline__ uint32_t codes_to_f16_hi(uint32_t x) {
  uint32_t r;
  asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, h;\n\t}" : "=r"(r) : "r"(x));
  return r;
}
// Two values as codes (lo in the low byte): nearest, ties to even, +-448 beyond the largest.
__device__ __forceinline__ uint32_t to_codes(float lo, float hi) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ float4 codes_to_f32(uint32_t x) {
  const uint32_t a = codes_to_f16(x), b = codes_to_f16_hi(x);
  const float2 lo = __half22float2(*reinterpret_cast<const __half2*>(&a)), hi = __half22float2(*reinterpret_cast<const __half2*>(&b));
  return make_float4(lo.x, lo.y, hi.x, hi.y);
}

// The scale for values up to m: 2^e with the smallest e for which m <= 448 * 2^e.  448 = 1.75 * 2^8.
__device__ __forceinline__ float scale_for(float m) {
  const uint32_t bits = __float_as_uint(m);
  int e = (int)(bits >> 23) - 127 - 8 + ((bits & 0x7fffffu) > 0x600000u ? 1 : 0);
  if (e < kLeastExponent || m == 0.f) e = kLeastExponent;   // (also for what is below the smallest normal float)
  if (e > kMostExponent) e = kMostExponent;
  return __uint_as_float((uint32_t)(e + 127) << 23);
}
// 1 / a power of two in [2^-126, 2^126].
__device__ __forceinline__ float inverse_pow2(float s) { return __uint_as_float(0x7f000000u - __float_as_uint(s)); }

// tanh(x) = 1 - 2 / (1 + e^2x), to 3e-7 of 1: the logits are off by that times the cap.  A NaN stays one.
__device__ __forceinline__ float tanh_ex2(float x) {
  float y;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(x * (2.f * kLog2e)), "f"(80.f));
  return 1.f - __fdividef(2.f, 1.f + ex2_approx(y));
}

cudaError_t launch_append(const Append& p, cudaStream_t stream, int* launches);
cudaError_t launch_attend_generic(const Attend& p, cudaStream_t stream);
// Few queries (csrc/kv8_split.cu): head sizes that are a multiple of 16, 16-byte aligned pools, no mask.  Without its workspace keys are not
// cut.  raised: a word of the handle, which kernels had their shared-memory limit raised.
bool split_supported(const Attend& p);
int64_t split_workspace_bytes(int head_dim, bool exact, int64_t batch, int64_t rows, int64_t seq_kv, int kv_count, int num_sms);
cudaError_t launch_attend_split(const Attend& p, int num_sms, void* workspace, int64_t workspace_bytes, uint64_t* raised, int* launches,
                                cudaStream_t stream);
// Many queries of 16 bits (csrc/kv8_sm100.cu): head sizes 64 and 128, blocks of a multiple of 16 tokens, 16-byte aligned pools, no mask.
bool sm100_supported(const Attend& p);
int64_t sm100_workspace_bytes(int head_dim, int num_sms);
cudaError_t launch_attend_sm100(const Attend& p, int num_sms, void* workspace, int64_t workspace_bytes, uint64_t* raised, int* launches,
                                cudaStream_t stream);

}  // namespace kv8
}  // namespace aidn
