// Attention over a paged pool held in 8 bits (kv8.cuh), for any shape: head sizes that are a multiple of 8 up to 256, any block
// size and strides, masks.  A warp owns one query: 32 keys at a time, one a lane, whose codes it multiplies with the query in fp32;
// then the softmax of the 32 with a running maximum, and the lanes change over to columns of the values.
//
// Everything is fp32 multiply-adds and every query reads its own keys (through L2): the kernel for what the others do not take, and
// what they are compared with in the tests.  (16 tokens over up to 2048 keys, 32 heads of 128 on 8: 1133 us, where the kernel for few queries takes 19.4.)
#include "kv8.cuh"

namespace aidn {
namespace kv8 {
namespace {

constexpr int kWarps = 4;
constexpr int kMaxD = 256;

template <typename T>
__global__ void __launch_bounds__(kWarps * 32) kv8_generic_kernel(const __grid_constant__ Attend p) {
  __shared__ __align__(16) float qs[kWarps][kMaxD];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int D = p.c.head_dim, b = blockIdx.y;
  const int heads = p.kv_count * p.group;
  const int64_t item = (int64_t)blockIdx.x * kWarps + warp;
  const int i = (int)(item / heads);
  const int h = p.kv_begin * p.group + (int)(item % heads), kvh = h / p.group;
  const Rows r = rows_of(p, b);
  if (i >= r.count) return;
  const int keys = keys_of(p, b), end = visible(p, keys, r.count, i);

  const T* q = static_cast<const T*>(p.q) + query_at(p, p.qs, r, b, h, i);
  for (int d = lane; d < D; d += 32) qs[warp][d] = to_float<T>(q[d]) * p.scale;
  __syncwarp();

  float acc[kMaxD / 32] = {};
  float m = -INFINITY, sum = 0.f;
  bool bad = false;
  for (int key0 = 0; key0 < end; key0 += 32) {
    const int key = key0 + lane;
    int block = -1;
    float s = -INFINITY, vs = 0.f;
    const uint8_t* vrow = nullptr;
    if (key < end) {
      const int at = block_of(p.c, key);
      block = checked_block(p.c, p.c.table[b * p.c.table_stride + at], bad);
      if (block >= 0) {
        const int64_t row = block * p.c.stride[0] + (key - at * p.c.block_size) * p.c.stride[1] + kvh * p.c.stride[2];
        const uint8_t* krow = p.c.k + row;
        vrow = p.c.v + row;
        vs = p.c.v_scale[(int64_t)block * p.c.kv_heads + kvh];
        float dot = 0.f;
        for (int d = 0; d < D; d += 4) {
          const float4 x = codes_to_f32(*reinterpret_cast<const uint32_t*>(krow + d));
          const float4 y = *reinterpret_cast<const float4*>(&qs[warp][d]);
          dot = fmaf(x.x, y.x, dot);
          dot = fmaf(x.y, y.y, dot);
          dot = fmaf(x.z, y.z, dot);
          dot = fmaf(x.w, y.w, dot);
        }
        s = dot * p.c.k_scale[(int64_t)block * p.c.kv_heads + kvh];
        if (p.softcap > 0.f) s = p.softcap * tanhf(s / p.softcap);
        if (p.mask_kind != AIDN_MASK_NONE) {
          const int64_t idx = b * p.mask_stride[0] + h * p.mask_stride[1] + i * p.mask_stride[2] + key * p.mask_stride[3];
          if (p.mask_kind == AIDN_MASK_KEEP_U8) {
            if (static_cast<const uint8_t*>(p.mask)[idx] == 0) s = -INFINITY;
          } else if (p.mask_kind == AIDN_MASK_KEEP_F32) {
            if (static_cast<const float*>(p.mask)[idx] == 0.f) s = -INFINITY;
          } else {
            s += static_cast<const float*>(p.mask)[idx];
          }
        }
      }
    }
    float top = s;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    const float now = fmaxf(m, top);
    if (now == -INFINITY && !__any_sync(0xffffffffu, isnan(s))) continue;
    const float base = now == -INFINITY ? 0.f : now;
    const float pr = s == -INFINITY ? 0.f : expf(s - base);
    const float keep = m == -INFINITY ? 0.f : expf(m - base);
    m = now;
    float part = pr;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) part += __shfl_xor_sync(0xffffffffu, part, o);
    sum = sum * keep + part;
#pragma unroll
    for (int c = 0; c < kMaxD / 32; ++c) acc[c] *= keep;
    // a masked key's values may be anything: they are not looked at
    unsigned left = __ballot_sync(0xffffffffu, s != -INFINITY && vrow != nullptr);
    while (left) {
      const int src = __ffs(left) - 1;
      left &= left - 1;
      const float w = __shfl_sync(0xffffffffu, pr, src) * __shfl_sync(0xffffffffu, vs, src);
      const uint8_t* v = reinterpret_cast<const uint8_t*>(__shfl_sync(0xffffffffu, reinterpret_cast<uint64_t>(vrow), src));
#pragma unroll
      for (int c = 0; c < kMaxD / 128; ++c) {   // lane: columns 128 c + 4 lane ..
        const int d = 128 * c + 4 * lane;
        if (d >= D) continue;
        const float4 x = codes_to_f32(*reinterpret_cast<const uint32_t*>(v + d));
        acc[4 * c] = fmaf(w, x.x, acc[4 * c]);
        acc[4 * c + 1] = fmaf(w, x.y, acc[4 * c + 1]);
        acc[4 * c + 2] = fmaf(w, x.z, acc[4 * c + 2]);
        acc[4 * c + 3] = fmaf(w, x.w, acc[4 * c + 3]);
      }
    }
  }
  const float inverse = sum == 0.f ? 0.f : 1.f / sum;
  const int64_t out = query_at(p, p.os, r, b, h, i);
#pragma unroll
  for (int c = 0; c < kMaxD / 128; ++c)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int d = 128 * c + 4 * lane + e;
      if (d < D) store_out<T>(p.out, out + d, acc[4 * c + e] * inverse, p.out_f32);
    }
  if (p.lse && lane == 0) *lse_at(p, r, h, i) = sum == 0.f ? -INFINITY : m + logf(sum);
  if (bad && p.status) atomicOr(p.status, kStatusBadBlock);
}

template <typename T>
cudaError_t launch(const Attend& p, cudaStream_t stream) {
  const int64_t items = p.seq_q * p.kv_count * p.group, grid = (items + kWarps - 1) / kWarps;
  if (grid > 0x7fffffff) return cudaErrorInvalidConfiguration;
  kv8_generic_kernel<T><<<dim3((unsigned)grid, (unsigned)p.batch), kWarps * 32, 0, stream>>>(p);
  return cudaGetLastError();
}

}  // namespace

cudaError_t launch_attend_generic(const Attend& p, cudaStream_t stream) {
  if (p.dtype == AIDN_F32) return launch<float>(p, stream);
  if (p.dtype == AIDN_F16) return launch<__half>(p, stream);
  return launch<__nv_bfloat16>(p, stream);
}

}  // namespace kv8
}  // namespace aidn
