// Append to a paged key / value pool held in 8 bits (kv8.cuh): a step's queries and keys are rotated by their positions, the
// queries written out, keys and values put into their sequences' blocks as E4M3 codes with a power-of-two scale per block and head.
//
//   (a, b) -> (a cos - b sin, a sin + b cos) for the pairs of a row        fp32, every product and sum rounded on its own
//   s = max(scale_for(largest new magnitude), the block's scale if it holds tokens already);   code = e4m3(x / s)
//
// 3 operations an element: bound by the bytes where there are many tokens and by the chain start -> table -> scale -> store where
// there are few.  (With many tokens by the latency of the loads, in fact: rows are held as the 32-bit floats that they became, and part of them on the
// stack.)  The scale is one for all tokens of a block, so that a block and head is the unit of work: a warp (several for
// blocks of more rows than its registers hold) loads the new rows of one block and head once, keeps them rotated in registers
// across the maximum, and stores codes.  Scales being powers of two, a block's older codes change only when its scale does, and
// then by an exponent: only then are they read.  8192 tokens of 32 + 2 x 8 heads of 128: 47 us, 4.0 TB/s (a warp a token, one element at a time:
// 99); one token: 3.8 us.
#include "kv8.cuh"

namespace aidn {
namespace kv8 {
namespace {

constexpr int kWarps = 8;
constexpr int kHeld = 4;    // row groups that a warp keeps in registers: 8 floats a lane each
constexpr int kQueryRounds = 4;   // row groups of queries of one token that share the token's cosines and sines

// How a lane's eight elements of a row lie: [d0, d0 + 4) and [d1, d1 + 4), which make four pairs of a rotation either way.
enum Form {
  kAny,      // element by element, in either layout: rows that are not 16-byte aligned
  kPairs,    // 16 bytes at a time; pairs (2i, 2i + 1), or no rotation
  kHalves    // pairs (i, i + D/2)
};
template <typename T>
__device__ __forceinline__ void load4(const T* p, bool vec, float* f) {
  if (!vec) {
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] = to_float<T>(p[i]);
  } else if constexpr (sizeof(T) == 4) {
    const float4 v = *reinterpret_cast<const float4*>(p);
    f[0] = v.x; f[1] = v.y; f[2] = v.z; f[3] = v.w;
  } else {
    const uint2 v = *reinterpret_cast<const uint2*>(p);
    const T* t = reinterpret_cast<const T*>(&v);
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] = to_float<T>(t[i]);
  }
}
template <typename T, Form F>
__device__ __forceinline__ void load8(const T* row, int d0, int d1, bool split, float* f) {
  if (sizeof(T) == 2 && F != kAny && !(F == kHalves && split)) {
    const uint4 v = *reinterpret_cast<const uint4*>(row + d0);
    const T* t = reinterpret_cast<const T*>(&v);
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = to_float<T>(t[i]);
  } else {
    load4(row + d0, F != kAny, f);
    load4(row + d1, F != kAny, f + 4);
  }
}
template <typename T, Form F>
__device__ __forceinline__ void store8(T* row, int d0, int d1, const float* f) {
  if constexpr (F == kAny) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      row[d0 + i] = from_float<T>(f[i]);
      row[d1 + i] = from_float<T>(f[4 + i]);
    }
  } else if constexpr (sizeof(T) == 4) {
    *reinterpret_cast<float4*>(row + d0) = make_float4(f[0], f[1], f[2], f[3]);
    *reinterpret_cast<float4*>(row + d1) = make_float4(f[4], f[5], f[6], f[7]);
  } else {
    uint4 v;
    T* t = reinterpret_cast<T*>(&v);
#pragma unroll
    for (int i = 0; i < 8; ++i) t[i] = from_float<T>(f[i]);
    if constexpr (F == kPairs) {
      *reinterpret_cast<uint4*>(row + d0) = v;
    } else {
      *reinterpret_cast<uint2*>(row + d0) = make_uint2(v.x, v.y);
      *reinterpret_cast<uint2*>(row + d1) = make_uint2(v.z, v.w);
    }
  }
}
__device__ __forceinline__ void store_codes(uint8_t* row, int d0, int d1, bool eight, const float* f) {
  const uint32_t a = to_codes(f[0], f[1]) | to_codes(f[2], f[3]) << 16, b = to_codes(f[4], f[5]) | to_codes(f[6], f[7]) << 16;
  if (eight) {
    *reinterpret_cast<uint2*>(row + d0) = make_uint2(a, b);
  } else {
    *reinterpret_cast<uint32_t*>(row + d0) = a;
    *reinterpret_cast<uint32_t*>(row + d1) = b;
  }
}

__device__ __forceinline__ void rotate_pair(float& a, float& b, float c, float s) {
  const float u = a, w = b;
  a = __fsub_rn(__fmul_rn(u, c), __fmul_rn(w, s));
  b = __fadd_rn(__fmul_rn(u, s), __fmul_rn(w, c));
}
// The pairs of a lane's eight elements have the rotations 4 l .. 4 l + 3 in both layouts.
template <Form F>
__device__ __forceinline__ void rotate8(float* x, const float* c, const float* s, bool halves) {
  if (F == kHalves || (F == kAny && halves)) {
#pragma unroll
    for (int i = 0; i < 4; ++i) rotate_pair(x[i], x[i + 4], c[i], s[i]);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) rotate_pair(x[2 * i], x[2 * i + 1], c[i], s[i]);
  }
}
template <Form F>
__device__ __forceinline__ void load_turn(const Append& p, int64_t position, int pair, float* c, float* s) {
  if (position < 0 || position >= p.max_position) {
#pragma unroll
    for (int i = 0; i < 4; ++i) { c[i] = 1.f; s[i] = 0.f; }
    return;
  }
  const int64_t at = position * (p.c.head_dim / 2) + pair;
  load4(p.cosine + at, F != kAny, c);
  load4(p.sine + at, F != kAny, s);
}

// The largest b in [0, n) with f(b) <= x, for an ascending f with f(0) <= x.  All lanes of the warp: 32 candidates a round.
template <typename F>
__device__ __forceinline__ int search(int n, int64_t x, F f) {
  const int lane = threadIdx.x & 31;
  int low = 0;
  while (n > 1) {
    const int step = (n + 31) / 32, at = lane * step;
    const unsigned below = __ballot_sync(0xffffffffu, at < n && f(low + at) <= x);
    const int k = below ? 31 - __clz(below) : 0;
    low += k * step;
    n = min(step, n - k * step);
  }
  return low;
}

struct Sequence {
  int64_t first;   // its first token
  int64_t count;
};
__device__ __forceinline__ Sequence sequence_of(const Append& p, int b) {
  if (!p.token_starts) return {b * p.each, p.each};
  const int64_t first = p.token_starts[b], last = p.token_starts[b + 1];
  // (what the host cannot see: no token outside [0, tokens) is touched whatever the starts are)
  const int64_t n = (last < p.tokens ? last : p.tokens) - first;
  return {first, first < 0 || n < 0 ? 0 : n};
}

// CTAs an SM: their loads have to cover one another's latency, and more of them are worth registers that are spilled.  8192 tokens of 32 and 8 heads of
// 128, pairs: 47.5 us with four (64 registers, 216 bytes of spill stores a thread), 50.6 with three (80, 12 bytes), 59.5 with two (115, none), and 99
// with two of eight row groups a warp; 13 prompts of 16 heads of 64, halves, whose loads are twice as many: 38 with four, 33.9 with three (80, 96
// bytes), 36.2 with two (118, none).
template <Form F>
constexpr int kMinCtas = F == kHalves ? 3 : 4;

template <typename T, int LPR, Form F>   // LPR lanes of eight elements make a row
__global__ void __launch_bounds__(kWarps * 32, kMinCtas<F>) kv8_append_kernel(const __grid_constant__ Append p, const int shift, const uint32_t slots,
                                                                            const uint32_t kv_ctas, const uint32_t per_sequence, const bool eight) {
  constexpr int RPI = 32 / LPR;   // rows that a warp loads at a time
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int sub = lane / LPR;
  const int D = p.c.head_dim;
  // lanes beyond a row's end take its first elements too, so that no load needs a condition (and store nothing)
  const bool mine = 8 * (lane % LPR) < D;
  const int l = mine ? lane % LPR : 0;
  const bool halves = F == kHalves || (F == kAny && p.rope == AIDN_ROPE_HALVES);
  __shared__ float maxima[kWarps];
  pdl_wait();
  pdl_trigger();

  if (blockIdx.x >= kv_ctas) {   // ---- queries: (token, kQueryRounds * RPI heads) a warp
    const uint32_t chunks = (p.heads + kQueryRounds * RPI - 1) / (kQueryRounds * RPI), item = (blockIdx.x - kv_ctas) * kWarps + warp;
    const uint32_t token = item / chunks;
    if (token >= (uint32_t)p.tokens) return;
    const int head0 = (int)(item - token * chunks) * kQueryRounds * RPI + sub;
    const int d0 = halves ? 4 * l : 8 * l, d1 = halves ? D / 2 + 4 * l : 8 * l + 4;
    const T* q = static_cast<const T*>(p.q) + token * p.qs[0];
    T* out = static_cast<T*>(p.q_out) + token * p.os[0];
    float x[kQueryRounds][8];
#pragma unroll
    for (int i = 0; i < kQueryRounds; ++i) load8<T, F>(q + min(head0 + i * RPI, p.heads - 1) * p.qs[1], d0, d1, halves, x[i]);
    if (p.rope != AIDN_ROPE_NONE) {
      int64_t position;
      if (p.positions) {
        position = p.positions[token];
      } else {
        const int b = p.token_starts ? search(p.batch, token, [&](int i) { return (int64_t)p.token_starts[i]; }) : (int)(token / (uint32_t)p.each);
        position = p.start[b] + (token - sequence_of(p, b).first);
      }
      float c[4], s[4];
      load_turn<F>(p, position, 4 * l, c, s);
#pragma unroll
      for (int i = 0; i < kQueryRounds; ++i) rotate8<F>(x[i], c, s, halves);
    }
#pragma unroll
    for (int i = 0; i < kQueryRounds; ++i)
      if (mine && head0 + i * RPI < p.heads) store8<T, F>(out + (head0 + i * RPI) * p.os[1], d0, d1, x[i]);
    return;
  }

  // ---- keys and values: (slot of a sequence's touched blocks, head, key or value) an item of 2^shift warps
  const uint32_t item = (blockIdx.x * kWarps + warp) >> shift, slot = item / (2u * p.c.kv_heads);
  const int warps = 1 << shift, part = warp & (warps - 1);
  const int kind = (int)(item - slot * 2u * p.c.kv_heads);
  const bool is_key = kind < p.c.kv_heads;
  const int head = is_key ? kind : kind - p.c.kv_heads;
  const bool turned = is_key && p.rope != AIDN_ROPE_NONE, split = turned && halves;
  const int d0 = split ? 4 * l : 8 * l, d1 = split ? D / 2 + 4 * l : 8 * l + 4;

  int held = 0, count = 0, entry = -1;   // tokens in the block before, new ones, and the block
  int64_t token = 0;                     // the first new one, and its position
  int position = 0;
  if (slot < slots) {
    int b, j;
    if (p.token_starts) {
      // a sequence of n tokens touches at most n / size + 2 blocks
      auto base = [&](int i) { return block_of(p.c, p.token_starts[i]) + 2 * (int64_t)i; };
      b = search(p.batch, slot, base);
      j = (int)(slot - base(b));
    } else {
      b = (int)(slot / per_sequence);
      j = (int)(slot - (uint32_t)b * per_sequence);
    }
    const Sequence q = sequence_of(p, b);
    const int start = p.start[b];
    const int64_t block = (start < 0 ? 0 : block_of(p.c, start)) + (int64_t)j, edge = block * p.c.block_size;
    const int64_t low = edge > start ? edge : start, end = min(edge + p.c.block_size, start + q.count);
    if (start >= 0 && j >= 0 && low < end && block < p.c.table_stride) {
      bool bad = false;
      entry = checked_block(p.c, p.c.table[b * p.c.table_stride + block], bad);
      held = (int)(low - edge);
      count = (int)(end - low);
      token = q.first + (low - start);
      position = (int)low;
    }
  }
  if (entry < 0) count = 0;

  const int first = part * RPI + sub, step = RPI << shift;   // rows of this lane: first, first + step, ...
  const T* const src = (is_key ? static_cast<const T*>(p.k) + head * p.ks[1] + token * p.ks[0] : static_cast<const T*>(p.v) + head * p.vs[1] + token * p.vs[0]);
  const int64_t src_stride = is_key ? p.ks[0] : p.vs[0];
  float* const scale = (is_key ? p.c.k_scale : p.c.v_scale) + (int64_t)entry * p.c.kv_heads + head;
  uint8_t* const dst = (is_key ? p.c.k : p.c.v) + (int64_t)entry * p.c.stride[0] + head * p.c.stride[2];
  const float had = count > 0 && held > 0 ? *scale : 0.f;

  const int chunks = (count + kHeld * step - 1) / (kHeld * step);   // of the rows that all lanes hold
  float x[kHeld][8];
  auto load = [&](int c) {   // (rows beyond the last are the last)
#pragma unroll
    for (int i = 0; i < kHeld; ++i) load8<T, F>(src + min((c * kHeld + i) * step + first, count - 1) * src_stride, d0, d1, split, x[i]);
    if (turned) {
#pragma unroll
      for (int i = 0; i < kHeld; ++i) {
        const int row = min((c * kHeld + i) * step + first, count - 1);
        float cs[4], sn[4];
        load_turn<F>(p, p.positions ? p.positions[token + row] : position + row, 4 * l, cs, sn);
        rotate8<F>(x[i], cs, sn, halves);
      }
    }
  };
  auto maximum = [&](bool finite) {
    float largest = 0.f;
    for (int c = 0; c < chunks; ++c) {
      load(c);
#pragma unroll
      for (int i = 0; i < kHeld; ++i)
#pragma unroll
        for (int e = 0; e < 8; ++e) largest = fmaxf(largest, finite && fabsf(x[i][e]) == INFINITY ? 0.f : fabsf(x[i][e]));
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) largest = fmaxf(largest, __shfl_xor_sync(0xffffffffu, largest, o));
    return largest;
  };
  float largest = maximum(false);
  if (largest == INFINITY) largest = maximum(true);   // only finite elements count
  if (shift > 0) {
    if (lane == 0) maxima[warp] = largest;
    __syncthreads();   // (and every warp of the item has read the block's scale)
    for (int w = 0; w < warps; ++w) largest = fmaxf(largest, maxima[warp - part + w]);
  }
  if (count == 0) return;
  const float s = fmaxf(scale_for(largest), had), inverse = 1.f / s;

  if (held > 0 && s > had && mine) {
    const float moved = had * inverse;
    for (int row = first; row < held; row += step) {
      uint8_t* at = dst + row * p.c.stride[1];
      const float4 a = codes_to_f32(*reinterpret_cast<const uint32_t*>(at + d0)), b = codes_to_f32(*reinterpret_cast<const uint32_t*>(at + d1));
      const float y[8] = {a.x * moved, a.y * moved, a.z * moved, a.w * moved, b.x * moved, b.y * moved, b.z * moved, b.w * moved};
      store_codes(at, d0, d1, eight && !split, y);
    }
  }
  for (int c = 0; c < chunks; ++c) {
    if (chunks > 1) load(c);
#pragma unroll
    for (int i = 0; i < kHeld; ++i) {
      const int row = (c * kHeld + i) * step + first;
      if (row < count && mine) {
#pragma unroll
        for (int e = 0; e < 8; ++e) x[i][e] *= inverse;
        store_codes(dst + (held + row) * p.c.stride[1], d0, d1, eight && !split, x[i]);
      }
    }
  }
  if (part == 0 && lane == 0) *scale = s;
}

template <typename T, int LPR>
cudaError_t launch(const Append& p, cudaStream_t stream, int* launches) {
  constexpr int RPI = 32 / LPR;
  auto aligned = [&](const void* ptr, const int64_t* s) {
    return (uintptr_t)ptr % 16 == 0 && s[0] * sizeof(T) % 16 == 0 && s[1] * sizeof(T) % 16 == 0;
  };
  // (rows of the cosines and sines are D / 2 floats, D a multiple of 8)
  const bool vec = aligned(p.k, p.ks) && aligned(p.v, p.vs) && (!p.q || (aligned(p.q, p.qs) && aligned(p.q_out, p.os))) &&
                   (uintptr_t)p.cosine % 16 == 0 && (uintptr_t)p.sine % 16 == 0;
  const bool eight = ((uintptr_t)p.c.k | (uintptr_t)p.c.v | (uint64_t)p.c.stride[0] | (uint64_t)p.c.stride[1] | (uint64_t)p.c.stride[2]) % 8 == 0;
  int shift = 0;   // warps of an item: those that hold a block's rows, up to all of a CTA
  while ((1 << shift) < kWarps && kHeld * (RPI << shift) < p.c.block_size && kHeld * (RPI << shift) < p.tokens) ++shift;
  const int64_t per_sequence = p.each == 1 ? 1 : (p.each + p.c.block_size - 2) / p.c.block_size + 1;
  const int64_t slots = p.token_starts ? p.tokens / p.c.block_size + 2 * (int64_t)p.batch : p.batch * per_sequence;
  const int64_t items = slots * 2 * p.c.kv_heads, per_cta = kWarps >> shift;
  const int64_t kv_ctas = (items + per_cta - 1) / per_cta;
  const int64_t q_items = p.q ? p.tokens * ((p.heads + kQueryRounds * RPI - 1) / (kQueryRounds * RPI)) : 0;
  const int64_t grid = kv_ctas + (q_items + kWarps - 1) / kWarps;
  if (grid > 0x0fffffff || slots > 0x7fffffff) return cudaErrorInvalidConfiguration;   // (warps are counted in 32 bits)
  *launches = 1;
  auto k = !vec ? kv8_append_kernel<T, LPR, kAny> : p.rope == AIDN_ROPE_HALVES ? kv8_append_kernel<T, LPR, kHalves> : kv8_append_kernel<T, LPR, kPairs>;
  return launch_dependent(k, dim3((unsigned)grid), kWarps * 32, 0, stream, p, shift, (uint32_t)slots, (uint32_t)kv_ctas, (uint32_t)per_sequence, eight);
}

template <typename T>
cudaError_t launch_t(const Append& p, cudaStream_t stream, int* launches) {
  if (p.c.head_dim <= 64) return launch<T, 8>(p, stream, launches);
  if (p.c.head_dim <= 128) return launch<T, 16>(p, stream, launches);
  return launch<T, 32>(p, stream, launches);
}

}  // namespace

cudaError_t launch_append(const Append& p, cudaStream_t stream, int* launches) {
  if (p.dtype == AIDN_F32) return launch_t<float>(p, stream, launches);
  if (p.dtype == AIDN_F16) return launch_t<__half>(p, stream, launches);
  return launch_t<__nv_bfloat16>(p, stream, launches);
}

}  // namespace kv8
}  // namespace aidn
