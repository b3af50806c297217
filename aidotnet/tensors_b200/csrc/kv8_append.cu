// Append to a paged key / value pool held in 8 bits (kv8.cuh): a step's queries and keys are rotated by their positions, the
// queries written out, keys and values put into their sequences' blocks as E4M3 codes with a power-of-two scale per block and head.
//
//   (a, b) -> (a cos - b sin, a sin + b cos) for the pairs of a row        fp32, every product and sum rounded on its own
//   s = max(scale_for(largest new magnitude), the block's scale if it holds tokens already);   code = e4m3(x / s)
//
// 3 operations an element: bound by the bytes where there are many tokens and by the chain start -> table -> scale -> store where
// there are few.  The scale is one for all tokens of a block, so that a block and head is the unit of work: a warp (several for
// blocks of more rows than its registers hold) loads the new rows of one block and head once, keeps them rotated in registers
// across the maximum, and stores codes.  Scales being powers of two, a block's older codes change only when its scale does, and
// then by an exponent: only then are they read.
#include "kv8.cuh"

namespace aidn {
namespace kv8 {
namespace {

constexpr int kWarps = 8;
constexpr int kHeld = 8;    // row groups that a warp keeps in registers: 8 floats a lane each
constexpr int kQueryRounds = 4;   // row groups of queries of one token that share the token's cosines and sines

template <typename T>
__device__ __forceinline__ void unpack4(const T* p, bool vec, float* f) {
  if constexpr (sizeof(T) == 4) {
    if (vec) {
      const float4 v = *reinterpret_cast<const float4*>(p);
      f[0] = v.x; f[1] = v.y; f[2] = v.z; f[3] = v.w;
      return;
    }
  } else {
    if (vec) {
      const uint2 v = *reinterpret_cast<const uint2*>(p);
      const T* t = reinterpret_cast<const T*>(&v);
#pragma unroll
      for (int i = 0; i < 4; ++i) f[i] = to_float<T>(t[i]);
      return;
    }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) f[i] = to_float<T>(p[i]);
}

// A lane's eight elements of a row: [d0, d0 + 4) and [d1, d1 + 4).  Contiguous rows are one load.
template <typename T>
__device__ __forceinline__ void load8(const T* row, int d0, int d1, bool vec, float* f) {
  if (sizeof(T) == 2 && vec && d1 == d0 + 4) {
    const uint4 v = *reinterpret_cast<const uint4*>(row + d0);
    const T* t = reinterpret_cast<const T*>(&v);
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = to_float<T>(t[i]);
  } else {
    unpack4(row + d0, vec, f);
    unpack4(row + d1, vec, f + 4);
  }
}
template <typename T>
__device__ __forceinline__ void store8(T* row, int d0, int d1, bool vec, const float* f) {
  if constexpr (sizeof(T) == 4) {
    if (vec) {
      *reinterpret_cast<float4*>(row + d0) = make_float4(f[0], f[1], f[2], f[3]);
      *reinterpret_cast<float4*>(row + d1) = make_float4(f[4], f[5], f[6], f[7]);
      return;
    }
  } else if (vec) {
    uint4 v;
    T* t = reinterpret_cast<T*>(&v);
#pragma unroll
    for (int i = 0; i < 8; ++i) t[i] = from_float<T>(f[i]);
    if (d1 == d0 + 4) {
      *reinterpret_cast<uint4*>(row + d0) = v;
    } else {
      *reinterpret_cast<uint2*>(row + d0) = make_uint2(v.x, v.y);
      *reinterpret_cast<uint2*>(row + d1) = make_uint2(v.z, v.w);
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    row[d0 + i] = from_float<T>(f[i]);
    row[d1 + i] = from_float<T>(f[4 + i]);
  }
}
__device__ __forceinline__ void store_codes(uint8_t* row, int d0, int d1, const float* f) {
  const uint32_t a = to_codes(f[0], f[1]) | to_codes(f[2], f[3]) << 16, b = to_codes(f[4], f[5]) | to_codes(f[6], f[7]) << 16;
  if (d1 == d0 + 4 && (reinterpret_cast<uintptr_t>(row) & 7) == 0) {
    *reinterpret_cast<uint2*>(row + d0) = make_uint2(a, b);
  } else {
    *reinterpret_cast<uint32_t*>(row + d0) = a;
    *reinterpret_cast<uint32_t*>(row + d1) = b;
  }
}

// The pairs of a lane's eight elements have the rotations 4 l .. 4 l + 3 in both layouts.
__device__ __forceinline__ void rotate_pair(float& a, float& b, float c, float s) {
  const float u = a, w = b;
  a = __fsub_rn(__fmul_rn(u, c), __fmul_rn(w, s));
  b = __fadd_rn(__fmul_rn(u, s), __fmul_rn(w, c));
}
__device__ __forceinline__ void rotate8(float* x, const float* c, const float* s, bool halves) {
  if (halves) {
#pragma unroll
    for (int i = 0; i < 4; ++i) rotate_pair(x[i], x[i + 4], c[i], s[i]);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) rotate_pair(x[2 * i], x[2 * i + 1], c[i], s[i]);
  }
}
__device__ __forceinline__ void load_turn(const Append& p, int64_t position, int pair, bool vec, float* c, float* s) {
  if (position < 0 || position >= p.max_position) {
#pragma unroll
    for (int i = 0; i < 4; ++i) { c[i] = 1.f; s[i] = 0.f; }
    return;
  }
  const int64_t at = position * (p.c.head_dim / 2) + pair;
  unpack4(p.cosine + at, vec, c);
  unpack4(p.sine + at, vec, s);
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

template <typename T, int LPR>   // LPR lanes of eight elements make a row
__global__ void __launch_bounds__(kWarps * 32) kv8_append_kernel(const __grid_constant__ Append p, const int warps_per_item, const int64_t slots,
                                                                  const unsigned kv_ctas, const int64_t per_sequence, const bool vec,
                                                                  const bool turn_vec) {
  constexpr int RPI = 32 / LPR;   // rows that a warp loads at a time
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int sub = lane / LPR, l = lane % LPR;
  const int D = p.c.head_dim;
  const bool halves = p.rope == AIDN_ROPE_HALVES;
  __shared__ float maxima[kWarps];
  pdl_wait();
  pdl_trigger();

  if (blockIdx.x >= kv_ctas) {   // ---- queries: (token, kQueryRounds * RPI heads) a warp
    const int chunks = (p.heads + kQueryRounds * RPI - 1) / (kQueryRounds * RPI);
    const int64_t item = (int64_t)(blockIdx.x - kv_ctas) * kWarps + warp;
    const int64_t token = item / chunks;
    if (token >= p.tokens) return;
    const int head0 = (int)(item % chunks) * kQueryRounds * RPI + sub;
    const int d0 = halves ? 4 * l : 8 * l, d1 = halves ? D / 2 + 4 * l : 8 * l + 4;
    const bool mine = 8 * l < D;
    const T* q = static_cast<const T*>(p.q) + token * p.qs[0];
    T* out = static_cast<T*>(p.q_out) + token * p.os[0];
    float x[kQueryRounds][8];
#pragma unroll
    for (int i = 0; i < kQueryRounds; ++i)
      if (mine && head0 + i * RPI < p.heads) load8(q + (head0 + i * RPI) * p.qs[1], d0, d1, vec, x[i]);
    if (p.rope != AIDN_ROPE_NONE) {
      int64_t position;
      if (p.positions) {
        position = p.positions[token];
      } else {
        const int b = p.token_starts ? search(p.batch, token, [&](int i) { return (int64_t)p.token_starts[i]; }) : (int)(token / p.each);
        position = p.start[b] + (token - sequence_of(p, b).first);
      }
      float c[4], s[4];
      if (mine) {
        load_turn(p, position, 4 * l, turn_vec, c, s);
#pragma unroll
        for (int i = 0; i < kQueryRounds; ++i) rotate8(x[i], c, s, halves);
      }
    }
#pragma unroll
    for (int i = 0; i < kQueryRounds; ++i)
      if (mine && head0 + i * RPI < p.heads) store8(out + (head0 + i * RPI) * p.os[1], d0, d1, vec, x[i]);
    return;
  }

  // ---- keys and values: (slot of a sequence's touched blocks, head, key or value) an item
  const int items_per_cta = kWarps / warps_per_item;
  const int64_t item = (int64_t)blockIdx.x * items_per_cta + warp / warps_per_item;
  const int part = warp % warps_per_item;
  const int64_t slot = item / (2 * p.c.kv_heads);
  const int kind = (int)(item % (2 * p.c.kv_heads));
  const bool is_key = kind < p.c.kv_heads;
  const int head = is_key ? kind : kind - p.c.kv_heads;
  const bool turned = is_key && p.rope != AIDN_ROPE_NONE;
  const bool split = turned && halves;
  const int d0 = split ? 4 * l : 8 * l, d1 = split ? D / 2 + 4 * l : 8 * l + 4;
  const bool mine = 8 * l < D;

  int held = 0, count = 0, entry = -1;   // tokens in the block before, new ones, and the block
  int64_t token = 0, position = 0;       // of the first new one
  if (slot < slots) {
    int b;
    int64_t j;
    if (p.token_starts) {
      // a sequence of n tokens touches at most n / size + 2 blocks
      auto base = [&](int i) { return p.token_starts[i] / p.c.block_size + 2 * (int64_t)i; };
      b = search(p.batch, slot, base);
      j = slot - base(b);
    } else {
      b = (int)(slot / per_sequence);
      j = slot % per_sequence;
    }
    const Sequence q = sequence_of(p, b);
    const int64_t start = p.start[b], block = start / p.c.block_size + j;
    const int64_t low = block * p.c.block_size > start ? block * p.c.block_size : start;
    const int64_t end = (block + 1) * p.c.block_size < start + q.count ? (block + 1) * p.c.block_size : start + q.count;
    if (start >= 0 && j >= 0 && low < end && block < p.c.table_stride) {
      bool bad = false;
      entry = checked_block(p.c, p.c.table[b * p.c.table_stride + block], bad);
      held = (int)(low - block * p.c.block_size);
      count = (int)(end - low);
      token = q.first + (low - start);
      position = low;
    }
  }
  if (entry < 0) count = 0;

  const T* src = is_key ? static_cast<const T*>(p.k) + head * p.ks[1] : static_cast<const T*>(p.v) + head * p.vs[1];
  const int64_t src_stride = is_key ? p.ks[0] : p.vs[0];
  float* scale = (is_key ? p.c.k_scale : p.c.v_scale) + (int64_t)entry * p.c.kv_heads + head;
  uint8_t* dst = (is_key ? p.c.k : p.c.v) + (int64_t)entry * p.c.stride[0] + head * p.c.stride[2];
  const float had = count > 0 && held > 0 ? *scale : 0.f;

  // row group i of chunk c: rows (c * kHeld + i) * RPI * warps_per_item + part * RPI + sub
  const int rows_per_group = RPI * warps_per_item;
  const int chunks = (count + kHeld * rows_per_group - 1) / (kHeld * rows_per_group);
  float x[kHeld][8];
  auto load = [&](int c) {
#pragma unroll
    for (int i = 0; i < kHeld; ++i) {
      const int row = (c * kHeld + i) * rows_per_group + part * RPI + sub;
      if (row < count && mine) {
        load8(src + (token + row) * src_stride, d0, d1, vec, x[i]);
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) x[i][e] = 0.f;
      }
    }
    if (turned) {
#pragma unroll
      for (int i = 0; i < kHeld; ++i) {
        const int row = (c * kHeld + i) * rows_per_group + part * RPI + sub;
        if (row < count && mine) {
          float cs[4], sn[4];
          load_turn(p, p.positions ? (int64_t)p.positions[token + row] : position + row, 4 * l, turn_vec, cs, sn);
          rotate8(x[i], cs, sn, halves);
        }
      }
    }
  };

  float largest = 0.f;
  for (int c = 0; c < chunks; ++c) {
    load(c);
#pragma unroll
    for (int i = 0; i < kHeld; ++i)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float a = fabsf(x[i][e]);
        largest = fmaxf(largest, a < INFINITY ? a : 0.f);
      }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) largest = fmaxf(largest, __shfl_xor_sync(0xffffffffu, largest, o));
  if (warps_per_item > 1) {
    if (lane == 0) maxima[warp] = largest;
    __syncthreads();   // (and every warp of the item has read the block's scale)
    for (int w = 0; w < warps_per_item; ++w) largest = fmaxf(largest, maxima[warp - part + w]);
  }
  if (count == 0) return;
  const float s = fmaxf(scale_for(largest), had);
  const float inverse = 1.f / s;

  if (held > 0 && s > had) {
    const float moved = had * inverse;
    for (int row = part * RPI + sub; row < held; row += rows_per_group) {
      if (!mine) continue;
      uint8_t* at = dst + row * p.c.stride[1];
      const float4 a = codes_to_f32(*reinterpret_cast<const uint32_t*>(at + d0)), b = codes_to_f32(*reinterpret_cast<const uint32_t*>(at + d1));
      const float y[8] = {a.x * moved, a.y * moved, a.z * moved, a.w * moved, b.x * moved, b.y * moved, b.z * moved, b.w * moved};
      store_codes(at, d0, d1, y);
    }
  }
  for (int c = 0; c < chunks; ++c) {
    if (chunks > 1) load(c);
#pragma unroll
    for (int i = 0; i < kHeld; ++i) {
      const int row = (c * kHeld + i) * rows_per_group + part * RPI + sub;
      if (row < count && mine) {
#pragma unroll
        for (int e = 0; e < 8; ++e) x[i][e] *= inverse;
        store_codes(dst + (held + row) * p.c.stride[1], d0, d1, x[i]);
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
  const bool vec = aligned(p.k, p.ks) && aligned(p.v, p.vs) && (!p.q || (aligned(p.q, p.qs) && aligned(p.q_out, p.os)));
  const bool turn_vec = (uintptr_t)p.cosine % 16 == 0 && (uintptr_t)p.sine % 16 == 0;   // rows of D / 2 floats, D a multiple of 8
  int warps = 1;
  while (warps < kWarps && warps * kHeld * RPI < p.c.block_size) warps *= 2;
  const int64_t per_sequence = p.each == 1 ? 1 : (p.each + p.c.block_size - 2) / p.c.block_size + 1;
  const int64_t slots = p.token_starts ? p.tokens / p.c.block_size + 2 * (int64_t)p.batch : p.batch * per_sequence;
  const int64_t items = slots * 2 * p.c.kv_heads, per_cta = kWarps / warps;
  const int64_t kv_ctas = (items + per_cta - 1) / per_cta;
  const int64_t q_items = p.q ? p.tokens * ((p.heads + kQueryRounds * RPI - 1) / (kQueryRounds * RPI)) : 0;
  const int64_t grid = kv_ctas + (q_items + kWarps - 1) / kWarps;
  if (grid > 0x7fffffff) return cudaErrorInvalidConfiguration;
  *launches = 1;
  return launch_dependent(kv8_append_kernel<T, LPR>, dim3((unsigned)grid), kWarps * 32, 0, stream, p, warps, slots, (unsigned)kv_ctas,
                          per_sequence, vec, turn_vec);
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
