// Attention of few queries over a paged pool held in 8 bits (kv8.cuh): decode steps, drafted tokens, short chunks.
//
//   S^T = K Q^T,  x = S c_r k_scale(block)   (base 2; c_r = scale log2(e) / the query's own factor)
//   P = 2^(x - m) with a running maximum m,   O^T += V^T (P v_scale(block) / v_ref)^T,   o = O v_ref / sum P
//
// Bound by the pool's bytes: 2 D bytes a key and KV head, a few operations a byte.  So every key is read once for all the queries of its
// sequence and KV head (a "line": up to 8 NR query rows = query heads of the group x queries), straight from global memory into the
// registers that feed mma.sync: a product does not care about the order of its terms, so the head dimension is permuted such
// that a lane's 16 bytes of a key are its own elements of four A fragments, and a lane's 16 bytes of a value row its own rows of eight
// (queries are laid out in the matching order once a line).  No shared memory and no transposition lie on the way of the keys; a
// code becomes fp16 exactly (cvt, two at a time), a query is scaled by a power of two into fp16 (two terms for fp32 results),
// and the scales of the blocks are applied to the products in fp32.  Weights are rounded to fp16 (11 bits, of 2^9 times their
// value so that they stay normal down to 2^-23 of the largest); for fp32 results they are two terms too.
//
// The lines' 16-key tiles are one row, cut into equal shares for the CTAs that are resident whatever the lengths are; the warps of a
// CTA take the tiles of its share in turn and merge through shared memory.  A line that is cut leaves one partial result a CTA in
// the workspace, and the CTA that arrives last (a counter that wraps to zero by itself) merges them in their order: the
// result does not depend on who was last, and there is no second launch.
#include "kv8.cuh"
#include "mma_sync.cuh"

namespace aidn {
namespace kv8 {
namespace {

constexpr int kTile = 16;           // keys
constexpr float kUnset = -1e30f;    // running maximum before any key
constexpr float kLazy = 6.f;        // the maximum follows when a logit is 2^6 above it: weights stay below 2^(9 + 6), in fp16's range
constexpr float kLift = 9.f;

struct Split {
  float* partial;    // [2 grid][8 NR][DP], or null: lines are not cut
  float2* stats;     // [2 grid][8 NR]: maximum and sum
  int least;         // tiles of a warp's share
  bool query_vec, out_vec;   // 16 bytes of the queries, four elements of the results are aligned
};

__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
  return r;
}
__device__ __forceinline__ uint2 ld_stream8(const void* ptr) {
  uint2 r;
  asm volatile("ld.global.L1::no_allocate.v2.u32 {%0,%1}, [%2];" : "=r"(r.x), "=r"(r.y) : "l"(ptr));
  return r;
}
// Sixteen elements of a query as they lie: eight words of 16-bit elements, sixteen of 32-bit ones.  (Volatile: issued where they stand.)
__device__ __forceinline__ void ld_words4(const void* ptr, uint32_t* w) {
  asm volatile("ld.global.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "l"(ptr));
}
template <int T>
__device__ __forceinline__ void load16(const Attend& p, int64_t at, bool vec, uint32_t* w) {
  if (T == 2 && p.dtype == AIDN_F32) {
    const float* q = static_cast<const float*>(p.q) + at;
#pragma unroll
    for (int e = 0; e < 8 * T; e += 4) {
      if (vec) {
        ld_words4(q + e, w + e);
      } else {
#pragma unroll
        for (int u = 0; u < 4; ++u) w[e + u] = __float_as_uint(q[e + u]);
      }
    }
    return;
  }
  const uint16_t* q = static_cast<const uint16_t*>(p.q) + at;
#pragma unroll
  for (int e = 0; e < 8; e += 4) {
    if (vec) {
      ld_words4(q + 2 * e, w + e);
    } else {
#pragma unroll
      for (int u = 0; u < 4; ++u) w[e + u] = q[2 * (e + u)] | (uint32_t)q[2 * (e + u) + 1] << 16;
    }
  }
}
template <int T>
__device__ __forceinline__ float widen(const Attend& p, const uint32_t* w, int e) {
  if (T == 2 && p.dtype == AIDN_F32) return __uint_as_float(w[T == 2 ? e : 0]);
  const uint32_t v = w[e >> 1] >> (16 * (e & 1)) & 0xffffu;
  return p.dtype == AIDN_F16 ? __half2float(__ushort_as_half((unsigned short)v)) : __uint_as_float(v << 16);
}
__device__ __forceinline__ void store4(const Attend& p, int64_t at, bool vec, float4 o) {
  if (p.out_f32) {
    float* to = static_cast<float*>(p.out) + at;
    if (vec) {
      *reinterpret_cast<float4*>(to) = o;
    } else {
      to[0] = o.x; to[1] = o.y; to[2] = o.z; to[3] = o.w;
    }
    return;
  }
  uint16_t* to = static_cast<uint16_t*>(p.out) + at;
  const uint32_t a = p.dtype == AIDN_F16 ? pack_pair<__half>(o.x, o.y) : pack_pair<__nv_bfloat16>(o.x, o.y);
  const uint32_t c = p.dtype == AIDN_F16 ? pack_pair<__half>(o.z, o.w) : pack_pair<__nv_bfloat16>(o.z, o.w);
  if (vec) {
    *reinterpret_cast<uint2*>(to) = make_uint2(a, c);
  } else {
    to[0] = (uint16_t)a; to[1] = (uint16_t)(a >> 16); to[2] = (uint16_t)c; to[3] = (uint16_t)(c >> 16);
  }
}
// tanh to 3e-7 of 1: the logits are off by that times the cap.
__device__ __forceinline__ float tanh_ex2(float x) { return 1.f - __fdividef(2.f, 1.f + ex2_approx(fminf(x * (2.f * kLog2e), 80.f))); }
// Whether any of four codes is a NaN.
__device__ __forceinline__ bool any_nan(uint32_t x) { return (((x & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u) != 0; }
__device__ __forceinline__ uint32_t without_nan(uint32_t x) {
  const uint32_t hit = (((x & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u) >> 7;   // 1 in the bytes that are
  return x & ~(hit * 0xffu);
}

template <int DP, int NR, int T, bool UB>
struct Config {
  static constexpr int kWarps = NR == 1 && DP < 256 ? 8 : 4;
  static constexpr int kMinCtas = DP == 256 ? 2 : (NR == 1 ? 2 : 3);
  static constexpr int kSteps = DP / 16;                 // of 16 elements: fragments of a key
  static constexpr int kRows = 8 * NR;
  static constexpr int kPitch = DP + 4;                  // floats between the rows of a partial result
  static constexpr int kQueryWords = T * NR * kSteps * 32 * 2;   // of a warp
  static constexpr size_t kSmem = (size_t)kWarps * (kQueryWords * 4 + 2 * kRows * kPitch * 4);
};

template <int DP, int NR, int T, bool UB>
__global__ void __launch_bounds__(Config<DP, NR, T, UB>::kWarps * 32, Config<DP, NR, T, UB>::kMinCtas)
    kv8_split_kernel(const __grid_constant__ Attend p, const Split sp) {
  using C = Config<DP, NR, T, UB>;
  constexpr int NW = C::kWarps, KS = C::kSteps, MT = DP / 16, ROWS = C::kRows;
  constexpr int KC = DP / 64;                     // 64-byte pieces of a key: 16 bytes a lane
  constexpr int VB = DP == 64 ? 8 : 16;           // bytes of a value row a lane reads at a time
  constexpr int VC = DP == 256 ? 2 : 1;
  extern __shared__ __align__(16) uint8_t smem[];
  float* const wacc = reinterpret_cast<float*>(smem + NW * C::kQueryWords * 4);   // [NW][2][ROWS][kPitch]: parts of cut lines
  __shared__ float row_c[NW][ROWS];
  __shared__ int row_lim[NW][ROWS];
  __shared__ float2 wstat[NW][2][ROWS];
  __shared__ int64_t wline[NW][2];      // the line's first tile, or -1
  __shared__ int winfo[NW][2][3];       // its sequence, number and tiles
  __shared__ int64_t scan[NW], prefix[NW * 32];
  __shared__ int last_flag[2];

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  uint2* const qfrag = reinterpret_cast<uint2*>(smem) + warp * (C::kQueryWords / 2);   // [T][NR][KS][32]
  const int D = p.c.head_dim, G = p.group;
  const bool cut = sp.partial != nullptr;
  pdl_wait();
  pdl_trigger();

  auto tiles_of = [&](int keys) { return keys > kTile ? (keys + kTile - 1) / kTile : 1; };
  auto lines_of = [&](int n) { return ((n * G + ROWS - 1) / ROWS) * p.kv_count; };
  auto weight_of = [&](int b) { return (int64_t)lines_of(rows_of(p, b).count) * (cut ? tiles_of(keys_of(p, b)) : 1); };

  // ---- the share of this CTA and of its warps: the threads sum up their sequences' tiles
  const int per = (p.batch + NW * 32 - 1) / (NW * 32);
  const int b_lo = min(tid * per, p.batch), b_hi = min(b_lo + per, p.batch);
  int64_t mine = 0;
  for (int b = b_lo; b < b_hi; ++b) mine += weight_of(b);
  int64_t upto = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t v = __shfl_up_sync(0xffffffffu, upto, o);
    if (lane >= o) upto += v;
  }
  if (lane == 31) scan[warp] = upto;
  if (lane < 2) wline[warp][lane] = -1;
  __syncthreads();
  int64_t total = 0, before = 0;
#pragma unroll
  for (int w = 0; w < NW; ++w) {
    if (w == warp) before = total;
    total += scan[w];
  }
  prefix[tid] = before + upto - mine;
  int64_t share = (total + (int64_t)gridDim.x * NW - 1) / ((int64_t)gridDim.x * NW);   // of a warp
  if (cut && share < sp.least) share = sp.least;
  const int64_t cta_pos = (int64_t)blockIdx.x * share * NW, cta_end = min(cta_pos + share * NW, total);
  if (cta_pos >= cta_end) return;
  __syncthreads();
  int64_t pos = min(cta_pos + warp * share, cta_end);
  const int64_t end = min(pos + share, cta_end);
  int b = 0;
  int64_t base = 0;
  if (pos < end) {   // the last thread whose sequences begin at or before pos, then the sequence among its own
    int at = 0;
#pragma unroll
    for (int w = 0; w < NW; ++w) at += __popc(__ballot_sync(0xffffffffu, prefix[w * 32 + lane] <= pos));
    b = (at - 1) * per;
    base = prefix[at - 1];
  }
  bool bad = false;

  while (pos < end) {
    const Rows rw = rows_of(p, b);
    const int keys = keys_of(p, b), lines = lines_of(rw.count);
    const int tiles = cut ? tiles_of(keys) : 1;
    if (pos >= base + (int64_t)lines * tiles) {   // on to the next sequence
      base += (int64_t)lines * tiles;
      ++b;
      continue;
    }
    const int64_t into = pos - base;   // (a division of 64 bits takes over a hundred instructions)
    const int off = into < 0x7fffffff ? (int)into / tiles : (int)(into / tiles), t0 = cut ? (int)(into - (int64_t)off * tiles) : 0;
    const int kvh = p.kv_begin + off % p.kv_count, r0 = off / p.kv_count * ROWS;
    const int rows = min(ROWS, rw.count * G - r0);
    const int t1 = cut ? (int)min((int64_t)tiles, t0 + (end - pos)) : tiles_of(keys);
    const bool whole = !cut || (t0 == 0 && t1 == tiles);
    const int64_t line_pos = pos - t0;
    pos += cut ? t1 - t0 : 1;

    // the queries are on their way while the first keys are looked up: lane (g, t) takes of row g (of eight) what it is to multiply with
    uint32_t qr[NR][KC][8 * T];
#pragma unroll
    for (int n = 0; n < NR; ++n) {
      const int r = 8 * n + g;
      if (r >= rows) continue;
      const int i = rw.count == 1 ? 0 : (r0 + r) / G, h = kvh * G + (r0 + r) - i * G;
      const int64_t at = query_at(p, p.qs, rw, b, h, i) + 16 * t;
#pragma unroll
      for (int j = 0; j < KC; ++j)
        if (64 * j + 16 * t < D) load16<T>(p, at + 64 * j, sp.query_vec, qr[n][j]);
    }

    const int lim_least = visible(p, keys, rw.count, rw.count == 1 ? 0 : r0 / G);
    const int lim_most = rw.count == 1 ? lim_least : visible(p, keys, rw.count, (r0 + rows - 1) / G);
    const int t_end = min(t1, (lim_most + kTile - 1) / kTile);
    // ---- tiles t0 .. t_end - 1.  The blocks of the next 32 are looked up together, a lane each.
    const int32_t* table = p.c.table + b * p.c.table_stride;
    const int64_t pitch = p.c.stride[1];
    const uint8_t* const klane = p.c.k + kvh * p.c.stride[2] + 16 * t + (UB ? g * pitch : 0);
    const uint8_t* const vlane = p.c.v + kvh * p.c.stride[2] + VB * g + (UB ? 2 * t * pitch : 0);
    int entry = -1;
    float ks_l = 0.f, vs_l = 0.f;
    auto look_up = [&](int tile) {   // this lane's tile (UB: a tile lies in one block)
      entry = -1;
      ks_l = vs_l = 0.f;
      if (tile < t_end) {
        entry = checked_block(p.c, table[block_of(p.c, tile * kTile)], bad);
        if (entry >= 0) {
          ks_l = p.c.k_scale[(int64_t)entry * p.c.kv_heads + kvh];
          vs_l = p.c.v_scale[(int64_t)entry * p.c.kv_heads + kvh];
        }
      }
    };
    // K fragments: keys g, g + 8 of the tile; V fragments: keys 2t, 2t + 1, 2t + 8, 2t + 9.
    uint4 kr[2][KC];
    uint4 vr[4][VC];
    float ks[2], vs[2], ks_n[2], vs_n[2];   // of keys g and g + 8: this tile's, and (not UB) the next one's
    bool full_n = false;                    // all keys of the tile are there, and a row has DP bytes
    bool ok_n[2];
    int64_t row_n = -1;                     // UB: offset of the tile's first row, -1 without one
    int64_t vrow[UB ? 1 : 4];               // else of the values' rows
    auto find = [&](int tile, int slot) {   // and loads the keys
      const int key0 = tile * kTile;
      if constexpr (UB) {
        const int ent = __shfl_sync(0xffffffffu, entry, slot);
        const int first = key0 - block_of(p.c, key0) * p.c.block_size;
        row_n = ent >= 0 ? ent * p.c.stride[0] + first * pitch : -1;
        full_n = ent >= 0 && key0 + kTile <= keys && D == DP;
        if (full_n) {
          const uint8_t* at = klane + row_n;
#pragma unroll
          for (int q = 0; q < KC; ++q) kr[0][q] = ld_stream16(at + 64 * q);
          at += 8 * pitch;
#pragma unroll
          for (int q = 0; q < KC; ++q) kr[1][q] = ld_stream16(at + 64 * q);
        } else {
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            ok_n[j] = ent >= 0 && key0 + g + 8 * j < keys;
#pragma unroll
            for (int q = 0; q < KC; ++q)
              kr[j][q] = ok_n[j] && 64 * q + 16 * t < D ? ld_stream16(klane + row_n + 8 * j * pitch + 64 * q) : make_uint4(0, 0, 0, 0);
          }
        }
      } else {
        auto lookup = [&](int key, float* ksv, float* vsv) -> int64_t {
          if (key >= keys) return -1;
          const int at = block_of(p.c, key);
          const int ent = checked_block(p.c, table[at], bad);
          if (ent < 0) return -1;
          if (ksv) {
            *ksv = p.c.k_scale[(int64_t)ent * p.c.kv_heads + kvh];
            *vsv = p.c.v_scale[(int64_t)ent * p.c.kv_heads + kvh];
          }
          return ent * p.c.stride[0] + (key - at * p.c.block_size) * pitch;
        };
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          ks_n[j] = vs_n[j] = 0.f;
          const int64_t row = lookup(key0 + g + 8 * j, &ks_n[j], &vs_n[j]);
          ok_n[j] = row >= 0;
#pragma unroll
          for (int q = 0; q < KC; ++q)
            kr[j][q] = ok_n[j] && 64 * q + 16 * t < D ? ld_stream16(klane + row + 64 * q) : make_uint4(0, 0, 0, 0);
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) vrow[UB ? 0 : j] = lookup(key0 + 2 * t + (j & 1) + 8 * (j >> 1), nullptr, nullptr);
      }
    };
    auto load_v = [&](int key0) {
      if (UB && full_n) {
        const uint8_t* at = vlane + row_n;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
#pragma unroll
          for (int q = 0; q < VC; ++q) {
            if (VB == 8) {
              const uint2 x = ld_stream8(at + 128 * q);
              vr[j][q].x = x.x; vr[j][q].y = x.y;
            } else {
              vr[j][q] = ld_stream16(at + 128 * q);
            }
          }
          at += j == 1 ? 7 * pitch : pitch;
        }
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int k = (j & 1) + 8 * (j >> 1);
          const int64_t row = UB ? (row_n >= 0 && key0 + 2 * t + k < keys ? row_n + k * pitch : -1) : vrow[UB ? 0 : j];
#pragma unroll
          for (int q = 0; q < VC; ++q) {
            const bool there = row >= 0 && 128 * q + VB * g < D;
            if (VB == 8) {
              const uint2 x = there ? ld_stream8(vlane + row) : make_uint2(0, 0);
              vr[j][q].x = x.x; vr[j][q].y = x.y;
            } else {
              vr[j][q] = there ? ld_stream16(vlane + row + 128 * q) : make_uint4(0, 0, 0, 0);
            }
          }
        }
      }
    };
    int tile = t0, slot = 0;
    if (tile < t_end) {   // (the first keys are on their way while the queries are laid out)
      if (UB) look_up(tile + lane);
      find(tile, 0);
      load_v(tile * kTile);
    }

    // ---- queries: scaled by a power of two so that the largest element is in [2^12, 2^13), as fragments
#pragma unroll
    for (int n = 0; n < NR; ++n) {
      const int r = 8 * n + g;
      const bool valid = r < rows;
      float largest = 0.f;
#pragma unroll
      for (int j = 0; j < KC; ++j)
        if (valid && 64 * j + 16 * t < D) {
#pragma unroll
          for (int e = 0; e < 16; ++e) largest = fmaxf(largest, fabsf(widen<T>(p, qr[n][j], e)));
        }
      largest = fmaxf(largest, __shfl_xor_sync(0xffffffffu, largest, 1));
      largest = fmaxf(largest, __shfl_xor_sync(0xffffffffu, largest, 2));
      int up = 12 - ((int)(__float_as_uint(largest) >> 23) - 127);   // (zeros and what is below the normal floats: 2^126)
      up = max(-110, min(up, 126));
      const float f = __uint_as_float((uint32_t)(up + 127) << 23);
#pragma unroll
      for (int j = 0; j < KC; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          __half2 hi[2] = {}, lo[2] = {};
          if (valid && 64 * j + 16 * t < D) {
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const float a = widen<T>(p, qr[n][j], 4 * i + 2 * e) * f, c = widen<T>(p, qr[n][j], 4 * i + 2 * e + 1) * f;
              hi[e] = __floats2half2_rn(a, c);
              if (T == 2) lo[e] = __floats2half2_rn(a - __low2float(hi[e]), c - __high2float(hi[e]));
            }
          }
          uint2* const dst = qfrag + (n * KS + 4 * j + i) * 32 + lane;
          dst[0] = make_uint2(*reinterpret_cast<uint32_t*>(&hi[0]), *reinterpret_cast<uint32_t*>(&hi[1]));
          if (T == 2) dst[NR * KS * 32] = make_uint2(*reinterpret_cast<uint32_t*>(&lo[0]), *reinterpret_cast<uint32_t*>(&lo[1]));
        }
      if (t == 0) {
        row_c[warp][r] = p.scale * __uint_as_float((uint32_t)(127 - up) << 23) * (p.softcap > 0.f ? 1.f : kLog2e);
        row_lim[warp][r] = !valid ? keys : (rw.count == 1 ? lim_least : visible(p, keys, rw.count, (r0 + r) / G));
      }
    }
    __syncwarp();

    float acc[NR][MT][4];
    float m[NR][2], l[NR][2], c[NR][2];
    int lim[NR][2];
    float vref = 0.f, inv_vref = 0.f;
#pragma unroll
    for (int n = 0; n < NR; ++n) {
#pragma unroll
      for (int j = 0; j < MT; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[n][j][e] = 0.f;
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        m[n][e] = kUnset;
        l[n][e] = 0.f;
        c[n][e] = row_c[warp][8 * n + 2 * t + e];
        lim[n][e] = row_lim[warp][8 * n + 2 * t + e];
      }
    }
    for (; tile < t_end; ++tile) {
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        ks[j] = UB ? __shfl_sync(0xffffffffu, ks_l, slot) : ks_n[j];
        vs[j] = UB ? __shfl_sync(0xffffffffu, vs_l, slot) : vs_n[j];
      }
      // rows of which not all keys of the tile are seen, or keys that are not there
      const int key0 = tile * kTile;
      const bool full = full_n, edge = !full || key0 + kTile > lim_least;
      bool ok[2] = {true, true};
      if (!full) {
        ok[0] = ok_n[0];
        ok[1] = ok_n[1];
      }
      float s[NR][4];
#pragma unroll
      for (int n = 0; n < NR; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[n][e] = 0.f;
#pragma unroll
      for (int q = 0; q < KC; ++q) {
        const uint32_t w0[4] = {kr[0][q].x, kr[0][q].y, kr[0][q].z, kr[0][q].w}, w1[4] = {kr[1][q].x, kr[1][q].y, kr[1][q].z, kr[1][q].w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint32_t a0 = codes_to_f16(w0[i]), a1 = codes_to_f16(w1[i]), a2 = codes_to_f16_hi(w0[i]), a3 = codes_to_f16_hi(w1[i]);
#pragma unroll
          for (int n = 0; n < NR; ++n)
#pragma unroll
            for (int term = 0; term < T; ++term) {
              const uint2 bq = qfrag[((term * NR + n) * KS + 4 * q + i) * 32 + lane];
              mma16816<__half>(s[n], a0, a1, a2, a3, bq.x, bq.y);
            }
        }
      }
      // the next tile's keys, while this one's weights are formed
      const int next = tile + 1;
      if (next < t_end) {
        if (++slot == 32) {
          slot = 0;
          if (UB) look_up(next + lane);
        }
        find(next, slot);
      }

      uint32_t nan_keys = 0;   // keys of which a value is NaN: where rows do not see the key it must not reach them, so that it goes through the logit
      if (edge) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          bool hit = false;
#pragma unroll
          for (int q = 0; q < VC; ++q) {
            hit = hit || any_nan(vr[j][q].x) || any_nan(vr[j][q].y);
            vr[j][q].x = without_nan(vr[j][q].x); vr[j][q].y = without_nan(vr[j][q].y);
            if (VB == 16) {
              hit = hit || any_nan(vr[j][q].z) || any_nan(vr[j][q].w);
              vr[j][q].z = without_nan(vr[j][q].z); vr[j][q].w = without_nan(vr[j][q].w);
            }
          }
          const uint32_t who = __ballot_sync(0xffffffffu, hit);   // lanes (g, t): key 2t + (j & 1) + 8 (j >> 1)
#pragma unroll
          for (int tt = 0; tt < 4; ++tt)
            if (who & (0x11111111u << tt)) nan_keys |= 1u << (2 * tt + (j & 1) + 8 * (j >> 1));
        }
      }
      bool grow = false;
#pragma unroll
      for (int n = 0; n < NR; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          float x = s[n][e] * (c[n][e & 1] * ks[e >> 1]);
          if (p.softcap > 0.f) x = p.softcap * kLog2e * (T == 2 ? tanhf(x / p.softcap) : tanh_ex2(x / p.softcap));
          if (edge) {
            const int k = g + 8 * (e >> 1);
            if (nan_keys >> k & 1) x = NAN;
            if (!ok[e >> 1] || key0 + k >= lim[n][e & 1]) x = -INFINITY;
          }
          s[n][e] = x;
          grow = grow || x > m[n][e & 1] + kLazy;
        }
      if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
        for (int n = 0; n < NR; ++n)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float top = fmaxf(s[n][e], s[n][e + 2]);
#pragma unroll
            for (int o = 4; o < 32; o <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
            const float now = fmaxf(m[n][e], top), keep = ex2_approx(m[n][e] - now);
            m[n][e] = now;
            l[n][e] *= keep;
#pragma unroll
            for (int j = 0; j < MT; ++j) {
              acc[n][j][e] *= keep;
              acc[n][j][e + 2] *= keep;
            }
          }
      }
      // scales of the values relative to the largest so far
      float vtop = fmaxf(vs[0], vs[1]);
      if (!UB) {
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) vtop = fmaxf(vtop, __shfl_xor_sync(0xffffffffu, vtop, o));
      }
      if (vtop > vref) {
        const float keep = vref / vtop;
        vref = vtop;
        inv_vref = 1.f / vtop;
#pragma unroll
        for (int n = 0; n < NR; ++n)
#pragma unroll
          for (int j = 0; j < MT; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[n][j][e] *= keep;
      }
      uint32_t ph[NR][2], pl[NR][2];
#pragma unroll
      for (int n = 0; n < NR; ++n)
#pragma unroll
        for (int j = 0; j < 2; ++j) {   // key g + 8 j, rows 2t and 2t + 1
          float a = ex2_approx(s[n][2 * j] - (m[n][0] - kLift)), w = ex2_approx(s[n][2 * j + 1] - (m[n][1] - kLift));
          l[n][0] += a;
          l[n][1] += w;
          const float f = vs[j] * inv_vref;
          a *= f;
          w *= f;
          const __half2 hi = __floats2half2_rn(a, w);
          ph[n][j] = transpose8x8(*reinterpret_cast<const uint32_t*>(&hi));
          if constexpr (T == 2) {
            const __half2 lo = __floats2half2_rn(a - __low2float(hi), w - __high2float(hi));
            pl[n][j] = transpose8x8(*reinterpret_cast<const uint32_t*>(&lo));
          }
        }
#pragma unroll
      for (int q = 0; q < VC; ++q) {
        const uint32_t w[4][4] = {{vr[0][q].x, vr[0][q].y, vr[0][q].z, vr[0][q].w}, {vr[1][q].x, vr[1][q].y, vr[1][q].z, vr[1][q].w},
                                  {vr[2][q].x, vr[2][q].y, vr[2][q].z, vr[2][q].w}, {vr[3][q].x, vr[3][q].y, vr[3][q].z, vr[3][q].w}};
#pragma unroll
        for (int i = 0; i < VB / 4; ++i)
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            const uint32_t u = __byte_perm(w[0][i], w[1][i], half ? 0x7362 : 0x5140), v = __byte_perm(w[2][i], w[3][i], half ? 0x7362 : 0x5140);
            const uint32_t a0 = codes_to_f16(u), a1 = codes_to_f16_hi(u), a2 = codes_to_f16(v), a3 = codes_to_f16_hi(v);
            const int j = (VB / 2) * q + 2 * i + half;
#pragma unroll
            for (int n = 0; n < NR; ++n) {
              mma16816<__half>(acc[n][j], a0, a1, a2, a3, ph[n][0], ph[n][1]);
              if constexpr (T == 2) mma16816<__half>(acc[n][j], a0, a1, a2, a3, pl[n][0], pl[n][1]);
            }
          }
      }
      if (next < t_end) load_v(next * kTile);
    }

    // ---- a whole line is written, a part of one kept: of the line that began before this warp's share, and of the one that goes on
    float sum[NR][2];
#pragma unroll
    for (int n = 0; n < NR; ++n)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        sum[n][e] = l[n][e];
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) sum[n][e] += __shfl_xor_sync(0xffffffffu, sum[n][e], o);
      }
    const int part = t0 == 0 ? 1 : 0;
#pragma unroll
    for (int n = 0; n < NR; ++n)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int r = 8 * n + 2 * t + e;
        if (r >= rows) continue;
        const float f = whole ? (sum[n][e] == 0.f ? 0.f : vref / sum[n][e]) : vref;
        const int i = rw.count == 1 ? 0 : (r0 + r) / G, h = kvh * G + (r0 + r) - i * G;
        const int64_t at = whole ? query_at(p, p.os, rw, b, h, i) : 0;
        float* const to = wacc + ((warp * 2 + part) * ROWS + r) * C::kPitch;
#pragma unroll
        for (int j = 0; j < MT; j += 2) {
          const int d = DP == 256 ? 128 * (j / 8) + 16 * g + 2 * (j % 8) : VB * g + 2 * j;
          const float4 o = make_float4(acc[n][j][e] * f, acc[n][j][e + 2] * f, acc[n][j + 1][e] * f, acc[n][j + 1][e + 2] * f);
          if (!whole) *reinterpret_cast<float4*>(to + d) = o;
          else if (d < D) store4(p, at + d, sp.out_vec, o);
        }
        if (g == 0) {
          if (!whole) wstat[warp][part][r] = make_float2(m[n][e] - kLift, sum[n][e]);
          else if (p.lse) *lse_at(p, rw, h, i) = sum[n][e] == 0.f ? -INFINITY : (m[n][e] - kLift + log2f(sum[n][e])) * kLn2;
        }
      }
    if (!whole && lane == 0) {
      wline[warp][part] = line_pos;
      winfo[warp][part][0] = b;
      winfo[warp][part][1] = off;
      winfo[warp][part][2] = tiles;
    }
    __syncwarp();
  }
  if (bad && p.status) atomicOr(p.status, kStatusBadBlock);
  __syncthreads();

  // ---- the parts of a line in this CTA are consecutive: merged by all threads, and written, or left in the workspace
  auto finish = [&](const Rows& rw, int b, int off, int r, int d, float4 o, float top, float sum) {
    const int kvh = p.kv_begin + off % p.kv_count, r0 = off / p.kv_count * ROWS;
    const int i = (r0 + r) / G, h = kvh * G + (r0 + r) - i * G;
    const float f = sum == 0.f ? 0.f : 1.f / sum;
    store4(p, query_at(p, p.os, rw, b, h, i) + d, sp.out_vec, make_float4(o.x * f, o.y * f, o.z * f, o.w * f));
    if (p.lse && d == 0) *lse_at(p, rw, h, i) = sum == 0.f ? -INFINITY : (top + log2f(sum)) * kLn2;
  };
  int64_t handed0 = -1, handed1 = -1;   // lines of which other CTAs have parts too: the one that began before, the one that goes on
  int at0 = 0, at1 = 0;
  unsigned used = 0;   // slots that hold a part
#pragma unroll
  for (int q = 0; q < 2 * NW; ++q) used |= (unsigned)(wline[q >> 1][q & 1] >= 0) << q;
  while (used) {
    const int at = __ffs(used) - 1;
    const int64_t line = wline[at >> 1][at & 1];
    unsigned group = 0;
    for (unsigned left = used; left; left &= left - 1) {
      const int q = __ffs(left) - 1;
      if (wline[q >> 1][q & 1] != line) break;
      group |= 1u << q;
    }
    used &= ~group;
    const int b = winfo[at >> 1][at & 1][0], off = winfo[at >> 1][at & 1][1], tiles = winfo[at >> 1][at & 1][2];
    const Rows rw = rows_of(p, b);
    const int rows = min(ROWS, rw.count * G - off / p.kv_count * ROWS);
    const bool early = line < cta_pos, late = line + tiles > cta_end, whole = !early && !late;
    const int64_t slot = 2 * (int64_t)blockIdx.x + (early ? 0 : 1);
    for (int x = tid; x < rows * (DP / 4); x += NW * 32) {
      const int r = x / (DP / 4), d = x % (DP / 4) * 4;
      if (d >= D) continue;
      float top = kUnset;
      for (unsigned left = group; left; left &= left - 1) top = fmaxf(top, (&wstat[0][0][0])[(__ffs(left) - 1) * ROWS + r].x);
      float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
      float sum = 0.f;
      for (unsigned left = group; left; left &= left - 1) {
        const int q = __ffs(left) - 1;
        const float2 st = (&wstat[0][0][0])[q * ROWS + r];
        const float f = ex2_approx(st.x - top);
        const float4 v = *reinterpret_cast<const float4*>(wacc + (q * ROWS + r) * C::kPitch + d);
        sum += f * st.y;
        o.x += f * v.x; o.y += f * v.y; o.z += f * v.z; o.w += f * v.w;
      }
      if (whole) {
        finish(rw, b, off, r, d, o, top, sum);
      } else {
        __stcg(reinterpret_cast<float4*>(sp.partial + (slot * ROWS + r) * DP + d), o);
        if (d == 0) __stcg(sp.stats + slot * ROWS + r, make_float2(top, sum));
      }
    }
    if (early) {
      handed0 = line;
      at0 = at;
    } else if (late) {
      handed1 = line;
      at1 = at;
    }
  }
  if (handed0 < 0 && handed1 < 0) return;
  // CTAs first .. first + parts - 1 have a part of such a line; in the CTA where it begins it is the last one, elsewhere the first
  const int64_t cta_share = share * NW;
  __syncthreads();
  if (tid < 2) {
    const int64_t line = tid ? handed1 : handed0;
    bool last = false;
    if (line >= 0) {
      const int at = tid ? at1 : at0, first = tid ? (int)blockIdx.x : (int)(line / cta_share);
      const int parts = (int)((line + winfo[at >> 1][at & 1][2] - 1) / cta_share) - first + 1;
      __threadfence();   // (what the other threads wrote, too: the barrier lies between)
      last = atomicInc(p.counters + first, parts - 1) == (unsigned)(parts - 1);
      __threadfence();
    }
    last_flag[tid] = last;
  }
  __syncthreads();
#pragma unroll 1
  for (int k = 0; k < 2; ++k) {
    if (!last_flag[k]) continue;
    const int64_t line = k ? handed1 : handed0;
    const int at = k ? at1 : at0;
    const int* info = winfo[at >> 1][at & 1];
    const int b = info[0], off = info[1], tiles = info[2];
    const int first = k ? (int)blockIdx.x : (int)(line / cta_share), parts = (int)((line + tiles - 1) / cta_share) - first + 1;
    const Rows rw = rows_of(p, b);
    const int rows = min(ROWS, rw.count * G - off / p.kv_count * ROWS);
    for (int x = tid; x < rows * (DP / 4); x += NW * 32) {
      const int r = x / (DP / 4), d = x % (DP / 4) * 4;
      if (d >= D) continue;
      float top = kUnset, sum = 0.f;
      float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
      for (int q = 0; q < parts; q += 8) {
        float2 st[8];
        float4 v[8];
#pragma unroll
        for (int u = 0; u < 8; ++u) {
          const int part = min(q + u, parts - 1);
          const int64_t from = (int64_t)(2 * (first + part) + (part == 0)) * ROWS + r;
          st[u] = __ldcg(sp.stats + from);
          v[u] = __ldcg(reinterpret_cast<const float4*>(sp.partial + from * DP + d));
        }
        float now = top;
#pragma unroll
        for (int u = 0; u < 8; ++u) now = fmaxf(now, st[u].x);
        const float keep = ex2_approx(top - now);
        top = now;
        sum *= keep;
        o.x *= keep; o.y *= keep; o.z *= keep; o.w *= keep;
#pragma unroll
        for (int u = 0; u < 8; ++u) {
          if (q + u >= parts) continue;
          const float f = ex2_approx(st[u].x - top);
          sum += f * st[u].y;
          o.x += f * v[u].x; o.y += f * v[u].y; o.z += f * v[u].z; o.w += f * v[u].w;
        }
      }
      finish(rw, b, off, r, d, o, top, sum);
    }
  }
}

template <int DP, int NR, int T, bool UB>
int resident(int num_sms) {
  static const int ctas = [] {
    int n = 0;
    auto k = kv8_split_kernel<DP, NR, T, UB>;
    if (cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)Config<DP, NR, T, UB>::kSmem) != cudaSuccess ||
        cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, k, Config<DP, NR, T, UB>::kWarps * 32, Config<DP, NR, T, UB>::kSmem) != cudaSuccess) {
      cudaGetLastError();
      return 0;
    }
    return n;
  }();
  const int n = ctas * num_sms;
  return n < 1 ? 1 : (n < kCounters ? n : kCounters);
}

// One instantiation: its workspace, or its launch (workspace null: the lines are not cut).
template <int DP, int NR, int T, bool UB>
cudaError_t one(const Attend* p, int num_sms, void* workspace, int64_t* bytes, uint64_t* raised, cudaStream_t stream) {
  using C = Config<DP, NR, T, UB>;
  const int grid = resident<DP, NR, T, UB>(num_sms);
  const int64_t acc = (int64_t)2 * grid * C::kRows * DP * 4;
  if (bytes) {
    *bytes = acc + (int64_t)2 * grid * C::kRows * 8;
    return cudaSuccess;
  }
  auto k = kv8_split_kernel<DP, NR, T, UB>;
  const int id = ((DP == 64 ? 0 : DP == 128 ? 1 : 2) * 2 + NR - 1) * 4 + (T - 1) * 2 + (UB ? 1 : 0);
  if (!(*raised >> id & 1)) {   // once a handle: the limit belongs to the context
    const cudaError_t e = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)C::kSmem);
    if (e != cudaSuccess) return e;
    *raised |= 1ull << id;
  }
  Split sp;
  sp.partial = static_cast<float*>(workspace);
  sp.stats = workspace ? reinterpret_cast<float2*>(static_cast<char*>(workspace) + acc) : nullptr;
  sp.least = 2;
  auto vec = [](const void* ptr, const int64_t* st, int esz, int bytes) {
    return ((uintptr_t)ptr | (uint64_t)(st[0] * esz) | (uint64_t)(st[1] * esz) | (uint64_t)(st[2] * esz)) % bytes == 0;
  };
  sp.query_vec = vec(p->q, p->qs, p->dtype == AIDN_F32 ? 4 : 2, 16);
  sp.out_vec = vec(p->out, p->os, p->out_f32 ? 4 : 2, p->out_f32 ? 16 : 8);
  return launch_dependent(k, dim3((unsigned)grid), C::kWarps * 32, C::kSmem, stream, *p, sp);
}

template <int DP, int NR, int T>
cudaError_t pick_block(bool ub, const Attend* p, int num_sms, void* workspace, int64_t* bytes, uint64_t* raised, cudaStream_t stream) {
  return ub ? one<DP, NR, T, true>(p, num_sms, workspace, bytes, raised, stream) : one<DP, NR, T, false>(p, num_sms, workspace, bytes, raised, stream);
}
template <int DP, int T>
cudaError_t pick_rows(int64_t rows, bool ub, const Attend* p, int num_sms, void* workspace, int64_t* bytes, uint64_t* raised, cudaStream_t stream) {
  if (rows <= 8) return pick_block<DP, 1, T>(ub, p, num_sms, workspace, bytes, raised, stream);
  return pick_block<DP, 2, T>(ub, p, num_sms, workspace, bytes, raised, stream);
}
template <int DP>
cudaError_t pick(bool exact, int64_t rows, bool ub, const Attend* p, int num_sms, void* workspace, int64_t* bytes, uint64_t* raised, cudaStream_t stream) {
  return exact ? pick_rows<DP, 2>(rows, ub, p, num_sms, workspace, bytes, raised, stream) : pick_rows<DP, 1>(rows, ub, p, num_sms, workspace, bytes, raised, stream);
}
cudaError_t pick_dim(int dim, bool exact, int64_t rows, bool ub, const Attend* p, int num_sms, void* workspace, int64_t* bytes, uint64_t* raised, cudaStream_t stream) {
  if (dim <= 64) return pick<64>(exact, rows, ub, p, num_sms, workspace, bytes, raised, stream);
  if (dim <= 128) return pick<128>(exact, rows, ub, p, num_sms, workspace, bytes, raised, stream);
  return pick<256>(exact, rows, ub, p, num_sms, workspace, bytes, raised, stream);
}

}  // namespace

bool split_supported(const Attend& p) {
  if (p.c.head_dim % 16 != 0 || p.mask_kind != AIDN_MASK_NONE) return false;
  if ((uintptr_t)p.c.k % 16 != 0 || (uintptr_t)p.c.v % 16 != 0) return false;
  for (int i = 0; i < 3; ++i)
    if (p.c.stride[i] % 16 != 0) return false;
  return true;
}
// (whatever the block size: the larger of the two kernels' needs)
int64_t split_workspace_bytes(int head_dim, bool exact, int64_t rows, int num_sms) {
  int64_t most = 0;
  for (int ub = 0; ub < 2; ++ub) {
    int64_t n = 0;
    pick_dim(head_dim, exact, rows, ub, nullptr, num_sms, nullptr, &n, nullptr, nullptr);
    if (n > most) most = n;
  }
  return most;
}
cudaError_t launch_attend_split(const Attend& p, int num_sms, void* workspace, int64_t workspace_bytes, uint64_t* raised, cudaStream_t stream) {
  const bool exact = p.out_f32 != 0;
  const int64_t rows = p.seq_q * p.group;
  const bool ub = p.c.block_size % kTile == 0;
  int64_t need = 0;
  pick_dim(p.c.head_dim, exact, rows, ub, nullptr, num_sms, nullptr, &need, nullptr, nullptr);
  if (workspace_bytes < need || (uintptr_t)workspace % 16 != 0) workspace = nullptr;
  return pick_dim(p.c.head_dim, exact, rows, ub, &p, num_sms, workspace, nullptr, raised, stream);
}

}  // namespace kv8
}  // namespace aidn
