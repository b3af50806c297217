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
  int least;         // tiles of a share
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
// tanh to 3e-7 of 1: the logits are off by that times the cap.
__device__ __forceinline__ float tanh_ex2(float x) { return 1.f - __fdividef(2.f, 1.f + ex2_approx(fminf(x * (2.f * kLog2e), 80.f))); }
// Whether any of four codes is a NaN.
__device__ __forceinline__ bool any_nan(uint32_t x) { return (((x & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u) != 0; }
__device__ __forceinline__ uint32_t without_nan(uint32_t x) {
  const uint32_t hit = (((x & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u) >> 7;   // 1 in the bytes that are
  return x & ~(hit * 0xffu);
}

// What lies past the D bytes of a key is never read: the fragments' elements from D on are zeros.
template <int DP, int NR, int T, bool UB>
struct Config {
  static constexpr int kWarps = NR == 1 ? 8 : 4;
  static constexpr int kMinCtas = DP == 256 ? (NR == 1 ? 1 : 1) : (NR == 1 ? 2 : (NR == 2 && DP == 64 ? 4 : (NR == 4 && DP == 128 ? 2 : 3)));
  static constexpr int kSteps = DP / 16;                 // of 16 elements: fragments of a key
  static constexpr int kRows = 8 * NR;
  static constexpr int kPitch = DP + 4;                  // floats between the rows of a warp's results
  static constexpr int kQueryWords = T * NR * kSteps * 32 * 2;
  static constexpr size_t kSmem = (size_t)kQueryWords * 4 + (size_t)kWarps * kRows * kPitch * 4;
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
  uint2* const qfrag = reinterpret_cast<uint2*>(smem);                          // [T][NR][KS][32]
  float* const wacc = reinterpret_cast<float*>(smem + C::kQueryWords * 4);      // [NW][ROWS][kPitch]
  __shared__ float row_c[ROWS];
  __shared__ int row_lim[ROWS];
  __shared__ float2 wstat[NW][ROWS];
  __shared__ float wref[NW];
  __shared__ int64_t scan[NW + 1];
  __shared__ int found_b;
  __shared__ int64_t found_base;
  __shared__ int last_flag;

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  const int D = p.c.head_dim, G = p.group;
  const bool cut = sp.partial != nullptr;
  pdl_wait();
  pdl_trigger();

  auto tiles_of = [&](int keys) { return keys > kTile ? (keys + kTile - 1) / kTile : 1; };
  auto lines_of = [&](int n) { return ((n * G + ROWS - 1) / ROWS) * p.kv_count; };

  // ---- the share of this CTA: all threads sum their sequences' tiles, the one whose sequences hold its first tile says so
  const int per = (p.batch + NW * 32 - 1) / (NW * 32);
  const int b_lo = min(tid * per, p.batch), b_hi = min(b_lo + per, p.batch);
  int64_t mine = 0;
  for (int b = b_lo; b < b_hi; ++b) {
    const int64_t lines = lines_of(rows_of(p, b).count);
    mine += cut ? lines * tiles_of(keys_of(p, b)) : lines;
  }
  int64_t upto = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t v = __shfl_up_sync(0xffffffffu, upto, o);
    if (lane >= o) upto += v;
  }
  if (lane == 31) scan[warp] = upto;
  __syncthreads();
  int64_t total = 0, before = 0;
#pragma unroll
  for (int w = 0; w < NW; ++w) {
    if (w == warp) before = total;
    total += scan[w];
  }
  before += upto - mine;
  int64_t share = (total + gridDim.x - 1) / gridDim.x;
  if (cut) {
    if (share < sp.least) share = sp.least;
    share = (share + NW - 1) / NW * NW;
  }
  int64_t pos = (int64_t)blockIdx.x * share;
  const int64_t end = min(pos + share, total);
  if (pos >= end) return;
  if (pos >= before && pos < before + mine) {
    int64_t base = before;
    for (int b = b_lo; b < b_hi; ++b) {
      const int64_t lines = lines_of(rows_of(p, b).count), w = cut ? lines * tiles_of(keys_of(p, b)) : lines;
      if (pos < base + w) {
        found_b = b;
        found_base = base;
        break;
      }
      base += w;
    }
  }
  __syncthreads();
  int b = found_b;
  int64_t base = found_base;
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
    const int off = (int)((pos - base) / tiles), t0 = cut ? (int)((pos - base) % tiles) : 0;
    const int kvh = p.kv_begin + off % p.kv_count, r0 = off / p.kv_count * ROWS;
    const int rows = min(ROWS, rw.count * G - r0);
    const int t1 = cut ? (int)min((int64_t)tiles, t0 + (end - pos)) : tiles_of(keys);
    const bool whole = !cut || (t0 == 0 && t1 == tiles);
    const int64_t line_pos = pos - t0;
    pos += cut ? t1 - t0 : 1;

    // ---- queries: scaled by a power of two so that the largest element is in [2^12, 2^13), as fragments
    for (int r = warp; r < ROWS; r += NW) {
      float x[DP / 128 > 0 ? DP / 128 : 1][4];
      float largest = 0.f;
      const bool valid = r < rows;
      const int i = (r0 + r) / G, h = kvh * G + (r0 + r) % G;
      const int64_t at = valid ? query_at(p, p.qs, rw, b, h, i) : 0;
#pragma unroll
      for (int j = 0; j < (DP + 127) / 128; ++j) {
        const int d = 128 * j + 4 * lane;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          float v = 0.f;
          if (valid && d < D) {
            if (p.dtype == AIDN_F32) v = static_cast<const float*>(p.q)[at + d + e];
            else if (p.dtype == AIDN_F16) v = __half2float(static_cast<const __half*>(p.q)[at + d + e]);
            else v = __bfloat162float(static_cast<const __nv_bfloat16*>(p.q)[at + d + e]);
          }
          x[j][e] = v;
          largest = fmaxf(largest, fabsf(v));
        }
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) largest = fmaxf(largest, __shfl_xor_sync(0xffffffffu, largest, o));
      int up = 12 - ((int)(__float_as_uint(largest) >> 23) - 127);   // (zeros and what is below the normal floats: 2^126)
      up = max(-110, min(up, 126));
      const float f = __uint_as_float((uint32_t)(up + 127) << 23);
#pragma unroll
      for (int j = 0; j < (DP + 127) / 128; ++j) {
        const int d = 128 * j + 4 * lane;
        if (d >= DP) continue;
        const int step = d / 64 * 4 + d % 16 / 4, to = (r % 8) * 4 + d % 64 / 16;
        __half2 hi[2], lo[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float a = x[j][2 * e] * f, c = x[j][2 * e + 1] * f;
          hi[e] = __floats2half2_rn(a, c);
          if (T == 2) lo[e] = __floats2half2_rn(a - __low2float(hi[e]), c - __high2float(hi[e]));
        }
        qfrag[((r / 8) * KS + step) * 32 + to] = make_uint2(*reinterpret_cast<uint32_t*>(&hi[0]), *reinterpret_cast<uint32_t*>(&hi[1]));
        if (T == 2)
          qfrag[((NR + r / 8) * KS + step) * 32 + to] = make_uint2(*reinterpret_cast<uint32_t*>(&lo[0]), *reinterpret_cast<uint32_t*>(&lo[1]));
      }
      if (lane == 0) {
        row_c[r] = p.scale * __uint_as_float((uint32_t)(127 - up) << 23) * (p.softcap > 0.f ? 1.f : kLog2e);
        row_lim[r] = valid ? visible(p, keys, rw.count, i) : keys;
      }
    }
    __syncthreads();

    const int lim_least = visible(p, keys, rw.count, r0 / G), lim_most = visible(p, keys, rw.count, (r0 + rows - 1) / G);
    const int t_end = min(t1, (lim_most + kTile - 1) / kTile);
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
        c[n][e] = row_c[8 * n + 2 * t + e];
        lim[n][e] = row_lim[8 * n + 2 * t + e];
      }
    }
    uint2 qreg[NR == 1 && T == 1 ? KS : 1];
    if constexpr (NR == 1 && T == 1) {
#pragma unroll
      for (int s = 0; s < KS; ++s) qreg[s] = qfrag[s * 32 + lane];
    }

    // ---- tiles of this warp: t0 + warp, + NW, ...  The blocks of the next 32 are looked up together, a lane each.
    const int32_t* table = p.c.table + b * p.c.table_stride;
    const uint8_t* const kbase = p.c.k + kvh * p.c.stride[2];
    const uint8_t* const vbase = p.c.v + kvh * p.c.stride[2];
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
    uint4 kr[2][KC];
    uint4 vr[4][VC];
    float ks[2], vs[2], ks_n[2], vs_n[2];   // of keys g and g + 8: this tile's, and the next one's
    bool ok[2], ok_n[2];
    int64_t vrow[4];
    // Rows and scales of a tile's keys.  K fragments: keys g, g + 8; V fragments: keys 2t, 2t + 1, 2t + 8, 2t + 9.
    auto find = [&](int tile, int slot) {
      const int key0 = tile * kTile;
      if constexpr (UB) {
        const int ent = __shfl_sync(0xffffffffu, entry, slot);
        ks_n[0] = ks_n[1] = __shfl_sync(0xffffffffu, ks_l, slot);
        vs_n[0] = vs_n[1] = __shfl_sync(0xffffffffu, vs_l, slot);
        const int first = key0 - block_of(p.c, key0) * p.c.block_size;
        const int64_t row = ent * p.c.stride[0] + first * p.c.stride[1];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          ok_n[j] = ent >= 0 && key0 + g + 8 * j < keys;
          const uint8_t* at = kbase + row + (g + 8 * j) * p.c.stride[1];
#pragma unroll
          for (int q = 0; q < KC; ++q)
            kr[j][q] = ok_n[j] && 64 * q + 16 * t < D ? ld_stream16(at + 64 * q + 16 * t) : make_uint4(0, 0, 0, 0);
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int k = 2 * t + (j & 1) + 8 * (j >> 1);
          vrow[j] = ent >= 0 && key0 + k < keys ? row + k * p.c.stride[1] : -1;
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
          return ent * p.c.stride[0] + (key - at * p.c.block_size) * p.c.stride[1];
        };
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          ks_n[j] = vs_n[j] = 0.f;
          const int64_t row = lookup(key0 + g + 8 * j, &ks_n[j], &vs_n[j]);
          ok_n[j] = row >= 0;
#pragma unroll
          for (int q = 0; q < KC; ++q)
            kr[j][q] = ok_n[j] && 64 * q + 16 * t < D ? ld_stream16(kbase + row + 64 * q + 16 * t) : make_uint4(0, 0, 0, 0);
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) vrow[j] = lookup(key0 + 2 * t + (j & 1) + 8 * (j >> 1), nullptr, nullptr);
      }
    };
    auto load_v = [&]() {
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int q = 0; q < VC; ++q) {
          const int d = 128 * q + VB * g;
          if (VB == 8) {
            const uint2 x = vrow[j] >= 0 && d < D ? ld_stream8(vbase + vrow[j] + d) : make_uint2(0, 0);
            vr[j][q] = make_uint4(x.x, x.y, 0, 0);
          } else {
            vr[j][q] = vrow[j] >= 0 && d < D ? ld_stream16(vbase + vrow[j] + d) : make_uint4(0, 0, 0, 0);
          }
        }
    };
    int tile = t0 + warp, slot = 0;
    if (tile < t_end) {
      if (UB) look_up(tile + NW * lane);
      find(tile, 0);
      load_v();
    }
    for (; tile < t_end; tile += NW) {
#pragma unroll
      for (int j = 0; j < 2; ++j) { ks[j] = ks_n[j]; vs[j] = vs_n[j]; ok[j] = ok_n[j]; }
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
              uint2 bq;
              if constexpr (NR == 1 && T == 1) bq = qreg[4 * q + i];
              else bq = qfrag[((term * NR + n) * KS + 4 * q + i) * 32 + lane];
              mma16816<__half>(s[n], a0, a1, a2, a3, bq.x, bq.y);
            }
        }
      }
      // the next tile's keys, while this one's weights are formed
      const int next = tile + NW;
      if (next < t_end) {
        if (++slot == 32) {
          slot = 0;
          if (UB) look_up(next + NW * lane);
        }
        find(next, slot);
      }

      const int key0 = tile * kTile;
      // rows of which not all keys of the tile are seen, or keys that are not there
      const bool edge = key0 + kTile > lim_least || __any_sync(0xffffffffu, !ok[0] || !ok[1]);
      uint32_t nan_keys = 0;   // keys of which a value is NaN: where rows do not see the key it must not reach them, so that it goes through the logit
      if (edge) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          bool hit = false;
#pragma unroll
          for (int q = 0; q < VC; ++q) {
            hit = hit || any_nan(vr[j][q].x) || any_nan(vr[j][q].y) || any_nan(vr[j][q].z) || any_nan(vr[j][q].w);
            vr[j][q].x = without_nan(vr[j][q].x); vr[j][q].y = without_nan(vr[j][q].y);
            vr[j][q].z = without_nan(vr[j][q].z); vr[j][q].w = without_nan(vr[j][q].w);
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
      if (next < t_end) load_v();
    }

    // ---- the warps' results meet in shared memory
#pragma unroll
    for (int n = 0; n < NR; ++n)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float sum = l[n][e];
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        if (g == 0) wstat[warp][8 * n + 2 * t + e] = make_float2(m[n][e] - kLift, sum);
        float* to = wacc + (warp * ROWS + 8 * n + 2 * t + e) * C::kPitch;
#pragma unroll
        for (int j = 0; j < MT; ++j) {
          const int d = DP == 256 ? 128 * (j / 8) + 16 * g + 2 * (j % 8) : VB * g + 2 * j;
          *reinterpret_cast<float2*>(to + d) = make_float2(acc[n][j][e], acc[n][j][e + 2]);
        }
      }
    if (lane == 0) wref[warp] = vref;
    __syncthreads();

    auto write = [&](int r, int d, float4 o, float top, float sum) {
      const int i = (r0 + r) / G, h = kvh * G + (r0 + r) % G;
      const float f = sum == 0.f ? 0.f : 1.f / sum;
      const int64_t at = query_at(p, p.os, rw, b, h, i) + d;
      const float v[4] = {o.x * f, o.y * f, o.z * f, o.w * f};
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if (p.out_f32) static_cast<float*>(p.out)[at + e] = v[e];
        else if (p.dtype == AIDN_F16) static_cast<__half*>(p.out)[at + e] = __float2half_rn(v[e]);
        else static_cast<__nv_bfloat16*>(p.out)[at + e] = __float2bfloat16_rn(v[e]);
      }
      if (p.lse && d == 0) *lse_at(p, rw, h, i) = sum == 0.f ? -INFINITY : (top + log2f(sum)) * kLn2;
    };
    const int slot_out = 2 * (int)blockIdx.x + (t0 == 0 ? 1 : 0);
    for (int at = tid; at < rows * (DP / 4); at += NW * 32) {
      const int r = at / (DP / 4), d = at % (DP / 4) * 4;
      if (d >= D) continue;
      float top = kUnset;
#pragma unroll
      for (int w = 0; w < NW; ++w) top = fmaxf(top, wstat[w][r].x);
      float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
      float sum = 0.f;
#pragma unroll
      for (int w = 0; w < NW; ++w) {
        const float2 st = wstat[w][r];
        const float f = ex2_approx(st.x - top), fv = f * wref[w];
        const float4 x = *reinterpret_cast<const float4*>(wacc + (w * ROWS + r) * C::kPitch + d);
        sum += f * st.y;
        o.x += fv * x.x; o.y += fv * x.y; o.z += fv * x.z; o.w += fv * x.w;
      }
      if (whole) {
        write(r, d, o, top, sum);
      } else {
        __stcg(reinterpret_cast<float4*>(sp.partial + ((int64_t)slot_out * ROWS + r) * DP + d), o);
        if (d == 0) __stcg(sp.stats + (int64_t)slot_out * ROWS + r, make_float2(top, sum));
      }
    }
    if (!whole) {
      // CTAs first .. first + parts - 1 have a part of the line; where it begins it is the CTA's last, elsewhere its first
      const int first = (int)(line_pos / share), parts = (int)((line_pos + tiles - 1) / share) - first + 1;
      __threadfence();
      __syncthreads();
      if (tid == 0) last_flag = atomicInc(p.counters + first, parts - 1) == (unsigned)(parts - 1);
      __syncthreads();
      if (last_flag) {
        __threadfence();
        for (int at = tid; at < rows * (DP / 4); at += NW * 32) {
          const int r = at / (DP / 4), d = at % (DP / 4) * 4;
          if (d >= D) continue;
          float top = kUnset;
#pragma unroll 8
          for (int q = 0; q < parts; ++q) top = fmaxf(top, __ldcg(sp.stats + (int64_t)(2 * (first + q) + (q == 0)) * ROWS + r).x);
          float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
          float sum = 0.f;
#pragma unroll 8
          for (int q = 0; q < parts; ++q) {
            const int64_t from = (int64_t)(2 * (first + q) + (q == 0)) * ROWS + r;
            const float2 st = __ldcg(sp.stats + from);
            const float4 x = __ldcg(reinterpret_cast<const float4*>(sp.partial + from * DP + d));
            const float f = ex2_approx(st.x - top);
            sum += f * st.y;
            o.x += f * x.x; o.y += f * x.y; o.z += f * x.z; o.w += f * x.w;
          }
          write(r, d, o, top, sum);
        }
      }
    }
    __syncthreads();   // (shared memory is filled again)
  }
  if (bad && p.status) atomicOr(p.status, kStatusBadBlock);
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
  const int id = ((DP == 64 ? 0 : DP == 128 ? 1 : 2) * 3 + (NR == 1 ? 0 : NR == 2 ? 1 : 2)) * 4 + (T - 1) * 2 + (UB ? 1 : 0);
  if (!(*raised >> id & 1)) {   // once a handle: the limit belongs to the context
    const cudaError_t e = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)C::kSmem);
    if (e != cudaSuccess) return e;
    *raised |= 1ull << id;
  }
  Split sp;
  sp.partial = static_cast<float*>(workspace);
  sp.stats = workspace ? reinterpret_cast<float2*>(static_cast<char*>(workspace) + acc) : nullptr;
  sp.least = 2 * C::kWarps;
  return launch_dependent(k, dim3((unsigned)grid), C::kWarps * 32, C::kSmem, stream, *p, sp);
}

template <int DP, int NR, int T>
cudaError_t pick_block(bool ub, const Attend* p, int num_sms, void* workspace, int64_t* bytes, uint64_t* raised, cudaStream_t stream) {
  return ub ? one<DP, NR, T, true>(p, num_sms, workspace, bytes, raised, stream) : one<DP, NR, T, false>(p, num_sms, workspace, bytes, raised, stream);
}
template <int DP, int T>
cudaError_t pick_rows(int64_t rows, bool ub, const Attend* p, int num_sms, void* workspace, int64_t* bytes, uint64_t* raised, cudaStream_t stream) {
  if (rows <= 8) return pick_block<DP, 1, T>(ub, p, num_sms, workspace, bytes, raised, stream);
  if (rows <= 16 || DP == 256) return pick_block<DP, 2, T>(ub, p, num_sms, workspace, bytes, raised, stream);
  if constexpr (DP < 256) return pick_block<DP, 4, T>(ub, p, num_sms, workspace, bytes, raised, stream);
  return cudaErrorInvalidValue;
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
