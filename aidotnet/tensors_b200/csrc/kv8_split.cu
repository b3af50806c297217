// Attention of few queries over a paged pool held in 8 bits (kv8.cuh): decode steps, drafted tokens, short chunks.
//
//   S^T = K Q^T,  x = S c_r k_scale(block)   (base 2; c_r = scale log2(e) / the query's own factor)
//   with running maxima m of x and b of (x - m) + log2(v_scale(block)) - 9 (rounded up):
//   P = 2^(x - m) (v_scale(block) 2^-b),   O^T += V^T P^T,   l += 2^(x - m),   o = O 2^b / l
//
// Bound by the pool's bytes: 2 D bytes a key and KV head, a few operations a byte.  So every key is read once for all the queries of its
// sequence and KV head (a "line": up to 8 NR query rows = query heads of the group x queries).  A warp has a line's next tiles of 16 keys
// in shared memory or on their way to it (asynchronous copies of 16 bytes), and reads them as fragments of mma.sync without transposing: a
// product does not care about the order of its terms, so the head dimension is permuted such that a lane's 16 bytes of a key are its
// own elements of four A fragments, and a lane's 16 bytes of a value row its own rows of eight (queries are laid out in the
// matching order once a line).  A code becomes fp16 exactly (cvt, two at a time), a query is scaled by a power of two into
// fp16 (two terms for fp32 results), the scales of the blocks are applied to the products in fp32 and those of the values to the weights, and
// these rounded to fp16: 11 bits, of up to 2^9 so that they stay normal down to 2^-23 of the row's largest product of weight and scale; for fp32
// results they are two terms too.  What a row does not see has no part in its maxima.
//
// The warps of a "unit" do the same tiles of neighbouring KV heads, whose rows are neighbours in the pool: memory is read in runs
// of up to 512 bytes (64 sequences of 512 to 4096 keys, 32 KV heads of 128: 228 us, and 265 us where each warp goes through lines of its own;
// 197 us, 5.9 TB/s, by now).  The lines' tiles are one row, cut into equal shares for the units that are resident whatever the lengths are.  No
// warp waits for another one: a line that is cut leaves a partial result a unit in the workspace, and a second launch merges them in their
// order, so that the result does not depend on which was first.
//
// Small calls are one latency after the other (16 sequences of up to 2048 keys, 8 KV heads: 19.4 us for 37 MB, of which the loop over
// tiles takes 6), and code that runs once is fetched once: what is not the loop stays small, in loops that are not unrolled.
#include "kv8.cuh"
#include "mma_sync.cuh"

namespace aidn {
namespace kv8 {
namespace {

constexpr int kTile = 16;           // keys
constexpr float kUnset = -3e38f;    // running maximum before any key: below every finite logit but the last few
constexpr float kLift = 9.f;        // the largest weight is 2^9
constexpr float kMost = 32768.f;    // the maxima follow when a weight is above this: all are in fp16's range
constexpr float kMostSum = 0x1p100f;   // or l: logits rise above m where blocks of small values follow large ones
constexpr float kMostFactor = 0x1p126f;
constexpr int kMergeThreads = 256;
constexpr int kMostUnits = 4096;   // (twelve bits in the merging kernel)

// A line that is cut, at the unit in which it begins: parts of it lie there and in the `parts - 1` units behind; 0: no such line.
struct Note {
  int parts, b, off, rows;
};
struct Split {
  float* partial;    // [2 units][heads of a unit][row_most][DP], or null: lines are not cut
  float2* stats;     // [2 units][heads of a unit][row_most]: maximum and sum
  Note* notes;       // [units]
  int units, heads_log2, row_most;
  int least;         // tiles of a unit's share
  bool query_vec, out_vec;   // 16 bytes of the queries, four elements of the results are aligned
};

__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
  return r;
}
__device__ __forceinline__ void copy16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void copy4(uint32_t dst, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ uint4 lds16(uint32_t at) {
  uint4 r;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w) : "r"(at));
  return r;
}
__device__ __forceinline__ uint2 lds8(uint32_t at) {
  uint2 r;
  asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(r.x), "=r"(r.y) : "r"(at));
  return r;
}
__device__ __forceinline__ float lds_f(uint32_t at) {
  float r;
  asm volatile("ld.shared.f32 %0, [%1];" : "=f"(r) : "r"(at));
  return r;
}
__device__ __forceinline__ float lg2_approx(float x) {
  float y;
  asm("lg2.approx.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float pow2(float e) { return __uint_as_float((uint32_t)((int)e + 127) << 23); }   // of a whole number in [-126, 127]
__device__ __forceinline__ float exponent_of(float x) { return (float)((int)(__float_as_uint(x) >> 23) - 127); }
__device__ __forceinline__ void copy8(uint32_t dst, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(dst), "l"(src) : "memory");
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
// Whether any of four codes is a NaN.
__device__ __forceinline__ bool any_nan(uint32_t x) { return (((x & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u) != 0; }
__device__ __forceinline__ uint32_t without_nan(uint32_t x) {
  const uint32_t hit = (((x & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u) >> 7;   // 1 in the bytes that are
  return x & ~(hit * 0xffu);
}

// What the host knows of a call.
struct Sizes {
  int64_t batch, rows, seq_kv;   // rows: of a sequence and KV head, at most
  int kv_count, num_sms;
  int64_t workspace_bytes;
};

template <int DP, int NR, int T, bool UB>
struct Config {
  static constexpr int kWarps = 4;   // (8 and 16: 2 % slower with 64 sequences, 6 to 10 % with one)
  // registers: 16 warps an SM with one fragment of rows (12: 64 tokens 194 -> 211 us; 20: 216), 12 with two (16: drafts 57 -> 77; 8: 66).  Fragments of 32
  // rows leave 8 warps (drafts 77), and passing over those without rows costs more than it saves (60).
  static constexpr int kMinCtas = DP == 256 ? 2 : (NR == 1 ? 4 : 3);
  static constexpr int kSteps = DP / 16;                 // of 16 elements: fragments of a key
  static constexpr int kRows = 8 * NR;
  static constexpr int kQueryBytes = T * NR * kSteps * 32 * 8;   // of a warp
  static constexpr int kScales = UB ? 16 : 128;                  // bytes of a stage: the block's two, or those of 16 keys
  static constexpr int kStage = 2 * kTile * DP + kScales;
  static constexpr int kStages = 2;   // tiles of a warp in shared memory or on their way to it (with three: 228 us, and 208, of the case above)
  static constexpr size_t kSmem = (size_t)kWarps * (kQueryBytes + kStages * kStage);
};

template <int DP, int NR, int T, bool UB>
__global__ void __launch_bounds__(Config<DP, NR, T, UB>::kWarps * 32, Config<DP, NR, T, UB>::kMinCtas)
    kv8_split_kernel(const __grid_constant__ Attend p, const __grid_constant__ Split sp) {
  using C = Config<DP, NR, T, UB>;
  constexpr int NW = C::kWarps, KS = C::kSteps, MT = DP / 16, ROWS = C::kRows, STAGES = C::kStages;
  constexpr int KC = DP / 64;                     // 16-byte pieces of a key a lane multiplies
  constexpr int VB = DP == 64 ? 8 : 16;           // bytes of a value row a lane reads at a time
  constexpr int VC = DP == 256 ? 2 : 1;
  constexpr int CPR = DP / 16, RPI = 32 / CPR, NI = kTile / RPI;   // 16-byte chunks of a row; rows and copies of a warp's instruction
  extern __shared__ __align__(128) uint8_t smem[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const uint32_t ring = (uint32_t)__cvta_generic_to_shared(smem) + warp * STAGES * C::kStage;
  // Fragments of the queries, [NR][SLOTS][32 lanes] of 16 bytes: two steps, or the two terms of one
  constexpr int SLOTS = T == 1 ? KS / 2 : KS, SLOT = T == 1 ? 8 : 4;   // elements
  uint4* const qfrag = reinterpret_cast<uint4*>(smem + NW * STAGES * C::kStage + warp * C::kQueryBytes);
  const int D = p.c.head_dim, G = p.group, groups = p.kv_count >> sp.heads_log2;
  const int unit = ((int)blockIdx.x * NW + warp) >> sp.heads_log2, sub = warp & ((1 << sp.heads_log2) - 1);
  const bool cut = sp.partial != nullptr;
  auto column = [](int j, int t) { return DP == 64 ? 16 * t : 128 * (j >> 1) + 32 * t + 16 * (j & 1); };   // first element of a lane's piece j
  pdl_wait();
  pdl_trigger();

  auto tiles_of = [&](int keys) { return keys > kTile ? (keys + kTile - 1) / kTile : 1; };
  auto lines_of = [&](int n) { return ((n * G + ROWS - 1) / ROWS) * groups; };
  auto weight_of = [&](int b) { return lines_of(rows_of(p, b).count) * (cut ? tiles_of(keys_of(p, b)) : 1); };

  // ---- the share of this unit: the lanes sum up their sequences' tiles (of each warp: there is nothing to wait for.  The host cuts lines
  // only where all tiles together are fewer than 2^31)
  const int per = (p.batch + 31) >> 5;
  const int b_lo = min(lane * per, p.batch), b_hi = min(b_lo + per, p.batch);
  int mine = 0;
#pragma unroll 4
  for (int b = b_lo; b < b_hi; ++b) mine += weight_of(b);
  int upto = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int v = __shfl_up_sync(0xffffffffu, upto, o);
    if (lane >= o) upto += v;
  }
  const int total = __shfl_sync(0xffffffffu, upto, 31);
  int share = (int)(((uint32_t)total + sp.units - 1) / (uint32_t)sp.units);
  if (cut && share < sp.least) share = sp.least;
  int pos = (int)min((int64_t)unit * share, (int64_t)total);
  const int end = min((uint32_t)pos + (uint32_t)share, (uint32_t)total);
  int b = 0, base = 0;
  if (pos < end) {   // the last lane whose sequences begin at or before pos, then the sequence among its own
    const int at = __popc(__ballot_sync(0xffffffffu, upto - mine <= pos)) - 1;
    b = at * per;
    base = __shfl_sync(0xffffffffu, upto - mine, at);
  }
  bool bad = false;
  Note note = {0, 0, 0, 0};

  while (pos < end) {
    const Rows rw = rows_of(p, b);
    const int keys = keys_of(p, b), lines = lines_of(rw.count);
    const int tiles = cut ? tiles_of(keys) : 1;
    const int into = pos - base;
    if (into >= lines * tiles) {   // on to the next sequence
      base += lines * tiles;
      ++b;
      continue;
    }
    const int off = into / tiles, t0 = cut ? into - off * tiles : 0;
    const int chunk = off < groups ? 0 : off / groups, kvh = p.kv_begin + ((off - chunk * groups) << sp.heads_log2) + sub, r0 = chunk * ROWS;
    const int rows = min(ROWS, rw.count * G - r0);
    const int t1 = cut ? min(tiles, t0 + (end - pos)) : tiles_of(keys);
    const bool whole = !cut || (t0 == 0 && t1 == tiles);
    if (!whole && t0 == 0) note = {pos + tiles - 1, b, off, rows};   // (parts: below)
    pos += cut ? t1 - t0 : 1;

    const int lim_least = visible(p, keys, rw.count, rw.count == 1 ? 0 : r0 / G);
    const int lim_most = rw.count == 1 ? lim_least : visible(p, keys, rw.count, (r0 + rows - 1) / G);
    const int t_end = min(t1, (lim_most + kTile - 1) / kTile);
    // ---- tiles t0 .. t_end - 1.  A lane holds the table's entry of one of 32 blocks, and of one of the next 32.
    const int32_t* table = p.c.table + b * p.c.table_stride;
    int window = 0, entry = 0, entry_n = 0, last_block = 0;
    if (t0 < t_end) {
      window = block_of(p.c, t0 * kTile);
      last_block = block_of(p.c, min(t_end * kTile, keys) - 1);
      if (window + lane <= last_block) entry = table[window + lane];
      if (window + 32 + lane <= last_block) entry_n = table[window + 32 + lane];
    }

    // The queries are on their way while the first keys are looked up.  Lane (g, t) copies of row g (of eight) what it will multiply with to where
    // the fragments of it will be.
    __syncwarp();   // (the last line's tiles and queries have been read)
#pragma unroll 1
    for (int n = 0; n < NR; ++n) {
      const int r = 8 * n + g, i = rw.count == 1 ? 0 : (r0 + r) / G, h = kvh * G + (r0 + r) - i * G;
      const int64_t at = r < rows ? query_at(p, p.qs, rw, b, h, i) : 0;
      const bool wide = T == 2 && p.dtype == AIDN_F32;
      const int64_t esz = wide ? 4 : 2;
#pragma unroll 4
      for (int x = 0; x < SLOTS; ++x) {
        const int d = T == 1 ? column(x >> 1, t) + 8 * (x & 1) : column(x >> 2, t) + 4 * (x & 3);
        uint4* const dst = qfrag + (n * SLOTS + x) * 32 + lane;
        const uint8_t* const src = static_cast<const uint8_t*>(p.q) + (at + d) * esz;
        if (r >= rows || d >= D) {
          *dst = make_uint4(0, 0, 0, 0);
        } else if (sp.query_vec) {
          const uint32_t to = (uint32_t)__cvta_generic_to_shared(dst);
          if (T == 1 || wide) copy16(to, src);
          else copy8(to, src);
        } else {
#pragma unroll 1
          for (int e = 0; e < SLOT; ++e) {
            if (wide) reinterpret_cast<uint32_t*>(dst)[e] = reinterpret_cast<const uint32_t*>(src)[e];
            else reinterpret_cast<uint16_t*>(dst)[e] = reinterpret_cast<const uint16_t*>(src)[e];
          }
        }
      }
    }
    cp_async_commit();

    // A tile's keys and values go to shared memory, 16 bytes a lane and copy.  All of them exist: where a row is shorter than DP bytes its
    // first chunk comes again (the queries are zero there, and those values are not written), and keys behind the last one, or of a
    // block outside the pool, are other rows of the pool, masked below.
    const int64_t pitch = p.c.stride[1];
    const int my_row = lane / CPR, my_chunk = lane % CPR;
    const int64_t from = kvh * p.c.stride[2] + (my_chunk * 16 < D ? my_chunk * 16 : 0) + (UB ? my_row * pitch : 0);
    auto key_chunk = [](int row, int chunk) { return row * DP + (DP == 64 ? chunk : chunk ^ (row & 7)) * 16; };
    // (64 bytes a row: rows 0 and 2 share a line of the banks, 1 and 3 the next)
    auto value_chunk = [](int row, int chunk) {
      return DP == 64 ? ((row >> 2) * 2 + (row & 1)) * 128 + (row & 2) * 32 + (chunk ^ (row >> 1 & 2)) * 16 : row * DP + (chunk ^ (row & 7)) * 16;
    };
    auto issue = [&](int tile, int stage) {
      const uint32_t at = ring + stage * C::kStage;
      const int key0 = tile * kTile, first = block_of(p.c, key0);
      if (first - window >= 32) {
        window += 32;
        entry = entry_n;
        if (window + 32 + lane <= last_block) entry_n = table[window + 32 + lane];
      }
      if constexpr (UB) {
        const int ent = checked_block(p.c, __shfl_sync(0xffffffffu, entry, first - window), bad);
        const int64_t row = (int64_t)max(ent, 0) * p.c.stride[0] + (key0 - first * p.c.block_size) * pitch + from;
        const uint8_t* k = p.c.k + row;
        const uint8_t* v = p.c.v + row;
#pragma unroll
        for (int i = 0; i < NI; ++i) {
          copy16(at + key_chunk(my_row + i * RPI, my_chunk), k);
          copy16(at + kTile * DP + value_chunk(my_row + i * RPI, my_chunk), v);
          k += RPI * pitch;
          v += RPI * pitch;
        }
        if (lane < 2) {
          const uint32_t to = at + 2 * kTile * DP + lane * 4;
          if (ent >= 0) copy4(to, (lane ? p.c.v_scale : p.c.k_scale) + (int64_t)ent * p.c.kv_heads + kvh);
          else asm volatile("st.shared.f32 [%0], %1;" ::"r"(to), "f"(-1.f) : "memory");
        }
      } else {
        auto entry_of = [&](int key, int& within) {
          key = min(key, keys - 1);
          const int block = block_of(p.c, key), rel = block - window;
          const int a = __shfl_sync(0xffffffffu, entry, rel & 31), c = __shfl_sync(0xffffffffu, entry_n, rel & 31);
          within = key - block * p.c.block_size;
          return checked_block(p.c, rel < 32 ? a : c, bad);
        };
#pragma unroll
        for (int i = 0; i < NI; ++i) {
          int within;
          const int ent = entry_of(key0 + my_row + i * RPI, within);
          const int64_t row = (int64_t)max(ent, 0) * p.c.stride[0] + within * pitch + from;
          copy16(at + key_chunk(my_row + i * RPI, my_chunk), p.c.k + row);
          copy16(at + kTile * DP + value_chunk(my_row + i * RPI, my_chunk), p.c.v + row);
        }
        int within;
        const int ent = entry_of(key0 + (lane & 15), within);
        const uint32_t to = at + 2 * kTile * DP + lane * 4;
        if (ent >= 0) copy4(to, (lane < 16 ? p.c.k_scale : p.c.v_scale) + (int64_t)ent * p.c.kv_heads + kvh);
        else asm volatile("st.shared.f32 [%0], %1;" ::"r"(to), "f"(-1.f) : "memory");
      }
    };
    int stage = 0;
#pragma unroll 1
    for (int a = 0; a < STAGES - 1; ++a) {
      if (t0 + a < t_end) issue(t0 + a, a);
      cp_async_commit();
    }

    // ---- queries: scaled by a power of two so that the largest element is in [2^12, 2^13), as fragments
    cp_async_wait<STAGES - 1>();   // (the tiles are behind them)
    auto values = [&](uint4 w, float* x) {
      const uint32_t u[4] = {w.x, w.y, w.z, w.w};
      if (T == 2 && p.dtype == AIDN_F32) {
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = __uint_as_float(u[e]);
      } else if (p.dtype == AIDN_F16) {
#pragma unroll
        for (int e = 0; e < SLOT / 2; ++e) {
          const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&u[e]));
          x[2 * e] = f.x;
          x[2 * e + 1] = f.y;
        }
      } else {
#pragma unroll
        for (int e = 0; e < SLOT / 2; ++e) {
          x[2 * e] = __uint_as_float(u[e] << 16);
          x[2 * e + 1] = __uint_as_float(u[e] & 0xffff0000u);
        }
      }
    };
    constexpr int UNROLL = SLOTS <= 4 ? SLOTS : 2;   // (code that runs once a line is fetched once a line)
    float c_row[NR];
    int lim_row[NR];
#pragma unroll
    for (int n = 0; n < NR; ++n) {
      const int r = 8 * n + g;
      uint4* const mine = qfrag + n * SLOTS * 32 + lane;
      uint32_t most = 0;   // the largest magnitudes by their bits (a NaN makes the row's logits NaN whatever the factor)
#pragma unroll UNROLL
      for (int x = 0; x < SLOTS; ++x) {
        const uint4 w = mine[x * 32];
        const uint32_t u[4] = {w.x, w.y, w.z, w.w};
        if (T == 2 && p.dtype == AIDN_F32) {
#pragma unroll
          for (int e = 0; e < 4; ++e) most = max(most, u[e] & 0x7fffffffu);
        } else {
#pragma unroll
          for (int e = 0; e < SLOT / 2; ++e) most = __vmaxu2(most, u[e] & 0x7fff7fffu);
        }
      }
      float largest = __uint_as_float(most);
      if (T == 1 || p.dtype != AIDN_F32) {
        most = max(most >> 16, most & 0xffffu);
        largest = p.dtype == AIDN_F16 ? __half2float(__ushort_as_half((unsigned short)most)) : __uint_as_float(most << 16);
      }
      largest = fmaxf(largest, __shfl_xor_sync(0xffffffffu, largest, 1));
      largest = fmaxf(largest, __shfl_xor_sync(0xffffffffu, largest, 2));
      int up = 12 - ((int)(__float_as_uint(largest) >> 23) - 127);   // (zeros and what is below the normal floats: 2^126)
      up = max(-110, min(up, 126));
      const float f = __uint_as_float((uint32_t)(up + 127) << 23);
#pragma unroll UNROLL
      for (int x = 0; x < SLOTS; ++x) {
        float v[SLOT];
        values(mine[x * 32], v);
        uint32_t w[4];
#pragma unroll
        for (int e = 0; e < SLOT / 2; ++e) {
          const float a = v[2 * e] * f, c = v[2 * e + 1] * f;
          const __half2 hi = __floats2half2_rn(a, c);
          w[e] = *reinterpret_cast<const uint32_t*>(&hi);
          if (T == 2) {
            const __half2 lo = __floats2half2_rn(a - __low2float(hi), c - __high2float(hi));
            w[T == 2 ? 2 + e : e] = *reinterpret_cast<const uint32_t*>(&lo);
          }
        }
        mine[x * 32] = make_uint4(w[0], w[1], w[2], w[3]);
      }
      c_row[n] = p.scale * __uint_as_float((uint32_t)(127 - up) << 23) * (p.softcap > 0.f ? 1.f : kLog2e);
      lim_row[n] = r >= rows ? keys : (rw.count == 1 ? lim_least : visible(p, keys, rw.count, (r0 + r) / G));
    }

    float acc[NR][MT][4];
    float m[NR][2], factor[NR][2], l[NR][2], c[NR][2];   // factor: 2^-b, exactly
    int lim[NR][2];
#pragma unroll
    for (int n = 0; n < NR; ++n) {
#pragma unroll
      for (int j = 0; j < MT; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[n][j][e] = 0.f;
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        m[n][e] = kUnset;
        factor[n][e] = 1.f;
        l[n][e] = 0.f;
        c[n][e] = __shfl_sync(0xffffffffu, c_row[n], 4 * (2 * t + e));
        lim[n][e] = __shfl_sync(0xffffffffu, lim_row[n], 4 * (2 * t + e));
      }
    }
#pragma unroll 1
    for (int tile = t0; tile < t_end; ++tile) {
      cp_async_wait<STAGES - 2>();
      __syncwarp();   // all lanes' copies have landed, and all have read the stage that is filled again now
      const uint32_t at = ring + stage * C::kStage;
      if (tile + STAGES - 1 < t_end) issue(tile + STAGES - 1, stage == 0 ? STAGES - 1 : stage - 1);
      cp_async_commit();
      stage = stage == STAGES - 1 ? 0 : stage + 1;

      const int key0 = tile * kTile;
      float ks[2], vs[2];
      if constexpr (UB) {
        const uint2 x = lds8(at + 2 * kTile * DP);
        ks[0] = ks[1] = __uint_as_float(x.x);
        vs[0] = vs[1] = __uint_as_float(x.y);
      } else {
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          ks[j] = lds_f(at + 2 * kTile * DP + (g + 8 * j) * 4);
          vs[j] = lds_f(at + 2 * kTile * DP + (16 + g + 8 * j) * 4);
        }
      }
      const bool ok[2] = {__float_as_int(ks[0]) >= 0, __float_as_int(ks[1]) >= 0};   // (a block outside the pool: -1)
      // rows of which not all keys of the tile are seen, or keys that are not there
      bool edge = key0 + kTile > lim_least || !ok[0];
      if constexpr (!UB) edge = edge || __any_sync(0xffffffffu, !ok[0] || !ok[1]);
      float s[NR][4];
#pragma unroll
      for (int n = 0; n < NR; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[n][e] = 0.f;
#pragma unroll
      for (int q = 0; q < KC; ++q) {
        const int chunk = DP == 64 ? t : 8 * (q >> 1) + 2 * t + (q & 1);
        const uint4 x0 = lds16(at + key_chunk(g, chunk)), x1 = lds16(at + key_chunk(g, chunk) + 8 * DP);
        const uint32_t w0[4] = {x0.x, x0.y, x0.z, x0.w}, w1[4] = {x1.x, x1.y, x1.z, x1.w};
        uint4 bq[NR];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint32_t a0 = codes_to_f16(w0[i]), a1 = codes_to_f16(w1[i]), a2 = codes_to_f16_hi(w0[i]), a3 = codes_to_f16_hi(w1[i]);
#pragma unroll
          for (int n = 0; n < NR; ++n) {
            if constexpr (T == 1) {
              if (i % 2 == 0) bq[n] = qfrag[(n * SLOTS + 2 * q + i / 2) * 32 + lane];
              if (i % 2 == 0) mma16816<__half>(s[n], a0, a1, a2, a3, bq[n].x, bq[n].y);
              else mma16816<__half>(s[n], a0, a1, a2, a3, bq[n].z, bq[n].w);
            } else {
              bq[n] = qfrag[(n * SLOTS + 4 * q + i) * 32 + lane];
              mma16816<__half>(s[n], a0, a1, a2, a3, bq[n].x, bq[n].y);
              mma16816<__half>(s[n], a0, a1, a2, a3, bq[n].z, bq[n].w);
            }
          }
        }
      }
      uint4 vr[4][VC];   // keys 2t, 2t + 1, 2t + 8, 2t + 9
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int q = 0; q < VC; ++q) {
          const uint32_t from_v = at + kTile * DP + value_chunk(2 * t + (j & 1) + 8 * (j >> 1), VB == 8 ? g >> 1 : g + 8 * q);
          if (VB == 8) {
            const uint2 x = lds8(from_v + (g & 1) * 8);
            vr[j][q].x = x.x; vr[j][q].y = x.y;
          } else {
            vr[j][q] = lds16(from_v);
          }
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
      // (a scale of the values that is no number makes the logits none, of the rows that see them)
#pragma unroll
      for (int j = 0; j < 2; ++j)
        if (!(vs[j] < INFINITY)) {
          ks[j] = NAN;
          vs[j] = 1.f;
        }
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
        }
      // The weights with the maxima so far; again, once, with the tile's own where one does not fit, or the sum may not.
      float a[NR][4], sum[NR][2];
#pragma unroll 1
      for (bool again = false;; again = true) {
        bool grow = false;
#pragma unroll
        for (int n = 0; n < NR; ++n)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const float x = ex2_approx(s[n][e] - m[n][e]), y = ex2_approx(s[n][e + 2] - m[n][e]);
            sum[n][e] = l[n][e] + x + y;
            // (factors that are finite, for keys that a row does not see)
            a[n][e] = x * fminf(vs[0] * factor[n][e], kMostFactor);
            a[n][e + 2] = y * fminf(vs[1] * factor[n][e], kMostFactor);
            grow = grow || fmaxf(a[n][e], a[n][e + 2]) > kMost || sum[n][e] > kMostSum;
          }
        if (again || !__any_sync(0xffffffffu, grow)) break;
        const float lv[2] = {lg2_approx(vs[0]), lg2_approx(vs[1])};
#pragma unroll
        for (int n = 0; n < NR; ++n)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float top = fmaxf(s[n][e], s[n][e + 2]);
#pragma unroll
            for (int o = 4; o < 32; o <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
            top = fmaxf(m[n][e], top);
            float most = fmaxf((s[n][e] - top) + lv[0], (s[n][e + 2] - top) + lv[1]);
#pragma unroll
            for (int o = 4; o < 32; o <<= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
            const float down = m[n][e] - top, before = exponent_of(factor[n][e]);
            const float now = fmaxf(-126.f, fminf(ceilf(fmaxf(down - before, most - kLift)), 126.f));   // b
            const float keep = ex2_approx(down - before - now);
            factor[n][e] = pow2(-now);
            m[n][e] = top;
            l[n][e] *= ex2_approx(down);
#pragma unroll
            for (int j = 0; j < MT; ++j) {
              acc[n][j][e] *= keep;
              acc[n][j][e + 2] *= keep;
            }
          }
      }
      uint32_t ph[NR][2], pl[NR][2];
#pragma unroll
      for (int n = 0; n < NR; ++n)
#pragma unroll
        for (int j = 0; j < 2; ++j) {   // key g + 8 j, rows 2t and 2t + 1
          l[n][j] = sum[n][j];
          const __half2 hi = __floats2half2_rn(a[n][2 * j], a[n][2 * j + 1]);
          ph[n][j] = transpose8x8(*reinterpret_cast<const uint32_t*>(&hi));
          if constexpr (T == 2) {
            const __half2 lo = __floats2half2_rn(a[n][2 * j] - __low2float(hi), a[n][2 * j + 1] - __high2float(hi));
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
    }

    // ---- a whole line is written, a part of one left in the workspace: of the line that began before this unit's share, or of the one that goes on
    float sum[NR][2];
#pragma unroll
    for (int n = 0; n < NR; ++n)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        sum[n][e] = l[n][e];
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) sum[n][e] += __shfl_xor_sync(0xffffffffu, sum[n][e], o);
      }
    // (row r's to lane r; its elements through the tiles' place, in which no copy is under way, groups of four in an order without conflicts)
    float my_top = 0.f, my_sum = 0.f, my_unit = 0.f;
    cp_async_wait<0>();
    __syncwarp();
    float* const rows_at = reinterpret_cast<float*>(smem + warp * STAGES * C::kStage);
#pragma unroll
    for (int n = 0; n < NR; ++n)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const float top_e = __shfl_sync(0xffffffffu, m[n][e], lane >> 1 & 3), sum_e = __shfl_sync(0xffffffffu, sum[n][e], lane >> 1 & 3);
        const float unit_e = __shfl_sync(0xffffffffu, inverse_pow2(factor[n][e]), lane >> 1 & 3);
        if (lane >> 3 == n && (lane & 1) == e) {
          my_top = top_e;
          my_sum = sum_e;
          my_unit = unit_e;
        }
        float* const to = rows_at + (8 * n + 2 * t + e) * DP;
#pragma unroll
        for (int j = 0; j < MT; j += 2) {
          const int d = DP == 256 ? 128 * (j / 8) + 16 * g + 2 * (j % 8) : VB * g + 2 * j;
          *reinterpret_cast<float4*>(to + (d ^ 4 * t)) = make_float4(acc[n][j][e], acc[n][j][e + 2], acc[n][j + 1][e], acc[n][j + 1][e + 2]);
        }
      }
    __syncwarp();
    const int64_t part = ((int64_t)(2 * unit + (t0 == 0 ? 1 : 0)) << sp.heads_log2) + sub;
    const float mine_f = !whole ? my_unit : (my_sum == 0.f ? 0.f : my_unit / my_sum);
    // (lane r knows where row r goes)
    const int my_i = rw.count == 1 ? 0 : (r0 + lane) / G, my_h = kvh * G + (r0 + lane) - my_i * G;
    const int64_t my_to = whole ? query_at(p, p.os, rw, b, my_h, my_i) : (part * sp.row_most + lane) * DP;
#pragma unroll 2
    for (int r = 0; r < rows; ++r) {
      const float f = __shfl_sync(0xffffffffu, mine_f, r);
      const int64_t to = __shfl_sync(0xffffffffu, my_to, r);
#pragma unroll 1
      for (int d = lane * 4; d < D; d += 128) {
        float4 o = *reinterpret_cast<const float4*>(rows_at + r * DP + (d ^ 4 * (r >> 1 & 3)));
        o.x *= f; o.y *= f; o.z *= f; o.w *= f;
        if (whole) store4(p, to + d, sp.out_vec, o);
        else __stcg(reinterpret_cast<float4*>(sp.partial + to + d), o);
      }
    }
    if (lane < rows) {
      if (!whole) __stcg(sp.stats + part * sp.row_most + lane, make_float2(my_top, my_sum));
      else if (p.lse) *lse_at(p, rw, my_h, my_i) = my_sum == 0.f ? -INFINITY : (my_top + log2f(my_sum)) * kLn2;
    }
  }
  if (cut && sub == 0 && lane == 0 && unit < sp.units) *reinterpret_cast<int4*>(sp.notes + unit) = make_int4(note.rows > 0 ? note.parts / share - unit + 1 : 0, note.b, note.off, note.rows);
  if (bad && p.status) atomicOr(p.status, kStatusBadBlock);
}

// The cut lines' parts: warps take rows in turn, or, where a line has many parts (and so there are few lines), CTAs; four elements a lane.
template <int DP>
__global__ void __launch_bounds__(kMergeThreads, 4) kv8_split_merge_kernel(const __grid_constant__ Attend p, const __grid_constant__ Split sp, int line_rows) {
  constexpr int C4 = DP / 4, PL = kMergeThreads / C4, WARPS = kMergeThreads / 32, AHEAD = 4;
  constexpr int SMALL = 16;
  __shared__ int counts[WARPS];
  __shared__ uint32_t list[kMostUnits];   // units, their lines' parts and rows
  __shared__ float4 held[PL][C4];
  __shared__ float2 held_stats[PL];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  pdl_wait();
  pdl_trigger();
  // the units that began a line which is cut
  const int per = (sp.units + kMergeThreads - 1) / kMergeThreads, u_lo = min(tid * per, sp.units), u_hi = min(u_lo + per, sp.units);
  int mine = 0;
  bool many = false;
  for (int u = u_lo; u < u_hi; ++u) {
    const int parts = sp.notes[u].parts;
    mine += parts > 0;
    many = many || parts > SMALL;
  }
  int upto = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int v = __shfl_up_sync(0xffffffffu, upto, o);
    if (lane >= o) upto += v;
  }
  if (lane == 31) counts[warp] = upto;
  many = __syncthreads_or(many);
  int total = 0, to = upto - mine;
#pragma unroll
  for (int w = 0; w < WARPS; ++w) {
    if (w < warp) to += counts[w];
    total += counts[w];
  }
  if (mine > 0)
    for (int u = u_lo; u < u_hi; ++u)
      if (sp.notes[u].parts > 0) list[to++] = (uint32_t)u | (uint32_t)sp.notes[u].parts << 12 | (uint32_t)sp.notes[u].rows << 25;
  __syncthreads();

  const int D = p.c.head_dim, G = p.group, H = 1 << sp.heads_log2, groups = p.kv_count >> sp.heads_log2;
  const int items = total * sp.row_most << sp.heads_log2;
  float top, sum;
  float4 o;
  // parts first, first + step, ... of row r: four elements from the 4 x-th on
  auto join = [&](int parts, int unit, int sub, int r, int x, int first, int step) {
    top = kUnset;
    sum = 0.f;
    o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 1
    for (int q = first; q < parts; q += AHEAD * step) {
      float2 st[AHEAD];
      float4 v[AHEAD];
#pragma unroll
      for (int u = 0; u < AHEAD; ++u) {
        const int part = min(q + u * step, parts - 1);
        const int64_t from = (((int64_t)(2 * (unit + part) + (part == 0)) << sp.heads_log2) + sub) * sp.row_most + r;
        st[u] = __ldcg(sp.stats + from);
        v[u] = __ldcg(reinterpret_cast<const float4*>(sp.partial + from * DP) + x);
      }
      float now = top;
#pragma unroll
      for (int u = 0; u < AHEAD; ++u) now = fmaxf(now, st[u].x);
      const float keep = ex2_approx(top - now);
      top = now;
      sum *= keep;
      o.x *= keep; o.y *= keep; o.z *= keep; o.w *= keep;
#pragma unroll
      for (int u = 0; u < AHEAD; ++u) {
        if (q + u * step >= parts) continue;
        const float f = ex2_approx(st[u].x - top);
        sum += f * st[u].y;
        o.x += f * v[u].x; o.y += f * v[u].y; o.z += f * v[u].z; o.w += f * v[u].w;
      }
    }
  };
  const int each = sp.row_most << sp.heads_log2, step = many ? gridDim.x : gridDim.x * WARPS;
#pragma unroll 1
  for (int item = many ? blockIdx.x : blockIdx.x * WARPS + warp; item < items; item += step) {
    const int line = item / each, rest = item - line * each, sub = rest & (H - 1), r = rest >> sp.heads_log2;
    const int unit = list[line] & 4095, parts = list[line] >> 12 & 8191;
    if (r >= list[line] >> 25) continue;
    const int b = sp.notes[unit].b, off = sp.notes[unit].off;
#pragma unroll 1
    for (int x = many ? tid % C4 : lane; x < C4; x += many ? C4 : 32) {
      join(parts, unit, sub, r, x, many ? tid / C4 : 0, many ? PL : 1);
      if (many) {
        const int pl = tid / C4;
        held[pl][x] = o;
        if (x == 0) held_stats[pl] = make_float2(top, sum);
        __syncthreads();
        if (pl == 0) {
#pragma unroll
          for (int u = 1; u < PL; ++u) top = fmaxf(top, held_stats[u].x);
          sum = 0.f;
          o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
          for (int u = 0; u < PL; ++u) {
            const float2 st = held_stats[u];
            const float4 v = held[u][x];
            const float f = ex2_approx(st.x - top);
            sum += f * st.y;
            o.x += f * v.x; o.y += f * v.y; o.z += f * v.z; o.w += f * v.w;
          }
        }
        __syncthreads();
        if (pl != 0) continue;
      }
      const int d = 4 * x;
      if (d >= D) continue;
      const Rows rw = rows_of(p, b);
      const int chunk = off / groups, kvh = p.kv_begin + ((off - chunk * groups) << sp.heads_log2) + sub, at = chunk * line_rows + r;
      const int i = at / G, h = kvh * G + at - i * G;
      const float f = sum == 0.f ? 0.f : 1.f / sum;
      store4(p, query_at(p, p.os, rw, b, h, i) + d, sp.out_vec, make_float4(o.x * f, o.y * f, o.z * f, o.w * f));
      if (p.lse && x == 0) *lse_at(p, rw, h, i) = sum == 0.f ? -INFINITY : (top + log2f(sum)) * kLn2;
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
  const int n = ctas * num_sms, most = kMostUnits / Config<DP, NR, T, UB>::kWarps;
  return n < 1 ? 1 : (n < most ? n : most);
}

// One instantiation: its workspace, or its launches (workspace null: the lines are not cut).
template <int DP, int NR, int T, bool UB>
cudaError_t one(const Attend* p, const Sizes& z, void* workspace, int64_t* bytes, uint64_t* raised, int* launches, cudaStream_t stream) {
  using C = Config<DP, NR, T, UB>;
  const int most = resident<DP, NR, T, UB>(z.num_sms);
  Split sp;
  sp.row_most = (int)(z.rows < C::kRows ? z.rows : C::kRows);
  sp.least = NR * T > 1 ? 1 : 2;   // (one query row of 16 bits, 1237 keys: 10.3 us, and 11.0 with one; nine rows of 32 bits: 24.1, and 19.1 with one)
  sp.heads_log2 = 0;
  while ((2 << sp.heads_log2) <= C::kWarps && z.kv_count % (2 << sp.heads_log2) == 0) ++sp.heads_log2;
  const int units_cta = C::kWarps >> sp.heads_log2;
  // no more units than there can be shares (or, uncut, lines)
  const int64_t lines = z.batch * ((z.rows + C::kRows - 1) / C::kRows) * (z.kv_count >> sp.heads_log2);
  const int64_t shares = (lines * (z.seq_kv > 0 ? (z.seq_kv + kTile - 1) / kTile : 1) + sp.least - 1) / sp.least;
  auto grid_for = [&](int64_t n) { return (int)((n + units_cta - 1) / units_cta < most ? (n + units_cta - 1) / units_cta : most); };
  int grid = grid_for(shares);   // (at least one: a call has sequences, queries and room for keys)
  sp.units = grid * units_cta;
  const int64_t rows = (int64_t)2 * grid * C::kWarps * sp.row_most, acc = rows * DP * 4;
  const int64_t need = acc + (rows * 8 + 15) / 16 * 16 + sp.units * (int64_t)sizeof(Note);
  if (bytes) {
    if (*bytes < need) *bytes = need;
    return cudaSuccess;
  }
  auto k = kv8_split_kernel<DP, NR, T, UB>;
  const int id = ((DP == 64 ? 0 : DP == 128 ? 1 : 2) * 2 + NR - 1) * 4 + (T - 1) * 2 + (UB ? 1 : 0);
  if (!(*raised >> id & 1)) {   // once a handle: the limit belongs to the context
    const cudaError_t e = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)C::kSmem);
    if (e != cudaSuccess) return e;
    *raised |= 1ull << id;
  }
  if (z.workspace_bytes < need || (uintptr_t)workspace % 16 != 0 || shares * sp.least >= 0x7fffffff - C::kWarps * most) workspace = nullptr;
  sp.partial = static_cast<float*>(workspace);
  sp.stats = workspace ? reinterpret_cast<float2*>(static_cast<char*>(workspace) + acc) : nullptr;
  sp.notes = workspace ? reinterpret_cast<Note*>(static_cast<char*>(workspace) + need) - sp.units : nullptr;
  if (!workspace) {
    grid = grid_for(lines);
    sp.units = grid * units_cta;
  }
  auto vec = [](const void* ptr, const int64_t* st, int esz, int bytes) {
    return ((uintptr_t)ptr | (uint64_t)(st[0] * esz) | (uint64_t)(st[1] * esz) | (uint64_t)(st[2] * esz)) % bytes == 0;
  };
  sp.query_vec = vec(p->q, p->qs, p->dtype == AIDN_F32 ? 4 : 2, 16);
  sp.out_vec = vec(p->out, p->os, p->out_f32 ? 4 : 2, p->out_f32 ? 16 : 8);
  const cudaError_t e = launch_dependent(k, dim3((unsigned)grid), C::kWarps * 32, C::kSmem, stream, *p, sp);
  *launches = 1;
  if (e != cudaSuccess || !workspace) return e;
  *launches = 2;
  const int64_t items = (lines < sp.units ? lines : sp.units) * ((int64_t)sp.row_most << sp.heads_log2);
  const int64_t merge = items < 8 * z.num_sms ? items : 8 * z.num_sms;
  return launch_dependent(kv8_split_merge_kernel<DP>, dim3((unsigned)merge), kMergeThreads, 0, stream, *p, sp, C::kRows);
}

template <int DP, int NR, int T>
cudaError_t pick_block(bool ub, const Attend* p, const Sizes& z, void* workspace, int64_t* bytes, uint64_t* raised, int* launches, cudaStream_t stream) {
  return ub ? one<DP, NR, T, true>(p, z, workspace, bytes, raised, launches, stream) : one<DP, NR, T, false>(p, z, workspace, bytes, raised, launches, stream);
}
template <int DP, int T>
cudaError_t pick_rows(bool ub, const Attend* p, const Sizes& z, void* workspace, int64_t* bytes, uint64_t* raised, int* launches, cudaStream_t stream) {
  if (z.rows <= 8) return pick_block<DP, 1, T>(ub, p, z, workspace, bytes, raised, launches, stream);
  return pick_block<DP, 2, T>(ub, p, z, workspace, bytes, raised, launches, stream);
}
template <int DP>
cudaError_t pick(bool exact, bool ub, const Attend* p, const Sizes& z, void* workspace, int64_t* bytes, uint64_t* raised, int* launches, cudaStream_t stream) {
  return exact ? pick_rows<DP, 2>(ub, p, z, workspace, bytes, raised, launches, stream) : pick_rows<DP, 1>(ub, p, z, workspace, bytes, raised, launches, stream);
}
cudaError_t pick_dim(int dim, bool exact, bool ub, const Attend* p, const Sizes& z, void* workspace, int64_t* bytes, uint64_t* raised, int* launches, cudaStream_t stream) {
  if (dim <= 64) return pick<64>(exact, ub, p, z, workspace, bytes, raised, launches, stream);
  if (dim <= 128) return pick<128>(exact, ub, p, z, workspace, bytes, raised, launches, stream);
  return pick<256>(exact, ub, p, z, workspace, bytes, raised, launches, stream);
}

}  // namespace

bool split_supported(const Attend& p) {
  if (p.c.head_dim % 16 != 0 || p.mask_kind != AIDN_MASK_NONE) return false;
  if ((uintptr_t)p.c.k % 16 != 0 || (uintptr_t)p.c.v % 16 != 0) return false;
  for (int i = 0; i < 3; ++i)
    if (p.c.stride[i] % 16 != 0) return false;
  return p.batch * ((p.seq_q * p.group + 7) / 8) * p.kv_count < 0x7ff00000;   // lines are counted in 32 bits
}
// (whatever the block size: the larger of the two kernels' needs)
int64_t split_workspace_bytes(int head_dim, bool exact, int64_t batch, int64_t rows, int64_t seq_kv, int kv_count, int num_sms) {
  int64_t most = 0;
  const Sizes z = {batch, rows, seq_kv, kv_count, num_sms, 0};
  for (int ub = 0; ub < 2; ++ub) pick_dim(head_dim, exact, ub, nullptr, z, nullptr, &most, nullptr, nullptr, nullptr);
  return most;
}
cudaError_t launch_attend_split(const Attend& p, int num_sms, void* workspace, int64_t workspace_bytes, uint64_t* raised, int* launches, cudaStream_t stream) {
  const Sizes z = {p.batch, p.seq_q * p.group, p.seq_kv, p.kv_count, num_sms, workspace_bytes};
  return pick_dim(p.c.head_dim, p.out_f32 != 0, p.c.block_size % kTile == 0, &p, z, workspace, nullptr, raised, launches, stream);
}

}  // namespace kv8
}  // namespace aidn
