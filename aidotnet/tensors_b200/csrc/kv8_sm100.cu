// Attention of many queries over a paged pool held in 8 bits (kv8.cuh) on tcgen05: prompt chunks, ragged batches, drafted tokens.
//
//   x = (Q K^T) c_r k_scale(block)      (base 2; c_r = scale log2(e) / the query's own factor)
//   P = 2^((x - m) + e - e_ref + lift),   e = log2(v_scale(block)),   O += P V,   l += 2^(x - m)
//   o = O 2^(e_ref - lift) / l,           m, e_ref: the largest x and (x - m) + e that the row has seen, when they were last taken
//
// A line is (sequence, KV head, pair of 128-row tiles); a row is a (query, query head of the group), so that a few queries of a
// group fill a tile as well as many of one head.  4 D operations a (row, key): bound by the tensor cores for two full tiles, and by the
// pool's bytes where a line has few rows.  Codes become fp16 on the way into shared memory, exactly; the scales of the blocks touch
// sixteen scores at a time, as a factor of the logits and an offset of the exponents, so that they cost nothing per score, and
// queries are scaled by a power of two into fp16 (bf16 and fp16 queries lose nothing that their largest element leaves visible).
// Weights are fp16, 11 bits, lifted so that they stay normal down to 2^-18 of the row's largest product of weight and scale.
//
//   warps 0-3, 4-7    softmax of tile 0 and 1, a row a thread: queries into shared memory, S from tensor memory, P back over it
//                     (16 bits), results.  A row keeps the maxima that it has until sixteen weights sum up to 2^15 (a product of weight
//                     and scale about 2^8 above them): then it takes the step's, scales its accumulator, and forms the weights again
//   warps 8-11        keys and values: 16-byte loads through the block table, codes to fp16, into rings of two 128-key tiles
//   warp 12           tcgen05.mma: S_a = Q_a K^T, O_a += P_a V, for 64 keys at a time
//
// Tensor memory: two score buffers of 64 columns for each row tile (P in the first half of each), O_0 | O_1.  The scores of 64 keys
// are formed while the softmax works on the 64 before: with one buffer of 128 keys a tile the chain softmax -> P V -> next scores
// was the period, 4500 to 5300 cycles for 128 keys where the products take 2050 and the softmax 2900.  The tiles of all lines are one row that is cut into
// equal shares for the CTAs, one an SM (a 128-key tile of a line with two row tiles weighs 4, of one 3).  A line that is cut leaves one
// partial result a CTA in the workspace, and the CTA in which it begins a note about it, from which a second launch merges them:
// 256 rows of up to 148 parts take one CTA 25 to 80 us (measured, merged by the last CTA to arrive), spread over all SMs 4 to 8.
//
// 2048 queries at 14336, 32 heads of 128 on 8: 510 us, 1010 TFLOP/s (bound by the softmax warps, 2300 cycles for 64 keys of two tiles, 46 bytes of
// spill stores and 288 of loads a thread among them; the products take 620); 12 sequences of up to 509 queries, 16 heads of 64 on 4, capped logits: 255 us (4 multiply-adds more a score and a look at its size).
#include <cstddef>
#include <type_traits>

#include "ffma2.cuh"
#include "kv8.cuh"
#include "sm100_ptx.cuh"

namespace aidn {
namespace kv8 {
namespace {

using namespace ptx;

constexpr int kKeys = 128;            // keys of a tile
constexpr int kTileRows = 128;
constexpr int kPairRows = 2 * kTileRows;
constexpr int kThreads = 512;
constexpr int kConvertWarp = 8, kMmaWarp = 12;
constexpr int kSoftmaxRegs = 176, kConvertRegs = 112, kMmaRegs = 48;
// setmaxnreg.inc waits without a bound for registers that are not there: the shares must not exceed what the CTA is launched with
static_assert(256 * kSoftmaxRegs + 128 * kConvertRegs + 128 * kMmaRegs <= kThreads * 128, "registers of the launch");
constexpr int kRing = 4;              // tiles whose scales are kept
constexpr float kUnset = -3e38f;      // maximum before any key: below every finite logit but the last few
constexpr float kLift = 4.f;
constexpr float kLeastScale = -110.f;     // log2 of a scale at least: below that of any block that an append wrote (2^-100); sixteen weights over it are in fp32's range
constexpr int kTileCost = 3, kPairCost = 4;   // of 128 keys with one row tile, and with two, which overlap (64 keys: 1700 cycles, and 2300)
constexpr float kMostWeights = 32768.f;   // of sixteen weights together: each is then in fp16's range
constexpr float kMostSum = 0x1p100f;      // of sixty-four weights without their scales: logits rise above m where blocks of small values follow large ones
constexpr float kLargeLogit = 1048576.f;  // (to base 2) a rounding of half a unit of its last place is 2^-4 here

template <int HD>
struct Cfg {
  static constexpr int kSlab = kKeys * 128;              // 64 elements of 128 rows, 128-byte swizzle
  static constexpr int kTile = kSlab * (HD / 64);        // a query, key or value tile in fp16
  static constexpr int kQ = 0, kK = 2 * kTile, kV = 4 * kTile;
  static constexpr int kMisc = 6 * kTile;
  static constexpr int kSmem = kMisc + 2048 + 1024 /* alignment */;
  static constexpr uint32_t kO = 256;                    // accumulators' first column
};
// barriers: q_full[2] k_full[2] k_empty[2] v_full[2] v_empty[2] s_full[2][2] p_full[2][2] o_done[2][2] scales[kRing]
enum { kQFull = 0, kKFull = 2, kKEmpty = 4, kVFull = 6, kVEmpty = 8, kSFull = 10, kPFull = 14, kODone = 18, kScales = 22, kBars = 22 + kRing };

struct Misc {
  uint64_t bars[kBars];
  uint32_t tmem;
  int abort;
  // of a tile's groups of sixteen keys: scale of the keys, log2 of the values' (-inf: no such keys) and its inverse (then 0)
  struct Scales {
    alignas(16) float k[8];
    float v_exp[8], v_inverse[8];
    uint32_t nan[4];   // keys with a NaN among their values, in tiles of which rows of the pair do not see all: their codes are zeros there
  } scales[kRing];
  int64_t scan[kThreads / 32];
  int64_t start_base;
  int start_b, start_u;
};
static_assert(sizeof(Misc) <= 2048, "");

// (a division of 64 bits takes over a hundred instructions)
__device__ __forceinline__ int64_t quotient(int64_t a, int64_t b) {
  return (uint64_t)(a | b) >> 32 ? a / b : (int64_t)((uint32_t)a / (uint32_t)b);
}

// A line that begins in a CTA's share and goes on behind it: in how many CTAs it has parts (0: there is none).
struct Note {
  int64_t first_row;
  int b, kvh, row, rows, parts;
};
struct Cut {
  float* partial;   // [2 grid][256][HD], or null: lines are not cut
  float2* stats;    // [2 grid][256]: maximum and sum
  Note* notes;      // [grid]
  bool query_vec, out_vec;
};

// The lines of this CTA's share, in order; every role walks them by itself.
struct Walk {
  const Attend* p;
  int64_t pos, end, share, base;   // base: position of the line's first tile
  bool cut;
  int b, u, kvh;
  Rows rw;
  int keys, pairs;
  // the line
  int rows, cost, tiles, t0, t1;
  bool whole;

  __device__ __forceinline__ void sequence() {
    rw = rows_of(*p, b);
    keys = keys_of(*p, b);
    pairs = (rw.count * p->group + kPairRows - 1) / kPairRows;
  }
  __device__ __forceinline__ void line() {
    const int left = rw.count * p->group - u * kPairRows;
    rows = left < kPairRows ? left : kPairRows;
    cost = rows > kTileRows ? kPairCost : kTileCost;
    tiles = tiles_of(*p, rw.count, keys, u);
  }
  __device__ __forceinline__ int tiles_before(int64_t cost_of_them) const {   // rounded up, all of the line's at most
    return cost_of_them >= (int64_t)tiles * cost ? tiles : ((int)cost_of_them + cost - 1) / cost;
  }
  static __device__ __forceinline__ int tiles_of(const Attend& p, int n, int keys, int u) {
    const int last = min(n * p.group, (u + 1) * kPairRows) - 1;
    const int end = visible(p, keys, n, last / p.group);
    return end > kKeys ? (end + kKeys - 1) / kKeys : 1;
  }
  // On to the next line that this CTA has tiles of; false at the end.
  __device__ __forceinline__ bool next(bool first) {
    for (;;) {
      if (!first) {
        base += (int64_t)tiles * cost;
        if (++kvh == p->kv_count) {
          kvh = 0;
          if (++u == pairs) {
            u = 0;
            do {
              if (++b >= p->batch || base >= end) return false;
              sequence();
            } while (pairs == 0);
          }
          line();
        }
      }
      first = false;
      if (base >= end) return false;
      if (cut) {
        t0 = pos > base ? tiles_before(pos - base) : 0;
        t1 = tiles_before(end - base);
        if (t0 >= t1) continue;
        whole = t0 == 0 && t1 == tiles;
      } else {
        if (base < pos) continue;   // a line belongs to the share that it begins in
        t0 = 0;
        t1 = tiles;
        whole = true;
      }
      return true;
    }
  }
};

__device__ __forceinline__ float4 ld_shared_f4(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ uint4 ld_shared_v4(uint32_t addr) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ uint32_t ld_shared_u32(uint32_t addr) {
  uint32_t v;
  asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ float log2_approx(float x) {
  float y;
  asm("lg2.approx.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// tanh of two numbers up to 1, to 7e-7 of itself: x q(x^2), q the polynomial of degree 5 with the least relative error (a weighted least-squares
// fit whose weights were adapted until the error was even).  Four multiply-adds an element in place of two of the special functions, of which a
// multiprocessor does 16 a cycle: with those, logits that are capped took three a score where others take one.
__device__ __forceinline__ uint64_t tanh_small(uint64_t x) {
  constexpr float q[6] = {0.999999404f, -0.333290428f, 0.132814333f, -0.0516056716f, 0.0167431142f, -0.00306705991f};
  const uint64_t w = mul2(x, x);
  uint64_t y = aidn::pack2(q[5], q[5]);
#pragma unroll
  for (int i = 4; i >= 0; --i) y = fma2(y, w, aidn::pack2(q[i], q[i]));
  return mul2(x, y);
}
__device__ __forceinline__ bool any_nan(uint32_t x) { return (((x & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u) != 0; }
__device__ __forceinline__ uint32_t without_nan(uint32_t x) {
  const uint32_t hit = (((x & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u) >> 7;
  return x & ~(hit * 0xffu);
}
// Two 16-bit elements of the queries as floats.
__device__ __forceinline__ float2 widen2(const Attend& p, uint32_t w) {
  if (p.dtype == AIDN_F16) return __half22float2(*reinterpret_cast<const __half2*>(&w));
  return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}
template <int HD, bool CAP>
__global__ void __launch_bounds__(kThreads, 1) kv8_sm100_kernel(const __grid_constant__ Attend p, const Cut cut) {
  using C = Cfg<HD>;
  extern __shared__ uint8_t raw[];
  uint8_t* const smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~(uintptr_t)1023);
  Misc& ms = *reinterpret_cast<Misc*>(smem + C::kMisc);
  volatile int* const abort_flag = &ms.abort;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, G = p.group;
  const uint32_t base = smem_u32(smem);
  const uint32_t bars = base + C::kMisc + (uint32_t)offsetof(Misc, bars), scales_at = base + C::kMisc + (uint32_t)offsetof(Misc, scales);
  auto bar = [&](uint32_t i) { return bars + 8 * i; };
  if (tid == 0) {
    ms.abort = 0;
    for (int i = 0; i < 2; ++i) {
      mbar_init(bar(kQFull + i), 4);
      mbar_init(bar(kKFull + i), 4);
      mbar_init(bar(kKEmpty + i), 1);
      mbar_init(bar(kVFull + i), 4);
      mbar_init(bar(kVEmpty + i), 1);
    }
    for (int i = 0; i < 4; ++i) {
      mbar_init(bar(kSFull + i), 1);
      mbar_init(bar(kODone + i), 1);
      mbar_init(bar(kPFull + i), 4);
    }
    for (int i = 0; i < kRing; ++i) mbar_init(bar(kScales + i), 4);
    fence_mbar_init();
  }
  if (warp == kMmaWarp) {
    tmem_alloc(smem_u32(&ms.tmem), 512);
    tmem_relinquish();
  }
  pdl_wait();
  pdl_trigger();

  // ---- shares: a thread sums up the lines of some sequences, or of some row pairs of one; their prefix gives where a share begins
  const bool is_cut = cut.partial != nullptr;
  const int spread = p.batch < kThreads ? kThreads / p.batch : 1, per = (p.batch + kThreads - 1) / kThreads;   // threads a sequence, sequences a thread
  const int b_lo = spread > 1 ? min(tid / spread, p.batch) : min(tid * per, p.batch);
  const int b_hi = spread > 1 ? min(b_lo + 1, p.batch) : min(b_lo + per, p.batch);
  auto pairs_of = [&](int n, int* lo, int* hi) {   // this thread's row pairs of a sequence of n queries
    const int pairs = (n * G + kPairRows - 1) / kPairRows, each = (pairs + spread - 1) / spread;
    *lo = spread > 1 ? min((tid % spread) * each, pairs) : 0;
    *hi = spread > 1 ? min(*lo + each, pairs) : pairs;
  };
  auto weight = [&](int n, int keys, int u) {
    return (int64_t)Walk::tiles_of(p, n, keys, u) * p.kv_count * (n * G - u * kPairRows > kTileRows ? kPairCost : kTileCost);
  };
  int64_t mine = 0;
  for (int b = b_lo; b < b_hi; ++b) {
    const int n = rows_of(p, b).count, keys = keys_of(p, b);
    int lo, hi;
    pairs_of(n, &lo, &hi);
    for (int u = lo; u < hi; ++u) mine += weight(n, keys, u);
  }
  int64_t upto = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t v = __shfl_up_sync(0xffffffffu, upto, o);
    if (lane >= o) upto += v;
  }
  if (lane == 31) ms.scan[warp] = upto;
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  int64_t total = 0, before = 0;
#pragma unroll
  for (int w = 0; w < kThreads / 32; ++w) {
    if (w == warp) before = total;
    total += ms.scan[w];
  }
  before += upto - mine;
  int64_t share = quotient(total + gridDim.x - 1, gridDim.x);
  if (share < 2 * kPairCost) share = 2 * kPairCost;   // (no line passes over a share)
  const int64_t pos = blockIdx.x * share, end = min(pos + share, total);
  const uint32_t tmem = ms.tmem;
  if (pos < end && pos >= before && pos < before + mine) {
    int64_t at = before;
    bool found = false;
    for (int b = b_lo; b < b_hi && !found; ++b) {
      const int n = rows_of(p, b).count, keys = keys_of(p, b);
      int lo, hi;
      pairs_of(n, &lo, &hi);
      for (int u = lo; u < hi; ++u) {
        const int64_t w = weight(n, keys, u);
        if (pos < at + w) {
          ms.start_b = b;
          ms.start_u = u;
          ms.start_base = at;
          found = true;
          break;
        }
        at += w;
      }
    }
  }
  __syncthreads();

  auto walk = [&]() {   // at the first line; the head within the pair is the quotient
    Walk w;
    w.p = &p;
    w.pos = pos;
    w.end = end;
    w.share = share;
    w.cut = is_cut;
    w.b = ms.start_b;
    w.u = ms.start_u;
    w.sequence();
    w.line();
    const int64_t a_line = (int64_t)w.tiles * w.cost;
    w.kvh = (int)quotient(pos - ms.start_base, a_line);
    w.base = ms.start_base + w.kvh * a_line;
    return w;
  };
  bool alive = pos < end;
  bool bad = false;
  if (is_cut && tid == 0) cut.notes[blockIdx.x].parts = 0;

  if (warp < kConvertWarp) {
    // ================================================= softmax =================================================
    setmaxnreg_inc<kSoftmaxRegs>();
    const int a = warp >> 2, row_in = tid & 127;
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t ts0 = tmem + lanes + (uint32_t)(a * 128), to = tmem + lanes + C::kO + (uint32_t)(a * HD);
    uint32_t steps = 0;        // of 64 keys, that this row tile took part in
    uint32_t tile_count = 0;   // of this CTA, for the scales' ring
    if (alive) {
      Walk w = walk();
      for (bool first = true; alive && w.next(first); first = false) {
        const int n_tiles = w.t1 - w.t0;
        if (a == 1 && w.rows <= kTileRows) {   // (tile 1 has no rows: not taken part in)
          tile_count += n_tiles;
          continue;
        }
        const int r = w.u * kPairRows + a * kTileRows + row_in;
        const bool valid = a * kTileRows + row_in < w.rows;
        const int i = valid ? r / G : 0, h = (p.kv_begin + w.kvh) * G + (valid ? r - i * G : 0);
        // ---- this warp's 32 queries: HD / 8 lanes a row, scaled by a power of two so that the largest element is in [2^8, 2^9)
        constexpr int kLanes = HD / 8, kAtOnce = 32 / kLanes;   // lanes of a row, rows of a load
        const int sub = lane / kLanes, chunk = lane % kLanes;
        const int warp_row = (warp & 3) * 32, warp_rows = min(32, w.rows - a * kTileRows - warp_row);   // (may be negative)
        float c;
        {
          // (loops, not unrolled: code that runs once a line costs its fetch from memory, 40 us over a step of 24 sequences)
          const uint32_t tile = base + C::kQ + a * C::kTile + warp_row * 128;
          const int first = w.u * kPairRows + a * kTileRows + warp_row;
#pragma unroll 2
          for (int j = 0; j < HD / 8; ++j) {
            const int row = j * kAtOnce + sub, qi = (first + row) / G, gh = (first + row) - qi * G;
            const uint32_t dst = tile + (chunk >> 3) * C::kSlab + row * 128 + (((chunk & 7) ^ (row & 7)) << 4);
            uint32_t x[4] = {0, 0, 0, 0};
            if (row < warp_rows) {
              const uint16_t* q = static_cast<const uint16_t*>(p.q) + query_at(p, p.qs, w.rw, w.b, (p.kv_begin + w.kvh) * G + gh, qi) + 8 * chunk;
              if (cut.query_vec) {
                asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(q) : "memory");
                continue;
              }
              for (int e = 0; e < 4; ++e) x[e] = q[2 * e] | (uint32_t)q[2 * e + 1] << 16;
            }
            st_shared_v4(dst, x[0], x[1], x[2], x[3]);
          }
          asm volatile("cp.async.wait_all;" ::: "memory");
          __syncwarp();
          // a thread its own row
          auto piece = [&](int j) { return tile + (j >> 3) * C::kSlab + lane * 128 + (((j & 7) ^ (lane & 7)) << 4); };
          float largest = 0.f;
#pragma unroll 2
          for (int j = 0; j < HD / 8; ++j) {
            const uint4 x = ld_shared_v4(piece(j));
            const float2 y0 = widen2(p, x.x), y1 = widen2(p, x.y), y2 = widen2(p, x.z), y3 = widen2(p, x.w);
            largest = fmaxf(largest, fmaxf(fmaxf(fmaxf(fabsf(y0.x), fabsf(y0.y)), fmaxf(fabsf(y1.x), fabsf(y1.y))),
                                           fmaxf(fmaxf(fabsf(y2.x), fabsf(y2.y)), fmaxf(fabsf(y3.x), fabsf(y3.y)))));
          }
          int up = 8 - ((int)(__float_as_uint(largest) >> 23) - 127);
          up = max(-110, min(up, 126));
          const float f = __uint_as_float((uint32_t)(up + 127) << 23);
          c = p.scale * __uint_as_float((uint32_t)(127 - up) << 23) * (CAP ? 1.f : kLog2e);
#pragma unroll 2
          for (int j = 0; j < HD / 8; ++j) {
            const uint4 x = ld_shared_v4(piece(j));
            const float2 y0 = widen2(p, x.x), y1 = widen2(p, x.y), y2 = widen2(p, x.z), y3 = widen2(p, x.w);
            st_shared_v4(piece(j), ptx::pack2<false>(y0.x * f, y0.y * f), ptx::pack2<false>(y1.x * f, y1.y * f), ptx::pack2<false>(y2.x * f, y2.y * f),
                         ptx::pack2<false>(y3.x * f, y3.y * f));
          }
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(bar(kQFull + a));
        const int lim = valid ? visible(p, w.keys, w.rw.count, i) : 0x7fffffff;
        const int lim_least = visible(p, w.keys, w.rw.count, (w.u * kPairRows + a * kTileRows) / G);
        const int lim_pair = visible(p, w.keys, w.rw.count, w.u * kPairRows / G);   // what the converters clean a tile by
        const float cap_inverse = CAP ? 1.f / p.softcap : 0.f;
        float m = kUnset, l = 0.f, eref = 0.f, l_unit = 0.f;   // l_unit = 2^(eref - lift): sums of weights over it and the scale are l's

        if (!w.whole && w.t0 == 0 && tid == 0) {
          const int parts = (int)quotient(w.base + (int64_t)(w.tiles - 1) * w.cost, share) - (int)blockIdx.x + 1;
          cut.notes[blockIdx.x] = {w.rw.first, w.b, w.kvh, w.u * kPairRows, w.rows, parts};
        }
        // The scores of a step are read as soon as the weights of the one before are formed; if they are there, beside the storing of those.
        uint32_t s[64];
        auto fetch = [&](uint32_t buf) {
          tc_fence_after();
          tmem_ld32(ts0 + 64 * buf, s);
          tmem_ld32(ts0 + 64 * buf + 32, s + 32);
        };
        // (a line's steps come in pairs: so does every buffer's phase)
        alive = mbar_wait(bar(kSFull + 2 * a), steps >> 1 & 1, abort_flag);
        fetch(0);
        // Its scales, of four groups of sixteen keys: factors of the scores, exponents of the weights and their inverses.  (Waited for behind
        // the first scores: once a tile's are there, its scales are the next that the ring's slot waits for.)
        float4 k4, v4, i4;
        auto scales = [&](uint32_t tile, uint32_t buf) {
          const uint32_t at = scales_at + tile % kRing * (uint32_t)sizeof(Misc::Scales) + 16 * buf;
          k4 = ld_shared_f4(at);
          v4 = ld_shared_f4(at + 32);
          i4 = ld_shared_f4(at + 64);
        };
        alive = alive && mbar_wait(bar(kScales + tile_count % kRing), tile_count / kRing & 1, abort_flag);
        scales(tile_count, 0);
        for (int u = 0; u < 2 * n_tiles && alive; ++u, ++steps) {
          const uint32_t buf = u & 1, next = buf ^ 1;
          const bool more = u + 1 < 2 * n_tiles;
          const uint32_t next_bar = bar(kSFull + 2 * a + next), next_phase = (steps + 1) >> 1 & 1;
          const uint32_t next_tile = tile_count + buf, scales_bar = bar(kScales + next_tile % kRing), scales_phase = next_tile / kRing & 1;
          bool scored = false, scaled = false;   // whether the next step's scores and scales are there
          const int key0 = (w.t0 + (u >> 1)) * kKeys + 64 * buf;
          auto step = [&](auto edge_t) {
            constexpr bool EDGE = decltype(edge_t)::value;
            const float cs = CAP ? c * cap_inverse : c;
            float ck[4] = {cs * k4.x, cs * k4.y, cs * k4.z, cs * k4.w};
            const float e[4] = {v4.x, v4.y, v4.z, v4.w};
            const float inverse[4] = {i4.x, i4.y, i4.z, i4.w};
            tc_wait_ld();
            if constexpr (CAP) {   // the scores become capped logits; factors of one are left
              float far = 0.f;
#pragma unroll
              for (int k = 0; k < 64; k += 2) {
                const uint64_t x = mul2(aidn::pack2(__uint_as_float(s[k]), __uint_as_float(s[k + 1])), aidn::pack2(ck[k / 16], ck[k / 16]));
                const float2 v = unpack2(x);
                far = fmax3(far, fabsf(v.x), fabsf(v.y));
                s[k] = __float_as_uint(v.x);
                s[k + 1] = __float_as_uint(v.y);
              }
              const float most = p.softcap * kLog2e;
              if (__any_sync(0xffffffffu, far > 1.f)) {
#pragma unroll
                for (int k = 0; k < 64; ++k) s[k] = __float_as_uint(most * tanh_ex2(__uint_as_float(s[k])));
              } else {
                const uint64_t most2 = aidn::pack2(most, most);
#pragma unroll
                for (int k = 0; k < 64; k += 2) {
                  const float2 v = unpack2(mul2(tanh_small(aidn::pack2(__uint_as_float(s[k]), __uint_as_float(s[k + 1]))), most2));
                  s[k] = __float_as_uint(v.x);
                  s[k + 1] = __float_as_uint(v.y);
                }
              }
#pragma unroll
              for (int g = 0; g < 4; ++g) ck[g] = 1.f;
            }
            if constexpr (EDGE) {   // what a row does not see is -inf, a key with a NaN among its values NaN
#pragma unroll
              for (int q = 0; q < 2; ++q) {
                const uint32_t nan = ld_shared_u32(scales_at + tile_count % kRing * (uint32_t)sizeof(Misc::Scales) + (uint32_t)offsetof(Misc::Scales, nan) + 8 * buf + 4 * q);
#pragma unroll
                for (int k = 0; k < 32; ++k) {
                  if (nan >> k & 1) s[32 * q + k] = 0x7fffffffu;
                  if (key0 + 32 * q + k >= lim) s[32 * q + k] = 0xff800000u;
                }
              }
            }
            // The weights are formed with the maximum so far: again, once, if their sum says that they may not fit, with the step's own.  From logits
            // of 2^20 on the exponents are formed from differences, of products that are rounded as the maximum was: none is then above it, where a
            // fused multiply-add has the product's rounding, 2^(p - 24) for a logit of 2^p, in the exponent.  Such rows take the maximum first.
            auto large = [&] { return __any_sync(0xffffffffu, fabsf(m) > kLargeLogit && m != kUnset); };
            bool again = large(), far = again;   // (again: of the warp)
            float sum, base_m = m;               // base_m: what the scores, or differences, have to come down by
            for (;;) {
              if (again) {
                float keep = 1.f;
                if (far) {
                  float top = m, y[4];   // of the groups of which the row sees a key
#pragma unroll
                  for (int g = 0; g < 4; ++g) {
                    float m0 = __uint_as_float(s[16 * g]);
#pragma unroll
                    for (int k = 1; k < 15; k += 2) m0 = fmax3(m0, __uint_as_float(s[16 * g + k]), __uint_as_float(s[16 * g + k + 1]));
                    m0 = fmaxf(m0, __uint_as_float(s[16 * g + 15]));
                    y[g] = e[g] != -INFINITY && m0 != -INFINITY ? m0 * ck[g] : -INFINITY;
                    top = fmaxf(top, y[g]);
                  }
                  const float down = m - top;
                  float now = eref + down;   // eref: the largest (x - m) + e
#pragma unroll
                  for (int g = 0; g < 4; ++g) now = fmaxf(now, (y[g] - top) + e[g]);
                  keep = ex2_approx(down + (eref - now));
                  l *= ex2_approx(down);
                  m = top;
                  eref = now;
                  l_unit = ex2_approx(eref - kLift);
                }
                if (u > 0 && __any_sync(0xffffffffu, keep != 1.f)) {   // (one product at most is on its way, that of the step before: the next needs these weights)
                  if (!mbar_wait(bar(kODone + 2 * a + (buf ^ 1)), (steps - 1) >> 1 & 1, abort_flag)) alive = false;
                  tc_fence_after();
#pragma unroll 1
                  for (int q = 0; q < HD / 16; ++q) {
                    uint32_t o[16];
                    tmem_ld16(to + 16 * q, o);
                    tc_wait_ld();
#pragma unroll
                    for (int k = 0; k < 16; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * keep);
                    tmem_st16(to + 16 * q, o);
                  }
                }
                base_m = m;
                if (large()) {
#pragma unroll
                  for (int k = 0; k < 64; ++k) {
                    const float x = __uint_as_float(s[k]);
                    if (!EDGE || x != -INFINITY) s[k] = __float_as_uint(__fsub_rn(__fmul_rn(x, ck[k / 16]), m));
                  }
#pragma unroll
                  for (int g = 0; g < 4; ++g) ck[g] = 1.f;
                  base_m = 0.f;
                }
              }
              float most = 0.f;
              sum = 0.f;
#pragma unroll
              for (int q = 0; q < 2; ++q) {
                if (q == 1) {   // (looked at beside the arithmetic: shared memory is busy with the products' operands, and answers in 200 cycles)
                  scored = mbar_test(next_bar, next_phase);
                  scaled = mbar_test(scales_bar, scales_phase);
                }
                uint32_t packed[16];
#pragma unroll
                for (int h2 = 0; h2 < 2; ++h2) {
                  const int g = 2 * q + h2;
                  const float off = e[g] - (eref + base_m - kLift);
                  const uint64_t ck2 = aidn::pack2(ck[g], ck[g]), off2 = aidn::pack2(off, off);
                  uint64_t sum_g = 0;
#pragma unroll
                  for (int k = 0; k < 16; k += 2) {
                    const float u0 = __uint_as_float(s[16 * g + k]), u1 = __uint_as_float(s[16 * g + k + 1]);
                    float2 y;
                    y = unpack2(fma2(aidn::pack2(u0, u1), ck2, off2));
                    y.x = ex2_approx(y.x);
                    y.y = ex2_approx(y.y);
                    if constexpr (EDGE) {   // (a scale of zero times -inf)
                      y.x = u0 == -INFINITY ? 0.f : y.x;
                      y.y = u1 == -INFINITY ? 0.f : y.y;
                    }
                    sum_g = add2(sum_g, aidn::pack2(y.x, y.y));
                    packed[8 * h2 + (k >> 1)] = ptx::pack2<false>(y.x, y.y);
                  }
                  const float part = sum2(sum_g);
                  most = fmaxf(most, part);
                  sum = fmaf(part, inverse[g], sum);
                }
                tmem_st16(ts0 + 64 * buf + 16 * q, packed);
              }
              if (again) break;
              far = most > kMostWeights || sum * l_unit > kMostSum;
              if (!__any_sync(0xffffffffu, far)) break;
              again = true;
            }
            l = fmaf(sum, l_unit, l);
          };
          // (uniform.  All of these rows may see all of these keys, and yet their tile be one that was cleaned, for its other keys or the pair's first rows)
          bool edge = key0 + 64 > lim_least || key0 + 64 > w.keys;
          if (!edge && key0 - 64 * (int)buf + kKeys > lim_pair) {
            const uint32_t nan = scales_at + tile_count % kRing * (uint32_t)sizeof(Misc::Scales) + (uint32_t)offsetof(Misc::Scales, nan) + 8 * buf;
            edge = (ld_shared_u32(nan) | ld_shared_u32(nan + 4)) != 0;
          }
          if (edge) step(std::true_type{});
          else step(std::false_type{});
          scored = __all_sync(0xffffffffu, scored) && more;
          scaled = __all_sync(0xffffffffu, scaled) && more;
          if (scaled) scales(next_tile, next);
          if (scored) fetch(next);
          tc_wait_st();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(bar(kPFull + 2 * a + buf));
          if (more && !scored) {
            alive = alive && mbar_wait(next_bar, next_phase, abort_flag);
            fetch(next);
          }
          if (more && !scaled) {
            alive = alive && mbar_wait(scales_bar, scales_phase, abort_flag);
            scales(next_tile, next);
          }
          tile_count += buf;
        }
        if (!alive) break;
        // ---- results (a line's last step is one of the second buffer)
        if (!mbar_wait(bar(kODone + 2 * a + 1), (steps - 1) >> 1 & 1, abort_flag)) {
          alive = false;
          break;
        }
        tc_fence_after();
        const float f = w.whole ? (l == 0.f ? 0.f : l_unit / l) : l_unit;
        // Rows go out through this warp's part of the queries' tile, which nothing reads any more: 256 bytes a row at a time, lanes along rows.
        const int slot = 2 * (int)blockIdx.x + (w.t0 == 0 ? 1 : 0), prow = a * kTileRows + row_in;
        const uint32_t stage = base + C::kQ + a * C::kTile + warp_row * 128;
        constexpr int kSlabs = HD / 64;
        auto put = [&](int at16, uint32_t x, uint32_t y, uint32_t z, uint32_t v) {   // sixteen bytes of this thread's row
          st_shared_v4(stage + (at16 >> 3) * C::kSlab + lane * 128 + (((at16 & 7) ^ (lane & 7)) << 4), x, y, z, v);
        };
        auto rows_out = [&](auto&& store) {   // store(row, sixteen bytes' number, them)
          __syncwarp();
          constexpr int kOut = 8 * kSlabs, kRowsAtOnce = 32 / kOut;
          const int at16 = lane % kOut, s2 = lane / kOut;
#pragma unroll 2
          for (int j = 0; j < 32 / kRowsAtOnce; ++j) {
            const int row = j * kRowsAtOnce + s2;
            const uint4 v = ld_shared_v4(stage + (at16 >> 3) * C::kSlab + row * 128 + (((at16 & 7) ^ (row & 7)) << 4));
            if (row < warp_rows) store(row, at16, v);
          }
          __syncwarp();
        };
        if (w.whole) {
#pragma unroll 1
          for (int q = 0; q < HD / 32; ++q) {
            uint32_t x[32];
            tmem_ld32(to + 32 * q, x);
            tc_wait_ld();
#pragma unroll
            for (int e = 0; e < 32; e += 2) {
              const float y = __uint_as_float(x[e]) * f, z = __uint_as_float(x[e + 1]) * f;
              x[e / 2] = p.dtype == AIDN_F16 ? ptx::pack2<false>(y, z) : ptx::pack2<true>(y, z);
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) put(4 * q + e, x[4 * e], x[4 * e + 1], x[4 * e + 2], x[4 * e + 3]);
          }
          const int first = w.u * kPairRows + a * kTileRows + warp_row;
          rows_out([&](int row, int at16, uint4 v) {
            const int qi = (first + row) / G, gh = (first + row) - qi * G;
            const int64_t at = query_at(p, p.os, w.rw, w.b, (p.kv_begin + w.kvh) * G + gh, qi) + 8 * at16;
            uint16_t* const dst = static_cast<uint16_t*>(p.out) + at;
            if (cut.out_vec) {
              *reinterpret_cast<uint4*>(dst) = v;
            } else {
              const uint32_t words[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                dst[2 * e] = (uint16_t)words[e];
                dst[2 * e + 1] = (uint16_t)(words[e] >> 16);
              }
            }
          });
        } else {
          float* const part = cut.partial + ((int64_t)slot * kPairRows + a * kTileRows + warp_row) * HD;
#pragma unroll 1
          for (int half = 0; half < 2; ++half) {   // HD / 2 floats: as many bytes as a row of queries
#pragma unroll 1
            for (int q = 0; q < HD / 64; ++q) {
              uint32_t x[32];
              tmem_ld32(to + half * (HD / 2) + 32 * q, x);
              tc_wait_ld();
#pragma unroll
              for (int e = 0; e < 32; ++e) x[e] = __float_as_uint(__uint_as_float(x[e]) * f);
#pragma unroll
              for (int e = 0; e < 8; ++e) put(8 * q + e, x[4 * e], x[4 * e + 1], x[4 * e + 2], x[4 * e + 3]);
            }
            rows_out([&](int row, int at16, uint4 v) {
              __stcg(reinterpret_cast<uint4*>(part + (int64_t)row * HD + half * (HD / 2) + 4 * at16), v);
            });
          }
        }
        if (valid && w.whole && p.lse) *lse_at(p, w.rw, h, i) = l == 0.f ? -INFINITY : (m + log2f(l)) * kLn2;
        if (valid && !w.whole) __stcg(cut.stats + (int64_t)slot * kPairRows + prow, make_float2(m, l));
        tc_fence_before();   // (the next line's products come behind this warp's next arrival)
      }
    }
  } else if (warp < kMmaWarp) {
    // ======================================= keys and values: codes to fp16 =======================================
    setmaxnreg_dec<kConvertRegs>();
    const int quarter = warp & 3, t4 = lane & 3, g8 = lane >> 2;   // this warp: keys 32 quarter .. + 31; a lane: row g8 (+ 8 i), 16 bytes t4
    constexpr int H = HD / 64;
    const int64_t pitch = p.c.stride[1];
    const uint32_t dst0 = base + (uint32_t)((32 * quarter + g8) * 128);
    uint32_t count = 0;
    if (alive) {
      Walk w = walk();
      for (bool first = true; alive && w.next(first); first = false) {
        const int kvh = p.kv_begin + w.kvh;
        const int64_t lane_at = kvh * p.c.stride[2] + 16 * t4 + g8 * pitch;
        const int32_t* const table = p.c.table + w.b * p.c.table_stride;
        // lane e of this: the block of keys 32 quarter + 16 (e & 1) .. of a tile
        auto entry_of = [&](int t) {
          const int key = t * kKeys + 32 * quarter + 16 * (lane & 1);
          return t < w.t1 && key < w.keys ? checked_block(p.c, table[block_of(p.c, key)], bad) : -1;
        };
        uint4 xk[4][H], xv[4][H];
        int entry = entry_of(w.t0), entry_n;   // of the tile that is loaded, and of the next
        auto load = [&](const uint8_t* pool, int t, uint4 (&x)[4][H]) {
          const int key0 = t * kKeys + 32 * quarter;
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const int ent = __shfl_sync(0xffffffffu, entry, j), key = key0 + 16 * j;
            const uint8_t* at = pool + lane_at + ent * p.c.stride[0] + (key - block_of(p.c, key) * p.c.block_size) * pitch;
            if (ent >= 0 && key + 16 <= w.keys) {
#pragma unroll
              for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int q = 0; q < H; ++q) x[2 * j + i][q] = ld_stream16(at + i * 8 * pitch + 64 * q);
            } else {
#pragma unroll
              for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int q = 0; q < H; ++q)
                  x[2 * j + i][q] = ent >= 0 && key + 8 * i + g8 < w.keys ? ld_stream16(at + i * 8 * pitch + 64 * q) : make_uint4(0, 0, 0, 0);
            }
          }
        };
        auto convert = [&](uint32_t dst, const uint4 (&x)[4][H]) {
#pragma unroll
          for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int q = 0; q < H; ++q) {
              const uint4 v = x[i][q];
              const uint32_t at = dst + i * 1024 + q * C::kSlab;   // 16 elements: chunks 2 t4 and 2 t4 + 1 of the row's eight
              st_shared_v4(at + (((2 * t4) ^ g8) << 4), codes_to_f16(v.x), codes_to_f16_hi(v.x), codes_to_f16(v.y), codes_to_f16_hi(v.y));
              st_shared_v4(at + (((2 * t4 + 1) ^ g8) << 4), codes_to_f16(v.z), codes_to_f16_hi(v.z), codes_to_f16(v.w), codes_to_f16_hi(v.w));
            }
          fence_proxy_async_smem();
          __syncwarp();
        };
        auto scale_of = [&](const float* scales) { return entry >= 0 ? scales[(int64_t)entry * p.c.kv_heads + kvh] : 0.f; };
        const int lim_least = visible(p, w.keys, w.rw.count, w.u * kPairRows / G);
        load(p.c.k, w.t0, xk);
        load(p.c.v, w.t0, xv);
        float ks = scale_of(p.c.k_scale), vs = scale_of(p.c.v_scale);
        entry_n = entry_of(w.t0 + 1);
        for (int t = w.t0; t < w.t1; ++t, ++count) {
          const uint32_t stage = count & 1, ring = count % kRing;
          const int before = entry;
          entry = entry_n;
          entry_n = entry_of(t + 2);
          if (!mbar_wait(bar(kKEmpty + stage), (count >> 1 & 1) ^ 1, abort_flag)) {
            alive = false;
            break;
          }
          convert(dst0 + C::kK + stage * C::kTile, xk);
          if (lane == 0) mbar_arrive(bar(kKFull + stage));
          if (t + 1 < w.t1) load(p.c.k, t + 1, xk);
          if (!mbar_wait(bar(kVEmpty + stage), (count >> 1 & 1) ^ 1, abort_flag)) {
            alive = false;
            break;
          }
          uint32_t nan = 0;
          if (t * kKeys + kKeys > lim_least) {   // NaN values of keys that some rows do not see
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              bool hit = false;
#pragma unroll
              for (int q = 0; q < H; ++q) {
                hit = hit || any_nan(xv[i][q].x) || any_nan(xv[i][q].y) || any_nan(xv[i][q].z) || any_nan(xv[i][q].w);
                xv[i][q].x = without_nan(xv[i][q].x); xv[i][q].y = without_nan(xv[i][q].y);
                xv[i][q].z = without_nan(xv[i][q].z); xv[i][q].w = without_nan(xv[i][q].w);
              }
              const uint32_t who = __ballot_sync(0xffffffffu, hit);
#pragma unroll
              for (int r = 0; r < 8; ++r)
                if (who >> (4 * r) & 15) nan |= 1u << (8 * i + r);
            }
          }
          if (lane < 2) {
            float exponent = log2_approx(vs);
            if (exponent < kLeastScale) exponent = kLeastScale;   // (a NaN stays one)
            Misc::Scales& sc = ms.scales[ring];
            sc.k[2 * quarter + lane] = ks;
            sc.v_exp[2 * quarter + lane] = before < 0 ? -INFINITY : exponent;
            // (of a NaN something finite: it is multiplied with zero for rows that do not see the keys)
            sc.v_inverse[2 * quarter + lane] = before < 0 ? 0.f : exponent == exponent ? ex2_approx(-exponent) : 1.f;
          }
          if (lane == 0) ms.scales[ring].nan[quarter] = nan;
          convert(dst0 + C::kV + stage * C::kTile, xv);
          if (lane == 0) {
            mbar_arrive(bar(kVFull + stage));
            mbar_arrive(bar(kScales + ring));
          }
          if (t + 1 < w.t1) {
            load(p.c.v, t + 1, xv);
            ks = scale_of(p.c.k_scale);
            vs = scale_of(p.c.v_scale);
          }
        }
      }
    }
  } else {
    // ================================================ products ================================================
    setmaxnreg_dec<kMmaRegs>();
    if (warp == kMmaWarp && alive) {
      const bool leader = elect_one();
      constexpr uint32_t idesc_s = make_idesc(kTileRows, 64, false, false), idesc_o = make_idesc(kTileRows, HD, false, true);
      const uint64_t qd = make_smem_desc(base + C::kQ, 16, 1024), kd = make_smem_desc(base + C::kK, 16, 1024);
      const uint64_t vd = make_smem_desc(base + C::kV, C::kSlab, 1024);
      uint32_t count = 0, q_uses[2] = {0, 0}, p_uses[2] = {0, 0};   // tiles of all lines; lines and steps of a row tile
      auto scores = [&](int a, uint32_t tile, int buf) {   // the 64 keys `buf` of a tile
        const uint64_t k0 = kd + (uint64_t)((tile & 1) * (C::kTile >> 4) + buf * (64 * 128 >> 4));
#pragma unroll
        for (int k = 0; k < HD / 16; ++k) {
          const uint64_t off = (uint64_t)((k >> 2) * (C::kSlab >> 4) + (k & 3) * 2);
          if (leader) mma_ss(tmem + a * 128 + 64 * buf, qd + (uint64_t)(a * (C::kTile >> 4)) + off, k0 + off, idesc_s, k > 0);
        }
        if (leader) tc_commit(bar(kSFull + 2 * a + buf));
      };
      Walk w = walk();
      for (bool first = true; alive && w.next(first); first = false) {
        const int two = w.rows > kTileRows ? 2 : 1, steps = 2 * (w.t1 - w.t0);
        for (int a = 0; a < two; ++a)
          alive = alive && mbar_wait(bar(kQFull + a), q_uses[a]++ & 1, abort_flag);
        alive = alive && mbar_wait(bar(kKFull + (count & 1)), count >> 1 & 1, abort_flag);
        if (!alive) break;
        tc_fence_after();
        for (int buf = 0; buf < 2; ++buf)
          for (int a = 0; a < two; ++a) scores(a, count, buf);
        if (leader) tc_commit(bar(kKEmpty + (count & 1)));
        for (int u = 0; u < steps; ++u) {
          const int buf = u & 1;
          const uint32_t tile = count + (u >> 1);
          const bool more = u + 2 < steps;
          if (buf == 0) {
            alive = alive && mbar_wait(bar(kVFull + (tile & 1)), tile >> 1 & 1, abort_flag);
            if (more) alive = alive && mbar_wait(bar(kKFull + ((tile + 1) & 1)), (tile + 1) >> 1 & 1, abort_flag);
          }
          if (!alive) break;
          for (int a = 0; a < two; ++a) {
            if (!mbar_wait(bar(kPFull + 2 * a + buf), p_uses[a]++ >> 1 & 1, abort_flag)) {
              alive = false;
              break;
            }
            tc_fence_after();
#pragma unroll
            for (int k = 0; k < 4; ++k)
              if (leader)
                mma_ts(tmem + C::kO + a * HD, tmem + a * 128 + 64 * buf + k * 8,
                       vd + (uint64_t)((tile & 1) * (C::kTile >> 4)) + (uint64_t)((4 * buf + k) * (2048 >> 4)), idesc_o, u > 0 || k > 0);
            if (leader) tc_commit(bar(kODone + 2 * a + buf));
            if (more) scores(a, tile + 1, buf);
          }
          if (!alive) break;
          if (buf == 1 && leader) {
            tc_commit(bar(kVEmpty + (tile & 1)));
            if (more) tc_commit(bar(kKEmpty + ((tile + 1) & 1)));
          }
        }
        count += steps >> 1;
      }
    }
  }

  // ---- teardown
  if (bad && p.status) atomicOr(p.status, kStatusBadBlock);
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  const bool gave_up = *abort_flag != 0;
  if (gave_up) {
    if (tid == 0) {
      abort_grace();
      if (p.status) atomicOr(p.status, kStatusTimeout);
    }
    __syncthreads();
  }
  if (warp == kMmaWarp) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// CTA (c, i): 16 rows of the line that begins in the share of CTA c and goes on behind it, a warp two of them.  (Bound by the latency of the parts: with
// four rows a warp and so many registers that an SM held one or two CTAs it took 19 us where it takes 12.)
constexpr int kMergeRows = 2;
template <int HD>
__global__ void __launch_bounds__(256, HD == 128 ? 3 : 4) kv8_sm100_merge_kernel(const __grid_constant__ Attend p, const Cut cut) {
  pdl_wait();
  pdl_trigger();
  const Note note = cut.notes[blockIdx.x];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, r0 = 8 * kMergeRows * blockIdx.y + kMergeRows * warp;
  if (note.parts == 0 || r0 >= note.rows) return;
  constexpr int N = HD / 32, R = kMergeRows;
  float top[R], sum[R] = {}, o[R][N] = {};
#pragma unroll
  for (int r = 0; r < R; ++r) top[r] = kUnset;
  for (int q = 0; q < note.parts; q += 4) {
    float2 st[4][R];
    float v[4][R][N];
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      const int part = min(q + x, note.parts - 1);
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const int64_t from = (int64_t)(2 * (blockIdx.x + part) + (part == 0)) * kPairRows + min(r0 + r, note.rows - 1);
        st[x][r] = cut.stats[from];
        const float* at = cut.partial + from * HD + N * lane;
        if constexpr (N == 4) {
          const float4 u = *reinterpret_cast<const float4*>(at);
          v[x][r][0] = u.x; v[x][r][1] = u.y; v[x][r][2] = u.z; v[x][r][3] = u.w;
        } else {
          const float2 u = *reinterpret_cast<const float2*>(at);
          v[x][r][0] = u.x; v[x][r][1] = u.y;
        }
      }
    }
#pragma unroll
    for (int r = 0; r < R; ++r) {
      float now = top[r];
#pragma unroll
      for (int x = 0; x < 4; ++x) now = fmaxf(now, st[x][r].x);
      const float keep = ex2_approx(top[r] - now);
      top[r] = now;
      sum[r] *= keep;
#pragma unroll
      for (int e = 0; e < N; ++e) o[r][e] *= keep;
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        if (q + x >= note.parts) continue;
        const float f = ex2_approx(st[x][r].x - now);
        sum[r] += f * st[x][r].y;
#pragma unroll
        for (int e = 0; e < N; ++e) o[r][e] += f * v[x][r][e];
      }
    }
  }
  const Rows rw = {note.first_row, 0};
#pragma unroll
  for (int r = 0; r < R; ++r) {
    if (r0 + r >= note.rows) continue;
    const int row = note.row + r0 + r, i = row / p.group, h = (p.kv_begin + note.kvh) * p.group + row - i * p.group;
    const float f = sum[r] == 0.f ? 0.f : 1.f / sum[r];
    const int64_t at = query_at(p, p.os, rw, note.b, h, i) + N * lane;
    uint16_t* const dst = static_cast<uint16_t*>(p.out) + at;
    uint32_t w[N / 2];
#pragma unroll
    for (int e = 0; e < N / 2; ++e)
      w[e] = p.dtype == AIDN_F16 ? ptx::pack2<false>(o[r][2 * e] * f, o[r][2 * e + 1] * f) : ptx::pack2<true>(o[r][2 * e] * f, o[r][2 * e + 1] * f);
    if (cut.out_vec) {
      if constexpr (N == 4) *reinterpret_cast<uint2*>(dst) = make_uint2(w[0], w[1]);
      else *reinterpret_cast<uint32_t*>(dst) = w[0];
    } else {
#pragma unroll
      for (int e = 0; e < N / 2; ++e) {
        dst[2 * e] = (uint16_t)w[e];
        dst[2 * e + 1] = (uint16_t)(w[e] >> 16);
      }
    }
    if (p.lse && lane == 0) *lse_at(p, rw, h, i) = sum[r] == 0.f ? -INFINITY : (top[r] + log2f(sum[r])) * kLn2;
  }
}

template <int HD, bool CAP>
cudaError_t launch(const Attend& p, int grid, const Cut& cut, uint64_t* raised, int* launches, cudaStream_t stream) {
  auto k = kv8_sm100_kernel<HD, CAP>;
  const int id = 60 + (HD == 128 ? 2 : 0) + (CAP ? 1 : 0);
  if (!(*raised >> id & 1)) {
    const cudaError_t e = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg<HD>::kSmem);
    if (e != cudaSuccess) return e;
    *raised |= 1ull << id;
  }
  const cudaError_t e = launch_dependent(k, dim3((unsigned)grid), kThreads, Cfg<HD>::kSmem, stream, p, cut);
  if (e != cudaSuccess || !cut.partial) return e;
  const int64_t rows = p.seq_q * p.group;
  const unsigned slices = (unsigned)((rows < kPairRows ? rows : kPairRows) + 8 * kMergeRows - 1) / (8 * kMergeRows);
  ++*launches;
  return launch_dependent(kv8_sm100_merge_kernel<HD>, dim3((unsigned)grid, slices), 256, 0, stream, p, cut);
}

}  // namespace

bool sm100_supported(const Attend& p) {
  if (p.dtype == AIDN_F32 || p.out_f32 || (p.c.head_dim != 64 && p.c.head_dim != 128) || p.mask_kind != AIDN_MASK_NONE) return false;
  if (p.c.block_size % 16 != 0 || (uintptr_t)p.c.k % 16 != 0 || (uintptr_t)p.c.v % 16 != 0) return false;
  for (int i = 0; i < 3; ++i)
    if (p.c.stride[i] % 16 != 0) return false;
  return p.seq_q * p.group < 0x7fffffff - kPairRows;
}
int64_t sm100_workspace_bytes(int head_dim, int num_sms) { return (int64_t)2 * num_sms * kPairRows * (head_dim * 4 + 8) + num_sms * (int64_t)sizeof(Note); }

cudaError_t launch_attend_sm100(const Attend& p, int num_sms, void* workspace, int64_t workspace_bytes, uint64_t* raised, int* launches, cudaStream_t stream) {
  const int grid = num_sms;
  if (workspace_bytes < sm100_workspace_bytes(p.c.head_dim, grid) || (uintptr_t)workspace % 16 != 0) workspace = nullptr;
  Cut cut;
  cut.partial = static_cast<float*>(workspace);
  cut.stats = workspace ? reinterpret_cast<float2*>(cut.partial + (int64_t)2 * grid * kPairRows * p.c.head_dim) : nullptr;
  cut.notes = workspace ? reinterpret_cast<Note*>(cut.stats + (int64_t)2 * grid * kPairRows) : nullptr;
  auto vec = [](const void* ptr, const int64_t* st) { return ((uintptr_t)ptr | (uint64_t)(st[0] * 2) | (uint64_t)(st[1] * 2) | (uint64_t)(st[2] * 2)) % 16 == 0; };
  cut.query_vec = vec(p.q, p.qs);
  cut.out_vec = vec(p.out, p.os);
  if (p.c.head_dim == 64) return p.softcap > 0.f ? launch<64, true>(p, grid, cut, raised, launches, stream) : launch<64, false>(p, grid, cut, raised, launches, stream);
  return p.softcap > 0.f ? launch<128, true>(p, grid, cut, raised, launches, stream) : launch<128, false>(p, grid, cut, raised, launches, stream);
}

}  // namespace kv8
}  // namespace aidn
