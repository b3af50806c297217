// The scan of linear.cuh for 16-bit tensors with sizes of 64 and 128, on tcgen05.  A CTA walks the rows of one sequence and head (or of one segment of
// them) in chunks of 64, with tensor memory lanes along c's columns, so that the state never leaves the registers of the threads that own it:
//
//     S   = A B^T                      scores, 64 x 64 (rows of A in lanes 0-63; the lanes above hold what is not looked at)
//     P   = S weighted by lam^(i-j), zeros where j follows i, as two 16-bit terms to shared memory
//     T^T = C~^T B                     C~ = rows of C weighted by lam^(n-lag-j), as two 16-bit terms (off by 2^-17 of a value in bf16, 2^-22
//                                      in fp16), or three for bf16 states that go out (2^-24, as fp32 rounds)
//     O^T = X^T A^T  and  C^T P^T      apart, since their columns have different factors; X^T in 16 bits in tensor memory
//     X   = lam^n X + T                in fp32 registers, then X^T rounded for the next chunk
//
// Rounded to 16 bits on the way to an output: X^T, as tensor memory has no columns for a second term of it at 128 (through shared memory it takes 67 -> 87 us of
// B4 S2048 H32 D128 in bf16, in tensor memory 54 -> 58 us of D64), and the output itself.  Against one rounding of what is exact, the errors are 1.0 times as large within a sequence's first chunk, 1.06 for a decay of 0.05 a row, and go to 1.41 where a state remembers
// everything.  (With P in one term they were 1.41 everywhere, up to 1.57 where its part and the state's cancel; its second term takes 2 to 10 %
// of a call: B4 S2048 H32 D128 in bf16 62.6 -> 66.6 us, 7 prompts to 8192 rows of the same heads 206 -> 228 us, with states 335 -> 345.  Columns by 32 in place of 16,
// or without those that are zeros for all rows of a warp: no faster.)
//
//   warps 0-1    P            warp 2   TMA producer (one thread)            warp 3   issues the products (one thread), owns tensor memory
//   warps 4-11   C~ and the state, a lane (column of c) and half of b's columns to a thread; C~^T goes to tensor memory by transposing loads
//   warps 12-15  output: O^T from tensor memory, weighted, by transposing stores to rows in shared memory, and out by TMA
//
// Rows are taken from a sequence's last to its first for the gradients of keys and values: a tile is loaded as it lies, and only masks and
// exponents turn around.  The last chunk's missing rows are zeros in C~, and in B and C, which multiply zeros.
//
// fp16: a row of P, a lane's row of X^T and a chunk's column of C~ are scaled by a power of two to their own largest value, as none is bound by fp16's
// range; the second term of C~ is held 2^11 times as large besides, and its product divided on the way into the first's.  A weighted value is then off by
// 2^-22 of itself, or by 2^-50 of the largest in its column and chunk, where fp16's smallest numbers cut the second term.  (Without C~'s scale that was
// 2^-36 whatever the values' size: a state of 7e-20 was zero, one of 1e-6 off by 6e-6.  It takes 67 -> 77 us of B4 S2048 H32 D64 with
// states, 83 -> 93 of D128, 233 -> 262 of that one's gradients; with scalar products and weights in registers 80, 101 and 284.  Formed by the output's
// warps in place of these, no less: what it costs are instructions.)
//
// What is not finite in C would reach earlier rows of its chunk as 0 * NaN in C^T P^T: columns that come out not finite are summed again, row by row, over
// what a row may see.
//
// Few sequences and heads: their rows are cut into segments.  A first launch forms what each segment adds to the state, a second one turns
// those into the states before the segments, and the scan then runs on all segments at once, at the price of b and c read twice.
//
// What bounds it: a chunk takes 1.4 us (sizes of 64) to 1.8 us (128), with 16 CTAs as with 128, where the bytes of 128 CTAs would take 1.28 us at 128:
// the chain of waits between the roles and their code, which is longer than the instruction cache holds (8 in 100 fetches of a line miss), not a unit.
// B4 S2048 H32 D128 in bf16: 65 to 72 us, 4.1 to 3.7 TB/s.  Measured on the way, with P in one term (us for that call, 63 to 71 then): roles unrolled over their rows 174, in loops 84, packed
// arithmetic and stores by TMA 70; C~ by shared memory in place of tensor memory 80; four more warps for C~ at 96 registers a thread 76; products issued by
// two warps, and those of T and O in turn, made no difference.
//
// Every wait is bounded; a CTA that gives up counts itself and leaves through the common teardown.
#include <cuda.h>

#include "ffma2.cuh"
#include "linear.cuh"
#include "sm100_ptx.cuh"
#include "tensor_map.hpp"

namespace aidn {
namespace lin {
namespace {

using namespace ptx;

// How many CTAs gave up a bounded wait in this context.  (The entry points have no handle whose status word could say so; never cleared, so that whoever asks
// can tell what is new to them.)
__device__ uint32_t g_linear_gave_up;

constexpr int kChunk = 64;
constexpr int kBlock = kChunk * 128;   // 64 rows of 64 16-bit elements
constexpr int kYBytes = kChunk * 64;   // 64 rows of 32
constexpr int kMaxSegments = 64;
constexpr int kMaxRanked = 64;         // sequences of a batch that is taken by lengths
constexpr int kThreads = 512;
constexpr int kWarpLoad = 2, kWarpMma = 3, kWarpState = 4, kWarpOut = 12;   // (warps 0 and 1: P)

template <int D1, int D2>
struct Cfg {
  static constexpr int kN1 = D1 / 64, kN2 = D2 / 64;
  static constexpr int kStageBytes = (2 * kN1 + kN2) * kBlock;
  static constexpr int kStages = 147456 / kStageBytes;            // 144 KB of tiles
  static constexpr int kOffB = kN1 * kBlock, kOffC = 2 * kN1 * kBlock;
  static constexpr int kOffP = kStages * kStageBytes;             // two buffers of two terms
  static constexpr int kOffY = kOffP + 4 * kBlock;                // output, 64 rows of 32 columns to a warp
  static constexpr int kOffTab = kOffY + 4 * kYBytes;
  // tables (floats): powers [65], weights of the scores by distance in four copies, each one element on from the one before (a row's begin anywhere
  // and are read by four), of the state's rows [64]; row scales of P [2][64], lane scales of X [4][128], exchange of the maxima of X and of C~, [2][2][128]
  // each, weights of C~'s rows with as many zeros [128], weights
  // of C~ by exponent, [2] 16-bit terms of [66], and of a whole chunk's pairs of rows as the threads take them, [2][2][4][4]
  static constexpr int kTabPower = 0, kTabScore = 68, kScorePitch = 136, kTabRow = kTabScore + 4 * kScorePitch, kTabP = kTabRow + 64, kTabX = kTabP + 128,
                       kTabMax = kTabX + 512, kTabC = kTabMax + 512, kTabRowsC = kTabC + 512, kTabW = kTabRowsC + 128, kTabPairs = kTabW + 68, kTabFloats = kTabPairs + 64;
  static constexpr int kOffBar = kOffTab + kTabFloats * 4;
  static constexpr int kBars = 2 * kStages + 24;
  static constexpr int kOffMisc = kOffBar + kBars * 8;
  static constexpr int kSmem = kOffMisc + 16 + 1024;
  // tensor memory columns: X^T in 16 bits, T^T, S, O^T (state part, row part), C~^T in 16 bits (two terms in two buffers, or three)
  static constexpr int kColX = 0, kColT = D1 / 2, kColS = kColT + D1, kColO = kColS + 64, kColC = kColO + 128;
  static_assert(kColC + 128 <= 512, "tensor memory");
};

struct Maps {
  CUtensorMap t[4];
  CUtensorMap y[3];
};

struct Args {
  Params p;
  int32_t ia[3], ib[3], ic[3];   // maps of a, b, c of each scan
  int32_t first, count;          // scans of this launch
  int32_t segments, seg_len;     // seg_len: a multiple of kChunk
  int32_t states_only;
  int32_t ranked;                // sequences from the longest to the shortest
  int32_t terms;                 // of C~: 2, or 3 for bf16 where states go out
  float* work;                   // [scan][sequence, head][segment][D1][D2]
  uint64_t wait_ns;
  int32_t withhold;              // test hook: no loads, so that the waits run out
};

__device__ __forceinline__ uint4 lds128(uint32_t a) {
  uint4 v;
  asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a));
  return v;
}
__device__ __forceinline__ uint32_t bf16x2_mul(uint32_t a, uint32_t b) {
  uint32_t d;
  asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  return d;
}
__device__ __forceinline__ uint32_t bf16x2_fma(uint32_t a, uint32_t b, uint32_t c) {
  uint32_t d;
  asm("fma.rn.bf16x2 %0, %1, %2, %3;" : "=r"(d) : "r"(a), "r"(b), "r"(c));
  return d;
}
template <bool BF16>
__device__ __forceinline__ float2 unpack16(uint32_t v) {
  if constexpr (BF16) return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u));
  else return __half22float2(*reinterpret_cast<__half2*>(&v));
}
template <bool BF16>
__device__ __forceinline__ float lds16(uint32_t a) {
  uint16_t v;
  asm volatile("ld.shared.b16 %0, [%1];" : "=h"(v) : "r"(a));
  if constexpr (BF16) return __uint_as_float((uint32_t)v << 16);
  else return __half2float(*reinterpret_cast<__half*>(&v));
}
// The rest of a wait that did not end at once, apart from the code of every place that waits: all of it has to stay in the instruction cache.
__device__ __noinline__ bool wait_on(uint32_t bar, uint32_t parity, volatile int* abort_flag, uint64_t wait_ns) {
  return mbar_wait(bar, parity, abort_flag, wait_ns);
}
// One term of the weights of rows j + 8 i, + 1 in a last chunk of n rows, zeros where there are none.
__device__ __noinline__ uint4 end_weights(const uint16_t* term, int j, int n, int lag, bool reverse) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    uint32_t v = 0;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const int at = reverse ? kChunk - 1 - (j + 8 * i + k) : j + 8 * i + k;
      if (at < n) v |= (uint32_t)term[n - lag - at] << (16 * k);
    }
    w[i] = v;
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}
// Powers of two that bring a largest value into [2^14, 2^15) and back.  (What is not finite, or so small that the power has no
// reciprocal, is left near where it is.)
__device__ __forceinline__ void scale_of(float largest, float& to, float& back) {
  int e = (__float_as_int(largest) >> 23) & 255;
  if (e == 255) {
    to = back = 1.f;
    return;
  }
  e = e < 15 ? 15 : e;
  to = __int_as_float((268 - e) << 23);
  back = __int_as_float((e - 14) << 23);
}

// D[tmem] = A[tmem] * B[smem] + D * 2^-11
__device__ __forceinline__ void mma_ts_down11(uint32_t d_tmem, uint32_t a_tmem, uint64_t b_desc, uint32_t idesc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.eq.b32 p, 0, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p, 11;\n\t}"
      ::"r"(d_tmem), "r"(a_tmem), "l"(b_desc), "r"(idesc)
      : "memory");
}
// Four 8 x 8 tiles of 16-bit elements, transposed: thread t holds row t / 4 and columns 2 (t % 4), + 1 of each.
__device__ __forceinline__ void ldmatrix_x4_trans(uint32_t addr, uint32_t* r) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
// The other way: four 8 x 8 tiles to shared memory, transposed.
__device__ __forceinline__ void stmatrix_x4_trans(uint32_t addr, const uint32_t* r) {
  asm volatile("stmatrix.sync.aligned.m8n8.x4.trans.shared.b16 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]) : "memory");
}
__device__ __forceinline__ void sts16(uint32_t addr, uint32_t v) { asm volatile("st.shared.b16 [%0], %1;" ::"r"(addr), "h"((uint16_t)v) : "memory"); }
// 16 lanes x 32 columns: r[4 i], r[4 i + 1] hold lane t / 4 and columns 8 i + 2 (t % 4), + 1; r[4 i + 2], r[4 i + 3] the lane 8 above.
__device__ __forceinline__ void tmem_ld_16x256b_x4(uint32_t taddr, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.16x256b.x4.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]),
        "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr)
      : "memory");
}
// 16 lanes x 16 columns: r[2 i] holds lane t / 4 and column 4 i + t % 4, r[2 i + 1] the lane 8 above.
__device__ __forceinline__ void tmem_st_16x128b_x4(uint32_t taddr, const uint32_t* r) {
  asm volatile("tcgen05.st.sync.aligned.16x128b.x4.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};"
               ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
               : "memory");
}

// The sequence that `rank` longer ones precede (of equal ones, the first first).  Called by all threads of a CTA.
__device__ __forceinline__ int sequence_of_rank(const Params& p, int rank) {
  __shared__ int64_t rows[kMaxRanked];
  __shared__ int found;
  const int mine = threadIdx.x;
  if (mine < p.batch) rows[mine] = p.starts ? (int64_t)p.starts[mine + 1] - p.starts[mine] : (int64_t)p.lengths[mine];
  __syncthreads();
  if (mine < p.batch) {
    int before = 0;
    for (int i = 0; i < p.batch; ++i) before += rows[i] > rows[mine] || (rows[i] == rows[mine] && i < mine) ? 1 : 0;
    if (before == rank) found = mine;
  }
  __syncthreads();
  return found;
}

template <int D1, int D2, bool BF16>
__global__ void __launch_bounds__(kThreads, 1) scan_sm100_kernel(const __grid_constant__ Maps maps, const __grid_constant__ Args args) {
  using C = Cfg<D1, D2>;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  uint8_t* gen = smem_raw + (base - smem_u32(smem_raw));
  float* table = reinterpret_cast<float*>(gen + C::kOffTab);
  const uint32_t bars = base + C::kOffBar;
  const uint32_t b_full = bars, b_empty = bars + 8 * C::kStages;
  // (in pairs: for chunks in turn, where more than one role waits, or one that may be a chunk behind)
  uint32_t next_bar = bars + 16 * C::kStages;
  auto bar = [&](int n) { const uint32_t at = next_bar; next_bar += 8 * n; return at; };
  const uint32_t b_s_full = bar(2), b_s_empty = bar(1), b_p_full = bar(2), b_o_full = bar(2), b_o_empty = bar(2), b_bt_full = bar(2);
  const uint32_t b_t_full = bar(1), b_t_empty = bar(1), b_x_full = bar(1), b_x_empty = bar(1);
  const uint32_t b_max = bar(4), b_most = bar(4);   // of the two warps that share lanes: X, C~
  uint32_t* tmem_ptr = reinterpret_cast<uint32_t*>(gen + C::kOffMisc);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(gen + C::kOffMisc + 4);

  const Params& p = args.p;
  const int which = args.first + (int)(blockIdx.x % (unsigned)args.count);
  const unsigned unit = blockIdx.x / (unsigned)args.count;
  const int seg = (int)(unit % (unsigned)args.segments);
  const int place = (int)(unit / (unsigned)args.segments) / p.heads, h = (int)(unit / (unsigned)args.segments) - place * p.heads;
  const int b = args.ranked ? sequence_of_rank(p, place) : place, item = b * p.heads + h;
  const Scan& s = p.scan[which];
  const bool states_only = args.states_only != 0;
  // (shuffled from lane 0: what depends on it is known to be the same in a warp, and stays in uniform registers)
  const int warp = __shfl_sync(0xffffffffu, (int)(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;
  const bool reverse = s.reverse != 0;
  const uint64_t wait_ns = args.wait_ns;

  const Sequence q = sequence_of(p, b);
  const int64_t t0 = (int64_t)seg * args.seg_len;
  const int rows = q.bad || q.n <= t0 ? 0 : (int)(q.n - t0 < args.seg_len ? q.n - t0 : args.seg_len);
  const int chunks = __shfl_sync(0xffffffffu, (rows + kChunk - 1) / kChunk, 0);
  const int64_t y0 = (p.starts ? 0 : b * s.ys[0]) + h * s.ys[1] + q.row0 * s.ys[2];
  // rows from tile row r of chunk c: token_of(c) + r, of the sequence
  auto token_of = [&](int c) { return reverse ? (int)(q.n - t0) - (c + 1) * kChunk : (int)t0 + c * kChunk; };

  // the segments that were empty have nothing before them either, but a state may have to be handed on
  const bool run = chunks > 0 || (!q.bad && args.segments == 1 && s.x_last && q.state >= 0);
  if (run) {
    if (threadIdx.x == 0) {
      *abort_flag = 0;
      for (int i = 0; i < C::kStages; ++i) {
        mbar_init(b_full + 8 * i, 1);
        mbar_init(b_empty + 8 * i, 1);
      }
      mbar_init(b_s_empty, 2);
      for (int i = 0; i < 2; ++i) {
        mbar_init(b_s_full + 8 * i, 1);
        mbar_init(b_p_full + 8 * i, 2);
        mbar_init(b_bt_full + 8 * i, 8);
        mbar_init(b_o_full + 8 * i, 1);
        mbar_init(b_o_empty + 8 * i, 4);
      }
      mbar_init(b_t_full, 1);
      mbar_init(b_t_empty, 8);
      mbar_init(b_x_full, 8);
      mbar_init(b_x_empty, 1);
      for (int i = 0; i < 4; ++i) {
        mbar_init(b_max + 8 * i, 2);
        mbar_init(b_most + 8 * i, 2);
      }
      fence_mbar_init();
    }
    const double g = log_decay(p.decay, h);
    if (threadIdx.x < 65) {
      const float w = decay_power(g, threadIdx.x);
      table[C::kTabPower + threadIdx.x] = w;
      if constexpr (BF16) {
        uint16_t* terms = reinterpret_cast<uint16_t*>(table + C::kTabW);
        float left = w * s.key_scale;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const uint32_t t = pack2<true>(left, 0.f) & 0xffffu;
          terms[i * 66 + threadIdx.x] = (uint16_t)t;
          const int j = reverse ? (int)threadIdx.x + s.lag - 1 : kChunk - s.lag - (int)threadIdx.x;   // the row of a whole chunk with this exponent
          if (j >= 0 && j < kChunk)
            reinterpret_cast<uint16_t*>(table + C::kTabPairs + i * 32)[((j / 32) * 16 + ((j % 8) / 2) * 4 + (j % 32) / 8) * 2 + (j & 1)] = (uint16_t)t;
          left -= __uint_as_float(t << 16);
        }
      } else {
        const int j = reverse ? (int)threadIdx.x + s.lag - 1 : kChunk - s.lag - (int)threadIdx.x;   // (as above)
        if (j >= 0 && j < kChunk) {
          table[C::kTabRowsC + j + (reverse ? kChunk : 0)] = w;
          table[C::kTabRowsC + j + (reverse ? 0 : kChunk)] = 0.f;
        }
      }
    }
    else if (threadIdx.x >= 96 && threadIdx.x < 160) {
      const int r = threadIdx.x - 96;
      table[C::kTabRow + r] = s.row_scale * decay_power(g, (reverse ? kChunk - 1 - r : r) + s.lag);
    } else if (threadIdx.x >= 256 && threadIdx.x < 384) {   // of row i and column j at 63 - i + j; zeros where j follows i
      const int x = (int)threadIdx.x - 256, d = reverse ? x - 63 : 63 - x;
      const float w = d >= 0 ? p.scale * decay_power(g, d) : 0.f;
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (x >= i) table[C::kTabScore + i * C::kScorePitch + x - i] = w;
    }
    if (warp == kWarpMma) {
      tmem_alloc(smem_u32(tmem_ptr), 512);
      tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = __shfl_sync(0xffffffffu, *tmem_ptr, 0);
    const float* power = table + C::kTabPower;
    auto wait = [&](uint32_t bar, uint32_t parity) {
      bool done = mbar_try_wait(bar, parity);
      if (!done) done = wait_on(bar, parity, abort_flag, wait_ns);
      return __all_sync(0xffffffffu, done) != 0;
    };
    // a single thread's
    auto wait1 = [&](uint32_t bar, uint32_t parity) { return mbar_try_wait(bar, parity) || wait_on(bar, parity, abort_flag, wait_ns); };
    auto arrive = [&](uint32_t bar) {
      __syncwarp();
      if (lane == 0) mbar_arrive(bar);
    };

    if (warp == kWarpLoad) {
      // ---- tiles in ----
      if (elect_one()) {
        const CUtensorMap* ma = &maps.t[args.ia[which]];
        const CUtensorMap* mb = &maps.t[args.ib[which]];
        const CUtensorMap* mc = &maps.t[args.ic[which]];
        const int ha = h / s.a_group, hb = h / s.b_group, hc = h / s.c_group, bb = p.starts ? 0 : b;
        int at = 0;
        uint32_t phase = 1;
        for (int c = 0; c < chunks; ++c) {
          if (!wait1(b_empty + 8 * at, phase)) break;
          if (!args.withhold) {
            const uint32_t bar = b_full + 8 * at, dst = base + (uint32_t)(at * C::kStageBytes);
            const int row = (int)q.row0 + token_of(c);
            mbar_expect_tx(bar, (uint32_t)(states_only ? C::kStageBytes - C::kOffB : C::kStageBytes));
#pragma unroll
            for (int i = 0; i < C::kN1; ++i) {
              if (!states_only) tma_load_4d(dst + i * kBlock, ma, bar, i * 64, row, ha, bb);
              tma_load_4d(dst + C::kOffB + i * kBlock, mb, bar, i * 64, row, hb, bb);
            }
#pragma unroll
            for (int i = 0; i < C::kN2; ++i) tma_load_4d(dst + C::kOffC + i * kBlock, mc, bar, i * 64, row, hc, bb);
          }
          if (++at == C::kStages) at = 0, phase ^= 1u;
        }
      }
    } else if (warp == kWarpMma) {
      // ---- products ----
      constexpr uint32_t kTransposeA = 1u << 15;
      constexpr uint32_t idesc_rows = make_idesc(128, 64, BF16, false);               // S: A and B along their rows; state part: X^T from tensor memory
      constexpr uint32_t idesc_p = make_idesc(128, 64, BF16, false) | kTransposeA;    // C^T, P along its rows
      constexpr uint32_t idesc_t = make_idesc(128, D1, BF16, true);                   // C~^T from tensor memory, B across its rows
      // (a descriptor's start address is counted in 16 bytes; what is added to it stays within its field)
      const uint64_t rows_desc = make_smem_desc(base, 16, 1024), cols_desc = make_smem_desc(base, kBlock, 1024);
      auto row_step = [](int k) { return (uint64_t)(((k / 4) * kBlock + (k % 4) * 32) >> 4); };   // 16 elements along a row
      // One thread for the waits too: a wait of the whole warp takes 100 cycles where there is nothing to wait for.
      if (elect_one()) {
        const bool third = args.terms == 3;
        int at = 0, ahead = 0;   // the chunk's stage; the next chunk whose scores are to be issued
        uint32_t phase = 0;
        for (int c = 0; c < chunks; ++c) {
          const uint64_t stage = (uint64_t)(at * (C::kStageBytes >> 4));
          const int next = at + 1 == C::kStages ? 0 : at + 1;
          const uint32_t next_phase = phase ^ (next == 0 ? 1u : 0u);
          // This chunk's scores, if they are not ahead; the next one's if its tiles are there; what is added to the state; and only then what waits for the
          // state and for P.
          bool ok = true;
          while (!states_only && ahead <= c + 1 && ahead < chunks) {
            const int slot = ahead == c ? at : next;
            const uint32_t slot_phase = ahead == c ? phase : next_phase;
            if (ahead > c ? !mbar_test(b_full + 8 * slot, slot_phase) : !(ok = wait1(b_full + 8 * slot, slot_phase))) break;
            if (!(ok = wait1(b_s_empty, (uint32_t)(ahead & 1) ^ 1u))) break;
            tc_fence_after();
            const uint64_t ad = rows_desc + (uint64_t)(slot * (C::kStageBytes >> 4)), bd = ad + (C::kOffB >> 4);
#pragma unroll
            for (int k = 0; k < D1 / 16; ++k) mma_ss(tmem + C::kColS, ad + row_step(k), bd + row_step(k), idesc_rows, k > 0);
            tc_commit(b_s_full + 8 * (ahead & 1));
            ++ahead;
          }
          // (the tiles have been waited for with the scores; a state that has been put down has left T's columns)
          if (!ok || !wait1(b_bt_full + 8 * (c & 1), (uint32_t)((c >> 1) & 1))) break;
          if (states_only ? !wait1(b_full + 8 * at, phase) || !wait1(b_t_empty, (uint32_t)(c & 1) ^ 1u) : !wait1(b_x_full, (uint32_t)(c & 1))) break;
          tc_fence_after();
          const uint64_t ct = cols_desc + stage + (C::kOffC >> 4), bt = cols_desc + stage + (C::kOffB >> 4);
          const uint32_t first = tmem + C::kColC + (third ? 0 : (c & 1) * 64);
          // the smallest term first (fp16 holds its second 2^11 times as large)
          if (third) {
#pragma unroll
            for (int k = 0; k < kChunk / 16; ++k) mma_ts(tmem + C::kColT, first + 64 + k * 8, bt + k * (2048 >> 4), idesc_t, k > 0);
          }
#pragma unroll
          for (int k = 0; k < kChunk / 16; ++k) mma_ts(tmem + C::kColT, first + 32 + k * 8, bt + k * (2048 >> 4), idesc_t, k > 0 || third);
#pragma unroll
          for (int k = 0; k < kChunk / 16; ++k) {
            if (!BF16 && k == 0) mma_ts_down11(tmem + C::kColT, first, bt, idesc_t);
            else mma_ts(tmem + C::kColT, first + k * 8, bt + k * (2048 >> 4), idesc_t, 1u);
          }
          tc_commit(b_t_full);
          if (!states_only) {
            if (c > 0 && !wait1(b_o_empty + 8 * ((c - 1) & 1), (uint32_t)(((c - 1) >> 1) & 1))) break;
            tc_fence_after();
#pragma unroll
            for (int k = 0; k < D1 / 16; ++k) mma_ts(tmem + C::kColO, tmem + C::kColX + k * 8, rows_desc + stage + row_step(k), idesc_rows, k > 0);
            tc_commit(b_x_empty);
            if (!wait1(b_p_full + 8 * (c & 1), (uint32_t)((c >> 1) & 1))) break;
            tc_fence_after();
            const uint64_t pd = rows_desc + (uint64_t)((C::kOffP + (c & 1) * (2 * kBlock)) >> 4);
#pragma unroll
            for (int k = 0; k < kChunk / 16; ++k) mma_ss(tmem + C::kColO + 64, ct + k * (2048 >> 4), pd + (kBlock >> 4) + k * (32 >> 4), idesc_p, k > 0);
#pragma unroll
            for (int k = 0; k < kChunk / 16; ++k) mma_ss(tmem + C::kColO + 64, ct + k * (2048 >> 4), pd + k * (32 >> 4), idesc_p, 1u);
            tc_commit(b_o_full + 8 * (c & 1));
          }
          tc_commit(b_empty + 8 * at);
          at = next;
          phase = next_phase;
        }
      }
    } else if (warp < kWarpLoad) {
      // ---- P ----
      if (!states_only && chunks > 0) {
        const int i = warp * 32 + lane;
        const uint32_t t_s = tmem + ((uint32_t)(warp * 32) << 16) + C::kColS;
        const int skip = 63 - i;
        const float* weight = table + C::kTabScore + (skip & 3) * C::kScorePitch + (skip & ~3);   // of column j at j
        for (int c = 0; c < chunks; ++c) {
          if (!wait(b_s_full + 8 * (c & 1), (uint32_t)((c >> 1) & 1))) break;
          tc_fence_after();
          if (c >= 2 && !wait(b_o_empty + 8 * (c & 1), (uint32_t)((c >> 1) & 1) ^ 1u)) break;
          const uint32_t row = base + C::kOffP + (c & 1) * (2 * kBlock) + i * 128;
          uint64_t to = 0;
          if constexpr (!BF16) {
            float most = 0.f, up, back;
#pragma unroll 1
            for (int j0 = 0; j0 < kChunk; j0 += 16) {
              uint32_t r[16];
              tmem_ld16(t_s + j0, r);
              tc_wait_ld();
#pragma unroll
              for (int j = 0; j < 16; j += 2) {
                const uint64_t w = *reinterpret_cast<const uint64_t*>(weight + j0 + j);
                const float2 f = unpack2(mul2(pack2(__uint_as_float(r[j]), __uint_as_float(r[j + 1])), w));
                most = fmax3(most, fabsf(f.x), fabsf(f.y));   // (NaN behind the row counts for nothing, an infinity there would be NaN)
              }
            }
            scale_of(most, up, back);
            to = pack2(up, up);
            table[C::kTabP + (c & 1) * 64 + i] = back;
          }
#pragma unroll 1
          for (int j0 = 0; j0 < kChunk; j0 += 16) {
            uint32_t r[16], v[8], left[8];
            tmem_ld16(t_s + j0, r);
            tc_wait_ld();
            uint64_t x[8], probe = 0;
#pragma unroll
            for (int j = 0; j < 16; j += 4) {
              const Pair2 w = lds_pairs(weight + j0 + j);
              x[j / 2] = mul2(pack2(__uint_as_float(r[j]), __uint_as_float(r[j + 1])), w.a);
              x[j / 2 + 1] = mul2(pack2(__uint_as_float(r[j + 2]), __uint_as_float(r[j + 3])), w.b);
              probe = fma2(x[j / 2], 0ull, fma2(x[j / 2 + 1], 0ull, probe));
            }
            const float2 odd_ones = unpack2(probe);
            const bool odd = __any_sync(0xffffffffu, odd_ones.x + odd_ones.y != 0.f);   // NaN: a score is not finite
            if (odd) {   // (behind the row it counts for nothing)
#pragma unroll
              for (int j = 0; j < 16; j += 2) {
                const float2 f = unpack2(x[j / 2]);
                const int at = j0 + j;
                x[j / 2] = pack2((reverse ? at < i : at > i) ? 0.f : f.x, (reverse ? at + 1 < i : at + 1 > i) ? 0.f : f.y);
              }
            }
#pragma unroll
            for (int k = 0; k < 8; ++k) {
              if constexpr (!BF16) x[k] = mul2(x[k], to);
              const float2 f = unpack2(x[k]);
              v[k] = pack2<BF16>(f.x, f.y);
              const float2 t = unpack16<BF16>(v[k]), e = unpack2(fma2(pack2(t.x, t.y), pack2(-1.f, -1.f), x[k]));
              left[k] = pack2<BF16>(e.x, e.y);
            }
            if (odd) {   // (of what is not finite nothing is left)
#pragma unroll
              for (int k = 0; k < 8; ++k) {
                const float2 e = unpack16<BF16>(left[k]);
                left[k] = pack2<BF16>(fabsf(e.x) < INFINITY ? e.x : 0.f, fabsf(e.y) < INFINITY ? e.y : 0.f);
              }
            }
            st_shared_v4(row + (((uint32_t)(j0 / 8) ^ (uint32_t)(i & 7)) << 4), v[0], v[1], v[2], v[3]);
            st_shared_v4(row + (((uint32_t)(j0 / 8 + 1) ^ (uint32_t)(i & 7)) << 4), v[4], v[5], v[6], v[7]);
            st_shared_v4(row + kBlock + (((uint32_t)(j0 / 8) ^ (uint32_t)(i & 7)) << 4), left[0], left[1], left[2], left[3]);
            st_shared_v4(row + kBlock + (((uint32_t)(j0 / 8 + 1) ^ (uint32_t)(i & 7)) << 4), left[4], left[5], left[6], left[7]);
          }
          tc_fence_before();
          arrive(b_s_empty);
          fence_proxy_async_smem();
          arrive(b_p_full + 8 * (c & 1));
        }
      }
    } else if (warp < kWarpOut) {
      // ---- C~ and the state ----
      const int tid = threadIdx.x - kWarpState * 32, quarter = warp & 3, half = (warp - kWarpState) >> 2;
      constexpr int kCols = D1 / 2;              // of a thread
      const int d2 = quarter * 32 + lane, d1 = half * kCols;
      const bool owner = d2 < D2;                // (with 64 columns, the lanes above hold nothing; whole warps)
      const uint32_t lanes = (uint32_t)(quarter * 32) << 16;
      const int64_t matrix = (int64_t)D1 * D2;
      const int lag = s.lag;
      const float key_scale = s.key_scale;   // in C~'s weights, for fp16 behind the product
      float t_scale = key_scale, t_scale_next = key_scale;   // fp16: of T's lane, for this chunk and the next
      float x[kCols];
#pragma unroll
      for (int i = 0; i < kCols; ++i) x[i] = 0.f;
      float* work = args.segments > 1 ? args.work + (((int64_t)which * p.batch * p.heads + item) * args.segments + seg) * matrix : nullptr;
      if (owner && !states_only) {
        const float* from = work ? work : (s.x_first && q.state >= 0 ? s.x_first + (q.state * p.heads + h) * matrix : nullptr);
        if (from) {
          const bool turned = !work && s.x_transposed;
          const int step = turned ? 1 : D2;
          from += turned ? d2 * D1 + d1 : d1 * D2 + d2;
#pragma unroll
          for (int i = 0; i < kCols; ++i) x[i] = from[i * step];
        }
      }
      // X^T of chunk c to tensor memory
      auto put_state = [&](int c) {
        if (owner) {
          float to = 1.f;
          if constexpr (!BF16) {
            float most = 0.f, back;
#pragma unroll
            for (int i = 0; i < kCols; ++i) most = fmaxf(most, fabsf(x[i]));
            float* most_of = table + C::kTabMax + (c & 1) * 256;   // (two in turn: the other warp has read c's before it takes part in c + 1)
            most_of[half * 128 + d2] = most;
            arrive(b_max + 8 * quarter);
            if (!wait(b_max + 8 * quarter, (uint32_t)(c & 1))) return false;
            most = fmaxf(most, most_of[(half ^ 1) * 128 + d2]);
            scale_of(most, to, back);
            if (half == 0) table[C::kTabX + (c & 3) * 128 + d2] = back;
          }
#pragma unroll
          for (int i0 = 0; i0 < kCols; i0 += 32) {
            uint32_t v[16];
#pragma unroll
            for (int i = 0; i < 32; i += 2) v[i / 2] = BF16 ? pack2<BF16>(x[i0 + i], x[i0 + i + 1]) : pack2<BF16>(x[i0 + i] * to, x[i0 + i + 1] * to);
            tmem_st16(tmem + lanes + C::kColX + (d1 + i0) / 2, v);
          }
          tc_wait_st();
        }
        tc_fence_before();
        arrive(b_x_full);
        return true;
      };
      // C~^T of chunk c to tensor memory: these lanes, rows 32 half .. + 31 of the chunk.  Two terms in two buffers in turn, so that they are formed while
      // the chunk before is multiplied, or three in one.
      const bool third = args.terms == 3;
      auto exponent = [&](int j, int n) { return reverse ? n - lag - (kChunk - 1 - j) : n - lag - j; };   // of tile row j, where it is one of n
      auto there = [&](int j, int n) { return reverse ? kChunk - 1 - j < n : j < n; };
      const int j_own = half * 32 + (lane & 3) * 2;   // + 8 i
      auto weigh = [&](int c) {
        const int n = rows - c * kChunk < kChunk ? rows - c * kChunk : kChunk;
        const uint32_t st = base + (uint32_t)((c % C::kStages) * C::kStageBytes) + C::kOffC;
        if (!wait(b_full + 8 * (c % C::kStages), (uint32_t)((c / C::kStages) & 1))) return false;
        if (owner) {
          uint32_t weights[2][4];   // of this thread's pairs of rows, as two terms
          if (BF16 && !third) {
            const uint16_t* terms = reinterpret_cast<const uint16_t*>(table + C::kTabW);
#pragma unroll
            for (int t = 0; t < 2; ++t) {
              uint4 w = *reinterpret_cast<const uint4*>(table + C::kTabPairs + t * 32 + half * 16 + (lane & 3) * 4);
              if (n < kChunk) w = end_weights(terms + t * 66, j_own, n, lag, reverse);
              weights[t][0] = w.x; weights[t][1] = w.y; weights[t][2] = w.z; weights[t][3] = w.w;
            }
          }
          const uint32_t to = tmem + lanes + C::kColC + (third ? 0 : (c & 1) * 64) + half * 16;
          // (matrices of a load: rows j .. j + 7 with columns d, d + 8; rows j + 8 .. j + 15 with the same)
          const int row = half * 32 + (lane & 7) + ((lane >> 4) << 3), col = quarter * 32 + (lane & 8);
          const uint32_t from = st + (col / 64) * kBlock + row * 128;
          // fp16: weights of row j and the next, zeros where there are none (a chunk of n rows ends with the last weight, and what is not there lies in the
          // zeros beside them)
          const float* row_weights = table + C::kTabRowsC + (reverse ? n : kChunk - n) + j_own;
          auto weights_of = [&](int i) { return pack2(row_weights[8 * i], row_weights[8 * i + 1]); };
          float up_all = 1.f;  // fp16: the power of two of column (lane & 3) * 8 + lane / 4
          if constexpr (!BF16) {
            float most[4] = {0.f, 0.f, 0.f, 0.f};   // of columns lane / 4, 8, 16 and 24 further
#pragma unroll
            for (int d = 0; d < 32; d += 16) {
              uint32_t v[8];
#pragma unroll
              for (int i = 0; i < 2; ++i) ldmatrix_x4_trans(from + i * (16 * 128) + (((uint32_t)(((col & 63) + d) >> 3) ^ (uint32_t)(row & 7)) << 4), v + 4 * i);
#pragma unroll
              for (int i = 0; i < 8; ++i) {
                const float2 c2 = unpack16<BF16>(v[i]), f = unpack2(mul2(pack2(c2.x, c2.y), weights_of(i / 2)));
                float& m = most[d / 8 + (i & 1)];
                m = fmax3(m, fabsf(f.x), fabsf(f.y));   // (NaN counts for nothing)
              }
            }
            // of four lanes and four columns, a column to each
            const bool odd = lane & 1, upper = lane & 2;
            const float m0 = fmaxf(odd ? most[1] : most[0], __shfl_xor_sync(0xffffffffu, odd ? most[0] : most[1], 1));
            const float m1 = fmaxf(odd ? most[3] : most[2], __shfl_xor_sync(0xffffffffu, odd ? most[2] : most[3], 1));
            float m = fmaxf(upper ? m1 : m0, __shfl_xor_sync(0xffffffffu, upper ? m0 : m1, 2));
            float* most_of = table + C::kTabC + (c & 1) * 256 + quarter * 32 + lane;   // of 32 rows; the other warp's 128 further (two in turn, as above)
            most_of[half * 128] = m;
            arrive(b_most + 8 * quarter);
            if (!wait(b_most + 8 * quarter, (uint32_t)(c & 1))) return false;
            float back;
            scale_of(fmaxf(m, most_of[(half ^ 1) * 128]), up_all, back);
            t_scale_next = key_scale * __shfl_sync(0xffffffffu, back, (lane & 7) * 4 + lane / 8);
          }
#pragma unroll 1
          for (int d = 0; d < 32; d += 16) {
            uint32_t v[8], a[8], e[8];
#pragma unroll
            for (int i = 0; i < 2; ++i) ldmatrix_x4_trans(from + i * (16 * 128) + (((uint32_t)(((col & 63) + d) >> 3) ^ (uint32_t)(row & 7)) << 4), v + 4 * i);
            if (n < kChunk) {   // (whatever stands in rows that are not there)
#pragma unroll
              for (int i = 0; i < 8; ++i) {
                const int j = j_own + 8 * (i / 2);
                v[i] &= (there(j, n) ? 0xffffu : 0u) | (there(j + 1, n) ? 0xffff0000u : 0u);
              }
            }
            if (BF16 && !third) {
              // c w as two terms by packed multiply-adds, with w = w0 + w1 of 8 bits each: c w0 has 16 bits, so that what its rounding leaves is exact.
              // (In fp32, with conversions there and back, it takes three times the instructions.)
#pragma unroll
              for (int i = 0; i < 8; ++i) {
                a[i] = bf16x2_mul(v[i], weights[0][i / 2]);
                e[i] = bf16x2_fma(v[i], weights[1][i / 2], bf16x2_fma(v[i], weights[0][i / 2], a[i] ^ 0x80008000u));
              }
            } else if constexpr (BF16) {
#pragma unroll
              for (int i = 0; i < 8; ++i) {
                const int j = j_own + 8 * (i / 2);
                float2 f = unpack16<BF16>(v[i]);
                f.x *= power[there(j, n) ? exponent(j, n) : 0] * key_scale;
                f.y *= power[there(j + 1, n) ? exponent(j + 1, n) : 0] * key_scale;
                a[i] = pack2<BF16>(f.x, f.y);
                float2 t = unpack16<BF16>(a[i]);
                f.x -= t.x;
                f.y -= t.y;
                e[i] = pack2<BF16>(f.x, f.y);
                t = unpack16<BF16>(e[i]);
                v[i] = pack2<BF16>(f.x - t.x, f.y - t.y);
              }
            } else {
              uint64_t up[2];
#pragma unroll
              for (int i = 0; i < 2; ++i) {
                const float f = __shfl_sync(0xffffffffu, up_all, (lane & ~3) + d / 8 + i);
                up[i] = pack2(f, f);
              }
              const uint64_t minus = pack2(-1.f, -1.f), kilo2 = pack2(2048.f, 2048.f);
#pragma unroll
              for (int i = 0; i < 8; ++i) {
                const float2 c2 = unpack16<BF16>(v[i]);
                const uint64_t f = mul2(pack2(c2.x, c2.y), mul2(weights_of(i / 2), up[i & 1]));   // (the weight first: it may be below what a product can hold)
                const float2 f2 = unpack2(f);
                a[i] = pack2<BF16>(f2.x, f2.y);
                const float2 t = unpack16<BF16>(a[i]), r = unpack2(mul2(fma2(pack2(t.x, t.y), minus, f), kilo2));
                e[i] = pack2<BF16>(r.x, r.y);
              }
            }
            tmem_st_16x128b_x4(to + ((uint32_t)d << 16), a);
            tmem_st_16x128b_x4(to + ((uint32_t)d << 16) + 32, e);
            if (third) tmem_st_16x128b_x4(to + ((uint32_t)d << 16) + 64, v);
          }
          tc_wait_st();
        }
        if (n < kChunk) {   // what multiplies a zero has to be finite: B's rows in the product with C~, C's in the one with P
          const int r0 = tid >> 3;   // this thread's rows are r0 and r0 + 32, of each block of 64 columns
          __syncwarp();
#pragma unroll
          for (int u = 0; u < 2 * (C::kN1 + C::kN2); ++u)   // (C lies behind B)
            if (!there(r0 + 32 * (u & 1), n)) st_shared_v4(st + C::kOffB - C::kOffC + u * (kBlock / 2) + tid * 16, 0, 0, 0, 0);
          fence_proxy_async_smem();
        }
        tc_fence_before();
        arrive(b_bt_full + 8 * (c & 1));
        return true;
      };
      // One place each for the next C~ and the state's step (their code is long): C~ in front of T, which is then being formed, with three terms behind
      // it.  c = -1: the first C~ and the first state.
      bool ok = chunks > 0;
      for (int c = -1; c < chunks && ok; ++c) {
#pragma unroll 1
        for (int turn = 0; turn < 2 && ok; ++turn) {
          if ((turn == 0) != third) {
            if (c + 1 < chunks) ok = weigh(c + 1);
            continue;
          }
          if (c >= 0) {
            const int n = rows - c * kChunk < kChunk ? rows - c * kChunk : kChunk;
            if (!(ok = wait(b_t_full, (uint32_t)(c & 1)))) break;
            tc_fence_after();
            if (owner) {
              const uint64_t keep = pack2(power[n], power[n]);
#pragma unroll
              for (int i0 = 0; i0 < kCols; i0 += 32) {
                uint32_t r[32];
                tmem_ld32(tmem + lanes + C::kColT + d1 + i0, r);
                tc_wait_ld();
#pragma unroll
                for (int i = 0; i < 32; i += 2) {
                  uint64_t t = pack2(__uint_as_float(r[i]), __uint_as_float(r[i + 1]));
                  if constexpr (!BF16) t = mul2(pack2(t_scale, t_scale), t);
                  const float2 f = unpack2(fma2(keep, pack2(x[i0 + i], x[i0 + i + 1]), t));
                  x[i0 + i] = f.x;
                  x[i0 + i + 1] = f.y;
                }
              }
            }
            tc_fence_before();
            arrive(b_t_empty);
          }
          t_scale = t_scale_next;
          if (!states_only && c + 1 < chunks) {
            if (c >= 0) {
              if (!(ok = wait(b_x_empty, (uint32_t)(c & 1)))) break;
              tc_fence_after();
            }
            ok = put_state(c + 1);
          }
        }
      }
      if (owner && !*abort_flag) {
        float* to = states_only ? work : args.segments == 1 && s.x_last && q.state >= 0 ? s.x_last + (q.state * p.heads + h) * matrix : nullptr;
        if (to) {
          const bool turned = !states_only && s.x_transposed;
          const int step = turned ? 1 : D2;
          to += turned ? d2 * D1 + d1 : d1 * D2 + d2;
#pragma unroll
          for (int i = 0; i < kCols; ++i) to[i * step] = x[i];
        }
      }
    } else if (!states_only) {
      // ---- output ----
      const int quarter = warp & 3, d2 = quarter * 32 + lane;
      const uint32_t lanes = (uint32_t)(quarter * 32) << 16;
      const bool owner = quarter * 32 < D2;
      const int64_t pitch = s.ys[2];
      const bool y_f32 = s.y_f32 != 0;
      const int group = lane >> 2, pair = (lane & 3) * 2;
      const uint32_t mine = base + C::kOffY + quarter * kYBytes;
      // 16 bytes of a row of this warp's 64 rows of 32 columns, swizzled as the stores out of it expect
      auto piece = [&](int row, int at) { return mine + (uint32_t)(row * 64) + (((uint32_t)at ^ ((uint32_t)(row >> 1) & 3u)) << 4); };
      const bool leader = elect_one();
      for (int c = 0; c < chunks; ++c) {
        const int n = rows - c * kChunk < kChunk ? rows - c * kChunk : kChunk;
        const int low = reverse ? kChunk - n : 0, high = reverse ? kChunk : n;   // the tile's rows
        const int token = token_of(c);
        if (!wait(b_o_full + 8 * (c & 1), (uint32_t)((c >> 1) & 1))) break;
        tc_fence_after();
        auto value = [&](int r, float state, float part) {   // of a lane's own column
          const float w = table[C::kTabRow + r];
          return BF16 ? fmaf(w, state, part) : fmaf(table[C::kTabP + (c & 1) * 64 + r], part, w * table[C::kTabX + (c & 3) * 128 + d2] * state);
        };
        if (owner) {
          if (leader) bulk_wait_read0();   // (the last chunk's stores have read its rows)
          __syncwarp();
          uint64_t probe = 0;   // NaN as soon as a value of the row part is not finite
          if (y_f32) {          // partial sums: a column to a lane
            float* at = static_cast<float*>(s.y) + y0 + (int64_t)token * pitch + d2;
#pragma unroll 1
            for (int r0 = 0; r0 < kChunk; r0 += 8) {
              uint32_t u[8], v[8];
              tmem_ld8(tmem + lanes + C::kColO + r0, u);
              tmem_ld8(tmem + lanes + C::kColO + 64 + r0, v);
              tc_wait_ld();
#pragma unroll
              for (int r = 0; r < 8; ++r) {
                const float f = value(r0 + r, __uint_as_float(u[r]), __uint_as_float(v[r]));
                probe = fma2(pack2(__uint_as_float(v[r]), 0.f), 0ull, probe);
                if (r0 + r >= low && r0 + r < high) *at = f;
                at += pitch;
              }
            }
          } else {
            // 16 lanes at a time, a thread with two rows of the chunk in eight groups and two lanes: pairs along the rows, transposed on the way to shared
            // memory
#pragma unroll 1
            for (int part_of = 0; part_of < 4; ++part_of) {
              const int up = (part_of & 1) * 16, half = part_of >> 1;
              const uint32_t t_o = tmem + lanes + ((uint32_t)up << 16) + C::kColO + half * 32;
              uint32_t u[16], v[16], m[8];
              tmem_ld_16x256b_x4(t_o, u);
              tmem_ld_16x256b_x4(t_o + 64, v);
              uint64_t xs[2] = {0, 0};
              if constexpr (!BF16) {
                const float* of = table + C::kTabX + (c & 3) * 128 + quarter * 32 + up + group;
                xs[0] = pack2(of[0], of[0]);
                xs[1] = pack2(of[8], of[8]);
              }
              const uint64_t* row_w = reinterpret_cast<const uint64_t*>(table + C::kTabRow + half * 32 + pair);   // of rows 8 g + pair and the next, at 4 g
              const uint64_t* row_p = reinterpret_cast<const uint64_t*>(table + C::kTabP + (c & 1) * 64 + half * 32 + pair);
              tc_wait_ld();
#pragma unroll
              for (int g = 0; g < 4; ++g) {
                const uint64_t w = row_w[4 * g];
                uint64_t ps = 0;
                if constexpr (!BF16) ps = row_p[4 * g];
#pragma unroll
                for (int k = 0; k < 2; ++k) {   // lanes group and group + 8
                  const uint64_t state = pack2(__uint_as_float(u[4 * g + 2 * k]), __uint_as_float(u[4 * g + 2 * k + 1]));
                  const uint64_t part = pack2(__uint_as_float(v[4 * g + 2 * k]), __uint_as_float(v[4 * g + 2 * k + 1]));
                  probe = fma2(part, 0ull, probe);   // (of rows that are not there too: at worst the sums below are formed again for nothing)
                  const float2 f = unpack2(BF16 ? fma2(w, state, part) : fma2(ps, part, mul2(mul2(w, xs[k]), state)));
                  m[2 * g + k] = pack2<BF16>(f.x, f.y);
                }
              }
#pragma unroll
              for (int g = 0; g < 4; g += 2)   // matrices: rows 8 g .. of columns up .. and up + 8 .., rows 8 (g + 1) .. of the same
                stmatrix_x4_trans(piece((half * 4 + g + (lane >> 4)) * 8 + (lane & 7), up / 8 + ((lane >> 3) & 1)), m + 2 * g);
            }
          }
          const float2 two = unpack2(probe);
          if (__any_sync(0xffffffffu, two.x + two.y != 0.f)) {
            // columns that came out not finite are summed again, a lane to each, over what a row may see (the tile of C may have been given
            // back: its column comes from memory once more)
            __syncwarp();
            const uint32_t pt = base + C::kOffP + (c & 1) * (2 * kBlock);
            const uint16_t* ct = static_cast<const uint16_t*>(s.c) + (p.starts ? 0 : b * s.cs[0]) + (h / s.c_group) * s.cs[1] + (q.row0 + token) * s.cs[2] + d2;
#pragma unroll 1
            for (int r = low; r < high; ++r) {
              uint32_t u, v;
              asm volatile("tcgen05.ld.sync.aligned.32x32b.x1.b32 {%0}, [%1];" : "=r"(u) : "r"(tmem + lanes + C::kColO + r) : "memory");
              asm volatile("tcgen05.ld.sync.aligned.32x32b.x1.b32 {%0}, [%1];" : "=r"(v) : "r"(tmem + lanes + C::kColO + 64 + r) : "memory");
              tc_wait_ld();
              float part = __uint_as_float(v);
              if (!(fabsf(part) < INFINITY)) {
                part = 0.f;
                for (int j = reverse ? r : low; j < (reverse ? high : r + 1); ++j) {
                  const uint32_t at = pt + r * 128 + (((uint32_t)(j >> 3) ^ (uint32_t)(r & 7)) << 4) + (j & 7) * 2;
                  part = fmaf(lds16<BF16>(at) + lds16<BF16>(at + kBlock), unpack16<BF16>(ct[j * s.cs[2]]).x, part);
                }
              }
              const float f = value(r, __uint_as_float(u), part);
              if (y_f32) static_cast<float*>(s.y)[y0 + (int64_t)(token + r) * pitch + d2] = f;
              else sts16(piece(r, lane >> 3) + (lane & 7) * 2, pack2<BF16>(f, 0.f));
            }
          }
        }
        tc_fence_before();
        arrive(b_o_empty + 8 * (c & 1));
        if (owner && !y_f32) {
          if (n == kChunk) {
            fence_proxy_async_smem();
            __syncwarp();
            if (leader) {
              tma_store_4d(&maps.y[which], mine, quarter * 32, (int)q.row0 + token, h, p.starts ? 0 : b);
              bulk_commit();
            }
          } else {   // not the rows beside the sequence
            __syncwarp();
            for (int e = lane; e < n * 4; e += 32) {
              const int r = low + e / 4;
              const uint4 f = lds128(piece(r, e & 3));
              *reinterpret_cast<uint4*>(static_cast<uint16_t*>(s.y) + y0 + (int64_t)(token + r) * pitch + quarter * 32 + (e & 3) * 8) = f;
            }
          }
        }
      }
      if (leader) bulk_wait_all();   // shared memory outlives the stores that read it
      __syncwarp();
    }

    // ---- teardown ----
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    if (*abort_flag) {
      if (threadIdx.x == 0) {
        abort_grace();
        atomicAdd(&g_linear_gave_up, 1u);
      }
      __syncthreads();
    }
    if (warp == kWarpMma) {
      tc_fence_after();
      tmem_dealloc(tmem, 512);
    }
  }
  // rows without a state, and rows of padding
  if (states_only || (!q.bad && p.starts)) return;
  const int64_t end = p.starts ? q.n : p.seq_len;
  const int64_t from = q.bad || q.n < t0 ? t0 : q.n, upto = end < t0 + args.seg_len ? end : t0 + args.seg_len;
  for (int64_t e = from * D2 + threadIdx.x; e < upto * D2; e += kThreads) {
    const int64_t r = e / D2;
    const float f = r < q.n ? __int_as_float(0x7fffffff) : 0.f;
    const int64_t at = y0 + r * s.ys[2] + (e - r * D2);
    if (s.y_f32) static_cast<float*>(s.y)[at] = f;
    else if constexpr (BF16) static_cast<__nv_bfloat16*>(s.y)[at] = from_float<__nv_bfloat16>(f);
    else static_cast<__half*>(s.y)[at] = from_float<__half>(f);
  }
}

template <int D1, int D2, bool BF16>
cudaError_t launch_t(const Maps& maps, Args& args, cudaStream_t stream, int* launches) {
  using C = Cfg<D1, D2>;
  auto kern = scan_sm100_kernel<D1, D2, BF16>;
  cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmem);
  if (e != cudaSuccess) return e;
  const unsigned items = (unsigned)args.p.batch * args.p.heads, grid = items * (unsigned)args.count * (unsigned)args.segments;
  if (args.segments > 1) {
    args.states_only = 1;
    kern<<<grid, kThreads, C::kSmem, stream>>>(maps, args);
    args.states_only = 0;
    e = cudaGetLastError();
    if (e != cudaSuccess) return e;
    e = launch_join(args.p, Segments{args.segments, args.seg_len, 0, args.work}, args.first, args.count, D1 * D2, stream);
    if (e != cudaSuccess) return e;
    *launches += 2;
  }
  kern<<<grid, kThreads, C::kSmem, stream>>>(maps, args);
  ++*launches;
  return cudaGetLastError();
}

template <bool BF16>
cudaError_t launch_sizes(const Maps& maps, Args& args, cudaStream_t stream, int* launches) {
  const Scan& s = args.p.scan[args.first];
  if (s.d1 == 128) return s.d2 == 128 ? launch_t<128, 128, BF16>(maps, args, stream, launches) : launch_t<128, 64, BF16>(maps, args, stream, launches);
  return s.d2 == 128 ? launch_t<64, 128, BF16>(maps, args, stream, launches) : launch_t<64, 64, BF16>(maps, args, stream, launches);
}

// How many segments the sequences are cut into: as many as bring work to all SMs, where that pays.  A row goes through both launches then, the first at 0.7
// of the second's cost, and the two launches more take the time of ten chunks.  One sequence and 16 heads of 64 in fp16, by host and device: 2048 rows 76 us
// uncut, 37 us in 9 segments; 1024 rows 41 and 30 us; 768 rows 33 us uncut, which is where the rule leaves off.  8192 rows of 16 heads of 128 in bf16: 215 and 84 us.
int segments_of(const Params& p, int num_sms) {
  const int64_t items = (int64_t)p.batch * p.heads * p.scans, chunks = (p.seq_len + kChunk - 1) / kChunk;
  int64_t n = num_sms / items;
  n = n < chunks ? n : chunks;
  n = n < kMaxSegments ? n : kMaxSegments;
  return n >= 2 && chunks * (10 * n - 17) >= 100 * n ? (int)n : 1;
}

// Whether sequences of unequal lengths are taken from the longest to the shortest: a long one at the end of a batch would run alone.  To find its sequence
// takes a CTA 0.2 us, so it is done where the longest may take a quarter of the call: seq_len * SMs against rows * heads * scans.  (32 heads of 128 in bf16,
// as they lie / longest first, us, with P in one term: 7 prompts of 1 to 8192, the shortest first, 221 / 206, with states 362 / 335, gradients 798 / 692; 32 of up to 1023
// 155 / 147; 63 of up to 63 and one of 2000 at the end 146 / 123; 16 of 512 each 74.8 / 76.8.)
bool by_length(const Params& p, int num_sms) {
  if ((!p.starts && !p.lengths) || p.batch < 2 || p.batch > kMaxRanked) return false;
  const int64_t ctas = (int64_t)p.batch * p.heads * p.scans, rows = p.starts ? p.tokens : p.batch * p.seq_len;
  return ctas > num_sms && 4 * p.seq_len * num_sms >= rows * p.heads * p.scans;
}

}  // namespace

uint32_t* sm100_gave_up() {
  void* addr = nullptr;
  if (cudaGetSymbolAddress(&addr, g_linear_gave_up) != cudaSuccess) {
    cudaGetLastError();
    return nullptr;
  }
  return static_cast<uint32_t*>(addr);
}

bool scan_sm100_supported(const Params& p) {
  if (p.dtype == AIDN_F32 || (p.starts && p.tokens == 0)) return false;
  if ((int64_t)p.batch * p.heads > (1 << 24)) return false;
  const int64_t rows = p.starts ? p.tokens : p.seq_len;
  for (int i = 0; i < p.scans; ++i) {
    const Scan& s = p.scan[i];
    if ((s.d1 != 64 && s.d1 != 128) || (s.d2 != 64 && s.d2 != 128)) return false;
    const void* ptr[3] = {s.a, s.b, s.c};
    const int64_t* stride[3] = {s.as, s.bs, s.cs};
    const int group[3] = {s.a_group, s.b_group, s.c_group};
    for (int t = 0; t < 3; ++t) {
      if ((uintptr_t)ptr[t] % 16 != 0) return false;
      const int64_t extent[3] = {p.starts ? 1 : p.batch, p.heads / group[t], rows};
      for (int d = 0; d < 3; ++d)
        if (extent[d] > 1 && (stride[t][d] <= 0 || stride[t][d] % 8 != 0 || stride[t][d] >= (1ll << 38))) return false;
    }
    if (!s.y_f32) {
      if ((uintptr_t)s.y % 16 != 0) return false;
      const int64_t extent[3] = {p.starts ? 1 : p.batch, p.heads, rows};
      for (int d = 0; d < 3; ++d)
        if (extent[d] > 1 && (s.ys[d] <= 0 || s.ys[d] % 8 != 0 || s.ys[d] >= (1ll << 38))) return false;
    }
  }
  return true;
}

int64_t scan_sm100_bytes(const Params& p, int num_sms) {
  if (p.dtype == AIDN_F32 || (p.scan[0].d1 != 64 && p.scan[0].d1 != 128) || (p.scan[0].d2 != 64 && p.scan[0].d2 != 128)) return 0;
  const int n = segments_of(p, num_sms);
  return n == 1 ? 0 : (int64_t)p.scans * p.batch * p.heads * n * p.scan[0].d1 * p.scan[0].d2 * 4;
}

cudaError_t launch_scan_sm100(const Params& p, int num_sms, float* work, int64_t work_bytes, bool expire, cudaStream_t stream, int* launches) {
  cudaError_t e = tmap::resolve_encode();
  if (e != cudaSuccess) return e;
  const bool bf16 = p.dtype == AIDN_BF16;
  const CUtensorMapDataType dt = bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  const int64_t rows = p.starts ? p.tokens : p.seq_len, batch = p.starts ? 1 : p.batch;
  Maps maps;
  Args args;
  args.p = p;
  // one map for each tensor (of the three scans' nine operands, four are different)
  int known = 0;
  struct Key {
    const void* ptr;
    int64_t stride[3];
    int size, group;
  } made[4];
  auto map_of = [&](const void* ptr, const int64_t* stride, int size, int group) {
    for (int i = 0; i < known; ++i)
      if (made[i].ptr == ptr && made[i].size == size && made[i].group == group && made[i].stride[0] == stride[0] && made[i].stride[1] == stride[1] &&
          made[i].stride[2] == stride[2])
        return i;
    if (known == 4) return -1;
    int64_t st[3] = {stride[0], stride[1], rows > 1 ? stride[2] : size};
    if (!tmap::encode_bhsd(&maps.t[known], dt, 2, CU_TENSOR_MAP_SWIZZLE_128B, ptr, size, rows, p.heads / group, batch, st, 64, kChunk)) return -1;
    made[known] = {ptr, {stride[0], stride[1], stride[2]}, size, group};
    return known++;
  };
  for (int i = 0; i < p.scans; ++i) {
    const Scan& s = p.scan[i];
    args.ia[i] = map_of(s.a, s.as, s.d1, s.a_group);
    args.ib[i] = map_of(s.b, s.bs, s.d1, s.b_group);
    args.ic[i] = map_of(s.c, s.cs, s.d2, s.c_group);
    if (args.ia[i] < 0 || args.ib[i] < 0 || args.ic[i] < 0) return cudaErrorInvalidValue;
    const int64_t st[3] = {s.ys[0], s.ys[1], rows > 1 ? s.ys[2] : s.d2};
    if (!s.y_f32 && !tmap::encode_bhsd(&maps.y[i], dt, 2, CU_TENSOR_MAP_SWIZZLE_64B, s.y, s.d2, rows, p.heads, batch, st, 32, kChunk)) return cudaErrorInvalidValue;
  }
  args.segments = work && work_bytes >= scan_sm100_bytes(p, num_sms) ? segments_of(p, num_sms) : 1;
  const int64_t per = (p.seq_len + args.segments - 1) / args.segments;
  args.seg_len = (int)((per + kChunk - 1) / kChunk * kChunk < 0x7fffffc0ll ? (per + kChunk - 1) / kChunk * kChunk : 0x7fffffc0ll);
  args.states_only = 0;
  args.ranked = args.segments == 1 && by_length(p, num_sms);
  // two bf16 terms leave 2^-17 of a key: enough for outputs of 8 bits, not for states that go out in 32
  args.terms = 2;
  if (bf16)
    for (int i = 0; i < p.scans; ++i)
      if (p.scan[i].x_last) args.terms = 3;
  args.work = work;
  args.wait_ns = expire ? 20000000ull : kWaitBudgetNs;
  args.withhold = expire ? 1 : 0;
  // scans of the same sizes share a launch
  for (args.first = 0; args.first < p.scans && e == cudaSuccess; args.first += args.count) {
    args.count = 1;
    while (args.first + args.count < p.scans && p.scan[args.first + args.count].d1 == p.scan[args.first].d1 &&
           p.scan[args.first + args.count].d2 == p.scan[args.first].d2)
      ++args.count;
    e = bf16 ? launch_sizes<true>(maps, args, stream, launches) : launch_sizes<false>(maps, args, stream, launches);
  }
  return e;
}

}  // namespace lin
}  // namespace aidn
