// Rotary positions: the pairs of the first rotary_dim elements of each head, turned by position * frequency.
//     (a, b) -> amplitude * (a cos - b sin, a sin + b cos);  the gradient is the same with the angle negated.
//
// Bound by memory: every element once in and once out.  The angles of a token serve all of its heads, so a CTA takes a few tokens
// with all heads, forms their cosines and sines once in shared memory and then streams.  An angle is formed in turns as
// two numbers of 64 bits each, the second what the first one's rounding leaves: the nearest whole turn is taken off the first, and what is left (at most
// half a turn) has an error of 2^-25 turns in 32 bits for every position that 64 bits hold as they are, up to 2^53.  (One number of 64 bits would be off by
// position * frequency * 2^-55 turns, a product in 32 bits by the position times 2^-24.)
//
// Two units of 32 bytes in flight to a thread and six CTAs an SM: 8192 tokens of 40 heads of 128 (bf16, out of a packed projection) 35.4 us, 4.7 TB/s
// (34.9 with angles of one number); four units and three CTAs 38.1 us, two units and twice the tokens to a CTA 36.2 us.
#include "linear.cuh"

namespace aidn {
namespace lin {
namespace {

constexpr int kThreads = 256;
constexpr int kBatch = 2;          // units of a thread whose loads are in flight together
constexpr int kMaxTokens = 16;     // of a CTA
constexpr double kPerRadian = 0.15915494309189535, kPerRadianLeft = -9.839338337591243e-18;   // 1 / 2 pi, and what its rounding leaves

template <int BYTES>
struct Raw;
template <> struct Raw<16> { using T = uint4; };
template <> struct Raw<8> { using T = uint2; };
template <> struct Raw<4> { using T = uint32_t; };
template <> struct Raw<2> { using T = uint16_t; };

// A unit is NP pairs: 2 * NP elements, for pairs (2i, 2i+1) side by side, else NP at i and NP at i + rotary_dim / 2.  Behind rotary_dim
// it is 2 * NP elements that stay as they are.
template <typename T, int NP, bool HALVES>
__global__ void __launch_bounds__(kThreads, 6) rotary_kernel(const Rotary p, const int tokens_per_cta, const bool copy_rest) {
  using R = typename Raw<NP * (int)sizeof(T)>::T;
  __shared__ float2 table[kMaxTokens * 128];
  const int half = p.rotary_dim / 2;
  const int64_t t0 = (int64_t)blockIdx.x * tokens_per_cta;
  const int tokens = (int)(p.tokens - t0 < tokens_per_cta ? p.tokens - t0 : tokens_per_cta);
  const int turned = half / NP;                                        // units of a head that are turned
  const int units = copy_rest ? p.head_dim / (2 * NP) : turned;
  const int heads = p.heads[0] + p.heads[1];
  const int per_token = heads * units, total = tokens * per_token;

  const T* src[kBatch];
  T* dst[kBatch];
  R lo[kBatch], hi[kBatch];
  int angle[kBatch];
  auto load = [&](int first) {
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      const int e = first + i * kThreads;
      if (e >= total) break;
      const int t = e / per_token, r = e - t * per_token;
      const int hh = r / units, u = r - hh * units;
      const int which = hh >= p.heads[0] ? 1 : 0;
      const int h = hh - (which ? p.heads[0] : 0);
      src[i] = static_cast<const T*>(p.x[which]) + (t0 + t) * p.xs[which][0] + h * p.xs[which][1];
      dst[i] = static_cast<T*>(p.y[which]) + (t0 + t) * p.ys[which][0] + h * p.ys[which][1];
      angle[i] = u < turned ? t * half + u * NP : -1;
      const int at = HALVES && u < turned ? u * NP : 2 * u * NP;
      const int step = HALVES && u < turned ? half : NP;
      src[i] += at;
      dst[i] += at;
      lo[i] = *reinterpret_cast<const R*>(src[i]);
      hi[i] = *reinterpret_cast<const R*>(src[i] + step);
    }
  };
  load(threadIdx.x);
  for (int e = threadIdx.x; e < tokens * half; e += kThreads) {
    const int t = e / half, i = e - t * half;
    int64_t pos;
    if (!p.positions) pos = p.start + (t0 + t) % p.seq_len;
    else if (p.wide_positions) pos = static_cast<const int64_t*>(p.positions)[t0 + t];
    else pos = static_cast<const int32_t*>(p.positions)[t0 + t];
    // turns a position, f / 2 pi, with 1 / 2 pi in two numbers; then turns, and what is left of them
    const double f = p.frequencies[i], x = (double)pos;
    const double per = f * kPerRadian, per_left = fma(f, kPerRadian, -per) + f * kPerRadianLeft;
    const double turns = x * per, turns_left = fma(x, per, -turns) + x * per_left;
    float s, c;
    sincospif(2.f * (float)((turns - rint(turns)) + turns_left), &s, &c);
    table[e] = make_float2(c * p.amplitude, s * p.amplitude * p.sign);
  }
  __syncthreads();
  for (int first = threadIdx.x; first < total; first += kThreads * kBatch) {
    if (first != threadIdx.x) load(first);
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      if (first + i * kThreads >= total) break;
      const int step = HALVES && angle[i] >= 0 ? half : NP;
      if (angle[i] >= 0) {
        alignas(16) T e[2 * NP];
        *reinterpret_cast<R*>(e) = lo[i];
        *reinterpret_cast<R*>(e + NP) = hi[i];
#pragma unroll
        for (int j = 0; j < NP; ++j) {
          const float2 cs = table[angle[i] + j];
          const int at = HALVES ? j : 2 * j, bt = HALVES ? NP + j : 2 * j + 1;
          const float x = to_float(e[at]), y = to_float(e[bt]);
          e[at] = from_float<T>(x * cs.x - y * cs.y);
          e[bt] = from_float<T>(x * cs.y + y * cs.x);
        }
        lo[i] = *reinterpret_cast<R*>(e);
        hi[i] = *reinterpret_cast<R*>(e + NP);
      }
      *reinterpret_cast<R*>(dst[i]) = lo[i];
      *reinterpret_cast<R*>(dst[i] + step) = hi[i];
    }
  }
}

template <typename T, int NP>
cudaError_t launch_t(const Rotary& p, bool copy_rest, cudaStream_t stream) {
  const int units = copy_rest ? p.head_dim / (2 * NP) : p.rotary_dim / (2 * NP);
  const int64_t per_token = (int64_t)(p.heads[0] + p.heads[1]) * units;
  // about four units to a thread
  int64_t tokens = kThreads * 4 / (per_token > 0 ? per_token : 1);
  if (tokens < 1) tokens = 1;
  if (tokens > kMaxTokens) tokens = kMaxTokens;
  const int64_t grid = (p.tokens + tokens - 1) / tokens;
  if (grid > 0x7fffffff) return cudaErrorInvalidConfiguration;
  auto kern = p.halves ? rotary_kernel<T, NP, true> : rotary_kernel<T, NP, false>;
  kern<<<(unsigned)grid, kThreads, 0, stream>>>(p, (int)tokens, copy_rest);
  return cudaGetLastError();
}

}  // namespace

cudaError_t launch_rotary(const Rotary& p, cudaStream_t stream) {
  const int esz = p.dtype == AIDN_F32 ? 4 : 2;
  bool in_place = true;
  int np = p.dtype == AIDN_F32 ? 4 : 8;
  auto fits = [&](int n) {
    if (p.rotary_dim % (2 * n) != 0 || p.head_dim % (2 * n) != 0) return false;
    const int bytes = n * esz;
    for (int i = 0; i < 2; ++i) {
      if (p.heads[i] == 0) continue;
      if ((uintptr_t)p.x[i] % bytes != 0 || (uintptr_t)p.y[i] % bytes != 0) return false;
      for (int j = 0; j < 2; ++j)
        if ((p.xs[i][j] * esz) % bytes != 0 || (p.ys[i][j] * esz) % bytes != 0) return false;
    }
    return true;
  };
  for (int i = 0; i < 2; ++i)
    if (p.heads[i] > 0 && p.x[i] != p.y[i]) in_place = false;
  while (np > 1 && !fits(np)) np = np == 8 ? 4 : 1;   // (the widest vectors that sizes and addresses allow)
  const bool copy = !in_place;
  if (p.dtype == AIDN_F32) return np == 4 ? launch_t<float, 4>(p, copy, stream) : launch_t<float, 1>(p, copy, stream);
  if (p.dtype == AIDN_F16)
    return np == 8 ? launch_t<__half, 8>(p, copy, stream) : np == 4 ? launch_t<__half, 4>(p, copy, stream) : launch_t<__half, 1>(p, copy, stream);
  return np == 8 ? launch_t<__nv_bfloat16, 8>(p, copy, stream) : np == 4 ? launch_t<__nv_bfloat16, 4>(p, copy, stream) : launch_t<__nv_bfloat16, 1>(p, copy, stream);
}

}  // namespace lin
}  // namespace aidn
