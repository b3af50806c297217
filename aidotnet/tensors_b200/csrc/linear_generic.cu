// The scan of linear.cuh on FFMA: any type, any head sizes.  A CTA takes some columns of c (and of the state) for one sequence and head, or one segment
// of them, and walks its rows in chunks, the state in shared memory in fp32; the chunk's products a . b are formed again for every slice of
// columns.  What bounds it is the reads of shared memory that feed the multiply-adds: all products are tiles of 2 x 2 (a . b), 2 x N (outputs) or
// 4 x N (state; N = 2 or 4 for 32 or 64 columns) to a thread, read by fours along the sizes.  Few sequences and heads are cut into segments as on the tensor cores.
#include "linear.cuh"

namespace aidn {
namespace lin {
namespace {

constexpr int kThreads = 256;
constexpr int kChunk = 32;
__host__ __device__ constexpr int pitch_of(int d) { return d + 4; }   // (rows begin in different banks, fours stay aligned)
constexpr int kPitchP = kChunk + 4;
// shared memory in floats: A, B [chunk][d1], C and weighted C [chunk][width], X [d1][width], P [chunk][chunk], powers
inline size_t smem_bytes(int d1, int width) {
  return sizeof(float) * (2 * kChunk * pitch_of(d1) + (2 * kChunk + (size_t)d1) * (width + 4) + kChunk * kPitchP + kChunk + 4);
}

__host__ __device__ constexpr int ctas_of(int width) { return width == 64 ? 2 : 3; }   // CTAs that an SM's registers hold

template <typename T>
__device__ __forceinline__ void put(const Scan& s, int64_t at, float x) {
  if (s.y_f32) static_cast<float*>(s.y)[at] = x;
  else static_cast<T*>(s.y)[at] = from_float<T>(x);
}

__device__ __forceinline__ float dot4(float4 a, float4 b, float c) { return fmaf(a.w, b.w, fmaf(a.z, b.z, fmaf(a.y, b.y, fmaf(a.x, b.x, c)))); }

// N floats side by side.
template <int N>
__device__ __forceinline__ void load_n(const float* from, float (&to)[N]) {
  if constexpr (N == 4) {
    const float4 v = *reinterpret_cast<const float4*>(from);
    to[0] = v.x; to[1] = v.y; to[2] = v.z; to[3] = v.w;
  } else {
    const float2 v = *reinterpret_cast<const float2*>(from);
    to[0] = v.x; to[1] = v.y;
  }
}

template <typename T, int kWidth>
__global__ void __launch_bounds__(kThreads, ctas_of(kWidth)) scan_kernel(const __grid_constant__ Params p, const Segments g) {
  constexpr int kPitchW = kWidth + 4, N = kWidth / 16;   // N: columns of a thread
  extern __shared__ float4 smem4[];
  float* smem = reinterpret_cast<float*>(smem4);
  const Scan& s = p.scan[blockIdx.y];
  const int slices = (s.d2 + kWidth - 1) / kWidth;
  if (blockIdx.x >= (int64_t)p.batch * p.heads * g.count * slices) return;   // (the scans of one launch may have different widths)
  const int slice = (int)(blockIdx.x % (unsigned)slices), w0 = slice * kWidth;
  const int unit = (int)(blockIdx.x / (unsigned)slices), seg = unit % g.count, item = unit / g.count;
  const int b = item / p.heads, h = item - b * p.heads;
  const int width = s.d2 - w0 < kWidth ? s.d2 - w0 : kWidth;
  const int d1 = s.d1, pitch = pitch_of(d1), tid = threadIdx.x;
  float* A = smem;
  float* B = A + kChunk * pitch;
  float* C = B + kChunk * pitch;
  float* Cw = C + kChunk * kPitchW;
  float* X = Cw + kChunk * kPitchW;
  float* P = X + d1 * kPitchW;
  float* power = P + kChunk * kPitchP;   // lam^0 .. lam^kChunk

  const Sequence q = sequence_of(p, b);
  const int64_t from = (int64_t)seg * g.rows;   // this segment's rows, counted as they are taken
  const int64_t rows = q.bad || q.n <= from ? 0 : (q.n - from < g.rows ? q.n - from : g.rows);
  const T* a = static_cast<const T*>(s.a) + (p.starts ? 0 : b * s.as[0]) + (h / s.a_group) * s.as[1] + q.row0 * s.as[2];
  const T* bb = static_cast<const T*>(s.b) + (p.starts ? 0 : b * s.bs[0]) + (h / s.b_group) * s.bs[1] + q.row0 * s.bs[2];
  const T* c = static_cast<const T*>(s.c) + (p.starts ? 0 : b * s.cs[0]) + (h / s.c_group) * s.cs[1] + q.row0 * s.cs[2] + w0;
  const int64_t y0 = (p.starts ? 0 : b * s.ys[0]) + h * s.ys[1] + q.row0 * s.ys[2] + w0;
  const bool hand_on = g.count == 1 && s.x_last && q.state >= 0 && !q.bad;   // (a sequence without rows leaves its state too)
  if (rows > 0 || hand_on) {
    const double decay = log_decay(p.decay, h);
    if (tid <= kChunk) power[tid] = decay_power(decay, tid);
    const int64_t matrix = (int64_t)d1 * s.d2;
    const int64_t state = (q.state * p.heads + h) * matrix;
    float* work = g.count > 1 ? g.work + (((int64_t)blockIdx.y * p.batch * p.heads + item) * g.count + seg) * matrix : nullptr;
    for (int e = tid; e < d1 * kWidth; e += kThreads) {
      const int r = e / kWidth, w = e - r * kWidth;
      float x = 0.f;
      if (w < width && !g.states_only) {
        if (work) x = work[(int64_t)r * s.d2 + w0 + w];
        else if (s.x_first && q.state >= 0) x = s.x_first[state + (s.x_transposed ? (int64_t)(w0 + w) * d1 + r : (int64_t)r * s.d2 + w0 + w)];
      }
      X[r * kPitchW + w] = x;
    }
    for (int64_t t0 = 0; t0 < rows; t0 += kChunk) {
      const int n = (int)(rows - t0 < kChunk ? rows - t0 : kChunk);
      auto row = [&](int i) { return s.reverse ? q.n - 1 - (from + t0 + i) : from + t0 + i; };
      __syncthreads();
      for (int e = tid; e < kChunk * d1; e += kThreads) {
        const int i = e / d1, d = e - i * d1;
        if (!g.states_only) A[i * pitch + d] = i < n ? to_float(a[row(i) * s.as[2] + d]) : 0.f;
        B[i * pitch + d] = i < n ? to_float(bb[row(i) * s.bs[2] + d]) : 0.f;
      }
      for (int e = tid; e < kChunk * kWidth; e += kThreads) {
        const int i = e / kWidth, w = e - i * kWidth;
        const float x = i < n && w < width ? to_float(c[row(i) * s.cs[2] + w]) : 0.f;
        C[i * kPitchW + w] = x;
        Cw[i * kPitchW + w] = i < n ? x * (power[n - s.lag - i] * s.key_scale) : 0.f;
      }
      __syncthreads();
      // this thread's rows and columns of the 32 x 32 products: i, i + 16 and j, j + 16
      const int i = tid / 16, j = tid % 16;
      if (!g.states_only) {
        float acc[2][2] = {};
        for (int d = 0; d < d1; d += 4) {
          const float4 a0 = *reinterpret_cast<const float4*>(A + i * pitch + d), a1 = *reinterpret_cast<const float4*>(A + (i + 16) * pitch + d);
          const float4 b0 = *reinterpret_cast<const float4*>(B + j * pitch + d), b1 = *reinterpret_cast<const float4*>(B + (j + 16) * pitch + d);
          acc[0][0] = dot4(a0, b0, acc[0][0]);
          acc[0][1] = dot4(a0, b1, acc[0][1]);
          acc[1][0] = dot4(a1, b0, acc[1][0]);
          acc[1][1] = dot4(a1, b1, acc[1][1]);
        }
#pragma unroll
        for (int x = 0; x < 2; ++x)
#pragma unroll
          for (int y = 0; y < 2; ++y) {
            const int ii = i + 16 * x, jj = j + 16 * y;
            if (jj <= ii) P[ii * kPitchP + jj] = acc[x][y] * (p.scale * power[ii - jj]);
          }
        __syncthreads();
        // outputs: rows i, i + 16, columns N j .. + N - 1
        float o[2][N] = {};
        for (int d = 0; d < d1; d += 4) {
          const float4 a0 = *reinterpret_cast<const float4*>(A + i * pitch + d), a1 = *reinterpret_cast<const float4*>(A + (i + 16) * pitch + d);
          const float va[4] = {a0.x, a0.y, a0.z, a0.w}, vb[4] = {a1.x, a1.y, a1.z, a1.w};
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            float x[N];
            load_n<N>(X + (d + k) * kPitchW + N * j, x);
#pragma unroll
            for (int m = 0; m < N; ++m) {
              o[0][m] = fmaf(va[k], x[m], o[0][m]);
              o[1][m] = fmaf(vb[k], x[m], o[1][m]);
            }
          }
        }
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          const int ii = i + 16 * x;
          const float w = s.row_scale * power[ii + s.lag];
#pragma unroll
          for (int m = 0; m < N; ++m) o[x][m] *= w;
          for (int k = 0; k <= ii; ++k) {   // (not a row behind: what stands there may not be finite)
            const float pk = P[ii * kPitchP + k];
            float ck[N];
            load_n<N>(C + k * kPitchW + N * j, ck);
#pragma unroll
            for (int m = 0; m < N; ++m) o[x][m] = fmaf(pk, ck[m], o[x][m]);
          }
          if (ii < n) {
#pragma unroll
            for (int m = 0; m < N; ++m)
              if (N * j + m < width) put<T>(s, y0 + row(ii) * s.ys[2] + N * j + m, o[x][m]);
          }
        }
        __syncthreads();
      }
      // the state: rows 4 i .. + 3 of every 64, columns N j .. + N - 1
      const float keep = power[n];
      for (int r = 4 * i; r < d1; r += 64) {
        float x[4][N] = {};
        for (int k = 0; k < n; ++k) {
          float v[4], ck[N];
          load_n<4>(B + k * pitch + r, v);
          load_n<N>(Cw + k * kPitchW + N * j, ck);
#pragma unroll
          for (int e = 0; e < 4; ++e)
#pragma unroll
            for (int m = 0; m < N; ++m) x[e][m] = fmaf(v[e], ck[m], x[e][m]);
        }
#pragma unroll
        for (int e = 0; e < 4; ++e)
#pragma unroll
          for (int m = 0; m < N; ++m) {
            float* at = X + (r + e) * kPitchW + N * j + m;
            *at = fmaf(keep, *at, x[e][m]);
          }
      }
    }
    __syncthreads();
    if (g.states_only || hand_on) {
      for (int e = tid; e < d1 * kWidth; e += kThreads) {
        const int r = e / kWidth, w = e - r * kWidth;
        if (w >= width) continue;
        if (g.states_only) work[(int64_t)r * s.d2 + w0 + w] = X[r * kPitchW + w];
        else s.x_last[state + (s.x_transposed ? (int64_t)(w0 + w) * d1 + r : (int64_t)r * s.d2 + w0 + w)] = X[r * kPitchW + w];
      }
    }
  }
  if (g.states_only) return;
  // rows without a state, and rows of padding
  if (!q.bad && p.starts) return;
  const int64_t end = p.starts ? q.n : p.seq_len, upto = end < from + g.rows ? end : from + g.rows;
  const int64_t first = q.bad || q.n < from ? from : q.n;
  for (int64_t e = first * width + tid; e < upto * width; e += kThreads)
    put<T>(s, y0 + (e / width) * s.ys[2] + e % width, e / width < q.n ? __int_as_float(0x7fffffff) : 0.f);
}

// The states before the segments, from what each adds, in place; and the state behind the last.  A thread has the same four elements of all
// segments of a scan, sequence and head.
__global__ void __launch_bounds__(256) join_kernel(const __grid_constant__ Params p, const Segments g, const int first, const int scans, const int matrix) {
  const int parts = (matrix + 1023) / 1024;
  const unsigned unit = blockIdx.x / (unsigned)parts;
  const int which = first + (int)(unit % (unsigned)scans), item = (int)(unit / (unsigned)scans);
  const int e = ((int)(blockIdx.x % (unsigned)parts) * 256 + threadIdx.x) * 4;
  const Scan& s = p.scan[which];
  const int b = item / p.heads, h = item - b * p.heads;
  const Sequence q = sequence_of(p, b);
  if (q.bad || e >= matrix) return;
  const double decay = log_decay(p.decay, h);
  float* work = g.work + ((int64_t)which * p.batch * p.heads + item) * g.count * matrix + e;
  const int64_t state = (q.state * p.heads + h) * (int64_t)matrix;
  const int d2 = s.d2, r = e / d2, c = e - r * d2;   // (sizes are multiples of 8: the four are of one row)
  float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
  if (s.x_first && q.state >= 0) {
    if (s.x_transposed) {
      const float* f = s.x_first + state + (int64_t)c * s.d1 + r;
      x = make_float4(f[0], f[s.d1], f[2 * s.d1], f[3 * s.d1]);
    } else {
      x = *reinterpret_cast<const float4*>(s.x_first + state + e);
    }
  }
  for (int i = 0; i < g.count; ++i) {
    const int64_t left = q.n - (int64_t)i * g.rows;
    if (left <= 0) break;
    const float keep = decay_power(decay, (double)(left < g.rows ? left : g.rows));
    float4* at = reinterpret_cast<float4*>(work + (int64_t)i * matrix);
    const float4 t = *at;
    *at = x;
    x.x = fmaf(keep, x.x, t.x);
    x.y = fmaf(keep, x.y, t.y);
    x.z = fmaf(keep, x.z, t.z);
    x.w = fmaf(keep, x.w, t.w);
  }
  if (s.x_last && q.state >= 0) {
    if (s.x_transposed) {
      float* f = s.x_last + state + (int64_t)c * s.d1 + r;
      f[0] = x.x;
      f[s.d1] = x.y;
      f[2 * s.d1] = x.z;
      f[3 * s.d1] = x.w;
    } else {
      *reinterpret_cast<float4*>(s.x_last + state + e) = x;
    }
  }
}

template <typename T>
__global__ void __launch_bounds__(256) group_sum_kernel(const GroupSum p, const int parts) {
  const int which = blockIdx.y, d = p.d[which];
  const int item = blockIdx.x / parts, part = blockIdx.x - item * parts;
  const int b = item / p.kv_heads, kh = item - b * p.kv_heads;
  int64_t row0 = 0, n = p.seq_len, live = p.seq_len;
  if (p.starts) {
    int64_t lo = p.starts[b], hi = p.starts[b + 1];
    lo = lo < 0 ? 0 : (lo > p.tokens ? p.tokens : lo);
    hi = hi < lo ? lo : (hi > p.tokens ? p.tokens : hi);
    row0 = lo;
    live = n = hi - lo < p.seq_len ? hi - lo : p.seq_len;
  } else if (p.lengths) {
    const int64_t l = p.lengths[b];
    live = l < 0 ? 0 : (l < n ? l : n);
  }
  const int heads = p.kv_heads * p.group;
  const float* in = p.partial[which] + (p.starts ? 0 : (int64_t)b * heads * p.rows * d) + (int64_t)kh * p.group * p.rows * d + row0 * d;
  T* out = static_cast<T*>(p.out[which]) + (p.starts ? 0 : b * p.os[which][0]) + kh * p.os[which][1] + row0 * p.os[which][2];
  for (int64_t e = (int64_t)part * 256 + threadIdx.x; e < n * d; e += (int64_t)parts * 256) {
    const int64_t r = e / d;
    float x = 0.f;
    if (r < live)
      for (int g = 0; g < p.group; ++g) x += in[(int64_t)g * p.rows * d + e];
    out[r * p.os[which][2] + (e - r * d)] = from_float<T>(x);
  }
}

}  // namespace

cudaError_t launch_join(const Params& p, const Segments& g, int first, int scans, int matrix, cudaStream_t stream) {
  const int64_t grid = (int64_t)p.batch * p.heads * scans * ((matrix + 1023) / 1024);
  if (grid > 0x7fffffff) return cudaErrorInvalidConfiguration;
  join_kernel<<<(unsigned)grid, 256, 0, stream>>>(p, g, first, scans, matrix);
  return cudaGetLastError();
}

namespace {
struct Plan { int width, segments; };
// Segments: two chunks each at least, where the slices of all sequences and heads are fewer than two CTAs an SM; fewer than three gain nothing, as both
// passes and the join cost about the uncut scan's work again.  Width: slices of 64 columns feed more multiply-adds from each read and form a . b half
// as often, but there are half as many, they take 7/6 of the time of 32 columns and fewer of them fit an SM.  So each is reckoned as passes x waves x
// chunks of a CTA (bf16, 16 heads, 32 against 64 columns, us): heads of 256, B4 S1024, 6057 / 3531 (four waves / two); 192: 2162 / 2386 (two / two);
// 160: 1517 / 1036 (two / one); 136, B1: 392 / 285 (3 / 6 segments); 256, B1 S128: 137 / 158 (one / one).
Plan plan_of(const Params& p, int num_sms) {
  Plan best{};
  int64_t least = 0;
  const int64_t chunks = ((int64_t)p.seq_len + kChunk - 1) / kChunk;
  for (int width = 32; width <= 64; width += 32) {
    int64_t ctas = 0;
    size_t smem = 0;
    for (int i = 0; i < p.scans; ++i) {
      ctas += (int64_t)p.batch * p.heads * ((p.scan[i].d2 + width - 1) / width);
      const size_t need = smem_bytes(p.scan[i].d1, width);
      smem = need > smem ? need : smem;
    }
    if (ctas == 0) return Plan{32, 1};
    const int64_t most = (chunks + 1) / 2;
    int64_t n = 2 * num_sms / ctas;
    n = n < most ? n : most;
    n = n < 64 ? n : 64;
    if (n < 3) n = 1;
    int64_t fit = (int64_t)(228 * 1024 / (smem + 1024));
    fit = fit < ctas_of(width) ? fit : ctas_of(width);
    const int64_t at_once = (fit > 1 ? fit : 1) * num_sms;
    const int64_t cost = (n > 1 ? 2 : 1) * ((ctas * n + at_once - 1) / at_once) * ((chunks + n - 1) / n) * (width == 64 ? 7 : 6);
    if (best.width == 0 || cost < least) {
      best = Plan{width, (int)n};
      least = cost;
    }
  }
  return best;
}
}  // namespace

int64_t scan_generic_bytes(const Params& p, int num_sms) {
  const int n = plan_of(p, num_sms).segments;
  return n == 1 ? 0 : (int64_t)p.scans * p.batch * p.heads * n * p.scan[0].d1 * p.scan[0].d2 * 4;
}

cudaError_t launch_scan_generic(const Params& p, int num_sms, float* work, int64_t work_bytes, cudaStream_t stream, int* launches) {
  int64_t grid = 0;
  size_t smem = 0;
  const Plan plan = plan_of(p, num_sms);
  const int width = plan.width;
  Segments g;
  g.count = work && work_bytes >= scan_generic_bytes(p, num_sms) ? plan.segments : 1;
  const int64_t per = (p.seq_len + g.count - 1) / g.count, rows = (per + kChunk - 1) / kChunk * kChunk;
  g.rows = (int)(rows < 0x7fffffe0ll ? rows : 0x7fffffe0ll);
  g.states_only = 0;
  g.work = work;
  for (int i = 0; i < p.scans; ++i) {
    const int64_t n = (int64_t)p.batch * p.heads * g.count * ((p.scan[i].d2 + width - 1) / width);
    grid = n > grid ? n : grid;
    const size_t need = smem_bytes(p.scan[i].d1, width);
    smem = need > smem ? need : smem;
  }
  if (grid > 0x7fffffff) return cudaErrorInvalidConfiguration;
  auto kern = width == 64 ? (p.dtype == AIDN_F32 ? scan_kernel<float, 64> : p.dtype == AIDN_F16 ? scan_kernel<__half, 64> : scan_kernel<__nv_bfloat16, 64>)
                          : (p.dtype == AIDN_F32 ? scan_kernel<float, 32> : p.dtype == AIDN_F16 ? scan_kernel<__half, 32> : scan_kernel<__nv_bfloat16, 32>);
  cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem_bytes(256, width));
  if (e != cudaSuccess) return e;
  if (g.count > 1) {
    g.states_only = 1;
    kern<<<dim3((unsigned)grid, (unsigned)p.scans), kThreads, smem, stream>>>(p, g);
    g.states_only = 0;
    e = cudaGetLastError();
    if (e == cudaSuccess) e = launch_join(p, g, 0, p.scans, p.scan[0].d1 * p.scan[0].d2, stream);
    if (e != cudaSuccess) return e;
    *launches += 2;
  }
  kern<<<dim3((unsigned)grid, (unsigned)p.scans), kThreads, smem, stream>>>(p, g);
  ++*launches;
  return cudaGetLastError();
}

cudaError_t launch_group_sum(const GroupSum& p, cudaStream_t stream) {
  const int widest = p.d[0] > p.d[1] ? p.d[0] : p.d[1];
  const int64_t items = (int64_t)p.batch * p.kv_heads;
  int64_t parts = (p.seq_len * widest + 1023) / 1024;
  if (parts > 1024) parts = 1024;
  if (parts * items > 0x7fffffff) parts = 0x7fffffff / items;
  const dim3 grid((unsigned)(items * parts), 2);
  if (p.dtype == AIDN_F32) group_sum_kernel<float><<<grid, 256, 0, stream>>>(p, (int)parts);
  else if (p.dtype == AIDN_F16) group_sum_kernel<__half><<<grid, 256, 0, stream>>>(p, (int)parts);
  else group_sum_kernel<__nv_bfloat16><<<grid, 256, 0, stream>>>(p, (int)parts);
  return cudaGetLastError();
}

}  // namespace lin
}  // namespace aidn
