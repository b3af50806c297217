// The scan of linear.cuh on FFMA: any type, any head sizes.  A CTA takes some columns of c (and of the state) for one sequence and head and walks
// its rows in chunks, the state in shared memory in fp32; the chunk's products a . b are formed again for every slice of columns.  What
// bounds it is arithmetic and the reads of shared memory that feed it.
#include "linear.cuh"

namespace aidn {
namespace lin {
namespace {

constexpr int kThreads = 256;
constexpr int kChunk = 32;
constexpr int kWidth = 32;   // columns of a slice

__host__ __device__ constexpr int pitch_of(int d) { return d + 1; }   // (odd: rows of a column lie in different banks)
inline size_t smem_bytes(int d1) {
  return sizeof(float) * (2 * kChunk * pitch_of(d1) + kChunk * kWidth + (size_t)d1 * kWidth + kChunk * (kChunk + 1) + kChunk + 1);
}

template <typename T>
__device__ __forceinline__ void put(const Scan& s, int64_t at, float x) {
  if (s.y_f32) static_cast<float*>(s.y)[at] = x;
  else static_cast<T*>(s.y)[at] = from_float<T>(x);
}

template <typename T>
__global__ void __launch_bounds__(kThreads) scan_kernel(const Params p) {
  extern __shared__ float smem[];
  const Scan& s = p.scan[blockIdx.y];
  const int slices = (s.d2 + kWidth - 1) / kWidth;
  if (blockIdx.x >= (int64_t)p.batch * p.heads * slices) return;   // (the scans of one launch may have different widths)
  const int item = blockIdx.x / slices, w0 = (blockIdx.x - item * slices) * kWidth;
  const int b = item / p.heads, h = item - b * p.heads;
  const int width = s.d2 - w0 < kWidth ? s.d2 - w0 : kWidth;
  const int d1 = s.d1, pitch = pitch_of(d1), tid = threadIdx.x;
  float* A = smem;
  float* B = A + kChunk * pitch;
  float* C = B + kChunk * pitch;
  float* X = C + kChunk * kWidth;
  float* P = X + d1 * kWidth;
  float* power = P + kChunk * (kChunk + 1);   // lam^0 .. lam^kChunk

  const Sequence q = sequence_of(p, b);
  const T* a = static_cast<const T*>(s.a) + (p.starts ? 0 : b * s.as[0]) + (h / s.a_group) * s.as[1] + q.row0 * s.as[2];
  const T* bb = static_cast<const T*>(s.b) + (p.starts ? 0 : b * s.bs[0]) + (h / s.b_group) * s.bs[1] + q.row0 * s.bs[2];
  const T* c = static_cast<const T*>(s.c) + (p.starts ? 0 : b * s.cs[0]) + (h / s.c_group) * s.cs[1] + q.row0 * s.cs[2] + w0;
  const int64_t y0 = (p.starts ? 0 : b * s.ys[0]) + h * s.ys[1] + q.row0 * s.ys[2] + w0;
  if (q.bad) {
    for (int64_t e = tid; e < q.n * width; e += kThreads) put<T>(s, y0 + (e / width) * s.ys[2] + e % width, __int_as_float(0x7fffffff));
  } else {
    const float g = log2_decay(p.decay, h);
    if (tid <= kChunk) power[tid] = exp2f(g * tid);
    const int64_t state = (q.state * p.heads + h) * (int64_t)s.d1 * s.d2;
    for (int e = tid; e < d1 * kWidth; e += kThreads) {
      const int r = e / kWidth, w = e - r * kWidth;
      X[e] = s.x_first && q.state >= 0 && w < width ? s.x_first[state + (s.x_transposed ? (int64_t)(w0 + w) * d1 + r : (int64_t)r * s.d2 + w0 + w)] : 0.f;
    }
    for (int64_t t0 = 0; t0 < q.n; t0 += kChunk) {
      const int n = (int)(q.n - t0 < kChunk ? q.n - t0 : kChunk);
      auto row = [&](int i) { return s.reverse ? q.n - 1 - (t0 + i) : t0 + i; };
      __syncthreads();
      for (int e = tid; e < kChunk * d1; e += kThreads) {
        const int i = e / d1, d = e - i * d1;
        A[i * pitch + d] = i < n ? to_float(a[row(i) * s.as[2] + d]) : 0.f;
        B[i * pitch + d] = i < n ? to_float(bb[row(i) * s.bs[2] + d]) : 0.f;
      }
      for (int e = tid; e < kChunk * kWidth; e += kThreads) {
        const int i = e / kWidth, w = e - i * kWidth;
        C[e] = i < n && w < width ? to_float(c[row(i) * s.cs[2] + w]) : 0.f;
      }
      __syncthreads();
      {
        // 2 x 2 products to a thread
        const int i = tid / 16, j = tid % 16;
        float acc[2][2] = {};
        for (int d = 0; d < d1; ++d) {
          const float a0 = A[i * pitch + d], a1 = A[(i + 16) * pitch + d], b0 = B[j * pitch + d], b1 = B[(j + 16) * pitch + d];
          acc[0][0] = fmaf(a0, b0, acc[0][0]);
          acc[0][1] = fmaf(a0, b1, acc[0][1]);
          acc[1][0] = fmaf(a1, b0, acc[1][0]);
          acc[1][1] = fmaf(a1, b1, acc[1][1]);
        }
#pragma unroll
        for (int x = 0; x < 2; ++x)
#pragma unroll
          for (int y = 0; y < 2; ++y) {
            const int ii = i + 16 * x, jj = j + 16 * y;
            if (jj <= ii) P[ii * (kChunk + 1) + jj] = acc[x][y] * (p.scale * power[ii - jj]);
          }
      }
      __syncthreads();
      {
        // a column of four rows to a thread
        const int w = tid % kWidth, i0 = tid / kWidth;
        float acc[4] = {};
        for (int d = 0; d < d1; ++d) {
          const float x = X[d * kWidth + w];
#pragma unroll
          for (int r = 0; r < 4; ++r) acc[r] = fmaf(A[(i0 + 8 * r) * pitch + d], x, acc[r]);
        }
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int i = i0 + 8 * r;
          float y = acc[r] * (s.row_scale * exp2f(g * (i + s.lag)));
          for (int j = 0; j <= i; ++j) y = fmaf(P[i * (kChunk + 1) + j], C[j * kWidth + w], y);
          if (i < n && w < width) put<T>(s, y0 + row(i) * s.ys[2] + w, y);
        }
      }
      __syncthreads();
      const float keep = power[n];
      for (int e = tid; e < d1 * kWidth; e += kThreads) {
        const int r = e / kWidth, w = e - r * kWidth;
        float acc = 0.f;
        for (int j = 0; j < n; ++j) acc = fmaf(B[j * pitch + r] * power[n - s.lag - j], C[j * kWidth + w], acc);
        X[e] = fmaf(keep, X[e], s.key_scale * acc);
      }
    }
    if (s.x_last && q.state >= 0) {
      for (int e = tid; e < d1 * kWidth; e += kThreads) {   // (each thread's own elements)
        const int r = e / kWidth, w = e - r * kWidth;
        if (w < width) s.x_last[state + (s.x_transposed ? (int64_t)(w0 + w) * d1 + r : (int64_t)r * s.d2 + w0 + w)] = X[e];
      }
    }
  }
  if (!p.starts)   // the rows of padding
    for (int64_t e = tid + q.n * width; e < p.seq_len * width; e += kThreads) put<T>(s, y0 + (e / width) * s.ys[2] + e % width, 0.f);
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

cudaError_t launch_scan_generic(const Params& p, cudaStream_t stream, int* launches) {
  int64_t grid = 0;
  size_t smem = 0;
  for (int i = 0; i < p.scans; ++i) {
    const int64_t n = (int64_t)p.batch * p.heads * ((p.scan[i].d2 + kWidth - 1) / kWidth);
    grid = n > grid ? n : grid;
    const size_t need = smem_bytes(p.scan[i].d1);
    smem = need > smem ? need : smem;
  }
  if (grid > 0x7fffffff) return cudaErrorInvalidConfiguration;
  auto kern = p.dtype == AIDN_F32 ? scan_kernel<float> : p.dtype == AIDN_F16 ? scan_kernel<__half> : scan_kernel<__nv_bfloat16>;
  const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem_bytes(256));
  if (e != cudaSuccess) return e;
  kern<<<dim3((unsigned)grid, (unsigned)p.scans), kThreads, smem, stream>>>(p);
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
