// Linear attention, one token of each sequence:  S = lam S + k v^T,  o = scale * q S, on states of fp32 that stay where they are.
//
// Bound by the states' bytes, once in and once out.  A CTA has some columns of one head's state: a thread four columns of every
// so many rows, whose loads are all issued before the first is used; a column's sum over the rows is joined through shared memory.  Columns
// need nothing of one another, so that few heads are cut by columns until the SMs have work.
#include "linear.cuh"

namespace aidn {
namespace lin {
namespace {

constexpr int kThreads = 256;
constexpr int kRows = 16;   // of a thread, in flight together

template <typename T>
__global__ void __launch_bounds__(kThreads) step_kernel(const Step p, const int width, const int slices) {
  __shared__ float qk[2][256];
  __shared__ float4 part[kThreads];
  const int item = blockIdx.x / slices, v0 = (blockIdx.x - item * slices) * width;
  const int b = item / p.heads, h = item - b * p.heads, kh = h / p.group;
  const int cols = p.value_dim - v0 < width ? p.value_dim - v0 : width;
  T* out = static_cast<T*>(p.out) + b * p.os[0] + h * p.os[1] + v0;
  int64_t slot = b;
  if (p.slots) {
    slot = p.slots[b];
    bool bad = slot >= p.num_slots;
    if (slot >= 0)
      for (int i = threadIdx.x; i < b; i += kThreads) bad = bad || p.slots[i] == slot;
    bad = __syncthreads_or(bad) != 0;
    if (slot < 0 || bad) {   // no state: a padding row, or a mistake that shows
      if (threadIdx.x < cols) out[threadIdx.x] = from_float<T>(slot < 0 ? 0.f : __int_as_float(0x7fffffff));
      return;
    }
  }
  const int quads = cols / 4, groups = kThreads / quads;
  const int group = threadIdx.x / quads, quad = threadIdx.x - group * quads;
  float4* state = reinterpret_cast<float4*>(p.states + (slot * p.heads + h) * ((int64_t)p.key_dim * p.value_dim) + v0) + quad;
  const int pitch = p.value_dim / 4;
  float4 s[kRows];
  auto load = [&](int r0) {
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
      const int r = r0 + i * groups;
      if (group < groups && r < p.key_dim) s[i] = state[(int64_t)r * pitch];
    }
  };
  load(group);
  const T* q = static_cast<const T*>(p.q) + b * p.qs[0] + h * p.qs[1];
  const T* k = static_cast<const T*>(p.k) + b * p.ks[0] + kh * p.ks[1];
  const T* v = static_cast<const T*>(p.v) + b * p.vs[0] + kh * p.vs[1] + v0 + quad * 4;
  if (threadIdx.x < p.key_dim) {
    qk[0][threadIdx.x] = to_float(q[threadIdx.x]) * p.scale;
    qk[1][threadIdx.x] = to_float(k[threadIdx.x]);
  }
  float4 vv = make_float4(0.f, 0.f, 0.f, 0.f);
  if (group < groups) vv = make_float4(to_float(v[0]), to_float(v[1]), to_float(v[2]), to_float(v[3]));
  const float lam = decay_power(log_decay(p.decay, h), 1.0);
  __syncthreads();
  float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int r0 = group; r0 < p.key_dim; r0 += kRows * groups) {
    if (r0 != group) load(r0);
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
      const int r = r0 + i * groups;
      if (group < groups && r < p.key_dim) {
        const float kr = qk[1][r], qr = qk[0][r];
        s[i].x = fmaf(kr, vv.x, lam * s[i].x);
        s[i].y = fmaf(kr, vv.y, lam * s[i].y);
        s[i].z = fmaf(kr, vv.z, lam * s[i].z);
        s[i].w = fmaf(kr, vv.w, lam * s[i].w);
        state[(int64_t)r * pitch] = s[i];
        sum.x = fmaf(qr, s[i].x, sum.x);
        sum.y = fmaf(qr, s[i].y, sum.y);
        sum.z = fmaf(qr, s[i].z, sum.z);
        sum.w = fmaf(qr, s[i].w, sum.w);
      }
    }
  }
  part[threadIdx.x] = sum;
  __syncthreads();
  if (threadIdx.x < cols) {
    const float* f = reinterpret_cast<const float*>(part) + threadIdx.x;
    float o = 0.f;
    for (int i = 0; i < groups; ++i) o += f[i * cols];
    out[threadIdx.x] = from_float<T>(o);
  }
}

}  // namespace

cudaError_t launch_step(const Step& p, int num_sms, cudaStream_t stream) {
  int width = p.value_dim;
  const int64_t items = (int64_t)p.batch * p.heads;
  while (width > 16 && width % 8 == 0 && items * ((p.value_dim + width - 1) / width) < 2 * num_sms) width /= 2;
  const int slices = (p.value_dim + width - 1) / width;
  if (items * slices > 0x7fffffff) return cudaErrorInvalidConfiguration;
  const unsigned grid = (unsigned)(items * slices);
  if (p.dtype == AIDN_F32) step_kernel<float><<<grid, kThreads, 0, stream>>>(p, width, slices);
  else if (p.dtype == AIDN_F16) step_kernel<__half><<<grid, kThreads, 0, stream>>>(p, width, slices);
  else step_kernel<__nv_bfloat16><<<grid, kThreads, 0, stream>>>(p, width, slices);
  return cudaGetLastError();
}

}  // namespace lin
}  // namespace aidn
