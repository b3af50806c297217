// Linear attention with a decay for each head: launch parameters shared by its kernels.
//
// Everything but the single-token step is one recurrence, the scan
//     X_(i+1) = lam X_i + key_scale * b_i c_i^T (times lam where lag is 0),   y_i = row_scale lam^lag a_i X_i + scale (a_i . b_i) c_i,
// which over a chunk of n rows behind the state X reads
//     y_i = row_scale lam^(i + lag) a_i X  +  sum over j <= i of scale lam^(i - j) (a_i . b_j) c_j
//     X'  = lam^n X + key_scale * sum over j of lam^(n - lag - j) b_j c_j^T          (lam = exp of the head's log decay)
// The forward pass is the scan (q, k, v) from the first state, with lag 1.  With U_t = scale q_t do_t^T + lam U_(t+1) the gradients are
//     dq: (do, v, k), lag 1, from the transposed first state;
//     dk: (v, do, q) and dv: (k, q, do) from the last row to the first, lag 0, from the gradient of the last state.
#pragma once

#include "common.cuh"

namespace aidn {
namespace lin {

struct Scan {
  const void* a;       // [.., d1]
  const void* b;       // [.., d1]
  const void* c;       // [.., d2]
  void* y;             // [.., d2]
  int64_t as[3], bs[3], cs[3], ys[3];   // element strides for (sequence, head, row)
  int32_t a_group, b_group, c_group;    // heads that share one of a's (b's, c's): head h reads h / group
  int32_t d1, d2;
  int32_t reverse;     // rows from a sequence's last to its first
  int32_t lag;
  int32_t y_f32;       // y is fp32 (partial sums over shared heads)
  float row_scale, key_scale;
  const float* x_first;   // [state, head, ..] or null: zeros
  float* x_last;          // or null
  int32_t x_transposed;   // the states are [d2][d1], else [d1][d2]
};

struct Params {
  Scan scan[3];
  int32_t scans;
  const float* decay;        // [heads] or null
  const int32_t* lengths;    // [batch] or null
  const int32_t* starts;     // [batch + 1] or null
  const int32_t* slots;      // [batch] or null: sequence b has state b
  int64_t tokens;            // rows of packed tensors
  int64_t seq_len;           // the most rows of a sequence
  int32_t batch, heads, num_slots, dtype;
  float scale;
};

// A sequence's rows and state.
struct Sequence {
  int64_t row0;    // its first row in packed tensors, else 0
  int64_t n;       // its rows
  int64_t state;   // its state, -1: none
  bool bad;        // its state is not there, or an earlier sequence's
};

// Called by all threads of a CTA.  `slots` may name a state twice by mistake; it is the first one's then.
__device__ __forceinline__ Sequence sequence_of(const Params& p, int b) {
  Sequence s;
  s.row0 = 0;
  s.n = p.seq_len;
  if (p.starts) {
    int64_t lo = p.starts[b], hi = p.starts[b + 1];
    lo = lo < 0 ? 0 : (lo > p.tokens ? p.tokens : lo);
    hi = hi < lo ? lo : (hi > p.tokens ? p.tokens : hi);
    s.row0 = lo;
    s.n = hi - lo < p.seq_len ? hi - lo : p.seq_len;
  } else if (p.lengths) {
    const int64_t l = p.lengths[b];
    s.n = l < 0 ? 0 : (l < s.n ? l : s.n);
  }
  s.state = b;
  s.bad = false;
  if (p.slots) {
    s.state = p.slots[b];
    bool bad = s.state >= p.num_slots;
    if (s.state < 0) s.state = -1;
    else
      for (int i = threadIdx.x; i < b; i += blockDim.x) bad = bad || p.slots[i] == s.state;
    s.bad = __syncthreads_or(bad) != 0;
  }
  return s;
}

// A head's log decay.  0 * -inf is no exponent, so that a decay to nothing is a large finite one; above 0 is refused by NaN.
__device__ __forceinline__ double log_decay(const float* decay, int h) {
  if (!decay) return 0.0;
  const float g = decay[h];
  if (!(g <= 0.f)) return __longlong_as_double(0x7ff8000000000000ll);
  return fmax((double)g, -1e30);
}
// Its factor over n rows, rounded once.  (A state is multiplied by the same one chunk after chunk: what exp2f is off by, up to two units in the last
// place, would add up over all the chunks that the state remembers.)
__device__ __forceinline__ float decay_power(double g, double n) { return (float)exp(g * n); }

// Sequences cut into segments: a first launch leaves what each adds to the state in `work` ([scan][sequence, head][segment][d1][d2]),
// launch_join turns those into the states before them and writes the last ones, and the scan then starts every segment from its own.
struct Segments {
  int32_t count;         // 1: uncut
  int32_t rows;          // of a segment
  int32_t states_only;   // the first launch
  float* work;
};
// The scans first .. first + scans - 1, of matrix elements a state.
cudaError_t launch_join(const Params& p, const Segments& g, int first, int scans, int matrix, cudaStream_t stream);

// a scan on FFMA, any sizes and types.  Without its workspace long sequences are not cut.
int64_t scan_generic_bytes(const Params& p, int num_sms);
cudaError_t launch_scan_generic(const Params& p, int num_sms, float* work, int64_t work_bytes, cudaStream_t stream, int* launches);

// 16-bit types with sizes of 64 and 128 on tcgen05 (csrc/linear_sm100.cu).  Without its workspace long sequences are not cut.
bool scan_sm100_supported(const Params& p);
int64_t scan_sm100_bytes(const Params& p, int num_sms);
// expire: test hook - the loads are withheld and bounded waits give up after 20 ms.
cudaError_t launch_scan_sm100(const Params& p, int num_sms, float* work, int64_t work_bytes, bool expire, cudaStream_t stream, int* launches);
uint32_t* sm100_gave_up();   // address of its count of CTAs that gave up in the current context, or null

// dk / dv of shared heads: fp32 partial sums [.., heads, .., d] summed over each group in order
struct GroupSum {
  const float* partial[2];
  void* out[2];
  int64_t os[2][3];
  int32_t d[2];
  int64_t rows;         // of a partial's head
  const int32_t* lengths;
  const int32_t* starts;
  int64_t tokens, seq_len;
  int32_t batch, kv_heads, group, dtype;
};
cudaError_t launch_group_sum(const GroupSum& p, cudaStream_t stream);

struct Step {
  const void* q;
  const void* k;
  const void* v;
  void* out;
  float* states;            // [num_slots, heads, key_dim, value_dim]
  const float* decay;
  const int32_t* slots;
  int64_t qs[2], ks[2], vs[2], os[2];   // element strides for (row, head)
  int32_t batch, heads, group, key_dim, value_dim, num_slots, dtype;
  float scale;
};
cudaError_t launch_step(const Step& p, int num_sms, cudaStream_t stream);

struct Rotary {
  const void* x[2];         // queries, keys
  void* y[2];
  int64_t xs[2][2], ys[2][2];   // element strides for (token, head)
  const double* frequencies;
  const void* positions;    // int32 or int64, or null: start + token % seq_len
  int64_t tokens, seq_len, start;
  int32_t heads[2];
  int32_t head_dim, rotary_dim, dtype, halves, wide_positions;
  float amplitude, sign;
};
cudaError_t launch_rotary(const Rotary& p, cudaStream_t stream);

}  // namespace lin
}  // namespace aidn
