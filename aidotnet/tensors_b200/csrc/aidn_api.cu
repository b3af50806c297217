// C ABI of libaidotnet_sdpa_sm100 (declared in include/aidn_sdpa.h): argument validation, kernel selection
// and launch.  No torch types, no allocation on the launch path, no CPU fallback: a request no CUDA kernel
// of this build can serve is an error.
#include <dlfcn.h>

#include <atomic>
#include <cmath>
#include <cstdarg>
#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <initializer_list>
#include <map>
#include <mutex>
#include <new>
#include <utility>

#include "common.cuh"
#include "kv8.cuh"
#include "linear.cuh"
#include "../../../include/aidn_sdpa_debug.h"

namespace {

thread_local char g_err[512] = "";
thread_local bool g_expire_linear = false;   // the same for aidn_linear_attention and its backward
thread_local int g_linear_launches = 0;      // of this thread's last aidn_linear_attention or its backward
thread_local bool g_expire_qkv = false;   // test hook: this thread's next aidn_qkv_rope_cache lets its bounded waits run out

int fail(int code, const char* fmt, ...) {
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(g_err, sizeof(g_err), fmt, ap);
  va_end(ap);
  return code;
}

int fail_cuda(cudaError_t e, const char* what) {
  return fail(AIDN_ECUDA, "%s: %s (%s)", what, cudaGetErrorString(e), cudaGetErrorName(e));
}

inline int64_t align_up(int64_t x, int64_t a) { return (x + a - 1) / a * a; }

// AIDOTNET_KERNEL_LAUNCH_CHECK=1, the reference's own debugging switch (CudaBackend.cs:5381-5421): every entry point
// then synchronises the stream right after its launches and reports a device error, or a bounded wait that gave up, as
// the failure of THAT call instead of some later one.  Skipped while the stream is being captured.  Read once.
bool launch_check_enabled() {
  static const bool on = [] {
    const char* v = std::getenv("AIDOTNET_KERNEL_LAUNCH_CHECK");
    return v && v[0] == '1' && v[1] == 0;
  }();
  return on;
}

// `reset`: the status word has no handle whose poll would clear it, so that reporting it does.
int post_launch_check(cudaStream_t stream, const char* what, int32_t* status_dev, bool reset = false) {
  if (!launch_check_enabled()) return AIDN_OK;
  cudaStreamCaptureStatus cap = cudaStreamCaptureStatusNone;
  if (cudaStreamIsCapturing(stream, &cap) != cudaSuccess || cap != cudaStreamCaptureStatusNone) {
    cudaGetLastError();
    return AIDN_OK;
  }
  cudaError_t e = cudaStreamSynchronize(stream);
  if (e != cudaSuccess) return fail(AIDN_ECUDA, "[LAUNCH-FAULT] %s: %s (%s)", what, cudaGetErrorString(e), cudaGetErrorName(e));
  if (status_dev) {
    int32_t st = 0;
    e = cudaMemcpy(&st, status_dev, sizeof(st), cudaMemcpyDeviceToHost);
    if (e != cudaSuccess) return fail_cuda(e, "launch check: status read");
    if (st && reset) cudaMemset(status_dev, 0, sizeof(st));
    if (st & aidn::kStatusTimeout) return fail(AIDN_ETIMEOUT, "[LAUNCH-FAULT] %s: a kernel gave up a bounded wait (status word 0x%x)", what, st);
  }
  return AIDN_OK;
}

size_t elem_size(int dtype) { return dtype == AIDN_F32 ? 4 : 2; }

// ---- NCCL, resolved lazily so that the library loads on machines without it --------------------------
struct Nccl {
  void* lib = nullptr;
  int (*AllGather)(const void*, void*, size_t, int, void*, cudaStream_t) = nullptr;
  int (*GroupStart)() = nullptr;
  int (*GroupEnd)() = nullptr;
  int (*CommUserRank)(void*, int*) = nullptr;
  int (*CommCount)(void*, int*) = nullptr;
  const char* (*GetErrorString)(int) = nullptr;
  bool ok = false;
};
Nccl g_nccl;
std::once_flag g_nccl_once;

void load_nccl() {
  const char* names[] = {"libnccl.so.2", "libnccl.so"};
  for (const char* n : names) {
    g_nccl.lib = dlopen(n, RTLD_NOW | RTLD_GLOBAL);
    if (g_nccl.lib) break;
  }
  if (!g_nccl.lib) return;
  g_nccl.AllGather = (decltype(g_nccl.AllGather))dlsym(g_nccl.lib, "ncclAllGather");
  g_nccl.GroupStart = (decltype(g_nccl.GroupStart))dlsym(g_nccl.lib, "ncclGroupStart");
  g_nccl.GroupEnd = (decltype(g_nccl.GroupEnd))dlsym(g_nccl.lib, "ncclGroupEnd");
  g_nccl.CommUserRank = (decltype(g_nccl.CommUserRank))dlsym(g_nccl.lib, "ncclCommUserRank");
  g_nccl.CommCount = (decltype(g_nccl.CommCount))dlsym(g_nccl.lib, "ncclCommCount");
  g_nccl.GetErrorString = (decltype(g_nccl.GetErrorString))dlsym(g_nccl.lib, "ncclGetErrorString");
  g_nccl.ok = g_nccl.AllGather && g_nccl.GroupStart && g_nccl.GroupEnd && g_nccl.CommUserRank && g_nccl.CommCount;
}

constexpr int kNcclFloat32 = 7, kNcclFloat16 = 6, kNcclBfloat16 = 9;  // ncclDataType_t values (nccl.h)

}  // namespace

struct aidn_sdpa {
  aidn_sdpa_desc d;
  int group;
  int head_count;
  int32_t* status_dev;   // [0] status word, [1..2] scheduler counters of the persistent prefill kernel
  int num_sms;
  void* scratch;
  int64_t scratch_bytes;
  int last_path;
  int last_launches;
  float* debug;
  int debug_mode;
  uint64_t kv8_raised;                  // which kernels over 8-bit pools had their shared-memory limit raised in this context
  aidn::PrefillMapCache prefill_maps;   // tensor maps of the last tcgen05 prefill launch (see common.cuh)
};

namespace {


// Keys per split of the decode kernel.  Enough CTAs to fill 148 SMs several times over, but never more than
// 512 keys per CTA so that ragged kv_len values balance, and never fewer than 64.
int pick_chunk(const aidn_sdpa* h, int64_t batch, int64_t seq_kv) {
  if (h->d.decode_chunk > 0) return h->d.decode_chunk;
  const int gt = h->group <= 2 ? h->group : (h->group <= 4 ? 4 : 8);  // as the FFMA decode launcher picks
  int gchunks = (h->group + gt - 1) / gt;
  int64_t cap = 512;
  // 16-bit inputs with up to 16 query heads per KV head run the tensor-core decode kernel: one CTA per KV head and
  // split, and chunks up to 1024 keys (its per-CTA prologue and merge are heavier, its steady state faster)
  if (h->d.qkv_dtype != AIDN_F32 && (h->d.head_dim == 64 || h->d.head_dim == 128) && h->group <= 16) {
    gchunks = 1;
    cap = 1024;
  }
  const int64_t items = batch * (h->head_count / h->group) * gchunks;
  const int64_t target = 148 * 8;
  int64_t splits = (target + items - 1) / items;
  if (splits < 1) splits = 1;
  int64_t chunk = align_up((seq_kv + splits - 1) / splits, 64);
  if (chunk > cap) chunk = cap;
  if (chunk < 64) chunk = 64;
  return (int)chunk;
}

int64_t decode_ws_bytes(const aidn_sdpa* h, int64_t batch, int64_t seq_kv, int* chunk_out, int* nchunks_out) {
  const int chunk = pick_chunk(h, batch, seq_kv);
  const int64_t nchunks = (seq_kv + chunk - 1) / chunk;
  if (chunk_out) *chunk_out = chunk;
  if (nchunks_out) *nchunks_out = (int)nchunks;
  if (nchunks <= 1) return 0;
  return align_up(batch * h->head_count * nchunks * (h->d.head_dim + 2) * (int64_t)sizeof(float), 256);
}

// What a decode can use: equal shares of all keys, for sequences with lengths, may take more than it needs.
int64_t decode_ws_most(const aidn_sdpa* h, int64_t batch, int64_t seq_kv) {
  aidn::DecodePlan chunks = {0, 0, 1, 0};
  const int64_t need = decode_ws_bytes(h, batch, seq_kv, &chunks.chunk, &chunks.nchunks);
  if (need == 0 || h->d.decode_chunk > 0 || batch > 0x7fffffff) return need;
  aidn::SdpaParams p;
  std::memset(&p, 0, sizeof(p));
  p.batch = (int32_t)batch;
  p.seq_q = 1;
  p.seq_kv = seq_kv;
  p.head_dim = h->d.head_dim;
  p.group = h->group;
  p.head_count = h->head_count;
  p.ks[2] = 1;   // (any layout: the one that takes the most)
  int ctas = 0;
  const int64_t stream = align_up(aidn::decode_stream_bytes(p, h->d.qkv_dtype, h->num_sms, chunks, &ctas), 256);
  return need > stream ? need : stream;
}

// Workspace of the split tcgen05 prefill for these sizes, 0 when it would not be split.
int64_t prefill_split_need(const aidn_sdpa* h, int64_t batch, int64_t seq_q, int64_t seq_kv) {
  aidn::SdpaParams p;
  std::memset(&p, 0, sizeof(p));
  p.batch = (int)batch;
  p.num_q_heads = h->d.num_q_heads;
  p.head_count = h->head_count;
  p.group = h->group;
  p.seq_q = seq_q;
  p.seq_kv = seq_kv;
  p.head_dim = h->d.head_dim;
  const int splits = aidn::prefill_splits(p, h->num_sms);
  return splits > 1 ? align_up(aidn::prefill_split_bytes(p, splits), 256) : 0;
}

bool aligned16(const void* ptr, const int64_t* stride, size_t esz) {
  if ((uintptr_t)ptr % 16 != 0) return false;
  for (int i = 0; i < 3; ++i)
    if ((stride[i] * (int64_t)esz) % 16 != 0) return false;
  return true;
}

void dense_strides(int64_t* s, int64_t heads, int64_t seq, int64_t d) {
  s[2] = d;
  s[1] = seq * d;
  s[0] = heads * seq * d;
}

bool all_zero(const int64_t* s) { return s[0] == 0 && s[1] == 0 && s[2] == 0; }

}  // namespace

extern "C" {

const char* aidn_sdpa_last_error(void) { return g_err; }

int aidn_sdpa_device_supported(int32_t device) {
  int major = 0;
  if (cudaDeviceGetAttribute(&major, cudaDevAttrComputeCapabilityMajor, device) != cudaSuccess) {
    cudaGetLastError();
    return 0;
  }
  return major == 10 ? 1 : 0;
}

int aidn_sdpa_create(const aidn_sdpa_desc* desc, aidn_sdpa_t* out) {
  g_err[0] = 0;
  if (!desc || !out) return fail(AIDN_EINVAL, "create: null argument");
  *out = nullptr;
  const aidn_sdpa_desc& d = *desc;
  if (d.qkv_dtype < AIDN_F32 || d.qkv_dtype > AIDN_BF16) return fail(AIDN_EINVAL, "create: unknown qkv_dtype %d", d.qkv_dtype);
  if (d.out_dtype != AIDN_F32 && d.out_dtype != d.qkv_dtype)
    return fail(AIDN_EINVAL, "create: out_dtype must be fp32 or equal to qkv_dtype");
  if (d.head_dim <= 0 || d.head_dim > 256) return fail(AIDN_EINVAL, "create: head_dim %d outside [1,256]", d.head_dim);
  if (d.num_q_heads <= 0 || d.num_kv_heads <= 0 || d.num_q_heads % d.num_kv_heads != 0)
    return fail(AIDN_EINVAL, "create: numHeads (%d) must be a positive multiple of numKVHeads (%d)", d.num_q_heads,
                d.num_kv_heads);
  if (d.mask_kind < AIDN_MASK_NONE || d.mask_kind > AIDN_MASK_ADD_F32) return fail(AIDN_EINVAL, "create: unknown mask_kind");
  if (d.path < AIDN_PATH_AUTO || d.path > AIDN_PATH_PREFILL_SM100) return fail(AIDN_EINVAL, "create: unknown path");
  if (!(d.softcap >= 0.f)) return fail(AIDN_EINVAL, "create: softcap must be >= 0");
  const int group = d.num_q_heads / d.num_kv_heads;
  const int head_count = d.head_count > 0 ? d.head_count : d.num_q_heads - d.head_begin;
  if (d.head_begin < 0 || head_count <= 0 || d.head_begin + head_count > d.num_q_heads)
    return fail(AIDN_EINVAL, "create: head shard [%d,%d) outside [0,%d)", d.head_begin, d.head_begin + head_count,
                d.num_q_heads);
  if (d.head_begin % group != 0 || head_count % group != 0)
    return fail(AIDN_EINVAL, "create: a head shard must cover whole KV groups (group size %d)", group);
  if (d.decode_chunk < 0 || (d.decode_chunk > 0 && d.decode_chunk % 8 != 0))
    return fail(AIDN_EINVAL, "create: decode_chunk must be 0 or a positive multiple of 8");

  int cur = -1;
  cudaError_t e = cudaGetDevice(&cur);
  if (e != cudaSuccess) return fail_cuda(e, "create: cudaGetDevice");
  if (cur != d.device) return fail(AIDN_EINVAL, "create: desc.device (%d) is not the current device (%d)", d.device, cur);
  if (!aidn_sdpa_device_supported(d.device))
    return fail(AIDN_EUNSUPPORTED, "create: device %d is not compute capability 10.x (this library carries sm_100a code only)",
                d.device);

  aidn_sdpa* h = new (std::nothrow) aidn_sdpa();
  if (!h) return fail(AIDN_ECUDA, "create: out of host memory");
  h->d = d;
  h->group = group;
  h->head_count = head_count;
  h->status_dev = nullptr;
  h->scratch = nullptr;
  h->scratch_bytes = 0;
  h->last_path = AIDN_PATH_AUTO;
  h->last_launches = 0;
  h->debug = nullptr;
  h->debug_mode = 0;
  h->num_sms = 0;
  h->kv8_raised = 0;
  std::memset(&h->prefill_maps, 0, sizeof(h->prefill_maps));
  e = cudaDeviceGetAttribute(&h->num_sms, cudaDevAttrMultiProcessorCount, d.device);
  if (e == cudaSuccess) e = cudaMalloc(&h->status_dev, 4 * sizeof(int32_t));
  if (e == cudaSuccess) e = cudaMemset(h->status_dev, 0, 4 * sizeof(int32_t));
  if (e != cudaSuccess) {
    if (h->status_dev) cudaFree(h->status_dev);
    delete h;
    return fail_cuda(e, "create: status word");
  }
  if (d.max_batch > 0 && d.max_seq_kv > 0) {
    const int64_t bytes = decode_ws_bytes(h, d.max_batch, d.max_seq_kv, nullptr, nullptr);
    if (bytes > 0) {
      e = cudaMalloc(&h->scratch, (size_t)bytes);
      if (e != cudaSuccess) {
        cudaFree(h->status_dev);
        delete h;
        return fail_cuda(e, "create: decode scratch");
      }
      h->scratch_bytes = bytes;
    }
  }
  *out = h;
  return AIDN_OK;
}

int aidn_sdpa_destroy(aidn_sdpa_t h) {
  if (!h) return AIDN_OK;
  if (h->scratch) cudaFree(h->scratch);
  if (h->status_dev) cudaFree(h->status_dev);
  delete h;
  return AIDN_OK;
}

int64_t aidn_sdpa_workspace_bytes(aidn_sdpa_t h, int64_t batch, int64_t seq_q, int64_t seq_kv) {
  if (!h || batch <= 0 || seq_q <= 0 || seq_kv <= 0) {
    fail(AIDN_EINVAL, "workspace_bytes: bad argument");
    return -1;
  }
  if (h->d.path == AIDN_PATH_GENERIC) return 0;
  // the decode kernel's partial results, or those of a tcgen05 prefill with fewer work items than SMs (which runs without
  // a workspace too, only slower)
  int64_t need = 0;
  if (seq_q == 1 && h->d.path != AIDN_PATH_PREFILL_SM100 && aidn::decode_supported(h->d.qkv_dtype, h->d.head_dim))
    need = decode_ws_most(h, batch, seq_kv);
  else if (h->d.path != AIDN_PATH_DECODE && h->d.qkv_dtype != AIDN_F32 && (h->d.head_dim == 64 || h->d.head_dim == 128) &&
           batch <= 65535)
    need = prefill_split_need(h, batch, seq_q, seq_kv);
  return need;
}

int aidn_sdpa_last_path(aidn_sdpa_t h) { return h ? h->last_path : -1; }
int aidn_sdpa_last_launch_count(aidn_sdpa_t h) { return h ? h->last_launches : -1; }

// Test and development hook, declared in include/aidn_sdpa_debug.h.
int aidn_sdpa_debug_set(aidn_sdpa_t h, float* buf, int mode) {
  if (!h) {
    g_expire_qkv = mode == 3;
    g_expire_linear = mode == 5;
    return mode == 0 || mode == 3 || mode == 5 ? AIDN_OK : AIDN_EINVAL;
  }
  h->debug = buf;
  h->debug_mode = (buf || mode == 3) ? mode : 0;
  return AIDN_OK;
}

int aidn_sdpa_poll(aidn_sdpa_t h, void* cu_stream) {
  g_err[0] = 0;
  if (!h) return fail(AIDN_EINVAL, "poll: null handle");
  cudaError_t e = cudaStreamSynchronize((cudaStream_t)cu_stream);
  if (e != cudaSuccess) return fail_cuda(e, "poll: stream");
  int32_t st = 0;
  e = cudaMemcpy(&st, h->status_dev, sizeof(st), cudaMemcpyDeviceToHost);
  if (e != cudaSuccess) return fail_cuda(e, "poll: status read");
  if (st != 0) {
    cudaMemset(h->status_dev, 0, 4 * sizeof(int32_t));
    if (st & aidn::kStatusTimeout)
      return fail(AIDN_ETIMEOUT, "poll: a kernel gave up a bounded wait (status word 0x%x)", st);
    return fail(AIDN_EINVAL, "poll: a block-table entry outside [0, num_blocks) was skipped (status word 0x%x)", st);
  }
  return AIDN_OK;
}

}  // extern "C"

namespace {

// Validates a launch request and flattens it into the kernels' parameter block (shared by the forward launches and
// the backward).
int build_params(aidn_sdpa_t h, const aidn_sdpa_args* a, const aidn_paged_kv* pg, aidn::SdpaParams& p) {
  g_err[0] = 0;
  if (!h || !a) return fail(AIDN_EINVAL, "launch: null argument");
  const aidn_sdpa_desc& d = h->d;
  if (!a->q || !a->k || !a->v || !a->out) return fail(AIDN_EINVAL, "launch: null tensor pointer");
  if (a->batch <= 0 || a->seq_q <= 0 || a->seq_kv <= 0)
    return fail(AIDN_EINVAL, "launch: attention dimensions must be positive");
  if (a->batch > 65535) return fail(AIDN_EINVAL, "launch: batch above 65535");
  if (d.emit_lse && !a->lse) return fail(AIDN_EINVAL, "launch: emit_lse set but lse pointer is null");
  if (d.mask_kind != AIDN_MASK_NONE && !a->mask) return fail(AIDN_EINVAL, "launch: mask_kind set but mask pointer is null");
  if (a->scale < 0.f || std::isnan(a->scale)) return fail(AIDN_EINVAL, "launch: scale must be >= 0");

  std::memset(&p, 0, sizeof(p));
  p.q = a->q;
  p.k = a->k;
  p.v = a->v;
  p.out = a->out;
  p.lse = d.emit_lse ? a->lse : nullptr;
  p.weights = a->weights;
  if (a->peer_count < 0 || a->peer_count > AIDN_MAX_PEERS) return fail(AIDN_EINVAL, "launch: peer_count out of range");
  p.peer_count = a->peer_count;
  for (int i = 0; i < a->peer_count; ++i) {
    if (!a->peer_out[i]) return fail(AIDN_EINVAL, "launch: peer_out[%d] is null", i);
    p.peer_out[i] = a->peer_out[i];
  }
  p.mask = d.mask_kind != AIDN_MASK_NONE ? a->mask : nullptr;
  p.mask_kind = d.mask_kind;
  p.kv_len = a->kv_len;
  for (int i = 0; i < 4; ++i) p.mask_stride[i] = a->mask_stride[i];
  p.seq_q = a->seq_q;
  p.seq_kv = a->seq_kv;
  p.batch = (int)a->batch;
  p.num_q_heads = d.num_q_heads;
  p.num_kv_heads = d.num_kv_heads;
  p.group = h->group;
  p.head_begin = d.head_begin;
  p.head_count = h->head_count;
  p.head_dim = d.head_dim;
  p.causal = d.causal ? 1 : 0;
  p.causal_offset = d.causal_bottom_right ? (a->seq_kv - a->seq_q) : d.causal_offset;
  p.out_f32 = d.out_dtype == AIDN_F32 ? 1 : 0;
  p.scale = a->scale > 0.f ? a->scale : 1.0f / std::sqrt((float)d.head_dim);
  p.softcap = d.softcap;
  p.status = h->status_dev;
  p.no_tcgen05 = d.path == AIDN_PATH_GENERIC ? 1 : 0;
  p.expire = h->debug_mode == 3 ? 1 : 0;
  const int64_t D = d.head_dim;
  if (all_zero(a->q_stride)) dense_strides(p.qs, d.num_q_heads, a->seq_q, D);
  else std::memcpy(p.qs, a->q_stride, sizeof(p.qs));
  if (pg) {
    if (!pg->block_table) return fail(AIDN_EINVAL, "launch_paged: null block table");
    if (pg->block_size <= 0) return fail(AIDN_EINVAL, "launch_paged: block_size must be positive");
    if (pg->num_blocks < 0 || pg->block_table_stride < 0) return fail(AIDN_EINVAL, "launch_paged: negative num_blocks or stride");
    if (a->seq_kv > 0x7fffffffll) return fail(AIDN_EINVAL, "launch_paged: seq_kv above 2^31-1");
    if (a->batch > 1 && pg->block_table_stride * pg->block_size < a->seq_kv && !a->kv_len)
      return fail(AIDN_EINVAL, "launch_paged: block_table_stride (%lld) holds fewer than seq_kv keys",
                  (long long)pg->block_table_stride);
    // kv_len lives on the device and cannot be checked here: no key beyond what a table row can address is ever
    // looked up, whatever kv_len[b] says (it would read the next sequence's row, or past the table)
    if (a->batch > 1 && pg->block_table_stride * pg->block_size < p.seq_kv) p.seq_kv = pg->block_table_stride * pg->block_size;
    p.block_table = pg->block_table;
    p.bt_stride = pg->block_table_stride;
    p.block_size = pg->block_size;
    p.block_shift = -1;
    for (int sft = 0; sft < 31; ++sft)
      if ((1 << sft) == pg->block_size) p.block_shift = sft;
    p.num_blocks = pg->num_blocks;
    const int64_t pool_dense[3] = {0, D, (int64_t)d.num_kv_heads * D};
    std::memcpy(p.ks, all_zero(a->k_stride) ? pool_dense : a->k_stride, sizeof(p.ks));
    std::memcpy(p.vs, all_zero(a->v_stride) ? pool_dense : a->v_stride, sizeof(p.vs));
    p.ks[0] = p.vs[0] = 0;
  } else {
    if (all_zero(a->k_stride)) dense_strides(p.ks, d.num_kv_heads, a->seq_kv, D);
    else std::memcpy(p.ks, a->k_stride, sizeof(p.ks));
    if (all_zero(a->v_stride)) dense_strides(p.vs, d.num_kv_heads, a->seq_kv, D);
    else std::memcpy(p.vs, a->v_stride, sizeof(p.vs));
  }
  if (all_zero(a->o_stride)) dense_strides(p.os, d.num_q_heads, a->seq_q, D);
  else std::memcpy(p.os, a->o_stride, sizeof(p.os));
  for (int i = 0; i < 3; ++i)
    if (p.qs[i] < 0 || p.ks[i] < 0 || p.vs[i] < 0 || p.os[i] < 0) return fail(AIDN_EINVAL, "launch: negative stride");
  if (p.head_count > 65535) return fail(AIDN_EINVAL, "launch: more than 65535 heads in one shard");
  return AIDN_OK;
}

// The launch shared by aidn_sdpa_launch (pg == nullptr) and aidn_sdpa_launch_paged.
int launch_common(aidn_sdpa_t h, const aidn_sdpa_args* a, const aidn_paged_kv* pg, void* cu_stream) {
  aidn::SdpaParams p;
  const int rc = build_params(h, a, pg, p);
  if (rc != AIDN_OK) return rc;
  const aidn_sdpa_desc& d = h->d;
  cudaStream_t stream = (cudaStream_t)cu_stream;
  const int64_t D = d.head_dim;

  const size_t esz = elem_size(d.qkv_dtype);
  const bool vec_ok = aligned16(p.q, p.qs, esz) && aligned16(p.k, p.ks, esz) && aligned16(p.v, p.vs, esz);
  const bool decode_ok = a->seq_q == 1 && aidn::decode_supported(d.qkv_dtype, d.head_dim) && vec_ok;
  const char* why = "";
  const bool prefill_ok = aidn::prefill_sm100_supported(p, d.qkv_dtype, &why);

  int path = d.path;
  if (path == AIDN_PATH_AUTO) path = decode_ok ? AIDN_PATH_DECODE : (prefill_ok ? AIDN_PATH_PREFILL_SM100 : AIDN_PATH_GENERIC);
  if (p.weights) {
    // the probabilities are written by the fp32 kernel only
    if (d.path != AIDN_PATH_AUTO && d.path != AIDN_PATH_GENERIC)
      return fail(AIDN_EUNSUPPORTED, "launch: attention weights are produced by the generic kernel (desc.path AUTO or GENERIC)");
    if ((uintptr_t)p.weights % 4 != 0) return fail(AIDN_EINVAL, "launch: weights must be 4-byte aligned");
    if (pg) return fail(AIDN_EUNSUPPORTED, "launch: attention weights over paged K/V are not defined");
    path = AIDN_PATH_GENERIC;
  }
  if (p.peer_count > 0) {
    // the stores to the other devices are issued by the tcgen05 kernel's epilogue
    if (path != AIDN_PATH_PREFILL_SM100 || !prefill_ok)
      return fail(AIDN_EUNSUPPORTED, "launch: peer_out needs the tcgen05 prefill kernel (16-bit inputs, head_dim 64 or 128)");
    if (a->gather_output) return fail(AIDN_EINVAL, "launch: peer_out and gather_output are two ways to the same result");
  }
  if (path == AIDN_PATH_DECODE && !decode_ok)
    return fail(AIDN_EUNSUPPORTED,
                "launch: decode kernel needs seq_q == 1, head_dim 64/128 (256 for 16-bit) and 16-byte aligned Q/K/V rows");
  if (path == AIDN_PATH_PREFILL_SM100 && !prefill_ok) return fail(AIDN_EUNSUPPORTED, "launch: %s", why);

  cudaError_t e = cudaSuccess;
  int launches = 0;
  if (path == AIDN_PATH_DECODE) {
    int chunk = 0, nchunks = 0;
    const int64_t need = decode_ws_bytes(h, a->batch, a->seq_kv, &chunk, &nchunks);
    float* ws = nullptr;
    if (need > 0) {
      if (a->workspace) {
        if (a->workspace_bytes < need)
          return fail(AIDN_EWORKSPACE, "launch: workspace of %lld bytes, need %lld", (long long)a->workspace_bytes,
                      (long long)need);
        if ((uintptr_t)a->workspace % 16 != 0) return fail(AIDN_EINVAL, "launch: workspace must be 16-byte aligned");
        ws = static_cast<float*>(a->workspace);
      } else if (h->scratch && h->scratch_bytes >= need) {
        ws = static_cast<float*>(h->scratch);
      } else {
        return fail(AIDN_EWORKSPACE, "launch: decode needs %lld bytes of workspace and the handle owns %lld",
                    (long long)need, (long long)h->scratch_bytes);
      }
    }
    aidn::DecodePlan plan = {chunk, nchunks, 1, 0};
    if (d.decode_chunk == 0 && nchunks > 1) {
      int ctas = 0;
      const int64_t stream_need = p.kv_len ? aidn::decode_stream_bytes(p, d.qkv_dtype, h->num_sms, plan, &ctas) : 0;
      if (stream_need > 0 && (ws == a->workspace ? a->workspace_bytes : h->scratch_bytes) >= stream_need) plan.stream_ctas = ctas;   // with less: as without
      else aidn::decode_plan_clusters(p, d.qkv_dtype, h->num_sms, &plan);
    }
    e = aidn::launch_decode(p, d.qkv_dtype, plan, ws, stream, &launches);
  } else if (path == AIDN_PATH_PREFILL_SM100) {
    // Keys of few items are split when the caller's workspace holds the partial results; without one they are not.  The
    // handle's own scratch is not used: it belongs to decode calls, which may be running on another stream.
    int splits = aidn::prefill_splits(p, h->num_sms);
    if (!a->workspace || (uintptr_t)a->workspace % 16 != 0 || h->debug || h->debug_mode) splits = 1;
    if (splits > 1 && a->workspace_bytes < aidn::prefill_split_bytes(p, splits)) splits = 1;
    e = aidn::launch_prefill_sm100(p, d.qkv_dtype, stream, h->status_dev + 1, h->num_sms, h->debug, h->debug_mode,
                                   &h->prefill_maps, splits, static_cast<float*>(a->workspace), &why);
    launches = splits > 1 ? 2 : 1;
    if (e != cudaSuccess && why[0]) return fail(AIDN_ECUDA, "launch: %s (%s)", why, cudaGetErrorName(e));
  } else {
    e = aidn::launch_generic(p, d.qkv_dtype, stream);
    launches = 1;
  }
  if (e != cudaSuccess) return fail_cuda(e, "launch");
  h->last_path = path;
  h->last_launches = launches;

  if (a->gather_output) {
    if (!d.nccl_comm) return fail(AIDN_ENCCL, "launch: gather_output needs desc.nccl_comm");
    std::call_once(g_nccl_once, load_nccl);
    if (!g_nccl.ok) return fail(AIDN_ENCCL, "launch: libnccl.so.2 could not be loaded");
    int nranks = 0, rank = -1;
    if (g_nccl.CommCount(d.nccl_comm, &nranks) != 0 || g_nccl.CommUserRank(d.nccl_comm, &rank) != 0)
      return fail(AIDN_ENCCL, "launch: cannot query the communicator");
    if (h->head_count * nranks != d.num_q_heads || d.head_begin != rank * h->head_count)
      return fail(AIDN_EINVAL, "launch: gather needs %d equal consecutive head shards, rank r owning heads [r*n,(r+1)*n)", nranks);
    if (p.os[2] != D || p.os[1] != a->seq_q * D)
      return fail(AIDN_EINVAL, "launch: gather needs a dense [B,H,S,D] output");
    const size_t osz = p.out_f32 ? 4 : 2;
    const int dt = p.out_f32 ? kNcclFloat32 : (d.qkv_dtype == AIDN_F16 ? kNcclFloat16 : kNcclBfloat16);
    const size_t count = (size_t)h->head_count * (size_t)a->seq_q * (size_t)D;
    int rc = g_nccl.GroupStart();
    for (int64_t b = 0; b < a->batch && rc == 0; ++b) {
      char* recv = static_cast<char*>(a->out) + (size_t)b * p.os[0] * osz;
      rc = g_nccl.AllGather(recv + (size_t)rank * count * osz, recv, count, dt, d.nccl_comm, stream);
    }
    const int rc2 = g_nccl.GroupEnd();
    if (rc == 0) rc = rc2;
    if (rc != 0)
      return fail(AIDN_ENCCL, "launch: ncclAllGather failed: %s", g_nccl.GetErrorString ? g_nccl.GetErrorString(rc) : "?");
    h->last_launches += 1;
  }
  return post_launch_check(stream, "aidn_sdpa_launch", h->status_dev);
}

}  // namespace

extern "C" {

int aidn_sdpa_launch(aidn_sdpa_t h, const aidn_sdpa_args* a, void* cu_stream) {
  return launch_common(h, a, nullptr, cu_stream);
}

int aidn_sdpa_launch_paged(aidn_sdpa_t h, const aidn_sdpa_args* a, const aidn_paged_kv* paged, void* cu_stream) {
  if (!paged) {
    g_err[0] = 0;
    return fail(AIDN_EINVAL, "launch_paged: null aidn_paged_kv");
  }
  return launch_common(h, a, paged, cu_stream);
}

int64_t aidn_sdpa_backward_workspace_bytes(aidn_sdpa_t h, int64_t batch, int64_t seq_q) {
  if (!h || batch <= 0 || seq_q <= 0) {
    fail(AIDN_EINVAL, "backward_workspace_bytes: bad argument");
    return -1;
  }
  int64_t bytes = align_up(batch * h->head_count * seq_q * (int64_t)sizeof(float), 256);   // delta
  if (h->d.qkv_dtype != AIDN_F32 && h->d.out_dtype == AIDN_F32)                              // dO in the input dtype
    bytes += align_up(batch * h->head_count * seq_q * (int64_t)h->d.head_dim * 2, 256);
  return bytes;
}

int aidn_sdpa_backward(aidn_sdpa_t h, const aidn_sdpa_bwd_args* a, void* cu_stream) {
  g_err[0] = 0;
  if (!h || !a) return fail(AIDN_EINVAL, "backward: null argument");
  if (!a->dout || !a->dq || !a->dk || !a->dv) return fail(AIDN_EINVAL, "backward: null gradient pointer");
  if (!a->fwd.lse) return fail(AIDN_EINVAL, "backward: the forward's log-sum-exp (fwd.lse) is required");
  if (h->d.softcap > 0.f) return fail(AIDN_EUNSUPPORTED, "backward: logit softcap is not differentiated here");
  aidn::BwdParams bp;
  const int rc = build_params(h, &a->fwd, a->paged, bp.p);
  if (rc != AIDN_OK) return rc;
  bp.p.lse = a->fwd.lse;   // read here, whatever desc.emit_lse says
  bp.p.weights = nullptr;
  const int64_t need = aidn_sdpa_backward_workspace_bytes(h, a->fwd.batch, a->fwd.seq_q);
  if (!a->fwd.workspace || a->fwd.workspace_bytes < need)
    return fail(AIDN_EWORKSPACE, "backward: workspace of %lld bytes, need %lld", (long long)a->fwd.workspace_bytes, (long long)need);
  if ((uintptr_t)a->fwd.workspace % 16 != 0) return fail(AIDN_EINVAL, "backward: workspace must be 16-byte aligned");
  bp.dout = a->dout;
  if (all_zero(a->do_stride)) std::memcpy(bp.dos, bp.p.os, sizeof(bp.dos));
  else std::memcpy(bp.dos, a->do_stride, sizeof(bp.dos));
  for (int i = 0; i < 3; ++i)
    if (bp.dos[i] < 0) return fail(AIDN_EINVAL, "backward: negative stride");
  bp.dq = a->dq; bp.dk = a->dk; bp.dv = a->dv;
  bp.delta = static_cast<float*>(a->fwd.workspace);
  bp.dout_t = nullptr;
  if (h->d.qkv_dtype != AIDN_F32 && h->d.out_dtype == AIDN_F32)
    bp.dout_t = static_cast<char*>(a->fwd.workspace) +
                align_up(a->fwd.batch * h->head_count * a->fwd.seq_q * (int64_t)sizeof(float), 256);
  bp.no_tcgen05 = h->d.path == AIDN_PATH_GENERIC ? 1 : 0;
  bp.round_dout = 0;
  bp.expire = h->debug_mode == 3 ? 1 : 0;
  int launches = 0, used_tcgen05 = 0;
  cudaError_t e = aidn::launch_backward(bp, h->d.qkv_dtype, (cudaStream_t)cu_stream, &launches, &used_tcgen05);
  if (e != cudaSuccess) return fail_cuda(e, "backward");
  h->last_path = used_tcgen05 ? AIDN_PATH_PREFILL_SM100 : AIDN_PATH_GENERIC;
  h->last_launches = launches;
  return post_launch_check((cudaStream_t)cu_stream, "aidn_sdpa_backward", h->status_dev);
}

// Decode for callers that cannot allocate device memory (no handle, no workspace): see include/aidn_sdpa.h.
int aidn_sdpa_decode_noalloc(const aidn_sdpa_desc* desc, const aidn_sdpa_args* a, void* cu_stream) {
  g_err[0] = 0;
  if (!desc || !a) return fail(AIDN_EINVAL, "decode_noalloc: null argument");
  const aidn_sdpa_desc& d = *desc;
  if (d.qkv_dtype < AIDN_F32 || d.qkv_dtype > AIDN_BF16) return fail(AIDN_EINVAL, "decode_noalloc: unknown qkv_dtype");
  if (d.out_dtype != AIDN_F32 && d.out_dtype != d.qkv_dtype)
    return fail(AIDN_EINVAL, "decode_noalloc: out_dtype must be fp32 or equal to qkv_dtype");
  if (d.num_q_heads <= 0 || d.num_kv_heads <= 0 || d.num_q_heads % d.num_kv_heads != 0)
    return fail(AIDN_EINVAL, "decode_noalloc: numHeads must be a positive multiple of numKVHeads");
  if (d.mask_kind < AIDN_MASK_NONE || d.mask_kind > AIDN_MASK_ADD_F32) return fail(AIDN_EINVAL, "decode_noalloc: unknown mask_kind");
  if (!(d.softcap >= 0.f)) return fail(AIDN_EINVAL, "decode_noalloc: softcap must be >= 0");
  if (d.decode_chunk < 0 || (d.decode_chunk > 0 && d.decode_chunk % 8 != 0))
    return fail(AIDN_EINVAL, "decode_noalloc: decode_chunk must be 0 or a positive multiple of 8");
  int cur = -1;
  cudaError_t ce = cudaGetDevice(&cur);
  if (ce != cudaSuccess) return fail_cuda(ce, "decode_noalloc: cudaGetDevice");
  if (cur != d.device)
    return fail(AIDN_EINVAL, "decode_noalloc: desc.device (%d) is not the current device (%d)", d.device, cur);
  if (!aidn_sdpa_device_supported(d.device))
    return fail(AIDN_EUNSUPPORTED, "decode_noalloc: device %d is not compute capability 10.x", d.device);
  aidn_sdpa tmp;  // on the stack: only the fields the chunk heuristic reads
  std::memset(&tmp, 0, sizeof(tmp));
  tmp.d = d;
  tmp.group = d.num_q_heads / d.num_kv_heads;
  tmp.head_count = d.head_count > 0 ? d.head_count : d.num_q_heads - d.head_begin;
  if (d.head_begin < 0 || tmp.head_count <= 0 || d.head_begin + tmp.head_count > d.num_q_heads ||
      d.head_begin % tmp.group != 0 || tmp.head_count % tmp.group != 0)
    return fail(AIDN_EINVAL, "decode_noalloc: the head shard must lie inside the tensor and cover whole KV groups");
  if (tmp.head_count > 65535) return fail(AIDN_EINVAL, "decode_noalloc: more than 65535 heads in one shard");
  if (!a->q || !a->k || !a->v || !a->out) return fail(AIDN_EINVAL, "decode_noalloc: null tensor pointer");
  if (a->batch <= 0 || a->batch > 65535 || a->seq_kv <= 0) return fail(AIDN_EINVAL, "decode_noalloc: bad batch or seq_kv");
  if (a->seq_q != 1) return fail(AIDN_EUNSUPPORTED, "decode_noalloc: seq_q must be 1");
  if (d.emit_lse && !a->lse) return fail(AIDN_EINVAL, "decode_noalloc: emit_lse set but lse pointer is null");
  if (d.mask_kind != AIDN_MASK_NONE && !a->mask) return fail(AIDN_EINVAL, "decode_noalloc: mask_kind set but mask pointer is null");
  if (a->scale < 0.f || std::isnan(a->scale)) return fail(AIDN_EINVAL, "decode_noalloc: scale must be >= 0");
  if (!aidn::decode_supported(d.qkv_dtype, d.head_dim))
    return fail(AIDN_EUNSUPPORTED, "decode_noalloc: head_dim must be 64 or 128 (256 for 16-bit inputs)");

  aidn::SdpaParams p;
  std::memset(&p, 0, sizeof(p));
  p.q = a->q; p.k = a->k; p.v = a->v; p.out = a->out;
  p.lse = d.emit_lse ? a->lse : nullptr;
  p.mask = d.mask_kind != AIDN_MASK_NONE ? a->mask : nullptr;
  p.mask_kind = d.mask_kind;
  p.kv_len = a->kv_len;
  for (int i = 0; i < 4; ++i) p.mask_stride[i] = a->mask_stride[i];
  p.seq_q = 1;
  p.seq_kv = a->seq_kv;
  p.batch = (int)a->batch;
  p.num_q_heads = d.num_q_heads;
  p.num_kv_heads = d.num_kv_heads;
  p.group = tmp.group;
  p.head_begin = d.head_begin;
  p.head_count = tmp.head_count;
  p.head_dim = d.head_dim;
  p.causal = d.causal ? 1 : 0;
  p.causal_offset = d.causal_bottom_right ? (a->seq_kv - 1) : d.causal_offset;
  p.out_f32 = d.out_dtype == AIDN_F32 ? 1 : 0;
  p.scale = a->scale > 0.f ? a->scale : 1.0f / std::sqrt((float)d.head_dim);
  p.softcap = d.softcap;
  p.status = nullptr;
  const int64_t D = d.head_dim;
  if (all_zero(a->q_stride)) dense_strides(p.qs, d.num_q_heads, 1, D); else std::memcpy(p.qs, a->q_stride, sizeof(p.qs));
  if (all_zero(a->k_stride)) dense_strides(p.ks, d.num_kv_heads, a->seq_kv, D); else std::memcpy(p.ks, a->k_stride, sizeof(p.ks));
  if (all_zero(a->v_stride)) dense_strides(p.vs, d.num_kv_heads, a->seq_kv, D); else std::memcpy(p.vs, a->v_stride, sizeof(p.vs));
  if (all_zero(a->o_stride)) dense_strides(p.os, d.num_q_heads, 1, D); else std::memcpy(p.os, a->o_stride, sizeof(p.os));
  for (int i = 0; i < 3; ++i)
    if (p.qs[i] < 0 || p.ks[i] < 0 || p.vs[i] < 0 || p.os[i] < 0) return fail(AIDN_EINVAL, "decode_noalloc: negative stride");
  const size_t esz = elem_size(d.qkv_dtype);
  if (!(aligned16(p.q, p.qs, esz) && aligned16(p.k, p.ks, esz) && aligned16(p.v, p.vs, esz)))
    return fail(AIDN_EUNSUPPORTED, "decode_noalloc: Q/K/V rows must be 16-byte aligned");

  int chunk = 0, nchunks = 0;
  const int64_t need = decode_ws_bytes(&tmp, a->batch, a->seq_kv, &chunk, &nchunks);
  const int64_t have = aidn::decode_static_scratch_bytes();
  if (need > have)
    return fail(AIDN_EWORKSPACE,
                "decode_noalloc: this shape needs %lld bytes of split-KV scratch but the library's static array holds %lld; "
                "lower batch*heads*ceil(seq_kv/chunk) (a larger decode_chunk helps) or use aidn_sdpa_launch with a workspace",
                (long long)need, (long long)have);
  int launches = 0;
  cudaError_t e = aidn::launch_decode_static(p, d.qkv_dtype, {chunk, nchunks, 1}, (cudaStream_t)cu_stream, &launches);
  if (e != cudaSuccess) return fail_cuda(e, "decode_noalloc");
  return post_launch_check((cudaStream_t)cu_stream, "aidn_sdpa_decode_noalloc", nullptr);
}

int aidn_qkv_rope_cache(const aidn_qkv_rope_args* a, void* cu_stream) {
  g_err[0] = 0;
  const bool expire = g_expire_qkv;
  g_expire_qkv = false;
  if (!a) return fail(AIDN_EINVAL, "qkv_rope_cache: null argument");
  if (!a->input || !a->weights || !a->cosine || !a->sine || !a->query || !a->key_cache || !a->value_cache)
    return fail(AIDN_EINVAL, "qkv_rope_cache: null buffer");
  if (a->heads <= 0) return fail(AIDN_EINVAL, "qkv_rope_cache: heads must be > 0");
  if (a->kv_heads <= 0 || a->kv_heads > a->heads || a->heads % a->kv_heads != 0)
    return fail(AIDN_EINVAL, "qkv_rope_cache: kv_heads must divide heads");
  if (a->head_dim <= 0 || a->head_dim > 256 || a->head_dim % 2 != 0)
    return fail(AIDN_EINVAL, "qkv_rope_cache: head_dim must be even and in [2, 256]");
  if (a->tokens <= 0) return fail(AIDN_EINVAL, "qkv_rope_cache: tokens must be > 0");
  if (a->cache_capacity <= 0 || a->max_position <= 0) return fail(AIDN_EINVAL, "qkv_rope_cache: cache_capacity and max_position must be > 0");
  if (!a->positions && (a->position < 0 || (int64_t)a->position + a->tokens > a->max_position))
    return fail(AIDN_EINVAL, "qkv_rope_cache: position outside the cos/sin tables");
  if (!a->positions && !a->cache_rows && (int64_t)a->position + a->tokens > a->cache_capacity)
    return fail(AIDN_EINVAL, "qkv_rope_cache: position outside the cache");   /* ArgumentOutOfRangeException(position) */
  if (a->weight_dtype != AIDN_F32 && a->weight_dtype != AIDN_BF16) return fail(AIDN_EINVAL, "qkv_rope_cache: weights are fp32 or bf16");
  if (a->query_dtype < AIDN_F32 || a->query_dtype > AIDN_BF16 || a->cache_dtype < AIDN_F32 || a->cache_dtype > AIDN_BF16)
    return fail(AIDN_EINVAL, "qkv_rope_cache: unknown output dtype");
  const int64_t model = (int64_t)a->heads * a->head_dim;
  if (model % 8 != 0) return fail(AIDN_EUNSUPPORTED, "qkv_rope_cache: heads * head_dim must be a multiple of 8");
  if (model > aidn::qkv_rope_max_model())
    return fail(AIDN_EUNSUPPORTED, "qkv_rope_cache: heads * head_dim above %lld", (long long)aidn::qkv_rope_max_model());
  if ((uintptr_t)a->weights % 16 != 0 || (uintptr_t)a->input % 16 != 0)
    return fail(AIDN_EINVAL, "qkv_rope_cache: input and weights must be 16-byte aligned");
  // per-device facts, looked up once: this entry point has no handle to keep them in.  Unsynchronised on purpose:
  // two threads racing here write the same values (the lookups are idempotent), and g_sms is written last.
  static int g_sms[64] = {0};
  static int g_ok[64] = {0};
  int dev = -1;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return fail_cuda(e, "qkv_rope_cache: device query");
  if (dev < 0 || dev >= 64) return fail(AIDN_EUNSUPPORTED, "qkv_rope_cache: device ordinal %d", dev);
  if (g_sms[dev] == 0) {
    int sms_q = 0;
    e = cudaDeviceGetAttribute(&sms_q, cudaDevAttrMultiProcessorCount, dev);
    if (e != cudaSuccess) return fail_cuda(e, "qkv_rope_cache: device query");
    g_ok[dev] = aidn_sdpa_device_supported(dev);
    g_sms[dev] = sms_q;
  }
  const int sms = g_sms[dev];
  if (!g_ok[dev]) return fail(AIDN_EUNSUPPORTED, "qkv_rope_cache: device %d is not compute capability 10.x", dev);
  aidn::QkvRopeParams p;
  std::memset(&p, 0, sizeof(p));
  p.input = a->input; p.weights = a->weights; p.bias = a->bias; p.cosine = a->cosine; p.sine = a->sine;
  p.query = a->query; p.key_cache = a->key_cache; p.value_cache = a->value_cache;
  p.positions = a->positions; p.cache_rows = a->cache_rows;
  p.tokens = a->tokens; p.heads = a->heads; p.kv_heads = a->kv_heads; p.head_dim = a->head_dim;
  p.position = a->position; p.query_dtype = a->query_dtype; p.cache_dtype = a->cache_dtype;
  p.cache_capacity = a->cache_capacity; p.max_position = a->max_position; p.model = (int32_t)model;
  int launches = 0;
  e = aidn::launch_qkv_rope_cache(p, a->weight_dtype, sms, (cudaStream_t)cu_stream, &launches, expire);
  if (e != cudaSuccess) return fail_cuda(e, "qkv_rope_cache");
  const bool waits = launch_check_enabled() && aidn::qkv_rope_sm100_supported(p, a->weight_dtype);   // the kernel with bounded waits
  return post_launch_check((cudaStream_t)cu_stream, "aidn_qkv_rope_cache", waits ? aidn::qkv_rope_sm100_status() : nullptr, true);
}

int aidn_qkv_rope_poll(void* cu_stream) {
  g_err[0] = 0;
  cudaError_t e = cudaStreamSynchronize((cudaStream_t)cu_stream);
  if (e != cudaSuccess) return fail_cuda(e, "qkv_rope_poll: stream");
  int32_t* status = aidn::qkv_rope_sm100_status();
  if (!status) return fail(AIDN_ECUDA, "qkv_rope_poll: no status word in the current context");
  int32_t st = 0;
  e = cudaMemcpy(&st, status, sizeof(st), cudaMemcpyDeviceToHost);
  if (e != cudaSuccess) return fail_cuda(e, "qkv_rope_poll: status read");
  if (st == 0) return AIDN_OK;
  cudaMemset(status, 0, sizeof(st));
  return fail(AIDN_ETIMEOUT, "qkv_rope_poll: a kernel gave up a bounded wait (status word 0x%x)", st);
}

int aidn_rope_interleaved(const float* input, const float* cosine, const float* sine, float* output, int64_t rows,
                          int32_t head_dim, int32_t seq_len, int32_t start_position, void* cu_stream) {
  g_err[0] = 0;
  if (rows <= 0 || head_dim <= 0 || seq_len <= 0) return fail(AIDN_EINVAL, "rope_interleaved: rows, headDim and seqLen must be > 0");
  if (head_dim % 2 != 0) return fail(AIDN_EINVAL, "rope_interleaved: headDim must be even");
  if (start_position < 0) return fail(AIDN_EINVAL, "rope_interleaved: startPosition must be >= 0");
  if (!input || !cosine || !sine || !output) return fail(AIDN_EINVAL, "rope_interleaved: null buffer");
  if ((uintptr_t)input % 8 != 0 || (uintptr_t)output % 8 != 0) return fail(AIDN_EINVAL, "rope_interleaved: buffers must be 8-byte aligned");
  cudaError_t e = aidn::launch_rope_interleaved(input, cosine, sine, output, rows, head_dim, seq_len, start_position,
                                                (cudaStream_t)cu_stream);
  if (e != cudaSuccess) return fail_cuda(e, "rope_interleaved");
  return AIDN_OK;
}

int aidn_paged_kv_append(const void* new_keys, const void* new_values, void* key_pool, void* value_pool,
                         const int32_t* block_table, int64_t start_position, int64_t tokens, int32_t block_size,
                         int32_t num_blocks, int64_t row_bytes, void* cu_stream) {
  g_err[0] = 0;
  if (tokens < 0 || start_position < 0) return fail(AIDN_EINVAL, "paged_kv_append: newLen and the start position must be >= 0");
  if (tokens == 0) return AIDN_OK;
  if (!new_keys || !new_values || !key_pool || !value_pool || !block_table) return fail(AIDN_EINVAL, "paged_kv_append: null buffer");
  if (block_size <= 0 || num_blocks <= 0) return fail(AIDN_EINVAL, "paged_kv_append: block_size and num_blocks must be > 0");
  if (row_bytes <= 0 || row_bytes % 16 != 0) return fail(AIDN_EINVAL, "paged_kv_append: row_bytes must be a positive multiple of 16");
  if (start_position + tokens > (int64_t)num_blocks * block_size)
    return fail(AIDN_EINVAL, "paged_kv_append: the sequence would reach %lld tokens, above the pool capacity %lld",
                (long long)(start_position + tokens), (long long)num_blocks * block_size);   /* InvalidOperationException there */
  if ((uintptr_t)new_keys % 16 || (uintptr_t)new_values % 16 || (uintptr_t)key_pool % 16 || (uintptr_t)value_pool % 16)
    return fail(AIDN_EINVAL, "paged_kv_append: buffers must be 16-byte aligned");
  cudaError_t e = aidn::launch_paged_append(new_keys, new_values, key_pool, value_pool, block_table, start_position, tokens,
                                            block_size, num_blocks, row_bytes, (cudaStream_t)cu_stream);
  if (e != cudaSuccess) return fail_cuda(e, "paged_kv_append");
  return AIDN_OK;
}

// ---- paged K / V held in 8 bits --------------------------------------------------------------------------------------
namespace {
// The pool's parameter block; `op` names the call in messages.
int build_pool(const char* op, const aidn_kv8_cache* c, aidn::kv8::Pool& pool) {
  if (!c) return fail(AIDN_EINVAL, "%s: null aidn_kv8_cache", op);
  if (!c->key_pool || !c->value_pool || !c->key_scale || !c->value_scale || !c->block_table)
    return fail(AIDN_EINVAL, "%s: null pool, scales or block table", op);
  if (c->block_size <= 0 || c->block_size > 65536) return fail(AIDN_EINVAL, "%s: block_size %d outside [1,65536]", op, c->block_size);
  if (c->num_blocks < 0 || c->block_table_stride <= 0) return fail(AIDN_EINVAL, "%s: num_blocks must be >= 0 and block_table_stride > 0", op);
  if (c->kv_heads <= 0 || c->kv_heads > 65535) return fail(AIDN_EINVAL, "%s: kv_heads outside [1,65535]", op);
  if (c->head_dim <= 0 || c->head_dim > 256) return fail(AIDN_EINVAL, "%s: head_dim %d outside [1,256]", op, c->head_dim);
  if (c->head_dim % 8 != 0) return fail(AIDN_EUNSUPPORTED, "%s: head_dim %d is not a multiple of 8", op, c->head_dim);
  pool.k = c->key_pool;
  pool.v = c->value_pool;
  pool.k_scale = c->key_scale;
  pool.v_scale = c->value_scale;
  pool.table = c->block_table;
  pool.table_stride = c->block_table_stride;
  const int64_t D = c->head_dim, dense[3] = {c->block_size * (c->kv_heads * D), c->kv_heads * D, D};
  std::memcpy(pool.stride, all_zero(c->pool_stride) ? dense : c->pool_stride, sizeof(pool.stride));
  for (int i = 0; i < 3; ++i)
    if (pool.stride[i] < 0 || pool.stride[i] % 4 != 0) return fail(AIDN_EINVAL, "%s: pool strides must be multiples of 4 and not negative", op);
  if ((uintptr_t)c->key_pool % 4 != 0 || (uintptr_t)c->value_pool % 4 != 0 || (uintptr_t)c->key_scale % 4 != 0 || (uintptr_t)c->value_scale % 4 != 0)
    return fail(AIDN_EINVAL, "%s: pools and scales must be 4-byte aligned", op);
  if ((uintptr_t)c->block_table % 4 != 0) return fail(AIDN_EINVAL, "%s: the block table is not aligned to its entries", op);
  pool.num_blocks = c->num_blocks;
  pool.block_size = c->block_size;
  pool.kv_heads = c->kv_heads;
  pool.head_dim = c->head_dim;
  pool.block_shift = -1;
  for (int sft = 0; sft < 31; ++sft)
    if ((1 << sft) == c->block_size) pool.block_shift = sft;
  return AIDN_OK;
}
}  // namespace

int aidn_kv8_append(const aidn_kv8_cache* cache, const aidn_kv8_append_args* a, void* cu_stream) {
  g_err[0] = 0;
  aidn::kv8::Append p;
  std::memset(&p, 0, sizeof(p));
  const int rc = build_pool("kv8_append", cache, p.c);
  if (rc != AIDN_OK) return rc;
  if (!a) return fail(AIDN_EINVAL, "kv8_append: null argument");
  if (a->tokens < 0 || a->batch <= 0) return fail(AIDN_EINVAL, "kv8_append: tokens must be >= 0 and batch > 0");
  if (a->tokens > 0x7fffffffll) return fail(AIDN_EINVAL, "kv8_append: more than 2^31-1 tokens");
  if (a->dtype < AIDN_F32 || a->dtype > AIDN_BF16) return fail(AIDN_EINVAL, "kv8_append: unknown dtype %d", a->dtype);
  if (a->rope < AIDN_ROPE_NONE || a->rope > AIDN_ROPE_HALVES) return fail(AIDN_EINVAL, "kv8_append: unknown rotation %d", a->rope);
  if (!a->token_starts && a->tokens % a->batch != 0)
    return fail(AIDN_EINVAL, "kv8_append: %lld tokens are not the same number for each of %d sequences, and token_starts is null",
                (long long)a->tokens, a->batch);
  if (a->tokens == 0) return AIDN_OK;
  if (!a->key || !a->value || !a->start) return fail(AIDN_EINVAL, "kv8_append: null buffer");
  if (a->query && (!a->query_out || a->heads <= 0)) return fail(AIDN_EINVAL, "kv8_append: queries need query_out and heads > 0");
  if (a->rope != AIDN_ROPE_NONE && (!a->cosine || !a->sine || a->max_position < 0))
    return fail(AIDN_EINVAL, "kv8_append: a rotation needs cosine, sine and max_position >= 0");
  const int64_t D = cache->head_dim;
  const size_t esz = elem_size(a->dtype);
  const void* ptrs[] = {a->query, a->key, a->value, a->query_out, a->cosine, a->sine, a->start, a->token_starts, a->positions};
  const size_t align[] = {esz, esz, esz, esz, 4, 4, 4, 4, 4};
  for (int i = 0; i < 9; ++i)
    if ((uintptr_t)ptrs[i] % align[i] != 0) return fail(AIDN_EINVAL, "kv8_append: a buffer is not aligned to its elements");
  auto strides = [&](const int64_t* given, int64_t heads, int64_t* to) {
    to[0] = given[0] == 0 && given[1] == 0 ? heads * D : given[0];
    to[1] = given[0] == 0 && given[1] == 0 ? D : given[1];
    return to[0] >= 0 && to[1] >= 0;
  };
  if (!strides(a->query_stride, a->heads, p.qs) || !strides(a->key_stride, cache->kv_heads, p.ks) ||
      !strides(a->value_stride, cache->kv_heads, p.vs) || !strides(a->query_out_stride, a->heads, p.os))
    return fail(AIDN_EINVAL, "kv8_append: negative stride");
  p.q = a->query;
  p.k = a->key;
  p.v = a->value;
  p.q_out = a->query_out;
  p.cosine = a->cosine;
  p.sine = a->sine;
  p.start = a->start;
  p.token_starts = a->token_starts;
  p.positions = a->positions;
  p.tokens = a->tokens;
  p.max_position = a->max_position;
  p.each = a->tokens / a->batch;
  p.batch = a->batch;
  p.heads = a->query ? a->heads : 0;
  p.dtype = a->dtype;
  p.rope = a->rope;
  int launches = 0;
  const cudaError_t e = aidn::kv8::launch_append(p, (cudaStream_t)cu_stream, &launches);
  if (e != cudaSuccess) return fail_cuda(e, "kv8_append");
  return post_launch_check((cudaStream_t)cu_stream, "aidn_kv8_append", nullptr);
}

int64_t aidn_sdpa_kv8_workspace_bytes(aidn_sdpa_t h, int64_t batch, int64_t seq_q, int64_t seq_kv) {
  g_err[0] = 0;
  if (!h || batch <= 0 || seq_q <= 0 || seq_kv <= 0) {
    fail(AIDN_EINVAL, "kv8_workspace_bytes: bad argument");
    return -1;
  }
  if (h->d.path == AIDN_PATH_GENERIC || h->d.mask_kind != AIDN_MASK_NONE || h->d.head_dim % 16 != 0) return 0;
  const int64_t few = aidn::kv8::split_workspace_bytes(h->d.head_dim, h->d.out_dtype == AIDN_F32, batch, seq_q * h->group, seq_kv,
                                                        h->head_count / h->group, h->num_sms);
  const int64_t many = seq_q * h->group > aidn::kv8::kFewRows && h->d.out_dtype != AIDN_F32 && (h->d.head_dim == 64 || h->d.head_dim == 128)
                           ? aidn::kv8::sm100_workspace_bytes(h->d.head_dim, h->num_sms) : 0;
  return align_up(few > many ? few : many, 256);
}

int aidn_sdpa_launch_kv8(aidn_sdpa_t h, const aidn_sdpa_args* a, const aidn_kv8_cache* cache, const int32_t* query_starts,
                         int64_t queries, void* cu_stream) {
  g_err[0] = 0;
  if (!h || !a) return fail(AIDN_EINVAL, "launch_kv8: null argument");
  const aidn_sdpa_desc& d = h->d;
  aidn::kv8::Attend p;
  std::memset(&p, 0, sizeof(p));
  const int rc = build_pool("launch_kv8", cache, p.c);
  if (rc != AIDN_OK) return rc;
  if (cache->head_dim != d.head_dim || cache->kv_heads != d.num_kv_heads)
    return fail(AIDN_EINVAL, "launch_kv8: the pool has %d heads of %d, the handle %d of %d", cache->kv_heads, cache->head_dim, d.num_kv_heads, d.head_dim);
  if (!a->q || !a->out) return fail(AIDN_EINVAL, "launch_kv8: null tensor pointer");
  if (a->batch <= 0 || a->batch > 65535 || a->seq_q <= 0 || a->seq_kv <= 0 || a->seq_q > 0x7fffffffll || a->seq_kv > 0x7fffffffll)
    return fail(AIDN_EINVAL, "launch_kv8: batch, seq_q and seq_kv must be positive, batch at most 65535, lengths at most 2^31-1");
  if (query_starts && (queries <= 0 || queries > 0x7fffffffll)) return fail(AIDN_EINVAL, "launch_kv8: query_starts needs the number of queries");
  if (d.emit_lse && !a->lse) return fail(AIDN_EINVAL, "launch_kv8: emit_lse set but lse pointer is null");
  if (d.mask_kind != AIDN_MASK_NONE && !a->mask) return fail(AIDN_EINVAL, "launch_kv8: mask_kind set but mask pointer is null");
  if (d.mask_kind != AIDN_MASK_NONE && query_starts) return fail(AIDN_EUNSUPPORTED, "launch_kv8: masks with query_starts are not defined");
  if (a->scale < 0.f || std::isnan(a->scale)) return fail(AIDN_EINVAL, "launch_kv8: scale must be >= 0");
  if (a->weights || a->peer_count != 0 || a->gather_output)
    return fail(AIDN_EUNSUPPORTED, "launch_kv8: attention weights, peer_out and gather_output are not served over an 8-bit pool");
  if (d.path == AIDN_PATH_DECODE || d.path == AIDN_PATH_PREFILL_SM100)
    return fail(AIDN_EUNSUPPORTED, "launch_kv8: desc.path must be AUTO or GENERIC");
  const size_t esz = elem_size(d.qkv_dtype);
  if ((uintptr_t)a->q % esz != 0 || (uintptr_t)a->out % elem_size(d.out_dtype) != 0) return fail(AIDN_EINVAL, "launch_kv8: q or out is not aligned to its elements");
  if ((uintptr_t)a->kv_len % 4 != 0 || (uintptr_t)query_starts % 4 != 0) return fail(AIDN_EINVAL, "launch_kv8: kv_len or query_starts is not aligned to its entries");
  if ((d.emit_lse && (uintptr_t)a->lse % 4 != 0) || (d.mask_kind > AIDN_MASK_KEEP_U8 && (uintptr_t)a->mask % 4 != 0))
    return fail(AIDN_EINVAL, "launch_kv8: lse or mask is not aligned to its elements");
  const int64_t D = d.head_dim;
  auto strides = [&](const int64_t* given, int64_t* to) {
    if (!all_zero(given)) std::memcpy(to, given, 3 * sizeof(int64_t));
    else if (query_starts) to[0] = 0, to[1] = D, to[2] = d.num_q_heads * D;
    else dense_strides(to, d.num_q_heads, a->seq_q, D);
    return to[0] >= 0 && to[1] >= 0 && to[2] >= 0;
  };
  if (!strides(a->q_stride, p.qs) || !strides(a->o_stride, p.os)) return fail(AIDN_EINVAL, "launch_kv8: negative stride");
  p.q = a->q;
  p.out = a->out;
  p.lse = d.emit_lse ? a->lse : nullptr;
  p.kv_len = a->kv_len;
  p.query_starts = query_starts;
  p.queries = query_starts ? queries : a->batch * a->seq_q;
  p.mask = d.mask_kind != AIDN_MASK_NONE ? a->mask : nullptr;
  p.mask_kind = d.mask_kind;
  for (int i = 0; i < 4; ++i) p.mask_stride[i] = a->mask_stride[i];
  p.seq_q = a->seq_q;
  // kv_len lives on the device: no key beyond what a table row can address is looked up, whatever it says
  const int64_t most = cache->block_table_stride < (0x7fffffffll / cache->block_size) ? cache->block_table_stride * cache->block_size : 0x7fffffffll;
  p.seq_kv = a->seq_kv < most ? a->seq_kv : most;
  p.causal = d.causal ? 1 : 0;
  p.bottom_right = d.causal_bottom_right ? 1 : 0;
  p.causal_offset = d.causal_offset;
  p.batch = (int32_t)a->batch;
  p.num_q_heads = d.num_q_heads;
  p.group = h->group;
  p.kv_begin = d.head_begin / h->group;
  p.kv_count = h->head_count / h->group;
  p.dtype = d.qkv_dtype;
  p.out_f32 = d.out_dtype == AIDN_F32 ? 1 : 0;
  p.scale = a->scale > 0.f ? a->scale : 1.0f / std::sqrt((float)d.head_dim);
  p.softcap = d.softcap;
  p.status = h->status_dev;
  cudaStream_t stream = (cudaStream_t)cu_stream;
  int launches = 1;
  cudaError_t e;
  p.rows_above = 0;
  p.rows_upto = INT64_MAX;
  if (d.path != AIDN_PATH_GENERIC && p.seq_q * p.group > aidn::kv8::kFewRows && aidn::kv8::sm100_supported(p)) {
    // sequences of few rows among others: a launch of their own, at the speed of memory.  (The launches take turns on the workspace.)
    int few = 0;
    e = cudaSuccess;
    if (query_starts && p.batch > 1 && p.group <= aidn::kv8::kFewRows && aidn::kv8::split_supported(p)) {
      aidn::kv8::Attend f = p;
      f.rows_upto = aidn::kv8::kFewRows;
      f.seq_q = aidn::kv8::kFewRows / p.group;
      e = aidn::kv8::launch_attend_split(f, h->num_sms, a->workspace, a->workspace_bytes, &h->kv8_raised, &few, stream);
      p.rows_above = aidn::kv8::kFewRows;
    }
    if (e == cudaSuccess) e = aidn::kv8::launch_attend_sm100(p, h->num_sms, a->workspace, a->workspace_bytes, &h->kv8_raised, &launches, stream);
    launches += few;
    h->last_path = AIDN_PATH_PREFILL_SM100;
  } else if (d.path != AIDN_PATH_GENERIC && aidn::kv8::split_supported(p)) {
    e = aidn::kv8::launch_attend_split(p, h->num_sms, a->workspace, a->workspace_bytes, &h->kv8_raised, &launches, stream);
    h->last_path = AIDN_PATH_DECODE;
  } else {
    e = aidn::kv8::launch_attend_generic(p, stream);
    h->last_path = AIDN_PATH_GENERIC;
  }
  if (e != cudaSuccess) return fail_cuda(e, "launch_kv8");
  h->last_launches = launches;
  return post_launch_check(stream, "aidn_sdpa_launch_kv8", h->status_dev);
}

// ---- rotary positions, linear attention ------------------------------------------------------------------------------
namespace {
// What a device is, looked up once (handle-less entry points have nowhere else to keep it): its SMs, negative where it is not served.  One value, so that a
// thread sees all of it or nothing; racing threads write the same.
int device_facts(const char* op, int* sms) {
  static std::atomic<int> facts[64];
  int dev = -1;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) {
    cudaGetLastError();
    return fail_cuda(e, op);
  }
  if (dev < 0 || dev >= 64) return fail(AIDN_EUNSUPPORTED, "%s: device ordinal %d", op, dev);
  int n = facts[dev].load(std::memory_order_relaxed);
  if (n == 0) {
    e = cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev);
    if (e != cudaSuccess) return fail_cuda(e, op);
    if (!aidn_sdpa_device_supported(dev)) n = -n;
    facts[dev].store(n, std::memory_order_relaxed);
  }
  if (n < 0) return fail(AIDN_EUNSUPPORTED, "%s: device %d is not compute capability 10.x", op, dev);
  *sms = n;
  return AIDN_OK;
}

// Element strides of a tensor: given, or dense.
bool take_strides(int n, const int64_t* given, const int64_t* dense, int64_t* to) {
  bool zero = true;
  for (int i = 0; i < n; ++i) zero = zero && given[i] == 0;
  for (int i = 0; i < n; ++i) {
    to[i] = zero ? dense[i] : given[i];
    if (to[i] < 0) return false;
  }
  return true;
}

// Whether rows of an output may share elements, which two threads would then write in any order: each stride has to hold what the smaller ones span.
bool rows_meet(int n, const int64_t* extent, const int64_t* stride, int64_t size) {
  bool done[3] = {false, false, false};
  for (int i = 0; i < n; ++i) {
    int least = -1;
    for (int j = 0; j < n; ++j)
      if (!done[j] && extent[j] > 1 && (least < 0 || stride[j] < stride[least])) least = j;
    if (least < 0) return false;
    if (stride[least] < size) return true;
    size += (extent[least] - 1) * stride[least];
    done[least] = true;
  }
  return false;
}
// Whether an output is one of the tensors that a call reads or writes besides.
bool is_one_of(const void* out, std::initializer_list<const void*> others) {
  for (const void* x : others)
    if (out && out == x) return true;
  return false;
}

constexpr int64_t kMostRows = 0x7fffffc0;   // of a sequence: a whole number of chunks below 2^31
constexpr int64_t kMostBytes = 1ll << 60;

// The sizes and pointers that a forward and a backward call share.
int linear_common(const char* op, const aidn_linear_args& a, aidn::lin::Params& p) {
  if (a.batch <= 0 || a.heads <= 0 || a.kv_heads <= 0) return fail(AIDN_EINVAL, "%s: batch, heads and kv_heads must be positive", op);
  if (a.batch > 65535 || a.heads > 65535) return fail(AIDN_EINVAL, "%s: batch and heads must be at most 65535", op);
  if (a.heads % a.kv_heads != 0) return fail(AIDN_EINVAL, "%s: kv_heads (%d) must divide heads (%d)", op, a.kv_heads, a.heads);
  if (a.key_dim <= 0 || a.key_dim > 256 || a.key_dim % 8 != 0 || a.value_dim <= 0 || a.value_dim > 256 || a.value_dim % 8 != 0)
    return fail(AIDN_EINVAL, "%s: key_dim (%d) and value_dim (%d) must be multiples of 8 in [8, 256]", op, a.key_dim, a.value_dim);
  if (a.dtype < AIDN_F32 || a.dtype > AIDN_BF16) return fail(AIDN_EINVAL, "%s: unknown dtype %d", op, a.dtype);
  if (a.path != AIDN_PATH_AUTO && a.path != AIDN_PATH_GENERIC) return fail(AIDN_EINVAL, "%s: path must be AUTO or GENERIC", op);
  if (a.seq_len <= 0 || a.seq_len > 0x7fffffffll) return fail(AIDN_EINVAL, "%s: seq_len must be in [1, 2^31-1]", op);
  if (!(a.scale >= 0.f) || std::isinf(a.scale)) return fail(AIDN_EINVAL, "%s: scale must be finite and >= 0", op);
  if (a.token_starts && a.lengths) return fail(AIDN_EINVAL, "%s: lengths and token_starts exclude one another", op);
  if (a.token_starts && (a.tokens < 0 || a.tokens > 0x7fffffffll)) return fail(AIDN_EINVAL, "%s: token_starts needs the number of tokens, at most 2^31-1", op);
  if ((uintptr_t)a.decay % 4 != 0 || (uintptr_t)a.lengths % 4 != 0 || (uintptr_t)a.token_starts % 4 != 0 || (uintptr_t)a.state_slots % 4 != 0)
    return fail(AIDN_EINVAL, "%s: decay, lengths, token_starts or state_slots is not aligned to its elements", op);
  if (a.state_slots && a.num_slots <= 0) return fail(AIDN_EINVAL, "%s: state_slots needs num_slots > 0", op);
  // The most rows that a sequence can have: of packed rows, no more than there are, however large a bound seq_len is.  A segment's rows are counted in 32 bits.
  int64_t longest = a.seq_len;
  if (a.token_starts && longest > a.tokens) longest = a.tokens > 0 ? a.tokens : 1;
  if (longest > kMostRows) return fail(AIDN_EINVAL, "%s: a sequence of %lld rows; seq_len and tokens may not both be above %lld", op, (long long)longest, (long long)kMostRows);
  const int64_t rows = a.token_starts ? a.tokens : a.batch * a.seq_len, row_bytes = (int64_t)a.heads * (a.key_dim > a.value_dim ? a.key_dim : a.value_dim) * 4;
  if (rows > kMostBytes / row_bytes) return fail(AIDN_EINVAL, "%s: sizes of more than 2^60 bytes", op);
  std::memset(&p, 0, sizeof(p));
  p.decay = a.decay;
  p.lengths = a.lengths;
  p.starts = a.token_starts;
  p.slots = a.state_slots;
  p.tokens = a.tokens;
  p.seq_len = longest;
  p.batch = a.batch;
  p.heads = a.heads;
  p.num_slots = a.state_slots ? a.num_slots : a.batch;
  p.dtype = a.dtype;
  p.scale = a.scale > 0.f ? a.scale : 1.0f / std::sqrt((float)a.key_dim);
  return AIDN_OK;
}

// One tensor of such a call: its pointer's alignment and its strides.
bool linear_tensor(const aidn_linear_args& a, const void* ptr, const int64_t* given, int64_t heads, int64_t size, int64_t* to) {
  const int64_t packed[3] = {0, size, heads * size}, dense[3] = {heads * a.seq_len * size, a.seq_len * size, size};
  return (uintptr_t)ptr % elem_size(a.dtype) == 0 && (a.token_starts ? take_strides(3, given, packed, to) : take_strides(3, given, dense, to));
}

bool no_rows(const aidn_linear_args& a) { return a.token_starts && a.tokens == 0; }

bool linear_rows_meet(const aidn_linear_args& a, int64_t heads, int64_t size, const int64_t* stride) {
  const int64_t extent[3] = {a.token_starts ? 1 : a.batch, heads, a.token_starts ? a.tokens : a.seq_len};
  return rows_meet(3, extent, stride, size);
}

// The scans of a call, and the check behind them.
cudaError_t run_scans(const aidn_linear_args& a, const aidn::lin::Params& p, int sms, char* work, int64_t work_bytes, cudaStream_t stream, bool* waits) {
  const bool expire = g_expire_linear;
  g_expire_linear = false;
  g_linear_launches = 0;
  *waits = a.path != AIDN_PATH_GENERIC && aidn::lin::scan_sm100_supported(p);
  return *waits ? aidn::lin::launch_scan_sm100(p, sms, reinterpret_cast<float*>(work), work_bytes, expire, stream, &g_linear_launches)
                : aidn::lin::launch_scan_generic(p, sms, reinterpret_cast<float*>(work), work_bytes, stream, &g_linear_launches);
}
// Waits for `stream` and reports a wait given up in its context that was not yet reported for this stream.  What each stream was told is kept here, and
// only where there was something to tell; a stream's id is never another one's, its handle may be.
int linear_report(const char* op, cudaStream_t stream, const char* prefix = "") {
  cudaStreamCaptureStatus cap = cudaStreamCaptureStatusNone;
  cudaError_t e = cudaStreamIsCapturing(stream, &cap);
  if (e != cudaSuccess) {
    cudaGetLastError();
    return fail_cuda(e, op);
  }
  if (cap != cudaStreamCaptureStatusNone) return fail(AIDN_EINVAL, "%s: the stream is being captured", op);   // (to wait for it would end the capture)
  e = cudaStreamSynchronize(stream);
  if (e != cudaSuccess) return fail_cuda(e, op);
  const uint32_t* word = aidn::lin::sm100_gave_up();
  if (!word) return fail(AIDN_ECUDA, "%s: no count of waits in the current context", op);
  uint32_t count = 0;
  unsigned long long id = 0;
  e = cudaMemcpyAsync(&count, word, sizeof(count), cudaMemcpyDeviceToHost, stream);   // (on this stream: no other is waited for)
  if (e == cudaSuccess) e = cudaStreamSynchronize(stream);
  if (e != cudaSuccess) return fail_cuda(e, op);
  if (count == 0) return AIDN_OK;
  e = cudaStreamGetId(stream, &id);
  if (e != cudaSuccess) return fail_cuda(e, op);
  static std::mutex lock;
  try {
    const std::lock_guard<std::mutex> guard(lock);
    static auto& told = *new std::map<std::pair<const uint32_t*, unsigned long long>, uint32_t>;   // (never destroyed: threads may outlive main)
    uint32_t& last = told[{word, id}];
    if (last == count) return AIDN_OK;
    last = count;
  } catch (...) {   // no memory to remember it in: it will be told again
  }
  return fail(AIDN_ETIMEOUT, "%s%s: a kernel gave up a bounded wait", prefix, op);
}
int linear_check(const char* what, cudaStream_t stream, bool waits) {
  const int rc = post_launch_check(stream, what, nullptr);
  if (rc != AIDN_OK || !waits || !launch_check_enabled()) return rc;
  cudaStreamCaptureStatus cap = cudaStreamCaptureStatusNone;
  if (cudaStreamIsCapturing(stream, &cap) != cudaSuccess || cap != cudaStreamCaptureStatusNone) {
    cudaGetLastError();
    return AIDN_OK;
  }
  return linear_report(what, stream, "[LAUNCH-FAULT] ");
}
}  // namespace

int aidn_rotary(const aidn_rotary_args* a, void* cu_stream) {
  g_err[0] = 0;
  if (!a) return fail(AIDN_EINVAL, "rotary: null argument");
  if (a->tokens < 0) return fail(AIDN_EINVAL, "rotary: tokens must be >= 0");
  if (a->heads <= 0 || a->heads > 65535 || a->kv_heads < 0 || a->kv_heads > 65535) return fail(AIDN_EINVAL, "rotary: heads must be in [1, 65535], kv_heads in [0, 65535]");
  if (a->head_dim <= 0 || a->head_dim > 256 || a->head_dim % 8 != 0) return fail(AIDN_EINVAL, "rotary: head_dim %d is not a multiple of 8 in [8, 256]", a->head_dim);
  if (a->rotary_dim < 2 || a->rotary_dim > a->head_dim || a->rotary_dim % 2 != 0) return fail(AIDN_EINVAL, "rotary: rotary_dim %d is not even and in [2, head_dim]", a->rotary_dim);
  if (a->dtype < AIDN_F32 || a->dtype > AIDN_BF16) return fail(AIDN_EINVAL, "rotary: unknown dtype %d", a->dtype);
  if (a->layout != AIDN_ROPE_INTERLEAVED && a->layout != AIDN_ROPE_HALVES) return fail(AIDN_EINVAL, "rotary: unknown layout %d", a->layout);
  if (a->positions && a->position_bytes != 4 && a->position_bytes != 8) return fail(AIDN_EINVAL, "rotary: position_bytes must be 4 or 8");
  if (!a->positions && (a->seq_len < 0 || a->start_position < 0)) return fail(AIDN_EINVAL, "rotary: seq_len and start_position must be >= 0");
  if (std::isnan(a->amplitude) || std::isinf(a->amplitude)) return fail(AIDN_EINVAL, "rotary: amplitude must be finite");
  if (a->tokens == 0) return AIDN_OK;
  if (!a->query || !a->query_out || !a->frequencies) return fail(AIDN_EINVAL, "rotary: null buffer");
  if ((a->kv_heads > 0) != (a->key != nullptr) || (a->key != nullptr) != (a->key_out != nullptr))
    return fail(AIDN_EINVAL, "rotary: key, key_out and kv_heads > 0 come together");
  const size_t esz = elem_size(a->dtype);
  if ((uintptr_t)a->query % esz || (uintptr_t)a->query_out % esz || (uintptr_t)a->key % esz || (uintptr_t)a->key_out % esz ||
      (uintptr_t)a->frequencies % 8 || (a->positions && (uintptr_t)a->positions % a->position_bytes))
    return fail(AIDN_EINVAL, "rotary: a buffer is not aligned to its elements");
  aidn::lin::Rotary p;
  std::memset(&p, 0, sizeof(p));
  p.x[0] = a->query; p.y[0] = a->query_out; p.x[1] = a->key; p.y[1] = a->key_out;
  p.heads[0] = a->heads; p.heads[1] = a->kv_heads;
  const int64_t* in[2] = {a->query_stride, a->key_stride};
  const int64_t* out[2] = {a->query_out_stride, a->key_out_stride};
  for (int i = 0; i < 2; ++i) {
    const int64_t dense[2] = {(int64_t)p.heads[i] * a->head_dim, a->head_dim};
    if (!take_strides(2, in[i], dense, p.xs[i]) || !take_strides(2, out[i], dense, p.ys[i])) return fail(AIDN_EINVAL, "rotary: negative stride");
    if (p.heads[i] > 0 && p.x[i] == p.y[i] && (p.xs[i][0] != p.ys[i][0] || p.xs[i][1] != p.ys[i][1]))
      return fail(AIDN_EINVAL, "rotary: in place needs the same strides in and out");
    const int64_t extent[2] = {a->tokens, p.heads[i]};
    if (p.heads[i] > 0 && rows_meet(2, extent, p.ys[i], a->head_dim)) return fail(AIDN_EINVAL, "rotary: rows of an output overlap");
  }
  if (is_one_of(a->query_out, {a->key, a->key_out}) || is_one_of(a->key_out, {a->query})) return fail(AIDN_EINVAL, "rotary: queries and keys overlap");
  p.frequencies = a->frequencies;
  p.positions = a->positions;
  p.tokens = a->tokens;
  p.seq_len = a->seq_len > 0 ? a->seq_len : a->tokens;
  p.start = a->start_position;
  p.head_dim = a->head_dim;
  p.rotary_dim = a->rotary_dim;
  p.dtype = a->dtype;
  p.halves = a->layout == AIDN_ROPE_HALVES;
  p.wide_positions = a->position_bytes == 8;
  p.amplitude = a->amplitude != 0.f ? a->amplitude : 1.f;
  p.sign = a->inverse ? -1.f : 1.f;
  int sms = 0;
  const int rc = device_facts("rotary", &sms);
  if (rc != AIDN_OK) return rc;
  const cudaError_t e = aidn::lin::launch_rotary(p, (cudaStream_t)cu_stream);
  if (e != cudaSuccess) return fail_cuda(e, "rotary");
  return post_launch_check((cudaStream_t)cu_stream, "aidn_rotary", nullptr);
}

// Bytes for the states of segments.  (Without a device, where no call runs either, none.)
static int64_t linear_segment_bytes(const aidn_linear_args& a, const aidn::lin::Params& p) {
  int sms = 0;
  if (device_facts("", &sms) != AIDN_OK) {
    g_err[0] = 0;
    return 0;
  }
  // (which kernels serve a call depends on its pointers and strides too: enough for either)
  const int64_t one = a.path != AIDN_PATH_GENERIC ? aidn::lin::scan_sm100_bytes(p, sms) : 0, other = aidn::lin::scan_generic_bytes(p, sms);
  return one > other ? one : other;
}

int64_t aidn_linear_attention_workspace_bytes(const aidn_linear_args* a) {
  g_err[0] = 0;
  aidn::lin::Params p;
  if (!a) return fail(AIDN_EINVAL, "linear_attention_workspace_bytes: null argument"), -1;
  if (linear_common("linear_attention_workspace_bytes", *a, p) != AIDN_OK) return -1;
  p.scans = 1;
  p.scan[0].d1 = a->key_dim;
  p.scan[0].d2 = a->value_dim;
  return linear_segment_bytes(*a, p);
}

int aidn_linear_attention(const aidn_linear_args* a, void* cu_stream) {
  g_err[0] = 0;
  if (!a) return fail(AIDN_EINVAL, "linear_attention: null argument");
  aidn::lin::Params p;
  int rc = linear_common("linear_attention", *a, p);
  if (rc != AIDN_OK) return rc;
  if (!no_rows(*a) && (!a->q || !a->k || !a->v || !a->out)) return fail(AIDN_EINVAL, "linear_attention: null tensor pointer");
  if ((uintptr_t)a->initial_state % 16 != 0 || (uintptr_t)a->final_state % 16 != 0) return fail(AIDN_EINVAL, "linear_attention: states must be 16-byte aligned");
  if ((uintptr_t)a->workspace % 256 != 0) return fail(AIDN_EINVAL, "linear_attention: workspace must be 256-byte aligned");
  aidn::lin::Scan& s = p.scan[0];
  if (!linear_tensor(*a, a->q, a->q_stride, a->heads, a->key_dim, s.as) || !linear_tensor(*a, a->k, a->k_stride, a->kv_heads, a->key_dim, s.bs) ||
      !linear_tensor(*a, a->v, a->v_stride, a->kv_heads, a->value_dim, s.cs) || !linear_tensor(*a, a->out, a->o_stride, a->heads, a->value_dim, s.ys))
    return fail(AIDN_EINVAL, "linear_attention: a tensor is not aligned to its elements, or a stride is negative");
  if (linear_rows_meet(*a, a->heads, a->value_dim, s.ys) || is_one_of(a->out, {a->q, a->k, a->v}))
    return fail(AIDN_EINVAL, "linear_attention: rows of out overlap one another or an input");
  p.scans = 1;
  s.a = a->q; s.b = a->k; s.c = a->v; s.y = a->out;
  s.a_group = 1;
  s.b_group = s.c_group = a->heads / a->kv_heads;
  s.d1 = a->key_dim; s.d2 = a->value_dim;
  s.lag = 1;
  s.row_scale = p.scale;
  s.key_scale = 1.f;
  s.x_first = a->initial_state;
  s.x_last = a->final_state;
  int sms = 0;
  rc = device_facts("linear_attention", &sms);
  if (rc != AIDN_OK) return rc;
  bool waits = false;
  const cudaError_t e = run_scans(*a, p, sms, static_cast<char*>(a->workspace), a->workspace_bytes, (cudaStream_t)cu_stream, &waits);
  if (e != cudaSuccess) return fail_cuda(e, "linear_attention");
  return linear_check("aidn_linear_attention", (cudaStream_t)cu_stream, waits);
}

// Bytes of the partial sums of dk and dv for shared heads.
static int64_t linear_partial_bytes(const aidn_linear_args& a, int64_t size) {
  const int64_t rows = a.token_starts ? a.tokens : a.batch * a.seq_len;
  return a.heads == a.kv_heads ? 0 : align_up(rows * a.heads * size * 4, 256);
}

int64_t aidn_linear_attention_backward_workspace_bytes(const aidn_linear_bwd_args* a) {
  g_err[0] = 0;
  aidn::lin::Params p;
  if (!a) return fail(AIDN_EINVAL, "linear_attention_backward_workspace_bytes: null argument"), -1;
  if (linear_common("linear_attention_backward_workspace_bytes", a->fwd, p) != AIDN_OK) return -1;
  p.scans = 3;
  for (int i = 0; i < 3; ++i) {
    p.scan[i].d1 = i == 2 ? a->fwd.key_dim : a->fwd.value_dim;
    p.scan[i].d2 = i == 2 ? a->fwd.value_dim : a->fwd.key_dim;
  }
  return linear_partial_bytes(a->fwd, a->fwd.key_dim) + linear_partial_bytes(a->fwd, a->fwd.value_dim) + linear_segment_bytes(a->fwd, p);
}

int aidn_linear_attention_backward(const aidn_linear_bwd_args* a, void* cu_stream) {
  g_err[0] = 0;
  if (!a) return fail(AIDN_EINVAL, "linear_attention_backward: null argument");
  const aidn_linear_args& f = a->fwd;
  aidn::lin::Params p;
  int rc = linear_common("linear_attention_backward", f, p);
  if (rc != AIDN_OK) return rc;
  if (f.state_slots) return fail(AIDN_EUNSUPPORTED, "linear_attention_backward: states are by sequence, state_slots must be NULL");
  if (!no_rows(f) && (!f.q || !f.k || !f.v || !a->dout || !a->dq || !a->dk || !a->dv)) return fail(AIDN_EINVAL, "linear_attention_backward: null tensor pointer");
  if ((uintptr_t)f.initial_state % 16 != 0 || (uintptr_t)a->d_final_state % 16 != 0 || (uintptr_t)a->d_initial_state % 16 != 0)
    return fail(AIDN_EINVAL, "linear_attention_backward: states must be 16-byte aligned");
  if ((uintptr_t)f.workspace % 256 != 0) return fail(AIDN_EINVAL, "linear_attention_backward: workspace must be 256-byte aligned");
  const int group = f.heads / f.kv_heads;
  const int64_t dk = f.key_dim, dv = f.value_dim, part[2] = {linear_partial_bytes(f, dk), linear_partial_bytes(f, dv)};
  int64_t qs[3], ks[3], vs[3], dos[3], dqs[3], dks[3], dvs[3];
  if (!linear_tensor(f, f.q, f.q_stride, f.heads, dk, qs) || !linear_tensor(f, f.k, f.k_stride, f.kv_heads, dk, ks) ||
      !linear_tensor(f, f.v, f.v_stride, f.kv_heads, dv, vs) || !linear_tensor(f, a->dout, a->do_stride, f.heads, dv, dos) ||
      !linear_tensor(f, a->dq, a->dq_stride, f.heads, dk, dqs) || !linear_tensor(f, a->dk, a->dk_stride, f.kv_heads, dk, dks) ||
      !linear_tensor(f, a->dv, a->dv_stride, f.kv_heads, dv, dvs))
    return fail(AIDN_EINVAL, "linear_attention_backward: a tensor is not aligned to its elements, or a stride is negative");
  if (group > 1 && part[0] + part[1] > 0 && (!f.workspace || f.workspace_bytes < part[0] + part[1]))
    return fail(AIDN_EWORKSPACE, "linear_attention_backward: workspace of %lld bytes, need %lld", (long long)(f.workspace ? f.workspace_bytes : 0),
                (long long)(part[0] + part[1]));
  if (linear_rows_meet(f, f.heads, dk, dqs) || linear_rows_meet(f, f.kv_heads, dk, dks) || linear_rows_meet(f, f.kv_heads, dv, dvs) ||
      is_one_of(a->dq, {f.q, f.k, f.v, a->dout, a->dk, a->dv}) || is_one_of(a->dk, {f.q, f.k, f.v, a->dout, a->dv}) ||
      is_one_of(a->dv, {f.q, f.k, f.v, a->dout}))
    return fail(AIDN_EINVAL, "linear_attention_backward: rows of gradients overlap one another or an input");
  auto copy3 = [](int64_t* to, const int64_t* from) { std::memcpy(to, from, 3 * sizeof(int64_t)); };
  const int64_t rows = f.token_starts ? f.tokens : f.seq_len;   // of a head of the partial sums
  p.scans = 3;
  aidn::lin::Scan& sq = p.scan[0];
  sq.a = a->dout; sq.b = f.v; sq.c = f.k; sq.y = a->dq;
  copy3(sq.as, dos); copy3(sq.bs, vs); copy3(sq.cs, ks); copy3(sq.ys, dqs);
  sq.a_group = 1; sq.b_group = sq.c_group = group;
  sq.d1 = (int)dv; sq.d2 = (int)dk;
  sq.lag = 1;
  sq.row_scale = p.scale; sq.key_scale = 1.f;
  sq.x_first = f.initial_state;
  sq.x_transposed = 1;
  aidn::lin::Scan& sk = p.scan[1];
  sk.a = f.v; sk.b = a->dout; sk.c = f.q; sk.y = group > 1 ? f.workspace : a->dk;
  copy3(sk.as, vs); copy3(sk.bs, dos); copy3(sk.cs, qs); copy3(sk.ys, dks);
  sk.a_group = group; sk.b_group = sk.c_group = 1;
  sk.d1 = (int)dv; sk.d2 = (int)dk;
  sk.x_first = a->d_final_state;
  sk.x_transposed = 1;
  aidn::lin::Scan& sv = p.scan[2];
  sv.a = f.k; sv.b = f.q; sv.c = a->dout; sv.y = group > 1 ? static_cast<char*>(f.workspace) + part[0] : a->dv;
  copy3(sv.as, ks); copy3(sv.bs, qs); copy3(sv.cs, dos); copy3(sv.ys, dvs);
  sv.a_group = group; sv.b_group = sv.c_group = 1;
  sv.d1 = (int)dk; sv.d2 = (int)dv;
  sv.x_first = a->d_final_state;
  sv.x_last = a->d_initial_state;
  for (aidn::lin::Scan* s : {&sk, &sv}) {
    s->reverse = 1;
    s->row_scale = 1.f;
    s->key_scale = p.scale;
    if (group > 1) {
      s->y_f32 = 1;
      s->ys[0] = f.heads * rows * s->d2;
      s->ys[1] = rows * s->d2;
      s->ys[2] = s->d2;
    }
  }
  int sms = 0;
  rc = device_facts("linear_attention_backward", &sms);
  if (rc != AIDN_OK) return rc;
  cudaStream_t stream = (cudaStream_t)cu_stream;
  bool waits = false;
  cudaError_t e = run_scans(f, p, sms, f.workspace ? static_cast<char*>(f.workspace) + part[0] + part[1] : nullptr,
                            f.workspace_bytes - part[0] - part[1], stream, &waits);
  if (e == cudaSuccess && group > 1) {
    aidn::lin::GroupSum g;
    std::memset(&g, 0, sizeof(g));
    g.partial[0] = static_cast<const float*>(sk.y);
    g.partial[1] = static_cast<const float*>(sv.y);
    g.out[0] = a->dk; g.out[1] = a->dv;
    copy3(g.os[0], dks); copy3(g.os[1], dvs);
    g.d[0] = (int)dk; g.d[1] = (int)dv;
    g.rows = rows;
    g.lengths = f.lengths; g.starts = f.token_starts;
    g.tokens = f.tokens; g.seq_len = p.seq_len;
    g.batch = f.batch; g.kv_heads = f.kv_heads; g.group = group; g.dtype = f.dtype;
    e = aidn::lin::launch_group_sum(g, stream);
    if (e == cudaSuccess) ++g_linear_launches;
  }
  if (e != cudaSuccess) return fail_cuda(e, "linear_attention_backward");
  return linear_check("aidn_linear_attention_backward", stream, waits);
}

int aidn_linear_attention_last_launch_count(void) { return g_linear_launches; }

int aidn_linear_attention_poll(void* cu_stream) {
  g_err[0] = 0;
  return linear_report("linear_attention_poll", (cudaStream_t)cu_stream);
}

int aidn_linear_attention_step(const aidn_linear_step_args* a, void* cu_stream) {
  g_err[0] = 0;
  if (!a) return fail(AIDN_EINVAL, "linear_attention_step: null argument");
  if (a->batch < 0 || a->heads <= 0 || a->kv_heads <= 0) return fail(AIDN_EINVAL, "linear_attention_step: batch must be >= 0, heads and kv_heads positive");
  if (a->batch > 65535 || a->heads > 65535) return fail(AIDN_EINVAL, "linear_attention_step: batch and heads must be at most 65535");
  if (a->heads % a->kv_heads != 0) return fail(AIDN_EINVAL, "linear_attention_step: kv_heads (%d) must divide heads (%d)", a->kv_heads, a->heads);
  if (a->key_dim <= 0 || a->key_dim > 256 || a->key_dim % 8 != 0 || a->value_dim <= 0 || a->value_dim > 256 || a->value_dim % 8 != 0)
    return fail(AIDN_EINVAL, "linear_attention_step: key_dim (%d) and value_dim (%d) must be multiples of 8 in [8, 256]", a->key_dim, a->value_dim);
  if (a->dtype < AIDN_F32 || a->dtype > AIDN_BF16) return fail(AIDN_EINVAL, "linear_attention_step: unknown dtype %d", a->dtype);
  if (!(a->scale >= 0.f) || std::isinf(a->scale)) return fail(AIDN_EINVAL, "linear_attention_step: scale must be finite and >= 0");
  if (a->state_slots && a->num_slots <= 0) return fail(AIDN_EINVAL, "linear_attention_step: state_slots needs num_slots > 0");
  if (a->batch == 0) return AIDN_OK;
  if (!a->q || !a->k || !a->v || !a->out || !a->states) return fail(AIDN_EINVAL, "linear_attention_step: null buffer");
  const size_t esz = elem_size(a->dtype);
  if ((uintptr_t)a->q % esz || (uintptr_t)a->k % esz || (uintptr_t)a->v % esz || (uintptr_t)a->out % esz || (uintptr_t)a->decay % 4 || (uintptr_t)a->state_slots % 4)
    return fail(AIDN_EINVAL, "linear_attention_step: a buffer is not aligned to its elements");
  if ((uintptr_t)a->states % 16 != 0) return fail(AIDN_EINVAL, "linear_attention_step: states must be 16-byte aligned");
  aidn::lin::Step p;
  std::memset(&p, 0, sizeof(p));
  const int64_t kd = a->key_dim, vd = a->value_dim;
  const int64_t dq[2] = {a->heads * kd, kd}, dk[2] = {a->kv_heads * kd, kd}, dv[2] = {a->kv_heads * vd, vd}, dout[2] = {a->heads * vd, vd};
  if (!take_strides(2, a->q_stride, dq, p.qs) || !take_strides(2, a->k_stride, dk, p.ks) || !take_strides(2, a->v_stride, dv, p.vs) || !take_strides(2, a->o_stride, dout, p.os))
    return fail(AIDN_EINVAL, "linear_attention_step: negative stride");
  const int64_t extent[2] = {a->batch, a->heads};
  if (rows_meet(2, extent, p.os, vd) || is_one_of(a->out, {a->q, a->k, a->v})) return fail(AIDN_EINVAL, "linear_attention_step: rows of out overlap one another or an input");
  p.q = a->q; p.k = a->k; p.v = a->v; p.out = a->out;
  p.states = a->states;
  p.decay = a->decay;
  p.slots = a->state_slots;
  p.batch = a->batch; p.heads = a->heads; p.group = a->heads / a->kv_heads;
  p.key_dim = a->key_dim; p.value_dim = a->value_dim;
  p.num_slots = a->state_slots ? a->num_slots : a->batch;
  p.dtype = a->dtype;
  p.scale = a->scale > 0.f ? a->scale : 1.0f / std::sqrt((float)a->key_dim);
  int sms = 0;
  const int rc = device_facts("linear_attention_step", &sms);
  if (rc != AIDN_OK) return rc;
  const cudaError_t e = aidn::lin::launch_step(p, sms, (cudaStream_t)cu_stream);
  if (e != cudaSuccess) return fail_cuda(e, "linear_attention_step");
  return post_launch_check((cudaStream_t)cu_stream, "aidn_linear_attention_step", nullptr);
}

// ---- fused multi-head attention forward ---------------------------------------------------------------------------
namespace {
struct MhaPlan {
  int64_t off_x, off_w, off_q, off_k, off_v, off_o, off_t[2], total;   // off_t: terms of the fp32 weights, Q / K / V and output
  aidn::ProjPlanF32 f32_plan[2];
};
// `images`: with the terms of the fp32 weights in the workspace, where that is faster.
MhaPlan mha_plan(const aidn_sdpa* h, int64_t batch, int64_t seq, int input_dtype, int weight_dtype, bool images) {
  const int64_t dm = (int64_t)h->d.num_q_heads * h->d.head_dim;
  const int64_t esz = (int64_t)elem_size(h->d.qkv_dtype);
  const int64_t act = align_up(batch * seq * dm * esz, 1024), wgt = align_up(dm * dm * esz, 1024);
  MhaPlan pl;
  std::memset(&pl, 0, sizeof(pl));
  int64_t off = 0;
  pl.off_x = off; off += input_dtype != h->d.qkv_dtype ? act : 0;
  pl.off_w = off; off += weight_dtype != h->d.qkv_dtype ? 4 * wgt : 0;
  pl.off_q = off; off += act;
  pl.off_k = off; off += act;
  pl.off_v = off; off += act;
  pl.off_o = off; off += act;
  for (int i = 0; i < 2; ++i) {
    pl.off_t[i] = off;
    if (h->d.qkv_dtype != AIDN_F32 || h->d.path == AIDN_PATH_GENERIC || !aidn::proj_gemm_f32_sm100_fits(dm, dm)) continue;
    const int mats = i == 0 ? 3 : 1;
    pl.f32_plan[i] = aidn::proj_gemm_f32_sm100_plan(batch * seq, dm, dm, mats, h->num_sms, images, i == 1 && !pl.f32_plan[0].cut_w);
    off += align_up(aidn::proj_gemm_f32_sm100_bytes(pl.f32_plan[i], dm, dm, mats), 1024);
  }
  pl.total = off;
  return pl;
}
int mha_check_handle(const aidn_sdpa* h) {
  const aidn_sdpa_desc& d = h->d;
  if (d.out_dtype != d.qkv_dtype)
    return fail(AIDN_EUNSUPPORTED, "mha: the handle must have out_dtype == qkv_dtype (the attention output feeds a projection)");
  if (d.num_kv_heads != d.num_q_heads || h->head_count != d.num_q_heads)
    return fail(AIDN_EUNSUPPORTED, "mha: the handle must cover all heads with num_kv_heads == num_q_heads");
  if (d.emit_lse || d.softcap > 0.f || d.nccl_comm)
    return fail(AIDN_EUNSUPPORTED, "mha: the handle must not ask for log-sum-exp, softcap or a gather");
  if (d.mask_kind == AIDN_MASK_ADD_F32) return fail(AIDN_EUNSUPPORTED, "mha: the mask is a keep-mask (Tensor<bool>) or absent");
  // desc.causal is honoured (causal self-attention without materialising the mask): an extension, the reference's
  // MultiHeadAttentionForward expresses causality through its boolean mask only.
  return AIDN_OK;
}
}  // namespace

int64_t aidn_mha_workspace_bytes(aidn_sdpa_t h, int64_t batch, int64_t seq, int32_t input_dtype, int32_t weight_dtype) {
  g_err[0] = 0;
  if (!h || batch <= 0 || seq <= 0) {
    fail(AIDN_EINVAL, "mha_workspace_bytes: bad argument");
    return -1;
  }
  if (mha_check_handle(h) != AIDN_OK) return -1;
  return mha_plan(h, batch, seq, input_dtype, weight_dtype, true).total;
}

int aidn_mha_forward(aidn_sdpa_t h, const aidn_mha_args* a, void* cu_stream) {
  g_err[0] = 0;
  if (!h || !a) return fail(AIDN_EINVAL, "mha: null argument");
  if (!a->input || !a->q_weight || !a->k_weight || !a->v_weight || !a->out_weight || !a->out)
    return fail(AIDN_EINVAL, "mha: null tensor pointer");
  if (a->batch <= 0 || a->seq <= 0) return fail(AIDN_EINVAL, "mha: batch and seq must be positive");
  int rc = mha_check_handle(h);
  if (rc != AIDN_OK) return rc;
  const aidn_sdpa_desc& d = h->d;
  auto dtype_ok = [&](int t) { return t == AIDN_F32 || t == d.qkv_dtype; };
  if (!dtype_ok(a->input_dtype) || !dtype_ok(a->weight_dtype) || !dtype_ok(a->out_dtype))
    return fail(AIDN_EINVAL, "mha: input, weight and output dtypes must be fp32 or the handle's qkv_dtype");
  if (d.mask_kind != AIDN_MASK_NONE && !a->mask) return fail(AIDN_EINVAL, "mha: mask_kind set but mask pointer is null");
  MhaPlan pl = mha_plan(h, a->batch, a->seq, a->input_dtype, a->weight_dtype, true);
  if (a->workspace && a->workspace_bytes < pl.total)   // no room for the images: the GEMMs cut the weights themselves
    pl = mha_plan(h, a->batch, a->seq, a->input_dtype, a->weight_dtype, false);
  if (!a->workspace || a->workspace_bytes < pl.total)
    return fail(AIDN_EWORKSPACE, "mha: workspace of %lld bytes, need %lld", (long long)(a->workspace ? a->workspace_bytes : 0),
                (long long)pl.total);
  if ((uintptr_t)a->workspace % 256 != 0) return fail(AIDN_EINVAL, "mha: workspace must be 256-byte aligned");
  cudaStream_t stream = (cudaStream_t)cu_stream;
  char* ws = static_cast<char*>(a->workspace);
  const int64_t H = d.num_q_heads, D = d.head_dim, dm = H * D, S = a->seq, B = a->batch;
  const int cast_kind = d.qkv_dtype == AIDN_BF16 ? 0 : 1;
  const int64_t esz = (int64_t)elem_size(d.qkv_dtype);
  // tcgen05 GEMMs for 16-bit arithmetic on head sizes 64 / 128, and for fp32 from three bf16 terms where the width allows; the fp32
  // FFMA GEMM for everything else
  const bool tensor_route = d.qkv_dtype != AIDN_F32 && (D == 64 || D == 128) && dm % 128 == 0 && d.path != AIDN_PATH_GENERIC;
  int launches = 0;
  cudaError_t e = cudaSuccess;

  const void* x = a->input;
  if (a->input_dtype != d.qkv_dtype) {
    e = aidn::launch_cast(cast_kind, a->input, ws + pl.off_x, B * S * dm, stream);
    if (e != cudaSuccess) return fail_cuda(e, "mha: input cast");
    x = ws + pl.off_x;
    ++launches;
  }
  const void* w[4] = {a->q_weight, a->k_weight, a->v_weight, a->out_weight};
  if (a->weight_dtype != d.qkv_dtype) {
    const int64_t wgt = align_up(dm * dm * esz, 1024);
    for (int i = 0; i < 4; ++i) {
      void* dst = ws + pl.off_w + i * wgt;
      e = aidn::launch_cast(cast_kind, w[i], dst, dm * dm, stream);
      if (e != cudaSuccess) return fail_cuda(e, "mha: weight cast");
      w[i] = dst;
      ++launches;
    }
  }

  const char* why = "";
  aidn::ProjGemm g;
  std::memset(&g, 0, sizeof(g));
  g.a = x;
  g.batch = B; g.seq = S; g.k = dm; g.n = dm;
  g.head_dim = (int)D;
  g.bf16 = d.qkv_dtype == AIDN_BF16;
  g.num_mats = 3;
  g.out_f32 = false;
  for (int i = 0; i < 3; ++i) g.w[i] = w[i];
  g.c[0] = ws + pl.off_q; g.c[1] = ws + pl.off_k; g.c[2] = ws + pl.off_v;
  g.c_stride[0] = H * S * D; g.c_stride[1] = S * D; g.c_stride[2] = D;    // [B, H, S, d]
  aidn::ProjGemm go = g;
  go.a = ws + pl.off_o;
  go.num_mats = 1;
  go.w[0] = w[3];
  go.c[0] = a->out;
  go.out_f32 = a->out_dtype == AIDN_F32;
  go.c_stride[0] = S * dm; go.c_stride[1] = D; go.c_stride[2] = dm;
  bool f32_sm100[2] = {false, false};   // projections of Q, K and V, and of the output
  if (d.qkv_dtype == AIDN_F32 && d.path != AIDN_PATH_GENERIC) {
    f32_sm100[0] = aidn::proj_gemm_f32_sm100_supported(g);
    f32_sm100[1] = aidn::proj_gemm_f32_sm100_supported(go);
    aidn::ProjGemm split[2];
    int count = 0;
    g.image = ws + pl.off_t[0];
    g.f32_plan = pl.f32_plan[0];
    go.image = ws + pl.off_t[1];
    go.f32_plan = pl.f32_plan[1];
    if (f32_sm100[0] && pl.off_t[1] > pl.off_t[0]) split[count++] = g;
    if (f32_sm100[1] && pl.total > pl.off_t[1]) split[count++] = go;
    if (count > 0) {
      e = aidn::launch_proj_split_f32(split, count, stream);
      if (e != cudaSuccess) return fail_cuda(e, "mha: terms of the weights");
      ++launches;
    }
  }
  auto gemm = [&](const aidn::ProjGemm& g, bool f32_sm100, const char* what) -> int {
    if (tensor_route) {
      if (!aidn::proj_gemm_sm100_supported(g, &why)) return fail(AIDN_EUNSUPPORTED, "mha: %s", why);
      e = aidn::launch_proj_gemm_sm100(g, stream, h->num_sms, h->status_dev, &why, h->debug_mode == 3);
    } else {
      if (!aidn::proj_gemm_generic_supported(g, &why)) return fail(AIDN_EUNSUPPORTED, "mha: %s", why);
      if (f32_sm100)
        e = aidn::launch_proj_gemm_f32_sm100(g, stream, h->status_dev, h->debug_mode == 3);
      else
        e = aidn::launch_proj_gemm_generic(g, d.qkv_dtype, stream);
    }
    if (e != cudaSuccess) return why[0] ? fail(AIDN_ECUDA, "mha: %s (%s)", why, cudaGetErrorName(e)) : fail_cuda(e, what);
    ++launches;
    return AIDN_OK;
  };
  rc = gemm(g, f32_sm100[0], "mha: QKV projection");
  if (rc != AIDN_OK) return rc;

  aidn_sdpa_args sa;
  std::memset(&sa, 0, sizeof(sa));
  sa.q = g.c[0]; sa.k = g.c[1]; sa.v = g.c[2];
  sa.out = ws + pl.off_o;
  sa.mask = a->mask;
  for (int i = 0; i < 4; ++i) sa.mask_stride[i] = a->mask_stride[i];
  sa.batch = B; sa.seq_q = S; sa.seq_kv = S;
  sa.o_stride[0] = S * dm; sa.o_stride[1] = D; sa.o_stride[2] = dm;      // heads side by side: [B, S, H*d]
  rc = launch_common(h, &sa, nullptr, cu_stream);
  if (rc != AIDN_OK) return rc;
  launches += h->last_launches;

  rc = gemm(go, f32_sm100[1], "mha: output projection");
  if (rc != AIDN_OK) return rc;
  h->last_launches = launches;
  return post_launch_check(stream, "aidn_mha_forward", h->status_dev);
}

static int cast_common(int kind, const void* src, void* dst, int64_t n, void* cu_stream) {
  g_err[0] = 0;
  if (n < 0 || (n > 0 && (!src || !dst))) return fail(AIDN_EINVAL, "cast: bad argument");
  cudaError_t e = aidn::launch_cast(kind, src, dst, n, (cudaStream_t)cu_stream);
  if (e != cudaSuccess) return fail_cuda(e, "cast");
  return AIDN_OK;
}

int aidn_peer_export(const void* dev_ptr, void* handle64, int64_t* offset) {
  g_err[0] = 0;
  if (!dev_ptr || !handle64 || !offset) return fail(AIDN_EINVAL, "peer_export: null argument");
  static_assert(sizeof(cudaIpcMemHandle_t) == 64, "CUDA IPC handle size");
  // the handle names a whole allocation: find its base
  typedef int (*GetRangeFn)(unsigned long long*, size_t*, unsigned long long);   // CUresult cuMemGetAddressRange_v2
  static GetRangeFn get_range = nullptr;
  if (!get_range) {
    void* raw = nullptr;
    cudaDriverEntryPointQueryResult qres;
    if (cudaGetDriverEntryPoint("cuMemGetAddressRange", &raw, cudaEnableDefault, &qres) != cudaSuccess || !raw ||
        qres != cudaDriverEntryPointSuccess)
      return fail(AIDN_ECUDA, "peer_export: cuMemGetAddressRange is not available from the driver");
    get_range = reinterpret_cast<GetRangeFn>(raw);
  }
  unsigned long long base = 0;
  size_t size = 0;
  if (get_range(&base, &size, (unsigned long long)(uintptr_t)dev_ptr) != 0)
    return fail(AIDN_EINVAL, "peer_export: not a device allocation");
  cudaIpcMemHandle_t hdl;
  cudaError_t e = cudaIpcGetMemHandle(&hdl, reinterpret_cast<void*>((uintptr_t)base));
  if (e != cudaSuccess) return fail_cuda(e, "peer_export");
  std::memcpy(handle64, &hdl, 64);
  *offset = (int64_t)((uintptr_t)dev_ptr - (uintptr_t)base);
  return AIDN_OK;
}

int aidn_peer_open(const void* handle64, void** base) {
  g_err[0] = 0;
  if (!handle64 || !base) return fail(AIDN_EINVAL, "peer_open: null argument");
  cudaIpcMemHandle_t hdl;
  std::memcpy(&hdl, handle64, 64);
  cudaError_t e = cudaIpcOpenMemHandle(base, hdl, cudaIpcMemLazyEnablePeerAccess);
  if (e != cudaSuccess) return fail_cuda(e, "peer_open");
  return AIDN_OK;
}

int aidn_peer_close(void* base) {
  g_err[0] = 0;
  if (!base) return fail(AIDN_EINVAL, "peer_close: null argument");
  cudaError_t e = cudaIpcCloseMemHandle(base);
  if (e != cudaSuccess) return fail_cuda(e, "peer_close");
  return AIDN_OK;
}

int aidn_cast_f32_to_bf16(const float* src, void* dst, int64_t n, void* s) { return cast_common(0, src, dst, n, s); }
int aidn_cast_f32_to_f16(const float* src, void* dst, int64_t n, void* s) { return cast_common(1, src, dst, n, s); }
int aidn_cast_bf16_to_f32(const void* src, float* dst, int64_t n, void* s) { return cast_common(2, src, dst, n, s); }
int aidn_cast_f16_to_f32(const void* src, float* dst, int64_t n, void* s) { return cast_common(3, src, dst, n, s); }

}  // extern "C"
