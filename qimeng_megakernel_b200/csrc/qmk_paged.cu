// C entry points of the paged KV cache: block tables, slot maps, attention with a shared prefix.
// Plain launches on the caller's stream; no handle, no library-owned memory.
#include <cuda_runtime.h>
#include <math.h>
#include <stdio.h>
#include <string.h>

#include "../../include/qmk_b200.h"
#include "qmk_paged_tables.cuh"
#include "qmk_prefix_attention.cuh"

using namespace qmkp;

static thread_local char g_paged_err[256];

extern "C" const char* qmk_paged_last_cuda_error(void) { return g_paged_err; }

static int paged_fail(cudaError_t e, const char* what) {
  snprintf(g_paged_err, sizeof(g_paged_err), "%s: %s", what, cudaGetErrorString(e));
  return QMK_ERR_CUDA;
}

// The launch goes to `device` whatever the caller's current device is, which is put back.
namespace {
struct DeviceScope {
  int before = -1;
  cudaError_t err;
  explicit DeviceScope(int device) {
    err = cudaGetDevice(&before);
    if (err == cudaSuccess && before != device) err = cudaSetDevice(device);
    else before = -1;
  }
  ~DeviceScope() {
    if (before >= 0) cudaSetDevice(before);
  }
};
}  // namespace

static int page_shift_of(int page_size) {
  for (int s = 4; s <= 8; ++s)
    if (page_size == (1 << s)) return s;
  return -1;
}
static bool aligned_to(const void* p, unsigned n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1u)) == 0; }

extern "C" int qmk_build_block_tables(const qmk_block_tables_args* a, int device, void* cuda_stream) {
  if (!a || a->seqs < 1 || a->max_pages < 1 || a->num_free < 0 || a->prefix_pages < 0) return QMK_ERR_INVALID_ARG;
  const int shift = page_shift_of(a->page_size);
  if (shift < 0 || !a->lengths || !a->tables || !a->used || (a->num_free > 0 && !a->free_pages) ||
      (a->prefix_pages > 0 && !a->prefix_table) || a->prefix_pages > a->max_pages)
    return QMK_ERR_INVALID_ARG;
  DeviceScope scope(device);
  if (scope.err != cudaSuccess) return paged_fail(scope.err, "cudaSetDevice");
  TableParams p;
  p.lengths = a->lengths; p.free_pages = a->free_pages; p.prefix_table = a->prefix_table;
  p.tables = a->tables; p.used = a->used;
  p.seqs = a->seqs; p.num_free = a->num_free; p.prefix_pages = a->prefix_pages; p.page_shift = shift; p.max_pages = a->max_pages;
  int rows = (a->seqs + 295) / 296;
  if (rows < 8) rows = 8;
  if (rows > kTableThreads) rows = kTableThreads;
  p.rows_per_cta = rows;
  block_tables_kernel<<<(unsigned)((a->seqs + rows - 1) / rows), kTableThreads, 0, (cudaStream_t)cuda_stream>>>(p);
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? QMK_OK : paged_fail(e, "block_tables_kernel");
}

extern "C" int qmk_build_slot_map(const qmk_slot_map_args* a, int device, void* cuda_stream) {
  if (!a || a->seqs < 1 || a->tokens < 1 || a->max_pages < 1) return QMK_ERR_INVALID_ARG;
  const int shift = page_shift_of(a->page_size);
  if (shift < 0 || !a->block_tables || !a->kv_lengths || !a->new_lengths || !a->slots || !a->positions || !a->seq_ids ||
      !a->active || !a->cu_tokens || !a->kv_lengths_out)
    return QMK_ERR_INVALID_ARG;
  if (a->kv_lengths_out == a->kv_lengths) return QMK_ERR_INVALID_ARG;   // other CTAs still read the lengths
  DeviceScope scope(device);
  if (scope.err != cudaSuccess) return paged_fail(scope.err, "cudaSetDevice");
  SlotParams p;
  p.tables = a->block_tables; p.kv_lengths = a->kv_lengths; p.new_lengths = a->new_lengths;
  p.slots = (long long*)a->slots; p.positions = a->positions; p.seq_ids = a->seq_ids; p.active = a->active;
  p.cu_tokens = a->cu_tokens; p.kv_out = a->kv_lengths_out;
  p.seqs = a->seqs; p.tokens = a->tokens; p.page_shift = shift; p.max_pages = a->max_pages;
  const unsigned grid = (unsigned)(((long long)a->tokens + kTableThreads - 1) / kTableThreads);
  slot_map_kernel<<<grid, kTableThreads, 0, (cudaStream_t)cuda_stream>>>(p);
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? QMK_OK : paged_fail(e, "slot_map_kernel");
}

extern "C" int64_t qmk_prefix_attention_workspace(int32_t tokens, int32_t seqs, int32_t num_heads, int32_t num_kv_heads,
                                                  int32_t head_dim, int32_t prefix_len, int device) {
  (void)tokens; (void)seqs; (void)num_heads; (void)num_kv_heads; (void)head_dim; (void)prefix_len; (void)device;
  return 0;
}

static int attention_args(const qmk_prefix_attention_args* a) {
  if (!a) return QMK_ERR_INVALID_ARG;
  if (a->tokens < 1 || a->seqs < 1 || a->max_pages < 1 || a->num_pages < 1 || a->prefix_len < 0) return QMK_ERR_INVALID_ARG;
  if (a->head_dim != 64 && a->head_dim != 128) return QMK_ERR_INVALID_ARG;
  if (a->num_kv_heads < 1 || a->num_heads < 1 || a->num_heads % a->num_kv_heads != 0 || a->num_heads / a->num_kv_heads > 16)
    return QMK_ERR_INVALID_ARG;
  if (page_shift_of(a->page_size) < 0 || a->prefix_len % a->page_size != 0) return QMK_ERR_INVALID_ARG;
  if (a->prefix_len > 0 && !a->prefix_table) return QMK_ERR_INVALID_ARG;
  if (!a->block_tables || !a->kv_lengths || !a->cu_tokens || !a->q || !a->out || !a->k_pages || !a->v_pages) return QMK_ERR_INVALID_ARG;
  const long long row = (long long)a->num_heads * a->head_dim;
  if (a->q_token_stride < row || a->out_token_stride < row || a->q_token_stride % 8 != 0 || a->out_token_stride % 8 != 0)
    return QMK_ERR_INVALID_ARG;
  if (!aligned_to(a->q, 16) || !aligned_to(a->out, 16) || !aligned_to(a->k_pages, 16) || !aligned_to(a->v_pages, 16))
    return QMK_ERR_INVALID_ARG;
  if (!(a->scale > 0.f) || isinf(a->scale)) return QMK_ERR_INVALID_ARG;
  return QMK_OK;
}

extern "C" int qmk_prefix_attention(const qmk_prefix_attention_args* a, int device, void* cuda_stream) {
  const int rc = attention_args(a);
  if (rc) return rc;
  DeviceScope scope(device);
  if (scope.err != cudaSuccess) return paged_fail(scope.err, "cudaSetDevice");
  AttnParams p;
  p.q = (const uint16_t*)a->q; p.out = (uint16_t*)a->out; p.lse = a->lse;
  p.k_pages = (const uint16_t*)a->k_pages; p.v_pages = (const uint16_t*)a->v_pages;
  p.tables = a->block_tables; p.kv_lengths = a->kv_lengths; p.cu_tokens = a->cu_tokens; p.prefix_table = a->prefix_table;
  p.q_stride = a->q_token_stride; p.out_stride = a->out_token_stride;
  p.tokens = a->tokens; p.seqs = a->seqs; p.NH = a->num_heads; p.NKV = a->num_kv_heads;
  p.page_shift = page_shift_of(a->page_size); p.num_pages = a->num_pages; p.max_pages = a->max_pages; p.prefix_len = a->prefix_len;
  p.scale_log2e = a->scale * 1.4426950408889634f;
  const unsigned grid = (unsigned)(((long long)a->tokens * a->num_heads + 3) / 4);
  if (a->head_dim == 64) prefix_attention_simple<64><<<grid, 128, 0, (cudaStream_t)cuda_stream>>>(p);
  else prefix_attention_simple<128><<<grid, 128, 0, (cudaStream_t)cuda_stream>>>(p);
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? QMK_OK : paged_fail(e, "prefix_attention_simple");
}
