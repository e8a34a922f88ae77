// C entry points of the paged KV cache: block tables, slot maps, attention with a shared prefix.
// Plain launches on the caller's stream; no handle, no library-owned memory.
#include <cuda.h>
#include <cuda_runtime.h>
#include <math.h>
#include <stdio.h>
#include <string.h>

#include <atomic>

#include "../../include/qmk_b200.h"
#include "qmk_paged_host.h"
#include "qmk_paged_tables.cuh"
#include "qmk_prefix_attention.cuh"

using namespace qmkp;

static thread_local char g_paged_err[256];

extern "C" const char* qmk_paged_last_cuda_error(void) { return g_paged_err; }

static int refuse(const char* why) {
  snprintf(g_paged_err, sizeof(g_paged_err), "%s", why);
  return QMK_ERR_INVALID_ARG;
}

// An operand's bytes.  Outputs may not cover any of an input or of one another: other CTAs still read, or write too.
struct Bytes {
  const char* name;
  const void* at;
  long long n;
};
static bool apart(const Bytes* out, int outs, const Bytes* in, int ins) {
  const auto meet = [](const Bytes& a, const Bytes& b) {
    const uintptr_t x = reinterpret_cast<uintptr_t>(a.at), y = reinterpret_cast<uintptr_t>(b.at);
    if (a.n <= 0 || b.n <= 0 || x + (uintptr_t)a.n <= y || y + (uintptr_t)b.n <= x) return false;
    snprintf(g_paged_err, sizeof(g_paged_err), "%s overlaps %s", a.name, b.name);
    return true;
  };
  for (int i = 0; i < outs; ++i) {
    for (int j = 0; j < ins; ++j)
      if (meet(out[i], in[j])) return false;
    for (int j = 0; j < i; ++j)
      if (meet(out[i], out[j])) return false;
  }
  return true;
}

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
  g_paged_err[0] = 0;
  if (!a || a->seqs < 1 || a->seqs > kMaxTableSeqs || a->max_pages < 1 || a->max_pages > kMaxTablePages || a->num_free < 0 ||
      a->prefix_pages < 0)
    return QMK_ERR_INVALID_ARG;
  const int shift = page_shift_of(a->page_size);
  if (shift < 0 || !a->lengths || !a->tables || !a->used || (a->num_free > 0 && !a->free_pages) ||
      (a->prefix_pages > 0 && !a->prefix_table) || a->prefix_pages > a->max_pages)
    return QMK_ERR_INVALID_ARG;
  const Bytes in[] = {{"lengths", a->lengths, 4ll * a->seqs}, {"free_pages", a->free_pages, 4ll * a->num_free},
                      {"prefix_table", a->prefix_table, 4ll * a->prefix_pages}};
  const Bytes out[] = {{"tables", a->tables, 4ll * a->seqs * a->max_pages}, {"used", a->used, 8}};
  if (!apart(out, 2, in, 3)) return QMK_ERR_INVALID_ARG;
  DeviceScope scope(device);
  if (scope.err != cudaSuccess) return paged_fail(scope.err, "cudaSetDevice");
  TableParams p;
  p.lengths = a->lengths; p.free_pages = a->free_pages; p.prefix_table = a->prefix_table;
  p.tables = a->tables; p.used = a->used;
  p.seqs = a->seqs; p.num_free = a->num_free; p.prefix_pages = a->prefix_pages; p.page_shift = shift; p.max_pages = a->max_pages;
  // a row per warp while the CTAs fit the machine at once (eight a multiprocessor), more beyond
  int rows = kTableThreads / 32;
  while ((long long)rows * 8 * 148 < a->seqs && rows < kTableThreads) rows *= 2;
  p.rows_per_cta = rows;
  block_tables_kernel<<<(unsigned)((a->seqs + rows - 1) / rows), kTableThreads, 0, (cudaStream_t)cuda_stream>>>(p);
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? QMK_OK : paged_fail(e, "block_tables_kernel");
}

extern "C" int qmk_build_slot_map(const qmk_slot_map_args* a, int device, void* cuda_stream) {
  g_paged_err[0] = 0;
  if (!a || a->seqs < 1 || a->seqs > kMaxTableSeqs || a->tokens < 1 || a->tokens > kMaxTableTokens || a->max_pages < 1 ||
      a->max_pages > kMaxTablePages)
    return QMK_ERR_INVALID_ARG;
  const int shift = page_shift_of(a->page_size);
  if (shift < 0 || !a->block_tables || !a->kv_lengths || !a->new_lengths || !a->slots || !a->positions || !a->seq_ids ||
      !a->active || !a->cu_tokens || !a->kv_lengths_out)
    return QMK_ERR_INVALID_ARG;
  const Bytes in[] = {{"block_tables", a->block_tables, 4ll * a->seqs * a->max_pages}, {"kv_lengths", a->kv_lengths, 4ll * a->seqs},
                      {"new_lengths", a->new_lengths, 4ll * a->seqs}};
  const Bytes out[] = {{"slots", a->slots, 8ll * a->tokens}, {"positions", a->positions, 4ll * a->tokens},
                       {"seq_ids", a->seq_ids, 4ll * a->tokens}, {"active", a->active, a->tokens},
                       {"cu_tokens", a->cu_tokens, 4ll * (a->seqs + 1)}, {"kv_lengths_out", a->kv_lengths_out, 4ll * a->seqs}};
  if (!apart(out, 6, in, 3)) return QMK_ERR_INVALID_ARG;
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

// ------------------------------------------------------------------------------------------------ attention
static int sm_count(int device) {
  static std::atomic<int> known[64];
  if (device < 0) return 0;
  int n = device < 64 ? known[device].load(std::memory_order_relaxed) : 0;
  if (n > 0) return n;
  if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, device) != cudaSuccess) {
    cudaGetLastError();
    return 0;
  }
  if (device < 64) known[device].store(n, std::memory_order_relaxed);
  return n;
}

// Regions of the workspace; every one starts on a 256-byte boundary.
struct WorkspaceLayout { long long refused, aborted, dense_ml, dense_o, strip_ml, strip_o, dense_desc, strip_desc, total; };
static WorkspaceLayout workspace_layout(const PlanDims& d, int head_dim) {
  WorkspaceLayout w;
  long long at = 0;
  auto take = [&](long long bytes) { const long long here = at; at += (bytes + 255) / 256 * 256; return here; };
  const long long records = max_dense_records(d), strips = max_strip_records(d);
  w.refused = take(4);
  w.aborted = take((long long)d.ctas * kStripWarps * 4);
  w.dense_ml = take(records * kUnitRows * 8);
  w.strip_ml = take(strips * kStripRows * 8);
  w.dense_desc = take((long long)d.tokens * d.NKV * 8);
  w.strip_desc = take((long long)d.tokens * d.NKV * d.G * 8);
  w.dense_o = take(records * kUnitRows * head_dim * 4);
  w.strip_o = take(strips * kStripRows * head_dim * 4);
  w.total = at;
  return w;
}

// The device counts blocks, pieces and records in 32 bits.
static bool counts_fit(const PlanDims& d) {
  const long long most = 0x7fffffffll, strips = max_strips(d), by_request = (long long)d.seqs * (kMostShort / kStripRows) * d.NKV;
  return max_units(d) * d.NKV * (d.room / kBlockKeys + 1) <= most && max_strip_records(d) <= most &&
         (strips < by_request ? strips : by_request) * (d.room / kPieceKeys + 1 + kStripCost) <= most;
}

static bool attention_sizes_ok(int tokens, int seqs, int num_heads, int num_kv_heads, int head_dim, int prefix_len) {
  return tokens >= 1 && tokens <= (1 << 20) && seqs >= 1 && seqs <= kMaxSeqs && (head_dim == 64 || head_dim == 128) &&
         num_kv_heads >= 1 && num_heads >= 1 && num_heads <= 1024 && num_heads % num_kv_heads == 0 &&
         num_heads / num_kv_heads <= kMaxGroup && prefix_len >= 0;
}

extern "C" int64_t qmk_prefix_attention_workspace(int32_t tokens, int32_t seqs, int32_t num_heads, int32_t num_kv_heads,
                                                  int32_t head_dim, int32_t prefix_len, int device) {
  if (!attention_sizes_ok(tokens, seqs, num_heads, num_kv_heads, head_dim, prefix_len)) return QMK_ERR_INVALID_ARG;
  const int ctas = sm_count(device);
  if (ctas < 1) return QMK_ERR_DEVICE;
  return workspace_layout(make_dims(tokens, seqs, num_heads / num_kv_heads, num_kv_heads, head_dim, prefix_len, 0, ctas), head_dim).total;
}

static int attention_args(const qmk_prefix_attention_args* a) {
  if (!a) return QMK_ERR_INVALID_ARG;
  if (a->num_heads > 1024) return refuse("more than 1024 query heads");
  if (!attention_sizes_ok(a->tokens, a->seqs, a->num_heads, a->num_kv_heads, a->head_dim, a->prefix_len)) return QMK_ERR_INVALID_ARG;
  if (a->max_pages < 1 || a->num_pages < 1) return QMK_ERR_INVALID_ARG;
  if (page_shift_of(a->page_size) < 0 || a->prefix_len % a->page_size != 0) return QMK_ERR_INVALID_ARG;
  // positions and rows of the pool are 32-bit coordinates
  if ((long long)a->max_pages * a->page_size > (1ll << 30) || a->prefix_len > (1 << 30) ||
      (long long)a->num_pages * a->page_size > (1ll << 31) - 1024)
    return refuse("more than 2^30 positions, or more than 2^31 - 1024 rows in the pool");
  if (a->prefix_len > 0 && !a->prefix_table) return QMK_ERR_INVALID_ARG;
  if (!a->block_tables || !a->kv_lengths || !a->cu_tokens || !a->q || !a->out || !a->k_pages || !a->v_pages || !a->workspace)
    return QMK_ERR_INVALID_ARG;
  const long long row = (long long)a->num_heads * a->head_dim;
  if (a->q_token_stride < row || a->out_token_stride < row || a->q_token_stride % 8 != 0 || a->out_token_stride % 8 != 0)
    return QMK_ERR_INVALID_ARG;
  if (!aligned_to(a->q, 16) || !aligned_to(a->out, 16)) return refuse("q and out must be 16-byte aligned");
  if (!aligned_to(a->k_pages, 16) || !aligned_to(a->v_pages, 16)) return refuse("the pages must be 16-byte aligned");
  if (!aligned_to(a->workspace, 256)) return refuse("the workspace must be 256-byte aligned");
  // (log2(e) * scale is what the kernel multiplies by)
  if (!(a->scale > 0.f) || isinf(a->scale * 1.4426950408889634f)) return refuse("the scale is not a positive number in 32 bits");
  return QMK_OK;
}

typedef CUresult (*encode_fn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                              const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                              CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
static encode_fn tensor_map_encoder() {
  static std::atomic<void*> known{nullptr};
  void* fn = known.load(std::memory_order_relaxed);
  if (fn) return (encode_fn)fn;
  cudaDriverEntryPointQueryResult q;
  if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &fn, cudaEnableDefault, &q) != cudaSuccess || !fn ||
      q != cudaDriverEntryPointSuccess) {
    cudaGetLastError();
    return nullptr;
  }
  known.store(fn, std::memory_order_relaxed);
  return (encode_fn)fn;
}
// The pool as {HD, NKV, rows}; boxes of 64 dimensions of one head, `box_rows` rows.  Rows outside read as zeros.
static bool pool_map(encode_fn enc, CUtensorMap* m, const void* base, const qmk_prefix_attention_args* a, int box_rows) {
  const cuuint64_t dims[3] = {(cuuint64_t)a->head_dim, (cuuint64_t)a->num_kv_heads, (cuuint64_t)a->num_pages * a->page_size};
  const cuuint64_t strides[2] = {(cuuint64_t)a->head_dim * 2, (cuuint64_t)a->head_dim * 2 * a->num_kv_heads};
  const cuuint32_t box[3] = {64, 1, (cuuint32_t)box_rows}, es[3] = {1, 1, 1};
  return enc(m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(base), dims, strides, box, es,
             CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_128B,
             CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// 32 rows of a KV head a block, and the fewer dimensions to a thread the fewer rows there are: all blocks of a small call run at
// once, a thread of a large one weighs the parts once for several quads.  9 pieces behind 8192 keys at 16/8 heads x 128: 342 us with
// a quad to a thread, 324 with eight, four of them read together; 32 rows at 32/8 x 64: 18.0 with one, 24.9 with four.
template <int HD>
static dim3 merge_grid(const PlanDims& d) {
  const long long blocks = (long long)((d.tokens * d.G + 31) / 32) * d.NKV;
  unsigned z = HD / 4 / (kMergeThreads / 32);
  while (z > 1 && blocks * z > kMergeBlocks) z /= 2;
  return dim3((unsigned)((d.tokens * d.G + 31) / 32), (unsigned)d.NKV, z);
}

template <int HD>
static int launch_attention(const qmk_prefix_attention_args* a, const AttnParams& p, const AttnMaps& maps, int device,
                            cudaStream_t stream) {
  using S = AttnSmem<HD>;
  static std::atomic<unsigned long long> ready{0};                  // devices whose kernel may use its shared memory
  cudaError_t e;
  const unsigned long long bit = device < 64 ? 1ull << device : 0ull;
  if (!(ready.load(std::memory_order_relaxed) & bit)) {
    e = cudaFuncSetAttribute(prefix_attention_kernel<HD>, cudaFuncAttributeMaxDynamicSharedMemorySize, S::total(kMaxSeqs));
    if (e != cudaSuccess) return paged_fail(e, "cudaFuncSetAttribute");
    ready.fetch_or(bit, std::memory_order_relaxed);
  }
  prefix_attention_kernel<HD><<<(unsigned)p.d.ctas, kAttnThreads, S::total(p.d.seqs), stream>>>(p, maps);
  e = cudaGetLastError();
  if (e != cudaSuccess) return paged_fail(e, "prefix_attention_kernel");
  cudaLaunchConfig_t cfg;
  memset(&cfg, 0, sizeof(cfg));
  cfg.gridDim = merge_grid<HD>(p.d);
  if (p.status) cfg.gridDim.x += 1;                                  // (the block that reports)
  cfg.blockDim = dim3(kMergeThreads);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;   // (the kernel waits for its predecessor itself)
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  e = cfg.gridDim.z < HD / 4 / (kMergeThreads / 32) ? cudaLaunchKernelEx(&cfg, merge_kernel<HD, true>, p)
                                                    : cudaLaunchKernelEx(&cfg, merge_kernel<HD, false>, p);
  return e == cudaSuccess ? QMK_OK : paged_fail(e, "merge_kernel");
}

static PlanDims call_dims(const qmk_prefix_attention_args* a, int ctas) {
  return make_dims(a->tokens, a->seqs, a->num_heads / a->num_kv_heads, a->num_kv_heads, a->head_dim, a->prefix_len,
                   a->max_pages * a->page_size, ctas);
}

int qmk_prefix_attention_check(const qmk_prefix_attention_args* a, int device) {
  g_paged_err[0] = 0;
  const int rc = attention_args(a);
  if (rc) return rc;
  const int ctas = sm_count(device);
  if (ctas < 2) return QMK_ERR_DEVICE;
  const PlanDims d = call_dims(a, ctas);
  if (!counts_fit(d))
    return refuse("rows and the room of prefix and tables: their units of 256 rows x 128 keys, or strips of 8 rows x 32 keys, do not count in "
                  "32 bits");
  if (a->workspace_bytes < workspace_layout(d, a->head_dim).total) return refuse("the workspace is too small");
  return QMK_OK;
}

extern "C" int qmk_prefix_attention(const qmk_prefix_attention_args* a, int device, void* cuda_stream) {
  const qmk_attention_watch nobody = {nullptr, 0, 4000000000ll, 0};   // (waits of about two seconds)
  return qmk_prefix_attention_launch(a, &nobody, device, cuda_stream);
}

int qmk_prefix_attention_launch(const qmk_prefix_attention_args* a, const qmk_attention_watch* watch, int device, void* cuda_stream) {
  const int rc = qmk_prefix_attention_check(a, device);
  if (rc) return rc;
  DeviceScope scope(device);
  if (scope.err != cudaSuccess) return paged_fail(scope.err, "cudaSetDevice");
  AttnParams p;
  memset(&p, 0, sizeof(p));
  p.d = call_dims(a, sm_count(device));
  const WorkspaceLayout w = workspace_layout(p.d, a->head_dim);
  p.q = (const uint16_t*)a->q; p.out = (uint16_t*)a->out; p.lse = a->lse;
  p.tables = a->block_tables; p.kv_lengths = a->kv_lengths; p.cu_tokens = a->cu_tokens; p.prefix_table = a->prefix_table;
  p.q_stride = a->q_token_stride; p.out_stride = a->out_token_stride;
  p.NH = a->num_heads; p.page_shift = page_shift_of(a->page_size); p.num_pages = a->num_pages; p.max_pages = a->max_pages;
  p.scale_log2e = a->scale * 1.4426950408889634f;
  p.status = watch->status; p.phase = watch->phase; p.wait_first = watch->wait_first;
  const long long budget = (watch->wait_cycles + 1023) / 1024;
  p.wait_budget = (unsigned)(budget < 1 ? 1 : (budget > 0xffffffffll ? 0xffffffffll : budget));
  unsigned char* ws = (unsigned char*)a->workspace;
  p.refused = (int*)(ws + w.refused); p.aborted = (unsigned*)(ws + w.aborted);
  p.dense_ml = (float2*)(ws + w.dense_ml); p.dense_o = (float4*)(ws + w.dense_o);
  p.strip_ml = (float2*)(ws + w.strip_ml); p.strip_o = (float*)(ws + w.strip_o);
  p.dense_desc = (int2*)(ws + w.dense_desc); p.strip_desc = (int2*)(ws + w.strip_desc);
  encode_fn enc = tensor_map_encoder();
  if (!enc) {
    snprintf(g_paged_err, sizeof(g_paged_err), "cudaGetDriverEntryPoint(cuTensorMapEncodeTiled)");
    return QMK_ERR_CUDA;
  }
  AttnMaps maps;
  const int box = a->page_size < 64 ? a->page_size : 64;
  if (!pool_map(enc, &maps.k, a->k_pages, a, box) || !pool_map(enc, &maps.v, a->v_pages, a, box) ||
      !pool_map(enc, &maps.k16, a->k_pages, a, 16) || !pool_map(enc, &maps.v16, a->v_pages, a, 16)) {
    snprintf(g_paged_err, sizeof(g_paged_err), "cuTensorMapEncodeTiled failed");
    return QMK_ERR_CUDA;
  }
  return a->head_dim == 64 ? launch_attention<64>(a, p, maps, device, (cudaStream_t)cuda_stream)
                           : launch_attention<128>(a, p, maps, device, (cudaStream_t)cuda_stream);
}
