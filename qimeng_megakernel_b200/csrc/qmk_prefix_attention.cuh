// Attention over a paged KV cache whose requests share a prefix.
//
//   row i of request s (n_s rows this step, kv_s tokens in the cache with them):  lim = kv_s - n_s + i + 1
//   o = sum_{j < lim} softmax_j(scale * q . k_j) v_j,    lse = log sum_{j < lim} exp(scale * q . k_j)
//   position j lies in page prefix_table[j / page] for j < prefix_len and in block_tables[s][j / page] behind it
//
// One persistent CTA per SM works through its share of the plan (qmk_prefix_plan.h): blocks or strips.
//
// Blocks.  Up to 256 rows against 128 keys at a time with tcgen05.mma, in the manner of a running softmax: S = Q K^T into
// tensor memory, softmax warps (one thread per row) turn S into P = exp2(S - m), rounded to bf16 and put over S, and O += P V.
// Two groups alternate, so that the tensor pipe works for one while the other does its exponentials: each has a tile of 128
// rows, or, where a unit has only one tile, they share it and take alternate blocks.  A group works in steps of 64 keys with
// two buffers for S, so that its next scores are there when it has written a P.  m is the row's first maximum and is raised
// (and O rescaled) only when a step's sum of exponentials passes 2^40: P keeps bf16's relative precision up to there, and a
// step looks for no maximum.
//   tensor memory: S (2 groups x 2 buffers x 64 columns, P over S), O0 | O1 (HD columns each)
//   warps 0-3, 4-7 softmax groups; 8 and 11 load K and V blocks (one TMA box per page and 64 dimensions); 9 and 10 issue the
//   products of a group each
//
// Strips.  What a short request holds behind the prefix: 8 rows x a run of 32-key pieces per warp, on mma.sync with the keys
// (for P V the dimensions) as the long side of the tile, K and V through a ring of the warp's own in shared memory.
//
// P is rounded to bf16 because the instruction takes one 16-bit type for both operands: 2^-8 of a probability at most, 0.0015 of the
// output in the root mean square (its own rounding is 0.0017); the sum l is over the unrounded values.
//
// What bounds it (B200, whole calls at 1965 MHz).  Many rows: the softmax warps' steps.  One of 64 keys for both groups (256 rows)
// takes about 1450 clocks, 1070 of them the exponentials of the two warps that share a scheduler (768 of the exponential unit), the
// rest reading S, writing P and the barriers, which nothing of the same warp runs beside; the products take 630 clocks of the tensor
// pipe at head size 64.  4 pieces of 500..1100 tokens behind 32768 shared keys at 32/8 heads x 64: 1079 us, 740 TFLOP/s; 9 pieces
// behind 8192 at 16/8 x 128, where a step has twice the products: 324 us, 1065 TFLOP/s (372 us at the 1660 MHz that the power limit
// leaves when it runs on).  Few rows: the latency of plan, first loads, last block and merge, about 11.4 us in all (2 rows), and
// the bytes: 64 rows behind 12288 keys at 16/8 x 128 44 us, 4.3 TB/s.
//
// Both parts leave partial results (m, l, unnormalised O, all in 32 bits) unless a row is complete; merge_kernel adds them
// up in a fixed order, so a call gives the same bits every time.  Nothing is kept between calls.
//
// Every wait is bounded: one that expires raises the CTA's abort word, all waits then return, the CTA's rows are NaN, and the
// caller's status record, if there is one, says so.
#pragma once
#include <cuda.h>
#include <stdint.h>

#include "qmk_device.cuh"
#include "qmk_params.h"
#include "qmk_prefix_plan.h"

namespace qmkp {

using namespace qmk;

struct AttnParams {
  const uint16_t* q;           // [tokens, NH, HD], q_stride elements from token to token
  uint16_t* out;               // [tokens, NH, HD], out_stride elements from token to token
  float* lse;                  // [tokens, NH] or null
  const int* tables;           // [seqs, max_pages]
  const int* kv_lengths;       // [seqs]
  const int* cu_tokens;        // [seqs + 1]
  const int* prefix_table;     // [prefix_len / page]
  long long q_stride, out_stride;
  PlanDims d;
  int NH, page_shift, num_pages, max_pages;
  float scale_log2e;
  // workspace
  float4* dense_o;             // [records, HD / 4, 256]   four dimensions of every row side by side
  float2* dense_ml;            // [records, 256]   (m in log2 units, l)
  float* strip_o;              // [records, 8, HD]
  float2* strip_ml;            // [records, 8]
  int2* dense_desc;            // [tokens, NKV]    {first record, records | row << 16}; records 0: none
  int2* strip_desc;            // [tokens, NH]     {first record, records | row << 16}
  int* refused;                // 1: cu_tokens does not ascend from 0 to at most `tokens`, nothing was computed
  unsigned* aborted;           // [CTAs, 8]  not 0: a wait expired there (one word for each warp with strips; blocks set all).  Zeroed at
                               // the CTA's start and set on failure only: a store at its end would make every call longer (0.2 us)
  // failures: the merge, which runs behind all CTAs, reports them
  unsigned* status;            // record of StatusWord, or null
  int phase;                   // of the step, for the record
  unsigned wait_budget;        // of every wait, in units of 1024 clocks
  int wait_first;              // failure test: every CTA waits for an arrival that nothing makes
};
struct AttnMaps {
  CUtensorMap k, v;            // {HD, NKV, slots}, box {64, 1, min(page, 64)}
  CUtensorMap k16, v16;        // the same, box {64, 1, 16}
};

constexpr int kAttnThreads = 384;
constexpr int kSoftmaxWarps = 8, kKeyWarp = 8, kIssueWarp = 9, kValueWarp = 11;   // (9 and 10 issue, one for each group)
struct Yes { static constexpr bool value = true; };
struct No { static constexpr bool value = false; };
constexpr int kPolyEvery = 4;                        // one pair of exponentials in so many goes to the multiply-add pipe

template <int HD>
struct AttnSmem {
  static constexpr int kHalves = HD / 64;
  static constexpr int kTileBytes = 128 * HD * 2;               // a 128-row Q tile
  static constexpr int kHalfBytes = 64 * HD * 2;                // K or V of half a block
  static constexpr int kStages = HD == 64 ? 8 : 4;              // halves of K, and of V, in the rings
  static constexpr int kOffQ = 0;
  static constexpr int kOffK = 2 * kTileBytes;
  static constexpr int kOffV = kOffK + kStages * kHalfBytes;
  static constexpr int kRing = kOffV + kStages * kHalfBytes;
  // strips: per warp a ring of kStripStages stages of 8 KiB
  static constexpr int kStripStages = 3, kStripStageBytes = 8192;
  static constexpr int kStageKeys = HD == 64 ? 32 : 16;         // keys of a stage
  static constexpr int kStripRing = kStripWarps * kStripStages * kStripStageBytes;
  static constexpr int kOffBars = kRing > kStripRing ? kRing : kStripRing;
  static constexpr int kDenseBars = 4 * kStages + 15;
  static constexpr int kNumBars = kDenseBars + kStripWarps * kStripStages;
  static constexpr int kOffCtl = kOffBars + kNumBars * 8;       // words: 0 abort, 1 tensor memory base
  static constexpr int kOffRed = (kOffCtl + 16 + 15) / 16 * 16;   // int4 [12] scratch of the scan
  static constexpr int kOffWork = kOffRed + kAttnThreads / 32 * 16;   // Work
  static constexpr int kOffMl = (kOffWork + 128 + 15) / 16 * 16;   // float2 [256]  m and l of the groups' rows
  static constexpr int kOffScan = kOffMl + 256 * 8;             // int [4][seqs + 1]
  static __host__ __device__ constexpr int total(int seqs) { return kOffScan + 4 * (seqs + 1) * 4; }
};

// ------------------------------------------------------------------------------------------------ primitives
__device__ __forceinline__ void tma_box(uint32_t dst, const CUtensorMap* map, int x, int y, int z, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(dst),
      "l"(map), "r"(x), "r"(y), "r"(z), "r"(bar)
      : "memory");
}
__device__ __forceinline__ void mbar_arrive(uint32_t bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void fence_async_shared() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
// Operand in shared memory, 128-byte swizzle.  K-major (Q, K): 8-row groups 1024 bytes apart.
__device__ __forceinline__ uint64_t desc_k_major(uint32_t addr) {
  return (uint64_t)((addr >> 4) & 0x3fffu) | (1ull << 16) | ((uint64_t)(1024u >> 4) << 32) | (1ull << 46) | (2ull << 61);
}
// V as the N x K operand, N (the dimensions) contiguous: 64-dimension atoms `half_bytes` apart, groups of 8 keys 1024 bytes.
__device__ __forceinline__ uint64_t desc_n_major(uint32_t addr, uint32_t half_bytes) {
  return (uint64_t)((addr >> 4) & 0x3fffu) | ((uint64_t)(half_bytes >> 4) << 16) | ((uint64_t)(1024u >> 4) << 32) |
         (1ull << 46) | (2ull << 61);
}
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t add) {
  asm volatile(
      "{\n.reg .pred p;\nsetp.ne.u32 p, %4, 0;\n"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}\n" ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(add)
      : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t add) {
  asm volatile(
      "{\n.reg .pred p;\nsetp.ne.u32 p, %4, 0;\n"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}\n" ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(add)
      : "memory");
}
__device__ __forceinline__ void mma_commit_to(uint32_t bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void tmem_ld32(float* r, uint32_t addr) {
  uint32_t* u = reinterpret_cast<uint32_t*>(r);
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,"
      "%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(u[0]), "=r"(u[1]), "=r"(u[2]), "=r"(u[3]), "=r"(u[4]), "=r"(u[5]), "=r"(u[6]), "=r"(u[7]), "=r"(u[8]), "=r"(u[9]),
        "=r"(u[10]), "=r"(u[11]), "=r"(u[12]), "=r"(u[13]), "=r"(u[14]), "=r"(u[15]), "=r"(u[16]), "=r"(u[17]), "=r"(u[18]),
        "=r"(u[19]), "=r"(u[20]), "=r"(u[21]), "=r"(u[22]), "=r"(u[23]), "=r"(u[24]), "=r"(u[25]), "=r"(u[26]), "=r"(u[27]),
        "=r"(u[28]), "=r"(u[29]), "=r"(u[30]), "=r"(u[31])
      : "r"(addr)
      : "memory");
}
__device__ __forceinline__ void tmem_st32(uint32_t addr, const uint32_t* u) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,"
      "%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(addr),
      "r"(u[0]), "r"(u[1]), "r"(u[2]), "r"(u[3]), "r"(u[4]), "r"(u[5]), "r"(u[6]), "r"(u[7]), "r"(u[8]), "r"(u[9]), "r"(u[10]),
      "r"(u[11]), "r"(u[12]), "r"(u[13]), "r"(u[14]), "r"(u[15]), "r"(u[16]), "r"(u[17]), "r"(u[18]), "r"(u[19]), "r"(u[20]),
      "r"(u[21]), "r"(u[22]), "r"(u[23]), "r"(u[24]), "r"(u[25]), "r"(u[26]), "r"(u[27]), "r"(u[28]), "r"(u[29]), "r"(u[30]),
      "r"(u[31])
      : "memory");
}
// Waits for loads; the 32 values are of use behind it only, whatever order the compiler gives the rest.
__device__ __forceinline__ void tmem_wait_ld_of(float* r) {
#define F4(i) "+f"(r[i]), "+f"(r[i + 1]), "+f"(r[i + 2]), "+f"(r[i + 3])
  asm volatile("tcgen05.wait::ld.sync.aligned;" : F4(0), F4(4), F4(8), F4(12), F4(16), F4(20), F4(24), F4(28)::"memory");
#undef F4
}
__device__ __forceinline__ float ex2(float x) {   // 2^x, 2 ulp; results below 2^-126 are zero
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  uint32_t u;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(u) : "f"(hi), "f"(lo));
  return u;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float y;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(y) : "f"(a), "f"(b), "f"(c));
  return y;
}
__device__ __forceinline__ float max3_nan(float a, float b, float c) {   // NaN if any of them is
  float y;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(y) : "f"(a), "f"(b), "f"(c));
  return y;
}
// Two floats in a register pair.
typedef unsigned long long f32x2;
__device__ __forceinline__ f32x2 pair(float lo, float hi) {
  f32x2 v;
  asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(lo), "f"(hi));
  return v;
}
__device__ __forceinline__ void unpair(f32x2 v, float& lo, float& hi) { asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v)); }
__device__ __forceinline__ f32x2 fma2(f32x2 a, f32x2 b, f32x2 c) {
  f32x2 v;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(v) : "l"(a), "l"(b), "l"(c));
  return v;
}
__device__ __forceinline__ f32x2 add2(f32x2 a, f32x2 b) {
  f32x2 v;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(v) : "l"(a), "l"(b));
  return v;
}
// 2^x of a pair on the fused multiply-add pipe, for x <= 127; below -126, and for a NaN, the result is about 2^-126 (whoever calls
// this looks for NaN himself).  x = n + f with n the
// nearest whole number (an addition of 1.5 * 2^23 rounds to it and leaves it in the low bits), 2^f on [-1/2, 1/2] by the
// polynomial of degree 4 with the smallest largest relative error (2.6e-6, found by Remez exchange), n into the exponent.
__device__ __forceinline__ void ex2_pair(f32x2 x, float& lo, float& hi) {
  float a, b;
  unpair(x, a, b);
  x = pair(fmaxf(a, -126.f), fmaxf(b, -126.f));
  const f32x2 magic = pair(12582912.f, 12582912.f), back = pair(-12582912.f, -12582912.f), minus = pair(-1.f, -1.f);
  const f32x2 t = add2(x, magic);
  const f32x2 f = fma2(add2(t, back), minus, x);
  f32x2 r = fma2(f, pair(0.009570102207362652f, 0.009570102207362652f), pair(0.05591785907745361f, 0.05591785907745361f));
  r = fma2(r, f, pair(0.240247443318367f, 0.240247443318367f));
  r = fma2(r, f, pair(0.6931217908859253f, 0.6931217908859253f));
  r = fma2(r, f, pair(0.9999992847442627f, 0.9999992847442627f));
  float n0, n1;
  unpair(t, n0, n1);
  unpair(r, lo, hi);
  lo = __uint_as_float(__float_as_uint(lo) + (__float_as_uint(n0) << 23));
  hi = __uint_as_float(__float_as_uint(hi) + (__float_as_uint(n1) << 23));
}
__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldsm4_t(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ uint32_t transpose8(uint32_t a) {   // of an 8 x 8 fragment of 16-bit values
  uint32_t d;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
  return d;
}
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// One lane of the (whole) warp.
__device__ __forceinline__ bool elect_one() {
  uint32_t one;
  asm volatile("{\n.reg .pred p;\nelect.sync _|p, 0xffffffff;\nselp.u32 %0, 1, 0, p;\n}\n" : "=r"(one));
  return one != 0u;
}
// Bounded wait on a phase of a barrier; false once the CTA has been aborted.  The hint (1 ms) lets the hardware park the warp:
// one that polls takes issue slots from the softmax warps of its scheduler (measured: 3 % of a long step).
__device__ __forceinline__ uint32_t mbar_try_wait_parked(uint32_t bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n.reg .pred p;\nmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\nselp.u32 %0, 1, 0, p;\n}\n"
      : "=r"(ok) : "r"(bar), "r"(parity), "r"(1000000u) : "memory");
  return ok;
}
__device__ __forceinline__ bool wait_bar(uint32_t bar, uint32_t parity, volatile unsigned* ctl, const AttnParams& p) {
  if (mbar_try_wait_parked(bar, parity)) return true;
  const long long t0 = clock64();
  while (!mbar_try_wait_parked(bar, parity)) {
    if (clock64() - t0 > (long long)p.wait_budget * 1024) ctl[0] = 1u;
    if (ctl[0] != 0u) return false;
  }
  return true;
}

// ------------------------------------------------------------------------------------------------ plan
struct Scans {                 // prefix sums over the requests, in shared memory, seqs + 1 entries each
  int* long_blocks;
  int* long_units;
  int* short_tokens;
  int* pieces;                 // of one KV head
};
__device__ __forceinline__ Req load_request(const AttnParams& p, int s) {
  return request(p.d, p.cu_tokens[s], p.cu_tokens[s + 1], p.kv_lengths[s]);
}
// The last entry of a[0 .. n] that is at most v (a[0] = 0 <= v < a[n]).
__device__ __forceinline__ int find_last(const int* a, int n, int v) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (a[mid] <= v) lo = mid; else hi = mid;
  }
  return lo;
}
struct Work {                  // in shared memory
  Totals t;
  Plan plan;
};
// Prefix sums of the requests' numbers and the plan.  One pass takes as many requests as the CTA has threads; only warps that
// have some take part in the sums.  False: cu_tokens does not ascend from 0 to at most `tokens`, so rows would belong to several
// requests or to none, and what they leave would not fit the workspace.
__device__ __forceinline__ bool build_plan(const AttnParams& p, const Scans& sc, int4* red, Work* out) {
  const int seqs = p.d.seqs, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int4 base = make_int4(0, 0, 0, 0);
  bool bad = false;
  for (int s0 = 0; s0 < seqs; s0 += kAttnThreads) {
    const int s = s0 + (int)threadIdx.x;
    const int warps = (min(seqs - s0, kAttnThreads) + 31) / 32;
    int4 v = make_int4(0, 0, 0, 0), x;
    if (warp < warps) {
      if (s < seqs) {
        const int c0 = p.cu_tokens[s], c1 = p.cu_tokens[s + 1];
        bad |= c0 > c1 || c1 > p.d.tokens || (s == 0 && c0 != 0);
        const Req r = request(p.d, c0, c1, p.kv_lengths[s]);
        if (is_long(p.d, r)) {
          const int n = units_of(p.d, r);
          for (int u = 0; u < n; ++u) v.x += unit_blocks(p.d, r, u);
          v.y = n;
        } else {
          v.z = r.n;
          v.w = strips_of(p.d, r) * pieces_of(p.d, r);
        }
      }
      x = v;
#pragma unroll 1
      for (int o = 1; o < 32; o <<= 1) {                     // (rolled, like what else runs once: its code comes from afar)
        const int a = __shfl_up_sync(kFullMask, x.x, o), b = __shfl_up_sync(kFullMask, x.y, o);
        const int c = __shfl_up_sync(kFullMask, x.z, o), d = __shfl_up_sync(kFullMask, x.w, o);
        if (lane >= o) { x.x += a; x.y += b; x.z += c; x.w += d; }
      }
      if (lane == 31) red[warp] = x;
    }
    __syncthreads();
    if (warp < warps) {
      int4 at = base;
      for (int w = 0; w < warps; ++w) {
        const int4 y = red[w];
        if (w < warp) { at.x += y.x; at.y += y.y; at.z += y.z; at.w += y.w; }
        base.x += y.x; base.y += y.y; base.z += y.z; base.w += y.w;
      }
      if (s < seqs) {
        sc.long_blocks[s] = at.x + x.x - v.x;
        sc.long_units[s] = at.y + x.y - v.y;
        sc.short_tokens[s] = at.z + x.z - v.z;
        sc.pieces[s] = at.w + x.w - v.w;
      }
    }
    if (s0 + kAttnThreads < seqs) __syncthreads();           // (the scratch is written again)
  }
  if (threadIdx.x == 0) {                                    // (its warp has taken part in every pass)
    sc.long_blocks[seqs] = base.x;
    sc.long_units[seqs] = base.y;
    sc.short_tokens[seqs] = base.z;
    sc.pieces[seqs] = base.w;
  }
  if (warp == 0) {                                           // each lane weighs one division of the CTAs
    const Totals t{base.x, base.y, base.z, base.w};
    Choice c = plan_choice(p.d, t, lane);
    // (times are positive: their bits order like them; the lane's number takes the last five, and breaks ties)
    const int best = (int)(__reduce_min_sync(kFullMask, (__float_as_uint(c.time) & ~31u) | (unsigned)lane) & 31u);
    c.ctas = __shfl_sync(kFullMask, c.ctas, best);
    c.each = __shfl_sync(kFullMask, c.each, best);
    if (lane == 0) {
      out->t = t;
      out->plan = make_plan(p.d, t, c);
    }
  }
  return !__syncthreads_or(bad);
}

// A unit of one KV head.
struct Unit {
  int kvh, index;       // index among the KV head's units
  int s, u;             // long: request and unit inside it; short: s = -1, u = unit among the short ones
  int blocks, limit;    // 128-key blocks; keys the unit's rows can see
  int rows;             // packed rows that exist
  Req r;
};
__device__ __forceinline__ Unit unit_at(const AttnParams& p, const Scans& sc, const Totals& t, const Plan& plan, int b,
                                        int& block) {
  Unit x;
  x.kvh = b / plan.blocks;
  int rest = b - x.kvh * plan.blocks;
  if (rest < t.long_blocks) {
    int lo = find_last(sc.long_blocks, p.d.seqs, rest);
    rest -= sc.long_blocks[lo];
    x.s = lo;
    x.r = load_request(p, lo);
    x.u = 0;
    for (;; ++x.u) {
      x.blocks = unit_blocks(p.d, x.r, x.u);
      if (rest < x.blocks) break;
      rest -= x.blocks;
    }
    x.index = sc.long_units[lo] + x.u;
    x.limit = unit_limit(p.d, x.r, x.u);
    x.rows = min(p.d.unit_tokens, x.r.n - x.u * p.d.unit_tokens) * p.d.G;
  } else {
    rest -= t.long_blocks;
    x.s = -1;
    x.blocks = p.d.prefix_blocks;
    x.u = rest / x.blocks;
    rest -= x.u * x.blocks;
    x.index = t.long_units + x.u;
    x.limit = p.d.prefix_len;
    x.rows = min(p.d.unit_tokens, t.short_tokens - x.u * p.d.unit_tokens) * p.d.G;
    x.r = Req{0, 0, 0};
  }
  block = rest;
  return x;
}
// The row `row` of a unit: token (-1: none) and the keys it sees of the unit's.
__device__ __forceinline__ int row_token(const AttnParams& p, const Scans& sc, const Unit& x, int row, int& lim) {
  lim = 0x7fffffff;
  if (row >= x.rows) return -1;
  const int i = p.d.by_G.div(row);
  if (x.s >= 0) {
    const int t = x.u * p.d.unit_tokens + i;
    lim = limit_of(p.d, x.r, t);
    return x.r.first + t;
  }
  const int at = x.u * p.d.unit_tokens + i;
  const int s = find_last(sc.short_tokens, p.d.seqs, at);
  const Req r = load_request(p, s);
  const int t = at - sc.short_tokens[s];
  lim = min(limit_of(p.d, r, t), p.d.prefix_len);
  return r.first + t;
}

// ------------------------------------------------------------------------------------------------ blocks
template <int HD>
struct Dense {
  using S = AttnSmem<HD>;
  const AttnParams& p;
  const AttnMaps& maps;
  unsigned char* smem;
  uint32_t base;               // shared address of smem
  volatile unsigned* ctl;
  Scans sc;
  const Totals& t;             // (in shared memory: read where they are needed, not held in registers)
  const Plan& plan;
  int lo, hi;                  // blocks of this CTA
  uint32_t tmem;
  int warp, lane;

  __device__ __forceinline__ uint32_t bar(int i) const { return base + S::kOffBars + i * 8; }
  __device__ __forceinline__ uint32_t k_full(int s) const { return bar(s); }
  __device__ __forceinline__ uint32_t k_empty(int s) const { return bar(S::kStages + s); }
  __device__ __forceinline__ uint32_t v_full(int s) const { return bar(2 * S::kStages + s); }
  __device__ __forceinline__ uint32_t v_empty(int s) const { return bar(3 * S::kStages + s); }
  // A waiter tells a phase by its parity alone, so every barrier below is one whose next phase cannot complete before all its
  // waiters have seen the last one.
  __device__ __forceinline__ uint32_t s_full(int g, int half) const { return bar(4 * S::kStages + 2 * g + half); }
  __device__ __forceinline__ uint32_t p_full(int g, int half) const { return bar(4 * S::kStages + 4 + 2 * g + half); }
  __device__ __forceinline__ uint32_t o_full(int g, int half) const { return bar(4 * S::kStages + 8 + 2 * g + half); }   // once a segment
  __device__ __forceinline__ uint32_t q_full(int g) const { return bar(4 * S::kStages + 12 + g); }   // segments in which g has steps
  __device__ __forceinline__ uint32_t v_clear() const { return bar(4 * S::kStages + 14); }

  // Steps of a group in a segment of nb blocks: halves of 64 keys of the blocks it takes (with two tiles every block, with
  // one the blocks of its parity).
  __device__ __forceinline__ static int steps_of(int nb, bool dual, int g) { return 2 * (dual ? (nb + 1 - g) >> 1 : nb); }
  __device__ __forceinline__ static int block_of(int j, bool dual, int g) { return dual ? (j & ~1) + g : j >> 1; }

  // keys of half a block of a unit that rows can see
  __device__ __forceinline__ static int valid_keys(const Unit& x, int b, int half) { return max(0, min(64, x.limit - b * kBlockKeys - 64 * half)); }

  __device__ __forceinline__ int page_of(const Unit& x, int key) const {
    int id;
    if (key < p.d.prefix_len) id = p.prefix_table[key >> p.page_shift];
    else id = x.s >= 0 ? p.tables[(size_t)x.s * p.max_pages + (key >> p.page_shift)] : -1;
    return id;
  }
  // K (or V) of the CTA's blocks, half by half: lane l loads box l of a half (a page, or 64 rows of one, of 64 dimensions).  K and
  // V have a warp each: the scores run up to a block ahead of the products with V.
  template <bool kV>
  __device__ __forceinline__ unsigned produce() {
    const int box_rows = min(1 << p.page_shift, 64);
    const int key_of_lane = (lane / S::kHalves) * box_rows, half_dims = lane % S::kHalves;
    const int boxes = 64 / box_rows * S::kHalves;
    const int oob = p.num_pages << p.page_shift;             // behind the last row: reads as zeros
    const uint32_t dst = base + (kV ? S::kOffV : S::kOffK) + (uint32_t)(half_dims * 8192 + key_of_lane * 128);
    unsigned n = 0;
    if (!kV && p.wait_first && !wait_bar(v_clear(), 0u, ctl, p)) return n;   // (V is cleared behind the first scores only)
    for (int b = lo; b < hi;) {
      int b0;
      const Unit x = unit_at(p, sc, t, plan, b, b0);
      const int nb = min(x.blocks - b0, hi - b), end = 2 * (b0 + nb);
      auto row_of = [&](int part) {                          // row of the pool that this lane's box of a half starts at, -1: no box
        const int key = part * 64 + key_of_lane;
        if (lane >= boxes || key >= x.limit) return -1;
        const int id = page_of(x, key);
        if (id < 0 || id >= p.num_pages) return oob;
        return (id << p.page_shift) + (key & ((1 << p.page_shift) - 1));
      };
      int row = row_of(2 * b0);
      for (int part = 2 * b0; part < end; ++part, ++n) {
        const int st = n % S::kStages;
        const uint32_t full = kV ? v_full(st) : k_full(st), empty = kV ? v_empty(st) : k_empty(st);
        const unsigned issue = __ballot_sync(kFullMask, row >= 0);
        const uint32_t bytes = (uint32_t)__popc(issue) * (uint32_t)(box_rows * 128);
        const int next = part + 1 < end ? row_of(part + 1) : -1;
        if (!wait_bar(empty, ((n / S::kStages) & 1u) ^ 1u, ctl, p)) return n;
        if (lane == 0) mbar_expect_tx(full, bytes);
        __syncwarp();
        if (row >= 0) tma_box(dst + st * S::kHalfBytes, kV ? &maps.v : &maps.k, half_dims * 64, x.kvh, row, full);
        row = next;
      }
      b += nb;
    }
    return n;
  }
  // After an abort: no copy stays in flight.
  template <bool kV>
  __device__ __forceinline__ void drain(unsigned issued) const {
    const unsigned from = issued > (unsigned)S::kStages ? issued - S::kStages : 0u;
    for (unsigned n = from; n < issued; ++n) {
      const long long t0 = clock64();
      while (!mbar_try_wait(kV ? v_full(n % S::kStages) : k_full(n % S::kStages), (n / S::kStages) & 1u))
        if (clock64() - t0 > 1000000) break;
    }
  }

  // S = Q K^T and O += P V of group g for the CTA's blocks (one lane of a warp per group: a lane spends about as long on
  // issuing a step as a group on its exponentials).  For every half of 64 keys: its P is waited for, P V is issued, and then the
  // scores of the same half of the next block into the buffer that P leaves; those of the other half are there already.
  // A block is released by both groups; with one tile the other group's part is an arrival without products.
  __device__ __forceinline__ void issue(int g) {
    constexpr uint32_t kIdescS = (1u << 4) | (1u << 7) | (1u << 10) | ((64u >> 3) << 17) | ((128u >> 4) << 24);
    constexpr uint32_t kIdescO = (1u << 4) | (1u << 7) | (1u << 10) | (1u << 16) | (((uint32_t)HD >> 3) << 17) | ((128u >> 4) << 24);
    const uint64_t kd0 = desc_k_major(base + S::kOffK), vd0 = desc_n_major(base + S::kOffV, 8192u);
    const uint32_t sd = tmem + (uint32_t)g * 128u, od = tmem + 256u + (uint32_t)g * 128u;
    unsigned n = 0, segs = 0, p_par = 0;                     // (p_par: parity of the next P, both halves)
    for (int b = lo; b < hi;) {
      int b0;
      const Unit x = unit_at(p, sc, t, plan, b, b0);
      const int nb = min(x.blocks - b0, hi - b);
      const bool dual = x.rows <= 128;
      const uint64_t qd = desc_k_major(base + S::kOffQ + (dual ? 0 : g) * S::kTileBytes);
      const int step = dual ? 2 : 1;
      auto score = [&](int st, int half) {
        const uint64_t kd = kd0 + (uint32_t)(st * (S::kHalfBytes >> 4));
#pragma unroll
        for (int k = 0; k < HD / 16; ++k) {
          const uint32_t q_off = (uint32_t)((k >> 2) * (16384 >> 4) + (k & 3) * (32 >> 4));
          const uint32_t k_off = (uint32_t)((k >> 2) * (8192 >> 4) + (k & 3) * (32 >> 4));
          if (k == 0) mma_ss(sd + 64u * half, qd + q_off, kd + k_off, kIdescS, 0u);
          else mma_ss(sd + 64u * half, qd + q_off, kd + k_off, kIdescS, 1u);
        }
        mma_commit_to(s_full(g, half));
      };
      auto release = [&](uint32_t empty) {
        mma_commit_to(empty);
        if (dual) mbar_arrive(empty);
      };
      int blk = dual ? g : 0;
      if (blk < nb) {
        if (!wait_bar(q_full(g), segs & 1u, ctl, p)) return;
        ++segs;
        // halves are numbered n, n + 1, ...: those of block blk are m and m + 1
        unsigned m = n + 2u * (unsigned)blk;
        auto score_when_there = [&](unsigned i, int half) {
          const int st = (int)(i % S::kStages);
          if (!wait_bar(k_full(st), (i / S::kStages) & 1u, ctl, p)) return false;
          tmem_fence_after_sync();
          score(st, half);
          release(k_empty(st));
          return true;
        };
        if (!score_when_there(m, 0) || !score_when_there(m + 1, 1)) return;
        uint32_t more = 0;                                   // 0 for the first products of the segment: O is overwritten
        for (; blk < nb; blk += step) {
          const bool next = blk + step < nb;
          const unsigned mn = m + 2u * (unsigned)step;
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            const int st = (int)((m + half) % S::kStages), valid = valid_keys(x, b0 + blk, half);
            const uint64_t vd = vd0 + (uint32_t)(st * (S::kHalfBytes >> 4));
            if (!wait_bar(v_full(st), ((m + half) / S::kStages) & 1u, ctl, p)) return;
            if (!wait_bar(p_full(g, half), p_par, ctl, p)) return;
            tmem_fence_after_sync();
            if (valid == 64) {
              mma_ts(od, sd + 64u * half, vd, kIdescO, more);
#pragma unroll
              for (int k = 1; k < 4; ++k) mma_ts(od, sd + 64u * half + 8u * k, vd + (uint32_t)(k * (2048 >> 4)), kIdescO, 1u);
              more = 1u;
            } else {
#pragma unroll 1
              for (int k = 0; 16 * k < valid; ++k) {
                mma_ts(od, sd + 64u * half + 8u * k, vd + (uint32_t)(k * (2048 >> 4)), kIdescO, more);
                more = 1u;
              }
            }
            release(v_empty(st));
            if (next) {
              if (!score_when_there(mn + half, half)) return;
            } else {
              mma_commit_to(o_full(g, half));
            }
          }
          p_par ^= 1u;
          m = mn;
        }
      }
      n += 2u * (unsigned)nb;
      b += nb;
    }
  }

  // Rows of V behind the last visible key of a half: cleared, so that 0 * V is 0 whatever the page holds there.  (One warp,
  // before its P is handed over; rows from the next multiple of 16 on are not read.)
  __device__ __forceinline__ void clear_rows(int st, int valid) {
    const int rows = 16 - (valid & 15);
    for (int i = lane; i < rows * 8 * S::kHalves; i += 32) {
      const int r = valid + i / (8 * S::kHalves), c = i % (8 * S::kHalves);
      *reinterpret_cast<uint4*>(smem + S::kOffV + st * S::kHalfBytes + (c >> 3) * 8192 + r * 128 + (c & 7) * 16) =
          make_uint4(0, 0, 0, 0);
    }
    fence_async_shared();
    __syncwarp();
  }

  __device__ __forceinline__ void softmax() {
    const int g = warp >> 2, row = g * 128 + (warp & 3) * 32 + lane;
    const uint32_t lane_base = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t s_col = tmem + g * 128 + lane_base, o_col = tmem + 256 + g * 128 + lane_base;
    unsigned s_par = 0;                                      // parity of the next S, both halves
    unsigned n = 0, clears = 0, o_par = 0;
    for (int b = lo; b < hi;) {
      int b0;
      const Unit x = unit_at(p, sc, t, plan, b, b0);
      const int nb = min(x.blocks - b0, hi - b);
      const bool dual = x.rows <= 128;
      // Q: thread `row` brings row `row` of the unit (with one tile the second group's threads have nothing to bring)
      int lim;
      const int tile_row = dual && g == 1 ? row - 128 : row;
      const int token = row_token(p, sc, x, tile_row, lim);
      const int head = x.kvh * p.d.G + p.d.by_G.mod(tile_row);
      if (!(dual && g == 1)) {
        const uint4* src = reinterpret_cast<const uint4*>(p.q + (size_t)max(token, 0) * p.q_stride + (size_t)head * HD);
        unsigned char* dst = smem + S::kOffQ + g * S::kTileBytes + (row & 127) * 128;
#pragma unroll
        for (int c = 0; c < HD / 8; ++c) {
          const uint4 v = token >= 0 ? __ldg(src + c) : make_uint4(0, 0, 0, 0);
          *reinterpret_cast<uint4*>(dst + (c >> 3) * 16384 + (((c & 7) ^ (row & 7)) << 4)) = v;
        }
        fence_async_shared();
      }
      tmem_fence_before_sync();                       // (the O of the segment before has been read)
      asm volatile("bar.sync 1, 256;" ::: "memory");  // (nobody arrives for a segment before all have left the last)
      mbar_arrive(q_full(0));
      if (steps_of(nb, dual, 1) > 0) mbar_arrive(q_full(1));
      const bool warp_works = __ballot_sync(kFullMask, token >= 0) != 0u;
      const int warp_lim = __reduce_min_sync(kFullMask, lim);
      float m = -INFINITY, l = 0.f;
      bool seen = false;                              // every row of the warp has an m
      const int steps = steps_of(nb, dual, g);
      // the step of the half in which the keys end inside 16 of them: its V is cleared behind them, by a warp of the group
      int clear_step = -1;
      if ((warp & 3) == 0 && (x.limit & 15) != 0) {
        const int blk = x.limit / kBlockKeys - b0;
        if (blk >= 0 && blk < nb && (!dual || (blk & 1) == g)) clear_step = (dual ? blk - g : 2 * blk) + ((x.limit >> 6) & 1);
      }
      bool ok = true;
      for (int j = 0; j < steps; ++j) {
        const int half = j & 1;
        const uint32_t sh = s_col + 64 * half;
        ok = wait_bar(s_full(g, half), s_par, ctl, p);
        if (!ok) break;
        tmem_fence_after_sync();
        if (warp_works) {
          float s[64];
          tmem_ld32(s, sh);
          tmem_wait_ld_of(s);
          tmem_ld32(s + 32, sh + 32);
          const int k0 = (b0 + block_of(j, dual, g)) * kBlockKeys + 64 * half;
          const f32x2 scale2 = pair(p.scale_log2e, p.scale_log2e);
          float sum = 0.f, most = -INFINITY;
          uint32_t pk[32];
          // 2^(scale s - m) of the row, packed, and their sum.  One pair in kPolyEvery goes to the multiply-add pipe; the
          // largest exponent of those is noted (a NaN before all), the others say themselves when they are too large or NaN.
          auto exps = [&](auto with_poly, int first) {       // of the 32 from `first` on
            const float off = m == -INFINITY ? 0.f : m;
            const f32x2 off2 = pair(-off, -off);
            f32x2 sum2[2] = {0ull, 0ull};
#pragma unroll
            for (int u = 0; u < 16; ++u) {
              const int i = first / 2 + u;
              const f32x2 e = fma2(pair(s[2 * i], s[2 * i + 1]), scale2, off2);
              float a, d;
              unpair(e, a, d);
              if (decltype(with_poly)::value && i % kPolyEvery == kPolyEvery - 1) {
                most = max3_nan(most, a, d);
                ex2_pair(e, a, d);
              } else {
                a = ex2(a);
                d = ex2(d);
              }
              sum2[i & 1] = add2(sum2[i & 1], pair(a, d));
              pk[i] = pack2(a, d);
            }
            float a, d;
            unpair(add2(sum2[0], sum2[1]), a, d);
            sum += a + d;
          };
          bool done = false;
          const bool plain = k0 + 64 <= warp_lim;
          if (plain && seen) {
            exps(Yes{}, 0);
            tmem_wait_ld_of(s + 32);
            exps(Yes{}, 32);
            done = __all_sync(kFullMask, sum <= 1099511627776.f && most <= 40.f);
          }
          if (!done) {                                  // the first step, hidden keys, a score far above m, or a NaN
            tmem_wait_ld_of(s + 32);
            tmem_ld32(s, sh);                           // (read again: they need not be kept for this)
            tmem_ld32(s + 32, sh + 32);
            tmem_wait_ld_of(s);
            tmem_wait_ld_of(s + 32);
            if (!plain) {
              const int vis = lim - k0;
#pragma unroll
              for (int c = 0; c < 64; ++c) s[c] = c < vis ? s[c] : -INFINITY;
            }
            float mx[4] = {s[0], s[1], s[2], s[3]};
#pragma unroll
            for (int i = 4; i + 8 <= 64; i += 8)
#pragma unroll
              for (int c = 0; c < 4; ++c) mx[c] = max3(mx[c], s[i + c], s[i + 4 + c]);
#pragma unroll
            for (int c = 0; c < 4; ++c) mx[c] = fmaxf(mx[c], s[60 + c]);
            // (NaN scores: the maximum passes them over, their own exponential keeps them)
            const float top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * p.scale_log2e;
            if (__any_sync(kFullMask, top > m)) {
              const float m_new = fmaxf(m, top);
              if (j > 0) {
                // O may be touched once P V of step j - 1 is through: the scores of step j + 1 were issued behind it
                ok = j + 1 < steps ? wait_bar(s_full(g, half ^ 1), half ? s_par ^ 1u : s_par, ctl, p) : wait_bar(o_full(g, 0), o_par, ctl, p);
                if (!ok) break;
                tmem_fence_after_sync();
                const float f = m_new == -INFINITY ? 1.f : ex2(m - m_new);
                l *= f;
#pragma unroll 1
                for (int c = 0; c < HD / 16; ++c) {
                  uint32_t o[16];
                  tmem_ld16(o, o_col + 16 * c);
                  tmem_wait_ld();
#pragma unroll
                  for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * f);
                  tmem_st16(o_col + 16 * c, o);
                }
              }
              m = m_new;
              seen = __all_sync(kFullMask, m != -INFINITY);
            }
            sum = 0.f;
            exps(No{}, 0);
            exps(No{}, 32);
          }
          l += sum;
          tmem_st32(sh, pk);
          tmem_wait_st();
        }
        if (j == clear_step) {
          const unsigned at = n + 2u * (unsigned)block_of(j, dual, g) + (unsigned)half;
          const int st = (int)(at % S::kStages);
          if (dual || g == 0) {
            ok = wait_bar(v_full(st), (at / S::kStages) & 1u, ctl, p);
            if (!ok) break;
            clear_rows(st, x.limit & 63);
            if (!dual && lane == 0) mbar_arrive(v_clear());
          } else {                                           // (the block of both groups is cleared by the first)
            ok = wait_bar(v_clear(), clears & 1u, ctl, p);
            if (!ok) break;
            ++clears;
          }
        }
        tmem_fence_before_sync();
        mbar_arrive(p_full(g, half));
        s_par ^= (unsigned)half;
      }
      if (ok && steps > 0) ok = wait_bar(o_full(g, 1), o_par, ctl, p);
      if (steps > 0) o_par ^= 1u;
      tmem_fence_after_sync();
      // ---- the unit's rows: complete, or a record.  With one tile both groups have a part of every row (in the same lanes
      // of tensor memory): they add the two up, half of the dimensions each ----
      const int cta = (int)blockIdx.x;
      const bool whole = b0 == 0 && nb == x.blocks && x.s >= 0;
      const int rec = cta + x.kvh * plan.unit_total + x.index;
      float f = 1.f, f_other = 0.f;                   // factors of this group's O and of the other's
      if (!ok) l = __int_as_float(0x7fffffff);
      if (dual) {
        float2* ml = reinterpret_cast<float2*>(smem + S::kOffMl);
        ml[row] = make_float2(m, l);
        tmem_fence_before_sync();
        asm volatile("bar.sync 2, 256;" ::: "memory");
        tmem_fence_after_sync();
        const float2 other = ml[row ^ 128];
        const float top = fmaxf(m, other.x);
        f = m == -INFINITY ? 0.f : ex2(m - top);
        f_other = other.x == -INFINITY ? 0.f : ex2(other.x - top);
        l = l * f + other.y * f_other;
        if (!(other.y == other.y) || !ok) l = __int_as_float(0x7fffffff);
        m = top;
      } else if (steps == 0 || m == -INFINITY) {
        f = 0.f;
      }
      if (warp_works) {
        const float inv = l == 0.f ? 0.f : 1.f / l;
        const uint32_t other_col = tmem + 256 + (g ^ 1) * 128 + lane_base;
        uint16_t* out = p.out + (size_t)max(token, 0) * p.out_stride + (size_t)head * HD;
        float4* part = p.dense_o + (size_t)rec * (HD / 4) * kUnitRows + tile_row;
        const int c0 = dual ? g * (HD / 32) : 0, c1 = dual ? c0 + HD / 32 : HD / 16;
#pragma unroll 1
        for (int c = c0; c < c1; ++c) {
          uint32_t o[16];
          tmem_ld16(o, o_col + 16 * c);
          if (dual) {
            uint32_t u[16];
            tmem_ld16(u, other_col + 16 * c);
            tmem_wait_ld();
#pragma unroll
            for (int i = 0; i < 16; ++i)               // (a factor of zero: whatever stands there does not count)
              o[i] = __float_as_uint((f != 0.f ? f * __uint_as_float(o[i]) : 0.f) + (f_other != 0.f ? f_other * __uint_as_float(u[i]) : 0.f));
          } else {
            tmem_wait_ld();
#pragma unroll
            for (int i = 0; i < 16; ++i) o[i] = f != 0.f ? o[i] : 0u;
          }
          if (token >= 0) {
            if (whole) {
#pragma unroll
              for (int i = 0; i < 2; ++i) {
                uint32_t w[4];
#pragma unroll
                for (int k = 0; k < 4; ++k) w[k] = pack2(__uint_as_float(o[8 * i + 2 * k]) * inv, __uint_as_float(o[8 * i + 2 * k + 1]) * inv);
                reinterpret_cast<uint4*>(out + 16 * c)[i] = make_uint4(w[0], w[1], w[2], w[3]);
              }
            } else {
#pragma unroll
              for (int i = 0; i < 4; ++i)
                part[(4 * c + i) * kUnitRows] = make_float4(__uint_as_float(o[4 * i]), __uint_as_float(o[4 * i + 1]),
                                                            __uint_as_float(o[4 * i + 2]), __uint_as_float(o[4 * i + 3]));
            }
          }
        }
        if (token >= 0 && !(dual && g == 1)) {
          if (whole) {
            if (p.lse) p.lse[(size_t)token * p.NH + head] = l == 0.f ? -INFINITY : (m + log2f(l)) * 0.6931471805599453f;
          } else {
            p.dense_ml[(size_t)rec * kUnitRows + tile_row] = make_float2(l == l ? m : l, l);
          }
          // whoever starts the unit says where its rows' parts are
          if (b0 == 0 && p.d.by_G.mod(tile_row) == 0) {
            const int parts = whole ? 0 : plan.dense_owner(b + x.blocks - 1) - cta + 1;
            p.dense_desc[(size_t)token * p.d.NKV + x.kvh] = make_int2(rec, parts | (tile_row << 16));
            if (x.s >= 0)
              for (int i = 0; i < p.d.G; ++i) p.strip_desc[(size_t)token * p.NH + head + i] = make_int2(0, 0);
          }
        }
      }
      n += 2u * (unsigned)nb;
      b += nb;
    }
  }
};

// ------------------------------------------------------------------------------------------------ strips
// g = lane / 4, t = lane % 4.  S^T = K Q^T: tiles of 16 keys x 8 rows (lane: keys g, g + 8 of rows 2t, 2t + 1); O^T = V^T P^T: tiles
// of 16 dimensions x 8 rows.  The P^T operand is the transpose of the S^T fragment: one movmatrix per 8 keys.  A lane's columns
// are the same two rows in both products, so a row's maximum and scale never leave its lanes.
// The part of a strip that a warp takes: pieces [c0, c0 + n), `stages` fills of the ring.
struct StripRun {
  Req r;
  int s, per, c0, n, kvh, strip, base_row, rows, k_lo, k_hi, stages;
};
__device__ __forceinline__ StripRun strip_at(const AttnParams& p, const Scans& sc, int f, int hi, int stage_keys) {
  StripRun x;
  x.s = find_last(sc.pieces, p.d.seqs, p.d.by_NKV.div(f));
  x.r = load_request(p, x.s);
  x.per = pieces_of(p.d, x.r);
  const int rest = f - sc.pieces[x.s] * p.d.NKV, column = rest / x.per;
  x.c0 = rest - column * x.per;
  x.n = min(x.per - x.c0, hi - f);
  x.strip = p.d.by_NKV.div(column);
  x.kvh = column - x.strip * p.d.NKV;
  x.base_row = x.strip * kStripRows;
  x.rows = min(kStripRows, x.r.n * p.d.G - x.base_row);
  x.k_lo = p.d.prefix_len + piece_lo(x.c0);
  x.k_hi = max(x.k_lo, min(p.d.prefix_len + piece_lo(x.c0 + x.n), limit_of(p.d, x.r, p.d.by_G.div(x.base_row + x.rows - 1))));
  x.stages = (x.k_hi - x.k_lo + stage_keys - 1) / stage_keys;
  return x;
}
template <int HD>
__device__ __forceinline__ void walk_strips(const AttnParams& p, const AttnMaps& maps, unsigned char* smem, volatile unsigned* ctl,
                                            const Scans& sc, const Plan& plan, int warp, int lane) {
  using S = AttnSmem<HD>;
  constexpr int KS = S::kStageKeys, TILES = KS / 16, HALVES = S::kHalves;
  constexpr int KBYTES = KS * HD * 2;                       // 4 KiB of K, then 4 KiB of V
  const uint32_t ring = smem_u32(smem) + warp * S::kStripStages * S::kStripStageBytes;
  const uint32_t bars = smem_u32(smem) + S::kOffBars + (S::kDenseBars + warp * S::kStripStages) * 8;
  const int g = lane >> 2, t4 = lane & 3;
  const int oob = p.num_pages << p.page_shift;
  int lo, hi;
  const int number = piece_range(p.d, plan, (int)blockIdx.x, warp, lo, hi);
  if (lo >= hi) return;
  // The fills run ahead of the products, into the next strips too: a short strip's table, pages and rows would otherwise be
  // waited for one after the other.
  unsigned sent = 0, used = 0;                              // stages filled and consumed by this warp
  int nf = lo, next = 0, held = -1, held_from = 0;          // strip being filled, its next stage, pool rows of 32 groups of 16 keys
  StripRun y = strip_at(p, sc, lo, hi, KS);
  auto group_row = [&](int grp) {
    const int key = y.k_lo + grp * 16;
    if (key >= y.k_hi) return -1;
    const int id = p.tables[(size_t)y.s * p.max_pages + (key >> p.page_shift)];
    if (id < 0 || id >= p.num_pages) return oob;
    return (id << p.page_shift) + (key & ((1 << p.page_shift) - 1));
  };
  held = group_row(lane);
  auto send = [&]() {                                        // the next fill; lane l < 2 * TILES * HALVES sends one box
    while (nf < hi && next >= y.stages) {
      nf += y.n;
      if (nf >= hi) return;
      y = strip_at(p, sc, nf, hi, KS);
      next = held_from = 0;
      held = group_row(lane);
      if (lane < y.rows) {                                   // (its rows of Q, for when it is taken up)
        const int i = y.base_row + lane;
        asm volatile("prefetch.global.L1 [%0];" ::"l"(p.q + (size_t)(y.r.first + p.d.by_G.div(i)) * p.q_stride +
                                                      (size_t)(y.kvh * p.d.G + p.d.by_G.mod(i)) * HD));
      }
    }
    if (nf >= hi) return;
    const int st = (int)(sent % S::kStripStages);
    const int grp0 = next * TILES;
    if (grp0 + TILES > held_from + 32) {
      held_from = grp0;
      held = group_row(grp0 + lane);
    }
    const int q = lane % (TILES * HALVES), kg = q / HALVES, half = q % HALVES;
    const bool is_v = lane >= TILES * HALVES;
    const int row = __shfl_sync(kFullMask, held, (grp0 + kg - held_from) & 31);
    const bool mine = lane < 2 * TILES * HALVES && row >= 0;
    const unsigned issue = __ballot_sync(kFullMask, mine);
    if (lane == 0) mbar_expect_tx(bars + st * 8, (uint32_t)__popc(issue) * 2048u);
    __syncwarp();
    if (mine)
      tma_box(ring + st * S::kStripStageBytes + (is_v ? KBYTES : 0) + (kg * HALVES + half) * 2048, is_v ? &maps.v16 : &maps.k16,
              half * 64, y.kvh, row, bars + st * 8);
    ++sent;
    ++next;
  };
  for (int i = 0; i < S::kStripStages; ++i) send();
  bool ok = true;
  if (p.wait_first) ok = wait_bar(smem_u32(smem) + S::kOffBars + (S::kDenseBars - 1) * 8, 0u, ctl, p);   // (a barrier of the blocks')
  for (int f = lo; f < hi;) {
    const StripRun x = strip_at(p, sc, f, hi, KS);
    const Req& r = x.r;
    const int s = x.s, per = x.per, c0 = x.c0, n = x.n, kvh = x.kvh, strip = x.strip, base_row = x.base_row, rows = x.rows;
    const int k_lo = x.k_lo, k_hi = x.k_hi, stages = x.stages;
    // row g of the strip as the column-major operand; the two rows this lane's results belong to
    uint32_t qb[HD / 16][2];
    {
      const int i = min(g, rows - 1) + base_row;
      const uint16_t* qp = p.q + (size_t)(r.first + p.d.by_G.div(i)) * p.q_stride + (size_t)(kvh * p.d.G + p.d.by_G.mod(i)) * HD + 2 * t4;
#pragma unroll
      for (int k = 0; k < HD / 16; ++k) {
        qb[k][0] = *reinterpret_cast<const uint32_t*>(qp + 16 * k);
        qb[k][1] = *reinterpret_cast<const uint32_t*>(qp + 16 * k + 8);
      }
    }
    const int lim0 = min(k_hi, limit_of(p.d, r, p.d.by_G.div(base_row + min(2 * t4, rows - 1))));
    const int lim1 = min(k_hi, limit_of(p.d, r, p.d.by_G.div(base_row + min(2 * t4 + 1, rows - 1))));
    float m0 = -INFINITY, m1 = -INFINITY, l0 = 0.f, l1 = 0.f;
    float o[HD / 16][4];
#pragma unroll
    for (int j = 0; j < HD / 16; ++j) o[j][0] = o[j][1] = o[j][2] = o[j][3] = 0.f;
    for (int i = 0; i < stages; ++i) {
      const int st = (int)(used % S::kStripStages);
      ok = ok && wait_bar(bars + st * 8, (used / S::kStripStages) & 1u, ctl, p);
      if (!ok) break;
      ++used;
      const uint32_t kb = ring + st * S::kStripStageBytes, vb = kb + KBYTES;
      const int key0 = k_lo + i * KS;
      const int valid = min(KS, k_hi - key0);
      if (valid < KS) {                                     // rows of V behind the last key: whatever they hold, 0 * V is to be 0
        unsigned char* vp = smem + warp * S::kStripStages * S::kStripStageBytes + st * S::kStripStageBytes + KBYTES;
        for (int e = lane; e < (KS - valid) * 8 * HALVES; e += 32) {
          const int rr = valid + e / (8 * HALVES), c = e % (8 * HALVES);
          *reinterpret_cast<uint4*>(vp + ((rr >> 4) * HALVES + (c >> 3)) * 2048 + (rr & 15) * 128 + (c & 7) * 16) = make_uint4(0, 0, 0, 0);
        }
        fence_async_shared();                               // (before a copy lands here again)
        __syncwarp();
      }
      float x[TILES][4];
#pragma unroll
      for (int j = 0; j < TILES; ++j) {
        float y[4] = {0.f, 0.f, 0.f, 0.f};
        x[j][0] = x[j][1] = x[j][2] = x[j][3] = 0.f;
        const int kr = lane & 15;
#pragma unroll
        for (int k = 0; k < HD / 16; ++k) {                 // (two chains of products)
          const int piece = 2 * k + (lane >> 4);
          uint32_t a[4];
          ldsm4(a, kb + (j * HALVES + (piece >> 3)) * 2048 + kr * 128 + (((piece & 7) ^ (kr & 7)) << 4));
          if (k & 1) mma16816(y, a, qb[k][0], qb[k][1]);
          else mma16816(x[j], a, qb[k][0], qb[k][1]);
        }
#pragma unroll
        for (int c = 0; c < 4; ++c) x[j][c] = (x[j][c] + y[c]) * p.scale_log2e;
      }
      if (key0 + KS > min(lim0, lim1)) {
#pragma unroll
        for (int j = 0; j < TILES; ++j) {
          const int key = key0 + 16 * j + g;
          x[j][0] = key < lim0 ? x[j][0] : -INFINITY;
          x[j][1] = key < lim1 ? x[j][1] : -INFINITY;
          x[j][2] = key + 8 < lim0 ? x[j][2] : -INFINITY;
          x[j][3] = key + 8 < lim1 ? x[j][3] : -INFINITY;
        }
      }
      float t0 = fmaxf(x[0][0], x[0][2]), t1 = fmaxf(x[0][1], x[0][3]);
#pragma unroll
      for (int j = 1; j < TILES; ++j) { t0 = max3(t0, x[j][0], x[j][2]); t1 = max3(t1, x[j][1], x[j][3]); }
      // m is raised only when a lane's part of a row asks for more than 2^8: then the row's lanes agree on the new one
      if (__any_sync(kFullMask, t0 > m0 + 8.f || t1 > m1 + 8.f)) {
#pragma unroll
        for (int d = 4; d < 32; d <<= 1) {
          t0 = fmaxf(t0, __shfl_xor_sync(kFullMask, t0, d));
          t1 = fmaxf(t1, __shfl_xor_sync(kFullMask, t1, d));
        }
        const float n0 = fmaxf(m0, t0), n1 = fmaxf(m1, t1);
        const float f0 = n0 == -INFINITY ? 1.f : ex2(m0 - n0), f1 = n1 == -INFINITY ? 1.f : ex2(m1 - n1);
        m0 = n0; m1 = n1;
        l0 *= f0; l1 *= f1;
#pragma unroll
        for (int j = 0; j < HD / 16; ++j) { o[j][0] *= f0; o[j][1] *= f1; o[j][2] *= f0; o[j][3] *= f1; }
      }
      const float off0 = m0 == -INFINITY ? 0.f : m0, off1 = m1 == -INFINITY ? 0.f : m1;
      uint32_t pb[TILES][2];
#pragma unroll
      for (int j = 0; j < TILES; ++j) {
        const float a = ex2(x[j][0] - off0), b = ex2(x[j][1] - off1), c = ex2(x[j][2] - off0), d = ex2(x[j][3] - off1);
        l0 += a + c;
        l1 += b + d;
        pb[j][0] = transpose8(pack2(a, b));
        pb[j][1] = transpose8(pack2(c, d));
      }
#pragma unroll
      for (int j = 0; j < TILES; ++j)
#pragma unroll
        for (int c = 0; c < HD / 16; ++c) {
          const int kr = (lane & 7) + ((lane >> 4) & 1) * 8, piece = 2 * c + ((lane >> 3) & 1);
          uint32_t a[4];
          ldsm4_t(a, vb + (j * HALVES + (piece >> 3)) * 2048 + kr * 128 + (((piece & 7) ^ (kr & 7)) << 4));
          mma16816(o[c], a, pb[j][0], pb[j][1]);
        }
      __syncwarp();                                         // every lane has read the stage
      send();
    }
#pragma unroll
    for (int d = 4; d < 32; d <<= 1) {
      l0 += __shfl_xor_sync(kFullMask, l0, d);
      l1 += __shfl_xor_sync(kFullMask, l1, d);
    }
    const float nan = __int_as_float(0x7fffffff);
    if (!ok) m0 = m1 = l0 = l1 = nan;
    const bool whole = p.d.prefix_len == 0 && n == per;
    const int rec = number + strip_number(p.d, s, sc.short_tokens[s], strip, kvh);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int row = 2 * t4 + h;
      if (row >= rows) continue;
      const float m = h ? m1 : m0, l = h ? l1 : l0;
      const int token = r.first + p.d.by_G.div(base_row + row), gq = p.d.by_G.mod(base_row + row), head = kvh * p.d.G + gq;
      if (whole) {
        const float inv = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : nan);
        uint16_t* dst = p.out + (size_t)token * p.out_stride + (size_t)head * HD + g;
#pragma unroll
        for (int j = 0; j < HD / 16; ++j) {
          dst[16 * j] = f32_to_bf16_bits(l == 0.f ? 0.f : o[j][h] * inv);
          dst[16 * j + 8] = f32_to_bf16_bits(l == 0.f ? 0.f : o[j][2 + h] * inv);
        }
        if (p.lse && g == 0) p.lse[(size_t)token * p.NH + head] = l == 0.f ? -INFINITY : (m + log2f(l)) * 0.6931471805599453f;
      } else {
        float* dst = p.strip_o + ((size_t)rec * kStripRows + row) * HD + g;
#pragma unroll
        for (int j = 0; j < HD / 16; ++j) {
          dst[16 * j] = o[j][h];
          dst[16 * j + 8] = o[j][2 + h];
        }
        // (a NaN is told from m: scores that are all NaN leave no maximum, and the merge would give such a part no weight)
        if (g == 0) p.strip_ml[(size_t)rec * kStripRows + row] = make_float2(l == l ? m : l, l);
      }
      if (c0 == 0 && g == 0) {                              // whoever starts the strip says where its rows' parts are
        const int parts = whole ? 0 : plan.strips.owner(f + per - 1) - number + 1;
        p.strip_desc[(size_t)token * p.NH + head] = make_int2(rec, parts | (row << 16));
        if (p.d.prefix_len == 0 && gq == 0) p.dense_desc[(size_t)token * p.d.NKV + kvh] = make_int2(0, 0);
      }
    }
    f += n;
  }
  for (; used < sent; ++used) {                             // after an abort: no copy stays in flight
    const long long w0 = clock64();
    while (!mbar_try_wait(bars + (used % S::kStripStages) * 8, (used / S::kStripStages) & 1u))
      if (clock64() - w0 > 1000000) break;
  }
}

// ------------------------------------------------------------------------------------------------ kernels
template <int HD>
__global__ void __launch_bounds__(kAttnThreads, 1)
prefix_attention_kernel(const __grid_constant__ AttnParams p, const __grid_constant__ AttnMaps maps) {
  using S = AttnSmem<HD>;
  extern __shared__ __align__(1024) unsigned char smem[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  volatile unsigned* ctl = reinterpret_cast<volatile unsigned*>(smem + S::kOffCtl);
  Scans sc;
  sc.long_blocks = reinterpret_cast<int*>(smem + S::kOffScan);
  sc.long_units = sc.long_blocks + p.d.seqs + 1;
  sc.short_tokens = sc.long_units + p.d.seqs + 1;
  sc.pieces = sc.short_tokens + p.d.seqs + 1;
  Work* work = reinterpret_cast<Work*>(smem + S::kOffWork);
  Dense<HD> w{p, maps, smem, smem_u32(smem), ctl, sc, work->t, work->plan, 0, 0, 0u, warp, lane};
  if (warp == kKeyWarp) {
    if (lane < 4) {
      const CUtensorMap* m = lane == 0 ? &maps.k : (lane == 1 ? &maps.v : (lane == 2 ? &maps.k16 : &maps.v16));
      asm volatile("prefetch.tensormap [%0];" ::"l"(m) : "memory");
    }
    // barriers: arrivals they wait for
    for (int i = lane; i < S::kNumBars; i += 32) {
      int count = 1;
      const int r = i - 4 * S::kStages;
      if (r < 0) count = (i / S::kStages) & 1 ? 2 : 1;       // full: the copy's bytes; empty: both groups
      else if (r >= 4 && r < 8) count = 128;                 // p_full: a group's four warps
      else if (r == 12 || r == 13) count = 256;              // q_full: all softmax warps
      mbar_init(w.bar(i), count);
    }
    if (lane == 0) ctl[0] = 0u;
    if (lane < kStripWarps) p.aborted[blockIdx.x * kStripWarps + lane] = 0u;
    fence_barrier_init();
  }
  if (warp == kIssueWarp) {                                  // (before it is known whether the CTA has blocks: it takes a while)
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(w.base + S::kOffCtl + 4) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    tmem_fence_before_sync();
  }
  const bool ok = build_plan(p, sc, reinterpret_cast<int4*>(smem + S::kOffRed), work);
  if (blockIdx.x == 0 && threadIdx.x == 0) *p.refused = !ok;
  if (!ok || (int)blockIdx.x >= work->plan.dense_ctas) {
    if (warp == kIssueWarp) {
      tmem_fence_after_sync();
      asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(ctl[1]) : "memory");
    }
    if (ok && warp < kStripWarps) {
      walk_strips<HD>(p, maps, smem, ctl, sc, work->plan, warp, lane);
      if (lane == 0 && ctl[0] != 0u) p.aborted[blockIdx.x * kStripWarps + warp] = 1u;
    }
    return;
  }
  dense_range(work->plan, (int)blockIdx.x, w.lo, w.hi);
  tmem_fence_after_sync();
  w.tmem = ctl[1];
  if (warp < kSoftmaxWarps) {
    w.softmax();
  } else if (warp == kKeyWarp) {
    const unsigned n = w.template produce<false>();
    __syncwarp();
    if (ctl[0] != 0u) w.template drain<false>(n);
  } else if (warp == kValueWarp) {
    const unsigned n = w.template produce<true>();
    __syncwarp();
    if (ctl[0] != 0u) w.template drain<true>(n);
  } else {
    if (elect_one()) w.issue(warp - kIssueWarp);
  }
  __syncwarp();
  tmem_fence_before_sync();
  __syncthreads();
  if (threadIdx.x < kStripWarps && ctl[0] != 0u) p.aborted[blockIdx.x * kStripWarps + threadIdx.x] = 1u;
  if (warp == kIssueWarp) {
    tmem_fence_after_sync();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(w.tmem) : "memory");
  }
}

constexpr int kMergeThreads = 128, kMergeParts = 8;
constexpr long long kMergeBlocks = 4 * 148 * 6;              // four waves of the blocks that fit the machine
// What failed goes to the status record, whose first entry stays.  A block beside those that merge does it, where there is a record.
static __device__ __noinline__ void report_failures(const int* refused, const unsigned* aborted, int ctas, unsigned* status, int phase,
                                                    int last, int tokens) {
  const bool offsets = *refused != 0;                        // (then no CTA has waited for anything)
#pragma unroll 4
  for (int i = (int)threadIdx.x; i < (offsets ? 1 : ctas * kStripWarps); i += kMergeThreads) {
    if (!offsets && aborted[i] == 0u) continue;
    if (atomicCAS(&status[kStCode], 0u, (unsigned)(offsets ? kErrRowOffsets : kErrCopyWait)) != 0u) continue;
    status[kStSm] = i / kStripWarps;
    status[kStWarp] = i % kStripWarps;
    status[kStPhase] = phase;
    status[kStSeen] = offsets ? last : 0;
    status[kStExpected] = offsets ? tokens : 0;
    status[kStDetail] = 0;
  }
}

// Adds a row's parts.  With M = max m_r and w_r = 2^(m_r - M):   o = sum_r w_r O_r / sum_r w_r l_r
// A thread takes four dimensions of a (row, KV head) at a time; neighbours take neighbouring rows, which is how the blocks' parts
// lie.  The statistics and values of eight parts are on their way at once, M is the running maximum (a part of weight zero may
// hold anything and is left out; one whose scores had a NaN has m = NaN and makes the row NaN).  A refused call's rows are NaN, all of
// them.  Launched as a programmatic dependent without an early trigger: blocks that wait on the SMs while the attention still runs
// cost it more (32 rows over 2048 shared keys: 24.6 us) than the plain order of launches (18.5 us); this takes 17.8 us (all before
// the present division of the CTAs, 16.5 us with it), of which about 4 us are the adding.
template <int HD, bool kMany>                                // kMany: a large call
__global__ void __launch_bounds__(kMergeThreads) merge_kernel(const __grid_constant__ AttnParams p) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if (p.status != nullptr && blockIdx.x == gridDim.x - 1) {
    if (blockIdx.y + blockIdx.z == 0)
      report_failures(p.refused, p.aborted, p.d.ctas, p.status, p.phase, p.cu_tokens[p.d.seqs], p.d.tokens);
    return;
  }
  const int row = (int)blockIdx.x * 32 + (int)(threadIdx.x & 31), kvh = (int)blockIdx.y;
  const int token = p.d.by_G.div(row), g = row - token * p.d.G, head = kvh * p.d.G + g;
  if (token >= p.d.tokens) return;
  const int rows = p.cu_tokens[p.d.seqs], refused = *p.refused;
  const int2 dd = p.dense_desc[(size_t)token * p.d.NKV + kvh], sd = p.strip_desc[(size_t)token * p.NH + head];
  const int nd = refused ? 0 : dd.y & 0xffff, ns = refused ? 0 : sd.y & 0xffff;
  if (!refused && (nd + ns == 0 || token >= rows)) return;
  const size_t drow = (size_t)dd.x * kUnitRows + ((unsigned)dd.y >> 16) + g, srow = (size_t)sd.x * kStripRows + ((unsigned)sd.y >> 16);
  const int parts = nd + ns, from = (int)blockIdx.z * (kMergeThreads / 32) + (int)(threadIdx.x >> 5);
  const int step = (int)gridDim.z * (kMergeThreads / 32);
  uint16_t* out = p.out + (size_t)token * p.out_stride + (size_t)head * HD;
  if (kMany && parts <= 2) {                                 // four quads on their way at once
    auto stat = [&](int r) { return __ldcg(r < nd ? p.dense_ml + drow + (size_t)r * kUnitRows : p.strip_ml + srow + (size_t)(r - nd) * kStripRows); };
    const float2 a = parts > 0 ? stat(0) : make_float2(-INFINITY, 0.f), b = parts > 1 ? stat(1) : make_float2(-INFINITY, 0.f);
    const float M = fmaxf(a.x, b.x);
    const float wa = M == -INFINITY ? 0.f : ex2(a.x - M), wb = M == -INFINITY ? 0.f : ex2(b.x - M);
    float L = (wa != 0.f ? wa * a.y : 0.f) + (wb != 0.f ? wb * b.y : 0.f);
    if (refused || a.x != a.x || b.x != b.x) L = __int_as_float(0x7fffffff);
    const bool none = L == 0.f;
    const float inv = none ? 0.f : 1.f / L;
#pragma unroll 1
    for (int c0 = from; c0 < HD / 4; c0 += 4 * step) {
      float4 va[4], vb[4];
      auto value = [&](int r, int c4) {
        return __ldcg(r < nd ? p.dense_o + (((size_t)dd.x + r) * (HD / 4) + c4) * kUnitRows + ((unsigned)dd.y >> 16) + g
                             : reinterpret_cast<const float4*>(p.strip_o + (srow + (size_t)(r - nd) * kStripRows) * HD + 4 * c4));
      };
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const bool there = c0 + i * step < HD / 4;
        va[i] = vb[i] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (there && wa != 0.f) va[i] = value(0, c0 + i * step);
        if (there && wb != 0.f) vb[i] = value(1, c0 + i * step);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float x = (wa * va[i].x + wb * vb[i].x) * inv, y = (wa * va[i].y + wb * vb[i].y) * inv;
        const float z = (wa * va[i].z + wb * vb[i].z) * inv, t = (wa * va[i].w + wb * vb[i].w) * inv;
        const uint2 w = none ? make_uint2(0u, 0u) : make_uint2(pack2(x, y), pack2(z, t));
        if (c0 + i * step < HD / 4) *reinterpret_cast<uint2*>(out + 4 * (c0 + i * step)) = w;
      }
    }
    if (p.lse && from == 0) p.lse[(size_t)token * p.NH + head] = none ? -INFINITY : (M + log2f(L)) * 0.6931471805599453f;
    return;
  }
  float2 ml[kMergeParts];
#pragma unroll 1
  for (int c4 = from, first = 1; c4 < HD / 4; c4 += step, first = 0) {      // dimensions 4 c4 ..
    const float4* dense = p.dense_o + ((size_t)dd.x * (HD / 4) + c4) * kUnitRows + ((unsigned)dd.y >> 16) + g;
    const float* strip = p.strip_o + srow * HD + 4 * c4;
    float M = -INFINITY, L = 0.f;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 1
    for (int r0 = 0; r0 < parts; r0 += kMergeParts) {
      float4 v[kMergeParts];
#pragma unroll
      for (int i = 0; i < kMergeParts; ++i) {
        const int r = r0 + i;
        if (first || parts > kMergeParts) {
          ml[i] = make_float2(-INFINITY, 0.f);
          if (r < parts) ml[i] = __ldcg(r < nd ? p.dense_ml + drow + (size_t)r * kUnitRows : p.strip_ml + srow + (size_t)(r - nd) * kStripRows);
        }
        v[i] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (r < parts)
          v[i] = __ldcg(r < nd ? dense + (size_t)r * (HD / 4) * kUnitRows
                               : reinterpret_cast<const float4*>(strip + (size_t)(r - nd) * kStripRows * HD));
      }
      float top = M;
      bool nan = false;
#pragma unroll
      for (int i = 0; i < kMergeParts; ++i) {
        top = fmaxf(top, ml[i].x);
        nan |= ml[i].x != ml[i].x;
      }
      const float f = M == -INFINITY ? 0.f : ex2(M - top);
      M = top;
      L = nan ? __int_as_float(0x7fffffff) : L * f;
      acc.x *= f; acc.y *= f; acc.z *= f; acc.w *= f;
#pragma unroll
      for (int i = 0; i < kMergeParts; ++i) {
        const float w = M == -INFINITY ? 0.f : ex2(ml[i].x - M);
        if (w != 0.f) {
          L += w * ml[i].y;
          acc.x += w * v[i].x; acc.y += w * v[i].y; acc.z += w * v[i].z; acc.w += w * v[i].w;
        }
      }
    }
    if (refused) L = __int_as_float(0x7fffffff);
    const bool none = L == 0.f;
    const float inv = none ? 0.f : 1.f / L;
    uint2 w = make_uint2(pack2(acc.x * inv, acc.y * inv), pack2(acc.z * inv, acc.w * inv));
    if (none) w = make_uint2(0u, 0u);
    *reinterpret_cast<uint2*>(out + 4 * c4) = w;
    if (p.lse && c4 == 0) p.lse[(size_t)token * p.NH + head] = none ? -INFINITY : (M + log2f(L)) * 0.6931471805599453f;
  }
}

}  // namespace qmkp
