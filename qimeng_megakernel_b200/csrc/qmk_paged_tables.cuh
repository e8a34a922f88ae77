// Block tables and slot maps of the paged KV cache, built on the device from request lengths.
//
// Both are a prefix sum over the requests followed by one write per table entry or token.  A CTA does not wait for
// another: it adds up what lies before its own share itself (the lengths of all requests are a few KB that every SM
// reads from L2), so a call is one launch without counters, scratch or atomics, and its result is the same every time.
#pragma once
#include <stdint.h>

#include "qmk_device.cuh"

namespace qmkp {

constexpr int kTableThreads = 256;
// A CTA reads the lengths of the requests before its own: a million of them keep a call within milliseconds.  Entries and tokens are
// counted in 32 bits with room for a pass's step.
constexpr int kMaxTableSeqs = 1 << 20, kMaxTablePages = 1 << 30, kMaxTableTokens = 1 << 24;

// Sum of v over the CTA, in every thread.  `red` has one word per warp.
__device__ __forceinline__ long long block_sum(long long v, long long* red) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(qmk::kFullMask, v, o);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  long long s = 0;
#pragma unroll
  for (int w = 0; w < kTableThreads / 32; ++w) s += red[w];
  return s;
}

// Inclusive prefix sum of v over the CTA's threads.
__device__ __forceinline__ long long block_scan(long long v, long long* red) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long u = __shfl_up_sync(qmk::kFullMask, v, o);
    if (lane >= o) v += u;
  }
  __syncthreads();
  if (lane == 31) red[warp] = v;
  __syncthreads();
  long long before = 0;
#pragma unroll
  for (int w = 0; w < kTableThreads / 32; ++w) before += w < warp ? red[w] : 0;
  return v + before;
}

struct TableParams {
  const int* lengths;        // [seqs]
  const int* free_pages;     // [num_free]
  const int* prefix_table;   // [prefix_pages]
  int* tables;               // [seqs, max_pages]
  int* used;                 // [2]
  int seqs, num_free, prefix_pages, page_shift, max_pages, rows_per_cta;
};

__device__ __forceinline__ int pages_wanted(int length, int page_shift) {
  return length > 0 ? (int)(((long long)length + (1 << page_shift) - 1) >> page_shift) : 0;
}
__device__ __forceinline__ int pages_own(const TableParams& p, int length) {
  const int n = min(pages_wanted(length, p.page_shift), p.max_pages) - p.prefix_pages;
  return n > 0 ? n : 0;
}

// Row s of the table:  n_s = min(ceil(len_s / page), max_pages) entries, the first prefix_pages of them the shared
// ones, the others taken from the free list behind those of the rows before:  first_s = sum_{t < s} own_t.
// Bound by the 4 * seqs * max_pages bytes written, or by the launch for a small batch.  A warp takes a row and a CTA eight: measured
// at 4096 requests x 512 entries 6.1 us by graph replay, 2.5 of it the launch.
__global__ void __launch_bounds__(kTableThreads) block_tables_kernel(const TableParams p) {
  __shared__ long long red[kTableThreads / 32];
  __shared__ long long first_s[kTableThreads];
  __shared__ int count_s[kTableThreads];
  const int r0 = (int)blockIdx.x * p.rows_per_cta, r1 = min(p.seqs, r0 + p.rows_per_cta);
  const int s = r0 + (int)threadIdx.x;
  const int len = s < r1 ? p.lengths[s] : 0;                 // (on its way with the others)
  long long v = 0, cut = 0;
  for (int s0 = 0; s0 < r0; s0 += 8 * kTableThreads) {       // (eight lengths on their way at a time)
    int before[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int t = s0 + i * kTableThreads + (int)threadIdx.x;
      before[i] = t < r0 ? p.lengths[t] : 0;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      v += pages_own(p, before[i]);
      cut += pages_wanted(before[i], p.page_shift) > p.max_pages;
    }
  }
  const long long base = block_sum(v, red);
  const int own = pages_own(p, len);
  const long long incl = block_scan(own, red);
  first_s[threadIdx.x] = base + incl - own;
  count_s[threadIdx.x] = min(pages_wanted(len, p.page_shift), p.max_pages);
  if (blockIdx.x == gridDim.x - 1) {   // the last CTA has seen every row
    cut += pages_wanted(len, p.page_shift) > p.max_pages;
    cut = block_sum(cut, red);
    const long long total = block_sum(own, red) + base;
    if (threadIdx.x == 0) {
      p.used[0] = (int)(total < 0x7fffffffll ? total : 0x7fffffffll);
      p.used[1] = (int)cut;
    }
  }
  __syncthreads();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (int r = warp; r0 + r < r1; r += kTableThreads / 32) {
    int* row = p.tables + (size_t)(r0 + r) * p.max_pages;
    const long long first = first_s[r] - p.prefix_pages;
    const int n = count_s[r];
    auto entry = [&](int j) {
      if (j >= n) return -1;
      if (j < p.prefix_pages) return p.prefix_table[j];
      return first + j < p.num_free ? p.free_pages[first + j] : -1;
    };
    // four passes of the row on their way at a time; entries four by four where rows start on 16 bytes
    if ((p.max_pages & 3) == 0 && (reinterpret_cast<uintptr_t>(p.tables) & 15u) == 0) {
      for (int j0 = 4 * lane; j0 < p.max_pages; j0 += 4 * 128) {
        int4 e[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int j = j0 + 128 * i;
          e[i] = make_int4(entry(j), entry(j + 1), entry(j + 2), entry(j + 3));
        }
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (j0 + 128 * i < p.max_pages) *reinterpret_cast<int4*>(row + j0 + 128 * i) = e[i];
      }
    } else {
      for (int j0 = lane; j0 < p.max_pages; j0 += 128) {
        int e[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) e[i] = entry(j0 + 32 * i);
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (j0 + 32 * i < p.max_pages) row[j0 + 32 * i] = e[i];
      }
    }
  }
}

struct SlotParams {
  const int* tables;         // [seqs, max_pages]
  const int* kv_lengths;     // [seqs]  tokens in the cache before the step
  const int* new_lengths;    // [seqs]  tokens the step appends
  long long* slots;          // [tokens]
  int* positions;            // [tokens]
  int* seq_ids;              // [tokens]
  unsigned char* active;     // [tokens]
  int* cu_tokens;            // [seqs + 1]
  int* kv_out;               // [seqs]
  int seqs, tokens, page_shift, max_pages;
};

constexpr int kSlotItems = 8;                                // requests per thread and pass
constexpr int kSlotChunk = kTableThreads * kSlotItems;       // requests per pass

// One thread per token.  Every CTA walks the requests in passes of kSlotChunk until it has met its own tokens:
//   cu_s = min(sum_{t < s} new_t, tokens)   position = kv_s + (token - cu_s)   slot = table[s][position / page] * page + position % page
// Pass c's cu_tokens and lengths are written by CTA c mod grid.  Bound by the launch and one pass's latency: 2.9 us for 64 requests of
// a token, 3.8 us for 16411 tokens of 777 by graph replay (where these took 3.5 and 4.3, kv_lengths kept beside cu in shared memory
// took 4.1 and 4.3).
__global__ void __launch_bounds__(kTableThreads) slot_map_kernel(const SlotParams p) {
  __shared__ long long red[kTableThreads / 32];
  __shared__ int cu_s[kSlotChunk + 1];
  const int passes = (p.seqs + kSlotChunk - 1) / kSlotChunk;
  int last_write = -1;                                       // the last pass this CTA writes out
  for (int c = (int)blockIdx.x; c < passes; c += (int)gridDim.x) last_write = c;
  const int t0 = (int)blockIdx.x * kTableThreads;
  const int token = t0 + (int)threadIdx.x;
  const long long t1 = (long long)t0 + kTableThreads;
  long long base = 0;
  int seq = -1, start = 0;
  for (int c = 0; c < passes && (base < t1 || c <= last_write); ++c) {
    long long sum = 0;
    int n[kSlotItems];
    const int s0 = c * kSlotChunk + (int)threadIdx.x * kSlotItems;
#pragma unroll
    for (int i = 0; i < kSlotItems; ++i) {
      n[i] = s0 + i < p.seqs ? max(p.new_lengths[s0 + i], 0) : 0;
      sum += n[i];
    }
    const long long incl = block_scan(sum, red);
    const long long all = block_sum(sum, red);
    long long at = base + incl - sum;
    __syncthreads();                                         // the searches of the pass before are done
#pragma unroll
    for (int i = 0; i < kSlotItems; ++i) {
      cu_s[threadIdx.x * kSlotItems + i] = (int)(at < p.tokens ? at : p.tokens);
      at += n[i];
    }
    if (threadIdx.x == kTableThreads - 1) cu_s[kSlotChunk] = (int)(at < p.tokens ? at : p.tokens);
    __syncthreads();
    if (c % (int)gridDim.x == (int)blockIdx.x) {
      for (int i = (int)threadIdx.x; i < kSlotChunk && c * kSlotChunk + i < p.seqs; i += kTableThreads) {
        const int s = c * kSlotChunk + i;
        p.cu_tokens[s] = cu_s[i];
        if (s == p.seqs - 1) p.cu_tokens[p.seqs] = cu_s[i + 1];
        const long long kv = (long long)max(p.kv_lengths[s], 0) + (cu_s[i + 1] - cu_s[i]);
        p.kv_out[s] = (int)(kv < 0x7fffffffll ? kv : 0x7fffffffll);
      }
    }
    if (seq < 0 && token < cu_s[kSlotChunk]) {               // (cu is clipped to `tokens`: a real token)
      int lo = 0, hi = kSlotChunk;                           // the last request of the pass that starts at or before the token
      while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (cu_s[mid] <= token) lo = mid; else hi = mid;
      }
      seq = c * kSlotChunk + lo;
      start = cu_s[lo];
    }
    base += all;
  }
  if (token >= p.tokens) return;
  long long slot = -1, pos = 0;
  if (seq >= 0) {
    pos = (long long)max(p.kv_lengths[seq], 0) + (token - start);
    const long long pg = pos >> p.page_shift;
    if (pg < p.max_pages) {
      const int page = p.tables[(size_t)seq * p.max_pages + pg];
      if (page >= 0) slot = ((long long)page << p.page_shift) + (pos & ((1 << p.page_shift) - 1));
    }
  }
  p.slots[token] = slot;
  p.positions[token] = (int)(pos < 0x7fffffffll ? pos : 0x7fffffffll);
  p.seq_ids[token] = seq;
  p.active[token] = slot >= 0 ? 1 : 0;
}

}  // namespace qmkp
