// Attention over a paged KV cache whose requests share a prefix.
//
//   row i of request s (n_s rows this step, kv_s tokens in the cache with them):  lim = kv_s - n_s + i + 1
//   o = sum_{j < lim} softmax_j(scale * q . k_j) v_j,    lse = log sum_{j < lim} exp(scale * q . k_j)
//   position j lies in page prefix_table[j / page] for j < prefix_len and in block_tables[s][j / page] behind it
#pragma once
#include <stdint.h>

#include "qmk_device.cuh"

namespace qmkp {

struct AttnParams {
  const uint16_t* q;           // [tokens, NH, HD], q_stride elements from token to token
  uint16_t* out;               // [tokens, NH, HD], out_stride elements from token to token
  float* lse;                  // [tokens, NH] or null
  const uint16_t* k_pages;     // [num_pages, page, NKV, HD]
  const uint16_t* v_pages;
  const int* tables;           // [seqs, max_pages]
  const int* kv_lengths;       // [seqs]
  const int* cu_tokens;        // [seqs + 1]
  const int* prefix_table;     // [prefix_len / page]
  long long q_stride, out_stride;
  int tokens, seqs, NH, NKV, page_shift, num_pages, max_pages, prefix_len;
  float scale_log2e;
};

// Request of a token: the last s with cu[s] <= token (empty requests before it share its start).
__device__ __forceinline__ int request_of(const int* cu, int seqs, int token) {
  int lo = 0, hi = seqs;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (cu[mid] <= token) lo = mid; else hi = mid;
  }
  return lo;
}

// One warp per (token, query head): lanes share the head's dimensions, the keys are walked one by one with the running
// maximum and sum of the softmax.
template <int HD>
__global__ void __launch_bounds__(128) prefix_attention_simple(const AttnParams p) {
  constexpr int PER = HD / 32;
  const int lane = threadIdx.x & 31;
  const long long row = (long long)blockIdx.x * 4 + (threadIdx.x >> 5);
  const int token = (int)(row / p.NH), head = (int)(row % p.NH);
  if (token >= p.tokens || token >= p.cu_tokens[p.seqs]) return;
  const int s = request_of(p.cu_tokens, p.seqs, token);
  const int n = p.cu_tokens[s + 1] - p.cu_tokens[s], i = token - p.cu_tokens[s];
  long long lim = (long long)p.kv_lengths[s] - n + i + 1;
  const long long room = max((long long)p.max_pages << p.page_shift, (long long)p.prefix_len);
  lim = lim < room ? lim : room;
  const int kvh = head / (p.NH / p.NKV);
  float q[PER], o[PER], m = -INFINITY, l = 0.f;
#pragma unroll
  for (int d = 0; d < PER; ++d) {
    q[d] = qmk::bf16_bits_to_f32(p.q[(size_t)token * p.q_stride + (size_t)head * HD + lane + 32 * d]);
    o[d] = 0.f;
  }
  const int page_mask = (1 << p.page_shift) - 1;
  for (int j = 0; j < lim; ++j) {
    const int page = j < p.prefix_len ? p.prefix_table[j >> p.page_shift] : p.tables[(size_t)s * p.max_pages + (j >> p.page_shift)];
    const bool held = page >= 0 && page < p.num_pages;
    const size_t at = ((((size_t)(held ? page : 0) << p.page_shift) + (j & page_mask)) * p.NKV + kvh) * HD + lane;
    float x = 0.f;
#pragma unroll
    for (int d = 0; d < PER; ++d) x += held ? q[d] * qmk::bf16_bits_to_f32(p.k_pages[at + 32 * d]) : 0.f;
    x = qmk::warp_sum(x) * p.scale_log2e;
    const float m_new = fmaxf(m, x);
    const float c = m_new == -INFINITY ? 1.f : exp2f(m - m_new), e = m_new == -INFINITY ? 0.f : exp2f(x - m_new);
    m = m_new;
    l = l * c + e;
#pragma unroll
    for (int d = 0; d < PER; ++d) o[d] = o[d] * c + (held ? e * qmk::bf16_bits_to_f32(p.v_pages[at + 32 * d]) : 0.f);
  }
  const float inv = l > 0.f ? 1.f / l : 0.f;
#pragma unroll
  for (int d = 0; d < PER; ++d)
    p.out[(size_t)token * p.out_stride + (size_t)head * HD + lane + 32 * d] = qmk::f32_to_bf16_bits(o[d] * inv);
  if (p.lse && lane == 0) p.lse[(size_t)token * p.NH + head] = l > 0.f ? (m + log2f(l)) * 0.6931471805599453f : -INFINITY;
}

}  // namespace qmkp
