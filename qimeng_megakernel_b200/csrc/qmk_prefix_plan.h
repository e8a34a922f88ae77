// Division of the work of one attention call (qmk_prefix_attention.cuh): pure integer arithmetic shared by the device code
// and by a host test that replays it.
//
// Rows of a KV head are the step's (token, query head of the group) pairs.  Requests come in two kinds:
//   long   (n * G >= kLongRows rows)  cut into units of up to 256 rows of ONE request; a unit walks all its keys, prefix
//          included, causal limits applied
//   short  (fewer rows: decoding, verification)  their tokens are strung together and cut into units of 256 rows, which
//          walk the shared prefix; what each request holds behind the prefix is walked by single warps in ITEMS of up to 16
//          rows x `ck` keys
// The 128-key blocks of all (KV head, unit) pairs, in that order, are dealt to `dense_ctas` CTAs as equal contiguous ranges;
// the items to all CTAs so that the sum comes out even.  A (CTA, unit) pair and an item each leave a partial result.
#pragma once
#include <stdint.h>

#if defined(__CUDACC__)
#define QMKP_HD __host__ __device__ __forceinline__
#else
#define QMKP_HD inline
#endif

namespace qmkp {

constexpr int kUnitRows = 256;      // two tensor-core tiles of 128 rows
constexpr int kBlockKeys = 128;     // keys of a block
constexpr int kLongRows = 128;      // a request with fewer rows shares its units
constexpr int kItemRows = 16;       // rows of an item (one mma.sync tile)
constexpr int kItemWarps = 8;       // warps of a CTA that walk items
constexpr int kMinItemKeys = 64;
constexpr int kMaxSeqs = 2048;      // requests of a call (their prefix sums are kept in shared memory)

struct PlanDims {
  int tokens, seqs, G, NKV, prefix_len, ctas;
  int room;                         // positions a request can have: max(prefix_len, max_pages * page_size)
  QMKP_HD int unit_tokens() const { return kUnitRows / G; }
  QMKP_HD int item_tokens() const { return kItemRows / G; }
  QMKP_HD int prefix_blocks() const { return (prefix_len + kBlockKeys - 1) / kBlockKeys; }
};

struct Req {
  int first, n;                     // first row (token) of the request in the step, tokens
  int base;                         // its token i sees positions below base + i + 1
};
QMKP_HD int imin(int a, int b) { return a < b ? a : b; }
QMKP_HD int imax(int a, int b) { return a > b ? a : b; }
QMKP_HD Req request(const PlanDims& d, int c0, int c1, int kv) {
  Req r;
  r.first = imin(imax(c0, 0), d.tokens);
  r.n = imax(imin(c1, d.tokens) - r.first, 0);
  // (a length below zero holds nothing; the difference cannot leave 32 bits)
  r.base = imax(kv, 0) - r.n;
  return r;
}
QMKP_HD int limit_of(const PlanDims& d, const Req& r, int i) {
  const long long l = (long long)r.base + i + 1;
  return l < 0 ? 0 : (l > d.room ? d.room : (int)l);
}
QMKP_HD bool is_long(const PlanDims& d, const Req& r) { return (long long)r.n * d.G >= kLongRows; }

// long requests
QMKP_HD int units_of(const PlanDims& d, const Req& r) { return (r.n + d.unit_tokens() - 1) / d.unit_tokens(); }
QMKP_HD int unit_limit(const PlanDims& d, const Req& r, int u) {
  return limit_of(d, r, imin((u + 1) * d.unit_tokens(), r.n) - 1);
}
QMKP_HD int unit_blocks(const PlanDims& d, const Req& r, int u) {
  return imax(1, (unit_limit(d, r, u) + kBlockKeys - 1) / kBlockKeys);
}
// short requests
QMKP_HD int own_keys(const PlanDims& d, const Req& r) { return r.n > 0 ? imax(0, limit_of(d, r, r.n - 1) - d.prefix_len) : 0; }
QMKP_HD int item_rows_blocks(const PlanDims& d, const Req& r) { return (r.n + d.item_tokens() - 1) / d.item_tokens(); }
QMKP_HD int item_chunks(int own, int ck) { return imax(1, (own + ck - 1) / ck); }

struct Totals {
  long long long_blocks;            // blocks of all long units (per KV head)
  int long_units;
  int short_tokens;
  long long item_keys;              // keys of all row blocks of all short requests (per KV head)
};

struct Plan {
  int short_units, unit_total;      // units per KV head
  long long blocks;                 // per KV head
  long long dense_blocks;           // all KV heads
  int dense_ctas;
  int ck;
};
constexpr int kMinSegment = 2;      // blocks a CTA takes at least

QMKP_HD Plan make_plan(const PlanDims& d, const Totals& t) {
  Plan p;
  p.short_units = d.prefix_len > 0 ? (t.short_tokens + d.unit_tokens() - 1) / d.unit_tokens() : 0;
  p.unit_total = t.long_units + p.short_units;
  p.blocks = t.long_blocks + (long long)p.short_units * d.prefix_blocks();
  p.dense_blocks = p.blocks * d.NKV;
  const long long want = (p.dense_blocks + kMinSegment - 1) / kMinSegment;
  p.dense_ctas = want < d.ctas ? (int)want : d.ctas;
  const long long warps = (long long)d.ctas * kItemWarps;
  long long ck = (t.item_keys * d.NKV + warps - 1) / warps;
  ck = (ck + 15) / 16 * 16;
  p.ck = (int)(ck < kMinItemKeys ? kMinItemKeys : (ck > (1 << 30) ? (1 << 30) : ck));
  return p;
}
// Blocks [lo, hi) of CTA c.
QMKP_HD void dense_range(const Plan& p, int c, long long& lo, long long& hi) {
  if (c >= p.dense_ctas) { lo = hi = 0; return; }
  lo = p.dense_blocks * c / p.dense_ctas;
  hi = p.dense_blocks * (c + 1) / p.dense_ctas;
}
QMKP_HD int dense_owner(const Plan& p, long long b) { return (int)(((b + 1) * p.dense_ctas - 1) / p.dense_blocks); }

// Items [lo, hi) of CTA c out of `items`: a CTA with a dense share takes fewer (a block counts as its 128 keys).
QMKP_HD void item_range(const PlanDims& d, const Plan& p, const Totals& t, long long items, int c, long long& lo, long long& hi) {
  const long long dense = p.dense_blocks * kBlockKeys, few = t.item_keys * d.NKV;
  const long long even = (dense + few) / d.ctas;                    // keys per CTA
  const long long mine = p.dense_ctas > 0 ? dense / p.dense_ctas : 0;
  long long with = even > mine ? even - mine : 0, without = even;
  if (with * p.dense_ctas + without * (d.ctas - p.dense_ctas) <= 0) with = without = 1;
  const long long total = with * p.dense_ctas + without * (d.ctas - p.dense_ctas);
  const int dc = p.dense_ctas;
  const long long a = c < dc ? c * with : dc * with + (c - dc) * without;
  const long long b = c + 1 < dc ? (c + 1) * with : dc * with + (c + 1 - dc) * without;
  // (shares scaled to 2^20 so that the products stay inside 64 bits)
  const long long sa = (long long)((double)a / (double)total * 1048576.0), sb = c + 1 == d.ctas ? 1048576 : (long long)((double)b / (double)total * 1048576.0);
  lo = items * sa >> 20;
  hi = items * sb >> 20;
}

// Upper bounds for the workspace.
QMKP_HD long long max_units(const PlanDims& d) {
  const long long per = d.unit_tokens(), a = 2ll * d.tokens / per + 2, b = d.tokens / per + (long long)d.seqs + 2;
  return a < b ? a : b;
}
QMKP_HD long long max_dense_records(const PlanDims& d) { return d.ctas + max_units(d) * d.NKV; }
QMKP_HD long long max_items(const PlanDims& d) {
  const long long a = d.tokens, b = (long long)d.tokens / d.item_tokens() + d.seqs;
  return (long long)d.ctas * kItemWarps + (a < b ? a : b) * d.NKV + 1;
}

}  // namespace qmkp
