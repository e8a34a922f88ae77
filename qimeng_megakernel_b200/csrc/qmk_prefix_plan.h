// Division of the work of one attention call (qmk_prefix_attention.cuh): pure integer arithmetic shared by the device code
// and by a host test that replays it.
//
// Rows of a KV head are the step's (token, query head of the group) pairs.  Requests come in two kinds:
//   long   (n * G >= kLongRows rows)  cut into units of up to 256 rows of ONE request; a unit walks all its keys, prefix
//          included, causal limits applied
//   short  (fewer rows: decoding, verification)  their tokens are strung together and cut into units of 256 rows, which
//          walk the shared prefix; what each request holds behind the prefix is walked by single warps, 8 rows at a time: a
//          STRIP is (request, 8 of its rows, KV head), cut into pieces of 32 keys
// The 128-key blocks of all (KV head, unit) pairs, in that order, are dealt to `dense_ctas` CTAs as equal contiguous ranges;
// the pieces of all strips to warps, so that a CTA's blocks and pieces together come out even.  Every (CTA, unit) and every
// (warp, strip) that meet leave a partial result: record number (CTA + unit) or (warp + strip), which no other pair has.
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
constexpr int kStripRows = 8;       // rows of a strip (the short side of an mma.sync tile)
constexpr int kMaxGroup = 16;       // query heads of a KV head
constexpr int kPieceKeys = 32;      // keys of a piece
constexpr int kStripWarps = 8;      // warps of a CTA that walk strips
constexpr int kMaxSeqs = 2048;      // requests of a call (their prefix sums are kept in shared memory)

struct PlanDims {
  int tokens, seqs, G, NKV, prefix_len, ctas;
  int room;                         // positions a request can have: max(prefix_len, max_pages * page_size)
  QMKP_HD int unit_tokens() const { return kUnitRows / G; }
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
QMKP_HD int strips_of(const PlanDims& d, const Req& r) { return (r.n * d.G + kStripRows - 1) / kStripRows; }   // of a KV head
QMKP_HD int pieces_of(const PlanDims& d, const Req& r) { return imax(1, (own_keys(d, r) + kPieceKeys - 1) / kPieceKeys); }

struct Totals {
  long long long_blocks;            // blocks of all long units (per KV head)
  int long_units;
  int short_tokens;
  long long pieces;                 // pieces of all short requests (per KV head)
};

struct Plan {
  int short_units, unit_total;      // units per KV head
  long long blocks;                 // per KV head
  long long dense_blocks;           // all KV heads
  int dense_ctas;
  // pieces: warps of the CTAs with blocks (class 0) and of those without (class 1); warps and pieces of a class
  int warps[2];
  long long share[2];
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
  // a block counts as four pieces (its keys)
  const long long all = t.pieces * d.NKV, load = p.dense_blocks * (kBlockKeys / kPieceKeys);
  const long long even = (load + all) / d.ctas, mine = p.dense_ctas > 0 ? load / p.dense_ctas : 0;
  const long long left = even > mine ? (even - mine) * p.dense_ctas : 0;       // room beside the blocks
  p.share[0] = p.dense_ctas == d.ctas ? all : (left < all ? left : all);
  p.share[1] = all - p.share[0];
  for (int c = 0; c < 2; ++c) {
    const long long w = (long long)kStripWarps * (c == 0 ? p.dense_ctas : d.ctas - p.dense_ctas);
    p.warps[c] = (int)(w < p.share[c] ? w : p.share[c]);
  }
  return p;
}
// Blocks [lo, hi) of CTA c.
QMKP_HD void dense_range(const Plan& p, int c, long long& lo, long long& hi) {
  if (c >= p.dense_ctas) { lo = hi = 0; return; }
  lo = p.dense_blocks * c / p.dense_ctas;
  hi = p.dense_blocks * (c + 1) / p.dense_ctas;
}
QMKP_HD int dense_owner(const Plan& p, long long b) { return (int)(((b + 1) * p.dense_ctas - 1) / p.dense_blocks); }

// Pieces [lo, hi) of a warp of CTA c, and the warp's number among all that have any (-1: none).  Neighbouring numbers are
// neighbouring CTAs.
QMKP_HD int piece_range(const PlanDims& d, const Plan& p, int c, int warp, long long& lo, long long& hi) {
  const int k = c < p.dense_ctas ? 0 : 1;
  const int i = k == 0 ? warp * p.dense_ctas + c : warp * (d.ctas - p.dense_ctas) + c - p.dense_ctas;
  lo = hi = 0;
  if (i >= p.warps[k]) return -1;
  const long long from = k == 0 ? 0 : p.share[0];
  lo = from + p.share[k] * i / p.warps[k];
  hi = from + p.share[k] * (i + 1) / p.warps[k];
  return (k == 0 ? 0 : p.warps[0]) + i;
}
QMKP_HD int piece_owner(const Plan& p, long long f) {
  if (f < p.share[0]) return (int)(((f + 1) * p.warps[0] - 1) / p.share[0]);
  f -= p.share[0];
  return p.warps[0] + (int)(((f + 1) * p.warps[1] - 1) / p.share[1]);
}
// Pieces are numbered request by request, inside it (strip of a KV head, KV head, piece), the piece fastest.  Strips are
// numbered in the same order, with gaps: `before` short tokens in front of request s leave room for their strips.
QMKP_HD int strip_number(const PlanDims& d, int s, int before, int strip, int kvh) {
  return ((int)((long long)before * d.G / kStripRows) + s + strip) * d.NKV + kvh;
}

// Upper bounds for the workspace.
QMKP_HD long long max_units(const PlanDims& d) {
  const long long per = d.unit_tokens(), a = 2ll * d.tokens / per + 2, b = d.tokens / per + (long long)d.seqs + 2;
  return a < b ? a : b;
}
QMKP_HD long long max_dense_records(const PlanDims& d) { return d.ctas + max_units(d) * d.NKV; }
QMKP_HD long long max_strips(const PlanDims& d) {
  return ((long long)d.tokens * d.G / kStripRows + d.seqs) * d.NKV;
}
QMKP_HD long long max_strip_records(const PlanDims& d) { return (long long)d.ctas * kStripWarps + max_strips(d); }

}  // namespace qmkp
