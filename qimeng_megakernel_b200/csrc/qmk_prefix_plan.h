// Division of the work of one attention call (qmk_prefix_attention.cuh): pure integer arithmetic shared by the device code
// and by a host test that replays it.
//
// Rows of a KV head are the step's (token, query head of the group) pairs.  Requests come in two kinds:
//   long   (n * G >= kLongRows rows)  cut into units of up to 256 rows of ONE request; a unit walks all its keys, prefix
//          included, causal limits applied
//   short  (fewer rows: decoding, verification)  their tokens are strung together and cut into units of 256 rows, which
//          walk the shared prefix; what each request holds behind the prefix is walked by single warps, 8 rows at a time: a
//          STRIP is (request, 8 of its rows, KV head), cut into pieces of 32 keys
// The 128-key blocks of all (KV head, unit) pairs, in that order, are dealt to the first CTAs as equal contiguous ranges, the
// pieces of all strips to the warps of the other CTAs, as many CTAs to either as its share of the work.  Every (CTA, unit) and every
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
constexpr int kBlockCost = 8;       // time of a block of 256 rows in pieces (a CTA's eight warps at one each)
constexpr int kMaxSeqs = 1536;      // requests of a call (their prefix sums are kept in shared memory)

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

// `total` things dealt to n takers as contiguous ranges that differ by one at most (with fewer things than takers the first
// ones get one each, so owners of neighbouring things are always neighbours).
struct Deal {
  int n, each, more;                // the first `more` takers get each + 1
  QMKP_HD int first(int i) const { return each * i + imin(i, more); }
  QMKP_HD int owner(int b) const {
    const int head = more * (each + 1);
    return b < head ? b / (each + 1) : more + (b - head) / each;
  }
};
QMKP_HD Deal deal(int total, int n) {
  Deal d;
  d.n = n;
  d.each = n > 0 ? total / n : 0;
  d.more = n > 0 ? total - d.each * n : 0;
  return d;
}

// (The entry point refuses sizes whose totals do not fit 32 bits.)
struct Totals {
  int long_blocks;                  // blocks of all long units (per KV head)
  int long_units;
  int short_tokens;
  int pieces;                       // pieces of all short requests (per KV head)
};

struct Plan {
  int unit_total;                   // units per KV head
  int blocks;                       // per KV head
  int dense_ctas;                   // CTAs with blocks; the others have pieces
  Deal dense, strips;               // all blocks to CTAs, all pieces to warps
};
constexpr int kMinSegment = 2;      // blocks a CTA takes at least

QMKP_HD Plan make_plan(const PlanDims& d, const Totals& t) {
  Plan p;
  const int short_units = d.prefix_len > 0 ? (t.short_tokens + d.unit_tokens() - 1) / d.unit_tokens() : 0;
  p.unit_total = t.long_units + short_units;
  const int short_blocks = short_units * d.prefix_blocks();
  p.blocks = t.long_blocks + short_blocks;
  const int all = p.blocks * d.NKV, pieces = t.pieces * d.NKV;
  // a block of two tiles counts as kBlockCost pieces, one of a single tile as four (its keys)
  const bool small = t.short_tokens * d.G <= kLongRows;
  const float dense = ((float)t.long_blocks * kBlockCost + (float)short_blocks * (small ? 4 : kBlockCost)) * (float)d.NKV;
  int ctas = pieces == 0 ? d.ctas : (int)((float)d.ctas * (dense / (dense + (float)pieces)) + 0.5f);
  ctas = imin(imax(ctas, 1), pieces == 0 ? d.ctas : d.ctas - 1);
  ctas = imin(ctas, (all + kMinSegment - 1) / kMinSegment);
  p.dense_ctas = ctas;
  p.dense = deal(all, ctas);
  p.strips = deal(pieces, (d.ctas - ctas) * kStripWarps);
  return p;
}
// Blocks [lo, hi) of CTA c.
QMKP_HD void dense_range(const Plan& p, int c, int& lo, int& hi) {
  lo = hi = 0;
  if (c >= p.dense_ctas) return;
  lo = p.dense.first(c);
  hi = p.dense.first(c + 1);
}
// Pieces [lo, hi) of a warp of CTA c and the warp's number among those that have any (neighbours sit in neighbouring CTAs).
QMKP_HD int piece_range(const PlanDims& d, const Plan& p, int c, int warp, int& lo, int& hi) {
  lo = hi = 0;
  if (c < p.dense_ctas) return -1;
  const int i = warp * (d.ctas - p.dense_ctas) + c - p.dense_ctas;
  lo = p.strips.first(i);
  hi = p.strips.first(i + 1);
  return i;
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
