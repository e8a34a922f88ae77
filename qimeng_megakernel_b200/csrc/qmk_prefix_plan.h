// Division of the work of one attention call (qmk_prefix_attention.cuh): pure integer arithmetic shared by the device code
// and by a host test that replays it.
//
// Rows of a KV head are the step's (token, query head of the group) pairs.  Requests come in two kinds:
//   long   (is_long: pieces of prompts)  cut into units of up to 256 rows of ONE request; a unit walks all its keys, prefix
//          included, causal limits applied
//   short  (few rows: decoding, verification, short pieces behind a long prefix)  their tokens are strung together and cut into units of 256 rows, which
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
constexpr int kMostShort = 512;     // one with as many or more does not
constexpr int kStripRows = 8;       // rows of a strip (the short side of an mma.sync tile)
constexpr int kMaxGroup = 16;       // query heads of a KV head
constexpr int kPieceKeys = 32;      // keys of a piece
constexpr int kStripCost = 3;       // pieces without keys at the head of a strip: what it costs to take one up (2 is 1 %
                                    // slower over 14 calls, 1 and 4 are 6 and 2 % over six)
constexpr int kStripWarps = 8;      // warps of a CTA that walk strips
constexpr int kMaxSeqs = 1536;      // requests of a call (their prefix sums are kept in shared memory)

// Division by a number known on the host, for 0 <= x < 2^31: with p = 31 + ceil(log2 d) and mul = ceil(2^p / d) < 2^32 the
// quotient is floor(x * mul / 2^p) (the rounding of mul adds less than x / 2^31 < 1 part of 1 / d).
struct Divider {
  unsigned mul;
  int d, shift;
  QMKP_HD int div(int x) const {
    if (d == 1) return x;
#if defined(__CUDA_ARCH__)
    return (int)(__umulhi((unsigned)x, mul) >> shift);
#else
    return (int)(((unsigned long long)(unsigned)x * mul >> 32) >> shift);
#endif
  }
  QMKP_HD int mod(int x) const { return x - div(x) * d; }
};
inline Divider make_divider(int d) {
  Divider v;
  v.d = d;
  int log = 0;
  while ((1ll << log) < d) ++log;
  v.shift = 31 + log - 32;
  v.mul = d == 1 ? 0u : (unsigned)(((1ull << (31 + log)) + (unsigned)d - 1) / (unsigned)d);
  return v;
}

struct PlanDims {
  int tokens, seqs, G, NKV, prefix_len, ctas, head_dim;
  int room;                         // positions a request can have: max(prefix_len, max_pages * page_size)
  int unit_tokens;                  // tokens of a unit
  Divider by_unit;
  int prefix_blocks;
  Divider by_G, by_NKV;
};
inline PlanDims make_dims(int tokens, int seqs, int G, int NKV, int head_dim, int prefix_len, int room, int ctas) {
  PlanDims d;
  d.tokens = tokens; d.seqs = seqs; d.G = G; d.NKV = NKV; d.prefix_len = prefix_len; d.ctas = ctas; d.head_dim = head_dim;
  d.room = room > prefix_len ? room : prefix_len;
  d.unit_tokens = kUnitRows / G;
  d.prefix_blocks = (prefix_len + kBlockKeys - 1) / kBlockKeys;
  d.by_unit = make_divider(d.unit_tokens);
  d.by_G = make_divider(G);
  d.by_NKV = make_divider(NKV);
  return d;
}

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
// long requests
QMKP_HD int units_of(const PlanDims& d, const Req& r) { return d.by_unit.div(r.n + d.unit_tokens - 1); }
QMKP_HD int unit_limit(const PlanDims& d, const Req& r, int u) {
  return limit_of(d, r, imin((u + 1) * d.unit_tokens, r.n) - 1);
}
QMKP_HD int unit_blocks(const PlanDims& d, const Req& r, int u) {
  return imax(1, (unit_limit(d, r, u) + kBlockKeys - 1) / kBlockKeys);
}
// short requests
QMKP_HD int own_keys(const PlanDims& d, const Req& r) { return r.n > 0 ? imax(0, limit_of(d, r, r.n - 1) - d.prefix_len) : 0; }
// Between kLongRows and kMostShort rows the cheaper way: units of its own are padded to whole ones and walk all keys so, shared ones
// are not, but a row and key of a strip cost 8 (head size 64; 13 at 128) of a block's.  Weighed with about twice that, as the blocks
// lack the strips' CTAs: 10 pieces of 64..90 tokens behind 28160 keys at 16/8 x 128 take 189 us against 243 us in units of their
// own, 5 of 70..120 behind 16384 at 32/8 x 64 115 against 127; 16 of 33..100 behind 2048 61 either way (64 weighed with once that).
QMKP_HD bool is_long(const PlanDims& d, const Req& r) {
  const long long rows = (long long)r.n * d.G;
  if (rows < kLongRows || rows >= kMostShort) return rows >= kLongRows;
  const int pad = rows == kLongRows ? 0 : units_of(d, r) * kUnitRows - (int)rows;
  return (long long)pad * limit_of(d, r, r.n - 1) <= (d.head_dim == 128 ? 26 : 14) * rows * (own_keys(d, r) + kStripCost * kPieceKeys);
}
QMKP_HD int strips_of(const PlanDims& d, const Req& r) { return (r.n * d.G + kStripRows - 1) / kStripRows; }   // of a KV head
QMKP_HD int pieces_of(const PlanDims& d, const Req& r) { return kStripCost + (own_keys(d, r) + kPieceKeys - 1) / kPieceKeys; }

// Quotients where the exact one takes too long: of small whole numbers (a < 2^21, exact: half a unit is far above the error of the
// reciprocal), and for estimates.
QMKP_HD float about(float a, float b) {
#if defined(__CUDA_ARCH__)
  return __fdividef(a, b);
#else
  return a / b;
#endif
}
QMKP_HD int small_div(int a, int b) { return (int)about((float)a + 0.5f, (float)b); }

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
  int span;                         // the blocks are dealt span by span: one unit of a KV head, or all there are
  Deal dense, strips;               // a span's blocks to CTAs, all pieces to warps
  QMKP_HD int dense_first(int c) const {
    const int s = small_div(c, dense.n);
    return s * span + dense.first(c - s * dense.n);
  }
  QMKP_HD int dense_owner(int b) const {
    const int s = b / span;
    return s * dense.n + dense.owner(b - s * span);
  }
};

// A way to divide the CTAs: `ctas` of them have the blocks, with `each` > 0 as many to every unit and each of them blocks of one
// unit only.
struct Choice {
  int ctas, each;
  float time;
};
// Estimated microseconds of a call, the longer of blocks and strips.  Measured on B200, per CTA: a block of one tile 0.95 us at head
// size 64 and 2.2 us at 128, of two tiles 1.65 and 2.2 us; a piece 0.105 and 0.22 us, or its share of 5.5 TB/s; 6 us to the first
// block's result and out again, 5 us for every unit more; 4 us for a strip.
QMKP_HD int short_units_of(const PlanDims& d, const Totals& t) {
  return d.prefix_len > 0 ? d.by_unit.div(t.short_tokens + d.unit_tokens - 1) : 0;
}
QMKP_HD float choice_time(const PlanDims& d, const Totals& t, int short_units, int ctas, int each) {
  const bool small = t.short_tokens * d.G <= kLongRows, wide = d.head_dim == 128;
  const float one = wide ? 2.2f : 0.95f, two = wide ? 2.2f : 1.65f, block = small ? one : two;
  const int units = (t.long_units + short_units) * d.NKV, rest = d.ctas - ctas;
  float dense = 0.f;
  if (units > 0 && ctas == 0) dense = 1e30f;
  else if (units > 0 && each > 0) dense = 6.f + (about((float)d.prefix_blocks, (float)each) + 0.5f) * block;
  else if (units > 0) {
    const float more = about((float)units, (float)ctas) + 1.f, most = (float)(units - 1);
    dense = 6.f + 5.f * (more < most ? more : most) +
            about(((float)t.long_blocks * two + (float)(short_units * d.prefix_blocks) * block) * (float)d.NKV, (float)ctas);
  }
  const float pieces = (float)t.pieces * (float)d.NKV, stream = pieces * (wide ? 0.003f : 0.0015f);
  const float work = rest > 0 ? about(pieces * (wide ? 0.22f : 0.105f), (float)rest) : 1e30f;
  const float few = t.pieces > 0 ? 4.f + (work > stream ? work : stream) : 0.f;
  return dense > few ? dense : few;
}
// The divisions that are weighed: i of kPlanChoices.
constexpr int kPlanChoices = 32;
QMKP_HD Choice plan_choice(const PlanDims& d, const Totals& t, int i) {
  const int short_units = short_units_of(d, t), units = short_units * d.NKV;
  const int blocks = (t.long_blocks + short_units * d.prefix_blocks) * d.NKV;
  Choice c;
  c.ctas = t.pieces == 0 ? d.ctas : (i + 1) * (d.ctas - 1) / kPlanChoices;
  c.ctas = imin(imax(c.ctas, 1), blocks);   // (no blocks: none)
  c.each = 0;
  c.time = choice_time(d, t, short_units, c.ctas, 0);
  if (t.long_units == 0 && units > 0 && c.ctas >= units) {
    const int each = imin(small_div(c.ctas, units), d.prefix_blocks);
    const float time = choice_time(d, t, short_units, units * each, each);
    if (time <= c.time) { c.ctas = units * each; c.each = each; c.time = time; }
  }
  return c;
}
QMKP_HD Plan make_plan(const PlanDims& d, const Totals& t, const Choice& c) {
  Plan p;
  const int short_units = short_units_of(d, t);
  p.unit_total = t.long_units + short_units;
  p.blocks = t.long_blocks + short_units * d.prefix_blocks;
  p.dense_ctas = c.ctas;
  p.span = c.each ? d.prefix_blocks : p.blocks * d.NKV;
  p.dense = deal(p.span, c.each ? c.each : c.ctas);
  p.strips = deal(t.pieces * d.NKV, (d.ctas - c.ctas) * kStripWarps);
  return p;
}
// Blocks [lo, hi) of CTA c.
QMKP_HD void dense_range(const Plan& p, int c, int& lo, int& hi) {
  lo = hi = 0;
  if (c >= p.dense_ctas) return;
  lo = p.dense_first(c);
  hi = p.dense_first(c + 1);
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

// First key behind the prefix of piece c of a strip.
QMKP_HD int piece_lo(int c) { return imax(0, c - kStripCost) * kPieceKeys; }
// Pieces are numbered request by request, inside it (strip of a KV head, KV head, piece), the piece fastest.  Strips are
// numbered in the same order, with gaps: `before` short tokens in front of request s leave room for their strips.
QMKP_HD int strip_number(const PlanDims& d, int s, int before, int strip, int kvh) {
  return ((int)((long long)before * d.G / kStripRows) + s + strip) * d.NKV + kvh;
}

// Upper bounds for the workspace.
QMKP_HD long long max_units(const PlanDims& d) {
  const long long per = d.unit_tokens, a = 2ll * d.tokens / per + 2, b = d.tokens / per + (long long)d.seqs + 2;
  return a < b ? a : b;
}
QMKP_HD long long max_dense_records(const PlanDims& d) { return d.ctas + max_units(d) * d.NKV; }
// (A short request has fewer than kMostShort rows.  With T short tokens in all, floor(before * G / 8) + strip <= floor(T * G / 8).)
QMKP_HD long long max_strips(const PlanDims& d) {
  const long long by_request = (long long)d.seqs * ((kMostShort - 1) / d.G);
  return ((by_request < d.tokens ? by_request : d.tokens) * d.G / kStripRows + d.seqs) * d.NKV;
}
QMKP_HD long long max_strip_records(const PlanDims& d) { return (long long)d.ctas * kStripWarps + max_strips(d); }

}  // namespace qmkp
