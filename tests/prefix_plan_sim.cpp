// Replays the plan of the prefix attention (qmk_prefix_plan.h) on the CPU: every (KV head, row, visible key) has to be
// walked exactly once, by a block of a unit or by a piece of a strip; every partial result has to have a record of its own inside the
// workspace's bounds; and the records that a row's description names have to be the ones that were written for it.
#include <cstdio>
#include <cstdlib>
#include <random>
#include <vector>

#include "../qimeng_megakernel_b200/csrc/qmk_prefix_plan.h"

using namespace qmkp;

#define CHECK(c)                                                      \
  do {                                                                \
    if (!(c)) {                                                       \
      std::printf("line %d: %s (case %d)\n", __LINE__, #c, g_case);  \
      std::exit(1);                                                   \
    }                                                                 \
  } while (0)
static int g_case;
static int aligned, middle;                            // middle: requests of some hundred rows that share their units

struct Walk { std::vector<std::vector<int>> seen; };   // [row of the step * NKV + kvh][key] -> times

int main() {
  std::mt19937 rng(7);
  auto pick = [&](int lo, int hi) { return lo + (int)(rng() % (unsigned)(hi - lo + 1)); };
  for (int d : {1, 2, 3, 5, 7, 8, 16, 48, 127, 1000, 1024}) {
    const Divider v = make_divider(d);
    for (int i = 0; i < 20000; ++i) {
      const int x = i < 5000 ? i : (i < 10000 ? 0x7fffffff - i : (int)(rng() >> 1));
      CHECK(v.div(x) == x / d && v.mod(x) == x % d);
    }
  }
  for (g_case = 0; g_case < 1500; ++g_case) {
    const int G = pick(1, 16), ctas = pick(0, 1) ? 148 : pick(2, 30), page = 16;
    const bool far = g_case % 25 == 24;                      // short pieces behind a long prefix
    const int prefix_len = far ? 16 * pick(200, 400) : (pick(0, 3) ? 16 * pick(0, 60) : 0);
    const int max_pages = prefix_len / page + pick(1, 40);
    PlanDims d = make_dims(1, far ? pick(1, 3) : pick(1, pick(0, 3) ? 6 : 40), G, far ? 1 : pick(1, 4), pick(0, 1) ? 64 : 128, prefix_len,
                           max_pages * page, ctas);
    std::vector<int> cu(1, 0), kv;
    const int kind = pick(0, 3);
    for (int s = 0; s < d.seqs; ++s) {
      const int n = far ? pick(128, 511) / d.G : kind == 0 ? 1 : (kind == 1 ? pick(0, 5) : (kind == 2 ? pick(0, 400 / d.G) : pick(0, 2) * pick(0, 600)));
      cu.push_back(cu.back() + n);
      if (far) kv.push_back(d.prefix_len + n + pick(0, 30));
      else kv.push_back(pick(0, 9) ? d.prefix_len + pick(0, max_pages * page - d.prefix_len + 5) : pick(-3, d.prefix_len + n));
    }
    d.tokens = cu.back() + pick(-3, 5);
    if (d.tokens < 1) d.tokens = 1;

    std::vector<Req> req;
    std::vector<int> lb(1, 0), lu(1, 0), stk(1, 0), pc(1, 0);
    Totals t{0, 0, 0, 0};
    for (int s = 0; s < d.seqs; ++s) {
      const Req r = request(d, cu[s], cu[s + 1], kv[s]);
      req.push_back(r);
      int blocks = 0;
      if (is_long(d, r)) {
        for (int u = 0; u < units_of(d, r); ++u) blocks += unit_blocks(d, r, u);
        t.long_blocks += blocks;
        t.long_units += units_of(d, r);
      } else {
        middle += r.n * d.G >= kLongRows;
        t.short_tokens += r.n;
        t.pieces += (long long)strips_of(d, r) * pieces_of(d, r);
      }
      lb.push_back((int)t.long_blocks);
      lu.push_back(t.long_units);
      stk.push_back(t.short_tokens);
      pc.push_back((int)t.pieces);
    }
    Choice choice = plan_choice(d, t, 0);
    for (int i = 1; i < kPlanChoices; ++i) {
      const Choice other = plan_choice(d, t, i);
      if (other.time < choice.time) choice = other;
    }
    if (g_case % 3 == 0) choice = plan_choice(d, t, pick(0, kPlanChoices - 1));   // (any of them has to do)
    aligned += choice.each > 0;
    const Plan p = make_plan(d, t, choice);
    const int pieces = t.pieces * d.NKV, all_blocks = p.blocks * d.NKV;
    CHECK(p.unit_total <= max_units(d));
    CHECK(p.dense_ctas <= d.ctas && (all_blocks == 0) == (p.dense_ctas == 0) && (pieces == 0 || p.dense_ctas < d.ctas));

    Walk w;
    w.seen.resize((size_t)d.tokens * d.NKV);
    std::vector<int> limit(d.tokens, -1), owner(d.tokens, -1);
    for (int s = 0; s < d.seqs; ++s)
      for (int i = 0; i < req[s].n; ++i) {
        CHECK(owner[req[s].first + i] < 0);
        owner[req[s].first + i] = s;
        limit[req[s].first + i] = limit_of(d, req[s], i);
      }
    for (int tok = 0; tok < d.tokens; ++tok)
      if (limit[tok] >= 0)
        for (int h = 0; h < d.NKV; ++h) w.seen[(size_t)tok * d.NKV + h].assign((size_t)limit[tok], 0);
    std::vector<char> record((size_t)max_dense_records(d), 0);
    struct Named { int rec, n; };
    std::vector<Named> named((size_t)d.tokens * d.NKV, Named{-1, 0});
    std::vector<std::vector<int>> written((size_t)d.tokens * d.NKV);
    int walked = 0;
    std::vector<char> strip_record((size_t)max_strip_records(d), 0), piece_done((size_t)pieces, 0);
    std::vector<Named> strip_named((size_t)d.tokens * d.G * d.NKV, Named{-1, 0});
    std::vector<std::vector<int>> strip_written((size_t)d.tokens * d.G * d.NKV);
    for (int c = 0; c < d.ctas; ++c) {
      int lo, hi;
      dense_range(p, c, lo, hi);
      if (c < p.dense_ctas) {
        CHECK(lo == walked && hi > lo);
        walked = hi;
      }
      for (int b = lo; b < hi;) {
        // the unit of block b, found by walking all of them
        const int kvh = (int)(b / p.blocks);
        int rest = b % p.blocks;
        int index = 0, blocks = 0, s = -1, u = 0;
        bool found = false;
        for (int q = 0; q < d.seqs && !found; ++q) {
          if (!is_long(d, req[q])) continue;
          for (u = 0; u < units_of(d, req[q]); ++u, ++index) {
            blocks = unit_blocks(d, req[q], u);
            if (rest < blocks) { s = q; found = true; break; }
            rest -= blocks;
          }
        }
        if (found) {
          CHECK(lb[s] <= b % p.blocks && b % p.blocks < lb[s + 1]);
          CHECK(index == lu[s] + u);
        } else {
          blocks = d.prefix_blocks;
          u = (int)(rest / blocks);
          rest -= (long long)u * blocks;
          index = t.long_units + u;
        }
        const int b0 = (int)rest, b1 = (int)(blocks - b0 < hi - b ? blocks : b0 + (hi - b));
        const int rec = c + kvh * p.unit_total + index;
        CHECK(rec < max_dense_records(d) && !record[rec]);
        record[rec] = 1;
        const int parts = p.dense_owner(b - b0 + blocks - 1) - p.dense_owner(b - b0) + 1;
        CHECK(p.dense_owner(b) == c && p.dense_owner(b + (b1 - b0) - 1) == c);
        for (int i = 0; i < d.unit_tokens; ++i) {
          int tok, lim;
          if (s >= 0) {
            const int k = u * d.unit_tokens + i;
            if (k >= req[s].n) break;
            tok = req[s].first + k;
            lim = limit_of(d, req[s], k);
            CHECK(lim <= unit_limit(d, req[s], u));
          } else {
            const int k = u * d.unit_tokens + i;
            if (k >= t.short_tokens) break;
            int q = 0;
            while (!(stk[q] <= k && k < stk[q + 1])) ++q;
            tok = req[q].first + k - stk[q];
            lim = limit_of(d, req[q], k - stk[q]);
            lim = lim < d.prefix_len ? lim : d.prefix_len;
          }
          auto& seen = w.seen[(size_t)tok * d.NKV + kvh];
          for (int key = b0 * kBlockKeys; key < b1 * kBlockKeys && key < lim; ++key) ++seen[key];
          if (b0 == 0) named[(size_t)tok * d.NKV + kvh] = Named{rec, parts};
          written[(size_t)tok * d.NKV + kvh].push_back(rec);
        }
        b += b1 - b0;
      }
      for (int warp = 0; warp < kStripWarps; ++warp) {
        int flo, fhi;
        const int number = piece_range(d, p, c, warp, flo, fhi);
        CHECK(number >= 0 || flo == fhi);
        for (int f = flo; f < fhi;) {
          int s = 0;
          while (!((long long)pc[s] * d.NKV <= f && f < (long long)pc[s + 1] * d.NKV)) ++s;
          CHECK(pc[s] <= f / d.NKV && f / d.NKV < pc[s + 1]);
          const Req& r = req[s];
          const int per = pieces_of(d, r);
          int rest = f - pc[s] * d.NKV;
          const int c0 = (int)(rest % per), n = (int)(per - c0 < fhi - f ? per - c0 : fhi - f);
          rest /= per;
          const int kvh = (int)(rest % d.NKV), strip = (int)(rest / d.NKV);
          const int rec = number + strip_number(d, s, stk[s], strip, kvh);
          CHECK(rec < max_strip_records(d) && !strip_record[rec]);
          strip_record[rec] = 1;
          for (int k = f; k < f + n; ++k) { CHECK(!piece_done[k]); piece_done[k] = 1; CHECK(p.strips.owner(k) == number); }
          const int row0 = strip * kStripRows, rows = imin(kStripRows, r.n * d.G - row0);
          CHECK(rows > 0);
          const int last = limit_of(d, r, (row0 + rows - 1) / d.G);
          const int k_lo = d.prefix_len + piece_lo(c0), k_hi = imin(d.prefix_len + piece_lo(c0 + n), last);
          for (int i = 0; i < rows; ++i) {
            const int tok = r.first + (row0 + i) / d.G, gq = (row0 + i) % d.G, lim = limit_of(d, r, (row0 + i) / d.G);
            CHECK(lim <= last);
            const size_t at = ((size_t)tok * d.NKV + kvh) * d.G + gq;
            if (gq == 0) {                                    // (heads of a token see the same keys)
              auto& seen = w.seen[(size_t)tok * d.NKV + kvh];
              for (int key = k_lo; key < k_hi && key < lim; ++key) ++seen[key];
            }
            if (c0 == 0) strip_named[at] = Named{rec, p.strips.owner(f + per - 1) - number + 1};
            strip_written[at].push_back(rec);
          }
          f += n;
        }
      }
    }
    for (char x : piece_done) CHECK(x);
    for (int tok = 0; tok < d.tokens; ++tok) {
      if (owner[tok] < 0 || is_long(d, req[owner[tok]])) continue;
      for (int h = 0; h < d.NKV * d.G; ++h) {
        const size_t at = (size_t)tok * d.NKV * d.G + h;
        std::vector<int>& v = strip_written[at];
        for (size_t a = 0; a < v.size(); ++a)                  // (warps are visited CTA by CTA, not in their order)
          for (size_t b2 = a + 1; b2 < v.size(); ++b2)
            if (v[b2] < v[a]) { const int x = v[a]; v[a] = v[b2]; v[b2] = x; }
        CHECK((int)v.size() == strip_named[at].n);
        for (int k = 0; k < strip_named[at].n; ++k) CHECK(v[k] == strip_named[at].rec + k);
      }
    }
    CHECK(walked == all_blocks);
    for (int tok = 0; tok < d.tokens; ++tok)
      for (int h = 0; h < d.NKV; ++h) {
        const size_t i = (size_t)tok * d.NKV + h;
        for (int n : w.seen[i]) CHECK(n == 1);
        CHECK((int)written[i].size() == named[i].n);
        for (int k = 0; k < named[i].n; ++k) CHECK(written[i][k] == named[i].rec + k);
      }
  }
  CHECK(aligned > 100);
  CHECK(middle > 30);
  std::printf("prefix plan ok\n");
  return 0;
}
