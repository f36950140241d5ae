// The cut of the attention's work (csrc/attention_plan.cuh) on the host, for test_attention_cut.py: every key of
// every row block is some part's, once; every segment gets its entry, and the joining kernel follows no entry that is
// none. Prints what is wrong and ends with 1, or ends with 0.
#include <cstdio>
#include <cstdlib>
#include <random>
#include <vector>

#include "attention_plan.cuh"

using namespace vtq;

#define WANT(x)                                                      \
  do {                                                               \
    if (!(x)) {                                                      \
      std::printf("line %d: %s does not hold\n", __LINE__, #x);      \
      std::exit(1);                                                  \
    }                                                                \
  } while (0)

// The plan that build_plan makes, by a plain loop.
struct Cut {
  AttnParams p = {};
  std::vector<int> ints;
  Plan pl;
  int B, H, total;
  Cut(const std::vector<int>& rows, const std::vector<int>& lens, int H_, int group, int tile, int keys_max, int shared, bool on_tiles)
      : ints(plan_ints((int)rows.size())), pl(plan_of(ints.data(), (int)rows.size())), B((int)rows.size()), H(H_) {
    p.group = group;
    p.tile = tile;
    while (1 << p.tile_shift < tile) p.tile_shift++;
    p.by_group = divisor(group);
    p.keys_max = keys_max;
    p.prefix = shared < keys_max ? shared : keys_max;
    p.on_tiles = on_tiles;
    p.a.kv.seqs = B, p.a.kv.kv_heads = H;
    bool any = false;
    for (int b = 0; b < B; b++) pl.q0[b + 1] = pl.q0[b] + rows[b], pl.len[b] = lens[b];
    for (int b = 0; b < B; b++) any |= sees_prefix(p, pl, b);
    p.a.tokens = pl.q0[B];
    pl.len[B] = any ? p.prefix : 0;
    int segs = 0;
    total = 0;
    for (int b = 0; b <= B; b++) {
      pl.tiles[b] = total, pl.segs[b] = segs;
      const Entry e = entry_of(p, pl, b, B);
      total += blocks_of(e) * H * tiles_of(p, e);
      segs += blocks_of(e) * H;
    }
    pl.tiles[B + 1] = total, pl.segs[B + 1] = segs;
  }
};

void check(const Cut& c, int parts) {
  const int W = c.total < parts ? c.total : parts, B = c.B, H = c.H, segs = c.pl.segs[B + 1];
  const int stale = (int)0xcdcdcdcd;
  std::vector<std::vector<int>> seen(segs);  // how often each key of a segment is taken
  std::vector<int2> entries(segs, make_int2(stale, stale));
  for (int w = 0; w < W; w++) {
    const int tile0 = first_tile(c.total, W, w), tile1 = first_tile(c.total, W, w + 1);
    WANT(tile0 < tile1);
    Cursor at = seek(c.p, c.pl, B, tile0);
    for (int tile = tile0; tile < tile1; tile++) {
      const Cursor again = seek(c.p, c.pl, B, tile);
      WANT(at.b == again.b && at.mb == again.mb && at.g == again.g && at.t == again.t && at.nt == again.nt && at.lo == again.lo && at.end == again.end);
      const int id = c.pl.segs[at.b] + at.mb * H + at.g, key0 = (at.lo & -c.p.tile) + at.t * c.p.tile;
      WANT(id >= 0 && id < segs && at.t >= 0 && at.t < at.nt);
      std::vector<int>& s = seen[id];
      s.resize(at.end);
      for (int k = key0; k < key0 + c.p.tile; k++)
        if (k >= at.lo && k < at.end) s[k]++;
      // The part's share of the segment ends here: its entry.
      if (tile + 1 == tile1 || at.t + 1 == at.nt) {
        if (tile - at.t >= tile0) entries[id].x = w;
        if (at.t + 1 == at.nt) entries[id].y = w;
      }
      if (tile + 1 < tile1) advance(c.p, c.pl, B, at);
    }
  }
  for (int b = 0; b <= B; b++) {
    const Entry e = entry_of(c.p, c.pl, b, B);
    if (!e.keys) continue;
    const int lo = b < B && sees_prefix(c.p, c.pl, b) ? c.p.prefix : 0, end = b < B ? std::min(c.pl.len[b], c.p.keys_max) : c.pl.len[B];
    for (int i = 0; i < blocks_of(e) * H; i++) {
      const int id = c.pl.segs[b] + i;
      WANT((int)seen[id].size() == end);
      for (int k = 0; k < end; k++) WANT(seen[id][k] == (k >= lo));
      WANT(parts_ok(entries[id], W));
    }
  }
  for (int t = 0; t < (int)c.p.a.tokens; t++) {
    const int b = owner(c.pl, B, t);
    WANT(b >= 0 && c.pl.q0[b] <= t && t < c.pl.q0[b + 1]);
  }
}

int main() {
  std::mt19937 rng(1);
  auto below = [&](int n) { return (int)(rng() % (unsigned)n); };
  // Words that no part left.
  for (int most : {1, 148, 1776})
    for (int x : {INT32_MIN, -1, 0, 1, most - 1, most, most + 1, INT32_MAX, (int)0xcdcdcdcd, 0x7f7f7f7f})
      for (int y : {INT32_MIN, -1, 0, 1, most - 1, most, most + 1, INT32_MAX, (int)0xcdcdcdcd, 0x7f7f7f7f})
        WANT(parts_ok(make_int2(x, y), most) == (x >= 0 && (int64_t)y - x >= 0 && y < most));
  // Divisors, over their whole range.
  for (int i = 0; i < 200000; i++) {
    const int64_t d = i < 3000 ? i + 1 : 1 + (int64_t)(rng() >> (1 + below(31)));
    const Divisor by = divisor(d);
    for (int64_t n : {(int64_t)0, d - 1, d, d + 1, 2 * d - 1, 7 * d, (int64_t)INT32_MAX, (int64_t)INT32_MAX - 1, (int64_t)(rng() >> 1), (int64_t)(rng() >> 12)})
      if (n >= 0 && n <= INT32_MAX) WANT(by((int)n) == (int)(n / d));
  }
  for (int i = 0; i < 400; i++) {
    const int B = 1 + below(i % 4 ? 6 : 40), H = 1 + below(4), group = 1 + below(20), tile = below(2) ? 32 : 16;
    const int keys_max = 1 + below(3000), shared = below(3) ? below(2000) : 0;
    std::vector<int> rows(B), lens(B);
    for (int b = 0; b < B; b++) {
      rows[b] = below(4) ? below(6) : 0;
      lens[b] = below(5) == 0 ? 0 : below(3) ? shared + below(700) : below(4000);
    }
    for (bool on_tiles : {false, true}) {
      const Cut c(rows, lens, H, group, tile, keys_max, shared, on_tiles);
      for (int parts : {1, 7, 8 * 148, 12 * 148}) check(c, parts);
    }
  }
  return 0;
}
