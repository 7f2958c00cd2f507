// latent_shares.cu -- the shares of a step over latent rows, made on the host by the code that
// the plan's kernel makes them with, and what must hold of them: test_latent_shares.py
// compiles and runs it.
//
// Reads steps, one a line: form (0 absorbed, 1 expanded), grow, heads, latent, most rows of a
// request, SMs, requests, then the rows and the tokens of each.  Answers, for each: workers,
// whole tiles of each, empty shares, steps of tiles that no part or more than one covers,
// parts that a join reads and nobody leaves, results left twice, borders that no join knows.
#include <algorithm>
#include <cstdio>
#include <map>
#include <vector>

#include "../graftrepository_b200/csrc/latent.cuh"

using namespace grm_b200;
using namespace grm_b200::latent;

struct Piece {
  int step0, steps, slot, worker;
};
struct Tile {
  int all = 0;  // steps that it has
  std::vector<Piece> pieces;
};

int main() {
  int form, grow, heads, latent, sms, n;
  long long most;
  while (scanf("%d %d %d %d %lld %d %d", &form, &grow, &heads, &latent, &most, &sms, &n) == 7) {
    std::vector<int32_t> fresh(n), lens(n), starts(n + 1, 0), tile(n + 1, 0);
    std::vector<int64_t> base(n + 1, 0);
    for (auto* v : {&fresh, &lens})
      for (auto& x : *v)
        if (scanf("%d", &x) != 1) return 1;
    for (int r = 0; r < n; ++r) starts[r + 1] = starts[r] + fresh[r];
    const Tiling tiling = form ? expanded_tiling(heads, sms)
                               : absorbed_tiling(heads, latent, most, sms);
    const View v{base.data(), tile.data(), starts.data(), lens.data(), n, tiling, grow, heads};
    for (int r = 0; r < n; ++r) {
      const Request q = request_of(v, r);
      base[r + 1] = base[r] + q.total * tiling.groups;
      tile[r + 1] = tile[r] + q.tiles * tiling.groups;
    }
    // the plan's kernel, with its sums over the block one after another
    Header h{0, form ? std::max(tile[n] / tiling.workers - 1, 0) : 0, 0};
    int64_t first = 0;
    if (h.waves > 0) {
      Walk walk;
      walk.enter(v, 0);
      walk.tile(v, h.waves * tiling.workers);
      first = base[walk.r] + walk.g * walk.q.total + units_before(walk.q, v, walk.j);
    }
    const int64_t rest = base[n] - first;
    h.workers = rest == 0 ? 0
                : h.waves ? tiling.workers
                          : (int)std::min<int64_t>(tiling.workers,
                                                   std::max<int64_t>(rest / kLeast, 1));
    const int workers = h.workers;
    std::vector<int64_t> cost(workers, 0), need(workers), raw(workers + 1);
    for (int r = 0; r < n && h.waves; ++r) {
      const Request q = request_of(v, r);
      for (int x = 0; x < q.tiles * tiling.groups && tile[r] + x < h.waves * workers; ++x)
        cost[(tile[r] + x) % workers] += tile_units(q, v, x % q.tiles);
    }
    auto sum_of = [](const std::vector<int64_t>& x) {
      int64_t s = 0;
      for (int64_t y : x) s += y;
      return s;
    };
    if (workers) {
      int64_t level = share_level(rest, sum_of(cost), workers, workers, tiling.start);
      for (int active = workers; h.waves > 0;) {
        int left = 0;
        int64_t sum = 0;
        for (int64_t c : cost)
          if (level - c >= tiling.start) {
            ++left;
            sum += c;
          }
        if (left == active) break;
        active = left;
        level = share_level(rest, sum, workers, active, tiling.start);
      }
      for (int w = 0; w < workers; ++w) need[w] = std::max<int64_t>(level - cost[w], tiling.start);
    }
    int64_t before = 0;
    const int64_t all = sum_of(need);
    for (int w = 0; w < workers; before += need[w++])
      raw[w] = first + (int64_t)((double)before * ((double)rest / (double)all));
    raw[workers] = base[n];
    std::vector<Start> start(workers + 1);
    std::vector<Join> join(workers);
    start[workers].u = base[n];
    int empty = 0;
    for (int w = 0; w < workers; ++w) {
      place_share(v, raw.data(), workers, w, form == 1, &start[w], &join[w]);
      empty += raw[w] >= raw[w + 1];
    }

    // what the workers do
    Params p{};
    p.l.header = &h;
    p.l.start = start.data();
    p.v = v;
    p.causal = grow;
    p.heads = heads;
    std::map<std::vector<int>, Tile> tiles;
    std::vector<int> left(2 * workers, 0);
    auto work = [&](auto parts, int w, int step) {
      Part x;
      while (parts.next(p, &x)) {
        const int toks = x.toks[0] + x.toks[1];
        const int sees = grow ? std::min(x.len, x.cached + x.tok0 + toks) : x.len;
        Tile& t = tiles[{x.r, x.g, x.tok0}];
        t.all = (sees + step - 1) / step;
        t.pieces.push_back({x.step0, x.steps, x.slot, w});
        if (x.slot >= 0) ++left[x.slot];
      }
    };
    for (int w = 0; w < workers; ++w) {
      if (form) work(Parts<2>(p, h, w, start[w], start[w + 1].u), w, kStep);
      else if (tiling.few) work(Parts<1, 128>(p, h, w, start[w], start[w + 1].u), w, 128);
      else work(Parts<1>(p, h, w, start[w], start[w + 1].u), w, kStep);
    }
    int uncovered = (int)tiles.size() != tile[n], unread = 0, unwritten = 0, twice = 0;
    std::vector<int> joined(2 * workers, 0);
    for (const Join& j : join)
      for (int k = 0; j.rows && k < j.parts; ++k) {
        const int slot = k == 0 ? j.slot : 2 * (j.worker + k);
        joined[slot] = 1;
        unwritten += left[slot] == 0;
      }
    for (int s = 0; s < 2 * workers; ++s) {
      twice += left[s] > 1;
      unread += left[s] && !joined[s];
    }
    for (auto& [key, t] : tiles) {
      std::sort(t.pieces.begin(), t.pieces.end(),
                [](const Piece& a, const Piece& b) { return a.worker < b.worker; });
      int at = 0;
      for (const Piece& x : t.pieces) {
        uncovered += x.step0 != at && x.steps > 0;
        uncovered += (x.slot < 0) != (t.pieces.size() == 1);
        at += x.steps;
      }
      uncovered += at != t.all;
    }
    printf("%d %d %d %d %d %d %d\n", workers, h.waves, empty, uncovered, unwritten, twice, unread);
  }
}
