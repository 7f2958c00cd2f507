// latent.cuh -- what the kernels over pages of latent rows share: how a step's
// attention is cut into shares, and the layout of a plan's work area.
#pragma once

#include <cuda.h>

#include "paged.cuh"

namespace grm_b200 {
namespace latent {

constexpr int kStep = 64;   // tokens of a step of the softmax
constexpr int kRows = 128;  // rows of a query tile
// Tokens of a request are expanded from a multiple of this on.
constexpr int kExpandAlign = 64;

// Both forms of attention go over tiles of query rows, each of which sees some of
// its request's tokens, and every worker (a block, one an SM) gets work of the same
// cost in units: a tile costs the tokens that it sees, and Tiling::start more for its
// queries, first scores and result.  Tiles lie one after another, a request's by group (a
// head of the expanded form; of the absorbed one 128 heads) and then by token; a worker's
// share may start and end inside a tile, whose parts join_kernel puts together.  The units
// of a tile's start come first, so that whoever takes some of its tokens from the
// beginning pays them; who goes on inside a tile pays once, as nearly everybody does.  A
// share does not begin among them, nor within a step after them: it takes the whole tile.
//
// A step of 64 tokens and a part of a tile take, by a fit over the blocks' times: 0.66 and
// 5.9 us (64 requests of 32 to 16,384 tokens, one row, 40 heads of 256 + 32), 1.2 and 5.5
// (16 of them with 5 rows), 0.97 and 6.0 expanded (8,449 rows on 31,000 tokens, 40 heads of 64
// + 32), 2.2 and 3.6 (3,499 rows, 16 heads of 128 + 64).
// Both sides, us of those four: absorbed 448 46.2 and 33.6, 512 45.3 and 33.7, 640 45.4 and
// 35.0; expanded 192 1,698 and 123.5, 256 1,697 and 117.0, 320 1,699 and 119.1.  Those four
// are all that stands behind them: a fit for one case alone would be 570, 290, 395 or 105, and
// latents of 128 and 512 and latent_few.cu's kernel go by the same without one.
constexpr int kAbsorbedStart = 512, kExpandedStart = 256;
// Fewest units of a worker: weighs the parts that join_kernel has to read against blocks
// that stand idle (with 1,024 the 16 requests of 5 rows take 39.0 us, with 640 33.4).
constexpr int kLeast = 640;
constexpr int kMostWorkers = 1024;
// A tile of the expanded form that has rows for one of its two query tiles takes about
// so many eighths for a token (6: the same times within 0.5 %).
constexpr int kAlone = 5;

// The expanded form's tiles are many where requests are long, and each head has keys and
// values of its own: in equal shares one after another the workers would be at as many
// heads as there are, whose keys and values L2 does not hold (8,449 rows of 40 heads:
// 6.5 GB from HBM).  So all but the last one or two tiles of a worker go out whole, tile i
// to worker i mod workers: 0.6 GB, in about the same time, as the softmax is what it is
// bound by, but not at HBM's cost in power.  The rest is shared so that all have the same.

struct Header {     // written by the schedule kernel, one for each form
  int32_t workers;  // that have a share
  int32_t waves;    // tiles of each worker that go out whole
  int32_t lost;     // more tokens to expand than there is room for
};

// Where a worker's share starts: the tile, its first unit, and the share's.
struct alignas(16) Start {
  int32_t r, g, j;       // request, group, tile
  int32_t from, n, len;  // the request's first packed row, rows, tokens
  int64_t first, u;
};

// A tile that lies in the shares of several workers, as join_kernel goes by: one for
// each border between two shares that is inside a tile.
struct alignas(32) Join {
  int64_t row;     // of the results, [tokens * heads], of the tile's first row
  int32_t rows;    // 0: the border is not inside a tile
  int32_t parts;
  int32_t slot;    // of the first part; the others' are 2 (worker + k)
  int32_t worker;  // of the first part
  int32_t border;  // of the tile's borders, from 0 on
};

struct Lists {
  Header* header;
  int64_t* base;  // [requests + 1] first unit of each request
  int32_t* tile;  // [requests + 1] first tile of each request (expanded form)
  Start* start;   // [workers + 1]
  Join* join;     // [workers], of the border where each begins
  float* part;    // [workers * splits * 2] partial results, see slot_floats
};

// Tiles of one form: tokens and groups of a request, and how a row of a tile is one
// of (token, head).
struct Tiling {
  int per;      // tokens of a tile
  int groups;   // tiles of the same tokens
  int splits;   // blocks that share a tile's values
  int workers;  // most
  int start;    // units of a tile's start
  int few;      // columns of latent_few.cu's kernel, which serves the step; 0: it does not
};
// The absorbed form's kernel for few rows (latent_few.cu) takes requests of up to 32 rows
// of a step over a latent of 512, where latent_attend.cu's needs two blocks for a tile and
// both work out the scores.  Both sides over 512 + 64, us: one request of 250,007 tokens, one
// row of 16 heads, 158 and with latent_few.cu's 71, of 32 heads 157 and 85; 64 of 4,096 171
// and 73, 173 and 87; 148 of 4,096, 16 heads, 344 and 124; 64 of 1,000 with 4 rows of 8 heads
// 51 and 42; one of 333, 16 heads, 21 and 17.  Its buffers have no room for more rows; over
// smaller latents it is the slower one (70 us against 102 us for 148 requests of 4,096
// tokens, 40 heads of 256 + 32).
__host__ __device__ inline Tiling absorbed_tiling(int heads, int latent, int64_t most_tokens,
                                                  int sms) {
  const int64_t most = most_tokens * heads;
  if (latent == 512 && most <= 32)
    return {(int)most_tokens, 1, 1, sms, kAbsorbedStart, most <= 16 ? 16 : 32};
  const int splits = latent > 256 ? latent / 256 : 1;
  return {heads <= kRows ? kRows / heads : 1, heads <= kRows ? 1 : (heads + kRows - 1) / kRows,
          splits, sms / splits, kAbsorbedStart, 0};
}
__host__ __device__ inline Tiling expanded_tiling(int heads, int sms) {
  return {2 * kRows, heads, 1, sms, kExpandedStart, 0};
}
// fp32 of a partial result: [rows][values], then [rows][4] of reference exponent, sum,
// sum of the rounded weights, and what there is of the row:
constexpr float kNoResult = 0.0f;    // the part has no steps, and left no values
constexpr float kSeesNothing = 1.0f;  // the row sees none of the part's tokens
constexpr float kSees = 2.0f;
// A row that sees tokens has a sum, but where all of their scores are -inf: that one is
// NaN, as 0 / 0 is, and its log-sum -inf.
__host__ __device__ constexpr int slot_floats(int rows, int values) { return rows * (values + 4); }

// Byte offsets in the work area, which follow from the plan's sizes alone.
struct Shape {
  Tiling tiling[2];  // absorbed, expanded
  int64_t off_header[2], off_base[2], off_tile[2], off_start[2], off_join[2];
  int64_t off_part, off_room, off_keys, off_values, bytes;
};

int make_shape(const grm_b200_latent_plan& p, int sms, Shape* s);

inline Lists lists_of(const Shape& s, int form, void* work) {
  char* b = static_cast<char*>(work);
  return {reinterpret_cast<Header*>(b + s.off_header[form]),
          reinterpret_cast<int64_t*>(b + s.off_base[form]),
          reinterpret_cast<int32_t*>(b + s.off_tile[form]),
          reinterpret_cast<Start*>(b + s.off_start[form]),
          reinterpret_cast<Join*>(b + s.off_join[form]),
          reinterpret_cast<float*>(b + s.off_part)};
}

// What the walk over a form's tiles goes by.
struct View {
  const int64_t* base;
  const int32_t* tile;
  const int32_t* starts;
  const int32_t* lens;
  int64_t requests;
  Tiling tiling;
  int grow, heads;
};

struct Params {
  Lists l;
  View v;
  unsigned probes;    // of a bounded wait: paged::kProbes, or less by GRM_B200_WAIT_LIMIT
  const int32_t* room;  // [requests + 1] first expanded token of each request
  uint16_t* keys;       // [heads][expand_tokens][2 * nope]: rounded, and what that left over
  uint16_t* values;     // [heads][expand_tokens][value]
  const int32_t* table;
  int64_t width, tokens, pages, expand_tokens;
  int page_shift, heads, latent, rope, nope, causal, dtype;
  const uint16_t* cache;
  const uint16_t* q;  // absorbed: the latent part; expanded: nope + rope values
  int64_t q_row, q_head;
  const uint16_t* qr;  // the positional part
  int64_t qr_row, qr_head;
  const uint16_t* weights;
  int64_t w_head, w_row;
  float scale_log2;
  uint16_t* out;
  float* lse;
  int32_t* status;
};

int launch_absorbed(const Params& p, cudaStream_t st);
int launch_few(const Params& p, cudaStream_t st);
int launch_expanded(const Params& p, cudaStream_t st);
int launch_expand(const Params& p, cudaStream_t st);

// cuTensorMapEncodeTiled of 16-bit rows: `rank` dims (2 or 3), strides of all but the
// first in elements.  The innermost box is 64 values (128-byte swizzle) or 32 (64).
int make_map(CUtensorMap* map, const void* base, int rank, const int64_t* dims,
             const int64_t* strides, const int* box);

// ---- the shares

template <typename I>
__host__ __device__ __forceinline__ I imin(I a, I b) {
  return a < b ? a : b;
}

struct Request {
  int start, n, len, cached, tiles;
  int64_t total;  // units of a group
};
// Units of tile j, which sees cached + (j + 1) * per tokens of a causal step, but no more
// than len.
__host__ __device__ __forceinline__ int64_t tile_units(const Request& q, const View& v, int j) {
  const int per = v.tiling.per;
  const bool last = j + 1 == q.tiles;
  const int64_t sees = !v.grow || last ? (int64_t)q.len : q.cached + (int64_t)(j + 1) * per;
  const bool alone = per == 2 * kRows && last && q.n - j * per <= kRows;
  return (alone ? sees * kAlone / 8 : sees) + v.tiling.start;
}
// Of the first j tiles of a group.
__host__ __device__ __forceinline__ int64_t units_before(const Request& q, const View& v, int j) {
  const int full = imin(j, q.tiles - 1);
  int64_t u = (int64_t)full * (q.cached + v.tiling.start);
  if (v.grow) u += (int64_t)v.tiling.per * full * (full + 1) / 2;
  return j < q.tiles ? u : u + tile_units(q, v, j - 1);
}
__host__ __device__ __forceinline__ Request request_of(const View& v, int r) {
  const int start = v.starts[r], n = v.starts[r + 1] - start, len = v.lens[r];
  Request q{start, n, len, v.grow ? len - n : len, (n + v.tiling.per - 1) / v.tiling.per, 0};
  q.total = q.tiles > 0 ? units_before(q, v, q.tiles) : 0;
  return q;
}

// The tile that holds a unit, and on from there.
struct Walk {
  int r, g, j;
  Request q;
  int64_t first, last;  // units of the tile

  __host__ __device__ __forceinline__ void enter(const View& v, int request) {
    r = request;
    q = request_of(v, r);
  }
  __host__ __device__ __forceinline__ void seek(const View& v, int64_t u, int request) {
    enter(v, request);
    const int64_t x = u - v.base[r];
    g = (int)(x / q.total);
    const int64_t y = x - g * q.total;
    int lo = 0, hi = q.tiles;  // the last tile that starts at y or before
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (units_before(q, v, mid) <= y) lo = mid;
      else hi = mid;
    }
    j = lo;
    first = v.base[r] + g * q.total + units_before(q, v, j);
    last = first + tile_units(q, v, j);
  }
  __host__ __device__ __forceinline__ void start(const View& v, const Start& s) {
    r = s.r;
    g = s.g;
    j = s.j;
    q = Request{s.from, s.n, s.len, v.grow ? s.len - s.n : s.len,
                (s.n + v.tiling.per - 1) / v.tiling.per, 0};
    first = s.first;
    last = first + tile_units(q, v, j);
  }
  // The i-th of all tiles, from the request where this one is on.
  __host__ __device__ __forceinline__ void tile(const View& v, int i) {
    if (i >= v.tile[r + 1]) {
      int lo = r + 1, hi = (int)v.requests;
      while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (v.tile[mid] <= i) lo = mid;
        else hi = mid;
      }
      enter(v, lo);
    }
    const int x = i - v.tile[r];
    g = x / q.tiles;
    j = x - g * q.tiles;
  }
  __host__ __device__ __forceinline__ void next(const View& v) {  // there is one
    first = last;
    if (++j == q.tiles) {
      j = 0;
      if (++g == v.tiling.groups) {
        g = 0;
        // the next request that has units
        int lo = r + 1;
        if (v.base[lo + 1] <= first) {
          int hi = (int)v.requests;
          while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (v.base[mid] <= first) lo = mid;
            else hi = mid;
          }
        }
        enter(v, lo);
      }
    }
    last = first + tile_units(q, v, j);
  }
};

// What whole tiles and share of a worker come to together: the same for all, but that a
// share is a tile's start at the least, which is what workers get whose whole tiles cost
// more than that leaves room for.  `active` workers, whose whole tiles cost `cost`, are not
// among those.  Found by taking out, from all on, those that the level leaves less, until
// there are none: it falls from step to step, and somebody is left, as the rest of the
// tiles is as many as there are workers, each a start or more.  No share is empty then,
// which join_kernel counts on: a worker that has a border inside a tile leaves a part.
// (Needs that were cut to fit instead left shares of no unit where whole tiles cost very
// different amounts: 64 heads of requests of 300, 10^6, 300, 300 and 300 tokens.)
__host__ __device__ __forceinline__ int64_t share_level(int64_t rest, int64_t cost, int workers,
                                                        int active, int start) {
  return (rest - (int64_t)(workers - active) * start + cost) / active;
}

// The worker whose share has unit u, the last one that starts there or before.
__host__ __device__ __forceinline__ int worker_of(const int64_t* raw, int workers, int64_t u) {
  int lo = 0, hi = workers;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (raw[mid] <= u) lo = mid;
    else hi = mid;
  }
  return lo;
}

// Where the share of worker w starts, which gets the units from raw[w] on, and the tile
// that it shares with the one before.  (Called: inlined into the plan's kernel it costs the
// loops before it registers, 4,096 requests of the expanded form 190 us, not 180.)
__host__ __device__ __noinline__ inline void place_share(const View& v, const int64_t* raw,
                                                     int workers, int w, bool expanded,
                                                     Start* start, Join* join) {
  const int snap = v.tiling.start + kStep;  // a share does not begin before that in a tile
  const int64_t u = raw[w];
  int lo = 0, hi = (int)v.requests;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (v.base[mid] <= u) lo = mid;
    else hi = mid;
  }
  Walk walk;
  walk.seek(v, u, lo);
  const bool inside = u - walk.first >= snap;
  *start = Start{walk.r, walk.g, walk.j, walk.q.start, walk.q.n, walk.q.len, walk.first,
                 inside ? u : walk.first};
  Join j{0, 0, 0, 0, 0, 0};
  if (inside) {
    // whose share has the tile's first token
    const int w0 = worker_of(raw, workers, walk.first + snap - 1);
    const int tok0 = walk.j * v.tiling.per, toks = imin(v.tiling.per, walk.q.n - tok0);
    const bool wide = !expanded && v.tiling.groups > 1;
    j.row = (int64_t)(walk.q.start + tok0) * v.heads +
            (expanded ? walk.g : wide ? walk.g * kRows : 0);
    j.rows = expanded ? toks : wide ? imin(kRows, v.heads - walk.g * kRows) : toks * v.heads;
    j.parts = worker_of(raw, workers, walk.last - 1) - w0 + 1;
    j.slot = 2 * w0 + (raw[w0] >= walk.first ? 0 : 1);
    j.worker = w0;
    j.border = w - 1 - w0;
  }
  *join = j;
}

// A worker's part of a tile.
struct Part {
  int r, g, tok0;       // request, group, first token of the tile within the step
  int toks[2];          // tokens of the two query tiles (the second one's: expanded form)
  int start, n, cached, len;
  int step0, steps;     // of STEP tokens
  int slot;             // where its result goes, -1: it is the whole tile's
};

// The parts of worker `w`, one after another.
template <int QUERIES, int STEP = kStep>
struct Parts {
  Walk walk;
  int64_t u, end;
  int w, whole, waves, count;

  // `until`: where the next worker's share starts
  __host__ __device__ __forceinline__ Parts(const Params& p, const Header& h, int worker,
                                            const Start& start, int64_t until)
      : u(start.u), end(until), w(worker), whole(0), waves(h.waves), count(0) {
    if (QUERIES == 2 && waves > 0) walk.enter(p.v, 0);
    else walk.start(p.v, start);
  }
  __host__ __device__ __forceinline__ bool next(const Params& p, Part* x) {
    const bool all_of_it = QUERIES == 2 && whole < waves;
    if (all_of_it) {
      walk.tile(p.v, whole * p.v.tiling.workers + w);
      ++whole;
    } else {
      if (u >= end) return false;
      if (QUERIES == 2 && waves > 0 && count == 0) walk.start(p.v, p.l.start[w]);
      if (count > 0) walk.next(p.v);
    }
    x->r = walk.r;
    x->g = walk.g;
    x->start = walk.q.start;
    x->n = walk.q.n;
    x->cached = walk.q.cached;
    x->len = walk.q.len;
    x->tok0 = walk.j * p.v.tiling.per;
    const int toks = imin(p.v.tiling.per, x->n - x->tok0);
    x->toks[0] = QUERIES == 2 ? imin(toks, kRows) : toks;
    x->toks[1] = QUERIES == 2 ? toks - x->toks[0] : 0;
    const int sees = p.causal ? imin(x->len, x->cached + x->tok0 + toks) : x->len;
    const int all = (sees + STEP - 1) / STEP;
    if (all_of_it) {
      x->step0 = 0;
      x->steps = all;
      x->slot = -1;
      return true;
    }
    // The step that a unit of the tile falls on.  Any rounding will do, as the workers on
    // both sides of a border round alike; a division in 64 bits is 100 instructions.
    const int start = p.v.tiling.start;
    const int units = (int)(walk.last - walk.first), from = (int)(u - walk.first);
    const int to = (int)(imin(end, walk.last) - walk.first);
    const float per_unit = (float)all / (float)(units - start);  // not used where that is 0
    x->step0 = from == 0 ? 0 : imin(all, (int)((float)(from - start) * per_unit));
    x->steps = (to == units ? all : imin(all, (int)((float)(to - start) * per_unit))) - x->step0;
    x->slot = from == 0 && to == units ? -1 : 2 * w + (count > 0 ? 1 : 0);
    u = imin(end, walk.last);
    ++count;
    return true;
  }
};

}  // namespace latent
}  // namespace grm_b200
