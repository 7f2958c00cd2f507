// paged_plan.cu -- a step of the 8-bit paged arena planned on the GPU: block
// table, slots, positions, and the work lists of append and attention, all
// from the requests' lengths in one launch.
//
// With have = ceil(cached / P) and need = ceil((cached + fresh) / P), request
// r takes need - have pages; page j in [have, need) is
//   ring[(taken + sum of the requests before r + j - have) mod pages],
// and token t of the step's packed rows, at position p of its request, has the
// slot page(p / P) * P + p % P.  Everything is a prefix sum over the requests
// followed by one independent write for each entry.
//
// One launch without a barrier between blocks: every block adds up all requests
// itself (8 bytes a request, from L2), in chunks of kPlanThreads, and keeps what
// stands before its own chunk; a prefix sum of that chunk alone then tells where
// each of its entries goes, and the block writes one kind of entries, finding an
// entry's request by a binary search in shared memory.  A new page's number comes
// from the ring, not from the table entry another block writes, so no block
// waits for another.  The kinds run side by side because each is a chain of
// dependent reads, and a step's plan is bound by those: one block for all of
// them, chunk after chunk, took 31 us for 4,096 requests and 262,694 rows, where
// this takes 13; 64 requests of one row take 6.5 us, about three such chains.  That
// every block adds up all requests makes the work grow with their square: 18 us for
// 16,384 requests of one row, 94 for 65,536, 1.2 ms for 2^18 and 18 ms for 2^20, the
// most that a plan takes.
#include <algorithm>

#include "paged.cuh"

namespace grm_b200 {
namespace paged {

namespace {

constexpr int kPlanThreads = 1024;
constexpr int kPlanWarps = kPlanThreads / 32;
// Segments of no more units are left whole.  us with 3, 5 and 8: one request of 333
// tokens 12.1, 10.0, 10.1; 8 of 300 tokens 13.6, 11.1, 11.2; 24 of 200 to 2,000 at
// head_dim 128 21.7, 21.8, 25.6; 24 of up to 3,000 at head_dim 64 18.5, 18.4, 19.9; 16
// of 100 to 1,000 at head_dim 256 16.2, 16.0, 24.1.
constexpr int kJoinUnits = 5;
constexpr int kBuckets = 256;  // of prompt tiles by what they see
// A part of a prompt tile has no fewer tokens.  us with 128, 256, 512 and 1,024: one
// request of 4,096 tokens, 32 pairs, head_dim 256 25.7, 24.3, 26.0, 32.4; of 1,024
// tokens, 160 pairs, head_dim 128 23.8, 23.6, 25.7, 31.7; 4 of 700 tokens at head_dim
// 64 17.6, 17.7, 19.5, 21.7; 2 of 2,000 tokens, 400 pairs 40.0, 40.0, 40.0, 45.1; one of
// 16,000 on 4 kv heads 39.9, 40.0, 38.1, 41.7.
constexpr int kPartTokens = 256;
// Most tokens of a request, its new rows included: what rounds up to tiles or looks
// one tile ahead stays below 2^31.
constexpr int64_t kMaxTokens = ((int64_t)1 << 31) - 1024;
constexpr int kSizes = 4;  // candidate part sizes, see plan_kernel
// The sums over requests: pages taken, rows, pages touched, prompt tiles or their
// parts (all of them below 2^31 in a step that can be planned) and the split
// kernel's units; and two that only totals are needed of, the split kernel's
// segments and the tokens of the requests of all prompt tiles.
constexpr int kSums = 7;
constexpr int kTake = 0, kRows = 1, kTouched = 2, kTiles = 3, kUnits = 4;
constexpr int kSegments = 5, kTokens = 6;

struct PlanParams {
  int64_t requests, tokens, max_fresh, width, ring_size;
  int page_shift, grow, kv_heads, sms;
  int block_shift, tile_shift;  // log2 of a segment's rows and a tile's tokens
  int chunks, row_blocks, page_blocks;  // blocks for a chunk's rows, and for its pages
  Shape s;
  const int32_t* cached;
  const int32_t* fresh;
  const int32_t* ring;
  const int64_t* cursor_in;
  int32_t* table;
  int32_t* lens;
  int32_t* starts;
  int32_t* positions;
  int32_t* rows;
  int64_t* slots;
  int64_t* cursor;
  int32_t* status;
  Lists l;
};

struct Request {
  int cached, fresh, after, have, need;
};

// Parts of a prompt request's tiles, for `part_tokens` in each (0: whole).
__device__ __forceinline__ int parts_of(int after, int part_tokens) {
  return part_tokens == 0 ? 1 : max(1, (after + part_tokens - 1) / part_tokens);
}

// What request r adds to each sum, its prompt tiles whole.
__device__ __forceinline__ void weigh(const PlanParams& p, const Request& q, int64_t (&v)[kSums]) {
  v[kTake] = q.need - q.have;
  v[kRows] = q.fresh;
  v[kTouched] = p.grow && q.fresh > 0 ? q.need - (q.cached >> p.page_shift) : 0;
  const int64_t pairs = (int64_t)q.fresh * p.s.group;
  const bool prompt = pairs > p.s.prompt_rows && p.s.qtile_cap > 0;
  v[kTiles] = prompt ? (int64_t)(((unsigned)q.fresh + p.s.qtile_tokens - 1) /
                                 (unsigned)p.s.qtile_tokens)
                     : 0;
  v[kTokens] = v[kTiles] * q.after;
  v[kSegments] = prompt ? 0 : p.kv_heads * ((pairs + p.s.block_rows - 1) >> p.block_shift);
  v[kUnits] = v[kSegments] * (((q.after + p.s.tile - 1) >> p.tile_shift) + 1);
}

// Sum of a warp's values in [0, 2^50), in two 32-bit reductions.
__device__ __forceinline__ int64_t warp_sum(int64_t v) {
  const unsigned lo = __reduce_add_sync(kFull, (unsigned)v & 0xFFFFFFu);
  const unsigned hi = __reduce_add_sync(kFull, (unsigned)(v >> 24));
  return ((int64_t)hi << 24) + lo;
}

// The last of the n + 1 ascending sums s[0..n] that is <= x (s[n] > x).
template <typename T>
__device__ __forceinline__ int find(const T* s, int n, T x) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (s[mid] <= x) lo = mid;
    else hi = mid;
  }
  return lo;
}

// Inclusive prefix sum over a warp.
template <typename T>
__device__ __forceinline__ T warp_scan(T v, int lane) {
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const T up = __shfl_up_sync(kFull, v, o);
    if (lane >= o) v += up;
  }
  return v;
}

// What a block writes of its chunk.
constexpr int kWriteRows = 0, kWriteRequests = 1, kWritePages = 2, kWriteWork = 3;

__global__ void __launch_bounds__(kPlanThreads) plan_kernel(const PlanParams p) {
  constexpr int kScans = kUnits + 1;
  __shared__ int sum[kScans][kPlanThreads + 1];  // before each request of the chunk, from the start
  __shared__ int s_cached[kPlanThreads], s_have[kPlanThreads];
  __shared__ int64_t part[2 * kSums][kPlanWarps];
  __shared__ int64_t total[2 * kSums];  // of all requests; of those before the chunk
  __shared__ int chunk_part[kScans][kPlanWarps];
  __shared__ int cut[2];  // parts of all tiles, and of those before the chunk
  __shared__ int bucket[kBuckets], most_seen;
  __shared__ int bad;

  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int page = 1 << p.page_shift;
  const int64_t taken0 = p.cursor_in[0], returned = p.cursor_in[1];
  int kind = kWriteRows, chunk = blockIdx.x / p.row_blocks, index = blockIdx.x % p.row_blocks;
  int blocks = p.row_blocks;  // of this kind and chunk
  if (chunk >= p.chunks) {
    const int x = blockIdx.x - p.chunks * p.row_blocks;
    chunk = x % p.chunks;
    const int y = x / p.chunks;  // of a chunk: page_blocks twice, then one
    kind = kWriteRequests + y / p.page_blocks;
    index = y % p.page_blocks;
    blocks = kind == kWriteWork ? 1 : p.page_blocks;
  }
  const int gid = index * kPlanThreads + tid, gsize = blocks * kPlanThreads;

  auto request = [&](int64_t r, int* flags) {
    Request q{0, 0, 0, 0, 0};
    if (r >= p.requests) return q;
    q.cached = p.cached[r];
    q.fresh = p.fresh[r];
    if (q.cached < 0 || q.fresh < 0 || (int64_t)q.cached + q.fresh > kMaxTokens) {
      *flags |= GRM_B200_PLAN_BAD_LENGTH;
      return Request{0, 0, 0, 0, 0};
    }
    if (q.fresh > p.max_fresh) *flags |= GRM_B200_PLAN_ROWS;
    q.after = q.cached + (p.grow ? q.fresh : 0);
    q.have = (q.cached + page - 1) >> p.page_shift;
    q.need = (q.after + page - 1) >> p.page_shift;
    if (q.need > p.width) *flags |= GRM_B200_PLAN_TABLE;
    return q;
  };

  if (tid == 0) bad = 0;

  // ---- totals, the chunk's own requests, and errors
  int64_t v[kSums] = {}, before[kSums] = {}, own[kSums] = {};
  Request q{0, 0, 0, 0, 0};
  int flags = 0;
  for (int c = 0; c < p.chunks; ++c) {
    int64_t a[kSums];
    const Request x = request((int64_t)c * kPlanThreads + tid, &flags);
    weigh(p, x, a);
    if (c == chunk) {
      q = x;
#pragma unroll
      for (int i = 0; i < kSums; ++i) {
        before[i] = v[i];
        own[i] = a[i];
      }
    }
#pragma unroll
    for (int i = 0; i < kSums; ++i) v[i] += a[i];
  }
#pragma unroll
  for (int i = 0; i < kSums; ++i) {
    const int64_t w = warp_sum(v[i]);
    if (lane == 0) part[i][warp] = w;
    if (p.chunks > 1) {
      const int64_t u = warp_sum(before[i]);
      if (lane == 0) part[kSums + i][warp] = u;
    }
  }
  __syncthreads();
  if (flags) atomicOr(&bad, flags);
  if (warp < 2 * kSums) {
    const int64_t w = warp < kSums || p.chunks > 1 ? warp_sum(part[warp][lane]) : 0;
    if (lane == 0) total[warp] = w;
  }
  __syncthreads();
  int failed = bad;

  // A prompt tile and head is one block; where they are fewer than half of the SMs,
  // tiles are cut along their tokens into parts that all run at once.  The fewest
  // tokens that a part can have are between Sum len / SMs and Sum len / (SMs - tiles),
  // which is always enough (Sum ceil(len / part) <= Sum len / part + tiles): of four
  // sizes in between, the smallest whose parts the SMs can hold (16 requests of 100 to
  // 8,192 tokens with 5 rows of head_dim 256: 40 us, 44 with the last one always).
  int part_tokens = 0;
  const int64_t whole = total[kTiles] * p.kv_heads;
  if (whole > 0 && whole <= p.sms / 2) {
#pragma unroll 1
    for (int k = 1; k <= kSizes; ++k) {
      const int64_t each = ceil_div64(total[kTokens] * p.kv_heads, p.sms - whole * k / kSizes);
      part_tokens = (int)(each < kPartTokens ? kPartTokens : each < (1 << 30) ? each : 1 << 30);
      int all = 0, all_before = 0;
#pragma unroll 1
      for (int c = 0; c < p.chunks; ++c) {
        const Request x = c == chunk ? q : request((int64_t)c * kPlanThreads + tid, &flags);
        int64_t a[kSums];
        weigh(p, x, a);
        if (c == chunk) all_before = all;
        all += (int)a[kTiles] * parts_of(x.after, part_tokens);
      }
      all = __reduce_add_sync(kFull, all);
      all_before = __reduce_add_sync(kFull, all_before);
      if (lane == 0) {
        part[0][warp] = all;
        part[1][warp] = all_before;
      }
      __syncthreads();
      if (warp < 2) {
        const int64_t w = warp_sum(part[warp][lane]);
        if (lane == 0) cut[warp] = (int)w;
      }
      __syncthreads();
      if ((int64_t)cut[0] * p.kv_heads <= p.sms) break;
    }
    own[kTiles] *= parts_of(q.after, part_tokens);
    if (tid == 0) {
      total[kTiles] = cut[0];
      total[kSums + kTiles] = cut[1];
    }
    __syncthreads();
  }

  if (total[kRows] > p.tokens || total[kUnits] > INT32_MAX - (1 << 20))
    failed |= GRM_B200_PLAN_ROWS;
  if (taken0 < 0 || returned - taken0 > p.ring_size || total[kTake] > returned - taken0)
    failed |= GRM_B200_PLAN_PAGES;
  const int units = failed ? 0 : (int)total[kUnits];
  const int all_rows = failed ? 0 : (int)total[kRows];
  // Few units: fewer workers.  Joining a segment costs about what kJoinUnits
  // tiles cost, so a step whose segments are no longer than that leaves them
  // whole; longer ones are split down to two units a worker.
  const int mean = units == 0 ? 1 : (int)((units + total[kSegments] - 1) / total[kSegments]);
  const int least = mean <= kJoinUnits ? (mean > 2 ? mean : 2) : 2;
  const int most = (units + least - 1) / least;
  const int workers = most < p.s.workers ? most : p.s.workers;

  if (kind == kWriteRequests && chunk == 0 && gid == 0) {
    p.status[0] = failed;
    p.cursor[0] = taken0 + (failed ? 0 : total[kTake]);
    p.cursor[1] = returned;
    p.starts[p.requests] = all_rows;
  }
  if (kind == kWriteWork && chunk == 0) {
    if (tid == 0) {
      p.l.base[p.requests] = units;
      *p.l.header = Header{units,
                           workers,
                           workers ? units / workers : 0,
                           workers ? units % workers : 0,
                           failed ? 0 : (int)total[kTouched],
                           failed ? 0 : (int)total[kTiles],
                           failed || part_tokens == 0 ? 0 : (int)total[kTiles],
                           all_rows,
                           failed ? 0 : (int)total[kTake],
                           0};
    }
    for (int i = tid; i < p.s.workers; i += kPlanThreads) p.l.count[i] = 0;
  }
  if (kind == kWriteRows)
    for (int64_t i = all_rows + (int64_t)chunk * gsize + gid; i < p.tokens;
         i += (int64_t)p.chunks * gsize) {
      p.positions[i] = -1;
      p.rows[i] = -1;
      p.slots[i] = -1;
    }
  const int64_t r0 = (int64_t)chunk * kPlanThreads;
  const int n = (int)(p.requests - r0 < kPlanThreads ? p.requests - r0 : kPlanThreads);
  if (failed) {
    if (gid < n && kind == kWriteRequests) {
      p.lens[r0 + tid] = p.cached[r0 + tid];
      p.starts[r0 + tid] = 0;
    }
    if (tid < n && kind == kWriteWork) p.l.base[r0 + tid] = 0;
    return;
  }

  // ---- prefix sums of the chunk
  int incl[kScans];
#pragma unroll
  for (int i = 0; i < kScans; ++i) {
    incl[i] = warp_scan((int)own[i], lane);
    if (lane == 31) chunk_part[i][warp] = incl[i];
  }
  s_cached[tid] = q.cached;
  s_have[tid] = q.have;
  __syncthreads();
  if (warp < kScans) {
    const int x = chunk_part[warp][lane];
    const int w = warp_scan(x, lane);
    const int from = (int)total[kSums + warp];
    chunk_part[warp][lane] = from + w - x;
    if (lane == 31) sum[warp][n] = from + w;  // n == kPlanThreads, or requests past n add nothing
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kScans; ++i)
    if (tid < n) sum[i][tid] = chunk_part[i][warp] + incl[i] - (int)own[i];
  __syncthreads();

  const int ring0 = (int)(taken0 % p.ring_size);
  auto ring_page = [&](int x) {  // the x-th page this step takes
    const int64_t at = (int64_t)ring0 + x;
    return p.ring[at < p.ring_size ? at : at - p.ring_size];
  };
  // page j of request r0 + i; one taken in this step is read from the ring
  auto page_of = [&](int i, int j) {
    return j < s_have[i] ? p.table[(r0 + i) * p.width + j]
                         : ring_page(sum[kTake][i] + j - s_have[i]);
  };
  if (kind == kWriteRows) {
    for (int x = sum[kRows][0] + gid; x < sum[kRows][n]; x += gsize) {
      const int i = find(sum[kRows], n, x);
      const int pos = s_cached[i] + x - sum[kRows][i];
      p.rows[x] = (int)(r0 + i);
      p.positions[x] = pos;
      p.slots[x] = p.grow ? ((int64_t)page_of(i, pos >> p.page_shift) << p.page_shift) +
                                (pos & (page - 1))
                          : -1;
    }
  } else if (kind == kWriteRequests) {
    if (gid < n) {
      p.lens[r0 + tid] = q.after;
      p.starts[r0 + tid] = sum[kRows][tid];
    }
    for (int x = sum[kTake][0] + gid; x < sum[kTake][n]; x += gsize) {
      const int i = find(sum[kTake], n, x);
      p.table[(r0 + i) * p.width + s_have[i] + x - sum[kTake][i]] = ring_page(x);
    }
  } else if (kind == kWritePages) {
    for (int x = sum[kTouched][0] + gid; x < sum[kTouched][n]; x += gsize) {
      const int i = find(sum[kTouched], n, x);
      const int j = (s_cached[i] >> p.page_shift) + x - sum[kTouched][i];
      const int first = j << p.page_shift, off = max(s_cached[i] - first, 0);
      const int after = s_cached[i] + sum[kRows][i + 1] - sum[kRows][i];
      p.l.pages[x] = make_int4(sum[kRows][i] + first + off - s_cached[i], page_of(i, j), off,
                               min(after - first, page) - off);
    }
  } else {
    if (tid < n) p.l.base[r0 + tid] = sum[kUnits][tid];
    const int tile0 = sum[kTiles][0], tiles = sum[kTiles][n] - tile0;
    if (tiles > 0) {
      // Parts of prompt tiles in the order of what they see, longest first (the blocks of
      // the prompt kernel start in this order, and the last ones to start decide
      // when it ends): counted into kBuckets, then placed.  The order within a
      // bucket does not matter.
      auto sees = [&](int i, int tok) {  // a causal step's; otherwise about as good
        return s_cached[i] + tok + p.s.qtile_tokens;
      };
      if (tid < kBuckets) bucket[tid] = 0;
      if (tid == 0) most_seen = 0;
      __syncthreads();
      const int top = __reduce_max_sync(kFull, tid < n && own[kTiles] > 0 ? q.cached + q.fresh : 0);
      if (lane == 0) atomicMax(&most_seen, top);
      __syncthreads();
      const int unit = (most_seen + p.s.qtile_tokens) / kBuckets + 1;
      auto entry = [&](int x, int* b) {
        const int i = find(sum[kTiles], n, x);
        const int after = s_cached[i] + (p.grow ? sum[kRows][i + 1] - sum[kRows][i] : 0);
        const int parts = parts_of(after, part_tokens), y = x - sum[kTiles][i];
        const int tok = y / parts * p.s.qtile_tokens, part = y % parts;
        *b = kBuckets - 1 - min(sees(i, tok) / unit, kBuckets - 1);
        return make_int4((int)(r0 + i), tok, part + 256 * parts, x - part);
      };
      int b;
      for (int x = tile0 + tid; x < tile0 + tiles; x += kPlanThreads) {
        entry(x, &b);
        atomicAdd(&bucket[b], 1);
      }
      __syncthreads();
      if (warp == 0) {
        int before = 0;
        for (int b = 0; b < kBuckets; b += 32) {
          const int x = bucket[b + lane], w = warp_scan(x, lane);
          bucket[b + lane] = before + w - x;
          before += __shfl_sync(kFull, w, 31);
        }
      }
      __syncthreads();
      for (int x = tile0 + tid; x < tile0 + tiles; x += kPlanThreads) {
        const int4 e = entry(x, &b);
        p.l.qtiles[tile0 + atomicAdd(&bucket[b], 1)] = e;
      }
    }
    const int share = workers ? units / workers : 0, more = workers ? units % workers : 0;
    for (int w = tid; w < workers; w += kPlanThreads) {
      const int u = w * share + (w < more ? w : more);
      if (u >= sum[kUnits][0] && u < sum[kUnits][n])
        p.l.start[w] = (int)(r0 + find(sum[kUnits], n, u));
    }
  }
}

constexpr int kCommitThreads = 1024;

// One block, as nothing is written before every row has been looked at: a step is
// taken up if its requests still hold what they held when it was planned and no
// page has been taken since.  Pages returned meanwhile and requests without rows in
// the step are left as they are.  (64 requests 1.7 us, 4,096 3.1, 65,536 34 beside a
// plan's 98.)
__global__ void __launch_bounds__(kCommitThreads)
    commit_kernel(int64_t requests, const int32_t* after, const int32_t* starts, Header* header,
                  const int64_t* cursor_after, int32_t* lens, int64_t* cursor, int32_t* status) {
  const int take = header->take;
  const bool again = header->committed != 0;
  bool ready = !again && (take == 0 || cursor[0] == cursor_after[0] - take), done = again;
#pragma unroll 4
  for (int64_t r = threadIdx.x; r < requests; r += blockDim.x) {
    const int n = starts[r + 1] - starts[r], held = lens[r], then = after[r];
    ready &= n <= 0 || held == then - n;
    done &= n <= 0 || held == then;
  }
  ready = __syncthreads_and(ready);
  done = __syncthreads_and(done);
  if (!ready) {
    if (!done && threadIdx.x == 0) atomicOr(status, GRM_B200_PLAN_STALE);
    return;
  }
#pragma unroll 4
  for (int64_t r = threadIdx.x; r < requests; r += blockDim.x) {
    const int n = starts[r + 1] - starts[r], then = after[r];
    if (n > 0) lens[r] = then;
  }
  if (threadIdx.x == 0) {
    if (take > 0) cursor[0] = cursor_after[0];
    header->committed = 1;
  }
}

constexpr int kReleaseThreads = 1024;

// One block: the list in chunks, a prefix sum of the page counts in each.  64
// requests of 1,000 tokens in pages of 64 take 8 us, of 8,000 tokens 24; 4,096 of one
// page 11.
__global__ void __launch_bounds__(kReleaseThreads)
    release_kernel(const int32_t* rows, int64_t count, int64_t requests, int64_t width,
                   int64_t ring_size, int page_shift, const int32_t* table, int32_t* lens,
                   int32_t* ring, int64_t* cursor) {
  __shared__ int64_t sum[kReleaseThreads + 1];
  __shared__ int64_t part[32];
  __shared__ int row_of[kReleaseThreads];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  int64_t returned = cursor[1];
  if (returned < 0) return;
  for (int64_t c0 = 0; c0 < count; c0 += kReleaseThreads) {
    int64_t n_pages = 0;
    int row = -1;
    if (c0 + tid < count) {
      row = rows[c0 + tid];
      // a row listed twice gives its pages to whichever of the two comes first
      if (row >= 0 && row < requests) {
        const int len = atomicExch(&lens[row], 0);
        n_pages = ((int64_t)(len > 0 ? len : 0) + (1 << page_shift) - 1) >> page_shift;
        n_pages = n_pages < width ? n_pages : width;
      }
    }
    const int64_t incl = warp_scan(n_pages, lane);
    __syncthreads();
    if (lane == 31) part[warp] = incl;
    row_of[tid] = row;
    __syncthreads();
    if (warp == 0) {
      const int64_t own = part[lane];
      const int64_t w = warp_scan(own, lane);
      part[lane] = w - own;
      if (lane == 31) sum[kReleaseThreads] = w;
    }
    __syncthreads();
    sum[tid] = part[warp] + incl - n_pages;
    __syncthreads();
    for (int64_t x = tid; x < sum[kReleaseThreads]; x += kReleaseThreads) {
      const int i = find(sum, kReleaseThreads, x);
      ring[(returned + x) % ring_size] = table[row_of[i] * width + (x - sum[i])];
    }
    returned += sum[kReleaseThreads];
  }
  if (tid == 0) cursor[1] = returned;
}

int64_t align256(int64_t v) { return (v + 255) & ~(int64_t)255; }

}  // namespace

int make_shape(const grm_b200_paged_plan& p, int sms, Shape* s) {
  s->group = p.query_heads / p.kv_heads;
  const int64_t most = std::min(p.max_fresh, p.tokens) * s->group;
  s->block_rows = most <= 8 ? 8 : 16;
  // (row, head) pairs a kv head up to which the split kernel serves a request, in
  // segments of 16 rows that read the codes again; a prompt tile costs the same for
  // 1 row and 128.  Split / prompt, us, at 16, 32 and 64 pairs, pages of 64:
  //   head_dim  kv heads  requests x tokens   16 pairs   32 pairs   64 pairs
  //      64        8          16 x 4,096       34 / 58    48 / 59    79 / 59
  //      64        8          64 x 2,048       54 / 121   89 / 121  152 / 121
  //     128        8          16 x 4,096       49 / 66    72 / 66   121 / 67
  //     128        8          64 x 2,048       80 / 136  133 / 138  234 / 140
  //     256        8          16 x 4,096       81 / 82   128 / 83   227 / 85
  //     256        8          64 x 2,048      135 / 172  239 / 177  442 / 180
  //     128        2          16 x 4,096       30 / 32    35 / 32    45 / 34
  //     256        2          16 x 4,096       46 / 36    53 / 39    76 / 44
  //     256        8          16 x 1,024       41 / 30    55 / 31    83 / 32
  // So the rule holds where there is work for all SMs.  Where there is not, the prompt
  // kernel is ahead from fewer pairs on, at head_dim 256 by a third at 16; the rule
  // does not look at that.
  s->prompt_rows = p.head_dim == 256 ? 16 : 32;
  const bool prompts = most > s->prompt_rows;
  s->qtile_tokens = (p.head_dim == 256 ? 1 : 2) * (128 / s->group);
  s->tile = split_tile(p.head_dim);
  s->workers = sms * split_blocks(p.head_dim, s->block_rows);
  const int64_t R = p.requests, T = p.tokens;
  s->page_cap = p.grow ? std::min(T, T / p.page_tokens + 2 * std::min(R, T)) : 0;
  // a tile for every qtile_tokens rows, one more for every prompt, and what the
  // parts add
  s->qtile_cap = prompts ? T / s->qtile_tokens + std::min(R, T * s->group / s->prompt_rows) +
                               ceil_div64(sms, p.kv_heads)
                         : 0;
  int64_t at = align256(sizeof(Header));
  auto take = [&](int64_t bytes) {
    const int64_t o = at;
    at += align256(bytes);
    return o;
  };
  s->off_base = take((R + 1) * 4);
  s->off_start = take((int64_t)s->workers * 4);
  s->off_count = take((int64_t)s->workers * 4);
  s->off_pages = take(std::min(T, T / p.page_tokens + 2 * std::min(R, T)) * 16);
  s->off_qtiles = take(s->qtile_cap * 16);
  s->off_part = take((int64_t)s->workers * 2 * split_slot(p.head_dim, s->block_rows) * 4);
  s->off_qpart = take(prompts ? (int64_t)sms * prompt_slot(p.head_dim) * 4 : 0);
  s->bytes = at;
  return 0;
}

int current_sms(int* sms) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) {
    set_thread_error("no current device: %s", cudaGetErrorString(e));
    return cuda_status(e);
  }
  DeviceInfo info;
  const int rc = device_info(dev, &info);
  if (rc != 0) {
    set_thread_error("device %d has no properties", dev);
    return rc;
  }
  *sms = info.sms;
  return 0;
}

int allow_shared(const void* kernel, int bytes, std::atomic<uint64_t>* done) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  const uint64_t bit = (uint64_t)1 << (dev & 63);
  if (e == cudaSuccess && (done->load(std::memory_order_relaxed) & bit)) return 0;
  if (e == cudaSuccess)
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e != cudaSuccess) {
    set_thread_error("paged attend: %s", cudaGetErrorString(e));
    return cuda_status(e);
  }
  done->fetch_or(bit, std::memory_order_relaxed);
  return 0;
}

int launch_status(const char* what) {
  const cudaError_t e = cudaGetLastError();
  if (e == cudaSuccess) return 0;
  set_thread_error("%s launch failed: %s", what, cudaGetErrorString(e));
  return cuda_status(e);
}

namespace {

bool page_ok(int v) { return v == 16 || v == 32 || v == 64 || v == 128; }
bool dim_ok(int v) { return v == 64 || v == 128 || v == 256; }

int check_sizes(const grm_b200_paged_plan* p) {
  if (!p) {
    set_thread_error("paged plan: null plan");
    return GRM_B200_EINVAL;
  }
  if (p->requests < 1 || p->requests > (1 << 20) || p->tokens < 1 || p->tokens > INT32_MAX ||
      p->max_fresh < 1 || p->table_width < 1 || p->table_width > (1 << 28) || p->pages < 1 ||
      p->pages > INT32_MAX) {
    set_thread_error("paged plan: sizes out of range (requests %lld, tokens %lld, max_fresh %lld, "
                     "table_width %lld, pages %lld)",
                     (long long)p->requests, (long long)p->tokens, (long long)p->max_fresh,
                     (long long)p->table_width, (long long)p->pages);
    return GRM_B200_EINVAL;
  }
  if (!page_ok(p->page_tokens) || !dim_ok(p->head_dim)) {
    set_thread_error("paged plan: page_tokens %d must be 16, 32, 64 or 128 and head_dim %d must be "
                     "64, 128 or 256", p->page_tokens, p->head_dim);
    return GRM_B200_EINVAL;
  }
  if (p->kv_heads < 1 || p->kv_heads > 1024 || p->query_heads < p->kv_heads ||
      p->query_heads % p->kv_heads || p->query_heads / p->kv_heads > 128) {
    set_thread_error("paged plan: query_heads %d must be a multiple of kv_heads %d, at most 128 "
                     "query heads for each", p->query_heads, p->kv_heads);
    return GRM_B200_EINVAL;
  }
  return 0;
}

}  // namespace

int check_plan(const grm_b200_paged_plan* p) {
  int rc = check_sizes(p);
  if (rc) return rc;
  if (!p->cached || !p->ring || !p->cursor_in || !p->table || !p->lens || !p->starts ||
      !p->positions || !p->rows || !p->slots || !p->cursor || !p->status || !p->scratch) {
    set_thread_error("paged plan: a buffer is missing");
    return GRM_B200_EINVAL;
  }
  if (p->cursor == p->cursor_in || p->lens == p->cached) {
    set_thread_error("paged plan: cursor and lens must not be the buffers they are made from");
    return GRM_B200_EINVAL;
  }
  if (reinterpret_cast<uintptr_t>(p->scratch) & 255) {
    set_thread_error("paged plan: scratch must be 256-byte aligned");
    return GRM_B200_EINVAL;
  }
  int64_t need = 0;
  rc = grm_b200_paged_scratch_bytes(p, &need);
  if (rc) return rc;
  if (p->scratch_bytes < need) {
    set_thread_error("paged plan: scratch of %lld bytes, %lld needed",
                     (long long)p->scratch_bytes, (long long)need);
    return GRM_B200_EINVAL;
  }
  return 0;
}

int check_arena(const grm_b200_paged_arena* a) {
  if (!a || !a->k_codes || !a->v_codes || !a->k_scales || !a->v_scales) {
    set_thread_error("paged arena: a buffer is missing");
    return GRM_B200_EINVAL;
  }
  if (a->pages < 1 || a->kv_heads < 1 || a->pages > INT32_MAX / a->kv_heads || a->kv_heads > 1024 ||
      !page_ok(a->page_tokens) || !dim_ok(a->head_dim)) {
    set_thread_error("paged arena: pages %lld, kv_heads %d, page_tokens %d (16, 32, 64, 128), "
                     "head_dim %d (64, 128, 256)",
                     (long long)a->pages, a->kv_heads, a->page_tokens, a->head_dim);
    return GRM_B200_EINVAL;
  }
  if ((reinterpret_cast<uintptr_t>(a->k_codes) | reinterpret_cast<uintptr_t>(a->v_codes)) & 15) {
    set_thread_error("paged arena: codes must be 16-byte aligned");
    return GRM_B200_EINVAL;
  }
  return 0;
}

int check_match(const grm_b200_paged_plan* p, const grm_b200_paged_arena* a) {
  if (a->pages != p->pages || a->kv_heads != p->kv_heads || a->page_tokens != p->page_tokens ||
      a->head_dim != p->head_dim) {
    set_thread_error("paged plan and arena differ: pages %lld / %lld, kv_heads %d / %d, "
                     "page_tokens %d / %d, head_dim %d / %d",
                     (long long)p->pages, (long long)a->pages, p->kv_heads, a->kv_heads,
                     p->page_tokens, a->page_tokens, p->head_dim, a->head_dim);
    return GRM_B200_EINVAL;
  }
  return 0;
}

}  // namespace paged
}  // namespace grm_b200

using namespace grm_b200;
using namespace grm_b200::paged;

extern "C" {

int grm_b200_paged_scratch_bytes(const grm_b200_paged_plan* plan, int64_t* out_bytes) {
  int rc = check_sizes(plan);
  if (rc) return rc;
  if (!out_bytes) {
    set_thread_error("paged plan: null out_bytes");
    return GRM_B200_EINVAL;
  }
  int sms = 0;
  rc = current_sms(&sms);
  if (rc) return rc;
  Shape s;
  make_shape(*plan, sms, &s);
  *out_bytes = s.bytes;
  return 0;
}

int grm_b200_paged_plan_step(const grm_b200_paged_plan* plan, const int32_t* fresh_device,
                             void* stream) {
  int rc = check_plan(plan);
  if (rc) return rc;
  if (!fresh_device) {
    set_thread_error("paged plan: null fresh");
    return GRM_B200_EINVAL;
  }
  int sms = 0;
  if ((rc = current_sms(&sms))) return rc;
  PlanParams p;
  p.requests = plan->requests;
  p.tokens = plan->tokens;
  p.max_fresh = plan->max_fresh;
  p.width = plan->table_width;
  p.ring_size = plan->pages;
  p.page_shift = shift_of(plan->page_tokens);
  p.grow = plan->grow ? 1 : 0;
  p.kv_heads = plan->kv_heads;
  p.sms = sms;
  make_shape(*plan, sms, &p.s);
  p.block_shift = p.s.block_rows == 8 ? 3 : 4;
  p.tile_shift = shift_of(p.s.tile);
  p.cached = plan->cached;
  p.fresh = fresh_device;
  p.ring = plan->ring;
  p.cursor_in = plan->cursor_in;
  p.table = plan->table;
  p.lens = plan->lens;
  p.starts = plan->starts;
  p.positions = plan->positions;
  p.rows = plan->rows;
  p.slots = plan->slots;
  p.cursor = plan->cursor;
  p.status = plan->status;
  p.l = lists_of(p.s, plan->scratch);
  // a block for every 2,048 rows or 1,024 pages of a chunk of requests and one for
  // its work lists, but no more than run at once (one an SM: 152 blocks took 21 us
  // where 144 take 14)
  p.chunks = (int)ceil_div64(plan->requests, kPlanThreads);
  const int64_t room = sms / p.chunks;
  const auto share = [&](int64_t entries, int64_t each, int64_t most) {
    return (int)std::max<int64_t>(1, std::min(ceil_div64(entries, p.chunks * each), most));
  };
  p.page_blocks = share(p.s.page_cap, kPlanThreads, room / 8);
  p.row_blocks = share(plan->tokens, 2 * kPlanThreads, room - 2 * p.page_blocks - 1);
  plan_kernel<<<p.chunks * (p.row_blocks + 2 * p.page_blocks + 1), kPlanThreads, 0,
                static_cast<cudaStream_t>(stream)>>>(p);
  return launch_status("paged plan");
}

int grm_b200_paged_commit(const grm_b200_paged_plan* plan, int32_t* lens, int64_t* cursor,
                          void* stream) {
  int rc = check_sizes(plan);
  if (rc) return rc;
  if (!plan->grow || lens != plan->cached || cursor != plan->cursor_in) {
    set_thread_error("paged commit: a step that joins (grow != 0), and the plan's own cached and "
                     "cursor_in");
    return GRM_B200_EINVAL;
  }
  int sms = 0;
  if ((rc = check_plan(plan)) || (rc = current_sms(&sms))) return rc;
  Shape s;
  make_shape(*plan, sms, &s);
  const int threads = (int)std::min<int64_t>(ceil_div64(plan->requests, 32) * 32, kCommitThreads);
  commit_kernel<<<1, threads, 0, static_cast<cudaStream_t>(stream)>>>(
      plan->requests, plan->lens, plan->starts, lists_of(s, plan->scratch).header, plan->cursor,
      lens, cursor, plan->status);
  return launch_status("paged commit");
}

int grm_b200_paged_release(const int32_t* rows_device, int64_t count, int64_t requests,
                           int64_t table_width, int64_t pages, int page_tokens,
                           const int32_t* table, int32_t* lens, int32_t* ring, int64_t* cursor,
                           void* stream) {
  if (!rows_device || !table || !lens || !ring || !cursor || count < 0 || requests < 1 ||
      table_width < 1 || pages < 1 || !page_ok(page_tokens)) {
    set_thread_error("invalid paged release arguments");
    return GRM_B200_EINVAL;
  }
  if (count == 0) return 0;
  release_kernel<<<1, kReleaseThreads, 0, static_cast<cudaStream_t>(stream)>>>(
      rows_device, count, requests, table_width, pages, shift_of(page_tokens), table, lens, ring,
      cursor);
  return launch_status("paged release");
}

}  // extern "C"
