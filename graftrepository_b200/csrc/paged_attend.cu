// paged_attend.cu -- attention of a step's query rows over the 8-bit paged arena.
//
// For a query row q and the tokens t that it sees, with key codes a_t and value
// codes b_t (int8), key scale s_t and value scale u_t of t's page and head,
//   z_t = scale * s_t * (q . a_t),  w_t = exp(z_t),
//   out = sum_t w_t u_t b_t / sum_t w_t,  lse = log sum_t w_t.
// One pass keeps, for a row, a reference exponent m (base 2), the sum and the
// unscaled result.  The value scale is folded into the exponent: with
//   y_t = z_t * log2(e) + log2(u_t),  p_t = 2^(y_t - m),
// p_t u-weighted is what multiplies b_t, and the sum of weights is
// sum_t p_t / u_t, so p_t never exceeds 2^8 whatever the scales are (m trails the
// largest y seen by at most 8: it moves only when a y passes m + 8, so the
// accumulators are rarely rescaled), and fp16 holds 2^7 p_t.  The log-sum-exp is
// m ln 2 + log of that sum.
//
// The split kernel serves few query rows a kv head (decoding, a few proposed
// tokens): it is bound by the bytes of the codes, 2 * head_dim a token and kv
// head.  Every resident block ("worker") gets the same share of all tiles of
// all requests and heads, whatever their lengths; a segment (request, kv head,
// up to 16 query rows) that several workers share is joined by the one that
// finishes it last, in the order of the workers, so results do not depend on
// timing.
//
// A warp owns a quarter of a tile's tokens (32 of 128; 16 of 64 at head_dim
// 256), in a private ring of shared-memory stages that tensor-map copies fill
// and that it drains without a barrier of the block.  Products run on
// mma.m16n8k16 with fp16 operands and fp32 accumulators, tokens (or value dims)
// on the M side and the query rows on the 8-wide N side: four query heads of a
// group waste half of the columns instead of three quarters.  Codes become fp16
// exactly: byte b of code + 128 under the exponent of 1024 is the half 1024 + b,
// less 1152.  Queries are fp16: a bf16 row is first scaled by the power of two
// that brings its largest value into [2^14, 2^15), so only values 2^29 times
// smaller than the largest round.
//
// 64 requests of 200 to 16,384 tokens, one row x 4 each on 8 kv heads of head_dim
// 128 (515 MB of codes), take 97 us, 5.3 TB/s (head_dim 64 67 us, 256 190); one
// request of 250,007 tokens 100 us.  In its stride the kernel reads 7.5 TB/s (1.94 us a tile and block); the
// rest is the start (first data after 4.3 us of dependent loads) and the spread
// of the blocks, which end between 61 and 90 us for equal shares.  Measured and
// dropped: a last sixth of the tiles handed out in small shares as blocks finish
// (98 -> 105 us: starts and joins cost more than the spread); score products in
// int8, the codes as stored and the query in three digits (17 % fewer
// instructions, the same time).
#include <cuda.h>

#include <algorithm>
#include <type_traits>

#include "paged.cuh"

namespace grm_b200 {
namespace paged {

namespace {

constexpr int kWarps = 4;
constexpr int kThreads = kWarps * 32;

struct SplitParams {
  CUtensorMap k_map, v_map;  // codes as [pages * kv_heads][page_tokens][head_dim] bytes
  AttendParams a;
};

template <int D, int NT>
struct Layout {
  static constexpr int kTokens = split_tile(D) / kWarps;  // of a warp's stage
  static constexpr int kBlocks16 = kTokens / 16;
  static constexpr int kBlocks = split_blocks(D, NT * 8);
  static constexpr int kStages = D == 64 ? 4 : kBlocks == 3 || D == 256 ? 2 : 3;
  static constexpr int kSide = kTokens * D;       // codes
  static constexpr int kStage = 2 * kSide;
  static constexpr int kRow = D + 4;              // floats of a row in the merge buffer
  static constexpr int kRing = kWarps * kStages * kStage;
  static constexpr int kMerge = 2 * 8 * kRow * 4;
  static constexpr int kScales = kWarps * kStages * 2 * 8;
  static constexpr int kML = 2 * kWarps * NT * 8 * 4;
  // Sixteen rows: their fragments in shared memory, the same for every warp (in
  // registers beside the results of 16 rows they would spill).
  static constexpr bool kQShared = NT == 2;
  static constexpr int kQ = kQShared ? (D / 16) * NT * 32 * 8 + NT * 8 * 4 : 0;
  static constexpr int kSmem = 1024 + kRing + kMerge + kScales + kML + kQ;
};

__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldsm4t(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ uint32_t transpose8(uint32_t v) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}
__device__ __forceinline__ void mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                    uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
      "{%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void tma_load_3d(uint32_t dst, const CUtensorMap* map, int x, int y,
                                            int z, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(dst),
      "l"(map), "r"(x), "r"(y), "r"(z), "r"(smem_u32(bar))
      : "memory");
}

__device__ __forceinline__ void cp_async4(uint32_t dst, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory");
}
// One of the barrier's arrivals, once this thread's copies above have landed.
__device__ __forceinline__ void cp_async_arrive(uint64_t* bar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(bar))
               : "memory");
}

// Byte of 16-code chunk c of row r in a warp's stage of `rows` rows.  The
// copies' swizzle (128 bytes; 64 at head_dim 64) puts eight rows of one chunk
// into eight different bank groups, which ldmatrix reads together; head_dim 256
// is two blocks of 128 codes.
template <int D>
__device__ __forceinline__ uint32_t tile_byte(int rows, int r, int c) {
  if (D == 64) return (r >> 1) * 128 + ((((r & 1) << 2) | (c ^ ((r >> 1) & 3))) << 4);
  return (c >> 3) * rows * 128 + r * 128 + (((c & 7) ^ (r & 7)) << 4);
}

// A segment: up to block_rows query rows of a kv head of a request.
struct Segment {
  int first;  // its first unit
  int request, tiles, len, start, pairs, head, cached;
  int row0, row0_token, row0_head;  // its first row: token, and head of the group
};

// The share of one worker, walked segment by segment.
template <int TILE>
struct Walk {
  const AttendParams& p;
  int begin, end;  // units
  int u;           // first unit of the next segment to look at
  int r;
  Segment s;
  int t, t1;       // tiles of s that are the worker's, from t on

  __device__ __forceinline__ Walk(const AttendParams& pp, int b, int e, int request)
      : p(pp), begin(b), end(e), u(b), r(request), t(0), t1(0) {}

  // Step to the next segment that reaches into the share; false at its end.
  __device__ __forceinline__ bool next() {
    if (u >= end) return false;
    int base = __ldg(p.l.base + r), after = __ldg(p.l.base + r + 1);
    while (after <= u) {
      ++r;
      base = after;
      after = __ldg(p.l.base + r + 1);
    }
    s.request = r;
    s.start = __ldg(p.starts + r);
    const int n = __ldg(p.starts + r + 1) - s.start;
    s.len = __ldg(p.lens + r);
    s.cached = s.len - n;
    s.pairs = n * p.group;
    s.tiles = (s.len + TILE - 1) / TILE;
    const int blocks = (s.pairs + p.block_rows - 1) / p.block_rows;
    const int i = (u - base) / (s.tiles + 1);
    s.first = base + i * (s.tiles + 1);
    s.head = i / blocks;
    s.row0 = (i - s.head * blocks) * p.block_rows;
    s.row0_token = s.row0 / p.group;
    s.row0_head = s.row0 - s.row0_token * p.group;
    u = s.first + s.tiles + 1;
    t = max(begin - s.first - 1, 0);
    t1 = min(end - s.first - 1, s.tiles);
    return true;
  }
};

// Row `row` of a segment whose n partial results workers wa, wa + 1, ... left:
// summed in that order by a warp, and written as packed row `out_row`.  A call
// of its own, so that its registers are not the tile loop's.
template <typename T, int D, int ROWS>
__device__ __noinline__ void join_row(const AttendParams& p, int wa, int n, int row,
                                      int64_t out_row) {
  constexpr int kDims = D / 32, kAhead = 8, kSlot = split_slot(D, ROWS);
  const int lane = threadIdx.x & 31;
  auto part = [&](int i) {  // the first left the segment unfinished, the others took it up
    return p.l.part + (2 * (wa + i) + (i == 0 ? 1 : 0)) * (int64_t)kSlot;
  };
  auto sums = [&](int i) {  // (reference exponent, sum)
    return i < n ? __ldcg(reinterpret_cast<const float2*>(part(i) + ROWS * D + 2 * row))
                 : make_float2(-INFINITY, 0.0f);
  };
  float top = -INFINITY;
  for (int i = lane; i < n; i += 32) top = fmaxf(top, sums(i).x);
#pragma unroll
  for (int i = 16; i >= 1; i >>= 1) top = fmaxf(top, __shfl_xor_sync(kFull, top, i));
  float sum = 0.0f, acc[kDims] = {};
  for (int i0 = 0; i0 < n; i0 += 32) {
    const float2 ml = sums(i0 + lane);
    const float a = ml.x == top ? 1.0f : ex2(ml.x - top);
    float l = ml.y == 0.0f ? 0.0f : ml.y * a;
#pragma unroll
    for (int i = 16; i >= 1; i >>= 1) l += __shfl_xor_sync(kFull, l, i);
    sum += l;
    for (int i1 = 0; i1 < 32 && i0 + i1 < n; i1 += kAhead) {
      float2 v[kAhead][kDims / 2];  // lane: D / 32 neighbouring dims
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        const float* src = part(min(i0 + i1 + i, n - 1)) + row * D + kDims * lane;
#pragma unroll
        for (int d = 0; d < kDims / 2; ++d)
          v[i][d] = __ldcg(reinterpret_cast<const float2*>(src) + d);
      }
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        const float w = __shfl_sync(kFull, a, i1 + i);
        if (i0 + i1 + i < n) {
#pragma unroll
          for (int d = 0; d < kDims / 2; ++d) {
            acc[2 * d] = fmaf(v[i][d].x, w, acc[2 * d]);
            acc[2 * d + 1] = fmaf(v[i][d].y, w, acc[2 * d + 1]);
          }
        }
      }
    }
  }
  const float inv = sum == 0.0f ? 0.0f : kUnlift / sum;
#pragma unroll
  for (int d = 0; d < kDims / 2; ++d)
    reinterpret_cast<uint32_t*>(p.out + out_row * D + kDims * lane)[d] =
        pack_out<T>(acc[2 * d] * inv, acc[2 * d + 1] * inv);
  if (p.lse && lane == 0)
    p.lse[out_row] = sum == 0.0f ? -INFINITY : (top + log2f(sum)) * 0.693147180559945309f;
}

// Prompt tiles that the prompt kernel left in parts: a warp takes eight rows and 16
// dims, four a lane, and adds the parts up in their order, eight loads in flight.
// As the last part's own work, by one block, it took 42 us for 256 rows of head_dim
// 128 in 8 parts; over all blocks it takes 3.
template <typename T, int D>
__device__ __noinline__ void join_prompts(const AttendParams& p, int entries) {
  constexpr int kRows = prompt_rows_of(D), kItems = kRows / 8 * (D / 16), kAhead = 8;
  const int lane = threadIdx.x & 31, warps = gridDim.x * kWarps;
  const int heads = p.kv_heads * p.group, items = p.kv_heads * kItems;
  const int64_t step = (int64_t)p.kv_heads * prompt_slot(D);
  int next = blockIdx.x * kWarps + (threadIdx.x >> 5);
  for (int e0 = 0; e0 < entries; e0 += 32) {
    const int4 mine = p.l.qtiles[min(e0 + lane, entries - 1)];
    const int my_parts = prompt_tile<D>(p, mine).parts;
    unsigned todo =
        __ballot_sync(kFull, e0 + lane < entries && (mine.z & 255) == 0 && my_parts > 1);
    for (; todo; todo &= todo - 1) {
      const int4 e = p.l.qtiles[e0 + __ffs(todo) - 1];
      const PromptTile t = prompt_tile<D>(p, e);
      for (; next < items; next += warps) {
        const int h = next / kItems, x = next % kItems;
        const int r = x / (D / 16) * 8 + (lane & 7), c = x % (D / 16) * 4 + (lane >> 3);
        const int q = r / 128, in = r % 128;
        if (in >= (q == 0 ? t.toks[0] : t.toks[1]) * p.group) continue;
        const float* part = p.l.qpart + ((int64_t)e.w * p.kv_heads + h) * prompt_slot(D);
        const float4* src = reinterpret_cast<const float4*>(part) + c * kRows + r;
        const float2* sums = reinterpret_cast<const float2*>(part + kRows * D) + r;
        float top = -INFINITY, sum = 0.0f;
        float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        for (int i0 = 0; i0 < t.parts; i0 += kAhead) {
          float2 ml[kAhead];
          float4 v[kAhead];
#pragma unroll
          for (int i = 0; i < kAhead; ++i) {
            const int64_t at = min(i0 + i, t.parts - 1) * step;
            ml[i] = __ldcg(sums + at / 2);
            v[i] = __ldcg(src + at / 4);
          }
          float high = top;
#pragma unroll
          for (int i = 0; i < kAhead; ++i) high = fmaxf(high, ml[i].x);
          const float a = top == high ? 1.0f : ex2(top - high);
          top = high;
          sum *= a;
          acc = make_float4(acc.x * a, acc.y * a, acc.z * a, acc.w * a);
#pragma unroll
          for (int i = 0; i < kAhead; ++i) {
            if (i0 + i >= t.parts) break;
            const float w = ml[i].x == top ? 1.0f : ex2(ml[i].x - top);
            sum += ml[i].y == 0.0f ? 0.0f : ml[i].y * w;
            acc.x = fmaf(v[i].x, w, acc.x);
            acc.y = fmaf(v[i].y, w, acc.y);
            acc.z = fmaf(v[i].z, w, acc.z);
            acc.w = fmaf(v[i].w, w, acc.w);
          }
        }
        const int64_t row = (int64_t)(t.start + t.tok0 + q * t.per + in / p.group) * heads +
                            h * p.group + in % p.group;
        const float inv = sum == 0.0f ? 0.0f : kUnlift / sum;
        reinterpret_cast<uint2*>(p.out + row * D)[c] =
            make_uint2(pack_out<T>(acc.x * inv, acc.y * inv),
                       pack_out<T>(acc.z * inv, acc.w * inv));
        if (p.lse && c == 0)
          p.lse[row] = sum == 0.0f ? -INFINITY : (top + log2f(sum)) * 0.693147180559945309f;
      }
      next -= items;
    }
  }
}

template <typename T, int D, int NT>
__global__ void __launch_bounds__(kThreads, (Layout<D, NT>::kBlocks))
    split_kernel(const __grid_constant__ SplitParams sp) {
  using LY = Layout<D, NT>;
  constexpr int kChunks = D / 16;
  constexpr int kTokens = LY::kTokens, kB = LY::kBlocks16;
  constexpr int kSums = NT * 8 * D, kSlot = split_slot(D, NT * 8);  // of a partial result
  const AttendParams& p = sp.a;
  extern __shared__ unsigned char raw_smem[];
  unsigned char* const smem = raw_smem + ((1024u - (smem_u32(raw_smem) & 1023u)) & 1023u);
  float* const merge = reinterpret_cast<float*>(smem + LY::kRing);
  float2* const scales = reinterpret_cast<float2*>(smem + LY::kRing + LY::kMerge);
  float* const sm_m = reinterpret_cast<float*>(smem + LY::kRing + LY::kMerge + LY::kScales);
  float* const sm_l = sm_m + kWarps * NT * 8;
  uint2* const sm_q = reinterpret_cast<uint2*>(sm_l + kWarps * NT * 8);
  float* const sm_unscale = reinterpret_cast<float*>(sm_q + kChunks * NT * 32);
  __shared__ __align__(8) uint64_t bars[kWarps][LY::kStages];
  __shared__ int sm_last, sm_fail;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, t4 = lane & 3;
  const int heads = p.kv_heads * p.group;
  const Header hd = *p.l.header;
  const int w = blockIdx.x;
  const int request0 = p.l.start[w];

  // rows past the step's last one
  for (int64_t i = hd.rows + (int64_t)blockIdx.x; i < p.tokens; i += gridDim.x) {
    for (int x = threadIdx.x; x < heads * D / 2; x += kThreads)
      reinterpret_cast<uint32_t*>(p.out + i * heads * D)[x] = 0;
    if (p.lse)
      for (int x = threadIdx.x; x < heads; x += kThreads) p.lse[i * heads + x] = -INFINITY;
  }
  if (hd.joins > 0) join_prompts<T, D>(p, hd.joins);
  if (w >= hd.workers) return;
  const int begin = worker_first(w, hd), end = worker_first(w + 1, hd);
  Walk<LY::kTokens * kWarps> walk(p, begin, end, request0);
  bool more;

  // ---- queries of a segment: column g of the B operand, dims 16c + 4 t4 .. + 3
  uint2 raw[LY::kQShared ? 1 : NT][kChunks];
  // packed row and head of row `x` of a segment (a block's rows are few, so the
  // division by the group is a multiplication)
  auto pair_of = [&](const Segment& s, int x, int* token, int* head) {
    const int j = s.row0_head + x;
    const int q = p.group == 1 ? j : (int)__umulhi(j, p.group_inv);
    *token = s.row0_token + q;
    *head = s.head * p.group + j - q * p.group;
  };
  auto fetch_queries = [&](const Segment& s) {
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const bool there = s.row0 + nt * 8 + g < s.pairs;
      int token, head;
      pair_of(s, nt * 8 + g, &token, &head);
      const uint16_t* qp = p.q + (int64_t)(s.start + token) * p.q_row + (int64_t)head * p.q_head +
                           t4 * 4;
#pragma unroll
      for (int c = 0; c < kChunks; ++c)
        raw[nt][c] = there ? __ldg(reinterpret_cast<const uint2*>(qp + c * 16))
                           : make_uint2(0, 0);
    }
  };
  // The same to shared memory, a warp the four rows 4 warp .. and eight lanes a row.
  auto share_queries = [&](const Segment& s) {
    const int x = warp * 4 + (lane >> 3), d0 = (lane & 7) * (D / 8);
    const bool there = s.row0 + x < s.pairs;
    int token, head;
    pair_of(s, x, &token, &head);
    const uint4* qp = reinterpret_cast<const uint4*>(
        p.q + (int64_t)(s.start + token) * p.q_row + (int64_t)head * p.q_head + d0);
    uint4 v[D / 64];
    unsigned m = 0;
#pragma unroll
    for (int i = 0; i < D / 64; ++i) {
      v[i] = there ? __ldg(qp + i) : make_uint4(0, 0, 0, 0);
      m = __vmaxu2(m, __vmaxu2(v[i].x & 0x7FFF7FFFu, v[i].y & 0x7FFF7FFFu));
      m = __vmaxu2(m, __vmaxu2(v[i].z & 0x7FFF7FFFu, v[i].w & 0x7FFF7FFFu));
    }
    float up = 1.0f, unscale = 1.0f;
    if constexpr (!std::is_same<T, __half>::value) {
      m = max(m & 0xFFFFu, m >> 16);
#pragma unroll
      for (int i = 1; i <= 4; i <<= 1) m = max(m, __shfl_xor_sync(kFull, m, i));
      row_scale(m, &up, &unscale);
#pragma unroll
      for (int i = 0; i < D / 64; ++i)
        v[i] = make_uint4(scale_pair(v[i].x, up), scale_pair(v[i].y, up), scale_pair(v[i].z, up),
                          scale_pair(v[i].w, up));
    }
    if ((lane & 7) == 0) sm_unscale[x] = unscale;
#pragma unroll
    for (int i = 0; i < D / 64; ++i) {
      const int d = d0 + 8 * i;
      uint2* to = sm_q + (d / 16 * NT + x / 8) * 32 + (x % 8) * 4 + d % 16 / 4;
      to[0] = make_uint2(v[i].x, v[i].y);
      to[1] = make_uint2(v[i].z, v[i].w);
    }
    __syncthreads();
  };
  auto next_segment = [&]() {
    more = walk.next();
    if (!LY::kQShared && more) fetch_queries(walk.s);
  };
  next_segment();

  if (lane == 0) {
    for (int i = 0; i < LY::kStages; ++i) mbar_init(&bars[warp][i], 2);
    mbar_fence_init();
  }
  if (threadIdx.x == 0) sm_fail = 0;
  __syncthreads();

  // ---- the loader: this warp's tokens of a tile, one stage at a time
  const uint32_t ring = smem_u32(smem) + warp * LY::kStages * LY::kStage;
  const float2* const ring_scales = scales + warp * LY::kStages * 2;
  Walk<LY::kTokens * kWarps> load = walk;
  int issued = 0, used = 0;        // stages
  // lane i: page ids_base + i of the request, and the page 32 further on
  int ids = 0, ids_ahead = 0, ids_base = 0, ids_request = -1;
  auto issue = [&]() {
    int tok = 0;
    for (;;) {  // the next tile of the share with tokens for this warp
      while (load.t >= load.t1)
        if (!load.next()) return;
      tok = load.t++ * kTokens * kWarps + warp * kTokens;
      if (tok < load.s.len) break;
    }
    const Segment& s = load.s;
    const int j = tok >> p.page_shift;
    if (s.request != ids_request || j >= ids_base + 32 || j < ids_base) {
      const int last = (s.len - 1) >> p.page_shift;
      const int32_t* row = p.table + s.request * p.width;
      const bool follows = s.request == ids_request && j == ids_base + 32;
      ids = follows ? ids_ahead : __ldg(row + min(j + lane, last));
      ids = min(max(ids, 0), (int)p.pages - 1);
      ids_ahead = __ldg(row + min(j + 32 + lane, last));
      ids_base = j;
      ids_request = s.request;
    }
    const int stage = issued % LY::kStages;
    ++issued;
    const int per = 1 << p.page_shift;
    const int rows = min(per, kTokens);  // of one copy
    uint64_t* bar = &bars[warp][stage];
    const int page0 = __shfl_sync(kFull, ids, j - ids_base);
    const int page1 = __shfl_sync(kFull, ids, min(j + 1 - ids_base, 31));
    if (lane == 0) {
      // a second copy where pages are smaller than the stage, unless it would
      // begin past the request's tokens (what then lies there is not read)
      const bool both = rows < kTokens && tok + rows < s.len;
      mbar_arrive_expect_tx(bar, (both ? 2 : 1) * 2 * rows * D);
      const uint32_t to = ring + stage * LY::kStage;
      const int y = tok & (per - 1);
      const int z0 = page0 * p.kv_heads + s.head;
      const int z1 = both ? page1 * p.kv_heads + s.head : z0;
#pragma unroll
      for (int x = 0; x < D; x += 128) {
        const uint32_t at = to + (x / 128) * kTokens * 128;
        tma_load_3d(at, &sp.k_map, x, y, z0, bar);
        tma_load_3d(at + LY::kSide, &sp.v_map, x, y, z0, bar);
        if (both) {
          const uint32_t at1 = at + rows * (D < 128 ? D : 128);
          tma_load_3d(at1, &sp.k_map, x, 0, z1, bar);
          tma_load_3d(at1 + LY::kSide, &sp.v_map, x, 0, z1, bar);
        }
      }
#pragma unroll
      for (int b = 0; b < kB; ++b) {  // scales of 16 tokens
        const uint32_t f = smem_u32(ring_scales + stage * 2 + b);
        cp_async4(f, p.ks + (b ? z1 : z0));
        cp_async4(f + 4, p.vs + (b ? z1 : z0));
      }
      cp_async_arrive(bar);
    }
  };
#pragma unroll 1
  for (int i = 0; i < LY::kStages; ++i) issue();

  // ldmatrix source of this lane: rows 0-7 / 8-15 of an even chunk, then of an odd one
  uint32_t lm[kChunks / 2];
#pragma unroll
  for (int c = 0; c < kChunks; c += 2)
    lm[c / 2] = tile_byte<D>(kTokens, lane & 15, c + (lane >> 4));
  constexpr uint32_t kNext16 = 16 * (D < 128 ? D : 128);  // bytes from 16 rows to the next

  bool failed = false;
  for (; more; next_segment()) {
    const Segment s = walk.s;
    const int rows = min(s.pairs - s.row0, NT * 8);
    auto out_row = [&](int x) {  // of row x of the segment
      int token, head;
      pair_of(s, x, &token, &head);
      return (int64_t)(s.start + token) * heads + head;
    };
    if (s.tiles == 0) {  // nothing cached: empty rows (the segment is its one unit)
      for (int x = threadIdx.x; x < rows * (D / 2); x += kThreads) {
        const int64_t row = out_row(x / (D / 2));
        reinterpret_cast<uint32_t*>(p.out + row * D)[x % (D / 2)] = 0;
        if (p.lse && x % (D / 2) == 0) p.lse[row] = -INFINITY;
      }
      continue;
    }
    if (walk.t >= walk.t1) continue;  // only its start is this worker's

    uint32_t qf[LY::kQShared ? 1 : kChunks][NT][2];
    float kq[NT][2];
    int lim[NT][2];
    if constexpr (LY::kQShared) share_queries(s);
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      float up = 1.0f, unscale = 1.0f;
      if constexpr (!LY::kQShared && !std::is_same<T, __half>::value) {
        unsigned m = 0;
#pragma unroll
        for (int c = 0; c < kChunks; ++c)
          m = __vmaxu2(m, __vmaxu2(raw[nt][c].x & 0x7FFF7FFFu, raw[nt][c].y & 0x7FFF7FFFu));
        m = max(m & 0xFFFFu, m >> 16);
        m = max(m, __shfl_xor_sync(kFull, m, 1));
        m = max(m, __shfl_xor_sync(kFull, m, 2));
        row_scale(m, &up, &unscale);
      }
#pragma unroll
      for (int c = 0; c < (LY::kQShared ? 0 : kChunks); ++c) {
        uint2 f = raw[nt][c];
        if constexpr (!std::is_same<T, __half>::value)
          f = make_uint2(scale_pair(f.x, up), scale_pair(f.y, up));
        qf[c][nt][0] = f.x;
        qf[c][nt][1] = f.y;
      }
      // columns 2 t4 and 2 t4 + 1 of the scores
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        kq[nt][x] = p.scale_log2 * (LY::kQShared ? sm_unscale[nt * 8 + 2 * t4 + x]
                                                 : __shfl_sync(kFull, unscale, (2 * t4 + x) * 4));
        int token, head;
        pair_of(s, nt * 8 + 2 * t4 + x, &token, &head);
        lim[nt][x] = p.causal && s.row0 + nt * 8 + 2 * t4 + x < s.pairs ? s.cached + token + 1
                                                                       : s.len;
      }
    }
    const int all_see = p.causal ? s.cached + s.row0_token + 1 : s.len;

    float o[kChunks][NT][4];
    float m[NT][2], l[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      m[nt][0] = m[nt][1] = -INFINITY;
      l[nt][0] = l[nt][1] = 0.0f;
#pragma unroll
      for (int c = 0; c < kChunks; ++c)
#pragma unroll
        for (int x = 0; x < 4; ++x) o[c][nt][x] = 0.0f;
    }

    // ---- this worker's tiles
#pragma unroll 1
    for (int t = walk.t; t < walk.t1; ++t) {
      const int tok = t * kTokens * kWarps + warp * kTokens;
      if (tok >= s.len) break;  // the last tile, and none of it is this warp's
      const int stage = used % LY::kStages;
      if (!failed)
        failed = !__all_sync(
            kFull, mbar_wait(&bars[warp][stage], (used / LY::kStages) & 1, p.probes));
      if (failed) break;  // `used` stays at the first stage that was not seen to land
      ++used;
      __syncwarp();
      const uint32_t kb = ring + stage * LY::kStage;
      // scores of kB x 16 tokens x 8 NT rows, two chains of products at least
      constexpr int kChains = kB * NT == 1 ? 2 : 1;
      float sum[kChains][kB][NT][4];
#pragma unroll
      for (int i = 0; i < kChains; ++i)
#pragma unroll
        for (int b = 0; b < kB; ++b)
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int x = 0; x < 4; ++x) sum[i][b][nt][x] = 0.0f;
      // (fragments one step ahead of their use)
      uint32_t fr[2][kB][4];
#pragma unroll
      for (int b = 0; b < kB; ++b) ldsm4(fr[0][b], kb + lm[0] + b * kNext16);
#pragma unroll
      for (int c = 0; c < kChunks; c += 2) {
#pragma unroll
        for (int b = 0; b < kB; ++b) {
          if (c + 2 < kChunks)
            ldsm4(fr[(c / 2 + 1) % 2][b], kb + lm[(c + 2) / 2 % (kChunks / 2)] + b * kNext16);
          else  // the first value fragments
            ldsm4t(fr[(c / 2 + 1) % 2][b], kb + lm[0] + (LY::kSide + b * kNext16));
        }
        uint2 qs[2][NT];
#pragma unroll
        for (int x = 0; x < 2; ++x)
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            if constexpr (LY::kQShared) qs[x][nt] = sm_q[((c + x) * NT + nt) * 32 + lane];
            else qs[x][nt] = make_uint2(qf[c + x][nt][0], qf[c + x][nt][1]);
          }
#pragma unroll
        for (int b = 0; b < kB; ++b) {
          const uint32_t* r = fr[(c / 2) % 2][b];
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            const uint32_t lo = r[2 * x] ^ 0x80808080u, hi = r[2 * x + 1] ^ 0x80808080u;
            const uint32_t a0 = halves(lo, 0x4140), a2 = halves(lo, 0x4342);
            const uint32_t a1 = halves(hi, 0x4140), a3 = halves(hi, 0x4342);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
              mma(sum[x % kChains][b][nt], a0, a1, a2, a3, qs[x][nt].x, qs[x][nt].y);
          }
        }
      }
      bool moves = false;
      float sc[kB][NT][4], inv[kB];
#pragma unroll
      for (int b = 0; b < kB; ++b) {
        const float2 f = ring_scales[stage * 2 + b];
        float log2_u;
        value_scale(f.y, &log2_u, &inv[b]);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            const float z = sum[0][b][nt][x] + (kChains == 2 ? sum[kChains - 1][b][nt][x] : 0.0f);
            sc[b][nt][x] = fmaf(z, kq[nt][x & 1] * f.x, log2_u);
          }
        }
      }
      if (tok + kTokens > all_see) {
#pragma unroll
        for (int b = 0; b < kB; ++b)
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int x = 0; x < 4; ++x)
              if (tok + 16 * b + g + (x >> 1) * 8 >= min(lim[nt][x & 1], s.len))
                sc[b][nt][x] = -INFINITY;
      }
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          float top = fmaxf(sc[0][nt][x], sc[0][nt][x + 2]);
          if (kB == 2) top = fmaxf(top, fmaxf(sc[kB - 1][nt][x], sc[kB - 1][nt][x + 2]));
          moves |= top > m[nt][x] + kLazy;
        }
      if (__any_sync(kFull, moves)) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            float top = fmaxf(sc[0][nt][x], sc[0][nt][x + 2]);
            if (kB == 2) top = fmaxf(top, fmaxf(sc[kB - 1][nt][x], sc[kB - 1][nt][x + 2]));
#pragma unroll
            for (int i = 4; i <= 16; i <<= 1) top = fmaxf(top, __shfl_xor_sync(kFull, top, i));
            // each row by its own scores, so that no row's rounding hangs on another's
            top = top > m[nt][x] + kLazy ? reference_of(top) : m[nt][x];
            const float a = top == m[nt][x] ? 1.0f : ex2(m[nt][x] - top);
            m[nt][x] = top;
            l[nt][x] *= a;
#pragma unroll
            for (int c = 0; c < kChunks; ++c) {
              o[c][nt][x] *= a;
              o[c][nt][x + 2] *= a;
            }
          }
      }
      uint32_t bp[kB][NT][2];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        float ref[2];
#pragma unroll
        for (int x = 0; x < 2; ++x) ref[x] = m[nt][x] == -INFINITY ? 0.0f : m[nt][x] - kLift;
#pragma unroll
        for (int b = 0; b < kB; ++b) {
          float pr[4];
#pragma unroll
          for (int x = 0; x < 4; ++x) pr[x] = ex2(sc[b][nt][x] - ref[x & 1]);
#pragma unroll
          for (int x = 0; x < 2; ++x) l[nt][x] = fmaf(pr[x] + pr[x + 2], inv[b], l[nt][x]);
          bp[b][nt][0] = transpose8(pack_half2(pr[0], pr[1]));
          bp[b][nt][1] = transpose8(pack_half2(pr[2], pr[3]));
        }
      }
      // result dims 16c + 2g (rows g) and 16c + 2g + 1 (rows g + 8)
#pragma unroll
      for (int c = 0; c < kChunks; c += 2) {
        constexpr int kFirst = kChunks / 2;  // the buffer that the loop above left them in
        if (c + 2 < kChunks) {
#pragma unroll
          for (int b = 0; b < kB; ++b)
            ldsm4t(fr[(c / 2 + kFirst + 1) % 2][b],
                   kb + lm[(c + 2) / 2 % (kChunks / 2)] + (LY::kSide + b * kNext16));
        }
#pragma unroll
        for (int b = 0; b < kB; ++b) {
          const uint32_t* r = fr[(c / 2 + kFirst) % 2][b];
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            const uint32_t lo = r[2 * x] ^ 0x80808080u, hi = r[2 * x + 1] ^ 0x80808080u;
            const uint32_t a0 = halves(lo, 0x4240), a1 = halves(lo, 0x4341);
            const uint32_t a2 = halves(hi, 0x4240), a3 = halves(hi, 0x4341);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
              mma(o[c + x][nt], a0, a1, a2, a3, bp[b][nt][0], bp[b][nt][1]);
          }
        }
      }
      __syncwarp();  // the stage is read: its place is free
      issue();
    }
    if (failed) {  // tokens are missing: no number for these rows
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) l[nt][0] = l[nt][1] = __int_as_float(0x7FC00000);
    }

    // ---- join the four warps
    float lt[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int x = 0; x < 2; ++x) {
#pragma unroll
        for (int i = 4; i <= 16; i <<= 1) l[nt][x] += __shfl_xor_sync(kFull, l[nt][x], i);
        if (g == 0) {
          sm_m[warp * NT * 8 + nt * 8 + 2 * t4 + x] = m[nt][x];
          sm_l[warp * NT * 8 + nt * 8 + 2 * t4 + x] = l[nt][x];
        }
      }
    __syncthreads();
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const int col = nt * 8 + 2 * t4 + x;
        float top = -INFINITY;
#pragma unroll
        for (int i = 0; i < kWarps; ++i) top = fmaxf(top, sm_m[i * NT * 8 + col]);
        lt[nt][x] = 0.0f;
#pragma unroll
        for (int i = 0; i < kWarps; ++i) {
          const float mi = sm_m[i * NT * 8 + col];
          if (mi != -INFINITY || sm_l[i * NT * 8 + col] != 0.0f)
            lt[nt][x] += sm_l[i * NT * 8 + col] * (mi == top ? 1.0f : ex2(mi - top));
        }
        const float a = m[nt][x] == top ? 1.0f : ex2(m[nt][x] - top);
        m[nt][x] = top;
#pragma unroll
        for (int c = 0; c < kChunks; ++c) {
          o[c][nt][x] *= a;
          o[c][nt][x + 2] *= a;
        }
      }
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {  // 8 rows at a time: 2, 3 to 0, 1, then 1 to 0
      auto at = [&](int buf, int c, int x) {
        return reinterpret_cast<float2*>(merge + (buf * 8 + 2 * t4 + x) * LY::kRow + 16 * c +
                                         2 * g);
      };
      auto put = [&](int buf) {
#pragma unroll
        for (int c = 0; c < kChunks; ++c)
#pragma unroll
          for (int x = 0; x < 2; ++x) *at(buf, c, x) = make_float2(o[c][nt][x], o[c][nt][x + 2]);
      };
      auto add = [&](int buf) {
#pragma unroll
        for (int c = 0; c < kChunks; ++c)
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            const float2 v = *at(buf, c, x);
            o[c][nt][x] += v.x;
            o[c][nt][x + 2] += v.y;
          }
      };
      if (warp >= 2) put(warp - 2);
      __syncthreads();
      if (warp < 2) add(warp);
      __syncthreads();
      if (warp == 1) put(0);
      __syncthreads();
      if (warp == 0) add(0);
      if (nt + 1 < NT) __syncthreads();
    }

    // ---- alone on the segment: done
    const int wa = worker_of(s.first + 1, hd), wb = worker_of(s.first + s.tiles, hd);
    if (wa == wb) {
      if (warp == 0) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            if (s.row0 + nt * 8 + 2 * t4 + x < s.pairs) {
              const int64_t row = out_row(nt * 8 + 2 * t4 + x);
              const float sum = lt[nt][x];
              const float inv = sum == 0.0f ? 0.0f : kUnlift / sum;
#pragma unroll
              for (int c = 0; c < kChunks; ++c)
                *reinterpret_cast<uint32_t*>(p.out + row * D + 16 * c + 2 * g) =
                    pack_out<T>(o[c][nt][x] * inv, o[c][nt][x + 2] * inv);
              if (p.lse && g == 0)
                p.lse[row] = sum == 0.0f ? -INFINITY
                                         : (m[nt][x] + log2f(sum)) * 0.693147180559945309f;
            }
          }
      }
      continue;
    }

    // ---- shared: leave the partial result; the last worker joins them
    if (warp == 0) {
      float* slot = p.l.part + (2 * w + (w == wa ? 1 : 0)) * (int64_t)kSlot;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          const int row = nt * 8 + 2 * t4 + x;
#pragma unroll
          for (int c = 0; c < kChunks; ++c)
            *reinterpret_cast<float2*>(slot + row * D + 16 * c + 2 * g) =
                make_float2(o[c][nt][x], o[c][nt][x + 2]);
          if (g == 0)
            *reinterpret_cast<float2*>(slot + kSums + 2 * row) = make_float2(m[nt][x], lt[nt][x]);
        }
      __syncwarp();
      if (lane == 0) {  // releases the warp's stores, acquires the other workers'
        unsigned arrived;
        asm volatile("atom.acq_rel.gpu.global.add.u32 %0, [%1], 1;"
                     : "=r"(arrived)
                     : "l"(p.l.count + wa)
                     : "memory");
        const int last = arrived + 1 == (unsigned)(wb - wa + 1);
        if (last) p.l.count[wa] = 0;  // for the next call
        sm_last = last;
      }
    }
    __syncthreads();
    if (sm_last) {
#pragma unroll 1
      for (int row = warp; row < rows; row += kWarps)  // a warp takes a row
        join_row<T, D, NT * 8>(p, wa, wb - wa + 1, row, out_row(row));
    }
  }
  if (failed) {  // copies still in flight end before the block does
    if (lane == 0) sm_fail = 1;
    for (; used < issued; ++used)
      mbar_wait(&bars[warp][used % LY::kStages], (used / LY::kStages) & 1, kProbes);
  }
  __syncthreads();
  if (threadIdx.x == 0 && sm_fail) atomicOr(p.status, GRM_B200_PLAN_WAIT);
}

template <typename T, int D, int NT>
int launch_split(const SplitParams& p, int workers, cudaStream_t st) {
  using LY = Layout<D, NT>;
  static_assert((LY::kSmem + 2048) * LY::kBlocks <= 228 * 1024, "blocks of an SM");
  auto kernel = split_kernel<T, D, NT>;
  static std::atomic<uint64_t> done{0};
  const int rc = allow_shared(reinterpret_cast<const void*>(kernel), LY::kSmem, &done);
  if (rc) return rc;
  kernel<<<workers, kThreads, LY::kSmem, st>>>(p);
  return launch_status("paged attend");
}

template <typename T>
int launch_split_any(int dim, int block_rows, const SplitParams& p, int workers,
                     cudaStream_t st) {
  if (dim == 64)
    return block_rows == 8 ? launch_split<T, 64, 1>(p, workers, st)
                           : launch_split<T, 64, 2>(p, workers, st);
  if (dim == 128)
    return block_rows == 8 ? launch_split<T, 128, 1>(p, workers, st)
                           : launch_split<T, 128, 2>(p, workers, st);
  return block_rows == 8 ? launch_split<T, 256, 1>(p, workers, st)
                         : launch_split<T, 256, 2>(p, workers, st);
}

// cuTensorMapEncodeTiled from the driver, looked up once (no libcuda link).
using EncodeTiled = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*,
                                 const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                                 const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                 CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
EncodeTiled encode_tiled() {
  static const EncodeTiled fn = [] {
    void* f = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &f, 12000, cudaEnableDefault,
                                         &q) != cudaSuccess ||
        q != cudaDriverEntryPointSuccess)
      f = nullptr;
    return reinterpret_cast<EncodeTiled>(f);
  }();
  return fn;
}

// The codes of one side as rows of bytes: a box is the rows that one copy brings
// (a page, at most a warp's stage) by 128 bytes.
int make_map(CUtensorMap* map, const int8_t* codes, const grm_b200_paged_arena& a) {
  const EncodeTiled encode = encode_tiled();
  const int stage = split_tile(a.head_dim) / kWarps;
  const cuuint64_t dims[3] = {(cuuint64_t)a.head_dim, (cuuint64_t)a.page_tokens,
                              (cuuint64_t)a.pages * a.kv_heads};
  const cuuint64_t strides[2] = {(cuuint64_t)a.head_dim,
                                 (cuuint64_t)a.head_dim * a.page_tokens};
  const cuuint32_t box[3] = {(cuuint32_t)std::min(a.head_dim, 128),
                             (cuuint32_t)std::min(a.page_tokens, stage), 1};
  const cuuint32_t step[3] = {1, 1, 1};
  if (!encode ||
      encode(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, const_cast<int8_t*>(codes), dims, strides, box,
             step, CU_TENSOR_MAP_INTERLEAVE_NONE,
             a.head_dim == 64 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_128B,
             CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
             CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS) {
    set_thread_error("paged attend: no tensor map of the arena (pages %lld, kv_heads %d)",
                     (long long)a.pages, a.kv_heads);
    return GRM_B200_EINVAL;
  }
  return 0;
}

}  // namespace
}  // namespace paged
}  // namespace grm_b200

using namespace grm_b200;
using namespace grm_b200::paged;

extern "C" {

int grm_b200_paged_attend(const grm_b200_paged_plan* plan, const grm_b200_paged_arena* arena,
                          const void* q_device, int dtype, int64_t q_row_stride,
                          int64_t q_head_stride, float softmax_scale, int causal,
                          void* out_device, float* lse_device, void* stream) {
  int rc;
  if ((rc = check_plan(plan)) || (rc = check_arena(arena)) || (rc = check_match(plan, arena)) ||
      (rc = check_rows("paged attend", q_device, dtype, q_row_stride, q_head_stride)))
    return rc;
  if (!out_device || (reinterpret_cast<uintptr_t>(out_device) & 15)) {
    set_thread_error("paged attend: out must be 16-byte aligned device memory");
    return GRM_B200_EINVAL;
  }
  if (causal && !plan->grow) {
    set_thread_error("paged attend: rows that do not join the arena (grow = 0) have no position "
                     "in it; attend with causal = 0");
    return GRM_B200_EINVAL;
  }
  if (!(softmax_scale > 0.0f) || !(softmax_scale < INFINITY)) {
    set_thread_error("paged attend: softmax_scale %g must be positive and finite",
                     (double)softmax_scale);
    return GRM_B200_EINVAL;
  }
  int sms = 0;
  if ((rc = current_sms(&sms))) return rc;
  Shape s;
  make_shape(*plan, sms, &s);
  SplitParams sp;
  if ((rc = make_map(&sp.k_map, arena->k_codes, *arena)) ||
      (rc = make_map(&sp.v_map, arena->v_codes, *arena)))
    return rc;
  AttendParams& p = sp.a;
  p.l = lists_of(s, plan->scratch);
  p.table = plan->table;
  p.lens = plan->lens;
  p.starts = plan->starts;
  p.width = plan->table_width;
  p.tokens = plan->tokens;
  p.pages = plan->pages;
  p.page_shift = shift_of(plan->page_tokens);
  p.kv_heads = plan->kv_heads;
  p.group = s.group;
  p.group_inv = (unsigned)(((uint64_t)1 << 32) / s.group) + 1;
  p.causal = causal ? 1 : 0;
  p.block_rows = s.block_rows;
  p.k = arena->k_codes;
  p.v = arena->v_codes;
  p.ks = arena->k_scales;
  p.vs = arena->v_scales;
  p.q = static_cast<const uint16_t*>(q_device);
  p.q_row = q_row_stride;
  p.q_head = q_head_stride;
  p.scale_log2 = softmax_scale * 1.44269504088896341f;
  p.out = static_cast<uint16_t*>(out_device);
  p.lse = lse_device;
  p.qtile_tokens = s.qtile_tokens;
  p.probes = std::min(scan_wait_limit(), kProbes);
  p.status = plan->status;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (s.qtile_cap > 0 &&
      (rc = launch_prompt(dtype, plan->head_dim, p, s.qtile_cap * plan->kv_heads, st)))
    return rc;
  return dtype == GRM_B200_F16
             ? launch_split_any<__half>(plan->head_dim, s.block_rows, sp, s.workers, st)
             : launch_split_any<__nv_bfloat16>(plan->head_dim, s.block_rows, sp, s.workers, st);
}

}  // extern "C"
