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
// sum_t p_t / u_t, so p_t never exceeds 2^8 whatever the scales are and fp16
// holds it (m trails the largest y seen by at most 8: it moves only when a y
// passes m + 8, so the accumulators are rarely rescaled).   The log-sum-exp is m ln 2 + log of that sum.
//
// The split kernel serves few query rows a kv head (decoding, a few proposed
// tokens): it is bound by the bytes of the codes, 2 * head_dim a token and kv
// head.  Every resident block ("worker") gets the same share of all tiles of
// all requests and heads, whatever their lengths; a segment (request, kv head,
// up to 16 query rows) that several workers share is joined by the one that
// finishes it last, in the order of the workers, so results do not depend on
// timing.
//
// A warp owns 16 of a tile's 64 tokens, in a private ring of shared-memory
// stages that it fills with 16-byte asynchronous copies and drains without a
// barrier of the block.  Products run on mma.m16n8k16 with fp16 operands and
// fp32 accumulators, tokens (or value dims) on the M side and the query rows on
// the 8-wide N side: four query heads of a group waste half of the columns
// instead of three quarters.  Codes become fp16 exactly: byte b of code + 128
// under the exponent of 1024 is the half 1024 + b, less 1152.  Queries are
// fp16: a bf16 row is first scaled by the power of two that brings its largest
// value into [2^14, 2^15), so only values 2^29 times smaller than the largest
// round.
#include <algorithm>
#include <type_traits>

#include "paged.cuh"

namespace grm_b200 {
namespace paged {

namespace {

constexpr int kWarps = 4;
constexpr int kThreads = kWarps * 32;

template <int D, int NT>
struct Layout {
  static constexpr int kStages = D == 256 ? 3 : D == 128 ? 3 : 5;
  static constexpr int kSide = 16 * D;            // codes of 16 tokens
  static constexpr int kStage = 2 * kSide;
  static constexpr int kRow = D + 4;              // floats of a row in the merge buffer
  static constexpr int kRing = kWarps * kStages * kStage;
  static constexpr int kMerge = 2 * NT * 8 * kRow * 4;
  static constexpr int kScales = kWarps * kStages * 2 * 4;
  static constexpr int kML = 2 * kWarps * NT * 8 * 4;
  static constexpr int kSmem = kRing + kMerge + kScales + kML + 16;
  static constexpr int kBlocks = D == 256 ? 2 : 3;
};

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async4(uint32_t dst, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

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
// Byte of chunk c (16 codes) of row r in a 16-row tile whose rows are D codes:
// 16-byte chunks are permuted so that eight rows of one chunk lie in eight
// different bank groups (ldmatrix reads them together).
template <int D>
__device__ __forceinline__ uint32_t tile_byte(int r, int c) {
  if (D == 64) return (r >> 1) * 128 + ((((r & 1) << 2) | (c ^ ((r >> 1) & 3))) << 4);
  return r * D + ((c ^ (r & 7)) << 4);
}

// A segment: up to block_rows query rows of a kv head of a request.
struct Segment {
  int64_t first;  // its first unit
  int request, tiles, len, start, pairs, head, row0, cached;
};

// The share of one worker, walked segment by segment.
struct Walk {
  const AttendParams& p;
  int64_t begin, end;  // units
  int64_t u;           // first unit of the next segment to look at
  int r;
  Segment s;
  int t, t1;           // tiles of s that are the worker's, from t on

  __device__ __forceinline__ Walk(const AttendParams& pp, int64_t b, int64_t e, int request)
      : p(pp), begin(b), end(e), u(b), r(request) {}

  // Step to the next segment that reaches into the share; false at its end.
  __device__ __forceinline__ bool next() {
    if (u >= end) return false;
    while (__ldg(p.l.base + r + 1) <= u) ++r;
    const int64_t base = __ldg(p.l.base + r);
    s.request = r;
    s.start = __ldg(p.starts + r);
    const int n = __ldg(p.starts + r + 1) - s.start;
    s.len = __ldg(p.lens + r);
    s.cached = s.len - n;
    s.pairs = n * p.group;
    s.tiles = (s.len + kTile - 1) / kTile;
    const int blocks = (s.pairs + p.block_rows - 1) / p.block_rows;
    const int64_t i = (u - base) / (s.tiles + 1);
    s.first = base + i * (s.tiles + 1);
    s.head = (int)(i / blocks);
    s.row0 = (int)(i - (int64_t)s.head * blocks) * p.block_rows;
    u = s.first + s.tiles + 1;
    const int64_t a = begin - s.first - 1, b = end - s.first - 1;
    t = a > 0 ? (int)a : 0;
    t1 = b < s.tiles ? (int)b : s.tiles;
    return true;
  }
};

template <typename T, int D, int NT>
__global__ void __launch_bounds__(kThreads, Layout<D, NT>::kBlocks)
    split_kernel(const AttendParams p) {
  using LY = Layout<D, NT>;
  constexpr int kChunks = D / 16;
  extern __shared__ __align__(128) unsigned char smem[];
  float* const merge = reinterpret_cast<float*>(smem + LY::kRing);
  float* const scales = reinterpret_cast<float*>(smem + LY::kRing + LY::kMerge);
  float* const sm_m = reinterpret_cast<float*>(smem + LY::kRing + LY::kMerge + LY::kScales);
  float* const sm_l = sm_m + kWarps * NT * 8;
  int* const sm_last = reinterpret_cast<int*>(sm_l + kWarps * NT * 8);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, t4 = lane & 3;
  const int heads = p.kv_heads * p.group;
  const Header hd = *p.l.header;

  // rows past the step's last one
  for (int64_t i = hd.rows + (int64_t)blockIdx.x; i < p.tokens; i += gridDim.x) {
    for (int x = threadIdx.x; x < heads * D / 2; x += kThreads)
      reinterpret_cast<uint32_t*>(p.out + i * heads * D)[x] = 0;
    if (p.lse)
      for (int x = threadIdx.x; x < heads; x += kThreads) p.lse[i * heads + x] = -INFINITY;
  }
  const int w = blockIdx.x;
  if (w >= hd.workers) return;
  const int64_t begin = worker_first(w, hd.units, hd.workers);
  const int64_t end = worker_first(w + 1, hd.units, hd.workers);
  const int request0 = p.l.start[w];

  // ---- the loader: 16 tokens of a tile for this warp, one stage at a time
  const uint32_t ring = smem_u32(smem) + warp * LY::kStages * LY::kStage;
  const uint32_t ring_scales = smem_u32(scales) + warp * LY::kStages * 8;
  Walk load(p, begin, end, request0);
  bool loading = true;
  load.t = load.t1 = 0;
  int ids = 0, ids_base = 0, ids_request = -1;  // lane i: page ids_base + i of the request
  auto issue = [&](int stage) {
    while (loading && load.t >= load.t1) loading = load.next();
    if (loading) {
      const Segment& s = load.s;
      const int tok = load.t * kTile + warp * 16;
      if (tok < s.len) {
        const int j = tok >> p.page_shift;
        if (s.request != ids_request || j >= ids_base + 32 || j < ids_base) {
          const int last = (s.len - 1) >> p.page_shift;
          ids = __ldg(p.table + s.request * p.width + min(j + lane, last));
          ids_base = j;
          ids_request = s.request;
        }
        int64_t page = __shfl_sync(kFull, ids, j - ids_base);
        page = min(max(page, (int64_t)0), p.pages - 1);
        const int64_t at = page * p.kv_heads + s.head;
        const int64_t off = ((at << p.page_shift) + (tok & ((1 << p.page_shift) - 1))) * D;
        const int8_t* kp = p.k + off;
        const int8_t* vp = p.v + off;
        const uint32_t dst = ring + stage * LY::kStage;
#pragma unroll
        for (int i = 0; i < kChunks / 2; ++i) {
          const int c = lane + 32 * i;
          const uint32_t to = dst + tile_byte<D>(c / kChunks, c % kChunks);
          cp_async16(to, kp + c * 16);
          cp_async16(to + LY::kSide, vp + c * 16);
        }
        if (lane < 2) cp_async4(ring_scales + stage * 8 + lane * 4, (lane ? p.vs : p.ks) + at);
      }
      ++load.t;
    }
    cp_commit();
  };
#pragma unroll
  for (int i = 0; i < LY::kStages - 1; ++i) issue(i);
  int stage = 0;

  // ldmatrix source of this lane: rows 0-7 / 8-15 of an even chunk, then of an odd one
  const int lm_row = lane & 15, lm_chunk = lane >> 4;

  Walk walk(p, begin, end, request0);
  while (walk.next()) {
    const Segment s = walk.s;
    const int rows = min(s.pairs - s.row0, NT * 8);
    if (s.tiles == 0) {  // nothing cached: empty rows (the segment is its one unit)
      for (int x = threadIdx.x; x < rows * (D / 2); x += kThreads) {
        const int j = s.row0 + x / (D / 2);
        const int64_t row = (int64_t)(s.start + j / p.group) * heads + s.head * p.group +
                            j % p.group;
        reinterpret_cast<uint32_t*>(p.out + row * D)[x % (D / 2)] = 0;
        if (p.lse && x % (D / 2) == 0) p.lse[row] = -INFINITY;
      }
      continue;
    }
    if (walk.t >= walk.t1) continue;  // only its start is this worker's

    // ---- queries: column g of the B operand, dims 16c + 4 t4 .. + 3
    uint32_t qf[kChunks][NT][2];
    float kq[NT][2];
    int lim[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int j = s.row0 + nt * 8 + g;
      uint2 raw[kChunks];
#pragma unroll
      for (int c = 0; c < kChunks; ++c) raw[c] = make_uint2(0, 0);
      if (j < s.pairs) {
        const uint16_t* qp = p.q + (int64_t)(s.start + j / p.group) * p.q_row +
                             (int64_t)(s.head * p.group + j % p.group) * p.q_head + t4 * 4;
#pragma unroll
        for (int c = 0; c < kChunks; ++c)
          raw[c] = __ldg(reinterpret_cast<const uint2*>(qp + c * 16));
      }
      float unscale = 1.0f;
      if constexpr (!std::is_same<T, __half>::value) {
        unsigned m = 0;
#pragma unroll
        for (int c = 0; c < kChunks; ++c)
          m = __vmaxu2(m, __vmaxu2(raw[c].x & 0x7FFF7FFFu, raw[c].y & 0x7FFF7FFFu));
        m = max(m & 0xFFFFu, m >> 16);
        m = max(m, __shfl_xor_sync(kFull, m, 1));
        m = max(m, __shfl_xor_sync(kFull, m, 2));
        float up;
        row_scale(m, &up, &unscale);
#pragma unroll
        for (int c = 0; c < kChunks; ++c) {
          qf[c][nt][0] = scale_pair(raw[c].x, up);
          qf[c][nt][1] = scale_pair(raw[c].y, up);
        }
      } else {
#pragma unroll
        for (int c = 0; c < kChunks; ++c) {
          qf[c][nt][0] = raw[c].x;
          qf[c][nt][1] = raw[c].y;
        }
      }
      // columns 2 t4 and 2 t4 + 1 of the scores
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        kq[nt][x] = p.scale_log2 * __shfl_sync(kFull, unscale, (2 * t4 + x) * 4);
        const int jc = s.row0 + nt * 8 + 2 * t4 + x;
        lim[nt][x] = p.causal && jc < s.pairs ? s.cached + jc / p.group + 1 : s.len;
      }
    }
    const int all_see = p.causal ? s.cached + s.row0 / p.group + 1 : s.len;

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
    for (int t = walk.t; t < walk.t1; ++t) {
      cp_wait<LY::kStages - 2>();
      __syncwarp();
      issue(stage == 0 ? LY::kStages - 1 : stage - 1);
      const int tok = t * kTile + warp * 16;
      if (tok < s.len) {
        const uint32_t kb = ring + stage * LY::kStage, vb = kb + LY::kSide;
        const float ks = scales[(warp * LY::kStages + stage) * 2];
        float lv, inv;
        value_scale(scales[(warp * LY::kStages + stage) * 2 + 1], &lv, &inv);
        // scores of 16 tokens x 8 NT rows, in two independent chains
        float sc[NT][2][4];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int x = 0; x < 4; ++x) sc[nt][0][x] = sc[nt][1][x] = 0.0f;
#pragma unroll
        for (int c = 0; c < kChunks; c += 2) {
          uint32_t r[4];
          ldsm4(r, kb + tile_byte<D>(lm_row, c + lm_chunk));
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            const uint32_t lo = r[2 * x] ^ 0x80808080u, hi = r[2 * x + 1] ^ 0x80808080u;
            const uint32_t a0 = halves(lo, 0x4140), a2 = halves(lo, 0x4342);
            const uint32_t a1 = halves(hi, 0x4140), a3 = halves(hi, 0x4342);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
              mma(sc[nt][x], a0, a1, a2, a3, qf[c + x][nt][0], qf[c + x][nt][1]);
          }
        }
        uint32_t b[NT][2];
        float y[NT][4];
        bool moves = false;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
          for (int x = 0; x < 4; ++x)
            y[nt][x] = fmaf(sc[nt][0][x] + sc[nt][1][x], kq[nt][x & 1] * ks, lv);
          if (tok + 16 > all_see) {
#pragma unroll
            for (int x = 0; x < 4; ++x)
              if (tok + g + (x >> 1) * 8 >= min(lim[nt][x & 1], s.len)) y[nt][x] = -INFINITY;
          }
#pragma unroll
          for (int x = 0; x < 4; ++x) moves |= y[nt][x] > m[nt][x & 1] + kLazy;
        }
        if (__any_sync(kFull, moves)) {
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int x = 0; x < 2; ++x) {
              float top = fmaxf(y[nt][x], y[nt][x + 2]);
#pragma unroll
              for (int i = 4; i <= 16; i <<= 1) top = fmaxf(top, __shfl_xor_sync(kFull, top, i));
              // each row by its own scores, so that no row's rounding hangs on another's
              if (!(top > m[nt][x] + kLazy)) top = m[nt][x];
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
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          float pr[4];
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            const float ref = m[nt][x & 1] == -INFINITY ? 0.0f : m[nt][x & 1];
            pr[x] = ex2(y[nt][x] - ref);
          }
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            l[nt][x] = fmaf(pr[x] + pr[x + 2], inv, l[nt][x]);
          }
          b[nt][0] = transpose8(pack_half2(pr[0], pr[1]));
          b[nt][1] = transpose8(pack_half2(pr[2], pr[3]));
        }
        // result dims 16c + 2g (rows g) and 16c + 2g + 1 (rows g + 8)
#pragma unroll
        for (int c = 0; c < kChunks; c += 2) {
          uint32_t r[4];
          ldsm4t(r, vb + tile_byte<D>(lm_row, c + lm_chunk));
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            const uint32_t lo = r[2 * x] ^ 0x80808080u, hi = r[2 * x + 1] ^ 0x80808080u;
            const uint32_t a0 = halves(lo, 0x4240), a1 = halves(lo, 0x4341);
            const uint32_t a2 = halves(hi, 0x4240), a3 = halves(hi, 0x4341);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) mma(o[c + x][nt], a0, a1, a2, a3, b[nt][0], b[nt][1]);
          }
        }
      }
      stage = stage + 1 == LY::kStages ? 0 : stage + 1;
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
    auto at = [&](int buf, int c, int nt, int x) {
      return reinterpret_cast<float2*>(merge + (buf * NT * 8 + nt * 8 + 2 * t4 + x) * LY::kRow +
                                       16 * c + 2 * g);
    };
    auto put = [&](int buf) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int c = 0; c < kChunks; ++c)
#pragma unroll
          for (int x = 0; x < 2; ++x) *at(buf, c, nt, x) = make_float2(o[c][nt][x], o[c][nt][x + 2]);
    };
    auto add = [&](int buf) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int c = 0; c < kChunks; ++c)
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            const float2 v = *at(buf, c, nt, x);
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

    // ---- alone on the segment: done
    const int64_t wa = worker_of(s.first + 1, hd.units, hd.workers);
    const int64_t wb = worker_of(s.first + s.tiles, hd.units, hd.workers);
    if (wa == wb) {
      if (warp == 0) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            const int j = s.row0 + nt * 8 + 2 * t4 + x;
            if (j < s.pairs) {
              const int64_t row = (int64_t)(s.start + j / p.group) * heads + s.head * p.group +
                                  j % p.group;
              const float sum = lt[nt][x];
              const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
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
      float* slot = p.l.part + (2 * w + (w == wa ? 1 : 0)) * (int64_t)kWorkerSlot;
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
            *reinterpret_cast<float2*>(slot + 2048 + 2 * row) = make_float2(m[nt][x], lt[nt][x]);
        }
      __threadfence();
      __syncwarp();
      if (lane == 0) {
        const unsigned arrived = atomicAdd(p.l.count + wa, 1u);
        const int last = arrived + 1 == (unsigned)(wb - wa + 1);
        if (last) p.l.count[wa] = 0;  // for the next call
        *sm_last = last;
        __threadfence();
      }
    }
    __syncthreads();
    if (*sm_last) {
      const int n = (int)(wb - wa + 1);
      auto part = [&](int i) {
        return p.l.part + (2 * (wa + i) + (i == 0 ? 1 : 0)) * (int64_t)kWorkerSlot;
      };
      for (int row = warp; row < rows; row += kWarps) {  // a warp takes a row
        float top = -INFINITY;
        for (int i = lane; i < n; i += 32) top = fmaxf(top, __ldcg(part(i) + 2048 + 2 * row));
#pragma unroll
        for (int i = 16; i >= 1; i >>= 1) top = fmaxf(top, __shfl_xor_sync(kFull, top, i));
        float sum = 0.0f, acc[D / 32] = {};
#pragma unroll 4
        for (int i = 0; i < n; ++i) {
          const float* src = part(i);
          const float2 ml = __ldcg(reinterpret_cast<const float2*>(src + 2048 + 2 * row));
          const float a = ml.x == top ? 1.0f : ex2(ml.x - top);
          sum += ml.y == 0.0f ? 0.0f : ml.y * a;
#pragma unroll
          for (int d = 0; d < D / 64; ++d) {
            const float2 v = __ldcg(reinterpret_cast<const float2*>(src + row * D + 64 * d + 2 * lane));
            acc[2 * d] = fmaf(v.x, a, acc[2 * d]);
            acc[2 * d + 1] = fmaf(v.y, a, acc[2 * d + 1]);
          }
        }
        const int j = s.row0 + row;
        const int64_t orow = (int64_t)(s.start + j / p.group) * heads + s.head * p.group +
                             j % p.group;
        const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
#pragma unroll
        for (int d = 0; d < D / 64; ++d)
          *reinterpret_cast<uint32_t*>(p.out + orow * D + 64 * d + 2 * lane) =
              pack_out<T>(acc[2 * d] * inv, acc[2 * d + 1] * inv);
        if (p.lse && lane == 0)
          p.lse[orow] = sum == 0.0f ? -INFINITY : (top + log2f(sum)) * 0.693147180559945309f;
      }
    }
  }
  cp_wait<0>();
}

template <typename T, int D, int NT>
int launch_split(const AttendParams& p, int workers, cudaStream_t st) {
  using LY = Layout<D, NT>;
  static_assert(NT * 8 * D <= 2048, "a partial result fits its slot");
  auto kernel = split_kernel<T, D, NT>;
  const cudaError_t e =
      cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, LY::kSmem);
  if (e != cudaSuccess) {
    set_thread_error("paged attend: %s", cudaGetErrorString(e));
    return cuda_status(e);
  }
  kernel<<<workers, kThreads, LY::kSmem, st>>>(p);
  return launch_status("paged attend");
}

template <typename T>
int launch_split_any(int dim, int block_rows, const AttendParams& p, int workers,
                     cudaStream_t st) {
  if (dim == 64)
    return block_rows == 8 ? launch_split<T, 64, 1>(p, workers, st)
                           : launch_split<T, 64, 2>(p, workers, st);
  if (dim == 128)
    return block_rows == 8 ? launch_split<T, 128, 1>(p, workers, st)
                           : launch_split<T, 128, 2>(p, workers, st);
  return launch_split<T, 256, 1>(p, workers, st);
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
  AttendParams p;
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
  p.status = plan->status;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  rc = dtype == GRM_B200_F16
           ? launch_split_any<__half>(plan->head_dim, s.block_rows, p, s.workers, st)
           : launch_split_any<__nv_bfloat16>(plan->head_dim, s.block_rows, p, s.workers, st);
  if (rc == 0 && s.qtile_cap > 0)
    rc = launch_prompt(dtype, plan->head_dim, p, s.qtile_cap * plan->kv_heads, st);
  return rc;
}

}  // extern "C"
