// latent_prompt.cu -- latent attention in the expanded form for heads of 64 + 64 values.
//
// The sums are latent_attend.cu's, whose kernel serves heads of 128 + 128.  A product
// of the tensor cores costs the same for 64 columns as for 128, so with scores of 64
// tokens at a time they are what that kernel waits for: 14 products of 64 clocks for
// 64 tokens of each of its two query tiles, 1,800 clocks, where the exponentials take
// 1,024.  Here scores are of 128 tokens (10 products) and results of 128 tokens and 64
// values (8), 1,152 clocks for 64 tokens.
//
// Tensor memory holds two results of 64 columns and three buffers of 128 scores, which
// the tiles' steps take in turn, weights over the scores they are made from: while one
// tile's softmax runs, the other's next scores are there and its own are on their way.
// One warp issues all products, in the order in which the softmax warps take turns.
// Queries are in shared memory.
//
// 8,449 rows of 3 requests of up to 16,000 tokens, 40 heads of 64 + 32, 64: 1.7 ms in
// latent_attend.cu's way, @@ here.
#include <algorithm>

#include "latent_device.cuh"

namespace grm_b200 {
namespace latent {

namespace {

using paged::ex2;
using paged::kLazy;
using paged::kProbes;
using paged::reference_of;

constexpr int kTokens = 128;          // of a step
constexpr int kHead = 64;             // values of a head's keys beside the positional part
constexpr int kAtom = kTokens * 128;  // 128 tokens or rows x 64 values
constexpr int kQ = 2;                 // query tiles
constexpr int kBuffers = 3;           // of scores
constexpr uint32_t kTmemCols = 512;

template <int ROPE>
struct Layout {
  // a stage: keys, what their rounding left over, positional part, values
  static constexpr int kRopeAt = 2 * kAtom;
  static constexpr int kRopeBytes = kTokens * ROPE * 2;
  static constexpr int kValueAt = kRopeAt + kRopeBytes;
  static constexpr int kStage = kValueAt + kAtom;
  static constexpr int kQuery = kAtom + kRows * ROPE * 2;  // the positional part last
  static constexpr int kStages = (232448 - 1024 - 1024 - kQ * kQuery) / kStage;
  static constexpr int kSmem = 1024 + kQ * kQuery + kStages * kStage;
  static constexpr uint32_t kResult = kBuffers * kTokens;
  static constexpr int kSoftWarps = 4 * kQ, kMmaWarp = kSoftWarps;  // and one that loads
  static constexpr int kThreads = (kMmaWarp + 2) * 32;
  static constexpr int kSlot = slot_floats(kRows * kQ, kHead);
  static_assert(kStages >= 2 && kResult + kQ * kHead <= kTmemCols, "tiles");
};

// fp32 accumulators, 16-bit operands, 128 rows, n columns; B K-major or (b_mn) not.
template <typename T>
__host__ __device__ constexpr uint32_t idesc(int n, bool b_mn) {
  return (1u << 4) | Kind<T>::kFormat | (b_mn ? 1u << 16 : 0u) | ((uint32_t)(n >> 3) << 17) |
         ((uint32_t)(kRows >> 4) << 24);
}

// The scores of a step from the first hidden one on set to -inf, in tensor memory;
// `bad`: the hidden tokens whose score was no finite number.
__device__ __forceinline__ void hide(uint32_t scores, int seen, unsigned (&bad)[4]) {
#pragma unroll 1
  for (int c = 0; c < kTokens; c += 16) {
    uint32_t v[16];
    tmem_ld16(scores + c, v);
    unsigned b = 0;
#pragma unroll
    for (int k = 0; k < 16; ++k)
      if (c + k >= seen) {
        if ((v[k] & 0x7F800000u) == 0x7F800000u) b |= 1u << k;
        v[k] = 0xFF800000u;
      }
    tmem_st16(scores + c, v);
#pragma unroll
    for (int w = 0; w < 4; ++w)
      if (c / 32 == w) bad[w] |= b << (c % 32);
  }
  tmem_wait_st();
}

// Numbers that are none among the values of 32 tokens from `t0` on, set to 0.
template <typename T>
__device__ __noinline__ void scrub(unsigned char* values, int t0, unsigned tokens) {
  while (tokens) {
    const int t = t0 + __ffs((int)tokens) - 1;
    tokens &= tokens - 1;
    for (int c = 0; c < 8; ++c) {
      uint4* at = reinterpret_cast<uint4*>(values + atom_byte(t, c));
      const uint4 v = *at;
      uint32_t x[4] = {v.x, v.y, v.z, v.w};
      bool bad = false;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        constexpr uint32_t e = Kind<T>::kNoNumber;
        if ((x[i] & e) == e) { x[i] &= 0xFFFF0000u; bad = true; }
        if ((x[i] >> 16 & e) == e) { x[i] &= 0x0000FFFFu; bad = true; }
      }
      if (bad) *at = make_uint4(x[0], x[1], x[2], x[3]);
    }
  }
}

// The rows of a worker in which a wait gave up: no numbers.
template <int ROPE>
__device__ __noinline__ void lose_rows(const Params& p, const Header& hd, int worker) {
  using LY = Layout<ROPE>;
  const float nan = __int_as_float(0x7FC00000);
  const int t = threadIdx.x >> 7, row = threadIdx.x & 127;
  Parts<kQ, kTokens> parts(p, hd, worker, p.l.start[worker]);
  Part x;
  while (parts.next(p, &x)) {
    const Row a = row_of<true>(p, x, t, row);
    if (x.slot >= 0) {
      float* slot = p.l.part + (int64_t)x.slot * LY::kSlot;
      *reinterpret_cast<float4*>(slot + kRows * kQ * kHead + 4 * (t * kRows + row)) =
          make_float4(-INFINITY, nan, nan, 0.0f);
    } else if (a.active) {
      const int64_t orow = (int64_t)(x.start + a.token) * p.heads + a.head;
      for (int c = 0; c < kHead / 8; ++c)
        reinterpret_cast<uint4*>(p.out + orow * kHead)[c] =
            make_uint4(0x7FFF7FFFu, 0x7FFF7FFFu, 0x7FFF7FFFu, 0x7FFF7FFFu);
      if (p.lse) p.lse[orow] = nan;
    }
  }
}

struct Maps {
  CUtensorMap keys;    // 64 values of a head's keys, of what was left over, of 128 tokens
  CUtensorMap rope;    // the positional part of rows of the cache
  CUtensorMap values;  // a head's values
};

template <typename T, int ROPE>
__global__ void __launch_bounds__(Layout<ROPE>::kThreads, 1)
    prompt_kernel(const __grid_constant__ Maps maps, const __grid_constant__ Params p) {
  using LY = Layout<ROPE>;
  constexpr int kStages = LY::kStages;
  extern __shared__ unsigned char raw[];
  unsigned char* const sm = raw + ((1024u - (smem_u32(raw) & 1023u)) & 1023u);
  unsigned char* const sm_q = sm;                         // [kQ]
  unsigned char* const sm_stage = sm + kQ * LY::kQuery;   // [kStages]
  __shared__ __align__(8) uint64_t full[kStages], empty[kStages], q_full[kQ], drained,
      s_full[kBuffers], p_full[kBuffers][2], o_full[kQ], o_done[kQ], turn[kQ][4];
  __shared__ uint32_t sh_tmem;
  __shared__ int sh_fail;

  const int worker = blockIdx.x;
  const Start begin = p.l.start[worker];  // on its way beside the header
  const Header hd = *p.l.header;
  asm volatile("griddepcontrol.launch_dependents;");
  if (worker >= hd.workers) return;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (hd.lost) {
    if (warp < LY::kSoftWarps) lose_rows<ROPE>(p, hd, worker);
    return;
  }
  if (threadIdx.x == 0) {
    for (int i = 0; i < kStages; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 1);
    }
    for (int i = 0; i < kBuffers; ++i) {
      mbar_init(&s_full[i], 1);
      for (int x = 0; x < 2; ++x) mbar_init(&p_full[i][x], 4);
    }
    for (int t = 0; t < kQ; ++t) {
      mbar_init(&q_full[t], 4);
      mbar_init(&o_full[t], 1);
      mbar_init(&o_done[t], 1);
      for (int x = 0; x < 4; ++x) mbar_init(&turn[t][x], 1);
    }
    mbar_init(&drained, 1);
    mbar_fence_init();
    sh_fail = 0;
  }
  if (warp == LY::kMmaWarp) {
    tmem_alloc(&sh_tmem, kTmemCols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = sh_tmem;
  auto wait = [&](uint64_t* bar, unsigned parity) {
    return warp_wait(bar, parity, &sh_fail, p.probes);
  };
  Parts<kQ, kTokens> parts(p, hd, worker, begin);
  Part x;

  if (warp < LY::kSoftWarps) {
    // ------------------------------------------------------------- softmax
    const int t = warp >> 2, row = (warp & 3) * 32 + lane;
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t o_col = tmem + lanes + LY::kResult + t * kHead;
    unsigned char* const my_q = sm_q + t * LY::kQuery;
    bool ok = true;
    int it = 0, tile = 0, stage0 = 0;  // steps and tiles of this query tile; stages so far
    int turns = 0;                     // steps of both query tiles so far
    unsigned scored = 0;               // scores of the parts before, of either tile
    // the row's query of a part, to shared memory
    auto queries = [&](const Part& y) {
      const Row b = row_of<true>(p, y, t, row);
      const uint16_t* qp = p.q + (int64_t)(y.start + b.token) * p.q_row + b.head * p.q_head;
      constexpr int kChunks = (kHead + ROPE) / 8;
      uint4 v[kChunks];
#pragma unroll
      for (int c = 0; c < kChunks; ++c)
        v[c] = b.active ? __ldg(reinterpret_cast<const uint4*>(qp) + c) : make_uint4(0, 0, 0, 0);
#pragma unroll
      for (int c = 0; c < kChunks; ++c) {
        const int r = c - 8;
        *reinterpret_cast<uint4*>(
            my_q + (c < 8 ? atom_byte(row, c)
                          : kAtom + (ROPE == 64 ? atom_byte(row, r) : half_atom_byte(row, r)))) = v[c];
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(&q_full[t]);
    };
    Part next;
    bool more = parts.next(p, &next), held = false;  // held: a tile whose result is to go out
    Row a{0, 0, false};
    bool idle = false;
    int steps = 0;
    float m = 0.0f, l = 0.0f, lr = 0.0f;
#pragma unroll 1
    while (true) {
      // The scores of the tile before are there, so its queries' place is free: the next
      // tile's first scores are worked out while this one's result goes out.
      if (more && next.steps > 0 && next.toks[t] > 0) queries(next);
      if (held) {
        if (steps > 0) {
          if (!(ok = wait(&o_done[t], tile & 1))) break;
          tc_fence_after();
          ++tile;
        }
        const int64_t orow = (int64_t)(x.start + a.token) * p.heads + a.head;
        float* const slot = p.l.part + (int64_t)x.slot * LY::kSlot;
        const float inv = lr == 0.0f ? 0.0f : 1.0f / lr;
        if (!idle)
#pragma unroll 1
          for (int c = 0; c < kHead; c += 32) {
            uint32_t o[32];
            if (steps > 0) {
              tmem_ld32_nowait(o_col + c, o);
              tmem_wait_ld32(o);
            }
            if (!a.active) continue;
            if (x.slot >= 0) {  // a part's result, for join_kernel
              float4* to = reinterpret_cast<float4*>(slot + (t * kRows + row) * kHead + c);
              if (steps > 0)
#pragma unroll
                for (int k = 0; k < 8; ++k)
                  to[k] = make_float4(__uint_as_float(o[4 * k]), __uint_as_float(o[4 * k + 1]),
                                      __uint_as_float(o[4 * k + 2]), __uint_as_float(o[4 * k + 3]));
            } else {
              uint4* to = reinterpret_cast<uint4*>(p.out + orow * kHead + c);
#pragma unroll
              for (int k = 0; k < 4; ++k) {
                uint32_t w[4];
#pragma unroll
                for (int y = 0; y < 4; ++y)
                  w[y] = lr == 0.0f ? 0u
                                    : Kind<T>::pack(__uint_as_float(o[8 * k + 2 * y]) * inv,
                                                    __uint_as_float(o[8 * k + 2 * y + 1]) * inv);
                to[k] = make_uint4(w[0], w[1], w[2], w[3]);
              }
            }
          }
        if (a.active) {
          if (x.slot >= 0)
            *reinterpret_cast<float4*>(slot + kRows * kQ * kHead + 4 * (t * kRows + row)) =
                make_float4(m, l, lr, 0.0f);
          else if (p.lse)
            p.lse[orow] = l == 0.0f ? -INFINITY
                                    : (m - Kind<T>::kLift + log2f(l)) * 0.693147180559945309f;
        }
        // what the next tile's products overwrite has been read
        tc_fence_before();
      }
      if (!more) break;
      x = next;
      steps = x.steps;
      const bool two = x.toks[1] > 0;
      const int stage_base = stage0;
      const unsigned scored0 = scored;
      stage0 += steps;
      scored += steps << two;
      held = x.toks[t] > 0;
      if (!held || steps == 0) more = parts.next(p, &next);
      if (!held) continue;
      a = row_of<true>(p, x, t, row);
      m = -INFINITY;
      l = lr = 0.0f;
      // tokens that the row sees, from the part's first on
      const int lim = (p.causal ? min(x.len, x.cached + a.token + 1) : x.len) - x.step0 * kTokens;
      idle = !__any_sync(kFull, a.active);
#pragma unroll 1
      for (int i = 0; i < steps; ++i, ++it) {
        const unsigned n = scored0 + (two ? 2 * i + t : i), buf = n % kBuffers;
        const uint32_t s_col = tmem + lanes + buf * kTokens;
        if (!(ok = wait(&s_full[buf], (n / kBuffers) & 1))) break;
        tc_fence_after();
        // The two softmax warps of a scheduler take turns at the exponentials, so that one's
        // other work lies under them.
        auto my_turn = [&] {
          const bool go = t == 1 || turns > 0 ? wait(&turn[t][warp & 3], (turns - 1 + t) & 1) : true;
          ++turns;
          return go;
        };
        if (idle) {
          if (two && !(ok = my_turn())) break;
          if (lane == 0) {
            mbar_arrive(&p_full[buf][0]);
            mbar_arrive(&p_full[buf][1]);
            if (two) mbar_arrive(&turn[1 - t][warp & 3]);
          }
          if (i == 0) more = parts.next(p, &next);
          continue;
        }
        if (__any_sync(kFull, (i + 1) * kTokens > lim)) {
          unsigned bad[4] = {0, 0, 0, 0};
          hide(s_col, lim - i * kTokens, bad);
          if (__any_sync(kFull, (bad[0] | bad[1] | bad[2] | bad[3]) != 0)) {
            const int st = stage_base + i;  // its copies landed before the scores were there
            if (!(ok = wait(&full[st % kStages], (st / kStages) & 1))) break;
#pragma unroll
            for (int w = 0; w < 4; ++w)
              scrub<T>(sm_stage + st % kStages * LY::kStage + LY::kValueAt, 32 * w, bad[w]);
            fence_proxy_async_smem();
          }
        }
        uint32_t v[2][32];
        float tops[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};  // chains side by side
#pragma unroll
        for (int c = 0; c < 4; c += 2) {
          tmem_ld32_nowait(s_col + 32 * c, v[0]);
          tmem_ld32_nowait(s_col + 32 * c + 32, v[1]);
          tmem_wait_ld32(v[0]);
          tmem_wait_ld32(v[1]);
#pragma unroll
          for (int k = 0; k < 64; k += 2)
            tops[k / 2 % 4] = max3(tops[k / 2 % 4], __uint_as_float(v[k / 32][k % 32]),
                                   __uint_as_float(v[k / 32][k % 32 + 1]));
        }
        const float top = fmaxf(max3(tops[0], tops[1], tops[2]), tops[3]) * p.scale_log2;
        if (__any_sync(kFull, top > m + kLazy)) {
          const float now = top > m + kLazy ? reference_of(top) : m;
          const float f = now == m ? 1.0f : ex2(m - now);
          m = now;
          l *= f;
          lr *= f;
          if (i > 0) {  // once the products of the step before have ended
            if (!(ok = wait(&o_full[t], (it - 1) & 1))) break;
            tc_fence_after();
#pragma unroll 1
            for (int c = 0; c < kHead / 16; ++c) {
              uint32_t o[16];
              tmem_ld16(o_col + 16 * c, o);
#pragma unroll
              for (int k = 0; k < 16; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * f);
              tmem_st16(o_col + 16 * c, o);
            }
          }
        }
        const float off = m == -INFINITY ? 0.0f : Kind<T>::kLift - m;
        if (two && !(ok = my_turn())) break;
        float2 sum = make_float2(0.0f, 0.0f), rounded = make_float2(0.0f, 0.0f);
        tmem_ld32_nowait(s_col, v[0]);
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          tmem_wait_ld32(v[c & 1]);
          if (c < 3) tmem_ld32_nowait(s_col + 32 * (c + 1), v[(c + 1) & 1]);
          uint32_t w[16];
#pragma unroll
          for (int k = 0; k < 32; k += 2) {
            const float2 y = fma2(__uint_as_float(v[c & 1][k]), __uint_as_float(v[c & 1][k + 1]),
                                  p.scale_log2, off);
            const float2 e = make_float2(ex2(y.x), ex2(y.y));
            sum = add2(sum, e);
            w[k / 2] = Kind<T>::pack(e.x, e.y);
            rounded = add2(rounded, Kind<T>::widen(w[k / 2]));
            // seven eighths done: the other's first ones fill the gaps of the last
            if (c == 3 && k == 14 && two && lane == 0) mbar_arrive(&turn[1 - t][warp & 3]);
          }
          tmem_st16(s_col + 16 * c, w);  // over scores that have been read
          if (c & 1) {  // half of the weights
            tmem_wait_st();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&p_full[buf][c >> 1]);
          }
        }
        l += sum.x + sum.y;
        lr += rounded.x + rounded.y;
        // a chain of loads that lies under the wait for the second scores
        if (i == 0) more = parts.next(p, &next);
      }
      if (!ok) break;
    }
  } else if (warp == LY::kMmaWarp) {
    // ---------------------------------------------------------- products
    const uint32_t base = __shfl_sync(kFull, tmem, 0);
    const uint32_t q_lo = (uint32_t)sw128_desc(sm_q);
    const uint32_t k_lo = (uint32_t)sw128_desc(sm_stage);
    const uint32_t v_lo = (uint32_t)sw128_mn_desc(sm_stage + LY::kValueAt, kAtom);
    auto desc = [&](uint32_t hi, uint32_t lo) { return (uint64_t)hi << 32 | lo; };
    int stage0 = 0;
    unsigned tiles = 0, scored = 0;  // tiles so far: 16 bits for each query tile
    bool ok = true;
    Part next;
    bool more = parts.next(p, &next);
#pragma unroll 1
    while (ok && more) {
      x = next;
      const int two = __shfl_sync(kFull, x.toks[1] > 0 ? 1 : 0, 0);
      const int count = __shfl_sync(kFull, x.steps, 0) << two;  // of scores
      if (count == 0) more = parts.next(p, &next);
      // Scores three ahead of results (of one tile alone no more steps than there are
      // stages), each of them in one place of the code.  The buffer that scores go to
      // held the weights of the products issued just before.
      const int ahead = two || kStages >= kBuffers ? kBuffers : kStages;
#pragma unroll 1
      for (int n = -ahead; n < count && ok; ++n) {
        if (n == 0) more = parts.next(p, &next);  // under the first softmax
        if (n >= 0) {
          const int t = n & two, i = n >> two, s = (stage0 + i) % kStages;
          const unsigned buf = (scored + n) % kBuffers, phase = (scored + n) / kBuffers & 1;
          const uint32_t vd = v_lo + (uint32_t)s * (LY::kStage / 16);
          const uint32_t o_at = base + LY::kResult + t * kHead;
#pragma unroll 1
          for (int half = 0; half < 2; ++half) {
            if (!(ok = wait(&p_full[buf][half], phase))) break;
            tc_fence_after();
            if (elect_one()) {
#pragma unroll
              for (int k = 0; k < 4; ++k)
                umma_f16_ts(o_at, base + buf * kTokens + half * 32 + 8 * k,
                            desc(kHi128, vd + (half * 4 + k) * (16 * 128 / 16)),
                            idesc<T>(kHead, true), i != 0 || half + k != 0);
              if (half) {
                umma_commit(&o_full[t]);
                if (t == two) umma_commit(&empty[s]);
                if (n + 1 + two - t >= count) umma_commit(&o_done[t]);
              }
            }
            __syncwarp();
          }
          if (!ok) break;
        }
        if (n + ahead < count) {
          const int e = n + ahead, t = e & two, i = e >> two, s = stage0 + i;
          const unsigned buf = (scored + e) % kBuffers;
          if (i == 0) {
            if (!(ok = wait(&q_full[t], tiles >> (16 * t) & 1))) break;
            tiles = t ? tiles + 0x10000u : (tiles & 0xFFFF0000u) | ((tiles + 1) & 0xFFFFu);
          }
          if (!(ok = wait(&full[s % kStages], (s / kStages) & 1))) break;
          tc_fence_after();
          const uint32_t kd = k_lo + (uint32_t)(s % kStages) * (LY::kStage / 16);
          const uint32_t qd = q_lo + t * (LY::kQuery / 16), to = base + buf * kTokens;
          if (elect_one()) {
#pragma unroll
            for (int half = 0; half < 2; ++half)
#pragma unroll
              for (int k = 0; k < kHead / 16; ++k)
                umma_f16(to, desc(kHi128, qd + k * 2),
                         desc(kHi128, kd + (half * kAtom + k * 32) / 16), idesc<T>(kTokens, false),
                         half + k != 0);
            constexpr uint32_t kHi = ROPE == 64 ? kHi128 : kHi64;
#pragma unroll
            for (int k = 0; k < ROPE / 16; ++k)
              umma_f16(to, desc(kHi, qd + (kAtom + k * 32) / 16),
                       desc(kHi, kd + (LY::kRopeAt + k * 32) / 16), idesc<T>(kTokens, false), 1);
            umma_commit(&s_full[buf]);
          }
          __syncwarp();
        }
      }
      stage0 += count >> two;
      scored += count;
    }
    // whatever happened, nothing is in flight when tensor memory is given back
    if (elect_one()) umma_commit(&drained);
    __syncwarp();
    mbar_wait(&drained, 0, kProbes);
  } else {
    // -------------------------------------- keys and values, positional parts from pages
    const int piece = min(1 << p.page_shift, kTokens), pieces = kTokens / piece;
    const int my_tok = lane % pieces * piece;
    int s = 0;  // stages so far
    // With no probes at all the block gives up here: nothing comes, and everybody's
    // waits run out.
    bool ok = p.probes > 0;
#pragma unroll 1
    while (ok && parts.next(p, &x)) {
      const int last = (x.len - 1) >> p.page_shift;
      auto row_at = [&](int i) {  // of this lane's piece of step i
        const int tok = (x.step0 + i) * kTokens + my_tok;
        const int at = min(tok >> p.page_shift, last);  // past the end: the last page again
        return min(max(__ldg(p.table + x.r * p.width + at), 0), (int)p.pages - 1) << p.page_shift;
      };
      int at = x.steps > 0 ? row_at(0) : 0;
      const int room = p.room[x.r];
#pragma unroll 1
      for (int i = 0; i < x.steps; ++i, ++s) {
        const int st = s % kStages, to_row = at;
        if (i + 1 < x.steps) at = row_at(i + 1);
        if (s >= kStages && !(ok = wait(&empty[st], (s / kStages - 1) & 1))) break;
        unsigned char* to = sm_stage + st * LY::kStage;
        if (lane == 0) mbar_arrive_expect_tx(&full[st], LY::kStage);
        __syncwarp();
        // keys and values 64 tokens at a time, as they were expanded; past those the same
        // again: what lies there was never written, or by others
        const int half = lane & 1, tok = (x.step0 + i) * kTokens;
        const int row = room + tok + (half && tok + 64 < x.len ? 64 : 0);
        if (lane < 4)
          tma_load(to + (lane >> 1) * kAtom + half * (kAtom / 2), &maps.keys, (lane >> 1) * 64, row,
                   x.g, &full[st]);
        else if (lane < 6)
          tma_load(to + LY::kValueAt + half * (kAtom / 2), &maps.values, 0, row, x.g, &full[st]);
        if (lane < pieces)
          tma_load(to + LY::kRopeAt + my_tok * ROPE * 2, &maps.rope, p.latent, to_row, &full[st]);
      }
    }
    // no copy is in flight when the block ends, whatever happened
    for (int i = max(s - kStages, 0); i < s; ++i)
      mbar_wait(&full[i % kStages], (i / kStages) & 1, kProbes);
  }

  __syncwarp();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == LY::kMmaWarp) tmem_dealloc(tmem, kTmemCols);
  if (sh_fail) {
    if (warp < LY::kSoftWarps) lose_rows<ROPE>(p, hd, worker);
    if (threadIdx.x == 0) atomicOr(p.status, GRM_B200_PLAN_WAIT);
  }
}

template <typename T, int ROPE>
int launch(const Params& p, cudaStream_t st) {
  using LY = Layout<ROPE>;
  Maps maps;
  const int64_t width = p.latent + p.rope;
  const int64_t cache[2] = {width, p.pages << p.page_shift};
  const int64_t keys[3] = {2 * kHead, p.expand_tokens, p.heads};
  const int64_t k_strides[2] = {2 * kHead, 2 * kHead * p.expand_tokens};
  const int64_t values[3] = {kHead, p.expand_tokens, p.heads};
  const int64_t v_strides[2] = {kHead, kHead * p.expand_tokens};
  const int rope[2] = {ROPE, 1 << p.page_shift}, tile[3] = {64, 64, 1};
  int rc;
  if ((rc = make_map(&maps.rope, p.cache, 2, cache, &width, rope)) ||
      (rc = make_map(&maps.keys, p.keys, 3, keys, k_strides, tile)) ||
      (rc = make_map(&maps.values, p.values, 3, values, v_strides, tile)))
    return rc;
  auto kernel = prompt_kernel<T, ROPE>;
  static std::atomic<uint64_t> done{0};
  if ((rc = paged::allow_shared(reinterpret_cast<const void*>(kernel), LY::kSmem, &done)))
    return rc;
  kernel<<<(unsigned)p.v.tiling.workers, LY::kThreads, LY::kSmem, st>>>(maps, p);
  if ((rc = paged::launch_status("latent attend"))) return rc;
  return launch_join<T, kHead, 1, kRows * kQ, true>(p, st);
}

template <int ROPE>
int launch_kind(const Params& p, cudaStream_t st) {
  return p.dtype == GRM_B200_F16 ? launch<__half, ROPE>(p, st) : launch<__nv_bfloat16, ROPE>(p, st);
}

}  // namespace

int launch_prompt(const Params& p, cudaStream_t st) {
  return p.rope == 32 ? launch_kind<32>(p, st) : launch_kind<64>(p, st);
}

}  // namespace latent
}  // namespace grm_b200
