// latent_attend.cu -- latent attention over pages of rows (c_t, r_t), both forms.
//
// With y_t = scale * log2(e) * (q . k_t) and the reference exponent m of a row,
//   p_t = 2^(y_t - m),  out = sum_t p_t v_t / sum_t p_t,  lse = ln 2 (m + log2 sum_t p_t).
// Absorbed: k_t = (c_t, r_t) and v_t = c_t, the same for all heads, so that a tile of
// 128 rows is several heads of a few tokens and one copy of a token's row serves its
// keys and its values.  Expanded: k_t and v_t are one head's (latent_expand.cu has made
// them), and a block takes 2 x 128 tokens of it.  There k_t is held as two numbers of
// the arena's type, the rounded key and what that left over, and multiplied twice:
// with the first alone a score is off by 2^-9 of its products' size, which the log-sum
// of a row of few tokens shows (1e-3 of it).  Values are rounded to the type, as
// weights are, since products take no wider operands and a second number of either would
// double the second products; a row is divided by the sum of its rounded weights, so that
// what they share is not off, and its log-sum is that of the exact ones.  Root mean square
// against 64 bits, beside fp32 arithmetic rounded once: absorbed 2.1e-3 and 1.7e-3 (bf16),
// expanded 1.8e-3 and 1.7e-3, 3.2e-4 and 2.1e-4 (fp16); the log-sum is off by 4e-6 at most.
//
// A block's warps:
//   4 a query tile  softmax, one row a thread: 64 scores from tensor memory, weights back
//                   over them in the arena's type, and when a row's reference exponent
//                   has to move (rarely: it trails by up to 8), its result rescaled
//   1 a query tile  its products, issued by one elected lane: S = Q K^T, O += P V
//   1               rows from their pages to shared memory by tensor-map copies, 64
//                   tokens a stage, as many stages as there is room for
// Scores are in two buffers of 64 tokens, so that products run under a softmax.
// Queries are in tensor memory where there is room beside scores and results, so that
// the products read keys and values alone from shared memory.  A result of 512 values
// would take all of tensor memory: two blocks take 256 values each there and both
// work out the scores.
//
// Work is shared by units (latent.cuh): a worker goes from tile to tile, its copies
// running ahead over their borders, and leaves parts of the tiles at its ends for
// join_kernel.
//
// Absorbed, a step of 64 tokens (40 heads of 256 + 32, one row) takes 0.66 to 0.87 us, up to
// 8 TB/s of all SMs: its copies and its products are about level.  64 requests of 32 to 16,384
// tokens (147 MB, 22.5 us at a copy's rate) take 42 us: 32 in this kernel's blocks, 5.5 of
// them a tile's start and end, then 5 in join_kernel and two launches.
// Expanded, heads of 64 + 32: 28 products for 64 tokens of both query tiles, 64 clocks each
// at least, are 1,792 of a step's 1,845 clocks, with the softmax of one tile under the products
// of the other; 8,449 rows on 31,000 tokens, 40 heads, take 1.5 ms, 0.7 PFLOP/s (keys count
// once).  Before the softmax warps' places left their registers it was they, 2,075 clocks, of
// which a warp's exponentials, their sums and roundings take 900, in turns.  Tried then (not
// since the products are the limit), and no faster: scores of 96 or 128 tokens at a time (a
// product with both operands in shared memory takes 100 clocks at 128 columns), keys and what
// they left over side by side in one product of 128 columns, the sum left to the softmax (2.25
// ms in all against 1.95), two threads a row (3.36 ms: 96 registers are too few).
//
// Tokens that a row does not see have weight 0, and a product of 0 and what is no
// number would be none: where a hidden token's score is not finite, the numbers of
// its values that are not are set to 0 in shared memory before the weights go out
// (scrub).  Rows of the tile that do see the token are told: a score of -inf has weight
// 0, and 0 times what was there is no number.
#include <algorithm>
#include <climits>
#include <type_traits>

#include "latent_device.cuh"

namespace grm_b200 {
namespace latent {

namespace {

using paged::ex2;
using paged::kLazy;
using paged::kProbes;
using paged::reference_of;

constexpr int kAtom = kStep * 128;       // 64 tokens x 64 values
constexpr int kQueryAtom = kRows * 128;  // 128 rows x 64 values
constexpr uint32_t kTmemCols = 512;
constexpr int kShared = 232448 - 1024;   // dynamic shared memory beside the barriers
constexpr float kBlind = -3.402823466e38f;

template <int MAIN, int ROPE, bool EXP>
struct Layout {
  static constexpr int kQueries = EXP ? 2 : 1;
  static constexpr int kV = EXP || MAIN <= 256 ? MAIN : 256;  // values of a block's results
  static constexpr int kSplits = MAIN / kV;
  static constexpr int kAtoms = MAIN / 64;
  static constexpr int kKeyAtoms = EXP ? 2 * kAtoms : kAtoms;
  // a stage: keys, positional part, values where they are not the keys
  static constexpr int kRopeAt = kKeyAtoms * kAtom;
  static constexpr int kRopeBytes = kStep * ROPE * 2;
  static constexpr int kValueAt = EXP ? kRopeAt + kRopeBytes : 0;
  static constexpr int kStage = kRopeAt + kRopeBytes + (EXP ? kAtoms * kAtom : 0);
  // tensor memory: scores, results, and queries in what is left
  static constexpr int kFree = (int)kTmemCols - kQueries * (2 * kStep + kV);
  static constexpr int kQTmem =
      kFree / kQueries * 2 >= MAIN ? MAIN : kFree / kQueries * 2 / 64 * 64;
  static constexpr uint32_t kScore = 0;
  static constexpr uint32_t kResult = kQueries * 2 * kStep;
  static constexpr uint32_t kQueryCol = kResult + kQueries * kV;
  // the rest of the queries in shared memory, the positional part last
  static constexpr int kQRopeAt = (MAIN - kQTmem) / 64 * kQueryAtom;
  static constexpr int kQuery = kQRopeAt + kRows * ROPE * 2;
  static constexpr int kWalks = EXP ? 1536 : 0;  // shared memory of the softmax warps' places
  static constexpr int kFit = (kShared - kWalks - 1024 - kQueries * kQuery) / kStage;
  static constexpr int kStages = kFit > 8 ? 8 : kFit;
  static constexpr int kUsed = 1024 + kQueries * kQuery + kStages * kStage;
  // one block an SM: it owns all of tensor memory
  static constexpr int kSmem = kUsed > 120 * 1024 ? kUsed : 120 * 1024;
  static constexpr int kSoftWarps = 4 * kQueries;
  static constexpr int kMmaWarp = kSoftWarps;
  static constexpr int kLoadWarp = kMmaWarp + kQueries;
  static constexpr int kThreads = (kLoadWarp + 1) * 32;
  static constexpr int kSlot = slot_floats(kRows * kQueries, kV);
  static_assert(kQueryCol + kQueries * kQTmem / 2 <= kTmemCols && kStages >= 2, "tiles");
  static_assert(kQTmem % 256 == 0 || kQTmem == MAIN, "queries come 256 values at a time");
};

// fp32 accumulators, 16-bit operands, 128 rows, n columns; B K-major or (b_mn) not.
template <typename T>
__host__ __device__ constexpr uint32_t idesc(int n, bool b_mn) {
  return (1u << 4) | Kind<T>::kFormat | (b_mn ? 1u << 16 : 0u) | ((uint32_t)(n >> 3) << 17) |
         ((uint32_t)(kRows >> 4) << 24);
}

// The scores of a step from the first hidden one on set to -inf, in tensor memory;
// returns the hidden tokens whose score was no finite number.  A step of its own, few
// instructions in a loop: unrolled into the softmax it took 5 us the first time a
// block came by, on instructions that were not in its cache.
__device__ __forceinline__ unsigned long long hide(uint32_t scores, int seen) {
  unsigned long long bad = 0;
#pragma unroll 1
  for (int c = 0; c < kStep; c += 16) {
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
    bad |= (unsigned long long)b << c;
  }
  tmem_wait_st();
  return bad;
}

// Numbers that are none among the V values of some tokens of a stage set to 0; returns
// the first token that had one (kStep: none).
template <typename T, int V>
__device__ __noinline__ int scrub(unsigned char* values, unsigned long long tokens) {
  int first = kStep;
  while (tokens) {
    const int t = __ffsll((long long)tokens) - 1;
    tokens &= tokens - 1;
    for (int c = 0; c < V / 8; ++c) {
      uint4* at = reinterpret_cast<uint4*>(values + (c / 8) * kAtom + atom_byte(t, c % 8));
      const uint4 v = *at;
      uint32_t x[4] = {v.x, v.y, v.z, v.w};
      bool bad = false;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t e = Kind<T>::kNoNumber;
        if ((x[i] & e) == e) { x[i] &= 0xFFFF0000u; bad = true; }
        if ((x[i] >> 16 & e) == e) { x[i] &= 0x0000FFFFu; bad = true; }
      }
      if (bad) {
        *at = make_uint4(x[0], x[1], x[2], x[3]);
        first = min(first, t);
      }
    }
  }
  return first;
}

// The rows of a worker in which a wait gave up: no numbers.
template <int MAIN, int ROPE, bool EXP>
__device__ __noinline__ void lose_rows(const Params& p, const Header& hd, int worker, int split) {
  using LY = Layout<MAIN, ROPE, EXP>;
  const float nan = __int_as_float(0x7FC00000);
  const int t = threadIdx.x >> 7, row = threadIdx.x & 127;
  Parts<LY::kQueries> parts(p, hd, worker, p.l.start[worker], p.l.start[worker + 1].u);
  Part x;
  while (parts.next(p, &x)) {
    const Row a = row_of<EXP>(p, x, t, row);
    if (x.slot >= 0) {
      float* slot = p.l.part + ((int64_t)x.slot * LY::kSplits + split) * LY::kSlot;
      *reinterpret_cast<float4*>(slot + kRows * LY::kQueries * LY::kV + 4 * (t * kRows + row)) =
          make_float4(-INFINITY, nan, nan, kSees);
    } else if (a.active) {
      const int64_t orow = (int64_t)(x.start + a.token) * p.heads + a.head;
      for (int c = 0; c < LY::kV / 8; ++c)
        reinterpret_cast<uint4*>(p.out + orow * MAIN + split * LY::kV)[c] =
            make_uint4(0x7FFF7FFFu, 0x7FFF7FFFu, 0x7FFF7FFFu, 0x7FFF7FFFu);
      if (p.lse && split == 0) p.lse[orow] = nan;
    }
  }
}

struct Maps {
  CUtensorMap main;    // absorbed: 64 values of rows of the cache; expanded: of its keys
  CUtensorMap rope;    // the positional part of rows of the cache
  CUtensorMap values;  // expanded: 64 values of its values
};

template <typename T, int MAIN, int ROPE, bool EXP>
__global__ void __launch_bounds__(Layout<MAIN, ROPE, EXP>::kThreads, 1)
    attend_kernel(const __grid_constant__ Maps maps, const __grid_constant__ Params p) {
  using LY = Layout<MAIN, ROPE, EXP>;
  constexpr int kStages = LY::kStages, kQ = LY::kQueries;
  extern __shared__ unsigned char raw[];
  unsigned char* const sm = raw + ((1024u - (smem_u32(raw) & 1023u)) & 1023u);
  unsigned char* const sm_q = sm;                         // [kQ]
  unsigned char* const sm_stage = sm + kQ * LY::kQuery;   // [kStages]
  __shared__ __align__(8) uint64_t full[kStages], empty[kStages], q_full[kQ], drained[kQ],
      s_full[kQ][2], p_full[kQ][2], o_full[kQ], o_done[kQ], turn[kQ][4];
  __shared__ uint32_t sh_tmem;
  __shared__ int sh_fail;
  // Where the expanded form's softmax warps are, and their next part: in registers it is
  // what their loop lacks (8,449 rows on 31,000 tokens: 1.86 ms, 1.72 from here).
  struct Place {
    Parts<kQ> parts;
    Part next;
    bool more;
  };
  constexpr int kPlace = EXP ? (sizeof(Place) + 15) / 16 * 16 : 16;
  static_assert(!EXP || kPlace * LY::kSoftWarps <= LY::kWalks, "places");
  __shared__ __align__(16) unsigned char sh_place[LY::kSoftWarps][kPlace];
  // First token of which each softmax warp took numbers out, in this tile and the one before.
  // (Expanded, a token whose values are none has no score either.)
  __shared__ int sh_scrubbed[2][4];

  const int worker = blockIdx.x / LY::kSplits, split = blockIdx.x % LY::kSplits;
  const Start begin = p.l.start[worker];  // on their way beside the header
  const int64_t until = p.l.start[worker + 1].u;
  const Header hd = *p.l.header;
  asm volatile("griddepcontrol.launch_dependents;");
  if (worker >= hd.workers) return;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (EXP && hd.lost) {
    if (warp < LY::kSoftWarps) lose_rows<MAIN, ROPE, EXP>(p, hd, worker, split);
    return;
  }
  if (threadIdx.x == 0) {
    for (int i = 0; i < kStages; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], kQ);
    }
    for (int t = 0; t < kQ; ++t) {
      mbar_init(&q_full[t], 4);
      mbar_init(&drained[t], 1);
      mbar_init(&o_full[t], 1);
      mbar_init(&o_done[t], 1);
      for (int x = 0; x < 2; ++x) {
        mbar_init(&s_full[t][x], 1);
        mbar_init(&p_full[t][x], 4);
      }
      for (int x = 0; x < 4; ++x) mbar_init(&turn[t][x], 1);
    }
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
  Parts<kQ> parts(p, hd, worker, begin, until);
  Part x;

  if (warp < LY::kSoftWarps) {
    // ------------------------------------------------------------- softmax
    const int t = warp >> 2, row = (warp & 3) * 32 + lane;
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t s_col = tmem + lanes + LY::kScore + t * 2 * kStep;
    const uint32_t o_col = tmem + lanes + LY::kResult + t * LY::kV;
    const uint32_t q_col = tmem + lanes + LY::kQueryCol + t * (LY::kQTmem / 2);
    unsigned char* const my_q = sm_q + t * LY::kQuery;
    bool ok = true;
    int it = 0, tile = 0, stage0 = 0;  // steps and tiles of this query tile; stages so far
    int turns = 0;  // steps of both query tiles so far
    // the row's query of a part, to tensor memory and shared memory
    auto queries = [&](const Part& y) {
      const Row b = row_of<EXP>(p, y, t, row);
      const uint16_t* qp = p.q + (int64_t)(y.start + b.token) * p.q_row + b.head * p.q_head;
      const uint16_t* rp = p.qr + (int64_t)(y.start + b.token) * p.qr_row + b.head * p.qr_head;
      auto chunk = [&](const uint16_t* from, int c) {
        return b.active ? __ldg(reinterpret_cast<const uint4*>(from) + c)
                        : make_uint4(0, 0, 0, 0);
      };
      // All loads in flight (of a latent of 512 half of them): in batches of sixteen, the
      // positional part after them, it was three trips to memory, 1.5 us more of a tile's start.
      constexpr int kBatch = MAIN / 8 < 32 ? MAIN / 8 : 32;
      uint4 positional[ROPE / 8];
#pragma unroll
      for (int c = 0; c < ROPE / 8; ++c) positional[c] = chunk(rp, c);
#pragma unroll 1
      for (int c = 0; c < MAIN / 8; c += kBatch) {
        uint4 v[kBatch];
#pragma unroll
        for (int i = 0; i < kBatch; ++i) v[i] = chunk(qp, c + i);
        if (c < LY::kQTmem / 8) {
#pragma unroll
          for (int i = 0; i < kBatch; i += 4) {
            const uint32_t w[16] = {v[i].x, v[i].y, v[i].z, v[i].w, v[i + 1].x, v[i + 1].y,
                                    v[i + 1].z, v[i + 1].w, v[i + 2].x, v[i + 2].y, v[i + 2].z,
                                    v[i + 2].w, v[i + 3].x, v[i + 3].y, v[i + 3].z, v[i + 3].w};
            tmem_st16(q_col + 4 * (c + i), w);
          }
        } else {
#pragma unroll
          for (int i = 0; i < kBatch; ++i) {
            const int z = c + i - LY::kQTmem / 8;
            *reinterpret_cast<uint4*>(my_q + (z / 8) * kQueryAtom + atom_byte(row, z % 8)) = v[i];
          }
        }
      }
#pragma unroll
      for (int c = 0; c < ROPE / 8; ++c)
        *reinterpret_cast<uint4*>(my_q + LY::kQRopeAt + (ROPE == 64 ? atom_byte(row, c)
                                                                    : half_atom_byte(row, c))) =
            positional[c];
      tmem_wait_st();
      tc_fence_before();
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(&q_full[t]);
    };
    Part own;
    Place* const place = reinterpret_cast<Place*>(sh_place[warp]);
    Part& next = EXP ? place->next : own;
    if (EXP && lane == 0) place->parts = parts;
    auto advance = [&] {
      if (!EXP) return parts.next(p, &own);
      __syncwarp();  // what is there has been read
      if (lane == 0) place->more = place->parts.next(p, &place->next);
      __syncwarp();
      return place->more;
    };
    bool more = advance(), held = false;  // held: a tile whose result is to go out
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
        if (!EXP && steps > 0) {  // (tile was counted above)
          const int* first = sh_scrubbed[(tile - 1) & 1];
          if (seen_by(p, x, a.token) > min(min(first[0], first[1]), min(first[2], first[3])))
            lr = __int_as_float(0x7FC00000);  // the row sees what is no number
        }
        const bool sees = m != kBlind || lr != 0.0f;
        if (x.slot >= 0) {  // a part's result, for join_kernel
          float* slot = p.l.part + ((int64_t)x.slot * LY::kSplits + split) * LY::kSlot;
          float4* to = reinterpret_cast<float4*>(slot + (t * kRows + row) * LY::kV);
          if (steps > 0 && !idle)
#pragma unroll 1
            for (int c = 0; c < LY::kV / 32; ++c) {
              uint32_t o[32];
              tmem_ld32_nowait(o_col + 32 * c, o);
              tmem_wait_ld32(o);
              if (a.active)
#pragma unroll
                for (int k = 0; k < 8; ++k)
                  to[8 * c + k] =
                      make_float4(__uint_as_float(o[4 * k]), __uint_as_float(o[4 * k + 1]),
                                  __uint_as_float(o[4 * k + 2]), __uint_as_float(o[4 * k + 3]));
            }
          if (a.active)
            *reinterpret_cast<float4*>(slot + kRows * kQ * LY::kV + 4 * (t * kRows + row)) =
                make_float4(m, l, lr, steps == 0 ? kNoResult : sees ? kSees : kSeesNothing);
        } else if (!idle) {
          const float inv = lr == 0.0f ? __int_as_float(0x7FC00000) : 1.0f / lr;
          uint16_t* out = p.out + orow * MAIN + split * LY::kV;
#pragma unroll 1
          for (int c = 0; c < LY::kV / 32; ++c) {
            uint32_t o[32];
            if (steps > 0) {
              tmem_ld32_nowait(o_col + 32 * c, o);
              tmem_wait_ld32(o);
            }
            if (a.active)
#pragma unroll
              for (int k = 0; k < 4; ++k) {
                uint32_t w[4];
#pragma unroll
                for (int y = 0; y < 4; ++y)
                  w[y] = sees ? Kind<T>::pack(__uint_as_float(o[8 * k + 2 * y]) * inv,
                                              __uint_as_float(o[8 * k + 2 * y + 1]) * inv)
                              : 0u;
                reinterpret_cast<uint4*>(out)[4 * c + k] = make_uint4(w[0], w[1], w[2], w[3]);
              }
          }
          if (a.active && p.lse && split == 0)
            p.lse[orow] = l == 0.0f ? -INFINITY
                                    : (m - Kind<T>::kLift + log2f(l)) * 0.693147180559945309f;
        }
        // what the next tile's products overwrite has been read
        tc_fence_before();
      }
      if (!more) break;
      x = next;
      steps = x.steps;
      const int stage_base = stage0;
      stage0 += steps;
      held = x.toks[t] > 0;
      if (!held || steps == 0) more = advance();
      if (!held) continue;
      a = row_of<EXP>(p, x, t, row);
      // tokens that the row sees, from the part's first on
      const int lim = seen_by(p, x, a.token) - x.step0 * kStep;
      // A row that sees none of the part's tokens keeps a reference exponent that says so (a
      // flag costs the expanded form's loop a register, 1 % of its time).
      m = lim > 0 ? -INFINITY : kBlind;
      l = lr = 0.0f;
      idle = !__any_sync(kFull, a.active);
      if (!EXP && steps > 0) {
        if (lane == 0) sh_scrubbed[tile & 1][warp] = INT_MAX;
        __syncwarp();
      }
#pragma unroll 1
      for (int i = 0; i < steps; ++i, ++it) {
        const int buf = it & 1;
        if (!(ok = wait(&s_full[t][buf], (it >> 1) & 1))) break;
        tc_fence_after();
        // The two softmax warps of a scheduler take turns at the exponentials, so that one's
        // other work lies under them (left to themselves they do both in step).
        const bool two = kQ == 2 && x.toks[kQ - 1] > 0;
        auto my_turn = [&] {
          const bool go = t == 1 || turns > 0 ? wait(&turn[t][warp & 3], (turns - 1 + t) & 1) : true;
          ++turns;
          return go;
        };
        auto your_turn = [&] {
          if (lane == 0) mbar_arrive(&turn[kQ - 1 - t][warp & 3]);
        };
        if (idle) {
          if (lane == 0) mbar_arrive(&p_full[t][buf]);
          if (i == 0) more = advance();
          if (two) {
            if (!(ok = my_turn())) break;
            your_turn();
          }
          continue;
        }
        if (__any_sync(kFull, (i + 1) * kStep > lim)) {
          const unsigned long long bad = hide(s_col + buf * kStep, lim - i * kStep);
          if (__any_sync(kFull, bad != 0)) {
            const int st = stage_base + i;  // its copies landed before the scores were there
            if (!(ok = wait(&full[st % kStages], (st / kStages) & 1))) break;
            const int first = scrub<T, LY::kV>(sm_stage + st % kStages * LY::kStage +
                                                   LY::kValueAt + split * (LY::kV / 64) * kAtom,
                                               bad);
            if (!EXP && first < kStep)
              atomicMin(&sh_scrubbed[tile & 1][warp], (x.step0 + i) * kStep + first);
            fence_proxy_async_smem();
          }
        }
        uint32_t v[2][32];
        tmem_ld32_nowait(s_col + buf * kStep, v[0]);
        tmem_ld32_nowait(s_col + buf * kStep + 32, v[1]);
        tmem_wait_ld32(v[0]);
        tmem_wait_ld32(v[1]);
        float tops[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};  // chains side by side
#pragma unroll
        for (int k = 0; k < kStep; k += 2)
          tops[k / 2 % 4] = max3(tops[k / 2 % 4], __uint_as_float(v[k / 32][k % 32]),
                                 __uint_as_float(v[k / 32][k % 32 + 1]));
        const float top = fmaxf(max3(tops[0], tops[1], tops[2]), tops[3]) * p.scale_log2;
        if (__any_sync(kFull, top > m + kLazy)) {
          const float next = top > m + kLazy ? reference_of(top) : m;
          const float f = next == m ? 1.0f : ex2(m - next);
          m = next;
          l *= f;
          lr *= f;
          if (i > 0) {  // once the products of the step before have ended
            if (!(ok = wait(&o_full[t], (it - 1) & 1))) break;
            tc_fence_after();
#pragma unroll 1
            for (int c = 0; c < LY::kV / 16; ++c) {
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
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          uint32_t w[16];
#pragma unroll
          for (int k = 0; k < 32; k += 2) {
            const float2 y = fma2(__uint_as_float(v[c][k]), __uint_as_float(v[c][k + 1]),
                                  p.scale_log2, off);
            const float2 e = make_float2(ex2(y.x), ex2(y.y));
            sum = add2(sum, e);
            w[k / 2] = Kind<T>::pack(e.x, e.y);
            rounded = add2(rounded, Kind<T>::widen(w[k / 2]));
            // three quarters done: the other's first ones fill the gaps of the last
            if (c == 1 && k == 14 && two) your_turn();
          }
          tmem_st16(s_col + buf * kStep + 16 * c, w);
        }
        l += sum.x + sum.y;
        lr += rounded.x + rounded.y;
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_full[t][buf]);
        // a chain of loads that lies under the wait for the second scores
        if (i == 0) more = advance();
      }
      if (!ok) break;
    }
  } else if (warp < LY::kLoadWarp) {
    // ---------------------------------------------------------- products
    // The whole warp runs this, an elected lane issues; what the instructions read is
    // the same in every lane and known to be (broadcast), so that it stays in uniform
    // registers.
    const int t = __shfl_sync(kFull, warp, 0) - LY::kMmaWarp;
    const uint32_t base = __shfl_sync(kFull, tmem, 0);
    const uint32_t s_at = base + LY::kScore + t * 2 * kStep;
    const uint32_t o_at = base + LY::kResult + t * LY::kV;
    const uint32_t q_at = base + LY::kQueryCol + t * (LY::kQTmem / 2);
    const uint32_t q_lo = (uint32_t)sw128_desc(sm_q + t * LY::kQuery);
    const uint32_t k_lo = (uint32_t)sw128_desc(sm_stage);
    const uint32_t v_lo = (uint32_t)sw128_mn_desc(
        sm_stage + LY::kValueAt + split * (LY::kV / 64) * kAtom, kAtom);
    auto desc = [&](uint32_t hi, uint32_t lo) { return (uint64_t)hi << 32 | lo; };
    int it = 0, tile = 0, stage0 = 0;
    bool ok = true;
    auto scores = [&](int i) {  // of the it + i-th step, in the stage of the part's i-th
      const uint32_t kd = k_lo + (uint32_t)((stage0 + i) % kStages) * (LY::kStage / 16);
      const uint32_t to = s_at + ((it + i) & 1) * kStep;
      if (elect_one()) {
#pragma unroll
        for (int part = 0; part < LY::kKeyAtoms / LY::kAtoms; ++part)
#pragma unroll
          for (int k = 0; k < MAIN / 16; ++k) {
            const uint32_t k_step = ((part * LY::kAtoms + k / 4) * kAtom + (k % 4) * 32) / 16;
            if (16 * k < LY::kQTmem) {
              umma_f16_ts(to, q_at + 8 * k, desc(kHi128, kd + k_step), idesc<T>(kStep, false),
                          part + k != 0);
            } else {
              const int y = k - LY::kQTmem / 16;
              umma_f16(to, desc(kHi128, q_lo + ((y / 4) * kQueryAtom + (y % 4) * 32) / 16),
                       desc(kHi128, kd + k_step), idesc<T>(kStep, false), part + k != 0);
            }
          }
#pragma unroll
        for (int k = 0; k < ROPE / 16; ++k) {
          constexpr uint32_t kHi = ROPE == 64 ? kHi128 : kHi64;
          umma_f16(to, desc(kHi, q_lo + (LY::kQRopeAt + k * 32) / 16),
                   desc(kHi, kd + (LY::kRopeAt + k * 32) / 16), idesc<T>(kStep, false), 1);
        }
        umma_commit(&s_full[t][(it + i) & 1]);
      }
      __syncwarp();
    };
    auto next_scores = [&](int i) {
      const int s = stage0 + i;
      if (!wait(&full[s % kStages], (s / kStages) & 1)) return false;
      tc_fence_after();
      scores(i);
      return true;
    };
    Part next;
    bool more = parts.next(p, &next);
#pragma unroll 1
    while (ok && more) {
      x = next;
      const int steps = __shfl_sync(kFull, x.steps, 0);
      if (x.toks[t] == 0 || steps == 0) more = parts.next(p, &next);
      if (x.toks[t] == 0) {  // nothing to do for this one: give the stages back
#pragma unroll 1
        for (int i = 0; i < steps && ok; ++i) {
          const int s = stage0 + i;
          ok = wait(&full[s % kStages], (s / kStages) & 1);
          if (ok && lane == 0) mbar_arrive(&empty[s % kStages]);
          __syncwarp();
        }
        stage0 += steps;
        continue;
      }
      if (steps == 0) continue;
      ok = wait(&q_full[t], tile & 1);
      if (!ok) break;
      tc_fence_after();
      // scores two steps ahead of results, each of them in one place of the code
#pragma unroll 1
      for (int i = -2; i < steps && ok; ++i) {
        if (i == 0) more = parts.next(p, &next);  // under the first softmax
        if (i >= 0) {
          const int s = (stage0 + i) % kStages, buf = (it + i) & 1;
          if (!(ok = wait(&p_full[t][buf], ((it + i) >> 1) & 1))) break;
          tc_fence_after();
          const uint32_t vd = v_lo + (uint32_t)s * (LY::kStage / 16);
          if (elect_one()) {
#pragma unroll
            for (int k = 0; k < kStep / 16; ++k)
              umma_f16_ts(o_at, s_at + buf * kStep + 8 * k, desc(kHi128, vd + k * (16 * 128 / 16)),
                          idesc<T>(LY::kV, true), i != 0 || k != 0);
            umma_commit(&o_full[t]);
            umma_commit(&empty[s]);
            if (i + 1 == steps) umma_commit(&o_done[t]);
          }
          __syncwarp();
        }
        if (i + 2 < steps) ok = next_scores(i + 2);  // in this step's place
      }
      stage0 += steps;
      it += steps;
      ++tile;
    }
    // whatever happened, nothing is in flight when tensor memory is given back
    if (elect_one()) umma_commit(&drained[t]);
    __syncwarp();
    mbar_wait(&drained[t], 0, kProbes);
  } else {
    // ------------------------------------------------ rows from their pages
    const int piece = min(1 << p.page_shift, kStep);  // tokens of one copy
    const int pieces = kStep / piece;
    const int my_tok = lane % pieces * piece;
    int s = 0;  // stages so far
    // With no probes at all the block gives up here: nothing comes, and everybody's
    // waits run out.
    bool ok = p.probes > 0;
#pragma unroll 1
    while (ok && parts.next(p, &x)) {
      const int last = (x.len - 1) >> p.page_shift;
      auto row_at = [&](int i) {  // of this lane's piece of step i
        const int tok = (x.step0 + i) * kStep + my_tok;
        const int at = min(tok >> p.page_shift, last);  // past the end: the last page again
        const int page = min(max(__ldg(p.table + x.r * p.width + at), 0), (int)p.pages - 1);
        return (page << p.page_shift) + (tok & ((1 << p.page_shift) - 1));
      };
      int at = x.steps > 0 ? row_at(0) : 0;
      int64_t room = 0;
      if (EXP) room = (int64_t)x.g * p.expand_tokens + p.room[x.r];
#pragma unroll 1
      for (int i = 0; i < x.steps; ++i, ++s) {
        const int st = s % kStages, to_row = at;
        if (i + 1 < x.steps) at = row_at(i + 1);
        if (s >= kStages && !(ok = wait(&empty[st], (s / kStages - 1) & 1))) break;
        unsigned char* to = sm_stage + st * LY::kStage;
        if (lane == 0) mbar_arrive_expect_tx(&full[st], LY::kStage);
        __syncwarp();
        if (EXP) {
          const int row = (int)(room + (int64_t)(x.step0 + i) * kStep);
          if (lane < LY::kKeyAtoms) tma_load(to + lane * kAtom, &maps.main, lane * 64, row, &full[st]);
          if (lane < LY::kAtoms)
            tma_load(to + LY::kValueAt + lane * kAtom, &maps.values, lane * 64, row, &full[st]);
        } else {
#pragma unroll
          for (int y = lane; y < LY::kAtoms * 4; y += 32) {
            const int atom = y / pieces;
            if (atom < LY::kAtoms)
              tma_load(to + atom * kAtom + my_tok * 128, &maps.main, atom * 64, to_row, &full[st]);
          }
        }
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
    if (warp < LY::kSoftWarps) lose_rows<MAIN, ROPE, EXP>(p, hd, worker, split);
    if (threadIdx.x == 0) atomicOr(p.status, GRM_B200_PLAN_WAIT);
  }
}

template <typename T, int MAIN, int ROPE, bool EXP>
int launch(const Params& p, cudaStream_t st) {
  using LY = Layout<MAIN, ROPE, EXP>;
  Maps maps;
  const int64_t width = p.latent + p.rope, slots = p.pages << p.page_shift;
  const int64_t cache[2] = {width, slots};
  const int tokens = std::min(1 << p.page_shift, kStep);
  const int box[2] = {64, tokens}, rope[2] = {ROPE, tokens}, tile[2] = {64, kStep};
  int rc = make_map(&maps.rope, p.cache, 2, cache, &width, rope);
  if (EXP) {
    const int64_t rows = (int64_t)p.heads * p.expand_tokens;
    const int64_t keys[2] = {2 * MAIN, rows}, values[2] = {MAIN, rows};
    if (rc || (rc = make_map(&maps.main, p.keys, 2, keys, keys, tile)) ||
        (rc = make_map(&maps.values, p.values, 2, values, values, tile)))
      return rc;
  } else {
    if (rc || (rc = make_map(&maps.main, p.cache, 2, cache, &width, box))) return rc;
    maps.values = maps.main;
  }
  auto kernel = attend_kernel<T, MAIN, ROPE, EXP>;
  static std::atomic<uint64_t> done{0};
  if ((rc = paged::allow_shared(reinterpret_cast<const void*>(kernel), LY::kSmem, &done)))
    return rc;
  kernel<<<(unsigned)(p.v.tiling.workers * LY::kSplits), LY::kThreads, LY::kSmem, st>>>(maps, p);
  if ((rc = paged::launch_status("latent attend"))) return rc;
  return launch_join<T, LY::kV, LY::kSplits, kRows * LY::kQueries, EXP>(p, st);
}

template <int MAIN, int ROPE, bool EXP>
int launch_kind(const Params& p, cudaStream_t st) {
  return p.dtype == GRM_B200_F16 ? launch<__half, MAIN, ROPE, EXP>(p, st)
                                 : launch<__nv_bfloat16, MAIN, ROPE, EXP>(p, st);
}

template <int MAIN, bool EXP>
int launch_rope(const Params& p, cudaStream_t st) {
  return p.rope == 32 ? launch_kind<MAIN, 32, EXP>(p, st) : launch_kind<MAIN, 64, EXP>(p, st);
}

}  // namespace

int launch_absorbed(const Params& p, cudaStream_t st) {
  return p.latent == 128   ? launch_rope<128, false>(p, st)
         : p.latent == 256 ? launch_rope<256, false>(p, st)
                           : launch_rope<512, false>(p, st);
}

int launch_expanded(const Params& p, cudaStream_t st) {
  return p.nope == 64 ? launch_rope<64, true>(p, st) : launch_rope<128, true>(p, st);
}

}  // namespace latent
}  // namespace grm_b200
