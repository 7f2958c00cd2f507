// latent_few.cu -- latent attention in the absorbed form for few query rows: decoding over
// a latent of 512, where a request brings a row of each head, up to 32 in all.
//
// The sums are latent_attend.cu's.  There rows are the 128 lanes of the tensor cores'
// products; with few of them most lanes would do nothing, and a latent of 512 needs
// two blocks.  Here tokens are the lanes of the scores and values those of the results:
//   S^T [128 tokens, rows] = K Q^T,   O^T [values, rows] += V^T P^T,
// the same copy of the tokens' rows being K (values of a token side by side) and V^T
// (read the other way).  Results are 128 values of all rows in a lane each, few
// columns, so that there are two of them and one goes out while the next tile is worked
// on.  Bound by HBM: 128 tokens of 512 + 64 values are 147 KB, 6,400 clocks of an SM's
// share, their products about 3,200 (shared memory: 4 KB of rows for each 16 x 128),
// their exponentials 600.  As the next step's rows have to be on their way while this one's
// are worked on, and there is room for 1.4 steps of them, a product waits for its rows: 250,007
// tokens (288 MB, 44 us) of 16 heads take 79 us, 13 of them join_kernel's.
// At latents of 128 and 256 that one is the faster (148 requests of 4,096 tokens, 40
// heads of 256 + 32: 70 us, 102 us with this one), whose products cost as much
// however few their columns are.
//
// A block's warps:
//   0-7   softmax, a token and half of the rows a lane: scores from tensor memory,
//         weights to shared memory.  Reference exponents are the rows', in shared
//         memory; they move (rarely, as they trail by up to 8) when a lane of the eight
//         warps finds a score too far above its row's
//   8-11  queries to shared memory, results out
//   12    products, issued by one elected lane
//   13    rows from their pages to shared memory, 128 values of 128 tokens a place.  The
//         next tokens' scores start on what has come while the weights of these are
//         worked out, and a place is free when the values in it have been added up
#include <algorithm>
#include <climits>

#include "latent_device.cuh"

namespace grm_b200 {
namespace latent {

namespace {

using paged::ex2;
using paged::kLazy;
using paged::kProbes;
using paged::reference_of;

constexpr int kTokens = 128;              // of a step
constexpr int kAtom = kTokens * 128;      // 128 tokens x 64 values
constexpr int kPlace = 2 * kAtom;
constexpr int kRopes = 2;
constexpr uint32_t kTmemCols = 512;
constexpr int kSoftWarps = 8, kOutWarps = 4, kMmaWarp = 12;  // and one that loads
constexpr int kSoftThreads = kSoftWarps * 32;
constexpr int kThreads = 14 * 32;
// What is added to the scores of a row that has no reference exponent yet: far above what
// one may be passed by for every finite score, and -inf for a score of -inf.
constexpr float kNoReference = 3.402823466e38f;

template <int LATENT, int ROPE, int N>
struct Layout {
  static constexpr int kPairs = LATENT / 128;  // places of a step's rows
  static constexpr int kRopeBytes = kTokens * ROPE * 2;
  // queries: 64 values of N rows apiece, the positional part last
  static constexpr int kQRopeAt = LATENT / 64 * N * 128;
  static constexpr int kQuery = kQRopeAt + N * ROPE * 2;
  static constexpr int kWeights = 2 * N * 128;  // 64 tokens of N rows, twice
  static constexpr int kWeightsAt = kQuery, kRopeAt = kWeightsAt + 2 * kWeights;
  static constexpr int kRingAt = kRopeAt + kRopes * kRopeBytes;
  // reference exponents and sums (static): below 6 KB
  static constexpr int kFit = (232448 - 6144 - 1024 - kRingAt) / kPlace;
  static constexpr int kRing = kFit > 8 ? 8 : kFit;
  static constexpr int kSmem = 1024 + kRingAt + kRing * kPlace;
  // places of the next step that can be there while this one's are held
  static constexpr int kPre = kRing - kPairs < kPairs ? kRing - kPairs : kPairs;
  static constexpr uint32_t kScore = 0, kResult = 2 * N;
  static constexpr int kSlot = slot_floats(N, LATENT);
  static_assert(kRing >= kPairs && kResult + 2 * kPairs * N <= kTmemCols && kSmem > 120 * 1024,
                "places");
};

// fp32 accumulators, 16-bit operands, 128 lanes, n columns; A K-major or (a_mn) not.
template <typename T>
__host__ __device__ constexpr uint32_t idesc(int n, bool a_mn) {
  return (1u << 4) | Kind<T>::kFormat | (a_mn ? 1u << 15 : 0u) | ((uint32_t)(n >> 3) << 17) |
         (128u >> 4 << 24);
}

// Whether `yes` holds in one of the softmax warps' threads.
__device__ __forceinline__ bool soft_any(bool yes) {
  unsigned r;
  asm volatile("{\n .reg .pred p, q;\n setp.ne.u32 p, %1, 0;\n"
               " barrier.cta.red.or.pred q, 1, 256, p;\n selp.u32 %0, 1, 0, q;\n}\n"
               : "=r"(r)
               : "r"((unsigned)yes)
               : "memory");
  return r != 0;
}
__device__ __forceinline__ void soft_sync() { asm volatile("bar.sync 1, 256;" ::: "memory"); }
__device__ __forceinline__ bool out_all(bool yes) {
  unsigned r;
  asm volatile("{\n .reg .pred p, q;\n setp.ne.u32 p, %1, 0;\n"
               " barrier.cta.red.and.pred q, 2, 128, p;\n selp.u32 %0, 1, 0, q;\n}\n"
               : "=r"(r)
               : "r"((unsigned)yes)
               : "memory");
  return r != 0;
}
__device__ __forceinline__ void out_sync() { asm volatile("bar.sync 2, 128;" ::: "memory"); }

// Sums over a warp's lanes of v[0..N), kSums<N> of them in a lane: those from
// first_sum<N>(lane) on.  Lanes halve what they hold from step to step, as long as
// that is an even number.
constexpr int halvings(int n) { return n % 2 == 0 && n > 1 ? 1 + halvings(n / 2) : 0; }
template <int N>
constexpr int kHalvings = halvings(N) < 5 ? halvings(N) : 5;
template <int N>
constexpr int kSums = N >> kHalvings<N>;
template <int N>
__device__ __forceinline__ int first_sum(int lane) {
  return (lane >> (5 - kHalvings<N>)) * kSums<N>;
}
template <int N>
__device__ __forceinline__ void sum_lanes(float (&v)[N], int lane) {
#pragma unroll
  for (int step = 0; step < 5; ++step) {
    const int o = 16 >> step;
    if (step < kHalvings<N>) {
      const int n = N >> (step + 1);
      const bool upper = lane & o;
#pragma unroll
      for (int i = 0; i < N / 2; ++i)
        if (i < n) {
          const float keep = upper ? v[n + i] : v[i], give = upper ? v[i] : v[n + i];
          v[i] = keep + __shfl_xor_sync(kFull, give, o);
        }
    } else {
#pragma unroll
      for (int i = 0; i < kSums<N>; ++i) v[i] += __shfl_xor_sync(kFull, v[i], o);
    }
  }
}

// Eight columns of a warp's 32 lanes; valid after a wait.
__device__ __forceinline__ void tmem_ld8_nowait(uint32_t taddr, uint32_t* v) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
               : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]),
                 "=r"(v[6]), "=r"(v[7])
               : "r"(taddr));
}
// A wait for such loads that also orders every use of v after it.
template <int N>
__device__ __forceinline__ void tmem_wait_all(uint32_t (&v)[N]) {
  tmem_wait_ld();
#pragma unroll
  for (int i = 0; i < N; ++i) asm volatile("" : "+r"(v[i]));
}

// The largest of a warp's 32 numbers, those that are none left out.
__device__ __forceinline__ float warp_max(float v) {
  float m;
  asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(m) : "f"(v));
  return m;
}

// Values of row `t` of a step's places that are no numbers, set to 0; whether there were
// any.
template <typename T, int PAIRS, int RING>
__device__ __noinline__ bool scrub(unsigned char* ring, unsigned place0, int t) {
  bool any = false;
  for (int c = 0; c < PAIRS * 16; ++c) {
    unsigned char* place = ring + (place0 + c / 16) % RING * kPlace;
    uint4* at = reinterpret_cast<uint4*>(place + c / 8 % 2 * kAtom + atom_byte(t, c % 8));
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
    any |= bad;
  }
  return any;
}

// The rows of a worker in which a wait gave up: no numbers.
template <int LATENT, int N>
__device__ __noinline__ void lose_rows(const Params& p, const Header& hd, int worker) {
  const float nan = __int_as_float(0x7FC00000);
  Parts<1, kTokens> parts(p, hd, worker, p.l.start[worker], p.l.start[worker + 1].u);
  Part x;
  while (parts.next(p, &x)) {
    const int rows = x.toks[0] * p.heads;
    const int64_t row0 = (int64_t)(x.start + x.tok0) * p.heads;
    for (int n = threadIdx.x; n < rows; n += kSoftThreads) {
      if (x.slot >= 0) {
        float* slot = p.l.part + (int64_t)x.slot * slot_floats(N, LATENT);
        *reinterpret_cast<float4*>(slot + N * LATENT + 4 * n) =
            make_float4(-INFINITY, nan, nan, kSees);
      } else {
        for (int c = 0; c < LATENT / 8; ++c)
          reinterpret_cast<uint4*>(p.out + (row0 + n) * LATENT)[c] =
              make_uint4(0x7FFF7FFFu, 0x7FFF7FFFu, 0x7FFF7FFFu, 0x7FFF7FFFu);
        if (p.lse) p.lse[row0 + n] = nan;
      }
    }
  }
}

struct Maps {
  CUtensorMap main, rope;
};

template <typename T, int LATENT, int ROPE, int N>
__global__ void __launch_bounds__(kThreads, 1)
    few_kernel(const __grid_constant__ Maps maps, const __grid_constant__ Params p) {
  using LY = Layout<LATENT, ROPE, N>;
  constexpr int kPairs = LY::kPairs, kRing = LY::kRing;
  constexpr int kMine = N / 2;  // rows of a softmax lane
  extern __shared__ unsigned char raw[];
  unsigned char* const sm = raw + ((1024u - (smem_u32(raw) & 1023u)) & 1023u);
  unsigned char* const sm_w = sm + LY::kWeightsAt;
  unsigned char* const sm_rope = sm + LY::kRopeAt;
  unsigned char* const sm_ring = sm + LY::kRingAt;
  __shared__ __align__(8) uint64_t full[kRing], empty[kRing], rope_full[kRopes],
      rope_empty[kRopes], q_full, q_empty, s_full[2], p_full[2], pv_done[2], o_done[2],
      fin_full[2], fin_empty[2], drained;
  __shared__ __align__(16) float ref[2][N];     // reference exponents of two tiles' rows
  __shared__ __align__(16) float off[N];        // what is added to a score: lift - reference
  __shared__ __align__(16) float factor[N];
  __shared__ float top[4][N];
  __shared__ float sums[2][4][2][N];            // of weights, and of the rounded ones
  __shared__ float inverse[N];
  __shared__ int scrubbed[2];  // first token of two tiles of which numbers were taken out
  __shared__ uint32_t sh_tmem;
  __shared__ int sh_fail;

  const int worker = blockIdx.x;
  const Start begin = p.l.start[worker];  // on their way beside the header
  const int64_t until = p.l.start[worker + 1].u;
  const Header hd = *p.l.header;
  asm volatile("griddepcontrol.launch_dependents;");
  if (worker >= hd.workers) return;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int i = 0; i < kRing; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&rope_full[i], 1);
      mbar_init(&rope_empty[i], 1);
      mbar_init(&s_full[i], 1);
      mbar_init(&p_full[i], kSoftWarps);
      mbar_init(&pv_done[i], 1);
      mbar_init(&o_done[i], 1);
      mbar_init(&fin_full[i], kSoftWarps);
      mbar_init(&fin_empty[i], kOutWarps);
    }
    mbar_init(&q_full, kOutWarps);
    mbar_init(&q_empty, 1);
    mbar_init(&drained, 1);
    mbar_fence_init();
    sh_fail = 0;
  }
  if (warp == kMmaWarp) {
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
  Parts<1, kTokens> parts(p, hd, worker, begin, until);
  Part x;

  if (warp < kSoftWarps) {
    // ------------------------------------------------------------- softmax
    const int tid = threadIdx.x, quarter = warp & 3, half = warp >> 2;
    const int row0 = half * kMine, lane_tok = quarter * 32 + lane;
    const uint32_t lanes = (uint32_t)(quarter * 32) << 16;
    bool ok = true;  // the same in the eight warps, which meet at barriers
    int it = 0, seg = 0;
    Part next;
    bool more = parts.next(p, &next);
#pragma unroll 1
    while (ok && more) {
      x = next;
      if (x.steps == 0) {
        more = parts.next(p, &next);
        continue;
      }
      const int ob = seg & 1;
      if (seg >= 2) ok = wait(&fin_empty[ob], ((seg >> 1) - 1) & 1);
      if (soft_any(!ok)) { ok = false; break; }
      if (tid < N) {
        ref[ob][tid] = -INFINITY;
        off[tid] = kNoReference;
        if (tid == 0) scrubbed[ob] = INT_MAX;
      }
      soft_sync();
      float l[kMine], lr[kMine];
#pragma unroll
      for (int n = 0; n < kMine; ++n) l[n] = lr[n] = 0.0f;
#pragma unroll 1
      for (int i = 0; i < x.steps; ++i, ++it) {
        const int buf = it & 1;
        const uint32_t s_col = tmem + lanes + LY::kScore + buf * N + row0;
        ok = wait(&s_full[buf], (it >> 1) & 1);
        // and the weights of the step before last have been used
        if (ok && it >= 2) ok = wait(&pv_done[buf], ((it >> 1) - 1) & 1);
        tc_fence_after();
        uint32_t v[kMine];
#pragma unroll
        for (int c = 0; c < kMine; c += 8) tmem_ld8_nowait(s_col + c, v + c);
        // rows from this one on (of the lane's) see the lane's token
        const int token = (x.step0 + i) * kTokens + lane_tok;
        const int ahead = p.causal ? token - (x.cached + x.tok0) : 0;
        const int from = (token >= x.len ? N : ahead > 0 ? min(ahead * p.heads, N) : 0) - row0;
        const bool hides = __any_sync(kFull, from > 0);
        tmem_wait_all(v);
        // exponents; does one pass its row's reference by more than it may?
        float y[kMine], far = -INFINITY;
        auto exponents = [&] {
#pragma unroll
          for (int k = 0; k < kMine; k += 4) {
            const float4 o = *reinterpret_cast<const float4*>(&off[row0 + k]);
            const float2 a = fma2(__uint_as_float(v[k]), __uint_as_float(v[k + 1]), p.scale_log2,
                                  make_float2(o.x, o.y));
            const float2 b = fma2(__uint_as_float(v[k + 2]), __uint_as_float(v[k + 3]),
                                  p.scale_log2, make_float2(o.z, o.w));
            y[k] = a.x;
            y[k + 1] = a.y;
            y[k + 2] = b.x;
            y[k + 3] = b.y;
          }
        };
        exponents();
        bool odd = false;  // a hidden score that is no finite number
        if (hides) {
#pragma unroll
          for (int k = 0; k < kMine; ++k)
            if (k < from) {
              odd |= (v[k] & 0x7F800000u) == 0x7F800000u;
              y[k] = -INFINITY;
            }
        }
#pragma unroll
        for (int k = 0; k < kMine; k += 2) far = max3(far, y[k], y[k + 1]);
        if (soft_any(!ok || far > kLazy + Kind<T>::kLift)) {
          // every row's largest score, its reference exponent, what was added up so far
          if (soft_any(!ok)) { ok = false; break; }
#pragma unroll
          for (int k = 0; k < kMine; ++k) {
            const float m = warp_max(k < from ? -INFINITY : __uint_as_float(v[k]) * p.scale_log2);
            if (lane == 0) top[quarter][row0 + k] = m;
          }
          soft_sync();
          if (tid < N) {
            const float m = fmaxf(fmaxf(top[0][tid], top[1][tid]), fmaxf(top[2][tid], top[3][tid]));
            const float old = ref[ob][tid];
            const float next = m > old + kLazy ? reference_of(m) : old;
            factor[tid] = next == old ? 1.0f : ex2(old - next);
            ref[ob][tid] = next;
            off[tid] = next == -INFINITY ? kNoReference : Kind<T>::kLift - next;
          }
          soft_sync();
          exponents();
          if (hides) {
#pragma unroll
            for (int k = 0; k < kMine; ++k)
              if (k < from) y[k] = -INFINITY;
          }
          if (i > 0) {
#pragma unroll
            for (int n = 0; n < kMine; ++n) {
              l[n] *= factor[row0 + n];
              lr[n] *= factor[row0 + n];
            }
            // once the products of the step before have ended
            ok = wait(&pv_done[(it - 1) & 1], ((it - 1) >> 1) & 1);
            if (soft_any(!ok)) { ok = false; break; }  // all of them, or the others would wait
            tc_fence_after();
#pragma unroll 1
            for (int c = half * 16; c < kPairs * N; c += 32) {
              const uint32_t at = tmem + lanes + LY::kResult + ob * kPairs * N + c;
              uint32_t o[16];
              tmem_ld16(at, o);
#pragma unroll
              for (int k = 0; k < 16; ++k)
                o[k] = __float_as_uint(__uint_as_float(o[k]) * factor[c % N + k]);
              tmem_st16(at, o);
            }
            tmem_wait_st();
          }
        }
        unsigned char* const weights =
            sm_w + buf * LY::kWeights + lane_tok / 64 * (N * 128) + row0 * 128 + lane % 8 * 2;
        const int chunk = lane_tok % 64 / 8;
#pragma unroll
        for (int k = 0; k < kMine; k += 2) {
          const float a = ex2(y[k]), b = ex2(y[k + 1]);
          const uint32_t w = Kind<T>::pack(a, b);
          const float2 r = Kind<T>::widen(w);
          l[k] += a;
          l[k + 1] += b;
          lr[k] += r.x;
          lr[k + 1] += r.y;
          // rows of a half start at a multiple of eight: their places in it are the swizzle's
          *reinterpret_cast<uint16_t*>(weights + atom_byte(k, chunk)) = (uint16_t)w;
          *reinterpret_cast<uint16_t*>(weights + atom_byte(k + 1, chunk)) = (uint16_t)(w >> 16);
        }
        if (hides && __any_sync(kFull, odd)) {
          // the copies landed before the scores were there; seen here before the look at them
          bool there = true;
          for (int j = 0; j < kPairs && there; ++j) {
            const unsigned s = (unsigned)it * kPairs + j;
            there = wait(&full[s % kRing], (s / kRing) & 1);
          }
          if (there && odd && scrub<T, kPairs, kRing>(sm_ring, (unsigned)it * kPairs, lane_tok))
            atomicMin(&scrubbed[ob], token);
        }
        fence_proxy_async_smem();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_full[buf]);
        // a chain of loads that lies under the wait for the next scores
        if (i == 0) more = parts.next(p, &next);
      }
      if (!ok) break;
      // sums over the tokens, for the warps that bring the results out
      sum_lanes<kMine>(l, lane);
      sum_lanes<kMine>(lr, lane);
#pragma unroll
      for (int k = 0; k < kSums<kMine>; ++k) {
        sums[ob][quarter][0][row0 + first_sum<kMine>(lane) + k] = l[k];
        sums[ob][quarter][1][row0 + first_sum<kMine>(lane) + k] = lr[k];
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&fin_full[ob]);
      ++seg;
    }
  } else if (warp < kMmaWarp) {
    // ------------------------------------------------- queries in, results out
    const int tid = threadIdx.x - kSoftThreads;
    const uint32_t lanes = (uint32_t)((warp - kSoftWarps) * 32) << 16;
    bool ok = true;  // the same in the four warps
    int loaded = 0, seg = 0;
    auto queries = [&](const Part& y) {
      if (loaded > 0 && !(ok = wait(&q_empty, (loaded - 1) & 1))) return;
      ++loaded;
      // a row's chunks of 16 bytes side by side, as many rows at a time as there are
      // threads for, eight loads in flight
      constexpr int kChunks = (LATENT + ROPE) / 8;
      constexpr int kRowLanes = kChunks <= 32 ? 32 : kChunks <= 64 ? 64 : 128;
      constexpr int kRowsPass = 128 / kRowLanes, kPasses = N / kRowsPass;
      constexpr int kBatch = 8;
      static_assert(kPasses % kBatch == 0, "rows");
      const int rows = y.toks[0] * p.heads;
#pragma unroll 1
      for (int c = tid % kRowLanes; c < kChunks; c += kRowLanes) {
        const bool wide = c < LATENT / 8;
        const int r = c - LATENT / 8;
        const uint16_t* const from = (wide ? p.q + c * 8 : p.qr + r * 8) +
                                     (y.start + y.tok0) * (wide ? p.q_row : p.qr_row);
        const int64_t row = wide ? p.q_row : p.qr_row, head = wide ? p.q_head : p.qr_head;
#pragma unroll 1
        for (int i0 = 0; i0 < kPasses; i0 += kBatch) {
          uint4 v[kBatch];
#pragma unroll
          for (int i = 0; i < kBatch; ++i) {
            const int n = (i0 + i) * kRowsPass + tid / kRowLanes;
            const int t = y.toks[0] == 1 ? 0 : n / p.heads;
            v[i] = n < rows ? __ldg(reinterpret_cast<const uint4*>(from + t * row +
                                                                   (n - t * p.heads) * head))
                            : make_uint4(0, 0, 0, 0);
          }
#pragma unroll
          for (int i = 0; i < kBatch; ++i) {
            const int n = (i0 + i) * kRowsPass + tid / kRowLanes;
            *reinterpret_cast<uint4*>(
                sm + (wide ? c / 8 * (N * 128) + atom_byte(n, c % 8)
                           : LY::kQRopeAt + (ROPE == 64 ? atom_byte(n, r) : half_atom_byte(n, r)))) =
                v[i];
          }
        }
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(&q_full);
    };
    Part next;
    bool more = parts.next(p, &next);
    if (more && next.steps > 0) queries(next);
#pragma unroll 1
    while (more) {
      x = next;
      more = parts.next(p, &next);
      if (ok && more && next.steps > 0) queries(next);
      const int ob = seg & 1, rows = x.toks[0] * p.heads;
      if (x.steps > 0) {
        ok = ok && wait(&fin_full[ob], (seg >> 1) & 1) && wait(&o_done[ob], (seg >> 1) & 1);
        tc_fence_after();
        ++seg;
      }
      if (!(ok = out_all(ok))) break;
      const int64_t row0 = (int64_t)(x.start + x.tok0) * p.heads;
      float* const slot = p.l.part + (int64_t)x.slot * LY::kSlot;
      if (tid < N) {
        float m = -INFINITY, l = 0.0f, lr = 0.0f;
        if (x.steps > 0) {
          m = ref[ob][tid];
#pragma unroll
          for (int w = 0; w < 4; ++w) {
            l += sums[ob][w][0][tid];
            lr += sums[ob][w][1][tid];
          }
        }
        const int seen = seen_by(p, x, x.tok0 + tid / p.heads);
        const bool sees = seen > x.step0 * kTokens;  // any of the part's tokens
        // one that held what is no number: 0 times it, if its score is -inf
        if (x.steps > 0 && seen > scrubbed[ob]) lr = __int_as_float(0x7FC00000);
        inverse[tid] = !sees ? 0.0f : lr == 0.0f ? __int_as_float(0x7FC00000) : 1.0f / lr;
        if (tid < rows) {
          if (x.slot >= 0)
            *reinterpret_cast<float4*>(slot + N * LATENT + 4 * tid) =
                make_float4(m, l, lr, x.steps == 0 ? kNoResult : sees ? kSees : kSeesNothing);
          else if (p.lse)
            p.lse[row0 + tid] =
                l == 0.0f ? -INFINITY : (m - Kind<T>::kLift + log2f(l)) * 0.693147180559945309f;
        }
      }
      out_sync();
      // a lane has one of the values, of all rows: sixteen at a time
#pragma unroll 1
      for (int c = 0; c < kPairs * N; c += 16) {
        const int j = c / N, n = c % N;  // 128 values, and the first row
        if (n >= rows) continue;
        uint32_t o[16];
        if (x.steps > 0) tmem_ld16(tmem + lanes + LY::kResult + ob * kPairs * N + c, o);
        if (x.slot >= 0) {
          float* const to = slot + n * LATENT + j * 128 + tid;
          if (x.steps > 0)
#pragma unroll
            for (int k = 0; k < 16; ++k)
              if (n + k < rows) to[k * LATENT] = __uint_as_float(o[k]);
        } else {
          uint16_t* const to = p.out + (row0 + n) * LATENT + j * 128 + tid;
#pragma unroll
          for (int k = 0; k < 16; ++k) {
            const float inv = inverse[n + k];
            if (n + k < rows)
              to[k * LATENT] =
                  inv == 0.0f ? (uint16_t)0
                              : (uint16_t)Kind<T>::pack(__uint_as_float(o[k]) * inv, 0.0f);
          }
        }
      }
      tc_fence_before();
      out_sync();  // and `inverse` has been read
      if (x.steps > 0 && lane == 0) mbar_arrive(&fin_empty[ob]);
    }
  } else if (warp == kMmaWarp) {
    // ---------------------------------------------------------- products
    const uint32_t base = __shfl_sync(kFull, tmem, 0);
    const uint32_t q_lo = (uint32_t)sw128_desc(sm), k_lo = (uint32_t)sw128_desc(sm_ring);
    const uint32_t r_lo = (uint32_t)sw128_desc(sm_rope), w_lo = (uint32_t)sw128_desc(sm_w);
    const uint32_t v_lo = (uint32_t)sw128_mn_desc(sm_ring, kAtom);
    auto desc = [&](uint32_t hi, uint32_t lo) { return (uint64_t)hi << 32 | lo; };
    int it = 0, seg = 0;
    bool ok = true;
    int part = 0;  // places of the step's scores that are done; kPairs: positional part next
    // Goes on with the scores of step s, up to `most` places of it (kPairs + 1: all).  With a
    // barrier `other` it gives way as soon as that one is through and rows are not there.
    auto scores = [&](int s, int most, uint64_t* other, unsigned parity) {
      const uint32_t to = base + LY::kScore + (s & 1) * N;
#pragma unroll 1
      while (part < most) {
        const unsigned place = (unsigned)s * kPairs + part;
        const bool last = part == kPairs;
        uint64_t* const bar = last ? &rope_full[s % kRopes] : &full[place % kRing];
        const unsigned phase = (last ? (unsigned)s / kRopes : place / kRing) & 1;
        if (other) {
          bool there = false;
          for (unsigned i = 0; i < p.probes; ++i) {
            if ((there = __all_sync(kFull, mbar_try_wait(bar, phase)))) break;
            if (__all_sync(kFull, mbar_try_wait(other, parity))) return;
            if (*(volatile int*)&sh_fail) break;
          }
          if (!there) {
            ok = wait(bar, phase);  // the limit is up, or somebody's was
            if (!ok) return;
          }
        } else if (!(ok = wait(bar, phase))) {
          return;
        }
        tc_fence_after();
        if (!last) {
          const uint32_t kd = k_lo + place % kRing * (kPlace / 16);
          const uint32_t qd = q_lo + part * (2 * N * 128 / 16);
          if (elect_one()) {
#pragma unroll
            for (int k = 0; k < 8; ++k)
              umma_f16(to, desc(kHi128, kd + (k / 4 * kAtom + k % 4 * 32) / 16),
                       desc(kHi128, qd + (k / 4 * (N * 128) + k % 4 * 32) / 16),
                       idesc<T>(N, false), part != 0 || k != 0);
          }
        } else if (elect_one()) {
          constexpr uint32_t kHi = ROPE == 64 ? kHi128 : kHi64;
#pragma unroll
          for (int k = 0; k < ROPE / 16; ++k)
            umma_f16(to, desc(kHi, r_lo + (s % kRopes * LY::kRopeBytes + k * 32) / 16),
                     desc(kHi, q_lo + (LY::kQRopeAt + k * 32) / 16), idesc<T>(N, false), 1);
          umma_commit(&rope_empty[s % kRopes]);
          umma_commit(&s_full[s & 1]);
        }
        __syncwarp();
        ++part;
      }
    };
    Part next;
    bool more = parts.next(p, &next);
#pragma unroll 1
    while (ok && more) {
      x = next;
      const int steps = __shfl_sync(kFull, x.steps, 0);
      if (steps == 0) {
        more = parts.next(p, &next);
        continue;
      }
      const int ob = seg & 1;
      ok = wait(&q_full, seg & 1) && (seg < 2 || wait(&fin_empty[ob], ((seg >> 1) - 1) & 1));
      if (!ok) break;
      tc_fence_after();
      part = 0;
      scores(it, kPairs + 1, nullptr, 0);
      if (ok && steps == 1 && elect_one()) umma_commit(&q_empty);
      __syncwarp();
      more = parts.next(p, &next);  // under the first softmax
#pragma unroll 1
      for (int i = 0; i < steps && ok; ++i) {
        const int s = it + i;
        part = 0;
        // the next scores on what has come, as long as the weights are not there
        if (i + 1 < steps)
          scores(s + 1, LY::kPre == kPairs ? kPairs + 1 : LY::kPre, &p_full[s & 1], (s >> 1) & 1);
        if (!ok || !(ok = wait(&p_full[s & 1], (s >> 1) & 1))) break;
        tc_fence_after();
        const uint32_t wd = w_lo + (s & 1) * (LY::kWeights / 16);
#pragma unroll 1
        for (int j = 0; j < kPairs; ++j) {
          const unsigned place = (unsigned)s * kPairs + j;
          const uint32_t vd = v_lo + place % kRing * (kPlace / 16);
          const uint32_t to = base + LY::kResult + (ob * kPairs + j) * N;
          if (elect_one()) {
#pragma unroll
            for (int k = 0; k < kTokens / 16; ++k)
              umma_f16(to, desc(kHi128, vd + k * (16 * 128 / 16)),
                       desc(kHi128, wd + (k / 4 * (N * 128) + k % 4 * 32) / 16),
                       idesc<T>(N, true), i != 0 || k != 0);
            umma_commit(&empty[place % kRing]);
            if (j + 1 == kPairs) {
              umma_commit(&pv_done[s & 1]);
              if (i + 1 == steps) umma_commit(&o_done[ob]);
            }
          }
          __syncwarp();
        }
        if (i + 1 < steps) {
          scores(s + 1, kPairs + 1, nullptr, 0);
          if (ok && i + 2 == steps && elect_one()) umma_commit(&q_empty);
          __syncwarp();
        }
      }
      it += steps;
      ++seg;
    }
    // whatever happened, nothing is in flight when tensor memory is given back
    if (elect_one()) umma_commit(&drained);
    __syncwarp();
    mbar_wait(&drained, 0, kProbes);
  } else {
    // ------------------------------------------------ rows from their pages
    const int piece = 1 << p.page_shift;  // tokens of one copy
    const int pieces = kTokens / piece;
    const int my_tok = lane % pieces * piece;
    int s = 0;           // steps begun
    unsigned places = 0, ropes = 0;
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
#pragma unroll 1
      for (int i = 0; i < x.steps && ok; ++i, ++s) {
        const int row = at;
        if (i + 1 < x.steps) at = row_at(i + 1);
#pragma unroll 1
        for (int j = 0; j < kPairs; ++j, ++places) {
          const unsigned st = places % kRing;
          if (places >= kRing && !(ok = wait(&empty[st], (places / kRing - 1) & 1))) break;
          if (lane == 0) mbar_arrive_expect_tx(&full[st], kPlace);
          __syncwarp();
          for (int y = lane; y < 2 * pieces; y += 32)
            tma_load(sm_ring + st * kPlace + y / pieces * kAtom + my_tok * 128, &maps.main,
                     j * 128 + y / pieces * 64, row, &full[st]);
        }
        if (!ok) break;
        if (s >= kRopes && !(ok = wait(&rope_empty[s % kRopes], (s / kRopes - 1) & 1))) break;
        if (lane == 0) mbar_arrive_expect_tx(&rope_full[s % kRopes], LY::kRopeBytes);
        __syncwarp();
        if (lane < pieces)
          tma_load(sm_rope + s % kRopes * LY::kRopeBytes + my_tok * ROPE * 2, &maps.rope, LATENT,
                   row, &rope_full[s % kRopes]);
        ++ropes;
      }
    }
    // no copy is in flight when the block ends, whatever happened
    for (unsigned i = places > kRing ? places - kRing : 0; i < places; ++i)
      mbar_wait(&full[i % kRing], (i / kRing) & 1, kProbes);
    for (unsigned i = ropes > kRopes ? ropes - kRopes : 0; i < ropes; ++i)
      mbar_wait(&rope_full[i % kRopes], (i / kRopes) & 1, kProbes);
  }

  __syncwarp();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == kMmaWarp) tmem_dealloc(tmem, kTmemCols);
  if (sh_fail) {
    if (warp < kSoftWarps) lose_rows<LATENT, N>(p, hd, worker);
    if (threadIdx.x == 0) atomicOr(p.status, GRM_B200_PLAN_WAIT);
  }
}

template <typename T, int LATENT, int ROPE, int N>
int launch(const Params& p, cudaStream_t st) {
  using LY = Layout<LATENT, ROPE, N>;
  Maps maps;
  const int64_t width = p.latent + p.rope;
  const int64_t cache[2] = {width, p.pages << p.page_shift};
  const int box[2] = {64, 1 << p.page_shift}, rope[2] = {ROPE, 1 << p.page_shift};
  int rc;
  if ((rc = make_map(&maps.main, p.cache, 2, cache, &width, box)) ||
      (rc = make_map(&maps.rope, p.cache, 2, cache, &width, rope)))
    return rc;
  auto kernel = few_kernel<T, LATENT, ROPE, N>;
  static std::atomic<uint64_t> done{0};
  if ((rc = paged::allow_shared(reinterpret_cast<const void*>(kernel), LY::kSmem, &done)))
    return rc;
  kernel<<<(unsigned)p.v.tiling.workers, kThreads, LY::kSmem, st>>>(maps, p);
  if ((rc = paged::launch_status("latent attend"))) return rc;
  return launch_join<T, LATENT, 1, N, false>(p, st);
}

template <int LATENT, int ROPE, int N>
int launch_kind(const Params& p, cudaStream_t st) {
  return p.dtype == GRM_B200_F16 ? launch<__half, LATENT, ROPE, N>(p, st)
                                 : launch<__nv_bfloat16, LATENT, ROPE, N>(p, st);
}

template <int LATENT, int ROPE>
int launch_columns(const Params& p, cudaStream_t st) {
  return p.v.tiling.few == 16 ? launch_kind<LATENT, ROPE, 16>(p, st)
                              : launch_kind<LATENT, ROPE, 32>(p, st);
}

}  // namespace

int launch_few(const Params& p, cudaStream_t st) {
  return p.rope == 32 ? launch_columns<512, 32>(p, st) : launch_columns<512, 64>(p, st);
}

}  // namespace latent
}  // namespace grm_b200
