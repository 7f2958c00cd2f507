// latent_expand.cu -- keys and values of each head from the rows of the cache,
//   k = W^k_h c,  v = W^v_h c,
// for the tokens of every request that has rows in the step: a product of [tokens,
// latent] and [heads * (nope + value), latent], on tcgen05.  A key goes out as two
// numbers of the arena's type, the rounded one and what that left over, a value as
// one.
//
// A block, one an SM, takes an equal share of (128 tokens, head) pairs, a tile of
// tokens after another: their rows come to shared memory once a tile, from their pages
// by tensor-map copies, and the heads' weights stream by, 128 rows of 64 columns at a
// time.  Results go from tensor memory (four buffers, so that products run under the
// conversion) through shared memory to global memory by tensor-map copies, one pair by
// one group of four warps and the next by the other: what holds a group up is the
// chain of conversion, barriers and copies.
//
// Bound by HBM's writes: 6 bytes for a token, head and value a head has of either kind, 476
// MB for 31,000 tokens of 40 heads of 64 + 64.  A fill of as many takes 124 us, this 156
// (210 with one group of four warps and two buffers; results 128 bytes of a row at a time,
// or two places of them a group, changed nothing).
#include <algorithm>

#include "latent_device.cuh"

namespace grm_b200 {
namespace latent {

namespace {

using paged::kProbes;

constexpr int kTile = 128;               // tokens
constexpr int kAtom = kTile * 128;       // 128 rows of 64 values
constexpr int kGroups = 2, kMmaWarp = 4 * kGroups;  // and one that loads
constexpr int kThreads = (kMmaWarp + 2) * 32;
constexpr int kBuffers = 4;              // of results in tensor memory
constexpr uint32_t kTmemCols = kBuffers * 128;
constexpr int kStages = 4;               // of weights
constexpr int kCols = 32;                // results that go out together
constexpr int kPlace = kTile * kCols * 2;

template <int LATENT>
struct Layout {
  static constexpr int kAtoms = LATENT / 64;
  static constexpr int kWeights = kAtoms * kAtom;          // after the rows
  // results on their way out: a group's numbers and what they left over
  static constexpr int kOut = kWeights + kStages * kAtom;
  static constexpr int kUsed = 1024 + kOut + 2 * kGroups * kPlace;
  static constexpr int kSmem = kUsed > 120 * 1024 ? kUsed : 120 * 1024;
};

struct Maps {
  CUtensorMap rows, weights, keys, values;
};

__device__ __forceinline__ void tma_store(const CUtensorMap* map, int x, int y, int z,
                                          const void* src) {
  asm volatile("cp.async.bulk.tensor.3d.global.shared::cta.tile.bulk_group [%0, {%1, %2, %3}], [%4];"
               ::"l"(map), "r"(x), "r"(y), "r"(z), "r"(smem_u32(src))
               : "memory");
}

__device__ __forceinline__ void group_sync(int group) {
  asm volatile("bar.sync %0, 128;" ::"r"(1 + group) : "memory");
}
// The same, and whether all of the group are fine.
__device__ __forceinline__ bool group_all(int group, bool ok) {
  unsigned r;
  asm volatile("{\n .reg .pred p, q;\n setp.ne.u32 p, %1, 0;\n"
               " barrier.cta.red.and.pred q, %2, 128, p;\n selp.u32 %0, 1, 0, q;\n}\n"
               : "=r"(r)
               : "r"((unsigned)ok), "r"(1 + group)
               : "memory");
  return r != 0;
}

template <typename T, int LATENT>
__global__ void __launch_bounds__(kThreads, 1)
    expand_kernel(const __grid_constant__ Maps maps, const __grid_constant__ Params p) {
  using LY = Layout<LATENT>;
  extern __shared__ unsigned char raw[];
  unsigned char* const sm = raw + ((1024u - (smem_u32(raw) & 1023u)) & 1023u);
  unsigned char* const sm_w = sm + LY::kWeights;
  unsigned char* const sm_out = sm + LY::kOut;
  __shared__ __align__(8) uint64_t a_full, a_empty, b_full[kStages], b_empty[kStages],
      d_full[kBuffers], d_empty[kBuffers], drained;
  __shared__ uint32_t sh_tmem;
  __shared__ int sh_fail;

  const int total = p.room[p.v.requests];  // tokens, a multiple of 64
  const int64_t pairs = ceil_div64(total, kTile) * p.heads;
  const int64_t first = pairs * blockIdx.x / gridDim.x;
  const int64_t end = pairs * (blockIdx.x + 1) / gridDim.x;
  if (first == end) return;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int units = p.nope == 64 ? 1 : 2;  // products of 128 weight rows of a head
  if (threadIdx.x == 0) {
    mbar_init(&a_full, 1);
    mbar_init(&a_empty, 1);
    for (int i = 0; i < kStages; ++i) {
      mbar_init(&b_full[i], 1);
      mbar_init(&b_empty[i], 1);
    }
    for (int i = 0; i < kBuffers; ++i) {
      mbar_init(&d_full[i], 1);
      mbar_init(&d_empty[i], 4);
    }
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
    bool ok = false;
    for (unsigned i = 0; i < p.probes; ++i) {
      if ((ok = mbar_try_wait(bar, parity))) break;
      if (*(volatile int*)&sh_fail) break;
    }
    ok = __all_sync(kFull, ok);
    if (!ok) *(volatile int*)&sh_fail = 1;
    return ok;
  };

  if (warp < kMmaWarp) {
    // ---------------------------------------- results to the arena's type and out
    const int group = warp >> 2, row = (warp & 3) * 32 + lane;
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    const bool copies = (threadIdx.x & 127) == 0;  // one thread of the group
    unsigned char* const to = sm_out + group * 2 * kPlace;
    bool ok = true;  // the same in a group's four warps, which meet at barriers below
#pragma unroll 1
    for (int64_t x = first + group; x < end && ok; x += kGroups) {
      int it = (int)(x - first) * units;
      const int t0 = (int)(x / p.heads) * kTile, h = (int)(x % p.heads);
      bool bad = false;  // a value that is no number
#pragma unroll 1
      for (int u = 0; u < units; ++u, ++it) {
        const int buf = it % kBuffers;
        if (!(ok = group_all(group, wait(&d_full[buf], (it / kBuffers) & 1)))) break;
        tc_fence_after();
        // values first: the upper half of a unit of both, or a unit of their own
#pragma unroll 1
        for (int y = 128 / kCols - 1; y >= 0; --y) {
          const bool value = units == 1 ? y >= 64 / kCols : u == 0;
          const int col = (units == 1 ? y % (64 / kCols) : y) * kCols;  // of the head's
          uint32_t v[32];
          tmem_ld32_nowait(tmem + lanes + buf * 128 + y * kCols, v);
          tmem_wait_ld32(v);
          // the copies before have left this place
          if (copies) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
          group_sync(group);
#pragma unroll
          for (int c = 0; c < kCols / 8; ++c) {
            uint32_t hi[4], lo[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const float a = __uint_as_float(v[8 * c + 2 * k]);
              const float b = __uint_as_float(v[8 * c + 2 * k + 1]);
              hi[k] = Kind<T>::pack(a, b);
              const float2 w = Kind<T>::widen(hi[k]);
              lo[k] = Kind<T>::pack(a - w.x, b - w.y);
              constexpr uint32_t e = Kind<T>::kNoNumber;
              if (value) bad |= (hi[k] & e) == e || (hi[k] >> 16 & e) == e;
            }
            // Keys of a token whose values are none in this type make its score none,
            // so that attention knows.
            if (bad && c == 0 && col == 0) lo[0] = 0x7FFFu | (lo[0] & 0xFFFF0000u);
            const uint32_t at = row * 64 + ((c ^ ((row >> 1) & 3)) << 4);
            *reinterpret_cast<uint4*>(to + at) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
            if (!value)
              *reinterpret_cast<uint4*>(to + kPlace + at) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
          }
          fence_proxy_async_smem();
          group_sync(group);
          if (copies) {
            for (int half = 0; half < 2; ++half) {
              const int t = t0 + half * 64, at = half * (kPlace / 2);
              if (t >= total) break;
              if (value) {
                tma_store(&maps.values, col, t, h, to + at);
              } else {
                tma_store(&maps.keys, col, t, h, to + at);
                tma_store(&maps.keys, p.nope + col, t, h, to + kPlace + at);
              }
            }
            asm volatile("cp.async.bulk.commit_group;" ::: "memory");
          }
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&d_empty[buf]);
      }
    }
    if (copies) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
  } else if (warp == kMmaWarp) {
    // ---------------------------------------------------------- products
    const uint32_t base = __shfl_sync(kFull, tmem, 0);
    constexpr uint32_t kIdesc = (1u << 4) | Kind<T>::kFormat | (128u >> 3 << 17) | (128u >> 4 << 24);
    const uint64_t a_desc = sw128_desc(sm), b_desc = sw128_desc(sm_w);
    bool ok = true;
    int it = 0, s = 0, tiles = 0;
    int64_t tile = -1;
#pragma unroll 1
    for (int64_t x = first; x < end && ok; ++x) {
      if (x / p.heads != tile) {
        tile = x / p.heads;
        ok = wait(&a_full, tiles & 1);
        ++tiles;
      }
#pragma unroll 1
      for (int u = 0; u < units && ok; ++u, ++it) {
        const int buf = it % kBuffers;
        if (it >= kBuffers && !(ok = wait(&d_empty[buf], (it / kBuffers - 1) & 1))) break;
        tc_fence_after();
#pragma unroll 1
        for (int c = 0; c < LY::kAtoms; ++c, ++s) {
          if (!(ok = wait(&b_full[s % kStages], (s / kStages) & 1))) break;
          tc_fence_after();
          if (elect_one()) {
#pragma unroll
            for (int k = 0; k < 4; ++k)
              umma_f16(base + buf * 128, a_desc + (c * kAtom + k * 32) / 16,
                       b_desc + (s % kStages * kAtom + k * 32) / 16, kIdesc, c + k != 0);
            umma_commit(&b_empty[s % kStages]);
          }
          __syncwarp();
        }
        if (ok && elect_one()) {
          umma_commit(&d_full[buf]);
          if (u + 1 == units && (x + 1) / p.heads != tile) umma_commit(&a_empty);
        }
        __syncwarp();
      }
    }
    if (elect_one()) umma_commit(&drained);
    __syncwarp();
    mbar_wait(&drained, 0, kProbes);
  } else {
    // ------------------------------- rows from their pages, weights as they stream by
    const int piece = min(1 << p.page_shift, 64), pieces = 64 / piece;
    bool ok = p.probes > 0;
    int s = 0, tiles = 0;
    int64_t tile = -1;
#pragma unroll 1
    for (int64_t x = first; x < end && ok; ++x) {
      if (x / p.heads != tile) {
        tile = x / p.heads;
        if (tiles > 0 && !(ok = wait(&a_empty, (tiles - 1) & 1))) break;
        const int halves = total - tile * kTile > 64 ? 2 : 1;
        if (lane == 0) mbar_arrive_expect_tx(&a_full, halves * LY::kAtoms * (kAtom / 2));
        __syncwarp();
        for (int half = 0; half < halves; ++half) {
          const int t0 = (int)(tile * kTile) + half * 64;
          int lo = 0, hi = (int)p.v.requests;
          while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (p.room[mid] <= t0) lo = mid;
            else hi = mid;
          }
          // past the request's end the last page again: nothing sees those rows
          const int tok = t0 - p.room[lo] + lane % pieces * piece;
          const int at = min(tok, p.v.lens[lo] - 1) >> p.page_shift;
          const int page = min(max(p.table[lo * p.width + at], 0), (int)p.pages - 1);
          const int y = (page << p.page_shift) + (tok & ((1 << p.page_shift) - 1));
          for (int i = lane; i < LY::kAtoms * pieces; i += 32)
            tma_load(sm + i / pieces * kAtom + (half * 64 + lane % pieces * piece) * 128,
                     &maps.rows, i / pieces * 64, y, &a_full);
        }
        ++tiles;
      }
      const int h = p.w_head ? (int)(x % p.heads) : 0;
#pragma unroll 1
      for (int u = 0; u < units && ok; ++u) {
        const int y = units == 2 ? (1 - u) * 128 : 0;  // values first
#pragma unroll 1
        for (int c = 0; c < LY::kAtoms; ++c, ++s) {
          if (s >= kStages && !(ok = wait(&b_empty[s % kStages], (s / kStages - 1) & 1))) break;
          if (lane == 0) {
            mbar_arrive_expect_tx(&b_full[s % kStages], kAtom);
            tma_load(sm_w + s % kStages * kAtom, &maps.weights, c * 64, y, h, &b_full[s % kStages]);
          }
          __syncwarp();
        }
      }
    }
    // no copy is in flight when the block ends, whatever happened
    if (tiles > 0) mbar_wait(&a_full, (tiles - 1) & 1, kProbes);
    for (int i = max(s - kStages, 0); i < s; ++i)
      mbar_wait(&b_full[i % kStages], (i / kStages) & 1, kProbes);
  }

  __syncwarp();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == kMmaWarp) tmem_dealloc(tmem, kTmemCols);
  if (sh_fail && threadIdx.x == 0) {  // attention then leaves no numbers
    atomicOr(p.status, GRM_B200_PLAN_WAIT);
    atomicExch(&p.l.header->lost, 1);
  }
}

template <typename T, int LATENT>
int launch(const Params& p, int sms, cudaStream_t st) {
  using LY = Layout<LATENT>;
  Maps maps;
  const int64_t width = p.latent + p.rope;
  const int64_t rows[2] = {width, p.pages << p.page_shift};
  const int64_t weights[3] = {p.latent, 2 * p.nope, p.w_head ? p.heads : 1};
  const int64_t w_strides[2] = {p.w_row, p.w_head ? p.w_head : 2 * p.nope * p.w_row};
  const int64_t keys[3] = {2 * p.nope, p.expand_tokens, p.heads};
  const int64_t k_strides[2] = {2 * p.nope, 2 * p.nope * p.expand_tokens};
  const int64_t values[3] = {p.nope, p.expand_tokens, p.heads};
  const int64_t v_strides[2] = {p.nope, p.nope * p.expand_tokens};
  const int piece[2] = {64, std::min(1 << p.page_shift, 64)}, box[3] = {64, 128, 1},
            out[3] = {kCols, 64, 1};
  int rc;
  if ((rc = make_map(&maps.rows, p.cache, 2, rows, &width, piece)) ||
      (rc = make_map(&maps.weights, p.weights, 3, weights, w_strides, box)) ||
      (rc = make_map(&maps.keys, p.keys, 3, keys, k_strides, out)) ||
      (rc = make_map(&maps.values, p.values, 3, values, v_strides, out)))
    return rc;
  auto kernel = expand_kernel<T, LATENT>;
  static std::atomic<uint64_t> done{0};
  if ((rc = paged::allow_shared(reinterpret_cast<const void*>(kernel), LY::kSmem, &done)))
    return rc;
  kernel<<<(unsigned)sms, kThreads, LY::kSmem, st>>>(maps, p);
  return paged::launch_status("latent expand");
}

template <typename T>
int launch_latent(const Params& p, int sms, cudaStream_t st) {
  return p.latent == 128   ? launch<T, 128>(p, sms, st)
         : p.latent == 256 ? launch<T, 256>(p, sms, st)
                           : launch<T, 512>(p, sms, st);
}

}  // namespace

int launch_expand(const Params& p, cudaStream_t st) {
  const int sms = p.v.tiling.workers;
  return p.dtype == GRM_B200_F16 ? launch_latent<__half>(p, sms, st)
                                 : launch_latent<__nv_bfloat16>(p, sms, st);
}

}  // namespace latent
}  // namespace grm_b200
