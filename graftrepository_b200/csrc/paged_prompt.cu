// paged_prompt.cu -- attention over the 8-bit paged arena for many query rows.
//
// The same sums as the split kernel's (paged_attend.cu): with key codes a_t and
// value codes b_t, key scale s_t and value scale u_t,
//   y_t = scale * log2(e) * s_t (q . a_t) + log2(u_t),  p_t = 2^(y_t - m),
//   out = sum_t p_t b_t / sum_t (p_t / u_t),
// here bound by arithmetic: 4 head_dim operations a (row, visible token) on the
// tensor cores and one exponential, 16 a clock and SM against 4,096 fp16
// multiply-adds, so at head_dim 128 a 128 x 128 tile costs the two units about
// the same 1,024 clocks.
//
// A block takes 2 x 128 query rows of one kv head (rows of the group's heads
// side by side, so a key tile serves all of them) and walks the visible tokens
// 128 at a time:
//   warps 0-3, 4-7  softmax of query tile 0 / 1, one row a thread: scores from
//                   tensor memory, p back as fp16 over them, and when a row's
//                   reference exponent has to move (rarely: it trails by up
//                   to 8), its result in tensor memory rescaled
//   warps 8-11      codes from their pages to fp16 key and value tiles in
//                   shared memory (two of each), read one tile ahead
//   warp 12         tensor memory, and one lane that issues the products
//                   S = Q K^T (both from shared memory) and O += P V (P from
//                   tensor memory)
// While one query tile's softmax runs, the tensor cores work for the other.
// Keys and values have the same layout in shared memory, 128-byte rows of 64
// dims with a 128-byte swizzle: K is read K-major, V with its dims contiguous.
// A block whose rows fit one tile leaves the other tile's work out.
#include <type_traits>

#include "paged.cuh"
#include "umma.cuh"

namespace grm_b200 {
namespace paged {

namespace {

constexpr int kM = 128;             // rows of a query tile
constexpr int kN = 128;             // tokens of a key tile
constexpr int kSoftWarps = 8;
constexpr int kConvWarps = 4;
constexpr int kMmaWarp = kSoftWarps + kConvWarps;
constexpr int kPromptThreads = (kMmaWarp + 1) * 32;
constexpr int kScaleRing = 4;       // key tiles whose scales are held
constexpr uint32_t kTmemCols = 512;
constexpr unsigned kProbes = 1u << 22;  // probes of a bounded wait

template <int D>
struct PromptLayout {
  static constexpr int kAtom = kN * 128;            // 128 rows x 64 halves
  static constexpr int kTile = (D / 64) * kAtom;    // a query, key or value tile
  static constexpr int kUsed = 1024 + 6 * kTile + kScaleRing * 8 * 16;
  // one block an SM: it owns all of tensor memory
  static constexpr int kSmem = kUsed > 120 * 1024 ? kUsed : 120 * 1024;
  static constexpr uint32_t kScore = 0;             // tensor memory columns
  static constexpr uint32_t kResult = 2 * kN;
  static_assert(2 * kN + 2 * D <= kTmemCols, "two score and two result tiles");
};

// fp32 accumulators, fp16 operands, 128 rows, N columns; B K-major or (bit 16) not.
__host__ __device__ constexpr uint32_t idesc(int n, bool b_mn) {
  return (1u << 4) | (b_mn ? 1u << 16 : 0u) | ((uint32_t)(n >> 3) << 17) |
         ((uint32_t)(kM >> 4) << 24);
}

// Byte of 16-byte chunk c (8 halves of 64) of row r in a swizzled atom.
__device__ __forceinline__ uint32_t atom_byte(int r, int c) { return r * 128 + ((c ^ (r & 7)) << 4); }

// Every lane of a warp waits; false, for all of them, when a wait gave up.
__device__ __forceinline__ bool warp_wait(uint64_t* bar, unsigned parity, volatile int* fail) {
  bool ok = false;
  for (unsigned i = 0; i < kProbes; ++i) {
    if ((ok = mbar_try_wait(bar, parity))) break;
    if (*fail) break;
  }
  ok = __all_sync(kFull, ok);
  if (!ok) *fail = 1;
  return ok;
}
__device__ __forceinline__ bool lane_wait(uint64_t* bar, unsigned parity, volatile int* fail) {
  for (unsigned i = 0; i < kProbes; ++i) {
    if (mbar_try_wait(bar, parity)) return true;
    if (*fail) return false;
  }
  *fail = 1;
  return false;
}

struct Scale {
  float key, log2_value, inv_value, unused;
};

template <typename T, int D>
__global__ void __launch_bounds__(kPromptThreads, 1) prompt_kernel(const AttendParams p) {
  using LY = PromptLayout<D>;
  extern __shared__ unsigned char raw[];
  unsigned char* const sm = raw + ((1024u - (smem_u32(raw) & 1023u)) & 1023u);
  unsigned char* const sm_q = sm;                       // [2]
  unsigned char* const sm_k = sm + 2 * LY::kTile;       // [2]
  unsigned char* const sm_v = sm + 4 * LY::kTile;       // [2]
  Scale* const sm_scale = reinterpret_cast<Scale*>(sm + 6 * LY::kTile);  // [kScaleRing][8]
  __shared__ __align__(8) uint64_t q_full, drained, k_full[2], k_empty[2], v_full[2], v_empty[2],
      scale_full[kScaleRing], s_full[2], p_full[2], o_done[2];
  __shared__ uint32_t sh_tmem;
  __shared__ int sh_fail;

  const Header hd = *p.l.header;
  // later tiles first: in a causal step they see the most tokens
  const int h = blockIdx.x % p.kv_heads;
  const int ti = hd.qtiles - 1 - (int)(blockIdx.x / p.kv_heads);
  if (ti < 0) return;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int2 tile = p.l.qtiles[ti];
  const int start = p.starts[tile.x];
  const int n = p.starts[tile.x + 1] - start;
  const int len = p.lens[tile.x];
  const int cached = len - n;
  const int per = p.qtile_tokens >> 1;  // tokens of one query tile
  const int tok0 = tile.y;
  const int toks[2] = {min(per, n - tok0), max(0, min(per, n - tok0 - per))};
  const bool two = toks[1] > 0;
  const int heads = p.kv_heads * p.group;
  const int sees = p.causal ? min(len, cached + tok0 + toks[0] + toks[1]) : len;
  const int tiles = (sees + kN - 1) / kN;

  if (tiles == 0) {  // nothing cached: empty rows
    for (int x = threadIdx.x; x < (toks[0] + toks[1]) * p.group * (D / 2); x += kPromptThreads) {
      const int j = x / (D / 2);
      const int64_t row = (int64_t)(start + tok0 + j / p.group) * heads + h * p.group + j % p.group;
      reinterpret_cast<uint32_t*>(p.out + row * D)[x % (D / 2)] = 0;
      if (p.lse && x % (D / 2) == 0) p.lse[row] = -INFINITY;
    }
    return;
  }

  if (threadIdx.x == 0) {
    mbar_init(&q_full, two ? kSoftWarps : kSoftWarps / 2);
    mbar_init(&drained, 1);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&k_full[i], kConvWarps);
      mbar_init(&k_empty[i], 1);
      mbar_init(&v_full[i], kConvWarps);
      mbar_init(&v_empty[i], 1);
      mbar_init(&s_full[i], 1);
      mbar_init(&p_full[i], kSoftWarps / 2);
      mbar_init(&o_done[i], 1);
    }
    for (int i = 0; i < kScaleRing; ++i) mbar_init(&scale_full[i], 1);
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
  volatile int* const fail = &sh_fail;

  if (warp < kSoftWarps) {
    // ------------------------------------------------------------- softmax
    const int t = warp >> 2;
    if (t == 0 || two) {
      const int row = (warp & 3) * 32 + lane;
      const bool active = row < (t == 0 ? toks[0] : toks[1]) * p.group;
      const int token = tok0 + t * per + row / p.group;
      const int64_t orow = (int64_t)(start + token) * heads + h * p.group + row % p.group;
      const int lim = active && p.causal ? cached + token + 1 : len;  // tokens that the row sees

      // the row as fp16 (a bf16 row scaled by a power of two), to shared memory
      float kq = p.scale_log2;
      {
        uint4 x[D / 8];
#pragma unroll
        for (int c = 0; c < D / 8; ++c) x[c] = make_uint4(0, 0, 0, 0);
        if (active) {
          const uint16_t* qp = p.q + (int64_t)(start + token) * p.q_row +
                               (int64_t)(h * p.group + row % p.group) * p.q_head;
#pragma unroll
          for (int c = 0; c < D / 8; ++c) x[c] = __ldg(reinterpret_cast<const uint4*>(qp) + c);
        }
        if constexpr (!std::is_same<T, __half>::value) {
          unsigned m = 0;
#pragma unroll
          for (int c = 0; c < D / 8; ++c) {
            m = __vmaxu2(m, __vmaxu2(x[c].x & 0x7FFF7FFFu, x[c].y & 0x7FFF7FFFu));
            m = __vmaxu2(m, __vmaxu2(x[c].z & 0x7FFF7FFFu, x[c].w & 0x7FFF7FFFu));
          }
          m = max(m & 0xFFFFu, m >> 16);
          float up;
          row_scale(m, &up, &kq);
          kq *= p.scale_log2;
#pragma unroll
          for (int c = 0; c < D / 8; ++c)
            x[c] = make_uint4(scale_pair(x[c].x, up), scale_pair(x[c].y, up),
                              scale_pair(x[c].z, up), scale_pair(x[c].w, up));
        }
#pragma unroll
        for (int c = 0; c < D / 8; ++c)
          *reinterpret_cast<uint4*>(sm_q + t * LY::kTile + (c / 8) * LY::kAtom +
                                    atom_byte(row, c % 8)) = x[c];
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(&q_full);

      const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
      const uint32_t s_col = tmem + lanes + LY::kScore + t * kN;
      const uint32_t o_col = tmem + lanes + LY::kResult + t * D;
      float m = -INFINITY, l = 0.0f;
      bool ok = true;
      for (int j = 0; j < tiles && ok; ++j) {
        ok = warp_wait(&scale_full[j % kScaleRing], (j / kScaleRing) & 1, fail) &&
             warp_wait(&s_full[t], j & 1, fail);
        if (!ok) break;
        tc_fence_after();
        const Scale* sc = sm_scale + (j % kScaleRing) * 8;
        const int t0 = j * kN;
        const bool masked = __any_sync(kFull, t0 + kN > lim);
        // the largest exponent of the row's 128 scores
        float top = -INFINITY;
        uint32_t v[32];
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          tmem_ld32_nowait(s_col + 32 * c, v);
          tmem_wait_ld32(v);
#pragma unroll
          for (int g = 0; g < 2; ++g) {
            const Scale x = sc[2 * c + g];
            const float k = kq * x.key;
            if (masked) {
#pragma unroll
              for (int i = 0; i < 16; ++i) {
                const float y = fmaf(__uint_as_float(v[16 * g + i]), k, x.log2_value);
                top = fmaxf(top, t0 + 32 * c + 16 * g + i < lim ? y : -INFINITY);
              }
            } else {
              float y = __uint_as_float(v[16 * g]);
#pragma unroll
              for (int i = 1; i < 16; ++i) y = fmaxf(y, __uint_as_float(v[16 * g + i]));
              top = fmaxf(top, fmaf(y, k, x.log2_value));
            }
          }
        }
        if (__any_sync(kFull, top > m + kLazy)) {
          const float next = top > m + kLazy ? top : m;
          const float a = next == m ? 1.0f : ex2(m - next);
          m = next;
          l *= a;
          if (j > 0) {  // the products up to tile j - 1 ended before these scores
#pragma unroll
            for (int c = 0; c < D / 32; ++c) {
              tmem_ld32_nowait(o_col + 32 * c, v);
              tmem_wait_ld32(v);
#pragma unroll
              for (int i = 0; i < 32; ++i) v[i] = __float_as_uint(__uint_as_float(v[i]) * a);
              tmem_st32(o_col + 32 * c, v);
            }
          }
        }
        const float ref = m == -INFINITY ? 0.0f : m;
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          tmem_ld32_nowait(s_col + 32 * c, v);
          tmem_wait_ld32(v);
          uint32_t w[16];
#pragma unroll
          for (int g = 0; g < 2; ++g) {
            const Scale x = sc[2 * c + g];
            const float k = kq * x.key, off = x.log2_value - ref;
            float pr[16];
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              float y = fmaf(__uint_as_float(v[16 * g + i]), k, off);
              if (masked && t0 + 32 * c + 16 * g + i >= lim) y = -INFINITY;
              pr[i] = ex2(y);
            }
            float sum = 0.0f;
#pragma unroll
            for (int i = 0; i < 16; i += 2) {
              sum += pr[i] + pr[i + 1];
              w[8 * g + i / 2] = pack_half2(pr[i], pr[i + 1]);
            }
            // a page without a number counts only where it is seen
            l += sum == 0.0f ? 0.0f : sum * x.inv_value;
          }
          tmem_st16(s_col + 16 * c, w);
        }
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_full[t]);
      }
      if (ok && warp_wait(&o_done[t], 0, fail)) {
        tc_fence_after();
        const float inv = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
        for (int c = 0; c < D / 32; ++c) {
          uint32_t v[32];
          tmem_ld32_nowait(o_col + 32 * c, v);
          tmem_wait_ld32(v);
          if (active) {
            uint4* out = reinterpret_cast<uint4*>(p.out + orow * D + 32 * c);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              uint32_t w[4];
#pragma unroll
              for (int x = 0; x < 4; ++x)
                w[x] = pack_out<T>(__uint_as_float(v[8 * i + 2 * x]) * inv,
                                   __uint_as_float(v[8 * i + 2 * x + 1]) * inv);
              out[i] = make_uint4(w[0], w[1], w[2], w[3]);
            }
          }
        }
        if (active && p.lse)
          p.lse[orow] = l == 0.0f ? -INFINITY : (m + log2f(l)) * 0.693147180559945309f;
      }
    }
  } else if (warp < kMmaWarp) {
    // ---------------------------------------------- codes to fp16 tiles
    constexpr int kLanes = D / 16;          // lanes of a row, 16 codes each
    constexpr int kRows = 32 / kLanes;      // rows of one load of the warp
    const int cw = warp - kSoftWarps;
    const int c = lane % kLanes;
    const int last = (len - 1) >> p.page_shift;
    const int mask = (1 << p.page_shift) - 1;
    const int32_t* table = p.table + tile.x * p.width;
    // pages of the two 16-token groups of this warp's 32 tokens of tile j
    auto page_of = [&](int j, int half) {
      const int i = min((j * kN + cw * 32 + half * 16) >> p.page_shift, last);
      return (int64_t)min(max((int64_t)__ldg(table + i), (int64_t)0), p.pages - 1);
    };
    auto load = [&](uint4 (&r)[kLanes], const int8_t* codes, int j, const int64_t (&page)[2]) {
#pragma unroll
      for (int i = 0; i < kLanes; ++i) {
        const int in = i * kRows + lane / kLanes;  // row of the warp's 32
        const int tok = j * kN + cw * 32 + in;
        const int64_t pg = i * kRows < 16 ? page[0] : page[1];
        r[i] = make_uint4(0, 0, 0, 0);
        if (tok < len)
          r[i] = __ldg(reinterpret_cast<const uint4*>(
              codes + ((((pg * p.kv_heads + h) << p.page_shift) + (tok & mask)) * D) + c * 16));
      }
    };
    auto convert = [&](unsigned char* dst, const uint4 (&r)[kLanes]) {
      // lanes of the upper half of a row write their second chunk first, so that
      // eight lanes of a store hit eight different bank groups
      const int swap = (c >> 2) & 1;
#pragma unroll
      for (int i = 0; i < kLanes; ++i) {
        const int row = cw * 32 + i * kRows + lane / kLanes;
        unsigned char* at = dst + (c / 4) * LY::kAtom;
        const uint32_t x[4] = {r[i].x ^ 0x80808080u, r[i].y ^ 0x80808080u, r[i].z ^ 0x80808080u,
                               r[i].w ^ 0x80808080u};
        const uint4 a = make_uint4(halves(x[0], 0x4140), halves(x[0], 0x4342),
                                   halves(x[1], 0x4140), halves(x[1], 0x4342));
        const uint4 b = make_uint4(halves(x[2], 0x4140), halves(x[2], 0x4342),
                                   halves(x[3], 0x4140), halves(x[3], 0x4342));
        const int ch = (c % 4) * 2;
        *reinterpret_cast<uint4*>(at + atom_byte(row, ch + swap)) = swap ? b : a;
        *reinterpret_cast<uint4*>(at + atom_byte(row, ch + 1 - swap)) = swap ? a : b;
      }
    };
    // lane g < 8 of the first of these warps: scales of the tile's group g
    float s_key = 0.0f, s_value = 0.0f;
    auto load_scales = [&](int j) {
      if (cw == 0 && lane < 8) {
        const int i = min((j * kN + lane * 16) >> p.page_shift, last);
        const int64_t pg = min(max((int64_t)__ldg(table + i), (int64_t)0), p.pages - 1);
        s_key = __ldg(p.ks + pg * p.kv_heads + h);
        s_value = __ldg(p.vs + pg * p.kv_heads + h);
      }
    };
    uint4 rk[kLanes], rv[kLanes];
    int64_t page[2] = {page_of(0, 0), page_of(0, 1)};
    load(rk, p.k, 0, page);
    load_scales(0);
    load(rv, p.v, 0, page);
    bool ok = true;
    for (int j = 0; j < tiles; ++j) {
      const int st = j & 1;
      const int64_t next[2] = {page_of(j + 1, 0), page_of(j + 1, 1)};
      if (j >= 2 && !(ok = warp_wait(&k_empty[st], ((j >> 1) - 1) & 1, fail))) break;
      convert(sm_k + st * LY::kTile, rk);
      if (cw == 0) {
        if (lane < 8) {
          Scale x{s_key, 0.0f, 0.0f, 0.0f};
          value_scale(s_value, &x.log2_value, &x.inv_value);
          sm_scale[(j % kScaleRing) * 8 + lane] = x;
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&scale_full[j % kScaleRing]);
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(&k_full[st]);
      if (j + 1 < tiles) {
        load(rk, p.k, j + 1, next);
        load_scales(j + 1);
      }
      if (j >= 2 && !(ok = warp_wait(&v_empty[st], ((j >> 1) - 1) & 1, fail))) break;
      convert(sm_v + st * LY::kTile, rv);
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(&v_full[st]);
      if (j + 1 < tiles) load(rv, p.v, j + 1, next);
    }
  } else if (lane == 0) {
    // ------------------------------------------------------------ products
    auto scores = [&](int t, int st) {
#pragma unroll
      for (int k = 0; k < D / 16; ++k)
        umma_f16(tmem + LY::kScore + t * kN,
                 sw128_desc(sm_q + t * LY::kTile + (k / 4) * LY::kAtom + (k % 4) * 32),
                 sw128_desc(sm_k + st * LY::kTile + (k / 4) * LY::kAtom + (k % 4) * 32),
                 idesc(kN, false), k != 0);
    };
    auto results = [&](int t, int st, bool first) {
#pragma unroll
      for (int k = 0; k < kN / 16; ++k)
        umma_f16_ts(tmem + LY::kResult + t * D, tmem + LY::kScore + t * kN + 8 * k,
                    sw128_mn_desc(sm_v + st * LY::kTile + k * 16 * 128, LY::kAtom),
                    idesc(D, true), !first || k != 0);
    };
    const int both = two ? 2 : 1;
    bool ok = lane_wait(&q_full, 0, fail) && lane_wait(&k_full[0], 0, fail);
    if (ok) {
      tc_fence_after();
      for (int t = 0; t < both; ++t) {
        scores(t, 0);
        umma_commit(&s_full[t]);
      }
      umma_commit(&k_empty[0]);
    }
    for (int j = 0; j < tiles && ok; ++j) {
      const int st = j & 1;
      ok = lane_wait(&v_full[st], (j >> 1) & 1, fail);
      for (int t = 0; t < both && ok; ++t) {
        if (!(ok = lane_wait(&p_full[t], j & 1, fail))) break;
        tc_fence_after();
        results(t, st, j == 0);
        if (t + 1 == both) umma_commit(&v_empty[st]);
        if (j + 1 < tiles) {
          if (t == 0 && !(ok = lane_wait(&k_full[st ^ 1], ((j + 1) >> 1) & 1, fail))) break;
          tc_fence_after();
          scores(t, st ^ 1);
          umma_commit(&s_full[t]);
          if (t + 1 == both) umma_commit(&k_empty[st ^ 1]);
        } else {
          umma_commit(&o_done[t]);
        }
      }
    }
    // whatever happened, nothing is in flight when tensor memory is given back
    umma_commit(&drained);
    mbar_wait(&drained, 0, kProbes);
  }

  __syncwarp();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == kMmaWarp) tmem_dealloc(tmem, kTmemCols);
  if (threadIdx.x == 0 && sh_fail) atomicOr(p.status, GRM_B200_PLAN_WAIT);
}

template <typename T, int D>
int launch(const AttendParams& p, int64_t blocks, cudaStream_t st) {
  auto kernel = prompt_kernel<T, D>;
  const cudaError_t e = cudaFuncSetAttribute(
      kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, PromptLayout<D>::kSmem);
  if (e != cudaSuccess) {
    set_thread_error("paged attend: %s", cudaGetErrorString(e));
    return cuda_status(e);
  }
  kernel<<<(unsigned)blocks, kPromptThreads, PromptLayout<D>::kSmem, st>>>(p);
  return launch_status("paged attend");
}

}  // namespace

int launch_prompt(int dtype, int dim, const AttendParams& p, int64_t blocks, cudaStream_t st) {
  if (dtype == GRM_B200_F16)
    return dim == 64 ? launch<__half, 64>(p, blocks, st) : launch<__half, 128>(p, blocks, st);
  return dim == 64 ? launch<__nv_bfloat16, 64>(p, blocks, st)
                   : launch<__nv_bfloat16, 128>(p, blocks, st);
}

}  // namespace paged
}  // namespace grm_b200
