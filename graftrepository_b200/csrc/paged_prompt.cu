// paged_prompt.cu -- attention over the 8-bit paged arena for many query rows.
//
// The same sums as the split kernel's (paged_attend.cu): with key codes a_t and
// value codes b_t, key scale s_t and value scale u_t,
//   y_t = scale * log2(e) * s_t (q . a_t) + log2(u_t),  p_t = 2^(y_t - m),
//   out = sum_t p_t b_t / sum_t (p_t / u_t), the fp16 operand being 2^7 p_t,
// here bound by arithmetic: 4 head_dim operations a (row, visible token) on the
// tensor cores and one exponential, 16 a clock and SM against 4,096 fp16
// multiply-adds, so at head_dim 128 a 128 x 128 tile costs the two units about
// the same 1,024 clocks.
//
// A block takes 2 x 128 query rows of one kv head (rows of the group's heads
// side by side, so a key tile serves all of them) and walks the visible tokens
// 128 at a time, 64 in a step of the softmax:
//   warps 0-3, 4-7  softmax of query tile 0 / 1, one row a thread: scores from
//                   tensor memory, p back as fp16 over them, and when a row's
//                   reference exponent has to move (rarely: it trails by up
//                   to 8), its result in tensor memory rescaled
//   warps 8-11      codes in shared memory to fp16 key and value tiles (two of
//                   each)
//   warps 12, 13    a query tile's products, S = Q K^T and O += P V (P from
//                   tensor memory), issued by one elected lane.  A thread that
//                   waits on a barrier first sees its own commits out of the
//                   queue of products, so with one thread for both tiles the
//                   tensor cores ran dry at every wait, about 250 clocks each
//   warp 14         codes from their pages to shared memory, one bulk copy a page
// While one query tile's softmax runs, the tensor cores work for the other, and
// the two softmax warps of a scheduler take turns at the exponentials.  At
// head_dim 256 a result tile takes half of tensor memory: one query tile, key
// tiles of 64 tokens, and warps 4-11 convert.  At head_dim 64 and 256 there is
// room for the queries in tensor memory, too, so that the products read keys and
// values alone from shared memory, and for two places of codes.
// Keys and values have the same layout in shared memory, 128-byte rows of 64
// dims with a 128-byte swizzle: K is read K-major, V with its dims contiguous.
// A block whose rows fit one tile leaves the other tile's work out.
//
// Few tiles over long contexts are cut along their tokens into parts, a block
// each; the split kernel, which runs after this one, joins them.
//
// 8,449 rows of 3 requests (1.4 TFLOP at 8 kv heads, 32 query heads, head_dim 128)
// take 1.27 ms alone, 1.12 PFLOP/s, and 1.39 to 1.44 in a row of calls, where the
// power cap lowers the clocks; at head_dim 64 1.13 ms (exponentials 0.60, products
// 0.42 at the units' rates), at head_dim 256 2.6 to 2.9 ms (products 1.66).  What
// bounds it now is the softmax warps' chain of dependent steps: per 64 tokens about
// 1,900 clocks, where the exponentials alone need 1,024 (both warps of a scheduler),
// the tensor cores as many, and shared memory 1,536.  On the way: both warps of a
// scheduler in the same phase 1.51 ms, in turns 1.43; then, where each product had
// had a predicate of its own (80 clocks of issue apiece), an elected branch 1.33;
// arithmetic two at a time 1.27.
#include <type_traits>

#include "paged.cuh"
#include "umma.cuh"

namespace grm_b200 {
namespace paged {

namespace {

constexpr int kM = 128;             // rows of a query tile
constexpr int kHalf = 64;           // tokens of one softmax step
constexpr int kQueryAtom = kM * 128;  // 128 rows x 64 halves
constexpr int kPromptThreads = 15 * 32;
constexpr int kMmaWarp = 12, kLoadWarp = 14;
constexpr uint32_t kTmemCols = 512;

// Two query tiles and key tiles of 128 tokens, in two steps of the softmax; at
// head_dim 256, whose results alone take half of tensor memory, one query tile
// and key tiles of one step, and the other tile's softmax warps convert codes.
template <int D>
struct PromptLayout {
  static constexpr int kQueries = prompt_rows_of(D) / kM;  // query tiles
  static constexpr int kN = prompt_step_of(D);          // tokens of a key tile
  static constexpr int kHalves = kN / kHalf;
  static constexpr int kSoftWarps = 4 * kQueries;
  static constexpr int kConvWarps = kMmaWarp - kSoftWarps;
  static constexpr int kRing = 16 / kHalves;            // key tiles whose scales are held
  // Queries in tensor memory, where the results leave room for them: the products
  // then read keys and values alone from shared memory.
  static constexpr bool kQTmem = kQueries * (2 * kHalf + D + D / 2) <= (int)kTmemCols;
  static constexpr int kQuery = kQTmem ? 0 : (D / 64) * kQueryAtom;  // a query tile
  static constexpr int kAtom = kN * 128;                // kN rows x 64 halves
  static constexpr int kTile = (D / 64) * kAtom;        // a key or value tile
  static constexpr int kRaw = kN * D;                   // its codes
  // places for a side's codes: two where shared memory has room, so that a copy's
  // latency hides behind a conversion
  static constexpr int kRaws = kQTmem ? 2 : 1;
  static constexpr int kGroups = kN / 16;               // pages' scales of a key tile
  static constexpr int kScaleBytes = kRing * kGroups * 16;
  static constexpr int kUsed =
      1024 + kQueries * kQuery + 4 * kTile + 2 * kRaws * kRaw + kScaleBytes;
  // one block an SM: it owns all of tensor memory
  static constexpr int kSmem = kUsed > 120 * 1024 ? kUsed : 120 * 1024;
  static constexpr uint32_t kScore = 0;                 // tensor memory columns
  static constexpr uint32_t kResult = kQueries * 2 * kHalf;
  static constexpr uint32_t kQueryCol = kResult + kQueries * D;
  static_assert(kQueryCol + (kQTmem ? kQueries * D / 2 : 0) <= kTmemCols, "tiles");
};

// fp32 accumulators, fp16 operands, 128 rows, N columns; B K-major or (bit 16) not.
__host__ __device__ constexpr uint32_t idesc(int n, bool b_mn) {
  return (1u << 4) | (b_mn ? 1u << 16 : 0u) | ((uint32_t)(n >> 3) << 17) |
         ((uint32_t)(kM >> 4) << 24);
}

// Byte of 16-byte chunk c (8 halves of 64) of row r in a swizzled atom.
__device__ __forceinline__ uint32_t atom_byte(int r, int c) {
  return r * 128 + ((c ^ (r & 7)) << 4);
}

__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
__device__ __forceinline__ float max3(uint32_t a, uint32_t b, uint32_t c) {
  return max3(__uint_as_float(a), __uint_as_float(b), __uint_as_float(c));
}
// Two numbers at a time.
__device__ __forceinline__ float2 fma2(float a, float b, float k, float o) {
  float2 r;
  asm("{\n .reg .b64 x, y, z;\n mov.b64 x, {%2, %3};\n mov.b64 y, {%4, %4};\n"
      " mov.b64 z, {%5, %5};\n fma.rn.f32x2 x, x, y, z;\n mov.b64 {%0, %1}, x;\n}\n"
      : "=f"(r.x), "=f"(r.y)
      : "f"(a), "f"(b), "f"(k), "f"(o));
  return r;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 r;
  asm("{\n .reg .b64 x, y;\n mov.b64 x, {%2, %3};\n mov.b64 y, {%4, %5};\n"
      " add.rn.f32x2 x, x, y;\n mov.b64 {%0, %1}, x;\n}\n"
      : "=f"(r.x), "=f"(r.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return r;
}
// Every lane of a warp waits; false, for all of them, when a wait gave up.
// The loops of this kernel share an instruction cache that they barely fit, so
// what is not the common path stays out of line.
__device__ __noinline__ bool wait_long(uint64_t* bar, unsigned parity, volatile int* fail,
                                       unsigned probes) {
  bool ok = false;
  for (unsigned i = 0; i < probes; ++i) {
    if ((ok = mbar_try_wait(bar, parity))) break;
    if (*fail) break;
  }
  ok = __all_sync(kFull, ok);
  if (!ok) *fail = 1;
  return ok;
}
__device__ __forceinline__ bool warp_wait(uint64_t* bar, unsigned parity, volatile int* fail,
                                          unsigned probes) {
  if (__all_sync(kFull, mbar_try_wait(bar, parity))) return true;
  return wait_long(bar, parity, fail, probes);
}

struct Scale {
  float key, log2_value, inv_value, unused;
};
static_assert(sizeof(Scale) == 16, "PromptLayout::kScaleBytes");

// Row `row` of query tile t of a block in which a wait gave up: no numbers.
template <int D>
__device__ __noinline__ void lose_row(const AttendParams& p, int4 e, int h, int t, int row) {
  const PromptTile pt = prompt_tile<D>(p, e);
  if (row >= (t == 0 ? pt.toks[0] : pt.toks[1]) * p.group) return;
  const float nan = __int_as_float(0x7FC00000);
  if (pt.parts > 1) {  // the sum of its part
    float* slot = p.l.qpart + ((int64_t)(e.w + (e.z & 255)) * p.kv_heads + h) * prompt_slot(D);
    *reinterpret_cast<float2*>(slot + prompt_rows_of(D) * D + 2 * (t * kM + row)) =
        make_float2(-INFINITY, nan);
    return;
  }
  const int64_t orow = (int64_t)(pt.start + pt.tok0 + t * pt.per + row / p.group) * p.kv_heads *
                           p.group + h * p.group + row % p.group;
  for (int c = 0; c < D / 8; ++c)
    reinterpret_cast<uint4*>(p.out + orow * D)[c] =
        make_uint4(0x7FFF7FFFu, 0x7FFF7FFFu, 0x7FFF7FFFu, 0x7FFF7FFFu);
  if (p.lse) p.lse[orow] = nan;
}

template <typename T, int D>
__global__ void __launch_bounds__(kPromptThreads, 1)
    prompt_kernel(const __grid_constant__ AttendParams p) {
  using LY = PromptLayout<D>;
  constexpr int kN = LY::kN, kHalves = LY::kHalves, kRing = LY::kRing, kRaws = LY::kRaws;
  extern __shared__ unsigned char raw[];
  unsigned char* const sm = raw + ((1024u - (smem_u32(raw) & 1023u)) & 1023u);
  unsigned char* const sm_q = sm;                                     // [kQueries]
  unsigned char* const sm_k = sm + LY::kQueries * LY::kQuery;         // [2]
  unsigned char* const sm_v = sm_k + 2 * LY::kTile;                   // [2]
  unsigned char* const sm_raw = sm_v + 2 * LY::kTile;                 // codes: [kRaws][2 sides]
  Scale* const sm_scale =
      reinterpret_cast<Scale*>(sm_raw + 2 * kRaws * LY::kRaw);        // [kRing][kGroups]
  __shared__ __align__(8) uint64_t q_full[2], drained[2], k_full[2], k_empty[2], v_full[2],
      v_empty[2], scale_full[kRing], raw_full[2][kRaws], raw_empty[2][kRaws], s_full[2][2],
      p_full[2][2], o_full[2], o_done[2], turn[2][4];
  __shared__ uint32_t sh_tmem;
  __shared__ int sh_fail;

  const Header hd = *p.l.header;
  const int h = blockIdx.x % p.kv_heads;
  const int ti = (int)(blockIdx.x / p.kv_heads);  // the longest come first in the list
  if (ti >= hd.qtiles) return;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int4 tile = p.l.qtiles[ti];
  const PromptTile pt = prompt_tile<D>(p, tile);
  const int start = pt.start, len = pt.len, cached = pt.cached, tok0 = pt.tok0, per = pt.per;
  const int all_tiles = pt.steps, parts = pt.parts, part = tile.z & 255;
  const bool two = pt.toks[1] > 0;
  const int heads = p.kv_heads * p.group;
  if (part >= parts) return;
  // the block's share of the key tiles, and the tokens that its rows see in it
  const int tile0 = (int)((int64_t)all_tiles * part / parts);
  const int tiles = (int)((int64_t)all_tiles * (part + 1) / parts) - tile0;
  const int tok_base = tile0 * kN;
  const int sees = p.causal ? min(len, cached + tok0 + pt.toks[0] + pt.toks[1]) : len;
  const int halves_seen = (min(sees - tok_base, tiles * kN) + kHalf - 1) / kHalf;

  if (all_tiles == 0) {  // nothing cached: empty rows
    const int values = (pt.toks[0] + pt.toks[1]) * p.group * (D / 2);
    for (int x = threadIdx.x; x < values; x += kPromptThreads) {
      const int j = x / (D / 2);
      const int64_t row = (int64_t)(start + tok0 + j / p.group) * heads + h * p.group + j % p.group;
      reinterpret_cast<uint32_t*>(p.out + row * D)[x % (D / 2)] = 0;
      if (p.lse && x % (D / 2) == 0) p.lse[row] = -INFINITY;
    }
    return;
  }

  if (threadIdx.x == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(&q_full[i], 4);
      mbar_init(&drained[i], 1);
      mbar_init(&k_full[i], LY::kConvWarps);
      mbar_init(&k_empty[i], two ? 2 : 1);
      mbar_init(&v_full[i], LY::kConvWarps);
      mbar_init(&v_empty[i], two ? 2 : 1);
      for (int x = 0; x < kRaws; ++x) {
        mbar_init(&raw_full[i][x], 1);
        mbar_init(&raw_empty[i][x], LY::kConvWarps);
      }
      for (int x = 0; x < 2; ++x) {
        mbar_init(&s_full[i][x], 1);
        mbar_init(&p_full[i][x], 4);
      }
      mbar_init(&o_full[i], 1);
      mbar_init(&o_done[i], 1);
      for (int x = 0; x < 4; ++x) mbar_init(&turn[i][x], 1);
    }
    for (int i = 0; i < kRing; ++i) mbar_init(&scale_full[i], 1);
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

  if (warp < LY::kSoftWarps) {
    // ------------------------------------------------------------- softmax
    const int t = warp >> 2;
    if (t == 0 || two) {
      const int row = (warp & 3) * 32 + lane;
      const bool active = row < (t == 0 ? pt.toks[0] : pt.toks[1]) * p.group;
      const int token = tok0 + t * per + row / p.group;
      // tokens that the row sees, from the part's first on
      const int lim = (active && p.causal ? cached + token + 1 : len) - tok_base;

      // the row as fp16 (a bf16 row scaled by a power of two), to shared memory
      float kq = p.scale_log2, up = 1.0f;
      const uint4* qp = reinterpret_cast<const uint4*>(
          p.q + (int64_t)(start + token) * p.q_row +
          (int64_t)(h * p.group + row % p.group) * p.q_head);
      if constexpr (!std::is_same<T, __half>::value) {
        unsigned m = 0;
        if (active)
#pragma unroll 8
          for (int c = 0; c < D / 8; ++c) {
            const uint4 x = __ldg(qp + c);
            m = __vmaxu2(m, __vmaxu2(x.x & 0x7FFF7FFFu, x.y & 0x7FFF7FFFu));
            m = __vmaxu2(m, __vmaxu2(x.z & 0x7FFF7FFFu, x.w & 0x7FFF7FFFu));
          }
        row_scale(max(m & 0xFFFFu, m >> 16), &up, &kq);
        kq *= p.scale_log2;
      }
      const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
      auto chunk = [&](int c) {  // eight values
        uint4 x = active ? __ldg(qp + c) : make_uint4(0, 0, 0, 0);
        if constexpr (!std::is_same<T, __half>::value)
          x = make_uint4(scale_pair(x.x, up), scale_pair(x.y, up), scale_pair(x.z, up),
                         scale_pair(x.w, up));
        return x;
      };
      if constexpr (LY::kQTmem) {
#pragma unroll 1
        for (int c = 0; c < D / 8; c += 4) {
          uint32_t w[16];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const uint4 x = chunk(c + i);
            w[4 * i] = x.x;
            w[4 * i + 1] = x.y;
            w[4 * i + 2] = x.z;
            w[4 * i + 3] = x.w;
          }
          tmem_st16(tmem + lanes + LY::kQueryCol + t * (D / 2) + 4 * c, w);
        }
        tmem_wait_st();
        tc_fence_before();
      } else {
#pragma unroll 4
        for (int c = 0; c < D / 8; ++c)
          *reinterpret_cast<uint4*>(sm_q + t * LY::kQuery + (c / 8) * kQueryAtom +
                                    atom_byte(row, c % 8)) = chunk(c);
        fence_proxy_async_smem();
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&q_full[t]);

      const uint32_t s_col = tmem + lanes + LY::kScore + t * 2 * kHalf;
      const uint32_t o_col = tmem + lanes + LY::kResult + t * D;
      float m = -INFINITY, l = 0.0f;
      bool ok = true;
#pragma unroll 1
      for (int i = 0; i < halves_seen; ++i) {
        const int j = i / kHalves, buf = i & 1;
        if (i % kHalves == 0 && !(ok = wait(&scale_full[j % kRing], (j / kRing) & 1)))
          break;
        if (!(ok = wait(&s_full[t][buf], (i >> 1) & 1))) break;
        tc_fence_after();
        // the row's 64 scores, in registers from here on
        uint32_t v[2][32];
        tmem_ld32_nowait(s_col + buf * kHalf, v[0]);
        tmem_ld32_nowait(s_col + buf * kHalf + 32, v[1]);
        // factors and offsets of the exponents of 4 x 16 tokens
        const Scale* sc = sm_scale + i % 16 * 4;  // the ring holds sixteen halves
        float fk[4], fo[4];
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          fk[g] = kq * sc[g].key;
          fo[g] = sc[g].log2_value;
        }
        tmem_wait_ld32(v[0]);
        tmem_wait_ld32(v[1]);
        // Hidden tokens: scores of -inf, with factors kept above 0.  16 tokens that
        // are all hidden from the row take factor 1 and offset 0, so that a page
        // without a number does not reach it.
        if (__any_sync(kFull, (i + 1) * kHalf > lim)) {
#pragma unroll
          for (int x = 0; x < kHalf; ++x)
            if (i * kHalf + x >= lim) v[x / 32][x % 32] = 0xFF800000u;
#pragma unroll
          for (int g = 0; g < 4; ++g) {
            const bool hidden = i * kHalf + 16 * g >= lim;
            fk[g] = hidden ? 1.0f : fk[g] == 0.0f ? 0x1p-126f : fk[g];
            fo[g] = hidden ? 0.0f : fo[g];
          }
        }
        float top = -INFINITY;
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const uint32_t* x = v[g / 2] + 16 * (g % 2);
          const float y = max3(max3(max3(x[0], x[1], x[2]), max3(x[3], x[4], x[5]),
                                    max3(x[6], x[7], x[8])),
                               max3(x[9], x[10], x[11]),
                               max3(max3(x[12], x[13], x[14]), __uint_as_float(x[15]),
                                    -INFINITY));
          top = fmaxf(top, fmaf(y, fk[g], fo[g]));
        }
        if (__any_sync(kFull, top > m + kLazy)) {
          const float next = top > m + kLazy ? reference_of(top) : m;
          const float a = next == m ? 1.0f : ex2(m - next);
          m = next;
          l *= a;
          if (i > 0) {  // once the products of the half before have ended
            if (!(ok = wait(&o_full[t], (i - 1) & 1))) break;
            tc_fence_after();
#pragma unroll 1
            for (int c = 0; c < D / 16; ++c) {
              uint32_t o[16];
              tmem_ld16(o_col + 16 * c, o);
#pragma unroll
              for (int x = 0; x < 16; ++x) o[x] = __float_as_uint(__uint_as_float(o[x]) * a);
              tmem_st16(o_col + 16 * c, o);
            }
          }
        }
        // The two warps of a scheduler take turns at the exponentials, so that one's
        // other work lies under them.
        if (two && t + i > 0 &&
            !(ok = wait(&turn[t][warp & 3], (i - 1 + t) & 1)))
          break;
        const float ref = m == -INFINITY ? 0.0f : m - kLift;
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          uint32_t w[16];
#pragma unroll
          for (int h2 = 0; h2 < 2; ++h2) {
            const int g = 2 * c + h2;
            const float k = fk[g], off = fo[g] - ref;
            float2 sum = make_float2(0.0f, 0.0f);
#pragma unroll
            for (int x = 0; x < 16; x += 2) {
              const float2 y = fma2(__uint_as_float(v[c][16 * h2 + x]),
                                    __uint_as_float(v[c][16 * h2 + x + 1]), k, off);
              const float2 e = make_float2(ex2(y.x), ex2(y.y));
              sum = add2(sum, e);
              w[8 * h2 + x / 2] = pack_half2(e.x, e.y);
            }
            l = fmaf(sum.x + sum.y, sc[g].inv_value, l);
            // three quarters done: the other's first ones fill the gaps of the last
            if (g == 2 && two && lane == 0) mbar_arrive(&turn[1 - t][warp & 3]);
          }
          tmem_st16(s_col + buf * kHalf + 16 * c, w);
        }
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_full[t][buf]);
      }
      if (ok && wait(&o_done[t], 0)) {
        tc_fence_after();
        // looked up again rather than kept in registers through the loop
        int tid;
        asm volatile("mov.u32 %0, %%tid.x;" : "=r"(tid));
        const int4 e = p.l.qtiles[ti];
        const PromptTile pt = prompt_tile<D>(p, e);
        const int t = tid >> 7, row = tid & 127;
        const bool active = row < (t == 0 ? pt.toks[0] : pt.toks[1]) * p.group;
        const int64_t orow = (int64_t)(pt.start + pt.tok0 + t * pt.per + row / p.group) * heads +
                             h * p.group + row % p.group;
        if (pt.parts > 1) {  // the part's result, for the split kernel to join
          float* slot = p.l.qpart +
                        ((int64_t)(e.w + (e.z & 255)) * p.kv_heads + h) * prompt_slot(D);
          float4* to = reinterpret_cast<float4*>(slot) + t * kM + row;
#pragma unroll 1
          for (int c = 0; c < D / 16; ++c) {
            uint32_t v[16];
            tmem_ld16(o_col + 16 * c, v);
            if (active)
#pragma unroll
              for (int i = 0; i < 4; ++i)
                to[(4 * c + i) * prompt_rows_of(D)] =
                    make_float4(__uint_as_float(v[4 * i]), __uint_as_float(v[4 * i + 1]),
                                __uint_as_float(v[4 * i + 2]), __uint_as_float(v[4 * i + 3]));
          }
          if (active)
            *reinterpret_cast<float2*>(slot + prompt_rows_of(D) * D + 2 * (t * kM + row)) =
                make_float2(m, l);
        } else {
          const float inv = l == 0.0f ? 0.0f : kUnlift / l;
#pragma unroll 1
          for (int c = 0; c < D / 16; ++c) {
            uint32_t v[16];
            tmem_ld16(o_col + 16 * c, v);
            if (active) {
              uint4* out = reinterpret_cast<uint4*>(p.out + orow * D + 16 * c);
#pragma unroll
              for (int i = 0; i < 2; ++i) {
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
    }
  } else if (warp < kMmaWarp) {
    // ---------------------------------------------- codes to fp16 tiles
    constexpr int kLanes = D / 16;          // lanes of a row, 16 codes each
    constexpr int kRows = 32 / kLanes;      // rows of one load of the warp
    // Eight lanes together take the first half of one row's codes and the second
    // half of the next row's: reads in 8 different bank groups, and writes too,
    // the swizzle putting what an even row's lanes write, 32 bytes apart, into
    // even places of 16 bytes and what an odd row's write into odd ones.
    const int odd = kLanes == 4 ? 0 : (lane >> 2) & 1;
    const int c = kLanes == 4 ? lane & 3
                              : (lane & 3) + (((lane >> 3) ^ odd) & (kLanes / 4 - 1)) * 4;
    const int row0 = (warp - LY::kSoftWarps) * (kN / LY::kConvWarps) +
                     (kLanes == 4 ? lane >> 2 : kLanes == 8 ? odd + (lane >> 4) * 2 : odd);
    // places of a lane's two chunks, less the row's: the swizzle repeats every 8 rows
    constexpr int kPlaces = 8 / kRows;
    uint32_t put[kPlaces][2];
#pragma unroll
    for (int i = 0; i < kPlaces; ++i)
#pragma unroll
      for (int x = 0; x < 2; ++x)
        put[i][x] = atom_byte(row0 + kRows * i, (c % 4) * 2 + x) - kRows * i * 128;
    bool ok = true;
#pragma unroll 1
    for (int x = 0; x < 2 * tiles; ++x) {  // keys, values, keys, ...
      const int j = x >> 1, side = x & 1, st = j & 1, place = j % kRaws;
      const unsigned char* src = sm_raw + (place * 2 + side) * LY::kRaw + row0 * D + c * 16;
      unsigned char* at = (side ? sm_v : sm_k) + st * LY::kTile + (c / 4) * LY::kAtom;
      if (!(ok = wait(&raw_full[side][place], (j / kRaws) & 1))) break;
      uint4 r[4];
      auto load = [&] {
#pragma unroll
        for (int i = 0; i < 4; ++i)
          r[i] = *reinterpret_cast<const uint4*>(src + i * kRows * D);
        src += 4 * kRows * D;
      };
      load();
      if (j >= 2 &&
          !(ok = wait(side ? &v_empty[st] : &k_empty[st], ((j >> 1) - 1) & 1)))
        break;
#pragma unroll 1
      for (int i0 = 0; i0 < kN / LY::kConvWarps / kRows; i0 += 4) {
        if (i0 > 0) load();
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint32_t x[4] = {r[i].x ^ 0x80808080u, r[i].y ^ 0x80808080u,
                                 r[i].z ^ 0x80808080u, r[i].w ^ 0x80808080u};
          const uint4 lo = make_uint4(halves(x[0], 0x4140), halves(x[0], 0x4342),
                                      halves(x[1], 0x4140), halves(x[1], 0x4342));
          const uint4 hi = make_uint4(halves(x[2], 0x4140), halves(x[2], 0x4342),
                                      halves(x[3], 0x4140), halves(x[3], 0x4342));
          *reinterpret_cast<uint4*>(at + i * kRows * 128 + put[i % kPlaces][0]) = lo;
          *reinterpret_cast<uint4*>(at + i * kRows * 128 + put[i % kPlaces][1]) = hi;
        }
        at += 4 * kRows * 128;
      }
      // the tile for the tensor cores, the codes' place for the next copy
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(&raw_empty[side][place]);
        mbar_arrive(side ? &v_full[st] : &k_full[st]);
      }
    }
  } else {
    if (warp < kLoadWarp) {
      // ---------------------------------------------------------- products
      // The whole warp runs this, an elected lane issues; what the instructions read
      // is the same in every lane and known to be (broadcast), so that it stays in
      // uniform registers.
      const int t = __shfl_sync(kFull, warp, 0) - kMmaWarp;
      const int steps = __shfl_sync(kFull, halves_seen, 0);
      const uint32_t base = __shfl_sync(kFull, tmem, 0);
      if (t == 0 || two) {
        // Descriptors of the first step; later steps and stages add to the address
        // field (16-byte units), which no tile of shared memory overflows.
        constexpr uint32_t kHi = (uint32_t)(((uint64_t)64 << 32 | (uint64_t)1 << 46 |
                                             (uint64_t)2 << 61) >> 32);
        constexpr uint32_t kTile16 = LY::kTile / 16, kHalf16 = kHalf * 128 / 16;
        const uint32_t q_lo = (uint32_t)sw128_desc(sm_q) + t * (LY::kQuery / 16);
        const uint32_t k_lo = (uint32_t)sw128_desc(sm_k);
        const uint32_t v_lo = (uint32_t)sw128_mn_desc(sm_v, LY::kAtom);
        const uint32_t s_at = base + LY::kScore + t * 2 * kHalf, o_at = base + LY::kResult + t * D;
        const uint32_t q_at = base + LY::kQueryCol + t * (D / 2);
        auto desc = [&](uint32_t lo) { return (uint64_t)kHi << 32 | lo; };
        auto scores = [&](int i) {  // half i of the tokens
          const uint32_t kd = k_lo + ((i / kHalves) & 1) * kTile16 + (i % kHalves) * kHalf16;
          const uint32_t to = s_at + (i & 1) * kHalf;
          if (elect_one()) {
#pragma unroll
            for (int k = 0; k < D / 16; ++k) {
              const uint32_t q_step = ((k / 4) * kQueryAtom + (k % 4) * 32) / 16;
              const uint32_t k_step = ((k / 4) * LY::kAtom + (k % 4) * 32) / 16;
              if constexpr (LY::kQTmem)
                umma_f16_ts(to, q_at + 8 * k, desc(kd + k_step), idesc(kHalf, false), k != 0);
              else
                umma_f16(to, desc(q_lo + q_step), desc(kd + k_step), idesc(kHalf, false), k != 0);
            }
            umma_commit(&s_full[t][i & 1]);
            if ((i + 1) % kHalves == 0) umma_commit(&k_empty[(i / kHalves) & 1]);
          }
          __syncwarp();
        };
        auto results = [&](int i) {
          const uint32_t vd = v_lo + ((i / kHalves) & 1) * kTile16 + (i % kHalves) * kHalf16;
          const uint32_t from = s_at + (i & 1) * kHalf;
          if (elect_one()) {
#pragma unroll
            for (int k = 0; k < kHalf / 16; ++k)
              umma_f16_ts(o_at, from + 8 * k, desc(vd + k * (16 * 128 / 16)), idesc(D, true),
                          i != 0 || k != 0);
            umma_commit(&o_full[t]);
            if ((i + 1) % kHalves == 0) umma_commit(&v_empty[(i / kHalves) & 1]);
            if (i + 1 == steps) umma_commit(&o_done[t]);
          }
          __syncwarp();
        };
        // scores of half i: the first half of a key tile waits for it, the last gives it back
        auto next_scores = [&](int i) {
          const int j = i / kHalves;
          if (i % kHalves == 0) {
            if (!wait(&k_full[j & 1], (j >> 1) & 1)) return false;
            tc_fence_after();
          }
          scores(i);
          return true;
        };
        bool ok = wait(&q_full[t], 0);
        tc_fence_after();
        ok = ok && next_scores(0);
        if (ok && steps > 1) ok = next_scores(1);
#pragma unroll 1
        for (int i = 0; i < steps && ok; ++i) {
          const int j = i / kHalves;
          if (i % kHalves == 0) ok = wait(&v_full[j & 1], (j >> 1) & 1);
          ok = ok && wait(&p_full[t][i & 1], (i >> 1) & 1);
          if (!ok) break;
          tc_fence_after();
          results(i);
          if (i + 2 < steps) ok = next_scores(i + 2);  // in this half's place
        }
        // whatever happened, nothing is in flight when tensor memory is given back
        if (elect_one()) umma_commit(&drained[t]);
        __syncwarp();
        mbar_wait(&drained[t], 0, kProbes);
      }
    } else if (warp == kLoadWarp) {
      // ------------------------------------- codes and scales from their pages
      const int last = (len - 1) >> p.page_shift;
      const int page_tokens = 1 << p.page_shift;
      const unsigned piece = (unsigned)(min(page_tokens, kN) * D);  // codes of a page in a tile
      constexpr int kGroups = LY::kGroups;  // 8 of a key tile, 4 at head_dim 256
      const int group16 = lane & (kGroups - 1);
      auto page_of = [&](int j) {  // lane g < kGroups: page of the tile's tokens 16 g ..
        const int i = min((tok_base + j * kN + group16 * 16) >> p.page_shift, last);
        return min(max(__ldg(p.table + tile.x * p.width + i), 0), (int)p.pages - 1);
      };
      int page = page_of(0);
      int issued[2] = {0, 0};
      // With no probes at all the block gives up here: nothing comes, and everybody's
      // waits run out.  (A look at the limit in every wait costs 2 % of the kernel.)
      bool ok = p.probes > 0;
      for (int j = 0; j < tiles && ok; ++j) {
        const int64_t at = (int64_t)page * p.kv_heads + h;
        const int t0 = tok_base + j * kN + group16 * 16;
        // a lane at the start of a page's share of the tile copies it; a page is
        // copied whole, past the request's last token too
        const bool leads =
            lane < kGroups && t0 <= len - 1 && ((lane * 16) & (page_tokens - 1)) == 0;
        const unsigned bytes = __popc(__ballot_sync(kFull, leads)) * piece;
        const int64_t off = ((at << p.page_shift) + (t0 & (page_tokens - 1))) * D;
        float s_key = 0.0f, s_value = 0.0f;
        if (lane < kGroups) {
          s_key = __ldg(p.ks + at);
          s_value = __ldg(p.vs + at);
        }
        page = page_of(j + 1);
#pragma unroll
        for (int side = 0; side < 2; ++side) {
          const int place = j % kRaws;
          if (j >= kRaws && !(ok = wait(&raw_empty[side][place], (j / kRaws - 1) & 1)))
            break;
          issued[side] = j + 1;
          if (lane == 0) mbar_arrive_expect_tx(&raw_full[side][place], bytes);
          __syncwarp();
          if (leads)
            bulk_g2s(sm_raw + (place * 2 + side) * LY::kRaw + lane * 16 * D,
                     (side ? p.v : p.k) + off, piece, &raw_full[side][place]);
          if (side == 0) {
            if (lane < kGroups) {
              Scale x{s_key, 0.0f, 0.0f, 0.0f};
              value_scale(s_value, &x.log2_value, &x.inv_value);
              sm_scale[(j % kRing) * kGroups + lane] = x;
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(&scale_full[j % kRing]);
          }
        }
      }
      // no copy is in flight when the block ends, whatever happened
#pragma unroll
      for (int side = 0; side < 2; ++side)
        for (int j = max(issued[side] - kRaws, 0); j < issued[side]; ++j)
          mbar_wait(&raw_full[side][j % kRaws], (j / kRaws) & 1, kProbes);
    }
  }

  __syncwarp();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == kMmaWarp) tmem_dealloc(tmem, kTmemCols);
  if (sh_fail) {
    if (warp < LY::kSoftWarps)
      lose_row<D>(p, p.l.qtiles[blockIdx.x / p.kv_heads], blockIdx.x % p.kv_heads,
                  threadIdx.x >> 7, threadIdx.x & 127);
    if (threadIdx.x == 0) atomicOr(p.status, GRM_B200_PLAN_WAIT);
  }
}

template <typename T, int D>
int launch(const AttendParams& p, int64_t blocks, cudaStream_t st) {
  auto kernel = prompt_kernel<T, D>;
  static std::atomic<uint64_t> done{0};
  const int rc =
      allow_shared(reinterpret_cast<const void*>(kernel), PromptLayout<D>::kSmem, &done);
  if (rc) return rc;
  kernel<<<(unsigned)blocks, kPromptThreads, PromptLayout<D>::kSmem, st>>>(p);
  return launch_status("paged attend");
}

}  // namespace

int launch_prompt(int dtype, int dim, const AttendParams& p, int64_t blocks, cudaStream_t st) {
  if (dtype == GRM_B200_F16)
    return dim == 64    ? launch<__half, 64>(p, blocks, st)
           : dim == 128 ? launch<__half, 128>(p, blocks, st)
                        : launch<__half, 256>(p, blocks, st);
  return dim == 64    ? launch<__nv_bfloat16, 64>(p, blocks, st)
         : dim == 128 ? launch<__nv_bfloat16, 128>(p, blocks, st)
                      : launch<__nv_bfloat16, 256>(p, blocks, st);
}

}  // namespace paged
}  // namespace grm_b200
