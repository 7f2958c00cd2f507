// latent_device.cuh -- what the kernels of latent attention share on the device.
#pragma once

#include <algorithm>

#include "latent.cuh"
#include "umma.cuh"

namespace grm_b200 {
namespace latent {
namespace {

template <typename T>
struct Kind;
template <>
struct Kind<__half> {
  static constexpr uint32_t kFormat = 0;
  // Weights times 2^7, at most 2^15: lost at the small end is then what lies below
  // 2^-32 of a row's largest, not 2^-25.
  static constexpr float kLift = paged::kLift;
  static __device__ __forceinline__ uint32_t pack(float a, float b) {
    return paged::pack_half2(a, b);
  }
  static __device__ __forceinline__ float2 widen(uint32_t v) {
    return __half22float2(*reinterpret_cast<const __half2*>(&v));
  }
  static constexpr uint32_t kNoNumber = 0x7C00u;  // exponent bits
};
template <>
struct Kind<__nv_bfloat16> {
  static constexpr uint32_t kFormat = (1u << 7) | (1u << 10);
  static constexpr float kLift = 0.0f;
  static __device__ __forceinline__ uint32_t pack(float a, float b) {
    return paged::pack_out<__nv_bfloat16>(a, b);
  }
  static __device__ __forceinline__ float2 widen(uint32_t v) {
    return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xFFFF0000u));
  }
  static constexpr uint32_t kNoNumber = 0x7F80u;
};

// Byte of 16-byte chunk c of row r: 128-byte rows of 8 chunks, 64-byte rows of 4.
__device__ __forceinline__ uint32_t atom_byte(int r, int c) {
  return r * 128 + ((c ^ (r & 7)) << 4);
}
__device__ __forceinline__ uint32_t half_atom_byte(int r, int c) {
  return r * 64 + ((c ^ ((r >> 1) & 3)) << 4);
}

// Upper word of a shared-memory descriptor (umma.cuh's sw128_desc): 8-row groups of
// 1024 bytes and a 128-byte swizzle, or of 512 and 64.
constexpr uint32_t kHi128 = (uint32_t)(((uint64_t)64 << 32 | (uint64_t)1 << 46 |
                                        (uint64_t)2 << 61) >> 32);
constexpr uint32_t kHi64 = (uint32_t)(((uint64_t)32 << 32 | (uint64_t)1 << 46 |
                                       (uint64_t)4 << 61) >> 32);

__device__ __forceinline__ void tma_load(void* dst, const CUtensorMap* map, int x, int y,
                                         uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%2, %3}], [%4];" ::"r"(smem_u32(dst)),
      "l"(map), "r"(x), "r"(y), "r"(smem_u32(bar))
      : "memory");
}

__device__ __forceinline__ void tma_load(void* dst, const CUtensorMap* map, int x, int y, int z,
                                         uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(smem_u32(dst)),
      "l"(map), "r"(x), "r"(y), "r"(z), "r"(smem_u32(bar))
      : "memory");
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
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
__device__ __forceinline__ float2 fma2(float a, float b, float k, float2 o) {
  float2 r;
  asm("{\n .reg .b64 x, y, z;\n mov.b64 x, {%2, %3};\n mov.b64 y, {%4, %4};\n"
      " mov.b64 z, {%5, %6};\n fma.rn.f32x2 x, x, y, z;\n mov.b64 {%0, %1}, x;\n}\n"
      : "=f"(r.x), "=f"(r.y)
      : "f"(a), "f"(b), "f"(k), "f"(o.x), "f"(o.y));
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

// Row of query tile t: its token within the step, its head, and whether there is one.
struct Row {
  int token, head;
  bool active;
};
// Tokens of its request that a row sees: the first so many.
__device__ __forceinline__ int seen_by(const Params& p, const Part& x, int token) {
  return p.causal ? min(x.len, x.cached + token + 1) : x.len;
}
template <bool EXP>
__device__ __forceinline__ Row row_of(const Params& p, const Part& x, int t, int row) {
  if (EXP) return {x.tok0 + t * kRows + row, x.g, row < x.toks[t]};
  if (p.v.tiling.groups > 1) {
    const int h = x.g * kRows + row;
    return {x.tok0, min(h, p.heads - 1), h < p.heads};
  }
  const int token = row / p.heads;
  return {x.tok0 + token, row - token * p.heads, token < x.toks[0]};
}

// ---- joining the parts of tiles

// Parts of tiles that lie in the shares of several workers, and the rows past the
// step's last one.  A tile in n parts has n - 1 borders inside, whose blocks (one for
// every eight of its rows) share the rows: one warp a row or several, each for some of its
// values; lanes beyond those take every so many of the parts.  A row in 148 parts is
// many warps' (16 rows of 512 values: 35 us with eight of them at most, 13 with 64).  What is here runs once
// in a launch, on instructions that are in no cache, so there are few of them: with
// the tiles looked up here rather than in the plan, and a batch of parts unrolled, it
// took 22 us where this takes 5 (64 requests of 32 to 16,384 tokens, one row each).
// ROWS of a tile, V values of a block's results, SPLITS blocks that share a tile's.
template <typename T, int V, int SPLITS, int ROWS, bool EXP>
__global__ void __launch_bounds__(256) join_kernel(const Params p) {
  constexpr int kWide = V * SPLITS, kSlot = slot_floats(ROWS, V);
  constexpr int kLanes = V / 4;  // float4 of a row
  constexpr int kMine = (kLanes + 31) / 32;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int b = blockIdx.x / SPLITS + 1, split = blockIdx.x % SPLITS;
  // the lists are the plan's, which were there before attention began
  Join j = p.l.join[b < p.v.tiling.workers ? b : 0];
  const int workers = p.l.header->workers, used = p.v.starts[p.v.requests];
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if (used < p.tokens) {
    const int64_t id = ((int64_t)blockIdx.y * gridDim.x + blockIdx.x) * 256 + threadIdx.x;
    for (int64_t i = (int64_t)used * p.heads * (kWide / 8) + id;
         i < p.tokens * p.heads * (kWide / 8); i += (int64_t)gridDim.x * gridDim.y * 256) {
      reinterpret_cast<uint4*>(p.out)[i] = make_uint4(0, 0, 0, 0);
      if (p.lse && i % (kWide / 8) == 0) p.lse[i / (kWide / 8)] = -INFINITY;
    }
  }
  if (b >= workers || j.rows == 0) return;
  // warps of a row: 1, 2, 4 or 8, as many as there are, and beyond that as long as each lane
  // has four parts or more to add up
  const int warps = (j.parts - 1) * gridDim.y * 8;
  int shift = 0;
  while ((j.rows << (shift + 1)) <= warps &&
         (shift < 3 || (j.parts * (kLanes >> (shift + 1)) >= 128 && (kLanes >> (shift + 1)) >= 2)))
    ++shift;
  const int width = kLanes >> shift;  // float4 of a warp's
  const int wide = width < 32 ? width : 32;
  const int id = (j.border * gridDim.y + blockIdx.y) * 8 + warp;
  const int of_row = id & ((1 << shift) - 1);
  const int column = of_row * width + (lane & (wide - 1));
  const float* const part = p.l.part + split * kSlot;
#pragma unroll 1
  for (int line = id >> shift; line < j.rows; line += warps >> shift) {
    float m = -INFINITY, l = 0.0f, lr = 0.0f;
    bool sees = false;
    float4 o[kMine] = {};
#pragma unroll 2
    for (int k = lane / wide; k < j.parts; k += 32 / wide) {
      const float* slot =
          part + (int64_t)(k == 0 ? j.slot : 2 * (j.worker + k)) * (SPLITS * kSlot);
      const float4 s = *reinterpret_cast<const float4*>(slot + ROWS * V + 4 * line);
      float4 v[kMine];
#pragma unroll
      for (int i = 0; i < kMine; ++i)
        if (32 * i < width) v[i] = (reinterpret_cast<const float4*>(slot + line * V) + column)[32 * i];
      if (s.w == kNoResult) continue;
      sees |= s.w == kSees;
      const float next = fmaxf(m, s.x);
      const float a = m == next ? 1.0f : paged::ex2(m - next);
      const float f = s.x == next ? 1.0f : paged::ex2(s.x - next);
      m = next;
      l = fmaf(l, a, s.y * f);
      lr = fmaf(lr, a, s.z * f);
#pragma unroll
      for (int i = 0; i < kMine; ++i)
        if (32 * i < width) {
          o[i].x = fmaf(o[i].x, a, v[i].x * f);
          o[i].y = fmaf(o[i].y, a, v[i].y * f);
          o[i].z = fmaf(o[i].z, a, v[i].z * f);
          o[i].w = fmaf(o[i].w, a, v[i].w * f);
        }
    }
#pragma unroll 1
    for (int d = wide; d < 32; d <<= 1) {  // lanes with other parts; there is one float4 then
      const float other = __shfl_xor_sync(kFull, m, d), next = fmaxf(m, other);
      const float f = m == next ? 1.0f : paged::ex2(m - next);
      m = next;
      l *= f;
      lr *= f;
      l += __shfl_xor_sync(kFull, l, d);
      lr += __shfl_xor_sync(kFull, lr, d);
      o[0] = make_float4(o[0].x * f, o[0].y * f, o[0].z * f, o[0].w * f);
      o[0].x += __shfl_xor_sync(kFull, o[0].x, d);
      o[0].y += __shfl_xor_sync(kFull, o[0].y, d);
      o[0].z += __shfl_xor_sync(kFull, o[0].z, d);
      o[0].w += __shfl_xor_sync(kFull, o[0].w, d);
    }
    sees = __any_sync(kFull, sees);
    if (lane >= wide) continue;
    const int64_t row = j.row + (int64_t)line * (EXP ? p.heads : 1);
    const float inv = lr == 0.0f ? __int_as_float(0x7FC00000) : 1.0f / lr;
#pragma unroll
    for (int i = 0; i < kMine; ++i)
      if (32 * i < width)
        reinterpret_cast<uint2*>(p.out + row * kWide + split * V)[column + 32 * i] =
            sees ? make_uint2(Kind<T>::pack(o[i].x * inv, o[i].y * inv),
                              Kind<T>::pack(o[i].z * inv, o[i].w * inv))
                 : make_uint2(0, 0);
    if (lane == 0 && of_row == 0 && split == 0 && p.lse)
      p.lse[row] = l == 0.0f ? -INFINITY : (m - Kind<T>::kLift + log2f(l)) * 0.693147180559945309f;
  }
}

template <typename T, int V, int SPLITS, int ROWS, bool EXP>
int launch_join(const Params& p, cudaStream_t st) {
  cudaLaunchConfig_t cfg{};
  const Tiling& t = p.v.tiling;
  const int rows = EXP ? t.per : (int)std::min((int64_t)kRows, (int64_t)t.per * p.heads);
  cfg.gridDim = dim3((unsigned)(std::max(t.workers - 1, 1) * SPLITS), (unsigned)(rows + 31) / 32);
  cfg.blockDim = dim3(256);
  cfg.stream = st;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, join_kernel<T, V, SPLITS, ROWS, EXP>, p);
  if (e != cudaSuccess) {
    set_thread_error("latent join launch failed: %s", cudaGetErrorString(e));
    return cuda_status(e);
  }
  return 0;
}

}  // namespace
}  // namespace latent
}  // namespace grm_b200
