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

constexpr int kJoinBlocks = 8;  // for every border between two shares

// Parts of tiles that lie in the shares of several workers, and the rows past the
// step's last one.  A tile in n parts has n - 1 borders inside, whose blocks share its
// rows: 1 to 8 warps a row, each for some of its values; lanes beyond those take every
// so many of the parts.  Takes no shared memory, so that blocks get their place, and
// find theirs in the lists, while attention still runs.
// ROWS of a tile, V values of a block's results, SPLITS blocks that share a tile's.
template <typename T, int V, int SPLITS, int ROWS, bool EXP>
__global__ void __launch_bounds__(256) join_kernel(const Params p) {
  constexpr int kWide = V * SPLITS, kSlot = slot_floats(ROWS, V);
  constexpr int kLanes = V / 4;  // float4 of a row
  constexpr int kMine = (kLanes + 31) / 32;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int b = blockIdx.x / SPLITS + 1, split = blockIdx.x % SPLITS;
  // the lists are the plan's, which was there before attention began
  const Start start = p.l.start[min(b, p.v.tiling.workers - 1)];
  const Header hd = *p.l.header;
  const int64_t used = p.v.starts[p.v.requests];
  bool joins = b < hd.workers;
  Walk walk;
  int w0 = 0, parts = 0;
  if (joins) {
    walk.start(p.v, start);
    joins = walk.first != worker_first(b, hd);  // a border inside the tile
    w0 = worker_of(walk.first, hd);             // worker of the tile's first part
    parts = worker_of(walk.last - 1, hd) - w0 + 1;
  }
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int64_t id = ((int64_t)blockIdx.y * gridDim.x + blockIdx.x) * 256 + threadIdx.x;
  for (int64_t i = used * p.heads * (kWide / 8) + id; i < p.tokens * p.heads * (kWide / 8);
       i += (int64_t)gridDim.x * gridDim.y * 256) {
    reinterpret_cast<uint4*>(p.out)[i] = make_uint4(0, 0, 0, 0);
    if (p.lse && i % (kWide / 8) == 0) p.lse[i / (kWide / 8)] = -INFINITY;
  }
  if (!joins) return;
  Part x;
  x.r = walk.r;
  x.g = walk.g;
  x.tok0 = walk.j * p.v.tiling.per;
  const int toks = min(p.v.tiling.per, walk.q.n - x.tok0);
  x.toks[0] = EXP ? min(toks, kRows) : toks;
  x.toks[1] = EXP ? toks - x.toks[0] : 0;
  const int rows = EXP ? toks
                       : min(kRows, toks * (p.v.tiling.groups > 1 ? kRows : p.heads));
  // rows of a block: 8, 4, 2 or 1, whichever is enough, and more where 8 are not
  const int blocks = (parts - 1) * kJoinBlocks;
  int each = 1;
  while (each < 8 && each * blocks < rows) each *= 2;
  const int warps = 8 / each;                // of a row
  const int width = kLanes / warps;          // float4 of a warp, wide * mine
  const int wide = width < 32 ? width : 32, mine = width / wide;
  const int column = warp % warps * width + lane % wide, group = lane / wide;
  const int slot0 = 2 * w0 + (walk.first == worker_first(w0, hd) ? 0 : 1);
  auto slot = [&](int k) {
    const int at = k == 0 ? slot0 : 2 * (w0 + k);
    return p.l.part + ((int64_t)at * SPLITS + split) * kSlot;
  };
  const int block = (b - 1 - w0) * kJoinBlocks + blockIdx.y;
#pragma unroll 1
  for (int row0 = block * each; row0 < rows; row0 += blocks * each) {
    const int line = row0 + warp / warps;  // of the tile's rows
    const Row a = row_of<EXP>(p, x, line / kRows, line % kRows);
    if (line >= rows || !a.active) continue;
    auto state = [&](int k) {
      return *reinterpret_cast<const float4*>(slot(k) + ROWS * V + 4 * line);
    };
    // the largest reference exponent of the parts that see something, and the sums,
    // lanes side by side
    float m = -INFINITY, l = 0.0f, lr = 0.0f;
    for (int k = lane; k < parts; k += 32) {
      const float4 s = state(k);
      if (s.y != 0.0f) m = fmaxf(m, s.x);
    }
#pragma unroll
    for (int i = 16; i; i >>= 1) m = fmaxf(m, __shfl_xor_sync(kFull, m, i));
    for (int k = lane; k < parts; k += 32) {
      const float4 s = state(k);
      const float f = s.x == m ? 1.0f : paged::ex2(s.x - m);
      if (s.y != 0.0f) {
        l = fmaf(s.y, f, l);
        lr = fmaf(s.z, f, lr);
      }
    }
#pragma unroll
    for (int i = 16; i; i >>= 1) {
      l += __shfl_xor_sync(kFull, l, i);
      lr += __shfl_xor_sync(kFull, lr, i);
    }
    float4 o[kMine] = {};
    const int groups = 32 / wide;
#pragma unroll 4
    for (int k = group; k < parts; k += groups) {
      const float4 s = state(k);
      const float f = s.x == m ? 1.0f : paged::ex2(s.x - m);
      const float4* from = reinterpret_cast<const float4*>(slot(k) + line * V) + column;
#pragma unroll
      for (int i = 0; i < kMine; ++i)
        if (i < mine && s.y != 0.0f) {
          const float4 v = from[32 * i];
          o[i].x = fmaf(v.x, f, o[i].x);
          o[i].y = fmaf(v.y, f, o[i].y);
          o[i].z = fmaf(v.z, f, o[i].z);
          o[i].w = fmaf(v.w, f, o[i].w);
        }
    }
    for (int d = wide; d < 32; d <<= 1) {  // there is one float4 then
      o[0].x += __shfl_xor_sync(kFull, o[0].x, d);
      o[0].y += __shfl_xor_sync(kFull, o[0].y, d);
      o[0].z += __shfl_xor_sync(kFull, o[0].z, d);
      o[0].w += __shfl_xor_sync(kFull, o[0].w, d);
    }
    if (group > 0) continue;
    const int64_t orow = (int64_t)(walk.q.start + a.token) * p.heads + a.head;
    const float inv = 1.0f / lr;
#pragma unroll
    for (int i = 0; i < kMine; ++i)
      if (i < mine)
        reinterpret_cast<uint2*>(p.out + orow * kWide + split * V)[column + 32 * i] =
            lr == 0.0f ? make_uint2(0, 0)
                       : make_uint2(Kind<T>::pack(o[i].x * inv, o[i].y * inv),
                                    Kind<T>::pack(o[i].z * inv, o[i].w * inv));
    if (lane == 0 && warp % warps == 0 && p.lse && split == 0)
      p.lse[orow] =
          l == 0.0f ? -INFINITY : (m - Kind<T>::kLift + log2f(l)) * 0.693147180559945309f;
  }
}

template <typename T, int V, int SPLITS, int ROWS, bool EXP>
int launch_join(const Params& p, cudaStream_t st) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)(std::max(p.v.tiling.workers - 1, 1) * SPLITS),
                     kJoinBlocks);
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
