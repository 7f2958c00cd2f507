// paged_store.cu -- rows into and out of the 8-bit paged arena.
//
// append: for a page and kv head that the step writes,
//   s  = max(s_old if the page holds older tokens, max |x| / 127)
//   c  = rint(x / s)                 the step's rows
//   c' = rint(c * s_old / s)         the page's older codes, when s > s_old
// in fp32 with IEEE division, so the codes are the same whatever block computes
// them and writing a step twice changes nothing (s_old = s then).  One group of
// threads owns a (page, kv head, keys or values): it needs the maximum over all
// of its rows before the first code, and holds the rows in registers meanwhile,
// so that every input is read once.
//
// Both are bound by HBM: a value of append is 2 bytes in and 1 out, one of read
// 1 byte in and 2 or 4 out.  11,198 fp16 rows of 8 heads of 128, keys and values,
// are 69 MB in and out each way, 10.7 us at the rate of a copy: append takes 18 to
// 20 us (the rows in flight are limited by the registers that hold them, at 30 %
// occupancy; no unit is busy more than half of the time), read 13 to 16-bit values
// and 29 to fp32, of which it writes 93 MB.
#include <algorithm>

#include "paged.cuh"
#include "rotary.cuh"

namespace grm_b200 {
namespace paged {

namespace {

struct AppendParams {
  const Header* header;
  const int4* pages;
  int64_t ring_size;
  int page_shift, kv_heads;
  const uint16_t* x[2];  // keys, values
  int64_t row_stride[2], head_stride[2];
  int8_t* codes[2];
  float* scales[2];
};

// Sixteen 16-bit values.
struct Chunk {
  uint4 a, b;
};

__device__ __forceinline__ Chunk load_chunk(const uint16_t* p) {
  return {ld_nc16(p), ld_nc16(p + 8)};
}

// Largest magnitude of a chunk as 16-bit patterns in both halves of the result.
// Magnitude bits order as numbers do, infinity above them and NaN above that.
__device__ __forceinline__ unsigned magnitude(const Chunk& c) {
  const unsigned m = 0x7FFF7FFFu;
  unsigned r = __vmaxu2(c.a.x & m, c.a.y & m);
  r = __vmaxu2(r, __vmaxu2(c.a.z & m, c.a.w & m));
  r = __vmaxu2(r, __vmaxu2(c.b.x & m, c.b.y & m));
  return __vmaxu2(r, __vmaxu2(c.b.z & m, c.b.w & m));
}

template <typename T>
__device__ __forceinline__ float2 widen(unsigned v);
template <>
__device__ __forceinline__ float2 widen<__nv_bfloat16>(unsigned v) {
  return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xFFFF0000u));
}
template <>
__device__ __forceinline__ float2 widen<__half>(unsigned v) {
  return __half22float2(*reinterpret_cast<const __half2*>(&v));
}

__device__ __forceinline__ unsigned pack4(unsigned a, unsigned b, unsigned c, unsigned d) {
  return __byte_perm(__byte_perm(a, b, 0x0040), __byte_perm(c, d, 0x0040), 0x5410);
}

// Codes of a chunk: rint(x / s) with the quotient rounded to fp32.  One fused
// multiply-add with 1 / s and 1.5 * 2^23 gives the nearest whole number of a
// product that is off by less than 127 * 2^-23, and the number's byte; only where
// that product lies within 2^-15 of half-way between two numbers can the
// division's answer differ, and there the division is done (1 value in 16,000).
// A division for every value took 34 us where this takes 19 (11,198 rows of 8
// heads, fp16, keys and values).
template <typename T>
__device__ __forceinline__ uint4 quantise(const Chunk& c, float s, float inv) {
  const unsigned w[8] = {c.a.x, c.a.y, c.a.z, c.a.w, c.b.x, c.b.y, c.b.z, c.b.w};
  constexpr float kBase = 12582912.0f;
  unsigned out[4];
  float far = inv < INFINITY ? 0.0f : 1.0f;  // largest distance from a whole number
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 u = widen<T>(w[2 * i]), v = widen<T>(w[2 * i + 1]);
    const float x[4] = {u.x, u.y, v.x, v.y};
    unsigned t[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const float y = fmaf(x[k], inv, kBase);
      far = fmaxf(far, fabsf(fmaf(x[k], inv, kBase - y)));
      t[k] = __float_as_uint(y);
    }
    out[i] = pack4(t[0], t[1], t[2], t[3]);
  }
  if (far > 0.5f - 0x1p-15f) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 u = widen<T>(w[2 * i]), v = widen<T>(w[2 * i + 1]);
      out[i] = pack4(__float2int_rn(__fdiv_rn(u.x, s)), __float2int_rn(__fdiv_rn(u.y, s)),
                     __float2int_rn(__fdiv_rn(v.x, s)), __float2int_rn(__fdiv_rn(v.y, s)));
    }
  }
  return make_uint4(out[0], out[1], out[2], out[3]);
}

__device__ __forceinline__ unsigned rescale4(unsigned v, float from, float to) {
  int c[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int code = (int)(int8_t)(v >> (8 * i));
    c[i] = __float2int_rn(__fdiv_rn(__fmul_rn((float)code, from), to));
  }
  return pack4(c[0], c[1], c[2], c[3]);
}

// GROUP threads of a block own one (page, kv head, keys or values) and hold
// CACHE x 16 values each in registers; rows that a larger page has beyond them are
// read again (from L1 or L2).  Everything a group has to look up is one entry of
// the step's list, so that two loads, not four, stand before the rows.
template <typename T, int D, int GROUP, int CACHE>
__device__ __forceinline__ void append_one(const AppendParams& p, const int4 entry, int side, int h,
                                           int t, int group, unsigned* warp_max) {
  constexpr int kLanes = D / 16;            // threads of a row
  constexpr int kRowsPass = GROUP / kLanes;
  const int off = entry.z;   // older tokens of the page
  const int rows = entry.w;  // the step's
  const int64_t page = min(max((int64_t)entry.y, (int64_t)0), p.ring_size - 1);
  const int64_t row_stride = side ? p.row_stride[1] : p.row_stride[0];
  const uint16_t* x = (side ? p.x[1] : p.x[0]) + (int64_t)entry.x * row_stride +
                      (int64_t)h * (side ? p.head_stride[1] : p.head_stride[0]) +
                      (t % kLanes) * 16;
  int8_t* codes = (side ? p.codes[1] : p.codes[0]) +
                  (((page * p.kv_heads + h) << p.page_shift) * D);
  float* scale = (side ? p.scales[1] : p.scales[0]) + page * p.kv_heads + h;

  const int r0 = t / kLanes;
  Chunk c[CACHE];
  unsigned m = 0;
#pragma unroll
  for (int i = 0; i < CACHE; ++i) {
    const int r = r0 + i * kRowsPass;
    c[i] = r < rows ? load_chunk(x + r * row_stride)
                    : Chunk{make_uint4(0, 0, 0, 0), make_uint4(0, 0, 0, 0)};
  }
  const float old = off > 0 ? *scale : 0.0f;
#pragma unroll
  for (int i = 0; i < CACHE; ++i) m = __vmaxu2(m, magnitude(c[i]));
  for (int r = r0 + CACHE * kRowsPass; r < rows; r += kRowsPass)
    m = __vmaxu2(m, magnitude(load_chunk(x + r * row_stride)));
  m = __reduce_max_sync(kFull, max(m & 0xFFFFu, m >> 16));
  if (GROUP > 32) {  // the group's warps exchange their maxima
    if (t % 32 == 0) warp_max[threadIdx.x / 32] = m;
    asm volatile("bar.sync %0, %1;" ::"r"(1 + group), "n"(GROUP) : "memory");
#pragma unroll
    for (int w = 0; w < GROUP / 32; ++w) m = max(m, warp_max[group * (GROUP / 32) + w]);
  }
  float s = __fdiv_rn(widen<T>(m).x, 127.0f);
  s = old > s || isnan(old) ? old : s;
  if (!(s < INFINITY)) s = __int_as_float(0x7FC00000);
  const bool zero = !(s > 0.0f);  // nothing but zeros, or no number: codes 0
  const float inv = __fdiv_rn(1.0f, s);

  int8_t* out = codes + (t % kLanes) * 16;
#pragma unroll
  for (int i = 0; i < CACHE; ++i) {
    const int r = r0 + i * kRowsPass;
    if (r < rows)
      *reinterpret_cast<uint4*>(out + (off + r) * D) =
          zero ? make_uint4(0, 0, 0, 0) : quantise<T>(c[i], s, inv);
  }
#pragma unroll 1
  for (int r = r0 + CACHE * kRowsPass; r < rows; r += kRowsPass)
    *reinterpret_cast<uint4*>(out + (off + r) * D) =
        zero ? make_uint4(0, 0, 0, 0)
             : quantise<T>(load_chunk(x + r * row_stride), s, inv);
  if (off > 0 && !(s == old)) {
#pragma unroll 1
    for (int r = r0; r < off; r += kRowsPass) {
      uint4* q = reinterpret_cast<uint4*>(out + r * D);
      uint4 v = make_uint4(0, 0, 0, 0);
      if (!zero) {
        v = *q;
        v = make_uint4(rescale4(v.x, old, s), rescale4(v.y, old, s), rescale4(v.z, old, s),
                       rescale4(v.w, old, s));
      }
      *q = v;
    }
  }
  if (GROUP == 32) __syncwarp();  // every lane has read the old scale (else: the barrier above)
  if (t == 0) *scale = s;
}

template <typename T, int D, int GROUP, int CACHE>
__global__ void __launch_bounds__(256) append_kernel(const AppendParams p) {
  __shared__ unsigned warp_max[8];
  const int64_t job = (int64_t)blockIdx.x * (256 / GROUP) + threadIdx.x / GROUP;
  const int heads2 = p.kv_heads * 2;
  const int64_t unit = job / heads2;
  if (unit >= p.header->pages) return;
  const int side = (int)(job % heads2) & 1, h = (int)(job % heads2) >> 1;
  append_one<T, D, GROUP, CACHE>(p, p.pages[unit], side, h, threadIdx.x % GROUP,
                                 threadIdx.x / GROUP, warp_max);
}

// ---- append with the keys rotated on the way
//
// As append_kernel, with the values held as fp32, 32 of them a thread.  A thread's 16
// values of a row are eight pairs whole: 8 values of the first half of the rotated
// part and the 8 that turn with them, or 16 in a row where pairs are side by side.
// A block is HEADS groups, for as many heads of one page, so that the angles of the
// rows that they hold (about 25 instructions a pair) are worked out once and read from
// shared memory; rows of a larger page beyond those work theirs out where they are
// used.  11,198 fp16 rows of 8 heads of 128, 64 values of each key's head rotated (69 MB
// in and out, 10.5 us at a copy's rate), take 26.7 us and without the rotation 18.1; a group of
// its own for each head took 44, four heads one after another 46.  At three blocks an SM, 80
// registers, 80 to 88 bytes a thread are spilled, but for groups of 256.  61 bf16 rows of single
// tokens take 4.2, with it or without: a launch and three dependent loads.

struct TurnedParams {
  AppendParams a;
  RotaryParams r;
  const int32_t* positions;
};

// The largest of three, NaN if one of them is.
__device__ __forceinline__ float max3_nan(float a, float b, float c) {
  float d;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

// Codes of 16 values in fp32, as quantise.
__device__ __forceinline__ void quantise_turned(const float (&x)[16], float s, float inv,
                                                unsigned (&out)[4]) {
  constexpr float kBase = 12582912.0f;
  float far = inv < INFINITY ? 0.0f : 1.0f;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    unsigned t[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const float y = fmaf(x[4 * i + k], inv, kBase);
      far = fmaxf(far, fabsf(fmaf(x[4 * i + k], inv, kBase - y)));
      t[k] = __float_as_uint(y);
    }
    out[i] = pack4(t[0], t[1], t[2], t[3]);
  }
  if (far > 0.5f - 0x1p-15f) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      int t[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) t[k] = __float2int_rn(__fdiv_rn(x[4 * i + k], s));
      out[i] = pack4(t[0], t[1], t[2], t[3]);
    }
  }
}

template <typename T, int D, int GROUP, int HEADS>
__global__ void __launch_bounds__(GROUP * HEADS, 3) append_turned_kernel(const TurnedParams tp) {
  const AppendParams& p = tp.a;
  constexpr int kLanes = D / 16;  // threads of a row
  constexpr int kRowsPass = GROUP / kLanes, kCache = 2, kHeld = kCache * kRowsPass;
  static_assert(GROUP * HEADS >= D / 2, "a thread a pair");
  __shared__ unsigned warp_max[GROUP * HEADS / 32];
  __shared__ float2 angle[kHeld * (D / 2)];  // [rows][pairs], each row's eights apart
  const int t = threadIdx.x % GROUP, group = threadIdx.x / GROUP;
  const int sets2 = (p.kv_heads + HEADS - 1) / HEADS * 2;
  const int64_t unit = blockIdx.x / sets2;
  if (unit >= p.header->pages) return;
  const int side = (int)(blockIdx.x % sets2) & 1;
  const int h = ((int)(blockIdx.x % sets2) >> 1) * HEADS + group;
  const bool there = h < p.kv_heads;
  const int4 entry = p.pages[unit];
  if (side) {
    if (there)
      append_one<T, D, GROUP, GROUP == 32 ? 2 : 4>(p, entry, side, h, t, group, warp_max);
    return;
  }
  const int off = entry.z, rows = there ? entry.w : 0;
  const int64_t page = min(max((int64_t)entry.y, (int64_t)0), p.ring_size - 1);
  const int64_t row_stride = p.row_stride[0];
  const uint16_t* const x = p.x[0] + (int64_t)entry.x * row_stride + h * p.head_stride[0];
  int8_t* const codes = p.codes[0] + (((page * p.kv_heads + h) << p.page_shift) * D);
  float* const scale = p.scales[0] + page * p.kv_heads + h;

  // where the thread's two runs of 8 values lie, and its first pair
  const int lane16 = (t % kLanes) * 16, within = lane16 - tp.r.offset;
  const bool halves = tp.r.layout == GRM_B200_ROTARY_HALF;
  const bool turns = within >= 0 && within < tp.r.dim;
  const int pair0 = within / 2;
  const int at0 = turns && halves ? tp.r.offset + pair0 : lane16;
  const int at1 = turns && halves ? at0 + tp.r.dim / 2 : lane16 + 8;
  const int r0 = t / kLanes;
  auto load = [&](int r) {
    const uint16_t* row = x + r * row_stride;
    return Chunk{ld_nc16(row + at0), ld_nc16(row + at1)};
  };
  Chunk raw[kCache];
#pragma unroll
  for (int i = 0; i < kCache; ++i)
    if (r0 + i * kRowsPass < rows) raw[i] = load(r0 + i * kRowsPass);
  const float old = there && off > 0 ? *scale : 0.0f;

  // Angle i of the pairs 8 n .. 8 n + 7 of row r is at (r * 8 + i) * eights + n: lanes
  // of a row, whose eights follow one another, read different banks.
  const int eights = tp.r.dim / 16;
  const int position0 = tp.positions[entry.x];
  const int pairs = tp.r.dim / 2, held = min(entry.w, kHeld);
  const int i = threadIdx.x % pairs, first = threadIdx.x / pairs;
  const int step = max(GROUP * HEADS / pairs, 1);  // rows of a pass
  const uint64_t turns_i = tp.r.turns[i];
  if (first < step)
    for (int r = first; r < held; r += step) {
      const Turn u = turn_of(position0 + r, turns_i);
      angle[(r * 8 + i % 8) * eights + i / 8] =
          make_float2(u.cos * tp.r.amplitude, u.sin * tp.r.amplitude);
    }
  __syncthreads();

  auto take = [&](const Chunk& c, const float2 (&a)[8], float (&v)[16]) {
    const unsigned w[8] = {c.a.x, c.a.y, c.a.z, c.a.w, c.b.x, c.b.y, c.b.z, c.b.w};
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float2 u = widen<T>(w[i]);
      v[2 * i] = u.x;
      v[2 * i + 1] = u.y;
    }
    if (turns) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float x1 = halves ? v[i] : v[2 * i], x2 = halves ? v[8 + i] : v[2 * i + 1];
        const float y1 = x1 * a[i].x - x2 * a[i].y, y2 = x2 * a[i].x + x1 * a[i].y;
        if (halves) {
          v[i] = y1;
          v[8 + i] = y2;
        } else {
          v[2 * i] = y1;
          v[2 * i + 1] = y2;
        }
      }
    }
  };
  auto again = [&](int r, float (&v)[16]) {  // a row that is not held
    float2 a[8];
    if (turns) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const Turn u = turn_of(position0 + r, tp.r.turns[pair0 + i]);
        a[i] = make_float2(u.cos * tp.r.amplitude, u.sin * tp.r.amplitude);
      }
    }
    take(load(r), a, v);
  };
  // largest magnitude as bits, which order as numbers do, NaN above infinity
  auto widest = [](const float (&v)[16]) {
    float m = 0.0f;
#pragma unroll
    for (int i = 0; i < 16; i += 2) m = max3_nan(m, fabsf(v[i]), fabsf(v[i + 1]));
    return __float_as_uint(m) & 0x7FFFFFFFu;
  };

  float c[kCache][16];
  unsigned m = 0;
#pragma unroll
  for (int i = 0; i < kCache; ++i) {
    const int r = r0 + i * kRowsPass;
    if (r < rows) {
      float2 a[8];
      if (turns)
#pragma unroll
        for (int k = 0; k < 8; ++k) a[k] = angle[(r * 8 + k) * eights + pair0 / 8];
      take(raw[i], a, c[i]);
      m = max(m, widest(c[i]));
    }
  }
#pragma unroll 1
  for (int r = r0 + kHeld; r < rows; r += kRowsPass) {
    float v[16];
    again(r, v);
    m = max(m, widest(v));
  }
  m = __reduce_max_sync(kFull, m);
  if (GROUP > 32) {  // the group's warps exchange their maxima
    if (t % 32 == 0) warp_max[threadIdx.x / 32] = m;
    asm volatile("bar.sync %0, %1;" ::"r"(1 + group), "n"(GROUP) : "memory");
#pragma unroll
    for (int w = 0; w < GROUP / 32; ++w) m = max(m, warp_max[group * (GROUP / 32) + w]);
  }
  float s = __fdiv_rn(__uint_as_float(m), 127.0f);
  s = old > s || isnan(old) ? old : s;
  if (!(s < INFINITY)) s = __int_as_float(0x7FC00000);
  const bool zero = !(s > 0.0f);  // nothing but zeros, or no number: codes 0
  const float inv = __fdiv_rn(1.0f, s);

  auto store = [&](int r, const float (&v)[16]) {
    unsigned w[4] = {0, 0, 0, 0};
    if (!zero) quantise_turned(v, s, inv, w);
    int8_t* to = codes + (off + r) * D;
    *reinterpret_cast<uint2*>(to + at0) = make_uint2(w[0], w[1]);
    *reinterpret_cast<uint2*>(to + at1) = make_uint2(w[2], w[3]);
  };
#pragma unroll
  for (int i = 0; i < kCache; ++i)
    if (r0 + i * kRowsPass < rows) store(r0 + i * kRowsPass, c[i]);
#pragma unroll 1
  for (int r = r0 + kHeld; r < rows; r += kRowsPass) {
    float v[16];
    again(r, v);
    store(r, v);
  }
  if (!there) return;
  if (off > 0 && !(s == old)) {
#pragma unroll 1
    for (int r = r0; r < off; r += kRowsPass) {
      uint4* q = reinterpret_cast<uint4*>(codes + r * D + lane16);
      uint4 v = make_uint4(0, 0, 0, 0);
      if (!zero) {
        v = *q;
        v = make_uint4(rescale4(v.x, old, s), rescale4(v.y, old, s), rescale4(v.z, old, s),
                       rescale4(v.w, old, s));
      }
      *q = v;
    }
  }
  if (GROUP == 32) __syncwarp();  // every lane has read the old scale (else: the barrier above)
  if (t == 0) *scale = s;
}

template <typename T, int D, int GROUP, int HEADS>
int launch_append_group(const TurnedParams& p, int64_t cap, cudaStream_t st) {
  const int64_t blocks = cap * ceil_div64(p.a.kv_heads, HEADS) * 2;
  append_turned_kernel<T, D, GROUP, HEADS><<<(unsigned)blocks, GROUP * HEADS, 0, st>>>(p);
  return launch_status("paged append");
}

template <typename T, int D>
int launch_append(const TurnedParams& p, int64_t cap, int64_t max_fresh, cudaStream_t st) {
  const int64_t values = std::min<int64_t>(max_fresh, (int64_t)1 << p.a.page_shift) * D;
  if (values <= 32 * 32) return launch_append_group<T, D, 32, 8>(p, cap, st);
  if (values <= 64 * 32) return launch_append_group<T, D, 64, 4>(p, cap, st);
  if (values <= 128 * 32) return launch_append_group<T, D, 128, 2>(p, cap, st);
  return launch_append_group<T, D, 256, 1>(p, cap, st);
}

template <typename T, int D, int GROUP, int CACHE>
int launch_append_group(const AppendParams& p, int64_t cap, cudaStream_t st) {
  const int64_t blocks = ceil_div64(cap * p.kv_heads * 2, 256 / GROUP);
  append_kernel<T, D, GROUP, CACHE><<<(unsigned)blocks, 256, 0, st>>>(p);
  return launch_status("paged append");
}

template <typename T, int D>
int launch_append(const AppendParams& p, int64_t cap, int64_t max_fresh, cudaStream_t st) {
  // Few rows a page (decoding): a warp with two passes.  Else 64 values a thread:
  // fewer leave a thread more to look up than to do, more leave too few warps to
  // load while others compute (11,198 rows of 8 x 128: 30 us with 16 values, 25
  // with 128).
  const int64_t values = std::min<int64_t>(max_fresh, (int64_t)1 << p.page_shift) * D;
  if (values <= 32 * 32) return launch_append_group<T, D, 32, 2>(p, cap, st);
  if (values <= 32 * 64) return launch_append_group<T, D, 32, 4>(p, cap, st);
  if (values <= 64 * 64) return launch_append_group<T, D, 64, 4>(p, cap, st);
  if (values <= 128 * 64) return launch_append_group<T, D, 128, 4>(p, cap, st);
  return launch_append_group<T, D, 256, 4>(p, cap, st);
}

template <typename T, typename P>
int launch_append_dim(int dim, const P& p, int64_t cap, int64_t max_fresh, cudaStream_t st) {
  if (dim == 64) return launch_append<T, 64>(p, cap, max_fresh, st);
  if (dim == 128) return launch_append<T, 128>(p, cap, max_fresh, st);
  return launch_append<T, 256>(p, cap, max_fresh, st);
}

// ---- read

struct ReadParams {
  const int64_t* slots;
  int64_t count, limit;  // limit: pages * page_tokens
  int page_shift, kv_heads;
  const int8_t* codes[2];
  const float* scales[2];
  void* out[2];
};

template <typename T>
struct Out;
template <>
struct Out<float> {
  static __device__ __forceinline__ void store(float* o, const float (&v)[16]) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      reinterpret_cast<float4*>(o)[i] = make_float4(v[4 * i], v[4 * i + 1], v[4 * i + 2],
                                                    v[4 * i + 3]);
  }
};
template <typename T>
__device__ __forceinline__ unsigned pack2(float a, float b);
template <>
__device__ __forceinline__ unsigned pack2<__half>(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const unsigned*>(&h);
}
template <>
__device__ __forceinline__ unsigned pack2<__nv_bfloat16>(float a, float b) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const unsigned*>(&h);
}
template <typename T>
struct Out {
  static __device__ __forceinline__ void store(T* o, const float (&v)[16]) {
#pragma unroll
    for (int i = 0; i < 2; ++i)
      reinterpret_cast<uint4*>(o)[i] =
          make_uint4(pack2<T>(v[8 * i], v[8 * i + 1]), pack2<T>(v[8 * i + 2], v[8 * i + 3]),
                     pack2<T>(v[8 * i + 4], v[8 * i + 5]), pack2<T>(v[8 * i + 6], v[8 * i + 7]));
  }
};

// One thread for 16 values; blockIdx.y: keys or values.
template <typename T, int D>
__global__ void __launch_bounds__(256) read_kernel(const ReadParams p) {
  constexpr int kLanes = D / 16;
  const int side = blockIdx.y;
  const int64_t per_row = (int64_t)p.kv_heads * kLanes;
  const int64_t x = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (x >= p.count * per_row) return;
  const int64_t i = x / per_row;
  const int hc = (int)(x - i * per_row);
  const int h = hc / kLanes, c = hc % kLanes;
  const int64_t slot = p.slots[i];
  float v[16] = {};
  if (slot >= 0 && slot < p.limit) {
    const int64_t at = (slot >> p.page_shift) * p.kv_heads + h;
    const float s = (side ? p.scales[1] : p.scales[0])[at];
    const int64_t in = slot & ((1 << p.page_shift) - 1);
    const uint4 q = *reinterpret_cast<const uint4*>(
        (side ? p.codes[1] : p.codes[0]) + ((at << p.page_shift) + in) * D + c * 16);
    const unsigned w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
    for (int j = 0; j < 16; ++j) v[j] = (float)(int)(int8_t)(w[j / 4] >> (8 * (j % 4))) * s;
  }
  Out<T>::store(static_cast<T*>(side ? p.out[1] : p.out[0]) + x * 16, v);
}

template <typename T>
int launch_read(int dim, const ReadParams& p, cudaStream_t st) {
  const dim3 grid((unsigned)ceil_div64(p.count * p.kv_heads * (dim / 16), 256), 2);
  if (dim == 64) read_kernel<T, 64><<<grid, 256, 0, st>>>(p);
  else if (dim == 128) read_kernel<T, 128><<<grid, 256, 0, st>>>(p);
  else read_kernel<T, 256><<<grid, 256, 0, st>>>(p);
  return launch_status("paged read");
}

}  // namespace

int check_rows(const char* what, const void* ptr, int dtype, int64_t row_stride,
               int64_t head_stride) {
  if (!ptr || (dtype != GRM_B200_F16 && dtype != GRM_B200_BF16)) {
    set_thread_error("%s: rows must be fp16 or bf16 in device memory", what);
    return GRM_B200_EINVAL;
  }
  if ((reinterpret_cast<uintptr_t>(ptr) & 15) || row_stride % 8 || head_stride % 8 ||
      row_stride < 0 || head_stride < 0) {
    set_thread_error("%s: rows must be 16-byte aligned with strides that are multiples of 8 "
                     "elements (row stride %lld, head stride %lld)",
                     what, (long long)row_stride, (long long)head_stride);
    return GRM_B200_EINVAL;
  }
  return 0;
}

}  // namespace paged
}  // namespace grm_b200

using namespace grm_b200;
using namespace grm_b200::paged;

namespace {

int append(const grm_b200_paged_plan* plan, const grm_b200_paged_arena* arena,
           const grm_b200_rotary* rotary, const void* k_device, const void* v_device, int dtype,
           int64_t k_row_stride, int64_t k_head_stride, int64_t v_row_stride,
           int64_t v_head_stride, void* stream) {
  int rc;
  if ((rc = check_plan(plan)) || (rc = check_arena(arena)) || (rc = check_match(plan, arena)) ||
      (rc = check_rows("paged append", k_device, dtype, k_row_stride, k_head_stride)) ||
      (rc = check_rows("paged append", v_device, dtype, v_row_stride, v_head_stride)))
    return rc;
  if (!plan->grow) {
    set_thread_error("paged append: the plan's rows do not join the arena (grow = 0)");
    return GRM_B200_EINVAL;
  }
  int sms = 0;
  if ((rc = current_sms(&sms))) return rc;
  Shape s;
  make_shape(*plan, sms, &s);
  const Lists l = lists_of(s, plan->scratch);
  if (s.page_cap * arena->kv_heads * 2 > INT32_MAX) {
    set_thread_error("paged append: %lld pages of %d heads in one step are too many",
                     (long long)s.page_cap, arena->kv_heads);
    return GRM_B200_EINVAL;
  }
  AppendParams p;
  p.header = l.header;
  p.pages = l.pages;
  p.ring_size = plan->pages;
  p.page_shift = shift_of(plan->page_tokens);
  p.kv_heads = plan->kv_heads;
  p.x[0] = static_cast<const uint16_t*>(k_device);
  p.x[1] = static_cast<const uint16_t*>(v_device);
  p.row_stride[0] = k_row_stride;
  p.row_stride[1] = v_row_stride;
  p.head_stride[0] = k_head_stride;
  p.head_stride[1] = v_head_stride;
  p.codes[0] = arena->k_codes;
  p.codes[1] = arena->v_codes;
  p.scales[0] = arena->k_scales;
  p.scales[1] = arena->v_scales;
  const int64_t fresh = std::min(plan->max_fresh, plan->tokens);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (rotary) {
    const TurnedParams tp{p, rotary_params(*rotary), plan->positions};
    return dtype == GRM_B200_F16
               ? launch_append_dim<__half>(plan->head_dim, tp, s.page_cap, fresh, st)
               : launch_append_dim<__nv_bfloat16>(plan->head_dim, tp, s.page_cap, fresh, st);
  }
  return dtype == GRM_B200_F16
             ? launch_append_dim<__half>(plan->head_dim, p, s.page_cap, fresh, st)
             : launch_append_dim<__nv_bfloat16>(plan->head_dim, p, s.page_cap, fresh, st);
}

}  // namespace

extern "C" {

int grm_b200_paged_append(const grm_b200_paged_plan* plan, const grm_b200_paged_arena* arena,
                          const void* k_device, const void* v_device, int dtype,
                          int64_t k_row_stride, int64_t k_head_stride, int64_t v_row_stride,
                          int64_t v_head_stride, void* stream) {
  return append(plan, arena, nullptr, k_device, v_device, dtype, k_row_stride, k_head_stride,
                v_row_stride, v_head_stride, stream);
}

int grm_b200_paged_append_rotary(const grm_b200_paged_plan* plan, const grm_b200_paged_arena* arena,
                                 const grm_b200_rotary* rotary, const void* k_device,
                                 const void* v_device, int dtype, int64_t k_row_stride,
                                 int64_t k_head_stride, int64_t v_row_stride,
                                 int64_t v_head_stride, void* stream) {
  const int rc = check_rotary("paged append", rotary);
  if (rc) return rc;
  if (plan && (rotary->layout == GRM_B200_ROTARY_PAIR_SWAP || rotary->dim % 16 ||
               rotary->offset % 16 || (int64_t)rotary->offset + rotary->dim > plan->head_dim)) {
    set_thread_error("paged append: rotates dims at multiples of 16 within head_dim %d, layout half "
                     "or interleaved; got offset %d, dim %d, layout %d", plan->head_dim,
                     rotary->offset, rotary->dim, rotary->layout);
    return GRM_B200_EINVAL;
  }
  return append(plan, arena, rotary, k_device, v_device, dtype, k_row_stride, k_head_stride,
                v_row_stride, v_head_stride, stream);
}

int grm_b200_paged_read(const grm_b200_paged_arena* arena, const int64_t* slots_device,
                        int64_t count, int out_dtype, void* out_k_device, void* out_v_device,
                        void* stream) {
  const int rc = check_arena(arena);
  if (rc) return rc;
  if (count == 0) return 0;
  if (!slots_device || count < 0 || !out_k_device || !out_v_device ||
      ((reinterpret_cast<uintptr_t>(out_k_device) | reinterpret_cast<uintptr_t>(out_v_device)) &
       15) ||
      count > (int64_t)INT32_MAX * 256 / (arena->kv_heads * (arena->head_dim / 16))) {
    set_thread_error("invalid paged read arguments (count %lld; outputs must be 16-byte aligned)",
                     (long long)count);
    return GRM_B200_EINVAL;
  }
  ReadParams p;
  p.slots = slots_device;
  p.count = count;
  p.limit = arena->pages * arena->page_tokens;
  p.page_shift = shift_of(arena->page_tokens);
  p.kv_heads = arena->kv_heads;
  p.codes[0] = arena->k_codes;
  p.codes[1] = arena->v_codes;
  p.scales[0] = arena->k_scales;
  p.scales[1] = arena->v_scales;
  p.out[0] = out_k_device;
  p.out[1] = out_v_device;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (out_dtype == GRM_B200_F32) return launch_read<float>(arena->head_dim, p, st);
  if (out_dtype == GRM_B200_F16) return launch_read<__half>(arena->head_dim, p, st);
  if (out_dtype == GRM_B200_BF16) return launch_read<__nv_bfloat16>(arena->head_dim, p, st);
  set_thread_error("paged read: unknown element type %d", out_dtype);
  return GRM_B200_EINVAL;
}

}  // extern "C"
