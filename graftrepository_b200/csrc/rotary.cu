// rotary.cu -- rotary positions of rows [tokens, heads, head_dim]: with a the
// amplitude and t the angle of (position, pair),
//   y1 = a (x1 cos t - x2 sin t),   y2 = a (x2 cos t + x1 sin t),
// and the inverse, which takes the same rotation off again (1 / a, -t).  fp32, one
// rounding.
//
// Bound by HBM where rows are many: each value is read and written once.  A warp takes
// a token, or some heads of one where tokens are few.  Its first values are on their
// way to registers, eight pairs a lane (two loads of 16 bytes), while it works out the
// token's angles, once for all heads (about 25 instructions a pair; by each thread
// anew they were half of the kernel's), into its own corner of shared memory, so that
// no warp waits for another.  One pair at a time where strides, sizes or pointers are
// not multiples of that.
//
// 8,449 bf16 rows of 32 heads of 128 (138 MB, 21.2 us at a copy's rate) take 25.0 us, 5.5
// TB/s; 33 with a block's angles shared behind a barrier, 41 with a thread's own.  (At three
// blocks an SM, 80 registers, the 16-bit kernels spill 12 to 48 bytes a thread.)  2,047 fp32
// rows of 8 heads of 128, half of each rotated (17 MB, 2.6 us), take 6.3 and 61 bf16 rows of
// 40 heads of 96 take 4.4: a launch, a token's angles and one trip to memory.
#include <algorithm>

#include "rotary.cuh"

namespace grm_b200 {

namespace {

// Heads that a lane holds at once: 128 bytes of values.
template <typename T>
constexpr int kHeldOf = sizeof(T) == 4 ? 2 : 4;
constexpr int kMostDim = 4096;
constexpr int kSharedAngles = 2048;  // of a block

struct RotateParams {
  RotaryParams r;
  const void* x;
  void* out;
  const int32_t* positions;
  int64_t x_row, x_head, out_row, out_head;
  int tokens, heads, head_dim, inverse, copy;  // copy: values beside the rotated ones, too
  int entries;  // places of V pairs, or of V values beside them, in a head
  int lanes;    // heads that a warp takes side by side
  int splits;   // warps that share a token's heads
  int warps;    // of a block
};

template <typename T, int V, bool IN, bool OUT>
__global__ void __launch_bounds__(256, 3) rotate_kernel(const RotateParams p) {
  using W = Values<T, V>;
  constexpr int kHeld = kHeldOf<T>;
  __shared__ float2 angles[kSharedAngles];
  const int pairs = p.r.dim >> 1, places = pairs / V, lane = threadIdx.x & 31;
  // pair V n + i of the warp's token at i * places + n
  float2* const angle = angles + (threadIdx.x >> 5) * pairs;
  const unsigned warp = blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5);
  const int t = warp / p.splits, split = warp - t * p.splits;
  if (t >= p.tokens) return;
  const int h0 = p.heads * split / p.splits, h1 = p.heads * (split + 1) / p.splits;
  const T* const x = static_cast<const T*>(p.x) + t * p.x_row;
  T* const out = static_cast<T*>(p.out) + t * p.out_row;
  const int first = lane / p.entries;  // of the heads side by side
  const int position = p.positions[t];
  bool turned = false;  // the angles are there
#pragma unroll 1
  for (int n = lane - first * p.entries; n - lane < p.entries; n += 32) {
    const bool mine = first < p.lanes && n < p.entries, turns = n < places;
    // where V pairs, or V values beside them, lie in a head
    int i0 = p.r.offset + (IN ? 2 * n : n) * V, i1 = IN ? i0 + V : i0 + pairs;
    int o0 = p.r.offset + (OUT ? 2 * n : n) * V, o1 = OUT ? o0 + V : o0 + pairs;
    if (!turns) {
      i0 = (n - places) * V;
      if (i0 >= p.r.offset) i0 += p.r.dim;
      i1 = o0 = o1 = i0;
    }
    const T* from = x + (h0 + first) * p.x_head;
    T* to = out + (h0 + first) * p.out_head;
#pragma unroll 1
    for (int h = h0 + first; h - first < h1; h += kHeld * p.lanes) {
      W a[kHeld], b[kHeld];
#pragma unroll
      for (int k = 0; k < kHeld; ++k)
        if (mine && h + k * p.lanes < h1) {
          a[k] = *reinterpret_cast<const W*>(from + k * p.lanes * p.x_head + i0);
          if (turns) b[k] = *reinterpret_cast<const W*>(from + k * p.lanes * p.x_head + i1);
        }
      from += kHeld * p.lanes * p.x_head;
      if (!turned) {
        turned = true;
        const float gain = p.inverse ? 1.0f / p.r.amplitude : p.r.amplitude;
        for (int i = lane; i < pairs && position >= 0; i += 32) {
          const Turn u = turn_of(position, p.r.turns[i]);
          angle[i % V * places + i / V] =
              make_float2(u.cos * gain, (p.inverse ? -u.sin : u.sin) * gain);
        }
        __syncwarp();
      }
      if (mine && turns && position >= 0) {
        float2 c[V];
#pragma unroll
        for (int i = 0; i < V; ++i) c[i] = angle[i * places + n];
#pragma unroll
        for (int k = 0; k < kHeld; ++k)
          if (h + k * p.lanes < h1) {
            W y0, y1;
            turn_values<T, V, IN, OUT>(c, a[k], b[k], &y0, &y1);
            *reinterpret_cast<W*>(to + k * p.lanes * p.out_head + o0) = y0;
            *reinterpret_cast<W*>(to + k * p.lanes * p.out_head + o1) = y1;
          }
      } else if (mine && p.copy) {
        // beside the rotated ones, or a row without a position: as they came
#pragma unroll
        for (int k = 0; k < kHeld; ++k)
          if (h + k * p.lanes < h1) {
            *reinterpret_cast<W*>(to + k * p.lanes * p.out_head + i0) = a[k];
            if (turns) *reinterpret_cast<W*>(to + k * p.lanes * p.out_head + i1) = b[k];
          }
      }
      to += kHeld * p.lanes * p.out_head;
    }
  }
}

template <typename T, bool IN, bool OUT>
void launch_layout(const RotateParams& p, bool wide, int64_t blocks, cudaStream_t st) {
  if (wide) rotate_kernel<T, 8, IN, OUT><<<(unsigned)blocks, 32 * p.warps, 0, st>>>(p);
  else rotate_kernel<T, 1, IN, OUT><<<(unsigned)blocks, 32 * p.warps, 0, st>>>(p);
}

template <typename T>
int launch(const RotateParams& p, bool wide, int64_t blocks, cudaStream_t st) {
  if (p.r.layout == GRM_B200_ROTARY_HALF) launch_layout<T, false, false>(p, wide, blocks, st);
  else if (p.r.layout == GRM_B200_ROTARY_INTERLEAVED)
    launch_layout<T, true, true>(p, wide, blocks, st);
  else if (p.inverse) launch_layout<T, false, true>(p, wide, blocks, st);
  else launch_layout<T, true, false>(p, wide, blocks, st);
  const cudaError_t e = cudaGetLastError();
  if (e == cudaSuccess) return 0;
  set_thread_error("rotate launch failed: %s", cudaGetErrorString(e));
  return cuda_status(e);
}

}  // namespace

int check_rotary(const char* what, const grm_b200_rotary* r) {
  if (!r || !r->turns || r->dim < 2 || r->dim % 2 || r->dim > kMostDim || r->offset < 0 ||
      r->layout < GRM_B200_ROTARY_HALF || r->layout > GRM_B200_ROTARY_PAIR_SWAP ||
      !(r->amplitude > 0.0f) || !(r->amplitude < INFINITY)) {
    set_thread_error("%s: a rotary needs its turns, an even dim of 2 to %d, an offset from 0 on, a "
                     "layout and a positive amplitude", what, kMostDim);
    return GRM_B200_EINVAL;
  }
  return 0;
}

}  // namespace grm_b200

using namespace grm_b200;

extern "C" int grm_b200_rotate(const grm_b200_rotary* rotary, const void* x_device, int dtype,
                               int64_t tokens, int64_t heads, int64_t head_dim,
                               int64_t x_row_stride, int64_t x_head_stride,
                               const int32_t* positions_device, int inverse, void* out_device,
                               int64_t out_row_stride, int64_t out_head_stride, void* stream) {
  const int rc = check_rotary("rotate", rotary);
  if (rc) return rc;
  if (tokens == 0) return 0;
  const int size = dtype == GRM_B200_F32 ? 4 : 2;
  if (!x_device || !out_device || !positions_device || tokens < 0 || tokens > INT32_MAX ||
      heads < 1 || heads > 65536 || head_dim > 65536 || heads * head_dim > (1 << 24) ||
      (int64_t)rotary->offset + rotary->dim > head_dim || x_row_stride < 0 || x_head_stride < 0 ||
      out_row_stride < 0 || out_head_stride < 0 ||
      (dtype != GRM_B200_F32 && dtype != GRM_B200_F16 && dtype != GRM_B200_BF16) ||
      ((reinterpret_cast<uintptr_t>(x_device) | reinterpret_cast<uintptr_t>(out_device)) &
       (size - 1))) {
    set_thread_error("rotate: rows [%lld, %lld, %lld] of fp32, fp16 or bf16 with dims %d to %d "
                     "rotated, in device memory", (long long)tokens, (long long)heads,
                     (long long)head_dim, rotary->offset, rotary->offset + rotary->dim);
    return GRM_B200_EINVAL;
  }
  if (x_device == out_device &&
      (rotary->layout == GRM_B200_ROTARY_PAIR_SWAP || x_row_stride != out_row_stride ||
       x_head_stride != out_head_stride)) {
    set_thread_error("rotate: in place takes the same strides, and no pair swap");
    return GRM_B200_EINVAL;
  }
  int dev = 0;
  DeviceInfo info;
  const cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess || device_info(dev, &info)) {
    set_thread_error("rotate: no current device");
    return cuda_status(e == cudaSuccess ? cudaErrorInvalidDevice : e);
  }
  RotateParams p;
  p.r = rotary_params(*rotary);
  p.x = x_device;
  p.out = out_device;
  p.positions = positions_device;
  p.tokens = (int)tokens;
  p.x_row = x_row_stride;
  p.x_head = x_head_stride;
  p.out_row = out_row_stride;
  p.out_head = out_head_stride;
  p.heads = (int)heads;
  p.head_dim = (int)head_dim;
  p.inverse = inverse ? 1 : 0;
  p.copy = x_device != out_device;
  // eight pairs at a time: 8 values are 16 bytes (32 of fp32), wherever they start
  const int64_t words = (int64_t)p.r.offset | head_dim | x_row_stride | x_head_stride |
                        out_row_stride | out_head_stride;
  const bool wide = words % 8 == 0 && p.r.dim % 16 == 0 &&
                    ((reinterpret_cast<uintptr_t>(x_device) |
                      reinterpret_cast<uintptr_t>(out_device)) & 15) == 0;
  const int v = wide ? 8 : 1;
  p.entries = p.r.dim / 2 / v + (p.copy ? (p.head_dim - p.r.dim) / v : 0);
  p.lanes = std::max(32 / p.entries, 1);
  // A token's heads by several warps where that is what it takes to give every SM twelve
  // (2,047 rows of 32 x 128, 40 x 96 and fp32 8 x 128: 5.8, 9.5 and 5.4 us; with sixteen, a
  // wave and a half, 6.7, 10.6 and 6.5; with eight 400 to 1,600 rows take up to a fifth more).
  p.splits = (int)std::max<int64_t>(
      1, std::min<int64_t>(ceil_div64(heads, p.lanes), ceil_div64(12 * info.sms, tokens)));
  const int64_t warps = tokens * p.splits;
  p.warps = std::min(8, kSharedAngles / (p.r.dim / 2));
  const int64_t blocks = ceil_div64(warps, p.warps);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return dtype == GRM_B200_F32   ? launch<float>(p, wide, blocks, st)
         : dtype == GRM_B200_F16 ? launch<__half>(p, wide, blocks, st)
                                 : launch<__nv_bfloat16>(p, wide, blocks, st);
}
