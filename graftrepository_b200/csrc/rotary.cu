// rotary.cu -- rotary positions of rows [tokens, heads, head_dim]: with a the
// amplitude and t the angle of (position, pair),
//   y1 = a (x1 cos t - x2 sin t),   y2 = a (x2 cos t + x1 sin t),
// and the inverse, which takes the same rotation off again (1 / a, -t).  fp32, one
// rounding.
//
// Bound by HBM where rows are many: each value is read and written once.  A block
// takes a few tokens: their angles go to shared memory once, whatever the number of
// heads, then every thread takes eight pairs at a time (two loads and two stores of
// 16 bytes), or one pair where strides, sizes or pointers are not multiples of that.
#include <algorithm>

#include "rotary.cuh"

namespace grm_b200 {

namespace {

constexpr int kThreads = 256;
constexpr int kAngles = 2048;  // pairs of a block's tokens: 16 KB of cos and sin
constexpr int kMostDim = 2 * kAngles;

struct RotateParams {
  RotaryParams r;
  const void* x;
  void* out;
  const int32_t* positions;
  int64_t tokens, x_row, x_head, out_row, out_head;
  int heads, head_dim, inverse, copy;  // copy: values beside the rotated ones, too
  int per_block;                       // tokens
  int splits;                          // blocks that share a token's heads
};

template <typename T, int V, bool IN, bool OUT>
__global__ void __launch_bounds__(kThreads) rotate_kernel(const RotateParams p) {
  __shared__ float2 angle[kAngles];
  const int pairs = p.r.dim >> 1;
  const int64_t t0 = (int64_t)(blockIdx.x / p.splits) * p.per_block;
  const int split = blockIdx.x % p.splits;
  const int tokens = (int)(p.tokens - t0 < p.per_block ? p.tokens - t0 : p.per_block);
  const float gain = p.inverse ? 1.0f / p.r.amplitude : p.r.amplitude;
  for (int x = threadIdx.x; x < tokens * pairs; x += kThreads) {
    const int position = p.positions[t0 + x / pairs];
    // a row without a position stays as it is
    Turn t{1.0f, 0.0f};
    float g = 1.0f;
    if (position >= 0) {
      t = turn_of(position, p.r.turns[x % pairs]);
      g = gain;
    }
    angle[x] = make_float2(t.cos * g, (p.inverse ? -t.sin : t.sin) * g);
  }
  __syncthreads();
  const int h0 = (int)((int64_t)p.heads * split / p.splits);
  const int h1 = (int)((int64_t)p.heads * (split + 1) / p.splits);
  const T* const x = static_cast<const T*>(p.x);
  T* const out = static_cast<T*>(p.out);
  const int turned = pairs / V;  // entries of a head: its pairs, then what is copied
  const int beside = p.copy ? (p.head_dim - p.r.dim) / V : 0;
  const int entries = turned + beside, per_token = (h1 - h0) * entries;
  for (int i = threadIdx.x; i < tokens * per_token; i += kThreads) {
    const int t = i / per_token, y = i - t * per_token, h = h0 + y / entries, e = y % entries;
    const T* from = x + (t0 + t) * p.x_row + h * p.x_head;
    T* to = out + (t0 + t) * p.out_row + h * p.out_head;
    if (e >= turned) {
      int at = (e - turned) * V;
      if (at >= p.r.offset) at += p.r.dim;
      *reinterpret_cast<Values<T, V>*>(to + at) = *reinterpret_cast<const Values<T, V>*>(from + at);
    } else if (p.positions[t0 + t] >= 0 || p.copy) {
      if (p.positions[t0 + t] < 0) {  // out of place: as they came
        for (int k = 0; k < 2 * V; ++k)
          to[p.r.offset + 2 * e * V + k] = from[p.r.offset + 2 * e * V + k];
        continue;
      }
      float2 a[V];
#pragma unroll
      for (int k = 0; k < V; ++k) a[k] = angle[t * pairs + e * V + k];
      turn_pairs<T, V, IN, OUT>(pairs, a, e * V, from + p.r.offset, to + p.r.offset);
    }
  }
}

template <typename T, bool IN, bool OUT>
void launch_layout(const RotateParams& p, bool wide, int64_t blocks, cudaStream_t st) {
  if (wide) rotate_kernel<T, 8, IN, OUT><<<(unsigned)blocks, kThreads, 0, st>>>(p);
  else rotate_kernel<T, 1, IN, OUT><<<(unsigned)blocks, kThreads, 0, st>>>(p);
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
  p.tokens = tokens;
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
  // about 4,096 values a block, fewer where that leaves SMs without one
  const int64_t values = heads * head_dim;
  const int64_t most = std::max<int64_t>(1, std::min<int64_t>(4096 / std::max<int64_t>(values, 1),
                                                              kAngles / (p.r.dim / 2)));
  p.per_block = (int)std::max<int64_t>(1, std::min(most, tokens / (2 * info.sms)));
  const int64_t groups = ceil_div64(tokens, p.per_block);
  p.splits = groups >= 2 * info.sms
                 ? 1
                 : (int)std::min<int64_t>(heads, ceil_div64(2 * info.sms, groups));
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const int64_t blocks = groups * p.splits;
  return dtype == GRM_B200_F32   ? launch<float>(p, wide, blocks, st)
         : dtype == GRM_B200_F16 ? launch<__half>(p, wide, blocks, st)
                                 : launch<__nv_bfloat16>(p, wide, blocks, st);
}
