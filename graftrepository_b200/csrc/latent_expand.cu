// latent_expand.cu -- keys and values of each head from the rows of the cache,
//   k = W^k_h c (as a rounded number and what that left over), v = W^v_h c,
// for the tokens of every request that has rows in the step.
#include "latent.cuh"

namespace grm_b200 {
namespace latent {

namespace {

template <typename T>
__device__ __forceinline__ float value_of(uint16_t v);
template <>
__device__ __forceinline__ float value_of<__half>(uint16_t v) {
  return __half2float(__ushort_as_half(v));
}
template <>
__device__ __forceinline__ float value_of<__nv_bfloat16>(uint16_t v) {
  return __uint_as_float((unsigned)v << 16);
}
template <typename T>
__device__ __forceinline__ uint16_t bits_of(float v);
template <>
__device__ __forceinline__ uint16_t bits_of<__half>(float v) {
  return __half_as_ushort(__float2half_rn(v));
}
template <>
__device__ __forceinline__ uint16_t bits_of<__nv_bfloat16>(float v) {
  return __bfloat16_as_ushort(__float2bfloat16_rn(v));
}

__device__ __forceinline__ const uint16_t* row_of(const Params& p, int64_t r, int t) {
  const int last = (1 << p.page_shift) - 1;
  const int page = min(max(p.table[r * p.width + (t >> p.page_shift)], 0), (int)p.pages - 1);
  return p.cache + (((int64_t)page << p.page_shift) + (t & last)) * (p.latent + p.rope);
}

// 64 tokens of a request and one head's keys and values: a thread an output.
template <typename T>
__global__ void __launch_bounds__(256) expand_kernel(const Params p) {
  const int64_t t0 = (int64_t)blockIdx.x * kExpandAlign;
  if (t0 >= p.room[p.requests]) return;
  int64_t lo = 0, hi = p.requests;
  while (hi - lo > 1) {
    const int64_t mid = (lo + hi) >> 1;
    if (p.room[mid] <= t0) lo = mid;
    else hi = mid;
  }
  const int h = blockIdx.y, n = 2 * p.nope;
  for (int x = threadIdx.x; x < kExpandAlign * n; x += 256) {
    const int j = x % n;
    const int t = (int)(t0 - p.room[lo]) + x / n;
    float y = 0.0f;
    if (t < p.lens[lo]) {
      const uint16_t* row = row_of(p, lo, t);
      const uint16_t* w = p.weights + h * p.w_head + j * p.w_row;
      for (int i = 0; i < p.latent; ++i) y = fmaf(value_of<T>(row[i]), value_of<T>(w[i]), y);
    }
    const int64_t at = (int64_t)h * p.expand_tokens + t0 + x / n;
    if (j < p.nope) {
      const uint16_t k = bits_of<T>(y);
      p.keys[at * n + j] = k;
      p.keys[at * n + p.nope + j] = bits_of<T>(y - value_of<T>(k));
    } else {
      p.values[at * p.nope + j - p.nope] = bits_of<T>(y);
    }
  }
}

}  // namespace

int launch_expand(const Params& p, cudaStream_t st) {
  const dim3 grid((unsigned)ceil_div64(p.expand_tokens, kExpandAlign), p.heads);
  if (p.dtype == GRM_B200_F16) expand_kernel<__half><<<grid, 256, 0, st>>>(p);
  else expand_kernel<__nv_bfloat16><<<grid, 256, 0, st>>>(p);
  return paged::launch_status("latent expand");
}

}  // namespace latent
}  // namespace grm_b200
