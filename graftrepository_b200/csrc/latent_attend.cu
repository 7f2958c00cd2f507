// latent_attend.cu -- attention over pages of latent rows, in its simplest form: a
// block for each query row and head walks the tokens that the row sees, 128 at a
// time, with the running maximum and sum of the softmax.
#include "latent.cuh"

namespace grm_b200 {
namespace latent {

namespace {

constexpr int kThreads = 128;

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

// Request of packed row x: the last whose first row is not past it.
__device__ __forceinline__ int64_t request_of(const Params& p, int64_t x) {
  int64_t lo = 0, hi = p.requests;
  while (hi - lo > 1) {
    const int64_t mid = (lo + hi) >> 1;
    if (p.starts[mid] <= x) lo = mid;
    else hi = mid;
  }
  return lo;
}

template <typename T, bool EXPANDED>
__global__ void __launch_bounds__(kThreads) attend_kernel(const Params p) {
  __shared__ float q[512 + 64], weight[kThreads], red[4];
  const int64_t x = blockIdx.x / p.heads;
  const int h = blockIdx.x % p.heads, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int wide = EXPANDED ? p.value : p.latent, main = EXPANDED ? p.nope : p.latent;
  const int64_t orow = x * p.heads + h;
  int n = 0;
  int64_t r = 0;
  if (x < p.starts[p.requests]) {
    r = request_of(p, x);
    n = p.lens[r];
    if (p.causal) n = n - (p.starts[r + 1] - p.starts[r]) + (int)(x - p.starts[r]) + 1;
  }
  for (int i = tid; i < main; i += kThreads)
    q[i] = value_of<T>(p.q[x * p.q_row + h * p.q_head + i]);
  for (int i = tid; i < p.rope; i += kThreads)
    q[main + i] = value_of<T>(p.qr[x * p.qr_row + h * p.qr_head + i]);
  __syncthreads();
  const bool lost = EXPANDED && p.w.header->overflow;
  const int64_t base = EXPANDED && !lost ? p.w.base[r] : 0;
  if (lost && n > 0) n = 1;
  float m = -INFINITY, l = 0.0f, acc[4] = {};
  for (int t0 = 0; t0 < n; t0 += kThreads) {
    const int t = t0 + tid;
    float s = -INFINITY;
    if (t < n && !lost) {
      const uint16_t* row = row_of(p, r, t);
      const uint16_t* k = EXPANDED ? p.w.keys + ((int64_t)h * p.expand_tokens + base + t) * main
                                   : row;
      float y = 0.0f;
      for (int i = 0; i < main; ++i) y = fmaf(q[i], value_of<T>(k[i]), y);
      for (int i = 0; i < p.rope; ++i) y = fmaf(q[main + i], value_of<T>(row[p.latent + i]), y);
      s = y * p.scale_log2;
    }
    if (lost) s = __int_as_float(0x7FC00000);
    float top = s;
    for (int o = 16; o; o >>= 1) {
      const float u = __shfl_xor_sync(kFull, top, o);
      top = u > top || u != u ? u : top;
    }
    if (lane == 0) red[warp] = top;
    __syncthreads();
    for (int w = 0; w < 4; ++w) top = red[w] > top || red[w] != red[w] ? red[w] : top;
    const float next = top > m || top != top ? top : m;
    const float ref = next == -INFINITY ? 0.0f : next;
    const float a = paged::ex2(m - ref), e = paged::ex2(s - ref);
    weight[tid] = e;
    m = next;
    float sum = e;
    for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(kFull, sum, o);
    __syncthreads();
    if (lane == 0) red[warp] = sum;
    __syncthreads();
    l = l * a + ((red[0] + red[1]) + (red[2] + red[3]));
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int d = tid + j * kThreads;
      if (d < wide) {
        float y = acc[j] * a;
        for (int i = 0; i < min(kThreads, n - t0) && !lost; ++i) {
          const uint16_t* v =
              EXPANDED ? p.w.values + ((int64_t)h * p.expand_tokens + base + t0 + i) * wide
                       : row_of(p, r, t0 + i);
          y = fmaf(weight[i], value_of<T>(v[d]), y);
        }
        acc[j] = y;
      }
    }
    __syncthreads();
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int d = tid + j * kThreads;
    if (d < wide) p.out[orow * wide + d] = bits_of<T>(l == 0.0f ? 0.0f : acc[j] / l);
  }
  if (tid == 0 && p.lse)
    p.lse[orow] = l == 0.0f ? -INFINITY : (m + log2f(l)) * 0.693147180559945309f;
}

// 64 tokens of a request and one head's keys or values: a thread an output.
template <typename T>
__global__ void __launch_bounds__(256) expand_kernel(const Params p) {
  if (p.w.header->overflow) return;
  const int64_t t0 = (int64_t)blockIdx.x * kExpandAlign;
  if (t0 >= p.w.base[p.requests]) return;
  int64_t lo = 0, hi = p.requests;
  while (hi - lo > 1) {
    const int64_t mid = (lo + hi) >> 1;
    if (p.w.base[mid] <= t0) lo = mid;
    else hi = mid;
  }
  const int h = blockIdx.y, n = p.nope + p.value;
  for (int x = threadIdx.x; x < kExpandAlign * n; x += 256) {
    const int j = x % n;
    const int t = (int)(t0 - p.w.base[lo]) + x / n;
    float y = 0.0f;
    if (t < p.lens[lo]) {
      const uint16_t* row = row_of(p, lo, t);
      const uint16_t* w = p.weights + h * p.w_head + j * p.w_row;
      for (int i = 0; i < p.latent; ++i) y = fmaf(value_of<T>(row[i]), value_of<T>(w[i]), y);
    }
    const int64_t at = (int64_t)h * p.expand_tokens + t0 + x / n;
    if (j < p.nope) p.w.keys[at * p.nope + j] = bits_of<T>(y);
    else p.w.values[at * p.value + j - p.nope] = bits_of<T>(y);
  }
}

template <typename T>
int absorbed(const Params& p, cudaStream_t st) {
  attend_kernel<T, false><<<(unsigned)(p.tokens * p.heads), kThreads, 0, st>>>(p);
  return paged::launch_status("latent attend");
}

template <typename T>
int expanded(const Params& p, cudaStream_t st) {
  const dim3 grid((unsigned)ceil_div64(p.expand_tokens, kExpandAlign), p.heads);
  expand_kernel<T><<<grid, 256, 0, st>>>(p);
  const int rc = paged::launch_status("latent expand");
  if (rc) return rc;
  attend_kernel<T, true><<<(unsigned)(p.tokens * p.heads), kThreads, 0, st>>>(p);
  return paged::launch_status("latent attend");
}

}  // namespace

int launch_absorbed(int dtype, const Params& p, cudaStream_t st) {
  return dtype == GRM_B200_F16 ? absorbed<__half>(p, st) : absorbed<__nv_bfloat16>(p, st);
}

int launch_expanded(int dtype, const Params& p, cudaStream_t st) {
  return dtype == GRM_B200_F16 ? expanded<__half>(p, st) : expanded<__nv_bfloat16>(p, st);
}

}  // namespace latent
}  // namespace grm_b200
