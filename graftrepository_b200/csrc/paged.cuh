// paged.cuh -- what the kernels of the 8-bit paged arena share: the layout of a
// plan's scratch (work lists and partial results) and the checks of arguments.
#pragma once

#include <atomic>

#include "common.cuh"

namespace grm_b200 {
namespace paged {

// The split kernel of attention walks a request's tokens in tiles and gives
// every worker (a resident block) the same number of units: a request, kv head
// and block of query rows ("segment") costs its tiles and one unit more for
// its start and end.
__host__ __device__ constexpr int split_tile(int dim) { return dim == 256 ? 64 : 128; }
// Its blocks on an SM, for segments of `rows` query rows.
__host__ __device__ constexpr int split_blocks(int dim, int rows) {
  return dim == 64 || (dim == 128 && rows == 8) ? 3 : 2;
}
// fp32 of one partial result: rows x dim, then (reference exponent, sum) a row.
__host__ __device__ constexpr int split_slot(int dim, int rows) { return rows * dim + 2 * rows; }

// Query rows and tokens of a step of a prompt tile, and fp32 of one part's result:
// [dim / 4][rows][4], then (reference exponent, sum) a row.
__host__ __device__ constexpr int prompt_rows_of(int dim) { return dim == 256 ? 128 : 256; }
__host__ __device__ constexpr int prompt_step_of(int dim) { return dim == 256 ? 64 : 128; }
__host__ __device__ constexpr int prompt_slot(int dim) { return prompt_rows_of(dim) * (dim + 2); }

struct Header {           // written by the plan kernel
  int32_t units;          // units of the split kernel's work, all requests
  int32_t workers;        // workers that share them (<= Shape::workers)
  int32_t share, more;    // units of a worker, and how many workers have one more
  int32_t pages;          // entries of the append list
  int32_t qtiles;         // entries of the prompt kernel's list: parts of prompt tiles
  int32_t joins;          // qtiles, where tiles are in more than one part; 0 where none is
  int32_t rows;           // packed rows of the step
  int32_t take;           // pages that it takes
  int32_t committed;      // whether a commit has taken it up
};

// Sizes that follow from the plan's sizes alone, so that the plan kernel and
// the kernels that read its lists agree without the host seeing a length.
struct Shape {
  int group;            // query heads of a kv head
  int prompt_rows;      // requests with more (row, head) pairs a kv head can be prompts
  int block_rows;       // rows of a segment: 8 or 16
  int qtile_tokens;     // tokens of a prompt tile
  int tile;             // tokens of a tile of the split kernel
  int workers;          // resident blocks of the split kernel
  int64_t page_cap;     // most pages a step can touch
  int64_t qtile_cap;    // most entries of the prompt kernel's list (0: no request can be a prompt)
  // byte offsets in the scratch
  int64_t off_base, off_start, off_count, off_pages, off_qtiles, off_part;
  int64_t off_qpart, bytes;
};

int make_shape(const grm_b200_paged_plan& p, int sms, Shape* s);

struct Lists {
  Header* header;
  int32_t* base;      // [requests + 1] first unit of each request
  int32_t* start;     // [workers] request of a worker's first unit
  unsigned* count;    // [workers] arrivals at the segment that a worker starts; 0 between calls
  int4* pages;        // [page_cap] (first packed row, page, older tokens in it, new rows)
  // [qtile_cap] (request, first row of the tile within the request, part + 256 *
  // parts, first entry of the tile)
  int4* qtiles;
  float* part;        // [workers * 2][split_slot]
  float* qpart;       // [sms][prompt_slot]
};

inline Lists lists_of(const Shape& s, void* scratch) {
  char* b = static_cast<char*>(scratch);
  return {reinterpret_cast<Header*>(b),
          reinterpret_cast<int32_t*>(b + s.off_base),
          reinterpret_cast<int32_t*>(b + s.off_start),
          reinterpret_cast<unsigned*>(b + s.off_count),
          reinterpret_cast<int4*>(b + s.off_pages),
          reinterpret_cast<int4*>(b + s.off_qtiles),
          reinterpret_cast<float*>(b + s.off_part),
          reinterpret_cast<float*>(b + s.off_qpart)};
}

// First unit of worker w, and the worker that holds unit u.
__host__ __device__ inline int worker_first(int w, const Header& h) {
  return w * h.share + (w < h.more ? w : h.more);
}
__host__ __device__ inline int worker_of(int u, const Header& h) {
  const int big = h.more * (h.share + 1);  // units of the workers that have one more
  return u < big ? u / (h.share + 1) : h.more + (u - big) / h.share;
}

// ---- attention

constexpr float kLazy = 8.0f;  // how far a row's scores may pass its reference exponent
// Weights are held as fp16 times 2^7: at most 2^15, and what is lost at the small end
// (fp16 ends at 2^-24) lies below 2^-32 of the row's largest.  Held as they are it
// would be 2^-25, which the many small weights beside one that takes nearly all of
// the sum reach (16,384 equal tokens e^-16 below one token: their part 6 % off).
// Sums are of the weights themselves, results of the lifted ones.
constexpr float kLift = 7.0f;
constexpr float kUnlift = 0x1p-7f;
// The reference exponent for a largest score `top`: a multiple of 2^-14 (below 256).
// Less 7 it stays exact, where the rounding of any other one would be a factor on the
// row's whole sum (1e-6 in its logarithm), and the largest weight is a power of two
// but for 2^-15, so that fp16 does not round the one that counts most (a whole number
// is as exact, but one row over 250,007 tokens is then off by 2.7e-4 in fp16, not 2.3).
__device__ __forceinline__ float reference_of(float top) {
  return __fadd_rn(__fadd_rn(top, 768.0f), -768.0f);
}

// Probes of a bounded wait.  A wait that gives up leaves NaN in its rows and
// GRM_B200_PLAN_WAIT in the plan's status; copies and products in flight are waited
// for (with this limit, whatever AttendParams::probes is) before the block ends.
constexpr unsigned kProbes = 1u << 18;

struct AttendParams {
  Lists l;
  unsigned probes;  // kProbes, or less by GRM_B200_WAIT_LIMIT
  const int32_t* table;
  const int32_t* lens;
  const int32_t* starts;
  int64_t width, tokens, pages;
  int page_shift, kv_heads, group, causal, block_rows, qtile_tokens;
  unsigned group_inv;  // above 2^32 / group: x / group for small x, where group > 1
  const int8_t* k;
  const int8_t* v;
  const float* ks;
  const float* vs;
  const uint16_t* q;
  int64_t q_row, q_head;
  float scale_log2;
  uint16_t* out;
  float* lse;
  int32_t* status;
};

// Rows of the requests that the plan made prompts (paged_prompt.cu).
int launch_prompt(int dtype, int dim, const AttendParams& p, int64_t blocks, cudaStream_t st);

// A prompt tile from its entry in the list: 128-row query tiles of `per` tokens,
// the second one empty where the rows fit one.
struct PromptTile {
  int start, cached, len, tok0, per, toks[2];
  int steps;  // of the tokens that its rows see
  int parts;  // blocks that share them
};
template <int D>
__device__ __forceinline__ PromptTile prompt_tile(const AttendParams& p, int4 e) {
  PromptTile t;
  t.start = p.starts[e.x];
  const int n = p.starts[e.x + 1] - t.start;
  t.len = p.lens[e.x];
  t.cached = t.len - n;
  t.per = p.qtile_tokens / (prompt_rows_of(D) / 128);
  t.tok0 = e.y;
  t.toks[0] = min(t.per, n - t.tok0);
  t.toks[1] = prompt_rows_of(D) == 256 ? max(0, min(t.per, n - t.tok0 - t.per)) : 0;
  const int sees = p.causal ? min(t.len, t.cached + t.tok0 + t.toks[0] + t.toks[1]) : t.len;
  t.steps = (sees + prompt_step_of(D) - 1) / prompt_step_of(D);
  t.parts = max(1, min(e.z >> 8, t.steps));
  return t;
}

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Two codes, chosen by `sel` from the four of w (already + 128), as halves.
__device__ __forceinline__ uint32_t halves(uint32_t w, uint32_t sel) {
  const uint32_t v = __byte_perm(w, 0x64646464u, sel);
  const __half2 h = __hsub2(*reinterpret_cast<const __half2*>(&v),
                            __halves2half2(__ushort_as_half(0x6480), __ushort_as_half(0x6480)));
  return *reinterpret_cast<const uint32_t*>(&h);
}

__device__ __forceinline__ uint32_t pack_half2(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}

template <typename T>
__device__ __forceinline__ uint32_t pack_out(float a, float b);
template <>
__device__ __forceinline__ uint32_t pack_out<__half>(float a, float b) { return pack_half2(a, b); }
template <>
__device__ __forceinline__ uint32_t pack_out<__nv_bfloat16>(float a, float b) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// The power of two that brings a bf16 row, whose largest magnitude has the bits
// m, into [2^14, 2^15), and its inverse; rows of zeros or below 2^-100 keep out
// of the way of overflow.
__device__ __forceinline__ void row_scale(unsigned m, float* up, float* down) {
  const int e = max((int)(m >> 7), 27);  // biased exponent
  *up = m ? __uint_as_float((unsigned)(127 + 14 + 127 - e) << 23) : 1.0f;
  *down = m ? __uint_as_float((unsigned)(e - 14) << 23) : 1.0f;
}
// Base-2 logarithm of a value scale and what takes a lifted weight out of it,
// 2^-7 / u.  A page of zeros (scale 0)
// takes 2^-40, any scale being right for it: small enough to leave the other
// pages' weights alone, large enough for its own to stay above 2^-126 when the
// reference exponent is another page's.  Scales below 2^-100 count as 2^-100, so
// the inverse is a number even where the scale is none.
__device__ __forceinline__ void value_scale(float u, float* log2_u, float* inv_u) {
  const float w = u == 0.0f ? 0x1p-40f : fmaxf(u, 0x1p-100f);
  *log2_u = u != u ? u : __log2f(w);
  *inv_u = __fdividef(1.0f, w) * kUnlift;
}
// Two bf16 times `up` as halves.
__device__ __forceinline__ uint32_t scale_pair(uint32_t v, float up) {
  return pack_half2(__uint_as_float(v << 16) * up, __uint_as_float(v & 0xFFFF0000u) * up);
}

int check_plan(const grm_b200_paged_plan* p);
int check_arena(const grm_b200_paged_arena* a);
// The two describe the same pages and heads.
int check_match(const grm_b200_paged_plan* p, const grm_b200_paged_arena* a);
int check_rows(const char* what, const void* ptr, int dtype, int64_t row_stride,
               int64_t head_stride);
int current_sms(int* sms);
// Lets a kernel use `bytes` of dynamic shared memory; `done` (one a kernel)
// remembers the devices where that is set.
int allow_shared(const void* kernel, int bytes, std::atomic<uint64_t>* done);
inline int shift_of(int page_tokens) {  // log2 of 16, 32, 64 or 128
  return page_tokens == 16 ? 4 : page_tokens == 32 ? 5 : page_tokens == 64 ? 6 : 7;
}
int launch_status(const char* what);

}  // namespace paged
}  // namespace grm_b200
