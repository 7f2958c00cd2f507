// paged.cuh -- what the kernels of the 8-bit paged arena share: the layout of a
// plan's scratch (work lists and partial results) and the checks of arguments.
#pragma once

#include "common.cuh"

namespace grm_b200 {
namespace paged {

// Attention walks a request's tokens in tiles of kTile.  The split kernel gives
// every worker (a resident block) the same number of units: a request, kv head
// and block of query rows ("segment") costs its tiles and one unit more for
// its start and end.
constexpr int kTile = 64;
constexpr int kWorkerSlot = 2048 + 64;  // fp32 of one partial result: rows x dim, then (M, L)

struct Header {           // written by the plan kernel
  int64_t units;          // units of the split kernel's work, all requests
  int32_t workers;        // workers that share them (<= Shape::workers)
  int32_t pages;          // entries of the append list
  int32_t qtiles;         // entries of the prompt kernel's list
  int32_t rows;           // packed rows of the step
};

// Sizes that follow from the plan's sizes alone, so that the plan kernel and
// the kernels that read its lists agree without the host seeing a length.
struct Shape {
  int group;            // query heads of a kv head
  int split_rows;       // requests with more (row, head) pairs a kv head than this are prompts
  int block_rows;       // rows of a segment: 8 or 16
  int qtile_tokens;     // tokens of a prompt tile
  int workers;          // resident blocks of the split kernel
  int64_t page_cap;     // most pages a step can touch
  int64_t qtile_cap;    // most prompt tiles (0: no request can be a prompt)
  // byte offsets in the scratch
  int64_t off_base, off_start, off_count, off_pages, off_qtiles, off_part, bytes;
};

int make_shape(const grm_b200_paged_plan& p, int sms, Shape* s);

struct Lists {
  Header* header;
  int64_t* base;      // [requests + 1] first unit of each request
  int32_t* start;     // [workers] request of a worker's first unit
  unsigned* count;    // [workers] arrivals at the segment that a worker starts; 0 between calls
  int2* pages;        // [page_cap] (request, page of the request)
  int2* qtiles;       // [qtile_cap] (request, first row of the tile within the request)
  float* part;        // [workers * 2][kWorkerSlot]
};

inline Lists lists_of(const Shape& s, void* scratch) {
  char* b = static_cast<char*>(scratch);
  return {reinterpret_cast<Header*>(b),
          reinterpret_cast<int64_t*>(b + s.off_base),
          reinterpret_cast<int32_t*>(b + s.off_start),
          reinterpret_cast<unsigned*>(b + s.off_count),
          reinterpret_cast<int2*>(b + s.off_pages),
          reinterpret_cast<int2*>(b + s.off_qtiles),
          reinterpret_cast<float*>(b + s.off_part)};
}

// First unit of worker w of `workers`, and the worker that holds unit u: the
// largest w with first(w) <= u.
__host__ __device__ inline int64_t worker_first(int64_t w, int64_t units, int64_t workers) {
  return w * units / workers;
}
__host__ __device__ inline int64_t worker_of(int64_t u, int64_t units, int64_t workers) {
  return ((u + 1) * workers - 1) / units;
}

int check_plan(const grm_b200_paged_plan* p);
int check_arena(const grm_b200_paged_arena* a);
// The two describe the same pages and heads.
int check_match(const grm_b200_paged_plan* p, const grm_b200_paged_arena* a);
int check_rows(const char* what, const void* ptr, int dtype, int64_t row_stride,
               int64_t head_stride);
int current_sms(int* sms);
inline int shift_of(int page_tokens) {  // log2 of 16, 32, 64 or 128
  return page_tokens == 16 ? 4 : page_tokens == 32 ? 5 : page_tokens == 64 ? 6 : 7;
}
int launch_status(const char* what);

}  // namespace paged
}  // namespace grm_b200
