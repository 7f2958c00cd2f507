// latent.cuh -- what the kernels over pages of latent rows share.
#pragma once

#include "paged.cuh"

namespace grm_b200 {
namespace latent {

// Tokens of a request are expanded from a multiple of this on.
constexpr int kExpandAlign = 64;

struct Header {      // written by the schedule kernel
  int32_t rows;      // packed rows of the step
  int32_t overflow;  // more tokens to expand than there is room for
};

// Byte offsets in the work area, which follow from the plan's sizes alone.
struct Shape {
  int64_t off_base, off_keys, off_values, bytes;
};

struct Work {
  Header* header;
  int32_t* base;     // [requests + 1] first expanded token of each request
  uint16_t* keys;    // [heads][expand_tokens][nope]
  uint16_t* values;  // [heads][expand_tokens][value]
};

int make_shape(const grm_b200_latent_plan& p, int sms, Shape* s);
inline Work work_of(const Shape& s, void* work) {
  char* b = static_cast<char*>(work);
  return {reinterpret_cast<Header*>(b), reinterpret_cast<int32_t*>(b + s.off_base),
          reinterpret_cast<uint16_t*>(b + s.off_keys),
          reinterpret_cast<uint16_t*>(b + s.off_values)};
}

struct Params {
  Work w;
  const int32_t* table;
  const int32_t* lens;
  const int32_t* starts;
  int64_t requests, width, tokens, pages, expand_tokens;
  int page_shift, heads, latent, rope, nope, value, causal;
  const uint16_t* cache;
  const uint16_t* q;      // absorbed: the latent part; expanded: nope + rope values
  int64_t q_row, q_head;
  const uint16_t* qr;     // the positional part
  int64_t qr_row, qr_head;
  const uint16_t* weights;
  int64_t w_head, w_row;
  float scale_log2;
  uint16_t* out;
  float* lse;
  int32_t* status;
};

int launch_absorbed(int dtype, const Params& p, cudaStream_t st);
int launch_expanded(int dtype, const Params& p, cudaStream_t st);

}  // namespace latent
}  // namespace grm_b200
