// latent.cu -- pages of latent rows: step plans, append, and the entry points of
// attention (latent_attend.cu).
#include <algorithm>

#include "latent.cuh"
#include "rotary.cuh"

namespace grm_b200 {
namespace latent {

namespace {

using paged::check_plan;
using paged::launch_status;

constexpr int kScheduleThreads = 1024;
constexpr int kForms = 2;  // absorbed, expanded

struct ScheduleParams {
  Lists l[kForms];
  View v[kForms];
  int forms;  // 1 where the plan has no expanded form
  int32_t* room;
  int32_t* status;
  int64_t expand_tokens;
};

// Inclusive prefix sum over the block; `part` is of the block's warps.
__device__ __forceinline__ int64_t block_scan(int64_t v, int64_t* part, int64_t* all) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t up = __shfl_up_sync(kFull, v, o);
    if (lane >= o) v += up;
  }
  __syncthreads();  // the sums of the call before have been read
  if (lane == 31) part[warp] = v;
  __syncthreads();
  if (warp == 0) {
    const int64_t own = part[lane];
    int64_t w = own;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t up = __shfl_up_sync(kFull, w, o);
      if (lane >= o) w += up;
    }
    part[lane] = w - own;
    if (lane == 31) part[32] = w;
  }
  __syncthreads();
  *all = part[32];
  return part[warp] + v;
}

// One block for each form, and one for the room of what is expanded: prefix sums over
// the requests, 1,024 at a time, then each worker's first tile by binary searches.
__global__ void __launch_bounds__(kScheduleThreads) schedule_kernel(const ScheduleParams p) {
  __shared__ int64_t part[33];
  __shared__ Header sh;
  __shared__ int64_t raw[kMostWorkers + 1], first;
  __shared__ unsigned long long whole[kScheduleThreads];
  const int tid = threadIdx.x, form = blockIdx.x;
  const bool sizes = form < p.forms;  // else: room
  const Lists l = p.l[sizes ? form : 0];
  const View v = p.v[sizes ? form : 0];
  const int64_t requests = v.requests;
  int64_t before = 0, room = 0, tiles = 0;
  for (int64_t r0 = 0; r0 < requests; r0 += kScheduleThreads) {
    const int64_t r = r0 + tid;
    int64_t n = 0, tokens = 0, own_tiles = 0;
    if (r < requests) {
      const Request q = request_of(v, (int)r);
      if (q.n > 0) {
        n = q.total * v.tiling.groups;
        own_tiles = (int64_t)q.tiles * v.tiling.groups;
        tokens = ((int64_t)q.len + kExpandAlign - 1) / kExpandAlign * kExpandAlign;
      }
    }
    int64_t all = 0;
    if (sizes) {
      const int64_t incl = block_scan(n, part, &all);
      if (r < requests) l.base[r] = before + incl - n;
      before += all;
    }
    if (sizes && form > 0) {
      const int64_t incl = block_scan(own_tiles, part, &all);
      if (r < requests) l.tile[r] = (int)(tiles + incl - own_tiles);
      tiles += all;
    }
    if (form > 0 || !sizes) {  // the second form's block wants to know if it has room
      const int64_t incl = block_scan(tokens, part, &all);
      if (!sizes && r < requests)
        p.room[r] = (int)min(room + incl - tokens, (int64_t)INT32_MAX);
      room += all;
    }
  }
  const bool lost = p.expand_tokens > 0 && room > p.expand_tokens;
  if (!sizes) {
    if (tid == 0) {
      p.room[requests] = lost ? 0 : (int)room;  // nothing is expanded then
      if (lost) atomicOr(p.status, GRM_B200_PLAN_EXPAND);
    }
    return;
  }
  if (tid == 0) {
    l.base[requests] = before;
    if (form > 0) l.tile[requests] = (int)tiles;
    // whole tiles of each worker, and the unit that follows them
    const int waves = form > 0 ? (int)(tiles / v.tiling.workers) - 1 : 0;
    sh = Header{0, max(waves, 0), lost};
    first = 0;
  }
  __syncthreads();  // and the block's own writes are there
  if (tid == 0) {
    if (sh.waves > 0) {
      Walk walk;
      walk.enter(v, 0);
      walk.tile(v, sh.waves * v.tiling.workers);
      first = l.base[walk.r] + walk.g * walk.q.total + units_before(walk.q, v, walk.j);
    }
    const int64_t units = before - first;
    sh.workers = units == 0      ? 0
                 : sh.waves > 0 ? v.tiling.workers
                                : (int)min((int64_t)v.tiling.workers,
                                           max(units / kLeast, (int64_t)1));
    *l.header = sh;
  }
  __syncthreads();
  // Shares that make up for what the whole tiles of a worker cost more or less than others'.
  const int workers = sh.workers;
  if (workers == 0) return;
  const int64_t rest = before - first;
  int64_t cost = 0, all = 0;
  if (sh.waves > 0) {  // a warp a request, a lane a tile; sums of integers in any order
    whole[tid] = 0;
    __syncthreads();
    const int count = sh.waves * workers;
    for (int64_t r = tid / 32; r < requests; r += kScheduleThreads / 32) {
      const Request q = request_of(v, (int)r);
      const int from = l.tile[r], tiles = min(q.tiles * v.tiling.groups, count - from);
      for (int x = tid % 32; x < tiles; x += 32)
        atomicAdd(&whole[(from + x) % workers],
                  (unsigned long long)tile_units(q, v, x % q.tiles));
    }
    __syncthreads();
    cost = tid < workers ? (int64_t)whole[tid] : 0;
    block_scan(cost, part, &all);
  }
  const int start = v.tiling.start;
  int64_t level = share_level(rest, all, workers, workers, start);
  for (int active = workers; sh.waves > 0;) {  // once where whole tiles cost much the same
    const bool mine = tid < workers && level - cost >= start;
    const int left = __syncthreads_count(mine);
    if (left == active) break;
    active = left;
    block_scan(mine ? cost : 0, part, &all);
    level = share_level(rest, all, workers, active, start);
  }
  const int64_t need = tid < workers ? max(level - cost, (int64_t)start) : 0;
  const int64_t incl = block_scan(need, part, &all);
  if (tid < workers)
    raw[tid] = first + (int64_t)((double)(incl - need) * ((double)rest / (double)all));
  if (tid == 0) {
    raw[workers] = before;
    l.start[workers].u = before;
  }
  __syncthreads();
  if (tid < workers) place_share(v, raw, workers, tid, form == 1, &l.start[tid], &l.join[tid]);
}

struct AppendParams {
  RotaryParams r;
  const int64_t* slots;
  const int32_t* positions;
  int64_t tokens, limit;  // limit: pages * page_tokens
  const uint16_t* latent_rows;
  const uint16_t* rope_rows;
  int64_t latent_stride, rope_stride;
  uint16_t* cache;
  int latent, rope, rotary;
  int copy_shift, rope_shift;  // threads of a row, as powers of two
};

// A thread for 8 values of a row, or for 8 pairs of its positional part, those of all
// rows behind the others, so that a warp has one or the other to do: 8,358 rows of 256 +
// 32 values (9.7 MB in and out, 1.5 us at a copy's rate) take 6.2 us with their positional
// part rotated and 4.2 without, a launch and three dependent loads; 8.2 where every warp
// had two lanes that rotate.
template <typename T, bool IN, bool OUT>
__global__ void __launch_bounds__(256) append_kernel(const AppendParams p) {
  const int copies = p.latent / 8;  // powers of two
  const int64_t x = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int64_t y = x - p.tokens * copies;
  const int shift = y < 0 ? p.copy_shift : p.rope_shift;
  const int64_t t = (y < 0 ? x : y) >> shift;
  if (t >= p.tokens) return;
  const int e = (int)((y < 0 ? x : y) & ((1 << shift) - 1)) + (y < 0 ? 0 : copies);
  const int64_t slot = p.slots[t];
  if (slot < 0 || slot >= p.limit) return;
  uint16_t* to = p.cache + slot * (p.latent + p.rope);
  if (e < copies) {
    reinterpret_cast<uint4*>(to)[e] = ld_nc16(p.latent_rows + t * p.latent_stride + e * 8);
    return;
  }
  const uint16_t* from = p.rope_rows + t * p.rope_stride;
  to += p.latent;
  const int c = (e - copies) * 8;
  if (!p.rotary) {
    *reinterpret_cast<uint4*>(to + c) = ld_nc16(from + c);
    return;
  }
  const int position = p.positions[t];
  float2 angle[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const Turn a = turn_of(position, p.r.turns[c + i]);
    angle[i] = make_float2(a.cos * p.r.amplitude, a.sin * p.r.amplitude);
  }
  turn_pairs<T, 8, IN, OUT>(p.rope / 2, angle, c, reinterpret_cast<const T*>(from),
                            reinterpret_cast<T*>(to));
}

template <typename T>
int launch_append(const AppendParams& p, cudaStream_t st) {
  const unsigned blocks = (unsigned)ceil_div64(
      p.tokens * ((1 << p.copy_shift) + (1 << p.rope_shift)), 256);
  if (!p.rotary || p.r.layout == GRM_B200_ROTARY_HALF)
    append_kernel<T, false, false><<<blocks, 256, 0, st>>>(p);
  else if (p.r.layout == GRM_B200_ROTARY_INTERLEAVED)
    append_kernel<T, true, true><<<blocks, 256, 0, st>>>(p);
  else
    append_kernel<T, true, false><<<blocks, 256, 0, st>>>(p);
  return launch_status("latent append");
}

int64_t align256(int64_t v) { return (v + 255) & ~(int64_t)255; }

bool latent_ok(int v) { return v == 128 || v == 256 || v == 512; }
bool rope_ok(int v) { return v == 32 || v == 64; }

int check_sizes(const grm_b200_latent_plan* p) {
  if (!p) {
    set_thread_error("latent plan: null plan");
    return GRM_B200_EINVAL;
  }
  if (!latent_ok(p->latent) || !rope_ok(p->rope)) {
    set_thread_error("latent plan: latent %d must be 128, 256 or 512 and rope %d 32 or 64",
                     p->latent, p->rope);
    return GRM_B200_EINVAL;
  }
  if (p->heads < 1 || p->heads > 1024) {
    set_thread_error("latent plan: heads %d must be 1 to 1024", p->heads);
    return GRM_B200_EINVAL;
  }
  if (p->step.tokens > INT32_MAX / p->heads) {
    set_thread_error("latent plan: %lld rows of %d heads are more than 2^31 - 1",
                     (long long)p->step.tokens, p->heads);
    return GRM_B200_EINVAL;
  }
  const bool none = p->nope == 0 && p->value == 0 && p->expand_tokens == 0;
  const bool some = (p->nope == 64 || p->nope == 128) && p->value == p->nope &&
                    p->expand_tokens >= 1 && p->expand_tokens <= (1 << 28) &&
                    p->expand_tokens * p->heads <= INT32_MAX;  // rows of keys
  if (!none && !some) {
    set_thread_error("latent plan: nope %d and value %d must both be 64 or both 128, with "
                     "expand_tokens %lld from 1 to 2^28 and below 2^31 times the heads (or all 0)",
                     p->nope, p->value, (long long)p->expand_tokens);
    return GRM_B200_EINVAL;
  }
  return 0;
}

// What does not need a device first, so that a call that cannot be right is refused
// without one.
int check_latent_plan(const grm_b200_latent_plan* p) {
  int rc = check_sizes(p);
  if (rc) return rc;
  if (!p->work || (reinterpret_cast<uintptr_t>(p->work) & 255)) {
    set_thread_error("latent plan: work must be 256-byte aligned device memory");
    return GRM_B200_EINVAL;
  }
  if ((rc = check_plan(&p->step))) return rc;
  int64_t need = 0;
  rc = grm_b200_latent_work_bytes(p, &need);
  if (rc) return rc;
  if (p->work_bytes < need) {
    set_thread_error("latent plan: work of %lld bytes, %lld needed", (long long)p->work_bytes,
                     (long long)need);
    return GRM_B200_EINVAL;
  }
  return 0;
}

int check_latent_arena(const grm_b200_latent_arena* a) {
  if (!a || !a->rows || (reinterpret_cast<uintptr_t>(a->rows) & 15)) {
    set_thread_error("latent arena: rows must be 16-byte aligned device memory");
    return GRM_B200_EINVAL;
  }
  if (a->pages < 1 || a->pages > INT32_MAX / 128 ||
      (a->page_tokens != 16 && a->page_tokens != 32 && a->page_tokens != 64 &&
       a->page_tokens != 128) ||
      !latent_ok(a->latent) || !rope_ok(a->rope) ||
      (a->dtype != GRM_B200_F16 && a->dtype != GRM_B200_BF16)) {
    set_thread_error("latent arena: pages %lld (at most 2^24 - 1), page_tokens %d (16, 32, 64, "
                     "128), latent %d (128, 256, 512), rope %d (32, 64), fp16 or bf16 rows",
                     (long long)a->pages, a->page_tokens, a->latent, a->rope);
    return GRM_B200_EINVAL;
  }
  return 0;
}

int check_match(const grm_b200_latent_plan* p, const grm_b200_latent_arena* a) {
  if (a->pages != p->step.pages || a->page_tokens != p->step.page_tokens ||
      a->latent != p->latent || a->rope != p->rope) {
    set_thread_error("latent plan and arena differ: pages %lld / %lld, page_tokens %d / %d, "
                     "latent %d / %d, rope %d / %d", (long long)p->step.pages, (long long)a->pages,
                     p->step.page_tokens, a->page_tokens, p->latent, a->latent, p->rope, a->rope);
    return GRM_B200_EINVAL;
  }
  return 0;
}

int check_attend(const grm_b200_latent_plan* plan, const grm_b200_latent_arena* arena,
                 float softmax_scale, int causal, const void* out) {
  int rc;
  if ((rc = check_sizes(plan)) || (rc = check_latent_arena(arena)) ||
      (rc = check_match(plan, arena)))
    return rc;
  if (!out || (reinterpret_cast<uintptr_t>(out) & 15)) {
    set_thread_error("latent attend: out must be 16-byte aligned device memory");
    return GRM_B200_EINVAL;
  }
  if (causal && !plan->step.grow) {
    set_thread_error("latent attend: rows that do not join the arena (grow = 0) have no position "
                     "in it; attend with causal = 0");
    return GRM_B200_EINVAL;
  }
  if (!(softmax_scale > 0.0f) || !(softmax_scale < INFINITY)) {
    set_thread_error("latent attend: softmax_scale %g must be positive and finite",
                     (double)softmax_scale);
    return GRM_B200_EINVAL;
  }
  return 0;
}

View view_of(const grm_b200_latent_plan& plan, const Shape& s, int form) {
  const Lists l = lists_of(s, form, plan.work);
  return {l.base, l.tile, plan.step.starts, plan.step.lens, plan.step.requests,
          s.tiling[form], plan.step.grow ? 1 : 0, plan.heads};
}

int fill(const grm_b200_latent_plan* plan, const grm_b200_latent_arena* arena, int form,
         float softmax_scale, int causal, void* out, float* lse, Params* p) {
  int sms = 0;
  int rc = paged::current_sms(&sms);
  if (rc) return rc;
  Shape s;
  make_shape(*plan, sms, &s);
  *p = Params{};
  p->l = lists_of(s, form, plan->work);
  p->v = view_of(*plan, s, form);
  p->probes = std::min(scan_wait_limit(), paged::kProbes);
  char* work = static_cast<char*>(plan->work);
  p->room = reinterpret_cast<const int32_t*>(work + s.off_room);
  p->keys = reinterpret_cast<uint16_t*>(work + s.off_keys);
  p->values = reinterpret_cast<uint16_t*>(work + s.off_values);
  p->table = plan->step.table;
  p->width = plan->step.table_width;
  p->tokens = plan->step.tokens;
  p->pages = plan->step.pages;
  p->expand_tokens = plan->expand_tokens;
  p->page_shift = paged::shift_of(plan->step.page_tokens);
  p->heads = plan->heads;
  p->latent = plan->latent;
  p->rope = plan->rope;
  p->nope = plan->nope;
  p->causal = causal ? 1 : 0;
  p->dtype = arena->dtype;
  p->cache = static_cast<const uint16_t*>(arena->rows);
  p->scale_log2 = softmax_scale * 1.44269504088896341f;
  p->out = static_cast<uint16_t*>(out);
  p->lse = lse;
  p->status = plan->step.status;
  return 0;
}

}  // namespace

int make_shape(const grm_b200_latent_plan& p, int sms, Shape* s) {
  sms = std::min(sms, kMostWorkers);
  s->tiling[0] = absorbed_tiling(p.heads, p.latent, std::min(p.step.max_fresh, p.step.tokens), sms);
  s->tiling[1] = expanded_tiling(p.heads, sms);
  int64_t at = 0;
  auto take = [&](int64_t bytes) {
    const int64_t o = at;
    at += align256(bytes);
    return o;
  };
  for (int f = 0; f < kForms; ++f) {
    s->off_header[f] = take(sizeof(Header));
    s->off_base[f] = take((p.step.requests + 1) * 8);
    s->off_tile[f] = take(f > 0 ? (p.step.requests + 1) * 4 : 0);
    s->off_start[f] = take((int64_t)(s->tiling[f].workers + 1) * (int64_t)sizeof(Start));
    s->off_join[f] = take((int64_t)s->tiling[f].workers * (int64_t)sizeof(Join));
  }
  const Tiling& t = s->tiling[0];
  const int64_t absorbed = (int64_t)t.workers * t.splits *
                           (t.few ? slot_floats(t.few, p.latent)
                                  : slot_floats(kRows, std::min(p.latent, 256)));
  const int64_t expanded =
      p.nope ? (int64_t)s->tiling[1].workers * slot_floats(2 * kRows, p.value) : 0;
  s->off_part = take(std::max(absorbed, expanded) * 2 * 4);
  s->off_room = take((p.step.requests + 1) * 4);
  s->off_keys = take(p.expand_tokens * p.heads * 2 * p.nope * 2);
  s->off_values = take(p.expand_tokens * p.heads * p.value * 2);
  s->bytes = at;
  return 0;
}

// cuTensorMapEncodeTiled from the driver, looked up once (no libcuda link).
using EncodeTiled = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*,
                                 const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                                 const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                 CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
static EncodeTiled encode_tiled() {
  static const EncodeTiled fn = [] {
    void* f = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &f, 12000, cudaEnableDefault,
                                         &q) != cudaSuccess ||
        q != cudaDriverEntryPointSuccess)
      f = nullptr;
    return reinterpret_cast<EncodeTiled>(f);
  }();
  return fn;
}

int make_map(CUtensorMap* map, const void* base, int rank, const int64_t* dims,
             const int64_t* strides, const int* box) {
  const EncodeTiled encode = encode_tiled();
  cuuint64_t d[3], s[2];
  cuuint32_t b[3];
  const cuuint32_t step[3] = {1, 1, 1};
  for (int i = 0; i < rank; ++i) {
    d[i] = (cuuint64_t)dims[i];
    b[i] = (cuuint32_t)box[i];
    if (i > 0) s[i - 1] = (cuuint64_t)strides[i - 1] * 2;
  }
  if (!encode ||
      encode(map, CU_TENSOR_MAP_DATA_TYPE_UINT16, rank, const_cast<void*>(base), d, s, b, step,
             CU_TENSOR_MAP_INTERLEAVE_NONE,
             box[0] == 64 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B,
             CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
             CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS) {
    set_thread_error("latent attend: no tensor map of rows of %lld values", (long long)dims[0]);
    return GRM_B200_EINVAL;
  }
  return 0;
}

}  // namespace latent
}  // namespace grm_b200

using namespace grm_b200;
using namespace grm_b200::latent;

extern "C" {

int grm_b200_latent_work_bytes(const grm_b200_latent_plan* plan, int64_t* out_bytes) {
  int rc = check_sizes(plan);
  if (rc) return rc;
  if (!out_bytes) {
    set_thread_error("latent plan: null out_bytes");
    return GRM_B200_EINVAL;
  }
  int64_t step = 0;
  int sms = 0;
  if ((rc = grm_b200_paged_scratch_bytes(&plan->step, &step)) || (rc = paged::current_sms(&sms)))
    return rc;
  Shape s;
  make_shape(*plan, sms, &s);
  *out_bytes = s.bytes;
  return 0;
}

int grm_b200_latent_plan_step(const grm_b200_latent_plan* plan, const int32_t* fresh_device,
                              void* stream) {
  int rc = check_latent_plan(plan);
  if (rc) return rc;
  int sms = 0;
  if ((rc = paged::current_sms(&sms)) ||
      (rc = grm_b200_paged_plan_step(&plan->step, fresh_device, stream)))
    return rc;
  Shape s;
  make_shape(*plan, sms, &s);
  ScheduleParams p;
  for (int f = 0; f < kForms; ++f) {
    p.l[f] = lists_of(s, f, plan->work);
    p.v[f] = view_of(*plan, s, f);
  }
  p.forms = plan->nope ? kForms : 1;
  p.room = reinterpret_cast<int32_t*>(static_cast<char*>(plan->work) + s.off_room);
  p.status = plan->step.status;
  p.expand_tokens = plan->expand_tokens;
  schedule_kernel<<<plan->nope ? kForms + 1 : 1, kScheduleThreads, 0,
                    static_cast<cudaStream_t>(stream)>>>(p);
  return launch_status("latent plan");
}

int grm_b200_latent_append(const grm_b200_latent_plan* plan, const grm_b200_latent_arena* arena,
                           const grm_b200_rotary* rotary, const void* latent_device,
                           int64_t latent_row_stride, const void* rope_device,
                           int64_t rope_row_stride, void* stream) {
  int rc;
  if ((rc = check_sizes(plan)) || (rc = check_latent_arena(arena)) ||
      (rc = check_match(plan, arena)) ||
      (rc = paged::check_rows("latent append", latent_device, arena->dtype, latent_row_stride,
                              0)) ||
      (rc = paged::check_rows("latent append", rope_device, arena->dtype, rope_row_stride, 0)) ||
      (rotary && (rc = check_rotary("latent append", rotary))))
    return rc;
  if (rotary && (rotary->dim != arena->rope || rotary->offset != 0)) {
    set_thread_error("latent append: the rotary's dim %d and offset %d must be %d and 0",
                     rotary->dim, rotary->offset, arena->rope);
    return GRM_B200_EINVAL;
  }
  if (!plan->step.grow) {
    set_thread_error("latent append: the plan's rows do not join the arena (grow = 0)");
    return GRM_B200_EINVAL;
  }
  if ((rc = check_latent_plan(plan))) return rc;
  AppendParams p;
  p.r = rotary ? rotary_params(*rotary) : RotaryParams{};
  p.slots = plan->step.slots;
  p.positions = plan->step.positions;
  p.tokens = plan->step.tokens;
  p.limit = arena->pages * arena->page_tokens;
  p.latent_rows = static_cast<const uint16_t*>(latent_device);
  p.rope_rows = static_cast<const uint16_t*>(rope_device);
  p.latent_stride = latent_row_stride;
  p.rope_stride = rope_row_stride;
  p.cache = static_cast<uint16_t*>(arena->rows);
  p.latent = arena->latent;
  p.rope = arena->rope;
  p.rotary = rotary != nullptr;
  auto log2_of = [](int n) { int s = 0; while (n > 1) { n >>= 1; ++s; } return s; };
  p.copy_shift = log2_of(arena->latent / 8);
  p.rope_shift = log2_of(arena->rope / (rotary ? 16 : 8));
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return arena->dtype == GRM_B200_F16 ? launch_append<__half>(p, st)
                                      : launch_append<__nv_bfloat16>(p, st);
}

int grm_b200_latent_attend(const grm_b200_latent_plan* plan, const grm_b200_latent_arena* arena,
                           const void* q_latent_device, int64_t q_latent_row_stride,
                           int64_t q_latent_head_stride, const void* q_rope_device,
                           int64_t q_rope_row_stride, int64_t q_rope_head_stride,
                           float softmax_scale, int causal, void* out_device, float* lse_device,
                           void* stream) {
  int rc;
  Params p;
  if ((rc = check_attend(plan, arena, softmax_scale, causal, out_device)) ||
      (rc = paged::check_rows("latent attend", q_latent_device, arena->dtype, q_latent_row_stride,
                              q_latent_head_stride)) ||
      (rc = paged::check_rows("latent attend", q_rope_device, arena->dtype, q_rope_row_stride,
                              q_rope_head_stride)) ||
      (rc = check_latent_plan(plan)) ||
      (rc = fill(plan, arena, 0, softmax_scale, causal, out_device, lse_device, &p)))
    return rc;
  p.q = static_cast<const uint16_t*>(q_latent_device);
  p.q_row = q_latent_row_stride;
  p.q_head = q_latent_head_stride;
  p.qr = static_cast<const uint16_t*>(q_rope_device);
  p.qr_row = q_rope_row_stride;
  p.qr_head = q_rope_head_stride;
  return p.v.tiling.few ? launch_few(p, static_cast<cudaStream_t>(stream))
                        : launch_absorbed(p, static_cast<cudaStream_t>(stream));
}

int grm_b200_latent_attend_expanded(const grm_b200_latent_plan* plan,
                                    const grm_b200_latent_arena* arena, const void* q_device,
                                    int64_t q_row_stride, int64_t q_head_stride,
                                    const void* weights_device, int64_t weights_head_stride,
                                    int64_t weights_row_stride, float softmax_scale, int causal,
                                    void* out_device, float* lse_device, void* stream) {
  int rc;
  Params p;
  if ((rc = check_attend(plan, arena, softmax_scale, causal, out_device)) ||
      (rc = paged::check_rows("latent attend", q_device, arena->dtype, q_row_stride,
                              q_head_stride)) ||
      (rc = paged::check_rows("latent attend", weights_device, arena->dtype, weights_row_stride,
                              weights_head_stride)))
    return rc;
  if (plan->nope == 0) {
    set_thread_error("latent attend: the plan has no room for the expanded form (expand_tokens)");
    return GRM_B200_EINVAL;
  }
  if (weights_row_stride < arena->latent ||
      (weights_head_stride != 0 && weights_head_stride < arena->latent)) {
    set_thread_error("latent attend: weights' rows overlap (head stride %lld, row stride %lld)",
                     (long long)weights_head_stride, (long long)weights_row_stride);
    return GRM_B200_EINVAL;
  }
  if ((rc = check_latent_plan(plan)) ||
      (rc = fill(plan, arena, 1, softmax_scale, causal, out_device, lse_device, &p)))
    return rc;
  p.q = static_cast<const uint16_t*>(q_device);
  p.q_row = q_row_stride;
  p.q_head = q_head_stride;
  p.qr = p.q + plan->nope;
  p.qr_row = q_row_stride;
  p.qr_head = q_head_stride;
  p.weights = static_cast<const uint16_t*>(weights_device);
  p.w_head = weights_head_stride;
  p.w_row = weights_row_stride;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if ((rc = launch_expand(p, st))) return rc;
  return launch_expanded(p, st);
}

}  // extern "C"
