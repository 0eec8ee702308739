// abi_block.cpp — extern "C" entry points of the operators of the attention
// block beside the cache (nkv_rope_tables, nkv_rotary, nkv_residual_norm,
// nkv_attend_*): argument checks, the plan object, launches.
#include <cuda_runtime.h>

#include <algorithm>
#include <cmath>
#include <functional>
#include <memory>
#include <string>
#include <vector>

#include "bank.h"
#include "nkv_kernels.h"
#include "nkv_packed.h"
#include "nomas_kv.h"

namespace nkv {
int guarded_call(const std::function<void()>& f);
}

using nkv::fail;

struct nkv_attend_plan {
  int device = 0;
  int32_t H = 0, kv_heads = 0, D = 0, causal = 0;
  int64_t block = 1;
  uint64_t q_tokens = 0, k_tokens = 0, part_rows = 0;
  int32_t n_items = 0, n_ctas = 0, n_units = 0, max_unit_rows = 0;
  // status word (64 bytes), items, where each CTA's begin, each one's first, units
  unsigned char* table = nullptr;
  size_t items_off = 64, ctas_off = 0, first_off = 0, units_off = 0;
  uint64_t workspace() const {  // partial rows, then their (max, sum)
    return part_rows * (uint64_t(D) * sizeof(float) + sizeof(float2));
  }
};

namespace {

void need(const void* p, const char* what) {
  if (!p) fail(NKV_ERR_ARGUMENT, std::string("null ") + what);
}

bool aligned(const void* p, uintptr_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

bool float_type(int32_t dt) { return dt == NKV_F32 || dt == NKV_BF16 || dt == NKV_F16; }

// The axes' pairs and frequencies.  The last configuration's are kept per
// thread: 64 powers take longer than a small call's other host work.
nkv::RopePositions rope_positions(const nkv_rope_axes& ax, const void* positions, int32_t type) {
  if (ax.n_axes < 1 || ax.n_axes > 4) fail(NKV_ERR_INVALID_CONFIG, "rotary positions need 1 to 4 axes");
  if (!(ax.theta > 0.0) || !std::isfinite(ax.theta))
    fail(NKV_ERR_INVALID_CONFIG, "theta must be finite and positive");
  if (type < NKV_POS_I32 || type > NKV_POS_F32)
    fail(NKV_ERR_ARGUMENT, "unknown position type " + std::to_string(type));
  struct Known {
    int32_t n_axes = 0, dims[4] = {0, 0, 0, 0};
    double theta = 0.0;
    nkv::RopePositions p{};
  };
  static thread_local Known known;
  if (known.n_axes != ax.n_axes || known.theta != ax.theta || !std::equal(ax.dims, ax.dims + ax.n_axes, known.dims)) {
    nkv::RopePositions p{};
    p.n_axes = ax.n_axes;
    for (int a = 0; a < ax.n_axes; ++a) {
      const int32_t d = ax.dims[a];
      if (d < 2 || d % 2 || d > nkv::kRotaryMaxDim || p.pairs + d / 2 > nkv::kRotaryMaxDim / 2)
        fail(NKV_ERR_INVALID_CONFIG, "rotary axes need even dims >= 2 with a sum of at most 256");
      for (int i = 0; i < d / 2; ++i) {
        p.axis[p.pairs] = uint8_t(a);
        p.freq[p.pairs++] = std::pow(ax.theta, -2.0 * i / d);
      }
    }
    known.n_axes = ax.n_axes;
    std::copy(ax.dims, ax.dims + ax.n_axes, known.dims);
    known.theta = ax.theta;
    known.p = p;
  }
  nkv::RopePositions p = known.p;
  p.data = positions;
  p.dtype = type;
  return p;
}

void check_positions(const void* positions, int32_t type) {
  need(positions, "positions");
  if (!aligned(positions, type == NKV_POS_I64 ? 8 : 4))
    fail(NKV_ERR_ARGUMENT, "positions must be aligned to their type");
}

void check_tokens(uint64_t tokens) {
  if (tokens >= (uint64_t(1) << 31)) fail(NKV_ERR_ARGUMENT, "tokens must be below 2^31");
}

nkv::RotarySide rotary_side(const nkv_rotary_side& s, size_t es, const char* name) {
  nkv::RotarySide r{};
  if (s.heads < 0 || s.heads > 65535) fail(NKV_ERR_ARGUMENT, std::string(name) + " heads must be 0 to 65535");
  if (s.heads == 0) return r;
  need(s.in, name);
  need(s.out, name);
  if (!aligned(s.in, es) || !aligned(s.out, es) || !aligned(s.weight, es))
    fail(NKV_ERR_ARGUMENT, std::string(name) + " must be aligned to its type");
  if (s.in_token_stride < 0 || s.in_head_stride < 0 || s.out_token_stride < 0 || s.out_head_stride < 0)
    fail(NKV_ERR_ARGUMENT, std::string(name) + " strides must not be negative");
  r.in = s.in, r.out = s.out;
  r.in_token = s.in_token_stride, r.in_head = s.in_head_stride;
  r.out_token = s.out_token_stride, r.out_head = s.out_head_stride;
  r.weight = s.weight;
  r.heads = s.heads;
  return r;
}

struct Lens {
  std::vector<int64_t> q, k;
  uint64_t q_tokens = 0, k_tokens = 0;
};

Lens check_lens(const uint64_t* q_lens, const uint64_t* k_lens, uint64_t n, int32_t heads, int32_t kv_heads,
                uint64_t block) {
  if (n) need(q_lens, "q_lens"), need(k_lens, "k_lens");
  if (heads < 1 || kv_heads < 1 || heads % kv_heads || heads > 65535)
    fail(NKV_ERR_GEOMETRY, "heads must be a positive multiple of kv_heads, at most 65535");
  if (heads / kv_heads > nkv::kPackedHalfRows)
    fail(NKV_ERR_GEOMETRY, "at most 128 query heads per key/value head");
  if (block < 1 || block >= (uint64_t(1) << 31)) fail(NKV_ERR_ARGUMENT, "block must be 1 to 2^31 - 1");
  // packed rows (tokens x group) and tile coordinates are 32-bit
  constexpr uint64_t kMax = (uint64_t(1) << 31) - 1024;
  const uint64_t group = uint64_t(heads / kv_heads);
  constexpr uint64_t kMaxItems = uint64_t(1) << 22;  // a quarter of a gigabyte of work list
  const uint64_t half = group * (nkv::kPackedHalfRows / group);
  uint64_t items = 0;
  Lens l;
  for (uint64_t s = 0; s < n; ++s) {
    if (q_lens[s] > kMax || k_lens[s] > kMax) fail(NKV_ERR_GEOMETRY, "sequence too long");
    l.q_tokens += q_lens[s];
    l.k_tokens += k_lens[s];
    if (l.q_tokens * group > kMax || l.k_tokens > kMax)
      fail(NKV_ERR_GEOMETRY, "packed tokens x heads per group, and packed keys, must be below 2^31");
    items += (q_lens[s] * group + half - 1) / half * uint64_t(kv_heads);
    if (items > kMaxItems) fail(NKV_ERR_GEOMETRY, "too many rows for one plan: at most 2^22 work items");
    l.q.push_back(int64_t(q_lens[s]));
    l.k.push_back(int64_t(k_lens[s]));
  }
  return l;
}

void check_strides(const void* p, int64_t token, int64_t head, int64_t tokens, int64_t heads, const char* name) {
  if (!aligned(p, 16) || token % 8 || head % 8)
    fail(NKV_ERR_ARGUMENT, std::string(name) + " must be 16-byte aligned with strides of multiples of 8 elements");
  // a stride counts only where there is a second element
  if ((tokens > 1 && token <= 0) || (heads > 1 && head <= 0))
    fail(NKV_ERR_ARGUMENT, std::string(name) + " strides must be positive");
  constexpr int64_t kMaxStride = int64_t(1) << 38;  // elements: the tensor map's byte strides are below 2^40
  if (token > kMaxStride || head > kMaxStride) fail(NKV_ERR_ARGUMENT, std::string(name) + " strides are too large");
}

// Makes `device` current for a scope.
struct OnDevice {
  int prev = 0;
  explicit OnDevice(int device) {
    nkv::check_cuda(cudaGetDevice(&prev), "cudaGetDevice");
    nkv::check_cuda(cudaSetDevice(device), "cudaSetDevice");
  }
  ~OnDevice() { cudaSetDevice(prev); }
};

// Lets this thread allocate, copy and free (a plan's table, none of it work of
// a stream's) while one of the process's streams is being captured.
struct DuringCapture {
  cudaStreamCaptureMode mode = cudaStreamCaptureModeRelaxed;
  DuringCapture() { nkv::check_cuda(cudaThreadExchangeStreamCaptureMode(&mode), "cudaThreadExchangeStreamCaptureMode"); }
  ~DuringCapture() { cudaThreadExchangeStreamCaptureMode(&mode); }
};

}  // namespace

extern "C" {

int nkv_rope_tables(const nkv_rope_axes* axes, const void* positions, int32_t position_type, uint64_t tokens,
                    float* cos_out, float* sin_out, void* stream) {
  return nkv::guarded_call([&] {
    need(axes, "axes");
    const nkv::RopePositions p = rope_positions(*axes, positions, position_type);
    check_tokens(tokens);
    if (tokens == 0) return;
    check_positions(positions, position_type);
    need(cos_out, "cos output"), need(sin_out, "sin output");
    if (!aligned(cos_out, 4) || !aligned(sin_out, 4)) fail(NKV_ERR_ARGUMENT, "tables must be aligned to f32");
    nkv::check_cuda(nkv::launch_rope_tables(p, tokens, cos_out, sin_out, static_cast<cudaStream_t>(stream)),
                    "rope tables launch");
  });
}

int nkv_rotary(const nkv_rotary_args* a, void* stream) {
  return nkv::guarded_call([&] {
    need(a, "args");
    nkv::RotaryParams p{};
    p.pos = rope_positions(a->axes, a->positions, a->position_type);
    if (!float_type(a->dtype)) fail(NKV_ERR_ARGUMENT, "unknown dtype " + std::to_string(a->dtype));
    if (a->head_dim < 2 || a->head_dim % 2 || a->head_dim > nkv::kRotaryMaxDim)
      fail(NKV_ERR_GEOMETRY, "head_dim must be even, 2 to 256");
    if (2 * p.pos.pairs > a->head_dim) fail(NKV_ERR_GEOMETRY, "rotary axes exceed head_dim");
    if (a->norm && !(a->eps >= 0.0f && std::isfinite(a->eps)))
      fail(NKV_ERR_ARGUMENT, "eps must be finite and not negative");
    check_tokens(a->tokens);
    const size_t es = nkv::dtype_size(a->dtype);
    if (a->tokens == 0) return;
    p.side[0] = rotary_side(a->q, es, "q");
    p.side[1] = rotary_side(a->k, es, "k");
    if (p.side[0].heads + p.side[1].heads == 0) return;
    check_positions(a->positions, a->position_type);
    p.tokens = a->tokens;
    p.D = a->head_dim;
    p.interleaved = a->axes.interleaved ? 1 : 0;
    p.norm = a->norm ? 1 : 0;
    p.eps = a->eps;
    nkv::check_cuda(nkv::launch_rotary(p, a->dtype, static_cast<cudaStream_t>(stream)), "rotary launch");
  });
}

int nkv_residual_norm(const nkv_residual_norm_args* a, void* stream) {
  return nkv::guarded_call([&] {
    need(a, "args");
    if (!float_type(a->dtype)) fail(NKV_ERR_ARGUMENT, "unknown dtype " + std::to_string(a->dtype));
    for (int32_t dt : {a->weight_dtype, a->mod_dtype})
      if (dt != NKV_F32 && dt != a->dtype)
        fail(NKV_ERR_ARGUMENT, "weights and modulation must be f32 or the stream's dtype");
    if (a->dim < 1 || a->dim > nkv::kResidualNormMaxDim) fail(NKV_ERR_GEOMETRY, "dim must be 1 to 32768");
    for (int32_t k : {a->post, a->norm})
      if (k < NKV_NORM_NONE || k > NKV_NORM_LAYER) fail(NKV_ERR_ARGUMENT, "unknown norm kind " + std::to_string(k));
    if (!(a->eps >= 0.0f && std::isfinite(a->eps))) fail(NKV_ERR_ARGUMENT, "eps must be finite and not negative");
    if (!a->branch && (a->post || a->gate || a->post_weight))
      fail(NKV_ERR_ARGUMENT, "post, post_weight and gate need a branch");
    if (!a->branch && !a->norm) fail(NKV_ERR_ARGUMENT, "nothing to do: no branch and no norm");
    if (!a->norm && (a->weight || a->scale || a->shift))
      fail(NKV_ERR_ARGUMENT, "weight, scale and shift need a norm");
    const bool mods = a->gate || a->scale || a->shift;
    if (mods && a->mod_rows < 1) fail(NKV_ERR_GEOMETRY, "mod_rows must be positive");
    if (mods && !a->mod_index && a->mod_rows != 1)
      fail(NKV_ERR_GEOMETRY, "several modulation rows need mod_index");
    check_tokens(a->tokens);
    if (a->tokens == 0) return;
    need(a->x, "x");
    if (a->branch) need(a->h_out, "h output");
    if (a->norm) need(a->y_out, "y output");
    const size_t es = nkv::dtype_size(a->dtype), ws = nkv::dtype_size(a->weight_dtype),
                 ms = nkv::dtype_size(a->mod_dtype);
    if (!aligned(a->x, es) || !aligned(a->branch, es) || !aligned(a->h_out, es) || !aligned(a->y_out, es) ||
        !aligned(a->post_weight, ws) || !aligned(a->weight, ws) || !aligned(a->gate, ms) || !aligned(a->scale, ms) ||
        !aligned(a->shift, ms) || !aligned(a->mod_index, 4))
      fail(NKV_ERR_ARGUMENT, "tensors must be aligned to their types");
    if (a->x_stride < 0 || a->branch_stride < 0 || a->h_stride < 0 || a->y_stride < 0)
      fail(NKV_ERR_ARGUMENT, "row strides must not be negative");
    if (a->tokens > 1 && ((a->branch && a->h_stride < a->dim) || (a->norm && a->y_stride < a->dim)))
      fail(NKV_ERR_ARGUMENT, "output rows must not overlap");
    nkv::ResidualNormParams p{};
    p.x = a->x, p.branch = a->branch;
    p.h_out = a->branch ? a->h_out : nullptr, p.y_out = a->norm ? a->y_out : nullptr;
    p.x_stride = a->x_stride, p.branch_stride = a->branch ? a->branch_stride : 0;
    p.h_stride = p.h_out ? a->h_stride : 0, p.y_stride = p.y_out ? a->y_stride : 0;
    p.post_weight = a->post_weight, p.weight = a->weight;
    p.gate = a->gate, p.scale = a->scale, p.shift = a->shift;
    p.mod_index = mods ? a->mod_index : nullptr;
    p.mod_rows = a->mod_rows;
    p.tokens = a->tokens, p.dim = a->dim;
    p.weight_dtype = a->weight_dtype, p.mod_dtype = a->mod_dtype;
    p.post = a->post, p.norm = a->norm;
    p.eps = a->eps;
    nkv::check_cuda(nkv::launch_residual_norm(p, a->dtype, static_cast<cudaStream_t>(stream)), "residual norm launch");
  });
}

int nkv_attend_schedule(const uint64_t* q_lens, const uint64_t* k_lens, uint64_t n, int32_t heads, int32_t kv_heads,
                        int32_t causal, uint64_t block, int32_t sms, int64_t* out, uint64_t cap, uint64_t* n_items) {
  return nkv::guarded_call([&] {
    need(n_items, "count output");
    if (sms < 1) fail(NKV_ERR_ARGUMENT, "sms must be positive");
    const Lens l = check_lens(q_lens, k_lens, n, heads, kv_heads, block);
    const nkv::PackedSchedule s = nkv::packed_schedule(l.q, l.k, heads, kv_heads, causal != 0, int64_t(block), sms);
    *n_items = s.items.size();
    if (!out) return;
    for (size_t i = 0; i < s.items.size() && i < cap; ++i) {
      const nkv::PackedItem& t = s.items[i];
      const int64_t v[8] = {t.q_start, t.k_start, t.row0, t.rows, t.kvh, t.t_lo, t.t_hi, t.part_row};
      std::copy(v, v + 8, out + 8 * i);
    }
  });
}

int nkv_attend_plan_create(const uint64_t* q_lens, const uint64_t* k_lens, uint64_t n, int32_t heads,
                           int32_t kv_heads, int32_t head_dim, int32_t causal, uint64_t block, int32_t device,
                           nkv_attend_plan** out) {
  return nkv::guarded_call([&] {
    need(out, "output handle");
    *out = nullptr;
    const Lens l = check_lens(q_lens, k_lens, n, heads, kv_heads, block);
    if (head_dim < 8 || head_dim > 128 || head_dim % 8)
      fail(NKV_ERR_GEOMETRY, "packed attention needs head_dim a multiple of 8, 8 to 128");
    int count = 0;
    if (cudaGetDeviceCount(&count) != cudaSuccess || count == 0) {
      cudaGetLastError();
      fail(NKV_ERR_CUDA, "no CUDA device: packed attention has no CPU fallback");
    }
    if (device < 0 || device >= count) fail(NKV_ERR_ARGUMENT, "device out of range");
    OnDevice on(device);
    int sms = 0;
    nkv::check_cuda(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, device), "cudaDeviceGetAttribute");
    const nkv::PackedSchedule s = nkv::packed_schedule(l.q, l.k, heads, kv_heads, causal != 0, int64_t(block), sms);
    auto p = std::make_unique<nkv_attend_plan>();
    p->device = device;
    p->H = heads, p->kv_heads = kv_heads, p->D = head_dim;
    p->causal = causal ? 1 : 0;
    p->block = int64_t(block);
    p->q_tokens = l.q_tokens, p->k_tokens = l.k_tokens;
    p->part_rows = uint64_t(s.part_rows);
    p->n_items = int32_t(s.items.size()), p->n_units = int32_t(s.units.size());
    p->n_ctas = int32_t(s.cta_begin.size()) - 1;
    p->max_unit_rows = s.max_unit_rows;
    DuringCapture relaxed;
    auto after = [](size_t at, size_t bytes) { return (at + bytes + 63) / 64 * 64; };
    p->ctas_off = after(p->items_off, s.items.size() * sizeof(nkv::PackedItem));
    p->first_off = after(p->ctas_off, s.cta_begin.size() * sizeof(int32_t));
    p->units_off = after(p->first_off, size_t(p->n_ctas) * sizeof(nkv::PackedItem));
    std::vector<unsigned char> host(after(p->units_off, s.units.size() * sizeof(nkv::PackedUnit)), 0);
    std::copy_n(reinterpret_cast<const unsigned char*>(s.items.data()), s.items.size() * sizeof(nkv::PackedItem),
                host.data() + p->items_off);
    std::copy_n(reinterpret_cast<const unsigned char*>(s.cta_begin.data()), s.cta_begin.size() * sizeof(int32_t),
                host.data() + p->ctas_off);
    for (int32_t c = 0; c < p->n_ctas; ++c)
      std::copy_n(reinterpret_cast<const unsigned char*>(&s.items[size_t(s.cta_begin[size_t(c)])]),
                  sizeof(nkv::PackedItem), host.data() + p->first_off + size_t(c) * sizeof(nkv::PackedItem));
    std::copy_n(reinterpret_cast<const unsigned char*>(s.units.data()), s.units.size() * sizeof(nkv::PackedUnit),
                host.data() + p->units_off);
    cudaError_t e = cudaMalloc(reinterpret_cast<void**>(&p->table), host.size());
    if (e == cudaSuccess) e = cudaMemcpy(p->table, host.data(), host.size(), cudaMemcpyHostToDevice);
    // a copy from pageable memory may return before it has landed, and the
    // plan's calls come on streams that do not wait for the default stream
    if (e == cudaSuccess) e = cudaStreamSynchronize(nullptr);
    if (e != cudaSuccess) {
      if (p->table) cudaFree(p->table);
      nkv::check_cuda(e, "attention plan upload");
    }
    *out = p.release();
  });
}

int nkv_attend_plan_destroy(nkv_attend_plan* plan) {
  return nkv::guarded_call([&] {
    if (!plan) return;
    {
      OnDevice on(plan->device);
      DuringCapture relaxed;
      if (plan->table) nkv::check_cuda(cudaFree(plan->table), "cudaFree");  // waits for work that reads the table
    }
    delete plan;
  });
}

int nkv_attend_plan_get_info(const nkv_attend_plan* plan, nkv_attend_plan_info* out) {
  return nkv::guarded_call([&] {
    need(plan, "plan");
    need(out, "output");
    out->q_tokens = plan->q_tokens;
    out->k_tokens = plan->k_tokens;
    out->items = uint64_t(plan->n_items);
    out->split_units = uint64_t(plan->n_units);
    out->workspace_bytes = plan->workspace();
  });
}

int nkv_attend_plan_status(const nkv_attend_plan* plan, uint32_t* status) {
  return nkv::guarded_call([&] {
    need(plan, "plan");
    need(status, "status output");
    OnDevice on(plan->device);
    nkv::check_cuda(cudaDeviceSynchronize(), "cudaDeviceSynchronize");
    nkv::check_cuda(cudaMemcpy(status, plan->table, sizeof(uint32_t), cudaMemcpyDeviceToHost), "cudaMemcpy");
  });
}

int nkv_attend_plan_set_status(nkv_attend_plan* plan, uint32_t status) {
  return nkv::guarded_call([&] {
    need(plan, "plan");
    OnDevice on(plan->device);
    nkv::check_cuda(cudaDeviceSynchronize(), "cudaDeviceSynchronize");
    nkv::check_cuda(cudaMemcpy(plan->table, &status, sizeof(uint32_t), cudaMemcpyHostToDevice), "cudaMemcpy");
    nkv::check_cuda(cudaStreamSynchronize(nullptr), "cudaStreamSynchronize");  // as in nkv_attend_plan_create
  });
}

int nkv_attend_packed(const nkv_attend_plan* plan, const nkv_attend_args* a, void* stream) {
  return nkv::guarded_call([&] {
    need(plan, "plan");
    need(a, "args");
    if (a->dtype != NKV_BF16 && a->dtype != NKV_F16)
      fail(NKV_ERR_GEOMETRY, "packed attention needs bf16 or f16 queries, keys and values");
    if (a->out_dtype != a->dtype && a->out_dtype != NKV_F32)
      fail(NKV_ERR_GEOMETRY, "the output must be f32 or of the queries' type");
    const float scale_log2 = a->scale * 1.4426950408889634f;
    if (!(scale_log2 > 0.0f) || !std::isfinite(scale_log2))
      fail(NKV_ERR_ARGUMENT, "scale must be finite and positive");
    if (a->q_rows < plan->q_tokens || a->k_rows < plan->k_tokens)
      fail(NKV_ERR_GEOMETRY, "q has " + std::to_string(a->q_rows) + " rows and k / v " + std::to_string(a->k_rows) +
                                 ", the plan " + std::to_string(plan->q_tokens) + " and " +
                                 std::to_string(plan->k_tokens));
    if (!a->hist_out != !a->hist_lse) fail(NKV_ERR_ARGUMENT, "hist_out and hist_lse go together");
    int current = 0;
    nkv::check_cuda(cudaGetDevice(&current), "cudaGetDevice");
    if (current != plan->device) fail(NKV_ERR_ARGUMENT, "the plan belongs to another device");
    if (plan->n_items == 0) return;
    need(a->q, "q"), need(a->out, "out"), need(a->lse, "lse");
    if (plan->k_tokens) need(a->k, "k"), need(a->v, "v");
    check_strides(a->q, a->q_token_stride, a->q_head_stride, int64_t(plan->q_tokens), plan->H, "q");
    if (plan->k_tokens) {
      check_strides(a->k, a->k_token_stride, a->k_head_stride, int64_t(plan->k_tokens), plan->kv_heads, "k");
      check_strides(a->v, a->v_token_stride, a->v_head_stride, int64_t(plan->k_tokens), plan->kv_heads, "v");
    }
    if (!aligned(a->out, 16) || !aligned(a->hist_out, 16)) fail(NKV_ERR_ARGUMENT, "out and hist_out must be 16-byte aligned");
    if (!aligned(a->lse, 4) || !aligned(a->hist_lse, 4)) fail(NKV_ERR_ARGUMENT, "lse must be 4-byte aligned");
    if (plan->workspace()) {
      need(a->workspace, "workspace");
      if (a->workspace_bytes < plan->workspace()) fail(NKV_ERR_ARGUMENT, "workspace too small");
      if (!aligned(a->workspace, 16)) fail(NKV_ERR_ARGUMENT, "workspace must be 16-byte aligned");
    }
    nkv::PackedArgs p{};
    p.items = reinterpret_cast<const nkv::PackedItem*>(plan->table + plan->items_off);
    p.units = reinterpret_cast<const nkv::PackedUnit*>(plan->table + plan->units_off);
    p.first = reinterpret_cast<const nkv::PackedItem*>(plan->table + plan->first_off);
    p.cta_begin = reinterpret_cast<const int32_t*>(plan->table + plan->ctas_off);
    p.n_ctas = plan->n_ctas, p.n_units = plan->n_units, p.max_unit_rows = plan->max_unit_rows;
    p.H = plan->H, p.G = plan->H / plan->kv_heads, p.D = plan->D;
    p.causal = plan->causal;
    p.block = plan->block;
    p.q = static_cast<const uint16_t*>(a->q);
    p.q_token = a->q_token_stride, p.q_head = a->q_head_stride;
    p.v = static_cast<const uint16_t*>(a->v);
    p.v_token = a->v_token_stride, p.v_head = a->v_head_stride;
    p.out = a->out;
    p.out_f32 = a->out_dtype == NKV_F32 ? 1 : 0;
    p.lse = a->lse;
    p.lse_head = int64_t(a->q_rows);
    p.hist_o = a->hist_out;
    p.hist_lse = a->hist_lse;
    p.hist_lse_head = int64_t(a->q_rows);
    p.scale_log2 = scale_log2;
    p.part_o = static_cast<float*>(a->workspace);
    p.part_ml = p.part_o ? p.part_o + plan->part_rows * uint64_t(plan->D) : nullptr;
    p.status = reinterpret_cast<uint32_t*>(plan->table);
    cudaError_t e = cudaSuccess;
    if (!nkv::launch_attend_packed(p, a->dtype, a->k, int64_t(plan->q_tokens), int64_t(plan->k_tokens),
                                   a->k_token_stride, a->k_head_stride, static_cast<cudaStream_t>(stream), &e))
      fail(NKV_ERR_CUDA, "the driver refused the layout of q, k or v");
    nkv::check_cuda(e, "packed attention launch");
  });
}

}  // extern "C"
