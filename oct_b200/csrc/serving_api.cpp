// serving_api.cpp -- the token-by-token serving entry points of the C ABI: head
// norm + rotation, the 4-bit cache's store and load, the attention over it.
// Each validates on the host what the host can see and enqueues; lengths, row
// ranges and page numbers on the device are checked by the kernels.
#include <cmath>

#include "runtime.h"
#include "serving.h"

using namespace oct::rt;

namespace {

int fail(int* detail, int code) {
  if (detail) *detail = code;
  return PROM_ERROR;
}

constexpr uint64_t kMaxStride = 1ull << 32;  // elements; times 2^31 rows it stays below 2^64

// Of the attention's scale: times 2^24 and log2(e), which the kernel makes of it, it stays finite.
constexpr float kMaxScale = 0x1p100f;

bool aligned16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

// Elements of `dtype` in 16 bytes; 0 for an unknown type.
uint32_t vector_elements(uint32_t dtype) {
  return dtype == OCT_B200_F32 ? 4u : (dtype == OCT_B200_BF16 || dtype == OCT_B200_F16 ? 8u : 0u);
}

// The stride of a dimension of one is not used.
uint64_t used(uint64_t stride, uint64_t extent) { return extent > 1 ? stride : 0; }

// A [tokens][heads][dim] tensor.  Rows of an output must not share elements.
int check_rows(const void* p, uint64_t tokens, uint32_t heads, uint32_t dim, uint64_t token_stride,
               uint64_t head_stride, uint32_t vec, bool output) {
  if (p == nullptr) return OCT_B200_DETAIL_INVALID_ARGUMENT;
  token_stride = used(token_stride, tokens);
  head_stride = used(head_stride, heads);
  if (!aligned16(p) || token_stride % vec != 0 || head_stride % vec != 0) return OCT_B200_DETAIL_UNALIGNED;
  if (token_stride > kMaxStride || head_stride > kMaxStride) return OCT_B200_DETAIL_INVALID_ARGUMENT;
  // one of an output's two strides steps over all that the other covers
  const bool by_token = tokens <= 1 || token_stride >= (heads - 1) * head_stride + dim;
  const bool by_head = heads <= 1 || head_stride >= (tokens - 1) * token_stride + dim;
  const bool rows_apart = (heads <= 1 || head_stride >= dim) && (tokens <= 1 || token_stride >= dim);
  if (output && !(rows_apart && (by_token || by_head))) return OCT_B200_DETAIL_INVALID_ARGUMENT;
  return 0;
}

// The call's GPU is the handle's: with several GPUs its kernels are launched there,
// whichever is current, and a pointer of another GPU is refused.
class OnDevice {
 public:
  explicit OnDevice(Runtime* rt) {
    static const int count = [] {
      int n = 0;
      return cudaGetDeviceCount(&n) == cudaSuccess ? n : 1;
    }();
    several_ = count > 1;
    if (several_ && cudaGetDevice(&before_) == cudaSuccess && before_ != rt->device)
      restore_ = cudaSetDevice(rt->device) == cudaSuccess;
    device_ = rt->device;
  }
  ~OnDevice() {
    if (restore_) cudaSetDevice(before_);
  }
  bool holds(const void* p) const {
    if (!several_ || p == nullptr) return true;
    cudaPointerAttributes at{};
    if (cudaPointerGetAttributes(&at, p) != cudaSuccess) {
      (void)cudaGetLastError();
      return false;
    }
    return at.type != cudaMemoryTypeDevice || at.device == device_;
  }

 private:
  int before_ = 0, device_ = 0;
  bool several_ = false, restore_ = false;
};

// Cache and batch of a call with `tokens` rows.
int check_cache(const OctB200Kv4Cache* c) {
  if (c == nullptr || c->struct_size < sizeof(OctB200Kv4Cache) || c->data == nullptr || c->pages == 0 ||
      c->kv_heads == 0 || c->reserved != 0)
    return OCT_B200_DETAIL_INVALID_ARGUMENT;
  if (c->page_size == 0 || c->page_size % oct::kKv4Tile != 0 || c->page_size > 65536u || c->kv_heads > 4096u ||
      !oct::kv4_attention_supported(c->head_dim))
    return OCT_B200_DETAIL_UNSUPPORTED_SHAPE;
  // tiles are counted in 32 bits (5 TB of cache)
  if (static_cast<uint64_t>(c->pages) * c->kv_heads * (c->page_size / oct::kKv4Tile) > 0xfffffff0ull)
    return OCT_B200_DETAIL_UNSUPPORTED_SHAPE;
  return aligned16(c->data) ? 0 : OCT_B200_DETAIL_UNALIGNED;
}
int check_batch(const OctB200Kv4Cache* c, const OctB200Kv4Batch* b, uint64_t tokens) {
  if (b == nullptr || b->struct_size < sizeof(OctB200Kv4Batch) || b->reserved != 0)
    return OCT_B200_DETAIL_INVALID_ARGUMENT;
  if (b->batch == 0) return 0;
  if (b->kv_lens == nullptr || (b->page_table == nullptr && b->page_table_width > 0) ||
      (b->batch > 1 && b->page_table_stride < b->page_table_width) ||
      b->max_kv_len > static_cast<uint64_t>(b->page_table_width) * c->page_size ||
      (b->cu_tokens == nullptr && (tokens != b->batch || b->max_tokens != 1)))
    return OCT_B200_DETAIL_INVALID_ARGUMENT;
  for (const int32_t* p : {b->page_table, b->kv_lens, b->cu_tokens})
    if (reinterpret_cast<uintptr_t>(p) % 4 != 0) return OCT_B200_DETAIL_UNALIGNED;
  if (b->batch > 65535u || b->max_kv_len > 0x7fff0000u || tokens > 0x7fffffffull || b->max_tokens > 0x7fffffffu ||
      static_cast<uint64_t>(b->max_tokens) * c->kv_heads * 2 > 0x7fffffffull)
    return OCT_B200_DETAIL_UNSUPPORTED_SHAPE;
  return 0;
}

oct::Kv4View view_of(const OctB200Kv4Cache* c, const OctB200Kv4Batch* b, uint64_t tokens, unsigned long long* skipped) {
  oct::Kv4View v;
  v.data = static_cast<uint8_t*>(c->data);
  v.pages = c->pages;
  v.page_tiles = c->page_size / oct::kKv4Tile;
  v.kv_heads = c->kv_heads;
  v.dim = c->head_dim;
  v.batch = b->batch;
  v.table = b->page_table;
  v.table_stride = b->page_table_stride;
  v.kv_lens = b->kv_lens;
  v.cu_tokens = b->cu_tokens;
  v.max_tokens = b->max_tokens;
  v.max_kv_len = b->max_kv_len;
  v.tokens = tokens;
  v.skipped = skipped;
  return v;
}

int run_rows(void* handle, const OctB200Kv4Cache* cache, const OctB200Kv4Batch* batch, const OctB200Kv4Rows* rows,
             bool store, void* stream, int* out_detail_code) {
  try {
    if (out_detail_code) *out_detail_code = 0;
    Runtime* rt = lookup(handle);
    if (rt == nullptr) return PROM_INVALID_HANDLE;
    if (rows == nullptr || rows->struct_size < sizeof(OctB200Kv4Rows))
      return fail(out_detail_code, OCT_B200_DETAIL_INVALID_ARGUMENT);
    const uint32_t vec = vector_elements(rows->dtype);
    int bad = vec == 0 ? OCT_B200_DETAIL_INVALID_ARGUMENT : check_cache(cache);
    if (bad == 0) bad = check_batch(cache, batch, rows->tokens);
    const bool any = bad == 0 && rows->tokens > 0 && batch->batch > 0 && batch->max_tokens > 0;
    if (any) {
      bad = check_rows(rows->k, rows->tokens, cache->kv_heads, cache->head_dim, rows->k_token_stride,
                       rows->k_head_stride, vec, !store);
      if (bad == 0)
        bad = check_rows(rows->v, rows->tokens, cache->kv_heads, cache->head_dim, rows->v_token_stride,
                         rows->v_head_stride, vec, !store);
    }
    if (any && bad == 0 && !store && rows->k == rows->v) bad = OCT_B200_DETAIL_INVALID_ARGUMENT;
    if (bad != 0) return fail(out_detail_code, bad);
    if (!rt->available) return fail(out_detail_code, PROM_DETAIL_CAPABILITY_MISMATCH);
    if (!any) return PROM_OK;
    std::lock_guard<std::mutex> lock(rt->mu);
    const OnDevice on(rt);
    for (const void* p : {static_cast<const void*>(cache->data), static_cast<const void*>(batch->page_table),
                          static_cast<const void*>(batch->kv_lens), static_cast<const void*>(batch->cu_tokens),
                          static_cast<const void*>(rows->k), static_cast<const void*>(rows->v)})
      if (!on.holds(p)) return fail(out_detail_code, OCT_B200_DETAIL_INVALID_ARGUMENT);
    oct::Kv4RowArgs a;
    a.view = view_of(cache, batch, rows->tokens, rt->skipped_word());
    a.type = static_cast<oct::ElementType>(rows->dtype);
    a.rows[0] = rows->k;
    a.rows[1] = rows->v;
    a.token_stride[0] = used(rows->k_token_stride, rows->tokens);
    a.token_stride[1] = used(rows->v_token_stride, rows->tokens);
    a.head_stride[0] = used(rows->k_head_stride, cache->kv_heads);
    a.head_stride[1] = used(rows->v_head_stride, cache->kv_heads);
    cudaStream_t s = static_cast<cudaStream_t>(stream);  // NULL is the CUDA default stream
    if ((store ? oct::kv4_store(a, s) : oct::kv4_load(a, s)) != cudaSuccess)
      return fail(out_detail_code, OCT_B200_DETAIL_CUDA_ERROR);
    return PROM_OK;
  } catch (...) {
    return PROM_INTERNAL_ERROR;
  }
}

// Everything of an attention call but its pointers; the plan on success.
int check_attention(const OctB200Kv4Cache* c, const OctB200Kv4Batch* b, const OctB200Kv4AttentionRequest* r,
                    oct::Kv4Plan* plan) {
  int bad = check_cache(c);
  if (bad != 0) return bad;
  if (r == nullptr || r->struct_size < sizeof(OctB200Kv4AttentionRequest) || vector_elements(r->dtype) == 0 ||
      r->q_heads == 0 || r->q_heads % c->kv_heads != 0 || !(std::fabs(r->scale) < kMaxScale) ||
      (r->window != 0 && r->causal == 0))
    return OCT_B200_DETAIL_INVALID_ARGUMENT;
  bad = check_batch(c, b, r->tokens);
  if (bad != 0) return bad;
  if (b->batch == 0 || b->max_tokens == 0 || r->tokens == 0) {
    *plan = oct::Kv4Plan{};
    return 0;
  }
  if (r->q_heads > 65535u || static_cast<uint64_t>(b->max_tokens) * r->q_heads > 0x7fffffffull)
    return OCT_B200_DETAIL_UNSUPPORTED_SHAPE;
  *plan = oct::kv4_attention_plan(c->head_dim, c->kv_heads, r->q_heads, b->batch, b->max_tokens, b->max_kv_len, r->window,
                                  static_cast<oct::ElementType>(r->dtype));
  // work is counted in 32 bits, in units of 64 or 128 keys of an item
  return plan->row_tiles * b->batch > 0x3fffffffull || plan->run > 0x3fffffffull ? OCT_B200_DETAIL_UNSUPPORTED_SHAPE : 0;
}

}  // namespace

extern "C" {

int oct_b200_qk_norm_rope_device(void* handle, const OctB200QkNormRopeRequest* r, void* stream, int* out_detail_code) {
  try {
    if (out_detail_code) *out_detail_code = 0;
    Runtime* rt = lookup(handle);
    if (rt == nullptr) return PROM_INVALID_HANDLE;
    if (r == nullptr || r->struct_size < sizeof(OctB200QkNormRopeRequest))
      return fail(out_detail_code, OCT_B200_DETAIL_INVALID_ARGUMENT);
    const uint32_t vec = vector_elements(r->dtype);
    uint64_t pairs = 0;
    for (uint32_t i = 0; i < r->axes && i < oct::kRopeMaxAxes; ++i) pairs += r->axis_pairs[i];
    if (vec == 0 || r->axes == 0 || r->axes > oct::kRopeMaxAxes || 2 * pairs != r->rotary_dim ||
        r->rotary_dim > r->head_dim || !std::isfinite(r->eps) || r->eps <= 0.f)
      return fail(out_detail_code, OCT_B200_DETAIL_INVALID_ARGUMENT);
    if (r->head_dim == 0 || r->head_dim % 16 != 0 || r->head_dim > oct::kRopeMaxHeadDim || r->rotary_dim == 0 ||
        r->rotary_dim % 16 != 0 || r->q_heads > 65535u || r->k_heads > 65535u || r->tokens > 0x7fffffffull)
      return fail(out_detail_code, OCT_B200_DETAIL_UNSUPPORTED_SHAPE);
    const bool any = r->tokens > 0 && (r->q_heads > 0 || r->k_heads > 0);
    oct::QkNormRopeArgs a;
    if (any) {
      if (r->positions == nullptr || r->frequencies == nullptr ||
          (r->tokens > 1 && r->position_stride < r->axes))
        return fail(out_detail_code, OCT_B200_DETAIL_INVALID_ARGUMENT);
      if (reinterpret_cast<uintptr_t>(r->positions) % 4 != 0 || reinterpret_cast<uintptr_t>(r->frequencies) % 8 != 0 ||
          !aligned16(r->q_weight) || !aligned16(r->k_weight))
        return fail(out_detail_code, OCT_B200_DETAIL_UNALIGNED);
      a.heads[0] = r->q_heads, a.heads[1] = r->k_heads;
      a.in[0] = r->q, a.in[1] = r->k;
      a.out[0] = r->q_out, a.out[1] = r->k_out;
      a.in_token[0] = used(r->q_token_stride, r->tokens), a.in_token[1] = used(r->k_token_stride, r->tokens);
      a.in_head[0] = used(r->q_head_stride, r->q_heads), a.in_head[1] = used(r->k_head_stride, r->k_heads);
      a.out_token[0] = used(r->q_out_token_stride, r->tokens), a.out_token[1] = used(r->k_out_token_stride, r->tokens);
      a.out_head[0] = used(r->q_out_head_stride, r->q_heads), a.out_head[1] = used(r->k_out_head_stride, r->k_heads);
      a.weight[0] = r->q_weight, a.weight[1] = r->k_weight;
      for (int i = 0; i < 2; ++i) {
        if (a.heads[i] == 0) continue;
        int bad = check_rows(a.in[i], r->tokens, a.heads[i], r->head_dim, a.in_token[i], a.in_head[i], vec, false);
        if (bad == 0)
          bad = check_rows(a.out[i], r->tokens, a.heads[i], r->head_dim, a.out_token[i], a.out_head[i], vec, true);
        // in place means row for row
        if (bad == 0 && a.in[i] == a.out[i] && (a.in_token[i] != a.out_token[i] || a.in_head[i] != a.out_head[i]))
          bad = OCT_B200_DETAIL_INVALID_ARGUMENT;
        if (bad == 0 && a.heads[0] > 0 && a.heads[1] > 0 && a.out[0] == a.out[1]) bad = OCT_B200_DETAIL_INVALID_ARGUMENT;
        if (bad != 0) return fail(out_detail_code, bad);
      }
    }
    if (!rt->available) return fail(out_detail_code, PROM_DETAIL_CAPABILITY_MISMATCH);
    if (!any) return PROM_OK;
    std::lock_guard<std::mutex> lock(rt->mu);
    const OnDevice on(rt);
    for (const void* p : {a.heads[0] ? a.in[0] : nullptr, a.heads[1] ? a.in[1] : nullptr,
                          static_cast<const void*>(a.heads[0] ? a.out[0] : nullptr),
                          static_cast<const void*>(a.heads[1] ? a.out[1] : nullptr),
                          static_cast<const void*>(r->positions), static_cast<const void*>(r->frequencies),
                          static_cast<const void*>(r->q_weight), static_cast<const void*>(r->k_weight)})
      if (!on.holds(p)) return fail(out_detail_code, OCT_B200_DETAIL_INVALID_ARGUMENT);
    a.type = static_cast<oct::ElementType>(r->dtype);
    a.tokens = r->tokens;
    a.dim = r->head_dim;
    a.rotary = r->rotary_dim;
    a.interleaved = r->interleaved != 0;
    a.normalize = r->normalize != 0;
    a.eps = r->eps;
    a.axes = r->axes;
    for (uint32_t i = 0; i < r->axes; ++i) a.axis_pairs[i] = r->axis_pairs[i];
    a.positions = r->positions;
    a.position_stride = r->position_stride;
    a.frequencies = r->frequencies;
    if (!a.normalize) a.weight[0] = a.weight[1] = nullptr;
    if (oct::qk_norm_rope(a, static_cast<cudaStream_t>(stream)) != cudaSuccess)
      return fail(out_detail_code, OCT_B200_DETAIL_CUDA_ERROR);
    return PROM_OK;
  } catch (...) {
    return PROM_INTERNAL_ERROR;
  }
}

uint64_t oct_b200_kv4_tile_bytes(uint32_t head_dim) {
  return oct::kv4_attention_supported(head_dim) ? oct::kv4_tile_bytes(head_dim) : 0;
}

int oct_b200_kv4_store_device(void* handle, const OctB200Kv4Cache* cache, const OctB200Kv4Batch* batch,
                              const OctB200Kv4Rows* rows, void* stream, int* out_detail_code) {
  return run_rows(handle, cache, batch, rows, true, stream, out_detail_code);
}

int oct_b200_kv4_load_device(void* handle, const OctB200Kv4Cache* cache, const OctB200Kv4Batch* batch,
                             const OctB200Kv4Rows* rows, void* stream, int* out_detail_code) {
  return run_rows(handle, cache, batch, rows, false, stream, out_detail_code);
}

int oct_b200_kv4_attention_workspace_bytes(const OctB200Kv4Cache* cache, const OctB200Kv4Batch* batch,
                                           const OctB200Kv4AttentionRequest* request, uint64_t* out_bytes,
                                           int* out_detail_code) {
  try {
    if (out_detail_code) *out_detail_code = 0;
    if (out_bytes == nullptr) return fail(out_detail_code, OCT_B200_DETAIL_INVALID_ARGUMENT);
    *out_bytes = 0;
    oct::Kv4Plan plan;
    const int bad = check_attention(cache, batch, request, &plan);
    if (bad != 0) return fail(out_detail_code, bad);
    *out_bytes = plan.workspace;
    return PROM_OK;
  } catch (...) {
    return PROM_INTERNAL_ERROR;
  }
}

int oct_b200_kv4_attention_device(void* handle, const OctB200Kv4Cache* cache, const OctB200Kv4Batch* batch,
                                  const OctB200Kv4AttentionRequest* r, void* stream, int* out_detail_code) {
  try {
    if (out_detail_code) *out_detail_code = 0;
    Runtime* rt = lookup(handle);
    if (rt == nullptr) return PROM_INVALID_HANDLE;
    oct::Kv4Plan plan;
    int bad = check_attention(cache, batch, r, &plan);
    if (bad != 0) return fail(out_detail_code, bad);
    const bool any = r->tokens > 0 && batch->batch > 0 && batch->max_tokens > 0;
    if (any) {
      const uint32_t vec = vector_elements(r->dtype);
      bad = check_rows(r->q, r->tokens, r->q_heads, cache->head_dim, r->q_token_stride, r->q_head_stride, vec, false);
      if (bad == 0)
        bad = check_rows(r->out, r->tokens, r->q_heads, cache->head_dim, r->out_token_stride, r->out_head_stride, vec,
                         true);
      // over the queries means row for row
      if (bad == 0 && r->q == r->out &&
          (used(r->q_token_stride, r->tokens) != used(r->out_token_stride, r->tokens) ||
           used(r->q_head_stride, r->q_heads) != used(r->out_head_stride, r->q_heads)))
        bad = OCT_B200_DETAIL_INVALID_ARGUMENT;
      if (bad == 0 && r->lse != nullptr && reinterpret_cast<uintptr_t>(r->lse) % 4 != 0) bad = OCT_B200_DETAIL_UNALIGNED;
      if (bad == 0 && plan.workspace > 0) {
        if (r->workspace == nullptr || r->workspace_bytes < plan.workspace)
          bad = OCT_B200_DETAIL_KV4_WORKSPACE;
        else if (!aligned16(r->workspace))
          bad = OCT_B200_DETAIL_UNALIGNED;
      }
      if (bad != 0) return fail(out_detail_code, bad);
    }
    if (!rt->available) return fail(out_detail_code, PROM_DETAIL_CAPABILITY_MISMATCH);
    if (!any) return PROM_OK;
    std::lock_guard<std::mutex> lock(rt->mu);
    const OnDevice on(rt);
    for (const void* p : {static_cast<const void*>(cache->data), static_cast<const void*>(batch->page_table),
                          static_cast<const void*>(batch->kv_lens), static_cast<const void*>(batch->cu_tokens), r->q,
                          static_cast<const void*>(r->out), static_cast<const void*>(r->lse),
                          static_cast<const void*>(plan.workspace > 0 ? r->workspace : nullptr)})
      if (!on.holds(p)) return fail(out_detail_code, OCT_B200_DETAIL_INVALID_ARGUMENT);
    oct::Kv4AttnArgs a;
    a.view = view_of(cache, batch, r->tokens, rt->skipped_word());
    a.type = static_cast<oct::ElementType>(r->dtype);
    a.heads = r->q_heads;
    a.q = r->q;
    a.out = r->out;
    a.q_token = used(r->q_token_stride, r->tokens);
    a.q_head = used(r->q_head_stride, r->q_heads);
    a.out_token = used(r->out_token_stride, r->tokens);
    a.out_head = used(r->out_head_stride, r->q_heads);
    a.lse = r->lse;
    a.scale = r->scale;
    a.causal = r->causal != 0;
    a.window = r->window;
    a.workspace = r->workspace;
    if (oct::kv4_attention(a, plan, static_cast<cudaStream_t>(stream)) != cudaSuccess)
      return fail(out_detail_code, OCT_B200_DETAIL_CUDA_ERROR);
    return PROM_OK;
  } catch (...) {
    return PROM_INTERNAL_ERROR;
  }
}

}  // extern "C"
