// serving.h -- host-side launchers of the token-by-token serving kernels:
// head norm + position rotation (qk_norm_rope.cu), the paged cache that holds
// keys and values in 4 bits (kv4_cache.cu) and the attention over it
// (kv4_attention.cu).  The entry points are in serving_api.cpp.
#pragma once

#include <cstdint>
#include <cuda_runtime.h>

namespace oct {

enum ElementType : uint32_t { kF32 = 0, kBf16 = 1, kF16 = 2 };

// ---------------------------------------------------------------- head norm + rotation
constexpr uint32_t kRopeMaxAxes = 4;
constexpr uint32_t kRopeMaxHeadDim = 512;
struct QkNormRopeArgs {
  ElementType type = kF32;
  uint64_t tokens = 0;
  uint32_t heads[2] = {0, 0};  // query heads, key heads (0: that input is absent)
  uint32_t dim = 0, rotary = 0;
  bool interleaved = false, normalize = false;
  float eps = 0.f;
  uint32_t axes = 0;
  uint32_t axis_pairs[kRopeMaxAxes] = {};
  const void* in[2] = {};
  void* out[2] = {};
  uint64_t in_token[2] = {}, in_head[2] = {}, out_token[2] = {}, out_head[2] = {};  // element strides
  const float* weight[2] = {};
  const int32_t* positions = nullptr;
  uint64_t position_stride = 0;
  const double* frequencies = nullptr;
};
cudaError_t qk_norm_rope(const QkNormRopeArgs& a, cudaStream_t stream);

// ---------------------------------------------------------------- 4-bit paged cache
// data: [pages][kv_heads][page_size / 16] tiles of 16 tokens; a tile is
//   key codes [16][dim/2] | key (s, z) [16][dim/32] | value codes | value (s, z).
constexpr uint32_t kKv4Tile = 16;
constexpr uint32_t kKv4Group = 32;
inline constexpr uint64_t kv4_tile_bytes(uint32_t dim) { return 2ull * kKv4Tile * (dim / 2 + dim / kKv4Group * 4); }

struct Kv4View {
  uint8_t* data = nullptr;
  uint32_t pages = 0, page_tiles = 0, kv_heads = 0, dim = 0;
  // sequences
  uint32_t batch = 0;
  const int32_t* table = nullptr;
  uint64_t table_stride = 0;
  const int32_t* kv_lens = nullptr;
  const int32_t* cu_tokens = nullptr;  // null: one token per sequence
  uint32_t max_tokens = 0, max_kv_len = 0;
  uint64_t tokens = 0;  // rows of the call's own tensors
  unsigned long long* skipped = nullptr;  // counts the device-side indices that are out of range
};

struct Kv4RowArgs {
  Kv4View view;
  ElementType type = kF32;
  void* rows[2] = {};  // keys, values: [tokens][kv_heads][dim]
  uint64_t token_stride[2] = {}, head_stride[2] = {};
};
cudaError_t kv4_store(const Kv4RowArgs& a, cudaStream_t stream);
cudaError_t kv4_load(const Kv4RowArgs& a, cudaStream_t stream);

// ---------------------------------------------------------------- attention over it
bool kv4_attention_supported(uint32_t dim);
// How a call is laid out over thread blocks, from sizes the host knows.
struct Kv4Plan {
  uint32_t row_tile = 0;   // query rows (token, head of a key head's share) of one item
  uint64_t row_tiles = 0;  // items per (sequence, key head)
  uint32_t blocks = 0;
  uint32_t cluster = 0;    // blocks per cluster where each cluster has one item; 0: equal runs of all items
  uint64_t run = 0;        // bound of the call's work in the kernel's units
  uint64_t workspace = 0;  // bytes; 0 when no item can be split
};
Kv4Plan kv4_attention_plan(uint32_t dim, uint32_t kv_heads, uint32_t heads, uint32_t batch, uint32_t max_tokens,
                           uint32_t max_kv_len, uint32_t window, ElementType type);
// The blocks of a cluster to launch where `wanted` (a power of two) are planned: halved until `places`, asked once
// per size, says that the device has room for one such cluster.  Every size gives the same parts of the work to
// some block, so what a smaller one costs is time.
template <typename Places>
uint32_t kv4_cluster_to_launch(uint32_t wanted, Places places) {
  while (wanted > 1 && !places(wanted)) wanted /= 2;
  return wanted;
}
struct Kv4AttnArgs {
  Kv4View view;
  ElementType type = kF32;
  uint32_t heads = 0;
  const void* q = nullptr;
  void* out = nullptr;
  uint64_t q_token = 0, q_head = 0, out_token = 0, out_head = 0;
  float* lse = nullptr;  // [tokens][heads], may be null
  float scale = 0.f;
  bool causal = true;
  uint32_t window = 0;
  void* workspace = nullptr;
};
cudaError_t kv4_attention(const Kv4AttnArgs& a, const Kv4Plan& plan, cudaStream_t stream);

}  // namespace oct
