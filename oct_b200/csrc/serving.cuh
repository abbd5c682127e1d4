// serving.cuh -- device helpers the serving kernels share: element types in
// groups of eight, and a sequence's place in a 4-bit cache call.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <type_traits>

#include "ptx.cuh"
#include "serving.h"

namespace oct {

// Launches a kernel whose threads all begin with griddep_wait(): its blocks may be placed while the
// stream's previous kernel ends, and touch no memory before that one's is all written.  Cluster: blocks
// per cluster along x, or 0.
template <typename... P, typename... A>
cudaError_t launch_dependent(void (*kernel)(P...), dim3 grid, uint32_t threads, size_t smem, cudaStream_t stream,
                             uint32_t cluster, const A&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = cluster;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = cluster > 0 ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, kernel, args...);
}
// Whether the current device has room for a cluster of that many blocks.
template <typename... P>
bool has_room(void (*kernel)(P...), uint32_t threads, size_t smem, uint32_t cluster) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(cluster);
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = cluster;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  int clusters = 0;
  if (cudaOccupancyMaxActiveClusters(&clusters, kernel, &cfg) != cudaSuccess) {
    (void)cudaGetLastError();
    return false;
  }
  return clusters > 0;
}

template <ElementType T> struct Element;
template <> struct Element<kF32> { using type = float; };
template <> struct Element<kBf16> { using type = __nv_bfloat16; };
template <> struct Element<kF16> { using type = __half; };

// Eight consecutive elements, 16-byte aligned, as fp32.
__device__ __forceinline__ void load8(const float* p, float (&v)[8]) {
  const float4 a = *reinterpret_cast<const float4*>(p), b = *reinterpret_cast<const float4*>(p + 4);
  v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
}
__device__ __forceinline__ void load8(const __nv_bfloat16* p, float (&v)[8]) {
  const uint4 a = *reinterpret_cast<const uint4*>(p);
  const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    v[2 * i] = __uint_as_float(w[i] << 16);
    v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
  }
}
__device__ __forceinline__ void load8(const __half* p, float (&v)[8]) {
  const uint4 a = *reinterpret_cast<const uint4*>(p);
  const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
    v[2 * i] = f.x;
    v[2 * i + 1] = f.y;
  }
}
__device__ __forceinline__ void store8(float* p, const float (&v)[8]) {
  *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
  *reinterpret_cast<float4*>(p + 4) = make_float4(v[4], v[5], v[6], v[7]);
}
__device__ __forceinline__ uint32_t pack2(float a, float b, __nv_bfloat16) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t pack2(float a, float b, __half) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
template <typename T>
__device__ __forceinline__ void store8(T* p, const float (&v)[8]) {
  uint4 w;
  w.x = pack2(v[0], v[1], T());
  w.y = pack2(v[2], v[3], T());
  w.z = pack2(v[4], v[5], T());
  w.w = pack2(v[6], v[7], T());
  *reinterpret_cast<uint4*>(p) = w;
}
__device__ __forceinline__ float min_nan(float a, float b) {
  float r;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
// What reads back from the cache may lie a step (half of s) behind a clamped row's 65504: as float16 it is
// clamped there, so that no finite row becomes infinite; NaN stays NaN.
constexpr float kF16Max = 65504.f;
template <typename T>
__device__ __forceinline__ float within(float x) {
  return std::is_same<T, __half>::value ? min_nan(max_nan(x, -kF16Max), kF16Max) : x;
}
// Four consecutive elements.
__device__ __forceinline__ void store4(float* p, float4 v) { *reinterpret_cast<float4*>(p) = v; }
template <typename T>
__device__ __forceinline__ void store4(T* p, float4 v) {
  *reinterpret_cast<uint2*>(p) = make_uint2(pack2(v.x, v.y, T()), pack2(v.z, v.w, T()));
}

// Two fp32 values in one register pair: sm_100 adds and multiplies both with one instruction.
typedef unsigned long long Pair;
__device__ __forceinline__ Pair pair_of(float a, float b) {
  Pair r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void split(Pair p, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(p)); }
__device__ __forceinline__ Pair add(Pair a, Pair b) {
  Pair r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ Pair fma(Pair a, Pair b, Pair c) {
  Pair r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ Pair mul(Pair a, Pair b) {
  Pair r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}

// What sequence `b` of a call brings and holds.  False, and counted, when the
// arrays on the device do not fit the bounds that the host was given: such a
// sequence is skipped and nothing of it is read or written.
struct Kv4Seq {
  uint64_t row0;  // first row of the call's tensors
  uint32_t n;     // rows
  uint32_t len;   // tokens in the cache, the n new ones among them
};
__device__ __forceinline__ bool kv4_seq(const Kv4View& v, uint32_t b, Kv4Seq* s) {
  const int32_t len = v.kv_lens[b];
  int32_t r0 = static_cast<int32_t>(b), r1 = r0 + 1;
  if (v.cu_tokens != nullptr) {
    r0 = v.cu_tokens[b];
    r1 = v.cu_tokens[b + 1];
  }
  const bool ok = len >= 0 && static_cast<uint32_t>(len) <= v.max_kv_len && r0 >= 0 && r1 >= r0 &&
                  static_cast<uint64_t>(r1) <= v.tokens && static_cast<uint32_t>(r1 - r0) <= v.max_tokens;
  if (!ok) {
    atomicAdd(v.skipped, 1ull);
    return false;
  }
  s->row0 = static_cast<uint64_t>(r0);
  s->n = static_cast<uint32_t>(r1 - r0);
  s->len = static_cast<uint32_t>(len);
  return true;
}

// The tile that holds a page's token `tile * 16 ..` of key head `h`.
__device__ __forceinline__ uint8_t* kv4_tile(const Kv4View& v, uint32_t page, uint32_t h, uint32_t tile_in_page,
                                             uint32_t tile_bytes) {
  return v.data + ((static_cast<uint64_t>(page) * v.kv_heads + h) * v.page_tiles + tile_in_page) * tile_bytes;
}

}  // namespace oct
