// kv4_cache.cu -- writing key and value rows into the 4-bit paged cache and
// reading them back.
//
// A row (one token, one key head, keys or values) is quantised in groups of 32
// channels.  With x clamped to +-65504 (infinities too):
//   z = the greatest float16 <= min x,  s = the least float16 with z + 15 s >= max x,
//   code = the integer nearest to (x - z) / s, ties to even (0 when s = 0),
// so every code is in 0..15 without clamping and the value z + s * code is
// within s / 2 of x.  A NaN makes its whole group read back as NaN (z = NaN,
// s = 0); the codes themselves are never anything but integers, which is what
// lets the attention multiply masked tokens by zero.
//
// In a row of dim/2 bytes the four codes of channels 32 j + 4 g + 0..3 form
// halfword g * (dim/32) + j: the attention's key fragments and its value
// fragments both read their operands from that one order without unpacking a
// code twice.
//
// Bound: HBM.  A lane holds 8 channels (one 16-byte load of a 16-bit type), a
// group is 4 lanes and a row dim/8, so the bounds of a group need two shuffles.
#include <type_traits>

#include "serving.cuh"

namespace oct {
namespace {

constexpr int kThreads = 256;
constexpr float kF16Max = 65504.f;

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

// The bounds (s, z) of a group with smallest value lo and largest hi.
__device__ __forceinline__ __half2 group_params(float lo, float hi) {
  const __half z = __float2half_rd(lo);
  const float zf = __half2float(z);
  // Rounding up at every step gives a candidate that covers hi; the step below
  // it is taken when that covers hi as well (in binary64, where both sides are exact).
  __half s = __float2half_ru(__fdiv_ru(__fsub_ru(hi, zf), 15.f));
  const unsigned short bits = __half_as_ushort(s);
  if (bits != 0 && bits < 0x7c00u) {
    const __half below = __ushort_as_half(static_cast<unsigned short>(bits - 1));
    if (static_cast<double>(zf) + 15.0 * static_cast<double>(__half2float(below)) >= static_cast<double>(hi)) s = below;
  }
  if (!(lo <= hi)) s = __ushort_as_half(0);  // NaN
  return __halves2half2(s, z);
}

// The integer nearest to (x - z) / s in 0..15, exactly: the quotient's guess is
// corrected where the remainder says so, and at a remainder of half a step the
// rounding error of x - z decides, or the even integer when there is none.
__device__ __forceinline__ uint32_t code_of(float x, float z, float s, float inv) {
  const float d = x - z;
  float c = rintf(d * inv);
  const float rem = fmaf(-c, s, d);  // one rounding: its comparison with s / 2 is exact
  const float half = 0.5f * s;
  if (fabsf(rem) >= half) {
    if (rem > half) c += 1.f;
    if (rem < -half) c -= 1.f;
    if (fabsf(rem) == half) {
      const float bb = d - x;  // two-sum error of x + (-z)
      const float err = (x - (d - bb)) + (-z - bb);
      const float low = rem > 0.f ? c : c - 1.f;  // d = (low + 1/2) s
      c = err > 0.f ? low + 1.f : (err < 0.f ? low : 2.f * rintf(0.5f * (low + 0.5f)));
    }
  }
  return static_cast<uint32_t>(c);
}

template <int D>
struct Geometry {
  static constexpr uint32_t kGroups = D / 32, kRowBytes = D / 2, kLanes = D / 8;
  static constexpr uint32_t kParams = 16 * kRowBytes;            // (s, z) pairs behind the codes
  static constexpr uint32_t kHalf = kParams + 16 * kGroups * 4;  // keys; the values behind them
  static constexpr uint32_t kBytes = 2 * kHalf;
};

// Lane's row of one sequence: rows go (token, key head, keys / values).
struct RowPlace {
  uint64_t in;   // element offset in the caller's tensor (keys or values)
  uint8_t* half; // the tile's keys or values
  uint32_t slot, which;
};
template <int D>
__device__ __forceinline__ bool row_place(const Kv4RowArgs& a, const Kv4Seq& s, uint32_t b, uint32_t row, RowPlace* p) {
  const Kv4View& v = a.view;
  const uint32_t which = row & 1u, th = row >> 1;
  const uint32_t t = th / v.kv_heads, h = th - t * v.kv_heads;
  const int64_t pos = static_cast<int64_t>(s.len) - s.n + t;
  uint32_t page = 0;
  bool ok = pos >= 0;
  const uint32_t tile = static_cast<uint32_t>(pos) / kKv4Tile;
  if (ok) {
    page = static_cast<uint32_t>(v.table[b * v.table_stride + tile / v.page_tiles]);
    ok = page < v.pages;
  }
  if (!ok) {
    atomicOr(v.bad, 1u);
    return false;
  }
  p->in = (s.row0 + t) * a.token_stride[which] + h * a.head_stride[which];
  p->half = kv4_tile(v, page, h, tile % v.page_tiles, Geometry<D>::kBytes) + which * Geometry<D>::kHalf;
  p->slot = static_cast<uint32_t>(pos) % kKv4Tile;
  p->which = which;
  return true;
}

template <typename T, int D>
__global__ void __launch_bounds__(kThreads) kv4_store_kernel(const Kv4RowArgs a) {
  using G = Geometry<D>;
  const uint32_t b = blockIdx.y;
  Kv4Seq s;
  if (!kv4_seq(a.view, b, &s)) return;
  const uint32_t rows = s.n * a.view.kv_heads * 2;
  const uint32_t lane = threadIdx.x % G::kLanes;
  const uint32_t j = lane / 4, g = 2 * (lane % 4);  // channels 32 j + 4 g .. + 7
  for (uint32_t r0 = blockIdx.x * (kThreads / G::kLanes); r0 < rows; r0 += gridDim.x * (kThreads / G::kLanes)) {
    const uint32_t row = r0 + threadIdx.x / G::kLanes;
    RowPlace p;
    const bool live = row < rows && row_place<D>(a, s, b, row, &p);
    float x[8] = {};
    if (live) load8(static_cast<const T*>(a.rows[p.which]) + p.in + 8 * lane, x);
    float lo, hi;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      x[i] = min_nan(max_nan(x[i], -kF16Max), kF16Max);
      lo = i == 0 ? x[0] : min_nan(lo, x[i]);
      hi = i == 0 ? x[0] : max_nan(hi, x[i]);
    }
#pragma unroll
    for (int o = 1; o < 4; o <<= 1) {
      lo = min_nan(lo, __shfl_xor_sync(0xffffffffu, lo, o));
      hi = max_nan(hi, __shfl_xor_sync(0xffffffffu, hi, o));
    }
    if (!live) continue;
    const __half2 sz = group_params(lo, hi);
    const float sf = __low2float(sz), zf = __high2float(sz);
    uint32_t codes = 0;
    if (sf > 0.f) {
      const float inv = 1.0f / sf;
#pragma unroll
      for (int i = 0; i < 8; ++i) codes |= code_of(x[i], zf, sf, inv) << (4 * i);
    }
    uint16_t* c = reinterpret_cast<uint16_t*>(p.half + p.slot * G::kRowBytes);
    c[g * G::kGroups + j] = static_cast<uint16_t>(codes);
    c[(g + 1) * G::kGroups + j] = static_cast<uint16_t>(codes >> 16);
    if (lane % 4 == 0) reinterpret_cast<__half2*>(p.half + G::kParams)[p.slot * G::kGroups + j] = sz;
  }
}

template <typename T, int D>
__global__ void __launch_bounds__(kThreads) kv4_load_kernel(const Kv4RowArgs a) {
  using G = Geometry<D>;
  const uint32_t b = blockIdx.y;
  Kv4Seq s;
  if (!kv4_seq(a.view, b, &s)) return;
  const uint32_t rows = s.n * a.view.kv_heads * 2;
  const uint32_t lane = threadIdx.x % G::kLanes;
  const uint32_t j = lane / 4, g = 2 * (lane % 4);
  for (uint32_t r0 = blockIdx.x * (kThreads / G::kLanes); r0 < rows; r0 += gridDim.x * (kThreads / G::kLanes)) {
    const uint32_t row = r0 + threadIdx.x / G::kLanes;
    RowPlace p;
    if (row >= rows || !row_place<D>(a, s, b, row, &p)) continue;
    const uint16_t* c = reinterpret_cast<const uint16_t*>(p.half + p.slot * G::kRowBytes);
    const uint32_t codes = c[g * G::kGroups + j] | (static_cast<uint32_t>(c[(g + 1) * G::kGroups + j]) << 16);
    const __half2 sz = reinterpret_cast<const __half2*>(p.half + G::kParams)[p.slot * G::kGroups + j];
    const float sf = __low2float(sz), zf = __high2float(sz);
    float x[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      x[i] = fmaf(static_cast<float>((codes >> (4 * i)) & 15u), sf, zf);
      // z + 15 s may lie a step behind a clamped row's 65504: no finite row reads back as infinite
      if constexpr (std::is_same<T, __half>::value) x[i] = min_nan(max_nan(x[i], -kF16Max), kF16Max);
    }
    store8(static_cast<T*>(a.rows[p.which]) + p.in + 8 * lane, x);
  }
}

template <typename T, int D>
cudaError_t launch(const Kv4RowArgs& a, bool store, cudaStream_t stream) {
  const uint64_t rows = static_cast<uint64_t>(a.view.max_tokens) * a.view.kv_heads * 2;
  const uint64_t per = kThreads / Geometry<D>::kLanes;
  const uint64_t blocks = (rows + per - 1) / per;
  const dim3 grid(static_cast<uint32_t>(blocks < 65536 ? blocks : 65536), a.view.batch);
  if (store)
    kv4_store_kernel<T, D><<<grid, kThreads, 0, stream>>>(a);
  else
    kv4_load_kernel<T, D><<<grid, kThreads, 0, stream>>>(a);
  return cudaGetLastError();
}

template <typename T>
cudaError_t dispatch(const Kv4RowArgs& a, bool store, cudaStream_t stream) {
  switch (a.view.dim) {
    case 64: return launch<T, 64>(a, store, stream);
    case 128: return launch<T, 128>(a, store, stream);
    case 256: return launch<T, 256>(a, store, stream);
    default: return cudaErrorInvalidValue;
  }
}

cudaError_t rows(const Kv4RowArgs& a, bool store, cudaStream_t stream) {
  if (a.view.batch == 0 || a.view.max_tokens == 0 || a.view.tokens == 0) return cudaSuccess;
  switch (a.type) {
    case kF32: return dispatch<float>(a, store, stream);
    case kBf16: return dispatch<__nv_bfloat16>(a, store, stream);
    default: return dispatch<__half>(a, store, stream);
  }
}

}  // namespace

cudaError_t kv4_store(const Kv4RowArgs& a, cudaStream_t stream) { return rows(a, true, stream); }
cudaError_t kv4_load(const Kv4RowArgs& a, cudaStream_t stream) { return rows(a, false, stream); }

}  // namespace oct
