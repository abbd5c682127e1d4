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
// Bound: HBM.  A warp takes one tile's keys or values of one head: one page
// lookup serves up to 16 rows, and the loads of four passes are in flight at
// once.  A lane holds 8 channels of a row (one 16-byte load of a 16-bit type),
// a group is 4 lanes and a row dim/8, so a group's bounds need two shuffles;
// one more pairs the halfwords of neighbouring groups into whole words.
#include <type_traits>

#include "serving.cuh"

namespace oct {
namespace {

constexpr int kWarps = 4;
constexpr int kThreads = kWarps * 32;
constexpr int kPasses = 4;  // row passes whose loads are issued together
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
__device__ __forceinline__ float min_nan(float a, float b, float c) {
  float r;
  asm("min.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
__device__ __forceinline__ float max_nan(float a, float b, float c) {
  float r;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

// What rounding d = x - z lost: x - z = d + the result, exactly.
__device__ __forceinline__ float difference_error(float x, float z, float d) {
  const float bb = d - x;
  return (x - (d - bb)) + (-z - bb);
}

// The bounds (s, z) of a group with smallest value lo and largest hi.
__device__ __forceinline__ __half2 group_params(float lo, float hi) {
  const __half z = __float2half_rd(lo);
  const float zf = __half2float(z);
  // the float16 nearest to (hi - z) / 15 covers hi, or the next one does; 15 s is exact in fp32
  const float h = hi - zf;
  __half s = __float2half_rn(h * (1.0f / 15.0f));
  const float reach = 15.f * __half2float(s);
  if (reach < h || (reach == h && difference_error(hi, zf, h) > 0.f))
    s = __ushort_as_half(static_cast<unsigned short>(__half_as_ushort(s) + 1));
  if (!(lo <= hi)) s = __ushort_as_half(0);  // NaN
  return __halves2half2(s, z);
}

// The integer nearest to (x - z) / s, exactly: where the remainder of the guess reaches half a
// step it decides, and at exactly half a step the rounding error of x - z does, or the even integer.
__device__ __noinline__ uint32_t exact_code(float x, float z, float s) {
  const float d = x - z;
  float c = rintf(d / s);
  const float rem = fmaf(-c, s, d);  // one rounding: its comparison with s / 2 is exact
  const float half = 0.5f * s;
  if (rem > half) {
    c += 1.f;
  } else if (rem < -half) {
    c -= 1.f;
  } else if (fabsf(rem) == half) {
    const float err = difference_error(x, z, d);
    const float low = rem > 0.f ? c : c - 1.f;  // d = (low + 1/2) s
    c = err > 0.f ? low + 1.f : (err < 0.f ? low : 2.f * rintf(0.5f * (low + 0.5f)));
  }
  return static_cast<uint32_t>(c);
}

// Eight codes, the first in the lowest bits.
__device__ __forceinline__ uint32_t codes_of(const float (&x)[8], float z, float s) {
  constexpr float kRound = 12582912.f;  // 1.5 * 2^23: adding it rounds to an integer, in the low bits
  constexpr uint32_t kRoundBits = 0x4B400000u;
  const float inv = __frcp_rn(s), half = 0.5f * s;
  uint32_t codes = 0, bias = 0;
  bool near = false;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float d = x[i] - z;
    const float t = fmaf(d, inv, kRound);
    near |= fabsf(fmaf(kRound - t, s, d)) >= half;
    codes += __float_as_uint(t) << (4 * i);
    bias += kRoundBits << (4 * i);
  }
  codes -= bias;
  if (near && s > 0.f) {
    codes = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) codes |= exact_code(x[i], z, s) << (4 * i);
  }
  return s > 0.f ? codes : 0u;
}

template <int D>
struct Geometry {
  static constexpr int kGroups = D / 32, kRowBytes = D / 2, kLanes = D / 8;
  static constexpr int kRowsPerPass = 32 / kLanes;
  static constexpr int kParams = 16 * kRowBytes;            // (s, z) pairs behind the codes
  static constexpr int kHalf = kParams + 16 * kGroups * 4;  // keys; the values behind them
  static constexpr int kBytes = 2 * kHalf;
};

// Eight elements as they lie in memory.
template <typename T> struct Raw { uint4 v[sizeof(T) / 2]; };
template <typename T>
__device__ __forceinline__ Raw<T> load_raw(const T* p) {
  Raw<T> r;
#pragma unroll
  for (int i = 0; i < static_cast<int>(sizeof(T) / 2); ++i) r.v[i] = reinterpret_cast<const uint4*>(p)[i];
  return r;
}

// Calls body(tile half, first live slot, last live slot, row of slot 0 relative to the call's first
// row, key head, keys / values) for each of the tile halves that this warp works on.
template <int D, typename Body>
__device__ __forceinline__ void each_half_tile(const Kv4View& v, const Kv4Seq& s, uint32_t b, Body body) {
  const int32_t first = static_cast<int32_t>(s.len) - static_cast<int32_t>(s.n);  // position of the first row
  if (first < 0 && threadIdx.x == 0 && blockIdx.x == 0) atomicOr(v.bad, 1u);  // rows before position 0 are skipped
  const uint32_t tile0 = static_cast<uint32_t>(max(first, 0)) / kKv4Tile;
  const uint32_t tiles = (s.len + kKv4Tile - 1) / kKv4Tile - tile0;
  if (s.n == 0 || s.len == 0) return;
  const uint32_t units = tiles * v.kv_heads * 2;
  for (uint32_t u = blockIdx.x * kWarps + threadIdx.x / 32; u < units; u += gridDim.x * kWarps) {
    const uint32_t which = u & 1u, th = u >> 1, t = th / v.kv_heads, h = th - t * v.kv_heads;
    const uint32_t tile = tile0 + t, in_table = tile / v.page_tiles;
    const uint32_t page = static_cast<uint32_t>(v.table[b * v.table_stride + in_table]);
    if (page >= v.pages) {
      if (threadIdx.x % 32 == 0) atomicOr(v.bad, 1u);
      continue;
    }
    const int32_t pos0 = static_cast<int32_t>(tile * kKv4Tile);
    const int32_t slot0 = max(first - pos0, 0);
    const int32_t slot1 = min(static_cast<int32_t>(s.len) - pos0, static_cast<int32_t>(kKv4Tile)) - 1;
    body(kv4_tile(v, page, h, tile - in_table * v.page_tiles, Geometry<D>::kBytes) + which * Geometry<D>::kHalf, slot0,
         slot1, pos0 - first, h, which);
  }
}

template <typename T, int D>
__global__ void __launch_bounds__(kThreads) kv4_store_kernel(const Kv4RowArgs a) {
  using G = Geometry<D>;
  Kv4Seq s;
  if (!kv4_seq(a.view, blockIdx.y, &s)) return;
  const int lane = threadIdx.x % G::kLanes, sub = threadIdx.x % 32 / G::kLanes;
  const int j = lane / 4, i4 = lane % 4;  // channels 32 j + 8 i4 .. + 7: halfwords 2 i4 and 2 i4 + 1 of group j
  const int word = (j & 1) ? ((2 * i4 + 1) * G::kGroups + j - 1) / 2 : (2 * i4 * G::kGroups + j) / 2;
  each_half_tile<D>(a.view, s, blockIdx.y, [&](uint8_t* half, int32_t slot0, int32_t slot1, int32_t row0, uint32_t h,
                                               uint32_t which) {
    const T* in = static_cast<const T*>(a.rows[which]) + h * a.head_stride[which] + 8 * lane;
    for (int32_t base = slot0 / G::kRowsPerPass * G::kRowsPerPass; base <= slot1; base += kPasses * G::kRowsPerPass) {
      Raw<T> raw[kPasses];
#pragma unroll
      for (int p = 0; p < kPasses; ++p) {
        const int32_t slot = base + p * G::kRowsPerPass + sub;
        if (slot >= slot0 && slot <= slot1)
          raw[p] = load_raw(in + (s.row0 + static_cast<uint64_t>(static_cast<int64_t>(row0 + slot))) * a.token_stride[which]);
        else
          raw[p] = Raw<T>{};
      }
#pragma unroll
      for (int p = 0; p < kPasses; ++p) {
        const int32_t slot = base + p * G::kRowsPerPass + sub;
        if (base + p * G::kRowsPerPass > slot1) break;
        float x[8];
        load8(reinterpret_cast<const T*>(raw[p].v), x);
        float lo = min_nan(min_nan(x[0], x[1], x[2]), min_nan(x[3], x[4], x[5]), min_nan(x[6], x[7]));
        float hi = max_nan(max_nan(x[0], x[1], x[2]), max_nan(x[3], x[4], x[5]), max_nan(x[6], x[7]));
#pragma unroll
        for (int o = 1; o < 4; o <<= 1) {
          lo = min_nan(lo, __shfl_xor_sync(0xffffffffu, lo, o));
          hi = max_nan(hi, __shfl_xor_sync(0xffffffffu, hi, o));
        }
        if (lo < -kF16Max || hi > kF16Max) {
#pragma unroll
          for (int i = 0; i < 8; ++i) x[i] = min_nan(max_nan(x[i], -kF16Max), kF16Max);
          lo = min_nan(max_nan(lo, -kF16Max), kF16Max);
          hi = min_nan(max_nan(hi, -kF16Max), kF16Max);
        }
        const __half2 sz = group_params(lo, hi);
        const uint32_t codes = codes_of(x, __high2float(sz), __low2float(sz));
        const uint32_t other = __shfl_xor_sync(0xffffffffu, (j & 1) ? codes & 0xffffu : codes >> 16, 4);
        if (slot < slot0 || slot > slot1) continue;
        reinterpret_cast<uint32_t*>(half + slot * G::kRowBytes)[word] =
            (j & 1) ? other | (codes & 0xffff0000u) : (codes & 0xffffu) | (other << 16);
        if (i4 == 0) reinterpret_cast<__half2*>(half + G::kParams)[slot * G::kGroups + j] = sz;
      }
    }
  });
}

template <typename T, int D>
__global__ void __launch_bounds__(kThreads) kv4_load_kernel(const Kv4RowArgs a) {
  using G = Geometry<D>;
  Kv4Seq s;
  if (!kv4_seq(a.view, blockIdx.y, &s)) return;
  const int lane = threadIdx.x % G::kLanes, sub = threadIdx.x % 32 / G::kLanes;
  const int j = lane / 4, i4 = lane % 4;
  const int word = (j & 1) ? ((2 * i4 + 1) * G::kGroups + j - 1) / 2 : (2 * i4 * G::kGroups + j) / 2;
  each_half_tile<D>(a.view, s, blockIdx.y, [&](const uint8_t* half, int32_t slot0, int32_t slot1, int32_t row0,
                                               uint32_t h, uint32_t which) {
    T* out = static_cast<T*>(a.rows[which]) + h * a.head_stride[which] + 8 * lane;
    for (int32_t base = slot0 / G::kRowsPerPass * G::kRowsPerPass; base <= slot1; base += kPasses * G::kRowsPerPass) {
      uint32_t words[kPasses], params[kPasses];
#pragma unroll
      for (int p = 0; p < kPasses; ++p) {
        const int32_t slot = min(base + p * G::kRowsPerPass + sub, static_cast<int32_t>(kKv4Tile) - 1);
        words[p] = reinterpret_cast<const uint32_t*>(half + slot * G::kRowBytes)[word];
        params[p] = reinterpret_cast<const uint32_t*>(half + G::kParams)[slot * G::kGroups + j];
      }
#pragma unroll
      for (int p = 0; p < kPasses; ++p) {
        const int32_t slot = base + p * G::kRowsPerPass + sub;
        const uint32_t other = __shfl_xor_sync(0xffffffffu, (j & 1) ? words[p] & 0xffffu : words[p] >> 16, 4);
        const uint32_t codes = (j & 1) ? other | (words[p] & 0xffff0000u) : (words[p] & 0xffffu) | (other << 16);
        if (slot < slot0 || slot > slot1) continue;
        const float2 sz = __half22float2(*reinterpret_cast<const __half2*>(&params[p]));
        float x[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          // 2^23 + code by its bits: exact, and no conversion instruction
          const float c = __uint_as_float(((codes >> (4 * i)) & 15u) | 0x4B000000u) - 8388608.f;
          x[i] = fmaf(c, sz.x, sz.y);
          // z + 15 s may lie a step behind a clamped row's 65504: no finite row reads back as infinite
          if constexpr (std::is_same<T, __half>::value) x[i] = min_nan(max_nan(x[i], -kF16Max), kF16Max);
        }
        store8(out + (s.row0 + static_cast<uint64_t>(static_cast<int64_t>(row0 + slot))) * a.token_stride[which], x);
      }
    }
  });
}

template <typename T, int D>
cudaError_t launch(const Kv4RowArgs& a, bool store, cudaStream_t stream) {
  // a sequence's rows may start and end inside a tile
  const uint64_t tiles = (static_cast<uint64_t>(a.view.max_tokens) + 2 * (kKv4Tile - 1)) / kKv4Tile;
  const uint64_t blocks = (tiles * a.view.kv_heads * 2 + kWarps - 1) / kWarps;
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
