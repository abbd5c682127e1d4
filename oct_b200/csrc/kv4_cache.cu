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
// Bound: HBM for the load (116 us for 701 MB: 6.0 TB/s, 0.92 of the measured copy
// rate), the issue slots for the store (170 us for 493 MB: 180 instructions for a
// warp's 256 channels, the schedulers issue in 73 % of the cycles).  A warp takes rows of one
// tile's keys or values of one head: one page lookup serves them all, and the loads
// of four passes over its lanes are in flight at once.  A lane holds 8 channels of
// a row (one 16-byte load of a 16-bit type), a group is 4 lanes and a row dim/8, so
// a group's bounds need two shuffles; one more pairs the halfwords of neighbouring
// groups into whole words.
#include <type_traits>

#include "serving.cuh"

namespace oct {
namespace {

constexpr int kWarps = 4;
constexpr int kThreads = kWarps * 32;
constexpr int kPasses = 4;  // row passes whose loads are issued together

__device__ __forceinline__ float min3_nan(float a, float b, float c) {
  float r;
  asm("min.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
__device__ __forceinline__ float max3_nan(float a, float b, float c) {
  float r;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

// What rounding d = x - z lost: x - z = d + the result, exactly (Knuth's two-sum, of x and -z).
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

// What a guess c of (x - z) / s is corrected by when its remainder d - c s reaches half a step: beyond
// it by one; at exactly half a step the rounding error of d = x - z decides, or the even integer.
__device__ __forceinline__ int correction(float x, float z, float s, float d, float c) {
  const float rem = fmaf(-c, s, d), half = 0.5f * s;  // one rounding: its comparison with s / 2 is exact
  if (rem > half) return 1;
  if (rem < -half) return -1;
  const bool above = rem > 0.f;  // c and, above or below it, the other neighbour are equally near d
  const float err = difference_error(x, z, d);
  const bool odd = (static_cast<int>(c) & 1) != 0;
  const bool other = err != 0.f ? (err > 0.f) == above : odd;
  return other ? (above ? 1 : -1) : 0;
}

// Eight codes, the first in the lowest bits: each the integer nearest to (x - z) / s, exactly.
__device__ __forceinline__ uint32_t codes_of(const float (&x)[8], float z, float s) {
  constexpr float kRound = 12582912.f;  // 1.5 * 2^23: adding it rounds to an integer, in the low bits
  constexpr uint32_t kRoundBits = 0x4B400000u;
  float inv;  // within an ulp: what a guess lacks the remainder shows
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(inv) : "f"(s));
  const float half = 0.5f * s;
  const Pair z2 = pair_of(-z, -z), s2 = pair_of(-s, -s), inv2 = pair_of(inv, inv);
  const Pair up = pair_of(kRound, kRound), down = pair_of(-kRound, -kRound);
  uint32_t codes = 0, bias = 0;
  bool near = false;
#pragma unroll
  for (int i = 0; i < 8; i += 2) {
    const Pair d = add(pair_of(x[i], x[i + 1]), z2);
    const Pair t = fma(d, inv2, up);
    const Pair rem = fma(add(t, down), s2, d);  // d - code * s
    float t0, t1, r0, r1;
    split(t, t0, t1);
    split(rem, r0, r1);
    near |= fabsf(r0) >= half || fabsf(r1) >= half;
    codes += (__float_as_uint(t0) << (4 * i)) + (__float_as_uint(t1) << (4 * i + 4));
    bias += (kRoundBits << (4 * i)) + (kRoundBits << (4 * i + 4));
  }
  codes -= bias;
  if (near && s > 0.f) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float d = x[i] - z, c = static_cast<float>((codes >> (4 * i)) & 15u);
      if (fabsf(fmaf(-c, s, d)) >= half) codes += static_cast<uint32_t>(correction(x[i], z, s, d, c)) << (4 * i);
    }
  }
  return s > 0.f ? codes : 0u;
}

// Eight elements as they lie in memory.
template <typename T> struct Raw { uint4 v[sizeof(T) / 2]; };
template <typename T>
__device__ __forceinline__ Raw<T> load_raw(const T* p) {
  Raw<T> r;
#pragma unroll
  for (int i = 0; i < static_cast<int>(sizeof(T) / 2); ++i) r.v[i] = reinterpret_cast<const uint4*>(p)[i];
  return r;
}

// Smallest and largest of a lane's eight elements, NaN where one is NaN.
__device__ __forceinline__ void bounds(const Raw<float>&, const float (&x)[8], float& lo, float& hi) {
  lo = min3_nan(min3_nan(x[0], x[1], x[2]), min3_nan(x[3], x[4], x[5]), min_nan(x[6], x[7]));
  hi = max3_nan(max3_nan(x[0], x[1], x[2]), max3_nan(x[3], x[4], x[5]), max_nan(x[6], x[7]));
}
template <typename T>
__device__ __forceinline__ void bounds(const Raw<T>& raw, const float (&)[8], float& lo, float& hi) {
  using T2 = typename std::conditional<std::is_same<T, __half>::value, __half2, __nv_bfloat162>::type;
  const T2* w = reinterpret_cast<const T2*>(raw.v);
  const T2 l = __hmin2_nan(__hmin2_nan(w[0], w[1]), __hmin2_nan(w[2], w[3]));
  const T2 h = __hmax2_nan(__hmax2_nan(w[0], w[1]), __hmax2_nan(w[2], w[3]));
  lo = static_cast<float>(__hmin_nan(l.x, l.y));
  hi = static_cast<float>(__hmax_nan(h.x, h.y));
}

template <int D>
struct Geometry {
  static constexpr int kGroups = D / 32, kRowBytes = D / 2, kLanes = D / 8;
  static constexpr int kRowsPerPass = 32 / kLanes;
  static constexpr int kStrips = 16 / (kRowsPerPass * kPasses);  // warps' shares of a tile's rows
  static constexpr int kParams = 16 * kRowBytes;            // (s, z) pairs behind the codes
  static constexpr int kHalf = kParams + 16 * kGroups * 4;  // keys; the values behind them
  static constexpr int kBytes = 2 * kHalf;
};

// What one warp works on: slots slot0 .. slot1 of a tile, from slot base0 on in runs of kPasses passes
// over its lanes; its keys and values, or one of them.
struct Strip {
  uint8_t* tile;
  int32_t base0, slot0, slot1;
  int64_t row;                 // row of slot 0 in the call's tensors (may lie before the sequence)
  uint32_t head, which0, which1;  // key head; first of keys (0) and values (1), and the one behind the last
};
// Strip u of a sequence.  Whole: (tile, key head), keys and values, so that one page lookup serves 32
// rows.  Else (tile, key head, keys or values, run of passes).
template <int D, bool kWhole>
__device__ __forceinline__ bool find_strip(const Kv4View& v, const Kv4Seq& s, uint32_t b, uint32_t u, Strip* p) {
  using G = Geometry<D>;
  const int32_t first = static_cast<int32_t>(s.len) - static_cast<int32_t>(s.n);  // position of the first row
  const uint32_t th = kWhole ? u : u / (2 * G::kStrips);
  const uint32_t t = th / v.kv_heads, tile = static_cast<uint32_t>(max(first, 0)) / kKv4Tile + t;
  const int32_t pos0 = static_cast<int32_t>(tile * kKv4Tile);
  p->head = th - t * v.kv_heads;
  constexpr int32_t kSlots = kWhole ? 16 : 16 / G::kStrips;
  const int32_t begin = kWhole ? 0 : static_cast<int32_t>(u % G::kStrips) * kSlots;
  p->which0 = kWhole ? 0 : u / G::kStrips % 2;
  p->which1 = kWhole ? 2 : p->which0 + 1;
  p->slot0 = max(first - pos0, begin);
  p->slot1 = min(static_cast<int32_t>(s.len) - pos0, begin + kSlots) - 1;
  if (p->slot0 > p->slot1) return false;
  p->base0 = p->slot0 / (kPasses * G::kRowsPerPass) * (kPasses * G::kRowsPerPass);
  const uint32_t in_table = tile / v.page_tiles;
  const uint32_t page = static_cast<uint32_t>(v.table[b * v.table_stride + in_table]);
  if (page >= v.pages) {
    if (threadIdx.x % 32 == 0) atomicAdd(v.skipped, 1ull);
    return false;
  }
  p->tile = kv4_tile(v, page, p->head, tile - in_table * v.page_tiles, G::kBytes);
  p->row = static_cast<int64_t>(s.row0) + pos0 - first;
  return true;
}
// Strips of a sequence; reports rows before position 0, which none covers.
template <int D, bool kWhole>
__device__ __forceinline__ uint32_t strips_of(const Kv4View& v, const Kv4Seq& s) {
  if (s.n > s.len && threadIdx.x == 0 && blockIdx.x == 0) atomicAdd(v.skipped, 1ull);
  if (s.n == 0 || s.len == 0) return 0;
  const uint32_t tile0 = (s.n > s.len ? 0u : s.len - s.n) / kKv4Tile;
  return ((s.len + kKv4Tile - 1) / kKv4Tile - tile0) * v.kv_heads * (kWhole ? 1 : 2 * Geometry<D>::kStrips);
}

// Runs of passes of a strip: keys first, then values.
template <int D>
struct Runs {
  static constexpr int kRun = kPasses * Geometry<D>::kRowsPerPass;
  int32_t per, count;  // of one half; of all
  __device__ __forceinline__ explicit Runs(const Strip& r)
      : per((r.slot1 - r.base0) / kRun + 1), count(per * static_cast<int32_t>(r.which1 - r.which0)) {}
  __device__ __forceinline__ uint32_t which(const Strip& r, int32_t q) const { return r.which0 + (q >= per ? 1u : 0u); }
  __device__ __forceinline__ int32_t base(const Strip& r, int32_t q) const { return r.base0 + (q >= per ? q - per : q) * kRun; }
};

template <typename T, int D, bool kWhole>
__global__ void __launch_bounds__(kThreads, 8) kv4_store_kernel(const Kv4RowArgs a) {
  using G = Geometry<D>;
  griddep_wait();
  Kv4Seq s;
  if (!kv4_seq(a.view, blockIdx.y, &s)) return;
  const int lane = threadIdx.x % G::kLanes, sub = threadIdx.x % 32 / G::kLanes;
  const int j = lane / 4, i4 = lane % 4;  // channels 32 j + 8 i4 .. + 7: halfwords 2 i4 and 2 i4 + 1 of group j
  const int word = (j & 1) ? ((2 * i4 + 1) * G::kGroups + j - 1) / 2 : (2 * i4 * G::kGroups + j) / 2;
  const uint32_t units = strips_of<D, kWhole>(a.view, s);
  for (uint32_t u = blockIdx.x * kWarps + threadIdx.x / 32; u < units; u += gridDim.x * kWarps) {
    Strip r;
    if (!find_strip<D, kWhole>(a.view, s, blockIdx.y, u, &r)) continue;
    const Runs<D> runs(r);
    auto fetch = [&](int32_t q, Raw<T>(&raw)[kPasses]) {
      const uint32_t which = runs.which(r, q);
      const int32_t base = runs.base(r, q);
      const int64_t stride = static_cast<int64_t>(a.token_stride[which]);
      const T* in = static_cast<const T*>(a.rows[which]) + r.head * a.head_stride[which] + 8 * lane + (r.row + base + sub) * stride;
#pragma unroll
      for (int p = 0; p < kPasses; ++p) {
        const int32_t slot = base + p * G::kRowsPerPass + sub;
        raw[p] = slot >= r.slot0 && slot <= r.slot1 ? load_raw(in + p * G::kRowsPerPass * stride) : Raw<T>{};
      }
    };
#pragma unroll 1
    for (int32_t q = 0; q < runs.count; ++q) {
      Raw<T> raw[kPasses];
      fetch(q, raw);
      uint8_t* const half = r.tile + runs.which(r, q) * G::kHalf;
      const int32_t base = runs.base(r, q);
#pragma unroll
      for (int p = 0; p < kPasses; ++p) {
        const int32_t slot0 = base + p * G::kRowsPerPass, slot = slot0 + sub;
        if (slot0 > r.slot1 || slot0 + G::kRowsPerPass <= r.slot0) continue;  // the whole warp's
        float x[8];
        load8(reinterpret_cast<const T*>(raw[p].v), x);
        float lo, hi;
        bounds(raw[p], x, lo, hi);
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
        if (slot < r.slot0 || slot > r.slot1) continue;
        reinterpret_cast<uint32_t*>(half + slot * G::kRowBytes)[word] =
            (j & 1) ? other | (codes & 0xffff0000u) : (codes & 0xffffu) | (other << 16);
        if (i4 == 0) reinterpret_cast<__half2*>(half + G::kParams)[slot * G::kGroups + j] = sz;
      }
    }
  }
}

template <typename T, int D, bool kWhole>
__global__ void __launch_bounds__(kThreads, 12) kv4_load_kernel(const Kv4RowArgs a) {
  using G = Geometry<D>;
  griddep_wait();
  Kv4Seq s;
  if (!kv4_seq(a.view, blockIdx.y, &s)) return;
  const int lane = threadIdx.x % G::kLanes, sub = threadIdx.x % 32 / G::kLanes;
  const int j = lane / 4, i4 = lane % 4;
  const int word = (j & 1) ? ((2 * i4 + 1) * G::kGroups + j - 1) / 2 : (2 * i4 * G::kGroups + j) / 2;
  const uint32_t units = strips_of<D, kWhole>(a.view, s);
  for (uint32_t u = blockIdx.x * kWarps + threadIdx.x / 32; u < units; u += gridDim.x * kWarps) {
    Strip r;
    if (!find_strip<D, kWhole>(a.view, s, blockIdx.y, u, &r)) continue;
    const Runs<D> runs(r);
    auto fetch = [&](int32_t q, uint32_t(&words)[kPasses], uint32_t(&params)[kPasses]) {
      const uint8_t* const half = r.tile + runs.which(r, q) * G::kHalf;
#pragma unroll
      for (int p = 0; p < kPasses; ++p) {
        const int32_t slot = runs.base(r, q) + p * G::kRowsPerPass + sub;  // inside the tile, whether live or not
        words[p] = reinterpret_cast<const uint32_t*>(half + slot * G::kRowBytes)[word];
        params[p] = reinterpret_cast<const uint32_t*>(half + G::kParams)[slot * G::kGroups + j];
      }
    };
#pragma unroll 1
    for (int32_t q = 0; q < runs.count; ++q) {
      uint32_t words[kPasses], params[kPasses];
      fetch(q, words, params);
      const uint32_t which = runs.which(r, q);
      const int32_t base = runs.base(r, q);
      const int64_t stride = static_cast<int64_t>(a.token_stride[which]);
      T* out = static_cast<T*>(a.rows[which]) + r.head * a.head_stride[which] + 8 * lane + (r.row + base + sub) * stride;
#pragma unroll
      for (int p = 0; p < kPasses; ++p) {
        const int32_t slot = base + p * G::kRowsPerPass + sub;
        const uint32_t other = __shfl_xor_sync(0xffffffffu, (j & 1) ? words[p] & 0xffffu : words[p] >> 16, 4);
        const uint32_t codes = (j & 1) ? other | (words[p] & 0xffff0000u) : (words[p] & 0xffffu) | (other << 16);
        if (slot < r.slot0 || slot > r.slot1) continue;
        const float2 sz = __half22float2(*reinterpret_cast<const __half2*>(&params[p]));
        float x[8];
        const uint32_t even = codes & 0x0f0f0f0fu, odd = (codes >> 4) & 0x0f0f0f0fu;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          // 2^23 + code, from the code's byte: exact, and no conversion instruction
          const Pair c = add(pair_of(__uint_as_float(__byte_perm(even, 0x4B000000u, 0x7440u + i)),
                                     __uint_as_float(__byte_perm(odd, 0x4B000000u, 0x7440u + i))),
                             pair_of(-8388608.f, -8388608.f));
          split(fma(c, pair_of(sz.x, sz.x), pair_of(sz.y, sz.y)), x[2 * i], x[2 * i + 1]);
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = within<T>(x[i]);
        store8(out + p * G::kRowsPerPass * stride, x);
      }
    }
  }
}

template <typename T, int D>
cudaError_t launch(const Kv4RowArgs& a, bool store, cudaStream_t stream) {
  // a sequence's rows may start and end inside a tile
  const uint64_t tiles = (static_cast<uint64_t>(a.view.max_tokens) + 2 * (kKv4Tile - 1)) / kKv4Tile;
  // A warp takes a whole tile of a head where that fills the SMs (one page lookup for 32 rows), else one
  // run of passes of its keys or values, so that a few tiles' rows are in flight at once (8.0 us against
  // 11.3 to store 8192 rows of 256).
  const uint64_t whole = tiles * a.view.kv_heads;
  const bool fills = whole * a.view.batch >= 148ull * 32;
  const uint64_t blocks = ((fills ? whole : whole * 2 * Geometry<D>::kStrips) + kWarps - 1) / kWarps;
  const dim3 grid(static_cast<uint32_t>(blocks < 65536 ? blocks : 65536), a.view.batch);
  const auto kernel = store ? (fills ? kv4_store_kernel<T, D, true> : kv4_store_kernel<T, D, false>)
                            : (fills ? kv4_load_kernel<T, D, true> : kv4_load_kernel<T, D, false>);
  return launch_dependent(kernel, grid, kThreads, 0, stream, 0, a);
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
