// qk_norm_rope.cu -- RMSNorm of every query and key head followed by the
// rotation to the token's position, in one pass over q and k.
//
// Per row of `dim` channels: y_c = x_c / sqrt(mean(x^2) + eps) * w_c (the norm
// and the weight are optional), then pairs of channels turn by
// position[axis of the pair] * frequency[pair]; half-split pairs are
// (j, j + rotary/2), interleaved pairs (2j, 2j + 1), channels behind `rotary`
// pass through.  It is the reference's head RMSNorm + RoPE
// (prometheus_reactor_runtime_gemma4e2b_m1_head_rmsnorm_rope,
// internal/prometheus/native/reactor_api.h:2700-2705) and, with interleaved
// pairs and three axes, its canonicalRope (internal/prometheus/zimage/
// canonical_reference.go:212-239), on device tensors and without stored tables.
//
// Bound: HBM, each element read and written once.  A row is spread over dim/16
// lanes, each with the two 8-element vectors that hold both halves of its eight
// pairs, so a rotation needs no exchange between lanes.  A thread keeps its row
// (head) and channels while it goes through a block's tokens: the weight stays in
// registers, the loads of the next tokens are on their way, and the tokens'
// cosines and sines, computed once per block into shared memory, serve all heads.
//
// Angles: position * frequency is reduced to a fraction of a turn in binary64
// before the fp32 sine and cosine, because a far position loses every digit of
// the fraction in fp32 (at 2^20 a fp32 product is off by 2^-4 turns).
#include "serving.cuh"

namespace oct {
namespace {

constexpr uint32_t kMaxThreads = 256;
constexpr int kInFlight = 4;              // tokens whose loads are issued together
constexpr uint32_t kMaxBlockTokens = 16;

template <typename T> struct Raw { uint4 v[sizeof(T)]; };  // two vectors of eight elements
template <typename T>
__device__ __forceinline__ Raw<T> load_raw(const T* a, const T* b) {
  constexpr int n = sizeof(T) / 2;
  Raw<T> r;
#pragma unroll
  for (int i = 0; i < n; ++i) {
    r.v[i] = reinterpret_cast<const uint4*>(a)[i];
    r.v[n + i] = reinterpret_cast<const uint4*>(b)[i];
  }
  return r;
}

// Grid x: runs of block_tokens tokens; y: runs of the rows (query heads, then key heads) of a token.
template <typename T, int LANES>
__global__ void __launch_bounds__(kMaxThreads) qk_norm_rope_kernel(const QkNormRopeArgs a, uint32_t block_tokens) {
  extern __shared__ float2 turns[];  // [block_tokens][8][rotary / 16] (cos, sin) of pair 8 lane + i at [i][lane]
  const uint32_t pairs = a.rotary / 2, strip = pairs / 8;
  const uint64_t t0 = static_cast<uint64_t>(blockIdx.x) * block_tokens;
  const uint32_t nt = static_cast<uint32_t>(min(static_cast<uint64_t>(block_tokens), a.tokens - t0));
  for (uint32_t e = threadIdx.x; e < nt * pairs; e += blockDim.x) {
    const uint32_t t = e / pairs, j = e - t * pairs;
    uint32_t axis = 0, end = a.axis_pairs[0];
    while (j >= end && axis + 1 < a.axes) end += a.axis_pairs[++axis];
    const double pos = static_cast<double>(a.positions[(t0 + t) * a.position_stride + axis]);
    const double turn = pos * a.frequencies[j] * 0.15915494309189533576888;  // 1 / (2 pi)
    const float f = static_cast<float>(turn - rint(turn));
    float s, c;
    sincospif(2.0f * f, &s, &c);
    turns[t * pairs + (j % 8) * strip + j / 8] = make_float2(c, s);
  }

  const uint32_t lane = threadIdx.x % LANES, r = blockIdx.y * (blockDim.x / LANES) + threadIdx.x / LANES;
  const uint32_t which = r < a.heads[0] ? 0 : 1, h = which == 0 ? r : r - a.heads[0];
  const bool live = lane < a.dim / 16 && r < a.heads[0] + a.heads[1];
  // this lane's two vectors of eight channels
  const bool rotates = lane < a.rotary / 16;
  const uint32_t ca = a.interleaved || !rotates ? 16 * lane : 8 * lane;
  const uint32_t cb = a.interleaved || !rotates ? 16 * lane + 8 : a.rotary / 2 + 8 * lane;
  const T* in = live ? static_cast<const T*>(a.in[which]) + t0 * a.in_token[which] + h * a.in_head[which] : nullptr;
  T* out = live ? static_cast<T*>(a.out[which]) + t0 * a.out_token[which] + h * a.out_head[which] : nullptr;
  float wa[8], wb[8];
  if (live && a.weight[which] != nullptr) {
    load8(a.weight[which] + ca, wa);
    load8(a.weight[which] + cb, wb);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) wa[i] = wb[i] = 1.f;
  }
  __syncthreads();
#pragma unroll 1
  for (uint32_t b0 = 0; b0 < nt; b0 += kInFlight) {
    Raw<T> raw[kInFlight];
#pragma unroll
    for (int i = 0; i < kInFlight; ++i) {
      const T* p = in + (b0 + i) * a.in_token[which];
      raw[i] = live && b0 + i < nt ? load_raw(p + ca, p + cb) : Raw<T>{};
    }
#pragma unroll
    for (int n = 0; n < kInFlight; ++n) {
      const uint32_t t = b0 + n;
      if (t >= nt) break;
      float x[8], y[8];
      load8(reinterpret_cast<const T*>(raw[n].v), x);
      load8(reinterpret_cast<const T*>(raw[n].v + sizeof(T) / 2), y);
      if (a.normalize) {
        float ss = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) ss = fmaf(x[i], x[i], fmaf(y[i], y[i], ss));
#pragma unroll
        for (int o = LANES / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
        const float inv = 1.0f / sqrtf(ss / static_cast<float>(a.dim) + a.eps);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          x[i] = x[i] * inv * wa[i];
          y[i] = y[i] * inv * wb[i];
        }
      }
      if (!live) continue;
      if (rotates) {
        const float2* cs = turns + t * pairs + lane;
        if (a.interleaved) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float2 u = cs[i * strip], v = cs[(4 + i) * strip];
            const float p = x[2 * i], q = x[2 * i + 1];
            x[2 * i] = p * u.x - q * u.y;
            x[2 * i + 1] = q * u.x + p * u.y;
            const float m = y[2 * i], n2 = y[2 * i + 1];
            y[2 * i] = m * v.x - n2 * v.y;
            y[2 * i + 1] = n2 * v.x + m * v.y;
          }
        } else {
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const float2 u = cs[i * strip];
            const float p = x[i], q = y[i];
            x[i] = p * u.x - q * u.y;
            y[i] = q * u.x + p * u.y;
          }
        }
      }
      T* o = out + t * a.out_token[which];
      store8(o + ca, x);
      store8(o + cb, y);
    }
  }
}

template <typename T, int LANES>
cudaError_t launch(const QkNormRopeArgs& a, cudaStream_t stream) {
  const uint32_t rows = a.heads[0] + a.heads[1];
  const uint32_t most = kMaxThreads / LANES;               // rows of a block
  const uint32_t runs = (rows + most - 1) / most, per = (rows + runs - 1) / runs;
  const uint32_t threads = (per * LANES + 31) / 32 * 32;
  const uint32_t row_runs = (rows + threads / LANES - 1) / (threads / LANES);
  // One token per block until the blocks fill the SMs several times over.
  const uint64_t share = a.tokens * row_runs / (148ull * 8);
  const uint32_t bt = static_cast<uint32_t>(share < 1 ? 1 : (share > kMaxBlockTokens ? kMaxBlockTokens : share));
  const uint64_t blocks = (a.tokens + bt - 1) / bt;
  const size_t smem = static_cast<size_t>(bt) * (a.rotary / 2) * sizeof(float2);
  qk_norm_rope_kernel<T, LANES><<<dim3(static_cast<uint32_t>(blocks), row_runs), threads, smem, stream>>>(a, bt);
  return cudaGetLastError();
}

template <typename T>
cudaError_t dispatch(const QkNormRopeArgs& a, cudaStream_t stream) {
  const uint32_t lanes = a.dim / 16;
  if (lanes <= 4) return launch<T, 4>(a, stream);
  if (lanes <= 8) return launch<T, 8>(a, stream);
  if (lanes <= 16) return launch<T, 16>(a, stream);
  return launch<T, 32>(a, stream);
}

}  // namespace

cudaError_t qk_norm_rope(const QkNormRopeArgs& a, cudaStream_t stream) {
  if (a.tokens == 0 || (a.heads[0] == 0 && a.heads[1] == 0)) return cudaSuccess;
  switch (a.type) {
    case kF32: return dispatch<float>(a, stream);
    case kBf16: return dispatch<__nv_bfloat16>(a, stream);
    default: return dispatch<__half>(a, stream);
  }
}

}  // namespace oct
