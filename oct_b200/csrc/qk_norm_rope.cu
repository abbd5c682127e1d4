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
// Bound: HBM, each element read and written once.  A block takes a few tokens:
// it computes their cosines and sines once into shared memory (a token's
// angles serve all its heads) and then streams their rows.  A row is spread
// over dim/16 lanes, each with the two 8-element vectors that hold both halves
// of its eight pairs, so a rotation needs no exchange between lanes.
//
// Angles: position * frequency is reduced to a fraction of a turn in binary64
// before the fp32 sine and cosine, because a far position loses every digit of
// the fraction in fp32 (at 2^20 a fp32 product is off by 2^-4 turns).
#include "serving.cuh"

namespace oct {
namespace {

constexpr int kThreads = 128;
constexpr uint32_t kMaxBlockTokens = 8;

template <typename T, int LANES>
__global__ void __launch_bounds__(kThreads) qk_norm_rope_kernel(const QkNormRopeArgs a, uint32_t block_tokens) {
  extern __shared__ float2 turns[];  // [block_tokens][rotary / 2] (cos, sin)
  const uint32_t pairs = a.rotary / 2;
  const uint64_t t0 = static_cast<uint64_t>(blockIdx.x) * block_tokens;
  const uint32_t nt = static_cast<uint32_t>(min(static_cast<uint64_t>(block_tokens), a.tokens - t0));
  for (uint32_t e = threadIdx.x; e < nt * pairs; e += kThreads) {
    const uint32_t t = e / pairs, j = e - t * pairs;
    uint32_t axis = 0, end = a.axis_pairs[0];
    while (j >= end && axis + 1 < a.axes) end += a.axis_pairs[++axis];
    const double pos = static_cast<double>(a.positions[(t0 + t) * a.position_stride + axis]);
    const double turn = pos * a.frequencies[j] * 0.15915494309189533576888;  // 1 / (2 pi)
    const float f = static_cast<float>(turn - rint(turn));
    float s, c;
    sincospif(2.0f * f, &s, &c);
    turns[e] = make_float2(c, s);
  }
  __syncthreads();

  constexpr uint32_t kRowsPerPass = kThreads / LANES;
  const uint32_t lane = threadIdx.x % LANES;
  const bool active = lane < a.dim / 16;
  // this lane's two vectors of eight channels, and its first pair
  const bool rotates = lane < a.rotary / 16;
  const uint32_t ca = a.interleaved || !rotates ? 16 * lane : 8 * lane;
  const uint32_t cb = a.interleaved || !rotates ? 16 * lane + 8 : a.rotary / 2 + 8 * lane;
#pragma unroll 1
  for (int which = 0; which < 2; ++which) {
    const uint32_t heads = a.heads[which];
    if (heads == 0) continue;
    const T* in = static_cast<const T*>(a.in[which]);
    T* out = static_cast<T*>(a.out[which]);
    float wa[8], wb[8];
    if (a.weight[which] != nullptr && active) {
      load8(a.weight[which] + ca, wa);
      load8(a.weight[which] + cb, wb);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) wa[i] = wb[i] = 1.f;
    }
    for (uint32_t r0 = 0; r0 < nt * heads; r0 += kRowsPerPass) {
      const uint32_t r = r0 + threadIdx.x / LANES;
      const bool live = active && r < nt * heads;
      const uint32_t t = r / heads, h = r - t * heads;
      float x[8] = {}, y[8] = {};
      if (live) {
        const T* p = in + (t0 + t) * a.in_token[which] + h * a.in_head[which];
        load8(p + ca, x);
        load8(p + cb, y);
      }
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
        const float2* cs = turns + t * pairs + 8 * lane;
        if (a.interleaved) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float2 u = cs[i], v = cs[4 + i];
            const float p = x[2 * i], q = x[2 * i + 1];
            x[2 * i] = p * u.x - q * u.y;
            x[2 * i + 1] = q * u.x + p * u.y;
            const float m = y[2 * i], n = y[2 * i + 1];
            y[2 * i] = m * v.x - n * v.y;
            y[2 * i + 1] = n * v.x + m * v.y;
          }
        } else {
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const float2 u = cs[i];
            const float p = x[i], q = y[i];
            x[i] = p * u.x - q * u.y;
            y[i] = q * u.x + p * u.y;
          }
        }
      }
      T* o = out + (t0 + t) * a.out_token[which] + h * a.out_head[which];
      store8(o + ca, x);
      store8(o + cb, y);
    }
  }
}

template <typename T>
cudaError_t launch(const QkNormRopeArgs& a, cudaStream_t stream) {
  // One token per block until the blocks fill the SMs several times over.
  const uint64_t per = a.tokens / (148ull * 16);
  const uint32_t bt = static_cast<uint32_t>(per < 1 ? 1 : (per > kMaxBlockTokens ? kMaxBlockTokens : per));
  const uint64_t blocks = (a.tokens + bt - 1) / bt;
  const size_t smem = static_cast<size_t>(bt) * (a.rotary / 2) * sizeof(float2);
  const dim3 grid(static_cast<uint32_t>(blocks));
  const uint32_t lanes = a.dim / 16;
  if (lanes <= 4)
    qk_norm_rope_kernel<T, 4><<<grid, kThreads, smem, stream>>>(a, bt);
  else if (lanes <= 8)
    qk_norm_rope_kernel<T, 8><<<grid, kThreads, smem, stream>>>(a, bt);
  else if (lanes <= 16)
    qk_norm_rope_kernel<T, 16><<<grid, kThreads, smem, stream>>>(a, bt);
  else
    qk_norm_rope_kernel<T, 32><<<grid, kThreads, smem, stream>>>(a, bt);
  return cudaGetLastError();
}

}  // namespace

cudaError_t qk_norm_rope(const QkNormRopeArgs& a, cudaStream_t stream) {
  if (a.tokens == 0 || (a.heads[0] == 0 && a.heads[1] == 0)) return cudaSuccess;
  switch (a.type) {
    case kF32: return launch<float>(a, stream);
    case kBf16: return launch<__nv_bfloat16>(a, stream);
    default: return launch<__half>(a, stream);
  }
}

}  // namespace oct
