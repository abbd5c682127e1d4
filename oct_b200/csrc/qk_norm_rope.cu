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
// pairs, so a rotation needs no exchange between lanes; first and second elements
// of two neighbouring pairs share a register pair, and every step works on both
// at once.  A thread keeps its row (head) and channels while it goes through a
// block's tokens: the weight stays in registers, the loads of the next tokens are
// on their way, and the tokens' cosines and sines, computed once per block into
// shared memory, serve all heads.  2 x 4096 tokens x 48 heads of 128 (bf16): 39 us,
// 5.1 TB/s (0.78 of the measured copy rate); 4096 tokens x 9 heads of 256 (fp32):
// 13-16 us, 4.7-5.8 TB/s; one token: 1.8 us from call to call in a graph.
//
// Angles: position * frequency is reduced to a fraction of a turn in binary64
// before the fp32 sine and cosine, because a far position loses every digit of
// the fraction in fp32 (at 2^20 a fp32 product is off by 2^-4 turns).
#include "serving.cuh"

namespace oct {
namespace {

constexpr uint32_t kMaxThreads = 256;
// Tokens whose loads are on their way at a time: 128 bytes a lane (16-bit types 45 us with two tokens, 41
// with four, for 2 x 4096 x 48 rows of 128; fp32 14.4 with two, 16.5 with four, for 4096 x 9 rows of 256).
template <typename T> constexpr int kTokensInFlight = sizeof(T) == 4 ? 2 : 4;
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
// The two vectors' sixteen elements as first and second elements of eight pairs: half-split, element i
// of either vector; interleaved, elements 2 i and 2 i + 1 of both in a row.
template <typename E>
__device__ __forceinline__ void to_pairs(const E (&e)[16], bool interleaved, E (&x)[8], E (&y)[8]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    x[i] = interleaved ? e[2 * i] : e[i];
    y[i] = interleaved ? e[2 * i + 1] : e[8 + i];
  }
}
__device__ __forceinline__ void as_pairs(const float (&x)[8], Pair (&p)[4]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) p[i] = pair_of(x[2 * i], x[2 * i + 1]);
}

// Grid x: runs of block_tokens tokens; y: runs of the rows (query heads, then key heads) of a token.
template <typename T, int LANES, bool kInterleaved>
__global__ void __launch_bounds__(kMaxThreads) qk_norm_rope_kernel(const QkNormRopeArgs a, uint32_t block_tokens) {
  constexpr int kInFlight = kTokensInFlight<T>;
  griddep_wait();
  extern __shared__ float2 turns[];  // [block_tokens][cos, sin][4][rotary / 16]: pairs 2 i and 2 i + 1 of a lane
  const uint32_t pairs = a.rotary / 2, strip = a.rotary / 16;
  const uint64_t t0 = static_cast<uint64_t>(blockIdx.x) * block_tokens;
  const uint32_t nt = static_cast<uint32_t>(min(static_cast<uint64_t>(block_tokens), a.tokens - t0));

  const uint32_t lane = threadIdx.x % LANES, r = blockIdx.y * (blockDim.x / LANES) + threadIdx.x / LANES;
  const uint32_t which = r < a.heads[0] ? 0 : 1, h = which == 0 ? r : r - a.heads[0];
  const bool live = lane < a.dim / 16 && r < a.heads[0] + a.heads[1];
  const bool rotates = lane < strip;
  const uint32_t ca = kInterleaved || !rotates ? 16 * lane : 8 * lane;
  const uint32_t cb = kInterleaved || !rotates ? 16 * lane + 8 : a.rotary / 2 + 8 * lane;
  const uint64_t in_step = a.in_token[which], out_step = a.out_token[which];
  const T* in = live ? static_cast<const T*>(a.in[which]) + t0 * in_step + h * a.in_head[which] : nullptr;
  T* out = live ? static_cast<T*>(a.out[which]) + t0 * out_step + h * a.out_head[which] : nullptr;
  Raw<T> raw[kInFlight];
#pragma unroll
  for (int i = 0; i < kInFlight; ++i) {
    raw[i] = live && i < static_cast<int>(nt) ? load_raw(in + ca, in + cb) : Raw<T>{};
    in += in_step;
  }
  // the table, while the first rows are on their way
  for (uint32_t e = threadIdx.x; e < nt * pairs; e += blockDim.x) {
    const uint32_t t = e / pairs, j = e - t * pairs;
    uint32_t axis = 0, end = a.axis_pairs[0];
    while (j >= end && axis + 1 < a.axes) end += a.axis_pairs[++axis];
    const double pos = static_cast<double>(a.positions[(t0 + t) * a.position_stride + axis]);
    const double turn = pos * a.frequencies[j] * 0.15915494309189533576888;  // 1 / (2 pi)
    const float f = static_cast<float>(turn - rint(turn));
    float s, c;
    sincospif(2.0f * f, &s, &c);
    float* to = reinterpret_cast<float*>(turns + t * pairs + j % 8 / 2 * strip + j / 8) + j % 2;
    to[0] = c;
    to[2 * 4 * strip] = s;
  }
  Pair wx[4], wy[4];
  {
    float e[16], x[8], y[8];
#pragma unroll
    for (int i = 0; i < 16; ++i) e[i] = 1.f;
    if (live && a.weight[which] != nullptr) {
      float va[8], vb[8];
      load8(a.weight[which] + ca, va);
      load8(a.weight[which] + cb, vb);
#pragma unroll
      for (int i = 0; i < 8; ++i) e[i] = va[i], e[8 + i] = vb[i];
    }
    to_pairs(e, kInterleaved, x, y);
    as_pairs(x, wx);
    as_pairs(y, wy);
  }
  const float mean = 1.0f / static_cast<float>(a.dim);
  __syncthreads();
#pragma unroll 1
  for (uint32_t b0 = 0; b0 < nt; b0 += kInFlight) {
#pragma unroll
    for (int n = 0; n < kInFlight; ++n) {
      const uint32_t t = b0 + n;
      if (t >= nt) break;
      Pair x[4], y[4];
      {
        float va[8], vb[8], e[16], u[8], v[8];
        load8(reinterpret_cast<const T*>(raw[n].v), va);
        load8(reinterpret_cast<const T*>(raw[n].v + sizeof(T) / 2), vb);
#pragma unroll
        for (int i = 0; i < 8; ++i) e[i] = va[i], e[8 + i] = vb[i];
        to_pairs(e, kInterleaved, u, v);
        as_pairs(u, x);
        as_pairs(v, y);
      }
      if (live && t + kInFlight < nt) raw[n] = load_raw(in + ca, in + cb);
      in += in_step;
      if (a.normalize) {
        Pair sum = 0ull;
#pragma unroll
        for (int i = 0; i < 4; ++i) sum = fma(x[i], x[i], fma(y[i], y[i], sum));
        float ss, other;
        split(sum, ss, other);
        ss += other;
#pragma unroll
        for (int o = LANES / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
        const float inv = rsqrtf(fmaf(ss, mean, a.eps));
        const Pair inv2 = pair_of(inv, inv);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          x[i] = mul(mul(x[i], inv2), wx[i]);
          y[i] = mul(mul(y[i], inv2), wy[i]);
        }
      }
      if (!live) continue;
      if (rotates) {
        const float2* cs = turns + t * pairs + lane;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float2 c = cs[i * strip], s = cs[(4 + i) * strip];
          const Pair c2 = pair_of(c.x, c.y), s2 = pair_of(s.x, s.y), n2 = pair_of(-s.x, -s.y);
          const Pair u = fma(x[i], c2, mul(y[i], n2));
          y[i] = fma(y[i], c2, mul(x[i], s2));
          x[i] = u;
        }
      }
      float va[8], vb[8];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float x0, x1, y0, y1;
        split(x[i], x0, x1);
        split(y[i], y0, y1);
        if constexpr (kInterleaved) {
          float(&to)[8] = i < 2 ? va : vb;
          to[4 * (i % 2)] = x0, to[4 * (i % 2) + 1] = y0, to[4 * (i % 2) + 2] = x1, to[4 * (i % 2) + 3] = y1;
        } else {
          va[2 * i] = x0, va[2 * i + 1] = x1, vb[2 * i] = y0, vb[2 * i + 1] = y1;
        }
      }
      store8(out + t * out_step + ca, va);
      store8(out + t * out_step + cb, vb);
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
  const dim3 grid(static_cast<uint32_t>(blocks), row_runs);
  return launch_dependent(a.interleaved ? qk_norm_rope_kernel<T, LANES, true> : qk_norm_rope_kernel<T, LANES, false>,
                          grid, threads, smem, stream, 0, a, bt);
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
