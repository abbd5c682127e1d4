// kv4_attention.cu -- attention of a few query tokens per sequence over the
// 4-bit paged cache (the single-token form of the attention that the blocks
// run over whole sequences; the reference has neither a cache nor this step).
//
// For a query row and the keys p it sees (p <= its own position, and within
// the window when there is one):
//   score_p = scale * sum_j (s_pj (q . code)_pj + z_pj sum(q)_j),   j over groups of 32 channels
//   out     = sum_p w_p (z_pj + s_pj code_p) / sum_p w_p,           w_p = exp(score_p - max)
// The codes enter the matrix products as integers; scales meet fp32 sums (keys)
// or the weights (values), the zeros are a small product of their own, maxima,
// sums and results stay in fp32.
//
// Codes as operands.  A code masked out of its word into the low bits of a
// float16 is the number code * 2^-24, and one nibble further up code * 2^-20.  So
// four ANDs and one shift turn eight codes into matrix operands, with no
// conversion; the powers of two are undone on the other operand (q / 16 for the
// upper nibbles) and at the end.  fp16 and fp32 scores and fp32 results take
// normal numbers instead (`centred`, below).  q is scaled per row by a power of
// two that puts its largest value near 2^10, so that as float16 (one part for
// 16-bit inputs, two for fp32) it keeps its digits; the weights likewise, in one
// part for bf16 (2^-12 of each, an eighth of the result's rounding) and two else.
//
// Tokens are the rows of both products (m16n8k16: 16 tokens, 8 query rows), so
// one warp works through 16 keys at a time for 8 query rows -- the query heads
// that share a key head -- and the scores' fragment becomes the second
// product's operand with one 8 x 8 transposition per 8 tokens.
//
// Bound: HBM at a decode batch, reading each cached key once: 268 instructions
// per tile of 16 keys (bf16, 128 channels), 2560 bytes, stream at 6.1 TB/s once
// the blocks run (0.93 of the measured copy rate), which leaves the tensor pipe
// at 15-30 % and is why this runs on warp-level matrix instructions whose
// operands come from registers instead of through tcgen05 and tensor memory.
// fp16 (about 350 instructions) and fp32 are bound by their warps' latencies:
// with 168 registers a thread 12 warps share an SM and issue in every second
// cycle.  Each warp streams its own tiles (keys and values side by side) through
// a private ring in shared memory, by 16-byte asynchronous copies: no barrier
// between warps until an item's end, and none of the per-copy cost that bulk
// copies have at these sizes (a bulk copy a tile streamed at 4.6 TB/s with no
// arithmetic at all).
//
// Short items (one or few sequences, short keys, windows) get a cluster of blocks
// each, which join their parts through distributed shared memory.  Else blocks
// take equal runs of the call's tiles, whatever the sequences' lengths: each adds
// up the lengths on the device and finds its own run (2 us), and an item that a
// run's end cuts leaves partial results, which a second kernel joins in order
// (4-5 us).  Measured, whole calls: 64 sequences of up to 16384 keys, 32 / 8
// heads of 128, bf16 124-135 us (587 MB, floor 89); one of 131071 keys, fp16 57 us
// (168 MB, floor 26); one of 1000 keys, 8 / 1 heads of 256, bf16 9.8 us (latency;
// 14.4 spread over the GPU and joined by a second kernel).
#include <algorithm>
#include <atomic>
#include <type_traits>

#include "kernels.h"
#include "ptx.cuh"
#include "serving.cuh"

namespace oct {
namespace {

constexpr int kWarps = 4;
constexpr int kThreads = kWarps * 32;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
// The running maximum is renewed only when a score exceeds it by this much (in
// powers of two): weights stay below 2^4, and most tiles skip the exchange.
constexpr float kSlack = 4.f;
constexpr uint32_t kNoTile = 0xffffffffu;
constexpr int32_t kNowhere = 0x7fffffff - 64;  // no sequence is that long
constexpr float kCodeLow = 16777216.f, kCodeHigh = 1048576.f;  // 2^24, 2^20

template <int D>
struct Geometry {
  static constexpr int kGroups = D / 32;
  static constexpr int kRowBytes = D / 2;
  static constexpr int kKeyParams = 16 * kRowBytes;
  static constexpr int kValues = kKeyParams + 16 * kGroups * 4;
  static constexpr int kValueParams = kValues + 16 * kRowBytes;
  static constexpr int kBytes = 2 * kValues;
  // ring of tiles per warp: 10 to 20 KB, and room for the warp's result at the end
  static constexpr int kStages = D == 64 ? 8 : (D == 128 ? 6 : 4);
};

// Tiles that a warp works through at a time: with two, one vote on the maximum and one on the scales
// serve 32 keys and their operands' latencies overlap.
constexpr int tiles_per_step(int dim, int row_groups) { return dim * row_groups <= 128 ? 2 : 1; }
// Blocks of a cluster that share one item, at most: more than the portable 8 (one token over 1000 keys of
// 256 channels: 10.8 us with up to 16, 12.3 with up to 8).
constexpr uint32_t kMaxCluster = 16;
// Units that each block of a cluster may get; longer items are spread over the whole GPU, which balances
// sequences of unequal lengths.  Clusters against equal runs, sequences of one length: 8 of 2048 keys, 32 / 8
// heads of 128, bf16, 12.2 us against 15.5 (4 units a block), of 4096 16.4 against 20.9 (8), 16 of 8192 45.5
// against 43.9 (32); fp32, 8 / 1 heads of 256, one of 4096 15.6 against 16.4 (4), of 8192 22.0 against 20.3 (8).
constexpr uint32_t cluster_units(ElementType type) { return type == kF32 ? 4 : 8; }
// Blocks per SM that the compiler leaves registers for, and that a launch fills.
constexpr int blocks_per_sm(int dim, int row_groups) { return dim * row_groups <= 128 ? 3 : 2; }
// Query rows of one block in groups of 8, by what the accumulators leave of the registers.
template <int D> constexpr int kMaxRowGroups = D == 64 ? 4 : (D == 128 ? 2 : 1);

__device__ __forceinline__ void mma_f16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                        uint32_t b1) {
  asm(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// Codes less 8 as normal numbers: code - 8 from the low nibble, 16 times that from the high one.  The
// subnormal codes are exact, but the tensor cores align their products as if they were 2^-14, so that the
// sums keep about 18 bits, and truncate as they add, which unsigned codes let grow with the sum of the
// weights while the zeros cancel most of it.  Scores are 5e-8 off with centred keys against up to 1.4e-6:
// 16-bit results differ by that in their lse alone, so bf16 takes the cheaper form (64 sequences: 126 us
// against 141, lse 3.2e-6 off against 1.4e-6, the results' error the same to three digits; the header tells
// the caller) and fp16, whose results keep eight times as many digits, does not (60 us against 55 for 131071
// keys).
// fp32 results over 512 keys are 2e-7 off with centred values against 1.6e-5 (there less 7.5, 16 times
// over, so that the codes' mean is near zero and a bias of the sums has nothing to act on).
constexpr uint32_t kMiddleLow = 0x64086408u, kMiddleHigh = 0x64806480u;  // 1024 + 8, 1024 + 128
constexpr uint32_t kMiddleHalf = 0x64786478u;                             // 1024 + 120
__device__ __forceinline__ uint32_t centred(uint32_t codes, uint32_t middle) {
  const uint32_t x = codes | 0x64006400u;  // 1024 + code
  const __half2 r = __hsub2(*reinterpret_cast<const __half2*>(&x), *reinterpret_cast<const __half2*>(&middle));
  return *reinterpret_cast<const uint32_t*>(&r);
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
  uint32_t r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
  return r;
}
// 8 x 8 matrices of 16-bit elements from shared memory, transposed: lanes 8 m .. 8 m + 7 name the rows of matrix m.
__device__ __forceinline__ void load_transposed(uint32_t& m0, uint32_t& m1, const void* row) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x2.trans.shared.b16 {%0, %1}, [%2];" : "=r"(m0), "=r"(m1) : "r"(smem_addr(row)) : "memory");
}
__device__ __forceinline__ void load_transposed(uint32_t& m0, uint32_t& m1, uint32_t& m2, uint32_t& m3, const void* row) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(m0), "=r"(m1), "=r"(m2), "=r"(m3)
               : "r"(smem_addr(row))
               : "memory");
}
// Loads from the shared memory of another block of the cluster.
__device__ __forceinline__ float2 ld_cluster_v2(uint32_t addr) {
  float2 v;
  asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ float4 ld_cluster_v4(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
               : "r"(addr)
               : "memory");
  return v;
}
__device__ __forceinline__ float exp2_approx(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
__device__ __forceinline__ uint32_t pack_half2(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t max_half2(uint32_t a, uint32_t b) {
  const __half2 h = __hmax2(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&b));
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ float max_half(uint32_t a) {
  const __half2 h = *reinterpret_cast<const __half2*>(&a);
  return __half2float(__hmax(__low2half(h), __high2half(h)));
}
__device__ __forceinline__ uint32_t times(uint32_t a, uint32_t b) {
  const __half2 h = __hmul2(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&b));
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t times_plus(uint32_t a, uint32_t b, uint32_t c) {
  const __half2 h = __hfma2(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&b),
                            *reinterpret_cast<const __half2*>(&c));
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t times_minus(uint32_t a, uint32_t b, uint32_t c) {
  const __half2 h = __hfma2(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&b),
                            __hneg2(*reinterpret_cast<const __half2*>(&c)));
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ float2 unpack_half2(uint32_t w) {
  return __half22float2(*reinterpret_cast<const __half2*>(&w));
}
// a power of two with the exponent of x shifted to `target`; 1 for zero and non-finite x
__device__ __forceinline__ float pow2_toward(float x, int target) {
  const int e = static_cast<int>((__float_as_uint(x) >> 23) & 255u);
  if (e == 0 || e == 255) return 1.f;
  const int f = target + 127 - (e - 127);
  return __uint_as_float(static_cast<uint32_t>(f < 1 ? 1 : (f > 254 ? 254 : f)) << 23);
}

// 16 bytes from global into shared memory, past the L1 cache; waits count commit groups.
__device__ __forceinline__ void copy16(void* to, const void* from) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_addr(to)), "l"(from) : "memory");
}
__device__ __forceinline__ void commit_copies() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void wait_copies() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

template <int N>
__device__ __forceinline__ void lds(uint32_t (&w)[N], const uint8_t* p) {
  if constexpr (N == 1) {
    w[0] = *reinterpret_cast<const uint32_t*>(p);
  } else if constexpr (N == 2) {
    const uint2 v = *reinterpret_cast<const uint2*>(p);
    w[0] = v.x, w[1] = v.y;
  } else {
#pragma unroll
    for (int i = 0; i < N / 4; ++i) {
      const uint4 v = *reinterpret_cast<const uint4*>(p + 16 * i);
      w[4 * i] = v.x, w[4 * i + 1] = v.y, w[4 * i + 2] = v.z, w[4 * i + 3] = v.w;
    }
  }
}

// A row's four channels from their sums and one over the sum of the weights.
template <typename T>
__device__ __forceinline__ float4 result(float4 sum, float inv) {
  return make_float4(within<T>(sum.x * inv), within<T>(sum.y * inv), within<T>(sum.z * inv), within<T>(sum.w * inv));
}

// What a block began and did not finish, for the join.
struct PartOf {
  uint32_t last1 = 0;  // the last block with a part of it, plus 1; 0: nothing was left unfinished
  uint32_t head = 0, first = 0, count = 0;  // its key head and rows
  uint64_t row0 = 0, pad = 0;
};
struct KernelArgs {
  Kv4View view;
  const void* q;
  void* out;
  uint64_t q_token, q_head, out_token, out_head;
  float* lse;
  float scale_log2;
  uint32_t heads, share;  // query heads, query heads of one key head
  uint32_t causal, window;
  uint32_t row_tiles;
  float* part_o;    // [blocks][2][rows of a tile][D]
  float2* part_ml;  // [blocks][2][rows of a tile]
  PartOf* part_of;  // [blocks]
  uint32_t cluster;  // blocks that share one item and join it among themselves; 0: equal runs of all items
};

// The keys that the rows of one row tile see: row r of a sequence is query
// token r / share, whose own position is last.
struct Rows {
  uint32_t first, count;  // rows of the tile inside the sequence
  int32_t lo_min, lo_max, hi_min, hi_max;
  int32_t t_begin, t_end;  // 16-key tiles
};
__device__ __forceinline__ int32_t row_hi(const KernelArgs& a, const Kv4Seq& s, uint32_t row) {
  return a.causal ? static_cast<int32_t>(s.len) - static_cast<int32_t>(s.n) + static_cast<int32_t>(row / a.share)
                  : static_cast<int32_t>(s.len) - 1;
}
__device__ __forceinline__ int32_t row_lo(const KernelArgs& a, int32_t hi) {
  const int64_t lo = static_cast<int64_t>(hi) - a.window + 1;
  return a.window == 0 || lo < 0 ? 0 : static_cast<int32_t>(lo);
}
__device__ __forceinline__ bool row_range(const KernelArgs& a, const Kv4Seq& s, uint32_t tile, uint32_t rows_per_tile,
                                          Rows* r) {
  const uint32_t rows = s.n * a.share;
  r->first = tile * rows_per_tile;
  if (r->first >= rows) return false;
  r->count = min(rows_per_tile, rows - r->first);
  r->hi_min = row_hi(a, s, r->first);
  r->hi_max = row_hi(a, s, r->first + r->count - 1);
  r->lo_min = row_lo(a, r->hi_min);
  r->lo_max = row_lo(a, r->hi_max);
  r->t_begin = r->lo_min / static_cast<int32_t>(kKv4Tile);
  r->t_end = r->hi_max < 0 ? r->t_begin : r->hi_max / static_cast<int32_t>(kKv4Tile) + 1;
  return true;
}

// An item is one (sequence, row tile, key head); its units are runs of one
// step's tiles for every warp, at least one so that a row without keys is written too.  Items stand
// in that order, and every block takes an equal run of all the call's units.
__device__ __forceinline__ uint32_t item_units(const Rows& r, int32_t unit_tiles) {
  return static_cast<uint32_t>(max(1, (r.t_end - r.t_begin + unit_tiles - 1) / unit_tiles));
}
__device__ __forceinline__ bool item_rows(const KernelArgs& a, uint32_t pair, uint32_t rows_per_tile, Kv4Seq* s,
                                          Rows* r) {
  const uint32_t b = pair / a.row_tiles;
  return kv4_seq(a.view, b, s) && row_range(a, *s, pair - b * a.row_tiles, rows_per_tile, r);
}
// What an item costs beside its units, in units: finding its pages, loading its queries, joining its
// warps.  Counted where blocks get several units, so that one with many short items gets fewer of them
// (64 sequences of up to 16384 keys: 151 us at a cost of 1, 127 at 5, 129 at 8).  Where units are few,
// latency counts: there no block gets parts of two items, an item's run is filled up to whole shares.
constexpr uint32_t kItemCost = 5;
struct Share {
  uint32_t begin, end, per;     // this block's run of all items' runs; every block's length
  uint32_t cost, pad;           // kItemCost or 0; shares that an item's run is filled up to, or 1
  uint32_t pair, head, offset;  // where it begins
  __device__ __forceinline__ uint32_t size(uint32_t units) const { return (units + cost + pad - 1) / pad * pad; }
};
// Called by the whole block.  Sums fit in 32 bits: the host refuses calls whose bounds do not.
__device__ __forceinline__ bool find_share(const KernelArgs& a, uint32_t rows_per_tile, int32_t unit_tiles, Share* out) {
  __shared__ uint32_t warp_sums[3][kWarps];
  __shared__ uint32_t found[3];
  const uint32_t pairs = a.view.batch * a.row_tiles, chunk = (pairs + kThreads - 1) / kThreads;
  const uint32_t p0 = min(pairs, threadIdx.x * chunk), p1 = min(pairs, p0 + chunk);
  const uint32_t lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  Kv4Seq s;
  Rows r;
  uint32_t units = 0, items = 0;
  for (uint32_t p = p0; p < p1; ++p)
    if (item_rows(a, p, rows_per_tile, &s, &r)) units += item_units(r, unit_tiles), ++items;
  const uint32_t unit_sum = __reduce_add_sync(0xffffffffu, units), item_sum = __reduce_add_sync(0xffffffffu, items);
  if (lane == 0) warp_sums[0][warp] = unit_sum, warp_sums[1][warp] = item_sum;
  __syncthreads();
  uint32_t total = 0, all_items = 0;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) total += warp_sums[0][w], all_items += warp_sums[1][w];
  total *= a.view.kv_heads;
  all_items *= a.view.kv_heads;
  const bool few = total <= 4 * gridDim.x && all_items <= gridDim.x / 2;
  // without a workspace every item is one unit and stays whole: no cost may be cut off it
  out->cost = few || a.part_o == nullptr ? 0 : kItemCost;
  const uint32_t run = total + out->cost * all_items, blocks = few ? gridDim.x - all_items : gridDim.x;
  out->per = max(1u, (run + blocks - 1) / blocks);
  out->pad = few ? out->per : 1;
  // runs of the threads before this one
  uint32_t mine = units + out->cost * items;
  if (few) {
    mine = 0;
    for (uint32_t p = p0; p < p1; ++p)
      if (item_rows(a, p, rows_per_tile, &s, &r)) mine += out->size(item_units(r, unit_tiles));
  }
  mine *= a.view.kv_heads;
  uint32_t upto = mine;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const uint32_t v = __shfl_up_sync(0xffffffffu, upto, d);
    if (lane >= static_cast<uint32_t>(d)) upto += v;
  }
  if (lane == 31) warp_sums[2][warp] = upto;
  __syncthreads();
  uint32_t all = 0;
#pragma unroll
  for (uint32_t w = 0; w < kWarps; ++w) {
    if (w < warp) upto += warp_sums[2][w];
    all += warp_sums[2][w];
  }
  out->begin = blockIdx.x * out->per;
  out->end = min(all, out->begin + out->per);
  if (out->begin >= all) return false;
  uint32_t at = upto - mine;
  if (out->begin >= at && out->begin < upto)
    for (uint32_t p = p0; p < p1; ++p)
      if (item_rows(a, p, rows_per_tile, &s, &r)) {
        const uint32_t size = out->size(item_units(r, unit_tiles));
        if (out->begin < at + size * a.view.kv_heads) {
          const uint32_t rest = out->begin - at;
          found[0] = p;
          found[1] = rest / size;
          found[2] = rest % size;
          break;
        }
        at += size * a.view.kv_heads;
      }
  __syncthreads();
  out->pair = found[0];
  out->head = found[1];
  out->offset = found[2];
  return true;
}

// A block's share where every cluster has one item: an equal run of its units.
__device__ __forceinline__ void cluster_share(const KernelArgs& a, uint32_t rows_per_tile, int32_t unit_tiles,
                                              Share* out, PartOf* item) {
  const uint32_t at = blockIdx.x / a.cluster, rank = blockIdx.x - at * a.cluster;
  out->pair = at / a.view.kv_heads;
  out->head = at - out->pair * a.view.kv_heads;
  Kv4Seq s;
  Rows r;
  uint32_t units = 0, count = 0;
  if (item_rows(a, out->pair, rows_per_tile, &s, &r)) units = item_units(r, unit_tiles), count = r.count;
  out->per = (units + a.cluster - 1) / a.cluster;
  out->begin = out->offset = min(units, rank * out->per);
  out->end = min(units, out->begin + out->per);
  out->cost = 0;
  out->pad = 1;
  if (threadIdx.x == 0) *item = PartOf{0, out->head, count > 0 ? r.first : 0, count, count > 0 ? s.row0 : 0, 0};
}

// float16 bits, zero for infinities and NaN
__device__ __forceinline__ uint32_t finite_half(uint32_t bits) { return (bits & 0x7c00u) == 0x7c00u ? 0u : bits; }

template <typename T, int D, int NT, int QP, int PP>
__global__ void __launch_bounds__(kThreads, blocks_per_sm(D, NT)) kv4_attention_kernel(const KernelArgs a) {
  using G = Geometry<D>;
  constexpr int NG = G::kGroups;
  constexpr int kRows = 8 * NT;
  constexpr int kZeroWords = NG == 8 ? 2 : 1;
  constexpr int H = tiles_per_step(D, NT), kUnit = kWarps * H;
  constexpr int kStages = G::kStages / H, kStageBytes = H * G::kBytes;
  constexpr bool kCentred = std::is_same<T, float>::value;  // value codes less 7.5
  constexpr bool kCentredKeys = PP == 2;                    // key codes less 8
  // fp32: every tile's part of the result is added rounded to nearest, since the tensor cores' truncation adds
  // up over the keys (2 x 64 rows over 77541 keys: 8e-6 of the result off, so 1e-7; the 512-key window 20.7 us,
  // so 22.5; 16-bit results do not show it).
  constexpr bool kNearest = kCentred;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ uint32_t loaded[kWarps][kStages];
  __shared__ float2 warp_ml[kWarps][kRows];

  __shared__ PartOf cluster_item;
  __shared__ float2 block_ml[kRows];

  griddep_wait();
  Share share;
  if (a.cluster != 0) {
    cluster_share(a, kRows, kUnit, &share, &cluster_item);
    if (share.begin >= share.end && threadIdx.x < kRows) block_ml[threadIdx.x] = make_float2(-INFINITY, 0.f);
  } else {
    if (a.part_o != nullptr) griddep_launch_dependents();  // the join
    const bool any = find_share(a, kRows, kUnit, &share);
    if (threadIdx.x == 0 && a.part_of != nullptr) a.part_of[blockIdx.x] = PartOf{};
    if (!any) return;
  }

  const uint32_t warp = threadIdx.x / 32, lane = threadIdx.x % 32, g = lane / 4, i4 = lane % 4;
  uint8_t* ring = smem + warp * (G::kStages * G::kBytes);
  // Token of score row g (and, 8 further, of row g + 8): an order in which a
  // quarter warp's key loads touch every bank once and the value loads twice.
  const int32_t tok_g = (g & 1) ? 4 + static_cast<int32_t>((g >> 1) ^ 1u) : static_cast<int32_t>(g >> 1);
  const int32_t tok_v[2] = {static_cast<int32_t>(i4), 4 + static_cast<int32_t>(i4 ^ 1u)};  // rows 2 i4, 2 i4 + 1

  const int32_t tok_ld = static_cast<int32_t>((lane & 1) ? 4 + (((lane % 8) >> 1) ^ 1u) : (lane % 8) >> 1) + 8 * static_cast<int32_t>((lane >> 3) & 1);
  const bool looks = g % 2 == 0 && g < 2 * NG;  // whether its row of the zeros' operand holds scales

  // The item at `unit`, if it is this block's.
  struct Item {
    Kv4Seq seq;
    Rows rows;
    uint32_t pair, head, offset, size, take;
    int32_t first_tile, t1, steps;  // of this warp: tiles of step 0, of step 1 kUnit further, ... up to t1
  };
  uint32_t unit = share.begin;
  auto open = [&](Item* it, uint32_t pair, uint32_t head, uint32_t offset) {
    if (unit >= share.end) return false;
    while (true) {
      if (pair >= a.view.batch * a.row_tiles) return false;  // lengths that changed under the call
      if (item_rows(a, pair, kRows, &it->seq, &it->rows)) break;
      ++pair;  // a sequence or row tile without rows has no units
    }
    it->pair = pair, it->head = head, it->offset = offset;
    it->size = share.size(item_units(it->rows, kUnit));
    it->take = min(it->size - offset, share.end - unit);
    // the item's cost comes first in its run; the units behind it are its tiles
    const uint32_t unit0 = max(offset, share.cost) - share.cost;
    const uint32_t unit1 = max(offset + it->take, share.cost) - share.cost;
    it->first_tile = it->rows.t_begin + static_cast<int32_t>(unit0 * kUnit + warp * H);
    it->t1 = min(it->rows.t_end, it->rows.t_begin + static_cast<int32_t>(unit1 * kUnit));
    it->steps = it->first_tile < it->t1 ? (it->t1 - it->first_tile + kUnit - 1) / kUnit : 0;
    return true;
  };
  // Which of the cache's tiles this warp's next 32 steps take, one step per lane (kNoTile: no page
  // of the cache, or behind the last key).
  uint32_t source[H];
  auto locate = [&](const Item& it, int32_t k0) {
    const int32_t* table = a.view.table + it.pair / a.row_tiles * a.view.table_stride;
    const int32_t t = it.first_tile + (k0 + static_cast<int32_t>(lane)) * kUnit;
#pragma unroll
    for (int h = 0; h < H; ++h) {
      source[h] = kNoTile;
      if (t + h >= it.t1) continue;
      const uint32_t in_table = static_cast<uint32_t>(t + h) / a.view.page_tiles;
      const uint32_t page = static_cast<uint32_t>(table[in_table]);
      if (page < a.view.pages)
        source[h] = (page * a.view.kv_heads + it.head) * a.view.page_tiles + (t + h) - in_table * a.view.page_tiles;
      else
        atomicAdd(a.view.skipped, 1ull);
    }
  };
  // The tiles of step k into its stage; one commit group per call, empty behind the last step.
  auto issue = [&](const Item& it, int32_t k) {
    if (k < it.steps) {
      if (k % 32 == 0) locate(it, k);
      const uint32_t st = static_cast<uint32_t>(k) % kStages;
      uint32_t there = 0;
#pragma unroll
      for (int h = 0; h < H; ++h) {
        const uint32_t tile = __shfl_sync(0xffffffffu, source[h], k % 32);
        if (tile == kNoTile) continue;
        there |= 1u << h;
        const uint8_t* from = a.view.data + static_cast<uint64_t>(tile) * G::kBytes + 16 * lane;
        uint8_t* to = ring + st * kStageBytes + h * G::kBytes + 16 * lane;
#pragma unroll
        for (int c = 0; c < G::kBytes; c += 512)
          if (c + 512 <= G::kBytes || c + 16 * static_cast<int>(lane) < G::kBytes) copy16(to + c, from + c);
      }
      if (lane == 0) loaded[warp][st] = there;
    }
    commit_copies();
  };
  // A warp's result lies in the last stages of its ring; the next item's first steps are on their way
  // to the stages before them while the block's warps are joined.
  constexpr int kResultStages = (kRows * D * 4 + kStageBytes - 1) / kStageBytes;
  constexpr int kAhead = kStages - kResultStages < kStages - 1 ? kStages - kResultStages : kStages - 1;
  static_assert(kAhead >= 0, "the ring holds the warp's result at the end");
  float* const mine = reinterpret_cast<float*>(ring + (kStages - kResultStages) * kStageBytes);  // [8 NT][D]

  Item item;
  bool more = open(&item, share.pair, share.head, share.offset);
  if (more)
    for (int32_t k = 0; k < kAhead; ++k) issue(item, k);
  while (more) {
    const Kv4Seq& seq = item.seq;
    const Rows& rows = item.rows;
    const uint32_t head = item.head;
    for (int32_t k = kAhead; k < kStages - 1; ++k) issue(item, k);

    // Query fragments: column g of group nt is row rows.first + 8 nt + g.
    uint32_t qf[NT][NG][2][2][QP];
    uint32_t qz[NT][2][kZeroWords];  // the sums of q over the groups, in two parts: the zeros' operand
    float kf[NT][2], zf[NT][2];  // factors of this lane's score columns 2 i4, 2 i4 + 1
    int32_t hi[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const uint32_t col = 8 * nt + g;
      float v[NG][8];
      float amax = 0.f;
      if (col < rows.count) {
        const uint32_t row = rows.first + col;
        const T* p = static_cast<const T*>(a.q) + (seq.row0 + row / a.share) * a.q_token +
                     (head * a.share + row % a.share) * a.q_head + 8 * i4;
#pragma unroll
        for (int j = 0; j < NG; ++j) load8(p + 32 * j, v[j]);
      } else {
#pragma unroll
        for (int j = 0; j < NG; ++j)
#pragma unroll
          for (int e = 0; e < 8; ++e) v[j][e] = 0.f;
      }
      float sums[NG];
      float smax = 0.f;
#pragma unroll
      for (int j = 0; j < NG; ++j) {
        float s = 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          s += v[j][e];
          amax = fmaxf(amax, fabsf(v[j][e]));
        }
        s += __shfl_xor_sync(0xffffffffu, s, 1);
        s += __shfl_xor_sync(0xffffffffu, s, 2);
        sums[j] = s;
        smax = fmaxf(smax, fabsf(s));
      }
      amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
      amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
      const float nq = pow2_toward(amax, 10), nz = pow2_toward(smax, 10);
      // The zeros' operand: slot 2 j of 16 meets the scale of group j, of which centred codes lack 8,
      // slot 2 j + 1 its zero.  Four groups (or two) fill eight slots: the sums' high part there, the low
      // part in the next eight; eight groups fill all sixteen, and the low part is a second operand.
#pragma unroll
      for (int x = 0; x < kZeroWords; ++x) {
        float mine = 0.f;
#pragma unroll
        for (int j = 0; j < 4 && j < NG; ++j)
          if (static_cast<int>(i4) == j) mine = sums[4 * x + j] * nz;
        const float lack = kCentredKeys ? 8.f * mine : 0.f;
        const uint32_t h = pack_half2(lack, mine);
        const float2 f = unpack_half2(h);
        qz[nt][0][x] = h;
        qz[nt][1][x] = pack_half2(lack - f.x, mine - f.y);
      }
      const float kfac = (kCentredKeys ? 1.f : kCodeLow) / nq * a.scale_log2, zfac = a.scale_log2 / nz;
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const int from = (2 * i4 + c) * 4;
        kf[nt][c] = __shfl_sync(0xffffffffu, kfac, from);
        zf[nt][c] = __shfl_sync(0xffffffffu, zfac, from);
        const uint32_t cc = 8 * nt + 2 * i4 + c;
        hi[nt][c] = cc < rows.count ? row_hi(a, seq, rows.first + cc) : -1;
      }
#pragma unroll
      for (int j = 0; j < NG; ++j)
#pragma unroll
        for (int m2 = 0; m2 < 2; ++m2)
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            const float f = r == 0 ? nq : nq * 0.0625f;  // the upper nibble's code is 16 times as large
            const float x = v[j][2 * m2 + r] * f, y = v[j][4 + 2 * m2 + r] * f;
            qf[nt][j][m2][r][0] = pack_half2(x, y);
            if constexpr (QP == 2) {
              const float2 h = unpack_half2(qf[nt][j][m2][r][0]);
              qf[nt][j][m2][r][1] = pack_half2(x - h.x, y - h.y);
            }
          }
    }

    float o[NT][NG][2][4];  // out^T: channels 32 j + 4 g + 2 m2 (+ 1, 16 times as large), columns 2 i4, 2 i4 + 1
    float oz[NT][4];        // the zeros' share, in the rows of their operand below (16-bit results)
    float zsum[NT][NG][2];  // the same of the zeros + 7.5 s, of this lane's tokens (fp32 results)
    float l[NT][2], m[NT][2], trigger[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        l[nt][c] = 0.f;
        m[nt][c] = 0.f;
        trigger[nt][c] = -INFINITY;
#pragma unroll
        for (int j = 0; j < NG; ++j) {
          zsum[nt][j][c] = 0.f;
#pragma unroll
          for (int e = 0; e < 4; ++e) o[nt][j][c][e] = 0.f;
        }
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) oz[nt][e] = 0.f;
    }
    // weights enter as w * pm and w * pm * s in float16: pm <= 2^11 and s <= pm_limit keep both below 2^15
    float pm = 0.f, pm_limit = -1.f;

    // One step: H tiles (key0: position of the first token; there: which of them are in the stage).
    auto step = [&](const uint8_t* stage, int32_t key0, uint32_t there, auto masked_tag) {
      constexpr bool kMasked = decltype(masked_tag)::value;
      int32_t at[H];            // position of a tile's first token; behind every key when it is not there
      bool vis[H][NT][4];
#pragma unroll
      for (int h = 0; h < H; ++h) at[h] = kMasked && !((there >> h) & 1u) ? kNowhere : key0 + 16 * h;
      // ---- scores
      float raw[H][NT][4];
#pragma unroll
      for (int h = 0; h < H; ++h) {
        const uint8_t* st = stage + h * G::kBytes;
        float zz[NT][4];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 4; ++e) raw[h][nt][e] = zz[nt][e] = 0.f;
        uint32_t w0[NG], w1[NG], p0[NG], p1[NG];
        lds(w0, st + tok_g * G::kRowBytes + i4 * 4 * NG);
        lds(w1, st + (tok_g + 8) * G::kRowBytes + i4 * 4 * NG);
        lds(p0, st + G::kKeyParams + tok_g * 4 * NG);
        lds(p1, st + G::kKeyParams + (tok_g + 8) * 4 * NG);
        uint32_t z0[kZeroWords], z1[kZeroWords];  // (s, z) of group i4 (and 4 + i4)
#pragma unroll
        for (int x = 0; x < kZeroWords; ++x) {
          const int to = G::kKeyParams + 4 * (static_cast<int>(i4) % NG) + 16 * x;
          z0[x] = *reinterpret_cast<const uint32_t*>(st + to + tok_g * 4 * NG);
          z1[x] = *reinterpret_cast<const uint32_t*>(st + to + (tok_g + 8) * 4 * NG);
        }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          if constexpr (NG == 8) {
            mma_f16(zz[nt], z0[0], z1[0], z0[1], z1[1], qz[nt][0][0], qz[nt][0][1]);
            mma_f16(zz[nt], z0[0], z1[0], z0[1], z1[1], qz[nt][1][0], qz[nt][1][1]);
          } else {
            mma_f16(zz[nt], z0[0], z1[0], z0[0], z1[0], qz[nt][0][0], qz[nt][1][0]);
          }
        }
#pragma unroll
        for (int j = 0; j < NG; ++j) {
          const uint32_t sel = (j & 1) ? 0x7632u : 0x5410u;
          uint32_t x0 = __byte_perm(w0[j / 2], w0[j / 2 + NG / 2], sel);
          uint32_t x1 = __byte_perm(w1[j / 2], w1[j / 2 + NG / 2], sel);
          float acc[NT][4];
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[nt][e] = 0.f;
#pragma unroll
          for (int m2 = 0; m2 < 2; ++m2) {
            uint32_t a0 = x0 & 0x000f000fu, a2 = x0 & 0x00f000f0u;
            uint32_t a1 = x1 & 0x000f000fu, a3 = x1 & 0x00f000f0u;
            if constexpr (kCentredKeys) {
              a0 = centred(a0, kMiddleLow), a2 = centred(a2, kMiddleHigh);
              a1 = centred(a1, kMiddleLow), a3 = centred(a3, kMiddleHigh);
            }
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
              for (int qp = 0; qp < QP; ++qp)
                mma_f16(acc[nt], a0, a1, a2, a3, qf[nt][j][m2][0][qp], qf[nt][j][m2][1][qp]);
            x0 >>= 8;
            x1 >>= 8;
          }
          const float s0 = unpack_half2(p0[j]).x, s1 = unpack_half2(p1[j]).x;
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int c = 0; c < 2; ++c) {
              raw[h][nt][c] = fmaf(s0, acc[nt][c], raw[h][nt][c]);
              raw[h][nt][2 + c] = fmaf(s1, acc[nt][2 + c], raw[h][nt][2 + c]);
            }
        }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int c = e & 1;
            float x = fmaf(raw[h][nt][e], kf[nt][c], zz[nt][e] * zf[nt][c]);
            vis[h][nt][e] = true;
            if constexpr (kMasked) {
              const int32_t pos = at[h] + tok_g + 8 * (e >> 1);
              vis[h][nt][e] = pos <= hi[nt][c] && pos >= row_lo(a, hi[nt][c]);
              if (!vis[h][nt][e]) x = -INFINITY;
            }
            raw[h][nt][e] = x;
          }
      }
      bool renew = false;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          float top = fmaxf(raw[0][nt][c], raw[0][nt][2 + c]);
          if constexpr (H == 2) top = max3(top, raw[H - 1][nt][c], raw[H - 1][nt][2 + c]);
          renew |= top > trigger[nt][c];
        }
      if (__any_sync(0xffffffffu, renew)) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            float top = fmaxf(raw[0][nt][c], raw[0][nt][2 + c]);
            if constexpr (H == 2) top = max3(top, raw[H - 1][nt][c], raw[H - 1][nt][2 + c]);
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 4));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 8));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 16));
            if (!(top > -INFINITY)) continue;  // this column still sees nothing, or nothing but NaN
            const bool first = trigger[nt][c] == -INFINITY;
            const float next = first ? top : fmaxf(m[nt][c], top);
            const float alpha = first ? 0.f : exp2_approx(m[nt][c] - next);
            m[nt][c] = next;
            trigger[nt][c] = next + kSlack;
            l[nt][c] *= alpha;
            oz[nt][c] *= alpha;
            oz[nt][2 + c] *= alpha;
#pragma unroll
            for (int j = 0; j < NG; ++j) {
              zsum[nt][j][c] *= alpha;
#pragma unroll
              for (int m2 = 0; m2 < 2; ++m2) {
                o[nt][j][m2][c] *= alpha;
                o[nt][j][m2][2 + c] *= alpha;
              }
            }
          }
      }
      // ---- weights, in place of the scores
#pragma unroll
      for (int h = 0; h < H; ++h)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            raw[h][nt][e] = exp2_approx(raw[h][nt][e] - m[nt][e & 1]);
            l[nt][e & 1] += raw[h][nt][e];
          }
      // ---- values.  Scales and zeros as a matrix: rows 2 j and 2 j + 1 are those of group j (of group
      // 4 + j from row 8 on), columns a tile's tokens.  It is the zeros' operand (16-bit results), and its
      // scale rows, dealt to all lanes, lie as the transposed weights do.
      uint32_t pa[H][4];
      [[maybe_unused]] uint32_t strange[H][4];  // kMasked: where a zero is no number
      float smax = 0.f;  // the largest scale that this lane looks at
#pragma unroll
      for (int h = 0; h < H; ++h) {
        const uint8_t* st = stage + h * G::kBytes;
#pragma unroll
        for (int r = 0; r < 4; ++r) pa[h][r] = 0u;
        if constexpr (NG == 8) {
          load_transposed(pa[h][0], pa[h][2], pa[h][1], pa[h][3],
                          st + G::kValueParams + tok_ld * 4 * NG + 16 * (lane / 16));
        } else if constexpr (NG == 4) {
          load_transposed(pa[h][0], pa[h][2], st + G::kValueParams + tok_ld * 4 * NG);
        } else if (g < 4) {
          uint32_t x[4];
#pragma unroll
          for (int r = 0; r < 4; ++r)
            x[r] = *reinterpret_cast<const uint16_t*>(st + G::kValueParams + (tok_v[r & 1] + 8 * (r >> 1)) * 4 * NG + 2 * g);
          pa[h][0] = x[0] | (x[1] << 16), pa[h][2] = x[2] | (x[3] << 16);
        }
        if constexpr (kMasked) {
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            // rows 2 i4 and 2 i4 + 1 (r < 2) of the order above, or 8 further on: zero where no row looks.
            // A zero that is no number reaches, through its codes' weights, the rows that see it
            const int32_t x = at[h] + 8 * (r >> 1) + tok_v[0], y = at[h] + 8 * (r >> 1) + tok_v[1];
            const uint32_t kept = (x >= rows.lo_min && x <= rows.hi_max ? 0xffffu : 0u) |
                                  (y >= rows.lo_min && y <= rows.hi_max ? 0xffff0000u : 0u);
            const uint32_t all = pa[h][r] & kept;
            pa[h][r] = finite_half(all & 0xffffu) | (finite_half(all >> 16) << 16);
            strange[h][r] = ((all & 0x7c00u) == 0x7c00u ? 0xffffu : 0u) | ((all & 0x7c000000u) == 0x7c000000u ? 0xffff0000u : 0u);
          }
        }
        smax = fmaxf(smax, max_half(max_half2(max_half2(pa[h][0], pa[h][2]), max_half2(pa[h][1], pa[h][3]))));
      }
      if (__any_sync(0xffffffffu, smax > (looks ? pm_limit : INFINITY))) {
        if (!looks) smax = 0.f;
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) smax = fmaxf(smax, __shfl_xor_sync(0xffffffffu, smax, d));
        // a largest scale of zero sets no measure for those to come
        const float next = fminf(pow2_toward(smax, 9), 2048.f);
        const float ratio = pm_limit < 0.f ? 0.f : next / pm;
        pm = next;
        pm_limit = smax > 0.f ? 2048.f / next : 0.f;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
          for (int j = 0; j < NG; ++j)
#pragma unroll
            for (int m2 = 0; m2 < 2; ++m2)
#pragma unroll
              for (int e = 0; e < 4; ++e) o[nt][j][m2][e] *= ratio;
#pragma unroll
          for (int e = 0; e < 4; ++e) oz[nt][e] *= ratio;
        }
      }
#pragma unroll
      for (int h = 0; h < H; ++h) {
        const uint8_t* st = stage + h * G::kBytes;
        uint32_t vw[4][NG / 2];
#pragma unroll
        for (int r = 0; r < 4; ++r)
          lds(vw[r], st + G::kValues + (tok_v[r & 1] + 8 * (r >> 1)) * G::kRowBytes + g * 2 * NG);
        if constexpr (kCentred) {  // zeros + 7.5 s, summed beside the weights and rounded to nearest
          uint32_t p0[NG], p1[NG];
          lds(p0, st + G::kValueParams + tok_g * 4 * NG);
          lds(p1, st + G::kValueParams + (tok_g + 8) * 4 * NG);
#pragma unroll
          for (int j = 0; j < NG; ++j) {
            const float2 f0 = unpack_half2(p0[j]), f1 = unpack_half2(p1[j]);
            const float z0 = fmaf(7.5f, f0.x, f0.y), z1 = fmaf(7.5f, f1.x, f1.y);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
              for (int c = 0; c < 2; ++c) {
                const float* w = raw[h][nt];
                if (vis[h][nt][c]) zsum[nt][j][c] = fmaf(w[c], z0, zsum[nt][j][c]);
                if (vis[h][nt][2 + c]) zsum[nt][j][c] = fmaf(w[2 + c], z1, zsum[nt][j][c]);
              }
          }
        }
        // w * pm in float16 and what that leaves, transposed: tokens 2 i4, 2 i4 + 1 (and 8 on) of column g
        uint32_t wh[NT][2];
        [[maybe_unused]] uint32_t wl[NT][2], seen[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            const float u = raw[h][nt][2 * r] * pm, v = raw[h][nt][2 * r + 1] * pm;
            const uint32_t x = pack_half2(u, v);
            if constexpr (PP == 2) {
              const float2 f = unpack_half2(x);
              wl[nt][r] = transpose8x8(pack_half2(u - f.x, v - f.y));
            }
            wh[nt][r] = transpose8x8(x);
            if constexpr (kMasked)
              seen[nt][r] = transpose8x8((vis[h][nt][2 * r] ? 0xffffu : 0u) | (vis[h][nt][2 * r + 1] ? 0xffff0000u : 0u));
          }
          if constexpr (!kCentred) {
            if constexpr (PP == 2) mma_f16(oz[nt], pa[h][0], pa[h][1], pa[h][2], pa[h][3], wl[nt][0], wl[nt][1]);
            mma_f16(oz[nt], pa[h][0], pa[h][1], pa[h][2], pa[h][3], wh[nt][0], wh[nt][1]);
          }
        }
#pragma unroll
        for (int j = 0; j < NG; ++j) {
          const uint32_t sel = (j & 1) ? 0x7632u : 0x5410u;
          uint32_t x01 = __byte_perm(vw[0][j / 2], vw[1][j / 2], sel);
          uint32_t x23 = __byte_perm(vw[2][j / 2], vw[3][j / 2], sel);
          uint32_t bf[NT][2][PP];
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            const uint32_t scales = __shfl_sync(0xffffffffu, pa[h][j < 4 ? 2 * r : 2 * r + 1], 8 * (j % 4) + i4);
            [[maybe_unused]] uint32_t odd = 0u;
            if constexpr (kMasked && !kCentred)
              odd = __shfl_sync(0xffffffffu, strange[h][j < 4 ? 2 * r : 2 * r + 1], 8 * (j % 4) + 4 + i4);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
              // weight * scale: the product rounded to float16, and in two parts what the rounding left,
              // exactly, plus the weight's own second part
              uint32_t x = times(wh[nt][r], scales);
              [[maybe_unused]] uint32_t rest = 0u;
              if constexpr (PP == 2) rest = times_plus(wl[nt][r], scales, times_minus(wh[nt][r], scales, x));
              if constexpr (kMasked) {
                x = ((x & ~odd) | (0x7fff7fffu & odd)) & seen[nt][r];
                rest &= ~odd & seen[nt][r];
              }
              bf[nt][r][0] = x;
              if constexpr (PP == 2) bf[nt][r][1] = rest;
            }
          }
#pragma unroll
          for (int m2 = 0; m2 < 2; ++m2) {
            uint32_t a0, a1, a2, a3;
            if constexpr (kCentred) {
              a0 = centred((x01 << 4) & 0x00f000f0u, kMiddleHalf), a1 = centred(x01 & 0x00f000f0u, kMiddleHalf);
              a2 = centred((x23 << 4) & 0x00f000f0u, kMiddleHalf), a3 = centred(x23 & 0x00f000f0u, kMiddleHalf);
              x01 >>= 8;
              x23 >>= 8;
            } else {  // the low nibble's code, and both as one byte, from which the end takes the low one
              a1 = __byte_perm(x01, 0u, m2 == 0 ? 0x4240u : 0x4341u), a0 = a1 & 0x000f000fu;
              a3 = __byte_perm(x23, 0u, m2 == 0 ? 0x4240u : 0x4341u), a2 = a3 & 0x000f000fu;
            }
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
              if constexpr (kNearest) {
                float part[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int pp = PP - 1; pp >= 0; --pp) mma_f16(part, a0, a1, a2, a3, bf[nt][0][pp], bf[nt][1][pp]);
#pragma unroll
                for (int e = 0; e < 4; ++e) o[nt][j][m2][e] += part[e];
              } else {
#pragma unroll
                for (int pp = 0; pp < PP; ++pp) mma_f16(o[nt][j][m2], a0, a1, a2, a3, bf[nt][0][pp], bf[nt][1][pp]);
              }
            }
          }
        }
      }
    };

    for (int32_t k = 0; k < item.steps; ++k) {
      issue(item, k + kStages - 1);
      wait_copies<kStages - 1>();  // this lane's share of step k
      __syncwarp();                // and every other lane's
      const uint32_t st = static_cast<uint32_t>(k) % kStages;
      const uint32_t there = loaded[warp][st];
      if (there != 0) {
        const int32_t key0 = (item.first_tile + k * kUnit) * static_cast<int32_t>(kKv4Tile);
        const uint8_t* p = ring + st * kStageBytes;
        if (there == (1u << H) - 1u && key0 >= rows.lo_max && key0 + 16 * H - 1 <= rows.hi_min)
          step(p, key0, there, std::false_type{});
        else
          step(p, key0, there, std::true_type{});
      }
      __syncwarp();  // every lane has read the stage before it is filled again
    }

    // ---- this warp's result, then the block's
    const float unit_f = pm_limit < 0.f ? 0.f : 1.f / pm;
    const float low = unit_f * (kCentred ? 0.0625f : kCodeLow), high = unit_f * (kCentred ? 0.0625f : kCodeHigh);
    __syncwarp();
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
#pragma unroll
        for (int d = 4; d < 32; d <<= 1) l[nt][c] += __shfl_xor_sync(0xffffffffu, l[nt][c], d);
        const int col = 8 * nt + 2 * static_cast<int>(i4) + c;
        // a column that saw no key; one whose scores are all NaN has l = NaN and is none
        const bool none = trigger[nt][c] == -INFINITY && l[nt][c] == 0.f;
        if (g == 0) warp_ml[warp][col] = make_float2(none ? -INFINITY : m[nt][c], l[nt][c]);
#pragma unroll
        for (int j = 0; j < NG; ++j) {
          float z;  // 16-bit results: from the rows of the zeros' accumulators
          if constexpr (kCentred) {
            z = zsum[nt][j][c];
#pragma unroll
            for (int d = 4; d < 32; d <<= 1) z += __shfl_xor_sync(0xffffffffu, z, d);
          } else {
            z = __shfl_sync(0xffffffffu, oz[nt][j < 4 ? c : 2 + c], 4 * (2 * (j % 4) + 1) + i4);
            z *= unit_f;
          }
          float2* to = reinterpret_cast<float2*>(mine + col * D + 32 * j + 4 * g);
#pragma unroll
          for (int m2 = 0; m2 < 2; ++m2)
            {
            const float lower = o[nt][j][m2][c], upper = o[nt][j][m2][2 + c] - (kCentred ? 0.f : lower);
            to[m2] = make_float2(fmaf(lower, low, z), fmaf(upper, high, z));
          }
        }
      }
    const uint64_t row0 = seq.row0;
    const uint32_t first_row = rows.first, count = rows.count;
    const bool whole = item.take == item.size;
    const uint32_t slot = blockIdx.x * 2 + (item.offset == 0 ? 1u : 0u);
    if (!whole && item.offset == 0 && threadIdx.x == 0 && a.part_o != nullptr) {
      const uint32_t last = (unit + item.size - 1) / share.per;
      a.part_of[blockIdx.x] = PartOf{min(last, gridDim.x - 1) + 1, head, first_row, count, row0};
    }
    unit += item.take;
    const bool next_pair = head + 1 == a.view.kv_heads;
    more = open(&item, item.pair + (next_pair ? 1 : 0), next_pair ? 0 : head + 1, 0);
    if (more)
      for (int32_t k = 0; k < kAhead; ++k) issue(item, k);
    __syncthreads();
    float* all = reinterpret_cast<float*>(smem + (kStages - kResultStages) * kStageBytes);
    constexpr int kWarpFloats = G::kStages * G::kBytes / 4;
    for (uint32_t e = threadIdx.x; e < count * (D / 4); e += kThreads) {
      const uint32_t col = e / (D / 4), c4 = e % (D / 4);
      float top = -INFINITY;
#pragma unroll
      for (int wi = 0; wi < kWarps; ++wi) top = fmaxf(top, warp_ml[wi][col].x);
      const float base = top == -INFINITY ? 0.f : top;
      float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
      float total = 0.f;
#pragma unroll
      for (int wi = 0; wi < kWarps; ++wi) {
        const float2 ml = warp_ml[wi][col];
        if (ml.x == -INFINITY) continue;
        const float f = exp2_approx(ml.x - base);
        const float4 x = *reinterpret_cast<const float4*>(all + wi * kWarpFloats + col * D + 4 * c4);
        total = fmaf(f, ml.y, total);
        sum.x = fmaf(f, x.x, sum.x);
        sum.y = fmaf(f, x.y, sum.y);
        sum.z = fmaf(f, x.z, sum.z);
        sum.w = fmaf(f, x.w, sum.w);
      }
      if (a.cluster != 0) {  // over the first warp's part, which no other thread reads here
        *reinterpret_cast<float4*>(all + col * D + 4 * c4) = sum;
        if (c4 == 0) block_ml[col] = make_float2(top, total);
      } else if (whole) {
        const uint32_t row = first_row + col;
        const uint64_t token = row0 + row / a.share;
        const uint32_t qh = head * a.share + row % a.share;
        const float inv = top == -INFINITY ? 0.f : 1.0f / total;
        store4(static_cast<T*>(a.out) + token * a.out_token + qh * a.out_head + 4 * c4, result<T>(sum, inv));
        if (c4 == 0 && a.lse != nullptr)
          a.lse[token * a.heads + qh] = top == -INFINITY ? -INFINITY : (top + log2f(total)) * kLn2;
      } else if (a.part_o != nullptr) {
        const uint64_t at = static_cast<uint64_t>(slot) * kRows + col;
        *reinterpret_cast<float4*>(a.part_o + at * D + 4 * c4) = sum;
        if (c4 == 0) a.part_ml[at] = make_float2(top, total);
      }
    }
    __syncthreads();  // the next item's copies overwrite what was written and read here
  }
  if (a.cluster == 0) return;
  // The cluster's blocks have their parts in shared memory; each joins its share of the item's results.
  __syncwarp();  // the barrier takes whole warps, and a block without a part comes here from a branch of its first threads
  cluster_sync();
  const uint32_t count = cluster_item.count;
  const float* const parts = reinterpret_cast<const float*>(smem + (kStages - kResultStages) * kStageBytes);
  for (uint32_t e = cluster_cta_rank() * kThreads + threadIdx.x; e < count * (D / 4); e += a.cluster * kThreads) {
    const uint32_t col = e / (D / 4), c4 = e % (D / 4);
    float2 ml[kMaxCluster];
    float4 x[kMaxCluster];
    float top = -INFINITY;
#pragma unroll
    for (uint32_t r = 0; r < kMaxCluster; ++r) {
      ml[r] = make_float2(-INFINITY, 0.f);
      if (r >= a.cluster) continue;
      ml[r] = ld_cluster_v2(cluster_smem_addr(block_ml + col, r));
      x[r] = ld_cluster_v4(cluster_smem_addr(parts + col * D + 4 * c4, r));
    }
#pragma unroll
    for (uint32_t r = 0; r < kMaxCluster; ++r) top = fmaxf(top, ml[r].x);
    const float base = top == -INFINITY ? 0.f : top;
    float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
    float total = 0.f;
#pragma unroll
    for (uint32_t r = 0; r < kMaxCluster; ++r) {
      if (ml[r].x == -INFINITY) continue;  // what such a block holds is no part
      const float f = exp2_approx(ml[r].x - base);
      total = fmaf(f, ml[r].y, total);
      sum.x = fmaf(f, x[r].x, sum.x);
      sum.y = fmaf(f, x[r].y, sum.y);
      sum.z = fmaf(f, x[r].z, sum.z);
      sum.w = fmaf(f, x[r].w, sum.w);
    }
    const uint32_t row = cluster_item.first + col;
    const uint64_t token = cluster_item.row0 + row / a.share;
    const uint32_t qh = cluster_item.head * a.share + row % a.share;
    const float inv = top == -INFINITY ? 0.f : 1.0f / total;
    store4(static_cast<T*>(a.out) + token * a.out_token + qh * a.out_head + 4 * c4, result<T>(sum, inv));
    if (c4 == 0 && a.lse != nullptr) a.lse[token * a.heads + qh] = top == -INFINITY ? -INFINITY : (top + log2f(total)) * kLn2;
  }
  __syncwarp();
  cluster_sync();  // no block's shared memory goes before the others have read it
}

// Joins the parts of every item that was split: block x looks at what block x of the first kernel
// began and did not finish, whose other parts lie in slot 0 of the blocks behind it; grid y deals out
// the channels.  The parts of a (row, four channels) are dealt to `lanes` threads and what they make
// of them is joined in a fixed order.
constexpr int kJoinThreads = 256;

template <typename T, int D, int kJoinColumns>  // float4 columns of a row per block
__global__ void __launch_bounds__(kJoinThreads) kv4_join_kernel(const KernelArgs a, uint32_t rows_per_tile) {
  constexpr uint32_t kWho = kJoinThreads / kJoinColumns;  // threads over (row, part)
  __shared__ float4 part[kJoinThreads];
  __shared__ float2 part_ml[kWho];
  griddep_wait();
  const PartOf of = a.part_of[blockIdx.x];
  if (of.last1 == 0u) return;
  const uint32_t parts = of.last1 - blockIdx.x;
  const uint32_t c4 = threadIdx.x % kJoinColumns, who = threadIdx.x / kJoinColumns;
  const uint32_t channel = 4 * (blockIdx.y * kJoinColumns + c4);
  uint32_t lanes = kWho;  // threads per row: a power of two
  while (lanes > 1 && lanes * of.count > kWho) lanes >>= 1;
  const uint32_t sub = who % lanes;
  for (uint32_t r0 = 0; r0 < of.count; r0 += kWho / lanes) {
    const uint32_t col = r0 + who / lanes;
    float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
    float2 ml = make_float2(-INFINITY, 0.f);
    auto add = [&](float2 n, float4 x) {
      const float top = fmaxf(ml.x, n.x), base = top == -INFINITY ? 0.f : top;
      const float f = exp2_approx(ml.x - base), g = exp2_approx(n.x - base);
      ml = make_float2(top, fmaf(f, ml.y, g * n.y));
      sum.x = fmaf(f, sum.x, g * x.x);
      sum.y = fmaf(f, sum.y, g * x.y);
      sum.z = fmaf(f, sum.z, g * x.z);
      sum.w = fmaf(f, sum.w, g * x.w);
    };
    if (col < of.count) {
      auto place = [&](uint32_t p) {
        return (static_cast<uint64_t>(blockIdx.x + p) * 2 + (p == 0 ? 1u : 0u)) * rows_per_tile + col;
      };
      uint32_t p = sub;
      for (; p + 3 * lanes < parts; p += 4 * lanes) {  // four parts' loads together
        float2 n[4];
        float4 x[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint64_t at = place(p + i * lanes);
          n[i] = a.part_ml[at];
          x[i] = *reinterpret_cast<const float4*>(a.part_o + at * D + channel);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) add(n[i], x[i]);
      }
      for (; p < parts; p += lanes) {
        const uint64_t at = place(p);
        add(a.part_ml[at], *reinterpret_cast<const float4*>(a.part_o + at * D + channel));
      }
    }
    part[threadIdx.x] = sum;
    if (c4 == 0) part_ml[who] = ml;
    __syncthreads();
    if (col < of.count && sub == 0) {
      for (uint32_t i = 1; i < lanes; ++i) add(part_ml[who + i], part[threadIdx.x + i * kJoinColumns]);
      const uint32_t row = of.first + col;
      const uint64_t token = of.row0 + row / a.share;
      const uint32_t qh = of.head * a.share + row % a.share;
      const float inv = ml.x == -INFINITY ? 0.f : 1.0f / ml.y;
      store4(static_cast<T*>(a.out) + token * a.out_token + qh * a.out_head + channel, result<T>(sum, inv));
      if (channel == 0 && a.lse != nullptr)
        a.lse[token * a.heads + qh] = ml.x == -INFINITY ? -INFINITY : (ml.x + log2f(ml.y)) * kLn2;
    }
    __syncthreads();
  }
}

template <typename T, int D, int kJoinColumns>
cudaError_t launch_join(const KernelArgs& a, const Kv4Plan& plan, cudaStream_t stream) {
  return launch_dependent(kv4_join_kernel<T, D, kJoinColumns>, dim3(plan.blocks, D / 4 / kJoinColumns), kJoinThreads, 0,
                          stream, 0, a, plan.row_tile);
}

template <typename T> constexpr int kQueryParts = sizeof(T) == 4 ? 2 : 1;
template <typename T, int D, int NT>
cudaError_t launch(const KernelArgs& a, const Kv4Plan& plan, cudaStream_t stream) {
  using G = Geometry<D>;
  constexpr int QP = kQueryParts<T>;
  constexpr int PP = std::is_same<T, __nv_bfloat16>::value ? 1 : 2;
  constexpr size_t kSmem = static_cast<size_t>(kWarps) * G::kStages * G::kBytes;
  const auto kernel = kv4_attention_kernel<T, D, NT, QP, PP>;
  // the attributes stay with the device's function, and so does the largest cluster that it has room for (a
  // part of a GPU may have less than all of one): set and asked once on each
  static std::atomic<uint32_t> most[64];
  int device = 0;
  cudaError_t e = cudaGetDevice(&device);
  if (e != cudaSuccess) return e;
  uint32_t fits = device < 64 ? most[device].load(std::memory_order_acquire) : 0;
  if (fits == 0) {
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(kSmem));
    if (e != cudaSuccess) return e;
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    if (e != cudaSuccess) return e;
    fits = kv4_cluster_to_launch(kMaxCluster, [&](uint32_t n) { return has_room(kernel, kThreads, kSmem, n); });
    if (device < 64) most[device].store(fits, std::memory_order_release);
  }
  uint32_t blocks = plan.blocks;
  KernelArgs args = a;
  if (plan.cluster > fits) {
    args.cluster = fits;
    blocks = plan.blocks / plan.cluster * fits;
  }
  e = launch_dependent(kernel, dim3(blocks), kThreads, kSmem, stream, args.cluster, args);
  if (e != cudaSuccess || plan.workspace == 0) return e;
  // Few items have many parts each: narrower blocks give a row's parts to more threads (8 items of 54
  // parts: 55 us against 58 of the whole call).  Many items have a few: fewer blocks start faster (439
  // cut items: 128 us against 131).
  return a.view.batch * a.view.kv_heads * a.row_tiles < 64 ? launch_join<T, D, 8>(a, plan, stream)
                                                           : launch_join<T, D, 16>(a, plan, stream);
}

template <typename T, int D>
cudaError_t dispatch(const KernelArgs& a, const Kv4Plan& plan, cudaStream_t stream) {
  switch (plan.row_tile) {
    case 8: return launch<T, D, 1>(a, plan, stream);
    case 16:
      if constexpr (kMaxRowGroups<D> >= 2) return launch<T, D, 2>(a, plan, stream);
      return cudaErrorInvalidValue;
    case 32:
      if constexpr (kMaxRowGroups<D> >= 4) return launch<T, D, 4>(a, plan, stream);
      return cudaErrorInvalidValue;
    default: return cudaErrorInvalidValue;
  }
}

template <typename T>
cudaError_t dispatch_dim(const KernelArgs& a, const Kv4Plan& plan, cudaStream_t stream) {
  switch (a.view.dim) {
    case 64: return dispatch<T, 64>(a, plan, stream);
    case 128: return dispatch<T, 128>(a, plan, stream);
    case 256: return dispatch<T, 256>(a, plan, stream);
    default: return cudaErrorInvalidValue;
  }
}

}  // namespace

bool kv4_attention_supported(uint32_t dim) { return dim == 64 || dim == 128 || dim == 256; }

Kv4Plan kv4_attention_plan(uint32_t dim, uint32_t kv_heads, uint32_t heads, uint32_t batch, uint32_t max_tokens,
                           uint32_t max_kv_len, uint32_t window, ElementType type) {
  Kv4Plan p;
  const uint64_t share = heads / kv_heads, rows = static_cast<uint64_t>(max_tokens) * share;
  const uint32_t most = dim == 64 ? 8 * kMaxRowGroups<64> : 8 * (dim == 128 ? kMaxRowGroups<128> : kMaxRowGroups<256>);
  p.row_tile = 8;
  while (p.row_tile < most && p.row_tile < rows) p.row_tile *= 2;
  p.row_tiles = (rows + p.row_tile - 1) / p.row_tile;
  // Most tiles that an item's rows see: those of the longest sequence the call allows, or of the window
  // and the tokens whose rows share the item, wherever that begins in a tile.
  uint64_t tiles = (static_cast<uint64_t>(max_kv_len) + kKv4Tile - 1) / kKv4Tile;
  if (window > 0) {
    const uint64_t tokens = std::min<uint64_t>(max_tokens, (p.row_tile + share - 2) / share + 1);
    tiles = std::min(tiles, (window + tokens - 2) / kKv4Tile + 2);
  }
  const uint64_t unit = kWarps * tiles_per_step(static_cast<int>(dim), static_cast<int>(p.row_tile / 8));
  const uint64_t item = tiles <= unit ? 1 : (tiles + unit - 1) / unit;
  const uint64_t items = static_cast<uint64_t>(batch) * kv_heads * p.row_tiles;
  const uint64_t resident = 148ull * blocks_per_sm(static_cast<int>(dim), static_cast<int>(p.row_tile / 8));
  p.run = items * (item + kItemCost);
  // Few items of a few units: a cluster of blocks for each, which joins it in shared memory, needs no
  // workspace and looks at no other sequence's length.
  if (item > 1 && 2 * items <= resident) {
    uint64_t cluster = 2;
    // a cluster's blocks share a GPC, of whose places clusters of 8 and 16 may leave some empty
    auto room = [&](uint64_t c) { return c > 4 ? resident / 4 * 3 : resident; };
    while (cluster < kMaxCluster && cluster < item && 2 * cluster * items <= room(2 * cluster)) cluster *= 2;
    if (item <= cluster * cluster_units(type)) {
      p.cluster = static_cast<uint32_t>(cluster);
      p.blocks = static_cast<uint32_t>(items * cluster);
      return p;
    }
  }
  // Else one wave: as many blocks as the SMs hold, each with an equal share of the units, or a block per
  // unit where there are fewer.
  p.blocks = static_cast<uint32_t>(items >= resident || items * (item + 1) >= resident ? resident : items * (item + 1));
  // an item of one unit is never split
  if (item > 1)
    p.workspace = static_cast<uint64_t>(p.blocks) * (2 * p.row_tile * (static_cast<uint64_t>(dim) * 4 + 8) + sizeof(PartOf));
  return p;
}

cudaError_t kv4_attention(const Kv4AttnArgs& in, const Kv4Plan& plan, cudaStream_t stream) {
  if (in.view.batch == 0 || in.view.tokens == 0 || in.view.max_tokens == 0) return cudaSuccess;
  KernelArgs a{};
  a.view = in.view;
  a.q = in.q;
  a.out = in.out;
  a.q_token = in.q_token;
  a.q_head = in.q_head;
  a.out_token = in.out_token;
  a.out_head = in.out_head;
  a.lse = in.lse;
  a.scale_log2 = in.scale * kLog2e;
  a.heads = in.heads;
  a.share = in.heads / in.view.kv_heads;
  a.causal = in.causal ? 1 : 0;
  a.window = in.window;
  a.row_tiles = static_cast<uint32_t>(plan.row_tiles);
  a.cluster = plan.cluster;
  if (plan.workspace > 0) {
    const uint64_t parts = 2ull * plan.blocks * plan.row_tile;
    a.part_o = static_cast<float*>(in.workspace);
    a.part_of = reinterpret_cast<PartOf*>(a.part_o + parts * in.view.dim);
    a.part_ml = reinterpret_cast<float2*>(a.part_of + plan.blocks);
  }
  switch (in.type) {
    case kF32: return dispatch_dim<float>(a, plan, stream);
    case kBf16: return dispatch_dim<__nv_bfloat16>(a, plan, stream);
    default: return dispatch_dim<__half>(a, plan, stream);
  }
}

}  // namespace oct
