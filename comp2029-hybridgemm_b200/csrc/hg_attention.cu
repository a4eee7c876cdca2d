// Attention of one new token a sequence over the paged MXFP8 cache, split over the cache's length and joined.
//
//   s_t = scale q . k_t      p_t = exp(s_t - max s)      out = sum_t p_t v_t / sum_t p_t
//
// One pass over the cache with a running maximum and sum, in one launch.  A unit of work is a sequence, a kv head and up to eight of its
// query heads.  A block takes a run of a unit's 16-token tiles, and each of its warps every fourth (or twelfth) of these; sums of warps
// meet in shared memory, of blocks there or in a workspace.  A tile comes in by TMA, a few tiles ahead, into a ring that the warp has for
// itself, and goes from there into the fragments of two matrix products,
//   S^T [16 tokens, 8 heads]     = K [16 tokens, d]   Q^T [d, 8 heads]       (m16n8k16, one accumulator for every scale group of 32 d)
//   O^T [16 d, 8 heads]          = V^T [16 d, tokens] P^T [tokens, 8 heads]
// so that the heads fill the narrow side of an instruction, whatever their number, and the cache its wide one.  (tcgen05 would
// take 128 rows where there are eight heads, and has no operand for scales along the summed axis of the second product; E4M3
// operands of mma.sync are converted by instructions too here.)  Codes become halves, which hold them exactly.  Scales stay outside:
// those of the keys multiply a group's partial sum, those of the values the probabilities, once for every group, before these are
// rounded to halves.
//
// What bounds it: bytes of the cache, and nearly as soon a warp's way through a tile (about 445 instructions for 4224 bytes, issued in half
// of the slots, with the ALU pipe busy as long; from L2 an SM keeps up with some 24 bytes a clock, and memory delivers 23.6).  28 heads on 4 of 128, bf16: 128 sequences of 1024 to 1150 tokens
// 32.6 us (0.70 of the measured copy rate), 128 x 4000 about 94 us (0.89), 4 x 32768 30.6 us (0.69); 1 x 1000 5.4 us, of which launch, three
// dependent loads and two meetings of blocks are all but 0.2.  (Where two sides are compared below, both are from before values were summed under a
// scale for each group, which adds 1 to 3 % to either.)
//
// Roundings: q keeps its 16 bits (a head's bf16 queries become halves under a power of two, which keeps eight bits of all that is
// not 2^-29 of the largest).  P times the scale of its values is rounded to 11 bits (2^-11 of it at most) where it is 2^-21 or more of the largest
// weight times the largest scale of its head and group so far, and off by up to 2^-32 of these where it is less: a bias of 2^7, a power of two for
// each group and lazy rescaling hold it in the range of a half.  Weights are exponentials by ex2.approx (two units of fp32).  Sums, maxima and outputs
// are fp32.  Where the output is quantised (EXACT) what the rounding of P left goes through a second product: an output beside the border of two scales
// changes the codes of its whole group, and a rounding to 16 bits no longer hides the difference.  (37 sequences, values of
// the codes against 64-bit arithmetic, relative: 0.015 with one product; with two, in five draws, 4e-20 to 3e-5, fp32 arithmetic 8e-8 to 1e-2: single
// codes beside a border, on either side.)
#include <algorithm>
#include <atomic>
#include <cmath>
#include <cstring>
#include <mutex>
#include <type_traits>

#include "hg_cache.cuh"
#include "hg_gemm_cluster.cuh"
#include "hg_tags.cuh"

namespace hg {
namespace {

constexpr int kTile = 16;            // tokens of a step of one warp
constexpr int kHeadTile = 8;         // query heads of a unit
constexpr int kWarps = 4, kWideWarps = 12;   // of a block; of one that has an SM for itself
constexpr int kMostRing = 4;        // tiles of a warp in shared memory or on their way there, at most
constexpr int kBlocksPerSm = 4, kLineBlocksPerSm = 3;   // of kWarps; of a line of no more units than that
constexpr int kWhole = 16;           // sequences of no more tiles are not split
// Costs in tiles.  A unit has one beside its tiles, by the warps that share these (16 for both: 37 of 1 to 4099 tokens on three blocks an SM 17.4
// us for 17.05; 16 of 10 to 16000 on wide ones 19.3 for 17.4), units that are split have kSplitCost (in a block of kWarps), and a block takes at
// least kLeastShare (40: 37 of 1 to 4099 18.4 us).
constexpr int kSplitCost = 28, kLeastShare = 24;
__host__ __device__ constexpr int unit_cost(int warps) { return warps == kWarps ? 12 : 24; }
// Tiles of all units up to which they are left to clusters: kFew where the clusters fill less than three quarters of the device, kMuch
// otherwise.  A cluster's blocks take equal parts of one unit, so the longest unit sets the time; a line has a slower beginning and end.
// Cluster and line, us, 4 kv heads of 128: 1 x 8000 tokens 8.3, 11.1; 1 x 32000 16.6, 16.7; 4 x 4000 12.1, 12.6; 4 x 16000 28.1, 19.4; 4 x 32768 50.5,
// 30.3; 8 x 4000 12.8, 15.0, 8 of 10 to 4000 10.3, 10.4; 8 x 16000 27.8, 29.7, 8 of 10 to 16000 26.4, 14.6; 16 x 2000 13.1, 16.2, 16 of 10 to
// 2000 8.8, 10.4; 36 x 4000 28.8, 28.6, 36 of 10 to 4000 25.0, 15.9.
constexpr int kFew = 6144, kMuch = 18432;
// Clusters of 1, 2, 4, 8 and 16 blocks that a device holds at once, per thousand SMs: blocks of kWarps (whose SMs hold several), and of
// kWideWarps.  GPCs differ in their SMs, so it is not a matter of division (148 SMs: 592, 296, 142, 71 and 31; 148, 74, 33, 15 and 7).
constexpr int kHeld[2][5] = {{4000, 2000, 959, 479, 209}, {1000, 500, 222, 101, 47}};
constexpr int kTableLines = 8192;    // lines of the table that are prefetched, at most: it may be far wider than its sequences
constexpr int kSmBytes = 228 << 10;  // shared memory of an SM
constexpr float kBias = 7.f, kSlack = 4.f;   // P is kept in [0, 2^(kBias + 2 kSlack)]
constexpr float kNone = -3e38f;      // maximum of nothing
constexpr int kLeastScale = 24, kMostScale = 250;   // values are summed under 2^-103 at least and 2^123 at most (bytes of E8M0)
constexpr uint32_t kZeros = 0x7f7f7f7fu;   // scale bytes of groups of zeros

// How units come to blocks.  Few units (CLUSTER): a cluster of `split` blocks each, whose sums meet in shared memory.  Many (LINE):
// the work is a line on which every unit (sequence and head unit, in this order) has its tiles behind what it costs
// besides, and a block takes an equal share of it, so whatever the lengths all blocks end together.  A unit that ends in another
// block than it begins in is added up by the one that it begins in, which comes to it last; the others come to their
// parts of it first, write their sums to a slot and set a tag behind them, and the first one waits for the tags and takes them back.
// It waits for blocks behind it alone, whose first parts wait for nothing, so the wait ends even where the device holds fewer blocks
// than there are: all but one of them end.  A tag is 64 bits that a workspace holds by accident once in 2^64 slots, so that
// it needs no clearing before a launch.  Every call has its own one; replays of a captured one share it, and find it taken back, where a wait was
// given up too (hg_tags.cuh).
constexpr uint64_t kTag = 0x9d3f6ac1e57b2481ull;

struct AttentionParams {
  hg_cache cache;
  hg_attention_call call;
  float* partial;       // LINE: [blocks][kHeadTile][head_dim + 2]: sums, maximum, sum of weights of a block's first part
  uint64_t* tags;       // LINE: [blocks]
  uint64_t tag;
  int least, more;      // LINE: units of a block, and blocks that have one more
  float by_blocks;      // LINE: 1 / blocks, rounded up
  int table_lines;      // 128-byte lines of a row of the table that are prefetched
  int head_units;       // kv heads x chunks of kHeadTile heads
  int chunks, group;
  int split;            // CLUSTER: blocks of a unit, 1, 2, 4, 8 or 16
  int ring;             // tiles of a warp in shared memory or on their way there
  uint32_t page_tiles, by_page_tiles;   // tiles of a page, and ceil(2^32 / page_tiles)
};

__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// The same on a sum of zero, which then takes no registers before.
__device__ __forceinline__ void mma_f16_first(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};"
               : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t v) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}
__device__ __forceinline__ uint32_t half2_bits(float low, float high) {
  const __half2 h = __floats2half2_rn(low, high);
  return *reinterpret_cast<const uint32_t*>(&h);
}
// 2^(byte - 127) of a pair of bytes, as bf16, and of one of them.
__device__ __forceinline__ uint32_t two_scales(uint32_t bytes) {
  uint32_t r;
  asm("cvt.rn.bf16x2.ue8m0x2 %0, %1;" : "=r"(r) : "h"(uint16_t(bytes)));
  return r;
}
__device__ __forceinline__ float scale_of(uint32_t pair, int g) { return __uint_as_float(g & 1 ? pair & 0xffff0000u : pair << 16); }
__device__ __forceinline__ uint32_t max_pairs(uint32_t a, uint32_t b) {
  const __nv_bfloat162 m = __hmax2(*reinterpret_cast<const __nv_bfloat162*>(&a), *reinterpret_cast<const __nv_bfloat162*>(&b));
  return *reinterpret_cast<const uint32_t*>(&m);
}
__device__ __forceinline__ uint32_t min_pairs(uint32_t a, uint32_t b) {
  const __nv_bfloat162 m = __hmin2(*reinterpret_cast<const __nv_bfloat162*>(&a), *reinterpret_cast<const __nv_bfloat162*>(&b));
  return *reinterpret_cast<const uint32_t*>(&m);
}
__device__ __forceinline__ uint32_t mul_pairs(uint32_t a, uint32_t b) {
  const __nv_bfloat162 m = __hmul2(*reinterpret_cast<const __nv_bfloat162*>(&a), *reinterpret_cast<const __nv_bfloat162*>(&b));
  return *reinterpret_cast<const uint32_t*>(&m);
}
// 2^(byte - 127) twice, and the inverse of a pair of powers of two.
__device__ __forceinline__ constexpr uint32_t pair_of(int byte) { return uint32_t(byte) * 0x00800080u; }
__device__ __forceinline__ uint32_t inverse_pair(uint32_t a) { return pair_of(254) - a; }
__device__ __forceinline__ float power_of(int biased) { return __uint_as_float(uint32_t(biased) << 23); }

__device__ __forceinline__ uint4 shared_16(uint32_t at) {
  uint4 v;
  asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at) : "memory");
  return v;
}
__device__ __forceinline__ uint2 shared_8(uint32_t at) {
  uint2 v;
  asm volatile("ld.shared.v2.b32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(at) : "memory");
  return v;
}
__device__ __forceinline__ uint32_t shared_4(uint32_t at) {
  uint32_t v;
  asm volatile("ld.shared.b32 %0, [%1];" : "=r"(v) : "r"(at) : "memory");
  return v;
}

// Tiles that sequence i has to look at: from .. to - 1 hold positions first .. length - 1.
struct Span { int first, length, from, to; };
__device__ __forceinline__ Span span_of(const AttentionParams& p, int i) {
  Span s;
  s.length = min(max(p.call.lengths[i], 0), p.call.table_width * p.cache.page_size);
  s.first = p.call.window ? max(0, s.length - p.call.window) : 0;
  s.from = s.first / kTile;
  s.to = s.length > 0 ? (s.length + kTile - 1) / kTile : s.from;
  return s;
}

// Sums of what the block's threads give, of all and of those up to this one.
struct Sums { int64_t all, upto; };
template <int WARPS>
__device__ __forceinline__ Sums block_sums(int64_t v, int64_t* parts) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int step = 1; step < 32; step <<= 1) {
    const int64_t other = __shfl_up_sync(0xffffffffu, v, step);
    if (lane >= step) v += other;
  }
  __syncthreads();
  if (lane == 31) parts[warp] = v;
  __syncthreads();
  Sums s{0, v};
#pragma unroll
  for (int i = 0; i < WARPS; ++i) {
    if (i < warp) s.upto += parts[i];
    s.all += parts[i];
  }
  return s;
}

// Codes of 32 elements (4 of a lane, 8 lanes) of one head of a row, and their scale.
__device__ __forceinline__ void store_packed(const AttentionParams& p, int seq, int head, int head_dim, int g, int x, const float (&v)[4], unsigned mask) {
  float amax = fmaxf(fmaxf(fabsf(v[0]), fabsf(v[1])), fmaxf(fabsf(v[2]), fabsf(v[3])));
#pragma unroll
  for (int step = 1; step < 8; step <<= 1) amax = fmaxf(amax, __shfl_xor_sync(mask, amax, step));
  const int e = mx_exponent<false>(amax);
  const float inv = mx_inverse_scale(e);
  const int k = p.call.heads * head_dim, col = head * head_dim + 32 * g;
  *reinterpret_cast<uint32_t*>(static_cast<uint8_t*>(p.call.codes) + int64_t(seq) * k + col + 4 * x) =
      cvt_e4m3x2(v[0] * inv, v[1] * inv) | (cvt_e4m3x2(v[2] * inv, v[3] * inv) << 16);
  if (x == 0) static_cast<uint8_t*>(p.call.scales)[scale_word_offset(seq, col >> 7, k) + ((col >> 5) & 3)] = uint8_t(e + 127);
}

// Four elements of a head from element d on, of their weighted sums, the sum of weights and its maximum; all eight lanes of a group of 32
// elements are here.
template <typename T, int GROUPS>
__device__ __forceinline__ void write_out(const AttentionParams& p, int seq, int head, int d, const float4& sum, float l, float m) {
  constexpr int kDim = 32 * GROUPS;
  const float inv = 1.f / l;
  float v[4] = {sum.x * inv, sum.y * inv, sum.z * inv, sum.w * inv};
  if (l == 0.f) v[0] = v[1] = v[2] = v[3] = 0.f;
  if (p.call.codes) store_packed(p, seq, head, kDim, d >> 5, (d >> 2) & 7, v, 0xffu << (threadIdx.x & 24));
  else
    *reinterpret_cast<uint2*>(static_cast<uint16_t*>(p.call.out) + (int64_t(seq) * p.call.heads + head) * kDim + d) =
        make_uint2(uint32_t(from_float<T>(v[0])) | (uint32_t(from_float<T>(v[1])) << 16), uint32_t(from_float<T>(v[2])) | (uint32_t(from_float<T>(v[3])) << 16));
  if (p.call.lse && d == 0) p.call.lse[int64_t(seq) * p.call.heads + head] = l == 0.f ? -INFINITY : (m + log2f(l)) * 0.69314718f;
}

// Adds the sums of `count` other blocks, in their order, to m, l and sum; `load(j, sums, {maximum, weight})` for some of them together.
template <int kMeet, typename Load>
__device__ __forceinline__ void meet(int count, float& m, float& l, float4& sum, Load load) {
  for (int first = 0; first < count; first += kMeet) {
    float4 x[kMeet];
    float2 y[kMeet];
#pragma unroll
    for (int j = 0; j < kMeet; ++j) load(min(first + j, count - 1), x[j], y[j]);
    const float before = m;
#pragma unroll
    for (int j = 0; j < kMeet; ++j) m = fmaxf(m, y[j].x);
    const float shrink = exp2_fast(before - m);
    l *= shrink;
    sum.x *= shrink; sum.y *= shrink; sum.z *= shrink; sum.w *= shrink;
#pragma unroll
    for (int j = 0; j < kMeet; ++j) {
      if (first + j >= count) continue;
      const float factor = exp2_fast(y[j].x - m);
      l += y[j].y * factor;
      sum.x += x[j].x * factor; sum.y += x[j].y * factor; sum.z += x[j].z * factor; sum.w += x[j].w * factor;
    }
  }
}

struct TagWord {
  uint64_t* at;
  // Until the tag is set; what was written before it is then visible.  False when it is not within about two seconds.
  __device__ __forceinline__ bool wait(uint64_t tag) const {
    const long long start = clock64();
    for (uint32_t spin = 1;; ++spin) {
      uint64_t now;
      asm volatile("ld.acquire.gpu.global.u64 %0, [%1];" : "=l"(now) : "l"(at) : "memory");
      if (now == tag) return true;
      if ((spin & 63u) == 0) {
        __nanosleep(100);
        if (clock64() - start > kWaitLimitCycles) return false;
      }
    }
  }
  // What was written before it is visible to whoever finds `to`.
  __device__ __forceinline__ uint64_t exchange(uint64_t to) const {
    uint64_t before;
    asm volatile("fence.acq_rel.gpu;\n atom.relaxed.gpu.global.exch.b64 %0, [%1], %2;" : "=l"(before) : "l"(at), "l"(to) : "memory");
    return before;
  }
  __device__ __forceinline__ void store(uint64_t to) const { asm volatile("st.relaxed.gpu.global.u64 [%0], %1;" ::"l"(at), "l"(to) : "memory"); }
};

// Whether sums have a place of their own on a line, so that the next unit's first tiles and queries come in while one's are added up: where three
// tiles to a warp are left beside them (4 x 32768 tokens 31.9 -> 30.3 us, 16 of 10 to 16000 22.6 -> 19.3, 37 of 1 to 4099 18.0 -> 17.4, 64 x 500 14.65 ->
// 14.1).
__host__ __device__ constexpr bool apart(int head_dim, int per_sm) { return head_dim == 64 || per_sm < kBlocksPerSm; }

// Shared memory of a block.  A tile of keys or values is 16 rows of head_dim bytes, whose 16-byte chunks the copy swizzles (with the
// period of 128-byte rows, or of 64-byte ones).  The warps' sums take the place of the rings when these are idle, or (apart)
// have their own, so that the next unit's first tiles come in meanwhile.
template <int GROUPS, int WARPS>
struct Shared {
  static constexpr int kDim = 32 * GROUPS, kCodes = kTile * kDim, kScales = kTile * 2 * GROUPS, kRow = kDim + 4;
  static constexpr int kStage = 2 * kCodes + kScales;   // of a warp
  static constexpr int kSums = WARPS * kHeadTile * kRow * 4;
  static constexpr int bytes(int ring, bool apart) {
    return (apart ? WARPS * ring * kStage + kSums : (WARPS * ring * kStage > kSums ? WARPS * ring * kStage : kSums)) + 1024;   // the beginning is brought to a multiple of 1024
  }
};
// Row r of a fragment's eight holds this token: two rows that are read in one pass, r and r ^ 1, then have their chunks in different
// banks, and so have the four tokens 2c that lanes read values of in one pass.
__device__ __forceinline__ int token_of(int r) { return r ^ ((r & 1) << 2); }
// Byte of a tile's 16-byte chunk.
template <int GROUPS>
__device__ __forceinline__ uint32_t chunk_at(int token, int chunk) {
  return uint32_t(token * 32 * GROUPS + ((chunk ^ (GROUPS == 4 ? token & 7 : (token >> 1) & 3)) << 4));
}

template <typename T, int GROUPS, int WARPS, int PER_SM, bool LINE, bool EXACT>
__global__ void __launch_bounds__(WARPS * 32, PER_SM)
attention_kernel(const __grid_constant__ AttentionParams p, const __grid_constant__ CUtensorMap map) {
  using S = Shared<GROUPS, WARPS>;
  constexpr int kDim = 32 * GROUPS, kThreads = WARPS * 32;
  constexpr int kUnitCost = unit_cost(WARPS);
  constexpr bool kApart = LINE && apart(kDim, PER_SM);
  extern __shared__ uint8_t dynamic[];
  __shared__ int given_up, there[WARPS][kMostRing];
  __shared__ float weights[WARPS][kHeadTile], maxima[WARPS][kHeadTile];
  __shared__ alignas(8) float2 block_weights[kHeadTile];   // maximum and sum of weights of the block
  __shared__ uint64_t full[WARPS][kMostRing];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, r = lane >> 2, c = lane & 3;
  const int ring = p.ring;
  const uint32_t base = (smem_u32(dynamic) + 1023u) & ~1023u, all_scales = base + uint32_t(WARPS * ring) * (2 * S::kCodes), bars = smem_u32(&full[warp][0]);
  float (*const sums)[kHeadTile][S::kRow] = reinterpret_cast<float (*)[kHeadTile][S::kRow]>(dynamic + (base - smem_u32(dynamic)) + (kApart ? WARPS * ring * S::kStage : 0));
  if (lane < p.ring) mbar_init(bars + 8 * lane, 1);
  if (threadIdx.x == 0) {
    given_up = 0;
    asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&map)) : "memory");
  }
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  __syncthreads();
  // Lengths and tables come as far as L2 while the kernel in front ends (from cold memory 4 x 32768 tokens took 31.8 us for 32.2 without);
  // what they hold is read behind the wait.
  {
    const unsigned at = blockIdx.x * kThreads + threadIdx.x, row = at / unsigned(p.table_lines), col = (at - row * p.table_lines) * 32;
    if (threadIdx.x * 32 < p.call.seqs) asm volatile("prefetch.global.L2 [%0];" ::"l"(p.call.lengths + threadIdx.x * 32));
    if (row < unsigned(p.call.seqs) && col < unsigned(p.call.table_width))
      asm volatile("prefetch.global.L2 [%0];" ::"l"(p.call.table + int64_t(row) * p.call.table_stride + col));
  }
  // Loads below are ordinary ones: the kernel in front may still be writing the cache when this one starts, so the data is not
  // read-only for its duration.
  pdl_wait();
  pdl_trigger();

  // Padding of the scale buffer behind the last sequence.
  if (p.call.codes) {
    const int k = p.call.heads * kDim, kblocks = k >> 7, pad_rows = ((p.call.seqs + 127) & ~127) - p.call.seqs;
    for (int64_t i = int64_t(blockIdx.x) * kThreads + threadIdx.x; i < int64_t(pad_rows) * kblocks; i += int64_t(gridDim.x) * kThreads)
      *reinterpret_cast<uint32_t*>(static_cast<uint8_t*>(p.call.scales) + scale_word_offset(p.call.seqs + int(i / kblocks), int(i % kblocks), k)) = 0x7f7f7f7fu;
  }

  // The block's units.
  int seq, offset = 0;                     // LINE: `offset` in the units of sequence `seq`, `remaining` of its share of the line, `position` on it
  int64_t remaining = 1, share = 1, position = 0;
  int head_unit = 0, rank = 0;
  bool whole = !LINE;                      // whole units, `remaining` of them from `position` on
  if constexpr (LINE) {
    __shared__ int64_t sums_of[WARPS];
    __shared__ int found[2], largest_of[WARPS];
    const unsigned blocks = gridDim.x;
    auto tiles_of = [&](int i) {
      if (i >= p.call.seqs) return -kUnitCost;
      const Span s = span_of(p, i);
      return s.to - s.from;
    };
    const int tiles = tiles_of(threadIdx.x);
    int largest = tiles;
    int64_t mine = int64_t(tiles + kUnitCost) * p.head_units, cost = mine;
    for (int i = threadIdx.x + kThreads; i < p.call.seqs; i += kThreads) {
      const int other = tiles_of(i);
      largest = max(largest, other);
      cost += int64_t(other + kUnitCost) * p.head_units;
    }
    largest = __reduce_max_sync(0xffffffffu, largest);
    if (lane == 0) largest_of[warp] = largest;
    Sums s = block_sums<WARPS>(cost, sums_of);
#pragma unroll
    for (int i = 0; i < WARPS; ++i) largest = max(largest, largest_of[i]);
    largest += kUnitCost;
    share = max(int64_t(kLeastShare), int64_t(float(s.all) * p.by_blocks) + 1);   // at least s.all / blocks
    // No unit is split where the longest of them, as many as a block gets, cost no more than an equal share and a split.  Whole and split, us:
    // 64 x 700 tokens of 4 heads 17.3, 18.5, 64 x 1000 22.2, 21.4, 64 x 2000 39.9, 31.4; 40 x 4000 72, 37; 96 x 2000 39.1, 43.7.
    whole = int64_t(largest) * (p.least + (p.more > 0)) <= share + kSplitCost * WARPS / kWarps;
    if (whole) {
      // blocks with one unit more are spread over the SMs
      const unsigned ahead = (blockIdx.x * unsigned(p.more) + blocks - 1) / blocks;
      position = int64_t(blockIdx.x) * p.least + ahead;
      remaining = p.least + int((blockIdx.x * unsigned(p.more) + p.more + blocks - 1) / blocks - ahead);
      if (remaining <= 0) return;
    } else {
      position = blockIdx.x * share;
      remaining = min(share, s.all - position);
      if (remaining <= 0) return;
      if (p.call.seqs > kThreads) s = block_sums<WARPS>(mine, sums_of);
      int64_t before = 0;
      for (int first = 0;;) {
        const int64_t end = before + s.upto;
        if (position < end && position >= end - mine) {
          found[0] = first + threadIdx.x;
          found[1] = int(position - (end - mine));
        }
        before += s.all;
        first += kThreads;
        if (first >= p.call.seqs || position < before) break;
        mine = int64_t(tiles_of(first + threadIdx.x) + kUnitCost) * p.head_units;
        s = block_sums<WARPS>(mine, sums_of);
      }
      __syncthreads();
      seq = found[0];
      offset = found[1];
    }
  }
  if constexpr (!LINE) {
    position = blockIdx.x / p.split;
    rank = blockIdx.x - int(position) * p.split;
  }

  const int record_rows = p.cache.page_size * 2 + p.cache.page_size / 16;
  auto place_of = [&](int t) { return int(p.page_tiles == 1 ? uint32_t(t) : __umulhi(uint32_t(t), p.by_page_tiles)); };
  int copied = 0;                          // stage of the next copy
  int stage = 0;
  uint32_t phase = 0;
  bool lost = false;   // a copy did not arrive: this warp's results become NaN
  const int my_token = token_of(r), value_token = token_of(2 * c), odd_token = token_of(2 * c + 1);
  const uint32_t key_at = chunk_at<GROUPS>(my_token, c);
  const uint32_t value_at = GROUPS == 4 ? chunk_at<4>(value_token, r) : chunk_at<2>(value_token, r >> 1) + 8 * (r & 1);
  const uint32_t odd_at = GROUPS == 4 ? chunk_at<4>(odd_token, r) : chunk_at<2>(odd_token, r >> 1) + 8 * (r & 1);
  // The unit at `position`: its tiles, heads and, on the line, the part of its cost that falls to this block.
  Span span;
  int begin, end, from = 0, to = 0, cost = 0, kv_head, head0, heads;
  const int* table;
  // Copies run ahead of the tiles that are multiplied.  The number of the next tile's page is on its way a tile earlier.
  int ahead_tile, ahead_page;
  auto enter = [&] {
    if (whole) {
      seq = int(position) / p.head_units;
      head_unit = int(position) - seq * p.head_units;
    }
    span = span_of(p, seq);
    if (!whole) {
      cost = span.to - span.from + kUnitCost;
      head_unit = int(uint32_t(offset) / uint32_t(cost));
      from = offset - head_unit * cost;
      to = int(min(int64_t(cost), from + remaining));
      begin = span.from + max(0, from - kUnitCost);
      end = span.from + max(0, to - kUnitCost);
    } else if (LINE) {
      begin = span.from;
      end = span.to;
    } else {
      const int tiles = (span.to - span.from + p.split - 1) / p.split;
      begin = min(span.to, span.from + rank * tiles);
      end = min(span.to, begin + tiles);
    }
    kv_head = head_unit / p.chunks;
    const int chunk = head_unit - kv_head * p.chunks;
    head0 = kv_head * p.group + chunk * kHeadTile;
    heads = min(kHeadTile, p.group - chunk * kHeadTile);
    table = p.call.table + seq * p.call.table_stride;
    ahead_tile = begin + warp;
    ahead_page = ahead_tile < end ? table[place_of(ahead_tile)] : 0;
  };
  auto copy_next = [&] {
    if (ahead_tile >= end) return;
    const int next_page = ahead_tile + WARPS < end ? table[place_of(ahead_tile + WARPS)] : 0;
    if (elect_one()) {
      // A page that is not there gives way to the first one, whose entries are then not used.
      const bool here = uint32_t(ahead_page) < uint32_t(p.cache.pages);
      const int record = (here ? ahead_page : 0) * p.cache.kv_heads + kv_head;
      const int entry = (ahead_tile - place_of(ahead_tile) * int(p.page_tiles)) * kTile, row = record * record_rows + entry;
      const uint32_t bar = bars + 8 * copied, slot = uint32_t(warp * ring + copied);
      there[warp][copied] = here;
      mbar_expect_tx(bar, 2 * S::kCodes + S::kScales);
      tma_load_2d(base + slot * (2 * S::kCodes), &map, bar, 0, row);
      tma_load_2d(base + slot * (2 * S::kCodes) + S::kCodes, &map, bar, 0, row + p.cache.page_size);
      bulk_load(all_scales + slot * S::kScales,
                static_cast<const uint8_t*>(p.cache.data) + (int64_t(record) * record_rows + 2 * p.cache.page_size) * kDim + entry * 2 * GROUPS, S::kScales, bar);
    }
    __syncwarp();
    copied = copied == ring - 1 ? 0 : copied + 1;
    ahead_tile += WARPS;
    ahead_page = next_page;
  };
  uint32_t q[GROUPS][2][2];
  auto fetch = [&] {   // the unit's first tiles and queries
#pragma unroll 1
    for (int i = 0; i < ring - 1 && !lost; ++i) copy_next();
    const uint16_t* const row = static_cast<const uint16_t*>(p.call.q) + seq * p.call.q_stride + int64_t(head0 + r) * kDim;
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int g = 0; g < GROUPS; ++g) {
        const int x = GROUPS == 4 ? 4 * j + c : 2 * c + j;
        const uint2 v = r < heads ? *reinterpret_cast<const uint2*>(row + 32 * g + 4 * x) : make_uint2(0, 0);
        q[g][j][0] = v.x;
        q[g][j][1] = v.y;
      }
  };
  if constexpr (kApart) {
    enter();
    fetch();
  }
  [[maybe_unused]] TagWord own_tag{p.tags + blockIdx.x};
  [[maybe_unused]] uint64_t tag_before = 0;   // looked at when the block ends: its way through memory is not waited for here
  for (;;) {
    if constexpr (!kApart) {
      enter();
      fetch();
    }
    // Queries as the second operand of the first product: column r is head r, rows the four elements at 32 g + 4 x.  A head's bf16 queries
    // become halves under a power of two that brings the largest to [2^14, 2^15).
    float2 to_log2;
    {
      uint32_t top = 0;
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int g = 0; g < GROUPS; ++g) {
          const uint32_t v0 = q[g][j][0], v1 = q[g][j][1];
          top = max(max(top, max(v0 & 0x7fffu, (v0 >> 16) & 0x7fffu)), max(v1 & 0x7fffu, (v1 >> 16) & 0x7fffu));
        }
      float back = p.call.scale * 1.44269504f;
      if constexpr (std::is_same<T, __nv_bfloat16>::value) {
#pragma unroll
        for (int step = 1; step < 4; step <<= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, step));
        const int biased = min(253, max(1, 127 + 14 + 127 - int(top >> 7)));
        const float factor = power_of(biased);
        back *= power_of(254 - biased);
#pragma unroll
        for (int g = 0; g < GROUPS; ++g)
#pragma unroll
          for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              const float2 pair = Packed<T>::widen(q[g][j][i]);
              q[g][j][i] = half2_bits(pair.x * factor, pair.y * factor);
            }
      }
      to_log2 = make_float2(__shfl_sync(0xffffffffu, back, 8 * c), __shfl_sync(0xffffffffu, back, 8 * c + 4));
    }

    float out[GROUPS][2][4];
#pragma unroll
    for (int g = 0; g < GROUPS; ++g)
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int i = 0; i < 4; ++i) out[g][h][i] = 0.f;
    // Heads 2c and 2c + 1.  Weights (of this lane's tokens) are summed over 2^(maximum - kBias), values over that and the scale of their group.
    float maximum[2] = {kNone, kNone}, weight[2] = {0.f, 0.f};
    float2 shift = make_float2(-kNone, -kNone);
    uint32_t inverse[GROUPS / 2];   // pairs of 1 / (the scale of a group's sums)
#pragma unroll
    for (int j = 0; j < GROUPS / 2; ++j) inverse[j] = pair_of(254 - kLeastScale);
    const auto scale_byte = [&](int g) { return 254 - int((inverse[g / 2] >> (g & 1 ? 23 : 7)) & 255u); };

    for (int t = begin + warp; t < end; t += WARPS) {
      if (!lost && !warp_wait(bars + 8 * stage, phase, &given_up)) {
        lost = true;
        given_up = 1;
      }
      if (lost) continue;
      const uint32_t slot = uint32_t(warp * ring + stage), keys = base + slot * (2 * S::kCodes), values = keys + S::kCodes;
      const uint32_t scales = all_scales + slot * S::kScales + uint32_t(my_token) * (2 * GROUPS);
      // Entries outside the span may hold anything: no score, no value and no scale of theirs is used.
      const int first_position = t * kTile, length = there[warp][stage] ? span.length : 0;
      const bool whole_tile = first_position >= span.first && first_position + kTile <= length;
      uint32_t k[2][2 * GROUPS], ks[2], vs[2];               // tokens my_token and my_token + 8
#pragma unroll
      for (int i = 0; i < 2; ++i) {
#pragma unroll
        for (int j = 0; j < GROUPS / 2; ++j) {
          const uint4 v = shared_16(keys + (key_at ^ (64 * j)) + i * 8 * kDim);
          k[i][4 * j] = v.x; k[i][4 * j + 1] = v.y; k[i][4 * j + 2] = v.z; k[i][4 * j + 3] = v.w;
        }
        if constexpr (GROUPS == 4) {
          const uint2 v = shared_8(scales + i * 16 * GROUPS);
          ks[i] = v.x; vs[i] = v.y;
        } else {
          const uint32_t v = shared_4(scales + i * 16 * GROUPS);
          ks[i] = v & 0xffffu; vs[i] = v >> 16;
        }
      }
      bool seen[2] = {true, true};
      if (!whole_tile) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int at_position = first_position + my_token + 8 * i;
          seen[i] = at_position >= span.first && at_position < length;
          if (!seen[i]) ks[i] = vs[i] = 0;
        }
      }
      // Scores: tokens my_token and my_token + 8, heads 2c and 2c + 1.
      float2 sum[2];
      uint32_t key_scales[2][GROUPS / 2], value_scales[2][GROUPS / 2];
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < GROUPS / 2; ++j) {
          key_scales[i][j] = two_scales(ks[i] >> (16 * j));
          value_scales[i][j] = mul_pairs(two_scales(vs[i] >> (16 * j)), inverse[j]);
        }
#pragma unroll
      for (int g = 0; g < GROUPS; ++g) {
        float part[4];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const int i = GROUPS * j + g;
          const uint32_t a[4] = {e4m3x2_to_half2(uint16_t(k[0][i])), e4m3x2_to_half2(uint16_t(k[1][i])),
                                 e4m3x2_to_half2(uint16_t(k[0][i] >> 16)), e4m3x2_to_half2(uint16_t(k[1][i] >> 16))};
          if (j == 0) mma_f16_first(part, a[0], a[1], a[2], a[3], q[g][j][0], q[g][j][1]);
          else mma_f16(part, a[0], a[1], a[2], a[3], q[g][j][0], q[g][j][1]);
        }
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const float by = scale_of(key_scales[i][g / 2], g);
          const float2 by2 = make_float2(by, by), part2 = make_float2(part[2 * i], part[2 * i + 1]);
          sum[i] = g == 0 ? mul2(by2, part2) : fma2(by2, part2, sum[i]);
        }
      }
      // The logarithms of the weights are rounded before the maximum is taken off, so the largest is off by nothing, whatever its size.
#pragma unroll
      for (int i = 0; i < 2; ++i) sum[i] = mul2(sum[i], to_log2);
      const float s[4] = {sum[0].x, sum[0].y, sum[1].x, sum[1].y};
      uint32_t v[4][GROUPS];                                 // tokens value_token, odd_token and those eight behind: elements 32 g + 4 r ...
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t from = values + (i & 1 ? odd_at : value_at) + (i >> 1) * 8 * kDim;
        if constexpr (GROUPS == 4) {
          const uint4 u = shared_16(from);
          v[i][0] = u.x; v[i][1] = u.y; v[i][2] = u.z; v[i][3] = u.w;
        } else {
          const uint2 u = shared_8(from);
          v[i][0] = u.x; v[i][1] = u.y;
        }
      }
      // The tile before this one has been multiplied by all lanes; its stage takes the next copy.
      __syncwarp();
      copy_next();
      if (!whole_tile) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int at_position = first_position + (i & 1 ? odd_token : value_token) + 8 * (i >> 1);
          if (at_position < span.first || at_position >= length) {
#pragma unroll
            for (int g = 0; g < GROUPS; ++g) v[i][g] = 0;
          }
        }
      }
      const float2 first = add2(sum[0], shift), second = add2(sum[1], shift);
      float x[4] = {first.x, first.y, second.x, second.y};
      if (!whole_tile) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (!seen[i >> 1]) x[i] = -INFINITY;
      }
      uint32_t tops = max_pairs(value_scales[0][0], value_scales[1][0]);
      if constexpr (GROUPS == 4) tops = max_pairs(tops, max_pairs(value_scales[0][1], value_scales[1][1]));

      // A new maximum, or a larger scale of a group's values, is taken up only when a weight could leave the range of a half.
      const bool larger = (tops + 0x3e003e00u) & 0x80008000u;   // more than 16 times
      const bool higher = fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])) > kBias + kSlack;
      if (__any_sync(0xffffffffu, larger || higher)) {
        // Groups of zeros have the scale 2^0, which says nothing of the others, so they do not count.  They are looked for where a byte could be theirs.
        // A group that holds nothing else brings every tile here (128 x 1100 tokens with the last group of 128 empty 39.8 us for 32.2); to know that of it
        // cost every tile 2 %.
        if (__builtin_expect(__any_sync(0xffffffffu, __vcmpeq4(vs[0], kZeros) | __vcmpeq4(vs[1], kZeros)), 0)) {
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            uint32_t codes[4] = {0, 0, 0, 0}, live = 0;   // of the groups, a quarter of them in a lane
#pragma unroll
            for (int j = 0; j < GROUPS / 2; ++j) {
              const uint4 w = shared_16(values + (key_at ^ (64 * j)) + i * 8 * kDim);
              codes[0] |= w.x; codes[1] |= w.y; codes[2 % GROUPS] |= w.z; codes[3 % GROUPS] |= w.w;
            }
#pragma unroll
            for (int g = 0; g < GROUPS; ++g) live |= codes[g] & 0x7f7f7f7fu ? 0xffu << (8 * g) : 0;
            live |= __shfl_xor_sync(0xffffffffu, live, 1);
            live |= __shfl_xor_sync(0xffffffffu, live, 2);
            vs[i] &= live;
          }
        }
        uint32_t shrink[GROUPS / 2];
#pragma unroll
        for (int j = 0; j < GROUPS / 2; ++j) {
          value_scales[0][j] = two_scales(vs[0] >> (16 * j));
          value_scales[1][j] = two_scales(vs[1] >> (16 * j));
          uint32_t top = max_pairs(value_scales[0][j], value_scales[1][j]);
#pragma unroll
          for (int step = 4; step < 32; step <<= 1) top = max_pairs(top, __shfl_xor_sync(0xffffffffu, top, step));
          top = min_pairs(top, pair_of(kMostScale));
          const uint32_t before = inverse_pair(inverse[j]);
          inverse[j] = inverse_pair(max_pairs(before, top));
          shrink[j] = mul_pairs(before, inverse[j]);
          value_scales[0][j] = mul_pairs(value_scales[0][j], inverse[j]);
          value_scales[1][j] = mul_pairs(value_scales[1][j], inverse[j]);
        }
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          float m = fmaxf(seen[0] ? s[h] : kNone, seen[1] ? s[h + 2] : kNone);
#pragma unroll
          for (int step = 4; step < 32; step <<= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, step));
          m = fmaxf(m, maximum[h]);
          const float factor = exp2_fast(maximum[h] - m);
          maximum[h] = m;
          (h ? shift.y : shift.x) = kBias - m;
          weight[h] *= factor;
#pragma unroll
          for (int i = 0; i < 2; ++i) x[h + 2 * i] = seen[i] ? s[h + 2 * i] + (h ? shift.y : shift.x) : -INFINITY;
#pragma unroll
          for (int g = 0; g < GROUPS; ++g) {
            const float by = factor * scale_of(shrink[g / 2], g);
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              out[g][i][h] *= by;
              out[g][i][h + 2] *= by;
            }
          }
        }
      }
      float scale[2][GROUPS];
#pragma unroll
      for (int g = 0; g < GROUPS; ++g)
#pragma unroll
        for (int i = 0; i < 2; ++i) scale[i][g] = scale_of(value_scales[i][g / 2], g);
      float2 probability[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) probability[i] = make_float2(exp2_fast(x[2 * i]), exp2_fast(x[2 * i + 1]));
      weight[0] += probability[0].x + probability[1].x;
      weight[1] += probability[0].y + probability[1].y;

#pragma unroll
      for (int g = 0; g < GROUPS; ++g) {
        uint32_t b[2], rest[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const float2 scaled = mul2(probability[i], make_float2(scale[i][g], scale[i][g]));
          const uint32_t rounded = half2_bits(scaled.x, scaled.y);
          b[i] = transpose8x8(rounded);
          if constexpr (EXACT) {
            const float2 back = Packed<__half>::widen(rounded);
            rest[i] = transpose8x8(half2_bits(scaled.x - back.x, scaled.y - back.y));
          }
        }
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const uint32_t near = __byte_perm(v[0][g], v[1][g], h ? 0x7362 : 0x5140), far = __byte_perm(v[2][g], v[3][g], h ? 0x7362 : 0x5140);
          const uint32_t a[4] = {e4m3x2_to_half2(uint16_t(near)), e4m3x2_to_half2(uint16_t(near >> 16)),
                                 e4m3x2_to_half2(uint16_t(far)), e4m3x2_to_half2(uint16_t(far >> 16))};
          if constexpr (EXACT) mma_f16(out[g][h], a[0], a[1], a[2], a[3], rest[0], rest[1]);
          mma_f16(out[g][h], a[0], a[1], a[2], a[3], b[0], b[1]);
        }
      }
      if (stage == ring - 1) {
        stage = 0;
        phase ^= 1u;
      } else {
        ++stage;
      }
    }

    // On to the next unit, whose first tiles come in while this one's sums are added up where these are apart.
    const bool begins = from == 0, ends = to == cost;   // whole units: both
    const int done_seq = seq, done_head0 = head0, done_heads = heads;
    int others = 0;   // where the unit ends in a block behind this one, this block waits for the parts of the blocks up to there
    auto find_others = [&] {
      if (!begins || ends) return;
      const int64_t last = position + cost - 1 - blockIdx.x * share;   // of the unit, behind this block's first place
      others = share >> 31 ? int(last >= share) : int(uint32_t(last) / uint32_t(share));
    };
    auto advance = [&] {
      if (whole) {
        --remaining;
        ++position;
      } else {
        remaining -= to - from;
        offset += to - from;
        position += to - from;
        if (offset == cost * p.head_units) {
          ++seq;
          offset = 0;
        }
      }
    };
    if constexpr (kApart) {
      find_others();
      advance();
      if (remaining > 0) {
        enter();
        fetch();
      }
    }

    // The block's warps meet: sums under a common maximum.
    __syncthreads();   // the rings are idle, and sums that were there have been read
    const float unit = lost ? __uint_as_float(0x7fc00000u) : power_of(127 - int(kBias));
#pragma unroll
    for (int h = 0; h < 2; ++h) {
#pragma unroll
      for (int step = 4; step < 32; step <<= 1) weight[h] += __shfl_xor_sync(0xffffffffu, weight[h], step);
      if (r == 0) {
        weights[warp][2 * c + h] = weight[h] * unit;
        maxima[warp][2 * c + h] = maximum[h];
      }
    }
#pragma unroll
    for (int g = 0; g < GROUPS; ++g) {
      const float group = lost ? unit : power_of(scale_byte(g) - int(kBias));
#pragma unroll
      for (int h = 0; h < 2; ++h)
        *reinterpret_cast<float4*>(&sums[warp][2 * c + h][32 * g + 4 * r]) =
            make_float4(out[g][0][h] * group, out[g][0][h + 2] * group, out[g][1][h] * group, out[g][1][h + 2] * group);
    }
    __syncthreads();
    if constexpr (LINE && !kApart) find_others();
    if (others) {
      for (int i = threadIdx.x; i < others; i += kThreads) {
        TagWord word{p.tags + blockIdx.x + 1 + i};
        if (!take_tag(word, p.tag)) given_up = 1;
      }
      __syncthreads();
    }
    for (int i = threadIdx.x; i < done_heads * kDim / 4; i += kThreads) {   // whole groups of eight lanes
      const int h = i / (kDim / 4), d = (i % (kDim / 4)) * 4;
      float m = maxima[0][h], l = 0.f;
      float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int j = 1; j < WARPS; ++j) m = fmaxf(m, maxima[j][h]);
#pragma unroll
      for (int j = 0; j < WARPS; ++j) {
        const float factor = exp2_fast(maxima[j][h] - m);
        const float4 part = *reinterpret_cast<const float4*>(&sums[j][h][d]);
        l += weights[j][h] * factor;
        sum.x += part.x * factor; sum.y += part.y * factor; sum.z += part.z * factor; sum.w += part.w * factor;
      }
      if constexpr (LINE) {
        constexpr int64_t kStride = kHeadTile * (kDim + 2);
        if (!begins) {
          float* const partial = p.partial + blockIdx.x * kStride;
          *reinterpret_cast<float4*>(partial + h * kDim + d) = sum;
          if (d == 0) *reinterpret_cast<float2*>(partial + kHeadTile * kDim + 2 * h) = make_float2(m, l);
          continue;
        }
        const float* const partial = p.partial + (blockIdx.x + 1) * kStride;
        const auto load = [&](int j, float4& x, float2& y) {
          x = __ldcg(reinterpret_cast<const float4*>(partial + j * kStride + h * kDim + d));
          y = __ldcg(reinterpret_cast<const float2*>(partial + j * kStride + kHeadTile * kDim + 2 * h));
        };
        // Few together where there are few: with sixteen at a time, most of them read again, 128 of 1000 to 2000 tokens took 44.4 us for 42.5.
        if (others <= 4) meet<2>(others, m, l, sum, load);
        else meet<16>(others, m, l, sum, load);
        if (others && given_up) l = __uint_as_float(0x7fc00000u);
        write_out<T, GROUPS>(p, done_seq, done_head0 + h, d, sum, l, m);
      } else if (p.split == 1) {
        write_out<T, GROUPS>(p, done_seq, done_head0 + h, d, sum, l, m);
      } else {
        *reinterpret_cast<float4*>(&sums[0][h][d]) = sum;   // read by this thread alone until here
        if (d == 0) block_weights[h] = make_float2(m, l);
      }
    }
    if constexpr (LINE) {
      if (!begins) {
        __syncthreads();
        if (threadIdx.x == 0) tag_before = leave_tag(own_tag, p.tag);
      }
      if constexpr (!kApart) advance();
      if (remaining <= 0) break;
      if constexpr (!kApart) {   // the sums have been read, and copies may take their place
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncthreads();
      }
    } else {
      if (p.split > 1) {
        // The cluster's blocks meet: each adds up its share of the columns over all blocks, in their order.
        cluster_sync();
        const int columns = kHeadTile * kDim / 4 / p.split, i = rank * columns + threadIdx.x;   // at least two blocks, 128 threads
        if (threadIdx.x < columns && i < done_heads * kDim / 4) {   // whole groups of eight lanes
          const int h = i / (kDim / 4), d = (i % (kDim / 4)) * 4;
          const uint32_t sums_at = smem_u32(&sums[0][h][d]), weights_at = smem_u32(&block_weights[h]);
          float m = kNone, l = 0.f;
          float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
          const auto load = [&](int j, float4& x, float2& y) {
            asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(x.x), "=f"(x.y), "=f"(x.z), "=f"(x.w) : "r"(map_to_rank(sums_at, uint32_t(j))) : "memory");
            asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(y.x), "=f"(y.y) : "r"(map_to_rank(weights_at, uint32_t(j))) : "memory");
          };
          if (p.split == 2) meet<2>(2, m, l, sum, load);
          else if (p.split == 4) meet<4>(4, m, l, sum, load);
          else meet<8>(p.split, m, l, sum, load);
          write_out<T, GROUPS>(p, done_seq, done_head0 + h, d, sum, l, m);
        }
        cluster_sync();   // no block leaves while another may read its sums
      }
      break;
    }
  }
  if constexpr (LINE) settle_tag(own_tag, p.tag, tag_before);
  if (lost) {   // time for what is still on its way to shared memory
    const long long start = clock64();
    while (clock64() - start < 400000ll) __nanosleep(1000);
  }
}

// How a call is spread over the device.
struct Split { int chunks, head_units; int64_t units; int warps, per_sm, split; bool line; int blocks, ring; };

Split split_of(const hg_cache& c, int seqs, int heads, int table_width, int window) {
  Split s{};
  const int group = heads / c.kv_heads, sms = sm_count();
  s.chunks = (group + kHeadTile - 1) / kHeadTile;
  s.head_units = c.kv_heads * s.chunks;
  s.units = int64_t(seqs) * s.head_units;
  int64_t longest = (int64_t(table_width) * c.page_size + kTile - 1) / kTile;
  if (window) longest = std::min<int64_t>(longest, (int64_t(window) + 2 * kTile - 2) / kTile);
  s.warps = kWarps;
  s.per_sm = kBlocksPerSm;
  s.split = 1;
  // The most warps of which the device holds all clusters at once.
  int64_t most = longest > kWhole ? 0 : INT64_MAX;
  for (int wide = 0; wide < 2; ++wide)
    for (int log = 0; log < 5; ++log) {
      const int warps = wide ? kWideWarps : kWarps, split = 1 << log;
      const int64_t all = s.units * split * warps;
      if (s.units * 1000 > int64_t(sms) * kHeld[wide][log] || all <= most || (split > 1 && longest <= int64_t(split / 2) * warps)) continue;
      most = all;
      s.warps = warps;
      s.per_sm = wide ? 1 : kBlocksPerSm;
      s.split = split;
    }
  // More units than SMs, or much work: a line.
  s.line = longest > kWhole && (s.units > sms || s.units * longest > kMuch || (s.units * longest > kFew && most * 4 < int64_t(sms) * kWideWarps * 3));
  s.blocks = int(s.units * s.split);
  if (s.line) {
    // Few units have many parts each: a wide block to an SM makes these a third as many, and its warps end together (4 x 32768: 31.9 us; three
    // blocks 34.5).  With more units, blocks that begin and end one at different times cover for one another (37 of 1 to 4099: 18.3;
    // one wide block 26.1).  Four blocks an SM have no room for sums beside rings of 128 elements (see kApart): they take what gives each of them
    // one unit at most (128 x 1100 31.7 us, three blocks 34.1; 128 of 1000 to 2000 42.5, 41.2).
    const bool wide = s.units <= sms;
    s.warps = wide ? kWideWarps : kWarps;
    s.per_sm = wide ? 1 : s.units <= sms * kLineBlocksPerSm || (s.units > sms * kBlocksPerSm && c.head_dim == 128) ? kLineBlocksPerSm : kBlocksPerSm;
    s.split = 1;
    s.blocks = int(std::min<int64_t>(sms * s.per_sm, (s.units * (longest + unit_cost(s.warps)) + kLeastShare - 1) / kLeastShare));
  }
  // As deep a ring as the blocks of an SM have room for, and use.
  const int sums = s.line && apart(c.head_dim, s.per_sm) ? s.warps * kHeadTile * (c.head_dim + 4) * 4 : 0;
  const int room = (kSmBytes / s.per_sm - 2048 - sums) / (s.warps * (c.head_dim == 128 ? Shared<4, kWarps>::kStage : Shared<2, kWarps>::kStage));
  s.ring = std::max(2, std::min({kMostRing, room, int((longest / s.split + s.warps - 1) / s.warps) + 1}));
  return s;
}

void validate_attention(const hg_cache& c, int seqs, int heads, int table_width, int window) {
  validate_cache(c);
  // rows of head_dim bytes, which the copies count in 32 bits
  if (int64_t(c.pages) * c.kv_heads * (c.page_size * 2 + c.page_size / 16) > 0x7fffffff) throw std::runtime_error("hg_attention: the cache has too many rows");
  if (seqs < 0 || heads <= 0 || heads % c.kv_heads) throw std::runtime_error("hg_attention: heads must be a multiple of kv_heads");
  if (table_width < 0 || window < 0 || int64_t(table_width) * c.page_size > (int64_t(1) << 30)) throw std::runtime_error("hg_attention: invalid table width or window");
  // a sequence's units are counted in 32 bits
  if (int64_t(seqs) * heads > (1 << 26) || (int64_t(table_width) * c.page_size / kTile + unit_cost(kWideWarps) + 1) * heads > 0x7fffffff) throw std::runtime_error("hg_attention: too much work for one call");
}

// The cache as rows of head_dim bytes; a copy takes sixteen.
CUtensorMap cache_map(const hg_cache& c) {
  static const EncodeTiled encode = encode_tiled();
  CUtensorMap map;
  std::memset(&map, 0, sizeof(map));
  const cuuint64_t dims[2] = {cuuint64_t(c.head_dim), cuuint64_t(c.pages) * c.kv_heads * (c.page_size * 2 + c.page_size / 16)};
  const cuuint64_t strides[1] = {cuuint64_t(c.head_dim)};
  const cuuint32_t box[2] = {cuuint32_t(c.head_dim), cuuint32_t(kTile)}, elem[2] = {1u, 1u};
  const CUresult r = encode(&map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, c.data, dims, strides, box, elem, CU_TENSOR_MAP_INTERLEAVE_NONE,
                            c.head_dim == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) throw std::runtime_error("cuTensorMapEncodeTiled failed with code " + std::to_string(int(r)));
  return map;
}

template <typename T, int GROUPS, int WARPS, int PER_SM, bool LINE, bool EXACT>
void launch_attention(const AttentionParams& p, const Split& s, cudaStream_t stream) {
  constexpr bool kApart = LINE && apart(32 * GROUPS, PER_SM);
  constexpr int kMost = Shared<GROUPS, WARPS>::bytes(kApart && GROUPS == 4 ? 3 : kMostRing, kApart);
  const int bytes = Shared<GROUPS, WARPS>::bytes(s.ring, kApart);
  if (bytes > kMost) throw std::runtime_error("hg_attention: shared memory");
  static std::once_flag once[64];   // limits of the function on each device
  int device = 0;
  check(cudaGetDevice(&device), "cudaGetDevice");
  if (device < 0 || device >= 64) throw std::runtime_error("Device ordinals 0..63 are supported");
  std::call_once(once[device], [] {
    check(cudaFuncSetAttribute(attention_kernel<T, GROUPS, WARPS, PER_SM, LINE, EXACT>, cudaFuncAttributeMaxDynamicSharedMemorySize, kMost), "attention");
    check(cudaFuncSetAttribute(attention_kernel<T, GROUPS, WARPS, PER_SM, LINE, EXACT>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1), "attention");
  });
  cudaLaunchConfig_t config{};
  config.gridDim = dim3(unsigned(s.blocks));
  config.blockDim = dim3(WARPS * 32);
  config.dynamicSmemBytes = size_t(bytes);
  config.stream = stream;
  cudaLaunchAttribute attribute[2];
  int count = 0;
  if (!LINE && s.split > 1) {
    attribute[count].id = cudaLaunchAttributeClusterDimension;
    attribute[count++].val.clusterDim = {unsigned(s.split), 1u, 1u};
  }
  if (pdl_enabled()) {
    attribute[count].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attribute[count++].val.programmaticStreamSerializationAllowed = 1;
  }
  config.attrs = attribute;
  config.numAttrs = unsigned(count);
  check(cudaLaunchKernelEx(&config, attention_kernel<T, GROUPS, WARPS, PER_SM, LINE, EXACT>, p, cache_map(p.cache)), "attention");
}

}  // namespace
}  // namespace hg

extern "C" {

int64_t hg_attention_workspace(const hg_cache* cache, int seqs, int heads, int table_width, int window) {
  try {
    if (!cache) throw std::runtime_error("Null argument to hg_attention_workspace");
    hg::validate_attention(*cache, seqs, heads, table_width, window);
    const hg::Split s = hg::split_of(*cache, seqs, heads, table_width, window);
    return !s.line || !seqs ? 0 : (s.blocks + 1 & ~1) * int64_t(sizeof(uint64_t)) + s.blocks * int64_t(hg::kHeadTile * (cache->head_dim + 2) * sizeof(float));
  } catch (std::exception const& e) {
    hg::last_error() = e.what();
    return -1;
  }
}

int hg_attention(const hg_cache* cache, const hg_attention_call* call, int dtype, void* stream) {
  HG_TRY
  if (!cache || !call) throw std::runtime_error("Null argument to hg_attention");
  const hg_attention_call& a = *call;
  hg::validate_attention(*cache, a.seqs, a.heads, a.table_width, a.window);
  if (dtype != HG_DTYPE_F16 && dtype != HG_DTYPE_BF16) throw std::runtime_error("hg_attention: unknown dtype");
  if (a.seqs == 0) return 0;
  if (!a.q || !a.lengths || (!a.table && a.table_width) || !a.codes == !a.out || !a.codes != !a.scales)
    throw std::runtime_error("hg_attention: queries, table, lengths and either out or codes with scales are needed");
  if (a.codes && a.heads * cache->head_dim % 128) throw std::runtime_error("hg_attention: quantisation needs heads * head_dim divisible by 128");
  if (reinterpret_cast<uintptr_t>(a.q) % 16 || a.q_stride % 8 || reinterpret_cast<uintptr_t>(a.out) % 16 || reinterpret_cast<uintptr_t>(a.codes) % 16 ||
      reinterpret_cast<uintptr_t>(a.scales) % 16 || reinterpret_cast<uintptr_t>(a.workspace) % 16)
    throw std::runtime_error("hg_attention: pointers must be aligned to 16 bytes and q_stride to 8 elements");
  const hg::Split s = hg::split_of(*cache, a.seqs, a.heads, a.table_width, a.window);
  const uint32_t page_tiles = uint32_t(cache->page_size / hg::kTile);
  hg::AttentionParams p{*cache, a, nullptr, nullptr, 0, 0, 0, 0.f, std::max(1, std::min(a.table_width / 32 + (a.table_width % 32 ? 1 : 0), hg::kTableLines / a.seqs)), s.head_units, s.chunks, a.heads / cache->kv_heads, s.split, s.ring, page_tiles,
                        uint32_t(((uint64_t(1) << 32) + page_tiles - 1) / page_tiles)};
  if (s.line) {
    if (!a.workspace) throw std::runtime_error("hg_attention: a workspace is needed");
    static std::atomic<uint64_t> calls{0};
    p.tag = hg::kTag * (2 * calls.fetch_add(1, std::memory_order_relaxed) + 1);   // odd numbers: none is zero, and no two are alike for 2^63 calls
    p.least = int(s.units / s.blocks);
    p.more = int(s.units % s.blocks);
    p.by_blocks = 1.000001f / float(s.blocks);
    p.tags = static_cast<uint64_t*>(a.workspace);
    p.partial = reinterpret_cast<float*>(p.tags + (s.blocks + 1 & ~1));
  }
  auto* const to = static_cast<cudaStream_t>(stream);
  const auto pick = [&](auto type, auto groups, auto exact) {
    using T = decltype(type);
    constexpr int G = decltype(groups)::value;
    constexpr bool E = decltype(exact)::value;
    if (s.line && s.warps == hg::kWideWarps) return hg::launch_attention<T, G, hg::kWideWarps, 1, true, E>;
    if (s.line)
      return s.per_sm == hg::kLineBlocksPerSm ? hg::launch_attention<T, G, hg::kWarps, hg::kLineBlocksPerSm, true, E> : hg::launch_attention<T, G, hg::kWarps, hg::kBlocksPerSm, true, E>;
    return s.warps == hg::kWideWarps ? hg::launch_attention<T, G, hg::kWideWarps, 1, false, E> : hg::launch_attention<T, G, hg::kWarps, hg::kBlocksPerSm, false, E>;
  };
  const auto pick_exact = [&](auto type, auto groups) { return a.codes ? pick(type, groups, std::true_type{}) : pick(type, groups, std::false_type{}); };
  using Two = std::integral_constant<int, 2>;
  using Four = std::integral_constant<int, 4>;
  const bool wide = cache->head_dim == 128;
  const auto launch = dtype == HG_DTYPE_BF16 ? (wide ? pick_exact(__nv_bfloat16{}, Four{}) : pick_exact(__nv_bfloat16{}, Two{}))
                                             : (wide ? pick_exact(__half{}, Four{}) : pick_exact(__half{}, Two{}));
  launch(p, s, to);
  HG_CATCH
}

}  // extern "C"
