// Attention of one new token a sequence over the paged MXFP8 cache, split over the cache's length and joined.
//
//   s_t = scale q . k_t      p_t = exp(s_t - max s)      out = sum_t p_t v_t / sum_t p_t
//
// One pass over the cache with a running maximum and sum.  A unit of work is a run of 16-token tiles of one sequence, kv head and
// up to eight of its query heads; a block of four warps takes one unit, its warps every fourth tile each, without shared memory on the
// way: a tile's codes go from global memory straight into the fragments of two matrix products,
//   S^T [16 tokens, 8 heads]     = K [16 tokens, d]   Q^T [d, 8 heads]       (m16n8k16, one accumulator for every scale group of 32 d)
//   O^T [16 d, 8 heads]          = V^T [16 d, tokens] P^T [tokens, 8 heads]
// so that the heads fill the narrow side of an instruction, whatever their number, and the cache its wide one.  Codes become halves,
// which hold them exactly.  Scales stay outside: those of the keys multiply a group's partial sum, those of the values the
// probabilities, once for every group, before these are rounded to halves for the second product.
//
// Roundings: q keeps its 16 bits (bf16 queries become halves under one power of two for the block, which keeps eight bits of
// all that is not 2^-30 of the largest).  P times the scale is rounded to 11 bits (2^-12 of each weight), held between 2^-32 and
// 2^8 of the largest so far by a bias of 2^7 and lazy rescaling.  Sums, maxima and outputs are fp32.
#include <algorithm>
#include <cmath>

#include "hg_cache.cuh"

namespace hg {
namespace {

constexpr int kTile = 16;            // tokens of a step of one warp
constexpr int kHeadTile = 8;         // query heads of a unit
constexpr int kWarps = 4;
constexpr int kUnitTiles = 16;       // a unit has no fewer tiles while its sequence has more
constexpr int kBlocksPerSm = 3;
constexpr float kBias = 7.f, kSlack = 4.f;   // P is kept in [0, 2^(kBias + 2 kSlack)]
constexpr float kNone = -1e30f;      // maximum of nothing

struct AttentionParams {
  hg_cache cache;
  hg_attention_call call;
  float* partial;       // [units][kHeadTile][head_dim + 2]: sums, maximum, sum of weights
  int2* pieces;         // [seqs][head units]: first unit and number of units
  int head_units;       // kv heads x chunks of kHeadTile heads
  int chunks, group, target;
};

__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t v) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}
__device__ __forceinline__ float exp2_approx(float x) { float r; asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x)); return r; }
__device__ __forceinline__ uint32_t half2_bits(float low, float high) {
  const __half2 h = __floats2half2_rn(low, high);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ float scale_of(uint32_t word, int g) { return __uint_as_float(((word >> (8 * g)) & 255u) << 23); }

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

__device__ __forceinline__ int block_sum(int v, int* parts) {
#pragma unroll
  for (int step = 16; step; step >>= 1) v += __shfl_xor_sync(0xffffffffu, v, step);
  if ((threadIdx.x & 31) == 0) parts[threadIdx.x >> 5] = v;
  __syncthreads();
  v = 0;
#pragma unroll
  for (int i = 0; i < kWarps; ++i) v += parts[i];
  return v;
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

// Results of one head unit: eight lanes a head and group of 32 elements, four elements a lane.  `value(h, d)` gives the four weighted
// sums of head h from element d on, `weight(h)` the sum of weights (over 2^maximum), `maximum(h)`.
template <typename T, int GROUPS, typename Value, typename Weight, typename Maximum>
__device__ __forceinline__ void finish(const AttentionParams& p, int seq, int head0, int heads, Value value, Weight weight, Maximum maximum) {
  constexpr int kDim = 32 * GROUPS;
  for (int i = threadIdx.x; i < kHeadTile * kDim / 4; i += kWarps * 32) {
    const int h = i / (kDim / 4), d = (i % (kDim / 4)) * 4;
    if (h >= heads) continue;   // whole groups of eight lanes
    const float l = weight(h), inv = l > 0.f || l != l ? 1.f / l : 0.f;
    const float4 sum = value(h, d);
    float v[4] = {sum.x * inv, sum.y * inv, sum.z * inv, sum.w * inv};
    if (l == 0.f) v[0] = v[1] = v[2] = v[3] = 0.f;
    const int head = head0 + h;
    if (p.call.codes) store_packed(p, seq, head, kDim, d >> 5, (d >> 2) & 7, v, 0xffu << (threadIdx.x & 24));
    else
      *reinterpret_cast<uint2*>(static_cast<uint16_t*>(p.call.out) + (int64_t(seq) * p.call.heads + head) * kDim + d) =
          make_uint2(uint32_t(from_float<T>(v[0])) | (uint32_t(from_float<T>(v[1])) << 16), uint32_t(from_float<T>(v[2])) | (uint32_t(from_float<T>(v[3])) << 16));
    if (p.call.lse && d == 0) p.call.lse[int64_t(seq) * p.call.heads + head] = l == 0.f ? -INFINITY : (maximum(h) - kBias + log2f(l)) * 0.69314718f;
  }
}

// Codes and scales of one tile, as a lane's part of the fragments.
template <int GROUPS>
struct Tile {
  uint32_t k[2][2 * GROUPS];   // tokens r and r + 8: for the steps (g, j) the word [GROUPS j + g]
  uint32_t v[4][GROUPS];       // tokens 2c, 2c + 1, 2c + 8, 2c + 9: elements 32 g + 4 r ...
  uint32_t ks[2], vs[2];       // scale bytes of the groups, tokens r and r + 8
};

template <int GROUPS>
__device__ __forceinline__ void load_tile(Tile<GROUPS>& t, const uint8_t* record, int page_size, int at, int r, int c) {
  constexpr int kDim = 32 * GROUPS;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const uint8_t* const row = record + (at + r + 8 * i) * kDim + 16 * c;
    const uint4 x = *reinterpret_cast<const uint4*>(row);
    t.k[i][0] = x.x; t.k[i][1] = x.y; t.k[i][2] = x.z; t.k[i][3] = x.w;
    if constexpr (GROUPS == 4) {
      const uint4 y = *reinterpret_cast<const uint4*>(row + 64);
      t.k[i][4] = y.x; t.k[i][5] = y.y; t.k[i][6] = y.z; t.k[i][7] = y.w;
    }
  }
  const uint8_t* const scales = record + 2 * page_size * kDim;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const uint8_t* const s = scales + (at + r + 8 * i) * 2 * GROUPS;
    if constexpr (GROUPS == 4) {
      const uint2 x = *reinterpret_cast<const uint2*>(s);
      t.ks[i] = x.x; t.vs[i] = x.y;
    } else {
      const uint32_t x = *reinterpret_cast<const uint32_t*>(s);
      t.ks[i] = x & 0xffffu; t.vs[i] = x >> 16;
    }
  }
  const uint8_t* const values = record + page_size * kDim;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint8_t* const row = values + (at + 2 * c + (i & 1) + 8 * (i >> 1)) * kDim + 4 * GROUPS * r;
    if constexpr (GROUPS == 4) {
      const uint4 x = *reinterpret_cast<const uint4*>(row);
      t.v[i][0] = x.x; t.v[i][1] = x.y; t.v[i][2] = x.z; t.v[i][3] = x.w;
    } else {
      const uint2 x = *reinterpret_cast<const uint2*>(row);
      t.v[i][0] = x.x; t.v[i][1] = x.y;
    }
  }
}

template <typename T, int GROUPS>
__global__ void __launch_bounds__(kWarps * 32, kBlocksPerSm)
attention_kernel(const AttentionParams p) {
  constexpr int kDim = 32 * GROUPS, kSteps = 2 * GROUPS;
  __shared__ int counts[2][kWarps];
  __shared__ int found[4];                                   // sequence, head unit, piece, pieces
  __shared__ float sums[kWarps][kHeadTile][kDim], weights[kWarps][kHeadTile], maxima[kWarps][kHeadTile];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, r = lane >> 2, c = lane & 3;
  // Loads below are ordinary ones: the kernel in front may still be writing the cache when this one starts, so the data is not
  // read-only for its duration.
  pdl_wait();
  pdl_trigger();

  // Padding of the scale buffer behind the last sequence.
  if (p.call.codes) {
    const int k = p.call.heads * kDim, kblocks = k >> 7, pad_rows = ((p.call.seqs + 127) & ~127) - p.call.seqs;
    for (int64_t i = int64_t(blockIdx.x) * blockDim.x + threadIdx.x; i < int64_t(pad_rows) * kblocks; i += int64_t(gridDim.x) * blockDim.x)
      *reinterpret_cast<uint32_t*>(static_cast<uint8_t*>(p.call.scales) + scale_word_offset(p.call.seqs + int(i / kblocks), int(i % kblocks), k)) = 0x7f7f7f7fu;
  }

  // This block's unit: sequences have ceil(tiles / size) units for each head unit, one at least.
  int tiles = 0;
  for (int i = threadIdx.x; i < p.call.seqs; i += kWarps * 32) {
    const Span s = span_of(p, i);
    tiles += s.to - s.from;
  }
  const int64_t all = int64_t(block_sum(tiles, counts[0])) * p.head_units;
  const int size = int(max(int64_t(kUnitTiles), (all + p.target - 1) / p.target));
  int before = 0;                                            // units of the sequences before this round's
  const int unit = blockIdx.x;
  if (threadIdx.x == 0) found[0] = -1;
  __syncwarp();
  for (int base = 0; base < p.call.seqs; base += 32) {       // every warp the same; warp 0 speaks
    int pieces = 0;
    if (base + lane < p.call.seqs) {
      const Span s = span_of(p, base + lane);
      pieces = max(1, (s.to - s.from + size - 1) / size);
    }
    int upto = pieces * p.head_units;
#pragma unroll
    for (int step = 1; step < 32; step <<= 1) {
      const int other = __shfl_up_sync(0xffffffffu, upto, step);
      if (lane >= step) upto += other;
    }
    const int start = before + upto - pieces * p.head_units;
    if (warp == 0 && unit >= start && unit < before + upto) {
      const int within = unit - start;
      found[0] = base + lane;
      found[1] = within / pieces;
      found[2] = within % pieces;
      found[3] = pieces;
    }
    before += __shfl_sync(0xffffffffu, upto, 31);
    if (unit < before) break;
  }
  __syncthreads();
  const int seq = found[0];
  if (seq < 0) return;
  const int head_unit = found[1], piece = found[2], pieces = found[3];
  const int kv_head = head_unit / p.chunks, chunk = head_unit - kv_head * p.chunks;
  const int head0 = kv_head * p.group + chunk * kHeadTile, heads = min(kHeadTile, p.group - chunk * kHeadTile);
  const Span span = span_of(p, seq);
  const int begin = span.from + piece * size, end = min(span.to, begin + size);
  if (threadIdx.x == 0 && piece == 0 && p.pieces) p.pieces[int64_t(seq) * p.head_units + head_unit] = make_int2(unit, pieces);

  // Queries as the second operand: column r is head r, rows the four elements at 32 g + 4 x of step (g, j).
  uint32_t q[kSteps][2];
  float q_scale = 1.f;
  {
    const uint16_t* const row = static_cast<const uint16_t*>(p.call.q) + seq * p.call.q_stride + int64_t(head0 + r) * kDim;
    uint2 raw[kSteps];
    uint32_t top = 0;
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int g = 0; g < GROUPS; ++g) {
        const int x = GROUPS == 4 ? 4 * j + c : 2 * c + j;
        raw[GROUPS * j + g] = r < heads ? *reinterpret_cast<const uint2*>(row + 32 * g + 4 * x) : make_uint2(0, 0);
        const uint2 w = raw[GROUPS * j + g];
        top = max(max(top, max(w.x & 0x7fffu, (w.x >> 16) & 0x7fffu)), max(w.y & 0x7fffu, (w.y >> 16) & 0x7fffu));
      }
    float factor = 1.f;
    if constexpr (std::is_same<T, __nv_bfloat16>::value) {
      // One power of two brings the largest of the block's queries to [2^14, 2^15).
      top = __reduce_max_sync(0xffffffffu, top);
      const int exponent = int(top >> 7);                    // biased
      const int biased = min(253, max(1, 127 + 14 + 127 - exponent));
      factor = __uint_as_float(uint32_t(biased) << 23);
      q_scale = __uint_as_float(uint32_t(254 - biased) << 23);
    }
#pragma unroll
    for (int i = 0; i < kSteps; ++i) {
      if constexpr (std::is_same<T, __half>::value) {
        q[i][0] = raw[i].x; q[i][1] = raw[i].y;
      } else {
        const float2 low = Packed<T>::widen(raw[i].x), high = Packed<T>::widen(raw[i].y);
        q[i][0] = half2_bits(low.x * factor, low.y * factor);
        q[i][1] = half2_bits(high.x * factor, high.y * factor);
      }
    }
  }
  const float to_log2 = p.call.scale * 1.44269504f * q_scale;

  float out[GROUPS][2][4];
#pragma unroll
  for (int g = 0; g < GROUPS; ++g)
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int i = 0; i < 4; ++i) out[g][h][i] = 0.f;
  float maximum[2] = {kNone, kNone}, weight[2] = {0.f, 0.f};   // heads 2c and 2c + 1; weights of this lane's tokens
  int value_scale = 0;                                         // exponent byte under which values are summed

  const int64_t record_bytes = cache_page_bytes(p.cache.page_size, kDim);
  const int* const table = p.call.table + seq * p.call.table_stride;
  for (int t = begin + warp; t < end; t += kWarps) {
    const int position = t * kTile, place = position / p.cache.page_size;
    const int page = table[place];
    if (uint32_t(page) >= uint32_t(p.cache.pages)) continue;
    const uint8_t* const record = static_cast<const uint8_t*>(p.cache.data) + (int64_t(page) * p.cache.kv_heads + kv_head) * record_bytes;
    Tile<GROUPS> tile;
    load_tile(tile, record, p.cache.page_size, position - place * p.cache.page_size, r, c);
    // Entries outside the span may hold anything: no score, no value and no scale of theirs is used.
    const bool whole = position >= span.first && position + kTile <= span.length;
    bool seen[2] = {true, true};
    if (!whole) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        seen[i] = position + r + 8 * i >= span.first && position + r + 8 * i < span.length;
        if (!seen[i]) tile.ks[i] = tile.vs[i] = 0;
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int at = position + 2 * c + (i & 1) + 8 * (i >> 1);
        if (at < span.first || at >= span.length) {
#pragma unroll
          for (int g = 0; g < GROUPS; ++g) tile.v[i][g] = 0;
        }
      }
    }
    // Scores: tokens r and r + 8, heads 2c and 2c + 1.
    float s[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int g = 0; g < GROUPS; ++g) {
      float part[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int w = GROUPS == 4 ? 4 * j + g : 2 * j + g;
        mma_f16(part, e4m3x2_to_half2(uint16_t(tile.k[0][w])), e4m3x2_to_half2(uint16_t(tile.k[1][w])),
                e4m3x2_to_half2(uint16_t(tile.k[0][w] >> 16)), e4m3x2_to_half2(uint16_t(tile.k[1][w] >> 16)), q[GROUPS * j + g][0], q[GROUPS * j + g][1]);
      }
      const float low = scale_of(tile.ks[0], g), high = scale_of(tile.ks[1], g);
      s[0] += low * part[0];
      s[1] += low * part[1];
      s[2] += high * part[2];
      s[3] += high * part[3];
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) s[i] = seen[i >> 1] ? s[i] * to_log2 : -INFINITY;

    // A new maximum, or larger scales of the values, is taken up only when a weight could leave the range of a half.
    const uint32_t tops = __vmaxu4(tile.vs[0], tile.vs[1]);
    const int top = max(max(int(tops & 255), int((tops >> 8) & 255)), max(int((tops >> 16) & 255), int(tops >> 24)));
    const bool rescale = fmaxf(s[0], s[2]) > maximum[0] + kSlack || fmaxf(s[1], s[3]) > maximum[1] + kSlack || top > value_scale + int(kSlack);
    if (__any_sync(0xffffffffu, rescale)) {
      const int new_scale = max(value_scale, __reduce_max_sync(0xffffffffu, top));
      const float shrink = __uint_as_float(uint32_t(max(0, 127 + value_scale - new_scale)) << 23);
      value_scale = new_scale;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        float m = fmaxf(s[h], s[h + 2]);
#pragma unroll
        for (int step = 4; step < 32; step <<= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, step));
        m = fmaxf(m, maximum[h]);
        const float factor = exp2_approx(maximum[h] - m);
        maximum[h] = m;
        weight[h] *= factor;
#pragma unroll
        for (int g = 0; g < GROUPS; ++g)
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            out[g][i][h] *= factor * shrink;
            out[g][i][h + 2] *= factor * shrink;
          }
      }
    }
    float probability[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) probability[i] = exp2_approx(s[i] - maximum[i & 1] + kBias);
    weight[0] += probability[0] + probability[2];
    weight[1] += probability[1] + probability[3];

#pragma unroll
    for (int g = 0; g < GROUPS; ++g) {
      const float low = __uint_as_float(uint32_t(max(0, 127 + int((tile.vs[0] >> (8 * g)) & 255) - value_scale)) << 23);
      const float high = __uint_as_float(uint32_t(max(0, 127 + int((tile.vs[1] >> (8 * g)) & 255) - value_scale)) << 23);
      const uint32_t b0 = transpose8x8(half2_bits(probability[0] * low, probability[1] * low));
      const uint32_t b1 = transpose8x8(half2_bits(probability[2] * high, probability[3] * high));
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint32_t near = __byte_perm(tile.v[0][g], tile.v[1][g], h ? 0x7362 : 0x5140), far = __byte_perm(tile.v[2][g], tile.v[3][g], h ? 0x7362 : 0x5140);
        mma_f16(out[g][h], e4m3x2_to_half2(uint16_t(near)), e4m3x2_to_half2(uint16_t(near >> 16)),
                e4m3x2_to_half2(uint16_t(far)), e4m3x2_to_half2(uint16_t(far >> 16)), b0, b1);
      }
    }
  }

  // The block's warps meet: sums under a common maximum.
#pragma unroll
  for (int h = 0; h < 2; ++h) {
#pragma unroll
    for (int step = 4; step < 32; step <<= 1) weight[h] += __shfl_xor_sync(0xffffffffu, weight[h], step);
    if (r == 0) {
      weights[warp][2 * c + h] = weight[h];
      maxima[warp][2 * c + h] = maximum[h];
    }
  }
  const float unit_scale = mx_scale(value_scale);
#pragma unroll
  for (int g = 0; g < GROUPS; ++g)
#pragma unroll
    for (int h = 0; h < 2; ++h)
      *reinterpret_cast<float4*>(&sums[warp][2 * c + h][32 * g + 4 * r]) =
          make_float4(out[g][0][h] * unit_scale, out[g][0][h + 2] * unit_scale, out[g][1][h] * unit_scale, out[g][1][h + 2] * unit_scale);
  __syncthreads();
  auto block_maximum = [&](int h) {
    float m = maxima[0][h];
#pragma unroll
    for (int w = 1; w < kWarps; ++w) m = fmaxf(m, maxima[w][h]);
    return m;
  };
  auto block_weight = [&](int h) {
    const float m = block_maximum(h);
    float l = 0.f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) l += weights[w][h] * exp2_approx(maxima[w][h] - m);
    return l;
  };
  auto block_value = [&](int h, int d) {
    const float m = block_maximum(h);
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const float factor = exp2_approx(maxima[w][h] - m);
      const float4 part = *reinterpret_cast<const float4*>(&sums[w][h][d]);
      v.x += part.x * factor; v.y += part.y * factor; v.z += part.z * factor; v.w += part.w * factor;
    }
    return v;
  };
  if (pieces == 1) {
    finish<T, GROUPS>(p, seq, head0, heads, block_value, block_weight, block_maximum);
    return;
  }
  float* const partial = p.partial + int64_t(unit) * kHeadTile * (kDim + 2);
  for (int i = threadIdx.x; i < kHeadTile * kDim / 4; i += kWarps * 32) {
    const int h = i / (kDim / 4), d = (i % (kDim / 4)) * 4;
    *reinterpret_cast<float4*>(partial + h * kDim + d) = block_value(h, d);
  }
  if (threadIdx.x < kHeadTile) {
    partial[kHeadTile * kDim + threadIdx.x] = block_maximum(threadIdx.x);
    partial[kHeadTile * (kDim + 1) + threadIdx.x] = block_weight(threadIdx.x);
  }
}

// Adds the units of a sequence and head unit, in their order.
template <typename T, int GROUPS>
__global__ void __launch_bounds__(kWarps * 32)
attention_join_kernel(const AttentionParams p) {
  constexpr int kDim = 32 * GROUPS, kStride = kHeadTile * (kDim + 2);
  pdl_trigger();
  const int seq = blockIdx.x / p.head_units, head_unit = blockIdx.x - seq * p.head_units;
  const int kv_head = head_unit / p.chunks, chunk = head_unit - kv_head * p.chunks;
  const int head0 = kv_head * p.group + chunk * kHeadTile, heads = min(kHeadTile, p.group - chunk * kHeadTile);
  pdl_wait();
  const int2 at = p.pieces[blockIdx.x];
  if (at.y == 1) return;
  const float* const first = p.partial + int64_t(at.x) * kStride;
  auto maximum = [&](int h) {
    float m = kNone;
    for (int i = 0; i < at.y; ++i) m = fmaxf(m, first[int64_t(i) * kStride + kHeadTile * kDim + h]);
    return m;
  };
  auto weight = [&](int h) {
    const float m = maximum(h);
    float l = 0.f;
    for (int i = 0; i < at.y; ++i) l += first[int64_t(i) * kStride + kHeadTile * (kDim + 1) + h] * exp2_approx(first[int64_t(i) * kStride + kHeadTile * kDim + h] - m);
    return l;
  };
  auto value = [&](int h, int d) {
    const float m = maximum(h);
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int i = 0; i < at.y; ++i) {
      const float* const from = first + int64_t(i) * kStride;
      const float factor = exp2_approx(from[kHeadTile * kDim + h] - m);
      const float4 part = *reinterpret_cast<const float4*>(from + h * kDim + d);
      v.x += part.x * factor; v.y += part.y * factor; v.z += part.z * factor; v.w += part.w * factor;
    }
    return v;
  };
  finish<T, GROUPS>(p, seq, head0, heads, value, weight, maximum);
}

// Blocks that share the work, and the units there can be at most.
struct Split { int chunks, head_units, target; int64_t units, longest; bool join; };
Split split_of(const hg_cache& c, int seqs, int heads, int table_width, int window) {
  static const int sms = [] {
    int device = 0, n = 148;
    if (cudaGetDevice(&device) != cudaSuccess || cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, device) != cudaSuccess) {
      cudaGetLastError();
      n = 148;
    }
    return n;
  }();
  Split s;
  const int group = heads / c.kv_heads;
  s.chunks = (group + kHeadTile - 1) / kHeadTile;
  s.head_units = c.kv_heads * s.chunks;
  s.target = sms * kBlocksPerSm;
  s.longest = (int64_t(table_width) * c.page_size + kTile - 1) / kTile;
  if (window) s.longest = std::min<int64_t>(s.longest, (int64_t(window) + 2 * kTile - 2) / kTile);
  s.join = s.longest > kUnitTiles;
  s.units = int64_t(seqs) * s.head_units + (s.join ? s.target : 0);
  return s;
}

void validate_attention(const hg_cache& c, int seqs, int heads, int table_width, int window) {
  validate_cache(c);
  if (seqs < 0 || heads <= 0 || heads % c.kv_heads) throw std::runtime_error("hg_attention: heads must be a multiple of kv_heads");
  if (table_width < 0 || window < 0 || int64_t(table_width) * c.page_size > (int64_t(1) << 30)) throw std::runtime_error("hg_attention: invalid table width or window");
  // sums of tiles and units are held in 32 bits
  const Split s = split_of(c, seqs, heads, table_width, window);
  if (s.units > (1 << 30) || int64_t(seqs) * s.longest > (1 << 30)) throw std::runtime_error("hg_attention: too many sequences in one call");
}

template <typename T, int GROUPS>
void launch_attention(const AttentionParams& p, const Split& s, cudaStream_t stream) {
  check(launch_kernel(attention_kernel<T, GROUPS>, dim3(unsigned(s.units)), dim3(kWarps * 32), 0, stream, p), "attention");
  if (s.join) check(launch_kernel(attention_join_kernel<T, GROUPS>, dim3(unsigned(p.call.seqs * p.head_units)), dim3(kWarps * 32), 0, stream, p), "attention join");
}

}  // namespace
}  // namespace hg

extern "C" {

int64_t hg_attention_workspace(const hg_cache* cache, int seqs, int heads, int table_width, int window) {
  try {
    if (!cache) throw std::runtime_error("Null argument to hg_attention_workspace");
    hg::validate_attention(*cache, seqs, heads, table_width, window);
    const hg::Split s = hg::split_of(*cache, seqs, heads, table_width, window);
    if (!s.join || !seqs) return 0;
    return ((int64_t(seqs) * s.head_units * 8 + 15) & ~int64_t(15)) + s.units * hg::kHeadTile * (cache->head_dim + 2) * 4;
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
  if (s.join && !a.workspace) throw std::runtime_error("hg_attention: a workspace is needed");
  hg::AttentionParams p{*cache, a, nullptr, nullptr, s.head_units, s.chunks, a.heads / cache->kv_heads, s.target};
  if (s.join) {
    p.pieces = static_cast<int2*>(a.workspace);
    p.partial = reinterpret_cast<float*>(static_cast<char*>(a.workspace) + ((int64_t(a.seqs) * s.head_units * 8 + 15) & ~int64_t(15)));
  }
  auto* const to = static_cast<cudaStream_t>(stream);
  if (dtype == HG_DTYPE_BF16) cache->head_dim == 128 ? hg::launch_attention<__nv_bfloat16, 4>(p, s, to) : hg::launch_attention<__nv_bfloat16, 2>(p, s, to);
  else cache->head_dim == 128 ? hg::launch_attention<__half, 4>(p, s, to) : hg::launch_attention<__half, 2>(p, s, to);
  HG_CATCH
}

}  // extern "C"
