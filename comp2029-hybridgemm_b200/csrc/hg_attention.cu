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
constexpr int kWarps = 4, kThreads = kWarps * 32;
constexpr int kBlocksPerSm = 3;
constexpr int kWhole = 16;           // sequences of no more tiles are not split
constexpr int kUnitCost = 8;         // cost of a unit beside its tiles, in tiles
constexpr int kLeastShare = 24;      // a block's share of the cost, where there is less for all blocks
constexpr float kBias = 7.f, kSlack = 4.f;   // P is kept in [0, 2^(kBias + 2 kSlack)]
constexpr float kNone = -1e30f;      // maximum of nothing

// The work of a split call is a line on which every unit (sequence and head unit, in this order) has its tiles behind kUnitCost
// for what it costs besides; a block takes an equal share of the line, so whatever the lengths all blocks end together.
// It holds parts of at most two units that other blocks have parts of, at its beginning and at its end.
struct Join { int seq, head_unit, first, parts; };   // sums of a unit: slots first, 2 * (first / 2 + 1), + 2, ...

struct AttentionParams {
  hg_cache cache;
  hg_attention_call call;
  float* partial;       // [2 per block][kHeadTile][head_dim + 2]: sums, maximum, sum of weights; null: no unit is split
  Join* joins;          // [blocks]: the unit whose second part begins the block's share; parts 0: none
  int head_units;       // kv heads x chunks of kHeadTile heads
  int chunks, group;
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

// Sums of what the block's threads give, of all and of those up to this one.
struct Sums { int64_t all, upto; };
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
  for (int i = 0; i < kWarps; ++i) {
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
  if (p.call.lse && d == 0) p.call.lse[int64_t(seq) * p.call.heads + head] = l == 0.f ? -INFINITY : (m - kBias + log2f(l)) * 0.69314718f;
}

// Results of one head unit.  `value(h, d)` gives the four weighted sums of head h from element d on.
template <typename T, int GROUPS, typename Value, typename Weight, typename Maximum>
__device__ __forceinline__ void finish(const AttentionParams& p, int seq, int head0, int heads, Value value, Weight weight, Maximum maximum) {
  constexpr int kDim = 32 * GROUPS;
  for (int i = threadIdx.x; i < heads * kDim / 4; i += kThreads) {   // whole groups of eight lanes
    const int h = i / (kDim / 4), d = (i % (kDim / 4)) * 4;
    write_out<T, GROUPS>(p, seq, head0 + h, d, value(h, d), weight(h), maximum(h));
  }
}

__device__ __forceinline__ uint4 load_16(const uint8_t* p) {
  uint4 v;
  asm volatile("ld.global.L1::no_allocate.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
  return v;
}
__device__ __forceinline__ uint2 load_8(const uint8_t* p) {
  uint2 v;
  asm volatile("ld.global.L1::no_allocate.v2.b32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "l"(p));
  return v;
}
__device__ __forceinline__ uint32_t load_4(const uint8_t* p) {
  uint32_t v;
  asm volatile("ld.global.L1::no_allocate.b32 %0, [%1];" : "=r"(v) : "l"(p));
  return v;
}

// A lane's part of one tile, as the fragments take it.
template <int GROUPS>
struct Tile {
  uint32_t k[2][2 * GROUPS];   // tokens r and r + 8: for the steps (g, j) the word [GROUPS j + g]
  uint32_t v[4][GROUPS];       // tokens 2c, 2c + 1, 2c + 8, 2c + 9: elements 32 g + 4 r ...
  uint32_t ks[2], vs[2];       // scale bytes of the groups, tokens r and r + 8
};

template <int GROUPS>
__device__ __forceinline__ void load_keys(Tile<GROUPS>& t, const uint8_t* record, int page_size, int at, int r, int c) {
  constexpr int kDim = 32 * GROUPS;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const uint8_t* const row = record + (at + r + 8 * i) * kDim + 16 * c;
    const uint4 x = load_16(row);
    t.k[i][0] = x.x; t.k[i][1] = x.y; t.k[i][2] = x.z; t.k[i][3] = x.w;
    if constexpr (GROUPS == 4) {
      const uint4 y = load_16(row + 64);
      t.k[i][4] = y.x; t.k[i][5] = y.y; t.k[i][6] = y.z; t.k[i][7] = y.w;
    }
  }
}
template <int GROUPS>
__device__ __forceinline__ void load_scales(uint32_t (&ks)[2], uint32_t (&vs)[2], const uint8_t* record, int page_size, int at, int r) {
  const uint8_t* const scales = record + 2 * page_size * (32 * GROUPS);
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const uint8_t* const s = scales + (at + r + 8 * i) * 2 * GROUPS;
    if constexpr (GROUPS == 4) {
      const uint2 x = load_8(s);
      ks[i] = x.x; vs[i] = x.y;
    } else {
      const uint32_t x = load_4(s);
      ks[i] = x & 0xffffu; vs[i] = x >> 16;
    }
  }
}
template <int GROUPS>
__device__ __forceinline__ void load_values(Tile<GROUPS>& t, const uint8_t* record, int page_size, int at, int r, int c) {
  constexpr int kDim = 32 * GROUPS;
  const uint8_t* const values = record + page_size * kDim;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint8_t* const row = values + (at + 2 * c + (i & 1) + 8 * (i >> 1)) * kDim + 4 * GROUPS * r;
    if constexpr (GROUPS == 4) {
      const uint4 x = load_16(row);
      t.v[i][0] = x.x; t.v[i][1] = x.y; t.v[i][2] = x.z; t.v[i][3] = x.w;
    } else {
      const uint2 x = load_8(row);
      t.v[i][0] = x.x; t.v[i][1] = x.y;
    }
  }
}

template <typename T, int GROUPS>
__global__ void __launch_bounds__(kThreads, kBlocksPerSm)
attention_kernel(const AttentionParams p) {
  constexpr int kDim = 32 * GROUPS, kSteps = 2 * GROUPS, kStride = kHeadTile * (kDim + 2);
  __shared__ int64_t parts[kWarps], found_offset;
  __shared__ int found_seq;
  __shared__ alignas(16) float sums[kWarps][kHeadTile][kDim];   // four at a time
  __shared__ float weights[kWarps][kHeadTile], maxima[kWarps][kHeadTile];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, r = lane >> 2, c = lane & 3;
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

  // This block's share of the line: `remaining` from `offset` in the units of sequence `seq` on.
  int seq;
  int64_t offset, remaining, share = 0, position0 = 0;
  if (p.partial) {
    auto cost_of = [&](int i) -> int64_t {
      if (i >= p.call.seqs) return 0;
      const Span s = span_of(p, i);
      return int64_t(s.to - s.from + kUnitCost) * p.head_units;
    };
    int64_t mine = cost_of(threadIdx.x), cost = mine;
    for (int i = threadIdx.x + kThreads; i < p.call.seqs; i += kThreads) cost += cost_of(i);
    Sums s = block_sums(cost, parts);
    const int64_t all = s.all;
    share = max(int64_t(kLeastShare), (all + gridDim.x - 1) / gridDim.x);
    position0 = blockIdx.x * share;
    remaining = min(share, all - position0);
    if (remaining <= 0) {
      if (threadIdx.x == 0) p.joins[blockIdx.x].parts = 0;
      return;
    }
    if (p.call.seqs > kThreads) s = block_sums(mine, parts);
    int64_t before = 0;
    for (int base = 0;;) {
      const int64_t end = before + s.upto;
      if (position0 < end && position0 >= end - mine) {
        found_seq = base + threadIdx.x;
        found_offset = position0 - (end - mine);
      }
      before += s.all;
      base += kThreads;
      if (base >= p.call.seqs || position0 < before) break;
      mine = cost_of(base + threadIdx.x);
      s = block_sums(mine, parts);
    }
    __syncthreads();
    seq = found_seq;
    offset = found_offset;
  } else {
    seq = blockIdx.x / p.head_units;
    offset = blockIdx.x - seq * p.head_units;
    remaining = 1;
  }

  const int64_t record_bytes = cache_page_bytes(p.cache.page_size, kDim);
  for (bool first = true; remaining > 0; first = false) {
    // The next unit, or this block's part of it.
    const Span span = span_of(p, seq);
    const int tiles = span.to - span.from;
    int head_unit = int(offset), begin = 0, end = tiles;
    bool whole_unit = true;
    if (p.partial) {
      const int cost = tiles + kUnitCost;
      head_unit = int(offset / cost);
      const int from = int(offset - int64_t(head_unit) * cost), to = int(min(int64_t(cost), from + remaining));
      begin = max(0, from - kUnitCost);
      end = max(0, to - kUnitCost);
      whole_unit = from == 0 && to == cost;
      if (first && threadIdx.x == 0) {
        // The second part of a unit is at the beginning of the block behind the one that holds the unit's beginning.
        const int64_t unit0 = position0 - from, before = position0 - share;
        Join j{seq, head_unit, 2 * int(blockIdx.x - 1) + (unit0 > before), 0};
        if (from > 0 && unit0 >= before) j.parts = int((unit0 + cost - 1) / share) - int(blockIdx.x) + 2;
        p.joins[blockIdx.x] = j;
      }
      remaining -= to - from;
      offset += to - from;
    } else {
      remaining = 0;
    }
    begin += span.from;
    end += span.from;
    const int kv_head = head_unit / p.chunks, chunk = head_unit - kv_head * p.chunks;
    const int head0 = kv_head * p.group + chunk * kHeadTile, heads = min(kHeadTile, p.group - chunk * kHeadTile);

    // The first tile, on its way while the queries are prepared.
    const int* const table = p.call.table + seq * p.call.table_stride;
    const uint8_t* const head_data = static_cast<const uint8_t*>(p.cache.data) + kv_head * record_bytes;
    auto page_of = [&](int t) { return t < end ? table[t * kTile / p.cache.page_size] : -1; };
    // A page that is not there gives way to the first one, whose entries are then not used.
    auto record_of = [&](int page) { return head_data + (uint32_t(page) < uint32_t(p.cache.pages) ? page : 0) * (record_bytes * p.cache.kv_heads); };
    auto place_of = [&](int t) { return t * kTile % p.cache.page_size; };
    int t = begin + warp, page = page_of(t), next_page = page_of(t + kWarps);
    Tile<GROUPS> tile;
    if (t < end) {
      load_keys(tile, record_of(page), p.cache.page_size, place_of(t), r, c);
      load_scales<GROUPS>(tile.ks, tile.vs, record_of(page), p.cache.page_size, place_of(t), r);
      load_values(tile, record_of(page), p.cache.page_size, place_of(t), r, c);
    }

    // Queries as the second operand: column r is head r, rows the four elements at 32 g + 4 x of step (g, j).
    uint32_t q[kSteps][2];
    float q_scale = 1.f;
    {
      const uint16_t* const row = static_cast<const uint16_t*>(p.call.q) + seq * p.call.q_stride + int64_t(head0 + r) * kDim;
      uint32_t top = 0;
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int g = 0; g < GROUPS; ++g) {
          const int x = GROUPS == 4 ? 4 * j + c : 2 * c + j;
          const uint2 w = r < heads ? *reinterpret_cast<const uint2*>(row + 32 * g + 4 * x) : make_uint2(0, 0);
          q[GROUPS * j + g][0] = w.x;
          q[GROUPS * j + g][1] = w.y;
          top = max(max(top, max(w.x & 0x7fffu, (w.x >> 16) & 0x7fffu)), max(w.y & 0x7fffu, (w.y >> 16) & 0x7fffu));
        }
      if constexpr (std::is_same<T, __nv_bfloat16>::value) {
        // One power of two brings the largest of the unit's queries to [2^14, 2^15).
        top = __reduce_max_sync(0xffffffffu, top);
        const int biased = min(253, max(1, 127 + 14 + 127 - int(top >> 7)));
        const float factor = __uint_as_float(uint32_t(biased) << 23);
        q_scale = __uint_as_float(uint32_t(254 - biased) << 23);
#pragma unroll
        for (int i = 0; i < kSteps; ++i)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const float2 pair = Packed<T>::widen(q[i][h]);
            q[i][h] = half2_bits(pair.x * factor, pair.y * factor);
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

    for (; t < end; t += kWarps) {
      const int position = t * kTile;
      const bool more = t + kWarps < end;
      const int after = page_of(t + 2 * kWarps);
      // Entries outside the span may hold anything: no score, no value and no scale of theirs is used.
      const int to = uint32_t(page) < uint32_t(p.cache.pages) ? span.length : 0;
      const bool whole = position >= span.first && position + kTile <= to;
      bool seen[2] = {true, true};
      if (!whole) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          seen[i] = position + r + 8 * i >= span.first && position + r + 8 * i < to;
          if (!seen[i]) tile.ks[i] = tile.vs[i] = 0;
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int at = position + 2 * c + (i & 1) + 8 * (i >> 1);
          if (at < span.first || at >= to) {
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
          const int w = GROUPS * j + g;
          mma_f16(part, e4m3x2_to_half2(uint16_t(tile.k[0][w])), e4m3x2_to_half2(uint16_t(tile.k[1][w])),
                  e4m3x2_to_half2(uint16_t(tile.k[0][w] >> 16)), e4m3x2_to_half2(uint16_t(tile.k[1][w] >> 16)), q[w][0], q[w][1]);
        }
        const float low = scale_of(tile.ks[0], g), high = scale_of(tile.ks[1], g);
        s[0] += low * part[0];
        s[1] += low * part[1];
        s[2] += high * part[2];
        s[3] += high * part[3];
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) s[i] = seen[i >> 1] ? s[i] * to_log2 : -INFINITY;
      // The next tile's keys take the place of these, as its values will.
      const uint8_t* const next = record_of(next_page);
      const int next_place = place_of(t + kWarps);
      uint32_t next_ks[2] = {0, 0}, next_vs[2] = {0, 0};
      if (more) {
        load_keys(tile, next, p.cache.page_size, next_place, r, c);
        load_scales<GROUPS>(next_ks, next_vs, next, p.cache.page_size, next_place, r);
      }

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
      if (more) load_values(tile, next, p.cache.page_size, next_place, r, c);
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        tile.ks[i] = next_ks[i];
        tile.vs[i] = next_vs[i];
      }
      page = next_page;
      next_page = after;
    }

    // The block's warps meet: sums under a common maximum.
    if (!first) __syncthreads();   // the unit before has been read
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
    if (whole_unit) {
      finish<T, GROUPS>(p, seq, head0, heads, block_value, block_weight, block_maximum);
    } else {
      float* const partial = p.partial + (2 * int64_t(blockIdx.x) + !first) * kStride;
      for (int i = threadIdx.x; i < heads * kDim / 4; i += kThreads) {
        const int h = i / (kDim / 4), d = (i % (kDim / 4)) * 4;
        *reinterpret_cast<float4*>(partial + h * kDim + d) = block_value(h, d);
      }
      if (threadIdx.x < kHeadTile) {
        partial[kHeadTile * kDim + threadIdx.x] = block_maximum(threadIdx.x);
        partial[kHeadTile * (kDim + 1) + threadIdx.x] = block_weight(threadIdx.x);
      }
    }
    if (p.partial && offset == int64_t(tiles + kUnitCost) * p.head_units) {
      ++seq;
      offset = 0;
    }
  }
}

// Adds the parts of a split unit, in their order; a block for each of its heads.
template <typename T, int GROUPS>
__global__ void __launch_bounds__(kThreads)
attention_join_kernel(const AttentionParams p) {
  constexpr int kDim = 32 * GROUPS, kStride = kHeadTile * (kDim + 2), kLanes = kDim / 4, kTeams = kThreads / kLanes;
  __shared__ float4 values[kTeams][kLanes];
  pdl_trigger();
  pdl_wait();
  const Join j = p.joins[blockIdx.x];
  if (j.parts == 0) return;
  const int kv_head = j.head_unit / p.chunks, chunk = j.head_unit - kv_head * p.chunks, h = blockIdx.y;
  if (h >= min(kHeadTile, p.group - chunk * kHeadTile)) return;
  const int head = kv_head * p.group + chunk * kHeadTile + h;
  auto part = [&](int i) { return p.partial + int64_t(i == 0 ? j.first : 2 * (j.first / 2 + i)) * kStride; };
  const int lane = threadIdx.x & 31;
  float m = kNone, l = 0.f;
  for (int i = lane; i < j.parts; i += 32) m = fmaxf(m, part(i)[kHeadTile * kDim + h]);
#pragma unroll
  for (int step = 16; step; step >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, step));
  for (int i = lane; i < j.parts; i += 32) l += part(i)[kHeadTile * (kDim + 1) + h] * exp2_approx(part(i)[kHeadTile * kDim + h] - m);
#pragma unroll
  for (int step = 16; step; step >>= 1) l += __shfl_xor_sync(0xffffffffu, l, step);
  const int team = threadIdx.x / kLanes, d = (threadIdx.x % kLanes) * 4;
  float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
  for (int i = team; i < j.parts; i += kTeams) {
    const float factor = exp2_approx(part(i)[kHeadTile * kDim + h] - m);
    const float4 x = *reinterpret_cast<const float4*>(part(i) + h * kDim + d);
    v.x += x.x * factor; v.y += x.y * factor; v.z += x.z * factor; v.w += x.w * factor;
  }
  values[team][d / 4] = v;
  __syncthreads();
  if (threadIdx.x >= kLanes) return;
#pragma unroll
  for (int i = 1; i < kTeams; ++i) {
    const float4 x = values[i][d / 4];
    v.x += x.x; v.y += x.y; v.z += x.z; v.w += x.w;
  }
  write_out<T, GROUPS>(p, j.seq, head, d, v, l, m);
}

// How a call is spread over the device.
struct Split { int chunks, head_units, blocks; int64_t longest; bool join; };
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
  s.longest = (int64_t(table_width) * c.page_size + kTile - 1) / kTile;
  if (window) s.longest = std::min<int64_t>(s.longest, (int64_t(window) + 2 * kTile - 2) / kTile);
  s.join = s.longest > kWhole;
  const int64_t units = int64_t(seqs) * s.head_units;
  s.blocks = int(s.join ? std::min<int64_t>(sms * kBlocksPerSm, (units * (s.longest + kUnitCost) + kLeastShare - 1) / kLeastShare) : units);
  return s;
}

void validate_attention(const hg_cache& c, int seqs, int heads, int table_width, int window) {
  validate_cache(c);
  if (seqs < 0 || heads <= 0 || heads % c.kv_heads) throw std::runtime_error("hg_attention: heads must be a multiple of kv_heads");
  if (table_width < 0 || window < 0 || int64_t(table_width) * c.page_size > (int64_t(1) << 30)) throw std::runtime_error("hg_attention: invalid table width or window");
  if (int64_t(seqs) * heads > (1 << 30)) throw std::runtime_error("hg_attention: too many sequences in one call");
}

template <typename T, int GROUPS>
void launch_attention(const AttentionParams& p, const Split& s, cudaStream_t stream) {
  check(launch_kernel(attention_kernel<T, GROUPS>, dim3(unsigned(s.blocks)), dim3(kThreads), 0, stream, p), "attention");
  if (s.join) check(launch_kernel(attention_join_kernel<T, GROUPS>, dim3(unsigned(s.blocks), unsigned(std::min(kHeadTile, p.group))), dim3(kThreads), 0, stream, p), "attention join");
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
    return int64_t(s.blocks) * (sizeof(hg::Join) + 2 * hg::kHeadTile * (cache->head_dim + 2) * sizeof(float));
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
  hg::AttentionParams p{*cache, a, nullptr, nullptr, s.head_units, s.chunks, a.heads / cache->kv_heads};
  if (s.join) {
    p.joins = static_cast<hg::Join*>(a.workspace);
    p.partial = reinterpret_cast<float*>(p.joins + s.blocks);
  }
  auto* const to = static_cast<cudaStream_t>(stream);
  if (dtype == HG_DTYPE_BF16) cache->head_dim == 128 ? hg::launch_attention<__nv_bfloat16, 4>(p, s, to) : hg::launch_attention<__nv_bfloat16, 2>(p, s, to);
  else cache->head_dim == 128 ? hg::launch_attention<__half, 4>(p, s, to) : hg::launch_attention<__half, 2>(p, s, to);
  HG_CATCH
}

}  // extern "C"
