// RMS norm between two blocks of a decoder, fused with what stands round it: the residual addition in front (with the gate, the
// residual scale and the norm of the block's output that some models have there) and the MXFP8 quantisation behind.
//
//   y = x                                         or, with a post weight, x / sqrt(mean(x^2) + post_eps) * post_weight
//   h = round16(residual + scale * gate * y)      the new residual stream, written out
//   n = h / sqrt(mean(h^2) + eps) * weight        E4M3 codes and E8M0 scales as hg_pack's, or rounded to 16 bits
//
// Sums and products are fp32.  h is rounded once, and n is computed from the rounded h, so that whoever reads the stream later
// finds the values that were normalised; n is not rounded to 16 bits before its codes are.
//
// A row stays in the registers of a block between the sum of its squares and its codes, so memory is passed over once; bytes bound many rows (2048 x
// 3584 with a residual 10.4 us, 0.76 of the measured copy rate), the chain load, barrier, store few ones (one row 1.8 us).
#include <algorithm>

#include "hg_common.cuh"

namespace hg {
namespace {

constexpr int kNormThreads = 1024, kNormVectors = 4;   // at most kNormThreads x kNormVectors x 8 columns
constexpr int kManyRows = 768, kWideRow = 3200, kMuch = 1 << 23;

// Sum over the block; `parts` holds a float for each warp and is used once.
__device__ __forceinline__ float block_sum(float v, float4* parts) {
#pragma unroll
  for (int step = 16; step; step >>= 1) v += __shfl_xor_sync(0xffffffffu, v, step);
  const int warps = blockDim.x >> 5, warp = threadIdx.x >> 5, lane = threadIdx.x & 31, all = (warps + 3) & ~3;
  float* const part = reinterpret_cast<float*>(parts);
  if (lane == 0) part[warp] = v;
  else if (warp == warps - 1 && warp + lane < all) part[warp + lane] = 0.f;
  __syncthreads();
  v = 0.f;
  for (int i = 0; i < all / 4; ++i) {   // four at a time: one by one they took 0.2 us
    const float4 x = parts[i];
    v += (x.x + x.y) + (x.z + x.w);
  }
  return v;
}

// Eight columns as pairs.
struct Eight { float2 v[4]; };
template <typename T>
__device__ __forceinline__ Eight widen8(const uint4& raw) {
  return {Packed<T>::widen(raw.x), Packed<T>::widen(raw.y), Packed<T>::widen(raw.z), Packed<T>::widen(raw.w)};
}
__device__ __forceinline__ void times(Eight& a, const Eight& b) {
#pragma unroll
  for (int i = 0; i < 4; ++i) a.v[i] = mul2(a.v[i], b.v[i]);
}
__device__ __forceinline__ void times(Eight& a, float b) {
#pragma unroll
  for (int i = 0; i < 4; ++i) a.v[i] = mul2(a.v[i], make_float2(b, b));
}
template <typename T>
__device__ __forceinline__ uint4 round8(const Eight& a) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) w[i] = Packed<T>::round(a.v[i]);
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// 1 / sqrt(m) with one step of Newton's method behind the approximation: a row's codes beside a border all move with its error.
__device__ __forceinline__ float inverse_root(float m) {
  const float r = rsqrtf(m), off = fmaf(-m * r, r, 1.f);
  return m > 1e-30f && m < 1e30f ? fmaf(0.5f * r, off, r) : r;   // beyond, a product may leave the range
}

__device__ __forceinline__ const uint4* at(const void* base, int64_t element) { return reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(base) + element); }
__device__ __forceinline__ uint4* at(void* base, int64_t element) { return reinterpret_cast<uint4*>(static_cast<uint16_t*>(base) + element); }

// Whether h differs from x.
__host__ __device__ __forceinline__ bool changes(const hg_norm_call& p) { return p.post_weight || p.gate || p.residual || p.scale != 1.f; }

// Eight columns of the new stream, from the block's output (r: of its norm) and their residual.
template <typename T>
__device__ __forceinline__ uint4 stream8(const hg_norm_call& p, int row, int col, const uint4& x, float r, const uint4& residual) {
  Eight v = widen8<T>(x);
  if (p.post_weight) {
    times(v, widen8<T>(*at(p.post_weight, col)));   // exact
    times(v, r);
  }
  if (p.gate) {
    if (p.gate_per_row) times(v, to_float<T>(static_cast<const uint16_t*>(p.gate)[row * p.gate_stride]));
    else times(v, widen8<T>(*at(p.gate, row * p.gate_stride + col)));
  }
  if (p.scale != 1.f) times(v, p.scale);
  if (p.residual) {
    const Eight other = widen8<T>(residual);
#pragma unroll
    for (int i = 0; i < 4; ++i) v.v[i] = add2(v.v[i], other.v[i]);
  }
  return round8<T>(v);
}

template <typename T>
__device__ __forceinline__ float squares8(const uint4& raw) {
  const Eight v = widen8<T>(raw);
  float2 sum = mul2(v.v[0], v.v[0]);
#pragma unroll
  for (int i = 1; i < 4; ++i) sum = fma2(v.v[i], v.v[i], sum);
  return sum.x + sum.y;
}

// Writes eight normalised columns.  When quantising all sixteen lanes of the K128 block are here.
template <typename T>
__device__ __forceinline__ void emit8(const hg_norm_call& p, int row, int col, const uint4& h, const uint4& weight, float r) {
  Eight v = widen8<T>(h);
  times(v, widen8<T>(weight));   // exact
  times(v, r);
  if (!p.codes) {
    *at(p.normed, int64_t(row) * p.k + col) = round8<T>(v);
    return;
  }
  const unsigned mask = 0xffffu << (threadIdx.x & 16);
  float amax = 0.f;
#pragma unroll
  for (int i = 0; i < 4; ++i) amax = fmaxf(fmaxf(amax, fabsf(v.v[i].x)), fabsf(v.v[i].y));
  amax = fmaxf(amax, __shfl_xor_sync(mask, amax, 1));
  amax = fmaxf(amax, __shfl_xor_sync(mask, amax, 2));
  const int e = mx_exponent<false>(amax);
  times(v, mx_inverse_scale(e));
  uint2 codes;
  codes.x = cvt_e4m3x2(v.v[0].x, v.v[0].y) | (cvt_e4m3x2(v.v[1].x, v.v[1].y) << 16);
  codes.y = cvt_e4m3x2(v.v[2].x, v.v[2].y) | (cvt_e4m3x2(v.v[3].x, v.v[3].y) << 16);
  *reinterpret_cast<uint2*>(static_cast<uint8_t*>(p.codes) + int64_t(row) * p.k + col) = codes;
  uint32_t word = uint32_t(e + 127) << (8 * ((threadIdx.x >> 2) & 3));
  word |= __shfl_xor_sync(mask, word, 4);
  word |= __shfl_xor_sync(mask, word, 8);
  if ((threadIdx.x & 15) == 0) *reinterpret_cast<uint32_t*>(static_cast<uint8_t*>(p.scales) + scale_word_offset(row, col >> 7, p.k)) = word;
}

// Scale bytes of the rows behind the last one, by the blocks from `first` on.
__device__ __forceinline__ void pad_scales(const hg_norm_call& p, int first) {
  const int kblocks = p.k >> 7, pad_rows = ((p.rows + 127) & ~127) - p.rows;
  pdl_wait();
  for (int64_t i = int64_t(blockIdx.x - first) * blockDim.x + threadIdx.x; i < int64_t(pad_rows) * kblocks; i += int64_t(gridDim.x - first) * blockDim.x)
    *reinterpret_cast<uint32_t*>(static_cast<uint8_t*>(p.scales) + scale_word_offset(p.rows + int(i / kblocks), int(i % kblocks), p.k)) = 0x7f7f7f7fu;
}

// Few or wide rows: a block to a row, eight columns to a thread and vector.
template <typename T, int VECTORS>
__global__ void __launch_bounds__(kNormThreads)
norm_kernel(const hg_norm_call p) {
  __shared__ float4 parts[2][8];
  pdl_trigger();
  const int row = blockIdx.x;
  if (row >= p.rows) return pad_scales(p, p.rows);
  pdl_wait();
  const float inv_k = 1.f / float(p.k);
  uint4 h[VECTORS], weight[VECTORS], residual[VECTORS];
  float sum = 0.f;
#pragma unroll
  for (int j = 0; j < VECTORS; ++j) {
    const int col = (j * blockDim.x + threadIdx.x) * 8;
    h[j] = residual[j] = weight[j] = make_uint4(0, 0, 0, 0);
    if (col >= p.k) continue;
    h[j] = *at(p.x, row * p.x_stride + col);
    if (p.residual) residual[j] = *at(p.residual, row * p.residual_stride + col);
    weight[j] = *at(p.weight, col);
  }
  float r = 1.f;
  if (p.post_weight) {
#pragma unroll
    for (int j = 0; j < VECTORS; ++j) sum += squares8<T>(h[j]);
    r = inverse_root(block_sum(sum, parts[0]) * inv_k + p.post_eps);
  }
  sum = 0.f;
#pragma unroll
  for (int j = 0; j < VECTORS; ++j) {
    const int col = (j * blockDim.x + threadIdx.x) * 8;
    if (changes(p) && col < p.k) {
      h[j] = stream8<T>(p, row, col, h[j], r, residual[j]);
      *at(p.stream_out, int64_t(row) * p.k + col) = h[j];
    }
    sum += squares8<T>(h[j]);
  }
  r = inverse_root(block_sum(sum, parts[1]) * inv_k + p.eps);
#pragma unroll
  for (int j = 0; j < VECTORS; ++j) {
    const int col = (j * blockDim.x + threadIdx.x) * 8;
    if (col < p.k) emit8<T>(p, row, col, h[j], weight[j], r);
  }
}

bool aligned(const void* p, int64_t stride = 0) { return reinterpret_cast<uintptr_t>(p) % 16 == 0 && stride % 8 == 0; }

template <typename T>
void launch_norm(const hg_norm_call& p, cudaStream_t stream) {
  const int pad_words = p.codes ? (((p.rows + 127) & ~127) - p.rows) * (p.k >> 7) : 0;
  // One vector gives the shorter chain while SMs hold few rows (3584 columns: one row 1.8 us, with two 2.1; 512 rows 4.0 and 4.4), two halve
  // the barriers and weigh less on issue where they hold many (2048 rows 11.6 us and 10.5; 1024 rows of 2432 with a post norm and a gate 7.5
  // and 6.6), and four leave an SM more rows at once where there are rows enough for that (16384 x 4096 85.7 us and 72.9, 2048 x 5120 15.7 and
  // 14.4, 2048 x 12288 47.7 and 35.8; but 2048 x 3584 10.5 and 10.8, 4096 x 2432 13.9 and 14.2, 8192 x 1152 14.4 and 16.1).  A warp to a row,
  // without barriers, was slower everywhere (2048 rows 16.2 us): too few rows under way.
  const bool much = p.k >= kWideRow && int64_t(p.rows) * p.k >= kMuch;
  const int vectors = much ? kNormVectors : p.k <= kNormThreads * 8 && (p.rows < kManyRows || p.k <= 1024) ? 1 : p.k <= kNormThreads * 16 ? 2 : kNormVectors;
  const int threads = ((p.k + 8 * vectors - 1) / (8 * vectors) + 31) & ~31, pad_blocks = std::min((pad_words + threads - 1) / threads, 16);
  const auto kernel = vectors == 1 ? norm_kernel<T, 1> : vectors == 2 ? norm_kernel<T, 2> : norm_kernel<T, kNormVectors>;
  check(launch_kernel(kernel, dim3(unsigned(p.rows + pad_blocks)), dim3(threads), 0, stream, p), "norm");
}

}  // namespace
}  // namespace hg

extern "C" int hg_norm(const hg_norm_call* call, int dtype, void* stream) {
  HG_TRY
  if (!call) throw std::runtime_error("Null argument to hg_norm");
  const hg_norm_call& p = *call;
  if (p.rows < 0 || p.k <= 0 || p.k % 8 || p.k > hg::kNormThreads * hg::kNormVectors * 8)
    throw std::runtime_error("hg_norm: k must be a multiple of 8 up to 32768");
  if (p.rows == 0) return 0;
  if (dtype != HG_DTYPE_F16 && dtype != HG_DTYPE_BF16) throw std::runtime_error("hg_norm: unknown dtype");
  if (!p.x || !p.weight || !p.codes == !p.normed || !p.codes != !p.scales) throw std::runtime_error("hg_norm: x, weight and either codes with scales or normed are needed");
  if (p.codes && p.k % 128) throw std::runtime_error("hg_norm: quantisation needs k divisible by 128");
  if (hg::changes(p) && !p.stream_out) throw std::runtime_error("hg_norm: a changed stream needs an output");
  if (!hg::aligned(p.x, p.x_stride) || !hg::aligned(p.residual, p.residual ? p.residual_stride : 0) || !hg::aligned(p.weight) ||
      !hg::aligned(p.post_weight) || (!p.gate_per_row && !hg::aligned(p.gate, p.gate ? p.gate_stride : 0)) || !hg::aligned(p.stream_out) ||
      !hg::aligned(p.normed) || !hg::aligned(p.codes) || !hg::aligned(p.scales))
    throw std::runtime_error("hg_norm: pointers and rows must be aligned to 16 bytes");
  if (dtype == HG_DTYPE_BF16) hg::launch_norm<__nv_bfloat16>(p, static_cast<cudaStream_t>(stream));
  else hg::launch_norm<__half>(p, static_cast<cudaStream_t>(stream));
  HG_CATCH
}
