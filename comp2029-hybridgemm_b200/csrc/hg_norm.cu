// RMS norm between two blocks of a decoder, fused with what stands round it: the residual addition in front (with the gate, the
// residual scale and the norm of the block's output that some models have there) and the MXFP8 quantisation behind.
//
//   y = x                                         or, with a post weight, x / sqrt(mean(x^2) + post_eps) * post_weight
//   h = round16(residual + scale * gate * y)      the new residual stream, written out
//   n = h / sqrt(mean(h^2) + eps) * weight        E4M3 codes and E8M0 scales as hg_pack's, or rounded to 16 bits
//
// Sums and products are fp32.  h is rounded once, and n is computed from the rounded h, so that whoever reads the stream later
// finds the values that were normalised; n is not rounded to 16 bits before its codes are.
#include <algorithm>

#include "hg_common.cuh"

namespace hg {
namespace {

constexpr int kNormThreads = 1024, kNormVectors = 4;   // at most kNormThreads x kNormVectors x 8 columns

// Sum over the block; `parts` holds a float for each warp and is used once.
__device__ __forceinline__ float block_sum(float v, float* parts) {
#pragma unroll
  for (int step = 16; step; step >>= 1) v += __shfl_xor_sync(0xffffffffu, v, step);
  const int warps = blockDim.x >> 5;
  if ((threadIdx.x & 31) == 0) parts[threadIdx.x >> 5] = v;
  __syncthreads();
  v = 0.f;
  for (int i = 0; i < warps; ++i) v += parts[i];
  return v;
}

template <typename T>
__device__ __forceinline__ void load8(const void* base, int64_t element, float (&v)[8]) {
  const uint4 raw = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(base) + element);
  const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 pair = Packed<T>::widen(w[i]);
    v[2 * i] = pair.x;
    v[2 * i + 1] = pair.y;
  }
}
template <typename T>
__device__ __forceinline__ uint4 round8(const float (&v)[8]) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) w[i] = uint32_t(from_float<T>(v[2 * i])) | (uint32_t(from_float<T>(v[2 * i + 1])) << 16);
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// One block to a row, eight columns to a thread and vector; blocks behind the rows write the padding of the scales.
template <typename T, int VECTORS>
__global__ void __launch_bounds__(kNormThreads)
norm_kernel(const hg_norm_call p) {
  __shared__ float parts[2][32];
  pdl_trigger();
  const int row = blockIdx.x, kblocks = p.k >> 7;
  if (row >= p.rows) {
    const int pad_rows = ((p.rows + 127) & ~127) - p.rows;
    const int64_t stride = int64_t(gridDim.x - p.rows) * blockDim.x;
    pdl_wait();
    for (int64_t i = int64_t(row - p.rows) * blockDim.x + threadIdx.x; i < int64_t(pad_rows) * kblocks; i += stride)
      *reinterpret_cast<uint32_t*>(static_cast<uint8_t*>(p.scales) + scale_word_offset(p.rows + int(i / kblocks), int(i % kblocks), p.k)) = 0x7f7f7f7fu;
    return;
  }
  pdl_wait();
  const float inv_k = 1.f / float(p.k);
  float v[VECTORS][8];
  float sum = 0.f;
#pragma unroll
  for (int j = 0; j < VECTORS; ++j) {
    const int col = (j * blockDim.x + threadIdx.x) * 8;
#pragma unroll
    for (int i = 0; i < 8; ++i) v[j][i] = 0.f;
    if (col >= p.k) continue;
    load8<T>(p.x, row * p.x_stride + col, v[j]);
#pragma unroll
    for (int i = 0; i < 8; ++i) sum += v[j][i] * v[j][i];
  }
  float r = 1.f;
  if (p.post_weight) r = rsqrtf(block_sum(sum, parts[0]) * inv_k + p.post_eps);
  const bool changed = p.post_weight || p.gate || p.residual || p.scale != 1.f;
  if (changed) {
    sum = 0.f;
#pragma unroll
    for (int j = 0; j < VECTORS; ++j) {
      const int col = (j * blockDim.x + threadIdx.x) * 8;
      if (col >= p.k) continue;
      float other[8];
      if (p.post_weight) {
        load8<T>(p.post_weight, col, other);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[j][i] = v[j][i] * r * other[i];
      }
      if (p.gate) {
        if (p.gate_per_row) {
          const float gate = to_float<T>(static_cast<const uint16_t*>(p.gate)[row * p.gate_stride]);
#pragma unroll
          for (int i = 0; i < 8; ++i) v[j][i] *= gate;
        } else {
          load8<T>(p.gate, row * p.gate_stride + col, other);
#pragma unroll
          for (int i = 0; i < 8; ++i) v[j][i] *= other[i];
        }
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) v[j][i] *= p.scale;
      if (p.residual) {
        load8<T>(p.residual, row * p.residual_stride + col, other);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[j][i] += other[i];
      }
      const uint4 h = round8<T>(v[j]);
      *reinterpret_cast<uint4*>(static_cast<uint16_t*>(p.stream_out) + int64_t(row) * p.k + col) = h;
      const uint32_t w[4] = {h.x, h.y, h.z, h.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 pair = Packed<T>::widen(w[i]);
        v[j][2 * i] = pair.x;
        v[j][2 * i + 1] = pair.y;
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) sum += v[j][i] * v[j][i];
    }
  }
  r = rsqrtf(block_sum(sum, parts[1]) * inv_k + p.eps);
#pragma unroll
  for (int j = 0; j < VECTORS; ++j) {
    const int col = (j * blockDim.x + threadIdx.x) * 8;
    if (col >= p.k) continue;
    const unsigned mask = 0xffffu << (threadIdx.x & 16);   // the 16 threads of a K128 block, all of them here when quantising
    float w[8];
    load8<T>(p.weight, col, w);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[j][i] = v[j][i] * r * w[i];
    if (!p.codes) {
      *reinterpret_cast<uint4*>(static_cast<uint16_t*>(p.normed) + int64_t(row) * p.k + col) = round8<T>(v[j]);
      continue;
    }
    float amax = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) amax = fmaxf(amax, fabsf(v[j][i]));
    amax = fmaxf(amax, __shfl_xor_sync(mask, amax, 1));
    amax = fmaxf(amax, __shfl_xor_sync(mask, amax, 2));
    const int e = mx_exponent<false>(amax);
    const float inv = mx_inverse_scale(e);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[j][i] *= inv;
    uint2 codes;
    codes.x = cvt_e4m3x2(v[j][0], v[j][1]) | (cvt_e4m3x2(v[j][2], v[j][3]) << 16);
    codes.y = cvt_e4m3x2(v[j][4], v[j][5]) | (cvt_e4m3x2(v[j][6], v[j][7]) << 16);
    *reinterpret_cast<uint2*>(static_cast<uint8_t*>(p.codes) + int64_t(row) * p.k + col) = codes;
    const int base = threadIdx.x & 16;
    const uint32_t byte = uint32_t(e + 127);
    const uint32_t word = __shfl_sync(mask, byte, base) | (__shfl_sync(mask, byte, base + 4) << 8) |
                          (__shfl_sync(mask, byte, base + 8) << 16) | (__shfl_sync(mask, byte, base + 12) << 24);
    if ((threadIdx.x & 15) == 0) *reinterpret_cast<uint32_t*>(static_cast<uint8_t*>(p.scales) + scale_word_offset(row, col >> 7, p.k)) = word;
  }
}

bool aligned(const void* p, int64_t stride = 0) { return reinterpret_cast<uintptr_t>(p) % 16 == 0 && stride % 8 == 0; }

template <typename T>
void launch_norm(const hg_norm_call& p, cudaStream_t stream) {
  const int vectors = p.k <= kNormThreads * 8 ? 1 : p.k <= kNormThreads * 16 ? 2 : kNormVectors;
  const int threads = ((p.k + 8 * vectors - 1) / (8 * vectors) + 31) & ~31;
  const int64_t pad_words = p.codes ? int64_t(((p.rows + 127) & ~127) - p.rows) * (p.k >> 7) : 0;
  const int pad_blocks = int(std::min<int64_t>((pad_words + threads - 1) / threads, 16));
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
  const bool changed = p.post_weight || p.gate || p.residual || p.scale != 1.f;
  if (changed && !p.stream_out) throw std::runtime_error("hg_norm: a changed stream needs an output");
  if (!hg::aligned(p.x, p.x_stride) || !hg::aligned(p.residual, p.residual ? p.residual_stride : 0) || !hg::aligned(p.weight) ||
      !hg::aligned(p.post_weight) || (!p.gate_per_row && !hg::aligned(p.gate, p.gate ? p.gate_stride : 0)) || !hg::aligned(p.stream_out) ||
      !hg::aligned(p.normed) || !hg::aligned(p.codes) || !hg::aligned(p.scales))
    throw std::runtime_error("hg_norm: pointers and rows must be aligned to 16 bytes");
  if (dtype == HG_DTYPE_BF16) hg::launch_norm<__nv_bfloat16>(p, static_cast<cudaStream_t>(stream));
  else hg::launch_norm<__half>(p, static_cast<cudaStream_t>(stream));
  HG_CATCH
}
