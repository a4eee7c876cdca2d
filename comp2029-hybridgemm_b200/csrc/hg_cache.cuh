// The paged MXFP8 cache, as its kernels see it.
#pragma once
#include "hg_common.cuh"

namespace hg {

// Per page and head, one after the other: key codes [page_size][head_dim], value codes [page_size][head_dim], scale bytes
// [page_size][keys, values][head_dim / 32].  A token's codes lie as [8][head_dim / 32][4], element d = 32 g + 4 x + i at
// (x, g, i): a lane that loads one run of head_dim / 8 bytes has four elements of every scale group, which is what the
// fragments of a matrix instruction take from it, for keys (summed over d) as for values (summed over tokens).
__host__ __device__ inline int64_t cache_page_bytes(int page_size, int head_dim) { return int64_t(page_size) * (2 * head_dim + head_dim / 16); }

void validate_cache(const hg_cache& c);   // throws

#ifdef __CUDACC__
// Two E4M3 codes to two halves (exact), the lower byte to the lower half.
__device__ __forceinline__ uint32_t e4m3x2_to_half2(uint16_t codes) {
  uint32_t r;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"(codes));
  return r;
}
__device__ __forceinline__ float2 e4m3x2_to_float2(uint16_t codes) { return Packed<__half>::widen(e4m3x2_to_half2(codes)); }
// 2^(byte - 127) as fp32; byte 0 is 2^-127.
__device__ __forceinline__ float mx_scale(int byte) { return __uint_as_float(byte ? uint32_t(byte) << 23 : 0x00400000u); }
#endif

}  // namespace hg
