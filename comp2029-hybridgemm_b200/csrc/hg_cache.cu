// A paged key-value cache held in MXFP8: quantising keys and values as they are written, and reading entries back.
//
// E4M3 codes with an E8M0 scale per 32 elements of a head, by the rule of hg_pack.  The layout is the one that
// hg_attention.cu's loads ask for (see hg_cache_layout in hg_cache.cuh).
#include <algorithm>

#include "hg_cache.cuh"

namespace hg {
namespace {

// Eight threads to a token, head and key or value; each has four elements of every group of 32, its 4 x GROUPS codes are consecutive in the cache.
template <typename T, int GROUPS>
__global__ void __launch_bounds__(256)
cache_write_kernel(const hg_cache c, const uint16_t* k, const uint16_t* v, int64_t k_token, int64_t k_head,
                   int64_t v_token, int64_t v_head, const int64_t* slots, int tokens) {
  pdl_trigger();
  const int64_t thread = int64_t(blockIdx.x) * blockDim.x + threadIdx.x;
  const int x = int(thread & 7);
  const int64_t row = thread >> 3;                       // token, head, key or value
  const int kind = int(row & 1);
  const int64_t pair = row >> 1;
  const int64_t token = pair / c.kv_heads;
  const int head = int(pair - token * c.kv_heads);
  pdl_wait();
  if (token >= tokens) return;                           // whole groups of eight
  const int64_t slot = slots[token];
  if (slot < 0 || slot >= int64_t(c.pages) * c.page_size) return;
  const unsigned mask = 0xffu << (threadIdx.x & 24);
  const uint16_t* const src = (kind ? v + token * v_token + head * v_head : k + token * k_token + head * k_head) + 4 * x;
  uint2 raw[GROUPS];
#pragma unroll
  for (int g = 0; g < GROUPS; ++g) raw[g] = *reinterpret_cast<const uint2*>(src + 32 * g);
  const int64_t page = slot / c.page_size;
  const int at = int(slot - page * c.page_size);
  uint8_t* const record = static_cast<uint8_t*>(c.data) + (page * c.kv_heads + head) * cache_page_bytes(c.page_size, 32 * GROUPS);
  uint32_t codes[GROUPS], scales = 0;
#pragma unroll
  for (int g = 0; g < GROUPS; ++g) {
    const float2 low = Packed<T>::widen(raw[g].x), high = Packed<T>::widen(raw[g].y);
    float amax = fmaxf(fmaxf(fmaxf(0.f, fabsf(low.x)), fabsf(low.y)), fmaxf(fabsf(high.x), fabsf(high.y)));
#pragma unroll
    for (int step = 1; step < 8; step <<= 1) amax = fmaxf(amax, __shfl_xor_sync(mask, amax, step));
    const int e = mx_exponent<false>(amax);
    const float inv = mx_inverse_scale(e);
    codes[g] = cvt_e4m3x2(low.x * inv, low.y * inv) | (cvt_e4m3x2(high.x * inv, high.y * inv) << 16);
    scales |= uint32_t(e + 127) << (8 * g);
  }
  uint8_t* const to = record + (int64_t(kind) * c.page_size + at) * (32 * GROUPS) + x * (4 * GROUPS);
  if constexpr (GROUPS == 4) *reinterpret_cast<uint4*>(to) = make_uint4(codes[0], codes[1], codes[2], codes[3]);
  else *reinterpret_cast<uint2*>(to) = make_uint2(codes[0], codes[1]);
  uint8_t* const scale = record + int64_t(2) * c.page_size * (32 * GROUPS) + (2 * at + kind) * GROUPS;
  if (x == 0) {
    if constexpr (GROUPS == 4) *reinterpret_cast<uint32_t*>(scale) = scales;
    else *reinterpret_cast<uint16_t*>(scale) = uint16_t(scales);
  }
}

template <typename T, int GROUPS>
__global__ void __launch_bounds__(256)
cache_read_kernel(const hg_cache c, uint16_t* k, uint16_t* v, const int64_t* slots, int tokens) {
  pdl_trigger();
  const int64_t thread = int64_t(blockIdx.x) * blockDim.x + threadIdx.x;
  const int x = int(thread & 7);
  const int64_t row = thread >> 3;
  const int kind = int(row & 1);
  const int64_t pair = row >> 1;
  const int64_t token = pair / c.kv_heads;
  const int head = int(pair - token * c.kv_heads);
  pdl_wait();
  if (token >= tokens) return;
  const int64_t slot = slots[token];
  uint32_t codes[GROUPS] = {}, scales = 0;
  if (slot >= 0 && slot < int64_t(c.pages) * c.page_size) {
    const int64_t page = slot / c.page_size;
    const int at = int(slot - page * c.page_size);
    const uint8_t* const record = static_cast<const uint8_t*>(c.data) + (page * c.kv_heads + head) * cache_page_bytes(c.page_size, 32 * GROUPS);
    const uint8_t* const from = record + (int64_t(kind) * c.page_size + at) * (32 * GROUPS) + x * (4 * GROUPS);
    const uint8_t* const scale = record + int64_t(2) * c.page_size * (32 * GROUPS) + (2 * at + kind) * GROUPS;
    if constexpr (GROUPS == 4) {
      const uint4 raw = *reinterpret_cast<const uint4*>(from);
      codes[0] = raw.x; codes[1] = raw.y; codes[2] = raw.z; codes[3] = raw.w;
      scales = *reinterpret_cast<const uint32_t*>(scale);
    } else {
      const uint2 raw = *reinterpret_cast<const uint2*>(from);
      codes[0] = raw.x; codes[1] = raw.y;
      scales = *reinterpret_cast<const uint16_t*>(scale);
    }
  }
  uint16_t* const to = (kind ? v : k) + pair * (32 * GROUPS) + 4 * x;
#pragma unroll
  for (int g = 0; g < GROUPS; ++g) {
    const float scale = mx_scale(int(scales >> (8 * g)) & 255);
    const float2 low = e4m3x2_to_float2(uint16_t(codes[g])), high = e4m3x2_to_float2(uint16_t(codes[g] >> 16));
    *reinterpret_cast<uint2*>(to + 32 * g) = make_uint2(
        uint32_t(from_float<T>(low.x * scale)) | (uint32_t(from_float<T>(low.y * scale)) << 16),
        uint32_t(from_float<T>(high.x * scale)) | (uint32_t(from_float<T>(high.y * scale)) << 16));
  }
}

unsigned row_blocks(const hg_cache& c, int tokens) {
  const int64_t blocks = (int64_t(tokens) * c.kv_heads * 16 + 255) / 256;
  if (blocks > 0x7fffffff) throw std::runtime_error("hg_cache: too many tokens in one call");
  return unsigned(blocks);
}
bool aligned16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

}  // namespace

void validate_cache(const hg_cache& c) {
  if (!c.data || c.pages <= 0 || c.kv_heads <= 0) throw std::runtime_error("hg_cache: a cache has pages and heads");
  if (c.head_dim != 64 && c.head_dim != 128) throw std::runtime_error("hg_cache: head_dim must be 64 or 128");
  if (c.page_size <= 0 || c.page_size % 16 || c.page_size > 1024) throw std::runtime_error("hg_cache: page_size must be a multiple of 16 up to 1024");
  if (!aligned16(c.data)) throw std::runtime_error("hg_cache: data must be aligned to 16 bytes");
}

}  // namespace hg

extern "C" {

int64_t hg_cache_page_bytes(int page_size, int head_dim) { return hg::cache_page_bytes(page_size, head_dim); }

int hg_cache_write(const hg_cache* cache, const void* k, const void* v, const int64_t* strides, const int64_t* slots, int tokens, int dtype, void* stream) {
  HG_TRY
  if (!cache || !strides) throw std::runtime_error("Null argument to hg_cache_write");
  hg::validate_cache(*cache);
  if (tokens < 0 || (dtype != HG_DTYPE_F16 && dtype != HG_DTYPE_BF16)) throw std::runtime_error("hg_cache_write: invalid tokens or dtype");
  if (tokens == 0) return 0;
  if (!k || !v || !slots) throw std::runtime_error("Null argument to hg_cache_write");
  if (reinterpret_cast<uintptr_t>(k) % 8 || reinterpret_cast<uintptr_t>(v) % 8 || reinterpret_cast<uintptr_t>(slots) % 8)
    throw std::runtime_error("hg_cache_write: keys and values must be aligned to 8 bytes");
  for (int i = 0; i < 4; ++i)
    if (strides[i] % 4) throw std::runtime_error("hg_cache_write: strides must be multiples of four elements");
  const auto* kk = static_cast<const uint16_t*>(k);
  const auto* vv = static_cast<const uint16_t*>(v);
  const bool bf16 = dtype == HG_DTYPE_BF16, wide = cache->head_dim == 128;
  const auto kernel = bf16 ? (wide ? hg::cache_write_kernel<__nv_bfloat16, 4> : hg::cache_write_kernel<__nv_bfloat16, 2>)
                           : (wide ? hg::cache_write_kernel<__half, 4> : hg::cache_write_kernel<__half, 2>);
  hg::check(hg::launch_kernel(kernel, dim3(hg::row_blocks(*cache, tokens)), dim3(256), 0, static_cast<cudaStream_t>(stream), *cache, kk, vv,
                              strides[0], strides[1], strides[2], strides[3], slots, tokens), "cache write");
  HG_CATCH
}

int hg_cache_read(const hg_cache* cache, void* k, void* v, const int64_t* slots, int tokens, int dtype, void* stream) {
  HG_TRY
  if (!cache) throw std::runtime_error("Null argument to hg_cache_read");
  hg::validate_cache(*cache);
  if (tokens < 0 || (dtype != HG_DTYPE_F16 && dtype != HG_DTYPE_BF16)) throw std::runtime_error("hg_cache_read: invalid tokens or dtype");
  if (tokens == 0) return 0;
  if (!k || !v || !slots) throw std::runtime_error("Null argument to hg_cache_read");
  if (!hg::aligned16(k) || !hg::aligned16(v) || reinterpret_cast<uintptr_t>(slots) % 8) throw std::runtime_error("hg_cache_read: outputs must be aligned to 16 bytes");
  const bool bf16 = dtype == HG_DTYPE_BF16, wide = cache->head_dim == 128;
  const auto kernel = bf16 ? (wide ? hg::cache_read_kernel<__nv_bfloat16, 4> : hg::cache_read_kernel<__nv_bfloat16, 2>)
                           : (wide ? hg::cache_read_kernel<__half, 4> : hg::cache_read_kernel<__half, 2>);
  hg::check(hg::launch_kernel(kernel, dim3(hg::row_blocks(*cache, tokens)), dim3(256), 0, static_cast<cudaStream_t>(stream), *cache,
                              static_cast<uint16_t*>(k), static_cast<uint16_t*>(v), slots, tokens), "cache read");
  HG_CATCH
}

}  // extern "C"
