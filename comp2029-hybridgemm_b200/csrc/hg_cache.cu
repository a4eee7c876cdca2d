// A paged key-value cache held in MXFP8: quantising keys and values as they are written, and reading entries back.
//
// E4M3 codes with an E8M0 scale per 32 elements of a head, by the rule of hg_pack.  The layout is the one that
// hg_attention.cu's loads ask for (see hg_cache.cuh).  Both are bound by memory, and in small calls by their chain: slot, entry.  Eight
// heads of 128, bf16, random slots: 65536 tokens written in 65 us and read in 73 (0.95 and 0.86 of the measured copy rate), 2048 in 3.9 and
// 3.2 (0.50 and 0.61), 128 tokens of four heads in 1.3.
#include <type_traits>

#include "hg_cache.cuh"

namespace hg {
namespace {

// Eight threads to a token, head and key or value; each has four elements of every group of 32, whose 4 x GROUPS codes are consecutive in
// the cache.  A block has kTokens tokens of one head.
constexpr int kTokens = 8, kThreads = kTokens * 16;
// Tokens times heads from which a thread has two tokens: more loads are under way, but fewer SMs have some while there are few (one token
// and two, us: 16384 x 8 heads written 19.5, 18.4, read 19.1, 14.5; 2048 x 8 written 3.9, 4.9, read 3.2, 3.6; at 4096 x 8 written 6.4, 6.6,
// read 5.9, 4.8).
constexpr int kMany = 32768;
struct Place { uint8_t *codes, *scales; };   // of one thread's part of an entry
template <int GROUPS>
__device__ __forceinline__ Place place_of(const hg_cache& c, uint64_t by_page_size, uint32_t slot, int head, int kind, int x) {
  const uint32_t page = uint32_t(__umul64hi(slot, by_page_size)), at = slot - page * uint32_t(c.page_size);
  uint8_t* const record = static_cast<uint8_t*>(c.data) + (int64_t(page) * c.kv_heads + head) * cache_page_bytes(c.page_size, 32 * GROUPS);
  return {record + (kind * c.page_size + int(at)) * (32 * GROUPS) + x * (4 * GROUPS), record + 2 * c.page_size * (32 * GROUPS) + (2 * int(at) + kind) * GROUPS};
}

// EACH tokens to a thread, their loads under way together.
template <typename T, int GROUPS, int EACH>
__global__ void __launch_bounds__(kThreads)
cache_write_kernel(const hg_cache c, uint64_t by_page_size, const uint16_t* k, const uint16_t* v, int64_t k_token, int64_t k_head,
                   int64_t v_token, int64_t v_head, const int64_t* slots, int tokens) {
  pdl_trigger();
  const int x = threadIdx.x & 7, kind = (threadIdx.x >> 3) & 1, head = blockIdx.y;
  const int64_t first = int64_t(blockIdx.x) * (kTokens * EACH) + (threadIdx.x >> 4), stride = kind ? v_token : k_token;
  const uint16_t* const src = (kind ? v + head * v_head : k + head * k_head) + 4 * x;
  const unsigned mask = 0xffu << (threadIdx.x & 24);
  if (first >= tokens) return;
  pdl_wait();
  int64_t slot[EACH];
  uint2 raw[EACH][GROUPS];
#pragma unroll
  for (int i = 0; i < EACH; ++i) {
    slot[i] = -1;
    if (i && first + i * kTokens >= tokens) continue;   // whole groups of eight
    slot[i] = slots[first + i * kTokens];
#pragma unroll
    for (int g = 0; g < GROUPS; ++g) raw[i][g] = *reinterpret_cast<const uint2*>(src + (first + i * kTokens) * stride + 32 * g);
  }
#pragma unroll
  for (int i = 0; i < EACH; ++i) {
    if (uint64_t(slot[i]) >= uint64_t(c.pages) * uint64_t(c.page_size)) continue;
    const Place to = place_of<GROUPS>(c, by_page_size, uint32_t(slot[i]), head, kind, x);
    uint32_t codes[GROUPS], scales = 0;
    // The largest of two groups at once, as pairs of 16-bit values; a NaN is skipped.
    float top[GROUPS];
#pragma unroll
    for (int g = 0; g < GROUPS; g += 2) {
      const uint32_t a = Packed<T>::max_abs(Packed<T>::max_abs(0u, raw[i][g].x), raw[i][g].y), b = Packed<T>::max_abs(Packed<T>::max_abs(0u, raw[i][g + 1].x), raw[i][g + 1].y);
      uint32_t both = Packed<T>::max_abs(__byte_perm(a, b, 0x5410), __byte_perm(a, b, 0x7632));
#pragma unroll
      for (int step = 1; step < 8; step <<= 1) both = Packed<T>::max_abs(both, __shfl_xor_sync(mask, both, step));
      const float2 ends = Packed<T>::widen(both);
      top[g] = fmaxf(0.f, ends.x);
      top[g + 1] = fmaxf(0.f, ends.y);
    }
#pragma unroll
    for (int g = 0; g < GROUPS; ++g) {
      const int e = mx_exponent<false>(top[g]);
      const float inv = mx_inverse_scale(e);
      const float2 low = mul2(Packed<T>::widen(raw[i][g].x), make_float2(inv, inv)), high = mul2(Packed<T>::widen(raw[i][g].y), make_float2(inv, inv));
      codes[g] = cvt_e4m3x2(low.x, low.y) | (cvt_e4m3x2(high.x, high.y) << 16);
      scales |= uint32_t(e + 127) << (8 * g);
    }
    if constexpr (GROUPS == 4) *reinterpret_cast<uint4*>(to.codes) = make_uint4(codes[0], codes[1], codes[2], codes[3]);
    else *reinterpret_cast<uint2*>(to.codes) = make_uint2(codes[0], codes[1]);
    if (x == 0) {
      if constexpr (GROUPS == 4) *reinterpret_cast<uint32_t*>(to.scales) = scales;
      else *reinterpret_cast<uint16_t*>(to.scales) = uint16_t(scales);
    }
  }
}

template <typename T, int GROUPS, int EACH>
__global__ void __launch_bounds__(kThreads)
cache_read_kernel(const hg_cache c, uint64_t by_page_size, uint16_t* k, uint16_t* v, const int64_t* slots, int tokens) {
  pdl_trigger();
  const int x = threadIdx.x & 7, kind = (threadIdx.x >> 3) & 1, head = blockIdx.y;
  const int64_t first = int64_t(blockIdx.x) * (kTokens * EACH) + (threadIdx.x >> 4);
  uint16_t* const to = (kind ? v : k) + head * (32 * GROUPS) + 4 * x;
  pdl_wait();
  int64_t slot[EACH];
#pragma unroll
  for (int i = 0; i < EACH; ++i) slot[i] = first + i * kTokens < tokens ? slots[first + i * kTokens] : -1;
  uint32_t codes[EACH][GROUPS], scales[EACH];
#pragma unroll
  for (int i = 0; i < EACH; ++i) {
#pragma unroll
    for (int g = 0; g < GROUPS; ++g) codes[i][g] = 0;
    scales[i] = 0;
    if (uint64_t(slot[i]) >= uint64_t(c.pages) * uint64_t(c.page_size)) continue;
    const Place from = place_of<GROUPS>(c, by_page_size, uint32_t(slot[i]), head, kind, x);
    if constexpr (GROUPS == 4) {
      const uint4 raw = *reinterpret_cast<const uint4*>(from.codes);
      codes[i][0] = raw.x; codes[i][1] = raw.y; codes[i][2] = raw.z; codes[i][3] = raw.w;
      scales[i] = *reinterpret_cast<const uint32_t*>(from.scales);
    } else {
      const uint2 raw = *reinterpret_cast<const uint2*>(from.codes);
      codes[i][0] = raw.x; codes[i][1] = raw.y;
      scales[i] = *reinterpret_cast<const uint16_t*>(from.scales);
    }
  }
#pragma unroll
  for (int i = 0; i < EACH; ++i) {
    if (first + i * kTokens >= tokens) return;
    uint16_t* const row = to + (first + i * kTokens) * c.kv_heads * (32 * GROUPS);
#pragma unroll
    for (int g = 0; g < GROUPS; ++g) {
      const float scale = mx_scale(int(scales[i] >> (8 * g)) & 255);
      const float2 low = mul2(e4m3x2_to_float2(uint16_t(codes[i][g])), make_float2(scale, scale)), high = mul2(e4m3x2_to_float2(uint16_t(codes[i][g] >> 16)), make_float2(scale, scale));
      *reinterpret_cast<uint2*>(row + 32 * g) = make_uint2(Packed<T>::round(low), Packed<T>::round(high));
    }
  }
}

dim3 token_blocks(const hg_cache& c, int tokens, int each) { return dim3(unsigned((tokens + kTokens * each - 1) / (kTokens * each)), unsigned(c.kv_heads)); }
uint64_t inverse_of(int n) { return ~uint64_t(0) / uint64_t(n) + 1; }   // ceil(2^64 / n) for n > 1; exact for 32-bit dividends
bool aligned16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

}  // namespace

int sm_count() {
  static const int sms = [] {
    int device = 0, n = 148;
    if (cudaGetDevice(&device) != cudaSuccess || cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, device) != cudaSuccess) {
      cudaGetLastError();
      n = 148;
    }
    return n;
  }();
  return sms;
}

void validate_cache(const hg_cache& c) {
  if (!c.data || c.pages <= 0 || c.kv_heads <= 0) throw std::runtime_error("hg_cache: a cache has pages and heads");
  if (c.head_dim != 64 && c.head_dim != 128) throw std::runtime_error("hg_cache: head_dim must be 64 or 128");
  if (c.page_size <= 0 || c.page_size % 16 || c.page_size > 1024) throw std::runtime_error("hg_cache: page_size must be a multiple of 16 up to 1024");
  if (c.kv_heads > 65535 || int64_t(c.pages) * c.page_size > 0x7fffffff) throw std::runtime_error("hg_cache: too many heads or entries");
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
  const bool many = int64_t(tokens) * cache->kv_heads >= hg::kMany;
  const auto pick = [&](auto type, auto groups) {
    using T = decltype(type);
    constexpr int G = decltype(groups)::value;
    return many ? hg::cache_write_kernel<T, G, 2> : hg::cache_write_kernel<T, G, 1>;
  };
  using Two = std::integral_constant<int, 2>;
  using Four = std::integral_constant<int, 4>;
  const auto kernel = bf16 ? (wide ? pick(__nv_bfloat16{}, Four{}) : pick(__nv_bfloat16{}, Two{})) : (wide ? pick(__half{}, Four{}) : pick(__half{}, Two{}));
  hg::check(hg::launch_kernel(kernel, hg::token_blocks(*cache, tokens, many ? 2 : 1), dim3(hg::kThreads), 0, static_cast<cudaStream_t>(stream), *cache, hg::inverse_of(cache->page_size), kk, vv,
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
  const bool many = int64_t(tokens) * cache->kv_heads >= hg::kMany;
  const auto pick = [&](auto type, auto groups) {
    using T = decltype(type);
    constexpr int G = decltype(groups)::value;
    return many ? hg::cache_read_kernel<T, G, 2> : hg::cache_read_kernel<T, G, 1>;
  };
  using Two = std::integral_constant<int, 2>;
  using Four = std::integral_constant<int, 4>;
  const auto kernel = bf16 ? (wide ? pick(__nv_bfloat16{}, Four{}) : pick(__nv_bfloat16{}, Two{})) : (wide ? pick(__half{}, Four{}) : pick(__half{}, Two{}));
  hg::check(hg::launch_kernel(kernel, hg::token_blocks(*cache, tokens, many ? 2 : 1), dim3(hg::kThreads), 0, static_cast<cudaStream_t>(stream), *cache, hg::inverse_of(cache->page_size),
                              static_cast<uint16_t*>(k), static_cast<uint16_t*>(v), slots, tokens), "cache read");
  HG_CATCH
}

}  // extern "C"
