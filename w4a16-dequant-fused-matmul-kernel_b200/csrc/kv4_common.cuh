// kv4_common.cuh -- the 4-bit paged key/value cache: its byte layout and the helpers its
// kernels share.
//
// A cached value is offset + scale * code, code in 0..15, with one fp16 (scale, offset)
// pair per token, kv head and group of G channels (G divides the head dimension D). A block
// holds 16 tokens of one kv head:
//   key codes    [16][D / 2] bytes   channel 2i in the low nibble of byte i (so a 32-bit word
//                                    holds channels 8w .. 8w + 7, channel 8w + j in nibble j,
//                                    the order of qweight's words)
//   value codes  [16][D / 2] bytes
//   key pairs    [16][D / G] (scale, offset) fp16
//   value pairs  [16][D / G] (scale, offset) fp16
// A page is page_size / 16 consecutive blocks per kv head and the pool is
// [layers][pages][kv heads][page_size / 16][block]. Sixteen tokens are what one step of the
// attention kernels' matrix instructions takes, so whatever the page size (a multiple of 16)
// a block arrives with one contiguous copy of a multiple of 16 bytes.
#pragma once

#include <type_traits>

#include "common.cuh"

namespace w4a16 {
namespace kv4 {

constexpr int BLK = 16;                       // tokens per block
constexpr float kMaxF16 = 65504.0f;           // keys and values beyond it are stored as it

__host__ __device__ constexpr int block_bytes(int D, int groups) { return BLK * (D + 8 * groups); }
__host__ __device__ constexpr int value_codes_at(int D) { return BLK * (D / 2); }
__host__ __device__ constexpr int key_pairs_at(int D) { return BLK * D; }
__host__ __device__ constexpr int value_pairs_at(int D, int groups) { return BLK * D + BLK * groups * 4; }

// Division of n < 2^31 by a number that the host knows: one multiplication, one addition and one
// shift, where the instruction sequence of a division takes about twenty.
// With s = ceil(log2 d) and m = floor(2^32 (2^s - d) / d) + 1, n / d = (hi(n m) + n) >> s.
struct Divisor {
  uint32_t m, s;
  Divisor() = default;
  explicit Divisor(uint32_t d) : m(0), s(0) {
    while (s < 31 && (1u << s) < d) ++s;
    m = static_cast<uint32_t>(((((1ull << s) - d) << 32) / d) + 1);
  }
  __device__ __forceinline__ uint32_t quotient(uint32_t n) const { return (__umulhi(n, m) + n) >> s; }
};

// The cache as the kernels see it (one layer's pool for all but the page copies).
struct CacheView {
  uint8_t* pool;            // first byte of the layer
  long long pages;          // pages of a layer
  int kv_heads;
  int page_size;            // tokens per page
  int page_blocks;          // page_size / 16
  Divisor blocks;           // by page_blocks
  int block_bytes;
  long long page_bytes;     // bytes of a page of one kv head
};

__device__ __forceinline__ uint8_t* block_ptr(const CacheView& c, long long page, int head, int block) {
  return c.pool + (page * c.kv_heads + head) * c.page_bytes + static_cast<long long>(block) * c.block_bytes;
}

template <typename T>
__device__ __forceinline__ float to_f32(T v);
template <>
__device__ __forceinline__ float to_f32<__half>(__half v) { return __half2float(v); }
template <>
__device__ __forceinline__ float to_f32<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
// Two fp32 values rounded to T, packed (lo in the low half).
template <typename T>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  if constexpr (std::is_same<T, __half>::value) {
    const __half2 v = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
  } else {
    const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
  }
}

}  // namespace kv4
}  // namespace w4a16
