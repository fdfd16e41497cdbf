// kv4_attend.cuh -- attention over the 4-bit paged cache: o = softmax(scale q k^T) v over the
// cached tokens a query may see. Query i of a sequence with n cached tokens, m of them new,
// stands at position n - m + i and sees tokens t with t <= position (and t > position - window
// when there is one). A query that sees nothing gives zeros and a log-sum-exp of -inf.
#pragma once

#include "kv4_common.cuh"

namespace w4a16 {
namespace kv4 {

struct AttendParams {
  const void* q;             // [T, heads, D], channels contiguous
  long long q_st, q_sh;      // strides, in elements
  void* o;                   // [T, heads, D] dense
  float* lse;                // [T, heads] or null
  CacheView cache;
  const int* table;          // [seqs, width] page ids
  int width;
  const int* lens;           // [seqs] cached tokens, the new ones among them
  const int* cu_q;           // [seqs + 1] first query of each sequence, or null: T / seqs each
  int seqs;
  int T;
  int heads;
  int share;                 // query heads per kv head
  float scale;
  int window;                // 0: all
  int groups;
};

// A sequence's queries [first, first + count) and its cached tokens.
__device__ __forceinline__ void sequence(const AttendParams& p, int b, int& first, int& count, int& len) {
  if (p.cu_q) {
    first = p.cu_q[b];
    count = p.cu_q[b + 1] - first;
  } else {
    count = p.T / p.seqs;
    first = b * count;
  }
  len = min(max(p.lens[b], 0), p.width * p.cache.page_size);
}

// One warp per query and head; 32 tokens at a time, one per lane for the scores, four (two)
// channels per lane for the sums.
template <typename T, int D>
__global__ void __launch_bounds__(128) kv4_attend_simple_kernel(const AttendParams p) {
  __shared__ float qs[4][D];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const long long row = blockIdx.x * 4LL + warp;
  if (row >= static_cast<long long>(p.T) * p.heads) return;
  const int tq = static_cast<int>(row / p.heads), h = static_cast<int>(row % p.heads), kh = h / p.share;
  int b = 0;
  if (p.cu_q) {
    int lo = 0, hi = p.seqs - 1;
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (p.cu_q[mid] <= tq) lo = mid; else hi = mid - 1;
    }
    b = lo;
  } else {
    b = tq / (p.T / p.seqs);
  }
  int first, count, len;
  sequence(p, b, first, count, len);
  const int pos = len - count + tq - first;
  const int to = min(len, pos + 1);                                   // tokens [from, to)
  const int from = p.window && pos - p.window + 1 > 0 ? pos - p.window + 1 : 0;
  const T* q = static_cast<const T*>(p.q) + tq * p.q_st + h * p.q_sh;
  for (int i = lane; i < D; i += 32) qs[warp][i] = to_f32<T>(q[i]) * p.scale;
  __syncwarp();
  constexpr int C = D / 32;
  float acc[C] = {}, m = -INFINITY, sum = 0.0f;
  const int G = D / p.groups;
  for (int t0 = from / 32 * 32; t0 < to; t0 += 32) {
    const int t = t0 + lane;
    float s = -INFINITY;
    int page = -1;
    if (t >= from && t < to) {
      page = p.table[static_cast<long long>(b) * p.width + t / p.cache.page_size];
      if (page < 0 || page >= p.cache.pages) {
        flag_error(kErrIndex);
        page = -1;
      }
    }
    if (page >= 0) {
      const int in_page = t % p.cache.page_size;
      const uint8_t* blk = block_ptr(p.cache, page, kh, in_page / BLK);
      const int tok = in_page % BLK;
      const uint32_t* codes = reinterpret_cast<const uint32_t*>(blk + tok * (D / 2));
      const __half2* pairs = reinterpret_cast<const __half2*>(blk + key_pairs_at(D)) + tok * p.groups;
      s = 0.0f;
      for (int w = 0; w < D / 8; ++w) {
        const float2 so = __half22float2(pairs[w * 8 / G]);
        const uint32_t c = codes[w];
#pragma unroll
        for (int j = 0; j < 8; ++j)
          s += qs[warp][8 * w + j] * (so.x * static_cast<float>((c >> (4 * j)) & 15u) + so.y);
      }
    }
    float mx = s;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
    if (mx == -INFINITY) continue;
    const float mn = fmaxf(m, mx), e = expf(s - mn), f = expf(m - mn);
    m = mn;
    sum = sum * f + e;
#pragma unroll
    for (int i = 0; i < C; ++i) acc[i] *= f;
    for (int j = 0; j < 32; ++j) {
      const float e1 = __shfl_sync(0xffffffffu, e, j);
      const int page1 = __shfl_sync(0xffffffffu, page, j);
      if (page1 < 0) continue;
      const int in_page = (t0 + j) % p.cache.page_size;
      const uint8_t* blk = block_ptr(p.cache, page1, kh, in_page / BLK);
      const int tok = in_page % BLK;
      const uint8_t* codes = blk + value_codes_at(D) + tok * (D / 2);
      const __half2* pairs = reinterpret_cast<const __half2*>(blk + value_pairs_at(D, p.groups)) + tok * p.groups;
#pragma unroll
      for (int i = 0; i < C; ++i) {
        const int d = lane * C + i;
        const float2 so = __half22float2(pairs[d / G]);
        acc[i] += e1 * (so.x * static_cast<float>((codes[d / 2] >> (4 * (d & 1))) & 15u) + so.y);
      }
    }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  T* out = static_cast<T*>(p.o) + row * D;
#pragma unroll
  for (int i = 0; i < C; ++i) out[lane * C + i] = from_f32<T>(sum > 0.0f ? acc[i] / sum : sum != sum ? sum : 0.0f);
  if (p.lse && lane == 0) p.lse[row] = sum > 0.0f ? m + logf(sum) : sum != sum ? sum : -INFINITY;
}

}  // namespace kv4
}  // namespace w4a16
