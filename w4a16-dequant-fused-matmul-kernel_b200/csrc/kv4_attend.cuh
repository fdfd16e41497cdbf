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
  int max_q;                 // most queries of a sequence (the workspace goes by it)
  int heads;
  int share;                 // query heads per kv head
  float scale;
  int window;                // 0: all
  int groups;
};

// The first token that the query at position `pos` sees; a window may be anything up to the largest int, and a
// position below zero (more new tokens than cached ones).
__device__ __forceinline__ int sees_from(const AttendParams& p, int pos) {
  return p.window && pos >= p.window ? pos - p.window + 1 : 0;
}

// A sequence's queries [first, first + count) and its cached tokens (none of what does not fit the
// arrays).
__device__ __forceinline__ void sequence(const AttendParams& p, int b, int& first, int& count, int& len) {
  if (p.cu_q) {
    first = p.cu_q[b];
    count = p.cu_q[b + 1] - first;
    if (first < 0 || count < 0 || count > p.max_q || first > p.T - count) {
      flag_error(kErrIndex);
      first = count = 0;
    }
  } else {
    count = p.T / p.seqs;
    first = b * count;
  }
  len = p.lens[b];
  if (len < 0 || len > p.width * p.cache.page_size) {
    flag_error(kErrIndex);
    len = 0;
  }
}

}  // namespace kv4
}  // namespace w4a16
