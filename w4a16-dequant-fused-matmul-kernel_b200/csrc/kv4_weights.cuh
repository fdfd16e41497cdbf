// kv4_weights.cuh -- the attention weight that cached tokens collect: for every token and kv head the sum, over the
// queries of its sequence that see it and the heads of the group, of p = exp(scale q . k - lse), lse the
// log-sum-exp that the attention of the same call gave. It is added to what the token had; a token that is new in
// this call (one of its queries' own positions) had nothing.
//
// The scores are those of the attention kernels, from the cache's codes: q . k = s_k (q . c) + b_k sum(q) per group of
// channels, codes masked out of their words as fp16 subnormals, queries scaled by a power of two of their own row
// (kv4_decode.cuh has the arithmetic). Tokens are the M side of mma.m16n8k16, eight query rows its N side, so
// the sum over rows stays in a lane but for its last two steps. Scores, exponentials and sums are fp32. The scaled
// queries are fp16 operands: channels down to 2^-24 of their row's largest are exact (odd nibbles hold 1/16 of
// theirs), smaller ones within 2^-35 of it, less than the fp32 sum rounds off.
//
// A launch before (kv4_weights_prep_kernel) writes the queries in the order of the second operand's fragments, with
// what a row's scores need (factor, sums, -lse log2(e)) beside them, and the prefix sums of the sequences' chunks:
// 64 tokens of a kv head. The chunks of all form one list that the warps of the second launch split evenly. Each
// warp feeds itself: while it goes over the rows that see a chunk, the next one's keys are copied into its other
// stage. Each sum has one owner and a fixed order, so results do not depend on timing. Sequences of more than 64 rows
// a kv head go to the tensor-memory kernel further down.
//
// Memory-bound by design (a token's keys are half of what the attention reads, and four bytes in and out), but no
// unit is full: 64 sequences of up to 8000 tokens, 64 heads of 128 channels on 8 kv heads (172 MB) 49 us, 3.5 TB/s,
// issue slots 56%, ALU pipe 49% (the codes' masks), 23% of an SM's warps there. What is left is latency: a warp
// waits 1.6 cycles an instruction for its own results and 1.4 for memory, with one chunk in flight. Three blocks an SM, of
// 80 registers and with spills, took 70 us; divisions by the group's heads 2.5 of now 49. One token over 777: 7 us, both
// launches.
#pragma once

#include "kv4_prefill.cuh"

namespace w4a16 {
namespace kv4 {

constexpr int WT_THREADS = 256, WT_WARPS = WT_THREADS / 32, WT_PER_SM = 2;
constexpr int WT_BLOCKS = 4, WT_TOKENS = WT_BLOCKS * BLK;       // blocks and tokens of a chunk
constexpr int WT_PREP = 256;

// Of a tile of eight rows: fragment words [D / 32][32 lanes][4], then eight rows' (factor, sum of group 0, sum of
// the last group, -lse log2(e)), then whether a row has a log-sum-exp of -inf. (Rows behind the last have channels and
// sums of 0 and -inf for the last: they give nothing to a token with a finite pair. One whose pair is not is NaN
// to the rows that see it.)
__host__ __device__ constexpr int wt_tile_words(int D) { return D / 32 * 128 + 8 * 4 + 4; }

struct WeightsParams {
  AttendParams a;            // lse is an input here, o unused
  const float* lse;          // [T, heads]
  const float* before;       // [seqs, kv heads, capacity]
  float* after;              // the same, may be `before`
  long long b_ss, b_sh, a_ss, a_sh;
  int capacity;
  int bf16;
  int tiles;                 // tiles of eight rows of a kv head: T share / 8 + seqs
  long long* prefix;         // [seqs + 1] chunks before a sequence
  uint32_t* queries;         // [kv heads][tiles][wt_tile_words]
  // sequences of more than `row_limit` rows a kv head (kv4_weights_tc_kernel)
  int row_limit;
  int tc_tiles;              // tiles of TcShape::N rows of a kv head: T share / N + seqs
  long long* tc_prefix;      // [seqs + 1] entries (WT_TC_TOKENS tokens) before a sequence
  long long* tc_steps;       // [entries + 1] steps (N rows of a kv head) before an entry
  uint8_t* tc_queries;       // [kv heads][tc_tiles][TcShape::TILE_BYTES]
  float* parts;              // [blocks][2][WT_TC_TOKENS] sums of tiles that several blocks share
  long long entries;         // that there is room for: all, unless cu_q gives queries to several sequences
  int blocks;
  unsigned long long wait_ns;
  int copies;                // blocks of the first launch that copy (0 in place)
};

template <int D, int NG>
struct WeightsShape {
  static constexpr int CODES = BLK * (D / 2), PAIRS = BLK * NG * 4, KEYS = CODES + PAIRS;   // of a block's keys
  static constexpr int STAGE = WT_BLOCKS * KEYS;
  static constexpr int SMEM_BYTES = WT_WARPS * 2 * (STAGE + 8);
  static_assert(WT_PER_SM * (SMEM_BYTES + 1024) <= 228 * 1024, "shared memory budget");
};

// The second kernel's shapes: tokens of a tile, rows of a step (two groups of channels have a product each).
constexpr int WT_TC_TOKENS = 512, WT_TC_QUARTERS = WT_TC_TOKENS / 128, WT_TC_SOFTMAX = 4 * WT_TC_QUARTERS;
constexpr int WT_TC_ISSUERS = 2, WT_TC_THREADS = (WT_TC_SOFTMAX + 1 + WT_TC_ISSUERS) * 32;   // (20 warps have 96 registers, 24 have 80)
constexpr int WT_TC_LEAST = 4;   // steps of a block, at least
template <int D, int NG>
struct TcShape {
  static constexpr int KB = D / 64, N = NG == 2 ? 64 : 128;
  // a step's queries as they lie in shared memory, two float4 for each two rows, a byte for each eight
  static constexpr int CONSTS_AT = N * D * 2, FLAGS_AT = CONSTS_AT + N * 16, TILE_BYTES = FLAGS_AT + 16;
  static constexpr int STAGE = (TILE_BYTES + 1023) / 1024 * 1024, RING = NG * D == 128 ? 2 : 4;
  static constexpr int KEY_BYTES = WT_TC_QUARTERS * KB * PF_TILE;
  static constexpr int SMEM_BYTES = 1024 + KEY_BYTES + RING * STAGE + 256;
  static_assert(SMEM_BYTES <= 227 * 1024, "shared memory budget");
};

// A sequence's first tile of eight rows. Sequences in order leave room for each one's last, partly filled tile.
__device__ __forceinline__ long long wt_first_tile(const AttendParams& a, int b, int first, int rows = 8) {
  return static_cast<long long>(first) * a.share / rows + b;
}

// Chunks of a sequence that some query sees: sinks' first, then the window's. Where the sums do not go where they were,
// what the other tokens have is copied: by the first launch, or (entries of the tensor-memory kernel, which are
// all of a sequence's then) by the join.
struct Chunks {
  int sinks, skip, n;        // chunk g is chunk g of the sequence below `sinks`, else chunk g + skip
};
template <int TOKENS = WT_TOKENS>
__device__ __forceinline__ Chunks wt_chunks(const WeightsParams& p, int count, int len) {
  Chunks c = {0, 0, (len + TOKENS - 1) / TOKENS};
  if (TOKENS == WT_TOKENS) {
    if (count == 0) {
      c.skip = c.n;
      c.n = 0;
      return c;
    }
    if (p.a.window == 0) return c;
  } else if (p.before != p.after) {
    return c;
  }
  const int first = sees_from(p.a, len - count) / TOKENS;
  c.sinks = min((min(p.a.sinks, len) + TOKENS - 1) / TOKENS, first);
  c.skip = first - c.sinks;
  c.n = max(0, c.n - c.skip);
  return c;
}

__device__ __forceinline__ void wt_sequence(const WeightsParams& p, int b, int& first, int& count, int& len) {
  sequence(p.a, b, first, count, len);
  if (len > p.capacity) {
    flag_error(kErrIndex);
    len = 0;
  }
}

// Whether a sequence is the tensor-memory kernel's, and its parts.
__device__ __forceinline__ bool wt_many(const WeightsParams& p, int count) {
  return static_cast<long long>(count) * p.a.share > p.row_limit;
}

// WT_TC_TOKENS tokens of a kv head against the rows that see some of them, in steps of N rows.
struct TcTile {
  int b, g, kh;              // sequence, entry of the sequence, kv head
  int first, count, len;
  Chunks c;
  int t0, j0, n;             // first token, first step, steps
  __device__ __forceinline__ int pos0() const { return len - count; }
};
__device__ __forceinline__ int wt_row_from(const WeightsParams& p, const TcTile& s, int t) { return max(0, t - s.pos0()) * p.a.share; }
// The first row behind those that see token t.
__device__ __forceinline__ int wt_row_to(const WeightsParams& p, const TcTile& s, int t) {
  const int rows = s.count * p.a.share;
  if (!p.a.window || t < p.a.sinks) return rows;
  return static_cast<int>(min(static_cast<long long>(rows), max(0LL, static_cast<long long>(t) + p.a.window - s.pos0()) * p.a.share));
}
template <int N>
__device__ __forceinline__ void wt_tile_rows(const WeightsParams& p, TcTile& s) {
  s.t0 = (s.g < s.c.sinks ? s.g : s.g + s.c.skip) * WT_TC_TOKENS;
  const int lo = wt_row_from(p, s, s.t0);
  const int hi = s.t0 < p.a.sinks ? s.count * p.a.share : wt_row_to(p, s, min(s.t0 + WT_TC_TOKENS, s.len) - 1);
  s.j0 = lo / N;
  s.n = hi > lo ? (hi + N - 1) / N - s.j0 : 0;
}
__device__ __forceinline__ void wt_tile_sequence(const WeightsParams& p, TcTile& s) {
  wt_sequence(p, s.b, s.first, s.count, s.len);
  s.c = wt_chunks<WT_TC_TOKENS>(p, s.count, s.len);
  if (!wt_many(p, s.count)) s.c.n = 0;
}
// The next tile with steps: heads of an entry, entries of a sequence, sequences (there is one).
template <int N>
__device__ __forceinline__ void wt_next_tile(const WeightsParams& p, TcTile& s) {
  if (++s.kh < p.a.cache.kv_heads) return;
  s.kh = 0;
  for (;;) {
    if (++s.g >= s.c.n) {
      if (s.b + 1 >= p.a.seqs) return;
      ++s.b;
      s.g = -1;
      wt_tile_sequence(p, s);
      continue;
    }
    wt_tile_rows<N>(p, s);
    if (s.n > 0) return;
  }
}

// The last entry of an ascending list of n at or below x, with every lane of a warp.
template <typename At>
__device__ __forceinline__ int wt_search(int n, At at_or_below) {
  const int lane = threadIdx.x & 31;
  int lo = 0, hi = n - 1;
  while (lo < hi) {
    const int step = (hi - lo + 31) / 32, b = lo + step * (lane + 1);
    const int past = __popc(__ballot_sync(0xffffffffu, b <= hi && at_or_below(min(b, hi))));
    lo += past * step;
    hi = min(hi, lo + step - 1);
  }
  return lo;
}

// Block 0: the prefix sums. The next ones: a warp per tile of eight rows of a kv head. The last `copies`: what tokens that
// nobody sees have.
template <int D, int NG>
__global__ void __launch_bounds__(WT_PREP) kv4_weights_prep_kernel(const WeightsParams p) {
  constexpr int KW = D / 32;
  let_next_launch();
  const AttendParams& a = p.a;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (blockIdx.x == 0) {
    __shared__ long long warp_sums[2][WT_PREP / 32];
    long long sum[2] = {0, 0};
    for (int base = 0; base < a.seqs; base += WT_PREP) {
      const int b = base + threadIdx.x;
      long long v[2] = {0, 0}, inc[2];
      if (b < a.seqs) {
        int first, count, len;
        wt_sequence(p, b, first, count, len);
        if (wt_many(p, count)) v[1] = wt_chunks<WT_TC_TOKENS>(p, count, len).n;
        else v[0] = static_cast<long long>(wt_chunks(p, count, len).n) * a.cache.kv_heads;
      }
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        inc[k] = v[k];
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const long long x = __shfl_up_sync(0xffffffffu, inc[k], o);
          if (lane >= o) inc[k] += x;
        }
      }
      __syncthreads();
      if (lane == 31) {
        warp_sums[0][warp] = inc[0];
        warp_sums[1][warp] = inc[1];
      }
      __syncthreads();
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        long long before = sum[k];
#pragma unroll
        for (int w = 0; w < WT_PREP / 32; ++w) {
          before += w < warp ? warp_sums[k][w] : 0;
          sum[k] += warp_sums[k][w];
        }
        if (b < a.seqs) (k ? p.tc_prefix : p.prefix)[b] = before + inc[k] - v[k];
      }
    }
    const long long entries = min(sum[1], p.entries);
    if (threadIdx.x == 0) {
      if (sum[1] > p.entries) flag_error(kErrIndex);
      p.prefix[a.seqs] = sum[0];
      p.tc_prefix[a.seqs] = entries;
    }
    if (entries == 0) {
      if (threadIdx.x == 0 && p.tc_steps) p.tc_steps[0] = 0;
      return;
    }
    __syncthreads();                     // tc_prefix is written
    long long steps = 0;
    for (long long base = 0; base < entries; base += WT_PREP) {
      const long long e = base + threadIdx.x;
      long long v = 0;
      if (e < entries) {
        TcTile s;
        int lo = 0, hi = a.seqs - 1;     // the last sequence that begins at or before it
        while (lo < hi) {
          const int mid = (lo + hi + 1) >> 1;
          if (p.tc_prefix[mid] <= e) lo = mid; else hi = mid - 1;
        }
        s.b = lo;
        s.g = static_cast<int>(e - p.tc_prefix[lo]);
        wt_tile_sequence(p, s);
        wt_tile_rows<TcShape<D, NG>::N>(p, s);
        v = static_cast<long long>(s.n) * a.cache.kv_heads;
      }
      long long inc = v;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const long long x = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += x;
      }
      __syncthreads();
      if (lane == 31) warp_sums[0][warp] = inc;
      __syncthreads();
      long long before = steps;
#pragma unroll
      for (int w = 0; w < WT_PREP / 32; ++w) {
        before += w < warp ? warp_sums[0][w] : 0;
        steps += warp_sums[0][w];
      }
      if (e < entries) p.tc_steps[e] = before + inc - v;
    }
    if (threadIdx.x == 0) p.tc_steps[entries] = steps;
    return;
  }
  if (blockIdx.x >= gridDim.x - p.copies) {
    for (long long i = blockIdx.x - (gridDim.x - p.copies); i < static_cast<long long>(a.seqs) * a.cache.kv_heads; i += p.copies) {
      const int b = static_cast<int>(i / a.cache.kv_heads), kh = static_cast<int>(i - static_cast<long long>(b) * a.cache.kv_heads);
      int first, count, len;
      wt_sequence(p, b, first, count, len);
      if (wt_many(p, count)) continue;           // (the join's)
      const Chunks c = wt_chunks(p, count, len);
      const int end = min(len, (c.sinks + c.skip) * WT_TOKENS);
      const float* from = p.before + b * p.b_ss + kh * p.b_sh;
      float* to = p.after + b * p.a_ss + kh * p.a_sh;
#pragma unroll 4
      for (int t = c.sinks * WT_TOKENS + threadIdx.x; t < end; t += WT_PREP) to[t] = from[t];
    }
    return;
  }
  const long long item = (blockIdx.x - 1) * static_cast<long long>(WT_PREP / 32) + warp;
  if (item >= static_cast<long long>(p.tiles) * a.cache.kv_heads) return;
  const int kh = static_cast<int>(item % a.cache.kv_heads), tile = static_cast<int>(item / a.cache.kv_heads);
  // the last sequence that begins at or before the tile
  const int lo = wt_search(a.seqs, [&](int b) {
    return wt_first_tile(a, b, a.cu_q ? min(max(a.cu_q[b], 0), a.T) : b * (a.T / a.seqs)) <= tile;
  });
  int first, count, len;
  wt_sequence(p, lo, first, count, len);
  const int t = tile - static_cast<int>(wt_first_tile(a, lo, first));
  if (t < 0 || static_cast<long long>(t) * 8 >= static_cast<long long>(count) * a.share) return;
  const int r = lane >> 2, q4 = lane & 3;
  const int row = t * 8 + r;
  const bool live = row < count * a.share;
  const uint16_t* src = static_cast<const uint16_t*>(a.q);
  float nlse = -INFINITY;
  if (live) {
    const int token = first + row / a.share, head = kh * a.share + row % a.share;
    src += token * a.q_st + head * a.q_sh;
    const float lse = p.lse[static_cast<long long>(token) * a.heads + head];
    if (lse != -INFINITY) nlse = -lse * kLog2e;
  }
  auto key_word = [&](int i) { return NG == 1 ? KW * q4 + i : (i < 2 ? 2 * q4 + i : 8 + 2 * q4 + i - 2); };
  float x[KW][8], sum[NG] = {}, top = 0.0f;
#pragma unroll
  for (int i = 0; i < KW; ++i) {
    uint4 v = make_uint4(0, 0, 0, 0);
    if (live) v = *reinterpret_cast<const uint4*>(src + 8 * key_word(i));
    const uint32_t vv[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (p.bf16) {
        x[i][2 * j] = __uint_as_float(vv[j] << 16);
        x[i][2 * j + 1] = __uint_as_float(vv[j] & 0xffff0000u);
      } else {
        const float2 h = __half22float2(*reinterpret_cast<const __half2*>(&vv[j]));
        x[i][2 * j] = h.x;
        x[i][2 * j + 1] = h.y;
      }
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      top = fmaxf(top, fabsf(x[i][j]));
      sum[NG == 1 ? 0 : i / 2] += x[i][j];
    }
  }
#pragma unroll
  for (int o = 1; o < 4; o <<= 1) {
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
#pragma unroll
    for (int g = 0; g < NG; ++g) sum[g] += __shfl_xor_sync(0xffffffffu, sum[g], o);
  }
  auto exponent = [](uint32_t bits) { return min(max(static_cast<int>(bits >> 23) - 127, -112), 127); };
  int e2 = exponent(__float_as_uint(top));
  const bool none = __any_sync(0xffffffffu, live && nlse == -INFINITY);
  bool apart = false;
  if (wt_many(p, count)) {
    // Eight rows share a power of two where their largest channels lie within 2^kPfSpread of one another, so that what
    // their scores are multiplied by is one number: 2^-24 of the largest is enough for each then. Rows of zeros, and
    // those with an infinity or NaN, have no say.
    const uint32_t bits = top > 0.0f && top < INFINITY ? __float_as_uint(top) : 0u;
    const int most = exponent(__reduce_max_sync(0xffffffffu, bits)), least = exponent(__reduce_min_sync(0xffffffffu, bits ? bits : 0x7f7fffffu));
    apart = least < most - kPfSpread;
    if (!apart) e2 = most;
  }
  const float down = __uint_as_float(static_cast<uint32_t>(127 + 14 - e2) << 23), units = a.scale * kLog2e;
  const float f = units * 1024.0f * __uint_as_float(static_cast<uint32_t>(127 + e2) << 23);
  // a word's eight channels, in the order of a masked word of codes: 0 4 1 5 2 6 3 7
  auto chunk = [&](int i, float sixteenth) {
    uint32_t w[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float by = (j & 1) ? down * sixteenth : down;
      w[j] = pack2<__half>(x[i][j] * by, x[i][j + 4] * by);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
  };
  if (!wt_many(p, count)) {
    uint32_t* out = p.queries + (static_cast<long long>(kh) * p.tiles + tile) * wt_tile_words(D);
#pragma unroll
    for (int i = 0; i < KW; ++i) *reinterpret_cast<uint4*>(out + (i * 32 + lane) * 4) = chunk(i, 0.0625f);
    if (q4 == 0) *reinterpret_cast<float4*>(out + KW * 128 + r * 4) = make_float4(f, sum[0] * units, sum[NG - 1] * units, nlse);
    if (lane == 0) out[KW * 128 + 32] = none;
  } else {
    using SH = TcShape<D, NG>;
    const int in_tile = t * 8 % SH::N + r;
    uint8_t* out = p.tc_queries + (static_cast<long long>(kh) * p.tc_tiles + wt_first_tile(a, lo, first, SH::N) + t * 8 / SH::N) * SH::TILE_BYTES;
#pragma unroll
    for (int i = 0; i < KW; ++i) {
      const int c = key_word(i);
      *reinterpret_cast<uint4*>(swizzled(out + (c >> 3) * SH::N * 128, in_tile, c & 7)) = chunk(i, 1.0f);
    }
    if (q4 == 0) {
      float* pair = reinterpret_cast<float*>(out + SH::CONSTS_AT + (in_tile >> 1) * 32) + (in_tile & 1);
      pair[0] = f * 0x1p-24f;            // (codes as they are, not 2^-24 of them)
      pair[2] = sum[0] * units;
      pair[4] = sum[NG - 1] * units;
      pair[6] = nlse;
    }
    if (lane == 0) out[SH::FLAGS_AT + in_tile / 8] = none || apart;
  }
}

template <int D, int NG>
__global__ void __launch_bounds__(WT_THREADS, WT_PER_SM) kv4_weights_kernel(const WeightsParams p) {
  using SH = WeightsShape<D, NG>;
  constexpr int KW = D / 32, TILE = wt_tile_words(D);
  extern __shared__ __align__(128) uint8_t smem[];
  after_launch_before();
  const AttendParams& a = p.a;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, r = lane >> 2, q4 = lane & 3;
  const long long total = p.prefix[a.seqs], warps = static_cast<long long>(gridDim.x) * WT_WARPS;
  const long long me = static_cast<long long>(blockIdx.x) * WT_WARPS + warp;
  const long long c0 = total * me / warps;
  int left = static_cast<int>(total * (me + 1) / warps - c0);
  if (left == 0) return;

  // ---- where a chunk is: its sequence, kv head and number; `next` walks a chunk ahead of the sums
  struct Place {
    int b, kh, g;
    int first, count, len;
    Chunks c;
  };
  auto enter = [&](Place& s) {
    wt_sequence(p, s.b, s.first, s.count, s.len);
    s.c = wt_chunks(p, s.count, s.len);
    if (wt_many(p, s.count)) s.c.n = 0;  // the other kernel's
  };
  Place next;
  {
    const int lo = wt_search(a.seqs, [&](int b) { return p.prefix[b] <= c0; });
    next.b = lo;
    enter(next);
    const int at = static_cast<int>(c0 - p.prefix[lo]);
    next.kh = at / next.c.n;
    next.g = at - next.kh * next.c.n;
  }
  auto advance = [&](Place& s) {
    if (++s.g < s.c.n) return;
    s.g = 0;
    if (++s.kh < a.cache.kv_heads) return;
    s.kh = 0;
    do {
      ++s.b;
      enter(s);
    } while (s.c.n == 0 && s.b + 1 < a.seqs);
  };
  auto chunk_of = [&](const Place& s) { return s.g < s.c.sinks ? s.g : s.g + s.c.skip; };

  // ---- this warp's copies: lane 2 k copies block k's codes, lane 2 k + 1 its pairs
  uint8_t* stages = smem + warp * 2 * SH::STAGE;
  uint64_t* bar = reinterpret_cast<uint64_t*>(smem + WT_WARPS * 2 * SH::STAGE) + 2 * warp;
  if (lane == 0) {
    mbar_init(&bar[0], 1);
    mbar_init(&bar[1], 1);
    mbar_fence_init();
  }
  __syncwarp();
  unsigned have = 0;                     // blocks that `next` has in its stage
  float had[2];                          // what tokens r and r + 8 of block q4 have
  auto load = [&](const Place& s, int st) {
    const int chunk = chunk_of(s), blk = chunk * WT_BLOCKS + (lane >> 1);
    const uint8_t* from = nullptr;
    if (lane < 2 * WT_BLOCKS && blk < (s.len + BLK - 1) / BLK) {
      const int col = a.cache.blocks.quotient(blk), page = a.table[static_cast<long long>(s.b) * a.width + col];
      if (static_cast<unsigned>(page) < static_cast<unsigned>(a.cache.pages))
        from = block_ptr(a.cache, page, s.kh, blk - col * a.cache.page_blocks);
      else
        flag_error(kErrIndex);
    }
    have = __ballot_sync(0xffffffffu, from != nullptr);
    if (lane == 0) mbar_arrive_expect_tx(&bar[st], __popc(have) / 2 * SH::KEYS);
    __syncwarp();
    if (from != nullptr) {
      uint8_t* to = stages + st * SH::STAGE + (lane >> 1) * SH::KEYS;
      if (lane & 1) bulk_load(to + SH::CODES, from + key_pairs_at(D), SH::PAIRS, &bar[st]);
      else bulk_load(to, from, SH::CODES, &bar[st]);
    }
    const float* w = p.before + s.b * p.b_ss + s.kh * p.b_sh;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int t = chunk * WT_TOKENS + q4 * BLK + r + 8 * h;
      had[h] = t < min(s.len - s.count, s.len) ? w[t] : 0.0f;
    }
  };
  load(next, 0);
  auto key_word = [&](int i) { return NG == 1 ? KW * q4 + i : (i < 2 ? 2 * q4 + i : 8 + 2 * q4 + i - 2); };

  int stage = 0;
  uint32_t phases = 0;
  for (;;) {
    const Place s = next;
    const float old[2] = {had[0], had[1]};
    const unsigned blocks = have;
    if (--left > 0) {
      advance(next);
      load(next, stage ^ 1);
    }
    if (!mbar_try_wait(&bar[stage], (phases >> stage) & 1u)) wait_for_copy(&bar[stage], (phases >> stage) & 1u, p.wait_ns);
    phases ^= 1u << stage;
    const uint8_t* keys = stages + stage * SH::STAGE;
    stage ^= 1;
    const int t0 = chunk_of(s) * WT_TOKENS, pos0 = s.len - s.count, rows = s.count * a.share;
    // rows that see some token of the chunk: from the first at t0's position to the last whose window reaches it
    const int last_token = min(t0 + WT_TOKENS, s.len) - 1;
    const int row_lo = max(0, t0 - pos0) * a.share;
    int row_hi = rows;
    if (a.window && t0 >= a.sinks)
      row_hi = static_cast<int>(min(static_cast<long long>(rows), max(0LL, static_cast<long long>(last_token) + a.window - pos0) * a.share));
    const uint32_t* tile = p.queries + (s.kh * static_cast<long long>(p.tiles) + wt_first_tile(a, s.b, s.first) + row_lo / 8) * TILE;
    float acc[WT_BLOCKS][2] = {};
    for (int row0 = row_lo & ~7; row0 < row_hi; row0 += 8, tile += TILE) {
      uint32_t qf[KW][4];
#pragma unroll
      for (int i = 0; i < KW; ++i) *reinterpret_cast<uint4*>(qf[i]) = *reinterpret_cast<const uint4*>(tile + (i * 32 + lane) * 4);
      float4 row[2];
#pragma unroll
      for (int c = 0; c < 2; ++c) row[c] = *reinterpret_cast<const float4*>(tile + KW * 128 + (2 * q4 + c) * 4);
      // whether each row sees each token of the chunk: the first row the last token, the last row the first
      const int last_row = min(row0 + 8, rows) - 1;
      const bool edge = blocks != (1u << 2 * WT_BLOCKS) - 1u || tile[KW * 128 + 32] || t0 + WT_TOKENS > s.len ||
                        pos0 + static_cast<int>(a.by_share.quotient(row0)) < last_token ||
                        (a.window && t0 < sees_from(a, pos0 + static_cast<int>(a.by_share.quotient(last_row))) && last_token >= a.sinks);
      auto step = [&](auto edge_tag) {
        constexpr bool EDGE = decltype(edge_tag)::value;
        int from[2], to[2];
        if constexpr (EDGE) {
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            const int i = row0 + 2 * q4 + c, pos = pos0 + static_cast<int>(a.by_share.quotient(i));
            const bool live = i < rows && row[c].w != -INFINITY;
            from[c] = live ? sees_from(a, pos) : 0;
            to[c] = live ? min(s.len, pos + 1) : 0;
          }
        }
#pragma unroll
        for (int k = 0; k < WT_BLOCKS; ++k) {
          const uint8_t* blk = keys + k * SH::KEYS;
          uint32_t kk[2][KW];
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const uint8_t* mine = blk + (r + 8 * h) * (D / 2);
            if constexpr (NG == 1 && KW == 4) {
              *reinterpret_cast<uint4*>(kk[h]) = *reinterpret_cast<const uint4*>(mine + 16 * q4);
            } else {
#pragma unroll
              for (int i = 0; i < KW; i += 2) *reinterpret_cast<uint2*>(kk[h] + i) = *reinterpret_cast<const uint2*>(mine + 4 * key_word(i));
            }
          }
          const uint32_t* pairs = reinterpret_cast<const uint32_t*>(blk + SH::CODES);
          float y[4];
#pragma unroll
          for (int c = 0; c < 4; ++c) y[c] = row[c & 1].w;
#pragma unroll
          for (int g = 0; g < NG; ++g) {
            float d[4];
#pragma unroll
            for (int i = g * (KW / NG); i < (g + 1) * (KW / NG); ++i) {
              const uint32_t w0 = kk[0][i], w1 = kk[1][i], u0 = w0 >> 8, u1 = w1 >> 8;
              if (i == g * (KW / NG))
                mma16816_first(d, w0 & 0x000f000fu, w1 & 0x000f000fu, w0 & 0x00f000f0u, w1 & 0x00f000f0u, qf[i][0], qf[i][1]);
              else
                mma16816(d, w0 & 0x000f000fu, w1 & 0x000f000fu, w0 & 0x00f000f0u, w1 & 0x00f000f0u, qf[i][0], qf[i][1]);
              mma16816(d, u0 & 0x000f000fu, u1 & 0x000f000fu, u0 & 0x00f000f0u, u1 & 0x00f000f0u, qf[i][2], qf[i][3]);
            }
            const float2 p0 = __half22float2(*reinterpret_cast<const __half2*>(&pairs[r * NG + g]));
            const float2 p1 = __half22float2(*reinterpret_cast<const __half2*>(&pairs[(r + 8) * NG + g]));
#pragma unroll
            for (int c = 0; c < 4; ++c)
              y[c] = fmaf(d[c], (c < 2 ? p0.x : p1.x) * row[c & 1].x,
                          fmaf(c < 2 ? p0.y : p1.y, g == 0 ? row[c & 1].y : row[c & 1].z, y[c]));
          }
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            float v = ex2(y[c]);
            if constexpr (EDGE) {
              const int t = t0 + k * BLK + r + (c < 2 ? 0 : 8);
              if ((t < from[c & 1] && t >= a.sinks) || t >= to[c & 1] || !((blocks >> 2 * k) & 1u)) v = 0.0f;
            }
            acc[k][c >> 1] += v;
          }
        }
      };
      if (edge) step(std::true_type()); else step(std::false_type());
    }
    // ---- sums over the rows, and block q4's tokens written by the lanes of q4
    float got[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
#pragma unroll
      for (int k = 0; k < WT_BLOCKS; ++k) {
        float v = acc[k][h];
        v += __shfl_xor_sync(0xffffffffu, v, 1);
        v += __shfl_xor_sync(0xffffffffu, v, 2);
        if (k == 0 || q4 == k) got[h] = v;
      }
    }
    float* w = p.after + s.b * p.a_ss + s.kh * p.a_sh;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int t = t0 + q4 * BLK + r + 8 * h;
      if (t < s.len) w[t] = old[h] + got[h];
    }
    if (left <= 0) break;
    __syncwarp();                        // the stage is copied into again
  }
}

// One word's eight codes less 8, (0,4) (1,5) (2,6) (3,7): 1024 + c - 1032 and 64 + c - 72, exact.
__device__ __forceinline__ uint4 centred_word(uint32_t w) {
  const uint32_t u = w >> 8;
  return make_uint4(hadd2_u32(lop3_and_or(w, 0x000F000Fu, 0x64006400u), 0xE408E408u),
                    hadd2_u32(lop3_and_or(w, 0x00F000F0u, 0x54005400u), 0xD480D480u),
                    hadd2_u32(lop3_and_or(u, 0x000F000Fu, 0x64006400u), 0xE408E408u),
                    hadd2_u32(lop3_and_or(u, 0x00F000F0u, 0x54005400u), 0xD480D480u));
}

// Rows [lo, hi) of a step, a bit each, but for those whose log-sum-exp is -inf (each lane looks at its rows').
template <int N>
__device__ __forceinline__ void wt_seen_rows(const float4* consts, int lo, int hi, uint32_t (&see)[N / 32]) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int w = 0; w < N / 32; ++w) {
    const float4 v = consts[(w * 32 + lane) | 1];
    const uint32_t none = __ballot_sync(0xffffffffu, (lane & 1 ? v.w : v.z) == -INFINITY);
    auto below = [&](int end) { return end >= 32 ? 0xffffffffu : end <= 0 ? 0u : (1u << end) - 1u; };
    see[w] = below(hi - w * 32) & ~below(lo - w * 32) & ~none;
  }
}

// Eight columns of this thread's TMEM lane at each of two places.
__device__ __forceinline__ void tmem_ld_two(uint32_t at0, uint32_t at1, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%16];\n\t"
      "tcgen05.ld.sync.aligned.32x32b.x8.b32 {%8,%9,%10,%11,%12,%13,%14,%15}, [%17];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(at0), "r"(at1));
}

// The same for sequences of many rows, on the 5th-generation tensor cores. A tile is 512 tokens of a kv head, as four
// quarters of 128 (the M side, a token to a TMEM lane), against all rows that see some of them, N at a step:
//   warps 0-15   a quarter each four: its key codes into shared memory as fp16, once a tile; then per step the scores
//                from TMEM (a token per thread), their exponentials and sum, which crosses no lane
//   warp 16      the rows' prepared queries, one copy a step, as many steps ahead as the ring has room
//   warps 17, 18 each issues two quarters' tcgen05.mma: while one quarter's products run, the others' warps are busy
// The steps of all tiles form one list that the blocks split evenly; where a block's share begins or ends inside a
// tile its sums go to a part of their own, which kv4_weights_join_kernel adds up in order. Within a tile sums are
// taken per step and then in pairs of fp32 numbers (rounded-off parts kept): thousands of steps would lose bits.
//
// Keys are codes less 8 (exact in fp16), so that a score's two terms are as small as they can be; eight rows share a
// power of two where they lie within 2^13 of one another, which leaves two packed multiply-adds a score and group. A
// row that far below its neighbours keeps its channels as fp16 down to 2^-15 of its own largest, and smaller ones
// within 2^-26 of it: half of what fp32 rounds off a product with the largest.
//
// The exponentials are 16 a cycle and SM, 2 D operations a score about twice as fast at the tensor cores' rate. Two
// prompts of 4001 and 2763 tokens over 6000 and 4145, 32 heads of 128 channels in two groups on 8 kv heads: 303 us,
// 0.64 PFLOP/s; the 757 million exponentials alone would take 168. By the counters the exponentials' pipe is 66%
// busy, issue slots 58%, tensor cores 53% (64 rows a product, which costs as much as 110 would): what is left is
// latency, at five warps to a scheduler of 96 registers each. Tried: two buffers of scores and two quarters (484 us), two
// tokens a thread in eight warps of 168 registers (435), codes looked up a tile ahead in registers (351 where 336),
// a block an item of a fixed part of the rows (674).
template <int D, int NG>
__global__ void __launch_bounds__(WT_TC_THREADS, 1) kv4_weights_tc_kernel(const WeightsParams p) {
  using SH = TcShape<D, NG>;
  constexpr int N = SH::N, KB = SH::KB, RING = SH::RING, CHUNKS = D / 8;
  after_launch_before();
  let_next_launch();
  const AttendParams& a = p.a;
  const long long entries = p.tc_prefix[a.seqs], total = p.tc_steps[entries];
  const long long each = max(static_cast<long long>(WT_TC_LEAST), (total + p.blocks - 1) / p.blocks);
  const long long x0 = blockIdx.x * each, x1 = min(total, x0 + each);
  if (x0 >= x1) return;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  uint8_t* ktile = smem;
  uint8_t* ring = ktile + SH::KEY_BYTES;
  uint64_t* qfull = reinterpret_cast<uint64_t*>(ring + RING * SH::STAGE);
  uint64_t *qempty = qfull + RING, *kfull = qempty + RING, *sfull = kfull + WT_TC_QUARTERS, *sfree = sfull + WT_TC_QUARTERS;
  uint64_t* drain = sfree + WT_TC_QUARTERS;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 1);

  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int i = 0; i < RING; ++i) {
      mbar_init(&qfull[i], 1);
      mbar_init(&qempty[i], WT_TC_ISSUERS + WT_TC_SOFTMAX);
    }
    for (int i = 0; i < WT_TC_QUARTERS; ++i) {
      mbar_init(&kfull[i], 4);
      mbar_init(&sfull[i], 1);
      mbar_init(&sfree[i], 4);
    }
    mbar_init(drain, WT_TC_ISSUERS);
    mbar_fence_init();
  }
  if (warp == WT_TC_SOFTMAX) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  // the block's first tile, and the place in it
  const int e0 = wt_search(static_cast<int>(entries), [&](int e) { return p.tc_steps[e] <= x0; });
  TcTile s;
  s.b = wt_search(a.seqs, [&](int b) { return p.tc_prefix[b] <= e0; });
  s.g = static_cast<int>(e0 - p.tc_prefix[s.b]);
  wt_tile_sequence(p, s);
  wt_tile_rows<N>(p, s);
  int at = static_cast<int>(x0 - p.tc_steps[e0]);
  s.kh = s.n ? at / s.n : 0;
  at -= s.kh * s.n;
  const int steps = static_cast<int>(x1 - x0);
  auto tile_steps = [&](int done) { return min(s.n - at, steps - done); };   // of the tile, this block's

  bool ok = true;
  if (warp < WT_TC_SOFTMAX) {
    const int t = warp >> 2, m = threadIdx.x & 127;
    // ---- this thread's token's codes and pairs (looked up a tile ahead they would hold registers that the steps need)
    uint4 codes[CHUNKS / 4];
    uint32_t pair[NG];
    bool gone = false;                           // its page is out of range: it gets nothing
    auto load = [&](const TcTile& s) {
      const int tok = s.t0 + t * 128 + m;
#pragma unroll
      for (int i = 0; i < CHUNKS / 4; ++i) codes[i] = make_uint4(0, 0, 0, 0);
#pragma unroll
      for (int i = 0; i < NG; ++i) pair[i] = 0;
      gone = false;
      if (tok >= s.len || wt_row_from(p, s, tok) >= wt_row_to(p, s, tok)) return;     // (nobody sees it)
      const int blk = tok / BLK, col = a.cache.blocks.quotient(blk), page = a.table[static_cast<long long>(s.b) * a.width + col];
      if (static_cast<unsigned>(page) < static_cast<unsigned>(a.cache.pages)) {
        const uint8_t* from = block_ptr(a.cache, page, s.kh, blk - col * a.cache.page_blocks);
#pragma unroll
        for (int i = 0; i < CHUNKS / 4; ++i) codes[i] = *reinterpret_cast<const uint4*>(from + tok % BLK * (D / 2) + i * 16);
#pragma unroll
        for (int i = 0; i < NG; ++i) pair[i] = *reinterpret_cast<const uint32_t*>(from + key_pairs_at(D) + (tok % BLK * NG + i) * 4);
      } else {
        flag_error(kErrIndex);
        gone = true;
      }
    };
    const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
    int ts = 0;                                  // steps of this quarter
    for (int done = 0; ok && done < steps;) {
      const int n = tile_steps(done);
      if (n <= 0) break;                         // (lengths that changed under the call)
      const bool some = s.t0 + t * 128 < s.len;  // the quarter has tokens (else it only lets the stages go)
      load(s);
      if (some) {
        // (the products of the tile before are over: their scores have been waited for)
#pragma unroll
        for (int i = 0; i < CHUNKS / 4; ++i) {
          const uint32_t w[4] = {codes[i].x, codes[i].y, codes[i].z, codes[i].w};
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const int c = i * 4 + k;
            *reinterpret_cast<uint4*>(swizzled(ktile + (t * KB + (c >> 3)) * PF_TILE, m, c & 7)) = centred_word(w[k]);
          }
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&kfull[t]);
      }
      float sk[NG], bk[NG];
#pragma unroll
      for (int i = 0; i < NG; ++i) {
        const float2 x = __half22float2(*reinterpret_cast<const __half2*>(&pair[i]));
        sk[i] = x.x;
        bk[i] = fmaf(8.0f, x.x, x.y);
      }
      // ---- the rows that see the token, and those that every token of the warp's is seen by
      const int tok = s.t0 + t * 128 + m, rows = s.count * a.share;
      const bool live = tok < s.len;
      const int lo = live ? wt_row_from(p, s, tok) : 0, hi = gone ? 0 : live ? wt_row_to(p, s, tok) : rows;
      const int all_lo = __reduce_max_sync(0xffffffffu, lo), all_hi = __reduce_min_sync(0xffffffffu, hi);
      // (rows that some token of the warp's is seen by)
      const int any_lo = __reduce_min_sync(0xffffffffu, live ? lo : rows), any_hi = __reduce_max_sync(0xffffffffu, live ? hi : 0);
      float high = 0.0f, low = 0.0f;
      for (int j = 0; j < n; ++j) {
        const int js = done + j, r = js % RING;
        ok = __all_sync(0xffffffffu, mbar_wait(&qfull[r], (js / RING) & 1, p.wait_ns));
        if (!ok) break;
        if (some) {
          ok = __all_sync(0xffffffffu, mbar_wait(&sfull[t], ts & 1, p.wait_ns));
          if (!ok) break;
          tc_fence_after();
          const uint32_t s_at = tmem + lanes + t * 128;
          const uint8_t* stage = ring + r * SH::STAGE;
          const float4* consts = reinterpret_cast<const float4*>(stage + SH::CONSTS_AT);
          const uint4 flags = *reinterpret_cast<const uint4*>(stage + SH::FLAGS_AT);
          const int row0 = (s.j0 + at + j) * N;
          const bool edge = row0 < all_lo || row0 + N > all_hi || (flags.x | flags.y | (N == 128 ? flags.z | flags.w : 0u));
          constexpr int BATCH = 16 / NG;         // rows at a time; the next ones' scores are under way meanwhile
          auto add = [&](auto edge_tag) {
            constexpr bool EDGE = decltype(edge_tag)::value;
            float2 sum = make_float2(0.0f, 0.0f);
            uint32_t see[N / 32];                // a bit for each row that sees the token
            if constexpr (EDGE) wt_seen_rows<N>(consts, lo - row0, hi - row0, see);
            uint32_t x[2][16];
            float2 skf[NG];                      // scales, times what eight rows' scores are multiplied by
            auto fetch = [&](int c0, uint32_t (&to)[16]) {
              if constexpr (NG == 2) tmem_ld_two(s_at + c0, s_at + N + c0, to);
              else tmem_ld_cols(s_at + c0, to);
            };
            fetch(0, x[0]);
#pragma unroll
            for (int c0 = 0; c0 < N; c0 += BATCH) {
              uint32_t(&now)[16] = x[c0 / BATCH & 1];
              tmem_ld_done(now);
              if (c0 + BATCH < N) {
                fetch(c0 + BATCH, x[(c0 / BATCH + 1) & 1]);
              } else {
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&sfree[t]);
              }
#pragma unroll
              for (int k = 0; k < BATCH; k += 2) {
                // (f, f, q0, q0), (q1, q1, n, n) of two rows
                const float4 u = consts[c0 + k], v = consts[c0 + k + 1];
                if (EDGE || k % 8 == 0)
#pragma unroll
                  for (int i = 0; i < NG; ++i) skf[i] = make_float2(sk[i] * u.x, sk[i] * (EDGE ? u.y : u.x));
                float2 y = __ffma2_rn(make_float2(u.z, u.w), make_float2(bk[0], bk[0]), make_float2(v.z, v.w));
                if (NG == 2) y = __ffma2_rn(make_float2(v.x, v.y), make_float2(bk[NG - 1], bk[NG - 1]), y);
#pragma unroll
                for (int i = 0; i < NG; ++i)
                  y = __ffma2_rn(make_float2(__uint_as_float(now[i * BATCH + k]), __uint_as_float(now[i * BATCH + k + 1])), skf[i], y);
                float2 e = make_float2(ex2(y.x), ex2(y.y));
                if (EDGE) {
                  const uint32_t word = see[(c0 + k) / 32] >> (c0 + k) % 32;
                  if (!(word & 1u)) e.x = 0.0f;
                  if (!(word & 2u)) e.y = 0.0f;
                }
                sum = __fadd2_rn(sum, e);
              }
            }
            return sum.x + sum.y;
          };
          float got = 0.0f;
          if (row0 + N <= any_lo || row0 >= any_hi) {
            tc_fence_before();
            if (lane == 0) mbar_arrive(&sfree[t]);
          } else {
            got = edge ? add(std::true_type()) : add(std::false_type());
          }
          const float q = __fadd_rn(high, got), z = __fsub_rn(q, high);
          low += __fadd_rn(__fsub_rn(high, __fsub_rn(q, z)), __fsub_rn(got, z));
          high = q;
          ++ts;
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&qempty[r]);
      }
      if (!ok) break;
      // ---- the whole of the tile's rows: added to what the token had; else a part
      const float sum = high + low;
      if (n == s.n) {
        if (live) {
          const float had = tok < s.pos0() ? p.before[s.b * p.b_ss + s.kh * p.b_sh + tok] : 0.0f;
          p.after[s.b * p.a_ss + s.kh * p.a_sh + tok] = had + sum;
        }
      } else {
        p.parts[(blockIdx.x * 2 + (at > 0 ? 0 : 1)) * WT_TC_TOKENS + t * 128 + m] = sum;
      }
      done += n;
      at = 0;
      if (done < steps) wt_next_tile<N>(p, s);
    }
  } else if (warp == WT_TC_SOFTMAX && elect_one()) {
    // ---- the queries
    int js = 0;
    for (int done = 0; ok && done < steps;) {
      const int n = tile_steps(done);
      if (n <= 0) break;                         // (lengths that changed under the call)
      const uint8_t* from = p.tc_queries + (static_cast<long long>(s.kh) * p.tc_tiles + wt_first_tile(a, s.b, s.first, N) + s.j0 + at) * SH::TILE_BYTES;
      for (int j = 0; j < n; ++j, ++js) {
        const int r = js % RING;
        if (!mbar_wait_backoff(&qempty[r], ((js / RING) & 1) ^ 1u, p.wait_ns, 64)) {
          ok = false;
          break;
        }
        mbar_arrive_expect_tx(&qfull[r], SH::TILE_BYTES);
        bulk_load(ring + r * SH::STAGE, from + j * static_cast<long long>(SH::TILE_BYTES), SH::TILE_BYTES, &qfull[r]);
      }
      done += n;
      at = 0;
      if (done < steps) wt_next_tile<N>(p, s);
    }
    // (after an expired wait the copies under way still end before the block does)
    if (!ok)
      for (int i = max(0, js - RING); i < js; ++i) mbar_wait(&qfull[i % RING], (i / RING) & 1, kWaitBudgetNs);
  } else if (warp > WT_TC_SOFTMAX && elect_one()) {
    // ---- the products
    constexpr int EACH = WT_TC_QUARTERS / WT_TC_ISSUERS;
    const int q0 = (warp - WT_TC_SOFTMAX - 1) * EACH;
    const uint32_t desc = umma_idesc_f16_f32(128, N);
    int ts[EACH] = {}, tiles[EACH] = {};         // a quarter's steps, and tiles (a quarter without tokens may be ahead)
    for (int done = 0; ok && done < steps;) {
      const int n = tile_steps(done);
      if (n <= 0) break;                         // (lengths that changed under the call)
#pragma unroll
      for (int k = 0; k < EACH; ++k)
        if (ok && s.t0 + (q0 + k) * 128 < s.len) ok = mbar_wait(&kfull[q0 + k], tiles[k]++ & 1, p.wait_ns);
      for (int j = 0; ok && j < n; ++j) {
        const int js = done + j, r = js % RING;
        ok = mbar_wait(&qfull[r], (js / RING) & 1, p.wait_ns);
        if (!ok) break;
#pragma unroll
        for (int k = 0; k < EACH; ++k) {
          const int t = q0 + k;
          if (s.t0 + t * 128 >= s.len) continue; // no such tokens
          ok = mbar_wait(&sfree[t], (ts[k] & 1) ^ 1u, p.wait_ns);
          if (!ok) break;
          tc_fence_after();
#pragma unroll
          for (int kb = 0; kb < KB; ++kb) {
            const uint64_t kd = umma_desc_sw128(smem_u32(ktile + (t * KB + kb) * PF_TILE));
            const uint64_t qd = umma_desc_sw128(smem_u32(ring + r * SH::STAGE + kb * N * 128));
#pragma unroll
            for (int kk = 0; kk < 4; ++kk)
              tc_mma_f16(tmem + t * 128 + (NG == 2 ? kb : 0) * N, kd + kk * 2, qd + kk * 2, desc, (NG == 1 && kb) || kk);
          }
          tc_commit(&sfull[t]);
          ++ts[k];
        }
        if (ok) tc_commit(&qempty[r]);
      }
      done += n;
      at = 0;
      if (done < steps) wt_next_tile<N>(p, s);
    }
    tc_commit(drain);
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  if (warp == WT_TC_SOFTMAX) {
    mbar_wait(drain, 0, kWaitBudgetNs);          // every product has finished before TMEM is released
    __syncwarp();
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// The tiles that several blocks share: their parts in order. Those without a row: what they had.
template <int D, int NG>
__global__ void __launch_bounds__(WT_TC_TOKENS) kv4_weights_join_kernel(const WeightsParams p) {
  after_launch_before();
  let_next_launch();
  const AttendParams& a = p.a;
  const long long entries = p.tc_prefix[a.seqs], total = p.tc_steps[entries];
  const long long each = max(static_cast<long long>(WT_TC_LEAST), (total + p.blocks - 1) / p.blocks);
  for (long long i = blockIdx.x; i < entries * a.cache.kv_heads; i += gridDim.x) {
    const long long e = i / a.cache.kv_heads;
    TcTile s;
    s.kh = static_cast<int>(i - e * a.cache.kv_heads);
    const long long n = (p.tc_steps[e + 1] - p.tc_steps[e]) / a.cache.kv_heads;
    const long long x = p.tc_steps[e] + s.kh * n, first = x / each, last = n ? (x + n - 1) / each : first;
    if (n && first == last) continue;
    s.b = wt_search(a.seqs, [&](int b) { return p.tc_prefix[b] <= e; });
    s.g = static_cast<int>(e - p.tc_prefix[s.b]);
    wt_tile_sequence(p, s);
    wt_tile_rows<TcShape<D, NG>::N>(p, s);
    const int t = s.t0 + threadIdx.x;
    if (t >= s.len) continue;
    float sum = t < s.pos0() ? p.before[s.b * p.b_ss + s.kh * p.b_sh + t] : 0.0f;
    if (n)
      for (long long b = first; b <= last; ++b) sum += p.parts[(b * 2 + (b * each > x ? 0 : 1)) * WT_TC_TOKENS + threadIdx.x];
    p.after[s.b * p.a_ss + s.kh * p.a_sh + t] = sum;
  }
}

}  // namespace kv4
}  // namespace w4a16
