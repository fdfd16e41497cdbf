// kv4_evict.cuh -- eviction from the 4-bit cache by accumulated attention weight: of a sequence longer than
// `keep` each layer and kv head keeps its first `sinks` tokens, its last `recent` ones, and the tokens with the
// largest weights of those between, `keep` in all, in their order (equal weights: the lowest positions; NaN: below
// every number, -0 as 0). Keys are rotated already, so a token may move. What is kept goes into fresh pages, in every
// layer at once; the old ones are given back. So no page that another row shares is written, and nothing is read
// that is being written.
//
// A first small launch decides who gets which pages (one block; the rules of kv4_reserve) and keeps what the
// second one changes: the rows' old pages and lengths. In the second a block, or a cluster of up to eight where
// there are few, takes a row's kv head of a layer. It finds the M-th largest of the weights by digits of 11, 11 and
// 10 bits (a histogram each), until so few share the digits that each is compared with all; a prefix sum of who stays, a run of tokens per thread, gives a list of them, and the
// list is copied 256 tokens at a time: their addresses by one thread each, then 16 bytes a thread. (The blocks of a
// cluster select alike and copy 256 tokens each in turn.)
//
// Memory-bound in the copies; the selection is a chain of a dozen block-wide steps that other blocks of
// the SM fill. Addresses worked out by every thread for its 16 bytes took half of all issue slots: 412 us where this
// takes 333 (40 rows of up to 2048 tokens to 1024, 16 layers, 8 kv heads of 128; 1.72 GB from and to memory, 5.2 TB/s).
// One row of 1100 tokens to 1000: 19.5 us, both launches.
#pragma once

#include <cooperative_groups.h>

#include "kv4_pages.cuh"

namespace w4a16 {
namespace kv4 {

constexpr int EVICT_THREADS = 256, EVICT_BINS = 2048;
constexpr int EVICT_KEYS = 4096;             // weights of a head that are kept in shared memory

struct EvictParams {
  CacheView cache;           // layer 0
  long long layer_bytes;
  Tables in, out;            // out may be in
  const float* weights;      // entry (layer, row, head, token)
  float* kept;               // where the kept tokens' weights go: may be weights
  long long w_sl, w_sr, w_sh, k_sl, k_sr, k_sh;
  int capacity;              // tokens per (layer, row, head) of both
  const int* rows;
  int n;
  int keep, sinks, recent;
  int need;                  // pages that `keep` tokens take
  int* ok;                   // [n]
  int* does;                 // [n] whether the row is evicted from
  int* start;                // [n + 1] pages asked for before request i
  int* lens;                 // [n] the rows' lengths
  int* fresh;                // [n need] new pages
  int* old;                  // [n][width] the rows' pages
  int* claim;                // [rows] scratch: the first request that names a row
  int key_limit;             // weights that shared memory holds
};

// One block, then as many as there are requests, then those that copy the tables.
__global__ void __launch_bounds__(SCAN_THREADS) kv4_evict_plan_kernel(const EvictParams p) {
  let_next_launch();
  const Tables& t = p.in;
  if (blockIdx.x > static_cast<unsigned>(p.n)) {
    const long long at = (blockIdx.x - 1 - p.n) * static_cast<long long>(SCAN_THREADS) + threadIdx.x;
    const long long step = (gridDim.x - 1 - p.n) * static_cast<long long>(SCAN_THREADS);
    copy_ints(p.out.refs, t.refs, t.pages, at, step);
    copy_ints(p.out.table, t.table, static_cast<long long>(t.rows) * t.width, at, step);
    copy_ints(p.out.lens, t.lens, t.rows, at, step);
    return;
  }
  if (blockIdx.x > 0) {      // the row's pages, as they are
    const int i = blockIdx.x - 1, r = p.rows[i];
    if (r < 0 || r >= t.rows) return;
    for (int c = threadIdx.x; c < t.width; c += SCAN_THREADS)
      p.old[static_cast<long long>(i) * t.width + c] = t.table[static_cast<long long>(r) * t.width + c];
    return;
  }
  // a row named twice is evicted from once, by the first request
  for (int pass = 0; p.n > 1 && pass < 2; ++pass) {
    for (int i = threadIdx.x; i < p.n; i += SCAN_THREADS) {
      const int r = p.rows[i];
      if (r < 0 || r >= t.rows) continue;
      if (pass == 0) p.claim[r] = p.n;
      else atomicMin(p.claim + r, i);
    }
    __syncthreads();
  }
  int before = 0;
  for (int base = 0; base < p.n; base += SCAN_THREADS) {
    const int i = base + threadIdx.x;
    int need = 0, good = 0;
    if (i < p.n) {
      const int r = p.rows[i];
      int len = 0;
      if (r < 0 || r >= t.rows) {
        flag_error(kErrIndex);
      } else {
        len = t.lens[r];
        if (len < 0 || static_cast<long long>(len) > static_cast<long long>(t.width) * t.page_size ||
            (len > p.keep && len > p.capacity)) {
          flag_error(kErrIndex);
          len = 0;
        } else {
          good = p.n == 1 || p.claim[r] == i;
          if (good && len > p.keep) need = p.need;
        }
      }
      p.lens[i] = len;
    }
    int total;
    const int at = before + block_exclusive_scan(need, &total);
    if (i < p.n) {
      p.start[i] = at;
      p.does[i] = need != 0;
      p.ok[i] = good;
    }
    before += total;
  }
  if (threadIdx.x == 0) p.start[p.n] = before;
  const int got = lowest_free(t.refs, t.pages, before, [&](int j, int id) { p.fresh[j] = id; });
  // (a thread's own requests: what it wrote above)
  for (int i = threadIdx.x; i < p.n; i += SCAN_THREADS)
    if (p.does[i] && p.start[i] + p.need > got) p.does[i] = p.ok[i] = 0;
}

// Weights in the order of unsigned numbers.
__device__ __forceinline__ uint32_t weight_key(float w) {
  const uint32_t u = w == 0.0f ? 0u : __float_as_uint(w);
  return w != w ? 0u : (u & 0x80000000u) ? ~u : u | 0x80000000u;
}

// Exclusive prefix sum over the block; *total gets the sum.
__device__ __forceinline__ int evict_scan(int v, int* total, int* warp_sums) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int inc = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int n = __shfl_up_sync(0xffffffffu, inc, o);
    if (lane >= o) inc += n;
  }
  __syncthreads();           // an earlier call's readers are done
  if (lane == 31) warp_sums[warp] = inc;
  __syncthreads();
  int before = 0, all = 0;
#pragma unroll
  for (int w = 0; w < EVICT_THREADS / 32; ++w) {
    const int s = warp_sums[w];
    before += w < warp ? s : 0;
    all += s;
  }
  *total = all;
  return before + inc - v;
}

template <int D, int NG>
__global__ void __launch_bounds__(EVICT_THREADS, 5) kv4_evict_kernel(const EvictParams p) {
  namespace cg = cooperative_groups;
  cg::cluster_group cluster = cg::this_cluster();
  const int split = cluster.num_blocks(), part = cluster.block_rank();
  extern __shared__ __align__(16) uint32_t keys[];           // [key_limit], then the list, 16 bits each
  uint16_t* list = reinterpret_cast<uint16_t*>(keys + p.key_limit);
  __shared__ int bins[EVICT_BINS];
  __shared__ int warp_sums[EVICT_THREADS / 32];
  __shared__ int found[2];
  // where the key codes of 256 kept tokens lie and go; the token's number in its block in the lowest four bits
  __shared__ unsigned long long from[2][EVICT_THREADS], to[2][EVICT_THREADS];
  const int item = blockIdx.x / split;
  const int kh = item % p.cache.kv_heads, i = item / p.cache.kv_heads % p.n, layer = item / p.cache.kv_heads / p.n;
  after_launch_before();
  if (!p.does[i]) return;
  const int r = p.rows[i], len = p.lens[i];
  const int lo = p.sinks, hi = len - p.recent, M = p.keep - p.sinks - p.recent;
  const float* w = p.weights + layer * p.w_sl + r * p.w_sr + kh * p.w_sh;
  const int* old = p.old + static_cast<long long>(i) * p.in.width;
  const int* fresh = p.fresh + p.start[i];

  // ---- the row's new pages, by the block of its first layer and head
  if (layer == 0 && kh == 0 && part == 0) {
    for (int c = threadIdx.x; c < p.in.width; c += EVICT_THREADS) {
      const int page = old[c], now = c < p.need ? fresh[c] : -1;
      if (page >= p.in.pages) flag_error(kErrIndex);
      else if (page >= 0) atomicSub(p.out.refs + page, 1);
      if (now >= 0) atomicExch(p.out.refs + now, 1);
      p.out.table[static_cast<long long>(r) * p.in.width + c] = now;
    }
    if (threadIdx.x == 0) p.out.lens[r] = p.keep;
  }

  // ---- the M-th largest weight between sinks and recent ones: `least`, and how many equal to it stay
  const bool held = hi - lo <= p.key_limit;
  auto key_at = [&](int t) { return held ? keys[t - lo] : weight_key(w[t]); };
  uint32_t least = 0xffffffffu;
  int equals = 0;
  if (M > 0) {
    uint32_t known = 0;                                      // the digits found so far
    int left = M;
#pragma unroll 1
    for (int digit = 0; digit < 3; ++digit) {
      const int shift = digit == 0 ? 21 : digit == 1 ? 10 : 0, mask = digit == 2 ? 1023 : 2047;
      const uint32_t above = digit == 0 ? 0u : digit == 1 ? 0xffe00000u : 0xfffffc00u;
      for (int c = threadIdx.x; c < EVICT_BINS; c += EVICT_THREADS) bins[c] = 0;
      __syncthreads();
      for (int t = lo + threadIdx.x; t < hi; t += EVICT_THREADS) {
        uint32_t k;
        if (digit == 0) {
          k = weight_key(w[t]);
          if (held) keys[t - lo] = k;
        } else {
          k = key_at(t);
        }
        if ((k & above) == known) atomicAdd(&bins[(k >> shift) & mask], 1);
      }
      __syncthreads();
      // bins from the largest down, eight a thread
      constexpr int EACH = EVICT_BINS / EVICT_THREADS;
      int mine[EACH], sum = 0;
#pragma unroll
      for (int c = 0; c < EACH; ++c) {
        mine[c] = bins[EVICT_BINS - 1 - (threadIdx.x * EACH + c)];
        sum += mine[c];
      }
      int total;
      int before = evict_scan(sum, &total, warp_sums);
      if (before < left && before + sum >= left) {
#pragma unroll
        for (int c = 0; c < EACH; ++c) {
          if (before < left && before + mine[c] >= left) {
            found[0] = EVICT_BINS - 1 - (threadIdx.x * EACH + c);
            found[1] = left - before;
          }
          before += mine[c];
        }
      }
      __syncthreads();
      known |= static_cast<uint32_t>(found[0]) << shift;
      left = found[1];
      const int same = bins[found[0]];                       // weights with these digits
      __syncthreads();
      if (same > EVICT_THREADS) continue;
      // so few that each can be compared with all
      if (threadIdx.x == 0) found[0] = 0;
      __syncthreads();
      const uint32_t upto = digit == 0 ? 0xffe00000u : digit == 1 ? 0xfffffc00u : 0xffffffffu;
      for (int t = lo + threadIdx.x; t < hi; t += EVICT_THREADS) {
        const uint32_t k = key_at(t);
        if ((k & upto) == known) bins[atomicAdd(&found[0], 1)] = static_cast<int>(k);
      }
      __syncthreads();
      int larger = 0, alike = 0;
      const uint32_t mine_key = static_cast<int>(threadIdx.x) < same ? static_cast<uint32_t>(bins[threadIdx.x]) : 0u;
      for (int j = 0; j < same; ++j) {
        const uint32_t k = static_cast<uint32_t>(bins[j]);
        larger += k > mine_key;
        alike += k == mine_key;
      }
      if (static_cast<int>(threadIdx.x) < same && larger < left && larger + alike >= left) {
        found[0] = static_cast<int>(mine_key);               // (equal ones write the same)
        found[1] = left - larger;
      }
      __syncthreads();
      known = static_cast<uint32_t>(found[0]);
      left = found[1];
      break;
    }
    least = known;
    equals = left;
  }
  // (in place, a block may write weights that another one of its cluster still selects by)
  if (split > 1 && p.kept == p.weights) cluster.sync();

  // ---- who stays, and their copies, `key_limit` tokens at a time
  constexpr int CODE = D / 32;                               // 16-byte pieces of a token's key codes, or value codes
  CacheView cache = p.cache;
  cache.pool += layer * p.layer_bytes;
  // the key codes of the token at place `at` of a sequence with these pages (0: a page out of range)
  auto codes_of = [&](const int* pages, uint32_t at) -> unsigned long long {
    const uint32_t block = at / BLK, col = cache.blocks.quotient(block);
    const int page = pages[col];
    if (static_cast<unsigned>(page) >= static_cast<unsigned>(p.in.pages)) return 0;
    return reinterpret_cast<unsigned long long>(block_ptr(cache, page, kh, block - col * cache.page_blocks)) + at % BLK * (D / 2) + at % BLK;
  };
  float* kept = p.kept + layer * p.k_sl + r * p.k_sr + kh * p.k_sh;
  const bool in_place = split > 1 && p.kept == p.weights;
  float* later = nullptr;                                    // in place: a kept weight, and where it goes
  float weight = 0.0f;
  int place = 0, equal_before = 0, turn = 0, buf = 0;        // tokens kept, and equal ones met, so far
  for (int base = 0; base < len; base += p.key_limit) {
    const int end = min(len, base + p.key_limit), each = (end - base + EVICT_THREADS - 1) / EVICT_THREADS;
    const int t0 = base + threadIdx.x * each, t1 = min(end, t0 + each);
    int surely = 0, equal = 0;
    for (int t = t0; t < t1; ++t) {
      if (t < lo || t >= hi) {
        ++surely;
      } else if (M > 0) {
        const uint32_t k = key_at(t);
        surely += k > least;
        equal += k == least;
      }
    }
    int total;
    const int at = evict_scan(surely | (equal << 16), &total, warp_sums);
    // of the equal ones the first `equals` stay
    int met = equal_before + (at >> 16), rank = (at & 0xffff) + min(met, equals) - min(equal_before, equals);
    for (int t = t0; t < t1; ++t) {
      bool stays = t < lo || t >= hi;
      if (!stays && M > 0) {
        const uint32_t k = key_at(t);
        stays = k > least || (k == least && met < equals);
        met += k == least;
      }
      if (stays) list[rank++] = static_cast<uint16_t>(t - base);
    }
    const int count = (total & 0xffff) + min(equal_before + (total >> 16), equals) - min(equal_before, equals);
    __syncthreads();
    for (int first = 0; first < count; first += EVICT_THREADS, turn = turn + 1 == split ? 0 : turn + 1) {
      const int n = min(EVICT_THREADS, count - first);
      if (turn == part) {
        const int dst = place + first + threadIdx.x;
        if (static_cast<int>(threadIdx.x) < n) {
          const int t = base + list[first + threadIdx.x];
          weight = w[t];
          const unsigned long long there = codes_of(old, t);
          if (there == 0) flag_error(kErrIndex);
          from[buf][threadIdx.x] = there;
          to[buf][threadIdx.x] = codes_of(fresh, dst);
        }
        __syncthreads();
        // (a place is never behind its token, and the 256 are read; other blocks of a cluster may not have come as far)
        if (static_cast<int>(threadIdx.x) < n) {
          if (in_place) later = kept + dst;
          else kept[dst] = weight;
        }
        // the codes: two or four pieces of keys, then as many of values
        constexpr int STEP = EVICT_THREADS / (2 * CODE), UN = 4;
#pragma unroll 1
        for (int round = 0; round < 2 * CODE / UN; ++round) {
          const int piece = threadIdx.x % (2 * CODE), j0 = threadIdx.x / (2 * CODE) + round * UN * STEP;
          const int within = (piece >= CODE ? value_codes_at(D) : 0) + piece % CODE * 16;
          uint4 v[UN];
#pragma unroll
          for (int u = 0; u < UN; ++u) {
            const int j = j0 + u * STEP;
            const unsigned long long src = j < n ? from[buf][j] & ~15ull : 0;
            if (src) v[u] = *reinterpret_cast<const uint4*>(src + within);
          }
#pragma unroll
          for (int u = 0; u < UN; ++u) {
            const int j = j0 + u * STEP;
            if (j < n && from[buf][j]) *reinterpret_cast<uint4*>((to[buf][j] & ~15ull) + within) = v[u];
          }
        }
        // the pairs: keys' and values', one word each and group
        {
          const int word = threadIdx.x % (2 * NG), which = word / NG, g = word % NG;
          auto pair_of = [&](unsigned long long codes) {
            const int i = static_cast<int>(codes & 15);
            return reinterpret_cast<uint32_t*>((codes & ~15ull) - i * (D / 2) + (which ? value_pairs_at(D, NG) : key_pairs_at(D)) + (i * NG + g) * 4);
          };
#pragma unroll
          for (int u = 0; u < 2 * NG; ++u) {
            const int j = threadIdx.x / (2 * NG) + u * (EVICT_THREADS / (2 * NG));
            if (j < n && from[buf][j]) *pair_of(to[buf][j]) = *pair_of(from[buf][j]);
          }
        }
        buf ^= 1;
      }
      // in place: every block has read the weights of `split` turns before any of their places is written
      if (in_place && turn == split - 1) {
        cluster.sync();
        if (later) *later = weight;
        later = nullptr;
      }
    }
    place += count;
    equal_before += total >> 16;
  }
  if (in_place && turn) {
    cluster.sync();
    if (later) *later = weight;
  }
}

}  // namespace kv4
}  // namespace w4a16
