// drafts.cuh -- verification of drafted tokens against the target's probabilities, from given random
// numbers: draft x_i of a sequence is accepted while u_i q_i(x_i) < p_i(x_i) (p the target's
// probabilities at its place, q the ones it was drawn from; 1 where it was looked up), so that what is
// accepted is distributed as the target's own tokens. The token behind the last accepted draft, at
// place a, is drawn by the last random number u from r = max(p_a - q_a, 0), or from p_a where no
// draft is left (or r is nothing): the first v with r_0 + ... + r_v > u (r_0 + r_1 + ...).
//
// u q is exact in fp64, p - q within 2^-53 of itself. The sums are fp64 of four values each (two, where rows lie at any
// place beside a draft) that are summed to 2^-45 of themselves; a thread adds V / 2048 such numbers at most, each addition
// rounded to 2^-53. So a border between two tokens is off by less than 2^-45 + V 2^-64 of the whole, however the sum
// is split (a fp32 sum of 10^5 probabilities would move it by more than many of them are wide). Values
// whose difference is not finite count as nothing, and so do negative ones.
//
// Memory-bound: of a sequence's rows one pair is read whole, after two dependent reads (the drafted
// tokens, then their probabilities) that say which. A cluster of up to eight blocks takes a sequence;
// a warp sums a contiguous range in four quarters at once, the warps' sums meet in shared memory of
// the cluster, and the one warp whose range the border falls into looks at the quarter once more, sixteen values to
// a lane, so that one prefix sum finds the lane.
//
// 64 sequences of up to 7 drafts, 131072 values, fp32: 20.3 us, in which 48 MB are read (a sequence whose drafts all
// stand reads one row): 2.4 TB/s, 36% of the copy rate. One sequence of 32000 values 7.4 us. 201 sequences of 50001
// values, whose rows begin at any multiple of 4 bytes: 18.5 us for looked-up drafts, 26 us beside a draft. No
// unit is full (issue 30%): it is the latency of a chain of four dependent reads, two joins in the cluster and
// the second look.
#pragma once

#include <cooperative_groups.h>

#include "kv4_common.cuh"

namespace w4a16 {
namespace drafts {

constexpr int THREADS = 256, WARPS = THREADS / 32, MOST_CLUSTER = 8;
constexpr int WALK = 16;      // values of a lane, one after another, that the second look takes at a time

struct VerifyParams {
  const void* target;         // [seqs, drafts + 1, vocab], the last axis contiguous
  const void* draft;          // [seqs, drafts, vocab], or null: drafts without probabilities
  long long t_sb, t_si, d_sb, d_si;
  const long long* tokens;    // [seqs, drafts]
  const float* uniforms;      // [seqs, drafts + 1]
  const int* counts;          // [seqs] drafts there are, or null: all
  long long* out;             // [seqs, drafts + 1]
  int* accepted;              // [seqs]
  int* kv_lens;               // lowered by what was rejected, or null
  const int* rows;            // [seqs] entry of kv_lens, or null: the sequence's number
  int n_lens;
  int seqs, drafts;
  long long vocab;
};

template <typename T>
__device__ __forceinline__ float as_f32(T v) { return kv4::to_f32<T>(v); }
template <>
__device__ __forceinline__ float as_f32<float>(float v) { return v; }

__device__ __forceinline__ void load4(const float* at, float (&v)[4]) {
  *reinterpret_cast<float4*>(v) = *reinterpret_cast<const float4*>(at);
}
template <typename T>
__device__ __forceinline__ void load4(const T* at, float (&v)[4]) {
  const uint2 w = *reinterpret_cast<const uint2*>(at);
  const T* x = reinterpret_cast<const T*>(&w);
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = as_f32(x[i]);
}

// What two fp32 numbers' sum is rounded to, and by how much (Knuth's two-sum).
__device__ __forceinline__ float two_sum(float a, float b, float& rest) {
  const float t = __fadd_rn(a, b), x = __fsub_rn(t, a);
  rest = __fadd_rn(__fsub_rn(a, __fsub_rn(t, x)), __fsub_rn(b, x));
  return t;
}

// The sum of N values, or of what they have over as many others, added to an fp64 number. The N are added in fp32 with
// what is rounded off kept (Dekker's rest for a difference: exact where neither number is negative), which leaves
// an error of 2^-45 of their sum at most: 8 roundings, each 2^-24 of a rest of 2^-24. fp64 from the first value on
// costs one or two conversions a value where this costs two for N values: the kernel took 87 us for 64 sequences
// of 131072. Infinities and NaN show in the sum.
template <bool MINUS, int N>
__device__ __forceinline__ void add_to(double& sum, const float (&p)[N], const float (&q)[N]) {
  static_assert(N == 2 || N == 4, "");
  float d[N], e[N] = {};
#pragma unroll
  for (int i = 0; i < N; ++i) {
    if (MINUS) {
      const float qv = fminf(q[i], p[i]);          // (a difference below zero is none)
      d[i] = __fsub_rn(p[i], qv);
      e[i] = __fsub_rn(__fsub_rn(p[i], d[i]), qv);
    } else {
      d[i] = fmaxf(p[i], 0.0f);
    }
  }
  float high, low;
  if (N == 2) {
    high = two_sum(d[0], d[1], low);
    if (MINUS) low = __fadd_rn(low, __fadd_rn(e[0], e[1]));
  } else {
    float r0, r1, r;
    const float t0 = two_sum(d[0], d[1], r0), t1 = two_sum(d[N - 2], d[N - 1], r1);
    high = two_sum(t0, t1, r);
    low = __fadd_rn(__fadd_rn(r0, r1), r);
    if (MINUS) low = __fadd_rn(low, __fadd_rn(__fadd_rn(e[0], e[1]), __fadd_rn(e[N - 2], e[N - 1])));
  }
  sum += static_cast<double>(high) + static_cast<double>(low);
}

__device__ __forceinline__ double warp_sum(double v) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
__device__ __forceinline__ double warp_prefix(double v, int lane) {      // inclusive
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const double x = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += x;
  }
  return v;
}

template <typename T, bool LOOKUP>
__global__ void __launch_bounds__(THREADS, 4) verify_kernel(const VerifyParams p) {
  namespace cg = cooperative_groups;
  cg::cluster_group cluster = cg::this_cluster();
  __shared__ double sums[WARPS];
  const int blocks = cluster.num_blocks(), rank = cluster.block_rank();
  const int b = blockIdx.x / blocks;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const T* target = static_cast<const T*>(p.target) + b * p.t_sb;
  const T* draft = LOOKUP ? nullptr : static_cast<const T*>(p.draft) + b * p.d_sb;
  const long long* tokens = p.tokens + static_cast<long long>(b) * p.drafts;
  const float* uniforms = p.uniforms + static_cast<long long>(b) * (p.drafts + 1);
  int count = p.drafts;
  if (p.counts) {
    count = p.counts[b];
    if (count < 0 || count > p.drafts) {
      if (threadIdx.x == 0 && rank == 0) flag_error(kErrIndex);
      count = min(max(count, 0), p.drafts);
    }
  }

  // ---- the first draft that is not accepted (every warp looks: a block-wide step would cost more)
  int a = count;
  for (int base = 0; base < p.drafts && base < count; base += 32) {
    const int i = base + lane;
    long long x = 0;
    float u = 0.0f;
    if (i < p.drafts) {
      x = tokens[i];
      u = uniforms[i];
    }
    bool take = true;
    if (i < count) {
      if (x < 0 || x >= p.vocab) {
        flag_error(kErrIndex);
        take = false;
      } else {
        const double q = LOOKUP ? 1.0 : static_cast<double>(as_f32(draft[i * p.d_si + x]));
        take = u * q < static_cast<double>(as_f32(target[i * p.t_si + x]));
      }
    }
    const unsigned stop = ~__ballot_sync(0xffffffffu, take);
    if (stop) {
      a = base + __ffs(stop) - 1;
      break;
    }
  }

  // ---- what is left of the target there
  const T* row = target + a * p.t_si;
  const T* minus = LOOKUP || a == count ? nullptr : draft + a * p.d_si;
  constexpr uint32_t NONE = 0xffffffffu;
  uint32_t except = NONE;                     // a looked-up token is the whole of what it was drawn from
  if (LOOKUP && a < count && tokens[a] >= 0 && tokens[a] < p.vocab) except = static_cast<uint32_t>(tokens[a]);
  auto left = [&](float pv, float qv, uint32_t v) {
    const double d = static_cast<double>(pv) - static_cast<double>(qv);
    return d > 0.0 && d < INFINITY && (!LOOKUP || v != except) ? d : 0.0;
  };
  // this warp's rows of 32 values, and its quarters: [first + k len / 4, first + (k + 1) len / 4)
  const uint32_t vocab = p.vocab, units = (vocab + 31) / 32, warps = blocks * WARPS, me = rank * WARPS + warp;
  auto share = [&](uint32_t w) { return static_cast<uint32_t>(static_cast<uint64_t>(units) * w / warps); };
  const uint32_t first = share(me), len = share(me + 1) - first;
  auto quarter = [&](int k) { return first + k * len / 4; };
  double s[4], total, prefix[2], sum[2];
  const bool vectors = vocab % 4 == 0 && (reinterpret_cast<uintptr_t>(row) | reinterpret_cast<uintptr_t>(minus)) % (4 * sizeof(T)) == 0;
  bool slow = false;
  for (;;) {
    // (minus: the pair's other half; without one the loads are of the row alone)
    auto add = [&](auto with) {
      constexpr bool WITH = decltype(with)::value;
#pragma unroll
      for (int k = 0; k < 4; ++k) s[k] = 0.0;
      if (vectors) {
        const uint32_t steps = ((len + 3) / 4 * 8 + 31) / 32;
#pragma unroll 1
        for (uint32_t j = 0; j < steps; ++j)
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const uint32_t v = quarter(k) * 32 + (j * 32 + lane) * 4;
            if (v >= min(quarter(k + 1) * 32, vocab)) continue;
            float pv[4], qv[4] = {};
            load4(row + v, pv);
            if (WITH) load4(minus + v, qv);
            if (LOOKUP) {
#pragma unroll
              for (int i = 0; i < 4; ++i)
                if (v + i == except) pv[i] = 0.0f;
            }
            add_to<WITH>(s[k], pv, qv);
          }
      } else {
        const uint32_t steps = (len + 3) / 4;
        constexpr int UN = WITH ? 2 : 4;
#pragma unroll 1
        for (uint32_t j = 0; j < steps; j += UN) {
          float pv[4][UN], qv[4][UN] = {};
#pragma unroll
          for (int i = 0; i < UN; ++i)
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const uint32_t unit = quarter(k) + j + i, v = unit * 32 + lane;
              const bool in = unit < quarter(k + 1) && v < vocab;
              pv[k][i] = in && (!LOOKUP || v != except) ? as_f32(row[v]) : 0.0f;
              if (WITH) qv[k][i] = in ? as_f32(minus[v]) : 0.0f;
            }
#pragma unroll
          for (int k = 0; k < 4; ++k) add_to<WITH>(s[k], pv[k], qv[k]);
        }
      }
    };
    if (slow) {                               // infinities, NaN or sums beyond fp32 among the values
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        s[k] = 0.0;
        for (uint32_t v = quarter(k) * 32 + lane; v < min(quarter(k + 1) * 32, vocab); v += 32)
          s[k] += left(as_f32(row[v]), minus ? as_f32(minus[v]) : 0.0f, v);
      }
    } else if (minus) {
      add(std::true_type());
    } else {
      add(std::false_type());
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) s[k] = warp_sum(s[k]);
    if (lane == 0) sums[warp] = (s[0] + s[1]) + (s[2] + s[3]);
    cluster.sync();
    // prefix sums of all warps, in every warp: lane's and lane + 32's
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const uint32_t w = h * 32 + lane;
      sum[h] = w < warps ? *cluster.map_shared_rank(&sums[w % WARPS], w / WARPS) : 0.0;
      prefix[h] = warp_prefix(sum[h], lane);
    }
    const double low = __shfl_sync(0xffffffffu, prefix[0], 31);
    prefix[1] += low;
    total = __shfl_sync(0xffffffffu, prefix[1], 31);
    cluster.barrier_arrive();                 // (waited for before the sums change again, or the block ends)
    if (!slow && !(total < INFINITY)) {
      slow = true;
      cluster.barrier_wait();
      continue;
    }
    if (total > 0.0 || (minus == nullptr && except == NONE)) break;
    cluster.barrier_wait();
    minus = nullptr;                          // the draft has all of it: the target's own probabilities
    except = NONE;
    slow = false;
  }

  // ---- the warp whose range holds the border, else the last one with anything
  // (a number below 0, or none, counts as 0; one of 1 or more lies behind every sum. Prefix sums of neighbours are
  // rounded apart, so that a range that holds nothing can seem to exceed the border first: it is passed over.)
  const double border = uniforms[p.drafts] >= 1.0f ? INFINITY : fmax(uniforms[p.drafts] * total, 0.0);
  const unsigned over0 = __ballot_sync(0xffffffffu, prefix[0] > border && sum[0] > 0.0);
  const unsigned over1 = __ballot_sync(0xffffffffu, prefix[1] > border && sum[1] > 0.0);
  const unsigned any0 = __ballot_sync(0xffffffffu, sum[0] > 0.0), any1 = __ballot_sync(0xffffffffu, sum[1] > 0.0);
  const int owner = over0 ? __ffs(over0) - 1 : over1 ? 31 + __ffs(over1) : any1 ? 63 - __clz(any1) : any0 ? 31 - __clz(any0) : 0;
  if (owner != static_cast<int>(me)) {
    cluster.barrier_wait();
    return;
  }
  long long found = -1;
  if (total > 0.0) {
    // what lies before the range; then the first quarter that exceeds the border, the last one where rounding says
    // that none does
    double before = __shfl_sync(0xffffffffu, owner <= 32 ? prefix[0] : prefix[1], (owner - 1) & 31);
    if (owner == 0) before = 0.0;
    int k = 0;
#pragma unroll
    for (int j = 0; j < 3; ++j)
      if (k == j && !(before + s[j] > border)) {
        before += s[j];
        ++k;
      }
    // 16 values to a lane, one after another, so that one prefix sum over the lanes finds the lane. (A border that
    // rounding moved past the quarter's end: on to the next one; past the range's end: its last value with anything.)
    const uint32_t end = min((first + len) * 32, vocab);
    long long last = -1;
    for (uint32_t at = quarter(k) * 32; at < end && found < 0; at += 32 * WALK) {
      double x[WALK], mine = 0.0;
#pragma unroll
      for (int j = 0; j < WALK; ++j) {
        const uint32_t v = at + lane * WALK + j;
        x[j] = v < end ? left(as_f32(row[v]), minus ? as_f32(minus[v]) : 0.0f, v) : 0.0;
        mine += x[j];
      }
      const double up_to = before + warp_prefix(mine, lane);
      const unsigned over = __ballot_sync(0xffffffffu, up_to > border && mine > 0.0), any = __ballot_sync(0xffffffffu, mine > 0.0);
      const int holder = over ? __ffs(over) - 1 : any ? 31 - __clz(any) : 0;
      double up = __shfl_up_sync(0xffffffffu, up_to, 1);
      if (lane == 0) up = before;
      int hit = -1, nonzero = -1;
#pragma unroll
      for (int j = 0; j < WALK; ++j) {
        up += x[j];
        if (x[j] > 0.0) nonzero = j;
        if (hit < 0 && up > border && x[j] > 0.0) hit = j;
      }
      const int in_lane = __shfl_sync(0xffffffffu, hit < 0 ? nonzero : hit, holder);
      if (any) last = at + holder * WALK + in_lane;
      if (over) found = last;
      before = __shfl_sync(0xffffffffu, up_to, 31);
    }
    if (found < 0 && last < 0)
      for (uint32_t at = first * 32; at < end; at += 32) {
        const uint32_t v = at + lane;
        const unsigned any = __ballot_sync(0xffffffffu, v < end && left(as_f32(row[v]), minus ? as_f32(minus[v]) : 0.0f, v) > 0.0);
        if (any) last = at + 31 - __clz(any);
      }
    if (found < 0) found = last;
  }
  for (int i = lane; i <= p.drafts; i += 32)
    p.out[static_cast<long long>(b) * (p.drafts + 1) + i] = i < a ? tokens[i] : i == a ? found : -1;
  if (lane == 0) {
    p.accepted[b] = a;
    if (p.kv_lens) {
      const int r = p.rows ? p.rows[b] : b;
      if (r < 0 || r >= p.n_lens) {
        flag_error(kErrIndex);
      } else if (count > a) {
        // (not below nothing: a length that was wrong before stays as it is)
        if (atomicSub(p.kv_lens + r, count - a) < count - a) {
          atomicAdd(p.kv_lens + r, count - a);
          flag_error(kErrIndex);
        }
      }
    }
  }
  cluster.barrier_wait();
}

}  // namespace drafts
}  // namespace w4a16
