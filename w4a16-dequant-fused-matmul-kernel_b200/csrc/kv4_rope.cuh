// kv4_rope.cuh -- queries and keys on their way to attention, in one pass over them: RMS norm
// of each head, rotary position embedding (one position per token, or time / height / width
// axes), and, for the form with a cache, the 4-bit quantisation of keys and values into their
// slots. And its inverse, reading cached tokens back.
//
//   y = x * (1 / sqrt(mean(x^2) + eps)) * w           (per head; skipped without w)
//   (a, b) -> (a cos - b sin, b cos + a sin)          (pairs (i, i + rot / 2), or (2i, 2i + 1))
//   offset = fp16(min), scale = fp16((max - offset) / 15) (1 when not > 0),
//   code = clamp(rint((x - offset) * (1 / scale)), 0, 15)        (per group of G channels)
//
// All arithmetic is fp32 with one rounding of the result; products are rounded one by one (no
// contraction into FMAs) so that a key's code does not depend on how the compiler fuses them.
// A group that holds an infinity or NaN gets the offset NaN: what reads it sees NaN instead of
// a value made up.
//
// Memory-bound. D / 8 lanes share a head, each with two quads of channels chosen so that a pair
// of the rotation lies in one lane: in the half-split form lane l holds channels 4l .. and
// rot / 2 + 4l ..; without exchange between lanes the rotation costs no shuffles, and every
// 8-byte access of the group still covers whole 32-byte sectors. A group handles UN heads of one
// token, so that their loads are in flight together and share the angles, and so that what is
// computed from a head's or group's statistics is computed by few lanes for all of them (reduce_scatter).
// A group's heads are of one kind, with one base address; pairs of fp32 go through one instruction.
//
// 4096 tokens of 32 + 8 heads of 128 fp16 channels (86 MB in and out): 17 us, 5.1 TB/s, 79% of a plain
// copy's rate. 8192 tokens of 64 + 8 heads of bf16 with their values into the cache (8 kv heads; 316 MB):
// 73 us, 4.3 TB/s; there 71% of the issue slots are full (54% of the ALU pipe with conversions
// of 16-bit pairs, minima and code packing), and blocks of 128 threads at 64 registers took 6% less time than
// blocks of 256 (the same occupancy, given back sooner). Reading 8192 tokens of 8 heads back: 10.4 us, 4.1 TB/s.
#pragma once

#include "kv4_common.cuh"

namespace w4a16 {
namespace kv4 {

constexpr int ROPE_THREADS = 128;
constexpr int UN = 4;             // heads of a token per group of lanes

struct RopeParams {
  const void *q, *k, *v;          // [T, heads, D] each, channels contiguous
  long long q_st, q_sh, k_st, k_sh, v_st, v_sh;   // token and head strides, in elements
  void *q_out, *k_out;            // [T, heads, D] dense
  long long T;
  int heads, kv_heads;
  int chunks, q_chunks, k_chunks; // groups per token; those of queries and of keys (then values)
  Divisor by_chunks;
  const long long* positions;     // [axes, T]
  int axes, end0, end1;           // frequencies < end0 turn by axis 0, < end1 by axis 1, else axis 2
  const float* cos_sin;           // [max_pos, rot]: cosines, then sines
  long long max_pos;
  int rot;                        // rotated channels (the first of each head), a multiple of 8
  int interleaved;
  const void *qw, *kw;            // [D] or null: no norm
  int w_f32;                      // weights fp32, else of the inputs' type
  float eps;
  int vec;                        // every quad of q, k, v is 8-byte aligned
  int w_vec;                      // and of 16-bit weights
  const long long* slots;         // APPEND: [T], page * page_size + offset; < 0: not cached
  CacheView cache;
  int groups;                     // D / G: 1 or 2
};

// Four channels as they lie in memory, and as fp32.
template <typename T>
__device__ __forceinline__ uint2 load_quad(const T* src, int vec) {
  if (vec) return __ldg(reinterpret_cast<const uint2*>(src));
  const unsigned short* v = reinterpret_cast<const unsigned short*>(src);
  return make_uint2(v[0] | static_cast<uint32_t>(v[1]) << 16, v[2] | static_cast<uint32_t>(v[3]) << 16);
}
template <typename T>
__device__ __forceinline__ void quad_f32(const uint2& v, float2* x) {
  const T* e = reinterpret_cast<const T*>(&v);
  x[0] = make_float2(to_f32<T>(e[0]), to_f32<T>(e[1]));
  x[1] = make_float2(to_f32<T>(e[2]), to_f32<T>(e[3]));
}

// Minimum of two that is NaN where one of them is.
__device__ __forceinline__ float min_nan(float a, float b) {
  float r;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// N values of every lane reduced over the L lanes of a group, each to L / N of its lanes: lane l
// ends with value l / (L / N). Every step halves the values that a lane still carries, so all N
// take N - 1 + log2(L / N) shuffles and not N log2(L), and what follows from a value is then
// computed once per group and not once per lane.
template <int N, int L, bool SUM>
__device__ __forceinline__ float reduce_scatter(float (&v)[N]) {
  static_assert(N <= L, "one value per lane at the end");
#pragma unroll
  for (int o = L / 2, n = N; o > 0; o >>= 1, n = n > 1 ? n / 2 : 1) {
    if (n > 1) {
      const bool up = threadIdx.x & o;
#pragma unroll
      for (int i = 0; i < n / 2; ++i) {
        const float got = __shfl_xor_sync(0xffffffffu, up ? v[i] : v[i + n / 2], o);
        const float own = up ? v[i + n / 2] : v[i];
        v[i] = SUM ? own + got : min_nan(own, got);
      }
    } else {
      const float got = __shfl_xor_sync(0xffffffffu, v[0], o);
      v[0] = SUM ? v[0] + got : min_nan(v[0], got);
    }
  }
  return v[0];
}

template <typename T>
__device__ __forceinline__ void store_quad(T* dst, const float2* x) {
  uint2 v;
  v.x = pack2<T>(x[0].x, x[0].y);
  v.y = pack2<T>(x[1].x, x[1].y);
  *reinterpret_cast<uint2*>(dst) = v;
}

// A lane's quads (channels e0 .. e0 + 3 and e1 .. e1 + 3) of UN heads quantised into their
// token's rows; every lane of the warp calls it. `block` is the block of the first head, the
// next `page_bytes` behind it, `store` how many of them are stored; `at` is where their codes
// begin in it, `pairs_at` their pairs.
template <int D, int GROUPS>
__device__ __forceinline__ void quantise_rows(const float2 (&x)[UN][4], int e0, int e1, int tok, uint8_t* block,
                                              long long page_bytes, int store, int at, int pairs_at) {
  constexpr int L = D / 8, N = UN * GROUPS * 2, R = L / N;
  const int l = threadIdx.x % L;
  const int g0 = GROUPS == 1 ? 0 : e0 / (D / 2), g1 = GROUPS == 1 ? 0 : e1 / (D / 2);
  float stat[N];                 // [head][group][minimum, -maximum]
#pragma unroll
  for (int u = 0; u < UN; ++u) {
    float lo[2], hi[2];
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      const float2 a = x[u][2 * q], b = x[u][2 * q + 1];
      lo[q] = min_nan(min_nan(a.x, a.y), min_nan(b.x, b.y));
      hi[q] = min_nan(min_nan(-a.x, -a.y), min_nan(-b.x, -b.y));
    }
    if constexpr (GROUPS == 1) {
      stat[2 * u] = min_nan(lo[0], lo[1]);
      stat[2 * u + 1] = min_nan(hi[0], hi[1]);
    } else {
#pragma unroll
      for (int g = 0; g < GROUPS; ++g) {
        stat[(u * GROUPS + g) * 2] = min_nan(g0 == g ? lo[0] : INFINITY, g1 == g ? lo[1] : INFINITY);
        stat[(u * GROUPS + g) * 2 + 1] = min_nan(g0 == g ? hi[0] : INFINITY, g1 == g ? hi[1] : INFINITY);
      }
    }
  }
  const float mine = reduce_scatter<N, L, false>(stat);
  const float other = __shfl_xor_sync(0xffffffffu, mine, R);
  const int j = l / R;           // this lane's group: j / 2, of head j / 2 / GROUPS
  float lo = j & 1 ? other : mine, hi = -(j & 1 ? mine : other);
  const bool finite = fabsf(lo) < INFINITY && fabsf(hi) < INFINITY;
  lo = finite ? fminf(fmaxf(lo, -kMaxF16), kMaxF16) : NAN;
  hi = fminf(fmaxf(hi, -kMaxF16), kMaxF16);
  const __half ho = __float2half_rn(lo);
  const float fo = __half2float(ho);
  __half hs = __float2half_rn(__fdiv_rn(__fsub_rn(hi, fo), 15.0f));
  if (!(__half2float(hs) > 0.0f)) hs = __float2half_rn(1.0f);
  const float fi = __frcp_rn(__half2float(hs));
  if (l % (2 * R) == 0 && j / 2 / GROUPS < store)
    reinterpret_cast<uint32_t*>(block + j / 2 / GROUPS * page_bytes + pairs_at)[tok * GROUPS + j / 2 % GROUPS] =
        static_cast<uint32_t>(__half_as_ushort(hs)) | (static_cast<uint32_t>(__half_as_ushort(ho)) << 16);
  uint8_t* codes = block + at + tok * (D / 2);
#pragma unroll
  for (int u = 0; u < UN; ++u) {
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      const int from = (u * GROUPS + (q ? g1 : g0)) * 2 * R;
      const float off = -__shfl_sync(0xffffffffu, fo, from, L), inv = __shfl_sync(0xffffffffu, fi, from, L);
      // rounding by the addition of 2^23: the code is what the sum's low bits hold
      uint32_t w = 0;
#pragma unroll
      for (int i = 1; i >= 0; --i) {
        float2 c = x[u][2 * q + i];
        c = make_float2(fminf(fmaxf(c.x, -kMaxF16), kMaxF16), fminf(fmaxf(c.y, -kMaxF16), kMaxF16));
        c = __fmul2_rn(__fadd2_rn(c, make_float2(off, off)), make_float2(inv, inv));
        c = make_float2(fminf(fmaxf(c.x, 0.0f), 15.0f), fminf(fmaxf(c.y, 0.0f), 15.0f));   // NaN: code 0
        c = __fadd2_rn(c, make_float2(8388608.0f, 8388608.0f));
        w = (w * 16 + __float_as_uint(c.y)) * 16 + __float_as_uint(c.x);
      }
      if (u < store) *reinterpret_cast<uint16_t*>(codes + u * page_bytes + (q ? e1 : e0) / 2) = static_cast<uint16_t>(w);
    }
  }
}

template <typename T, int D, bool APPEND>
__global__ void __launch_bounds__(ROPE_THREADS, 8) qk_norm_rope_kernel(const RopeParams p) {
  constexpr int L = D / 8;
  const int l = threadIdx.x % L;
  uint32_t g = blockIdx.x * (ROPE_THREADS / L) + threadIdx.x / L;
  const bool live = g < p.T * p.chunks;
  if (!live) g = 0;   // stays for the warp's shuffles, stores nothing
  const uint32_t token = p.by_chunks.quotient(g);
  const long long t = token;
  const int chunk = g - token * p.chunks;
  // a group's heads are all of one kind
  const bool is_q = chunk < p.q_chunks, is_k = !is_q && chunk < p.q_chunks + p.k_chunks;
  const int first = (chunk - (is_q ? 0 : is_k ? p.q_chunks : p.q_chunks + p.k_chunks)) * UN;
  const int count = min(UN, (is_q ? p.heads : p.kv_heads) - first);
  const long long sh = is_q ? p.q_sh : is_k ? p.k_sh : p.v_sh;
  const T* src = static_cast<const T*>(is_q ? p.q : is_k ? p.k : p.v) + t * (is_q ? p.q_st : is_k ? p.k_st : p.v_st) +
                 first * sh;

  const bool turns = l < p.rot / 8;
  const int e0 = turns && !p.interleaved ? 4 * l : 8 * l;
  const int e1 = turns && !p.interleaved ? p.rot / 2 + 4 * l : 8 * l + 4;

  uint2 raw[UN][2];
#pragma unroll
  for (int u = 0; u < UN; ++u) raw[u][0] = raw[u][1] = make_uint2(0, 0);
  if (p.vec) {
#pragma unroll
    for (int u = 0; u < UN; ++u)
      if (u < count) {
        raw[u][0] = __ldg(reinterpret_cast<const uint2*>(src + u * sh + e0));
        raw[u][1] = __ldg(reinterpret_cast<const uint2*>(src + u * sh + e1));
      }
  } else {
#pragma unroll
    for (int u = 0; u < UN; ++u)
      if (u < count) {
        raw[u][0] = load_quad<T>(src + u * sh + e0, 0);
        raw[u][1] = load_quad<T>(src + u * sh + e1, 0);
      }
  }

  float cs[4], sn[4];
  if (turns && (is_q || is_k)) {
    const int f = 4 * l;
    long long pos = p.positions[t];
    if (pos < 0 || pos >= p.max_pos) {
      flag_error(kErrIndex);
      pos = 0;
    }
    if (p.axes == 1) {
      const float4 c4 = __ldg(reinterpret_cast<const float4*>(p.cos_sin + pos * p.rot + f));
      const float4 s4 = __ldg(reinterpret_cast<const float4*>(p.cos_sin + pos * p.rot + p.rot / 2 + f));
      cs[0] = c4.x; cs[1] = c4.y; cs[2] = c4.z; cs[3] = c4.w;
      sn[0] = s4.x; sn[1] = s4.y; sn[2] = s4.z; sn[3] = s4.w;
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        long long a = p.positions[(f + i < p.end0 ? 0 : f + i < p.end1 ? 1 : 2) * p.T + t];
        if (a < 0 || a >= p.max_pos) {
          flag_error(kErrIndex);
          a = 0;
        }
        cs[i] = __ldg(p.cos_sin + a * p.rot + f + i);
        sn[i] = __ldg(p.cos_sin + a * p.rot + p.rot / 2 + f + i);
      }
    }
  }

  float2 x[UN][4];
  float sums[UN];
#pragma unroll
  for (int u = 0; u < UN; ++u) {
    quad_f32<T>(raw[u][0], x[u]);
    quad_f32<T>(raw[u][1], x[u] + 2);
  }
  const void* w = is_q ? p.qw : is_k ? p.kw : nullptr;
  if (__any_sync(0xffffffffu, w != nullptr)) {
#pragma unroll
    for (int u = 0; u < UN; ++u) {
      float2 sum = __fmul2_rn(x[u][0], x[u][0]);
#pragma unroll
      for (int i = 1; i < 4; ++i) sum = __ffma2_rn(x[u][i], x[u][i], sum);
      sums[u] = sum.x + sum.y;
    }
    const float norm = __frcp_rn(__fsqrt_rn(__fadd_rn(reduce_scatter<UN, L, true>(sums) / D, p.eps)));
    float2 wv[4];
    if (w == nullptr) {
#pragma unroll
      for (int i = 0; i < 4; ++i) wv[i] = make_float2(1.0f, 1.0f);
    } else if (p.w_f32) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float* wf = static_cast<const float*>(w) + (i < 2 ? e0 : e1 - 4) + 2 * i;
        wv[i] = make_float2(__ldg(wf), __ldg(wf + 1));
      }
    } else {
      quad_f32<T>(load_quad<T>(static_cast<const T*>(w) + e0, p.w_vec), wv);
      quad_f32<T>(load_quad<T>(static_cast<const T*>(w) + e1, p.w_vec), wv + 2);
    }
#pragma unroll
    for (int u = 0; u < UN; ++u) {
      float r = __shfl_sync(0xffffffffu, norm, u * (L / UN), L);
      if (w == nullptr) r = 1.0f;
#pragma unroll
      for (int i = 0; i < 4; ++i) x[u][i] = __fmul2_rn(__fmul2_rn(x[u][i], make_float2(r, r)), wv[i]);
    }
  }
  if (turns && (is_q || is_k)) {
    if (p.interleaved) {
#pragma unroll
      for (int u = 0; u < UN; ++u)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          x[u][i] = __fadd2_rn(__fmul2_rn(x[u][i], make_float2(cs[i], cs[i])),
                               __fmul2_rn(make_float2(x[u][i].y, x[u][i].x), make_float2(-sn[i], sn[i])));
    } else {
#pragma unroll
      for (int u = 0; u < UN; ++u)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const float2 a = x[u][i], b = x[u][i + 2], c = make_float2(cs[2 * i], cs[2 * i + 1]);
          const float2 s = make_float2(sn[2 * i], sn[2 * i + 1]);
          x[u][i] = __fadd2_rn(__fmul2_rn(a, c), __fmul2_rn(b, make_float2(-s.x, -s.y)));
          x[u][i + 2] = __fadd2_rn(__fmul2_rn(b, c), __fmul2_rn(a, s));
        }
    }
  }
  if (live && (is_q || !APPEND)) {
    T* dst = (is_q ? static_cast<T*>(p.q_out) + t * p.heads * D : static_cast<T*>(p.k_out) + t * p.kv_heads * D) + first * D;
#pragma unroll
    for (int u = 0; u < UN; ++u)
      if (u < count) {
        store_quad<T>(dst + u * D + e0, x[u]);
        store_quad<T>(dst + u * D + e1, x[u] + 2);
      }
  }

  if constexpr (APPEND) {
    // the lanes of a warp may hold different kinds: all of them take part where any has keys or
    // values
    if (__all_sync(0xffffffffu, is_q)) return;
    const long long slot = is_q ? -1 : p.slots[t];
    bool cached = live && slot >= 0;
    if (cached && slot >= p.cache.pages * p.cache.page_size) {
      flag_error(kErrIndex);
      cached = false;
    }
    // (below 2^32, as the host checks for the whole layer)
    const uint32_t block = cached ? static_cast<uint32_t>(slot) / BLK : 0;
    const uint32_t page = p.cache.blocks.quotient(block);
    uint8_t* blk = block_ptr(p.cache, page, first, block - page * p.cache.page_blocks);
    const int tok = static_cast<int>(slot % BLK), store = cached ? count : 0;
    const int at = is_k ? 0 : value_codes_at(D);
    if constexpr (D == 128) {
      if (p.groups == 2) {
        quantise_rows<D, 2>(x, e0, e1, tok, blk, p.cache.page_bytes, store, at, is_k ? key_pairs_at(D) : value_pairs_at(D, 2));
        return;
      }
    }
    quantise_rows<D, 1>(x, e0, e1, tok, blk, p.cache.page_bytes, store, at, is_k ? key_pairs_at(D) : value_pairs_at(D, 1));
  }
}

// Cached tokens as T: out [2][n][kv heads][D], keys then values; a negative slot gives zeros.
// D / 8 lanes per token and head, one word of eight channels each.
struct GatherParams {
  const long long* slots;
  long long n;
  void* out;
  CacheView cache;
  int groups;
  Divisor by_heads;
};

template <typename T, int D>
__global__ void __launch_bounds__(256) kv4_gather_kernel(const GatherParams p) {
  constexpr int L = D / 8;
  const int l = threadIdx.x % L;
  const uint32_t g = blockIdx.x * (256 / L) + threadIdx.x / L;
  if (g >= p.n * p.cache.kv_heads) return;
  const uint32_t t = p.by_heads.quotient(g);
  const int head = g - t * p.cache.kv_heads;
  long long slot = p.slots[t];
  if (slot >= p.cache.pages * p.cache.page_size) {
    flag_error(kErrIndex);
    slot = -1;
  }
  uint32_t word[2] = {0, 0}, pair[2] = {0, 0};
  if (slot >= 0) {
    const uint32_t block = static_cast<uint32_t>(slot) / BLK;   // (the host checks for 2^32)
    const uint32_t page = p.cache.blocks.quotient(block);
    const uint8_t* blk = block_ptr(p.cache, page, head, block - page * p.cache.page_blocks);
    const int tok = static_cast<int>(slot % BLK);
    const int grp = l * 8 / (D / p.groups);
    word[0] = *reinterpret_cast<const uint32_t*>(blk + tok * (D / 2) + 4 * l);
    word[1] = *reinterpret_cast<const uint32_t*>(blk + value_codes_at(D) + tok * (D / 2) + 4 * l);
    pair[0] = *reinterpret_cast<const uint32_t*>(blk + key_pairs_at(D) + (tok * p.groups + grp) * 4);
    pair[1] = *reinterpret_cast<const uint32_t*>(blk + value_pairs_at(D, p.groups) + (tok * p.groups + grp) * 4);
  }
#pragma unroll
  for (int s = 0; s < 2; ++s) {
    const float2 so = __half22float2(*reinterpret_cast<const __half2*>(&pair[s]));
    uint4 v;
    uint32_t* vp = &v.x;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      // 2^23 + code, exactly, less 2^23
      const float a = __uint_as_float(0x4B000000u | ((word[s] >> (8 * i)) & 15u)) - 8388608.0f;
      const float b = __uint_as_float(0x4B000000u | ((word[s] >> (8 * i + 4)) & 15u)) - 8388608.0f;
      vp[i] = pack2<T>(__fadd_rn(__fmul_rn(so.x, a), so.y), __fadd_rn(__fmul_rn(so.x, b), so.y));
    }
    *reinterpret_cast<uint4*>(static_cast<T*>(p.out) + ((s * p.n + t) * p.cache.kv_heads + head) * D + 8 * l) = v;
  }
}

}  // namespace kv4
}  // namespace w4a16
