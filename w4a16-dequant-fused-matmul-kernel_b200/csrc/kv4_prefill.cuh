// kv4_prefill.cuh -- attention over the 4-bit cache for many query rows per kv head (prompts and
// their chunks): o = softmax(scale q k^T) v on the 5th-generation tensor cores.
//
// Compute-bound: 4 D operations per row and token. A block takes 256 rows (query token, head of
// the group) of one kv head as two tiles of 128, and 64 tokens at a time (32 with two groups):
//   warps 0-3, 4-7  softmax of row tile 0 and 1, one row per thread (TMEM lane): queries scaled and
//                   written to shared memory once; then per step the scores from TMEM, the running
//                   maximum, probabilities as fp16 over their scores' columns (the A operand of the
//                   second product), and at the end the sums, divided
//   warps 8-11      the cache: a token's keys (8, 9) or values (10, 11), or one group of them, per thread,
//                   read a step ahead; key codes as fp16 into the K ring, values as fp16 into the V ring,
//                   key pairs as fp32 beside them
//   warps 12, 13    each issues its row tile's tcgen05.mma: O_t += P_t V (P from TMEM, V as it lies,
//                   token-major, through the transposing descriptor), then S_t = Q_t K^T two steps ahead
// Each tile has two buffers of scores, so its softmax goes on with step j + 1 while the tensor cores
// take up step j's probabilities and write over them the scores of step j + 2 (the products of one thread
// run in order). With one buffer of 128 tokens softmax and products took turns: 3700 and 3500 cycles
// per 128 tokens.
//
// Three prompts of up to 4096 tokens over up to 8192, 32 heads of 128 channels on 8 kv heads: 1.18 ms, 0.79
// PFLOP/s, 47% of what a plain bf16 matrix product reaches; in two groups per head 1.46 ms, with heads of 64 1.04 ms.
// A step of 64 tokens takes 2600 cycles, its products 1000 of them: what bounds it is the softmax warps'
// instructions (traced at 2500: 1950 cycles a step, two warps to an SM quarter, 128 registers) with the cache
// warps' in the same issue slots; without exponentials, key pairs and expansion the schedule took 0.76 ms of then
// 1.14. Four softmax warps to a quarter of 80 registers each (even and odd steps by different threads) took 1.28 ms.
//
// As in the decode kernel the tensor cores see a key's codes, and its scale and offset act on its
// scores in fp32, so the scores carry no rounding of keys (values rounded to fp16 first move a
// log-sum-exp by some 1e-3 where scores reach 80). The codes are masked words, c 2^-24 (queries carry
// the 1/16 of odd nibbles). With two groups of channels each has its own product S. A value is
// rounded once, to fp16, as a 16-bit cache would hold it: 2^-11 of it at most, like its
// probability. (Value scales on the probabilities instead took two more floats per token and row
// out of shared memory and three more instructions per score.)
// A value pair that is not finite becomes zeros in V, where a row that does not see the token would
// meet it as 0 NaN; the rows that do see it are marked and get NaN in those channels at the end.
//
// The block's queries are scaled by one power of two, to a largest finite magnitude in [2^14, 2^15), which fits
// fp16. It keeps the channels of a row down to 2^-24 of the block's largest (odd nibbles with their 1/16): enough for
// rows whose largest channel is within 2^kPfSpread of that. Where some row lies below, each row has its own power
// of two, and its products the ratio of it to the block's: one packed multiplication per two products, which only the
// steps at the causal edge and those of such blocks carry.
//
// TMEM columns: S0 2 x 64, S1 2 x 64 (with P over them), O0 128, O1 128: all 512. Channels lie in the
// order 0 4 1 5 2 6 3 7 inside each eight (how a masked word gives them): in Q and K alike, which
// leaves the scores as they are, and in V, which the last step undoes.
//
// The probabilities of a step are taken with the running maximum as it stands, and again in the
// rare case that some score of the warp's rows exceeds it by kPfLazyMax: one pass over the scores
// instead of two. Every wait is bounded; on expiry the block raises the device error bit and leaves.
#pragma once

#include "kv4_decode.cuh"

namespace w4a16 {
namespace kv4 {

constexpr int PF_ROWS = 256;         // query rows per block (two tiles)
constexpr int PF_THREADS = 14 * 32;
// A row's maximum is raised when a score exceeds it by this (base 2): probabilities up to 256, as exact in
// fp16 as those below 1. At 2.9 (the decode kernel's, whose probabilities carry a scale) 14% of a long
// prompt's steps took the rescaling path.
constexpr float kPfLazyMax = 8.0f;
// A score's two terms are at most 65504 |scale| log2(e) sum|q|. Up to this sum they are below 2^25, and taking the
// maximum off inside the sum moves a score by a few units at most. A block with a row beyond takes it off afterwards, so that
// the largest score is zero exactly (at scores of 1e12 all others were off by 1e5, and sums of nothing).
constexpr float kPfPlainSum = 512.0f;
constexpr int kPfSpread = 13;
constexpr int PF_TILE = 128 * 128;   // bytes of a [128][64] fp16 tile
constexpr int PF_RING = 4;           // K tiles, and V tiles
constexpr int PF_PARS = 8;           // steps whose pairs are kept

// B operand as it lies with its N index contiguous: [k][64 n] rows of 128 bytes, 128-byte swizzle, blocks
// of 64 n `block_bytes` apart, 8-row groups 1024 bytes apart.
__device__ __forceinline__ uint64_t umma_desc_sw128_mn(uint32_t smem_addr, uint32_t block_bytes) {
  uint64_t d = 0;
  d |= static_cast<uint64_t>((smem_addr & 0x3FFFFu) >> 4);
  d |= static_cast<uint64_t>(block_bytes >> 4) << 16;
  d |= static_cast<uint64_t>(1024u >> 4) << 32;
  d |= static_cast<uint64_t>(1u) << 46;
  d |= static_cast<uint64_t>(2u) << 61;
  return d;
}
constexpr uint32_t kTransposeB = 1u << 16;   // instruction descriptor: B's N index contiguous

struct PrefillParams {
  AttendParams a;
  int bf16;
  int row_limit;             // sequences with at most so many rows are left to the other kernel
  unsigned long long wait_ns;
};

template <int D, int NG>
struct PrefillShape {
  static constexpr int KB = D / 64;                       // 64-channel blocks
  static constexpr int TOK = 64 / NG;                     // tokens per step
  static constexpr int Q_BYTES = 2 * KB * PF_TILE;
  static constexpr int BLOCK_BYTES = TOK * 128;           // [TOK][64] fp16
  static constexpr int KV_BYTES = KB * BLOCK_BYTES;       // one K or V tile
  static constexpr int PAR_BYTES = PF_PARS * 64 * 8;
  static constexpr int SMEM_BYTES = 1024 + Q_BYTES + 2 * PF_RING * KV_BYTES + PAR_BYTES + 512;
  static_assert(SMEM_BYTES <= 227 * 1024, "shared memory budget");
};

// One word's eight codes, (0,4) (1,5) (2,6) (3,7): c 2^-24 and 16 c 2^-24 in turn.
__device__ __forceinline__ uint4 masked_word(uint32_t w) {
  const uint32_t u = w >> 8;
  return make_uint4(w & 0x000f000fu, w & 0x00f000f0u, u & 0x000f000fu, u & 0x00f000f0u);
}
// Their values offset + scale c, each rounded once; within +-65504 with `clamp`.
__device__ __forceinline__ uint4 value_word(uint32_t w, __half2 scale, __half2 offset, bool clamp) {
  const uint32_t u = w >> 8;
  // 1024 + c and 64 + c, less 1024 and 64: exact
  const uint32_t c[4] = {hadd2_u32(lop3_and_or(w, 0x000F000Fu, 0x64006400u), 0xE400E400u),
                         hadd2_u32(lop3_and_or(w, 0x00F000F0u, 0x54005400u), 0xD400D400u),
                         hadd2_u32(lop3_and_or(u, 0x000F000Fu, 0x64006400u), 0xE400E400u),
                         hadd2_u32(lop3_and_or(u, 0x00F000F0u, 0x54005400u), 0xD400D400u)};
  uint4 o;
  uint32_t* ow = &o.x;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    __half2 v = __hfma2(*reinterpret_cast<const __half2*>(&c[i]), scale, offset);
    if (clamp) v = __hmin2(__hmax2(v, __float2half2_rn(-kMaxF16)), __float2half2_rn(kMaxF16));
    ow[i] = *reinterpret_cast<const uint32_t*>(&v);
  }
  return o;
}

// Whether the phase with this parity is over, without waiting.
__device__ __forceinline__ bool mbar_test(uint64_t* bar, uint32_t parity) {
  uint32_t is;
  asm volatile("{ .reg .pred p; mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2; selp.u32 %0, 1, 0, p; }"
               : "=r"(is) : "r"(smem_u32(bar)), "r"(parity) : "memory");
  return is != 0;
}

// One lane of a converged warp. The compiler knows of it that it is one thread, so the operands of the
// products go through uniform registers (with the warp's number taken from one lane, too: 1.28 -> 1.16 ms
// for three prompts of 4096 tokens, 32 heads).
__device__ __forceinline__ bool elect_one() {
  uint32_t is;
  asm volatile("{ .reg .pred p; elect.sync _|p, 0xffffffff; selp.u32 %0, 1, 0, p; }" : "=r"(is));
  return is != 0;
}

// Columns of this thread's TMEM lane. Neither a load nor its wait says anything of other memory, so that
// loads from shared memory may be moved over them; the wait takes the registers through.
__device__ __forceinline__ void tmem_ld_cols(uint32_t at, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(at));
}
template <int N>
__device__ __forceinline__ void tmem_ld_done(uint32_t (&r)[N]) {
#pragma unroll
  for (int i = 0; i < N; i += 16)
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(r[i]), "+r"(r[i + 1]), "+r"(r[i + 2]), "+r"(r[i + 3]), "+r"(r[i + 4]), "+r"(r[i + 5]),
                   "+r"(r[i + 6]), "+r"(r[i + 7]), "+r"(r[i + 8]), "+r"(r[i + 9]), "+r"(r[i + 10]), "+r"(r[i + 11]),
                   "+r"(r[i + 12]), "+r"(r[i + 13]), "+r"(r[i + 14]), "+r"(r[i + 15]));
}

__device__ __forceinline__ uint8_t* swizzled(uint8_t* tile, int row, int chunk) {
  return tile + row * 128 + ((chunk ^ (row & 7)) << 4);
}

// A step's probabilities with the maximum m: h in fp16, packed by token pairs, and their sum; returns
// the largest score. EDGE: some row does not see every token (this one sees [rel_from, rel_to) of the step),
// or has large scores or a power of two of its own: its products are to be multiplied by `ratio`.
template <int NG, int TOK, bool EDGE>
__device__ __forceinline__ float step_probabilities(uint32_t s_at, const float4* par, float m, const float (&qs)[NG],
                                                    int rel_from, int rel_to, float ratio, uint32_t (&h)[TOK / 2], float& l_add) {
  constexpr int COLS = 16, CHUNK = TOK / COLS;
  float top = -INFINITY;
  float2 sum = make_float2(0.0f, 0.0f);
  uint32_t x[CHUNK][NG][COLS];
#pragma unroll
  for (int c = 0; c < CHUNK; ++c)
#pragma unroll
    for (int g = 0; g < NG; ++g) tmem_ld_cols(s_at + g * TOK + c * COLS, x[c][g]);
#pragma unroll
  for (int c = 0; c < CHUNK; ++c)
#pragma unroll
    for (int g = 0; g < NG; ++g) tmem_ld_done(x[c][g]);
#pragma unroll
  for (int c = 0; c < CHUNK; ++c) {
#pragma unroll
    for (int i = 0; i < COLS; i += 2) {
      float4 q[NG];
      float2 y = EDGE ? make_float2(0.0f, 0.0f) : make_float2(-m, -m);
#pragma unroll
      for (int g = 0; g < NG; ++g) {
        q[g] = par[(c * COLS + i) / 2 * NG + g];
        y = __ffma2_rn(make_float2(q[g].z, q[g].w), make_float2(qs[g], qs[g]), y);
      }
#pragma unroll
      for (int g = 0; g < NG; ++g) {
        float2 s = make_float2(__uint_as_float(x[c][g][i]), __uint_as_float(x[c][g][i + 1]));
        if (EDGE) s = __fmul2_rn(s, make_float2(ratio, ratio));
        y = __ffma2_rn(s, make_float2(q[g].x, q[g].y), y);
      }
      if (EDGE) {
        const int tok = c * COLS + i;
        if (tok < rel_from || tok >= rel_to) y.x = -INFINITY;
        if (tok + 1 < rel_from || tok + 1 >= rel_to) y.y = -INFINITY;
      }
      top = fmaxf(top, fmaxf(y.x, y.y));
      if (EDGE) y = __fadd2_rn(y, make_float2(-m, -m));
      const float2 e = make_float2(ex2(y.x), ex2(y.y));
      sum = __fadd2_rn(sum, e);
      h[(c * COLS + i) / 2] = pack2<__half>(e.x, e.y);
    }
  }
  l_add = sum.x + sum.y;
  return EDGE ? top : m + top;
}

template <int D, int NG>
__global__ void __launch_bounds__(PF_THREADS, 1) kv4_prefill_kernel(const PrefillParams p) {
  using SH = PrefillShape<D, NG>;
  constexpr int KB = SH::KB, CHUNKS = D / 8, TOK = SH::TOK;
  const AttendParams& a = p.a;
  // longest first: the last row tiles see the most tokens
  int first, count, len;
  const int kh = blockIdx.x % a.cache.kv_heads, b = blockIdx.x / a.cache.kv_heads % a.seqs;
  const int back = blockIdx.x / a.cache.kv_heads / a.seqs;
  sequence(a, b, first, count, len);
  const int rows = count * a.share;
  const int row0 = ((rows + PF_ROWS - 1) / PF_ROWS - 1 - back) * PF_ROWS;
  if (rows <= p.row_limit || row0 < 0) return;
  const int last_row = min(rows, row0 + PF_ROWS) - 1;
  // tokens some row of the block sees, in steps of TOK
  const int pos0 = len - count + row0 / a.share, pos1 = len - count + last_row / a.share;
  const int from = sees_from(a, pos0), to = min(len, pos1 + 1);
  const int step0 = from / TOK;
  const int steps = max(0, (to + TOK - 1) / TOK - step0);
  const bool two = row0 + 128 <= last_row;

  extern __shared__ __align__(1024) uint8_t smem_raw[];
  // an offset, not a cast: the compiler then knows its loads to be from shared memory
  uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  uint8_t* qtile = smem;
  uint8_t* ktile = qtile + SH::Q_BYTES;                   // K's ring, then V's
  uint8_t* vtile = ktile + PF_RING * SH::KV_BYTES;
  float4* pars = reinterpret_cast<float4*>(vtile + PF_RING * SH::KV_BYTES);   // [PF_PARS][TOK / 2][NG]
  uint2* bad = reinterpret_cast<uint2*>(pars + PF_PARS * 32);     // [PF_PARS]: tokens whose value pair is not finite
  uint64_t* bars = reinterpret_cast<uint64_t*>(bad + PF_PARS);
  uint64_t *kfull = bars, *kempty = kfull + PF_RING, *vfull = kempty + PF_RING, *vempty = vfull + PF_RING;
  uint64_t* parfull = vempty + PF_RING;
  uint64_t *sfull = parfull + PF_PARS, *pfull = sfull + 4;        // [tile][buffer of S], pvdone too
  uint64_t *pvdone = pfull + 4, *drain = pvdone + 4;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 1);
  uint32_t *qmax = tmem_slot + 1, *qmin = tmem_slot + 2;   // largest and smallest of the rows' largest magnitudes

  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int i = 0; i < PF_RING; ++i) {
      mbar_init(&kfull[i], 2);
      mbar_init(&kempty[i], two ? 2 : 1);
      mbar_init(&vfull[i], 2);
      mbar_init(&vempty[i], two ? 2 : 1);
    }
    for (int i = 0; i < PF_PARS; ++i) mbar_init(&parfull[i], 4);
    for (int i = 0; i < 4; ++i) {
      mbar_init(&sfull[i], 1);
      mbar_init(&pfull[i], 4);
      mbar_init(&pvdone[i], 1);
    }
    mbar_init(drain, two ? 2 : 1);
    *qmax = 0;
    *qmin = 0x7f800000u;
    mbar_fence_init();
  }
  if (warp == 12) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }

  __syncthreads();
  // ---- queries: thread = row
  float qs[NG];                    // sums of the row's queries per group, times scale log2(e)
  float top = 0.0f;                // the row's largest magnitude
  int row = 0;
  uint4 v[CHUNKS];
  bool special = false;            // some row has large scores, or a power of two of its own
  if (warp < 8) {
    row = row0 + threadIdx.x;
    const bool live = row <= last_row;
    const uint16_t* src = static_cast<const uint16_t*>(a.q);
    if (live) src += (first + row / a.share) * a.q_st + (kh * a.share + row % a.share) * a.q_sh;
    float all = 0.0f;
#pragma unroll
    for (int i = 0; i < NG; ++i) qs[i] = 0.0f;
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c) {
      v[c] = live ? *reinterpret_cast<const uint4*>(src + 8 * c) : make_uint4(0, 0, 0, 0);
      const uint32_t* w = &v[c].x;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float2 h;
        if (p.bf16) h = make_float2(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xffff0000u));
        else h = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
        top = fmaxf(top, fmaxf(fabsf(h.x), fabsf(h.y)));
        all += fabsf(h.x) + fabsf(h.y);
        qs[c / (CHUNKS / NG)] += h.x + h.y;
      }
    }
    special = fabsf(a.scale * kLog2e) * all > kPfPlainSum;
#pragma unroll
    for (int i = 0; i < NG; ++i) qs[i] *= a.scale * kLog2e;
    // rows of zeros, and those with an infinity (which have no result to be exact in), have no say
    if (!(top < INFINITY)) top = 0.0f;
    const uint32_t hi = __reduce_max_sync(0xffffffffu, __float_as_uint(top));
    const uint32_t lo = __reduce_min_sync(0xffffffffu, top > 0.0f ? __float_as_uint(top) : 0x7f800000u);
    if (lane == 0) {
      atomicMax(qmax, hi);
      atomicMin(qmin, lo);
    }
  }
  special = __syncthreads_or(special);
  // exponents, kept where the powers of two below are normal
  auto exponent = [](uint32_t bits) { return max(static_cast<int>(bits >> 23) - 127, -112); };
  const int e2 = exponent(*qmax);
  const bool apart = e2 - exponent(*qmin) > kPfSpread;
  special |= apart;
  const int e_row = apart && top > 0.0f ? exponent(__float_as_uint(top)) : e2;
  const float ratio = e_row < e2 - 126 ? 0.0f : __uint_as_float(static_cast<uint32_t>(127 + e_row - e2) << 23);
  // what a product of codes c 2^-24 and queries scaled to 2^14 is multiplied by, with the key's scale
  const float f = a.scale * kLog2e * 1024.0f * __uint_as_float(static_cast<uint32_t>(127 + e2) << 23);
  if (warp < 8) {
    const float down = __uint_as_float(static_cast<uint32_t>(127 + 14 - e_row) << 23), down16 = down * 0.0625f;
    uint8_t* tile = qtile + (threadIdx.x >> 7) * KB * PF_TILE;
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c) {
      float x[8];
      const uint32_t* w = &v[c].x;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float2 h;
        if (p.bf16) h = make_float2(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xffff0000u));
        else h = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
        x[2 * i] = h.x;
        x[2 * i + 1] = h.y;
      }
      uint4 o;
      o.x = pack2<__half>(x[0] * down, x[4] * down);
      o.y = pack2<__half>(x[1] * down16, x[5] * down16);
      o.z = pack2<__half>(x[2] * down, x[6] * down);
      o.w = pack2<__half>(x[3] * down16, x[7] * down16);
      *reinterpret_cast<uint4*>(swizzled(tile + (c >> 3) * PF_TILE, threadIdx.x & 127, c & 7)) = o;
    }
    fence_proxy_async_smem();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  if (warp >= 12) {
    // ------------------------------ products ------------------------------
    const int t = warp - 12;
    if ((t == 0 || two) && elect_one()) {
      const uint32_t qk_desc = umma_idesc_f16_f32(128, TOK), pv_desc = umma_idesc_f16_f32(128, D) | kTransposeB;
      // the scores of step j into their buffer, after the products that read the probabilities there
      auto qk = [&](int j, bool ready) {
        if (!ready && !mbar_wait(&kfull[j % PF_RING], (j / PF_RING) & 1, p.wait_ns)) return false;
        tc_fence_after();
        const uint8_t* q = qtile + t * KB * PF_TILE;
        const uint8_t* k = ktile + (j % PF_RING) * SH::KV_BYTES;
        const uint32_t to = tmem + t * 128 + (j & 1) * 64;
#pragma unroll
        for (int kb = 0; kb < KB; ++kb) {
          const uint64_t qd = umma_desc_sw128(smem_u32(q + kb * PF_TILE)), kd = umma_desc_sw128(smem_u32(k + kb * SH::BLOCK_BYTES));
          const int g = NG == 2 ? kb : 0;
#pragma unroll
          for (int kk = 0; kk < 4; ++kk) tc_mma_f16(to + g * TOK, qd + kk * 2, kd + kk * 2, qk_desc, (NG == 1 && kb) || kk);
        }
        tc_commit(&sfull[t * 2 + (j & 1)]);
        tc_commit(&kempty[j % PF_RING]);
        return true;
      };
      bool ok = true;
      for (int j = 0; ok && j < min(2, steps); ++j) ok = qk(j, false);
      for (int j = 0; ok && j < steps; ++j) {
        // (the keys of step j + 2 are mostly there: looked at while the probabilities are not)
        const bool ready = j + 2 < steps && mbar_test(&kfull[(j + 2) % PF_RING], ((j + 2) / PF_RING) & 1);
        ok = mbar_wait(&vfull[j % PF_RING], (j / PF_RING) & 1, p.wait_ns) && mbar_wait(&pfull[t * 2 + (j & 1)], (j >> 1) & 1, p.wait_ns);
        if (!ok) break;
        tc_fence_after();
        const uint64_t vd = umma_desc_sw128_mn(smem_u32(vtile + (j % PF_RING) * SH::KV_BYTES), SH::BLOCK_BYTES);
#pragma unroll
        for (int kk = 0; kk < TOK / 16; ++kk)
          tc_mma_f16_ts(tmem + 256 + t * 128, tmem + t * 128 + (j & 1) * 64 + kk * 8, vd + kk * 128, pv_desc, j || kk);
        tc_commit(&pvdone[t * 2 + (j & 1)]);
        tc_commit(&vempty[j % PF_RING]);
        if (j + 2 < steps) ok = qk(j + 2, ready);
      }
      tc_commit(drain);
    }
  } else if (warp >= 8) {
    // ------------------------------ the cache: warps 8, 9 keys, 10, 11 values ------------------------------
    constexpr int CPT = CHUNKS / NG;                     // eights of channels per thread: one group's
    const bool values = warp >= 10;
    const int tok = threadIdx.x % TOK, g = threadIdx.x % 64 / TOK;
    uint4 next[CPT / 4];
    uint32_t next_pair;
    // this thread's bytes of a block, and the steps [lo, hi) whose token some row sees
    const int in_block = tok % BLK * (D / 2) + g * (CPT * 4) + (values ? value_codes_at(D) : 0);
    const int to_pair = (values ? value_pairs_at(D, NG) : key_pairs_at(D)) + (tok % BLK * NG + g) * 4 - in_block;
    const uint8_t* mine = a.cache.pool + kh * a.cache.page_bytes + in_block;
    const long long page_stride = a.cache.kv_heads * a.cache.page_bytes;
    const int* row_pages = a.table + static_cast<long long>(b) * a.width;
    const int tok_first = step0 * TOK + tok;
    const int lo = tok_first < from, hi = min(steps, tok_first < len ? (len - tok_first + TOK - 1) / TOK : 0);
    int page, block;                  // of the step after the next: looked up a step before its codes are read
    auto look_up = [&](int j) {
      page = 0;
      if (j < lo || j >= hi) return;
      const int at = (tok_first + j * TOK) / BLK, col = a.cache.blocks.quotient(at);
      page = row_pages[col];
      block = at - col * a.cache.page_blocks;
    };
    auto load = [&](int j) {
#pragma unroll
      for (int i = 0; i < CPT / 4; ++i) next[i] = make_uint4(0, 0, 0, 0);
      next_pair = 0;
      if (j < lo || j >= hi) return;
      if (static_cast<unsigned>(page) >= static_cast<unsigned>(a.cache.pages)) {
        flag_error(kErrIndex);                           // read as zeros
        return;
      }
      const uint8_t* codes = mine + page * page_stride + block * a.cache.block_bytes;
#pragma unroll
      for (int i = 0; i < CPT / 4; ++i) next[i] = *reinterpret_cast<const uint4*>(codes + 16 * i);
      next_pair = *reinterpret_cast<const uint32_t*>(codes + to_pair);
    };
    // the codes of a token as K, or with its scale and offset as V
    auto expand = [&](bool is_v, uint8_t* tile, const uint4 (&codes)[CPT / 4], __half2 scale, __half2 offset, bool clamp) {
      const uint32_t at = smem_u32(tile) + tok * 128 + ((tok & 7) << 4);     // of chunk 0; chunk c swaps bits with c
#pragma unroll
      for (int i = 0; i < CPT / 4; ++i) {
        const uint32_t* w = &codes[i].x;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const int c = g * CPT + 4 * i + k;
          uint4 o;
          if (is_v) o = value_word(w[k], scale, offset, clamp);
          else o = masked_word(w[k]);
          asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"((at ^ ((c & 7) << 4)) + (c >> 3) * SH::BLOCK_BYTES),
                       "r"(o.x), "r"(o.y), "r"(o.z), "r"(o.w) : "memory");
        }
      }
      fence_proxy_async_smem();
      __syncwarp();
    };
    uint64_t *full = values ? vfull : kfull, *empty = values ? vempty : kempty;
    look_up(0);
    load(0);
    look_up(1);
    bool ok = true;
    for (int j = 0; ok && j < steps; ++j) {
      uint4 codes[CPT / 4];
#pragma unroll
      for (int i = 0; i < CPT / 4; ++i) codes[i] = next[i];
      const uint32_t pair = next_pair;
      load(j + 1);
      look_up(j + 2);
      const float2 so = __half22float2(*reinterpret_cast<const __half2*>(&pair));
      const bool finite = fabsf(so.x) < INFINITY && fabsf(so.y) < INFINITY;
      // The pairs of step j - PF_PARS have been read: this warp has seen step j - 1 - PF_RING leave its
      // ring, a value tile after that step's probabilities, a key tile after those two steps before it.
      const int slot = j % PF_PARS, ring = j % PF_RING;
      uint8_t* tile = (values ? vtile : ktile) + ring * SH::KV_BYTES;
      if (values) {
        const uint32_t word = __ballot_sync(0xffffffffu, !finite);
        if (lane == 0) reinterpret_cast<uint32_t*>(bad + slot)[warp - 10] = word;
      } else {
        float* par = reinterpret_cast<float*>(pars + slot * 32 + (tok >> 1) * NG + g) + (tok & 1);
        par[0] = so.x * f;
        par[2] = so.y;
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&parfull[slot]);
      ok = mbar_wait_backoff(&empty[ring], ((j / PF_RING) & 1) ^ 1u, p.wait_ns, 64);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      if (values) {
        const uint32_t held = finite ? pair : 0;
        const __half2 h = *reinterpret_cast<const __half2*>(&held), sc = __low2half2(h), of = __high2half2(h);
        if (__any_sync(0xffffffffu, finite && 15.0f * fabsf(so.x) + fabsf(so.y) > kMaxF16)) expand(true, tile, codes, sc, of, true);
        else expand(true, tile, codes, sc, of, false);
      } else {
        expand(false, tile, codes, __half2(), __half2(), false);
      }
      if (lane == 0) mbar_arrive(&full[ring]);
    }
  } else if (warp < 4 || two) {
    // ------------------------------ softmax ------------------------------
    const int t = warp >> 2;
    const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const uint32_t s_at = tmem + lanes + t * 128, o_at = tmem + lanes + 256 + t * 128;
    const bool live = row <= last_row;
    const int pos = len - count + row / a.share;
    const int see_to = live ? min(len, pos + 1) : len, see_from = live ? sees_from(a, pos) : 0;
    // tokens every row of this tile sees
    const int tile_last = min(last_row, row0 + t * 128 + 127);
    const int all_to = min(len, len - count + (row0 + t * 128) / a.share + 1);
    const int all_from = sees_from(a, len - count + tile_last / a.share);
    float m = 0.0f, l = 0.0f;
    uint32_t nan_groups = 0;         // groups whose values are NaN in some token this row sees
    bool fresh = true, ok = true, scores = false, pairs = false;   // the next step's are there
    for (int j = 0; j < steps; ++j) {
      const int slot = j % PF_PARS;
      const uint32_t buf = s_at + (j & 1) * 64;
      ok = (pairs || mbar_wait(&parfull[slot], (j / PF_PARS) & 1, p.wait_ns)) &&
           (scores || mbar_wait(&sfull[t * 2 + (j & 1)], (j >> 1) & 1, p.wait_ns));
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      tc_fence_after();
      const int tok0 = (step0 + j) * TOK;
      const bool edge = special || tok0 < all_from || tok0 + TOK > all_to;
      const float4* par = pars + slot * 32;
      uint32_t h[TOK / 2];
      float l_add;
#pragma unroll 1
      for (int pass = 0; pass < 2; ++pass) {
        const float most = edge ? step_probabilities<NG, TOK, true>(buf, par, m, qs, see_from - tok0, see_to - tok0, ratio, h, l_add)
                                : step_probabilities<NG, TOK, false>(buf, par, m, qs, 0, 0, 1.0f, h, l_add);
        const float over = most - m;
        const bool grow = over > (fresh ? -INFINITY : kPfLazyMax);
        if (pass || !__any_sync(0xffffffffu, grow)) break;
        const float by = grow && !fresh ? ex2(-over) : 1.0f;
        if (grow) {
          m = most;
          fresh = false;
        }
        l *= by;
        if (j > 0) {                     // the sums so far
          ok = __all_sync(0xffffffffu, mbar_wait(&pvdone[t * 2 + ((j - 1) & 1)], ((j - 1) >> 1) & 1, p.wait_ns));
          if (!ok) break;
          tc_fence_after();
#pragma unroll 1
          for (int c = 0; c < D; c += 16) {
            uint32_t x[16];
            tmem_ld_cols(o_at + c, x);
            tmem_ld_done(x);
#pragma unroll
            for (int i = 0; i < 16; ++i) x[i] = __float_as_uint(__uint_as_float(x[i]) * by);
            tmem_st_32x32b_x16(o_at + c, x);
          }
        }
      }
      if (!ok) break;
      l += l_add;
#pragma unroll
      for (int c = 0; c < TOK / 2; c += 16) {
        uint32_t r[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) r[i] = h[c + i];
        tmem_st_32x32b_x16(buf + c, r);
      }
      const uint2 bads = bad[slot];
      if (bads.x | bads.y) {
        const uint32_t words[2] = {bads.x, bads.y};
#pragma unroll
        for (int w = 0; w < 2; ++w)
          for (uint32_t left = words[w]; left; left &= left - 1) {
            const int tok = tok0 + w * 32 % TOK + __ffs(left) - 1;
            if (tok >= see_from && tok < see_to) nan_groups |= 1u << (w * 32 / TOK);
          }
        __syncwarp();
      }
      // the next step's barriers, while the stores are under way
      pairs = j + 1 < steps && mbar_test(&parfull[(j + 1) % PF_PARS], ((j + 1) / PF_PARS) & 1);
      scores = j + 1 < steps && mbar_test(&sfull[t * 2 + ((j + 1) & 1)], ((j + 1) >> 1) & 1);
      tmem_st_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&pfull[t * 2 + (j & 1)]);
    }
    // ---- the row's result
    // (a barrier per buffer: the scores of the last step have shown its phase before to be over)
    if (ok && steps > 0)
      ok = __all_sync(0xffffffffu, mbar_wait(&pvdone[t * 2 + ((steps - 1) & 1)], ((steps - 1) >> 1) & 1, p.wait_ns));
    tc_fence_after();
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    const long long at = static_cast<long long>(first + row / a.share) * a.heads + kh * a.share + row % a.share;
    uint16_t* out = static_cast<uint16_t*>(a.o) + at * D;
#pragma unroll 1
    for (int c = 0; c < D; c += 16) {
      uint32_t x[16];
      __syncwarp();
      if (steps > 0) {
        tmem_ld_cols(o_at + c, x);
        tmem_ld_done(x);
      }
      const bool gone = nan_groups >> (c < D / NG ? 0 : NG - 1) & 1;
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        float y[8];
#pragma unroll
        for (int i = 0; i < 8; ++i)     // column order 0 4 1 5 2 6 3 7
          y[(i >> 1) + (i & 1) * 4] = gone ? NAN : steps > 0 && l != 0.0f ? __uint_as_float(x[8 * k + i]) * inv : 0.0f;
        uint4 o;
        uint32_t* ow = &o.x;
#pragma unroll
        for (int i = 0; i < 4; ++i)
          ow[i] = p.bf16 ? pack2<__nv_bfloat16>(y[2 * i], y[2 * i + 1]) : pack2<__half>(y[2 * i], y[2 * i + 1]);
        if (live && ok) *reinterpret_cast<uint4*>(out + c + 8 * k) = o;
      }
    }
    if (live && ok && a.lse) a.lse[at] = l == 0.0f ? -INFINITY : (m + log2f(l)) * kLn2;
  }

  __syncwarp();
  tc_fence_before();
  __syncthreads();
  if (warp == 12) {
    mbar_wait(drain, 0, kWaitBudgetNs);   // every product has finished before TMEM is released
    __syncwarp();
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

}  // namespace kv4
}  // namespace w4a16
