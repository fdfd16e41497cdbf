// kv4_prefill.cuh -- attention over the 4-bit cache for many query rows per kv head (prompts and
// their chunks): o = softmax(scale q k^T) v on the 5th-generation tensor cores.
//
// Compute-bound: 4 D operations per row and token. A block takes 256 rows (query token, head of
// the group) of one kv head as two tiles of 128, and 128 tokens at a time (64 with two groups):
//   warps 0-3, 4-7  softmax of row tile 0 and 1, one row per thread (TMEM lane): queries scaled and
//                   written to shared memory once; then per step the scores from TMEM, the running
//                   maximum, probabilities times value scales as fp16 over their scores' columns
//                   (the A operand of the second product), and at the end the sums, divided
//   warps 8-11      the cache: a token (or one group of it) per thread, read a step ahead; its codes
//                   as fp16 into the K and V tiles, its pairs as fp32 beside them
//   warp 12         issues tcgen05.mma: S_t = Q_t K^T (both operands in shared memory), O_t += P_t V
//                   (P from TMEM, V as it lies, token-major, through the transposing descriptor)
// While one row tile's softmax runs, the tensor cores work on the other's products:
//   PV0(j) QK0(j+1) | PV1(j) QK1(j+1) | ...
// The products of one thread run in order, so QK_t(j+1) may write over P_t(j) after PV_t(j).
//
// As in the decode kernel the tensor cores see codes, not values: a key's scale and offset act on its
// scores, a value's scale on its probability, in fp32, so the scores carry no rounding of keys
// (values rounded to fp16 first move a log-sum-exp by some 1e-3 where scores reach 80) and p s is
// the one rounding to 16 bits. Keys' codes are masked words, c 2^-24 (queries carry the 1/16 of odd
// nibbles); values' are c - 8, so that what p s loses meets centred numbers, and
// sum p v = sum (p s)(c - 8) + sum p (b + 8 s). With two groups of channels each has its own product
// S, probabilities and half of V.
//
// TMEM columns: S0 128, S1 128 (with P over them), O0 128, O1 128: all 512. Channels lie in the
// order 0 4 1 5 2 6 3 7 inside each eight (how a masked word gives them): in Q and K alike, which
// leaves the scores as they are, and in V, which the last step undoes.
//
// The probabilities of half a step are taken with the running maximum as it stands, and again in
// the rare case that some score of the warp's rows exceeds it by kLazyMax: one pass over the scores
// instead of two. Every wait is bounded; on expiry the block raises the device error bit and leaves.
#pragma once

#include "kv4_decode.cuh"

namespace w4a16 {
namespace kv4 {

constexpr int PF_ROWS = 256;         // query rows per block (two tiles)
constexpr int PF_THREADS = 13 * 32;
constexpr int PF_TILE = 128 * 128;   // bytes of a [128][64] fp16 tile
constexpr int PF_PARS = 4;           // steps whose pairs are kept

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
  static constexpr int TOK = 128 / NG;                    // tokens per step
  static constexpr int Q_BYTES = 2 * KB * PF_TILE;
  static constexpr int BLOCK_BYTES = TOK * 128;           // [TOK][64] fp16
  static constexpr int KV_BYTES = KB * BLOCK_BYTES;       // one K or V tile
  static constexpr int PAR_BYTES = PF_PARS * 128 * 16;
  static constexpr int SMEM_BYTES = 1024 + Q_BYTES + 4 * KV_BYTES + PAR_BYTES + 256;
  static_assert(SMEM_BYTES <= 227 * 1024, "shared memory budget");
};

// One word's eight codes, (0,4) (1,5) (2,6) (3,7): c 2^-24 and 16 c 2^-24 in turn, or c - 8.
__device__ __forceinline__ uint4 masked_word(uint32_t w) {
  const uint32_t u = w >> 8;
  return make_uint4(w & 0x000f000fu, w & 0x00f000f0u, u & 0x000f000fu, u & 0x00f000f0u);
}
__device__ __forceinline__ uint4 centred_word(uint32_t w) {
  const uint32_t u = w >> 8;
  // 1024 + c and 64 + c, less 1032 and 72
  return make_uint4(hadd2_u32(lop3_and_or(w, 0x000F000Fu, 0x64006400u), 0xE408E408u),
                    hadd2_u32(lop3_and_or(w, 0x00F000F0u, 0x54005400u), 0xD480D480u),
                    hadd2_u32(lop3_and_or(u, 0x000F000Fu, 0x64006400u), 0xE408E408u),
                    hadd2_u32(lop3_and_or(u, 0x00F000F0u, 0x54005400u), 0xD480D480u));
}

__device__ __forceinline__ uint8_t* swizzled(uint8_t* tile, int row, int chunk) {
  return tile + row * 128 + ((chunk ^ (row & 7)) << 4);
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
  const int from = a.window ? max(0, pos0 - a.window + 1) : 0, to = min(len, pos1 + 1);
  const int step0 = from / TOK;
  const int steps = max(0, (to + TOK - 1) / TOK - step0);
  const bool two = row0 + 128 <= last_row;

  extern __shared__ __align__(1024) uint8_t smem_raw[];
  // an offset, not a cast: the compiler then knows its loads to be from shared memory
  uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  uint8_t* qtile = smem;
  uint8_t* ktile = qtile + SH::Q_BYTES;                   // two buffers, then V's two
  uint8_t* vtile = ktile + 2 * SH::KV_BYTES;
  float4* pars = reinterpret_cast<float4*>(vtile + 2 * SH::KV_BYTES);   // [PF_PARS][NG][TOK]
  uint64_t* bars = reinterpret_cast<uint64_t*>(pars + PF_PARS * 128);
  uint64_t *kfull = bars, *kempty = bars + 2, *vfull = bars + 4, *vempty = bars + 6;
  uint64_t *sfull = bars + 8, *pfull = bars + 10, *pvdone = bars + 12, *drain = bars + 14;
  uint64_t* parfull = bars + 15;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 15 + PF_PARS);
  uint32_t* qmax = tmem_slot + 1;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(&kfull[i], 4);
      mbar_init(&kempty[i], 1);
      mbar_init(&vfull[i], 4);
      mbar_init(&vempty[i], 1);
      mbar_init(&sfull[i], 1);
      mbar_init(&pfull[i], 4);
      mbar_init(&pvdone[i], 1);
    }
    for (int i = 0; i < PF_PARS; ++i) mbar_init(&parfull[i], 4);
    mbar_init(drain, 1);
    *qmax = 0;
    mbar_fence_init();
  }
  if (warp == 12) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }

  __syncthreads();
  // ---- queries: thread = row; all of the block's scaled by one power of two to a largest magnitude in
  // [1, 2) (exact), so bf16 ones fit fp16
  float qs[NG];                    // sums of the row's queries per group, times scale log2(e)
  int row = 0;
  uint4 v[CHUNKS];
  if (warp < 8) {
    row = row0 + threadIdx.x;
    const bool live = row <= last_row;
    const uint16_t* src = static_cast<const uint16_t*>(a.q);
    if (live) src += (first + row / a.share) * a.q_st + (kh * a.share + row % a.share) * a.q_sh;
    float top = 0.0f;
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
        qs[c / (CHUNKS / NG)] += h.x + h.y;
      }
    }
#pragma unroll
    for (int i = 0; i < NG; ++i) qs[i] *= a.scale * kLog2e;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    if (lane == 0) atomicMax(qmax, __float_as_uint(top));
  }
  __syncthreads();
  const int e2 = min(max(static_cast<int>(*qmax >> 23) - 127, -100), 100);
  // what a product of codes c 2^-24 and scaled queries is multiplied by, with the key's scale
  const float f = a.scale * kLog2e * 16777216.0f * __uint_as_float(static_cast<uint32_t>(127 + e2) << 23);
  if (warp < 8) {
    const float down = __uint_as_float(static_cast<uint32_t>(127 - e2) << 23), down16 = down * 0.0625f;
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

  if (warp == 12) {
    // ------------------------------ products ------------------------------
    if (lane == 0) {
      const uint32_t qk_desc = umma_idesc_f16_f32(128, TOK), pv_desc = umma_idesc_f16_f32(128, D / NG) | kTransposeB;
      auto qk = [&](int t, int j) {
        const uint8_t* q = qtile + t * KB * PF_TILE;
        const uint8_t* k = ktile + (j & 1) * SH::KV_BYTES;
#pragma unroll
        for (int kb = 0; kb < KB; ++kb) {
          const uint64_t qd = umma_desc_sw128(smem_u32(q + kb * PF_TILE)), kd = umma_desc_sw128(smem_u32(k + kb * SH::BLOCK_BYTES));
          const int g = NG == 2 ? kb : 0;
#pragma unroll
          for (int kk = 0; kk < 4; ++kk)
            tc_mma_f16(tmem + t * 128 + g * TOK, qd + kk * 2, kd + kk * 2, qk_desc, (NG == 1 && kb) || kk);
        }
        tc_commit(&sfull[t]);
      };
      bool ok = true;
      if (steps > 0) {
        ok = mbar_wait(&kfull[0], 0, p.wait_ns);
        tc_fence_after();
        if (ok) {
          qk(0, 0);
          if (two) qk(1, 0);
          tc_commit(&kempty[0]);
        }
      }
      for (int j = 0; ok && j < steps; ++j) {
        for (int t = 0; ok && t < (two ? 2 : 1); ++t) {
          ok = (t || mbar_wait(&vfull[j & 1], (j >> 1) & 1, p.wait_ns)) && mbar_wait(&pfull[t], j & 1, p.wait_ns);
          if (!ok) break;
          tc_fence_after();
#pragma unroll
          for (int g = 0; g < NG; ++g) {
            const uint64_t vd = umma_desc_sw128_mn(smem_u32(vtile + (j & 1) * SH::KV_BYTES + g * SH::BLOCK_BYTES), SH::BLOCK_BYTES);
#pragma unroll
            for (int kk = 0; kk < TOK / 16; ++kk)
              tc_mma_f16_ts(tmem + 256 + t * 128 + g * 64, tmem + t * 128 + g * TOK + kk * 8, vd + kk * 128, pv_desc, j || kk);
          }
          tc_commit(&pvdone[t]);
          if (t == 1 || !two) tc_commit(&vempty[j & 1]);
          if (j + 1 < steps) {
            if (t == 0) {
              ok = mbar_wait(&kfull[(j + 1) & 1], ((j + 1) >> 1) & 1, p.wait_ns);
              if (!ok) break;
              tc_fence_after();
            }
            qk(t, j + 1);
            if (t == 1 || !two) tc_commit(&kempty[(j + 1) & 1]);
          }
        }
      }
      tc_commit(drain);
    }
  } else if (warp >= 8) {
    // ------------------------------ the cache ------------------------------
    constexpr int CPT = CHUNKS / NG;                     // eights of channels per thread: one group's
    const int tok = (threadIdx.x - 256) % TOK, g = (threadIdx.x - 256) / TOK;
    uint4 kc[CPT / 4], vc[CPT / 4];
    uint32_t kp, vp;
    auto page_of = [&](int j) {       // the page of this thread's token of step j, or -1
      const int t = (step0 + j) * TOK + tok;
      if (j >= steps || t >= len || t < from) return -1;
      const int page = a.table[static_cast<long long>(b) * a.width + (t / BLK) / a.cache.page_blocks];
      if (static_cast<unsigned>(page) < static_cast<unsigned>(a.cache.pages)) return page;
      flag_error(kErrIndex);          // read as zeros
      return -1;
    };
    auto load = [&](int j, int page) {
      const int t = (step0 + j) * TOK + tok;
      if (page < 0) {
#pragma unroll
        for (int i = 0; i < CPT / 4; ++i) kc[i] = vc[i] = make_uint4(0, 0, 0, 0);
        kp = vp = 0;
        return;
      }
      const uint8_t* blk = block_ptr(a.cache, page, kh, t / BLK % a.cache.page_blocks);
      const int tb = t % BLK;
#pragma unroll
      for (int i = 0; i < CPT / 4; ++i) {
        kc[i] = *reinterpret_cast<const uint4*>(blk + tb * (D / 2) + g * (CPT * 4) + 16 * i);
        vc[i] = *reinterpret_cast<const uint4*>(blk + value_codes_at(D) + tb * (D / 2) + g * (CPT * 4) + 16 * i);
      }
      kp = *reinterpret_cast<const uint32_t*>(blk + key_pairs_at(D) + (tb * NG + g) * 4);
      vp = *reinterpret_cast<const uint32_t*>(blk + value_pairs_at(D, NG) + (tb * NG + g) * 4);
    };
    auto expand = [&](uint8_t* tile, const uint4 (&codes)[CPT / 4], bool centred) {
#pragma unroll
      for (int i = 0; i < CPT / 4; ++i) {
        const uint32_t* w = &codes[i].x;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const int c = g * CPT + 4 * i + k;
          *reinterpret_cast<uint4*>(swizzled(tile + (c >> 3) * SH::BLOCK_BYTES, tok, c & 7)) = centred ? centred_word(w[k]) : masked_word(w[k]);
        }
      }
      fence_proxy_async_smem();
      __syncwarp();
    };
    int page = page_of(0);
    load(0, page);
    page = page_of(1);
    bool ok = true;
    for (int j = 0; ok && j < steps; ++j) {
      uint4 kc1[CPT / 4], vc1[CPT / 4];
#pragma unroll
      for (int i = 0; i < CPT / 4; ++i) {
        kc1[i] = kc[i];
        vc1[i] = vc[i];
      }
      const float2 ks = __half22float2(*reinterpret_cast<const __half2*>(&kp)), vs = __half22float2(*reinterpret_cast<const __half2*>(&vp));
      load(j + 1, page);
      page = page_of(j + 2);
      // the pairs of step j - PF_PARS have been read: its products were done before step j - 2's V tile
      // was written over
      pars[((j % PF_PARS) * NG + g) * TOK + tok] = make_float4(ks.x * f, ks.y, vs.x, fmaf(8.0f, vs.x, vs.y));
      __syncwarp();
      if (lane == 0) mbar_arrive(&parfull[j % PF_PARS]);
      ok = mbar_wait_backoff(&kempty[j & 1], ((j >> 1) & 1) ^ 1u, p.wait_ns, 64);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      expand(ktile + (j & 1) * SH::KV_BYTES, kc1, false);
      if (lane == 0) mbar_arrive(&kfull[j & 1]);
      ok = mbar_wait_backoff(&vempty[j & 1], ((j >> 1) & 1) ^ 1u, p.wait_ns, 64);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      expand(vtile + (j & 1) * SH::KV_BYTES, vc1, true);
      if (lane == 0) mbar_arrive(&vfull[j & 1]);
    }
  } else if (warp < 4 || two) {
    // ------------------------------ softmax ------------------------------
    const int t = warp >> 2;
    const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const uint32_t s_at = tmem + lanes + t * 128, o_at = tmem + lanes + 256 + t * 128;
    const bool live = row <= last_row;
    const int pos = len - count + row / a.share;
    const int see_to = live ? min(len, pos + 1) : len, see_from = live && a.window ? max(0, pos - a.window + 1) : 0;
    // tokens every row of this tile sees
    const int tile_last = min(last_row, row0 + t * 128 + 127);
    const int all_to = min(len, len - count + (row0 + t * 128) / a.share + 1);
    const int all_from = a.window ? max(0, len - count + tile_last / a.share - a.window + 1) : 0;
    constexpr int HT = 64 / NG;                          // tokens of half a step
    float m = 0.0f, l = 0.0f, corr[NG];                  // l = sum p, corr = sum p (b + 8 s)
#pragma unroll
    for (int g = 0; g < NG; ++g) corr[g] = 0.0f;
    bool fresh = true, ok = true;
    // The probabilities of half a step with the maximum m: h = p s in fp16, packed by token pairs, and
    // what l and corr gain; returns the largest score over m.
    auto half_step = [&](auto edge_tag, const float4* par, uint32_t s_half, int tok0, uint32_t (&h)[NG][HT / 2],
                         float& l_add, float (&c_add)[NG]) {
      constexpr bool EDGE = decltype(edge_tag)::value;
      float top = -INFINITY;
      l_add = 0.0f;
#pragma unroll
      for (int g = 0; g < NG; ++g) c_add[g] = 0.0f;
#pragma unroll
      for (int c = 0; c < HT; c += 32) {
        uint32_t x[NG][32];
#pragma unroll
        for (int g = 0; g < NG; ++g) tmem_ld_32x32b_x32(s_half + g * TOK + c, x[g]);
        tmem_ld_wait();
#pragma unroll
        for (int i = 0; i < 32; i += 2) {
          float ps[NG][2];
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            float4 q[NG];
            float y = -m;
#pragma unroll
            for (int g = 0; g < NG; ++g) {
              q[g] = par[g * TOK + c + i + k];
              y = fmaf(q[g].y, qs[g], y);
            }
#pragma unroll
            for (int g = 0; g < NG; ++g) y = fmaf(__uint_as_float(x[g][i + k]), q[g].x, y);
            if (EDGE && (tok0 + c + i + k < see_from || tok0 + c + i + k >= see_to)) y = -INFINITY;
            top = fmaxf(top, y);
            const float e = ex2(y);
            l_add += e;
#pragma unroll
            for (int g = 0; g < NG; ++g) {
              if (EDGE && e == 0.0f) {     // a token that is not seen may have any pair, NaN too
                ps[g][k] = 0.0f;
              } else {
                ps[g][k] = e * q[g].z;
                c_add[g] = fmaf(e, q[g].w, c_add[g]);
              }
            }
          }
#pragma unroll
          for (int g = 0; g < NG; ++g) h[g][(c + i) / 2] = pack2<__half>(ps[g][0], ps[g][1]);
        }
      }
      return top;
    };
    auto store_half = [&](uint32_t at, const uint32_t (&h)[HT / 2]) {
#pragma unroll
      for (int c = 0; c < HT / 2; c += 16) {
        uint32_t r[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) r[i] = h[c + i];
        tmem_st_32x32b_x16(at + c, r);
      }
    };
    for (int j = 0; ok && j < steps; ++j) {
      ok = mbar_wait(&sfull[t], j & 1, p.wait_ns) && mbar_wait(&parfull[j % PF_PARS], (j / PF_PARS) & 1, p.wait_ns);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      tc_fence_after();
      const int tok0 = (step0 + j) * TOK;
      const bool edge = tok0 < all_from || tok0 + TOK > all_to;
#pragma unroll 1
      for (int half = 0; half < 2; ++half) {
        const float4* par = pars + (j % PF_PARS) * NG * TOK + half * HT;
        uint32_t h[NG][HT / 2];
        float l_add, c_add[NG];
        auto take = [&]() {
          return edge ? half_step(std::true_type(), par, s_at + half * HT, tok0 + half * HT, h, l_add, c_add)
                      : half_step(std::false_type(), par, s_at + half * HT, tok0 + half * HT, h, l_add, c_add);
        };
        float top = take();
        const bool grow = top > (fresh ? -INFINITY : kLazyMax);
        if (__any_sync(0xffffffffu, grow)) {
          const float by = grow && !fresh ? ex2(-top) : 1.0f;
          if (grow) {
            m += top;
            fresh = false;
          }
          l *= by;
#pragma unroll
          for (int g = 0; g < NG; ++g) corr[g] *= by;
          if (j > 0) {                   // the sums so far
            ok = __all_sync(0xffffffffu, mbar_wait(&pvdone[t], (j - 1) & 1, p.wait_ns));
            if (!ok) break;
            tc_fence_after();
#pragma unroll 1
            for (int c = 0; c < D; c += 16) {
              uint32_t x[16];
              tmem_ld_32x32b_x16(o_at + c, x);
              tmem_ld_wait();
#pragma unroll
              for (int i = 0; i < 16; ++i) x[i] = __float_as_uint(__uint_as_float(x[i]) * by);
              tmem_st_32x32b_x16(o_at + c, x);
            }
          }
          if (half) {                    // and this step's first half, stored already
            tmem_st_wait();
            const __half2 by2 = __float2half2_rn(by);
#pragma unroll 1
            for (int c = 0; c < HT / 2 * NG; c += 16) {
              uint32_t x[16];
              const uint32_t at = s_at + c / (HT / 2) * TOK + c % (HT / 2);
              tmem_ld_32x32b_x16(at, x);
              tmem_ld_wait();
#pragma unroll
              for (int i = 0; i < 16; ++i) {
                const __half2 z = __hmul2(*reinterpret_cast<const __half2*>(&x[i]), by2);
                x[i] = *reinterpret_cast<const uint32_t*>(&z);
              }
              tmem_st_32x32b_x16(at, x);
            }
          }
          top = take();
        }
        l += l_add;
#pragma unroll
        for (int g = 0; g < NG; ++g) {
          corr[g] += c_add[g];
          store_half(s_at + g * TOK + half * (HT / 2), h[g]);
        }
      }
      if (!ok) break;
      tmem_st_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&pfull[t]);
    }
    // ---- the row's result
    if (ok && steps > 0) ok = __all_sync(0xffffffffu, mbar_wait(&pvdone[t], (steps - 1) & 1, p.wait_ns));
    tc_fence_after();
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    const long long at = static_cast<long long>(first + row / a.share) * a.heads + kh * a.share + row % a.share;
    uint16_t* out = static_cast<uint16_t*>(a.o) + at * D;
#pragma unroll 1
    for (int c = 0; c < D; c += 16) {
      uint32_t x[16];
      __syncwarp();
      if (steps > 0) {
        tmem_ld_32x32b_x16(o_at + c, x);
        tmem_ld_wait();
      }
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        float y[8];
#pragma unroll
        for (int i = 0; i < 8; ++i)     // column order 0 4 1 5 2 6 3 7
          y[(i >> 1) + (i & 1) * 4] = steps > 0 && l != 0.0f ? (__uint_as_float(x[8 * k + i]) + (c < D / NG ? corr[0] : corr[NG - 1])) * inv : 0.0f;
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
