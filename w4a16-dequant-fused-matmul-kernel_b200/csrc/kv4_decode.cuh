// kv4_decode.cuh -- attention over the 4-bit cache for few query rows per kv head (single new
// tokens, drafted tokens, the heads that share a kv head): o = softmax(scale q k^T) v.
//
// Memory-bound by design: a token of a kv head is D + 8 D / G bytes, read once for all the query
// rows (query token, head of the group) that share it. What a row costs beside is arithmetic on
// codes, so codes are never turned into values:
//   q . k = s_k (q . c) + b_k sum(q)          (per group of G channels; s, b the token's pair)
//   sum_t p_t v_t = sum_t (p_t s_t) c_t + sum_t p_t b_t
// A code masked out of its word, (w & 0x000f000f), is a pair of fp16 subnormals c * 2^-24, which
// the tensor cores multiply exactly: no conversion, one AND per two codes. Nibbles at bits 4-7
// give 16 c * 2^-24; the queries' fragments for them carry 1/16, and the sums of the values'
// channels with an odd nibble are divided by 16 at the end.
//
// Each row's queries are scaled by a power of two of its own to a largest magnitude in [2^14, 2^15): any bf16
// query then fits fp16, its channels are exact down to 2^-24 of the row's largest (odd nibbles with their 1/16),
// and no row's magnitude (an infinity, say) tells on its neighbours. It costs two multiplications per 16 tokens
// and group: 1 us of 73 for the long case below, nothing measurable with one group per head.
//
// p s is the one rounding to 16 bits, h (2^-11). Rounded against codes of 7.5 on average it would cost more than a
// rounding of p against centred values, so the sum is taken as sum h (c - 7.5) + sum p (b + 7.5 s), the second term
// in fp32; the sum of h comes from one more product, with ones. So that h has its 11 bits for small values too, the
// values' scales are multiplied by 2^10 (p s >= 2^-24 is then a normal number; unscaled, a mean of values of 1e-4 is off
// by 2%), and by less from the first scale above 8 on that a warp meets, so that p s stays finite. A group without
// spread has the scale 1 and codes of zero: its scale is taken as zero, or 7.5 times the rounding of its p would stand
// beside its offset, which may be nothing. Looking for both costs 0.2 us for one token and 2 of 76 for a batch.
//
// Both products take the cache as the M side of mma.m16n8k16 (16 tokens, or 16 channels) and
// eight query rows as its N side, so no row of the tensor core is wasted on padding queries when
// eight heads share a kv head. S^T comes out with tokens along lanes; movmatrix turns it into the
// B fragment of the second product.
//
// Work: a segment is a kv head of a sequence (and a tile of 8 NT of its rows), a tile TB blocks
// of 16 tokens. All tiles form one list that N teams of warps split evenly, whatever the lengths
// (a segment counts `seg_cost` tiles more than it has, for its queries and its epilogue); a team that holds a
// part of a segment leaves (m, l, o) in the workspace and, when all its tiles are done, the last of the segment's
// teams to arrive joins the parts in team order, so results do not depend on timing. (Where there are teams enough
// and no segment is much longer than the others, each team takes one whole segment.) Each warp feeds itself: two
// stages of a tile, filled by copies that its own lane 0 issues. A piece's end passes through shared memory once:
// each warp leaves its sums in the stage it has just read, and each then adds up some rows over all warps.
//
// Two sequences of 131071 and 107000 tokens, 32 heads of 128 channels in groups of 64 on 8 kv heads (274 MB): 74.5 us,
// 3.7 TB/s; 61 of up to 8000 tokens, 64 heads on 8 (298 MB): 80 us, 3.7 TB/s; one of 777 tokens: 12.1 us. By the
// batch's counters no unit is full: 54% of the issue slots, 54% of the ALU pipe (masking codes, packing), 22% of
// the tensor pipe, with four warps to a scheduler (128 registers), which mostly wait for an instruction before theirs.
// Timed inside the kernel, when the long case took 74 us: 51 in the tile loop (5.4 TB/s), 3 until the first copy is
// issued (lengths, prefix sums, the table), 4 at a piece's end, 5 in joining parts; the other 11 have no name yet.
#pragma once

#include <type_traits>

#include "kv4_attend.cuh"

namespace w4a16 {
namespace kv4 {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr float kNoMax = -1e30f;           // running maximum before any token
// The running maximum follows only when a score exceeds it by this much (log2): p <= 7.46, and
// p * s stays finite in fp16 as the scales are brought to at most kMostScale.
constexpr float kLazyMax = 2.9f, kMostScale = 8192.0f;
constexpr int MAX_SEQS = 2048;             // sequences per launch (their prefix sums lie in shared memory)

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ uint32_t movmatrix_trans(uint32_t a) {
  uint32_t d;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
  return d;
}

__device__ __forceinline__ void mma16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// The same with accumulators that start at zero.
__device__ __forceinline__ void mma16816_first(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                               uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.0f));
}

// Bulk copy of `bytes` (a multiple of 16) into shared memory, completing on `bar`.
__device__ __forceinline__ void bulk_load(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
                   smem_u32(dst)),
               "l"(src), "r"(bytes), "r"(smem_u32(bar))
               : "memory");
}

struct DecodeParams {
  AttendParams a;
  int bf16;                // q and o bf16, else fp16
  int row_limit;           // sequences with more rows than this are left to the other kernel
  int before, after;       // whether queries before cu_q[0], and from cu_q[seqs] on, are this launch's
  int team_warps;          // warps per team: 1, 2, 4, ... W
  int seg_cost;            // tiles that a segment counts more than it has
  int teams;               // most teams (CTAs * W / team_warps)
  int* counters;           // [teams] arrivals at a segment that several teams share, by the first of them; left zero
  float* parts;            // [teams * 2] partial results
  unsigned long long wait_ns;
};

template <int D, int NG, int NT, int W, int TB>
struct DecodeShape {
  static constexpr int SETS = D / 64;                    // sets of 8 words per token
  static constexpr int BLOCK = block_bytes(D, NG);
  static constexpr int STAGE = TB * BLOCK;
  static constexpr int R4 = NT * SETS * 4;               // rows of 32 float4: a warp's (or team's) sums
  static constexpr int SMALL = 8 * NT * (2 + NG);        // and for each query row m, l, corr [NG]
  static constexpr int PART = R4 * 128 + SMALL;          // floats of a part in the workspace
  static constexpr int RING_BYTES = W * 2 * STAGE;
  static constexpr int SMEM_BYTES = RING_BYTES + W * SMALL * 4 + MAX_SEQS * 20 + 16 + W * 2 * 8 + W * 16 + 64;
  static_assert(STAGE % 16 == 0 && STAGE >= R4 * 512, "a stage holds a warp's sums");
  static_assert(SMEM_BYTES <= 227 * 1024, "shared memory budget");
};

// A sequence as the list of tiles has it: where its tiles and its segments begin, its queries (none:
// it has no tile in this launch) and cached tokens.
struct Sequence {
  int prefix, segments, first, count, len;
};
// A team takes one whole segment each, and nothing is joined, where there are teams enough and no segment
// has many more tiles per warp than the warps' average share: kWholeTiles + 0.9 x the share more, at most
// kWholeMost. Joining costs what four tiles of a warp alone take, and more where the memory is busy. Measured
// (whole, split; us): 24 sequences with a window of 1024, 5 rows, 16 kv heads of 64: 19.7, 24.6; 48 of 777, 20
// rows, 8 kv heads of 128: 50, 90; 16 of 6000, 4 rows: 32, 41; one of 6000: 30, 16.7; 24 of 6000 on one kv head: 30,
// 19.5; 48 of 3000, 16 kv heads of 64: 66, 57; one of 777: 11.8, 14.4.
constexpr float kWholeTiles = 4.0f, kWholeMost = 9.0f;

struct Segment {
  int start;               // its first tile's place in the list (after the seg_cost places without a tile)
  int n;                   // its tiles
  int b, kh, rt;           // sequence, kv head, row tile
  int first, count, len;   // the sequence's queries and cached tokens
  int tile0;               // the sequence's first tile some query sees
};

// Waits for a copy that takes longer than a try; whatever happens, not without it.
__device__ __noinline__ void wait_for_copy(uint64_t* bar, uint32_t parity, uint64_t budget_ns) {
  if (!mbar_wait(bar, parity, budget_ns)) mbar_wait(bar, parity, kWaitBudgetNs);
}

// Row i of a segment's sums, divided and rounded: channels 8 (r + 8 set) + j and + 4 of query rows
// 2 q4 and 2 q4 + 1 of row tile nt, i = (nt SETS + set) 4 + j.
template <int D, int NG, int NT>
__device__ __forceinline__ void finish_row(const DecodeParams& p, const Segment& s, int i, int r, int q4, const float4& v,
                                           const float (&mm)[2], const float (&ll)[2], const float (&cc)[2][NG]) {
  constexpr int SETS = D / 64;
  const AttendParams& a = p.a;
  const int nt = i / (SETS * 4), set = i / 4 % SETS, j = i % 4;
  const float by = (j & 1) ? 1048576.0f : 16777216.0f;     // codes are c 2^-24, 16 c 2^-24 where j is odd
#pragma unroll
  for (int c = 0; c < 2; ++c) {
    const int row = s.rt * 8 * NT + nt * 8 + 2 * q4 + c;
    if (row >= s.count * a.share) continue;
    const float inv = ll[c] == 0.0f ? 0.0f : 1.0f / ll[c];
    const float add = NG == 1 || set == 0 ? cc[c][0] : cc[c][NG - 1];
    const float y0 = ((c ? v.y : v.x) * by + add) * inv, y1 = ((c ? v.w : v.z) * by + add) * inv;
    const long long at = static_cast<long long>(s.first + row / a.share) * a.heads + s.kh * a.share + row % a.share;
    const uint32_t both = p.bf16 ? pack2<__nv_bfloat16>(y0, y1) : pack2<__half>(y0, y1);
    uint16_t* o = static_cast<uint16_t*>(a.o) + at * D + 8 * (r + 8 * set) + j;
    o[0] = static_cast<uint16_t>(both);
    o[4] = static_cast<uint16_t>(both >> 16);
    if (a.lse && r == 0 && set == 0 && j == 0) a.lse[at] = ll[c] == 0.0f ? -INFINITY : (mm[c] + log2f(ll[c])) * kLn2;
  }
}

template <int D, int NG, int NT, int W, int TB>
__global__ void __launch_bounds__(W * 32, 1) kv4_decode_kernel(const DecodeParams p) {
  using SH = DecodeShape<D, NG, NT, W, TB>;
  constexpr int ROWS = 8 * NT, TT = TB * BLK, SETS = SH::SETS;
  constexpr int R4 = SH::R4, SMALL = SH::SMALL;
  extern __shared__ __align__(128) uint8_t smem[];
  uint8_t* ring = smem;
  float* smalls = reinterpret_cast<float*>(smem + SH::RING_BYTES);
  Sequence* seqs = reinterpret_cast<Sequence*>(smalls + W * SMALL);
  uint64_t* bars = reinterpret_cast<uint64_t*>((reinterpret_cast<uintptr_t>(seqs + MAX_SEQS) + 15) & ~static_cast<uintptr_t>(15));
  unsigned long long* scan = reinterpret_cast<unsigned long long*>(bars + 2 * W);
  int* flags = reinterpret_cast<int*>(scan);             // two per team, then each warp's stage with its sums
  int* ends = flags + 3 * W;                             // cu_q's ends

  const AttendParams& a = p.a;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int r = lane >> 2, q4 = lane & 3;

  if (lane == 0) {
    mbar_init(&bars[2 * warp], 1);
    mbar_init(&bars[2 * warp + 1], 1);
    mbar_fence_init();
  }

  // the first tile that some query of a sequence sees, how many there are, and its segments
  auto tile0_of = [&](int count, int len) { return sees_from(a, len - count) / TT; };
  auto tiles_of = [&](int count, int len) { return count ? max(0, (len + TT - 1) / TT - tile0_of(count, len)) : 0; };
  auto segments_of = [&](int count) { return a.cache.kv_heads * ((count * a.share + ROWS - 1) / ROWS); };

  const int TW = p.team_warps;
  // prefix sums of the sequences' tiles (low half) and segments (high half)
  unsigned long long sums = 0;
  for (int base = 0; base < a.seqs; base += W * 32) {
    const int b = base + threadIdx.x;
    Sequence q = {0, 0, 0, 0, 0};
    unsigned long long v = 0;
    if (b < a.seqs) {
      sequence(a, b, q.first, q.count, q.len);
      if (a.cu_q && b == 0) ends[0] = a.cu_q[0];
      if (a.cu_q && b == a.seqs - 1) ends[1] = a.cu_q[a.seqs];
      if (static_cast<long long>(q.count) * a.share > p.row_limit) q.count = 0;
      const int n = tiles_of(q.count, q.len);
      if (n) {
        const unsigned h = segments_of(q.count);
        v = (static_cast<unsigned long long>(h) << 32) | h * (n + p.seg_cost);
      }
    }
    unsigned long long inc = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const unsigned long long x = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += x;
    }
    if (base) __syncthreads();
    if (lane == 31) scan[warp] = inc;
    __syncthreads();
    unsigned long long before = sums + inc - v;
#pragma unroll
    for (int w = 0; w < W; ++w) {
      const unsigned long long x = scan[w];
      if (w < warp) before += x;
      sums += x;
    }
    q.prefix = static_cast<int>(before);
    q.segments = static_cast<int>(before >> 32);
    if (b < a.seqs) seqs[b] = q;
  }
  __syncthreads();
  const int total = static_cast<int>(sums), segments = static_cast<int>(sums >> 32);
  // whether every segment is one team's: team i then takes segment i
  bool direct = segments <= p.teams;
  if (direct) {
    const float share = static_cast<float>(total - segments * p.seg_cost) / (p.teams * TW);
    const int whole = static_cast<int>(TW * (share + fminf(kWholeTiles + 0.9f * share, kWholeMost)));
    bool longer = false;
    for (int b = threadIdx.x; b < a.seqs; b += W * 32) longer |= tiles_of(seqs[b].count, seqs[b].len) > whole;
    direct = !__syncthreads_or(longer);
  }

  const int team_in_cta = warp / TW, wt = warp % TW;
  const int team = blockIdx.x * (W / TW) + team_in_cta;
  auto team_sync = [&]() {
    if (TW == 1) __syncwarp();
    else asm volatile("bar.sync %0, %1;" ::"r"(1 + team_in_cta), "r"(TW * 32) : "memory");
  };

  // sequences without a tile: their queries see nothing
  for (int b = team; b < a.seqs; b += p.teams) {
    const Sequence q = seqs[b];
    if (q.count == 0 || tiles_of(q.count, q.len) != 0) continue;
    const long long rows = static_cast<long long>(q.count) * a.heads, at = static_cast<long long>(q.first) * a.heads;
    uint4* o = reinterpret_cast<uint4*>(static_cast<uint16_t*>(a.o) + at * D);
    for (long long i = wt * 32 + lane; i < rows * (D / 8); i += TW * 32) o[i] = make_uint4(0, 0, 0, 0);
    if (a.lse)
      for (long long i = wt * 32 + lane; i < rows; i += TW * 32) a.lse[at + i] = -INFINITY;
  }

  // queries of no sequence
  if (a.cu_q) {
    const int head = p.before ? min(max(ends[0], 0), a.T) : 0, tail = p.after ? max(ends[1], head) : a.T;
    const long long step = static_cast<long long>(gridDim.x) * W * 32, at = blockIdx.x * W * 32LL + threadIdx.x;
    auto nothing = [&](long long first, long long rows) {
      uint4* o = reinterpret_cast<uint4*>(static_cast<uint16_t*>(a.o) + first * a.heads * D);
      for (long long i = at; i < rows * a.heads * (D / 8); i += step) o[i] = make_uint4(0, 0, 0, 0);
      if (a.lse)
        for (long long i = at; i < rows * a.heads; i += step) a.lse[first * a.heads + i] = -INFINITY;
    };
    if (head > 0) nothing(0, head);
    if (tail < a.T) nothing(tail, a.T - tail);
  }

  // The team's share [t0, t1) of the list: no more teams than give each warp a tile; the first
  // `more` teams have one place more than the others.
  const int N = direct ? segments : min(p.teams, (total + TW - 1) / TW);
  if (team >= N) return;
  const int each = total / N, more = total - each * N;
  int t0 = team * each + min(team, more), t1 = t0 + each + (team < more ? 1 : 0);
  auto team_of = [&](int t) { return t < more * (each + 1) ? t / (each + 1) : more + (t - more * (each + 1)) / each; };

  auto locate = [&](int t) {
    int lo = 0, hi = a.seqs - 1;   // last b that begins at or before t: the one that holds t
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if ((direct ? seqs[mid].segments : seqs[mid].prefix) <= (direct ? team : t)) lo = mid; else hi = mid - 1;
    }
    const Sequence q = seqs[lo];
    Segment s;
    s.b = lo;
    s.first = q.first;
    s.count = q.count;
    s.len = q.len;
    s.tile0 = tile0_of(q.count, q.len);
    s.n = tiles_of(q.count, q.len);
    const int seg = direct ? team - q.segments : (t - q.prefix) / (s.n + p.seg_cost);
    s.rt = seg / a.cache.kv_heads;
    s.kh = seg - s.rt * a.cache.kv_heads;
    s.start = direct ? 0 : q.prefix + seg * (s.n + p.seg_cost) + p.seg_cost;
    return s;
  };
  if (direct) {
    t0 = 0;
    t1 = locate(0).n;
  }

  // ------------------------------ this warp's copies ------------------------------
  // A tile arrives with one copy where it lies in one page (`whole_tiles`), else block by block. The
  // sources of the next 32 copies are looked up together, one per lane; lane 0 issues them in turn.
  uint8_t* stages = ring + warp * 2 * SH::STAGE;
  uint64_t* bar = &bars[2 * warp];
  const bool whole_tiles = a.cache.page_blocks % TB == 0;
  const int per_tile = whole_tiles ? 1 : TB;
  int pt = t0 + wt;                    // the next tile to copy
  int pleft = 0, ptaken = 32;          // tiles of its segment left for this warp, and sources used
  int pblk = 0, plast = 0;             // its first block, and the sequence's blocks
  const int* prow = nullptr;           // the sequence's row of the table
  const uint8_t* phead = nullptr;      // its kv head in page 0
  unsigned long long psrc = 0;         // this lane's source (0: none)
  unsigned have = 0;                   // blocks of each stage that hold tokens, 8 bits a stage
  auto refill = [&]() {                // called with every lane, at a new segment or after 32 sources
    while (pleft == 0 && pt < t1) {    // on to the segment that holds pt, past places without a tile
      const Segment s = locate(pt);
      if (pt < s.start) {
        pt += (s.start - pt + TW - 1) / TW * TW;
        if (pt >= s.start + s.n) continue;
      }
      if (pt >= t1) break;
      pleft = (min(t1, s.start + s.n) - pt + TW - 1) / TW;
      pblk = (s.tile0 + pt - s.start) * TB;
      plast = (s.len + BLK - 1) / BLK;
      prow = a.table + static_cast<long long>(s.b) * a.width;
      phead = a.cache.pool + s.kh * a.cache.page_bytes;
    }
    ptaken = 0;
    psrc = 0;
    const int tile = lane / per_tile, blk = pblk + tile * TW * TB + lane % per_tile;
    if (tile < pleft && blk < plast) {
      const int col = a.cache.blocks.quotient(blk), page = prow[col];
      if (static_cast<unsigned>(page) < static_cast<unsigned>(a.cache.pages))
        psrc = reinterpret_cast<unsigned long long>(phead + page * (a.cache.kv_heads * a.cache.page_bytes) +
                                                    (blk - col * a.cache.page_blocks) * SH::BLOCK);
      else
        flag_error(kErrIndex);
    }
    __syncwarp();
  };
  auto issue = [&](int st) {           // copy the next tile into stage st
    if (pleft == 0 || ptaken + per_tile > 32) refill();
    if (pleft == 0) return;
    const int blocks = min(TB, plast - pblk);
    uint8_t* dst = stages + st * SH::STAGE;
    unsigned ok = 0;
    if (whole_tiles) {
      const unsigned long long src = __shfl_sync(0xffffffffu, psrc, ptaken);
      if (src) ok = (1u << blocks) - 1u;
      if (lane == 0) {
        mbar_arrive_expect_tx(&bar[st], src ? blocks * SH::BLOCK : 0);
        if (src) bulk_load(dst, reinterpret_cast<const void*>(src), blocks * SH::BLOCK, &bar[st]);
      }
    } else {
      ok = (__ballot_sync(0xffffffffu, psrc != 0) >> ptaken) & ((1u << TB) - 1u);
      if (lane == 0) mbar_arrive_expect_tx(&bar[st], __popc(ok) * SH::BLOCK);
#pragma unroll 1
      for (int j = 0; j < TB; ++j) {
        const unsigned long long src = __shfl_sync(0xffffffffu, psrc, ptaken + j);
        if (lane == 0 && src) bulk_load(dst + j * SH::BLOCK, reinterpret_cast<const void*>(src), SH::BLOCK, &bar[st]);
      }
    }
    have = st ? (have & 0xffu) | (ok << 8) : (have & 0xff00u) | ok;
    ptaken += per_tile;
    pblk += TW * TB;
    pt += TW;
    --pleft;
  };
  int stage = 0;
  uint32_t phases = 0;
  issue(0);

  // word of the token's codes that this lane's i-th fragment word is
  auto key_word = [&](int i) { return NG == 1 ? (D / 32) * q4 + i : (i < 2 ? 2 * q4 + i : 8 + 2 * q4 + i - 2); };
  constexpr int KW = D / 32;
  const bool odd = q4 & 1;
  const uint32_t sel_lo = odd ? 0x1054u : 0x5410u, sel_hi = odd ? 0x3276u : 0x7632u;

  bool parts = false;         // some piece was part of a segment
  for (int t = t0; t < t1;) {
    const Segment s = locate(t);
    if (t < s.start) {
      t = s.start;
      if (t >= t1) break;
    }
    const int end = min(t1, s.start + s.n);

    // ---- the rows' queries as B fragments, their sums, and what a score is scaled by
    uint32_t qf[NT][KW][4];
    float qs[NT][2][NG];
    float f[NT][2];                   // what a product is multiplied by, with the key's scale
    int to[NT][2], from[NT][2];       // tokens [from, to) that a row sees
    const float units = a.scale * kLog2e;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int row = s.rt * ROWS + nt * 8 + r;
      const bool live = row < s.count * a.share;
      const uint16_t* src = static_cast<const uint16_t*>(a.q);
      if (live) src += (s.first + row / a.share) * a.q_st + (s.kh * a.share + row % a.share) * a.q_sh;
      float x[KW][8], sum[NG], top = 0.0f;
#pragma unroll
      for (int i = 0; i < NG; ++i) sum[i] = 0.0f;
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
      for (int o = 1; o < 4; o <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
      // 2^e <= top < 2^(e+1), kept where the powers of two below are normal (an infinity stays one)
      const int e2 = min(max(static_cast<int>(__float_as_uint(top) >> 23) - 127, -112), 127);
      const float down = __uint_as_float(static_cast<uint32_t>(127 + 14 - e2) << 23);
      const float row_f = units * 1024.0f * __uint_as_float(static_cast<uint32_t>(127 + e2) << 23);   // 2^24 2^(e - 14)
#pragma unroll
      for (int i = 0; i < KW; ++i)
        // fragment words: nibbles (0, 4), (1, 5) / 16, (2, 6), (3, 7) / 16 of word key_word(i)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float by = (j & 1) ? down * 0.0625f : down;
          const __half2 h = __floats2half2_rn(x[i][j] * by, x[i][j + 4] * by);
          qf[nt][i][j] = *reinterpret_cast<const uint32_t*>(&h);
        }
#pragma unroll
      for (int i = 0; i < NG; ++i) {
        sum[i] += __shfl_xor_sync(0xffffffffu, sum[i], 1);
        sum[i] += __shfl_xor_sync(0xffffffffu, sum[i], 2);
      }
      const int pos = s.len - s.count + row / a.share;
#pragma unroll
      for (int c = 0; c < 2; ++c) {   // accumulators hold rows 2 q4 and 2 q4 + 1
        const int src_lane = 4 * (2 * q4 + c);
#pragma unroll
        for (int i = 0; i < NG; ++i) qs[nt][c][i] = __shfl_sync(0xffffffffu, sum[i] * units, src_lane);
        f[nt][c] = __shfl_sync(0xffffffffu, row_f, src_lane);
        // a row past the last sees everything, so that it makes no tile an edge
        to[nt][c] = __shfl_sync(0xffffffffu, live ? min(s.len, pos + 1) : s.len, src_lane);
        from[nt][c] = __shfl_sync(0xffffffffu, live ? sees_from(a, pos) : 0, src_lane);
      }
    }
    // tokens that some row of the tile sees
    const int last_row = min((s.rt + 1) * ROWS, s.count * a.share) - 1, pos0 = s.len - s.count;
    const int any_to = min(s.len, pos0 + last_row / a.share + 1);
    const int any_from = sees_from(a, pos0 + s.rt * ROWS / a.share);
    int all_from = 0, all_to = 0x7fffffff;   // tokens that every row of this warp's tile sees
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        all_from = max(all_from, from[nt][c]);
        all_to = min(all_to, to[nt][c]);
      }
#pragma unroll
    for (int o = 1; o < 4; o <<= 1) {
      all_from = max(all_from, __shfl_xor_sync(0xffffffffu, all_from, o));
      all_to = min(all_to, __shfl_xor_sync(0xffffffffu, all_to, o));
    }

    float acc[NT][SETS * 4][4] = {}, hsum[NT][NG][4] = {};
    float m[NT][2], l[NT][2], corr[NT][2][NG];
    float vs = kMostScale / 8;                 // what the values' scales are multiplied by,
    uint32_t vs_for = 0x4800;                  // up to this one (fp16: 8)
    unsigned fresh = (1u << (2 * NT)) - 1u;    // rows that have seen no token yet (their m is 0 until then)
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        m[nt][c] = 0.0f;
        l[nt][c] = 0.0f;
#pragma unroll
        for (int i = 0; i < NG; ++i) corr[nt][c][i] = 0.0f;
      }

    // this warp's tiles of the piece: those at t0 + wt + k TW
    int g = t - s.start + ((wt - (t - t0)) & (TW - 1));
    const int stop = end - s.start;
    // tiles [inside_lo, inside_hi) of the segment lie within what every row sees
    const int inside_lo = (all_from + TT - 1) / TT - s.tile0, inside_hi = all_to / TT - s.tile0;
    const uint32_t lane_k = (NG == 1 && KW == 4) ? r * (D / 2) + 16 * q4 : r * (D / 2);
    const uint32_t lane_va = value_codes_at(D) + (2 * q4 + (odd ? 1 : 0)) * (D / 2) + 4 * r;
    const uint32_t lane_vb = value_codes_at(D) + (2 * q4 + (odd ? 0 : 1)) * (D / 2) + 4 * r;

    // One tile. EDGE: some row may not see some token of it.
    auto step = [&](auto edge_tag, const uint8_t* tile, unsigned blocks, int tok0) {
      constexpr bool EDGE = decltype(edge_tag)::value;
      // ---- scores over the running maximum, log2 units
      float y[TB][NT][4];
#pragma unroll
      for (int k = 0; k < TB; ++k) {
        const uint8_t* blk = tile + k * SH::BLOCK;
        uint32_t w0[KW], w1[KW];       // this lane's words of tokens r and r + 8
        if constexpr (NG == 1 && KW == 4) {
          *reinterpret_cast<uint4*>(w0) = *reinterpret_cast<const uint4*>(blk + lane_k);
          *reinterpret_cast<uint4*>(w1) = *reinterpret_cast<const uint4*>(blk + lane_k + 4 * D);
        } else {
#pragma unroll
          for (int i = 0; i < KW; i += 2) {
            *reinterpret_cast<uint2*>(w0 + i) = *reinterpret_cast<const uint2*>(blk + lane_k + 4 * key_word(i));
            *reinterpret_cast<uint2*>(w1 + i) = *reinterpret_cast<const uint2*>(blk + lane_k + 4 * D + 4 * key_word(i));
          }
        }
        const uint32_t* pairs = reinterpret_cast<const uint32_t*>(blk + key_pairs_at(D));
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int c = 0; c < 4; ++c) y[k][nt][c] = -m[nt][c & 1];
#pragma unroll
        for (int gr = 0; gr < NG; ++gr) {
          float d[NT][4];
#pragma unroll
          for (int i = gr * (KW / NG); i < (gr + 1) * (KW / NG); ++i) {
            const uint32_t u0 = w0[i] >> 8, u1 = w1[i] >> 8;
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
              if (i == gr * (KW / NG))
                mma16816_first(d[nt], w0[i] & 0x000f000fu, w1[i] & 0x000f000fu, w0[i] & 0x00f000f0u, w1[i] & 0x00f000f0u,
                               qf[nt][i][0], qf[nt][i][1]);
              else
                mma16816(d[nt], w0[i] & 0x000f000fu, w1[i] & 0x000f000fu, w0[i] & 0x00f000f0u, w1[i] & 0x00f000f0u,
                         qf[nt][i][0], qf[nt][i][1]);
              mma16816(d[nt], u0 & 0x000f000fu, u1 & 0x000f000fu, u0 & 0x00f000f0u, u1 & 0x00f000f0u, qf[nt][i][2],
                       qf[nt][i][3]);
            }
          }
          const float2 pr0 = __half22float2(*reinterpret_cast<const __half2*>(&pairs[r * NG + gr]));
          const float2 pr1 = __half22float2(*reinterpret_cast<const __half2*>(&pairs[(r + 8) * NG + gr]));
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int c = 0; c < 4; ++c)
              y[k][nt][c] = fmaf(d[nt][c], (c < 2 ? pr0.x : pr1.x) * f[nt][c & 1],
                                 fmaf(c < 2 ? pr0.y : pr1.y, qs[nt][c & 1][gr], y[k][nt][c]));
        }
      }
      if constexpr (EDGE) {
#pragma unroll
        for (int k = 0; k < TB; ++k)
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int c = 0; c < 4; ++c) {
              const int tok = tok0 + k * BLK + r + (c < 2 ? 0 : 8);
              if (!((blocks >> k) & 1u) || tok < from[nt][c & 1] || tok >= to[nt][c & 1]) y[k][nt][c] = -INFINITY;
            }
      }

      // ---- the values' scales, a token and group per lane at a time: is one too large, or perhaps no scale
      constexpr int SCALES = TT * NG / 32;
      auto pair_of = [&](int i) {
        const int at = i * 32 + lane;
        return tile + at / (BLK * NG) * SH::BLOCK + value_pairs_at(D, NG) + at % (BLK * NG) * 4;
      };
      bool look = false;
#pragma unroll
      for (int i = 0; i < SCALES; ++i) {
        const uint32_t sc = *reinterpret_cast<const uint16_t*>(pair_of(i)) & 0x7fffu;
        look |= sc > vs_for || sc == 0x3c00u;
      }

      // ---- running maximum
      float top_y[NT][2];
      bool grows = fresh != 0 || look;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          float v = fmaxf(y[0][nt][c], y[0][nt][c + 2]);
#pragma unroll
          for (int k = 1; k < TB; ++k) v = fmaxf(v, fmaxf(y[k][nt][c], y[k][nt][c + 2]));
          top_y[nt][c] = v;
          grows |= v > kLazyMax;
        }
      if (__any_sync(0xffffffffu, grows)) {
        if (__any_sync(0xffffffffu, look)) {
          uint32_t most = 0;
#pragma unroll 1
          for (int i = 0; i < SCALES; ++i) {
            const int at = i * 32 + lane, k = at / (BLK * NG), tok = tok0 + at / NG;
            uint16_t* pair = const_cast<uint16_t*>(reinterpret_cast<const uint16_t*>(pair_of(i)));
            uint32_t sc = *pair & 0x7fffu;
            if (sc == 0x3c00u) {
              const uint4* codes = reinterpret_cast<const uint4*>(tile + k * SH::BLOCK + value_codes_at(D) +
                                                                  at % (BLK * NG) * (D / 2 / NG));
              uint32_t any = 0;
#pragma unroll
              for (int j = 0; j < D / 32 / NG; ++j) any |= codes[j].x | codes[j].y | codes[j].z | codes[j].w;
              if (any == 0) {
                *pair = 0;
                fence_proxy_async_smem();      // the stage is copied into again
                sc = 0;
              }
            }
            // (tokens that no row sees, and scales that are not finite, have no say)
            const bool seen = !EDGE || (((blocks >> k) & 1u) && tok >= any_from && tok < any_to);
            if (seen && sc < 0x7c00u) most = max(most, sc);
          }
          most = __reduce_max_sync(0xffffffffu, most);
          if (most > vs_for) {
            const int e = static_cast<int>(most >> 10) - 15;       // most < 2^(e + 1)
            vs_for = (most & 0x7c00u) + 0x400u;
            const float to = __uint_as_float(static_cast<uint32_t>(127 + 12 - e) << 23);
            const float by = to / vs;
            vs = to;
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
              for (int c = 0; c < 4; ++c) {
#pragma unroll
                for (int i = 0; i < NG; ++i) hsum[nt][i][c] *= by;
#pragma unroll
                for (int i = 0; i < SETS * 4; ++i) acc[nt][i][c] *= by;
              }
          }
          __syncwarp();
        }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            float v = top_y[nt][c];
#pragma unroll
            for (int o = 4; o < 32; o <<= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
            const unsigned bit = 1u << (2 * nt + c);
            const bool first = (fresh & bit) != 0;
            const float up = v > (first ? -INFINITY : kLazyMax) ? v : 0.0f;
            const float by = first ? 1.0f : ex2(-up);      // nothing to scale yet
            if (v > -INFINITY) fresh &= ~bit;
            m[nt][c] += up;
            l[nt][c] *= by;
#pragma unroll
            for (int k = 0; k < TB; ++k) {
              y[k][nt][c] -= up;
              y[k][nt][c + 2] -= up;
            }
#pragma unroll
            for (int i = 0; i < NG; ++i) {
              corr[nt][c][i] *= by;
              hsum[nt][i][c] *= by;
            }
#pragma unroll
            for (int i = 0; i < SETS * 4; ++i) {
              acc[nt][i][c] *= by;
              acc[nt][i][c + 2] *= by;
            }
          }
      }

      // ---- probabilities and the second product
#pragma unroll
      for (int k = 0; k < TB; ++k) {
        const uint8_t* blk = tile + k * SH::BLOCK;
        const uint32_t* pairs = reinterpret_cast<const uint32_t*>(blk + value_pairs_at(D, NG));
        uint32_t b[NT][NG][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            // (minus zero: not seen. The weight of a token that is seen may vanish, but a NaN of it does not)
            y[k][nt][c] = EDGE && y[k][nt][c] == -INFINITY ? -0.0f : ex2(y[k][nt][c]);
            l[nt][c & 1] += y[k][nt][c];
          }
#pragma unroll
        for (int gr = 0; gr < NG; ++gr) {
          const float2 pr0 = __half22float2(*reinterpret_cast<const __half2*>(&pairs[r * NG + gr]));
          const float2 pr1 = __half22float2(*reinterpret_cast<const __half2*>(&pairs[(r + 8) * NG + gr]));
          const float o0 = fmaf(7.5f, pr0.x, pr0.y), o1 = fmaf(7.5f, pr1.x, pr1.y);
          const float sv0 = pr0.x * vs, sv1 = pr1.x * vs;
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            float ps[4];
            if constexpr (EDGE) {            // a token that is not seen may have any pair, NaN too
#pragma unroll
              for (int c = 0; c < 4; ++c) {
                const float pv = y[k][nt][c];
                const bool seen = __float_as_uint(pv) != 0x80000000u;
                ps[c] = seen ? pv * (c < 2 ? sv0 : sv1) : 0.0f;
                if (seen) corr[nt][c & 1][gr] = fmaf(pv, c < 2 ? o0 : o1, corr[nt][c & 1][gr]);
              }
            } else {
#pragma unroll
              for (int c = 0; c < 4; ++c) {
                ps[c] = y[k][nt][c] * (c < 2 ? sv0 : sv1);
                corr[nt][c & 1][gr] = fmaf(y[k][nt][c], c < 2 ? o0 : o1, corr[nt][c & 1][gr]);
              }
            }
            b[nt][gr][0] = movmatrix_trans(pack2<__half>(ps[0], ps[1]));
            b[nt][gr][1] = movmatrix_trans(pack2<__half>(ps[2], ps[3]));
            mma16816(hsum[nt][gr], 0x3c003c00u, 0x3c003c00u, 0x3c003c00u, 0x3c003c00u, b[nt][gr][0], b[nt][gr][1]);
          }
        }
        // channels: set s of this lane's row r is word r + 8 s, nibble j (rows 0-7) and j + 4 (rows 8-15).
        // Odd q4 load the second token of their pair first, so a load's lanes cover both halves of
        // the banks (rows of 16 words).
#pragma unroll
        for (int s2 = 0; s2 < SETS; ++s2) {
          const uint32_t wa = *reinterpret_cast<const uint32_t*>(blk + lane_va + 32 * s2);
          const uint32_t wb = *reinterpret_cast<const uint32_t*>(blk + lane_vb + 32 * s2);
          const uint32_t wc = *reinterpret_cast<const uint32_t*>(blk + lane_va + 4 * D + 32 * s2);
          const uint32_t wd = *reinterpret_cast<const uint32_t*>(blk + lane_vb + 4 * D + 32 * s2);
          const uint32_t v[4] = {prmt(wa, wb, sel_lo), prmt(wa, wb, sel_hi), prmt(wc, wd, sel_lo), prmt(wc, wd, sel_hi)};
          const uint32_t z[4] = {v[0] >> 8, v[1] >> 8, v[2] >> 8, v[3] >> 8};
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            const uint32_t* bb = b[nt][NG == 1 ? 0 : s2];
            mma16816(acc[nt][4 * s2], v[0] & 0x000f000fu, v[1] & 0x000f000fu, v[2] & 0x000f000fu, v[3] & 0x000f000fu, bb[0], bb[1]);
            mma16816(acc[nt][4 * s2 + 1], v[0] & 0x00f000f0u, v[1] & 0x00f000f0u, v[2] & 0x00f000f0u, v[3] & 0x00f000f0u, bb[0], bb[1]);
            mma16816(acc[nt][4 * s2 + 2], z[0] & 0x000f000fu, z[1] & 0x000f000fu, z[2] & 0x000f000fu, z[3] & 0x000f000fu, bb[0], bb[1]);
            mma16816(acc[nt][4 * s2 + 3], z[0] & 0x00f000f0u, z[1] & 0x00f000f0u, z[2] & 0x00f000f0u, z[3] & 0x00f000f0u, bb[0], bb[1]);
          }
        }
      }
    };
    for (; g < stop; g += TW) {
      const unsigned blocks = (stage ? have >> 8 : have) & 0xffu;
      issue(stage ^ 1);
      if (!mbar_try_wait(&bar[stage], (phases >> stage) & 1u)) wait_for_copy(&bar[stage], (phases >> stage) & 1u, p.wait_ns);
      phases ^= 1u << stage;
      const uint8_t* tile = stages + stage * SH::STAGE;
      if (blocks == (1u << TB) - 1u && g >= inside_lo && g < inside_hi)
        step(std::false_type(), tile, blocks, 0);
      else
        step(std::true_type(), tile, blocks, (s.tile0 + g) * TT);
      __syncwarp();
      stage ^= 1;
    }

    // ---- this warp's sums over its lanes of tokens
    const float back = 1.0f / vs;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int c = 0; c < 2; ++c)
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) {
          l[nt][c] += __shfl_xor_sync(0xffffffffu, l[nt][c], o);
#pragma unroll
          for (int i = 0; i < NG; ++i) corr[nt][c][i] += __shfl_xor_sync(0xffffffffu, corr[nt][c][i], o);
        }
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        if ((fresh >> (2 * nt + c)) & 1u) m[nt][c] = kNoMax;
#pragma unroll
        for (int i = 0; i < NG; ++i) corr[nt][c][i] = fmaf(-7.5f * back, hsum[nt][i][c], corr[nt][c][i]);
      }

    // ---- the warp's sums into the stage it has just read, the rest beside
    {
      float4* sums = reinterpret_cast<float4*>(stages + (stage ^ 1) * SH::STAGE) + lane;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
        for (int i = 0; i < SETS * 4; ++i)
          sums[(nt * SETS * 4 + i) * 32] = make_float4(acc[nt][i][0] * back, acc[nt][i][1] * back, acc[nt][i][2] * back, acc[nt][i][3] * back);
        if (r == 0) {
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            float* e = smalls + warp * SMALL + (nt * 8 + 2 * q4 + c) * (2 + NG);
            e[0] = m[nt][c];
            e[1] = l[nt][c];
#pragma unroll
            for (int i = 0; i < NG; ++i) e[2 + i] = corr[nt][c][i];
          }
        }
      }
      if (lane == 0) flags[2 * W + warp] = stage ^ 1;
    }
    team_sync();
    // ---- row i of the sums over the team's warps: finished, or left as a part
    const bool whole = end - t == s.n;
    parts |= !whole;
    float* part = p.parts + (2 * team + (t0 >= s.start ? 0 : 1)) * static_cast<long long>(SH::PART);
    for (int i = wt; i < R4; i += TW) {
      const int col = i / (SETS * 4) * 8 + 2 * q4;
      const float* e = smalls + team_in_cta * TW * SMALL + col * (2 + NG);
      float mm[2] = {kNoMax, kNoMax}, ll[2] = {0.0f, 0.0f}, cc[2][NG] = {};
      for (int w = 0; w < TW; ++w) {
        mm[0] = fmaxf(mm[0], e[w * SMALL]);
        mm[1] = fmaxf(mm[1], e[w * SMALL + 2 + NG]);
      }
      float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      for (int w = 0; w < TW; ++w) {
        float by[2];
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const float* ec = e + w * SMALL + c * (2 + NG);
          by[c] = ex2(ec[0] - mm[c]);
          ll[c] = fmaf(by[c], ec[1], ll[c]);
#pragma unroll
          for (int k = 0; k < NG; ++k) cc[c][k] = fmaf(by[c], ec[2 + k], cc[c][k]);
        }
        const int from_warp = team_in_cta * TW + w;
        const float4 x = *(reinterpret_cast<const float4*>(ring + (2 * from_warp + flags[2 * W + from_warp]) * SH::STAGE) + i * 32 + lane);
        v.x = fmaf(by[0], x.x, v.x);
        v.y = fmaf(by[1], x.y, v.y);
        v.z = fmaf(by[0], x.z, v.z);
        v.w = fmaf(by[1], x.w, v.w);
      }
      if (whole) {
        finish_row<D, NG, NT>(p, s, i, r, q4, v, mm, ll, cc);
      } else {
        reinterpret_cast<float4*>(part)[i * 32 + lane] = v;
        if (i % (SETS * 4) == 0 && r == 0) {
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            float* ec = part + R4 * 128 + (col + c) * (2 + NG);
            ec[0] = mm[c];
            ec[1] = ll[c];
#pragma unroll
            for (int k = 0; k < NG; ++k) ec[2 + k] = cc[c][k];
          }
        }
      }
    }
    fence_proxy_async_smem();   // the stages are copied into again
    team_sync();
    t = end;
  }

  // ---- parts: the segment the team starts in, and the one it ends in
  auto shared_segment = [&](int k, Segment& s) {
    s = locate(k ? t1 - 1 : t0);
    if (k ? s.start <= t0 || s.start >= t1 : s.start > t0) return false;
    return s.start < t0 || s.start + s.n > t1;
  };
  if (!parts) return;
  {
    __threadfence();
    team_sync();
    if (wt == 0 && lane < 2) {
      Segment s;
      int last = 0;
      if (shared_segment(lane, s)) {
        const int first = team_of(s.start), all = team_of(s.start + s.n - 1) - first;
        last = atomicAdd(p.counters + first, 1) == all;
        if (last) p.counters[first] = 0;     // every team has arrived: left zero for the next launch
      }
      flags[2 * team_in_cta + lane] = last;
    }
    team_sync();
  }
  for (int k = 0; k < 2; ++k) {
    if (!flags[2 * team_in_cta + k]) continue;
    __threadfence();
    Segment s;
    shared_segment(k, s);
    const int first = team_of(s.start), count = team_of(s.start + s.n - 1) - first + 1;
    const int first_t0 = first * each + min(first, more);
    // the first team's part is its second unless its own share starts at the segment's
    const float* part0 = p.parts + (2 * first + (first_t0 >= s.start ? 0 : 1)) * static_cast<long long>(SH::PART);
    const float* rest = p.parts + 2 * first * static_cast<long long>(SH::PART);
    // RUN rows at a time, which share the query rows' m, l and corr; the maximum runs along, so that
    // all loads of four parts are in flight together
    constexpr int RUN = 4;
    const int rows = max(1, R4 / TW);
    for (int i0 = wt * rows; i0 < min(R4, (wt + 1) * rows); i0 += RUN) {
      const int col = i0 / (SETS * 4) * 8 + 2 * q4, n = min(RUN, rows);
      float mm[2] = {kNoMax, kNoMax}, ll[2] = {0.0f, 0.0f}, cc[2][NG] = {};
      float4 v[RUN];
#pragma unroll
      for (int j = 0; j < RUN; ++j) v[j] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 4
      for (int w = 0; w < count; ++w) {
        const float* base = w ? rest + 2 * w * static_cast<long long>(SH::PART) : part0;
        const float* e = base + R4 * 128 + col * (2 + NG);
        float4 x[RUN];
#pragma unroll
        for (int j = 0; j < RUN; ++j)
          x[j] = j < n ? __ldcg(reinterpret_cast<const float4*>(base) + (i0 + j) * 32 + lane) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        float mine[2], theirs[2];
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const float* ec = e + c * (2 + NG);
          const float mo = __ldcg(ec), mn = fmaxf(mm[c], mo);
          mine[c] = ex2(mm[c] - mn);
          theirs[c] = ex2(mo - mn);
          mm[c] = mn;
          ll[c] = fmaf(theirs[c], __ldcg(ec + 1), ll[c] * mine[c]);
#pragma unroll
          for (int j = 0; j < NG; ++j) cc[c][j] = fmaf(theirs[c], __ldcg(ec + 2 + j), cc[c][j] * mine[c]);
        }
#pragma unroll
        for (int j = 0; j < RUN; ++j) {
          v[j].x = fmaf(theirs[0], x[j].x, v[j].x * mine[0]);
          v[j].y = fmaf(theirs[1], x[j].y, v[j].y * mine[1]);
          v[j].z = fmaf(theirs[0], x[j].z, v[j].z * mine[0]);
          v[j].w = fmaf(theirs[1], x[j].w, v[j].w * mine[1]);
        }
      }
#pragma unroll
      for (int j = 0; j < RUN; ++j)
        if (j < n) finish_row<D, NG, NT>(p, s, i0 + j, r, q4, v[j], mm, ll, cc);
    }
  }
}

}  // namespace kv4
}  // namespace w4a16
