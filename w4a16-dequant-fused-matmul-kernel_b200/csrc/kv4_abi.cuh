// kv4_abi.cuh -- the C entry points of the 4-bit paged cache, its attention and the query/key
// preparation: argument checks and launches. Included once, by w4a16_b200.cu.
#pragma once

#include "kv4_evict.cuh"
#include "kv4_prefill.cuh"
#include "kv4_pages.cuh"
#include "kv4_rope.cuh"
#include "kv4_weights.cuh"

namespace w4a16 {
namespace kv4 {
namespace {

// The checks every entry point makes of a cache; those that need no device, and all.
int check_cache(const w4a16_kv4_cache* c) {
  if (c == nullptr || c->layers < 1 || c->layers > 0x7fffffffLL || c->pages < 1 || c->pages > 0x7fffffffLL || c->kv_heads < 1 ||
      c->kv_heads > 65535 || (c->head_dim != 64 && c->head_dim != 128) || c->page_size < BLK ||
      c->page_size % BLK != 0 || c->page_size > 4096 || c->pages * c->page_size > 0xffffffffLL || (c->group_size != 64 && c->group_size != c->head_dim))
    return W4A16_ERR_INVALID;
  if (c->pool == nullptr) return W4A16_ERR_INVALID;
  if (!aligned16(c->pool)) return W4A16_ERR_ALIGNMENT;
  return W4A16_OK;
}
int check_cache(const w4a16_kv4_cache* c, DeviceState** dev) {
  const int st = check_cache(c);
  return st != W4A16_OK ? st : current_device_state(dev);
}

// Collected weights as they lie in memory: up to three axes of n entries at a stride, each entry `tokens` floats.
struct WeightsAxis {
  long long n, stride;
};
struct WeightsMemory {
  const float* at;
  WeightsAxis given[3], axes[3];   // those of more than one entry: as they came, and from the largest stride down
  int count = 0;
  long long tokens;
  __int128 low = 0, high;    // floats from `at`: the first, and the one behind the last

  WeightsMemory(const float* p, std::initializer_list<WeightsAxis> all, long long tokens_) : at(p), tokens(tokens_), high(tokens_) {
    for (const WeightsAxis& a : all) {
      if (a.n <= 0) tokens = 0;          // nothing at all
      if (a.n <= 1) continue;
      given[count] = a;
      int i = count++;
      for (; i > 0 && magnitude(axes[i - 1].stride) < magnitude(a.stride); --i) axes[i] = axes[i - 1];
      axes[i] = a;
      (a.stride < 0 ? low : high) += static_cast<__int128>(a.n - 1) * a.stride;
    }
  }
  static __int128 magnitude(__int128 x) { return x < 0 ? -x : x; }
  // Whether each entry of an axis holds all of the axes below it without reaching the next.
  bool nested() const {
    __int128 extent = tokens;
    for (int i = count - 1; i >= 0; --i) {
      if (magnitude(axes[i].stride) < extent) return false;
      extent += magnitude(axes[i].stride) * (axes[i].n - 1);
    }
    return true;
  }
  // Whether entries that lie `by` floats apart, and at any two places of the axes from i on, share some (nested ones).
  bool meets(int i, __int128 by) const {
    if (i == count) return magnitude(by) < tokens;
    const __int128 s = magnitude(axes[i].stride);
    const __int128 k = by / s - (by % s < 0);             // rounded down: only this one and the next come near enough
    for (int next = 0; next < 2; ++next)
      if (magnitude(k + next) < axes[i].n && meets(i + 1, by - (k + next) * s)) return true;
    return false;
  }
};

// Whether `to` can be written while `from` is read: no two entries of `to` share memory, and none of them
// with another's of `from` (they are the same, or apart).
bool can_write(const WeightsMemory& from, const WeightsMemory& to) {
  if (to.tokens <= 0) return true;       // (fewer than none are refused elsewhere)
  if (!to.nested()) return false;
  bool same = from.count == to.count, alike = same;
  for (int i = 0; i < std::min(from.count, to.count); ++i) {
    same = same && from.given[i].stride == to.given[i].stride;
    alike = alike && from.axes[i].n == to.axes[i].n && from.axes[i].stride == to.axes[i].stride;
  }
  const __int128 bytes = static_cast<__int128>(reinterpret_cast<uintptr_t>(to.at)) - static_cast<__int128>(reinterpret_cast<uintptr_t>(from.at));
  if (bytes == 0) return same;
  if (bytes + 4 * to.low >= 4 * from.high || bytes + 4 * to.high <= 4 * from.low) return true;
  return alike && bytes % 4 == 0 && !to.meets(0, bytes / 4);
}

CacheView view_of(const w4a16_kv4_cache& c, int64_t layer) {
  CacheView v;
  v.pages = c.pages;
  v.kv_heads = c.kv_heads;
  v.page_size = c.page_size;
  v.page_blocks = c.page_size / BLK;
  v.blocks = Divisor(v.page_blocks);
  v.block_bytes = block_bytes(c.head_dim, c.head_dim / c.group_size);
  v.page_bytes = static_cast<long long>(v.page_blocks) * v.block_bytes;
  v.pool = static_cast<uint8_t*>(c.pool) + layer * c.pages * c.kv_heads * v.page_bytes;
  return v;
}

int launched() {
  if (cudaGetLastError() != cudaSuccess) return W4A16_ERR_LAUNCH;
  return W4A16_OK;
}

// A launch that may begin before the kernel before it in the stream has ended: the kernel waits for that itself
// (after_launch_before). Blocks in clusters of `cluster`.
template <typename P>
int launch_after(void (*kernel)(P), unsigned grid, unsigned block, int bytes, int cluster, cudaStream_t s, const P& p) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(block);
  cfg.dynamicSmemBytes = bytes;
  cfg.stream = s;
  cudaLaunchAttribute attr[2] = {};
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = cluster;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  if (cudaLaunchKernelEx(&cfg, kernel, p) != cudaSuccess) {
    cudaGetLastError();
    return W4A16_ERR_LAUNCH;
  }
  return W4A16_OK;
}

// What routing and workspace go by: nothing that lies in device memory.
struct AttendPlan {
  long long seqs;
  int kv_heads;
  long long rows;          // most query rows of a sequence's kv head
};

struct RopeArgs {
  const void *q, *k, *v;
  int dtype;
  int64_t T;
  int heads, kv_heads, head_dim;
  int64_t q_st, q_sh, k_st, k_sh, v_st, v_sh;
  const int64_t* positions;
  int axes, end0, end1;
  const float* cos_sin;
  int64_t max_pos;
  int rot, interleaved;
  const void *qw, *kw;
  int w_dtype;
  float eps;
};

template <typename T, bool APPEND>
void launch_rope(const RopeParams& p, int head_dim, cudaStream_t s) {
  const long long lanes = p.T * p.chunks * (head_dim / 8);
  const unsigned grid = static_cast<unsigned>((lanes + ROPE_THREADS - 1) / ROPE_THREADS);
  if (head_dim == 128)
    qk_norm_rope_kernel<T, 128, APPEND><<<grid, ROPE_THREADS, 0, s>>>(p);
  else
    qk_norm_rope_kernel<T, 64, APPEND><<<grid, ROPE_THREADS, 0, s>>>(p);
}

int rope(const RopeArgs& a, void* q_out, void* k_out, const w4a16_kv4_cache* cache, int64_t layer,
         const int64_t* slots, void* stream) {
  const bool append = cache != nullptr;
  if (a.T < 0 || a.T > 0x7fffffffLL || a.heads < 0 || a.kv_heads < 0 || a.heads > 65535 || a.kv_heads > 65535 ||
      (a.head_dim != 64 && a.head_dim != 128) || (a.dtype != W4A16_DTYPE_F16 && a.dtype != W4A16_DTYPE_BF16) ||
      a.rot < 0 || a.rot > a.head_dim || a.rot % 8 != 0 || (a.axes != 1 && a.axes != 3) || a.max_pos < 1 ||
      !(a.eps >= 0.0f) || (a.w_dtype != a.dtype && a.w_dtype != W4A16_DTYPE_F32))
    return W4A16_ERR_INVALID;
  if (a.axes == 3 && (a.end0 < 0 || a.end1 < a.end0 || a.end1 > a.rot / 2)) return W4A16_ERR_INVALID;
  DeviceState* dev = nullptr;
  RopeParams p = {};
  if (append) {
    const int st = check_cache(cache, &dev);
    if (st != W4A16_OK) return st;
    if (layer < 0 || layer >= cache->layers || cache->kv_heads != a.kv_heads || cache->head_dim != a.head_dim)
      return W4A16_ERR_INVALID;
    p.cache = view_of(*cache, layer);
    p.groups = cache->head_dim / cache->group_size;
  } else {
    const int st = current_device_state(&dev);
    if (st != W4A16_OK) return st;
  }
  const int items = a.heads + (append ? 2 : 1) * a.kv_heads;
  if (a.T == 0 || items == 0) return W4A16_OK;
  if ((a.heads && (a.q == nullptr || q_out == nullptr)) || (a.kv_heads && a.k == nullptr) ||
      (a.kv_heads && !append && k_out == nullptr) || (append && (a.v == nullptr || slots == nullptr)) ||
      (a.rot && (a.positions == nullptr || a.cos_sin == nullptr)))
    return W4A16_ERR_INVALID;
  if (!aligned16(q_out) || (!append && !aligned16(k_out)) || !aligned16(a.cos_sin)) return W4A16_ERR_ALIGNMENT;
  p.q = a.q; p.k = a.k; p.v = a.v;
  p.q_st = a.q_st; p.q_sh = a.q_sh; p.k_st = a.k_st; p.k_sh = a.k_sh; p.v_st = a.v_st; p.v_sh = a.v_sh;
  p.q_out = q_out; p.k_out = k_out;
  p.T = a.T;
  p.heads = a.heads; p.kv_heads = a.kv_heads;
  p.q_chunks = (a.heads + UN - 1) / UN;
  p.k_chunks = (a.kv_heads + UN - 1) / UN;
  p.chunks = p.q_chunks + (append ? 2 : 1) * p.k_chunks;
  p.by_chunks = Divisor(p.chunks);
  p.positions = reinterpret_cast<const long long*>(a.positions);
  p.axes = a.axes; p.end0 = a.end0; p.end1 = a.end1;
  p.cos_sin = a.cos_sin;
  p.max_pos = a.max_pos;
  p.rot = a.rot;
  p.interleaved = a.interleaved;
  p.qw = a.qw; p.kw = a.kw;
  p.w_f32 = a.w_dtype == W4A16_DTYPE_F32;
  p.eps = a.eps;
  p.slots = reinterpret_cast<const long long*>(slots);
  auto quads = [](const void* x, int64_t st, int64_t sh) {
    return reinterpret_cast<uintptr_t>(x) % 8 == 0 && st % 4 == 0 && sh % 4 == 0;
  };
  p.vec = quads(a.q, a.q_st, a.q_sh) && quads(a.k, a.k_st, a.k_sh) && (!append || quads(a.v, a.v_st, a.v_sh));
  p.w_vec = reinterpret_cast<uintptr_t>(a.qw) % 8 == 0 && reinterpret_cast<uintptr_t>(a.kw) % 8 == 0;
  if (p.T * p.chunks > 0x7fffffffLL) return W4A16_ERR_INVALID;   // the kernel counts groups in 32 bits
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (a.dtype == W4A16_DTYPE_F16) {
    if (append) launch_rope<__half, true>(p, a.head_dim, s);
    else launch_rope<__half, false>(p, a.head_dim, s);
  } else {
    if (append) launch_rope<__nv_bfloat16, true>(p, a.head_dim, s);
    else launch_rope<__nv_bfloat16, false>(p, a.head_dim, s);
  }
  return launched();
}

int check_tables(const w4a16_kv4_tables* t) {
  if (t == nullptr || t->pages < 1 || t->rows < 1 || t->width < 1 || t->page_size < BLK || t->page_size % BLK != 0 ||
      t->page_size > 4096 || t->refs == nullptr || t->block_table == nullptr || t->kv_lens == nullptr ||
      static_cast<int64_t>(t->width) * t->page_size > 0x7fffffffLL)
    return W4A16_ERR_INVALID;
  return W4A16_OK;
}

Tables tables_of(const w4a16_kv4_tables& t) {
  Tables v;
  v.refs = t.refs; v.table = t.block_table; v.lens = t.kv_lens;
  v.pages = t.pages; v.rows = t.rows; v.width = t.width; v.page_size = t.page_size;
  return v;
}

bool same_shape(const w4a16_kv4_tables& a, const w4a16_kv4_tables& b) {
  return a.pages == b.pages && a.rows == b.rows && a.width == b.width && a.page_size == b.page_size;
}

unsigned table_blocks(const w4a16_kv4_tables& t, int threads, const DeviceState& dev) {
  const long long n = std::max<long long>(static_cast<long long>(t.rows) * t.width, t.pages);
  return static_cast<unsigned>(std::min<long long>((n + threads - 1) / threads, 4LL * dev.num_sms));
}

// Decode attention: query rows per tile, warps and blocks per tile of each shape. Eight rows (NT = 1)
// leave room for 16 warps of 128 registers with two blocks per stage; sixteen rows need 8 warps of
// twice the registers, which take four blocks per stage so that as many bytes are in flight.
template <int D, int NG, int NT, bool SK>
struct DecodeConfig {
  static constexpr int W = NT == 1 ? 16 : 8, TB = NT == 1 ? 2 : 4;
  using Shape = DecodeShape<D, NG, NT, W, TB>;
  static auto kernel() { return kv4_decode_kernel<D, NG, NT, W, TB, SK>; }
};

template <bool SK = false, typename F>
int with_decode_config(const w4a16_kv4_cache& c, int nt, F f) {
  if (c.head_dim == 64) return nt == 1 ? f(DecodeConfig<64, 1, 1, SK>()) : f(DecodeConfig<64, 1, 2, SK>());
  if (c.group_size == 128) return nt == 1 ? f(DecodeConfig<128, 1, 1, SK>()) : f(DecodeConfig<128, 1, 2, SK>());
  return nt == 1 ? f(DecodeConfig<128, 2, 1, SK>()) : f(DecodeConfig<128, 2, 2, SK>());
}

int decode_nt(const AttendPlan& p) { return p.rows <= 8 ? 1 : 2; }

// Warps per team: as many as there are for each segment, a power of two.
int decode_team_warps(const AttendPlan& p, int W, const DeviceState& dev) {
  const int rows = 8 * decode_nt(p);
  const long long segments = std::min<long long>(p.seqs, MAX_SEQS) * p.kv_heads * ((p.rows + rows - 1) / rows);
  int tw = 1;
  while (tw < W && 2 * tw * segments <= static_cast<long long>(dev.num_sms) * W) tw *= 2;
  return tw;
}

// The workspace begins with the teams' counters, always at the same place: what one call leaves zero
// the next one finds zero, whatever its shape.
constexpr int kCounterBytes = 65536;

long long decode_workspace(const w4a16_kv4_cache& c, const AttendPlan& p, const DeviceState& dev) {
  long long parts = 0;
  with_decode_config(c, decode_nt(p), [&](auto cfg) {
    using C = decltype(cfg);
    parts = static_cast<long long>(dev.num_sms) * (C::W / decode_team_warps(p, C::W, dev)) * 2 * C::Shape::PART * 4;
    return 0;
  });
  return kCounterBytes + parts;
}

int launch_decode(const w4a16_kv4_cache& c, const AttendParams& all, const AttendPlan& plan, int bf16, int row_limit,
                  void* workspace, const DeviceState& dev, cudaStream_t s) {
  const int nt = decode_nt(plan);
  auto launch = [&](auto cfg) {
    using C = decltype(cfg);
    const int tw = decode_team_warps(plan, C::W, dev);
    if (dev.num_sms * (C::W / tw) > kCounterBytes / 4) return W4A16_ERR_DEVICE;
    auto k = C::kernel();
    static std::atomic<uint64_t> ready{0};   // devices whose shared memory limit is set
    int d = 0;
    if (cudaGetDevice(&d) != cudaSuccess) return W4A16_ERR_DEVICE;
    if (!(ready.load(std::memory_order_acquire) >> d & 1)) {
      if (cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, C::Shape::SMEM_BYTES) != cudaSuccess) {
        cudaGetLastError();
        return W4A16_ERR_LAUNCH;
      }
      ready.fetch_or(1ull << d, std::memory_order_release);
    }
    // places in a launch's list of tiles fit 31 bits: as many sequences per launch as that allows
    const long long row_tiles = (std::min<long long>(plan.rows, row_limit) + 8 * nt - 1) / (8 * nt);
    const long long tiles = static_cast<long long>(all.width) * all.cache.page_size / (C::TB * BLK) + 1 + 3 * tw;
    if (plan.kv_heads * row_tiles > 0x7fffffffLL / tiles) return W4A16_ERR_INVALID;
    const int step = static_cast<int>(std::min<long long>(MAX_SEQS, 0x7fffffffLL / (plan.kv_heads * row_tiles * tiles)));
    for (int b0 = 0; b0 < all.seqs; b0 += step) {
      DecodeParams p = {};
      p.a = all;
      p.a.seqs = std::min(all.seqs - b0, step);
      p.a.table += static_cast<long long>(b0) * all.width;
      p.a.lens += b0;
      if (p.a.cu_q) {
        p.a.cu_q += b0;
      } else if (p.a.seqs < all.seqs) {     // uniform queries: this launch's own
        const long long each = all.T / all.seqs;
        p.a.q = static_cast<const uint16_t*>(all.q) + b0 * each * all.q_st;
        p.a.o = static_cast<uint16_t*>(all.o) + b0 * each * all.heads * c.head_dim;
        if (all.lse) p.a.lse = all.lse + b0 * each * all.heads;
        p.a.T = static_cast<int>(each * p.a.seqs);
      }
      p.bf16 = bf16;
      p.row_limit = row_limit;
      p.before = b0 == 0;
      p.after = b0 + p.a.seqs == all.seqs;
      p.team_warps = tw;
      // a piece's queries and end cost a team about what three tiles of each of its warps do (6 us
      // where a tile takes 2)
      p.seg_cost = 3 * tw;
      p.teams = dev.num_sms * (C::W / tw);
      p.wait_ns = g_wait_budget_ns.load(std::memory_order_relaxed);
      p.counters = static_cast<int*>(workspace);
      p.parts = reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + kCounterBytes);
      k<<<dev.num_sms, C::W * 32, C::Shape::SMEM_BYTES, s>>>(p);
      const int st = launched();
      if (st != W4A16_OK) return st;
    }
    return static_cast<int>(W4A16_OK);
  };
  return all.sinks ? with_decode_config<true>(c, nt, launch) : with_decode_config(c, nt, launch);
}

// Which kernel takes a sequence goes by its query rows (new tokens x heads of a group) per kv head.
// The tensor-memory kernel reads the cache once per 256 rows but has a block for no less, so a batch of few
// such blocks leaves most SMs idle and takes as long as its longest sequence; the decode kernel reads it
// once per 8 or 16 rows and splits it over all SMs. Up to kDecodeRows rows the decode kernel takes the
// sequence, and every sequence of a batch of at most kDecodeWork rows x kv heads x sequences. Measured, 32
// heads of 128 channels on 8 kv heads (decode kernel against the other, us): one sequence of 8192 tokens, 128
// rows: 34, 138; 1024 rows: 166, 188; 1536 rows: 243, 188; of 1500 tokens, 512 rows: 26, 50; 1024: 43, 49;
// 1536: 78, 50; 16 sequences of 8192, 64 rows: 167, 141; 96: 244, 141 (with many segments the crossing lies
// somewhat below 64). In two groups per head, one of 8192, 512 rows: 102, 234; 1024: 197, 236; 1536: 315, 235;
// with heads of 64, 512: 61, 167; 1024: 116, 168; 1536: 166, 168.
constexpr long long kDecodeRows = 64, kDecodeWork = 8192;

long long decode_rows(const AttendPlan& plan) {
  return plan.rows <= kDecodeWork / std::max(1LL, plan.kv_heads * plan.seqs) ? plan.rows : std::min(plan.rows, kDecodeRows);
}

template <int D, int NG, bool SK>
int launch_prefill_as(const PrefillParams& p, long long blocks, cudaStream_t s) {
  auto k = kv4_prefill_kernel<D, NG, SK>;
  constexpr int bytes = PrefillShape<D, NG>::SMEM_BYTES;
  static std::atomic<uint64_t> ready{0};
  int d = 0;
  if (cudaGetDevice(&d) != cudaSuccess) return W4A16_ERR_DEVICE;
  if (!(ready.load(std::memory_order_acquire) >> d & 1)) {
    if (cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) != cudaSuccess) {
      cudaGetLastError();
      return W4A16_ERR_LAUNCH;
    }
    ready.fetch_or(1ull << d, std::memory_order_release);
  }
  k<<<static_cast<unsigned>(blocks), PF_THREADS, bytes, s>>>(p);
  return launched();
}

template <bool SK>
int launch_prefill_of(const w4a16_kv4_cache& c, const PrefillParams& p, long long blocks, cudaStream_t s) {
  if (c.head_dim == 64) return launch_prefill_as<64, 1, SK>(p, blocks, s);
  if (c.group_size == 128) return launch_prefill_as<128, 1, SK>(p, blocks, s);
  return launch_prefill_as<128, 2, SK>(p, blocks, s);
}

int launch_prefill(const w4a16_kv4_cache& c, const AttendParams& a, const AttendPlan& plan, int bf16, long long row_limit,
                   cudaStream_t s) {
  PrefillParams p = {};
  p.a = a;
  p.bf16 = bf16;
  p.row_limit = static_cast<int>(row_limit);
  p.wait_ns = g_wait_budget_ns.load(std::memory_order_relaxed);
  const long long tiles = (plan.rows + PF_ROWS - 1) / PF_ROWS;
  if (plan.seqs * plan.kv_heads > 0x7fffffffLL / tiles) return W4A16_ERR_INVALID;
  const long long blocks = tiles * plan.seqs * plan.kv_heads;
  return a.sinks ? launch_prefill_of<true>(c, p, blocks, s) : launch_prefill_of<false>(c, p, blocks, s);
}

// Which kernel collects a sequence's weights goes by its query rows per kv head, as for the attention itself.
constexpr long long kWeightsRows = 64;

// The collected weights' workspace: the sequences' prefix sums, the prepared queries of each kernel, and the parts
// of tiles that several of the tensor-memory kernel's blocks share.
struct WeightsLayout {
  long long tiles, tc_tiles, entries;
  long long tc_prefix_at, tc_steps_at, queries_at, tc_queries_at, parts_at, bytes;
  bool many;                 // there may be sequences for the tensor-memory kernel
};
WeightsLayout weights_layout(const w4a16_kv4_cache& c, int64_t T, int heads, int64_t seqs, int64_t max_q, int64_t capacity,
                             int num_sms) {
  WeightsLayout l;
  const int64_t share = heads / c.kv_heads, most = std::min(max_q, T) * share;
  const int n = c.head_dim == 128 && c.group_size == 64 ? 64 : 128;
  l.many = most > kWeightsRows;
  l.tiles = T * share / 8 + seqs;
  l.tc_tiles = l.many ? T * share / n + seqs : 0;
  l.entries = l.many ? std::min<int64_t>(seqs, T * share / kWeightsRows + 1) * ((capacity + WT_TC_TOKENS - 1) / WT_TC_TOKENS) : 0;
  auto up = [](int64_t x) { return (x + 255) / 256 * 256; };
  l.tc_prefix_at = up((seqs + 1) * 8);
  l.tc_steps_at = l.tc_prefix_at + up((seqs + 1) * 8);
  l.queries_at = l.tc_steps_at + up((l.entries + 1) * 8);
  l.tc_queries_at = l.queries_at + up(l.tiles * c.kv_heads * wt_tile_words(c.head_dim) * 4);
  l.parts_at = l.tc_queries_at + up(l.tc_tiles * c.kv_heads * (n * c.head_dim * 2 + n * 16 + 16));
  l.bytes = l.parts_at + (l.many ? 2LL * num_sms * WT_TC_TOKENS * 4 : 0);
  return l;
}

template <typename K>
int allow_shared_memory(K k, int bytes, std::atomic<uint64_t>& ready) {
  int d = 0;
  if (cudaGetDevice(&d) != cudaSuccess) return W4A16_ERR_DEVICE;
  if (!(ready.load(std::memory_order_acquire) >> d & 1)) {
    if (cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) != cudaSuccess) {
      cudaGetLastError();
      return W4A16_ERR_LAUNCH;
    }
    ready.fetch_or(1ull << d, std::memory_order_release);
  }
  return W4A16_OK;
}

template <int D, int NG>
int launch_weights_as(const WeightsParams& p, bool many, bool few, const DeviceState& dev, cudaStream_t s) {
  static_assert(TcShape<D, NG>::N == (D == 128 && NG == 2 ? 64 : 128), "weights_layout's");
  static std::atomic<uint64_t> ready{0}, tc_ready{0};
  const long long items = static_cast<long long>(p.tiles) * p.a.cache.kv_heads;
  kv4_weights_prep_kernel<D, NG><<<static_cast<unsigned>(1 + (items + WT_PREP / 32 - 1) / (WT_PREP / 32) + p.copies), WT_PREP, 0, s>>>(p);
  int st = launched();
  if (st != W4A16_OK) return st;
  if (many) {
    constexpr int bytes = TcShape<D, NG>::SMEM_BYTES;
    if ((st = allow_shared_memory(kv4_weights_tc_kernel<D, NG>, bytes, tc_ready)) != W4A16_OK) return st;
    if ((st = launch_after(kv4_weights_tc_kernel<D, NG>, p.blocks, WT_TC_THREADS, bytes, 1, s, p)) != W4A16_OK) return st;
    if ((st = launch_after(kv4_weights_join_kernel<D, NG>, 4 * dev.num_sms, WT_TC_TOKENS, 0, 1, s, p)) != W4A16_OK) return st;
  }
  if (few) {
    constexpr int bytes = WeightsShape<D, NG>::SMEM_BYTES;
    if ((st = allow_shared_memory(kv4_weights_kernel<D, NG>, bytes, ready)) != W4A16_OK) return st;
    st = launch_after(kv4_weights_kernel<D, NG>, WT_PER_SM * dev.num_sms, WT_THREADS, bytes, 1, s, p);
  }
  return st;
}

// Pages that `keep` tokens take: a row that holds more has as many, at least.
int64_t evict_pages(const w4a16_kv4_tables& t, int keep) {
  return std::min<int64_t>((static_cast<int64_t>(keep) + t.page_size - 1) / t.page_size, t.width);
}

// Blocks of a cluster that share a row's kv head of a layer: a power of two, more than one where there are not four
// blocks for each SM.
int evict_split(long long items, int num_sms) {
  int split = 1;
  while (split < 8 && 2 * split * items <= 4LL * num_sms) split *= 2;
  return split;
}

template <int D, int NG>
int launch_evict_as(const EvictParams& p, long long items, int split, cudaStream_t s) {
  return launch_after(kv4_evict_kernel<D, NG>, static_cast<unsigned>(items * split), EVICT_THREADS, p.key_limit * 6, split, s, p);
}

// The copies of pages, and how many blocks share them.
CopyParams copy_params(const w4a16_kv4_cache& c, const int* src, const int* dst, const int* count, int n,
                       const DeviceState& dev, unsigned* blocks) {
  const CacheView v = view_of(c, 0);
  CopyParams p = {};
  p.pool = v.pool;
  p.copy_bytes = c.kv_heads * v.page_bytes;
  p.layer_bytes = c.pages * p.copy_bytes;
  p.layers = static_cast<int>(c.layers);
  p.pages = static_cast<int>(c.pages);
  p.src = src; p.dst = dst; p.count = count; p.n = n;
  const long long per_part = 16LL * COPY_THREADS * COPY_VECS;
  p.parts = static_cast<int>((p.copy_bytes + per_part - 1) / per_part);
  const long long work = static_cast<long long>(n) * c.layers * p.parts;
  *blocks = static_cast<unsigned>(std::min<long long>(work, 8LL * dev.num_sms));
  return p;
}

}  // namespace
}  // namespace kv4
}  // namespace w4a16

extern "C" {

int w4a16_kv4_page_bytes(int head_dim, int page_size, int group_size, int64_t* bytes_out) {
  if (bytes_out == nullptr || (head_dim != 64 && head_dim != 128) || page_size < kv4::BLK || page_size % kv4::BLK != 0 ||
      page_size > 4096 || (group_size != 64 && group_size != head_dim))
    return W4A16_ERR_INVALID;
  *bytes_out = static_cast<int64_t>(page_size / kv4::BLK) * kv4::block_bytes(head_dim, head_dim / group_size);
  return W4A16_OK;
}

int w4a16_qk_norm_rope(const void* q, const void* k, int dtype, int64_t T, int heads, int kv_heads, int head_dim,
                       int64_t q_token_stride, int64_t q_head_stride, int64_t k_token_stride, int64_t k_head_stride,
                       const int64_t* positions, int axes, int axis0_end, int axis1_end, const float* cos_sin,
                       int64_t max_position, int rot, int interleaved, const void* q_weight, const void* k_weight,
                       int weight_dtype, float eps, void* q_out, void* k_out, void* stream) {
  kv4::RopeArgs a = {q, k, nullptr, dtype, T, heads, kv_heads, head_dim, q_token_stride, q_head_stride, k_token_stride,
                     k_head_stride, 0, 0, positions, axes, axis0_end, axis1_end, cos_sin, max_position, rot, interleaved,
                     q_weight, k_weight, weight_dtype, eps};
  return kv4::rope(a, q_out, k_out, nullptr, 0, nullptr, stream);
}

int w4a16_qk_norm_rope_append(const void* q, const void* k, const void* v, int dtype, int64_t T, int heads,
                              int64_t q_token_stride, int64_t q_head_stride, int64_t k_token_stride,
                              int64_t k_head_stride, int64_t v_token_stride, int64_t v_head_stride,
                              const int64_t* positions, int axes, int axis0_end, int axis1_end, const float* cos_sin,
                              int64_t max_position, int rot, int interleaved, const void* q_weight,
                              const void* k_weight, int weight_dtype, float eps, void* q_out,
                              const w4a16_kv4_cache* cache, int64_t layer, const int64_t* slots, void* stream) {
  if (cache == nullptr) return W4A16_ERR_INVALID;
  kv4::RopeArgs a = {q, k, v, dtype, T, heads, cache->kv_heads, cache->head_dim, q_token_stride, q_head_stride,
                     k_token_stride, k_head_stride, v_token_stride, v_head_stride, positions, axes, axis0_end, axis1_end,
                     cos_sin, max_position, rot, interleaved, q_weight, k_weight, weight_dtype, eps};
  return kv4::rope(a, q_out, nullptr, cache, layer, slots, stream);
}

int w4a16_kv4_gather(const w4a16_kv4_cache* cache, int64_t layer, const int64_t* slots, int64_t n, void* out, int dtype,
                     void* stream) {
  DeviceState* dev = nullptr;
  const int st = kv4::check_cache(cache, &dev);
  if (st != W4A16_OK) return st;
  if (layer < 0 || layer >= cache->layers || n < 0 || n > 0x7fffffffLL ||
      (dtype != W4A16_DTYPE_F16 && dtype != W4A16_DTYPE_BF16))
    return W4A16_ERR_INVALID;
  if (n == 0) return W4A16_OK;
  if (slots == nullptr || out == nullptr) return W4A16_ERR_INVALID;
  if (!aligned16(out)) return W4A16_ERR_ALIGNMENT;
  kv4::GatherParams p = {};
  p.slots = reinterpret_cast<const long long*>(slots);
  p.n = n;
  p.out = out;
  p.cache = kv4::view_of(*cache, layer);
  p.groups = cache->head_dim / cache->group_size;
  p.by_heads = kv4::Divisor(cache->kv_heads);
  if (n * cache->kv_heads > 0x7fffffffLL) return W4A16_ERR_INVALID;   // counted in 32 bits
  const unsigned grid = static_cast<unsigned>((n * cache->kv_heads * (cache->head_dim / 8) + 255) / 256);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (dtype == W4A16_DTYPE_F16) {
    if (cache->head_dim == 128) kv4::kv4_gather_kernel<__half, 128><<<grid, 256, 0, s>>>(p);
    else kv4::kv4_gather_kernel<__half, 64><<<grid, 256, 0, s>>>(p);
  } else {
    if (cache->head_dim == 128) kv4::kv4_gather_kernel<__nv_bfloat16, 128><<<grid, 256, 0, s>>>(p);
    else kv4::kv4_gather_kernel<__nv_bfloat16, 64><<<grid, 256, 0, s>>>(p);
  }
  return kv4::launched();
}

int w4a16_kv4_attention_workspace_size(const w4a16_kv4_cache* cache, int64_t T, int heads, int64_t seqs, int64_t max_q,
                                       int64_t* bytes_out) {
  DeviceState* dev = nullptr;
  if (bytes_out == nullptr) return W4A16_ERR_INVALID;
  *bytes_out = 0;
  const int st = kv4::check_cache(cache, &dev);
  if (st != W4A16_OK) return st;
  if (T < 0 || T > 0x7fffffffLL || heads < 1 || heads % cache->kv_heads != 0 || seqs < 0 || max_q < 0)
    return W4A16_ERR_INVALID;
  if (T == 0 || seqs == 0) return W4A16_OK;
  kv4::AttendPlan plan = {seqs, cache->kv_heads, std::min(max_q, T) * (heads / cache->kv_heads)};
  plan.rows = kv4::decode_rows(plan);
  *bytes_out = kv4::decode_workspace(*cache, plan, *dev);
  return W4A16_OK;
}

int w4a16_kv4_attention(const void* q, int dtype, int64_t T, int heads, int64_t q_token_stride, int64_t q_head_stride,
                        const w4a16_kv4_cache* cache, int64_t layer, const int32_t* block_table, int64_t table_width,
                        const int32_t* kv_lens, const int32_t* cu_q, int64_t seqs, int64_t max_q, float scale,
                        int window, void* o, float* lse, void* workspace, int64_t workspace_bytes, void* stream) {
  return w4a16_kv4_attention_sinks(q, dtype, T, heads, q_token_stride, q_head_stride, cache, layer, block_table,
                                   table_width, kv_lens, cu_q, seqs, max_q, scale, window, 0, o, lse, workspace,
                                   workspace_bytes, stream);
}

int w4a16_kv4_attention_sinks(const void* q, int dtype, int64_t T, int heads, int64_t q_token_stride,
                              int64_t q_head_stride, const w4a16_kv4_cache* cache, int64_t layer,
                              const int32_t* block_table, int64_t table_width, const int32_t* kv_lens,
                              const int32_t* cu_q, int64_t seqs, int64_t max_q, float scale, int window, int sinks,
                              void* o, float* lse, void* workspace, int64_t workspace_bytes, void* stream) {
  DeviceState* dev = nullptr;
  const int st = kv4::check_cache(cache, &dev);
  if (st != W4A16_OK) return st;
  if (T < 0 || T > 0x7fffffffLL || (dtype != W4A16_DTYPE_F16 && dtype != W4A16_DTYPE_BF16) || heads < 1 ||
      heads > 65535 || heads % cache->kv_heads != 0 || layer < 0 || layer >= cache->layers || seqs < 0 ||
      seqs > 0x7fffffffLL || table_width < 0 || max_q < 0 || window < 0 || sinks < 0 || workspace_bytes < 0 || !(scale == scale) ||
      table_width * cache->page_size > 0x7fffffffLL || T * (heads / cache->kv_heads) > (1LL << 30))
    return W4A16_ERR_INVALID;
  if (T == 0 || seqs == 0) return T == 0 ? W4A16_OK : W4A16_ERR_INVALID;
  if (cu_q == nullptr && T % seqs != 0) return W4A16_ERR_INVALID;
  if (q == nullptr || o == nullptr || kv_lens == nullptr || (table_width > 0 && block_table == nullptr))
    return W4A16_ERR_INVALID;
  if (!aligned16(q) || !aligned16(o) || q_token_stride % 8 != 0 || q_head_stride % 8 != 0) return W4A16_ERR_ALIGNMENT;
  kv4::AttendParams p = {};
  p.q = q; p.q_st = q_token_stride; p.q_sh = q_head_stride;
  p.o = o; p.lse = lse;
  p.cache = kv4::view_of(*cache, layer);
  p.table = block_table; p.width = static_cast<int>(table_width);
  p.lens = kv_lens; p.cu_q = cu_q;
  p.seqs = static_cast<int>(seqs); p.T = static_cast<int>(T);
  p.max_q = static_cast<int>(std::min<int64_t>(max_q, T));
  p.heads = heads; p.share = heads / cache->kv_heads;
  p.scale = scale; p.window = window;
  p.sinks = window ? sinks : 0;
  p.by_share = kv4::Divisor(p.share);
  p.groups = cache->head_dim / cache->group_size;
  const kv4::AttendPlan plan = {seqs, cache->kv_heads, (cu_q ? std::min(max_q, T) : T / seqs) * p.share};
  kv4::AttendPlan few = plan;      // the sequences that the decode kernel takes
  few.rows = kv4::decode_rows(plan);
  const int64_t need = kv4::decode_workspace(*cache, few, *dev);
  if (workspace == nullptr || workspace_bytes < need || reinterpret_cast<uintptr_t>(workspace) % 256 != 0)
    return W4A16_ERR_WORKSPACE;
  const int bf16 = dtype == W4A16_DTYPE_BF16;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (plan.rows > few.rows) {
    const int st2 = kv4::launch_prefill(*cache, p, plan, bf16, few.rows, s);
    if (st2 != W4A16_OK || cu_q == nullptr) return st2;
  }
  // sequences with few rows (every one, unless the batch is mixed)
  return kv4::launch_decode(*cache, p, few, bf16, static_cast<int>(few.rows), workspace, *dev, s);
}

int w4a16_kv4_attention_weights_workspace_size(const w4a16_kv4_cache* cache, int64_t T, int heads, int64_t seqs,
                                               int64_t max_q, int64_t capacity, int64_t* bytes_out) {
  DeviceState* dev = nullptr;
  if (bytes_out == nullptr) return W4A16_ERR_INVALID;
  *bytes_out = 0;
  const int st = kv4::check_cache(cache, &dev);
  if (st != W4A16_OK) return st;
  if (T < 0 || T > 0x7fffffffLL || heads < 1 || heads > 65535 || heads % cache->kv_heads != 0 || seqs < 0 || seqs > 0x7fffffffLL ||
      max_q < 0 || capacity < 0 || capacity > 0x7fffffffLL || T * (heads / cache->kv_heads) > (1LL << 30))
    return W4A16_ERR_INVALID;
  *bytes_out = kv4::weights_layout(*cache, T, heads, seqs, max_q, capacity, dev->num_sms).bytes;
  return W4A16_OK;
}

int w4a16_kv4_attention_weights(const void* q, int dtype, int64_t T, int heads, int64_t q_token_stride,
                                int64_t q_head_stride, const w4a16_kv4_cache* cache, int64_t layer,
                                const int32_t* block_table, int64_t table_width, const int32_t* kv_lens,
                                const int32_t* cu_q, int64_t seqs, int64_t max_q, float scale, int window, int sinks,
                                const float* lse, const float* before, int64_t before_seq_stride,
                                int64_t before_head_stride, float* after, int64_t after_seq_stride,
                                int64_t after_head_stride, int64_t capacity, void* workspace, int64_t workspace_bytes,
                                void* stream) {
  DeviceState* dev = nullptr;
  int st = kv4::check_cache(cache);
  if (st != W4A16_OK) return st;
  if (!kv4::can_write({before, {{seqs, before_seq_stride}, {cache->kv_heads, before_head_stride}}, capacity},
                      {after, {{seqs, after_seq_stride}, {cache->kv_heads, after_head_stride}}, capacity}))
    return W4A16_ERR_INVALID;
  if ((st = current_device_state(&dev)) != W4A16_OK) return st;
  int64_t need = 0;
  if (seqs > 0 && cu_q == nullptr) max_q = T / seqs;
  if (w4a16_kv4_attention_weights_workspace_size(cache, T, heads, seqs, max_q, capacity, &need) != W4A16_OK ||
      (dtype != W4A16_DTYPE_F16 && dtype != W4A16_DTYPE_BF16) || layer < 0 || layer >= cache->layers || table_width < 0 ||
      max_q < 0 || window < 0 || sinks < 0 || workspace_bytes < 0 || !(scale == scale) || capacity < 0 ||
      capacity > 0x7fffffffLL || table_width * cache->page_size > 0x7fffffffLL)
    return W4A16_ERR_INVALID;
  if (seqs == 0) return T == 0 ? W4A16_OK : W4A16_ERR_INVALID;
  if (cu_q == nullptr && T % seqs != 0) return W4A16_ERR_INVALID;
  if (kv_lens == nullptr || (T > 0 && (q == nullptr || lse == nullptr)) || (table_width > 0 && block_table == nullptr) ||
      (capacity > 0 && (before == nullptr || after == nullptr)))
    return W4A16_ERR_INVALID;
  if (!aligned16(q) || q_token_stride % 8 != 0 || q_head_stride % 8 != 0) return W4A16_ERR_ALIGNMENT;
  if (workspace == nullptr || workspace_bytes < need || reinterpret_cast<uintptr_t>(workspace) % 256 != 0)
    return W4A16_ERR_WORKSPACE;
  const kv4::WeightsLayout layout = kv4::weights_layout(*cache, T, heads, seqs, max_q, capacity, dev->num_sms);
  if (layout.tiles * cache->kv_heads > 0x7fffffffLL) return W4A16_ERR_INVALID;
  kv4::WeightsParams p = {};
  p.a.q = q; p.a.q_st = q_token_stride; p.a.q_sh = q_head_stride;
  p.a.cache = kv4::view_of(*cache, layer);
  p.a.table = block_table; p.a.width = static_cast<int>(table_width);
  p.a.lens = kv_lens; p.a.cu_q = cu_q;
  p.a.seqs = static_cast<int>(seqs); p.a.T = static_cast<int>(T);
  p.a.max_q = static_cast<int>(std::min<int64_t>(max_q, T));
  p.a.heads = heads; p.a.share = heads / cache->kv_heads;
  p.a.scale = scale; p.a.window = window;
  p.a.sinks = window ? sinks : 0;
  p.a.groups = cache->head_dim / cache->group_size;
  p.lse = lse;
  p.before = before; p.b_ss = before_seq_stride; p.b_sh = before_head_stride;
  p.after = after; p.a_ss = after_seq_stride; p.a_sh = after_head_stride;
  p.capacity = static_cast<int>(capacity);
  p.bf16 = dtype == W4A16_DTYPE_BF16;
  p.wait_ns = g_wait_budget_ns.load(std::memory_order_relaxed);
  p.tiles = static_cast<int>(layout.tiles);
  p.a.by_share = kv4::Divisor(p.a.share);
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  p.prefix = reinterpret_cast<long long*>(ws);
  p.queries = reinterpret_cast<uint32_t*>(ws + layout.queries_at);
  p.row_limit = static_cast<int>(kv4::kWeightsRows);
  p.tc_tiles = static_cast<int>(layout.tc_tiles);
  p.copies = before == after || (window == 0 && cu_q == nullptr && T > 0)
                 ? 0 : static_cast<int>(std::min<int64_t>(2 * dev->num_sms, seqs * cache->kv_heads));
  p.entries = layout.entries;
  p.blocks = dev->num_sms;
  p.tc_prefix = reinterpret_cast<long long*>(ws + layout.tc_prefix_at);
  p.tc_queries = ws + layout.tc_queries_at;
  p.tc_steps = reinterpret_cast<long long*>(ws + layout.tc_steps_at);
  p.parts = reinterpret_cast<float*>(ws + layout.parts_at);
  const bool few = cu_q != nullptr || !layout.many;    // (every sequence has the same rows without cu_q)
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (cache->head_dim == 64) return kv4::launch_weights_as<64, 1>(p, layout.many, few, *dev, s);
  if (cache->group_size == 128) return kv4::launch_weights_as<128, 1>(p, layout.many, few, *dev, s);
  return kv4::launch_weights_as<128, 2>(p, layout.many, few, *dev, s);
}

int w4a16_kv4_copy_pages(const w4a16_kv4_cache* cache, const int32_t* src, const int32_t* dst, int64_t n, void* stream) {
  DeviceState* dev = nullptr;
  const int st = kv4::check_cache(cache, &dev);
  if (st != W4A16_OK) return st;
  if (n < 0 || n > 0x7fffffffLL) return W4A16_ERR_INVALID;
  if (n == 0) return W4A16_OK;
  if (src == nullptr || dst == nullptr) return W4A16_ERR_INVALID;
  unsigned blocks = 0;
  const kv4::CopyParams p = kv4::copy_params(*cache, src, dst, nullptr, static_cast<int>(n), *dev, &blocks);
  kv4::kv4_copy_pages_kernel<<<blocks, kv4::COPY_THREADS, 0, static_cast<cudaStream_t>(stream)>>>(p);
  return kv4::launched();
}

int w4a16_kv4_reserve(const w4a16_kv4_tables* tables, const int32_t* rows, const int32_t* lens, int64_t n, int32_t* ok,
                      int32_t* scratch, void* stream) {
  const int st = kv4::check_tables(tables);
  if (st != W4A16_OK) return st;
  if (n < 0 || n > (1 << 30)) return W4A16_ERR_INVALID;
  if (n == 0) return W4A16_OK;
  if (rows == nullptr || lens == nullptr || ok == nullptr || scratch == nullptr) return W4A16_ERR_INVALID;
  DeviceState* dev = nullptr;
  const int ds = current_device_state(&dev);
  if (ds != W4A16_OK) return ds;
  kv4::ReserveParams p = {kv4::tables_of(*tables), rows, lens, static_cast<int>(n), ok, scratch};
  kv4::kv4_reserve_kernel<<<1, kv4::SCAN_THREADS, 0, static_cast<cudaStream_t>(stream)>>>(p);
  return kv4::launched();
}

int w4a16_kv4_fork(const w4a16_kv4_cache* cache, const w4a16_kv4_tables* in, const w4a16_kv4_tables* out,
                   const int32_t* parents, const int32_t* children, int64_t n, int32_t* ok, int32_t* scratch,
                   void* stream) {
  DeviceState* dev = nullptr;
  int st = kv4::check_cache(cache, &dev);
  if (st != W4A16_OK) return st;
  if ((st = kv4::check_tables(in)) != W4A16_OK || (st = kv4::check_tables(out)) != W4A16_OK) return st;
  if (!kv4::same_shape(*in, *out) || in->pages != cache->pages || in->page_size != cache->page_size || n < 0 ||
      n > (1 << 30))
    return W4A16_ERR_INVALID;
  if (n > 0 && (parents == nullptr || children == nullptr || ok == nullptr || scratch == nullptr))
    return W4A16_ERR_INVALID;
  kv4::ForkParams p = {kv4::tables_of(*in), kv4::tables_of(*out), parents, children, static_cast<int>(n), ok, scratch,
                       scratch + n};
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (n == 0) {
    kv4::kv4_copy_tables_kernel<<<kv4::table_blocks(*in, 256, *dev), 256, 0, s>>>(p.in, p.out);
    return kv4::launched();
  }
  kv4::kv4_fork_plan_kernel<<<1 + kv4::table_blocks(*in, kv4::SCAN_THREADS, *dev), kv4::SCAN_THREADS, 0, s>>>(p);
  unsigned blocks = 0;
  const kv4::CopyParams copy = kv4::copy_params(*cache, p.src, p.dst, nullptr, p.n, *dev, &blocks);
  kv4::kv4_fork_rows_kernel<<<static_cast<unsigned>(n) + blocks, kv4::COPY_THREADS, 0, s>>>(p, copy);
  return kv4::launched();
}

int w4a16_kv4_release(const w4a16_kv4_tables* in, const w4a16_kv4_tables* out, const int32_t* rows, int64_t n,
                      void* stream) {
  int st;
  if ((st = kv4::check_tables(in)) != W4A16_OK || (st = kv4::check_tables(out)) != W4A16_OK) return st;
  if (!kv4::same_shape(*in, *out) || n < 0 || n > 0x7fffffffLL || (n > 0 && rows == nullptr)) return W4A16_ERR_INVALID;
  DeviceState* dev = nullptr;
  if ((st = current_device_state(&dev)) != W4A16_OK) return st;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const kv4::Tables ti = kv4::tables_of(*in), to = kv4::tables_of(*out);
  if (ti.refs != to.refs || ti.table != to.table || ti.lens != to.lens)
    kv4::kv4_copy_tables_kernel<<<kv4::table_blocks(*in, 256, *dev), 256, 0, s>>>(ti, to);
  if (n > 0) {
    kv4::ReleaseParams p = {to, rows};
    kv4::kv4_release_kernel<<<static_cast<unsigned>(n), 256, 0, s>>>(p);
  }
  return kv4::launched();
}

int w4a16_kv4_evict_scratch_ints(const w4a16_kv4_tables* in, int64_t n, int keep, int64_t* ints_out) {
  if (ints_out == nullptr) return W4A16_ERR_INVALID;
  *ints_out = 0;
  const int st = kv4::check_tables(in);
  if (st != W4A16_OK) return st;
  // (the device adds up in 32 bits how many pages are asked for)
  if (n < 0 || n > (1 << 20) || keep < 1 || n * kv4::evict_pages(*in, keep) > 0x7fffffffLL) return W4A16_ERR_INVALID;
  *ints_out = n * (3 + kv4::evict_pages(*in, keep) + in->width) + 1 + in->rows;
  return W4A16_OK;
}

int w4a16_kv4_evict(const w4a16_kv4_cache* cache, const w4a16_kv4_tables* in, const w4a16_kv4_tables* out,
                    const float* weights, int64_t w_layer_stride, int64_t w_row_stride, int64_t w_head_stride, float* kept,
                    int64_t k_layer_stride, int64_t k_row_stride, int64_t k_head_stride, int64_t capacity,
                    const int32_t* rows, int64_t n, int keep, int sinks, int recent, int32_t* ok, int32_t* scratch,
                    void* stream) {
  DeviceState* dev = nullptr;
  int st = kv4::check_cache(cache);
  if (st != W4A16_OK) return st;
  if ((st = kv4::check_tables(in)) != W4A16_OK || (st = kv4::check_tables(out)) != W4A16_OK) return st;
  if (n > 0 && !kv4::can_write(
          {weights, {{cache->layers, w_layer_stride}, {in->rows, w_row_stride}, {cache->kv_heads, w_head_stride}}, capacity},
          {kept, {{cache->layers, k_layer_stride}, {in->rows, k_row_stride}, {cache->kv_heads, k_head_stride}}, capacity}))
    return W4A16_ERR_INVALID;
  if ((st = current_device_state(&dev)) != W4A16_OK) return st;
  int64_t ints = 0;
  if ((st = w4a16_kv4_evict_scratch_ints(in, n, keep, &ints)) != W4A16_OK) return st;
  if (!kv4::same_shape(*in, *out) || in->pages != cache->pages || in->page_size != cache->page_size || sinks < 0 ||
      recent < 0 || static_cast<int64_t>(sinks) + recent > keep || capacity < 0 || capacity > 0x7fffffffLL)
    return W4A16_ERR_INVALID;
  const long long items = cache->layers * n * cache->kv_heads;
  if (n > 0 && (weights == nullptr || kept == nullptr || rows == nullptr || ok == nullptr || scratch == nullptr ||
                cache->layers > 0x7fffffffLL / 8 / (n * cache->kv_heads)))
    return W4A16_ERR_INVALID;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  kv4::EvictParams p = {};
  p.cache = kv4::view_of(*cache, 0);
  p.layer_bytes = cache->pages * cache->kv_heads * p.cache.page_bytes;
  p.in = kv4::tables_of(*in);
  p.out = kv4::tables_of(*out);
  p.weights = weights; p.w_sl = w_layer_stride; p.w_sr = w_row_stride; p.w_sh = w_head_stride;
  p.kept = kept; p.k_sl = k_layer_stride; p.k_sr = k_row_stride; p.k_sh = k_head_stride;
  p.capacity = static_cast<int>(capacity);
  p.rows = rows;
  p.n = static_cast<int>(n);
  p.keep = keep; p.sinks = sinks; p.recent = recent;
  p.need = static_cast<int>(kv4::evict_pages(*in, keep));
  p.ok = ok;
  p.does = scratch;
  p.lens = p.does + n;
  p.start = p.lens + n;
  p.fresh = p.start + n + 1;
  p.old = p.fresh + n * p.need;
  p.claim = p.old + n * in->width;
  p.key_limit = static_cast<int>(std::min<int64_t>((std::max<int64_t>(capacity, 1) + 1) / 2 * 2, kv4::EVICT_KEYS));
  const bool apart = p.in.refs != p.out.refs || p.in.table != p.out.table || p.in.lens != p.out.lens;
  if (n == 0 && !apart) return W4A16_OK;
  const unsigned copies = apart ? kv4::table_blocks(*in, kv4::SCAN_THREADS, *dev) : 0;
  kv4::kv4_evict_plan_kernel<<<1 + static_cast<unsigned>(n) + copies, kv4::SCAN_THREADS, 0, s>>>(p);
  if ((st = kv4::launched()) != W4A16_OK || n == 0) return st;
  const int split = kv4::evict_split(items, dev->num_sms);
  if (cache->head_dim == 64) return kv4::launch_evict_as<64, 1>(p, items, split, s);
  if (cache->group_size == 128) return kv4::launch_evict_as<128, 1>(p, items, split, s);
  return kv4::launch_evict_as<128, 2>(p, items, split, s);
}

int w4a16_kv4_compact(const w4a16_kv4_cache* cache, const w4a16_kv4_tables* in, const w4a16_kv4_tables* out,
                      int32_t* scratch, void* stream) {
  DeviceState* dev = nullptr;
  int st = kv4::check_cache(cache, &dev);
  if (st != W4A16_OK) return st;
  if ((st = kv4::check_tables(in)) != W4A16_OK || (st = kv4::check_tables(out)) != W4A16_OK) return st;
  if (!kv4::same_shape(*in, *out) || in->pages != cache->pages || in->page_size != cache->page_size ||
      scratch == nullptr)
    return W4A16_ERR_INVALID;
  const int pages = in->pages, half = pages / 2;
  kv4::CompactParams p = {kv4::tables_of(*in), kv4::tables_of(*out), scratch, scratch + pages, scratch + pages + half,
                          scratch + pages + 2 * half, static_cast<int>(kv4::table_blocks(*in, kv4::COPY_THREADS, *dev))};
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  kv4::kv4_compact_plan_kernel<<<1, kv4::SCAN_THREADS, 0, s>>>(p);
  unsigned blocks = 0;
  const kv4::CopyParams copy = kv4::copy_params(*cache, p.src, p.dst, p.count, half, *dev, &blocks);
  kv4::kv4_compact_tables_kernel<<<static_cast<unsigned>(p.table_blocks) + blocks, kv4::COPY_THREADS, 0, s>>>(p, copy);
  return kv4::launched();
}

}  // extern "C"
