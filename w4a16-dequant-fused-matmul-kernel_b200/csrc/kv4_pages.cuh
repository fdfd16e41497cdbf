// kv4_pages.cuh -- page management of the 4-bit cache on the device, without a host round trip:
// growing sequences (reserve), copying pages, forking sequences (shared full pages, a copy of
// the partly filled last one), releasing them, and compacting the pool.
//
// State: refs [pages] (how many sequences hold a page; 0: free), block_table [rows][width]
// (-1: none) and kv_lens [rows]. Free pages are handed out lowest id first, in the order of the
// request, so results do not depend on timing; reference counts change by integer atomics.
//
// The copies are memory-bound: 400 pages of 70 KB in each of 16 layers (891 MB in and out) take 150 us, 5.9
// TB/s, 93% of a plain copy's rate. What decides (which page goes where) is a scan of the reference
// counts by one block, 5 to 7 us for 1200 to 2048 pages: more blocks would need a grid-wide join
// between their counts, which costs as much. Everything after it is one launch.
#pragma once

#include "kv4_common.cuh"

namespace w4a16 {
namespace kv4 {

constexpr int SCAN_THREADS = 1024;

// Exclusive prefix sum over the block of one value per thread; *total gets the sum.
__device__ __forceinline__ int block_exclusive_scan(int v, int* total) {
  __shared__ int warp_sums[SCAN_THREADS / 32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int inc = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int n = __shfl_up_sync(0xffffffffu, inc, o);
    if (lane >= o) inc += n;
  }
  __syncthreads();   // an earlier call's readers are done
  if (lane == 31) warp_sums[warp] = inc;
  __syncthreads();
  if (warp == 0) {
    int s = warp_sums[lane];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int n = __shfl_up_sync(0xffffffffu, s, o);
      if (lane >= o) s += n;
    }
    warp_sums[lane] = s;
  }
  __syncthreads();
  *total = warp_sums[SCAN_THREADS / 32 - 1];
  return inc - v + (warp ? warp_sums[warp - 1] : 0);
}

struct Tables {
  int* refs;
  int* table;
  int* lens;
  int pages, rows, width, page_size;
};

// ---------------------------------------------------------------------------
// Copies of pages: pair i copies page src[i] to dst[i] in every layer (all kv heads).
// ---------------------------------------------------------------------------
struct CopyParams {
  uint8_t* pool;             // layer 0
  long long layer_bytes;     // bytes of a layer
  long long copy_bytes;      // bytes of a page, all kv heads: a multiple of 16
  int layers, pages;
  int parts;                 // pieces of a page: at most COPY_THREADS * COPY_VECS uint4 each
  const int *src, *dst;      // [n]; a pair with a negative entry is skipped
  const int* count;          // how many pairs there are, or null: n
  int n;
};

// A page is copied in `parts` near-equal pieces of at most COPY_VECS uint4 a thread, so that each
// piece's loads are in flight together and a handful of pages still fills the SMs.
constexpr int COPY_THREADS = 256, COPY_VECS = 4;

// This block's share, the `block`-th of `blocks`.
__device__ __forceinline__ void copy_pages(const CopyParams& p, unsigned block, unsigned blocks) {
  const int n = p.count ? min(*p.count, p.n) : p.n;
  const long long work = static_cast<long long>(n) * p.layers * p.parts;
  const long long vecs = p.copy_bytes / 16;
  for (long long w = block; w < work; w += blocks) {
    const long long item = w / p.parts;
    const int part = static_cast<int>(w - item * p.parts);
    const long long layer = item / n;
    const int i = static_cast<int>(item - layer * n);
    const int s = p.src[i], d = p.dst[i];
    if (s < 0 || d < 0) continue;
    if (s >= p.pages || d >= p.pages) {
      if (threadIdx.x == 0) flag_error(kErrIndex);
      continue;
    }
    uint8_t* base = p.pool + layer * p.layer_bytes;
    const uint4* from = reinterpret_cast<const uint4*>(base + s * p.copy_bytes);
    uint4* to = reinterpret_cast<uint4*>(base + d * p.copy_bytes);
    const long long first = part * vecs / p.parts + threadIdx.x, end = (part + 1) * vecs / p.parts;
    uint4 v[COPY_VECS];
#pragma unroll
    for (int c = 0; c < COPY_VECS; ++c)
      if (first + c * COPY_THREADS < end) v[c] = from[first + c * COPY_THREADS];
#pragma unroll
    for (int c = 0; c < COPY_VECS; ++c)
      if (first + c * COPY_THREADS < end) to[first + c * COPY_THREADS] = v[c];
  }
}

__global__ void __launch_bounds__(COPY_THREADS) kv4_copy_pages_kernel(const CopyParams p) {
  copy_pages(p, blockIdx.x, gridDim.x);
}

// ---------------------------------------------------------------------------
// Free pages: put(j, id) for the lowest `need` free ids of refs, j-th lowest first (as many as
// there are). One block of SCAN_THREADS threads.
// ---------------------------------------------------------------------------
template <typename Put>
__device__ __forceinline__ void lowest_free(const int* refs, int pages, int need, Put put) {
  int found = 0;
  for (int base = 0; base < pages && found < need; base += SCAN_THREADS) {
    const int id = base + threadIdx.x;
    const int is_free = id < pages && refs[id] == 0;
    int total;
    const int at = found + block_exclusive_scan(is_free, &total);
    if (is_free && at < need) put(at, id);
    found += total;
  }
}

// Growth: row rows[i] gets pages up to lens[i] tokens. ok[i] = 1 where it has them (its kv_lens
// is then lens[i]); 0, and nothing changed, where the free pages before it in the order of the
// request do not reach, the table is too narrow, or lens[i] is less than it has. Pages that the row
// has beyond its length (which was lowered) are used before free ones.
struct ReserveParams {
  Tables t;
  const int *req_rows, *req_lens;
  int n;
  int* ok;                   // [n]
  int* start;                // [n + 1] scratch: pages asked for before request i
};

__global__ void __launch_bounds__(SCAN_THREADS) kv4_reserve_kernel(const ReserveParams p) {
  const Tables& t = p.t;
  int before = 0;
  for (int base = 0; base < p.n; base += SCAN_THREADS) {
    const int i = base + threadIdx.x;
    int need = 0, good = 0;
    if (i < p.n) {
      const int r = p.req_rows[i], len = p.req_lens[i];
      if (r < 0 || r >= t.rows) {
        flag_error(kErrIndex);
      } else {
        const int have = t.lens[r];
        const int want = len / t.page_size + (len % t.page_size != 0);
        if (have >= 0 && len >= have && want <= t.width) {
          good = 1;
          int held = have / t.page_size + (have % t.page_size != 0);
          for (; held < want; ++held) {
            const int page = t.table[static_cast<long long>(r) * t.width + held];
            if (page < 0 || page >= t.pages || t.refs[page] <= 0) break;
          }
          need = want - held;
        }
      }
    }
    int total;
    const int at = before + block_exclusive_scan(need, &total);
    if (i < p.n) {
      p.start[i] = at;
      p.ok[i] = good ? need : -1;
    }
    before += total;
  }
  if (threadIdx.x == 0) p.start[p.n] = before;
  // free pages, as far as they are asked for: they say who gets what before a page is given away
  int got = 0;
  for (int base = 0; base < t.pages && got < before; base += SCAN_THREADS) {
    const int id = base + threadIdx.x;
    got += __syncthreads_count(id < t.pages && t.refs[id] == 0);
  }
  got = min(got, before);
  __syncthreads();
  // the j-th free page goes to the request whose range holds j
  lowest_free(t.refs, t.pages, got, [&](int j, int id) {
    int lo = 0, hi = p.n - 1;   // last i with start[i] <= j: among equal starts the one with a need
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (p.start[mid] <= j) lo = mid; else hi = mid - 1;
    }
    if (p.start[lo + 1] > got) return;   // refused
    const int r = p.req_rows[lo], len = p.req_lens[lo];
    const int col = len / t.page_size + (len % t.page_size != 0) - p.ok[lo] + j - p.start[lo];
    t.table[static_cast<long long>(r) * t.width + col] = id;
    t.refs[id] = 1;
  });
  __syncthreads();
  for (int i = threadIdx.x; i < p.n; i += SCAN_THREADS) {
    const int need = p.ok[i];
    const bool good = need == 0 || (need > 0 && p.start[i + 1] <= got);
    if (good) t.lens[p.req_rows[i]] = p.req_lens[i];
    p.ok[i] = good;
  }
}

// ---------------------------------------------------------------------------
// Fork, step 1 (block 0): a free page for each pair whose parent's last page is partly filled.
// The other blocks copy the tables where the result goes to tables of its own.
// ---------------------------------------------------------------------------
struct ForkParams {
  Tables in, out;            // out may be in
  const int *parents, *children;
  int n;
  int* ok;                   // [n]
  int *src, *dst;            // [n] scratch: the copies of last pages (-1: none)
};

__device__ __forceinline__ void copy_ints(int* to, const int* from, long long n, long long at, long long step) {
  if (to == from) return;
  for (long long i = at; i < n; i += step) to[i] = from[i];
}

__global__ void __launch_bounds__(SCAN_THREADS) kv4_fork_plan_kernel(const ForkParams p) {
  const Tables& t = p.in;
  if (blockIdx.x > 0) {
    const long long at = (blockIdx.x - 1) * static_cast<long long>(SCAN_THREADS) + threadIdx.x;
    const long long step = (gridDim.x - 1) * static_cast<long long>(SCAN_THREADS);
    copy_ints(p.out.refs, t.refs, t.pages, at, step);
    copy_ints(p.out.table, t.table, static_cast<long long>(t.rows) * t.width, at, step);
    copy_ints(p.out.lens, t.lens, t.rows, at, step);
    return;
  }
  // src[i] holds request i's rank among those that need a page until the pages are known
  int before = 0;
  for (int base = 0; base < p.n; base += SCAN_THREADS) {
    const int i = base + threadIdx.x;
    int need = 0, good = 0;
    if (i < p.n) {
      const int a = p.parents[i], c = p.children[i];
      if (a < 0 || a >= t.rows || c < 0 || c >= t.rows) {
        flag_error(kErrIndex);
      } else {
        const int len = t.lens[a];
        if (len < 0 || len / t.page_size + (len % t.page_size != 0) > t.width) {
          flag_error(kErrIndex);
        } else {
          good = 1;
          need = len % t.page_size != 0;
        }
      }
    }
    int total;
    const int at = before + block_exclusive_scan(need, &total);
    if (i < p.n) {
      p.ok[i] = good;
      p.src[i] = need ? at : -1;
      if (need) p.dst[at] = -1;   // rank -> page, filled below
    }
    before += total;
  }
  __syncthreads();
  lowest_free(t.refs, t.pages, before, [&](int j, int id) { p.dst[j] = id; });
  __syncthreads();
  // ranks to pages: dst[rank] is read before dst[i] is written over; rank <= i, so go downwards
  for (int base = (p.n - 1) / SCAN_THREADS * SCAN_THREADS; base >= 0; base -= SCAN_THREADS) {
    const int i = base + threadIdx.x;
    int page = -1, old = -1;
    if (i < p.n && p.src[i] >= 0) {
      page = p.dst[p.src[i]];
      const int a = p.parents[i], len = t.lens[a];
      old = t.table[static_cast<long long>(a) * t.width + len / t.page_size];
      if (page < 0) p.ok[i] = 0;
    }
    __syncthreads();
    if (i < p.n) {
      p.dst[i] = page;
      p.src[i] = page >= 0 ? old : -1;
    }
    __syncthreads();
  }
}

// Fork, step 2: block i < n writes child i's row and counts its pages; the others copy the last pages.
__global__ void __launch_bounds__(COPY_THREADS) kv4_fork_rows_kernel(const ForkParams p, const CopyParams copy) {
  if (blockIdx.x >= static_cast<unsigned>(p.n)) {
    copy_pages(copy, blockIdx.x - p.n, gridDim.x - p.n);
    return;
  }
  const Tables& t = p.out;
  const int i = blockIdx.x;
  const int a = p.parents[i], c = p.children[i];
  if (a < 0 || a >= t.rows || c < 0 || c >= t.rows) return;   // flagged in step 1
  const int len = p.ok[i] ? p.in.lens[a] : 0;
  const int held = len / t.page_size + (len % t.page_size != 0);
  for (int col = threadIdx.x; col < t.width; col += COPY_THREADS) {
    int page = -1;
    if (col < held) {
      page = col == held - 1 && p.dst[i] >= 0 ? p.dst[i] : p.in.table[static_cast<long long>(a) * t.width + col];
      if (page >= 0 && page < t.pages) atomicAdd(t.refs + page, 1);
      else flag_error(kErrIndex);
    }
    t.table[static_cast<long long>(c) * t.width + col] = page;
  }
  if (threadIdx.x == 0) t.lens[c] = len;
}

// ---------------------------------------------------------------------------
// Release: block i gives back the pages of row rows[i] (a row named twice gives them back once).
// ---------------------------------------------------------------------------
struct ReleaseParams {
  Tables t;
  const int* rows;
};

__global__ void __launch_bounds__(256) kv4_release_kernel(const ReleaseParams p) {
  const Tables& t = p.t;
  const int r = p.rows[blockIdx.x];
  if (r < 0 || r >= t.rows) {
    if (threadIdx.x == 0) flag_error(kErrIndex);
    return;
  }
  for (int col = threadIdx.x; col < t.width; col += 256) {
    const int page = atomicExch(t.table + static_cast<long long>(r) * t.width + col, -1);
    if (page >= 0 && page < t.pages) atomicSub(t.refs + page, 1);
    else if (page >= t.pages) flag_error(kErrIndex);
  }
  if (threadIdx.x == 0) t.lens[r] = 0;
}

__global__ void __launch_bounds__(256) kv4_copy_tables_kernel(const Tables in, const Tables out) {
  const long long at = blockIdx.x * 256LL + threadIdx.x, step = gridDim.x * 256LL;
  copy_ints(out.refs, in.refs, in.pages, at, step);
  copy_ints(out.table, in.table, static_cast<long long>(in.rows) * in.width, at, step);
  copy_ints(out.lens, in.lens, in.rows, at, step);
}

// ---------------------------------------------------------------------------
// Compact: with `live` pages in use, the i-th page in use with an id >= live moves to the i-th
// free page with an id < live; pages below `live` stay where they are, so as few pages move as
// can. Step 1 (one block): the moves and the map of ids. Step 2: the first `table_blocks` blocks the
// tables, the others the pages.
// ---------------------------------------------------------------------------
struct CompactParams {
  Tables in, out;
  int* map;                  // [pages]: new id of a page
  int *src, *dst;            // [pages / 2] moves
  int* count;                // [1]
  int table_blocks;
};

__global__ void __launch_bounds__(SCAN_THREADS) kv4_compact_plan_kernel(const CompactParams p) {
  const Tables& t = p.in;
  int live = 0;
  for (int base = 0; base < t.pages; base += SCAN_THREADS) {
    const int id = base + threadIdx.x;
    live += __syncthreads_count(id < t.pages && t.refs[id] > 0);
  }
  int holes = 0, movers = 0;
  for (int base = 0; base < t.pages; base += SCAN_THREADS) {
    const int id = base + threadIdx.x;
    const bool used = id < t.pages && t.refs[id] > 0;
    const int hole = id < live && !used, mover = used && id >= live;
    int total;
    const int at = block_exclusive_scan(hole | (mover << 16), &total);
    if (hole) p.dst[holes + (at & 0xffff)] = id;
    if (mover) p.src[movers + (at >> 16)] = id;
    holes += total & 0xffff;
    movers += total >> 16;
    if (id < t.pages && !mover) p.map[id] = id;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < movers; i += SCAN_THREADS) p.map[p.src[i]] = p.dst[i];
  if (threadIdx.x == 0) *p.count = movers;
  __syncthreads();
  // reference counts: read all, then write, chunk by chunk (out may be in: a mover's new place
  // lies below `live` and was free, so its count is not read again)
  for (int base = 0; base < t.pages; base += SCAN_THREADS) {
    const int id = base + threadIdx.x;
    const int r = id < t.pages ? t.refs[id] : 0;
    __syncthreads();
    if (id < t.pages && id < live && r > 0) p.out.refs[id] = r;
    if (id >= live && id < t.pages) {
      if (r > 0) p.out.refs[p.map[id]] = r;
      p.out.refs[id] = 0;
    }
  }
}

__global__ void __launch_bounds__(COPY_THREADS) kv4_compact_tables_kernel(const CompactParams p, const CopyParams copy) {
  if (blockIdx.x >= static_cast<unsigned>(p.table_blocks)) {
    copy_pages(copy, blockIdx.x - p.table_blocks, gridDim.x - p.table_blocks);
    return;
  }
  const Tables& t = p.in;
  const long long n = static_cast<long long>(t.rows) * t.width;
  const long long at = blockIdx.x * static_cast<long long>(COPY_THREADS) + threadIdx.x;
  const long long step = p.table_blocks * static_cast<long long>(COPY_THREADS);
  for (long long i = at; i < n; i += step) {
    int page = t.table[i];
    if (page >= t.pages) {
      flag_error(kErrIndex);
    } else if (page >= 0) {
      page = p.map[page];
    }
    p.out.table[i] = page;
  }
  copy_ints(p.out.lens, t.lens, t.rows, at, step);
}

}  // namespace kv4
}  // namespace w4a16
