// The pages of a paged cache (dsv4_pages of dsv4.h): handing them out, giving them back, branching a
// sequence and closing the gaps. A page belongs to as many sequences as its count says; 0 is free.
// Full pages of a branch are shared, because nothing is ever written to a full page again; the
// partly filled last page is copied, so a sequence always writes to pages of its own.
//
// Every step runs on the device, on the caller's stream, without a host round trip, and gives the
// same tables for the same input: free pages are handed out from the lowest index up, in the order
// of the call. One CTA makes the plan (the pages are counted with ballots and a block scan, no
// atomics decide an order), the copies run on the whole GPU and are bound by HBM. Measured: eight branches of
// a slot with 16384 entries (136 MB written) 39 us, of which 27 the copy; 1991 of 8192 pages of 64 rows moved
// (261 MB read and written) 38 us, 6.8 TB/s, behind a plan of 8 us; small calls 7 to 11 us, two or three
// launches.
#include <algorithm>

#include "common.cuh"

namespace dsv4 {
namespace pg {

constexpr int PLAN = 1024;                // threads of a planning CTA
constexpr int COPY = 256;                 // threads of a copying CTA
constexpr int UNIT = 16384;               // bytes a copying CTA takes at a time: four 16-byte loads a thread in flight
constexpr int SEGS = 8;                   // parts of a branch (fork_job)

// exclusive sum of v over the CTA's threads in order; *total the whole sum. Ends with a barrier.
__device__ __forceinline__ int block_scan(int v, int* total) {
  __shared__ int warps[33];
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  int s = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int x = __shfl_up_sync(0xffffffffu, s, o);
    if (lane >= o) s += x;
  }
  if (lane == 31) warps[w] = s;
  __syncthreads();
  if (w == 0) {
    int x = lane < (blockDim.x >> 5) ? warps[lane] : 0;
    int y = x;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int z = __shfl_up_sync(0xffffffffu, y, o);
      if (lane >= o) y += z;
    }
    warps[lane] = y - x;
    if (lane == 31) warps[32] = y;
  }
  __syncthreads();
  const int r = warps[w] + s - v;
  *total = warps[32];
  __syncthreads();
  return r;
}

// The lowest `want` free pages in ascending order into out; returns how many there are (at most want).
__device__ __forceinline__ int lowest_free(const int32_t* refs, int n_pages, int want, int32_t* out) {
  int have = 0;
  for (int base = 0; base < n_pages && have < want; base += PLAN) {  // uniform over the CTA
    const int i = base + threadIdx.x;
    const bool free = i < n_pages && refs[i] == 0;
    int total;
    const int r = have + block_scan(free ? 1 : 0, &total);
    if (free && r < want) out[r] = i;
    have += total;
  }
  __syncthreads();
  return have < want ? have : want;
}

// one CTA per sequence: its pages given back (its count lowered), its table row emptied. Bound by two
// dependent reads (the row, then nothing waits for the counts).
__global__ void __launch_bounds__(COPY) free_kernel(dsv4_pages p, const int32_t* seqs, int n) {
  pdl_wait();
  pdl_trigger();
  const int k = blockIdx.x, s = seqs[k];
  bool skip = s < 0 || s >= p.slots;
  if (skip && threadIdx.x == 0) raise_device_error(DSV4_ERR_INDEX_OUT_OF_RANGE);
  for (int i = threadIdx.x; i < k; i += COPY) skip |= seqs[i] == s;  // a sequence named twice gives its pages back once
  if (__syncthreads_or(skip)) return;
  for (int j = threadIdx.x; j < p.bt_stride; j += COPY) {
    int32_t* cell = p.block_table + static_cast<int64_t>(s) * p.bt_stride + j;
    const int32_t pg = *cell;
    *cell = -1;
    if (pg >= 0 && pg < p.n_pages) atomicSub(p.refs + pg, 1);
  }
}

// pages of its own for the entries of `tokens[k] + add` tokens of sequence seqs[k]; a sequence that
// finds too few free pages gets none of them (DSV4_ERR_NO_PAGES on the error word), and those behind it are
// served from what it leaves. There are enough pages for all almost always, and then a scan hands them out; one
// thread goes through the sequences in order where there are not.
__global__ void __launch_bounds__(PLAN) reserve_kernel(dsv4_pages p, const int32_t* seqs, const int32_t* tokens, int add,
                                                       int n, int32_t* free_list) {
  pdl_wait();
  pdl_trigger();
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  __shared__ int want[PLAN], held[PLAN], from[PLAN];
  for (int base = 0; base < n; base += PLAN) {  // PLAN sequences at a time
    const int m = min(PLAN, n - base);
    for (int k = w; k < m; k += PLAN / 32) {
      const int s = seqs ? seqs[base + k] : base + k;
      int need = 0, have = 0;
      // a sequence named twice asks once, by its first mention, for the largest count (and again among the next
      // PLAN, for what it does not have by then)
      bool again = false;
      int count = tokens[base + k];
      if (seqs != nullptr)
        for (int i = lane; i < m; i += 32)
          if (seqs[base + i] == s) {
            again |= i < k;
            count = max(count, tokens[base + i]);
          }
      again = __any_sync(0xffffffffu, again);
      count = __reduce_max_sync(0xffffffffu, count);
      if (s >= 0 && s < p.slots) {
        const int64_t all = max(static_cast<int64_t>(0), static_cast<int64_t>(count) + add) / p.ratio;
        if (all > p.max_comp && lane == 0) raise_device_error(DSV4_ERR_INDEX_OUT_OF_RANGE);
        const int e = static_cast<int>(min(all, static_cast<int64_t>(p.max_comp)));
        need = (e + p.page - 1) / p.page;
        // pages fill a row from the left
        for (int j = lane; j < p.bt_stride; j += 32)
          have += p.block_table[static_cast<int64_t>(s) * p.bt_stride + j] >= 0;
        have = __reduce_add_sync(0xffffffffu, have);
      } else if (lane == 0) {
        raise_device_error(DSV4_ERR_INDEX_OUT_OF_RANGE);
      }
      if (lane == 0) {
        want[k] = again ? 0 : max(0, need - have);
        held[k] = have;
      }
    }
    __syncthreads();
    int total;
    const int mine = threadIdx.x < m ? want[threadIdx.x] : 0;
    const int at = block_scan(mine, &total);
    if (total == 0) continue;  // uniform
    const int got = lowest_free(p.refs, p.n_pages, total, free_list);
    from[threadIdx.x] = at;
    __syncthreads();
    if (got < total && threadIdx.x == 0) {
      for (int k = 0, used = 0; k < m; ++k) {
        const bool fits = want[k] <= got - used;
        from[k] = fits ? used : -1;
        if (fits) used += want[k];
      }
    }
    __syncthreads();
    if (mine > 0) {
      const int first = from[threadIdx.x];
      if (first < 0) {
        raise_device_error(DSV4_ERR_NO_PAGES);
      } else {
        const int s = seqs ? seqs[base + threadIdx.x] : base + static_cast<int>(threadIdx.x);
        for (int j = 0; j < mine; ++j) {
          const int32_t pg = free_list[first + j];
          p.block_table[static_cast<int64_t>(s) * p.bt_stride + held[threadIdx.x] + j] = pg;
          p.refs[pg] = 1;
        }
      }
    }
    __syncthreads();
  }
}

// ---- a branch: what one (src, dst) pair copies
struct Fork {
  int32_t src, dst, entries, ok;
  int32_t from, to;    // the partly filled last page and its copy, -1: none
  int32_t lead, next;  // the first branch that copies the same, the one after this, -1: none
};

struct Part {
  const uint8_t* src;
  uint8_t* dst;
  int64_t bytes;
};
__device__ __forceinline__ int64_t part_bytes(const dsv4_pages& p, const Fork& f, int s) {
  const int64_t tiles = (f.entries + 127) / 128;
  switch (s) {
    case 0: return p.k_idx ? static_cast<int64_t>(f.entries) * p.idx_dim * 4 : 0;
    case 1: return p.key_image ? tiles * DSV4_KEY_TILE_BYTES : 0;
    case 2: return p.key_image ? tiles * 512 : 0;
    case 3: return static_cast<int64_t>(p.window) * p.head_dim * 2;
    case 4:
    case 5: return p.ring_kv ? static_cast<int64_t>(4) * p.ratio * p.head_dim * 4 : 0;
    case 6:
    case 7: return p.ring_k_idx ? static_cast<int64_t>(4) * p.ratio * p.idx_dim * 4 : 0;
    default: return f.from >= 0 ? static_cast<int64_t>(f.entries % p.page) * p.head_dim * 2 : 0;
  }
}
__device__ __forceinline__ Part part(const dsv4_pages& p, const Fork& f, int s) {
  const int64_t all = (p.max_comp + 127) / 128;
  uint8_t* base = nullptr;
  int64_t from = f.src, to = f.dst, stride = 0;
  switch (s) {
    case 0: base = reinterpret_cast<uint8_t*>(p.k_idx), stride = static_cast<int64_t>(p.max_comp) * p.idx_dim * 4; break;
    case 1: base = p.key_image, stride = all * DSV4_KEY_TILE_BYTES; break;
    case 2: base = reinterpret_cast<uint8_t*>(p.key_inv), stride = all * 512; break;
    case 3:
      base = reinterpret_cast<uint8_t*>(p.pool), stride = static_cast<int64_t>(p.head_dim) * 2;
      from = p.win_base[f.src], to = p.win_base[f.dst];
      break;
    case 4: base = reinterpret_cast<uint8_t*>(p.ring_kv), stride = static_cast<int64_t>(4) * p.ratio * p.head_dim * 4; break;
    case 5: base = reinterpret_cast<uint8_t*>(p.ring_score), stride = static_cast<int64_t>(4) * p.ratio * p.head_dim * 4; break;
    case 6: base = reinterpret_cast<uint8_t*>(p.ring_k_idx), stride = static_cast<int64_t>(4) * p.ratio * p.idx_dim * 4; break;
    case 7: base = reinterpret_cast<uint8_t*>(p.ring_s_idx), stride = static_cast<int64_t>(4) * p.ratio * p.idx_dim * 4; break;
    default:
      base = reinterpret_cast<uint8_t*>(p.pool) + p.comp_base * p.head_dim * 2;
      stride = static_cast<int64_t>(p.page) * p.head_dim * 2;
      from = f.from, to = f.to;
  }
  return {base + from * stride, base + to * stride, part_bytes(p, f, s)};
}

// workspace of a fork: forks [n], then the running number of copy units before each (fork, part)
// [n * (SEGS + 1) + 1], then the free pages found [n]
__device__ __forceinline__ int64_t* unit_starts(Fork* forks, int n) { return reinterpret_cast<int64_t*>(forks + n); }

__global__ void __launch_bounds__(PLAN) fork_plan_kernel(dsv4_pages p, const int32_t* src, const int32_t* dst,
                                                         const int32_t* tokens, int n, Fork* forks, int32_t* free_list) {
  pdl_wait();
  pdl_trigger();
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  int64_t* starts = unit_starts(forks, n);
  // a warp per branch: what it asks for, and whether it may have it
  for (int k = w; k < n; k += PLAN / 32) {
    const int a = src[k], b = dst[k];
    const int e = p.max_comp == 0 ? 0 : tokens[k] / p.ratio;  // a window-only cache has rings alone
    int bad = 0;
    if (a < 0 || a >= p.slots || b < 0 || b >= p.slots || a == b || tokens[k] < 0 || e > p.max_comp) {
      bad = 1;
    } else {
      const int pages = (e + p.page - 1) / p.page;
      // every page of the source there, the branch's row empty, and no slot written twice or read after
      const int32_t *ra = p.block_table + static_cast<int64_t>(a) * p.bt_stride;
      const int32_t *rb = p.block_table + static_cast<int64_t>(b) * p.bt_stride;
#pragma unroll 8
      for (int j = lane; j < p.bt_stride; j += 32) {
        const int32_t pg = ra[j], own = rb[j];
        bad |= (j < pages && (pg < 0 || pg >= p.n_pages)) | (own >= 0);
      }
      for (int i = lane; i < n; i += 32) bad |= (i < k && dst[i] == b) || src[i] == b;
    }
    bad = __any_sync(0xffffffffu, bad);
    if (lane == 0) {
      if (bad) raise_device_error(DSV4_ERR_INDEX_OUT_OF_RANGE);
      forks[k] = {a, b, e, bad ? 0 : 1, -1, -1, 0, -1};
    }
  }
  __syncthreads();
  // the last pages: ranks in the order of the call
  int asked = 0;
  for (int base = 0; base < n; base += PLAN) {
    const int k = base + threadIdx.x;
    const bool t = k < n && forks[k].ok && forks[k].entries % p.page != 0;
    int total;
    const int r = block_scan(t ? 1 : 0, &total);
    if (t) forks[k].to = asked + r;
    asked += total;
  }
  __syncthreads();
  const int got = asked ? lowest_free(p.refs, p.n_pages, asked, free_list) : 0;
  for (int k = threadIdx.x; k < n; k += PLAN) {
    Fork f = forks[k];
    if (f.ok && f.to >= 0) {
      if (f.to >= got) {
        raise_device_error(DSV4_ERR_NO_PAGES);
        f.ok = 0;
        f.to = -1;
      } else {
        f.to = free_list[f.to];
        f.from = p.block_table[static_cast<int64_t>(f.src) * p.bt_stride + f.entries / p.page];
        p.refs[f.to] = 1;
        p.block_table[static_cast<int64_t>(f.dst) * p.bt_stride + f.entries / p.page] = f.to;
      }
      forks[k] = f;
    }
    if (f.ok && p.key_norm_max) p.key_norm_max[f.dst] = p.key_norm_max[f.src];
  }
  __syncthreads();
  for (int k = w; k < n; k += PLAN / 32) {
    const Fork f = forks[k];
    if (!f.ok) continue;
    // the other branches of what this one copies
    bool before = false;
    int next = -1;
    for (int i0 = 0; i0 < n && next < 0; i0 += 32) {
      const int i = i0 + lane;
      const bool same = i < n && forks[i].ok && forks[i].src == f.src && forks[i].entries == f.entries;
      before |= __any_sync(0xffffffffu, same && i < k);
      const uint32_t after = __ballot_sync(0xffffffffu, same && i > k);
      if (after != 0) next = i0 + __ffs(after) - 1;
    }
    if (lane == 0) {
      forks[k].lead = !before;
      forks[k].next = next;
    }
    const int32_t* ra = p.block_table + static_cast<int64_t>(f.src) * p.bt_stride;
    int32_t* rb = p.block_table + static_cast<int64_t>(f.dst) * p.bt_stride;
    const int full = f.entries / p.page;
    for (int j0 = lane; j0 < full; j0 += 8 * 32) {
      int32_t pg[8];
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (j0 + 32 * i < full) pg[i] = ra[j0 + 32 * i];
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (j0 + 32 * i < full) {
          rb[j0 + 32 * i] = pg[i];
          atomicAdd(p.refs + pg[i], 1);
        }
    }
  }
  __syncthreads();
  // copy units before each part
  int64_t before = 0;
  const int parts = n * (SEGS + 1);
  for (int base = 0; base < parts; base += PLAN) {
    const int i = base + threadIdx.x;
    int units = 0;
    if (i < parts && forks[i / (SEGS + 1)].lead)
      units = static_cast<int>((part_bytes(p, forks[i / (SEGS + 1)], i % (SEGS + 1)) + UNIT - 1) / UNIT);
    int total;
    const int r = block_scan(units, &total);
    if (i < parts) starts[i] = before + r;
    before += total;
  }
  if (threadIdx.x == 0) starts[parts] = before;
}

// up to UNIT bytes (a multiple of 16): all of a thread's loads before its first store
struct Piece {
  uint4 v[UNIT / 16 / COPY];
  __device__ __forceinline__ void load(const uint8_t* src, int bytes) {
    const uint4* s = reinterpret_cast<const uint4*>(src) + threadIdx.x;
    const int n16 = bytes / 16 - static_cast<int>(threadIdx.x);
#pragma unroll
    for (int i = 0; i < UNIT / 16 / COPY; ++i)
      if (i * COPY < n16) v[i] = __ldcs(s + i * COPY);
  }
  __device__ __forceinline__ void store(uint8_t* dst, int bytes) const {
    uint4* d = reinterpret_cast<uint4*>(dst) + threadIdx.x;
    const int n16 = bytes / 16 - static_cast<int>(threadIdx.x);
#pragma unroll
    for (int i = 0; i < UNIT / 16 / COPY; ++i)
      if (i * COPY < n16) __stcs(d + i * COPY, v[i]);
  }
};

// A CTA takes neighbouring units: it looks its first part up and walks on from there. A unit is read once for
// all branches of it (eight branches of 16384 entries: 30.7 us when each read it, with HBM at 40%). No early launch of
// the next kernel: the decode attention reads window rows before it waits for the kernel before it.
__global__ void __launch_bounds__(COPY) fork_copy_kernel(dsv4_pages p, int n, Fork* forks) {
  pdl_wait();
  const int64_t* starts = unit_starts(forks, n);
  const int parts = n * (SEGS + 1);
  const int64_t units = starts[parts];
  const int64_t u1 = units * (blockIdx.x + 1) / gridDim.x;
  int64_t u = units * blockIdx.x / gridDim.x;
  if (u >= u1) return;
  int lo = 0, hi = parts - 1;  // the last part that starts at or before u (parts without units are passed over)
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (starts[mid] <= u)
      lo = mid;
    else
      hi = mid - 1;
  }
  while (u < u1) {
    while (starts[lo + 1] <= u) ++lo;  // u < units = starts[parts]
    const int lead = lo / (SEGS + 1), seg = lo % (SEGS + 1);
    const Part q = part(p, forks[lead], seg);
    const int64_t first = starts[lo], end = min(starts[lo + 1], u1);
    for (; u < end; ++u) {
      const int64_t off = (u - first) * UNIT;
      const int bytes = static_cast<int>(min(static_cast<int64_t>(UNIT), q.bytes - off));
      Piece x;
      x.load(q.src + off, bytes);
      x.store(q.dst + off, bytes);
      for (int k = forks[lead].next; k >= 0; k = forks[k].next) x.store(part(p, forks[k], seg).dst + off, bytes);
    }
  }
}

// ---- compaction: the k-th free page below the number of pages in use takes the k-th page in use above it.
// With live(i) pages in use before page i and nl in all, the free page i < nl is the (i - live(i))-th, and the
// used page i >= nl the (live(i) - live(nl))-th: one scan ranks both. holes[k] is the k-th of the first,
// movers[live(i)] = i of the second, so that movers[nl - n_moves + k] goes to holes[k]. (A scan each took 11.0 us
// for 8192 pages.)
__global__ void __launch_bounds__(PLAN) compact_plan_kernel(dsv4_pages p, int32_t* n_live, int32_t* holes, int32_t* movers,
                                                            int32_t* to, int32_t* n_moves) {
  pdl_wait();
  pdl_trigger();
  __shared__ int live_nl;  // live(nl)
  // a stretch of pages per thread, in order
  const int per = (p.n_pages + PLAN - 1) / PLAN;
  const int i0 = min(p.n_pages, per * static_cast<int>(threadIdx.x)), i1 = min(p.n_pages, i0 + per);
  int live = 0;
#pragma unroll 8
  for (int i = i0; i < i1; ++i) live += p.refs[i] > 0;
  int nl;
  live = block_scan(live, &nl);
  if (threadIdx.x == 0 && nl == p.n_pages) live_nl = nl;
#pragma unroll 8
  for (int i = i0; i < i1; ++i) {
    const bool used = p.refs[i] > 0;
    if (i == nl) live_nl = live;
    if (used && i >= nl) movers[live] = i;
    if (!used) {
      if (i < nl) holes[i - live] = i;
      to[i] = -1;  // for a cell that names a page which is not counted
    }
    live += used;
  }
  __syncthreads();
  const int nm = nl - live_nl;
  for (int k = threadIdx.x; k < nm; k += PLAN) {
    const int a = movers[live_nl + k], b = holes[k];
    p.refs[b] = p.refs[a];
    p.refs[a] = 0;
    to[a] = b;
  }
  if (threadIdx.x == 0) {
    *n_live = nl;
    *n_moves = nm;
  }
}

__global__ void __launch_bounds__(COPY) compact_copy_kernel(dsv4_pages p, const int32_t* n_live, const int32_t* holes,
                                                            const int32_t* movers, const int32_t* to,
                                                            const int32_t* n_moves) {
  pdl_wait();
  pdl_trigger();
  const int64_t bytes = static_cast<int64_t>(p.page) * p.head_dim * 2;
  const int nl = *n_live, nm = *n_moves;
  const int64_t per = (bytes + UNIT - 1) / UNIT, units = nm * per;
  uint8_t* base = reinterpret_cast<uint8_t*>(p.pool) + p.comp_base * p.head_dim * 2;
  for (int64_t u = blockIdx.x; u < units; u += gridDim.x) {
    const int64_t k = u / per, off = (u - k * per) * UNIT;
    const int some = static_cast<int>(min(static_cast<int64_t>(UNIT), bytes - off));
    Piece x;
    x.load(base + movers[nl - nm + k] * bytes + off, some);
    x.store(base + holes[k] * bytes + off, some);
  }
  const int64_t cells = static_cast<int64_t>(p.slots) * p.bt_stride;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * COPY + threadIdx.x; i < cells;
       i += static_cast<int64_t>(gridDim.x) * COPY) {
    const int32_t pg = p.block_table[i];
    if (pg >= nl && pg < p.n_pages) p.block_table[i] = to[pg];
  }
}

DSV4_ERROR_READER(pages)

static int check_pages(const dsv4_pages* p, const char* who) {
  DSV4_CHECK_ARG(p && p->pool && p->win_base && (p->max_comp == 0 || (p->block_table && p->refs)),
                 "%s: NULL pointer in the cache", who);
  DSV4_CHECK_ARG(p->slots > 0 && p->n_pages >= 0 && p->page > 0 && p->max_comp >= 0 && p->ratio > 0 && p->window > 0 &&
                     (p->max_comp == 0 ? p->bt_stride == 0 && p->n_pages == 0
                                       : p->bt_stride * static_cast<int64_t>(p->page) >= p->max_comp) &&
                     p->comp_base >= 0,
                 "%s: bad sizes", who);
  DSV4_CHECK_ARG(p->head_dim > 0 && p->head_dim % 8 == 0 && p->idx_dim >= 0 && p->idx_dim % 4 == 0,
                 "%s: rows must be a multiple of 16 bytes", who);
  DSV4_CHECK_ARG(p->key_image == nullptr || (p->key_inv && p->key_norm_max), "%s: a key image has three parts", who);
  DSV4_CHECK_ARG((p->ring_kv == nullptr) == (p->ring_score == nullptr) &&
                     (p->ring_k_idx == nullptr) == (p->ring_s_idx == nullptr),
                 "%s: a compressor ring has two parts", who);
  const void* all[] = {p->pool, p->k_idx, p->key_image, p->key_inv, p->ring_kv, p->ring_score, p->ring_k_idx, p->ring_s_idx};
  for (const void* q : all)
    DSV4_CHECK_ARG((reinterpret_cast<uintptr_t>(q) & 15) == 0, "%s: tensors must be 16-byte aligned", who);
  return DSV4_OK;
}

}  // namespace pg
}  // namespace dsv4

using namespace dsv4;
using pg::Fork;

extern "C" {

size_t dsv4_pages_workspace_size(const dsv4_pages* p, int32_t n) {
  if (p == nullptr || n < 0 || p->n_pages < 0) return 0;
  // a fork's plan, the free pages of a reservation, or a compaction's lists and new places
  const size_t fork = static_cast<size_t>(n) * (sizeof(Fork) + (pg::SEGS + 1) * 8 + 4) + 8;
  const size_t lists = (3 * static_cast<size_t>(p->n_pages) + 1) * 4;
  return (std::max(fork, lists) + 15) / 16 * 16;
}

int dsv4_pages_free(const dsv4_pages* p, const int32_t* seqs, int32_t n, void* stream) {
  const int rc = pg::check_pages(p, "dsv4_pages_free");
  if (rc != DSV4_OK) return rc;
  DSV4_CHECK_ARG(n >= 0 && (n == 0 || seqs), "dsv4_pages_free: NULL sequences");
  if (n == 0) return DSV4_OK;
  DSV4_CUDA_CHECK(launch_pdl(pg::free_kernel, dim3(n), dim3(pg::COPY), 0, as_stream(stream), *p, seqs, n));
  return DSV4_OK;
}

int dsv4_pages_reserve(const dsv4_pages* p, const int32_t* seqs, const int32_t* tokens, int32_t add, int32_t n,
                       void* workspace, size_t workspace_bytes, void* stream) {
  const int rc = pg::check_pages(p, "dsv4_pages_reserve");
  if (rc != DSV4_OK) return rc;
  DSV4_CHECK_ARG(n >= 0 && (n == 0 || tokens) && (seqs || n <= p->slots), "dsv4_pages_reserve: bad sequences");
  if (n == 0 || p->max_comp == 0) return DSV4_OK;
  if (workspace == nullptr || workspace_bytes < dsv4_pages_workspace_size(p, n)) {
    set_error("dsv4_pages_reserve: workspace missing or too small");
    return DSV4_ERR_WORKSPACE;
  }
  DSV4_CUDA_CHECK(launch_pdl(pg::reserve_kernel, dim3(1), dim3(pg::PLAN), 0, as_stream(stream), *p, seqs, tokens, add, n,
                             reinterpret_cast<int32_t*>(workspace)));
  return DSV4_OK;
}

int dsv4_pages_fork(const dsv4_pages* p, const int32_t* src, const int32_t* dst, const int32_t* tokens, int32_t n,
                    void* workspace, size_t workspace_bytes, void* stream) {
  const int rc = pg::check_pages(p, "dsv4_pages_fork");
  if (rc != DSV4_OK) return rc;
  DSV4_CHECK_ARG(n >= 0 && n <= p->slots && (n == 0 || (src && dst && tokens)), "dsv4_pages_fork: bad sequences");
  if (n == 0) return DSV4_OK;
  if (workspace == nullptr || workspace_bytes < dsv4_pages_workspace_size(p, n) ||
      (reinterpret_cast<uintptr_t>(workspace) & 15) != 0) {
    set_error("dsv4_pages_fork: workspace missing, too small or not 16-byte aligned");
    return DSV4_ERR_WORKSPACE;
  }
  Fork* forks = reinterpret_cast<Fork*>(workspace);
  int32_t* free_list = reinterpret_cast<int32_t*>(reinterpret_cast<uint8_t*>(workspace) + static_cast<size_t>(n) * sizeof(Fork) +
                                                  (static_cast<size_t>(n) * (pg::SEGS + 1) + 1) * 8);
  DSV4_CUDA_CHECK(launch_pdl(pg::fork_plan_kernel, dim3(1), dim3(pg::PLAN), 0, as_stream(stream), *p, src, dst, tokens, n,
                             forks, free_list));
  DSV4_CUDA_CHECK(launch_pdl(pg::fork_copy_kernel, dim3(8 * num_sms()), dim3(pg::COPY), 0, as_stream(stream), *p, n, forks));
  return DSV4_OK;
}

int dsv4_pages_compact(const dsv4_pages* p, int32_t* n_live, void* workspace, size_t workspace_bytes, void* stream) {
  const int rc = pg::check_pages(p, "dsv4_pages_compact");
  if (rc != DSV4_OK) return rc;
  DSV4_CHECK_ARG(n_live, "dsv4_pages_compact: NULL n_live");
  if (workspace == nullptr || workspace_bytes < dsv4_pages_workspace_size(p, 0)) {
    set_error("dsv4_pages_compact: workspace missing or too small");
    return DSV4_ERR_WORKSPACE;
  }
  int32_t* holes = reinterpret_cast<int32_t*>(workspace);
  int32_t *movers = holes + p->n_pages, *to = movers + p->n_pages, *n_moves = to + p->n_pages;
  DSV4_CUDA_CHECK(launch_pdl(pg::compact_plan_kernel, dim3(1), dim3(pg::PLAN), 0, as_stream(stream), *p, n_live, holes, movers,
                             to, n_moves));
  DSV4_CUDA_CHECK(launch_pdl(pg::compact_copy_kernel, dim3(8 * num_sms()), dim3(pg::COPY), 0, as_stream(stream), *p,
                             static_cast<const int32_t*>(n_live), static_cast<const int32_t*>(holes),
                             static_cast<const int32_t*>(movers), static_cast<const int32_t*>(to),
                             static_cast<const int32_t*>(n_moves)));
  return DSV4_OK;
}

}  // extern "C"
