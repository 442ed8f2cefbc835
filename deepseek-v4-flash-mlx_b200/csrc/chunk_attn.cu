// Attention of a chunk of new tokens over the paged cache, every token over its window and all of its
// compressed rows (the list of oracle/decode_engine.py:110-116), on the 5th-generation tensor cores.
//
// All 64 heads share the 512-wide row that is both key and value, so the tokens of a chunk are rows of
// one matrix: two neighbouring tokens times 64 heads are the M = 128 rows of a CTA pair
// (cta_group::2), one token in each CTA, against tiles of 128 cached rows:
//   S[row, j]   = Q[row, :] . K[j, :]        M = 128, N = 128, K = 512   (tensor memory, two buffers)
//   P[row, j]   = 2^(S * scale * log2 e - m[row])  as bf16               (shared memory, two buffers)
//   O[row, :]  += P[row, :] . K[:, :]        M = 128, N = 2 x 256, K = 128 (tensor memory, 256 columns)
// A pair because of space: O alone is 128 KB a token. M = 128 over two CTAs gives each CTA its 64 rows
// with the columns folded over the 128 TMEM lanes (lane l: row l % 64, columns of half l / 64), so O
// takes 256 of the 512 TMEM columns and two S buffers 128; and each operand tile is brought into the
// pair once for S and half of it once more for O, not twice into each CTA:
//   as K (N = 128 rows, split over the pair): CTA r holds rows 64 r .. 64 r + 63, all 512 dims;
//   as V (N = 512 dims, split over the pair): CTA r holds dims 256 r .., all 128 rows.
// A tile buffer has two 32 KB slots, X and Y. For S the CTA's own 64 rows are in X (dims 0-255) and Y
// (dims 256-511). For O X holds rows 0-63 and Y rows 64-127 of the CTA's dims: of the two slots one is
// already that (X in CTA 0, Y in CTA 1), the other is loaded again once S has been computed. 96 KB per
// tile and CTA instead of 128, and two tiles fit beside Q (64 KB) and P (2 x 16 KB).
//
// Rows come in halves of 64: the ring's rows of before the chunk, in slot order; the staged rows of
// the chunk itself; the compressed entries, page by page. Every half is a run of the pool, so TMA
// brings it in (boxes of min(64, the power of two that divides the page) rows), coordinates past the
// pool for what is not there (TMA fills zeros). Visibility is a 64-bit mask per half and token. Rows
// that neither token of the pair sees are zeroed in shared memory before they are used as values, so
// that whatever they hold stays out. A row that one of the two sees alone (the window's oldest, the second
// token's own, the entry that it completes) is a value of both, with a weight of 0 for the other: what of it
// is not finite is zeroed too, by the warp that loads V, which knows these rows for the whole unit (2,048 tokens at
// 16,384 at full clock: 948 us, 933 without; in the softmax warps, whichever way it was written, 960 to 978, in a
// warp of its own 970, since one more that looks at a barrier slows the others). The token that sees the row has it
// from its scores, which are not finite either; a head that scores it -inf weighs it 0 and leaves it out.
//
// The kernel is persistent: a cluster takes pairs of tokens from a static list, the longest first, and
// the next pair's loads and S run under the last pair's epilogue.
// Roles (13 warps a CTA): in CTA 0 one thread of warp 0 issues the S MMAs, a quarter (two slabs of a slot)
// as its rows arrive, and one of warp 12 the O MMAs; an O frees the buffer quarter by quarter, in the order
// in which the next S takes them. (One thread for both that looked at two barriers in turn lost 300 cycles
// and more at each look: the MMAs keep shared memory busy, and a look waits for it.) Warps 1 and 2 load Q
// and the tiles as K, a slot each (one warp for both: 1.04 instead of 0.97 ms for 2048 tokens at position 16384); warp 3
// loads the second slot as V; warps 4-11 softmax and epilogue (warp w: TMEM lanes 32 (w % 4) .., half of the
// columns). The running maximum is lazy (raised only when a score passes it by 2^8; O and the sums are then
// rescaled), the sums are fp32. P is rounded to bf16 (the MMA takes both operands in the rows' type), O is
// rounded once at the end.
// Long lists with few tokens are split over clusters; fp32 partials and a merging kernel follow.
// All waits inside a CTA are bounded (1 s): DSV4_ERR_WAIT_TIMEOUT, and the pair drains and leaves.
//
// Measured on a B200: 2048 tokens at position 16384 (1.2 TFLOP) take 0.95 ms at full clock, 1.27 PFLOP/s or 0.76 of a
// large library product's burst rate, with the tensor pipe active 72% of the time and HBM at 3%; 1.03 ms under the power
// cap (1545 MHz), 0.83 of the same product's sustained rate. A tile's MMAs take 2093 cycles and a tile 2900: of
// two buffers one is being refilled (a load's latency, S behind the other tile's O, softmax), and a third does
// not fit. A pair of tokens costs 7000 cycles beside its tiles (the last O, the epilogue, the next unit's first
// softmax, by the same warps). Few tokens are bound by latency: 32 at position 2048 take 17.9 us and one at
// 65536 17.0 us (16 MB of rows, 2.6 us of HBM), of which the launch and the first rows are 5, the partials'
// stores 1 (an SM writes 32 bytes a cycle; 17.8 us when one CTA of the pair stored them all) and the merging
// kernel 6.
#include <cudaTypedefs.h>

#include <algorithm>
#include <atomic>

#include "chunk.cuh"
#include "common.cuh"
#include "tcgen05.cuh"

namespace dsv4 {
namespace ca {

using namespace tc5;

constexpr int D = 512, HB = 64, BN = 128;
constexpr int SMX_WARPS = 8, SMX_THREADS = 256, THREADS = 416;
constexpr int SLAB = 64 * 128;           // 64 rows of 64 bf16 dims, 128-byte swizzled
constexpr int SLOT = 4 * SLAB;           // 64 rows of 256 dims
constexpr int TMEM_COLS = 512, COL_O = 0, COL_S = 256;
constexpr int MAX_WINDOW = 1024;         // the ring's halves are kept as 4-bit numbers
constexpr float LOG2E = 1.4426950408889634f;
constexpr float RESCALE = 8.0f;          // log2 units a score may pass the running maximum by

struct Smem {
  uint8_t q[8 * SLAB];
  uint8_t kv[2][2][SLOT];                // [tile buffer][X, Y]
  uint8_t p[2][2 * SLAB];                // [buffer][rows 0-63 of the tile, rows 64-127]
  float red[4][HB];
  uint64_t fin[2], q_full, o_free, kv_full[2][4], kv_free[2][4], s_full[2], p_full[2], v_full[2];
  uint32_t tmem_base;
  int abort;
  volatile int unit_tiles[2];            // tiles of a unit, handed to the S thread with its Q; -1: no more
};
static_assert(sizeof(Smem) + 1024 <= 232448, "shared memory above the 227 KB a CTA may opt into");

// Division by a number of the call, as a product: floor(x / d) = x * ceil(2^(31 + s) / d) >> (31 + s) for
// 0 <= x < 2^31 and s = ceil(log2 d): the rounding up adds less than x / 2^(31 + s) < 2^-s <= 1 / d to the quotient.
// (A division takes over 100 cycles, and a unit needs a dozen before its first load: 2000 of 5000 cycles.)
struct Div {
  uint32_t mul;
  int32_t d, shift;
  Div() = default;
  explicit Div(int by) : d(by), shift(31) {
    while ((1LL << (shift - 31)) < by) ++shift;
    mul = static_cast<uint32_t>(((1ULL << shift) + by - 1) / by);
  }
  __device__ __forceinline__ int quot(int x) const {
    return static_cast<int>(static_cast<uint64_t>(static_cast<uint32_t>(x)) * mul >> shift);
  }
  __device__ __forceinline__ int rem(int x) const { return x - quot(x) * d; }
};

struct Params {
  CUtensorMap pool;  // [pool_rows, 512] bf16, box 64 dims x box_rows
  CUtensorMap q;     // [total * 64, 512] bf16, box 64 dims x 64 rows
  CUtensorMap o;     // out, if bf16 and not split: as q
  dsv4_chunk c;
  const float* sink;
  void* out;
  float* part;       // splits > 1: O [total][splits][512 / 4][64 heads][4 dims], then (m, l) [total][splits][64][2]
  const float* freqs;
  int rope_dim, out_dtype, splits, box_rows;
  float scale_log2;
  Div by_window, by_ratio, by_page, by_splits;
};

// ---- the pair
__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;\n" : "=r"(r));
  return r;
}
__device__ __forceinline__ uint32_t in_cta(const void* p, uint32_t rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;\n" : "=r"(r) : "r"(smem_u32(p)), "r"(rank));
  return r;
}
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;\n" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;\n" ::: "memory"); }
// Arrive on a barrier of either CTA. What it tells of is read by the tensor cores from the arriving
// CTA's own shared memory, and its writes there are complete for them once fence.proxy.async has been
// passed, so the arrival need not release at cluster scope (which took 1000 to 1800 cycles a tile).
__device__ __forceinline__ void arrive_at(uint32_t bar) {
  asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];\n" ::"r"(bar) : "memory");
}
// a tile load into this CTA's shared memory that completes on a barrier of CTA 0 of the pair
__device__ __forceinline__ void load_pair(void* dst, const void* map, int x, int y, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, "
      "%3}], [%4];\n" ::"r"(smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(bar)
      : "memory");
}
// a 64 x 64 tile of this CTA's shared memory to a tensor, and the wait until such tiles have been read (what
// was written is complete with the grid)
__device__ __forceinline__ void store_tile(const void* map, int x, int y, const void* src) {
  asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.tile.bulk_group [%0, {%1, %2}], [%3];\n" ::"l"(
                   reinterpret_cast<uint64_t>(map)),
               "r"(x), "r"(y), "r"(smem_u32(src))
               : "memory");
  asm volatile("cp.async.bulk.commit_group;\n" ::: "memory");
}
__device__ __forceinline__ void stores_read() { asm volatile("cp.async.bulk.wait_group.read 0;\n" ::: "memory"); }
__device__ __forceinline__ void mma_pair(uint32_t d, uint64_t a, uint64_t b, uint32_t id, uint32_t acc) {
  asm volatile(
      "{\n.reg .pred p;\nsetp.ne.b32 p, %4, 0;\n"
      "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n}\n" ::"r"(d),
      "l"(a), "l"(b), "r"(id), "r"(acc));
}
// arrive on `bar` of both CTAs once the MMAs issued before have completed
__device__ __forceinline__ void commit_pair(uint64_t* bar) {
  asm volatile(
      "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;\n" ::"r"(
          smem_u32(bar)),
      "h"(static_cast<uint16_t>(3))
      : "memory");
}
// after an error: everything this thread issued completes (bounded) before its CTA leaves
__device__ __forceinline__ void drain_issued(uint64_t* fin) {
  commit_pair(fin);
  bar_wait(fin, 0);
}
__device__ __forceinline__ float ex2(float x) {  // 2^x, relative error about 2^-22, 2^-inf = +0
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;\n" : "=f"(y) : "f"(x));
  return y;
}
// a pair of bf16 with 0 in place of what is not finite
__device__ __forceinline__ uint32_t finite_bf16x2(uint32_t v) {
  if ((v & 0x7f80u) == 0x7f80u) v &= 0xffff0000u;
  if ((v & 0x7f800000u) == 0x7f800000u) v &= 0xffffu;
  return v;
}
__device__ __forceinline__ void smx_bar() { asm volatile("bar.sync 1, %0;\n" ::"n"(SMX_THREADS) : "memory"); }
// the two warps that hold the same columns of O
__device__ __forceinline__ void column_bar(int group) { asm volatile("bar.sync %0, 64;\n" ::"r"(2 + group) : "memory"); }
__device__ __forceinline__ bool smx_any(bool v) {
  uint32_t r;
  asm volatile(
      "{\n.reg .pred p, q;\nsetp.ne.u32 p, %1, 0;\nbar.red.or.pred q, 1, %2, p;\nselp.u32 %0, 1, 0, q;\n}\n"
      : "=r"(r)
      : "r"(static_cast<uint32_t>(v)), "n"(SMX_THREADS)
      : "memory");
  return r != 0;
}
__device__ __forceinline__ void set_abort(Smem& sm) {
  if (!*reinterpret_cast<volatile int*>(&sm.abort)) {
    *reinterpret_cast<volatile int*>(&sm.abort) = 1;
    raise_device_error(DSV4_ERR_WAIT_TIMEOUT);
  }
}

// ---- the halves of 64 rows that a pair of tokens attends to
struct Unit {
  int first, start;       // the sequence's first token in the batch and its position
  int t0, n;              // the pair's first token, tokens of the pair (1 or 2)
  int p0;                 // its position
  int slot;               // cache slot
  int stage_pos;          // position of the first staged row it sees
  int newest;             // ring slot of the newest row of before the chunk
  int nring, nstage, nh;  // halves: ring, stage, all
  uint64_t ring;          // the ring's halves, 4 bits each
  int seen[2];            // compressed entries that the first and the last token see
};
__device__ __forceinline__ int entries_seen(const Params& P, int pos) {  // as chunk_seen
  return P.c.max_comp == 0 ? 0 : min(P.by_ratio.quot(pos + 1), P.c.max_comp);
}
__device__ __forceinline__ Unit make_unit(const Params& P, int first, int start, int slot, int t0, int n) {
  const dsv4_chunk& c = P.c;
  Unit u;
  u.first = first;
  u.start = start;
  u.t0 = t0;
  u.n = n;
  u.p0 = u.start + (t0 - u.first);
  u.slot = slot;
  const int lo = max(0, u.p0 - c.window + 1);  // oldest position in the first token's window
  u.ring = 0;
  u.nring = 0;
  const int old = u.start - lo;                // rows of before the chunk: slots lo % window .., cyclic
  const int oldest = P.by_window.rem(lo);
  u.newest = u.start > 0 ? P.by_window.rem(u.start - 1) : 0;
  if (old > 0)
    for (int h = 0; 64 * h < c.window; ++h) {
      const int gap = h * 64 - oldest + (h * 64 < oldest ? c.window : 0);  // slots from the oldest row to the half
      if (gap < old || gap > c.window - 64) u.ring |= static_cast<uint64_t>(h) << (4 * u.nring++);
    }
  u.stage_pos = max(u.start, lo);
  u.nstage = (u.p0 + n - u.stage_pos + 63) / 64;
  u.seen[0] = entries_seen(P, u.p0);
  u.seen[1] = entries_seen(P, u.p0 + n - 1);
  u.nh = u.nring + u.nstage + (u.seen[1] + 63) / 64;
  return u;
}
// first pool row of box b of half h; the row behind the pool where there is nothing to load
__device__ __forceinline__ int half_row(const Params& P, const Unit& u, int h, int b) {
  const dsv4_chunk& c = P.c;
  const int r = b * P.box_rows;
  if (h < u.nring) return static_cast<int>(c.win_base[u.slot]) + 64 * static_cast<int>((u.ring >> (4 * h)) & 15) + r;
  h -= u.nring;
  if (h < u.nstage) return static_cast<int>(c.stage_base) + u.first + (u.stage_pos - u.start) + 64 * h + r;
  const int e = 64 * (h - u.nstage) + r;
  if (e >= u.seen[1]) return static_cast<int>(c.pool_rows);
  const int j = P.by_page.quot(e);
  const int32_t pg = c.block_table[static_cast<int64_t>(u.slot) * c.bt_stride + j];
  if (pg < 0) {
    raise_device_error(DSV4_ERR_INDEX_OUT_OF_RANGE);
    return static_cast<int>(c.pool_rows);
  }
  const int64_t row = c.comp_base + static_cast<int64_t>(pg) * c.page + (e - j * c.page);
  return row < c.pool_rows ? static_cast<int>(row) : static_cast<int>(c.pool_rows);
}
// One token and split: each CTA has 32 of its heads in rows 0-31, since storing the partials (32 bytes a cycle
// and SM) is what the pair is slow at; otherwise each has its own token.
__device__ __forceinline__ bool heads_shared(const Params& P, const Unit& u) { return P.splits > 1 && u.n == 1; }
// the same for lane `b` of a warp that loads a half together; nothing to load past the last half or box
__device__ __forceinline__ int tile_row(const Params& P, const Unit& u, int h, int b, int boxes) {
  return h < u.nh && b < boxes ? half_row(P, u, h, b) : static_cast<int>(P.c.pool_rows);
}
// whether the token at position p (entries: what it sees of them) sees row j of half h
__device__ __forceinline__ bool half_sees(const dsv4_chunk& c, const Unit& u, int h, int j, int p, int entries) {
  if (h < u.nring) {
    const int back = u.newest - 64 * static_cast<int>((u.ring >> (4 * h)) & 15) - j;
    const int pos = u.start - 1 - (back < 0 ? back + c.window : back);
    return pos >= 0 && pos > p - c.window;
  }
  h -= u.nring;
  if (h < u.nstage) {
    const int pos = u.stage_pos + 64 * h + j;
    return pos <= p && pos > p - c.window;
  }
  return 64 * (h - u.nstage) + j < entries;
}

// The rows of a pair's halves (64 * half + row) that one of its two tokens alone sees, a lane each: 0 the oldest of the
// first's window, 1 the second's own, 2 the entry that it completes. -1 where there is none.
__device__ __forceinline__ int alone_row(const Params& P, const Unit& u, int lane) {
  if (u.n < 2 || lane > 2) return -1;
  if (lane == 1) return 64 * u.nring + (u.p0 + 1 - u.stage_pos);
  if (lane == 2) return u.seen[1] > u.seen[0] ? 64 * (u.nring + u.nstage) + u.seen[0] : -1;
  const int pos = u.p0 - P.c.window + 1;
  if (pos < 0) return -1;
  if (pos >= u.start) return 64 * u.nring + (pos - u.stage_pos);
  const int slot = P.by_window.rem(pos);
  for (int k = 0; k < u.nring; ++k)
    if (static_cast<int>((u.ring >> (4 * k)) & 15) == slot >> 6) return 64 * k + (slot & 63);
  return -1;
}

// The work of a cluster: units (pair of tokens, split) number `at`, at + clusters, ...; the pairs are counted
// through the sequences and taken from the last to the first, since the last see the most rows. A warp looks
// together, a lane per sequence, 32 at a time (and keeps the first 32).
struct Work {
  struct Seq {
    int first, len, start, slot, pairs;
  };
  Unit u;
  Seq head;
  int pairs, at, split, tile0, nt;

  // this lane's sequence of those from b0 on
  static __device__ __forceinline__ Seq load(const Params& P, int b0) {
    const int b = b0 + (threadIdx.x & 31);
    Seq q = {0, 0, 0, 0, 0};
    if (b < P.c.n) {
      q.first = P.c.cu_seqlens[b];
      const int end = P.c.cu_seqlens[b + 1];
      q.start = P.c.start[b];
      q.slot = P.c.seqs ? P.c.seqs[b] : b;
      if (chunk_valid(q.first, end, P.c.total, q.start, q.slot, P.c.slots)) {
        q.len = end - q.first;
        q.pairs = (q.len + 1) / 2;
      } else {
        raise_device_error(DSV4_ERR_INDEX_OUT_OF_RANGE);
      }
    }
    return q;
  }
  __device__ __forceinline__ explicit Work(const Params& P) : head(load(P, 0)), at(static_cast<int>(blockIdx.x >> 1)) {
    pairs = __reduce_add_sync(0xffffffffu, head.pairs);
    for (int b0 = 32; b0 < P.c.n; b0 += 32) pairs += __reduce_add_sync(0xffffffffu, load(P, b0).pairs);
  }
  __device__ __forceinline__ bool next(const Params& P) {
    if (at >= pairs * P.splits) return false;
    const int pair = P.by_splits.quot(at);
    split = at - pair * P.splits;
    const int find = pairs - 1 - pair;
    at += gridDim.x >> 1;
    int before = 0;
    for (int b0 = 0;; b0 += 32) {  // ends: find < pairs
      const Seq q = b0 == 0 ? head : load(P, b0);
      int s = q.pairs;
      if (P.c.n > 1) {
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const int x = __shfl_up_sync(0xffffffffu, s, o);
          if ((threadIdx.x & 31) >= o) s += x;
        }
      }
      const int own = before + s - q.pairs;
      const uint32_t hit = __ballot_sync(0xffffffffu, find >= own && find < own + q.pairs);
      if (hit != 0) {
        const int l = __ffs(hit) - 1, t0 = q.first + 2 * (find - own);
        u = make_unit(P, __shfl_sync(0xffffffffu, q.first, l), __shfl_sync(0xffffffffu, q.start, l),
                      __shfl_sync(0xffffffffu, q.slot, l), __shfl_sync(0xffffffffu, t0, l),
                      __shfl_sync(0xffffffffu, min(2, q.first + q.len - t0), l));
        break;
      }
      before += __shfl_sync(0xffffffffu, s, 31);
    }
    const int tiles = (u.nh + 1) / 2;  // below 2^24 + 16: 64 times that is an int
    tile0 = P.by_splits.quot(tiles * split);
    nt = P.by_splits.quot(tiles * (split + 1)) - tile0;
    return true;
  }
};

__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(THREADS, 1) chunk_attn_kernel(const __grid_constant__ Params P) {
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  Smem& sm = *reinterpret_cast<Smem*>(smem_raw + ((1024 - (smem_u32(smem_raw) & 1023)) & 1023));
  const int tid = threadIdx.x, lane = tid & 31;
  const int warp = __shfl_sync(0xffffffffu, tid >> 5, 0);  // the same register in every lane
  const uint32_t rank = cluster_rank();

  if (warp == 0) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;\n" ::"r"(smem_u32(&sm.tmem_base)),
                 "r"(TMEM_COLS)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;\n" ::: "memory");
  }
  if (tid == 32) {
    bar_init(&sm.q_full, 1);
    bar_init(&sm.fin[0], 1);
    bar_init(&sm.fin[1], 1);
    bar_init(&sm.o_free, 2 * SMX_WARPS);
    for (int i = 0; i < 2; ++i) {
      for (int x = 0; x < 4; ++x) {
        bar_init(&sm.kv_full[i][x], 1);
        bar_init(&sm.kv_free[i][x], 1);
      }
      bar_init(&sm.s_full[i], 1);
      bar_init(&sm.p_full[i], 2 * (SMX_WARPS + 1));  // and the warps that load V
      bar_init(&sm.v_full[i], 1);
    }
    sm.abort = 0;
    bar_init_fence();
    tma_prefetch_map(&P.pool);
    tma_prefetch_map(&P.q);
  }
  before_sync();
  __syncthreads();
  cluster_arrive();
  pdl_wait();  // what follows reads memory that the kernels before may have written
  // one launch: the next kernel may move in beside it (the merging kernel: see the end)
  if (P.splits == 1) pdl_trigger();
  Work w(P);
  bool has = w.next(P);
  // the loading warps' first rows (the table's words) are on their way while the pair meets
  const int boxes = 64 / P.box_rows;
  int first_row = 0;
  if (warp >= 1 && warp <= 3 && has) first_row = tile_row(P, w.u, 2 * w.tile0 + static_cast<int>(warp == 3 ? 1 - rank : rank), lane, boxes);
  cluster_wait();
  after_sync();
  const uint32_t tmem = sm.tmem_base;
  const volatile int* abort = &sm.abort;
  const uint32_t box_bytes = static_cast<uint32_t>(P.box_rows) * 128;

  // Tiles and units are counted through the whole work (g, ord): a barrier of two buffers is in phase
  // (g / 2) % 2 at tile g.
  if (warp == 1 || warp == 2) {
    // ---------------------------------------------------------------- the tiles as K: slot X (and Q), slot Y
    // (the warp goes together: lane k finds the row of box k, a tile ahead; one lane issues the loads)
    const int x = warp - 1;
    bool ok = true, looked = true;  // looked: first_row is the unit's
    int g = 0, ord = 0, issued = 0;
    for (; ok && has; has = w.next(P), looked = false) {
      if (w.nt == 0) continue;
      int row = looked ? first_row : tile_row(P, w.u, 2 * w.tile0 + static_cast<int>(rank), lane, boxes);
      // Q follows the last S of the unit before
      if (x == 0 && g > 0) ok = bar_wait_or_abort(&sm.s_full[(g - 1) & 1], ((g - 1) >> 1) & 1, abort);
      if (x == 0 && ok && elect_one()) {
        sm.unit_tiles[ord & 1] = w.nt;
        const uint32_t qb = in_cta(&sm.q_full, 0);
        if (rank == 0) bar_expect_tx(&sm.q_full, 2 * 8 * SLAB);
        const int qrow = heads_shared(P, w.u) ? w.u.t0 * HB + 32 * static_cast<int>(rank)
                                    : static_cast<int>(rank) < w.u.n ? (w.u.t0 + static_cast<int>(rank)) * HB : P.c.total * HB;
        for (int e = 0; e < 8; ++e) load_pair(sm.q + e * SLAB, &P.q, e * 64, qrow, qb);  // behind q: zeros
      }
      __syncwarp();
      for (int i = 0; i < w.nt && ok; ++i, ++g) {
        const int b = g & 1;
#pragma unroll
        for (int y = 0; y < 2; ++y) {  // two slabs at a time, as the O of the tile before last frees them
          const int qr = 2 * y + x;
          if (g >= 2 && !(ok = __all_sync(0xffffffffu, bar_wait_or_abort(&sm.kv_free[b][qr], ((g >> 1) - 1) & 1, abort)))) break;
          const uint32_t fb = in_cta(&sm.kv_full[b][qr], 0);
          const bool one = elect_one();
          if (one && rank == 0) bar_expect_tx(&sm.kv_full[b][qr], 4 * SLAB);
          for (int k = 0; k < boxes; ++k) {
            const int at = __shfl_sync(0xffffffffu, row, k);
            if (one) {
#pragma unroll
              for (int e = 0; e < 2; ++e)
                load_pair(sm.kv[b][x] + (2 * y + e) * SLAB + k * box_bytes, &P.pool, (4 * x + 2 * y + e) * 64, at, fb);
            }
          }
          ++issued;
        }
        if (i + 1 < w.nt) row = tile_row(P, w.u, 2 * (w.tile0 + i + 1) + static_cast<int>(rank), lane, boxes);
      }
      if (!ok) {
        if (lane == 0) set_abort(sm);
        // what both CTAs have under way into the pair's tiles lands before the pair leaves
        if (rank == 0) {
          if (x == 0) bar_wait(&sm.q_full, ord & 1);
          for (int e = max(0, issued - 4); e < issued; ++e)
            bar_wait(&sm.kv_full[(e >> 1) & 1][2 * (e & 1) + x], (e >> 2) & 1);
        }
      }
      ++ord;
    }
    if (x == 0 && ok && g > 0) ok = bar_wait_or_abort(&sm.s_full[(g - 1) & 1], ((g - 1) >> 1) & 1, abort);
    if (x == 0 && lane == 0) {
      if (!ok) set_abort(sm);
      sm.unit_tiles[ord & 1] = -1;
      if (ok) bar_arrive(&sm.q_full);
    }
  } else if (warp == 3) {
    // ---------------------------------------------------------------- the other half's rows as V
    bool ok = true, looked = true;
    int g = 0;
    for (; ok && has; has = w.next(P), looked = false) {
      if (w.nt == 0) continue;
      int row = looked ? first_row : tile_row(P, w.u, 2 * w.tile0 + 1 - static_cast<int>(rank), lane, boxes);
      int alone = alone_row(P, w.u, lane);  // lanes 0 to 2
      if (alone >= 0) alone -= 128 * w.tile0;
      for (int i = 0; i < w.nt; ++i, ++g) {
        const int b = g & 1;
        if (!(ok = __all_sync(0xffffffffu, bar_wait_or_abort(&sm.s_full[b], (g >> 1) & 1, abort)))) break;
        uint8_t* slot = sm.kv[b][1 - rank];  // CTA 0: Y takes rows 64-127, CTA 1: X takes rows 0-63
        const bool one = elect_one();
        if (one) bar_expect_tx(&sm.v_full[b], SLOT);
        for (int k = 0; k < boxes; ++k) {
          const int at = __shfl_sync(0xffffffffu, row, k);
          if (one) {
#pragma unroll
            for (int e = 0; e < 4; ++e)
              tma_load_2d(slot + e * SLAB + k * box_bytes, &P.pool, (4 * static_cast<int>(rank) + e) * 64, at, &sm.v_full[b]);
          }
        }
        if (i + 1 < w.nt) row = tile_row(P, w.u, 2 * (w.tile0 + i + 1) + 1 - static_cast<int>(rank), lane, boxes);
        uint32_t here = __ballot_sync(0xffffffffu, alone >> 7 == i);
        if (here != 0) {  // rows of this tile that one token alone sees: 512 bytes of this CTA's dims each, 16 a lane
          if (!(ok = __all_sync(0xffffffffu, bar_wait_or_abort(&sm.v_full[b], (g >> 1) & 1, abort)))) {
            ++g;  // its load is under way
            break;
          }
          for (; here != 0; here &= here - 1) {
            const int r = __shfl_sync(0xffffffffu, alone, __ffs(here) - 1) & 127;
            uint4* at = reinterpret_cast<uint4*>(sm.kv[b][r >> 6] + (lane >> 3) * SLAB + (r & 63) * 128 + (lane & 7) * 16);
            const uint4 v = *at;
            *at = make_uint4(finite_bf16x2(v.x), finite_bf16x2(v.y), finite_bf16x2(v.z), finite_bf16x2(v.w));
          }
          fence_async_smem();
          __syncwarp();
        }
        if (lane == 0) arrive_at(in_cta(&sm.p_full[b], 0));
      }
      if (!ok) {
        if (lane == 0) set_abort(sm);
        for (int e = max(0, g - 2); e < g; ++e) bar_wait(&sm.v_full[e & 1], (e >> 1) & 1);
      }
    }
  } else if (warp == 0) {
    // ---------------------------------------------------------------- S (CTA 0, one thread)
    if (rank == 0 && elect_one()) {
      constexpr uint32_t id_s = idesc_bf16<128, 128>(false, false);
      const uint64_t qd = sdesc(smem_u32(sm.q), 16, 1024), kd = sdesc(smem_u32(sm.kv), 16, 1024);
      bool ok = true;
      int g = 0;
      for (int ord = 0; ok; ++ord) {
        if (!(ok = bar_wait_or_abort(&sm.q_full, ord & 1, abort))) break;
        const int n = sm.unit_tiles[ord & 1];
        if (n < 0) break;
        for (int i = 0; i < n && ok; ++i, ++g) {
          const int b = g & 1;
          const uint32_t d = tmem + COL_S + 64 * b;
          // Quarter qr: slabs 2 (qr / 2) .. of slot qr % 2. Its rows say that the buffer of the tile before last
          // has been through O, and so that its S has been read.
#pragma unroll
          for (int qr = 0; qr < 4; ++qr) {
            if (!(ok = bar_wait_or_abort(&sm.kv_full[b][qr], (g >> 1) & 1, abort))) break;
            if (qr == 0) after_sync();
            const uint64_t a = qd + ((4 * (qr & 1) + (qr & 2)) * SLAB >> 4);
            const uint64_t k = kd + b * (2 * SLOT >> 4) + ((qr & 1) * SLOT + (qr & 2) * SLAB >> 4);
#pragma unroll
            for (int e = 0; e < 8; ++e)
              mma_pair(d, a + ((e >> 2) * SLAB + (e & 3) * 32 >> 4), k + ((e >> 2) * SLAB + (e & 3) * 32 >> 4), id_s,
                       (qr | e) ? 1u : 0u);
          }
          if (ok) commit_pair(&sm.s_full[b]);
        }
      }
      if (!ok) {
        set_abort(sm);
        drain_issued(&sm.fin[0]);
      }
    }
  } else if (warp == 12) {
    // ---------------------------------------------------------------- O (CTA 0, one thread)
    if (rank == 0) {
      constexpr uint32_t id_o = idesc_bf16<128, 256>(false, true);
      const uint64_t pd = sdesc(smem_u32(sm.p), 16, 1024), vd = sdesc(smem_u32(sm.kv), SLAB, 1024);
      bool ok = true;
      int g = 0, ord = 0;
      for (; ok && has; has = w.next(P)) {
        if (w.nt == 0) continue;
        uint32_t leader;
        if (elect_one(&leader)) {
          // the epilogue of the unit before has read O
          if (ord > 0) ok = bar_wait_or_abort(&sm.o_free, (ord - 1) & 1, abort);
          for (int i = 0; i < w.nt && ok; ++i, ++g) {
            const int b = g & 1;
            if (!(ok = bar_wait_or_abort(&sm.p_full[b], (g >> 1) & 1, abort))) break;
            after_sync();
            const uint64_t a = pd + b * (2 * SLAB >> 4), v = vd + b * (2 * SLOT >> 4);
            const uint32_t acc = i > 0 ? 1u : 0u;
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
              for (int kk = 0; kk < 8; ++kk) {
                mma_pair(tmem + COL_O + 128 * j, a + ((kk >> 2) * SLAB + (kk & 3) * 32 >> 4),
                         v + ((kk >> 2) * SLOT + 2 * j * SLAB + (kk & 3) * 2048 >> 4), id_o, kk ? 1u : acc);
                if ((kk & 3) == 3) commit_pair(&sm.kv_free[b][2 * j + (kk >> 2)]);
              }
          }
          if (!ok) {
            set_abort(sm);
            drain_issued(&sm.fin[1]);
          }
        }
        ok = __shfl_sync(0xffffffffu, ok, leader);
        g = __shfl_sync(0xffffffffu, g, leader);
        ++ord;
      }
    }
  } else {
    // ---------------------------------------------------------------- softmax, epilogue (warps 4-11)
    const int quad = warp & 3, ch = (warp >> 2) - 1;
    const uint32_t lanes = static_cast<uint32_t>(quad * 32) << 16;
    const int head = (quad & 1) * 32 + lane, kvh = quad >> 1;  // TMEM lane: head + 64 kvh
    const float sink = P.sink[head] * LOG2E;
    bool ok = true;
    int g = 0;
    while (has) {
      const Unit& u = w.u;
      const bool shared = heads_shared(P, u);
      const bool second = rank != 0 && !shared;  // this CTA has the pair's second token
      const int token = u.t0 + second;
      // the row's head, -1: none of a token
      const int whose = shared ? ((quad & 1) == 0 ? 32 * static_cast<int>(rank) + lane : -1) : second >= u.n ? -1 : head;
      const int pos = u.p0 + static_cast<int>(rank), split = w.split;
      if (w.nt == 0) {  // splits > 1: no rows for this one, its O is not read
        if (whose >= 0 && kvh == 0 && ch == 0) {
          float* ml = P.part + static_cast<int64_t>(P.c.total) * P.splits * (HB * D) +
                      ((static_cast<int64_t>(token) * P.splits + split) * HB + whose) * 2;
          ml[0] = -INFINITY;
          ml[1] = 0.f;
        }
        has = w.next(P);
        continue;
      }
      float m = -INFINITY, l = 0.f;
      for (int i = 0; i < w.nt; ++i, ++g) {
        const int b = g & 1;
        // what of this warp's 32 rows is seen, by the CTA's token and by either token of the pair: all of
        // them, but for the ring, the stage and the last entries
        const int h = 2 * (w.tile0 + i) + kvh;
        uint32_t see = 0xffffffffu, either = 0xffffffffu;
        if (h < u.nring + u.nstage || 64 * (h - u.nring - u.nstage) + 64 > u.seen[0]) {
          const int j = 32 * ch + lane;
          const bool v0 = h < u.nh && half_sees(P.c, u, h, j, u.p0, u.seen[0]);
          const bool v1 = h < u.nh && u.n > 1 && half_sees(P.c, u, h, j, u.p0 + 1, u.seen[1]);
          see = __ballot_sync(0xffffffffu, second ? v1 : v0);
          either = __ballot_sync(0xffffffffu, v0 || v1);
        }
        // a wait that ran out takes the CTA's warps to the end together, from the next smx_any
        ok = ok && __all_sync(0xffffffffu, bar_wait_or_abort(&sm.s_full[b], (g >> 1) & 1, abort));
        float x[32];
        float mx = -INFINITY;
        if (ok) {
          after_sync();
          tmem_ld16(tmem + lanes + COL_S + 64 * b + 32 * ch, x);
          tmem_ld16(tmem + lanes + COL_S + 64 * b + 32 * ch + 16, x + 16);
          tmem_wait_ld();
#pragma unroll
          for (int c = 0; c < 32; ++c) x[c] *= P.scale_log2;
          if (see != 0xffffffffu) {
#pragma unroll
            for (int c = 0; c < 32; ++c) x[c] = (see >> c) & 1 ? x[c] : -INFINITY;
          }
          float mc[4];
#pragma unroll
          for (int c = 0; c < 4; ++c) mc[c] = x[c];
#pragma unroll
          for (int c = 4; c < 32; ++c) mc[c & 3] = fmaxf(mc[c & 3], x[c]);
          mx = fmaxf(fmaxf(mc[0], mc[1]), fmaxf(mc[2], mc[3]));
        }
        if (smx_any(!ok || mx > m + RESCALE)) {
          if (smx_any(!ok)) {
            if (lane == 0) set_abort(sm);
            ok = false;
            break;
          }
          sm.red[kvh * 2 + ch][head] = mx;
          smx_bar();
          const float mn = fmaxf(m, fmaxf(fmaxf(sm.red[0][head], sm.red[1][head]), fmaxf(sm.red[2][head], sm.red[3][head])));
          const float alpha = m == -INFINITY ? 0.f : ex2(m - mn);
          const bool moved = mn != m && m != -INFINITY;
          m = mn;
          l *= alpha;
          smx_bar();  // red is free again
          if (i > 0 && __any_sync(0xffffffffu, moved)) {
            // O of the tiles before has been added up: rescale this warp's half of its columns
            ok = __all_sync(0xffffffffu, bar_wait_or_abort(&sm.kv_free[b ^ 1][3], ((g - 1) >> 1) & 1, abort));
            if (ok) {
              after_sync();
#pragma unroll 1
              for (int c = 0; c < 128; c += 32) {
                float v[32];
                tmem_ld16(tmem + lanes + COL_O + 128 * ch + c, v);
                tmem_ld16(tmem + lanes + COL_O + 128 * ch + c + 16, v + 16);
                tmem_wait_ld();
#pragma unroll
                for (int e = 0; e < 32; ++e) v[e] *= moved ? alpha : 1.f;
                tmem_st16(tmem + lanes + COL_O + 128 * ch + c, v);
                tmem_st16(tmem + lanes + COL_O + 128 * ch + c + 16, v + 16);
              }
              tmem_wait_st();
            }
          }
        }
        // P: 32 columns of this row, four 16-byte chunks of the 128-byte-swizzled slab (free: the S that was
        // waited for needed the tile before last's O, which read it)
        uint8_t* prow = sm.p[b] + kvh * SLAB + head * 128;
        const float mm = m == -INFINITY ? 0.f : m;  // nothing seen yet: every x is -inf and p is 0
        float ls[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int c4 = 0; c4 < 4; ++c4) {
          uint32_t e2[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float p0 = ex2(x[c4 * 8 + 2 * e] - mm), p1 = ex2(x[c4 * 8 + 2 * e + 1] - mm);
            e2[e] = pack_bf16x2(p0, p1);
            ls[e] += p0 + p1;
          }
          *reinterpret_cast<uint4*>(prow + (((ch * 4 + c4) ^ (head & 7)) << 4)) = make_uint4(e2[0], e2[1], e2[2], e2[3]);
        }
        l += (ls[0] + ls[1]) + (ls[2] + ls[3]);
        ok = ok && __all_sync(0xffffffffu, bar_wait_or_abort(&sm.v_full[b], (g >> 1) & 1, abort));
        if (!ok) {  // the CTA's other warps end at their next wait or at smx_any
          if (lane == 0) set_abort(sm);
        } else if (either != 0xffffffffu && h < u.nh) {
          // values of rows that neither token sees: two slabs of the slot for this warp, 16 lanes a row
          uint8_t* slab = sm.kv[b][kvh] + (2 * (quad & 1) + ((lane >> 3) & 1)) * SLAB;
          for (int e = lane >> 4; e < 32; e += 2)
            if (!((either >> e) & 1))
              *reinterpret_cast<uint4*>(slab + (32 * ch + e) * 128 + (lane & 7) * 16) = make_uint4(0, 0, 0, 0);
        }
        fence_async_smem();
        before_sync();
        __syncwarp();
        if (lane == 0) arrive_at(in_cta(&sm.p_full[b], 0));
      }
      // the row's sum of its four parts; the unit's last O (a warp whose wait ran out goes on to the barriers)
      if (smx_any(!ok)) {
        if (lane == 0) set_abort(sm);
        ok = false;
        break;
      }
      sm.red[kvh * 2 + ch][head] = l;
      smx_bar();
      l = (sm.red[0][head] + sm.red[1][head]) + (sm.red[2][head] + sm.red[3][head]);
      smx_bar();
      has = w.next(P);  // found while the last O is being computed; u is the next unit's from here
      ok = __all_sync(0xffffffffu, bar_wait_or_abort(&sm.kv_free[(g - 1) & 1][3], ((g - 1) >> 1) & 1, abort));
      after_sync();
      const uint32_t src = tmem + lanes + COL_O + 128 * ch;
      const int d0 = 256 * kvh + 128 * ch, group = 2 * kvh + ch;
      if (P.splits > 1) {
        // partials by four dims of every head: a warp stores 512 bytes at a time
        if (ok && whose >= 0) {
          const int64_t at = static_cast<int64_t>(token) * P.splits + split;
          float4* po = reinterpret_cast<float4*>(P.part) + (at * (D / 4) + d0 / 4) * HB + whose;
#pragma unroll 1
          for (int c = 0; c < 128; c += 32) {
            float v[32];
            tmem_ld16(src + c, v);
            tmem_ld16(src + c + 16, v + 16);
            tmem_wait_ld();
#pragma unroll
            for (int e = 0; e < 8; ++e) po[(c / 4 + e) * HB] = make_float4(v[4 * e], v[4 * e + 1], v[4 * e + 2], v[4 * e + 3]);
          }
          if (group == 0)
            *reinterpret_cast<float2*>(P.part + static_cast<int64_t>(P.c.total) * P.splits * (HB * D) + (at * HB + whose) * 2) =
                make_float2(m, l);
        }
      } else {
        const float inv = 1.f / (l + exp2f(sink - m));
        const int64_t off = (static_cast<int64_t>(token) * HB + head) * D + d0;
        // Rows leave by way of P's space, which is out of use until the next unit's first P: 64 rows by 64 dims
        // of two warps at a time, 128-byte swizzled, to the tensor by TMA (16 bytes a lane straight from the
        // registers took 5700 cycles a unit).
        uint8_t* const tile = sm.p[0] + group * SLAB;
        const bool storer = (quad & 1) == 0 && lane == 0;
        float rc = 1.f, rs = 0.f;  // lane f: the rotation of pair f
        if (P.freqs != nullptr && d0 + 128 > D - P.rope_dim && lane < P.rope_dim / 2)
          rope_cos_sin(pos, P.freqs[lane], &rc, &rs);
        const bool store = whose >= 0 && P.out_dtype == DSV4_BF16;
#pragma unroll 1
        for (int c = 0; c < 128; c += 32) {
          float v[32];
          tmem_ld16(src + c, v);
          tmem_ld16(src + c + 16, v + 16);
          tmem_wait_ld();
#pragma unroll
          for (int e = 0; e < 32; ++e) v[e] *= inv;
          if (d0 + c + 32 > D - P.rope_dim) {
#pragma unroll
            for (int e = 0; e < 32; e += 2) {
              const int f = (d0 + c + e - (D - P.rope_dim)) >> 1;
              const float cs = __shfl_sync(0xffffffffu, rc, f & 31), sn = __shfl_sync(0xffffffffu, rs, f & 31);
              if (f >= 0) rotate_pair(v[e], v[e + 1], cs, sn, true, &v[e], &v[e + 1]);
            }
          }
          if (P.out_dtype == DSV4_BF16) {
            if (c == 64) {  // the first 64 dims have left the space
              if (storer) stores_read();
              column_bar(group);
            }
#pragma unroll
            for (int e = 0; e < 4; ++e)
              *reinterpret_cast<uint4*>(tile + head * 128 + (((((c >> 3) & 4) + e) ^ (head & 7)) << 4)) =
                  make_uint4(pack_bf16x2(v[8 * e], v[8 * e + 1]), pack_bf16x2(v[8 * e + 2], v[8 * e + 3]),
                             pack_bf16x2(v[8 * e + 4], v[8 * e + 5]), pack_bf16x2(v[8 * e + 6], v[8 * e + 7]));
            if (c & 32) {
              fence_async_smem();
              column_bar(group);
              if (store && ok && storer)
                store_tile(&P.o, d0 + c - 32, token * HB, tile);
            }
          } else if (ok && whose >= 0) {
            float4* dst = reinterpret_cast<float4*>(reinterpret_cast<float*>(P.out) + off + c);
#pragma unroll
            for (int e = 0; e < 8; ++e) dst[e] = make_float4(v[4 * e], v[4 * e + 1], v[4 * e + 2], v[4 * e + 3]);
          }
        }
        if (storer) stores_read();
      }
      if (!ok && lane == 0) set_abort(sm);
      // O has been read: the next unit's may be begun
      before_sync();
      __syncwarp();
      if (lane == 0) arrive_at(in_cta(&sm.o_free, 0));
    }
    // every commit of the last two tiles has arrived here before the CTA leaves
    for (int e = max(0, g - 2); e < g; ++e)
      for (int x = 0; x < 4; ++x)
        ok = ok && __all_sync(0xffffffffu, bar_wait_or_abort(&sm.kv_free[e & 1][x], (e >> 1) & 1, abort));
    if (!ok && lane == 0) set_abort(sm);
  }
  __syncwarp();
  before_sync();
  __syncthreads();
  // (not earlier: the merging kernel's blocks would all be placed on the few SMs without a cluster)
  if (P.splits > 1) pdl_trigger();
  cluster_arrive();
  cluster_wait();  // no CTA leaves while the pair's MMAs, loads or arrivals may touch it
  after_sync();
  if (warp == 0)
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;\n" ::"r"(tmem), "r"(TMEM_COLS));
}

// One CTA per (token, MD dims): the splits' partials weighed by 2^(m - max), the sink, the inverse
// rotation. At most 64 splits. A float4 (four dims of a head) per thread of a group and split; MG groups take
// every MG-th split, the first PF of a thread's loads on their way before the weights are known. <8, 4> for
// as many tokens as have all their CTAs resident at once (2 an SM), so that the 64 CTAs of a single token have
// enough loads in flight; <16, 1> otherwise. The sum turns round in shared memory, so that a head's dims leave
// together. What the attention kernel had to wait for is complete before this one starts (its launch is
// triggered behind that wait), so the sequences are looked up before its own wait.
template <int MD, int MG, int PF>
__global__ void __launch_bounds__(MG * MD * HB / 4) chunk_merge_kernel(const __grid_constant__ Params P) {
  constexpr int MT = MG * MD * HB / 4, MH = MT / HB, MS = 64 / MH;  // threads; per head; splits a thread weighs
  constexpr int BLOCKS = D / MD;
  const int64_t t = blockIdx.x / BLOCKS;
  const int d0 = static_cast<int>(blockIdx.x % BLOCKS) * MD;
  const ChunkToken k = chunk_token(P.c, static_cast<int>(t));
  __shared__ float w[64][HB];   // [split][head]
  __shared__ float red[2][MH][HB];
  __shared__ float4 o[MG][MD / 4][HB];
  const int tid = threadIdx.x, h = tid & (HB - 1);
  const float sink = P.sink[h] * LOG2E;
  pdl_wait();
  if (k.seq < 0) return;
  // this thread's four dims of head h, splits gd, gd + MG, ...
  const int gd = tid / (MD * HB / 4), quad = tid / HB % (MD / 4);
  const float4* src = reinterpret_cast<const float4*>(P.part) + (t * P.splits * (D / 4) + d0 / 4 + quad) * HB + h;
  float4 x[PF];
  auto fetch = [&](int s0) {
#pragma unroll
    for (int i = 0; i < PF; ++i)
      if (s0 + i * MG < P.splits) x[i] = src[static_cast<int64_t>(s0 + i * MG) * (HB * D / 4)];
  };
  {
    const int g = tid / HB;
    const float2* ml = reinterpret_cast<const float2*>(P.part + static_cast<int64_t>(P.c.total) * P.splits * (HB * D)) +
                       t * P.splits * HB + h;
    float2 v[MS];
#pragma unroll
    for (int i = 0; i < MS; ++i) {
      const int s = g + i * MH;
      v[i] = s < P.splits ? ml[s * HB] : make_float2(-INFINITY, 0.f);
    }
    fetch(gd);
    float M = v[0].x;
#pragma unroll
    for (int i = 1; i < MS; ++i) M = fmaxf(M, v[i].x);
    red[0][g][h] = M;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < MH; ++i) M = fmaxf(M, red[0][i][h]);
    float L = 0.f;
#pragma unroll
    for (int i = 0; i < MS; ++i) {
      const int s = g + i * MH;
      const float e = v[i].x == -INFINITY ? 0.f : exp2f(v[i].x - M);
      if (s < P.splits) w[s][h] = e;
      L = fmaf(e, v[i].y, L);
    }
    red[1][g][h] = L;
    __syncthreads();
    if (g == 0) {
      L = 0.f;
#pragma unroll
      for (int i = 0; i < MH; ++i) L += red[1][i][h];
      red[0][0][h] = 1.f / (L + exp2f(sink - M));
    }
  }
  float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int s0 = gd; s0 < P.splits; s0 += PF * MG) {
    if (s0 != gd) fetch(s0);
#pragma unroll
    for (int i = 0; i < PF; ++i) {
      const int s = s0 + i * MG;
      const float f = s < P.splits ? w[s][h] : 0.f;
      if (f != 0.f) {  // a split without rows has written no O
        a.x = fmaf(f, x[i].x, a.x);
        a.y = fmaf(f, x[i].y, a.y);
        a.z = fmaf(f, x[i].z, a.z);
        a.w = fmaf(f, x[i].w, a.w);
      }
    }
  }
  o[gd][quad][h] = a;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < MD * HB / 2; i += MT) {  // a pair of dims of a head
    if (i + tid >= MD * HB / 2) break;
    const int head = (i + tid) / (MD / 2), e = (i + tid) % (MD / 2) * 2;
    float y = 0.f, z = 0.f;
#pragma unroll
    for (int g = 0; g < MG; ++g) {
      const float2 v = *(reinterpret_cast<const float2*>(&o[g][e / 4][head]) + (e / 2 & 1));
      y += v.x;
      z += v.y;
    }
    y *= red[0][0][head];
    z *= red[0][0][head];
    const int f = (d0 + e - (D - P.rope_dim)) >> 1;
    if (P.freqs != nullptr && f >= 0) {
      float c, s;
      rope_cos_sin(k.pos, P.freqs[f], &c, &s);
      rotate_pair(y, z, c, s, true, &y, &z);
    }
    const int64_t off = (t * HB + head) * D + d0 + e;
    if (P.out_dtype == DSV4_BF16)
      *reinterpret_cast<uint32_t*>(reinterpret_cast<__nv_bfloat16*>(P.out) + off) = pack_bf16x2(y, z);
    else
      *reinterpret_cast<float2*>(reinterpret_cast<float*>(P.out) + off) = make_float2(y, z);
  }
}

DSV4_ERROR_READER(chunk_attn)

static int encode(CUtensorMap* map, const void* base, uint64_t rows, uint32_t box_rows) {
  static std::atomic<void*> fn{nullptr};
  void* f = fn.load(std::memory_order_acquire);
  if (!f) {
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &q) != cudaSuccess ||
        q != cudaDriverEntryPointSuccess) {
      set_error("dsv4_chunk_attn: cuTensorMapEncodeTiled is not available from the driver");
      return DSV4_ERR_CUDA;
    }
    fn.store(f, std::memory_order_release);
  }
  const cuuint64_t dims[2] = {D, rows};
  const cuuint64_t strides[1] = {D * 2};
  const cuuint32_t box[2] = {64, box_rows};
  const cuuint32_t estr[2] = {1, 1};
  const CUresult r = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(f)(
      map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, const_cast<void*>(base), dims, strides, box, estr,
      CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
      CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) {
    set_error("dsv4_chunk_attn: cuTensorMapEncodeTiled failed (%d) for %llu rows", static_cast<int>(r),
              static_cast<unsigned long long>(rows));
    return DSV4_ERR_CUDA;
  }
  return DSV4_OK;
}

// Over how many clusters the rows of a pair are split: the number with the least time, by this account in
// hundredths of a tile (1.43 us for 128 rows): the tiles of a split in every round of the clusters, 1.4 a round
// after the first, and for a split 2.4 for the merging kernel and 0.05 a token and split for its partials.
// Measured (us): 32 tokens at 2048: 19.0 whole, 23.1 in 3; 1 at 65536: 196 whole, 20.6 in 44, 21.8 in 64; 80 at
// 64548 (40 pairs for 74 clusters): 199 whole, 161 in 3, 177 in 8; 300 at 16384: 173 whole, 217 in 2.
// A last round of eight or more that is not full is not worth it. Of the splits with as many tiles each the
// fewest are the best, so only those are looked at.
static int plan_splits(const dsv4_chunk_attn_params* p) {
  if (p->num_splits > 0) return std::min(p->num_splits, 64);
  const int64_t total = p->chunk.total;
  const uint32_t clusters = std::max(1, num_sms() / 2);
  if ((total + p->chunk.n) / 2 >= 8 * static_cast<int64_t>(clusters)) return 1;
  const uint32_t units = static_cast<uint32_t>((total + p->chunk.n) / 2);
  const uint32_t tiles = (static_cast<uint32_t>(p->chunk.max_comp) + 2u * p->chunk.window) / BN + 1;  // at most
  int best = 1;
  int64_t least = INT64_MAX;
  for (uint32_t s = 1, each = tiles; s <= 64; s = (tiles + each - 2) / (each - 1)) {  // the fewest with fewer tiles each
    each = (tiles + s - 1) / s;
    const uint32_t rounds = (units * s + clusters - 1) / clusters;
    const int64_t cost = static_cast<int64_t>(rounds) * each * 100 + (static_cast<int64_t>(rounds) - 1) * 140 +
                         (s > 1 ? 240 + 5 * s * total : 0);
    if (cost < least) least = cost, best = static_cast<int>(s);
    if (each == 1) break;
  }
  return best;
}

}  // namespace ca
}  // namespace dsv4

using namespace dsv4;

extern "C" {

static size_t partial_bytes(const dsv4_chunk_attn_params* p, int splits) {
  return splits == 1 ? 0 : static_cast<size_t>(p->chunk.total) * splits * (ca::HB * ca::D + ca::HB * 2) * sizeof(float);
}
size_t dsv4_chunk_attn_workspace_size(const dsv4_chunk_attn_params* p) {
  if (p == nullptr || p->chunk.total <= 0 || p->chunk.n <= 0) return 0;
  return partial_bytes(p, ca::plan_splits(p));
}

int dsv4_chunk_attn(const dsv4_chunk_attn_params* p, void* stream) {
  DSV4_CHECK_ARG(p != nullptr, "dsv4_chunk_attn: params is NULL");
  const int rc = check_chunk(&p->chunk, "dsv4_chunk_attn");
  if (rc != DSV4_OK) return rc;
  DSV4_CHECK_ARG(p->q && p->pool && p->sink && p->out, "dsv4_chunk_attn: NULL tensor");
  DSV4_CHECK_ARG(((reinterpret_cast<uintptr_t>(p->q) | reinterpret_cast<uintptr_t>(p->pool) |
                   reinterpret_cast<uintptr_t>(p->out)) & 15) == 0,
                 "dsv4_chunk_attn: q, pool and out must be 16-byte aligned");
  DSV4_CHECK_ARG(p->chunk.window <= ca::MAX_WINDOW, "dsv4_chunk_attn: window %d above %d", p->chunk.window, ca::MAX_WINDOW);
  DSV4_CHECK_ARG(p->chunk.max_comp == 0 || p->chunk.page % 8 == 0, "dsv4_chunk_attn: page %d is not a multiple of 8",
                 p->chunk.page);
  DSV4_CHECK_DTYPE(p->out_dtype == DSV4_F32 || p->out_dtype == DSV4_BF16, "dsv4_chunk_attn: out dtype");
  DSV4_CHECK_ARG(p->rope_freqs == nullptr || (p->rope_dim > 0 && p->rope_dim <= 64 && p->rope_dim % 2 == 0),
                 "dsv4_chunk_attn: 0 < rope_dim <= 64");
  DSV4_CHECK_ARG(p->num_splits >= 0 && p->num_splits <= 64, "dsv4_chunk_attn: 0 to 64 splits");
  DSV4_CHECK_ARG(static_cast<int64_t>(p->chunk.total) * ca::HB <= 0x7fffffffLL - ca::HB, "dsv4_chunk_attn: too many tokens");
  if (p->chunk.n == 0 || p->chunk.total == 0) return DSV4_OK;
  ca::Params P = {};
  P.splits = ca::plan_splits(p);
  const size_t need = partial_bytes(p, P.splits);
  if (need > 0 && (p->workspace == nullptr || p->workspace_bytes < need ||
                   (reinterpret_cast<uintptr_t>(p->workspace) & 15) != 0)) {
    set_error("dsv4_chunk_attn: workspace of %zu bytes needed, %zu given", need, p->workspace_bytes);
    return DSV4_ERR_WORKSPACE;
  }
  P.box_rows = 64;
  if (p->chunk.max_comp > 0)
    while (p->chunk.page % P.box_rows != 0) P.box_rows /= 2;
  int st = ca::encode(&P.pool, p->pool, static_cast<uint64_t>(p->chunk.pool_rows), static_cast<uint32_t>(P.box_rows));
  if (st != DSV4_OK) return st;
  st = ca::encode(&P.q, p->q, static_cast<uint64_t>(p->chunk.total) * ca::HB, 64);
  if (st != DSV4_OK) return st;
  if (P.splits == 1 && p->out_dtype == DSV4_BF16)
    st = ca::encode(&P.o, p->out, static_cast<uint64_t>(p->chunk.total) * ca::HB, 64);
  if (st != DSV4_OK) return st;
  P.c = p->chunk;
  P.sink = p->sink;
  P.out = p->out;
  P.part = reinterpret_cast<float*>(p->workspace);
  P.freqs = p->rope_freqs;
  P.rope_dim = p->rope_freqs ? p->rope_dim : 0;
  P.out_dtype = p->out_dtype;
  P.scale_log2 = p->scale * ca::LOG2E;
  P.by_window = ca::Div(P.c.window);
  P.by_ratio = ca::Div(std::max(1, P.c.ratio));
  P.by_page = ca::Div(std::max(1, P.c.page));
  P.by_splits = ca::Div(P.splits);
  // one cluster per pair of SMs, or per unit where there are fewer
  const int64_t units = (static_cast<int64_t>(P.c.total) + P.c.n) / 2 * P.splits;
  DSV4_CHECK_ARG(static_cast<int64_t>(P.c.total) * P.splits * ca::HB <= 0x7fffffffLL, "dsv4_chunk_attn: too many tokens");
  static PerDeviceOnce attr;
  const int smem = static_cast<int>(sizeof(ca::Smem)) + 1024;
  DSV4_CUDA_CHECK(set_smem_once(attr, ca::chunk_attn_kernel, smem));
  DSV4_CUDA_CHECK(launch_pdl(ca::chunk_attn_kernel, dim3(static_cast<unsigned>(2 * std::min<int64_t>(units, num_sms() / 2))),
                             dim3(ca::THREADS), smem, as_stream(stream), P));
  if (P.splits > 1 && P.c.total * (ca::D / 8) <= 2 * num_sms())
    DSV4_CUDA_CHECK(launch_pdl(ca::chunk_merge_kernel<8, 4, 8>, dim3(static_cast<unsigned>(P.c.total) * (ca::D / 8)),
                               dim3(4 * 8 * ca::HB / 4), 0, as_stream(stream), P));
  else if (P.splits > 1)
    DSV4_CUDA_CHECK(launch_pdl(ca::chunk_merge_kernel<16, 1, 4>, dim3(static_cast<unsigned>(P.c.total) * (ca::D / 16)),
                               dim3(16 * ca::HB / 4), 0, as_stream(stream), P));
  return DSV4_OK;
}

}  // extern "C"
