// Row bookkeeping of a chunk of new tokens over the device-resident sparse-MLA state: where each
// token's kv row is staged, which pool rows it attends to, and the move of the last rows into the
// window rings once the chunk has been attended. The reference keeps this state on the host and
// takes one token at a time (oracle/v4_fast.py:93-118); a chunk cannot go through the ring first,
// because the token at position p would overwrite the row of position p - window that earlier
// tokens of the same chunk still see. So the chunk's rows are staged behind the pages of the pool,
// token i of the chunk at row stage_base + i, and reach the ring only after the attention.
//
// Both kernels move a few words or rows per token and are bound by their launch (256 lists of 640 entries: 4.8 us).
#include "chunk.cuh"
#include "common.cuh"

namespace dsv4 {
namespace chk {

// one CTA per token: positions[t], rows[t] (the staged row) and, when asked for, the explicit list
// [window rows in ascending position | cols columns]: the given rows of the token, or every
// compressed entry it sees, mapped through the block table
__global__ void chunk_rows_kernel(dsv4_chunk c, int32_t* positions, int64_t* stage_rows, int32_t* index,
                                  int64_t index_stride, int32_t cols, const int32_t* given) {
  pdl_wait();
  pdl_trigger();
  const int t = blockIdx.x;
  const ChunkToken k = chunk_token(c, t);
  if (threadIdx.x == 0) {
    if (positions) positions[t] = k.pos;
    if (stage_rows) stage_rows[t] = c.stage_base + t;
  }
  if (index == nullptr) return;
  int32_t* row = index + t * index_stride;
  const int slot = k.seq < 0 ? 0 : c.seqs ? c.seqs[k.seq] : k.seq;
  for (int j = threadIdx.x; j < c.window; j += blockDim.x) {
    const int p = k.pos - c.window + 1 + j;
    int64_t r = -1;
    if (k.seq >= 0 && p >= 0) r = p >= k.start ? c.stage_base + k.first + (p - k.start) : c.win_base[slot] + p % c.window;
    row[j] = static_cast<int32_t>(r);
  }
  const int seen = k.seq < 0 ? 0 : chunk_seen(c, k.pos);
  for (int j = threadIdx.x; j < cols; j += blockDim.x) {
    int64_t r = -1;
    if (given) {
      r = k.seq < 0 ? -1 : given[static_cast<int64_t>(t) * cols + j];
    } else if (j < seen) {
      const int32_t pg = c.block_table[static_cast<int64_t>(slot) * c.bt_stride + j / c.page];
      if (pg >= 0)
        r = c.comp_base + static_cast<int64_t>(pg) * c.page + j % c.page;
      else
        raise_device_error(DSV4_ERR_INDEX_OUT_OF_RANGE);
    }
    row[c.window + j] = static_cast<int32_t>(r);
  }
}

// one CTA per (sequence, ring slot): the slot's newest token of the chunk, if it has one. A slot named
// twice has no newest token: DSV4_ERR_INDEX_OUT_OF_RANGE, and the first to name it has the ring.
// No early launch of the next kernel: the decode attention reads window rows before it waits for the
// kernel before it, and counts on those that wrote them being complete.
__global__ void chunk_commit_kernel(dsv4_chunk c, uint4* pool, int row16) {
  pdl_wait();
  const int b = blockIdx.y, j = blockIdx.x;
  const int first = c.cu_seqlens[b], last = c.cu_seqlens[b + 1];
  const int slot = c.seqs ? c.seqs[b] : b;
  bool bad = !chunk_valid(first, last, c.total, c.start[b], slot, c.slots);
  if (c.seqs != nullptr && last > first)
    for (int i = threadIdx.x; i < b; i += blockDim.x) bad |= c.seqs[i] == slot && c.cu_seqlens[i + 1] > c.cu_seqlens[i];
  if (__syncthreads_or(bad)) {
    if (j == 0 && threadIdx.x == 0) raise_device_error(DSV4_ERR_INDEX_OUT_OF_RANGE);
    return;
  }
  if (last == first) return;
  const int end = c.start[b] + (last - first);  // the largest p < end with p % window == j
  const int p = end - 1 - (end - 1 - j % c.window + c.window) % c.window;
  if (p < c.start[b]) return;
  const uint4* src = pool + (c.stage_base + first + (p - c.start[b])) * row16;
  uint4* dst = pool + (c.win_base[slot] + j) * row16;
  for (int i = threadIdx.x; i < row16; i += blockDim.x) dst[i] = src[i];
}

DSV4_ERROR_READER(chunk_rows)

}  // namespace chk

int check_chunk(const dsv4_chunk* c, const char* who) {
  DSV4_CHECK_ARG(c && c->cu_seqlens && c->start && c->win_base, "%s: NULL pointer in the chunk", who);
  DSV4_CHECK_ARG(c->n >= 0 && c->total >= 0 && c->slots > 0 && c->window > 0 && c->window % 64 == 0,
                 "%s: bad chunk sizes (window must be a multiple of 64)", who);
  DSV4_CHECK_ARG(c->seqs || c->n <= c->slots, "%s: more sequences than the cache has slots", who);
  DSV4_CHECK_ARG(c->max_comp >= 0 && (c->max_comp == 0 || (c->block_table && c->ratio > 0 && c->page > 0 &&
                                                           c->bt_stride * static_cast<int64_t>(c->page) >= c->max_comp)),
                 "%s: compressed rows need a block table that covers max_comp, a ratio and a page size", who);
  DSV4_CHECK_ARG(c->comp_base >= 0 && c->stage_base >= c->comp_base && c->pool_rows >= c->stage_base + c->total,
                 "%s: the staged rows do not fit behind the pages", who);
  DSV4_CHECK_ARG(c->pool_rows <= 0x7fffffffLL, "%s: at most 2^31 - 1 pool rows", who);
  return DSV4_OK;
}

}  // namespace dsv4

using namespace dsv4;

extern "C" int dsv4_chunk_rows(const dsv4_chunk* c, int32_t* positions, int64_t* stage_rows, int32_t* index,
                               int64_t index_stride, int32_t cols, const int32_t* given, void* stream) {
  const int rc = check_chunk(c, "dsv4_chunk_rows");
  if (rc != DSV4_OK) return rc;
  DSV4_CHECK_ARG(index == nullptr || (cols >= 0 && index_stride >= static_cast<int64_t>(c->window) + cols),
                 "dsv4_chunk_rows: index_stride holds less than window + cols");
  DSV4_CHECK_ARG(given == nullptr || index != nullptr, "dsv4_chunk_rows: given rows need an index to go to");
  if (c->n == 0 || c->total == 0) return DSV4_OK;
  const int threads = index ? 256 : 32;
  DSV4_CUDA_CHECK(launch_pdl(chk::chunk_rows_kernel, dim3(c->total), dim3(threads), 0, as_stream(stream), *c, positions,
                             stage_rows, index, index_stride, cols, given));
  return DSV4_OK;
}

extern "C" int dsv4_chunk_commit(const dsv4_chunk* c, void* pool, int32_t dim, void* stream) {
  const int rc = check_chunk(c, "dsv4_chunk_commit");
  if (rc != DSV4_OK) return rc;
  DSV4_CHECK_ARG(pool && dim > 0 && dim % 8 == 0 && (reinterpret_cast<uintptr_t>(pool) & 15) == 0,
                 "dsv4_chunk_commit: the pool must be 16-byte aligned bf16 rows of a multiple of 8 dims");
  if (c->n == 0 || c->total == 0) return DSV4_OK;
  DSV4_CHECK_ARG(c->n <= 65535, "dsv4_chunk_commit: at most 65535 sequences");
  DSV4_CUDA_CHECK(launch_pdl(chk::chunk_commit_kernel, dim3(c->window, c->n), dim3(64), 0, as_stream(stream), *c,
                             reinterpret_cast<uint4*>(pool), dim / 8));
  return DSV4_OK;
}
