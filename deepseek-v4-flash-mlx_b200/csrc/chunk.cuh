// A chunk of new tokens over the paged cache, as the kernels read it (dsv4_chunk of dsv4.h).
#pragma once
#include "common.cuh"

namespace dsv4 {

struct ChunkToken {
  int seq;    // index of the chunk's sequence, -1 behind the last one
  int first;  // its first token
  int start;  // position of that token
  int pos;    // position of this token
};

// whether a sequence is one that can be read: its tokens in the batch, positions that stay far from
// the end of an int, a slot of the cache
__device__ __forceinline__ bool chunk_valid(int first, int end, int total, int start, int slot, int slots) {
  return first >= 0 && end >= first && end <= total && start >= 0 && start <= 0x7fff0000 - total && slot >= 0 && slot < slots;
}

// the sequence of token t: the last b with cu_seqlens[b] <= t (empty sequences own no token); a token
// of a sequence that is not valid belongs to none
__device__ __forceinline__ ChunkToken chunk_token(const dsv4_chunk& c, int t) {
  ChunkToken k = {-1, 0, 0, 0};
  if (t >= c.cu_seqlens[c.n]) return k;
  int lo = 0, hi = c.n - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (c.cu_seqlens[mid] <= t)
      lo = mid;
    else
      hi = mid - 1;
  }
  k.first = c.cu_seqlens[lo];
  k.start = c.start[lo];
  const int end = c.cu_seqlens[lo + 1];
  if (t < k.first || t >= end) return k;
  if (chunk_valid(k.first, end, c.total, k.start, c.seqs ? c.seqs[lo] : lo, c.slots)) {
    k.seq = lo;
    k.pos = k.start + (t - k.first);
  } else {
    raise_device_error(DSV4_ERR_INDEX_OUT_OF_RANGE);
  }
  return k;
}

// compressed entries seen at position pos
__device__ __forceinline__ int chunk_seen(const dsv4_chunk& c, int pos) {
  if (c.max_comp == 0) return 0;
  const int e = (pos + 1) / c.ratio;
  return e < c.max_comp ? e : c.max_comp;
}

int check_chunk(const dsv4_chunk* c, const char* who);

}  // namespace dsv4
