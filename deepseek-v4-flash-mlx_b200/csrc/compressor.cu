// KV block compressor (ref_torch/compressor.py:21-50; decode ring oracle/decode_engine.py:96-105).
//
// Input: the two projections kv = x wkv^T and score = x wgate^T (fp32, [b, s, 2d]) from the
// projection GEMM. For compressed row g of a sequence, dim c in [0, d):
//   slots 0..3: kv[4g-4+r, c],      score[4g-4+r, c]   + ape[r, c]      (group 0: 0 / -inf)
//   slots 4..7: kv[4g+r,   d + c],  score[4g+r,   d + c] + ape[r, d + c]
//   pooled[c] = sum_slot softmax_slot(score) * kv
// then RMSNorm(norm_w), RoPE of the last rope_dim dims at position ratio*g (+pos0), and one
// 128-bit vectorised store per thread into the cache (bf16) or a plain fp32 output; rows can be
// scattered into a paged pool through out_rows. One CTA per compressed row, one thread per two
// dims (up to 256 threads, whole warps). The decode kernel keeps the per-sequence ring [2*ratio, 2d] on the device.
#include <algorithm>

#include "chunk.cuh"
#include "common.cuh"
#include "key_image.cuh"
#include "tcgen05.cuh"

namespace dsv4 {
namespace cmp {

constexpr int THREADS = 256;

__device__ __forceinline__ float block_sum(float v, float* red) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  v = warp_sum(v);
  if (lane == 0) red[warp] = v;
  __syncthreads();
  float t = 0.f;
  if (threadIdx.x < 32) {
    t = threadIdx.x < (blockDim.x >> 5) ? red[threadIdx.x] : 0.f;
    t = warp_sum(t);
    if (threadIdx.x == 0) red[32] = t;
  }
  __syncthreads();
  return red[32];
}

__device__ __forceinline__ float block_max(float v, float* red) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  v = warp_max(v);
  if (lane == 0) red[warp] = v;
  __syncthreads();
  float t = 0.f;
  if (threadIdx.x < 32) {
    t = threadIdx.x < (blockDim.x >> 5) ? red[threadIdx.x] : 0.f;
    t = warp_max(t);
    if (threadIdx.x == 0) red[32] = t;
  }
  __syncthreads();
  return red[32];
}

__device__ __forceinline__ void store_pair(float v0, float v1, int c, int d, void* out, int64_t orow, int out_dtype) {
  if (orow < 0) return;  // an entry whose page is not assigned: dsv4_decode_rows has raised the error word
  const int64_t off = orow * d + c;
  if (out_dtype == DSV4_BF16)
    *reinterpret_cast<uint32_t*>(reinterpret_cast<__nv_bfloat16*>(out) + off) = pack_bf16x2(v0, v1);
  else
    *reinterpret_cast<float2*>(reinterpret_cast<float*>(out) + off) = make_float2(v0, v1);
}

// The indexer compressor's key simulation (act_quant mode 2; v4mlx/compressor.py:57-59 with
// v4mlx/qat.py:8-31) on a 128-dim row held as pairs (2 tid, 2 tid + 1) by threads 0..63: the
// normalised Walsh-Hadamard transform (width-1 butterflies in the thread, widths 2..32 across lanes,
// width 64 across the two warps through `xch`, then float32(128^-0.5)), and the fp4-e2m1 round
// trip per 32-dim block (16 lanes). Every thread of the CTA calls it (one barrier).
__device__ __forceinline__ void hadamard_fp4_128(float& v0, float& v1, float* xch) {
  const int tid = threadIdx.x, lane = tid & 31;
  const bool mine = tid < 64;
  const float a = v0 + v1, b = v0 - v1;
  v0 = a;
  v1 = b;
#pragma unroll
  for (int o = 1; o <= 16; o <<= 1) {
    const float p0 = __shfl_xor_sync(0xffffffffu, v0, o), p1 = __shfl_xor_sync(0xffffffffu, v1, o);
    if (lane & o) {
      v0 = p0 - v0;
      v1 = p1 - v1;
    } else {
      v0 = v0 + p0;
      v1 = v1 + p1;
    }
  }
  if (mine) {
    xch[2 * tid] = v0;
    xch[2 * tid + 1] = v1;
  }
  __syncthreads();
  if (mine) {
    const float p0 = xch[2 * (tid ^ 32)], p1 = xch[2 * (tid ^ 32) + 1];
    if (tid & 32) {
      v0 = p0 - v0;
      v1 = p1 - v1;
    } else {
      v0 = v0 + p0;
      v1 = v1 + p1;
    }
    v0 *= 0.08838834764831845f;  // float32(128^-0.5)
    v1 *= 0.08838834764831845f;
  }
  float m = fmaxf(fabsf(v0), fabsf(v1));
#pragma unroll
  for (int o = 1; o <= 8; o <<= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  if (mine) {
    const int e = fp4_exp(m);
    const float dn = __uint_as_float(static_cast<uint32_t>(127 - e) << 23);
    const float up = __uint_as_float(static_cast<uint32_t>(127 + e) << 23);
    v0 = e2m1_round(fminf(fmaxf(v0 * dn, -6.f), 6.f)) * up;
    v1 = e2m1_round(fminf(fmaxf(v1 * dn, -6.f), 6.f)) * up;
  }
}

// normalise, rope and store two adjacent dims (c, c+1) of one compressed row; the stored values
// (before the cast) are left in v0, v1. In act_quant mode 2 the pair is left unstored for
// hadamard_fp4_128 and store_pair.
__device__ __forceinline__ void finish_pair(float& v0, float& v1, int c, int d, int rope_dim,
                                            const void* norm_w, int norm_dtype, float rinv,
                                            const float* freqs, int pos, void* out, int64_t orow,
                                            int out_dtype, int act_quant) {
  v0 = v0 * rinv;
  v1 = v1 * rinv;
  if (norm_w) {
    v0 = load_as_float(norm_w, c, norm_dtype) * v0;
    v1 = load_as_float(norm_w, c + 1, norm_dtype) * v1;
  }
  if (c >= d - rope_dim) {
    float cs, sn;
    rope_cos_sin(pos, freqs[(c - (d - rope_dim)) >> 1], &cs, &sn);
    rotate_pair(v0, v1, cs, sn, false, &v0, &v1);
  }
  // fp8 act-quant simulation of the nope dims: a 64-dim block is the 32 pairs of one warp (the
  // condition is warp-uniform)
  if (act_quant == 1 && c < d - rope_dim) {
    const int ex = act_quant_exp(warp_max(fmaxf(fabsf(v0), fabsf(v1))));
    v0 = fp8_round_pow2(v0, ex);
    v1 = fp8_round_pow2(v1, ex);
  }
  if (act_quant == 2) return;
  store_pair(v0, v1, c, d, out, orow, out_dtype);
}

// softmax over 8 slots (max-subtracted, as torch.softmax) and the weighted sum
__device__ __forceinline__ float pool8(const float* kv8, const float* sc8) {
  float m = sc8[0];
#pragma unroll
  for (int i = 1; i < 8; ++i) m = fmaxf(m, sc8[i]);
  float den = 0.f, num = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    float e = expf(sc8[i] - m);
    den += e;
    num = fmaf(e, kv8[i], num);
  }
  return num / den;
}

// One CTA per compressed row; blockDim = the row's pairs of dims rounded up to whole warps (at
// most THREADS), so a 128-dim row (the indexer compressor) runs 64 threads, none idle.
__global__ void __launch_bounds__(THREADS) pool_kernel(dsv4_compressor_params p) {
  pdl_wait();  // programmatic dependent launch: the previous kernel is complete from here
  pdl_trigger();
  __shared__ float red[33];
  const int groups = p.s / p.ratio;
  const int64_t rowid = blockIdx.x;  // b * groups + g
  const int b = static_cast<int>(rowid / groups);
  const int g = static_cast<int>(rowid % groups);
  const int d = p.head_dim, d2 = 2 * d;
  const int R = p.ratio;
  const float* kvb = p.kv + static_cast<int64_t>(b) * p.s * d2;
  const float* scb = p.score + static_cast<int64_t>(b) * p.s * d2;
  float vals[2][2];  // up to 2 pairs per thread (d <= 1024)
  float ss = 0.f;
  int npairs = 0;
  for (int c = threadIdx.x * 2; c < d; c += blockDim.x * 2, ++npairs) {
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      float kv8[16], sc8[16];
      const int cc = c + e;
      for (int r = 0; r < R; ++r) {
        if (g > 0) {
          const int64_t t = static_cast<int64_t>(g - 1) * R + r;
          kv8[r] = kvb[t * d2 + cc];
          sc8[r] = scb[t * d2 + cc] + p.ape[r * d2 + cc];
        } else {
          kv8[r] = 0.f;
          sc8[r] = -INFINITY;
        }
        const int64_t t2 = static_cast<int64_t>(g) * R + r;
        kv8[R + r] = kvb[t2 * d2 + d + cc];
        sc8[R + r] = scb[t2 * d2 + d + cc] + p.ape[r * d2 + d + cc];
      }
      float v;
      if (R == 4) {
        v = pool8(kv8, sc8);
      } else {
        float m = sc8[0];
        for (int i = 1; i < 2 * R; ++i) m = fmaxf(m, sc8[i]);
        float den = 0.f, num = 0.f;
        for (int i = 0; i < 2 * R; ++i) {
          float ex = expf(sc8[i] - m);
          den += ex;
          num = fmaf(ex, kv8[i], num);
        }
        v = num / den;
      }
      vals[npairs][e] = v;
      ss = fmaf(v, v, ss);
    }
  }
  ss = block_sum(ss, red);
  const float rinv = rsqrtf(ss / static_cast<float>(d) + p.eps);
  const int64_t orow = p.out_rows ? p.out_rows[rowid] : rowid;
  npairs = 0;
  for (int c = threadIdx.x * 2; c < d; c += blockDim.x * 2, ++npairs)
    finish_pair(vals[npairs][0], vals[npairs][1], c, d, p.rope_dim, p.norm_w, p.norm_dtype, rinv,
                p.freqs, p.pos0 + R * g, p.out, orow, p.out_dtype, p.act_quant);
  if (p.act_quant == 2) {  // head_dim 128: threads 0..63 hold the row (uniform over the CTA)
    __shared__ float xch[128];
    hadamard_fp4_128(vals[0][0], vals[0][1], xch);
    if (threadIdx.x < 64) store_pair(vals[0][0], vals[0][1], 2 * threadIdx.x, d, p.out, orow, p.out_dtype);
  }
}

// decode hand-off ring (ref_torch/compressor.py:67-74; seeding as oracle/decode_engine.py:91-95):
// rows [0, R) = last full block (kv, score+ape), rows [R, R+rem) = remainder, rest 0 / -inf.
__global__ void ring_seed_kernel(dsv4_compressor_params p) {
  pdl_wait();  // programmatic dependent launch: the previous kernel is complete from here
  pdl_trigger();
  const int b = blockIdx.y;
  const int slot = blockIdx.x;  // 0 .. 2R-1
  const int R = p.ratio, d2 = 2 * p.head_dim;
  const int cutoff = p.s - p.s % R;
  const int rem = p.s % R;
  int64_t t = -1;
  int ape_r = 0;
  if (slot < R) {
    if (cutoff >= R) {
      t = cutoff - R + slot;
      ape_r = slot;
    }
  } else if (slot - R < rem) {
    t = cutoff + (slot - R);
    ape_r = slot - R;
  }
  float* rk = p.ring_kv + (static_cast<int64_t>(b) * 2 * R + slot) * d2;
  float* rs = p.ring_score + (static_cast<int64_t>(b) * 2 * R + slot) * d2;
  const float* kvb = p.kv + static_cast<int64_t>(b) * p.s * d2;
  const float* scb = p.score + static_cast<int64_t>(b) * p.s * d2;
  for (int c = threadIdx.x; c < d2; c += blockDim.x) {
    if (t >= 0) {
      rk[c] = kvb[t * d2 + c];
      rs[c] = scb[t * d2 + c] + p.ape[ape_r * d2 + c];
    } else {
      rk[c] = 0.f;
      rs[c] = -INFINITY;
    }
  }
}

// one decode token per sequence: ring row R + p%R <- (kv, score + ape[p%R]); when (p+1)%R == 0
// emit the pooled row at position p+1-R and shift rows [R,2R) to [0,R). Block 0 has none before it: rows
// [0,R) then count as empty (kv 0, score -inf) whatever they hold, so that a slot that begins again takes
// nothing from the sequence it held.
// ratio 4 (the model's): the same step with every thread owning column pairs (c, c+1) of both
// halves. The ring rows it reads were written by earlier steps and the current token's row stays
// in registers, so all of a thread's loads go out at once and the only barrier is the norm's
// reduction (the generic kernel below re-reads the ring it just wrote, behind a barrier, with
// runtime-sized loops). Same operations in the same order: identical results.
__device__ __forceinline__ float2 ld2(const float* p) { return *reinterpret_cast<const float2*>(p); }
__device__ __forceinline__ void st2(float* p, float2 v) { *reinterpret_cast<float2*>(p) = v; }

// the emitted row (indexer key, head_dim 128 = 64 pairs held by threads 0..63, fp32 values as
// stored) added to the key image: scaled and split as dsv4_indexer_key_image does it, its inverse
// scale, and the entry's norm maximum raised
__device__ __forceinline__ void append_key_row(float v0, float v1, int head_dim, uint8_t* key_image, float* key_inv,
                                               float* key_norm_max, int64_t image_stride, int64_t seq, int64_t j,
                                               float* red) {
  const int tid = threadIdx.x;
  const bool mine = 2 * tid < head_dim;
  if (!mine) v0 = v1 = 0.f;
  const float mx = block_max(fmaxf(fabsf(v0), fabsf(v1)), red);
  const float ss = block_sum(fmaf(v1, v1, v0 * v0), red);
  const int64_t tiles = (image_stride + 127) / 128;
  const int sh = itc::row_shift(mx);
  if (mine) {
    uint32_t hi, lo;
    const float up = itc::pow2(sh);
    itc::split2(v0 * up, v1 * up, &hi, &lo);
    const int c = 2 * tid;
    uint8_t* img = key_image + (seq * tiles + j / 128) * itc::IMG_TILE_BYTES;
    const uint32_t off = itc::key_off(static_cast<int>(j % 128), c >> 2) + ((c >> 1) & 1) * 4;
    *reinterpret_cast<uint32_t*>(img + off) = hi;
    *reinterpret_cast<uint32_t*>(img + off + itc::IMG_SLAB_K) = lo;
  }
  if (tid == 0) {
    key_inv[seq * tiles * 128 + j] = itc::pow2(-sh);
    atomicMax(reinterpret_cast<unsigned int*>(key_norm_max + seq), __float_as_uint(sqrtf(ss)));
  }
}
template <int NP>
__device__ __forceinline__ void append_key_image(const dsv4_compressor_decode_params& p, const float (&vals)[NP][2],
                                                 float* red) {
  const bool mine = 2 * static_cast<int>(threadIdx.x) < p.head_dim;
  const int64_t orow = p.out_rows[blockIdx.x];
  append_key_row(mine ? vals[0][0] : 0.f, mine ? vals[0][1] : 0.f, p.head_dim, p.key_image, p.key_inv, p.key_norm_max,
                 p.image_stride, orow / p.image_stride, orow % p.image_stride, red);
}

// the ratio-4 step of sequence blockIdx.x for one compressor (the body of decode_r4_kernel)
template <int NP>
__device__ __forceinline__ void decode_r4_row(const dsv4_compressor_decode_params& p) {
  constexpr int R = 4;
  __shared__ float red[33];
  const int b = blockIdx.x, tid = threadIdx.x;
  const int d = p.head_dim, d2 = 2 * d;
  const int pos = p.positions[b];
  const int slot = R + pos % R;
  float* rk = p.ring_kv + static_cast<int64_t>(b) * 2 * R * d2;
  float* rs = p.ring_score + static_cast<int64_t>(b) * 2 * R * d2;
  const float* kin = p.kv + static_cast<int64_t>(b) * d2;
  const float* sin_ = p.score + static_cast<int64_t>(b) * d2;
  const float* ape = p.ape + (pos % R) * d2;
  const bool emit = (pos + 1) % R == 0;
  float2 nk[NP][2], ns[NP][2];  // this token's kv and score + ape, columns c and d + c
  float2 K[NP][8], S[NP][8], F[NP][3], G[NP][3];  // pooled inputs; rows 4..6 of the first half (shift)
#pragma unroll
  for (int np = 0; np < NP; ++np) {
    const int c = 2 * (tid + np * THREADS);
    if (c >= d) continue;
    nk[np][0] = ld2(kin + c);
    nk[np][1] = ld2(kin + d + c);
    const float2 s0 = ld2(sin_ + c), s1 = ld2(sin_ + d + c), a0 = ld2(ape + c), a1 = ld2(ape + d + c);
    ns[np][0] = make_float2(s0.x + a0.x, s0.y + a0.y);
    ns[np][1] = make_float2(s1.x + a1.x, s1.y + a1.y);
    if (emit) {
#pragma unroll
      for (int r = 0; r < R; ++r) {
        K[np][r] = pos < R ? make_float2(0.f, 0.f) : ld2(rk + r * d2 + c);
        S[np][r] = pos < R ? make_float2(-INFINITY, -INFINITY) : ld2(rs + r * d2 + c);
      }
#pragma unroll
      for (int r = 0; r < R - 1; ++r) {
        K[np][R + r] = ld2(rk + (R + r) * d2 + d + c);
        S[np][R + r] = ld2(rs + (R + r) * d2 + d + c);
        F[np][r] = ld2(rk + (R + r) * d2 + c);
        G[np][r] = ld2(rs + (R + r) * d2 + c);
      }
      K[np][2 * R - 1] = nk[np][1];  // row 2R - 1 is this token's slot
      S[np][2 * R - 1] = ns[np][1];
    }
    // the slot is written in every case (after an emission the ring holds what the generic kernel
    // leaves: this token's row both in its slot and, shifted, in row R - 1)
    st2(rk + slot * d2 + c, nk[np][0]);
    st2(rk + slot * d2 + d + c, nk[np][1]);
    st2(rs + slot * d2 + c, ns[np][0]);
    st2(rs + slot * d2 + d + c, ns[np][1]);
  }
  if (!emit) return;  // uniform over the CTA
  float vals[NP][2];
  float ss = 0.f;
#pragma unroll
  for (int np = 0; np < NP; ++np) {
    const int c = 2 * (tid + np * THREADS);
    if (c >= d) continue;
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      float m = e ? S[np][0].y : S[np][0].x;
#pragma unroll
      for (int i = 1; i < 2 * R; ++i) m = fmaxf(m, e ? S[np][i].y : S[np][i].x);
      float den = 0.f, num = 0.f;
#pragma unroll
      for (int i = 0; i < 2 * R; ++i) {
        const float ex = expf((e ? S[np][i].y : S[np][i].x) - m);
        den += ex;
        num = fmaf(ex, e ? K[np][i].y : K[np][i].x, num);
      }
      vals[np][e] = num / den;
      ss = fmaf(vals[np][e], vals[np][e], ss);
    }
  }
  ss = block_sum(ss, red);
  const float rinv = rsqrtf(ss / static_cast<float>(d) + p.eps);
#pragma unroll
  for (int np = 0; np < NP; ++np) {
    const int c = 2 * (tid + np * THREADS);
    if (c >= d) continue;
    finish_pair(vals[np][0], vals[np][1], c, d, p.rope_dim, p.norm_w, p.norm_dtype, rinv, p.freqs, pos + 1 - R,
                p.out, p.out_rows[b], p.out_dtype, p.act_quant);
    // the block's rows become the previous block (rows 0..R-1); this token's row is the last
#pragma unroll
    for (int r = 0; r < R - 1; ++r) {
      st2(rk + r * d2 + c, F[np][r]);
      st2(rs + r * d2 + c, G[np][r]);
      st2(rk + r * d2 + d + c, K[np][R + r]);
      st2(rs + r * d2 + d + c, S[np][R + r]);
    }
    st2(rk + (R - 1) * d2 + c, nk[np][0]);
    st2(rs + (R - 1) * d2 + c, ns[np][0]);
    st2(rk + (R - 1) * d2 + d + c, nk[np][1]);
    st2(rs + (R - 1) * d2 + d + c, ns[np][1]);
  }
  if (p.act_quant == 2) {  // head_dim 128: threads 0..63 hold the row (uniform over the CTA)
    __shared__ float xch[128];
    hadamard_fp4_128(vals[0][0], vals[0][1], xch);
    if (tid < 64) store_pair(vals[0][0], vals[0][1], 2 * tid, d, p.out, p.out_rows[b], p.out_dtype);
  }
  if (p.key_image) append_key_image<NP>(p, vals, red);
}

template <int NP>
__global__ void __launch_bounds__(THREADS) decode_r4_kernel(dsv4_compressor_decode_params p) {
  pdl_wait();  // programmatic dependent launch: the previous kernel is complete from here
  pdl_trigger();
  decode_r4_row<NP>(p);
}

// two compressors' steps in one launch (grid.y = 2; the same batch): a decode block's main and
// indexer compressors, which read the same token's projections and write disjoint rings and rows
template <int NP>
__global__ void __launch_bounds__(THREADS) decode_r4_pair_kernel(dsv4_compressor_decode_params p0,
                                                                 dsv4_compressor_decode_params p1) {
  pdl_wait();
  pdl_trigger();
  const dsv4_compressor_decode_params& p = blockIdx.y ? p1 : p0;
  decode_r4_row<NP>(p);
}

__global__ void __launch_bounds__(THREADS) decode_kernel(dsv4_compressor_decode_params p) {
  pdl_wait();  // programmatic dependent launch: the previous kernel is complete from here
  pdl_trigger();
  __shared__ float red[33];
  const int b = blockIdx.x;
  const int R = p.ratio, d = p.head_dim, d2 = 2 * d;
  const int pos = p.positions[b];
  const int slot = R + pos % R;
  float* rk = p.ring_kv + static_cast<int64_t>(b) * 2 * R * d2;
  float* rs = p.ring_score + static_cast<int64_t>(b) * 2 * R * d2;
  const float* kin = p.kv + static_cast<int64_t>(b) * d2;
  const float* sin_ = p.score + static_cast<int64_t>(b) * d2;
  for (int c = threadIdx.x; c < d; c += blockDim.x) {
    rk[slot * d2 + c] = kin[c];
    rk[slot * d2 + d + c] = kin[d + c];
    rs[slot * d2 + c] = sin_[c] + p.ape[(pos % R) * d2 + c];
    rs[slot * d2 + d + c] = sin_[d + c] + p.ape[(pos % R) * d2 + d + c];
  }
  if ((pos + 1) % R != 0) return;
  __syncthreads();  // the pooled read below covers dims written by other threads
  float vals[2][2];
  float ss = 0.f;
  int np = 0;
  for (int c = threadIdx.x * 2; c < d; c += THREADS * 2, ++np) {
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int cc = c + e;
      float kv8[16], sc8[16];
      for (int r = 0; r < R; ++r) {
        kv8[r] = pos < R ? 0.f : rk[r * d2 + cc];
        sc8[r] = pos < R ? -INFINITY : rs[r * d2 + cc];
        kv8[R + r] = rk[(R + r) * d2 + d + cc];
        sc8[R + r] = rs[(R + r) * d2 + d + cc];
      }
      float m = sc8[0];
      for (int i = 1; i < 2 * R; ++i) m = fmaxf(m, sc8[i]);
      float den = 0.f, num = 0.f;
      for (int i = 0; i < 2 * R; ++i) {
        float ex = expf(sc8[i] - m);
        den += ex;
        num = fmaf(ex, kv8[i], num);
      }
      vals[np][e] = num / den;
      ss = fmaf(vals[np][e], vals[np][e], ss);
    }
  }
  ss = block_sum(ss, red);  // its barrier also orders the pooled reads before the shift below
  const float rinv = rsqrtf(ss / static_cast<float>(d) + p.eps);
  np = 0;
  for (int c = threadIdx.x * 2; c < d; c += THREADS * 2, ++np)
    finish_pair(vals[np][0], vals[np][1], c, d, p.rope_dim, p.norm_w, p.norm_dtype, rinv, p.freqs,
                pos + 1 - R, p.out, p.out_rows[b], p.out_dtype, p.act_quant);
  if (p.act_quant == 2) {  // head_dim 128: threads 0..63 hold the row (uniform over the CTA)
    __shared__ float xch[128];
    hadamard_fp4_128(vals[0][0], vals[0][1], xch);
    if (threadIdx.x < 64)
      store_pair(vals[0][0], vals[0][1], 2 * threadIdx.x, d, p.out, p.out_rows[b], p.out_dtype);
  }
  for (int c = threadIdx.x; c < d2; c += blockDim.x)
    for (int r = 0; r < R; ++r) {
      rk[r * d2 + c] = rk[(R + r) * d2 + c];
      rs[r * d2 + c] = rs[(R + r) * d2 + c];
    }
}

// ---- a chunk of new tokens per sequence (dsv4_compressor_chunk): what R = ratio calls of the
// decode step per emitted row would leave, in one launch. Block g of a sequence is emitted when its
// last token, position R g + R - 1, is in the chunk; its tokens and those of block g - 1 come from
// the chunk where it has them and from the ring otherwise (rows [0, R): the last complete block,
// rows R + p % R: the tokens of the block begun before the chunk; before position 0 there are none, kv 0 and
// score -inf whatever the ring holds).
//
// Every element of the projections is used once (the first half of a token's columns by the next
// block's row, the second half by its own), so the kernel is a stream of 16 * head_dim bytes per
// token and bound by HBM. A CTA takes the rows emitted by four neighbouring tokens, one in a long
// chunk, up to four where every sequence has a token or two; each thread owns pairs of columns and
// has all 4 R of its loads in flight before the first is used. The rows that read the ring (at most
// the first two of a sequence) and the ring's own update belong to one CTA per sequence, so no
// order between CTAs is needed: a thread reads the ring's columns it owns before it writes them.
// The prefix grid (the sequences' CTAs, the slowest) is launched first.
template <int R>
struct ChunkSeq {
  int first, n, start, slot;  // first token, tokens, position of the first, cache slot
};

// the table's word on entry g of a slot (0 without a table), to be asked for well before chunk_row needs it
__device__ __forceinline__ int32_t chunk_page(const dsv4_compressor_chunk_params& p, int slot, int g) {
  return p.block_table != nullptr && g < p.max_comp ? p.block_table[static_cast<int64_t>(slot) * p.bt_stride + g / p.page] : 0;
}
// where entry g of a slot goes; -1 (and the error word) past the cache, without a page or outside of out
__device__ __forceinline__ int64_t chunk_row(const dsv4_compressor_chunk_params& p, int slot, int g, int32_t page) {
  int64_t row = -1;
  if (g < p.max_comp && page >= 0)
    row = p.out_base + (p.block_table == nullptr ? static_cast<int64_t>(slot) * p.max_comp + g
                                                 : static_cast<int64_t>(page) * p.page + g % p.page);
  if (row < 0 || row >= p.out_rows) {
    raise_device_error(DSV4_ERR_INDEX_OUT_OF_RANGE);
    return -1;
  }
  return row;
}
// one column of a row: the softmax over its 2 R slots
template <int R>
__device__ __forceinline__ float chunk_pool(const float2 (&K)[2 * R], const float2 (&S)[2 * R], int e) {
  float m = e ? S[0].y : S[0].x;
#pragma unroll
  for (int i = 1; i < 2 * R; ++i) m = fmaxf(m, e ? S[i].y : S[i].x);
  float den = 0.f, num = 0.f;
#pragma unroll
  for (int i = 0; i < 2 * R; ++i) {
    const float ex = expf((e ? S[i].y : S[i].x) - m);
    den += ex;
    num = fmaf(ex, e ? K[i].y : K[i].x, num);
  }
  return num / den;
}

template <int R>
__device__ __forceinline__ void chunk_emit(const dsv4_compressor_chunk_params& p, const ChunkSeq<R>& q, int g,
                                           float* red, float* xch) {
  const int d = p.head_dim, d2 = 2 * d;
  const float* rk = p.ring_kv + static_cast<int64_t>(q.slot) * 2 * R * d2;
  const float* rs = p.ring_score + static_cast<int64_t>(q.slot) * 2 * R * d2;
  const int block = q.start / R * R;  // the block the chunk begins in
  const int32_t page = chunk_page(p, q.slot, g);
  float vals[2][2];
  float ss = 0.f;
#pragma unroll
  for (int np = 0; np < 2; ++np) {
    const int c = 2 * (threadIdx.x + np * THREADS);
    if (c >= d) continue;
    float2 K[2 * R], S[2 * R];
#pragma unroll
    for (int i = 0; i < 2 * R; ++i) {
      const int pos = (g - 1) * R + i;  // slots [0, R): block g - 1, first half of the columns
      const int col = c + (i < R ? 0 : d);
      if (pos >= q.start) {
        const int64_t off = static_cast<int64_t>(q.first + (pos - q.start)) * d2 + col;
        K[i] = ld2(p.kv + off);
        const float2 s = ld2(p.score + off), a = ld2(p.ape + (i % R) * d2 + col);
        S[i] = make_float2(s.x + a.x, s.y + a.y);
      } else if (pos < 0) {  // not the ring's rows: they may be those of another sequence
        K[i] = make_float2(0.f, 0.f);
        S[i] = make_float2(-INFINITY, -INFINITY);
      } else {
        const int row = (pos >= block ? R : 0) + i % R;
        K[i] = ld2(rk + row * d2 + col);
        S[i] = ld2(rs + row * d2 + col);
      }
    }
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      vals[np][e] = chunk_pool<R>(K, S, e);
      ss = fmaf(vals[np][e], vals[np][e], ss);
    }
  }
  ss = block_sum(ss, red);
  const int64_t orow = chunk_row(p, q.slot, g, page);
  const float rinv = rsqrtf(ss / static_cast<float>(d) + p.eps);
#pragma unroll
  for (int np = 0; np < 2; ++np) {
    const int c = 2 * (threadIdx.x + np * THREADS);
    if (c >= d) continue;
    finish_pair(vals[np][0], vals[np][1], c, d, p.rope_dim, p.norm_w, p.norm_dtype, rinv, p.freqs, R * g, p.out, orow,
                p.out_dtype, p.act_quant);
  }
  if (p.act_quant == 2) {  // head_dim 128: threads 0..63 hold the row (uniform over the CTA)
    hadamard_fp4_128(vals[0][0], vals[0][1], xch);
    if (threadIdx.x < 64) store_pair(vals[0][0], vals[0][1], 2 * threadIdx.x, d, p.out, orow, p.out_dtype);
  }
  if (p.key_image && g < p.max_comp)
    append_key_row(vals[0][0], vals[0][1], d, p.key_image, p.key_inv, p.key_norm_max, p.max_comp, q.slot, g, red);
  __syncthreads();  // red and xch are free for the next row
}

// the chunk's sequence b; n == 0 where there is nothing to do or the chunk is not a valid one
template <int R>
__device__ __forceinline__ ChunkSeq<R> chunk_seq(const dsv4_compressor_chunk_params& p, int b) {
  ChunkSeq<R> q;
  q.first = p.cu_seqlens[b];
  const int end = p.cu_seqlens[b + 1];
  q.start = p.start[b];
  q.slot = p.seqs ? p.seqs[b] : b;
  q.n = end - q.first;
  if (!chunk_valid(q.first, end, p.total, q.start, q.slot, p.slots)) {
    raise_device_error(DSV4_ERR_INDEX_OUT_OF_RANGE);
    q.n = 0;
  }
  return q;
}

// the rows of sequence b that read its ring (at most two), then the ring
// (any number of threads that covers a row: those past it add nothing)
template <int R>
__device__ __forceinline__ void chunk_sequence(const dsv4_compressor_chunk_params& p, int b, float* red, float* xch) {
  const ChunkSeq<R> q = chunk_seq<R>(p, b);
  if (q.n <= 0) return;
  // a slot named twice: an error (nothing waits for the look), and the rows and ring of that slot are either's
  if (p.seqs != nullptr)
    for (int i = threadIdx.x; i < b; i += blockDim.x)
      if (p.seqs[i] == q.slot && p.cu_seqlens[i + 1] > p.cu_seqlens[i]) raise_device_error(DSV4_ERR_INDEX_OUT_OF_RANGE);
  const int end = q.start + q.n, g0 = q.start / R, g1 = end / R;
  for (int g = g0; g < g1 && (g - 1) * R < q.start; ++g) chunk_emit<R>(p, q, g, red, xch);
  // the ring after the chunk: rows [0, R) the last complete block, rows R + p % R the newest token
  const int d2 = 2 * p.head_dim;
  float* rk = p.ring_kv + static_cast<int64_t>(q.slot) * 2 * R * d2;
  float* rs = p.ring_score + static_cast<int64_t>(q.slot) * 2 * R * d2;
  for (int c = 2 * threadIdx.x; c < d2; c += 2 * blockDim.x) {
#pragma unroll
    for (int i = 0; i < R; ++i) {
      const int last = end - 1 - (end - 1 - i + R) % R;  // newest position with p % R == i
      if (g1 > g0) {
        const int pos = (g1 - 1) * R + i;
        if (pos >= q.start) {
          const int64_t off = static_cast<int64_t>(q.first + (pos - q.start)) * d2 + c;
          const float2 s = ld2(p.score + off), a = ld2(p.ape + i * d2 + c);
          st2(rk + i * d2 + c, ld2(p.kv + off));
          st2(rs + i * d2 + c, make_float2(s.x + a.x, s.y + a.y));
        } else {
          st2(rk + i * d2 + c, ld2(rk + (R + i) * d2 + c));
          st2(rs + i * d2 + c, ld2(rs + (R + i) * d2 + c));
        }
      }
      if (last >= q.start) {
        const int64_t off = static_cast<int64_t>(q.first + (last - q.start)) * d2 + c;
        const float2 s = ld2(p.score + off), a = ld2(p.ape + i * d2 + c);
        st2(rk + (R + i) * d2 + c, ld2(p.kv + off));
        st2(rs + (R + i) * d2 + c, make_float2(s.x + a.x, s.y + a.y));
      }
    }
  }
}

// The long-chunk form of the rows that need no ring (R = 4, head_dim a multiple of 64 up to 512): a CTA
// takes up to `run` blocks of a sequence one after the other, G rows at a time, a group of threads each. A
// block's tokens are consecutive, so one bulk copy each brings kv and score (16 KB each at 512 dims) into a
// ring of 2 G + 1 buffers, G blocks ahead of those that are computed and without a thread waiting for any
// address; every block is read once and serves two rows, but for the one before a run (half of its columns
// again, 1 / run). The arithmetic is about 490 instructions a warp and row (16 exponentials and 2 divisions
// a thread, as the decode step has them), so as many warps as registers allow run at once: 512 dims with G = 3
// (24 warps, 224 KB) in one CTA an SM. The row-at-a-time form above looks its row up, loads, sums and stores in
// turn: 53 us for 16384 tokens; two CTAs of G = 1 took 33 us, this 30 (139 MB, 4.6 TB/s). Neither the issue slots
// (40% used) nor HBM (50%) bound it: the CTA's barrier of every round, at which three groups wait for the slowest, is the
// longest stall.
template <int D, int G>  // D: head_dim where it is known (addresses fold into the loads), 0: any
struct Run {
  static constexpr int STAGES = 2 * G + 1;
};
template <int D, int G>
__global__ void __launch_bounds__(G == 1 ? THREADS : G * D / 2, G == 1 ? 2 : 1)
    chunk_run_kernel(dsv4_compressor_chunk_params p, int run) {
  constexpr int R = 4, STAGES = Run<D, G>::STAGES;
  static_assert(G == 1 || D == 2 * THREADS, "groups of THREADS");
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ float red[33];
  __shared__ float sums[G][THREADS / 32];
  __shared__ int64_t where[G];
  __shared__ float xch[128];
  if (static_cast<int>(blockIdx.x) < p.n) {
    pdl_wait();
    pdl_trigger();
    chunk_sequence<R>(p, blockIdx.x, red, xch);
    return;
  }
  __shared__ uint64_t full[STAGES];
  __shared__ int unit[3];  // sequence, first block of the run, blocks
  const int lane = threadIdx.x & 31, group = G == 1 ? 0 : threadIdx.x / THREADS;
  const int tid = G == 1 ? threadIdx.x : threadIdx.x % THREADS;  // in the group
  const int d = D ? D : p.head_dim, d2 = 2 * d;
  const uint32_t half = static_cast<uint32_t>(R * d2 * 4), stage = 2 * half;  // bytes of a block's kv, of both
  if (threadIdx.x == 0) {
    for (int i = 0; i < STAGES; ++i) tc5::bar_init(&full[i], 1);
    tc5::bar_init_fence();
  }
  pdl_wait();
  pdl_trigger();
  if (threadIdx.x < 32) {  // the run of this CTA, counted through the sequences
    int before = 0;
    bool found = false;
    for (int b0 = 0; b0 < p.n && !found; b0 += 32) {
      const int b = b0 + lane;
      int gs = 0, ge = 0;
      if (b < p.n) {
        const int first = p.cu_seqlens[b], last = p.cu_seqlens[b + 1], start = p.start[b];
        const int slot = p.seqs ? p.seqs[b] : b;
        // the blocks whose row needs no token of before the chunk (invalid sequences: reported elsewhere)
        if (chunk_valid(first, last, p.total, start, slot, p.slots)) {
          gs = (start + R - 1) / R + 1;
          ge = max(gs, (start + last - first) / R);
        }
      }
      const int cnt = (ge - gs + run - 1) / run;
      int s = cnt;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int x = __shfl_up_sync(0xffffffffu, s, o);
        if (lane >= o) s += x;
      }
      const int at = before + s - cnt, want = static_cast<int>(blockIdx.x) - p.n;
      const bool hit = want >= at && want < at + cnt;
      if (hit) {
        unit[0] = b;
        unit[1] = gs + (want - at) * run;
        unit[2] = min(run, ge - unit[1]);
      }
      found = __any_sync(0xffffffffu, hit);
      before += __shfl_sync(0xffffffffu, s, 31);
    }
    if (!found && lane == 0) unit[2] = 0;
  }
  __syncthreads();
  const int nb = unit[2];
  if (nb == 0) return;
  const int b = unit[0], g0 = unit[1];
  const int first = p.cu_seqlens[b], start = p.start[b], slot = p.seqs ? p.seqs[b] : b;
  const float* kv = p.kv + static_cast<int64_t>(first + (g0 - 1) * R - start) * d2;  // block g0 - 1
  const float* sc = p.score + static_cast<int64_t>(first + (g0 - 1) * R - start) * d2;
  int issued = 0;
  auto load_to = [&](int end) {  // blocks g0 - 1 + issued .. g0 - 1 + end - 1
    if (threadIdx.x == 0)
      for (int i = issued; i < end; ++i) {
        uint8_t* dst = smem + (i % STAGES) * stage;
        tc5::bar_expect_tx(&full[i % STAGES], stage);
        tc5::bulk_g2s(dst, kv + static_cast<int64_t>(i) * R * d2, half, &full[i % STAGES]);
        tc5::bulk_g2s(dst + half, sc + static_cast<int64_t>(i) * R * d2, half, &full[i % STAGES]);
      }
    issued = max(issued, end);
  };
  load_to(min(STAGES, nb + 1));
  const int c = 2 * tid;  // this thread's columns c, c + 1 and d + c, d + c + 1
  const bool mine = c < d;
  float2 A[2 * R];
#pragma unroll
  for (int i = 0; i < 2 * R; ++i)
    A[i] = mine ? ld2(p.ape + (i % R) * d2 + c + (i < R ? 0 : d)) : make_float2(0.f, 0.f);
  // one thread of a group finds where its rows go, a round ahead
  int32_t next_page = tid == 0 && group < nb ? chunk_page(p, slot, g0 + group) : 0;
  bool ok = true;
  int sp = group, sc_ = group + 1;          // buffers of the row's two blocks, and their phases
  uint32_t pp = 0, pc = 0;
  for (int i0 = 1; i0 <= nb; i0 += G) {
    const int i = i0 + group, g = g0 - 1 + i;
    const bool row = i <= nb;
    float2 K[2 * R], S[2 * R];
    if (row) {
      if (tid == 0) {
        where[group] = chunk_row(p, slot, g, next_page);
        if (i + G <= nb) next_page = chunk_page(p, slot, g + G);
      }
      ok = tc5::bar_wait(&full[sp], pp) && tc5::bar_wait(&full[sc_], pc);
      if (mine) {
        const uint8_t* prev = smem + sp * stage + c * 4;
        const uint8_t* cur = smem + sc_ * stage + (d + c) * 4;
#pragma unroll
        for (int j = 0; j < 2 * R; ++j) {
          const uint8_t* src = (j < R ? prev : cur) + (j % R) * d2 * 4;
          K[j] = *reinterpret_cast<const float2*>(src);
          const float2 s = *reinterpret_cast<const float2*>(src + half);
          S[j] = make_float2(s.x + A[j].x, s.y + A[j].y);
        }
      }
    }
    sp += G;
    if (sp >= STAGES) sp -= STAGES, pp ^= 1;
    sc_ += G;
    if (sc_ >= STAGES) sc_ -= STAGES, pc ^= 1;
    if (__syncthreads_or(!ok)) {
      if (threadIdx.x == 0) raise_device_error(DSV4_ERR_WAIT_TIMEOUT);
      ok = false;  // of every thread: the one that waits for the copies below is not the one whose wait ran out
      break;
    }
    load_to(min(nb + 1, i0 + G - 1 + STAGES));  // blocks up to i0 + G - 2 have been read
    if (!row) continue;
    // Between the CTA's barrier above, behind which the write of `where` lies, and the group's barrier below, ahead
    // of the next round's write: read behind the group's barrier it would race with that write.
    const int64_t orow = where[group];
    float vals[1][2] = {{0.f, 0.f}};
    float ss = 0.f;
    if (mine) {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        vals[0][e] = chunk_pool<R>(K, S, e);
        ss = fmaf(vals[0][e], vals[0][e], ss);
      }
    }
    // the group's sum, in block_sum's order; the next round writes sums behind its CTA barrier, so that frees them
    ss = warp_sum(ss);
    if (lane == 0) sums[group][tid >> 5] = ss;
    if (G == 1)
      __syncthreads();
    else
      asm volatile("bar.sync %0, %1;\n" ::"r"(1 + group), "n"(THREADS) : "memory");
    ss = warp_sum(lane < (d + 63) / 64 ? sums[group][lane] : 0.f);
    const float rinv = rsqrtf(ss / static_cast<float>(d) + p.eps);
    if (mine)
      finish_pair(vals[0][0], vals[0][1], c, d, p.rope_dim, p.norm_w, p.norm_dtype, rinv, p.freqs, R * g, p.out, orow,
                  p.out_dtype, p.act_quant);
    if (G == 1 && p.act_quant == 2) {  // head_dim 128: threads 0..63 hold the row (uniform over the CTA)
      hadamard_fp4_128(vals[0][0], vals[0][1], xch);
      if (tid < 64) store_pair(vals[0][0], vals[0][1], c, d, p.out, orow, p.out_dtype);
    }
    if (G == 1 && p.key_image && g < p.max_comp)
      append_key_row(vals[0][0], vals[0][1], d, p.key_image, p.key_inv, p.key_norm_max, p.max_comp, slot, g, red);
  }
  if (!ok && threadIdx.x == 0)  // what was asked for lands before the CTA leaves
    for (int i = max(0, issued - STAGES); i < issued; ++i) tc5::bar_wait(&full[i % STAGES], (i / STAGES) & 1);
}

template <int R>
__global__ void __launch_bounds__(THREADS) chunk_kernel(dsv4_compressor_chunk_params p) {
  pdl_wait();
  pdl_trigger();
  __shared__ float red[33];
  __shared__ float xch[128];
  __shared__ int own[4];  // sequence of each of the four tokens, -1: nothing to emit
  if (static_cast<int>(blockIdx.x) >= p.n) {
    const int t = 4 * (blockIdx.x - p.n) + threadIdx.x;
    if (threadIdx.x < 4) {
      int b = -1;
      if (t < p.total && t < p.cu_seqlens[p.n]) {
        int lo = 0, hi = p.n - 1;
        while (lo < hi) {
          const int mid = (lo + hi + 1) >> 1;
          if (p.cu_seqlens[mid] <= t)
            lo = mid;
          else
            hi = mid - 1;
        }
        // a block whose row needs no token of before the chunk
        const int start = p.start[lo], pos = start + (t - p.cu_seqlens[lo]);
        if ((pos + 1) % R == 0 && pos + 1 - 2 * R >= start) b = lo;
      }
      own[threadIdx.x] = b;
    }
    __syncthreads();
    for (int i = 0; i < 4; ++i) {
      const int b = own[i];
      if (b < 0) continue;
      const ChunkSeq<R> q = chunk_seq<R>(p, b);
      const int pos = q.start + (4 * (static_cast<int>(blockIdx.x) - p.n) + i - q.first);
      if (q.n > 0) chunk_emit<R>(p, q, pos / R, red, xch);
    }
    return;
  }
  chunk_sequence<R>(p, blockIdx.x, red, xch);
}

DSV4_ERROR_READER(compressor)

}  // namespace cmp
}  // namespace dsv4

using namespace dsv4;

extern "C" int dsv4_compressor_pool(const dsv4_compressor_params* p, void* stream) {
  DSV4_CHECK_ARG(p == nullptr || p->act_quant == 0 ||
                     (p->act_quant == 1 && p->head_dim % 64 == 0 && (p->head_dim - p->rope_dim) % 64 == 0) ||
                     (p->act_quant == 2 && p->head_dim == 128),
                 "dsv4_compressor_pool: act_quant 1 needs head_dim and head_dim - rope_dim multiples of 64, "
                 "act_quant 2 (Hadamard + fp4) head_dim 128");
  DSV4_CHECK_ARG(p && p->kv && p->score && p->ape && p->out && p->freqs, "dsv4_compressor_pool: NULL tensor");
  DSV4_CHECK_ARG(p->b > 0 && p->s >= 0 && p->ratio > 0 && p->ratio <= 8, "dsv4_compressor_pool: bad sizes");
  DSV4_CHECK_ARG(p->head_dim % 2 == 0 && p->head_dim <= 4 * cmp::THREADS && p->head_dim >= p->rope_dim &&
                     p->rope_dim % 2 == 0,
                 "dsv4_compressor_pool: head_dim %d unsupported", p->head_dim);
  DSV4_CHECK_DTYPE(p->out_dtype == DSV4_F32 || p->out_dtype == DSV4_BF16, "dsv4_compressor_pool: out dtype");
  DSV4_CHECK_DTYPE(p->norm_w == nullptr || p->norm_dtype == DSV4_F32 || p->norm_dtype == DSV4_BF16,
                   "dsv4_compressor_pool: norm dtype");
  const int groups = p->s / p->ratio;
  if (groups > 0) {
    // one thread per pair of dims, whole warps, at most THREADS (2 pairs a thread above 512 dims)
    const int threads = std::min(cmp::THREADS, (p->head_dim / 2 + 31) / 32 * 32);
    const dim3 grid(static_cast<unsigned>(static_cast<int64_t>(p->b) * groups));
    DSV4_CUDA_CHECK(launch_pdl(cmp::pool_kernel, grid, dim3(threads), 0, as_stream(stream), *p));
    DSV4_LAUNCH_CHECK("compressor pool_kernel");
  }
  if (p->ring_kv && p->ring_score) {
    dim3 g(2 * p->ratio, p->b);
    DSV4_CUDA_CHECK(launch_pdl(cmp::ring_seed_kernel, dim3(g), dim3(256), 0, as_stream(stream), *p));
    DSV4_LAUNCH_CHECK("compressor ring_seed_kernel");
  }
  return DSV4_OK;
}

static int check_decode_params(const dsv4_compressor_decode_params* p) {
  DSV4_CHECK_ARG(p == nullptr || p->act_quant == 0 ||
                     (p->act_quant == 1 && p->head_dim % 64 == 0 && (p->head_dim - p->rope_dim) % 64 == 0) ||
                     (p->act_quant == 2 && p->head_dim == 128),
                 "dsv4_compressor_decode: act_quant 1 needs head_dim and head_dim - rope_dim multiples of 64, "
                 "act_quant 2 (Hadamard + fp4) head_dim 128");
  DSV4_CHECK_ARG(p && p->kv && p->score && p->ape && p->ring_kv && p->ring_score && p->positions &&
                     p->out && p->out_rows && p->freqs,
                 "dsv4_compressor_decode: NULL tensor");
  DSV4_CHECK_ARG(p->b > 0 && p->ratio > 0 && p->ratio <= 8 && p->head_dim % 2 == 0 &&
                     p->head_dim <= 4 * cmp::THREADS && p->rope_dim % 2 == 0 && p->rope_dim <= p->head_dim,
                 "dsv4_compressor_decode: bad sizes");
  DSV4_CHECK_DTYPE(p->out_dtype == DSV4_F32 || p->out_dtype == DSV4_BF16, "dsv4_compressor_decode: out dtype");
  DSV4_CHECK_ARG(p->key_image == nullptr || (p->key_inv && p->key_norm_max && p->image_stride > 0 && p->ratio == 4 &&
                                              p->head_dim == 128 && p->out_dtype == DSV4_F32 &&
                                              reinterpret_cast<uintptr_t>(p->key_image) % 16 == 0),
                 "dsv4_compressor_decode: a key image needs ratio 4, head_dim 128, fp32 out, inv, norm_max, "
                 "image_stride and a 16-byte aligned image");
  return DSV4_OK;
}

extern "C" int dsv4_compressor_decode(const dsv4_compressor_decode_params* p, void* stream) {
  const int rc = check_decode_params(p);
  if (rc != DSV4_OK) return rc;
  if (p->ratio == 4 && p->head_dim <= 2 * cmp::THREADS)
    DSV4_CUDA_CHECK(launch_pdl(cmp::decode_r4_kernel<1>, dim3(p->b), dim3(cmp::THREADS), 0, as_stream(stream), *p));
  else if (p->ratio == 4)
    DSV4_CUDA_CHECK(launch_pdl(cmp::decode_r4_kernel<2>, dim3(p->b), dim3(cmp::THREADS), 0, as_stream(stream), *p));
  else
    DSV4_CUDA_CHECK(launch_pdl(cmp::decode_kernel, dim3(p->b), dim3(cmp::THREADS), 0, as_stream(stream), *p));
  DSV4_LAUNCH_CHECK("compressor decode_kernel");
  return DSV4_OK;
}

extern "C" int dsv4_compressor_decode_pair(const dsv4_compressor_decode_params* a,
                                           const dsv4_compressor_decode_params* b, void* stream) {
  int rc = check_decode_params(a);
  if (rc != DSV4_OK) return rc;
  rc = check_decode_params(b);
  if (rc != DSV4_OK) return rc;
  const bool one = a->b == b->b && a->ratio == 4 && b->ratio == 4 && a->head_dim <= 2 * cmp::THREADS &&
                   b->head_dim <= 2 * cmp::THREADS;
  if (!one) {
    rc = dsv4_compressor_decode(a, stream);
    return rc != DSV4_OK ? rc : dsv4_compressor_decode(b, stream);
  }
  DSV4_CUDA_CHECK(launch_pdl(cmp::decode_r4_pair_kernel<1>, dim3(a->b, 2), dim3(cmp::THREADS), 0, as_stream(stream),
                             *a, *b));
  DSV4_LAUNCH_CHECK("compressor decode_r4_pair_kernel");
  return DSV4_OK;
}

extern "C" int dsv4_compressor_chunk(const dsv4_compressor_chunk_params* p, void* stream) {
  DSV4_CHECK_ARG(p && p->kv && p->score && p->ape && p->ring_kv && p->ring_score && p->out && p->freqs && p->cu_seqlens &&
                     p->start,
                 "dsv4_compressor_chunk: NULL tensor");
  DSV4_CHECK_ARG(p->act_quant == 0 ||
                     (p->act_quant == 1 && p->head_dim % 64 == 0 && (p->head_dim - p->rope_dim) % 64 == 0) ||
                     (p->act_quant == 2 && p->head_dim == 128),
                 "dsv4_compressor_chunk: act_quant 1 needs head_dim and head_dim - rope_dim multiples of 64, "
                 "act_quant 2 (Hadamard + fp4) head_dim 128");
  DSV4_CHECK_ARG(p->n >= 0 && p->total >= 0 && p->slots > 0 && p->max_comp >= 0 && p->ratio > 0 && p->ratio <= 8,
                 "dsv4_compressor_chunk: bad sizes (ratio 1 to 8)");
  DSV4_CHECK_ARG(p->head_dim > 0 && p->head_dim % 2 == 0 && p->head_dim <= 4 * cmp::THREADS && p->rope_dim >= 0 &&
                     p->rope_dim % 2 == 0 && p->rope_dim <= p->head_dim,
                 "dsv4_compressor_chunk: head_dim %d, rope_dim %d unsupported", p->head_dim, p->rope_dim);
  DSV4_CHECK_ARG(p->seqs || p->n <= p->slots, "dsv4_compressor_chunk: more sequences than the ring has slots");
  DSV4_CHECK_ARG(p->block_table == nullptr ||
                     (p->page > 0 && p->bt_stride * static_cast<int64_t>(p->page) >= p->max_comp),
                 "dsv4_compressor_chunk: the block table does not cover max_comp");
  DSV4_CHECK_DTYPE(p->out_dtype == DSV4_F32 || p->out_dtype == DSV4_BF16, "dsv4_compressor_chunk: out dtype");
  DSV4_CHECK_DTYPE(p->norm_w == nullptr || p->norm_dtype == DSV4_F32 || p->norm_dtype == DSV4_BF16,
                   "dsv4_compressor_chunk: norm dtype");
  DSV4_CHECK_ARG(((reinterpret_cast<uintptr_t>(p->kv) | reinterpret_cast<uintptr_t>(p->score) |
                   reinterpret_cast<uintptr_t>(p->ape) | reinterpret_cast<uintptr_t>(p->ring_kv) |
                   reinterpret_cast<uintptr_t>(p->ring_score) | reinterpret_cast<uintptr_t>(p->out)) & 7) == 0,
                 "dsv4_compressor_chunk: tensors must be 8-byte aligned");
  DSV4_CHECK_ARG(p->key_image == nullptr || (p->key_inv && p->key_norm_max && p->max_comp > 0 && p->head_dim == 128 &&
                                              p->out_dtype == DSV4_F32 &&
                                              reinterpret_cast<uintptr_t>(p->key_image) % 16 == 0),
                 "dsv4_compressor_chunk: a key image needs head_dim 128, fp32 out, inv, norm_max and a 16-byte aligned image");
  if (p->n == 0 || p->total == 0) return DSV4_OK;
  const int threads = std::min(cmp::THREADS, (p->head_dim / 2 + 31) / 32 * 32);
  // Long chunks: runs of blocks, all CTAs resident at once: one an SM at 512 dims, as many as keep 192 KB an SM
  // under way below. Under two blocks a run there is nothing to stream ahead; the bulk copies want 16-byte
  // alignment.
  int run = 0;
  const bool wide = p->head_dim == 512 && p->act_quant != 2 && p->key_image == nullptr;
  if (p->ratio == 4 && p->head_dim % 64 == 0 && p->head_dim <= 2 * cmp::THREADS) {
    const int ctas = (wide ? 1 : 2 * (2 * cmp::THREADS / p->head_dim)) * num_sms() - 2 * p->n;
    run = ctas > 0 ? (p->total / 4 + ctas - 1) / ctas : 0;
  }
  if (run >= 2 && ((reinterpret_cast<uintptr_t>(p->kv) | reinterpret_cast<uintptr_t>(p->score)) & 15) == 0) {
    using cmp::Run;
    const int which = wide ? 0 : p->head_dim == 128 ? 1 : 2;
    void (*k)(dsv4_compressor_chunk_params, int) =
        wide ? cmp::chunk_run_kernel<512, 3> : which == 1 ? cmp::chunk_run_kernel<128, 1> : cmp::chunk_run_kernel<0, 1>;
    const int smem = (wide ? Run<512, 3>::STAGES : Run<0, 1>::STAGES) * 4 * 2 * p->head_dim * 8;
    static PerDeviceOnce attr[3];
    DSV4_CUDA_CHECK(set_smem_once(attr[which], k, which == 2 ? Run<0, 1>::STAGES * 4 * 2 * 2 * cmp::THREADS * 8 : smem));
    // at most one run a sequence is not full
    DSV4_CUDA_CHECK(launch_pdl(k, dim3(p->n + p->total / 4 / run + p->n), dim3(wide ? 3 * cmp::THREADS : threads), smem,
                               as_stream(stream), *p, run));
    return DSV4_OK;
  }
  const dim3 grid(p->n + (p->total + 3) / 4);
  void (*k)(dsv4_compressor_chunk_params) = nullptr;
  switch (p->ratio) {
    case 1: k = cmp::chunk_kernel<1>; break;
    case 2: k = cmp::chunk_kernel<2>; break;
    case 3: k = cmp::chunk_kernel<3>; break;
    case 4: k = cmp::chunk_kernel<4>; break;
    case 5: k = cmp::chunk_kernel<5>; break;
    case 6: k = cmp::chunk_kernel<6>; break;
    case 7: k = cmp::chunk_kernel<7>; break;
    default: k = cmp::chunk_kernel<8>; break;
  }
  DSV4_CUDA_CHECK(launch_pdl(k, grid, dim3(threads), 0, as_stream(stream), *p));
  DSV4_LAUNCH_CHECK("compressor chunk_kernel");
  return DSV4_OK;
}
