// rv_prefix.cuh -- attention of a batch of sequences that share a prefix
// (rv_prefix_attention).
//
// Query row (b, i, h) -- token i of the n_q newest of sequence b, query head h,
// kv head h / G -- sees every prefix position and the suffix positions of its
// own sequence up to its own: seen = lens[b] - n_q + 1 + i of them.
//   s_j = scale * q . k_j,   o = sum_j exp(s_j) v_j / sum_j exp(s_j)
// Any split of the keys can be joined: a part gives its maximum m, the sum
// l = sum exp(s_j - m) and o = sum exp(s_j - m) v_j, and the parts add up as
// sum_p exp(m_p - M) (l_p, o_p) with M = max m_p.  A row that sees nothing is 0.
#pragma once
#include "rv_kv.cuh"

#define RV_LOG2E 1.4426950408889634f

struct PrefixArgs {
  const void *q;         // [n_seqs][n_q][n_heads][hd]: strides below, heads contiguous
  void *out;             // [n_seqs][n_q][n_heads][hd], contiguous
  const void *pk, *pv;   // prefix planes [prefix_cap][n_kv][hd]
  const float *pks, *pvs;  // their scales (8-bit cache)
  const void *sk, *sv;   // suffix planes [n_seqs][cap][n_kv][hd]
  const float *sks, *svs;
  const int32_t *lens;   // [n_seqs] suffix lengths, the queries' own tokens included
  size_t q_seq_stride, q_token_stride;
  uint32_t prefix_len, cap, n_seqs, n_q, n_heads, n_kv, hd;
  float scale_log2;      // scale * log2(e)
};

// A sequence's suffix length, held inside its cache.
RV_DEVFN int prefix_suffix_len(const PrefixArgs &a, uint32_t b) {
  const int n = a.lens[b];
  if (n < 0 || n > (int)a.cap) rv_dev_fail(RV_ERR_CAPACITY_EXCEEDED);
  return min(max(n, 0), (int)a.cap);
}

// Any head_dim that is a multiple of 8 up to 256: one CTA of eight warps per
// query row, a warp per key in turn, head_dim spread over the lanes, so a
// score is one warp sum.  The keys and values of the prefix are read once per
// query row, not once per batch.
template <typename T, bool Q8>
__global__ void __launch_bounds__(256) k_prefix_any(PrefixArgs a) {
  __shared__ float s_m[8], s_l[8], s_o[8][256];
  const uint32_t h = blockIdx.x, i = blockIdx.y, b = blockIdx.z, kvh = h / (a.n_heads / a.n_kv);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int own = min(prefix_suffix_len(a, b), max(0, prefix_suffix_len(a, b) - (int)a.n_q + 1 + (int)i));
  const long long total = (long long)a.prefix_len + own;
  const uint32_t e = lane * 8;
  const bool on = e < a.hd;
  float q[8] = {0, 0, 0, 0, 0, 0, 0, 0}, o[8] = {0, 0, 0, 0, 0, 0, 0, 0}, m = -INFINITY, l = 0;
  if (on) kv_load8((const T *)a.q + b * a.q_seq_stride + i * a.q_token_stride + (size_t)h * a.hd + e, false, q);
  for (long long j = warp; j < total; j += 8) {
    const bool pre = j < a.prefix_len;
    const size_t at = (pre ? (size_t)j : (size_t)b * a.cap + (size_t)(j - a.prefix_len)) * a.n_kv + kvh;
    float kx[8] = {0, 0, 0, 0, 0, 0, 0, 0}, vx[8] = {0, 0, 0, 0, 0, 0, 0, 0}, s = 0, vs = 1;
    if (on) {
      if constexpr (Q8) {
        const uint2 kw = *(const uint2 *)((const int8_t *)(pre ? a.pk : a.sk) + at * a.hd + e);
        const uint2 vw = *(const uint2 *)((const int8_t *)(pre ? a.pv : a.sv) + at * a.hd + e);
#pragma unroll
        for (int t = 0; t < 8; t++) {
          kx[t] = (float)(int8_t)((t < 4 ? kw.x : kw.y) >> (8 * (t & 3)));
          vx[t] = (float)(int8_t)((t < 4 ? vw.x : vw.y) >> (8 * (t & 3)));
        }
      } else {
        kv_load8((const __half *)(pre ? a.pk : a.sk) + at * a.hd + e, true, kx);
        kv_load8((const __half *)(pre ? a.pv : a.sv) + at * a.hd + e, true, vx);
      }
    }
#pragma unroll
    for (int t = 0; t < 8; t++) s = fmaf(q[t], kx[t], s);
    for (int x = 16; x; x >>= 1) s += __shfl_xor_sync(RV_FULL, s, x);
    if constexpr (Q8) {
      s *= (pre ? a.pks : a.sks)[at];
      vs = (pre ? a.pvs : a.svs)[at];
    }
    s *= a.scale_log2;
    const float mn = fmaxf(m, s), c = m == mn ? 1.0f : exp2f(m - mn);
    // A score of -infinity adds nothing, and neither does it as the maximum.
    const float p = s == -INFINITY ? 0.0f : exp2f(s - mn);
    l = fmaf(l, c, p);
#pragma unroll
    for (int t = 0; t < 8; t++) o[t] = fmaf(o[t], c, p * (vx[t] * vs));
    m = mn;
  }
  if (lane == 0) {
    s_m[warp] = m;
    s_l[warp] = l;
  }
#pragma unroll
  for (int t = 0; t < 8; t++)
    if (on) s_o[warp][e + t] = o[t];
  __syncthreads();
  float M = -INFINITY, L = 0;
  for (int w = 0; w < 8; w++) M = fmaxf(M, s_m[w]);
  for (int w = 0; w < 8; w++) L += s_m[w] == -INFINITY ? s_l[w] : exp2f(s_m[w] - M) * s_l[w];
  for (uint32_t d = threadIdx.x; d < a.hd; d += 256) {
    float x = 0;
    for (int w = 0; w < 8; w++) x += s_m[w] == -INFINITY ? s_o[w][d] : exp2f(s_m[w] - M) * s_o[w][d];
    ((T *)a.out)[(((size_t)b * a.n_q + i) * a.n_heads + h) * a.hd + d] = (T)(L == 0 ? 0.0f : x / L);
  }
}
