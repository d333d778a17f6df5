// rv_sample.cuh -- drawing a token of each row of logits (rv_sample).
//
//   z_i = (l_i - max l) * (1/T), 0 where l_i is the maximum;  e_i = exp(z_i)
//   w_i = floor(e_i * 2^40), an integer: sums of weights are exact, so neither
//         the order of a sum nor the number of threads changes a result
//   order: l descending, equal values by index ascending (NaN counts as -inf)
//   top-k: the first k;  top-p: of those, the tokens whose preceding weight is
//   below floor(p * W_k), and the first;  min-p: of those, e_i >= min_p
// Each filter keeps a prefix of the order, so each is one cutoff (value, index).
//   draw: target = floor(u * W) of the kept weight W; the token is the first
//   kept one in index order whose running weight passes the target
//   logprob = z_token - ln(W 2^-40)
// The weights' step of 2^-40 loses less than 2^-40 of the largest weight a
// token; n < 2^23 keeps every sum below 2^63.
#pragma once
#include "rv_internal.cuh"

#define RV_SAMPLE_ONE 0x1p40f
#define RV_SAMPLE_THREADS 1024

struct SampleArgs {
  const float *logits;
  size_t row_stride;
  uint32_t n;
  const float *u, *temperature, *top_p, *min_p;
  const int32_t *top_k;
  int32_t *tokens;
  float *logprobs;
};

typedef unsigned long long u64;

RV_DEVFN float sample_value(float l) { return isnan(l) ? -INFINITY : l + 0.0f; }  // -0 -> +0
// Ascending integer order of the token order: (value, index descending).
RV_DEVFN u64 sample_key(float l, uint32_t i) {
  const uint32_t b = __float_as_uint(l);
  return ((u64)(b & 0x80000000u ? ~b : b | 0x80000000u) << 32) | (uint32_t)~i;
}
RV_DEVFN float sample_key_value(u64 key) {
  const uint32_t b = (uint32_t)(key >> 32);
  return __uint_as_float(b & 0x80000000u ? b & 0x7FFFFFFFu : ~b);
}
RV_DEVFN float sample_z(float l, float top, float inv_t) { return l == top ? 0.0f : __fmul_rn(__fsub_rn(l, top), inv_t); }
RV_DEVFN u64 sample_weight(float e) { return (u64)__fmul_rn(e, RV_SAMPLE_ONE); }

template <typename V, typename F>
RV_DEVFN V sample_reduce(V v, V *sh, F f) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (int o = 16; o; o >>= 1) v = f(v, __shfl_xor_sync(RV_FULL, v, o));
  __syncthreads();
  if (lane == 0) sh[warp] = v;
  __syncthreads();
  v = sh[0];
  for (int w = 1; w < (int)(blockDim.x >> 5); w++) v = f(v, sh[w]);
  return v;
}

// One CTA a row.
__global__ void __launch_bounds__(RV_SAMPLE_THREADS) k_sample(SampleArgs a) {
  __shared__ u64 s_red[32], s_hist[256], s_pick[2];
  const float *x = a.logits + (size_t)blockIdx.x * a.row_stride;
  const uint32_t n = a.n, t = threadIdx.x, nt = blockDim.x;
  const auto mx = [](u64 p, u64 q) { return p > q ? p : q; };
  const auto add = [](u64 p, u64 q) { return p + q; };
  u64 best = 0;
  for (uint32_t i = t; i < n; i += nt) best = mx(best, sample_key(sample_value(x[i]), i));
  best = sample_reduce(best, s_red, mx);
  const float top = sample_key_value(best), temp = a.temperature ? a.temperature[blockIdx.x] : 1.0f;
  if (top == -INFINITY || !(temp > 0.0f)) {  // nothing to draw from, or greedy
    if (t == 0) {
      a.tokens[blockIdx.x] = top == -INFINITY ? 0 : (int32_t)~(uint32_t)best;
      if (a.logprobs) a.logprobs[blockIdx.x] = top == -INFINITY ? -INFINITY : 0.0f;
    }
    return;
  }
  const float inv_t = __fdiv_rn(1.0f, temp);
  const auto weight = [&](float l) { return sample_weight(expf(sample_z(l, top, inv_t))); };
  // The largest key whose tokens at or above it amount to `goal` in number
  // (by weight: in weight), eight bits of the key at a time.
  const auto cutoff = [&](u64 from, u64 goal, bool by_weight) {
    u64 prefix = 0, above = 0;
    for (int shift = 56; shift >= 0; shift -= 8) {
      __syncthreads();
      for (uint32_t i = t; i < 256; i += nt) s_hist[i] = 0;
      __syncthreads();
      for (uint32_t i = t; i < n; i += nt) {
        const float l = sample_value(x[i]);
        const u64 k = sample_key(l, i);
        if (k >= from && (shift == 56 || (k >> (shift + 8)) == prefix))
          atomicAdd(&s_hist[(k >> shift) & 255], by_weight ? weight(l) : 1ull);
      }
      __syncthreads();
      if (t == 0) {
        int d = 255;
        u64 sum = above;
        for (; d > 0 && sum + s_hist[d] < goal; d--) sum += s_hist[d];
        s_pick[0] = (u64)d;
        s_pick[1] = sum;
      }
      __syncthreads();
      prefix = prefix << 8 | s_pick[0];
      above = s_pick[1];
    }
    return prefix;
  };
  const auto kept_weight = [&](u64 from) {
    u64 s = 0;
    for (uint32_t i = t; i < n; i += nt) {
      const float l = sample_value(x[i]);
      if (sample_key(l, i) >= from) s += weight(l);
    }
    return sample_reduce(s, s_red, add);
  };
  u64 from = 0;
  const int k = a.top_k ? a.top_k[blockIdx.x] : 0;
  if (k > 0 && (uint32_t)k < n) from = cutoff(0, (u64)k, false);
  const float p = a.top_p ? a.top_p[blockIdx.x] : 1.0f;
  if (p < 1.0f) {
    const double goal = __dmul_rn((double)p, (double)kept_weight(from));
    from = goal >= 1.0 ? cutoff(from, (u64)goal, true) : best;
  }
  const float mp = a.min_p ? a.min_p[blockIdx.x] : 0.0f;
  const auto kept = [&](float l, uint32_t i) -> u64 {
    const float e = expf(sample_z(l, top, inv_t));
    return sample_key(l, i) >= from && (e >= mp || l == top) ? sample_weight(e) : 0;
  };
  // Each thread owns a run of consecutive tokens.
  const uint32_t per = (n + nt - 1) / nt, i0 = min(n, t * per), i1 = min(n, i0 + per);
  u64 mine = 0;
  for (uint32_t i = i0; i < i1; i++) mine += kept(sample_value(x[i]), i);
  const u64 W = sample_reduce(mine, s_red, add);
  u64 before = mine;
  for (int o = 1; o < 32; o <<= 1) {
    const u64 v = __shfl_up_sync(RV_FULL, before, o);
    if ((t & 31) >= (uint32_t)o) before += v;
  }
  __syncthreads();
  if ((t & 31) == 31) s_red[t >> 5] = before;
  __syncthreads();
  for (uint32_t w = 0; w < t >> 5; w++) before += s_red[w];
  before -= mine;
  const float u = a.u[blockIdx.x];
  u64 target = u > 0.0f ? (u64)__dmul_rn((double)u, (double)W) : 0;  // u >= 1 is clamped below, NaN is 0
  if (target >= W) target = W - 1;
  if (before <= target && target < before + mine) {
    for (uint32_t i = i0; i < i1; i++) {
      const float l = sample_value(x[i]);
      const u64 w = kept(l, i);
      if (target < before + w) {
        a.tokens[blockIdx.x] = (int32_t)i;
        if (a.logprobs)
          a.logprobs[blockIdx.x] = __fsub_rn(sample_z(l, top, inv_t), (float)log((double)W * 0x1p-40));
        break;
      }
      before += w;
    }
  }
}
