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
// token; n < 2^22 keeps every sum below 2^63.
//
// One cluster of CTAs a row: each CTA reads its slice of the row once into
// shared memory (as values with NaN and -0 folded) and every later step works
// on that, so the row crosses the memory bus once and a call is one launch.  A
// cutoff is found in two steps instead of a sort: a histogram over 1024 bins of
// max - l (counts for top-k, weights for top-p), summed over the cluster
// through distributed shared memory, gives the bin that holds the cutoff; the
// tokens of that bin (a few out of a vocabulary) are gathered in one CTA, which
// ranks them against each other.  Bins with more tokens than the list holds
// (many equal logits) are searched eight bits of the order's key at a time
// instead.  Weights enter the histogram as three words of 14 bits each, which
// shared memory adds as 32-bit integers: 2^18 tokens of a slice cannot overflow
// one.
#pragma once
#include "rv_internal.cuh"

#define RV_SAMPLE_ONE 0x1p40f
#define RV_SAMPLE_THREADS 512
#define RV_SAMPLE_BINS 1024
#define RV_SAMPLE_LIST 1024    // tokens of one bin that are ranked directly
#define RV_SAMPLE_SLICE (1u << 18)
#define RV_SAMPLE_K_BINS 32.0f  // top-k's bins per unit of logit
#define RV_SAMPLE_P_BINS 64.0f  // top-p's per unit of z

typedef unsigned long long u64;

struct SampleArgs {
  const float *logits;
  size_t row_stride;
  uint32_t n, slice, size;  // logits of a row, of a CTA; CTAs of a cluster
  int in_smem;        // the slice is kept in shared memory
  const float *u, *temperature, *top_p, *min_p;
  const int32_t *top_k;
  int32_t *tokens;
  float *logprobs;
};

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
RV_DEVFN float sample_z(float l, float top, float inv_t) {
  return l == top ? 0.0f : __fmul_rn(__fsub_rn(l, top), inv_t);
}
RV_DEVFN u64 sample_weight(float e) { return (u64)__fmul_rn(e, RV_SAMPLE_ONE); }

// Shared memory of a CTA besides its slice.
struct SampleShared {
  u64 red[RV_SAMPLE_THREADS / 32];
  u64 best, sum;          // this CTA's, for the cluster
  u64 pick[4];            // results one thread hands to the others
  u64 list_key[RV_SAMPLE_LIST];
  u64 list_w[RV_SAMPLE_LIST];
  uint32_t list_n;
  uint32_t hist[3][RV_SAMPLE_BINS];  // counts, or words of weights, the lowest first
  u64 part[RV_SAMPLE_BINS];          // cluster sums of this CTA's share of the bins
};
// A weight (at most 2^40) into bin b.
RV_DEVFN void sample_add(SampleShared &sh, int b, u64 w) {
  atomicAdd(&sh.hist[0][b], (uint32_t)w & 0x3FFFu);
  atomicAdd(&sh.hist[1][b], (uint32_t)(w >> 14) & 0x3FFFu);
  atomicAdd(&sh.hist[2][b], (uint32_t)(w >> 28));
}

RV_DEVFN u64 ld_cluster_u64(uint32_t a) {
  u64 v;
  asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(v) : "r"(a) : "memory");
  return v;
}
RV_DEVFN uint32_t ld_cluster_u32(uint32_t a) {
  uint32_t v;
  asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(a) : "memory");
  return v;
}
RV_DEVFN void st_cluster_u64(uint32_t a, u64 v) {
  asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(a), "l"(v) : "memory");
}
RV_DEVFN uint32_t atom_add_cluster(uint32_t a, uint32_t v) {
  uint32_t r;
  asm volatile("atom.shared::cluster.add.u32 %0, [%1], %2;" : "=r"(r) : "r"(a), "r"(v) : "memory");
  return r;
}

struct SampleRow {
  const float *x;  // this CTA's slice (shared memory, or global where it does not fit)
  uint32_t i0, n;  // its first index and length
  uint32_t rank, size;  // the CTA in the cluster
  float top, inv_t, bin_scale;
  bool raw;        // x is as given: NaN and -0 are not folded yet
  RV_DEVFN float at(uint32_t i) const { return raw ? sample_value(x[i]) : x[i]; }
  RV_DEVFN float e(float l) const { return expf(sample_z(l, top, inv_t)); }
  RV_DEVFN u64 w(float l) const { return sample_weight(e(l)); }
  RV_DEVFN int bin(float l) const {  // monotone: a larger value has no larger bin
    return min((int)fminf((top - l) * bin_scale, (float)RV_SAMPLE_BINS), RV_SAMPLE_BINS - 1);
  }
};

// Sum (or maximum) over the CTA; every thread gets it.
template <typename F>
RV_DEVFN u64 sample_reduce(u64 v, SampleShared &sh, F f) {
  for (int o = 16; o; o >>= 1) v = f(v, __shfl_xor_sync(RV_FULL, v, o));
  __syncthreads();
  if ((threadIdx.x & 31) == 0) sh.red[threadIdx.x >> 5] = v;
  __syncthreads();
  v = sh.red[threadIdx.x & (RV_SAMPLE_THREADS / 32 - 1)];
  for (int o = RV_SAMPLE_THREADS / 64; o; o >>= 1) v = f(v, __shfl_xor_sync(RV_FULL, v, o));
  return v;
}
// Sum (or maximum) over the cluster.  `slot` of every CTA is written before and
// read after one barrier; a caller passes each slot once.
template <typename F>
RV_DEVFN u64 sample_cluster_reduce(u64 v, u64 *slot, const SampleRow &r, F f) {
  if (r.size == 1) return v;
  if (threadIdx.x == 0) *slot = v;
  cluster_sync_all();
  u64 x = (threadIdx.x & 31) < r.size ? ld_cluster_u64(dsmem_addr(slot, threadIdx.x & 31)) : 0;  // 0: neutral for both
  for (int o = 16; o; o >>= 1) x = f(x, __shfl_xor_sync(RV_FULL, x, o));
  return x;
}

// The bin where the running total (counts or weights, from bin 0 on) reaches
// `goal`, and the total before it.  Every CTA gets both.
RV_DEVFN int sample_find_bin(SampleShared &sh, const SampleRow &r, bool weights, u64 goal, u64 &before) {
  const uint32_t t = threadIdx.x;
  cluster_sync_all();  // the histograms are complete
  // Each CTA sums its share of the bins over the cluster; then every CTA reads
  // all the sums.
  const uint32_t share = RV_SAMPLE_BINS / r.size, f0 = r.rank * share;
  for (uint32_t b = f0 + t; b < f0 + share; b += RV_SAMPLE_THREADS) {
    u64 s = 0;
    for (uint32_t c = 0; c < r.size; c++) {
      s += ld_cluster_u32(dsmem_addr(&sh.hist[0][b], c));
      if (weights)
        s += ((u64)ld_cluster_u32(dsmem_addr(&sh.hist[1][b], c)) << 14) +
             ((u64)ld_cluster_u32(dsmem_addr(&sh.hist[2][b], c)) << 28);
    }
    sh.part[b] = s;
  }
  cluster_sync_all();
  constexpr int PER = RV_SAMPLE_BINS / RV_SAMPLE_THREADS;
  u64 v[PER], mine = 0;
#pragma unroll
  for (int j = 0; j < PER; j++) {
    const uint32_t b = t * PER + j;
    v[j] = ld_cluster_u64(dsmem_addr(&sh.part[b], b / share));
    mine += v[j];
  }
  u64 run = mine;
  for (int o = 1; o < 32; o <<= 1) {
    const u64 x = __shfl_up_sync(RV_FULL, run, o);
    if ((t & 31) >= (uint32_t)o) run += x;
  }
  __syncthreads();
  if ((t & 31) == 31) sh.red[t >> 5] = run;
  __syncthreads();
  for (uint32_t w = 0; w < t >> 5; w++) run += sh.red[w];
  run -= mine;
  if (run < goal && goal <= run + mine) {
#pragma unroll
    for (int j = 0; j < PER; j++) {
      if (run < goal && goal <= run + v[j]) {
        sh.pick[0] = t * PER + j;
        sh.pick[1] = run;
      }
      run += v[j];
    }
  }
  __syncthreads();
  before = sh.pick[1];
  return (int)sh.pick[0];
}

// The key of the last token kept when tokens from the largest on are kept until
// their number (weights: their weight) reaches `goal`; only tokens at or above
// `from` count.  1 <= goal <= the total.  Every CTA of the cluster gets it.
RV_DEVFN u64 sample_cutoff(SampleShared &sh, const SampleRow &r, u64 from, u64 goal, bool weights, u64 least) {
  const uint32_t t = threadIdx.x;
  cluster_sync_all();  // nobody still reads the histograms of an earlier cutoff
  for (uint32_t b = t; b < RV_SAMPLE_BINS; b += RV_SAMPLE_THREADS) sh.hist[0][b] = sh.hist[1][b] = sh.hist[2][b] = 0;
  if (t == 0) sh.list_n = 0;
  __syncthreads();
  // Tokens of less than `least` weight cannot lie at or above the cutoff.
  for (uint32_t i = t; i < r.n; i += RV_SAMPLE_THREADS) {
    const float l = r.at(i);
    if (!weights) {
      const int b = r.bin(l);
      // The last bin holds the far tail, which k seldom reaches: its count
      // is what the others leave.
      if (b < RV_SAMPLE_BINS - 1) atomicAdd(&sh.hist[0][b], 1u);
    } else if (sample_key(l, r.i0 + i) >= from) {
      const u64 w = r.w(l);
      if (w >= least) sample_add(sh, r.bin(l), w);
    }
  }
  if (!weights) {
    __syncthreads();
    u64 s = 0;
    for (uint32_t b = t; b < RV_SAMPLE_BINS - 1; b += RV_SAMPLE_THREADS) s += sh.hist[0][b];
    s = sample_reduce(s, sh, [](u64 p, u64 q) { return p + q; });
    if (t == 0) sh.hist[0][RV_SAMPLE_BINS - 1] = r.n - (uint32_t)s;
  }
  u64 before;
  const int bin = sample_find_bin(sh, r, weights, goal, before);
  // The bin's tokens go to CTA 0 of the cluster.
  const uint32_t list_n = dsmem_addr(&sh.list_n, 0);
  for (uint32_t i = t; i < r.n; i += RV_SAMPLE_THREADS) {
    const float l = r.at(i);
    if (r.bin(l) != bin) continue;
    const u64 key = sample_key(l, r.i0 + i);
    if (key < from) continue;
    const uint32_t at = atom_add_cluster(list_n, 1u);
    if (at < RV_SAMPLE_LIST) {
      st_cluster_u64(dsmem_addr(&sh.list_key[at], 0), key);
      st_cluster_u64(dsmem_addr(&sh.list_w[at], 0), weights ? r.w(l) : 1ull);
    }
  }
  cluster_sync_all();
  const uint32_t cnt = ld_cluster_u32(list_n);
  if (cnt <= RV_SAMPLE_LIST) {
    // Each thread of CTA 0 places its tokens among the list's.
    if (r.rank == 0) {
      for (uint32_t i = t; i < cnt; i += RV_SAMPLE_THREADS) {
        const u64 key = sh.list_key[i];
        u64 sum = before;
        for (uint32_t j = 0; j < cnt; j++) sum += sh.list_key[j] > key ? sh.list_w[j] : 0;
        if (sum < goal && goal <= sum + sh.list_w[i])
          for (uint32_t c = 0; c < r.size; c++) st_cluster_u64(dsmem_addr(&sh.pick[2], c), key);
      }
    }
    cluster_sync_all();
    return sh.pick[2];
  }
  // Too many for the list: eight bits of the key at a time, within the bin.
  u64 prefix = 0, above = before;
  for (int shift = 56; shift >= 0; shift -= 8) {
    cluster_sync_all();
    for (uint32_t b = t; b < RV_SAMPLE_BINS; b += RV_SAMPLE_THREADS) sh.hist[0][b] = sh.hist[1][b] = sh.hist[2][b] = 0;
    __syncthreads();
    for (uint32_t i = t; i < r.n; i += RV_SAMPLE_THREADS) {
      const float l = r.at(i);
      if (r.bin(l) != bin) continue;
      const u64 key = sample_key(l, r.i0 + i);
      if (key < from || (shift < 56 && (key >> (shift + 8)) != prefix)) continue;
      const int d = 255 - (int)((key >> shift) & 255);  // descending
      if (weights) sample_add(sh, d, r.w(l));
      else atomicAdd(&sh.hist[0][d], 1u);
    }
    u64 sum;
    const int d = sample_find_bin(sh, r, weights, goal - above, sum);
    prefix = prefix << 8 | (u64)(255 - d);
    above += sum;
  }
  return prefix;
}

__global__ void __launch_bounds__(RV_SAMPLE_THREADS) k_sample(SampleArgs a) {
  extern __shared__ __align__(16) uint8_t s_raw[];
  SampleShared &sh = *(SampleShared *)s_raw;
  float *s_slice = (float *)(s_raw + (sizeof(SampleShared) + 15) / 16 * 16);
  const auto mx = [](u64 p, u64 q) { return p > q ? p : q; };
  const auto add = [](u64 p, u64 q) { return p + q; };
  const uint32_t t = threadIdx.x, row = blockIdx.x / a.size;
  SampleRow r;
  r.rank = blockIdx.x - row * a.size;
  r.size = a.size;
  r.i0 = min(a.n, r.rank * a.slice);
  r.n = min(a.n - r.i0, a.slice);
  const float *x = a.logits + (size_t)row * a.row_stride + r.i0;
  r.x = a.in_smem ? s_slice : x;
  r.raw = !a.in_smem;
  u64 best = 0;
  const bool wide = a.in_smem && (((uintptr_t)x) & 15) == 0;
  const uint32_t n4 = wide ? r.n / 4 : 0;
#pragma unroll 4
  for (uint32_t i = t; i < n4; i += RV_SAMPLE_THREADS) {
    const float4 v = __ldcs((const float4 *)x + i);
    const float4 y = make_float4(sample_value(v.x), sample_value(v.y), sample_value(v.z), sample_value(v.w));
    ((float4 *)s_slice)[i] = y;
    best = mx(best, mx(mx(sample_key(y.x, r.i0 + 4 * i), sample_key(y.y, r.i0 + 4 * i + 1)),
                       mx(sample_key(y.z, r.i0 + 4 * i + 2), sample_key(y.w, r.i0 + 4 * i + 3))));
  }
#pragma unroll 8
  for (uint32_t i = 4 * n4 + t; i < r.n; i += RV_SAMPLE_THREADS) {
    const float l = sample_value(__ldcs(x + i));
    if (a.in_smem) s_slice[i] = l;
    best = mx(best, sample_key(l, r.i0 + i));
  }
  best = sample_cluster_reduce(sample_reduce(best, sh, mx), &sh.best, r, mx);
  r.top = sample_key_value(best);
  const float temp = a.temperature ? a.temperature[row] : 1.0f;
  if (r.top == -INFINITY || !(temp > 0.0f)) {  // nothing to draw from, or greedy
    if (t == 0 && r.rank == 0) {
      a.tokens[row] = r.top == -INFINITY ? 0 : (int32_t)~(uint32_t)best;
      if (a.logprobs) a.logprobs[row] = r.top == -INFINITY ? -INFINITY : 0.0f;
    }
    if (r.size > 1) cluster_sync_all();  // the others may still read this CTA's maximum
    return;
  }
  r.inv_t = __fdiv_rn(1.0f, temp);
  r.bin_scale = RV_SAMPLE_K_BINS;
  u64 from = 0;
  const int k = a.top_k ? a.top_k[row] : 0;
  if (k > 0 && (uint32_t)k < a.n) from = sample_cutoff(sh, r, 0, (u64)k, false, 0);
  const float p = a.top_p ? a.top_p[row] : 1.0f;
  if (p < 1.0f) {
    u64 s = 0;
    for (uint32_t i = t; i < r.n; i += RV_SAMPLE_THREADS) {
      const float l = r.at(i);
      if (sample_key(l, r.i0 + i) >= from) s += r.w(l);
    }
    const u64 total = sample_cluster_reduce(sample_reduce(s, sh, add), &sh.sum, r, add);
    const double goal = __dmul_rn((double)p, (double)total);
    if (goal >= 1.0) {
      // The tokens of less than (total - goal) / n each do not amount to what
      // lies beyond the cutoff, so they lie beyond it.
      const u64 g = (u64)goal;
      r.bin_scale = RV_SAMPLE_P_BINS * fminf(r.inv_t, 0x1p40f);
      from = sample_cutoff(sh, r, from, g, true, (total - g) / a.n);
    } else {
      from = best;
    }
  }
  const float mp = a.min_p ? a.min_p[row] : 0.0f;
  const auto kept = [&](float l, uint32_t i) -> u64 {
    if (sample_key(l, r.i0 + i) < from) return 0;
    const float e = r.e(l);
    return e >= mp || l == r.top ? sample_weight(e) : 0;
  };
  // Each warp owns a run of the slice, 32 consecutive tokens at a time.
  const uint32_t lane = t & 31, warps = RV_SAMPLE_THREADS / 32, per = ((r.n + warps * 32 - 1) / (warps * 32)) * 32,
                 w0 = min(r.n, (t >> 5) * per), w1 = min(r.n, w0 + per);
  u64 mine = 0;
  for (uint32_t i = w0 + lane; i < w1; i += 32) mine += kept(r.at(i), i);
  u64 warp_sum = mine;
  for (int o = 16; o; o >>= 1) warp_sum += __shfl_xor_sync(RV_FULL, warp_sum, o);
  __syncthreads();
  if (lane == 0) sh.red[t >> 5] = warp_sum;
  __syncthreads();
  u64 cta = 0, before = 0;
  for (uint32_t w = 0; w < warps; w++) {
    before += w < t >> 5 ? sh.red[w] : 0;
    cta += sh.red[w];
  }
  u64 W = cta;
  if (r.size > 1) {
    if (t == 0) sh.pick[3] = cta;
    cluster_sync_all();
    u64 c = lane < r.size ? ld_cluster_u64(dsmem_addr(&sh.pick[3], lane)) : 0, lower = lane < r.rank ? c : 0;
    for (int o = 16; o; o >>= 1) {
      c += __shfl_xor_sync(RV_FULL, c, o);
      lower += __shfl_xor_sync(RV_FULL, lower, o);
    }
    W = c;
    before += lower;
  }
  const float u = a.u[row];
  u64 target = u > 0.0f ? (u64)__dmul_rn((double)u, (double)W) : 0;  // NaN is 0
  if (target >= W) target = W - 1;
  if (before <= target && target < before + warp_sum) {
    for (uint32_t b = w0; b < w1; b += 32) {
      const float l = b + lane < w1 ? r.at(b + lane) : -INFINITY;
      const u64 w = b + lane < w1 ? kept(l, b + lane) : 0;
      u64 run = w;
      for (int o = 1; o < 32; o <<= 1) {
        const u64 v = __shfl_up_sync(RV_FULL, run, o);
        if (lane >= (uint32_t)o) run += v;
      }
      const u64 all = __shfl_sync(RV_FULL, run, 31);
      if (target < before + all) {
        const int hit = __ffs(__ballot_sync(RV_FULL, target < before + run)) - 1;
        if ((int)lane == hit) {
          a.tokens[row] = (int32_t)(r.i0 + b + lane);
          if (a.logprobs)
            a.logprobs[row] = __fsub_rn(sample_z(l, r.top, r.inv_t), (float)log((double)W * 0x1p-40));
        }
        break;
      }
      before += all;
    }
  }
  if (r.size > 1) cluster_sync_all();  // the others may still read this CTA's sums
}
