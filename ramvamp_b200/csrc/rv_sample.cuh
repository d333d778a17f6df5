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
// token; every sum stays below 2^60.
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
// shared memory adds as 32-bit integers: the tokens of a slice (fewer than
// 2^18) cannot overflow one.
//
// What bounds it: one row of 151,936 is a chain of cluster barriers and
// reductions (13.8 us; its bytes are 0.1 us).  Many rows alternate passes that
// issue -- a token costs its comparisons, one exponential and the histograms'
// shared-memory additions in each pass that weighs it -- with barriers: issue
// slots 0.45 to 0.51 used, the barrier the largest stall (64 rows of 151,936,
// top-p: 68 us of GPU time, 0.57 TB/s; 300 rows of 49,999, top-k 5,000 and top-p,
// 164 us).  Clusters also come in rounds: 37 of 8 CTAs or 74 of 4 at a time, so 64
// rows take two and 300 take five, the last nearly empty.
#pragma once
#include "rv_internal.cuh"

#define RV_SAMPLE_WARPS 32  // at most
#define RV_SAMPLE_BINS 1024
#define RV_SAMPLE_LIST 1024    // tokens of one bin that are ranked directly
#define RV_SAMPLE_MOST 720896  // logits a row: 16 slices of 45,056 (16-bit places)
#define RV_SAMPLE_K_BINS 32.0f  // top-k's bins per unit of logit
#define RV_SAMPLE_P_BINS 64.0f  // top-p's per unit of z

typedef unsigned long long u64;

struct SampleArgs {
  const float *logits;
  size_t row_stride;
  uint32_t n, slice, size;  // logits of a row, of a CTA; CTAs of a cluster
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
// floor(e * 2^40) for 0 <= e <= 1, from the bits: conversions to 64-bit
// integers are a tenth of the rate of shifts.
RV_DEVFN u64 sample_weight(float e) {
  const uint32_t b = __float_as_uint(e), m = (b & 0x7FFFFFu) | 0x800000u;
  const int up = (int)(b >> 23) - 110;  // e = m * 2^(up - 40), up <= 17
  return up >= 0 ? (u64)m * (1u << up) : (u64)(m >> min(-up, 31));
}

static_assert(RV_SAMPLE_BINS <= RV_SAMPLE_LIST, "sums of the bins in the list's space");
// Shared memory of a CTA besides its slice.
struct SampleShared {
  u64 red[RV_SAMPLE_WARPS];
  u64 best, sum;          // this CTA's, for the cluster
  u64 pick[4];            // results one thread hands to the others
  u64 list_key[RV_SAMPLE_LIST];      // also the [CTA][bin] sums of a share of the bins, before the list is filled
  u64 list_w[RV_SAMPLE_LIST];
  uint32_t list_n, found_n, found_at;  // found: this CTA's tokens for the list
  uint16_t found[RV_SAMPLE_LIST];
  u64 part_bin;           // the found bin's total
  uint32_t hist[3][RV_SAMPLE_BINS];  // counts, or words of weights, the lowest first
  u64 part[RV_SAMPLE_BINS];          // cluster sums of this CTA's share of the bins
};
// A weight (at most 2^40) into bin b.
RV_DEVFN void sample_add(SampleShared &sh, int b, u64 w) {
  atomicAdd(&sh.hist[0][b], (uint32_t)w & 0x3FFFu);
  atomicAdd(&sh.hist[1][b], (uint32_t)(w >> 14) & 0x3FFFu);
  if (w >> 28) atomicAdd(&sh.hist[2][b], (uint32_t)(w >> 28));  // most weights are below 2^-12
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
  const float *x;        // this CTA's slice, padded with -infinity to a multiple of 4
  uint32_t i0, n;        // its first index and length
  uint32_t rank, size;   // the CTA in the cluster
  float top, inv_t, bin_scale;
  float fv;              // kept: values above fv, and equal ones up to index fi
  uint32_t fi;
  RV_DEVFN float e(float l) const { return expf(sample_z(l, top, inv_t)); }
  RV_DEVFN u64 w(float l) const { return sample_weight(e(l)); }
  RV_DEVFN bool keeps(float l, uint32_t i) const { return l > fv || (l == fv && i0 + i <= fi); }
  RV_DEVFN int bin(float l) const {  // monotone: a larger value has no larger bin
    return min((int)fminf((top - l) * bin_scale, (float)RV_SAMPLE_BINS), RV_SAMPLE_BINS - 1);
  }
  // bin(l) == b, without the conversion.
  RV_DEVFN bool in_bin(float l, int b) const {
    const float d = (top - l) * bin_scale;
    return b == RV_SAMPLE_BINS - 1 ? !(d < (float)b) : d >= (float)b && d < (float)(b + 1);
  }
  RV_DEVFN void keep_from(u64 key) {
    fv = sample_key_value(key);
    fi = ~(uint32_t)key;
  }
  // f(value, index) for every token that is kept: 32 tokens a thread are looked
  // at first, so a warp works on kept tokens only, however few there are.
  template <int THREADS, typename F>
  RV_DEVFN void each_kept(F f) const {
    for (uint32_t base = 0; base < (n + 3) / 4; base += 8 * THREADS) {
      uint32_t m = 0;
#pragma unroll
      for (int j = 0; j < 8; j++) {
        const uint32_t i = base + j * THREADS + threadIdx.x;
        if (i < (n + 3) / 4) {
          const float4 v = ((const float4 *)x)[i];
          m |= (uint32_t)keeps(v.x, 4 * i) << (4 * j) | (uint32_t)keeps(v.y, 4 * i + 1) << (4 * j + 1) |
               (uint32_t)keeps(v.z, 4 * i + 2) << (4 * j + 2) | (uint32_t)keeps(v.w, 4 * i + 3) << (4 * j + 3);
        }
      }
      for (; m; m &= m - 1) {
        const uint32_t b = __ffs(m) - 1, i = 4 * (base + (b >> 2) * THREADS + threadIdx.x) + (b & 3);
        if (i < n) f(x[i], i);
      }
    }
  }
  // f(value, index) for every token of the slice; the padding comes as tokens
  // of -infinity with indexes from n on.
  template <int THREADS, typename F>
  RV_DEVFN void each(F f) const {
    for (uint32_t i = threadIdx.x; i < (n + 3) / 4; i += THREADS) {
      const float4 v = ((const float4 *)x)[i];
      f(v.x, 4 * i);
      f(v.y, 4 * i + 1);
      f(v.z, 4 * i + 2);
      f(v.w, 4 * i + 3);
    }
  }
};

// Sum (or maximum) over the CTA; every thread gets it.
template <int THREADS, typename F>
RV_DEVFN u64 sample_reduce(u64 v, SampleShared &sh, F f) {
  for (int o = 16; o; o >>= 1) v = f(v, __shfl_xor_sync(RV_FULL, v, o));
  __syncthreads();
  if ((threadIdx.x & 31) == 0) sh.red[threadIdx.x >> 5] = v;
  __syncthreads();
  v = sh.red[threadIdx.x & (THREADS / 32 - 1)];
  for (int o = THREADS / 64; o; o >>= 1) v = f(v, __shfl_xor_sync(RV_FULL, v, o));
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
// `goal`, and the total before it.  With p >= 0 the goal is first formed: p of
// all the weight, the bins' and every CTA's sh.sum (what its histogram left
// out), at least 1.  Every CTA gets all three.
template <int THREADS>
RV_DEVFN int sample_find_bin(SampleShared &sh, const SampleRow &r, bool weights, float p, u64 &goal, u64 &before) {
  const uint32_t t = threadIdx.x;
  cluster_sync_all();  // the histograms are complete
  // Each CTA sums its share of the bins over the cluster (a warp reads
  // consecutive bins of one CTA); then every CTA reads all the sums.
  const uint32_t share = RV_SAMPLE_BINS / r.size;
#pragma unroll
  for (int j = 0; j < RV_SAMPLE_BINS / THREADS; j++) {
    const uint32_t id = t + j * THREADS, c = id / share, b = r.rank * share + id % share;
    u64 s = ld_cluster_u32(dsmem_addr(&sh.hist[0][b], c));
    if (weights)
      s += ((u64)ld_cluster_u32(dsmem_addr(&sh.hist[1][b], c)) << 14) +
           ((u64)ld_cluster_u32(dsmem_addr(&sh.hist[2][b], c)) << 28);
    sh.list_key[id] = s;
  }
  __syncthreads();
  for (uint32_t b = t; b < share; b += THREADS) {
    u64 s = 0;
    for (uint32_t c = 0; c < r.size; c++) s += sh.list_key[c * share + b];
    sh.part[r.rank * share + b] = s;
  }
  cluster_sync_all();
  constexpr int PER = RV_SAMPLE_BINS / THREADS;
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
  // Warp sums: lane w holds warp w's; the sum of those before this warp.
  u64 total = (t & 31) < THREADS / 32 ? sh.red[t & 31] : 0, lower = (t & 31) < t >> 5 ? total : 0;
  if (p >= 0.0f && (t & 31) < r.size) total += ld_cluster_u64(dsmem_addr(&sh.sum, t & 31));
  for (int o = 16; o; o >>= 1) {
    lower += __shfl_xor_sync(RV_FULL, lower, o);
    total += __shfl_xor_sync(RV_FULL, total, o);
  }
  if (p >= 0.0f) goal = max((u64)__dmul_rn((double)p, (double)total), 1ull);
  run += lower - mine;
  if (run < goal && goal <= run + mine) {
#pragma unroll
    for (int j = 0; j < PER; j++) {
      if (run < goal && goal <= run + v[j]) {
        sh.pick[0] = t * PER + j;
        sh.pick[1] = run;
        sh.part_bin = v[j];
      }
      run += v[j];
    }
  }
  __syncthreads();
  before = sh.pick[1];
  return (int)sh.pick[0];
}

template <int THREADS>
RV_DEVFN void sample_clear(SampleShared &sh) {
  for (uint32_t b = threadIdx.x; b < RV_SAMPLE_BINS; b += THREADS) sh.hist[0][b] = sh.hist[1][b] = sh.hist[2][b] = 0;
  if (threadIdx.x == 0) sh.list_n = sh.found_n = 0;
}

// What a cutoff leaves.
struct SampleCut {
  u64 key;       // of the last token kept; 0: counts left so few candidates that all are in every CTA's list
  uint32_t cnt;  // tokens in the list
  bool sums;     // W and own are known (weights, and the list held its bin)
  u64 W, own;    // the weight kept, by all CTAs and by this one
};
// Tokens from the largest on are kept until their number reaches k (p < 0) or
// their weight p of the total, of the tokens that the row keeps so far.  Every
// CTA of the cluster gets the result.  fresh: the row's first cutoff (the
// histogram is zero and everything is kept).
template <int THREADS>
RV_DEVFN SampleCut sample_cutoff(SampleShared &sh, const SampleRow &r, uint32_t k, float p, uint32_t n, bool fresh) {
  const uint32_t t = threadIdx.x;
  const bool weights = p >= 0.0f;
  const auto add = [](u64 x, u64 y) { return x + y; };
  if (!fresh) {
    cluster_sync_all();  // nobody still reads the histograms of the earlier cutoff
    sample_clear<THREADS>(sh);
    __syncthreads();
  }
  if (!weights) {
    // The last bin holds the far tail, which k seldom reaches: its count is
    // what the others leave.
    r.each<THREADS>([&](float l, uint32_t) {
      const int b = r.bin(l);
      if (b < RV_SAMPLE_BINS - 1) atomicAdd(&sh.hist[0][b], 1u);
    });
    __syncthreads();
    u64 s = 0;
    for (uint32_t b = t; b < RV_SAMPLE_BINS - 1; b += THREADS) s += sh.hist[0][b];
    s = sample_reduce<THREADS>(s, sh, add);
    if (t == 0) sh.hist[0][RV_SAMPLE_BINS - 1] = r.n - (uint32_t)s;
  } else {
    // The total is at least 2^40, so the tokens of less than (1 - p) 2^40 / n
    // each do not amount to what lies beyond the cutoff: they lie beyond it,
    // and only the total needs them.
    const u64 least = (u64)(fmax(0.999 - (double)p, 0.0) * 0x1p40 / (double)n);
    u64 rest = 0;
    const auto put = [&](float l, uint32_t) {
      const u64 w = r.w(l);
      if (w >= least) sample_add(sh, r.bin(l), w);
      else rest += w;
    };
    if (fresh) r.each<THREADS>(put);  // everything is kept; the padding weighs nothing
    else r.each_kept<THREADS>(put);
    rest = sample_reduce<THREADS>(rest, sh, add);
    if (t == 0) sh.sum = rest;
  }
  SampleCut c;
  u64 goal = k, before;
  const int bin = sample_find_bin<THREADS>(sh, r, weights, p, goal, before);
  // The bin's tokens -- all up to it, where they are known to fit -- go to the
  // list of every CTA: first this CTA's, then one place in the list for all.
  const bool all = !weights && before + sh.part_bin <= RV_SAMPLE_LIST;
  const uint32_t list_n = dsmem_addr(&sh.list_n, 0);
  r.each<THREADS>([&](float l, uint32_t i) {
    if (!(all ? r.bin(l) <= bin : r.in_bin(l, bin)) || i >= r.n || !r.keeps(l, i)) return;
    const uint32_t at = atomicAdd(&sh.found_n, 1u);
    if (at < RV_SAMPLE_LIST) sh.found[at] = (uint16_t)i;
  });
  __syncthreads();
  const uint32_t found = sh.found_n;
  if (t == 0) sh.found_at = atom_add_cluster(list_n, found);
  __syncthreads();
  for (uint32_t j = t; j < min(found, RV_SAMPLE_LIST); j += THREADS) {
    const uint32_t at = sh.found_at + j, i = sh.found[j];
    if (at >= RV_SAMPLE_LIST) break;
    const float l = r.x[i];
    const u64 key = sample_key(l, r.i0 + i), w = weights || all ? r.w(l) : 1ull;
    for (uint32_t cta = 0; cta < r.size; cta++) {
      st_cluster_u64(dsmem_addr(&sh.list_key[at], cta), key);
      st_cluster_u64(dsmem_addr(&sh.list_w[at], cta), w);
    }
  }
  cluster_sync_all();
  c.cnt = ld_cluster_u32(list_n);
  c.key = 0;
  c.sums = false;
  if (all) return c;
  if (c.cnt <= RV_SAMPLE_LIST) {
    // A warp places a token among the list's; the CTAs share the tokens.
    for (uint32_t i = (t >> 5) * r.size + r.rank; i < c.cnt; i += THREADS / 32 * r.size) {
      const u64 key = sh.list_key[i];
      u64 sum = 0;
      if (weights) {
#pragma unroll 4
        for (uint32_t j = t & 31; j < c.cnt; j += 32) sum += sh.list_key[j] > key ? sh.list_w[j] : 0;
        for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(RV_FULL, sum, o);
      } else {
        uint32_t ahead = 0;
#pragma unroll 4
        for (uint32_t j = t & 31; j < c.cnt; j += 32) ahead += sh.list_key[j] > key;
        sum = __reduce_add_sync(RV_FULL, ahead);
      }
      sum += before;
      if (sum < goal && goal <= sum + sh.list_w[i] && (t & 31) < r.size) {
        st_cluster_u64(dsmem_addr(&sh.pick[2], t & 31), key);
        st_cluster_u64(dsmem_addr(&sh.pick[3], t & 31), sum + sh.list_w[i]);
      }
    }
    // Meanwhile, what this CTA keeps of the bins before.
    u64 own = 0;
    if (weights)
      for (int b = (int)t; b < bin; b += THREADS)
        own += sh.hist[0][b] + ((u64)sh.hist[1][b] << 14) + ((u64)sh.hist[2][b] << 28);
    cluster_sync_all();
    c.key = sh.pick[2];
    c.W = sh.pick[3];
    c.sums = weights;
    if (weights) {
      for (uint32_t i = t; i < c.cnt; i += THREADS) {
        const uint32_t id = ~(uint32_t)sh.list_key[i];
        if (sh.list_key[i] >= c.key && id - r.i0 < r.n) own += sh.list_w[i];
      }
      c.own = sample_reduce<THREADS>(own, sh, add);
    }
    return c;
  }
  // Too many for the list: eight bits of the key at a time, within the bin.
  u64 prefix = 0, above = before;
  for (int shift = 56; shift >= 0; shift -= 8) {
    cluster_sync_all();
    sample_clear<THREADS>(sh);
    __syncthreads();
    r.each<THREADS>([&](float l, uint32_t i) {
      if (!r.in_bin(l, bin) || i >= r.n || !r.keeps(l, i)) return;
      const u64 key = sample_key(l, r.i0 + i);
      if (shift < 56 && (key >> (shift + 8)) != prefix) return;
      const int d = 255 - (int)((key >> shift) & 255);  // descending
      if (weights) sample_add(sh, d, r.w(l));
      else atomicAdd(&sh.hist[0][d], 1u);
    });
    u64 sum, left = goal - above;
    const int d = sample_find_bin<THREADS>(sh, r, weights, -1.0f, left, sum);
    prefix = prefix << 8 | (u64)(255 - d);
    above += sum;
  }
  c.key = prefix;
  return c;
}

// The draw from a list of all candidates (`cnt` of them, more than k only by the
// last bin's), in one CTA: a warp a token, every filter by sums over the list.
template <int THREADS>
RV_DEVFN void sample_from_list(SampleShared &sh, const SampleRow &r, uint32_t cnt, uint32_t k, float p, float mp,
                               float u, int32_t *token, float *logprob) {
  const uint32_t t = threadIdx.x, lane = t & 31;
  const auto add = [](u64 x, u64 y) { return x + y; };
  // sh.part: the weight before each token in the order, or ~0 past the first k.
  u64 mine = 0;
  for (uint32_t i = t >> 5; i < cnt; i += THREADS / 32) {
    const u64 key = sh.list_key[i];
    u64 sum = 0;
    uint32_t rank = 0;
    for (uint32_t j = lane; j < cnt; j += 32) {
      const bool ahead = sh.list_key[j] > key;
      rank += ahead;
      sum += ahead ? sh.list_w[j] : 0;
    }
    rank = __reduce_add_sync(RV_FULL, rank);
    for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(RV_FULL, sum, o);
    if (lane == 0) {
      sh.part[i] = rank < k ? sum : ~0ull;
      if (rank < k) mine += sh.list_w[i];
    }
  }
  const u64 total = sample_reduce<THREADS>(mine, sh, add);
  const u64 goal = p < 1.0f ? (u64)fmax(__dmul_rn((double)p, (double)total), 0.0) : ~0ull;
  mine = 0;
  for (uint32_t i = t; i < cnt; i += THREADS) {
    const u64 key = sh.list_key[i], before = sh.part[i];
    const float l = sample_key_value(key);
    const bool keep = before != ~0ull && (before < goal || before == 0) && (r.e(l) >= mp || l == r.top);
    sh.list_w[i] = keep ? sh.list_w[i] : 0;
    mine += sh.list_w[i];
  }
  const u64 W = sample_reduce<THREADS>(mine, sh, add);
  u64 target = u > 0.0f ? (u64)__dmul_rn((double)u, (double)W) : 0;  // NaN is 0
  if (target >= W) target = W - 1;
  for (uint32_t i = t >> 5; i < cnt; i += THREADS / 32) {
    const uint32_t id = ~(uint32_t)sh.list_key[i];
    const u64 w = sh.list_w[i];
    if (w == 0) continue;
    u64 sum = 0;  // the kept weight of smaller indexes
    for (uint32_t j = lane; j < cnt; j += 32) sum += ~(uint32_t)sh.list_key[j] < id ? sh.list_w[j] : 0;
    for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(RV_FULL, sum, o);
    if (lane == 0 && sum <= target && target < sum + w) {
      *token = (int32_t)id;
      if (logprob)
        *logprob = __fsub_rn(sample_z(sample_key_value(sh.list_key[i]), r.top, r.inv_t),
                             (float)log((double)W * 0x1p-40));
    }
  }
}

template <int THREADS>
__global__ void __launch_bounds__(THREADS) k_sample(SampleArgs a) {
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
  r.x = s_slice;
  const float *x = a.logits + (size_t)row * a.row_stride + r.i0;
  sample_clear<THREADS>(sh);
  float top = -INFINITY;
  const uint32_t n4 = ((uintptr_t)x & 15) == 0 ? r.n / 4 : 0;
#pragma unroll 4
  for (uint32_t i = t; i < n4; i += THREADS) {
    const float4 v = __ldcs((const float4 *)x + i);
    const float4 y = make_float4(sample_value(v.x), sample_value(v.y), sample_value(v.z), sample_value(v.w));
    ((float4 *)s_slice)[i] = y;
    top = fmaxf(top, fmaxf(fmaxf(y.x, y.y), fmaxf(y.z, y.w)));
  }
#pragma unroll 8
  for (uint32_t i = 4 * n4 + t; i < r.n; i += THREADS) {
    const float l = sample_value(__ldcs(x + i));
    s_slice[i] = l;
    top = fmaxf(top, l);
  }
  if (t < 3 && r.n + t < (r.n + 3) / 4 * 4) s_slice[r.n + t] = -INFINITY;
  // The maximum as the key of index 0: only its value is used.
  u64 best = sample_cluster_reduce(sample_reduce<THREADS>(sample_key(top, 0), sh, mx), &sh.best, r, mx);
  r.top = sample_key_value(best);
  r.fv = -INFINITY;  // everything
  r.fi = 0xFFFFFFFFu;
  const float temp = a.temperature ? a.temperature[row] : 1.0f, p = a.top_p ? a.top_p[row] : 1.0f;
  const int k = a.top_k ? a.top_k[row] : 0;
  const bool none = r.top == -INFINITY, greedy = !(temp > 0.0f);
  // The first of the largest, where only that can be drawn.
  const auto first = [&]() {
    u64 b = 0;
    r.each<THREADS>([&](float l, uint32_t i) {
      if (l == r.top && i < r.n) b = mx(b, sample_key(l, r.i0 + i));
    });
    return sample_cluster_reduce(sample_reduce<THREADS>(b, sh, mx), &sh.sum, r, mx);
  };
  if (none || greedy) {
    if (!none) best = first();
    if (t == 0 && r.rank == 0) {
      a.tokens[row] = none ? 0 : (int32_t)~(uint32_t)best;
      if (a.logprobs) a.logprobs[row] = none ? -INFINITY : 0.0f;
    }
    cluster_sync_all();  // the others may still read this CTA's maximum
    return;
  }
  r.inv_t = fmaxf(__fdiv_rn(1.0f, temp), 0x1p-126f);  // so that -infinity times it stays one
  r.bin_scale = RV_SAMPLE_K_BINS;
  const float mp = a.min_p ? a.min_p[row] : 0.0f, u = a.u[row];
  bool fresh = true;
  SampleCut cut;
  cut.sums = false;
  if (k > 0 && (uint32_t)k < a.n) {
    cut = sample_cutoff<THREADS>(sh, r, (uint32_t)k, -1.0f, a.n, true);
    if (cut.key == 0) {
      if (r.rank == 0)
        sample_from_list<THREADS>(sh, r, cut.cnt, (uint32_t)k, p, mp, u, a.tokens + row,
                                  a.logprobs ? a.logprobs + row : nullptr);
      cluster_sync_all();  // the others may still read this CTA's shared memory
      return;
    }
    r.keep_from(cut.key);
    fresh = false;
  }
  if (p < 1.0f) {
    r.bin_scale = RV_SAMPLE_P_BINS * fminf(r.inv_t, 0x1p40f);
    cut = sample_cutoff<THREADS>(sh, r, 0, fmaxf(p, 0.0f), a.n, fresh);
    r.keep_from(cut.key);
  }
  const auto kept = [&](float l, uint32_t i) -> u64 {
    if (!r.keeps(l, i)) return 0;
    const float e = r.e(l);
    return e >= mp || l == r.top ? sample_weight(e) : 0;
  };
  const uint32_t lane = t & 31;
  // The kept weight of block b of 128 consecutive tokens of CTA c, whose first
  // index is i0 and length n (its slice is read over the cluster).
  const auto weigh = [&](uint32_t slice, uint32_t b, uint32_t i0, uint32_t n) {
    const uint32_t i = 128 * b + 4 * lane;
    u64 w = 0;
    if (i < n) {
      float4 v;
      asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
                   : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
                   : "r"(slice + 4 * i)
                   : "memory");
      const uint32_t at = i0 + i - r.i0;  // kept() adds this CTA's first index
      w = kept(v.x, at) + kept(v.y, at + 1) + kept(v.z, at + 2) + kept(v.w, at + 3);  // the padding weighs nothing
    }
    for (int o = 16; o; o >>= 1) w += __shfl_xor_sync(RV_FULL, w, o);
    return w;
  };
  // Without min-p the cutoff by weight knows what each CTA keeps, and only the
  // slice that holds the target is weighed, by all CTAs of the cluster.
  const bool known = cut.sums && !(mp > 0.0f);
  u64 own = cut.own;
  if (!known) {
    cluster_sync_all();  // sh.part is read by all in the cutoffs
    own = 0;
    for (uint32_t b = t >> 5; b < (r.n + 127) / 128; b += THREADS / 32) {
      const u64 w = weigh(smem_addr(s_slice), b, r.i0, r.n);
      if (lane == 0) {
        sh.part[b] = w;
        own += w;
      }
    }
    own = sample_reduce<THREADS>(own, sh, add);
  }
  if (t == 0) sh.best = own;
  cluster_sync_all();
  const u64 mine = lane < r.size ? ld_cluster_u64(dsmem_addr(&sh.best, lane)) : 0;
  u64 upto = mine;  // the kept weight up to each CTA's end
  for (int o = 1; o < 32; o <<= 1) {
    const u64 v = __shfl_up_sync(RV_FULL, upto, o);
    if (lane >= (uint32_t)o) upto += v;
  }
  const u64 W = __shfl_sync(RV_FULL, upto, 31);
  u64 target = u > 0.0f ? (u64)__dmul_rn((double)u, (double)W) : 0;  // NaN is 0
  if (target >= W) target = W - 1;
  const int where = __ffs(__ballot_sync(RV_FULL, target < upto)) - 1;
  u64 before = __shfl_sync(RV_FULL, upto - mine, where);
  const uint32_t i0 = min(a.n, (uint32_t)where * a.slice), blocks = (min(a.n - i0, a.slice) + 127) / 128;
  if (known) {
    const uint32_t slice = dsmem_addr(s_slice, where), part = dsmem_addr(sh.part, where);
    for (uint32_t b = (t >> 5) * r.size + r.rank; b < blocks; b += THREADS / 32 * r.size) {
      const u64 w = weigh(slice, b, i0, min(a.n - i0, a.slice));
      if (lane == 0) st_cluster_u64(part + 8 * b, w);
    }
    cluster_sync_all();
  }
  if ((uint32_t)where == r.rank) {
    if (t < 32) {
      const auto scan = [&](u64 v) {
        for (int o = 1; o < 32; o <<= 1) {
          const u64 x = __shfl_up_sync(RV_FULL, v, o);
          if (lane >= (uint32_t)o) v += x;
        }
        return v;
      };
      // The block that holds the target, then its tokens four a lane.
      for (uint32_t b0 = 0; b0 < blocks; b0 += 32) {
        const u64 v = b0 + lane < blocks ? sh.part[b0 + lane] : 0, end = before + scan(v);
        const uint32_t hits = __ballot_sync(RV_FULL, target < end);
        if (!hits) {
          before = __shfl_sync(RV_FULL, end, 31);
          continue;
        }
        const int which = __ffs(hits) - 1;
        before = __shfl_sync(RV_FULL, end - v, which);
        const uint32_t i = 128 * (b0 + which) + 4 * lane;
        u64 w[4], sum = 0;
        for (int j = 0; j < 4; j++) sum += w[j] = i + j < r.n ? kept(s_slice[i + j], i + j) : 0;
        before += scan(sum) - sum;
        for (int j = 0; j < 4; j++) {
          if (before <= target && target < before + w[j]) {
            a.tokens[row] = (int32_t)(r.i0 + i + j);
            if (a.logprobs)
              a.logprobs[row] = __fsub_rn(sample_z(s_slice[i + j], r.top, r.inv_t), (float)log((double)W * 0x1p-40));
          }
          before += w[j];
        }
        break;
      }
    }
  }
  cluster_sync_all();  // the others may still read this CTA's sums
}
