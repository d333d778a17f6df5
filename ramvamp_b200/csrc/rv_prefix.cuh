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
#include "rv_tc.cuh"

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

// Head dims other than 64 and 128 (multiples of 8 up to 256): one CTA of eight warps per
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

// ======================================================= tensor-core path
// head_dim 64 and 128.  For one kv head the rows of the whole batch that see
// the same keys are a matrix: S = Q K^T (128 rows x 128 keys a tile), P =
// exp(S - m), O += P V, with the running maximum and sum of every row kept in
// registers and S, P and O in tensor memory.
//
// Work: a segment is up to 256 (f32: 128) query rows of one kv head against the prefix or
// against one sequence's suffix, cut into units of 128 keys.  The units of all
// segments form one line that the CTAs (one per SM) split evenly, so a CTA
// walks one to a few pieces of segments whatever the lengths are; each piece
// leaves (m, l, O) of its rows in scratch and k_prefix_join adds the pieces of
// a row up.  Piece and slot numbers follow from the lengths alone, so the
// result does not depend on timing.
//
// Per CTA two streams of tiles run through the tensor cores, each with its own
// S, P and O columns and its own softmax warpgroup (thread = row), so one
// stream's products run under the other's exponentials.  Segments of more than
// 128 rows (f16 queries) pair the streams: each takes 128 of the rows and both
// read the same key and value tiles.  Otherwise the streams take alternate
// tiles of the same rows and leave a part each; f32 queries, whose two operands
// fill the space of the paired streams' query tiles, have segments of at most
// 128 rows.
//
// f32 queries are held to 2^-22 of their row's largest value as a sum of two
// f16 (after scaling by a power of two), and so is P: products of f16 with the
// f16 (or 8-bit) keys and values are exact, so the result carries f32's
// rounding only; the price is twice the products.  f16 queries round P to f16
// once, the size of the output's own rounding.  P is scaled by 2^7 and the
// reference maximum may lag by 2^8, so P stays below 2^15 and a weight is a
// normal f16 down to 2^-21 of the largest.
//
// 8-bit cache: levels are exact in f16, so the products run on levels.  With
// sk and sv the tokens' scales, t = s * sk + log2(sv): P = 2^(t - m) already
// holds sv, and l adds P / sv.
#define RV_PFX_CTAS 148       // CTAs at most: one per SM of a B200
#define RV_PFX_M 128          // rows of a stream's tile
#define RV_PFX_N 128          // keys of a tile
#define RV_PFX_LAG 8.0f       // the reference maximum may lag by this (log2)
#define RV_PFX_LIFT 7.0f      // P is lifted by 2^7
#define RV_PFX_SCALE_SLOTS 8  // tiles whose token scales are in shared memory
#define RV_PFX_O 256          // first tensor-memory column of O (S and P: 0..255)

struct PfxWork {
  int tp;              // prefix tiles
  int rows_p, rows_s;  // query rows of one kv head: all sequences', one sequence's
  int sr;              // rows of a segment: 256 (f16 queries) or 128 (f32)
  int nrt_p, nrt_s;    // segments of sr rows in them
  int rw_s;            // rows of a part of a suffix piece: min(128, rows_s)
  int grid;
  int q_aligned, out_aligned;  // 16-byte loads and stores
  int *cum;            // [n_seqs + 1] suffix tiles before sequence b, written by CTA 0
  float4 *o_p, *o_s;   // parts: [slot][stream][hd / 4][rows]
  float2 *ml_p, *ml_s; // [slot][stream][rows] (m, l)
};

template <int D, typename T, bool Q8>
struct PfxCfg {
  static constexpr bool PRECISE = sizeof(T) == 4;
  static constexpr int TILE = RV_PFX_M * D * 2;                 // bytes of a Q, K or V tile
  static constexpr int R = D == 64 ? 8 : Q8 ? 4 : 5;            // K/V ring stages
  static constexpr int SCALES = Q8 ? RV_PFX_SCALE_SLOTS * 3 * RV_PFX_N * 4 : 0;
  static constexpr int THREADS = Q8 ? 512 : 384;
  static constexpr int NBARS = 2 * R + 8 + RV_PFX_SCALE_SLOTS + 1;
  static constexpr size_t ring = 2 * TILE, scales = ring + (size_t)R * TILE, bars = scales + SCALES;
  static constexpr size_t total = 1024 + bars + NBARS * 8 + 32 * 4 + 64 + 2 * RV_PFX_M * 4;
};

struct PfxPiece {
  bool suffix, pair;
  int b, kvh, row0, nrows, keys, tile0, n, slot;
};

// A CTA's way along the line of units [u, end).
struct PfxWalk {
  int u, end, wp, ub;  // wp: units of the prefix; ub: suffix units before sequence b
  int b, c;
};
RV_DEVFN int pfx_tiles(int keys) { return (keys + RV_PFX_N - 1) / RV_PFX_N; }

RV_DEVFN bool pfx_next(const PrefixArgs &a, const PfxWork &w, PfxWalk &k, PfxPiece &p) {
  if (k.u >= k.end) return false;
  int seg, tiles, rt, nrt;
  if (k.u < k.wp) {
    tiles = w.tp;
    seg = k.u / tiles;
    p.tile0 = k.u - seg * tiles;
    nrt = w.nrt_p;
    p.suffix = false;
    p.b = 0;
    p.keys = (int)a.prefix_len;
    p.kvh = seg / nrt;
    rt = seg - p.kvh * nrt;
    p.nrows = min(w.sr, w.rows_p - rt * w.sr);
    p.slot = seg + k.c;
  } else {
    const int segs = (int)a.n_kv * w.nrt_s;
    const int us = k.u - k.wp;
    for (;;) {
      p.keys = prefix_suffix_len(a, (uint32_t)k.b);
      tiles = pfx_tiles(p.keys);
      if (us < k.ub + tiles * segs) break;
      k.ub += tiles * segs;
      k.b++;
    }
    const int local = (us - k.ub) / tiles;
    p.tile0 = us - k.ub - local * tiles;
    nrt = w.nrt_s;
    p.suffix = true;
    p.b = k.b;
    p.kvh = local / nrt;
    rt = local - p.kvh * nrt;
    p.nrows = min(w.sr, w.rows_s - rt * w.sr);
    p.slot = k.b * segs + local + k.c;
  }
  p.row0 = rt * w.sr;
  p.n = min(tiles - p.tile0, k.end - k.u);
  p.pair = p.nrows > RV_PFX_M;
  k.u += p.n;
  return true;
}

RV_DEVFN float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// 32 consecutive 32-bit columns of this thread's tensor-memory lane, loaded
// when it returns (one statement, so no use can be moved before the wait).
RV_DEVFN void tc_ld32(uint32_t taddr, uint32_t (&v)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
      "%15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];\n"
      " tcgen05.wait::ld.sync.aligned;"
      : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]),
        "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]), "=r"(v[16]),
        "=r"(v[17]), "=r"(v[18]), "=r"(v[19]), "=r"(v[20]), "=r"(v[21]), "=r"(v[22]), "=r"(v[23]), "=r"(v[24]),
        "=r"(v[25]), "=r"(v[26]), "=r"(v[27]), "=r"(v[28]), "=r"(v[29]), "=r"(v[30]), "=r"(v[31])
      : "r"(taddr)
      : "memory");
}
RV_DEVFN void tc_st16(uint32_t taddr, const uint32_t *v) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
      "%15, %16};" ::"r"(taddr),
      "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]),
      "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
      : "memory");
}
RV_DEVFN void tc_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
// D[tmem] (+)= A[tmem] * B[smem], kind::f16, issued by one thread.
RV_DEVFN void tc_mma_f16_ta(uint32_t d_tmem, uint32_t a_tmem, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
      " tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}\n" ::"r"(d_tmem),
      "r"(a_tmem), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}
RV_DEVFN uint32_t pack_f16(float lo, float hi) {  // element order: lo first
  const __half2 h = __floats2half2_rn(lo, hi);
  return *(const uint32_t *)&h;
}

// Load number of K(t) and V(t) within a piece of n tiles, in the order of first
// use by the products.  Paired streams: K0 V0 K1 V1 ...; alternating streams:
// K0 K1 V0 K2 V1 ... K(n-1) V(n-2) V(n-1).
RV_DEVFN int pfx_k_at(bool pair, int t) { return pair ? 2 * t : t == 0 ? 0 : 2 * t - 1; }
RV_DEVFN int pfx_v_at(bool pair, int t, int n) { return pair ? 2 * t + 1 : min(2 * t + 2, 2 * n - 1); }
RV_DEVFN void pfx_load_at(bool pair, int i, int n, bool &is_k, int &t) {
  if (pair) {
    is_k = !(i & 1);
    t = i >> 1;
  } else {
    is_k = i == 0 || ((i & 1) && i != 2 * n - 1);
    t = i == 0 ? 0 : i == 2 * n - 1 ? n - 1 : is_k ? (i + 1) >> 1 : (i - 2) >> 1;
  }
}

// Query row r of a segment: its sequence, token and head.
struct PfxRow {
  int b, i, h;
};
RV_DEVFN PfxRow pfx_row(const PrefixArgs &a, bool suffix, int b, int kvh, int r) {
  const int G = (int)(a.n_heads / a.n_kv), per = (int)a.n_q * G;
  PfxRow o;
  o.b = suffix ? b : r / per;
  const int x = suffix ? r : r - o.b * per;
  o.i = x / G;
  o.h = kvh * G + x - o.i * G;
  return o;
}

// The query rows of a stream's tile into the A operand(s) (K-major, 128-byte
// swizzle, 64 values a half tile), by the stream's 128 threads: D / 8 threads a
// row, so a row's loads are contiguous, and four rows a thread in flight.  f32
// rows are divided by a power of two first (2^e in `up`, the largest value
// then lies in [1, 2)) and held as hi + lo.  With store = false only `up` is
// formed.  neg: the queries change sign.
template <int D, typename T>
RV_DEVFN void pfx_load_q(const PrefixArgs &a, const PfxPiece &p, int r0, int nr, bool aligned, bool neg, int tid,
                         uint8_t *hi, uint8_t *lo, float *up, bool store) {
  constexpr int LPR = D / 8, RP = RV_PFX_M / LPR;  // threads a row, rows a pass
  constexpr bool F32 = sizeof(T) == 4;
  if (!F32 && !store) return;
  const int c = tid % LPR;
  for (int b0 = 0; b0 < nr; b0 += 4 * RP) {
    float x[4][8];
#pragma unroll
    for (int k = 0; k < 4; k++) {
      const int row = b0 + k * RP + tid / LPR;
      if (row < nr) {
        const PfxRow pr = pfx_row(a, p.suffix, p.b, p.kvh, r0 + row);
        const T *q = (const T *)a.q + (size_t)pr.b * a.q_seq_stride + (size_t)pr.i * a.q_token_stride +
                     (size_t)pr.h * D + 8 * c;
        if (aligned) {
          if constexpr (F32) {
            *(float4 *)x[k] = __ldg((const float4 *)q);
            *(float4 *)(x[k] + 4) = __ldg((const float4 *)q + 1);
          } else {
            *(uint4 *)x[k] = __ldg((const uint4 *)q);  // eight f16, taken apart below
          }
        } else {
#pragma unroll
          for (int j = 0; j < 8; j++)
            if constexpr (F32) x[k][j] = q[j];
            else ((T *)x[k])[j] = q[j];
        }
      }
    }
#pragma unroll
    for (int k = 0; k < 4; k++) {
      const int row = b0 + k * RP + tid / LPR;
      const uint32_t off = (uint32_t)(c >> 3) * (RV_PFX_M * 128) + tc_sw_off(row, c & 7);
      if constexpr (F32) {
        float m = 0;
#pragma unroll
        for (int j = 0; j < 8; j++) m = fmaxf(m, fabsf(x[k][j]));
        if (row >= nr) m = 0;
#pragma unroll
        for (int o = LPR / 2; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(RV_FULL, m, o));
        // Both 2^e and 2^-e are normal floats.
        const int e = min(max((int)(__float_as_uint(m) >> 23) - 127, -100), 126);
        const float down = __uint_as_float((uint32_t)(127 - e) << 23), sg = neg ? -down : down;
        if (row >= nr) continue;
        if (c == 0) up[row] = __uint_as_float((uint32_t)(e + 127) << 23);
        if (!store) continue;
        uint32_t o[4], r[4];
#pragma unroll
        for (int j = 0; j < 4; j++) {
          const float x0 = x[k][2 * j] * sg, x1 = x[k][2 * j + 1] * sg;
          o[j] = pack_f16(x0, x1);
          const float2 f = __half22float2(*(const __half2 *)&o[j]);
          r[j] = pack_f16(x0 - f.x, x1 - f.y);
        }
        *(uint4 *)(hi + off) = make_uint4(o[0], o[1], o[2], o[3]);
        *(uint4 *)(lo + off) = make_uint4(r[0], r[1], r[2], r[3]);
      } else if (row < nr) {
        uint4 v = *(const uint4 *)x[k];
        const uint32_t sg = neg ? 0x80008000u : 0;
        *(uint4 *)(hi + off) = make_uint4(v.x ^ sg, v.y ^ sg, v.z ^ sg, v.w ^ sg);
      }
    }
  }
}

// Four int8 levels of a word as two half2, in order.
RV_DEVFN void pfx_levels(uint32_t w, uint32_t &a, uint32_t &b) {
  const uint32_t x = w ^ 0x80808080u;  // level + 128
  const __half2 bias = __floats2half2_rn(1152.0f, 1152.0f);
  uint32_t lo = __byte_perm(x, 0x64646464u, 0x4140), hi = __byte_perm(x, 0x64646464u, 0x4342);  // 1024 + level + 128
  __half2 l = __hsub2(*(const __half2 *)&lo, bias), h = __hsub2(*(const __half2 *)&hi, bias);
  a = *(const uint32_t *)&l;
  b = *(const uint32_t *)&h;
}

// Barrier phases that a warp role waits for, with the CTA's failure flag.
RV_DEVFN bool pfx_wait(uint64_t *bar, uint32_t parity) {
  return __all_sync(RV_FULL, mbar_wait_bounded(bar, parity));
}

// One 32-key chunk of a row's scores as t = log2 of the unnormalised weights.
template <bool PRECISE, bool Q8>
RV_DEVFN void pfx_scores(const uint32_t (&v)[32], float c, const float *ck, const float *lv, float (&t)[32]) {
#pragma unroll
  for (int j = 0; j < 32; j += 4) {
    if constexpr (Q8) {
      const float4 k4 = *(const float4 *)(ck + j), l4 = *(const float4 *)(lv + j);
      const float kk[4] = {k4.x, k4.y, k4.z, k4.w}, ll[4] = {l4.x, l4.y, l4.z, l4.w};
#pragma unroll
      for (int x = 0; x < 4; x++) {
        const float s = __uint_as_float(v[j + x]);
        t[j + x] = fmaf(PRECISE ? s * c : s, kk[x], ll[x]);
      }
    } else {
#pragma unroll
      for (int x = 0; x < 4; x++) t[j + x] = __uint_as_float(v[j + x]) * c;
    }
  }
}

template <int D, typename T, bool Q8>
__global__ void __launch_bounds__(PfxCfg<D, T, Q8>::THREADS, 1)
    k_prefix_tc(PrefixArgs a, PfxWork w, const __grid_constant__ CUtensorMap map_pk,
                const __grid_constant__ CUtensorMap map_pv, const __grid_constant__ CUtensorMap map_sk,
                const __grid_constant__ CUtensorMap map_sv) {
  using C = PfxCfg<D, T, Q8>;
  constexpr bool PRECISE = C::PRECISE;
  constexpr int R = C::R, TILE = C::TILE;
  extern __shared__ __align__(16) uint8_t sm_raw_[];
  uint8_t *sm = (uint8_t *)(((uintptr_t)sm_raw_ + 1023) & ~(uintptr_t)1023);
  uint8_t *ring = sm + C::ring;
  float *s_scale = (float *)(sm + C::scales);  // [slot][ck, lv, 1 / sv][128]
  uint64_t *bars = (uint64_t *)(sm + C::bars);
  uint64_t *kv_full = bars, *kv_empty = bars + R, *s_full = bars + 2 * R, *p_ready = s_full + 2, *o_full = p_ready + 2,
           *q_ready = o_full + 2, *sc_full = q_ready + 2, *drained = sc_full + RV_PFX_SCALE_SLOTS;
  int *s_scan = (int *)(bars + C::NBARS);  // [16] warp sums, [17] the first sequence's ub
  int *s_int = s_scan + 32;
  uint32_t *s_tmem = (uint32_t *)s_int;
  volatile int *s_fail = s_int + 1;
  int *s_b = s_int + 2;
  float *s_up = (float *)(s_int + 16);  // [stream][128] powers of two of f32 query rows
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  pdl_trigger();
  if (threadIdx.x == 0) {
    for (int i = 0; i < R; i++) {
      mbar_init(&kv_full[i], Q8 ? 4 : 1);
      mbar_init(&kv_empty[i], 1);
    }
    for (int i = 0; i < 2; i++) {
      mbar_init(&s_full[i], 1);
      mbar_init(&p_ready[i], 4);
      mbar_init(&o_full[i], 1);
      mbar_init(&q_ready[i], 4);
    }
    for (int i = 0; i < RV_PFX_SCALE_SLOTS; i++) mbar_init(&sc_full[i], 4);
    mbar_init(drained, 1);
    *s_fail = 0;
    *s_b = 0;
    s_scan[17] = 0;
  }
  if (warp == 0) {
    __syncwarp();
    tc_alloc(s_tmem, 512);
    tc_relinquish();
  }
  // The line of units: each thread counts the tiles of a run of sequences.
  const int run = ((int)a.n_seqs + (int)blockDim.x - 1) / (int)blockDim.x;
  const int b0 = min((int)threadIdx.x * run, (int)a.n_seqs), b1 = min(b0 + run, (int)a.n_seqs);
  int mine = 0, before;
  for (int b = b0; b < b1; b++) mine += pfx_tiles(prefix_suffix_len(a, (uint32_t)b));
  before = mine;
  for (int o = 1; o < 32; o <<= 1) {
    const int v = __shfl_up_sync(RV_FULL, before, o);
    if (lane >= o) before += v;
  }
  if (lane == 31) s_scan[warp] = before;
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *s_tmem;
  int all = 0;
  for (int i = 0; i < (int)blockDim.x / 32; i++) {
    if (i < warp) before += s_scan[i];
    all += s_scan[i];
  }
  before -= mine;
  const int segs = (int)a.n_kv * w.nrt_s;
  PfxWalk walk;
  walk.wp = (int)a.n_kv * w.nrt_p * w.tp;
  const int W = walk.wp + all * segs, per = (W + w.grid - 1) / w.grid;
  walk.c = blockIdx.x;
  walk.u = min(W, blockIdx.x * per);
  walk.end = min(W, walk.u + per);
  if (blockIdx.x == 0) {
    int x = before;
    for (int b = b0; b < b1; b++) {
      w.cum[b] = x;
      x += pfx_tiles(prefix_suffix_len(a, (uint32_t)b));
    }
    if (threadIdx.x == 0) w.cum[a.n_seqs] = all;
  }
  if (walk.u >= walk.wp && walk.u < W) {  // the sequence whose units hold the first
    const int us = walk.u - walk.wp;
    if (us >= before * segs && us < (before + mine) * segs) {
      int x = before;
      int b = b0;
      for (;; b++) {
        const int t = pfx_tiles(prefix_suffix_len(a, (uint32_t)b));
        if (us < (x + t) * segs) break;
        x += t;
      }
      *s_b = b;
      s_scan[17] = x * segs;
    }
  }
  __syncthreads();
  walk.b = *s_b;
  walk.ub = s_scan[17];
  PfxPiece p;

  if (!Q8 && warp == 0) {
    // ------------------------------------------------------------ loads
    if (lane == 0) {
      bool ok = true;
      int n0 = 0;  // loads of earlier pieces
      while (ok && !*s_fail && pfx_next(a, w, walk, p)) {
        const CUtensorMap *mk = p.suffix ? &map_sk : &map_pk, *mv = p.suffix ? &map_sv : &map_pv;
        for (int i = 0; i < 2 * p.n; i++) {
          bool is_k;
          int t;
          pfx_load_at(p.pair, i, p.n, is_k, t);
          const int n = n0 + i, slot = n % R;
          if (!mbar_wait_bounded(&kv_empty[slot], ((n / R) & 1) ^ 1)) {
            ok = false;
            n0 = n - 2 * p.n;  // loads issued so far are n (see the drain below)
            break;
          }
          mbar_arrive_expect_tx(&kv_full[slot], (uint32_t)TILE);
#pragma unroll
          for (int h = 0; h < D / 64; h++)
            tma_load_4d(ring + (size_t)slot * TILE + h * (RV_PFX_N * 128), is_k ? mk : mv, 64 * h, p.kvh,
                        (p.tile0 + t) * RV_PFX_N, p.suffix ? p.b : 0, &kv_full[slot]);
        }
        n0 += 2 * p.n;
      }
      if (!ok) *s_fail = 1;
      if (*s_fail)  // let the copies in flight land before the CTA ends
        for (int n = max(0, n0 - R); n < n0; n++) mbar_wait_bounded(&kv_full[n % R], (n / R) & 1);
    }
    __syncwarp();
  } else if (warp == 1) {
    // ------------------------------------------------------- MMA issue
    const uint32_t hi_sw = (1024u >> 4) | (1u << 14) | (2u << 29);
    const uint32_t lbo_k = 1u << 16, lbo_v = (uint32_t)(RV_PFX_N * 128 >> 4) << 16;
    const uint32_t q_lo = smem_addr(sm) >> 4, ring_lo = smem_addr(ring) >> 4;
    const uint32_t idesc_s = tc_idesc(RV_PFX_N), idesc_o = tc_idesc(D) | (1u << 16);  // B of P V: keys down the rows
    auto mk = [](uint32_t lo, uint32_t hi) { return ((uint64_t)hi << 32) | lo; };
    bool ok = true;
    int n0 = 0, np[2] = {0, 0}, nq[2] = {0, 0};
    while (ok && !*s_fail && pfx_next(a, w, walk, p)) {
      const int step = p.pair ? 1 : 2;
      // S of tile t of stream s; the key tile is released by its last reader.
      auto qk = [&](int s, int t) {
        const int n = n0 + pfx_k_at(p.pair, t), slot = n % R;
        if (!pfx_wait(&kv_full[slot], (n / R) & 1)) return false;
        tc_fence_after();
        if (lane == 0) {
          const uint32_t qa = q_lo + (p.pair && s ? TILE >> 4 : 0), kb = ring_lo + (uint32_t)(slot * (TILE >> 4));
#pragma unroll
          for (int kk = 0; kk < D / 16; kk++) {
            const uint32_t o = (uint32_t)(kk >> 2) * (RV_PFX_M * 128 >> 4) + 2 * (kk & 3);
            tc_mma_f16(tmem + 128 * s, mk(lbo_k | (qa + o), hi_sw), mk(lbo_k | (kb + o), hi_sw), idesc_s, kk != 0);
            if (PRECISE)
              tc_mma_f16(tmem + 128 * s, mk(lbo_k | (qa + (TILE >> 4) + o), hi_sw), mk(lbo_k | (kb + o), hi_sw),
                         idesc_s, 1u);
          }
          if (!p.pair || s) tc_commit(&kv_empty[slot]);
          tc_commit(&s_full[s]);
        }
        __syncwarp();
        return true;
      };
      auto pv = [&](int s, int t, bool first, bool last) {
        const int n = n0 + pfx_v_at(p.pair, t, p.n), slot = n % R;
        if (!pfx_wait(&kv_full[slot], (n / R) & 1)) return false;
        const int valid = min(RV_PFX_N, p.keys - (p.tile0 + t) * RV_PFX_N);
        if (!Q8 && p.suffix && (valid & 15) && !(p.pair && s)) {
          // Rows past the sequence's end hold whatever the cache held: zero
          // those the last K step reads (0 * NaN is not 0).
          const int rows = ((valid + 15) & ~15) - valid;
          for (int i = lane; i < rows * (D / 8); i += 32) {
            const int r = valid + i / (D / 8), ch = i % (D / 8);
            *(uint4 *)(ring + (size_t)slot * TILE + (ch >> 3) * (RV_PFX_N * 128) + tc_sw_off(r, ch & 7)) =
                make_uint4(0, 0, 0, 0);
          }
          fence_proxy_async();
          __syncwarp();
        }
        if (!pfx_wait(&p_ready[s], np[s] & 1)) return false;
        np[s]++;
        tc_fence_after();
        if (lane == 0) {
          const uint32_t vb = ring_lo + (uint32_t)(slot * (TILE >> 4)), d = tmem + RV_PFX_O + 128 * s;
          const int steps = (valid + 15) >> 4;
          for (int kk = 0; kk < steps; kk++) {
            const uint32_t pa = tmem + 128 * s + 32 * (kk >> 1) + 8 * (kk & 1);
            const uint64_t bd = mk(lbo_v | (vb + (uint32_t)kk * (2048 >> 4)), hi_sw);
            tc_mma_f16_ta(d, pa, bd, idesc_o, !(first && kk == 0));
            if (PRECISE) tc_mma_f16_ta(d, pa + 16, bd, idesc_o, 1u);
          }
          if (!p.pair || s) tc_commit(&kv_empty[slot]);
          if (last) tc_commit(&o_full[s]);
        }
        __syncwarp();
        return true;
      };
      // The query tiles: one for both streams, or one each.
      for (int s = 0; ok && s < (p.pair ? 2 : 1); s++) {
        ok = pfx_wait(&q_ready[s], nq[s] & 1);
        nq[s]++;
      }
      tc_fence_after();
      for (int s = 0; ok && s < 2; s++)
        if (p.pair || s < p.n) ok = qk(s, p.pair ? 0 : s);
      for (int j = 0; ok && j < p.n; j += step)
        for (int s = 0; ok && s < 2; s++) {
          const int t = p.pair ? j : j + s;
          if (t >= p.n) break;
          const bool more = t + step < p.n;
          ok = pv(s, t, j == 0, !more);
          if (ok && more) ok = qk(s, t + step);
        }
      n0 += 2 * p.n;
    }
    if (!ok) *s_fail = 1;
    if (*s_fail) {  // products in flight end before tensor memory is freed
      if (lane == 0) {
        tc_commit(drained);
        mbar_wait_bounded(drained, 0);
      }
      __syncwarp();
    }
  } else if (warp >= 4 && warp < 12) {
    // --------------------------------------------------------- softmax
    const int s = (warp - 4) >> 2, quad = warp & 3, row = 32 * quad + lane;
    const uint32_t tl = tmem + ((uint32_t)(32 * quad) << 16), tS = tl + 128 * s, tO = tl + RV_PFX_O + 128 * s;
    const bool neg = a.scale_log2 < 0;  // the sign of the scale goes to the queries
    const float scale = fabsf(a.scale_log2);
    bool ok = true;
    int ns = 0, no = 0;
    int gt = 0;  // tiles of earlier pieces
    while (ok && !*s_fail && pfx_next(a, w, walk, p)) {
      const int step = p.pair ? 1 : 2, t_first = p.pair ? 0 : s;
      const int rr = (p.pair ? RV_PFX_M * s : 0) + row;
      const bool on = rr < p.nrows;
      const bool warp_on = __any_sync(RV_FULL, on);
      const PfxRow pr = pfx_row(a, p.suffix, p.b, p.kvh, p.row0 + (on ? rr : 0));
      int seen = p.keys;  // keys of the segment that this row sees
      if (p.suffix) seen = min(max(p.keys - (int)a.n_q + 1 + pr.i, 0), p.keys);
      if (!on) seen = 0;
      pfx_load_q<D, T>(a, p, p.row0 + (p.pair ? RV_PFX_M * s : 0), min(RV_PFX_M, p.nrows - (p.pair ? RV_PFX_M * s : 0)),
                       w.q_aligned, neg, row, sm + (p.pair && s ? TILE : 0), sm + TILE, s_up + RV_PFX_M * s,
                       p.pair || s == 0);
      if (p.pair || s == 0) {
        fence_proxy_async();
        __syncwarp();
        if (lane == 0) mbar_arrive(&q_ready[s]);
      }
      float up = 1.0f;
      if constexpr (PRECISE) {
        asm volatile("bar.sync %0, 128;" ::"r"(1 + s) : "memory");  // the stream's four warps
        if (on) up = s_up[RV_PFX_M * s + row];
        // The next piece's are written once every warp has read these: a
        // stream with tiles waits for its O, which needs all four warps' P.
        if (t_first >= p.n) asm volatile("bar.sync %0, 128;" ::"r"(1 + s) : "memory");
      }
      const float c = Q8 ? up : up * scale;
      float m_ref = -INFINITY, l = 0.0f;
      for (int t = t_first; ok && t < p.n; t += step) {
        const int tile = p.tile0 + t, valid = min(RV_PFX_N, p.keys - tile * RV_PFX_N), nch = (valid + 31) >> 5;
        const int lim = min(max(seen - tile * RV_PFX_N, 0), RV_PFX_N);
        const float *sc = s_scale + (size_t)((gt + t) % RV_PFX_SCALE_SLOTS) * 3 * RV_PFX_N;
        if (Q8) ok = pfx_wait(&sc_full[(gt + t) % RV_PFX_SCALE_SLOTS], (uint32_t)((gt + t) / RV_PFX_SCALE_SLOTS) & 1);
        ok = ok && pfx_wait(&s_full[s], ns & 1);
        ns++;
        if (!ok) break;
        tc_fence_after();
        if (warp_on) {
          const bool full = __all_sync(RV_FULL, lim == RV_PFX_N || !on);
          float mx = -INFINITY;
          for (int ch = 0; ch < nch; ch++) {
            uint32_t v[32];
            float x[32];
            tc_ld32(tS + 32 * ch, v);
            pfx_scores<PRECISE, Q8>(v, c, sc + 32 * ch, sc + RV_PFX_N + 32 * ch, x);
            if (full) {
#pragma unroll
              for (int j = 0; j < 32; j++) mx = fmaxf(mx, x[j]);
            } else {
#pragma unroll
              for (int j = 0; j < 32; j++) mx = fmaxf(mx, 32 * ch + j < lim ? x[j] : -INFINITY);
            }
          }
          if (!on) mx = -INFINITY;
          if (t == t_first) {
            m_ref = mx;
          } else if (const bool move = mx > m_ref + RV_PFX_LAG; __any_sync(RV_FULL, move)) {
            // Every product issued so far is done (S came after them).
            const float f = move ? ex2(m_ref - mx) : 1.0f;
            if (move) m_ref = mx;
            l *= f;
            for (int ch = 0; ch < D / 32; ch++) {
              uint32_t v[32];
              tc_ld32(tO + 32 * ch, v);
#pragma unroll
              for (int j = 0; j < 32; j++) v[j] = __float_as_uint(__uint_as_float(v[j]) * f);
              tc_st16(tO + 32 * ch, v);
              tc_st16(tO + 32 * ch + 16, v + 16);
            }
          }
          const float m_use = m_ref == -INFINITY ? 0.0f : m_ref - RV_PFX_LIFT;
          float l0 = 0, l1 = 0;
          for (int ch = 0; ch < nch; ch++) {
            uint32_t v[32];
            float x[32];
            tc_ld32(tS + 32 * ch, v);
            pfx_scores<PRECISE, Q8>(v, c, sc + 32 * ch, sc + RV_PFX_N + 32 * ch, x);
#pragma unroll
            for (int j = 0; j < 32; j++) x[j] = ex2(x[j] - m_use);
            if (!full) {
#pragma unroll
              for (int j = 0; j < 32; j++) x[j] = 32 * ch + j < lim ? x[j] : 0.0f;
            }
            if constexpr (Q8) {
#pragma unroll
              for (int j = 0; j < 32; j += 4) {
                const float4 r4 = *(const float4 *)(sc + 2 * RV_PFX_N + 32 * ch + j);
                const float rs[4] = {r4.x, r4.y, r4.z, r4.w};
                // A hidden token's 1 / scale may be NaN: its weight is 0 all the same.
#pragma unroll
                for (int y = 0; y < 4; y++) {
                  const float add = full || 32 * ch + j + y < lim ? x[j + y] * rs[y] : 0.0f;
                  if (y & 1) l1 += add;
                  else l0 += add;
                }
              }
            } else {
#pragma unroll
              for (int j = 0; j < 32; j += 2) {
                l0 += x[j];
                l1 += x[j + 1];
              }
            }
            uint32_t o[16], r[16];
#pragma unroll
            for (int j = 0; j < 16; j++) {
              o[j] = pack_f16(x[2 * j], x[2 * j + 1]);
              if constexpr (PRECISE) {
                const float2 f = __half22float2(*(const __half2 *)&o[j]);
                r[j] = pack_f16(x[2 * j] - f.x, x[2 * j + 1] - f.y);
              }
            }
            // P takes the columns its scores came from.
            tc_st16(tS + 32 * ch, o);
            if constexpr (PRECISE) tc_st16(tS + 32 * ch + 16, r);
          }
          l += l0 + l1;
          tc_wait_st();
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_ready[s]);
      }
      gt += p.n;
      // ------------------------------------------- the piece's (m, l, O)
      const int rw = p.suffix ? w.rw_s : RV_PFX_M;
      const size_t part = (size_t)p.slot * 2 + s;
      float4 *po = (p.suffix ? w.o_s : w.o_p) + part * (D / 4) * rw + row;
      float2 *pm = (p.suffix ? w.ml_s : w.ml_p) + part * rw + row;
      if (ok && t_first < p.n) {
        ok = pfx_wait(&o_full[s], no & 1);
        no++;
        if (!ok) break;
        tc_fence_after();
        if (warp_on) {
          for (int ch = 0; ch < D / 32; ch++) {
            uint32_t v[32];
            tc_ld32(tO + 32 * ch, v);
            if (on) {
#pragma unroll
              for (int j = 0; j < 8; j++)
                po[(size_t)(8 * ch + j) * rw] =
                    make_float4(__uint_as_float(v[4 * j]), __uint_as_float(v[4 * j + 1]), __uint_as_float(v[4 * j + 2]),
                                __uint_as_float(v[4 * j + 3]));
            }
          }
          tc_fence_before();
        }
      }
      if (on) *pm = make_float2(m_ref == -INFINITY ? -INFINITY : m_ref - RV_PFX_LIFT, l);
    }
    if (!ok) *s_fail = 1;
  } else if (Q8 && warp >= 12) {
    // ------------------------------------ 8-bit rows into f16 operands
    // 16 levels a thread and load: D / 16 threads a token.  The next tile's
    // levels are in registers before its stage is free.
    constexpr int TPT = D / 16, TOK = 128 / TPT, IT = RV_PFX_N / TOK;
    const int ct = threadIdx.x - 384, tok0 = ct / TPT, e = (ct % TPT) * 16;
    bool ok = true;
    int n0 = 0, gt = 0;
    while (ok && !*s_fail && pfx_next(a, w, walk, p)) {
      const size_t first = (p.suffix ? (size_t)p.b * a.cap : 0) + (size_t)p.tile0 * RV_PFX_N;
      const int left = p.keys - p.tile0 * RV_PFX_N;  // keys from the piece's first tile on
      for (int i = 0; ok && i < 2 * p.n; i++) {
        bool is_k;
        int t;
        pfx_load_at(p.pair, i, p.n, is_k, t);
        const int n = n0 + i, slot = n % R, valid = min(RV_PFX_N, left - t * RV_PFX_N);
        const int8_t *src = (const int8_t *)(is_k ? (p.suffix ? a.sk : a.pk) : (p.suffix ? a.sv : a.pv));
        uint4 x[IT];
#pragma unroll
        for (int j = 0; j < IT; j++) {
          const int tok = tok0 + j * TOK;
          x[j] = tok < valid
                     ? __ldcs((const uint4 *)(src + ((first + (size_t)t * RV_PFX_N + tok) * a.n_kv + p.kvh) * D + e))
                     : make_uint4(0, 0, 0, 0);
        }
        float ks = 0, vs = 0;
        if (is_k && ct < valid) {
          const size_t at = (first + (size_t)t * RV_PFX_N + ct) * a.n_kv + p.kvh;
          ks = (p.suffix ? a.sks : a.pks)[at];
          vs = (p.suffix ? a.svs : a.pvs)[at];
        }
        ok = pfx_wait(&kv_empty[slot], ((n / R) & 1) ^ 1);
        if (!ok) break;
        if (is_k) {
          float *sc = s_scale + (size_t)((gt + t) % RV_PFX_SCALE_SLOTS) * 3 * RV_PFX_N;
          // A scale of 0 stands for a row of zeros: any scale does.  NaN and
          // infinity pass on.
          const float v1 = vs < 0x1p-60f ? 0x1p-60f : vs;
          sc[ct] = ks * fabsf(a.scale_log2);
          sc[RV_PFX_N + ct] = log2f(v1);
          sc[2 * RV_PFX_N + ct] = __frcp_rn(v1);
          __syncwarp();
          if (lane == 0) mbar_arrive(&sc_full[(gt + t) % RV_PFX_SCALE_SLOTS]);
        }
        uint8_t *dst = ring + (size_t)slot * TILE + (e >> 6) * (RV_PFX_N * 128);
#pragma unroll
        for (int j = 0; j < IT; j++) {
          const int tok = tok0 + j * TOK, ch = (e & 63) >> 3;
          uint32_t o[8];
          pfx_levels(x[j].x, o[0], o[1]);
          pfx_levels(x[j].y, o[2], o[3]);
          pfx_levels(x[j].z, o[4], o[5]);
          pfx_levels(x[j].w, o[6], o[7]);
          *(uint4 *)(dst + tc_sw_off(tok, ch)) = make_uint4(o[0], o[1], o[2], o[3]);
          *(uint4 *)(dst + tc_sw_off(tok, ch + 1)) = make_uint4(o[4], o[5], o[6], o[7]);
        }
        fence_proxy_async();
        __syncwarp();
        if (lane == 0) mbar_arrive(&kv_full[slot]);
      }
      n0 += 2 * p.n;
      gt += p.n;
    }
    if (!ok) *s_fail = 1;
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 0) {
    tc_fence_after();
    tc_dealloc(tmem, 512);
  }
}

// The parts of each query row added up: out = sum 2^(m_p - M) O_p / sum
// 2^(m_p - M) l_p.  grid = (8-row groups of a kv head's rows, kv heads); a warp
// holds eight rows times four part lanes (each takes every fourth part) and
// two groups of four values, so a load is 128 contiguous bytes a part.
#define RV_PFX_JOIN_ROWS 8
template <int D, typename T>
__global__ void __launch_bounds__(D * 4) k_prefix_join(PrefixArgs a, PfxWork w) {
  const int lane = threadIdx.x & 31, d4 = threadIdx.x >> 5, kvh = blockIdx.y, pl = lane >> 3;
  const int r = min((int)blockIdx.x * RV_PFX_JOIN_ROWS + (lane & 7), w.rows_p - 1);
  const bool on = (int)blockIdx.x * RV_PFX_JOIN_ROWS + (lane & 7) < w.rows_p;
  const PfxRow pr = pfx_row(a, false, 0, kvh, r);
  const int segs = (int)a.n_kv * w.nrt_s, wp = (int)a.n_kv * w.nrt_p * w.tp;
  pdl_wait();  // cum and the parts are k_prefix_tc's
  const int W = wp + w.cum[a.n_seqs] * segs, per = max(1, (W + w.grid - 1) / w.grid);
  // The row's parts: those of its prefix segment, then of its sequence's
  // suffix segment; each a run with a constant step.
  const float2 *ml[2];
  const float4 *po[2];
  int n[2], step[2], rw[2];
#pragma unroll
  for (int s = 0; s < 2; s++) {
    const int rows = s ? w.rows_s : w.rows_p, x = s ? r - pr.b * w.rows_s : r, in = x % w.sr;
    const int c0 = s ? w.cum[pr.b] : 0, tiles = s ? w.cum[pr.b + 1] - c0 : w.tp;
    const int local = kvh * (s ? w.nrt_s : w.nrt_p) + x / w.sr, seg = s ? pr.b * segs + local : local;
    const int u0 = s ? wp + c0 * segs + local * tiles : seg * tiles;
    const bool pair = min(w.sr, rows - (x - in)) > RV_PFX_M;
    const int first = u0 / per, last = (u0 + tiles - 1) / per;
    const size_t part = (size_t)(seg + first) * 2 + (pair ? in / RV_PFX_M : 0);
    rw[s] = s ? w.rw_s : RV_PFX_M;
    step[s] = pair ? 2 : 1;
    n[s] = tiles == 0 ? 0 : (last - first + 1) * (pair ? 1 : 2);
    ml[s] = (s ? w.ml_s : w.ml_p) + part * rw[s] + in % RV_PFX_M;
    po[s] = (s ? w.o_s : w.o_p) + (part * (D / 4) + d4) * rw[s] + in % RV_PFX_M;
  }
  float M = -INFINITY, L = 0;
#pragma unroll
  for (int s = 0; s < 2; s++)
#pragma unroll 4
    for (int i = pl; i < n[s]; i += 4) M = fmaxf(M, ml[s][(size_t)i * step[s] * rw[s]].x);
  M = fmaxf(M, __shfl_xor_sync(RV_FULL, M, 8));
  M = fmaxf(M, __shfl_xor_sync(RV_FULL, M, 16));
  float o[8] = {0, 0, 0, 0, 0, 0, 0, 0};
#pragma unroll
  for (int s = 0; s < 2; s++)
#pragma unroll 4
    for (int i = pl; i < n[s]; i += 4) {
      const float2 x = ml[s][(size_t)i * step[s] * rw[s]];
      const float4 *q = po[s] + (size_t)i * step[s] * (D / 4) * rw[s];
      const float4 v[2] = {q[0], q[(D / 8) * rw[s]]};
      // -infinity: the row saw none of the part's keys, whose O may be anything.
      const bool sees = x.x != -INFINITY;
      const float f = sees ? exp2f(x.x - M) : 0.0f;
      L += sees ? x.y * f : 0.0f;
#pragma unroll
      for (int j = 0; j < 2; j++) {
        o[4 * j] += sees ? v[j].x * f : 0.0f;
        o[4 * j + 1] += sees ? v[j].y * f : 0.0f;
        o[4 * j + 2] += sees ? v[j].z * f : 0.0f;
        o[4 * j + 3] += sees ? v[j].w * f : 0.0f;
      }
    }
#pragma unroll
  for (int k = 8; k <= 16; k *= 2) {
    L += __shfl_xor_sync(RV_FULL, L, k);
#pragma unroll
    for (int j = 0; j < 8; j++) o[j] += __shfl_xor_sync(RV_FULL, o[j], k);
  }
  if (!on || pl >= 2) return;
  const float inv = L == 0.0f ? 0.0f : 1.0f / L;
  T *out = (T *)a.out + (((size_t)pr.b * a.n_q + pr.i) * a.n_heads + pr.h) * D + 4 * (d4 + pl * (D / 8));
  float v[4];
#pragma unroll
  for (int j = 0; j < 4; j++) v[j] = (pl ? o[4 + j] : o[j]) * inv;
  if (!w.out_aligned) {
#pragma unroll
    for (int j = 0; j < 4; j++) out[j] = (T)v[j];
  } else if constexpr (sizeof(T) == 4) {
    *(float4 *)out = make_float4(v[0], v[1], v[2], v[3]);
  } else {
    *(uint2 *)out = make_uint2(pack_f16(v[0], v[1]), pack_f16(v[2], v[3]));
  }
}
