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
#include <limits.h>

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

// The power of two of a scale's size: f32 queries take it before they meet the
// levels of 8-bit keys (exactly), so that large ones do not overflow there.
RV_DEVFN float prefix_pow2(float scale) {
  return __uint_as_float(max(__float_as_uint(scale) & 0x7F800000u, 0x00800000u));
}

// A sequence's suffix length, held inside its cache.
RV_DEVFN int prefix_suffix_len(const PrefixArgs &a, uint32_t b) {
  const int n = a.lens[b];
  if (n < 0 || n > (int)a.cap) rv_dev_fail(RV_ERR_CAPACITY_EXCEEDED);
  return min(max(n, 0), (int)a.cap);
}

// Head dims other than 64 and 128 (multiples of 8 up to 256): one CTA of eight warps per
// query row, a warp per key in turn, head_dim spread over the lanes, so a
// score is one warp sum.  The keys and values of the prefix are read once per
// query row, not once per batch, and a key waits for the sum before it: bound by
// that latency (head_dim 96, f16 rows, 16 query and 4 kv heads: one sequence over
// 1,024 positions 55 us, 64 over 8,192 1.17 ms; head_dim 128 through the tensor
// cores 13 and 27 us, f32 queries 14 and 42).
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
  const float p2 = prefix_pow2(a.scale_log2), rest = a.scale_log2 / p2;
#pragma unroll
  for (int t = 0; t < 8; t++) q[t] *= p2;
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
    s *= rest;
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
// Work: a segment is a run of query rows of one kv head against the prefix or
// against one sequence's suffix, cut into units of 128 keys.  The segments'
// units stand on a line, with RV_PFX_OV places more for each segment's fixed
// cost (one place costs about what a tile does: the loads of Q, the first tiles
// and the parts' stores), and the line is split evenly; every stretch of a segment is a piece
// that leaves (m, l, O) of its rows in scratch, and k_prefix_join adds the
// pieces of a row up.  The split follows from the lengths alone, so the result
// does not depend on timing.
//
// Per CTA (one an SM) two streams run through the tensor cores, each with its
// own S, P and O columns and its own softmax warpgroup (thread = row), so one
// stream's products run under the other's exponentials.
//   solo: each stream walks a stretch of the line of its own.
//   pair: more than 128 query rows of a kv head share the prefix (f16 queries):
//   the streams take 128 rows each of a segment of 256 and read the same key
//   and value tiles, halving the traffic per product.  The prefix then has a
//   line of its own, over a share of the CTAs that follows the costs (8 query
//   heads a kv head; 128 sequences over an f16 32K prompt 98 us, solo 113, at
//   head_dim 64 77 and 94; 64 over an 8-bit 16K one 62 and 72, at head_dim 64 53
//   and 60; 17 sequences, 136 rows: 38 and 41, 8-bit 39 and 45; with 128 rows or
//   fewer there is no second stream to pair).
//
// What bounds it: a unit is 2,048 cycles of products and as many of
// exponentials (16 a cycle and SM), and a stream's chain S -> exponentials -> P
// V -> next S takes about twice that, so two streams keep the tensor pipe 0.42
// active at 128 sequences over 32K positions (its floor is 40 us; K and V are
// read from memory once, 119 MB).  Over an 8-bit cache the pipe is 0.20 active
// and no memory or issue slot is full: a tile's conversion to f16 by three warps
// stands in the chain before its products.  f32 queries: 278 us there, the pipe
// 0.52 active with four times the products, and half the rows of each are empty
// at head_dim 128.  Small calls are bound by the fixed chain of planning, loading
// Q, one unit, and the join: 13 us at one short sequence.
//
// f32 queries are held to 2^-22 of their row's largest value as a sum of two
// f16 (after scaling by a power of two), and so is P: products of f16 with the
// f16 (or 8-bit) keys and values are exact, so the result carries f32's
// rounding only.  The tensor cores' accumulator truncates, so O leaves it every
// RV_PFX_RUN tiles and is summed up in the part, by f32 additions in memory that
// nothing waits for and that the row's own thread gives in order (8 sequences over 4K positions: 6e-7 of the norm against 64
// bits, f32 sums 1.6e-6; 1,024 tokens over 32K: 1.8e-6 and 3.5e-6, values of one sign
// 3.3e-6 and 4.9e-6; in one accumulation these were 6e-5 and 2e-4.  Runs of 8
// tiles: up to 7e-6, and 2 % faster on 128 sequences over 32K).  The price of f32 is
// twice the products, and for head_dim 128 query tiles of 64 rows (two operands a
// stream in shared memory).
// f16 queries round P to f16 once, the size of the output's own rounding
// (together 2.9e-4 of the norm, where the output's alone is 2.1e-4), and sum a
// piece in one accumulation (values of one sign over 32K positions: 2.4e-4, the
// output's rounding alone 1.8e-4).  P in two terms took 48 sequences' own tokens
// from 36 to 40 us, 64 over an 8-bit 16K prompt from 62 to 72, 128 over 32K from
// 98 to 123.  P is lifted by 2^7 and the reference maximum may lag by 2^8, so P stays below 2^15 and a weight is a
// normal f16 down to 2^-21 of the largest.
//
// 8-bit cache: levels are exact in f16, so the products run on levels; a token's
// key scale multiplies its score and its value scale its weight, both in f32
// (f32 queries take the attention scale's power of two first, so that large ones
// do not overflow against the levels).
// P holds the value scale, so the reference is that of the products: with 2^e
// above a token's value scale, the largest s + e of the keys that the row sees.
// What a row does not see, or sees with next to no weight, does not move it
// (with one exponent a tile, for its largest value, it did, and 64 sequences took
// 58 us for 62, f32 queries 155 for 162).
#define RV_PFX_CTAS 148       // CTAs at most: one per SM of a B200
#define RV_PFX_THREADS 384    // loads, products and conversion; two softmax warpgroups
#define RV_PFX_CONV 96        // threads that turn 8-bit rows into f16 (warps 0, 2, 3)
#define RV_PFX_M 128          // rows of a product
#define RV_PFX_N 128          // keys of a tile
#define RV_PFX_OV 1           // a segment's fixed cost, in units
#define RV_PFX_LAG 8.0f       // the reference maximum may lag by this (log2)
#define RV_PFX_RUN 4          // tiles that an f32 row's O is summed over in tensor memory
#define RV_PFX_LIFT 7.0f      // P is lifted by 2^7
#define RV_PFX_SCALE_SLOTS 8  // tiles a stream whose token scales are in shared memory
#define RV_PFX_SCALE (3 * RV_PFX_N)  // floats of a tile's scales: keys', values', the values' exponents
#define RV_PFX_TABLE 32       // pieces a stream works through between plans: one a lane
#define RV_PFX_O 256          // first tensor-memory column of O (S and P: 0..255)

// n / d for 0 <= n < 2^31 by a multiplication (Granlund and Montgomery, 1994).
struct PfxDiv {
  uint32_t mul, shift;
  PfxDiv() = default;
  __host__ explicit PfxDiv(uint32_t d) {
    shift = 0;
    while (shift < 31 && (1u << shift) < d) shift++;
    mul = (uint32_t)((((1ull << shift) - d) << 32) / d + 1);
  }
  RV_DEVFN int operator()(int n) const { return (int)((__umulhi((uint32_t)n, mul) + (uint32_t)n) >> shift); }
};

struct PfxWork {
  int tp;              // prefix tiles
  int rows_p, rows_s;  // query rows of one kv head: all sequences', one sequence's
  int sr_p, sr_s;      // rows of a prefix / suffix segment
  int nrt_p, nrt_s;    // segments per kv head (per sequence)
  int rw_p, rw_s;      // rows of a part
  int pair;            // the prefix runs on paired streams
  float pair_cost;     // a paired unit's cost in solo places
  PfxDiv by_g, by_row; // divisions by the query heads of a kv head, by the query rows of a sequence's
  int grid;
  int q_aligned, out_aligned;  // 16-byte loads and stores
  int *cum;            // [2 n_seqs + 1]: suffix tiles, then suffixes that are not empty, before sequence b
  float4 *o_p, *o_s;   // parts: [part][hd / 4][rows]
  float2 *ml_p, *ml_s; // [part][rows] (m, l)
};

// How the lines are split: the same on every CTA and in the join.
struct PfxLine {
  int gp;            // CTAs of the paired prefix (0: none)
  int per_p, per;    // places a paired CTA / a solo stream takes
  int wp, w;         // places of the paired prefix; of the solo line
  int solo_p;        // places of the prefix on the solo line (they come first)
};
RV_DEVFN int pfx_tiles(int keys) { return (keys + RV_PFX_N - 1) / RV_PFX_N; }
RV_DEVFN PfxLine pfx_line(const PrefixArgs &a, const PfxWork &w, int tiles, int filled) {
  PfxLine l;
  const int seg_p = (int)a.n_kv * w.nrt_p, seg_s = (int)a.n_kv * w.nrt_s;
  const int suffix = (tiles + filled * RV_PFX_OV) * seg_s;
  l.solo_p = w.pair || w.tp == 0 ? 0 : seg_p * (w.tp + RV_PFX_OV);
  l.wp = w.pair ? seg_p * w.tp : 0;
  l.w = l.solo_p + suffix;
  // A paired segment costs about three units more than its own.
  l.gp = 0;
  if (l.wp) {
    const float cost = __fmul_rn(w.pair_cost, (float)(l.wp + 3 * seg_p));
    const float share = __fdiv_rn(cost, __fadd_rn(cost, (float)l.w));
    l.gp = min(max(__float2int_rn(__fmul_rn(share, (float)w.grid)), 1), l.w ? w.grid - 1 : w.grid);
  }
  l.per_p = l.gp ? (l.wp + l.gp - 1) / l.gp : 1;
  const int streams = 2 * (w.grid - l.gp);
  l.per = max(1, streams ? (l.w + streams - 1) / streams : 1);
  return l;
}

// A piece: a stretch of a segment.  n = 0: nothing to do.
struct __align__(16) PfxPiece {
  int b, head, row0, keys;  // head: 2 * kv head + (1: a suffix)
  int tile0, n, part, pad;
};
// A stream's stretch of its line: places [u, end), which is stretch v.
struct PfxStretch {
  int u, end, v;
};
// Segment [at, at + len) of the line (fixed cost ov, then tiles) cut to a stretch.
RV_DEVFN void pfx_cut(PfxPiece &p, const PfxStretch &k, int at, int tiles, int ov) {
  const int x0 = max(k.u - at, 0), x1 = min(k.end - at, tiles + ov);
  p.tile0 = max(0, x0 - ov);
  p.n = max(0, x1 - ov - p.tile0);
}

template <int D, typename T, bool Q8>
struct PfxCfg {
  static constexpr bool PRECISE = sizeof(T) == 4;
  static constexpr int SR = PRECISE && D == 128 ? 64 : 128;     // query rows of a stream
  static constexpr int QT = SR * D * 2;                         // bytes of one query operand
  static constexpr int QS = QT * (PRECISE ? 2 : 1);             // of a stream's
  static constexpr int TILE = RV_PFX_N * D * 2;                 // of a K or V tile
  static constexpr bool RUNS = PRECISE;                         // O leaves tensor memory every RV_PFX_RUN tiles
  static constexpr int R = D == 64 ? (Q8 ? 6 : 8) : Q8 ? 3 : 5;  // K/V ring stages
  static constexpr int RAW = Q8 ? 2 * RV_PFX_N * D : 0;         // two tiles of levels on their way
  static constexpr int SCALES = Q8 ? 2 * RV_PFX_SCALE_SLOTS * RV_PFX_SCALE * 4 : 0;
  static constexpr int NBARS = 2 * R + 8 + 2 * RV_PFX_SCALE_SLOTS + 1;
  static constexpr size_t ring = 2 * QS, raw = ring + (size_t)R * TILE, scales = raw + RAW, table = scales + SCALES,
                          ups = table + 2 * RV_PFX_TABLE * sizeof(PfxPiece), bars = ups + (PRECISE ? 4 * SR : 0);
  static constexpr size_t total = bars + NBARS * 8 + 8 * 4;
  static_assert(total <= 227 * 1024, "shared memory of a CTA");
};

// The order in which K and V tiles are first used, for the warps that bring
// them in: K of each stream's first unit, then in turn for each stream V of its
// unit and K of its next.  Paired streams use the same tiles: one stream here.
RV_DEVFN void pfx_entry(const PfxPiece *tab, int count, int &i, int &n) {
  for (n = 0; i < count; i++)
    if ((n = tab[i].n) > 0) return;
}
struct PfxSide {  // a stream
  int at, left, tile, unit;  // table entry, its units not loaded yet, the next one's tile; units so far
  int b, head, keys;
  bool begun;  // K of the next unit is loaded
  RV_DEVFN void enter(const PfxPiece *tab, int count) {
    pfx_entry(tab, count, at, left);
    if (left) {
      tile = tab[at].tile0;
      b = tab[at].b;
      head = tab[at].head;
      keys = tab[at].keys;
    }
  }
};
struct PfxFeed {
  PfxSide c, o;  // the stream in turn and the other
  int s;         // which c is
  bool v_done;   // of this turn
  // The current load.
  bool is_k;
  int stream, tile, b, head, keys, unit;
};
RV_DEVFN void pfx_feed_start(const PfxPiece (*tab)[RV_PFX_TABLE], const int (&count)[2], bool pair, PfxFeed &f) {
  if (f.s) {
    const PfxSide t = f.c;
    f.c = f.o;
    f.o = t;
  }
  f.s = f.c.at = f.o.at = 0;
  f.c.begun = f.o.begun = f.v_done = false;
  f.c.enter(tab[0], count[0]);
  f.o.left = 0;
  if (!pair) f.o.enter(tab[1], count[1]);
}
RV_DEVFN bool pfx_feed(const PfxPiece (*tab)[RV_PFX_TABLE], const int (&count)[2], bool pair, PfxFeed &f) {
  while (f.c.left || f.o.left) {
    f.is_k = f.v_done || !f.c.begun;
    f.stream = f.s;
    f.tile = f.c.tile;
    f.b = f.c.b;
    f.head = f.c.head;
    f.keys = f.c.keys;
    f.unit = f.c.unit;
    if (!f.is_k) {  // V of the unit whose K came last
      f.v_done = true;
      f.c.unit++;
      f.c.tile++;
      if (--f.c.left == 0) {
        f.c.at++;
        f.c.enter(tab[f.s], count[f.s]);
      }
      return true;
    }
    const bool has = f.c.left != 0;  // K of the next unit; then it is the other's turn
    f.c.begun = has;
    f.v_done = false;
    if (!pair) {
      const PfxSide t = f.c;
      f.c = f.o;
      f.o = t;
      f.s ^= 1;
    }
    if (has) return true;
  }
  return false;
}

RV_DEVFN float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// Two f32 operations an instruction.
RV_DEVFN float2 fma_f32x2(float2 a, float2 b, float2 c) {
  float2 d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;"
      : "=l"(*(unsigned long long *)&d)
      : "l"(*(unsigned long long *)&a), "l"(*(unsigned long long *)&b), "l"(*(unsigned long long *)&c));
  return d;
}
RV_DEVFN float2 add_f32x2(float2 a, float2 b) {
  float2 d;
  asm("add.rn.f32x2 %0, %1, %2;"
      : "=l"(*(unsigned long long *)&d)
      : "l"(*(unsigned long long *)&a), "l"(*(unsigned long long *)&b));
  return d;
}
// Consecutive 32-bit columns of this thread's tensor-memory lane, loaded when
// it returns (one statement, so no use can be moved before the wait).
RV_DEVFN void tc_ld_wait(uint32_t taddr, uint32_t (&v)[64]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x64.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
      "%15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32, %33, %34, %35, "
      "%36, %37, %38, %39, %40, %41, %42, %43, %44, %45, %46, %47, %48, %49, %50, %51, %52, %53, %54, %55, %56, "
      "%57, %58, %59, %60, %61, %62, %63}, [%64];\n"
      " tcgen05.wait::ld.sync.aligned;"
      : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]),
        "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]), "=r"(v[16]),
        "=r"(v[17]), "=r"(v[18]), "=r"(v[19]), "=r"(v[20]), "=r"(v[21]), "=r"(v[22]), "=r"(v[23]), "=r"(v[24]),
        "=r"(v[25]), "=r"(v[26]), "=r"(v[27]), "=r"(v[28]), "=r"(v[29]), "=r"(v[30]), "=r"(v[31]), "=r"(v[32]),
        "=r"(v[33]), "=r"(v[34]), "=r"(v[35]), "=r"(v[36]), "=r"(v[37]), "=r"(v[38]), "=r"(v[39]), "=r"(v[40]),
        "=r"(v[41]), "=r"(v[42]), "=r"(v[43]), "=r"(v[44]), "=r"(v[45]), "=r"(v[46]), "=r"(v[47]), "=r"(v[48]),
        "=r"(v[49]), "=r"(v[50]), "=r"(v[51]), "=r"(v[52]), "=r"(v[53]), "=r"(v[54]), "=r"(v[55]), "=r"(v[56]),
        "=r"(v[57]), "=r"(v[58]), "=r"(v[59]), "=r"(v[60]), "=r"(v[61]), "=r"(v[62]), "=r"(v[63])
      : "r"(taddr)
      : "memory");
}
RV_DEVFN void tc_ld_wait(uint32_t taddr, uint32_t (&v)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
      "%15}, [%16];\n"
      " tcgen05.wait::ld.sync.aligned;"
      : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]),
        "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
      : "r"(taddr)
      : "memory");
}
RV_DEVFN void tc_st16(uint32_t taddr, const uint32_t *v) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, "
      "%13, %14, %15, %16};" ::"r"(taddr), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]),
      "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]),
      "r"(v[15])
               : "memory");
}
RV_DEVFN void tc_st32(uint32_t taddr, const uint32_t *v) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, "
      "%13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, "
      "%32};" ::"r"(taddr), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]),
      "r"(v[7]), "r"(v[8]), "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15]),
      "r"(v[16]), "r"(v[17]), "r"(v[18]), "r"(v[19]), "r"(v[20]), "r"(v[21]), "r"(v[22]), "r"(v[23]), "r"(v[24]),
      "r"(v[25]), "r"(v[26]), "r"(v[27]), "r"(v[28]), "r"(v[29]), "r"(v[30]), "r"(v[31])
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

// Query row r of a segment's row space: its sequence, token and head.
struct PfxRow {
  int b, i, h;
};
RV_DEVFN PfxRow pfx_row(const PfxWork &w, int G, bool suffix, int b, int kvh, int r) {
  PfxRow o;
  o.b = suffix ? b : w.by_row(r);
  const int x = suffix ? r : r - o.b * w.rows_s;
  o.i = w.by_g(x);
  o.h = kvh * G + x - o.i * G;
  return o;
}

// The query rows of a stream's tile into its A operand(s) (K-major, 128-byte
// swizzle, 64 values a half tile), by the stream's 128 threads: D / 8 threads a
// row, so a row's loads are contiguous, and 64 registers of loads a thread in
// flight.  f32 rows are divided by a power of two first (2^e, e in `up`; the
// largest value then lies in [1, 2)) and held as hi + lo.  neg: the queries
// change sign.
template <int D, typename T, int SR>
RV_DEVFN void pfx_load_q(const PrefixArgs &a, const PfxWork &w, const PfxPiece &p, int r0, int nr, bool neg, int tid,
                         uint8_t *hi, int8_t *up) {
  constexpr int LPR = D / 8, RP = RV_PFX_M / LPR;  // threads a row, rows a pass
  constexpr bool F32 = sizeof(T) == 4;
  constexpr int W4 = F32 ? 2 : 1, NB = 2;  // 16-byte words; rows a thread in flight
  uint8_t *lo = hi + SR * D * 2;
  const int c = tid % LPR, G = (int)(a.n_heads / a.n_kv);
  const auto at = [&](int row) {
    const PfxRow pr = pfx_row(w, G, p.head & 1, p.b, p.head >> 1, r0 + row);
    return (const T *)a.q + (size_t)pr.b * a.q_seq_stride + (size_t)pr.i * a.q_token_stride + (size_t)pr.h * D + 8 * c;
  };
  if (!F32 && w.q_aligned && !neg) {  // as they are: copied past the registers
#pragma unroll 1
    for (int row = tid / LPR; row < nr; row += RP)
      asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(
                       smem_addr(hi + (uint32_t)(c >> 3) * (SR * 128) + tc_sw_off(row, c & 7))),
                   "l"(at(row))
                   : "memory");
    asm volatile("cp.async.wait_all;" ::: "memory");
    return;
  }
  for (int b0 = 0; b0 < nr; b0 += NB * RP) {
    uint4 x[NB][W4];
#pragma unroll
    for (int k = 0; k < NB; k++) {
      const int row = b0 + k * RP + tid / LPR;
      if (row < nr) {
        const T *q = at(row);
        if (w.q_aligned) {
#pragma unroll
          for (int i = 0; i < W4; i++) x[k][i] = __ldg((const uint4 *)q + i);
        } else {
          __align__(16) T t[8];
#pragma unroll
          for (int j = 0; j < 8; j++) t[j] = q[j];
#pragma unroll
          for (int i = 0; i < W4; i++) x[k][i] = ((const uint4 *)t)[i];
        }
      }
    }
#pragma unroll
    for (int k = 0; k < NB; k++) {
      const int row = b0 + k * RP + tid / LPR;
      const uint32_t off = (uint32_t)(c >> 3) * (SR * 128) + tc_sw_off(row, c & 7);
      if constexpr (F32) {
        const float f[8] = {__uint_as_float(x[k][0].x), __uint_as_float(x[k][0].y), __uint_as_float(x[k][0].z),
                            __uint_as_float(x[k][0].w), __uint_as_float(x[k][1].x), __uint_as_float(x[k][1].y),
                            __uint_as_float(x[k][1].z), __uint_as_float(x[k][1].w)};
        float m = 0;
#pragma unroll
        for (int j = 0; j < 8; j++) m = fmaxf(m, fabsf(f[j]));
        if (row >= nr) m = 0;
#pragma unroll
        for (int o = LPR / 2; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(RV_FULL, m, o));
        // Both 2^e and 2^-e are normal floats.
        const int e = min(max((int)(__float_as_uint(m) >> 23) - 127, -126), 126);
        const float down = __uint_as_float((uint32_t)(127 - e) << 23), sg = neg ? -down : down;
        if (row >= nr) continue;
        if (c == 0) up[row] = (int8_t)e;
        uint32_t o[4], r[4];
#pragma unroll
        for (int j = 0; j < 4; j++) {
          const float x0 = f[2 * j] * sg, x1 = f[2 * j + 1] * sg;
          o[j] = pack_f16(x0, x1);
          const float2 h = __half22float2(*(const __half2 *)&o[j]);
          r[j] = pack_f16(x0 - h.x, x1 - h.y);
        }
        *(uint4 *)(hi + off) = make_uint4(o[0], o[1], o[2], o[3]);
        *(uint4 *)(lo + off) = make_uint4(r[0], r[1], r[2], r[3]);
      } else if (row < nr) {
        const uint4 v = x[k][0];
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

// One lane of a converged warp, known to the compiler as one: the operands of
// the products it issues are then uniform without a check per lane.
RV_DEVFN bool elect_one() {
  uint32_t p;
  asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}\n" : "=r"(p));
  return p != 0;
}
// The bounded wait of mbar_wait_bounded in few instructions: this kernel's
// roles are limited by the instruction cache.
RV_DEVFN bool pfx_wait1(uint64_t *bar, uint32_t parity) {
  long long t0 = 0;
  for (uint32_t i = 1; !mbar_try_wait(bar, parity); i++) {
    if (i & 31) continue;
    const long long now = clock64();
    if (i == 32) t0 = now;
    if (now - t0 > RV_WAIT_CYCLES) {
      rv_dev_fail(RV_ERR_TIMEOUT);
      return false;
    }
  }
  return true;
}
// The same by a whole warp.
RV_DEVFN bool pfx_wait(uint64_t *bar, uint32_t parity) { return __all_sync(RV_FULL, pfx_wait1(bar, parity)); }
// Whether a role has given up, asked by a whole warp: its lanes leave together.
RV_DEVFN bool pfx_failed(const volatile int *fail) { return __any_sync(RV_FULL, *fail); }

template <int D, typename T, bool Q8>
__global__ void __launch_bounds__(RV_PFX_THREADS, 1)
    k_prefix_tc(PrefixArgs a, PfxWork w, const __grid_constant__ CUtensorMap map_pk,
                const __grid_constant__ CUtensorMap map_pv, const __grid_constant__ CUtensorMap map_sk,
                const __grid_constant__ CUtensorMap map_sv) {
  using C = PfxCfg<D, T, Q8>;
  constexpr bool PRECISE = C::PRECISE;
  constexpr int R = C::R, TILE = C::TILE, SLOTS = RV_PFX_SCALE_SLOTS;
  extern __shared__ __align__(1024) uint8_t sm[];  // the operand tiles are whole swizzle atoms
  uint8_t *ring = sm + C::ring;
  float *s_scale = (float *)(sm + C::scales);  // [stream][slot][RV_PFX_SCALE]
  PfxPiece(*tab)[RV_PFX_TABLE] = (PfxPiece(*)[RV_PFX_TABLE])(sm + C::table);
  int8_t *s_up = (int8_t *)(sm + C::ups);  // [stream][piece & 1][SR] exponents of f32 query rows
  uint64_t *bars = (uint64_t *)(sm + C::bars);
  uint64_t *kv_full = bars, *kv_empty = bars + R, *s_full = bars + 2 * R, *p_ready = s_full + 2, *o_full = p_ready + 2,
           *q_ready = o_full + 2, *sc_full = q_ready + 2, *drained = sc_full + 2 * SLOTS;
  int *s_scan = (int *)(bars + C::NBARS);  // pieces in the streams' tables
  uint32_t *s_tmem = (uint32_t *)(s_scan + 2);
  volatile int *s_fail = s_scan + 3, *s_bad = s_scan + 4;  // s_bad: [stream][piece & 1]
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  pdl_trigger();
  if (smem_addr(sm) & 1023) {
    rv_dev_fail(RV_ERR_CUDA);
    return;
  }
  if (threadIdx.x == 32) {
    for (int i = 0; i < R; i++) {
      mbar_init(&kv_full[i], Q8 ? RV_PFX_CONV / 32 : 1);
      mbar_init(&kv_empty[i], 1);
    }
    for (int i = 0; i < 2; i++) {
      mbar_init(&s_full[i], 1);
      mbar_init(&p_ready[i], 4);
      mbar_init(&o_full[i], 1);
      mbar_init(&q_ready[i], 4);
    }
    if (Q8)
      for (int i = 0; i < 2 * SLOTS; i++) mbar_init(&sc_full[i], RV_PFX_CONV / 32);
    mbar_init(drained, 1);
    *s_fail = 0;
  }
  if (warp == 0) {
    tc_alloc(s_tmem, 512);
    tc_relinquish();
  }
  // Counters that run on over the plans (each role uses its own).
  int n = 0, np[2] = {0, 0}, nq[2] = {0, 0}, unit = 0, piece = 0, run = 0;
  bool ok = true;
  PfxFeed feed{};
  for (int base = 0;; base += RV_PFX_TABLE) {
  // ------------------------------------------------ the next pieces
  // (Planned from the lengths each time, so that nothing of it stays in
  // registers while the roles run.)  Every warp adds up the lengths for itself;
  // warps 2 and 3 write the streams' pieces, a sequence a lane.
  bool pair;
  {
    int all = 0, fall = 0;
    for (uint32_t b = lane; b < ((a.n_seqs + 31) & ~31u); b += 32) {
      const int t = b < a.n_seqs ? pfx_tiles(prefix_suffix_len(a, b)) : 0;
      all += t;
      fall += t != 0;
    }
    all = __reduce_add_sync(RV_FULL, all);
    fall = __reduce_add_sync(RV_FULL, fall);
    const PfxLine line = pfx_line(a, w, all, fall);
    pair = (int)blockIdx.x < line.gp;
    const int segs = (int)a.n_kv * w.nrt_s;
    const bool cums = blockIdx.x == 0 && base == 0 && warp == 1;
    if (cums || warp == 2 || warp == 3) {
      const int s = warp - 2, ov_p = pair ? 0 : RV_PFX_OV, len_p = w.tp + ov_p;
      const int seg_p = pair || line.solo_p ? (int)a.n_kv * w.nrt_p : 0;  // prefix segments on this CTA's line
      // Solo streams: first stream 0 of every CTA, then stream 1, so few units
      // spread over all SMs.
      PfxStretch k;
      k.v = pair ? (int)blockIdx.x : (int)blockIdx.x - line.gp + s * (w.grid - line.gp);
      const int end = pair ? line.wp : line.w, per = pair ? line.per_p : line.per;
      k.u = min(end, k.v * per);
      k.end = min(end, k.u + per);
      // The first and last segment of the stretch, counted along the line.
      const int lim = seg_p * len_p;
      int g0 = -1, g1 = -1;
      if (k.u < min(k.end, lim)) {
        g0 = k.u / len_p;
        g1 = (min(k.end, lim) - 1) / len_p;
      }
      PfxPiece p{};
      if (g0 >= 0 && g0 + base + lane <= g1) {
        const int g = g0 + base + lane, kvh = g / w.nrt_p;
        p.head = 2 * kvh;
        p.row0 = (g - kvh * w.nrt_p) * w.sr_p;
        p.keys = (int)a.prefix_len;
        p.part = (g + k.v) * (pair ? 2 : 1);
        pfx_cut(p, k, g * len_p, w.tp, ov_p);
      }
      if (!cums) tab[s][lane] = p;
      __syncwarp();
      if (cums || (!pair && k.end > lim && k.u < k.end)) {
        int x0 = line.solo_p, c0 = 0, f0 = 0;  // the place, tiles and filled sequences before the 32
        for (uint32_t b0 = 0; b0 < a.n_seqs && (cums || x0 < k.end); b0 += 32) {
          const int b = (int)b0 + lane, keys = b < (int)a.n_seqs ? prefix_suffix_len(a, (uint32_t)b) : 0;
          const int t = pfx_tiles(keys), len = t ? t + RV_PFX_OV : 0;
          int upto = t;
          for (int o = 1; o < 32; o <<= 1) {
            const int v = __shfl_up_sync(RV_FULL, upto, o);
            if (lane >= o) upto += v;
          }
          const uint32_t some = __ballot_sync(RV_FULL, t != 0);
          const int c = c0 + upto - t, f = f0 + __popc(some & ((1u << lane) - 1));
          const int x = line.solo_p + (c + f * RV_PFX_OV) * segs;  // where the sequence's segments begin
          if (cums) {
            if (b < (int)a.n_seqs) {
              w.cum[b] = c;
              w.cum[a.n_seqs + 1 + b] = f;
            }
          } else {
            const int lo = max(k.u, x), hi = min(k.end, x + len * segs);  // its places on the stretch
            const uint32_t hit = __ballot_sync(RV_FULL, lo < hi);
            if (hit) {
              const int l0 = lo < hi ? (lo - x) / len : 0, l1 = lo < hi ? (hi - 1 - x) / len : -1, g = seg_p + b * segs;
              if (g0 < 0) g0 = __shfl_sync(RV_FULL, g + l0, __ffs(hit) - 1);
              g1 = __shfl_sync(RV_FULL, g + l1, 31 - __clz(hit));
              for (int i = max(l0, g0 + base - g); i <= min(l1, g0 + base + RV_PFX_TABLE - 1 - g); i++) {
                const int kvh = i / w.nrt_s;
                p.b = b;
                p.head = 2 * kvh + 1;
                p.row0 = (i - kvh * w.nrt_s) * w.sr_s;
                p.keys = keys;
                p.part = b * segs + i + k.v;
                pfx_cut(p, k, x + i * len, t, RV_PFX_OV);
                tab[s][g + i - g0 - base] = p;
              }
            }
          }
          c0 = __shfl_sync(RV_FULL, c + t, 31);
          f0 += __popc(some);
          x0 = line.solo_p + (c0 + f0 * RV_PFX_OV) * segs;
        }
        if (cums && lane == 0) {
          w.cum[a.n_seqs] = c0;
          w.cum[2 * a.n_seqs + 1] = f0;
        }
      }
      if (!cums && lane == 0) s_scan[s] = g0 < 0 ? 0 : min(max(g1 - g0 + 1 - base, 0), RV_PFX_TABLE);
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const int count[2] = {s_scan[0], s_scan[1]};
  if (count[0] + count[1] == 0) break;
  const uint32_t tmem = *s_tmem;
  if (warp < 4) {
    if (!Q8 && warp == 0) {
    if (elect_one()) {
      // ---------------------------------------------------------- loads
      PfxFeed &f = feed;
      pfx_feed_start(tab, count, pair, f);
      for (; ok && !*s_fail && pfx_feed(tab, count, pair, f); n++) {
        const int slot = n % R;
        if (!mbar_wait_bounded(&kv_empty[slot], ((n / R) & 1) ^ 1)) {
          ok = false;
          break;
        }
        mbar_arrive_expect_tx(&kv_full[slot], (uint32_t)TILE);
        const bool suffix = f.head & 1;
        const CUtensorMap *m = suffix ? (f.is_k ? &map_sk : &map_sv) : (f.is_k ? &map_pk : &map_pv);
#pragma unroll
        for (int h = 0; h < D / 64; h++)
          tma_load_4d(ring + (size_t)slot * TILE + h * (RV_PFX_N * 128), m, 64 * h, f.head >> 1, f.tile * RV_PFX_N, f.b,
                      &kv_full[slot]);
      }
      if (!ok) *s_fail = 1;
    }
    __syncwarp();
    n = __reduce_max_sync(RV_FULL, n);  // another lane may be elected in the next plan
    } else if (warp == 1) {
      // ----------------------------------------------------- MMA issue
      const uint32_t hi_sw = (1024u >> 4) | (1u << 14) | (2u << 29);
      const uint32_t lbo_k = 1u << 16, lbo_v = (uint32_t)(RV_PFX_N * 128 >> 4) << 16;
      const uint32_t q_lo = smem_addr(sm) >> 4, ring_lo = smem_addr(ring) >> 4;
      const uint32_t idesc_s = tc_idesc(RV_PFX_N), idesc_o = tc_idesc(D) | (1u << 16);  // B of P V: keys down the rows
      auto mk = [](uint32_t lo, uint32_t hi) { return ((uint64_t)hi << 32) | lo; };
      // A stream's place: table entry, its units (0: none left), the next one to
      // multiply (-1: S of the piece's first is still to come), phases passed.
      struct Place {
        int at, len, j, np, nq;
      } c = {0, 0, -1, np[0], nq[0]}, o = {0, 0, -1, np[1], nq[1]};
      const auto wait_full = [&](int i) { return pfx_wait(&kv_full[i % R], (i / R) & 1); };
      int nk = 0, nv = 0;
      pfx_entry(tab[0], count[0], c.at, c.len);
      if (pair) o.len = c.len, o.at = c.at;
      else pfx_entry(tab[1], count[1], o.at, o.len);
      // The streams in turn: O += P V of a unit and S = Q K^T of the stream's
      // next one.  Paired streams share tiles: stream 0 takes them from the ring,
      // stream 1 gives them back.
      int s = 0;
#pragma unroll 1
      for (; ok && (c.len || o.len) && !pfx_failed(s_fail); s ^= 1) {
        if (c.len) {
          const bool take = !(pair && s), give = !pair || s;
          const PfxPiece *p = &tab[pair ? 0 : s][c.at];
          bool next = c.j + 1 < c.len;  // an S is to come: of this piece, or
          if (c.j >= 0) {
            const int valid = min(RV_PFX_N, p->keys - (p->tile0 + c.j) * RV_PFX_N), steps = (valid + 15) >> 4;
            if (take) {
              nv = n++;
              ok = wait_full(nv);
              if (!Q8 && (p->head & 1) && (valid & 15)) {
                // Rows past the sequence's end hold whatever the cache held:
                // zero those the last K step reads (0 * NaN is not 0).
                for (int i = lane; i < (16 * steps - valid) * (D / 8); i += 32) {
                  const int r = valid + i / (D / 8), ch = i % (D / 8);
                  *(uint4 *)(ring + (size_t)(nv % R) * TILE + (ch >> 3) * (RV_PFX_N * 128) + tc_sw_off(r, ch & 7)) =
                      make_uint4(0, 0, 0, 0);
                }
                fence_proxy_async();
                __syncwarp();
              }
              if (!Q8 && a.n_q > 1 && (p->head & 1)) {
                // Values among the sequence's newest tokens are hidden from some
                // of its queries, and 0 * NaN is not 0: a row that is not finite
                // is taken out here, and its first key kept for the queries that
                // see it, whose outputs become NaN.
                // (The piece before may still be read: two places in turn.)
                volatile int *const mark = s_bad + 2 * s + ((c.nq - 1) & 1);
                int bad = c.j == 0 ? INT_MAX : *mark;
                const int hidden = p->keys - (int)a.n_q + 1 - (p->tile0 + c.j) * RV_PFX_N;
                for (int r = max(hidden, 0); r < valid; r++) {
                  uint4 *x = (uint4 *)(ring + (size_t)(nv % R) * TILE + (lane >> 3) * (RV_PFX_N * 128) +
                                       tc_sw_off(r, lane & 7));
                  uint4 v = make_uint4(0, 0, 0, 0);
                  if (lane < D / 8) v = *x;
                  const auto odd = [](uint32_t u) {
                    return (u & 0x7C00u) == 0x7C00u || (u & 0x7C000000u) == 0x7C000000u;
                  };
                  if (__any_sync(RV_FULL, odd(v.x) || odd(v.y) || odd(v.z) || odd(v.w))) {
                    if (lane < D / 8) *x = make_uint4(0, 0, 0, 0);
                    bad = min(bad, (p->tile0 + c.j) * RV_PFX_N + r);
                  }
                }
                if (lane == 0) *mark = bad;
                fence_proxy_async();
                __syncwarp();
              }
              if (next) {
                nk = n++;
                ok = ok && wait_full(nk);
              }
            }
            ok = ok && pfx_wait(&p_ready[s], c.np & 1);
            c.np++;
            if (!ok) break;
            tc_fence_after();
            if (elect_one()) {
              const uint32_t vb = ring_lo + (uint32_t)(nv % R * (TILE >> 4)), p0 = tmem + 128 * s, d = p0 + RV_PFX_O;
              // The accumulator truncates, by its own size: the low terms go
              // first, while it is small (here and for S; the error over 128
              // keys 7.4e-7 -> 3.7e-7 of the norm, plain f32 sums 3.8e-7).
#pragma unroll 1
              for (int lo = PRECISE; lo >= 0; lo--) {
#pragma unroll
                for (int kk = 0; kk < 8; kk++) {
                  if (kk < steps) {
                    const uint32_t pa = p0 + 32 * (kk >> 1) + 8 * (kk & 1) + 16 * lo;
                    const uint64_t bd = mk(lbo_v | (vb + (uint32_t)kk * (2048 >> 4)), hi_sw);
                    tc_mma_f16_ta(d, pa, bd, idesc_o, kk != 0 || (C::RUNS ? c.j % RV_PFX_RUN : c.j) != 0 || lo != PRECISE);
                  }
                }
              }
              if (!next || (C::RUNS && (c.j + 1) % RV_PFX_RUN == 0)) tc_commit(&o_full[s]);
              if (give) tc_commit(&kv_empty[nv % R]);
            }
            __syncwarp();
          }
          c.j++;
          if (c.j == c.len) {  // of the next piece
            c.at++;
            pfx_entry(tab[pair ? 0 : s], count[pair ? 0 : s], c.at, c.len);
            c.j = 0;
            next = c.len != 0;
          }
          if (next) {
            if (c.j == 0) {
              ok = pfx_wait(&q_ready[s], c.nq & 1);
              c.nq++;
              if (take) {
                nk = n++;
                ok = ok && wait_full(nk);
              }
              if (!ok) break;
              tc_fence_after();
            }
            if (elect_one()) {
              const uint32_t qa = q_lo + s * (C::QS >> 4), kb = ring_lo + (uint32_t)(nk % R * (TILE >> 4)),
                             d = tmem + 128 * s;
#pragma unroll 1
              for (int lo = PRECISE; lo >= 0; lo--) {
#pragma unroll
                for (int kk = 0; kk < D / 16; kk++) {
                  const uint32_t q = qa + (uint32_t)lo * (C::QT >> 4),
                                 oq = (uint32_t)(kk >> 2) * (C::SR * 128 >> 4) + 2 * (kk & 3),
                                 okk = (uint32_t)(kk >> 2) * (RV_PFX_N * 128 >> 4) + 2 * (kk & 3);
                  tc_mma_f16(d, mk(lbo_k | (q + oq), hi_sw), mk(lbo_k | (kb + okk), hi_sw), idesc_s,
                             kk != 0 || lo != PRECISE);
                }
              }
              tc_commit(&s_full[s]);
              if (give) tc_commit(&kv_empty[nk % R]);
            }
            __syncwarp();
          }
        }
        const Place t = c;
        c = o;
        o = t;
      }
      if (s) {  // an odd number of turns: c is stream 1's
        const Place t = c;
        c = o;
        o = t;
      }
      np[0] = c.np, nq[0] = c.nq, np[1] = o.np, nq[1] = o.nq;
      if (!ok) *s_fail = 1;
    } else if (Q8) {
      // ---------------------------------- 8-bit rows into f16 operands
      // 16 levels a load, D / 16 loads a token.  The next tile's levels are
      // copied to shared memory while this one's are converted; every thread
      // converts what it copied.
      constexpr int TPT = D / 16, LOADS = RV_PFX_N * TPT, IT = (LOADS + RV_PFX_CONV - 1) / RV_PFX_CONV;
      const int ct = (warp == 0 ? 0 : 32 * (warp - 1)) + lane;
      PfxFeed &f = feed;
      pfx_feed_start(tab, count, pair, f);
      // A tile on its way: its scales in registers.
      struct Load {
        float ks[2], vs[2];
        int at;  // scale slot of a K tile, -1: a V tile
      } cur, nxt;
      uint8_t *raw = sm + C::raw;
      const auto fetch = [&](Load &o, int half) {
        if (!pfx_feed(tab, count, pair, f)) return false;
        const bool suffix = f.head & 1;
        const int kvh = f.head >> 1, valid = min(RV_PFX_N, f.keys - f.tile * RV_PFX_N);
        const size_t first = (size_t)f.b * a.cap * suffix + (size_t)f.tile * RV_PFX_N;
        const int8_t *src = (const int8_t *)(f.is_k ? (suffix ? a.sk : a.pk) : (suffix ? a.sv : a.pv)) +
                            (first * a.n_kv + kvh) * D;
        const size_t pitch = (size_t)a.n_kv * D;
#pragma unroll
        for (int j = 0; j < IT; j++) {
          const int id = j * RV_PFX_CONV + ct, tok = id / TPT;
          if (tok < RV_PFX_N)  // tokens past the end read as zeros
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_addr(raw + half + 16 * id)),
                         "l"(tok < valid ? src + tok * pitch + (id % TPT) * 16 : src), "r"(tok < valid ? 16 : 0)
                         : "memory");
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
        o.at = f.is_k ? f.stream * SLOTS + f.unit % SLOTS : -1;
#pragma unroll
        for (int j = 0; j < 2; j++) {
          o.ks[j] = o.vs[j] = 0;
          if (f.is_k && ct + j * RV_PFX_CONV < valid) {
            const size_t at = (first + ct + j * RV_PFX_CONV) * a.n_kv + kvh;
            o.ks[j] = (suffix ? a.sks : a.pks)[at];
            o.vs[j] = (suffix ? a.svs : a.pvs)[at];
          }
        }
        return true;
      };
      int half = 0;
      bool any = fetch(cur, 0);
      for (; ok && any && !pfx_failed(s_fail); n++) {
        any = fetch(nxt, half ^ RV_PFX_N * D);  // in flight while this tile is converted
        if (any) asm volatile("cp.async.wait_group 1;" ::: "memory");
        else asm volatile("cp.async.wait_group 0;" ::: "memory");
        const int slot = n % R;
        ok = pfx_wait(&kv_empty[slot], ((n / R) & 1) ^ 1);
        if (!ok) break;
        if (cur.at >= 0) {
          float *sc = s_scale + cur.at * RV_PFX_SCALE;
          const float scale = PRECISE ? fabsf(a.scale_log2) / prefix_pow2(a.scale_log2) : fabsf(a.scale_log2);
#pragma unroll
          for (int j = 0; j < 2; j++) {
            const int tok = ct + j * RV_PFX_CONV;
            // A value scale that is not finite makes the token's weight NaN
            // through its key scale; as a factor it is 0, for the rows that do
            // not see the token.  Exponents from -80 up: the weights of tokens
            // without a value then stay below 2^95.
            const float size = fabsf(cur.vs[j]);
            const bool fine = size < INFINITY;
            if (tok < RV_PFX_N) {
              sc[tok] = fine ? cur.ks[j] * scale : __uint_as_float(0x7FC00000u);
              sc[RV_PFX_N + tok] = fine ? cur.vs[j] : 0.0f;
              sc[2 * RV_PFX_N + tok] = (float)max((int)(__float_as_uint(size) >> 23) - 126, -80);
            }
          }
          __syncwarp();
          if (lane == 0) mbar_arrive(&sc_full[cur.at]);
        }
        uint8_t *dst = ring + (size_t)slot * TILE;
#pragma unroll
        for (int j = 0; j < IT; j++) {
          const int id = j * RV_PFX_CONV + ct, tok = id / TPT, ch = (id % TPT) * 2;
          if (tok < RV_PFX_N) {
            const uint4 x = *(const uint4 *)(raw + half + 16 * id);
            uint32_t o[8];
            pfx_levels(x.x, o[0], o[1]);
            pfx_levels(x.y, o[2], o[3]);
            pfx_levels(x.z, o[4], o[5]);
            pfx_levels(x.w, o[6], o[7]);
            uint8_t *d = dst + (ch >> 3) * (RV_PFX_N * 128);
            *(uint4 *)(d + tc_sw_off(tok, ch & 7)) = make_uint4(o[0], o[1], o[2], o[3]);
            *(uint4 *)(d + tc_sw_off(tok, (ch & 7) + 1)) = make_uint4(o[4], o[5], o[6], o[7]);
          }
        }
        fence_proxy_async();
        __syncwarp();
        if (lane == 0) mbar_arrive(&kv_full[slot]);
        cur = nxt;
        half ^= RV_PFX_N * D;
      }
      asm volatile("cp.async.wait_all;" ::: "memory");
      if (!ok) *s_fail = 1;
    }
  } else {
    // --------------------------------------------------------- softmax
    const int s = (warp - 4) >> 2, quad = warp & 3, row = 32 * quad + lane;
    const uint32_t tl = tmem + ((uint32_t)(32 * quad) << 16), tS = tl + 128 * s, tO = tl + RV_PFX_O + 128 * s;
    const bool neg = a.scale_log2 < 0;  // the sign of the scale goes to the queries
    const float scale = fabsf(a.scale_log2);
    uint8_t *q_dst = sm + s * C::QS;
    const PfxPiece *mytab = tab[pair ? 0 : s];
    const int mycount = pair ? count[0] : s ? count[1] : count[0];
    // Queries of a piece into shared memory, for the products.
    auto give_q = [&](const PfxPiece &x, int which) {
      const int r0 = x.row0 + (pair ? RV_PFX_M * s : 0);
      const int rows = x.head & 1 ? w.rows_s : w.rows_p;
      pfx_load_q<D, T, C::SR>(a, w, x, r0, min(C::SR, rows - r0), neg, row, q_dst,
                              s_up + (2 * s + (which & 1)) * C::SR);
      fence_proxy_async();
      __syncwarp();
      if (lane == 0) mbar_arrive(&q_ready[s]);
    };
    int at = 0, left;
    pfx_entry(mytab, mycount, at, left);
    // What the run before leaves, written while this one's first scores are on
    // their way.
    int p_head = 0, p_part = -1, p_seen = 0;
    bool p_on = false, p_warp = false, p_add = false;
    float p_m = 0, p_l = 0, p_up = 0;
    int t = 0;  // the piece's next tile
    float m_ref = -INFINITY, m_part = -INFINITY, l = 0;  // m_part: the reference of what the part holds
#pragma unroll 1
    while (ok && !pfx_failed(s_fail)) {
      if (left && (!C::RUNS || t == 0)) give_q(mytab[at], piece);
      if (p_part >= 0) {
        const int rw = p_head & 1 ? w.rw_s : w.rw_p;
        const size_t part = (size_t)p_part + (pair ? s : 0);
        float4 *po = (p_head & 1 ? w.o_s : w.o_p) + part * (D / 4) * rw + row;
        ok = pfx_wait(&o_full[s], (run - 1) & 1);
        if (!ok) break;
        tc_fence_after();
        if (!Q8 && a.n_q > 1 && (p_head & 1) && p_seen > s_bad[2 * s + ((piece - 1) & 1)])
          p_l = __uint_as_float(0x7FC00000u);
        if (p_on) (p_head & 1 ? w.ml_s : w.ml_p)[part * rw + row] = make_float2(p_m, p_l);
        if (p_warp) {
#pragma unroll 1
          for (int ch = 0; ch < D / 16; ch++) {
            uint32_t v[16];
            tc_ld_wait(tO + 16 * ch, v);
            if (p_on) {
#pragma unroll
              for (int j = 0; j < 4; j++) {
                float4 x = make_float4(__uint_as_float(v[4 * j]), __uint_as_float(v[4 * j + 1]),
                                       __uint_as_float(v[4 * j + 2]), __uint_as_float(v[4 * j + 3]));
                if constexpr (C::RUNS) x = make_float4(x.x * p_up, x.y * p_up, x.z * p_up, x.w * p_up);
                float4 *const to = po + (4 * ch + j) * rw;
                if (C::RUNS && p_add)
                  asm volatile("red.relaxed.gpu.global.add.v4.f32 [%0], {%1, %2, %3, %4};" ::"l"(to), "f"(x.x),
                               "f"(x.y), "f"(x.z), "f"(x.w)
                               : "memory");
                else
                  *to = x;
              }
            }
          }
          tc_fence_before();
        }
      }
      if (!left) break;
      const PfxPiece p = mytab[at];
      const bool suffix = p.head & 1;
      const int r = p.row0 + (pair ? RV_PFX_M * s : 0) + row;  // this thread's query row
      const bool on = row < C::SR && r < (suffix ? w.rows_s : w.rows_p), warp_on = __any_sync(RV_FULL, on);
      int seen = on ? p.keys : 0;  // keys of the segment that this row sees
      if (suffix && on) seen = min(max(p.keys - (int)a.n_q + 1 + w.by_g(r), 0), p.keys);
      // Scores times c are in units of log2 (8-bit keys: their scales hold
      // the attention scale, for f32 queries but its power of two).  At least
      // 2^-126, so that -infinity stays one.
      float c = !Q8 ? scale : PRECISE ? prefix_pow2(scale) : 1.0f;
      if constexpr (PRECISE) {
        // The exponents of the stream's four warps: each arrives with its rows'.
        // A named barrier here would wait for ever on a warp that gave up.
        ok = pfx_wait(&q_ready[s], piece & 1);
        if (!ok) break;
        if (on) c *= __uint_as_float((uint32_t)(s_up[(2 * s + (piece & 1)) * C::SR + row] + 127) << 23);
      }
      c = fmaxf(c, 0x1p-126f);
      const int t0 = C::RUNS ? t : 0, end = C::RUNS ? min(p.n, t0 + RV_PFX_RUN) : p.n;  // of the run
      if (t0 == 0) m_ref = m_part = -INFINITY, l = 0;
      for (t = t0; t < end; t++, unit++) {
        const int tile = p.tile0 + t, valid = min(RV_PFX_N, p.keys - tile * RV_PFX_N);
        const int lim = min(max(seen - tile * RV_PFX_N, 0), RV_PFX_N);
        const int slot = (pair ? 0 : s) * SLOTS + unit % SLOTS;
        const float *sc = s_scale + slot * RV_PFX_SCALE;
        if (Q8) ok = pfx_wait(&sc_full[slot], (uint32_t)(unit / SLOTS) & 1);
        ok = ok && pfx_wait(&s_full[s], unit & 1);
        if (!ok) break;
        tc_fence_after();
        if (warp_on) {
          const int halves = valid > 64 ? 2 : 1;
          const bool full = __all_sync(RV_FULL, lim == RV_PFX_N || !on);
#pragma unroll 1
          for (int h = 0; h < halves; h++) {
            uint32_t v[64];
            tc_ld_wait(tS + 64 * h, v);
            float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
            if (!full) {
#pragma unroll
              for (int j = 0; j < 64; j++) v[j] = 64 * h + j < lim ? v[j] : 0xFF800000u;
            }
            if constexpr (Q8) {
              const float2 c2 = make_float2(c, c), zero = make_float2(0, 0);
#pragma unroll
              for (int j = 0; j < 64; j += 4) {
                const float4 k4 = *(const float4 *)(sc + 64 * h + j);
                const float4 e4 = *(const float4 *)(sc + 2 * RV_PFX_N + 64 * h + j);
                float2 x0 = make_float2(__uint_as_float(v[j]), __uint_as_float(v[j + 1]));
                float2 x1 = make_float2(__uint_as_float(v[j + 2]), __uint_as_float(v[j + 3]));
                if constexpr (PRECISE) {  // by a power of two: exact
                  x0 = fma_f32x2(x0, c2, zero);
                  x1 = fma_f32x2(x1, c2, zero);
                }
                // f32 queries use t for the maximum alone: the exponent comes with it.
                const float2 t0 = fma_f32x2(x0, make_float2(k4.x, k4.y), PRECISE ? make_float2(e4.x, e4.y) : zero),
                             t1 = fma_f32x2(x1, make_float2(k4.z, k4.w), PRECISE ? make_float2(e4.z, e4.w) : zero);
                const float t[4] = {t0.x, t0.y, t1.x, t1.y}, x[4] = {x0.x, x0.y, x1.x, x1.y}, e[4] = {e4.x, e4.y, e4.z, e4.w};
#pragma unroll
                for (int i = 0; i < 4; i++) {
                  // Hidden scores stay -infinity whatever the token's scale is.
                  const float u = full || x[i] != -INFINITY ? t[i] : -INFINITY;
                  mx[i] = fmaxf(mx[i], PRECISE ? u : u + e[i]);
                  v[j + i] = __float_as_uint(PRECISE ? x[i] : u);
                }
              }
            } else {
#pragma unroll
              for (int j = 0; j < 64; j++) mx[j & 3] = fmaxf(mx[j & 3], __uint_as_float(v[j]));
            }
            float top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
            if constexpr (!Q8) top *= c;
            top = on ? ceilf(top) : -INFINITY;
            if (t == 0 && h == 0) {
              m_ref = top;
            } else if (const bool move = top > m_ref + RV_PFX_LAG; __any_sync(RV_FULL, move)) {
              // A new reference, a whole number of powers of two away: O and P
              // change their exponents.  Every product issued so far is done
              // (S came after them).
              const int d = move && m_ref != -INFINITY ? (int)fmaxf(m_ref - top, -200.0f) : 0;
              const bool none = move && (m_ref == -INFINITY || d < -126);
              const float f = none ? 0.0f : __uint_as_float((uint32_t)(127 + d) << 23);
              if (move) m_ref = top;
              l *= f;
              const __half2 f2 = __float2half2_rn(f);
#pragma unroll 1
              for (int ch = t > t0 ? 0 : D / 16; ch < D / 16 + 4 * h; ch++) {
                uint32_t o[16];
                const bool is_p = ch >= D / 16;  // P of the tile's first half
                const uint32_t at = is_p ? tS + 16 * (ch - D / 16) : tO + 16 * ch;
                tc_ld_wait(at, o);
#pragma unroll
                for (int j = 0; j < 16; j++) {
                  const __half2 x = __hmul2(*(const __half2 *)&o[j], f2);
                  o[j] = is_p ? *(const uint32_t *)&x : __float_as_uint(__uint_as_float(o[j]) * f);
                }
                tc_st16(at, o);
              }
            }
            const float m_use = m_ref == -INFINITY ? 0.0f : m_ref - RV_PFX_LIFT;
            const float2 c2 = make_float2(c, c), m2 = make_float2(-m_use, -m_use);
            float2 l2[2] = {make_float2(0, 0), make_float2(0, 0)};
#pragma unroll
            for (int ch = 0; ch < 2; ch++) {
              uint32_t o[32];
#pragma unroll
              for (int j = 0; j < 16; j++) {
                const int e = 32 * ch + 2 * j;
                float2 x = make_float2(__uint_as_float(v[e]), __uint_as_float(v[e + 1]));
                if constexpr (PRECISE && Q8) {
                  // One rounding from the score to the exponent; a hidden
                  // token's scale may be anything.
                  const float2 k = *(const float2 *)(sc + 64 * h + e), y = fma_f32x2(x, k, m2);
                  x = make_float2(x.x == -INFINITY ? x.x : y.x, x.y == -INFINITY ? x.y : y.y);
                } else {
                  x = Q8 ? add_f32x2(x, m2) : fma_f32x2(x, c2, m2);
                }
                x.x = ex2(x.x);
                x.y = ex2(x.y);
                l2[j & 1] = add_f32x2(l2[j & 1], x);
                if constexpr (Q8)
                  x = fma_f32x2(x, *(const float2 *)(sc + RV_PFX_N + 64 * h + e), make_float2(0, 0));
                o[j] = pack_f16(x.x, x.y);
                if constexpr (PRECISE) {
                  const float2 f = __half22float2(*(const __half2 *)&o[j]);
                  o[16 + j] = pack_f16(x.x - f.x, x.y - f.y);
                }
              }
              // P takes the columns its scores came from: 16 of hi, then lo.
              if constexpr (PRECISE) tc_st32(tS + 64 * h + 32 * ch, o);
              else tc_st16(tS + 64 * h + 32 * ch, o);
            }
            l += (l2[0].x + l2[1].x) + (l2[0].y + l2[1].y);
          }
          tc_wait_st();
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_ready[s]);
      }
      if (!ok) break;
      if constexpr (C::RUNS) {
        // The run's O goes to the part, times a power of two where the reference
        // has moved since.  Past these limits what the part holds counts for
        // nothing (below them O and l stay in range).
        const float d = m_ref - m_part;
        p_add = t0 > 0 && d <= (Q8 ? 48.0f : 80.0f);
        p_up = p_add ? __uint_as_float((uint32_t)(127 + (int)d) << 23) : 1.0f;
      }
      if (!p_add) m_part = m_ref;
      p_head = p.head;
      p_part = p.part;
      p_on = on;
      p_seen = seen;
      p_warp = warp_on;
      p_m = m_part == -INFINITY ? -INFINITY : m_part - RV_PFX_LIFT;
      p_l = C::RUNS ? l * p_up : l;
      run++;
      if (C::RUNS && t < p.n) continue;
      // The products have read this piece's queries (S came after them), so the
      // next piece's may take their place under the last P V.
      t = 0;
      at++;
      pfx_entry(mytab, mycount, at, left);
      piece++;
    }
    if (!ok) *s_fail = 1;
  }
  tc_fence_before();
  __syncthreads();  // the table may be written again
  if (*s_fail) {
    // A role gave up, perhaps after others had ended theirs: copies and products
    // in flight end before the CTA does and tensor memory is freed.
    if (!Q8 && warp == 0 && elect_one())
      for (int i = max(0, n - R); i < n; i++) mbar_wait_bounded(&kv_full[i % R], (i / R) & 1);
    if (warp == 1 && elect_one()) {
      tc_commit(drained);
      mbar_wait_bounded(drained, 0);
    }
    tc_fence_before();
    __syncthreads();
    break;
  }
  }
  if (warp == 0) {
    tc_fence_after();
    tc_dealloc(*s_tmem, 512);
  }
}

// The parts of each query row added up: out = sum 2^(m_p - M) O_p / sum
// 2^(m_p - M) l_p.  grid = (8-row groups of a kv head's rows, kv heads); a warp
// holds eight rows times four part lanes (each takes every fourth part) and
// two groups of four values, so a load is 128 contiguous bytes a part.  Bound
// by the latency of few loads a lane: 3 to 11 us of a call.
#define RV_PFX_JOIN_ROWS 8
template <int D, typename T>
__global__ void __launch_bounds__(D * 4) k_prefix_join(PrefixArgs a, PfxWork w) {
  const int lane = threadIdx.x & 31, d4 = threadIdx.x >> 5, kvh = blockIdx.y, pl = lane >> 3;
  const int r = min((int)blockIdx.x * RV_PFX_JOIN_ROWS + (lane & 7), w.rows_p - 1);
  const bool on = (int)blockIdx.x * RV_PFX_JOIN_ROWS + (lane & 7) < w.rows_p;
  const PfxRow pr = pfx_row(w, (int)(a.n_heads / a.n_kv), false, 0, kvh, r);
  const int segs = (int)a.n_kv * w.nrt_s;
  pdl_wait();  // cum and the parts are k_prefix_tc's
  const int *fcum = w.cum + a.n_seqs + 1;
  const PfxLine line = pfx_line(a, w, w.cum[a.n_seqs], fcum[a.n_seqs]);
  // The row's parts: those of its prefix segment, then of its sequence's
  // suffix segment; each a run with a constant step.
  const float2 *ml[2];
  const float4 *po[2];
  int n[2], step[2], rw[2];
#pragma unroll
  for (int s = 0; s < 2; s++) {
    const bool pair = !s && w.pair;
    const int sr = s ? w.sr_s : w.sr_p, x = s ? r - pr.b * w.rows_s : r, in = x % sr;
    const int c0 = s ? w.cum[pr.b] : 0, tiles = s ? w.cum[pr.b + 1] - c0 : w.tp, ov = pair ? 0 : RV_PFX_OV;
    const int local = kvh * (s ? w.nrt_s : w.nrt_p) + x / sr, seg = s ? pr.b * segs + local : local;
    // The places of the segment's tiles on its line.
    const int u0 = (s ? line.solo_p + (c0 + fcum[pr.b] * RV_PFX_OV) * segs : 0) + local * (tiles + ov) + ov;
    const int per = pair ? line.per_p : line.per;
    const int first = u0 / per, last = (u0 + tiles - 1) / per;
    const size_t part = (size_t)(seg + first) * (pair ? 2 : 1) + (pair ? in / RV_PFX_M : 0);
    rw[s] = s ? w.rw_s : w.rw_p;
    step[s] = pair ? 2 : 1;
    n[s] = tiles == 0 ? 0 : last - first + 1;
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
#pragma unroll 2
    for (int i = pl; i < n[s]; i += 4) {
      const float2 x = ml[s][(size_t)i * step[s] * rw[s]];
      const float4 *q = po[s] + (size_t)i * step[s] * (D / 4) * rw[s];
      const float4 v[2] = {q[0], q[(D / 8) * rw[s]]};
      // -infinity: the row saw none of the part's keys, whose O may be anything --
      // unless its sum is NaN: then every score it saw was (maxima pass NaN over).
      const bool sees = x.x != -INFINITY || isnan(x.y);
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
