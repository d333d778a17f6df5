// rv_kv.cuh -- KV cache rows in f16 or in 8 bits: rv_kv_append, rv_kv_read.
//
// A row is the head_dim values of one (token, kv head).  The 8-bit format
// holds one f32 scale a row and int8 levels:
//   amax = max |x_i|,  scale = amax * (1/127),  level_i = rint(x_i * ((1/amax) * 127))
// every operation in f32 with one rounding each, ties to even; the value read
// back is level_i * scale.  A row whose amax is below 2^-50 is stored as zero
// (scale 0, levels 0), so a stored scale is 0 or at least 2^-57 and its
// logarithm and reciprocal are ordinary floats.  A row that holds an infinity
// or a NaN reads back as NaN everywhere (its scale is not finite), it never
// turns into finite values.  One scale for the whole row, not one per 32
// values, lets the attention products run on the levels alone: a key's scale
// multiplies its score and a value's scale its probability, both in f32.
//
// Both kernels move each byte once and are bound by that.  Eight values a
// thread (one 16-byte load of f16, two of f32) and 16 lanes a row of 128, so
// the row's maximum is four shuffles; two rows a thread in flight (one: 69 us).
// Written and read back: 32,768 tokens of 4 heads x 128 in f32, 8-bit
// cache, 65.6 us for 338 MB (5.1 TB/s; 0.80 of a plain copy's rate); 16 rows 4.0 us,
// which is two launches.
#pragma once
#include <cuda_bf16.h>

#include "rv_internal.cuh"

#define RV_KV_THREADS 256
#define RV_KV_UNROLL 2
#define RV_KV_TINY 0x1p-50f

struct KvArgs {
  void *k, *v;                    // cache planes [n_seqs][capacity][n_kv][hd]
  float *k_scale, *v_scale;       // [n_seqs][capacity][n_kv] (8-bit cache)
  void *k_io, *v_io;              // the rows written from / read to
  const int32_t *lens;            // sequence b's rows end at lens[b]; null: start at `position`
  size_t seq_stride, token_stride;  // of k_io / v_io, in elements
  size_t position, capacity;
  uint32_t n, n_kv, hd;           // rows per sequence, heads, row length
  uint32_t lanes;                 // threads per row: the power of two >= hd / 8
  int aligned;                    // k_io, v_io and their strides are multiples of 16 bytes
};

// Eight consecutive elements as f32.
template <typename T>
RV_DEVFN void kv_load8(const T *p, bool aligned, float (&x)[8]) {
  __align__(16) T t[8];
  if (aligned) {
#pragma unroll
    for (int i = 0; i < (int)sizeof t / 16; i++) ((uint4 *)t)[i] = __ldcs((const uint4 *)p + i);
  } else {
#pragma unroll
    for (int i = 0; i < 8; i++) t[i] = p[i];
  }
#pragma unroll
  for (int i = 0; i < 8; i++) x[i] = (float)t[i];
}
template <typename T>
RV_DEVFN void kv_store8(T *p, bool aligned, const float (&x)[8]) {
  __align__(16) T t[8];
#pragma unroll
  for (int i = 0; i < 8; i++) t[i] = (T)x[i];
  if (aligned) {
#pragma unroll
    for (int i = 0; i < (int)sizeof t / 16; i++) __stcs((uint4 *)p + i, ((uint4 *)t)[i]);
  } else {
#pragma unroll
    for (int i = 0; i < 8; i++) p[i] = t[i];
  }
}

// The cache position of row i of sequence b, -1 when it has none (an earlier
// token than the sequence's first) or when it lies past the cache, which sets
// the device error word.
RV_DEVFN long long kv_position(const KvArgs &a, uint32_t b, uint32_t i) {
  const long long pos = a.lens ? (long long)a.lens[b] - a.n + i : (long long)a.position + i;
  if (pos >= (long long)a.capacity) {
    rv_dev_fail(RV_ERR_CAPACITY_EXCEEDED);
    return -1;
  }
  return pos < 0 ? -1 : pos;
}

// Both kernels move RV_KV_UNROLL rows a thread (their loads in flight together).
// grid = (row blocks of one sequence, sequences, 2: keys and values).
struct KvRow {
  uint32_t i, h;
  long long pos;
  size_t at;  // the row in the cache
};
RV_DEVFN KvRow kv_row(const KvArgs &a, uint32_t b, int u) {
  const uint32_t per = RV_KV_THREADS / a.lanes, row = (blockIdx.x * RV_KV_UNROLL + u) * per + threadIdx.x / a.lanes;
  KvRow r;
  r.i = row / a.n_kv;
  r.h = row - r.i * a.n_kv;
  r.pos = r.i < a.n ? kv_position(a, b, r.i) : -1;
  r.at = ((size_t)b * a.capacity + (size_t)(r.pos < 0 ? 0 : r.pos)) * a.n_kv + r.h;
  return r;
}

// Rows into the cache.
template <typename T, bool Q8>
__global__ void __launch_bounds__(RV_KV_THREADS) k_kv_append(KvArgs a) {
  const uint32_t lane = threadIdx.x % a.lanes, b = blockIdx.y, e = lane * 8;
  const bool val = blockIdx.z != 0;
  float x[RV_KV_UNROLL][8];
  KvRow r[RV_KV_UNROLL];
#pragma unroll
  for (int u = 0; u < RV_KV_UNROLL; u++) {
    r[u] = kv_row(a, b, u);
#pragma unroll
    for (int j = 0; j < 8; j++) x[u][j] = 0;
    if (r[u].pos >= 0 && e < a.hd)
      kv_load8((const T *)(val ? a.v_io : a.k_io) + b * a.seq_stride + r[u].i * a.token_stride +
                   (size_t)r[u].h * a.hd + e,
               a.aligned, x[u]);
  }
#pragma unroll
  for (int u = 0; u < RV_KV_UNROLL; u++) {
    const bool on = r[u].pos >= 0 && e < a.hd;
    if constexpr (!Q8) {
      if (on) kv_store8((__half *)(val ? a.v : a.k) + r[u].at * a.hd + e, true, x[u]);
    } else {
      // max |x| as bits: for non-negative floats the integer order is the
      // float order with NaN above infinity, so a NaN is not lost.  Every lane
      // of a row's group reaches the shuffles.
      uint32_t m = 0;
#pragma unroll
      for (int j = 0; j < 8; j++) m = max(m, __float_as_uint(x[u][j]) & 0x7FFFFFFFu);
      for (uint32_t o = a.lanes / 2; o; o >>= 1) m = max(m, __shfl_xor_sync(RV_FULL, m, o));
      const float amax = __uint_as_float(m);
      const bool zero = amax < RV_KV_TINY;
      const float inv = zero ? 0.0f : __fmul_rn(__frcp_rn(amax), 127.0f);
      uint32_t w[2] = {0, 0};
#pragma unroll
      for (int j = 0; j < 8; j++) {
        const int level = __float2int_rn(__fmul_rn(x[u][j], inv));  // NaN -> 0
        w[j >> 2] |= (uint32_t)(level & 255) << (8 * (j & 3));
      }
      if (on) {
        *(uint2 *)((int8_t *)(val ? a.v : a.k) + r[u].at * a.hd + e) = make_uint2(w[0], w[1]);
        if (lane == 0) (val ? a.v_scale : a.k_scale)[r[u].at] = zero ? 0.0f : __fmul_rn(amax, 1.0f / 127.0f);
      }
    }
  }
}

// Rows out of the cache, as f32, f16 or bf16 (one rounding of level * scale).
// A row without a position is written as zeros.
template <typename T, bool Q8>
__global__ void __launch_bounds__(RV_KV_THREADS) k_kv_read(KvArgs a) {
  const uint32_t b = blockIdx.y, e = threadIdx.x % a.lanes * 8;
  const bool val = blockIdx.z != 0;
  float x[RV_KV_UNROLL][8], s[RV_KV_UNROLL];
  uint2 w[RV_KV_UNROLL];
  KvRow r[RV_KV_UNROLL];
#pragma unroll
  for (int u = 0; u < RV_KV_UNROLL; u++) {
    r[u] = kv_row(a, b, u);
    w[u] = make_uint2(0, 0);
    s[u] = 0;
#pragma unroll
    for (int j = 0; j < 8; j++) x[u][j] = 0;
    if (r[u].pos >= 0 && e < a.hd) {
      if constexpr (Q8) {
        w[u] = *(const uint2 *)((const int8_t *)(val ? a.v : a.k) + r[u].at * a.hd + e);
        s[u] = (val ? a.v_scale : a.k_scale)[r[u].at];
      } else {
        kv_load8((const __half *)(val ? a.v : a.k) + r[u].at * a.hd + e, true, x[u]);
      }
    }
  }
#pragma unroll
  for (int u = 0; u < RV_KV_UNROLL; u++) {
    if constexpr (Q8) {
#pragma unroll
      for (int j = 0; j < 8; j++)
        x[u][j] = __fmul_rn((float)(int8_t)((j < 4 ? w[u].x : w[u].y) >> (8 * (j & 3))), s[u]);
    }
    if (r[u].i < a.n && e < a.hd)
      kv_store8((T *)(val ? a.v_io : a.k_io) + b * a.seq_stride + r[u].i * a.token_stride + (size_t)r[u].h * a.hd + e,
                a.aligned, x[u]);
  }
}
