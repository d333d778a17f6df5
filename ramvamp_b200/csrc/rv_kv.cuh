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
// Both kernels move each byte once.  Eight values a thread (one 16-byte load of
// f16, two of f32) and 16 lanes a row of 128, so the row's maximum is four
// shuffles.
#pragma once
#include <cuda_bf16.h>

#include "rv_internal.cuh"

#define RV_KV_THREADS 256
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

// Rows into the cache.  grid = (row blocks of one sequence, sequences, 2: keys
// and values).
template <typename T, bool Q8>
__global__ void __launch_bounds__(RV_KV_THREADS) k_kv_append(KvArgs a) {
  const uint32_t per = RV_KV_THREADS / a.lanes, lane = threadIdx.x % a.lanes;
  const uint32_t row = blockIdx.x * per + threadIdx.x / a.lanes, b = blockIdx.y;
  const uint32_t i = row / a.n_kv, h = row - i * a.n_kv, e = lane * 8;
  const bool val = blockIdx.z != 0;
  // Every lane of a row's group reaches the shuffles.
  const long long pos = i < a.n ? kv_position(a, b, i) : -1;
  const bool on = pos >= 0 && e < a.hd;
  float x[8] = {0, 0, 0, 0, 0, 0, 0, 0};
  if (on)
    kv_load8((const T *)(val ? a.v_io : a.k_io) + b * a.seq_stride + i * a.token_stride + (size_t)h * a.hd + e, a.aligned,
             x);
  const size_t at = ((size_t)b * a.capacity + (size_t)(pos < 0 ? 0 : pos)) * a.n_kv + h;
  if constexpr (!Q8) {
    if (on) kv_store8((__half *)(val ? a.v : a.k) + at * a.hd + e, true, x);
  } else {
    // max |x| as bits: for non-negative floats the integer order is the
    // float order with NaN above infinity, so a NaN is not lost.
    uint32_t m = 0;
#pragma unroll
    for (int j = 0; j < 8; j++) m = max(m, __float_as_uint(x[j]) & 0x7FFFFFFFu);
    for (uint32_t o = a.lanes / 2; o; o >>= 1) m = max(m, __shfl_xor_sync(RV_FULL, m, o));
    const float amax = __uint_as_float(m);
    const bool zero = amax < RV_KV_TINY;
    const float inv = zero ? 0.0f : __fmul_rn(__frcp_rn(amax), 127.0f);
    uint32_t w[2] = {0, 0};
#pragma unroll
    for (int j = 0; j < 8; j++) {
      const int level = __float2int_rn(__fmul_rn(x[j], inv));  // NaN -> 0
      w[j >> 2] |= (uint32_t)(level & 255) << (8 * (j & 3));
    }
    if (on) {
      *(uint2 *)((int8_t *)(val ? a.v : a.k) + at * a.hd + e) = make_uint2(w[0], w[1]);
      if (lane == 0) (val ? a.v_scale : a.k_scale)[at] = zero ? 0.0f : __fmul_rn(amax, 1.0f / 127.0f);
    }
  }
}

// Rows out of the cache, as f32, f16 or bf16 (one rounding of level * scale).
// A row without a position is written as zeros.
template <typename T, bool Q8>
__global__ void __launch_bounds__(RV_KV_THREADS) k_kv_read(KvArgs a) {
  const uint32_t per = RV_KV_THREADS / a.lanes, e = threadIdx.x % a.lanes * 8;
  const uint32_t row = blockIdx.x * per + threadIdx.x / a.lanes, b = blockIdx.y;
  const uint32_t i = row / a.n_kv, h = row - i * a.n_kv;
  const bool val = blockIdx.z != 0;
  if (i >= a.n || e >= a.hd) return;
  const long long pos = kv_position(a, b, i);
  float x[8] = {0, 0, 0, 0, 0, 0, 0, 0};
  if (pos >= 0) {
    const size_t at = ((size_t)b * a.capacity + (size_t)pos) * a.n_kv + h;
    if constexpr (Q8) {
      const uint2 w = *(const uint2 *)((const int8_t *)(val ? a.v : a.k) + at * a.hd + e);
      const float s = (val ? a.v_scale : a.k_scale)[at];
#pragma unroll
      for (int j = 0; j < 8; j++)
        x[j] = __fmul_rn((float)(int8_t)((j < 4 ? w.x : w.y) >> (8 * (j & 3))), s);
    } else {
      kv_load8((const __half *)(val ? a.v : a.k) + at * a.hd + e, true, x);
    }
  }
  kv_store8((T *)(val ? a.v_io : a.k_io) + b * a.seq_stride + i * a.token_stride + (size_t)h * a.hd + e, a.aligned, x);
}
