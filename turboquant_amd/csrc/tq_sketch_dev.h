// tq_sketch_dev.h -- the QJL sketch of a key's residual: 16 vectors' products
// with the rows of R on the matrix cores, and the residual that they take.
// Shared by the TQ append of contiguous caches and of pages.
#pragma once

#include "tq_pqo_dev.h"

namespace tqs {

using namespace tqp;

typedef float f32x4 __attribute__((ext_vector_type(4)));

constexpr int kVecs = 16;  // vectors (or query rows) per workgroup

template <int D>
struct Geo {
  static constexpr int NQB = D / 32, NW = D / 32, WAVES = D / 32, THREADS = 64 * WAVES;
  static constexpr int RS = D + 4;  // floats per staged row: the chain's reads hit 64 banks
};

// Sign words of R's rows 16 (T wave + t) + l16, shifted so that column
// 4 k + lg of word w is bit 4 k.
template <int D, int T>
__device__ __forceinline__ void load_rows(const uint32_t *__restrict__ rbits, int wave, int l16, int lg,
                                          uint32_t (&rb)[T][Geo<D>::NW]) {
#pragma unroll
  for (int t = 0; t < T; t++)
#pragma unroll
    for (int w = 0; w < Geo<D>::NW; w++) rb[t][w] = rbits[(16 * (T * wave + t) + l16) * Geo<D>::NW + w] >> lg;
}

// acc[t][i] = sum_c R[16 (T wave + t) + 4 lg + i][c] v[l16][c] (R = +-1), in
// column order from -0.0, for the 16 vectors staged in LDS.
template <int D, int T>
__device__ __forceinline__ void row_products(const float *s_v, const uint32_t (&rb)[T][Geo<D>::NW], int l16, int lg,
                                             f32x4 (&acc)[T]) {
#pragma unroll
  for (int t = 0; t < T; t++) acc[t] = f32x4{-0.0f, -0.0f, -0.0f, -0.0f};
  const float *v = s_v + l16 * Geo<D>::RS + lg;
#pragma unroll
  for (int w = 0; w < Geo<D>::NW; w++) {
    float x[8];
#pragma unroll
    for (int k = 0; k < 8; k++) x[k] = v[32 * w + 4 * k];
#pragma unroll
    for (int k = 0; k < 8; k++)
#pragma unroll
      for (int t = 0; t < T; t++) {
        const float a = u2f(((rb[t][w] << (31 - 4 * k)) & 0x80000000u) | 0x3f800000u);
        acc[t] = __builtin_amdgcn_mfma_f32_16x16x4f32(a, x[k], acc[t], 0, 0, 0);
      }
  }
}

// The residual x - x_hat of block qb of the workgroup's vector vi, x_hat the
// block's record (codes w, scale s >= 0) as polar_dequantize's CPU branch gives
// it (quantize_tensor.rs:197-219, butterflies), into s_v; returns the lane's
// part of the vector's sum of squares: in element order through the vector's
// lanes, whole in its last one.  s_cb: the centroids times the decode factor.
template <int D, int BITS>
__device__ __forceinline__ float stage_residual(float (&x)[32], const uint32_t (&w)[BITS], float s, const float *s_cb,
                                                float *s_v, int vi, int qb) {
  float y[32];
#pragma unroll
  for (int j = 0; j < 32; j++) {
    const float c = s_cb[field<BITS>(w, j)];
    y[j] = pqo_neg(j) ? -c : c;
  }
  butterfly<32>(y);
#pragma unroll
  for (int j = 0; j < 32; j++) x[j] = x[j] - (y[j] * kInvSqrt32) * s;
  float4 *dst = reinterpret_cast<float4 *>(s_v + vi * Geo<D>::RS + 32 * qb);
#pragma unroll
  for (int j = 0; j < 8; j++) dst[j] = make_float4(x[4 * j], x[4 * j + 1], x[4 * j + 2], x[4 * j + 3]);
  // lane qb continues the sum of lane qb - 1; after NQB rounds the last
  // lane's has run over the whole key
#pragma unroll
  for (int j = 0; j < 32; j++) x[j] = x[j] * x[j];
  float ss = 0.f;
#pragma unroll
  for (int round = 0; round < Geo<D>::NQB; round++) {
    const float before = __shfl_up(ss, 1, 64);
    ss = qb == 0 ? 0.f : before;
#pragma unroll
    for (int j = 0; j < 32; j++) ss = ss + x[j];
  }
  return ss;
}

// Bits j = (R r)_j >= 0 (qjl.rs:305-319) of the wave's 32 rows, one word of the
// key in every lane l16 of it.
__device__ __forceinline__ uint32_t sign_word(const f32x4 (&acc)[2], float inv_sqrt_d, int lg) {
  uint32_t bits = 0;
#pragma unroll
  for (int t = 0; t < 2; t++)
#pragma unroll
    for (int i = 0; i < 4; i++) bits |= (acc[t][i] * inv_sqrt_d >= 0.0f ? 1u : 0u) << (16 * t + 4 * lg + i);
  bits |= __shfl_xor(bits, 16, 64);
  bits |= __shfl_xor(bits, 32, 64);
  return bits;
}

}  // namespace tqs
