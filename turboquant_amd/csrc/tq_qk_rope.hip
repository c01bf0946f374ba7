// tq_qk_rope.hip -- RMS norm of each query and key head and the position
// rotation in one pass.
//
// A head is a row of head_dim elements; lanes of one wave hold it, eight
// elements each, so a row is read and written by 16-byte accesses, its sum of
// squares is a reduction over its lanes, and the partner of a rotated element
// comes from another lane.  The rotation's angle is position x frequency: at
// position 10^6 an f32 product is off by up to 0.03 rad, so it is formed in
// f64, reduced to [-pi/4, pi/4] there, and sine and cosine of what is left
// are their Taylor series in f32.  Bound by HBM, one read and one write of
// every row: 8,192 tokens of 32 + 8 heads of 128 bf16 elements, 168 MB, take
// 36.4 us where nothing of them is in a cache (4.6 TB/s; a copy reaches 5.1).  A lane
// that forms its own elements' turns for every row takes 74 us; 16 tokens take
// 4.8, the launch and two dependent reads.
#include "tq_mfma.h"
#include "tq_paged.h"

#include <algorithm>
#include <type_traits>

namespace {

using namespace tqm;

struct RopeArgs {
  const void *x[2];         // queries, keys
  void *out[2];
  const void *weight[2];    // null: no norm
  long long in_stride[2], out_stride[2];
  int heads[2];
  const int *positions;
  const float *inv_freq;
  int tokens, head_dim, rot, half;
  int splits;               // waves that share a token's rows
  int through;              // tqh::store16
  float eps, inv_dim;
};

// cos and sin of position x frequency.  The turn is reduced by multiples of
// pi / 2 in f64 (the product's own rounding, 2^-53 of it, is what is lost:
// 2.4e-7 rad at 2^31 rad); on [-pi/4, pi/4] the series' next terms, r^11 / 11!
// and r^12 / 12!, are below 1.8e-9 and 1.2e-10.
__device__ __forceinline__ void turn(int pos, float freq, float &c, float &s) {
  const double t = (double)pos * (double)freq;
  const double n = __builtin_rint(t * 0.63661977236758134308);
  double rd = __builtin_fma(n, -1.57079632679489655800, t);
  rd = __builtin_fma(n, -6.12323399573676603587e-17, rd);
  const float r = (float)rd, z = r * r;
  float sp = __builtin_fmaf(z, 2.7557319e-6f, -1.9841270e-4f);
  sp = __builtin_fmaf(z, sp, 8.3333333e-3f);
  sp = __builtin_fmaf(z, sp, -1.6666667e-1f);
  const float sn = __builtin_fmaf(r * z, sp, r);
  float cp = __builtin_fmaf(z, -2.7557319e-7f, 2.4801587e-5f);
  cp = __builtin_fmaf(z, cp, -1.3888889e-3f);
  cp = __builtin_fmaf(z, cp, 4.1666667e-2f);
  cp = __builtin_fmaf(z, cp, -0.5f);
  const float cs = __builtin_fmaf(z, cp, 1.0f);
  const int q = (int)(long long)n & 3;
  const float a = q & 1 ? sn : cs, b = q & 1 ? cs : sn;
  c = (q + 1) & 2 ? -a : a;
  s = q & 2 ? -b : b;
}

template <int DT>
__device__ __forceinline__ float load1(const void *p, long long i) {
  if constexpr (DT == kF32) return static_cast<const float *>(p)[i];
  const uint16_t h = static_cast<const uint16_t *>(p)[i];
  return DT == kBF16 ? bf16_to_f32(h) : f16_to_f32(h);
}
// Elements i .. i + 7, in 16-byte accesses where VEC.
template <int DT, bool VEC>
__device__ __forceinline__ void load8(const void *p, long long i, float (&x)[8]) {
  if constexpr (!VEC) {
#pragma unroll
    for (int j = 0; j < 8; j++) x[j] = load1<DT>(p, i + j);
  } else if constexpr (DT == kF32) {
    const float4 *q = reinterpret_cast<const float4 *>(static_cast<const float *>(p) + i);
    const float4 a = q[0], b = q[1];
    x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w;
    x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
  } else {
    const uint4 v = *reinterpret_cast<const uint4 *>(static_cast<const uint16_t *>(p) + i);
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int j = 0; j < 4; j++) {
      x[2 * j] = DT == kBF16 ? u2f(w[j] << 16) : f16_to_f32((uint16_t)(w[j] & 0xffffu));
      x[2 * j + 1] = DT == kBF16 ? u2f(w[j] & 0xffff0000u) : f16_to_f32((uint16_t)(w[j] >> 16));
    }
  }
}
template <int DT, bool VEC>
__device__ __forceinline__ void store8(void *p, long long i, const float (&x)[8], int through) {
  if constexpr (DT == kF32) {
    float *q = static_cast<float *>(p) + i;
    if constexpr (VEC) {
      tqh::store16(q, u32x4{f2u(x[0]), f2u(x[1]), f2u(x[2]), f2u(x[3])}, through);
      tqh::store16(q + 4, u32x4{f2u(x[4]), f2u(x[5]), f2u(x[6]), f2u(x[7])}, through);
    } else {
#pragma unroll
      for (int j = 0; j < 8; j++) q[j] = x[j];
    }
  } else {
    uint32_t w[4];
#pragma unroll
    for (int j = 0; j < 4; j++)
      w[j] = DT == kBF16 ? pack_bf16x2(x[2 * j], x[2 * j + 1])
                         : (uint32_t)f32_to_f16(x[2 * j]) | ((uint32_t)f32_to_f16(x[2 * j + 1]) << 16);
    uint16_t *q = static_cast<uint16_t *>(p) + i;
    if constexpr (VEC) {
      tqh::store16(q, u32x4{w[0], w[1], w[2], w[3]}, through);
    } else {
#pragma unroll
      for (int j = 0; j < 8; j++) q[j] = (uint16_t)(w[j >> 1] >> (16 * (j & 1)));
    }
  }
}

template <int LPR>
__device__ __forceinline__ float row_sum(float v) {
  v += lane_xor<1>(v);
  v += lane_xor<2>(v);
  if constexpr (LPR >= 8) v += lane_xor<4>(v);
  if constexpr (LPR >= 16) v += lane_xor<8>(v);
  if constexpr (LPR >= 32) v += lane_xor<16>(v);
  return v;
}

// Where a rotated element's partner is: its neighbour in the lane; the same
// element of lane ^ LPR / 2 (the whole row of 8 LPR elements turns); any
// element of the row.
enum Partner : int { kNeighbour = 0, kHalfRow = 1, kAny = 2 };

constexpr int kWaves = 2048;  // waves that a launch of few tokens is split into
constexpr int kBatch = 4;  // rows a lane has in flight

// LPR lanes a row (a power of two, eight elements a lane; lanes past head_dim
// hold zeros).  A wave takes one token, or one of `splits` parts of its rows,
// 64 / LPR rows a pass: the turns are formed once, a pair a lane, and kept as
// each lane's eight through LDS.
template <int LPR, int DT, bool VEC, int PARTNER>
__global__ __launch_bounds__(256) void qk_norm_rope_kernel(RopeArgs a) {
  constexpr int RPW = 64 / LPR, NT = PARTNER == kNeighbour ? 4 : 8;
  __shared__ float2 s_turn[4][4 * LPR];
  __shared__ __attribute__((aligned(16))) float s_row[PARTNER == kAny ? 4 : 1][PARTNER == kAny ? 512 : 1];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int l = lane % LPR, e0 = 8 * l, r = lane / LPR;
  const int id = blockIdx.x * 4 + wave;
  const int t = id / a.splits, part = id - t * a.splits;
  if (t >= a.tokens) return;
  const int pos = a.positions[t];
  if (pos < 0) return;  // no token
  const bool in = e0 < a.head_dim;
  const int passes_q = (a.heads[0] + RPW - 1) / RPW, passes = passes_q + (a.heads[1] + RPW - 1) / RPW;
  const int p1 = (int)((long long)(part + 1) * passes / a.splits);
  float x[kBatch][8];
  auto head_of = [&](int p, int which) { return (which ? p - passes_q : p) * RPW + r; };
  auto load = [&](int p0) {
#pragma unroll
    for (int u = 0; u < kBatch; u++) {
      const int p = p0 + u, which = p >= passes_q, h = head_of(p, which);
#pragma unroll
      for (int j = 0; j < 8; j++) x[u][j] = 0.f;
      if (p < p1 && in && h < a.heads[which])
        load8<DT, VEC>(a.x[which], t * a.in_stride[which] + (long long)h * a.head_dim + e0, x[u]);
    }
  };
  int p0 = (int)((long long)part * passes / a.splits);
  load(p0);
  float w[2][8] = {};
#pragma unroll
  for (int k = 0; k < 2; k++)
    if (a.weight[k] && in) load8<DT, false>(a.weight[k], e0, w[k]);
  for (int i = lane; i < a.half; i += 64) {
    float c, s;
    turn(pos, a.inv_freq[i], c, s);
    s_turn[wave][i] = make_float2(c, s);
  }
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
  float c[NT], s[NT];
#pragma unroll
  for (int j = 0; j < NT; j++) {
    const int e = PARTNER == kNeighbour ? e0 + 2 * j : e0 + j;
    const int i = PARTNER == kNeighbour ? e >> 1 : (e < a.half ? e : e - a.half);
    c[j] = 1.f;
    s[j] = 0.f;
    if (e < a.rot) {
      const float2 v = s_turn[wave][i];
      c[j] = v.x;
      s[j] = PARTNER != kNeighbour && e < a.half ? -v.y : v.y;  // the sign of the partner's part
    }
  }
  for (;;) {
#pragma unroll
    for (int u = 0; u < kBatch; u++) {
      const int p = p0 + u;
      if (p >= p1) break;  // uniform
      const int which = p >= passes_q, h = head_of(p, which);
      if (a.weight[which]) {
        float ss = 0.f;
#pragma unroll
        for (int j = 0; j < 8; j++) ss = __builtin_fmaf(x[u][j], x[u][j], ss);
        const float scale = 1.0f / sqrtf(__builtin_fmaf(row_sum<LPR>(ss), a.inv_dim, a.eps));
#pragma unroll
        for (int j = 0; j < 8; j++) x[u][j] = x[u][j] * scale * w[which][j];
      }
      float y[8];
      if constexpr (PARTNER == kNeighbour) {
#pragma unroll
        for (int j = 0; j < 4; j++) {  // past rot a neighbour has no part, an infinite one neither
          const bool on = e0 + 2 * j < a.rot;
          const float x0 = x[u][2 * j], x1 = x[u][2 * j + 1];
          y[2 * j] = x0 * c[j] - (on ? x1 : 0.f) * s[j];
          y[2 * j + 1] = x1 * c[j] + (on ? x0 : 0.f) * s[j];
        }
      } else if constexpr (PARTNER == kHalfRow) {
#pragma unroll
        for (int j = 0; j < 8; j++) y[j] = x[u][j] * c[j] + lane_xor<LPR / 2>(x[u][j]) * s[j];
      } else {
        float *mine = s_row[wave] + r * (8 * LPR);
        __builtin_amdgcn_wave_barrier();
        reinterpret_cast<float4 *>(mine + e0)[0] = make_float4(x[u][0], x[u][1], x[u][2], x[u][3]);
        reinterpret_cast<float4 *>(mine + e0)[1] = make_float4(x[u][4], x[u][5], x[u][6], x[u][7]);
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
#pragma unroll
        for (int j = 0; j < 8; j++) {
          const int e = e0 + j, o = e >= a.rot ? e : (e < a.half ? e + a.half : e - a.half);
          y[j] = x[u][j] * c[j] + (e >= a.rot ? 0.f : mine[o]) * s[j];
        }
      }
      if (in && h < a.heads[which])
        store8<DT, VEC>(a.out[which], t * a.out_stride[which] + (long long)h * a.head_dim + e0, y, a.through);
    }
    p0 += kBatch;
    if (p0 >= p1) break;
    load(p0);
  }
}

}  // namespace

extern "C" int tq_qk_norm_rope(const void *q, long long q_stride, const void *k, long long k_stride, int dtype,
                               const int *positions, int tokens, int num_heads, int num_kv_heads, int head_dim,
                               const float *inv_freq, int rot_dim, int interleaved, const void *q_weight,
                               const void *k_weight, float eps, void *q_out, long long q_out_stride, void *k_out,
                               long long k_out_stride, hipStream_t stream) {
  if (!tqh::valid_dtype(dtype)) return tqh::fail(TQ_ERR_INVALID_ARGUMENT, "unknown dtype %d", dtype);
  if (head_dim <= 0 || head_dim % 32 != 0 || head_dim > 256)
    return tqh::fail(TQ_ERR_INVALID_DIMENSION, "head_dim %d is no multiple of 32 up to 256", head_dim);
  if (rot_dim < 0 || rot_dim > head_dim || rot_dim % 2 != 0)
    return tqh::fail(TQ_ERR_INVALID_DIMENSION, "rot_dim %d is no even number up to head_dim %d", rot_dim, head_dim);
  if (tokens < 0 || num_heads < 0 || num_kv_heads < 0 || num_heads > 65535 || num_kv_heads > 65535)
    return tqh::fail(TQ_ERR_INVALID_ARGUMENT, "negative shape, or more than 65,535 heads");
  if (!(eps >= 0.0f)) return tqh::fail(TQ_ERR_INVALID_ARGUMENT, "eps must not be negative");
  const long long rows = (long long)tokens * (num_heads + num_kv_heads);
  if (rows == 0) return TQ_OK;
  if (!positions || (rot_dim && !inv_freq) || (num_heads && (!q || !q_out)) || (num_kv_heads && (!k || !k_out)))
    return tqh::fail(TQ_ERR_INVALID_ARGUMENT, "null pointer");
  const long long qd = (long long)num_heads * head_dim, kd = (long long)num_kv_heads * head_dim;
  if (q_stride < qd || k_stride < kd || q_out_stride < qd || k_out_stride < kd)
    return tqh::fail(TQ_ERR_DIMENSION_MISMATCH, "a row stride is shorter than a token's heads");
  RopeArgs a{};
  a.x[0] = q;
  a.x[1] = k;
  a.out[0] = q_out;
  a.out[1] = k_out;
  a.weight[0] = q_weight;
  a.weight[1] = k_weight;
  a.in_stride[0] = q_stride;
  a.in_stride[1] = k_stride;
  a.out_stride[0] = q_out_stride;
  a.out_stride[1] = k_out_stride;
  a.heads[0] = num_heads;
  a.heads[1] = num_kv_heads;
  a.positions = positions;
  a.inv_freq = inv_freq;
  a.tokens = tokens;
  a.head_dim = head_dim;
  a.rot = rot_dim;
  a.half = rot_dim / 2;
  a.eps = eps;
  a.inv_dim = 1.0f / (float)head_dim;
  const int size = tqh::dtype_size(dtype);
  a.through = rows * head_dim * size > tqh::kThroughBytes;
  const bool vec = (!num_heads || (tqh::rows_aligned(q, q_stride, size) && tqh::rows_aligned(q_out, q_out_stride, size))) &&
                   (!num_kv_heads || (tqh::rows_aligned(k, k_stride, size) && tqh::rows_aligned(k_out, k_out_stride, size)));
  const int lpr = head_dim <= 32 ? 4 : (head_dim <= 64 ? 8 : (head_dim <= 128 ? 16 : 32)), rpw = 64 / lpr;
  const int passes = (num_heads + rpw - 1) / rpw + (num_kv_heads + rpw - 1) / rpw;
  // few tokens: their rows are shared out until the card has waves enough
  a.splits = (int)std::min<long long>(passes, std::max<long long>(1, kWaves / tokens));
  const long long blocks = ((long long)tokens * a.splits + 3) / 4;
  if (blocks >= 1ll << 24) return tqh::fail(TQ_ERR_INVALID_ARGUMENT, "too many rows in one call");
  auto go = [&](auto l, auto d, auto v, auto p) {
    hipLaunchKernelGGL((qk_norm_rope_kernel<l.value, d.value, v.value, p.value>), dim3((unsigned)blocks), dim3(256), 0,
                       stream, a);
  };
  auto by_partner = [&](auto l, auto d, auto v) {
    if (interleaved) go(l, d, v, std::integral_constant<int, kNeighbour>{});
    else if (rot_dim == 8 * lpr) go(l, d, v, std::integral_constant<int, kHalfRow>{});
    else go(l, d, v, std::integral_constant<int, kAny>{});
  };
  auto by_vec = [&](auto l, auto d) {
    if (vec) by_partner(l, d, std::true_type{});
    else by_partner(l, d, std::false_type{});
  };
  auto by_type = [&](auto l) {
    if (dtype == kF32) by_vec(l, std::integral_constant<int, kF32>{});
    else if (dtype == kBF16) by_vec(l, std::integral_constant<int, kBF16>{});
    else by_vec(l, std::integral_constant<int, kF16>{});
  };
  if (lpr == 4) by_type(std::integral_constant<int, 4>{});
  else if (lpr == 8) by_type(std::integral_constant<int, 8>{});
  else if (lpr == 16) by_type(std::integral_constant<int, 16>{});
  else by_type(std::integral_constant<int, 32>{});
  return tqh::check_launch("qk_norm_rope_kernel");
}
