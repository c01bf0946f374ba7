// tq_paged_store.hip -- keys and values into the records of pages and back.
//
// The codec is the contiguous cache's (tq_pqo_dev.h: one lane a 32-element
// block); what differs is where a record lies: slot s of KV head g is record
// ((s / page_size) num_kv_heads + g) page_size + s % page_size.  Consecutive
// lanes take consecutive blocks of the activations, which are four to five
// times the records' bytes; a workgroup's eight tokens (8 heads of 128) still
// make runs of 384 bytes in each head's records.  Bound by HBM for prompts and
// by the launch for a token per request: 8,000 tokens of 3-bit codes, 8 heads
// of 128, are stored in 13.5 us and loaded in 11.5 (40 MB each, 3.0 and 3.5
// TB/s), 64,000 in 80 and 53 (4.0 and 6.0 TB/s).  Lanes along the tokens of one
// head, so that records are one run and activations pieces of a head, store
// them in 87.
#include "tq_paged.h"
#include "tq_sketch_dev.h"

#include <type_traits>

namespace {

using namespace tqs;

struct Pages {
  const long long *slots;
  long long num_slots;
  int heads, shift, tokens;
};

// Record of token t of head g, or -1 where its slot names no token.
__device__ __forceinline__ long long paged_record(const Pages &p, int t, int g) {
  if (t >= p.tokens) return -1;
  const long long s = p.slots[t];
  if (s < 0 || s >= p.num_slots) return -1;
  return (((s >> p.shift) * p.heads + g) << p.shift) + (s & ((1 << p.shift) - 1));
}

// Consecutive workgroups go to the eight dies in turn; this gives each die a run
// of the work, so that a line of records that two workgroups write is whole in
// one L2 (64,000 tokens stored in 91 us in turn, in 82 so).
__device__ __forceinline__ int die_order(int b, int n) {
  const int q = n >> 3;
  return b < 8 * q ? (b & 7) * q + (b >> 3) : b;
}

// Block at element i of x, by 16-byte loads where `vec`.
template <int DT>
__device__ __forceinline__ void load_at(const void *x, long long i, int vec, float (&r)[32]) {
  if (vec) {
    if constexpr (DT == kF32) load_block<DT>(static_cast<const float *>(x) + i, 0, r);
    else load_block<DT>(static_cast<const uint16_t *>(x) + i, 0, r);
  } else {
#pragma unroll
    for (int j = 0; j < 32; j++) {
      if constexpr (DT == kF32) r[j] = static_cast<const float *>(x)[i + j];
      else r[j] = DT == kBF16 ? bf16_to_f32(static_cast<const uint16_t *>(x)[i + j])
                              : f16_to_f32(static_cast<const uint16_t *>(x)[i + j]);
    }
  }
}

struct StoreArgs {
  Pages pages;
  const void *x[2];  // keys, values
  long long stride[2];
  int vec[2];
  uint8_t *idx[2];
  uint16_t *sc[2];
  int num_blocks;    // blocks of a head
  QuantConsts qc;
  // TQ
  uint32_t *signs;
  uint16_t *norms;
  const uint32_t *rbits;
  float cb[16], decode_factor, inv_sqrt_d;
};

// grid (tokens x heads x blocks, keys and values)
template <int BITS, int CB, int DT, int NORM>
__global__ __launch_bounds__(256) void paged_store_kernel(StoreArgs a) {
  const int lin = die_order(blockIdx.x, gridDim.x) * 256 + threadIdx.x, z = blockIdx.y;
  const int v = lin / a.num_blocks, qb = lin - v * a.num_blocks;
  const int t = v / a.pages.heads, g = v - t * a.pages.heads;
  if (t >= a.pages.tokens) return;
  // encoded whether its slot names a token or not: the block's load does not wait for the slot's
  float r[32];
  load_at<DT>(a.x[z], t * a.stride[z] + ((long long)g * a.num_blocks + qb) * 32, a.vec[z], r);
  const long long rec = paged_record(a.pages, t, g);
  uint32_t w[BITS];
  const float s = encode_block<BITS, CB, true, NORM>(r, a.qc, w);
  if (rec < 0) return;
  const long long blk = rec * a.num_blocks + qb;
  store_packed<BITS>(a.idx[z], blk, w);
  a.sc[z][blk] = f32_to_f16(s * a.qc.scale_sign);
}

// The TQ append (tq_qjl_sketch.hip) with its records in pages: a workgroup
// takes 16 tokens of one head.
template <int D, int BITS, int DT, int NORM>
__global__ __launch_bounds__(Geo<D>::THREADS) void paged_store_tq_kernel(StoreArgs a) {
  using G = Geo<D>;
  constexpr int NQB = G::NQB;
  __shared__ __attribute__((aligned(16))) float s_v[kVecs * G::RS];
  __shared__ float s_cb[16];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int l16 = lane & 15, lg = lane >> 4;
  const int t0 = blockIdx.x * kVecs, g = blockIdx.y;
  uint32_t rb[2][G::NW];
  load_rows<D>(a.rbits, wave, l16, lg, rb);
#pragma unroll
  for (int i = 0; i < 16; i++)
    if (tid == i) s_cb[i] = a.cb[i] * a.decode_factor;
  const int qb = tid % NQB, vi = (tid / NQB) % kVecs;
  const int z = tid >= kVecs * NQB;
  const long long rec = tid < 2 * kVecs * NQB ? paged_record(a.pages, t0 + vi, g) : -1;
  uint32_t w[BITS];
  float x[32], s = 0.f;
  if (rec >= 0) {
    load_at<DT>(a.x[z], (t0 + vi) * a.stride[z] + ((long long)g * NQB + qb) * 32, a.vec[z], x);
    float r[32];
#pragma unroll
    for (int j = 0; j < 32; j++) r[j] = x[j];
    s = encode_block<BITS, BITS - 1, true, NORM>(r, a.qc, w);
    const long long blk = rec * NQB + qb;
    store_packed<BITS>(a.idx[z], blk, w);
    const uint16_t h = f32_to_f16(s * a.qc.scale_sign);
    a.sc[z][blk] = h;
    s = fabsf(f16_to_f32(h));
  }
  __syncthreads();
  if (rec >= 0 && z == 0) {
    const float ss = stage_residual<D, BITS>(x, w, s, s_cb, s_v, vi, qb);
    if (qb == NQB - 1) a.norms[rec] = f32_to_f16(sqrtf(ss));
  }
  __syncthreads();
  f32x4 acc[2];
  row_products<D>(s_v, rb, l16, lg, acc);
  const uint32_t bits = sign_word(acc, a.inv_sqrt_d, lg);
  const long long srec = paged_record(a.pages, t0 + l16, g);
  if (lg == 0 && srec >= 0) a.signs[srec * G::NW + wave] = bits;
}

struct LoadArgs {
  Pages pages;
  const uint8_t *idx[2];
  const uint16_t *sc[2];
  void *out[2];
  int num_blocks, through;  // through: tqh::store16
  float cb[16], sgm;  // the centroids and the decode signs' magnitude
};

// out_j = fl(fl(W_j * fl(1/sqrt(32))) * |scale|), W = butterfly(cb[code] sign),
// the values of tq_polar_dequantize.
// A wave's 64 blocks are staged in LDS (rows padded by 16 bytes), so that a
// store instruction writes 1 KB in one run instead of 16 bytes into each of 64
// places (8,000 tokens in 17 -> 12 us).
template <int BITS, int DT>
__global__ __launch_bounds__(256) void paged_load_kernel(LoadArgs a) {
  constexpr int NDW = DT == kF32 ? 32 : 16, RS = NDW + 4;  // words of a block
  __shared__ float lut[16];
  __shared__ __attribute__((aligned(16))) uint32_t s_out[4][64 * RS];
#pragma unroll
  for (int i = 0; i < 16; i++)
    if (threadIdx.x == i) lut[i] = a.cb[i] * a.sgm;
  __syncthreads();
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, z = blockIdx.y;
  const int lin0 = blockIdx.x * 256 + 64 * wave, lin = lin0 + lane;  // blocks in the output's order
  const int v = lin / a.num_blocks, qb = lin - v * a.num_blocks;
  const int t = v / a.pages.heads, g = v - t * a.pages.heads;
  const long long rec = paged_record(a.pages, t, g);
  const unsigned long long live = __ballot(rec >= 0);
  uint32_t *row = s_out[wave] + lane * RS;
  if (rec >= 0) {
    const long long blk = rec * a.num_blocks + qb;
    const uint32_t *p = reinterpret_cast<const uint32_t *>(a.idx[z] + blk * (4 * BITS));
    uint32_t w[BITS];
    if constexpr (BITS == 4) {
      const uint4 v = *reinterpret_cast<const uint4 *>(p);
      w[0] = v.x; w[1] = v.y; w[2] = v.z; w[3] = v.w;
    } else {
#pragma unroll
      for (int i = 0; i < BITS; i++) w[i] = p[i];
    }
    const float s = fabsf(f16_to_f32(a.sc[z][blk]));
    float y[32];
#pragma unroll
    for (int j = 0; j < 32; j++) {
      const float c = lut[field<BITS>(w, j)];
      y[j] = pqo_neg(j) ? -c : c;
    }
    butterfly<32>(y);
#pragma unroll
    for (int j = 0; j < 32; j++) y[j] = (y[j] * kInvSqrt32) * s;
    uint32_t o[NDW];
#pragma unroll
    for (int j = 0; j < NDW; j++) {
      if constexpr (DT == kF32) o[j] = f2u(y[j]);
      else if constexpr (DT == kBF16) o[j] = pack_bf16x2(y[2 * j], y[2 * j + 1]);
      else o[j] = (uint32_t)f32_to_f16(y[2 * j]) | ((uint32_t)f32_to_f16(y[2 * j + 1]) << 16);
    }
#pragma unroll
    for (int j = 0; j < NDW / 4; j++)
      *reinterpret_cast<uint4 *>(row + 4 * j) = make_uint4(o[4 * j], o[4 * j + 1], o[4 * j + 2], o[4 * j + 3]);
  }
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
  uint32_t *const out = static_cast<uint32_t *>(a.out[z]) + (long long)lin0 * NDW;
#pragma unroll
  for (int q = 0; q < NDW / 4; q++) {
    const int f = 256 * q + 4 * lane, r = f / NDW, c = f % NDW;  // block r of the wave, its words c .. c + 3
    if ((live >> r) & 1)
      tqh::store16(out + f, *reinterpret_cast<const tqh::words4 *>(s_out[wave] + r * RS + c), a.through);
  }
}

float decode_factor() {
  volatile float thirty_two = 32.0f;
  volatile float sq = sqrtf(thirty_two);
  volatile float inv = 1.0f / sq;
  return inv * sq;  // fl(fl(1/sqrt 32) * sqrt 32) (wht_tensor.rs:28-41)
}

// f(integral_constant DT) for a valid element type
template <class F>
void by_type(int dt, F &&f) {
  if (dt == kF32) f(std::integral_constant<int, kF32>{});
  else if (dt == kBF16) f(std::integral_constant<int, kBF16>{});
  else f(std::integral_constant<int, kF16>{});
}

}  // namespace

extern "C" int tq_paged_store(const void *k, long long k_stride, const void *v, long long v_stride, int dtype,
                              const long long *slots, int tokens, uint8_t *k_indices, uint16_t *k_scales,
                              uint8_t *v_indices, uint16_t *v_scales, uint8_t *signs, uint16_t *norms,
                              const uint32_t *sign_matrix, long long num_pages, int num_kv_heads, int page_size,
                              int head_dim, int bits, size_t outlier_blocks, int norm_mode, hipStream_t stream) {
  StoreArgs a{};
  tqh::PolarCodec codec;
  int rc = tqh::check_pages(num_pages, num_kv_heads, page_size, head_dim, bits, outlier_blocks, norm_mode,
                            a.pages.shift, codec);
  if (rc) return rc;
  if (!tqh::valid_dtype(dtype)) return tqh::fail(TQ_ERR_INVALID_ARGUMENT, "unknown dtype %d", dtype);
  if (tokens < 0) return tqh::fail(TQ_ERR_INVALID_ARGUMENT, "negative tokens");
  if (signs && head_dim != 64 && head_dim != 128 && head_dim != 256)
    return tqh::fail(TQ_ERR_INVALID_DIMENSION, "cache QJL kernels take head_dim 64, 128 or 256 (got %d)", head_dim);
  if (signs && codec.outlier)
    return tqh::fail(TQ_ERR_INVALID_ARGUMENT, "QJL correction applies to the standard codebook (outlier_blocks 0)");
  const long long row = (long long)num_kv_heads * head_dim;
  if (k_stride < row || v_stride < row)
    return tqh::fail(TQ_ERR_DIMENSION_MISMATCH, "a row stride is shorter than a token's %lld elements", row);
  if (tokens == 0 || num_pages == 0) return TQ_OK;
  if (!k || !v || !slots || !k_indices || !k_scales || !v_indices || !v_scales || (signs && (!norms || !sign_matrix)))
    return tqh::fail(TQ_ERR_INVALID_ARGUMENT, "null pointer");
  rc = tqh::check_pools({k_indices, v_indices, k_scales, v_scales, signs});
  if (rc) return rc;
  const long long lanes = (long long)tokens * num_kv_heads * (head_dim / 32);
  if (lanes >= 1ll << 30) return tqh::fail(TQ_ERR_INVALID_ARGUMENT, "too many tokens in one call");
  const int size = tqh::dtype_size(dtype);
  a.pages.slots = slots;
  a.pages.num_slots = num_pages << a.pages.shift;
  a.pages.heads = num_kv_heads;
  a.pages.tokens = tokens;
  a.x[0] = k;
  a.x[1] = v;
  a.stride[0] = k_stride;
  a.stride[1] = v_stride;
  a.vec[0] = tqh::rows_aligned(k, k_stride, size);
  a.vec[1] = tqh::rows_aligned(v, v_stride, size);
  a.idx[0] = k_indices;
  a.idx[1] = v_indices;
  a.sc[0] = k_scales;
  a.sc[1] = v_scales;
  a.num_blocks = head_dim / 32;
  a.qc = make_quant_consts(codec.cb, codec.outer, codec.scale_sign);
  const bool l2 = norm_mode == kL2Norm;
  if (signs) {
    a.signs = reinterpret_cast<uint32_t *>(signs);
    a.norms = norms;
    a.rbits = sign_matrix;
    for (int i = 0; i < codec.cb.nc; i++) a.cb[i] = codec.cb.c[i];
    a.decode_factor = decode_factor();
    a.inv_sqrt_d = tqh::inv_sqrt_dim(head_dim);
    const dim3 grid((unsigned)((tokens + kVecs - 1) / kVecs), (unsigned)num_kv_heads);
    by_type(dtype, [&](auto dt) {
      auto go = [&](auto d, auto b) {
        constexpr int D = decltype(d)::value, B = decltype(b)::value, DT = decltype(dt)::value;
        if (l2) hipLaunchKernelGGL((paged_store_tq_kernel<D, B, DT, kL2Norm>), grid, dim3(Geo<D>::THREADS), 0, stream, a);
        else hipLaunchKernelGGL((paged_store_tq_kernel<D, B, DT, kMaxNorm>), grid, dim3(Geo<D>::THREADS), 0, stream, a);
      };
      auto by_bits = [&](auto d) {
        if (bits == 3) go(d, std::integral_constant<int, 3>{});
        else go(d, std::integral_constant<int, 4>{});
      };
      if (head_dim == 64) by_bits(std::integral_constant<int, 64>{});
      else if (head_dim == 128) by_bits(std::integral_constant<int, 128>{});
      else by_bits(std::integral_constant<int, 256>{});
    });
    return tqh::check_launch("paged_store_tq_kernel");
  }
  const dim3 grid((unsigned)((lanes + 255) / 256), 2);
  by_type(dtype, [&](auto dt) {
    auto go = [&](auto b, auto c) {
      constexpr int B = decltype(b)::value, C = decltype(c)::value, DT = decltype(dt)::value;
      if (l2) hipLaunchKernelGGL((paged_store_kernel<B, C, DT, kL2Norm>), grid, dim3(256), 0, stream, a);
      else hipLaunchKernelGGL((paged_store_kernel<B, C, DT, kMaxNorm>), grid, dim3(256), 0, stream, a);
    };
    using I2 = std::integral_constant<int, 2>;
    using I3 = std::integral_constant<int, 3>;
    using I4 = std::integral_constant<int, 4>;
    if (bits == 3 && codec.outlier) go(I3{}, I3{});
    else if (bits == 3) go(I3{}, I2{});
    else if (codec.outlier) go(I4{}, I4{});
    else go(I4{}, I3{});
  });
  return tqh::check_launch("paged_store_kernel");
}

extern "C" int tq_paged_load(const uint8_t *k_indices, const uint16_t *k_scales, const uint8_t *v_indices,
                             const uint16_t *v_scales, const long long *slots, int tokens, long long num_pages,
                             int num_kv_heads, int page_size, int head_dim, int bits, size_t outlier_blocks,
                             int norm_mode, void *k_out, void *v_out, int out_dtype, hipStream_t stream) {
  LoadArgs a{};
  tqh::PolarCodec codec;
  int rc = tqh::check_pages(num_pages, num_kv_heads, page_size, head_dim, bits, outlier_blocks, norm_mode,
                            a.pages.shift, codec);
  if (rc) return rc;
  if (!tqh::valid_dtype(out_dtype)) return tqh::fail(TQ_ERR_INVALID_ARGUMENT, "unknown dtype %d", out_dtype);
  if (tokens < 0) return tqh::fail(TQ_ERR_INVALID_ARGUMENT, "negative tokens");
  if (tokens == 0 || num_pages == 0) return TQ_OK;
  if (!slots || !k_indices || !k_scales || !v_indices || !v_scales || !k_out || !v_out)
    return tqh::fail(TQ_ERR_INVALID_ARGUMENT, "null pointer");
  rc = tqh::check_pools({k_indices, v_indices, k_scales, v_scales});
  if (rc) return rc;
  if (!tqh::rows_aligned(k_out, 0, 1) || !tqh::rows_aligned(v_out, 0, 1))
    return tqh::fail(TQ_ERR_INVALID_ARGUMENT, "outputs start on 16-byte boundaries");
  const long long lanes = (long long)tokens * num_kv_heads * (head_dim / 32);
  if (lanes >= 1ll << 30) return tqh::fail(TQ_ERR_INVALID_ARGUMENT, "too many tokens in one call");
  a.pages.slots = slots;
  a.pages.num_slots = num_pages << a.pages.shift;
  a.pages.heads = num_kv_heads;
  a.pages.tokens = tokens;
  a.idx[0] = k_indices;
  a.idx[1] = v_indices;
  a.sc[0] = k_scales;
  a.sc[1] = v_scales;
  a.out[0] = k_out;
  a.out[1] = v_out;
  a.num_blocks = head_dim / 32;
  a.through = 2 * lanes * 32 * tqh::dtype_size(out_dtype) > tqh::kThroughBytes;
  for (int i = 0; i < codec.cb.nc; i++) a.cb[i] = codec.cb.c[i];
  a.sgm = decode_factor();
  const dim3 grid((unsigned)((lanes + 255) / 256), 2);
  by_type(out_dtype, [&](auto dt) {
    constexpr int DT = decltype(dt)::value;
    if (bits == 3) hipLaunchKernelGGL((paged_load_kernel<3, DT>), grid, dim3(256), 0, stream, a);
    else hipLaunchKernelGGL((paged_load_kernel<4, DT>), grid, dim3(256), 0, stream, a);
  });
  return tqh::check_launch("paged_load_kernel");
}
