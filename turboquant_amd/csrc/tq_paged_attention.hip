// tq_paged_attention.hip -- one new token per request over its pages.
//
// One workgroup a (request, query head): 256 tokens at a time, a lane scores
// one token against the rotated query (keys are never inverse-rotated), the
// softmax runs on with a rescale, and a lane of every element sums the values
// in the rotated domain; the inverse rotation follows once.
#include "tq_mfma.h"
#include "tq_paged.h"

namespace {

using namespace tqm;

struct PagedArgs {
  const void *q;
  int q_dtype;
  const uint8_t *k_idx, *v_idx;
  const uint16_t *k_sc, *v_sc;
  const uint32_t *signs;
  const uint16_t *norms;
  const uint32_t *rbits;
  const int *table, *lens;
  int width, heads, kv_heads, head_dim, shift, max_len;
  long long num_pages;
  float scale, qjl_c, inv_sqrt_d;
  float cb[16];
  void *out;
  int out_dtype;
};

template <int BITS>
__device__ __forceinline__ int code_at(const uint8_t *rec, int e) {
  const int pos = e * BITS;
  const int w = rec[pos >> 3] | ((pos & 7) + BITS > 8 ? rec[(pos >> 3) + 1] << 8 : 0);
  return (w >> (pos & 7)) & ((1 << BITS) - 1);
}

template <int BITS>
__global__ __launch_bounds__(256) void paged_decode_kernel(PagedArgs a) {
  __shared__ float s_q[256], s_rq[256], s_x[256], s_p[256], s_cb[16], s_red[8];
  __shared__ long long s_rec[256];
  const int tid = threadIdx.x, h = blockIdx.x, b = blockIdx.y, d = a.head_dim, nb = d / 32;
  const int g = h / (a.heads / a.kv_heads);
  const long long q0 = ((long long)b * a.heads + h) * d;
#pragma unroll
  for (int i = 0; i < 16; i++)
    if (tid == i) s_cb[i] = a.cb[i];
  float x = 0.f;
  if (tid < d) {
    if (a.q_dtype == kF32) x = static_cast<const float *>(a.q)[q0 + tid];
    else if (a.q_dtype == kBF16) x = bf16_to_f32(static_cast<const uint16_t *>(a.q)[q0 + tid]);
    else x = f16_to_f32(static_cast<const uint16_t *>(a.q)[q0 + tid]);
  }
  s_x[tid] = x;
  s_q[tid] = wht32_lanes(x, tid & 31) * (decode_sign(tid & 31) * kInvSqrt32);
  __syncthreads();
  if (a.signs && tid < d) {
    float r = 0.f;
    for (int c = 0; c < d; c++) r += (a.rbits[tid * nb + (c >> 5)] >> (c & 31)) & 1 ? -s_x[c] : s_x[c];
    s_rq[tid] = r * a.inv_sqrt_d;
  }
  const int len = min(max(a.lens[b], 0), a.max_len);
  float m = -INFINITY, l = 0.f, acc = 0.f;
  for (int t0 = 0; t0 < len; t0 += 256) {
    __syncthreads();
    const int t = t0 + tid;
    long long rec = -1;
    if (t < len) {
      const int page = a.table[(long long)b * a.width + (t >> a.shift)];
      if (page >= 0 && page < a.num_pages)
        rec = (((long long)page * a.kv_heads + g) << a.shift) + (t & ((1 << a.shift) - 1));
    }
    float s = -INFINITY;
    if (rec >= 0) {
      const uint8_t *p = a.k_idx + rec * (d * BITS / 8);
      s = 0.f;
      for (int qb = 0; qb < nb; qb++) {
        float y = 0.f;
        for (int j = 0; j < 32; j++) y += s_cb[code_at<BITS>(p, 32 * qb + j)] * s_q[32 * qb + j];
        s += y * fabsf(f16_to_f32(a.k_sc[rec * nb + qb]));
      }
      if (a.signs) {
        float y = 0.f;
        for (int j = 0; j < d; j++) y += (a.signs[rec * nb + (j >> 5)] >> (j & 31)) & 1 ? s_rq[j] : -s_rq[j];
        s += y * (f16_to_f32(a.norms[rec]) * a.qjl_c);
      }
      s *= a.scale * kLog2e;
    }
    s_rec[tid] = rec;
    float mx = wave_max(s);
    if ((tid & 63) == 0) s_red[tid >> 6] = mx;
    __syncthreads();
    mx = fmaxf(fmaxf(s_red[0], s_red[1]), fmaxf(s_red[2], s_red[3]));
    const float mn = fmaxf(m, mx), f = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - mn);
    const float p = s == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(s - mn);
    s_p[tid] = p;
    const float ws = wave_sum(p);
    if ((tid & 63) == 0) s_red[4 + (tid >> 6)] = ws;
    __syncthreads();
    l = l * f + ((s_red[4] + s_red[5]) + (s_red[6] + s_red[7]));
    m = mn;
    if (tid < d) {
      acc *= f;
      for (int i = 0; i < 256 && t0 + i < len; i++) {
        const long long r = s_rec[i];
        if (r < 0) continue;
        const float v = s_cb[code_at<BITS>(a.v_idx + r * (d * BITS / 8), tid)];
        acc += s_p[i] * (v * fabsf(f16_to_f32(a.v_sc[r * nb + (tid >> 5)])));
      }
    }
  }
  const float v = wht32_lanes(acc * decode_sign(tid & 31), tid & 31);
  const float o = l > 0.f ? v * kInvSqrt32 / l : 0.f;
  if (tid < d) {
    if (a.out_dtype == kF32) static_cast<float *>(a.out)[q0 + tid] = o;
    else if (a.out_dtype == kBF16) static_cast<uint16_t *>(a.out)[q0 + tid] = f32_to_bf16(o);
    else static_cast<uint16_t *>(a.out)[q0 + tid] = f32_to_f16(o);
  }
}

}  // namespace

extern "C" int tq_paged_decode_attention(const void *q, int q_dtype, const uint8_t *k_indices,
                                         const uint16_t *k_scales, const uint8_t *v_indices, const uint16_t *v_scales,
                                         const uint8_t *signs, const uint16_t *norms, const uint32_t *sign_matrix,
                                         const int *block_table, int table_width, const int *kv_lens, int batch,
                                         int num_heads, int num_kv_heads, int head_dim, int bits,
                                         size_t outlier_blocks, int norm_mode, int page_size, long long num_pages,
                                         int max_kv_len, float softmax_scale, void *out, int out_dtype,
                                         void *workspace, size_t workspace_bytes, hipStream_t stream) {
  PagedArgs a{};
  tqh::PolarCodec codec;
  const int rc = tqh::check_pages(num_pages, num_kv_heads, page_size, head_dim, bits, outlier_blocks, norm_mode,
                                  a.shift, codec);
  if (rc) return rc;
  if (head_dim != 32 && head_dim != 64 && head_dim != 128 && head_dim != 256)
    return tqh::fail(TQ_ERR_INVALID_ARGUMENT, "fused decode attention supports head_dim 32, 64, 128 or 256, got %d",
                     head_dim);
  if (signs && head_dim == 32)
    return tqh::fail(TQ_ERR_INVALID_ARGUMENT, "the QJL-corrected decode takes head_dim 64, 128 or 256");
  if (signs && codec.outlier)
    return tqh::fail(TQ_ERR_INVALID_ARGUMENT, "QJL correction applies to the standard codebook (outlier_blocks 0)");
  if (num_heads <= 0 || num_heads % num_kv_heads != 0)
    return tqh::fail(TQ_ERR_INVALID_ARGUMENT, "num_heads (%d) must be a multiple of num_kv_heads (%d)", num_heads,
                     num_kv_heads);
  if (!tqh::valid_dtype(q_dtype) || !tqh::valid_dtype(out_dtype))
    return tqh::fail(TQ_ERR_INVALID_ARGUMENT, "unknown dtype");
  if (batch < 0 || batch > 65535) return tqh::fail(TQ_ERR_INVALID_ARGUMENT, "batch %d outside 0 to 65,535", batch);
  if (table_width < 0 || max_kv_len < 0 || max_kv_len > (long long)table_width << a.shift)
    return tqh::fail(TQ_ERR_INVALID_ARGUMENT, "max_kv_len %d exceeds a table row of %d pages", max_kv_len, table_width);
  if (batch == 0) return TQ_OK;
  if (!q || !out || !kv_lens || !k_indices || !k_scales || !v_indices || !v_scales || (max_kv_len && !block_table) ||
      (signs && (!norms || !sign_matrix)) || !workspace)
    return tqh::fail(TQ_ERR_INVALID_ARGUMENT, "null pointer");
  const size_t need = tq_attention_workspace_size(batch, num_heads, num_kv_heads, head_dim, max_kv_len);
  if (workspace_bytes < need)
    return tqh::fail(TQ_ERR_INVALID_ARGUMENT, "workspace too small: %zu < %zu", workspace_bytes, need);
  a.q = q;
  a.q_dtype = q_dtype;
  a.k_idx = k_indices;
  a.k_sc = k_scales;
  a.v_idx = v_indices;
  a.v_sc = v_scales;
  a.signs = reinterpret_cast<const uint32_t *>(signs);
  a.norms = norms;
  a.rbits = sign_matrix;
  a.table = block_table;
  a.lens = kv_lens;
  a.width = table_width;
  a.heads = num_heads;
  a.kv_heads = num_kv_heads;
  a.head_dim = head_dim;
  a.max_len = max_kv_len;
  a.num_pages = num_pages;
  a.scale = softmax_scale;
  a.qjl_c = tq_qjl_bias_scale(head_dim);
  a.inv_sqrt_d = tqh::inv_sqrt_dim(head_dim);
  for (int i = 0; i < codec.cb.nc; i++) a.cb[i] = codec.cb.c[i];
  a.out = out;
  a.out_dtype = out_dtype;
  const dim3 grid((unsigned)num_heads, (unsigned)batch);
  if (bits == 3) hipLaunchKernelGGL((paged_decode_kernel<3>), grid, dim3(256), 0, stream, a);
  else hipLaunchKernelGGL((paged_decode_kernel<4>), grid, dim3(256), 0, stream, a);
  return tqh::check_launch("paged_decode_kernel");
}
