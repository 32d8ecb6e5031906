// Causal grouped-query attention over a cache held in 8 bits (cache8.cu):
//     o[t] = sum_j p_j sv_j cv_j / sum_j p_j,   p_j = exp(scale sk_j (q . ck_j) - max)
// over the keys j that token t sees: positions up to its own, within the window, on pages that the request still holds.
// A token that sees none gets 0.  One warp a token and head.
#include "common.cuh"
#include <float.h>

using namespace tkb;

namespace {

constexpr int MAX_PER_LANE = 8;  // head sizes up to 256

template <typename T>
__global__ void __launch_bounds__(128)
attn_kv8_kernel(const T* __restrict__ q, long long q_stride, T* __restrict__ out, long long out_stride, const int8_t* __restrict__ kcache,
                const int8_t* __restrict__ vcache, const float* __restrict__ k_scale, const float* __restrict__ v_scale,
                const int* __restrict__ q_start, const int* __restrict__ q_len, const int* __restrict__ kv_len,
                const int* __restrict__ page_indptr, const int* __restrict__ page_ids, int nh, int nkv, int hd, int ps, float scale,
                int window, int num_pages, int* __restrict__ status) {
  trigger_dependents();
  grid_dependency_wait();
  const int s = blockIdx.y, lane = threadIdx.x & 31;
  const int h = blockIdx.z;
  const int kvh = h / (nh / nkv);
  bool bad = false;
  const int* table = page_ids + page_indptr[s];
  for (int i = blockIdx.x * 4 + (threadIdx.x >> 5); i < q_len[s]; i += gridDim.x * 4) {
    const int pos = kv_len[s] - q_len[s] + i;
    const T* qr = q + (q_start[s] + i) * q_stride + (long long)h * hd;
    float qv[MAX_PER_LANE], o[MAX_PER_LANE];
#pragma unroll
    for (int e = 0; e < MAX_PER_LANE; e++) {
      const int d = lane + 32 * e;
      qv[e] = d < hd ? to_float(qr[d]) * scale : 0.f;
      o[e] = 0.f;
    }
    float m = -FLT_MAX, l = 0.f;
    for (int j = window > 0 ? max(0, pos - window + 1) : 0; j <= pos; j++) {
      const int page = checked_page(table[j / ps], num_pages, bad);
      if (page < 0) continue;
      const long long block = (long long)page * nkv + kvh;
      const int8_t* kr = kcache + (block * ps + j % ps) * hd;
      const int8_t* vr = vcache + (block * ps + j % ps) * hd;
      float dot = 0.f;
#pragma unroll
      for (int e = 0; e < MAX_PER_LANE; e++)
        if (lane + 32 * e < hd) dot = fmaf(qv[e], (float)kr[lane + 32 * e], dot);
      dot = warp_sum(dot) * k_scale[block];
      const float top = dot > m || dot != dot ? dot : m;
      const float a = expf(m - top), p = expf(dot - top);
      l = l * a + p;
      const float w = p * v_scale[block];
#pragma unroll
      for (int e = 0; e < MAX_PER_LANE; e++)
        if (lane + 32 * e < hd) o[e] = o[e] * a + w * (float)vr[lane + 32 * e];
      m = top;
    }
    T* dst = out + (q_start[s] + i) * out_stride + (long long)h * hd;
#pragma unroll
    for (int e = 0; e < MAX_PER_LANE; e++)
      if (lane + 32 * e < hd) dst[lane + 32 * e] = from_float<T>(l == 0.f ? 0.f : o[e] / l);
  }
  report_bad_page(bad, status);
}

}  // namespace

TKB_EXPORT int tkb_attn_kv8(const void* q, long long q_stride, void* out, long long out_stride, int f32, const void* kcache,
                            const void* vcache, const float* k_scale, const float* v_scale, const int* q_start, const int* q_len,
                            const int* kv_len, const int* page_indptr, const int* page_ids, int n_seqs, int max_q, int nh, int nkv, int hd,
                            int ps, float scale, int window, int num_pages, int* status, void* st_) {
  if (n_seqs <= 0 || max_q <= 0) return 0;
  if (nkv <= 0 || nh <= 0 || nh % nkv || hd <= 0 || (hd & 15) || hd > 256 || ps <= 0 || window < 0) return -2;
  if (n_seqs > 65535 || nh > 65535) return -3;
  cudaStream_t st = (cudaStream_t)st_;
  const dim3 grid((max_q + 3) / 4, n_seqs, nh);
  if (f32)
    return launch_pdl(attn_kv8_kernel<float>, grid, dim3(128), 0, st, (const float*)q, q_stride, (float*)out, out_stride,
                      (const int8_t*)kcache, (const int8_t*)vcache, k_scale, v_scale, q_start, q_len, kv_len, page_indptr, page_ids, nh,
                      nkv, hd, ps, scale, window, num_pages, status);
  return launch_pdl(attn_kv8_kernel<__nv_bfloat16>, grid, dim3(128), 0, st, (const __nv_bfloat16*)q, q_stride, (__nv_bfloat16*)out,
                    out_stride, (const int8_t*)kcache, (const int8_t*)vcache, k_scale, v_scale, q_start, q_len, kv_len, page_indptr,
                    page_ids, nh, nkv, hd, ps, scale, window, num_pages, status);
}
