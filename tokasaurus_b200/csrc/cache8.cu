// A cache of keys and values held in 8 bits: codes int8 [page, kv head, slot in page, hd] and one float32 scale for every
// page and kv head.  A number is its code times its block's scale.
//
// Writing a step's tokens: the tokens of one request that fall into one page are a SEGMENT; its first token leads it.  For a
// segment, head and side (k or v), with m = max |new numbers|:
//     s' = max(s, m * (1 / 127)),  s the block's scale so far, 0 if the segment starts in the page's first slot
//     new codes  code(x, s') = rint(x / s') held to [-127, 127], 0 where s' is 0
//     the block's other codes c -> code(c * s, s'), where s' differs from s (a scale only grows while a page is filled)
// each step rounded once in float32.  A page's first slot always starts it afresh: what an earlier request left there does
// not count.  An infinity or NaN among the numbers makes the block's scale NaN: all that is read from the block is NaN then.
// Writing the same tokens again changes nothing (their scale has been reached).
#include "common.cuh"

using namespace tkb;

namespace {

constexpr float ONE_127TH = 1.f / 127.f;

__device__ __forceinline__ int code_of(float x, float s) {
  return (int)fminf(fmaxf(rintf(__fdiv_rn(x, s)), -127.f), 127.f);
}

// Element d of a head after the rotation (half-split pairs), at angles pos * inv_freq.
template <typename T>
__device__ __forceinline__ float rotated(const T* x, int d, int half, int rot, float pos, const float* __restrict__ inv_freq) {
  if (d >= rot) return to_float(x[d]);
  const int j = d < half ? d : d - half;
  float sn, c;
  sincosf(pos * inv_freq[j], &sn, &c);
  return d < half ? to_float(x[d]) * c - to_float(x[d + half]) * sn : to_float(x[d]) * c + to_float(x[j]) * sn;
}

constexpr int W_THREADS = 256;

template <typename T>
__global__ void __launch_bounds__(W_THREADS)
rope_kv8_write_kernel(T* __restrict__ qkv, const int* __restrict__ positions, const int* __restrict__ token_seq,
                      const int* __restrict__ page_indptr, const int* __restrict__ page_ids, const float* __restrict__ inv_freq,
                      int8_t* __restrict__ kcache, int8_t* __restrict__ vcache, float* __restrict__ k_scale,
                      float* __restrict__ v_scale, int T_, int nh, int nkv, int hd, int rot, int ps, int num_pages, int write_cache,
                      int* __restrict__ status) {
  trigger_dependents();
  const int t = blockIdx.x;
  const int s = token_seq[t];
  if (s < 0) return;  // padding
  const int pos = positions[t];
  const int half = rot >> 1;
  const long long C = (long long)(nh + 2 * nkv) * hd;
  grid_dependency_wait();
  T* row = qkv + t * C;
  for (int i = threadIdx.x; i < nh * half; i += W_THREADS) {
    const int h = i / half, j = i - h * half;
    T* p = row + h * hd + j;
    const float a = to_float(p[0]), b = to_float(p[half]);
    float sn, c;
    sincosf((float)pos * inv_freq[j], &sn, &c);
    p[0] = from_float<T>(a * c - b * sn);
    p[half] = from_float<T>(b * c + a * sn);
  }
  if (!write_cache) return;
  const int slot = pos % ps;
  if (slot != 0 && t > 0 && token_seq[t - 1] == s) return;  // an earlier token leads this one's segment
  int n = 1;
  while (slot + n < ps && t + n < T_ && token_seq[t + n] == s) n++;
  const int page = page_ids[page_indptr[s] + pos / ps];
  if (page < 0 || page >= num_pages) {
    if (threadIdx.x == 0) atomicOr(status, TKB_STATUS_BAD_PAGE);
    return;
  }
  const int lane = threadIdx.x & 31;
  for (int task = threadIdx.x >> 5; task < 2 * nkv; task += W_THREADS / 32) {
    const int h = task >> 1;
    const bool is_v = task & 1;
    const T* src = row + (long long)(nh + (is_v ? nkv : 0) + h) * hd;
    const int r = is_v ? 0 : rot;
    int8_t* dst = (is_v ? vcache : kcache) + ((long long)page * nkv + h) * ps * hd;
    float* scale = (is_v ? v_scale : k_scale) + (long long)page * nkv + h;
    unsigned top = 0;
    for (int i = 0; i < n; i++)
      for (int d = lane; d < hd; d += 32)
        top = max(top, __float_as_uint(rotated(src + i * C, d, r >> 1, r, (float)(pos + i), inv_freq)) & 0x7fffffffu);
    top = __reduce_max_sync(0xffffffffu, top);
    const float old = slot == 0 ? 0.f : *scale;
    float s2 = top < 0x7f800000u ? __uint_as_float(top) * ONE_127TH : NAN;
    if (!(s2 > old)) s2 = (s2 == s2) ? old : s2;  // (a NaN stays one, whichever side it is on)
    const bool some = s2 > 0.f;
    if (s2 != old) {
      for (int i = lane; i < ps * hd; i += 32) {
        const int sl = i / hd;
        if (sl < slot || sl >= slot + n) dst[i] = some ? (int8_t)code_of((float)dst[i] * old, s2) : (int8_t)0;
      }
    }
    for (int i = 0; i < n; i++)
      for (int d = lane; d < hd; d += 32) {
        const float x = rotated(src + i * C, d, r >> 1, r, (float)(pos + i), inv_freq);
        dst[(slot + i) * hd + d] = some ? (int8_t)code_of(x, s2) : (int8_t)0;
      }
    if (lane == 0) *scale = s2;
  }
}

__global__ void __launch_bounds__(256)
read_kv8_kernel(const int8_t* __restrict__ kcache, const int8_t* __restrict__ vcache, const float* __restrict__ k_scale,
                const float* __restrict__ v_scale, const int* __restrict__ pages, float* __restrict__ k_out, float* __restrict__ v_out,
                int nkv, int block, int num_pages, int* __restrict__ status) {
  trigger_dependents();
  grid_dependency_wait();
  const int n = blockIdx.x / nkv, h = blockIdx.x % nkv;
  const bool is_v = blockIdx.y;
  const int page = pages[n];
  float* out = (is_v ? v_out : k_out) + (long long)blockIdx.x * block;
  const bool ok = page >= 0 && page < num_pages;
  if (page >= num_pages && threadIdx.x == 0) atomicOr(status, TKB_STATUS_BAD_PAGE);
  const long long at = (long long)page * nkv + h;
  const int8_t* src = (is_v ? vcache : kcache) + (ok ? at * block : 0);
  const float s = ok ? (is_v ? v_scale : k_scale)[at] : 0.f;
  for (int i = threadIdx.x * 4; i < block; i += 1024) {
    const char4 c = *reinterpret_cast<const char4*>(src + i);
    *reinterpret_cast<float4*>(out + i) = ok ? make_float4(c.x * s, c.y * s, c.z * s, c.w * s) : make_float4(0.f, 0.f, 0.f, 0.f);
  }
}

}  // namespace

// qkv [tokens, (nh + 2 nkv) hd] float32 (f32 != 0) or bfloat16, contiguous; q rotated in place, k and v to the cache.
TKB_EXPORT int tkb_rope_kv8_write(void* qkv, int f32, const int* positions, const int* token_seq, const int* page_indptr,
                                  const int* page_ids, const float* inv_freq, void* kcache, void* vcache, float* k_scale, float* v_scale,
                                  int tokens, int nh, int nkv, int hd, int rot, int ps, int num_pages, int write_cache, int* status, void* st_) {
  if (tokens <= 0) return 0;
  if (rot < 0 || rot > hd || (rot & 1) || (hd & 15) || nh <= 0 || nkv <= 0 || ps <= 0) return -2;
  cudaStream_t st = (cudaStream_t)st_;
  if (f32)
    return launch_pdl(rope_kv8_write_kernel<float>, dim3(tokens), dim3(W_THREADS), 0, st, (float*)qkv, positions, token_seq, page_indptr,
                      page_ids, inv_freq, (int8_t*)kcache, (int8_t*)vcache, k_scale, v_scale, tokens, nh, nkv, hd, rot, ps, num_pages,
                      write_cache, status);
  return launch_pdl(rope_kv8_write_kernel<__nv_bfloat16>, dim3(tokens), dim3(W_THREADS), 0, st, (__nv_bfloat16*)qkv, positions, token_seq,
                    page_indptr, page_ids, inv_freq, (int8_t*)kcache, (int8_t*)vcache, k_scale, v_scale, tokens, nh, nkv, hd, rot, ps,
                    num_pages, write_cache, status);
}

// k_out, v_out: float32 [n, nkv, block]; block = page size * head size (a multiple of 16).
TKB_EXPORT int tkb_read_kv8(const void* kcache, const void* vcache, const float* k_scale, const float* v_scale, const int* pages,
                            float* k_out, float* v_out, int n, int nkv, int block, int num_pages, int* status, void* st) {
  if (n <= 0) return 0;
  if (nkv <= 0 || block <= 0 || (block & 15)) return -2;
  if ((long long)n * nkv > 2147483647ll) return -3;
  return launch_pdl(read_kv8_kernel, dim3(n * nkv, 2), dim3(256), 0, (cudaStream_t)st, (const int8_t*)kcache, (const int8_t*)vcache,
                    k_scale, v_scale, pages, k_out, v_out, nkv, block, num_pages, status);
}
