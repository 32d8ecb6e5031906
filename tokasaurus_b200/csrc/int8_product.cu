// Products in 8-bit integers:  y[m, n] = (sum_k c[m, k] w[n, k]) * (s[m] t[n])
//
// c, s: a token's codes and scale, made here from its float32 or bfloat16 numbers (quantise_rows):
//     s = max_k |x| * (1 / 127),   c = rint(x / s) held to [-127, 127], 0 where s is 0,
// each step rounded once in float32, so that the codes do not depend on how the work is cut.  A row with an infinity or
// NaN gets the scale NaN and the codes 0: its results are NaN, those of other rows are not touched.
// w, t: an output channel's codes and scale.  The sum is a 32-bit integer, exact for K up to 132,103 (127 * 128 * K < 2^31).
#include "common.cuh"

using namespace tkb;

namespace {

constexpr float ONE_127TH = 1.f / 127.f;

// rint(x / s) with the quotient rounded as float32 division rounds it, held to [-127, 127].  x * (1 / s) is within 3e-5 of
// it, which settles all but quotients next to a half: those (2 in 10,000) are divided.
__device__ __forceinline__ int code_of(float x, float s, float inv) {
  const float t = x * inv;
  float q = rintf(t);
  if (!(fabsf(t - q) <= 0.4999f)) q = rintf(__fdiv_rn(x, s));
  return (int)fminf(fmaxf(q, -127.f), 127.f);
}

constexpr int Q_THREADS = 256;

template <typename T>
__global__ void __launch_bounds__(Q_THREADS)
quantise_rows_kernel(const T* __restrict__ x, long long ldx, int8_t* __restrict__ codes, long long ldc, float* __restrict__ scale,
                     int K) {
  __shared__ unsigned s_top[Q_THREADS / 32];
  trigger_dependents();
  grid_dependency_wait();
  const T* row = x + (long long)blockIdx.x * ldx;
  int8_t* dst = codes + (long long)blockIdx.x * ldc;
  // magnitudes as integers: NaN > infinity > every number
  unsigned top = 0;
  for (int k = threadIdx.x; k < K; k += Q_THREADS) top = max(top, __float_as_uint(to_float(row[k])) & 0x7fffffffu);
  top = __reduce_max_sync(0xffffffffu, top);
  if ((threadIdx.x & 31) == 0) s_top[threadIdx.x >> 5] = top;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < Q_THREADS / 32; i++) top = max(top, s_top[i]);
  const bool finite = top < 0x7f800000u;
  const float s = finite ? __uint_as_float(top) * ONE_127TH : NAN;
  const float inv = 1.f / s;
  const bool some = finite && s > 0.f;
  for (int k = threadIdx.x; k < K; k += Q_THREADS) dst[k] = some ? (int8_t)code_of(to_float(row[k]), s, inv) : (int8_t)0;
  if (threadIdx.x == 0) scale[blockIdx.x] = s;
}

// 64 tokens x 64 channels a block, 32 codes of K at a time through shared memory, four by four results a thread.
constexpr int TILE = 64, KSTEP = 32;

template <typename T>
__global__ void __launch_bounds__(256)
product_kernel(const int8_t* __restrict__ a, long long lda, const float* __restrict__ a_scale, const int8_t* __restrict__ w,
               long long ldw, const float* __restrict__ w_scale, T* __restrict__ out, long long ldo, int M, int N, int K, int gated) {
  __shared__ int sa[TILE][KSTEP / 4 + 1], sw[TILE][KSTEP / 4 + 1];
  __shared__ float tile[TILE][TILE + 1];
  trigger_dependents();
  grid_dependency_wait();
  const int m0 = blockIdx.y * TILE, n0 = blockIdx.x * TILE;
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  int acc[4][4] = {};
  for (int k0 = 0; k0 < K; k0 += KSTEP) {
    for (int i = threadIdx.x; i < TILE * KSTEP / 4; i += 256) {
      const int r = i / (KSTEP / 4), c = i % (KSTEP / 4), k = k0 + 4 * c;
      int va = 0, vw = 0;
      for (int e = 0; e < 4; e++)
        if (k + e < K) {
          if (m0 + r < M) va |= (int)(uint8_t)a[(m0 + r) * lda + k + e] << (8 * e);
          if (n0 + r < N) vw |= (int)(uint8_t)w[(n0 + r) * ldw + k + e] << (8 * e);
        }
      sa[r][c] = va;
      sw[r][c] = vw;
    }
    __syncthreads();
#pragma unroll
    for (int c = 0; c < KSTEP / 4; c++)
#pragma unroll
      for (int i = 0; i < 4; i++)
#pragma unroll
        for (int j = 0; j < 4; j++) acc[i][j] = __dp4a(sa[ty + 16 * i][c], sw[tx + 16 * j][c], acc[i][j]);
    __syncthreads();
  }
#pragma unroll
  for (int i = 0; i < 4; i++)
#pragma unroll
    for (int j = 0; j < 4; j++) {
      const int m = m0 + ty + 16 * i, n = n0 + tx + 16 * j;
      if (m < M && n < N) tile[ty + 16 * i][tx + 16 * j] = (float)acc[i][j] * (a_scale[m] * w_scale[n]);
    }
  __syncthreads();
  for (int i = threadIdx.x; i < TILE * TILE; i += 256) {
    const int r = i / TILE, c = i % TILE, m = m0 + r, n = n0 + c;
    if (m >= M || n >= N) continue;
    if (!gated) {
      out[m * ldo + n] = from_float<T>(tile[r][c]);
    } else if ((c & 8) == 0) {
      const float g = tile[r][c], u = tile[r][c + 8];
      out[m * ldo + (n >> 4) * 8 + (c & 7)] = from_float<T>(g / (1.f + expf(-g)) * u);
    }
  }
}

}  // namespace

// codes [M, ldc] int8 and scale [M] of x [M, K] (float32: f32 != 0, else bfloat16; row stride ldx elements).
TKB_EXPORT int tkb_quantise_rows(const void* x, long long ldx, int f32, void* codes, long long ldc, void* scale, int M, int K, void* st_) {
  if (M <= 0) return 0;
  if (K <= 0) return -2;
  cudaStream_t st = (cudaStream_t)st_;
  if (f32)
    return launch_pdl(quantise_rows_kernel<float>, dim3(M), dim3(Q_THREADS), 0, st, (const float*)x, ldx, (int8_t*)codes, ldc, (float*)scale, K);
  return launch_pdl(quantise_rows_kernel<__nv_bfloat16>, dim3(M), dim3(Q_THREADS), 0, st, (const __nv_bfloat16*)x, ldx, (int8_t*)codes, ldc, (float*)scale, K);
}

// out [M, N] (gated: [M, N / 2], rows of w interleaving gate and up in eights) float32 or bfloat16, row stride ldo elements.
TKB_EXPORT int tkb_int8_product(const void* a, long long lda, const void* a_scale, const void* w, long long ldw, const void* w_scale,
                                void* out, long long ldo, int f32, int M, int N, int K, int gated, int* status, void* st_) {
  if (M <= 0 || N <= 0) return 0;
  if (K <= 0 || K > 132103 || (gated && (N & 15))) return -2;
  if ((M + TILE - 1) / TILE > 65535) return -3;
  cudaStream_t st = (cudaStream_t)st_;
  const dim3 grid((N + TILE - 1) / TILE, (M + TILE - 1) / TILE);
  if (f32)
    return launch_pdl(product_kernel<float>, grid, dim3(256), 0, st, (const int8_t*)a, lda, (const float*)a_scale, (const int8_t*)w, ldw,
                      (const float*)w_scale, (float*)out, ldo, M, N, K, gated);
  return launch_pdl(product_kernel<__nv_bfloat16>, grid, dim3(256), 0, st, (const int8_t*)a, lda, (const float*)a_scale, (const int8_t*)w, ldw,
                    (const float*)w_scale, (__nv_bfloat16*)out, ldo, M, N, K, gated);
}
