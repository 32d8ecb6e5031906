// Causal grouped-query attention over a cache held in 8 bits (cache8.cu); compile with -DTKB_HD (a multiple of 16 to 256):
//     o[t] = sum_j p_j sv_j cv_j / sum_j p_j,   p_j = exp(scale sk_j (q . ck_j) - max)
// over the keys j that token t sees: positions up to its own, within the window, on pages that the request still holds.
// A token that sees none gets 0.
//
// Any mix of single tokens and portions.  The (token, head) pairs of one request and kv head are COLUMNS; a block takes 8 or 16
// of them (NT tiles of 8) and walks keys in tiles of 64, which a fifth warp brings into a ring: codes by TMA, a box a page
// (swizzled, so that the reads below meet no bank twice), or by plain bulk copies where pages or heads have other sizes; beside
// them each key's scale, the logarithm of its value's scale, and its position.  Each of four warps takes 16 keys of a tile:
//     S^T = K Q^T    mma.sync 16 keys x 8 columns x 32 in 8-bit integers: the cache's codes go in as they lie there, a query as
//                    two pieces (three in float32 steps) of a 16-bit (24-bit) fixed-point number whose unit is its largest / 32,512
//                    (/ 8,323,072).  The sums are exact; the rounding is 2^-16 of a query's largest number
//     O^T += V^T W   mma.sync 16 numbers x 8 columns x 16 in halves, W = 2^(s + log2 sv - M): the values' scales are in the
//                    weights, and a code is made a half exactly (its bits under an exponent of 2^10, less 1,152)
// Keys on the rows: 16 of them fill an instruction whose 8 columns a group of heads fills, where queries as rows would leave
// three quarters of the products empty.  Scores, sums and output are float32.  s and s + log2 sv have references of their own
// (m and M; a column's largest so far, moved when topped by 2^8): weights are at most 2^8 in half precision whatever the
// scales are, and lose nothing that the largest of them would not drown.  In float32 steps weights go in as two halves (22 bits).
//
// Work is cut on the device: the tiles of all items (request, column tile) stand in a row, and each of the blocks of a kv head
// takes an even share of them, whatever the requests' lengths are; what a share holds of an item that it does not hold whole
// is left as (O, M, m, l) and put together by a second small kernel, in the order of the shares (same bits every time).
// For short contexts shares are rounded to whole items and the second kernel is not launched.
// Every wait is bounded (TKB_STATUS_WAIT_TIMEOUT).
#include "tcgen05.cuh"
#include "per_device.h"
#include <cuda_fp16.h>

#ifndef TKB_HD
#error "compile with -DTKB_HD=<head size>"
#endif

using namespace tkb5;

namespace {

constexpr int HD = TKB_HD;
static_assert(HD % 16 == 0 && HD >= 16 && HD <= 256, "head size");
constexpr int BKV = 64;              // keys a tile
constexpr int WARPS = 4;             // 16 keys of a tile each
constexpr int THREADS = (WARPS + 1) * 32;
constexpr int KV_BYTES = BKV * HD;
constexpr int STAGES = HD <= 64 ? 4 : HD <= 128 ? 3 : 2;
constexpr int DTILES = HD / 16;      // 16-row tiles of O^T; words of codes that a lane takes of a key
constexpr int KSTEPS = (HD + 31) / 32;  // products along the head size
constexpr bool SWIZZLES = HD == 64 || HD == 128;
constexpr float SLACK = 8.f;
constexpr float LOWEST = -1e30f;  // a reference before the first key

__host__ __device__ constexpr int max_nt() { return HD <= 128 ? 2 : 1; }

template <typename T, int NT> struct Layout {
  static constexpr int QP = sizeof(T) == 4 ? 3 : 2;  // pieces of a query
  static constexpr int WP = sizeof(T) == 4 ? 2 : 1;  // pieces of a weight
  static constexpr int COLS = 8 * NT;
  static constexpr int RING = 2 * STAGES * KV_BYTES;
  static constexpr int QF = QP * KSTEPS * NT * 32 * 8;   // queries as the instructions take them
  static constexpr int OUT = COLS * (HD + 4) * 4;            // output of the four warps together
  static constexpr int BYTES = 1024 + RING + QF + OUT;
};

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ void bulk_copy(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(smem_u32(dst)), "l"(src),
               "r"(bytes), "r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma8(int (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
// The codes in bytes 0 and 2 of x as two halves: 0x64cc with the sign bit turned is 1152 + c.
__device__ __forceinline__ uint32_t halves(uint32_t x) {
  const uint32_t y = (x & 0x00ff00ffu) ^ 0x64806480u;
  const __half2 h = __hsub2(*reinterpret_cast<const __half2*>(&y), __floats2half2_rn(1152.f, 1152.f));
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t pack_half(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
// what of two numbers their halves leave over, as halves
__device__ __forceinline__ uint32_t rest_half(uint32_t h, float lo, float hi) {
  const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h));
  return pack_half(lo - f.x, hi - f.y);
}
// The key (of a warp's 16) in row r of the products: rows 2c and 2c + 1 of a lane group stand in different halves of the
// swizzle, so that neither the reads of K (rows next to one another) nor those of V (every second row) meet a bank twice.
__device__ __forceinline__ int key_of_row(int r) { return (r & 8) | ((r & 1) ? (r & 6) ^ 5 : r & 6); }

// O / l under their references.  Nothing seen: zeros.  Weights that were all zero (values' scales of zero) leave M where it was.
__device__ __forceinline__ float last_factor(float M, float m, float l) {
  return l == 0.f ? 0.f : M == LOWEST ? 1.f : ex2(M - m) / l;
}

struct Args {
  const void* q;
  void* out;
  const int8_t *kcache, *vcache;
  const float *k_scale, *v_scale;
  const int *q_start, *q_len, *kv_len, *page_indptr, *page_ids;
  float* parts;          // [kv heads][blocks][2][Layout::COLS][HD + 4]: O, M, m, l
  int* base;             // [requests]: where a request's tiles start in the row of all tiles; [requests]: how many there are
  long long q_stride, out_stride;
  int n_seqs, group, nkv, ps, ps_shift, window, num_pages, which, whole, tma_rows;
  float scale_log2;
  int* status;
};
constexpr int SINGLE = 1, PORTION = 2;  // `which`

// One request's part of the work.
struct Request {
  int s, q_len, kv_len, col_tiles, k0, tiles;
  __device__ __forceinline__ bool load(const Args& a, int s_, int cols) {
    s = s_;
    q_len = a.q_len[s];
    kv_len = a.kv_len[s];
    if (q_len <= 0 || !(a.which & (q_len == 1 ? SINGLE : PORTION))) return false;
    col_tiles = (q_len * a.group + cols - 1) / cols;
    const int first = a.window > 0 ? max(0, kv_len - q_len - a.window + 1) : 0;
    k0 = first & ~(BKV - 1);
    tiles = max(1, (kv_len - k0 + BKV - 1) / BKV);
    return true;
  }
  __device__ __forceinline__ int work() const { return col_tiles * tiles; }
};

// The row of all tiles in `n` even shares: the first `rest` of them hold one tile more.
struct Shares {
  int each, rest;
  __device__ __forceinline__ Shares(int total, int n) : each(total / n), rest(total % n) {}
  __device__ __forceinline__ int start(int b) const { return b * each + min(b, rest); }
  // the share that holds tile x
  __device__ __forceinline__ int of(int x) const {
    const int longer = rest * (each + 1);
    return x < longer ? x / (each + 1) : rest + (x - longer) / max(each, 1);
  }
};

// A block's share as it is walked: item after item, tile after tile.
struct Walk {
  Request r;
  int ct, tile;          // tile: the next one of this item
  int tile_end;          // one past the last one of this item in the share
  int at, end;           // in the row of all tiles
  bool live, opens;      // opens: the share starts with this item
  __device__ __forceinline__ void clip() { tile_end = end - at < r.tiles - tile ? tile + (end - at) : r.tiles; }
  __device__ __forceinline__ void next_item(const Args& a, int cols) {
    at += tile_end - tile;
    opens = false;
    live = at < end;
    if (!live) return;
    tile = 0;
    if (++ct == r.col_tiles) {
      ct = 0;
      int s = r.s + 1;
      while (s < a.n_seqs && !r.load(a, s, cols)) s++;
      if (s >= a.n_seqs) { live = false; return; }
    }
    clip();
  }
};

template <typename T, int NT>
__global__ void __launch_bounds__(THREADS, HD <= 64 ? 4 : HD <= 128 ? 3 : 1)
attn_kv8_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, const Args a) {
  using L = Layout<T, NT>;
  constexpr int COLS = L::COLS, QP = L::QP, WP = L::WP;
  extern __shared__ unsigned char smem_raw[];
  __shared__ __align__(8) uint64_t full[STAGES], empty[STAGES];
  __shared__ float s_sk[STAGES][BKV], s_lsv[STAGES][BKV];
  __shared__ int s_pos[STAGES][BKV];
  __shared__ float s_qs[COLS], s_M[WARPS][COLS], s_m[WARPS][COLS], s_l[WARPS][COLS];
  __shared__ int s_scan[THREADS / 32], s_offset, s_seq;
  __shared__ bool s_whole[STAGES];  // every key of the tile is there
  __shared__ int failed;
  unsigned char* ring = reinterpret_cast<unsigned char*>(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  uint32_t* qf = reinterpret_cast<uint32_t*>(ring + L::RING);
  float* s_out = reinterpret_cast<float*>(ring + L::RING + L::QF);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int kvh = blockIdx.y;
  trigger_dependents();
  if (threadIdx.x == 0) {
    for (int i = 0; i < STAGES; i++) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], WARPS);
    }
    failed = 0;
    s_seq = -1;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  grid_dependency_wait();

  // ---------------- this block's share of the row of all tiles
  const int per = (a.n_seqs + THREADS - 1) / THREADS;
  const int lo = min(a.n_seqs, (int)threadIdx.x * per), hi = min(a.n_seqs, lo + per);
  int mine = 0;
  Request rq;
  for (int s = lo; s < hi; s++)
    if (rq.load(a, s, COLS)) mine += rq.work();
  int before = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int v = __shfl_up_sync(0xffffffffu, before, o);
    if (lane >= o) before += v;
  }
  if (lane == 31) s_scan[warp] = before;
  __syncthreads();
  int total = 0;
  before -= mine;
#pragma unroll
  for (int i = 0; i < THREADS / 32; i++) {
    if (i < warp) before += s_scan[i];
    total += s_scan[i];
  }
  const Shares shares(total, gridDim.x);
  const int start = shares.start(blockIdx.x), end = shares.start(blockIdx.x + 1);
  if (start >= before && start < before + mine) {
    int at = before;
    for (int s = lo; s < hi; s++)
      if (rq.load(a, s, COLS)) {
        if (start < at + rq.work()) {
          s_seq = s;
          s_offset = start - at;
          break;
        }
        at += rq.work();
      }
  }
  if (!a.whole && blockIdx.x == 0 && blockIdx.y == 0) {
    // for the second kernel
    int at = before;
    for (int s = lo; s < hi; s++) {
      a.base[s] = at;
      if (rq.load(a, s, COLS)) at += rq.work();
    }
    if (threadIdx.x == 0) a.base[a.n_seqs] = total;
  }
  __syncthreads();
  Walk w;
  w.live = s_seq >= 0 && start < end;
  if (w.live) {
    w.r.load(a, s_seq, COLS);
    w.ct = s_offset / w.r.tiles;
    w.tile = s_offset - w.ct * w.r.tiles;
    w.at = start;
    w.end = end;
    w.opens = true;
    w.clip();
    if (a.whole) {
      // a share holds the items that start in it, whole
      if (w.tile > 0) w.next_item(a, COLS);
      if (w.live) {
        w.end = 0x7fffffff;
        w.clip();
      }
    }
  }
  // (whole items: the share is over with the first item that starts behind `end`)
  auto more = [&]() { return w.live && (!a.whole || w.at < end); };

  // keys that some column of the item sees, as tiles of the item
  auto visible = [&](int& t_lo, int& t_hi) {
    const int tok_lo = w.ct * COLS / a.group, tok_hi = min(w.r.q_len - 1, (w.ct * COLS + COLS - 1) / a.group);
    const int p0 = w.r.kv_len - w.r.q_len;
    const int first = a.window > 0 ? max(0, p0 + tok_lo - a.window + 1) : 0;
    t_lo = max(w.tile, (first - w.r.k0) / BKV);
    t_hi = min(w.tile_end, (p0 + tok_hi - w.r.k0) / BKV + 1);
  };

  if (warp == WARPS) {
    // ---------------- keys and values into the ring
    // Pages come in windows of 64: each lane holds two of them with their scales, and the ids of the window behind, so that
    // a tile waits for no lookup.
    uint32_t it = 0;
    bool ok = true, bad = false;
    for (; more() && ok; w.next_item(a, COLS)) {
      int t_lo, t_hi;
      visible(t_lo, t_hi);
      const int* table = a.page_ids + a.page_indptr[w.r.s];
      const int last_page = (w.r.kv_len - 1) / a.ps;
      auto page_at = [&](int p) { return p <= last_page ? __ldg(table + p) : -1; };
      int base = -1, id[2], next_id[2] = {-1, -1};
      float sk[2], lsv[2];
      for (int t = t_lo; t < t_hi; t++, it++) {
        const int st = it % STAGES;
        const int key0 = w.r.k0 + t * BKV, key1 = min(key0 + BKV, w.r.kv_len);
        const int page0 = a.ps_shift >= 0 ? key0 >> a.ps_shift : key0 / a.ps;
        const int page1 = a.ps_shift >= 0 ? (key1 - 1) >> a.ps_shift : (key1 - 1) / a.ps;
        const bool fresh = base < 0 || page1 >= base + 64;
        if (fresh) {
          const bool follows = base >= 0 && page0 == base + 64;
          base = page0;
#pragma unroll
          for (int i = 0; i < 2; i++) {
            id[i] = checked_page(follows ? next_id[i] : page_at(base + lane + 32 * i), a.num_pages, bad);
            const long long block = (long long)max(id[i], 0) * a.nkv + kvh;
            sk[i] = a.k_scale[block];
            lsv[i] = a.v_scale[block];
            next_id[i] = page_at(base + 64 + lane + 32 * i);
          }
        }
        if (it >= STAGES && !mbar_wait(&empty[st], ((it / STAGES) - 1) & 1)) { ok = false; break; }
        unsigned char* dk = ring + st * 2 * KV_BYTES;
        uint32_t bytes = 0;
#pragma unroll
        for (int i = 0; i < 2; i++) {
          const int p = page0 + lane + 32 * i, at = min(p - base, 63);
          const int id0 = __shfl_sync(0xffffffffu, id[0], at & 31), id1 = __shfl_sync(0xffffffffu, id[1], at & 31);
          const int page = at < 32 ? id0 : id1;
          if (p <= page1 && page >= 0) {
            const int from = max(key0, p * a.ps);
            const long long row = ((long long)page * a.nkv + kvh) * a.ps + (from - p * a.ps);
            unsigned char* dst = dk + (from - key0) * HD;
            if (a.tma_rows > 0) {
              tma_load_2d(dst, &map_k, &full[st], 0, (int)row);
              tma_load_2d(dst + KV_BYTES, &map_v, &full[st], 0, (int)row);
              bytes += 2 * HD * a.tma_rows;
            } else {
              const uint32_t n = (min(key1, (p + 1) * a.ps) - from) * HD;
              bulk_copy(dst, a.kcache + row * HD, n, &full[st]);
              bulk_copy(dst + KV_BYTES, a.vcache + row * HD, n, &full[st]);
              bytes += 2 * n;
            }
          }
        }
        // (the codes are on their way; the scales of a window's first tile may still be)
        if (fresh) lsv[0] = log2f(lsv[0]), lsv[1] = log2f(lsv[1]);
        bool there = true;
#pragma unroll
        for (int i = 0; i < 2; i++) {
          const int key = key0 + lane + 32 * i;
          const int at = min((a.ps_shift >= 0 ? key >> a.ps_shift : key / a.ps) - base, 63);
          const int id0 = __shfl_sync(0xffffffffu, id[0], at & 31), id1 = __shfl_sync(0xffffffffu, id[1], at & 31);
          const float sk0 = __shfl_sync(0xffffffffu, sk[0], at & 31), sk1 = __shfl_sync(0xffffffffu, sk[1], at & 31);
          const float lv0 = __shfl_sync(0xffffffffu, lsv[0], at & 31), lv1 = __shfl_sync(0xffffffffu, lsv[1], at & 31);
          const bool real = (at < 32 ? id0 : id1) >= 0 && key < key1;
          s_sk[st][lane + 32 * i] = at < 32 ? sk0 : sk1;
          s_lsv[st][lane + 32 * i] = at < 32 ? lv0 : lv1;
          s_pos[st][lane + 32 * i] = real ? key : 0x7fffffff;
          there &= real;
        }
        there = __all_sync(0xffffffffu, there);
        bytes = __reduce_add_sync(0xffffffffu, bytes);
        __syncwarp();
        if (lane == 0) {
          s_whole[st] = there;
          if (bytes) mbar_expect_tx(&full[st], bytes);
          else mbar_arrive(&full[st]);
        }
      }
    }
    if (!ok) failed = 1;
    report_bad_page(bad, a.status);
  } else {
    // ---------------- scores, weights, output
    const int g = lane >> 2, c = lane & 3;
    const int row0 = warp * 16 + key_of_row(g);  // this lane's key rows of a tile: row0, row0 + 8
    uint32_t it = 0;
    bool ok = true;
    for (; more(); w.next_item(a, COLS)) {
      const int cols = w.r.q_len * a.group, col0 = w.ct * COLS, p0 = w.r.kv_len - w.r.q_len;
      asm volatile("bar.sync 1, 128;" ::: "memory");  // the item before is through with the queries and s_out
      for (int j = warp; j < COLS; j += WARPS) {
        const int col = col0 + j;
        const bool real = col < cols;
        const T* src = reinterpret_cast<const T*>(a.q) + (a.q_start[w.r.s] + (real ? col / a.group : 0)) * a.q_stride +
                       (long long)(kvh * a.group + (real ? col % a.group : 0)) * HD;
        constexpr int N4 = (HD / 4 + 31) / 32;  // four numbers (a word of codes) a lane and turn
        float v[N4][4];
        unsigned top = 0;
#pragma unroll
        for (int i = 0; i < N4; i++)
#pragma unroll
          for (int e = 0; e < 4; e++) {
            const int d = (lane + 32 * i) * 4 + e;
            v[i][e] = real && d < HD ? to_float(src[d]) : 0.f;
            top = max(top, __float_as_uint(v[i][e]) & 0x7fffffffu);
          }
        top = __reduce_max_sync(0xffffffffu, top);
        // by a power of two to [1, 2) (what is below 2^-126 stays there), then to the fixed point's unit
        const int e = max(1, (int)(top >> 23)) - 127;
        const float down = __uint_as_float(e == 127 ? 0x00400000u : (unsigned)(127 - e) << 23), up = __uint_as_float(e == -126 ? 0x00800000u : (unsigned)(127 + e) << 23);
        const float most = __uint_as_float(top) * down;
        const float units = QP == 3 ? 8323072.f : 32512.f;
        const bool some = top > 0 && top < 0x7f800000u;
        const float f = some ? units / most : 0.f;
        if (lane == 0) s_qs[j] = top < 0x7f800000u ? a.scale_log2 * (most / units) * up : NAN;
#pragma unroll
        for (int i = 0; i < N4; i++) {
          const int word = lane + 32 * i;
          if (word < HD / 4) {
            uint32_t piece[QP] = {};
#pragma unroll
            for (int b = 0; b < 4; b++) {
              int x = some ? __float2int_rn(v[i][b] * down * f) : 0;
#pragma unroll
              for (int p = QP - 1; p >= 0; p--) {
                const int low = p == 0 ? x : (int)(int8_t)(x & 0xff);
                piece[p] |= (uint32_t)(low & 0xff) << (8 * b);
                x = (x - low) >> 8;
              }
            }
            // which of a lane's words the word is, and which lane's
            const int u = HD % 64 == 0 ? (word >> 4) * 4 + (word & 3) : word >> 2, cc = HD % 64 == 0 ? (word >> 2) & 3 : word & 3;
#pragma unroll
            for (int p = 0; p < QP; p++) qf[(((p * KSTEPS + (u >> 1)) * NT + (j >> 3)) * 32 + (j & 7) * 4 + cc) * 2 + (u & 1)] = piece[p];
          }
        }
      }
      asm volatile("bar.sync 1, 128;" ::: "memory");
      float qs[NT][2], m[NT][2], M[NT][2], l[NT][2], o[DTILES][NT][4];
      int pos[NT][2];  // the last key that a column sees (columns behind the last: as it)
#pragma unroll
      for (int n = 0; n < NT; n++)
#pragma unroll
        for (int e = 0; e < 2; e++) {
          const int j = n * 8 + 2 * c + e;
          qs[n][e] = s_qs[j];
          pos[n][e] = p0 + min(col0 + j, cols - 1) / a.group;
          m[n][e] = M[n][e] = LOWEST;
          l[n][e] = 0.f;
        }
#pragma unroll
      for (int k = 0; k < DTILES; k++)
#pragma unroll
        for (int n = 0; n < NT; n++)
#pragma unroll
          for (int e = 0; e < 4; e++) o[k][n][e] = 0.f;

      uint2 q_own[NT == 1 ? QP * KSTEPS : 1];  // one column tile's queries stay in registers
      if (NT == 1) {
#pragma unroll
        for (int i = 0; i < (NT == 1 ? QP * KSTEPS : 1); i++) q_own[i] = reinterpret_cast<const uint2*>(qf)[i * 32 + lane];
      }
      int t_lo, t_hi;
      visible(t_lo, t_hi);
      // tiles that every column sees whole, if their pages are there
      const int whole_lo = a.window > 0 ? p0 + min(w.r.q_len - 1, (col0 + COLS - 1) / a.group) - a.window + 1 : 0;
      const int whole_hi = p0 + col0 / a.group - BKV + 1;
      for (int t = t_lo; t < t_hi; t++, it++) {
        const int st = it % STAGES, key0 = w.r.k0 + t * BKV;
        ok = ok && mbar_wait(&full[st], (it / STAGES) & 1);
        if (!ok) break;
        const unsigned char* kt = ring + st * 2 * KV_BYTES;
        const unsigned char* vt = kt + KV_BYTES;
        [[maybe_unused]] const bool swz = SWIZZLES && a.tma_rows > 0;
        // S^T
        uint32_t k0[DTILES + 1], k1[DTILES + 1];
        if constexpr (HD % 64 == 0) {
          // the swizzle of rows of 128 (64) bytes: 16-byte chunks exclusive-or the row (half the row)
          const int x = !swz ? 0 : HD == 128 ? row0 & 7 : (row0 >> 1) & 3;
#pragma unroll
          for (int i = 0; i < HD / 64; i++) {
            const uint4 u = *reinterpret_cast<const uint4*>(kt + row0 * HD + (((4 * i + c) ^ x) << 4));
            const uint4 v = *reinterpret_cast<const uint4*>(kt + (row0 + 8) * HD + (((4 * i + c) ^ x) << 4));
            k0[4 * i] = u.x, k0[4 * i + 1] = u.y, k0[4 * i + 2] = u.z, k0[4 * i + 3] = u.w;
            k1[4 * i] = v.x, k1[4 * i + 1] = v.y, k1[4 * i + 2] = v.z, k1[4 * i + 3] = v.w;
          }
        } else {
#pragma unroll
          for (int i = 0; i < DTILES; i++) {
            k0[i] = *reinterpret_cast<const uint32_t*>(kt + row0 * HD + i * 16 + c * 4);
            k1[i] = *reinterpret_cast<const uint32_t*>(kt + (row0 + 8) * HD + i * 16 + c * 4);
          }
        }
        k0[DTILES] = k1[DTILES] = 0;  // (an odd number of words: the last product's second half)
        float s[NT][4];
#pragma unroll
        for (int n = 0; n < NT; n++) {
          int sum[QP][4] = {};
#pragma unroll
          for (int p = 0; p < QP; p++)
#pragma unroll
            for (int i = 0; i < KSTEPS; i++) {
              const uint2 b = NT == 1 ? q_own[NT == 1 ? p * KSTEPS + i : 0] : reinterpret_cast<const uint2*>(qf)[((p * KSTEPS + i) * NT + n) * 32 + lane];
              mma8(sum[p], k0[2 * i], k1[2 * i], k0[2 * i + 1], k1[2 * i + 1], b.x, b.y);
            }
#pragma unroll
          for (int e = 0; e < 4; e++) {
            const float low = (float)(sum[QP - 2][e] * 256 + sum[QP - 1][e]);
            s[n][e] = QP == 3 ? fmaf((float)sum[0][e], 65536.f, low) : low;
          }
        }
        // scores in powers of two less their reference, and the weights' exponents less theirs; what a column does not see has none
        const float sk0 = s_sk[st][row0], sk1 = s_sk[st][row0 + 8], lv0 = s_lsv[st][row0], lv1 = s_lsv[st][row0 + 8];
        float z[NT][4], top = -INFINITY;
#pragma unroll
        for (int n = 0; n < NT; n++)
#pragma unroll
          for (int e = 0; e < 4; e++) {
            s[n][e] *= (e < 2 ? sk0 : sk1) * qs[n][e & 1];
            z[n][e] = s[n][e] + (e < 2 ? lv0 : lv1);
          }
        if (!(s_whole[st] && key0 >= whole_lo && key0 <= whole_hi)) {
          const int kp0 = s_pos[st][row0], kp1 = s_pos[st][row0 + 8];
#pragma unroll
          for (int n = 0; n < NT; n++)
#pragma unroll
            for (int e = 0; e < 4; e++) {
              const int kp = e < 2 ? kp0 : kp1, q = pos[n][e & 1];
              if (kp > q || (a.window > 0 && kp <= q - a.window)) s[n][e] = z[n][e] = -INFINITY;
            }
        }
#pragma unroll
        for (int n = 0; n < NT; n++)
#pragma unroll
          for (int e = 0; e < 4; e++) top = fmaxf(top, fmaxf(s[n][e] - m[n][e & 1], z[n][e] - M[n][e & 1]));
        if (__any_sync(0xffffffffu, top > SLACK)) {
#pragma unroll
          for (int n = 0; n < NT; n++)
#pragma unroll
            for (int e = 0; e < 2; e++) {
              float top = fmaxf(s[n][e], s[n][e + 2]), topz = fmaxf(z[n][e], z[n][e + 2]);
#pragma unroll
              for (int d = 4; d < 32; d <<= 1) {
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
                topz = fmaxf(topz, __shfl_xor_sync(0xffffffffu, topz, d));
              }
              // (references are numbers: a column that has seen nothing yet keeps the lowest)
              const float m2 = fmaxf(m[n][e], top), M2 = fmaxf(M[n][e], topz);
              l[n][e] *= ex2(m[n][e] - m2);
              const float f = ex2(M[n][e] - M2);
#pragma unroll
              for (int k = 0; k < DTILES; k++) {
                o[k][n][e] *= f;
                o[k][n][e + 2] *= f;
              }
              m[n][e] = m2;
              M[n][e] = M2;
            }
        }
        uint32_t b0[WP][NT], b1[WP][NT];
#pragma unroll
        for (int n = 0; n < NT; n++) {
          float wt[4];
#pragma unroll
          for (int e = 0; e < 4; e++) {
            l[n][e & 1] += ex2(s[n][e] - m[n][e & 1]);
            wt[e] = ex2(z[n][e] - M[n][e & 1]);
          }
          const uint32_t h0 = pack_half(wt[0], wt[1]), h1 = pack_half(wt[2], wt[3]);
          b0[0][n] = transpose8x8(h0);
          b1[0][n] = transpose8x8(h1);
          if (WP == 2) {
            b0[WP - 1][n] = transpose8x8(rest_half(h0, wt[0], wt[1]));
            b1[WP - 1][n] = transpose8x8(rest_half(h1, wt[2], wt[3]));
          }
        }
        // O^T: lane group g holds numbers g * HD / 8 and on of the keys in rows 2c, 2c + 1, 2c + 8, 2c + 9
        constexpr int W = HD / 8;
        const int r0 = warp * 16 + key_of_row(2 * c), r1 = warp * 16 + key_of_row(2 * c + 1);
        auto with_pair = [&](int k, uint32_t lo01, uint32_t hi01) {
          // lo01: two numbers of the keys in rows 2c and 2c + 1 (bytes: number 0, number 1 of the one, then of the other)
          const uint32_t a0 = halves(lo01), a1 = halves(lo01 >> 8), a2 = halves(hi01), a3 = halves(hi01 >> 8);
#pragma unroll
          for (int p = 0; p < WP; p++)
#pragma unroll
            for (int n = 0; n < NT; n++) mma(o[k][n], a0, a1, a2, a3, b0[p][n], b1[p][n]);
        };
        if constexpr (W % 4 == 0) {
          uint32_t v[4][W / 4];
          constexpr int VEC = W % 16 == 0 ? 16 : W % 8 == 0 ? 8 : 4;  // bytes a read
#pragma unroll
          for (int i = 0; i < 4; i++) {
            const int r = (i & 1 ? r1 : r0) + (i >> 1) * 8;
#pragma unroll
            for (int u = 0; u < W / VEC; u++) {
              const int at = g * W + u * VEC;
              const int x = !swz ? 0 : HD == 128 ? r & 7 : (r >> 1) & 3;
              const unsigned char* src = vt + r * HD + ((((at >> 4) ^ x) << 4) | (at & 15));
              if constexpr (VEC == 16) {
                const uint4 y = *reinterpret_cast<const uint4*>(src);
                v[i][4 * u] = y.x, v[i][4 * u + 1] = y.y, v[i][4 * u + 2] = y.z, v[i][4 * u + 3] = y.w;
              } else if constexpr (VEC == 8) {
                const uint2 y = *reinterpret_cast<const uint2*>(src);
                v[i][2 * u] = y.x, v[i][2 * u + 1] = y.y;
              } else {
                v[i][u] = *reinterpret_cast<const uint32_t*>(src);
              }
            }
          }
#pragma unroll
          for (int u = 0; u < W / 4; u++) {
            with_pair(2 * u, __byte_perm(v[0][u], v[1][u], 0x5410), __byte_perm(v[2][u], v[3][u], 0x5410));
            with_pair(2 * u + 1, __byte_perm(v[0][u], v[1][u], 0x7632), __byte_perm(v[2][u], v[3][u], 0x7632));
          }
        } else {
#pragma unroll
          for (int k = 0; k < DTILES; k++) {
            uint32_t v[4];
#pragma unroll
            for (int i = 0; i < 4; i++)
              v[i] = *reinterpret_cast<const uint16_t*>(vt + ((i & 1 ? r1 : r0) + (i >> 1) * 8) * HD + g * W + 2 * k);
            with_pair(k, v[0] | v[1] << 16, v[2] | v[3] << 16);
          }
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&empty[st]);
      }
      if (!ok) failed = 1;

      // ---------------- the four warps together
#pragma unroll
      for (int n = 0; n < NT; n++)
#pragma unroll
        for (int e = 0; e < 2; e++) {
#pragma unroll
          for (int d = 4; d < 32; d <<= 1) l[n][e] += __shfl_xor_sync(0xffffffffu, l[n][e], d);
          if (g == 0) {
            const int j = n * 8 + 2 * c + e;
            s_m[warp][j] = m[n][e];
            s_M[warp][j] = M[n][e];
            s_l[warp][j] = l[n][e];
          }
        }
      asm volatile("bar.sync 1, 128;" ::: "memory");
      float f[NT][2];
#pragma unroll
      for (int n = 0; n < NT; n++)
#pragma unroll
        for (int e = 0; e < 2; e++) {
          const int j = n * 8 + 2 * c + e;
          float top = s_M[0][j];
#pragma unroll
          for (int i = 1; i < WARPS; i++) top = fmaxf(top, s_M[i][j]);
          f[n][e] = ex2(M[n][e] - top);
        }
      for (int turn = 0; turn < WARPS; turn++) {
        if (warp == turn) {
#pragma unroll
          for (int k = 0; k < DTILES; k++)
#pragma unroll
            for (int n = 0; n < NT; n++)
#pragma unroll
              for (int e = 0; e < 4; e++) {
                // row (of O^T) g of tile k is number g * HD / 8 + 2 k, row g + 8 the one behind it
                float* dst = s_out + (n * 8 + 2 * c + (e & 1)) * (HD + 4) + g * (HD / 8) + 2 * k + (e >> 1);
                const float x = o[k][n][e] * f[n][e & 1];
                *dst = turn == 0 ? x : *dst + x;
              }
        }
        asm volatile("bar.sync 1, 128;" ::: "memory");
      }
      const bool all = w.tile == 0 && w.tile_end == w.r.tiles;  // the share holds the item whole
      for (int j = warp; j < COLS; j += WARPS) {
        float top = s_m[0][j], topM = s_M[0][j], sum = 0.f;
#pragma unroll
        for (int i = 1; i < WARPS; i++) {
          top = fmaxf(top, s_m[i][j]);
          topM = fmaxf(topM, s_M[i][j]);
        }
#pragma unroll
        for (int i = 0; i < WARPS; i++) sum += s_l[i][j] * ex2(s_m[i][j] - top);
        const float* src = s_out + j * (HD + 4);
        if (all) {
          if (col0 + j < cols) {
            T* dst = reinterpret_cast<T*>(a.out) + (a.q_start[w.r.s] + (col0 + j) / a.group) * a.out_stride +
                     (long long)(kvh * a.group + (col0 + j) % a.group) * HD;
            const float r = last_factor(topM, top, sum);
            for (int d = lane; d < HD; d += 32) dst[d] = from_float<T>(src[d] * r);
          }
        } else {
          float* dst = a.parts + ((((long long)kvh * gridDim.x + blockIdx.x) * 2 + (w.opens ? 0 : 1)) * COLS + j) * (HD + 4);
          for (int d = lane; d < HD; d += 32) dst[d] = src[d];
          if (lane == 0) {
            dst[HD] = topM;
            dst[HD + 1] = top;
            dst[HD + 2] = sum;
          }
        }
      }
    }
  }
  __syncthreads();
  if (threadIdx.x == 0 && failed) atomicOr(a.status, TKB_STATUS_WAIT_TIMEOUT);
}

// The parts of items that no share holds whole, in the order of the shares.  A block a request and kv head, a warp a column.
template <typename T, int NT>
__global__ void __launch_bounds__(128) attn_kv8_join_kernel(const Args a, int blocks) {
  constexpr int COLS = 8 * NT;
  trigger_dependents();
  grid_dependency_wait();
  Request r;
  const int total = a.base[a.n_seqs], base = a.base[blockIdx.x];
  if (!r.load(a, blockIdx.x, COLS)) return;
  const Shares shares(total, blocks);
  const int kvh = blockIdx.y, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (int ct = 0; ct < r.col_tiles; ct++) {
    const int at = base + ct * r.tiles, b0 = shares.of(at), b1 = shares.of(at + r.tiles - 1);
    if (b0 == b1) continue;
    // the share's first item, or its last
    const float* first = a.parts + (((long long)kvh * blocks + b0) * 2 + (shares.start(b0) >= at ? 0 : 1)) * COLS * (HD + 4);
    const float* rest = a.parts + ((long long)kvh * blocks + b0 + 1) * 2 * COLS * (HD + 4);
    const int n = b1 - b0 + 1;
    for (int j = warp; j < COLS && ct * COLS + j < r.q_len * a.group; j += 4) {
      auto part = [&](int i) { return (i == 0 ? first : rest + (long long)(i - 1) * 2 * COLS * (HD + 4)) + j * (HD + 4); };
      float top = LOWEST, topM = LOWEST;
      for (int i = lane; i < n; i += 32) {
        const float* p = part(i);
        topM = fmaxf(topM, p[HD]);
        top = fmaxf(top, p[HD + 1]);
      }
      top = warp_max(top);
      topM = warp_max(topM);
      float sum = 0.f, acc[(HD + 31) / 32];
#pragma unroll
      for (int i = 0; i < (HD + 31) / 32; i++) acc[i] = 0.f;
#pragma unroll 4
      for (int b = 0; b < n; b++) {
        const float* p = part(b);
        sum += p[HD + 2] * ex2(p[HD + 1] - top);
        const float f = ex2(p[HD] - topM);
#pragma unroll
        for (int i = 0; i < (HD + 31) / 32; i++)
          if (lane + 32 * i < HD) acc[i] += p[lane + 32 * i] * f;
      }
      const float f = last_factor(topM, top, sum);
      const int col = ct * COLS + j;
      T* dst = reinterpret_cast<T*>(a.out) + (a.q_start[r.s] + col / a.group) * a.out_stride + (long long)(kvh * a.group + col % a.group) * HD;
#pragma unroll
      for (int i = 0; i < (HD + 31) / 32; i++)
        if (lane + 32 * i < HD) dst[lane + 32 * i] = from_float<T>(acc[i] * f);
    }
  }
}

int make_map_codes(CUtensorMap* map, const void* base, long long rows, int box_rows) {
  cuuint64_t dims[2] = {(cuuint64_t)HD, (cuuint64_t)rows};
  cuuint64_t strides[1] = {(cuuint64_t)HD};
  cuuint32_t box[2] = {(cuuint32_t)HD, (cuuint32_t)box_rows};
  cuuint32_t estr[2] = {1, 1};
  CUresult r = g_encode(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(base), dims, strides, box, estr,
                        CU_TENSOR_MAP_INTERLEAVE_NONE, HD == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B,
                        CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? 0 : 1000 + (int)r;
}

// How many blocks a kv head gets, and whether shares are whole items.  Both from bounds: `col_tiles` items of at most `tiles`.
struct Cut {
  int blocks, whole;
};
Cut cut(int col_tiles, int tiles, int nkv) {
  const int slots = sm_count() * (HD <= 64 ? 4 : HD <= 128 ? 3 : 1) / nkv;
  Cut c;
  const long long total = (long long)col_tiles * tiles;
  c.whole = tiles <= 4;
  long long b = c.whole ? col_tiles : total / 2;  // two tiles a share at least
  if (b > slots) b = slots;
  c.blocks = b < 1 ? 1 : (int)b;
  return c;
}

template <typename T, int NT>
int launch(Args a, int col_tiles, int tiles, cudaStream_t st) {
  constexpr int BYTES = Layout<T, NT>::BYTES;
  static SharedMemoryRequest ask;
  int rc = ask({{(const void*)attn_kv8_kernel<T, NT>, BYTES}});
  if (rc) return rc;
  CUtensorMap map_k, map_v;
  memset(&map_k, 0, sizeof(map_k));
  memset(&map_v, 0, sizeof(map_v));
  const long long rows = (long long)a.num_pages * a.nkv * a.ps;
  a.tma_rows = 0;
  if (SWIZZLES && a.ps_shift >= 3 && rows < (1ll << 31)) {
    a.tma_rows = a.ps < BKV ? a.ps : BKV;
    if ((rc = get_encode()) || (rc = make_map_codes(&map_k, a.kcache, rows, a.tma_rows)) || (rc = make_map_codes(&map_v, a.vcache, rows, a.tma_rows)))
      return rc;
  }
  const Cut c = cut(col_tiles, tiles, a.nkv);
  a.whole = c.whole;
  rc = launch_pdl(attn_kv8_kernel<T, NT>, dim3(c.blocks, a.nkv), dim3(THREADS), (size_t)BYTES, st, map_k, map_v, a);
  if (rc || c.whole) return rc;
  return launch_pdl(attn_kv8_join_kernel<T, NT>, dim3(a.n_seqs, a.nkv), dim3(128), 0, st, a, c.blocks);
}

// where the parts start in the scratch
long long parts_at(int n_seqs) { return ((long long)n_seqs + 1 + 3) / 4 * 16; }

// column tiles of all requests, at most, when a block takes `cols` of them
int most_col_tiles(int n_seqs, int singles, int tokens, int group, int cols) {
  const int one = (group + cols - 1) / cols;
  return singles * one + (int)(((long long)(tokens - singles) * group + cols - 1) / cols) + (n_seqs - singles);
}

}  // namespace

// Bytes of scratch that tkb_attn_kv8 wants with the same sizes.
TKB_EXPORT long long tkb_attn_kv8_scratch(int n_seqs, int singles, int tokens, int max_kv, int nkv, int group) {
  long long most = 0;
  for (int nt = 1; nt <= max_nt(); nt++) {
    const Cut c = cut(most_col_tiles(n_seqs, singles, tokens, group, 8 * nt), (max_kv + BKV - 1) / BKV + 1, nkv);
    const long long n = (long long)nkv * c.blocks * 2 * 8 * nt * (HD + 4) * 4;
    if (n > most) most = n;
  }
  return most + parts_at(n_seqs);
}

// q, out: rows of heads (f32 != 0: float32, else bfloat16).  singles: requests that bring one token; tokens: rows of q;
// max_kv: no request has more keys.  scratch: see above, on a 16-byte boundary.
TKB_EXPORT int tkb_attn_kv8(const void* q, long long q_stride, void* out, long long out_stride, int f32, const void* kcache,
                            const void* vcache, const float* k_scale, const float* v_scale, const int* q_start, const int* q_len,
                            const int* kv_len, const int* page_indptr, const int* page_ids, void* scratch, int n_seqs, int singles, int tokens,
                            int max_kv, int nh, int nkv, int ps, float scale, int window, int num_pages, int* status, void* st_) {
  if (n_seqs <= 0 || tokens <= 0) return 0;
  if (nkv <= 0 || nh <= 0 || nh % nkv || ps <= 0 || window < 0 || singles < 0 || singles > n_seqs || singles > tokens || max_kv < 0) return -2;
  if (nkv > 65535) return -3;
  Args a = {};
  a.q = q, a.out = out, a.q_stride = q_stride, a.out_stride = out_stride;
  a.kcache = (const int8_t*)kcache, a.vcache = (const int8_t*)vcache, a.k_scale = k_scale, a.v_scale = v_scale;
  a.q_start = q_start, a.q_len = q_len, a.kv_len = kv_len, a.page_indptr = page_indptr, a.page_ids = page_ids;
  a.base = (int*)scratch;
  a.parts = (float*)((char*)scratch + parts_at(n_seqs));
  a.n_seqs = n_seqs, a.group = nh / nkv, a.nkv = nkv, a.ps = ps, a.window = window, a.num_pages = num_pages, a.status = status;
  a.ps_shift = (ps & (ps - 1)) == 0 ? 31 - __builtin_clz(ps) : -1;
  a.scale_log2 = scale * 1.4426950408889634f;
  a.which = SINGLE | PORTION;
  cudaStream_t st = (cudaStream_t)st_;
  // one tile of 8 columns for single tokens of up to 8 heads a kv head, two where there are more columns to fill them
  const int nt = max_nt() == 2 && (singles < n_seqs || a.group > 8) ? 2 : 1;
  const int col_tiles = most_col_tiles(n_seqs, singles, tokens, a.group, 8 * nt), tiles = (max_kv + BKV - 1) / BKV + 1;
  if ((long long)col_tiles * tiles > 0x7fffffffll) return -3;
  if constexpr (max_nt() == 2) {
    if (nt == 2) return f32 ? launch<float, 2>(a, col_tiles, tiles, st) : launch<bf16, 2>(a, col_tiles, tiles, st);
  }
  return f32 ? launch<float, 1>(a, col_tiles, tiles, st) : launch<bf16, 1>(a, col_tiles, tiles, st);
}
