// A K/V cache in pages (gfx950): tables of different sizes share one pool, a test row or a few attend over the cached rows
// of their table, the attention weights add up per cached row, and a cache over its budget keeps the rows that drew most.
//
//   s_i = scale q . K_i  (i < len),   p = exp(s - max s),   out = sum_i p_i V_i / sum_i p_i   (len = 0: 0)
//   weights_i += sum over heads and query rows of p_i / sum p
#include "common.h"
#include "launch.h"
#include "paged.h"

namespace {

__device__ __forceinline__ int pool_length(const PagedPool& c, int n) {
  const int64_t cap = (int64_t)c.max_pages << c.shift;
  const int64_t len = c.lengths[n];
  return (int)(len < 0 ? 0 : len < cap ? len : cap);
}

// Element offset of row `row`, head h of sequence n in the pool, or -1 where its page is none of the pool's.
__device__ __forceinline__ int64_t pool_row(const PagedPool& c, int n, int h, int row) {
  const int32_t page = c.table[n * c.table_sn + (row >> c.shift)];
  if (page < 0 || page >= c.pages) return -1;
  const int R = 1 << c.shift;
  return page * c.page_sp + ((int64_t)h * R + (row & (R - 1))) * c.D;
}

// ---------------------------------------------------------------------------------------------
// attention
// ---------------------------------------------------------------------------------------------
// Bound by the bytes of K and V, which are read once: a workgroup takes `chunk` rows of one (sequence, K/V head) and up
// to 16 QT of its query rows (the heads of a group and the query rows together), its four waves take turns of KS rows.
// Nothing of K and V is shared between waves, so they go from memory straight into the registers of the matrix products,
// a turn ahead of their use; LDS only joins the four waves at the end.
//   S^T = K Q^T  (16 keys x 16 queries): the A operand is 16 bytes of a K row per lane, the result holds query l % 16,
//                keys 4 (l / 16) + i, which is the B operand of
//   O^T = V^T P^T with the keys in that order: the A operand holds the values of column group l % 16 (D / 16 columns, one
//                per product) of those keys; in bf16 the halves of pairs of rows are regrouped by v_perm_b32.
// bf16 probabilities enter as two bf16 terms (2^-16 of each left out), so that the output is off by its own rounding
// alone; the second product costs nothing beside the loads. fp32 runs on the fp32 matrix unit.
// Softmax: p = 2^(s - ref) with ref the running maximum + PA_SHIFT, moved only when a score passes it by more than 2^8
// (one test per turn); the shift keeps sums of 2^30 products with values near the largest float finite.
constexpr int PA_NW = 4;
constexpr float PA_SHIFT = 24.f, PA_SLACK = 8.f;
constexpr float PA_REF0 = -3.4028234663852886e38f;

struct PagedSplit {
  int chunk, splits, qtiles;
  int turn;      // (split turn + blockIdx) % 8 advances by one from split to split
  float* part;   // [N H][splits][rows][D] unnormalised outputs
  float2* ml;    // [N H][splits][rows] (ref, sum)
  float2* stat;  // [N H][rows] (ref, 1 / sum), for the weights
  float* score;  // [N H][rows][score_sn] scores in log2 units, for the weights
  int64_t score_sn;
};

template <typename T, int D>
struct PagedTile {
  static constexpr int ES = sizeof(T), SUB = ES == 2 ? 2 : 1, KS = 16 * SUB;  // 16-key subtiles, keys of a turn
  static constexpr int NC = D * ES / 64;                                      // 16-byte chunks of a K row per lane
  static constexpr int DE = D / 16, DW = DE * ES / 4;                         // values and dwords of a V row per lane
  uint4 k[SUB][NC];
  uint32_t v[SUB][4][DW];
};

template <int DW>
__device__ __forceinline__ void load_dwords(uint32_t* d, const char* p) {
  if constexpr (DW == 1) {
    d[0] = *(const uint32_t*)p;
  } else if constexpr (DW == 2) {
    const uint2 x = *(const uint2*)p;
    d[0] = x.x, d[1] = x.y;
  } else {
#pragma unroll
    for (int i = 0; i < DW; i += 4) {
      const uint4 x = *(const uint4*)(p + 4 * i);
      d[i] = x.x, d[i + 1] = x.y, d[i + 2] = x.z, d[i + 3] = x.w;
    }
  }
}

// The products of one tile with the 16 queries of a query tile.
template <typename T, int D>
__device__ __forceinline__ f32x4 paged_scores(const PagedTile<T, D>& t, int sub, const uint4* q) {
  f32x4 s = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int c = 0; c < PagedTile<T, D>::NC; ++c) {
    if constexpr (sizeof(T) == 2)
      s = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, t.k[sub][c]), __builtin_bit_cast(bf16x8, q[c]), s,
                                                  0, 0, 0);
    else
      s = mfma16x16x16(__builtin_bit_cast(f32x4, t.k[sub][c]), __builtin_bit_cast(f32x4, q[c]), s);
  }
  return s;
}

template <int D>
__device__ __forceinline__ void paged_values(const PagedTile<bf16, D>& t, const float (*p)[4], f32x4* o) {
  // hi: p cut to bf16, lo: the rest and 2^-18 of hi, so that neither term is 0 for a p > 0 nor of the other sign: an
  // infinite value stays infinite
  uint32_t hw[4];
  bf16x4 l4[2];
#pragma unroll
  for (int sub = 0; sub < 2; ++sub) {
    f32x4 lo32;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      lo32[i] = __builtin_fmaf(__uint_as_float(__float_as_uint(p[sub][i]) & 0xffff0000u), -(1.f - 0x1p-18f), p[sub][i]);
    l4[sub] = cvt_bf16x4(lo32);
#pragma unroll
    for (int i = 0; i < 2; ++i)
      hw[2 * sub + i] = __builtin_amdgcn_perm(__float_as_uint(p[sub][2 * i + 1]), __float_as_uint(p[sub][2 * i]), 0x07060302u);
  }
  const bf16x8 hi = __builtin_bit_cast(bf16x8, (uint4{hw[0], hw[1], hw[2], hw[3]}));
  const bf16x8 lo = __builtin_shufflevector(l4[0], l4[1], 0, 1, 2, 3, 4, 5, 6, 7);
#pragma unroll
  for (int e = 0; e < D / 16; ++e) {
    const uint32_t sel = e & 1 ? 0x07060302u : 0x05040100u;
    const int w = e / 2;
    const uint4 a = {__builtin_amdgcn_perm(t.v[0][1][w], t.v[0][0][w], sel), __builtin_amdgcn_perm(t.v[0][3][w], t.v[0][2][w], sel),
                     __builtin_amdgcn_perm(t.v[1][1][w], t.v[1][0][w], sel), __builtin_amdgcn_perm(t.v[1][3][w], t.v[1][2][w], sel)};
    const bf16x8 va = __builtin_bit_cast(bf16x8, a);
    o[e] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(va, hi, o[e], 0, 0, 0);
    o[e] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(va, lo, o[e], 0, 0, 0);
  }
  }
template <int D>
__device__ __forceinline__ void paged_values(const PagedTile<float, D>& t, const float (*p)[4], f32x4* o) {
  const f32x4 pv = {p[0][0], p[0][1], p[0][2], p[0][3]};
#pragma unroll
  for (int e = 0; e < D / 16; ++e) {
    const f32x4 va = {__uint_as_float(t.v[0][0][e]), __uint_as_float(t.v[0][1][e]), __uint_as_float(t.v[0][2][e]),
                      __uint_as_float(t.v[0][3][e])};
    o[e] = mfma16x16x16(va, pv, o[e]);
  }
}

template <typename T, int D, int QT, bool W>
__global__ __launch_bounds__(64 * PA_NW, 2) void pa_kernel(PagedAttn a, PagedSplit z) {
  typedef PagedTile<T, D> Tile;
  constexpr int SUB = Tile::SUB, KS = Tile::KS, NC = Tile::NC, DE = Tile::DE, ES = Tile::ES;
  __shared__ float sh_o[PA_NW / 2][16 * QT][D + 4];
  __shared__ float2 sh_ml[PA_NW / 2][16 * QT];
  const PagedPool& c = a.pool;
  // Workgroup b runs on XCD b % 8. The splits of a sequence and the first splits of all sequences go to all XCDs alike
  // (short sequences leave the later splits empty: with the splits of a sequence in a row, 16 of them, 64 sequences of 500
  // to 10,000 rows took 160 us, this way 87).
  const int items = a.N * c.H * z.qtiles, split = blockIdx.x / items;
  const int item = (blockIdx.x % items + items - split % items * (int)z.turn % items) % items;
  const int qt0 = item % z.qtiles, nh = item / z.qtiles;
  const int n = nh / c.H, h = nh % c.H, G = a.Hq / c.H, rows = G * a.Tq;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lr = lane & 15, lg = lane >> 4;
  const int len = c.pages > 0 ? pool_length(c, n) : 0;
  const int c0 = split * z.chunk, c1 = c0 + z.chunk < len ? c0 + z.chunk : len;
  if (c0 >= c1 && split) return;  // nothing here, and the merge knows

  // this lane's query rows: 16 QT of the (head of the group, query row) pairs
  uint4 q[QT][NC];
#pragma unroll
  for (int t = 0; t < QT; ++t) {
    const int r = (qt0 * QT + t) * 16 + lr;
#pragma unroll
    for (int i = 0; i < NC; ++i) q[t][i] = uint4{0, 0, 0, 0};
    if (r < rows) {
      const char* qp = (const char*)a.q + (n * a.q_sn + (h * G + r / a.Tq) * a.q_sh + (r % a.Tq) * a.q_st) * ES + lg * 16;
#pragma unroll
      for (int i = 0; i < NC; ++i) q[t][i] = ldg16(qp + i * 64);
    }
  }
  f32x4 o[QT][DE];
  float ref[QT], l[QT];
#pragma unroll
  for (int t = 0; t < QT; ++t) {
    ref[t] = PA_REF0;
    l[t] = 0.f;
#pragma unroll
    for (int e = 0; e < DE; ++e) o[t][e] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  const float sc = a.scale * TA_LOG2E;
  const int32_t* table = c.table + n * c.table_sn;
  // 64 page ids of the table at a time, one per lane
  int pg0 = c0 >> c.shift, pg = pg0 + lane < c.max_pages ? table[pg0 + lane] : -1;
  const int64_t head = (int64_t)h << c.shift;
  const uint32_t koff = lr * D * ES + lg * 16, voff = lg * 4 * D * ES + lr * DE * ES;

  // loads the turn at `key`; bit s of the result: subtile s has rows in the pool
  auto fetch = [&](Tile& t, int key) -> int {
    int live = 0;
#pragma unroll
    for (int s = 0; s < SUB; ++s) {
      const int k0 = key + 16 * s;
      int i = (k0 >> c.shift) - pg0;
      if (i >= 64) {
        pg0 += i;
        pg = pg0 + lane < c.max_pages ? table[pg0 + lane] : -1;
        i = 0;
      }
      const int page = __builtin_amdgcn_readlane(pg, i);
      const bool ok = k0 < c1 && page >= 0 && page < c.pages;
      live |= ok ? 1 << s : 0;
      // rows nobody has: any page's, for the address alone
      const int64_t off = ((ok ? page : 0) * c.page_sp + (head + (k0 & ((1 << c.shift) - 1))) * D) * ES;
      const char* kp = (const char*)c.k + off;
      const char* vp = (const char*)c.v + off;
#pragma unroll
      for (int i2 = 0; i2 < NC; ++i2) t.k[s][i2] = ldg16(kp + koff + i2 * 64);
#pragma unroll
      for (int j = 0; j < 4; ++j) load_dwords<Tile::DW>(t.v[s][j], vp + voff + j * D * ES);
    }
    return live;
  };
  auto compute = [&](Tile& t, int key, int live) {
    const bool full = live == (1 << SUB) - 1 && key + KS <= c1;
    if (!full) {
#pragma unroll
      for (int s = 0; s < SUB; ++s)
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (!(live >> s & 1) || key + 16 * s + lg * 4 + j >= c1)
#pragma unroll
            for (int w = 0; w < Tile::DW; ++w) t.v[s][j][w] = 0;
    }
#pragma unroll
    for (int qt = 0; qt < QT; ++qt) {
      float x[SUB][4];
      bool above = false;
#pragma unroll
      for (int s = 0; s < SUB; ++s) {
        const f32x4 sv = paged_scores<T, D>(t, s, q[qt]);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          x[s][i] = sv[i] * sc;
          if (!full && (!(live >> s & 1) || key + 16 * s + lg * 4 + i >= c1)) x[s][i] = TA_NEG_INF;
          above |= x[s][i] - ref[qt] > PA_SLACK - PA_SHIFT;
        }
        if constexpr (W) {
          const int r = (qt0 * QT + qt) * 16 + lr;
          if (r < rows)
            *(f32x4*)(z.score + ((int64_t)nh * rows + r) * z.score_sn + key + 16 * s + lg * 4) =
                f32x4{x[s][0], x[s][1], x[s][2], x[s][3]};
        }
      }
      if (wave_any(above)) {
        float m = x[0][0];
#pragma unroll
        for (int s = 0; s < SUB; ++s)
#pragma unroll
          for (int i = 0; i < 4; ++i) m = fmaxf(m, x[s][i]);
        const float to = fmaxf(ref[qt], quad_max(m) + PA_SHIFT), f = __builtin_amdgcn_exp2f(ref[qt] - to);
        ref[qt] = to;
        l[qt] *= f;
#pragma unroll
        for (int e = 0; e < DE; ++e) o[qt][e] *= f;
      }
      float p[SUB][4];
#pragma unroll
      for (int s = 0; s < SUB; ++s)
#pragma unroll
        for (int i = 0; i < 4; ++i) p[s][i] = __builtin_amdgcn_exp2f(x[s][i] - ref[qt]);
#pragma unroll
      for (int s = 0; s < SUB; ++s) l[qt] += (p[s][0] + p[s][1]) + (p[s][2] + p[s][3]);
      paged_values<D>(t, p, o[qt]);
    }
  };

  int key = c0 + wave * KS;
  if (key < c1) {
    Tile ta, tb;
    int la = fetch(ta, key), lb = 0;
    for (;;) {
      int next = key + PA_NW * KS;
      if (next < c1) lb = fetch(tb, next);
      compute(ta, key, la);
      key = next;
      if (key >= c1) break;
      next = key + PA_NW * KS;
      if (next < c1) la = fetch(ta, next);
      compute(tb, key, lb);
      key = next;
      if (key >= c1) break;
    }
  }

  // join the four waves: the upper half hands over to the lower half, twice
#pragma unroll
  for (int t = 0; t < QT; ++t) l[t] = quad_sum(l[t]);
#pragma unroll
  for (int half = PA_NW / 2; half >= 1; half >>= 1) {
    if (wave >= half && wave < 2 * half) {
#pragma unroll
      for (int t = 0; t < QT; ++t) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int e = 0; e < DE; ++e) sh_o[wave - half][t * 16 + lr][(lg * 4 + i) * DE + e] = o[t][e][i];
        if (lg == 0) sh_ml[wave - half][t * 16 + lr] = make_float2(ref[t], l[t]);
      }
    }
    __syncthreads();
    if (wave < half) {
#pragma unroll
      for (int t = 0; t < QT; ++t) {
        const float2 ml = sh_ml[wave][t * 16 + lr];
        const float to = fmaxf(ref[t], ml.x), f0 = __builtin_amdgcn_exp2f(ref[t] - to), f1 = __builtin_amdgcn_exp2f(ml.x - to);
        ref[t] = to;
        l[t] = l[t] * f0 + ml.y * f1;
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int e = 0; e < DE; ++e) o[t][e][i] = o[t][e][i] * f0 + sh_o[wave][t * 16 + lr][(lg * 4 + i) * DE + e] * f1;
      }
    }
    __syncthreads();
  }
  if (wave) return;
#pragma unroll
  for (int t = 0; t < QT; ++t) {
    const int r = (qt0 * QT + t) * 16 + lr;
    if (r >= rows) continue;
    if (z.splits > 1) {
      const int64_t at = ((int64_t)nh * z.splits + split) * rows + r;
      float* po = z.part + at * D + lg * 4 * DE;
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int e = 0; e < DE; ++e) po[i * DE + e] = o[t][e][i];
      if (lg == 0) z.ml[at] = make_float2(ref[t], l[t]);
    } else {
      const float inv = l[t] == 0.f ? 0.f : 1.f / l[t];
      T* op = (T*)a.out + n * a.o_sn + (h * G + r / a.Tq) * a.o_sh + (r % a.Tq) * a.o_st + lg * 4 * DE;
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int e = 0; e < DE; ++e) op[i * DE + e] = (T)(o[t][e][i] * inv);
      if (W && lg == 0) z.stat[(int64_t)nh * rows + r] = make_float2(ref[t], inv);
    }
  }
}

// Joins the splits of one query row per wave: 4 values of a partial output per lane, 256 / D partials at a time.
template <typename T, int D, bool W>
__global__ __launch_bounds__(256) void pa_merge_kernel(PagedAttn a, PagedSplit z) {
  constexpr int LPR = D / 4, GR = 64 / LPR;
  const int lane = threadIdx.x & 63, rows = a.Hq / a.pool.H * a.Tq;
  const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (row >= (int64_t)a.N * a.pool.H * rows) return;
  const int r = (int)(row % rows), nh = (int)(row / rows), n = nh / a.pool.H, h = nh % a.pool.H, G = a.Hq / a.pool.H;
  const int len = a.pool.pages > 0 ? pool_length(a.pool, n) : 0;
  const int used = (int)(((int64_t)len + z.chunk - 1) / z.chunk);
  const float2* ml = z.ml + (int64_t)nh * z.splits * rows + r;
  float m = PA_REF0;
  for (int s = lane; s < used; s += 64) m = fmaxf(m, ml[(int64_t)s * rows].x);
  for (int x = 32; x >= 1; x >>= 1) m = fmaxf(m, __shfl_xor(m, x, 64));
  float l = 0.f;
  for (int s = lane; s < used; s += 64) {
    const float2 v = ml[(int64_t)s * rows];
    l += v.y * __builtin_amdgcn_exp2f(v.x - m);
  }
  for (int x = 32; x >= 1; x >>= 1) l += __shfl_xor(l, x, 64);
  const float inv = l == 0.f ? 0.f : 1.f / l;
  const float* part = z.part + ((int64_t)nh * z.splits * rows + r) * D + lane % LPR * 4;
  f32x4 o = {0.f, 0.f, 0.f, 0.f};
  for (int s = lane / LPR; s < used; s += GR) {
    const float f = __builtin_amdgcn_exp2f(ml[(int64_t)s * rows].x - m) * inv;
    o += *(const f32x4*)(part + (int64_t)s * rows * D) * f;
  }
  for (int x = LPR; x < 64; x <<= 1)
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] += __shfl_xor(o[i], x, 64);
  if (lane < LPR) {
    T* op = (T*)a.out + n * a.o_sn + (h * G + r / a.Tq) * a.o_sh + (r % a.Tq) * a.o_st + lane * 4;
#pragma unroll
    for (int i = 0; i < 4; ++i) op[i] = (T)o[i];
  }
  if (W && lane == 0) z.stat[row] = make_float2(m, inv);
}

// weights[n, i] += sum over the query rows of p: 64 keys per workgroup, 4 per thread, the query rows over 16 threads
// (each in steps of 16), joined in a fixed order.
__global__ __launch_bounds__(256) void pa_weights_kernel(PagedAttn a, PagedSplit z) {
  __shared__ f32x4 sh[16][16];
  const int n = blockIdx.y, len = a.pool.pages > 0 ? pool_length(a.pool, n) : 0, k0 = blockIdx.x * 64;
  if (k0 >= len) return;
  const int all = a.Hq * a.Tq, kt = threadIdx.x & 15, rt = threadIdx.x >> 4;
  const int64_t first = (int64_t)n * all;
  f32x4 w = {0.f, 0.f, 0.f, 0.f};
  for (int r = rt; r < all; r += 16) {
    const float2 st = z.stat[first + r];
    const f32x4 s = *(const f32x4*)(z.score + (first + r) * z.score_sn + k0 + kt * 4);
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = __builtin_fmaf(__builtin_amdgcn_exp2f(s[i] - st.x), st.y, w[i]);
  }
  sh[rt][kt] = w;
  __syncthreads();
  if (threadIdx.x < 64) {
    const int key = k0 + threadIdx.x;
    float t = 0.f;
    for (int r = 0; r < 16; ++r) t += sh[r][threadIdx.x >> 2][threadIdx.x & 3];
    if (key < len) a.weights[n * a.weights_sn + key] += t;
  }
}

// ---------------------------------------------------------------------------------------------
// append: rows lengths[n] + t of the pages <- k, v; 16 bytes of K and of V per thread
// ---------------------------------------------------------------------------------------------
__global__ __launch_bounds__(256) void paged_append_kernel(PagedAppend a, int es) {
  const int n = blockIdx.y, chunks = a.pool.D * es / 16;
  const int64_t cap = (int64_t)a.pool.max_pages << a.pool.shift, start = pool_length(a.pool, n);
  const int T = a.count ? (a.count[n] < a.T ? a.count[n] : a.T) : a.T;
  const int64_t total = (int64_t)(T < 0 ? 0 : T) * a.pool.H * chunks;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
    const int c = (int)(i % chunks), h = (int)(i / chunks % a.pool.H);
    const int64_t t = i / chunks / a.pool.H;
    if (start + t >= cap) break;
    const int64_t off = pool_row(a.pool, n, h, (int)(start + t));
    if (off < 0) continue;
    *(uint4*)((char*)a.pool.k + off * es + c * 16) = ldg16((const char*)a.k + (n * a.k_sn + h * a.k_sh + t * a.k_st) * es + c * 16);
    *(uint4*)((char*)a.pool.v + off * es + c * 16) = ldg16((const char*)a.v + (n * a.v_sn + h * a.v_sh + t * a.v_st) * es + c * 16);
  }
}

// ---------------------------------------------------------------------------------------------
// eviction: one workgroup per sequence selects, a second kernel moves
// ---------------------------------------------------------------------------------------------
// Order of the weights as unsigned integers: larger weight, larger code; -0 as +0, NaN as -infinity.
__device__ __forceinline__ uint32_t weight_code(float w) {
  if (w != w) w = TA_NEG_INF;
  const uint32_t u = __float_as_uint(w + 0.f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

constexpr int PE_NT = 1024;

struct EvictSizes {
  int len, kept, recent;
};
__device__ __forceinline__ EvictSizes evict_sizes(const PagedEvict& a, int n) {
  EvictSizes z;
  z.len = pool_length(a.pool, n);
  int keep = a.keep ? a.keep[n] : a.keep_all;
  keep = keep < 0 ? 0 : keep < a.K ? keep : a.K;
  z.kept = keep < z.len ? keep : z.len;
  z.recent = a.recent < z.kept ? a.recent : z.kept;
  return z;
}

// Selection, one workgroup per sequence: the threshold code by three digits (11, 11 and 10 bits) of a histogram in LDS,
// then ranks. Wave w holds the rows [w seg, (w + 1) seg), lane l of step i row w seg + 64 i + l, so that a rank is the
// count of earlier flags of the wave (ballots) and of the waves before it: two barriers per rank, none per step. Up to
// PE_HELD steps the codes stay in registers from the first pass on; longer sequences read their weights again (from L2)
// in each of the six passes.
constexpr int PE_NW = PE_NT / 64, PE_HELD = 16, PE_BINS = 2048;

// The exclusive sums over the waves of three counts each, in sh; returns this wave's, total in *all.
__device__ __forceinline__ int wave_scan(int count, int* sh, int* all) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  __syncthreads();
  if (lane == 0) sh[wave] = count;
  __syncthreads();
  int before = 0, sum = 0;
#pragma unroll
  for (int w = 0; w < PE_NW; ++w) {
    const int x = sh[w];
    before += w < wave ? x : 0;
    sum += x;
  }
  *all = sum;
  return before;
}

template <bool HELD>
__device__ __forceinline__ void evict_select(const PagedEvict& a, int n, const EvictSizes z, int64_t* pairs, int32_t* npairs,
                                             int* hist, int* sh) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const float* w = a.weights + n * a.weights_sn;
  const int64_t cap = (int64_t)a.pool.max_pages << a.pool.shift;
  const int free_rows = z.len - z.recent;  // the rows that compete
  const int steps = ((z.len + PE_NT - 1) / PE_NT), base = wave * steps * 64 + lane;
  uint32_t held[HELD ? PE_HELD : 1];
  if constexpr (HELD) {
#pragma unroll
    for (int i = 0; i < PE_HELD; ++i) {
      const int r = base + i * 64;
      held[i] = i < steps && r < free_rows ? weight_code(w[r]) : 0;
    }
  }
  // f(step, row, code) over this lane's rows in order
  auto each = [&](auto f) {
    if constexpr (HELD) {
#pragma unroll
      for (int i = 0; i < PE_HELD; ++i)
        if (i < steps) f(base + i * 64, held[i]);
    } else {
      for (int i = 0; i < steps; i += 8) {
        uint32_t c[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const int r = base + (i + j) * 64;
          c[j] = i + j < steps && r < free_rows ? weight_code(w[r]) : 0;
        }
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (i + j < steps) f(base + (i + j) * 64, c[j]);
      }
    }
  };
  int want = z.kept - z.recent;  // of the rows [0, free_rows); in the end, of those of the threshold's weight
  const bool any = want > 0;
  uint32_t prefix = 0;
  if (any) {
#pragma unroll
    for (int digit = 0; digit < 3; ++digit) {
      const int shift = digit == 0 ? 21 : digit == 1 ? 10 : 0, bits = digit == 2 ? 10 : 11;
      for (int i = tid; i < PE_BINS; i += PE_NT) hist[i] = 0;
      __syncthreads();
      each([&](int r, uint32_t c) {
        const bool in = r < free_rows && (digit == 0 || (c >> (shift + bits)) == (prefix >> (shift + bits)));
        if (in) atomicAdd(&hist[(c >> shift) & ((1u << bits) - 1)], 1);
      });
      __syncthreads();
      // thread t sums the bins 2 t' and 2 t' + 1 with t' counted from the top: the first digit whose count from above
      // reaches `want`
      const int top = PE_BINS - 2 * tid - 1;
      const int h1 = hist[top], h0 = hist[top - 1];
      int incl = h0 + h1;
#pragma unroll
      for (int d = 1; d < 64; d <<= 1) {
        const int y = __shfl_up(incl, d, 64);
        if (lane >= d) incl += y;
      }
      int all;
      const int before = wave_scan(__shfl(incl, 63, 64), sh, &all) + incl - h0 - h1;
      __syncthreads();
      if (before < want && before + h0 + h1 >= want) {  // one thread
        const bool first = before + h1 >= want;
        sh[0] = first ? top : top - 1;
        sh[1] = want - before - (first ? 0 : h1);
      }
      __syncthreads();
      prefix |= (uint32_t)sh[0] << shift;
      want = sh[1];
      __syncthreads();
    }
  }
  const uint64_t below = (1ull << lane) - 1;
  int ties = 0, all;
  each([&](int r, uint32_t c) { ties += __popcll(__ballot(any && r < free_rows && c == prefix)); });
  const int tie0 = wave_scan(ties, sh, &all);
  auto kept = [&](int r, uint32_t c, int& at) {
    const bool tie = any && r < free_rows && c == prefix;
    const uint64_t b = __ballot(tie);
    const bool k = r < z.len && (r >= free_rows || (any && c > prefix) || (tie && at + __popcll(b & below) < want));
    at += __popcll(b);
    return k;
  };
  int holes = 0, tails = 0, at = tie0;
  each([&](int r, uint32_t c) {
    const bool k = kept(r, c, at);
    holes += __popcll(__ballot(r < z.kept && !k));
    tails += __popcll(__ballot(r >= z.kept && k));
  });
  int hole = wave_scan(holes, sh, &all), tail = wave_scan(tails, sh, &all);
  const int moves = all;
  int32_t* pr = (int32_t*)(pairs + (int64_t)n * a.K);
  int32_t* index = a.index + (int64_t)n * a.K;
  float* kw = a.kept_weights + n * cap;
  at = tie0;
  each([&](int r, uint32_t c) {
    const bool k = kept(r, c, at), is_hole = r < z.kept && !k, is_tail = r >= z.kept && k;
    const uint64_t bh = __ballot(is_hole), bt = __ballot(is_tail);
    if (is_hole) pr[2 * (hole + __popcll(bh & below))] = r;
    if (is_tail) pr[2 * (tail + __popcll(bt & below)) + 1] = r;
    hole += __popcll(bh);
    tail += __popcll(bt);
    if (k && r < z.kept) {
      index[r] = r;
      kw[r] = w[r];
    }
  });
  __syncthreads();
  for (int i = tid; i < moves; i += PE_NT) {
    const int to = pr[2 * i], from = pr[2 * i + 1];
    index[to] = from;
    kw[to] = w[from];
  }
  for (int r = z.kept + tid; r < a.K; r += PE_NT) index[r] = -1;
  for (int64_t r = z.kept + tid; r < cap; r += PE_NT) kw[r] = 0.f;
  if (tid == 0) {
    npairs[n] = moves;
    a.kept_lengths[n] = z.kept;
  }
}

// pairs [N, K]: (place, source row) of the rows that move, their count in npairs[n].
__global__ __launch_bounds__(PE_NT) void paged_select_kernel(PagedEvict a, int64_t* pairs, int32_t* npairs) {
  __shared__ int hist[PE_BINS], sh[PE_NW];
  const int n = blockIdx.x;
  const EvictSizes z = evict_sizes(a, n);
  if (z.len <= PE_HELD * PE_NT)
    evict_select<true>(a, n, z, pairs, npairs, hist, sh);
  else
    evict_select<false>(a, n, z, pairs, npairs, hist, sh);
}

__global__ __launch_bounds__(256) void paged_move_kernel(PagedEvict a, const int64_t* pairs, const int32_t* npairs, int es) {
  const int n = blockIdx.z, chunks = a.pool.D * es / 16;
  const int64_t total = (int64_t)npairs[n] * a.pool.H * chunks;
  char* kb = (char*)a.pool.k + blockIdx.y * a.block_sp * es;
  char* vb = (char*)a.pool.v + blockIdx.y * a.block_sp * es;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
    const int c = (int)(i % chunks), h = (int)(i / chunks % a.pool.H);
    const int32_t* p = (const int32_t*)(pairs + (int64_t)n * a.K + i / chunks / a.pool.H);
    const int64_t to = pool_row(a.pool, n, h, p[0]), from = pool_row(a.pool, n, h, p[1]);
    if (to < 0 || from < 0) continue;
    *(uint4*)(kb + to * es + c * 16) = ldg16(kb + from * es + c * 16);
    *(uint4*)(vb + to * es + c * 16) = ldg16(vb + from * es + c * 16);
  }
}

int64_t align256(int64_t b) { return (b + 255) & ~(int64_t)255; }

}  // namespace

namespace {

int paged_qt(int64_t rows, int64_t D, int dtype) {
  const int most = D == 128 ? 1 : D == 64 && dtype ? 2 : 4;  // more queries do not fit the registers
  return rows <= 16 || most == 1 ? 1 : rows <= 32 || most == 2 ? 2 : 4;
}

int cu_count() {
  static int count[64];
  int dev = 0;
  if (hipGetDevice(&dev) != hipSuccess || dev < 0 || dev >= 64) return 256;
  if (!count[dev]) {
    int n = 0;
    count[dev] = hipDeviceGetAttribute(&n, hipDeviceAttributeMultiprocessorCount, dev) == hipSuccess && n > 0 ? n : 256;
  }
  return count[dev];
}

// The split of a call and the bytes of its workspace; `rows`: the most rows a sequence can have.
int64_t paged_split(PagedSplit* z, char* ws, int64_t N, int64_t Hq, int64_t H, int64_t Tq, int64_t D, int64_t rows,
                    bool weights, int dtype) {
  const int64_t qrows = Hq / H * Tq, qt = paged_qt(qrows, D, dtype);
  z->qtiles = (int)((qrows + 16 * qt - 1) / (16 * qt));
  const int64_t items = N * H * z->qtiles;
  const int64_t target = 8 * cu_count(), least = 256;
  z->turn = (int)((9 - items % 8) % 8);
  int64_t chunk = (rows * items + target - 1) / target;
  chunk = (chunk + 127) / 128 * 128;
  if (chunk < least) chunk = least;
  const int64_t whole = rows > 0 ? (rows + 127) / 128 * 128 : 128;
  if (chunk > whole) chunk = whole;
  z->chunk = (int)chunk;
  z->splits = (int)(rows > chunk ? (rows + chunk - 1) / chunk : 1);
  int64_t at = 0;
  auto take = [&](int64_t bytes) {
    char* p = ws + at;
    at += align256(bytes);
    return p;
  };
  const int64_t all = N * H * qrows;
  z->part = (float*)take(z->splits > 1 ? all * z->splits * D * 4 : 0);
  z->ml = (float2*)take(z->splits > 1 ? all * z->splits * 8 : 0);
  z->score_sn = (rows + 63) / 64 * 64;
  z->stat = (float2*)take(weights ? all * 8 : 0);
  z->score = (float*)take(weights ? all * z->score_sn * 4 : 0);
  return at;
}

template <typename T, int D, int QT>
void launch_pa(const PagedAttn& a, const PagedSplit& z, hipStream_t stream) {
  const unsigned grid = (unsigned)((int64_t)a.N * a.pool.H * z.splits * z.qtiles);
  const unsigned merge = (unsigned)(((int64_t)a.N * a.Hq * a.Tq + 3) / 4);
  if (a.weights) {
    hipLaunchKernelGGL((pa_kernel<T, D, QT, true>), dim3(grid), dim3(64 * PA_NW), 0, stream, a, z);
    if (z.splits > 1) hipLaunchKernelGGL((pa_merge_kernel<T, D, true>), dim3(merge), dim3(256), 0, stream, a, z);
    const unsigned wx = (unsigned)(z.score_sn / 64);
    if (wx) hipLaunchKernelGGL(pa_weights_kernel, dim3(wx, a.N), dim3(256), 0, stream, a, z);
  } else {
    hipLaunchKernelGGL((pa_kernel<T, D, QT, false>), dim3(grid), dim3(64 * PA_NW), 0, stream, a, z);
    if (z.splits > 1) hipLaunchKernelGGL((pa_merge_kernel<T, D, false>), dim3(merge), dim3(256), 0, stream, a, z);
  }
}

template <typename T, int D>
void launch_pa_d(const PagedAttn& a, const PagedSplit& z, int qt, hipStream_t stream) {
  if (qt == 1) return launch_pa<T, D, 1>(a, z, stream);
  if constexpr (D < 128)
    if (qt == 2) return launch_pa<T, D, 2>(a, z, stream);
  if constexpr (D * sizeof(T) <= 128) launch_pa<T, D, 4>(a, z, stream);
}

template <typename T>
void launch_pa_t(const PagedAttn& a, const PagedSplit& z, int qt, hipStream_t stream) {
  if (a.pool.D == 32) launch_pa_d<T, 32>(a, z, qt, stream);
  else if (a.pool.D == 64) launch_pa_d<T, 64>(a, z, qt, stream);
  else launch_pa_d<T, 128>(a, z, qt, stream);
}

}  // namespace

int64_t tabicl_launch_paged_attn_ws_bytes(int64_t N, int64_t Hq, int64_t H, int64_t Tq, int64_t D, int64_t rows, int weights,
                                          int dtype) {
  PagedSplit z;
  return paged_split(&z, nullptr, N, Hq, H, Tq, D, rows, weights != 0, dtype);
}

int tabicl_launch_paged_attn(const PagedAttn& a, int dtype, void* ws, hipStream_t stream) {
  PagedSplit z;
  paged_split(&z, (char*)ws, a.N, a.Hq, a.pool.H, a.Tq, a.pool.D, (int64_t)a.pool.max_pages << a.pool.shift,
              a.weights != nullptr, dtype);
  const int qt = paged_qt((int64_t)a.Hq / a.pool.H * a.Tq, a.pool.D, dtype);
  if (dtype == 0) launch_pa_t<bf16>(a, z, qt, stream);
  else launch_pa_t<float>(a, z, qt, stream);
  return (int)hipGetLastError();
}

int tabicl_launch_paged_append(const PagedAppend& a, int dtype, hipStream_t stream) {
  const int es = dtype == 0 ? 2 : 4;
  const int64_t per_n = (int64_t)a.T * a.pool.H * (a.pool.D * es / 16);
  int64_t gx = (per_n + 255) / 256;
  if (gx > 4096) gx = 4096;
  hipLaunchKernelGGL(paged_append_kernel, dim3((unsigned)gx, (unsigned)a.N), dim3(256), 0, stream, a, es);
  return (int)hipGetLastError();
}

int64_t tabicl_launch_paged_evict_ws_bytes(int64_t N, int64_t K) { return align256(N * 4) + N * K * 8; }

int tabicl_launch_paged_evict(const PagedEvict& a, int dtype, void* ws, hipStream_t stream) {
  const int es = dtype == 0 ? 2 : 4;
  int32_t* npairs = (int32_t*)ws;
  int64_t* pairs = (int64_t*)((char*)ws + align256((int64_t)a.N * 4));
  hipLaunchKernelGGL(paged_select_kernel, dim3((unsigned)a.N), dim3(PE_NT), 0, stream, a, pairs, npairs);
  if (a.K > 0 && a.blocks > 0) {
    const int64_t per = (int64_t)a.K * a.pool.H * (a.pool.D * es / 16);
    int64_t gx = (per + 255) / 256;
    if (gx > 1024) gx = 1024;
    hipLaunchKernelGGL(paged_move_kernel, dim3((unsigned)gx, (unsigned)a.blocks, (unsigned)a.N), dim3(256), 0, stream, a,
                       pairs, npairs, es);
  }
  return (int)hipGetLastError();
}
