// A K/V cache in pages (gfx950): tables of different sizes share one pool, a test row or a few attend over the cached rows
// of their table, the attention weights add up per cached row, and a cache over its budget keeps the rows that drew most.
//
//   s_i = scale q . K_i  (i < len),   p = exp(s - max s),   out = sum_i p_i V_i / sum_i p_i   (len = 0: 0)
//   weights_i += sum over heads and query rows of p_i / sum p
#include "common.h"
#include "launch.h"
#include "paged.h"

#include <numeric>

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
// Bound by the bytes of K and V, which are read once (one row over 8 x 45,000 cached rows of 8 heads: 124 us, 5.9 TB/s). A
// workgroup takes a run of rows of one item: a sequence, a K/V head and up to 16 QT query rows (the heads of a group and
// the query rows together); its NW waves take turns of KS rows. Nothing of K and V is shared between waves, so they go from
// memory straight into the registers of the matrix products, a turn ahead of their use; LDS only joins the waves at the end.
//   S^T = K Q^T  (16 keys x 16 queries): the A operand is 16 bytes of a K row per lane, the result holds query l % 16,
//                keys 4 (l / 16) + i, which is the B operand of
//   O^T = V^T P^T with the keys in that order: the A operand holds the values of column group l % 16 (D / 16 columns, one
//                per product) of those keys; in bf16 the halves of pairs of rows are regrouped by v_perm_b32.
// One query row leaves 15 of the 16 columns empty: the products stay far below the loads all the same.
// bf16 probabilities enter as two bf16 terms (2^-16 of each left out), so that the output is off by its own rounding
// alone; the second product costs nothing beside the loads. fp32 runs on the fp32 matrix unit.
// Softmax: p = 2^(s - ref), ref moved to the running maximum when a score passes it by more than PA_SLACK (one test per turn).
// The products with V take 2^-24 p, so that sums with values near the largest float stay finite. bf16 has the 24 in ref,
// where it costs no instruction and rounds the exponent to 2^-20; fp32 would lose four bits of a mild score by that, and
// multiplies.
constexpr float PA_SHIFT = 24.f, PA_SLACK = 8.f;
template <typename T>
struct PagedShift {
  static constexpr float REF = sizeof(T) == 2 ? PA_SHIFT : 0.f, VALUE = sizeof(T) == 2 ? 1.f : 0x1p-24f;
};
constexpr float PA_REF0 = -3.4028234663852886e38f;

// The work is cut on the device, by the lengths as they are: a unit is PA_UNIT rows of one item, units are counted item after
// item, and G workgroups (pa_waves per CU) take equal runs of them, whatever the lengths. An item that one workgroup covers
// is written at once; of the others each workgroup leaves a partial (at most two: one of an item begun before it, one of an
// item it begins), which pa_merge_kernel joins. (A fixed number of rows per workgroup instead: 64 sequences of 500 to
// 10,000 rows took 97 us at 8 workgroups per CU and 146 at 2, one sequence of 45,000 rows 39 and 27; this way 84 and 26.)
constexpr int PA_UNIT = 128, PA_WHOLE = 1024;

struct PagedSplit {
  int groups;    // G, or 0: a workgroup of eight waves for each item
  int least;     // units a workgroup takes at least
  int few;       // below so many units, half of the workgroups share them
  int qtiles;
  float* part;   // [2 G][16 QT][D] unnormalised outputs
  float2* ml;    // [2 G][16 QT] (ref, sum)
  int2* ends;    // [N H qtiles] the workgroups that hold the first and the last unit of an item
  float2* stat;  // [N Hq Tq] (ref, 1 / sum) for the weights, or null
  float* score;  // [N Hq Tq][score_sn] scores in log2 units for the weights, or null: from K once more
  int64_t score_sn;
};

__device__ __forceinline__ int pa_len(const PagedAttn& a, int n) { return a.pool.pages > 0 ? pool_length(a.pool, n) : 0; }

__device__ __forceinline__ int pa_units(int len) { return (len + PA_UNIT - 1) / PA_UNIT; }

// Inclusive sum over the lanes of a wave, in the registers.
__device__ __forceinline__ int wave_sum_scan(int x) {
  x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, false);  // row_shr:1, 2, 4, 8 within 16 lanes
  x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xa, 0xf, false);  // row_bcast:15 into rows 1 and 3
  x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xc, 0xf, false);  // row_bcast:31 into rows 2 and 3
  return x;
}

// The units of the sequences, 64 sequences at a time, one per lane.
struct PagedUnits {
  const PagedAttn& a;
  int per, lane;  // items of a sequence
  int own, upto;  // sequence `lane`: its units, and theirs up to it
  int total;      // of all sequences
  __device__ __forceinline__ int load(int base) const {
    const int n = base + lane;
    return n < a.N ? pa_units(pa_len(a, n)) * per : 0;
  }
  __device__ __forceinline__ PagedUnits(const PagedAttn& args, int items, int l) : a(args), per(items), lane(l) {
    own = load(0);
    upto = wave_sum_scan(own);
    total = __builtin_amdgcn_readlane(upto, 63);
    for (int base = 64; base < a.N; base += 64) total += __builtin_amdgcn_readlane(wave_sum_scan(load(base)), 63);
  }
  // the sequence that unit t < total belongs to, and its first unit
  __device__ __forceinline__ int find(int t, int* first) const {
    int u = own, s = upto;
    for (int base = 0;;) {
      const uint64_t past = __ballot(s > t);
      if (past) {
        const int k = __builtin_ctzll(past);
        *first = __builtin_amdgcn_readlane(s - u, k);
        return base + k;
      }
      base += 64;
      if (base >= a.N) return *first = 0;  // not reached
      const int before = __builtin_amdgcn_readlane(s, 63);
      u = load(base);
      s = wave_sum_scan(u) + before;
    }
  }
};

// Equal shares: `groups` workgroups (half of them below `few` units, and fewer if they would get less than `least` units) of
// `share` units, the first `more` of them one more.
struct PagedShares {
  int groups, share, more;
  __device__ __forceinline__ PagedShares(const PagedSplit& z, int total) {
    groups = total / z.least;
    const int most = total < z.few ? z.groups / 2 : z.groups;
    groups = groups < 1 ? 1 : groups < most ? groups : most;
    share = total / groups;
    more = total - share * groups;
  }
  __device__ __forceinline__ int first(int w) const { return w * share + (w < more ? w : more); }
};

template <typename T, int D>
struct PagedTile {
  static constexpr int ES = sizeof(T), SUB = ES == 2 ? 2 : 1, KS = 16 * SUB;  // 16-key subtiles, keys of a turn
  static constexpr int NC = D * ES / 64;                                      // 16-byte chunks of a K row per lane
  static constexpr int DE = D / 16, DW = DE * ES / 4;                         // values and dwords of a V row per lane
  uint4 k[SUB][NC];
  uint32_t v[SUB][4][DW];
};

typedef uint32_t u32v2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32v4 __attribute__((ext_vector_type(4)));
template <int DW>
__device__ __forceinline__ void load_dwords(uint32_t* d, __amdgpu_buffer_rsrc_t r, uint32_t off) {
  if constexpr (DW == 1) {
    d[0] = __builtin_amdgcn_raw_buffer_load_b32(r, off, 0, 0);
  } else if constexpr (DW == 2) {
    const u32v2 x = __builtin_bit_cast(u32v2, __builtin_amdgcn_raw_buffer_load_b64(r, off, 0, 0));
    d[0] = x[0], d[1] = x[1];
  } else {
#pragma unroll
    for (int i = 0; i < DW; i += 4) {
      const u32v4 x = __builtin_bit_cast(u32v4, __builtin_amdgcn_raw_buffer_load_b128(r, off + 4 * i, 0, 0));
      d[i] = x[0], d[i + 1] = x[1], d[i + 2] = x[2], d[i + 3] = x[3];
    }
  }
}

// The scores of 16 keys (chunks k of their rows) for 16 queries: key 4 (l / 16) + i, query l % 16. fp32 sums in four chains:
// one of D products would be the largest rounding of all (2-norm of the output's error for sharp scores, D = 64 and 128:
// 9.4e-7 and 1.1e-6 with one chain and the 24 in ref, 4.5e-7 this way; of mild ones 4.2e-7 and 1.8e-7).
template <typename T, int NC>
__device__ __forceinline__ f32x4 tile_scores(const uint4* k, const uint4* q) {
  if constexpr (sizeof(T) == 2) {
    f32x4 s = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int c = 0; c < NC; ++c)
      s = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, k[c]), __builtin_bit_cast(bf16x8, q[c]), s, 0, 0, 0);
    return s;
  } else {
    f32x4 s[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      s[i] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int c = 0; c < NC; ++c)
        s[i] = __builtin_amdgcn_mfma_f32_16x16x4f32(__builtin_bit_cast(f32x4, k[c])[i], __builtin_bit_cast(f32x4, q[c])[i], s[i], 0,
                                                    0, 0);
    }
    return (s[0] + s[1]) + (s[2] + s[3]);
  }
}

// A score in log2 units, rounded before the reference is taken off: the difference of the largest one is then exact, however
// large it is, and the same wherever it is formed. (A fused product would leave the rounding of the product in the exponent:
// at scores of 10^9 the probabilities of a row added up to 10^7.)
__device__ __forceinline__ float log2_score(float s, float sc) {
#pragma clang fp contract(off)
  return s * sc;
}

// Sum over the 16 lanes of a row, in the registers (row_ror).
template <int N>
__device__ __forceinline__ float row_add(float x) {
  return x + __uint_as_float(__builtin_amdgcn_update_dpp(0, __float_as_uint(x), 0x120 + N, 0xf, 0xf, false));
}
__device__ __forceinline__ float row16_sum(float x) { return row_add<1>(row_add<2>(row_add<4>(row_add<8>(x)))); }

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
  const f32x4 pv = f32x4{p[0][0], p[0][1], p[0][2], p[0][3]} * PagedShift<float>::VALUE;
#pragma unroll
  for (int e = 0; e < D / 16; ++e) {
    const f32x4 va = {__uint_as_float(t.v[0][0][e]), __uint_as_float(t.v[0][1][e]), __uint_as_float(t.v[0][2][e]),
                      __uint_as_float(t.v[0][3][e])};
    o[e] = mfma16x16x16(va, pv, o[e]);
  }
}

// N values to p, 16 bytes at a time.
template <typename T, int N>
__device__ __forceinline__ void store_row(T* p, const float* x) {
  constexpr int C = 16 / sizeof(T);
#pragma unroll
  for (int j = 0; j < N; j += C) {
    if constexpr (C == 4) {
      *(f32x4*)(p + j) = f32x4{x[j], x[j + 1], x[j + 2], x[j + 3]};
    } else {
      const bf16x4 lo = cvt_bf16x4(f32x4{x[j], x[j + 1], x[j + 2], x[j + 3]});
      const bf16x4 hi = cvt_bf16x4(f32x4{x[j + 4], x[j + 5], x[j + 6], x[j + 7]});
      *(bf16x8*)(p + j) = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
    }
  }
}

// Rows [c0, c1) of an item by the NW waves of a workgroup: the output, or (slot >= 0) a partial of it.
template <typename T, int D, int QT, bool W, int NW>
__device__ __forceinline__ void pa_segment(const PagedAttn& a, const PagedSplit& z, int n, int item, int c0, int c1, int slot) {
  typedef PagedTile<T, D> Tile;
  constexpr int SUB = Tile::SUB, KS = Tile::KS, NC = Tile::NC, DE = Tile::DE, ES = Tile::ES;
  __shared__ float sh_o[NW / 2][16 * QT][D + 4];
  __shared__ float2 sh_ml[NW / 2][16 * QT];
  const PagedPool& c = a.pool;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lr = lane & 15, lg = lane >> 4;
  const int G = a.Hq / c.H, rows = G * a.Tq;
  const float sc = a.scale * TA_LOG2E;
  const uint32_t koff = lr * D * ES + lg * 16, voff = lg * 4 * D * ES + lr * DE * ES;
  const int qt0 = item % z.qtiles, h = item / z.qtiles, nh = n * c.H + h;

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
  const int32_t* table = c.table + n * c.table_sn;
  // 64 page ids of the table at a time, one per lane
  int pg0 = c0 >> c.shift, pg = pg0 + lane < c.max_pages ? table[pg0 + lane] : -1;
  const int64_t head = (int64_t)h << c.shift;

  // Loads the turn at `key`; returns the live rows of its subtiles, 8 bits each. The rows past c1 and those of a page the
  // pool does not have lie behind their buffer's end: the loads return 0 for them and touch no memory, so every turn issues
  // the same loads (waits that count them need no branch) and a value nobody wrote meets no product.
  auto fetch = [&](Tile& t, int key) -> int {
    int live = 0;
#pragma unroll
    for (int s = 0; s < SUB; ++s) {
      const int k0 = key + 16 * s, left = c1 - k0;
      int i = left > 0 ? (k0 >> c.shift) - pg0 : 0;
      if (i >= 64) {
        pg0 += i;
        pg = pg0 + lane < c.max_pages ? table[pg0 + lane] : -1;
        asm volatile("" : "+v"(pg));  // waited for here, not wherever the paths join (there: for every load in flight)
        i = 0;
      }
      const int page = __builtin_amdgcn_readlane(pg, i);
      const int have = page < 0 || page >= c.pages || left <= 0 ? 0 : left < 16 ? left : 16;
      live |= have << (8 * s);
      const int64_t off = ((have ? page : 0) * c.page_sp + (head + (k0 & ((1 << c.shift) - 1))) * D) * ES;
      const __amdgpu_buffer_rsrc_t kr = __builtin_amdgcn_make_buffer_rsrc((char*)c.k + off, 0, have * D * ES, TA_BUF_WORD3);
      const __amdgpu_buffer_rsrc_t vr = __builtin_amdgcn_make_buffer_rsrc((char*)c.v + off, 0, have * D * ES, TA_BUF_WORD3);
#pragma unroll
      for (int i2 = 0; i2 < NC; ++i2)
        t.k[s][i2] = __builtin_bit_cast(uint4, __builtin_amdgcn_raw_buffer_load_b128(kr, koff + i2 * 64, 0, 0));
#pragma unroll
      for (int j = 0; j < 4; ++j) load_dwords<Tile::DW>(t.v[s][j], vr, voff + j * D * ES);
    }
    return live;
  };
  auto compute = [&](Tile& t, int key, int live) {
    const bool full = live == (SUB == 2 ? 16 << 8 | 16 : 16);
#pragma unroll
    for (int qt = 0; qt < QT; ++qt) {
      float x[SUB][4], top = TA_NEG_INF;
#pragma unroll
      for (int s = 0; s < SUB; ++s) {
        const f32x4 sv = tile_scores<T, NC>(t.k[s], q[qt]);
#pragma unroll
        for (int i = 0; i < 4; ++i) x[s][i] = log2_score(sv[i], sc);
      }
      if (!full) {
#pragma unroll
        for (int s = 0; s < SUB; ++s)
#pragma unroll
          for (int i = 0; i < 4; ++i) x[s][i] = lg * 4 + i < (live >> (8 * s) & 255) ? x[s][i] : TA_NEG_INF;
      }
#pragma unroll
      for (int s = 0; s < SUB; ++s) {
#pragma unroll
        for (int i = 0; i < 4; ++i) top = fmaxf(top, x[s][i]);
        if constexpr (W) {
          const int r = (qt0 * QT + qt) * 16 + lr;
          if (r < rows && key < c1)
            *(f32x4*)(z.score + ((int64_t)nh * rows + r) * z.score_sn + key + 16 * s + lg * 4) =
                f32x4{x[s][0], x[s][1], x[s][2], x[s][3]};
        }
      }
      if (wave_any(top - ref[qt] > PA_SLACK - PagedShift<T>::REF)) {
        const float to = fmaxf(ref[qt], quad_max(top) + PagedShift<T>::REF), f = __builtin_amdgcn_exp2f(ref[qt] - to);
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
      // one query tile's scores and probabilities live at a time, where stored scores take the registers too (12 dwords a
      // lane spilled without it; elsewhere the tiles overlap: 64 query rows of 64 dims over 8 x 12,000 rows 57.5 -> 56 us)
      if constexpr (QT > 1 && W) __builtin_amdgcn_sched_barrier(0);
    }
  };

  int key = c0 + wave * KS;
  if (key < c1) {
    Tile ta, tb;
    int la = fetch(ta, key);
    for (; key < c1; key += 2 * NW * KS) {
      const int lb = fetch(tb, key + NW * KS);
      compute(ta, key, la);
      la = fetch(ta, key + 2 * NW * KS);
      if (key + NW * KS < c1) compute(tb, key + NW * KS, lb);
    }
  }

  // join the waves: the upper half hands over to the lower half, until one has all
#pragma unroll
  for (int t = 0; t < QT; ++t) l[t] = quad_sum(l[t]);
#pragma unroll
  for (int half = NW / 2; half >= 1; half >>= 1) {
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
  if (wave == 0) {
#pragma unroll
    for (int t = 0; t < QT; ++t) {
      const int r = (qt0 * QT + t) * 16 + lr;
      if (r >= rows) continue;
      const float inv = l[t] == 0.f ? 0.f : 1.f / l[t], out = slot >= 0 ? 1.f : inv * (1.f / PagedShift<T>::VALUE);
      float x[4 * DE];  // columns 4 DE lg + j of the row
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int e = 0; e < DE; ++e) x[i * DE + e] = o[t][e][i] * out;
      if (slot >= 0) {
        const int64_t at = (int64_t)slot * 16 * QT + t * 16 + lr;
        store_row<float, 4 * DE>(z.part + at * D + lg * 4 * DE, x);
        if (lg == 0) z.ml[at] = make_float2(ref[t], l[t]);
      } else {
        store_row<T, 4 * DE>((T*)a.out + n * a.o_sn + (h * G + r / a.Tq) * a.o_sh + (r % a.Tq) * a.o_st + lg * 4 * DE, x);
        if (z.stat && lg == 0) z.stat[(int64_t)nh * rows + r] = make_float2(ref[t], inv);
      }
    }
  }
}

// Waves per SIMD that the registers of a kernel allow: one for tiles of 32 and 64 query rows of 128 dims. In tiles of 16 with
// two waves every tile reads K and V again (tiles of 16 / larger: bf16, 32 query rows a head over 8 x 5,000 rows 57 / 42 us,
// 64 rows 104 / 48; fp32, 17 rows 102 / 70, 34 rows over 49 x 5,311 372 / 304).
constexpr int pa_waves(int D, int QT) { return D == 128 && QT > 1 ? 1 : 2; }

// Equal shares of all items' units.
template <typename T, int D, int QT, bool W>
__global__ __launch_bounds__(256, pa_waves(D, QT)) void pa_kernel(PagedAttn a, PagedSplit z) {
  const int per = a.pool.H * z.qtiles;
  const PagedUnits units(a, per, threadIdx.x & 63);
  const PagedShares shares(z, units.total);
  if ((int)blockIdx.x >= shares.groups) return;
  int unit = shares.first(blockIdx.x);
  const int end = shares.first(blockIdx.x + 1);
  while (unit < end) {
    int first;
    const int n = units.find(unit, &first);
    const int len = __builtin_amdgcn_readfirstlane(pa_len(a, n)), each = pa_units(len);
    const int item = (unit - first) / each, u0 = unit - first - item * each;
    const int u1 = u0 + end - unit < each ? u0 + end - unit : each;
    if (threadIdx.x == 0 && u0 == 0) z.ends[n * per + item].x = blockIdx.x;
    if (threadIdx.x == 0 && u1 == each) z.ends[n * per + item].y = blockIdx.x;
    pa_segment<T, D, QT, W, 4>(a, z, n, item, u0 * PA_UNIT, u1 * PA_UNIT < len ? u1 * PA_UNIT : len,
                               u1 - u0 < each ? 2 * blockIdx.x + (u0 == 0) : -1);
    unit += u1 - u0;
  }
}

// A workgroup of eight waves for each item, where no sequence is long.
template <typename T, int D, int QT, bool W>
__global__ __launch_bounds__(512) void pa_whole_kernel(PagedAttn a, PagedSplit z) {
  const int per = a.pool.H * z.qtiles, n = blockIdx.x / per;
  pa_segment<T, D, QT, W, 8>(a, z, n, blockIdx.x % per, 0, __builtin_amdgcn_readfirstlane(pa_len(a, n)), -1);
}

__device__ __forceinline__ void store4(float* p, f32x4 x) { *(f32x4*)p = x; }
__device__ __forceinline__ void store4(bf16* p, f32x4 x) { *(bf16x4*)p = cvt_bf16x4(x); }

// Where the partials of query row r (of all rows of K/V head h of sequence n) are: `parts` of them, from workgroup w0 on;
// one: pa_kernel has written the row.
template <int QT>
struct PagedParts {
  int w0, parts, at;
  __device__ __forceinline__ PagedParts(const PagedSplit& z, int nh, int r) {
    const int2 w = z.ends[nh * z.qtiles + r / (16 * QT)];
    w0 = w.x;
    parts = w.y - w0 + 1;
    at = r % (16 * QT);
  }
  __device__ __forceinline__ int64_t slot(int i) const { return (int64_t)(2 * (w0 + i) + (i == 0)) * (16 * QT) + at; }
};

// Joins the partials of a query row in a wave: 4 values of a partial output per lane, 256 / D partials at a time. Rows that
// pa_kernel has written are left alone; rows without a key become 0.
template <typename T, int D, int QT>
__device__ __forceinline__ void pa_merge_row(const PagedAttn& a, const PagedSplit& z, int64_t row) {
  constexpr int LPR = D / 4, GR = 64 / LPR;
  const int lane = threadIdx.x & 63, G = a.Hq / a.pool.H, rows = G * a.Tq;
  if (row >= (int64_t)a.N * a.pool.H * rows) return;
  const int r = (int)(row % rows), nh = (int)(row / rows), n = nh / a.pool.H, h = nh % a.pool.H;
  PagedParts<QT> p(z, nh, r);
  p.w0 = __builtin_amdgcn_readfirstlane(p.w0);
  p.parts = __builtin_amdgcn_readfirstlane(p.parts);
  const int len = pa_len(a, n);
  T* op = (T*)a.out + n * a.o_sn + (h * G + r / a.Tq) * a.o_sh + (r % a.Tq) * a.o_st + lane * 4;
  if (len == 0) {
    if (lane < LPR) store4(op, f32x4{0.f, 0.f, 0.f, 0.f});
    return;
  }
  if (p.parts == 1) return;
  // every group of lanes joins its share of the partials by itself (their loads wait for nothing but the lengths), then
  // the groups are joined
  float m = PA_REF0, l = 0.f;
  f32x4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
  for (int i = lane / LPR; i < p.parts; i += GR) {
    const float2 v = z.ml[p.slot(i)];
    const f32x4 x = *(const f32x4*)(z.part + p.slot(i) * D + lane % LPR * 4);
    const float to = fmaxf(m, v.x), f0 = __builtin_amdgcn_exp2f(m - to), f1 = __builtin_amdgcn_exp2f(v.x - to);
    m = to;
    l = l * f0 + v.y * f1;
#pragma unroll
    for (int j = 0; j < 4; ++j) o[j] = o[j] * f0 + x[j] * f1;
  }
#pragma unroll
  for (int x = LPR; x < 64; x <<= 1) {
    const float mo = __shfl_xor(m, x, 64), lo = __shfl_xor(l, x, 64);
    const float to = fmaxf(m, mo), f0 = __builtin_amdgcn_exp2f(m - to), f1 = __builtin_amdgcn_exp2f(mo - to);
    m = to;
    l = l * f0 + lo * f1;
#pragma unroll
    for (int j = 0; j < 4; ++j) o[j] = o[j] * f0 + __shfl_xor(o[j], x, 64) * f1;
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
  if (lane < LPR) store4(op, o * (inv * (1.f / PagedShift<T>::VALUE)));
  if (z.stat && lane == 0) z.stat[row] = make_float2(m, inv);
}

template <typename T, int D, int QT>
__global__ __launch_bounds__(256) void pa_merge_kernel(PagedAttn a, PagedSplit z) {
  pa_merge_row<T, D, QT>(a, z, (int64_t)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6));
}

// weights[n, i] += sum over the query rows of p (stat: their references and sums): the 64 keys from k0 on, 4 per thread, the
// query rows over 16 threads (each in steps of 16), joined in a fixed order.
__device__ __forceinline__ void pa_weights_keys64(const PagedAttn& a, const PagedSplit& z, int n, int len, int k0,
                                                  const float2* stat) {
  __shared__ f32x4 sh[16][16];
  const int all = a.Hq * a.Tq, kt = threadIdx.x & 15, rt = threadIdx.x >> 4;
  const int64_t first = (int64_t)n * all;
  f32x4 w = {0.f, 0.f, 0.f, 0.f};
  // Eight loads in flight: of few cached rows their latency is all there is (61 query rows in two heads a group over 22 x 9
  // rows: the whole call 71 -> 45 us; 59 over 5 x 1,700 39 -> 33).
#pragma unroll 8
  for (int r = rt; r < all; r += 16) {
    const float2 st = stat[r];
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

__global__ __launch_bounds__(256) void pa_weights_kernel(PagedAttn a, PagedSplit z) {
  const int n = blockIdx.y, len = pa_len(a, n), k0 = blockIdx.x * 64;
  if (k0 < len) pa_weights_keys64(a, z, n, len, k0, z.stat + (int64_t)n * a.Hq * a.Tq);
}

// Both in one launch for up to PA_JOIN query rows of a sequence: the first workgroups merge, the others join the references
// and sums of their sequence's rows for themselves and add the weights up.
constexpr int PA_JOIN = 32;

template <typename T, int D, int QT>
__global__ __launch_bounds__(256) void pa_merge_weights_kernel(PagedAttn a, PagedSplit z, int merges) {
  __shared__ float2 stat[PA_JOIN];
  if ((int)blockIdx.x < merges)
    return pa_merge_row<T, D, QT>(a, z, (int64_t)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6));
  const int at = blockIdx.x - merges, blocks = (int)(z.score_sn / 64), n = at / blocks, k0 = at % blocks * 64;
  const int len = pa_len(a, n), rows = a.Hq / a.pool.H * a.Tq, all = a.Hq * a.Tq;
  if (k0 >= len) return;
#pragma unroll 2
  for (int i = threadIdx.x / 16; i < all; i += 16) {  // 16 lanes a row
    const PagedParts<QT> p(z, n * a.pool.H + i / rows, i % rows);
    float m = PA_REF0, l = 0.f;
    for (int j = threadIdx.x % 16; j < p.parts; j += 16) {
      const float2 v = z.ml[p.slot(j)];
      const float to = fmaxf(m, v.x);
      l = l * __builtin_amdgcn_exp2f(m - to) + v.y * __builtin_amdgcn_exp2f(v.x - to);
      m = to;
    }
#pragma unroll
    for (int x = 1; x < 16; x <<= 1) {
      const float mo = __shfl_xor(m, x, 64), lo = __shfl_xor(l, x, 64), to = fmaxf(m, mo);
      l = l * __builtin_amdgcn_exp2f(m - to) + lo * __builtin_amdgcn_exp2f(mo - to);
      m = to;
    }
    if (threadIdx.x % 16 == 0)  // one part: pa_kernel has left the pair, and nothing in ml
      stat[i] = p.parts == 1 ? z.stat[(int64_t)n * all + i] : make_float2(m, l == 0.f ? 0.f : 1.f / l);
  }
  __syncthreads();
  pa_weights_keys64(a, z, n, len, k0, stat);
}

// The same from K itself, for many query rows per K/V head: the scores of 64 keys per wave once more, head after head (a
// head's K rows are loaded while the one before is multiplied), normalised and summed in the registers, then over the 16
// queries of a tile. Reads D values of a key per head where the scores are 8 bytes per query row, written and read.
template <int D>
__global__ __launch_bounds__(256) void pa_weights_keys_kernel(PagedAttn a, PagedSplit z) {
  typedef bf16 T;
  constexpr int ES = 2, NC = D * ES / 64, SUB = 4, KEYS = 16 * SUB;
  struct Tile {
    uint4 k[SUB][NC];
  };
  const PagedPool& c = a.pool;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lr = lane & 15, lg = lane >> 4;
  const int n = blockIdx.y, len = __builtin_amdgcn_readfirstlane(pa_len(a, n)), key0 = (blockIdx.x * 4 + wave) * KEYS;
  if (key0 >= len) return;
  const int G = a.Hq / c.H, rows = G * a.Tq, tiles = (rows + 15) / 16, at = (key0 + 16 * lane) >> c.shift;
  const int pg = lane < SUB && at < c.max_pages ? c.table[n * c.table_sn + at] : -1;
  const float sc = a.scale * TA_LOG2E;
  const uint32_t koff = lr * D * ES + lg * 16;
  int64_t off[SUB];
  int have[SUB];
#pragma unroll
  for (int s = 0; s < SUB; ++s) {
    const int page = __builtin_amdgcn_readlane(pg, s), left = len - key0 - 16 * s;
    have[s] = page < 0 || page >= c.pages || left <= 0 ? 0 : left < 16 ? left : 16;
    off[s] = ((have[s] ? page : 0) * c.page_sp + ((key0 + 16 * s) & ((1 << c.shift) - 1)) * D) * ES;
  }
  auto fetch = [&](Tile& t, int h) {  // past the last head: nothing
#pragma unroll
    for (int s = 0; s < SUB; ++s) {
      const __amdgpu_buffer_rsrc_t kr = __builtin_amdgcn_make_buffer_rsrc(
          (char*)c.k + off[s] + ((int64_t)(h < c.H ? h : 0) << c.shift) * D * ES, 0, h < c.H ? have[s] * D * ES : 0, TA_BUF_WORD3);
#pragma unroll
      for (int i = 0; i < NC; ++i)
        t.k[s][i] = __builtin_bit_cast(uint4, __builtin_amdgcn_raw_buffer_load_b128(kr, koff + i * 64, 0, 0));
    }
  };
  float w[SUB][4];
#pragma unroll
  for (int s = 0; s < SUB; ++s)
#pragma unroll
    for (int i = 0; i < 4; ++i) w[s][i] = 0.f;
  auto compute = [&](Tile& t, int h) {
    if (h >= c.H) return;
    for (int qt = 0; qt < tiles; ++qt) {
      const int r = qt * 16 + lr;
      uint4 q[NC];
      float2 st = make_float2(0.f, 0.f);
#pragma unroll
      for (int i = 0; i < NC; ++i) q[i] = uint4{0, 0, 0, 0};
      if (r < rows) {
        const char* qp = (const char*)a.q + (n * a.q_sn + (h * G + r / a.Tq) * a.q_sh + (r % a.Tq) * a.q_st) * ES + lg * 16;
#pragma unroll
        for (int i = 0; i < NC; ++i) q[i] = ldg16(qp + i * 64);
        st = z.stat[((int64_t)n * c.H + h) * rows + r];
      }
#pragma unroll
      for (int s = 0; s < SUB; ++s) {
        const f32x4 sv = tile_scores<T, NC>(t.k[s], q);
#pragma unroll
        for (int i = 0; i < 4; ++i)
          // a padded query row adds nothing, its product with an infinite key (0 times infinity) neither
          w[s][i] = r < rows ? __builtin_fmaf(__builtin_amdgcn_exp2f(log2_score(sv[i], sc) - st.x), st.y, w[s][i]) : w[s][i];
      }
    }
  };
  Tile ta, tb;
  fetch(ta, 0);
  for (int h = 0; h < c.H; h += 2) {
    fetch(tb, h + 1);
    compute(ta, h);
    fetch(ta, h + 2);
    compute(tb, h + 1);
  }
  float* out = a.weights + n * a.weights_sn + key0 + lg * 4;
#pragma unroll
  for (int s = 0; s < SUB; ++s)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float sum = row16_sum(w[s][i]);
      if (lr == 0 && lg * 4 + i < have[s]) out[16 * s + i] += sum;
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

// gather: k, v [N, H, T, D] <- the first min(lengths[n], T) rows of the pages (0 where there is no page), the same way back
__global__ __launch_bounds__(256) void paged_gather_kernel(PagedGather a, int es) {
  const int n = blockIdx.y, chunks = a.pool.D * es / 16, len = pool_length(a.pool, n), rows = len < a.T ? len : a.T;
  const int64_t total = (int64_t)rows * a.pool.H * chunks;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
    const int c = (int)(i % chunks), row = (int)(i / chunks % rows), h = (int)(i / chunks / rows);
    const int64_t from = pool_row(a.pool, n, h, row), to = (((int64_t)n * a.pool.H + h) * a.T + row) * a.pool.D * es + c * 16;
    *(uint4*)((char*)a.k + to) = from < 0 ? uint4{0, 0, 0, 0} : ldg16((const char*)a.pool.k + from * es + c * 16);
    *(uint4*)((char*)a.v + to) = from < 0 ? uint4{0, 0, 0, 0} : ldg16((const char*)a.pool.v + from * es + c * 16);
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

// Three launches: the threshold (one workgroup per sequence), the ranks (a workgroup per 1,024 rows, or more rows where there
// are many), the moves; the first two are one where no sequence has more than 1,024 rows.
//
// A row competes if it is none of the recent ones; it stays if its code is above the threshold, or equal to it and among the
// first `even` such rows. With before(r) the rows that stay below row r, the i-th place to fill is the row r < cut that goes
// with r - before(r) = i, and the i-th last row to move is the row r >= cut that stays with cut - 1 - before(r) = i: each
// row knows its rank by a count of the rows before it alone.
struct EvictCut {
  uint32_t threshold;
  int even;
};
constexpr int PE_NW = PE_NT / 64, PE_BINS = 2048;

__device__ __forceinline__ int lanes_before(uint64_t mask) {
  return __builtin_amdgcn_mbcnt_hi((uint32_t)(mask >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)mask, 0));
}
// f(row, code) for this thread's share of rows [0, end); load(row) gives the code, eight at a time in flight.
template <typename L, typename F>
__device__ __forceinline__ void each_code(int end, L load, F f) {
  int base = 0;
  for (; base + 8 * PE_NT <= end; base += 8 * PE_NT) {
    uint32_t c[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) c[j] = load(base + j * PE_NT + (int)threadIdx.x);
#pragma unroll
    for (int j = 0; j < 8; ++j) f(base + j * PE_NT + (int)threadIdx.x, c[j]);
  }
  for (int r = base + threadIdx.x; r < end; r += PE_NT) f(r, load(r));
}

// The sum of `count` (uniform) over the waves before this one, and over all.
__device__ __forceinline__ int wave_offset(int count, int* sh, int* all) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  __syncthreads();
  if (lane == 0) sh[wave] = count;
  __syncthreads();
  const int upto = wave_sum_scan(lane < PE_NW ? sh[lane] : 0);
  *all = __builtin_amdgcn_readlane(upto, PE_NW - 1);
  return __builtin_amdgcn_readlane(upto, __builtin_amdgcn_readfirstlane(wave)) - count;
}

// The threshold by three digits (11, 11 and 10 bits) of a histogram in LDS. One CU does it, bound by the latency and issue
// of its passes over the weights (from L2), so it does nothing else, keeps eight loads a thread in flight and stops at the
// digit that decides (mostly the second): 16,384 rows take 14 us, 45,000 rows 15 us (21 with all three digits, 42 with four
// loads in flight; with the ranks in it too, 16,384 rows took 29).
__device__ __forceinline__ EvictCut evict_threshold(const PagedEvict& a, int n, const EvictSizes z) {
  __shared__ int hist[PE_BINS], sh[PE_NW], pick[3];
  const int tid = threadIdx.x, free_rows = z.len - z.recent;
  const float* w = a.weights + n * a.weights_sn;
  int want = z.kept - z.recent;  // of the rows that compete; in the end, of those of the threshold's code
  if (want == 0 || want == free_rows) return EvictCut{want == 0 ? 0xffffffffu : 0u, 0};  // no code is 0 or 2^32 - 1
  for (int i = tid; i < PE_BINS; i += PE_NT) hist[i] = 0;
  __syncthreads();
  auto weight = [&](int r) { return weight_code(w[r]); };
  uint32_t threshold = 0;
  for (int digit = 0; digit < 3; ++digit) {
    const int shift = digit == 0 ? 21 : digit == 1 ? 10 : 0, above = digit == 1 ? 21 : 10;
    if (digit == 0)
      each_code(free_rows, weight, [&](int, uint32_t c) { atomicAdd(&hist[c >> 21], 1); });
    else
      each_code(free_rows, weight, [&](int, uint32_t c) {
        if ((c ^ threshold) >> above == 0) atomicAdd(&hist[c >> shift & ((1u << (above - shift)) - 1)], 1);
      });
    __syncthreads();
    // thread t takes two bins, counted from the top: the first digit whose count from above reaches `want`
    const int top = PE_BINS - 2 * tid - 1;
    const int h1 = hist[top], h0 = hist[top - 1], upto = wave_sum_scan(h0 + h1);
    hist[top] = hist[top - 1] = 0;
    int all;
    const int before = wave_offset(__builtin_amdgcn_readlane(upto, 63), sh, &all) + upto - h0 - h1;
    if (before < want && before + h0 + h1 >= want) {  // one thread
      const bool one = before + h1 >= want;
      pick[0] = one ? top : top - 1;
      pick[1] = want - before - (one ? 0 : h1);
      pick[2] = one ? h1 : h0;
    }
    __syncthreads();
    threshold |= (uint32_t)pick[0] << shift;
    want = pick[1];
    if (want == pick[2]) return EvictCut{threshold - 1, 0};  // all codes of these digits stay: no need to look further
  }
  return EvictCut{threshold, want};
}

__global__ __launch_bounds__(PE_NT) void paged_threshold_kernel(PagedEvict a, EvictCut* cuts) {
  const EvictCut e = evict_threshold(a, blockIdx.x, evict_sizes(a, blockIdx.x));
  if (threadIdx.x == 0) cuts[blockIdx.x] = e;
}

// `span` blocks of 1,024 rows of sequence n, one row per thread at a time: what stays in place, the places to fill (holes
// [N, K], in order) and the rows to move (tails [N, K], from the last one back), their number in moves[n]. ONE: the only block
// of its sequence, which finds the threshold itself. Each workgroup counts the rows before its first one; the span keeps the
// workgroups of a sequence to PE_GROUPS, and the time in proportion to the rows (2^22 rows 4.9 -> 2.0 ms, 2^24 61 -> 8.1,
// against a span of one; 2^30, which the entry point takes, would run for minutes).
constexpr int PE_GROUPS = 256;

template <bool ONE>
__global__ __launch_bounds__(PE_NT) void paged_ranks_kernel(PagedEvict a, const EvictCut* cuts, int32_t* holes, int32_t* tails,
                                                            int32_t* moves, int span) {
  __shared__ int sh[PE_NW];
  const int n = blockIdx.y, tid = threadIdx.x;
  const EvictSizes z = evict_sizes(a, n);
  const int64_t cap = (int64_t)a.pool.max_pages << a.pool.shift, start = (int64_t)blockIdx.x * span * PE_NT;
  const int64_t stop = start + (int64_t)span * PE_NT;
  const int free_rows = z.len - z.recent, cut = z.kept;
  EvictCut e;
  if constexpr (ONE) e = evict_threshold(a, n, z);
  else e = cuts[n];
  const float* w = a.weights + n * a.weights_sn;
  int32_t* index = a.index + (int64_t)n * a.K;
  float* kw = a.kept_weights + n * cap;
  if (blockIdx.x == 0 && tid == 0) {
    a.kept_lengths[n] = cut;
    if (cut == z.len) moves[n] = 0;
  }
  for (int64_t r = start + tid; r < stop; r += PE_NT) {
    if (r >= cut && r < a.K) index[r] = -1;
    if (r >= cut && r < cap) kw[r] = 0.f;
  }
  if (start >= z.len) return;
  // the rows before: those above the threshold, and those equal to it
  int more = 0, even = 0;
  each_code(
      start < free_rows ? (int)start : free_rows, [&](int i) { return weight_code(w[i]); },
      [&](int, uint32_t c) {
        more += c > e.threshold;
        even += c == e.threshold;
      });
  int more_before, even_before;
  wave_offset(__builtin_amdgcn_readlane(wave_sum_scan(more), 63), sh, &more_before);
  wave_offset(__builtin_amdgcn_readlane(wave_sum_scan(even), 63), sh, &even_before);
  const int end = stop < z.len ? (int)stop : z.len;
  for (int first = (int)start; first < end; first += PE_NT) {
    const int r = first + tid;
    const float x = r < z.len ? w[r] : 0.f;
    const uint32_t c = r < free_rows ? weight_code(x) : 0;
    int all, evens_here;
    const uint64_t evens = __ballot(r < free_rows && c == e.threshold);
    const int even_rank = even_before + wave_offset(__popcll(evens), sh, &evens_here) + lanes_before(evens);
    const bool keep = r < z.len && (r >= free_rows || c > e.threshold || (c == e.threshold && even_rank < e.even));
    const uint64_t keeps = __ballot(keep);
    const int before = more_before + (even_before < e.even ? even_before : e.even) +
                       (first > free_rows ? first - free_rows : 0) + wave_offset(__popcll(keeps), sh, &all) + lanes_before(keeps);
    if (r < z.len) {
      if (r < cut) {
        if (keep) {
          index[r] = r;
          kw[r] = x;
        } else {
          holes[(int64_t)n * a.K + r - before] = r;
        }
      } else {
        if (r == cut) moves[n] = cut - before;
        if (keep) tails[(int64_t)n * a.K + cut - 1 - before] = r;
      }
    }
    if (first + PE_NT < end) {  // the next block's rows before
      wave_offset(__popcll(__ballot(r < free_rows && c > e.threshold)), sh, &all);
      more_before += all;
      even_before += evens_here;
    }
  }
}

// Moves: 16 bytes of K and of V per thread and block, PM_BLOCKS blocks at a time behind one look at the pair and the table.
constexpr int PM_BLOCKS = 4;

__global__ __launch_bounds__(256) void paged_move_kernel(PagedEvict a, const int32_t* holes, const int32_t* tails,
                                                         const int32_t* moves, int es) {
  const int n = blockIdx.z, chunks = a.pool.D * es / 16, b0 = blockIdx.y * PM_BLOCKS, count = moves[n];
  const int64_t total = (int64_t)count * a.pool.H * chunks, cap = (int64_t)a.pool.max_pages << a.pool.shift;
  char* kb = (char*)a.pool.k + b0 * a.block_sp * es;
  char* vb = (char*)a.pool.v + b0 * a.block_sp * es;
  const int64_t step = a.block_sp * es;
  const int blocks = a.blocks - b0 < PM_BLOCKS ? (int)(a.blocks - b0) : PM_BLOCKS;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
    const int c = (int)(i % chunks), h = (int)(i / chunks % a.pool.H), pair = (int)(i / chunks / a.pool.H);
    const int to_row = holes[(int64_t)n * a.K + pair], from_row = tails[(int64_t)n * a.K + count - 1 - pair];
    if (b0 == 0 && h == 0 && c == 0) {
      a.index[(int64_t)n * a.K + to_row] = from_row;
      a.kept_weights[n * cap + to_row] = a.weights[n * a.weights_sn + from_row];
    }
    const int64_t to = pool_row(a.pool, n, h, to_row), from = pool_row(a.pool, n, h, from_row);
    if (to < 0 || from < 0) continue;
    const int64_t fo = from * es + c * 16, so = to * es + c * 16;
    uint4 k[PM_BLOCKS], v[PM_BLOCKS];
#pragma unroll
    for (int b = 0; b < PM_BLOCKS; ++b)
      if (b < blocks) {
        k[b] = ldg16(kb + b * step + fo);
        v[b] = ldg16(vb + b * step + fo);
      }
#pragma unroll
    for (int b = 0; b < PM_BLOCKS; ++b)
      if (b < blocks) {
        *(uint4*)(kb + b * step + so) = k[b];
        *(uint4*)(vb + b * step + so) = v[b];
      }
  }
}

int64_t align256(int64_t b) { return (b + 255) & ~(int64_t)255; }

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

// Scores kept for the weights take at most this many bytes, or those of 16 query rows of every K/V head where these are
// more (an eighth of an fp32 cache of 64 dims): tracked queries by the hundred go in slices (pa_slice), which read the cache
// as often as one launch does where they are whole tiles (bf16, 5,000 query rows over 1 x 45,000 rows: 4.4 ms with 6.9 GB, 4.8
// in slices; fp32, 1,000 over 8 x 45,000: 11.1 ms with 11 GB, 12.1).
constexpr int64_t PA_SCORE_BYTES = 1ll << 30;

// Whether the weights of a call take scores kept by the first pass, or K again (pa_weights_keys_kernel). 8 x 45,000 rows in
// bf16, D = 64, us kept / K again: 8 query rows a head 195 / 213, 16: 231 / 214, 64 (8 x 12,000): 133 / 103. Of few cached rows
// too few waves share the heads (8 x 2,000, 16 and 64 query rows: 23 / 32, 43 / 52), and in fp32 the products bound it
// (8 x 12,000, 64: 207 / 231).
template <typename T, int D>
bool pa_keeps_scores(int64_t N, int64_t Hq, int64_t H, int64_t Tq, int64_t rows) {
  if (sizeof(T) == 4 || N * rows < 65536) return true;
  return 16 * (Hq / H * Tq) <= 3 * D && N * Hq * Tq * ((rows + 63) / 64 * 64) * 4 <= PA_SCORE_BYTES;
}

// Query rows (of each head) that a launch takes: all, or as many as its counters hold (PAGED_MAX_QUERIES, PAGED_MAX_UNITS) and
// as keep their scores within PA_SCORE_BYTES, in whole tiles where that many are left.
template <typename T, int D>
int64_t pa_slice(int64_t N, int64_t Hq, int64_t H, int64_t Tq, int64_t rows, bool weights) {
  const int64_t G = Hq / H, units = N * H * (rows / 128 + 1);
  int64_t t = PAGED_MAX_QUERIES / (N * Hq);
  const int64_t counted = PAGED_MAX_UNITS / units * 16 / G;
  t = counted < t ? counted : t;
  if (weights && pa_keeps_scores<T, D>(N, Hq, H, Tq, rows)) {
    int64_t kept = PA_SCORE_BYTES / (N * Hq * ((rows + 63) / 64 * 64) * 4);
    if (kept < 16 / G) kept = 16 / G;
    t = kept < t ? kept : t;
  }
  if (t < 1) t = 1;
  if (t >= Tq) return Tq;
  for (int64_t tile = 64; tile >= 16; tile /= 2) {
    const int64_t step = tile / std::gcd(tile, G);
    if (t >= step) return t - t % step;
  }
  return t;
}

// The split of a call and the bytes of its workspace; `rows`: the most rows a sequence can have.
template <typename T, int D, int QT>
int64_t paged_split(PagedSplit* z, char* ws, int64_t N, int64_t Hq, int64_t H, int64_t Tq, int64_t rows, bool weights) {
  const int64_t qrows = Hq / H * Tq;
  z->qtiles = (int)((qrows + 16 * QT - 1) / (16 * QT));
  // Two workgroups per CU keep enough loads in flight (three: 3% slower on long caches, 30% at 64 query rows). Up to
  // PA_WHOLE rows an item goes to one workgroup of eight waves, without a merge: much the same on the GPU (split / whole:
  // one row over 8 x 700 rows 10.4 / 10.4 us, over 1 x 1,000 9.1 / 10.4, over 64 x 1,000 30.6 / 27.8), but a launch and a
  // workspace less, and such calls wait for the host (16.5 / 12.7 us).
  z->groups = rows <= PA_WHOLE ? 0 : pa_waves(D, QT) * cu_count();
  z->least = 2;
  // Of few units one workgroup per CU: half the partials, half the waves to join, and the loads of four waves are enough for
  // as long as the call then takes (us, two per CU / one: 64 query rows over 8 x 5,000 rows 30.3 / 28.9, over 1 x 45,000
  // 36.5 / 31.5, one row over 1 x 45,000 26.0 / 23.4, over 8 x 5,000 21.6 / 20.2; fp32, 32 rows over 8 x 5,000 43.9 / 40.2.
  // With the limit at 24 units a workgroup, one row over 64 x 2,000 51.4 / 52.9; rows of 32 dims, 64 query rows over
  // 8 x 5,000 22.1 / 23.2).
  z->few = D > 32 && pa_waves(D, QT) == 2 ? 12 * z->groups : 0;
  int64_t at = 0;
  auto take = [&](int64_t bytes) {
    char* p = ws + at;
    at += align256(bytes);
    return p;
  };
  const int64_t all = N * H * qrows;
  z->part = (float*)take((int64_t)z->groups * 2 * 16 * QT * D * 4);
  z->ml = (float2*)take((int64_t)z->groups * 2 * 16 * QT * 8);
  z->ends = (int2*)take(z->groups ? N * H * z->qtiles * 8 : 0);
  z->score_sn = (rows + 63) / 64 * 64;
  z->stat = nullptr;
  z->score = nullptr;
  if (weights) {
    z->stat = (float2*)take(all * 8);
    if (pa_keeps_scores<T, D>(N, Hq, H, Tq, rows)) z->score = (float*)take(all * z->score_sn * 4);
  }
  return at;
}

template <typename T, int D, int QT, bool W>
void launch_pa_w(const PagedAttn& a, const PagedSplit& z, hipStream_t stream) {
  if (z.groups == 0) {
    if constexpr (pa_waves(D, QT) == 2)
      hipLaunchKernelGGL((pa_whole_kernel<T, D, QT, W>), dim3((unsigned)(a.N * a.pool.H * z.qtiles)), dim3(512), 0, stream, a, z);
  } else {
    hipLaunchKernelGGL((pa_kernel<T, D, QT, W>), dim3((unsigned)z.groups), dim3(256), 0, stream, a, z);
    const unsigned merge = (unsigned)(((int64_t)a.N * a.Hq * a.Tq + 3) / 4);
    // In one launch where the workgroups of the weights all fit on the GPU at once and each has few rows to join (us of the
    // whole call, apart / in one, 8 heads: one query row over 8 x 2,000 rows 17.5 / 14.5, over 8 x 15,000 60.6 / 58.1, over
    // 64 x 4,000 111.2 / 112.1; 4 rows 18.2 / 16.1, 67.1 / 65.4, 125.9 / 130.0; 8 rows over 1 x 45,000 32.4 / 34.3).
    if constexpr (W && QT <= 2)  // more query rows a tile, more than PA_JOIN a sequence
      if (a.Hq * a.Tq <= PA_JOIN && a.N * z.score_sn <= 64 * 8 * (int64_t)cu_count()) {
        const unsigned blocks = (unsigned)(z.score_sn / 64 * a.N);
        hipLaunchKernelGGL((pa_merge_weights_kernel<T, D, QT>), dim3(merge + blocks), dim3(256), 0, stream, a, z, (int)merge);
        return;
      }
    hipLaunchKernelGGL((pa_merge_kernel<T, D, QT>), dim3(merge), dim3(256), 0, stream, a, z);
  }
  if (W)
    hipLaunchKernelGGL(pa_weights_kernel, dim3((unsigned)(z.score_sn / 64), a.N), dim3(256), 0, stream, a, z);
  else if (sizeof(T) == 2 && z.stat)
    hipLaunchKernelGGL(pa_weights_keys_kernel<D>, dim3((unsigned)((z.score_sn + 255) / 256), a.N), dim3(256), 0, stream, a, z);
}

// Launches (a != null) or sizes the workspace.
template <typename T, int D, int QT>
int64_t run_pa(const PagedAttn* a, void* ws, int64_t N, int64_t Hq, int64_t H, int64_t Tq, int64_t rows, bool weights,
               hipStream_t stream) {
  PagedSplit z;
  const int64_t bytes = paged_split<T, D, QT>(&z, (char*)ws, N, Hq, H, Tq, rows, weights && rows > 0);
  if (a && z.score) launch_pa_w<T, D, QT, true>(*a, z, stream);
  else if (a) launch_pa_w<T, D, QT, false>(*a, z, stream);
  return bytes;
}

template <typename T, int D>
int64_t run_pa_rows(const PagedAttn* a, void* ws, int64_t N, int64_t Hq, int64_t H, int64_t Tq, int64_t rows, bool weights,
                    hipStream_t stream) {
  const int64_t qrows = Hq / H * Tq;
  // Query rows of a tile: 16 to 64. fp32 of 64 dims keeps to 32 (64 would be one wave per SIMD; 64 query rows over 8 x 5,000
  // rows 62 / 66 us), and of 128 dims the kernel of whole items to 16: short caches are read from L2 anyhow, and two waves
  // hide more of it (8 x 900 rows, tiles of 16 / larger: bf16, 64 query rows 23.5 / 24.9 us, fp32, 32 rows 27 / 40).
  const int most = D == 128 ? (rows <= PA_WHOLE ? 16 : 64) : D * sizeof(T) > 128 ? 32 : 64;
  if constexpr (D == 128 || D * sizeof(T) <= 128)
    if (qrows > 32 && most == 64) return run_pa<T, D, 4>(a, ws, N, Hq, H, Tq, rows, weights, stream);
  if (qrows > 16 && most >= 32) return run_pa<T, D, 2>(a, ws, N, Hq, H, Tq, rows, weights, stream);
  return run_pa<T, D, 1>(a, ws, N, Hq, H, Tq, rows, weights, stream);
}

// The query rows in slices, one launch after the other on the stream (the weights add up in this order); they share a
// workspace.
template <typename T, int D>
int64_t run_pa_d(const PagedAttn* a, void* ws, int64_t N, int64_t Hq, int64_t H, int64_t Tq, int64_t rows, bool weights,
                 hipStream_t stream) {
  const int64_t slice = pa_slice<T, D>(N, Hq, H, Tq, rows, weights && rows > 0);
  int64_t bytes = 0;
  for (int64_t t = 0; t < Tq; t += slice) {
    const int64_t left = Tq - t < slice ? Tq - t : slice;
    if (!a && t > 0 && left == slice) continue;  // the last one may be sized otherwise
    PagedAttn part;
    if (a) {
      part = *a;
      part.q = (const char*)a->q + t * a->q_st * sizeof(T);
      part.out = (char*)a->out + t * a->o_st * sizeof(T);
      part.Tq = (int)left;
    }
    const int64_t b = run_pa_rows<T, D>(a ? &part : nullptr, ws, N, Hq, H, left, rows, weights, stream);
    bytes = b > bytes ? b : bytes;
  }
  return bytes;
}

int64_t run_pa_any(const PagedAttn* a, void* ws, int64_t N, int64_t Hq, int64_t H, int64_t Tq, int64_t D, int64_t rows,
                   bool weights, int dtype, hipStream_t stream) {
  if (dtype == 0)
    return D == 32   ? run_pa_d<bf16, 32>(a, ws, N, Hq, H, Tq, rows, weights, stream)
           : D == 64 ? run_pa_d<bf16, 64>(a, ws, N, Hq, H, Tq, rows, weights, stream)
                     : run_pa_d<bf16, 128>(a, ws, N, Hq, H, Tq, rows, weights, stream);
  return D == 32   ? run_pa_d<float, 32>(a, ws, N, Hq, H, Tq, rows, weights, stream)
         : D == 64 ? run_pa_d<float, 64>(a, ws, N, Hq, H, Tq, rows, weights, stream)
                   : run_pa_d<float, 128>(a, ws, N, Hq, H, Tq, rows, weights, stream);
}

}  // namespace

int64_t tabicl_launch_paged_attn_ws_bytes(int64_t N, int64_t Hq, int64_t H, int64_t Tq, int64_t D, int64_t rows, int weights,
                                          int dtype) {
  return run_pa_any(nullptr, nullptr, N, Hq, H, Tq, D, rows, weights != 0, dtype, nullptr);
}

int tabicl_launch_paged_attn(const PagedAttn& a, int dtype, void* ws, hipStream_t stream) {
  run_pa_any(&a, ws, a.N, a.Hq, a.pool.H, a.Tq, a.pool.D, (int64_t)a.pool.max_pages << a.pool.shift, a.weights != nullptr,
             dtype, stream);
  return (int)hipGetLastError();
}

int tabicl_launch_paged_append(const PagedAppend& a, int dtype, hipStream_t stream) {
  const int es = dtype == 0 ? 2 : 4;
  const int64_t per_n = (int64_t)a.T * a.pool.H * (a.pool.D * es / 16);
  int64_t gx = (per_n + 255) / 256;
  if (gx > PAGED_MAX_GRID / a.N) gx = PAGED_MAX_GRID / a.N;
  if (gx > 4096) gx = 4096;
  hipLaunchKernelGGL(paged_append_kernel, dim3((unsigned)gx, (unsigned)a.N), dim3(256), 0, stream, a, es);
  return (int)hipGetLastError();
}

int tabicl_launch_paged_gather(const PagedGather& a, int dtype, hipStream_t stream) {
  const int es = dtype == 0 ? 2 : 4;
  int64_t gx = ((int64_t)a.T * a.pool.H * (a.pool.D * es / 16) + 255) / 256;
  if (gx > PAGED_MAX_GRID / a.N) gx = PAGED_MAX_GRID / a.N;
  if (gx > 4096) gx = 4096;
  hipLaunchKernelGGL(paged_gather_kernel, dim3((unsigned)gx, (unsigned)a.N), dim3(256), 0, stream, a, es);
  return (int)hipGetLastError();
}

int64_t tabicl_launch_paged_evict_ws_bytes(int64_t N, int64_t K) {
  return align256(N * sizeof(EvictCut)) + align256(N * 4) + 2 * align256(N * K * 4);
}

int tabicl_launch_paged_evict(const PagedEvict& a, int dtype, void* ws, hipStream_t stream) {
  const int es = dtype == 0 ? 2 : 4;
  char* at = (char*)ws;
  EvictCut* cuts = (EvictCut*)at;
  at += align256((int64_t)a.N * sizeof(EvictCut));
  int32_t* moves = (int32_t*)at;
  at += align256((int64_t)a.N * 4);
  int32_t* holes = (int32_t*)at;
  int32_t* tails = (int32_t*)(at + align256((int64_t)a.N * a.K * 4));
  const int64_t rows = (int64_t)a.pool.max_pages << a.pool.shift;
  const int64_t blocks = (rows + PE_NT - 1) / PE_NT, span = (blocks + PE_GROUPS - 1) / PE_GROUPS;
  const dim3 nt(PE_NT);
  if (rows <= PE_NT) {
    hipLaunchKernelGGL(paged_ranks_kernel<true>, dim3(1, (unsigned)a.N), nt, 0, stream, a, cuts, holes, tails, moves, 1);
  } else {
    hipLaunchKernelGGL(paged_threshold_kernel, dim3((unsigned)a.N), nt, 0, stream, a, cuts);
    hipLaunchKernelGGL(paged_ranks_kernel<false>, dim3((unsigned)((blocks + span - 1) / span), (unsigned)a.N), nt, 0, stream, a,
                       cuts, holes, tails, moves, (int)span);
  }
  if (a.K > 0) {
    const int64_t per = (int64_t)a.K * a.pool.H * (a.pool.D * es / 16);
    const unsigned gy = a.blocks > PM_BLOCKS ? (unsigned)((a.blocks + PM_BLOCKS - 1) / PM_BLOCKS) : 1;
    int64_t gx = (per + 255) / 256;
    if (gx > PAGED_MAX_GRID / ((int64_t)gy * a.N)) gx = PAGED_MAX_GRID / ((int64_t)gy * a.N);
    if (gx > 1024) gx = 1024;
    hipLaunchKernelGGL(paged_move_kernel, dim3((unsigned)gx, gy, (unsigned)a.N), dim3(256), 0, stream, a, holes, tails, moves,
                       es);
  }
  return (int)hipGetLastError();
}
