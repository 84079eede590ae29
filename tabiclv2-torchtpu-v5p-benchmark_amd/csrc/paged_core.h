// What the attention kernels over paged K/V caches share (paged.hip, paged_q8.hip, paged_sparse.hip): the pool, the cut of
// the work, one segment of cached rows in one workgroup, the join of partial results.
#pragma once
#include "common.h"
#include "paged.h"

#include <type_traits>

namespace {

// 16 bytes that are read once: nothing else of the caches has to make room for them.
__device__ __forceinline__ uint4 ldg16_once(const void* p) {
  typedef uint32_t words __attribute__((ext_vector_type(4)));
  return __builtin_bit_cast(uint4, __builtin_nontemporal_load((const words*)p));
}

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
template <typename T, typename C = T>  // values in 8 bits multiply their page's scale into p, and the 24 with it
struct PagedShift {
  static constexpr bool IN_REF = sizeof(T) == 2 && sizeof(C) == 2;
  static constexpr float REF = IN_REF ? PA_SHIFT : 0.f, VALUE = IN_REF ? 1.f : 0x1p-24f;
};
constexpr float PA_REF0 = -3.4028234663852886e38f;

// The work is cut on the device, by the lengths as they are: a unit is PA_UNIT rows of one item, units are counted item after
// item, and G workgroups (pa_waves per CU) take equal runs of them, whatever the lengths. An item that one workgroup covers
// is written at once; of the others each workgroup leaves a partial (at most two: one of an item begun before it, one of an
// item it begins), which pa_merge_kernel joins. (A fixed number of rows per workgroup instead: 64 sequences of 500 to
// 10,000 rows took 97 us at 8 workgroups per CU and 146 at 2, one sequence of 45,000 rows 39 and 27; this way 84 and 26.)
constexpr int PA_UNIT = 128, PA_WHOLE = 1024;

// Units that an item of 8-bit rows counts for beyond its own, where some sequence is shorter than a workgroup's share: a
// workgroup that begins several items has the latency of each beginning, and a turn of 8-bit rows holds half the bytes of one of
// bf16 to hide it behind (us with 2 / 4 / 6 units, one row of 64 dims: 64 sequences of 100 to 3,000 rows 29.0 / 23.8 / 22.8, 200 of
// 1,100 to 2,000 over 2 heads 28.2 / 25.6 / 26.5; 40 rows over 32 of 300 to 30,000 and 4 heads 47.5 / 45.4 / 47.4; of 128 dims and
// fp32, 12 rows over 16 of 500 to 10,000, 31.3 / 30.3 / 30.1).
constexpr int PA_EXTRA8 = 4;

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
__device__ __forceinline__ int pa_each(int len, int extra) { return len ? pa_units(len) + extra : 0; }

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
  int per, extra, lane;  // items of a sequence; units that an item counts for beyond its rows
  int own, upto;  // sequence `lane`: its units, and theirs up to it
  int total;      // of all sequences
  __device__ __forceinline__ int load(int base) const {
    const int n = base + lane;
    return n < a.N ? pa_each(pa_len(a, n), extra) * per : 0;
  }
  __device__ __forceinline__ void count() {
    own = load(0);
    upto = wave_sum_scan(own);
    total = __builtin_amdgcn_readlane(upto, 63);
    for (int base = 64; base < a.N; base += 64) total += __builtin_amdgcn_readlane(wave_sum_scan(load(base)), 63);
  }
  __device__ __forceinline__ PagedUnits(const PagedAttn& args, int items, int l) : a(args), per(items), extra(0), lane(l) { count(); }
  // Counts again with `more` units for each item, if there is a sequence with rows of fewer than `share` units.
  __device__ __forceinline__ void weigh(int share, int more) {
    const int64_t least = (int64_t)share * per;
    bool some = wave_any(own > 0 && own < least);
    for (int base = 64; base < a.N && !some; base += 64) {
      const int u = load(base);
      some = wave_any(u > 0 && u < least);
    }
    if (!some) return;
    extra = more;
    count();
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
template <int DW, int POLICY = 0>
__device__ __forceinline__ void load_dwords(uint32_t* d, __amdgpu_buffer_rsrc_t r, uint32_t off) {
  if constexpr (DW == 1) {
    d[0] = __builtin_amdgcn_raw_buffer_load_b32(r, off, 0, POLICY);
  } else if constexpr (DW == 2) {
    const u32v2 x = __builtin_bit_cast(u32v2, __builtin_amdgcn_raw_buffer_load_b64(r, off, 0, POLICY));
    d[0] = x[0], d[1] = x[1];
  } else {
#pragma unroll
    for (int i = 0; i < DW; i += 4) {
      const u32v4 x = __builtin_bit_cast(u32v4, __builtin_amdgcn_raw_buffer_load_b128(r, off + 4 * i, 0, POLICY));
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

// Cells of 8 bits: value = code * the scale of its page and head (one for K, one for V).
struct E4M3 {
  uint8_t code;
};
struct I8 {
  int8_t code;
};

// Turns of 32 keys, as in bf16. (64 would keep as many bytes in flight; the code is twice as long then, and takes longer to come in
// than the loads: 64 x 1,000 rows 20.2 us for 14.2, 12 query rows of 128 dims in fp32 over 16 sequences of 501 to 10,001 rows 34
// for 26.6, where some registers do not fit either.)
template <int D>
struct PagedTile8 {
  static constexpr int SUB = 2, KS = 32, NC = D / 32, DE = D / 16;
  static constexpr int KW = D / 16, VW = (DE + 3) / 4;  // dwords of a K and of a V row per lane
  uint32_t k[SUB][KW], v[SUB][4][VW];
  float ks[SUB], vs[SUB];
};
template <typename T, typename C, int D>
struct PagedTileOf {
  typedef PagedTile<T, D> type;
};
template <typename T, int D>
struct PagedTileOf<T, E4M3, D> {
  typedef PagedTile8<D> type;
};
template <typename T, int D>
struct PagedTileOf<T, I8, D> {
  typedef PagedTile8<D> type;
};

// Codes to bf16, exactly: the four of a dword, in order. int8 goes through fp32, whose upper half is the bf16 value.
template <typename C>
__device__ __forceinline__ uint2 codes_bf16(uint32_t x);
template <>
__device__ __forceinline__ uint2 codes_bf16<E4M3>(uint32_t x) {
  return uint2{__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(x, 1.f, false)),
               __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(x, 1.f, true))};
}
template <>
__device__ __forceinline__ uint2 codes_bf16<I8>(uint32_t x) {
  const float a = (float)(int8_t)x, b = (float)(int8_t)(x >> 8), c = (float)(int8_t)(x >> 16), d = (float)(int8_t)(x >> 24);
  return uint2{__builtin_amdgcn_perm(__float_as_uint(b), __float_as_uint(a), 0x07060302u),
               __builtin_amdgcn_perm(__float_as_uint(d), __float_as_uint(c), 0x07060302u)};
}

// The V operands of the 32 keys, one for each of the D / 16 columns of a lane. e4m3: bytes of four rows are
// regrouped by column, then converted in pairs; int8: converted byte by byte, then regrouped.
template <typename C, int D>
__device__ __forceinline__ void paged_operands8(const PagedTile8<D>& t, bf16x8* va) {
  constexpr int DE = D / 16, VW = PagedTile8<D>::VW, DP = DE < 4 ? DE : 4;  // columns of a dword
  uint32_t w[DE][4];
#pragma unroll
  for (int u = 0; u < 2; ++u)
#pragma unroll
    for (int v = 0; v < VW; ++v) {
      const uint32_t r[4] = {t.v[u][0][v], t.v[u][1][v], t.v[u][2][v], t.v[u][3][v]};
      if constexpr (std::is_same<C, I8>::value) {
#pragma unroll
        for (int e = 0; e < DP; ++e)
#pragma unroll
          for (int p = 0; p < 2; ++p)
            w[4 * v + e][2 * u + p] = __builtin_amdgcn_perm(__float_as_uint((float)(int8_t)(r[2 * p + 1] >> (8 * e))),
                                                            __float_as_uint((float)(int8_t)(r[2 * p] >> (8 * e))), 0x07060302u);
      } else {
#pragma unroll
        for (int half = 0; half < DP / 2; ++half) {
          const uint32_t sel = half ? 0x07030602u : 0x05010400u;
          const uint32_t x01 = __builtin_amdgcn_perm(r[1], r[0], sel), x23 = __builtin_amdgcn_perm(r[3], r[2], sel);
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const uint2 y = codes_bf16<C>(__builtin_amdgcn_perm(x23, x01, e ? 0x07060302u : 0x05040100u));
            w[4 * v + 2 * half + e][2 * u] = y.x, w[4 * v + 2 * half + e][2 * u + 1] = y.y;
          }
        }
      }
    }
#pragma unroll
  for (int e = 0; e < DE; ++e) va[e] = __builtin_bit_cast(bf16x8, (uint4{w[e][0], w[e][1], w[e][2], w[e][3]}));
}

__device__ __forceinline__ float upper_half(float x) { return __uint_as_float(__float_as_uint(x) & 0xffff0000u); }

// Two fp32 values cut to their upper halves, packed.
__device__ __forceinline__ uint32_t pack_upper(float a, float b) {
  return __builtin_amdgcn_perm(__float_as_uint(b), __float_as_uint(a), 0x07060302u);
}

// Eight fp32 values as the sum of N bf16 terms (the first ones cut, so that nothing is lost up to the last; it is rounded where
// N < 3). The rest of an infinite value is NaN.
template <int N>
__device__ __forceinline__ void bf16_terms(const float* x, bf16x8* term) {
  float r[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) r[i] = x[i];
#pragma unroll
  for (int k = 0; k < N; ++k) {
    if (k == N - 1 && N < 3) {
      const bf16x4 a = cvt_bf16x4(f32x4{r[0], r[1], r[2], r[3]}), b = cvt_bf16x4(f32x4{r[4], r[5], r[6], r[7]});
      term[k] = __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
    } else {
      uint32_t w[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) w[i] = pack_upper(r[2 * i], r[2 * i + 1]);
      term[k] = __builtin_bit_cast(bf16x8, (uint4{w[0], w[1], w[2], w[3]}));
#pragma unroll
      for (int i = 0; i < 8; ++i) r[i] = r[i] - upper_half(r[i]);
    }
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

// Rows [c0, c1) of an item (query tile qt0 of K/V head h of sequence n) by the NW waves of a workgroup: the output, or
// (slot >= 0) a partial of it. SEL: the rows of the pages that `index` lists for query row t0, R for each of its entries;
// the query rows are those of the group's heads. ONCE: nothing reads these rows again.
template <typename T, typename C, int D, int QT, bool W, bool SEL, int NW, bool ONCE>
__device__ __forceinline__ void pa_segment(const PagedAttn& a, const PagedSplit& z, int n, int h, int t0, int qt0, int c0, int c1,
                                           int slot, const int32_t* index = nullptr) {
  typedef typename PagedTileOf<T, C, D>::type Tile;
  typedef PagedShift<T, C> Shift;
  constexpr bool Q8 = sizeof(C) == 1;
  constexpr int SUB = Tile::SUB, KS = Tile::KS, NC = Tile::NC, DE = Tile::DE, ES = sizeof(C), TS = sizeof(T);
  constexpr int NQ = Q8 ? (TS == 2 ? 1 : 3) : 1, NP = TS == 2 ? 2 : 3;  // bf16 terms of q and of p, where C has 8 bits
  // Rows in 8 bits of up to 64 dims that one tile of query rows reads are loaded past the caches (from them / past them: one row over
  // 8 x 45,000 rows 72.8 / 66.7 us, 32 fp32 rows 104.3 / 101.9; a second tile would have to go to memory again, 64 fp32 rows 187 / 195,
  // 200 over 8 x 5,000 80 / 87, over 64 x 300 66 / 73, and so would the second half of a row of 128 dims).
  constexpr int POLICY = ONCE ? 2 : 0;
  __shared__ float sh_o[NW / 2][16 * QT][D + 4];
  __shared__ float2 sh_ml[NW / 2][16 * QT];
  const PagedPool& c = a.pool;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lr = lane & 15, lg = lane >> 4;
  const int G = a.Hq / c.H, Tn = SEL ? 1 : a.Tq, rows = G * Tn;
  const float sc = a.scale * TA_LOG2E;
  const uint32_t koff = Q8 ? lr * D + lg * (D == 32 ? 8 : 16) : lr * D * ES + lg * 16, voff = lg * 4 * D * ES + lr * DE * ES;
  const int nh = n * c.H + h;

  // this lane's query rows: 16 QT of the (head of the group, query row) pairs
  uint4 q[QT][NQ][NC];
  auto row = [&](int r) { return (const char*)a.q + (n * a.q_sn + (h * G + r / Tn) * a.q_sh + (t0 + r % Tn) * a.q_st) * TS; };
  auto dims = [&](int i) { return D == 32 ? lg * 8 : i / 2 * 64 + lg * 16 + i % 2 * 8; };  // Q8: as the chunks of a K row lie
  float finite = 0.f;  // neither infinite nor NaN while no value is (fp32 queries over 8 bits)
#pragma unroll
  for (int t = 0; t < QT; ++t) {
    const int r = (qt0 * QT + t) * 16 + lr;
#pragma unroll
    for (int j = 0; j < NQ; ++j)
#pragma unroll
      for (int i = 0; i < NC; ++i) q[t][j][i] = uint4{0, 0, 0, 0};
    if (r < rows) {
      const char* qp = row(r);
      if constexpr (!Q8) {
#pragma unroll
        for (int i = 0; i < NC; ++i) q[t][0][i] = ldg16(qp + lg * 16 + i * 64);
      } else {
#pragma unroll
        for (int i = 0; i < NC; ++i) {
          const int dim = dims(i);
          if constexpr (TS == 2) {
            q[t][0][i] = ldg16(qp + dim * 2);
          } else {
            const f32x4 x = *(const f32x4*)(qp + dim * 4), y = *(const f32x4*)(qp + dim * 4 + 16);
            const float v[8] = {x[0], x[1], x[2], x[3], y[0], y[1], y[2], y[3]};
#pragma unroll
            for (int e = 0; e < 8; e += 2) finite = __builtin_fmaf(v[e], v[e + 1], finite);
            bf16x8 term[3];
            bf16_terms<3>(v, term);
#pragma unroll
            for (int j = 0; j < 3; ++j) q[t][j][i] = __builtin_bit_cast(uint4, term[j]);
          }
        }
      }
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
  // 64 page ids of the table at a time, one per lane; with a selection the rows that each has, for 8 bits its scales
  int pg0 = c0 >> c.shift, pg, has = 0;
  float2 cs;
  const int len = SEL ? __builtin_amdgcn_readfirstlane(pa_len(a, n)) : 0;
  auto pages = [&]() {
    if constexpr (!SEL) {
      pg = pg0 + lane < c.max_pages ? table[pg0 + lane] : -1;
    } else {
      const int at = pg0 + lane < a.K ? index[pg0 + lane] : -1;
      const bool in = at >= 0 && at < c.max_pages;
      pg = in ? table[at] : -1;
      has = in ? len - (at << c.shift) : 0;
    }
    if constexpr (Q8) {
      // 0 for a page without rows: nobody may have written its scales, and the probabilities of its rows, 0, are multiplied by them
      cs = make_float2(0.f, 0.f);
      if (pg >= 0 && pg < c.pages && (!SEL || has > 0)) cs = *(const float2*)(a.scales + ((int64_t)pg * c.H + h) * 2);
    }
  };
  pages();
  const int64_t head = (int64_t)h << c.shift;

  // Loads the turn at `key`; returns the live rows of its subtiles, 8 bits each. The rows past c1 and those of a page the
  // pool does not have lie behind their buffer's end: the loads return 0 for them and touch no memory, so every turn issues
  // the same loads (waits that count them need no branch) and a value nobody wrote meets no product.
  auto fetch = [&](Tile& t, int key) -> int {
    int live = 0, id[SUB];
#pragma unroll
    for (int s = 0; s < SUB; ++s) {
      const int k0 = key + 16 * s;
      int left = c1 - k0, i = left > 0 ? (k0 >> c.shift) - pg0 : 0;
      if ((!Q8 || s == 0) && i >= 64) {  // 8 bits: a turn's pages are among the same 64 (c0 and the turns are multiples of 32)
        pg0 += i;
        pages();
        // waited for here, not wherever the paths join (there: for every load in flight)
        if constexpr (Q8) asm volatile("" : "+v"(pg), "+v"(cs.x), "+v"(cs.y));
        else asm volatile("" : "+v"(pg));
        i = 0;
      }
      id[s] = i;
      const int page = __builtin_amdgcn_readlane(pg, i);
      if constexpr (SEL) {
        const int in = __builtin_amdgcn_readlane(has, i) - (k0 & ((1 << c.shift) - 1));
        left = in < left ? in : left;
      }
      const int have = page < 0 || page >= c.pages || left <= 0 ? 0 : left < 16 ? left : 16;
      live |= have << (8 * s);
      const int64_t off = ((have ? page : 0) * c.page_sp + (head + (k0 & ((1 << c.shift) - 1))) * D) * ES;
      const __amdgpu_buffer_rsrc_t kr = __builtin_amdgcn_make_buffer_rsrc((char*)c.k + off, 0, have * D * ES, TA_BUF_WORD3);
      const __amdgpu_buffer_rsrc_t vr = __builtin_amdgcn_make_buffer_rsrc((char*)c.v + off, 0, have * D * ES, TA_BUF_WORD3);
      if constexpr (Q8) {
        if constexpr (D == 128) {
          load_dwords<4, POLICY>(t.k[s], kr, koff);
          load_dwords<4, POLICY>(t.k[s] + 4, kr, koff + 64);
        } else {
          load_dwords<Tile::KW, POLICY>(t.k[s], kr, koff);
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          if constexpr (D == 32) t.v[s][j][0] = (uint16_t)__builtin_amdgcn_raw_buffer_load_b16(vr, voff + j * D, 0, POLICY);
          else load_dwords<Tile::VW, POLICY>(t.v[s][j], vr, voff + j * D);
        }
      } else {
#pragma unroll
        for (int i2 = 0; i2 < NC; ++i2)
          t.k[s][i2] = __builtin_bit_cast(uint4, __builtin_amdgcn_raw_buffer_load_b128(kr, koff + i2 * 64, 0, POLICY));
#pragma unroll
        for (int j = 0; j < 4; ++j) load_dwords<Tile::DW, POLICY>(t.v[s][j], vr, voff + j * D * ES);
      }
    }
    if constexpr (Q8) {  // behind the loads: the first turn waits for its scales here
#pragma unroll
      for (int s = 0; s < SUB; ++s) {
        t.ks[s] = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(cs.x), id[s]));
        t.vs[s] = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(cs.y), id[s]));
      }
    }
    return live;
  };
  auto compute = [&](Tile& t, int key, int live) {
    if constexpr (!Q8) {
      const bool full = live == (SUB == 2 ? 16 << 8 | 16 : 16);
#pragma unroll
      for (int qt = 0; qt < QT; ++qt) {
        float x[SUB][4], top = TA_NEG_INF;
#pragma unroll
        for (int s = 0; s < SUB; ++s) {
          const f32x4 sv = tile_scores<T, NC>(t.k[s], q[qt][0]);
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
        if (wave_any(top - ref[qt] > PA_SLACK - Shift::REF)) {
          const float to = fmaxf(ref[qt], quad_max(top) + Shift::REF), f = __builtin_amdgcn_exp2f(ref[qt] - to);
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
    } else {
      const bool full = live == (16 << 8 | 16);
      bf16x8 kb[2][NC], va[DE];
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int i = 0; i < NC; ++i) {
          const uint2 x = codes_bf16<C>(t.k[u][2 * i]), y = codes_bf16<C>(t.k[u][2 * i + 1]);
          kb[u][i] = __builtin_bit_cast(bf16x8, (uint4{x.x, x.y, y.x, y.y}));
        }
      paged_operands8<C, D>(t, va);
#pragma unroll
      for (int qt = 0; qt < QT; ++qt) {
        float x[2][4], top = TA_NEG_INF;
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          f32x4 sv = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int j = NQ - 1; j >= 0; --j)  // the smallest terms first
#pragma unroll
            for (int i = 0; i < NC; ++i)
              sv = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kb[u][i], __builtin_bit_cast(bf16x8, q[qt][j][i]), sv, 0, 0, 0);
          const float f = sc * t.ks[u];
#pragma unroll
          for (int i = 0; i < 4; ++i) x[u][i] = log2_score(sv[i], f);
        }
        if (!full) {
#pragma unroll
          for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int i = 0; i < 4; ++i) x[u][i] = lg * 4 + i < (live >> (8 * u) & 255) ? x[u][i] : TA_NEG_INF;
        }
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
          for (int i = 0; i < 4; ++i) top = fmaxf(top, x[u][i]);
        if (wave_any(top - ref[qt] > PA_SLACK)) {
          const float to = fmaxf(ref[qt], quad_max(top)), f = __builtin_amdgcn_exp2f(ref[qt] - to);
          ref[qt] = to;
          l[qt] *= f;
#pragma unroll
          for (int e = 0; e < DE; ++e) o[qt][e] *= f;
        }
        float p[8];
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
          for (int i = 0; i < 4; ++i) p[4 * u + i] = __builtin_amdgcn_exp2f(x[u][i] - ref[qt]);
#pragma unroll
        for (int u = 0; u < 2; ++u) l[qt] += (p[4 * u] + p[4 * u + 1]) + (p[4 * u + 2] + p[4 * u + 3]);
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
          for (int i = 0; i < 4; ++i) p[4 * u + i] *= t.vs[u] * Shift::VALUE;
        bf16x8 pt[NP];
        bf16_terms<NP>(p, pt);
#pragma unroll
        for (int e = 0; e < DE; ++e)
#pragma unroll
          for (int j = NP - 1; j >= 0; --j) o[qt][e] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(va[e], pt[j], o[qt][e], 0, 0, 0);
      }
    }
  };

  int key = c0 + wave * KS;
  if (key < c1) {
    Tile ta, tb;
    int la = fetch(ta, key);
    // The first term of an infinite value is all of it: NaN from the others would hide scores of -inf, which take no part. Looked
    // for in products of pairs, and behind the first loads, so that they need not wait for the queries (16 sequences of 501 to
    // 10,001 rows 31.0 us as without it; 31.6 before the loads, or with a choice for each value).
    if constexpr (NQ == 3)
      if (wave_any(!(__builtin_fabsf(finite) < -TA_NEG_INF))) {
#pragma unroll
        for (int t = 0; t < QT; ++t) {
          const int r = (qt0 * QT + t) * 16 + lr;
          if (r >= rows) continue;
#pragma unroll
          for (int i = 0; i < NC; ++i) {
            const uint32_t* v = (const uint32_t*)(row(r) + dims(i) * 4);
            uint32_t keep[4];
#pragma unroll
            for (int e = 0; e < 4; ++e)
              keep[e] = ((v[2 * e] & 0x7fffffffu) == 0x7f800000u ? 0u : 0xffffu) | ((v[2 * e + 1] & 0x7fffffffu) == 0x7f800000u ? 0u : 0xffff0000u);
#pragma unroll
            for (int j = 1; j < NQ; ++j) {
              q[t][j][i].x &= keep[0], q[t][j][i].y &= keep[1], q[t][j][i].z &= keep[2], q[t][j][i].w &= keep[3];
            }
          }
        }
      }
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
      const float inv = l[t] == 0.f ? 0.f : 1.f / l[t], out = slot >= 0 ? 1.f : inv * (1.f / Shift::VALUE);
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
        store_row<T, 4 * DE>((T*)a.out + n * a.o_sn + (h * G + r / Tn) * a.o_sh + (t0 + r % Tn) * a.o_st + lg * 4 * DE, x);
        if (z.stat && lg == 0) z.stat[(int64_t)nh * rows + r] = make_float2(ref[t], inv);
      }
    }
  }
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

// Joins the partials of a query row in a wave, 4 values of a partial output per lane, 256 / D partials at a time: `slot(i)` is
// the i-th one's place. Every group of lanes joins its share by itself (their loads wait for nothing but the slots), then the
// groups are joined. Returns the normalised values of columns 4 (lane % (D / 4)) on; m, inv: the reference and 1 / sum.
template <typename Shift, int D, typename F>
__device__ __forceinline__ f32x4 pa_join(const PagedSplit& z, int parts, F slot, float* ref, float* inverse) {
  constexpr int LPR = D / 4, GR = 64 / LPR;
  const int lane = threadIdx.x & 63;
  float m = PA_REF0, l = 0.f;
  f32x4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
  for (int i = lane / LPR; i < parts; i += GR) {
    const float2 v = z.ml[slot(i)];
    const f32x4 x = *(const f32x4*)(z.part + slot(i) * D + lane % LPR * 4);
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
  *ref = m;
  *inverse = l == 0.f ? 0.f : 1.f / l;
  return o * (*inverse * (1.f / Shift::VALUE));
}

// A query row of pa_kernel's: rows that it has written itself are left alone; rows without a key become 0.
template <typename T, typename C, int D, int QT>
__device__ __forceinline__ void pa_merge_row(const PagedAttn& a, const PagedSplit& z, int64_t row) {
  constexpr int LPR = D / 4;
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
  float m, inv;
  const f32x4 o = pa_join<PagedShift<T, C>, D>(z, p.parts, [&](int i) { return p.slot(i); }, &m, &inv);
  if (lane < LPR) store4(op, o);
  if (z.stat && lane == 0) z.stat[row] = make_float2(m, inv);
}

// Waves per SIMD that the registers of a kernel allow: one for tiles of 32 and 64 query rows of 128 dims. In tiles of 16 with
// two waves every tile reads K and V again (tiles of 16 / larger: bf16, 32 query rows a head over 8 x 5,000 rows 57 / 42 us,
// 64 rows 104 / 48; fp32, 17 rows 102 / 70, 34 rows over 49 x 5,311 372 / 304).
// Over 8-bit rows 32 bf16 query rows of 128 dims fit beside a second wave.
constexpr int pa_waves(int D, int QT) { return D == 128 && QT > 1 ? 1 : 2; }
template <typename T, typename C>
constexpr int pa_waves_of(int D, int QT) { return sizeof(C) > 1 ? pa_waves(D, QT) : D == 128 && QT > 1 && sizeof(T) == 4 ? 1 : 2; }

// Equal shares of all items' units.
template <typename T, typename C, int D, int QT, bool W, bool ONCE = false>
__global__ __launch_bounds__(256, (pa_waves_of<T, C>(D, QT))) void pa_kernel(PagedAttn a, PagedSplit z) {
  const int per = a.pool.H * z.qtiles;
  PagedUnits units(a, per, threadIdx.x & 63);
  if constexpr (sizeof(C) == 1) units.weigh(PagedShares(z, units.total).share, PA_EXTRA8);
  const PagedShares shares(z, units.total);
  if ((int)blockIdx.x >= shares.groups) return;
  int unit = shares.first(blockIdx.x);
  const int end = shares.first(blockIdx.x + 1);
  while (unit < end) {
    int first;
    const int n = units.find(unit, &first);
    const int len = __builtin_amdgcn_readfirstlane(pa_len(a, n)), each = pa_each(len, units.extra);
    const int item = (unit - first) / each, u0 = unit - first - item * each;
    const int u1 = u0 + end - unit < each ? u0 + end - unit : each;
    if (threadIdx.x == 0 && u0 == 0) z.ends[n * per + item].x = blockIdx.x;
    if (threadIdx.x == 0 && u1 == each) z.ends[n * per + item].y = blockIdx.x;
    pa_segment<T, C, D, QT, W, false, 4, ONCE>(a, z, n, item / z.qtiles, 0, item % z.qtiles, u0 * PA_UNIT < len ? u0 * PA_UNIT : len,
                                               u1 * PA_UNIT < len ? u1 * PA_UNIT : len,
                                               u1 - u0 < each ? 2 * blockIdx.x + (u0 == 0) : -1);
    unit += u1 - u0;
  }
}

// A workgroup of NW waves for each item, where no sequence is long.
template <typename T, typename C, int D, int QT, bool W, int NW = 8, bool ONCE = false>
__global__ __launch_bounds__(64 * NW, 2) void pa_whole_kernel(PagedAttn a, PagedSplit z) {
  const int per = a.pool.H * z.qtiles, n = blockIdx.x / per, item = blockIdx.x % per;
  pa_segment<T, C, D, QT, W, false, NW, ONCE>(a, z, n, item / z.qtiles, 0, item % z.qtiles, 0,
                                             __builtin_amdgcn_readfirstlane(pa_len(a, n)), -1);
}

template <typename T, typename C, int D, int QT>
__global__ __launch_bounds__(256) void pa_merge_kernel(PagedAttn a, PagedSplit z) {
  pa_merge_row<T, C, D, QT>(a, z, (int64_t)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6));
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

}  // namespace
