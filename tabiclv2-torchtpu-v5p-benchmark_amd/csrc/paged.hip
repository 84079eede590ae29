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
// to 16 QT of its query rows (the heads of a group and the query rows together), its NW waves take turns of KS rows.
// Nothing of K and V is shared between waves, so they go from memory straight into the registers of the matrix products,
// a turn ahead of their use; LDS only joins the waves at the end.
//   S^T = K Q^T  (16 keys x 16 queries): the A operand is 16 bytes of a K row per lane, the result holds query l % 16,
//                keys 4 (l / 16) + i, which is the B operand of
//   O^T = V^T P^T with the keys in that order: the A operand holds the values of column group l % 16 (D / 16 columns, one
//                per product) of those keys; in bf16 the halves of pairs of rows are regrouped by v_perm_b32.
// bf16 probabilities enter as two bf16 terms (2^-16 of each left out), so that the output is off by its own rounding
// alone; the second product costs nothing beside the loads. fp32 runs on the fp32 matrix unit.
// Softmax: p = 2^(s - ref) with ref the running maximum + PA_SHIFT, moved only when a score passes it by more than 2^8
// (one test per turn); the shift keeps sums of 2^30 products with values near the largest float finite.
constexpr float PA_SHIFT = 24.f, PA_SLACK = 8.f;
constexpr float PA_REF0 = -3.4028234663852886e38f;

// The work is cut on the device, by the lengths as they are: a unit is PA_UNIT rows of one item (sequence, K/V head, query
// tile), units are counted item after item, and workgroup w of G takes the units [w T / G, (w + 1) T / G) of all T: an equal
// share whatever the lengths, with G two per CU. An item that one workgroup covers is
// written at once; of the others each workgroup leaves a partial (at most two: one of an item begun before it, one of an
// item it begins), which pa_merge_kernel joins. (A fixed number of rows per workgroup: 64 sequences of 500 to 10,000 rows
// took 97 us at 8 workgroups per CU and 146 at 2, one sequence of 45,000 rows 39 and 27.)
constexpr int PA_UNIT = 128, PA_WHOLE = 1024;

struct PagedSplit {
  int groups;    // G, or 0: a workgroup of eight waves for each item
  int least;     // units a workgroup takes at least
  int qtiles;
  float* part;   // [2 G][16 QT][D] unnormalised outputs
  float2* ml;    // [2 G][16 QT] (ref, sum)
  float2* stat;  // [N Hq Tq] (ref, 1 / sum), for the weights
  float* score;  // [N Hq Tq][score_sn] scores in log2 units, for the weights
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
  // the first unit of sequence n
  __device__ __forceinline__ int before(int n) const {
    int u = own, s = upto;
    for (int base = 64; base <= n; base += 64) {
      const int sum = __builtin_amdgcn_readlane(s, 63);
      u = load(base);
      s = wave_sum_scan(u) + sum;
    }
    return __builtin_amdgcn_readlane(s - u, n & 63);
  }
};

// Equal shares: `groups` workgroups (fewer, if they would get less than `least` units) of `share` units, the first `more`
// of them one more.
struct PagedShares {
  int groups, share, more;
  __device__ __forceinline__ PagedShares(const PagedSplit& z, int total) {
    groups = total / z.least;
    groups = groups < 1 ? 1 : groups < z.groups ? groups : z.groups;
    share = total / groups;
    more = total - share * groups;
  }
  __device__ __forceinline__ int first(int w) const { return w * share + (w < more ? w : more); }
  // the workgroup that holds unit t
  __device__ __forceinline__ int holder(int t) const {
    const int big = more * (share + 1);
    return t < big ? t / (share + 1) : more + (t - big) / share;
  }
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

template <typename T, int D, int QT, bool W, int NW>
__global__ __launch_bounds__(64 * NW, 2) void pa_kernel(PagedAttn a, PagedSplit z) {
  typedef PagedTile<T, D> Tile;
  constexpr int SUB = Tile::SUB, KS = Tile::KS, NC = Tile::NC, DE = Tile::DE, ES = Tile::ES;
  __shared__ float sh_o[NW / 2][16 * QT][D + 4];
  __shared__ float2 sh_ml[NW / 2][16 * QT];
  const PagedPool& c = a.pool;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lr = lane & 15, lg = lane >> 4;
  const int G = a.Hq / c.H, rows = G * a.Tq;
  const float sc = a.scale * TA_LOG2E;
  const uint32_t koff = lr * D * ES + lg * 16, voff = lg * 4 * D * ES + lr * DE * ES;
  const int per = c.H * z.qtiles;
  int unit = 0, end = 1, n = 0, first = 0;
  const PagedUnits units(a, per, lane);
  if (z.groups) {
    const PagedShares shares(z, units.total);
    if ((int)blockIdx.x >= shares.groups) return;
    unit = shares.first(blockIdx.x);
    end = shares.first(blockIdx.x + 1);
  }
  while (unit < end) {
  // the segment: rows [c0, c1) of an item
  int item, c0, c1, slot = -1;
  if (z.groups) {
    n = units.find(unit, &first);
    const int len = __builtin_amdgcn_readfirstlane(pa_len(a, n)), each = pa_units(len);
    item = (unit - first) / each;
    const int u0 = unit - first - item * each, u1 = u0 + end - unit < each ? u0 + end - unit : each;
    c0 = u0 * PA_UNIT;
    c1 = u1 * PA_UNIT < len ? u1 * PA_UNIT : len;
    if (u1 - u0 < each) slot = 2 * blockIdx.x + (u0 == 0);
    unit += u1 - u0;
  } else {
    n = blockIdx.x / per;
    item = blockIdx.x % per;
    c0 = 0;
    c1 = __builtin_amdgcn_readfirstlane(pa_len(a, n));
    unit = end;
  }
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
          x[s][i] = lg * 4 + i < (live >> (8 * s) & 255) ? x[s][i] : TA_NEG_INF;
          above |= x[s][i] - ref[qt] > PA_SLACK - PA_SHIFT;
        }
        if constexpr (W) {
          const int r = (qt0 * QT + qt) * 16 + lr;
          if (r < rows && key < c1)
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
      if constexpr (QT > 1) __builtin_amdgcn_sched_barrier(0);  // one query tile's scores and probabilities live at a time
    }
  };

  int key = c0 + wave * KS;
  if (key < c1) {
    Tile ta, tb;
    int la = fetch(ta, key);
    for (; key < c1; key += 2 * NW * KS) {  // two turns: the second may be past the end, then its weights are 0
      const int lb = fetch(tb, key + NW * KS);
      compute(ta, key, la);
      la = fetch(ta, key + 2 * NW * KS);
      compute(tb, key + NW * KS, lb);
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
      if (slot >= 0) {
        const int64_t at = (int64_t)slot * 16 * QT + t * 16 + lr;
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
  }
}

// Joins the partials of one query row per wave: 4 values of a partial output per lane, 256 / D partials at a time. Rows
// that pa_kernel has written are left alone; rows without a key become 0.
template <typename T, int D, int QT, bool W>
__global__ __launch_bounds__(256) void pa_merge_kernel(PagedAttn a, PagedSplit z) {
  constexpr int LPR = D / 4, GR = 64 / LPR;
  const int lane = threadIdx.x & 63, G = a.Hq / a.pool.H, rows = G * a.Tq;
  const int64_t row = (int64_t)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (row >= (int64_t)a.N * a.pool.H * rows) return;
  const int r = (int)(row % rows), nh = (int)(row / rows), n = nh / a.pool.H, h = nh % a.pool.H;
  const PagedUnits units(a, a.pool.H * z.qtiles, lane);
  const PagedShares shares(z, units.total);
  const int each = pa_units(__builtin_amdgcn_readfirstlane(pa_len(a, n)));
  T* op = (T*)a.out + n * a.o_sn + (h * G + r / a.Tq) * a.o_sh + (r % a.Tq) * a.o_st + lane * 4;
  if (each == 0) {
    if (lane < LPR)
#pragma unroll
      for (int i = 0; i < 4; ++i) op[i] = (T)0.f;
    return;
  }
  // the workgroups of the item's first and last unit
  const int t0 = units.before(n) + (h * z.qtiles + r / (16 * QT)) * each;
  const int w0 = shares.holder(t0), w1 = shares.holder(t0 + each - 1);
  if (w0 == w1) return;
  const int parts = w1 - w0 + 1, at = r % (16 * QT);
  auto slot = [&](int i) { return (int64_t)(2 * (w0 + i) + (i == 0)) * (16 * QT) + at; };
  // every group of lanes joins its share of the partials by itself (their loads wait for nothing but the lengths), then
  // the groups are joined
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
  const float inv = l == 0.f ? 0.f : 1.f / l;
  if (lane < LPR)
#pragma unroll
    for (int i = 0; i < 4; ++i) op[i] = (T)(o[i] * inv);
  if (W && lane == 0) z.stat[row] = make_float2(m, inv);
}

// weights[n, i] += sum over the query rows of p: 64 keys per workgroup, 4 per thread, the query rows over 16 threads
// (each in steps of 16), joined in a fixed order.
__global__ __launch_bounds__(256) void pa_weights_kernel(PagedAttn a, PagedSplit z) {
  __shared__ f32x4 sh[16][16];
  const int n = blockIdx.y, len = pa_len(a, n), k0 = blockIdx.x * 64;
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
template <typename T, int D, int QT>
int64_t paged_split(PagedSplit* z, char* ws, int64_t N, int64_t Hq, int64_t H, int64_t Tq, int64_t rows, bool weights) {
  const int64_t qrows = Hq / H * Tq;
  z->qtiles = (int)((qrows + 16 * QT - 1) / (16 * QT));
  // Two workgroups per CU keep enough loads in flight (three: 3% slower on long caches, 30% at 64 query rows). Up to
  // PA_WHOLE rows an item goes to one workgroup of eight waves, without a merge: one row over 8 x 700 rows 10.9 us on the
  // GPU against 11.2 and a launch less for the host; over 8 x 2,000 rows 16.7 against 15.2.
  z->groups = rows <= PA_WHOLE ? 0 : 2 * cu_count();
  z->least = 2;
  int64_t at = 0;
  auto take = [&](int64_t bytes) {
    char* p = ws + at;
    at += align256(bytes);
    return p;
  };
  const int64_t all = N * H * qrows;
  z->part = (float*)take((int64_t)z->groups * 2 * 16 * QT * D * 4);
  z->ml = (float2*)take((int64_t)z->groups * 2 * 16 * QT * 8);
  z->score_sn = (rows + 63) / 64 * 64;
  z->stat = (float2*)take(weights ? all * 8 : 0);
  z->score = (float*)take(weights ? all * z->score_sn * 4 : 0);
  return at;
}

template <typename T, int D, int QT, bool W>
void launch_pa_w(const PagedAttn& a, const PagedSplit& z, hipStream_t stream) {
  if (z.groups == 0) {
    hipLaunchKernelGGL((pa_kernel<T, D, QT, W, 8>), dim3((unsigned)(a.N * a.pool.H * z.qtiles)), dim3(512), 0, stream, a, z);
  } else {
    hipLaunchKernelGGL((pa_kernel<T, D, QT, W, 4>), dim3((unsigned)z.groups), dim3(256), 0, stream, a, z);
    const unsigned merge = (unsigned)(((int64_t)a.N * a.Hq * a.Tq + 3) / 4);
    hipLaunchKernelGGL((pa_merge_kernel<T, D, QT, W>), dim3(merge), dim3(256), 0, stream, a, z);
  }
  if (W && z.score_sn)
    hipLaunchKernelGGL(pa_weights_kernel, dim3((unsigned)(z.score_sn / 64), a.N), dim3(256), 0, stream, a, z);
}

// Launches (a != null) or sizes the workspace.
template <typename T, int D, int QT>
int64_t run_pa(const PagedAttn* a, void* ws, int64_t N, int64_t Hq, int64_t H, int64_t Tq, int64_t rows, bool weights,
               hipStream_t stream) {
  PagedSplit z;
  const int64_t bytes = paged_split<T, D, QT>(&z, (char*)ws, N, Hq, H, Tq, rows, weights);
  if (a && weights) launch_pa_w<T, D, QT, true>(*a, z, stream);
  else if (a) launch_pa_w<T, D, QT, false>(*a, z, stream);
  return bytes;
}

template <typename T, int D>
int64_t run_pa_d(const PagedAttn* a, void* ws, int64_t N, int64_t Hq, int64_t H, int64_t Tq, int64_t rows, bool weights,
                 hipStream_t stream) {
  const int64_t qrows = Hq / H * Tq;
  constexpr int most = D == 128 ? 1 : D * sizeof(T) > 128 ? 2 : 4;  // more queries do not fit the registers
  if constexpr (most >= 4)
    if (qrows > 32) return run_pa<T, D, 4>(a, ws, N, Hq, H, Tq, rows, weights, stream);
  if constexpr (most >= 2)
    if (qrows > 16) return run_pa<T, D, 2>(a, ws, N, Hq, H, Tq, rows, weights, stream);
  return run_pa<T, D, 1>(a, ws, N, Hq, H, Tq, rows, weights, stream);
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
