// Attention of few query rows over selected pages of a paged K/V cache (gfx950): bounds of the keys of each page, the pages
// whose bounds promise a query row the largest scores, attention over those pages alone.
//
//   hi_d = ceil(max_i K_id / s),  lo_d = floor(min_i K_id / s)           int8, one s = 2^k per page and head
//   u_d = round(q_d / 2^j)                                              int8, one j per query row (of all heads of a group)
//   bound = max over the group's heads of sum_d (u+_d hi_d + u-_d lo_d) s,   u+ hi + u- lo = max(u hi, u lo)
//
// A sum of whole numbers below 2^24 times a power of two is exact in fp32: the K pages of largest bound (ties: the lower page)
// are the same however it is added up. hi and lo take 2 D bytes per page and head, 1/64 of a page of 64 bf16 rows.
#include "launch.h"
#include "paged_core.h"

#include <type_traits>

namespace {

typedef int i32x4 __attribute__((ext_vector_type(4)));

// The exponent k of the smallest 2^k, k in [-60, 100], with m <= 127 2^k (m: the bits of a finite value >= 0).
__device__ __forceinline__ int step_exponent(uint32_t m) {
  const int k = (int)(m >> 23) - 133 + ((m & 0x7fffffu) > 0x7e0000u);  // 127 = 1.984375 2^6
  return k < -60 ? -60 : k < 100 ? k : 100;
}
__device__ __forceinline__ float pow2(int k) { return __uint_as_float((uint32_t)(k + 127) << 23); }
__device__ __forceinline__ uint32_t finite_bits(float x) {
  const uint32_t u = __float_as_uint(x) & 0x7fffffffu;
  return u < 0x7f800000u ? u : 0;
}
__device__ __forceinline__ uint32_t umax(uint32_t a, uint32_t b) { return a > b ? a : b; }

// ---------------------------------------------------------------------------------------------
// bounds
// ---------------------------------------------------------------------------------------------
// 16 bytes of a row as fp32 values (codes without their scale).
template <typename C>
__device__ __forceinline__ void values16(uint4 u, float* x);
template <>
__device__ __forceinline__ void values16<bf16>(uint4 u, float* x) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) x[2 * i] = __uint_as_float(w[i] << 16), x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
}
template <>
__device__ __forceinline__ void values16<float>(uint4 u, float* x) {
  x[0] = __uint_as_float(u.x), x[1] = __uint_as_float(u.y), x[2] = __uint_as_float(u.z), x[3] = __uint_as_float(u.w);
}
template <>
__device__ __forceinline__ void values16<E4M3>(uint4 u, float* x) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8(w[i], false), hi = __builtin_amdgcn_cvt_pk_f32_fp8(w[i], true);
    x[4 * i] = lo[0], x[4 * i + 1] = lo[1], x[4 * i + 2] = hi[0], x[4 * i + 3] = hi[1];
  }
}
template <>
__device__ __forceinline__ void values16<I8>(uint4 u, float* x) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 16; ++i) x[i] = (float)(int8_t)(w[i / 4] >> (8 * (i % 4)));
}

// The largest and the smallest value of each dim in a lane's 16 bytes, over the rows added. Two 16-bit numbers at a time:
// 8-bit codes take the upper byte of one (even and odd bytes apart; what the lower byte holds decides nothing). Numbers in
// sign and magnitude (bf16, e4m3) order as integers apart from their signs: the largest as signed is the largest value, if there
// is one >= 0; the largest as unsigned the smallest, if there is a negative one; else the smallest as unsigned is either. A NaN
// shows as a magnitude beyond infinity (or the e4m3 NaN), and its page is gone through again value by value. (fp32 values one
// by one, with unpacking: 12 instructions for 16 bytes instead of 28 in bf16; 45,000 rows of 8 sequences and heads 79 -> 68 us,
// bound by the reads of K then.)
typedef short s16x2 __attribute__((ext_vector_type(2)));
typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
template <typename F>
__device__ __forceinline__ uint32_t across(uint32_t x, int lanes, F f) {
  if (lanes == 16) {
    const auto r = __builtin_amdgcn_permlane16_swap(x, x, false, false);
    return f(r[0], r[1]);
  }
  if (lanes == 32) {
    const auto r = __builtin_amdgcn_permlane32_swap(x, x, false, false);
    return f(r[0], r[1]);
  }
  return f(x, (uint32_t)__shfl_xor((int)x, lanes, 64));
}
__device__ __forceinline__ uint32_t max_i16(uint32_t a, uint32_t b) {
  return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(s16x2, a), __builtin_bit_cast(s16x2, b)));
}
__device__ __forceinline__ uint32_t min_i16(uint32_t a, uint32_t b) {
  return __builtin_bit_cast(uint32_t, __builtin_elementwise_min(__builtin_bit_cast(s16x2, a), __builtin_bit_cast(s16x2, b)));
}
__device__ __forceinline__ uint32_t max_u16(uint32_t a, uint32_t b) {
  return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(u16x2, a), __builtin_bit_cast(u16x2, b)));
}
__device__ __forceinline__ uint32_t min_u16(uint32_t a, uint32_t b) {
  return __builtin_bit_cast(uint32_t, __builtin_elementwise_min(__builtin_bit_cast(u16x2, a), __builtin_bit_cast(u16x2, b)));
}
__device__ __forceinline__ uint32_t max_f32(uint32_t a, uint32_t b) { return __float_as_uint(fmaxf(__uint_as_float(a), __uint_as_float(b))); }
__device__ __forceinline__ uint32_t min_f32(uint32_t a, uint32_t b) { return __float_as_uint(fminf(__uint_as_float(a), __uint_as_float(b))); }

// One of N registers by a number that differs between lanes (by masks: a choice between array elements would become an
// address, and the array go to memory).
template <int N>
__device__ __forceinline__ uint32_t choose(const uint32_t* x, int i) {
  if constexpr (N == 1) {
    return x[0];
  } else {
    const uint32_t upper = i & (N / 2) ? 0xffffffffu : 0u;
    return (choose<N / 2>(x + N / 2, i) & upper) | (choose<N / 2>(x, i) & ~upper);
  }
}

template <typename C>
struct Extremes {
  static constexpr int ES = sizeof(C), W = ES == 1 ? 8 : 4, VPC = 16 / ES;  // registers, values of 16 bytes
  static constexpr bool SIGNED = std::is_same<C, I8>::value, FLOAT = ES == 4;
  uint32_t a[W], b[W], c[W];  // max signed, max unsigned, min unsigned; int8, fp32: max, min
  __device__ __forceinline__ Extremes() {
#pragma unroll
    for (int i = 0; i < W; ++i) {
      a[i] = FLOAT ? 0xff800000u : 0x80008000u;
      b[i] = FLOAT ? 0x7f800000u : SIGNED ? 0x7fff7fffu : 0u;
      c[i] = 0xffffffffu;
    }
  }
  __device__ __forceinline__ void merge(int i, uint32_t x, uint32_t y, uint32_t z) {
    a[i] = FLOAT ? max_f32(a[i], x) : max_i16(a[i], x);
    b[i] = FLOAT ? min_f32(b[i], y) : SIGNED ? min_i16(b[i], y) : max_u16(b[i], y);
    if (!FLOAT && !SIGNED) c[i] = min_u16(c[i], z);
  }
  __device__ __forceinline__ void add(uint4 u) {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (ES == 1) {
        const uint32_t even = w[i] << 8;
        merge(2 * i, even, even, even);
        merge(2 * i + 1, w[i], w[i], w[i]);
      } else {
        merge(i, w[i], w[i], w[i]);
      }
    }
  }
  __device__ __forceinline__ void join(int lanes) {
#pragma unroll
    for (int i = 0; i < W; ++i) {
      a[i] = across(a[i], lanes, FLOAT ? max_f32 : max_i16);
      b[i] = across(b[i], lanes, FLOAT ? min_f32 : SIGNED ? min_i16 : max_u16);
      if (!FLOAT && !SIGNED) c[i] = across(c[i], lanes, min_u16);
    }
  }
  // The extremes of value e (of the 16 bytes; e differs between lanes); false where a NaN hides them.
  __device__ __forceinline__ bool value(int e, float* hi, float* lo) const {
    if constexpr (FLOAT) {
      *hi = __uint_as_float(choose<4>(a, e)), *lo = __uint_as_float(choose<4>(b, e));
      return true;  // fmaxf and fminf pass a NaN by
    } else {
      const int w = ES == 1 ? e / 4 * 2 + (e & 1) : e / 2, shift = (ES == 1 ? e >> 1 & 1 : e & 1) * 16;
      const uint32_t x = choose<W>(a, w) >> shift & 0xffffu, y = choose<W>(b, w) >> shift & 0xffffu;
      if constexpr (SIGNED) {
        *hi = (float)(int8_t)(x >> 8), *lo = (float)(int8_t)(y >> 8);
        return true;
      } else {
        const uint32_t z = choose<W>(c, w) >> shift & 0xffffu, p = x & 0x8000u ? z : x, m = y & 0x8000u ? y : z;
        if constexpr (ES == 2) {
          *hi = __uint_as_float(p << 16), *lo = __uint_as_float(m << 16);
          return !((x & 0x8000u) == 0 && x > 0x7f80u) && y <= 0xff80u;
        } else {
          const auto v = __builtin_amdgcn_cvt_pk_f32_fp8(p >> 8 | (m & 0xff00u), false);
          *hi = v[0], *lo = v[1];
          return x >> 8 != 0x7f && y >> 8 != 0xff;
        }
      }
    }
  }
};

// One wave per page and head. Bound by the bytes of K, which nothing reads again soon: loads that leave the caches alone (8 x
// 45,000 rows in bf16 78 -> 62 us).
template <typename C, int D>
__global__ __launch_bounds__(256) void paged_bounds_kernel(PagedBounds a) {
  constexpr int ES = sizeof(C), VPC = 16 / ES, LPR = D / VPC, RPP = 64 / LPR;  // values of 16 bytes, lanes of a row, rows of a pass
  constexpr int DPL = D < 64 ? 1 : D / 64;                                     // dims that a lane finishes
  const PagedPool& c = a.pool;
  const int n = blockIdx.y, item = blockIdx.x * 4 + (threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int h = item % c.H, len = pool_length(c, n), R = 1 << c.shift;
  int first = a.start ? a.start[n] : 0;
  first = first < 0 ? 0 : first;
  const int64_t p = (first >> c.shift) + (int64_t)(item / c.H), row0 = p << c.shift;
  if (row0 >= len) return;
  const int page = c.table[n * c.table_sn + p];
  if (page < 0 || page >= c.pages) return;
  const int live = len - row0 < R ? (int)(len - row0) : R;
  const char* k = (const char*)c.k + (page * c.page_sp + (int64_t)h * R * D) * ES + lane % LPR * 16;
  Extremes<C> ext;
  int r = lane / LPR;
  for (; r + 7 * RPP < live; r += 8 * RPP) {
    uint4 u[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) u[i] = ldg16_once(k + (int64_t)(r + i * RPP) * D * ES);
#pragma unroll
    for (int i = 0; i < 8; ++i) ext.add(u[i]);
  }
  for (; r < live; r += RPP) ext.add(ldg16(k + (int64_t)r * D * ES));
#pragma unroll
  for (int x = LPR; x < 64; x <<= 1) ext.join(x);
  // every lane has the extremes of its VPC dims now, and finishes DPL of them (D = 32: two lanes or more the same one)
  const int e0 = lane / LPR * DPL % VPC, dim = lane % LPR * VPC + e0;
  float hi[DPL], lo[DPL];
  bool fine = true;
#pragma unroll
  for (int i = 0; i < DPL; ++i) fine &= ext.value(e0 + i, &hi[i], &lo[i]);
  if (wave_any(!fine)) {
#pragma unroll
    for (int i = 0; i < DPL; ++i) hi[i] = TA_NEG_INF, lo[i] = -TA_NEG_INF;
    for (int row = 0; row < live; ++row) {
      float x[VPC];
      values16<C>(ldg16(k + (int64_t)row * D * ES), x);
#pragma unroll
      for (int e = 0; e < VPC; ++e)
#pragma unroll
        for (int i = 0; i < DPL; ++i)
          if (e == e0 + i) hi[i] = fmaxf(hi[i], x[e]), lo[i] = fminf(lo[i], x[e]);
    }
  }
  uint32_t most = 0;
#pragma unroll
  for (int i = 0; i < DPL; ++i) {
    if constexpr (ES == 1) {
      const float s = a.scales[((int64_t)page * c.H + h) * 2];
      hi[i] *= s, lo[i] *= s;
    }
    if (hi[i] < lo[i]) hi[i] = lo[i] = 0.f;  // a dim of NaN alone
    most = umax(most, umax(finite_bits(lo[i]), finite_bits(hi[i])));
  }
#pragma unroll
  for (int x = 1; x < 64; x <<= 1) most = across(most, x, umax);
  const int e2 = step_exponent(most);
  const float inv = pow2(-e2);
  int8_t* out = a.bounds + ((int64_t)page * c.H + h) * 2 * D + dim;
#pragma unroll
  for (int i = 0; i < DPL; ++i) {
    // infinite bounds, and finite ones beyond the largest scale, at the end of the range
    out[i] = (int8_t)(int)fminf(fmaxf(ceilf(hi[i] * inv), -127.f), 127.f);
    out[D + i] = (int8_t)(int)fminf(fmaxf(floorf(lo[i] * inv), -127.f), 127.f);
  }
  if (lane == 0) a.bound_scales[(int64_t)page * c.H + h] = pow2(e2);
}

template <int D>
void launch_bounds(const PagedBounds& a, int format, dim3 grid, hipStream_t stream) {
  const dim3 nt(256);
  if (format == 0) hipLaunchKernelGGL((paged_bounds_kernel<bf16, D>), grid, nt, 0, stream, a);
  else if (format == 1) hipLaunchKernelGGL((paged_bounds_kernel<float, D>), grid, nt, 0, stream, a);
  else if (format == 2) hipLaunchKernelGGL((paged_bounds_kernel<E4M3, D>), grid, nt, 0, stream, a);
  else hipLaunchKernelGGL((paged_bounds_kernel<I8, D>), grid, nt, 0, stream, a);
}

// ---------------------------------------------------------------------------------------------
// selection
// ---------------------------------------------------------------------------------------------
// A workgroup of 16 waves (or 4) takes up to TT query rows of one sequence and K/V head: the bounds of 16 pages for 16 (query row,
// head of the group) pairs at a time on the 8-bit matrix unit, kept as ordered codes [TT][pages] in LDS (0: no such page); then
// the K-th largest code of each query row by four 8-bit digits of a histogram, 16 / TT (4 / TT) waves a row; then the pages above it,
// and the first ones equal to it, in order. Bound by its chain of loads and barriers (64 query rows of 704 pages: a few MB), so
// the first tile's table entries and bounds are on their way before the queries are looked at, the histograms of all
// digits are cleared at once, every wave of a row finds the digit for itself (one barrier a digit), and there is little code:
// most of it runs once, as fast as instructions come in (two tiles of bounds on their way instead of one: 0.4 us more). One row of 8
// sequences of 704 pages and 8 heads takes 8.4 us call after call in a graph (10.3 between other kernels, which leave it neither the
// bounds nor its code in the caches), of which the digits take 1.7; 64 pages 6.3, 16 of 16, unscored, 2.5.
constexpr int PS_LDS = 32768;  // codes kept in LDS

__device__ __forceinline__ uint32_t bound_code(float x) {  // larger bound, larger code; none is 0
  const uint32_t u = __float_as_uint(x + 0.f);
  const uint32_t v = u & 0x80000000u ? ~u : u | 0x80000000u;
  return v ? v : 1;
}
__device__ __forceinline__ int lanes_below(uint64_t mask) {
  return __builtin_amdgcn_mbcnt_hi((uint32_t)(mask >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)mask, 0));
}

// A tile of 16 pages (the waves take turns): their bounds as operands, their scales and whether they are there. The table is
// read up to its width, not the sequence's, so that its entries need not wait for the length. Lanes without a page load another
// one's: a load under a condition would have every wait wait for all loads.
__device__ __forceinline__ int tile_page(const PagedSelect& a, const int32_t* table, int tile, int lr) {
  const uint32_t p = tile * 16 + lr, last = a.pool.max_pages - 1, at = p < last ? p : last;
  const int id = table[at];
  return p <= last ? id : -1;
}
// The bounds come in with four lanes side by side on 64 bytes of a page (16 lanes on 16 pages, as the operands lie, are 16 lines
// of the cache for every 16 lanes: 8 heads of a sequence of 3,125 pages 22.8 us for 16.6) and are passed on through LDS.
template <int KB>
struct BoundTile {
  i32x4 b[KB];  // 16 bytes from 16 (lane % 4) on of each 64, of page lane / 4
  float scale;  // of page lane % 16
  bool in;
  // bounds, scales: page 0's, from this head and lane's on; page: page lane % 16
  __device__ __forceinline__ void load(const PagedSelect& a, const int8_t* bounds, const float* scales, int page, int p, int P) {
    in = (uint32_t)page < (uint32_t)a.pool.pages && p < P;
    const uint32_t at = in ? page : 0, mine = __shfl((int)at, (threadIdx.x & 63) >> 2, 64);
    scale = *(const float*)((const char*)scales + (uint64_t)at * (uint32_t)(a.pool.H * 4));
    const int8_t* from = bounds + (uint64_t)mine * (uint32_t)(a.pool.H * (KB * 64));
#pragma unroll
    for (int i = 0; i < KB; ++i) b[i] = *(const i32x4*)(from + i * 64);
  }
};

// Grid (tiles of TT = 2^tshift query rows, H, N). per16: 256 / G, rounded up (x / G = x * per16 >> 8 for x < 16; G <= 16).
template <typename T, int D, bool GLOBAL, int NW>
__global__ __launch_bounds__(NW * 64) void paged_select_kernel(PagedSelect a, int tshift, int per16, uint32_t* store) {
  extern __shared__ uint32_t lds[];  // [4][TT][256] histograms, [TT][max_pages] codes
  constexpr int KB = 2 * D / 64, NV = (D + 63) / 64, COLS = 16 / NW, LOGW = NW == 16 ? 4 : 2;
  __shared__ __attribute__((aligned(16))) int8_t sh_q[16][2 * D], sh_b[NW][1024];
  __shared__ uint32_t sh_most[16];
  __shared__ int2 part[NW];
  const PagedPool& c = a.pool;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lr = lane & 15, lg = lane >> 4;
  const int n = blockIdx.z, h = blockIdx.y, TT = 1 << tshift, t0 = blockIdx.x << tshift;
  const int G = a.Hq / c.H, R = 1 << c.shift, len = __builtin_amdgcn_readfirstlane(pool_length(c, n));
  const int P = c.pages > 0 ? (len + R - 1) >> c.shift : 0, stride = c.max_pages;
  const int32_t* table = c.table + n * c.table_sn;
  int* hist = (int*)lds;
  const int64_t nh = (int64_t)n * c.H + h;
  uint32_t* codes = GLOBAL ? store + (nh * a.Tq + t0) * stride : lds + (1024 << tshift);
  const int8_t* bounds = a.bounds + h * (2 * D) + (lane & 3) * 16;
  // 64 bytes of a tile's pages in LDS, their sixteenths in an order by which neither side meets itself in a bank
  int8_t* const put = sh_b[wave] + (lane >> 2) * 64 + ((lane ^ lane >> 3) & 3) * 16;
  const int8_t* const get = sh_b[wave] + lr * 64 + ((lg ^ lr >> 1) & 3) * 16;
  const float* scales = a.bound_scales + h;
  BoundTile<KB> b;
  int page = c.max_pages > 0 ? tile_page(a, table, wave, lr) : -1;  // of the tile after b's
  auto first = [&]() {
    b.load(a, bounds, scales, page, wave * 16 + lr, P);
    page = tile_page(a, table, wave + NW, lr);
  };
  if (a.K < P) {
    first();
    // columns wave, wave + NW, ... of the queries: with up to 16 heads in the group (query row, head), else 16 heads at a time
    const char* q = (const char*)a.q + (n * a.q_sn + (int64_t)h * G * a.q_sh) * sizeof(T);
    const bool wide = G > 16;
    float x[COLS][NV];
    auto columns = [&](int g0) {
#pragma unroll
      for (int s = 0; s < COLS; ++s) {
        const int col = wave + s * NW, row = wide ? 0 : col * per16 >> 8, g = g0 + col - row * G;
        const bool in = row < TT && t0 + row < a.Tq && g < G;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
          const int d = lane + 64 * i;
          x[s][i] = in && d < D ? (float)*(const T*)(q + (g * a.q_sh + (t0 + row) * a.q_st + d) * (int64_t)sizeof(T)) : 0.f;
        }
      }
    };
    uint32_t most[COLS] = {};
#pragma unroll 1
    for (int g0 = 0; g0 < G; g0 += 16) {
      columns(g0);
#pragma unroll
      for (int s = 0; s < COLS; ++s)
#pragma unroll
        for (int i = 0; i < NV; ++i) most[s] = umax(most[s], finite_bits(x[s][i]));
    }
#pragma unroll 1
    for (int i = threadIdx.x; i < 1024 << tshift; i += NW * 64) hist[i] = 0;
#pragma unroll 1
    for (int t = 0; t < TT; ++t)
#pragma unroll 1
      for (int i = threadIdx.x; i < P; i += NW * 64) codes[t * stride + i] = 0;
#pragma unroll
    for (int s = 0; s < COLS; ++s) {
#pragma unroll
      for (int y = 1; y < 64; y <<= 1) most[s] = across(most[s], y, umax);
      if (lane == 0) sh_most[wave + s * NW] = most[s];
    }
    __syncthreads();
    // the step of a column's query row: the largest of its group's
    float inv[COLS];
#pragma unroll
    for (int s = 0; s < COLS; ++s) {
      uint32_t m = 0;
      const int w0 = wide ? 0 : ((wave + s * NW) * per16 >> 8) * G, w1 = wide || w0 + G > 16 ? 16 : w0 + G;
#pragma unroll 1
      for (int w = w0; w < w1; ++w) m = umax(m, sh_most[w]);
      inv[s] = pow2(-step_exponent(m));
    }

#pragma unroll 1
    for (int g0 = 0; g0 < G; g0 += 16) {
      if (wide) columns(g0);
#pragma unroll
      for (int s = 0; s < COLS; ++s) {
        const int col = wave + s * NW;
        int8_t* place = sh_q[(col & 3) * 4 + (col >> 2)];
#pragma unroll
        for (int i = 0; i < NV; ++i) {
          const int d = lane + 64 * i;
          const int u = x[s][i] != x[s][i] ? 0 : (int)fminf(fmaxf(__builtin_rintf(x[s][i] * inv[s]), -127.f), 127.f);
          if (d < D) {
            place[d] = (int8_t)(u > 0 ? u : 0);
            place[D + d] = (int8_t)(u < 0 ? u : 0);
          }
        }
      }
      __syncthreads();
      // this lane's products are those of page lr with columns lg, lg + 4, ...
      const int left = wide ? G - g0 : TT * G, values = left < 16 ? (left + 3) >> 2 : 4;
      int to[4];
      bool mine[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int j = lg + 4 * i, t = wide ? 0 : j * per16 >> 8, g = g0 + j - t * G;
        mine[i] = t < TT && g < G && t0 + t < a.Tq;
        to[i] = t * stride + lr;
      }
      i32x4 qb[KB];
#pragma unroll
      for (int i = 0; i < KB; ++i) qb[i] = *(const i32x4*)(&sh_q[lr][i * 64 + lg * 16]);
      if (g0 > 0) {
        page = tile_page(a, table, wave, lr);
        first();
      }
      // a tile's bounds are on their way while the one before becomes codes, its table entries a tile earlier
#pragma unroll 1
      for (int tile = wave; tile * 16 < P; tile += NW) {
        const int p0 = tile * 16;
        i32x4 sum = {0, 0, 0, 0};
#pragma unroll
        for (int i = 0; i < KB; ++i) {
          *(i32x4*)put = b.b[i];
          __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");  // what other lanes of the wave wrote, in order
          const i32x4 operand = *(const i32x4*)get;
          __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
          sum = __builtin_amdgcn_mfma_i32_16x16x64_i8(qb[i], operand, sum, 0, 0, 0);
        }
        const bool in = b.in;
        const float scale = b.scale;
        b.load(a, bounds, scales, page, p0 + NW * 16 + lr, P);
        page = tile_page(a, table, tile + 2 * NW, lr);
        if (mine[0] && in) atomicMax(codes + to[0] + p0, bound_code((float)sum[0] * scale));
        if (values > 1)
#pragma unroll
          for (int i = 1; i < 4; ++i)
            if (mine[i] && in) atomicMax(codes + to[i] + p0, bound_code((float)sum[i] * scale));
      }
      __syncthreads();
    }
  } else {  // every page that is there, whatever its bound
#pragma unroll 1
    for (int i = threadIdx.x; i < P; i += NW * 64) {
      const uint32_t there = (uint32_t)table[i] < (uint32_t)c.pages;
#pragma unroll 1
      for (int t = 0; t < TT; ++t) codes[t * stride + i] = there;
    }
    __syncthreads();
  }

  // the rows in groups of waves
  const int wshift = LOGW - tshift, wpr = 1 << wshift, t = wave >> wshift, sub = wave & (wpr - 1), member = sub * 64 + lane, members = wpr * 64;
  const uint32_t* mycodes = codes + t * stride;
  int want = a.K < P ? a.K : 0;  // of the pages of the threshold's code, in the end; every page there is: 0
  uint32_t threshold = 0;
  if (a.K < P) {
    int* bins = hist + t * 256;
#pragma unroll 1
    for (int shift = 24; shift >= 0; shift -= 8, bins += 256 << tshift) {
#pragma unroll 1
      for (int i = member; i < P; i += members) {
        const uint32_t v = mycodes[i];
        if (shift == 24 || (v ^ threshold) >> (shift + 8) == 0) atomicAdd(&bins[v >> shift & 255], 1);
      }
      __syncthreads();
      // four bins a lane, counted from the top; the digit's bin is one lane's
      const int4 b = *(const int4*)(bins + 252 - 4 * lane);
      const int sum = b.x + b.y + b.z + b.w, before = wave_sum_scan(sum) - sum;
      const uint64_t hit = __ballot(before < want && before + sum >= want);
      const int at = hit ? __builtin_ctzll(hit) : 0;
      const int bw = __builtin_amdgcn_readlane(b.w, at), bz = __builtin_amdgcn_readlane(b.z, at), by = __builtin_amdgcn_readlane(b.y, at);
      int rest = want - __builtin_amdgcn_readlane(before, at), digit = 255 - 4 * at;
      if (rest > bw) {
        rest -= bw;
        --digit;
        if (rest > bz) {
          rest -= bz;
          --digit;
          if (rest > by) {
            rest -= by;
            --digit;
          }
        }
      }
      threshold |= (uint32_t)digit << shift;
      want = rest;
    }
  }
  if (threshold == 0) want = 0;  // fewer pages than K: those that are there
  // a run of pages per wave: what is taken before it, then the places
  const int run = ((P + members - 1) >> (6 + wshift)) * 64, p0 = sub * run, p1 = p0 + run < P ? p0 + run : P;
  int more = 0, even = 0;
#pragma unroll 1
  for (int p = p0 + lane; p - lane < p1; p += 64) {
    const uint32_t v = p < p1 ? mycodes[p] : 0;
    more += __popcll(__ballot(v > threshold));
    even += __popcll(__ballot(v == threshold && v != 0));
  }
  if (lane == 0) part[wave] = make_int2(more, even);
  __syncthreads();
  if (t0 + t >= a.Tq) return;
  const int2 mine = lane < wpr ? part[(t << wshift) + lane] : make_int2(0, 0);
  const int upm = wave_sum_scan(mine.x), upe = wave_sum_scan(mine.y);
  int more0 = sub ? __builtin_amdgcn_readlane(upm, sub - 1) : 0, even0 = sub ? __builtin_amdgcn_readlane(upe, sub - 1) : 0;
  const int evens = __builtin_amdgcn_readlane(upe, 63), all = __builtin_amdgcn_readlane(upm, 63) + (evens < want ? evens : want);
  int32_t* out = a.index + (nh * a.Tq + t0 + t) * a.K;
#pragma unroll 1
  for (int p = p0 + lane; p - lane < p1; p += 64) {
    const uint32_t v = p < p1 ? mycodes[p] : 0;
    const uint64_t above = __ballot(v > threshold), equal = __ballot(v == threshold && v != 0);
    const int rank = even0 + lanes_below(equal);
    if (v > threshold || (v == threshold && v != 0 && rank < want)) out[more0 + lanes_below(above) + (rank < want ? rank : want)] = p;
    more0 += __popcll(above);
    even0 += __popcll(equal);
  }
#pragma unroll 1
  for (int i = all + member; i < a.K; i += members) out[i] = -1;
}

// The query rows of a workgroup as a shift: a power of two with up to 16 (query row, head) pairs and a wave a row, whose codes and
// histograms fit in LDS.
int select_shift(int64_t G, int64_t Tq, int64_t max_pages, int most) {
  int s = 0;
  while (s < most && (1 << s) < Tq && (2 << s) * G <= 16 && (2 << s) * (max_pages + 1024) <= PS_LDS) ++s;
  return s;
}

template <typename T, int D>
void launch_select(const PagedSelect& a, void* ws, hipStream_t stream) {
  const int64_t G = a.Hq / a.pool.H, M = a.pool.max_pages;
  // Four waves for tables of up to 256 pages, so that many workgroups share a CU (us with 16 / 4 waves: 8 heads of 8 sequences of 64
  // pages 7.2 / 7.2, of 256 7.9 / 8.6, of 512 9.3 / 11.2; of 64 sequences of 64 pages 12.9 / 8.1, of 256 14.4 / 10.2; 23 query rows and 4
  // heads a group over 51 of 11 pages 70 / 22; 32 query rows over 32 of 256 24 / 28).
  const bool few = M <= 256;
  const int shift = select_shift(G, a.Tq, M, few ? 2 : 4), per16 = (int)((256 + G - 1) / G);
  const dim3 grid((unsigned)((a.Tq + (1 << shift) - 1) >> shift), (unsigned)a.pool.H, (unsigned)a.N), nt(few ? 256 : 1024);
  const size_t bins = (size_t)4096 << shift, lds = bins + (M > PS_LDS ? 0 : ((size_t)M << shift) * 4);
  if (M > PS_LDS) {
    hipLaunchKernelGGL((paged_select_kernel<T, D, true, 16>), grid, nt, lds, stream, a, shift, per16, (uint32_t*)ws);
    return;
  }
  if (few) {
    hipLaunchKernelGGL((paged_select_kernel<T, D, false, 4>), grid, nt, lds, stream, a, shift, per16, (uint32_t*)nullptr);
    return;
  }
  static bool set[64];  // per device: more LDS than a kernel may have unasked
  int dev = 0;
  (void)hipGetDevice(&dev);
  if (lds > 49152 && (dev < 0 || dev >= 64 || !set[dev])) {
    (void)hipFuncSetAttribute((const void*)paged_select_kernel<T, D, false, 16>, hipFuncAttributeMaxDynamicSharedMemorySize,
                              PS_LDS * 4 + 4096);  // one row's codes and histograms; 20 KB more for the queries and bounds
    if (dev >= 0 && dev < 64) set[dev] = true;
  }
  hipLaunchKernelGGL((paged_select_kernel<T, D, false, 16>), grid, nt, lds, stream, a, shift, per16, (uint32_t*)nullptr);
}

// ---------------------------------------------------------------------------------------------
// attention
// ---------------------------------------------------------------------------------------------
// The segments of paged_core.h over the listed pages: an item is a query row with its K/V head (16 heads of the group a tile), a
// workgroup takes one, or one of `splits` runs of `chunk` rows of its list where there are too few items for the GPU: up to a
// quarter of the CUs (us of both launches, split / whole: 64 items of 4,096 rows of 64 dims 20 / 27, 128 of 1,536 rows of 128 dims
// 23 / 20.6, 256 of 2,048 rows in 8 bits 19 / 14.4). A workgroup has eight waves, or two where the rows are few or the workgroups
// fill the chip (us with 8 / 2 waves in bf16, in 8 bits: 1,024 items of 64 rows 10.6 / 6.8, 11.0 / 6.2, of 2,048 rows 50 / 47, 34 / 35;
// 256 items of 256 rows 7.2 / 6.1, 6.7 / 6.7, of 1,024 rows 14.7 / 13.8, 9.7 / 15.1).
template <typename T, typename C, int D, int NW>
__global__ __launch_bounds__(64 * NW, 2) void ps_kernel(PagedAttn a, PagedSplit z, int splits, int chunk) {
  const int b = xcd_remap(blockIdx.x, gridDim.x), part = b % splits;  // an XCD's workgroups share pages in its L2
  const int64_t item = b / splits;
  const int qt = (int)(item % z.qtiles), t = (int)(item / z.qtiles % a.Tq), nh = (int)(item / z.qtiles / a.Tq);
  const int64_t all = (int64_t)a.K << a.pool.shift, c0 = (int64_t)part * chunk;
  const int c1 = (int)(c0 + chunk < all ? c0 + chunk : all);
  pa_segment<T, C, D, 1, false, true, NW, false>(a, z, nh / a.pool.H, nh % a.pool.H, t, qt, (int)(c0 < all ? c0 : all), c1,
                                                splits > 1 ? b : -1, a.index + ((int64_t)nh * a.Tq + t) * a.K);
}

// A wave joins a query row's partials.
template <typename T, typename C, int D>
__global__ __launch_bounds__(256) void ps_merge_kernel(PagedAttn a, PagedSplit z, int splits) {
  constexpr int LPR = D / 4;
  const int64_t row = (int64_t)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (row >= (int64_t)a.N * a.Hq * a.Tq) return;
  const int lane = threadIdx.x & 63, G = a.Hq / a.pool.H, g = (int)(row % G);
  const int64_t item = row / G;
  const int t = (int)(item % a.Tq), nh = (int)(item / a.Tq), n = nh / a.pool.H, h = nh % a.pool.H;
  const int64_t first = (item * z.qtiles + g / 16) * splits;
  float m, inv;
  const f32x4 o = pa_join<PagedShift<T, C>, D>(z, splits, [&](int i) { return (first + i) * 16 + g % 16; }, &m, &inv);
  if (lane < LPR) store4((T*)a.out + n * a.o_sn + (h * G + g) * a.o_sh + t * a.o_st + lane * 4, o);
}

struct SparseCut {
  int64_t items, chunk;
  int splits;
  SparseCut(int64_t N, int64_t Hq, int64_t H, int64_t Tq, int64_t rows) {
    items = N * H * Tq * ((Hq / H + 15) / 16);
    int64_t s = items > 0 && items * 4 <= cu_count() ? cu_count() / items : 1;
    const int64_t most = (rows + 511) / 512;  // two turns a wave at least
    s = s < 1 ? 1 : s < most ? s : most;
    if (s < 1) s = 1;
    chunk = ((rows + s - 1) / s + 127) / 128 * 128;
    if (chunk < 128) chunk = 128;
    splits = rows > 0 ? (int)((rows + chunk - 1) / chunk) : 1;
  }
};

int64_t sparse_split(PagedSplit* z, char* ws, int64_t Hq, int64_t H, int64_t D, const SparseCut& cut) {
  *z = {};
  z->qtiles = (int)((Hq / H + 15) / 16);
  if (cut.splits == 1) return 0;
  const int64_t slots = cut.items * cut.splits * 16, part = align256(slots * D * 4);
  z->part = (float*)ws;
  z->ml = (float2*)(ws + part);
  return part + align256(slots * 8);
}

template <typename T, typename C, int D>
void launch_sparse(const PagedAttn& a, void* ws, hipStream_t stream) {
  const SparseCut cut(a.N, a.Hq, a.pool.H, a.Tq, (int64_t)a.K << a.pool.shift);
  PagedSplit z;
  sparse_split(&z, (char*)ws, a.Hq, a.pool.H, D, cut);
  const dim3 grid((unsigned)(cut.items * cut.splits));
  if (cut.chunk <= 256 || cut.items * cut.splits > 2 * cu_count())
    hipLaunchKernelGGL((ps_kernel<T, C, D, 2>), grid, dim3(128), 0, stream, a, z, cut.splits, (int)cut.chunk);
  else
    hipLaunchKernelGGL((ps_kernel<T, C, D, 8>), grid, dim3(512), 0, stream, a, z, cut.splits, (int)cut.chunk);
  if (cut.splits > 1)
    hipLaunchKernelGGL((ps_merge_kernel<T, C, D>), dim3((unsigned)(((int64_t)a.N * a.Hq * a.Tq + 3) / 4)), dim3(256), 0, stream, a,
                       z, cut.splits);
}

template <typename T, typename C>
void launch_sparse_d(const PagedAttn& a, void* ws, hipStream_t stream) {
  if (a.pool.D == 32) launch_sparse<T, C, 32>(a, ws, stream);
  else if (a.pool.D == 64) launch_sparse<T, C, 64>(a, ws, stream);
  else launch_sparse<T, C, 128>(a, ws, stream);
}

}  // namespace

int tabicl_launch_paged_bounds(const PagedBounds& a, int format, int64_t rows, hipStream_t stream) {
  int64_t pages = (rows >> a.pool.shift) + 2;
  if (pages > a.pool.max_pages) pages = a.pool.max_pages;
  if (pages == 0 || a.N == 0) return 0;
  const int64_t gx = (pages * a.pool.H + 3) / 4;
  int64_t some = PAGED_MAX_GRID / gx;  // sequences of a launch
  if (some > a.N) some = a.N;
  for (int64_t n = 0; n < a.N; n += some) {
    PagedBounds part = a;
    part.pool.table += n * a.pool.table_sn;
    part.pool.lengths += n;
    if (a.start) part.start += n;
    const dim3 grid((unsigned)gx, (unsigned)(a.N - n < some ? a.N - n : some));
    if (a.pool.D == 32) launch_bounds<32>(part, format, grid, stream);
    else if (a.pool.D == 64) launch_bounds<64>(part, format, grid, stream);
    else launch_bounds<128>(part, format, grid, stream);
  }
  return (int)hipGetLastError();
}

int64_t tabicl_launch_paged_select_ws_bytes(int64_t N, int64_t H, int64_t Tq, int64_t max_pages) {
  return max_pages > PS_LDS ? N * H * Tq * max_pages * 4 : 0;  // one query row a workgroup then
}

int tabicl_launch_paged_select(const PagedSelect& a, int dtype, void* ws, hipStream_t stream) {
  const int D = a.pool.D;
  if (dtype == 0) {
    if (D == 32) launch_select<bf16, 32>(a, ws, stream);
    else if (D == 64) launch_select<bf16, 64>(a, ws, stream);
    else launch_select<bf16, 128>(a, ws, stream);
  } else {
    if (D == 32) launch_select<float, 32>(a, ws, stream);
    else if (D == 64) launch_select<float, 64>(a, ws, stream);
    else launch_select<float, 128>(a, ws, stream);
  }
  return (int)hipGetLastError();
}

int64_t tabicl_launch_paged_sparse_ws_bytes(int64_t N, int64_t Hq, int64_t H, int64_t Tq, int64_t D, int64_t rows) {
  PagedSplit z;
  return sparse_split(&z, nullptr, Hq, H, D, SparseCut(N, Hq, H, Tq, rows));
}

int tabicl_launch_paged_sparse(const PagedAttn& a, int format, int dtype, void* ws, hipStream_t stream) {
  if (format == 0) launch_sparse_d<bf16, bf16>(a, ws, stream);
  else if (format == 1) launch_sparse_d<float, float>(a, ws, stream);
  else if (dtype == 0) format == 2 ? launch_sparse_d<bf16, E4M3>(a, ws, stream) : launch_sparse_d<bf16, I8>(a, ws, stream);
  else format == 2 ? launch_sparse_d<float, E4M3>(a, ws, stream) : launch_sparse_d<float, I8>(a, ws, stream);
  return (int)hipGetLastError();
}
