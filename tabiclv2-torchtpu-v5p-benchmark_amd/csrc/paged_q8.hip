// K/V pages of 8-bit codes (gfx950): value = code * scale, e4m3 or int8 codes, one scale for K and one for V of each page and
// head. Attention of few query rows over them, rows written into them, rows read back.
//
// A scale is a power of two: the smallest 2^k, k in [-60, 100], with max |x| <= Q 2^k over the new rows' finite values (Q = 448
// or 127). A page that already holds rows keeps the larger of its scale and theirs; where it grows, the held codes are rounded
// again to the new step. So a page filled row by row is rounded again at most once per doubling (int8: the errors add up to
// less than one step; e4m3: exact but for its subnormals), codes times scale are bf16 values, and no result depends on the
// order of a division.
#include "launch.h"
#include "paged_core.h"

namespace {

typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));

template <typename C>
struct Code;
template <>
struct Code<E4M3> {
  static constexpr int SHIFT = 8;               // 448 = 1.75 2^8
  static constexpr uint32_t MANT = 0x600000u;   // .75 of a mantissa
};
template <>
struct Code<I8> {
  static constexpr int SHIFT = 6;               // 127 = 1.984375 2^6
  static constexpr uint32_t MANT = 0x7e0000u;
};

// Four values to codes, rounded to the nearest (ties to even), saturating; NaN stays NaN in e4m3 and is 0 in int8.
template <typename C>
__device__ __forceinline__ uint32_t to_codes(const float* x);
template <>
__device__ __forceinline__ uint32_t to_codes<E4M3>(const float* x) {
  float y[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) y[i] = x[i] != x[i] ? x[i] : fminf(fmaxf(x[i], -448.f), 448.f);
  const int lo = __builtin_amdgcn_cvt_pk_fp8_f32(y[0], y[1], 0, false);
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(y[2], y[3], lo, true);
}
template <>
__device__ __forceinline__ uint32_t to_codes<I8>(const float* x) {
  uint32_t w = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float y = x[i] != x[i] ? 0.f : fminf(fmaxf(__builtin_rintf(x[i]), -127.f), 127.f);
    w |= (uint32_t)((int)y & 255) << (8 * i);
  }
  return w;
}

template <typename C>
__device__ __forceinline__ void from_codes(uint32_t w, float* x);
template <>
__device__ __forceinline__ void from_codes<E4M3>(uint32_t w, float* x) {
  const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8(w, false), hi = __builtin_amdgcn_cvt_pk_f32_fp8(w, true);
  x[0] = lo[0], x[1] = lo[1], x[2] = hi[0], x[3] = hi[1];
}
template <>
__device__ __forceinline__ void from_codes<I8>(uint32_t w, float* x) {
#pragma unroll
  for (int i = 0; i < 4; ++i) x[i] = (float)(int8_t)(w >> (8 * i));
}

// Eight consecutive values as they lie in memory; in fp32; the largest magnitude among them as an integer (16 bits of one, twice,
// in bf16).
template <typename T>
struct Raw8 {
  uint4 u[sizeof(T) / 2];
  __device__ __forceinline__ void load(const T* p) {
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i) u[i] = ldg16_once(p + i * (16 / sizeof(T)));
  }
  __device__ __forceinline__ void values(float* x) const {
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i) {
      const uint32_t w[4] = {u[i].x, u[i].y, u[i].z, u[i].w};
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if constexpr (sizeof(T) == 2) x[2 * j] = __uint_as_float(w[j] << 16), x[2 * j + 1] = __uint_as_float(w[j] & 0xffff0000u);
        else x[4 * i + j] = __uint_as_float(w[j]);
    }
  }
  __device__ __forceinline__ uint32_t most(uint32_t m) const {
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i) {
      const uint32_t w[4] = {u[i].x, u[i].y, u[i].z, u[i].w};
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if constexpr (sizeof(T) == 2)
          m = __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(u16x2, m), __builtin_bit_cast(u16x2, w[j] & 0x7fff7fffu)));
        else m = (w[j] & 0x7fffffffu) > m ? w[j] & 0x7fffffffu : m;
    }
    return m;
  }
};

// Four values, none beyond the largest code times the step, to codes: to_codes without its limits. int8: added to 1.5 2^23, a
// value is rounded to a whole number in the sum's lowest bits.
template <typename C>
__device__ __forceinline__ uint32_t to_codes_within(const float* x, float inv);
template <>
__device__ __forceinline__ uint32_t to_codes_within<E4M3>(const float* x, float inv) {
  const int lo = __builtin_amdgcn_cvt_pk_fp8_f32(x[0] * inv, x[1] * inv, 0, false);
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(x[2] * inv, x[3] * inv, lo, true);
}
template <>
__device__ __forceinline__ uint32_t to_codes_within<I8>(const float* x, float inv) {
  uint32_t y[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) y[i] = __float_as_uint(__builtin_fmaf(x[i], inv, 12582912.f));
  return __builtin_amdgcn_perm(__builtin_amdgcn_perm(y[3], y[2], 0x0c0c0400u), __builtin_amdgcn_perm(y[1], y[0], 0x0c0c0400u), 0x05040100u);
}

// ---------------------------------------------------------------------------------------------
// append
// ---------------------------------------------------------------------------------------------
// LANES threads take the new rows of one page and head, of K or of V: the largest |x|, the scale, the codes. Up to LANES * 8
// chunks of eight values are read once and kept; a larger page's are read again for their codes. A wave takes a page of up to 64 *
// 8 chunks, a workgroup of 256 or 512 threads a larger one (10 x 16,907 rows of 128 dims in fp32 to pages of 256 rows, which 512
// threads keep and 256 do not: 283 -> 214 us with their way back). Where a value is not finite, or beyond the largest scale, they are gone through value by value.
// Bound by the bytes of the rows and codes: 8 x 45,000 rows in bf16 to int8 268 us -> 238 with magnitudes compared in pairs and
// codes without limits (15 -> 4 instructions a value), 221 with loads that leave the caches alone (stores that do: 217, and what
// reads the codes next takes 10 us more).
constexpr int PQ_KEEP = 8;

template <typename T, typename C, int LANES>
__global__ __launch_bounds__(LANES == 64 ? 256 : LANES) void paged_append8_kernel(PagedAppend8 a) {
  const PagedPool& c = a.rows.pool;
  const int n = blockIdx.y, v = blockIdx.z, D = c.D, R = 1 << c.shift;
  const int item = LANES == 64 ? blockIdx.x * 4 + threadIdx.x / 64 : blockIdx.x, lane = threadIdx.x % LANES;
  const int h = item % c.H, j = item / c.H;
  const int64_t cap = (int64_t)c.max_pages << c.shift;
  const int start = pool_length(c, n);
  int64_t add = a.rows.count ? a.rows.count[n] : a.rows.T;
  const int64_t from = a.starts ? a.starts[n] : 0, most_rows = from < 0 ? 0 : a.rows.T - from;  // packed: T rows in all
  add = add < 0 ? 0 : add < most_rows ? add : most_rows;
  const int64_t end = start + add < cap ? start + add : cap, p = (start >> c.shift) + (int64_t)j;
  const int64_t r0 = p << c.shift > start ? p << c.shift : start, r1 = (p + 1) << c.shift < end ? (p + 1) << c.shift : end;
  if (r0 >= r1) return;
  const int page = c.table[n * c.table_sn + p];
  if (page < 0 || page >= c.pages) return;
  const int held = (int)(r0 - (p << c.shift)), cpr = __builtin_ctz(D / 8);  // rows in place; chunks of a row: 1 << cpr
  const int chunks = (int)(r1 - r0) << cpr;
  const int64_t st = v ? a.rows.v_st : a.rows.k_st;
  const T* src = (const T*)(v ? a.rows.v : a.rows.k) + (a.starts ? from * st : n * (v ? a.rows.v_sn : a.rows.k_sn)) +
                 h * (v ? a.rows.v_sh : a.rows.k_sh) + (r0 - start) * st;
  char* dst = (char*)(v ? c.v : c.k) + page * c.page_sp + (int64_t)h * R * D;
  float* scale = a.scales + ((int64_t)page * c.H + h) * 2 + v;
  const float old = held ? *scale : 0.f;
  auto chunk = [&](int at) { return src + (at >> cpr) * st + (at & ((1 << cpr) - 1)) * 8; };
  auto all = [&](uint32_t m) {  // the largest over the LANES threads
#pragma unroll
    for (int x = 1; x < 64; x <<= 1) {
      const uint32_t o = __shfl_xor(m, x, 64);
      m = o > m ? o : m;
    }
    if constexpr (LANES > 64) {
      __shared__ uint32_t sh[LANES / 64];
      __syncthreads();
      if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = m;
      __syncthreads();
#pragma unroll
      for (int i = 0; i < LANES / 64; ++i) m = sh[i] > m ? sh[i] : m;
    }
    return m;
  };

  Raw8<T> x[PQ_KEEP];
  uint32_t most = 0;
  const bool once = chunks <= LANES * PQ_KEEP;
  for (int base = 0; base < chunks; base += LANES * PQ_KEEP) {
#pragma unroll
    for (int i = 0; i < PQ_KEEP; ++i) {
      const int at = base + i * LANES + lane;
      if (at < chunks) x[i].load(chunk(at));
    }
#pragma unroll
    for (int i = 0; i < PQ_KEEP; ++i)
      if (base + i * LANES + lane < chunks) most = x[i].most(most);
  }
  if constexpr (sizeof(T) == 2) most = (most >> 16 > (most & 0xffffu) ? most >> 16 : most & 0xffffu) << 16;
  most = all(most);
  bool within = most < 0x7f800000u;
  if (!within) {  // uniform over the LANES threads: the largest finite one
    most = 0;
    for (int at = lane; at < chunks; at += LANES) {
      Raw8<T> y;
      float f[8];
      y.load(chunk(at));
      y.values(f);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const uint32_t u = __float_as_uint(f[e]) & 0x7fffffffu;
        most = u < 0x7f800000u && u > most ? u : most;
      }
    }
    most = all(most);
  }
  int k = (int)(most >> 23) - 127 - Code<C>::SHIFT + ((most & 0x7fffffu) > Code<C>::MANT);
  within = within && k <= 100;
  k = k < -60 ? -60 : k < 100 ? k : 100;
  float s = __uint_as_float((uint32_t)(k + 127) << 23);
  if (old > s) s = old;  // the held rows' (a NaN there gives way)
  const float inv = 1.f / s;
  for (int base = 0; base < chunks; base += LANES * PQ_KEEP)
#pragma unroll
    for (int i = 0; i < PQ_KEEP; ++i) {
      const int at = base + i * LANES + lane;
      if (at >= chunks) continue;
      if (!once) x[i].load(chunk(at));
      float y[8];
      uint2 w;
      x[i].values(y);
      if (within) {
        w = uint2{to_codes_within<C>(y, inv), to_codes_within<C>(y + 4, inv)};
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) y[e] *= inv;
        w = uint2{to_codes<C>(y), to_codes<C>(y + 4)};
      }
      *(uint2*)(dst + ((int64_t)held << cpr) * 8 + (int64_t)at * 8) = w;
    }
  if (held && s != old) {
    const float ratio = old / s;
    for (int at = lane; at < held << cpr; at += LANES) {
      const uint2 w = *(const uint2*)(dst + (int64_t)at * 8);
      float y[8];
      from_codes<C>(w.x, y);
      from_codes<C>(w.y, y + 4);
#pragma unroll
      for (int e = 0; e < 8; ++e) y[e] *= ratio;
      *(uint2*)(dst + (int64_t)at * 8) = uint2{to_codes<C>(y), to_codes<C>(y + 4)};
    }
  }
  // every thread has its `old` by now: within a wave by program order, across waves by the barriers above
  if (lane == 0) *scale = s;
}

// ---------------------------------------------------------------------------------------------
// gather: k, v [N, H, T, D] <- the values of the first min(lengths[n], T) rows (0 where there is no page)
// ---------------------------------------------------------------------------------------------
__device__ __forceinline__ void store16(bf16* p, const float* x) { store_row<bf16, 16>(p, x); }
__device__ __forceinline__ void store16(float* p, const float* x) { store_row<float, 16>(p, x); }

template <typename T, typename C>
__global__ __launch_bounds__(256) void paged_gather8_kernel(PagedGather a, const float* scales) {
  const PagedPool& c = a.pool;
  const int n = blockIdx.y, cpr = __builtin_ctz(c.D / 16), len = pool_length(c, n), rows = len < a.T ? len : a.T;
  const int64_t total = (int64_t)rows * c.H << cpr;
  const bool narrow = total >> cpr <= 0x7fffffff;  // a 64-bit division takes as long as a load
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
    const int64_t j = i >> cpr;
    const int h = narrow ? (int)((uint32_t)j / (uint32_t)rows) : (int)(j / rows), row = (int)(j - (int64_t)h * rows);
    const int ch = (int)i & ((1 << cpr) - 1);
    const int page = c.table[n * c.table_sn + (row >> c.shift)];
    const int64_t to = (((int64_t)n * c.H + h) * a.T + row) * c.D + ch * 16;
    uint4 k = {0, 0, 0, 0}, v = {0, 0, 0, 0};
    float2 s = make_float2(0.f, 0.f);
    if (page >= 0 && page < c.pages) {
      const int64_t from = page * c.page_sp + (((int64_t)h << c.shift) + (row & ((1 << c.shift) - 1))) * c.D + ch * 16;
      k = ldg16((const char*)c.k + from);
      v = ldg16((const char*)c.v + from);
      s = *(const float2*)(scales + ((int64_t)page * c.H + h) * 2);
    }
    const uint32_t kw[4] = {k.x, k.y, k.z, k.w}, vw[4] = {v.x, v.y, v.z, v.w};
    float x[16];
#pragma unroll
    for (int w = 0; w < 4; ++w) from_codes<C>(kw[w], x + 4 * w);
#pragma unroll
    for (int e = 0; e < 16; ++e) x[e] *= s.x;
    store16((T*)a.k + to, x);
#pragma unroll
    for (int w = 0; w < 4; ++w) from_codes<C>(vw[w], x + 4 * w);
#pragma unroll
    for (int e = 0; e < 16; ++e) x[e] *= s.y;
    store16((T*)a.v + to, x);
  }
}

// ---------------------------------------------------------------------------------------------
// attention: the kernels of paged_core.h; the codes become bf16 operands in the registers (exactly), K's scale goes into the
// scores and V's into the probabilities. fp32 queries and probabilities enter as three bf16 terms: nothing of them is lost.
// ---------------------------------------------------------------------------------------------
// The widest tile of query rows, in sixteens.
template <typename T>
constexpr int pa8_most(int D) { return sizeof(T) == 4 || D == 128 ? 2 : 4; }

// ONCE: the query rows are one tile.
template <typename T, typename C, int D, int QT, bool ONCE>
int64_t run_pa8(const PagedAttn* a, void* ws, int64_t N, int64_t Hq, int64_t H, int64_t Tq, int64_t rows, hipStream_t stream) {
  const int64_t qrows = Hq / H * Tq;
  PagedSplit z = {};
  z.qtiles = (int)((qrows + 16 * QT - 1) / (16 * QT));
  constexpr int waves = pa_waves_of<T, C>(D, QT);
  constexpr bool splits = ONCE || D == 128 || QT == pa8_most<T>(D);  // several narrow tiles: over short caches alone
  z.groups = !splits || (rows <= PA_WHOLE && waves == 2) ? 0 : waves * cu_count();
  z.least = 2;
  z.few = D > 32 && waves == 2 ? 12 * z.groups : 0;
  int64_t at = 0;
  auto take = [&](int64_t bytes) {
    char* p = (char*)ws + at;
    at += align256(bytes);
    return p;
  };
  z.part = (float*)take((int64_t)z.groups * 2 * 16 * QT * D * 4);
  z.ml = (float2*)take((int64_t)z.groups * 2 * 16 * QT * 8);
  z.ends = (int2*)take(z.groups ? N * H * z.qtiles * 8 : 0);
  if (!a) return at;
  if (z.groups == 0) {
    // Two waves for each item up to 256 rows and four beyond, so that many items share a CU; eight for more than 512 rows where
    // every item has a CU (us with 2 / 4 / 8 waves: 2,048 items of one query row of 64 dims and 64 rows 7.7 / - / 18.1, of 512 rows
    // 24 / 25 / 32; of 60 query rows 20 / - / 74 and 48 / 59 / 102; 64 items of one query row and 256 rows 6.2 / - / 6.1, of 1,024 13.2 /
    // 9.0 / 8.2; 16 items in fp32 of 800 rows - / 9.6 / 8.1).
    const int64_t items = N * H * z.qtiles;
    const dim3 grid((unsigned)items);
    if constexpr (waves == 2) {
      if (rows <= 256) hipLaunchKernelGGL((pa_whole_kernel<T, C, D, QT, false, 2, ONCE>), grid, dim3(128), 0, stream, *a, z);
      else if (rows <= 512 || items > cu_count())
        hipLaunchKernelGGL((pa_whole_kernel<T, C, D, QT, false, 4, ONCE>), grid, dim3(256), 0, stream, *a, z);
      else hipLaunchKernelGGL((pa_whole_kernel<T, C, D, QT, false, 8, ONCE>), grid, dim3(512), 0, stream, *a, z);
    }
  } else if constexpr (splits) {
    hipLaunchKernelGGL((pa_kernel<T, C, D, QT, false, ONCE>), dim3((unsigned)z.groups), dim3(256), 0, stream, *a, z);
    hipLaunchKernelGGL((pa_merge_kernel<T, C, D, QT>), dim3((unsigned)((N * Hq * Tq + 3) / 4)), dim3(256), 0, stream, *a, z);
  }
  return at;
}

// Tiles of 16 QT query rows; a single one in the form that loads past the caches.
template <typename T, typename C, int D, int QT>
int64_t run_pa8_tiles(const PagedAttn* a, void* ws, int64_t N, int64_t Hq, int64_t H, int64_t Tq, int64_t rows, hipStream_t stream) {
  if constexpr (D <= 64 && QT <= 2)
    if (Hq / H * Tq <= 16 * QT) return run_pa8<T, C, D, QT, true>(a, ws, N, Hq, H, Tq, rows, stream);
  return run_pa8<T, C, D, QT, false>(a, ws, N, Hq, H, Tq, rows, stream);
}

template <typename T, typename C, int D>
int64_t run_pa8_rows(const PagedAttn* a, void* ws, int64_t N, int64_t Hq, int64_t H, int64_t Tq, int64_t rows,
                     hipStream_t stream) {
  const int64_t qrows = Hq / H * Tq;
  // Tiles of 16 query rows or, up to what the registers hold, 32 or 64: every tile converts K and V again (us in tiles of 16 / 32 /
  // 64: 64 query rows over 48 x 6,239 rows and 2 heads of 128 dims 97 / 66 / -, in fp32 104 / 83 / -, in fp32 of 64 dims 63 / 50 /
  // 71). Up to PA_WHOLE rows only as far as the items fill the chip (64 dims, bf16: 64 rows over 8 x 300 6.9 / 8.5 / 11.9, 200 over
  // 57 x 1,000 and 2 heads 35 / 30 / 27, 64 over 256 x 300 77 / 54 / 50).
  constexpr int most = pa8_most<T>(D);
  auto wider = [&](int qt) {  // than 16 qt rows
    return qrows > 16 * qt && (rows > PA_WHOLE || N * H * ((qrows + 16 * qt - 1) / (16 * qt)) > 2 * cu_count());
  };
  if constexpr (most == 4)
    if (wider(1) && wider(2)) return run_pa8_tiles<T, C, D, 4>(a, ws, N, Hq, H, Tq, rows, stream);
  if ((rows > PA_WHOLE || pa_waves_of<T, C>(D, 2) == 2) && wider(1)) return run_pa8_tiles<T, C, D, 2>(a, ws, N, Hq, H, Tq, rows, stream);
  return run_pa8_tiles<T, C, D, 1>(a, ws, N, Hq, H, Tq, rows, stream);
}

// The query rows in slices of what a launch counts, one after the other over one workspace.
template <typename T, typename C, int D>
int64_t run_pa8_d(const PagedAttn* a, void* ws, int64_t N, int64_t Hq, int64_t H, int64_t Tq, int64_t rows, hipStream_t stream) {
  const int64_t G = Hq / H, units = N * H * (rows / PA_UNIT + 1 + PA_EXTRA8), counted = PAGED_MAX_UNITS / units * 16 / G;
  int64_t slice = PAGED_MAX_QUERIES / (N * Hq);
  slice = counted < slice ? counted : slice;
  slice = slice < 1 ? 1 : slice;
  int64_t bytes = 0;
  for (int64_t t = 0; t < Tq; t += slice) {
    const int64_t left = Tq - t < slice ? Tq - t : slice;
    if (!a && t > 0 && left == slice) continue;  // the last one may be sized otherwise
    PagedAttn part = {};
    if (a) {
      part = *a;
      part.q = (const char*)a->q + t * a->q_st * sizeof(T);
      part.out = (char*)a->out + t * a->o_st * sizeof(T);
      part.Tq = (int)left;
    }
    const int64_t b = run_pa8_rows<T, C, D>(a ? &part : nullptr, ws, N, Hq, H, left, rows, stream);
    bytes = b > bytes ? b : bytes;
  }
  return bytes;
}

template <typename T, typename C>
int64_t run_pa8_c(const PagedAttn* a, void* ws, int64_t N, int64_t Hq, int64_t H, int64_t Tq, int64_t D, int64_t rows,
                  hipStream_t stream) {
  return D == 32   ? run_pa8_d<T, C, 32>(a, ws, N, Hq, H, Tq, rows, stream)
         : D == 64 ? run_pa8_d<T, C, 64>(a, ws, N, Hq, H, Tq, rows, stream)
                   : run_pa8_d<T, C, 128>(a, ws, N, Hq, H, Tq, rows, stream);
}

int64_t run_pa8_any(const PagedAttn* a, void* ws, int64_t N, int64_t Hq, int64_t H, int64_t Tq, int64_t D, int64_t rows, int dtype,
                    int code, hipStream_t stream) {
  if (dtype == 0)
    return code == 0 ? run_pa8_c<bf16, E4M3>(a, ws, N, Hq, H, Tq, D, rows, stream)
                     : run_pa8_c<bf16, I8>(a, ws, N, Hq, H, Tq, D, rows, stream);
  return code == 0 ? run_pa8_c<float, E4M3>(a, ws, N, Hq, H, Tq, D, rows, stream)
                   : run_pa8_c<float, I8>(a, ws, N, Hq, H, Tq, D, rows, stream);
}

template <typename T, typename C>
void launch_append8(const PagedAppend8& a, hipStream_t stream) {
  const PagedPool& c = a.rows.pool;
  int64_t pages = ((int64_t)a.rows.T >> c.shift) + 2;  // that T rows can touch
  if (pages > c.max_pages) pages = c.max_pages;
  const int64_t items = pages * c.H;
  // chunks of a page's new rows
  const int64_t chunks = (a.rows.T < (1 << c.shift) ? (int64_t)a.rows.T : 1ll << c.shift) * (c.D / 8);
  const bool wave = chunks <= 64 * PQ_KEEP;
  const int64_t gx = wave ? (items + 3) / 4 : items;
  int64_t some = PAGED_MAX_GRID / (2 * gx);  // sequences of a launch
  if (some > a.rows.N) some = a.rows.N;
  for (int64_t n = 0; n < a.rows.N; n += some) {
    PagedAppend8 part = a;
    part.rows.pool.table += n * c.table_sn;
    part.rows.pool.lengths += n;
    if (a.rows.count) part.rows.count += n;
    if (a.starts) {
      part.starts += n;
    } else {
      part.rows.k = (const T*)a.rows.k + n * a.rows.k_sn;
      part.rows.v = (const T*)a.rows.v + n * a.rows.v_sn;
    }
    const dim3 grid((unsigned)gx, (unsigned)(a.rows.N - n < some ? a.rows.N - n : some), 2);
    if (wave) hipLaunchKernelGGL((paged_append8_kernel<T, C, 64>), grid, dim3(256), 0, stream, part);
    else if (chunks <= 256 * PQ_KEEP) hipLaunchKernelGGL((paged_append8_kernel<T, C, 256>), grid, dim3(256), 0, stream, part);
    else hipLaunchKernelGGL((paged_append8_kernel<T, C, 512>), grid, dim3(512), 0, stream, part);
  }
}

}  // namespace

int64_t tabicl_launch_paged_attn_q8_ws_bytes(int64_t N, int64_t Hq, int64_t H, int64_t Tq, int64_t D, int64_t rows, int dtype) {
  return run_pa8_any(nullptr, nullptr, N, Hq, H, Tq, D, rows, dtype, 0, nullptr);
}

int tabicl_launch_paged_attn_q8(const PagedAttn& a, int dtype, int code, void* ws, hipStream_t stream) {
  run_pa8_any(&a, ws, a.N, a.Hq, a.pool.H, a.Tq, a.pool.D, (int64_t)a.pool.max_pages << a.pool.shift, dtype, code, stream);
  return (int)hipGetLastError();
}

int tabicl_launch_paged_append_q8(const PagedAppend8& a, int dtype, int code, hipStream_t stream) {
  if (a.rows.pool.max_pages == 0) return 0;
  if (dtype == 0) code == 0 ? launch_append8<bf16, E4M3>(a, stream) : launch_append8<bf16, I8>(a, stream);
  else code == 0 ? launch_append8<float, E4M3>(a, stream) : launch_append8<float, I8>(a, stream);
  return (int)hipGetLastError();
}

int tabicl_launch_paged_gather_q8(const PagedGather& a, const float* scales, int dtype, int code, hipStream_t stream) {
  int64_t gx = ((int64_t)a.T * a.pool.H * (a.pool.D / 16) + 255) / 256;
  if (gx > PAGED_MAX_GRID / a.N) gx = PAGED_MAX_GRID / a.N;
  if (gx > 4096) gx = 4096;
  const dim3 grid((unsigned)gx, (unsigned)a.N);
  if (dtype == 0) {
    if (code == 0) hipLaunchKernelGGL((paged_gather8_kernel<bf16, E4M3>), grid, dim3(256), 0, stream, a, scales);
    else hipLaunchKernelGGL((paged_gather8_kernel<bf16, I8>), grid, dim3(256), 0, stream, a, scales);
  } else {
    if (code == 0) hipLaunchKernelGGL((paged_gather8_kernel<float, E4M3>), grid, dim3(256), 0, stream, a, scales);
    else hipLaunchKernelGGL((paged_gather8_kernel<float, I8>), grid, dim3(256), 0, stream, a, scales);
  }
  return (int)hipGetLastError();
}
