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

// One wave per page and head. Bound by the bytes of K.
template <typename C>
__global__ __launch_bounds__(256) void paged_bounds_kernel(PagedBounds a) {
  constexpr int VPC = 16 / sizeof(C), ES = sizeof(C);  // values of a lane's 16 bytes
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
  const int lpr = c.D * ES / 16, rpp = 64 / lpr;  // lanes of a row, rows of a pass
  const char* k = (const char*)c.k + (page * c.page_sp + (int64_t)h * R * c.D) * ES + lane % lpr * 16;
  float lo[VPC], hi[VPC];
#pragma unroll
  for (int e = 0; e < VPC; ++e) lo[e] = -TA_NEG_INF, hi[e] = TA_NEG_INF;
  auto add = [&](uint4 u) {
    float x[VPC];
    values16<C>(u, x);
#pragma unroll
    for (int e = 0; e < VPC; ++e) lo[e] = fminf(lo[e], x[e]), hi[e] = fmaxf(hi[e], x[e]);  // a NaN changes neither
  };
  int r = lane / lpr;
  for (; r + 7 * rpp < live; r += 8 * rpp) {
    uint4 u[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) u[i] = ldg16(k + (int64_t)(r + i * rpp) * c.D * ES);
#pragma unroll
    for (int i = 0; i < 8; ++i) add(u[i]);
  }
  for (; r < live; r += rpp) add(ldg16(k + (int64_t)r * c.D * ES));
  for (int x = lpr; x < 64; x <<= 1)
#pragma unroll
    for (int e = 0; e < VPC; ++e) lo[e] = fminf(lo[e], __shfl_xor(lo[e], x, 64)), hi[e] = fmaxf(hi[e], __shfl_xor(hi[e], x, 64));
  if constexpr (ES == 1) {
    const float s = a.scales[((int64_t)page * c.H + h) * 2];
#pragma unroll
    for (int e = 0; e < VPC; ++e) lo[e] *= s, hi[e] *= s;
  }
  uint32_t most = 0;
#pragma unroll
  for (int e = 0; e < VPC; ++e) {
    if (hi[e] < lo[e]) lo[e] = hi[e] = 0.f;  // a dim of NaN alone
    most = umax(most, umax(finite_bits(lo[e]), finite_bits(hi[e])));
  }
  for (int x = 1; x < lpr; x <<= 1) most = umax(most, (uint32_t)__shfl_xor(most, x, 64));
  const int e2 = step_exponent(most);
  const float inv = pow2(-e2);
  if (lane >= lpr) return;
  uint32_t wh[(VPC + 3) / 4], wl[(VPC + 3) / 4];
#pragma unroll
  for (int e = 0; e < VPC; ++e) {
    // infinite bounds, and finite ones beyond the largest scale, at the end of the range
    const int x = (int)fminf(fmaxf(ceilf(hi[e] * inv), -127.f), 127.f), y = (int)fminf(fmaxf(floorf(lo[e] * inv), -127.f), 127.f);
    if (e % 4 == 0) wh[e / 4] = wl[e / 4] = 0;
    wh[e / 4] |= (uint32_t)(x & 255) << (8 * (e % 4));
    wl[e / 4] |= (uint32_t)(y & 255) << (8 * (e % 4));
  }
  int8_t* out = a.bounds + ((int64_t)page * c.H + h) * 2 * c.D + lane * VPC;
#pragma unroll
  for (int w = 0; w < VPC / 4; ++w) {
    *(uint32_t*)(out + 4 * w) = wh[w];
    *(uint32_t*)(out + c.D + 4 * w) = wl[w];
  }
  if (lane == 0) a.bound_scales[(int64_t)page * c.H + h] = pow2(e2);
}

// ---------------------------------------------------------------------------------------------
// selection
// ---------------------------------------------------------------------------------------------
// A workgroup of 16 waves takes up to TT query rows of one sequence and K/V head: the bounds of 16 pages for 16 (query row,
// head of the group) pairs at a time on the 8-bit matrix unit, kept as ordered codes [TT][pages] in LDS (0: no such page); then
// the K-th largest code of each query row by four 8-bit digits of a histogram, 16 / TT waves a row; then the pages above it,
// and the first ones equal to it, in order.
constexpr int PS_NW = 16, PS_LDS = 32768;  // codes kept in LDS

__device__ __forceinline__ uint32_t bound_code(float x) {  // larger bound, larger code; none is 0
  const uint32_t u = __float_as_uint(x + 0.f);
  const uint32_t v = u & 0x80000000u ? ~u : u | 0x80000000u;
  return v ? v : 1;
}
__device__ __forceinline__ int lanes_below(uint64_t mask) {
  return __builtin_amdgcn_mbcnt_hi((uint32_t)(mask >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)mask, 0));
}

template <typename T, int D, bool GLOBAL>
__global__ __launch_bounds__(PS_NW * 64) void paged_select_kernel(PagedSelect a, int TT, int qtiles, uint32_t* store) {
  extern __shared__ uint32_t lds_codes[];
  constexpr int KB = 2 * D / 64;  // products of 64 bounds
  __shared__ __attribute__((aligned(16))) int8_t sh_q[16][2 * D];
  __shared__ float sh_inv[16];
  __shared__ int hist[16][256], pick[16][2], part[PS_NW][2];
  const PagedPool& c = a.pool;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lr = lane & 15, lg = lane >> 4;
  const int qt = blockIdx.x % qtiles, nh = blockIdx.x / qtiles, n = nh / c.H, h = nh % c.H, t0 = qt * TT;
  const int G = a.Hq / c.H, R = 1 << c.shift, len = __builtin_amdgcn_readfirstlane(pool_length(c, n));
  const int P = (len + R - 1) >> c.shift, stride = c.max_pages;
  uint32_t* codes = GLOBAL ? store + (int64_t)blockIdx.x * TT * stride : lds_codes;
  const char* q = (const char*)a.q + (n * a.q_sn + (int64_t)h * G * a.q_sh) * sizeof(T);
  auto value = [&](int g, int t, int d) {
    return (float)*(const T*)(q + (g * a.q_sh + t * a.q_st + d) * (int64_t)sizeof(T));
  };

  // the step of each query row: wave t looks at the group's heads
  if (wave < TT) {
    uint32_t most = 0;
    if (t0 + wave < a.Tq)
      for (int i = lane; i < G * D; i += 64) most = umax(most, finite_bits(value(i / D, t0 + wave, i % D)));
#pragma unroll
    for (int x = 1; x < 64; x <<= 1) most = umax(most, (uint32_t)__shfl_xor(most, x, 64));
    if (lane == 0) sh_inv[wave] = pow2(-step_exponent(most));
  }
  for (int i = threadIdx.x; i < TT * P; i += PS_NW * 64) codes[i / P * stride + i % P] = 0;
  __syncthreads();

  for (int g0 = 0; g0 < G; g0 += 16) {  // TT > 1: all heads at once
    {
      const int t = TT > 1 ? wave / G : 0, g = TT > 1 ? wave % G : g0 + wave;
      const bool in = t < TT && g < G && t0 + t < a.Tq;
      for (int d = lane; d < D; d += 64) {
        int u = 0;
        if (in) {
          const float x = value(g, t0 + t, d);
          u = x != x ? 0 : (int)fminf(fmaxf(__builtin_rintf(x * sh_inv[t]), -127.f), 127.f);
        }
        sh_q[wave][d] = (int8_t)(u > 0 ? u : 0);
        sh_q[wave][D + d] = (int8_t)(u < 0 ? u : 0);
      }
    }
    __syncthreads();
    const int t = TT > 1 ? lr / G : 0, g = TT > 1 ? lr % G : g0 + lr;
    const bool mine = t < TT && g < G && t0 + t < a.Tq;
    i32x4 qb[KB];
#pragma unroll
    for (int i = 0; i < KB; ++i) qb[i] = *(const i32x4*)(&sh_q[lr][i * 64 + lg * 16]);
    for (int p0 = wave * 16; p0 < P; p0 += PS_NW * 16) {
      int page = p0 + lr < P ? c.table[n * c.table_sn + p0 + lr] : -1;
      const bool have = page >= 0 && page < c.pages;
      const int64_t at = ((int64_t)(have ? page : 0) * c.H + h);
      i32x4 sum = {0, 0, 0, 0};
      float scale = 0.f;
      if (have) scale = a.bound_scales[at];
#pragma unroll
      for (int i = 0; i < KB; ++i) {
        i32x4 b = {0, 0, 0, 0};
        if (have) b = *(const i32x4*)(a.bounds + at * 2 * D + i * 64 + lg * 16);
        sum = __builtin_amdgcn_mfma_i32_16x16x64_i8(b, qb[i], sum, 0, 0, 0);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float s = __shfl(scale, lg * 4 + i, 64);
        const int there = __shfl((int)have, lg * 4 + i, 64);
        if (there && mine) {
          const uint32_t code = bound_code((float)sum[i] * s);
          uint32_t* to = codes + t * stride + p0 + lg * 4 + i;
          if (G == 1) *to = code;
          else atomicMax(to, code);
        }
      }
    }
    __syncthreads();
  }

  // the rows in groups of waves
  const int wpr = PS_NW / TT, t = wave / wpr, member = wave % wpr * 64 + lane, members = wpr * 64;
  const uint32_t* mycodes = codes + t * stride;
  int want = a.K < P ? a.K : 0;  // of the pages of the threshold's code, in the end; every page there is: 0
  uint32_t threshold = 0;
  if (a.K < P) {
    for (int shift = 24; shift >= 0; shift -= 8) {
      for (int i = member; i < 256; i += members) hist[t][i] = 0;
      __syncthreads();
      for (int i = member; i < P; i += members) {
        const uint32_t x = mycodes[i];
        if (shift == 24 || (x ^ threshold) >> (shift + 8) == 0) atomicAdd(&hist[t][x >> shift & 255], 1);
      }
      __syncthreads();
      if (wave % wpr == 0) {  // four bins a lane, counted from the top
        int b[4], sum = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) sum += b[i] = hist[t][255 - 4 * lane - i];
        int before = wave_sum_scan(sum) - sum;
        if (before < want && before + sum >= want) {  // one lane
          int i = 0;
          while (before + b[i] < want) before += b[i++];
          pick[t][0] = 255 - 4 * lane - i;
          pick[t][1] = want - before;
        }
      }
      __syncthreads();
      threshold |= (uint32_t)pick[t][0] << shift;
      want = pick[t][1];
    }
  }
  if (threshold == 0) want = 0;  // fewer pages than K: those that are there
  // a run of pages per wave: what is taken before it, then the places
  const int run = ((P + members - 1) / members) * 64, p0 = wave % wpr * run, p1 = p0 + run < P ? p0 + run : P;
  int more = 0, even = 0;
  for (int p = p0 + lane; p - lane < p1; p += 64) {
    const uint32_t x = p < p1 ? mycodes[p] : 0;
    more += __popcll(__ballot(x > threshold));
    even += __popcll(__ballot(x == threshold && x != 0));
  }
  if (lane == 0) part[wave][0] = more, part[wave][1] = even;
  __syncthreads();
  if (t0 + t >= a.Tq) return;
  int more0 = 0, even0 = 0, all = 0, evens = 0;
  for (int w = 0; w < wpr; ++w) {
    const int m = part[t * wpr + w][0], e = part[t * wpr + w][1];
    if (w < wave % wpr) more0 += m, even0 += e;
    all += m;
    evens += e;
  }
  all += evens < want ? evens : want;
  int32_t* out = a.index + ((int64_t)nh * a.Tq + t0 + t) * a.K;
  for (int p = p0 + lane; p - lane < p1; p += 64) {
    const uint32_t x = p < p1 ? mycodes[p] : 0;
    const uint64_t above = __ballot(x > threshold), equal = __ballot(x == threshold && x != 0);
    const int rank = even0 + lanes_below(equal);
    if (x > threshold || (x == threshold && x != 0 && rank < want)) out[more0 + lanes_below(above) + (rank < want ? rank : want)] = p;
    more0 += __popcll(above);
    even0 += __popcll(equal);
  }
  for (int i = all + member; i < a.K; i += members) out[i] = -1;
}

// Query rows of a workgroup: a power of two with up to 16 (query row, head) pairs whose codes fit in LDS.
int select_rows(int64_t G, int64_t Tq, int64_t max_pages) {
  int tt = 1;
  while (tt < 16 && tt < Tq && 2 * tt * G <= 16 && 2 * tt * max_pages <= PS_LDS) tt *= 2;
  return tt;
}

template <typename T, int D>
void launch_select(const PagedSelect& a, void* ws, hipStream_t stream) {
  const int64_t G = a.Hq / a.pool.H, M = a.pool.max_pages;
  const int tt = select_rows(G, a.Tq, M), qtiles = (a.Tq + tt - 1) / tt;
  const dim3 grid((unsigned)((int64_t)a.N * a.pool.H * qtiles)), nt(PS_NW * 64);
  if (M > PS_LDS) {
    hipLaunchKernelGGL((paged_select_kernel<T, D, true>), grid, nt, 0, stream, a, tt, qtiles, (uint32_t*)ws);
  } else {
    const size_t lds = (size_t)tt * M * 4;
    static bool set[64];  // per device: more LDS than a kernel may have unasked
    int dev = 0;
    (void)hipGetDevice(&dev);
    if (lds > 32768 && (dev < 0 || dev >= 64 || !set[dev])) {
      (void)hipFuncSetAttribute((const void*)paged_select_kernel<T, D, false>, hipFuncAttributeMaxDynamicSharedMemorySize,
                                PS_LDS * 4);
      if (dev >= 0 && dev < 64) set[dev] = true;
    }
    hipLaunchKernelGGL((paged_select_kernel<T, D, false>), grid, nt, lds, stream, a, tt, qtiles, (uint32_t*)nullptr);
  }
}

// ---------------------------------------------------------------------------------------------
// attention
// ---------------------------------------------------------------------------------------------
// The segments of paged_core.h over the listed pages: an item is a query row with its K/V head (16 heads of the group a tile),
// cut into `splits` runs of `chunk` rows of its list where there are too few items for the GPU.
template <typename T, typename C, int D>
__global__ __launch_bounds__(256, 2) void ps_kernel(PagedAttn a, PagedSplit z, int splits, int chunk) {
  const int b = xcd_remap(blockIdx.x, gridDim.x), part = b % splits;  // an XCD's workgroups share pages in its L2
  const int64_t item = b / splits;
  const int qt = (int)(item % z.qtiles), t = (int)(item / z.qtiles % a.Tq), nh = (int)(item / z.qtiles / a.Tq);
  const int64_t all = (int64_t)a.K << a.pool.shift, c0 = (int64_t)part * chunk;
  const int c1 = (int)(c0 + chunk < all ? c0 + chunk : all);
  pa_segment<T, C, D, 1, false, true, 4>(a, z, nh / a.pool.H, nh % a.pool.H, t, qt, (int)(c0 < all ? c0 : all), c1,
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
    int64_t s = items > 0 ? 2 * cu_count() / items : 1;
    const int64_t most = (rows + 255) / 256;  // 256 rows at least
    s = s < 1 ? 1 : s < most ? s : most;
    if (s < 1) s = 1;
    chunk = ((rows + s - 1) / s + 127) / 128 * 128;  // whole turns
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
  hipLaunchKernelGGL((ps_kernel<T, C, D>), dim3((unsigned)(cut.items * cut.splits)), dim3(256), 0, stream, a, z, cut.splits,
                     (int)cut.chunk);
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
    const dim3 grid((unsigned)gx, (unsigned)(a.N - n < some ? a.N - n : some)), nt(256);
    if (format == 0) hipLaunchKernelGGL(paged_bounds_kernel<bf16>, grid, nt, 0, stream, part);
    else if (format == 1) hipLaunchKernelGGL(paged_bounds_kernel<float>, grid, nt, 0, stream, part);
    else if (format == 2) hipLaunchKernelGGL(paged_bounds_kernel<E4M3>, grid, nt, 0, stream, part);
    else hipLaunchKernelGGL(paged_bounds_kernel<I8>, grid, nt, 0, stream, part);
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
