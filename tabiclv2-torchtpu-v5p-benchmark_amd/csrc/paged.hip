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
// attention: one workgroup per (sequence, head, query row), a key per thread, keys in steps of 256
// ---------------------------------------------------------------------------------------------
constexpr int PA_NT = 256;

__device__ __forceinline__ float block_reduce(float x, float* sh, bool is_max) {
  for (int m = 32; m >= 1; m >>= 1) {
    const float y = __shfl_xor(x, m, 64);
    x = is_max ? fmaxf(x, y) : x + y;
  }
  __syncthreads();
  if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = x;
  __syncthreads();
  x = sh[0];
  for (int w = 1; w < PA_NT / 64; ++w) x = is_max ? fmaxf(x, sh[w]) : x + sh[w];
  return x;
}

template <typename T>
__device__ float key_score(const PagedAttn& a, int n, int hkv, int row, const float* sq) {
  const int64_t off = pool_row(a.pool, n, hkv, row);
  if (off < 0) return TA_NEG_INF;
  const T* k = (const T*)a.pool.k + off;
  float s = 0.f;
  for (int d = 0; d < a.pool.D; ++d) s = __builtin_fmaf(sq[d], (float)k[d], s);
  return s * a.scale;
}

template <typename T>
__global__ __launch_bounds__(PA_NT) void pa_kernel(PagedAttn a, float2* stat) {
  __shared__ float sq[128], sp[PA_NT], sh[PA_NT / 64], acc[PA_NT];
  const int t = blockIdx.x % a.Tq, h = (blockIdx.x / a.Tq) % a.Hq, n = blockIdx.x / a.Tq / a.Hq;
  const int hkv = h / (a.Hq / a.pool.H), D = a.pool.D, len = pool_length(a.pool, n), tid = threadIdx.x;
  if (tid < D) sq[tid] = (float)((const T*)a.q)[n * a.q_sn + h * a.q_sh + t * a.q_st + tid];
  __syncthreads();
  float m = TA_NEG_INF;
  for (int r = tid; r < len; r += PA_NT) m = fmaxf(m, key_score<T>(a, n, hkv, r, sq));
  m = block_reduce(m, sh, true);
  const int groups = PA_NT / D, d = tid % D, grp = tid / D;
  float l = 0.f, o = 0.f;
  for (int r0 = 0; r0 < len; r0 += PA_NT) {
    const int r = r0 + tid;
    // 2^-31: sums of up to 2^30 products with values near the largest float stay finite
    const float p = r < len && m > TA_NEG_INF ? __expf(key_score<T>(a, n, hkv, r, sq) - m) * 0x1p-31f : 0.f;
    l += p;
    __syncthreads();
    sp[tid] = p;
    __syncthreads();
    for (int j = grp; j < PA_NT && r0 + j < len; j += groups) {
      const int64_t off = pool_row(a.pool, n, hkv, r0 + j);
      if (off >= 0) o = __builtin_fmaf(sp[j], (float)((const T*)a.pool.v)[off + d], o);
    }
  }
  l = block_reduce(l, sh, false);
  acc[tid] = o;
  __syncthreads();
  if (tid < D) {
    o = 0.f;
    for (int g = 0; g < groups; ++g) o += acc[g * D + d];
    ((T*)a.out)[n * a.o_sn + h * a.o_sh + t * a.o_st + d] = (T)(l == 0.f ? 0.f : o / l);
  }
  if (stat && tid == 0) stat[blockIdx.x] = make_float2(m, l);
}

template <typename T>
__global__ __launch_bounds__(PA_NT) void pa_weights_kernel(PagedAttn a, const float2* stat) {
  __shared__ float sq[128];
  const int n = blockIdx.y, len = pool_length(a.pool, n), tid = threadIdx.x, row = blockIdx.x * PA_NT + tid;
  if ((int)blockIdx.x * PA_NT >= len) return;
  float w = 0.f;
  for (int i = 0; i < a.Hq * a.Tq; ++i) {
    const int h = i / a.Tq, t = i % a.Tq;
    __syncthreads();
    if (tid < a.pool.D) sq[tid] = (float)((const T*)a.q)[n * a.q_sn + h * a.q_sh + t * a.q_st + tid];
    __syncthreads();
    const float2 ml = stat[(int64_t)n * a.Hq * a.Tq + i];
    if (row < len && ml.y != 0.f) w += __expf(key_score<T>(a, n, h / (a.Hq / a.pool.H), row, sq) - ml.x) * 0x1p-31f / ml.y;
  }
  if (row < len) a.weights[n * a.weights_sn + row] += w;
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

// The number of set flags before this thread's, and the workgroup's total.
__device__ __forceinline__ int block_rank(bool flag, int* sh, int* total) {
  const uint64_t b = __ballot(flag);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  __syncthreads();
  if (lane == 0) sh[wave] = __popcll(b);
  __syncthreads();
  int before = __popcll(b & ((1ull << lane) - 1)), sum = 0;
  for (int w = 0; w < PE_NT / 64; ++w) {
    before += w < wave ? sh[w] : 0;
    sum += sh[w];
  }
  *total = sum;
  return before;
}

// pairs [N, K]: (source row << 32 | place) of the rows that move, count in npairs[n].
__global__ __launch_bounds__(PE_NT) void paged_select_kernel(PagedEvict a, int64_t* pairs, int32_t* npairs) {
  __shared__ int hist[256], sh[PE_NT / 64], pick[2];
  const int n = blockIdx.x, tid = threadIdx.x;
  const EvictSizes z = evict_sizes(a, n);
  const float* w = a.weights + n * a.weights_sn;
  const int64_t cap = (int64_t)a.pool.max_pages << a.pool.shift;
  const int free_rows = z.len - z.recent;
  int want = z.kept - z.recent;  // of the rows [0, free_rows)
  // threshold code: the want-th largest, one digit of 8 bits at a time
  uint32_t prefix = 0;
  for (int shift = 24; shift >= 0 && want > 0; shift -= 8) {
    if (tid < 256) hist[tid] = 0;
    __syncthreads();
    for (int r = tid; r < free_rows; r += PE_NT) {
      const uint32_t c = weight_code(w[r]);
      if (shift == 24 || (c >> (shift + 8)) == (prefix >> (shift + 8))) atomicAdd(&hist[(c >> shift) & 255], 1);
    }
    __syncthreads();
    if (tid == 0) {
      int left = want, b = 255;
      for (; b > 0 && hist[b] < left; --b) left -= hist[b];
      pick[0] = b;
      pick[1] = left;
    }
    __syncthreads();
    prefix |= (uint32_t)pick[0] << shift;
    want = pick[1];
    __syncthreads();
  }
  // want: rows of exactly the threshold's weight that are kept, the lowest ones
  const bool any = z.kept > z.recent;
  int64_t* pr = pairs + (int64_t)n * a.K;
  int32_t* index = a.index + (int64_t)n * a.K;
  float* kw = a.kept_weights + n * cap;
  int ties = 0, holes = 0, tails = 0;
  for (int r0 = 0; r0 < z.len; r0 += PE_NT) {
    const int r = r0 + tid;
    const uint32_t c = r < free_rows ? weight_code(w[r]) : 0;
    int total;
    const bool tie = any && r < free_rows && c == prefix;
    const int tie_rank = ties + block_rank(tie, sh, &total);
    ties += total;
    const bool keep = r < z.len && (r >= free_rows || (any && c > prefix) || (tie && tie_rank < want));
    const bool hole = r < z.kept && !keep, tail = r >= z.kept && keep;
    const int hole_rank = holes + block_rank(hole, sh, &total);
    holes += total;
    const int tail_rank = tails + block_rank(tail, sh, &total);
    tails += total;
    if (hole) ((int32_t*)(pr + hole_rank))[0] = r;
    if (tail) ((int32_t*)(pr + tail_rank))[1] = r;
    if (keep && r < z.kept) {
      index[r] = r;
      kw[r] = w[r];
    }
  }
  __syncthreads();
  for (int i = tid; i < holes; i += PE_NT) {
    const int to = ((int32_t*)(pr + i))[0], from = ((int32_t*)(pr + i))[1];
    index[to] = from;
    kw[to] = w[from];
  }
  for (int r = z.kept + tid; r < a.K; r += PE_NT) index[r] = -1;
  for (int64_t r = z.kept + tid; r < cap; r += PE_NT) kw[r] = 0.f;
  if (tid == 0) {
    npairs[n] = holes;
    a.kept_lengths[n] = z.kept;
  }
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

int64_t tabicl_launch_paged_attn_ws_bytes(int64_t N, int64_t Hq, int64_t H, int64_t Tq, int64_t D, int64_t rows, int weights,
                                          int dtype) {
  return weights ? N * Hq * Tq * 8 : 0;
}

int tabicl_launch_paged_attn(const PagedAttn& a, int dtype, void* ws, hipStream_t stream) {
  const unsigned grid = (unsigned)((int64_t)a.N * a.Hq * a.Tq);
  float2* stat = a.weights ? (float2*)ws : nullptr;
  const unsigned wx = (unsigned)((((int64_t)a.pool.max_pages << a.pool.shift) + PA_NT - 1) / PA_NT);
  if (dtype == 0) {
    hipLaunchKernelGGL(pa_kernel<bf16>, dim3(grid), dim3(PA_NT), 0, stream, a, stat);
    if (stat && wx) hipLaunchKernelGGL(pa_weights_kernel<bf16>, dim3(wx, a.N), dim3(PA_NT), 0, stream, a, stat);
  } else {
    hipLaunchKernelGGL(pa_kernel<float>, dim3(grid), dim3(PA_NT), 0, stream, a, stat);
    if (stat && wx) hipLaunchKernelGGL(pa_weights_kernel<float>, dim3(wx, a.N), dim3(PA_NT), 0, stream, a, stat);
  }
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
