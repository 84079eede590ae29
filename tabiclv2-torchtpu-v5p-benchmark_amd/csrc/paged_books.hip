// The books of a paged K/V cache on the GPU (gfx950): pages for the rows that requests get (from a stack of free ones), back to
// the stack when rows are withdrawn, the slot of each row of a packed batch, and such rows into their slots. Everything stays
// on the device, so that a step of a serving loop can be captured and replayed while the requests grow.
//
//   reserve: entries p of the table, ceil(len / R) <= p < ceil((len + count) / R), that hold no page get one: the r-th such
//            entry (by sequence, then p) the r-th page from the top of the stack, as far as it goes; granted: the rows before
//            the first without a page, none where row len joins a page (len / R, not among those) that is not there
//   release: entries p >= ceil(len / R) that hold a page give it back and become -1: the last one first, so that a release
//            undoes a reserve, stack and all
//   slots:   row j of a packed batch, the t-th of sequence n: table[n, (len + t) / R] R + (len + t) % R, or -1
//
// All are bound by the latency of their launches (a few bytes a row): tables of up to 65,536 entries are gone through by one
// workgroup in one launch, larger ones by many in two (the first counts).
#include "launch.h"
#include "paged_core.h"

namespace {

constexpr int PB_GROUPS = 256;  // workgroups that share the sequences of the second launch

__device__ __forceinline__ int below(uint64_t mask) {
  return __builtin_amdgcn_mbcnt_hi((uint32_t)(mask >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)mask, 0));
}

struct BookRange {
  int64_t len, add;
  int first, last;  // the entries of the table that are looked at
  __device__ __forceinline__ BookRange(const PagedBooks& a, int n, bool release) {
    const int64_t cap = (int64_t)a.max_pages << a.shift, R = 1ll << a.shift;
    len = a.lengths[n];
    len = len < 0 ? 0 : len < cap ? len : cap;
    add = release ? 0 : a.count[n];
    add = add < 0 ? 0 : add;
    first = (int)((len + R - 1) >> a.shift);
    const int64_t end = (len + add + R - 1) >> a.shift;
    last = release || end > a.max_pages ? a.max_pages : (int)end;
  }
};

__device__ __forceinline__ bool book_has(const PagedBooks& a, int id) { return id >= 0 && id < a.pages; }

// The page that row `len` of sequence n joins, 0 where it begins one.
__device__ __forceinline__ int book_joins(const PagedBooks& a, int n, int64_t len) {
  return len & ((1ll << a.shift) - 1) ? a.table[n * a.table_sn + (len >> a.shift)] : 0;
}

// need[n]: the entries of sequence n that get (or give back) a page; need[N]: the pages on the stack. A wave per sequence.
template <bool RELEASE>
__global__ __launch_bounds__(256) void paged_need_kernel(PagedBooks a, int32_t* need) {
  const int n = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  if (blockIdx.x == 0 && threadIdx.x == 0) {
    const int f = *a.free_count;
    need[a.N] = f < 0 ? 0 : f < a.pages ? f : a.pages;
  }
  if (n >= a.N) return;
  const BookRange r(a, n, RELEASE);
  int count = 0;
  for (int p = r.first; p < r.last; p += 64) {
    const bool in = p + lane < r.last;
    const int id = in ? a.table[n * a.table_sn + p + lane] : 0;
    count += __popcll(__ballot(in && book_has(a, id) == RELEASE));
  }
  if (lane == 0) need[n] = count;
}

// A workgroup takes `per` sequences, a wave one at a time.
template <bool RELEASE>
__global__ __launch_bounds__(256) void paged_books_kernel(PagedBooks a, const int32_t* need, int per) {
  __shared__ int64_t sh[2][4];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int n0 = blockIdx.x * per, n1 = n0 + per < a.N ? n0 + per : a.N, have = need[a.N];
  int64_t before = 0, all = 0;  // entries of the sequences before the first one; of all
  for (int n = threadIdx.x; n < (RELEASE || n1 == a.N ? a.N : n0); n += 256) {
    const int x = need[n];
    all += x;
    before += n < n0 ? x : 0;
  }
#pragma unroll
  for (int x = 1; x < 64; x <<= 1) {
    before += __shfl_xor(before, x, 64);
    all += __shfl_xor(all, x, 64);
  }
  if (lane == 0) sh[0][wave] = before, sh[1][wave] = all;
  __syncthreads();
  before = sh[0][0] + sh[0][1] + sh[0][2] + sh[0][3];
  all = sh[1][0] + sh[1][1] + sh[1][2] + sh[1][3];
  for (int n = n0; n < n1; ++n) {
    const int mine = need[n];
    if ((n - n0) % 4 == wave) {
      const BookRange r(a, n, RELEASE);
      const int joins = RELEASE ? 0 : book_joins(a, n, r.len);
      int64_t rank = before;
      int missing = a.max_pages;
      for (int p = r.first; p < r.last; p += 64) {
        const bool in = p + lane < r.last;
        int32_t* entry = a.table + n * a.table_sn + p + lane;
        int id = in ? *entry : 0;
        const bool has = in && book_has(a, id), moves = in && has == RELEASE;
        const uint64_t m = __ballot(moves);
        const int64_t at = rank + below(m);
        rank += __popcll(m);
        if constexpr (RELEASE) {
          if (moves) {
            const int64_t to = have + all - 1 - at;
            if (to < a.pages) a.free_pages[to] = id;
            *entry = -1;
          }
        } else {
          if (moves && at < have) {
            id = a.free_pages[have - 1 - at];
            *entry = id;
          }
          const uint64_t none = __ballot(in && !book_has(a, id));
          if (none && missing == a.max_pages) missing = p + __builtin_ctzll(none);
        }
      }
      if (!RELEASE && lane == 0) {  // rows up to the first page that is not there
        const int64_t rows = ((int64_t)missing << a.shift) - r.len;
        a.granted[n] = (int)(rows < 0 || !book_has(a, joins) ? 0 : rows < r.add ? rows : r.add);
      }
    }
    before += mine;
  }
  if (n1 == a.N && threadIdx.x == 0) {
    const int64_t left = RELEASE ? have + all : have - all;
    *a.free_count = (int)(left < 0 ? 0 : left < a.pages ? left : a.pages);
  }
}

// One workgroup for up to 256 sequences and BOOKS_ONE entries: counts, running sums and the entries in one launch. The entries to
// look at are cut into runs of 64 of one sequence; a wave takes 16 runs at a time, all of them in its registers at once. (us of
// a reserve on the GPU, two launches / this: 256 requests of one row 6.3 / 6.2, 64 of up to 10,000 rows 7.6 / 8.9; of reserve,
// slots, a copy and release as a program calls them, host included: 32.5 / 25.4 and 32.5 / 25.2.)
constexpr int BOOKS_SEQS = 256, BOOKS_ONE = 65536, BOOKS_RUNS = BOOKS_ONE / 64 + BOOKS_SEQS, PB_NW = 16, PB_EACH = 16;

template <bool RELEASE>
__global__ __launch_bounds__(PB_NW * 64) void paged_books_one_kernel(PagedBooks a) {
  __shared__ int2 run[BOOKS_RUNS], rows[BOOKS_SEQS];  // (sequence, first entry | entries - 1); the rows in place and those wanted
  __shared__ int need[BOOKS_RUNS], miss[BOOKS_SEQS], sums[PB_NW];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int claimed = *a.free_count, have = claimed < 0 ? 0 : claimed < a.pages ? claimed : a.pages;
  // the sum of x over the threads before this one, and over all
  auto before = [&](int x, int* all) {
    const int upto = wave_sum_scan(x);
    if (lane == 63) sums[wave] = upto;
    __syncthreads();
    const int waves = wave_sum_scan(lane < PB_NW ? sums[lane] : 0);
    __syncthreads();
    *all = __builtin_amdgcn_readlane(waves, 63);
    return (wave ? __builtin_amdgcn_readlane(waves, wave - 1) : 0) + upto - x;
  };
  int first = 0, last = 0, runs, joins = 0;
  if (tid < a.N) {
    const BookRange r(a, tid, RELEASE);
    first = r.first, last = r.last > r.first ? r.last : r.first;
    rows[tid] = make_int2((int)r.len, (int)r.add);
    miss[tid] = a.max_pages;
    if (!RELEASE) joins = book_joins(a, tid, r.len);
  }
  int at = before((last - first + 63) / 64, &runs);
#pragma unroll 1
  for (int p = first; p < last; p += 64) run[at++] = make_int2(tid, p << 6 | ((last - p < 64 ? last - p : 64) - 1));
  __syncthreads();
  int32_t* entry[PB_EACH];
  int id[PB_EACH], rank[PB_EACH];
  bool moves[PB_EACH];
  auto load = [&](int k0) {  // every load is issued, so that none waits for the one before
#pragma unroll
    for (int u = 0; u < PB_EACH; ++u) {
      const int k = k0 + wave * PB_EACH + u;
      const int2 r = k < runs ? run[k] : make_int2(0, 0);
      const bool in = k < runs && lane <= (r.y & 63);
      entry[u] = in ? a.table + r.x * a.table_sn + (r.y >> 6) + lane : a.table;
      id[u] = *entry[u];
      moves[u] = in;
    }
#pragma unroll
    for (int u = 0; u < PB_EACH; ++u) moves[u] = moves[u] && book_has(a, id[u]) == RELEASE;
  };
#pragma unroll 1
  for (int k0 = 0; k0 < runs; k0 += PB_NW * PB_EACH) {
    if (k0 + wave * PB_EACH >= runs) break;  // none left for this wave
    load(k0);
    int mine = 0;
#pragma unroll
    for (int u = 0; u < PB_EACH; ++u) {
      const int count = __popcll(__ballot(moves[u]));
      mine = lane == u ? count : mine;
    }
    if (lane < PB_EACH && k0 + wave * PB_EACH + lane < runs) need[k0 + wave * PB_EACH + lane] = mine;
  }
  __syncthreads();
  int all;
  const int x0 = 2 * tid < runs ? need[2 * tid] : 0, x1 = 2 * tid + 1 < runs ? need[2 * tid + 1] : 0;
  const int start = before(x0 + x1, &all);
  if (2 * tid < runs) need[2 * tid] = start;
  if (2 * tid + 1 < runs) need[2 * tid + 1] = start + x0;
  __syncthreads();
#pragma unroll 1
  for (int k0 = 0; k0 < runs; k0 += PB_NW * PB_EACH) {
    if (k0 + wave * PB_EACH >= runs) break;
    if (runs > PB_NW * PB_EACH) load(k0);  // else they are here
#pragma unroll
    for (int u = 0; u < PB_EACH; ++u) {
      const int k = k0 + wave * PB_EACH + u;
      rank[u] = (k < runs ? need[k] : 0) + below(__ballot(moves[u]));
      if constexpr (RELEASE) {
        const int64_t to = (int64_t)have + all - 1 - rank[u];
        if (moves[u] && to < a.pages) a.free_pages[to] = id[u];
        if (moves[u]) *entry[u] = -1;
      }
    }
    if (!RELEASE && have > 0) {
      int page[PB_EACH];
#pragma unroll
      for (int u = 0; u < PB_EACH; ++u) page[u] = a.free_pages[moves[u] && rank[u] < have ? have - 1 - rank[u] : 0];
#pragma unroll
      for (int u = 0; u < PB_EACH; ++u) id[u] = moves[u] && rank[u] < have ? page[u] : id[u];
    }
    if constexpr (!RELEASE) {
#pragma unroll
      for (int u = 0; u < PB_EACH; ++u) {
        const int k = k0 + wave * PB_EACH + u;
        if (moves[u]) *entry[u] = id[u];  // as it was, if the stack had none left
        if (moves[u] && !book_has(a, id[u])) atomicMin(&miss[run[k].x], (run[k].y >> 6) + lane);
      }
    }
  }
  if constexpr (!RELEASE) {  // rows up to the first page that is not there
    __syncthreads();
    if (tid < a.N) {
      const int64_t there = ((int64_t)miss[tid] << a.shift) - rows[tid].x;
      a.granted[tid] = (int)(there < 0 || !book_has(a, joins) ? 0 : there < rows[tid].y ? there : rows[tid].y);
    }
  }
  if (tid == 0) {
    const int64_t left = RELEASE ? (int64_t)have + all : (int64_t)have - all;
    *a.free_count = (int)(left < 0 ? 0 : left < a.pages ? left : a.pages);
  }
}

// The slots of `per` rows of the batch by a workgroup: the counts' running sums, PS_SEQS sequences at a time in LDS, a row's
// sequence by bisection, four rows of a thread side by side.
constexpr int PS_SEQS = 1024, PS_ROWS = 4;

__global__ __launch_bounds__(256) void paged_slots_kernel(PagedBooks a, int64_t* slots, int32_t* starts, int64_t total, int per) {
  __shared__ int64_t sum[PS_SEQS + 1];
  __shared__ int64_t wsum[4];
  __shared__ int32_t held[PS_SEQS];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int64_t j0 = (int64_t)blockIdx.x * per, j1 = j0 + per < total ? j0 + per : total, cap = (int64_t)a.max_pages << a.shift;
  constexpr int EACH = PS_SEQS / 256;
  int64_t base = 0;
  for (int s0 = 0; s0 < a.N && (base < j1 || blockIdx.x == 0); s0 += PS_SEQS) {
    int64_t c[EACH], mine = 0;
    int x[EACH];
#pragma unroll
    for (int i = 0; i < EACH; ++i) {
      const int n = s0 + tid * EACH + i;
      x[i] = n < a.N ? a.count[n] : 0;
      held[tid * EACH + i] = n < a.N ? a.lengths[n] : 0;
    }
#pragma unroll
    for (int i = 0; i < EACH; ++i) {
      c[i] = mine;
      mine += x[i] < 0 ? 0 : x[i];
    }
    int64_t upto = mine;
#pragma unroll
    for (int y = 1; y < 64; y <<= 1) {
      const int64_t z = __shfl_up(upto, y, 64);
      if (lane >= y) upto += z;
    }
    if (lane == 63) wsum[wave] = upto;
    __syncthreads();
    int64_t off = base + upto - mine;
    for (int w = 0; w < wave; ++w) off += wsum[w];
#pragma unroll
    for (int i = 0; i < EACH; ++i) {
      const int n = s0 + tid * EACH + i;
      sum[tid * EACH + i] = off + c[i];
      if (blockIdx.x == 0 && n < a.N) starts[n] = (int32_t)(off + c[i]);
    }
    const int64_t next = base + wsum[0] + wsum[1] + wsum[2] + wsum[3];
    if (tid == 0) sum[PS_SEQS] = next;
    __syncthreads();
    const int64_t lo = j0 > base ? j0 : base, hi = j1 < next ? j1 : next;
    const int seqs = a.N - s0 < PS_SEQS ? a.N - s0 : PS_SEQS;  // sum[seqs] = next
    for (int64_t j = lo + tid; j < hi; j += 256 * PS_ROWS) {
      int l[PS_ROWS], id[PS_ROWS];
      int64_t row[PS_ROWS];
#pragma unroll
      for (int i = 0; i < PS_ROWS; ++i) l[i] = 0;
      for (int step = PS_SEQS / 2; step > 0; step >>= 1) {
        if (step >= seqs) continue;
#pragma unroll
        for (int i = 0; i < PS_ROWS; ++i)
          if (l[i] + step < seqs && sum[l[i] + step] <= j + 256 * i) l[i] += step;  // the last sum <= j + 256 i
      }
#pragma unroll
      for (int i = 0; i < PS_ROWS; ++i) {
        row[i] = (held[l[i]] < 0 ? 0 : held[l[i]]) + j + 256 * i - sum[l[i]];
        const bool in = j + 256 * i < hi && row[i] < cap;
        id[i] = in ? a.table[(s0 + l[i]) * a.table_sn + (row[i] >> a.shift)] : -1;
      }
#pragma unroll
      for (int i = 0; i < PS_ROWS; ++i)
        if (j + 256 * i < hi)
          slots[j + 256 * i] = book_has(a, id[i]) ? ((int64_t)id[i] << a.shift) + (row[i] & ((1ll << a.shift) - 1)) : -1;
    }
    base = next;
    __syncthreads();
  }
  if (blockIdx.x == 0 && tid == 0) starts[a.N] = (int32_t)base;
  for (int64_t j = (j0 > base ? j0 : base) + tid; j < j1; j += 256) slots[j] = -1;  // behind the last row
}

// Rows j of k, v [total, H, D] into their slots; 16 bytes of K and of V per thread.
__global__ __launch_bounds__(256) void paged_append_slots_kernel(PagedAppend a, const int64_t* slots, int64_t total, int es) {
  const PagedPool& c = a.pool;
  const int chunks = c.D * es / 16, per = c.H * chunks;
  const int64_t all = total * per, most = (int64_t)c.pages << c.shift;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < all; i += (int64_t)gridDim.x * 256) {
    const int64_t j = i / per;
    const int x = (int)(i - j * per), h = x / chunks, ch = x % chunks;
    const int64_t slot = slots[j];
    if (slot < 0 || slot >= most) continue;
    const int64_t to = ((slot >> c.shift) * c.page_sp + (((int64_t)h << c.shift) + (slot & ((1ll << c.shift) - 1))) * c.D) * es + ch * 16;
    *(uint4*)((char*)c.k + to) = ldg16((const char*)a.k + (h * a.k_sh + j * a.k_st) * es + ch * 16);
    *(uint4*)((char*)c.v + to) = ldg16((const char*)a.v + (h * a.v_sh + j * a.v_st) * es + ch * 16);
  }
}

template <bool RELEASE>
int launch_books(const PagedBooks& a, void* ws, hipStream_t stream) {
  if (a.N <= BOOKS_SEQS && (int64_t)a.N * a.max_pages <= BOOKS_ONE) {
    hipLaunchKernelGGL(paged_books_one_kernel<RELEASE>, dim3(1), dim3(PB_NW * 64), 0, stream, a);
    return (int)hipGetLastError();
  }
  const int per = (a.N + PB_GROUPS - 1) / PB_GROUPS < 4 ? 4 : (a.N + PB_GROUPS - 1) / PB_GROUPS;
  hipLaunchKernelGGL(paged_need_kernel<RELEASE>, dim3((unsigned)((a.N + 3) / 4)), dim3(256), 0, stream, a, (int32_t*)ws);
  hipLaunchKernelGGL(paged_books_kernel<RELEASE>, dim3((unsigned)((a.N + per - 1) / per)), dim3(256), 0, stream, a,
                     (const int32_t*)ws, per);
  return (int)hipGetLastError();
}

}  // namespace

int64_t tabicl_launch_paged_books_ws_bytes(int64_t N) { return align256((N + 1) * 4); }

int tabicl_launch_paged_reserve(const PagedBooks& a, void* ws, hipStream_t stream) { return launch_books<false>(a, ws, stream); }

int tabicl_launch_paged_release(const PagedBooks& a, void* ws, hipStream_t stream) { return launch_books<true>(a, ws, stream); }

int tabicl_launch_paged_slots(const PagedBooks& a, int64_t* slots, int32_t* starts, int64_t total, hipStream_t stream) {
  int64_t per = 1024, groups = (total + per - 1) / per;
  if (groups > 2048) {
    per = (total + 2047) / 2048;
    groups = (total + per - 1) / per;
  }
  if (groups < 1) groups = 1;  // the starts all the same
  hipLaunchKernelGGL(paged_slots_kernel, dim3((unsigned)groups), dim3(256), 0, stream, a, slots, starts, total, (int)per);
  return (int)hipGetLastError();
}

int tabicl_launch_paged_append_slots(const PagedAppend& a, const int64_t* slots, int64_t total, int dtype, hipStream_t stream) {
  const int es = dtype == 0 ? 2 : 4;
  int64_t gx = (total * a.pool.H * (a.pool.D * es / 16) + 255) / 256;
  if (gx > 65536) gx = 65536;
  hipLaunchKernelGGL(paged_append_slots_kernel, dim3((unsigned)gx), dim3(256), 0, stream, a, slots, total, es);
  return (int)hipGetLastError();
}
