// A K/V cache in pages (gfx950): tables of different sizes share one pool, a test row or a few attend over the cached rows
// of their table, the attention weights add up per cached row, and a cache over its budget keeps the rows that drew most.
//
//   s_i = scale q . K_i  (i < len),   p = exp(s - max s),   out = sum_i p_i V_i / sum_i p_i   (len = 0: 0)
//   weights_i += sum over heads and query rows of p_i / sum p
#include "launch.h"
#include "paged_core.h"

#include <numeric>

namespace {

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
    return pa_merge_row<T, T, D, QT>(a, z, (int64_t)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6));
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
      hipLaunchKernelGGL((pa_whole_kernel<T, T, D, QT, W>), dim3((unsigned)(a.N * a.pool.H * z.qtiles)), dim3(512), 0, stream, a, z);
  } else {
    hipLaunchKernelGGL((pa_kernel<T, T, D, QT, W>), dim3((unsigned)z.groups), dim3(256), 0, stream, a, z);
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
    hipLaunchKernelGGL((pa_merge_kernel<T, T, D, QT>), dim3(merge), dim3(256), 0, stream, a, z);
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
