// Arguments of the paged K/V cache kernels (paged.hip), shared with the argument checks in abi.hip.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

// A pool of pages [pages, H, R, D] (element stride page_sp between pages, the rest contiguous; R = 1 << shift) and the
// page table [N, max_pages] (row stride table_sn) of the sequences that live in it. Row i of sequence n is row i % R of
// page table[n, i / R]. lengths[n] (device) is clamped to [0, max_pages R]; a page id outside [0, pages) holds no rows.
struct PagedPool {
  void* k;
  void* v;
  int64_t pages, page_sp;
  int H, D, shift;
  const int32_t* table;
  int64_t table_sn;
  int max_pages;
  const int32_t* lengths;
};

struct PagedAttn {
  PagedPool pool;
  const void* q;
  int64_t q_sn, q_sh, q_st;
  void* out;
  int64_t o_sn, o_sh, o_st;
  float* weights;  // [N, max_pages R] (row stride weights_sn) or null
  int64_t weights_sn;
  int N, Hq, Tq;
  float scale;
  const float* scales;   // of 8-bit pools: [pages, H, 2] (K, V)
  const int32_t* index;  // [N, H, Tq, K]: the pages (their places in the table) that each query row attends to, or null: all
  int K;
};

struct PagedAppend {
  PagedPool pool;
  const void *k, *v;
  int64_t k_sn, k_sh, k_st, v_sn, v_sh, v_st;
  const int32_t* count;  // [N] or null: every row
  int N, T;
};

struct PagedGather {
  PagedPool pool;
  void *k, *v;  // [N, H, T, D] contiguous
  int N, T;
};

struct PagedEvict {
  PagedPool pool;  // k, v: block 0
  int64_t blocks, block_sp;
  const float* weights;
  int64_t weights_sn;
  const int32_t* keep;  // [N] or null: keep_all
  int keep_all, recent;
  int32_t* index;  // [N, K]
  int K;
  float* kept_weights;  // [N, max_pages R]
  int32_t* kept_lengths;
  int N;
};

// Workgroups of a launch (256 threads, or 1,024 for a quarter of them): below the 2^32 threads beyond which a launch leaves
// workgroups out without an error.
#define PAGED_MAX_GRID (1ll << 23)

// Query rows over all sequences and heads that a launch of the attention takes, and units (128 rows of a sequence, K/V head
// and tile of 16 query rows), which it counts in 32 bits. Calls of more query rows go in slices.
#define PAGED_MAX_QUERIES (1ll << 22)
#define PAGED_MAX_UNITS (1ll << 30)

// dtype codes 0 bf16, 1 fp32. Return value: hipGetLastError() after the launches.
int tabicl_launch_paged_attn(const PagedAttn& a, int dtype, void* ws, hipStream_t stream);
int64_t tabicl_launch_paged_attn_ws_bytes(int64_t N, int64_t Hq, int64_t H, int64_t Tq, int64_t D, int64_t rows, int weights,
                                          int dtype);
int tabicl_launch_paged_append(const PagedAppend& a, int dtype, hipStream_t stream);
int tabicl_launch_paged_gather(const PagedGather& a, int dtype, hipStream_t stream);
int tabicl_launch_paged_evict(const PagedEvict& a, int dtype, void* ws, hipStream_t stream);
int64_t tabicl_launch_paged_evict_ws_bytes(int64_t N, int64_t rows);

// Pools of 8-bit codes (paged_q8.hip): code 0 e4m3, 1 int8; scales [pages, H, 2]; dtype: of q, out and the rows.
struct PagedAppend8 {
  PagedAppend rows;
  float* scales;
  const int32_t* starts;  // [N]: row t of sequence n is row starts[n] + t of k and v (k_sn, v_sn unused), or null
};
int tabicl_launch_paged_attn_q8(const PagedAttn& a, int dtype, int code, void* ws, hipStream_t stream);
int64_t tabicl_launch_paged_attn_q8_ws_bytes(int64_t N, int64_t Hq, int64_t H, int64_t Tq, int64_t D, int64_t rows, int dtype);
int tabicl_launch_paged_append_q8(const PagedAppend8& a, int dtype, int code, hipStream_t stream);
int tabicl_launch_paged_gather_q8(const PagedGather& a, const float* scales, int dtype, int code, hipStream_t stream);

// Attention over selected pages (paged_sparse.hip). Pool formats: 0 bf16, 1 fp32, 2 e4m3, 3 int8.
struct PagedBounds {
  PagedPool pool;  // v unused
  const float* scales;
  const int32_t* start;  // [N] or null: pages wholly below this row keep their bounds
  int8_t* bounds;        // [pages, H, 2, D]
  float* bound_scales;   // [pages, H]
  int N;
};
struct PagedSelect {
  PagedPool pool;  // k, v unused
  const void* q;
  int64_t q_sn, q_sh, q_st;
  const int8_t* bounds;
  const float* bound_scales;
  int32_t* index;  // [N, H, Tq, K]
  int N, Hq, Tq, K;
};
int tabicl_launch_paged_bounds(const PagedBounds& a, int format, int64_t rows, hipStream_t stream);
int tabicl_launch_paged_select(const PagedSelect& a, int dtype, void* ws, hipStream_t stream);
int64_t tabicl_launch_paged_select_ws_bytes(int64_t N, int64_t H, int64_t Tq, int64_t max_pages);
int tabicl_launch_paged_sparse(const PagedAttn& a, int format, int dtype, void* ws, hipStream_t stream);
int64_t tabicl_launch_paged_sparse_ws_bytes(int64_t N, int64_t Hq, int64_t H, int64_t Tq, int64_t D, int64_t rows);

// The books of a pool (paged_books.hip).
struct PagedBooks {
  int32_t* table;
  int64_t table_sn;
  int max_pages, pages, shift, N;
  const int32_t* lengths;
  const int32_t* count;
  int32_t* free_pages;  // a stack of up to `pages` ids, *free_count of them
  int32_t* free_count;
  int32_t* granted;
};
int tabicl_launch_paged_reserve(const PagedBooks& a, void* ws, hipStream_t stream);
int tabicl_launch_paged_release(const PagedBooks& a, void* ws, hipStream_t stream);
int64_t tabicl_launch_paged_books_ws_bytes(int64_t N);
int tabicl_launch_paged_slots(const PagedBooks& a, int64_t* slots, int32_t* starts, int64_t total, hipStream_t stream);
int tabicl_launch_paged_append_slots(const PagedAppend& a, const int64_t* slots, int64_t total, int dtype, hipStream_t stream);
