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
