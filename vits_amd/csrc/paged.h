// Launchers of the paged-cache operators (kernels_paged.hip): page plan, rotary rows stored to the cache, attention of
// single rows over it.  Layouts and rules: include/vits_amd.h, which declares the entry points over them.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace vits {

constexpr int PAGED_MAX_DIM = 256;          // channels of a head
constexpr int PAGED_MAX_HEADS = 1024;
constexpr int PAGED_MAX_ROWS = 1 << 23;
constexpr int PAGED_PAGE_UNIT = 16;         // page_size is a multiple of it: 16 keys never straddle two pages

struct PagePlanArgs {
  const int *lengths, *grow;
  int requests;
  int* table; long long table_stride; int width;
  int* ring; int pages;
  const int64_t* cursor;
  int page_size;
  int* lengths_out; int64_t* cursor_out;
  int *row_start, *row_request, *row_position;
  int64_t* row_slot;
  int rows;
  int* status;
};
hipError_t launch_page_plan(const PagePlanArgs& a, hipStream_t s);

struct RotaryArgs {
  const void* q; long long q_row, q_head;             // strides in elements
  void* out; long long out_row, out_head;
  int heads;
  const void* k; long long k_row, k_head;
  const void* v; long long v_row, v_head;
  void *k_cache, *v_cache; long long page_stride;
  int pages, page_size, kv_heads, dim, dtype;
  const int* position; const int64_t* slot;
  int rows;
  const double* freq; int pairs; float scale; int interleaved;
  int* err_flag;
};
hipError_t launch_rotary_store(const RotaryArgs& a, hipStream_t s);

struct PagedAttArgs {
  const void* q; long long q_row, q_head;
  const void *k_cache, *v_cache; long long page_stride;
  int pages, page_size;
  const int* table; long long table_stride; int width, requests;
  const int *row_request, *row_position;
  int rows, heads, kv_heads, dim, dtype;
  float scale; int window;
  void* out; long long out_row, out_head;
  float* lse;
  int* err_flag;
};
int64_t paged_attention_workspace(int requests, int rows, int heads, int kv_heads, int dim, int dtype, long long max_keys);
hipError_t launch_paged_attention(const PagedAttArgs& a, long long max_keys, void* ws, hipStream_t s);

}  // namespace vits
