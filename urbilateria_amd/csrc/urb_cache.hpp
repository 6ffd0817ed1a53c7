// urb_cache.hpp -- host-side launch interface of the paged cache's kernels (include/urb_cache.h).
#pragma once

#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

namespace urb {

// Status bits of the cache's contexts.
constexpr int kCacheArgument = 1;
constexpr int kCacheMemory = 2;

// Division by a page size d <= 1024: n / d = n * magic >> shift for n < 2^31.  With 2^s < d <= 2^(s + 1) and shift
// 32 + s the magic number ceil(2^shift / d) has 32 bits, and its excess (below d / 2^shift) times n is below 1 / d.
struct PageDivision {
  uint32_t size, magic, shift;
  static PageDivision by(uint32_t size) {
    PageDivision d{size, 0, 31};
    while (size > 1u << (d.shift - 31)) ++d.shift;
    d.magic = (uint32_t)(((1ull << d.shift) + size - 1) / size);
    return d;
  }
  __host__ __device__ uint32_t of(uint32_t n) const { return (uint32_t)((uint64_t)n * magic >> shift); }
  __host__ __device__ uint32_t up(uint32_t n) const { return of(n + size - 1); }
};

// One layer's cache; strides in bytes.
struct KvCache {
  uint8_t *k, *v;
  uint8_t *k_scales, *v_scales;  // E4M3, else null
  uint32_t pages, heads, page, dim;
  uint64_t page_stride, head_stride, token_stride;
};

// ---- pages (urb_pages.hip) ----
struct AppendArgs {
  KvCache cache;
  const uint8_t *k, *v;  // strides in bytes
  uint64_t k_token, k_head, v_token, v_head;
  const int64_t* slots;
  uint32_t tokens;
};
void launch_append(const AppendArgs& a, bool rows_bf16, hipStream_t s);

// A row's first token, its length before, and the place on the stack of its first new page (-1: the row is
// not served).
struct __attribute__((aligned(16))) PlanRow {
  int32_t start, have, top, pad;
};
struct PlanArgs {
  uint32_t rows, tokens, pages, max_blocks;
  PageDivision page;
  uint64_t table_stride;
  const int32_t *lengths, *added;
  int32_t* tables;
  const int32_t *free_pages, *free_count;
  int32_t *lengths_out, *starts, *token_rows;
  int64_t *positions, *slots;
  int32_t* free_count_out;
  PlanRow* row_plans;  // workspace, [max_rows + 1]
  int* status;
};
void launch_plan(const PlanArgs& a, hipStream_t s);

constexpr int kForkCaches = 16;  // of a launch
constexpr int kForkWidth = 64, kForkRequests = 4096;
struct ForkCopy {
  uint32_t from, to, tokens;  // pages; 0 tokens: nothing
};
struct ForkArgs {
  uint32_t requests, width, pages, max_blocks;
  PageDivision page;
  uint64_t table_stride, table_out_stride;
  const int32_t *parents, *tables, *lengths;
  int32_t *tables_out, *lengths_out;
  int32_t* free_pages;
  const int32_t* free_count;
  int32_t* free_count_out;
  // workspace: lengths before [max_rows]; pages dropped and copies needed by each request; the dropped
  // pages of request r from r * width * max_blocks on; the free pages before
  int32_t *old_lengths, *drops, *copies, *dropped, *count;
  ForkCopy* page_copies;  // of each row
  int* status;
};
void launch_fork(const ForkArgs& a, hipStream_t s);
struct ForkCaches {
  KvCache c[kForkCaches];
};
// The copies of pages that the fork before it found, in n caches.
void launch_fork_copies(const ForkArgs& a, const ForkCaches& caches, uint32_t n, hipStream_t s);

// ---- attention (urb_attend.hip) ----
struct AttendArgs {
  KvCache cache;
  uint32_t rows, queries, q_heads, window, max_length;
  float scale;
  const uint8_t* q;
  uint8_t* out;
  uint64_t q_row, q_token, q_head, out_row, out_token, out_head;  // bytes
  const int32_t* tables;
  uint64_t table_stride;
  const int32_t* lengths;
  const float* sinks;
  float* lse;
  float* parts;  // attend_work_bytes
  int* status;
};
size_t attend_work_bytes(uint32_t dim, bool f8, bool rows_bf16);
void launch_attend(const AttendArgs& a, bool rows_bf16, hipStream_t s);

}  // namespace urb
