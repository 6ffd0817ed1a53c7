// urb_step.hpp -- host-side launch interface of the decoder-step kernels (include/urb_step.h).
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include <algorithm>

namespace urb {

// Status bits of the step contexts (urb_proj_ctx, urb_sampler).
constexpr int kStepNonFinite = 1;
constexpr int kStepArgument = 2;

// ---- norms of queries and keys with the rotation (urb_rotate.hip) ----
struct HeadRows {
  const void* in;
  void* out;
  const float* weight;
  uint64_t in_token, in_head, out_token, out_head;  // strides in values
};
struct RotateArgs {
  HeadRows q, k;
  int q_heads, heads;  // query heads; all heads
  int dim, rotary, interleaved;
  float offset;        // added to the weights: 1 for zero-centred ones
  float eps;
  const int64_t* positions;
  const float* inv_freq;
  uint32_t tokens;
};
void launch_rotate(const RotateArgs& a, bool bf16, hipStream_t s);

// ---- sampling (urb_sample.hip) ----
struct SampleArgs {
  const void* logits;
  uint64_t row_stride;  // values
  int vocab, rows;
  const float* temperature;
  const int32_t* top_k;
  const float* top_p;
  const float* min_p;
  const float* uniform;
  int32_t* ids;
  float* probs;
  int* status;
  void* work;  // sample_work_bytes(vocab, the most rows of a call)
};
// Rows per pass of a call (longer calls run in passes of this many).
constexpr int kSamplePass = 512;
size_t sample_work_bytes(int vocab, int rows);
void launch_sample(const SampleArgs& a, bool bf16, hipStream_t s);

// ---- projections with adapters (urb_project.hip) ----
// Ranks are kept in units of 8 in B and in 16-rank panels in A.
constexpr int kRankUnit = 8;
inline int rank_units(int rank) { return (rank + kRankUnit - 1) / kRankUnit; }
inline int rank_panels(int rank) { return (rank + 15) / 16; }

struct AdapterEntry {
  int rank;  // 0: empty slot
  float scale;
};

struct ProjArgs {
  int format;
  int rows, cols;
  const uint8_t* data;    // panel layout
  const uint8_t* scales;
  bool x_bf16, y_bf16;
  const void* x;
  uint64_t x_stride;
  void* y;
  uint64_t y_stride;
  int tokens;
  // adapters; ids NULL = none
  const int32_t* ids;
  int slots, max_rank;
  const AdapterEntry* table;
  const uint16_t* a;      // slot i at a + i * a_slot
  const uint16_t* b;
  size_t a_slot, b_slot;  // values
  void* work;             // proj_work_bytes
  int* status;
};
// The workspace of calls of up to max_tokens rows (of the geometry, types, slots and ranks in p).
size_t proj_work_bytes(const ProjArgs& p, int max_tokens);
void launch_project(const ProjArgs& a, hipStream_t s);
// Lays an adapter out in its slot and enters it in the table.
void launch_set_adapter(const uint16_t* a, const uint16_t* b, int rank, float scale, int rows,
                        int cols, uint16_t* slot_a, uint16_t* slot_b, AdapterEntry* entry,
                        int* flag, int* status, hipStream_t s);

}  // namespace urb
