// Host-side launchers of the attention operators' kernels (attend.hip): attention with shaped
// scores, forward and backward, its form over a paged cache, and the joint norm of many tensors.
// Operands and results are those of include/rg_plan.h; a null result is not written.
#pragma once
#include <hip/hip_runtime.h>

#include <cstdint>

#include "../../../include/rg_plan.h"
#include "kernels.h"

namespace rgk {

// A launch's threads have to stay below 2^32: blocks of 256 below this.
constexpr uint64_t ATTEND_BLOCKS = 1ull << 24;

struct AttendArgs {
  uint32_t batch, length, heads, keys, head;
  bool causal, joined;
  double scale, cap;            // cap 0: none
  const void *q, *k, *v, *slopes;
  const int32_t *documents, *prefix, *lengths;
  void *y, *sums;               // forward; `sums` is read by the backward
  const void *y_in, *sums_in, *dy;
  void *dq, *dk, *dv;           // joined: dk and dv point into dq's rows
  void *dslopes_rows;           // attend_slope_rows of [heads], to be folded
  void *workspace;              // attend_workspace or paged_workspace bytes
  // Paged.
  uint32_t pages, page, table_pages;
  const void *k_pages, *v_pages;
  const int32_t *table, *first;
  void *k_out, *v_out;          // the pages with the new rows; may be k_pages and v_pages
  // Set by the launchers.
  int64_t q_row, k_row;         // values from one position to the next, of q and of k and v
  uint32_t tiles, splits, parts, join_width, join_step;
  void *partial;
  FastDiv page_div;
};
uint64_t attend_blocks(int dtype, const AttendArgs& a);
uint64_t attend_workspace(int dtype, const AttendArgs& a);
uint32_t attend_slope_rows(int dtype, const AttendArgs& a);
void attend(hipStream_t s, int dtype, const AttendArgs& a);
void attend_grad(hipStream_t s, int dtype, const AttendArgs& a);

uint64_t paged_blocks(int dtype, const AttendArgs& a);
uint64_t paged_workspace(int dtype, const AttendArgs& a);
void paged_attend(hipStream_t s, int dtype, const AttendArgs& a);

// The norm's tensors, NORM_TENSORS a launch: `first_block` is the block that begins each.
constexpr int NORM_TENSORS = 128;
struct NormTensors {
  const void* x[NORM_TENSORS];
  uint64_t n[NORM_TENSORS];
  uint32_t first_block[NORM_TENSORS];
  uint32_t count;
};
uint32_t norm_blocks(uint64_t n);  // x is 16 bytes aligned
// The blocks' sums of squares in `partial` (64 bits, from `first_partial` on), then their root.
void norm_squares(hipStream_t s, int dtype, const NormTensors& t, uint32_t blocks, double* partial);
void norm_root(hipStream_t s, int dtype, const double* partial, uint32_t blocks, void* out);

}  // namespace rgk
