// Host-side launchers of the sequence operators' kernels (sequence.hip): the causal convolution,
// the selective scan and the norm with rotation, forward and backward. Operands and results are
// those of include/rg_plan.h; a null result is not written. Sums over the batch and its positions
// leave partial rows, which the caller folds (`*_rows` says how many) in row order.
#pragma once
#include <hip/hip_runtime.h>

#include <cstdint>

#include "../../../include/rg_plan.h"

namespace rgk {

// A launch's threads have to stay below 2^32: `*_blocks` of 256 below this.
constexpr uint64_t SEQUENCE_BLOCKS = 1ull << 24;

struct ConvArgs {
  uint32_t batch, length, width, taps;
  bool silu;
  const void *x, *w, *bias, *state;
  const int32_t* lengths;
  void *y, *next;               // forward
  const void *dy, *carry;       // backward
  void *dx, *dstate, *dw_rows, *db_rows;
};
uint64_t conv_blocks(int dtype, const ConvArgs& a);
uint32_t conv_grad_rows(int dtype, const ConvArgs& a);
void causal_conv(hipStream_t s, int dtype, const ConvArgs& a);
void causal_conv_grad(hipStream_t s, int dtype, const ConvArgs& a);

struct ScanArgs {
  uint32_t batch, length, width, states, groups;
  uint32_t map_stride;          // rows of states from one position to the next, in b and in c
  bool softplus, logs;          // logs: `a` holds the rates' logarithms
  const void *x, *dt, *dt_bias, *a, *b, *c, *skip, *gate, *state;
  const int32_t* lengths;
  void *y, *last, *marks;       // forward; `marks` is read by the backward
  const void *dy, *carry;       // backward
  void *dx, *ddt, *dz, *dstate;
  // Partial rows: of b and c one per tile of a group's channels, each [batch, length, map_stride,
  // states]; of a ([width, states]), the skip and the dt bias ([width]) scan_rows of them.
  void *db_rows, *dc_rows, *da_rows, *dd_rows, *dt_bias_rows;
  void* workspace;              // scan_workspace bytes
  // Set by the launchers: tiles of positions a chunk, chunks a sequence and a block of the gradient,
  // and the chunks' ends and sums of steps.
  uint32_t chunk_tiles, chunks, split;
  void *ends, *totals;
};
uint64_t scan_workspace(int dtype, const ScanArgs& a);
uint64_t scan_blocks(int dtype, const ScanArgs& a);
uint32_t scan_rows(int dtype, const ScanArgs& a);
uint32_t scan_group_tiles(int dtype, const ScanArgs& a);
void selective_scan(hipStream_t s, int dtype, const ScanArgs& a);
void selective_scan_grad(hipStream_t s, int dtype, const ScanArgs& a);

constexpr int ROTARY_SECTIONS = 4;
struct RotaryArgs {
  uint32_t batch, length, heads, head, turn;
  uint32_t sections, last[ROTARY_SECTIONS];  // head past the end of each section
  double eps;
  bool normed, shared_positions, positions_from;
  const void *x, *gain;
  const int32_t* positions;
  const double2* turns;         // turns per position of each pair, as high and low parts
  void* y;
  const void* dy;               // backward
  void *dx, *dgain_rows;        // rows of [sections, head]
};
uint32_t rotary_grad_rows(int dtype, const RotaryArgs& a);
void rotary_norm(hipStream_t s, int dtype, const RotaryArgs& a);
void rotary_norm_grad(hipStream_t s, int dtype, const RotaryArgs& a);

}  // namespace rgk
