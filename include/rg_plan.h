/* rg plan descriptor: the flat, C-ABI form of rg's `Plan` (reference src/plan.rs:75-164).
 *
 * A device backend receives a plan as one array of int64 words plus one byte blob holding the
 * constant tensors. The words encode, in order:
 *
 *   header     RG_PLAN_MAGIC, RG_PLAN_VERSION
 *   slots      n_slots, then per slot: dtype, capacity (elements), pinned (0/1)
 *              (plan.rs:151-154: `slots`, `pinned`)
 *   consts     n_consts, then per const: slot, n (elements), byte offset into the blob
 *              (plan.rs:155 `consts`; values are row-major, native-endian, dtype sizes 4/8/4)
 *   inputs     n_inputs, then per input: slot, n                (plan.rs:156-157)
 *   outputs    n_outputs, then per output: slot, n, rank, dims  (plan.rs:142-147, 158)
 *   steps      n_steps, then per step a tagged record:
 *     RG_STEP_INSTR  op, dtype, dst, n, mode, node,
 *                    rank, dims (output shape),
 *                    n_args, per arg: slot, rank, dims,
 *                    n_attr, attr words (op specific, below)   (plan.rs:127-140 `Instr`)
 *     RG_STEP_FUSED  dtype, n, regs, rank, dims,
 *                    n_in, per input: slot, kind, row_len, reg, rank, dims,
 *                    n_ops, per micro-op: op, reg, n_args, per arg: is_reg, index,
 *                    n_out, per output: reg, slot                (plan.rs:85-111 `Fused`)
 *     RG_STEP_ROWS   dtype, n, row_len, regs, rank, dims,
 *                    n_in, per input: slot, kind, row_len, reg, rank, dims,
 *                    n_ops, per micro-op: op, reg, aux, n_args, per arg: is_reg, index,
 *                    n_out, per output: reg, slot
 *                    A row group (no reference counterpart; device plans only): `dims` is
 *                    [rows..., row_len], and each row is computed independently. A register
 *                    holds either a whole row (element level) or one value per row (row level:
 *                    per-row inputs, reductions, and ops on row-level values only). RG_OP_REDUCE
 *                    micro-ops reduce an element-level register over the row, `aux` being the
 *                    rg_reduce_kind. Inputs are read per element like a fused group's; a
 *                    Broadcast input whose last dimension is 1 is row level. Outputs of
 *                    row-level registers hold one value per row. An RG_OP_REDUCE whose `aux`
 *                    has RG_ROWS_COLUMN added reduces an element-level register over all the
 *                    rows instead (every axis but the last): its register is column level, one
 *                    value per position of the row, read by no other micro-op, and its outputs
 *                    hold row_len values.
 *     RG_STEP_ATTN   dtype, backward (0/1), bh, heads, tq, tk, hd, div (f64 bits), fill (f64 bits),
 *                    mask_slot (-1: none), mask strides (4 words), mask_bits_slot, build_bits (0/1),
 *                    stats_slot,
 *                    n_in, per in: slot, offset, sb, sh, st,  n_out, per out: the same,  node
 *                    Fused attention (no reference counterpart; device plans only) over bh
 *                    independent problems b * heads + h; row t, column d of an operand lies at
 *                    offset + b * sb + h * sh + t * st + d in its slot (so operands may be
 *                    slices and transposes of other values, and outputs may share a slot):
 *                      forward   in q, k, v        out O = softmax(where(mask, q k^T / div, fill)) v
 *                      backward  in q, k, v, O, dO out dq, dk, dv (the gradients of O's graph)
 *                    The softmax is over keys; the mask (f32, nonzero = visible) is read at
 *                    b * s0 + h * s1 + q * s2 + k * s3 for problem b * heads + h. The stats
 *                    slot holds 3 * bh * tq words of per-query statistics (written by the
 *                    forward, read by the backward). With a mask, mask_bits_slot holds
 *                    slices * (2 * tq * tk / 32 + tq) words of packed mask bits, slices being
 *                    (s0 ? bh / heads : 1) * (s1 ? heads : 1); the step with build_bits set
 *                    packs them, and later steps reading the same mask reuse them. Planned
 *                    only for hd in {16, 32, 64} and tq, tk multiples of 32 up to
 *                    RG_ATTN_MAX_T.
 *
 * Operands: MATMUL and MATMUL_T (f32, device plans) may carry a third argument, a vector of
 * the product's column count added to every row of the finished product (a bias add folded
 * into the product; no reference counterpart).
 *
 * Attribute words per op:
 *   MATMUL_T       ta, tb
 *   REDUCE         kind, keepdims, n_axes, axes...
 *   TRANSPOSE      perm...
 *   BROADCAST_TO   shape...            RESHAPE  shape...
 *   SLICE          rank, starts..., stops...
 *   PAD            rank, starts..., shape...
 *   CAST           target dtype
 *   TAKE           axis                TAKE_GRAD  axis, shape...
 *   TAKE_ALONG_GRAD shape...           CONCAT     axis
 *   RAND_UNIFORM / RAND_NORMAL  dtype, shape...
 *   KEY_SPLIT      n                   ARG_TOP_K  k          CUMSUM reverse
 *   SCAN           n_carry, n_x, length, reverse, RESULTS, BODIES
 *   WHILE          n_carry, max_iterations, RESULTS, BODIES
 *   COND           RESULTS, BODIES
 *     RESULTS      n_results, per result the program reads: result index, slot
 *     BODIES       n_bodies, per body: n_words, then a whole plan descriptor (header included)
 *                  whose constants lie in the same blob (scan: body; while: condition, body;
 *                  cond: then, else)
 *   CAUSAL_CONV, CAUSAL_CONV_GRAD, SELECTIVE_SCAN, SELECTIVE_SCAN_GRAD, ROTARY_NORM,
 *   ROTARY_NORM_GRAD, ATTENTION, ATTENTION_GRAD, PAGED_ATTENTION, JOINT_NORM
 *                  flags, rotary dims, base (f64 bits), eps (f64 bits), n_sections, sections...,
 *                  n_results, per result the program reads: result index, slot
 *   Sequence operators (no reference counterpart; `sequence_of` says which operands follow which
 *   flags, and their shapes). ROTARY_NORM writes `dst`; the others' `dst` is -1.
 *     CAUSAL_CONV  in x[B,T,D], w[K,D] (, bias[D]) (, state[B,K-1,D]) (, lengths[B])
 *                  out 0: y[t] = act(bias + sum_k w[k] past[t + k]), past = state (zeros without
 *                  one) then x; 1: the K - 1 rows of past that end the sequence
 *       _GRAD      in the same, dy (, d of result 1); out dx, dw, dbias, dstate
 *     SELECTIVE_SCAN in x, dt[B,T,D], a[D,N], b, c[B,T,G,N] (, d[D]) (, z[B,T,D]) (, state[B,D,N])
 *                  (, lengths[B]) (, dt bias[D], added to dt first) (with RG_SCAN_JOINED one
 *                  b[B,T,2 G,N], b's groups then c's, and no c; with RG_SCAN_LOG a holds log(-a));
 *                  h[t] = exp(dt[t] a) h[t-1] + dt[t] x[t] b[t];
 *                  out 0: (c[t] . h[t] + d x[t]) silu(z[t]); 1: the last h; 2: marks, h before
 *                  positions 0, RG_SCAN_MARK, 2 RG_SCAN_MARK, ..., for the gradient alone
 *       _GRAD      in the same, marks, dy (, d of result 1); out dx, ddt, da, db, dc, dd, dz, dstate,
 *                  d of the dt bias
 *     ROTARY_NORM  in x[B,T,H,hd], positions[T], [B,T] or [B,1] (the first of each sequence)
 *                  (, gain[S,hd]); out x with the heads of
 *                  section s divided by their root mean square and scaled by gain[s], and their
 *                  pairs (i, i + R / 2), i < R / 2, turned by position * base^(-2 i / R)
 *       _GRAD      in the same, dy; out dx, dgain
 *     ATTENTION    in q[B,T,H,hd], k, v[B,T,G,hd] (with RG_ATTEND_JOINED one x[B,T,H + 2 G,hd], the
 *                  heads of q, k and v in order) (, slopes[H]) (, documents[B,T]) (, prefix[B])
 *                  (, lengths[B]); base is the scale, eps the cap (0: none), sections H, G;
 *                  s = cap tanh(scale q.k / cap) - slope |i - j|; key j is seen by query i when
 *                  (j <= i, or not RG_ATTEND_CAUSAL, or j < prefix) and both have the same document,
 *                  not negative; query head h reads head h G / H of k and v;
 *                  out 0: y[B,T,H,hd], the softmax of s over the keys seen, times v (0 where none is);
 *                  1: for the gradient alone, [2,B,H,T]: what scores to base 2 were lowered by before
 *                  their powers of two were summed, and one over that sum; the dtype's largest value
 *                  and 0 where no key is seen
 *       _GRAD      in the same, y, result 1, dy; out dq (joined: dx), dk, dv, dslopes
 *     PAGED_ATTENTION in q, k, v or x as above, k and v pages[P,page,G,hd], table[B,N], first[B]
 *                  (, slopes[H]) (, lengths[B]); position p of sequence b lies in row p % page of
 *                  page table[b, p / page]; the T new positions follow the first[b] that the pages
 *                  hold, and see those and each other in causal order; out y and the pages with the
 *                  new rows of k and v. Positions whose page is not one of the P are not there: not
 *                  read, not written
 *     JOINT_NORM   in tensors; out 0: the square root of the sum of all their squares
 *   With lengths, positions from lengths[b] on (clamped to 0..T) are outside sequence b: their
 *   results and gradients are 0, their inputs are not read into any other value.
 *   Control flow (plan.rs:737-831): the step's `dst` is -1 and its results go to the listed
 *   slots. Scan runs its body `length` times (from the last position when `reverse`) over
 *   inputs (carries, one slice of each x, captures); its results by index are the final
 *   carries, the ys stacked along a new leading axis, then the carries as they were before each
 *   step, stacked. While runs its condition and, while that is nonzero and fewer than
 *   max_iterations steps ran, its body over (carries, captures); results are the final carries,
 *   then the step count (int32). Cond runs `then` when its first argument is nonzero, else
 *   `else`, over the remaining arguments; results are that body's outputs. A body's carry
 *   results are written back to its carry inputs after every step, all read before any is
 *   written.
 *
 * Slot buffers hold at least `capacity` elements (at least 4 bytes) and start zeroed; a value
 * is the row-major prefix of `n` elements of its slot.
 */
#ifndef RG_PLAN_H
#define RG_PLAN_H

#include <stddef.h>
#include <stdint.h>

#define RG_PLAN_MAGIC 0x4c50475244ll /* "DRGPL" */
#define RG_PLAN_VERSION 1

enum rg_dtype { RG_F32 = 0, RG_F64 = 1, RG_I32 = 2 };

/* Operation codes: the variants of `Op` (reference src/graph.rs:47-114) that can reach a plan. */
enum rg_op {
  RG_OP_INPUT = 0, RG_OP_CONST, RG_OP_NEG, RG_OP_EXP, RG_OP_LOG, RG_OP_SQRT, RG_OP_SIN, RG_OP_COS,
  RG_OP_TANH, RG_OP_ABS, RG_OP_SIGN, RG_OP_ADD, RG_OP_SUB, RG_OP_MUL, RG_OP_DIV, RG_OP_POW,
  RG_OP_MAX, RG_OP_MIN, RG_OP_GT, RG_OP_GE, RG_OP_WHERE, RG_OP_MATMUL, RG_OP_MATMUL_T,
  RG_OP_REDUCE, RG_OP_RESHAPE, RG_OP_TRANSPOSE, RG_OP_BROADCAST_TO, RG_OP_SLICE, RG_OP_PAD,
  RG_OP_CAST, RG_OP_STOP_GRADIENT, RG_OP_FLOOR, RG_OP_TAKE, RG_OP_TAKE_ALONG, RG_OP_TAKE_GRAD,
  RG_OP_TAKE_ALONG_GRAD, RG_OP_CONCAT, RG_OP_ARGMAX, RG_OP_RAND_UNIFORM, RG_OP_RAND_NORMAL,
  RG_OP_KEY_SPLIT, RG_OP_ARG_TOP_K, RG_OP_CUMSUM, RG_OP_SCAN, RG_OP_WHILE, RG_OP_COND,
  RG_OP_OUTPUT, RG_OP_PLACEHOLDER, RG_OP_CUSTOM, RG_OP_CAUSAL_CONV, RG_OP_CAUSAL_CONV_GRAD,
  RG_OP_SELECTIVE_SCAN, RG_OP_SELECTIVE_SCAN_GRAD, RG_OP_ROTARY_NORM, RG_OP_ROTARY_NORM_GRAD,
  RG_OP_ATTENTION, RG_OP_ATTENTION_GRAD, RG_OP_PAGED_ATTENTION, RG_OP_JOINT_NORM,
  RG_OP_COUNT
};

/* Flags of the sequence operators: which optional operands are present, and the variants. */
enum rg_conv_flags { RG_CONV_BIAS = 1, RG_CONV_STATE = 2, RG_CONV_LENGTHS = 4, RG_CONV_SILU = 8, RG_CONV_CARRY = 16 };
enum rg_scan_flags {
  RG_SCAN_SKIP = 1, RG_SCAN_GATE = 2, RG_SCAN_STATE = 4, RG_SCAN_LENGTHS = 8, RG_SCAN_SOFTPLUS = 16, RG_SCAN_CARRY = 32,
  RG_SCAN_JOINED = 64, /* b holds b and c: [B,T,2 G,N], and c is no operand */
  RG_SCAN_BIAS = 128, RG_SCAN_LOG = 256 /* a holds the rates' logarithms: the rates are -e^a */
};
enum rg_rotary_flags { RG_ROTARY_GAIN = 1 };
enum rg_attend_flags {
  RG_ATTEND_JOINED = 1, RG_ATTEND_SLOPES = 2, RG_ATTEND_DOCUMENTS = 4, RG_ATTEND_PREFIX = 8, RG_ATTEND_LENGTHS = 16, RG_ATTEND_CAUSAL = 32
};
/* The longest head of an attention operator. */
#define RG_ATTEND_MAX_HEAD 256
/* Taps of a causal convolution, states of a selective scan, and the length of a head. */
#define RG_CONV_MAX_TAPS 8
#define RG_SCAN_MAX_STATES 64
#define RG_ROTARY_MAX_HEAD 256
/* A selective scan keeps its state before every RG_SCAN_MARK-th position for its gradient. */
#define RG_SCAN_MARK 16

enum rg_reduce_kind { RG_REDUCE_SUM = 0, RG_REDUCE_MAX = 1, RG_REDUCE_MIN = 2 };
/* Added to a row group's RG_OP_REDUCE `aux`: the reduction runs over the rows (a column reduction). */
#define RG_ROWS_COLUMN 4
/* Input kinds of a fused group (plan.rs:75-83). */
enum rg_arg_kind { RG_ARG_FULL = 0, RG_ARG_SPLAT = 1, RG_ARG_ROW = 2, RG_ARG_BROADCAST = 3 };
/* Binary broadcast modes of a single elementwise instruction (plan.rs:119-125). */
enum rg_mode { RG_MODE_SAME = 0, RG_MODE_ASCALAR = 1, RG_MODE_BSCALAR = 2, RG_MODE_GENERAL = 3 };
enum rg_step_kind { RG_STEP_INSTR = 0, RG_STEP_FUSED = 1, RG_STEP_ROWS = 2, RG_STEP_ATTN = 3 };
/* Longest query or key sequence of a fused attention step. */
#define RG_ATTN_MAX_T 256

#ifdef __cplusplus
#include <algorithm>
#include <cstring>
#include <stdexcept>
#include <string>
#include <vector>

namespace rgplan {

struct Arg {
  int64_t slot;
  std::vector<int64_t> shape;
};

/* The attributes of a sequence operator, before its results. */
struct SequenceAttr {
  int64_t flags = 0, turn = 0;
  double base = 0, eps = 0;
  std::vector<int64_t> sections;
};

struct Instr {
  int32_t op, dtype;
  int64_t dst, n, mode, node;
  std::vector<int64_t> shape;
  std::vector<Arg> args;
  std::vector<int64_t> attr;
  SequenceAttr sequence;                         /* sequence operators */
  std::vector<std::pair<int64_t, int64_t>> outs; /* theirs: (result index, slot) */
};

inline bool is_sequence(int32_t op) { return op >= RG_OP_CAUSAL_CONV && op <= RG_OP_JOINT_NORM; }
/* Those whose results are numbered; ROTARY_NORM has one, in `dst`. */
inline bool is_multi_result(int32_t op) { return is_sequence(op) && op != RG_OP_ROTARY_NORM; }

/* A sequence operator's sizes, where its operands are among the arguments (-1: absent), and the
 * shapes of its results. The one definition that the engine, the backend and the parser share. */
struct Sequence {
  int64_t batch = 0, length = 0, width = 0, taps = 0, states = 0, groups = 0, heads = 0, head = 0, used = 0, keys = 0, pages = 0, page = 0,
          table_pages = 0;
  int x = 0, w = -1, bias = -1, dt = -1, a = -1, b = -1, c = -1, skip = -1, gate = -1, state = -1, lengths = -1, marks = -1, dy = -1,
      carry = -1, positions = -1, gain = -1, dt_bias = -1, k = -1, v = -1, slopes = -1, documents = -1, prefix = -1, k_pages = -1, v_pages = -1,
      table = -1, first = -1, y = -1, sums = -1;
  bool shared_positions = false; /* positions of [length], the same for every sequence */
  bool positions_from = false;   /* positions of [batch, 1], the first of each sequence */
  std::vector<std::vector<int64_t>> results;
  std::string wrong; /* empty when the operands fit */
  /* Operands of whole numbers (int32). */
  bool is_index(int operand) const {
    for (int at : {lengths, positions, documents, prefix, table, first})
      if (at >= 0 && at == operand) return true;
    return false;
  }
};

/* Attention and its paged form, whose sections are the heads of q and of k and v. */
inline Sequence attention_of(int32_t op, const SequenceAttr& at, const std::vector<std::vector<int64_t>>& s) {
  Sequence q;
  auto fail = [&](const char* what) {
    if (q.wrong.empty()) q.wrong = what;
  };
  const int64_t f = at.flags;
  const bool joined = (f & RG_ATTEND_JOINED) != 0, paged = op == RG_OP_PAGED_ATTENTION, grad = op == RG_OP_ATTENTION_GRAD;
  int next = 1;
  auto take = [&](bool present) { return present ? next++ : -1; };
  q.k = take(!joined);
  q.v = take(!joined);
  q.k_pages = take(paged);
  q.v_pages = take(paged);
  q.table = take(paged);
  q.first = take(paged);
  q.slopes = take((f & RG_ATTEND_SLOPES) != 0);
  q.documents = take((f & RG_ATTEND_DOCUMENTS) != 0);
  q.prefix = take((f & RG_ATTEND_PREFIX) != 0);
  q.lengths = take((f & RG_ATTEND_LENGTHS) != 0);
  q.y = take(grad);
  q.sums = take(grad);
  q.dy = take(grad);
  if ((int)s.size() != next || (paged && (f & (RG_ATTEND_DOCUMENTS | RG_ATTEND_PREFIX)))) {
    fail("operand_count_does_not_match_the_flags");
    return q;
  }
  for (const auto& v : s)
    for (int64_t d : v)
      if (d < 1) {
        fail("empty_operand");
        return q;
      }
  if (at.sections.size() != 2 || at.sections[0] < 1 || at.sections[1] < 1 || at.sections[0] % at.sections[1] != 0) {
    fail("heads_must_be_a_multiple_of_the_key_heads");
    return q;
  }
  q.heads = at.sections[0];
  q.keys = at.sections[1];
  const std::vector<int64_t>& x = s[0];
  if (x.size() != 4 || x[2] != q.heads + (joined ? 2 * q.keys : 0)) {
    fail(joined ? "x_must_be_batch_length_heads_and_twice_the_key_heads_head" : "q_must_be_batch_length_heads_head");
    return q;
  }
  q.batch = x[0];
  q.length = x[1];
  q.head = x[3];
  if (q.head > RG_ATTEND_MAX_HEAD) fail("head_must_be_at_most_256");
  auto dims = [&](int k, const std::vector<int64_t>& want, const char* what) {
    if (k >= 0 && s[(size_t)k] != want) fail(what);
  };
  const std::vector<int64_t> keys = {q.batch, q.length, q.keys, q.head}, out = {q.batch, q.length, q.heads, q.head};
  const std::vector<int64_t> sums = {2, q.batch, q.heads, q.length};
  dims(q.k, keys, "k_must_be_batch_length_key_heads_head");
  dims(q.v, keys, "v_must_be_batch_length_key_heads_head");
  dims(q.slopes, {q.heads}, "slopes_must_be_one_per_head");
  dims(q.documents, {q.batch, q.length}, "documents_must_be_batch_length");
  dims(q.prefix, {q.batch}, "prefix_must_be_one_per_sequence");
  dims(q.lengths, {q.batch}, "lengths_must_be_one_per_sequence");
  dims(q.first, {q.batch}, "first_must_be_one_per_sequence");
  dims(q.y, out, "result_shape");
  dims(q.sums, sums, "sums_shape");
  dims(q.dy, out, "cotangent_shape_differs_from_the_result");
  if (paged) {
    const std::vector<int64_t>&p = s[(size_t)q.k_pages], &t = s[(size_t)q.table];
    if (p.size() != 4 || p[2] != q.keys || p[3] != q.head) {
      fail("pages_must_be_pages_page_key_heads_head");
      return q;
    }
    dims(q.v_pages, p, "pages_of_k_and_v_differ");
    if (t.size() != 2 || t[0] != q.batch) {
      fail("table_must_be_batch_by_pages");
      return q;
    }
    q.pages = p[0];
    q.page = p[1];
    q.table_pages = t[1];
    if (q.page > (1ll << 30) / t[1] || q.length > (1ll << 30)) fail("more_than_2_to_the_30_positions");
    q.results = {out, p, p};
  } else if (grad) {
    if (joined) q.results = {x, keys, keys, {q.heads}};
    else q.results = {out, keys, keys, {q.heads}};
  } else {
    if (q.length > (1ll << 30)) fail("more_than_2_to_the_30_positions");
    q.results = {out, sums};
  }
  return q;
}

inline Sequence sequence_of(int32_t op, const SequenceAttr& at, const std::vector<std::vector<int64_t>>& s) {
  Sequence q;
  auto fail = [&](const char* what) {
    if (q.wrong.empty()) q.wrong = what;
  };
  auto dims = [&](int k, const std::vector<int64_t>& want, const char* what) {
    if (s[(size_t)k] != want) fail(what);
  };
  if (op == RG_OP_ATTENTION || op == RG_OP_ATTENTION_GRAD || op == RG_OP_PAGED_ATTENTION) return attention_of(op, at, s);
  if (op == RG_OP_JOINT_NORM) {
    if (s.empty()) fail("operand_count_does_not_match_the_flags");
    for (const auto& v : s)
      for (int64_t d : v)
        if (d < 1) fail("empty_operand");
    q.results = {{}};
    return q;
  }
  const int64_t f = at.flags;
  int next = 1;
  auto take = [&](bool present) { return present ? next++ : -1; };
  const bool conv = op == RG_OP_CAUSAL_CONV || op == RG_OP_CAUSAL_CONV_GRAD, rotary = op == RG_OP_ROTARY_NORM || op == RG_OP_ROTARY_NORM_GRAD;
  const bool grad = op == RG_OP_CAUSAL_CONV_GRAD || op == RG_OP_SELECTIVE_SCAN_GRAD || op == RG_OP_ROTARY_NORM_GRAD;
  if (conv) {
    q.w = take(true);
    q.bias = take(f & RG_CONV_BIAS);
    q.state = take(f & RG_CONV_STATE);
    q.lengths = take(f & RG_CONV_LENGTHS);
    q.dy = take(grad);
    q.carry = take(grad && (f & RG_CONV_CARRY));
  } else if (rotary) {
    q.positions = take(true);
    q.gain = take(f & RG_ROTARY_GAIN);
    q.dy = take(grad);
  } else {
    q.dt = take(true);
    q.a = take(true);
    q.b = take(true);
    q.c = take(!(f & RG_SCAN_JOINED));
    q.skip = take(f & RG_SCAN_SKIP);
    q.gate = take(f & RG_SCAN_GATE);
    q.state = take(f & RG_SCAN_STATE);
    q.lengths = take(f & RG_SCAN_LENGTHS);
    q.dt_bias = take(f & RG_SCAN_BIAS);
    q.marks = take(grad);
    q.dy = take(grad);
    q.carry = take(grad && (f & RG_SCAN_CARRY));
  }
  if ((int)s.size() != next) {
    fail("operand_count_does_not_match_the_flags");
    return q;
  }
  const std::vector<int64_t>& x = s[0];
  if (x.size() != (rotary ? 4u : 3u)) {
    fail(rotary ? "x_must_be_batch_length_heads_head" : "x_must_be_batch_length_width");
    return q;
  }
  for (const auto& v : s)
    for (int64_t d : v)
      if (d < 1) {
        fail("empty_operand");
        return q;
      }
  q.batch = x[0];
  q.length = x[1];
  q.width = x[2];
  if (q.dy >= 0) dims(q.dy, x, "cotangent_shape_differs_from_x");
  if (q.lengths >= 0) dims(q.lengths, {q.batch}, "lengths_must_be_one_per_sequence");
  if (conv) {
    const std::vector<int64_t>& w = s[(size_t)q.w];
    if (w.size() != 2 || w[1] != q.width) {
      fail("weights_must_be_taps_width");
      return q;
    }
    q.taps = w[0];
    if (q.taps < 2 || q.taps > RG_CONV_MAX_TAPS) fail("taps_must_be_two_to_eight");
    const std::vector<int64_t> past = {q.batch, q.taps - 1, q.width};
    if (q.bias >= 0) dims(q.bias, {q.width}, "bias_must_be_width");
    if (q.state >= 0) dims(q.state, past, "state_must_be_batch_taps_less_one_width");
    if (q.carry >= 0) dims(q.carry, past, "state_cotangent_shape");
    if (grad) q.results = {x, w, {q.width}, past};
    else q.results = {x, past};
  } else if (rotary) {
    q.heads = x[2];
    q.head = x[3];
    q.width = q.heads * q.head;
    for (int64_t n : at.sections) {
      if (n < 1) fail("sections_must_be_positive");
      q.used += n;
    }
    if (at.sections.empty() || at.sections.size() > 4 || q.used > q.heads || q.used < 1) fail("sections_must_be_one_to_four_within_the_heads");
    if (q.head % 2 != 0 || q.head > RG_ROTARY_MAX_HEAD) fail("head_must_be_even_and_at_most_256");
    if (at.turn < 0 || at.turn % 2 != 0 || at.turn > q.head) fail("rotary_dims_must_be_even_and_within_the_head");
    const std::vector<int64_t>& p = s[(size_t)q.positions];
    q.shared_positions = p.size() == 1;
    q.positions_from = p.size() == 2 && p[1] == 1;
    if (q.shared_positions) dims(q.positions, {q.length}, "positions_must_be_length_or_batch_length");
    else if (q.positions_from) dims(q.positions, {q.batch, 1}, "positions_must_be_length_or_batch_length");
    else dims(q.positions, {q.batch, q.length}, "positions_must_be_length_or_batch_length");
    const std::vector<int64_t> gain = {(int64_t)at.sections.size(), q.head};
    if (q.gain >= 0) dims(q.gain, gain, "gain_must_be_sections_head");
    q.results = {x};
    if (grad) q.results.push_back(gain);
  } else {
    const std::vector<int64_t>&a = s[(size_t)q.a], &b = s[(size_t)q.b];
    if (a.size() != 2 || a[0] != q.width || a[1] > RG_SCAN_MAX_STATES) {
      fail("a_must_be_width_by_at_most_64_states");
      return q;
    }
    q.states = a[1];
    const int64_t maps = q.c < 0 ? 2 : 1;
    if (b.size() != 4 || b[0] != q.batch || b[1] != q.length || b[3] != q.states || b[2] % maps != 0 || q.width % (b[2] / maps) != 0) {
      fail("b_must_be_batch_length_groups_states_with_groups_dividing_the_width");
      return q;
    }
    q.groups = b[2] / maps;
    const std::vector<int64_t> state = {q.batch, q.width, q.states};
    const std::vector<int64_t> marks = {q.batch, (q.length + RG_SCAN_MARK - 1) / RG_SCAN_MARK, q.width, q.states};
    dims(q.dt, x, "dt_shape_differs_from_x");
    if (q.c >= 0) dims(q.c, b, "c_shape_differs_from_b");
    if (q.skip >= 0) dims(q.skip, {q.width}, "d_must_be_width");
    if (q.gate >= 0) dims(q.gate, x, "z_shape_differs_from_x");
    if (q.dt_bias >= 0) dims(q.dt_bias, {q.width}, "dt_bias_must_be_width");
    if (q.state >= 0) dims(q.state, state, "state_must_be_batch_width_states");
    if (q.carry >= 0) dims(q.carry, state, "state_cotangent_shape");
    if (q.marks >= 0) dims(q.marks, marks, "marks_shape");
    if (grad) q.results = {x, x, a, b, b, {q.width}, x, state, {q.width}};
    else q.results = {x, state, marks};
  }
  return q;
}

inline Sequence sequence_of(const Instr& in) {
  std::vector<std::vector<int64_t>> shapes;
  for (const Arg& a : in.args) shapes.push_back(a.shape);
  return sequence_of(in.op, in.sequence, shapes);
}

struct FusedInput {
  int64_t slot, kind, row_len, reg;
  std::vector<int64_t> shape;
};

struct MicroOp {
  int32_t op;
  int64_t reg;
  int64_t aux = 0; /* RG_STEP_ROWS: the reduce kind of an RG_OP_REDUCE */
  std::vector<std::pair<int64_t, int64_t>> args; /* (is_reg, index) */
};

/* RG_STEP_FUSED, or RG_STEP_ROWS when row_len > 0. */
struct Fused {
  int32_t dtype;
  int64_t n, regs;
  int64_t row_len = 0;
  std::vector<int64_t> shape;
  std::vector<FusedInput> inputs;
  std::vector<MicroOp> ops;
  std::vector<std::pair<int64_t, int64_t>> outputs; /* (reg, slot) */
};

/* RG_STEP_ATTN */
struct AttnView {
  int64_t slot, offset, sb, sh, st;
};
struct Attn {
  int32_t dtype;
  bool backward;
  int64_t bh, heads, tq, tk, hd;
  double div, fill;
  int64_t mask_slot;
  int64_t mask_strides[4];
  int64_t mask_bits_slot;
  bool build_bits;
  int64_t stats_slot;
  std::vector<AttnView> in, out;
  int64_t node;
};

struct Step {
  int32_t kind;
  Instr instr;
  Fused fused;
  Attn attn;
};

struct Slot {
  int32_t dtype;
  int64_t cap;
  bool pinned;
};

struct Const {
  int64_t slot, n, offset;
};

struct Output {
  int64_t slot, n;
  std::vector<int64_t> shape;
};

struct Plan {
  std::vector<Slot> slots;
  std::vector<Const> consts;
  std::vector<std::pair<int64_t, int64_t>> inputs; /* (slot, n) */
  std::vector<Output> outputs;
  std::vector<Step> steps;
};

inline int64_t dtype_size(int32_t d) { return d == RG_F64 ? 8 : 4; }

/* Refuses a plan whose steps name slots it does not have or reach beyond a slot's capacity:
 * constants, inputs and outputs within their slots; every instruction argument's elements and
 * its `n` outputs within their slots; fused inputs by their read extent (Full n, Row row_len,
 * Splat 1, Broadcast the source size) and outputs by what they write; attention views by the
 * largest offset they touch, the statistics and the mask tables by their sizes. Called by
 * `parse`, so a backend never launches a kernel on a plan that would index past its buffers. */
inline void check_refs(const Plan& pl) {
  const int64_t ns = (int64_t)pl.slots.size();
  auto fail = [](const std::string& what) { throw std::runtime_error("plan descriptor: " + what); };
  auto prod_of = [](const std::vector<int64_t>& v) {
    int64_t n = 1;
    for (int64_t d : v) {
      if (d < 0) return (int64_t)-1;
      n *= d;
    }
    return n;
  };
  auto fits = [&](int64_t slot, int64_t n, const char* what) {
    if (slot < 0 || slot >= ns) fail(std::string(what) + " names slot " + std::to_string(slot) + " of " + std::to_string(ns));
    if (n < 0 || n > pl.slots[(size_t)slot].cap)
      fail(std::string(what) + " needs " + std::to_string(n) + " values of slot " + std::to_string(slot) + ", which holds " +
           std::to_string(pl.slots[(size_t)slot].cap));
  };
  for (const Slot& s : pl.slots)
    if ((s.dtype != RG_F32 && s.dtype != RG_F64 && s.dtype != RG_I32) || s.cap < 0) fail("a slot has a bad dtype or capacity");
  for (const Const& c : pl.consts) {
    fits(c.slot, c.n, "a constant");
    if (c.offset < 0) fail("a constant has a negative offset");
  }
  for (const auto& in : pl.inputs) fits(in.first, in.second, "an input");
  for (const Output& o : pl.outputs) {
    fits(o.slot, o.n, "an output");
    if (prod_of(o.shape) != o.n) fail("an output's shape does not hold its n values");
  }
  for (size_t k = 0; k < pl.steps.size(); k++) {
    const Step& st = pl.steps[k];
    const std::string at = "step " + std::to_string(k);
    if (st.kind == RG_STEP_INSTR) {
      const Instr& in = st.instr;
      if (in.dst != -1) fits(in.dst, in.n, (at + " output").c_str());
      for (const Arg& a : in.args)
        if (a.slot != -1) fits(a.slot, prod_of(a.shape), (at + " argument").c_str());
      if (is_sequence(in.op)) {
        const Sequence q = sequence_of(in);
        if (!q.wrong.empty()) fail(at + ": " + q.wrong);
        if (in.dtype != RG_F32 && in.dtype != RG_F64) fail(at + " is not of a floating-point dtype");
        for (size_t j = 0; j < in.args.size(); j++) {
          const int32_t want = q.is_index((int)j) ? (int32_t)RG_I32 : in.dtype;
          if (in.args[j].slot < 0 || pl.slots[(size_t)in.args[j].slot].dtype != want) fail(at + " has an argument of another dtype");
        }
        if (!is_multi_result(in.op) && (in.dst < 0 || in.n != prod_of(q.results[0]) || pl.slots[(size_t)in.dst].dtype != in.dtype))
          fail(at + " has a result of another size or dtype");
        for (const auto& o : in.outs) {
          if (o.first < 0 || (size_t)o.first >= q.results.size()) fail(at + " names a result it does not have");
          for (const auto& other : in.outs)
            if (&other != &o && other.first == o.first) fail(at + " names a result twice");
          fits(o.second, prod_of(q.results[(size_t)o.first]), (at + " result").c_str());
          if (pl.slots[(size_t)o.second].dtype != in.dtype) fail(at + " has a result of another dtype");
        }
      }
    } else if (st.kind == RG_STEP_FUSED || st.kind == RG_STEP_ROWS) {
      const Fused& f = st.fused;
      const int64_t rows = f.row_len > 0 ? f.n / f.row_len : 0;
      for (const FusedInput& fi : f.inputs) {
        int64_t extent = fi.kind == RG_ARG_FULL ? f.n : fi.kind == RG_ARG_ROW ? fi.row_len : fi.kind == RG_ARG_SPLAT ? 1 : prod_of(fi.shape);
        if (fi.kind < RG_ARG_FULL || fi.kind > RG_ARG_BROADCAST) fail(at + " has an input of unknown kind");
        fits(fi.slot, extent, (at + " input").c_str());
      }
      for (const auto& o : f.outputs)
        fits(o.second, f.row_len > 0 ? std::min(rows, f.row_len) : f.n, (at + " output").c_str());
    } else if (st.kind == RG_STEP_ATTN) {
      const Attn& a = st.attn;
      const int64_t batch = a.bh / a.heads;
      auto view = [&](const AttnView& v, int64_t t, const char* what) {
        if (v.offset < 0 || v.sb < 0 || v.sh < 0 || v.st < 0 || t <= 0 || a.hd <= 0) fail(at + " has a bad " + what + " view");
        fits(v.slot, v.offset + (batch - 1) * v.sb + (a.heads - 1) * v.sh + (t - 1) * v.st + a.hd, (at + " " + what).c_str());
      };
      const int64_t in_t[5] = {a.tq, a.tk, a.tk, a.tq, a.tq}, out_t[3] = {a.tq, a.tk, a.tk};
      for (size_t j = 0; j < a.in.size(); j++) view(a.in[j], in_t[j], "operand");
      for (size_t j = 0; j < a.out.size(); j++) view(a.out[j], a.backward ? out_t[j] : a.tq, "result");
      fits(a.stats_slot, 3 * a.bh * a.tq, (at + " statistics").c_str());
      if (a.mask_slot != -1) {
        const int64_t* m = a.mask_strides;
        if (m[0] < 0 || m[1] < 0 || m[2] < 0 || m[3] < 0) fail(at + " has a negative mask stride");
        fits(a.mask_slot, (batch - 1) * m[0] + (a.heads - 1) * m[1] + (a.tq - 1) * m[2] + (a.tk - 1) * m[3] + 1, (at + " mask").c_str());
        const int64_t slices = (m[0] ? batch : 1) * (m[1] ? a.heads : 1);
        fits(a.mask_bits_slot, slices * (2 * a.tq * a.tk / 32 + a.tq), (at + " mask bits").c_str());
      }
    }
  }
}

/* Parses the word array; throws std::runtime_error on a malformed descriptor. */
inline Plan parse(const int64_t* w, size_t nw) {
  size_t p = 0;
  auto next = [&]() -> int64_t {
    if (p >= nw) throw std::runtime_error("plan descriptor truncated");
    return w[p++];
  };
  auto vec = [&](int64_t n) {
    if (n < 0 || (size_t)n > nw) throw std::runtime_error("plan descriptor has a bad length");
    std::vector<int64_t> v((size_t)n);
    for (auto& x : v) x = next();
    return v;
  };
  if (next() != RG_PLAN_MAGIC) throw std::runtime_error("not an rg plan descriptor");
  if (next() != RG_PLAN_VERSION) throw std::runtime_error("unsupported plan descriptor version");
  Plan pl;
  int64_t ns = next();
  for (int64_t i = 0; i < ns; i++) {
    Slot s;
    s.dtype = (int32_t)next();
    s.cap = next();
    s.pinned = next() != 0;
    pl.slots.push_back(s);
  }
  int64_t nc = next();
  for (int64_t i = 0; i < nc; i++) {
    Const c;
    c.slot = next();
    c.n = next();
    c.offset = next();
    pl.consts.push_back(c);
  }
  int64_t ni = next();
  for (int64_t i = 0; i < ni; i++) {
    int64_t s = next();
    int64_t n = next();
    pl.inputs.push_back({s, n});
  }
  int64_t no = next();
  for (int64_t i = 0; i < no; i++) {
    Output o;
    o.slot = next();
    o.n = next();
    o.shape = vec(next());
    pl.outputs.push_back(o);
  }
  int64_t nst = next();
  for (int64_t i = 0; i < nst; i++) {
    Step st;
    st.kind = (int32_t)next();
    if (st.kind == RG_STEP_INSTR) {
      Instr& in = st.instr;
      in.op = (int32_t)next();
      in.dtype = (int32_t)next();
      in.dst = next();
      in.n = next();
      in.mode = next();
      in.node = next();
      in.shape = vec(next());
      int64_t na = next();
      for (int64_t a = 0; a < na; a++) {
        Arg arg;
        arg.slot = next();
        arg.shape = vec(next());
        in.args.push_back(arg);
      }
      in.attr = vec(next());
      if (is_sequence(in.op)) {
        size_t q = 0;
        auto word = [&]() -> int64_t {
          if (q >= in.attr.size()) throw std::runtime_error("sequence attributes truncated");
          return in.attr[q++];
        };
        auto real = [&]() {
          const int64_t bits = word();
          double v;
          memcpy(&v, &bits, 8);
          return v;
        };
        in.sequence.flags = word();
        in.sequence.turn = word();
        in.sequence.base = real();
        in.sequence.eps = real();
        const int64_t ns2 = word();
        for (int64_t j = 0; j < ns2; j++) in.sequence.sections.push_back(word());
        const int64_t nr = word();
        for (int64_t j = 0; j < nr; j++) {
          const int64_t index = word();
          in.outs.push_back({index, word()});
        }
      }
    } else if (st.kind == RG_STEP_FUSED || st.kind == RG_STEP_ROWS) {
      const bool rows = st.kind == RG_STEP_ROWS;
      Fused& f = st.fused;
      f.dtype = (int32_t)next();
      f.n = next();
      if (rows) {
        f.row_len = next();
        if (f.row_len <= 0) throw std::runtime_error("row group with an empty row");
      }
      f.regs = next();
      f.shape = vec(next());
      int64_t nin = next();
      for (int64_t a = 0; a < nin; a++) {
        FusedInput fi;
        fi.slot = next();
        fi.kind = next();
        fi.row_len = next();
        fi.reg = next();
        fi.shape = vec(next());
        f.inputs.push_back(fi);
      }
      int64_t nops = next();
      for (int64_t a = 0; a < nops; a++) {
        MicroOp m;
        m.op = (int32_t)next();
        m.reg = next();
        if (rows) m.aux = next();
        int64_t nargs = next();
        for (int64_t b = 0; b < nargs; b++) {
          int64_t is_reg = next();
          int64_t idx = next();
          m.args.push_back({is_reg, idx});
        }
        f.ops.push_back(m);
      }
      int64_t nout = next();
      for (int64_t a = 0; a < nout; a++) {
        int64_t r = next();
        int64_t s = next();
        f.outputs.push_back({r, s});
      }
    } else if (st.kind == RG_STEP_ATTN) {
      Attn& a = st.attn;
      a.dtype = (int32_t)next();
      a.backward = next() != 0;
      a.bh = next();
      a.heads = next();
      a.tq = next();
      a.tk = next();
      a.hd = next();
      int64_t bits = next();
      memcpy(&a.div, &bits, 8);
      bits = next();
      memcpy(&a.fill, &bits, 8);
      a.mask_slot = next();
      for (int k = 0; k < 4; k++) a.mask_strides[k] = next();
      a.mask_bits_slot = next();
      a.build_bits = next() != 0;
      a.stats_slot = next();
      for (int side = 0; side < 2; side++) {
        int64_t n = next();
        if (n < 0 || n > 8) throw std::runtime_error("malformed attention step");
        for (int64_t k = 0; k < n; k++) {
          AttnView v;
          v.slot = next();
          v.offset = next();
          v.sb = next();
          v.sh = next();
          v.st = next();
          (side ? a.out : a.in).push_back(v);
        }
      }
      a.node = next();
      if (a.in.size() != (a.backward ? 5u : 3u) || a.out.size() != (a.backward ? 3u : 1u) || a.bh <= 0 || a.heads <= 0 ||
          a.bh % a.heads != 0)
        throw std::runtime_error("malformed attention step");
    } else {
      throw std::runtime_error("unknown plan step kind");
    }
    pl.steps.push_back(std::move(st));
  }
  if (p != nw) throw std::runtime_error("plan descriptor has trailing words");
  check_refs(pl);
  return pl;
}

/* The attributes of a control-flow step (SCAN, WHILE, COND). Bodies point into the step's
 * attribute words; parse each with `parse`. */
struct ControlAttr {
  int64_t n_carry = 0, n_x = 0, length = 0, max_iterations = 0;
  bool reverse = false;
  std::vector<std::pair<int64_t, int64_t>> results; /* (result index, slot) */
  std::vector<std::pair<const int64_t*, size_t>> bodies;
};

inline bool is_control(int32_t op) { return op == RG_OP_SCAN || op == RG_OP_WHILE || op == RG_OP_COND; }

inline ControlAttr parse_control(const Instr& in) {
  const std::vector<int64_t>& a = in.attr;
  size_t q = 0;
  auto next = [&]() -> int64_t {
    if (q >= a.size()) throw std::runtime_error("control-flow attributes truncated");
    return a[q++];
  };
  ControlAttr c;
  if (in.op == RG_OP_SCAN) {
    c.n_carry = next();
    c.n_x = next();
    c.length = next();
    c.reverse = next() != 0;
  } else if (in.op == RG_OP_WHILE) {
    c.n_carry = next();
    c.max_iterations = next();
  }
  int64_t n = next();
  if (n < 0 || (size_t)n > a.size()) throw std::runtime_error("control-flow attributes have a bad length");
  for (int64_t j = 0; j < n; j++) {
    int64_t index = next();
    c.results.push_back({index, next()});
  }
  n = next();
  if (n < 0 || n > 2) throw std::runtime_error("control-flow step has a bad body count");
  for (int64_t j = 0; j < n; j++) {
    int64_t len = next();
    if (len < 0 || q + (size_t)len > a.size()) throw std::runtime_error("control-flow body truncated");
    c.bodies.push_back({a.data() + q, (size_t)len});
    q += (size_t)len;
  }
  const size_t want = in.op == RG_OP_SCAN ? 1 : 2;
  if (c.bodies.size() != want || c.n_carry < 0 || c.n_x < 0 || c.length < 0 || c.max_iterations < 0 ||
      (size_t)(c.n_carry + c.n_x) > in.args.size())
    throw std::runtime_error("control-flow step is malformed");
  return c;
}

}  // namespace rgplan
#endif /* __cplusplus */

#endif /* RG_PLAN_H */
