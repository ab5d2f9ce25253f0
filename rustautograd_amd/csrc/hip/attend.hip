// Attention with shaped scores: for query i and key j of one head
//
//   s = cap tanh(scale q.k / cap) - slope |i - j|,   p = softmax of s over the keys seen,   y = p v
//
// and its reverse form, with D = dy.y per query,
//
//   dp = dy.v,  ds = p (dp - D),  dslope = -sum ds |i - j|,  du = ds (1 - tanh^2) scale,
//   dv = p^T dy,  dq = du k,  dk = du^T q.
//
// No score is kept: the forward walks the keys once with a running maximum and sum, and leaves the
// logarithm of each query's sum, from which the backward forms p again.
//
// A block of four waves takes 64 rows (queries, or keys where the gradients of k and v are formed),
// a wave 16 of them, and the other side passes through LDS in tiles of 32. Products run on the
// 16x16x4 matrix instructions of the type. A score tile is formed so that a lane holds one of its
// wave's rows and four of the other side's, and feeds the next product from where it lies: that
// product's four steps each take, from every lane, the value of one register, and the other
// operand's rows in the same order (`row_of`). Results have 16 rows of the tile's other dimension,
// the head, spread so that a lane ends with consecutive values of its row.
//
// Scores, sums, maxima and results are held in the type, scores to base 2.
#include "attend.h"

#include <algorithm>
#include <type_traits>

#include "ops.h"

namespace rgk {

namespace {

typedef float floatx2 __attribute__((ext_vector_type(2)));
typedef float floatx4 __attribute__((ext_vector_type(4)));
typedef double doublex2 __attribute__((ext_vector_type(2)));
typedef double doublex4 __attribute__((ext_vector_type(4)));

template <class T>
struct Type;
template <>
struct Type<float> {
  typedef floatx4 acc;
  typedef floatx4 vec;  // 16 bytes
  static constexpr int V = 4;
  static __device__ __forceinline__ acc mfma(float a, float b, acc c) { return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0); }
  // The tile row of register r in a lane of group g (its lane number over 16).
  static __device__ __forceinline__ int row_of(int r, int g) { return 4 * g + r; }
  static __device__ __forceinline__ float exp2_of(float x) { return __builtin_amdgcn_exp2f(x); }
  static __device__ __forceinline__ float log2_of(float x) { return __builtin_amdgcn_logf(x); }
  static __device__ __forceinline__ float max_of(float a, float b) { return fmaxf(a, b); }
  // Below 0.7 the fifth convergent of Lambert's continued fraction x / (1 + x^2 / (3 + ...)), off
  // by 2e-9 of it there; from there on (e^2x - 1) / (e^2x + 1). One division for either.
  static __device__ __forceinline__ float tanh_of(float x) {
    const float a = fminf(fabsf(x), 16.0f), z = a * a;
    const float e = __builtin_amdgcn_exp2f(2.8853900817779268f * a);
    const bool low = a < 0.7f;
    const float num = low ? a * fmaf(z, z + 105.0f, 945.0f) : e - 1.0f, den = low ? fmaf(z, fmaf(15.0f, z, 420.0f), 945.0f) : e + 1.0f;
    const float r = __builtin_amdgcn_rcpf(den), q = num * r;
    return x != x ? x : copysignf(fmaf(fmaf(-den, q, num), r, q), x);
  }
};
template <>
struct Type<double> {
  typedef doublex4 acc;
  typedef doublex2 vec;
  static constexpr int V = 2;
  static __device__ __forceinline__ acc mfma(double a, double b, acc c) { return __builtin_amdgcn_mfma_f64_16x16x4f64(a, b, c, 0, 0, 0); }
  static __device__ __forceinline__ int row_of(int r, int g) { return 4 * r + g; }
  static __device__ __forceinline__ double exp2_of(double x) { return exp2(x); }
  static __device__ __forceinline__ double log2_of(double x) { return log2(x); }
  static __device__ __forceinline__ double max_of(double a, double b) { return fmax(a, b); }
  static __device__ __forceinline__ double tanh_of(double x) { return tanh(x); }
};

// Over the four lanes that hold one row (l, l + 16, l + 32, l + 48), the same in all of them.
template <class T>
__device__ __forceinline__ T row_max(T x) {
  T a, b;
  rg_swap16(x, &a, &b);
  rg_swap32(Type<T>::max_of(a, b), &a, &b);
  return Type<T>::max_of(a, b);
}
template <class T>
__device__ __forceinline__ T row_sum(T x) {
  T a, b;
  rg_swap16(x, &a, &b);
  rg_swap32(a + b, &a, &b);
  return a + b;
}

constexpr int ROWS = 64, TILE = 32, NT = 256;  // rows of a block, rows of a tile, threads

// Rows of HD values in LDS lie 16 bytes further apart than that: 16 lanes reading 16 bytes of 16
// rows each reach every bank once.
template <class T, int HD>
constexpr int PITCH = HD + 16 / (int)sizeof(T);

// N values from LDS or memory at 16 bytes (8 where N values of float are only that).
template <int N, class T>
__device__ __forceinline__ void take(const T* p, T* out) {
  typedef typename Type<T>::vec vec;
  if constexpr (N % Type<T>::V == 0) {
#pragma unroll
    for (int i = 0; i < N; i += Type<T>::V) {
      const vec v = *(const vec*)(p + i);
#pragma unroll
      for (int j = 0; j < Type<T>::V; j++) out[i + j] = v[j];
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; i += 2) {
      const floatx2 v = *(const floatx2*)(p + i);
      out[i] = v[0];
      out[i + 1] = v[1];
    }
  }
}

// A row of `head` values, of which the V from d on are loaded; those past its end are 0.
template <class T>
__device__ __forceinline__ typename Type<T>::vec row_vec(const T* row, uint32_t d, uint32_t head, bool whole) {
  typename Type<T>::vec v = 0;
  if (!row) return v;
  if (whole) {  // rows are 16 bytes aligned and end with a vector
    if (d < head) v = *(const typename Type<T>::vec*)(row + d);
  } else {
#pragma unroll
    for (uint32_t j = 0; j < Type<T>::V; j++)
      if (d + j < head) v[j] = row[d + j];
  }
  return v;
}

// Row `l16`'s fragment of a product over the head: element n * 16 + 4 g + j in frag[4 n + j].
template <class T, int HD>
__device__ __forceinline__ void row_frag(const T* row, int g, uint32_t head, bool whole, T* frag) {
#pragma unroll
  for (int n = 0; n < HD / 16; n++)
#pragma unroll
    for (int j = 0; j < 4; j += Type<T>::V) {
      const auto v = row_vec(row, (uint32_t)(n * 16 + 4 * g + j), head, whole);
#pragma unroll
      for (int i = 0; i < Type<T>::V; i++) frag[4 * n + j + i] = v[i];
    }
}

// Two score tiles (rows 0..15 and 16..31 of `lds` against the lane's row).
template <class T, int HD>
__device__ __forceinline__ void score(const T* lds, int l16, int g, const T* frag, typename Type<T>::acc* s) {
  s[0] = s[1] = typename Type<T>::acc{0, 0, 0, 0};
#pragma unroll
  for (int n = 0; n < HD / 16; n++) {
    T a[4], b[4];
    take<4>(lds + l16 * PITCH<T, HD> + n * 16 + 4 * g, a);
    take<4>(lds + (16 + l16) * PITCH<T, HD> + n * 16 + 4 * g, b);
#pragma unroll
    for (int j = 0; j < 4; j++) {
      s[0] = Type<T>::mfma(a[j], frag[4 * n + j], s[0]);
      s[1] = Type<T>::mfma(b[j], frag[4 * n + j], s[1]);
    }
  }
}

// acc of the lane's row += the tile's 32 rows weighed by w[t][r]: value row_of(r, g) HD / 16 + n of the
// head in acc[n][r].
template <class T, int HD>
__device__ __forceinline__ void weigh(const T* lds, int l16, int g, const typename Type<T>::acc* w, typename Type<T>::acc* acc) {
  constexpr int ND = HD / 16;
#pragma unroll
  for (int t = 0; t < 2; t++)
#pragma unroll
    for (int r = 0; r < 4; r++) {
      T v[ND];
      take<ND>(lds + (t * 16 + Type<T>::row_of(r, g)) * PITCH<T, HD> + l16 * ND, v);
#pragma unroll
      for (int n = 0; n < ND; n++) acc[n] = Type<T>::mfma(v[n], w[t][r], acc[n]);
    }
}

// The lane's share of its row of a result, times `by`.
template <class T, int HD>
__device__ __forceinline__ void put_row(T* row, int g, uint32_t head, const typename Type<T>::acc* acc, T by) {
  constexpr int ND = HD / 16;
#pragma unroll
  for (int r = 0; r < 4; r++)
#pragma unroll
    for (int n = 0; n < ND; n++) {
      const uint32_t d = (uint32_t)(Type<T>::row_of(r, g) * ND + n);
      if (d < head) row[d] = acc[n][r] * by;
    }
}

// The scores of one head, to base 2: cap log2(e) tanh(dot mul) or dot mul, less slope log2(e) times
// the distance.
template <class T>
struct Scorer {
  T mul, cap, slope;  // cap and slope times log2(e)
  bool capped;
  __device__ __forceinline__ Scorer(const AttendArgs& a, uint32_t h) {
    constexpr double LOG2E = 1.4426950408889634;
    capped = a.cap > 0;
    mul = (T)(capped ? a.scale / a.cap : a.scale * LOG2E);
    cap = (T)(a.cap * LOG2E);
    slope = a.slopes ? (T)((double)((const T*)a.slopes)[h] * LOG2E) : (T)0;
  }
  // The score, and the slope of the cap there (1 without one).
  __device__ __forceinline__ T operator()(T dot, int distance, T* bend) const {
    T s = dot * mul;
    *bend = 1;
    if (capped) {
      const T t = Type<T>::tanh_of(s);
      *bend = 1 - t * t;
      s = cap * t;
    }
    return s - slope * (T)distance;
  }
};

// The sequence of a batch that a block works in: its positions, which of them belong to it, and
// which keys a query sees.
struct Sight {
  const int32_t* documents;
  int length, prefix;
  bool causal;
  __device__ __forceinline__ Sight(const AttendArgs& a, uint32_t b) {
    documents = a.documents ? a.documents + (uint64_t)b * a.length : nullptr;
    length = a.lengths ? min(max(a.lengths[b], 0), (int)a.length) : (int)a.length;
    prefix = a.prefix ? a.prefix[b] : 0;
    causal = a.causal;
  }
  __device__ __forceinline__ int document(int i) const { return i >= length ? -1 : documents ? documents[i] : 0; }
  // With the documents of both at hand; those of no sequence are negative.
  __device__ __forceinline__ bool sees(int i, int di, int j, int dj) const { return di >= 0 && di == dj && (!causal || j <= i || j < prefix); }
  // Keys [0, this) hold every one that a query before `end` sees.
  __device__ __forceinline__ int keys_to(int end) const { return min(causal ? max(end, prefix) : length, length); }
  // Queries [this, length) hold every one that sees a key from j on.
  __device__ __forceinline__ int queries_from(int j) const { return causal && j >= prefix ? j : 0; }
};

// One tile of `TILE` rows of two operands on its way to LDS: 16 bytes a thread and step.
template <class T, int HD>
struct Staged {
  static constexpr int PER = TILE * HD / Type<T>::V / NT > 0 ? TILE * HD / Type<T>::V / NT : 1;
  static constexpr bool ALL = TILE * HD / Type<T>::V >= NT;
  typedef typename Type<T>::vec vec;
  vec x[PER], y[PER];
  // `rows(r)` gives the pointers of row r of the two operands, null where there is none.
  template <class R>
  __device__ __forceinline__ void load(const R& rows, uint32_t head, bool whole) {
#pragma unroll
    for (int i = 0; i < PER; i++) {
      const int at = (int)threadIdx.x + i * NT;
      if (!ALL && at >= TILE * HD / Type<T>::V) continue;
      const auto p = rows(at / (HD / Type<T>::V));
      const uint32_t d = (uint32_t)(at % (HD / Type<T>::V)) * Type<T>::V;
      x[i] = row_vec(p.x, d, head, whole);
      y[i] = row_vec(p.y, d, head, whole);
    }
  }
  __device__ __forceinline__ void store(T* xs, T* ys) const {
#pragma unroll
    for (int i = 0; i < PER; i++) {
      const int at = (int)threadIdx.x + i * NT;
      if (!ALL && at >= TILE * HD / Type<T>::V) continue;
      const int o = at / (HD / Type<T>::V) * PITCH<T, HD> + at % (HD / Type<T>::V) * Type<T>::V;
      *(vec*)(xs + o) = x[i];
      *(vec*)(ys + o) = y[i];
    }
  }
};
template <class T>
struct RowPair {
  const T *x, *y;
};

// Block `blockIdx.x`'s head and tile of rows: the heads of a batch next to each other, so that blocks
// of one head meet in the same L2 where their number is a multiple of the eight dies, and the tiles
// with the most work under a causal order first (`last_first`).
struct Place {
  uint32_t b, h, tile;
  __device__ __forceinline__ Place(uint32_t batch, uint32_t heads, uint32_t tiles, bool last_first) {
    const uint32_t bh = blockIdx.x % (batch * heads), at = blockIdx.x / (batch * heads);
    b = bh / heads;
    h = bh % heads;
    tile = last_first ? tiles - 1 - at : at;
  }
};

// The running softmax of a row over its keys: maximum, sum (of the lane's own keys until the end)
// and weighed values.
template <class T, int HD>
struct Running {
  typename Type<T>::acc out[HD / 16];
  T top = -(T)__builtin_huge_val(), sum = 0;
  __device__ __forceinline__ Running() {
#pragma unroll
    for (int n = 0; n < HD / 16; n++) out[n] = typename Type<T>::acc{0, 0, 0, 0};
  }
  // Takes in two tiles of scores, minus infinity where a key is not seen, and leaves their weights.
  __device__ __forceinline__ void add(typename Type<T>::acc* s) {
    T high = s[0][0];
#pragma unroll
    for (int t = 0; t < 2; t++)
#pragma unroll
      for (int r = 0; r < 4; r++) high = Type<T>::max_of(high, s[t][r]);
    const T next = Type<T>::max_of(top, row_max(high));
    // A row that has seen nothing keeps weights of 0.
    const T at = next == -(T)__builtin_huge_val() ? (T)0 : next;
    if (__ballot(next != top) != 0) {
      const T by = Type<T>::exp2_of(top - at);
      sum *= by;
#pragma unroll
      for (int n = 0; n < HD / 16; n++) out[n] *= by;
      top = next;
    }
#pragma unroll
    for (int t = 0; t < 2; t++)
#pragma unroll
      for (int r = 0; r < 4; r++) {
        s[t][r] = Type<T>::exp2_of(s[t][r] - at);
        sum += s[t][r];
      }
  }
};

template <class T, int HD>
__global__ void __launch_bounds__(NT) k_attend(AttendArgs a) {
  __shared__ __align__(16) T ks[TILE * PITCH<T, HD>];
  __shared__ __align__(16) T vs[TILE * PITCH<T, HD>];
  __shared__ int docs[TILE];
  const Place at(a.batch, a.heads, a.tiles, a.causal);
  const Sight sight(a, at.b);
  const int lane = threadIdx.x & 63, l16 = lane & 15, g = lane >> 4;
  const int begin = (int)at.tile * ROWS, i = begin + (int)(threadIdx.x >> 6) * 16 + l16;
  const uint32_t kh = at.h / (a.heads / a.keys);
  const bool whole = a.head % Type<T>::V == 0;
  const Scorer<T> scorer(a, at.h);
  const int di = sight.document(i);
  T frag[HD / 4];
  row_frag<T, HD>(di >= 0 ? (const T*)a.q + ((int64_t)at.b * a.length + i) * a.q_row + at.h * a.head : nullptr, g, a.head, whole, frag);
  const T *kb = (const T*)a.k + (int64_t)at.b * a.length * a.k_row + kh * a.head, *vb = (const T*)a.v + (int64_t)at.b * a.length * a.k_row + kh * a.head;
  const int end = begin < sight.length ? sight.keys_to(min(begin + ROWS, sight.length)) : 0;
  Running<T, HD> run;
  Staged<T, HD> next;
  auto load = [&](int first) {
    next.load([&](int r) {
      const bool in = sight.document(first + r) >= 0;
      const int64_t o = (int64_t)(first + r) * a.k_row;
      return RowPair<T>{in ? kb + o : nullptr, in ? vb + o : nullptr};
    }, a.head, whole);
  };
  if (end > 0) load(0);
  for (int first = 0; first < end; first += TILE) {
    __syncthreads();
    next.store(ks, vs);
    if (threadIdx.x < TILE) docs[threadIdx.x] = sight.document(first + (int)threadIdx.x);
    __syncthreads();
    if (first + TILE < end) load(first + TILE);
    typename Type<T>::acc s[2];
    score<T, HD>(ks, l16, g, frag, s);
#pragma unroll
    for (int t = 0; t < 2; t++)
#pragma unroll
      for (int r = 0; r < 4; r++) {
        const int row = t * 16 + Type<T>::row_of(r, g), j = first + row;
        T bend;
        const T v = scorer(s[t][r], abs(i - j), &bend);
        s[t][r] = sight.sees(i, di, j, docs[row]) ? v : -(T)__builtin_huge_val();
      }
    run.add(s);
    weigh<T, HD>(vs, l16, g, s, run.out);
  }
  const T sum = row_sum(run.sum);
  if (i >= (int)a.length) return;
  const uint64_t row = ((uint64_t)at.b * a.length + i) * a.heads + at.h;
  const bool none = sum == 0;
  if (a.y) put_row<T, HD>((T*)a.y + row * a.head, g, a.head, run.out, none ? (T)0 : 1 / sum);
  // Of a query that sees nothing infinity, so that the backward forms weights of 0.
  if (a.sums && g == 0) ((T*)a.sums)[((uint64_t)at.b * a.heads + at.h) * a.length + i] = none ? (T)__builtin_huge_val() : run.top + Type<T>::log2_of(sum);
}

// The gradient of q, of the slopes, and each query's dy.y for the kernel of the others.
template <class T, int HD>
__global__ void __launch_bounds__(NT) k_attend_dq(AttendArgs a) {
  __shared__ __align__(16) T ks[TILE * PITCH<T, HD>];
  __shared__ __align__(16) T vs[TILE * PITCH<T, HD>];
  __shared__ int docs[TILE];
  __shared__ T waves[NT / 64];
  const Place at(a.batch, a.heads, a.tiles, a.causal);
  const Sight sight(a, at.b);
  const int lane = threadIdx.x & 63, l16 = lane & 15, g = lane >> 4;
  const int begin = (int)at.tile * ROWS, i = begin + (int)(threadIdx.x >> 6) * 16 + l16;
  const uint32_t kh = at.h / (a.heads / a.keys);
  const bool whole = a.head % Type<T>::V == 0;
  const Scorer<T> scorer(a, at.h);
  const int di = sight.document(i);
  const uint64_t row = ((uint64_t)at.b * a.length + i) * a.heads + at.h, stat = ((uint64_t)at.b * a.heads + at.h) * a.length + i;
  T frag[HD / 4], grad[HD / 4];
  row_frag<T, HD>(di >= 0 ? (const T*)a.q + ((int64_t)at.b * a.length + i) * a.q_row + at.h * a.head : nullptr, g, a.head, whole, frag);
  row_frag<T, HD>(di >= 0 ? (const T*)a.dy + row * a.head : nullptr, g, a.head, whole, grad);
  T dot = 0;
  {
    T y[HD / 4];
    row_frag<T, HD>(di >= 0 ? (const T*)a.y_in + row * a.head : nullptr, g, a.head, whole, y);
#pragma unroll
    for (int n = 0; n < HD / 4; n++) dot += y[n] * grad[n];
  }
  dot = row_sum(dot);
  const T sums = di >= 0 ? ((const T*)a.sums_in)[stat] : (T)__builtin_huge_val();
  if (g == 0 && i < (int)a.length) ((T*)a.workspace)[stat] = dot;
  const T *kb = (const T*)a.k + (int64_t)at.b * a.length * a.k_row + kh * a.head, *vb = (const T*)a.v + (int64_t)at.b * a.length * a.k_row + kh * a.head;
  const int end = begin < sight.length ? sight.keys_to(min(begin + ROWS, sight.length)) : 0;
  typename Type<T>::acc out[HD / 16];
#pragma unroll
  for (int n = 0; n < HD / 16; n++) out[n] = typename Type<T>::acc{0, 0, 0, 0};
  T dslope = 0;
  Staged<T, HD> next;
  auto load = [&](int first) {
    next.load([&](int r) {
      const bool in = sight.document(first + r) >= 0;
      const int64_t o = (int64_t)(first + r) * a.k_row;
      return RowPair<T>{in ? kb + o : nullptr, in ? vb + o : nullptr};
    }, a.head, whole);
  };
  if (end > 0) load(0);
  for (int first = 0; first < end; first += TILE) {
    __syncthreads();
    next.store(ks, vs);
    if (threadIdx.x < TILE) docs[threadIdx.x] = sight.document(first + (int)threadIdx.x);
    __syncthreads();
    if (first + TILE < end) load(first + TILE);
    typename Type<T>::acc s[2], dp[2];
    score<T, HD>(ks, l16, g, frag, s);
    score<T, HD>(vs, l16, g, grad, dp);
#pragma unroll
    for (int t = 0; t < 2; t++)
#pragma unroll
      for (int r = 0; r < 4; r++) {
        const int row_in = t * 16 + Type<T>::row_of(r, g), j = first + row_in, distance = abs(i - j);
        T bend;
        const T v = scorer(s[t][r], distance, &bend);
        const bool seen = sight.sees(i, di, j, docs[row_in]);
        const T ds = seen ? Type<T>::exp2_of(v - sums) * (dp[t][r] - dot) : (T)0;
        dslope -= ds * (T)distance;
        s[t][r] = ds * bend;
      }
    weigh<T, HD>(ks, l16, g, s, out);
  }
  if (a.dq && i < (int)a.length) put_row<T, HD>((T*)a.dq + ((int64_t)at.b * a.length + i) * a.q_row + at.h * a.head, g, a.head, out, (T)a.scale);
  if (a.dslopes_rows) {
    dslope = rg_wave_sum(dslope);
    if (lane == 0) waves[threadIdx.x >> 6] = dslope;
    __syncthreads();
    if (threadIdx.x == 0)
      ((T*)a.dslopes_rows)[((uint64_t)at.b * a.tiles + at.tile) * a.heads + at.h] = ((waves[0] + waves[1]) + waves[2]) + waves[3];
  }
}

// The gradients of k and v: a block's 64 keys against the queries of every head that reads them.
template <class T, int HD>
__global__ void __launch_bounds__(NT) k_attend_dkv(AttendArgs a) {
  __shared__ __align__(16) T qs[TILE * PITCH<T, HD>];
  __shared__ __align__(16) T gs[TILE * PITCH<T, HD>];
  __shared__ int docs[TILE];
  __shared__ T sums[TILE], dots[TILE];
  const Place at(a.batch, a.keys, a.tiles, false);
  const Sight sight(a, at.b);
  const int lane = threadIdx.x & 63, l16 = lane & 15, g = lane >> 4;
  const int begin = (int)at.tile * ROWS, j = begin + (int)(threadIdx.x >> 6) * 16 + l16;
  const uint32_t group = a.heads / a.keys;
  const bool whole = a.head % Type<T>::V == 0;
  const int dj = sight.document(j);
  const int64_t key = ((int64_t)at.b * a.length + j) * a.k_row + at.h * a.head;
  T frag[HD / 4], value[HD / 4];
  row_frag<T, HD>(dj >= 0 ? (const T*)a.k + key : nullptr, g, a.head, whole, frag);
  row_frag<T, HD>(dj >= 0 ? (const T*)a.v + key : nullptr, g, a.head, whole, value);
  typename Type<T>::acc dk[HD / 16], dv[HD / 16];
#pragma unroll
  for (int n = 0; n < HD / 16; n++) dk[n] = dv[n] = typename Type<T>::acc{0, 0, 0, 0};
  const int from = sight.queries_from(begin) / TILE * TILE, end = begin < sight.length ? sight.length : 0;
  const uint32_t per_head = end > from ? (uint32_t)(end - from + TILE - 1) / TILE : 0, steps = per_head * group;
  Staged<T, HD> next;
  auto load = [&](uint32_t step) {
    const uint32_t h = at.h * group + step / per_head;
    const int first = from + (int)(step % per_head) * TILE;
    next.load([&](int r) {
      const bool in = sight.document(first + r) >= 0;
      const int64_t t = (int64_t)at.b * a.length + first + r;
      return RowPair<T>{in ? (const T*)a.q + t * a.q_row + h * a.head : nullptr, in ? (const T*)a.dy + (t * a.heads + h) * a.head : nullptr};
    }, a.head, whole);
  };
  if (steps > 0) load(0);
  for (uint32_t step = 0; step < steps; step++) {
    const uint32_t h = at.h * group + step / per_head;
    const int first = from + (int)(step % per_head) * TILE;
    const Scorer<T> scorer(a, h);
    __syncthreads();
    next.store(qs, gs);
    if (threadIdx.x < TILE) {
      const int i = first + (int)threadIdx.x, di = sight.document(i);
      const uint64_t stat = ((uint64_t)at.b * a.heads + h) * a.length + i;
      docs[threadIdx.x] = di;
      sums[threadIdx.x] = di >= 0 ? ((const T*)a.sums_in)[stat] : (T)__builtin_huge_val();
      dots[threadIdx.x] = di >= 0 ? ((const T*)a.workspace)[stat] : (T)0;
    }
    __syncthreads();
    if (step + 1 < steps) load(step + 1);
    typename Type<T>::acc s[2], dp[2];
    score<T, HD>(qs, l16, g, frag, s);
    score<T, HD>(gs, l16, g, value, dp);
#pragma unroll
    for (int t = 0; t < 2; t++)
#pragma unroll
      for (int r = 0; r < 4; r++) {
        const int row = t * 16 + Type<T>::row_of(r, g), i = first + row;
        T bend;
        const T v = scorer(s[t][r], abs(i - j), &bend);
        const bool seen = sight.sees(i, docs[row], j, dj);
        const T p = seen ? Type<T>::exp2_of(v - sums[row]) : (T)0;
        s[t][r] = p;
        dp[t][r] = seen ? p * (dp[t][r] - dots[row]) * bend : (T)0;
      }
    weigh<T, HD>(gs, l16, g, s, dv);
    weigh<T, HD>(qs, l16, g, dp, dk);
  }
  if (j >= (int)a.length) return;
  if (a.dk) put_row<T, HD>((T*)a.dk + key, g, a.head, dk, (T)a.scale);
  if (a.dv) put_row<T, HD>((T*)a.dv + key, g, a.head, dv, (T)1);
}

// ---- over a paged cache ----------------------------------------------------------------------------

constexpr int FIRST_MOST = 1 << 30;  // positions before the new tokens that are told apart

// A sequence's keys in order: those that its pages hold, then the new tokens'.
struct Cache {
  const int32_t* table;
  int first, past, count;  // positions before the new tokens, those within the table, new tokens
  uint32_t pages, page;
  FastDiv div;
  __device__ __forceinline__ Cache(const AttendArgs& a, uint32_t b) {
    table = a.table + (uint64_t)b * a.table_pages;
    first = min(max(a.first[b], 0), FIRST_MOST);
    past = min(first, (int)(a.table_pages * a.page));
    count = a.lengths ? min(max(a.lengths[b], 0), (int)a.length) : (int)a.length;
    pages = a.pages;
    page = a.page;
    div = a.page_div;
  }
  // Row number of position p among the pages, or -1.
  __device__ __forceinline__ int64_t row(uint32_t p) const {
    const uint32_t n = div.div(p), at = (uint32_t)table[n];
    return at < pages ? (int64_t)at * page + (p - n * page) : -1;
  }
};

// Rows of a sequence's queries: the heads of one key head side by side, token after token.
template <class T, int HD>
__global__ void __launch_bounds__(NT) k_paged(AttendArgs a) {
  __shared__ __align__(16) T ks[TILE * PITCH<T, HD>];
  __shared__ __align__(16) T vs[TILE * PITCH<T, HD>];
  __shared__ int there[TILE];
  const uint32_t split = blockIdx.x % a.splits, rest = blockIdx.x / a.splits;
  const uint32_t bh = rest % (a.batch * a.keys), tile = rest / (a.batch * a.keys), b = bh / a.keys, kh = bh % a.keys, group = a.heads / a.keys;
  const Cache cache(a, b);
  const int lane = threadIdx.x & 63, l16 = lane & 15, g = lane >> 4;
  const uint32_t begin = tile * ROWS, r0 = begin + (threadIdx.x >> 6) * 16 + l16;
  const int i = (int)(r0 / group);
  const uint32_t h = kh * group + r0 % group;
  const bool whole = a.head % Type<T>::V == 0, in = i < cache.count;
  const Scorer<T> scorer(a, h);
  T frag[HD / 4];
  row_frag<T, HD>(in ? (const T*)a.q + ((int64_t)b * a.length + i) * a.q_row + h * a.head : nullptr, g, a.head, whole, frag);
  // Keys in order: `past` of the pages, then the new tokens up to the last query of the tile.
  const int last = min((int)((begin + ROWS - 1) / group), cache.count - 1);
  const int all = (int)(begin / group) < cache.count ? cache.past + last + 1 : 0;
  const int from = (int)min((uint64_t)split * a.split_keys, (uint64_t)all), end = (int)min((uint64_t)(split + 1) * a.split_keys, (uint64_t)all);
  const T *kb = (const T*)a.k + (int64_t)b * a.length * a.k_row + kh * a.head, *vb = (const T*)a.v + (int64_t)b * a.length * a.k_row + kh * a.head;
  Running<T, HD> run;
  Staged<T, HD> next;
  auto load = [&](int at) {
    next.load([&](int r) {
      const int c = at + r;
      if (c >= end) return RowPair<T>{nullptr, nullptr};
      if (c >= cache.past) {
        const int64_t o = (int64_t)(c - cache.past) * a.k_row;
        return RowPair<T>{kb + o, vb + o};
      }
      const int64_t row = cache.row((uint32_t)c);
      if (row < 0) return RowPair<T>{nullptr, nullptr};
      const int64_t o = (row * a.keys + kh) * a.head;
      return RowPair<T>{(const T*)a.k_pages + o, (const T*)a.v_pages + o};
    }, a.head, whole);
  };
  if (from < end) load(from);
  for (int at = from; at < end; at += TILE) {
    __syncthreads();
    next.store(ks, vs);
    if (threadIdx.x < TILE) {
      const int c = at + (int)threadIdx.x;
      there[threadIdx.x] = c < end && (c >= cache.past || cache.row((uint32_t)c) >= 0);
    }
    __syncthreads();
    if (at + TILE < end) load(at + TILE);
    typename Type<T>::acc s[2];
    score<T, HD>(ks, l16, g, frag, s);
#pragma unroll
    for (int t = 0; t < 2; t++)
#pragma unroll
      for (int r = 0; r < 4; r++) {
        const int row = t * 16 + Type<T>::row_of(r, g), c = at + row;
        const bool old = c < cache.past;
        const int distance = old ? cache.first + i - c : i - (c - cache.past);
        T bend;
        const T v = scorer(s[t][r], distance, &bend);
        s[t][r] = in && there[row] && distance >= 0 ? v : -(T)__builtin_huge_val();
      }
    run.add(s);
    weigh<T, HD>(vs, l16, g, s, run.out);
  }
  const T sum = row_sum(run.sum);
  if (i >= (int)a.length) return;
  const uint64_t row = ((uint64_t)b * a.length + i) * a.heads + h;
  if (a.splits == 1) {
    if (a.y) put_row<T, HD>((T*)a.y + row * a.head, g, a.head, run.out, sum == 0 ? (T)0 : 1 / sum);
    return;
  }
  // A split's maximum, sum and weighed values: [rows][splits] of 2 + head.
  T* part = (T*)a.partial + (row * a.splits + split) * (a.head + 2);
  put_row<T, HD>(part + 2, g, a.head, run.out, (T)1);
  if (g == 0) {
    part[0] = run.top;
    part[1] = sum;
  }
}

// Joins the splits of each row, a wave a row, and then (blocks from `join_blocks` on) puts the new
// tokens' keys and values into their pages, a wave a token and key head. Rows that a later sequence
// writes too are left to it, so that the result does not depend on which comes first.
template <class T>
__global__ void __launch_bounds__(NT) k_paged_finish(AttendArgs a, uint32_t join_blocks) {
  const uint32_t lane = threadIdx.x & 63;
  if (blockIdx.x < join_blocks) {
    const uint64_t row = (uint64_t)blockIdx.x * (NT / 64) + (threadIdx.x >> 6);
    if (row >= (uint64_t)a.batch * a.length * a.heads) return;
    const T* part = (const T*)a.partial + row * a.splits * (a.head + 2);
    T top = -(T)__builtin_huge_val();
    for (uint32_t p = lane; p < a.splits; p += 64) top = Type<T>::max_of(top, part[(uint64_t)p * (a.head + 2)]);
    top = rg_wave_max(top);
    if (top == -(T)__builtin_huge_val()) top = 0;
    T sum = 0;
    for (uint32_t p = lane; p < a.splits; p += 64) sum += part[(uint64_t)p * (a.head + 2) + 1] * Type<T>::exp2_of(part[(uint64_t)p * (a.head + 2)] - top);
    sum = rg_wave_sum(sum);
    for (uint32_t d = lane; d < a.head; d += 64) {
      T v = 0;
      for (uint32_t p = 0; p < a.splits; p++) v += part[(uint64_t)p * (a.head + 2) + 2 + d] * Type<T>::exp2_of(part[(uint64_t)p * (a.head + 2)] - top);
      ((T*)a.y)[row * a.head + d] = sum == 0 ? (T)0 : v / sum;
    }
    return;
  }
  const uint64_t item = (uint64_t)(blockIdx.x - join_blocks) * (NT / 64) + (threadIdx.x >> 6);
  if (item >= (uint64_t)a.batch * a.length * a.keys) return;
  const uint32_t kh = (uint32_t)(item % a.keys), i = (uint32_t)(item / a.keys % a.length), b = (uint32_t)(item / a.keys / a.length);
  const Cache cache(a, b);
  const uint32_t p = (uint32_t)cache.first + i;
  if ((int)i >= cache.count || p >= a.table_pages * a.page) return;
  const int64_t row = cache.row(p);
  if (row < 0) return;
  bool later = false;
  for (uint32_t other = b + 1 + lane; other < a.batch; other += 64) {
    const Cache c(a, other);
    // Its new positions that have this row's place in a page, page by page.
    const uint32_t in = (uint32_t)(row % a.page), begin = (uint32_t)c.first, stop = (uint32_t)min((uint64_t)c.first + c.count, (uint64_t)a.table_pages * a.page);
    for (uint32_t n = c.div.div(begin); n < a.table_pages && n * a.page < stop; n++) {
      const uint32_t at = n * a.page + in;
      if (at >= begin && at < stop && c.row(at) == row) later = true;
    }
  }
  if (__ballot(later) != 0) return;
  const int64_t src = ((int64_t)b * a.length + i) * a.k_row + kh * a.head, dst = (row * a.keys + kh) * a.head;
  for (uint32_t d = lane; d < a.head; d += 64) {
    if (a.k_out) ((T*)a.k_out)[dst + d] = ((const T*)a.k)[src + d];
    if (a.v_out) ((T*)a.v_out)[dst + d] = ((const T*)a.v)[src + d];
  }
}

// ---- the joint norm --------------------------------------------------------------------------------

constexpr uint64_t NORM_PER_BLOCK = 16384;

template <class T>
__global__ void __launch_bounds__(NT) k_norm_squares(NormTensors t, double* partial) {
  uint32_t k = 0;
  while (k + 1 < t.count && blockIdx.x >= t.first_block[k + 1]) k++;
  const uint64_t begin = (uint64_t)(blockIdx.x - t.first_block[k]) * NORM_PER_BLOCK, end = min(begin + NORM_PER_BLOCK, t.n[k]);
  const T* x = (const T*)t.x[k];
  double sum = 0;
  for (uint64_t i = begin + threadIdx.x; i < end; i += NT) {
    const double v = (double)x[i];
    sum += v * v;
  }
  __shared__ double waves[NT / 64];
  sum = rg_wave_sum(sum);
  if ((threadIdx.x & 63) == 0) waves[threadIdx.x >> 6] = sum;
  __syncthreads();
  if (threadIdx.x == 0) partial[blockIdx.x] = ((waves[0] + waves[1]) + waves[2]) + waves[3];
}

template <class T>
__global__ void __launch_bounds__(1024) k_norm_root(const double* partial, uint32_t blocks, T* out) {
  __shared__ double waves[16];
  double sum = 0;
  for (uint32_t i = threadIdx.x; i < blocks; i += 1024) sum += partial[i];
  sum = rg_wave_sum(sum);
  if ((threadIdx.x & 63) == 0) waves[threadIdx.x >> 6] = sum;
  __syncthreads();
  if (threadIdx.x == 0) {
    sum = 0;
    for (int w = 0; w < 16; w++) sum += waves[w];
    *out = (T)sqrt(sum);
  }
}

// ---- launchers -------------------------------------------------------------------------------------

// Calls f with the type and the padded head as constants.
template <class F>
void by_head(int dtype, uint32_t head, const F& f) {
  auto of = [&](auto t) {
    if (head <= 32) f(t, std::integral_constant<int, 32>{});
    else if (head <= 64) f(t, std::integral_constant<int, 64>{});
    else if (head <= 96) f(t, std::integral_constant<int, 96>{});
    else if (head <= 128) f(t, std::integral_constant<int, 128>{});
    else f(t, std::integral_constant<int, 256>{});
  };
  if (dtype == RG_F32) of(float{});
  else of(double{});
}

void set_rows(AttendArgs& a) {
  a.q_row = (int64_t)(a.joined ? a.heads + 2 * a.keys : a.heads) * a.head;
  a.k_row = a.joined ? a.q_row : (int64_t)a.keys * a.head;
  a.tiles = (a.length + ROWS - 1) / ROWS;
}

uint64_t size_of(int dtype) { return dtype == RG_F32 ? 4 : 8; }

// Tiles of a sequence's rows in the paged form, and over how many blocks their keys are split: as
// many as leave each 256 keys and the device four blocks for every CU.
uint32_t paged_tiles(const AttendArgs& a) { return (uint32_t)(((uint64_t)a.length * (a.heads / a.keys) + ROWS - 1) / ROWS); }
void set_splits(AttendArgs& a) {
  const uint64_t keys = (uint64_t)a.table_pages * a.page + a.length, blocks = (uint64_t)a.batch * a.keys * paged_tiles(a);
  const uint64_t most = (keys + 255) / 256, want = (1024 + blocks - 1) / blocks;
  uint64_t n = std::max<uint64_t>(1, std::min(most, want));
  const uint64_t per = ((keys + n - 1) / n + TILE - 1) / TILE * TILE;
  a.splits = (uint32_t)((keys + per - 1) / per);
  a.split_keys = (uint32_t)per;
}

}  // namespace

uint64_t attend_blocks(int, const AttendArgs& a) { return (uint64_t)a.batch * a.heads * ((a.length + ROWS - 1) / ROWS); }
uint64_t attend_workspace(int dtype, const AttendArgs& a) { return (uint64_t)a.batch * a.heads * a.length * size_of(dtype); }
uint32_t attend_slope_rows(int, const AttendArgs& a) { return a.batch * ((a.length + ROWS - 1) / ROWS); }

void attend(hipStream_t s, int dtype, const AttendArgs& args) {
  AttendArgs a = args;
  set_rows(a);
  by_head(dtype, a.head, [&](auto t, auto hd) {
    k_attend<decltype(t), decltype(hd)::value><<<a.tiles * a.batch * a.heads, NT, 0, s>>>(a);
  });
}

void attend_grad(hipStream_t s, int dtype, const AttendArgs& args) {
  AttendArgs a = args;
  set_rows(a);
  by_head(dtype, a.head, [&](auto t, auto hd) {
    k_attend_dq<decltype(t), decltype(hd)::value><<<a.tiles * a.batch * a.heads, NT, 0, s>>>(a);
    if (a.dk || a.dv) k_attend_dkv<decltype(t), decltype(hd)::value><<<a.tiles * a.batch * a.keys, NT, 0, s>>>(a);
  });
}

uint64_t paged_blocks(int, const AttendArgs& args) {
  AttendArgs a = args;
  set_splits(a);
  const uint64_t rows = (uint64_t)a.batch * a.length * (a.heads + a.keys) / (NT / 64) + 2;
  return std::max((uint64_t)a.batch * a.keys * paged_tiles(a) * a.splits, rows);
}

uint64_t paged_workspace(int dtype, const AttendArgs& args) {
  AttendArgs a = args;
  set_splits(a);
  return a.splits == 1 ? 0 : (uint64_t)a.batch * a.length * a.heads * a.splits * (a.head + 2) * size_of(dtype);
}

void paged_attend(hipStream_t s, int dtype, const AttendArgs& args) {
  AttendArgs a = args;
  set_rows(a);
  set_splits(a);
  a.partial = a.workspace;
  a.page_div = FastDiv(a.page);
  const uint64_t values = (uint64_t)a.pages * a.page * a.keys * a.head * size_of(dtype);
  if (a.k_out && a.k_out != a.k_pages) copy_bytes(s, a.k_out, a.k_pages, values);
  if (a.v_out && a.v_out != a.v_pages) copy_bytes(s, a.v_out, a.v_pages, values);
  const uint32_t blocks = a.batch * a.keys * paged_tiles(a) * a.splits;
  by_head(dtype, a.head, [&](auto t, auto hd) {
    if (a.y) k_paged<decltype(t), decltype(hd)::value><<<blocks, NT, 0, s>>>(a);
  });
  const uint32_t join = a.y && a.splits > 1 ? (uint32_t)(((uint64_t)a.batch * a.length * a.heads + NT / 64 - 1) / (NT / 64)) : 0;
  const uint32_t append = a.k_out || a.v_out ? (uint32_t)(((uint64_t)a.batch * a.length * a.keys + NT / 64 - 1) / (NT / 64)) : 0;
  if (join + append == 0) return;
  if (dtype == RG_F32) k_paged_finish<float><<<join + append, NT, 0, s>>>(a, join);
  else k_paged_finish<double><<<join + append, NT, 0, s>>>(a, join);
}

uint32_t norm_blocks(uint64_t n) { return (uint32_t)((n + NORM_PER_BLOCK - 1) / NORM_PER_BLOCK); }

void norm_squares(hipStream_t s, int dtype, const NormTensors& t, uint32_t blocks, double* partial) {
  if (dtype == RG_F32) k_norm_squares<float><<<blocks, NT, 0, s>>>(t, partial);
  else k_norm_squares<double><<<blocks, NT, 0, s>>>(t, partial);
}

void norm_root(hipStream_t s, int dtype, const double* partial, uint32_t blocks, void* out) {
  if (dtype == RG_F32) k_norm_root<float><<<1, 1024, 0, s>>>(partial, blocks, (float*)out);
  else k_norm_root<double><<<1, 1024, 0, s>>>(partial, blocks, (double*)out);
}

}  // namespace rgk
