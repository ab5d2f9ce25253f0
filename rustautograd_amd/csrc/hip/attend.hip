// Attention with shaped scores: for query i and key j of one head
//
//   s = cap tanh(scale q.k / cap) - slope |i - j|,   p = softmax of s over the keys seen,   y = p v
//
// and its reverse form, with D = dy.y per query,
//
//   dp = dy.v,  ds = p (dp - D),  dslope = -sum ds |i - j|,  du = ds (1 - tanh^2) scale,
//   dv = p^T dy,  dq = du k,  dk = du^T q.
//
// No score is kept: the forward walks the keys once with a running maximum and sum, and leaves both of
// each query, from which the backward forms p again.
//
// A block takes 64 rows (queries, or keys where the gradients of k and v are formed), a wave 16 of
// them, and the other side passes through LDS, 32 rows at a time for each set of four waves: with
// two sets a block walks two such tiles at once and joins its halves at the end. Products run on the
// 16x16x4 matrix instructions of the type. A score tile is formed so that a lane holds one of its
// wave's rows and four of the other side's, and feeds the next product from where it lies: that
// product's four steps each take, from every lane, the value of one register, and the other
// operand's rows in the same order (`row_of`). Results have 16 rows of the tile's other dimension,
// the head, spread so that a lane ends with consecutive values of its row.
//
// Scores, sums, maxima and results are held in the type. The logarithm's base enters with the bound that a
// weight's score is lowered by, 2^(log2(e) s - bound) with one rounding, of a difference that is small where
// the weight is not: scores kept to base 2, and rounded as such, left the slopes' gradients half again as far off.
//
// Times below are of one MI355X, whose fp32 matrix product of 8192^3 reaches 154 TFLOP/s and whose copy
// of 2 GB 4.9 TB/s. "The causal case" is 2 sequences of 2048, 8 heads of 64, capped: 8.6 GFLOP forward.
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
  static constexpr float MOST = __FLT_MAX__;
  static __device__ __forceinline__ acc mfma(float a, float b, acc c) { return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0); }
  // The tile row of register r in a lane of group g (its lane number over 16).
  static __device__ __forceinline__ int row_of(int r, int g) { return 4 * g + r; }
  // Of a tile of results the one of row and column l16, from the lane that holds it.
  static __device__ __forceinline__ float diagonal(acc x, int l16) {
    const int r = l16 & 3;
    return __shfl(r == 0 ? x[0] : r == 1 ? x[1] : r == 2 ? x[2] : x[3], l16 + 16 * (l16 >> 2));
  }
  static __device__ __forceinline__ float exp2_of(float x) { return __builtin_amdgcn_exp2f(x); }
  static __device__ __forceinline__ float max_of(float a, float b) { return fmaxf(a, b); }
  // What tanh(x) of up to 1 in size lacks of x, as a share of it: z q(z) with z = x^2, q the polynomial
  // whose largest relative error of the tanh over that range is least (4e-9).
  static __device__ __forceinline__ float tanh_share(float x) {
    const float z = x * x;
    float q = -3.5334553103893995e-4f;
    q = fmaf(q, z, 2.282229484990239e-3f);
    q = fmaf(q, z, -7.917444221675396e-3f);
    q = fmaf(q, z, 2.1464820951223373e-2f);
    q = fmaf(q, z, -5.387091264128685e-2f);
    q = fmaf(q, z, 1.333215981721878e-1f);
    return fmaf(q, z, -3.333327770233154e-1f) * z;
  }
  // Of any size: below 0.7 the fifth convergent of Lambert's continued fraction x / (1 + x^2 / (3 +
  // ...)), off by 2e-9 of it there, from there on (e^2x - 1) / (e^2x + 1), with one division.
  static __device__ __forceinline__ float tanh_of(float x) {
    const float a = fminf(fabsf(x), 16.0f), z = a * a, e = __builtin_amdgcn_exp2f(2.8853900817779268f * a);
    const bool low = a < 0.7f;
    const float num = low ? a * fmaf(z, z + 105.0f, 945.0f) : e - 1.0f, den = low ? fmaf(z, fmaf(15.0f, z, 420.0f), 945.0f) : e + 1.0f;
    const float r = __builtin_amdgcn_rcpf(den), q = num * r, t = fmaf(fmaf(-den, q, num), r, q);
    return copysignf(x == x ? t : x, x);
  }
  static constexpr bool LOW = true;
};
template <>
struct Type<double> {
  typedef doublex4 acc;
  typedef doublex2 vec;
  static constexpr int V = 2;
  static constexpr double MOST = __DBL_MAX__;
  static __device__ __forceinline__ acc mfma(double a, double b, acc c) { return __builtin_amdgcn_mfma_f64_16x16x4f64(a, b, c, 0, 0, 0); }
  static __device__ __forceinline__ int row_of(int r, int g) { return 4 * r + g; }
  static __device__ __forceinline__ double diagonal(acc x, int l16) {
    const int r = l16 >> 2;
    return __shfl(r == 0 ? x[0] : r == 1 ? x[1] : r == 2 ? x[2] : x[3], l16 + 16 * (l16 & 3));
  }
  static __device__ __forceinline__ double exp2_of(double x) { return exp2(x); }
  static __device__ __forceinline__ double max_of(double a, double b) { return fmax(a, b); }
  static __device__ __forceinline__ double tanh_share(double x) { return 0; }  // not called (LOW)
  // (e^2x - 1) / (e^2x + 1), where e^2x - 1 = (2^n - 1) + 2^n (e^y - 1) with y of at most ln 2 / 2 in size,
  // and e^y - 1 is its Taylor series to the 14th power (off by 2e-19 of it): no digit is lost near 0, where
  // n = 0. Within 3 of 2^-53 of the tanh; the library's, also within few, takes the forward of 2 x 130 x 4
  // heads of 32 from 18 to 22 us.
  static __device__ __forceinline__ double tanh_of(double x) {
    const double a = fmin(2 * fabs(x), 40.0), n = __builtin_rint(a * 1.4426950408889634);
    const double y = fma(n, -0.6931471805599453, a);
    double p = 1.0 / 87178291200.0;
    p = fma(p, y, 1.0 / 6227020800.0);
    p = fma(p, y, 1.0 / 479001600.0);
    p = fma(p, y, 1.0 / 39916800.0);
    p = fma(p, y, 1.0 / 3628800.0);
    p = fma(p, y, 1.0 / 362880.0);
    p = fma(p, y, 1.0 / 40320.0);
    p = fma(p, y, 1.0 / 5040.0);
    p = fma(p, y, 1.0 / 720.0);
    p = fma(p, y, 1.0 / 120.0);
    p = fma(p, y, 1.0 / 24.0);
    p = fma(p, y, 1.0 / 6.0);
    p = fma(p, y, 0.5);
    const double e = fma(p, y * y, y), two = __builtin_ldexp(1.0, (int)n), up = fma(two, e, two - 1);
    return copysign(x == x ? up / (up + 2) : x, x);
  }
  static constexpr bool LOW = false;
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

// 2^(log2(e) s - bound): a weight.
template <class T>
__device__ __forceinline__ T weight(T s, T bound) {
  return Type<T>::exp2_of(fma(s, (T)1.4426950408889634, -bound));
}

constexpr int TILE = 32;  // rows of the other side in a wave's tile

// A block's waves: RW of them take 16 rows each, in SETS sets, and each set has a tile of its own of the
// STAGE rows staged at once. Eight waves where four fit a SIMD (two blocks a CU), else four, of which two
// fit, in blocks of their own.
template <class T, int HD, int RW_>
struct Geo {
  static constexpr int SIZE = (int)sizeof(T) * HD, RW = RW_;
  static constexpr bool NARROW = SIZE <= 256;
  static constexpr int WAVES = NARROW ? 8 : 4, SETS = WAVES / RW, NT = 64 * WAVES, ROWS = 16 * RW, STAGE = TILE * SETS;
  // Waves a SIMD that the registers are to leave room for.
  static constexpr int FORWARD = SIZE <= 256 && sizeof(T) == 4 ? (SIZE == 256 && RW == 2 ? 2 : 4) : SIZE <= 512 ? 2 : 1;
  static constexpr int BACKWARD = SIZE <= 256 && sizeof(T) == 4 ? (SIZE == 256 && RW == 2 ? 2 : 4) : SIZE <= 512 && sizeof(T) == 4 ? 2 : SIZE <= 256 ? 2 : 1;
  // The backward's own rows lie in LDS and not in registers.
  static constexpr bool KEPT = NARROW && sizeof(T) == 4;
};

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

// A lane's row as the fragments of a product over the head: in registers, or in LDS where the waves of
// all sets share it.
template <class T, int HD>
struct Registers {
  T frag[HD / 4];
  __device__ __forceinline__ void get(int n, T* out) const {
#pragma unroll
    for (int j = 0; j < 4; j++) out[j] = frag[4 * n + j];
  }
};
template <class T, int HD>
struct Kept {
  const T* at;  // the row's place 4 g
  __device__ __forceinline__ void get(int n, T* out) const { take<4>(at + n * 16, out); }
};

// Two score tiles (rows 0..15 and 16..31 of `lds` against the lane's row), each half of the head summed by
// itself, which halves the length of the chain of roundings (gradients of heads of 64 a third further off with
// one; dq of the causal case 182 us for 190).
template <class T, int HD, class F>
__device__ __forceinline__ void score(const T* lds, int l16, int g, const F& own, typename Type<T>::acc* s) {
  constexpr int HALF = HD / 32;
  typename Type<T>::acc late[2];
  s[0] = s[1] = late[0] = late[1] = typename Type<T>::acc{0, 0, 0, 0};
#pragma unroll
  for (int m = 0; m < HALF; m++)
#pragma unroll
    for (int half = 0; half < 2; half++) {
      const int n = half * HALF + m;
      T a[4], b[4], x[4];
      take<4>(lds + l16 * PITCH<T, HD> + n * 16 + 4 * g, a);
      take<4>(lds + (16 + l16) * PITCH<T, HD> + n * 16 + 4 * g, b);
      own.get(n, x);
      typename Type<T>::acc* to = half == 0 ? s : late;
#pragma unroll
      for (int j = 0; j < 4; j++) {
        to[0] = Type<T>::mfma(a[j], x[j], to[0]);
        to[1] = Type<T>::mfma(b[j], x[j], to[1]);
      }
    }
  s[0] += late[0];
  s[1] += late[1];
}

// acc of the lane's row += the tile's 32 rows weighed by w[t][r]: value row_of(r, g) HD / 16 + n of the
// head in acc[n][r]. Keys that are not seen have weights of 0, which would not keep infinities and NaN
// out: the rows have none (make_finite).
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

// The lane's share of its row of a result, times `by`; 0 where there is none.
template <class T, int HD>
__device__ __forceinline__ void put_row(T* row, int g, uint32_t head, const typename Type<T>::acc* acc, T by, bool none) {
  constexpr int ND = HD / 16;
#pragma unroll
  for (int r = 0; r < 4; r++)
#pragma unroll
    for (int n = 0; n < ND; n++) {
      const uint32_t d = (uint32_t)(Type<T>::row_of(r, g) * ND + n);
      if (d < head) row[d] = none ? (T)0 : acc[n][r] * by;
    }
}

// Positions from 0 of the tile rows that a lane's scores [t][r] belong to.
template <class T>
__device__ __forceinline__ constexpr int tile_row(int t, int r) {
  return 16 * t + Type<T>::row_of(r, 0);
}

// The scores of one head: cap tanh(dot scale / cap) or dot scale, less slope times the distance.
template <class T>
struct Scorer {
  typedef typename Type<T>::acc acc;
  T mul, part, cap, slope;  // the scale, and over the cap
  bool capped, sloped;
  __device__ __forceinline__ Scorer(const AttendArgs& a, uint32_t h) {
    capped = a.cap > 0;
    sloped = a.slopes != nullptr;
    mul = (T)a.scale;
    part = (T)(capped ? a.scale / a.cap : 0);
    cap = (T)a.cap;
    slope = sloped ? ((const T*)a.slopes)[h] : (T)0;
  }
  // Makes scores of dot products, and leaves the tanh of each (0 without a cap) where asked to.
  // `apart` is the signed distance between the lane's row and row row_of(0, g) of the tile.
  template <bool TANH>
  __device__ __forceinline__ void operator()(acc* s, acc* bent, int apart) const {
    if (capped) {
      // Scores below the cap, as most are, differ from the uncapped by a share, which spares them two
      // roundings beside the quotient.
      bool high = !Type<T>::LOW;
      if constexpr (Type<T>::LOW) {
        T most = 0;
#pragma unroll
        for (int t = 0; t < 2; t++)
#pragma unroll
          for (int r = 0; r < 4; r++) most = Type<T>::max_of(most, abs_of(s[t][r]));
        high = __ballot(most * abs_of(part) > 1) != 0;
      }
      if (high) {
#pragma unroll
        for (int t = 0; t < 2; t++)
#pragma unroll
          for (int r = 0; r < 4; r++) {
            const T b = Type<T>::tanh_of(s[t][r] * part);
            if (TANH) bent[t][r] = b;
            s[t][r] = b * cap;
          }
      } else {
#pragma unroll
        for (int t = 0; t < 2; t++)
#pragma unroll
          for (int r = 0; r < 4; r++) {
            const T x = s[t][r] * part, u = s[t][r] * mul, share = Type<T>::tanh_share(x);
            if (TANH) bent[t][r] = fma(x, share, x);
            s[t][r] = fma(u, share, u);
          }
      }
    } else {
#pragma unroll
      for (int t = 0; t < 2; t++) s[t] *= mul;
    }
    if (sloped) {
      const T d = (T)apart;
#pragma unroll
      for (int t = 0; t < 2; t++)
#pragma unroll
        for (int r = 0; r < 4; r++) s[t][r] -= slope * abs_of(d - (T)tile_row<T>(t, r));
    }
  }
  static __device__ __forceinline__ T abs_of(T x) { return x < 0 ? -x : x; }
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
  // Position i's document, of which `doc` is the one that LDS holds where there are documents.
  __device__ __forceinline__ int in(int i, int doc) const { return documents ? doc : i < length ? 0 : -1; }
  // With the documents of both at hand; those of no sequence are negative.
  __device__ __forceinline__ bool sees(int i, int di, int j, int dj) const { return di >= 0 && di == dj && (!causal || j <= i || j < prefix); }
  // Whether every query from i on that there is sees every key of [j, end).
  __device__ __forceinline__ bool all_see(int i, int end) const { return !documents && end <= length && (!causal || end - 1 <= i || end <= prefix); }
  // Keys [0, this) hold every one that a query before `end` sees.
  __device__ __forceinline__ int keys_to(int end) const { return min(causal ? max(end, prefix) : length, length); }
  // Queries [this, length) hold every one that sees a key from j on.
  __device__ __forceinline__ int queries_from(int j) const { return causal && j >= prefix ? j : 0; }
};

__device__ __forceinline__ int wave_min(int x) {
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) x = min(x, __shfl_xor(x, o));
  return x;
}

// The stages of the other side, [from, end) of them, that may hold a position of the documents of a
// block's rows; all of them without documents. Every thread of the block calls it alike.
template <class G>
struct Stages {
  const Sight& sight;
  int low, high;  // documents of the rows
  int from, end;
  int chunk = -1;  // of 64 stages
  uint64_t live = 0;
  uint64_t* shared;
  static constexpr int STAGE = G::STAGE, WAVES = G::WAVES;
  __device__ __forceinline__ Stages(const Sight& s, int rows, int from_, int end_, uint64_t* shared_) : sight(s), from(from_), end(end_), shared(shared_) {
    if (!sight.documents) return;
    const int d = sight.document(rows + (int)(threadIdx.x & 63) % G::ROWS);
    low = wave_min(d < 0 ? 0x7fffffff : d);
    high = -wave_min(-max(d, -1));
  }
  // Each wave looks at every WAVES-th stage of the chunk; a wave's lanes take its positions.
  __device__ __forceinline__ void look(int c) {
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    uint64_t mine = 0;
    for (int k = wave; k < 64; k += WAVES) {
      const int first = (c * 64 + k) * STAGE;
      if (c * 64 + k < from || c * 64 + k >= end) continue;
      int least = 0x7fffffff, most = -1;
      for (int p = lane; p < STAGE; p += 64) {
        const int d = sight.document(first + p);
        least = min(least, d < 0 ? 0x7fffffff : d);
        most = max(most, d);
      }
      if (wave_min(least) <= high && -wave_min(-most) >= low) mine |= 1ull << k;
    }
    __syncthreads();
    if (lane == 0) shared[wave] = mine;
    __syncthreads();
    live = 0;
    for (int w = 0; w < WAVES; w++) live |= shared[w];
    chunk = c;
  }
  // The first live stage from k on, or `end`.
  __device__ __forceinline__ int at(int k) {
    if (!sight.documents) return min(k, end);
    while (k < end) {
      if (k / 64 != chunk) look(k / 64);
      const uint64_t left = live >> (k % 64);
      if (left) return k + __builtin_ctzll(left);
      k = (k / 64 + 1) * 64;
    }
    return end;
  }
};

// Sixteen bytes of a buffer, and one value, 0 past its end. The whole place is the vector offset: a
// scalar one past the end would be taken from the buffer's size without a check.
template <class T>
__device__ __forceinline__ typename Type<T>::vec buffer_vec(__amdgpu_buffer_rsrc_t from, uint32_t at) {
  typedef uint32_t words __attribute__((ext_vector_type(4)));
  const words w = __builtin_amdgcn_raw_buffer_load_b128(from, (int)at, 0, 0);
  return __builtin_bit_cast(typename Type<T>::vec, w);
}
__device__ __forceinline__ float buffer_value(__amdgpu_buffer_rsrc_t from, uint32_t at, float) {
  return __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(from, (int)at, 0, 0));
}
__device__ __forceinline__ double buffer_value(__amdgpu_buffer_rsrc_t from, uint32_t at, double) {
  typedef uint32_t words __attribute__((ext_vector_type(2)));
  const words w = __builtin_amdgcn_raw_buffer_load_b64(from, (int)at, 0, 0);
  return __builtin_bit_cast(double, w);
}

// Makes infinities and NaN among a thread's N vectors 0; whether there were any. Rows to be weighed go
// through it, and what a seen one of them does is made up for after the loop, in `for_odd_rows`: there is
// no place for it inside (it cost the forward of heads of 128 a third, in registers).
template <class T, int N, class... More>
__device__ __forceinline__ bool make_finite(typename Type<T>::vec (&x)[N], More&... more) {
  T z = 0;
  auto look = [&](auto& v) {
#pragma unroll
    for (int i = 0; i < N; i++)
#pragma unroll
      for (int j = 0; j < Type<T>::V; j++) z = fma(v[i][j], (T)0, z);
  };
  auto clear = [&](auto& v) {
#pragma unroll
    for (int i = 0; i < N; i++)
#pragma unroll
      for (int j = 0; j < Type<T>::V; j++) v[i][j] = v[i][j] * (T)0 == 0 ? v[i][j] : (T)0;
  };
  look(x);
  (look(more), ...);
  const bool odd = z != z;
  if (odd) {
    clear(x);
    (clear(more), ...);
  }
  return odd;
}

// Calls f(n) for each n of [from, to) whose row at(n) of `head` values holds an infinity or NaN; a wave's
// lanes look at 64 rows at once. `at` gives nullptr where there is no row.
template <class At, class F>
__device__ __forceinline__ void for_odd_rows(int from, int to, uint32_t head, const At& at, const F& f) {
  for (int base = from; base < to; base += 64) {
    const int n = base + (int)(threadIdx.x & 63);
    bool odd = false;
    if (n < to)
      if (const auto* row = at(n))
        for (uint32_t d = 0; d < head; d++) odd |= row[d] * 0 != 0;
    for (uint64_t left = __ballot(odd); left; left &= left - 1) f(base + (int)__builtin_ctzll(left));
  }
}
// To a lane's share of the result of a row that sees it, a row's infinities and NaN, whatever its weight.
template <class T, int HD>
__device__ __forceinline__ void add_odd(const T* row, int g, uint32_t head, typename Type<T>::acc* acc) {
  constexpr int ND = HD / 16;
#pragma unroll
  for (int n = 0; n < ND; n++)
#pragma unroll
    for (int r = 0; r < 4; r++) {
      const uint32_t d = (uint32_t)(Type<T>::row_of(r, g) * ND + n);
      const T x = d < head ? row[d] : (T)0;
      acc[n][r] += x * 0 == 0 ? (T)0 : x;
    }
}

// N rows of one operand on their way to LDS, 16 bytes a thread and step. They are read as a buffer that
// ends with the sequence, and columns past the head from past its end, so that what does not belong
// is 0 as it arrives, with no selection that would wait for it.
template <class T, int HD, class G, int N = G::STAGE>
struct Staged {
  static constexpr int V = Type<T>::V, NT = G::NT, LANES = HD / V, PER = N * LANES / NT;
  // Where all of a thread's steps have one column, its place is held once.
  static constexpr bool EVEN = NT % LANES == 0;
  static_assert(PER * NT == N * LANES, "whole steps");
  typedef typename Type<T>::vec vec;
  static constexpr uint32_t OUTSIDE = 0x80000000u;  // past a stage's rows (lower_attend)
  vec x[PER];
  uint32_t at[EVEN ? 1 : PER], pitch;
  static __device__ __forceinline__ int row(int i) { return ((int)threadIdx.x + i * NT) / LANES; }
  static __device__ __forceinline__ uint32_t column(int i) { return (uint32_t)(((int)threadIdx.x + i * NT) % LANES) * V; }
  // `step` values from one row to the next.
  __device__ __forceinline__ Staged(int64_t step, uint32_t head) : pitch((uint32_t)step * (uint32_t)sizeof(T)) {
#pragma unroll
    for (int i = 0; i < (EVEN ? 1 : PER); i++) at[i] = column(i) < head ? (uint32_t)row(i) * pitch + column(i) * (uint32_t)sizeof(T) : OUTSIDE;
  }
  // The rows from `p` on, of which `rows` are there.
  __device__ __forceinline__ void load(const T* p, int rows, uint32_t head, bool whole) {
    const uint64_t bytes = rows > 0 ? (uint64_t)(min(rows, N) - 1) * pitch + head * sizeof(T) : 0;
    const __amdgpu_buffer_rsrc_t from = __builtin_amdgcn_make_buffer_rsrc((void*)p, 0, (int)bytes, 0x00027000);
#pragma unroll
    for (int i = 0; i < PER; i++) {
      const uint32_t place = EVEN ? at[0] + (uint32_t)(i * (NT / LANES)) * pitch : at[i];
      if (whole) {
        x[i] = buffer_vec<T>(from, place);
      } else {
#pragma unroll
        for (uint32_t j = 0; j < V; j++)
          x[i][j] = buffer_value(from, column(i) + j < head ? place + j * (uint32_t)sizeof(T) : OUTSIDE, (T)0);
      }
    }
  }
  __device__ __forceinline__ void store(T* xs) const {
#pragma unroll
    for (int i = 0; i < PER; i++) *(vec*)(xs + row(i) * PITCH<T, HD> + (int)column(i)) = x[i];
  }
  // Makes 0, once they are there, the rows whose entry in `docs` is negative.
  static __device__ __forceinline__ void clear(T* xs, const int* docs) {
#pragma unroll
    for (int i = 0; i < PER; i++)
      if (docs[row(i)] < 0) *(vec*)(xs + row(i) * PITCH<T, HD> + (int)column(i)) = 0;
  }
};

// The end of a stage's arrival in LDS, for the whole block: its documents, where there are any, go to
// `docs`, and the rows of none are made 0.
template <class T, int HD, class G>
__device__ __forceinline__ void settle(const Sight& sight, int first, int doc, int* docs, T* xs, T* ys) {
  if (!sight.documents) {
    __syncthreads();
    return;
  }
  const bool mine = threadIdx.x < G::STAGE;
  if (mine) docs[threadIdx.x] = doc;
  if (__syncthreads_or(mine && doc < 0 && first + (int)threadIdx.x < sight.length)) {
    Staged<T, HD, G>::clear(xs, docs);
    Staged<T, HD, G>::clear(ys, docs);
    __syncthreads();
  }
}

// Rows of two operands anywhere in memory on their way to LDS; their places in both, and whether they are
// there, lie in LDS. Loads are of rows and columns that there are, so the places of rows that are not may
// be any that can be read; what does not belong is made 0 as it is stored.
template <class T, int HD, class G>
struct Gathered {
  static constexpr int V = Type<T>::V, NT = G::NT, PER = G::STAGE * HD / V / NT;
  static_assert(PER * NT * V == G::STAGE * HD && PER <= 32, "whole steps");
  typedef typename Type<T>::vec vec;
  vec x[PER], y[PER];
  uint32_t off;  // bit i: step i is not there
  static __device__ __forceinline__ int row(int i) { return ((int)threadIdx.x + i * NT) / (HD / V); }
  static __device__ __forceinline__ uint32_t column(int i) { return (uint32_t)(((int)threadIdx.x + i * NT) % (HD / V)) * V; }
  __device__ __forceinline__ void load(const T* xs, const T* ys, const int64_t* x_at, const int64_t* y_at, const int* there, uint32_t head, bool whole) {
    off = 0;
#pragma unroll
    for (int i = 0; i < PER; i++) {
      const T *u_row = xs + x_at[row(i)], *v_row = ys + y_at[row(i)];
      const uint32_t c = column(i);
      off |= there[row(i)] && c < head ? 0u : 1u << i;
      if (whole) {
        const uint32_t d = c < head ? c : 0;
        x[i] = *(const vec*)(u_row + d);
        y[i] = *(const vec*)(v_row + d);
      } else {
#pragma unroll
        for (uint32_t j = 0; j < V; j++) {
          const uint32_t d = c + j < head ? c + j : 0;
          const T u = u_row[d], v = v_row[d];
          x[i][j] = c + j < head ? u : (T)0;
          y[i][j] = c + j < head ? v : (T)0;
        }
      }
    }
  }
  __device__ __forceinline__ void store(T* xs, T* ys) const {
#pragma unroll
    for (int i = 0; i < PER; i++) {
      const int o = row(i) * PITCH<T, HD> + (int)column(i);
      const bool none = off >> i & 1;
      vec u = x[i], v = y[i];
#pragma unroll
      for (int j = 0; j < V; j++) {
        u[j] = none ? (T)0 : u[j];
        v[j] = none ? (T)0 : v[j];
      }
      *(vec*)(xs + o) = u;
      *(vec*)(ys + o) = v;
    }
  }
};

// A block's head and tile of rows. Heads of a batch lie next to each other, so that blocks of one head
// meet in the same L2 where their number is a multiple of the eight dies. Under a causal order the tiles
// with the most work come first (`last_first`: the last), so that short ones fill up at the end; where
// two blocks share a CU (`paired`), every second round of as many blocks as there are CUs runs the other
// way, since they all start at once and a long and a short one are to meet.
constexpr uint32_t CUS = 256;
struct Place {
  uint32_t b, h, tile;
  __device__ __forceinline__ Place(uint32_t at, uint32_t batch, uint32_t heads, uint32_t tiles, bool last_first, bool paired) {
    const uint32_t blocks = batch * heads * tiles, round = at / CUS * CUS;
    if (paired && round / CUS % 2 == 1) at = round + min(CUS, blocks - round) - 1 - (at - round);
    const uint32_t bh = at % (batch * heads), n = at / (batch * heads);
    b = bh / heads;
    h = bh % heads;
    tile = last_first ? tiles - 1 - n : n;
  }
};

// The running softmax of a row over its keys: a bound that its scores stay near (to base 2), the sum (of
// the lane's own keys until the end) and the weighed values. The bound is the largest score when it was
// last moved; it moves once a score is more than 2^8 times as heavy, and then what there is is scaled.
template <class T, int HD>
struct Running {
  typedef typename Type<T>::acc acc;
  acc out[HD / 16];
  T top = -(T)__builtin_huge_val(), sum = 0;
  __device__ __forceinline__ Running() {
#pragma unroll
    for (int n = 0; n < HD / 16; n++) out[n] = acc{0, 0, 0, 0};
  }
  __device__ __forceinline__ void scale(T by) {
    sum *= by;
#pragma unroll
    for (int n = 0; n < HD / 16; n++) out[n] *= by;
  }
  // What the bound is to scores: a row that has seen nothing keeps weights of 0.
  static __device__ __forceinline__ T base(T top) { return top == -(T)__builtin_huge_val() ? (T)0 : top; }
  // Takes in two tiles of scores, minus infinity where a key is not seen, and leaves their weights.
  __device__ __forceinline__ void add(acc* s) {
    T most = s[0][0];
#pragma unroll
    for (int t = 0; t < 2; t++)
#pragma unroll
      for (int r = 0; r < 4; r++) most = Type<T>::max_of(most, s[t][r]);
    most = row_max(most) * (T)1.4426950408889634;
    if (__ballot(most > top + 8) != 0) {
      const T next = Type<T>::max_of(top, most);
      scale(Type<T>::exp2_of(top - base(next)));
      top = next;
    }
    const T at = base(top);
#pragma unroll
    for (int t = 0; t < 2; t++)
#pragma unroll
      for (int r = 0; r < 4; r++) {
        s[t][r] = weight(s[t][r], at);
        sum += s[t][r];
      }
  }
};

// The sets' shares of a lane's results, added up in set 0 in the sets' order through LDS; `buffer`
// holds G::ROWS * HD values.
template <class T, int HD, class G>
__device__ __forceinline__ void join(typename Type<T>::acc* out, T* buffer, int set) {
  constexpr int N = 64 * G::RW;
  const int at = (int)threadIdx.x % N;
#pragma unroll
  for (int other = 1; other < G::SETS; other++) {
    __syncthreads();
    if (set == other)
#pragma unroll
      for (int n = 0; n < HD / 16; n++)
#pragma unroll
        for (int r = 0; r < 4; r++) buffer[(n * 4 + r) * N + at] = out[n][r];
    __syncthreads();
    if (set == 0)
#pragma unroll
      for (int n = 0; n < HD / 16; n++)
#pragma unroll
        for (int r = 0; r < 4; r++) out[n][r] += buffer[(n * 4 + r) * N + at];
  }
}
// The same of running softmaxes: afterwards set 0 has the whole.
template <class T, int HD, class G>
__device__ __forceinline__ void join(Running<T, HD>& run, T* buffer, T* tops, T* sums, int set) {
  constexpr int N = 64 * G::RW;
  const int at = (int)threadIdx.x % N;
  tops[threadIdx.x] = run.top;
  sums[threadIdx.x] = run.sum;
  __syncthreads();
  T top = tops[at];
#pragma unroll
  for (int other = 1; other < G::SETS; other++) top = Type<T>::max_of(top, tops[other * N + at]);
  const T base = Running<T, HD>::base(top);
  run.scale(Type<T>::exp2_of(run.top - base));
  run.top = top;
  run.sum = 0;
#pragma unroll
  for (int other = 0; other < G::SETS; other++) run.sum += sums[other * N + at] * Type<T>::exp2_of(tops[other * N + at] - base);
  join<T, HD, G>(run.out, buffer, set);
}

// A lane's set, its row among the block's and the wave's first row.
template <int RW>
struct Lane {
  int l16, g, set, row, first;
  __device__ __forceinline__ Lane() {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    l16 = lane & 15;
    g = lane >> 4;
    set = wave / RW;
    first = wave % RW * 16;
    row = first + l16;
  }
};

// A block's own rows, in registers or in LDS (Geo::KEPT).
template <class T, int HD, class G>
struct Own {
  T* kept;
  Registers<T, HD> held;
  __device__ __forceinline__ Own(T* k) : kept(k) {}
  __device__ __forceinline__ void set(const T* x, const Lane<G::RW>& l) {
    if constexpr (G::KEPT) {
      if (l.set == 0)
#pragma unroll
        for (int n = 0; n < HD / 16; n++)
#pragma unroll
          for (int j = 0; j < 4; j++) kept[l.row * PITCH<T, HD> + n * 16 + 4 * l.g + j] = x[4 * n + j];
    } else {
#pragma unroll
      for (int n = 0; n < HD / 4; n++) held.frag[n] = x[n];
    }
  }
  __device__ __forceinline__ auto of(const Lane<G::RW>& l) const {
    if constexpr (G::KEPT) return Kept<T, HD>{kept + l.row * PITCH<T, HD> + 4 * l.g};
    else return held;
  }
};

// Two products a pair. Bound by the matrix unit and the vector unit, which share a SIMD's issue: of the
// causal case's 118 us (73 TFLOP/s) the first is busy for 57 % and the second, with some 220 instructions
// for a wave's 16 x 32 scores, for 33 %. Heads of 128 over 5000 positions: 332 us, 77 TFLOP/s.
template <class T, int HD, int RW>
__global__ void __launch_bounds__((Geo<T, HD, RW>::NT), (Geo<T, HD, RW>::FORWARD)) k_attend(AttendArgs a) {
  typedef Geo<T, HD, RW> G;
  typedef typename Type<T>::acc acc;
  constexpr int STAGE = G::STAGE, SETS = G::SETS, NT = G::NT, ROWS = G::ROWS;
  __shared__ __align__(16) T smem[2 * STAGE * PITCH<T, HD>];
  __shared__ __align__(16) int docs[STAGE];
  __shared__ T tops[SETS > 1 ? NT : 1], sums[SETS > 1 ? NT : 1];
  __shared__ uint64_t found[NT / 64];
  T *ks = smem, *vs = smem + STAGE * PITCH<T, HD>;
  const Place at(blockIdx.x, a.batch, a.heads, a.tiles, a.causal, G::FORWARD * 4 == 2 * G::WAVES);
  const Sight sight(a, at.b);
  const Lane<RW> l;
  const int begin = (int)at.tile * ROWS, i = begin + l.row, i0 = begin + l.first;
  const uint32_t kh = at.h / (a.heads / a.keys);
  const bool whole = a.head % Type<T>::V == 0;
  const Scorer<T> scorer(a, at.h);
  const int di = sight.document(i);
  Registers<T, HD> own;
  row_frag<T, HD>(di >= 0 ? (const T*)a.q + ((int64_t)at.b * a.length + i) * a.q_row + at.h * a.head : nullptr, l.g, a.head, whole, own.frag);
  const T *kb = (const T*)a.k + (int64_t)at.b * a.length * a.k_row + kh * a.head, *vb = (const T*)a.v + (int64_t)at.b * a.length * a.k_row + kh * a.head;
  const int end = begin < sight.length ? sight.keys_to(min(begin + ROWS, sight.length)) : 0;
  const int seen_to = i0 < sight.length ? sight.keys_to(min(i0 + 16, sight.length)) : 0;
  Stages<G> stages(sight, begin, 0, (end + STAGE - 1) / STAGE, found);
  Running<T, HD> run;
  bool odd = false;
  Staged<T, HD, G> next_k(a.k_row, a.head), next_v(a.k_row, a.head);
  int doc = 0;
  auto load = [&](int stage) {
    const int first = stage * STAGE;
    next_k.load(kb + first * a.k_row, sight.length - first, a.head, whole);
    next_v.load(vb + first * a.k_row, sight.length - first, a.head, whole);
    if (sight.documents && threadIdx.x < STAGE) doc = sight.document(first + (int)threadIdx.x);
  };
  int k = stages.at(0);
  if (k < stages.end) load(k);
  while (k < stages.end) {
    __syncthreads();
    odd |= make_finite<T>(next_v.x);
    next_k.store(ks);
    next_v.store(vs);
    settle<T, HD, G>(sight, k * STAGE, doc, docs, ks, vs);
    const int here = k, first = here * STAGE + l.set * TILE;
    k = stages.at(here + 1);
    if (k < stages.end) load(k);
    if (first >= seen_to) continue;
    acc s[2];
    score<T, HD>(ks + l.set * TILE * PITCH<T, HD>, l.l16, l.g, own, s);
    scorer.template operator()<false>(s, nullptr, i - (first + Type<T>::row_of(0, l.g)));
    if (!sight.all_see(i0, first + TILE)) {
#pragma unroll
      for (int t = 0; t < 2; t++)
#pragma unroll
        for (int r = 0; r < 4; r++) {
          const int row = 16 * t + Type<T>::row_of(r, l.g);
          s[t][r] = sight.sees(i, di, first + row, sight.in(first + row, docs[l.set * TILE + row])) ? s[t][r] : -(T)__builtin_huge_val();
        }
    }
    run.add(s);
    weigh<T, HD>(vs + l.set * TILE * PITCH<T, HD>, l.l16, l.g, s, run.out);
  }
  run.sum = row_sum(run.sum);
  if constexpr (SETS > 1) join<T, HD, G>(run, smem, tops, sums, l.set);
  if (__syncthreads_or(odd) && l.set == 0) {
    for_odd_rows(0, seen_to, a.head, [&](int j) { return vb + (int64_t)j * a.k_row; }, [&](int j) {
      if (sight.sees(i, di, j, sight.document(j))) add_odd<T, HD>(vb + (int64_t)j * a.k_row, l.g, a.head, run.out);
    });
  }
  if (l.set != 0 || i >= (int)a.length) return;
  const uint64_t row = ((uint64_t)at.b * a.length + i) * a.heads + at.h;
  const bool none = run.sum == 0 || di < 0;
  if (a.y) put_row<T, HD>((T*)a.y + row * a.head, l.g, a.head, run.out, 1 / run.sum, none);
  // For the backward, which so forms the weights that were used here: the bound and the sum's
  // reciprocal; of a query that sees nothing the type's largest value and 0, weights of 0. (With the
  // logarithm of the sum in their place, 12 of 2^-24 each, the gradient of q was a tenth further off.)
  if (a.sums && l.g == 0) {
    const uint64_t stat = ((uint64_t)at.b * a.heads + at.h) * a.length + i;
    ((T*)a.sums)[stat] = none ? Type<T>::MOST : run.top;
    ((T*)a.sums)[stat + (uint64_t)a.batch * a.heads * a.length] = none ? (T)0 : 1 / run.sum;
  }
}

// The gradient of q, of the slopes, and each query's dy.y for the kernel of the others. Three products a
// pair, bound as the forward is: 190 us in the causal case, 68 TFLOP/s, the matrix unit busy for 59 %.
template <class T, int HD, int RW>
__global__ void __launch_bounds__((Geo<T, HD, RW>::NT), (Geo<T, HD, RW>::BACKWARD)) k_attend_dq(AttendArgs a) {
  typedef Geo<T, HD, RW> G;
  typedef typename Type<T>::acc acc;
  constexpr int STAGE = G::STAGE, SETS = G::SETS, NT = G::NT, ROWS = G::ROWS;
  __shared__ __align__(16) T smem[2 * STAGE * PITCH<T, HD>];
  __shared__ __align__(16) T kept[G::KEPT ? 2 * ROWS * PITCH<T, HD> : 4];
  __shared__ __align__(16) int docs[STAGE];
  __shared__ T waves[NT / 64], lefts[SETS > 1 ? SETS * ROWS : 1];
  __shared__ uint64_t found[NT / 64];
  T *ks = smem, *vs = smem + STAGE * PITCH<T, HD>;
  const Place at(blockIdx.x, a.batch, a.heads, a.tiles, a.causal, G::BACKWARD * 4 == 2 * G::WAVES);
  const Sight sight(a, at.b);
  const Lane<RW> l;
  const int begin = (int)at.tile * ROWS, i = begin + l.row, i0 = begin + l.first;
  const uint32_t kh = at.h / (a.heads / a.keys);
  const bool whole = a.head % Type<T>::V == 0;
  const Scorer<T> scorer(a, at.h);
  const int di = sight.document(i);
  const uint64_t row = ((uint64_t)at.b * a.length + i) * a.heads + at.h, stat = ((uint64_t)at.b * a.heads + at.h) * a.length + i;
  const T *qb = (const T*)a.q + (int64_t)at.b * a.length * a.q_row + at.h * a.head, *gb = (const T*)a.dy + ((int64_t)at.b * a.length * a.heads + at.h) * a.head;
  const T* yb = (const T*)a.y_in + ((int64_t)at.b * a.length * a.heads + at.h) * a.head;
  T dot = 0;
  Own<T, HD, G> own(kept), grad(kept + (G::KEPT ? ROWS * PITCH<T, HD> : 0));
  {
    // In registers for dy.y; the ones in LDS are there after the first stage's barriers.
    T y[HD / 4], x[HD / 4];
    row_frag<T, HD>(di >= 0 ? yb + (int64_t)i * a.heads * a.head : nullptr, l.g, a.head, whole, y);
    row_frag<T, HD>(di >= 0 ? gb + (int64_t)i * a.heads * a.head : nullptr, l.g, a.head, whole, x);
    // On the matrix instructions in the order of the products dy.v, so that where one key is all that a
    // query sees both are the same number, and near it nearly so: their difference is the gradient.
    acc all = {0, 0, 0, 0}, late = {0, 0, 0, 0};
#pragma unroll
    for (int n = 0; n < HD / 8; n++) {
      all = Type<T>::mfma(y[n], x[n], all);
      late = Type<T>::mfma(y[n + HD / 8], x[n + HD / 8], late);
    }
    dot = Type<T>::diagonal(all + late, l.l16);
    grad.set(x, l);
    row_frag<T, HD>(di >= 0 ? qb + (int64_t)i * a.q_row : nullptr, l.g, a.head, whole, x);
    own.set(x, l);
  }
  const T top = di >= 0 ? ((const T*)a.sums_in)[stat] : Type<T>::MOST, by = di >= 0 ? ((const T*)a.sums_in)[stat + (uint64_t)a.batch * a.heads * a.length] : (T)0;
  const T *kb = (const T*)a.k + (int64_t)at.b * a.length * a.k_row + kh * a.head, *vb = (const T*)a.v + (int64_t)at.b * a.length * a.k_row + kh * a.head;
  const int end = begin < sight.length ? sight.keys_to(min(begin + ROWS, sight.length)) : 0;
  const int seen_to = i0 < sight.length ? sight.keys_to(min(i0 + 16, sight.length)) : 0;
  Stages<G> stages(sight, begin, 0, (end + STAGE - 1) / STAGE, found);
  acc out[HD / 16];
#pragma unroll
  for (int n = 0; n < HD / 16; n++) out[n] = acc{0, 0, 0, 0};
  T dslope = 0, left = 0;
  bool odd = false;
  Staged<T, HD, G> next_k(a.k_row, a.head), next_v(a.k_row, a.head);
  int doc = 0;
  auto load = [&](int stage) {
    const int first = stage * STAGE;
    next_k.load(kb + first * a.k_row, sight.length - first, a.head, whole);
    next_v.load(vb + first * a.k_row, sight.length - first, a.head, whole);
    if (sight.documents && threadIdx.x < STAGE) doc = sight.document(first + (int)threadIdx.x);
  };
  int k = stages.at(0);
  if (k < stages.end) load(k);
  while (k < stages.end) {
    __syncthreads();
    odd |= make_finite<T>(next_k.x);
    next_k.store(ks);
    next_v.store(vs);
    settle<T, HD, G>(sight, k * STAGE, doc, docs, ks, vs);
    const int here = k, first = here * STAGE + l.set * TILE;
    k = stages.at(here + 1);
    if (k < stages.end) load(k);
    if (first >= seen_to) continue;
    acc s[2], dp[2], bent[2];
    score<T, HD>(ks + l.set * TILE * PITCH<T, HD>, l.l16, l.g, own.of(l), s);
    score<T, HD>(vs + l.set * TILE * PITCH<T, HD>, l.l16, l.g, grad.of(l), dp);
    const int apart = i - (first + Type<T>::row_of(0, l.g));
    scorer.template operator()<true>(s, bent, apart);
    if (!sight.all_see(i0, first + TILE)) {
#pragma unroll
      for (int t = 0; t < 2; t++)
#pragma unroll
        for (int r = 0; r < 4; r++) {
          const int row_in = 16 * t + Type<T>::row_of(r, l.g);
          const bool sees = sight.sees(i, di, first + row_in, sight.in(first + row_in, docs[l.set * TILE + row_in]));
          s[t][r] = sees ? s[t][r] : -(T)__builtin_huge_val();
          dp[t][r] = sees ? dp[t][r] : (T)0;
          if (scorer.capped) bent[t][r] = sees ? bent[t][r] : (T)0;
        }
    }
#pragma unroll
    for (int t = 0; t < 2; t++)
#pragma unroll
      for (int r = 0; r < 4; r++) s[t][r] = weight(s[t][r], top) * by;
    if (seen_to <= TILE) {
      // All keys of the wave's queries are in this tile: dy.y as the mean of the products dy.v that it is
      // of few, whose roundings then meet in the differences.
      T mean = 0;
#pragma unroll
      for (int t = 0; t < 2; t++)
#pragma unroll
        for (int r = 0; r < 4; r++) mean += s[t][r] * (s[t][r] == 0 ? (T)0 : dp[t][r]);
      dot = row_sum(mean);
    }
#pragma unroll
    for (int t = 0; t < 2; t++)
#pragma unroll
      for (int r = 0; r < 4; r++) {
        s[t][r] *= dp[t][r] - dot;
        left += s[t][r];
      }
    if (scorer.sloped) {
#pragma unroll
      for (int t = 0; t < 2; t++)
#pragma unroll
        for (int r = 0; r < 4; r++) dslope -= s[t][r] * Scorer<T>::abs_of((T)apart - (T)tile_row<T>(t, r));
    }
    if (scorer.capped) {
#pragma unroll
      for (int t = 0; t < 2; t++) s[t] -= s[t] * (bent[t] * bent[t]);
    }
    weigh<T, HD>(ks + l.set * TILE * PITCH<T, HD>, l.l16, l.g, s, out);
  }
  if (__syncthreads_or(odd)) {
    // The key's scores are no numbers either: nothing is left of a query that sees one.
    bool hit = false;
    for_odd_rows(0, seen_to, a.head, [&](int j) { return kb + (int64_t)j * a.k_row; }, [&](int j) { hit |= sight.sees(i, di, j, sight.document(j)); });
    if (hit) {
      left = dslope = (T)__builtin_nan("");
#pragma unroll
      for (int n = 0; n < HD / 16; n++) out[n] = acc{left, left, left, left};
    }
  }
  // What the differences leave over goes to dy.y, as the gradients of k and v take it: their sum over a
  // query's keys is 0.
  left = row_sum(left);
  if constexpr (SETS > 1) {
    lefts[l.set * ROWS + l.row] = left;
    __syncthreads();
    left = 0;
#pragma unroll
    for (int other = 0; other < SETS; other++) left += lefts[other * ROWS + l.row];
  }
  if (l.set == 0 && l.g == 0 && i < (int)a.length) ((T*)a.workspace)[stat] = di < 0 ? (T)0 : dot + left;
  if constexpr (SETS > 1) join<T, HD, G>(out, smem, l.set);
  if (a.dq && l.set == 0 && i < (int)a.length)
    put_row<T, HD>((T*)a.dq + ((int64_t)at.b * a.length + i) * a.q_row + at.h * a.head, l.g, a.head, out, (T)a.scale, di < 0);
  if (a.dslopes_rows) {
    dslope = rg_wave_sum(di < 0 ? (T)0 : dslope);
    if ((threadIdx.x & 63) == 0) waves[threadIdx.x >> 6] = dslope;
    __syncthreads();
    if (threadIdx.x == 0) {
      dslope = waves[0];
      for (int w = 1; w < NT / 64; w++) dslope += waves[w];
      ((T*)a.dslopes_rows)[((uint64_t)at.b * a.tiles + at.tile) * a.heads + at.h] = dslope;
    }
  }
}

// The gradients of k and v: a block's 64 keys against the queries of the heads that read them, all
// of a group's or, where that leaves too few blocks, a part of them, whose sums k_attend_parts adds up.
// Four products a pair: 228 us in the causal case, 75 TFLOP/s, the matrix unit busy for 60 %. Scores and
// dy.v are formed here a second time; one kernel for all five products would have to add to dq from many
// blocks, with atomics in an order of their own or a row of partial sums for every 64 keys.
template <class T, int HD, int RW>
__global__ void __launch_bounds__((Geo<T, HD, RW>::NT), (Geo<T, HD, RW>::BACKWARD)) k_attend_dkv(AttendArgs a) {
  typedef Geo<T, HD, RW> G;
  typedef typename Type<T>::acc acc;
  constexpr int STAGE = G::STAGE, SETS = G::SETS, NT = G::NT, ROWS = G::ROWS;
  __shared__ __align__(16) T smem[2 * STAGE * PITCH<T, HD>];
  __shared__ __align__(16) T kept[G::KEPT ? 2 * ROWS * PITCH<T, HD> : 4];
  __shared__ __align__(16) int docs[STAGE];
  __shared__ __align__(16) T tops[STAGE];
  __shared__ __align__(16) T sums[STAGE];
  __shared__ __align__(16) T dots[STAGE];
  __shared__ uint64_t found[NT / 64];
  T *qs = smem, *gs = smem + STAGE * PITCH<T, HD>;
  const Place at(blockIdx.x, a.batch, a.keys * a.parts, a.tiles, false, G::BACKWARD * 4 == 2 * G::WAVES);
  const uint32_t kh = at.h / a.parts, part = at.h % a.parts, group = a.heads / a.keys, per_part = group / a.parts;
  const Sight sight(a, at.b);
  const Lane<RW> l;
  const int begin = (int)at.tile * ROWS, j = begin + l.row, j0 = begin + l.first;
  const bool whole = a.head % Type<T>::V == 0;
  const int dj = sight.document(j);
  const int64_t key = ((int64_t)at.b * a.length + j) * a.k_row + kh * a.head;
  Own<T, HD, G> own(kept), value(kept + (G::KEPT ? ROWS * PITCH<T, HD> : 0));
  {
    T x[HD / 4];
    row_frag<T, HD>(dj >= 0 ? (const T*)a.k + key : nullptr, l.g, a.head, whole, x);
    own.set(x, l);
    row_frag<T, HD>(dj >= 0 ? (const T*)a.v + key : nullptr, l.g, a.head, whole, x);
    value.set(x, l);
  }
  acc dk[HD / 16], dv[HD / 16];
#pragma unroll
  for (int n = 0; n < HD / 16; n++) dk[n] = dv[n] = acc{0, 0, 0, 0};
  const int end = begin < sight.length ? (sight.length + STAGE - 1) / STAGE : 0;
  Stages<G> stages(sight, begin, min(sight.queries_from(begin) / STAGE, end), end, found);
  // The wave's keys are seen by no query before this.
  const int seen_from = sight.queries_from(j0);
  uint32_t h = kh * group + part * per_part;
  const uint32_t last = h + per_part;
  Staged<T, HD, G> next_q(a.q_row, a.head), next_g((int64_t)a.heads * a.head, a.head);
  int doc = 0;
  T top = 0, sum = 0, dot = 0;
  bool odd = false;
  auto load = [&](uint32_t of, int stage) {
    const int first = stage * STAGE;
    const int64_t t = (int64_t)at.b * a.length + first;
    next_q.load((const T*)a.q + t * a.q_row + of * a.head, sight.length - first, a.head, whole);
    next_g.load((const T*)a.dy + (t * a.heads + of) * a.head, sight.length - first, a.head, whole);
    if (threadIdx.x < STAGE) {
      const int i = first + (int)threadIdx.x;
      doc = sight.document(i);
      const uint64_t stat = ((uint64_t)at.b * a.heads + of) * a.length + min(i, sight.length - 1);
      top = ((const T*)a.sums_in)[stat];
      sum = ((const T*)a.sums_in)[stat + (uint64_t)a.batch * a.heads * a.length];
      dot = ((const T*)a.workspace)[stat];
    }
  };
  int k = stages.at(stages.from);
  const bool some = k < stages.end;
  if (G::NARROW && some) load(h, k);
  while (some && h < last) {
    if (!G::NARROW) load(h, k);  // its registers are the accumulators' while it computes
    __syncthreads();
    odd |= make_finite<T>(next_q.x, next_g.x);
    next_q.store(qs);
    next_g.store(gs);
    if (threadIdx.x < STAGE) {
      tops[threadIdx.x] = doc < 0 ? Type<T>::MOST : top;  // weights of 0
      sums[threadIdx.x] = doc < 0 ? (T)0 : sum;
      dots[threadIdx.x] = doc < 0 ? (T)0 : dot;
    }
    settle<T, HD, G>(sight, k * STAGE, doc, docs, qs, gs);
    const int here = k, first = here * STAGE + l.set * TILE;
    const Scorer<T> scorer(a, h);
    k = stages.at(here + 1);
    if (k >= stages.end) {
      h++;
      if (h < last) k = stages.at(stages.from);
    }
    if (G::NARROW && h < last) load(h, k);
    if (first + TILE <= seen_from || first >= sight.length) continue;
    acc s[2], dp[2], bent[2];
    score<T, HD>(qs + l.set * TILE * PITCH<T, HD>, l.l16, l.g, own.of(l), s);
    score<T, HD>(gs + l.set * TILE * PITCH<T, HD>, l.l16, l.g, value.of(l), dp);
    scorer.template operator()<true>(s, bent, j - (first + Type<T>::row_of(0, l.g)));
    const bool all = !sight.documents && (!sight.causal || j0 + 15 <= first || j0 + 15 < sight.prefix);
#pragma unroll
    for (int t = 0; t < 2; t++)
#pragma unroll
      for (int r = 0; r < 4; r++) {
        const int row = l.set * TILE + 16 * t + Type<T>::row_of(r, l.g);
        s[t][r] = weight(s[t][r], tops[row]) * sums[row];
        dp[t][r] = s[t][r] * (dp[t][r] - dots[row]);
      }
    if (scorer.capped) {
#pragma unroll
      for (int t = 0; t < 2; t++) dp[t] -= dp[t] * (bent[t] * bent[t]);
    }
    // After all of it: a query that does not see the key may hold anything.
    if (!all) {
#pragma unroll
      for (int t = 0; t < 2; t++)
#pragma unroll
        for (int r = 0; r < 4; r++) {
          const int row = l.set * TILE + 16 * t + Type<T>::row_of(r, l.g);
          const bool sees = sight.sees(here * STAGE + row, sight.in(here * STAGE + row, docs[row]), j, dj);
          s[t][r] = sees ? s[t][r] : (T)0;
          dp[t][r] = sees ? dp[t][r] : (T)0;
        }
    }
    weigh<T, HD>(gs + l.set * TILE * PITCH<T, HD>, l.l16, l.g, s, dv);
    weigh<T, HD>(qs + l.set * TILE * PITCH<T, HD>, l.l16, l.g, dp, dk);
  }
  if constexpr (SETS > 1) {
    join<T, HD, G>(dk, smem, l.set);
    join<T, HD, G>(dv, smem, l.set);
  }
  if (__syncthreads_or(odd) && l.set == 0) {
    // Of queries or gradients that are no numbers nothing is left to the keys that they see.
    bool hit = false;
    for (uint32_t of = last - per_part; of < last; of++) {
      auto see = [&](int i) { hit |= sight.sees(i, sight.document(i), j, dj); };
      for_odd_rows(seen_from, sight.length, a.head, [&](int i) { return (const T*)a.q + ((int64_t)at.b * a.length + i) * a.q_row + of * a.head; }, see);
      for_odd_rows(seen_from, sight.length, a.head, [&](int i) { return (const T*)a.dy + (((int64_t)at.b * a.length + i) * a.heads + of) * a.head; }, see);
    }
    if (hit) {
      const T none = (T)__builtin_nan("");
#pragma unroll
      for (int n = 0; n < HD / 16; n++) dk[n] = dv[n] = acc{none, none, none, none};
    }
  }
  if (l.set != 0 || j >= (int)a.length) return;
  const bool none = dj < 0;
  if (a.parts == 1) {
    if (a.dk) put_row<T, HD>((T*)a.dk + key, l.g, a.head, dk, (T)a.scale, none);
    if (a.dv) put_row<T, HD>((T*)a.dv + key, l.g, a.head, dv, (T)1, none);
    return;
  }
  // A part's rows: [parts][batch, length, keys, head] of k, then of v.
  const uint64_t all_rows = (uint64_t)a.batch * a.length * a.keys, at_row = ((uint64_t)at.b * a.length + j) * a.keys + kh;
  put_row<T, HD>((T*)a.partial + (part * all_rows + at_row) * a.head, l.g, a.head, dk, (T)a.scale, none);
  put_row<T, HD>((T*)a.partial + ((a.parts + part) * all_rows + at_row) * a.head, l.g, a.head, dv, (T)1, none);
}

// Adds up the parts of the gradients of k and v, in order.
template <class T>
__global__ void __launch_bounds__(256) k_attend_parts(AttendArgs a) {
  const uint64_t n = (uint64_t)a.batch * a.length * a.keys * a.head, per = a.keys * a.head;
  for (uint64_t i = (uint64_t)blockIdx.x * 256 + threadIdx.x; i < 2 * n; i += (uint64_t)gridDim.x * 256) {
    const uint64_t at = i < n ? i : i - n;
    const T* from = (const T*)a.partial + (i < n ? 0 : a.parts * n) + at;
    T sum = from[0];
    for (uint32_t p = 1; p < a.parts; p++) sum += from[p * n];
    T* into = (T*)(i < n ? a.dk : a.dv);
    if (into) into[at / per * a.k_row + at % per] = sum;
  }
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

// Rows of a sequence's queries: the heads of one key head side by side, token after token. A block
// takes 64 of them (32 of heads past 256 bytes) and a split of the keys. Bound as the forward is, at two
// waves a SIMD: four chunks of 256, 8 heads of 128, over 0 to 3800 positions 176 us in the mean, 58 TFLOP/s.
template <class T, int HD, int RW>
__global__ void __launch_bounds__((Geo<T, HD, RW>::NT), (Geo<T, HD, RW>::FORWARD)) k_paged(AttendArgs a) {
  typedef Geo<T, HD, RW> G;
  typedef typename Type<T>::acc acc;
  constexpr int STAGE = G::STAGE, SETS = G::SETS, NT = G::NT, ROWS = G::ROWS;
  __shared__ __align__(16) T smem[2 * STAGE * PITCH<T, HD>];
  __shared__ __align__(16) int there[STAGE];
  __shared__ int coming[STAGE];
  __shared__ int64_t k_at[STAGE], v_at[STAGE];
  __shared__ T tops[SETS > 1 ? NT : 1], sums[SETS > 1 ? NT : 1];
  T *ks = smem, *vs = smem + STAGE * PITCH<T, HD>;
  const uint32_t split = blockIdx.x % a.splits, rest = blockIdx.x / a.splits;
  const Place at(rest, a.batch, a.keys, a.tiles, true, false);
  const uint32_t b = at.b, kh = at.h, group = a.heads / a.keys;
  const Cache cache(a, b);
  const Lane<RW> l;
  const uint32_t begin = at.tile * ROWS, r0 = begin + l.row;
  const int i = (int)(r0 / group);
  const uint32_t h = kh * group + r0 % group;
  const bool whole = a.head % Type<T>::V == 0, in = i < cache.count;
  const Scorer<T> scorer(a, h);
  Registers<T, HD> own;
  row_frag<T, HD>(in ? (const T*)a.q + ((int64_t)b * a.length + i) * a.q_row + h * a.head : nullptr, l.g, a.head, whole, own.frag);
  // Keys in order: `past` of the pages, then the new tokens up to the last query of the tile.
  const int last = min((int)((begin + ROWS - 1) / group), cache.count - 1), least = (int)((begin + l.first) / group);
  const int all = (int)(begin / group) < cache.count ? cache.past + last + 1 : 0;
  // Split evenly, in whole stages.
  const int per = ((all + (int)a.splits - 1) / (int)a.splits + STAGE - 1) / STAGE * STAGE;
  const int from = (int)min((int64_t)split * per, (int64_t)all), end = min(from + per, all);
  // New rows as places in the pages' operands: their distance from those.
  const int64_t kn = (const T*)a.k + (int64_t)b * a.length * a.k_row + kh * a.head - (const T*)a.k_pages;
  const int64_t vn = (const T*)a.v + (int64_t)b * a.length * a.k_row + kh * a.head - (const T*)a.v_pages;
  Running<T, HD> run;
  bool odd = false;
  Gathered<T, HD, G> next;
  // Where a stage's rows lie is looked up by its first threads a stage before it is loaded, two before
  // it is used, so that no load waits for the table.
  const bool looks = threadIdx.x < STAGE;
  int64_t k_mine = 0, v_mine = 0;
  int has = 0;
  auto look = [&](int first) {
    const int c = first + (int)threadIdx.x;
    has = looks && c < end;
    if (!has) return;
    if (c >= cache.past) {
      k_mine = kn + (int64_t)(c - cache.past) * a.k_row;
      v_mine = vn + (int64_t)(c - cache.past) * a.k_row;
    } else {
      const int64_t row = cache.row((uint32_t)c);
      has = row >= 0;
      k_mine = v_mine = (max(row, (int64_t)0) * a.keys + kh) * a.head;
    }
  };
  auto leave = [&] {
    if (!looks) return;
    k_at[threadIdx.x] = has ? k_mine : 0;
    v_at[threadIdx.x] = has ? v_mine : 0;
    coming[threadIdx.x] = has;
  };
  auto load = [&] { next.load((const T*)a.k_pages, (const T*)a.v_pages, k_at, v_at, coming, a.head, whole); };
  if (from < end) {
    look(from);
    leave();
    __syncthreads();
    load();
    look(from + STAGE);
  }
  for (int stage = from; stage < end; stage += STAGE) {
    __syncthreads();
    odd |= make_finite<T>(next.y);
    next.store(ks, vs);
    if (looks) there[threadIdx.x] = coming[threadIdx.x];
    leave();
    __syncthreads();
    if (stage + STAGE < end) {
      load();
      look(stage + 2 * STAGE);
    }
    const int first = stage + l.set * TILE;
    if (first >= end || least >= cache.count) continue;
    acc s[2];
    score<T, HD>(ks + l.set * TILE * PITCH<T, HD>, l.l16, l.g, own, s);
    // Positions of old keys run on to the new ones' unless the table ends before them.
    const int apart = i + (first >= cache.past ? cache.past : cache.first) - first - Type<T>::row_of(0, l.g);
    const bool one = first + TILE <= cache.past || first >= cache.past || cache.first == cache.past;
    scorer.template operator()<false>(s, nullptr, apart);
    if (!one && scorer.sloped) {
      // A tile with keys on both sides of a gap: the new ones are nearer than their place says.
#pragma unroll
      for (int t = 0; t < 2; t++)
#pragma unroll
        for (int r = 0; r < 4; r++) {
          const int c = first + 16 * t + Type<T>::row_of(r, l.g);
          if (c >= cache.past)
            s[t][r] += scorer.slope * (Scorer<T>::abs_of((T)apart - (T)tile_row<T>(t, r)) - Scorer<T>::abs_of((T)(i - (c - cache.past))));
        }
    }
#pragma unroll
    for (int t = 0; t < 2; t++)
#pragma unroll
      for (int r = 0; r < 4; r++) {
        const int row = 16 * t + Type<T>::row_of(r, l.g), c = first + row;
        s[t][r] = in && there[l.set * TILE + row] && c - cache.past <= i ? s[t][r] : -(T)__builtin_huge_val();
      }
    run.add(s);
    weigh<T, HD>(vs + l.set * TILE * PITCH<T, HD>, l.l16, l.g, s, run.out);
  }
  run.sum = row_sum(run.sum);
  if constexpr (SETS > 1) join<T, HD, G>(run, smem, tops, sums, l.set);
  if (__syncthreads_or(odd) && l.set == 0) {
    auto value = [&](int c) -> const T* {
      if (c >= cache.past) return (const T*)a.v_pages + vn + (int64_t)(c - cache.past) * a.k_row;
      const int64_t row = cache.row((uint32_t)c);
      return row < 0 ? nullptr : (const T*)a.v_pages + (row * a.keys + kh) * a.head;
    };
    for_odd_rows(from, end, a.head, value, [&](int c) {
      if (in && c - cache.past <= i) add_odd<T, HD>(value(c), l.g, a.head, run.out);
    });
  }
  if (l.set != 0 || i >= (int)a.length) return;
  const uint64_t row = ((uint64_t)b * a.length + i) * a.heads + h;
  if (a.splits == 1) {
    if (a.y) put_row<T, HD>((T*)a.y + row * a.head, l.g, a.head, run.out, 1 / run.sum, run.sum == 0);
    return;
  }
  // A split's bound, sum and weighed values: [rows][splits] of 2 + head.
  T* part = (T*)a.partial + (row * a.splits + split) * (a.head + 2);
  put_row<T, HD>(part + 2, l.g, a.head, run.out, (T)1, false);
  if (l.g == 0) {
    part[0] = run.top;
    part[1] = run.sum;
  }
}

// Rows that one wave's tile holds, of single tokens and a few: a wave of the block's four takes every
// fourth step of the split's keys, straight from memory into the fragments of both products, while the
// rows of its next step are looked up. A key's row is read by the four lanes that hold it 16 bytes
// apart, a value's by sixteen. Three waves a SIMD, with 16 KB on the way each, hide what they wait for;
// a second step's fragments in registers left room for one and took three times as long. Bound by memory:
// 62 MB of 60000 positions, 2 key heads of 64, in 14 to 16 us (4.0 TB/s); by the latency of a split's few
// steps where there are many sequences: 28 MB of sixteen of 300 to 2300 in 10 to 12 us, for which the
// kernel of whole tiles takes 23.
// WHOLE: heads of whole 16 bytes.
template <class T, int HD>
struct FewGeo {
  static constexpr int TILES = (int)sizeof(T) * HD <= 256 ? 2 : 1, STEP = 16 * TILES;  // keys of a wave's step
  static constexpr bool FITS = (int)sizeof(T) * HD <= 512;
};
constexpr int FEW_ROWS = 16;

template <class T, int HD, bool WHOLE>
__global__ void __launch_bounds__(256, (WHOLE ? FewGeo<T, HD>::TILES + 1 : 2)) k_paged_few(AttendArgs a) {
  typedef typename Type<T>::acc acc;
  typedef typename Type<T>::vec vec;
  constexpr int TILES = FewGeo<T, HD>::TILES, STEP = FewGeo<T, HD>::STEP, ND = HD / 16, V = Type<T>::V;
  constexpr int KV = HD / 4 / V;  // vectors of a key's quarter
  __shared__ T outs[4][16 * (HD + 1)], tops[4][16], sums[4][16];
  const uint32_t split = blockIdx.x % a.splits, rest = blockIdx.x / a.splits, b = rest / a.keys, kh = rest % a.keys, group = a.heads / a.keys;
  const Cache cache(a, b);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, l16 = lane & 15, g = lane >> 4;
  const int i = l16 / (int)group;
  const uint32_t h = kh * group + l16 % group;
  const bool in = l16 < (int)(a.length * group) && i < cache.count;
  // The old keys split evenly, in whole rounds of the four waves; the new ones go to the last split.
  const int per = ((cache.past + (int)a.splits - 1) / (int)a.splits + 4 * STEP - 1) / (4 * STEP) * (4 * STEP);
  const int from = (int)min((int64_t)split * per, (int64_t)cache.past), end = min(from + per, cache.past);
  const bool own = cache.count > 0 && split == a.splits - 1;
  const Scorer<T> scorer(a, in ? h : kh * group);
  T frag[HD / 4];
  row_frag<T, HD>(in ? (const T*)a.q + ((int64_t)b * a.length + i) * a.q_row + h * a.head : nullptr, g, a.head, WHOLE, frag);
  Running<T, HD> run;
  struct Rows {
    vec k[TILES][KV];
    T v[TILES][4][ND];
    uint64_t there[TILES];
  };
  // Rows of a step's keys, a lane's own of each tile: places in both operands or -1.
  auto look = [&](int first, int64_t* row) {
#pragma unroll
    for (int t = 0; t < TILES; t++) {
      const int c = first + 16 * t + l16;
      row[t] = c < end ? cache.row((uint32_t)c) : -1;
    }
  };
  auto fetch = [&](const T* ks, const T* vs, int64_t pitch, const int64_t* row, Rows& x) {
#pragma unroll
    for (int t = 0; t < TILES; t++) {
      x.there[t] = __ballot(row[t] >= 0);
      const T* k = ks + max(row[t], (int64_t)0) * pitch;
#pragma unroll
      for (int n = 0; n < KV; n++) {
        const uint32_t d = (uint32_t)(n * V / 4 * 16 + 4 * g + n * V % 4);
        if constexpr (WHOLE) {
          x.k[t][n] = *(const vec*)(k + (d < a.head ? d : 0));
        } else {
#pragma unroll
          for (uint32_t j = 0; j < V; j++) x.k[t][n][j] = k[d + j < a.head ? d + j : 0];
        }
      }
    }
#pragma unroll
    for (int t = 0; t < TILES; t++)
#pragma unroll
      for (int r = 0; r < 4; r++) {
        const T* v = vs + max((int64_t)__shfl(row[t], Type<T>::row_of(r, g)), (int64_t)0) * pitch;
        const uint32_t d = (uint32_t)(l16 * ND);
        constexpr int VN = !WHOLE ? 1 : ND % V == 0 ? V : 2;  // whole heads are a multiple of it
#pragma unroll
        for (int n = 0; n < ND; n += VN) {
          const T* from = v + (d + n < a.head ? d + n : 0);
          if constexpr (WHOLE) take<VN>(from, x.v[t][r] + n);
          else x.v[t][r][n] = *from;
        }
      }
  };
  // Makes 0 what was loaded in the place of columns past the head and of rows that are not there; not
  // as it is loaded, which would wait for it.
  auto clear = [&](Rows& x) {
    if (a.head < HD) {
#pragma unroll
      for (int t = 0; t < TILES; t++) {
#pragma unroll
        for (int n = 0; n < KV; n++)
#pragma unroll
          for (uint32_t j = 0; j < V; j++)
            if ((uint32_t)(n * V / 4 * 16 + 4 * g + n * V % 4) + j >= a.head) x.k[t][n][j] = 0;
#pragma unroll
        for (int r = 0; r < 4; r++)
#pragma unroll
          for (uint32_t n = 0; n < ND; n++)
            if ((uint32_t)(l16 * ND) + n >= a.head) x.v[t][r][n] = 0;
      }
    }
#pragma unroll
    for (int t = 0; t < TILES; t++)
      if (x.there[t] != ~0ull) {
#pragma unroll
        for (int r = 0; r < 4; r++)
#pragma unroll
          for (int n = 0; n < ND; n++)
            if (!(x.there[t] >> Type<T>::row_of(r, g) & 1)) x.v[t][r][n] = 0;
      }
  };
  // `apart`: the distance of the lane's row from the step's first key. `news`: the values of the new
  // tokens, where the step is of them.
  auto work = [&](Rows& x, int apart, const T* news) {
    const bool ordered = news != nullptr;
    clear(x);
    bool odd = false;
    if (ordered && a.length > 1) {
      // Of tokens that earlier ones do not see, infinities and NaN are kept out as by make_finite.
#pragma unroll
      for (int r = 0; r < 4; r++)
#pragma unroll
        for (int n = 0; n < ND; n++)
          if (x.v[0][r][n] * 0 != 0) {
            odd = true;
            x.v[0][r][n] = 0;
          }
    }
    acc s[2] = {acc{0, 0, 0, 0}, acc{0, 0, 0, 0}};
#pragma unroll
    for (int n = 0; n < KV; n++)
#pragma unroll
      for (int j = 0; j < V; j++)
#pragma unroll
        for (int t = 0; t < TILES; t++) s[t] = Type<T>::mfma(x.k[t][n][j], frag[n * V + j], s[t]);
    scorer.template operator()<false>(s, nullptr, apart - Type<T>::row_of(0, g));
#pragma unroll
    for (int t = 0; t < 2; t++)
#pragma unroll
      for (int r = 0; r < 4; r++) {
        const int of = Type<T>::row_of(r, g);
        const bool sees = t < TILES && in && (x.there[t < TILES ? t : 0] >> of & 1) && (!ordered || 16 * t + of <= apart);
        s[t][r] = sees ? s[t][r] : -(T)__builtin_huge_val();
      }
    run.add(s);
#pragma unroll
    for (int t = 0; t < TILES; t++)
#pragma unroll
      for (int r = 0; r < 4; r++)
#pragma unroll
        for (int n = 0; n < ND; n++) run.out[n] = Type<T>::mfma(x.v[t][r][n], s[t][r], run.out[n]);
    if (ordered && __ballot(odd) != 0)
      for (int c = 0; c < cache.count; c++)
        if (in && c <= i) add_odd<T, HD>(news + c * a.k_row, g, a.head, run.out);
  };
  const T *kp = (const T*)a.k_pages + kh * a.head, *vp = (const T*)a.v_pages + kh * a.head;
  const int64_t pitch = (int64_t)a.keys * a.head;
  int64_t row[TILES];
  Rows x;
  int first = from + wave * STEP;
  if (first < end) look(first, row);
  for (; first < end; first += 4 * STEP) {
    fetch(kp, vp, pitch, row, x);
    look(first + 4 * STEP, row);
    work(x, cache.first + i - first, nullptr);
  }
  if (own && wave == 3) {
#pragma unroll
    for (int t = 0; t < TILES; t++) row[t] = t == 0 && l16 < cache.count ? l16 : -1;
    const int64_t at = (int64_t)b * a.length * a.k_row + kh * a.head;
    fetch((const T*)a.k + at, (const T*)a.v + at, a.k_row, row, x);
    work(x, i, (const T*)a.v + at);
  }
  // The four waves' results, joined in order.
  const T sum = row_sum(run.sum);
  if (g == 0) {
    tops[wave][l16] = run.top;
    sums[wave][l16] = sum;
  }
#pragma unroll
  for (int r = 0; r < 4; r++)
#pragma unroll
    for (int n = 0; n < ND; n++) outs[wave][l16 * (HD + 1) + Type<T>::row_of(r, g) * ND + n] = run.out[n][r];
  __syncthreads();
  const uint32_t rows = a.length * group;
  for (uint32_t at = threadIdx.x; at < rows * HD; at += 256) {
    const uint32_t r = at / HD, d = at % HD;
    if (d >= a.head) continue;
    T top = tops[0][r];
#pragma unroll
    for (int w = 1; w < 4; w++) top = Type<T>::max_of(top, tops[w][r]);
    const T base = Running<T, HD>::base(top);
    T all = 0, v = 0;
#pragma unroll
    for (int w = 0; w < 4; w++) {
      const T by = Type<T>::exp2_of(tops[w][r] - base);
      all += sums[w][r] * by;
      v += outs[w][r * (HD + 1) + d] * by;
    }
    const uint64_t row = ((uint64_t)b * a.length + r / group) * a.heads + kh * group + r % group;
    if (a.splits == 1) {
      ((T*)a.y)[row * a.head + d] = all == 0 ? (T)0 : v / all;
      continue;
    }
    T* part = (T*)a.partial + (row * a.splits + split) * (a.head + 2);
    part[2 + d] = v;
    if (d == 0) {
      part[0] = top;
      part[1] = all;
    }
  }
}

// Joins the splits of each row, and then (blocks from `join_blocks` on) puts the new
// tokens' keys and values into their pages, a wave a token and key head. Rows that a later sequence
// writes too are left to it, so that the result does not depend on which comes first. It comes after
// every read of the pages, so that it may write into the ones that were read.
template <class T>
__global__ void __launch_bounds__(512) k_paged_finish(AttendArgs a, uint32_t join_blocks) {
  const uint32_t lane = threadIdx.x & 63;
  if (blockIdx.x < join_blocks) {
    // Threads side by side on the head, `join_step` such rows of them on the splits, each over its own
    // with a maximum of its own, so that nothing waits for a first look at them all; the rest of the
    // block on other rows.
    __shared__ T lanes[512], tops[512], sums[512];
    const uint32_t width = a.join_width, step = a.join_step, pitch = a.head + 2;
    const uint64_t rows = (uint64_t)a.batch * a.length * a.heads, mine = (uint64_t)blockIdx.x * (512 / (width * step)) + threadIdx.x / (width * step);
    const uint64_t row = min(mine, rows - 1);
    const T* part = (const T*)a.partial + row * a.splits * pitch;
    const uint32_t d = threadIdx.x % width, first = threadIdx.x / width % step, column = 2 + min(d, a.head - 1);
    T top = -(T)__builtin_huge_val(), sum = 0, v = 0;
    constexpr uint32_t N = 8;
    for (uint32_t p = first; p < a.splits; p += N * step) {
      T high[N], of[N], x[N];
#pragma unroll
      for (uint32_t k = 0; k < N; k++) {
        const T* from = part + (uint64_t)min(p + k * step, a.splits - 1) * pitch;
        high[k] = from[0];
        of[k] = from[1];
        x[k] = from[column];
      }
      T next = top;
#pragma unroll
      for (uint32_t k = 0; k < N; k++) {
        if (p + k * step >= a.splits) high[k] = -(T)__builtin_huge_val();
        next = Type<T>::max_of(next, high[k]);
      }
      const T base = next == -(T)__builtin_huge_val() ? (T)0 : next, by = Type<T>::exp2_of(top - base);
      top = next;
      sum *= by;
      v *= by;
#pragma unroll
      for (uint32_t k = 0; k < N; k++) {
        // A split that has seen nothing adds nothing.
        const T w = Type<T>::exp2_of(high[k] - base);
        sum += w == 0 ? (T)0 : of[k] * w;
        v += w == 0 ? (T)0 : x[k] * w;
      }
    }
    lanes[threadIdx.x] = v;
    tops[threadIdx.x] = top;
    sums[threadIdx.x] = sum;
    __syncthreads();
    if (first != 0 || d >= a.head || mine >= rows) return;
    for (uint32_t k = 1; k < step; k++) top = Type<T>::max_of(top, tops[threadIdx.x + k * width]);
    const T base = top == -(T)__builtin_huge_val() ? (T)0 : top;
    sum = v = 0;
    for (uint32_t k = 0; k < step; k++) {
      const T w = Type<T>::exp2_of(tops[threadIdx.x + k * width] - base);
      sum += sums[threadIdx.x + k * width] * w;
      v += lanes[threadIdx.x + k * width] * w;
    }
    ((T*)a.y)[row * a.head + d] = sum == 0 ? (T)0 : v / sum;
    return;
  }
  const uint64_t item = (uint64_t)(blockIdx.x - join_blocks) * (512 / 64) + (threadIdx.x >> 6);
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

// Squares are exact in 64 bits and summed there. Values of a block: four 16 bytes a thread of float32 on
// their way at once. 19 MB in 64 tensors: 4.3 to 5.3 us (3.7 TB/s or more, from the caches) and 1.8 for the
// root of the blocks' sums.
constexpr uint64_t NORM_PER_BLOCK = 4096;

template <class T>
__global__ void __launch_bounds__(256) k_norm_squares(NormTensors t, double* partial) {
  typedef typename Type<T>::vec vec;
  constexpr int V = Type<T>::V, N = (int)(NORM_PER_BLOCK / (256 * V));
  uint32_t k = 0;
#pragma unroll
  for (uint32_t half = NORM_TENSORS / 2; half > 0; half /= 2)
    if (k + half < t.count && blockIdx.x >= t.first_block[k + half]) k += half;
  const uint64_t begin = (uint64_t)(blockIdx.x - t.first_block[k]) * NORM_PER_BLOCK;
  const T* x = (const T*)t.x[k] + begin;
  const uint32_t n = (uint32_t)min(NORM_PER_BLOCK, t.n[k] - begin);
  double sum = 0;
  if (n == NORM_PER_BLOCK) {
    vec v[N];
#pragma unroll
    for (int i = 0; i < N; i++) v[i] = *(const vec*)(x + (i * 256 + threadIdx.x) * V);
#pragma unroll
    for (int i = 0; i < N; i++)
#pragma unroll
      for (int j = 0; j < V; j++) sum = fma((double)v[i][j], (double)v[i][j], sum);
  } else {
    for (uint32_t i = threadIdx.x; i < n; i += 256) sum = fma((double)x[i], (double)x[i], sum);
  }
  __shared__ double waves[4];
  sum = rg_wave_sum(sum);
  if ((threadIdx.x & 63) == 0) waves[threadIdx.x >> 6] = sum;
  __syncthreads();
  if (threadIdx.x == 0) partial[blockIdx.x] = ((waves[0] + waves[1]) + waves[2]) + waves[3];
}

template <class T>
__global__ void __launch_bounds__(1024) k_norm_root(const double* partial, uint32_t blocks, T* out) {
  __shared__ double waves[16];
  double sum = 0;
#pragma unroll 4
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

// Calls f with the type, the padded head and the row waves as constants.
template <class F>
void by_head(int dtype, uint32_t head, uint32_t rows, const F& f) {
  auto of = [&](auto t) {
    auto by_rows = [&](auto hd) {
      constexpr int SIZE = (int)sizeof(t) * decltype(hd)::value;
      if constexpr (SIZE <= 512)
        if (rows == 32) return f(t, hd, std::integral_constant<int, 2>{});
      if constexpr (SIZE <= 256 || SIZE > 512) f(t, hd, std::integral_constant<int, 4>{});
    };
    if (head <= 32) by_rows(std::integral_constant<int, 32>{});
    else if (head <= 64) by_rows(std::integral_constant<int, 64>{});
    else if (head <= 96) by_rows(std::integral_constant<int, 96>{});
    else if (head <= 128) by_rows(std::integral_constant<int, 128>{});
    else if constexpr (sizeof(t) == 4) by_rows(std::integral_constant<int, 256>{});
  };
  if (dtype == RG_F32) of(float{});
  else of(double{});
}

// Heads of more than 256 and of more than 512 bytes.
bool wide_head(int dtype, uint32_t head) { return head > (dtype == RG_F32 ? 64u : 32u); }
bool widest_head(int dtype, uint32_t head) { return head > (dtype == RG_F32 ? 128u : 64u); }
// Rows of a block: 64, or 32 where those leave fewer than two blocks for every CU, and for heads whose
// blocks have four waves. Forward, dq, dk and dv of the causal case (512 blocks of 64) 122, 182, 230 us, with 32
// rows 152, 201, 242; of 3 sequences of 777, 6 heads of 44 (234 blocks of 64) 31, 40, 47 with 32 rows, with 64
// 46, 68, 90.
uint32_t rows_of(int dtype, const AttendArgs& a) {
  if (widest_head(dtype, a.head)) return 64;
  return wide_head(dtype, a.head) || (uint64_t)a.batch * a.heads * ((a.length + 63) / 64) < 2 * CUS ? 32 : 64;
}
uint32_t tiles_of(int dtype, const AttendArgs& a) { return (a.length + rows_of(dtype, a) - 1) / rows_of(dtype, a); }

void set_rows(int dtype, AttendArgs& a) {
  a.q_row = (int64_t)(a.joined ? a.heads + 2 * a.keys : a.heads) * a.head;
  a.k_row = a.joined ? a.q_row : (int64_t)a.keys * a.head;
  a.tiles = tiles_of(dtype, a);
}

uint64_t size_of(int dtype) { return dtype == RG_F32 ? 4 : 8; }

// Whether the rows of a key head are few enough for one wave, and the heads for its registers.
bool few_rows(int dtype, const AttendArgs& a) { return (uint64_t)a.length * (a.heads / a.keys) <= FEW_ROWS && !widest_head(dtype, a.head); }
// Rows of a block in the paged form, and tiles of a sequence's rows.
uint32_t paged_rows(int dtype, const AttendArgs& a) { return wide_head(dtype, a.head) && !widest_head(dtype, a.head) ? 32 : 64; }
uint32_t paged_tiles(int dtype, const AttendArgs& a) {
  return (uint32_t)(((uint64_t)a.length * (a.heads / a.keys) + paged_rows(dtype, a) - 1) / paged_rows(dtype, a));
}
// Over how many blocks a sequence's keys are split, by the room of its table, since only the device
// knows how much of it is used: three blocks of few rows for every CU, of whole tiles two (176 us for 4
// chunks of 256 at 8 heads of 128 over up to 4096 positions; with four of them 193), but not so many that
// a full table leaves one fewer keys than a stage of the block has (float64, 3 x 17 x 6 heads of 40 over 600
// positions: 12 us, with 256 at least 27).
void set_splits(int dtype, AttendArgs& a) {
  const bool few = few_rows(dtype, a);
  const uint64_t keys = (uint64_t)a.table_pages * a.page + (few ? 0 : a.length), blocks = (uint64_t)a.batch * a.keys * (few ? 1 : paged_tiles(dtype, a));
  const uint64_t least = few ? 128 : 64, want = std::max<uint64_t>(1, (few ? 3 * CUS : 2 * CUS) / blocks);
  uint64_t per = std::max(least, (keys + want - 1) / want);
  per = (per + least - 1) / least * least;
  a.splits = (uint32_t)((keys + per - 1) / per);
}

// A gradient's workspace: dy.y of every query, then the parts of dk and dv.
uint64_t dots_bytes(int dtype, const AttendArgs& a) { return ((uint64_t)a.batch * a.heads * a.length * size_of(dtype) + 255) / 256 * 256; }
// Parts of a group's heads: as few as leave two blocks for every CU. Packed documents, 4 sequences of 1024, 8
// heads on 2 of 64 (128 blocks): 135 us and 6 for the sums of four parts, 445 in one; the 3 of 777 above, 6
// heads on 3: 47 and 5, 84 in one.
uint32_t parts_of(int dtype, const AttendArgs& a) {
  const uint32_t group = a.heads / a.keys;
  const uint64_t blocks = (uint64_t)a.batch * a.keys * tiles_of(dtype, a);
  for (uint32_t p = 1; p < group; p++)
    if (group % p == 0 && blocks * p >= 2 * CUS) return p;
  return group;
}

}  // namespace

uint64_t attend_blocks(int dtype, const AttendArgs& a) { return 2 * (uint64_t)a.batch * a.heads * tiles_of(dtype, a); }
uint64_t attend_workspace(int dtype, const AttendArgs& a) {
  const uint32_t parts = parts_of(dtype, a);
  return dots_bytes(dtype, a) + (parts > 1 ? 2 * (uint64_t)parts * a.batch * a.length * a.keys * a.head * size_of(dtype) : 0);
}
uint32_t attend_slope_rows(int dtype, const AttendArgs& a) { return a.batch * tiles_of(dtype, a); }

void attend(hipStream_t s, int dtype, const AttendArgs& args) {
  AttendArgs a = args;
  set_rows(dtype, a);
  by_head(dtype, a.head, rows_of(dtype, a), [&](auto t, auto hd, auto rw) {
    typedef decltype(t) T;
    constexpr int HD = decltype(hd)::value, RW = decltype(rw)::value;
    k_attend<T, HD, RW><<<a.tiles * a.batch * a.heads, Geo<T, HD, RW>::NT, 0, s>>>(a);
  });
}

void attend_grad(hipStream_t s, int dtype, const AttendArgs& args) {
  AttendArgs a = args;
  set_rows(dtype, a);
  a.parts = parts_of(dtype, a);
  a.partial = (char*)a.workspace + dots_bytes(dtype, a);
  by_head(dtype, a.head, rows_of(dtype, a), [&](auto t, auto hd, auto rw) {
    typedef decltype(t) T;
    constexpr int HD = decltype(hd)::value, RW = decltype(rw)::value;
    k_attend_dq<T, HD, RW><<<a.tiles * a.batch * a.heads, Geo<T, HD, RW>::NT, 0, s>>>(a);
    if (!a.dk && !a.dv) return;
    k_attend_dkv<T, HD, RW><<<a.tiles * a.batch * a.keys * a.parts, Geo<T, HD, RW>::NT, 0, s>>>(a);
    if (a.parts == 1) return;
    const uint64_t n = 2 * (uint64_t)a.batch * a.length * a.keys * a.head;
    k_attend_parts<T><<<(uint32_t)std::min<uint64_t>((n + 255) / 256, 8192), 256, 0, s>>>(a);
  });
}

uint64_t paged_blocks(int dtype, const AttendArgs& args) {
  AttendArgs a = args;
  set_splits(dtype, a);
  const uint64_t rows = (uint64_t)a.batch * a.length * (a.heads + a.keys / 8 + 1) + 1;
  return 2 * std::max((uint64_t)a.batch * a.keys * paged_tiles(dtype, a) * a.splits, rows);
}

uint64_t paged_workspace(int dtype, const AttendArgs& args) {
  AttendArgs a = args;
  set_splits(dtype, a);
  return a.splits == 1 ? 0 : (uint64_t)a.batch * a.length * a.heads * a.splits * (a.head + 2) * size_of(dtype);
}

void paged_attend(hipStream_t s, int dtype, const AttendArgs& args) {
  AttendArgs a = args;
  set_rows(dtype, a);
  set_splits(dtype, a);
  a.tiles = paged_tiles(dtype, a);
  a.partial = a.workspace;
  a.page_div = FastDiv(a.page);
  const uint64_t values = (uint64_t)a.pages * a.page * a.keys * a.head * size_of(dtype);
  if (a.k_out && a.k_out != a.k_pages) copy_bytes(s, a.k_out, a.k_pages, values);
  if (a.v_out && a.v_out != a.v_pages) copy_bytes(s, a.v_out, a.v_pages, values);
  const bool few = few_rows(dtype, a);
  if (a.y)
    by_head(dtype, a.head, paged_rows(dtype, a), [&](auto t, auto hd, auto rw) {
      typedef decltype(t) T;
      constexpr int HD = decltype(hd)::value, RW = decltype(rw)::value;
      if constexpr (FewGeo<T, HD>::FITS) {
        if (few) {
          const uint32_t blocks = a.batch * a.keys * a.splits;
          if (a.head % Type<T>::V == 0) k_paged_few<T, HD, true><<<blocks, 256, 0, s>>>(a);
          else k_paged_few<T, HD, false><<<blocks, 256, 0, s>>>(a);
          return;
        }
      }
      if constexpr ((RW == 2) == ((int)sizeof(T) * HD > 256 && (int)sizeof(T) * HD <= 512))
        k_paged<T, HD, RW><<<a.batch * a.keys * a.tiles * a.splits, Geo<T, HD, RW>::NT, 0, s>>>(a);
    });
  // A thread of the join takes eight splits in one round of loads, and a block as many rows as that leaves.
  a.join_width = a.join_step = 1;
  while (a.join_width < a.head) a.join_width *= 2;
  while (a.join_step * 8 < a.splits && a.join_step * 2 * a.join_width <= 512) a.join_step *= 2;
  const uint64_t rows = (uint64_t)a.batch * a.length * a.heads, per_block = 512 / (a.join_width * a.join_step);
  const uint32_t join = a.y && a.splits > 1 ? (uint32_t)((rows + per_block - 1) / per_block) : 0;
  const uint32_t append = a.k_out || a.v_out ? (uint32_t)(((uint64_t)a.batch * a.length * a.keys + 7) / 8) : 0;
  if (join + append == 0) return;
  if (dtype == RG_F32) k_paged_finish<float><<<join + append, 512, 0, s>>>(a, join);
  else k_paged_finish<double><<<join + append, 512, 0, s>>>(a, join);
}

uint32_t norm_blocks(uint64_t n) { return (uint32_t)((n + NORM_PER_BLOCK - 1) / NORM_PER_BLOCK); }

void norm_squares(hipStream_t s, int dtype, const NormTensors& t, uint32_t blocks, double* partial) {
  if (dtype == RG_F32) k_norm_squares<float><<<blocks, 256, 0, s>>>(t, partial);
  else k_norm_squares<double><<<blocks, 256, 0, s>>>(t, partial);
}

void norm_root(hipStream_t s, int dtype, const double* partial, uint32_t blocks, void* out) {
  if (dtype == RG_F32) k_norm_root<float><<<1, 1024, 0, s>>>(partial, blocks, (float*)out);
  else k_norm_root<double><<<1, 1024, 0, s>>>(partial, blocks, (double*)out);
}

}  // namespace rgk
