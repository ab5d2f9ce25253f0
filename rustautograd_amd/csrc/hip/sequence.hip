// The sequence operators (include/rg_plan.h, CAUSAL_CONV ... ROTARY_NORM_GRAD).
#include "sequence.h"

#include <algorithm>
#include <cmath>

namespace rgk {

namespace {

constexpr int TPB = 256;

__device__ __forceinline__ float fma_(float a, float b, float c) { return __builtin_fmaf(a, b, c); }
__device__ __forceinline__ double fma_(double a, double b, double c) { return __builtin_fma(a, b, c); }
// e^v for -infinity <= v <= 88: the hardware's power of two of v log2 e, times what the rounding of
// that product leaves out (half the instructions of the full range). Below -104 it is 0.
__device__ __forceinline__ float exp_(float v) {
  constexpr float L = 1.44269504088896341f, REST = 1.92596303e-8f, LN2 = 0.693147180559945309f;  // log2 e = L + REST
  v = v < -200.0f ? -200.0f : v;
  const float t = v * L, r = fma_(v, REST, fma_(v, L, -t)), e = __builtin_amdgcn_exp2f(t);
  return fma_(e, r * LN2, e);
}
__device__ __forceinline__ double exp_(double v) { return exp(v); }
__device__ __forceinline__ float sqrt_(float v) { return sqrtf(v); }
__device__ __forceinline__ double sqrt_(double v) { return sqrt(v); }
// a / b for a finite a and a positive, finite, normal b: the hardware's reciprocal and one step of Newton's method,
// within a unit in the last place or two (the full division, for every b, takes three times as long).
__device__ __forceinline__ float over(float a, float b) {
  const float r = __builtin_amdgcn_rcpf(b), q = a * r;
  return fma_(fma_(-b, q, a), r, q);
}
__device__ __forceinline__ double over(double a, double b) { return a / b; }
__device__ __forceinline__ float abs_(float v) { return __builtin_fabsf(v); }
__device__ __forceinline__ double abs_(double v) { return __builtin_fabs(v); }
// 1 / (1 + e^-v), below zero as e^v / (1 + e^v): it goes to 0 as the exponential does, so that v times it is 0
// for the lowest values of the type, as masks have them.
template <class T>
__device__ __forceinline__ T sigmoid(T v) {
  const T u = exp_(-abs_(v));
  return over(v > T(0) ? T(1) : u, T(1) + u);
}
template <class T>
__device__ __forceinline__ T silu(T v) { return v * sigmoid(v); }
// silu'(v) from s = sigmoid(v).
template <class T>
__device__ __forceinline__ T silu_slope(T v, T s) { return s * fma_(v, T(1) - s, T(1)); }
// log(1 + u), 0 <= u <= 1, to full relative precision: u + u^2 p(u), where 1 + u p(u) is the least
// squares fit of degree 9 to log(1 + u) / u in Chebyshev polynomials of [0, 1]; with its roundings
// 2.31 x 2^-24 off at most (every float from 1/4 on, every seventh below).
__device__ __forceinline__ float log1p_(float u) {
  float p = -0.00325637846f;
  p = fma_(p, u, 0.0199071616f);
  p = fma_(p, u, -0.0570642017f);
  p = fma_(p, u, 0.106142648f);
  p = fma_(p, u, -0.153118625f);
  p = fma_(p, u, 0.196781173f);
  p = fma_(p, u, -0.249545589f);
  p = fma_(p, u, 0.333300054f);
  p = fma_(p, u, -0.499999046f);
  return fma_(u * p, u, u);
}
__device__ __forceinline__ double log1p_(double u) { return log1p(u); }
// log(1 + e^v) without overflow, small steps to full relative precision.
template <class T>
__device__ __forceinline__ T softplus(T v) { return (v > T(0) ? v : T(0)) + log1p_(exp_(v > T(0) ? -v : v)); }
// The same with its slope, the logistic function of v.
template <class T>
__device__ __forceinline__ T softplus(T v, T* slope) {
  const T u = exp_(v > T(0) ? -v : v);
  *slope = over(v > T(0) ? T(1) : u, T(1) + u);
  return (v > T(0) ? v : T(0)) + log1p_(u);
}

__device__ __forceinline__ uint32_t end_of(const int32_t* lengths, uint32_t b, uint32_t length) {
  if (!lengths) return length;
  const int32_t n = lengths[b];
  return n < 0 ? 0u : min((uint32_t)n, length);
}

// V consecutive values, moved as one access of up to 16 bytes.
template <class T, int V>
struct alignas(sizeof(T) * V > 16 ? 16 : sizeof(T) * V) Vec {
  T v[V];
};
template <class T, int V>
__device__ __forceinline__ Vec<T, V> load(const T* p) { return *(const Vec<T, V>*)p; }
template <class T, int V>
__device__ __forceinline__ void store(T* p, const Vec<T, V>& v) { *(Vec<T, V>*)p = v; }

// ---- causal convolution -----------------------------------------------------------------------

// A wave takes 64 V neighbouring channels over a run of R positions and keeps the last K inputs
// in registers, so that x is read once but for the K - 1 positions before a run. Bound by memory:
// 8 x 4096 x 2048, four taps 90 us, 6.0 TB/s; below some 20 MB by the latency of a block's loads,
// all of which are in flight at once (4 x 1024 x 512 5.3 us, 3.3 at the rate of a copy).
template <class T, int K, int V, int R>
__global__ void __launch_bounds__(TPB) k_conv(ConvArgs a, uint32_t nx, uint32_t runs) {
  const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const uint32_t bx = blockIdx.x % nx, by = blockIdx.x / nx;
  const uint32_t b = by / runs, t0 = ((by % runs) * (TPB / 64) + wave) * R;
  const uint32_t d = (bx * 64 + lane) * V;
  if (d >= a.width || t0 >= a.length) return;
  const uint32_t n = end_of(a.lengths, b, a.length);
  const T* x = (const T*)a.x + (uint64_t)b * a.length * a.width + d;
  const T* state = a.state ? (const T*)a.state + (uint64_t)b * (K - 1) * a.width + d : nullptr;
  auto past = [&](uint32_t i) {  // i < n + K - 1
    Vec<T, V> v{};
    if (i >= K - 1) v = load<T, V>(x + (uint64_t)(i - (K - 1)) * a.width);
    else if (state) v = load<T, V>(state + (uint64_t)i * a.width);
    return v;
  };
  if (a.next && t0 == 0) {
    T* next = (T*)a.next + (uint64_t)b * (K - 1) * a.width + d;
#pragma unroll
    for (int j = 0; j < K - 1; j++) store<T, V>(next + (uint64_t)j * a.width, past(n + j));
  }
  if (!a.y) return;
  Vec<T, V> w[K], bias{}, in[R + K - 1];
#pragma unroll
  for (int k = 0; k < K; k++) w[k] = load<T, V>((const T*)a.w + (uint64_t)k * a.width + d);
  if (a.bias) bias = load<T, V>((const T*)a.bias + d);
#pragma unroll
  for (int i = 0; i < R + K - 1; i++) {
    in[i] = Vec<T, V>{};
    if (t0 + i < n + (K - 1)) in[i] = past(t0 + i);
  }
  T* y = (T*)a.y + ((uint64_t)b * a.length + t0) * a.width + d;
#pragma unroll
  for (int i = 0; i < R; i++) {
    if (t0 + i >= a.length) break;
    Vec<T, V> out{};
    if (t0 + i < n) {
#pragma unroll
      for (int v = 0; v < V; v++) {
        T pre = bias.v[v];
#pragma unroll
        for (int k = 0; k < K; k++) pre = fma_(w[k].v[v], in[i + k].v[v], pre);
        out.v[v] = a.silu ? silu(pre) : pre;
      }
    }
    store<T, V>(y + (uint64_t)i * a.width, out);
  }
}

// The gradient: with gp[t] = dy[t] act'(pre[t]) (0 outside the sequence), the gradient of past[i]
// is sum_k w[k] gp[i - k], and dw[k] sums gp[t] past[t + k]. A run forms the gp of the K - 1
// positions after it again rather than exchange them. Positions outside the sequence are left out
// rather than multiplied by 0, which an infinite input or weight would make NaN. Bound as the forward
// pass is: 8 x 4096 x 2048 146 us, 5.5 TB/s, 4 x 1024 x 512 9.2 us. The sums for w and the bias stay
// in a lane's registers over its run, meet once in LDS and leave a row a block, of four runs.
template <class T, int K, int V, int R>
__global__ void __launch_bounds__(TPB) k_conv_grad(ConvArgs a, uint32_t nx, uint32_t runs) {
  __shared__ T part[TPB / 64][K + 1][64 * V];
  const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const uint32_t bx = blockIdx.x % nx, by = blockIdx.x / nx;
  const uint32_t b = by / runs, t0 = ((by % runs) * (TPB / 64) + wave) * R;
  const uint32_t d = (bx * 64 + lane) * V;
  const bool active = d < a.width && t0 < a.length;
  Vec<T, V> dw[K], db{};
#pragma unroll
  for (int k = 0; k < K; k++) dw[k] = Vec<T, V>{};
  if (active) {
    const uint32_t n = end_of(a.lengths, b, a.length);
    const T* x = (const T*)a.x + (uint64_t)b * a.length * a.width + d;
    const T* dy = (const T*)a.dy + (uint64_t)b * a.length * a.width + d;
    const T* state = a.state ? (const T*)a.state + (uint64_t)b * (K - 1) * a.width + d : nullptr;
    const T* carry = a.carry ? (const T*)a.carry + (uint64_t)b * (K - 1) * a.width + d : nullptr;
    const uint32_t live = __builtin_amdgcn_readfirstlane(n > t0 ? n - t0 : 0u);  // positions from t0 on; a wave has one t0
    Vec<T, V> w[K], bias{}, in[R + 2 * (K - 1)], g[R + K - 1];
#pragma unroll
    for (int k = 0; k < K; k++) w[k] = load<T, V>((const T*)a.w + (uint64_t)k * a.width + d);
    if (a.bias) bias = load<T, V>((const T*)a.bias + d);
#pragma unroll
    for (int i = 0; i < R + 2 * (K - 1); i++) {
      in[i] = Vec<T, V>{};
      const uint32_t p = t0 + i;
      if (p < n + (K - 1)) {
        if (p >= K - 1) in[i] = load<T, V>(x + (uint64_t)(p - (K - 1)) * a.width);
        else if (state) in[i] = load<T, V>(state + (uint64_t)p * a.width);
      }
    }
#pragma unroll
    for (int i = 0; i < R + K - 1; i++) {
      g[i] = Vec<T, V>{};
      if ((uint32_t)i < live) g[i] = load<T, V>(dy + (uint64_t)(t0 + i) * a.width);
    }
#pragma unroll
    for (int i = 0; i < R + K - 1; i++)
#pragma unroll
      for (int v = 0; v < V; v++) {
        if ((uint32_t)i >= live) continue;
        if (a.silu) {
          T pre = bias.v[v];
#pragma unroll
          for (int k = 0; k < K; k++) pre = fma_(w[k].v[v], in[i + k].v[v], pre);
          g[i].v[v] *= silu_slope(pre, sigmoid(pre));
        }
        if (i < R) {
          db.v[v] += g[i].v[v];
#pragma unroll
          for (int k = 0; k < K; k++) dw[k].v[v] = fma_(g[i].v[v], in[i + k].v[v], dw[k].v[v]);
        }
      }
    T* dx = a.dx ? (T*)a.dx + (uint64_t)b * a.length * a.width + d : nullptr;
    T* dstate = a.dstate ? (T*)a.dstate + (uint64_t)b * (K - 1) * a.width + d : nullptr;
#pragma unroll
    for (int i = 0; i < R + K - 1; i++) {
      // The gradient of past[t0 + i]: of x[t0 + i - K + 1], or in the first run of the state.
      if (i < K - 1 && t0 != 0) continue;
      const uint32_t p = t0 + i;
      Vec<T, V> out{};
#pragma unroll
      for (int k = 0; k < K; k++)
        if (i >= k && (uint32_t)(i - k) < live)
#pragma unroll
          for (int v = 0; v < V; v++) out.v[v] = fma_(w[k].v[v], g[i - k].v[v], out.v[v]);
      if (carry && p >= n && p < n + (K - 1)) {
        const Vec<T, V> c = load<T, V>(carry + (uint64_t)(p - n) * a.width);
#pragma unroll
        for (int v = 0; v < V; v++) out.v[v] += c.v[v];
      }
      if (i < K - 1) {
        if (dstate) store<T, V>(dstate + (uint64_t)p * a.width, out);
      } else if (dx && p - (K - 1) < a.length) {
        store<T, V>(dx + (uint64_t)(p - (K - 1)) * a.width, out);
      }
    }
  }
  if (!a.dw_rows && !a.db_rows) return;
#pragma unroll
  for (int v = 0; v < V; v++) {
#pragma unroll
    for (int k = 0; k < K; k++) part[wave][k][lane * V + v] = dw[k].v[v];
    part[wave][K][lane * V + v] = db.v[v];
  }
  __syncthreads();
  for (uint32_t i = threadIdx.x; i < (K + 1) * 64 * V; i += TPB) {
    const uint32_t k = i / (64 * V), c = i % (64 * V), at = bx * 64 * V + c;
    if (at >= a.width) continue;
    T sum = part[0][k][c];
#pragma unroll
    for (int q = 1; q < TPB / 64; q++) sum += part[q][k][c];
    if (k < K) {
      if (a.dw_rows) ((T*)a.dw_rows)[(uint64_t)by * K * a.width + (uint64_t)k * a.width + at] = sum;
    } else if (a.db_rows) {
      ((T*)a.db_rows)[(uint64_t)by * a.width + at] = sum;
    }
  }
}

template <class F>
void conv_taps(uint32_t taps, F launch) {
  using std::integral_constant;
  switch (taps) {
    case 2: launch(integral_constant<int, 2>()); break;
    case 3: launch(integral_constant<int, 3>()); break;
    case 4: launch(integral_constant<int, 4>()); break;
    case 5: launch(integral_constant<int, 5>()); break;
    case 6: launch(integral_constant<int, 6>()); break;
    case 7: launch(integral_constant<int, 7>()); break;
    case 8: launch(integral_constant<int, 8>()); break;
    default: break;
  }
}

// Channels a lane takes (wide accesses) and the positions of a run (fewer of them read twice), as far
// as that leaves eight waves a SIMD, or of runs two: 8 x 4096 x 2048 takes 90 us forward and 146
// backward with four channels (6.0 and 5.5 TB/s; 95 and 162 with one), 4 x 1024 x 512 5.3 and 9.2 us
// with one (7.1 and 11.6 with four), 5 x 333 x 77 backward 4.6 us in runs of four, 5.6 in runs of eight.
struct ConvCut {
  uint32_t v, r;
};
uint32_t conv_runs(const ConvArgs& a, uint32_t r) { return (a.length + 4 * r - 1) / (4 * r); }
ConvCut conv_cut(int dtype, const ConvArgs& a) {
  auto waves = [&](uint32_t v, uint32_t r) { return (uint64_t)a.batch * conv_runs(a, r) * 4 * ((a.width + 64 * v - 1) / (64 * v)); };
  ConvCut cut{1, a.length <= 4 ? 1u : waves(1, 8) < 2048 ? 4u : 8u};
  for (uint32_t v = dtype == RG_F32 ? 4 : 2; v > 1; v /= 2)
    if (a.width % v == 0 && waves(v, cut.r) >= 8192) {
      cut.v = v;
      break;
    }
  return cut;
}

template <class T, int V, int R, bool GRAD>
void launch_conv(hipStream_t s, const ConvArgs& a) {
  const uint32_t nx = (a.width + 64 * V - 1) / (64 * V), runs = conv_runs(a, R);
  const dim3 grid(nx * runs * a.batch);
  conv_taps(a.taps, [&](auto k) {
    if constexpr (GRAD) hipLaunchKernelGGL((k_conv_grad<T, decltype(k)::value, V, R>), grid, dim3(TPB), 0, s, a, nx, runs);
    else hipLaunchKernelGGL((k_conv<T, decltype(k)::value, V, R>), grid, dim3(TPB), 0, s, a, nx, runs);
  });
}

template <class T, bool GRAD>
void conv(hipStream_t s, int dtype, const ConvArgs& a) {
  constexpr int MOST = sizeof(T) == 4 ? 4 : 2;
  const ConvCut cut = conv_cut(dtype, a);
  auto runs = [&](auto v) {
    constexpr int V = decltype(v)::value;
    if (cut.r == 8) launch_conv<T, V, 8, GRAD>(s, a);
    else if (cut.r == 4) launch_conv<T, V, 4, GRAD>(s, a);
    else launch_conv<T, V, 1, GRAD>(s, a);
  };
  if (cut.v == MOST) runs(std::integral_constant<int, MOST>());
  else if (cut.v == MOST / 2) runs(std::integral_constant<int, MOST / 2>());
  else runs(std::integral_constant<int, 1>());
}

}  // namespace

uint64_t conv_blocks(int dtype, const ConvArgs& a) {
  const ConvCut cut = conv_cut(dtype, a);
  return (uint64_t)a.batch * conv_runs(a, cut.r) * ((a.width + 64 * cut.v - 1) / (64 * cut.v));
}
uint32_t conv_grad_rows(int dtype, const ConvArgs& a) { return a.batch * conv_runs(a, conv_cut(dtype, a).r); }

void causal_conv(hipStream_t s, int dtype, const ConvArgs& a) {
  if (dtype == RG_F32) conv<float, false>(s, dtype, a);
  else conv<double, false>(s, dtype, a);
}
void causal_conv_grad(hipStream_t s, int dtype, const ConvArgs& a) {
  if (dtype == RG_F32) conv<float, true>(s, dtype, a);
  else conv<double, true>(s, dtype, a);
}

// ---- selective scan ---------------------------------------------------------------------------

namespace {

constexpr int TILE = RG_SCAN_MARK;

// NL neighbouring lanes share a channel, NS of its states each; a block holds CH channels, of one
// group. Tiles of TILE positions pass through LDS, channels' values transposed so that a lane
// reads four positions at once.
template <class T_, int NL_, int NS_>
struct ScanShape {
  using T = T_;
  static constexpr int NL = NL_, NS = NS_, NP = NL * NS, CH = TPB / NL, EPT = CH / 16, LD = TILE + 16 / sizeof(T);
  static constexpr int MAPS = (TILE * NP + TPB - 1) / TPB;  // values of b or c a thread brings in a tile
};

// What a block works on: a tile of CH channels of a group, over one chunk of a sequence.
struct ScanPlace {
  uint32_t b, group, tile, chunk;
  uint32_t ch0, chs;        // first channel and how many
  uint32_t first, last;     // tiles of positions, [first, last)
  uint32_t n, marks;        // positions of the sequence; tiles of the padded one
};
template <class S>
__device__ __forceinline__ ScanPlace scan_place(const ScanArgs& a, uint32_t tiles, uint32_t first_chunk, uint32_t chunks, uint32_t chunk_tiles) {
  ScanPlace p;
  const uint32_t per = a.width / a.groups;
  uint32_t at = blockIdx.x;
  p.tile = at % tiles;
  at /= tiles;
  p.group = at % a.groups;
  at /= a.groups;
  p.chunk = at % chunks + first_chunk;
  p.b = at / chunks;
  p.ch0 = p.group * per + p.tile * S::CH;
  p.chs = min((uint32_t)S::CH, per - p.tile * S::CH);
  p.n = end_of(a.lengths, p.b, a.length);
  p.marks = (a.length + TILE - 1) / TILE;
  p.first = p.chunk * chunk_tiles;
  p.last = min(p.marks, p.first + chunk_tiles);
  return p;
}

// The part of a tile that a thread moves: EPT neighbouring channels of one position. A wave moves the
// channels that its own lanes compute, so that what passes through LDS needs no barrier; and no two of
// its lanes use a bank (four channels and four floats between them: rows of 20) at once.
template <class S>
struct ScanMover {
  uint32_t row, col, left;
  bool vec;
  __device__ __forceinline__ ScanMover(const ScanPlace& p, bool v) : row(threadIdx.x % 64 / 4), col((threadIdx.x / 64 * 4 + threadIdx.x % 4) * S::EPT), vec(v) {
    left = col < p.chs ? p.chs - col : 0;
  }
  __device__ __forceinline__ uint64_t at(const ScanArgs& a, const ScanPlace& p, uint32_t m) const {
    return ((uint64_t)p.b * a.length + m * TILE + row) * a.width + p.ch0 + col;
  }
  __device__ __forceinline__ bool inside(const ScanPlace& p, uint32_t m) const { return m * TILE + row < p.n && left > 0; }
  // Zeros outside the sequence.
  template <class T>
  __device__ __forceinline__ Vec<T, S::EPT> load_from(const void* src, uint64_t at, bool inside) const {
    Vec<T, S::EPT> v{};
    if (!inside) return v;
    const T* p = (const T*)src + at;
    if (vec && left >= (uint32_t)S::EPT) return load<T, S::EPT>(p);
#pragma unroll
    for (int j = 0; j < S::EPT; j++)
      if ((uint32_t)j < left) v.v[j] = p[j];
    return v;
  }
  template <class T>
  __device__ __forceinline__ void store_to(void* dst, uint64_t at, const Vec<T, S::EPT>& v, bool within) const {
    if (!dst || !within) return;
    T* p = (T*)dst + at;
    if (vec && left >= (uint32_t)S::EPT) {
      store<T, S::EPT>(p, v);
      return;
    }
#pragma unroll
    for (int j = 0; j < S::EPT; j++)
      if ((uint32_t)j < left) p[j] = v.v[j];
  }
};

// The values of b or c of a tile that a thread brings; zeros outside the sequence.
template <class S>
struct ScanMaps {
  typename S::T v[S::MAPS];
  __device__ __forceinline__ void read(const ScanArgs& a, const ScanPlace& p, const void* src, uint32_t m) {
#pragma unroll
    for (int q = 0; q < S::MAPS; q++) {
      const uint32_t i = threadIdx.x + q * TPB, t = m * TILE + i / S::NP, k = i % S::NP;
      v[q] = typename S::T(0);
      if (i < TILE * S::NP && t < p.n && k < a.states)
        v[q] = ((const typename S::T*)src)[(((uint64_t)p.b * a.length + t) * a.map_stride + p.group) * a.states + k];
    }
  }
  __device__ __forceinline__ void put(typename S::T* dst) const {
#pragma unroll
    for (int q = 0; q < S::MAPS; q++)
      if (threadIdx.x + q * TPB < TILE * S::NP) dst[threadIdx.x + q * TPB] = v[q];
  }
};

// The decay e^(dt a) of one position. In 32 bits `a` comes multiplied by log2 e, for the
// hardware's power of two.
__device__ __forceinline__ float decay(float dt, float a) { return __builtin_amdgcn_exp2f(dt * a); }
__device__ __forceinline__ double decay(double dt, double a) { return exp(dt * a); }
__device__ __forceinline__ float decay_rate(float a) { return a * 1.44269504088896341f; }
__device__ __forceinline__ double decay_rate(double a) { return a; }
// LDS written by lanes of this wave is read by others of it after this.
__device__ __forceinline__ void wave_sync() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}
// Keeps the scheduler from bringing in the operands of later positions of an unrolled tile early,
// which costs more registers than a wave has.
__device__ __forceinline__ void hold(int position) {
  if (position % 4 == 0) __builtin_amdgcn_sched_barrier(0);
}
// An infinite rate becomes a very large finite one: the decay of a step is the same 0 (or infinity),
// and positions outside the sequence, whose steps are 0, leave the state as it is.
__device__ __forceinline__ float finite_rate(float a) { return a > 2e38f ? 2e38f : a < -2e38f ? -2e38f : a; }
__device__ __forceinline__ double finite_rate(double a) { return a > 1e308 ? 1e308 : a < -1e308 ? -1e308 : a; }

// The rate of a decay from the operand's value: itself, or minus its exponential.
template <class T>
__device__ __forceinline__ T rate_of(T v, bool logs) {
  return finite_rate(logs ? -exp_(sizeof(T) == 4 && v > T(88) ? T(88) : v) : v);
}

template <int C>
__device__ __forceinline__ float dpp(float x) {
  return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), C, 0xf, 0xf, false));
}
template <int C>
__device__ __forceinline__ double dpp(double x) {
  const int2 v = __builtin_bit_cast(int2, x);
  return __builtin_bit_cast(double, make_int2(__builtin_amdgcn_update_dpp(0, v.x, C, 0xf, 0xf, false), __builtin_amdgcn_update_dpp(0, v.y, C, 0xf, 0xf, false)));
}
// The sum over the NL lanes of a channel, in all of them: exchanges within quads, then mirrors.
template <int NL, class T>
__device__ __forceinline__ T channel_sum(T v) {
  v += dpp<0xB1>(v);   // quad_perm [1,0,3,2]
  v += dpp<0x4E>(v);   // quad_perm [2,3,0,1]
  if (NL >= 8) v += dpp<0x141>(v);   // row_half_mirror
  if (NL >= 16) v += dpp<0x140>(v);  // row_mirror
  return v;
}

// a + b over both halves (rows) of the wave: a's sum in the lower half (even rows), b's in the
// upper (odd).
__device__ __forceinline__ float halves(float a, float b) {
  const auto p = __builtin_amdgcn_permlane32_swap(__float_as_uint(a), __float_as_uint(b), false, false);
  return __uint_as_float(p[0]) + __uint_as_float(p[1]);
}
__device__ __forceinline__ float rows(float a, float b) {
  const auto p = __builtin_amdgcn_permlane16_swap(__float_as_uint(a), __float_as_uint(b), false, false);
  return __uint_as_float(p[0]) + __uint_as_float(p[1]);
}
__device__ __forceinline__ double halves(double a, double b) {
  const uint2 x = __builtin_bit_cast(uint2, a), y = __builtin_bit_cast(uint2, b);
  const auto lo = __builtin_amdgcn_permlane32_swap(x.x, y.x, false, false), hi = __builtin_amdgcn_permlane32_swap(x.y, y.y, false, false);
  return __builtin_bit_cast(double, make_uint2(lo[0], hi[0])) + __builtin_bit_cast(double, make_uint2(lo[1], hi[1]));
}
__device__ __forceinline__ double rows(double a, double b) {
  const uint2 x = __builtin_bit_cast(uint2, a), y = __builtin_bit_cast(uint2, b);
  const auto lo = __builtin_amdgcn_permlane16_swap(x.x, y.x, false, false), hi = __builtin_amdgcn_permlane16_swap(x.y, y.y, false, false);
  return __builtin_bit_cast(double, make_uint2(lo[0], hi[0])) + __builtin_bit_cast(double, make_uint2(lo[1], hi[1]));
}

// M values of every lane summed over a wave's channels (lanes q, q + NL, q + 2 NL, ...). The sums
// are spread as they halve: out[i] is that of value value_at<M>(i) of this lane, the same in the
// 16 / NL lanes of a row with equal q.
template <int M>
constexpr int SUMS = M >= 4 ? M / 4 : 1;
template <int M>
__device__ __forceinline__ int value_at(int i) {
  const int lane = threadIdx.x % 64, odd = lane / 16 % 2, upper = lane / 32;
  return i + (M >= 4 ? M / 4 * odd : 0) + M / 2 * upper;
}
template <int NL, int M, class T>
__device__ __forceinline__ void sum_channels(const T (&v)[M], T (&out)[SUMS<M>]) {
  T half[M / 2];
#pragma unroll
  for (int i = 0; i < M / 2; i++) half[i] = halves(v[i], v[i + M / 2]);
#pragma unroll
  for (int i = 0; i < SUMS<M>; i++) {
    out[i] = M >= 4 ? rows(half[i], half[(i + M / 4) % (M / 2)]) : rows(half[0], half[0]);
    if (NL <= 8) out[i] += dpp<0x128>(out[i]);  // row_ror:8
    if (NL <= 4) out[i] += dpp<0x124>(out[i]);  // row_ror:4
  }
}

// The NS states from k0 on of a row of them, zeros past the last; `whole`: NS divides their number.
template <class T, int NS>
__device__ __forceinline__ Vec<T, NS> load_states(const void* src, uint64_t row, uint32_t k0, uint32_t states, bool whole) {
  const T* p = (const T*)src + row * states;
  Vec<T, NS> v;
  if (whole) {
    v = load<T, NS>(p + (k0 < states ? k0 : 0));
  } else {
#pragma unroll
    for (int j = 0; j < NS; j++) v.v[j] = p[k0 + j < states ? k0 + j : 0];
  }
#pragma unroll
  for (int j = 0; j < NS; j++)
    if (k0 + j >= states) v.v[j] = T(0);
  return v;
}
template <class T, int NS>
__device__ __forceinline__ void store_states(void* dst, uint64_t row, uint32_t k0, uint32_t states, bool whole, const T (&h)[NS]) {
  T* p = (T*)dst + row * states + k0;
  if (whole) {
    Vec<T, NS> v;
#pragma unroll
    for (int j = 0; j < NS; j++) v.v[j] = h[j];
    if (k0 < states) store<T, NS>(p, v);
    return;
  }
#pragma unroll
  for (int j = 0; j < NS; j++)
    if (k0 + j < states) p[j] = h[j];
}

// A long sequence is cut into chunks. What each makes of an empty state (k_scan_ends) and the sum
// of its steps suffice to start them all: the decay over a chunk is one exponential of that sum,
// so that joining them (k_scan_join) is one product a chunk and state.
//   forward:  end[c]  = state after the chunk's last position, from zero before its first
//   backward: end[c]  = gradient carried out of the chunk's first position, from zero after its last
// Bound by vector instructions, an exponential and four others a state of 29 in all a position and
// lane: 4 x 2048 x 2048, 16 states 59 us forward and 69 backward; 2 x 2048 x 512 12.0 and
// 13.4 us, three quarters of the slots taken by two waves a SIMD.
template <class T, int NL, int NS, bool BACK>
__global__ void __launch_bounds__(TPB) k_scan_ends(ScanArgs a, uint32_t tiles, uint32_t chunks, bool vec) {
  using S = ScanShape<T, NL, NS>;
  __shared__ __align__(16) T sdt[S::CH][S::LD], su[S::CH][S::LD], smaps[2][TILE][S::NP];  // maps of every other tile: one barrier a tile
  const ScanPlace p = scan_place<S>(a, tiles, BACK ? 1 : 0, chunks - 1, a.chunk_tiles);
  const uint32_t c = threadIdx.x / NL, q = threadIdx.x % NL, d = p.ch0 + c;
  const bool on = c < p.chs;
  const bool whole = a.states % NS == 0;
  T rate[NS], h[NS], total = T(0);
  const Vec<T, NS> rates = load_states<T, NS>(a.a, on ? d : p.ch0, q * NS, a.states, whole);
#pragma unroll
  for (int j = 0; j < NS; j++) {
    rate[j] = decay_rate(rate_of(rates.v[j], a.logs));
    h[j] = T(0);
  }
  const ScanMover<S> mv(p, vec);
  const uint32_t count = p.last - p.first;
  Vec<T, S::EPT> dt, u, z{};
  ScanMaps<S> map;
  auto read = [&](uint32_t i) {
    const uint32_t m = BACK ? p.last - 1 - i : p.first + i;
    const bool in = mv.inside(p, m);
    const uint64_t at = mv.at(a, p, m);
    dt = mv.template load_from<T>(a.dt, at, in);
    u = mv.template load_from<T>(BACK ? a.dy : a.x, at, in);
    if (BACK && a.gate) z = mv.template load_from<T>(a.gate, at, in);
    map.read(a, p, BACK ? a.c : a.b, m);
  };
  const Vec<T, S::EPT> bias = mv.template load_from<T>(a.dt_bias, p.ch0 + mv.col, a.dt_bias && mv.left > 0);
  read(0);
  for (uint32_t i = 0; i < count; i++) {
    const bool in = mv.inside(p, BACK ? p.last - 1 - i : p.first + i);
    if (a.dt_bias)
#pragma unroll
      for (int j = 0; j < S::EPT; j++) dt.v[j] = in ? dt.v[j] + bias.v[j] : T(0);
    if (a.softplus)
#pragma unroll
      for (int j = 0; j < S::EPT; j++) {
        const T soft = softplus(dt.v[j]);
        dt.v[j] = in ? soft : T(0);
      }
    if (BACK && a.gate)
#pragma unroll
      for (int j = 0; j < S::EPT; j++) u.v[j] *= silu(z.v[j]);
#pragma unroll
    for (int j = 0; j < S::EPT; j++) {
      sdt[mv.col + j][mv.row] = dt.v[j];
      su[mv.col + j][mv.row] = u.v[j];
    }
    auto& smap = smaps[i % 2];
    map.put(&smap[0][0]);
    __syncthreads();
    if (i + 1 < count) read(i + 1);
#pragma unroll
    for (int k = 0; k < TILE; k++) {
      hold(k);
      const int t = BACK ? TILE - 1 - k : k;
      const T step = sdt[c][t], v = su[c][t];
      total += step;
#pragma unroll
      for (int j = 0; j < NS; j++) {
        const T e = decay(step, rate[j]), w = smap[t][q * NS + j];
        h[j] = BACK ? e * fma_(v, w, h[j]) : fma_(e, h[j], step * v * w);
      }
    }
    wave_sync();
  }
  if (!on) return;
  const uint64_t at = ((uint64_t)p.b * chunks + p.chunk) * a.width + d;
  store_states<T, NS>(a.ends, at, q * NS, a.states, whole, h);
  if (q == 0) ((T*)a.totals)[at] = total;
}

// Chunks' ends into their starts, in place: the state carried from the sequence's start (backward:
// the gradient from its end) to each chunk, a thread a state. Bound by the latency of its loads:
// the operands of 32 chunks are in flight at a time. Where states grow, the decay over a chunk may
// overflow though its product with a small state does not: it is applied in two halves, and an empty
// state stays empty.
template <class T, bool BACK>
__global__ void __launch_bounds__(64) k_scan_join(ScanArgs a, uint32_t chunks) {
  const uint32_t i = blockIdx.x * 64 + threadIdx.x;
  if (i >= a.batch * a.width * a.states) return;
  const uint32_t k = i % a.states, d = i / a.states % a.width, b = i / a.states / a.width;
  const T rate = decay_rate(rate_of(((const T*)a.a)[(uint64_t)d * a.states + k], a.logs));
  const T* given = (const T*)(BACK ? a.carry : a.state);
  T h = given ? given[i] : T(0);
  constexpr uint32_t FLIGHT = 32;
  auto row = [&](uint32_t c) { return ((uint64_t)b * chunks + (BACK ? chunks - 1 - c : c)) * a.width + d; };
  for (uint32_t c = 0; c < chunks; c += FLIGHT) {
    T end[FLIGHT], total[FLIGHT];
#pragma unroll
    for (uint32_t j = 0; j < FLIGHT; j++) {
      const uint64_t r = row(min(c + j, chunks - 1));
      total[j] = ((const T*)a.totals)[r];
      end[j] = ((const T*)a.ends)[r * a.states + k];
    }
    // Backward the compiler would use each load as it comes (256 chunks 44 us, 28 so; forward 19, 27).
    if (BACK) __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (uint32_t j = 0; j < FLIGHT; j++) {
      if (c + j >= chunks) break;
      ((T*)a.ends)[row(c + j) * a.states + k] = h;
      const T half = decay(T(0.5) * total[j], rate);
      h = h == T(0) ? end[j] : fma_(half, half * h, end[j]);
    }
  }
}

// Forward: h[t] = e^(dt a) h[t - 1] + dt x b, y = c . h + d x, gated. Each lane's states stay in
// registers, x, dt, z and y pass once (2 x 2048 x 512 moves 34 MB, 6.5 us of the 18.2 it takes); bound by
// vector instructions, of which an exponential and four others a state are the recurrence, and what a
// lane does for its channel (its part of a softplus and a gate, the sum over the lanes, five reads of
// LDS) is spread over four states: 4 x 2048 x 2048, 16 states 94 us. Two states a lane took 23.8 us
// where four took 19, eight 31.5 (twice the chunks for as many waves).
template <class T, int NL, int NS>
__global__ void __launch_bounds__(TPB) k_scan(ScanArgs a, uint32_t tiles, uint32_t chunks, bool vec) {
  using S = ScanShape<T, NL, NS>;
  __shared__ __align__(16) T sx[S::CH][S::LD], sdt[S::CH][S::LD], sbs[2][TILE][S::NP], scs[2][TILE][S::NP];
  const ScanPlace p = scan_place<S>(a, tiles, 0, chunks, a.chunk_tiles);
  const uint32_t c = threadIdx.x / NL, q = threadIdx.x % NL, d = p.ch0 + c;
  const bool on = c < p.chs;
  const bool whole = a.states % NS == 0;
  T rate[NS], h[NS];
  const Vec<T, NS> rates = load_states<T, NS>(a.a, on ? d : p.ch0, q * NS, a.states, whole);
  Vec<T, NS> from{};
  if (on && chunks > 1) from = load_states<T, NS>(a.ends, ((uint64_t)p.b * chunks + p.chunk) * a.width + d, q * NS, a.states, whole);
  else if (on && a.state) from = load_states<T, NS>(a.state, (uint64_t)p.b * a.width + d, q * NS, a.states, whole);
#pragma unroll
  for (int j = 0; j < NS; j++) {
    rate[j] = decay_rate(rate_of(rates.v[j], a.logs));
    h[j] = from.v[j];
  }
  const T skip = on && q == 0 && a.skip ? ((const T*)a.skip)[d] : T(0);
  const ScanMover<S> mv(p, vec);
  Vec<T, S::EPT> x, dt, z{};
  ScanMaps<S> bs, cs;
  auto read = [&](uint32_t m) {
    const bool in = mv.inside(p, m);
    const uint64_t at = mv.at(a, p, m);
    x = mv.template load_from<T>(a.x, at, in);
    dt = mv.template load_from<T>(a.dt, at, in);
    if (a.gate) z = mv.template load_from<T>(a.gate, at, in);
    bs.read(a, p, a.b, m);
    cs.read(a, p, a.c, m);
  };
  const Vec<T, S::EPT> bias = mv.template load_from<T>(a.dt_bias, p.ch0 + mv.col, a.dt_bias && mv.left > 0);
  read(p.first);
  for (uint32_t m = p.first; m < p.last; m++) {
    const bool in = mv.inside(p, m);
    if (a.dt_bias)
#pragma unroll
      for (int j = 0; j < S::EPT; j++) dt.v[j] = in ? dt.v[j] + bias.v[j] : T(0);
    if (a.softplus)
#pragma unroll
      for (int j = 0; j < S::EPT; j++) {
        const T soft = softplus(dt.v[j]);
        dt.v[j] = in ? soft : T(0);
      }
#pragma unroll
    for (int j = 0; j < S::EPT; j++) {
      sx[mv.col + j][mv.row] = x.v[j];
      sdt[mv.col + j][mv.row] = dt.v[j];
    }
    auto &sb = sbs[m % 2], &sc = scs[m % 2];
    bs.put(&sb[0][0]);
    cs.put(&sc[0][0]);
    const Vec<T, S::EPT> gate = z;
    __syncthreads();
    if (m + 1 < p.last) read(m + 1);
    if (a.marks && on) store_states<T, NS>(a.marks, ((uint64_t)p.b * p.marks + m) * a.width + d, q * NS, a.states, whole, h);
    T mine = T(0);
#pragma unroll
    for (int i = 0; i < TILE; i++) {
      hold(i);
      const T step = sdt[c][i], u = sx[c][i], drive = step * u;
      T y = skip * u;
#pragma unroll
      for (int j = 0; j < NS; j++) {
        h[j] = fma_(decay(step, rate[j]), h[j], drive * sb[i][q * NS + j]);
        y = fma_(sc[i][q * NS + j], h[j], y);
      }
      y = channel_sum<NL>(y);
      if (i % NL == (int)q) mine = y;
      if (i % NL == NL - 1) sx[c][i - (NL - 1) + q] = mine;
    }
    wave_sync();
    Vec<T, S::EPT> y;
#pragma unroll
    for (int j = 0; j < S::EPT; j++) y.v[j] = in ? sx[mv.col + j][mv.row] : T(0);
    if (a.gate)
#pragma unroll
      for (int j = 0; j < S::EPT; j++) y.v[j] *= silu(gate.v[j]);
    mv.store_to(a.y, mv.at(a, p, m), y, m * TILE + mv.row < a.length);
    wave_sync();
  }
  if (a.last && on && p.last == p.marks) store_states<T, NS>(a.last, (uint64_t)p.b * a.width + d, q * NS, a.states, whole, h);
}

// A few positions, single tokens above all: no tiles, every operand of a position loaded at once.
// Bound by the latency of one round of loads, and for many sequences by the states, read and
// written once (16 x 2048 channels, 16 states, one position: 4 MB).
constexpr uint32_t SCAN_FEW = 4;
template <class T, int NL, int NS>
__global__ void __launch_bounds__(TPB) k_scan_few(ScanArgs a, uint32_t tiles) {
  using S = ScanShape<T, NL, NS>;
  const ScanPlace p = scan_place<S>(a, tiles, 0, 1, a.chunk_tiles);
  const uint32_t c = threadIdx.x / NL, q = threadIdx.x % NL, d = p.ch0 + c;
  if (c >= p.chs) return;  // whole channels: the lanes that sum stay together
  const bool whole = a.states % NS == 0;
  const Vec<T, NS> rates = load_states<T, NS>(a.a, d, q * NS, a.states, whole);
  Vec<T, NS> from{};
  if (a.state) from = load_states<T, NS>(a.state, (uint64_t)p.b * a.width + d, q * NS, a.states, whole);
  const T skip = q == 0 && a.skip ? ((const T*)a.skip)[d] : T(0);
  const T bias = a.dt_bias ? ((const T*)a.dt_bias)[d] : T(0);
  T rate[NS], h[NS];
#pragma unroll
  for (int j = 0; j < NS; j++) {
    rate[j] = decay_rate(rate_of(rates.v[j], a.logs));
    h[j] = from.v[j];
  }
  for (uint32_t t = 0; t < a.length; t++) {
    const uint64_t at = ((uint64_t)p.b * a.length + t) * a.width + d, row = ((uint64_t)p.b * a.length + t) * a.map_stride + p.group;
    T y = T(0);
    if (t < p.n) {
      const T u = ((const T*)a.x)[at];
      T step = ((const T*)a.dt)[at], z = T(0);
      if (a.gate) z = ((const T*)a.gate)[at];
      const Vec<T, NS> b = load_states<T, NS>(a.b, row, q * NS, a.states, whole), m = load_states<T, NS>(a.c, row, q * NS, a.states, whole);
      step += bias;
      if (a.softplus) step = softplus(step);
      const T drive = step * u;
      y = skip * u;
#pragma unroll
      for (int j = 0; j < NS; j++) {
        h[j] = fma_(decay(step, rate[j]), h[j], drive * b.v[j]);
        y = fma_(m.v[j], h[j], y);
      }
      y = channel_sum<NL>(y);
      if (a.gate) y *= silu(z);
    }
    if (a.y && q == 0) ((T*)a.y)[at] = y;
  }
  if (a.last) store_states<T, NS>(a.last, (uint64_t)p.b * a.width + d, q * NS, a.states, whole, h);
}

// Backward, tile by tile from the last of `split` chunks. From the state kept before the tile, its decays e
// and the decayed states p = e h[t - 1] are formed again, then with G = dL/dh[t] carried back:
//   dx = dt sum G b + d gy, ddt = x sum G b + sum G p a, da += dt G p, db = G dt x, dc = gy h.
// The sums over channels that db and dc take leave one partial row per tile of channels.
// Bound by vector instructions, 120 a position and lane of which 56 are the formulas' own: 2 x 2048 x
// 512, 16 states 46 us, 78 % of the slots taken by two waves a SIMD; 4 x 2048 x 2048 332 us. A tile's
// decays and decayed states fill 128 registers; two states a lane would leave room for three waves but
// share what is done for a channel among fewer (57.6 us, 48 then).
template <class T, int NL, int NS, bool GATE>
__global__ void __launch_bounds__(TPB, sizeof(T) == 8 && NS > 1 ? 1 : 2) k_scan_grad(ScanArgs a, uint32_t tiles, uint32_t chunks, bool vec) {
  using S = ScanShape<T, NL, NS>;
  constexpr int WAVES = TPB / 64, COPIES = 16 / NL, M = 2 * NS;
  __shared__ __align__(16) T sx[S::CH][S::LD], sdt[S::CH][S::LD], sg[S::CH][S::LD], sy[S::CH][S::LD], sb[TILE][S::NP], sc[TILE][S::NP];
  __shared__ T red[WAVES][TILE][2 * S::NP];
  __shared__ __align__(16) T sbias[S::CH], sdbias[TILE][S::CH];  // the steps' bias, and each thread's sums for its gradient
  // A thread's d dt / d raw and dy silu'(z), kept here while a tile's states fill the registers.
  __shared__ __align__(16) T sslope[TILE][S::CH], sgate[TILE][S::CH];
  const ScanPlace p = scan_place<S>(a, tiles, 0, chunks, a.chunk_tiles * a.split);
  const uint32_t c = threadIdx.x / NL, q = threadIdx.x % NL, d = p.ch0 + c, wave = threadIdx.x / 64;
  const int copy = threadIdx.x % 16 / NL;
  const bool on = c < p.chs;
  const bool whole = a.states % NS == 0;
  T rate[NS], rate_e[NS], back[NS], da[NS], dd = T(0);
  const Vec<T, NS> rates = load_states<T, NS>(a.a, on ? d : p.ch0, q * NS, a.states, whole);
  Vec<T, NS> from{};
  if (on && a.chunks > 1)
    from = load_states<T, NS>(a.ends, ((uint64_t)p.b * a.chunks + min((p.chunk + 1) * a.split, a.chunks) - 1) * a.width + d, q * NS, a.states, whole);
  else if (on && a.carry) from = load_states<T, NS>(a.carry, (uint64_t)p.b * a.width + d, q * NS, a.states, whole);
#pragma unroll
  for (int j = 0; j < NS; j++) {
    // A lane without a channel may have a step (softplus of 0): with a rate of 0 its decays are 1, where a
    // growing rate's overflow would reach the sums over channels as infinity times 0.
    rate[j] = on ? rate_of(rates.v[j], a.logs) : T(0);
    rate_e[j] = decay_rate(rate[j]);
    back[j] = from.v[j];
    da[j] = T(0);
  }
  const T skip = on && a.skip ? ((const T*)a.skip)[d] : T(0);
  const ScanMover<S> mv(p, vec);
  Vec<T, S::EPT> x, raw, g, z{};
  ScanMaps<S> bs, cs;
  Vec<T, NS> start{};
  auto read = [&](uint32_t m) {
    const bool in = mv.inside(p, m);
    const uint64_t at = mv.at(a, p, m);
    x = mv.template load_from<T>(a.x, at, in);
    raw = mv.template load_from<T>(a.dt, at, in);
    g = mv.template load_from<T>(a.dy, at, in);
    if (GATE) z = mv.template load_from<T>(a.gate, at, in);
    bs.read(a, p, a.b, m);
    cs.read(a, p, a.c, m);
    if (on) start = load_states<T, NS>(a.marks, ((uint64_t)p.b * p.marks + m) * a.width + d, q * NS, a.states, whole);
  };
  read(p.last - 1);
  if (a.dt_bias) {
    if (threadIdx.x < S::CH) sbias[threadIdx.x] = threadIdx.x < p.chs ? ((const T*)a.dt_bias)[p.ch0 + threadIdx.x] : T(0);
    store<T, S::EPT>(&sdbias[mv.row][mv.col], Vec<T, S::EPT>{});
    __syncthreads();
  }
  for (uint32_t m = p.last; m-- > p.first;) {
    const bool in = mv.inside(p, m);
    if (a.dt_bias) {
      const Vec<T, S::EPT> bias = load<T, S::EPT>(&sbias[mv.col]);
#pragma unroll
      for (int j = 0; j < S::EPT; j++) raw.v[j] = in ? raw.v[j] + bias.v[j] : T(0);
    }
    Vec<T, S::EPT> slope, gate_g;
    Vec<T, S::EPT> step = raw, gy = g;
    if (a.softplus) {
#pragma unroll
      for (int j = 0; j < S::EPT; j++) {
        const T soft = softplus(raw.v[j], &slope.v[j]);
        step.v[j] = in ? soft : T(0);
      }
    } else {
#pragma unroll
      for (int j = 0; j < S::EPT; j++) slope.v[j] = T(1);
    }
    if (GATE)
#pragma unroll
      for (int j = 0; j < S::EPT; j++) {
        const T s = sigmoid(z.v[j]);
        gate_g.v[j] = g.v[j] * silu_slope(z.v[j], s);
        gy.v[j] = g.v[j] * (z.v[j] * s);
      }
    store<T, S::EPT>(&sslope[mv.row][mv.col], slope);
    if (GATE) store<T, S::EPT>(&sgate[mv.row][mv.col], gate_g);
#pragma unroll
    for (int j = 0; j < S::EPT; j++) {
      sx[mv.col + j][mv.row] = x.v[j];
      sdt[mv.col + j][mv.row] = step.v[j];
      sg[mv.col + j][mv.row] = gy.v[j];
    }
    bs.put(&sb[0][0]);
    cs.put(&sc[0][0]);
    T h[NS];
#pragma unroll
    for (int j = 0; j < NS; j++) h[j] = start.v[j];
    __syncthreads();
    if (m > p.first) read(m - 1);
    T e[TILE][NS], kept[TILE][NS], mine = T(0), mine2 = T(0);
#pragma unroll
    for (int i = 0; i < TILE; i++) {
      hold(i);
      const T step = sdt[c][i], u = sx[c][i], drive = step * u;
      T y = q == 0 ? skip * u : T(0);
#pragma unroll
      for (int j = 0; j < NS; j++) {
        e[i][j] = decay(step, rate_e[j]);
        kept[i][j] = e[i][j] * h[j];
        h[j] = fma_(drive, sb[i][q * NS + j], kept[i][j]);
        y = fma_(sc[i][q * NS + j], h[j], y);
      }
      if (GATE) {
        y = channel_sum<NL>(y);
        if (i % NL == (int)q) mine = y;
        if (i % NL == NL - 1) sy[c][i - (NL - 1) + q] = mine;
      }
    }
    T sums[SUMS<M>];
#pragma unroll
    for (int i = TILE - 1; i >= 0; i--) {
      hold(i + 1);
      const T step = sdt[c][i], u = sx[c][i], gy = sg[c][i], drive = step * u;
      T sum_b = T(0), sum_a = T(0), over[M];
#pragma unroll
      for (int j = 0; j < NS; j++) {
        const T bj = sb[i][q * NS + j], G = fma_(gy, sc[i][q * NS + j], back[j]), gp = G * kept[i][j];
        over[j] = G * drive;
        over[NS + j] = gy * fma_(drive, bj, kept[i][j]);
        sum_b = fma_(G, bj, sum_b);
        sum_a = fma_(gp, rate[j], sum_a);
        da[j] = fma_(gp, step, da[j]);
        back[j] = e[i][j] * G;
      }
      dd = fma_(gy, u, dd);
      T of[SUMS<M>];
      sum_channels<NL>(over, of);
#pragma unroll
      for (int k = 0; k < SUMS<M>; k++) {
        if (i % COPIES == copy) sums[k] = of[k];
        if (i % COPIES == 0) red[wave][i + copy][value_at<M>(k) * NL + q] = sums[k];
      }
      sum_b = channel_sum<NL>(sum_b);
      sum_a = channel_sum<NL>(sum_a);
      const T dx = fma_(step, sum_b, skip * gy), ddt = fma_(u, sum_b, sum_a);
      if (i % NL == (int)q) mine = dx, mine2 = ddt;
      if (i % NL == 0) {
        sx[c][i + q] = mine;
        sdt[c][i + q] = mine2;
      }
    }
    __syncthreads();
    Vec<T, S::EPT> dx, ddt, dz;
    slope = load<T, S::EPT>(&sslope[mv.row][mv.col]);
    if (GATE) gate_g = load<T, S::EPT>(&sgate[mv.row][mv.col]);
#pragma unroll
    for (int j = 0; j < S::EPT; j++) {
      dx.v[j] = in ? sx[mv.col + j][mv.row] : T(0);
      ddt.v[j] = in ? sdt[mv.col + j][mv.row] * slope.v[j] : T(0);
      dz.v[j] = in && GATE ? sy[mv.col + j][mv.row] * gate_g.v[j] : T(0);
    }
    if (a.dt_bias) {
      Vec<T, S::EPT> sum = load<T, S::EPT>(&sdbias[mv.row][mv.col]);
#pragma unroll
      for (int j = 0; j < S::EPT; j++) sum.v[j] += ddt.v[j];
      store<T, S::EPT>(&sdbias[mv.row][mv.col], sum);
    }
    const bool within = m * TILE + mv.row < a.length;
    const uint64_t at = mv.at(a, p, m);
    mv.store_to(a.dx, at, dx, within);
    mv.store_to(a.ddt, at, ddt, within);
    if (GATE) mv.store_to(a.dz, at, dz, within);
    for (uint32_t i = threadIdx.x; i < TILE * 2 * S::NP; i += TPB) {
      // Value w NS + j of lane q is the gradient of b (w = 0) or c of state q NS + j.
      const uint32_t r = i / (2 * S::NP), w = i / S::NP % 2, k = i % S::NP, t = m * TILE + r;
      T* to = (T*)(w ? a.dc_rows : a.db_rows);
      if (!to || k >= a.states || t >= a.length) continue;
      const uint32_t from = (w * NS + k % NS) * NL + k / NS;
      T sum = T(0);
      if (t < p.n)
#pragma unroll
        for (int v = 0; v < WAVES; v++) sum += red[v][r][from];
      const uint64_t rows = (uint64_t)a.batch * a.length * a.map_stride * a.states;
      to[p.tile * rows + (((uint64_t)p.b * a.length + t) * a.map_stride + p.group) * a.states + k] = sum;
    }
    wave_sync();
  }
  if (a.dt_bias) __syncthreads();
  const uint64_t row = (uint64_t)p.b * chunks + p.chunk;
  if (a.dt_bias_rows && threadIdx.x < p.chs) {
    T sum = T(0);
#pragma unroll
    for (int t = 0; t < TILE; t++) sum += sdbias[t][threadIdx.x];
    ((T*)a.dt_bias_rows)[row * a.width + p.ch0 + threadIdx.x] = sum;
  }
  if (!on) return;
  if (a.logs)
#pragma unroll
    for (int j = 0; j < NS; j++) da[j] *= rate[j];
  if (a.da_rows) store_states<T, NS>(a.da_rows, row * a.width + d, q * NS, a.states, whole, da);
  if (a.dstate && p.chunk == 0) store_states<T, NS>(a.dstate, (uint64_t)p.b * a.width + d, q * NS, a.states, whole, back);
  if (a.dd_rows && q == 0) ((T*)a.dd_rows)[row * a.width + d] = dd;
}

// The lanes and states a channel is spread over: f(NL, NS).
template <class T, class F>
void scan_shape(uint32_t states, F f) {
  using std::integral_constant;
  if constexpr (sizeof(T) == 4) {
    if (states <= 4) f(integral_constant<int, 4>(), integral_constant<int, 1>());
    else if (states <= 8) f(integral_constant<int, 4>(), integral_constant<int, 2>());
    else if (states <= 16) f(integral_constant<int, 4>(), integral_constant<int, 4>());
    else if (states <= 32) f(integral_constant<int, 8>(), integral_constant<int, 4>());
    else f(integral_constant<int, 16>(), integral_constant<int, 4>());
  } else {
    if (states <= 8) f(integral_constant<int, 8>(), integral_constant<int, 1>());
    else if (states <= 16) f(integral_constant<int, 16>(), integral_constant<int, 1>());
    else if (states <= 32) f(integral_constant<int, 16>(), integral_constant<int, 2>());
    else f(integral_constant<int, 16>(), integral_constant<int, 4>());
  }
}

// Tiles of a group's channels, and the chunks a sequence is cut into: as many as bring the launch to
// SCAN_BLOCKS blocks, two a CU (3 x 777 x 200, 8 states: 25 chunks 46 us forward and backward, 13
// chunks 62). Joining takes about 0.2 us a chunk and a tile of positions 6 us, both ways, so that few
// channels are cut into no more than 4 sqrt(tiles) chunks (2 x 2048 x 512, 16 states: 64 chunks take a
// tenth longer than 32). Chunks of four tiles or more are cut further, to eight blocks a CU, whose waves
// cover each other's latency (4 x 2048 x 2048, 16 states: 16 chunks 169 us forward, 4 chunks 209 then; 2 x
// 2048 x 512, 64 states 87 and 100). k_scan_grad has registers for two blocks a CU and takes `split` of
// those chunks a block.
constexpr uint32_t SCAN_BLOCKS = 512, SCAN_MOST_BLOCKS = 2048;

struct ScanCut {
  uint32_t tiles = 1, chunk_tiles = 1, chunks = 1, split = 1, runs = 1;
};
template <class T>
ScanCut scan_cut(const ScanArgs& a, bool grad) {
  ScanCut cut;
  scan_shape<T>(a.states, [&](auto nl, auto) {
    const uint32_t ch = TPB / decltype(nl)::value;
    cut.tiles = (a.width / a.groups + ch - 1) / ch;
  });
  const uint32_t marks = (a.length + TILE - 1) / TILE;
  const uint64_t blocks = (uint64_t)a.batch * a.groups * cut.tiles, most = (uint64_t)std::ceil(4.0 * std::sqrt((double)marks));
  auto filling = [&](uint64_t n) { return std::min((n + blocks - 1) / blocks, most); };
  const uint64_t few = filling(SCAN_BLOCKS), wanted = std::max(few, std::min<uint64_t>(filling(SCAN_MOST_BLOCKS), marks / 4));
  cut.chunk_tiles = (uint32_t)((marks + wanted - 1) / wanted);
  cut.chunks = (marks + cut.chunk_tiles - 1) / cut.chunk_tiles;
  if (grad) cut.split = (uint32_t)((cut.chunks + few - 1) / few);
  cut.runs = (cut.chunks + cut.split - 1) / cut.split;
  return cut;
}
ScanCut scan_cut_of(int dtype, const ScanArgs& a, bool grad) { return dtype == RG_F32 ? scan_cut<float>(a, grad) : scan_cut<double>(a, grad); }

template <class T, bool GRAD>
void launch_scan(hipStream_t s, ScanArgs a) {
  const ScanCut cut = scan_cut<T>(a, GRAD);
  a.chunk_tiles = cut.chunk_tiles;
  a.chunks = cut.chunks;
  a.split = cut.split;
  a.ends = a.workspace;
  a.totals = (T*)a.workspace + (uint64_t)a.batch * cut.chunks * a.width * a.states;
  scan_shape<T>(a.states, [&](auto nl, auto ns) {
    constexpr int NL = decltype(nl)::value, NS = decltype(ns)::value, EPT = ScanShape<T, NL, NS>::EPT;
    const bool vec = a.width % EPT == 0 && (a.width / a.groups) % EPT == 0;
    const uint32_t blocks = a.batch * a.groups * cut.tiles;
    if (!GRAD && a.length <= SCAN_FEW && !a.marks) {
      hipLaunchKernelGGL((k_scan_few<T, NL, NS>), dim3(blocks), dim3(TPB), 0, s, a, cut.tiles);
      return;
    }
    if (cut.chunks > 1) {
      const uint32_t joins = (a.batch * a.width * a.states + 63) / 64;
      hipLaunchKernelGGL((k_scan_ends<T, NL, NS, GRAD>), dim3(blocks * (cut.chunks - 1)), dim3(TPB), 0, s, a, cut.tiles, cut.chunks, vec);
      hipLaunchKernelGGL((k_scan_join<T, GRAD>), dim3(joins), dim3(64), 0, s, a, cut.chunks);
    }
    const dim3 grid(blocks * cut.runs);
    if constexpr (GRAD) {
      if (a.gate) hipLaunchKernelGGL((k_scan_grad<T, NL, NS, true>), grid, dim3(TPB), 0, s, a, cut.tiles, cut.runs, vec);
      else hipLaunchKernelGGL((k_scan_grad<T, NL, NS, false>), grid, dim3(TPB), 0, s, a, cut.tiles, cut.runs, vec);
    } else {
      hipLaunchKernelGGL((k_scan<T, NL, NS>), grid, dim3(TPB), 0, s, a, cut.tiles, cut.runs, vec);
    }
  });
}

}  // namespace

uint64_t scan_blocks(int dtype, const ScanArgs& a) {
  const ScanCut cut = scan_cut_of(dtype, a, false);
  return (uint64_t)a.batch * a.groups * cut.tiles * cut.chunks;
}
uint32_t scan_rows(int dtype, const ScanArgs& a) { return a.batch * scan_cut_of(dtype, a, true).runs; }
uint32_t scan_group_tiles(int dtype, const ScanArgs& a) { return scan_cut_of(dtype, a, true).tiles; }
uint64_t scan_workspace(int dtype, const ScanArgs& a) {
  const uint32_t chunks = scan_cut_of(dtype, a, true).chunks;
  return chunks > 1 ? (uint64_t)a.batch * chunks * a.width * (a.states + 1) * (dtype == RG_F64 ? 8 : 4) : 0;
}

void selective_scan(hipStream_t s, int dtype, const ScanArgs& a) {
  if (dtype == RG_F32) launch_scan<float, false>(s, a);
  else launch_scan<double, false>(s, a);
}
void selective_scan_grad(hipStream_t s, int dtype, const ScanArgs& a) {
  if (dtype == RG_F32) launch_scan<float, true>(s, a);
  else launch_scan<double, true>(s, a);
}

// ---- norm with rotation -----------------------------------------------------------------------

namespace {

// Sine and cosine of f turns, |f| <= 1/2: the nearest quarter taken off in 64 bits, then the Taylor
// series of the remaining angle, at most pi / 4, whose next terms are below 2e-9.
__device__ __forceinline__ void sin_cos_turns(double f, float* sn, float* cs) {
  const double quarter = rint(4.0 * f);
  const float t = (float)(fma(quarter, -0.25, f) * 6.283185307179586477), w = t * t;
  const int q = (int)quarter;
  float s = fma_(w, 2.7557319e-6f, -1.9841270e-4f);
  s = fma_(w, s, 8.3333333e-3f);
  s = fma_(w, s, -1.6666667e-1f);
  s = fma_(t * w, s, t);
  float c = fma_(w, -2.7557319e-7f, 2.4801587e-5f);
  c = fma_(w, c, -1.3888889e-3f);
  c = fma_(w, c, 4.1666667e-2f);
  c = fma_(w, c, -0.5f);
  c = fma_(w, c, 1.0f);
  const float x = q & 1 ? c : s, y = q & 1 ? s : c;
  *sn = q & 2 ? -x : x;
  *cs = (q + 1) & 2 ? -y : y;
}
__device__ __forceinline__ void sin_cos_turns(double f, double* sn, double* cs) { sincospi(2.0 * f, sn, cs); }

// The sum over the LG lanes of a group, in all of them (every lane of the wave takes part).
template <int LG, class T>
__device__ __forceinline__ T group_sum(T v) {
  v = channel_sum<LG>(v);
  if (LG >= 32) v = rows(v, v);
  if (LG >= 64) v = halves(v, v);
  return v;
}

// LG lanes share a head, each with UPL units of V pairs: both halves of a pair lie in one lane, so
// the turn needs no exchange. A group of lanes keeps one head, its gain and its angles per position
// in registers and walks the tokens. Bound by memory: 4 x 1024 x 24 heads of 64, the values' passing,
// are 50 MB forward, 11 us or 4.7 TB/s, and 75 MB backward, 18 us or 4.2 TB/s; 8 x 4096 x 48 heads of 128
// 337 and 507 us, 4.8 both.
template <class T, int V, int LG, int UPL, bool GRAD>
__global__ void __launch_bounds__(TPB) k_rotary(RotaryArgs a) {
  constexpr int GROUPS = TPB / LG;
  const uint32_t group = blockIdx.x * GROUPS + threadIdx.x / LG, lane = threadIdx.x % LG;
  const uint32_t walkers = gridDim.x * GROUPS / a.heads, steps = (a.batch * a.length + walkers - 1) / walkers;
  const uint32_t head = group % a.heads, first = group / a.heads;
  const uint32_t half = a.turn / 2, rest = (a.head - a.turn) / 2, tokens = a.batch * a.length;
  uint32_t section = 0;
  while (section < a.sections && head >= a.last[section]) section++;
  const bool on = first < walkers, used = section < a.sections, normed = used && a.normed;
  // Where this lane's units lie in a head: their first and second halves.
  uint32_t lo[UPL], hi[UPL];
  bool has[UPL];
  Vec<T, V> g_lo[UPL], g_hi[UPL], d_lo[UPL], d_hi[UPL];
  double2 turns[UPL][V];
#pragma unroll
  for (int k = 0; k < UPL; k++) {
    const uint32_t u = (lane + k * LG) * V;
    has[k] = u < a.head / 2;
    lo[k] = u < half ? u : a.turn + (u - half);
    hi[k] = lo[k] + (u < half ? half : rest);
    d_lo[k] = d_hi[k] = Vec<T, V>{};
#pragma unroll
    for (int v = 0; v < V; v++) {
      g_lo[k].v[v] = g_hi[k].v[v] = T(1);
      turns[k][v] = has[k] && used && u + v < half ? a.turns[u + v] : make_double2(0.0, 0.0);
    }
    if (has[k] && normed) {
      g_lo[k] = load<T, V>((const T*)a.gain + section * a.head + lo[k]);
      g_hi[k] = load<T, V>((const T*)a.gain + section * a.head + hi[k]);
    }
  }
  for (uint32_t i = 0; i < steps; i++) {
    const uint32_t token = first + i * walkers;
    const bool valid = on && token < tokens;
    const uint64_t at = ((uint64_t)token * a.heads + head) * a.head;
    double pos = 0.0;
    if (valid) {
      const uint32_t b = token / a.length, t = token - b * a.length;
      pos = a.positions_from ? (double)a.positions[b] + (double)t : (double)a.positions[a.shared_positions ? t : token];
    }
    Vec<T, V> x_lo[UPL], x_hi[UPL], w_lo[UPL], w_hi[UPL];
    T ss = T(0);
#pragma unroll
    for (int k = 0; k < UPL; k++) {
      x_lo[k] = x_hi[k] = w_lo[k] = w_hi[k] = Vec<T, V>{};
      if (valid && has[k]) {
        x_lo[k] = load<T, V>((const T*)a.x + at + lo[k]);
        x_hi[k] = load<T, V>((const T*)a.x + at + hi[k]);
        if (GRAD) {
          w_lo[k] = load<T, V>((const T*)a.dy + at + lo[k]);
          w_hi[k] = load<T, V>((const T*)a.dy + at + hi[k]);
        }
      }
#pragma unroll
      for (int v = 0; v < V; v++) ss = fma_(x_lo[k].v[v], x_lo[k].v[v], fma_(x_hi[k].v[v], x_hi[k].v[v], ss));
    }
    ss = group_sum<LG>(ss);
    // A group without a token adds nothing: 1, as eps may be 0 and 0 / 0 would reach the gain's sums.
    const T r = normed && valid ? T(1) / sqrt_(ss / T(a.head) + T(a.eps)) : T(1);
    T mean = T(0);
#pragma unroll
    for (int k = 0; k < UPL; k++) {
#pragma unroll
      for (int v = 0; v < V; v++) {
        T sn, cs;
        const double2 turn = turns[k][v];
        sin_cos_turns(fma(pos, turn.y, fma(pos, turn.x, -rint(pos * turn.x))), &sn, &cs);
        const T nf = x_lo[k].v[v] * r, ns = x_hi[k].v[v] * r;
        if (!GRAD) {
          const T f = nf * g_lo[k].v[v], s = ns * g_hi[k].v[v];
          w_lo[k].v[v] = used ? fma_(f, cs, -(s * sn)) : x_lo[k].v[v];
          w_hi[k].v[v] = used ? fma_(s, cs, f * sn) : x_hi[k].v[v];
        } else if (used) {
          const T f = w_lo[k].v[v], s = w_hi[k].v[v];
          const T uf = fma_(f, cs, s * sn), us = fma_(s, cs, -(f * sn));
          d_lo[k].v[v] = fma_(uf, nf, d_lo[k].v[v]);
          d_hi[k].v[v] = fma_(us, ns, d_hi[k].v[v]);
          w_lo[k].v[v] = uf * g_lo[k].v[v];
          w_hi[k].v[v] = us * g_hi[k].v[v];
          mean = fma_(w_lo[k].v[v], nf, fma_(w_hi[k].v[v], ns, mean));
        }
      }
    }
    if (GRAD) {
      mean = group_sum<LG>(mean) / T(a.head);
      if (normed)
#pragma unroll
        for (int k = 0; k < UPL; k++)
#pragma unroll
          for (int v = 0; v < V; v++) {
            w_lo[k].v[v] = r * fma_(-(x_lo[k].v[v] * r), mean, w_lo[k].v[v]);
            w_hi[k].v[v] = r * fma_(-(x_hi[k].v[v] * r), mean, w_hi[k].v[v]);
          }
    }
    T* out = (T*)(GRAD ? a.dx : a.y);
    if (out && valid)
#pragma unroll
      for (int k = 0; k < UPL; k++) {
        if (!has[k]) continue;
        store<T, V>(out + at + lo[k], w_lo[k]);
        store<T, V>(out + at + hi[k], w_hi[k]);
      }
  }
  if constexpr (GRAD) {
    if (!a.dgain_rows) return;
    // One partial row a block: the groups of a section summed in order.
    __shared__ T part[GROUPS][2 * LG * UPL * V];
    __shared__ uint32_t of[GROUPS];
    const uint32_t mine = threadIdx.x / LG;
    if (lane == 0) of[mine] = on && used ? section : a.sections;
#pragma unroll
    for (int k = 0; k < UPL; k++)
      if (has[k])
#pragma unroll
        for (int v = 0; v < V; v++) {
          part[mine][lo[k] + v] = d_lo[k].v[v];
          part[mine][hi[k] + v] = d_hi[k].v[v];
        }
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < a.sections * a.head; i += TPB) {
      const uint32_t s = i / a.head, k = i % a.head;
      T sum = T(0);
#pragma unroll 8
      for (int g = 0; g < GROUPS; g++) sum += of[g] == s ? part[g][k] : T(0);
      ((T*)a.dgain_rows)[(uint64_t)blockIdx.x * a.sections * a.head + i] = sum;
    }
  }
}

// Lanes per head and units per lane for `units` units: f(LG, UPL).
template <class F>
void rotary_shape(uint32_t units, F f) {
  using std::integral_constant;
  if (units <= 4) f(integral_constant<int, 4>(), integral_constant<int, 1>());
  else if (units <= 8) f(integral_constant<int, 8>(), integral_constant<int, 1>());
  else if (units <= 16) f(integral_constant<int, 16>(), integral_constant<int, 1>());
  else if (units <= 32) f(integral_constant<int, 32>(), integral_constant<int, 1>());
  else if (units <= 64) f(integral_constant<int, 64>(), integral_constant<int, 1>());
  else f(integral_constant<int, 64>(), integral_constant<int, 2>());
}

// Pairs a unit holds: 16 bytes where both parts of a head divide into them.
uint32_t rotary_unit(int dtype, const RotaryArgs& a) {
  const uint32_t v = dtype == RG_F32 ? 4 : 2;
  return a.turn % (2 * v) == 0 && a.head % (2 * v) == 0 ? v : 1;
}

// Blocks: as many as there are heads of tokens for, up to eight a CU; backward two, each of which
// leaves a partial row for the fold to sum (4 x 1024 x 24 heads of 64: 512 rows fold in 5 us, 1024 in 9).
constexpr uint32_t ROTARY_BLOCKS = 2048, ROTARY_GRAD_BLOCKS = 512;

uint32_t rotary_blocks(int dtype, const RotaryArgs& a, bool grad) {
  uint32_t blocks = 0;
  rotary_shape(a.head / 2 / rotary_unit(dtype, a), [&](auto lg, auto) {
    const uint64_t per = TPB / decltype(lg)::value, items = (uint64_t)a.batch * a.length * a.heads;
    blocks = (uint32_t)std::max<uint64_t>(std::min<uint64_t>((items + per - 1) / per, grad ? ROTARY_GRAD_BLOCKS : ROTARY_BLOCKS), (a.heads + per - 1) / per);
  });
  return blocks;
}

template <class T, int V, bool GRAD>
void launch_rotary(hipStream_t s, int dtype, const RotaryArgs& a) {
  const uint32_t blocks = rotary_blocks(dtype, a, GRAD);
  rotary_shape(a.head / 2 / V, [&](auto lg, auto upl) {
    hipLaunchKernelGGL((k_rotary<T, V, decltype(lg)::value, decltype(upl)::value, GRAD>), dim3(blocks), dim3(TPB), 0, s, a);
  });
}

template <bool GRAD>
void rotary(hipStream_t s, int dtype, const RotaryArgs& a) {
  const uint32_t v = rotary_unit(dtype, a);
  if (dtype == RG_F32) {
    if (v == 4) launch_rotary<float, 4, GRAD>(s, dtype, a);
    else launch_rotary<float, 1, GRAD>(s, dtype, a);
  } else {
    if (v == 2) launch_rotary<double, 2, GRAD>(s, dtype, a);
    else launch_rotary<double, 1, GRAD>(s, dtype, a);
  }
}

}  // namespace

uint32_t rotary_grad_rows(int dtype, const RotaryArgs& a) { return rotary_blocks(dtype, a, true); }
void rotary_norm(hipStream_t s, int dtype, const RotaryArgs& a) { rotary<false>(s, dtype, a); }
void rotary_norm_grad(hipStream_t s, int dtype, const RotaryArgs& a) { rotary<true>(s, dtype, a); }

}  // namespace rgk
