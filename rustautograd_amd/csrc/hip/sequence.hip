// The sequence operators (include/rg_plan.h, CAUSAL_CONV ... ROTARY_NORM_GRAD).
#include "sequence.h"

#include <algorithm>

namespace rgk {

namespace {

constexpr int TPB = 256;

__device__ __forceinline__ float fma_(float a, float b, float c) { return __builtin_fmaf(a, b, c); }
__device__ __forceinline__ double fma_(double a, double b, double c) { return __builtin_fma(a, b, c); }
__device__ __forceinline__ float exp_(float v) { return expf(v); }
__device__ __forceinline__ double exp_(double v) { return exp(v); }
__device__ __forceinline__ float log1p_(float v) { return log1pf(v); }
__device__ __forceinline__ double log1p_(double v) { return log1p(v); }
__device__ __forceinline__ float sqrt_(float v) { return sqrtf(v); }
__device__ __forceinline__ double sqrt_(double v) { return sqrt(v); }
template <class T>
__device__ __forceinline__ T sigmoid(T v) { return T(1) / (T(1) + exp_(-v)); }
template <class T>
__device__ __forceinline__ T silu(T v) { return v / (T(1) + exp_(-v)); }
// silu'(v) from s = sigmoid(v).
template <class T>
__device__ __forceinline__ T silu_slope(T v, T s) { return s * fma_(v, T(1) - s, T(1)); }
// log(1 + e^v) without overflow; log1p keeps the relative precision of small steps.
template <class T>
__device__ __forceinline__ T softplus(T v) { return (v > T(0) ? v : T(0)) + log1p_(exp_(v > T(0) ? -v : v)); }

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
// in registers, so that x is read once but for the K - 1 positions before a run.
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
// positions after it again rather than exchange them.
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
      if (t0 + i < n) g[i] = load<T, V>(dy + (uint64_t)(t0 + i) * a.width);
    }
#pragma unroll
    for (int i = 0; i < R + K - 1; i++)
#pragma unroll
      for (int v = 0; v < V; v++) {
        if (a.silu && t0 + i < n) {
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
        if (i >= k)
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

constexpr int CONV_RUN = 8;

template <class T, int V, class F>
void conv_taps(const ConvArgs& a, F launch) {
  switch (a.taps) {
    case 2: launch(std::integral_constant<int, 2>()); break;
    case 3: launch(std::integral_constant<int, 3>()); break;
    case 4: launch(std::integral_constant<int, 4>()); break;
    case 5: launch(std::integral_constant<int, 5>()); break;
    case 6: launch(std::integral_constant<int, 6>()); break;
    case 7: launch(std::integral_constant<int, 7>()); break;
    case 8: launch(std::integral_constant<int, 8>()); break;
    default: break;
  }
}

template <class T, int V>
void launch_conv(hipStream_t s, const ConvArgs& a, bool grad) {
  const uint32_t nx = (a.width + 64 * V - 1) / (64 * V), runs = (a.length + 4 * CONV_RUN - 1) / (4 * CONV_RUN);
  conv_taps<T, V>(a, [&](auto k) {
    if (grad) hipLaunchKernelGGL((k_conv_grad<T, decltype(k)::value, V, CONV_RUN>), dim3(nx * runs * a.batch), dim3(TPB), 0, s, a, nx, runs);
    else hipLaunchKernelGGL((k_conv<T, decltype(k)::value, V, CONV_RUN>), dim3(nx * runs * a.batch), dim3(TPB), 0, s, a, nx, runs);
  });
}

}  // namespace

uint32_t conv_grad_rows(int, const ConvArgs& a) { return a.batch * ((a.length + 4 * CONV_RUN - 1) / (4 * CONV_RUN)); }

static void conv(hipStream_t s, int dtype, const ConvArgs& a, bool grad) {
  if (dtype == RG_F32) {
    if (a.width % 4 == 0) launch_conv<float, 4>(s, a, grad);
    else launch_conv<float, 1>(s, a, grad);
  } else {
    if (a.width % 2 == 0) launch_conv<double, 2>(s, a, grad);
    else launch_conv<double, 1>(s, a, grad);
  }
}
void causal_conv(hipStream_t s, int dtype, const ConvArgs& a) { conv(s, dtype, a, false); }
void causal_conv_grad(hipStream_t s, int dtype, const ConvArgs& a) { conv(s, dtype, a, true); }

// ---- selective scan ---------------------------------------------------------------------------

namespace {

constexpr int TILE = RG_SCAN_MARK;

// NL neighbouring lanes share a channel, NS of its states each; a block holds CH channels, of one
// group. Tiles of TILE positions pass through LDS, channels' values transposed so that a lane
// reads four positions at once.
template <class T, int NL_, int NS_>
struct ScanShape {
  static constexpr int NL = NL_, NS = NS_, NP = NL * NS, CH = TPB / NL, EPT = CH / 16, LD = TILE + 16 / sizeof(T);
};

struct ScanPlace {
  uint32_t b, group, ch0, chs;  // sequence, group, first channel of the tile and how many
  uint32_t tile;                // tile of the group's channels
};
template <class S>
__device__ __forceinline__ ScanPlace scan_place(const ScanArgs& a, uint32_t tiles) {
  ScanPlace p;
  const uint32_t per = a.width / a.groups;
  p.tile = blockIdx.x % tiles;
  p.group = blockIdx.x / tiles % a.groups;
  p.b = blockIdx.x / tiles / a.groups;
  p.ch0 = p.group * per + p.tile * S::CH;
  p.chs = min((uint32_t)S::CH, per - p.tile * S::CH);
  return p;
}

// EPT neighbouring channels of one position of a [batch, length, width] value; zeros outside.
template <class S, class T>
__device__ __forceinline__ Vec<T, S::EPT> scan_load(const T* p, bool inside, uint32_t left, bool vec) {
  Vec<T, S::EPT> v{};
  if (!inside) return v;
  if (vec && left >= (uint32_t)S::EPT) return load<T, S::EPT>(p);
#pragma unroll
  for (int j = 0; j < S::EPT; j++)
    if ((uint32_t)j < left) v.v[j] = p[j];
  return v;
}
template <class S, class T>
__device__ __forceinline__ void scan_store(T* p, const Vec<T, S::EPT>& v, bool inside, uint32_t left, bool vec) {
  if (!inside) return;
  if (vec && left >= (uint32_t)S::EPT) {
    store<T, S::EPT>(p, v);
    return;
  }
#pragma unroll
  for (int j = 0; j < S::EPT; j++)
    if ((uint32_t)j < left) p[j] = v.v[j];
}

// The decay e^(dt a) of one position. In 32 bits `a` comes multiplied by log2 e, for the
// hardware's power of two.
__device__ __forceinline__ float decay(float dt, float a) { return __builtin_amdgcn_exp2f(dt * a); }
__device__ __forceinline__ double decay(double dt, double a) { return exp(dt * a); }
__device__ __forceinline__ float decay_rate(float a) { return a * 1.44269504088896341f; }
__device__ __forceinline__ double decay_rate(double a) { return a; }
// An infinite rate becomes the largest finite one: the decay of a step is the same 0 (or infinity),
// and positions outside the sequence, whose steps are 0, leave the state as it is.
template <class T>
__device__ __forceinline__ T finite_rate(T a, T most) { return a > most ? most : a < -most ? -most : a; }

// The sum over the NL lanes of a channel, in all of them.
template <int NL, class T>
__device__ __forceinline__ T channel_sum(T v) {
#pragma unroll
  for (int m = 1; m < NL; m <<= 1) v += __shfl_xor(v, m);
  return v;
}

template <class S, class T>
__device__ __forceinline__ void scan_maps(const ScanArgs& a, const ScanPlace& p, uint32_t t0, uint32_t n, const T* src, T (*dst)[S::NP]) {
  for (uint32_t i = threadIdx.x; i < TILE * S::NP; i += TPB) {
    const uint32_t row = i / S::NP, k = i % S::NP;
    T v = T(0);
    if (t0 + row < n && k < a.states) v = src[(((uint64_t)p.b * a.length + t0 + row) * a.groups + p.group) * a.states + k];
    dst[row][k] = v;
  }
}

// Forward: h[t] = e^(dt a) h[t - 1] + dt x b, y = c . h + d x, gated.
template <class T, int NL, int NS>
__global__ void __launch_bounds__(TPB) k_scan(ScanArgs a, uint32_t tiles, bool vec) {
  using S = ScanShape<T, NL, NS>;
  __shared__ __align__(16) T sx[S::CH][S::LD], sdt[S::CH][S::LD], sb[TILE][S::NP], sc[TILE][S::NP];
  const ScanPlace p = scan_place<S>(a, tiles);
  const uint32_t n = end_of(a.lengths, p.b, a.length);
  const uint32_t c = threadIdx.x / NL, q = threadIdx.x % NL, d = p.ch0 + c;
  const bool on = c < p.chs;
  T rate[NS], h[NS];
#pragma unroll
  for (int j = 0; j < NS; j++) {
    const uint32_t k = q * NS + j;
    const bool has = on && k < a.states;
    rate[j] = has ? decay_rate(finite_rate(((const T*)a.a)[(uint64_t)d * a.states + k], sizeof(T) == 4 ? T(2e38f) : T(1e308))) : T(0);
    h[j] = has && a.state ? ((const T*)a.state)[((uint64_t)p.b * a.width + d) * a.states + k] : T(0);
  }
  const T skip = on && q == 0 && a.skip ? ((const T*)a.skip)[d] : T(0);
  const uint32_t row = threadIdx.x / 16, col = threadIdx.x % 16 * S::EPT;
  const uint32_t left = col < p.chs ? p.chs - col : 0;
  const uint32_t marks = (a.length + TILE - 1) / TILE;
  for (uint32_t m = 0; m < marks; m++) {
    const uint32_t t0 = m * TILE, t = t0 + row;
    const uint64_t at = ((uint64_t)p.b * a.length + t) * a.width + p.ch0 + col;
    const bool inside = t < n && left > 0;
    const auto x = scan_load<S>((const T*)a.x + at, inside, left, vec);
    auto dt = scan_load<S>((const T*)a.dt + at, inside, left, vec);
    Vec<T, S::EPT> z{};
    if (a.gate) z = scan_load<S>((const T*)a.gate + at, inside, left, vec);
#pragma unroll
    for (int j = 0; j < S::EPT; j++) {
      if (a.softplus && inside) dt.v[j] = softplus(dt.v[j]);
      sx[col + j][row] = x.v[j];
      sdt[col + j][row] = dt.v[j];
    }
    scan_maps<S>(a, p, t0, n, (const T*)a.b, sb);
    scan_maps<S>(a, p, t0, n, (const T*)a.c, sc);
    __syncthreads();
    if (a.marks && on)
#pragma unroll
      for (int j = 0; j < NS; j++)
        if (q * NS + j < a.states) ((T*)a.marks)[(((uint64_t)p.b * marks + m) * a.width + d) * a.states + q * NS + j] = h[j];
    T mine = T(0);
#pragma unroll 4
    for (int i = 0; i < TILE; i++) {
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
    __syncthreads();
    if (a.y) {
      Vec<T, S::EPT> y;
#pragma unroll
      for (int j = 0; j < S::EPT; j++) y.v[j] = !inside ? T(0) : a.gate ? sx[col + j][row] * silu(z.v[j]) : sx[col + j][row];
      scan_store<S>((T*)a.y + at, y, t < a.length, left, vec);
    }
    __syncthreads();
  }
  if (a.last && on)
#pragma unroll
    for (int j = 0; j < NS; j++)
      if (q * NS + j < a.states) ((T*)a.last)[((uint64_t)p.b * a.width + d) * a.states + q * NS + j] = h[j];
}

// Backward, tile by tile from the last. From the state kept before the tile, its decays e and the
// decayed states p = e h[t - 1] are formed again, then with G = dL/dh[t] carried back:
//   dx = dt sum G b + d gy, ddt = x sum G b + sum G p a, da += dt G p, db = G dt x, dc = gy h.
// The sums over channels that db and dc take leave one partial row per tile of channels.
template <class T, int NL, int NS>
__global__ void __launch_bounds__(TPB) k_scan_grad(ScanArgs a, uint32_t tiles, bool vec) {
  using S = ScanShape<T, NL, NS>;
  constexpr int WAVES = TPB / 64;
  __shared__ __align__(16) T sx[S::CH][S::LD], sdt[S::CH][S::LD], sg[S::CH][S::LD], sy[S::CH][S::LD], sb[TILE][S::NP], sc[TILE][S::NP];
  __shared__ T red[WAVES][TILE][2][S::NP];
  const ScanPlace p = scan_place<S>(a, tiles);
  const uint32_t n = end_of(a.lengths, p.b, a.length);
  const uint32_t c = threadIdx.x / NL, q = threadIdx.x % NL, d = p.ch0 + c, wave = threadIdx.x / 64;
  const bool on = c < p.chs;
  T rate[NS], rate_e[NS], back[NS], da[NS], dd = T(0);
#pragma unroll
  for (int j = 0; j < NS; j++) {
    const uint32_t k = q * NS + j;
    const bool has = on && k < a.states;
    rate[j] = has ? finite_rate(((const T*)a.a)[(uint64_t)d * a.states + k], sizeof(T) == 4 ? T(2e38f) : T(1e308)) : T(0);
    rate_e[j] = decay_rate(rate[j]);
    back[j] = has && a.carry ? ((const T*)a.carry)[((uint64_t)p.b * a.width + d) * a.states + k] : T(0);
    da[j] = T(0);
  }
  const T skip = on && a.skip ? ((const T*)a.skip)[d] : T(0);
  const uint32_t row = threadIdx.x / 16, col = threadIdx.x % 16 * S::EPT;
  const uint32_t left = col < p.chs ? p.chs - col : 0;
  const uint32_t marks = (a.length + TILE - 1) / TILE;
  for (uint32_t m = marks; m-- > 0;) {
    const uint32_t t0 = m * TILE, t = t0 + row;
    const uint64_t at = ((uint64_t)p.b * a.length + t) * a.width + p.ch0 + col;
    const bool inside = t < n && left > 0;
    const auto x = scan_load<S>((const T*)a.x + at, inside, left, vec);
    const auto raw = scan_load<S>((const T*)a.dt + at, inside, left, vec);
    const auto g = scan_load<S>((const T*)a.dy + at, inside, left, vec);
    Vec<T, S::EPT> z{};
    if (a.gate) z = scan_load<S>((const T*)a.gate + at, inside, left, vec);
    T h[NS];
#pragma unroll
    for (int j = 0; j < NS; j++)
      h[j] = on && q * NS + j < a.states ? ((const T*)a.marks)[(((uint64_t)p.b * marks + m) * a.width + d) * a.states + q * NS + j] : T(0);
#pragma unroll
    for (int j = 0; j < S::EPT; j++) {
      sx[col + j][row] = x.v[j];
      sdt[col + j][row] = a.softplus && inside ? softplus(raw.v[j]) : raw.v[j];
      sg[col + j][row] = a.gate ? g.v[j] * silu(z.v[j]) : g.v[j];
    }
    scan_maps<S>(a, p, t0, n, (const T*)a.b, sb);
    scan_maps<S>(a, p, t0, n, (const T*)a.c, sc);
    __syncthreads();
    T e[TILE][NS], kept[TILE][NS], mine = T(0), mine2 = T(0);
#pragma unroll
    for (int i = 0; i < TILE; i++) {
      const T step = sdt[c][i], u = sx[c][i], drive = step * u;
      T y = q == 0 ? skip * u : T(0);
#pragma unroll
      for (int j = 0; j < NS; j++) {
        e[i][j] = decay(step, rate_e[j]);
        kept[i][j] = e[i][j] * h[j];
        h[j] = fma_(drive, sb[i][q * NS + j], kept[i][j]);
        y = fma_(sc[i][q * NS + j], h[j], y);
      }
      if (a.gate) {
        y = channel_sum<NL>(y);
        if (i % NL == (int)q) mine = y;
        if (i % NL == NL - 1) sy[c][i - (NL - 1) + q] = mine;
      }
    }
#pragma unroll
    for (int i = TILE - 1; i >= 0; i--) {
      const T step = sdt[c][i], u = sx[c][i], gy = sg[c][i], drive = step * u;
      T sum_b = T(0), sum_a = T(0);
#pragma unroll
      for (int j = 0; j < NS; j++) {
        const T bj = sb[i][q * NS + j], G = fma_(gy, sc[i][q * NS + j], back[j]);
        T dc = gy * fma_(drive, bj, kept[i][j]), db = G * drive;
        const T gp = G * kept[i][j];
        sum_b = fma_(G, bj, sum_b);
        sum_a = fma_(gp, rate[j], sum_a);
        da[j] = fma_(gp, step, da[j]);
        back[j] = e[i][j] * G;
#pragma unroll
        for (int l = NL; l < 64; l <<= 1) {
          db += __shfl_xor(db, l);
          dc += __shfl_xor(dc, l);
        }
        if (threadIdx.x % 64 < NL) {
          red[wave][i][0][q * NS + j] = db;
          red[wave][i][1][q * NS + j] = dc;
        }
      }
      dd = fma_(gy, u, dd);
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
#pragma unroll
    for (int j = 0; j < S::EPT; j++) {
      dx.v[j] = inside ? sx[col + j][row] : T(0);
      ddt.v[j] = !inside ? T(0) : a.softplus ? sdt[col + j][row] * sigmoid(raw.v[j]) : sdt[col + j][row];
      dz.v[j] = inside && a.gate ? g.v[j] * sy[col + j][row] * silu_slope(z.v[j], sigmoid(z.v[j])) : T(0);
    }
    const bool within = t < a.length;
    if (a.dx) scan_store<S>((T*)a.dx + at, dx, within, left, vec);
    if (a.ddt) scan_store<S>((T*)a.ddt + at, ddt, within, left, vec);
    if (a.dz) scan_store<S>((T*)a.dz + at, dz, within, left, vec);
    for (uint32_t i = threadIdx.x; i < TILE * 2 * S::NP; i += TPB) {
      const uint32_t r = i / (2 * S::NP), w = i / S::NP % 2, k = i % S::NP;
      T* to = (T*)(w ? a.dc_rows : a.db_rows);
      if (!to || k >= a.states || t0 + r >= a.length) continue;
      T sum = T(0);
      if (t0 + r < n)
#pragma unroll
        for (int v = 0; v < WAVES; v++) sum += red[v][r][w][k];
      const uint64_t rows = (uint64_t)a.batch * a.length * a.groups * a.states;
      to[p.tile * rows + (((uint64_t)p.b * a.length + t0 + r) * a.groups + p.group) * a.states + k] = sum;
    }
    __syncthreads();
  }
  if (!on) return;
#pragma unroll
  for (int j = 0; j < NS; j++) {
    if (q * NS + j >= a.states) continue;
    const uint64_t at = ((uint64_t)p.b * a.width + d) * a.states + q * NS + j;
    if (a.da_rows) ((T*)a.da_rows)[at] = da[j];
    if (a.dstate) ((T*)a.dstate)[at] = back[j];
  }
  if (a.dd_rows && q == 0) ((T*)a.dd_rows)[(uint64_t)p.b * a.width + d] = dd;
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

template <class T>
uint32_t scan_tiles(const ScanArgs& a) {
  uint32_t tiles = 0;
  scan_shape<T>(a.states, [&](auto nl, auto) {
    const uint32_t ch = TPB / decltype(nl)::value;
    tiles = (a.width / a.groups + ch - 1) / ch;
  });
  return tiles;
}

template <class T>
void launch_scan(hipStream_t s, const ScanArgs& a, bool grad) {
  const uint32_t tiles = scan_tiles<T>(a);
  scan_shape<T>(a.states, [&](auto nl, auto ns) {
    constexpr int NL = decltype(nl)::value, NS = decltype(ns)::value, EPT = ScanShape<T, NL, NS>::EPT;
    const bool vec = a.width % EPT == 0 && (a.width / a.groups) % EPT == 0;
    const dim3 grid(a.batch * a.groups * tiles);
    if (grad) hipLaunchKernelGGL((k_scan_grad<T, NL, NS>), grid, dim3(TPB), 0, s, a, tiles, vec);
    else hipLaunchKernelGGL((k_scan<T, NL, NS>), grid, dim3(TPB), 0, s, a, tiles, vec);
  });
}

}  // namespace

uint32_t scan_rows(int, const ScanArgs& a) { return a.batch; }
uint32_t scan_group_tiles(int dtype, const ScanArgs& a) { return dtype == RG_F32 ? scan_tiles<float>(a) : scan_tiles<double>(a); }

void selective_scan(hipStream_t s, int dtype, const ScanArgs& a) {
  if (dtype == RG_F32) launch_scan<float>(s, a, false);
  else launch_scan<double>(s, a, false);
}
void selective_scan_grad(hipStream_t s, int dtype, const ScanArgs& a) {
  if (dtype == RG_F32) launch_scan<float>(s, a, true);
  else launch_scan<double>(s, a, true);
}

// ---- norm with rotation -----------------------------------------------------------------------

namespace {

__device__ __forceinline__ void sin_cos_turns(double f, float* sn, float* cs) { sincospif(2.0f * (float)f, sn, cs); }
__device__ __forceinline__ void sin_cos_turns(double f, double* sn, double* cs) { sincospi(2.0 * f, sn, cs); }

// LG lanes share a head, each with UPL units of V pairs: both halves of a pair lie in one lane, so
// the turn needs no exchange. A group of lanes keeps one head and walks the tokens.
template <class T, int V, int LG, int UPL, bool GRAD>
__global__ void __launch_bounds__(TPB) k_rotary(RotaryArgs a) {
  constexpr int GROUPS = TPB / LG;
  const uint32_t group = blockIdx.x * GROUPS + threadIdx.x / LG, lane = threadIdx.x % LG;
  const uint32_t all = gridDim.x * GROUPS, walkers = all / a.heads;
  const uint32_t head = group % a.heads, first = group / a.heads;
  const uint32_t half = a.turn / 2, rest = (a.head - a.turn) / 2, tokens = a.batch * a.length;
  uint32_t section = 0;
  while (section < a.sections && head >= a.last[section]) section++;
  const bool on = first < walkers;
  const bool used = section < a.sections;
  // Where this lane's units lie in a head: their first and second halves.
  uint32_t lo[UPL], hi[UPL];
  bool has[UPL];
  Vec<T, V> g_lo[UPL], g_hi[UPL], d_lo[UPL], d_hi[UPL];
#pragma unroll
  for (int k = 0; k < UPL; k++) {
    const uint32_t u = (lane + k * LG) * V;
    has[k] = u < a.head / 2;
    lo[k] = u < half ? u : a.turn + (u - half);
    hi[k] = lo[k] + (u < half ? half : rest);
    d_lo[k] = d_hi[k] = Vec<T, V>{};
#pragma unroll
    for (int v = 0; v < V; v++) g_lo[k].v[v] = g_hi[k].v[v] = T(1);
    if (has[k] && used && a.normed) {
      g_lo[k] = load<T, V>((const T*)a.gain + section * a.head + lo[k]);
      g_hi[k] = load<T, V>((const T*)a.gain + section * a.head + hi[k]);
    }
  }
  for (uint32_t token = on ? first : tokens; token < tokens; token += walkers) {
    const uint64_t at = ((uint64_t)token * a.heads + head) * a.head;
    const double pos = (double)a.positions[a.shared_positions ? token % a.length : token];
    Vec<T, V> x_lo[UPL], x_hi[UPL], w_lo[UPL], w_hi[UPL];
    T ss = T(0);
#pragma unroll
    for (int k = 0; k < UPL; k++) {
      x_lo[k] = x_hi[k] = w_lo[k] = w_hi[k] = Vec<T, V>{};
      if (!has[k]) continue;
      x_lo[k] = load<T, V>((const T*)a.x + at + lo[k]);
      x_hi[k] = load<T, V>((const T*)a.x + at + hi[k]);
      if (GRAD) {
        w_lo[k] = load<T, V>((const T*)a.dy + at + lo[k]);
        w_hi[k] = load<T, V>((const T*)a.dy + at + hi[k]);
      }
#pragma unroll
      for (int v = 0; v < V; v++) ss = fma_(x_lo[k].v[v], x_lo[k].v[v], fma_(x_hi[k].v[v], x_hi[k].v[v], ss));
    }
    T r = T(1);
    if (a.normed && used) {
#pragma unroll
      for (int m = 1; m < LG; m <<= 1) ss += __shfl_xor(ss, m);
      r = T(1) / sqrt_(ss / T(a.head) + T(a.eps));
    }
    T mean = T(0);
#pragma unroll
    for (int k = 0; k < UPL; k++) {
      if (!has[k] || !used) continue;
#pragma unroll
      for (int v = 0; v < V; v++) {
        T sn = T(0), cs = T(1);
        if (lo[k] + v < half) {
          const double2 turn = a.turns[lo[k] + v];
          const double whole = rint(pos * turn.x);
          sin_cos_turns(fma(pos, turn.y, fma(pos, turn.x, -whole)), &sn, &cs);
        }
        if (!GRAD) {
          const T f = x_lo[k].v[v] * r * g_lo[k].v[v], s = x_hi[k].v[v] * r * g_hi[k].v[v];
          w_lo[k].v[v] = fma_(f, cs, -(s * sn));
          w_hi[k].v[v] = fma_(s, cs, f * sn);
        } else {
          const T f = w_lo[k].v[v], s = w_hi[k].v[v];
          const T uf = fma_(f, cs, s * sn), us = fma_(s, cs, -(f * sn));
          const T nf = x_lo[k].v[v] * r, ns = x_hi[k].v[v] * r;
          d_lo[k].v[v] = fma_(uf, nf, d_lo[k].v[v]);
          d_hi[k].v[v] = fma_(us, ns, d_hi[k].v[v]);
          w_lo[k].v[v] = uf * g_lo[k].v[v];
          w_hi[k].v[v] = us * g_hi[k].v[v];
          mean = fma_(w_lo[k].v[v], nf, fma_(w_hi[k].v[v], ns, mean));
        }
      }
    }
    if (GRAD && a.normed && used) {
#pragma unroll
      for (int m = 1; m < LG; m <<= 1) mean += __shfl_xor(mean, m);
      mean /= T(a.head);
#pragma unroll
      for (int k = 0; k < UPL; k++)
#pragma unroll
        for (int v = 0; v < V; v++) {
          w_lo[k].v[v] = r * fma_(-(x_lo[k].v[v] * r), mean, w_lo[k].v[v]);
          w_hi[k].v[v] = r * fma_(-(x_hi[k].v[v] * r), mean, w_hi[k].v[v]);
        }
    }
    T* out = (T*)(GRAD ? a.dx : a.y);
    if (out)
#pragma unroll
      for (int k = 0; k < UPL; k++) {
        if (!has[k]) continue;
        const bool pass = !GRAD && !used;
        store<T, V>(out + at + lo[k], pass ? x_lo[k] : w_lo[k]);
        store<T, V>(out + at + hi[k], pass ? x_hi[k] : w_hi[k]);
      }
  }
  if (!GRAD || !a.dgain_rows) return;
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
    for (int g = 0; g < GROUPS; g++)
      if (of[g] == s) sum += part[g][k];
    ((T*)a.dgain_rows)[(uint64_t)blockIdx.x * a.sections * a.head + i] = sum;
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

uint32_t rotary_blocks(int dtype, const RotaryArgs& a) {
  uint32_t blocks = 0;
  rotary_shape(a.head / 2 / rotary_unit(dtype, a), [&](auto lg, auto) {
    const uint64_t per = TPB / decltype(lg)::value, items = (uint64_t)a.batch * a.length * a.heads;
    blocks = (uint32_t)std::max<uint64_t>(std::min<uint64_t>((items + per - 1) / per, 1024), (a.heads + per - 1) / per);
  });
  return blocks;
}

template <class T, int V, bool GRAD>
void launch_rotary(hipStream_t s, int dtype, const RotaryArgs& a) {
  const uint32_t blocks = rotary_blocks(dtype, a);
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

uint32_t rotary_grad_rows(int dtype, const RotaryArgs& a) { return rotary_blocks(dtype, a); }
void rotary_norm(hipStream_t s, int dtype, const RotaryArgs& a) { rotary<false>(s, dtype, a); }
void rotary_norm_grad(hipStream_t s, int dtype, const RotaryArgs& a) { rotary<true>(s, dtype, a); }

}  // namespace rgk
