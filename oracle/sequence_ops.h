// The sequence operators of include/rg_plan.h on the CPU: every value computed in 64 bits from the
// formulas, one position after another, and rounded once to the operator's dtype when stored. The
// angles of a rotation, whose error grows with the position, are formed in extended precision.
#pragma once
#include <algorithm>
#include <cmath>
#include <cstdint>
#include <limits>
#include <vector>

#include "../include/rg_plan.h"

namespace rgseq {

inline double sigmoid(double v) { return 1.0 / (1.0 + std::exp(-v)); }
inline double softplus(double v) { return std::fmax(v, 0.0) + std::log1p(std::exp(-std::fabs(v))); }

// The operands and results of a step as typed pointers; absent ones are null.
template <class T>
struct Operands {
  const rgplan::Instr& in;
  rgplan::Sequence q;
  std::vector<void*> slot;  // of each argument
  std::vector<T*> out;      // of each result
  const T* arg(int k) const { return k < 0 ? nullptr : (const T*)slot[(size_t)k]; }
  int64_t end(int64_t b) const {
    if (q.lengths < 0) return q.length;
    const int64_t n = ((const int32_t*)slot[(size_t)q.lengths])[b];
    return n < 0 ? 0 : n > q.length ? q.length : n;
  }
  bool has(int64_t flag) const { return (in.sequence.flags & flag) != 0; }
};

template <class T>
void causal_conv(const Operands<T>& o) {
  const auto& q = o.q;
  const T *x = o.arg(q.x), *w = o.arg(q.w), *bias = o.arg(q.bias), *state = o.arg(q.state), *dy = o.arg(q.dy), *carry = o.arg(q.carry);
  const int64_t K = q.taps, D = q.width, T_ = q.length;
  const bool grad = dy != nullptr, silu = o.has(RG_CONV_SILU);
  std::vector<double> dw((size_t)(K * D), 0.0), db((size_t)D, 0.0);
  for (int64_t b = 0; b < q.batch; b++) {
    const int64_t n = o.end(b);
    for (int64_t d = 0; d < D; d++) {
      auto past = [&](int64_t i) -> double {
        if (i >= K - 1) return (double)x[(b * T_ + i - K + 1) * D + d];
        return state ? (double)state[(b * (K - 1) + i) * D + d] : 0.0;
      };
      std::vector<double> dpast(grad ? (size_t)(n + K - 1) : 0, 0.0);
      for (int64_t t = 0; t < n; t++) {
        double pre = bias ? (double)bias[d] : 0.0;
        for (int64_t k = 0; k < K; k++) pre += (double)w[k * D + d] * past(t + k);
        const double s = sigmoid(pre);
        if (!grad) {
          if (o.out[0]) o.out[0][(b * T_ + t) * D + d] = (T)(silu ? pre * s : pre);
          continue;
        }
        const double g = (double)dy[(b * T_ + t) * D + d] * (silu ? s * (1.0 + pre * (1.0 - s)) : 1.0);
        db[(size_t)d] += g;
        for (int64_t k = 0; k < K; k++) {
          dw[(size_t)(k * D + d)] += g * past(t + k);
          dpast[(size_t)(t + k)] += g * (double)w[k * D + d];
        }
      }
      if (!grad) {
        if (o.out[0])
          for (int64_t t = n; t < T_; t++) o.out[0][(b * T_ + t) * D + d] = (T)0;
        if (o.out[1])
          for (int64_t j = 0; j < K - 1; j++) o.out[1][(b * (K - 1) + j) * D + d] = (T)past(n + j);
        continue;
      }
      if (carry)
        for (int64_t j = 0; j < K - 1; j++) dpast[(size_t)(n + j)] += (double)carry[(b * (K - 1) + j) * D + d];
      if (o.out[0])
        for (int64_t t = 0; t < T_; t++) o.out[0][(b * T_ + t) * D + d] = (T)(t < n ? dpast[(size_t)(t + K - 1)] : 0.0);
      if (o.out[3])
        for (int64_t j = 0; j < K - 1; j++) o.out[3][(b * (K - 1) + j) * D + d] = (T)dpast[(size_t)j];
    }
  }
  if (grad && o.out[1])
    for (size_t k = 0; k < dw.size(); k++) o.out[1][k] = (T)dw[k];
  if (grad && o.out[2])
    for (size_t k = 0; k < db.size(); k++) o.out[2][k] = (T)db[k];
}

template <class T>
void selective_scan(const Operands<T>& o) {
  const auto& q = o.q;
  const T *x = o.arg(q.x), *raw = o.arg(q.dt), *a = o.arg(q.a), *bm = o.arg(q.b), *cm = o.arg(q.c), *skip = o.arg(q.skip), *z = o.arg(q.gate),
          *state = o.arg(q.state), *dy = o.arg(q.dy), *carry = o.arg(q.carry), *bias = o.arg(q.dt_bias);
  const int64_t D = q.width, N = q.states, L = q.length, G = q.groups, per = D / G;
  const bool joined = q.c < 0;  // c's groups follow b's in one operand
  const int64_t GM = joined ? 2 * G : G, cg = joined ? G * N : 0;
  if (joined) cm = bm;
  const bool grad = dy != nullptr, soft = o.has(RG_SCAN_SOFTPLUS), logs = o.has(RG_SCAN_LOG);
  auto rate = [&](int64_t k) { return logs ? -std::exp((double)a[k]) : (double)a[k]; };
  auto given = [&](int64_t at, int64_t d) { return (double)raw[at] + (bias ? (double)bias[d] : 0.0); };
  std::vector<double> da((size_t)(D * N), 0.0), dd((size_t)D, 0.0), dbias((size_t)D, 0.0);
  std::vector<double> db, dc;
  if (grad) {
    db.assign((size_t)(q.batch * L * GM * N), 0.0);
    dc.assign(db.size(), 0.0);
    for (int r : {0, 1, 6})  // positions outside a sequence
      if (o.out[(size_t)r]) std::fill(o.out[(size_t)r], o.out[(size_t)r] + q.batch * L * D, (T)0);
  } else {
    if (o.out[0]) std::fill(o.out[0], o.out[0] + q.batch * L * D, (T)0);
    if (o.out[2]) std::fill(o.out[2], o.out[2] + q.batch * ((L + RG_SCAN_MARK - 1) / RG_SCAN_MARK) * D * N, (T)0);
  }
  for (int64_t b = 0; b < q.batch; b++) {
    const int64_t n = o.end(b);
    for (int64_t d = 0; d < D; d++) {
      const int64_t g = d / per;
      std::vector<double> h((size_t)((n + 1) * N), 0.0);  // h[t + 1] after position t
      if (state)
        for (int64_t s = 0; s < N; s++) h[(size_t)s] = (double)state[(b * D + d) * N + s];
      std::vector<double> y((size_t)n, 0.0);
      for (int64_t t = 0; t < n; t++) {
        const int64_t at = (b * L + t) * D + d, row = ((b * L + t) * GM + g) * N;
        const double given_dt = given(at, d), dt = soft ? softplus(given_dt) : given_dt, u = (double)x[at];
        for (int64_t s = 0; s < N; s++) {
          const double v = std::exp(dt * rate(d * N + s)) * h[(size_t)(t * N + s)] + dt * u * (double)bm[row + s];
          h[(size_t)((t + 1) * N + s)] = v;
          y[(size_t)t] += (double)cm[row + cg + s] * v;
        }
        if (skip) y[(size_t)t] += (double)skip[d] * u;
        if (!grad && o.out[0]) o.out[0][at] = (T)(z ? y[(size_t)t] * (double)z[at] * sigmoid((double)z[at]) : y[(size_t)t]);
      }
      if (!grad) {
        if (o.out[1])
          for (int64_t s = 0; s < N; s++) o.out[1][(b * D + d) * N + s] = (T)h[(size_t)(n * N + s)];
        continue;
      }
      std::vector<double> G_((size_t)N, 0.0);  // the gradient carried back into h[t]
      if (carry)
        for (int64_t s = 0; s < N; s++) G_[(size_t)s] = (double)carry[(b * D + d) * N + s];
      for (int64_t t = n; t-- > 0;) {
        const int64_t at = (b * L + t) * D + d, row = ((b * L + t) * GM + g) * N;
        const double given_dt = given(at, d), dt = soft ? softplus(given_dt) : given_dt, u = (double)x[at];
        double gy = (double)dy[at];
        if (z) {
          const double v = (double)z[at], s = sigmoid(v);
          if (o.out[6]) o.out[6][at] = (T)(gy * y[(size_t)t] * s * (1.0 + v * (1.0 - s)));
          gy *= v * s;
        }
        double sb = 0, sa = 0;
        for (int64_t s = 0; s < N; s++) {
          const double e = std::exp(dt * rate(d * N + s)), p = e * h[(size_t)(t * N + s)];
          const double gr = G_[(size_t)s] + gy * (double)cm[row + cg + s];
          (joined ? db : dc)[(size_t)(row + cg + s)] += gy * h[(size_t)((t + 1) * N + s)];
          db[(size_t)(row + s)] += gr * dt * u;
          sb += gr * (double)bm[row + s];
          sa += gr * p * rate(d * N + s);
          da[(size_t)(d * N + s)] += gr * p * dt * (logs ? rate(d * N + s) : 1.0);
          G_[(size_t)s] = gr * e;
        }
        if (o.out[0]) o.out[0][at] = (T)(dt * sb + (skip ? gy * (double)skip[d] : 0.0));
        const double ddt = (u * sb + sa) * (soft ? sigmoid(given_dt) : 1.0);
        if (o.out[1]) o.out[1][at] = (T)ddt;
        dbias[(size_t)d] += ddt;
        dd[(size_t)d] += gy * u;
      }
      if (o.out[7])
        for (int64_t s = 0; s < N; s++) o.out[7][(b * D + d) * N + s] = (T)G_[(size_t)s];
    }
  }
  auto store = [&](size_t r, const std::vector<double>& v) {
    if (grad && o.out[r])
      for (size_t k = 0; k < v.size(); k++) o.out[r][k] = (T)v[k];
  };
  if (grad) {
    store(2, da);
    store(3, db);
    if (!joined) store(4, dc);
    store(5, dd);
    store(8, dbias);
  }
}

template <class T>
void rotary_norm(const Operands<T>& o) {
  const auto& q = o.q;
  const T *x = o.arg(q.x), *gain = o.arg(q.gain), *dy = o.arg(q.dy);
  const int32_t* pos = (const int32_t*)o.slot[(size_t)q.positions];
  const int64_t R = o.in.sequence.turn, half = R / 2, hd = q.head, S = (int64_t)o.in.sequence.sections.size();
  std::vector<double> dgain((size_t)(S * hd), 0.0), v((size_t)hd), u((size_t)hd);
  for (int64_t b = 0; b < q.batch; b++)
    for (int64_t t = 0; t < q.length; t++) {
      const long double p = q.positions_from ? (long double)pos[b] + t : (long double)pos[q.shared_positions ? t : b * q.length + t];
      for (int64_t h = 0; h < q.heads; h++) {
        const int64_t at = ((b * q.length + t) * q.heads + h) * hd;
        int64_t s = 0, last = 0;
        for (; s < S; s++) {
          last += o.in.sequence.sections[(size_t)s];
          if (h < last) break;
        }
        if (s == S) {  // a head that passes
          if (o.out[0])
            for (int64_t i = 0; i < hd; i++) o.out[0][at + i] = dy ? dy[at + i] : x[at + i];
          continue;
        }
        double ss = 0;
        for (int64_t i = 0; i < hd; i++) ss += (double)x[at + i] * (double)x[at + i];
        const double r = gain ? 1.0 / std::sqrt(ss / (double)hd + o.in.sequence.eps) : 1.0;
        auto scale = [&](int64_t i) { return gain ? (double)gain[s * hd + i] : 1.0; };
        auto angle = [&](int64_t i) { return p * powl((long double)o.in.sequence.base, -2.0L * i / R); };
        if (!dy) {
          for (int64_t i = 0; i < hd; i++) v[(size_t)i] = (double)x[at + i] * r * scale(i);
          for (int64_t i = 0; i < half; i++) {
            const double c = (double)cosl(angle(i)), sn = (double)sinl(angle(i)), f = v[(size_t)i], g = v[(size_t)(i + half)];
            v[(size_t)i] = f * c - g * sn;
            v[(size_t)(i + half)] = g * c + f * sn;
          }
          for (int64_t i = 0; i < hd; i++) o.out[0][at + i] = (T)v[(size_t)i];
          continue;
        }
        for (int64_t i = 0; i < hd; i++) u[(size_t)i] = (double)dy[at + i];
        for (int64_t i = 0; i < half; i++) {
          const double c = (double)cosl(angle(i)), sn = (double)sinl(angle(i)), f = u[(size_t)i], g = u[(size_t)(i + half)];
          u[(size_t)i] = f * c + g * sn;
          u[(size_t)(i + half)] = g * c - f * sn;
        }
        double m = 0;
        for (int64_t i = 0; i < hd; i++) {
          dgain[(size_t)(s * hd + i)] += u[(size_t)i] * (double)x[at + i] * r;
          m += u[(size_t)i] * scale(i) * (double)x[at + i] * r;
        }
        m /= (double)hd;
        if (o.out[0])
          for (int64_t i = 0; i < hd; i++)
            o.out[0][at + i] = (T)(gain ? r * (u[(size_t)i] * scale(i) - (double)x[at + i] * r * m) : u[(size_t)i]);
      }
    }
  if (dy && o.out[1])
    for (size_t k = 0; k < dgain.size(); k++) o.out[1][k] = (T)dgain[k];
}

// The rows of a query, key or value operand: `heads` of them from `at` on in rows of `stride` values.
template <class T>
struct Rows {
  const T* p;
  int64_t stride, head;
  const T* operator()(int64_t position, int64_t h) const { return p + position * stride + h * head; }
};

template <class T>
void attention(const Operands<T>& o) {
  const auto& q = o.q;
  const int64_t L = q.length, H = q.heads, G = q.keys, hd = q.head, per = H / G, row = q.k < 0 ? (H + 2 * G) * hd : H * hd;
  const bool joined = q.k < 0, grad = q.dy >= 0, causal = o.has(RG_ATTEND_CAUSAL);
  const Rows<T> qs{o.arg(q.x), row, hd}, ks{joined ? o.arg(q.x) + H * hd : o.arg(q.k), joined ? row : G * hd, hd},
      vs{joined ? o.arg(q.x) + (H + G) * hd : o.arg(q.v), joined ? row : G * hd, hd};
  const T *slopes = o.arg(q.slopes), *dy = o.arg(q.dy);
  const int32_t* docs = q.documents < 0 ? nullptr : (const int32_t*)o.slot[(size_t)q.documents];
  const int32_t* prefix = q.prefix < 0 ? nullptr : (const int32_t*)o.slot[(size_t)q.prefix];
  const double scale = o.in.sequence.base, cap = o.in.sequence.eps;
  std::vector<double> dq, dk, dv, dslope((size_t)(q.batch * H), 0.0);
  if (grad) {
    dq.assign((size_t)(q.batch * L * H * hd), 0.0);
    dk.assign((size_t)(q.batch * L * G * hd), 0.0);
    dv.assign(dk.size(), 0.0);
  }
#pragma omp parallel for
  for (int64_t bg = 0; bg < q.batch * G; bg++) {
    const int64_t b = bg / G, g = bg % G, n = o.end(b);
    std::vector<double> s((size_t)L), slope_of(s.size());
    for (int64_t h = g * per; h < (g + 1) * per; h++)
      for (int64_t i = 0; i < L; i++) {
        const T* qi = qs(b * L + i, h);
        std::vector<int64_t> seen;
        const bool in = i < n && (!docs || docs[b * L + i] >= 0);
        for (int64_t j = 0; in && j < n; j++)
          if ((!causal || j <= i || (prefix && j < prefix[b])) && (!docs || docs[b * L + j] == docs[b * L + i])) seen.push_back(j);
        double top = -INFINITY, sum = 0.0;
        for (int64_t j : seen) {
          double u = 0.0;
          const T* kj = ks(b * L + j, g);
          for (int64_t d = 0; d < hd; d++) u += (double)qi[d] * (double)kj[d];
          u *= scale;
          slope_of[(size_t)j] = 1.0;
          if (cap > 0) {
            const double t = std::tanh(u / cap);
            u = cap * t;
            slope_of[(size_t)j] = 1.0 - t * t;
          }
          if (slopes) u -= (double)slopes[h] * (double)std::llabs(i - j);
          s[(size_t)j] = u;
          top = u > top || std::isnan(u) ? u : top;
        }
        for (int64_t j : seen) sum += s[(size_t)j] = std::exp(s[(size_t)j] - top);
        for (int64_t j : seen) s[(size_t)j] /= sum;
        if (!grad) {
          if (o.out[0])
            for (int64_t d = 0; d < hd; d++) {
              double y = 0.0;
              for (int64_t j : seen) y += s[(size_t)j] * (double)vs(b * L + j, g)[d];
              o.out[0][((b * L + i) * H + h) * hd + d] = (T)y;
            }
          if (o.out[1]) {
            o.out[1][(b * H + h) * L + i] = seen.empty() ? std::numeric_limits<T>::max() : (T)(top / std::log(2.0));
            o.out[1][(q.batch * H + b * H + h) * L + i] = seen.empty() ? (T)0 : (T)(1.0 / sum);
          }
          continue;
        }
        const T* gi = dy + ((b * L + i) * H + h) * hd;
        double dot = 0.0;
        std::vector<double> dp(seen.size(), 0.0);
        for (size_t c = 0; c < seen.size(); c++) {
          for (int64_t d = 0; d < hd; d++) dp[c] += (double)gi[d] * (double)vs(b * L + seen[c], g)[d];
          dot += s[(size_t)seen[c]] * dp[c];
        }
        for (size_t c = 0; c < seen.size(); c++) {
          const int64_t j = seen[c];
          const double p = s[(size_t)j], ds = p * (dp[c] - dot), du = ds * slope_of[(size_t)j] * scale;
          const T* kj = ks(b * L + j, g);
          for (int64_t d = 0; d < hd; d++) {
            dv[(size_t)(((b * L + j) * G + g) * hd + d)] += p * (double)gi[d];
            dq[(size_t)(((b * L + i) * H + h) * hd + d)] += du * (double)kj[d];
            dk[(size_t)(((b * L + j) * G + g) * hd + d)] += du * (double)qi[d];
          }
          dslope[(size_t)(b * H + h)] -= ds * (double)std::llabs(i - j);
        }
      }
  }
  if (!grad) return;
  auto put = [&](size_t r, const std::vector<double>& v, int64_t heads, int64_t stride, int64_t at) {
    if (!o.out[r]) return;
    for (int64_t t = 0; t < q.batch * L; t++)
      for (int64_t d = 0; d < heads * hd; d++) o.out[r][t * stride + at + d] = (T)v[(size_t)(t * heads * hd + d)];
  };
  put(0, dq, H, row, 0);
  put(joined ? 0 : 1, dk, G, joined ? row : G * hd, joined ? H * hd : 0);
  put(joined ? 0 : 2, dv, G, joined ? row : G * hd, joined ? (H + G) * hd : 0);
  if (o.out[3])
    for (int64_t h = 0; h < H; h++) {
      double sum = 0.0;
      for (int64_t b = 0; b < q.batch; b++) sum += dslope[(size_t)(b * H + h)];
      o.out[3][h] = (T)sum;
    }
}

template <class T>
void paged_attention(const Operands<T>& o) {
  const auto& q = o.q;
  const int64_t L = q.length, H = q.heads, G = q.keys, hd = q.head, per = H / G, row = q.k < 0 ? (H + 2 * G) * hd : H * hd;
  const bool joined = q.k < 0;
  const Rows<T> qs{o.arg(q.x), row, hd}, ks{joined ? o.arg(q.x) + H * hd : o.arg(q.k), joined ? row : G * hd, hd},
      vs{joined ? o.arg(q.x) + (H + G) * hd : o.arg(q.v), joined ? row : G * hd, hd};
  const T *slopes = o.arg(q.slopes), *kp = o.arg(q.k_pages), *vp = o.arg(q.v_pages);
  const int32_t *table = (const int32_t*)o.slot[(size_t)q.table], *first = (const int32_t*)o.slot[(size_t)q.first];
  const double scale = o.in.sequence.base, cap = o.in.sequence.eps;
  const int64_t room = q.table_pages * q.page;
  // The first value of position p's row among the pages, or -1 where it has none.
  auto place = [&](int64_t b, int64_t p) -> int64_t {
    if (p < 0 || p >= room) return -1;
    const int64_t page = table[b * q.table_pages + p / q.page];
    return page < 0 || page >= q.pages ? -1 : (page * q.page + p % q.page) * G * hd;
  };
  auto begin_of = [&](int64_t b) { return std::min<int64_t>(std::max<int64_t>(0, first[b]), 1ll << 30); };
  for (int64_t b = 0; b < q.batch; b++) {
    const int64_t n = o.end(b), begin = begin_of(b);
    for (int64_t i = 0; i < L; i++)
      for (int64_t h = 0; h < H && o.out[0]; h++) {
        T* y = o.out[0] + ((b * L + i) * H + h) * hd;
        std::fill(y, y + hd, (T)0);
        if (i >= n) continue;
        const int64_t g = h / per;
        std::vector<double> s;
        std::vector<const T*> value;
        double top = -INFINITY, sum = 0.0;
        auto add = [&](const T* k, const T* v, int64_t distance) {
          double u = 0.0;
          for (int64_t d = 0; d < hd; d++) u += (double)qs(b * L + i, h)[d] * (double)k[d];
          u *= scale;
          if (cap > 0) u = cap * std::tanh(u / cap);
          if (slopes) u -= (double)slopes[h] * (double)distance;
          s.push_back(u);
          value.push_back(v);
          top = u > top || std::isnan(u) ? u : top;
        };
        for (int64_t p = 0; p < std::min(begin, room); p++) {
          const int64_t at = place(b, p);
          if (at >= 0) add(kp + at + g * hd, vp + at + g * hd, begin + i - p);
        }
        for (int64_t j = 0; j <= i; j++) add(ks(b * L + j, g), vs(b * L + j, g), i - j);
        for (double& u : s) sum += u = std::exp(u - top);
        for (int64_t d = 0; d < hd; d++) {
          double v = 0.0;
          for (size_t c = 0; c < s.size(); c++) v += s[c] / sum * (double)value[c][d];
          y[d] = (T)v;
        }
      }
  }
  const int64_t all = q.pages * q.page * G * hd;
  for (int r : {1, 2}) {
    T* out = o.out[(size_t)r];
    if (!out) continue;
    const T* from = r == 1 ? kp : vp;
    if (out != from) std::copy(from, from + all, out);
    for (int64_t b = 0; b < q.batch; b++)
      for (int64_t i = 0; i < o.end(b); i++) {
        const int64_t at = place(b, begin_of(b) + i);
        if (at < 0) continue;
        for (int64_t g = 0; g < G; g++) {
          const T* src = (r == 1 ? ks : vs)(b * L + i, g);
          std::copy(src, src + hd, out + at + g * hd);
        }
      }
  }
}

template <class T, class Slot>
void joint_norm(const rgplan::Instr& in, const Operands<T>& o, Slot slot_bytes) {
  long double sum = 0.0L;
  for (auto& a : in.args) {
    int64_t n = 1;
    for (int64_t d : a.shape) n *= d;
    const T* x = (const T*)slot_bytes(a.slot);
    for (int64_t k = 0; k < n; k++) sum += (long double)x[k] * (long double)x[k];
  }
  if (o.out[0]) o.out[0][0] = (T)std::sqrt(sum);
}

template <class T, class Slot>
void run(const rgplan::Instr& in, Slot slot_bytes) {
  Operands<T> o{in, rgplan::sequence_of(in), {}, {}};
  for (auto& a : in.args) o.slot.push_back(slot_bytes(a.slot));
  o.out.assign(std::max<size_t>(o.q.results.size(), 1), nullptr);
  if (!rgplan::is_multi_result(in.op)) o.out[0] = (T*)slot_bytes(in.dst);
  for (auto& r : in.outs) o.out[(size_t)r.first] = (T*)slot_bytes(r.second);
  if (in.op == RG_OP_CAUSAL_CONV || in.op == RG_OP_CAUSAL_CONV_GRAD) causal_conv(o);
  else if (in.op == RG_OP_ATTENTION || in.op == RG_OP_ATTENTION_GRAD) attention(o);
  else if (in.op == RG_OP_PAGED_ATTENTION) paged_attention(o);
  else if (in.op == RG_OP_JOINT_NORM) joint_norm(in, o, slot_bytes);
  else if (in.op == RG_OP_SELECTIVE_SCAN || in.op == RG_OP_SELECTIVE_SCAN_GRAD) selective_scan(o);
  else rotary_norm(o);
}

}  // namespace rgseq
