// The sequence operators of include/rg_plan.h on the CPU: every value computed in 64 bits from the
// formulas, one position after another, and rounded once to the operator's dtype when stored. The
// angles of a rotation, whose error grows with the position, are formed in extended precision.
#pragma once
#include <cmath>
#include <cstdint>
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

template <class T, class Slot>
void run(const rgplan::Instr& in, Slot slot_bytes) {
  Operands<T> o{in, rgplan::sequence_of(in), {}, {}};
  for (auto& a : in.args) o.slot.push_back(slot_bytes(a.slot));
  o.out.assign(std::max<size_t>(o.q.results.size(), 1), nullptr);
  if (!rgplan::is_multi_result(in.op)) o.out[0] = (T*)slot_bytes(in.dst);
  for (auto& r : in.outs) o.out[(size_t)r.first] = (T*)slot_bytes(r.second);
  if (in.op == RG_OP_CAUSAL_CONV || in.op == RG_OP_CAUSAL_CONV_GRAD) causal_conv(o);
  else if (in.op == RG_OP_SELECTIVE_SCAN || in.op == RG_OP_SELECTIVE_SCAN_GRAD) selective_scan(o);
  else rotary_norm(o);
}

}  // namespace rgseq
