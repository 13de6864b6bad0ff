// pkv_verify.hip -- verification of drafted tokens against the target's
// probabilities, from given random numbers (gfx950).
//
// A request with n drafts d_0 .. d_{n-1} has n + 1 target rows.  With p_i =
// softmax(target row i / T) and q_i = softmax(draft row i / T) (or all of q_i on
// d_i without draft rows), draft i is kept while u_i q_i(d_i) < p_i(d_i); at
// the first one that is not, the next token is drawn from max(p_i - q_i, 0),
// after the last draft from p_n: the first token whose running sum of weights
// passes v times their total.  Greedy requests keep drafts that are the
// row's first maximum and end with a row's first maximum.
//
// Every decision is that of 64-bit arithmetic: exponentials, sums and
// comparisons are doubles.  On this GPU a double multiply-add issues at the
// rate of a float one, so 2^x is kept to such operations: x is split into an
// integer n and z in [-1/2, 1/2] by adding and subtracting 1.5 2^52, 2^z is a
// polynomial of degree 10 (interpolated at the Chebyshev nodes, error 3e-16
// relative), and n is added to the exponent field: 17 operations an element
// against 2 or 4 bytes read.  A sum needs no maximum, only a reference near
// the row's size, for a double holds 2^500 times its weight as well: a thread
// keeps the largest logit of its first group and moves it only when a logit
// is past that range.
//
// Three launches: statistics of every row (reference and sum, or the argmax of
// greedy rows) in chunks; per request the kept drafts and the last row's
// weights, summed in segments of 512 tokens (a wave's load); the segment in
// which the running sum passes and the token in it.  128 requests, 1-5 drafts,
// vocabulary 128,256, bf16 against bf16: 92 + 34 + 6.7 us under a profiler, bound by
// the issue of the f64 instructions (35 M of a wave, vector units 70 % busy); the
// logits alone would take 48 us at the rate of a copy.  6 requests of 32,000
// (f32): 5.9 + 5.8 + 4.0 us, three chains of memory round trips.
#include <algorithm>

#include "pkv_device.h"
#include "pkv_internal.h"

namespace pkv {
namespace {

constexpr int kVT = 256;  // threads
constexpr int kVW = kVT / kWave;

struct RowPart {  // of one chunk of a row
  float m;        // a logit near its largest (greedy: the largest)
  int arg;        // greedy: its first index
  double s;       // sum of 2^((l - m) c)
};
constexpr int kSeg = 512;  // tokens of a segment: 8 per lane of a wave
struct Decision {
  double inv_p, inv_q;  // 1 / sum of the target and the draft row (0: none)
  float m_p, m_q;
  int row;      // target row of the next token
  int draft;    // its draft row, or -1
  int not_tok;  // token whose weight is taken out (no draft rows), or -1
  int token;    // >= 0: the token itself
  int at;       // where it goes
  int pad;
};

struct VerifyKArgs {
  const char* target;
  const char* draft;  // or null
  long long t_stride, d_stride;  // elements
  int draft_dt;
  const int32_t* tokens;
  const int32_t* cu;
  const float* u;
  const float* u_last;
  const float* temps;  // or null: greedy
  int batch, total, vocab;
  int g1, len1;  // chunks of the statistics
  int g2, segs;  // workgroups and segments of the weights
  RowPart* rows;      // [total + batch target rows, total draft rows][g1]
  double* parts;      // [batch][segs]
  Decision* decide;   // [batch]
  int32_t* out;       // [total + batch]
  int32_t* accepted;  // [batch]
};

// 2^t for |t| <= 1000.
__device__ __forceinline__ double exp2_near(double t) {
  const double shift = 6755399441055744.0;  // 1.5 2^52: rounds t to an integer
  const double r = t + shift;
  const double z = t - (r - shift);
  double p = 7.072585949269223e-09;
  p = fma(p, z, 1.0208690299958306e-07);
  p = fma(p, z, 1.321544258792169e-06);
  p = fma(p, z, 1.5252657260200837e-05);
  p = fma(p, z, 0.0001540353044173605);
  p = fma(p, z, 0.0013333558230164974);
  p = fma(p, z, 0.009618129107606888);
  p = fma(p, z, 0.05550410866444772);
  p = fma(p, z, 0.24022650695910097);
  p = fma(p, z, 0.69314718055995);
  p = fma(p, z, 1.0);
  // r's low word is the integer
  const unsigned hi = (unsigned)__double2hiint(p) + ((unsigned)__double2loint(r) << 20);
  return __hiloint2double((int)hi, __double2loint(p));
}
// NaN as -inf, +inf as the largest float: the maximum and all that equal it
// weigh 1, the others nothing.
__device__ __forceinline__ float kept(float l) {
  return l > -INFINITY ? fminf(l, 3.402823466e+38f) : -INFINITY;
}
// Weight 2^((l - m) c) of a logit against reference m, at most 2^532; less
// than 2^-1000 is 0.
__device__ __forceinline__ double weight(float l, float m, double c) {
  const double t = ((double)kept(l) - (double)m) * c;
  const double w = exp2_near(fmin(fmax(t, -1000.0), 1000.0));
  return t > -1000.0 ? w : 0.0;  // (false for NaN: -inf against -inf)
}

// A row's reference and the logits around it whose weights are about 2^-500 to
// 2^500: [lo, hi].  far: these are not to be told from m itself (m is a type's
// lowest value, say) or end past the largest float (temperatures from 1e35 on), so
// every logit needs care.  Else |m| < 2^20 span, so rounding m +- span to 32 bits
// moves either end by at most (2^-4 + 2^-24) span: the weights of lo and hi are
// 2^-532 .. 2^-468 and 2^468 .. 2^532.
struct Ref {
  float m, lo, hi;
  bool far;
  double c, m64;
};
__device__ __forceinline__ void set_ref(Ref& r, float m) {
  const float span = (float)(500.0 / r.c);
  r.m = m;
  r.far = !(span > fabsf(m) * 0x1p-20f && span + fabsf(m) < 3.4e38f);
  r.lo = m - span;
  r.hi = m + span;
  r.m64 = m;
}
// A term of a sum: logits below the range count as its lower end, those above it
// as its upper end.  (One instruction; min and max of unpacked words cost another
// each, to quiet NaN.)
__device__ __forceinline__ double weight_clamped(float l, const Ref& r) {
  float x;
  asm("v_med3_f32 %0, %1, %2, %3" : "=v"(x) : "v"(l), "v"(r.lo), "v"(r.hi));
  // (a product and one addition would be off by the rounding of m c)
  return exp2_near(((double)x - r.m64) * r.c);
}
// Below the weight of any hi: a group whose sum is less has no logit past hi.
constexpr double kNearEnd = 0x1p460;
__device__ __forceinline__ float largest(const float (&x)[8]) {
  float top = kept(x[0]);
#pragma unroll
  for (int e = 1; e < 8; ++e) top = fmaxf(top, kept(x[e]));
  return top;
}

template <int DT>
__device__ __forceinline__ float logit(const char* row, long long i) {
  if constexpr (DT == PKV_F32) return reinterpret_cast<const float*>(row)[i];
  const uint16_t w = reinterpret_cast<const uint16_t*>(row)[i];
  return DT == PKV_BF16 ? bf16lo(w) : f16lo(w);
}
__device__ __forceinline__ float logit_dt(int dt, const char* row, long long i) {
  return dt == PKV_F32 ? logit<PKV_F32>(row, i)
                       : dt == PKV_F16 ? logit<PKV_F16>(row, i) : logit<PKV_BF16>(row, i);
}
__device__ __forceinline__ int bytes_of(int dt) { return dt == PKV_F32 ? 4 : 2; }

// c of exp(l / T) = 2^(l c); 0: greedy (T is not positive or not finite: 1 / inf is 0).
__device__ __forceinline__ double exponent(const VerifyKArgs& a, int b) {
  const float t = a.temps ? a.temps[b] : 0.0f;
  return t > 0.0f ? 1.4426950408889634074 / (double)t : 0.0;
}
// Drafts of request b, within the call's total.
__device__ __forceinline__ int first_draft(const VerifyKArgs& a, int b) {
  return min(max(a.cu[b], 0), a.total);
}
// The last request k with cu[k] + step k <= x (0 if none has): the request of
// target row x (step 1) or of draft x (step 0).  64 at a time, a wave's ballot.
__device__ __forceinline__ int request_of(const VerifyKArgs& a, int x, int step) {
  const int lane = threadIdx.x & 63;
  int first = 0, n = a.batch;
  while (n > 1) {
    const int stride = (n + kWave - 1) / kWave;
    const int k = first + lane * stride;
    const bool ok = lane * stride < n && first_draft(a, k) + step * k <= x;
    first += max(__popcll(__ballot(ok)) - 1, 0) * stride;
    n = min(stride, a.batch - first);
  }
  return first;
}

// What RowPart holds, of a part of a row.
struct Stat {
  float m;
  int arg;
  double s;
};
constexpr Stat kNoStat{-INFINITY, 0, 0.0};
__device__ __forceinline__ void join(Stat& x, const Stat& y, double c) {
  const float m = fmaxf(x.m, y.m);
  if (y.m > x.m || (y.m == x.m && y.arg < x.arg)) x.arg = y.arg;
  if (c != 0.0) x.s = x.s * weight(x.m, m, c) + y.s * weight(y.m, m, c);
  x.m = m;
}

// Elements i .. i + 7 of a row as floats, i a multiple of 8; those from n on
// are -inf.  VEC: rows start on 16 bytes.
constexpr int kN = 8;
template <int DT, bool VEC>
__device__ __forceinline__ void load8(const char* row, int i, int n, float (&x)[kN]) {
  if (VEC && i + kN <= n) {
    if constexpr (DT == PKV_F32) {
      float y[4], z[4];
      widen16<DT, 4>(ld16(row + (size_t)i * 4), y);
      widen16<DT, 4>(ld16(row + (size_t)i * 4 + 16), z);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        x[e] = y[e];
        x[4 + e] = z[e];
      }
    } else {
      widen16<DT, 8>(ld16(row + (size_t)i * 2), x);
    }
    return;
  }
#pragma unroll
  for (int e = 0; e < kN; ++e) x[e] = i + e < n ? logit<DT>(row, i + e) : -INFINITY;
}

// Statistics of elements c0 .. c1 - 1 by the workgroup; thread 0 has them.
template <int DT, bool VEC>
__device__ __forceinline__ Stat chunk_stat(const char* row, int c0, int c1, double c, Stat* lds) {
  Stat st = kNoStat;
  if (c == 0.0) {
    for (int i = c0 + (int)threadIdx.x * kN; i < c1; i += kVT * kN) {
      float x[kN];
      load8<DT, VEC>(row, i, c1, x);
#pragma unroll
      for (int e = 0; e < kN; ++e)
        if (x[e] > st.m) {
          st.m = x[e];
          st.arg = i + e;
        }
    }
  } else {
    Ref r;
    r.c = c;
    const int step = kVT * kN;
    float x[kN];
    // the reference: the largest of the first group with anything in it
    int i = c0 + (int)threadIdx.x * kN;
    float top = -INFINITY;
    for (; i < c1; i += step) {
      load8<DT, VEC>(row, i, c1, x);
      top = largest(x);
      if (top > -INFINITY) break;
    }
    set_ref(r, top);
    double sum = 0.0;
    while (i < c1) {
      float y[kN];  // the next group, on its way
      if (i + step < c1) load8<DT, VEC>(row, i + step, c1, y);
      double g = 0.0;
#pragma unroll
      for (int e = 0; e < kN; ++e) g += weight_clamped(x[e], r);
      if (g < kNearEnd && !r.far) {
        sum += g;
      } else {  // a logit near the range's upper end or past it, or NaN
        top = largest(x);
        if (top > r.hi) {
          sum *= weight(r.m, top, c);
          set_ref(r, top);
        }
#pragma unroll
        for (int e = 0; e < kN; ++e) sum += weight(x[e], r.m, c);
      }
      i += step;
#pragma unroll
      for (int e = 0; e < kN; ++e) x[e] = y[e];
    }
    st.m = r.m;
    st.s = sum;
  }
  // over the wave: the largest reference, and every sum against it once
  float m = st.m;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) m = fmaxf(m, __shfl_xor(m, o, kWave));
  if (c == 0.0) {
    int arg = st.m == m ? st.arg : INT32_MAX;  // (0 where nothing is above -inf)
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) arg = min(arg, __shfl_xor(arg, o, kWave));
    st.arg = arg;
  } else {
    st.s = wave_sum(st.s * weight(st.m, m, c));
  }
  st.m = m;
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = st;
  __syncthreads();
  if (threadIdx.x == 0)
    for (int w = 1; w < kVW; ++w) join(st, lds[w], c);
  return st;
}

// Grid rows x g1: target rows first, then draft rows.  Draft rows of greedy
// requests are not read.
template <int DT, int DDT, bool VEC>
__global__ void __launch_bounds__(kVT) verify_stat_kernel(VerifyKArgs a) {
  __shared__ Stat lds[kVW];
  const int n_target = a.total + a.batch;
  const int r = blockIdx.x / a.g1, chunk = blockIdx.x % a.g1;
  const bool draft = r >= n_target;
  const int b = draft ? request_of(a, r - n_target, 0) : request_of(a, r, 1);
  const double c = exponent(a, b);
  if (draft && c == 0.0) return;
  const int c0 = chunk * a.len1, c1 = min(c0 + a.len1, a.vocab);
  const Stat st =
      draft ? chunk_stat<DDT, VEC>(a.draft + (r - n_target) * a.d_stride * bytes_of(DDT), c0, c1, c, lds)
            : chunk_stat<DT, VEC>(a.target + r * a.t_stride * bytes_of(DT), c0, c1, c, lds);
  if (threadIdx.x == 0) a.rows[(size_t)r * a.g1 + chunk] = {st.m, st.arg, st.s};
}

// A row's statistics from its chunks', four at a time side by side.
__device__ __forceinline__ Stat row_stat(const VerifyKArgs& a, int r, double c) {
  constexpr int U = 4;
  Stat st = kNoStat;
  for (int k0 = 0; k0 < a.g1; k0 += U) {
    RowPart y[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      y[u] = a.rows[(size_t)r * a.g1 + min(k0 + u, a.g1 - 1)];
      if (k0 + u >= a.g1) y[u].m = -INFINITY;
    }
    Stat x = kNoStat;
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (y[u].m > x.m) {
        x.m = y[u].m;
        x.arg = y[u].arg;
      }
    if (c != 0.0) {
#pragma unroll
      for (int u = 0; u < U; ++u) x.s += y[u].s * weight(y[u].m, x.m, c);
    }
    if (k0 == 0) st = x;
    else join(st, x, c);
  }
  return st;
}

// The drafts of request b that are kept and what its next token is drawn
// from, in every thread.  Thread i has draft i and its rows; one past the last
// draft stands for the request's end.
__device__ __forceinline__ Decision decide(const VerifyKArgs& a, int b, int& n, int& kept, int* lds,
                                           Decision& shared) {
  const int d0 = first_draft(a, b);
  n = max(first_draft(a, b + 1) - d0, 0);
  const double c = exponent(a, b);
  const int n_target = a.total + a.batch;
  const int tdt = a.draft_dt >> 8, ddt = a.draft_dt & 255;
  for (int i0 = 0;; i0 += kVT) {  // uniform, ends at i = n
    const int i = i0 + (int)threadIdx.x;
    bool keep = true;
    Decision d{};
    if (i <= n) {
      const int r = d0 + b + i;
      const bool some = i < n, drawn = some && c != 0.0 && a.draft;
      const int tok = some ? a.tokens[d0 + i] : -1;
      const double u = some && c != 0.0 ? (double)a.u[d0 + i] : 0.0;
      const bool known = tok >= 0 && tok < a.vocab;
      float lp = 0.0f, lq = 0.0f;
      if (known && c != 0.0) {
        lp = logit_dt(tdt, a.target + r * a.t_stride * bytes_of(tdt), tok);
        if (drawn) lq = logit_dt(ddt, a.draft + (d0 + i) * a.d_stride * bytes_of(ddt), tok);
      }
      const Stat p = row_stat(a, r, c);
      const Stat q = drawn ? row_stat(a, n_target + d0 + i, c) : kNoStat;
      if (!known) {
        keep = false;
      } else if (c == 0.0) {
        keep = tok == p.arg && p.m > -INFINITY;
      } else {
        // u q(d) < p(d); a draft row without weight has q = 0
        const double pd = p.s > 0.0 ? weight(lp, p.m, c) / p.s : 0.0;
        const double qd = !a.draft ? 1.0 : q.s > 0.0 ? weight(lq, q.m, c) / q.s : 0.0;
        keep = u * qd < pd;
      }
      d.row = d.at = r;
      d.draft = drawn && q.s > 0.0 ? d0 + i : -1;
      d.not_tok = some && c != 0.0 && !a.draft ? tok : -1;
      d.token = c == 0.0 ? p.arg : p.s > 0.0 ? -1 : 0;
      d.m_p = p.m;
      d.inv_p = p.s > 0.0 ? 1.0 / p.s : 0.0;
      d.m_q = d.draft >= 0 ? q.m : 0.0f;
      d.inv_q = d.draft >= 0 ? 1.0 / q.s : 0.0;
    }
    const unsigned long long lost = __ballot(!keep);
    if ((threadIdx.x & 63) == 0)
      lds[threadIdx.x >> 6] = lost ? (int)threadIdx.x + __ffsll((long long)lost) - 1 : INT32_MAX;
    __syncthreads();
    int first = INT32_MAX;
#pragma unroll
    for (int w = 0; w < kVW; ++w) first = min(first, lds[w]);
    if (first != INT32_MAX) {
      kept = i0 + first;
      if ((int)threadIdx.x == first) shared = d;
      __syncthreads();
      return shared;
    }
    __syncthreads();
  }
}

// Probabilities below this count as 0 in a draw: the weight of a logit below
// the reference's range is that of its lower end, 2^-468 at most, not 0.
constexpr double kNothing = 0x1p-400;

// Probabilities of eight logits.
__device__ __forceinline__ void probs8(const float (&x)[kN], const Ref& r, double inv, double (&p)[kN]) {
  float sum = x[0];
#pragma unroll
  for (int e = 1; e < kN; ++e) sum += x[e];
  if (sum == sum && !r.far) {
#pragma unroll
    for (int e = 0; e < kN; ++e) p[e] = weight_clamped(x[e], r) * inv;
  } else {  // NaN, or both infinities
#pragma unroll
    for (int e = 0; e < kN; ++e) p[e] = weight(x[e], r.m, r.c) * inv;
  }
}
// What the next token of a request is drawn from.
struct Draw {
  Ref p, q;
};
__device__ __forceinline__ Draw draw_of(const Decision& d, double c) {
  Draw w;
  w.p.c = w.q.c = c;
  set_ref(w.p, d.m_p);
  set_ref(w.q, d.m_q);
  return w;
}
// Weights of tokens i .. i + 7, i a multiple of 8.
template <int DT, int DDT, bool VEC>
__device__ __forceinline__ void weigh8(const VerifyKArgs& a, const Decision& d, const Draw& r, int i,
                                       double (&w)[kN]) {
  float lp[kN], lq[kN];
  load8<DT, VEC>(a.target + d.row * a.t_stride * bytes_of(DT), i, a.vocab, lp);
  if (d.draft >= 0) {
    load8<DDT, VEC>(a.draft + d.draft * a.d_stride * bytes_of(DDT), i, a.vocab, lq);
    double q[kN];
    probs8(lq, r.q, d.inv_q, q);
    probs8(lp, r.p, d.inv_p, w);
#pragma unroll
    for (int e = 0; e < kN; ++e) w[e] = fmax(w[e] - q[e], 0.0);
  } else {
    probs8(lp, r.p, d.inv_p, w);
    if ((unsigned)(d.not_tok - i) < (unsigned)kN) {
#pragma unroll
      for (int e = 0; e < kN; ++e)
        if (i + e == d.not_tok) w[e] = 0.0;
    }
  }
}

// Grid batch x g2; a wave takes every (4 g2)-th segment.
template <int DT, int DDT, bool VEC>
__global__ void __launch_bounds__(kVT) verify_weight_kernel(VerifyKArgs a) {
  __shared__ int lds[kVW];
  __shared__ Decision shared;
  const int b = blockIdx.x / a.g2, chunk = blockIdx.x % a.g2;
  int n = 0, n_kept = 0;
  const Decision d = decide(a, b, n, n_kept, lds, shared);
  if (chunk == 0) {
    const int d0 = d.row - b - n_kept;
    if (threadIdx.x == 0) {
      a.decide[b] = d;
      a.accepted[b] = n_kept;
    }
    for (int i = threadIdx.x; i <= n; i += kVT)
      a.out[d0 + b + i] = i < n_kept ? a.tokens[d0 + i] : i == n_kept ? max(d.token, 0) : -1;
  }
  if (d.token >= 0) return;
  const Draw r = draw_of(d, exponent(a, b));
  const int lane = threadIdx.x & 63;
  for (int k = chunk * kVW + (int)(threadIdx.x >> 6); k < a.segs; k += a.g2 * kVW) {
    double w[kN], x = 0.0;
    weigh8<DT, DDT, VEC>(a, d, r, k * kSeg + lane * kN, w);
#pragma unroll
    for (int e = 0; e < kN; ++e) x += w[e];
    x = wave_sum(x);
    if (lane == 0) a.parts[(size_t)b * a.segs + k] = x;
  }
}

// Where the running sum of x(0), x(1), .. x(n - 1) first passes `want` (the last
// that counts if rounding leaves it short), and the sum before it; -1 if none
// counts.  One wave, consecutive numbers per lane.
template <class X>
__device__ int first_past(int n, double want, double& before, X x) {
  const int lane = threadIdx.x & 63;
  const int per = (n + kWave - 1) / kWave;
  const int k0 = min(lane * per, n), k1 = min(k0 + per, n);
  double mine = 0.0;
  bool some = false;
  for (int k = k0; k < k1; ++k) {
    const double v = x(k);
    mine += v;
    some |= v > kNothing;
  }
  const double upto = before + wave_incl_scan(mine);
  const unsigned long long hit = __ballot(some && upto > want), any = __ballot(some);
  if (!any) return -1;
  const int l = hit ? __ffsll((long long)hit) - 1 : 63 - __clzll((long long)any);
  double run = upto - mine, at = run;
  int pick = -1;
  for (int k = k0; k < k1; ++k) {
    const double v = x(k);
    if (v > kNothing) {
      pick = k;
      at = run;
      if (run + v > want) break;
    }
    run += v;
  }
  before = __shfl(at, l, kWave);
  return __shfl(pick, l, kWave);
}

// Grid batch, one wave: the segment in which the running sum passes, then the
// token in it.
template <int DT, int DDT, bool VEC>
__global__ void __launch_bounds__(kWave) verify_token_kernel(VerifyKArgs a) {
  const int b = blockIdx.x, lane = threadIdx.x;
  Decision d = a.decide[b];
  if (d.token >= 0) return;
  const Draw r = draw_of(d, exponent(a, b));
  double* parts = a.parts + (size_t)b * a.segs;
  auto sum_parts = [&]() {
    double x = 0.0;
    for (int k = lane; k < a.segs; k += kWave) x += parts[k];
    return wave_sum(x);
  };
  double total = sum_parts();
  if (!(total > kNothing) && (d.draft >= 0 || d.not_tok >= 0)) {
    // p <= q everywhere (only by rounding, or when all of p is on the draft):
    // the draw is from p
    d.draft = d.not_tok = -1;
    for (int k = 0; k < a.segs; ++k) {
      double w[kN], x = 0.0;
      weigh8<DT, DDT, VEC>(a, d, r, k * kSeg + lane * kN, w);
      for (int e = 0; e < kN; ++e) x += w[e];
      x = wave_sum(x);
      if (lane == 0) parts[k] = x;
    }
    __threadfence_block();
    __syncthreads();
    total = sum_parts();
  }
  const double want = (double)a.u_last[b] * total;
  double before = 0.0;
  const int seg = first_past(a.segs, want, before, [&](int k) { return parts[k]; });
  if (seg < 0) return;  // (token 0 is there)
  double w[kN], x = 0.0;
  weigh8<DT, DDT, VEC>(a, d, r, seg * kSeg + lane * kN, w);
#pragma unroll
  for (int e = 0; e < kN; ++e) x += w[e];
  const int l = first_past(kWave, want, before, [&](int) { return x; });
  if (lane != l) return;
  int pick = 0;
#pragma unroll
  for (int e = 0; e < kN; ++e)
    if (w[e] > kNothing) pick = e;
  bool done = false;
#pragma unroll
  for (int e = 0; e < kN; ++e) {
    before += w[e];
    if (!done && w[e] > kNothing && before > want) {
      pick = e;
      done = true;
    }
  }
  a.out[d.at] = seg * kSeg + lane * kN + pick;
}

template <int DT, int DDT>
hipError_t launch_dt(const VerifyKArgs& a, bool vec, int rows, hipStream_t s) {
  const unsigned g1 = (unsigned)rows * a.g1, g2 = (unsigned)a.batch * a.g2;
  if (vec) {
    verify_stat_kernel<DT, DDT, true><<<g1, kVT, 0, s>>>(a);
    verify_weight_kernel<DT, DDT, true><<<g2, kVT, 0, s>>>(a);
    if (a.temps) verify_token_kernel<DT, DDT, true><<<a.batch, kWave, 0, s>>>(a);
  } else {
    verify_stat_kernel<DT, DDT, false><<<g1, kVT, 0, s>>>(a);
    verify_weight_kernel<DT, DDT, false><<<g2, kVT, 0, s>>>(a);
    if (a.temps) verify_token_kernel<DT, DDT, false><<<a.batch, kWave, 0, s>>>(a);
  }
  return hipGetLastError();
}

template <int DT>
hipError_t launch_ddt(int ddt, const VerifyKArgs& a, bool vec, int rows, hipStream_t s) {
  switch (ddt) {
    case PKV_F32: return launch_dt<DT, PKV_F32>(a, vec, rows, s);
    case PKV_F16: return launch_dt<DT, PKV_F16>(a, vec, rows, s);
    default: return launch_dt<DT, PKV_BF16>(a, vec, rows, s);
  }
}

struct VerifyPlan {
  int rows, g1, len1, g2, segs;
  size_t parts, decide, bytes;
};

// Rows are cut into as many chunks as give about 4096 workgroups, of 4096
// elements or more, a multiple of 8 long; the last rows into as many workgroups,
// a segment or more for each wave.
VerifyPlan verify_plan(const VerifyArgs& a) {
  VerifyPlan p{};
  p.rows = a.total_drafts + a.batch + (a.has_draft ? a.total_drafts : 0);
  const int g = std::max(1, std::min(4096 / p.rows, a.vocab / 4096));
  p.len1 = ((a.vocab + g - 1) / g + 7) / 8 * 8;
  p.g1 = (a.vocab + p.len1 - 1) / p.len1;
  p.segs = (a.vocab + kSeg - 1) / kSeg;
  p.g2 = std::max(1, std::min(1024 / a.batch, (p.segs + kVW - 1) / kVW));
  auto up = [](size_t x) { return (x + 255) / 256 * 256; };
  p.parts = up((size_t)p.rows * p.g1 * sizeof(RowPart));
  p.decide = p.parts + up((size_t)a.batch * p.segs * sizeof(double));
  p.bytes = p.decide + up((size_t)a.batch * sizeof(Decision));
  return p;
}

}  // namespace

size_t verify_workspace_bytes(const VerifyArgs& a) { return verify_plan(a).bytes; }

bool verify_fits(const VerifyArgs& a) {
  const VerifyPlan p = verify_plan(a);
  return grid_fits((long long)p.rows * p.g1, kVT) && grid_fits((long long)a.batch * p.g2, kVT);
}

hipError_t launch_verify(const VerifyArgs& a, char* ws, hipStream_t stream) {
  const VerifyPlan pl = verify_plan(a);
  VerifyKArgs k{};
  k.target = static_cast<const char*>(a.target_logits);
  k.draft = static_cast<const char*>(a.draft_logits);
  k.t_stride = a.target_stride;
  k.d_stride = a.draft_stride;
  k.draft_dt = a.target_dtype << 8 | a.draft_dtype;
  k.tokens = a.draft_tokens;
  k.cu = a.cu_drafts;
  k.u = a.uniforms;
  k.u_last = a.final_uniforms;
  k.temps = a.temperatures;
  k.batch = a.batch;
  k.total = a.total_drafts;
  k.vocab = a.vocab;
  k.g1 = pl.g1;
  k.len1 = pl.len1;
  k.g2 = pl.g2;
  k.segs = pl.segs;
  k.rows = reinterpret_cast<RowPart*>(ws);
  k.parts = reinterpret_cast<double*>(ws + pl.parts);
  k.decide = reinterpret_cast<Decision*>(ws + pl.decide);
  k.out = a.out_tokens;
  k.accepted = a.n_accepted;
  // 16-byte loads where every row starts on 16 bytes
  auto al = [](const void* p, long long stride, int dt) {
    return ((reinterpret_cast<uintptr_t>(p) | (uintptr_t)(stride * (long long)dtype_bytes(dt))) & 15) == 0;
  };
  const bool vec = al(k.target, k.t_stride, a.target_dtype) &&
                   (!k.draft || al(k.draft, k.d_stride, a.draft_dtype));
  const int ddt = k.draft ? a.draft_dtype : a.target_dtype;
  switch (a.target_dtype) {
    case PKV_F32: return launch_ddt<PKV_F32>(ddt, k, vec, pl.rows, stream);
    case PKV_F16: return launch_ddt<PKV_F16>(ddt, k, vec, pl.rows, stream);
    default: return launch_ddt<PKV_BF16>(ddt, k, vec, pl.rows, stream);
  }
}

}  // namespace pkv
