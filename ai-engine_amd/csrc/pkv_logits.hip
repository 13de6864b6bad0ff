// pkv_logits.hip -- penalties, biases and masks on logits before a token is chosen
// (gfx950).
//
// A workgroup has a slice of one request's row.  It first counts the request's tokens
// that fall into the slice in LDS (integers, so in any order), and finds the last
// bias entry of each token there; then every logit of the slice is read, changed
// and written once.
#include "pkv_device.h"
#include "pkv_internal.h"

namespace pkv {
namespace {

constexpr int kLogitThreads = 512;
constexpr int kAtOnce = 4;  // of the request's tokens a thread reads at once

constexpr uint32_t kSeen = 1u << 31;  // among the request's tokens; below: times generated

// Entries [lo, hi) of request b in an array of `total` (at most kMaxLen, so that the
// strides of a loop over them stay in 32 bits).
__device__ __forceinline__ void range_of(const int32_t* cu, int total, int b, int& lo, int& hi) {
  lo = min(max(cu[b], 0), total);
  hi = min(max(cu[b + 1], 0), total);
}

// Sixteen bytes of logits; rows start at any element.
typedef uint32_t u32x4_at2 __attribute__((ext_vector_type(4), aligned(2)));
template <int DT>
struct Vec {
  static constexpr int E = DT == PKV_F32 ? 4 : 2, N = 16 / E;
};
// Elements at .. of the row at p, which has n.
template <int DT>
__device__ __forceinline__ u32x4 load_logits(const char* p, int at, int n) {
  using V = Vec<DT>;
  p += (size_t)at * V::E;
  if (at + V::N <= n) return *reinterpret_cast<const u32x4_at2*>(p);
  u32x4 w = {0, 0, 0, 0};
#pragma unroll
  for (int e = 0; e < V::N; ++e) {
    if (at + e >= n) break;
    if constexpr (DT == PKV_F32) w[e] = reinterpret_cast<const uint32_t*>(p)[e];
    else w[e / 2] |= (uint32_t)reinterpret_cast<const uint16_t*>(p)[e] << (16 * (e % 2));
  }
  return w;
}
template <int DT>
__device__ __forceinline__ void store_logits(char* p, int at, int n, u32x4 w) {
  using V = Vec<DT>;
  p += (size_t)at * V::E;
  if (at + V::N <= n) {
    *reinterpret_cast<u32x4_at2*>(p) = w;
    return;
  }
#pragma unroll
  for (int e = 0; e < V::N; ++e) {
    if (at + e >= n) break;
    if constexpr (DT == PKV_F32) reinterpret_cast<uint32_t*>(p)[e] = w[e];
    else reinterpret_cast<uint16_t*>(p)[e] = (uint16_t)(w[e / 2] >> (16 * (e % 2)));
  }
}

// NV: sixteen bytes of logits a thread.  A slice's counts (and last bias entries) are
// in planes of four tokens of each of its threads' sixteen bytes, so that lanes read
// neighbouring 16 bytes of LDS.
template <int DT, int NV>
__global__ void __launch_bounds__(kLogitThreads) logits_kernel(LogitsArgs a, int slices) {
#pragma clang fp contract(off)  // each operation is rounded
  using V = Vec<DT>;
  constexpr int N = V::N, P = N / 4, S = kLogitThreads * N * NV, PLANE = S / P;
  __shared__ __attribute__((aligned(16))) uint32_t count[S];
  __shared__ __attribute__((aligned(16))) int bias_at[S];  // 1 + the token's last entry, 0: none
  auto place = [](int t) { return P == 1 ? t : (t / 8) * 4 + t % 4 + (t / 4 % 2) * PLANE; };
  const int b = blockIdx.x / slices, t0 = (blockIdx.x % slices) * S;
  const int n = min(S, a.vocab - t0), tid = threadIdx.x;

  // everything that can be read at once: logits, masks, ranges and the first tokens
  const char* in = static_cast<const char*>(a.logits) + ((size_t)b * a.row_stride + t0) * V::E;
  const int row = !a.mask ? -1 : a.mask_rows ? a.mask_rows[b] : b;
  const bool none = a.mask && row >= a.n_masks, masked = row >= 0 && !none;
  u32x4 w[NV];
  uint32_t allow[NV];
#pragma unroll
  for (int v = 0; v < NV; ++v) {
    const int at = (v * kLogitThreads + tid) * N;
    allow[v] = none ? 0u : ~0u;
    if (at >= n) continue;
    w[v] = load_logits<DT>(in, at, n);
    if (masked)
      allow[v] = a.mask[(size_t)row * a.mask_row_words + ((t0 + at) >> 5)] >> ((t0 + at) & 31);
  }
  int lo = 0, hi = 0, blo = 0, bhi = 0;
  long long first_new = 0;
  if (a.cu_tokens) {
    range_of(a.cu_tokens, a.total_tokens, b, lo, hi);
    first_new = (long long)a.cu_tokens[b] + (a.prompt_lens ? a.prompt_lens[b] : 0);
  }
  if (a.cu_bias) range_of(a.cu_bias, a.total_bias, b, blo, bhi);
  int tk[kAtOnce];
  auto tokens_at = [&](int from) {
#pragma unroll
    for (int e = 0; e < kAtOnce; ++e) {
      const int i = from + e * kLogitThreads + tid;
      tk[e] = i < hi ? a.tokens[i] : -1;
    }
  };
  if (lo < hi) tokens_at(lo);

  const u32x4 zero = {0, 0, 0, 0};
  if (lo < hi)
    for (int i = tid * 4; i < S; i += kLogitThreads * 4) *reinterpret_cast<u32x4*>(&count[i]) = zero;
  if (blo < bhi)
    for (int i = tid * 4; i < S; i += kLogitThreads * 4)
      *reinterpret_cast<u32x4*>(&bias_at[i]) = zero;
  __syncthreads();
  for (int from = lo; from < hi; from += kAtOnce * kLogitThreads) {
#pragma unroll
    for (int e = 0; e < kAtOnce; ++e) {
      const uint32_t t = (uint32_t)tk[e] - (uint32_t)t0;
      if (tk[e] < 0 || t >= (uint32_t)n) continue;
      if (from + e * kLogitThreads + tid >= first_new) atomicAdd(&count[place(t)], 1u);
      else atomicOr(&count[place(t)], kSeen);
    }
    tokens_at(from + kAtOnce * kLogitThreads);
  }
  for (int i = blo + tid; i < bhi; i += kLogitThreads) {
    const uint32_t t = (uint32_t)a.bias_tokens[i] - (uint32_t)t0;
    if (t < (uint32_t)n) atomicMax(&bias_at[place(t)], i + 1);
  }
  __syncthreads();

  float r = a.repetition ? a.repetition[b] : 1.0f;
  if (!(r > 0.0f && r < INFINITY)) r = 1.0f;
  const float pres = a.presence ? a.presence[b] : 0.0f;
  const float freq = a.frequency ? a.frequency[b] : 0.0f;
  char* out = static_cast<char*>(a.out) + ((size_t)b * a.out_row_stride + t0) * V::E;
#pragma unroll
  for (int v = 0; v < NV; ++v) {
    const int at = (v * kLogitThreads + tid) * N;
    if (at >= n) continue;
    uint32_t c[N] = {}, bi[N] = {}, any = 0;
#pragma unroll
    for (int p = 0; p < P; ++p) {
      const int from = p * PLANE + (v * kLogitThreads + tid) * 4;
      const u32x4 x = lo < hi ? *reinterpret_cast<const u32x4*>(&count[from]) : zero;
      const u32x4 y = blo < bhi ? *reinterpret_cast<const u32x4*>(&bias_at[from]) : zero;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        c[4 * p + e] = x[e];
        bi[4 * p + e] = y[e];
        any |= x[e] | y[e];
      }
    }
    if (any) {
      float x[N];
      widen16<DT>(w[v], x);
#pragma unroll
      for (int e = 0; e < N; ++e) {
        if (!(c[e] | bi[e])) continue;
        if (c[e]) x[e] = x[e] > 0.0f ? __fdiv_rn(x[e], r) : x[e] * r;
        if (c[e] & ~kSeen) {
          const float f = freq * (float)(c[e] & ~kSeen);
          x[e] = x[e] - f;
          x[e] = x[e] - pres;
        }
        if (bi[e]) x[e] = x[e] + a.bias_values[bi[e] - 1];
        if constexpr (DT == PKV_F32) {
          w[v][e] = __float_as_uint(x[e]);
        } else {
          const uint32_t h = cvt_pk16<DT>(x[e], 0.0f) & 0xffffu;
          w[v][e / 2] = e % 2 ? (w[v][e / 2] & 0xffffu) | h << 16 : (w[v][e / 2] & 0xffff0000u) | h;
        }
      }
    }
    // -infinity where the bit is clear
#pragma unroll
    for (int e = 0; e < N; ++e) {
      const bool no = !(allow[v] >> e & 1);
      if constexpr (DT == PKV_F32) {
        if (no) w[v][e] = 0xff800000u;
      } else {
        constexpr uint32_t inf = DT == PKV_F16 ? 0xfc00u : 0xff80u;
        if (no)
          w[v][e / 2] = e % 2 ? (w[v][e / 2] & 0xffffu) | inf << 16
                              : (w[v][e / 2] & 0xffff0000u) | inf;
      }
    }
    store_logits<DT>(out, at, n, w[v]);
  }
}

constexpr int kNV = 2;
int slices_of(const LogitsArgs& a) {
  const int s = kLogitThreads * (a.dtype == PKV_F32 ? 4 : 8) * kNV;
  return (a.vocab + s - 1) / s;
}

}  // namespace

bool logits_fits(const LogitsArgs& a) {
  return grid_fits((long long)a.batch * slices_of(a), kLogitThreads);
}

hipError_t launch_logits(const LogitsArgs& a, hipStream_t stream) {
  const int slices = slices_of(a);
  const unsigned blocks = (unsigned)((long long)a.batch * slices);
  if (a.dtype == PKV_F32) logits_kernel<PKV_F32, kNV><<<blocks, kLogitThreads, 0, stream>>>(a, slices);
  else if (a.dtype == PKV_F16) logits_kernel<PKV_F16, kNV><<<blocks, kLogitThreads, 0, stream>>>(a, slices);
  else logits_kernel<PKV_BF16, kNV><<<blocks, kLogitThreads, 0, stream>>>(a, slices);
  return hipGetLastError();
}

}  // namespace pkv
