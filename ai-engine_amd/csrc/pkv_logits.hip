// pkv_logits.hip -- penalties, biases and masks on logits before a token is chosen
// (gfx950).
//
// A workgroup has a slice of one request's row: two or one 16 bytes of logits a thread,
// 16,384 or 8192 tokens of 16 bits (with biases the tables in LDS are two).  It counts the
// request's tokens that fall into the slice (integers, so in any order), marks the ones
// seen by a bit, and finds the last bias entry of each token; a thread then computes the
// logits of its own that have a bit one after another, and writes all of them once.
//
// Bound by the histories: each slice goes through the whole of its request's.  128 rows of
// 128,256 bf16 logits with histories up to 8000 take 27 us, 13.4 (the copy rate) without
// any; some 60 % of the cycles are vector instructions, the rest the waits of four rounds
// of workgroups.  With slices of 4096 and every logit computed in place, so that a wave of 512
// went through the division for a few of them, they took 34; a list of the changed
// tokens made by a shared counter, 42.
#include "pkv_device.h"
#include "pkv_internal.h"

namespace pkv {
namespace {

constexpr int kLogitThreads = 1024;
constexpr int kAtOnce = 4;  // of the request's tokens a thread reads at once

// Entries [lo, hi) of a request in an array of `total` (at most kMaxLen, so that the
// strides of a loop over them stay in 32 bits).
__device__ __forceinline__ void range_of(const int32_t* cu, int total, int& lo, int& hi) {
  lo = min(max(cu[0], 0), total);
  hi = min(max(cu[1], 0), total);
}

// What arrays that are not given stand for: read in place of them, so that a workgroup
// waits once for all of a request's numbers.
__device__ const int32_t kNoInts[2] = {0, 0};
__device__ const float kNoFloats[2] = {0.0f, 1.0f};

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

// The elements of w whose bit is set become those of x.
template <int DT>
__device__ __forceinline__ void set_logits(u32x4& w, uint32_t bits, u32x4 x) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    uint32_t m;
    if constexpr (DT == PKV_F32) {
      m = __builtin_amdgcn_sbfe(bits, i, 1);
    } else {
      const uint32_t lo = __builtin_amdgcn_sbfe(bits, 2 * i, 1);
      const uint32_t hi = __builtin_amdgcn_sbfe(bits, 2 * i + 1, 1);
      m = (lo & 0xffffu) | (hi & ~0xffffu);
    }
    w[i] = (x[i] & m) | (w[i] & ~m);
  }
}
// Element e.
template <int DT>
__device__ __forceinline__ float logit_at(u32x4 w, int e) {
  const int i = DT == PKV_F32 ? e : e / 2;
  const uint32_t lo = i & 1 ? w[1] : w[0], hi = i & 1 ? w[3] : w[2], x = i & 2 ? hi : lo;
  if constexpr (DT == PKV_F32) return __uint_as_float(x);
  else if constexpr (DT == PKV_F16) return e & 1 ? f16hi(x) : f16lo(x);
  else return e & 1 ? bf16hi(x) : bf16lo(x);
}

// A thread has NV pieces of 16 bytes.  The tables of a slice have a word for each token,
// in planes of four tokens of every piece, so that lanes read neighbouring 16 bytes.
template <int DT, bool BIAS>
struct Slice {
  static constexpr int N = Vec<DT>::N, NV = BIAS ? 1 : 2, S = kLogitThreads * N * NV;
};

template <int DT, bool BIAS>
__global__ void __launch_bounds__(kLogitThreads) logits_kernel(LogitsArgs a) {
#pragma clang fp contract(off)  // each operation is rounded
  using V = Vec<DT>;
  using SL = Slice<DT, BIAS>;
  constexpr int N = V::N, NV = SL::NV, P = N / 4, S = SL::S, PLANE = S / P, T = kLogitThreads;
  __shared__ __attribute__((aligned(16))) uint32_t count[S];  // then: the new logit's bits
  __shared__ __attribute__((aligned(16))) int bias_at[BIAS ? S : 1];  // 1 + the last entry
  __shared__ uint32_t seen[S / 32], biased[BIAS ? S / 32 : 1];
  // slices of small token ids first: they tend to be the ones with most of a text
  const int b = blockIdx.x % a.batch, t0 = blockIdx.x / a.batch * S;
  const int n = min(S, a.vocab - t0), tid = threadIdx.x;
  auto place = [](uint32_t t) { return t / N * 4 + t % 4 + (P == 2 ? (t / 4 % 2) * PLANE : 0); };

  const char* in = static_cast<const char*>(a.logits) + ((size_t)b * a.row_stride + t0) * V::E;
  u32x4 w[NV];
#pragma unroll
  for (int v = 0; v < NV; ++v) {
    const int at = (v * T + tid) * N;
    if (at < n) w[v] = load_logits<DT>(in, at, n);
  }
  int lo, hi, blo = 0, bhi = 0;
  const int32_t* cu = a.cu_tokens ? a.cu_tokens + b : kNoInts;
  const int prompt = *(a.prompt_lens ? a.prompt_lens + b : kNoInts);
  const int mask_row = *(a.mask_rows ? a.mask_rows + b : kNoInts);
  float r = *(a.repetition ? a.repetition + b : kNoFloats + 1);
  const float pres = *(a.presence ? a.presence + b : kNoFloats);
  const float freq = *(a.frequency ? a.frequency + b : kNoFloats);
  const long long first_new = (long long)cu[0] + prompt;
  range_of(cu, a.total_tokens, lo, hi);
  if constexpr (BIAS) range_of(a.cu_bias + b, a.total_bias, blo, bhi);
  if (!(r > 0.0f && r < INFINITY)) r = 1.0f;
  const int mid = (int)max((long long)lo, min((long long)hi, first_new));
  const int row = !a.mask ? -1 : a.mask_rows ? mask_row : b;
  const bool none = a.mask && row >= a.n_masks, masked = row >= 0 && !none;
  uint32_t allow[NV];
#pragma unroll
  for (int v = 0; v < NV; ++v) {
    const int at = (v * T + tid) * N;
    allow[v] = none ? 0u : ~0u;
    if (masked && at < n)
      allow[v] = a.mask[(size_t)row * a.mask_row_words + ((t0 + at) >> 5)] >> ((t0 + at) & 31);
  }
  const bool work = lo < hi || blo < bhi;
  if (work) {
    int tk[kAtOnce], bias_token = -1;
    auto tokens_from = [&](int from, int (&to)[kAtOnce]) {
      const int32_t* tokens = a.tokens + from;
      const int left = hi - from;
      if (left >= kAtOnce * T) {
#pragma unroll
        for (int e = 0; e < kAtOnce; ++e) to[e] = (tokens + e * T)[tid];
      } else {
#pragma unroll
        for (int e = 0; e < kAtOnce; ++e) {
          to[e] = -1;
          if (e * T + tid < left) to[e] = (tokens + e * T)[tid];
        }
      }
    };
    tokens_from(lo, tk);
    if constexpr (BIAS) {
      if (blo + tid < bhi) bias_token = a.bias_tokens[blo + tid];
    }
    const u32x4 zero = {0, 0, 0, 0};
#pragma unroll
    for (int i = tid * 4; i < S; i += T * 4) {
      *reinterpret_cast<u32x4*>(&count[i]) = zero;
      if constexpr (BIAS) *reinterpret_cast<u32x4*>(&bias_at[i]) = zero;
    }
    if (tid < S / 32) {
      seen[tid] = 0;
      if constexpr (BIAS) biased[tid] = 0;
    }
    __syncthreads();
    for (int from = lo; from < hi; from += kAtOnce * T) {
      int next[kAtOnce];
      tokens_from(min(from + kAtOnce * T, hi), next);
#pragma unroll
      for (int e = 0; e < kAtOnce; ++e) {
        const uint32_t t = (uint32_t)tk[e] - (uint32_t)t0;  // (t0 < 2^24: large if tk < 0)
        if (t < (uint32_t)n) {
          atomicOr(&seen[t >> 5], 1u << (t & 31));
          if (from + e * T + tid >= mid) atomicAdd(&count[place(t)], 1u);
        }
        tk[e] = next[e];
      }
    }
    if constexpr (BIAS) {
      for (int i = blo + tid; i < bhi; i += T) {
        const uint32_t t = (uint32_t)bias_token - (uint32_t)t0;
        if (t < (uint32_t)n) {
          atomicMax(&bias_at[place(t)], i + 1);
          atomicOr(&biased[t >> 5], 1u << (t & 31));
        }
        if (i + T < bhi) bias_token = a.bias_tokens[i + T];
      }
    }
    __syncthreads();
  }
  char* out = static_cast<char*>(a.out) + ((size_t)b * a.out_row_stride + t0) * V::E;
#pragma unroll
  for (int v = 0; v < NV; ++v) {
    const int at = (v * T + tid) * N;
    if (at >= n) continue;
    if (work) {
      constexpr uint32_t ALL = (1u << N) - 1;
      const uint32_t sb = seen[at >> 5] >> (at & 31) & ALL;
      const uint32_t bb = BIAS ? biased[at >> 5] >> (at & 31) & ALL : 0u;
      const uint32_t changed = sb | bb;
      for (uint32_t left = changed; left; left &= left - 1) {
        const int e = __builtin_ctz(left), where = place(at + e);
        float x = logit_at<DT>(w[v], e);
        if (sb >> e & 1) {
          x = x > 0.0f ? __fdiv_rn(x, r) : x * r;
          if (const uint32_t c = count[where]) {
            const float f = freq * (float)c;
            x = x - f;
            x = x - pres;
          }
        }
        if constexpr (BIAS) {
          if (bb >> e & 1) x = x + a.bias_values[bias_at[where] - 1];
        }
        if constexpr (DT == PKV_F32) count[where] = __float_as_uint(x);
        else count[where] = cvt_pk16<DT>(x, 0.0f) & 0xffffu;
      }
      if (changed) {
        u32x4 x[P];
#pragma unroll
        for (int p = 0; p < P; ++p)
          x[p] = *reinterpret_cast<const u32x4*>(&count[p * PLANE + (v * T + tid) * 4]);
        if constexpr (P == 2)
          x[0] = u32x4{x[0][0] | x[0][1] << 16, x[0][2] | x[0][3] << 16, x[1][0] | x[1][1] << 16,
                       x[1][2] | x[1][3] << 16};
        set_logits<DT>(w[v], changed, x[0]);
      }
    }
    if (a.mask) {
      constexpr uint32_t inf = DT == PKV_F32 ? 0xff800000u : DT == PKV_F16 ? 0xfc00fc00u : 0xff80ff80u;
      set_logits<DT>(w[v], ~allow[v], u32x4{inf, inf, inf, inf});
    }
    store_logits<DT>(out, at, n, w[v]);
  }
}

long long logit_blocks(const LogitsArgs& a) {
  const int s = a.dtype == PKV_F32 ? (a.cu_bias ? Slice<PKV_F32, true>::S : Slice<PKV_F32, false>::S)
                                   : (a.cu_bias ? Slice<PKV_F16, true>::S : Slice<PKV_F16, false>::S);
  return (long long)a.batch * ((a.vocab + s - 1) / s);
}

template <int DT>
void adjust(const LogitsArgs& a, hipStream_t stream) {
  const unsigned blocks = (unsigned)logit_blocks(a);
  if (a.cu_bias) logits_kernel<DT, true><<<blocks, kLogitThreads, 0, stream>>>(a);
  else logits_kernel<DT, false><<<blocks, kLogitThreads, 0, stream>>>(a);
}

}  // namespace

bool logits_fits(const LogitsArgs& a) {
  return grid_fits(logit_blocks(a), kLogitThreads);
}

hipError_t launch_logits(const LogitsArgs& a, hipStream_t stream) {
  if (a.dtype == PKV_F32) adjust<PKV_F32>(a, stream);
  else if (a.dtype == PKV_F16) adjust<PKV_F16>(a, stream);
  else adjust<PKV_BF16>(a, stream);
  return hipGetLastError();
}

}  // namespace pkv
