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

constexpr int kLogitThreads = 256;
constexpr int kSlice = 4096;  // tokens of a workgroup

constexpr uint32_t kSeen = 1u << 31;  // among the request's tokens; below: times generated

// Entries [lo, hi) of request b in an array of `total` (at most kMaxLen, so that the
// strides of a loop over them stay in 32 bits).
__device__ __forceinline__ void range_of(const int32_t* cu, int total, int b, int& lo, int& hi) {
  lo = min(max(cu[b], 0), total);
  hi = min(max(cu[b + 1], 0), total);
}

template <int DT>
__device__ __forceinline__ float load1(const void* p, size_t i) {
  if constexpr (DT == PKV_F32) return static_cast<const float*>(p)[i];
  else if constexpr (DT == PKV_F16) return (float)static_cast<const _Float16*>(p)[i];
  else return bf16lo(static_cast<const uint16_t*>(p)[i]);
}
template <int DT>
__device__ __forceinline__ void store1(void* p, size_t i, float x) {
  if constexpr (DT == PKV_F32) static_cast<float*>(p)[i] = x;
  else if constexpr (DT == PKV_F16) static_cast<_Float16*>(p)[i] = (_Float16)x;
  else static_cast<uint16_t*>(p)[i] = (uint16_t)f32_to_bf16_bits(x);
}

template <int DT>
__global__ void __launch_bounds__(kLogitThreads) logits_kernel(LogitsArgs a, int slices) {
#pragma clang fp contract(off)  // each operation is rounded
  __shared__ uint32_t count[kSlice];
  __shared__ int bias_at[kSlice];  // 1 + the last entry of the token, 0: none
  const int b = blockIdx.x / slices, t0 = (blockIdx.x % slices) * kSlice;
  const int n = min(kSlice, a.vocab - t0);
  for (int i = threadIdx.x; i < n; i += kLogitThreads) {
    count[i] = 0;
    bias_at[i] = 0;
  }
  __syncthreads();
  int lo = 0, hi = 0;
  if (a.cu_tokens) {
    range_of(a.cu_tokens, a.total_tokens, b, lo, hi);
    const long long first_new = (long long)a.cu_tokens[b] + (a.prompt_lens ? a.prompt_lens[b] : 0);
    for (int i = lo + threadIdx.x; i < hi; i += kLogitThreads) {
      const int t = a.tokens[i] - t0;
      if ((unsigned)t < (unsigned)n) {
        atomicOr(&count[t], kSeen);
        if (i >= first_new) atomicAdd(&count[t], 1u);
      }
    }
  }
  if (a.cu_bias) {
    range_of(a.cu_bias, a.total_bias, b, lo, hi);
    for (int i = lo + threadIdx.x; i < hi; i += kLogitThreads) {
      const int t = a.bias_tokens[i] - t0;
      if ((unsigned)t < (unsigned)n) atomicMax(&bias_at[t], i + 1);
    }
  }
  __syncthreads();
  float r = a.repetition ? a.repetition[b] : 1.0f;
  if (!(r > 0.0f && r < INFINITY)) r = 1.0f;
  const float pres = a.presence ? a.presence[b] : 0.0f;
  const float freq = a.frequency ? a.frequency[b] : 0.0f;
  const int row = !a.mask ? -1 : a.mask_rows ? a.mask_rows[b] : b;
  const uint32_t* mask = row < 0 || row >= a.n_masks ? nullptr
                                                     : a.mask + (size_t)row * a.mask_row_words;
  const bool none = a.mask && row >= a.n_masks;
  for (int i = threadIdx.x; i < n; i += kLogitThreads) {
    const int t = t0 + i;
    float x = load1<DT>(a.logits, (size_t)b * a.row_stride + t);
    const uint32_t c = count[i];
    if (c & kSeen) x = x > 0.0f ? __fdiv_rn(x, r) : x * r;
    if (c & ~kSeen) {
      const float f = freq * (float)(c & ~kSeen);
      x = x - f;
      x = x - pres;
    }
    if (bias_at[i]) x = x + a.bias_values[bias_at[i] - 1];
    if (none || (mask && !((mask[t >> 5] >> (t & 31)) & 1))) x = -INFINITY;
    store1<DT>(a.out, (size_t)b * a.out_row_stride + t, x);
  }
}

int slices_of(const LogitsArgs& a) { return (a.vocab + kSlice - 1) / kSlice; }

}  // namespace

bool logits_fits(const LogitsArgs& a) {
  return grid_fits((long long)a.batch * slices_of(a), kLogitThreads);
}

hipError_t launch_logits(const LogitsArgs& a, hipStream_t stream) {
  const int slices = slices_of(a);
  const unsigned blocks = (unsigned)((long long)a.batch * slices);
  if (a.dtype == PKV_F32) logits_kernel<PKV_F32><<<blocks, kLogitThreads, 0, stream>>>(a, slices);
  else if (a.dtype == PKV_F16) logits_kernel<PKV_F16><<<blocks, kLogitThreads, 0, stream>>>(a, slices);
  else logits_kernel<PKV_BF16><<<blocks, kLogitThreads, 0, stream>>>(a, slices);
  return hipGetLastError();
}

}  // namespace pkv
