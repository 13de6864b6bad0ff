// pkv_prompt.hip -- causal attention of whole prompts over their own rows, packed
// (gfx950): out_i = sum_{j <= i} softmax_j(scale q_i . k_j) v_j.
//
// One wave per (token, query head): a lane scores one key of 64, the weights go
// through LDS, and a lane then sums the values of its channels, with a running
// maximum and sum.
#include <algorithm>

#include "pkv_device.h"
#include "pkv_internal.h"

namespace pkv {
namespace {

template <int DT>
__device__ __forceinline__ float elem(const char* p, size_t i) {
  if constexpr (DT == PKV_F32) return reinterpret_cast<const float*>(p)[i];
  else if constexpr (DT == PKV_F16) return (float)reinterpret_cast<const _Float16*>(p)[i];
  else return bf16lo(reinterpret_cast<const uint16_t*>(p)[i]);
}
__device__ __forceinline__ void put(void* out, int dt, size_t i, float x) {
  if (dt == PKV_F32) static_cast<float*>(out)[i] = x;
  else if (dt == PKV_F16) static_cast<_Float16*>(out)[i] = (_Float16)x;
  else static_cast<uint16_t*>(out)[i] = (uint16_t)f32_to_bf16_bits(x);
}
__device__ __forceinline__ float wave_max(float x) {
  return row_group_max(row_max16(x));
}
__device__ __forceinline__ float wave_add(float x) {
  return swap32_sum(swap16_sum(row_sum16(x)));
}

template <int DT, int HD>
__global__ void __launch_bounds__(64) prompt_kernel(PromptArgs a, int rows_grid) {
  constexpr int PER = HD / 64;
  __shared__ float q[HD];
  __shared__ float p[64];
  const int lane = threadIdx.x;
  const int h = blockIdx.x % a.n_head;
  const long long u = blockIdx.x / a.n_head;
  const int s = (int)(u / rows_grid);
  const int lo = a.cu_lens[s], hi = a.cu_lens[s + 1];
  if (lo < 0 || hi > a.total) return;
  const int g = h / (a.n_head / a.n_kv_head);
  const char *Q = static_cast<const char*>(a.q), *K = static_cast<const char*>(a.k),
             *V = static_cast<const char*>(a.v);
  for (long long row = lo + u % rows_grid; row < hi; row += rows_grid) {
    __syncthreads();
    for (int j = 0; j < PER; ++j) {
      const int d = lane + 64 * j;
      q[d] = elem<DT>(Q, (size_t)row * a.q_stride + (size_t)h * HD + d) * a.scale * 1.44269504f;
    }
    __syncthreads();
    float m = -INFINITY, l = 0.0f, o[PER] = {};
    for (long long k0 = lo; k0 <= row; k0 += 64) {
      float x = -INFINITY;
      if (k0 + lane <= row) {
        x = 0.0f;
        const size_t at = (size_t)(k0 + lane) * a.k_stride + (size_t)g * HD;
        for (int d = 0; d < HD; ++d) x = fmaf(q[d], elem<DT>(K, at + d), x);
      }
      const float mn = fmaxf(m, wave_max(x));
      const float w = fast_exp2(x - mn), c = fast_exp2(m - mn);
      l = l * c + wave_add(w);
      m = mn;
      p[lane] = w;
      __syncthreads();
      for (int j = 0; j < PER; ++j) o[j] *= c;
      const int n = (int)min(64LL, row + 1 - k0);
      for (int i = 0; i < n; ++i) {
        const size_t at = (size_t)(k0 + i) * a.v_stride + (size_t)g * HD + lane;
        for (int j = 0; j < PER; ++j) o[j] = fmaf(p[i], elem<DT>(V, at + 64 * j), o[j]);
      }
      __syncthreads();
    }
    for (int j = 0; j < PER; ++j)
      put(a.out, a.out_dtype, ((size_t)row * a.n_head + h) * HD + lane + 64 * j, o[j] / l);
  }
}

long long prompt_blocks(const PromptArgs& a) {
  return (long long)a.n_seqs * std::min(a.max_len, a.total) * a.n_head;
}

template <int DT>
hipError_t run(const PromptArgs& a, hipStream_t stream) {
  const unsigned blocks = (unsigned)prompt_blocks(a);
  const int rows = std::min(a.max_len, a.total);
  if (a.head_dim == 64) prompt_kernel<DT, 64><<<blocks, 64, 0, stream>>>(a, rows);
  else if (a.head_dim == 128) prompt_kernel<DT, 128><<<blocks, 64, 0, stream>>>(a, rows);
  else prompt_kernel<DT, 256><<<blocks, 64, 0, stream>>>(a, rows);
  return hipGetLastError();
}

}  // namespace

bool prompt_fits(const PromptArgs& a) { return grid_fits(prompt_blocks(a), 64); }

hipError_t launch_prompt(const PromptArgs& a, hipStream_t stream) {
  if (a.dtype == PKV_F32) return run<PKV_F32>(a, stream);
  if (a.dtype == PKV_F16) return run<PKV_F16>(a, stream);
  return run<PKV_BF16>(a, stream);
}

}  // namespace pkv
