// pkv_step.hip -- block tables, slots and positions of a step, from request
// lengths that stay on the device (gfx950).
//
// The host allocator (block_table.cpp) serves a step whose lengths the host
// knows.  After a speculative step they are the verification's counts, on the
// device; this kernel gives the next step its arrays without a round trip.
//
// Request i holds seq[i] tokens in have[i] blocks and writes new[i] more:
//   need_i = max(0, ceil((seq_i + new_i) / bs) - have_i),   P_i = sum_{k<i} need_k
//   its j-th new block is free[count - 1 - P_i - j]   (taken from the list's
//   end in request order, as BlockAllocator::ensure_capacity, block_table.rs:32-47)
//   token t of the step (request i, cu_i <= t < cu_{i+1}) is at position
//   seq_i + t - cu_i, in slot table_i[pos / bs] * bs + pos % bs.
//
// Bound by latency: a step of 256 requests under a 32k limit moves 3 MB (0.5 us
// of HBM time), a small one nothing.  So one launch, with no order between
// workgroups: each adds up the requests' counts itself (n loads out of L2),
// which takes less than a second launch would, and outputs are apart from the
// inputs that other workgroups read.  7 requests: 4.2 us, 256 under a 32k limit: 6.8.
#include <algorithm>

#include "pkv_device.h"
#include "pkv_internal.h"

namespace pkv {
namespace {

constexpr int kStepThreads = 256;

constexpr int kStepWaves = kStepThreads / kWave;
constexpr int kSums = 5;

// Sums over the workgroup, in every thread, behind one barrier.
__device__ __forceinline__ void wg_sums(long long (&x)[kSums], long long (&lds)[kSums][kStepWaves]) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1)
#pragma unroll
    for (int k = 0; k < kSums; ++k) x[k] += __shfl_xor(x[k], o, kWave);
  if ((threadIdx.x & 63) == 0)
#pragma unroll
    for (int k = 0; k < kSums; ++k) lds[k][threadIdx.x >> 6] = x[k];
  __syncthreads();
#pragma unroll
  for (int k = 0; k < kSums; ++k) {
    x[k] = 0;
#pragma unroll
    for (int w = 0; w < kStepWaves; ++w) x[k] += lds[k][w];
  }
}

__global__ void __launch_bounds__(kStepThreads) step_tables_kernel(StepArgs a) {
  __shared__ long long red[kSums][kStepWaves];
  const int me = blockIdx.x;
  const int tid = threadIdx.x;
  const int bsl = a.bs_log2, bs = 1 << bsl;
  // counts of the requests before this one and of all; a request whose
  // lengths its table cannot hold makes the step invalid
  enum { kNeedBefore, kNeed, kNewBefore, kNew, kBad };
  long long sum[kSums] = {};
  for (int i = tid; i < a.n_seqs; i += kStepThreads) {
    const long long seq = a.seq_lens[i], nw = a.new_lens[i], have = a.n_blocks[i];
    const long long upto = (seq + nw + bs - 1) >> bsl;
    if (seq < 0 || nw < 0 || have < 0 || have > a.width || upto > a.width) {
      sum[kBad] = 1;
      continue;
    }
    const long long need = upto > have ? upto - have : 0;
    sum[kNeed] += need;
    sum[kNew] += nw;
    sum[kNeedBefore] += i < me ? need : 0;
    sum[kNewBefore] += i < me ? nw : 0;
  }
  const int count = *a.free_count;
  // (a step without requests still has its buffers filled)
  const bool any = me < a.n_seqs;
  const int seq = any ? a.seq_lens[me] : 0, have_raw = any ? a.n_blocks[me] : 0;
  const int new_raw = any ? a.new_lens[me] : 0;
  wg_sums(sum, red);
  const long long need_b = sum[kNeedBefore], need_t = sum[kNeed];
  const long long new_b = sum[kNewBefore], new_t = sum[kNew];
  const bool bad = sum[kBad] || count < 0 || count > a.free_len || new_t > a.max_tokens;
  const long long lacking = need_t - count;
  const bool ok = !bad && lacking <= 0;

  const int have = min(max(have_raw, 0), a.width);
  const int nw = ok ? new_raw : 0;
  const int total = ok ? (int)new_t : 0;
  const int upto = ok ? (int)(((long long)seq + nw + bs - 1) >> bsl) : 0;
  const int blocks = max(have, upto);
  const int32_t* in = a.tables_in + (size_t)me * a.width;
  int32_t* out = a.tables_out + (size_t)me * a.width;
  // block j of the request: held, or taken from the free list's end
  const int top = count - 1 - (int)(ok ? need_b : 0) + have;
  auto block = [&](int j) { return j < have ? in[j] : a.free_list[top - j]; };

  const int first = blockIdx.y * kStepThreads + tid, stride = gridDim.y * kStepThreads;
  for (int j = first; any && j < a.width; j += stride) out[j] = j < blocks ? block(j) : 0;
  const int cu = ok ? (int)new_b : 0;
  for (int t = first; t < nw; t += stride) {
    const int pos = seq + t;
    const int id = block(pos >> bsl);
    a.positions[cu + t] = pos;
    a.slots[cu + t] = id >= 0 && id < a.num_blocks ? (id << bsl) | (pos & (bs - 1)) : INT32_MAX;
  }
  // the buffers' rest, shared by all workgroups
  const long long all = (long long)gridDim.x * stride;
  for (long long t = total + (long long)me * stride + first; t < a.max_tokens; t += all) {
    a.positions[t] = -1;
    a.slots[t] = -1;
  }
  if (blockIdx.y != 0 || tid != 0) return;
  if (any) {
    a.n_blocks_out[me] = ok ? blocks : have_raw;
    a.context_lens[me] = seq + nw;
    a.cu_q_lens[me] = cu;
  }
  if (me == 0) {
    a.cu_q_lens[a.n_seqs] = total;
    *a.free_count_out = ok ? count - (int)need_t : count;
    *a.status = bad ? -1 : ok ? 0 : (int)(lacking < INT32_MAX ? lacking : INT32_MAX);
  }
}

}  // namespace

hipError_t launch_step_tables(const StepArgs& a, hipStream_t stream) {
  // up to about 1024 workgroups, none without 256 entries of its own
  const int most = std::max(a.width, a.max_tokens);
  const int n = std::max(a.n_seqs, 1);
  const int y = std::max(1, std::min(1024 / n, (most + kStepThreads - 1) / kStepThreads));
  if (!grid_fits((long long)n * y, kStepThreads)) return hipErrorInvalidValue;
  step_tables_kernel<<<dim3(n, y), kStepThreads, 0, stream>>>(a);
  return hipGetLastError();
}

}  // namespace pkv
