// pkv_q4_attn.hip -- attention over a pool held in 4 bits (gfx950).
//
// One wave per (query row, query head): a lane scores one key of 64, the weights go
// through LDS, and a lane then sums the values of its channels, with a running
// maximum and sum.
#include "pkv_internal.h"
#include "pkv_q4_dev.h"

namespace pkv {
namespace {

__device__ __forceinline__ float elem(const void* p, int dt, size_t i) {
  if (dt == PKV_F32) return static_cast<const float*>(p)[i];
  if (dt == PKV_F16) return (float)static_cast<const _Float16*>(p)[i];
  return bf16lo(static_cast<const uint16_t*>(p)[i]);
}
__device__ __forceinline__ void put(void* out, int dt, size_t i, float x) {
  if (dt == PKV_F32) static_cast<float*>(out)[i] = x;
  else if (dt == PKV_F16) static_cast<_Float16*>(out)[i] = (_Float16)x;
  else static_cast<uint16_t*>(out)[i] = (uint16_t)f32_to_bf16_bits(x);
}
__device__ __forceinline__ float half_at(const char* p) {
  return (float)*reinterpret_cast<const _Float16*>(p);
}

struct Q4KArgs {
  Q4Args a;
  const char* k;
  const char* v;
  int kvh;
  int bs_log2;
  int num_blocks;
  uint32_t* err;
};

template <int HD>
__global__ void __launch_bounds__(64) q4_attn_kernel(Q4KArgs ka) {
  using L = Q4Layout<HD>;
  constexpr int PER = HD / 64;
  const Q4Args& a = ka.a;
  __shared__ float q[HD];
  __shared__ float p[64];
  const int lane = threadIdx.x, bs = 1 << ka.bs_log2;
  const int h = blockIdx.x % a.n_head;
  const int u = blockIdx.x / a.n_head;
  const int s = u / a.max_q_len, i = u % a.max_q_len;
  const int q0 = a.cu_q_lens ? a.cu_q_lens[s] : s, q1 = a.cu_q_lens ? a.cu_q_lens[s + 1] : s + 1;
  const int ctx = a.context_lens[s];
  const int m_rows = q0 >= 0 && q1 >= q0 && q1 <= a.total_q ? q1 - q0 : -1;
  if (m_rows < 0 || m_rows > a.max_q_len || ctx < 0 ||
      ctx > a.max_context_len || ctx > (long long)a.max_blocks_per_seq * bs) {
    if (i == 0 && h == 0 && lane == 0) atomicOr(ka.err, PKV_EBIT_LENGTH);
    return;
  }
  if (i >= m_rows) return;
  const int n = ctx - m_rows + i + 1;  // keys of the row
  const int row = q0 + i;
  const int g = h / (a.n_head / ka.kvh);
  const int32_t* table = a.block_tables + (size_t)s * a.max_blocks_per_seq;
  for (int j = 0; j < PER; ++j) {
    const int d = lane + 64 * j;
    q[d] = elem(a.q, a.q_dtype, (size_t)row * a.q_stride + (size_t)h * HD + d) * a.scale *
           1.44269504f;
  }
  __syncthreads();
  float m = -INFINITY, l = 0.0f, o[PER] = {};
  for (int k0 = 0; k0 < n; k0 += 64) {
    float x = -INFINITY;
    const int key = k0 + lane;
    if (key < n) {
      const int blk = table[key >> ka.bs_log2], at = key & (bs - 1);
      if ((unsigned)blk >= (unsigned)ka.num_blocks) {
        atomicOr(ka.err, PKV_EBIT_BLOCK);
      } else {
        const char* c = ka.k + ((size_t)blk * ka.kvh + g) * L::chunk(bs);
        x = 0.0f;
        for (int gr = 0; gr < L::G; ++gr) {
          float dot = 0.0f, sum = 0.0f;
          for (int w4 = 0; w4 < 4; ++w4) {
            const uint32_t w = *reinterpret_cast<const uint32_t*>(c + L::k_word(at, w4, gr));
            for (int e = 0; e < 8; ++e) {
              const float qq = q[32 * gr + 8 * w4 + e];
              dot = fmaf(qq, (float)((w >> q4_k_bit(e)) & 15), dot);
              sum += qq;
            }
          }
          x = fmaf(half_at(c + L::s_at(bs, at, gr)), dot, x);
          x = fmaf(half_at(c + L::km_at(bs, at, gr)), sum, x);
        }
      }
    }
    const float mn = fmaxf(m, row_group_max(row_max16(x)));
    const float ref = mn == -INFINITY ? 0.0f : mn;
    const float w = fast_exp2(x - ref), c = fast_exp2(m - ref);
    l = l * c + swap32_sum(swap16_sum(row_sum16(w)));
    m = mn;
    p[lane] = w;
    __syncthreads();
    for (int j = 0; j < PER; ++j) o[j] *= c;
    for (int kk = 0; kk < min(64, n - k0); ++kk) {
      const int pos = k0 + kk, blk = table[pos >> ka.bs_log2], at = pos & (bs - 1);
      if ((unsigned)blk >= (unsigned)ka.num_blocks) continue;
      const char* c = ka.v + ((size_t)blk * ka.kvh + g) * L::chunk(bs);
      for (int j = 0; j < PER; ++j) {
        const int d = lane + 64 * j, t = d / 16;
        const uint8_t b = c[L::v_bytes(bs, at, d % 16) + t / 2];
        const float v = fmaf(half_at(c + L::s_at(bs, at, d / 32)), (float)((b >> (4 * (t & 1))) & 15),
                             half_at(c + L::vm_at(bs, at, d / 32)));
        o[j] = fmaf(p[kk], v, o[j]);
      }
    }
    __syncthreads();
  }
  for (int j = 0; j < PER; ++j)
    put(a.out, a.out_dtype, ((size_t)row * a.n_head + h) * HD + lane + 64 * j,
        l > 0.0f ? o[j] / l : 0.0f);
}

}  // namespace

size_t q4_workspace_bytes(const pkv_pool*, const Q4Args&) { return 0; }

bool q4_fits(const pkv_pool*, const Q4Args& a) {
  return grid_fits((long long)a.n_seqs * a.max_q_len, 64) &&
         grid_fits((long long)a.n_seqs * a.max_q_len * a.n_head, 64);
}

hipError_t launch_q4_attention(const pkv_pool* p, int layer, const Q4Args& a, char*,
                               hipStream_t stream) {
  Q4KArgs ka{a, p->layer_k(layer), p->layer_v(layer), p->n_kv_head, 0, p->num_blocks, p->err};
  while ((1 << ka.bs_log2) < p->block_size) ++ka.bs_log2;
  const unsigned blocks = (unsigned)((long long)a.n_seqs * a.max_q_len * a.n_head);
  if (p->head_dim == 64) q4_attn_kernel<64><<<blocks, 64, 0, stream>>>(ka);
  else if (p->head_dim == 128) q4_attn_kernel<128><<<blocks, 64, 0, stream>>>(ka);
  else q4_attn_kernel<256><<<blocks, 64, 0, stream>>>(ka);
  return hipGetLastError();
}

}  // namespace pkv
