// pkv_q4.hip -- rows into a pool held in 4 bits and the values back (gfx950).
//
// A group of 32 channels with smallest element m (in f16) and s = f16((max - m) / 15)
// holds element x as c = round((x - m) / s), 0 .. 15; it stands for m + s c.  The
// choice of c is the one of 64-bit arithmetic, so equal rows give equal bytes
// wherever they are stored.
#include "pkv_internal.h"
#include "pkv_q4_dev.h"

namespace pkv {
namespace {

constexpr int kQ4Threads = 256;

// Eight elements of type DT from `at`, NaN as 0 and limited so that what they are held
// as stays in the f16 range (m + 15 s is above the largest by 2^-11 of 15 s at most).
constexpr float kLimit = 65024.0f;
template <int DT>
__device__ __forceinline__ void load8(const char* at, float (&x)[8]) {
  if constexpr (DT == PKV_F32) {
    float a[4], b[4];
    widen16<PKV_F32>(ld16(at), a);
    widen16<PKV_F32>(ld16(at + 16), b);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      x[e] = a[e];
      x[4 + e] = b[e];
    }
  } else {
    widen16<DT>(ld16(at), x);
  }
#pragma unroll
  for (int e = 0; e < 8; ++e) x[e] = x[e] != x[e] ? 0.0f : fminf(fmaxf(x[e], -kLimit), kLimit);
}

// Over the four lanes of a group.
template <int CTRL>
__device__ __forceinline__ float quad(float x) {
  return dpp_f<CTRL>(x);
}
__device__ __forceinline__ float quad_min(float x) {
  x = fminf(x, quad<0xB1>(x));  // quad_perm 1, 0, 3, 2
  return fminf(x, quad<0x4E>(x));  // quad_perm 2, 3, 0, 1
}
__device__ __forceinline__ float quad_max(float x) {
  x = fmaxf(x, quad<0xB1>(x));
  return fmaxf(x, quad<0x4E>(x));
}

// Codes of this lane's eight elements, and the group's m and s.
__device__ __forceinline__ void quantize8(const float (&x)[8], int (&c)[8], _Float16& m,
                                          _Float16& s) {
  float lo = x[0], hi = x[0];
#pragma unroll
  for (int e = 1; e < 8; ++e) {
    lo = fminf(lo, x[e]);
    hi = fmaxf(hi, x[e]);
  }
  lo = quad_min(lo);
  hi = quad_max(hi);
  m = (_Float16)lo;
  s = (_Float16)__fdiv_rn(__fsub_rn(hi, (float)m), 15.0f);
  const double md = (double)m, sd = (double)s;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const double y = s > (_Float16)0.0f ? rint(((double)x[e] - md) / sd) : 0.0;
    c[e] = (int)fmin(fmax(y, 0.0), 15.0);
  }
}

// HD / 8 lanes a row (token, kv head): eight channels each, of K and of V.
template <int DT, int HD>
__global__ void __launch_bounds__(kQ4Threads)
    q4_append_kernel(char* kp, char* vp, const char* k, const char* v, long long k_stride,
                     long long v_stride, const int32_t* __restrict__ slots, long long rows,
                     int kvh, int bs_log2, long long n_slots, uint32_t* err) {
  using L = Q4Layout<HD>;
  constexpr int LANES = HD / 8, E = DT == PKV_F32 ? 4 : 2;
  __shared__ __attribute__((aligned(16))) uint8_t codes[kQ4Threads * 8];  // [row][i][t]
  const int bs = 1 << bs_log2;
  const int lane = threadIdx.x % LANES, local = threadIdx.x / LANES;
  const long long r = (long long)blockIdx.x * (kQ4Threads / LANES) + local;
  const long long tok = r / kvh;
  const int h = (int)(r - tok * kvh);
  int slot = r < rows ? slots[tok] : -1;
  if (slot >= n_slots) {
    if (lane == 0 && h == 0) atomicOr(err, PKV_EBIT_SLOT);
    slot = -1;
  }
  const bool live = slot >= 0;
  const int at = live ? slot & (bs - 1) : 0;
  const size_t chunk = ((size_t)(live ? slot >> bs_log2 : 0) * kvh + h) * L::chunk(bs);
  uint8_t* mine = codes + local * HD;
  if (live) {
    float x[8];
    int c[8];
    _Float16 m, s;
    const int g = lane / 4, i = lane % 4;
    load8<DT>(k + ((size_t)tok * k_stride + (size_t)h * HD + lane * 8) * E, x);
    quantize8(x, c, m, s);
    uint32_t w = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) w |= (uint32_t)c[e] << q4_k_bit(e);
    char* o = kp + chunk;
    *reinterpret_cast<uint32_t*>(o + L::k_word(at, i, g)) = w;
    if (i == 0) {
      *reinterpret_cast<_Float16*>(o + L::s_at(bs, at, g)) = s;
      *reinterpret_cast<_Float16*>(o + L::m_at(bs, at, g)) = m;
    }
    load8<DT>(v + ((size_t)tok * v_stride + (size_t)h * HD + lane * 8) * E, x);
    quantize8(x, c, m, s);
    o = vp + chunk;
    if (i == 0) {
      *reinterpret_cast<_Float16*>(o + L::s_at(bs, at, g)) = s;
      *reinterpret_cast<_Float16*>(o + L::m_at(bs, at, g)) = m;
    }
    // channel 8 lane + e is (i, t) = (8 (lane % 2) + e, lane / 2)
#pragma unroll
    for (int e = 0; e < 8; ++e) mine[(8 * (lane & 1) + e) * L::T + lane / 2] = (uint8_t)c[e];
  }
  __syncthreads();
  if (!live) return;
  uint32_t w = 0;  // codes 8 lane .. of [i][t]
#pragma unroll
  for (int e = 0; e < 8; ++e) w |= (uint32_t)mine[lane * 8 + e] << (4 * e);
  char* o = vp + chunk;
  if constexpr (HD == 64) {  // two columns of four
    *reinterpret_cast<uint16_t*>(o + L::v_bytes(bs, at, 2 * lane)) = (uint16_t)w;
    *reinterpret_cast<uint16_t*>(o + L::v_bytes(bs, at, 2 * lane + 1)) = (uint16_t)(w >> 16);
  } else {
    constexpr int PER = L::T / 8;  // words of a column
    *reinterpret_cast<uint32_t*>(o + L::v_bytes(bs, at, lane / PER) + 4 * (lane % PER)) = w;
  }
}

// Eight values as DT (round to nearest even).
template <int DT>
__device__ __forceinline__ void store8(char* at, const float (&x)[8]) {
  if constexpr (DT == PKV_F32) {
#pragma unroll
    for (int e = 0; e < 8; e += 4)
      st16(at + 4 * e, u32x4{__float_as_uint(x[e]), __float_as_uint(x[e + 1]),
                             __float_as_uint(x[e + 2]), __float_as_uint(x[e + 3])});
  } else {
    u32x4 w;
#pragma unroll
    for (int e = 0; e < 4; ++e) w[e] = cvt_pk16<DT>(x[2 * e], x[2 * e + 1]);
    st16(at, w);
  }
}

template <int DT, int HD>
__global__ void __launch_bounds__(kQ4Threads)
    q4_gather_kernel(const char* __restrict__ kp, const char* __restrict__ vp, char* __restrict__ ok,
                     char* __restrict__ ov, const int32_t* __restrict__ slots, long long rows,
                     int kvh, int bs_log2, long long n_slots, uint32_t* err) {
  using L = Q4Layout<HD>;
  constexpr int LANES = HD / 8, E = DT == PKV_F32 ? 4 : 2;
  const int bs = 1 << bs_log2;
  const int lane = threadIdx.x % LANES;
  const long long r = (long long)blockIdx.x * (kQ4Threads / LANES) + threadIdx.x / LANES;
  if (r >= rows) return;
  const long long tok = r / kvh;
  const int h = (int)(r - tok * kvh);
  int slot = slots[tok];
  if (slot >= n_slots) {
    if (lane == 0 && h == 0) atomicOr(err, PKV_EBIT_SLOT);
    slot = -1;
  }
  float x[8] = {}, y[8] = {};
  if (slot >= 0) {
    const int at = slot & (bs - 1), g = lane / 4, i = lane % 4, t = lane / 2;
    const size_t chunk = ((size_t)(slot >> bs_log2) * kvh + h) * L::chunk(bs);
    const char* o = kp + chunk;
    const uint32_t w = *reinterpret_cast<const uint32_t*>(o + L::k_word(at, i, g));
    float s = *reinterpret_cast<const _Float16*>(o + L::s_at(bs, at, g));
    float m = *reinterpret_cast<const _Float16*>(o + L::m_at(bs, at, g));
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = fmaf(s, (float)((w >> q4_k_bit(e)) & 15), m);
    o = vp + chunk;
    s = *reinterpret_cast<const _Float16*>(o + L::s_at(bs, at, g));
    m = *reinterpret_cast<const _Float16*>(o + L::m_at(bs, at, g));
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const uint8_t b = o[L::v_bytes(bs, at, 8 * (lane & 1) + e) + t / 2];
      y[e] = fmaf(s, (float)((b >> (4 * (t & 1))) & 15), m);
    }
  }
  const size_t off = ((size_t)r * HD + lane * 8) * E;
  store8<DT>(ok + off, x);
  store8<DT>(ov + off, y);
}

int log2_of(int x) {
  int n = 0;
  while ((1 << n) < x) ++n;
  return n;
}

long long q4_blocks(const pkv_pool* p, int n) {
  const long long per = kQ4Threads / (p->head_dim / 8);
  return ((long long)n * p->n_kv_head + per - 1) / per;
}

template <int DT, int HD>
hipError_t append(const pkv_pool* p, int layer, const void* k, const void* v, long long ks,
                  long long vs, const int32_t* slots, int n, hipStream_t stream) {
  q4_append_kernel<DT, HD><<<(unsigned)q4_blocks(p, n), kQ4Threads, 0, stream>>>(
      p->layer_k(layer), p->layer_v(layer), static_cast<const char*>(k),
      static_cast<const char*>(v), ks, vs, slots, (long long)n * p->n_kv_head, p->n_kv_head,
      log2_of(p->block_size), (long long)p->num_blocks * p->block_size, p->err);
  return hipGetLastError();
}

template <int DT, int HD>
hipError_t gather(const pkv_pool* p, int layer, const int32_t* slots, int n, void* ok, void* ov,
                  hipStream_t stream) {
  q4_gather_kernel<DT, HD><<<(unsigned)q4_blocks(p, n), kQ4Threads, 0, stream>>>(
      p->layer_k(layer), p->layer_v(layer), static_cast<char*>(ok), static_cast<char*>(ov), slots,
      (long long)n * p->n_kv_head, p->n_kv_head, log2_of(p->block_size),
      (long long)p->num_blocks * p->block_size, p->err);
  return hipGetLastError();
}

}  // namespace

bool q4_rows_fit(const pkv_pool* p, int n) { return grid_fits(q4_blocks(p, n), kQ4Threads); }

#define PKV_BY_TYPE(dt, hd, F, ...)                                                     \
  switch ((dt) * 1000 + (hd)) {                                                         \
    case PKV_F32 * 1000 + 64: return F<PKV_F32, 64>(__VA_ARGS__);                       \
    case PKV_F32 * 1000 + 128: return F<PKV_F32, 128>(__VA_ARGS__);                     \
    case PKV_F32 * 1000 + 256: return F<PKV_F32, 256>(__VA_ARGS__);                     \
    case PKV_F16 * 1000 + 64: return F<PKV_F16, 64>(__VA_ARGS__);                       \
    case PKV_F16 * 1000 + 128: return F<PKV_F16, 128>(__VA_ARGS__);                     \
    case PKV_F16 * 1000 + 256: return F<PKV_F16, 256>(__VA_ARGS__);                     \
    case PKV_BF16 * 1000 + 64: return F<PKV_BF16, 64>(__VA_ARGS__);                     \
    case PKV_BF16 * 1000 + 128: return F<PKV_BF16, 128>(__VA_ARGS__);                   \
    case PKV_BF16 * 1000 + 256: return F<PKV_BF16, 256>(__VA_ARGS__);                   \
  }                                                                                     \
  return hipErrorInvalidValue

hipError_t launch_q4_append(const pkv_pool* p, int layer, const void* k, const void* v, int dtype,
                            long long ks, long long vs, const int32_t* slots, int n,
                            hipStream_t stream) {
  PKV_BY_TYPE(dtype, p->head_dim, append, p, layer, k, v, ks, vs, slots, n, stream);
}

hipError_t launch_q4_gather(const pkv_pool* p, int layer, const int32_t* slots, int n, void* ok,
                            void* ov, int dtype, hipStream_t stream) {
  PKV_BY_TYPE(dtype, p->head_dim, gather, p, layer, slots, n, ok, ov, stream);
}

}  // namespace pkv
