// pkv_q4.hip -- rows into a pool held in 4 bits and the values back (gfx950).
//
// A group of 32 channels with smallest element m (in f16) and s = f16((max - m) / 15)
// holds element x as c = round((x - m) / s), 0 .. 15; it stands for m + s c.  The
// choice of c is the one of 64-bit arithmetic, so equal rows give equal bytes
// wherever they are stored.
//
// Both directions move bytes: rows of 2 or 4 bytes an element and a pool of 5 bits, each
// once.  60,001 tokens of 8 heads of 128 in f16 take 85 us to store and 48 to read
// back (3.8 and 6.7 TB/s; a large copy moves 5.0), 126 one after the other.  The store spends
// 83 % of its cycles on some 360 vector instructions a wave of 1024 elements; with 64-bit
// divisions throughout, and 2 tokens of 8 heads a workgroup, it took 150.
#include <algorithm>

#include "pkv_internal.h"
#include "pkv_q4_dev.h"

namespace pkv {
namespace {

constexpr int kQ4Threads = 256;

// Eight elements of type DT from `at`, which nothing here reads again.
template <int DT>
__device__ __forceinline__ void load8(const char* at, float (&x)[8]) {
  if constexpr (DT == PKV_F32) {
    float a[4], b[4];
    widen16<PKV_F32>(ld16_stream(at), a);
    widen16<PKV_F32>(ld16_stream(at + 16), b);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      x[e] = a[e];
      x[4 + e] = b[e];
    }
  } else {
    widen16<DT>(ld16_stream(at), x);
  }
}

// Over the four lanes of a group, of finite numbers (med3 with an infinity: fminf and
// fmaxf would quiet their operands first).
template <int CTRL>
__device__ __forceinline__ float quad(float x) {
  const int i = __float_as_int(x);
  return __int_as_float(__builtin_amdgcn_update_dpp(i, i, CTRL, 0xf, 0xf, true));
}
__device__ __forceinline__ float quad_min(float x) {
  x = __builtin_amdgcn_fmed3f(x, quad<0xB1>(x), -INFINITY);  // quad_perm 1, 0, 3, 2
  return __builtin_amdgcn_fmed3f(x, quad<0x4E>(x), -INFINITY);  // quad_perm 2, 3, 0, 1
}
__device__ __forceinline__ float quad_max(float x) {
  x = __builtin_amdgcn_fmed3f(x, quad<0xB1>(x), INFINITY);
  return __builtin_amdgcn_fmed3f(x, quad<0x4E>(x), INFINITY);
}

// Elements are limited so that what they are held as stays in the f16 range (m + 15 s is
// above the largest by 2^-11 of 15 s at most).
constexpr float kLimit = 65024.0f;

// x / 15 rounded to nearest, for normal quotients (below them an f16 is 0): with y = 1/15
// rounded and q = x y, the remainder x - 15 q is exact and q + y (x - 15 q) rounds to the
// quotient (Markstein, 1990).
__device__ __forceinline__ float by_15(float x) {
  const float y = 1.0f / 15.0f, q = x * y;
  float z = fmaf(fmaf(-15.0f, q, x), y, q);
  asm("" : "+v"(z));  // (else the rounding to f16 becomes part of the fma, and there is one only)
  return z;
}

// Nibble of channel e in a word of K codes, and in one as the exchange below has it.
__device__ __forceinline__ constexpr int k_nibble(int e) { return q4_k_bit(e) / 4; }
__device__ __forceinline__ constexpr int plain_nibble(int e) { return e; }

// Codes of this lane's eight elements, that of element e in nibble AT(e), and the group's
// m and s.  Kept to few instructions, which bound the store: NaN and large elements, and
// quotients close to the middle between two codes, take a path of their own.
//   t = d / s + 1.5 * 2^23 in one fma, d = x - m, rounds d / s to an integer in t's low
// bits.  d and the reciprocal of s are off by 2^-24 and 2^-23 of their size, so the
// quotient is within 2^-18 below 16: unless its distance from t's is as close to 1/2,
// the integer is that of 64 bits.  Eight words t shifted and added up modulo 2^32 are the
// codes plus a constant.
template <int (*AT)(int)>
__device__ __forceinline__ uint32_t quantize8(float (&x)[8], _Float16& m, _Float16& s) {
  auto range = [&](float& lo, float& hi) {
    lo = fminf(x[0], x[1]);
    hi = fmaxf(x[0], x[1]);
#pragma unroll
    for (int e = 2; e < 8; e += 2) {
      lo = fminf(fminf(x[e], x[e + 1]), lo);
      hi = fmaxf(fmaxf(x[e], x[e + 1]), hi);
    }
  };
  float lo, hi, odd = 0.0f;  // odd: NaN if an element is not finite
  range(lo, hi);
#pragma unroll
  for (int e = 0; e < 8; ++e) odd = fmaf(x[e], 0.0f, odd);
  if (!(odd == 0.0f && lo >= -kLimit && hi <= kLimit)) {
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = x[e] != x[e] ? 0.0f : fminf(fmaxf(x[e], -kLimit), kLimit);
    range(lo, hi);
  }
  lo = quad_min(lo);
  hi = quad_max(hi);
  m = (_Float16)lo;
  s = (_Float16)by_15(__fsub_rn(hi, (float)m));
  if (!(s > (_Float16)0.0f)) return 0;
  const float mf = (float)m, inv = __builtin_amdgcn_rcpf((float)s), magic = 12582912.0f;
  float t[8], off = 0.0f;  // t: in the order of the nibbles
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const float d = x[e] - mf;
    const float r = fmaf(d, inv, magic);
    off = fmaxf(off, fabsf(fmaf(d, inv, magic - r)));
    t[AT(e)] = __builtin_amdgcn_fmed3f(r, magic, magic + 15.0f);
  }
  uint32_t w = 0;
  if (off < 0.5f - 0x1p-15f) {
#pragma unroll
    for (int e = 7; e >= 0; --e) w = (w << 4) + __float_as_uint(t[e]);
    return w - 0x4b400000u * 0x11111111u;
  }
  const double md = (double)m, sd = (double)s;
#pragma unroll
  for (int e = 0; e < 8; ++e)
    w |= (uint32_t)fmin(fmax(rint(((double)x[e] - md) / sd), 0.0), 15.0) << (4 * AT(e));
  return w;
}

// Where a workgroup's tokens go: HD / 8 lanes a row, kRows<HD> tokens of one kv head,
// because neighbouring tokens share the cache lines of a block's codes, scales and
// offsets, and another workgroup's part of a line is written from another XCD.
template <int HD>
constexpr int kRows = kQ4Threads * 8 / HD;

// The slot of a token, -1: none.  n_slots: at most 2^31.
__device__ __forceinline__ int slot_of(const int32_t* slots, bool live, uint32_t tok,
                                       uint32_t n_slots, bool reporter, uint32_t* err) {
  const int slot = live ? slots[tok] : -1;
  if (slot < 0 || (uint32_t)slot < n_slots) return slot;
  if (reporter) atomicOr(err, PKV_EBIT_SLOT);
  return -1;
}

// Words of a row of codes in LDS, padded so that 16 rows' 16-byte reads meet no bank twice.
template <int HD>
constexpr int kRowWords = HD / 8 + 4;

template <int DT, int HD>
__global__ void __launch_bounds__(kQ4Threads)
    q4_append_kernel(char* kp, char* vp, const char* k, const char* v, long long k_stride,
                     long long v_stride, const int32_t* __restrict__ slots, int n, int kvh,
                     int bs_log2, uint32_t n_slots, uint32_t* err) {
  using L = Q4Layout<HD>;
  constexpr int LANES = HD / 8, E = DT == PKV_F32 ? 4 : 2, T = L::T;
  // V codes [row][lane % 2][lane / 2]: channel 8 lane + e is (i, t) = (8 (lane % 2) + e, lane / 2)
  __shared__ __attribute__((aligned(16))) uint32_t codes[kRows<HD>][kRowWords<HD>];
  const int bs = 1 << bs_log2;
  const int h = blockIdx.x % kvh;
  const uint32_t tok0 = blockIdx.x / kvh * kRows<HD>, left = n - tok0;  // left: 1 or more
  const uint32_t lane = threadIdx.x % LANES, local = threadIdx.x / LANES;
  // V codes are written by threads in the order of their bytes
  constexpr int W = T >= 8 ? T / 8 : 1;  // words of a column (HD 64: two columns' halves)
  constexpr uint32_t COLS = HD == 64 ? 8 : 16;
  const uint32_t wl = (threadIdx.x / W & 3) | threadIdx.x / (4 * W * COLS) << 2;
  const uint32_t col = threadIdx.x / (4 * W) % COLS;
  const int slot = slot_of(slots + tok0, local < left, local, n_slots, lane == 0 && h == 0, err);
  const int wslot = slot_of(slots + tok0, wl < left, wl, n_slots, false, err);
  const size_t blk_bytes = (size_t)kvh * L::chunk(bs), head_at = (size_t)h * L::chunk(bs);
  const size_t head = (size_t)h * HD * E;
  // read whether there is a slot or not, and not only once it is known; strides are at
  // most 2^24 elements
  const uint32_t row = min(local, left - 1);
  float x[8], y[8];
  load8<DT>(k + ((size_t)tok0 * k_stride * E + head) +
                (row * (uint32_t)(k_stride * E) + lane * 8 * E), x);
  load8<DT>(v + ((size_t)tok0 * v_stride * E + head) +
                (row * (uint32_t)(v_stride * E) + lane * 8 * E), y);
  if (slot >= 0) {
    _Float16 m, s;
    const int g = lane / 4, i = lane % 4, at = slot & (bs - 1);
    const size_t chunk = (uint32_t)(slot >> bs_log2) * blk_bytes + head_at;
    const uint32_t w = quantize8<k_nibble>(x, m, s);
    char* o = kp + chunk;
    *reinterpret_cast<uint32_t*>(o + L::k_word(at, i, g)) = w;
    if (i == 0) {
      *reinterpret_cast<_Float16*>(o + L::s_at(bs, at, g)) = s;
      *reinterpret_cast<_Float16*>(o + L::m_at(bs, at, g)) = m;
    }
    codes[local][(lane & 1) * T + lane / 2] = quantize8<plain_nibble>(y, m, s);
    o = vp + chunk;
    if (i == 0) {
      *reinterpret_cast<_Float16*>(o + L::s_at(bs, at, g)) = s;
      *reinterpret_cast<_Float16*>(o + L::m_at(bs, at, g)) = m;
    }
  }
  __syncthreads();
  if (wslot < 0) return;
  char* o = vp + ((uint32_t)(wslot >> bs_log2) * blk_bytes + head_at);
  const int at = wslot & (bs - 1);
  if constexpr (HD == 64) {  // columns 2 col, 2 col + 1
    const u32x4 x = *reinterpret_cast<const u32x4*>(&codes[wl][(col / 4) * T]);
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int i = 2 * col + j;
      uint32_t w = 0;
#pragma unroll
      for (int t = 3; t >= 0; --t) w = w << 4 | __builtin_amdgcn_ubfe(x[t], 4 * (i & 7), 4);
      *reinterpret_cast<uint16_t*>(o + L::v_bytes(at, i)) = (uint16_t)w;
    }
  } else {
    const int word = threadIdx.x % W;
    const uint32_t* c = &codes[wl][(col / 8) * T + 8 * word];
    const u32x4 x0 = *reinterpret_cast<const u32x4*>(c);
    const u32x4 x1 = *reinterpret_cast<const u32x4*>(c + 4);
    uint32_t w = 0;
#pragma unroll
    for (int t = 7; t >= 0; --t)
      w = w << 4 | __builtin_amdgcn_ubfe(t < 4 ? x0[t % 4] : x1[t % 4], 4 * (col & 7), 4);
    *reinterpret_cast<uint32_t*>(o + L::v_bytes(at, col) + 4 * word) = w;
  }
}

__device__ __forceinline__ void stream16(char* p, u32x4 v) {
  __builtin_nontemporal_store(v, reinterpret_cast<u32x4*>(p));
}
// Eight values as DT, which nothing here reads again (round to nearest even).
template <int DT>
__device__ __forceinline__ void store8(char* at, const float (&x)[8]) {
  if constexpr (DT == PKV_F32) {
#pragma unroll
    for (int e = 0; e < 8; e += 4)
      stream16(at + 4 * e, u32x4{__float_as_uint(x[e]), __float_as_uint(x[e + 1]),
                             __float_as_uint(x[e + 2]), __float_as_uint(x[e + 3])});
  } else {
    u32x4 w;
#pragma unroll
    for (int e = 0; e < 4; ++e) w[e] = cvt_pk16<DT>(x[2 * e], x[2 * e + 1]);
    stream16(at, w);
  }
}

template <int DT, int HD>
__global__ void __launch_bounds__(kQ4Threads)
    q4_gather_kernel(const char* __restrict__ kp, const char* __restrict__ vp, char* __restrict__ ok,
                     char* __restrict__ ov, const int32_t* __restrict__ slots, int n, int kvh,
                     int bs_log2, uint32_t n_slots, uint32_t* err) {
  using L = Q4Layout<HD>;
  constexpr int LANES = HD / 8, E = DT == PKV_F32 ? 4 : 2, T = L::T;
  constexpr int W = T >= 8 ? T / 8 : 1;
  // V codes: words [row][word of a column][column] (HD 64: 16 bits a column)
  __shared__ __attribute__((aligned(16))) uint32_t codes[kRows<HD>][kRowWords<HD>];
  const int bs = 1 << bs_log2;
  const int h = blockIdx.x % kvh;
  const uint32_t tok0 = blockIdx.x / kvh * kRows<HD>, left = n - tok0;  // left: 1 or more
  const uint32_t lane = threadIdx.x % LANES, local = threadIdx.x / LANES;
  constexpr uint32_t COLS = HD == 64 ? 8 : 16;
  const uint32_t wl = (threadIdx.x / W & 3) | threadIdx.x / (4 * W * COLS) << 2;
  const uint32_t col = threadIdx.x / (4 * W) % COLS;
  const int slot = slot_of(slots + tok0, local < left, local, n_slots, lane == 0 && h == 0, err);
  const int wslot = slot_of(slots + tok0, wl < left, wl, n_slots, false, err);
  if (wslot >= 0) {
    const char* o = vp + ((size_t)(wslot >> bs_log2) * kvh + h) * L::chunk(bs);
    const int at = wslot & (bs - 1);
    if constexpr (HD == 64) {
      codes[wl][col] = *reinterpret_cast<const uint16_t*>(o + L::v_bytes(at, 2 * col)) |
                       *reinterpret_cast<const uint16_t*>(o + L::v_bytes(at, 2 * col + 1)) << 16;
    } else {
      const int word = threadIdx.x % W;
      codes[wl][16 * word + col] =
          *reinterpret_cast<const uint32_t*>(o + L::v_bytes(at, col) + 4 * word);
    }
  }
  const int at = slot & (bs - 1), g = lane / 4, i = lane % 4, t = lane / 2;
  float x[8] = {}, y[8] = {}, s = 0.0f, m = 0.0f;
  if (slot >= 0) {
    const size_t chunk = ((size_t)(slot >> bs_log2) * kvh + h) * L::chunk(bs);
    const char* o = kp + chunk;
    const uint32_t w = *reinterpret_cast<const uint32_t*>(o + L::k_word(at, i, g));
    s = *reinterpret_cast<const _Float16*>(o + L::s_at(bs, at, g));
    m = *reinterpret_cast<const _Float16*>(o + L::m_at(bs, at, g));
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = fmaf(s, (float)((w >> q4_k_bit(e)) & 15), m);
    o = vp + chunk;
    s = *reinterpret_cast<const _Float16*>(o + L::s_at(bs, at, g));
    m = *reinterpret_cast<const _Float16*>(o + L::m_at(bs, at, g));
  }
  __syncthreads();
  if (local >= left) return;
  if (slot >= 0) {
    if constexpr (HD == 64) {
      const u32x4 w = *reinterpret_cast<const u32x4*>(&codes[local][4 * (lane & 1)]);
#pragma unroll
      for (int e = 0; e < 8; ++e)
        y[e] = fmaf(s, (float)((w[e / 2] >> (16 * (e % 2) + 4 * t)) & 15), m);
    } else {
      const uint32_t* c = &codes[local][16 * (t / 8) + 8 * (lane & 1)];
      const u32x4 w0 = *reinterpret_cast<const u32x4*>(c);
      const u32x4 w1 = *reinterpret_cast<const u32x4*>(c + 4);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        y[e] = fmaf(s, (float)((w0[e] >> (4 * (t & 7))) & 15), m);
        y[4 + e] = fmaf(s, (float)((w1[e] >> (4 * (t & 7))) & 15), m);
      }
    }
  }
  const size_t off = (((size_t)(tok0 + local) * kvh + h) * HD + lane * 8) * E;
  store8<DT>(ok + off, x);
  store8<DT>(ov + off, y);
}

int log2_of(int x) {
  int n = 0;
  while ((1 << n) < x) ++n;
  return n;
}

// (slots are int32: those from 2^31 on have no number)
uint32_t slots_of(const pkv_pool* p) {
  return (uint32_t)std::min((long long)p->num_blocks * p->block_size, 1LL << 31);
}

long long q4_blocks(const pkv_pool* p, int n) {
  const int per = kQ4Threads * 8 / p->head_dim;
  return ((long long)n + per - 1) / per * p->n_kv_head;
}

template <int DT, int HD>
hipError_t append(const pkv_pool* p, int layer, const void* k, const void* v, long long ks,
                  long long vs, const int32_t* slots, int n, hipStream_t stream) {
  q4_append_kernel<DT, HD><<<(unsigned)q4_blocks(p, n), kQ4Threads, 0, stream>>>(
      p->layer_k(layer), p->layer_v(layer), static_cast<const char*>(k),
      static_cast<const char*>(v), ks, vs, slots, n, p->n_kv_head,
      log2_of(p->block_size), slots_of(p), p->err);
  return hipGetLastError();
}

template <int DT, int HD>
hipError_t gather(const pkv_pool* p, int layer, const int32_t* slots, int n, void* ok, void* ov,
                  hipStream_t stream) {
  q4_gather_kernel<DT, HD><<<(unsigned)q4_blocks(p, n), kQ4Threads, 0, stream>>>(
      p->layer_k(layer), p->layer_v(layer), static_cast<char*>(ok), static_cast<char*>(ov), slots,
      n, p->n_kv_head, log2_of(p->block_size),
      slots_of(p), p->err);
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
