// pkv_select.hip -- key bounds of blocks and the choice of a context's blocks
// by them (gfx950).
//
// For block j of a kv head let lo_j and hi_j be the elementwise smallest and
// largest of its keys.  No key of the block scores above
//   s_hj = sum_d max(q_hd lo_jd, q_hd hi_jd) = q+ . hi_j + q- . lo_j
// against query head h (q+ = max(q, 0), q- = min(q, 0)): two rows stand for
// bs keys.  The choice of a query row and kv head is its first and last blocks
// and, of those between, the ones with the largest max_h s_hj.
//
// Choosing is exact: the blocks are those that the sums in 64 bits choose
// (lower index first among equals), while almost all of the work is done on
// the matrix cores in 32 bits.  With S~ the 32-bit sum and T = sum_d of the
// terms' magnitudes, |S~ - s| <= E = (hd + 16) 2^-23 T: half of the 2 hd
// products are zero, adding zero is exact, and each of the other hd adds
// rounds or truncates by at most 2^-23 of a partial sum, which T bounds; the
// 16 cover the products' own rounding in f32 pools.  If tau is the n-th
// largest S~ of a row and E the row's largest bound, n blocks have s >= tau -
// E, so one with S~ < tau - 2E is not chosen; at most n - 1 others reach tau + E,
// so one with S~ > tau + 2E is.  Only what lies between is summed again in 64 bits,
// mostly nothing or a few blocks.
//
// A block with a bound that is not finite (or a score past the f32 range)
// scores +inf, and so does every block for such a query.  E leaves out what
// falls below the f32 range: scores that differ by less than some hd 2^-126 may
// be taken for equal or in either order.
#include <algorithm>

#include "pkv_device.h"
#include "pkv_internal.h"

namespace pkv {
namespace {

// ---- key bounds --------------------------------------------------------------

struct BoundsKArgs {
  const char* k_pool;
  char* bounds;  // [num_blocks][kvh][2][hd]
  const int32_t* tables;
  int mbps;
  const int32_t* first;  // null: 0
  const int32_t* ctx;
  int n_seqs;
  int span;  // blocks per sequence at most
  int max_new;
  int num_blocks;
  int bs_log2;
  int kvh;
  uint32_t* err;
};

template <int DT>
__device__ __forceinline__ u32x4 narrow16(const float* x) {
  if constexpr (DT == PKV_F32) {
    return u32x4{__float_as_uint(x[0]), __float_as_uint(x[1]), __float_as_uint(x[2]),
                 __float_as_uint(x[3])};
  } else {
    u32x4 w;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t a = DT == PKV_BF16 ? f32_to_bf16_bits(x[2 * i]) : f32_to_f16_bits(x[2 * i]);
      const uint32_t b =
          DT == PKV_BF16 ? f32_to_bf16_bits(x[2 * i + 1]) : f32_to_f16_bits(x[2 * i + 1]);
      w[i] = a | (b << 16);
    }
    return w;
  }
}

// One thread per 16-byte chunk of a block's token rows: it walks the block's
// tokens, so a wave reads 1 KB of consecutive bytes per load, with up to 16
// loads in flight.  The keys are read once and the bound rows written once.
// Bound by HBM: 161 MB (12 prompts of 2-9k tokens, 8 kv heads of 128) in 33 us,
// 4.9 TB/s, the rate of a copy; the last block of 256 sequences in 4.4 us, a chain
// of two reads.  (Plain instead of streaming loads 38 us; 8 in flight 31.8, within the
// runs' spread.)
template <int DT, int HD>
__global__ void __launch_bounds__(256) bounds_kernel(BoundsKArgs a) {
  constexpr int E = DT == PKV_F32 ? 4 : 2;
  constexpr int EPL = 16 / E;
  constexpr int RB = HD * E;
  constexpr int CH = RB / 16;
  const int cpr = a.kvh * CH;  // chunks of a token's row
  const long long flat = (long long)blockIdx.x * 256 + threadIdx.x;
  const long long item = flat / cpr;
  const int c = (int)(flat - item * cpr);
  const int s = (int)(item / a.span);
  const int rel = (int)(item - (long long)s * a.span);
  if (s >= a.n_seqs) return;
  const int bsl = a.bs_log2, bs = 1 << bsl;
  const int ctx = a.ctx[s];
  const int first = a.first ? a.first[s] : 0;
  if (first < 0 || ctx < first || (ctx + (long long)bs - 1) >> bsl > a.mbps ||
      ctx - first > a.max_new) {
    if (c == 0 && rel == 0) atomicOr(a.err, PKV_EBIT_LENGTH);
    return;
  }
  const int j = (first >> bsl) + rel;
  if (ctx == first || j > (ctx - 1) >> bsl) return;
  const int id = a.tables[(size_t)s * a.mbps + j];
  if (id < 0 || id >= a.num_blocks) {
    if (c == 0) atomicOr(a.err, PKV_EBIT_BLOCK);
    return;
  }
  const int n = min(bs, ctx - (j << bsl));  // its keys
  const size_t stride = (size_t)cpr * 16;
  const char* k = a.k_pool + ((size_t)id << bsl) * stride + (size_t)c * 16;
  float lo[EPL], hi[EPL];
#pragma unroll
  for (int e = 0; e < EPL; ++e) {
    lo[e] = INFINITY;
    hi[e] = -INFINITY;
  }
  for (int t0 = 0; t0 < n; t0 += 16) {
    u32x4 w[16];
#pragma unroll
    for (int i = 0; i < 16; ++i)  // past the last key: the last one again
      w[i] = ld16_stream(k + (size_t)min(t0 + i, n - 1) * stride);
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      float x[EPL];
      widen16<DT, EPL>(w[i], x);
#pragma unroll
      for (int e = 0; e < EPL; ++e) {
        lo[e] = fminf(lo[e], x[e]);
        hi[e] = fmaxf(hi[e], x[e]);
      }
    }
  }
  const int g = c / CH, cc = c - g * CH;
  char* o = a.bounds + (((size_t)id * a.kvh + g) * 2) * RB + cc * 16;
  st16(o, narrow16<DT>(lo));
  st16(o + RB, narrow16<DT>(hi));
}

// ---- scores ------------------------------------------------------------------

struct SelectKArgs {
  const char* q;       // [total_q][n_head][hd]
  const char* bounds;  // [num_blocks][kvh][2][hd]
  const int32_t* tables;
  int mbps;
  const int32_t* cu;  // null: one row per sequence
  const int32_t* ctx;
  int n_seqs;
  int total_q;
  int tiles;   // row tiles per sequence
  int chunks;  // waves along the blocks
  int per;     // blocks per wave (a multiple of 16)
  int nb_max;  // blocks of a row at most
  int pitch;   // of score and again: nb_max in whole lines
  int num_blocks;
  int bs_log2;
  int kvh;
  int rtot;  // query heads per kv head
  int top;
  int n_first;
  int n_last;
  int max_q;
  float* score;  // [total_q][kvh][pitch]
  float* emax;   // [total_q][kvh][chunks]
  double* again; // [total_q][kvh][pitch], written where a sum is made again
  int32_t* out;  // [total_q][kvh][top]
  uint32_t* err;
};

// Rows of sequence s: r0 .. r0 + n - 1; row i of them has ctx - n + i + 1 keys.
struct SeqRows {
  int r0, n, ctx;
};
__device__ __forceinline__ SeqRows seq_rows(const int32_t* cu, const int32_t* ctx, int s,
                                            int total_q) {
  if (!cu) return {s, 1, ctx[s]};
  const int r0 = min(max(cu[s], 0), total_q), r1 = min(max(cu[s + 1], r0), total_q);
  return {r0, r1 - r0, ctx[s]};
}
// Blocks of row i, at most what the tables hold.
__device__ __forceinline__ int row_blocks(const SeqRows& r, int i, int bsl, int nb_max) {
  const long long keys = (long long)r.ctx - r.n + i + 1;
  const long long nb = keys > 0 ? (keys + (1 << bsl) - 1) >> bsl : 0;
  return (int)(nb < nb_max ? nb : nb_max);
}

// max(x, 0) and min(x, 0) of the elements of a 16-byte chunk; NaN stays in one.
template <int DT>
__device__ __forceinline__ void split_sign(const u32x4& w, u32x4& p, u32x4& m) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (DT == PKV_F32) {
      const bool neg = w[i] >> 31;
      p[i] = neg ? 0u : w[i];
      m[i] = neg ? w[i] : 0u;
    } else {
      const uint32_t neg = ((w[i] >> 15) & 0x00010001u) * 0xffffu;
      p[i] = w[i] & ~neg;
      m[i] = w[i] & neg;
    }
  }
}
template <int DT>
__device__ __forceinline__ u32x4 magnitude(const u32x4& w) {
  u32x4 r;
#pragma unroll
  for (int i = 0; i < 4; ++i) r[i] = w[i] & (DT == PKV_F32 ? 0x7fffffffu : 0x7fff7fffu);
  return r;
}

// One wave: 16 / R query rows of a sequence (a row tile: the 16 rows of the
// matrix operand, R heads each) against `per` blocks of one kv head, 16 at a
// time.  Lane l supplies 16-byte pieces of block l % 16's bound rows, as the
// K fragments of the decode kernel; S~ takes 2 NF matrix instructions, the
// two halves of T as many.  Bound by HBM: 360 MB of bounds (64 contexts of
// 12-32k tokens, 8 kv heads of 128) in 80 us, reads of the same rows
// alone in 74; scores leave through LDS in whole lines, for 64 bytes at a time
// (16 blocks) made it 83.  More loads in flight (the next 16 blocks' beside
// these: 85-117 us), non-temporal ones (93) and longer runs per wave (87 with
// 256 blocks) are slower.
constexpr int kFlush = 64;  // blocks whose scores a wave gathers

template <int DT, int HD, int R>
__global__ void __launch_bounds__(256) score_kernel(SelectKArgs a) {
  constexpr int E = DT == PKV_F32 ? 4 : 2;
  constexpr int RB = HD * E;
  constexpr int NF = RB / 64;
  constexpr int RP = 16 / R;  // query rows per tile
  __shared__ float buf_all[4][RP][kFlush];
  auto& buf = buf_all[threadIdx.x >> 6];
  const int lane = threadIdx.x & 63;
  const int G = lane >> 4, col = lane & 15;
  const long long wave = (long long)blockIdx.x * 4 + (threadIdx.x >> 6);
  // (sequence, tile, chunk, kv head), the head fastest
  const int g = (int)(wave % a.kvh);
  long long rest = wave / a.kvh;
  const int chunk = (int)(rest % a.chunks);
  rest /= a.chunks;
  const int tile = (int)(rest % a.tiles);
  const int s = (int)(rest / a.tiles);
  if (s >= a.n_seqs) return;
  const int bsl = a.bs_log2;
  const SeqRows sr = seq_rows(a.cu, a.ctx, s, a.total_q);
  const int i0 = tile * RP;
  if (i0 >= sr.n) return;
  const int nrow = min(RP, sr.n - i0);
  // blocks that some row of the tile ranks: the last row has the most
  const int nb = row_blocks(sr, i0 + nrow - 1, bsl, a.nb_max);
  const int j0 = max(chunk * a.per, a.n_first / 16 * 16);
  const int j1 = min((chunk + 1) * a.per, nb - a.n_last);
  float* em = a.emax + ((size_t)(sr.r0 + i0) * a.kvh + g) * a.chunks + chunk;
  const size_t em_row = (size_t)a.kvh * a.chunks;
  if (nb <= a.top || j0 >= j1) {
    if (lane < nrow) em[lane * em_row] = 0.0f;
    return;
  }

  const char* brow = a.bounds + (size_t)g * 2 * RB + 16 * G;
  const size_t bstride = (size_t)a.kvh * 2 * RB;
  const int32_t* tab = a.tables + (size_t)s * a.mbps;
  auto block_row = [&](int j) {
    const int id = tab[min(j + col, nb - 1)];
    const bool bad = id < 0 || id >= a.num_blocks;
    if (bad) atomicOr(a.err, PKV_EBIT_BLOCK);
    return brow + (size_t)(bad ? 0 : id) * bstride;
  };

  // slices of 16 heads (one for ratios up to 16)
  float etop = 0.0f;  // the largest T
  for (int h0 = 0; h0 < a.rtot; h0 += 16) {
    const int rq = min(a.rtot - h0, R);
    // operand row m = (query row m / R, head m % R)
    u32x4 qp[NF], qm[NF];
    const int mr = col / R, mh = col % R;
    const bool live = mr < nrow && mh < rq;
    const char* qrow = a.q + (((size_t)(sr.r0 + i0 + (live ? mr : 0)) * a.kvh + g) * a.rtot + h0 +
                              (live ? mh : 0)) * RB + 16 * G;
#pragma unroll
    for (int f = 0; f < NF; ++f) {
      const u32x4 w = live ? ld16(qrow + 64 * f) : u32x4{0, 0, 0, 0};
      split_sign<DT>(w, qp[f], qm[f]);
    }
    const char* next = block_row(j0);
    for (int j = j0; j < j1; j += 16) {
      u32x4 lo[NF], hi[NF];
#pragma unroll
      for (int f = 0; f < NF; ++f) {
        lo[f] = ld16(next + 64 * f);
        hi[f] = ld16(next + RB + 64 * f);
      }
      if (j + 16 < j1) next = block_row(j + 16);
      f32x4 sum = {0, 0, 0, 0}, tp = {0, 0, 0, 0}, tm = {0, 0, 0, 0};
#pragma unroll
      for (int f = 0; f < NF; ++f) {
        mfma_frag<DT>(qp[f], hi[f], sum);
        mfma_frag<DT>(qm[f], lo[f], sum);
        mfma_frag<DT>(qp[f], magnitude<DT>(hi[f]), tp);
        mfma_frag<DT>(qm[f], magnitude<DT>(lo[f]), tm);
      }
      // lane: rows 4 G + i of block j + col.  NaN and infinity become +inf.
      float sc[4], er[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float t = tp[i] - tm[i];
        const bool fin = t < INFINITY;  // (false for NaN)
        const bool mine = (4 * G + i) % R < rq;
        sc[i] = !mine ? -INFINITY : fin ? sum[i] : INFINITY;
        er[i] = mine && fin ? t : 0.0f;
      }
      // maximum over the R heads: registers first, then lane groups
#pragma unroll
      for (int w = 1; w < (R < 4 ? R : 4); w <<= 1)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (i % (2 * w) == 0) {
            sc[i] = fmaxf(sc[i], sc[i + w]);
            er[i] = fmaxf(er[i], er[i + w]);
          }
      if constexpr (R >= 8) {
        sc[0] = fmaxf(sc[0], shfl_xor_f(sc[0], 16));
        er[0] = fmaxf(er[0], shfl_xor_f(er[0], 16));
      }
      if constexpr (R >= 16) {
        sc[0] = fmaxf(sc[0], shfl_xor_f(sc[0], 32));
        er[0] = fmaxf(er[0], shfl_xor_f(er[0], 32));
      }
      const bool in = j + col < j1 && j + col >= a.n_first;
#pragma unroll
      for (int i = 0; i < 4; i += (R < 4 ? R : 4)) {
        const int m = 4 * G + i;
        const int qr = m / R;
        if (m % R == 0 && qr < nrow) buf[qr][(j + col) % kFlush] = sc[i];
        if (in) etop = fmaxf(etop, er[i]);
      }
      // every kFlush blocks, and at the end: the scores so far, lane by lane
      if ((j + 16) % kFlush == 0 || j + 16 >= j1) {
        const int k = (j / kFlush) * kFlush + lane;
        __builtin_amdgcn_wave_barrier();
        for (int qr = 0; qr < nrow; ++qr)
          if (k >= max(j0, a.n_first) && k < j1) {
            float* o = a.score + ((size_t)(sr.r0 + i0 + qr) * a.kvh + g) * a.pitch + k;
            *o = h0 ? fmaxf(*o, buf[qr][lane]) : buf[qr][lane];
          }
        __builtin_amdgcn_wave_barrier();
      }
    }
  }
  // one bound for the tile's rows: the largest
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) etop = fmaxf(etop, shfl_xor_f(etop, o));
  if (lane < nrow) em[lane * em_row] = etop;
}

// ---- choice ------------------------------------------------------------------

constexpr int kSelThreads = 256;
constexpr int kSelWaves = kSelThreads / kWave;
constexpr int kSelLds = 8192;  // scores of a row kept in LDS
constexpr int kNear = 64;      // blocks near the border ranked by one wave

// Order-preserving integers: larger value, larger key; +inf the largest.
__device__ __forceinline__ uint32_t key32(float x) {
  const uint32_t u = __float_as_uint(x + 0.0f);  // (-0 and 0 are equal)
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float unkey32(uint32_t k) {
  return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k);
}
__device__ __forceinline__ unsigned long long key64(double x) {
  const unsigned long long u = (unsigned long long)__double_as_longlong(x + 0.0);
  return u >> 63 ? ~u : u | (1ull << 63);
}

struct SelSmem {
  float score[kSelLds];
  int hist[2][256];
  int part[2][kSelWaves];
  unsigned long long bound[2][kSelWaves];
  float emax[kSelWaves];
  int digit, above;
  int list[kNear];
  double sum[kNear];
};

// Sums of x and y over the workgroup's threads before this one, and over all.
struct Scan {
  int x, y, all_x, all_y;
};
__device__ __forceinline__ Scan wg_scan(int x, int y, SelSmem& sm) {
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const int ix = wave_incl_scan(x), iy = wave_incl_scan(y);
  __syncthreads();
  if (lane == 63) {
    sm.part[0][w] = ix;
    sm.part[1][w] = iy;
  }
  __syncthreads();
  Scan s{ix - x, iy - y, 0, 0};
#pragma unroll
  for (int i = 0; i < kSelWaves; ++i) {
    if (i < w) {
      s.x += sm.part[0][i];
      s.y += sm.part[1][i];
    }
    s.all_x += sm.part[0][i];
    s.all_y += sm.part[1][i];
  }
  return s;
}

// The smallest and largest of the threads' l and h, in every thread; `em` as
// well becomes the largest.  Ends with a barrier's worth of order: what was
// stored to LDS before is visible after.
template <class Key>
__device__ __forceinline__ void wg_extremes(Key& l, Key& h, float& em, SelSmem& sm) {
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const Key l2 = __shfl_xor(l, o, kWave), h2 = __shfl_xor(h, o, kWave);
    l = l2 < l ? l2 : l;
    h = h2 > h ? h2 : h;
    em = fmaxf(em, __shfl_xor(em, o, kWave));
  }
  __syncthreads();
  if (lane == 0) {
    sm.bound[0][w] = l;
    sm.bound[1][w] = h;
    sm.emax[w] = em;
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kSelWaves; ++i) {
    l = sm.bound[0][i] < l ? (Key)sm.bound[0][i] : l;
    h = sm.bound[1][i] > h ? (Key)sm.bound[1][i] : h;
    em = fmaxf(em, sm.emax[i]);
  }
}

// The want-th largest key (1 <= want <= number of keys) of those that
// get(i, key) admits, i < n, and how many are larger, given the smallest and
// largest: digits of 8 bits from the highest in which the keys differ, two
// barriers each.
template <class Key, class Get>
__device__ Key kth_largest(int n, int want, Key lo, Key hi, Get get, SelSmem& sm, int& larger) {
  constexpr int kBits = (int)sizeof(Key) * 8;
  const int tid = threadIdx.x, lane = tid & 63;
  larger = 0;
  if (lo == hi) return hi;
  int bits = 64 - __clzll((long long)((unsigned long long)lo ^ hi));  // the keys agree above these
  Key prefix = bits >= kBits ? 0 : (Key)(hi >> bits);
  sm.hist[0][tid] = 0;
  __syncthreads();
  for (int pass = 0; bits > 0; ++pass) {
    int* hist = sm.hist[pass & 1];
    const int take = bits < 8 ? bits : 8;
    const int shift = bits - take;
    sm.hist[~pass & 1][tid] = 0;  // the next pass's
    for (int i = tid; i < n; i += kSelThreads) {
      Key k;
      if (get(i, k) && (bits >= kBits || (Key)(k >> bits) == prefix))
        atomicAdd(&hist[(int)((k >> shift) & ((1 << take) - 1))], 1);
    }
    __syncthreads();
    if (tid < kWave) {  // from the largest digit down, four a lane
      int c[4], sum = 0;
#pragma unroll
      for (int j = 0; j < 4; ++j) sum += c[j] = hist[255 - 4 * lane - j];
      int before = wave_incl_scan(sum) - sum;
      if (before < want - larger && before + sum >= want - larger) {
        int j = 0;
#pragma unroll
        for (int i = 0; i < 3; ++i)
          if (j == i && before + c[i] < want - larger) {
            before += c[i];
            j = i + 1;
          }
        sm.digit = 255 - 4 * lane - j;
        sm.above = before;
      }
    }
    __syncthreads();
    larger += sm.above;
    prefix = (Key)(prefix << take) | (Key)sm.digit;
    bits = shift;
  }
  return prefix;
}

// The score of a block in 64 bits, by a wave: 16 lanes a query head, four heads
// at a time, 16 bytes of a row per lane and step.  Every lane has the result.
template <int DT, int HD>
__device__ __forceinline__ double score64(const char* q, const char* bound, int heads) {
  constexpr int EPL = DT == PKV_F32 ? 4 : 8;
  constexpr int RB = HD * (DT == PKV_F32 ? 4 : 2);
  const int lane = threadIdx.x & 63;
  double best = -INFINITY;
  for (int h0 = 0; h0 < heads; h0 += 4) {
    const int h = min(h0 + (lane >> 4), heads - 1);
    double t = 0.0;
#pragma unroll
    for (int o = (lane & 15) * 16; o < RB; o += 256) {
      float x[EPL], lo[EPL], hi[EPL];
      widen16<DT, EPL>(ld16(q + (size_t)h * RB + o), x);
      widen16<DT, EPL>(ld16(bound + o), lo);
      widen16<DT, EPL>(ld16(bound + RB + o), hi);
#pragma unroll
      for (int e = 0; e < EPL; ++e)
        t = fma((double)x[e], (double)(x[e] > 0.0f ? hi[e] : lo[e]), t);
    }
#pragma unroll
    for (int o = 1; o < 16; o <<= 1) t += __shfl_xor(t, o, kWave);
    best = t > best ? t : best;
  }
#pragma unroll
  for (int o = 16; o < 64; o <<= 1) {
    const double y = __shfl_xor(best, o, kWave);
    best = y > best ? y : best;
  }
  return best;
}

// One workgroup per query row and kv head.  Bound by its chain of digits and
// barriers: 14.4 us for 512 of 750-2000 blocks, 7.4 for 24 of 310-560.
template <int DT, int HD>
__global__ void __launch_bounds__(kSelThreads) choose_kernel(SelectKArgs a) {
  constexpr int RB = HD * (DT == PKV_F32 ? 4 : 2);
  __shared__ SelSmem sm;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int g = blockIdx.x % a.kvh;
  const int slot = blockIdx.x / a.kvh;  // (sequence, row of it)
  const int s = slot / a.max_q, i = slot % a.max_q;
  const int bsl = a.bs_log2;
  const SeqRows sr = seq_rows(a.cu, a.ctx, s, a.total_q);
  if (i == 0 && g == 0 && tid == 0 &&
      (sr.n > a.max_q || row_blocks(sr, sr.n - 1, bsl, INT32_MAX) > a.nb_max))
    atomicOr(a.err, PKV_EBIT_LENGTH);
  if (i >= sr.n) return;
  const size_t row = (size_t)(sr.r0 + i) * a.kvh + g;
  int32_t* out = a.out + row * a.top;
  const int nb = row_blocks(sr, i, bsl, a.nb_max);
  if (nb <= a.top) {
    for (int k = tid; k < a.top; k += kSelThreads) out[k] = k < nb ? k : -1;
    return;
  }
  const int n = nb - a.n_first - a.n_last;         // blocks to rank
  const int want = a.top - a.n_first - a.n_last;   // of which this many are taken
  for (int k = tid; k < a.n_first; k += kSelThreads) out[k] = k;
  for (int k = tid; k < a.n_last; k += kSelThreads)
    out[a.top - a.n_last + k] = nb - a.n_last + k;
  if (want == 0) return;

  const float* score = a.score + row * a.pitch + a.n_first;
  const bool in_lds = n <= kSelLds;
  uint32_t klo = ~0u, khi = 0;
  float em = 0.0f;
  for (int k = tid; k < a.chunks; k += kSelThreads) em = fmaxf(em, a.emax[row * a.chunks + k]);
  constexpr int U = 8;  // loads in flight
  for (int k = tid; k < n; k += U * kSelThreads) {
    float x[U];
#pragma unroll
    for (int u = 0; u < U; ++u) x[u] = score[min(k + u * kSelThreads, n - 1)];
#pragma unroll
    for (int u = 0; u < U; ++u) {  // (the last one again changes nothing)
      if (in_lds) sm.score[min(k + u * kSelThreads, n - 1)] = x[u];
      klo = min(klo, key32(x[u]));
      khi = max(khi, key32(x[u]));
    }
  }
  wg_extremes(klo, khi, em, sm);
  // twice the row's bound, and a little for the border's own rounding below
  const float E2 = 2.02f * (HD + 16) * 0x1p-23f * em;
  auto at = [&](int k) { return in_lds ? sm.score[k] : score[k]; };
  int larger = 0;
  const uint32_t tkey = kth_largest<uint32_t>(
      n, want, klo, khi, [&](int k, uint32_t& key) { key = key32(at(k)); return true; }, sm, larger);
  const float tau = unkey32(tkey);
  // 2: taken, 1: within the bound of the border, 0: not taken.  An infinite
  // score is what it is: above any finite border, also one whose bound is past
  // the largest float.
  const float above = tau < INFINITY ? fminf(tau + E2, 3.402823466e+38f) : tau;
  const float below = tau < INFINITY ? tau - E2 : tau;
  auto cls = [&](int k) {
    const float x = at(k);
    return x > above ? 2 : x >= below ? 1 : 0;
  };
  // consecutive blocks per thread, so one scan gives every place in index order
  const int per = (n + kSelThreads - 1) / kSelThreads;
  const int k0 = min(tid * per, n), k1 = min(k0 + per, n);
  int n2 = 0, n1 = 0;
  for (int k = k0; k < k1; ++k) {
    const int c = cls(k);
    n2 += c == 2;
    n1 += c == 1;
  }
  const Scan sc = wg_scan(n2, n1, sm);
  const int need = want - sc.all_x, near = sc.all_y;  // of the near ones, `need` are taken
  // All of them, or the first ones where they are equal (the 32-bit sums are
  // exact where the bound is 0 or tau infinite); else by their 64-bit sums.
  const bool sum64 = near > need && E2 > 0.0f && tau < INFINITY;
  if (!sum64 || near <= kNear) {
    unsigned long long mask = ~0ull;  // near ones taken (while there are up to 64)
    if (sum64) {
      int j = sc.y;
      for (int k = k0; k < k1; ++k)
        if (cls(k) == 1) sm.list[j++] = k;
      __syncthreads();
      const char* q = a.q + row * a.rtot * (size_t)RB;
      const int32_t* tab = a.tables + (size_t)s * a.mbps + a.n_first;
      for (int e = wave; e < near; e += kSelWaves) {
        int id = tab[sm.list[e]];
        if (id < 0 || id >= a.num_blocks) id = 0;  // as its score (reported there)
        const double t =
            score64<DT, HD>(q, a.bounds + ((size_t)id * a.kvh + g) * 2 * RB, a.rtot);
        if (lane == 0) sm.sum[e] = t;
      }
      __syncthreads();
      const double mine = lane < near ? sm.sum[lane] : -INFINITY;
      int rank = 0;
      for (int e = 0; e < near; ++e) {
        const double y = sm.sum[e];
        rank += y > mine || (y == mine && e < lane);
      }
      mask = __ballot(lane < near && rank < need);
    }
    int p2 = sc.x, p1 = sc.y;  // taken for sure, and near, before block k
    for (int k = k0; k < k1; ++k) {
      const int c = cls(k);
      bool take = c == 2;
      int before = min(p1, need);
      if (sum64) {
        before = __popcll(p1 < 64 ? mask & ((1ull << p1) - 1) : mask);
        if (c == 1) take = mask >> p1 & 1;
      } else if (c == 1) {
        take = p1 < need;
      }
      if (take) out[a.n_first + p2 + before] = a.n_first + k;
      p2 += c == 2;
      p1 += c == 1;
    }
    return;
  }
  // many near ones: their sums go to the workspace, and a second search
  double* again = a.again + row * a.pitch;
  {
    const char* q = a.q + row * a.rtot * (size_t)RB;
    const int32_t* tab = a.tables + (size_t)s * a.mbps + a.n_first;
    for (int b0 = wave * kWave; b0 < n; b0 += kSelThreads) {
      unsigned long long todo = __ballot(b0 + lane < n && cls(min(b0 + lane, n - 1)) == 1);
      while (todo) {  // wave-uniform
        const int k = b0 + __ffsll((long long)todo) - 1;
        todo &= todo - 1;
        int id = tab[k];
        if (id < 0 || id >= a.num_blocks) id = 0;
        const double t =
            score64<DT, HD>(q, a.bounds + ((size_t)id * a.kvh + g) * 2 * RB, a.rtot);
        if (lane == 0) again[k] = t;
      }
    }
    __syncthreads();  // (read back by this workgroup only)
  }
  auto get = [&](int k, unsigned long long& key) {
    if (cls(k) != 1) return false;
    key = key64(again[k]);
    return true;
  };
  unsigned long long lo64 = ~0ull, hi64 = 0;
  for (int k = tid; k < n; k += kSelThreads) {
    unsigned long long key;
    if (get(k, key)) {
      lo64 = key < lo64 ? key : lo64;
      hi64 = key > hi64 ? key : hi64;
    }
  }
  wg_extremes(lo64, hi64, em, sm);
  int more = 0;
  const unsigned long long kappa =
      kth_largest<unsigned long long>(n, need, lo64, hi64, get, sm, more);
  const int ties = need - more;  // of those equal to kappa, lowest index first
  int taken = 0, equal = 0;
  for (int k = k0; k < k1; ++k) {
    unsigned long long key;
    const int c = cls(k);
    taken += c == 2 || (c == 1 && get(k, key) && key > kappa);
    equal += c == 1 && get(k, key) && key == kappa;
  }
  const Scan s2 = wg_scan(taken, equal, sm);
  int p2 = s2.x, p1 = s2.y;
  for (int k = k0; k < k1; ++k) {
    unsigned long long key = 0;
    const int c = cls(k);
    if (c == 1) (void)get(k, key);
    const bool eq = c == 1 && key == kappa, sure = c == 2 || (c == 1 && key > kappa);
    if (sure || (eq && p1 < ties)) out[a.n_first + p2 + min(p1, ties)] = a.n_first + k;
    p2 += sure;
    p1 += eq;
  }
}

template <int DT, int HD>
hipError_t launch_score(int R, const SelectKArgs& a, long long waves, hipStream_t s) {
  if (!grid_fits((waves + 3) / 4, 256)) return hipErrorInvalidValue;
  const unsigned grid = (unsigned)((waves + 3) / 4);
  switch (R) {
    case 1: score_kernel<DT, HD, 1><<<grid, 256, 0, s>>>(a); break;
    case 2: score_kernel<DT, HD, 2><<<grid, 256, 0, s>>>(a); break;
    case 4: score_kernel<DT, HD, 4><<<grid, 256, 0, s>>>(a); break;
    case 8: score_kernel<DT, HD, 8><<<grid, 256, 0, s>>>(a); break;
    default: score_kernel<DT, HD, 16><<<grid, 256, 0, s>>>(a); break;
  }
  return hipGetLastError();
}

template <int DT>
hipError_t launch_select_dt(int HD, int R, const SelectKArgs& a, long long waves,
                            hipStream_t s) {
  const unsigned rows = (unsigned)((long long)a.n_seqs * a.max_q * a.kvh);
  hipError_t e;
  switch (HD) {
    case 64:
      if ((e = launch_score<DT, 64>(R, a, waves, s)) != hipSuccess) return e;
      choose_kernel<DT, 64><<<rows, kSelThreads, 0, s>>>(a);
      break;
    case 128:
      if ((e = launch_score<DT, 128>(R, a, waves, s)) != hipSuccess) return e;
      choose_kernel<DT, 128><<<rows, kSelThreads, 0, s>>>(a);
      break;
    default:
      if ((e = launch_score<DT, 256>(R, a, waves, s)) != hipSuccess) return e;
      choose_kernel<DT, 256><<<rows, kSelThreads, 0, s>>>(a);
      break;
  }
  return hipGetLastError();
}

int log2_of(int x) {
  int r = 0;
  while ((1 << r) < x) ++r;
  return r;
}

size_t round256(size_t x) { return (x + 255) / 256 * 256; }

// Layout of a call's workspace.
struct SelectPlan {
  int R, tiles, per, chunks, nb_max, pitch;
  long long waves;
  size_t score, emax, again, bytes;
};

SelectPlan select_plan(const pkv_pool* p, const SelectArgs& a) {
  SelectPlan pl{};
  const int bsl = log2_of(p->block_size);
  pl.R = group_width(a.n_head / p->n_kv_head);
  pl.tiles = (a.max_q_len + 16 / pl.R - 1) / (16 / pl.R);
  pl.nb_max = (int)std::min<long long>(((long long)a.max_context_len + p->block_size - 1) >> bsl,
                                       a.max_blocks_per_seq);
  // 64 blocks per wave; fewer while that leaves fewer than 2048 waves
  const long long rows = (long long)a.n_seqs * pl.tiles * p->n_kv_head;
  pl.per = 64;
  while (pl.per > 16 && rows * ((pl.nb_max + pl.per - 1) / pl.per) < 2048) pl.per >>= 1;
  pl.chunks = (pl.nb_max + pl.per - 1) / pl.per;
  pl.waves = rows * pl.chunks;
  const size_t pairs = (size_t)a.total_q * p->n_kv_head;
  pl.score = 0;
  pl.pitch = (pl.nb_max + kFlush - 1) / kFlush * kFlush;
  pl.emax = round256(pairs * pl.pitch * 4);
  pl.again = pl.emax + round256(pairs * pl.chunks * 4);
  pl.bytes = pl.again + round256(pairs * pl.pitch * 8);
  return pl;
}

}  // namespace

size_t select_workspace_bytes(const pkv_pool* p, const SelectArgs& a) {
  return select_plan(p, a).bytes;
}

bool select_fits(const pkv_pool* p, const SelectArgs& a) {
  return grid_fits((select_plan(p, a).waves + 3) / 4, 256) &&
         grid_fits((long long)a.n_seqs * a.max_q_len * p->n_kv_head, kSelThreads);
}

hipError_t launch_select(const pkv_pool* p, const void* bounds, const SelectArgs& a, char* ws,
                         hipStream_t stream) {
  const SelectPlan pl = select_plan(p, a);
  SelectKArgs k{};
  k.q = static_cast<const char*>(a.q);
  k.bounds = static_cast<const char*>(bounds);
  k.tables = a.block_tables;
  k.mbps = a.max_blocks_per_seq;
  k.cu = a.cu_q_lens;
  k.ctx = a.context_lens;
  k.n_seqs = a.n_seqs;
  k.total_q = a.total_q;
  k.tiles = pl.tiles;
  k.chunks = pl.chunks;
  k.per = pl.per;
  k.nb_max = pl.nb_max;
  k.pitch = pl.pitch;
  k.num_blocks = p->num_blocks;
  k.bs_log2 = log2_of(p->block_size);
  k.kvh = p->n_kv_head;
  k.rtot = a.n_head / p->n_kv_head;
  k.top = a.top_blocks;
  k.n_first = a.first_blocks;
  k.n_last = a.last_blocks;
  k.max_q = a.max_q_len;
  k.score = reinterpret_cast<float*>(ws + pl.score);
  k.emax = reinterpret_cast<float*>(ws + pl.emax);
  k.again = reinterpret_cast<double*>(ws + pl.again);
  k.out = a.blocks;
  k.err = p->err;
  switch (p->dtype) {
    case PKV_F32: return launch_select_dt<PKV_F32>(p->head_dim, pl.R, k, pl.waves, stream);
    case PKV_F16: return launch_select_dt<PKV_F16>(p->head_dim, pl.R, k, pl.waves, stream);
    default: return launch_select_dt<PKV_BF16>(p->head_dim, pl.R, k, pl.waves, stream);
  }
}

namespace {
template <int DT>
hipError_t launch_bounds_dt(int HD, const BoundsKArgs& a, unsigned grid, hipStream_t s) {
  switch (HD) {
    case 64: bounds_kernel<DT, 64><<<grid, 256, 0, s>>>(a); break;
    case 128: bounds_kernel<DT, 128><<<grid, 256, 0, s>>>(a); break;
    default: bounds_kernel<DT, 256><<<grid, 256, 0, s>>>(a); break;
  }
  return hipGetLastError();
}

// Blocks that max_new_len consecutive positions can touch, within the tables.
int bounds_span(const pkv_pool* p, int max_new_len, int mbps) {
  return (int)std::min<long long>(((long long)max_new_len + p->block_size - 2) / p->block_size + 1,
                                  mbps);
}
long long bounds_grid(const pkv_pool* p, int n_seqs, int max_new_len, int mbps) {
  const long long cpr = (long long)p->n_kv_head * (p->row_bytes / 16);
  return ((long long)n_seqs * bounds_span(p, max_new_len, mbps) * cpr + 255) / 256;
}
}  // namespace

bool bounds_fits(const pkv_pool* p, int n_seqs, int max_new_len, int mbps) {
  return grid_fits(bounds_grid(p, n_seqs, max_new_len, mbps), 256);
}

hipError_t launch_bounds(const pkv_pool* p, int layer, void* bounds, const int32_t* tables,
                         int mbps, const int32_t* first, const int32_t* ctx, int n_seqs,
                         int max_new_len, hipStream_t stream) {
  BoundsKArgs k{};
  k.k_pool = p->layer_k(layer);
  k.bounds = static_cast<char*>(bounds);
  k.tables = tables;
  k.mbps = mbps;
  k.first = first;
  k.ctx = ctx;
  k.n_seqs = n_seqs;
  k.span = bounds_span(p, max_new_len, mbps);
  k.max_new = max_new_len;
  k.num_blocks = p->num_blocks;
  k.bs_log2 = log2_of(p->block_size);
  k.kvh = p->n_kv_head;
  k.err = p->err;
  const unsigned grid = (unsigned)bounds_grid(p, n_seqs, max_new_len, mbps);
  switch (p->dtype) {
    case PKV_F32: return launch_bounds_dt<PKV_F32>(p->head_dim, k, grid, stream);
    case PKV_F16: return launch_bounds_dt<PKV_F16>(p->head_dim, k, grid, stream);
    default: return launch_bounds_dt<PKV_BF16>(p->head_dim, k, grid, stream);
  }
}

}  // namespace pkv
