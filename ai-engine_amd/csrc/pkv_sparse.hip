// pkv_sparse.hip -- paged attention over chosen blocks (gfx950).
//
// Query row r of a sequence (single decode tokens, or the rows of a short
// chunk) attends, for kv head g, the keys of its context that lie in the
// blocks listed for (r, g):
//   out_h = sum_k softmax_k(scale q_h . k) v_k,  k over those keys.
//
// Bound by HBM: every listed block's K and V rows of a head (2 bs hd
// elements) are read once for the group's query heads.  The list is laid out
// as one run of tokens and cut into parts, a wavefront each, as the decode
// kernel cuts a context; a wave's tiles, matrix instructions, online softmax
// and P.V are those of pkv_decode.hip.  What differs is where a token is:
//  - a wave reads its slice of the list, then the table entries of those
//    blocks (two dependent loads in place of one), and moves the valid ones
//    to the front, so an entry that is no block costs nothing;
//  - each block has its own number of keys, since the context may end in any
//    of them: tokens past it read the block's last key with weight 0.
// Every row's list is equally long, so parts are the same for all rows and
// need no context lengths in the merge.
#include <algorithm>

#include "pkv_decode_dev.h"

namespace pkv {
namespace {

struct SparseKArgs {
  const char* k_pool;
  const char* v_pool;
  const char* q;  // [total_q][n_head][hd]
  void* out;
  int out_f32;
  const int32_t* blocks;  // [total_q][kvh][top]
  int top;
  const int32_t* tables;
  int mbps;
  const int32_t* cu;  // null: one row per sequence
  const int32_t* ctx;
  int n_seqs;
  int total_q;
  int max_q;
  int kvh;
  int num_blocks;
  int bs_log2;
  int part_tokens;
  int parts;
  float scale_log2;
  float* part_ml;
  float* part_o;
  uint32_t* err;
  int rq;  // query heads of this launch per group, h0 .. h0 + rq - 1 of rtot
  int rtot;
  int h0;
};

// Running maxima never go below this, so a tile without a valid token has
// weights 2^(-inf) = 0 and not 2^(inf - inf).
constexpr float kLowest = -3.0e38f;

struct RowAt {
  int row, keys;  // row < 0: none
};
__device__ __forceinline__ RowAt row_at(const SparseKArgs& a, int s, int i) {
  if (!a.cu) return {s, a.ctx[s]};
  const int r0 = min(max(a.cu[s], 0), a.total_q), r1 = min(max(a.cu[s + 1], r0), a.total_q);
  if (i >= r1 - r0) return {-1, 0};
  const long long keys = (long long)a.ctx[s] - (r1 - r0) + i + 1;
  return {r0 + i, (int)(keys > 0 ? keys : 0)};
}

template <int DT, int HD, int R>
struct SparseSmem {
  using C = DCfg<DT, HD, R, false>;
  float p[kWavesPerBlock][C::TILE * C::PP];
};

// SB: block_size below 16, the tokens of a sub-tile span several blocks.
// ONCE: one row per sequence, so no other wave reads a block's rows of a head,
// and the loads say so.  The rows of a chunk choose much the same blocks: their
// loads stay in the caches (42 rows of 12 chunks, 64 heads of 128, 75 blocks
// each: 40 us against 50 with such loads; the other way 64 single rows of 128
// blocks, 32 heads: 98 against 86).
template <int DT, int HD, int R, bool SB, bool ONCE>
__global__ void __launch_bounds__(kWavesPerBlock * kWave) sparse_kernel(SparseKArgs a) {
  using C = DCfg<DT, HD, R, false>;
  __shared__ SparseSmem<DT, HD, R> sm;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lane = threadIdx.x & 63;
  float* p_lds = sm.p[wave];
  const int H = a.kvh * a.rtot;
  const int lg = a.bs_log2, BS = 1 << lg, tmask = BS - 1;
  // item = ((sequence, row of it), part, kv head), the head fastest
  const unsigned item = blockIdx.x * kWavesPerBlock + wave;
  const unsigned rest = item / (unsigned)a.kvh;
  const int g = (int)(item - rest * (unsigned)a.kvh);
  const unsigned slot = rest / (unsigned)a.parts;
  const int p = (int)(rest - slot * (unsigned)a.parts);
  const unsigned s = slot / (unsigned)a.max_q;
  const int i = (int)(slot - s * (unsigned)a.max_q);
  if (s >= (unsigned)a.n_seqs) return;
  const RowAt at = row_at(a, (int)s, i);
  if (at.row < 0) return;
  const int b = at.row;
  const size_t pair = (size_t)b * a.kvh + g;

  const int G = lane >> 4, col = lane & 15;
  const int c = lane % C::CH;   // 16-byte chunk of a row (PV / output mapping)
  const int tg = lane / C::CH;  // token group of a V load
  const int PT = a.part_tokens;
  const int u0 = p * PT;
  const int e0 = u0 >> lg;    // the part's first list entry
  const int o0 = u0 & tmask;  // and offset in it (parts shorter than a block)
  const int span = PT >> lg > 1 ? PT >> lg : 1;  // entries, at most 64
  int sel = -1;
  if (lane < span && e0 + lane < a.top) sel = a.blocks[pair * a.top + e0 + lane];
  u32x4 qf[C::NF];
  {
    const char* qrow = a.q + ((size_t)b * H + g * a.rtot + a.h0 + (col < a.rq ? col : 0)) * C::RB;
#pragma unroll
    for (int f = 0; f < C::NF; ++f)
      qf[f] = col < a.rq ? ld16(qrow + 64 * f + 16 * G) : u32x4{0, 0, 0, 0};
  }
  const bool too_long = (long long)at.keys > (long long)a.mbps << lg;
  const int keys = too_long ? a.mbps << lg : at.keys;
  const int nb = (int)(((long long)keys + tmask) >> lg);
  bool valid = sel >= 0 && sel < nb;
  bool odd = sel >= nb;  // no block of this context
  int id = 0;
  if (valid) {
    id = a.tables[(size_t)s * a.mbps + sel];
    if (id < 0 || id >= a.num_blocks) valid = false, odd = true;
  }
  if (odd) atomicOr(a.err, PKV_EBIT_BLOCK);
  if (too_long && lane == 0) atomicOr(a.err, PKV_EBIT_LENGTH);
  int lim = valid ? min(BS, keys - (sel << lg)) : 0;  // the block's keys
  valid = lim > o0;
  const unsigned long long have = __ballot(valid);
  const int nv = __popcll(have);

  // where the part's result goes
  float* ml = a.part_ml + (pair * a.parts + p) * kMlFloats;
  float* po = a.part_o + (pair * a.parts + p) * R * HD;
  if (nv == 0) {
    if (a.parts > 1) {  // (the merge reads no rows of a part whose l is 0)
      if (lane < kMlFloats) ml[lane] = lane & 1 ? 0.0f : kLowest;
    } else if (lane < C::CH) {
      float z[C::EPL];
#pragma unroll
      for (int e = 0; e < C::EPL; ++e) z[e] = 0.0f;
      for (int h = 0; h < a.rq; ++h)
        store_out<C::EPL>(a.out, ((size_t)b * H + g * a.rtot + a.h0 + h) * HD + c * C::EPL,
                          a.out_f32, DT, z);
    }
    return;
  }
  // valid entries to the front, the others behind them
  {
    const int below = __builtin_amdgcn_mbcnt_hi((uint32_t)(have >> 32),
                                                __builtin_amdgcn_mbcnt_lo((uint32_t)have, 0));
    const int to = (valid ? below : nv + lane - below) << 2;
    id = __builtin_amdgcn_ds_permute(to, id);
    lim = __builtin_amdgcn_ds_permute(to, lim);
  }
  // tokens 0 .. T - 1 of the part: token t is at offset (t + o0) % BS of entry
  // (t + o0) / BS
  const int T = o0 || PT < BS ? min(PT, readlane_i(lim, 0) - o0)
                              : ((nv - 1) << lg) + readlane_i(lim, nv - 1);

  const size_t head_off = (size_t)g * C::RB;
  const size_t slot_stride = (size_t)a.kvh * C::RB;
  const char* kh = a.k_pool + head_off;
  const char* vh = a.v_pool + head_off;
  const size_t blk_stride = (size_t)BS * slot_stride;
  auto ld = [](const char* x) { return ONCE ? ld16_stream(x) : ld16(x); };
  auto lane_of = [&](int v, int t) {
    return __builtin_amdgcn_ds_bpermute(((t + o0) >> lg) << 2, v);
  };
  // Row of token t in `pool`; t0: a wave-uniform token of the same block.
  auto row_of = [&](const char* pool, int t0, int t) {
    const int off = (t + o0) & tmask;
    if constexpr (SB)
      return pool + (size_t)lane_of(id, t) * blk_stride +
             (uint32_t)(min(off, lane_of(lim, t) - 1) * slot_stride);
    const int e = (t0 + o0) >> lg;
    return pool + (size_t)readlane_i(id, e) * blk_stride +
           (uint32_t)(min(off, readlane_i(lim, e) - 1) * slot_stride);
  };
  auto k_row = [&](int tile_base, int st) {
    const int t0 = min(tile_base + 16 * st, T - 1);
    return row_of(kh, t0, min(tile_base + 16 * st + col, T - 1)) + 16 * G;
  };
  auto v_chunk = [&](int tile_base, int k) {
    const int t0 = min(tile_base + k * C::TPL, T - 1);
    return row_of(vh, t0, min(tile_base + k * C::TPL + tg, T - 1)) + 16 * c;
  };
  // whether token t (sub-tile token t0 + col) is attended
  auto live = [&](int t0, int t) {
    const int off = (t + o0) & tmask;
    if constexpr (SB) {
      const int l = lane_of(lim, min(t, T - 1));
      return t < T && off < l;
    }
    return t < T && off < readlane_i(lim, (min(t0, T - 1) + o0) >> lg);
  };

  float m[4], lsum[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    m[j] = kLowest;
    lsum[j] = 0.0f;
  }
  float o[R][C::EPL];
#pragma unroll
  for (int h = 0; h < R; ++h)
#pragma unroll
    for (int e = 0; e < C::EPL; ++e) o[h][e] = 0.0f;

  const int ntiles = (T + C::TILE - 1) / C::TILE;
  u32x4 kf[C::NST][C::NF];
  u32x4 vf[C::NV];
#pragma unroll
  for (int st = 0; st < C::NST; ++st) {
    const char* r = k_row(0, st);
#pragma unroll
    for (int f = 0; f < C::NF; ++f) kf[st][f] = ld(r + 64 * f);
  }
#pragma unroll
  for (int k = 0; k < C::NV; ++k) vf[k] = ld(v_chunk(0, k));

  // One tile, the next one's loads issued as the registers come free.
  auto tile_body = [&](const int tile_base, auto prefetch) {
    constexpr bool PF = decltype(prefetch)::value;
    const int next = tile_base + C::TILE;
    f32x4 acc[C::NST];
#pragma unroll
    for (int st = 0; st < C::NST; ++st) {
      acc[st] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int f = 0; f < C::NF; ++f) mfma_frag<DT>(qf[f], kf[st][f], acc[st]);
      if constexpr (PF) {
        const char* r = k_row(next, st);
#pragma unroll
        for (int f = 0; f < C::NF; ++f) kf[st][f] = ld(r + 64 * f);
      }
    }
    float sc[C::NST][4];
#pragma unroll
    for (int st = 0; st < C::NST; ++st) {
      const int t0 = tile_base + 16 * st;
      const bool ok = live(t0, t0 + col);
#pragma unroll
      for (int j = 0; j < 4; ++j) sc[st][j] = ok ? acc[st][j] * a.scale_log2 : -INFINITY;
    }
    float alpha[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      float tmax = sc[0][j];
#pragma unroll
      for (int st = 1; st < C::NST; ++st) tmax = fmaxf(tmax, sc[st][j]);
      tmax = row_max16(tmax);
      const float mnew = fmaxf(m[j], tmax);
      alpha[j] = fast_exp2(m[j] - mnew);
      m[j] = mnew;
      float ssum = 0.0f;
#pragma unroll
      for (int st = 0; st < C::NST; ++st) {
        sc[st][j] = fast_exp2(sc[st][j] - mnew);
        ssum += sc[st][j];
      }
      lsum[j] = lsum[j] * alpha[j] + ssum;
    }
    if (G < C::RG) {
#pragma unroll
      for (int st = 0; st < C::NST; ++st)
        *reinterpret_cast<f32x4*>(p_lds + (16 * st + col) * C::PP + 4 * G) =
            f32x4{sc[st][0], sc[st][1], sc[st][2], sc[st][3]};
    }
    __builtin_amdgcn_wave_barrier();
    // the running sums follow a new maximum (after the first tiles seldom)
    if (__any(alpha[0] != 1.0f || alpha[1] != 1.0f || alpha[2] != 1.0f || alpha[3] != 1.0f)) {
#pragma unroll
      for (int h = 0; h < R; ++h) {
        const float ah = readlane_f(alpha[h & 3], 16 * (h >> 2));
#pragma unroll
        for (int e = 0; e < C::EPL; ++e) o[h][e] *= ah;
      }
    }
#pragma unroll
    for (int k = 0; k < C::NV; ++k) {
      const float* pr = p_lds + (k * C::TPL + tg) * C::PP;
      float ph[R];
      if constexpr (R >= 4) {
#pragma unroll
        for (int h = 0; h < R; h += 4) {
          const f32x4 t4 = *reinterpret_cast<const f32x4*>(pr + h);
          ph[h] = t4[0];
          ph[h + 1] = t4[1];
          ph[h + 2] = t4[2];
          ph[h + 3] = t4[3];
        }
      } else {
#pragma unroll
        for (int h = 0; h < R; ++h) ph[h] = pr[h];
      }
      float x[C::EPL];
      widen16<DT, C::EPL>(vf[k], x);
      if constexpr (PF) vf[k] = ld(v_chunk(next, k));
#pragma unroll
      for (int h = 0; h < R; ++h)
#pragma unroll
        for (int e = 0; e < C::EPL; ++e) o[h][e] = fmaf(ph[h], x[e], o[h][e]);
    }
    __builtin_amdgcn_wave_barrier();
  };
  for (int t = 0; t + 1 < ntiles; ++t) tile_body(t * C::TILE, std::true_type{});
  tile_body((ntiles - 1) * C::TILE, std::false_type{});

  // sums over the token groups; every group then holds the full row
  constexpr int NG = 64 / C::CH;
#pragma unroll
  for (int j = 0; j < 4; ++j) lsum[j] = row_sum16(lsum[j]);
#pragma unroll
  for (int h = 0; h < R; ++h)
#pragma unroll
    for (int e = 0; e < C::EPL; ++e) o[h][e] = group_sum<C::CH>(o[h][e]);
  float mh[R], lh[R];
#pragma unroll
  for (int h = 0; h < R; ++h) {
    mh[h] = readlane_f(m[h & 3], 16 * (h >> 2));
    lh[h] = readlane_f(lsum[h & 3], 16 * (h >> 2));
  }
  if (a.parts == 1) {
#pragma unroll
    for (int h = 0; h < R; ++h) {
      if (h % NG != tg || h >= a.rq) continue;
      const float inv = lh[h] == 0.0f ? 0.0f : 1.0f / lh[h];
      float x[C::EPL];
#pragma unroll
      for (int e = 0; e < C::EPL; ++e) x[e] = o[h][e] * inv;
      store_out<C::EPL>(a.out, ((size_t)b * H + g * a.rtot + a.h0 + h) * HD + c * C::EPL,
                        a.out_f32, DT, x);
    }
    return;
  }
  // partials in whole lines, as the decode kernel's: quad j of a lane's
  // elements goes to float 4 CH j + 4 c of the head's partial row
#pragma unroll
  for (int h = 0; h < R; ++h) {
    if (h % NG != tg || h >= a.rq) continue;
#pragma unroll
    for (int e = 0; e < C::EPL; e += 4)
      __builtin_nontemporal_store(f32x4{o[h][e], o[h][e + 1], o[h][e + 2], o[h][e + 3]},
                                  reinterpret_cast<f32x4*>(po + h * HD + C::CH * e + 4 * c));
  }
  if (lane < kMlFloats) {
    float v = 0.0f;
#pragma unroll
    for (int h = 0; h < R; ++h)
      if ((lane >> 1) == h) v = (lane & 1) ? lh[h] : mh[h];
    __builtin_nontemporal_store(v, ml + lane);
  }
}

// Joins the parts: M = max m_p, L = sum l_p 2^(m_p - M), O = sum O_p 2^(m_p - M) / L;
// L = 0 (no key at all) gives a zero row.  One wave per query head: HD / 4
// lanes read a partial row, 64 / (HD / 4) rows per load, U loads in flight; the
// first ones and the (m, l) pairs of up to 64 parts go out together.
template <int HD>
__global__ void __launch_bounds__(kWavesPerBlock * kWave)
    sparse_merge_kernel(SparseKArgs a, int R, int dt) {
  constexpr int LPR = HD / 4;
  constexpr int PPI = kWave / LPR;
  constexpr int U = HD == 64 ? 4 : 8;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lane = threadIdx.x & 63;
  const unsigned qh = blockIdx.x * kWavesPerBlock + wave;
  const unsigned sp = qh / (unsigned)a.rq;  // ((sequence, row), kv head)
  const int h = (int)(qh - sp * (unsigned)a.rq);
  const unsigned slot = sp / (unsigned)a.kvh;
  const int g = (int)(sp - slot * (unsigned)a.kvh);
  const unsigned s = slot / (unsigned)a.max_q;
  if (s >= (unsigned)a.n_seqs) return;
  const RowAt at = row_at(a, (int)s, (int)(slot - s * (unsigned)a.max_q));
  if (at.row < 0) return;
  const size_t pair = (size_t)at.row * a.kvh + g;
  const float* ml = a.part_ml + pair * a.parts * kMlFloats + 2 * h;
  const int q = lane / LPR, c = lane % LPR;
  const float* po = a.part_o + (pair * a.parts * R + h) * HD + 4 * c;
  const size_t row = (size_t)R * HD;
  f32x4 ov[U];
  auto load = [&](int p0) {
#pragma unroll
    for (int u = 0; u < U; ++u)
      ov[u] = *reinterpret_cast<const f32x4*>(po + (size_t)min(p0 + u * PPI + q, a.parts - 1) * row);
  };
  load(0);
  float m0 = kLowest, l0 = 0.0f;  // part `lane`
  if (lane < a.parts) {
    m0 = ml[(size_t)lane * kMlFloats];
    l0 = ml[(size_t)lane * kMlFloats + 1];
  }
  float M = m0;
  for (int p = kWave + lane; p < a.parts; p += kWave) M = fmaxf(M, ml[(size_t)p * kMlFloats]);
#pragma unroll
  for (int x = 1; x < 64; x <<= 1) M = fmaxf(M, shfl_xor_f(M, x));
  const float w0 = fast_exp2(m0 - M);
  float L = w0 * l0;
  for (int p = kWave + lane; p < a.parts; p += kWave)
    L += fast_exp2(ml[(size_t)p * kMlFloats] - M) * ml[(size_t)p * kMlFloats + 1];
#pragma unroll
  for (int x = 1; x < 64; x <<= 1) L += shfl_xor_f(L, x);
  f32x4 acc = {0, 0, 0, 0};
  for (int p0 = 0; p0 < a.parts; p0 += PPI * U) {
    if (p0) load(p0);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int p = p0 + u * PPI + q;
      // weight and l of the part; one without a key (l = 0) wrote no rows
      float w = __int_as_float(__builtin_amdgcn_ds_bpermute((p & 63) << 2, __float_as_int(w0)));
      float l = __int_as_float(__builtin_amdgcn_ds_bpermute((p & 63) << 2, __float_as_int(l0)));
      if (p >= kWave && p < a.parts) {
        w = fast_exp2(ml[(size_t)p * kMlFloats] - M);
        l = ml[(size_t)p * kMlFloats + 1];
      }
      if (p < a.parts && l != 0.0f)
#pragma unroll
        for (int k = 0; k < 4; ++k) acc[k] = fmaf(w, ov[u][k], acc[k]);
    }
  }
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    if constexpr (LPR <= 16) acc[k] += shfl_xor_f(acc[k], 16);
    if constexpr (LPR <= 32) acc[k] += shfl_xor_f(acc[k], 32);
  }
  if (lane >= LPR) return;
  const float inv = L == 0.0f ? 0.0f : 1.0f / L;
  // chunk c of a partial row holds elements (c % CH) EPL + 4 (c / CH) ..
  const int epl = dt == PKV_F32 ? 4 : 8;
  const int chs = HD / epl;
  const size_t eo = ((size_t)at.row * a.kvh * a.rtot + g * a.rtot + a.h0 + h) * HD +
                    (c % chs) * epl + 4 * (c / chs);
  if (a.out_f32) {
    *reinterpret_cast<f32x4*>(reinterpret_cast<float*>(a.out) + eo) =
        f32x4{acc[0] * inv, acc[1] * inv, acc[2] * inv, acc[3] * inv};
  } else {
    uint32_t w[4];
#pragma unroll
    for (int k = 0; k < 4; ++k)
      w[k] = dt == PKV_BF16 ? f32_to_bf16_bits(acc[k] * inv) : f32_to_f16_bits(acc[k] * inv);
    typedef unsigned int u32x2 __attribute__((ext_vector_type(2)));
    *reinterpret_cast<u32x2*>(reinterpret_cast<uint16_t*>(a.out) + eo) =
        u32x2{w[0] | (w[1] << 16), w[2] | (w[3] << 16)};
  }
}

template <int DT, int HD, int R>
void launch_main(const SparseKArgs& k, unsigned grid, hipStream_t s) {
  constexpr int kThreads = kWavesPerBlock * kWave;
  if (k.bs_log2 < 4) sparse_kernel<DT, HD, R, true, false><<<grid, kThreads, 0, s>>>(k);
  else if (k.max_q > 1) sparse_kernel<DT, HD, R, false, false><<<grid, kThreads, 0, s>>>(k);
  else sparse_kernel<DT, HD, R, false, true><<<grid, kThreads, 0, s>>>(k);
}

template <int DT, int HD>
hipError_t launch_r(int R, const SparseKArgs& k, unsigned grid, hipStream_t s) {
  switch (R) {
    case 1: launch_main<DT, HD, 1>(k, grid, s); break;
    case 2: launch_main<DT, HD, 2>(k, grid, s); break;
    case 4: launch_main<DT, HD, 4>(k, grid, s); break;
    case 8: launch_main<DT, HD, 8>(k, grid, s); break;
    default: launch_main<DT, HD, 16>(k, grid, s); break;
  }
  return hipGetLastError();
}

template <int DT>
hipError_t launch_hd(int HD, int R, const SparseKArgs& k, unsigned grid, hipStream_t s) {
  switch (HD) {
    case 64: return launch_r<DT, 64>(R, k, grid, s);
    case 128: return launch_r<DT, 128>(R, k, grid, s);
    default: return launch_r<DT, 256>(R, k, grid, s);
  }
}

struct SparsePlan {
  int bs_log2, part_tokens, parts, R;
  size_t ml, bytes;
};

// Parts of 1024 tokens, halved (down to 64) while the call has fewer than
// 1024 waves, one per SIMD, and while a part has more than the 64 list entries of
// a wave.  Eight heads and more keep a wave at P.V for longer, so they get half
// as many waves again.  (us, main kernel and merge, parts of 128 / 256 / 512 /
// 1024: 64 rows of 2048 tokens, 32 heads on 8 of 128: 112 / 101 / 95 / 91; 42 rows
// of 1200, 64 heads: 64 / 57 / 80 / 87.)
SparsePlan sparse_plan(const pkv_pool* p, const SparseArgs& a) {
  SparsePlan pl{};
  while ((1 << pl.bs_log2) < p->block_size) ++pl.bs_log2;
  pl.R = group_width(a.n_head / p->n_kv_head);
  const long long len = (long long)a.top_blocks << pl.bs_log2;
  const long long pairs = (long long)a.total_q * p->n_kv_head;
  int pt = 1024;
  while (pt > 64 && pairs * ((len + pt - 1) / pt) < (pl.R < 8 ? 1024 : 1536)) pt >>= 1;
  while (pt > 64 && (pt >> pl.bs_log2) > 64) pt >>= 1;
  pl.part_tokens = pt;
  pl.parts = (int)((len + pt - 1) / pt);
  if (pl.parts > 1) {
    pl.ml = ((size_t)pairs * pl.parts * kMlFloats * 4 + 255) / 256 * 256;
    pl.bytes = pl.ml + (size_t)pairs * pl.parts * pl.R * p->head_dim * 4;
  }
  return pl;
}

long long sparse_items(const pkv_pool* p, const SparseArgs& a, int parts) {
  return (long long)a.n_seqs * a.max_q_len * p->n_kv_head * parts;
}

}  // namespace

size_t sparse_workspace_bytes(const pkv_pool* p, const SparseArgs& a) {
  return sparse_plan(p, a).bytes;
}

bool sparse_fits(const pkv_pool* p, const SparseArgs& a) {
  const SparsePlan pl = sparse_plan(p, a);
  const int heads = std::min(a.n_head / p->n_kv_head, 16);
  return sparse_items(p, a, std::max(pl.parts, heads)) < (1LL << 26) - 4;
}

hipError_t launch_sparse(const pkv_pool* p, int layer, const SparseArgs& a, char* ws,
                         hipStream_t stream) {
  const SparsePlan pl = sparse_plan(p, a);
  SparseKArgs k{};
  k.k_pool = p->layer_k(layer);
  k.v_pool = p->layer_v(layer);
  k.q = static_cast<const char*>(a.q);
  k.out = a.out;
  k.out_f32 = a.out_dtype == PKV_F32;
  k.blocks = a.blocks;
  k.top = a.top_blocks;
  k.tables = a.block_tables;
  k.mbps = a.max_blocks_per_seq;
  k.cu = a.cu_q_lens;
  k.ctx = a.context_lens;
  k.n_seqs = a.n_seqs;
  k.total_q = a.total_q;
  k.max_q = a.max_q_len;
  k.kvh = p->n_kv_head;
  k.num_blocks = p->num_blocks;
  k.bs_log2 = pl.bs_log2;
  k.part_tokens = pl.part_tokens;
  k.parts = pl.parts;
  k.scale_log2 = a.scale * 1.4426950408889634f;
  k.part_ml = reinterpret_cast<float*>(ws);
  k.part_o = reinterpret_cast<float*>(ws + pl.ml);
  k.err = p->err;
  k.rtot = a.n_head / p->n_kv_head;
  const unsigned grid =
      (unsigned)((sparse_items(p, a, pl.parts) + kWavesPerBlock - 1) / kWavesPerBlock);
  // slices of at most 16 query heads per group share the workspace in turn
  for (k.h0 = 0; k.h0 < k.rtot; k.h0 += 16) {
    k.rq = std::min(k.rtot - k.h0, pl.R);
    hipError_t e;
    switch (p->dtype) {
      case PKV_F32: e = launch_hd<PKV_F32>(p->head_dim, pl.R, k, grid, stream); break;
      case PKV_F16: e = launch_hd<PKV_F16>(p->head_dim, pl.R, k, grid, stream); break;
      default: e = launch_hd<PKV_BF16>(p->head_dim, pl.R, k, grid, stream); break;
    }
    if (e != hipSuccess) return e;
    if (pl.parts == 1) continue;
    const unsigned mgrid =
        (unsigned)((sparse_items(p, a, k.rq) + kWavesPerBlock - 1) / kWavesPerBlock);
    switch (p->head_dim) {
      case 64: sparse_merge_kernel<64><<<mgrid, kWavesPerBlock * kWave, 0, stream>>>(k, pl.R, p->dtype); break;
      case 128: sparse_merge_kernel<128><<<mgrid, kWavesPerBlock * kWave, 0, stream>>>(k, pl.R, p->dtype); break;
      default: sparse_merge_kernel<256><<<mgrid, kWavesPerBlock * kWave, 0, stream>>>(k, pl.R, p->dtype); break;
    }
    if ((e = hipGetLastError()) != hipSuccess) return e;
  }
  return hipSuccess;
}

}  // namespace pkv
