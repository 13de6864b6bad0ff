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
// kernel cuts a context.  What differs is where a token is:
//  - a wave reads its slice of the list, then the table entries of those
//    blocks (two dependent loads in place of one), and moves the valid ones
//    to the front, so an entry that is no block costs nothing;
//  - each block has its own number of keys, since the context may end in any
//    of them: tokens past it read the block's last key with weight 0.
// Every row's list is equally long, so parts are the same for all rows and
// need no context lengths in the merge.
//
// Both products of 16-bit pools run on the matrix cores, the heads as the 16
// columns: S^T = K Q^T, O^T = V^T P^T (sparse16_kernel).  f32 pools take the
// decode kernel's way, P.V in f32 multiply-adds (sparse32_kernel).
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
  int width;  // heads a partial has room for
  int joined;  // 16-bit pools: a workgroup's waves are the parts of one (row, kv head)
  int rq;     // query heads of this launch per group, h0 .. h0 + rq - 1 of rtot
  int rtot;
  int h0;
};

// Running maxima never go below this, so a tile without a valid token has
// weights 2^(-inf) = 0 and not 2^(inf - inf).
constexpr float kLowest = -3.0e38f;

struct RowAt {
  int row, keys;  // row < 0: none; keys < 0: none (bounded where it is used: the
                  // list's loads do not wait for the context)
  bool over;      // its chunk has more rows than max_q
};
__device__ __forceinline__ RowAt row_at(const SparseKArgs& a, int s, int i) {
  if (!a.cu) return {s, a.ctx[s], false};
  const int r0 = min(max(a.cu[s], 0), a.total_q), r1 = min(max(a.cu[s + 1], r0), a.total_q);
  if (i >= r1 - r0) return {-1, 0, false};
  const long long keys = (long long)a.ctx[s] - (r1 - r0) + i + 1;
  return {r0 + i, (int)(keys > 0 ? keys : 0), r1 - r0 > a.max_q};
}

// What a wave computes: part p of the list of (row, kv head g).
struct Part {
  int s, row, keys, g, p;
  bool over;    // its chunk has more rows than max_q
  size_t pair;  // row * kvh + g
  int o0;       // offset in its first block (parts shorter than a block)
  int T;        // tokens 0 .. T - 1; token t is at offset (t + o0) % bs of entry (t + o0) / bs
  int id, lim;  // lane e: block and number of keys of entry e
};

// Item = ((sequence, row of it), part, kv head), the head fastest; joined: the
// workgroup's ((sequence, row), kv head) and the wave's part.
__device__ __forceinline__ bool locate(const SparseKArgs& a, int wave, Part& w) {
  const unsigned item = a.joined ? blockIdx.x : blockIdx.x * kWavesPerBlock + wave;
  const unsigned rest = item / (unsigned)a.kvh;
  w.g = (int)(item - rest * (unsigned)a.kvh);
  const unsigned slot = a.joined ? rest : rest / (unsigned)a.parts;
  w.p = a.joined ? wave : (int)(rest - slot * (unsigned)a.parts);
  w.s = (int)(slot / (unsigned)a.max_q);
  if (w.s >= a.n_seqs) return false;
  const RowAt at = row_at(a, w.s, (int)(slot - (unsigned)w.s * (unsigned)a.max_q));
  w.row = at.row;
  w.keys = at.keys;
  w.over = at.over;
  w.pair = (size_t)w.row * a.kvh + w.g;
  return at.row >= 0;
}

// The part's list entries, the valid ones first.  T = 0: no key.
__device__ __forceinline__ void take_list(const SparseKArgs& a, int lane, Part& w) {
  const int lg = a.bs_log2, BS = 1 << lg, tmask = BS - 1, PT = a.part_tokens;
  const int u0 = w.p * PT;
  const int e0 = u0 >> lg;  // the part's first list entry
  w.o0 = u0 & tmask;
  const int span = PT >> lg > 1 ? PT >> lg : 1;  // entries, at most 64
  int sel = -1;
  if (lane < span && e0 + lane < a.top) sel = a.blocks[w.pair * a.top + e0 + lane];
  const bool too_long = (long long)w.keys > (long long)a.mbps << lg;
  const int keys = too_long ? a.mbps << lg : max(w.keys, 0);
  const int nb = (int)(((long long)keys + tmask) >> lg);
  bool valid = sel >= 0 && sel < nb;
  bool odd = sel >= nb;  // no block of this context
  int id = 0;
  if (valid) {
    id = a.tables[(size_t)w.s * a.mbps + sel];
    if (id < 0 || id >= a.num_blocks) valid = false, odd = true;
  }
  if (odd) atomicOr(a.err, PKV_EBIT_BLOCK);
  if ((too_long || w.over) && lane == 0) atomicOr(a.err, PKV_EBIT_LENGTH);
  int lim = valid ? min(BS, keys - (sel << lg)) : 0;  // the block's keys
  valid = lim > w.o0;
  const unsigned long long have = __ballot(valid);
  const int nv = __popcll(have);
  const int below = __builtin_amdgcn_mbcnt_hi((uint32_t)(have >> 32),
                                              __builtin_amdgcn_mbcnt_lo((uint32_t)have, 0));
  const int to = (valid ? below : nv + lane - below) << 2;
  w.id = __builtin_amdgcn_ds_permute(to, id);
  w.lim = __builtin_amdgcn_ds_permute(to, lim);
  w.T = nv == 0                ? 0
        : w.o0 || PT < BS      ? min(PT, readlane_i(w.lim, 0) - w.o0)
                               : ((nv - 1) << lg) + readlane_i(w.lim, nv - 1);
}

// A part without keys: zero rows, or l = 0 for the merge (which reads no rows
// of such a part).
__device__ __forceinline__ void store_nothing(const SparseKArgs& a, const Part& w, int lane, int hd) {
  if (a.parts > 1) {
    float* ml = a.part_ml + (w.pair * a.parts + w.p) * kMlFloats;
    if (lane < kMlFloats) ml[lane] = lane & 1 ? 0.0f : kLowest;
    return;
  }
  const size_t at = (w.pair * a.rtot + a.h0) * hd;
  for (int i = lane; i < a.rq * hd; i += kWave) {
    if (a.out_f32) reinterpret_cast<float*>(a.out)[at + i] = 0.0f;
    else reinterpret_cast<uint16_t*>(a.out)[at + i] = 0;
  }
}

// Rows of a part's tokens in a pool of one kv head.  SB: block_size below 16,
// so the tokens of a sub-tile span several blocks.
template <bool SB>
struct Rows {
  const Part& w;
  int lg, tmask;
  size_t slot_stride, blk_stride;
  __device__ __forceinline__ Rows(const SparseKArgs& a, const Part& p, int row_bytes)
      : w(p), lg(a.bs_log2), tmask((1 << a.bs_log2) - 1), slot_stride((size_t)a.kvh * row_bytes),
        blk_stride(slot_stride << a.bs_log2) {}
  __device__ __forceinline__ int lane_of(int v, int t) const {
    return __builtin_amdgcn_ds_bpermute(((t + w.o0) >> lg) << 2, v);
  }
  // Row of token t; t0: a wave-uniform token of the same block.  Tokens past
  // the block's keys give its last one.
  __device__ __forceinline__ const char* row(const char* pool, int t0, int t) const {
    const int off = (t + w.o0) & tmask;
    if constexpr (SB)
      return pool + (size_t)lane_of(w.id, t) * blk_stride +
             (uint32_t)(min(off, lane_of(w.lim, t) - 1) * slot_stride);
    const int e = (t0 + w.o0) >> lg;
    return pool + (size_t)readlane_i(w.id, e) * blk_stride +
           (uint32_t)(min(off, readlane_i(w.lim, e) - 1) * slot_stride);
  }
  // Row of token base + i of a run of up to 16, in one block without SB.
  __device__ __forceinline__ const char* run(const char* pool, int base, int i) const {
    return row(pool, min(base, w.T - 1), min(base + i, w.T - 1));
  }
  // How many tokens of the 16 from t0 on are attended (not SB).
  __device__ __forceinline__ int live16(int t0) const {
    const int at = t0 + w.o0;
    return t0 < w.T ? min(w.T - t0, readlane_i(w.lim, at >> lg) - (at & tmask)) : 0;
  }
  __device__ __forceinline__ bool live(int t) const {
    const int lim = lane_of(w.lim, min(t, w.T - 1));
    return t < w.T && ((t + w.o0) & tmask) < lim;
  }
};

// ONCE: one row per sequence, so no other wave reads a block's rows of a head,
// and the loads say so.  The rows of a chunk choose much the same blocks: their
// loads stay in the caches (43 rows of 12 chunks, 64 heads of 128, 75 blocks
// each: 35 us against 47 with such loads; the other way 64 single rows of 128
// blocks, 32 heads: 95 against 84).
template <bool ONCE>
__device__ __forceinline__ u32x4 ld_row(const char* x) {
  return ONCE ? ld16_stream(x) : ld16(x);
}

// ---- 16-bit pools ------------------------------------------------------------

template <int HD>
struct Cfg16 {
  static constexpr int RB = HD * 2;
  static constexpr int NF = RB / 64;   // 16-byte fragments per lane of a row
  static constexpr int CH = RB / 16;   // 16-byte chunks of a row
  static constexpr int TPL = 64 / CH;  // tokens per V load
  static constexpr int TILE = 32;      // tokens: two sub-tiles of S^T, one k-step of O^T
  static constexpr int NV = TILE / TPL;
  static constexpr int ND = HD / 16;   // 16-dim tiles of O^T
  static constexpr int VP = RB + 32;   // pitch of a V row in LDS
  static constexpr int LDS = TILE * VP;  // of a wave: its V tile, later its O
  // Most waves of a workgroup: their registers fit with 4, 2 and 1 per SIMD.
  static constexpr int WAVES = HD == 64 ? 16 : HD == 128 ? 8 : 4;
  static_assert(16 * HD * 4 <= LDS, "O of 16 heads");
};

// Weights above 2^kRise raise the running maximum: until then the sums need no
// rescaling.  f16 weights carry 2^kLift more, out of the range of its subnormals.
constexpr float kRise = 8.0f, kLift = 7.0f;

// One wave, 32 tokens a tile.
//  S^T = K Q^T: K fragments from the pool are the A operand (lane: token lane %
//   16, 64 contiguous bytes of a row per four lanes), the heads' Q the B
//   operand, so lane (G, c) gets head c's scores of tokens 4 G .. 4 G + 3 of each
//   sub-tile: the softmax state of a head sits in its column's four lanes.
//  O^T = V^T P^T: those scores are the lane's slice of the B operand as they
//   are, with the k-step's tokens taken in that order; V goes through the wave's
//   LDS and is read transposed.  P enters as the sum of three bf16 parts (24
//   bits) or two f16 ones (22), so the weights lose nothing: error against 64
//   bits as with P.V in f32 multiply-adds, which took 1020 vector instructions a
//   tile at 8 heads of 128.
// The next tile's rows are loaded when this one's scores are there and its V is
// in LDS.
//  Joined: the parts of a (row, kv head), equally long, are one workgroup, and
//   their results meet in LDS: one launch, and no partial leaves the CU.
// 64 single rows of 2048 tokens, 32 heads on 8 of 128: 84 us (537 MB, 6.4 TB/s, bound
// by HBM) and the merge 4.7; 43 chunk rows of 1200, 64 heads: 35 us joined, bound by
// the waves' own steps; 8 rows of 1000, 8 kv heads of 64: 7.2 + 3.4, round trips.
template <int DT, int HD, bool SB, bool ONCE>
__global__ void __launch_bounds__(Cfg16<HD>::WAVES * kWave) sparse16_kernel(SparseKArgs a) {
  using C = Cfg16<HD>;
  extern __shared__ __attribute__((aligned(16))) char v_lds_all[];  // LDS bytes a wave
  __shared__ float ml_lds[C::WAVES][kMlFloats];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lane = threadIdx.x & 63;
  const int G = lane >> 4, col = lane & 15;
  char* v_lds = v_lds_all + wave * C::LDS;
  Part w;
  if (!locate(a, wave, w)) return;
  u32x4 qf[C::NF];
  {
    const char* qrow = a.q + (w.pair * a.rtot + a.h0 + (col < a.rq ? col : 0)) * C::RB;
#pragma unroll
    for (int f = 0; f < C::NF; ++f)
      qf[f] = col < a.rq ? ld16(qrow + 64 * f + 16 * G) : u32x4{0, 0, 0, 0};
  }
  take_list(a, lane, w);
  if (w.T == 0 && !a.joined) {
    store_nothing(a, w, lane, HD);
    return;
  }
  const Rows<SB> rows(a, w, C::RB);
  const char* kh = a.k_pool + (size_t)w.g * C::RB + 16 * G;
  const int c = lane % C::CH, tg = lane / C::CH;
  const char* vh = a.v_pool + (size_t)w.g * C::RB + 16 * c;

  u32x4 kf[2][C::NF], vf[C::NV];
  auto load_k = [&](int base) {
#pragma unroll
    for (int st = 0; st < 2; ++st) {
      const char* r = rows.run(kh, base + 16 * st, col);
#pragma unroll
      for (int f = 0; f < C::NF; ++f) kf[st][f] = ld_row<ONCE>(r + 64 * f);
    }
  };
  auto load_v = [&](int base) {
#pragma unroll
    for (int i = 0; i < C::NV; ++i) vf[i] = ld_row<ONCE>(rows.run(vh, base + i * C::TPL, tg));
  };
  float m = kLowest, l = 0.0f;
  f32x4 o[C::ND];
#pragma unroll
  for (int d = 0; d < C::ND; ++d) o[d] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  if (w.T > 0) {
    load_k(0);
    load_v(0);
  }

  for (int base = 0; base < w.T; base += C::TILE) {
    const bool more = base + C::TILE < w.T;
    f32x4 sc[2];
#pragma unroll
    for (int st = 0; st < 2; ++st) {
      sc[st] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int f = 0; f < C::NF; ++f) mfma_frag<DT>(kf[st][f], qf[f], sc[st]);
    }
    // V rows to LDS: token i TPL + tg of the tile
#pragma unroll
    for (int i = 0; i < C::NV; ++i) st16(v_lds + (i * C::TPL + tg) * C::VP + 16 * c, vf[i]);
    __builtin_amdgcn_wave_barrier();
    if (more) {
      load_v(base + C::TILE);
      load_k(base + C::TILE);
    }
    // scores in the exp2 domain, tokens that are not attended at -inf
#pragma unroll
    for (int st = 0; st < 2; ++st) {
      const int t0 = base + 16 * st;
#pragma unroll
      for (int j = 0; j < 4; ++j) sc[st][j] *= a.scale_log2;
      if constexpr (SB) {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (!rows.live(t0 + 4 * G + j)) sc[st][j] = -INFINITY;
      } else {
        const int n = rows.live16(t0);
        if (n < 16) {  // wave-uniform
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if (4 * G + j >= n) sc[st][j] = -INFINITY;
        }
      }
    }
    float top = fmaxf(fmaxf(sc[0][0], sc[0][1]), fmaxf(sc[0][2], sc[0][3]));
    top = fmaxf(top, fmaxf(fmaxf(sc[1][0], sc[1][1]), fmaxf(sc[1][2], sc[1][3])));
    if (__any(top > m + kRise)) {  // the first tile, and seldom after it
      top = row_group_max(top);
      if (top > m + kRise) {
        const float alpha = fast_exp2(m - top);
        m = top;
        l *= alpha;
#pragma unroll
        for (int d = 0; d < C::ND; ++d) o[d] *= alpha;
      }
    }
    const float shift = DT == PKV_F16 ? kLift - m : -m;
    float p[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      p[i] = fast_exp2(sc[i >> 2][i & 3] + shift);
      l += p[i];
    }
    // the weights' parts as B operands
    constexpr int NP = DT == PKV_BF16 ? 3 : 2;
    u32x4 part[NP];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float x0 = p[2 * i], x1 = p[2 * i + 1];
#pragma unroll
      for (int k = 0; k < NP; ++k) {
        const uint32_t b = cvt_pk16<DT>(x0, x1);
        part[k][i] = b;
        x0 -= DT == PKV_BF16 ? bf16lo(b) : f16lo(b);
        x1 -= DT == PKV_BF16 ? bf16hi(b) : f16hi(b);
      }
    }
    // A operand: lane (dim 16 d + col, group G) needs tokens 4 G .. 4 G + 3 of
    // both sub-tiles.  ds_read_b64_tr_b16 gives lane i of a 16-lane group, element
    // j, the (i & 3)-th value at the address of lane 4 j + (i >> 2).
    typedef short s4 __attribute__((ext_vector_type(4)));
    typedef __attribute__((address_space(3))) s4 lds_s4;
    const char* vt = v_lds + (4 * G + (col >> 2)) * C::VP + 8 * (col & 3);
#pragma unroll
    for (int d = 0; d < C::ND; ++d) {
      const uint2 lo = __builtin_bit_cast(
          uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4*)(vt + 32 * d)));
      const uint2 hi = __builtin_bit_cast(
          uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4*)(vt + 32 * d + 16 * C::VP)));
      const u32x4 va{lo.x, lo.y, hi.x, hi.y};
#pragma unroll
      for (int k = 0; k < NP; ++k) mfma_frag<DT>(va, part[k], o[d]);
    }
    __builtin_amdgcn_wave_barrier();
  }
  l = swap32_sum(swap16_sum(l));

  // lane: head col, dims 16 d + 4 G .. + 3
  auto store = [&](size_t at, const f32x4& x) {
    if (a.out_f32)
      *reinterpret_cast<f32x4*>(reinterpret_cast<float*>(a.out) + at) = x;
    else
      *reinterpret_cast<uint2*>(reinterpret_cast<uint16_t*>(a.out) + at) =
          uint2{cvt_pk16<DT>(x[0], x[1]), cvt_pk16<DT>(x[2], x[3])};
  };
  const size_t out0 = (w.pair * a.rtot + a.h0) * HD;
  if (a.joined) {
    float* mine = reinterpret_cast<float*>(v_lds) + col * HD + 4 * G;
#pragma unroll
    for (int d = 0; d < C::ND; ++d) *reinterpret_cast<f32x4*>(mine + 16 * d) = o[d];
    if (G == 0) {
      ml_lds[wave][2 * col] = m;
      ml_lds[wave][2 * col + 1] = l;
    }
    __syncthreads();
    for (int i = threadIdx.x; i < a.rq * (HD / 4); i += a.parts * kWave) {
      const int h = i / (HD / 4);
      float M = kLowest, L = 0.0f;
      for (int p = 0; p < a.parts; ++p) M = fmaxf(M, ml_lds[p][2 * h]);
      f32x4 acc{0.0f, 0.0f, 0.0f, 0.0f};
      for (int p = 0; p < a.parts; ++p) {
        const float f = fast_exp2(ml_lds[p][2 * h] - M);
        L += f * ml_lds[p][2 * h + 1];
        acc += f * *reinterpret_cast<const f32x4*>(v_lds_all + p * C::LDS + i * 16);
      }
      store(out0 + 4 * i, acc * (L == 0.0f ? 0.0f : 1.0f / L));
    }
    return;
  }
  if (a.parts > 1) {
    float* ml = a.part_ml + (w.pair * a.parts + w.p) * kMlFloats;
    float* po = a.part_o + ((w.pair * a.parts + w.p) * a.width + col) * HD + 4 * G;
    if (G == 0) {
      ml[2 * col] = m;
      ml[2 * col + 1] = l;
    }
    if (col < a.rq) {
#pragma unroll
      for (int d = 0; d < C::ND; ++d) *reinterpret_cast<f32x4*>(po + 16 * d) = o[d];
    }
    return;
  }
  if (col >= a.rq) return;
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
  for (int d = 0; d < C::ND; ++d) store(out0 + col * HD + 16 * d + 4 * G, o[d] * inv);
}

// ---- f32 pools ---------------------------------------------------------------

// The decode kernel's tile: scores on v_mfma_f32_16x16x4f32, P.V in f32
// multiply-adds with the weights handed over through LDS.
template <int HD, int R, bool SB, bool ONCE>
__global__ void __launch_bounds__(kWavesPerBlock * kWave) sparse32_kernel(SparseKArgs a) {
  constexpr int DT = PKV_F32;
  using C = DCfg<DT, HD, R, false>;
  __shared__ float p_lds_all[kWavesPerBlock][C::TILE * C::PP];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lane = threadIdx.x & 63;
  float* p_lds = p_lds_all[wave];
  const int G = lane >> 4, col = lane & 15;
  Part w;
  if (!locate(a, wave, w)) return;
  u32x4 qf[C::NF];
  {
    const char* qrow = a.q + (w.pair * a.rtot + a.h0 + (col < a.rq ? col : 0)) * C::RB;
#pragma unroll
    for (int f = 0; f < C::NF; ++f)
      qf[f] = col < a.rq ? ld16(qrow + 64 * f + 16 * G) : u32x4{0, 0, 0, 0};
  }
  take_list(a, lane, w);
  if (w.T == 0) {
    store_nothing(a, w, lane, HD);
    return;
  }
  const Rows<SB> rows(a, w, C::RB);
  const int c = lane % C::CH;   // 16-byte chunk of a row (PV / output mapping)
  const int tg = lane / C::CH;  // token group of a V load
  const char* kh = a.k_pool + (size_t)w.g * C::RB + 16 * G;
  const char* vh = a.v_pool + (size_t)w.g * C::RB + 16 * c;
  auto k_row = [&](int base, int st) { return rows.run(kh, base + 16 * st, col); };
  auto v_chunk = [&](int base, int k) { return rows.run(vh, base + k * C::TPL, tg); };

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

  const int ntiles = (w.T + C::TILE - 1) / C::TILE;
  u32x4 kf[C::NST][C::NF];
  u32x4 vf[C::NV];
#pragma unroll
  for (int st = 0; st < C::NST; ++st) {
    const char* r = k_row(0, st);
#pragma unroll
    for (int f = 0; f < C::NF; ++f) kf[st][f] = ld_row<ONCE>(r + 64 * f);
  }
#pragma unroll
  for (int k = 0; k < C::NV; ++k) vf[k] = ld_row<ONCE>(v_chunk(0, k));

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
        for (int f = 0; f < C::NF; ++f) kf[st][f] = ld_row<ONCE>(r + 64 * f);
      }
    }
    float sc[C::NST][4];
#pragma unroll
    for (int st = 0; st < C::NST; ++st) {
      const int t0 = tile_base + 16 * st;
      const bool ok = SB ? rows.live(t0 + col) : col < rows.live16(t0);
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
      if constexpr (PF) vf[k] = ld_row<ONCE>(v_chunk(next, k));
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
  float* ml = a.part_ml + (w.pair * a.parts + w.p) * kMlFloats;
  float* po = a.part_o + (w.pair * a.parts + w.p) * a.width * HD;
#pragma unroll
  for (int h = 0; h < R; ++h) {
    const float mh = readlane_f(m[h & 3], 16 * (h >> 2));
    const float lh = readlane_f(lsum[h & 3], 16 * (h >> 2));
    if (a.parts > 1 && lane == 0) {
      ml[2 * h] = mh;
      ml[2 * h + 1] = lh;
    }
    if (h % NG != tg || h >= a.rq) continue;
    f32x4 x{o[h][0], o[h][1], o[h][2], o[h][3]};
    if (a.parts > 1) {
      *reinterpret_cast<f32x4*>(po + h * HD + 4 * c) = x;
    } else {
      x *= lh == 0.0f ? 0.0f : 1.0f / lh;
      *reinterpret_cast<f32x4*>(reinterpret_cast<float*>(a.out) +
                                (w.pair * a.rtot + a.h0 + h) * HD + 4 * c) = x;
    }
  }
}

// Joins the parts: M = max m_p, L = sum l_p 2^(m_p - M), O = sum O_p 2^(m_p - M) / L;
// L = 0 (no key at all) gives a zero row.  One wave per query head: HD / 4
// lanes read a partial row, 64 / (HD / 4) rows per load, U loads in flight; the
// first ones and the (m, l) pairs of up to 64 parts go out together.
template <int HD>
__global__ void __launch_bounds__(kWavesPerBlock * kWave)
    sparse_merge_kernel(SparseKArgs a, int dt) {
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
  const float* po = a.part_o + (pair * a.parts * a.width + h) * HD + 4 * c;
  const size_t row = (size_t)a.width * HD;
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
  const size_t eo = (pair * a.rtot + a.h0 + h) * HD + 4 * c;
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

constexpr int kThreads = kWavesPerBlock * kWave;

template <int DT, int HD>
void launch16(const SparseKArgs& k, unsigned grid, hipStream_t s) {
  const int waves = k.joined ? k.parts : kWavesPerBlock;
  const int threads = waves * kWave, lds = waves * Cfg16<HD>::LDS;
  if (k.bs_log2 < 4) sparse16_kernel<DT, HD, true, false><<<grid, threads, lds, s>>>(k);
  else if (k.max_q > 1) sparse16_kernel<DT, HD, false, false><<<grid, threads, lds, s>>>(k);
  else sparse16_kernel<DT, HD, false, true><<<grid, threads, lds, s>>>(k);
}

template <int HD, int R>
void launch32_r(const SparseKArgs& k, unsigned grid, hipStream_t s) {
  if (k.bs_log2 < 4) sparse32_kernel<HD, R, true, false><<<grid, kThreads, 0, s>>>(k);
  else if (k.max_q > 1) sparse32_kernel<HD, R, false, false><<<grid, kThreads, 0, s>>>(k);
  else sparse32_kernel<HD, R, false, true><<<grid, kThreads, 0, s>>>(k);
}

template <int HD>
void launch32(const SparseKArgs& k, unsigned grid, hipStream_t s) {
  switch (k.width) {
    case 1: launch32_r<HD, 1>(k, grid, s); break;
    case 2: launch32_r<HD, 2>(k, grid, s); break;
    case 4: launch32_r<HD, 4>(k, grid, s); break;
    case 8: launch32_r<HD, 8>(k, grid, s); break;
    default: launch32_r<HD, 16>(k, grid, s); break;
  }
}

template <int HD>
hipError_t launch_hd(int dt, const SparseKArgs& k, unsigned grid, unsigned merge_grid,
                     hipStream_t s) {
  switch (dt) {
    case PKV_F32: launch32<HD>(k, grid, s); break;
    case PKV_F16: launch16<PKV_F16, HD>(k, grid, s); break;
    default: launch16<PKV_BF16, HD>(k, grid, s); break;
  }
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess || k.parts == 1 || k.joined) return e;
  sparse_merge_kernel<HD><<<merge_grid, kThreads, 0, s>>>(k, dt);
  return hipGetLastError();
}

constexpr int kJoinTokens = 256, kJoinPairs = 160, kJoinSinglePairs = 256;

struct SparsePlan {
  int bs_log2, part_tokens, parts, R;
  bool joined;
  size_t ml, bytes;
};

int most_waves(int head_dim) {
  return head_dim == 64    ? Cfg16<64>::WAVES
         : head_dim == 128 ? Cfg16<128>::WAVES
                           : Cfg16<256>::WAVES;
}

// Parts of 1024 tokens, halved (down to 64) while a part has more than the 64
// list entries of a wave, and while the call has fewer than 1024 waves, one per
// SIMD; 2048 for chunks, whose rows hit the caches and are bound by the waves'
// own steps.  (us, main kernel and merge, from 1024 / 2048 waves, bf16: 43 chunk rows
// of 1200 tokens, 64 heads on 8 of 128: 53 / 38; single rows: 64 of 2048 tokens, 32
// heads: 93 / 90; 32 of 2048, 64 heads: 49 / 53; 32 of 1600, 16 heads of 256 (f16):
// 81 / 93.)
// The parts of a row and kv head of a 16-bit pool are joined in one workgroup if
// there are four or more, a workgroup can have that many and the workgroups cover
// most CUs.  Chunks and heads of 256: parts too many for a workgroup are lengthened
// for it, up to 256 tokens.  Single rows with smaller heads read their blocks from
// HBM whichever way and gain only the merge's launch; they are joined with five to
// seven parts while the workgroups are one a CU at most, and with four whose last
// is half full at most (with more in it the merge is level or ahead).  A call,
// joined / with the merge, us, bf16, 8 kv heads, 4 query heads each (2 at heads of
// 256):
//   pairs, tokens      chunks 64   chunks 128   chunks 256   single 64    single 128
//   160    768         9.0/10.8    13.3/15.3    26/26        14.0/11.9 x  20.5/19.1 x
//   160    1600        13/20       22/32        55/56        24.9/24.1    36.8/40.7
//   192    1312                                              21.2/24.0    32.8/40.4
//   256    768         9.3/13.1    13.6/20.6    36/36        14.8/17.0    22.8/26.7
//   256    1024        10.0/13.9   16.6/20.3    27/35        18.6/18.3 x  28.3/28.2 x
//   256    1200        12/17       18/30        53/53        21/25        33/42
//   256    1600        13/25       22/42        81/80        26.4/27.8    41.4/44.6
//   256    1920                                              31/29 x      49/48 x
//   256    2048        15/19       26/30        53/53        32/29 x      52/49 x
//   288    768         15.1/14.6   24.6/23.4    44/44        23/18 x      39/28 x
//   320    1568                                              42.3/41.5    68/74
//   320    2048        25.5/24.2   47/39        75/75        54/43 x      87/79 x
//   384    1600        23/33       41/62        105/105      45.1/44.3    72/77
//   448    832                                               26.3/26.6    43/47
//   512    1600        23/28       38/48        84/92        49/48 x      86/86 x
// (x: not joined; single rows of heads of 256: 160 of 1024 40/47, 256 of 1600 71/84, 320
// of 1600 121/140, 512 of 2048 185/177, as chunks else.)  Fewer pairs, joined / with
// the merge: 128 of 2048, 128: 41 / 28, 64 of 1536: 30 / 19.
SparsePlan sparse_plan(const pkv_pool* p, const SparseArgs& a) {
  SparsePlan pl{};
  while ((1 << pl.bs_log2) < p->block_size) ++pl.bs_log2;
  pl.R = group_width(a.n_head / p->n_kv_head);
  const long long len = (long long)a.top_blocks << pl.bs_log2;
  const long long pairs = (long long)a.total_q * p->n_kv_head;
  auto parts = [&](int pt) { return (len + pt - 1) / pt; };
  int pt = 1024;
  while (pt > 64 && pairs * parts(pt) < (a.max_q_len > 1 ? 2048 : 1024)) pt >>= 1;
  while (pt > 64 && (pt >> pl.bs_log2) > 64) pt >>= 1;
  if (p->dtype != PKV_F32 && pairs >= kJoinPairs) {
    const int most = most_waves(p->head_dim);
    if (a.max_q_len > 1 || p->head_dim == 256) {
      int longer = pt;
      while (parts(longer) > most && longer < kJoinTokens && (2 * longer >> pl.bs_log2) <= 64)
        longer <<= 1;
      pl.joined = parts(longer) >= 4 && parts(longer) <= most;
      if (pl.joined) pt = longer;
    } else {
      const long long last = len % pt;
      pl.joined = parts(pt) == 4 ? last && last <= pt / 2
                                 : pairs <= kJoinSinglePairs && parts(pt) >= 5 && parts(pt) <= 7;
    }
  }
  pl.part_tokens = pt;
  pl.parts = (int)parts(pt);
  if (pl.parts > 1 && !pl.joined) {
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
  SparseArgs x = a;  // of single rows and of chunks, whichever is more
  size_t most = 0;
  for (x.max_q_len = 1; x.max_q_len <= 2; ++x.max_q_len)
    most = std::max(most, sparse_plan(p, x).bytes);
  return most;
}

bool sparse_fits(const pkv_pool* p, const SparseArgs& a) {
  const SparsePlan pl = sparse_plan(p, a);
  // a wave per part, and one per query head where the parts are merged
  const bool merged = pl.parts > 1 && !pl.joined;
  const int heads = merged ? std::min(a.n_head / p->n_kv_head, 16) : 1;
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
  k.width = pl.R;
  k.rtot = a.n_head / p->n_kv_head;
  k.joined = pl.joined;
  const unsigned grid = (unsigned)(
      pl.joined ? sparse_items(p, a, 1)
                : (sparse_items(p, a, pl.parts) + kWavesPerBlock - 1) / kWavesPerBlock);
  // slices of at most 16 query heads per group share the workspace in turn
  for (k.h0 = 0; k.h0 < k.rtot; k.h0 += 16) {
    k.rq = std::min(k.rtot - k.h0, pl.R);
    const unsigned merge_grid =
        (unsigned)((sparse_items(p, a, k.rq) + kWavesPerBlock - 1) / kWavesPerBlock);
    hipError_t e;
    switch (p->head_dim) {
      case 64: e = launch_hd<64>(p->dtype, k, grid, merge_grid, stream); break;
      case 128: e = launch_hd<128>(p->dtype, k, grid, merge_grid, stream); break;
      default: e = launch_hd<256>(p->dtype, k, grid, merge_grid, stream); break;
    }
    if (e != hipSuccess) return e;
  }
  return hipSuccess;
}

}  // namespace pkv
