// pkv_q4_attn.hip -- attention over a pool held in 4 bits (gfx950).
//
// With group g's codes c, scale s and offset m, a key's score is
//   q . k = sum_g s_g (q_g . c_g) + m_g sum(q_g)
// and the values' sum
//   o_g = sum_k (p_k s_kg) c_k + sum_k p_k m_kg,
// so both products run on the matrix cores over the codes themselves.  A code's four
// bits in the low bits of an f16 are the number c 2^-24, and in the next four 16 c
// 2^-24 (subnormals, which v_mfma_f32_16x16x32_f16 takes exactly): one mask makes
// two of them, a second one the next two, and nothing is converted.
//
// A column is a query row of a chunk and one of the heads of a kv head's group.  A
// wave takes 32 keys a step: two tiles S^T = K Q^T of 16 keys, whose lanes then hold
// just the weights that they feed into the second product as its left operand.
// Weights are two f16 (2^-22): one would be off by 2^-11 of p s c, and where offset and
// code nearly cancel that is several times what rounding the result to f16 costs.
// Two kernels share this: one for few columns (decoding), one for many (chunks).
#include <algorithm>

#include "pkv_internal.h"
#include "pkv_q4_dev.h"

namespace pkv {
namespace {

constexpr int kWaves = 4;                  // of a workgroup; they take the steps in turn
constexpr int kStep = 32;                  // keys of a wave's step
constexpr float kNone = -3.0e38f;          // reference of a column without keys
constexpr float kLog2e = 1.44269504088896340736f;

typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));

struct Q4KArgs {
  Q4Args a;
  const char* k;
  const char* v;
  int kvh;
  int r;         // query heads of a kv head
  int bs_log2;
  int num_blocks;
  int cols;        // columns of a workgroup
  int tiles;       // workgroups that a sequence's and kv head's columns take
  int part_keys;   // keys of a part, a multiple of kWaves * kStep
  int max_parts;
  float* o_part;   // [row * n_head + head][part][hd]
  float2* ml_part; // [row * n_head + head][part] (reference, sum)
  uint32_t* err;
};

// Rows and keys of sequence s; false: it is left out (reported by one thread).
__device__ __forceinline__ bool sequence(const Q4KArgs& ka, int s, bool reporter, int& q0,
                                         int& rows, int& ctx) {
  const Q4Args& a = ka.a;
  q0 = a.cu_q_lens ? a.cu_q_lens[s] : s;
  const int q1 = a.cu_q_lens ? a.cu_q_lens[s + 1] : s + 1;
  ctx = a.context_lens[s];
  rows = q0 >= 0 && q1 >= q0 && q1 <= a.total_q ? q1 - q0 : -1;
  if (rows < 0 || rows > a.max_q_len || ctx < 0 || ctx > a.max_context_len ||
      ctx > ((long long)a.max_blocks_per_seq << ka.bs_log2)) {
    if (reporter) atomicOr(ka.err, PKV_EBIT_LENGTH);
    return false;
  }
  return true;
}

// A workgroup's share: columns col0 .. of sequence s and kv head g, keys k0 .. k1 - 1.
struct Item {
  int s, g, q0, rows, ctx;
  int col0, cols;       // first column, columns of the sequence and kv head
  int part, parts, k0, k1;
  int all;              // keys that every column of the share has
};

__device__ __forceinline__ int parts_of(const Q4KArgs& ka, int col0, int cols, int rows, int ctx,
                                        int& end) {
  const int last_row = (min(col0 + ka.cols, cols) - 1) / ka.r;
  end = ctx - rows + last_row + 1;
  return min(max((int)(((long long)end + ka.part_keys - 1) / ka.part_keys), 1), ka.max_parts);
}

__device__ __forceinline__ bool item_of(const Q4KArgs& ka, Item& it) {
  // parts are the slowest index: the first ones are full, the last ones empty or short
  int u = blockIdx.x;
  it.g = u % ka.kvh;
  u /= ka.kvh;
  const int tile = u % ka.tiles;
  u /= ka.tiles;
  it.s = u % ka.a.n_seqs;
  it.part = u / ka.a.n_seqs;
  if (!sequence(ka, it.s, it.part == 0 && tile == 0 && it.g == 0 && threadIdx.x == 0, it.q0,
                it.rows, it.ctx))
    return false;
  it.cols = it.rows * ka.r;
  it.col0 = tile * ka.cols;
  if (it.col0 >= it.cols) return false;
  int end;
  it.parts = parts_of(ka, it.col0, it.cols, it.rows, it.ctx, end);
  if (it.part >= it.parts) return false;
  it.k0 = it.part * ka.part_keys;
  it.k1 = min(end, it.k0 + ka.part_keys);
  it.all = min(it.ctx - it.rows + it.col0 / ka.r + 1, it.k1);
  return true;
}

// N bytes (a multiple of 4) of consecutive words.
template <int N>
__device__ __forceinline__ void load_words(const char* p, uint32_t (&w)[N / 4]) {
  if constexpr (N == 4) {
    w[0] = *reinterpret_cast<const uint32_t*>(p);
  } else if constexpr (N == 8) {
    const uint2 x = *reinterpret_cast<const uint2*>(p);
    w[0] = x.x;
    w[1] = x.y;
  } else {
#pragma unroll
    for (int i = 0; i < N / 16; ++i) {
      const u32x4 x = ld16(p + 16 * i);
#pragma unroll
      for (int j = 0; j < 4; ++j) w[4 * i + j] = x[j];
    }
  }
}

__device__ __forceinline__ float half_of(uint32_t w, int hi) {
  return (float)__builtin_bit_cast(f16x2, w)[hi];
}
__device__ __forceinline__ uint32_t pack_half(float x, float y) {
  const f16x2 h = {(_Float16)x, (_Float16)y};
  return __builtin_bit_cast(uint32_t, h);
}
// (x, y) in two f16 each: high and low parts.
__device__ __forceinline__ void split_half(float x, float y, uint32_t& hi, uint32_t& lo) {
  hi = pack_half(x, y);
  lo = pack_half(x - half_of(hi, 0), y - half_of(hi, 1));
}
// (x a, y b) likewise, a and b the halves of w (each product a v_fma_mix).
__device__ __forceinline__ void split_scaled(float x, float y, uint32_t w, uint32_t& hi,
                                             uint32_t& lo) {
  const float a = half_of(w, 0), b = half_of(w, 1);
  hi = pack_half(fmaf(x, a, 0.0f), fmaf(y, b, 0.0f));
  lo = pack_half(fmaf(x, a, -half_of(hi, 0)), fmaf(y, b, -half_of(hi, 1)));
}
__device__ __forceinline__ f32x4 mfma16(const uint32_t (&a)[4], const uint32_t (&b)[4], f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(
      __builtin_bit_cast(f16x8, u32x4{a[0], a[1], a[2], a[3]}),
      __builtin_bit_cast(f16x8, u32x4{b[0], b[1], b[2], b[3]}), c, 0, 0, 0);
}
__device__ __forceinline__ float lane_of(float x, int lane) {
  return __int_as_float(__builtin_amdgcn_ds_bpermute(lane << 2, __float_as_int(x)));
}

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
}

__device__ __forceinline__ void put(void* out, int dt, size_t i, float x) {
  if (dt == PKV_F32) static_cast<float*>(out)[i] = x;
  else if (dt == PKV_F16) static_cast<_Float16*>(out)[i] = (_Float16)x;
  else static_cast<uint16_t*>(out)[i] = (uint16_t)f32_to_bf16_bits(x);
}

// Four words of a K code word: its channels 2 e, 2 e + 1 as f16 pairs.
__device__ __forceinline__ void k_pairs(uint32_t w, uint32_t (&f)[4]) {
  const uint32_t w8 = w >> 8;
  f[0] = w & 0x000f000fu;
  f[1] = w & 0x00f000f0u;
  f[2] = w8 & 0x000f000fu;
  f[3] = w8 & 0x00f000f0u;
}

// V codes of a lane's four tokens (T / 2 bytes each): for channels 4 h .. 4 h + 3 of the
// column, tokens 0 and 1, 2 and 3 side by side in 16 bits each.
template <int T>
__device__ __forceinline__ void v_pairs(const uint32_t (&code)[T / 2], uint32_t (&pair)[2][T / 4]) {
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    if constexpr (T == 4) {
      pair[e][0] = code[e];
    } else {
      constexpr int W = T / 8;  // words of a token
#pragma unroll
      for (int w = 0; w < W; ++w) {
        const uint32_t t0 = code[2 * e * W + w], t1 = code[(2 * e + 1) * W + w];
        pair[e][2 * w] = __builtin_amdgcn_perm(t1, t0, 0x05040100u);
        pair[e][2 * w + 1] = __builtin_amdgcn_perm(t1, t0, 0x07060302u);
      }
    }
  }
}
// Right operand of channels i + 16 t from the pairs of both 16-token tiles.
template <int T>
__device__ __forceinline__ void v_frag(const uint32_t (&pair)[2][2][T / 4], int t,
                                       uint32_t (&f)[4]) {
#pragma unroll
  for (int j = 0; j < 2; ++j)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const uint32_t w = pair[j][e][t / 4];
      f[2 * j + e] = ((t & 2) ? w >> 8 : w) & ((t & 1) ? 0x00f000f0u : 0x000f000fu);
    }
}

// The block ids of a wave's steps, 64 tiles of 16 keys at a time: lane 2 n + j has the
// id of tile j of the n-th step from `first` on, -1 where it is outside the pool (or
// beyond the last key).  Lanes of the same block report it.
__device__ __forceinline__ int ids_of(const Q4KArgs& ka, const int32_t* table, int first, int k1) {
  const int lane = threadIdx.x & 63;
  const long long key = (long long)first + (lane >> 1) * (kWaves * kStep) + 16 * (lane & 1);
  int id = -1;
  if (key < k1) {
    id = table[key >> ka.bs_log2];
    if ((unsigned)id >= (unsigned)ka.num_blocks) {
      atomicOr(ka.err, PKV_EBIT_BLOCK);
      id = -1;
    }
  }
  return id;
}

// Keeps a column's running reference: weights 2^(x - ref) are at most 2^top, 14, so that
// with values' scales below 2 a weight times a scale stays within f16; a new one leaves
// room for growth by 2^6.  From the first scale of 2 or more on (scales are below
// 2^14) top is 1.  m: the column's largest score of the step.
__device__ __forceinline__ float new_ref(float ref, float m, float top, bool less) {
  if (less) return fmaxf(m, ref + 14.0f) - top;  // (scores up to ref + 14 were let in)
  return m - ref > top ? m - (top > 1.0f ? top - 6.0f : top) : ref;
}

// ---- few columns -------------------------------------------------------------
// The 16 columns of the tiles are 16 / G query columns times the G groups: column
// (c, g) of Q^T has the channels of group g alone, so one accumulator collects every
// group's product, a lane scales it once, and the G lanes of a query column add
// up.  A lane's weights then are for its group alone: rows (c, g) of the second product
// give o_g in the tiles of group g, the others are not used.  DT: type of q.  NT: such
// tiles, 16 / G query columns each.
template <int DT, int HD, int NT>
__global__ void __launch_bounds__(kWaves * 64) q4_few_kernel(Q4KArgs ka) {
  using L = Q4Layout<HD>;
  constexpr int G = L::G, T = L::T, NP = DT == PKV_F32 ? 2 : 1, E = DT == PKV_F32 ? 4 : 2;
  constexpr int C = 16 / G;  // query columns of a tile
  __shared__ float sm_m[kWaves][NT * C], sm_l[kWaves][NT * C];
  __shared__ float sm_o[kWaves][NT][8][64];

  const Q4Args& a = ka.a;
  Item it;
  if (!item_of(ka, it)) return;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lane = threadIdx.x & 63, kq = lane >> 4, n16 = lane & 15;
  const int cl = n16 / G, gp = n16 % G;

  // over the G lanes of a query column
  auto col_add = [](float x) {
    x += dpp_f<0xB1>(x);
    if constexpr (G >= 4) x += dpp_f<0x4E>(x);
    if constexpr (G == 8) x += dpp_f<0x141>(x);  // row_half_mirror: the other four
    return x;
  };
  auto col_max = [](float x) {
    x = fmaxf(x, dpp_f<0xB1>(x));
    if constexpr (G >= 4) x = fmaxf(x, dpp_f<0x4E>(x));
    if constexpr (G == 8) x = fmaxf(x, dpp_f<0x141>(x));
    return x;
  };

  // ---- the columns' queries ----
  uint32_t qf[NT][NP][G][4];   // right operand: channels 32 g + 8 kq + e where g is gp
  float qs[NT], f[NT];         // sum of the group; a score is f times what the products give
  int lim[NT];                 // a column's keys
#pragma unroll
  for (int c = 0; c < NT; ++c) {
    const int col = it.col0 + c * C + cl;
    const bool live = col < it.cols;
    const int i = live ? col / ka.r : 0, h = it.g * ka.r + (live ? col - i * ka.r : 0);
    lim[c] = live ? it.ctx - it.rows + i + 1 : 0x7fffffff;
    float x[8], big = 0.0f, sum = 0.0f;
    load8<DT>(static_cast<const char*>(a.q) +
                  ((size_t)(it.q0 + i) * a.q_stride + (size_t)h * HD + 32 * gp + 8 * kq) * E, x);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      if (!live || a.scale == 0.0f) x[e] = 0.0f;
      big = fmaxf(big, fabsf(x[e]));
    }
    big = col_max(row_group_max(big));
    const int ex = big > 0.0f ? 14 - __builtin_amdgcn_frexp_expf(big) : 0;  // below 2^14
    f[c] = fmaxf(ldexpf(fabsf(a.scale) * kLog2e, 24 - ex), 0x1p-126f);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      x[e] = ldexpf(a.scale < 0.0f ? -x[e] : x[e], ex);
      sum += x[e];
    }
    qs[c] = swap32_sum(swap16_sum(sum)) * 0x1p-24f;
#pragma unroll
    for (int e = 0; e < 8; e += 2) {
      const float by = (e & 2) ? 0.0625f : 1.0f;  // these codes are 16 times larger
      uint32_t w[2];
      if constexpr (NP == 2) split_half(x[e] * by, x[e + 1] * by, w[0], w[1]);
      else w[0] = pack_half(x[e] * by, x[e + 1] * by);
#pragma unroll
      for (int p = 0; p < NP; ++p)
#pragma unroll
        for (int g = 0; g < G; ++g) qf[c][p][g][e / 2] = g == gp ? w[p] : 0u;
    }
  }

  // ---- the steps ----
  const int bs = 1 << ka.bs_log2;
  const size_t blk_stride = (size_t)ka.kvh * L::chunk(bs);
  const char* kh = ka.k + (size_t)it.g * L::chunk(bs);
  const char* vh = ka.v + (size_t)it.g * L::chunk(bs);
  const int32_t* table = a.block_tables + (size_t)it.s * a.max_blocks_per_seq;
  const int s_off = bs * (HD / 2) + (kq * G + gp) * 8, m_off = s_off + bs * G * 2;
  const int k_off = (n16 * 4 + kq) * G * 4, v_off = (n16 * bs + kq * 4) * (T / 2);

  struct KV {
    uint32_t code[HD / 32], s[2], m[2];
  };
  auto load = [&](const char* base, int id, int key, bool keys, KV& t) {
    const int at = key & (bs - 1);
    const char* p = base + (size_t)max(id, 0) * blk_stride;
    load_words<HD / 8>(p + at * (keys ? HD / 2 : T / 2) + (keys ? k_off : v_off), t.code);
    load_words<8>(p + at * (G * 2) + s_off, t.s);
    load_words<8>(p + at * (G * 2) + m_off, t.m);
  };

  f32x4 o[NT][T];   // row (c, g) = 4 kq + i: channel n16 + 16 t
  float ref[NT], l[NT], om[NT];
#pragma unroll
  for (int c = 0; c < NT; ++c) {
    ref[c] = kNone;
    l[c] = om[c] = 0.0f;
#pragma unroll
    for (int t = 0; t < T; ++t) o[c][t] = f32x4{0, 0, 0, 0};
  }
  float top = 14.0f;

  constexpr int stride = kWaves * kStep;
  int key = it.k0 + wave * kStep;
  int ids = ids_of(ka, table, key, it.k1), left = 32;
  int id[2] = {readlane_i(ids, 0), readlane_i(ids, 1)};
  KV kt[2], vt[2];
  if (key < it.k1) {
#pragma unroll
    for (int j = 0; j < 2; ++j) load(kh, id[j], key + 16 * j, true, kt[j]);
#pragma unroll
    for (int j = 0; j < 2; ++j) load(vh, id[j], key + 16 * j, false, vt[j]);
  }
  for (; key < it.k1; key += stride) {
    const bool masked = key + kStep > it.all || (id[0] | id[1]) < 0;
    const bool in[2] = {id[0] >= 0, id[1] >= 0};
    float x[NT][2][4];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      f32x4 d[NT];
#pragma unroll
      for (int c = 0; c < NT; ++c) d[c] = f32x4{0, 0, 0, 0};
#pragma unroll
      for (int g = 0; g < G; ++g) {
        uint32_t kf[4];
        k_pairs(kt[j].code[g], kf);
#pragma unroll
        for (int c = 0; c < NT; ++c)
#pragma unroll
          for (int p = 0; p < NP; ++p) d[c] = mfma16(kf, qf[c][p][g], d[c]);
      }
#pragma unroll
      for (int c = 0; c < NT; ++c)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          x[c][j][i] = col_add(fmaf(half_of(kt[j].s[i / 2], i % 2), d[c][i],
                                    half_of(kt[j].m[i / 2], i % 2) * qs[c]));
    }
    // the next step's keys
    if (--left == 0) {
      ids = ids_of(ka, table, key + stride, it.k1);
      left = 32;
    }
    const int next = key + stride;
    const bool more = next < it.k1;
    if (more) {
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        id[j] = readlane_i(ids, 2 * (32 - left) + j);
        load(kh, id[j], next + 16 * j, true, kt[j]);
      }
    }
    if (masked) {
#pragma unroll
      for (int c = 0; c < NT; ++c)
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (key + 16 * j + 4 * kq + i >= min(lim[c], it.k1) || !in[j]) x[c][j][i] = -INFINITY;
    }
    // a large scale of values, or a score far above its column's reference
    const bool big = (vt[0].s[0] | vt[0].s[1] | vt[1].s[0] | vt[1].s[1]) & 0x40004000u;
    float mx[NT];
    bool far = top > 1.0f && big;
#pragma unroll
    for (int c = 0; c < NT; ++c) {
      mx[c] = x[c][0][0];
#pragma unroll
      for (int e = 1; e < 8; ++e) mx[c] = fmaxf(mx[c], x[c][e / 4][e % 4]);
      mx[c] *= f[c];
      far |= mx[c] - ref[c] > top;
    }
    if (__builtin_amdgcn_ballot_w64(far)) {
      const bool less = top > 1.0f && __builtin_amdgcn_ballot_w64(big);
      if (less) top = 1.0f;
#pragma unroll
      for (int c = 0; c < NT; ++c) {
        const float old = ref[c];
        ref[c] = new_ref(old, row_group_max(mx[c]), top, less);
        const float by = fast_exp2(old - ref[c]);
        l[c] *= by;
        om[c] *= by;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float b = lane_of(by, 4 * kq + i);
#pragma unroll
          for (int t = 0; t < T; ++t) o[c][t][i] *= b;
        }
      }
    }
    uint32_t wf[NT][2][4];
#pragma unroll
    for (int c = 0; c < NT; ++c)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        float p[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          p[i] = fast_exp2(fmaf(x[c][j][i], f[c], -ref[c]));
          l[c] += p[i];
          om[c] = fmaf(half_of(vt[j].m[i / 2], i % 2), p[i], om[c]);
        }
#pragma unroll
        for (int e = 0; e < 2; ++e)
          split_scaled(p[2 * e], p[2 * e + 1], vt[j].s[e], wf[c][0][2 * j + e],
                       wf[c][1][2 * j + e]);
      }
    uint32_t pair[2][2][T / 4];
#pragma unroll
    for (int j = 0; j < 2; ++j) v_pairs<T>(vt[j].code, pair[j]);
    if (more) {
#pragma unroll
      for (int j = 0; j < 2; ++j) load(vh, id[j], next + 16 * j, false, vt[j]);
    }
#pragma unroll
    for (int t = 0; t < T; ++t) {
      uint32_t vf[4];
      v_frag<T>(pair, t, vf);
#pragma unroll
      for (int c = 0; c < NT; ++c)
#pragma unroll
        for (int p = 0; p < 2; ++p) o[c][t] = mfma16(wf[c][p], vf, o[c][t]);
    }
  }

  // ---- join the waves ----
#pragma unroll
  for (int c = 0; c < NT; ++c) {
    l[c] = swap32_sum(swap16_sum(l[c]));
    om[c] = swap32_sum(swap16_sum(om[c]));
    if (kq == 0 && gp == 0) {
      sm_m[wave][c * C + cl] = ref[c];
      sm_l[wave][c * C + cl] = l[c];
    }
  }
  // Eight of a lane's values are used: slot e is channel n16 + 16 t of query column qc.
  auto slot = [&](int e, int k, int& t, int& qc) {
    if constexpr (HD == 64) {  // rows 4 k + i: columns 2 k + i / 2, group i % 2
      t = e / 2;
      qc = 2 * k + e % 2;
    } else if constexpr (HD == 128) {  // column k, group i
      t = e;
      qc = k;
    } else {  // column k / 2, group 4 (k % 2) + i
      t = 8 * (k & 1) + e;
      qc = k / 2;
    }
  };
#pragma unroll
  for (int c = 0; c < NT; ++c)
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      int t, qc;
      slot(e, kq, t, qc);
      float y;
      if constexpr (HD == 64) y = o[c][e / 2][2 * (e % 2) + e / 4];
      else if constexpr (HD == 128) y = o[c][e][e / 2];
      else y = (kq & 1) ? o[c][8 + e][e / 2] : o[c][e][e / 2];
      const float by = (HD == 64 ? e / 2 : e) % 2 ? 0x1p20f : 0x1p24f;
      sm_o[wave][c][e][lane] = fmaf(y, by, lane_of(om[c], qc * G + t / 2));
    }
  __syncthreads();
  for (int j = threadIdx.x; j < NT * 512; j += kWaves * 64) {
    const int c = j / 512, e = j / 64 % 8;
    int t, qc;
    slot(e, (j & 63) >> 4, t, qc);
    const int r = c * C + qc, col = it.col0 + r, d = 16 * t + (j & 15);
    if (col >= it.cols) continue;
    float m = kNone, sum = 0.0f, y = 0.0f;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) m = fmaxf(m, sm_m[w][r]);
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      const float by = fast_exp2(sm_m[w][r] - m);
      sum = fmaf(sm_l[w][r], by, sum);
      y = fmaf(sm_o[w][c][e][j & 63], by, y);
    }
    const int row = col / ka.r;
    const size_t at = (size_t)(it.q0 + row) * a.n_head + it.g * ka.r + (col - row * ka.r);
    if (it.parts == 1) {
      put(a.out, a.out_dtype, at * HD + d, sum > 0.0f ? y / sum : 0.0f);
    } else {
      const size_t pa = at * ka.max_parts + it.part;
      if (d == 0) ka.ml_part[pa] = float2{m, sum};
      ka.o_part[pa * HD + d] = y;
    }
  }
}

// ---- many columns ------------------------------------------------------------
// Tiles of 16 query columns: a product per group, scaled and added up in the lane; the
// offsets' products are one v_mfma_f32_16x16x4_f32 (its four k are groups).  DT: type of
// q.  NT: tiles.
template <int DT, int HD, int NT>
__global__ void __launch_bounds__(kWaves * 64) q4_many_kernel(Q4KArgs ka) {
  using L = Q4Layout<HD>;
  constexpr int G = L::G, T = L::T, NP = DT == PKV_F32 ? 2 : 1, E = DT == PKV_F32 ? 4 : 2;
  constexpr int GM = (G + 3) / 4;  // products of four groups' offsets
  __shared__ float sm_m[kWaves][NT * 16], sm_l[kWaves][NT * 16];
  __shared__ float sm_o[2][NT * 16 * HD];

  const Q4Args& a = ka.a;
  Item it;
  if (!item_of(ka, it)) return;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lane = threadIdx.x & 63, kq = lane >> 4, n16 = lane & 15;

  uint32_t qf[NT][NP][G][4];   // right operand: column n16, channels 32 g + 8 kq + e
  float qs[NT][GM];            // sum of group 4 b + kq
  float f[NT];
  int lim[NT];
#pragma unroll
  for (int c = 0; c < NT; ++c) {
    const int col = it.col0 + c * 16 + n16;
    const bool live = col < it.cols;
    const int i = live ? col / ka.r : 0, h = it.g * ka.r + (live ? col - i * ka.r : 0);
    lim[c] = live ? it.ctx - it.rows + i + 1 : 0x7fffffff;
    const char* src = static_cast<const char*>(a.q) +
                      ((size_t)(it.q0 + i) * a.q_stride + (size_t)h * HD + 8 * kq) * E;
    float x[G][8], big = 0.0f;
#pragma unroll
    for (int g = 0; g < G; ++g) {
      load8<DT>(src + 32 * g * E, x[g]);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        if (!live || a.scale == 0.0f) x[g][e] = 0.0f;
        big = fmaxf(big, fabsf(x[g][e]));
      }
    }
    big = row_group_max(big);
    const int ex = big > 0.0f ? 14 - __builtin_amdgcn_frexp_expf(big) : 0;
    f[c] = fmaxf(ldexpf(fabsf(a.scale) * kLog2e, 24 - ex), 0x1p-126f);
#pragma unroll
    for (int b = 0; b < GM; ++b) qs[c][b] = 0.0f;
#pragma unroll
    for (int g = 0; g < G; ++g) {
      float sum = 0.0f;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        x[g][e] = ldexpf(a.scale < 0.0f ? -x[g][e] : x[g][e], ex);
        sum += x[g][e];
      }
      sum = swap32_sum(swap16_sum(sum)) * 0x1p-24f;
      if (kq == g % 4) qs[c][g / 4] = sum;
#pragma unroll
      for (int e = 0; e < 8; e += 2) {
        const float by = (e & 2) ? 0.0625f : 1.0f;
        if constexpr (NP == 2)
          split_half(x[g][e] * by, x[g][e + 1] * by, qf[c][0][g][e / 2], qf[c][1][g][e / 2]);
        else
          qf[c][0][g][e / 2] = pack_half(x[g][e] * by, x[g][e + 1] * by);
      }
    }
  }

  const int bs = 1 << ka.bs_log2;
  const size_t blk_stride = (size_t)ka.kvh * L::chunk(bs);
  const char* kh = ka.k + (size_t)it.g * L::chunk(bs);
  const char* vh = ka.v + (size_t)it.g * L::chunk(bs);
  const int32_t* table = a.block_tables + (size_t)it.s * a.max_blocks_per_seq;
  const int s_off = bs * (HD / 2) + kq * G * 8;
  const int k_off = (n16 * 4 + kq) * G * 4, v_off = (n16 * bs + kq * 4) * (T / 2);
  // offsets: key n16 of group kq (and kq + 4); tokens 4 kq .. of group n16
  const int km_off = bs * (HD / 2) + bs * G * 2 + ((n16 >> 2) * G + kq % G) * 8 + (n16 & 3) * 2;
  const int vm_off = bs * (HD / 2) + bs * G * 2 + (kq * G + n16 % G) * 8;

  struct KTile {
    uint32_t code[HD / 32], s[2 * G];
    _Float16 m[GM];
  };
  struct VTile {
    uint32_t code[HD / 32], s[2 * G], m[2];
  };
  auto load_k = [&](int id, int key, KTile& t) {
    const int at = key & (bs - 1);
    const char* p = kh + (size_t)max(id, 0) * blk_stride;
    load_words<HD / 8>(p + at * (HD / 2) + k_off, t.code);
    load_words<G * 8>(p + at * (G * 2) + s_off, t.s);
#pragma unroll
    for (int b = 0; b < GM; ++b)
      t.m[b] = *reinterpret_cast<const _Float16*>(p + at * (G * 2) + km_off + 32 * b);
  };
  auto load_v = [&](int id, int key, VTile& t) {
    const int at = key & (bs - 1);
    const char* p = vh + (size_t)max(id, 0) * blk_stride;
    load_words<HD / 8>(p + at * (T / 2) + v_off, t.code);
    load_words<G * 8>(p + at * (G * 2) + s_off, t.s);
    load_words<8>(p + at * (G * 2) + vm_off, t.m);
  };

  f32x4 o[NT][T], om[NT];  // row 4 kq + i: channel n16 + 16 t; offsets' sum of group n16
  float ref[NT], l[NT];
#pragma unroll
  for (int c = 0; c < NT; ++c) {
    ref[c] = kNone;
    l[c] = 0.0f;
    om[c] = f32x4{0, 0, 0, 0};
#pragma unroll
    for (int t = 0; t < T; ++t) o[c][t] = f32x4{0, 0, 0, 0};
  }
  float top = 14.0f;

  constexpr int stride = kWaves * kStep;
  int key = it.k0 + wave * kStep;
  int ids = ids_of(ka, table, key, it.k1), left = 32;
  int id[2] = {readlane_i(ids, 0), readlane_i(ids, 1)};
  KTile kt[2];
  VTile vt[2];
  if (key < it.k1) {
#pragma unroll
    for (int j = 0; j < 2; ++j) load_k(id[j], key + 16 * j, kt[j]);
  }
  for (; key < it.k1; key += stride) {
#pragma unroll
    for (int j = 0; j < 2; ++j) load_v(id[j], key + 16 * j, vt[j]);
    const bool masked = key + kStep > it.all || (id[0] | id[1]) < 0;
    const bool in[2] = {id[0] >= 0, id[1] >= 0};
    float x[NT][2][4];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      f32x4 acc[NT];
#pragma unroll
      for (int c = 0; c < NT; ++c) {
        acc[c] = f32x4{0, 0, 0, 0};
#pragma unroll
        for (int b = 0; b < GM; ++b)
          acc[c] = __builtin_amdgcn_mfma_f32_16x16x4f32((float)kt[j].m[b], qs[c][b], acc[c], 0, 0, 0);
      }
#pragma unroll
      for (int g = 0; g < G; ++g) {
        uint32_t kf[4];
        k_pairs(kt[j].code[g], kf);
#pragma unroll
        for (int c = 0; c < NT; ++c) {
          f32x4 d = mfma16(kf, qf[c][0][g], f32x4{0, 0, 0, 0});
          if constexpr (NP == 2) d = mfma16(kf, qf[c][1][g], d);
#pragma unroll
          for (int i = 0; i < 4; ++i)
            acc[c][i] = fmaf(half_of(kt[j].s[2 * g + i / 2], i % 2), d[i], acc[c][i]);
        }
      }
#pragma unroll
      for (int c = 0; c < NT; ++c)
#pragma unroll
        for (int i = 0; i < 4; ++i) x[c][j][i] = acc[c][i];
    }
    if (--left == 0) {
      ids = ids_of(ka, table, key + stride, it.k1);
      left = 32;
    }
    const int next = key + stride;
    if (next < it.k1) {
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        id[j] = readlane_i(ids, 2 * (32 - left) + j);
        load_k(id[j], next + 16 * j, kt[j]);
      }
    }
    if (masked) {
#pragma unroll
      for (int c = 0; c < NT; ++c)
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (key + 16 * j + 4 * kq + i >= min(lim[c], it.k1) || !in[j]) x[c][j][i] = -INFINITY;
    }
    uint32_t sw = 0;
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int e = 0; e < 2 * G; ++e) sw |= vt[j].s[e];
    const bool big = sw & 0x40004000u;
    float mx[NT];
    bool far = top > 1.0f && big;
#pragma unroll
    for (int c = 0; c < NT; ++c) {
      mx[c] = x[c][0][0];
#pragma unroll
      for (int e = 1; e < 8; ++e) mx[c] = fmaxf(mx[c], x[c][e / 4][e % 4]);
      mx[c] *= f[c];
      far |= mx[c] - ref[c] > top;
    }
    if (__builtin_amdgcn_ballot_w64(far)) {
      const bool less = top > 1.0f && __builtin_amdgcn_ballot_w64(big);
      if (less) top = 1.0f;
#pragma unroll
      for (int c = 0; c < NT; ++c) {
        const float old = ref[c];
        ref[c] = new_ref(old, row_group_max(mx[c]), top, less);
        const float by = fast_exp2(old - ref[c]);
        l[c] *= by;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float b = lane_of(by, 4 * kq + i);
          om[c][i] *= b;
#pragma unroll
          for (int t = 0; t < T; ++t) o[c][t][i] *= b;
        }
      }
    }
    uint32_t mf[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) mf[e] = n16 < G ? vt[e / 2].m[e % 2] : 0u;
    float p[NT][2][4];
#pragma unroll
    for (int c = 0; c < NT; ++c) {
      uint32_t pf[2][4];
#pragma unroll
      for (int j = 0; j < 2; ++j) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          p[c][j][i] = fast_exp2(fmaf(x[c][j][i], f[c], -ref[c]));
          l[c] += p[c][j][i];
        }
#pragma unroll
        for (int e = 0; e < 2; ++e)
          split_half(p[c][j][2 * e], p[c][j][2 * e + 1], pf[0][2 * j + e], pf[1][2 * j + e]);
      }
      om[c] = mfma16(pf[0], mf, om[c]);
      om[c] = mfma16(pf[1], mf, om[c]);
    }
    uint32_t pair[2][2][T / 4];
#pragma unroll
    for (int j = 0; j < 2; ++j) v_pairs<T>(vt[j].code, pair[j]);
#pragma unroll
    for (int g = 0; g < G; ++g) {
      uint32_t wf[NT][2][4];
#pragma unroll
      for (int c = 0; c < NT; ++c)
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
          for (int e = 0; e < 2; ++e)
            split_scaled(p[c][j][2 * e], p[c][j][2 * e + 1], vt[j].s[2 * g + e],
                         wf[c][0][2 * j + e], wf[c][1][2 * j + e]);
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        uint32_t vf[4];
        v_frag<T>(pair, 2 * g + b, vf);
#pragma unroll
        for (int c = 0; c < NT; ++c)
#pragma unroll
          for (int q = 0; q < 2; ++q) o[c][2 * g + b] = mfma16(wf[c][q], vf, o[c][2 * g + b]);
      }
    }
  }

  // ---- join the waves ----
#pragma unroll
  for (int c = 0; c < NT; ++c) {
    l[c] = swap32_sum(swap16_sum(l[c]));
    if (kq == 0) {
      sm_m[wave][c * 16 + n16] = ref[c];
      sm_l[wave][c * 16 + n16] = l[c];
    }
    // offsets: group g of row 4 kq + i is in lane 16 kq + g
#pragma unroll
    for (int g = 0; g < G; ++g)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float m = lane_of(om[c][i], 16 * kq + g);
        o[c][2 * g][i] = fmaf(o[c][2 * g][i], 0x1p24f, m);
        o[c][2 * g + 1][i] = fmaf(o[c][2 * g + 1][i], 0x1p20f, m);
      }
  }
  __syncthreads();
  float best[NT][4], sum[NT][4];
#pragma unroll
  for (int c = 0; c < NT; ++c)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int r = c * 16 + 4 * kq + i;
      float m = kNone, t = 0.0f;
      for (int w = 0; w < kWaves; ++w) m = fmaxf(m, sm_m[w][r]);
      for (int w = 0; w < kWaves; ++w) t = fmaf(sm_l[w][r], fast_exp2(sm_m[w][r] - m), t);
      best[c][i] = m;
      sum[c][i] = t;
      const float by = fast_exp2(sm_m[wave][r] - m);
#pragma unroll
      for (int t2 = 0; t2 < T; ++t2) o[c][t2][i] *= by;
    }
  // waves 2 and 3 into 0 and 1, then 1 into 0
#pragma unroll
  for (int half = 2; half >= 1; half >>= 1) {
    if (wave >= half && wave < 2 * half) {
#pragma unroll
      for (int c = 0; c < NT; ++c)
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int t = 0; t < T; ++t)
            sm_o[wave - half][(c * 16 + 4 * kq + i) * HD + 16 * t + n16] = o[c][t][i];
    }
    __syncthreads();
    if (wave < half) {
#pragma unroll
      for (int c = 0; c < NT; ++c)
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int t = 0; t < T; ++t)
            o[c][t][i] += sm_o[wave][(c * 16 + 4 * kq + i) * HD + 16 * t + n16];
    }
    __syncthreads();
  }
  if (wave != 0) return;
#pragma unroll
  for (int c = 0; c < NT; ++c)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int col = it.col0 + c * 16 + 4 * kq + i;
      if (col >= it.cols) continue;
      const int row = col / ka.r;
      const size_t at = (size_t)(it.q0 + row) * a.n_head + it.g * ka.r + (col - row * ka.r);
      if (it.parts == 1) {
        const float inv = sum[c][i] > 0.0f ? 1.0f / sum[c][i] : 0.0f;
#pragma unroll
        for (int t = 0; t < T; ++t) put(a.out, a.out_dtype, at * HD + 16 * t + n16, o[c][t][i] * inv);
      } else {
        const size_t pa = at * ka.max_parts + it.part;
        if (n16 == 0) ka.ml_part[pa] = float2{best[c][i], sum[c][i]};
#pragma unroll
        for (int t = 0; t < T; ++t) ka.o_part[pa * HD + 16 * t + n16] = o[c][t][i];
      }
    }
}

// Joins the parts of a query row and head: one wave each.
template <int HD>
__global__ void __launch_bounds__(256) q4_join_kernel(Q4KArgs ka) {
  constexpr int PER = HD / 64;
  const Q4Args& a = ka.a;
  const int lane = threadIdx.x & 63;
  long long u = (long long)blockIdx.x * 4 + (threadIdx.x >> 6);
  const int h = (int)(u % a.n_head);
  u /= a.n_head;
  const int i = (int)(u % a.max_q_len);
  u /= a.max_q_len;
  if (u >= a.n_seqs) return;
  int q0, rows, ctx, end;
  if (!sequence(ka, (int)u, false, q0, rows, ctx) || i >= rows) return;
  const int col = i * ka.r + h % ka.r;
  const int parts = parts_of(ka, col / ka.cols * ka.cols, rows * ka.r, rows, ctx, end);
  if (parts == 1) return;
  const size_t at = (size_t)(q0 + i) * a.n_head + h;
  const float2* ml = ka.ml_part + at * ka.max_parts;
  const float* o = ka.o_part + at * ka.max_parts * HD + lane * PER;
  float m = kNone;
  for (int p = lane; p < parts; p += 64) m = fmaxf(m, ml[p].x);
  m = row_group_max(row_max16(m));
  float l = 0.0f, x[PER] = {};
  for (int p = 0; p < parts; ++p) {
    const float2 t = ml[p];
    const float by = fast_exp2(t.x - m);
    l = fmaf(t.y, by, l);
#pragma unroll
    for (int j = 0; j < PER; ++j) x[j] = fmaf(o[(size_t)p * HD + j], by, x[j]);
  }
  const float inv = l > 0.0f ? 1.0f / l : 0.0f;
#pragma unroll
  for (int j = 0; j < PER; ++j) put(a.out, a.out_dtype, at * HD + lane * PER + j, x[j] * inv);
}

struct Plan {
  bool few;
  int nt, cols, tiles, part_keys, max_parts;
};

Plan plan_of(const pkv_pool* p, const Q4Args& a) {
  Plan pl;
  const int c = 16 / (p->head_dim / 32);  // query columns of a tile for few
  const long long cols = (long long)a.max_q_len * (a.n_head / p->n_kv_head);
  pl.few = cols <= 2 * c;
  pl.nt = pl.few ? (cols > c ? 2 : 1) : p->head_dim <= 128 && cols > 16 ? 2 : 1;
  pl.cols = pl.nt * (pl.few ? c : 16);
  pl.tiles = (int)std::min((cols + pl.cols - 1) / pl.cols, (long long)INT32_MAX);
  const long long items = (long long)a.n_seqs * p->n_kv_head * pl.tiles;
  // enough workgroups to fill the GPU several times over; a part is worth its join
  // from 256 keys on
  const long long want = std::max(1LL, 2048 / std::max(items, 1LL));
  const int unit = kWaves * kStep;
  long long keys = (a.max_context_len + want - 1) / want;
  keys = std::max(256LL, (keys + unit - 1) / unit * unit);
  pl.part_keys = (int)keys;
  pl.max_parts = (int)((a.max_context_len + keys - 1) / keys);
  return pl;
}

size_t part_rows(const Q4Args& a, const Plan& pl) {
  return (size_t)a.total_q * a.n_head * pl.max_parts;
}

template <int DT, int HD>
void attend(const Q4KArgs& ka, const Plan& pl, unsigned blocks, hipStream_t stream) {
  constexpr int T = kWaves * 64;
  if (pl.few && pl.nt == 1) q4_few_kernel<DT, HD, 1><<<blocks, T, 0, stream>>>(ka);
  else if (pl.few) q4_few_kernel<DT, HD, 2><<<blocks, T, 0, stream>>>(ka);
  else if (pl.nt == 1) q4_many_kernel<DT, HD, 1><<<blocks, T, 0, stream>>>(ka);
  else if constexpr (HD <= 128) q4_many_kernel<DT, HD, 2><<<blocks, T, 0, stream>>>(ka);
}

template <int DT>
void attend_dt(const Q4KArgs& ka, int hd, const Plan& pl, unsigned blocks, hipStream_t stream) {
  if (hd == 256) attend<DT, 256>(ka, pl, blocks, stream);
  else if (hd == 128) attend<DT, 128>(ka, pl, blocks, stream);
  else attend<DT, 64>(ka, pl, blocks, stream);
}

long long join_blocks(const Q4Args& a) {
  return ((long long)a.n_seqs * a.max_q_len * a.n_head + 3) / 4;
}

}  // namespace

size_t q4_workspace_bytes(const pkv_pool* p, const Q4Args& a) {
  const Plan pl = plan_of(p, a);
  return pl.max_parts == 1 ? 0 : part_rows(a, pl) * (p->head_dim + 2) * 4;
}

bool q4_fits(const pkv_pool* p, const Q4Args& a) {
  const Plan pl = plan_of(p, a);
  if ((long long)a.max_q_len * a.n_head > INT32_MAX / 2) return false;
  const long long pairs = (long long)a.n_seqs * p->n_kv_head;
  if (pairs > (1LL << 40) / pl.tiles) return false;
  const long long items = pairs * pl.tiles;
  return items <= (1LL << 40) / pl.max_parts && grid_fits(items * pl.max_parts, kWaves * 64) &&
         (long long)a.n_seqs * a.max_q_len <= (1LL << 40) / a.n_head &&
         grid_fits(join_blocks(a), 256);
}

hipError_t launch_q4_attention(const pkv_pool* p, int layer, const Q4Args& a, char* ws,
                               hipStream_t stream) {
  const Plan pl = plan_of(p, a);
  Q4KArgs ka{};
  ka.a = a;
  ka.k = p->layer_k(layer);
  ka.v = p->layer_v(layer);
  ka.kvh = p->n_kv_head;
  ka.r = a.n_head / p->n_kv_head;
  while ((1 << ka.bs_log2) < p->block_size) ++ka.bs_log2;
  ka.num_blocks = p->num_blocks;
  ka.cols = pl.cols;
  ka.tiles = pl.tiles;
  ka.part_keys = pl.part_keys;
  ka.max_parts = pl.max_parts;
  if (pl.max_parts > 1) {
    ka.o_part = reinterpret_cast<float*>(ws);
    ka.ml_part = reinterpret_cast<float2*>(ka.o_part + part_rows(a, pl) * p->head_dim);
  }
  ka.err = p->err;
  const unsigned blocks = (unsigned)((long long)a.n_seqs * p->n_kv_head * pl.tiles * pl.max_parts);
  if (a.q_dtype == PKV_F32) attend_dt<PKV_F32>(ka, p->head_dim, pl, blocks, stream);
  else if (a.q_dtype == PKV_F16) attend_dt<PKV_F16>(ka, p->head_dim, pl, blocks, stream);
  else attend_dt<PKV_BF16>(ka, p->head_dim, pl, blocks, stream);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess || pl.max_parts == 1) return e;
  const unsigned jb = (unsigned)join_blocks(a);
  if (p->head_dim == 64) q4_join_kernel<64><<<jb, 256, 0, stream>>>(ka);
  else if (p->head_dim == 128) q4_join_kernel<128><<<jb, 256, 0, stream>>>(ka);
  else q4_join_kernel<256><<<jb, 256, 0, stream>>>(ka);
  return hipGetLastError();
}

}  // namespace pkv
