// pkv_q4_attn.hip -- attention over a pool held in 4 bits (gfx950).
//
// With group g's codes c, scale s and offset m, a key's score is
//   q . k = sum_g s_g (q_g . c_g) + m_g sum(q_g)
// and the values' sum
//   o_g = sum_k (p_k s_kg) c_k + sum_k p_k m_kg,
// so both products run on the matrix cores over the codes themselves, as f16 numbers
// that two instructions make of two codes.  As f16 subnormals, bits masked out of the
// words, they need fewer, and v_mfma_f32_16x16x32_f16 takes them exactly.  But it aligns
// eight products by their operands' exponents, subnormals counting as 2^-14, and
// drops bits, downwards, that a normal number would keep: of codes as c 2^-24 up to 2^-13 of the
// largest weight (of 1 in c) each.  In the values' sum, where offsets and codes cancel, that
// was 2^-15 of results over 2000 keys.  Keys' codes of single tokens are c 2^-20, which leaves
// 2^-17 of the largest of eight query elements, times the step s: as exact as normal
// numbers where one channel in 32 is 64 times the others (2^-20 of results in norm; c 2^-24: 2^-16).
//
// A column is a query row of a chunk and one of the heads of a kv head's group.  A
// wave takes 32 keys a step: two tiles S^T = K Q^T of 16 keys, whose lanes then hold
// just the weights that they feed into the second product as its left operand.
// Weights are two f16 (2^-22): one would be off by 2^-11 of p s c, and where offset and
// code nearly cancel that is several times what rounding the result to f16 costs.
// One kernel is for few columns (decoding), one for more and for f32 queries, on f32
// instructions; chunks of 16-bit queries have one that rounds the values a tile stands
// for to f16 first, for 128 columns at once.
#include <algorithm>

#include "pkv_internal.h"
#include "pkv_q4_dev.h"

namespace pkv {
namespace {

constexpr int kWaves = 4;                  // of a workgroup; they take the steps in turn
constexpr int kStep = 32;                  // keys of a wave's step
constexpr int kIdSteps = 32;               // steps that a wave has the block ids of at once
constexpr int kFewKeys = kIdSteps * kWaves * kStep;  // keys of a part at most, for few columns
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
  int min_cols;    // a sequence with fewer columns of a kv head, or more than max_cols, is
  int max_cols;    // another launch's
  int cols;        // columns of a workgroup
  int tiles;       // workgroups that a sequence's and kv head's columns take at most
  int part_keys;   // keys of a part, a multiple of kWaves * kStep
  int max_parts;
  int join_rows;   // rows of a sequence that the join goes through
  int seq_rows;    // rows of a sequence in the partial results; 0: they are at the row's place
  float* o_part;   // [row][head][part][hd]
  float2* ml_part; // [row][head][part] (reference, sum)
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

// Place of the first part of row i (row q0 + i of all) of sequence s and a head.
__device__ __forceinline__ size_t part_at(const Q4KArgs& ka, int s, int q0, int i, int head) {
  const size_t row = ka.seq_rows ? (size_t)s * ka.seq_rows + i : (size_t)q0 + i;
  return (row * ka.a.n_head + head) * ka.max_parts;
}

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
  if (it.col0 >= it.cols || it.cols < ka.min_cols || it.cols > ka.max_cols) return false;
  int end;
  it.parts = parts_of(ka, it.col0, it.cols, it.rows, it.ctx, end);
  if (it.part >= it.parts) return false;
  it.k0 = it.part * ka.part_keys;
  it.k1 = min(end, it.k0 + ka.part_keys);
  it.all = min(it.ctx - it.rows + it.col0 / ka.r + 1, it.k1);
  return true;
}

// N bytes (a multiple of 4) of consecutive words.  ONCE: nothing else of the launch reads
// them, so the caches need not keep them.
template <int N, bool ONCE = false>
__device__ __forceinline__ void load_words(const char* p, uint32_t (&w)[N / 4]) {
  if constexpr (N == 4) {
    w[0] = *reinterpret_cast<const uint32_t*>(p);
  } else if constexpr (N == 8) {
    typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
    const u32x2* q = reinterpret_cast<const u32x2*>(p);
    const u32x2 x = ONCE ? __builtin_nontemporal_load(q) : *q;
    w[0] = x[0];
    w[1] = x[1];
  } else {
#pragma unroll
    for (int i = 0; i < N / 16; ++i) {
      const u32x4 x = ONCE ? ld16_stream(p + 16 * i) : ld16(p + 16 * i);
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

// Codes 4 bits apart in 16-bit halves as f16 numbers; hi: they are in bits 4 .. 7.  (w &
// mask) | 1024.0 is 1024 + c or 1024 + 16 c, and one packed instruction makes c of it; the
// constants are kept in registers so that the first is one instruction too.
struct CodeMasks {
  uint32_t lo = 0x000f000fu, hi = 0x00f000f0u, one = 0x64006400u;
  __device__ __forceinline__ CodeMasks() { asm("" : "+v"(lo), "+v"(hi), "+v"(one)); }
};
__device__ __forceinline__ f16x2 code_pair(const CodeMasks& k, uint32_t w, bool hi) {
  const f16x2 x = __builtin_bit_cast(f16x2, (w & (hi ? k.hi : k.lo)) | k.one);
  const f16x2 a = {(_Float16)1024.0f, (_Float16)1024.0f}, b = {(_Float16)64.0f, (_Float16)64.0f};
  const f16x2 by = {(_Float16)0.0625f, (_Float16)0.0625f};
  return hi ? x * by - b : x - a;
}

// Four words of a K code word: its channels 2 e, 2 e + 1 as f16 pairs; or as subnormals,
// c 2^-20.
__device__ __forceinline__ void k_subnormals(uint32_t w, uint32_t (&f)[4]) {
#pragma unroll
  for (int e = 0; e < 4; ++e) f[e] = (e ? w >> 4 * (e - 1) : w << 4) & 0x00f000f0u;
}
__device__ __forceinline__ void k_pairs(const CodeMasks& k, uint32_t w, uint32_t (&f)[4]) {
#pragma unroll
  for (int e = 0; e < 4; ++e)
    f[e] = __builtin_bit_cast(uint32_t, code_pair(k, e & 2 ? w >> 8 : w, e & 1));
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
__device__ __forceinline__ void v_frag(const CodeMasks& k, const uint32_t (&pair)[2][2][T / 4],
                                       int t, uint32_t (&f)[4]) {
#pragma unroll
  for (int j = 0; j < 2; ++j)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const uint32_t w = pair[j][e][t / 4];
      f[2 * j + e] = __builtin_bit_cast(uint32_t, code_pair(k, t & 2 ? w >> 8 : w, t & 1));
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
// give o_g in the tiles of group g, the others are not used.  DT: type of q, 16 bits.
// NT: such tiles, 16 / G query columns each.
//
// Bound by the reads of codes, scales and offsets, each once and past the caches (6.5
// TB/s for blocks anywhere, 5.7 through them): 256 sequences of 512 .. 4096 keys, 8 kv
// heads of 128 and 32 heads, 163 us, 48 of 12 .. 32 thousand 249, 4.8 and 5.1 TB/s.  Of the
// codes' forms above, keys' as c 2^-24 took 1.5 % less and as normal numbers 2.5 % more, values'
// as subnormals 2.5 % less.  A few
// sequences are a chain of waits (lengths, ids, keys and values, the join): 8 of
// 600 .. 9000, heads of 64, 16.9 us and 4.0 for the join.
template <int DT, int HD, int NT>
__global__ void __launch_bounds__(kWaves * 64) q4_few_kernel(Q4KArgs ka) {
  using L = Q4Layout<HD>;
  constexpr int G = L::G, T = L::T, E = 2;
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

  // ---- the first step's keys and values, under way while the queries are taken ----
  const int bs = 1 << ka.bs_log2;
  const size_t blk_stride = (size_t)ka.kvh * L::chunk(bs);
  const char* kh = ka.k + (size_t)it.g * L::chunk(bs);
  const char* vh = ka.v + (size_t)it.g * L::chunk(bs);
  const int32_t* table = a.block_tables + (size_t)it.s * a.max_blocks_per_seq;
  const int s_off = bs * (HD / 2) + (kq * G + gp) * 8, m_off = s_off + bs * G * 2;
  const int k_off = (n16 * 4 + kq) * G * 4, v_off = (kq * 16 + n16) * (2 * T);

  struct KV {
    uint32_t code[HD / 32], s[2], m[2];
  };
  auto load = [&](const char* base, int id, int key, bool keys, KV& t) {
    const int at = key & (bs - 1);
    const char* p = base + (size_t)max(id, 0) * blk_stride;
    load_words<HD / 8, true>(p + at * (HD / 2) + (keys ? k_off : v_off), t.code);
    load_words<8, true>(p + at * (G * 2) + s_off, t.s);
    load_words<8, true>(p + at * (G * 2) + m_off, t.m);
  };

  constexpr int stride = kWaves * kStep;
  int key = it.k0 + wave * kStep;
  const int ids = ids_of(ka, table, key, it.k1);  // (of all steps: parts are kFewKeys at most)
  int id[2] = {readlane_i(ids, 0), readlane_i(ids, 1)};
  KV kt[2], vt[2];
  if (key < it.k1) {
#pragma unroll
    for (int j = 0; j < 2; ++j) load(kh, id[j], key + 16 * j, true, kt[j]);
#pragma unroll
    for (int j = 0; j < 2; ++j) load(vh, id[j], key + 16 * j, false, vt[j]);
  }

  // ---- the columns' queries ----
  uint32_t qf[NT][G][4];   // right operand: channels 32 g + 8 kq + e where g is gp
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
    f[c] = fmaxf(ldexpf(fabsf(a.scale) * kLog2e, 20 - ex), 0x1p-126f);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      x[e] = ldexpf(a.scale < 0.0f ? -x[e] : x[e], ex);
      sum += x[e];
    }
    qs[c] = swap32_sum(swap16_sum(sum)) * 0x1p-20f;
#pragma unroll
    for (int e = 0; e < 8; e += 2) {
      const uint32_t w = pack_half(x[e], x[e + 1]);
#pragma unroll
      for (int g = 0; g < G; ++g) qf[c][g][e / 2] = g == gp ? w : 0u;
    }
  }

  // ---- the steps ----
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
  const CodeMasks masks;
  for (int step = 1; key < it.k1; key += stride, ++step) {
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
        k_subnormals(kt[j].code[g], kf);
#pragma unroll
        for (int c = 0; c < NT; ++c) d[c] = mfma16(kf, qf[c][g], d[c]);
      }
#pragma unroll
      for (int c = 0; c < NT; ++c)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          x[c][j][i] = col_add(fmaf(half_of(kt[j].s[i / 2], i % 2), d[c][i],
                                    half_of(kt[j].m[i / 2], i % 2) * qs[c]));
    }
    // the next step's keys
    const int next = key + stride;
    const bool more = next < it.k1;
    if (more) {
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        id[j] = readlane_i(ids, 2 * step + j);
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
      v_frag<T>(masks, pair, t, vf);
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
      sm_o[wave][c][e][lane] = y + lane_of(om[c], qc * G + t / 2);
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
    const int head = it.g * ka.r + (col - row * ka.r);
    if (it.parts == 1) {
      put(a.out, a.out_dtype, ((size_t)(it.q0 + row) * a.n_head + head) * HD + d,
          sum > 0.0f ? y / sum : 0.0f);
    } else {
      const size_t pa = part_at(ka, it.s, it.q0, row, head) + it.part;
      if (d == 0) ka.ml_part[pa] = float2{m, sum};
      ka.o_part[pa * HD + d] = y;
    }
  }
}

// ---- many columns ------------------------------------------------------------
// Tiles of 16 query columns: a product per group, scaled and added up in the lane; the
// offsets' products are one v_mfma_f32_16x16x4_f32 (its four k are groups).  f32 queries
// have all their calls here, with keys and values as f32 on f32 instructions, which
// take eight times as long: in two f16 parts queries and weights would be off by 2^-22, and
// sums by what the f16 ones drop of small products.  64 sequences of 4096 keys, 8 kv heads of 128, 32
// heads, f32: 207 us.  DT: type of q.  NT: tiles.
template <int DT, int HD, int NT>
__global__ void __launch_bounds__(kWaves * 64) q4_many_kernel(Q4KArgs ka) {
  using L = Q4Layout<HD>;
  constexpr int G = L::G, T = L::T, E = DT == PKV_F32 ? 4 : 2;
  constexpr bool F32 = DT == PKV_F32;
  constexpr int GM = (G + 3) / 4;  // products of four groups' offsets
  __shared__ float sm_m[kWaves][NT * 16], sm_l[kWaves][NT * 16];
  __shared__ float sm_o[2][NT * 16 * HD];

  const Q4Args& a = ka.a;
  Item it;
  if (!item_of(ka, it)) return;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lane = threadIdx.x & 63, kq = lane >> 4, n16 = lane & 15;

  // right operand: column n16, channels 32 g + 8 kq + e
  uint32_t qf[F32 ? 1 : NT][G][4];
  float qx[F32 ? NT : 1][G][8];
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
    const int ex = !F32 && big > 0.0f ? 14 - __builtin_amdgcn_frexp_expf(big) : 0;
    f[c] = fmaxf(ldexpf(fabsf(a.scale) * kLog2e, -ex), 0x1p-126f);
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
      sum = swap32_sum(swap16_sum(sum));
      if (kq == g % 4) qs[c][g / 4] = sum;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        if constexpr (F32) qx[c][g][e] = x[g][e];
        else if (e % 2 == 0)
          qf[c][g][e / 2] = pack_half(x[g][e], x[g][e + 1]);
      }
    }
  }

  const int bs = 1 << ka.bs_log2;
  const size_t blk_stride = (size_t)ka.kvh * L::chunk(bs);
  const char* kh = ka.k + (size_t)it.g * L::chunk(bs);
  const char* vh = ka.v + (size_t)it.g * L::chunk(bs);
  const int32_t* table = a.block_tables + (size_t)it.s * a.max_blocks_per_seq;
  const int s_off = bs * (HD / 2) + kq * G * 8;
  const int k_off = (n16 * 4 + kq) * G * 4, v_off = (kq * 16 + n16) * (2 * T);
  const int quad_off = bs * (HD / 2) + (n16 >> 2) * G * 8;
  // offsets: key n16 of group kq (and kq + 4); tokens 4 kq .. of group n16
  const int km_off = bs * (HD / 2) + bs * G * 2 + ((n16 >> 2) * G + kq % G) * 8 + (n16 & 3) * 2;
  const int vm_off = bs * (HD / 2) + bs * G * 2 + (kq * G + n16 % G) * 8;

  struct KTile {  // s: of tokens 4 kq .., for f32 queries of the four that n16 is among
    uint32_t code[HD / 32], s[2 * G], all_m[F32 ? 2 * G : 1];
    _Float16 m[GM];
  };
  struct VTile {
    uint32_t code[HD / 32], s[2 * G], m[F32 ? 2 * G : 2];  // (m: of group n16 or all)
  };
  auto load_k = [&](int id, int key, KTile& t) {
    const int at = key & (bs - 1);
    const char* p = kh + (size_t)max(id, 0) * blk_stride;
    load_words<HD / 8>(p + at * (HD / 2) + k_off, t.code);
    if constexpr (F32) {
      load_words<G * 8>(p + at * (G * 2) + quad_off, t.s);
      load_words<G * 8>(p + at * (G * 2) + quad_off + bs * G * 2, t.all_m);
    } else {
      load_words<G * 8>(p + at * (G * 2) + s_off, t.s);
#pragma unroll
      for (int b = 0; b < GM; ++b)
        t.m[b] = *reinterpret_cast<const _Float16*>(p + at * (G * 2) + km_off + 32 * b);
    }
  };
  auto load_v = [&](int id, int key, VTile& t) {
    const int at = key & (bs - 1);
    const char* p = vh + (size_t)max(id, 0) * blk_stride;
    load_words<HD / 8>(p + at * (HD / 2) + v_off, t.code);
    load_words<G * 8>(p + at * (G * 2) + s_off, t.s);
    load_words<F32 ? G * 8 : 8>(p + at * (G * 2) + (F32 ? s_off + bs * G * 2 : vm_off), t.m);
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
  const CodeMasks masks;

  constexpr int stride = kWaves * kStep;
  int key = it.k0 + wave * kStep;
  int ids = ids_of(ka, table, key, it.k1), left = kIdSteps;
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
        for (int b = 0; b < (F32 ? 0 : GM); ++b)
          acc[c] = __builtin_amdgcn_mfma_f32_16x16x4f32((float)kt[j].m[b], qs[c][b], acc[c], 0, 0, 0);
      }
#pragma unroll
      for (int g = 0; g < G; ++g) {
        if constexpr (F32) {
          const uint32_t ws = n16 & 2 ? kt[j].s[2 * g + 1] : kt[j].s[2 * g];
          const uint32_t wm = n16 & 2 ? kt[j].all_m[2 * g + 1] : kt[j].all_m[2 * g];
          const float ks = n16 & 1 ? half_of(ws, 1) : half_of(ws, 0);
          const float km = n16 & 1 ? half_of(wm, 1) : half_of(wm, 0);
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const float k = fmaf(ks, (float)(kt[j].code[g] >> q4_k_bit(e) & 15), km);
#pragma unroll
            for (int c = 0; c < NT; ++c)
              acc[c] = __builtin_amdgcn_mfma_f32_16x16x4f32(k, qx[c][g][e], acc[c], 0, 0, 0);
          }
        } else {
          uint32_t kf[4];
          k_pairs(masks, kt[j].code[g], kf);
#pragma unroll
          for (int c = 0; c < NT; ++c) {
            const f32x4 d = mfma16(kf, qf[c][g], f32x4{0, 0, 0, 0});
#pragma unroll
            for (int i = 0; i < 4; ++i)
              acc[c][i] = fmaf(half_of(kt[j].s[2 * g + i / 2], i % 2), d[i], acc[c][i]);
          }
        }
      }
#pragma unroll
      for (int c = 0; c < NT; ++c)
#pragma unroll
        for (int i = 0; i < 4; ++i) x[c][j][i] = acc[c][i];
    }
    if (--left == 0) {
      ids = ids_of(ka, table, key + stride, it.k1);
      left = kIdSteps;
    }
    const int next = key + stride;
    if (next < it.k1) {
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        id[j] = readlane_i(ids, 2 * (kIdSteps - left) + j);
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
    const bool big = !F32 && sw & 0x40004000u;
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
          if constexpr (!F32) om[c][i] *= b;
#pragma unroll
          for (int t = 0; t < T; ++t) o[c][t][i] *= b;
        }
      }
    }
    float p[NT][2][4];
#pragma unroll
    for (int c = 0; c < NT; ++c)
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          p[c][j][i] = fast_exp2(fmaf(x[c][j][i], f[c], -ref[c]));
          l[c] += p[c][j][i];
        }
    if constexpr (F32) {
      // token 4 kq + i's nibbles of channels n16 + 16 t follow those of i - 1
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int t = 0; t < T; ++t) {
            const int g = t / 2, at = i * T + t;
            const float code = (float)(vt[j].code[at / 8] >> (4 * (at % 8)) & 15);
            const float v = fmaf(half_of(vt[j].s[2 * g + i / 2], i % 2), code,
                                 half_of(vt[j].m[2 * g + i / 2], i % 2));
#pragma unroll
            for (int c = 0; c < NT; ++c)
              o[c][t] = __builtin_amdgcn_mfma_f32_16x16x4f32(p[c][j][i], v, o[c][t], 0, 0, 0);
          }
    } else {
      uint32_t mf[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) mf[e] = n16 < G ? vt[e / 2].m[e % 2] : 0u;
#pragma unroll
      for (int c = 0; c < NT; ++c) {
        uint32_t pf[2][4];
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
          for (int e = 0; e < 2; ++e)
            split_half(p[c][j][2 * e], p[c][j][2 * e + 1], pf[0][2 * j + e], pf[1][2 * j + e]);
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
          v_frag<T>(masks, pair, 2 * g + b, vf);
#pragma unroll
          for (int c = 0; c < NT; ++c)
#pragma unroll
            for (int q = 0; q < 2; ++q) o[c][2 * g + b] = mfma16(wf[c][q], vf, o[c][2 * g + b]);
        }
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
    for (int g = 0; g < (F32 ? 0 : G); ++g)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float m = lane_of(om[c][i], 16 * kq + g);
        o[c][2 * g][i] += m;
        o[c][2 * g + 1][i] += m;
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
      const int head = it.g * ka.r + (col - row * ka.r);
      const size_t at = (size_t)(it.q0 + row) * a.n_head + head;
      if (it.parts == 1) {
        const float inv = sum[c][i] > 0.0f ? 1.0f / sum[c][i] : 0.0f;
#pragma unroll
        for (int t = 0; t < T; ++t) put(a.out, a.out_dtype, at * HD + 16 * t + n16, o[c][t][i] * inv);
      } else {
        const size_t pa = part_at(ka, it.s, it.q0, row, head) + it.part;
        if (n16 == 0) ka.ml_part[pa] = float2{best[c][i], sum[c][i]};
#pragma unroll
        for (int t = 0; t < T; ++t) ka.o_part[pa * HD + 16 * t + n16] = o[c][t][i];
      }
    }
}

// ---- chunks of 16-bit queries ---------------------------------------------------
// Four waves of 32 columns share tiles of 32 keys: every thread turns some codes into
// f16 in LDS, so that the work on them is done once for 128 columns, and the products are
// those of 32x32x16 matrix instructions: S^T = K Q^T leaves a column's scores in a lane
// and the one 32 further, in the order in which they enter O^T = V^T P^T.  Values are
// rounded to f16 (2^-11 of each, at random), as weights are.  For f16 queries, whose
// results show more of that: keys stay codes, a product per group is scaled in the lane
// and the offsets' products are f32 ones, and weights are two f16.
//
// Bound by vector instructions: for a tile of 32 keys a wave needs 512 cycles of matrix
// ones and, for codes to f16, exp2, maximum and sums, some 760 of vector ones.  8
// sequences of 256 rows over 4096 keys, 8 kv heads of 128 and 64 heads: bf16 372 us, 0.72
// PFLOP/s, f16 517.  Ragged chunks leave CUs idle at the end, since keys are not split once
// there are 768 workgroups: 12 chunks of up to 200 rows over 500 to 8000 keys have
// instructions in 45 % of the cycles (27 vector, 18 matrix).  bf16 with 128 channels spills seven registers.
constexpr int kTile = 32;
constexpr float kTau = 8.0f;  // weights are at most 2^8 of their reference

template <int HD>
struct CT {
  static constexpr int G = HD / 32, T = HD / 16;
  static constexpr int KP = HD * 2 + 16;            // pitch of a key's row
  static constexpr int VP = kTile * 2 + 16;         // of a channel's values
  static constexpr int K_ITEMS = 4 * G * 8;         // (i, group, quad of keys): a word of each key
  static constexpr int VW = T >= 8 ? T / 8 : 1;     // items of a column and quad: eight channels
  static constexpr int V_ITEMS = 16 * 8 * VW;
  static constexpr int NI = (K_ITEMS + V_ITEMS + 255) / 256;
  static constexpr int GS = G < 4 ? G : 4;          // groups of a V item's channels
  static constexpr int SM = 8 * G * 8;              // bytes of a tile's scales
  static constexpr int STAGE = kTile * KP + HD * VP + 2 * SM;
};

__device__ __forceinline__ f32x16 mfma32(const u32x4& a, const u32x4& b, const f32x16& c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a),
                                                __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}
__device__ __forceinline__ float half_max(float x) {  // over a lane and the one 32 away
  auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}

template <int DT, int HD>
__global__ void __launch_bounds__(kWaves * 64)
    __attribute__((amdgpu_waves_per_eu(HD == 64 ? 3 : HD == 128 ? (DT == PKV_BF16 ? 3 : 2) : 1))) q4_chunk_kernel(Q4KArgs ka) {
  using L = Q4Layout<HD>;
  using C = CT<HD>;
  constexpr int G = C::G, T = C::T, NS = HD / 16, ND = HD / 32;
  constexpr bool EXACT = DT == PKV_F16;  // keys as codes, weights in two parts
  constexpr int NP = EXACT ? 2 : 1;
  __shared__ __attribute__((aligned(16))) char lds[2 * C::STAGE];
  const Q4Args& a = ka.a;
  Item it;
  if (!item_of(ka, it)) return;
  const int tid = threadIdx.x, lane = tid & 63, half = lane >> 5, cl = lane & 31;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);

  // ---- this wave's columns' queries ----
  const int first = it.col0 + wave * 32;
  const bool any = first < it.cols;
  const int col = first + cl;
  const bool live = col < it.cols;
  const int qi = live ? col / ka.r : 0, head = it.g * ka.r + (live ? col - qi * ka.r : 0);
  const int lim = live ? it.ctx - it.rows + qi + 1 : 0x7fffffff;
  // keys that all the wave's columns have, that any has
  const int all = min(it.ctx - it.rows + first / ka.r + 1, it.k1);
  const int most = any ? min(it.ctx - it.rows + (min(first + 32, it.cols) - 1) / ka.r + 1, it.k1) : 0;
  u32x4 qf[NS];
  float qs[EXACT ? (G + 1) / 2 : 1];
  float f;
  {
    const char* q = static_cast<const char*>(a.q) +
                    ((size_t)(it.q0 + qi) * a.q_stride + (size_t)head * HD + 8 * half) * 2;
    float x[NS][8], big = 0.0f;
#pragma unroll
    for (int i = 0; i < NS; ++i) {
      widen16<DT>(ld16(q + 32 * i), x[i]);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        if (!live || a.scale == 0.0f) x[i][e] = 0.0f;
        big = fmaxf(big, fabsf(x[i][e]));
      }
    }
    big = half_max(big);
    const int ex = big > 0.0f ? 14 - __builtin_amdgcn_frexp_expf(big) : 0;  // below 2^14
    f = fmaxf(ldexpf(fabsf(a.scale) * kLog2e, -ex), 0x1p-126f);
#pragma unroll
    for (int i = 0; i < NS; ++i) {
#pragma unroll
      for (int e = 0; e < 8; ++e) x[i][e] = ldexpf(a.scale < 0.0f ? -x[i][e] : x[i][e], ex);
#pragma unroll
      for (int e = 0; e < 8; e += 2) qf[i][e / 2] = pack_half(x[i][e], x[i][e + 1]);
    }
    if constexpr (EXACT) {  // sums of groups 2 j + half
#pragma unroll
      for (int g = 0; g < G; ++g) {
        float t = 0.0f;
#pragma unroll
        for (int e = 0; e < 8; ++e) t += x[2 * g][e] + x[2 * g + 1][e];
        t = swap32_sum(t);
        if (half == g % 2) qs[g / 2] = t;
      }
    }
  }

  // ---- tiles: a thread's items ----
  const int bs = 1 << ka.bs_log2;
  const size_t blk_stride = (size_t)ka.kvh * L::chunk(bs);
  const char* kh = ka.k + (size_t)it.g * L::chunk(bs);
  const char* vh = ka.v + (size_t)it.g * L::chunk(bs);
  const int32_t* table = a.block_tables + (size_t)it.s * a.max_blocks_per_seq;
  const CodeMasks masks;

  // block ids, 64 blocks' parts of 16 keys at a time: lane n has the n-th from `from` on
  // (-1 outside the pool and from the last key on)
  int from = it.k0, ids = 0;
  auto fetch = [&]() {
    const long long key = (long long)from + 16 * lane;
    ids = -1;
    if (key < it.k1) {
      ids = table[key >> ka.bs_log2];
      if ((unsigned)ids >= (unsigned)ka.num_blocks) {
        atomicOr(ka.err, PKV_EBIT_BLOCK);
        ids = -1;
      }
    }
  };
  fetch();

  constexpr int SG = C::GS * 2;
  uint32_t code[C::NI][4], sc[C::NI][SG], of[C::NI][SG];
  // Item j of this thread, alike for a wave: 0 of K (i, group, quad), 1 of V (word, i,
  // quad), 2 none.  The quads of a wave's items lie in one half of the tile but for
  // keys of 64 channels.
  auto kind = [&](int j) {
    const int x = wave * 64 + 256 * j;
    return x < C::K_ITEMS ? 0 : x < C::K_ITEMS + C::V_ITEMS ? 1 : 2;
  };
  auto k_quad = [&](int x) { return x / (4 * G); };
  auto v_quad = [&](int x) { return x / (16 * C::VW); };
  auto load = [&](int k0) __attribute__((always_inline)) {  // (steps of kTile from k0 = it.k0 on)
    if (k0 - from >= 64 * 16) {
      from = k0;
      fetch();
    }
    const int n = (k0 - from) / 16;
    const int id0 = max(readlane_i(ids, n), 0), id1 = max(readlane_i(ids, n + 1), 0);
#pragma unroll
    for (int j = 0; j < C::NI; ++j) {
      const int idx = tid + 256 * j, k = kind(j);
      if (k == 2) continue;
      const int x = k == 0 ? idx : idx - C::K_ITEMS;
      const int quad = k == 0 ? k_quad(x) : v_quad(x);
      const int at = (k0 + 4 * quad) & (bs - 1);
      const int id = (HD == 64 && k == 0 ? quad >> 2 : __builtin_amdgcn_readfirstlane(quad >> 2))
                         ? id1 : id0;
      const char* p = (k == 0 ? kh : vh) + (size_t)id * blk_stride;
      if (k == 0) {
        const int i = x / G % 4, g = x % G;
        const char* c = p + (uint32_t)L::k_word(at, i, g);
#pragma unroll
        for (int e = 0; e < 4; ++e) code[j][e] = *reinterpret_cast<const uint32_t*>(c + e * 16 * G);
        const char* sm = p + (uint32_t)L::s_at(bs, at, g);
        const uint2 y = *reinterpret_cast<const uint2*>(sm);
        const uint2 z = *reinterpret_cast<const uint2*>(sm + bs * G * 2);
        sc[j][0] = y.x, sc[j][1] = y.y, of[j][0] = z.x, of[j][1] = z.y;
      } else {
        const int i = x / C::VW % 16, w = x % C::VW;
        const char* c = p + (uint32_t)(L::v_bytes(at, i) + 4 * w);
        if constexpr (T == 4) {
          const uint2 y = *reinterpret_cast<const uint2*>(c);
          code[j][0] = y.x, code[j][1] = y.y;
        } else if constexpr (T == 8) {
          load_words<16>(c, code[j]);
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e) code[j][e] = *reinterpret_cast<const uint32_t*>(c + e * (T / 2));
        }
        const char* sm = p + (uint32_t)L::s_at(bs, at, 4 * w);
        load_words<C::GS * 8>(sm, sc[j]);
        load_words<C::GS * 8>(sm + bs * G * 2, of[j]);
      }
    }
    return (readlane_i(ids, n) >= 0 ? 1 : 0) | (readlane_i(ids, n + 1) >= 0 ? 2 : 0);
  };
  auto store = [&](int b) __attribute__((always_inline)) {
    char* kl = lds + b * C::STAGE;
    char* vl = kl + kTile * C::KP;
    char* sl = vl + HD * C::VP;
#pragma unroll
    for (int j = 0; j < C::NI; ++j) {
      const int idx = tid + 256 * j, k = kind(j);
      if (k == 2) continue;
      const int x = k == 0 ? idx : idx - C::K_ITEMS;
      if (k == 0) {
        const int i = x / G % 4, g = x % G, quad = k_quad(x);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          u32x4 y;
          if constexpr (EXACT) {
            uint32_t w[4];
            k_pairs(masks, code[j][e], w);
            y = u32x4{w[0], w[1], w[2], w[3]};
          } else {
            const f16x2 s2 = __builtin_bit_cast(f16x2, sc[j][e / 2]);
            const f16x2 m2 = __builtin_bit_cast(f16x2, of[j][e / 2]);
            const f16x2 s = {s2[e % 2], s2[e % 2]}, m = {m2[e % 2], m2[e % 2]};
#pragma unroll
            for (int c = 0; c < 4; ++c) {
              const f16x2 v = code_pair(masks, c & 2 ? code[j][e] >> 8 : code[j][e], c & 1) * s + m;
              y[c] = __builtin_bit_cast(uint32_t, v);
            }
          }
          st16(kl + (4 * quad + e) * C::KP + (32 * g + 8 * i) * 2, y);
        }
        if constexpr (EXACT) {
          if (i == 0) {
            *reinterpret_cast<uint2*>(sl + (quad * G + g) * 8) = uint2{sc[j][0], sc[j][1]};
            *reinterpret_cast<uint2*>(sl + C::SM + (quad * G + g) * 8) = uint2{of[j][0], of[j][1]};
          }
        }
      } else {
        // channel i + 16 t: quad 4 s + 2 b + h at (s, h, b)
        const int i = x / C::VW % 16, w = x % C::VW, quad = v_quad(x);
        const int pos = (quad >> 2) * 32 + (quad & 1) * 16 + ((quad >> 1) & 1) * 8;
        constexpr int TC = T < 8 ? T : 8;
#pragma unroll
        for (int t = 0; t < TC; ++t) {
          uint32_t y[2];
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            uint32_t pair;
            if constexpr (T == 4) pair = code[j][e];
            else pair = __builtin_amdgcn_perm(code[j][2 * e + 1], code[j][2 * e],
                                              t & 4 ? 0x07060302u : 0x05040100u);
            const f16x2 s = __builtin_bit_cast(f16x2, sc[j][t / 2 * 2 + e]);
            const f16x2 m = __builtin_bit_cast(f16x2, of[j][t / 2 * 2 + e]);
            const f16x2 v = code_pair(masks, t & 2 ? pair >> 8 : pair, t & 1) * s + m;
            y[e] = __builtin_bit_cast(uint32_t, v);
          }
          *reinterpret_cast<uint2*>(vl + (i + 16 * (t + 8 * w)) * C::VP + pos) = uint2{y[0], y[1]};
        }
      }
    }
  };

  f32x16 o[ND];
  float ref = kNone, l = 0.0f;
#pragma unroll
  for (int d = 0; d < ND; ++d)
#pragma unroll
    for (int i = 0; i < 16; ++i) o[d][i] = 0.0f;

  int in = load(it.k0);  // bit h: the block of the tile's half h is in the pool
  store(0);
  int in_next = load(it.k0 + kTile);
  __syncthreads();
  int b = 0;
  for (int k0 = it.k0; k0 < it.k1; k0 += kTile, b ^= 1) {
    if (k0 < most) {
      const char* kl = lds + b * C::STAGE;
      const char* vl = kl + kTile * C::KP;
      const char* sl = vl + HD * C::VP;
      f32x16 x;
#pragma unroll
      for (int i = 0; i < 16; ++i) x[i] = 0.0f;
      if constexpr (EXACT) {
        // offsets: key cl of group 2 j + half
#pragma unroll
        for (int j = 0; j < (G + 1) / 2; ++j) {
          const float m = *reinterpret_cast<const _Float16*>(
              sl + C::SM + ((cl >> 2) * G + 2 * j + half) * 8 + (cl & 3) * 2);
          x = __builtin_amdgcn_mfma_f32_32x32x2f32(m, qs[j], x, 0, 0, 0);
        }
#pragma unroll
        for (int g = 0; g < G; ++g) {
          f32x16 d;
#pragma unroll
          for (int i = 0; i < 16; ++i) d[i] = 0.0f;
#pragma unroll
          for (int i = 2 * g; i < 2 * g + 2; ++i)
            d = mfma32(ld16(kl + cl * C::KP + i * 32 + half * 16), qf[i], d);
#pragma unroll
          for (int i = 0; i < 16; i += 4) {
            uint32_t w[2];
            load_words<8>(sl + ((i / 2 + half) * G + g) * 8, w);
#pragma unroll
            for (int e = 0; e < 4; ++e) x[i + e] = fmaf(half_of(w[e / 2], e % 2), d[i + e], x[i + e]);
          }
        }
      } else {
#pragma unroll
        for (int i = 0; i < NS; ++i)
          x = mfma32(ld16(kl + cl * C::KP + i * 32 + half * 16), qf[i], x);
      }
      if (k0 + kTile > all || in != 3) {
#pragma unroll
        for (int i = 0; i < 16; ++i)
          if (k0 + 8 * (i / 4) + 4 * half + i % 4 >= min(lim, it.k1) || !(in >> (i / 8) & 1))
            x[i] = -INFINITY;
      }
      float mx = x[0];
#pragma unroll
      for (int i = 1; i < 16; ++i) mx = fmaxf(mx, x[i]);
      mx *= f;
      if (__builtin_amdgcn_ballot_w64(mx - ref > kTau)) {
        mx = half_max(mx);
        if (mx - ref > kTau) {
          const float by = fast_exp2(ref - mx);
          ref = mx;
          l *= by;
#pragma unroll
          for (int d = 0; d < ND; ++d)
#pragma unroll
            for (int i = 0; i < 16; ++i) o[d][i] *= by;
        }
      }
      u32x4 pf[NP][2];
#pragma unroll
      for (int i = 0; i < 16; ++i) x[i] = fast_exp2(fmaf(x[i], f, -ref));
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        if constexpr (EXACT) {
          uint32_t hi, lo;
          split_half(x[2 * e], x[2 * e + 1], hi, lo);
          pf[0][e / 4][e % 4] = hi;
          pf[1][e / 4][e % 4] = lo;
          l += x[2 * e];
          l += x[2 * e + 1];
        } else {  // the sum of what enters the product
          const uint32_t w = pack_half(x[2 * e], x[2 * e + 1]);
          const f16x2 one = {(_Float16)1.0f, (_Float16)1.0f};
          pf[0][e / 4][e % 4] = w;
          l = __builtin_amdgcn_fdot2(__builtin_bit_cast(f16x2, w), one, l, false);
        }
      }
#pragma unroll
      for (int ks = 0; ks < 2; ++ks)
#pragma unroll
        for (int d = 0; d < ND; ++d) {
          const u32x4 vf = ld16(vl + (32 * d + cl) * C::VP + 32 * ks + 16 * half);
#pragma unroll
          for (int p = 0; p < NP; ++p) o[d] = mfma32(vf, pf[p][ks], o[d]);
        }
    }
    store(b ^ 1);
    in = in_next;
    in_next = load(k0 + 2 * kTile);
    __syncthreads();
  }

  // lane: column cl, channels 32 d + 8 (i / 4) + 4 half + i % 4
  l = swap32_sum(l);
  if (!live) return;
  const size_t at = (size_t)(it.q0 + qi) * a.n_head + head;
  const size_t pa = part_at(ka, it.s, it.q0, qi, head) + it.part;
  const float by = it.parts > 1 ? 1.0f : l > 0.0f ? 1.0f / l : 0.0f;
  if (it.parts > 1 && half == 0) ka.ml_part[pa] = float2{ref, l};
#pragma unroll
  for (int d = 0; d < ND; ++d)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int ch = 32 * d + 8 * i + 4 * half;
      float y[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) y[e] = o[d][4 * i + e] * by;
      if (it.parts > 1)
        *reinterpret_cast<f32x4*>(ka.o_part + pa * HD + ch) = f32x4{y[0], y[1], y[2], y[3]};
      else if (a.out_dtype == PKV_F32)
        *reinterpret_cast<f32x4*>(static_cast<float*>(a.out) + at * HD + ch) = f32x4{y[0], y[1], y[2], y[3]};
      else
        *reinterpret_cast<uint2*>(static_cast<uint16_t*>(a.out) + at * HD + ch) =
            uint2{cvt_pk16<DT>(y[0], y[1]), cvt_pk16<DT>(y[2], y[3])};
    }
}

// Joins the parts of a query row and head: one wave each.
template <int HD>
__global__ void __launch_bounds__(256) q4_join_kernel(Q4KArgs ka) {
  constexpr int PER = HD / 64, kAtOnce = 8;  // (kAtOnce divides 64)
  const Q4Args& a = ka.a;
  const int lane = threadIdx.x & 63;
  long long u = (long long)blockIdx.x * 4 + (threadIdx.x >> 6);
  const int h = (int)(u % a.n_head);
  u /= a.n_head;
  const int i = (int)(u % ka.join_rows);
  u /= ka.join_rows;
  if (u >= a.n_seqs) return;
  int q0, rows, ctx, end;
  if (!sequence(ka, (int)u, false, q0, rows, ctx) || i >= rows || rows * ka.r < ka.min_cols ||
      rows * ka.r > ka.max_cols)
    return;
  const int col = i * ka.r + h % ka.r;
  const int parts = parts_of(ka, col / ka.cols * ka.cols, rows * ka.r, rows, ctx, end);
  if (parts == 1) return;
  const size_t at = (size_t)(q0 + i) * a.n_head + h;
  const size_t pa = part_at(ka, (int)u, q0, i, h);
  const float2* ml = ka.ml_part + pa;
  const float* o = ka.o_part + pa * HD + lane * PER;
  float m = kNone;
  for (int p = lane; p < parts; p += 64) m = fmaxf(m, ml[p].x);
  m = row_group_max(row_max16(m));
  float l = 0.0f, x[PER] = {};
  for (int from = 0; from < parts; from += 64) {
    float by = 0.0f;  // lane n: weight of part from + n
    if (from + lane < parts) {
      const float2 t = ml[from + lane];
      by = fast_exp2(t.x - m);
      l = fmaf(t.y, by, l);
    }
    for (int p = from; p < min(from + 64, parts); p += kAtOnce) {
      float y[kAtOnce][PER];
#pragma unroll
      for (int e = 0; e < kAtOnce; ++e)
#pragma unroll
        for (int j = 0; j < PER; ++j) y[e][j] = o[(size_t)min(p + e, parts - 1) * HD + j];
#pragma unroll
      for (int e = 0; e < kAtOnce; ++e) {
        const float w = lane_of(by, p - from + e);  // 0 behind the last part
#pragma unroll
        for (int j = 0; j < PER; ++j) x[j] = fmaf(y[e][j], w, x[j]);
      }
    }
  }
  l = swap32_sum(swap16_sum(row_sum16(l)));
  const float inv = l > 0.0f ? 1.0f / l : 0.0f;
#pragma unroll
  for (int j = 0; j < PER; ++j) put(a.out, a.out_dtype, at * HD + lane * PER + j, x[j] * inv);
}

// A call is one launch, or two: sequences of few columns a kv head, and chunks.
enum Kind { kFew, kMany, kChunk };
struct Launch {
  Kind kind;
  int nt, min_cols, max_cols, cols, tiles, part_keys, max_parts, seq_rows;
  size_t part_rows;  // rows that partial results are kept of
};
struct Plan {
  Launch at[2];
  int n;
};

Launch launch_of(const pkv_pool* p, const Q4Args& a, Kind kind, int nt, int min_cols, int max_cols,
                 int cols) {
  Launch l{kind, nt, min_cols, max_cols, cols, 0, 0, 0, 0, (size_t)a.total_q};
  if (max_cols < INT32_MAX && (size_t)a.n_seqs * (max_cols / (a.n_head / p->n_kv_head)) < l.part_rows) {
    l.seq_rows = max_cols / (a.n_head / p->n_kv_head);
    l.part_rows = (size_t)a.n_seqs * l.seq_rows;
  }
  const long long most = std::min((long long)a.max_q_len * (a.n_head / p->n_kv_head), (long long)max_cols);
  l.tiles = (int)std::min((most + cols - 1) / cols, (long long)INT32_MAX);
  const long long items = (long long)a.n_seqs * p->n_kv_head * l.tiles;
  // Three workgroups a CU, and for ragged batches of long contexts parts of 4096 keys at
  // most: with 2048 workgroups wanted and no limit, and with these, 64 sequences of 4096
  // keys took 107 and 92 us, 8 of 600 .. 9000 23.6 and 21.3, one of 32,000 24 and 21,
  // 48 of 12 .. 32 thousand 252 and 247, but 32 of 500 .. 16,000 79 and 85.  A part is
  // worth its join from 256 keys on, for 128 columns from 1024.  Chunks, whose rows' partial
  // results would take gigabytes, have no such limit: f32, without and with it, 16 of
  // 64 rows over 500 .. 16,000 keys took 1643 and 1581 us, 8 of 128 over 8192 1439 and 1479.
  const long long want = std::max(1LL, 768 / std::max(items, 1LL));
  const int unit = kWaves * kStep;
  long long keys = (a.max_context_len + want - 1) / want;
  keys = std::max(kind == kChunk ? 1024LL : 256LL, (keys + unit - 1) / unit * unit);
  if (most <= 32) keys = std::min(keys, (long long)kFewKeys);
  l.part_keys = (int)keys;
  l.max_parts = (int)((a.max_context_len + keys - 1) / keys);
  return l;
}

Plan plan_of(const pkv_pool* p, const Q4Args& a) {
  Plan pl{};
  const int c = 16 / (p->head_dim / 32);  // query columns of a tile for few
  const long long cols = (long long)a.max_q_len * (a.n_head / p->n_kv_head);
  if (cols <= 2 * c && a.q_dtype != PKV_F32) {
    const int nt = cols > c ? 2 : 1;
    pl.at[pl.n++] = launch_of(p, a, kFew, nt, 0, INT32_MAX, nt * c);
  } else if (cols <= 32 || a.q_dtype == PKV_F32) {
    const int nt = p->head_dim <= 128 && cols > 16 ? 2 : 1;
    pl.at[pl.n++] = launch_of(p, a, kMany, nt, 0, INT32_MAX, nt * 16);
  } else {
    if (a.n_head / p->n_kv_head <= 2 * c) {  // (some sequences may have few)
      const int nt = 2;
      pl.at[pl.n++] = launch_of(p, a, kFew, nt, 0, 2 * c, nt * c);
      pl.at[pl.n++] = launch_of(p, a, kChunk, 1, 2 * c + 1, INT32_MAX, 128);
    } else {
      pl.at[pl.n++] = launch_of(p, a, kChunk, 1, 0, INT32_MAX, 128);
    }
  }
  return pl;
}

// (row, head, part) places of a call's partial results, which its launches use in turn.
size_t part_places(const Q4Args& a, const Plan& pl) {
  size_t n = 0;
  for (int i = 0; i < pl.n; ++i)
    if (pl.at[i].max_parts > 1)
      n = std::max(n, pl.at[i].part_rows * a.n_head * pl.at[i].max_parts);
  return n;
}

template <int DT, int HD>
void attend(const Q4KArgs& ka, const Launch& l, unsigned blocks, hipStream_t stream) {
  constexpr int T = kWaves * 64;
  if (l.kind == kMany) {
    if (l.nt == 1) q4_many_kernel<DT, HD, 1><<<blocks, T, 0, stream>>>(ka);
    else if constexpr (HD <= 128) q4_many_kernel<DT, HD, 2><<<blocks, T, 0, stream>>>(ka);
  } else if constexpr (DT != PKV_F32) {
    if (l.kind == kChunk) q4_chunk_kernel<DT, HD><<<blocks, T, 0, stream>>>(ka);
    else if (l.nt == 1) q4_few_kernel<DT, HD, 1><<<blocks, T, 0, stream>>>(ka);
    else q4_few_kernel<DT, HD, 2><<<blocks, T, 0, stream>>>(ka);
  }
}

template <int DT>
void attend_dt(const Q4KArgs& ka, int hd, const Launch& l, unsigned blocks, hipStream_t stream) {
  if (hd == 256) attend<DT, 256>(ka, l, blocks, stream);
  else if (hd == 128) attend<DT, 128>(ka, l, blocks, stream);
  else attend<DT, 64>(ka, l, blocks, stream);
}

// Rows of a sequence that a launch may have parts of.
int join_rows(const pkv_pool* p, const Q4Args& a, const Launch& l) {
  return std::min(a.max_q_len, l.max_cols / (a.n_head / p->n_kv_head));
}
long long join_blocks(const Q4Args& a, int rows) {
  return ((long long)a.n_seqs * rows * a.n_head + 3) / 4;
}

}  // namespace

size_t q4_workspace_bytes(const pkv_pool* p, const Q4Args& a) {
  return part_places(a, plan_of(p, a)) * (p->head_dim + 2) * 4;
}

bool q4_fits(const pkv_pool* p, const Q4Args& a) {
  if ((long long)a.max_q_len * a.n_head > INT32_MAX / 2) return false;
  const long long pairs = (long long)a.n_seqs * p->n_kv_head;
  const Plan pl = plan_of(p, a);
  for (int i = 0; i < pl.n; ++i) {
    const Launch& l = pl.at[i];
    if (pairs > (1LL << 40) / l.tiles || pairs * l.tiles > (1LL << 40) / l.max_parts ||
        !grid_fits(pairs * l.tiles * l.max_parts, kWaves * 64))
      return false;
    const int rows = join_rows(p, a, l);
    if (l.max_parts > 1 && ((long long)a.n_seqs * rows > (1LL << 40) / a.n_head ||
                            !grid_fits(join_blocks(a, rows), 256)))
      return false;
  }
  return true;
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
  ka.err = p->err;
  ka.o_part = reinterpret_cast<float*>(ws);
  ka.ml_part = reinterpret_cast<float2*>(ka.o_part + part_places(a, pl) * p->head_dim);
  for (int i = 0; i < pl.n; ++i) {
    const Launch& l = pl.at[i];
    ka.min_cols = l.min_cols;
    ka.max_cols = l.max_cols;
    ka.cols = l.cols;
    ka.tiles = l.tiles;
    ka.part_keys = l.part_keys;
    ka.max_parts = l.max_parts;
    ka.seq_rows = l.seq_rows;
    ka.join_rows = join_rows(p, a, l);
    const unsigned blocks = (unsigned)((long long)a.n_seqs * p->n_kv_head * l.tiles * l.max_parts);
    if (a.q_dtype == PKV_F32) attend_dt<PKV_F32>(ka, p->head_dim, l, blocks, stream);
    else if (a.q_dtype == PKV_F16) attend_dt<PKV_F16>(ka, p->head_dim, l, blocks, stream);
    else attend_dt<PKV_BF16>(ka, p->head_dim, l, blocks, stream);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    if (l.max_parts == 1) continue;
    const unsigned jb = (unsigned)join_blocks(a, ka.join_rows);
    if (p->head_dim == 64) q4_join_kernel<64><<<jb, 256, 0, stream>>>(ka);
    else if (p->head_dim == 128) q4_join_kernel<128><<<jb, 256, 0, stream>>>(ka);
    else q4_join_kernel<256><<<jb, 256, 0, stream>>>(ka);
    e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  return hipSuccess;
}

}  // namespace pkv
