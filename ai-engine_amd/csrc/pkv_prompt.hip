// pkv_prompt.hip -- causal attention of whole prompts over their own rows, packed
// (gfx950): out_i = sum_{j <= i} softmax_j(scale q_i . k_j) v_j.
//
// A unit is 32 tokens of a prompt for one query head, a wave's; a workgroup has four
// units of the same kv head in a row (all heads of a token tile, then the next tile's),
// so that a tile of keys and values serves the whole group.  Tiles of 32 keys come
// through registers into double-buffered LDS.  S^T = K Q^T on 32x32 matrix
// instructions leaves the scores of a query in a lane and its partner 32 lanes
// away, in the order in which they are the right operand of O^T = V^T P^T: weights
// never leave registers.  V stays row-major in LDS and is read transposed.
//
// Weights of 16-bit inputs are rounded to the inputs' type (by half a step at most, 2^-8 for
// bf16, of which a sum takes the average) and the denominator is the sum of the
// rounded ones: bf16 results are off by 2.0e-3 in norm, with weights in 32 bits by 1.6e-3.  A
// high and a low part of each would be half as many matrix instructions again.
//
// Bound by the matrix instructions and the vector ones beside them (exp2, maximum, sums):
// 8000 tokens, 64 heads of 128, bf16: 976 us, 1.07 PFLOP/s (a product of 8192^3 here
// reaches 1.24), 55 % of the cycles in matrix and 43 % in vector instructions.  Tiles of 64
// keys, two units a wave, two waves a SIMD and scores computed a tile ahead were all slower.
#include <algorithm>
#include <type_traits>

#include "pkv_device.h"
#include "pkv_internal.h"

namespace pkv {
namespace {

typedef short s16x4 __attribute__((ext_vector_type(4)));

constexpr int kWaves = 4;
constexpr int kTok = 32;  // tokens of a unit
constexpr int kRsrcWord3 = 0x00027000;  // raw buffers: 32-bit data format
constexpr float kTau = 8.0f;  // weights are at most 2^8 of their reference

template <int DT, int HD>
struct PT {
  static constexpr int E = DT == PKV_F32 ? 4 : 2;
  static constexpr int RB = HD * E;                       // bytes of a row
  static constexpr int KEYS = 32;                         // of a tile
  static constexpr int KP = RB + 16;                      // pitch of K rows in LDS
  static constexpr int VP = DT == PKV_F32 ? RB : RB + 32; // of V rows
  static constexpr int STAGE = KEYS * (KP + VP);
  static constexpr int CH = RB / 16;                      // 16-byte chunks of a row
  static constexpr int WPE = RB >= 512 ? 1 : 3;           // waves per SIMD that registers are for
};

template <int DT>
__device__ __forceinline__ f32x16 mfma32(const u32x4& a, const u32x4& b, const f32x16& c) {
  if constexpr (DT == PKV_BF16)
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a),
                                                   __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a),
                                                  __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}
__device__ __forceinline__ float half_max(float x) {  // over a lane and the one 32 away
  auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}

// Takes what is not finite out of 16 bytes of values, 0 in its place; false: all are finite.
template <int DT>
__device__ __forceinline__ bool take_odd(u32x4& w) {
  constexpr uint32_t top = DT == PKV_F32 ? 0x7f800000u : DT == PKV_F16 ? 0x7c007c00u : 0x7f807f80u;
  // an exponent of ones and 1 carry into the sign's place
  constexpr uint32_t one = DT == PKV_F32 ? 0x00800000u : DT == PKV_F16 ? 0x04000400u : 0x00800080u;
  constexpr uint32_t sign = DT == PKV_F32 ? 0x80000000u : 0x80008000u;
  uint32_t any = 0;
#pragma unroll
  for (int e = 0; e < 4; ++e) any |= (w[e] & top) + one;
  if (!(any & sign)) return false;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const uint32_t m = ((w[e] & top) + one) & sign;
    w[e] &= ~(DT == PKV_F32 ? 0u - (m >> 31) : (m >> 15) * 0xffffu);
  }
  return true;
}
// The same of one value: what is not finite, else 0.
__device__ __forceinline__ float odd_of(float x) { return fabsf(x) < INFINITY ? 0.0f : x; }

// Four neighbouring channels, widened.
template <int DT>
__device__ __forceinline__ void get4(const char* at, float (&x)[4]) {
  if constexpr (DT == PKV_F32) {
    const f32x4 w = *reinterpret_cast<const f32x4*>(at);
#pragma unroll
    for (int e = 0; e < 4; ++e) x[e] = w[e];
  } else {
    const uint2 w = *reinterpret_cast<const uint2*>(at);
    x[0] = DT == PKV_F16 ? f16lo(w.x) : bf16lo(w.x);
    x[1] = DT == PKV_F16 ? f16hi(w.x) : bf16hi(w.x);
    x[2] = DT == PKV_F16 ? f16lo(w.y) : bf16lo(w.y);
    x[3] = DT == PKV_F16 ? f16hi(w.y) : bf16hi(w.y);
  }
}

// Sum of the two 16-bit values of w, and x.
template <int DT>
__device__ __forceinline__ float pair_add(uint32_t w, float x) {
  if constexpr (DT == PKV_BF16) {
    typedef __bf16 b2 __attribute__((ext_vector_type(2)));
    return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(b2, w),
                                           __builtin_bit_cast(b2, 0x3f803f80u), x, false);
  } else {
    typedef _Float16 h2 __attribute__((ext_vector_type(2)));
    return __builtin_amdgcn_fdot2(__builtin_bit_cast(h2, w), __builtin_bit_cast(h2, 0x3c003c00u), x,
                                  false);
  }
}

// Four neighbouring channels of the output, times inv.
template <int DT>
__device__ __forceinline__ void put4(const PromptArgs& a, size_t e, const float (&x)[4], float inv) {
  const float y[4] = {x[0] * inv, x[1] * inv, x[2] * inv, x[3] * inv};
  if (DT == PKV_F32 || a.out_dtype == PKV_F32)
    *reinterpret_cast<f32x4*>(static_cast<float*>(a.out) + e) = f32x4{y[0], y[1], y[2], y[3]};
  else
    *reinterpret_cast<uint2*>(static_cast<uint16_t*>(a.out) + e) =
        uint2{cvt_pk16<DT == PKV_BF16 ? PKV_BF16 : PKV_F16>(y[0], y[1]),
              cvt_pk16<DT == PKV_BF16 ? PKV_BF16 : PKV_F16>(y[2], y[3])};
}

// Adds to four channels of a token's output what is not finite among its values in the
// rows v .. v + n - 1: their weights are above 0, however small.
template <int DT>
__device__ __forceinline__ void add_odd4(const PromptArgs& a, size_t e, const char* v, size_t st,
                                         int n) {
  float x[4] = {}, y[4];
#pragma unroll 1
  for (int j = 0; j < n; ++j) {
    get4<DT>(v + (size_t)j * st, y);
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] += odd_of(y[i]);
  }
  if (x[0] == 0.0f && x[1] == 0.0f && x[2] == 0.0f && x[3] == 0.0f) return;
  if (DT == PKV_F32 || a.out_dtype == PKV_F32) get4<PKV_F32>(static_cast<const char*>(a.out) + 4 * e, y);
  else get4<DT>(static_cast<const char*>(a.out) + 2 * e, y);
#pragma unroll
  for (int i = 0; i < 4; ++i) x[i] += y[i];
  put4<DT>(a, e, x, 1.0f);
}

// SPLIT: the four waves have one unit, and every fourth tile of its keys each, with a
// stage of LDS of their own; they join at the end.
template <int DT, int HD, bool SPLIT>
__global__ void __launch_bounds__(kWaves * 64)
    __attribute__((amdgpu_waves_per_eu(SPLIT ? 1 : PT<DT, HD>::WPE)))
    prompt_kernel(PromptArgs a, int max_groups) {
  using C = PT<DT, HD>;
  constexpr int NS = HD / 16, ND = HD / 32;          // k-steps of Q K, 32-channel tiles of O
  constexpr int QR = DT == PKV_F32 ? HD / 8 : NS;    // 16-byte pieces of a lane's query
  constexpr bool F32 = DT == PKV_F32;
  constexpr int UNITS = SPLIT ? 1 : kWaves;          // of a workgroup
  constexpr int LOADERS = SPLIT ? 64 : kWaves * 64;  // threads that a tile's loads are spread over
  constexpr int NL = C::KEYS * C::CH / LOADERS;      // 16-byte pieces a thread loads, of K and of V
  __shared__ __attribute__((aligned(16))) char lds[(SPLIT ? kWaves : 2) * C::STAGE];
  __shared__ float sm_m[SPLIT ? kWaves : 1][kTok], sm_l[SPLIT ? kWaves : 1][kTok];
  __shared__ int sm_odd;  // whether something was taken out of the values (here: ever)

  const int tid = threadIdx.x, lane = tid & 63, half = lane >> 5, col = lane & 31;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int pairs = a.n_seqs * a.n_kv_head, r = a.n_head / a.n_kv_head;
  // longest first: groups of units by their place in a prompt of max_len, from the end
  const int place = blockIdx.x / pairs, first = max_groups - 1 - place;
  // Workgroups go to the 8 XCDs in turn, so a pair would stay on one, good for its keys
  // in that cache, but prompts differ in length: unless every XCD has each prompt by
  // its heads, pairs move on from place to place (16 prompts, 2 kv heads: 186 and 121 us;
  // one prompt, where nothing is gained: 110 and 117).
  const int pair = (int)((blockIdx.x + (a.n_kv_head % 8 && a.n_seqs > 1 ? (unsigned)place : 0u)) % pairs);
  const int s = pair / a.n_kv_head, g = pair % a.n_kv_head;
  const int lo = a.cu_lens[s], hi = a.cu_lens[s + 1];
  if (lo < 0 || hi > a.total || lo >= hi) return;
  const int len = hi - lo;
  const int units = ((len - 1) / kTok + 1) * r, groups = (units + UNITS - 1) / UNITS;
  const char* kp = static_cast<const char*>(a.k) + ((size_t)lo * a.k_stride + (size_t)g * HD) * C::E;
  const char* vp = static_cast<const char*>(a.v) + ((size_t)lo * a.v_stride + (size_t)g * HD) * C::E;
  const size_t kst = (size_t)a.k_stride * C::E, vst = (size_t)a.v_stride * C::E;
  // a query is taken negated for a negative scale, and as 0 for 0
  const float c = a.scale == 0.0f ? 1.0f : fabsf(a.scale) * 1.44269504088896340736f;

  if (tid == 0) sm_odd = 0;
  for (int grp = first; grp < groups; grp += max_groups) {
    const int last_tile = (min(grp * UNITS + UNITS, units) - 1) / r;
    const int n_keys = min(len, (last_tile + 1) * kTok);
    const int n_tiles = (n_keys + C::KEYS - 1) / C::KEYS;

    // ---- this wave's unit: tokens tb .. tb + 31 of a head; none if tb < 0 ----
    const int un = grp * UNITS + (SPLIT ? 0 : wave);
    const int tb = un < units ? un / r * kTok : -1;
    const int head = g * r + (un < units ? un % r : 0);

    // A thread's pieces of a tile: rows row0 + RPT i of it, a 16-byte piece each.
    constexpr int RPT = LOADERS / C::CH;
    const int loader = SPLIT ? lane : tid, row0 = loader / C::CH;
    const uint32_t kb = 16 * (loader % C::CH);
    u32x4 kr[NL], vr[NL];
    // Buffer loads: rows behind the prompt, which may hold anything, come as 0.
    const uint32_t k_at = row0 * (uint32_t)kst + kb, v_at = row0 * (uint32_t)vst + kb;
    auto load = [&](int t) __attribute__((always_inline)) {
      const int n = min(len - t * C::KEYS, C::KEYS);  // (strides are below 2^26 bytes)
      auto rows = [&](const char* p, size_t st) {
        return __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(p + (size_t)(t * C::KEYS) * st), 0,
                                                 n > 0 ? (n - 1) * (int)st + C::RB : 0, kRsrcWord3);
      };
      const __amdgpu_buffer_rsrc_t ks = rows(kp, kst), vs = rows(vp, vst);
#pragma unroll
      for (int i = 0; i < NL; ++i) {
        kr[i] = __builtin_amdgcn_raw_buffer_load_b128(ks, k_at, RPT * i * (uint32_t)kst, 0);
        vr[i] = __builtin_amdgcn_raw_buffer_load_b128(vs, v_at, RPT * i * (uint32_t)vst, 0);
      }
    };
    // A token that is behind a query has the weight 0 there, but 0 times what is not finite is
    // not 0.  From the first unit's own tokens on, values that are not finite are taken out
    // of the tiles, and added to the results that have them at the end (one prompt of 8000
    // tokens, 64 heads of 128: 975 us without and 977 with; f32, 16 of 200: 33.5 and 36).
    const int clean = grp * UNITS / r * kTok;
    auto store = [&](int t) __attribute__((always_inline)) {
      char* l = lds + (SPLIT ? wave : t & 1) * C::STAGE;
      if (t * C::KEYS >= clean) {
        bool odd = false;
#pragma unroll
        for (int i = 0; i < NL; ++i) odd |= take_odd<DT>(vr[i]);
        if (odd) sm_odd = 1;
      }
#pragma unroll
      for (int i = 0; i < NL; ++i) {
        st16(l + (row0 + RPT * i) * C::KP + kb, kr[i]);
        st16(l + C::KEYS * C::KP + (row0 + RPT * i) * C::VP + kb, vr[i]);
      }
    };

    // ---- the queries: right operand ----
    load(SPLIT ? wave : 0);
    u32x4 qf[QR];
    {
      const int tok = min(max(tb, 0) + col, len - 1);
      const char* q = static_cast<const char*>(a.q) +
                      ((size_t)(lo + tok) * a.q_stride + (size_t)head * HD) * C::E + half * 16;
#pragma unroll
      for (int i = 0; i < QR; ++i) qf[i] = ld16(q + i * 32);
      if (a.scale <= 0.0f) {
#pragma unroll
        for (int i = 0; i < QR; ++i)
          qf[i] = a.scale < 0.0f ? qf[i] ^ (F32 ? 0x80000000u : 0x80008000u) : u32x4{0, 0, 0, 0};
      }
    }

    f32x16 o[ND];
    float m = -INFINITY, l = 0.0f;
#pragma unroll
    for (int d = 0; d < ND; ++d)
#pragma unroll
      for (int i = 0; i < 16; ++i) o[d][i] = 0.0f;

    // 32 keys; diag: the unit's own tokens
    auto step = [&](const char* kl, const char* vl, bool diag) __attribute__((always_inline)) {
      f32x16 x;
#pragma unroll
      for (int i = 0; i < 16; ++i) x[i] = 0.0f;
#pragma unroll
      for (int i = 0; i < QR; ++i) {
        const u32x4 kf = ld16(kl + col * C::KP + i * 32 + half * 16);
        if constexpr (F32) {
#pragma unroll
          for (int e = 0; e < 4; ++e)
            x = __builtin_amdgcn_mfma_f32_32x32x2f32(
                __uint_as_float(kf[e]), __uint_as_float(qf[i][e]), x, 0, 0, 0);
        } else {
          x = mfma32<DT>(kf, qf[i], x);
        }
      }
      if (diag) {
#pragma unroll
        for (int i = 0; i < 16; ++i)
          if (8 * (i / 4) + 4 * half + i % 4 > col) x[i] = -INFINITY;
      }
      float mx = x[0];
#pragma unroll
      for (int i = 1; i < 16; ++i) mx = fmaxf(mx, x[i]);
      mx *= c;
      if (__builtin_amdgcn_ballot_w64(mx - m > kTau)) {
        mx = half_max(mx);
        if (mx - m > kTau) {
          const float by = fast_exp2(m - mx);
          m = mx;
          l *= by;
#pragma unroll
          for (int d = 0; d < ND; ++d)
#pragma unroll
            for (int i = 0; i < 16; ++i) o[d][i] *= by;
        }
      }
      u32x4 pf[2];
#pragma unroll
      for (int i = 0; i < 16; ++i) x[i] = fast_exp2(fmaf(x[i], c, -m));
      if constexpr (F32) {
#pragma unroll
        for (int i = 0; i < 16; ++i) l += x[i];
        // k-step i: keys 8 (i / 4) + 4 half + i % 4
#pragma unroll
        for (int i = 0; i < 16; ++i)
#pragma unroll
          for (int d = 0; d < ND; ++d) {
            const float vf = *reinterpret_cast<const float*>(
                vl + (8 * (i / 4) + 4 * half + i % 4) * C::VP + (32 * d + col) * 4);
            o[d] = __builtin_amdgcn_mfma_f32_32x32x2f32(vf, x[i], o[d], 0, 0, 0);
          }
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          pf[e / 4][e % 4] = cvt_pk16<DT>(x[2 * e], x[2 * e + 1]);
          l = pair_add<DT>(pf[e / 4][e % 4], l);
        }
        // lane i of 16 gets, as element j, channel i of the row that lanes 4 j .. 4 j + 3
        // point into
        typedef __attribute__((address_space(3))) s16x4 lds_s4;
        const int i16 = lane & 15;
        const char* base = vl + (4 * half + (i16 >> 2)) * C::VP +
                           (16 * ((lane >> 4) & 1) + 4 * (i16 & 3)) * 2;
#pragma unroll
        for (int ks = 0; ks < 2; ++ks)
#pragma unroll
          for (int d = 0; d < ND; ++d) {
            const char* at = base + 16 * ks * C::VP + 64 * d;
            const uint2 v0 = __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4*)at));
            const uint2 v1 = __builtin_bit_cast(
                uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4*)(at + 8 * C::VP)));
            o[d] = mfma32<DT>(u32x4{v0.x, v0.y, v1.x, v1.y}, pf[ks], o[d]);
          }
      }
    };

    __syncthreads();  // (the last group's LDS is read)
    if constexpr (SPLIT) {
      for (int t = wave; t < n_tiles; t += kWaves) {
        store(t);
        load(t + kWaves);
        // the wave's LDS operations are done in this order
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
        const char* kl = lds + wave * C::STAGE;
        step(kl, kl + C::KEYS * C::KP, t * C::KEYS == tb);
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
      }
      // ---- join ----
      l = swap32_sum(l);
      if (half == 0) {
        sm_m[wave][col] = m;  // (the same in both halves)
        sm_l[wave][col] = l;
      }
      __syncthreads();  // (tiles are read)
      float* sums = reinterpret_cast<float*>(lds);  // [wave][d][i][lane]
#pragma unroll
      for (int d = 0; d < ND; ++d)
#pragma unroll
        for (int i = 0; i < 16; ++i) sums[((wave * ND + d) * 16 + i) * 64 + lane] = o[d][i];
      __syncthreads();
      float by[kWaves], top = -INFINITY;
      l = 0.0f;
#pragma unroll
      for (int w = 0; w < kWaves; ++w) top = fmaxf(top, sm_m[w][col]);
#pragma unroll
      for (int w = 0; w < kWaves; ++w) {
        by[w] = w < n_tiles ? fast_exp2(sm_m[w][col] - top) : 0.0f;
        l = fmaf(sm_l[w][col], by[w], l);
      }
      const int tok = tb + col;
      if (tok >= len) continue;
#pragma unroll
      for (int d = 0; d < ND; ++d) {  // channels 32 d + 8 wave + 4 half ..
        float y[4] = {};
#pragma unroll
        for (int w = 0; w < kWaves; ++w)
          if (w < n_tiles)
#pragma unroll
            for (int i = 0; i < 4; ++i)
              y[i] = fmaf(sums[((w * ND + d) * 16 + 4 * wave + i) * 64 + lane], by[w], y[i]);
        put4<DT>(a, ((size_t)(lo + tok) * a.n_head + head) * HD + 32 * d + 8 * wave + 4 * half, y,
                 1.0f / l);
      }
      if (sm_odd) {
#pragma unroll 1
        for (int ch = 8 * wave + 4 * half; ch < HD; ch += 32)
          add_odd4<DT>(a, ((size_t)(lo + tok) * a.n_head + head) * HD + ch,
                       vp + (size_t)clean * vst + ch * C::E, vst, tok - clean + 1);
      }
      continue;
    }
    store(0);
    load(1);
    __syncthreads();
    for (int t = 0; t < n_tiles; ++t) {
      const char* kl = lds + (t & 1) * C::STAGE;
      const char* vl = kl + C::KEYS * C::KP;
      const int k0 = t * C::KEYS;
      if (k0 <= tb) step(kl, vl, k0 == tb);
      store(t + 1);
      load(t + 2);
      __syncthreads();
    }

    // lane: query col, channels 32 d + 8 (i / 4) + 4 half + i % 4
    const float inv = 1.0f / swap32_sum(l);
    const int tok = tb + col;
    if (tb < 0 || tok >= len) continue;
    const size_t at = ((size_t)(lo + tok) * a.n_head + head) * HD + 4 * half;
#pragma unroll
    for (int d = 0; d < ND; ++d)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float y[4] = {o[d][4 * i], o[d][4 * i + 1], o[d][4 * i + 2], o[d][4 * i + 3]};
        put4<DT>(a, at + 32 * d + 8 * i, y, inv);
      }
    if (sm_odd) {
#pragma unroll 1
      for (int ch = 0; ch < HD; ch += 8)
        add_odd4<DT>(a, at + ch, vp + (size_t)clean * vst + (ch + 4 * half) * C::E, vst,
                     tok - clean + 1);
    }
  }
}

long long units_of(const PromptArgs& a) {
  return (long long)((std::min(a.max_len, a.total) + kTok - 1) / kTok) * (a.n_head / a.n_kv_head);
}
// Whether the waves of a workgroup share a unit: with so few units that the longest
// prompt's last ones take the time.  Not sharing and sharing took, us:
//   f32, 64 channels     1624 units 31, 18    3248  100, 59    6496 122, 136
//   f32, 128             512 units 74, 38     1024  76, 71     3648  86, 104   4032  537, 684
//   16 bits, 128         512 units 18, 14     1024  32, 26     2048  56, 65
//   16 bits, 64          2016 units 38, 36    2048 (of 500 tokens) 15, 19
// (f32 with 256 channels has no room for it.)
bool split_of(const PromptArgs& a) {
  const __int128 units = (__int128)units_of(a) * a.n_seqs * a.n_kv_head;
  if (a.dtype == PKV_F32) return a.head_dim <= 128 && units <= 4096 * 64 / a.head_dim;
  return units <= 1024;
}
// Groups that a prompt's kv heads have workgroups for: the bound's, or what one launch
// takes of them (workgroups then have several in turn).
long long max_groups_of(const PromptArgs& a) {
  const long long groups = split_of(a) ? units_of(a) : (units_of(a) + kWaves - 1) / kWaves;
  const long long most = 0xFFFFFFFFLL / (kWaves * 64) / ((long long)a.n_seqs * a.n_kv_head);
  return std::max(std::min(groups, most), 1LL);
}

template <int DT, int HD>
hipError_t run(const PromptArgs& a, hipStream_t stream) {
  const long long groups = max_groups_of(a);
  const unsigned blocks = (unsigned)(groups * a.n_seqs * a.n_kv_head);
  if constexpr (DT != PKV_F32 || HD != 256) {
    if (split_of(a)) {
      prompt_kernel<DT, HD, true><<<blocks, kWaves * 64, 0, stream>>>(a, (int)groups);
      return hipGetLastError();
    }
  }
  prompt_kernel<DT, HD, false><<<blocks, kWaves * 64, 0, stream>>>(a, (int)groups);
  return hipGetLastError();
}

template <int DT>
hipError_t run_hd(const PromptArgs& a, hipStream_t stream) {
  if (a.head_dim == 64) return run<DT, 64>(a, stream);
  if (a.head_dim == 128) return run<DT, 128>(a, stream);
  return run<DT, 256>(a, stream);
}

}  // namespace

bool prompt_fits(const PromptArgs& a) {
  const long long pairs = (long long)a.n_seqs * a.n_kv_head;
  return pairs <= INT32_MAX &&
         ((long long)a.total / kTok + 1) * (a.n_head / a.n_kv_head) <= INT32_MAX / 2 &&
         grid_fits(max_groups_of(a) * pairs, kWaves * 64);
}

hipError_t launch_prompt(const PromptArgs& a, hipStream_t stream) {
  if (a.dtype == PKV_F32) return run_hd<PKV_F32>(a, stream);
  if (a.dtype == PKV_F16) return run_hd<PKV_F16>(a, stream);
  return run_hd<PKV_BF16>(a, stream);
}

}  // namespace pkv
