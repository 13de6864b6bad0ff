// pkv_prompt.hip -- causal attention of whole prompts over their own rows, packed
// (gfx950): out_i = sum_{j <= i} softmax_j(scale q_i . k_j) v_j.
//
// A unit is 32 tokens of a prompt for one query head; a workgroup of four waves has 4 QT
// units of the same kv head in a row (all heads of a token tile, then the next tile's),
// so that a tile of keys and values serves the whole group.  Tiles of 64 keys come
// through registers into double-buffered LDS.  S^T = K Q^T on 32x32 matrix
// instructions leaves the scores of a query in a lane and its partner 32 lanes
// away, in the order in which they are the right operand of O^T = V^T P^T: weights
// never leave registers.  V stays row-major in LDS and is read transposed.
#include <algorithm>

#include "pkv_device.h"
#include "pkv_internal.h"

namespace pkv {
namespace {

typedef short s16x4 __attribute__((ext_vector_type(4)));

constexpr int kWaves = 4;
constexpr int kTok = 32;  // tokens of a unit
constexpr float kTau = 8.0f;  // weights are at most 2^8 of their reference

template <int DT, int HD>
struct PT {
  static constexpr int E = DT == PKV_F32 ? 4 : 2;
  static constexpr int RB = HD * E;                       // bytes of a row
  static constexpr int KEYS = RB >= 512 ? 32 : 64;        // of a tile
  static constexpr int KP = RB + 16;                      // pitch of K rows in LDS
  static constexpr int VP = DT == PKV_F32 ? RB : RB + 32; // of V rows
  static constexpr int STAGE = KEYS * (KP + VP);
  static constexpr int CH = RB / 16;                      // 16-byte chunks of a row
  static constexpr int NL = KEYS * CH / (kWaves * 64);    // chunks a thread loads, of K and of V
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

template <int DT, int HD, int QT>
__global__ void __launch_bounds__(kWaves * 64) prompt_kernel(PromptArgs a, int max_groups) {
  using C = PT<DT, HD>;
  constexpr int NS = HD / 16, ND = HD / 32;          // k-steps of Q K, 32-channel tiles of O
  constexpr int QR = DT == PKV_F32 ? HD / 8 : NS;    // 16-byte pieces of a lane's query
  constexpr bool F32 = DT == PKV_F32;
  __shared__ __attribute__((aligned(16))) char lds[2 * C::STAGE];

  const int tid = threadIdx.x, lane = tid & 63, half = lane >> 5, col = lane & 31;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int pairs = a.n_seqs * a.n_kv_head, r = a.n_head / a.n_kv_head;
  // longest first: groups of units by their place in a prompt of max_len, from the end
  const int pair = blockIdx.x % pairs, first = max_groups - 1 - (int)(blockIdx.x / pairs);
  const int s = pair / a.n_kv_head, g = pair % a.n_kv_head;
  const int lo = a.cu_lens[s], hi = a.cu_lens[s + 1];
  if (lo < 0 || hi > a.total || lo >= hi) return;
  const int len = hi - lo;
  const long long units = (long long)((len + kTok - 1) / kTok) * r;
  const int groups = (int)((units + kWaves * QT - 1) / (kWaves * QT));
  const char* kp = static_cast<const char*>(a.k) + ((size_t)lo * a.k_stride + (size_t)g * HD) * C::E;
  const char* vp = static_cast<const char*>(a.v) + ((size_t)lo * a.v_stride + (size_t)g * HD) * C::E;
  const size_t kst = (size_t)a.k_stride * C::E, vst = (size_t)a.v_stride * C::E;
  // a query is taken negated for a negative scale, and as 0 for 0
  const float c = a.scale == 0.0f ? 1.0f : fabsf(a.scale) * 1.44269504088896340736f;

  for (long long grp = first; grp < groups; grp += max_groups) {
    const long long u0 = grp * (kWaves * QT);
    const int last_tile = (int)((min(u0 + kWaves * QT, units) - 1) / r);
    const int n_keys = min(len, (last_tile + 1) * kTok);
    const int n_tiles = (n_keys + C::KEYS - 1) / C::KEYS;

    // ---- the units' queries: right operand ----
    int tb[QT], head[QT];  // first token; -1: no unit
    u32x4 qf[QT][QR];
#pragma unroll
    for (int u = 0; u < QT; ++u) {
      const long long un = u0 + wave * QT + u;
      const bool live = un < units;
      const int tile = live ? (int)(un / r) : 0;
      tb[u] = live ? tile * kTok : -1;
      head[u] = g * r + (live ? (int)(un - (long long)tile * r) : 0);
      const int tok = min(max(tb[u], 0) + col, len - 1);
      const char* q = static_cast<const char*>(a.q) +
                      ((size_t)(lo + tok) * a.q_stride + (size_t)head[u] * HD) * C::E + half * 16;
#pragma unroll
      for (int i = 0; i < QR; ++i) {
        qf[u][i] = ld16(q + i * 32);
        if (a.scale < 0.0f) qf[u][i] ^= F32 ? 0x80000000u : 0x80008000u;
        if (a.scale == 0.0f) qf[u][i] = u32x4{0, 0, 0, 0};
      }
    }

    u32x4 kr[C::NL], vr[C::NL];
    auto load = [&](int t) __attribute__((always_inline)) {
#pragma unroll
      for (int i = 0; i < C::NL; ++i) {
        const int idx = tid + kWaves * 64 * i, key = t * C::KEYS + idx / C::CH;
        const size_t row = min(key, len - 1), b = 16 * (idx % C::CH);
        kr[i] = ld16(kp + row * kst + b);
        vr[i] = ld16(vp + row * vst + b);
        if (key >= len) {  // what lies behind the prompt may be anything
          kr[i] = u32x4{0, 0, 0, 0};
          vr[i] = u32x4{0, 0, 0, 0};
        }
      }
    };
    auto store = [&](int t) __attribute__((always_inline)) {
      char* l = lds + (t & 1) * C::STAGE;
#pragma unroll
      for (int i = 0; i < C::NL; ++i) {
        const int idx = tid + kWaves * 64 * i, key = idx / C::CH, b = 16 * (idx % C::CH);
        st16(l + key * C::KP + b, kr[i]);
        st16(l + C::KEYS * C::KP + key * C::VP + b, vr[i]);
      }
    };

    f32x16 o[QT][ND];
    float m[QT], l[QT];
#pragma unroll
    for (int u = 0; u < QT; ++u) {
      m[u] = -INFINITY;
      l[u] = 0.0f;
#pragma unroll
      for (int d = 0; d < ND; ++d)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[u][d][i] = 0.0f;
    }

    // 32 keys from k0 on for the units in [ua, ub); diag: the last keys of the units
    auto step = [&](const char* kl, const char* vl, int k0, auto ua_, auto ub_, bool diag)
                    __attribute__((always_inline)) {
      constexpr int UA = decltype(ua_)::value, UB = decltype(ub_)::value;
      f32x16 x[QT];
#pragma unroll
      for (int u = UA; u < UB; ++u)
#pragma unroll
        for (int i = 0; i < 16; ++i) x[u][i] = 0.0f;
#pragma unroll
      for (int i = 0; i < QR; ++i) {
        const u32x4 kf = ld16(kl + col * C::KP + i * 32 + half * 16);
#pragma unroll
        for (int u = UA; u < UB; ++u) {
          if constexpr (F32) {
#pragma unroll
            for (int e = 0; e < 4; ++e)
              x[u] = __builtin_amdgcn_mfma_f32_32x32x2f32(
                  __uint_as_float(kf[e]), __uint_as_float(qf[u][i][e]), x[u], 0, 0, 0);
          } else {
            x[u] = mfma32<DT>(kf, qf[u][i], x[u]);
          }
        }
      }
      u32x4 pf[QT][2];
#pragma unroll
      for (int u = UA; u < UB; ++u) {
        if (diag) {
#pragma unroll
          for (int i = 0; i < 16; ++i)
            if (8 * (i / 4) + 4 * half + i % 4 > col) x[u][i] = -INFINITY;
        }
        float mx = x[u][0];
#pragma unroll
        for (int i = 1; i < 16; ++i) mx = fmaxf(mx, x[u][i]);
        mx *= c;
        if (__builtin_amdgcn_ballot_w64(mx - m[u] > kTau)) {
          mx = half_max(mx);
          if (mx - m[u] > kTau) {
            const float by = fast_exp2(m[u] - mx);
            m[u] = mx;
            l[u] *= by;
#pragma unroll
            for (int d = 0; d < ND; ++d)
#pragma unroll
              for (int i = 0; i < 16; ++i) o[u][d][i] *= by;
          }
        }
#pragma unroll
        for (int i = 0; i < 16; ++i) x[u][i] = fast_exp2(fmaf(x[u][i], c, -m[u]));
#pragma unroll
        for (int i = 0; i < 16; ++i) l[u] += x[u][i];
        if constexpr (!F32) {
#pragma unroll
          for (int e = 0; e < 8; ++e)
            pf[u][e / 4][e % 4] = cvt_pk16<DT>(x[u][2 * e], x[u][2 * e + 1]);
        }
      }
      if constexpr (F32) {
        // k-step i: keys 8 (i / 4) + 4 half + i % 4
#pragma unroll
        for (int i = 0; i < 16; ++i)
#pragma unroll
          for (int d = 0; d < ND; ++d) {
            const float vf = *reinterpret_cast<const float*>(
                vl + (8 * (i / 4) + 4 * half + i % 4) * C::VP + (32 * d + col) * 4);
#pragma unroll
            for (int u = UA; u < UB; ++u)
              o[u][d] = __builtin_amdgcn_mfma_f32_32x32x2f32(vf, x[u][i], o[u][d], 0, 0, 0);
          }
      } else {
        // lane i of 16 gets, as element j, channel i of the row that lanes 4 j .. 4 j + 3
        // point into
        typedef __attribute__((address_space(3))) s16x4 lds_s4;
        const int i16 = lane & 15;
        const char* base = vl + (4 * half + (i16 >> 2)) * C::VP + (16 * ((lane >> 4) & 1) + 4 * (i16 & 3)) * 2;
#pragma unroll
        for (int ks = 0; ks < 2; ++ks)
#pragma unroll
          for (int d = 0; d < ND; ++d) {
            const char* b = base + 16 * ks * C::VP + 64 * d;
            const uint2 v0 = __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4*)b));
            const uint2 v1 = __builtin_bit_cast(
                uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4*)(b + 8 * C::VP)));
            const u32x4 vf = {v0.x, v0.y, v1.x, v1.y};
#pragma unroll
            for (int u = UA; u < UB; ++u) o[u][d] = mfma32<DT>(vf, pf[u][ks], o[u][d]);
          }
      }
    };

    load(0);
    __syncthreads();  // (the last group's tiles are read)
    store(0);
    load(1);
    __syncthreads();
    for (int t = 0; t < n_tiles; ++t) {
      const char* kl = lds + (t & 1) * C::STAGE;
      const char* vl = kl + C::KEYS * C::KP;
#pragma unroll
      for (int sub = 0; sub < C::KEYS / 32; ++sub) {
        const int k0 = t * C::KEYS + 32 * sub;
        const char *ks = kl + 32 * sub * C::KP, *vs = vl + 32 * sub * C::VP;
        typedef std::integral_constant<int, 0> I0;
        typedef std::integral_constant<int, 1> I1;
        typedef std::integral_constant<int, QT> IQ;
        if constexpr (QT == 1) {
          if (k0 <= tb[0]) step(ks, vs, k0, I0{}, I1{}, k0 == tb[0]);
        } else {
          if (k0 < tb[0] && k0 < tb[1]) {
            step(ks, vs, k0, I0{}, IQ{}, false);
          } else {
            if (k0 <= tb[0]) step(ks, vs, k0, I0{}, I1{}, k0 == tb[0]);
            if (k0 <= tb[1]) step(ks, vs, k0, I1{}, IQ{}, k0 == tb[1]);
          }
        }
      }
      store(t + 1);
      load(t + 2);
      __syncthreads();
    }

    // lane: query col, channels 32 d + 8 (i / 4) + 4 half + i % 4
#pragma unroll
    for (int u = 0; u < QT; ++u) {
      const float sum = swap32_sum(l[u]);
      const int tok = tb[u] + col;
      if (tb[u] < 0 || tok >= len) continue;
      const float inv = 1.0f / sum;
      const size_t at = ((size_t)(lo + tok) * a.n_head + head[u]) * HD + 4 * half;
#pragma unroll
      for (int d = 0; d < ND; ++d)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const size_t e = at + 32 * d + 8 * i;
          float y[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) y[j] = o[u][d][4 * i + j] * inv;
          if (F32 || a.out_dtype == PKV_F32) {
            *reinterpret_cast<f32x4*>(static_cast<float*>(a.out) + e) = f32x4{y[0], y[1], y[2], y[3]};
          } else {
            *reinterpret_cast<uint2*>(static_cast<uint16_t*>(a.out) + e) =
                uint2{cvt_pk16<DT>(y[0], y[1]), cvt_pk16<DT>(y[2], y[3])};
          }
        }
    }
  }
}

struct Plan {
  int qt, max_groups;
  long long blocks;
};

Plan plan_of(const PromptArgs& a) {
  Plan pl;
  pl.qt = a.dtype != PKV_F32 && a.head_dim <= 128 ? 2 : 1;
  const long long units =
      (long long)((std::min(a.max_len, a.total) + kTok - 1) / kTok) * (a.n_head / a.n_kv_head);
  const long long groups = (units + kWaves * pl.qt - 1) / (kWaves * pl.qt);
  pl.max_groups = (int)std::min(groups, (long long)INT32_MAX);
  pl.blocks = groups * a.n_seqs * a.n_kv_head;
  return pl;
}

template <int DT, int HD, int QT>
hipError_t run(const PromptArgs& a, const Plan& pl, hipStream_t stream) {
  prompt_kernel<DT, HD, QT><<<(unsigned)pl.blocks, kWaves * 64, 0, stream>>>(a, pl.max_groups);
  return hipGetLastError();
}

template <int DT, int QT>
hipError_t run_hd(const PromptArgs& a, const Plan& pl, hipStream_t stream) {
  if (a.head_dim == 64) return run<DT, 64, QT>(a, pl, stream);
  if (a.head_dim == 128) return run<DT, 128, QT>(a, pl, stream);
  return run<DT, 256, 1>(a, pl, stream);
}

}  // namespace

bool prompt_fits(const PromptArgs& a) {
  return (long long)a.n_seqs * a.n_kv_head <= INT32_MAX && grid_fits(plan_of(a).blocks, kWaves * 64);
}

hipError_t launch_prompt(const PromptArgs& a, hipStream_t stream) {
  const Plan pl = plan_of(a);
  if (a.dtype == PKV_F32) return run_hd<PKV_F32, 1>(a, pl, stream);
  if (a.dtype == PKV_F16) return run_hd<PKV_F16, 2>(a, pl, stream);
  return run_hd<PKV_BF16, 2>(a, pl, stream);
}

}  // namespace pkv
