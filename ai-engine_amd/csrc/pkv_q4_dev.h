// pkv_q4_dev.h -- layout of PKV_Q4 pools on the device (include/pagedkv.h, "a cache
// held in 4 bits"): a layer's K or V is [num_blocks][n_kv_head][chunk], the chunk of a
// block and kv head holding its codes, then the scales s, then the offsets m.
#pragma once

#include "pkv_device.h"

namespace pkv {

template <int HD>
struct Q4Layout {
  static constexpr int G = HD / 32;  // groups of a row
  static constexpr int T = HD / 16;  // V channels of a column i: i + 16 t
  static constexpr size_t chunk(int bs) { return (size_t)bs * HD * 5 / 8; }
  // byte offsets within a chunk
  static __device__ __forceinline__ int k_word(int tok, int i, int g) {
    return ((tok * 4 + i) * G + g) * 4;
  }
  static __device__ __forceinline__ int v_bytes(int tok, int i) {
    return (((tok >> 2) * 16 + i) * 4 + (tok & 3)) * (T / 2);
  }
  static __device__ __forceinline__ int s_at(int bs, int tok, int g) {
    return bs * (HD / 2) + (((tok >> 2) * G + g) * 4 + (tok & 3)) * 2;
  }
  static __device__ __forceinline__ int m_at(int bs, int tok, int g) {
    return s_at(bs, tok, g) + bs * G * 2;
  }
};

// Bit of channel e (of eight) in a word of K codes: even and odd channels in its two
// halves, so that one mask leaves a pair of them in 16 bits each.
__device__ __forceinline__ constexpr int q4_k_bit(int e) { return 4 * (e / 2 + 4 * (e % 2)); }

}  // namespace pkv
