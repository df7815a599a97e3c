// Argument blocks and device pieces shared by the kernels that read a key /
// value cache beside the plain decode: the drafted tree (attn_tree.hip), the
// decode that accumulates attention weights (attn_accum.hip), a prompt's key
// weights (attn_keyw.hip) and the eviction (kv_evict.hip).
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "attn_mfma_dev.h"
#include "kat_common.h"

namespace kat {

// t = 2 sigma(s) of the rational sigmoid, r = 1 / (|s| + 1) (v_rcp_f32, 1 ulp):
// s / (|s| + 1) + 1 is r for s < 0 and 2 - r for s >= 0. The first form has no
// cancellation, so keys far below the query keep their relative precision
// (1 + s r, one instruction less, has lost 5 bits at s = -30).
__device__ __forceinline__ float sig2(float s) {
  const float r = __builtin_amdgcn_rcpf(fabsf(s) + 1.f);
  return s < 0.f ? r : 2.f - r;
}
// t^4 = 16 sigma^4
__device__ __forceinline__ float sig2_pow4(float s) {
  const float t = sig2(s), t2 = t * t;
  return t2 * t2;
}

// 16 bytes of a cache row that is read once per call (non-temporal, see attn_decode.hip)
__device__ __forceinline__ mfma::i16x8 ld_piece_nt(const char* p) {
  return __builtin_bit_cast(mfma::i16x8, __builtin_nontemporal_load(reinterpret_cast<const mfma::i32x4*>(p)));
}

// c += A B^T over one 64-byte column block of 16 rows on each side; lane
// (g = lane / 16, li = lane % 16) holds bytes 16 g .. 16 g + 15 of row li of A
// and of row li of B; C[4 g + j][li], rows of A by rows of B. 16-bit types: one
// 16x16x32 product. fp32: four 16x16x4 products, step j taking column 4 g + j.
template <typename T> __device__ __forceinline__ mfma::f32x4 dot64(const mfma::i16x8& a, const mfma::i16x8& b,
                                                                   mfma::f32x4 c) {
  if constexpr (sizeof(T) == 2) {
    return mfma::Mfma<T>::mma(a, b, c);
  } else {
    const mfma::f32x4 x = __builtin_bit_cast(mfma::f32x4, a), y = __builtin_bit_cast(mfma::f32x4, b);
#pragma unroll
    for (int j = 0; j < 4; ++j) c = __builtin_amdgcn_mfma_f32_16x16x4f32(x[j], y[j], c, 0, 0, 0);
    return c;
  }
}

// 1 / d; 0 for a row sum of 0 with eps = 0, whose numerators are 0 too
__device__ __forceinline__ float inv_sum(float d) { return d != 0.f ? 1.f / d : 0.f; }

// Layout width of a head dim in the kernels over a cache: the width of its
// columns padded to 32 (fp32 only), 64, 128 or 256; 0 if none serves (16-bit
// types: multiples of 8 up to 256; fp32: multiples of 4 up to 128 -- the sets
// of kat_attn_decode).
inline int cache_layout(int64_t D, int dtype) {
  if (dtype == KAT_F32) return D < 4 || D > 128 || D % 4 ? 0 : D <= 32 ? 32 : D <= 64 ? 64 : 128;
  if (dtype == KAT_BF16 || dtype == KAT_F16) return D < 8 || D > 256 || D % 8 ? 0 : D <= 64 ? 64 : D <= 128 ? 128 : 256;
  return 0;
}

}  // namespace kat
