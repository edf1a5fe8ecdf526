// MX4 token cache (MXFP4: E2M1 codes, one E8M0 scale byte per 32 channels): device helpers shared by the cache's writer / reader
// (ep_mx4.hip) and the attention over it (ep_mx4_pool.hip), and the internal interface of the latter.
#pragma once
#include "ep_common.h"

namespace ep {

constexpr int MX_BLOCK = 128;                 // channels of a row block: 64 code bytes + 4 scale bytes
constexpr int MX_MAX_D = 4096;

typedef __bf16 mx_bf2 __attribute__((ext_vector_type(2)));

inline int mx_blocks(int D) { return (D + MX_BLOCK - 1) / MX_BLOCK; }

// two codes (byte SEL of w) -> two bf16 values times the power of two in scale's exponent bits.  Exact: E2M1 has two significant
// bits.  The instruction looks at nothing but bits 30:23 of the scale; 255 there makes both values NaN.
template <int SEL>
__device__ __forceinline__ uint32_t mx_pair(uint32_t w, float scale) {
  return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, SEL));
}
// scale byte g (0 .. 3) of the dword of a row block, moved to the exponent bits (the other bytes are left beside it)
__device__ __forceinline__ float mx_scale(uint32_t four, int g) {
  return __uint_as_float(__builtin_amdgcn_alignbit(four, four, (uint32_t)(8 * g + 9)));
}
__device__ __forceinline__ void mx_decode8(uint32_t w, float scale, float (&v)[8]) {
  const uint32_t p[4] = {mx_pair<0>(w, scale), mx_pair<1>(w, scale), mx_pair<2>(w, scale), mx_pair<3>(w, scale)};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    v[2 * i] = __uint_as_float(p[i] << 16);
    v[2 * i + 1] = __uint_as_float(p[i] & 0xffff0000u);
  }
}

// A word of a per-image table at a wave-uniform place, through the scalar cache: a vector load would have to wait for every tile load
// in front of it.  (Nothing writes these tables while the kernel runs.)
__device__ __forceinline__ int mx_uniform_load(const int32_t* p) {
  int v;
  const uint64_t a = (uint64_t)p;
  const uint64_t u = (uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)a) | (uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)(a >> 32)) << 32;
  asm volatile("s_load_dword %0, %1, 0x0\n\ts_waitcnt lgkmcnt(0)" : "=s"(v) : "s"(u) : "memory");
  return v;
}

// image of the call -> image of the cache (-1: an index outside the cache) and its token count
__device__ __forceinline__ int mx_image(const ep_mx4_tokens& t, int b, int& len) {
  int64_t img = t.image_index ? (int64_t)t.image_index[b] : (int64_t)b;
  len = 0;
  if (img < 0 || img >= t.M) return -1;
  len = t.lengths ? t.lengths[img] : t.N;
  len = len < 0 ? 0 : (len > t.N ? t.N : len);
  return (int)img;
}

// the same for a wave-uniform b
__device__ __forceinline__ int mx_image_uniform(const ep_mx4_tokens& t, int b, int& len) {
  const int img = t.image_index ? mx_uniform_load(t.image_index + b) : b;
  len = 0;
  if (img < 0 || (int64_t)img >= t.M) return -1;
  len = t.lengths ? mx_uniform_load(t.lengths + img) : t.N;
  len = len < 0 ? 0 : (len > t.N ? t.N : len);
  return img;
}

int mx4_check(const ep_mx4_tokens* t, const char* what);

}  // namespace ep
