// MX4 token cache: writer and reader.
//
// Writer: a lane takes eight channels of a token, four lanes one 32-channel group: amax over the group in two DPP steps, the
// exponent from its bits, eight codes by the E2M1 conversion instruction (round to nearest, ties to even, cut off at 6).
// Reader: the inverse, through an optional image index.  Bound: HBM (the writer reads 4 or 2 bytes a value and writes 17/32).
#include "ep_mx4.h"

namespace ep {

template <int DT> struct MxElem;               // 0 fp32, 1 bf16, 2 fp16
template <> struct MxElem<0> { typedef float T; };
template <> struct MxElem<1> { typedef uint16_t T; };
template <> struct MxElem<2> { typedef _Float16 T; };

template <int DT>
__device__ __forceinline__ float mx_to_f32(typename MxElem<DT>::T v) {
  if constexpr (DT == 1) return __uint_as_float((uint32_t)v << 16);
  else return (float)v;
}

template <int DT, bool VEC>
__device__ __forceinline__ void mx_load8(const typename MxElem<DT>::T* p, int valid, float (&v)[8]) {
  if constexpr (VEC) {
    if constexpr (DT == 0) {
      const f4 a = reinterpret_cast<const f4*>(p)[0], b = reinterpret_cast<const f4*>(p)[1];
      v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
    } else {
      const uint4 w = *reinterpret_cast<const uint4*>(p);
      const uint32_t r[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const f4 f = h16x4_to_f4(uint2{r[i], 0u}, DT == 2);
        v[2 * i] = f.x; v[2 * i + 1] = f.y;
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = i < valid ? mx_to_f32<DT>(p[i]) : 0.f;
  }
}

// exponent byte of a group from its largest magnitude: floor(log2) - 2, one more from 1.75 * 2^floor on
__device__ __forceinline__ int mx_exponent(float amax) {
  const uint32_t u = __float_as_uint(amax);
  const int ex = (int)(u >> 23);
  if (ex == 255) return 255;                             // an infinity or a NaN among the group
  int s = ex - 2 + ((u & 0x7fffffu) >= 0x600000u ? 1 : 0);
  return s < 2 ? 2 : (s > 252 ? 252 : s);
}

// one lane per eight channels; grid.x over B * N * Dp / 8
template <int DT, bool VEC>
__global__ __launch_bounds__(256) void ep_mx4_quantize_kernel(const typename MxElem<DT>::T* __restrict__ x, int64_t xb, int64_t xt, int64_t first, int64_t total,
                                                              int N, int D, int words, uint8_t* __restrict__ codes,
                                                              uint8_t* __restrict__ scales, int64_t cb, int64_t sb) {
  const int64_t id = first + (int64_t)blockIdx.x * 256 + threadIdx.x;
  const bool in = id < total;
  const int64_t row = in ? id / words : 0;
  const int j = in ? (int)(id - row * words) : 0;
  const int64_t b = row / N;
  const int n = (int)(row - b * N);
  float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  if (in && 8 * j < D) mx_load8<DT, VEC>(x + b * xb + (int64_t)n * xt + 8 * j, D - 8 * j, v);
  // magnitudes are compared as bit patterns: an infinity or a NaN is larger than every number
  uint32_t am = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) { const uint32_t a = __float_as_uint(v[i]) & 0x7fffffffu; am = a > am ? a : am; }
#pragma unroll
  for (int step = 0; step < 2; ++step) {
    const uint32_t o = step == 0 ? __builtin_amdgcn_update_dpp(0u, am, 0xB1, 0xF, 0xF, true) : __builtin_amdgcn_update_dpp(0u, am, 0x4E, 0xF, 0xF, true);
    am = o > am ? o : am;
  }
  if (!in) return;
  const int s = mx_exponent(__uint_as_float(am));
  uint32_t w = 0;
  if (s != 255) {
    const float sc = __uint_as_float((uint32_t)s << 23);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[0], v[1], sc, 0);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[2], v[3], sc, 1);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[4], v[5], sc, 2);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[6], v[7], sc, 3);
    // the conversion leaves code 8 (-0) for small negative values: one code per value, so that equal tokens have equal bytes
    w &= 0x77777777u | ((w | w << 1 | w << 2) << 1 & 0x88888888u);
  }
  *reinterpret_cast<uint32_t*>(codes + b * cb + ((int64_t)n * words + j) * 4) = w;
  if ((j & 3) == 0) scales[b * sb + (int64_t)n * (words / 4) + j / 4] = (uint8_t)s;
}

template <int DT>
__device__ __forceinline__ uint32_t mx_out_pair(uint32_t bf2) {      // two bf16 -> two 16-bit outputs
  if constexpr (DT == 1) return bf2;
  typedef _Float16 h2v __attribute__((ext_vector_type(2)));
  const h2v h = {(_Float16)__uint_as_float(bf2 << 16), (_Float16)__uint_as_float(bf2 & 0xffff0000u)};
  return __builtin_bit_cast(uint32_t, h);
}

// one lane per eight channels of the output; VEC: D % 8 == 0
template <int DT, bool VEC>
__global__ __launch_bounds__(256) void ep_mx4_dequantize_kernel(ep_mx4_tokens t, int64_t first, int64_t total, int words, int words_out, typename MxElem<DT>::T* __restrict__ out) {
  const int64_t id = first + (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (id >= total) return;
  const int64_t row = id / words_out;
  const int j = (int)(id - row * words_out);
  const int b = (int)(row / t.N);
  const int n = (int)(row - (int64_t)b * t.N);
  int len;
  const int img = mx_image(t, b, len);
  uint32_t w = 0;
  float sc = __uint_as_float(0x7f800000u);                   // outside the cache: NaN
  if (img >= 0) {
    w = *reinterpret_cast<const uint32_t*>(t.codes + (int64_t)img * t.codes_bstride + ((int64_t)n * words + j) * 4);
    sc = __uint_as_float((uint32_t)t.scales[(int64_t)img * t.scales_bstride + (int64_t)n * (words / 4) + j / 4] << 23);
  }
  const uint32_t p[4] = {mx_pair<0>(w, sc), mx_pair<1>(w, sc), mx_pair<2>(w, sc), mx_pair<3>(w, sc)};
  typename MxElem<DT>::T* o = out + row * t.D + 8 * j;
  if constexpr (VEC) {
    if constexpr (DT == 0) {
      reinterpret_cast<f4*>(o)[0] = f4{__uint_as_float(p[0] << 16), __uint_as_float(p[0] & 0xffff0000u), __uint_as_float(p[1] << 16), __uint_as_float(p[1] & 0xffff0000u)};
      reinterpret_cast<f4*>(o)[1] = f4{__uint_as_float(p[2] << 16), __uint_as_float(p[2] & 0xffff0000u), __uint_as_float(p[3] << 16), __uint_as_float(p[3] & 0xffff0000u)};
    } else {
      *reinterpret_cast<uint4*>(o) = uint4{mx_out_pair<DT>(p[0]), mx_out_pair<DT>(p[1]), mx_out_pair<DT>(p[2]), mx_out_pair<DT>(p[3])};
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if (8 * j + i >= t.D) break;
      const float f = __uint_as_float((i & 1) ? p[i / 2] & 0xffff0000u : p[i / 2] << 16);
      if constexpr (DT == 0) o[i] = f;
      else if constexpr (DT == 1) o[i] = (uint16_t)(__float_as_uint(f) >> 16);
      else o[i] = (_Float16)f;
    }
  }
}

constexpr int64_t MX_SLICE = 1 << 30;            // threads of a launch (HIP takes less than 2^32)
static unsigned mx_slice(int64_t first, int64_t total) { return (unsigned)(((total - first < MX_SLICE ? total - first : MX_SLICE) + 255) / 256); }

int mx4_check(const ep_mx4_tokens* t, const char* what) {
  EP_REQUIRE(t && t->codes && t->scales, EP_E_ARG, "%s: null pointer", what);
  EP_REQUIRE(t->B > 0 && t->N > 0 && t->D > 0 && t->M > 0 && t->M <= 2147483647 && t->N <= 1 << 30, EP_E_ARG, "%s: B %d, N %d, D %d, M %lld must be positive", what, t->B, t->N,
             t->D, (long long)t->M);
  EP_REQUIRE(t->image_index || t->B <= t->M, EP_E_ARG, "%s: a batch of %d images from a cache of %lld needs an image_index", what, t->B, (long long)t->M);
  const int64_t nb = mx_blocks(t->D);
  EP_REQUIRE(t->M == 1 || (t->codes_bstride >= t->N * nb * 64 && t->scales_bstride >= t->N * nb * 4), EP_E_SHAPE,
             "%s: image strides %lld / %lld below one image of %d x %d", what, (long long)t->codes_bstride, (long long)t->scales_bstride, t->N, t->D);
  EP_REQUIRE(aligned16(t->codes) && t->codes_bstride % 16 == 0 && (reinterpret_cast<uintptr_t>(t->scales) & 3u) == 0 && t->scales_bstride % 4 == 0,
             EP_E_ALIGN, "%s: codes must be 16-byte and scales 4-byte aligned (pointers and image strides)", what);
  return 0;
}

}  // namespace ep

using namespace ep;

extern "C" {

int ep_mx4_quantize(const void* x, int x_dtype, int64_t x_bstride, int64_t x_tstride, int B, int N, int D, uint8_t* codes, uint8_t* scales,
                    int64_t codes_bstride, int64_t scales_bstride, ep_stream_t stream) {
  ep_mx4_tokens t{};
  t.codes = codes; t.scales = scales; t.codes_bstride = codes_bstride; t.scales_bstride = scales_bstride; t.M = B; t.B = B; t.N = N; t.D = D;
  EP_REQUIRE(x, EP_E_ARG, "ep_mx4_quantize: null pointer");
  EP_TRY(mx4_check(&t, "ep_mx4_quantize"));
  EP_REQUIRE(x_dtype >= EP_DTYPE_F32 && x_dtype <= EP_DTYPE_F16, EP_E_UNSUPPORTED, "ep_mx4_quantize: dtype %d", x_dtype);
  EP_REQUIRE((N == 1 || x_tstride >= 0) && (B == 1 || x_bstride >= 0), EP_E_ARG, "ep_mx4_quantize: negative stride");
  const int words = mx_blocks(D) * 16;
  const int64_t total = (int64_t)B * N * words;
  const int per16 = x_dtype == EP_DTYPE_F32 ? 4 : 8;
  const bool vec = D % 8 == 0 && aligned16(x) && (B == 1 || x_bstride % per16 == 0) && (N == 1 || x_tstride % per16 == 0);
  hipStream_t st = (hipStream_t)stream;
#define EP_MXQ(DT, V)                                                                                                                    \
  hipLaunchKernelGGL((ep_mx4_quantize_kernel<DT, V>), dim3(mx_slice(first, total)), dim3(256), 0, st, (const MxElem<DT>::T*)x, x_bstride, x_tstride, first, \
                     total, N, D, words, codes, scales, codes_bstride, scales_bstride)
  for (int64_t first = 0; first < total; first += MX_SLICE) {
    if (x_dtype == EP_DTYPE_F32) { if (vec) EP_MXQ(0, true); else EP_MXQ(0, false); }
    else if (x_dtype == EP_DTYPE_BF16) { if (vec) EP_MXQ(1, true); else EP_MXQ(1, false); }
    else { if (vec) EP_MXQ(2, true); else EP_MXQ(2, false); }
#undef EP_MXQ
    EP_LAUNCH_CHECK("ep_mx4_quantize_kernel");
  }
  return 0;
}

int ep_mx4_dequantize(const ep_mx4_tokens* t, void* out, int out_dtype, ep_stream_t stream) {
  EP_TRY(mx4_check(t, "ep_mx4_dequantize"));
  EP_REQUIRE(out, EP_E_ARG, "ep_mx4_dequantize: null pointer");
  EP_REQUIRE(aligned16(out), EP_E_ALIGN, "ep_mx4_dequantize: out must be 16-byte aligned");
  EP_REQUIRE(out_dtype >= EP_DTYPE_F32 && out_dtype <= EP_DTYPE_F16, EP_E_UNSUPPORTED, "ep_mx4_dequantize: dtype %d", out_dtype);
  const int words = mx_blocks(t->D) * 16, words_out = (t->D + 7) / 8;
  const int64_t total = (int64_t)t->B * t->N * words_out;
  const bool vec = t->D % 8 == 0;
  hipStream_t st = (hipStream_t)stream;
#define EP_MXD(DT, V) \
  hipLaunchKernelGGL((ep_mx4_dequantize_kernel<DT, V>), dim3(mx_slice(first, total)), dim3(256), 0, st, *t, first, total, words, words_out, (MxElem<DT>::T*)out)
  for (int64_t first = 0; first < total; first += MX_SLICE) {
    if (out_dtype == EP_DTYPE_F32) { if (vec) EP_MXD(0, true); else EP_MXD(0, false); }
    else if (out_dtype == EP_DTYPE_BF16) { if (vec) EP_MXD(1, true); else EP_MXD(1, false); }
    else { if (vec) EP_MXD(2, true); else EP_MXD(2, false); }
#undef EP_MXD
    EP_LAUNCH_CHECK("ep_mx4_dequantize_kernel");
  }
  return 0;
}

}  // extern "C"
