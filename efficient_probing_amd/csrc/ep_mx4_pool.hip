// Attention pooling over the MX4 token cache, forward and backward (S = scale q.x, A = softmax over the image's tokens, P = A x;
// dA = dP.x, dS = A (dA - delta), dq = scale sum dS x), x the decoded tokens.
//
// Plain form: one workgroup per (image, query) row, a wave per token for the dot products, a lane per eight channels for the sums.
#include "ep_mx4.h"

namespace ep {

constexpr int MXP_WAVES = 4;

struct MxPool {
  ep_mx4_tokens t;
  const float* q; int64_t qb;      // forward: queries; backward: dP (B, Q, D)
  int Q; float scale;
  float* P; float* S; float* ML;   // forward outputs (S: never null here)
  const float* Pin;                // backward: P, or null (delta from ML)
  float* dS;                       // backward scratch (B, Q, N)
  float* dq;                       // backward: (B, Q, D) per-image gradients
};

// out[n] = scale * row . x[n] for the image's tokens (waves stride over them)
__device__ __forceinline__ void mx_dots(const ep_mx4_tokens& t, const uint8_t* codes, const uint8_t* scales, int len, const float* row, float scale,
                                        float* out) {
  const int words = (t.D + MX_BLOCK - 1) / MX_BLOCK * 16;
  const int lane = lane_id(), w = (int)(threadIdx.x >> 6);
  for (int n = w; n < len; n += MXP_WAVES) {
    float s = 0.f;
    for (int j = lane; 8 * j < t.D; j += 64) {
      float v[8];
      mx_decode8(*reinterpret_cast<const uint32_t*>(codes + ((int64_t)n * words + j) * 4),
                 __uint_as_float((uint32_t)scales[(int64_t)n * (words / 4) + j / 4] << 23), v);
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (8 * j + i < t.D) s += row[8 * j + i] * v[i];
    }
    s = wave_sum(s);
    if (lane == 0) out[n] = s * scale;
  }
}

__device__ __forceinline__ float mx_block_reduce(float v, bool mx, float* lds) {
  v = mx ? wave_max(v) : wave_sum(v);
  __syncthreads();
  if (lane_id() == 0) lds[threadIdx.x >> 6] = v;
  __syncthreads();
  float r = lds[0];
  for (int i = 1; i < MXP_WAVES; ++i) r = mx ? fmaxf(r, lds[i]) : r + lds[i];
  return r;
}

// out[d] = sum_n f(n) x[n][d]
template <typename F>
__device__ __forceinline__ void mx_weighted(const ep_mx4_tokens& t, const uint8_t* codes, const uint8_t* scales, int len, F&& f, float mul, float* out) {
  const int words = (t.D + MX_BLOCK - 1) / MX_BLOCK * 16;
  for (int j = (int)threadIdx.x; 8 * j < t.D; j += 64 * MXP_WAVES) {
    float acc[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    for (int n = 0; n < len; ++n) {
      float v[8];
      mx_decode8(*reinterpret_cast<const uint32_t*>(codes + ((int64_t)n * words + j) * 4),
                 __uint_as_float((uint32_t)scales[(int64_t)n * (words / 4) + j / 4] << 23), v);
      const float a = f(n);
#pragma unroll
      for (int i = 0; i < 8; ++i) acc[i] += a * v[i];
    }
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (8 * j + i < t.D) out[8 * j + i] = acc[i] * mul;
  }
}

__global__ __launch_bounds__(64 * MXP_WAVES) void ep_mx4_pool_fwd_kernel(MxPool p) {
  __shared__ float red[MXP_WAVES];
  const ep_mx4_tokens& t = p.t;
  const int b = (int)(blockIdx.x / (unsigned)p.Q), q = (int)(blockIdx.x % (unsigned)p.Q);
  int len;
  const int img = mx_image(t, b, len);
  const float bad = img < 0 ? __uint_as_float(0x7fc00000u) : 0.f;
  const uint8_t* codes = t.codes + (int64_t)(img < 0 ? 0 : img) * t.codes_bstride;
  const uint8_t* scales = t.scales + (int64_t)(img < 0 ? 0 : img) * t.scales_bstride;
  const int64_t r = (int64_t)b * p.Q + q;
  float* S = p.S + r * t.N;
  mx_dots(t, codes, scales, len, p.q + (int64_t)b * p.qb + (int64_t)q * t.D, p.scale, S);
  __syncthreads();
  float m = -INFINITY;
  for (int n = (int)threadIdx.x; n < len; n += 64 * MXP_WAVES) m = fmaxf(m, S[n]);
  m = mx_block_reduce(m, true, red);
  if (m == -INFINITY) m = 0.f;                                // no tokens
  float l = 0.f;
  for (int n = (int)threadIdx.x; n < len; n += 64 * MXP_WAVES) l += expf(S[n] - m);
  l = mx_block_reduce(l, false, red);
  for (int n = len + (int)threadIdx.x; n < t.N; n += 64 * MXP_WAVES) S[n] = -INFINITY;
  if (threadIdx.x == 0) *reinterpret_cast<f4*>(p.ML + r * 4) = f4{m + bad, l + bad, 0.f, 0.f};
  float* out = p.P + r * t.D;
  const float inv = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);
  mx_weighted(t, codes, scales, len, [&](int n) { return expf(S[n] - m); }, inv + bad, out);
}

__global__ __launch_bounds__(64 * MXP_WAVES) void ep_mx4_pool_bwd_kernel(MxPool p) {
  __shared__ float red[MXP_WAVES];
  const ep_mx4_tokens& t = p.t;
  const int b = (int)(blockIdx.x / (unsigned)p.Q), q = (int)(blockIdx.x % (unsigned)p.Q);
  int len;
  const int img = mx_image(t, b, len);
  const uint8_t* codes = t.codes + (int64_t)(img < 0 ? 0 : img) * t.codes_bstride;
  const uint8_t* scales = t.scales + (int64_t)(img < 0 ? 0 : img) * t.scales_bstride;
  const int64_t r = (int64_t)b * p.Q + q;
  const float* dP = p.q + r * t.D;
  float delta;
  if (p.Pin) {
    delta = 0.f;
    for (int d = (int)threadIdx.x; d < t.D; d += 64 * MXP_WAVES) delta += dP[d] * p.Pin[r * t.D + d];
    delta = mx_block_reduce(delta, false, red);
  } else {
    delta = p.ML[r * 4 + 2];
  }
  const float m = p.ML[r * 4], l = p.ML[r * 4 + 1], inv = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);
  float* dS = p.dS + r * t.N;
  mx_dots(t, codes, scales, len, dP, 1.f, dS);
  __syncthreads();
  for (int n = (int)threadIdx.x; n < len; n += 64 * MXP_WAVES) dS[n] = expf(p.S[r * t.N + n] - m) * inv * (dS[n] - delta);
  __syncthreads();
  mx_weighted(t, codes, scales, len, [&](int n) { return dS[n]; }, p.scale, p.dq + r * t.D);
}

__global__ __launch_bounds__(256) void ep_mx4_sum_images_kernel(const float* __restrict__ part, int B, int64_t QD, float* __restrict__ dq, int accumulate) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= QD) return;
  float s = accumulate ? dq[i] : 0.f;
  for (int b = 0; b < B; ++b) s += part[(int64_t)b * QD + i];
  dq[i] = s;
}

}  // namespace ep

using namespace ep;

extern "C" {

size_t ep_mx4_pool_workspace_bytes(int B, int N, int D, int Q) {
  if (B <= 0 || N <= 0 || D <= 0 || Q <= 0) return 0;
  return round_up(((size_t)B * Q * N + (size_t)B * Q * D) * sizeof(float), 256);
}

static int mx_pool_check(const ep_mx4_tokens* t, int Q, void* ws, size_t bytes, const char* what) {
  EP_TRY(mx4_check(t, what));
  EP_REQUIRE(Q > 0, EP_E_ARG, "%s: Q = %d", what, Q);
  EP_REQUIRE(t->D <= MX_MAX_D, EP_E_SHAPE, "%s: D = %d > %d", what, t->D, MX_MAX_D);
  EP_REQUIRE(ws && aligned16(ws), EP_E_ARG, "%s: the workspace must be given and 16-byte aligned", what);
  const size_t need = ep_mx4_pool_workspace_bytes(t->B, t->N, t->D, Q);
  EP_REQUIRE(bytes >= need, EP_E_WORKSPACE, "%s: workspace %zu < %zu", what, bytes, need);
  return 0;
}

int ep_mx4_pool_forward(const ep_mx4_tokens* t, const float* queries, int64_t q_bstride, int Q, float scale, float* P, float* S, float* ML, void* workspace,
                        size_t workspace_bytes, ep_stream_t stream) {
  EP_TRY(mx_pool_check(t, Q, workspace, workspace_bytes, "ep_mx4_pool_forward"));
  EP_REQUIRE(queries && P && ML, EP_E_ARG, "ep_mx4_pool_forward: null pointer");
  EP_REQUIRE(aligned16(ML), EP_E_ALIGN, "ep_mx4_pool_forward: ML must be 16-byte aligned");
  EP_REQUIRE(q_bstride == 0 || q_bstride >= (int64_t)Q * t->D, EP_E_SHAPE, "ep_mx4_pool_forward: query batch stride %lld", (long long)q_bstride);
  MxPool p{};
  p.t = *t; p.q = queries; p.qb = q_bstride; p.Q = Q; p.scale = scale; p.P = P; p.S = S ? S : (float*)workspace; p.ML = ML;
  hipLaunchKernelGGL(ep_mx4_pool_fwd_kernel, dim3((unsigned)t->B * Q), dim3(64 * MXP_WAVES), 0, (hipStream_t)stream, p);
  EP_LAUNCH_CHECK("ep_mx4_pool_fwd_kernel");
  return 0;
}

int ep_mx4_pool_backward(const ep_mx4_tokens* t, int Q, float scale, const float* S, const float* ML, const float* P, const float* dP, float* dq,
                         int per_image, int accumulate, void* workspace, size_t workspace_bytes, ep_stream_t stream) {
  EP_TRY(mx_pool_check(t, Q, workspace, workspace_bytes, "ep_mx4_pool_backward"));
  EP_REQUIRE(S && ML && dP && dq, EP_E_ARG, "ep_mx4_pool_backward: null pointer");
  EP_REQUIRE(aligned16(ML), EP_E_ALIGN, "ep_mx4_pool_backward: ML must be 16-byte aligned");
  EP_REQUIRE(!(per_image && accumulate), EP_E_UNSUPPORTED, "ep_mx4_pool_backward: accumulate is for shared queries");
  MxPool p{};
  p.t = *t; p.q = dP; p.Q = Q; p.scale = scale; p.S = const_cast<float*>(S); p.ML = const_cast<float*>(ML); p.Pin = P;
  p.dS = (float*)workspace;
  p.dq = per_image ? dq : p.dS + (size_t)t->B * Q * t->N;
  hipStream_t st = (hipStream_t)stream;
  hipLaunchKernelGGL(ep_mx4_pool_bwd_kernel, dim3((unsigned)t->B * Q), dim3(64 * MXP_WAVES), 0, st, p);
  EP_LAUNCH_CHECK("ep_mx4_pool_bwd_kernel");
  if (!per_image) {
    const int64_t QD = (int64_t)Q * t->D;
    hipLaunchKernelGGL(ep_mx4_sum_images_kernel, dim3((unsigned)((QD + 255) / 256)), dim3(256), 0, st, p.dq, t->B, QD, dq, accumulate);
    EP_LAUNCH_CHECK("ep_mx4_sum_images_kernel");
  }
  return 0;
}

}  // extern "C"
