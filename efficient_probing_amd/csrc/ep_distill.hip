// Distillation from a teacher's top logits: loss and logit gradient of one row (formulas: include/ep_hip.h, ep_distill_topk).
//
// Plain form: one workgroup per row, three passes over it (maximum; sums of exponentials at both temperatures; gradient).  The
// classes that the teacher lists are marked in an LDS bit map, so the mass of all others is summed without them and not formed
// as a difference.  The listed classes' gradients are rewritten last, each by its first entry, which also adds up repeated ones
// in entry order: no atomics, one result.
#include "ep_common.h"

namespace ep {

constexpr int DIST_MAX_K = 1024;
constexpr int DIST_MAX_C = 1 << 20;               // bit map of a row: 128 KiB of the 160 KiB LDS

template <int DT> struct DistElem { typedef float T; };
template <> struct DistElem<1> { typedef uint16_t T; };
template <> struct DistElem<2> { typedef _Float16 T; };
template <int DT>
__device__ __forceinline__ float dist_load(const typename DistElem<DT>::T* p) {
  if constexpr (DT == 1) return __uint_as_float((uint32_t)*p << 16);
  else return (float)*p;
}
template <int DT>
__device__ __forceinline__ void dist_store(typename DistElem<DT>::T* p, float v) {
  if constexpr (DT == 1) { const __bf16 h = (__bf16)v; *p = __builtin_bit_cast(uint16_t, h); }
  else *p = (typename DistElem<DT>::T)v;
}

__device__ __forceinline__ float dist_reduce(float v, bool mx, float* lds) {       // over the 4 waves of the workgroup
  v = mx ? wave_max(v) : wave_sum(v);
  __syncthreads();
  if (lane_id() == 0) lds[threadIdx.x >> 6] = v;
  __syncthreads();
  return mx ? fmaxf(fmaxf(lds[0], lds[1]), fmaxf(lds[2], lds[3])) : (lds[0] + lds[1]) + (lds[2] + lds[3]);
}

template <int DT>
__global__ __launch_bounds__(256) void ep_distill_kernel(ep_distill_args a) {
  extern __shared__ char dyn[];
  __shared__ float red[4];
  __shared__ int bad_s;
  typedef typename DistElem<DT>::T T;
  int* idx = reinterpret_cast<int*>(dyn);
  float* pk = reinterpret_cast<float*>(idx + a.K);
  uint32_t* bits = reinterpret_cast<uint32_t*>(pk + a.K);
  const int b = (int)blockIdx.x, tid = (int)threadIdx.x, C = a.C, K = a.K;
  const float nan = __uint_as_float(0x7fc00000u), invT = 1.f / a.temperature;
  const T* z = static_cast<const T*>(a.logits) + (int64_t)b * a.ldl;
  const int64_t r = a.teacher_rows ? (int64_t)a.teacher_rows[b] : (int64_t)b;
  const bool row_ok = r >= 0 && r < a.R;
  const bool label = a.targets && a.alpha != 1.f;
  const int64_t tg64 = label ? a.targets[b] : -1;
  const bool tg_bad = tg64 >= C;
  const int tg = tg64 < 0 || tg_bad ? -1 : (int)tg64;
  if (tid == 0) bad_s = 0;
  if (a.teacher_tail)
    for (int i = tid; i < (C + 31) / 32; i += 256) bits[i] = 0u;
  __syncthreads();
  // teacher
  float tm = -INFINITY;
  for (int k = tid; k < K; k += 256) {
    int i = row_ok ? a.teacher_index[r * a.ldi + k] : -1;
    float t = row_ok ? a.teacher_values[r * a.ldv + k] * invT : 0.f;
    if (i >= C) { bad_s = 1; i = -1; }
    if (i < 0) t = -INFINITY;
    idx[k] = i; pk[k] = t;
    if (t != t) tm = t;
    tm = fmaxf(tm, t);
    if (i >= 0 && a.teacher_tail) atomicOr(&bits[i >> 5], 1u << (i & 31));
  }
  const float tail = a.teacher_tail && row_ok ? a.teacher_tail[r] : -INFINITY;
  tm = fmaxf(dist_reduce(tm, true, red), tail);
  const bool bad = bad_s || !row_ok || tg_bad;
  const bool soft = tm > -INFINITY || tail != tail;
  float ts = 0.f;
  for (int k = tid; k < K; k += 256) ts += soft && idx[k] >= 0 ? expf(pk[k] - tm) : 0.f;
  ts = dist_reduce(ts, false, red) + (soft ? expf(tail - tm) : 0.f);
  const float tl = tm + logf(ts);
  // student
  float m = -INFINITY;
  for (int i = tid; i < C; i += 256) m = fmaxf(m, dist_load<DT>(z + i));
  m = dist_reduce(m, true, red);
  float sall = 0.f, sout = 0.f, s1 = 0.f;
  for (int i = tid; i < C; i += 256) {
    const float v = dist_load<DT>(z + i) - m;
    const float e = expf(v * invT);
    sall += e;
    if (a.teacher_tail && !(bits[i >> 5] >> (i & 31) & 1u)) sout += e;
    if (label) s1 += expf(v);
  }
  sall = dist_reduce(sall, false, red);
  if (a.teacher_tail) sout = dist_reduce(sout, false, red);
  if (label) s1 = dist_reduce(s1, false, red);
  const float lsall = logf(sall);
  // loss
  float kl = 0.f;
  for (int k = tid; k < K; k += 256) {
    const int i = idx[k];
    if (!soft || i < 0) { pk[k] = 0.f; continue; }
    const float lp = pk[k] - tl, p = expf(lp);
    pk[k] = p;
    if (p > 0.f || p != p) kl += p * (lp - ((dist_load<DT>(z + i) - m) * invT - lsall));
  }
  kl = dist_reduce(kl, false, red);
  const float ptail = soft && a.teacher_tail ? expf(tail - tl) : 0.f;
  if (ptail > 0.f || ptail != ptail) kl += ptail * ((tail - tl) - (logf(sout) - lsall));
  if (tid == 0) {
    float loss = soft ? a.alpha * a.temperature * a.temperature * kl : 0.f;
    if (tg >= 0) loss += (1.f - a.alpha) * (logf(s1) - (dist_load<DT>(z + tg) - m));
    a.loss_rows[b] = bad ? nan : loss;
  }
  if (!a.dlogits) return;
  // gradient
  T* dz = static_cast<T*>(a.dlogits) + (int64_t)b * a.ldd;
  const float g = a.grad_scale * (a.grad_scale_dev ? *a.grad_scale_dev : 1.f) / (float)a.B;
  const float cs = soft ? a.alpha * a.temperature * g : 0.f, ch = tg >= 0 ? (1.f - a.alpha) * g : 0.f;
  const float is = 1.f / sall, ih = label ? 1.f / s1 : 0.f, io = ptail > 0.f ? ptail / sout : 0.f;
  auto grad = [&](int i, float zi, bool listed, float psum) {
    const float v = zi - m;
    const float e = expf(v * invT);
    float d = cs * (e * is - (listed ? 0.f : e * io) - psum);
    if (tg >= 0) d += ch * (expf(v) * ih - (i == tg ? 1.f : 0.f));
    return bad ? nan : d;
  };
  for (int i = tid; i < C; i += 256)
    dist_store<DT>(dz + i, grad(i, dist_load<DT>(z + i), a.teacher_tail && (bits[i >> 5] >> (i & 31) & 1u), 0.f));
  __syncthreads();
  for (int k = tid; k < K; k += 256) {
    const int i = idx[k];
    if (i < 0) continue;
    float ps = 0.f;
    bool first = true;
    for (int j = 0; j < K; ++j)
      if (idx[j] == i) { ps += pk[j]; first = first && j >= k; }
    if (first) dist_store<DT>(dz + i, grad(i, dist_load<DT>(z + i), a.teacher_tail != nullptr, ps));
  }
}

}  // namespace ep

using namespace ep;

extern "C" {

size_t ep_distill_workspace_bytes(int B, int C, int K) { return B > 0 && C > 0 && K > 0 ? 256 : 0; }

int ep_distill_topk(const ep_distill_args* a, void* workspace, size_t workspace_bytes, ep_stream_t stream) {
  EP_REQUIRE(a && a->logits && a->teacher_values && a->teacher_index && a->loss_rows && workspace, EP_E_ARG, "ep_distill_topk: null pointer");
  EP_REQUIRE(a->B > 0 && a->C > 0 && a->K > 0 && a->R > 0, EP_E_ARG, "ep_distill_topk: B %d, C %d, K %d, R %lld must be positive", a->B, a->C, a->K,
             (long long)a->R);
  EP_REQUIRE(a->C <= DIST_MAX_C && a->K <= DIST_MAX_K, EP_E_SHAPE, "ep_distill_topk: C %d (at most %d), K %d (at most %d)", a->C, DIST_MAX_C, a->K, DIST_MAX_K);
  EP_REQUIRE(a->dtype >= EP_DTYPE_F32 && a->dtype <= EP_DTYPE_F16, EP_E_UNSUPPORTED, "ep_distill_topk: dtype %d", a->dtype);
  EP_REQUIRE(a->teacher_rows || a->R >= a->B, EP_E_ARG, "ep_distill_topk: %lld teacher rows for a batch of %d need teacher_rows", (long long)a->R, a->B);
  EP_REQUIRE((a->B == 1 || (a->ldl >= a->C && (!a->dlogits || a->ldd >= a->C))) && (a->R == 1 || (a->ldv >= a->K && a->ldi >= a->K)), EP_E_SHAPE,
             "ep_distill_topk: a row stride is below its row");
  EP_REQUIRE(a->temperature > 0.f && a->temperature <= 3.0e38f && a->alpha >= 0.f && a->alpha <= 1.f, EP_E_ARG,
             "ep_distill_topk: temperature %g must be positive and alpha %g within [0, 1]", (double)a->temperature, (double)a->alpha);
  EP_REQUIRE(a->targets || a->alpha == 1.f, EP_E_ARG, "ep_distill_topk: alpha < 1 needs targets");
  EP_REQUIRE(workspace_bytes >= ep_distill_workspace_bytes(a->B, a->C, a->K), EP_E_WORKSPACE, "ep_distill_topk: workspace %zu < %zu", workspace_bytes,
             ep_distill_workspace_bytes(a->B, a->C, a->K));
  const size_t lds = (size_t)a->K * 8 + (a->teacher_tail ? ((size_t)a->C + 31) / 32 * 4 : 0);
  hipStream_t st = (hipStream_t)stream;
#define EP_DIST(DT)                                                                                                                       \
  do {                                                                                                                                    \
    if (lds > 48 * 1024) EP_HIP(hipFuncSetAttribute((const void*)ep_distill_kernel<DT>, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds)); \
    hipLaunchKernelGGL(ep_distill_kernel<DT>, dim3(a->B), dim3(256), lds, st, *a);                                                          \
  } while (0)
  if (a->dtype == EP_DTYPE_F32) EP_DIST(0);
  else if (a->dtype == EP_DTYPE_BF16) EP_DIST(1);
  else EP_DIST(2);
#undef EP_DIST
  EP_LAUNCH_CHECK("ep_distill_kernel");
  return 0;
}

}  // extern "C"
