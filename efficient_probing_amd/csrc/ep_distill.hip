// Distillation from a teacher's top logits: loss and logit gradient of one row (formulas: include/ep_hip.h, ep_distill_topk).
//
// Bound: the logits' bytes, read once and written once (gradient).  Rows of up to 32768 classes stay in the registers of one workgroup
// (a wave for up to 1024 classes, four rows a workgroup; 4 or 8 waves above): one read, then maximum, sums of exponentials, gradient.
// Longer rows are cut into pieces of 4096 over many workgroups in two launches: partial maxima and sums, then each piece's gradient.
// Measured with 64 listed classes and a tail (bytes read and written per second; a copy of the same size reaches 4.7 TB/s):
// 2048 x 32768 bf16 61 us (4.4 TB/s), 2048 x 21841 bf16 48 us (3.7), 4096 x 10000 fp32 68 us (4.8), 16384 x 1000 fp32 36 us (3.6);
// in pieces 512 x 100000 fp32 129 us (3.2: the second launch reads the logits again), 6 x 131071 fp32 14 us (one workgroup a row:
// 310 us).  bf16 rows are also near the vector unit's rate: about 16 instructions a class, two of them exponentials.
//
// The classes that the teacher lists are marked in an LDS bit map, so that the mass of all others is summed without them and not formed
// as a difference.  The gradient is written for every class as if none were listed; then the listed ones and the label are written
// again.  Where a class is listed more than once, each of its entries adds up all of them in entry order and writes the same value: no
// atomics on values, one result.
#include "ep_common.h"

namespace ep {

constexpr int DIST_MAX_K = 1024;
constexpr int DIST_MAX_C = 1 << 20;               // (256 pieces, one for each thread that joins them)
constexpr float DIST_MIN_T = 1e-15f, DIST_MAX_T = 1e15f;      // T^2, and a logit over T, stay within fp32
constexpr int DIST_PIECE = 4096;                  // classes of a workgroup where a row is cut
constexpr int DIST_SLICE = 1 << 22;               // workgroups of a launch (HIP takes less than 2^32 threads)
// A sum of exponentials below this is taken again relative to its own maximum: an exponential below 2^-126 is zero, which a sum of 1e-30
// would still feel (classes 20 below it, with shares of 1e-8 of the tail, took no gradient); of 1e-16 it loses shares below 1e-22.
constexpr float DIST_LOW = 1e-16f;
constexpr float DIST_LOG2E = 1.4426950408889634f;

template <int DT> struct DistElem { typedef float T; static constexpr int VEC = 4; };
template <> struct DistElem<1> { typedef uint16_t T; static constexpr int VEC = 8; };
template <> struct DistElem<2> { typedef _Float16 T; static constexpr int VEC = 8; };
template <int DT>
__device__ __forceinline__ float dist_load(const typename DistElem<DT>::T* p) {
  if constexpr (DT == 1) return __uint_as_float((uint32_t)*p << 16);
  else return (float)*p;
}
template <int DT>
__device__ __forceinline__ uint32_t dist_pair(float x, float y) {                     // two 16-bit values, rounded to nearest even
  if constexpr (DT == 1) {
    typedef __bf16 b2 __attribute__((ext_vector_type(2)));
    const b2 h = {(__bf16)x, (__bf16)y};
    return __builtin_bit_cast(uint32_t, h);
  } else {
    typedef _Float16 h2 __attribute__((ext_vector_type(2)));
    const h2 h = {(_Float16)x, (_Float16)y};
    return __builtin_bit_cast(uint32_t, h);
  }
}
template <int DT>
__device__ __forceinline__ void dist_store(typename DistElem<DT>::T* p, float v) {
  if constexpr (DT == 1) { const __bf16 h = (__bf16)v; *p = __builtin_bit_cast(uint16_t, h); }
  else *p = (typename DistElem<DT>::T)v;
}
typedef uint32_t dist_u4 __attribute__((ext_vector_type(4)));
template <int DT>
__device__ __forceinline__ void dist_unpack(const dist_u4& r, float (&v)[DistElem<DT>::VEC]) {
  const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (DT == 0) v[i] = __uint_as_float(w[i]);
    else { const f4 f = h16x4_to_f4(uint2{w[i], 0u}, DT == 2); v[2 * i] = f.x; v[2 * i + 1] = f.y; }
  }
}

// threads of one row work together: a whole workgroup, or one wave of it
template <int TH>
__device__ __forceinline__ void dist_sync() {
  if constexpr (TH == 64) {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "workgroup");
    __builtin_amdgcn_wave_barrier();
  } else {
    __syncthreads();
  }
}
template <int TH>
__device__ __forceinline__ float dist_max(float v, float* lds) {
  v = wave_max(v);
  if constexpr (TH > 64) {
    __syncthreads();
    if (lane_id() == 0) lds[threadIdx.x >> 6] = v;
    __syncthreads();
    v = wave_max(lds[lane_id() & (TH / 64 - 1)]);
  }
  return v;
}
template <int TH, int N>
__device__ __forceinline__ void dist_sums(float (&v)[N], float* lds) {
#pragma unroll
  for (int j = 0; j < N; ++j) v[j] = wave_sum(v[j]);
  if constexpr (TH > 64) {
    __syncthreads();
    if (lane_id() == 0)
#pragma unroll
      for (int j = 0; j < N; ++j) lds[(threadIdx.x >> 6) * N + j] = v[j];
    __syncthreads();
#pragma unroll
    for (int j = 0; j < N; ++j) v[j] = wave_sum(lane_id() < TH / 64 ? lds[lane_id() * N + j] : 0.f);
  }
}

// ---- one row's teacher, label and what follows from them ------------------------------------------------------------------
struct DistEntries {            // in LDS, K entries and the label, padded to whole quads
  int* idx;                     // class, -1 none (also the label's place and the padding)
  float* pk;                    // teacher's value / T, then its probability
  float* zk;                    // the logit, then the gradient
};
struct DistRow {
  int64_t r;                    // row of the teacher's tables
  int tg;                       // label, or -1
  bool bad, soft;               // something out of range; there is a distillation term
  float tail, tl, ptail;        // log mass behind the list; logsumexp over list and tail; the tail's probability
  float ml, ms;                 // student's statistics: maximum of the logits; log of the sum of exp((z - ml) / T)
  float mo;                     // what the sum over the classes behind the list is relative to
};

__host__ __device__ __forceinline__ int dist_quads(int K) { return (K + 4) / 4; }
__device__ __forceinline__ DistEntries dist_entries(int* p, int K) {
  const int n = 4 * dist_quads(K);
  return DistEntries{p, reinterpret_cast<float*>(p + n), reinterpret_cast<float*>(p + 2 * n)};
}
// entries to LDS, marks of the listed classes to `bits`
template <int DT, int TH>
__device__ __forceinline__ void dist_teacher(const ep_distill_args& a, int b, int tid, const typename DistElem<DT>::T* z, const DistEntries& e, uint32_t* bits,
                                             int* flag, float* red, DistRow& d) {
  const float invT = 1.f / a.temperature;
  d.r = a.teacher_rows ? (int64_t)a.teacher_rows[b] : (int64_t)b;
  const bool row_ok = d.r >= 0 && d.r < a.R;
  const int64_t tg64 = a.targets && a.alpha != 1.f ? a.targets[b] : -1;
  const bool tg_bad = tg64 >= a.C;
  d.tg = tg64 < 0 || tg_bad ? -1 : (int)tg64;
  if (tid == 0) *flag = 0;
  if (bits)
    for (int i = tid; i < (a.C + 31) / 32; i += TH) bits[i] = 0u;
  dist_sync<TH>();
  float tm = -INFINITY;
  bool nan = false;
  _Pragma("unroll 1") for (int k = tid; k < 4 * dist_quads(a.K); k += TH) {
    if (k >= a.K) {
      e.idx[k] = -1; e.pk[k] = 0.f;
      if (k == a.K) e.zk[k] = d.tg >= 0 ? dist_load<DT>(z + d.tg) : 0.f;
      continue;
    }
    int i = row_ok ? a.teacher_index[d.r * a.ldi + k] : -1;
    float t = row_ok ? a.teacher_values[d.r * a.ldv + k] * invT : 0.f;
    if (i >= a.C) { atomicOr(flag, 1); i = -1; }
    if (i < 0) t = -INFINITY;
    e.idx[k] = i; e.pk[k] = t; e.zk[k] = i >= 0 ? dist_load<DT>(z + i) : 0.f;
    nan |= t != t;
    tm = fmaxf(tm, t);
    if (bits && i >= 0) atomicOr(&bits[i >> 5], 1u << (i & 31));
  }
  d.tail = a.teacher_tail && row_ok ? a.teacher_tail[d.r] : -INFINITY;
  if (nan) atomicOr(flag, 2);
  tm = fmaxf(dist_max<TH>(tm, red), d.tail);
  dist_sync<TH>();
  const int f = *flag;
  d.bad = (f & 1) || !row_ok || tg_bad;
  d.soft = a.alpha > 0.f && (tm > -INFINITY || (f & 2) || d.tail != d.tail);   // (no 0 times infinity)
  float ts[1] = {0.f};
  _Pragma("unroll 1") for (int k = tid; k < a.K; k += TH) ts[0] += d.soft && e.idx[k] >= 0 ? __builtin_amdgcn_exp2f((e.pk[k] - tm) * DIST_LOG2E) : 0.f;
  dist_sums<TH, 1>(ts, red);
  ts[0] += d.soft ? __builtin_amdgcn_exp2f((d.tail - tm) * DIST_LOG2E) : 0.f;
  d.tl = tm + logf(ts[0]);
  d.ptail = d.soft && a.teacher_tail ? expf(d.tail - d.tl) : 0.f;
}

// loss of the row; turns pk into probabilities.  s[0..2]: sums of exp over all classes at T, over those not listed (relative to mo), over all at 1
template <int TH>
__device__ __forceinline__ void dist_loss(const ep_distill_args& a, int b, int tid, const DistEntries& e, const DistRow& d, const float (&s)[3], float* red,
                                          bool write) {
  const float invT = 1.f / a.temperature;
  float kl[1] = {0.f};
  _Pragma("unroll 1") for (int k = tid; k < a.K; k += TH) {
    if (!d.soft || e.idx[k] < 0) { e.pk[k] = 0.f; continue; }
    const float lp = e.pk[k] - d.tl, p = expf(lp);
    e.pk[k] = p;
    if (write && (p > 0.f || p != p)) kl[0] += p * (lp - ((e.zk[k] - d.ml) * invT - d.ms));
  }
  if (!write) return;
  dist_sums<TH, 1>(kl, red);
  if (d.ptail > 0.f || d.ptail != d.ptail) kl[0] += d.ptail * ((d.tail - d.tl) - ((d.mo - d.ml) * invT + (logf(s[1]) - d.ms)));
  if (tid == 0) {
    float loss = d.soft ? a.alpha * a.temperature * a.temperature * kl[0] : 0.f;
    if (d.tg >= 0) loss += (1.f - a.alpha) * (logf(s[2]) - (e.zk[a.K] - d.ml));
    a.loss_rows[b] = d.bad ? __uint_as_float(0x7fc00000u) : loss;
  }
}

struct DistGrad {               // d(class) = soft (e / s0 - [not listed] e io - sum of p) + hard (e1 / s2 - [label])
  float m, mo, kT, soft, hard, is, ih;
  float plain, label;           // factors of e and e1 for a class that is neither listed nor the label
};
__device__ __forceinline__ DistGrad dist_coeffs(const ep_distill_args& a, const DistRow& d, const float (&s)[3]) {
  DistGrad g;
  const float gs = a.grad_scale * (a.grad_scale_dev ? *a.grad_scale_dev : 1.f) / (float)a.B + (d.bad ? __uint_as_float(0x7fc00000u) : 0.f);
  g.m = d.ml; g.mo = d.mo; g.kT = DIST_LOG2E / a.temperature;
  g.soft = d.soft || d.bad ? a.alpha * a.temperature * gs : 0.f;
  g.hard = d.tg >= 0 ? (1.f - a.alpha) * gs : 0.f;
  g.is = 1.f / s[0]; g.ih = d.tg >= 0 ? 1.f / s[2] : 0.f;
  g.plain = g.soft * (g.is * __builtin_amdgcn_exp2f((d.mo - d.ml) * g.kT) - (d.ptail > 0.f || d.ptail != d.ptail ? d.ptail / s[1] : 0.f));
  g.label = g.hard * g.ih;
  return g;
}
__device__ __forceinline__ float dist_grad(const DistGrad& g, float z, bool listed, float psum, bool label) {
  const float v = z - g.m;
  float d = listed ? g.soft * (g.is * __builtin_amdgcn_exp2f(v * g.kT) - psum) : g.plain * __builtin_amdgcn_exp2f((z - g.mo) * g.kT);
  if (g.hard != 0.f) d += g.hard * (__builtin_amdgcn_exp2f(v * DIST_LOG2E) * g.ih - (label ? 1.f : 0.f));
  return d;
}
template <bool LABEL>
__device__ __forceinline__ float dist_grad_plain(const DistGrad& g, float z) {
  float d = g.plain * __builtin_amdgcn_exp2f((z - g.mo) * g.kT);
  if (LABEL) d += g.label * __builtin_amdgcn_exp2f((z - g.m) * DIST_LOG2E);
  return d;
}
// gradients of the listed classes in [lo, lo + n) and of the label, in place of their logits (every thread's probabilities must be there)
template <int TH>
__device__ __forceinline__ void dist_listed(const ep_distill_args& a, int tid, const DistEntries& e, const DistRow& d, const DistGrad& g, int lo, int n) {
  const int4* id4 = reinterpret_cast<const int4*>(e.idx);
  const f4* pk4 = reinterpret_cast<const f4*>(e.pk);
  _Pragma("unroll 1") for (int k = tid; k <= a.K; k += TH) {
    const int i = k < a.K ? e.idx[k] : d.tg;
    if (i < lo || i >= lo + n) continue;
    float ps = 0.f;
    bool listed = false;
#pragma unroll 2
    for (int j = 0; j < dist_quads(a.K); ++j) {
      const int4 v = id4[j];
      const f4 p = pk4[j];
      ps += v.x == i ? p.x : 0.f; ps += v.y == i ? p.y : 0.f; ps += v.z == i ? p.z : 0.f; ps += v.w == i ? p.w : 0.f;
      listed |= v.x == i || v.y == i || v.z == i || v.w == i;
    }
    e.zk[k] = dist_grad(g, e.zk[k], listed, ps, i == d.tg);
  }
}
template <int DT, int TH>
__device__ __forceinline__ void dist_store_listed(const ep_distill_args& a, int tid, const DistEntries& e, const DistRow& d, typename DistElem<DT>::T* dz, int lo, int n) {
  _Pragma("unroll 1") for (int k = tid; k <= a.K; k += TH) {
    const int i = k < a.K ? e.idx[k] : d.tg;
    if (i >= lo && i < lo + n) dist_store<DT>(dz + i, e.zk[k]);
  }
}

// A run of n classes in registers, in 16-byte pieces from its first class on and up to VEC - 1 single ones behind.  Rows of odd length start
// at any element: the pieces' loads and stores are of element alignment, which costs less than moving the pieces to the 16-byte grid
// would in code, and a class's place in the sums does not depend on the tensor's address.
template <int DT, int TH, int NV>
struct DistRun {
  typedef typename DistElem<DT>::T T;
  static constexpr int VEC = DistElem<DT>::VEC;
  struct __attribute__((packed, aligned(sizeof(T)))) Piece { dist_u4 v; };
  static_assert(alignof(Piece) == sizeof(T), "(a class type such as uint4 would not be packed, and 16 bytes promised to the compiler)");
  int nv, edge;                 // pieces, single classes
  dist_u4 raw[NV];
  float one;                    // the thread's single class (thread < edge)
  __device__ __forceinline__ int edge_class(int t) const { return nv * VEC + t; }
  __device__ __forceinline__ void load(const T* z, int n, int tid) {
    nv = n / VEC;
    edge = n - nv * VEC;
    const Piece* p = reinterpret_cast<const Piece*>(z);
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      const int i = tid + v * TH;
      raw[v] = i < nv ? p[i].v : dist_u4{0u, 0u, 0u, 0u};
    }
    one = tid < edge ? dist_load<DT>(z + edge_class(tid)) : 0.f;
  }
};

template <int DT, int TH, int NV>
__device__ __forceinline__ float dist_run_max(const DistRun<DT, TH, NV>& r, int tid, float* red) {
  float m = -INFINITY;
#pragma unroll
  for (int v = 0; v < NV; ++v) {
    float f[DistElem<DT>::VEC];
    dist_unpack<DT>(r.raw[v], f);
    if (tid + v * TH < r.nv) {
#pragma unroll
      for (int i = 0; i < DistElem<DT>::VEC; ++i) m = fmaxf(m, f[i]);
    }
  }
  if (tid < r.edge) m = fmaxf(m, r.one);
  return dist_max<TH>(m, red);
}
// v where bit i of `other` is set, else 0 (as a comparison and a selection it would be two instructions, one of them scalar)
__device__ __forceinline__ float dist_keep(float v, uint32_t other, int i) {
  int mask;
  asm("v_bfe_i32 %0, %1, %2, 1" : "=v"(mask) : "v"(other), "i"(i));
  return __int_as_float(__float_as_int(v) & mask);
}
template <int DT, int TH, int NV, bool LABEL>
__device__ __forceinline__ void dist_run_sums(const DistRun<DT, TH, NV>& r, int tid, float m, float kT, const uint32_t* bits, float (&s)[3]) {
  s[0] = s[1] = s[2] = 0.f;
  constexpr int VEC = DistElem<DT>::VEC;
#pragma unroll
  for (int v = 0; v < NV; ++v) {
    const int p = tid + v * TH;
    if (p >= r.nv) continue;
    float f[VEC];
    dist_unpack<DT>(r.raw[v], f);
    uint32_t other = 0;
    if (bits) other = ~(bits[p * VEC / 32] >> (p * VEC % 32));
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      const float e = __builtin_amdgcn_exp2f((f[i] - m) * kT);
      s[0] += e;
      if (bits) s[1] += dist_keep(e, other, i);
      if (LABEL) s[2] += __builtin_amdgcn_exp2f((f[i] - m) * DIST_LOG2E);
    }
  }
  if (tid < r.edge) {
    const int bit = r.edge_class(tid);
    const float e = __builtin_amdgcn_exp2f((r.one - m) * kT);
    s[0] += e;
    if (bits) s[1] += bits[bit >> 5] >> (bit & 31) & 1u ? 0.f : e;
    if (LABEL) s[2] += __builtin_amdgcn_exp2f((r.one - m) * DIST_LOG2E);
  }
}
// Where the classes behind the list lie so far below the listed ones that their sum has left fp32's normal range, it is taken again
// relative to their own maximum, so that their share keeps its logarithm and its gradient.
template <int DT, int TH, int NV>
__device__ __forceinline__ void dist_run_others(const DistRun<DT, TH, NV>& r, int tid, float kT, const uint32_t* bits, float* red, float& mo, float& s1) {
  constexpr int VEC = DistElem<DT>::VEC;
  float m = -INFINITY, s[1] = {0.f};
  _Pragma("unroll 1") for (int pass = 0; pass < 2; ++pass) {
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      const int p = tid + v * TH;
      if (p >= r.nv) continue;
      float f[VEC];
      dist_unpack<DT>(r.raw[v], f);
      const uint32_t listed = bits[p * VEC / 32] >> (p * VEC % 32);
#pragma unroll
      for (int i = 0; i < VEC; ++i)
        if (!(listed >> i & 1u)) { if (pass) s[0] += __builtin_amdgcn_exp2f((f[i] - mo) * kT); else m = fmaxf(m, f[i]); }
    }
    const int bit = r.edge_class(tid);
    if (tid < r.edge && !(bits[bit >> 5] >> (bit & 31) & 1u)) { if (pass) s[0] += __builtin_amdgcn_exp2f((r.one - mo) * kT); else m = fmaxf(m, r.one); }
    if (!pass) { m = dist_max<TH>(m, red); if (m > -INFINITY) mo = m; }
  }
  dist_sums<TH, 1>(s, red);
  s1 = s[0];
}
template <int DT, int TH, int NV, bool LABEL>
__device__ __forceinline__ void dist_run_grad(const DistRun<DT, TH, NV>& r, int tid, const DistGrad& g, typename DistElem<DT>::T* dz) {
  constexpr int VEC = DistElem<DT>::VEC;
#pragma unroll
  for (int v = 0; v < NV; ++v) {
    const int p = tid + v * TH;
    if (p >= r.nv) continue;
    float f[VEC];
    dist_unpack<DT>(r.raw[v], f);
#pragma unroll
    for (int i = 0; i < VEC; ++i) f[i] = dist_grad_plain<LABEL>(g, f[i]);
    dist_u4 w;
    if constexpr (DT == 0) w = dist_u4{__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3])};
    else w = dist_u4{dist_pair<DT>(f[0], f[1]), dist_pair<DT>(f[2], f[3]), dist_pair<DT>(f[4], f[5]), dist_pair<DT>(f[6], f[7])};
    reinterpret_cast<typename DistRun<DT, TH, NV>::Piece*>(dz)[p].v = w;
  }
  if (tid < r.edge) dist_store<DT>(dz + r.edge_class(tid), dist_grad_plain<LABEL>(g, r.one));
}

__device__ __forceinline__ void dist_stores_done() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }

// ---- a row in the registers of TH threads ---------------------------------------------------------------------------------
template <int DT, int TH, int NV, bool LABEL>
__global__ __launch_bounds__(TH < 256 ? 256 : TH, TH == 256 ? 8 : NV * DistElem<DT>::VEC > 32 && DT == 0 ? 4 : 6) void ep_distill_rows_kernel(ep_distill_args a, int row0, int row_lds) {
  extern __shared__ __align__(16) char dyn[];
  typedef typename DistElem<DT>::T T;
  constexpr int RPW = TH < 256 ? 256 / TH : 1;                          // rows of a workgroup
  const int sub = TH < 256 ? (int)threadIdx.x / TH : 0, tid = (int)threadIdx.x - sub * TH;
  const int b = row0 + (int)blockIdx.x * RPW + sub;
  if (b >= a.B) return;                                                 // (a whole wave: nothing below waits for it)
  char* mine = dyn + sub * row_lds;
  float* red = reinterpret_cast<float*>(mine);                          // 48 floats
  int* flag = reinterpret_cast<int*>(red + 48);
  const DistEntries e = dist_entries(flag + 4, a.K);
  uint32_t* bits = a.teacher_tail ? reinterpret_cast<uint32_t*>(e.zk + 4 * dist_quads(a.K)) : nullptr;
  const T* z = static_cast<const T*>(a.logits) + (int64_t)b * a.ldl;
  DistRun<DT, TH, NV> run;
  run.load(z, a.C, tid);
  DistRow d;
  dist_teacher<DT, TH>(a, b, tid, z, e, bits, flag, red, d);
  d.ml = dist_run_max(run, tid, red);
  float s[3];
  dist_run_sums<DT, TH, NV, LABEL>(run, tid, d.ml, DIST_LOG2E / a.temperature, bits, s);
  dist_sums<TH, 3>(s, red);
  d.ms = logf(s[0]); d.mo = d.ml;
  if (bits && s[1] < DIST_LOW) dist_run_others(run, tid, DIST_LOG2E / a.temperature, bits, red, d.mo, s[1]);
  dist_loss<TH>(a, b, tid, e, d, s, red, true);
  if (!a.dlogits) return;
  T* dz = static_cast<T*>(a.dlogits) + (int64_t)b * a.ldd;
  const DistGrad g = dist_coeffs(a, d, s);
  dist_sync<TH>();
  dist_listed<TH>(a, tid, e, d, g, 0, a.C);
  dist_run_grad<DT, TH, NV, LABEL>(run, tid, g, dz);
  dist_stores_done();
  dist_sync<TH>();
  dist_store_listed<DT, TH>(a, tid, e, d, dz, 0, a.C);
}

// ---- rows cut into pieces: partial statistics, then loss and gradient -------------------------------------------------------
struct DistPart { float m, s0, s2, mo, s1; };     // a piece's maximum and sums; the sum over its unlisted classes is relative to mo

template <int DT, bool LABEL>
__global__ __launch_bounds__(256) void ep_distill_part_kernel(ep_distill_args a, int row0, int pieces, DistPart* __restrict__ part) {
  extern __shared__ __align__(16) char dyn[];
  typedef typename DistElem<DT>::T T;
  constexpr int NV = DIST_PIECE / 256 / DistElem<DT>::VEC;
  float* red = reinterpret_cast<float*>(dyn);
  uint32_t* bits = reinterpret_cast<uint32_t*>(dyn + 256);
  const int b = row0 + (int)(blockIdx.x / (unsigned)pieces), pc = (int)(blockIdx.x % (unsigned)pieces), tid = (int)threadIdx.x;
  const int lo = pc * DIST_PIECE, n = a.C - lo < DIST_PIECE ? a.C - lo : DIST_PIECE;
  const T* z = static_cast<const T*>(a.logits) + (int64_t)b * a.ldl + lo;
  DistRun<DT, 256, NV> run;
  run.load(z, n, tid);
  if (a.teacher_tail) {
    const int64_t r = a.teacher_rows ? (int64_t)a.teacher_rows[b] : (int64_t)b;
    for (int i = tid; i < (n + 31) / 32; i += 256) bits[i] = 0u;
    __syncthreads();
    if (r >= 0 && r < a.R)
      for (int k = tid; k < a.K; k += 256) {
        const int i = a.teacher_index[r * a.ldi + k] - lo;
        if (i >= 0 && i < n) atomicOr(&bits[i >> 5], 1u << (i & 31));
      }
    __syncthreads();
  }
  const float m = dist_run_max(run, tid, red);                          // -inf where every class is masked: the sums are zero then
  float s[3];
  dist_run_sums<DT, 256, NV, LABEL>(run, tid, m == -INFINITY ? 0.f : m, DIST_LOG2E / a.temperature, a.teacher_tail ? bits : nullptr, s);
  dist_sums<256, 3>(s, red);
  float mo = m == -INFINITY ? 0.f : m;
  if (a.teacher_tail && s[1] < DIST_LOW) dist_run_others(run, tid, DIST_LOG2E / a.temperature, bits, red, mo, s[1]);
  if (tid == 0) part[(int64_t)b * pieces + pc] = DistPart{m, s[0], s[2], mo, s[1]};
}

template <int DT, bool LABEL>
__global__ __launch_bounds__(256) void ep_distill_join_kernel(ep_distill_args a, int row0, int pieces, const DistPart* __restrict__ part) {
  extern __shared__ __align__(16) char dyn[];
  typedef typename DistElem<DT>::T T;
  constexpr int NV = DIST_PIECE / 256 / DistElem<DT>::VEC;
  float* red = reinterpret_cast<float*>(dyn);
  int* flag = reinterpret_cast<int*>(dyn + 192);
  const DistEntries e = dist_entries(reinterpret_cast<int*>(dyn + 256), a.K);
  const int b = row0 + (int)blockIdx.x, pc = (int)blockIdx.y, tid = (int)threadIdx.x;
  const int lo = pc * DIST_PIECE, n = a.C - lo < DIST_PIECE ? a.C - lo : DIST_PIECE;
  const T* row = static_cast<const T*>(a.logits) + (int64_t)b * a.ldl;
  DistRun<DT, 256, NV> run;
  if (a.dlogits) run.load(row + lo, n, tid);
  DistRow d;
  dist_teacher<DT, 256>(a, b, tid, row, e, nullptr, flag, red, d);
  part += (int64_t)b * pieces;
  const float kT = DIST_LOG2E / a.temperature;
  const DistPart none = {-INFINITY, 0.f, 0.f, -INFINITY, 0.f};
  const DistPart p = tid < pieces ? part[tid] : none;                   // (at most 256 pieces)
  d.ml = dist_max<256>(p.m, red);
  d.mo = dist_max<256>(p.s1 == 0.f ? -INFINITY : p.mo, red);
  if (d.mo == -INFINITY) d.mo = d.ml;
  const float wT = p.m == d.ml ? 1.f : __builtin_amdgcn_exp2f((p.m - d.ml) * kT), w1 = p.m == d.ml ? 1.f : __builtin_amdgcn_exp2f((p.m - d.ml) * DIST_LOG2E);
  float s[3] = {p.s0 * wT, p.s1 == 0.f ? 0.f : p.s1 * __builtin_amdgcn_exp2f((p.mo - d.mo) * kT), p.s2 * w1};
  if (tid >= pieces) s[0] = s[1] = s[2] = 0.f;
  dist_sums<256, 3>(s, red);
  d.ms = logf(s[0]);
  dist_loss<256>(a, b, tid, e, d, s, red, pc == 0);
  if (!a.dlogits) return;
  T* dz = static_cast<T*>(a.dlogits) + (int64_t)b * a.ldd;
  const DistGrad g = dist_coeffs(a, d, s);
  __syncthreads();
  dist_listed<256>(a, tid, e, d, g, lo, n);
  dist_run_grad<DT, 256, NV, LABEL>(run, tid, g, dz + lo);
  dist_stores_done();
  __syncthreads();
  dist_store_listed<DT, 256>(a, tid, e, d, dz, lo, n);
}

static int dist_pieces(int C) { return (C + DIST_PIECE - 1) / DIST_PIECE; }
// threads of a row that stays in registers, 0 where it is cut into pieces
static int dist_row_threads(int C) { return C <= 1024 ? 64 : C <= 4096 ? 256 : C <= 32768 ? 512 : 0; }

template <int DT, bool LABEL>
static int dist_launch(const ep_distill_args& a, void* ws, hipStream_t st) {
  constexpr int VEC = DistElem<DT>::VEC;
  const int th = dist_row_threads(a.C);
  if (th) {
    const size_t lds = round_up(192 + 16 + (size_t)dist_quads(a.K) * 48 + (a.teacher_tail ? ((size_t)a.C + 31) / 32 * 4 : 0), 16);
#define EP_DIST_ROWS(TH, NV)                                                                                              \
  do {                                                                                                                    \
    constexpr int rpw = TH < 256 ? 256 / TH : 1;                                                                          \
    for (int64_t row = 0; row < a.B; row += (int64_t)rpw * DIST_SLICE) {                                                  \
      const int64_t n = a.B - row < (int64_t)rpw * DIST_SLICE ? a.B - row : (int64_t)rpw * DIST_SLICE;                    \
      hipLaunchKernelGGL((ep_distill_rows_kernel<DT, TH, NV, LABEL>), dim3((unsigned)((n + rpw - 1) / rpw)), dim3(TH < 256 ? 256 : TH), rpw * lds, st, a, \
                         (int)row, (int)lds);                                                                             \
    }                                                                                                                     \
  } while (0)
    if (th == 64) EP_DIST_ROWS(64, 16 / VEC);
    else if (th == 256) EP_DIST_ROWS(256, 16 / VEC);
    else if (a.C <= 16384) EP_DIST_ROWS(512, 32 / VEC);
    else EP_DIST_ROWS(512, 64 / VEC);
#undef EP_DIST_ROWS
    EP_LAUNCH_CHECK("ep_distill_rows_kernel");
    return 0;
  }
  const int pieces = dist_pieces(a.C), most = DIST_SLICE / pieces;
  for (int64_t row = 0; row < a.B; row += most) {
    const int n = a.B - row < most ? (int)(a.B - row) : most;
    hipLaunchKernelGGL((ep_distill_part_kernel<DT, LABEL>), dim3((unsigned)(n * pieces)), dim3(256), 256 + DIST_PIECE / 8, st, a, (int)row, pieces,
                       static_cast<DistPart*>(ws));
    EP_LAUNCH_CHECK("ep_distill_part_kernel");
    hipLaunchKernelGGL((ep_distill_join_kernel<DT, LABEL>), dim3((unsigned)n, a.dlogits ? pieces : 1), dim3(256), 256 + (size_t)dist_quads(a.K) * 48, st, a, (int)row,
                       pieces, static_cast<const DistPart*>(ws));
    EP_LAUNCH_CHECK("ep_distill_join_kernel");
  }
  return 0;
}

}  // namespace ep

using namespace ep;

extern "C" {

size_t ep_distill_workspace_bytes(int B, int C, int K) {
  if (B <= 0 || C <= 0 || K <= 0 || dist_row_threads(C)) return 0;
  return (size_t)B * dist_pieces(C) * sizeof(DistPart);
}

int ep_distill_topk(const ep_distill_args* a, void* workspace, size_t workspace_bytes, ep_stream_t stream) {
  EP_REQUIRE(a && a->logits && a->teacher_values && a->teacher_index && a->loss_rows, EP_E_ARG, "ep_distill_topk: null pointer");
  EP_REQUIRE(a->B > 0 && a->C > 0 && a->K > 0 && a->R > 0, EP_E_ARG, "ep_distill_topk: B %d, C %d, K %d, R %lld must be positive", a->B, a->C, a->K,
             (long long)a->R);
  EP_REQUIRE(a->C <= DIST_MAX_C && a->K <= DIST_MAX_K, EP_E_SHAPE, "ep_distill_topk: C %d (at most %d), K %d (at most %d)", a->C, DIST_MAX_C, a->K, DIST_MAX_K);
  EP_REQUIRE(a->dtype >= EP_DTYPE_F32 && a->dtype <= EP_DTYPE_F16, EP_E_UNSUPPORTED, "ep_distill_topk: dtype %d", a->dtype);
  EP_REQUIRE(a->teacher_rows || a->R >= a->B, EP_E_ARG, "ep_distill_topk: %lld teacher rows for a batch of %d need teacher_rows", (long long)a->R, a->B);
  EP_REQUIRE((a->B == 1 || (a->ldl >= a->C && (!a->dlogits || a->ldd >= a->C))) && (a->R == 1 || (a->ldv >= a->K && a->ldi >= a->K)), EP_E_SHAPE,
             "ep_distill_topk: a row stride is below its row");
  EP_REQUIRE(a->temperature >= DIST_MIN_T && a->temperature <= DIST_MAX_T && a->alpha >= 0.f && a->alpha <= 1.f, EP_E_ARG,
             "ep_distill_topk: temperature %g must lie within [1e-15, 1e15] and alpha %g within [0, 1]", (double)a->temperature, (double)a->alpha);
  EP_REQUIRE(a->targets || a->alpha == 1.f, EP_E_ARG, "ep_distill_topk: alpha < 1 needs targets");
  const size_t need = ep_distill_workspace_bytes(a->B, a->C, a->K);
  EP_REQUIRE(workspace_bytes >= need, EP_E_WORKSPACE, "ep_distill_topk: workspace %zu < %zu", workspace_bytes, need);
  EP_REQUIRE(!need || (workspace && aligned16(workspace)), EP_E_ARG, "ep_distill_topk: the workspace must be given and 16-byte aligned");
  hipStream_t st = (hipStream_t)stream;
  const bool label = a->alpha != 1.f;
#define EP_DIST(DT) (label ? dist_launch<DT, true>(*a, workspace, st) : dist_launch<DT, false>(*a, workspace, st))
  return a->dtype == EP_DTYPE_F32 ? EP_DIST(0) : a->dtype == EP_DTYPE_BF16 ? EP_DIST(1) : EP_DIST(2);
#undef EP_DIST
}

}  // extern "C"
