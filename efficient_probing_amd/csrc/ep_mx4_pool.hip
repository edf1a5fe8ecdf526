// Attention pooling over the MX4 token cache, forward and backward (x: the decoded tokens):
//     S = scale q.x     A = softmax over the image's tokens     P = A x
//     dA = dP.x         dS = A (dA - dP.P)                       dq = scale sum dS x
//
// Both passes are the same two contractions with a per-token weight between them, and every byte of the cache is read once in each.  A
// wave owns one 128-channel block of the rows (pipelined form, up to 14 blocks) or four (wide-row form) for all tokens of a tile of 32.
//
//   * Tiles come HBM -> LDS by LDS-DMA into a ring of stages that the wave keeps to itself (no barrier on the data path).
//   * First contraction (scores / dA), on the matrix cores in the cache's own format: v_mfma_scale_f32_16x16x128_f8f6f4 takes the
//     E2M1 codes and their E8M0 scale bytes as they lie in LDS, no decoding.  The fp32 operand (queries, dP) becomes seven (wide
//     rows: six) E2M3 terms with a scale per 32 channels, 2^-5 apart.  The grid of a term is 1/8 below 2 and 1/4 up to 4, so every term
//     takes five more bits: values down to 2^-11 (2^-6) of the largest of their 32 channels are exact, of smaller ones at most 2^-35
//     (2^-30) of that largest is left over.  (Five terms would leave 2^-25: rows whose channels differ by 100 to 10000, which meet
//     tokens sized inversely, then give scores up to 4e-4 off.)  All products of codes and terms are exact, the sums fp32.
//   * The blocks' parts of a score are added through LDS in block order.
//   * Weights (exp(S - max), or dS) are split into three bf16 terms, exactly.
//   * Second contraction: codes are decoded to bf16 (exact; v_cvt_scalef32_pk_bf16_fp4 applies the token's own scale, which is why
//     this side cannot stay in 4 bits: the contraction runs over tokens and every token has its own scale), transposed between
//     token pairs by v_perm, v_mfma_f32_16x16x32_bf16.
//
// QM 8: up to 8 queries, rows of a 16-row matrix instruction = 8 queries x 2 terms.  QM 16: up to 16.  More: blockIdx.y.
//
// Bound: the chain from a tile's arrival to its weights, and the start of a launch, more than any one unit.  1024 x 256 x 768, 8 queries:
// forward 42 us (38 back to back), 142 MB from and to HBM at 3.4 TB/s, matrix units busy 17 % of the time, waves waiting 43 % of their
// cycles (barriers and loads) and stalled at issue 27 %; backward 51 us, 208 MB at 4.1 TB/s, 14 %, 49 % and 25 %.  Twice the images take
// 67 and 99 us back to back: some 10 us a launch lie before the first tile and behind the last.
#include "ep_mx4.h"
#include "ep_mx4_pool.h"

namespace ep {

typedef int mx_i8 __attribute__((ext_vector_type(8)));
typedef uint32_t mx_u6 __attribute__((ext_vector_type(6)));
typedef uint32_t mx_u4 __attribute__((ext_vector_type(4)));
typedef float mx_f16 __attribute__((ext_vector_type(16)));
typedef float mx_f32 __attribute__((ext_vector_type(32)));
typedef __bf16 mx_bf8 __attribute__((ext_vector_type(8)));
typedef __attribute__((address_space(3))) void* mx_lds_t;
typedef const __attribute__((address_space(1))) void* mx_gptr_t;

constexpr float MX_LOG2E = 1.4426950408889634f;
constexpr int MX_NT = 2;                         // cache policy of the code loads: streamed once
constexpr float MX_LAZY = 12.0f;                 // the running maximum follows a score only when it lies this far above it

// Terms of an fp32 operand row.  Pipelined form: seven (five cost 2 - 7 % less: 1024 x 256 x 768, 8 queries: 40 us forward and 50 backward
// instead of 42 and 53).  Wide rows: six, what the registers hold (five: 1 % less).
constexpr int MX_TERMS = 7, MX_WIDE_TERMS = 6;

template <int QM> struct MxDims {
  static_assert(MX_TERMS <= 7, "scores() multiplies up to seven operands");
  static constexpr int SETS = QM == 8 ? (MX_TERMS + 1) / 2 : MX_TERMS;       // matrix operands of the fp32 rows: two terms in one at QM 8
  static constexpr int SCB = (SETS + 3) / 4;     // dwords of their scale bytes
  static constexpr int SV = QM == 8 ? 4 : 8;     // scores per lane and tile
  static constexpr int PSETS = QM == 8 ? 2 : 3;  // operands of the weights
};

// the lane number once more, opaque to the compiler: what is derived from it is made where it is used and not kept in registers
// across the tile loop, where they are scarce
__device__ __forceinline__ int mx_fresh(int lane) {
  asm volatile("" : "+v"(lane));
  return lane;
}
template <int N>
__device__ __forceinline__ void mx_wait_vm() {
  static_assert(N >= 0 && N <= 63, "vmcnt");
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}
__device__ __forceinline__ void mx_barrier() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }
__device__ __forceinline__ float mx_ror8(float v) { return dpp_f<0x128>(v); }
__device__ __forceinline__ uint32_t mx_ror8u(uint32_t v) { return __float_as_uint(mx_ror8(__uint_as_float(v))); }
__device__ __forceinline__ float mx_over_groups_max(float v) {       // over the four 16-lane rows
  v = fmaxf(v, __shfl_xor(v, 16, 64));
  return fmaxf(v, __shfl_xor(v, 32, 64));
}
__device__ __forceinline__ float mx_over_groups_sum(float v) {
  v = fold16(v, v);
  return fold32(v, v);
}
__device__ __forceinline__ f4 mx_mfma(mx_u4 a, mx_u4 b, f4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(mx_bf8, a), __builtin_bit_cast(mx_bf8, b), c, 0, 0, 0);
}
template <int BYTE>
__device__ __forceinline__ f4 mx_mfma_codes(const mx_u4& codes, uint32_t scale, const mx_u6& row, uint32_t row_scales, f4 c) {
  const mx_i8 a = {(int)codes[0], (int)codes[1], (int)codes[2], (int)codes[3], 0, 0, 0, 0};
  const mx_i8 b = {(int)row[0], (int)row[1], (int)row[2], (int)row[3], (int)row[4], (int)row[5], 0, 0};
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, c, 4 /* E2M1 */, 2 /* E2M3 */, 0, (int)scale, BYTE, (int)row_scales);
}

// 16 + 16 consecutive fp32 values (the even and the odd channels) -> E2M3 at a scale, and back.  Both instructions write their results
// before they have read all of their sources (the scale among them), which the compiler's own form of them does not say: a result placed
// over a source that dies there makes the low terms differ from run to run.  Hence early-clobber results; and since a matrix instruction
// may read the result of the inline assembly next, its two wait states come along.
__device__ __forceinline__ mx_u6 mx_to_fp6(const mx_f16& even, const mx_f16& odd, float scale) {
  mx_u6 k;
  asm("v_cvt_scalef32_2xpk16_fp6_f32 %0, %1, %2, %3\n\ts_nop 1" : "=&v"(k) : "v"(even), "v"(odd), "v"(scale));
  return k;
}
__device__ __forceinline__ mx_f32 mx_from_fp6(const mx_u6& k, float scale) {
  mx_f32 d;
  asm("v_cvt_scalef32_pk32_f32_fp6 %0, %1, %2\n\ts_nop 1" : "=&v"(d) : "v"(k), "v"(scale));
  return d;
}

// 32 consecutive fp32 values of an operand row -> TERMS E2M3 terms; term t has scale byte s0 - 5 t.  The row's largest value lies in
// [2, 4) times the first scale; what a term leaves is at most 1/8 of its scale (1/16 of values up to 2), which is 4 (2) of the next one's.
template <int QM>
struct MxOperand { mx_u6 b[MxDims<QM>::SETS]; uint32_t sc[MxDims<QM>::SCB]; };

// `take` gets each term with its scale byte (255 where the row holds an infinity or a NaN: its scores become NaN)
template <int TERMS, typename F>
__device__ __forceinline__ void mx_terms(mx_f16 a, mx_f16 b, F&& take) {                     // a, b: the row's even and odd channels
  uint32_t am = 0;
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const uint32_t x = __float_as_uint(a[i]) & 0x7fffffffu, y = __float_as_uint(b[i]) & 0x7fffffffu;
    am = x > am ? x : am;
    am = y > am ? y : am;
  }
  const int ex = (int)(am >> 23);
  const bool bad = ex == 255;
  const int s0 = bad ? 252 : (ex <= 5 * TERMS ? 5 * TERMS : ex - 1);      // (every term has a normal scale: below 2^-91 a row keeps what lies above 2^-126)
#pragma unroll
  for (int t = 0; t < TERMS; ++t) {
    const float sc = __uint_as_float((uint32_t)(s0 - 5 * t) << 23);
    const mx_u6 k = mx_to_fp6(a, b, sc);
    if (t < TERMS - 1) {
      const mx_f32 d = mx_from_fp6(k, sc);
#pragma unroll
      for (int i = 0; i < 16; ++i) { a[i] -= d[2 * i]; b[i] -= d[2 * i + 1]; }
    }
    take(t, k, bad ? 255u : (uint32_t)(s0 - 5 * t));
    __builtin_amdgcn_sched_barrier(0);
  }
}

// the operand of one row block for this lane's column; QM 8: two terms share an operand, columns 8-15 take the odd ones
template <int QM>
__device__ __forceinline__ void mx_operand(const mx_f16& a, const mx_f16& b, int c, MxOperand<QM>& o) {
  const bool odd = QM == 8 && (c & 8) != 0;
  uint32_t bytes[2] = {0, 0};
  mx_terms<MX_TERMS>(a, b, [&](int t, const mx_u6& k, uint32_t byte) {
    if constexpr (QM == 8) {
      if (t % 2 == 0) { o.b[t / 2] = k; bytes[0] |= (odd ? 0u : byte) << (8 * (t / 2)); }
      else {
#pragma unroll
        for (int i = 0; i < 6; ++i) o.b[t / 2][i] = odd ? k[i] : o.b[t / 2][i];
        bytes[0] |= (odd ? byte : 0u) << (8 * (t / 2));
      }
    } else {
      o.b[t] = k;
      bytes[t / 4] |= byte << (8 * (t % 4));
    }
  });
  if constexpr (QM == 8 && MX_TERMS % 2 != 0) {                // the last operand has one term
#pragma unroll
    for (int i = 0; i < 6; ++i) o.b[MX_TERMS / 2][i] = odd ? 0u : o.b[MX_TERMS / 2][i];
  }
  o.sc[0] = bytes[0];
  if constexpr (MxDims<QM>::SCB > 1) o.sc[1] = bytes[1];
}

// 32 values of an operand row from `row` on, times mul; `valid` of them exist, the others are 0.  vec (uniform) says how they lie: 2 rows
// of whole 128-channel blocks, 1 whole 16-byte pieces, 0 anything
__device__ __forceinline__ void mx_load_row(const float* row, int valid, int vec, float mul, mx_f16& a, mx_f16& b) {
  f4 x[8];
  if (vec == 2) {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = reinterpret_cast<const f4*>(row)[i];
  } else if (vec == 1) {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = 4 * i < valid ? reinterpret_cast<const f4*>(row)[i] : f4{0.f, 0.f, 0.f, 0.f};
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) x[i][j] = 4 * i + j < valid ? row[4 * i + j] : 0.f;
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    a[2 * i] = x[i][0] * mul; b[2 * i] = x[i][1] * mul;
    a[2 * i + 1] = x[i][2] * mul; b[2 * i + 1] = x[i][3] * mul;
  }
}

// a wave's sequence of (unit, tile): units u, u + ustep, ..., of each the tiles t_off, t_off + tstep, ...
struct MxCursor {
  int u, ustep, units, tile, hi, len, toff, tstep, tps, splits;
  int b, img;
  __device__ __forceinline__ bool valid() const { return u < units; }
  __device__ __forceinline__ void open(const ep_mx4_tokens& t) {       // first unit from u on that has a tile
    for (; u < units; u += ustep) {
      b = u / splits;
      const int s = u - b * splits;
      img = mx_image_uniform(t, b, len);
      const int n = (len + 31) >> 5;
      hi = (s + 1) * tps < n ? (s + 1) * tps : n;
      tile = s * tps + toff;
      if (tile < hi) return;
    }
    b = img = tile = hi = 0; len = 1;                                   // nothing left: loads go on, from the cache's first row
  }
  __device__ __forceinline__ bool next(const ep_mx4_tokens& t) {       // true: the next tile is another unit's (or there is none)
    tile += tstep;
    if (tile < hi) return false;
    u += ustep;
    open(t);
    return true;
  }
};

// ---- the wide-row form ---------------------------------------------------------------------------------------------------
// Rows of more than 14 blocks.  A wave owns four blocks of the row for all tokens and up to 8 queries; `groups` such sets of waves share
// a workgroup and take turns at the tiles (forward: of one image; backward: a group per image).  Every wave makes the weights itself,
// in the very lanes in which its second contraction wants them.  Accumulators and operand rows of four blocks fill 200 of 256 registers:
// lane constants are made again where they are used and the operands' scale bytes lie in LDS, since a register reloaded from scratch waits
// for the tiles in flight.  Bound:
// matrix and vector units with two waves a SIMD (256 x 784 x 4096, 4 queries: 126 us forward, 3.5 TB/s), and about 20 us for the operand
// rows, the first tile and the way out (128 x 196 x 4096: 36 us and 8 us to join two runs an image).
template <bool BWD, bool OPENS>
__global__ __launch_bounds__(512, 2) void ep_mx4_wide_kernel(MxPool p) {
  constexpr int QM = 8, CPW = 4, NST = MX_STAGES, REC = 1024;          // REC: bytes of an exchange record, the lane's four scores
  constexpr int CODES = 2048 * CPW, STAGE = CODES + 128 * CPW, OPS = 2 * CPW + CPW / 2;
  extern __shared__ __align__(16) char lds[];
  const int lane = lane_id();
  const int wave = wave_id_uniform();
  const int nw = p.nw, groups = p.groups;
  const int grp = wave / nw, dw = wave - grp * nw;
  const ep_mx4_tokens& t = p.t;
  const int nc = p.nc, rowC = nc * 64, rowS = nc * 4;
  const int chunk0 = dw * CPW;
  const int q0 = (int)blockIdx.y * p.qblk, qn = p.Q - q0 < p.qblk ? p.Q - q0 : p.qblk;      // queries of this workgroup
  char* ring = lds + wave * (NST * STAGE);
  char* exch = lds + nw * groups * (NST * STAGE);                      // [2][groups][nw][REC]
  char* opsc = exch + (2 * nw * groups + wave) * REC;                  // the wave's own: scale bytes of its operands, a dword a block

  // LDS row r of a tile holds token 8 (r % 4) + r / 4, its 16-byte pieces XOR-ed with r / 4: both contractions then read all banks
  auto issue = [&](const MxCursor& cu, int slot) {
    char* st = ring + slot * STAGE;
    const int t0 = cu.tile << 5, rows = cu.len - t0;
    const uint8_t* src = t.codes + (int64_t)cu.img * t.codes_bstride + (int64_t)t0 * rowC;
    const uint8_t* scl = t.scales + (int64_t)cu.img * t.scales_bstride + (int64_t)t0 * rowS;
    const int ln = mx_fresh(lane);
    const int tok = 8 * ((ln >> 2) & 3) + (ln >> 4), last = rows - 1;  // rows behind the image's end repeat its last one
    const unsigned seg = (unsigned)(((ln & 3) ^ (ln >> 4)) * 16);
    const unsigned off0 = (unsigned)((tok < last ? tok : last) * rowC) + seg, off1 = (unsigned)((tok + 4 < last ? tok + 4 : last) * rowC) + seg;
    const unsigned offs = (unsigned)(((ln & 31) < last ? (ln & 31) : last) * rowS);
#pragma unroll
    for (int k = 0; k < CPW; ++k) {
      const int ch = chunk0 + k < nc ? chunk0 + k : nc - 1;            // a slice that the row does not fill repeats its last block
      __builtin_amdgcn_global_load_lds((mx_gptr_t)(src + ch * 64 + off0), (mx_lds_t)(st + k * 2048), 16, 0, MX_NT);
      __builtin_amdgcn_global_load_lds((mx_gptr_t)(src + ch * 64 + off1), (mx_lds_t)(st + k * 2048 + 1024), 16, 0, MX_NT);
    }
#pragma unroll
    for (int k = 0; k < CPW; k += 2) {                                 // lanes 32-63: the second block
      const int ch0 = chunk0 + k < nc ? chunk0 + k : nc - 1, ch1 = ch0 + 1 < nc ? ch0 + 1 : ch0;
      __builtin_amdgcn_global_load_lds((mx_gptr_t)(scl + (offs + (unsigned)(ln < 32 ? ch0 : ch1) * 4u)), (mx_lds_t)(st + CODES + k * 128), 4, 0, 0);
    }
  };

  MxCursor cu;                                                          // the tile being worked on
  cu.units = p.units; cu.splits = p.splits; cu.tps = p.tps;
  if constexpr (BWD) { cu.u = (int)blockIdx.x * groups + grp; cu.ustep = (int)gridDim.x * groups; cu.toff = 0; cu.tstep = 1; }
  else { cu.u = (int)blockIdx.x; cu.ustep = (int)gridDim.x; cu.toff = grp; cu.tstep = groups; }
  MxCursor ahead = cu;                                                  // the next tile to load
  ahead.open(t);
  f4 sg;                                                                // backward: saved scores of the next tile
  auto load_scores = [&](const MxCursor& cu) {
    const int ln = mx_fresh(lane), q = ln & 7, n = (cu.tile << 5) + 8 * (ln >> 4) + 4 * ((ln >> 3) & 1);
    const float* row = p.S + ((int64_t)cu.b * p.Q + q0) * p.lds_;
    sg = *reinterpret_cast<const f4*>(row + (unsigned)((q < qn ? q : 0) * (int)p.lds_ + (n < p.lds_ ? n : (int)p.lds_ - 4)));
  };
  if constexpr (BWD) load_scores(ahead);
#pragma unroll
  for (int i = 0; i < NST; ++i) { issue(ahead, i); ahead.next(t); }

  // ---- operand rows.  Columns q and q + 8 belong to one query: lanes of the first make blocks 0 and 1, of the second blocks 2 and 3,
  // and they exchange the terms that the other's columns take.  One block at a time (as straight code this part would be several KiB of
  // instructions that run once), the operands moving up by one.
  struct { mx_u6 b[MX_WIDE_TERMS / 2]; } op[CPW];
  static_assert(MX_WIDE_TERMS == 6, "two terms an operand, as tile_step multiplies them");
  auto load_operand = [&](const float* rows, const float* prows, float mul) {
    const int ln = mx_fresh(lane), c = ln & 15, q = c & 7;
    const bool up = (c & 8) != 0;
    const int64_t at = (int64_t)(q0 + (q < qn ? q : 0)) * t.D;          // (rows without a query: the first one's, times 0)
    const int mine = chunk0 + (up ? 2 : 0);
    float sum = 0.f;
    uint32_t sc[CPW];
    mx_f16 ve, vo;
    auto load = [&](int i) {
      const bool in = mine + i < nc;
      const int d = (in ? mine + i : nc - 1) * MX_BLOCK + 32 * (ln >> 4);
      mx_load_row(rows + at + d, t.D - d, p.vecq, in && q < qn ? mul : 0.f, ve, vo);
    };
    load(1);
#pragma unroll 1
    for (int i = 1; i >= 0; --i) {
      if (BWD && prows) {
        mx_f16 we, wo;
        const int d = (mine + i < nc ? mine + i : nc - 1) * MX_BLOCK + 32 * (ln >> 4);
        mx_load_row(prows + at + d, t.D - d, p.vecq, 1.f, we, wo);
#pragma unroll
        for (int j = 0; j < 16; ++j) sum = fmaf(vo[j], wo[j], fmaf(ve[j], we[j], sum));
        __builtin_amdgcn_sched_barrier(0);
      }
      op[1] = op[0]; op[3] = op[2]; sc[1] = sc[0]; sc[3] = sc[2];
      const mx_f16 ue = ve, uo = vo;
      if (i > 0) load(0);
      __builtin_amdgcn_sched_barrier(0);
      mx_u6 even;
      uint32_t eb = 0;
      sc[0] = sc[2] = 0;
      mx_terms<MX_WIDE_TERMS>(ue, uo, [&](int t, const mx_u6& k, uint32_t byte) {
        if (t % 2 == 0) {
          even = k; eb = byte;
        } else {                                                        // columns 0-7 take the even term, 8-15 the odd one
#pragma unroll
          for (int w = 0; w < 6; ++w) {
            const uint32_t other = mx_ror8u(up ? even[w] : k[w]);
            op[0].b[t / 2][w] = up ? other : even[w];
            op[2].b[t / 2][w] = up ? k[w] : other;
          }
          const uint32_t other = mx_ror8u(up ? eb : byte);
          sc[0] |= (up ? other : eb) << (8 * (t / 2));
          sc[2] |= (up ? byte : other) << (8 * (t / 2));
        }
      });
      __builtin_amdgcn_sched_barrier(0);
    }
    *reinterpret_cast<mx_u4*>(opsc + ln * 16) = mx_u4{sc[0], sc[1], sc[2], sc[3]};
    return BWD && prows ? mx_over_groups_sum(sum + mx_ror8(sum)) : 0.f;
  };
  float delta = 0.f, m_run, l_run, t_max, invl;                         // m_run: what weights are taken against (-inf: no token yet)
  auto base = [](float m) { return m == -INFINITY ? 0.f : m; };
  auto open_unit = [&](int b) {                                         // backward: dP's rows and the saved statistics
    delta = load_operand(p.q + (int64_t)b * p.Q * t.D, p.Pin ? p.Pin + (int64_t)b * p.Q * t.D : nullptr, 1.f);
    const int q = mx_fresh(lane) & 7;
    f4 ml = {0.f, 0.f, 0.f, 0.f};
    if (q < qn) ml = *reinterpret_cast<const f4*>(p.ML + ((int64_t)b * p.Q + q0 + q) * 4);
    m_run = ml.x;
    invl = ml.y == 0.f ? 0.f : 1.f / ml.y;
    if (!p.Pin && dw == 0) delta = ml.z;                                // (each D-slice takes off its own part of delta)
  };
  f4 acc[CPW][8];
  auto clear = [&]() {
#pragma unroll
    for (int k = 0; k < CPW; ++k)
#pragma unroll
      for (int j = 0; j < 8; ++j) acc[k][j] = f4{0.f, 0.f, 0.f, 0.f};
  };
  clear();
  int slot = 0, buf = 0;

  // acc rows 4 g + i are queries (4 g + i) % 8; multiply each by the value that lane (c = query) holds
  auto scale_rows = [&](float f) {
    const int g = mx_fresh(lane) >> 4;
    float r[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) r[i] = __shfl(f, (4 * g + i) & 7, 64);
#pragma unroll
    for (int k = 0; k < CPW; ++k)
#pragma unroll
      for (int j = 0; j < 8; ++j) { acc[k][j].x *= r[0]; acc[k][j].y *= r[1]; acc[k][j].z *= r[2]; acc[k][j].w *= r[3]; }
  };

  auto tile_step = [&](int b, int t0, int len) {
    const char* st = ring + slot * STAGE;
    f4 s;
    {
      mx_wait_vm<(NST - 1) * OPS>();
      // first contraction, sixteen tokens at a time.  Leading and lower terms are kept apart: an addition to a large sum costs its last bit
      const int ln = mx_fresh(lane), c = ln & 15, g = ln >> 4;
      const char* codes = st + (4 * (c & 3) + (c >> 2)) * 64 + ((g ^ (c & 3)) << 4);
      const char* scl = st + CODES + (8 * (c >> 2) + (c & 3)) * 4;
      const mx_u4 osc = *reinterpret_cast<const mx_u4*>(opsc + ln * 16);
      f4 sum[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        __builtin_amdgcn_sched_barrier(0);
        f4 sa = {0.f, 0.f, 0.f, 0.f}, sl = sa;
#pragma unroll
        for (int k = 0; k < CPW; ++k) {
          const mx_u4 w = *reinterpret_cast<const mx_u4*>(codes + k * 2048 + h * 1024);
          const uint32_t sc = *reinterpret_cast<const uint32_t*>(scl + k * 128 + h * 16) >> (8 * g);
          sa = mx_mfma_codes<0>(w, sc, op[k].b[0], osc[k], sa);
          sl = mx_mfma_codes<2>(w, sc, op[k].b[2], osc[k], sl);
          sl = mx_mfma_codes<1>(w, sc, op[k].b[1], osc[k], sl);
        }
        sum[h] = sa + sl;
      }
      const bool up = (c & 8) != 0;                                    // columns q and q + 8 are terms of one query
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float own = up ? sum[1][i] : sum[0][i], oth = up ? sum[0][i] : sum[1][i];
        s[i] = own + mx_ror8(oth) - (BWD ? delta : 0.f);
      }
    }
    __builtin_amdgcn_sched_barrier(0);
    if (nw > 1) {                                                       // add the D-slices
      char* ex = exch + (buf * groups + grp) * nw * REC + mx_fresh(lane) * 16;
      *reinterpret_cast<f4*>(ex + dw * REC) = s;
      mx_barrier();
      buf ^= 1;
      s = *reinterpret_cast<const f4*>(ex);
#pragma unroll 4
      for (int o = 1; o < nw; ++o) s += *reinterpret_cast<const f4*>(ex + o * REC);
    }
    const bool tail = t0 + 32 > len;
    // weights
    mx_u4 wt[2];
    {
      const int ln = mx_fresh(lane), c = ln & 15, tok0 = 8 * (ln >> 4) + 4 * (c >> 3);      // the lane's first token in the tile
      float pv[4];
      if constexpr (!BWD) {
        if (tail) {
#pragma unroll
          for (int i = 0; i < 4; ++i) s[i] = t0 + tok0 + i < len ? s[i] : -INFINITY;
        }
        if (p.S && dw == 0) {
          const int q = c & 7;
          if (q < qn && t0 + tok0 < t.N) *reinterpret_cast<f4*>(p.S + ((int64_t)b * p.Q + q0 + q) * p.lds_ + t0 + tok0) = s;
        }
        float mx = fmaxf(fmaxf(s[0], s[1]), fmaxf(s[2], s[3]));
        t_max = fmaxf(t_max, mx);
        if (__any(mx > m_run + MX_LAZY)) {
          mx = mx_over_groups_max(fmaxf(mx, mx_ror8(mx)));
          const float mn = fmaxf(m_run, mx);
          const float f = mn == m_run ? 1.f : __builtin_amdgcn_exp2f((m_run - mn) * MX_LOG2E);
          m_run = mn;
          l_run *= f;
          scale_rows(f);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) { pv[i] = __builtin_amdgcn_exp2f((s[i] - base(m_run)) * MX_LOG2E); l_run += pv[i]; }
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) pv[i] = __builtin_amdgcn_exp2f((sg[i] - m_run) * MX_LOG2E) * invl * s[i];
        if (tail) {
#pragma unroll
          for (int i = 0; i < 4; ++i) pv[i] = t0 + tok0 + i < len ? pv[i] : 0.f;
        }
      }
      // three bf16 terms, exact: the upper half of the bits, of what is left, and of what is left then
      uint32_t H[2], M[2], L[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const float a = pv[2 * i], b2 = pv[2 * i + 1];
        const float ra = a - __uint_as_float(__float_as_uint(a) & 0xffff0000u), rb = b2 - __uint_as_float(__float_as_uint(b2) & 0xffff0000u);
        const float la = ra - __uint_as_float(__float_as_uint(ra) & 0xffff0000u), lb = rb - __uint_as_float(__float_as_uint(rb) & 0xffff0000u);
        H[i] = __builtin_amdgcn_perm(__float_as_uint(b2), __float_as_uint(a), 0x07060302u);
        M[i] = __builtin_amdgcn_perm(__float_as_uint(rb), __float_as_uint(ra), 0x07060302u);
        L[i] = __builtin_amdgcn_perm(__float_as_uint(lb), __float_as_uint(la), 0x07060302u);
      }
      const bool up = (c & 8) != 0;                                     // rows 0-7: first and third term, rows 8-15: second; 8 slots = both halves
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const uint32_t r1 = mx_ror8u(up ? H[i] : M[i]), r2 = mx_ror8u(L[i]);
        wt[0][i] = up ? r1 : H[i];
        wt[0][2 + i] = up ? M[i] : r1;
        wt[1][i] = up ? 0u : L[i];
        wt[1][2 + i] = up ? 0u : r2;
      }
    }
    // second contraction
    __builtin_amdgcn_sched_barrier(0);
    {
      const int ln = mx_fresh(lane), c = ln & 15, g = ln >> 4;
      const int p_off = g * 64 + c * 4;                                 // slot i: (p_off ^ 16 (i % 4)) + 256 i
      const uint32_t rot = (uint32_t)(8 * (c >> 2) + 9);
#pragma unroll
      for (int k = 0; k < CPW; ++k) {
        uint32_t w[8];
        float sc[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          w[i] = *reinterpret_cast<const uint32_t*>(st + k * 2048 + i * 256 + (p_off ^ ((i & 3) << 4)));
          const uint32_t four = *reinterpret_cast<const uint32_t*>(st + CODES + k * 128 + g * 32 + i * 4);
          sc[i] = __uint_as_float(__builtin_amdgcn_alignbit(four, four, rot));
        }
#define EP_MX_PAIR(PR)                                                                                                   \
  do {                                                                                                                   \
    uint32_t x[8];                                                                                                       \
    _Pragma("unroll") for (int i = 0; i < 8; ++i) x[i] = mx_pair<PR>(w[i], sc[i]);                                      \
    mx_u4 ev, od;                                                                                                        \
    _Pragma("unroll") for (int i = 0; i < 4; ++i) {                                                                     \
      ev[i] = __builtin_amdgcn_perm(x[2 * i + 1], x[2 * i], 0x05040100u);                                                \
      od[i] = __builtin_amdgcn_perm(x[2 * i + 1], x[2 * i], 0x07060302u);                                                \
    }                                                                                                                    \
    _Pragma("unroll") for (int z = 1; z >= 0; --z) {                                                                    \
      acc[k][2 * PR] = mx_mfma(wt[z], ev, acc[k][2 * PR]);                                                               \
      acc[k][2 * PR + 1] = mx_mfma(wt[z], od, acc[k][2 * PR + 1]);                                                       \
    }                                                                                                                    \
  } while (0)
        EP_MX_PAIR(0); EP_MX_PAIR(1); EP_MX_PAIR(2); EP_MX_PAIR(3);
        __builtin_amdgcn_sched_barrier(0);
#undef EP_MX_PAIR
      }
    }
  };
  // the stage is read: load the tile NST further on into it.  The loads always are the same number (at the end of the sequence they
  // repeat one row), so a counted wait means the same everywhere; the next tile's scores are asked for in front of them, so that
  // waiting for the scores does not wait for the tile.
  auto refill = [&]() {
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    if constexpr (BWD) load_scores(cu);
    issue(ahead, slot);
    ahead.next(t);
    slot = slot + 1 == NST ? 0 : slot + 1;
  };

  // store (or add) acc times inv(query) as rows of out (row stride D), the two term rows added first
  auto store_rows = [&](float* out, float inv, bool add) {
    const int ln = mx_fresh(lane), c = ln & 15, g = ln >> 4;
    float r[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) r[i] = __shfl(inv, 4 * (g & 1) + i, 64);
#pragma unroll
    for (int k = 0; k < CPW; ++k)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int q = 4 * (g & 1) + i;
        float* o = out + (int64_t)(q0 + q) * t.D;
        __builtin_amdgcn_sched_barrier(0);                               // row by row: the added values of all rows at once would not fit
        f4 x;
#pragma unroll
        for (int j = 0; j < 4; ++j) x[j] = fold32(acc[k][j][i], acc[k][j + 4][i]) * r[i];
        const int d = (chunk0 + k) * MX_BLOCK + 8 * c + 4 * (g >> 1);
        if (q < qn && chunk0 + k < nc) {
          if (p.veco) {
            if (d < t.D) {
              if (BWD && add) x += *reinterpret_cast<const f4*>(o + d);
              *reinterpret_cast<f4*>(o + d) = x;
            }
          } else {
#pragma unroll
            for (int j = 0; j < 4; ++j)
              if (d + j < t.D) o[d + j] = BWD && add ? o[d + j] + x[j] : x[j];
          }
        }
      }
  };
  // add the groups' accumulators into group 0's, half a row block at a time, through the exchange records (2 groups nw of them, at
  // least 4 KiB a wave of a group)
  auto add_groups = [&]() {
    const int ln = mx_fresh(lane);
    for (int o = 1; o < groups; ++o) {
#pragma unroll
      for (int k = 0; k < CPW; ++k)
#pragma unroll
        for (int j0 = 0; j0 < 8; j0 += 4) {
          if (grp == o) {
#pragma unroll
            for (int j = 0; j < 4; ++j) *reinterpret_cast<f4*>(exch + (dw * 4 + j) * 1024 + ln * 16) = acc[k][j0 + j];
          }
          mx_barrier();
          if (grp == 0) {
#pragma unroll
            for (int j = 0; j < 4; ++j) acc[k][j0 + j] += *reinterpret_cast<const f4*>(exch + (dw * 4 + j) * 1024 + ln * 16);
          }
          mx_barrier();
        }
    }
  };

  if constexpr (!BWD) {
    if constexpr (!OPENS) load_operand(p.q, nullptr, p.scale);
    for (int u = (int)blockIdx.x; u < p.units; u += (int)gridDim.x) {
      const int b = u / p.splits, sp = u - b * p.splits;
      int len;
      const int img = mx_image_uniform(t, b, len);
      const int n = (len + 31) >> 5, lo = sp * p.tps, hi = (sp + 1) * p.tps < n ? (sp + 1) * p.tps : n;
      if constexpr (OPENS) load_operand(p.q + (int64_t)b * p.qb, nullptr, p.scale);
      m_run = t_max = -INFINITY; l_run = 0.f;
      clear();
      int tl = lo;
      for (; tl + grp < hi; tl += groups) {
        tile_step(b, (tl + grp) << 5, len);
        refill();
      }
      if (tl < hi && nw > 1) mx_barrier();                              // a group without a tile in the last round keeps the others' barrier
      const int ln = mx_fresh(lane), c = ln & 15, g = ln >> 4;
      if (p.S && sp == p.splits - 1 && dw == 0 && grp == 0) {           // scores behind the image's tiles
        for (int q = 0; q < qn; ++q)
          for (int i = (n << 5) + ln; i < t.N; i += 64) p.S[((int64_t)b * p.Q + q0 + q) * p.lds_ + i] = img < 0 ? __uint_as_float(0x7fc00000u) : -INFINITY;
      }
      l_run = mx_over_groups_sum(l_run + mx_ror8(l_run));               // over the lanes of a query
      t_max = mx_over_groups_max(fmaxf(t_max, mx_ror8(t_max)));
      if (groups > 1) {
        float* ml = reinterpret_cast<float*>(exch);                     // [groups][16][3]
        mx_barrier();
        if (dw == 0 && g == 0) {
          float* e = ml + (grp * 16 + c) * 3;
          e[0] = m_run; e[1] = l_run; e[2] = t_max;
        }
        mx_barrier();
        float M = -INFINITY, T = -INFINITY, l = 0.f;
        for (int o = 0; o < groups; ++o) { const float* e = ml + (o * 16 + c) * 3; M = fmaxf(M, e[0]); T = fmaxf(T, e[2]); }
        for (int o = 0; o < groups; ++o) {
          const float* e = ml + (o * 16 + c) * 3;
          l += e[0] == M ? e[1] : e[1] * __builtin_amdgcn_exp2f((e[0] - M) * MX_LOG2E);
        }
        const float own = m_run == M ? 1.f : __builtin_amdgcn_exp2f((m_run - M) * MX_LOG2E);
        scale_rows(own);
        m_run = M; l_run = l; t_max = T;
        mx_barrier();                                                   // (the records are read: they carry accumulators next)
        add_groups();
      }
      if (grp == 0) {
        const float bad = img < 0 ? __uint_as_float(0x7fc00000u) : 0.f;
        const bool none = t_max == -INFINITY && l_run == 0.f;                                 // no token
        const float m = none ? (p.splits > 1 ? -INFINITY : 0.f) : t_max;
        const float e = none ? 0.f : __builtin_amdgcn_exp2f((base(m_run) - m) * MX_LOG2E);             // from the running to the true maximum
        if (dw == 0 && g == 0 && c < 8 && c < qn) {
          if (p.splits > 1) *reinterpret_cast<f2*>(p.part_ml + ((int64_t)u * p.Q + q0 + c) * 2) = f2{m + bad, l_run * e + bad};
          else *reinterpret_cast<f4*>(p.ML + ((int64_t)b * p.Q + q0 + c) * 4) = f4{m + bad, l_run * e + bad, 0.f, 0.f};
        }
        store_rows(p.splits > 1 ? p.part + (int64_t)u * p.Q * t.D : p.P + (int64_t)b * p.Q * t.D, (p.splits > 1 ? e : (none ? 0.f : 1.f / l_run)) + bad, false);
      }
    }
  } else {
    const int rounds = (p.units + cu.ustep - 1) / cu.ustep;
    int u = cu.u;
    cu.open(t);
    for (int r = 0; r < rounds; ++r, u += cu.ustep) {                   // a group's r-th unit; the sum over rounds and groups is in a fixed order
      if (cu.valid() && cu.u == u) open_unit(cu.b);
      clear();
      int it = 0;
      for (; cu.u == u && u < p.units; ++it) {
        tile_step(cu.b, cu.tile << 5, cu.len);
        cu.next(t);
        refill();
      }
      if (nw > 1)
        for (; it < p.tps; ++it) mx_barrier();                          // groups with fewer tiles keep the others' barriers
      if (p.per_unit) {                                                 // one gradient per image (and split)
        if (u < p.units) store_rows(p.part + (int64_t)u * p.Q * t.D, p.scale, false);
      } else {
        if (groups > 1) { mx_barrier(); add_groups(); }
        if (grp == 0) store_rows(p.part + (int64_t)blockIdx.x * p.Q * t.D, p.scale, r > 0);
      }
    }
  }
  mx_wait_vm<0>();                                                      // no load into LDS outlives its wave
}

// ---- the pipelined form --------------------------------------------------------------------------------------------------
// One 128-channel block per wave (nw pool waves) and one wave more that makes the weights.  Per tile j of the workgroup's sequence:
//     pool waves   first contraction of tile j -> record j | barrier j | second contraction of tile j - 1, refill its stage
//     weight wave                                          | barrier j | sums the records of tile j, softmax (or dS), weights j
// so that the long chain exchange -> maximum -> exponentials -> split runs beside the contractions of other tiles, once per tile
// instead of once per wave, and the pool waves' registers (accumulators and operand of one block) leave room for 4 waves a SIMD.
// OPENS: the operand rows change with the image (backward, per-image queries); else they are made once.  QM 16 and the backward pass make the
// lane constants of a step where they are used: with seven terms there are no registers to keep them in.
template <int QM, bool BWD, bool OPENS>
__global__ __launch_bounds__(1024, 4) void ep_mx4_pipe_kernel(MxPool p) {
  typedef MxDims<QM> DM;
  constexpr int SV = DM::SV, PREC = 2048;            // a record: the accumulators as they are
  constexpr int NST = MX_PIPE_STAGES, STAGE = 2048 + 128, OPS = 3;
  constexpr int WREC = DM::PSETS * 1024, WALL = WREC + 128 + 64;      // weights, rescaling factors, row factors, flags
  extern __shared__ __align__(16) char lds[];
  const int lane = lane_id(), c = lane & 15, g = lane >> 4;
  const int wave = wave_id_uniform();
  const ep_mx4_tokens& t = p.t;
  const int nw = p.nw, rowC = p.nc * 64, rowS = p.nc * 4;
  const int q0 = (int)blockIdx.y * p.qblk, qn = p.Q - q0 < p.qblk ? p.Q - q0 : p.qblk;      // queries of this workgroup
  char* recs = lds + nw * (NST * STAGE);                                // [2][nw][REC]
  char* wbuf = recs + 2 * nw * PREC;                                 // [2][WALL]
  float* dbuf = reinterpret_cast<float*>(wbuf + 2 * WALL);              // [2][nw][16]: the blocks' parts of delta, by parity of the unit
  const int tok0 = 8 * g + (QM == 8 ? 4 * (c >> 3) : 0);                // first token of the lane's scores in a tile
  const float NANF = __uint_as_float(0x7fc00000u);

  MxCursor start;
  start.units = p.units; start.splits = p.splits; start.tps = p.tps;
  start.u = (int)blockIdx.x; start.ustep = (int)gridDim.x; start.toff = 0; start.tstep = 1;

  if (wave < nw) {                                                      // ================= pool waves
    char* ring = lds + wave * (NST * STAGE);
    // lane offsets of a whole tile; rows behind an image's end repeat its last one
    const int dtok = 8 * ((lane >> 2) & 3) + g;
    const unsigned dseg = (unsigned)(((lane & 3) ^ g) * 16);
    const unsigned full0 = (unsigned)(dtok * rowC) + dseg, fulls = (unsigned)((lane & 31) * rowS);
    MxCursor ahead;                                                     // the tile to load, and where it lies
    const uint8_t *src, *scl;
    auto locate = [&]() {
      const int64_t t0 = (int64_t)ahead.tile << 5;
      src = t.codes + (int64_t)ahead.img * t.codes_bstride + t0 * rowC + wave * 64;
      scl = t.scales + (int64_t)ahead.img * t.scales_bstride + t0 * rowS + wave * 4;
    };
    auto load_tile = [&](int slot) {                                    // ... into the ring; and on to the next
      char* st = ring + slot * STAGE;
      const int last = ahead.len - (ahead.tile << 5) - 1;
      unsigned off0 = full0, off1 = full0 + 4 * rowC, offs = fulls;
      if (last < 31) {
        off0 = (unsigned)((dtok < last ? dtok : last) * rowC) + dseg;
        off1 = (unsigned)((dtok + 4 < last ? dtok + 4 : last) * rowC) + dseg;
        offs = (unsigned)(((lane & 31) < last ? (lane & 31) : last) * rowS);
      }
      __builtin_amdgcn_global_load_lds((mx_gptr_t)(src + off0), (mx_lds_t)st, 16, 0, MX_NT);
      __builtin_amdgcn_global_load_lds((mx_gptr_t)(src + off1), (mx_lds_t)(st + 1024), 16, 0, MX_NT);
      if (lane < 32) __builtin_amdgcn_global_load_lds((mx_gptr_t)(scl + offs), (mx_lds_t)(st + 2048), 4, 0, 0);
      src += 32 * rowC; scl += 32 * rowS;
      if (ahead.next(t)) locate();
    };

    MxCursor cs = start;                                                // the tile to score
    cs.open(t);
    ahead = cs;
    locate();
#pragma unroll
    for (int i = 0; i < NST; ++i) load_tile(i);
    MxCursor cp = cs;                                                   // the tile to pool

    MxOperand<QM> op;
    int parity = 0;
    auto open_unit = [&](int b) {                                       // the operand rows; backward: this block's part of delta = dP . P
      const int ln = mx_fresh(lane), c = ln & 15, g = ln >> 4;
      const float* rows = p.q + (BWD ? (int64_t)b * p.Q * t.D : (int64_t)b * p.qb);
      const int q = QM == 8 ? c & 7 : c;
      const int lo = wave * MX_BLOCK + 32 * g;
      const int64_t at = (int64_t)(q0 + (q < qn ? q : 0)) * t.D + lo;   // (rows without a query: the first one's, times 0)
      mx_f16 ve, vo;
      mx_load_row(rows + at, t.D - lo, p.vecq, q < qn ? (BWD ? 1.f : p.scale) : 0.f, ve, vo);
      if (BWD && p.Pin) {
        float d = 0.f;
        mx_f16 we, wo;
        mx_load_row(p.Pin + (int64_t)b * p.Q * t.D + at, t.D - lo, p.vecq, 1.f, we, wo);
#pragma unroll
        for (int i = 0; i < 16; ++i) d = fmaf(vo[i], wo[i], fmaf(ve[i], we[i], d));
        d = mx_over_groups_sum(d);
        if (g == 0) dbuf[((parity * nw + wave)) * 16 + c] = d;
        __builtin_amdgcn_sched_barrier(0);
      }
      mx_operand<QM>(ve, vo, c, op);
      __builtin_amdgcn_sched_barrier(0);
      parity ^= 1;
    };

    f4 acc[8];
    auto clear = [&]() {
#pragma unroll
      for (int j = 0; j < 8; ++j) acc[j] = f4{0.f, 0.f, 0.f, 0.f};
    };
    // acc times r (one factor per row 4 g + i) as rows of out: QM 8 adds the two term rows first
    auto store_rows = [&](float* out, const f4 (&r), bool add) {
      const int ln = mx_fresh(lane), c = ln & 15, g = ln >> 4;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int q = QM == 8 ? 4 * (g & 1) + i : 4 * g + i;
        float* o = out + (int64_t)(q0 + q) * t.D;
        __builtin_amdgcn_sched_barrier(0);
        constexpr int NV = QM == 8 ? 1 : 2;
#pragma unroll
        for (int v = 0; v < NV; ++v) {
          f4 x;
#pragma unroll
          for (int j = 0; j < 4; ++j) x[j] = (QM == 8 ? fold32(acc[j][i], acc[j + 4][i]) : acc[4 * v + j][i]) * r[i];
          const int d = wave * MX_BLOCK + 8 * c + (QM == 8 ? 4 * (g >> 1) : 4 * v);
          if (q < qn) {
            if (p.veco) {
              if (d < t.D) {
                if (BWD && add) x += *reinterpret_cast<const f4*>(o + d);
                *reinterpret_cast<f4*>(o + d) = x;
              }
            } else {
#pragma unroll
              for (int j = 0; j < 4; ++j)
                if (d + j < t.D) o[d + j] = BWD && add ? o[d + j] + x[j] : x[j];
            }
          }
        }
      }
    };
    int sslot = 0, pslot = 0, buf = 0;

    auto scores = [&]() {                                               // first contraction of the ring's stage sslot -> record
      mx_wait_vm<(NST - 2) * OPS>();
      const int ln = QM == 8 && !BWD ? lane : mx_fresh(lane), c = ln & 15, g = ln >> 4;
      const int sc_off = (8 * (c >> 2) + (c & 3)) * 4;                  // + 16 h: scale dword of the score row
      const int a_off = (4 * (c & 3) + (c >> 2)) * 64 + ((g ^ (c & 3)) << 4);
      const char* st = ring + sslot * STAGE;
      char* rec = recs + (buf * nw + wave) * PREC;
      mx_u4 w[2];
      uint32_t sc[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        w[h] = *reinterpret_cast<const mx_u4*>(st + h * 1024 + a_off);
        sc[h] = *reinterpret_cast<const uint32_t*>(st + 2048 + h * 16 + sc_off) >> (8 * g);
      }
      // lower terms first: only the last addition, the leading term's, rounds at the size of the score
      f4 s[2];
      const MxOperand<QM>& o = op;
      s[0] = s[1] = f4{0.f, 0.f, 0.f, 0.f};
#define EP_MX_TERM(Z)                                                                                                    \
  if constexpr (DM::SETS > Z) {                                                                                          \
    _Pragma("unroll") for (int h = 0; h < 2; ++h) s[h] = mx_mfma_codes<Z % 4>(w[h], sc[h], o.b[Z], o.sc[Z / 4], s[h]);   \
  }
      EP_MX_TERM(6) EP_MX_TERM(5) EP_MX_TERM(4) EP_MX_TERM(3) EP_MX_TERM(2) EP_MX_TERM(1) EP_MX_TERM(0)
#undef EP_MX_TERM
#pragma unroll
      for (int h = 0; h < 2; ++h) *reinterpret_cast<f4*>(rec + h * 1024 + ln * 16) = s[h];
      sslot = sslot + 1 == NST ? 0 : sslot + 1;
    };

    uint32_t w[8], s4[8];
    auto fetch = [&]() {                                                // the codes and scales of stage pslot: asked for in front of the barrier
      const char* st = ring + pslot * STAGE;
      const int ln = QM == 8 && !BWD ? lane : mx_fresh(lane), c = ln & 15, g = ln >> 4;
      const int p_off = g * 64 + c * 4;                                 // slot i: (p_off ^ 16 (i % 4)) + 256 i
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        w[i] = *reinterpret_cast<const uint32_t*>(st + i * 256 + (p_off ^ ((i & 3) << 4)));
        s4[i] = *reinterpret_cast<const uint32_t*>(st + 2048 + g * 32 + i * 4);
      }
    };
    auto pool = [&]() {                                                 // second contraction of stage pslot with the weights of buffer buf
      const char* wr = wbuf + buf * WALL;
      const int ln = QM == 8 && !BWD ? lane : mx_fresh(lane), c = ln & 15, g = ln >> 4;
      const uint32_t rot = (uint32_t)(8 * (c >> 2) + 9);
      mx_u4 wt[DM::PSETS];
#pragma unroll
      for (int z = 0; z < DM::PSETS; ++z) wt[z] = *reinterpret_cast<const mx_u4*>(wr + z * 1024 + ln * 16);
      if constexpr (!BWD) {
        if (__builtin_amdgcn_readfirstlane(*reinterpret_cast<const int*>(wr + WREC + 128))) {        // the running maximum has moved
          const f4 r = *reinterpret_cast<const f4*>(wr + WREC + (QM == 8 ? 16 * (g & 1) : 16 * g));
#pragma unroll
          for (int j = 0; j < 8; ++j) acc[j] *= r;
        }
      }
      float sc[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) sc[i] = __uint_as_float(__builtin_amdgcn_alignbit(s4[i], s4[i], rot));
#define EP_MX_PAIR(PR)                                                                                                   \
  do {                                                                                                                   \
    uint32_t x[8];                                                                                                       \
    _Pragma("unroll") for (int i = 0; i < 8; ++i) x[i] = mx_pair<PR>(w[i], sc[i]);                                      \
    mx_u4 ev, od;                                                                                                        \
    _Pragma("unroll") for (int i = 0; i < 4; ++i) {                                                                     \
      ev[i] = __builtin_amdgcn_perm(x[2 * i + 1], x[2 * i], 0x05040100u);                                                \
      od[i] = __builtin_amdgcn_perm(x[2 * i + 1], x[2 * i], 0x07060302u);                                                \
    }                                                                                                                    \
    _Pragma("unroll") for (int z = DM::PSETS - 1; z >= 0; --z) {     \
      acc[2 * PR] = mx_mfma(wt[z], ev, acc[2 * PR]);                                                         \
      acc[2 * PR + 1] = mx_mfma(wt[z], od, acc[2 * PR + 1]);                                                 \
    }                                                                                                                    \
  } while (0)
      EP_MX_PAIR(0); EP_MX_PAIR(1); EP_MX_PAIR(2); EP_MX_PAIR(3);
#undef EP_MX_PAIR
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");                // the stage is read
      load_tile(pslot);
      pslot = pslot + 1 == NST ? 0 : pslot + 1;
    };

    // The sequence of tiles; where the operand changes with the image, one sequence per unit: the accumulators are written out (added to
    // the workgroup's partial gradient) before the next rows are made, for which there would be no registers beside them.
    bool first = true;
    while (cs.valid()) {
      open_unit(cs.b);
      clear();
      const int unit = cs.u;
      scores();
      buf ^= 1;
      cs.next(t);
      mx_barrier();
      for (;;) {
        const bool more = cs.valid() && (!OPENS || cs.u == unit);
        fetch();
        if (more) scores();
        mx_barrier();
        buf ^= 1;                                                       // (the parity of the tile before)
        pool();
        const int u = cp.u, b = cp.b;
        const bool done = cp.next(t);                                   // that was the unit's last tile
        if constexpr (!BWD) {
          if (done) {
            f4 r;
            r = *reinterpret_cast<const f4*>(wbuf + buf * WALL + WREC + 64 + (QM == 8 ? 16 * (g & 1) : 16 * g));
            store_rows(p.splits > 1 ? p.part + (int64_t)u * p.Q * t.D : p.P + (int64_t)b * p.Q * t.D, r, false);
            if (!OPENS) clear();
          }
        }
        if (!more) break;
        cs.next(t);
      }
      buf ^= 1;
      if constexpr (BWD) {
        f4 one;
        one = f4{p.scale, p.scale, p.scale, p.scale};
        store_rows(p.part + (int64_t)(p.per_unit ? unit : (int)blockIdx.x) * p.Q * t.D, one, !p.per_unit && !first);
      }
      first = false;
    }
    if (!BWD || p.per_unit) {                                           // units without a token
      clear();
      for (int u = (int)blockIdx.x; u < p.units; u += (int)gridDim.x) {
        const int b = u / p.splits, sp = u - b * p.splits;
        int len;
        const int img = mx_image_uniform(t, b, len);
        if (sp * p.tps < (len + 31) >> 5) continue;
        const float f = !BWD && img < 0 ? NANF : 0.f;
        f4 r;
        r = f4{f, f, f, f};
        store_rows(BWD || p.splits > 1 ? p.part + (int64_t)u * p.Q * t.D : p.P + (int64_t)b * p.Q * t.D, r, false);
      }
    } else if (first) {                                                 // no unit of this workgroup had a token
      clear();
      f4 r;
      r = f4{0.f, 0.f, 0.f, 0.f};
      store_rows(p.part + (int64_t)blockIdx.x * p.Q * t.D, r, false);
    }
    mx_wait_vm<0>();                                                    // no load into LDS outlives its wave
  } else {                                                              // ================= weight wave
    __builtin_amdgcn_s_setprio(3);                                      // the pool waves wait for it at every barrier
    MxCursor cw = start;
    cw.open(t);
    float m_run, mz, l_run, t_max, invl, dml, sg[SV];
    auto load_scores = [&](const MxCursor& cu) {                        // backward: the saved scores of a tile
      const int q = QM == 8 ? c & 7 : c;
      const float* row = p.S + ((int64_t)cu.b * p.Q + q0) * p.lds_;
#pragma unroll
      for (int h = 0; h < SV / 4; ++h) {
        const int n = (cu.tile << 5) + tok0 + 4 * h;
        const f4 v = *reinterpret_cast<const f4*>(row + (unsigned)((q < qn ? q : 0) * (int)p.lds_ + (n < p.lds_ ? n : (int)p.lds_ - 4)));
        sg[4 * h] = v.x; sg[4 * h + 1] = v.y; sg[4 * h + 2] = v.z; sg[4 * h + 3] = v.w;
      }
    };
    auto open_unit = [&](int b) {
      m_run = t_max = -INFINITY; mz = l_run = 0.f;
      if constexpr (BWD) {
        const int q = QM == 8 ? c & 7 : c;
        f4 ml = {0.f, 0.f, 0.f, 0.f};
        if (q < qn) ml = *reinterpret_cast<const f4*>(p.ML + ((int64_t)b * p.Q + q0 + q) * 4);
        mz = ml.x;
        invl = ml.y == 0.f ? 0.f : 1.f / ml.y;
        dml = ml.z;
      }
    };
    bool fresh = true;
    int buf = 0, parity = 0;
    if (BWD) load_scores(cw);
    while (cw.valid()) {
      if (fresh) open_unit(cw.b);
      mx_barrier();
      const int b = cw.b, u = cw.u, t0 = cw.tile << 5, len = cw.len;
      if (BWD && fresh && p.Pin) {                                      // delta from the blocks' parts
        float d = 0.f;
        for (int o = 0; o < nw; ++o) d += dbuf[((parity * nw + o)) * 16 + c];
        dml = d;
        parity ^= 1;
      }
      const bool tail = t0 + 32 > len;
      char* wr = wbuf + buf * WALL;
      bool moved = false;
      const int q = QM == 8 ? c & 7 : c;
      float s[SV], pv[SV];
      f4 v[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) v[h] = f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
      for (int o = 0; o < nw; ++o) {                                  // the blocks' parts, in their order
        const char* r = recs + (buf * nw + o) * PREC + lane * 16;
        v[0] += *reinterpret_cast<const f4*>(r);
        v[1] += *reinterpret_cast<const f4*>(r + 1024);
      }
      if constexpr (QM == 8) {                                        // columns q and q + 8 are terms of one query; a lane keeps one half
        const bool up = (c & 8) != 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float own = up ? v[1][i] : v[0][i], oth = up ? v[0][i] : v[1][i];
          s[i] = own + mx_ror8(oth);
        }
      } else {
#pragma unroll
        for (int i = 0; i < SV; ++i) s[i] = v[i / 4][i % 4];
      }
      if constexpr (!BWD) {
        if (tail) {
#pragma unroll
          for (int i = 0; i < SV; ++i) s[i] = t0 + tok0 + i < len ? s[i] : -INFINITY;
        }
        if (p.S && q < qn) {
          float* sp = p.S + ((int64_t)b * p.Q + q0 + q) * p.lds_ + t0 + tok0;
#pragma unroll
          for (int h = 0; h < SV / 4; ++h)
            if (t0 + tok0 + 4 * h < t.N) *reinterpret_cast<f4*>(sp + 4 * h) = f4{s[4 * h], s[4 * h + 1], s[4 * h + 2], s[4 * h + 3]};
        }
        float mx = s[0];
#pragma unroll
        for (int i = 1; i < SV; ++i) mx = fmaxf(mx, s[i]);
        t_max = fmaxf(t_max, mx);
        float f = 1.f;
        if (__any(mx > m_run + MX_LAZY)) {
          if (QM == 8) mx = fmaxf(mx, mx_ror8(mx));
          mx = mx_over_groups_max(mx);
          const float mn = fmaxf(m_run, mx);
          f = mn == m_run ? 1.f : __builtin_amdgcn_exp2f((m_run - mn) * MX_LOG2E);
          m_run = mn;
          mz = mn == -INFINITY ? 0.f : mn;
          l_run *= f;
          moved = !fresh;                                             // (nothing is accumulated in front of the first tile)
        }
        if (g == 0 && (QM != 8 || c < 8)) *reinterpret_cast<float*>(wr + WREC + c * 4) = f;
#pragma unroll
        for (int i = 0; i < SV; ++i) { pv[i] = __builtin_amdgcn_exp2f((s[i] - mz) * MX_LOG2E); l_run += pv[i]; }
      } else {
#pragma unroll
        for (int i = 0; i < SV; ++i) {
          const float a = __builtin_amdgcn_exp2f((sg[i] - mz) * MX_LOG2E) * invl;
          pv[i] = a * (s[i] - dml);
        }
        if (tail) {
#pragma unroll
          for (int i = 0; i < SV; ++i) pv[i] = t0 + tok0 + i < len ? pv[i] : 0.f;
        }
      }
      // three bf16 terms, exact: the upper half of the bits, of what is left, and of what is left then
      uint32_t H[SV / 2], M[SV / 2], L[SV / 2];
#pragma unroll
      for (int i = 0; i < SV / 2; ++i) {
        const float x = pv[2 * i], y = pv[2 * i + 1];
        const float rx = x - __uint_as_float(__float_as_uint(x) & 0xffff0000u), ry = y - __uint_as_float(__float_as_uint(y) & 0xffff0000u);
        const float lx = rx - __uint_as_float(__float_as_uint(rx) & 0xffff0000u), ly = ry - __uint_as_float(__float_as_uint(ry) & 0xffff0000u);
        H[i] = __builtin_amdgcn_perm(__float_as_uint(y), __float_as_uint(x), 0x07060302u);
        M[i] = __builtin_amdgcn_perm(__float_as_uint(ry), __float_as_uint(rx), 0x07060302u);
        L[i] = __builtin_amdgcn_perm(__float_as_uint(ly), __float_as_uint(lx), 0x07060302u);
      }
      mx_u4 wt[DM::PSETS];
      if constexpr (QM == 8) {                                        // rows 0-7: first and third term, rows 8-15: second; 8 slots = both halves
        const bool up = (c & 8) != 0;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const uint32_t r1 = mx_ror8u(up ? H[i] : M[i]), r2 = mx_ror8u(L[i]);
          wt[0][i] = up ? r1 : H[i];
          wt[0][2 + i] = up ? M[i] : r1;
          wt[1][i] = up ? 0u : L[i];
          wt[1][2 + i] = up ? 0u : r2;
        }
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) { wt[0][i] = H[i]; wt[1][i] = M[i]; wt[DM::PSETS - 1][i] = L[i]; }
      }
#pragma unroll
      for (int z = 0; z < DM::PSETS; ++z) *reinterpret_cast<mx_u4*>(wr + z * 1024 + lane * 16) = wt[z];
      fresh = cw.next(t);
      if constexpr (BWD) load_scores(cw);
      else {
        if (lane == 0) *reinterpret_cast<int*>(wr + WREC + 128) = moved;
        if (fresh) {                                                    // the unit is done: statistics, row factors, the scores behind its tiles
          const int spl = u - b * p.splits;
          const int q = QM == 8 ? c & 7 : c;
          float l = l_run, tm = t_max;
          if (QM == 8) { l += mx_ror8(l); tm = fmaxf(tm, mx_ror8(tm)); }
          l = mx_over_groups_sum(l);
          tm = mx_over_groups_max(tm);
          const float e = __builtin_amdgcn_exp2f((mz - tm) * MX_LOG2E);               // from the running to the true maximum
          if (g == 0 && (QM != 8 || c < 8)) {
            if (q < qn) {
              if (p.splits > 1) *reinterpret_cast<f2*>(p.part_ml + ((int64_t)u * p.Q + q0 + q) * 2) = f2{tm, l * e};
              else *reinterpret_cast<f4*>(p.ML + ((int64_t)b * p.Q + q0 + q) * 4) = f4{tm, l * e, 0.f, 0.f};
            }
            *reinterpret_cast<float*>(wr + WREC + 64 + c * 4) = p.splits > 1 ? e : 1.f / l;
          }
          if (p.S && spl == p.splits - 1)
            for (int q = 0; q < qn; ++q)
              for (int i = (((len + 31) >> 5) << 5) + lane; i < t.N; i += 64) p.S[((int64_t)b * p.Q + q0 + q) * p.lds_ + i] = -INFINITY;
        }
      }
      buf ^= 1;
      if (OPENS ? fresh : !cw.valid()) mx_barrier();                    // the sequence's last weights are done
    }
    if constexpr (!BWD) {                                               // units without a token
      for (int u = (int)blockIdx.x; u < p.units; u += (int)gridDim.x) {
        const int b = u / p.splits, sp = u - b * p.splits;
        int len;
        const int img = mx_image_uniform(t, b, len);
        const int n = (len + 31) >> 5;
        if (sp * p.tps < n) continue;
        const float bad = img < 0 ? NANF : 0.f;
        for (int q = lane; q < qn; q += 64) {
          if (p.splits > 1) *reinterpret_cast<f2*>(p.part_ml + ((int64_t)u * p.Q + q0 + q) * 2) = f2{img < 0 ? NANF : -INFINITY, bad};
          else *reinterpret_cast<f4*>(p.ML + ((int64_t)b * p.Q + q0 + q) * 4) = f4{bad, bad, 0.f, 0.f};
        }
        if (p.S && sp == p.splits - 1)
          for (int q = 0; q < qn; ++q)
            for (int i = (n << 5) + lane; i < t.N; i += 64) p.S[((int64_t)b * p.Q + q0 + q) * p.lds_ + i] = img < 0 ? NANF : -INFINITY;
      }
    }
  }
}

// joins the splits of an image: blockIdx.x = (image, query); CH chains of splits side by side, 1024 / CH channels a workgroup
template <int CH>
__global__ __launch_bounds__(256) void ep_mx4_join_kernel(const float* __restrict__ part, const float* __restrict__ ml, int splits, int Q, int D,
                                                          float* __restrict__ P, float* __restrict__ ML) {
  constexpr int LN = 256 / CH;
  __shared__ f4 red[CH][LN + 1];
  const int b = (int)(blockIdx.x / (unsigned)Q), q = (int)(blockIdx.x % (unsigned)Q);
  const float* e = ml + ((int64_t)b * splits * Q + q) * 2;             // {maximum, sum} of split s at e[s * 2 Q]
  const int lane = lane_id();
  float m = -INFINITY, l = 0.f;
  bool bad = false;
  for (int s = lane; s < splits; s += 64) { const float v = e[(int64_t)s * 2 * Q]; bad |= v != v; m = fmaxf(m, v); }
  m = wave_max(m);
  for (int s = lane; s < splits; s += 64) {
    const float v = e[(int64_t)s * 2 * Q + 1];
    if (v != 0.f) l += v * __builtin_amdgcn_exp2f((e[(int64_t)s * 2 * Q] - m) * MX_LOG2E);
  }
  l = wave_sum(l);
  if (__any(bad)) m = l = __uint_as_float(0x7fc00000u);
  if (threadIdx.x == 0 && blockIdx.y == 0) *reinterpret_cast<f4*>(ML + ((int64_t)b * Q + q) * 4) = f4{l == 0.f ? 0.f : m, l, 0.f, 0.f};
  const int x = (int)threadIdx.x % LN, y = (int)threadIdx.x / LN, d = ((int)blockIdx.y * LN + x) * 4;
  f4 a = {0.f, 0.f, 0.f, 0.f};
  // (a run without tokens has sum 0 and rows of zeros; nothing here waits for a comparison, so that several rows are on their way)
#pragma unroll 4
  for (int s = y; s < splits; s += CH) {
    const f2 st = *reinterpret_cast<const f2*>(e + (int64_t)s * 2 * Q);
    const float f = st.y == 0.f ? 0.f : __builtin_amdgcn_exp2f((st.x - m) * MX_LOG2E);
    const float* row = part + (((int64_t)b * splits + s) * Q + q) * D + d;
    f4 v = {0.f, 0.f, 0.f, 0.f};
    if (D % 4 == 0) { if (d < D) v = *reinterpret_cast<const f4*>(row); }
    else {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (d + j < D) v[j] = row[j];
    }
    a += f * v;
  }
  red[y][x] = a;
  __syncthreads();
  if (y) return;
  for (int k = 1; k < CH; ++k) a += red[k][x];
  const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
  for (int j = 0; j < 4; ++j)
    if (d + j < D) P[((int64_t)b * Q + q) * D + d + j] = a[j] * inv;
}

// out[i] (+)= sum over n of part[n][i]: CH interleaved chains and then these in order; blockIdx.y selects the output.  A workgroup takes
// 1024 / CH columns: few columns take 64 chains, so that the launch still fills the chip (6144 x 512: 5.5 us, with 16 chains 11.4;
// 32768 x 256: 11.5 and 6.6).
template <int CH>
__global__ __launch_bounds__(256) void ep_mx4_sum_kernel(const float* __restrict__ part, int n, int64_t len, float* __restrict__ out, int accumulate) {
  constexpr int LN = 256 / CH;
  __shared__ float red[CH][4 * LN + 1];
  const int x = (int)threadIdx.x % LN, y = (int)threadIdx.x / LN;
  const int64_t i = (int64_t)blockIdx.x * (4 * LN) + 4 * x;
  const float* src = part + (int64_t)blockIdx.y * n * len;
  f4 s = {0.f, 0.f, 0.f, 0.f};
  if (len % 4 == 0) {
    if (i < len) {
#pragma unroll 4
      for (int r = y; r < n; r += CH) s += *reinterpret_cast<const f4*>(src + (int64_t)r * len + i);
    }
  } else {
    for (int r = y; r < n; r += CH)
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (i + j < len) s[j] += src[(int64_t)r * len + i + j];
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) red[y][4 * x + j] = s[j];
  __syncthreads();
  const int64_t o = (int64_t)blockIdx.x * (4 * LN) + threadIdx.x;
  if (threadIdx.x < 4 * LN && o < len) {
    float a = 0.f;
    for (int k = 0; k < CH; ++k) a += red[k][threadIdx.x];
    float* dst = out + (int64_t)blockIdx.y * len + o;
    *dst = accumulate ? *dst + a : a;
  }
}

struct MxPlan {
  int qm, nw, groups, splits, tps, units, grid, yblk, qblk;
  bool pipe;                                                            // the pipelined form, or the wide-row form
  size_t lds, ws;                                                       // bytes
};

static size_t mx_pipe_lds(int qm, int nw) {
  const size_t wall = (qm == 8 ? 2 : 3) * 1024 + 2 * 64 + 64;
  return (size_t)nw * MX_PIPE_STAGES * 2176 + 2 * (size_t)nw * 2048 + 2 * wall + 2 * (size_t)nw * 64;
}

static MxPlan mx_plan(int B, int N, int D, int Q, bool bwd, bool per_image) {
  MxPlan p{};
  const int nc = mx_blocks(D), cus = cu_count(), tiles = (N + 31) / 32;
  constexpr int LDS = 160 * 1024;
  int cap;                                                              // workgroups that run at the same time
  if (nc <= 14) {                                                       // a wave per block and the weight wave: what 160 KiB of LDS hold.
    // (512 x 256 x 1792, 8 queries: 44 us forward and 60 backward; wide-row form 53 and 64.  Narrower rows gain more.)  More than 8
    // queries: blocks of 16 (512 x 256 x 768: 16 queries 31 us forward, as two blocks of 8 37; 8 queries as a block of 16 28, of 8 25)
    p.qm = Q <= 8 ? 8 : 16;
    p.nw = nc; p.groups = 1;
    constexpr int waves = 16;                                           // four a SIMD
    p.pipe = true;
    p.lds = mx_pipe_lds(p.qm, nc);
    const int n = (int)(LDS / p.lds);
    cap = cus * (waves / (nc + 1) < n ? waves / (nc + 1) : n);
  } else {                                                              // four blocks per wave
    p.qm = 8;
    p.nw = (nc + 3) / 4;
    p.groups = bwd || B <= cus ? 8 / p.nw : 1;
    const int waves = p.nw * p.groups;
    p.lds = (size_t)waves * (MX_STAGES * (2048 * 4 + 512)) + 3 * (size_t)waves * 1024;
    const int n = (int)(LDS / p.lds);
    cap = cus * (8 / waves < n ? 8 / waves : n);
  }
  p.yblk = (Q + p.qm - 1) / p.qm;
  p.qblk = (Q + p.yblk - 1) / p.yblk;
  // ... for each block of queries: a second round of workgroups would make its operands and fill its ring once more (256 x 196 x 1024, 32
  // queries: 36 us forward instead of 43, 50 backward instead of 58)
  cap = cap / p.yblk > 1 ? cap / p.yblk : 1;
  // few images: their token axis is cut into runs of at least `least` tiles.  Forward the runs have to be joined by a second launch, so
  // they are kept longer (64 x 257 x 768, 8 queries: 8 tiles 15.8 us, 4 17 us); backward every run opens its operand rows (128 x 196 x
  // 768: 4 tiles 20 us, 2 25 us), which wide rows still gain from (128 x 196 x 4096: 2 tiles 40 us, 4 49 us)
  const int per = p.pipe ? 1 : p.groups, least = p.pipe ? (bwd ? 4 : 8) : (bwd ? 2 : 2 * per);
  p.splits = B < cap * (bwd ? per : 1) ? (cap * (bwd ? per : 1)) / B : 1;
  if (p.splits > tiles / least) p.splits = tiles / least;
  if (p.splits < 1 || (int64_t)B * Q > 1 << 22) p.splits = 1;            // (the joining launch has a workgroup per row)
  p.tps = (tiles + p.splits - 1) / p.splits;
  p.splits = (tiles + p.tps - 1) / p.tps;
  p.units = B * p.splits;
  if (p.pipe) {
    p.grid = p.units < cap ? p.units : cap;
  } else if (bwd) {
    p.grid = (p.units + p.groups - 1) / p.groups < cap ? (p.units + p.groups - 1) / p.groups : cap;
  } else {
    p.grid = p.groups > 1 || p.units < cap ? p.units : cap;             // several groups share one unit: a workgroup each
  }
  if (bwd) p.ws = !per_image ? (size_t)p.grid * Q * D * 4 : p.splits > 1 ? (size_t)p.units * Q * D * 4 : 0;
  else p.ws = p.splits > 1 ? (size_t)p.units * Q * (D + 2) * 4 : 0;
  return p;
}

// how the operand rows lie (mx_load_row)
static int mx_rows(int D, const float* a, const float* b) { return D % 4 || !aligned16(a) || !aligned16(b) ? 0 : D % MX_BLOCK ? 1 : 2; }

template <typename K>
static int mx_launch_kernel(K* fn, const MxPool& p, const MxPlan& pl, int threads, hipStream_t st) {
  if (pl.lds > 64 * 1024) EP_HIP(hipFuncSetAttribute(reinterpret_cast<const void*>(fn), hipFuncAttributeMaxDynamicSharedMemorySize, (int)pl.lds));
  hipLaunchKernelGGL(fn, dim3((unsigned)pl.grid, (unsigned)pl.yblk), dim3((unsigned)threads), pl.lds, st, p);
  EP_LAUNCH_CHECK("MX4 attention kernel");
  return 0;
}
template <bool BWD>
static int mx_launch(const MxPool& p, const MxPlan& pl, hipStream_t st) {
  const int threads = 64 * (pl.nw + 1);
  const bool opens = BWD || p.qb;
  if (!pl.pipe) return mx_launch_kernel(opens ? ep_mx4_wide_kernel<BWD, true> : ep_mx4_wide_kernel<BWD, BWD>, p, pl, 64 * pl.nw * pl.groups, st);
  if (pl.qm == 8) return opens ? mx_launch_kernel(ep_mx4_pipe_kernel<8, BWD, true>, p, pl, threads, st) : mx_launch_kernel(ep_mx4_pipe_kernel<8, BWD, BWD>, p, pl, threads, st);
  return opens ? mx_launch_kernel(ep_mx4_pipe_kernel<16, BWD, true>, p, pl, threads, st) : mx_launch_kernel(ep_mx4_pipe_kernel<16, BWD, BWD>, p, pl, threads, st);
}

static MxPool mx_pool_params(const ep_mx4_tokens* t, int Q, float scale, const MxPlan& pl) {
  MxPool p{};
  p.t = *t; p.Q = Q; p.scale = scale; p.nc = mx_blocks(t->D);
  p.nw = pl.nw; p.groups = pl.groups; p.splits = pl.splits; p.tps = pl.tps; p.units = pl.units; p.qblk = pl.qblk;
  return p;
}

int mx4_pool_forward(const ep_mx4_tokens* t, const float* queries, int64_t q_bstride, int Q, float scale, float* P, float* S, int64_t s_stride, float* ML, void* ws,
                     size_t ws_bytes, hipStream_t st) {
  const MxPlan pl = mx_plan(t->B, t->N, t->D, Q, false, q_bstride != 0);
  EP_REQUIRE(ws_bytes >= pl.ws, EP_E_WORKSPACE, "ep_mx4_pool_forward: workspace %zu < %zu", ws_bytes, pl.ws);
  MxPool p = mx_pool_params(t, Q, scale, pl);
  p.q = queries; p.qb = q_bstride; p.vecq = mx_rows(t->D, queries, nullptr); p.P = P; p.S = S; p.ML = ML;
  p.part = static_cast<float*>(ws); p.part_ml = p.part + (size_t)pl.units * Q * t->D;
  p.veco = t->D % 4 == 0 && aligned16(pl.splits > 1 ? (const void*)p.part : (const void*)P);
  p.lds_ = s_stride;
  EP_TRY(mx_launch<false>(p, pl, st));
  if (pl.splits > 1) {
    // few runs: one chain (128 x 196 x 4096, two runs: 41 us in all, sixteen chains 70); many: sixteen (2 x 50001 x 1024: 43 us, one 83)
    if (pl.splits <= 4)
      hipLaunchKernelGGL(ep_mx4_join_kernel<1>, dim3((unsigned)t->B * Q, (unsigned)((t->D + 1023) / 1024)), dim3(256), 0, st, p.part, p.part_ml, pl.splits, Q, t->D, P, ML);
    else
      hipLaunchKernelGGL(ep_mx4_join_kernel<16>, dim3((unsigned)t->B * Q, (unsigned)((t->D + 63) / 64)), dim3(256), 0, st, p.part, p.part_ml, pl.splits, Q, t->D, P, ML);
    EP_LAUNCH_CHECK("ep_mx4_join_kernel");
  }
  return 0;
}

int mx4_pool_backward(const ep_mx4_tokens* t, int Q, float scale, const float* S, int64_t s_stride, const float* ML, const float* P, const float* dP, float* dq,
                      int per_image, int accumulate, void* ws, size_t ws_bytes, hipStream_t st) {
  const MxPlan pl = mx_plan(t->B, t->N, t->D, Q, true, per_image != 0);
  EP_REQUIRE(ws_bytes >= pl.ws, EP_E_WORKSPACE, "ep_mx4_pool_backward: workspace %zu < %zu", ws_bytes, pl.ws);
  MxPool p = mx_pool_params(t, Q, scale, pl);
  p.q = dP; p.Pin = P; p.vecq = mx_rows(t->D, dP, P);
  p.S = const_cast<float*>(S); p.ML = const_cast<float*>(ML);
  p.per_unit = per_image != 0;
  p.part = per_image && pl.splits == 1 ? dq : static_cast<float*>(ws);
  p.veco = t->D % 4 == 0 && aligned16(p.part);
  p.lds_ = s_stride;
  const int64_t QD = (int64_t)Q * t->D;
  EP_TRY(mx_launch<true>(p, pl, st));
  if (!per_image || pl.splits > 1) {
    const int n = per_image ? pl.splits : pl.grid;
    const unsigned outs = per_image ? (unsigned)t->B : 1u;
    if (QD * outs < 16384)
      hipLaunchKernelGGL(ep_mx4_sum_kernel<64>, dim3((unsigned)((QD + 15) / 16), outs), dim3(256), 0, st, p.part, n, QD, dq, accumulate);
    else
      hipLaunchKernelGGL(ep_mx4_sum_kernel<16>, dim3((unsigned)((QD + 63) / 64), outs), dim3(256), 0, st, p.part, n, QD, dq, accumulate);
    EP_LAUNCH_CHECK("ep_mx4_sum_kernel");
  }
  return 0;
}

}  // namespace ep

using namespace ep;

extern "C" {

size_t ep_mx4_pool_workspace_bytes(int B, int N, int D, int Q) {
  if (B <= 0 || N <= 0 || D <= 0 || Q <= 0 || D > MX_MAX_D) return 0;
  size_t n = 0;
  for (int k = 0; k < 4; ++k) {
    const size_t w = mx_plan(B, N, D, Q, (k & 1) != 0, (k & 2) != 0).ws;
    n = w > n ? w : n;
  }
  return round_up(n, 256);
}

static int mx_pool_check(const ep_mx4_tokens* t, int Q, void* ws, size_t bytes, const char* what) {
  EP_TRY(mx4_check(t, what));
  EP_REQUIRE(Q > 0, EP_E_ARG, "%s: Q = %d", what, Q);
  EP_REQUIRE(t->D <= MX_MAX_D, EP_E_SHAPE, "%s: D = %d > %d", what, t->D, MX_MAX_D);
  EP_REQUIRE(Q <= 65535 * 8 && (int64_t)Q * t->D < 1 << 28, EP_E_SHAPE, "%s: %d queries of %d channels in one call", what, Q, t->D);
  EP_REQUIRE((int64_t)t->B * Q <= 1 << 30, EP_E_SHAPE, "%s: %d x %d rows in one call", what, t->B, Q);
  const size_t need = ep_mx4_pool_workspace_bytes(t->B, t->N, t->D, Q);
  EP_REQUIRE(bytes >= need, EP_E_WORKSPACE, "%s: workspace %zu < %zu", what, bytes, need);
  EP_REQUIRE(!need || (ws && aligned16(ws)), EP_E_ARG, "%s: the workspace must be given and 16-byte aligned", what);
  return 0;
}

int ep_mx4_pool_forward(const ep_mx4_tokens* t, const float* queries, int64_t q_bstride, int Q, float scale, float* P, float* S, int64_t s_stride, float* ML, void* workspace,
                        size_t workspace_bytes, ep_stream_t stream) {
  EP_TRY(mx_pool_check(t, Q, workspace, workspace_bytes, "ep_mx4_pool_forward"));
  EP_REQUIRE(queries && P && ML, EP_E_ARG, "ep_mx4_pool_forward: null pointer");
  EP_REQUIRE(!S || (aligned16(S) && s_stride % 4 == 0 && s_stride >= t->N && Q * s_stride <= 2147483647), EP_E_ALIGN,
             "ep_mx4_pool_forward: S must be 16-byte aligned, its row stride (%lld) a multiple of 4, at least N", (long long)s_stride);
  EP_REQUIRE(aligned16(ML), EP_E_ALIGN, "ep_mx4_pool_forward: ML must be 16-byte aligned");
  EP_REQUIRE(q_bstride == 0 || q_bstride == (int64_t)Q * t->D, EP_E_SHAPE, "ep_mx4_pool_forward: query batch stride %lld", (long long)q_bstride);
  EP_REQUIRE(t->D % MX_BLOCK || aligned16(queries), EP_E_ALIGN, "ep_mx4_pool_forward: queries must be 16-byte aligned");
  return mx4_pool_forward(t, queries, q_bstride, Q, scale, P, S, s_stride, ML, workspace, workspace_bytes, (hipStream_t)stream);
}

int ep_mx4_pool_backward(const ep_mx4_tokens* t, int Q, float scale, const float* S, int64_t s_stride, const float* ML, const float* P, const float* dP, float* dq,
                         int per_image, int accumulate, void* workspace, size_t workspace_bytes, ep_stream_t stream) {
  EP_TRY(mx_pool_check(t, Q, workspace, workspace_bytes, "ep_mx4_pool_backward"));
  EP_REQUIRE(S && ML && dP && dq, EP_E_ARG, "ep_mx4_pool_backward: null pointer");
  EP_REQUIRE(aligned16(S) && s_stride % 4 == 0 && s_stride >= t->N && Q * s_stride <= 2147483647, EP_E_ALIGN,
             "ep_mx4_pool_backward: S must be 16-byte aligned, its row stride (%lld) a multiple of 4, at least N", (long long)s_stride);
  EP_REQUIRE(aligned16(ML), EP_E_ALIGN, "ep_mx4_pool_backward: ML must be 16-byte aligned");
  EP_REQUIRE(t->D % MX_BLOCK || (aligned16(dP) && aligned16(P)), EP_E_ALIGN, "ep_mx4_pool_backward: dP and P must be 16-byte aligned");
  EP_REQUIRE(!(per_image && accumulate), EP_E_UNSUPPORTED, "ep_mx4_pool_backward: accumulate is for shared queries");
  return mx4_pool_backward(t, Q, scale, S, s_stride, ML, P, dP, dq, per_image, accumulate, workspace, workspace_bytes, (hipStream_t)stream);
}

}  // extern "C"
