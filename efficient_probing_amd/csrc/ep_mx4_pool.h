// Internal interface of the attention over the MX4 token cache (ep_mx4_pool.hip).
#pragma once
#include "ep_mx4.h"

namespace ep {

constexpr int MX_STAGES = 2;             // tiles of a wave's ring: wide-row form
constexpr int MX_PIPE_STAGES = 3;        // ... and pipelined form

struct MxPool {
  ep_mx4_tokens t;
  const float* q; int64_t qb;            // operand rows of the first contraction: queries (qb: batch stride, 0 = shared), backward: dP
  int Q, qblk;                           // all queries; queries of a blockIdx.y
  float scale;
  float* P; float* S; float* ML;
  int64_t lds_;                          // row stride of S, a multiple of 4
  const float* Pin;                      // backward: P, or null (delta in ML[..][2])
  float* part; float* part_ml;           // partial results of units (forward splits, backward)
  int nc, nw, groups;                    // 128-channel blocks of a row; waves a row is cut over; such groups of waves in a workgroup
  int splits, tps, units;                // an image's tiles are cut into `splits` runs of `tps`; unit = image * splits + run
  int per_unit;                          // backward: a gradient per unit instead of per workgroup
  int vecq;                              // how the operand rows lie: 2 whole blocks, 1 whole 16-byte pieces, 0 anything
  int veco;                              // 16-byte stores to the outputs
};

int mx4_pool_forward(const ep_mx4_tokens* t, const float* queries, int64_t q_bstride, int Q, float scale, float* P, float* S, int64_t s_stride, float* ML, void* ws,
                     size_t ws_bytes, hipStream_t st);
int mx4_pool_backward(const ep_mx4_tokens* t, int Q, float scale, const float* S, int64_t s_stride, const float* ML, const float* P, const float* dP, float* dq,
                      int per_image, int accumulate, void* ws, size_t ws_bytes, hipStream_t st);

}  // namespace ep
