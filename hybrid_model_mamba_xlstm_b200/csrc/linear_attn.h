// linear_attn.h — shared parameter blocks of the linear attention kernels (host + device).
//
// One `Problem` is a run of the recurrence over all (batch, head) pairs.  With g the head's decay
// and u = 0 .. n-1 the steps in processing order (time, or time reversed),
//   out_u = scale * [ sum_{w <= u} g^(u-w) (q_u . k_w) v_w  +  g^u q_u^T X_0 ].
// The carried matrix is kept as X = g S (the entering state already decayed once), so that chunk
// after chunk
//   out_i = scale * [ sum_{j <= i} g^(i-j) (q_i . k_j) v_j + g^i q_i^T X ]     (i, j: steps in the chunk)
//   X    <- g^C X + sum_j g^(C-j) k_j v_j^T.
// Forward in time X_0 = g s0 and the last state is S = X / g, formed without the division by taking
// exponents one lower in the last chunk.  The gradients are three more runs: with G the adjoint of S,
//   dq: (q, k, v) = (dout, v, k) from s0^T;
//   dv: (k, q, dout) and dk: (v, dout, q) in reversed time from X_0 = dsT / scale (its transpose),
// where G_(n-1) starts undecayed (x0_shift 0) and ds0 = scale * X_end keeps the last decay (end_shift 1).
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

#include "../../include/hxm.h"

namespace hxm {
namespace lattn {

struct Problem {
  const void* q;
  const void* k;
  const void* v;
  void* o;
  int64_t sq[3], sk[3], sv[3], so[3];  // element strides (b, t, h)
  int dk, dv;
  const float* s0;  // or NULL; element strides (b, h, k, v)
  int64_t s0s[4];
  float* sT;  // or NULL
  int64_t sTs[4];
  float scale, s0_scale, sT_scale;
  int reverse;
  float* ws;  // (b, h, nseg - 1, dk, dv): each earlier segment's own X_end, with nseg > 1
};

// Sizes shared by the runs of one call.
struct Common {
  int batch, heads, seqlen;
  const float* log_decay;
  const int32_t* lengths;
  int nseg, seg_len;  // time segments of seg_len steps (whole chunks) in processing order
  int* error_flag;
  long long wait_limit;
};

// Whether the tensor-core kernel takes this run (bf16; see linear_attn_tc.cu).
bool tc_ok(const Problem& p, int seqlen, hxm_dtype io);
// Runs np <= 3 problems of equal padded dk; state_only: the segment sums of pass one.
hxm_status launch_tc(const Common& c, const Problem* p, int np, bool state_only, cudaStream_t st);

}  // namespace lattn
}  // namespace hxm
