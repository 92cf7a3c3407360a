// What the two kernels behind b200_linear share: their arguments and the
// activations.
#pragma once

#include "common.cuh"

namespace b200 {

struct LinearArgs {
  const float* x_scale;  // nullable together
  const float* w_scale;
  const __nv_bfloat16* bias;      // nullable
  const __nv_bfloat16* residual;  // nullable
  __nv_bfloat16* out;
  int64_t r_row, o_row;
  int m, n;
  int k_blocks;          // stages of K
  int m_tiles, n_tiles;
  int gated;
  int act;
  int splits;            // CTAs of a cluster, each with a share of K
  int stages;
  int wide;              // out and residual take 16-byte accesses
  int32_t* dev_status;
};

// v / (1 + e^-v'): the quotient stays right at both ends (v' large and negative: 0)
B200_DEVICE float gate_by(float v, float z) { return __fdividef(v, 1.0f + __expf(-z)); }

template <int N>
B200_DEVICE void activate(float (&v)[N], int act) {
  switch (act) {  // outside the loops: one branch for N values
    case B200_ACT_RELU:
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] = v[i] < 0.0f ? 0.0f : v[i];  // NaN stays
      break;
    case B200_ACT_SILU:
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] = gate_by(v[i], v[i]);
      break;
    case B200_ACT_GELU:
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] = 0.5f * v[i] * (1.0f + erff(v[i] * 0.70710678118654752f));
      break;
    case B200_ACT_GELU_TANH:  // (1 + tanh z) / 2 = 1 / (1 + e^-2z)
#pragma unroll
      for (int i = 0; i < N; ++i)
        v[i] = gate_by(v[i], 1.5957691216057308f * (v[i] + 0.044715f * v[i] * v[i] * v[i]));
      break;
    default: break;
  }
}

}  // namespace b200

namespace b200host {

// Products of few tokens (linear_small.cu): whether one is, and its launch.
bool linear_is_small(const b200::LinearArgs& a, int k, bool fp8);
cudaError_t linear_small(const b200::LinearArgs& a, const void* x, int64_t x_stride, const void* w,
                         int64_t w_stride, int k, bool fp8, int sms, cudaStream_t stream);

}  // namespace b200host
