// RMS norm with the residual's addition, output in bf16 or in 8 bits (e4m3)
// with a scale a row, and the same 8-bit output without a norm:
//   h = x + r                        fp32 (returned rounded to bf16)
//   y = h / sqrt(mean(h^2) + eps) * w      fp32, from the unrounded h
//   s = max(max |y|, 1e-12) / 448    fp32, q = e4m3(y / s)
// The 8-bit form returns (q, s): q s is y to e4m3's 3 mantissa bits, and s is
// the row factor that the matrix product applies in its epilogue.
//
// Bound by memory: x and r are read once, h and y (or q, s) written once, so
// a row stays in registers between the reduction and the output.  A row is
// held by one group of threads, up to four 8-element vectors (or up to 8
// single elements where a row is not aligned) each; rows wider than a group
// of 1024 threads can hold are read again for the output.
// One reduction a row serves both statistics: y is h w times a positive row
// factor, so max |y| = rstd max |h w|, and (sum h^2, max |h w|) travel through
// the shuffles together.  Sums, maxima and scales are fp32; NaN propagates into
// the scale (max.NaN), so a row that holds one is NaN throughout, as its
// definition says.
#include "common.cuh"

#include <cuda_fp8.h>

namespace {

constexpr float kE4m3Max = 448.0f;
constexpr float kTiny = 1e-12f;  // floor of max |y|: a zero row gets a finite scale

struct NormArgs {
  const __nv_bfloat16* x;
  const __nv_bfloat16* r;  // nullable
  const __nv_bfloat16* w;  // nullable: no norm (y = x)
  void* y;                 // bf16, or e4m3 when scale is given
  float* scale;            // nullable
  __nv_bfloat16* h;        // given exactly when r is
  int64_t x_row, r_row, y_row, h_row;
  int64_t rows;
  int hidden;
  int group;  // threads of a row, a multiple of 32
  float eps;
};

B200_DEVICE float max_nan(float a, float b) {
  float d;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}

// 8 consecutive elements (VEC == 8, 16-byte aligned) or one
template <int VEC>
B200_DEVICE void load(const __nv_bfloat16* p, float (&v)[VEC]) {
  if constexpr (VEC == 8) {
    const uint4 u = *reinterpret_cast<const uint4*>(p);
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[2 * i] = b200::bf16_lo(w[i]);
      v[2 * i + 1] = b200::bf16_hi(w[i]);
    }
  } else {
    v[0] = __bfloat162float(*p);
  }
}

template <int VEC>
B200_DEVICE void store_bf16(__nv_bfloat16* p, const float (&v)[VEC]) {
  if constexpr (VEC == 8) {
    uint4 u;
    u.x = b200::pack_bf16x2(v[0], v[1]);
    u.y = b200::pack_bf16x2(v[2], v[3]);
    u.z = b200::pack_bf16x2(v[4], v[5]);
    u.w = b200::pack_bf16x2(v[6], v[7]);
    *reinterpret_cast<uint4*>(p) = u;
  } else {
    *p = __float2bfloat16_rn(v[0]);
  }
}

template <int VEC>
B200_DEVICE void store_e4m3(uint8_t* p, const float (&v)[VEC]) {
  if constexpr (VEC == 8) {
    uint32_t w[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(v[4 * i], v[4 * i + 1]),
                                                   __NV_SATFINITE, __NV_E4M3);
      const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(v[4 * i + 2], v[4 * i + 3]),
                                                   __NV_SATFINITE, __NV_E4M3);
      w[i] = lo | (hi << 16);
    }
    *reinterpret_cast<uint2*>(p) = make_uint2(w[0], w[1]);
  } else {
    *p = __nv_cvt_float_to_fp8(v[0], __NV_SATFINITE, __NV_E4M3);
  }
}

// sum and maximum over the `group` threads of a row; every thread of the block calls
B200_DEVICE void row_reduce(float& sum, float& top, int group, float2* part) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    sum += __shfl_xor_sync(0xffffffffu, sum, o);
    top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, o));
  }
  if (group == 32) return;
  const int warp = threadIdx.x >> 5, warps = group >> 5;
  if ((threadIdx.x & 31) == 0) part[warp] = make_float2(sum, top);
  __syncthreads();
  const int first = warp / warps * warps;
  float2 t = part[first];
  for (int i = 1; i < warps; ++i) {
    const float2 u = part[first + i];
    t.x += u.x;
    t.y = max_nan(t.y, u.y);
  }
  sum = t.x;
  top = t.y;
}

// HELD: the row fits the group's registers (NV vectors a thread); otherwise
// the row is read once for the statistics and again for the output.
template <int VEC, int NV, bool HELD>
__global__ void __launch_bounds__(1024) rms_norm_kernel(const NormArgs a) {
  b200::pdl_begin();
  __shared__ float2 part[32];
  const int64_t row = static_cast<int64_t>(blockIdx.x) * (blockDim.x / a.group) +
                      threadIdx.x / a.group;
  const int t = threadIdx.x % a.group;
  const bool live = row < a.rows;
  const __nv_bfloat16* x = a.x + row * a.x_row;
  const __nv_bfloat16* r = a.r != nullptr ? a.r + row * a.r_row : nullptr;
  const int step = a.group * VEC;
  const int span = HELD ? NV * step : (a.hidden + step - 1) / step * step;

  // elements e .. e + VEC - 1 of h (zero past the row's end)
  auto read_h = [&](int e, float (&v)[VEC]) {
    if (live && e < a.hidden) {
      load<VEC>(x + e, v);
      if (r != nullptr) {
        float u[VEC];
        load<VEC>(r + e, u);
#pragma unroll
        for (int i = 0; i < VEC; ++i) v[i] += u[i];
      }
    } else {
#pragma unroll
      for (int i = 0; i < VEC; ++i) v[i] = 0.0f;
    }
  };
  float sum = 0.0f, top = 0.0f;
  auto take = [&](int e, const float (&v)[VEC]) {
    float w[VEC];
    const bool norm = a.w != nullptr && e < a.hidden;
    if (norm) load<VEC>(a.w + e, w);
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      sum += v[i] * v[i];
      top = max_nan(top, fabsf(norm ? v[i] * w[i] : v[i]));
    }
  };

  float held[HELD ? NV : 1][VEC];
  if constexpr (HELD) {
#pragma unroll
    for (int j = 0; j < NV; ++j) read_h(t * VEC + j * step, held[j]);
#pragma unroll
    for (int j = 0; j < NV; ++j) take(t * VEC + j * step, held[j]);
  } else {
    for (int e = t * VEC; e < span; e += step) {
      read_h(e, held[0]);
      take(e, held[0]);
    }
  }
  row_reduce(sum, top, a.group, part);
  if (!live) return;

  float rstd = 1.0f, inv = 1.0f;
  if (a.w != nullptr) rstd = rsqrtf(sum / static_cast<float>(a.hidden) + a.eps);
  if (a.scale != nullptr) {
    const float most = max_nan(top * rstd, kTiny);
    if (t == 0) a.scale[row] = most / kE4m3Max;
    inv = kE4m3Max / most;
  }
  auto write = [&](int e, float (&v)[VEC]) {
    if (e >= a.hidden) return;
    if (a.h != nullptr) store_bf16<VEC>(a.h + row * a.h_row + e, v);
    if (a.w != nullptr) {
      float w[VEC];
      load<VEC>(a.w + e, w);
#pragma unroll
      for (int i = 0; i < VEC; ++i) v[i] = v[i] * w[i] * rstd;
    }
    if (a.scale != nullptr) {
#pragma unroll
      for (int i = 0; i < VEC; ++i) v[i] *= inv;
      store_e4m3<VEC>(static_cast<uint8_t*>(a.y) + row * a.y_row + e, v);
    } else {
      store_bf16<VEC>(static_cast<__nv_bfloat16*>(a.y) + row * a.y_row + e, v);
    }
  };
  if constexpr (HELD) {
#pragma unroll
    for (int j = 0; j < NV; ++j) write(t * VEC + j * step, held[j]);
  } else {
    for (int e = t * VEC; e < span; e += step) {
      read_h(e, held[0]);
      write(e, held[0]);
    }
  }
}

bool multiple8(int64_t s) { return (s & 7) == 0; }
bool aligned_to(const void* p, uintptr_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

}  // namespace

extern "C" int b200_rms_norm(const void* x, int64_t x_stride, const void* residual,
                             int64_t r_stride, const void* weight, void* y, int64_t y_stride,
                             float* scale, void* residual_out, int64_t h_stride, int64_t rows,
                             int hidden, float eps, void* stream) {
  if (rows < 0 || hidden <= 0 || rows > 0x7fffffff) return B200_ERR_INVALID_ARGUMENT;
  if (rows == 0) return B200_OK;
  if (!x || !y || (residual == nullptr) != (residual_out == nullptr))
    return B200_ERR_INVALID_ARGUMENT;
  if (weight == nullptr && (scale == nullptr || residual != nullptr))
    return B200_ERR_INVALID_ARGUMENT;  // without a norm only the 8-bit output has a use
  NormArgs a{};
  a.x = static_cast<const __nv_bfloat16*>(x);
  a.r = static_cast<const __nv_bfloat16*>(residual);
  a.w = static_cast<const __nv_bfloat16*>(weight);
  a.y = y;
  a.scale = scale;
  a.h = static_cast<__nv_bfloat16*>(residual_out);
  a.x_row = x_stride;
  a.r_row = r_stride;
  a.y_row = y_stride;
  a.h_row = h_stride;
  a.rows = rows;
  a.hidden = hidden;
  a.eps = eps;
  const bool vec = hidden % 8 == 0 && multiple8(x_stride) && multiple8(y_stride) &&
                   aligned_to(x, 16) && aligned_to(y, scale != nullptr ? 8 : 16) &&
                   (weight == nullptr || aligned_to(weight, 16)) &&
                   (residual == nullptr ||
                    (multiple8(r_stride) && multiple8(h_stride) && aligned_to(residual, 16) &&
                     aligned_to(residual_out, 16)));
  const int per = vec ? 32 : 8;  // elements a thread holds: 4 vectors, or 8 single elements
  int group = (hidden + per - 1) / per;
  group = (group + 31) / 32 * 32;
  const bool held = group <= 1024;
  if (!held) group = 1024;
  a.group = group;
  const int rows_a_block = group >= 256 ? 1 : 256 / group;
  const int64_t blocks = (rows + rows_a_block - 1) / rows_a_block;
  const dim3 grid(static_cast<unsigned>(blocks)), block(group * rows_a_block);
  cudaStream_t cs = static_cast<cudaStream_t>(stream);
  cudaError_t e;
  if (vec && held) e = b200host::launch_pdl(rms_norm_kernel<8, 4, true>, grid, block, 0, cs, a);
  else if (vec) e = b200host::launch_pdl(rms_norm_kernel<8, 1, false>, grid, block, 0, cs, a);
  else if (held) e = b200host::launch_pdl(rms_norm_kernel<1, 8, true>, grid, block, 0, cs, a);
  else e = b200host::launch_pdl(rms_norm_kernel<1, 1, false>, grid, block, 0, cs, a);
  return b200host::status_from_cuda(e);
}
