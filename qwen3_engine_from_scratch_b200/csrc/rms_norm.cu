// RMS norm with the residual's addition, output in bf16 or in 8 bits (e4m3)
// with a scale a row, and the same 8-bit output without a norm:
//   h = x + r                        fp32 (returned rounded to bf16)
//   y = h / sqrt(mean(h^2) + eps) * w      fp32, from the unrounded h
//   s = max(max |y|, 1e-12) / 448    fp32, q = e4m3(y / s)
// The 8-bit form returns (q, s): q s is y to e4m3's 3 mantissa bits, and s is
// the row factor that the matrix product applies in its epilogue.
//
// Bound by memory: x and r are read once, h and y (or q, s) written once, so a
// row stays on chip between the reduction and the output.  Three forms:
//   held    a group of threads holds the row in registers, up to four 8-element
//           vectors each (8 single elements where a row is not aligned);
//   stream  many wide aligned rows: persistent CTAs with a ring of rows in
//           shared memory filled by bulk copies;
//   wide    rows beyond 16,384 elements (8,192 unaligned) are read again for the
//           output.
// One reduction a row serves both statistics: y is h w times a positive row
// factor, so max |y| = rstd max |h w|, and (sum h^2, max |h w|) travel through
// the shuffles together.  Sums, maxima and scales are fp32; NaN propagates into
// the scale (max.NaN), so a row that holds one is NaN throughout, as its
// definition says.
// Measured: 8192 x 4096 with residual to e4m3 40.5 us (5.8 TB/s, 0.88 of the copy
// rate), to bf16 44 us (0.93); 8192 x 12288 to e4m3 without a norm 49.2 us (0.93); one
// row of 1024 1.5 us in a graph, its latency.
#include "common.cuh"
#include "words.cuh"

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
  int group;   // threads of a row, a multiple of 32
  int stages;  // rows in flight of a streaming CTA
  int32_t* dev_status;
  float eps;
};

B200_DEVICE float max_nan(float a, float b) {
  float d;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}

// 8 consecutive elements (VEC == 8, 16-byte aligned) or one, as they lie in memory
template <int VEC>
struct Word {
  uint4 w = make_uint4(0, 0, 0, 0);
};
template <>
struct Word<1> {
  __nv_bfloat16 w = __nv_bfloat16(__nv_bfloat16_raw{0});
};

template <int VEC>
B200_DEVICE Word<VEC> read(const __nv_bfloat16* p) {
  Word<VEC> r;
  if constexpr (VEC == 8) r.w = *reinterpret_cast<const uint4*>(p);
  else r.w = *p;
  return r;
}

template <int VEC>
B200_DEVICE void unpack(const Word<VEC>& u, float (&v)[VEC]) {
  if constexpr (VEC == 8) {
    const uint32_t w[4] = {u.w.x, u.w.y, u.w.z, u.w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[2 * i] = b200::bf16_lo(w[i]);
      v[2 * i + 1] = b200::bf16_hi(w[i]);
    }
  } else {
    v[0] = __bfloat162float(u.w);
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

// sum and (TOP) maximum over the `group` threads of a row; every thread of the block calls
template <bool TOP>
B200_DEVICE void row_reduce(float& sum, float& top, int group, float2* part) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (TOP) top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, o));
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
    if (TOP) t.y = max_nan(t.y, u.y);
  }
  sum = t.x;
  top = t.y;
}

// max |y| -> the row's scale; returns 1 / scale
B200_DEVICE float put_scale(const NormArgs& a, int64_t row, float most, bool writer) {
  most = max_nan(most, kTiny);
  if (writer) a.scale[row] = most / kE4m3Max;
  return kE4m3Max / most;
}

template <int VEC, bool FP8>
B200_DEVICE void put_y(const NormArgs& a, int64_t row, int e, const float (&v)[VEC]) {
  if constexpr (FP8)
    store_e4m3<VEC>(static_cast<uint8_t*>(a.y) + row * a.y_row + e, v);
  else
    store_bf16<VEC>(static_cast<__nv_bfloat16*>(a.y) + row * a.y_row + e, v);
}

// A row in the registers of its group, NV vectors a thread: fp32 h w behind a
// norm (h has left by then), the row's own bf16 words without one (half the
// registers, so twice the rows in flight: 8192 x 12288 in 103 us with fp32).
template <int VEC, int NV, bool NORM, bool FP8>
__global__ void __launch_bounds__(VEC == 8 ? 512 : 1024) rms_norm_kernel(const NormArgs a) {
  b200::pdl_begin();
  __shared__ float2 part[32];
  const int64_t row = static_cast<int64_t>(blockIdx.x) * (blockDim.x / a.group) +
                      threadIdx.x / a.group;
  const int t = threadIdx.x % a.group;
  const bool live = row < a.rows;
  const int step = a.group * VEC;
  const __nv_bfloat16* x = a.x + row * a.x_row;

  float sum = 0.0f, top = 0.0f;
  if constexpr (NORM) {
    const __nv_bfloat16* r = a.r != nullptr ? a.r + row * a.r_row : nullptr;
    Word<VEC> xw[NV], rw[NV], ww[NV];
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int e = t * VEC + j * step;
      const bool in = live && e < a.hidden;
      xw[j] = in ? read<VEC>(x + e) : Word<VEC>{};
      rw[j] = in && r != nullptr ? read<VEC>(r + e) : Word<VEC>{};
      ww[j] = in ? read<VEC>(a.w + e) : Word<VEC>{};
    }
    float v[NV][VEC];
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int e = t * VEC + j * step;
      unpack<VEC>(xw[j], v[j]);
      if (r != nullptr) {
        float u[VEC];
        unpack<VEC>(rw[j], u);
#pragma unroll
        for (int i = 0; i < VEC; ++i) v[j][i] += u[i];
        if (live && e < a.hidden) store_bf16<VEC>(a.h + row * a.h_row + e, v[j]);
      }
      float w[VEC];
      unpack<VEC>(ww[j], w);
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        sum += v[j][i] * v[j][i];
        v[j][i] *= w[i];
        if (FP8) top = max_nan(top, fabsf(v[j][i]));
      }
    }
    row_reduce<FP8>(sum, top, a.group, part);
    if (!live) return;
    float factor = rsqrtf(sum / static_cast<float>(a.hidden) + a.eps);
    float inv = 1.0f;
    if (FP8) inv = put_scale(a, row, top * factor, t == 0);
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int e = t * VEC + j * step;
      if (e >= a.hidden) break;
#pragma unroll
      for (int i = 0; i < VEC; ++i) v[j][i] = FP8 ? v[j][i] * factor * inv : v[j][i] * factor;
      put_y<VEC, FP8>(a, row, e, v[j]);
    }
  } else {
    Word<VEC> xw[NV];
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int e = t * VEC + j * step;
      xw[j] = live && e < a.hidden ? read<VEC>(x + e) : Word<VEC>{};
    }
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      float v[VEC];
      unpack<VEC>(xw[j], v);
#pragma unroll
      for (int i = 0; i < VEC; ++i) top = max_nan(top, fabsf(v[i]));
    }
    row_reduce<true>(sum, top, a.group, part);
    if (!live) return;
    const float inv = put_scale(a, row, top, t == 0);
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int e = t * VEC + j * step;
      if (e >= a.hidden) break;
      float v[VEC];
      unpack<VEC>(xw[j], v);
#pragma unroll
      for (int i = 0; i < VEC; ++i) v[i] *= inv;
      put_y<VEC, FP8>(a, row, e, v);
    }
  }
}

constexpr int kMaxStages = 8;
constexpr int kStreamSmem = 216 * 1024;             // of an SM, for its CTAs' stages
constexpr uint64_t kWaitLimitNs = 1000000000ull;   // 1 s a stage

B200_DEVICE void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
          dst),
      "l"(reinterpret_cast<uint64_t>(src)), "r"(bytes), "r"(bar)
      : "memory");
}

// Many aligned rows: persistent CTAs, each with a ring of whole rows in shared
// memory that bulk copies fill ahead, so the loads never wait for a reduction
// or an output.  One block barrier a row: it joins the partial sums, and after
// it the row's stage is free for the next copy.  The weight stays in registers.
template <int NV, bool NORM, bool FP8>
__global__ void __launch_bounds__(512) rms_norm_stream_kernel(const NormArgs a) {
  extern __shared__ __align__(128) uint8_t ring[];
  __shared__ __align__(8) uint64_t full[kMaxStages];
  __shared__ float2 part[2][16];
  const int t = threadIdx.x, warps = blockDim.x >> 5;
  const uint32_t row_bytes = static_cast<uint32_t>(a.hidden) * 2;
  const uint32_t stage_bytes = a.r != nullptr ? 2 * row_bytes : row_bytes;
  const int step = blockDim.x * 8;
  // a pipeline gave up before this launch: no new work until the host clears the
  // status.  Thread 0 reads it, so that the block agrees, and before the wait for the
  // previous kernel, off the launch's path; once more after it where it is set, since
  // that kernel may be the one that clears it.
  __shared__ bool aborted;
  if (t == 0) {
    for (int s = 0; s < a.stages; ++s) b200::mbar_init(b200::smem_u32(&full[s]), 1);
    b200::fence_mbar_init();
    aborted = b200::timeout_on_record(a.dev_status);
  }
  __syncthreads();
  b200::pdl_begin();
  if (aborted) {
    __syncthreads();
    if (t == 0) aborted = b200::timeout_on_record(a.dev_status);
    __syncthreads();
    if (aborted) return;
  }
  auto fetch = [&](int64_t row, int s) {
    const uint32_t bar = b200::smem_u32(&full[s]);
    const uint32_t dst = b200::smem_u32(ring) + s * stage_bytes;
    b200::mbar_arrive_expect_tx(bar, stage_bytes);
    bulk_load(dst, a.x + row * a.x_row, row_bytes, bar);
    if (a.r != nullptr) bulk_load(dst + row_bytes, a.r + row * a.r_row, row_bytes, bar);
  };
  int issued = 0, taken = 0;  // copies (of thread 0), rows done; copy n is in stage n % stages
  if (t == 0) {
    for (int64_t row = blockIdx.x; issued < a.stages && row < a.rows; row += gridDim.x)
      fetch(row, issued++);
  }
  Word<8> ww[NORM ? NV : 1];
  if constexpr (NORM) {
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int e = t * 8 + j * step;
      if (e < a.hidden) ww[j] = read<8>(a.w + e);
    }
  }

  int s = 0;
  uint32_t phase = 0;
  int odd = 0;
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x, odd ^= 1, ++taken) {
    bool ok = b200::mbar_wait_abortable(b200::smem_u32(&full[s]), phase, a.dev_status, kWaitLimitNs);
    const __nv_bfloat16* xr = reinterpret_cast<const __nv_bfloat16*>(ring + s * stage_bytes);
    float sum = 0.0f, top = 0.0f;
    Word<8> xw[NV];
    float v[NORM ? NV : 1][8];
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int e = t * 8 + j * step;
      xw[j] = e < a.hidden ? read<8>(xr + e) : Word<8>{};
      if constexpr (NORM) {
        unpack<8>(xw[j], v[j]);
        if (a.r != nullptr && e < a.hidden) {
          float u[8];
          unpack<8>(read<8>(xr + a.hidden + e), u);
#pragma unroll
          for (int i = 0; i < 8; ++i) v[j][i] += u[i];
          if (ok) store_bf16<8>(a.h + row * a.h_row + e, v[j]);
        }
        float w[8];
        unpack<8>(ww[j], w);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          sum += v[j][i] * v[j][i];
          v[j][i] *= w[i];
          if (FP8) top = max_nan(top, fabsf(v[j][i]));
        }
      } else {
        float u[8];
        unpack<8>(xw[j], u);
#pragma unroll
        for (int i = 0; i < 8; ++i) top = max_nan(top, fabsf(u[i]));
      }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      if (NORM) sum += __shfl_xor_sync(0xffffffffu, sum, o);
      if (FP8) top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, o));
    }
    if ((t & 31) == 0) part[odd][t >> 5] = make_float2(sum, top);
    if (!__syncthreads_and(ok)) {
      if (t == 0) b200::flag_error(a.dev_status, B200_DEV_TIMEOUT);
      break;
    }
    if (t == 0) {
      const int64_t next = row + static_cast<int64_t>(a.stages) * gridDim.x;
      if (next < a.rows) {
        fetch(next, s);
        ++issued;
      }
    }
    float2 all = part[odd][0];
    for (int i = 1; i < warps; ++i) {
      const float2 p = part[odd][i];
      all.x += p.x;
      all.y = max_nan(all.y, p.y);
    }
    const float factor =
        NORM ? rsqrtf(all.x / static_cast<float>(a.hidden) + a.eps) : 1.0f;
    float inv = 1.0f;
    if (FP8) inv = put_scale(a, row, all.y * factor, t == 0);
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int e = t * 8 + j * step;
      if (e >= a.hidden) break;
      float y[8];
      if constexpr (NORM) {
#pragma unroll
        for (int i = 0; i < 8; ++i) y[i] = FP8 ? v[j][i] * factor * inv : v[j][i] * factor;
      } else {
        unpack<8>(xw[j], y);
#pragma unroll
        for (int i = 0; i < 8; ++i) y[i] *= inv;
      }
      put_y<8, FP8>(a, row, e, y);
    }
    if (++s == a.stages) {
      s = 0;
      phase ^= 1;
    }
  }
  // after a give-up the copies in flight land before the shared memory goes away
  // (otherwise every copy was taken and there is none)
  if (t == 0) {
    for (; taken < issued; ++taken)
      b200::mbar_wait_abortable(b200::smem_u32(&full[taken % a.stages]), (taken / a.stages) & 1,
                                nullptr, kWaitLimitNs / 10);
  }
}

// Rows wider than a block's registers: read for the statistics and again for
// the output.  (h leaves in the second pass only: it may be x or the residual.)
template <int VEC, bool NORM, bool FP8>
__global__ void __launch_bounds__(1024) rms_norm_wide_kernel(const NormArgs a) {
  b200::pdl_begin();
  __shared__ float2 part[32];
  const int64_t row = blockIdx.x;
  const __nv_bfloat16* x = a.x + row * a.x_row;
  const __nv_bfloat16* r = a.r != nullptr ? a.r + row * a.r_row : nullptr;
  auto read_h = [&](int e, float (&v)[VEC]) {
    unpack<VEC>(read<VEC>(x + e), v);
    if (r != nullptr) {
      float u[VEC];
      unpack<VEC>(read<VEC>(r + e), u);
#pragma unroll
      for (int i = 0; i < VEC; ++i) v[i] += u[i];
    }
  };
  auto weigh = [&](int e, float (&v)[VEC]) {
    float w[VEC];
    unpack<VEC>(read<VEC>(a.w + e), w);
#pragma unroll
    for (int i = 0; i < VEC; ++i) v[i] *= w[i];
  };
  float sum = 0.0f, top = 0.0f;
  for (int e = threadIdx.x * VEC; e < a.hidden; e += blockDim.x * VEC) {
    float v[VEC];
    read_h(e, v);
    if (NORM) {
#pragma unroll
      for (int i = 0; i < VEC; ++i) sum += v[i] * v[i];
      weigh(e, v);
    }
    if (FP8) {
#pragma unroll
      for (int i = 0; i < VEC; ++i) top = max_nan(top, fabsf(v[i]));
    }
  }
  row_reduce<FP8>(sum, top, blockDim.x, part);
  float factor = NORM ? rsqrtf(sum / static_cast<float>(a.hidden) + a.eps) : 1.0f;
  float inv = 1.0f;
  if (FP8) inv = put_scale(a, row, top * factor, threadIdx.x == 0);
  for (int e = threadIdx.x * VEC; e < a.hidden; e += blockDim.x * VEC) {
    float v[VEC];
    read_h(e, v);
    if (r != nullptr) store_bf16<VEC>(a.h + row * a.h_row + e, v);
    if (NORM) weigh(e, v);
#pragma unroll
    for (int i = 0; i < VEC; ++i) v[i] = FP8 ? v[i] * factor * inv : v[i] * factor;
    put_y<VEC, FP8>(a, row, e, v);
  }
}

template <int NV, bool NORM, bool FP8>
cudaError_t launch_stream(const NormArgs& a, unsigned grid, int threads, int smem,
                          cudaStream_t cs) {
  const cudaError_t e =
      cudaFuncSetAttribute(rms_norm_stream_kernel<NV, NORM, FP8>,
                           cudaFuncAttributeMaxDynamicSharedMemorySize, kStreamSmem);
  if (e != cudaSuccess) return e;
  return b200host::launch_pdl(rms_norm_stream_kernel<NV, NORM, FP8>, dim3(grid), dim3(threads),
                              smem, cs, a);
}

template <int NV>
cudaError_t launch_stream(const NormArgs& a, unsigned grid, int threads, int smem,
                          cudaStream_t cs) {
  if (a.w == nullptr) return launch_stream<NV, false, true>(a, grid, threads, smem, cs);
  if (a.scale != nullptr) return launch_stream<NV, true, true>(a, grid, threads, smem, cs);
  return launch_stream<NV, true, false>(a, grid, threads, smem, cs);
}

template <int VEC, int NV>
cudaError_t launch_held(const NormArgs& a, dim3 grid, dim3 block, cudaStream_t cs) {
  if (a.w == nullptr)
    return b200host::launch_pdl(rms_norm_kernel<VEC, NV, false, true>, grid, block, 0, cs, a);
  if (a.scale != nullptr)
    return b200host::launch_pdl(rms_norm_kernel<VEC, NV, true, true>, grid, block, 0, cs, a);
  return b200host::launch_pdl(rms_norm_kernel<VEC, NV, true, false>, grid, block, 0, cs, a);
}

template <int VEC>
cudaError_t launch_wide(const NormArgs& a, dim3 grid, dim3 block, cudaStream_t cs) {
  if (a.w == nullptr)
    return b200host::launch_pdl(rms_norm_wide_kernel<VEC, false, true>, grid, block, 0, cs, a);
  if (a.scale != nullptr)
    return b200host::launch_pdl(rms_norm_wide_kernel<VEC, true, true>, grid, block, 0, cs, a);
  return b200host::launch_pdl(rms_norm_wide_kernel<VEC, true, false>, grid, block, 0, cs, a);
}

// a thread's element index steps past the row's end by a block's vectors at most
constexpr int kMaxHidden = 0x7fffffff - 1024 * 8;

bool multiple8(int64_t s) { return (s & 7) == 0; }
bool aligned_to(const void* p, uintptr_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

}  // namespace

extern "C" int b200_rms_norm(const void* x, int64_t x_stride, const void* residual,
                             int64_t r_stride, const void* weight, void* y, int64_t y_stride,
                             float* scale, void* residual_out, int64_t h_stride, int64_t rows,
                             int hidden, float eps, int32_t* dev_status,
                             void* stream) {
  if (rows < 0 || hidden <= 0 || hidden > kMaxHidden || rows > 0x7fffffff)
    return B200_ERR_INVALID_ARGUMENT;
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
  a.dev_status = dev_status;
  const bool vec = hidden % 8 == 0 && multiple8(x_stride) && multiple8(y_stride) &&
                   aligned_to(x, 16) && aligned_to(y, scale != nullptr ? 8 : 16) &&
                   (weight == nullptr || aligned_to(weight, 16)) &&
                   (residual == nullptr ||
                    (multiple8(r_stride) && multiple8(h_stride) && aligned_to(residual, 16) &&
                     aligned_to(residual_out, 16)));
  // A thread holds 4 vectors (or 8 single elements); few rows of up to 4096 elements
  // spread over more threads, one vector each, since their latency is all that counts.
  // Beyond that 4 vectors are as fast or faster: in a graph, 1 x 8192 with residual to
  // bf16 takes 2.4 us (3.0 with one vector and 1024 threads), 64 x 5120 to e4m3 2.35
  // (2.44); 1 x 4104 to bf16 2.1 (2.0).
  cudaStream_t cs = static_cast<cudaStream_t>(stream);
  const int sms = b200host::sm_count(b200host::current_device());
  if (sms <= 0) return B200_ERR_CUDA;
  const bool few = vec && hidden <= 4096 && rows <= sms;
  const int per = few ? 8 : vec ? 32 : 8;
  // Wide rows in numbers stream.  The CTAs an SM takes were swept from 1 to 8 for
  // rows of 1024 to 16384 elements: 8192 x 12288 to e4m3 without a norm takes
  // 48.0 us with 6 (66 held), 2000 x 12288 with norm and residual 29.8 with 2
  // (37.6 held), 8192 x 4096 39.6 with 8 (43.7 held).  Below the limits the held
  // form is as fast or faster (8192 x 1024: 11.7 us, streamed 14.1).
  const int64_t stage_bytes = (residual != nullptr ? int64_t{4} : 2) * hidden;
  const int wide_from = weight != nullptr ? 2048 : 4096;
  if (vec && hidden >= wide_from && hidden <= 16384 &&
      rows >= static_cast<int64_t>(sms) * (weight != nullptr ? 2 : 4)) {
    int ctas = weight != nullptr ? (hidden <= 4096 ? 8 : hidden <= 6144 ? 4 : 2)
                                 : (hidden <= 4096 ? 8 : hidden <= 12288 ? 6 : 4);
    while (kStreamSmem / ctas < stage_bytes) ctas /= 2;
    a.stages = static_cast<int>(kStreamSmem / ctas / stage_bytes);
    if (a.stages > kMaxStages) a.stages = kMaxStages;
    const int64_t most = static_cast<int64_t>(sms) * ctas;
    const int threads = ((hidden + 31) / 32 + 31) / 32 * 32;
    return b200host::status_from_cuda(launch_stream<4>(
        a, static_cast<unsigned>(rows < most ? rows : most), threads,
        static_cast<int>(a.stages * stage_bytes), cs));
  }
  a.group = ((hidden + per - 1) / per + 31) / 32 * 32;
  cudaError_t e;
  if (a.group > (vec ? 512 : 1024)) {
    a.group = 1024;
    const dim3 grid(static_cast<unsigned>(rows)), block(1024);
    e = vec ? launch_wide<8>(a, grid, block, cs) : launch_wide<1>(a, grid, block, cs);
  } else {
    const int rows_a_block = few || a.group >= 256 ? 1 : 256 / a.group;
    const dim3 grid(static_cast<unsigned>((rows + rows_a_block - 1) / rows_a_block));
    const dim3 block(a.group * rows_a_block);
    e = few ? launch_held<8, 1>(a, grid, block, cs)
            : vec ? launch_held<8, 4>(a, grid, block, cs) : launch_held<1, 8>(a, grid, block, cs);
  }
  return b200host::status_from_cuda(e);
}

extern "C" int b200_rms_norm_words(const int64_t* words) {
  if (!words) return B200_ERR_INVALID_ARGUMENT;
  b200host::Words w{words};
  const int hidden = w.integer(11);
  if (!w.fit) return B200_ERR_INVALID_ARGUMENT;
  return b200_rms_norm(w.pointer(0), w.wide(1), w.pointer(2), w.wide(3), w.pointer(4), w.pointer(5),
                       w.wide(6), w.pointer<float>(7), w.pointer(8), w.wide(9), w.wide(10), hidden,
                       w.real(12), w.pointer<int32_t>(13), w.pointer(14));
}
