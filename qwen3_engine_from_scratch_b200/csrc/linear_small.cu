// The matrix product of linear.cu for a few tokens (a decode step): the weight is
// read once and everything else is small, so the kernel is bound by memory and,
// at these sizes, by its own latency.  It therefore has no tensor maps, no TMEM
// and no pipeline to fill: every thread loads its 16-byte pieces of W and X
// straight into the registers of mma.sync, whose rate is far from the limit.
//   m16n8k16 (bf16) or m16n8k32 (e4m3): 16 weight rows x 8 tokens; a thread's four
// words of a row's 16 bytes are the k pairs (quads) of two instructions.  Which
// k an instruction sees at which place does not matter as long as W and X agree.
// The 8 or 16 warps of a block split K of the block's rows and add their sums in warp
// order through shared memory.  Gated: rows 0-7 of a tile are gate rows and rows
// 8-15 the up rows of the same outputs.
// Measured: 8 x 1024 x 4096 3.4 us in a graph, of which 1.3 are the weight's bytes;
// 8 rows of 151,936 logits over 1024 inputs 53.6 us (5.9 TB/s, 0.89 of the copy rate).
#include "linear.cuh"

namespace {

using namespace b200;

constexpr int kRows = 16;  // weight rows of a block
constexpr int kStep = 64;  // bytes of K a warp takes of every row in a step

struct SmallArgs {
  LinearArgs e;
  const uint8_t* x;
  const uint8_t* w;
  int64_t x_row, w_row;  // bytes
  int k_bytes;
};

template <bool FP8>
B200_DEVICE void mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                     uint32_t b1) {
  if constexpr (FP8) {
    asm volatile(
        "mma.sync.aligned.m16n8k32.row.col.f32.e4m3.e4m3.f32 {%0, %1, %2, %3}, "
        "{%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  } else {
    mma_bf16_16816(d, a0, a1, a2, a3, b0, b1);
  }
}

// 16 bytes of a row on their way
template <bool ALIGNED>
struct Piece {
  uint4 w;
};
template <>
struct Piece<false> {
  Unaligned16 w;
};
B200_DEVICE uint4 value(const Piece<true>& p) { return p.w; }
B200_DEVICE uint4 value(const Piece<false>& p) { return shifted(p.w); }

// 16 bytes of a row from byte `at` on, zero past its end
template <bool FP8, bool ALIGNED>
B200_DEVICE Piece<ALIGNED> piece(const uint8_t* row, int at, int end) {
  Piece<ALIGNED> p;
  if (at + 16 <= end) {
    if constexpr (ALIGNED) p.w = *reinterpret_cast<const uint4*>(row + at);
    else p.w = load_unaligned16(row + at);
    return p;
  }
  uint32_t w[4] = {0, 0, 0, 0};
  if (at < end) {
#pragma unroll
    for (int i = 0; i < 16; i += FP8 ? 1 : 2)
      if (at + i < end) {
        const uint32_t v = FP8 ? row[at + i] : *reinterpret_cast<const uint16_t*>(row + at + i);
        w[i / 4] |= v << (8 * (i % 4));
      }
  }
  const uint4 u = make_uint4(w[0], w[1], w[2], w[3]);
  if constexpr (ALIGNED) p.w = u;
  else p.w = Unaligned16{u, u, 0};
  return p;
}

// TT token tiles of 8; a warp reads AHEAD steps before it multiplies the first
template <int TT, int AHEAD, int WARPS, bool FP8, bool ALIGNED>
__global__ void __launch_bounds__(WARPS * 32) linear_small_kernel(const SmallArgs a) {
  constexpr int kWarps = WARPS, kThreads = WARPS * 32;
  __shared__ float sums[kWarps][kRows][TT * 8 + 1];
  const LinearArgs& e = a.e;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, t = lane & 3;
  const int tile_n = e.gated ? kRows / 2 : kRows;
  const int n0 = blockIdx.x * tile_n;

  // row 0 .. 15 of the block (n past the end repeats the last)
  auto weight_row = [&](int row) {
    if (!e.gated) return a.w + min(n0 + row, e.n - 1) * a.w_row;
    const int64_t n = min(n0 + (row & 7), e.n - 1);
    return a.w + (row < 8 ? n : e.n + n) * a.w_row;
  };
  const uint8_t* w[2] = {weight_row(g), weight_row(g + 8)};
  const uint8_t* x[TT];
#pragma unroll
  for (int i = 0; i < TT; ++i) x[i] = a.x + min(i * 8 + g, e.m - 1) * a.x_row;

  // The block's first loads start towards L2 while the previous kernel drains.
  // (A prefetch returns no data: what that kernel still writes to W is read after
  // the wait, from L2 as always.)
  {
    const int at = (threadIdx.x % (kThreads / kRows)) * 128;
    if (at < a.k_bytes) prefetch_l2(weight_row(threadIdx.x / (kThreads / kRows)) + at);
  }
  pdl_begin();
  float d[TT][4] = {};
  for (int k0 = warp * kStep; k0 < a.k_bytes; k0 += kWarps * kStep * AHEAD) {
    Piece<ALIGNED> wv[AHEAD][2], xv[AHEAD][TT];
#pragma unroll
    for (int s = 0; s < AHEAD; ++s) {
      const int at = k0 + s * kWarps * kStep + t * 16;
      wv[s][0] = piece<FP8, ALIGNED>(w[0], at, a.k_bytes);
      wv[s][1] = piece<FP8, ALIGNED>(w[1], at, a.k_bytes);
#pragma unroll
      for (int i = 0; i < TT; ++i) xv[s][i] = piece<FP8, ALIGNED>(x[i], at, a.k_bytes);
    }
#pragma unroll
    for (int s = 0; s < AHEAD; ++s) {
      const uint4 p = value(wv[s][0]), q = value(wv[s][1]);
#pragma unroll
      for (int i = 0; i < TT; ++i) {
        const uint4 v = value(xv[s][i]);
        mma<FP8>(d[i], p.x, q.x, p.y, q.y, v.x, v.y);
        mma<FP8>(d[i], p.z, q.z, p.w, q.w, v.z, v.w);
      }
    }
  }
#pragma unroll
  for (int i = 0; i < TT; ++i) {
    sums[warp][g][i * 8 + 2 * t] = d[i][0];
    sums[warp][g][i * 8 + 2 * t + 1] = d[i][1];
    sums[warp][g + 8][i * 8 + 2 * t] = d[i][2];
    sums[warp][g + 8][i * 8 + 2 * t + 1] = d[i][3];
  }
  __syncthreads();

  for (int at = threadIdx.x; at < tile_n * e.m; at += kThreads) {
    const int token = at / tile_n, col = at - token * tile_n;
    const int n = n0 + col;
    if (n >= e.n) continue;
    auto total = [&](int r, int w_row) {
      float v = sums[0][r][token];
#pragma unroll
      for (int i = 1; i < kWarps; ++i) v += sums[i][r][token];
      if (e.w_scale != nullptr) v *= e.w_scale[w_row] * e.x_scale[token];
      if (e.bias != nullptr) v += __bfloat162float(e.bias[w_row]);
      return v;
    };
    float v[1] = {total(col, n)};
    activate(v, e.act);
    if (e.gated) v[0] *= total(col + 8, e.n + n);
    if (e.residual != nullptr) v[0] += __bfloat162float(e.residual[token * e.r_row + n]);
    e.out[token * e.o_row + n] = __float2bfloat16_rn(v[0]);
  }
}

template <int TT, int AHEAD, int WARPS, bool ALIGNED>
cudaError_t launch(const SmallArgs& a, bool fp8, unsigned blocks, cudaStream_t stream) {
  return b200host::launch_pdl(fp8 ? linear_small_kernel<TT, AHEAD, WARPS, true, ALIGNED>
                                  : linear_small_kernel<TT, AHEAD, WARPS, false, ALIGNED>,
                              dim3(blocks), dim3(WARPS * 32), 0, stream, a);
}

}  // namespace

namespace b200host {

// Up to 8 tokens always; 9 to 16, whose X costs as many loads as W, where W is
// small enough for latency to count: 16 x 1024 x 4096 takes 3.6 us (6.8 on the
// tcgen05 tiles), 16 x 12288 x 4096 26 (22.5).
bool linear_is_small(const b200::LinearArgs& e, int k, bool fp8) {
  if (e.m <= 8) return true;
  const int64_t bytes = static_cast<int64_t>(e.n) * (e.gated ? 2 : 1) * k * (fp8 ? 1 : 2);
  return e.m <= 16 && bytes <= (20 << 20);
}

cudaError_t linear_small(const b200::LinearArgs& e, const void* x, int64_t x_stride, const void* w,
                         int64_t w_stride, int k, bool fp8, int sms, cudaStream_t stream) {
  SmallArgs a{};
  const int size = fp8 ? 1 : 2;
  a.e = e;
  a.x = static_cast<const uint8_t*>(x);
  a.w = static_cast<const uint8_t*>(w);
  a.x_row = x_stride * size;
  a.w_row = w_stride * size;
  a.k_bytes = k * size;
  const int tile_n = e.gated ? kRows / 2 : kRows;
  const unsigned blocks = static_cast<unsigned>((e.n + tile_n - 1) / tile_n);
  const bool aligned = aligned16(x) && aligned16(w) && a.x_row % 16 == 0 && a.w_row % 16 == 0;
  // 16 warps a block where there is about one block an SM, or less, and K feeds
  // them: 8 x 4096 x 2048 6.3 -> 5.5 us, 1 x 2048 x 1024 3.2 -> 2.5; with two blocks an
  // SM 8 warps are faster (8 x 4096 x 4096 8.5, 10.3 with 16).
  const bool wide = blocks <= static_cast<unsigned>(sms) && a.k_bytes >= 8 * 8 * kStep;
  if (!aligned)  // at most 8 tokens: b200_linear_unaligned takes no more
    return wide ? launch<1, 2, 16, false>(a, fp8, blocks, stream)
                : launch<1, 2, 8, false>(a, fp8, blocks, stream);
  if (e.m > 8) return launch<2, 4, 8, true>(a, fp8, blocks, stream);
  if (wide) return launch<1, 4, 16, true>(a, fp8, blocks, stream);
  // Eight steps ahead with up to two blocks an SM: 8 x 12288 x 4096 23.3 -> 20.7; with
  // more the registers cost more (8 x 4096 x 6144 10.7 -> 14.4).
  if (blocks <= 2u * sms && a.k_bytes >= 8 * 8 * kStep)
    return launch<1, 8, 8, true>(a, fp8, blocks, stream);
  return launch<1, 4, 8, true>(a, fp8, blocks, stream);
}

}  // namespace b200host
