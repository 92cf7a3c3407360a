// Rotary positions: every pair (a, b) of a head's first rotary_dim elements is
// turned by the angle position * f_i and scaled by the plan's gain,
//   a' = gain (a cos - b sin),  b' = gain (b cos + a sin),
// pairs (i, i + rotary_dim / 2) in the half layout, (2i, 2i + 1) in the
// interleaved one; the rest of the head is copied.
//
// Angles: the plan holds f_i / 2 pi as a 64-bit binary fraction of a turn, so
// position * f_i modulo one turn is one 64-bit integer product, at any position
// (negative ones included).  Its top 32 bits, rounded to fp32 (2^-26 turns near half a
// turn), go through sincospi.  The fractions come from float64 frequencies and are off
// by up to 2^-54 turns a position, less than that rounding up to position 2^28.  A
// product in fp32 would lose position * 2^-24 radians: 0.008 at position 131,072.
//
// Bound by memory for prefills: q and k are read and written once.  A block
// takes a few tokens: it computes their sines and cosines once into shared
// memory, then its threads (16 elements of a head each: 8 pairs, or 16 copied
// elements; neighbours in a head, then in heads) walk over the tokens' heads.
#include "common.cuh"
#include "words.cuh"

namespace {

struct RotaryArgs {
  const __nv_bfloat16* in[2];   // q, k
  __nv_bfloat16* out[2];
  int64_t in_b[2], in_h[2], in_s[2], out_b[2], out_h[2], out_s[2];
  const void* positions;
  int64_t pos_b, pos_s;
  int pos64;
  const uint64_t* turns;        // rotary_dim / 2 fractions of a turn a position
  float gain;
  int heads_q, heads;           // q heads, q + k heads
  int seq;                      // tokens of a sequence
  int dim, rotary_dim;
  int slots;                    // slots of a head: 16 elements, or one pair / element
  int slot_threads;             // threads of a head (a divisor of the block with the next two)
  int groups;                   // heads at work at a time
  int block_tokens;
  int interleaved;
  int64_t tokens;
};

B200_DEVICE void angle(const uint64_t* turns, int i, int64_t position, float gain, float& c,
                       float& s) {
  const uint64_t phase = static_cast<uint64_t>(position) * turns[i];
  // the fraction of a turn in [-1/2, 1/2), in half turns
  const float half_turns =
      static_cast<float>(static_cast<int32_t>(phase >> 32)) * 4.656612873077393e-10f;
  sincospif(half_turns, &s, &c);
  c *= gain;
  s *= gain;
}

struct Place {
  int64_t b, s;
};
B200_DEVICE Place place_of(const RotaryArgs& a, int64_t token) {
  Place p{0, token};
  if (a.tokens > a.seq) {  // several sequences
    if (a.tokens <= 0x7fffffff) {
      p.b = static_cast<uint32_t>(token) / static_cast<uint32_t>(a.seq);
      p.s = static_cast<uint32_t>(token) % static_cast<uint32_t>(a.seq);
    } else {
      p.b = token / a.seq;
      p.s = token - p.b * a.seq;
    }
  }
  return p;
}

B200_DEVICE int64_t position_of(const RotaryArgs& a, int64_t token) {
  const Place p = place_of(a, token);
  const int64_t at = p.b * a.pos_b + p.s * a.pos_s;
  return a.pos64 ? static_cast<const int64_t*>(a.positions)[at]
                 : static_cast<const int32_t*>(a.positions)[at];
}

// VEC: slots of 16 elements moved as two 16-byte vectors; otherwise any size,
// stride and alignment, and a slot is one pair or one copied element.
// Two heads ahead of a thread and three blocks an SM: 16,384 tokens of 32 + 8
// heads of 128 in 57.6 us (5.8 TB/s, 0.89 of the copy rate) with half of the head
// turning, 59.6 with all of it.  One head ahead: 61 to 66 us; four heads and two
// blocks, 62.8.
template <bool VEC, bool INTERLEAVED>
__global__ void __launch_bounds__(256, 3) rotary_kernel(const RotaryArgs a) {
  extern __shared__ float2 turn[];  // [token of the block][pair]: cos, sin
  b200::pdl_begin();
  const int half = a.rotary_dim / 2;
  const int64_t token0 = static_cast<int64_t>(blockIdx.x) * a.block_tokens;
  const int block_tokens =
      static_cast<int>(a.tokens - token0 < a.block_tokens ? a.tokens - token0 : a.block_tokens);
  for (int i = threadIdx.x; i < block_tokens * half; i += blockDim.x) {
    const int t = i / half;
    float2 v;
    angle(a.turns, i - t * half, position_of(a, token0 + t), a.gain, v.x, v.y);
    turn[i] = v;
  }
  __syncthreads();
  int rest = threadIdx.x / a.slot_threads;
  const int slot0 = threadIdx.x - rest * a.slot_threads;
  const int t = rest / a.groups;
  const int group = rest - t * a.groups;
  if (t >= block_tokens) return;
  const Place p = place_of(a, token0 + t);
  // where the token lies in q and k, in and out
  const __nv_bfloat16* in_q = a.in[0] + p.b * a.in_b[0] + p.s * a.in_s[0];
  const __nv_bfloat16* in_k = a.in[1] + p.b * a.in_b[1] + p.s * a.in_s[1];
  __nv_bfloat16* out_q = a.out[0] + p.b * a.out_b[0] + p.s * a.out_s[0];
  __nv_bfloat16* out_k = a.out[1] + p.b * a.out_b[1] + p.s * a.out_s[1];
  auto in_at = [&](int head) {
    return head < a.heads_q ? in_q + head * a.in_h[0] : in_k + (head - a.heads_q) * a.in_h[1];
  };
  auto out_at = [&](int head) {
    return head < a.heads_q ? out_q + head * a.out_h[0] : out_k + (head - a.heads_q) * a.out_h[1];
  };

  for (int slot = slot0; slot < a.slots; slot += a.slot_threads) {
    if constexpr (VEC) {
      const bool turns = slot * 16 < a.rotary_dim;
      const bool split = turns && !INTERLEAVED;
      const int e0 = split ? slot * 8 : slot * 16;
      const int e1 = split ? e0 + half : e0 + 8;
      float c[8], sn[8];
      if (turns) {
        const float4* from = reinterpret_cast<const float4*>(turn + t * half + slot * 8);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float4 v = from[j];
          c[2 * j] = v.x;
          sn[2 * j] = v.y;
          c[2 * j + 1] = v.z;
          sn[2 * j + 1] = v.w;
        }
      }
      // kAhead heads are read before the first of them is written
      constexpr int kAhead = 2;
      for (int first = group; first < a.heads; first += kAhead * a.groups) {
        uint4 u[kAhead][2];
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
          const int head = first + i * a.groups;
          if (head < a.heads) {
            const __nv_bfloat16* in = in_at(head);
            u[i][0] = *reinterpret_cast<const uint4*>(in + e0);
            u[i][1] = *reinterpret_cast<const uint4*>(in + e1);
          }
        }
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
          const int head = first + i * a.groups;
          if (head >= a.heads) break;
          uint32_t w0[4] = {u[i][0].x, u[i][0].y, u[i][0].z, u[i][0].w};
          uint32_t w1[4] = {u[i][1].x, u[i][1].y, u[i][1].z, u[i][1].w};
          if (split) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const float a0 = b200::bf16_lo(w0[j]), a1 = b200::bf16_hi(w0[j]);
              const float b0 = b200::bf16_lo(w1[j]), b1 = b200::bf16_hi(w1[j]);
              w0[j] = b200::pack_bf16x2(a0 * c[2 * j] - b0 * sn[2 * j],
                                        a1 * c[2 * j + 1] - b1 * sn[2 * j + 1]);
              w1[j] = b200::pack_bf16x2(b0 * c[2 * j] + a0 * sn[2 * j],
                                        b1 * c[2 * j + 1] + a1 * sn[2 * j + 1]);
            }
          } else if (turns) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const float a0 = b200::bf16_lo(w0[j]), b0 = b200::bf16_hi(w0[j]);
              const float a1 = b200::bf16_lo(w1[j]), b1 = b200::bf16_hi(w1[j]);
              w0[j] = b200::pack_bf16x2(a0 * c[j] - b0 * sn[j], b0 * c[j] + a0 * sn[j]);
              w1[j] = b200::pack_bf16x2(a1 * c[4 + j] - b1 * sn[4 + j],
                                        b1 * c[4 + j] + a1 * sn[4 + j]);
            }
          }
          __nv_bfloat16* out = out_at(head);
          *reinterpret_cast<uint4*>(out + e0) = make_uint4(w0[0], w0[1], w0[2], w0[3]);
          *reinterpret_cast<uint4*>(out + e1) = make_uint4(w1[0], w1[1], w1[2], w1[3]);
        }
      }
    } else {
      const bool turns = slot < half;
      const int e0 = !turns ? half + slot : INTERLEAVED ? 2 * slot : slot;
      const int e1 = INTERLEAVED ? e0 + 1 : e0 + half;
      const float2 v = turns ? turn[t * half + slot] : make_float2(1.0f, 0.0f);
      for (int head = group; head < a.heads; head += a.groups) {
        const __nv_bfloat16* in = in_at(head);
        __nv_bfloat16* out = out_at(head);
        if (turns) {
          const float x = __bfloat162float(in[e0]), y = __bfloat162float(in[e1]);
          out[e0] = __float2bfloat16_rn(x * v.x - y * v.y);
          out[e1] = __float2bfloat16_rn(y * v.x + x * v.y);
        } else {
          out[e0] = in[e0];
        }
      }
    }
  }
}

// cos and sin rows of some tokens, each angle at both elements of its pair.
__global__ void __launch_bounds__(256)
    rotary_tables_kernel(const RotaryArgs a, float* cos_out, float* sin_out) {
  b200::pdl_begin();
  const int64_t i = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x;
  const int half = a.rotary_dim / 2;
  if (i >= a.tokens * half) return;
  const int pair = static_cast<int>(i % half);
  const int64_t token = i / half;
  float c, sn;
  angle(a.turns, pair, position_of(a, token), a.gain, c, sn);
  const int64_t e0 = token * a.rotary_dim + (a.interleaved ? 2 * pair : pair);
  const int64_t e1 = e0 + (a.interleaved ? 1 : half);
  cos_out[e0] = c;
  cos_out[e1] = c;
  sin_out[e0] = sn;
  sin_out[e1] = sn;
}

int plan_args(RotaryArgs& a, const void* positions, int64_t pos_stride_b, int64_t pos_stride_s,
              int positions_64, const uint64_t* turns, float gain, int batch, int seq,
              int rotary_dim, int interleaved) {
  if (batch < 0 || seq < 0 || rotary_dim < 2 || (rotary_dim & 1)) return B200_ERR_INVALID_ARGUMENT;
  if (batch != 0 && seq != 0 && (!positions || !turns)) return B200_ERR_INVALID_ARGUMENT;
  a.positions = positions;
  a.pos_b = pos_stride_b;
  a.pos_s = pos_stride_s;
  a.pos64 = positions_64 != 0;
  a.turns = turns;
  a.gain = gain;
  a.tokens = static_cast<int64_t>(batch) * seq;
  a.seq = seq;
  a.rotary_dim = rotary_dim;
  a.interleaved = interleaved != 0;
  return B200_OK;
}

constexpr int64_t kMaxBlocks = 0x7fffffff;
constexpr int kMaxRotary = 8192;  // 32 KB of angles a token
// a thread's head and slot indexes step past their ends by two blocks at most
constexpr int kMaxHeads = 0x7fffffff - 1024, kMaxDim = kMaxHeads;

}  // namespace

extern "C" int b200_rotary(const void* q, int64_t q_stride_b, int64_t q_stride_h,
                           int64_t q_stride_s, const void* k, int64_t k_stride_b,
                           int64_t k_stride_h, int64_t k_stride_s, void* q_out,
                           int64_t qo_stride_b, int64_t qo_stride_h, int64_t qo_stride_s,
                           void* k_out, int64_t ko_stride_b, int64_t ko_stride_h,
                           int64_t ko_stride_s, const void* positions, int64_t pos_stride_b,
                           int64_t pos_stride_s, int positions_64, const uint64_t* turns,
                           float gain, int batch, int seq, int num_heads, int num_kv_heads,
                           int head_dim, int rotary_dim, int interleaved, void* stream) {
  RotaryArgs a{};
  const int st = plan_args(a, positions, pos_stride_b, pos_stride_s, positions_64, turns, gain,
                           batch, seq, rotary_dim, interleaved);
  if (st != B200_OK) return st;
  if (num_heads < 0 || num_kv_heads < 0 || head_dim < rotary_dim || head_dim > kMaxDim ||
      static_cast<int64_t>(num_heads) + num_kv_heads > kMaxHeads)
    return B200_ERR_INVALID_ARGUMENT;
  a.heads = num_heads + num_kv_heads;
  if (a.tokens == 0 || a.heads == 0) return B200_OK;
  if (rotary_dim > kMaxRotary) return B200_ERR_UNSUPPORTED;
  if ((num_heads > 0 && (!q || !q_out)) || (num_kv_heads > 0 && (!k || !k_out)))
    return B200_ERR_INVALID_ARGUMENT;
  a.heads_q = num_heads;
  a.dim = head_dim;
  const void* in[2] = {q, k};
  void* out[2] = {q_out, k_out};
  const int64_t strides[2][6] = {
      {q_stride_b, q_stride_h, q_stride_s, qo_stride_b, qo_stride_h, qo_stride_s},
      {k_stride_b, k_stride_h, k_stride_s, ko_stride_b, ko_stride_h, ko_stride_s}};
  bool vec = head_dim % 16 == 0 && rotary_dim % 16 == 0;
  for (int i = 0; i < 2; ++i) {
    a.in[i] = static_cast<const __nv_bfloat16*>(in[i]);
    a.out[i] = static_cast<__nv_bfloat16*>(out[i]);
    a.in_b[i] = strides[i][0];
    a.in_h[i] = strides[i][1];
    a.in_s[i] = strides[i][2];
    a.out_b[i] = strides[i][3];
    a.out_h[i] = strides[i][4];
    a.out_s[i] = strides[i][5];
    if ((i == 0 ? num_heads : num_kv_heads) == 0) continue;
    vec = vec && b200host::aligned16(in[i]) && b200host::aligned16(out[i]);
    for (int64_t v : strides[i]) vec = vec && (v & 7) == 0;
  }
  a.slots = vec ? head_dim / 16 : rotary_dim / 2 + (head_dim - rotary_dim);
  a.slot_threads = a.slots < 256 ? a.slots : 256;
  // Tokens of a block: as many as still leave four blocks an SM, so that a
  // decode step spreads over the GPU (64 tokens: one a block) and a prefill
  // computes few angles twice (8 tokens a block, 10 heads a thread).
  const int sms = b200host::sm_count(b200host::current_device());
  if (sms <= 0) return B200_ERR_CUDA;
  const int room = 256 / a.slot_threads;  // (token, head) places of a block
  a.block_tokens = 1;
  const int most = room / 8 >= a.heads ? 16 : 8;  // 16 where 8 leave a thread one head
  while (a.block_tokens < most && a.block_tokens * 2 <= room &&
         a.block_tokens * 2 * rotary_dim * 4 <= 32768 &&
         a.tokens / (a.block_tokens * 2) >= static_cast<int64_t>(sms) * 4)
    a.block_tokens *= 2;
  a.groups = room / a.block_tokens < a.heads ? room / a.block_tokens : a.heads;
  const int64_t blocks = (a.tokens + a.block_tokens - 1) / a.block_tokens;
  if (blocks > kMaxBlocks) return B200_ERR_INVALID_ARGUMENT;
  const int threads = (a.slot_threads * a.groups * a.block_tokens + 31) / 32 * 32;
  const auto kernel = vec ? (interleaved ? rotary_kernel<true, true> : rotary_kernel<true, false>)
                          : (interleaved ? rotary_kernel<false, true> : rotary_kernel<false, false>);
  const cudaError_t e = b200host::launch_pdl(kernel, dim3(static_cast<unsigned>(blocks)), dim3(threads),
                                             a.block_tokens * rotary_dim * 4,
                                             static_cast<cudaStream_t>(stream), a);
  return b200host::status_from_cuda(e);
}

extern "C" int b200_rotary_tables(const void* positions, int64_t pos_stride_b,
                                  int64_t pos_stride_s, int positions_64, const uint64_t* turns,
                                  float gain, float* cos_out, float* sin_out, int batch, int seq,
                                  int rotary_dim, int interleaved, void* stream) {
  RotaryArgs a{};
  const int st = plan_args(a, positions, pos_stride_b, pos_stride_s, positions_64, turns, gain,
                           batch, seq, rotary_dim, interleaved);
  if (st != B200_OK) return st;
  const int64_t work = a.tokens * (rotary_dim / 2);
  if (work == 0) return B200_OK;
  if (!cos_out || !sin_out) return B200_ERR_INVALID_ARGUMENT;
  const int64_t blocks = (work + 255) / 256;
  if (blocks > kMaxBlocks) return B200_ERR_INVALID_ARGUMENT;
  const cudaError_t e = b200host::launch_pdl(rotary_tables_kernel,
                                             dim3(static_cast<unsigned>(blocks)), dim3(256), 0,
                                             static_cast<cudaStream_t>(stream), a, cos_out, sin_out);
  return b200host::status_from_cuda(e);
}

extern "C" int b200_rotary_words(const int64_t* words) {
  if (!words) return B200_ERR_INVALID_ARGUMENT;
  b200host::Words w{words};
  const int wide_positions = w.integer(19), batch = w.integer(22), seq = w.integer(23);
  const int heads = w.integer(24), kv_heads = w.integer(25), dim = w.integer(26);
  const int rotary_dim = w.integer(27), interleaved = w.integer(28);
  if (!w.fit) return B200_ERR_INVALID_ARGUMENT;
  return b200_rotary(w.pointer(0), w.wide(1), w.wide(2), w.wide(3), w.pointer(4), w.wide(5),
                     w.wide(6), w.wide(7), w.pointer(8), w.wide(9), w.wide(10), w.wide(11),
                     w.pointer(12), w.wide(13), w.wide(14), w.wide(15), w.pointer(16), w.wide(17),
                     w.wide(18), wide_positions, w.pointer<uint64_t>(20), w.real(21), batch, seq,
                     heads, kv_heads, dim, rotary_dim, interleaved, w.pointer(29));
}
