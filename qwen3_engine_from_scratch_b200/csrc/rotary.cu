// Rotary positions: every pair (a, b) of a head's first rotary_dim elements is
// turned by the angle position * f_i and scaled by the plan's gain,
//   a' = gain (a cos - b sin),  b' = gain (b cos + a sin),
// pairs (i, i + rotary_dim / 2) in the half layout, (2i, 2i + 1) in the
// interleaved one; the rest of the head is copied.
//
// Angles: the plan holds f_i / 2 pi as a 64-bit binary fraction of a turn, so
// position * f_i modulo one turn is one 64-bit integer product, exact to
// position * 2^-64 turns at any position (negative ones included); the top 32
// bits then go through sincospi.  A product in fp32 would lose position * 2^-24
// radians: 0.008 at position 131,072.
//
// Bound by memory for prefills: q and k are read and written once.  A thread
// takes one slot of 16 elements (8 pairs, or 16 copied elements) of one token
// and walks over some of the token's heads, so its 8 sines and cosines are
// computed once for several heads.
#include "common.cuh"

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
  int slots;                    // slots of a head
  int groups;                   // threads that share a (token, slot), each with some heads
  int interleaved;
  int64_t work;                 // threads with work
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

B200_DEVICE int64_t position_of(const RotaryArgs& a, int64_t token) {
  const int64_t b = token / a.seq, s = token - b * a.seq;
  const int64_t at = b * a.pos_b + s * a.pos_s;
  return a.pos64 ? static_cast<const int64_t*>(a.positions)[at]
                 : static_cast<const int32_t*>(a.positions)[at];
}

// first element of a token's head in q or k (`which`)
B200_DEVICE const __nv_bfloat16* head_in(const RotaryArgs& a, int64_t b, int64_t s, int head,
                                         int& which) {
  which = head >= a.heads_q;
  const int h = which ? head - a.heads_q : head;
  return which ? a.in[1] + b * a.in_b[1] + h * a.in_h[1] + s * a.in_s[1]
               : a.in[0] + b * a.in_b[0] + h * a.in_h[0] + s * a.in_s[0];
}
B200_DEVICE __nv_bfloat16* head_out(const RotaryArgs& a, int64_t b, int64_t s, int head) {
  const int which = head >= a.heads_q;
  const int h = which ? head - a.heads_q : head;
  return which ? a.out[1] + b * a.out_b[1] + h * a.out_h[1] + s * a.out_s[1]
               : a.out[0] + b * a.out_b[0] + h * a.out_h[0] + s * a.out_s[0];
}

// Slots of 16 elements, moved as two 16-byte vectors.
__global__ void __launch_bounds__(256) rotary_vector_kernel(const RotaryArgs a) {
  b200::pdl_begin();
  const int64_t i = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x;
  if (i >= a.work) return;
  const int slot = static_cast<int>(i % a.slots);
  const int64_t rest = i / a.slots;
  const int group = static_cast<int>(rest % a.groups);
  const int64_t token = rest / a.groups;
  const int64_t b = token / a.seq, s = token - b * a.seq;
  const bool turn = slot * 16 < a.rotary_dim;
  const bool split = turn && !a.interleaved;
  const int e0 = split ? slot * 8 : slot * 16;
  const int e1 = split ? e0 + a.rotary_dim / 2 : e0 + 8;

  float c[8], sn[8];
  if (turn) {
    const int64_t position = position_of(a, token);
#pragma unroll
    for (int j = 0; j < 8; ++j) angle(a.turns, slot * 8 + j, position, a.gain, c[j], sn[j]);
  }
  for (int head = group; head < a.heads; head += a.groups) {
    int which;
    const __nv_bfloat16* in = head_in(a, b, s, head, which);
    __nv_bfloat16* out = head_out(a, b, s, head);
    const uint4 u0 = *reinterpret_cast<const uint4*>(in + e0);
    const uint4 u1 = *reinterpret_cast<const uint4*>(in + e1);
    uint32_t w0[4] = {u0.x, u0.y, u0.z, u0.w}, w1[4] = {u1.x, u1.y, u1.z, u1.w};
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
    } else if (turn) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float a0 = b200::bf16_lo(w0[j]), b0 = b200::bf16_hi(w0[j]);
        const float a1 = b200::bf16_lo(w1[j]), b1 = b200::bf16_hi(w1[j]);
        w0[j] = b200::pack_bf16x2(a0 * c[j] - b0 * sn[j], b0 * c[j] + a0 * sn[j]);
        w1[j] = b200::pack_bf16x2(a1 * c[4 + j] - b1 * sn[4 + j], b1 * c[4 + j] + a1 * sn[4 + j]);
      }
    }
    *reinterpret_cast<uint4*>(out + e0) = make_uint4(w0[0], w0[1], w0[2], w0[3]);
    *reinterpret_cast<uint4*>(out + e1) = make_uint4(w1[0], w1[1], w1[2], w1[3]);
  }
}

// Any size, stride and alignment: a slot is one pair, or one copied element.
__global__ void __launch_bounds__(256) rotary_scalar_kernel(const RotaryArgs a) {
  b200::pdl_begin();
  const int64_t i = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x;
  if (i >= a.work) return;
  const int slot = static_cast<int>(i % a.slots);
  const int64_t rest = i / a.slots;
  const int group = static_cast<int>(rest % a.groups);
  const int64_t token = rest / a.groups;
  const int64_t b = token / a.seq, s = token - b * a.seq;
  const int half = a.rotary_dim / 2;
  const bool turn = slot < half;
  const int e0 = !turn ? half + slot : a.interleaved ? 2 * slot : slot;
  const int e1 = a.interleaved ? e0 + 1 : e0 + half;
  float c = 1.0f, sn = 0.0f;
  if (turn) angle(a.turns, slot, position_of(a, token), a.gain, c, sn);
  for (int head = group; head < a.heads; head += a.groups) {
    int which;
    const __nv_bfloat16* in = head_in(a, b, s, head, which);
    __nv_bfloat16* out = head_out(a, b, s, head);
    if (turn) {
      const float x = __bfloat162float(in[e0]), y = __bfloat162float(in[e1]);
      out[e0] = __float2bfloat16_rn(x * c - y * sn);
      out[e1] = __float2bfloat16_rn(y * c + x * sn);
    } else {
      out[e0] = in[e0];
    }
  }
}

// cos and sin rows of some tokens, each angle at both elements of its pair.
__global__ void __launch_bounds__(256)
    rotary_tables_kernel(const RotaryArgs a, float* cos_out, float* sin_out) {
  b200::pdl_begin();
  const int64_t i = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x;
  if (i >= a.work) return;
  const int half = a.rotary_dim / 2;
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
  a.seq = seq;
  a.rotary_dim = rotary_dim;
  a.interleaved = interleaved != 0;
  return B200_OK;
}

constexpr int64_t kMaxBlocks = 0x7fffffff;

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
  if (num_heads < 0 || num_kv_heads < 0 || head_dim < rotary_dim) return B200_ERR_INVALID_ARGUMENT;
  const int64_t tokens = static_cast<int64_t>(batch) * seq;
  a.heads = num_heads + num_kv_heads;
  if (tokens == 0 || a.heads == 0) return B200_OK;
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
  // threads that share a token's slot: 8 heads each, fewer when the tokens
  // alone do not fill the GPU
  a.groups = (a.heads + 7) / 8;
  const int sms = b200host::sm_count(b200host::current_device());
  if (sms <= 0) return B200_ERR_CUDA;
  while (a.groups < a.heads && tokens * a.slots * a.groups < static_cast<int64_t>(sms) * 1024)
    a.groups = a.groups * 2 < a.heads ? a.groups * 2 : a.heads;
  a.work = tokens * a.slots * a.groups;
  const int64_t blocks = (a.work + 255) / 256;
  if (blocks > kMaxBlocks) return B200_ERR_INVALID_ARGUMENT;
  const cudaError_t e = b200host::launch_pdl(vec ? rotary_vector_kernel : rotary_scalar_kernel,
                                             dim3(static_cast<unsigned>(blocks)), dim3(256), 0,
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
  a.work = static_cast<int64_t>(batch) * seq * (rotary_dim / 2);
  if (a.work == 0) return B200_OK;
  if (!cos_out || !sin_out) return B200_ERR_INVALID_ARGUMENT;
  const int64_t blocks = (a.work + 255) / 256;
  if (blocks > kMaxBlocks) return B200_ERR_INVALID_ARGUMENT;
  const cudaError_t e = b200host::launch_pdl(rotary_tables_kernel,
                                             dim3(static_cast<unsigned>(blocks)), dim3(256), 0,
                                             static_cast<cudaStream_t>(stream), a, cos_out, sin_out);
  return b200host::status_from_cuda(e);
}
