// Matrix product with a fused epilogue, for sm_100a's tcgen05 tensor cores:
//   out = act(sx_t sw_n (X W^T)_tn + b_n) + r_tn                    plain
//   out = act(gate_tn) up_tn + r_tn, W = [gate rows; up rows]       gated
// X (m, k) and W (n or 2n, k) in bf16, or in e4m3 with an fp32 scale a row of
// each; accumulators, scales, bias, activation and residual in fp32, one
// rounding to bf16 at the end.
//
// The weight's rows are the M side of the instruction (128 TMEM lanes) and the
// tokens its N side: a decode step of a few tokens then streams W through full
// 128-row tiles and pads only the small token side, and one kernel serves nine
// tokens and thousands.  Token tiles of BN columns; two accumulators of BN
// columns, so the epilogue of one tile overlaps the product of the next.
//   warps 0-15   epilogue: lane l of warp w owns accumulator lane 32 (w % 4) + l,
//                of every fourth 16 token columns
//   warps 16, 17 TMA producers of W and X: 128-byte swizzled K-major panels, 128
//                weight rows and BN tokens x 128 bytes of K, one or two a stage
//   warp 18      MMA issuer: 4 instructions a panel (K = 32 bytes each)
// Gated: lanes 0-15 of every warp hold gate rows and lanes 16-31 the up rows
// of the same 16 outputs, so the two meet by one shuffle; the tile's rows
// come from one 4-D box (k, 16, gate/up, group), where n is no multiple of 16 the
// last tile's from 8 boxes of 16 rows.
//
// Many tokens: pairs of CTAs (cta_group::2) compute 256 weight rows x 128 or 256
// tokens, each with its own 128 weight rows and half of the tokens in shared
// memory: 64 KB a panel where two single tiles of 256 tokens load 96.
//
// Few tiles (a decode step): the CTAs (or pairs) of a cluster share one tile and
// split K; every CTA sends its fp32 partial to the CTA that owns its token columns
// through distributed shared memory, and the owners add the partials in rank
// order, so the result does not depend on timing.  Up to 8 tokens (16 with a small
// weight) go to the direct kernel of linear_small.cu.
//
// Bounds and what it measured (B200): large products by the tensor pipe, 97 %
// active in bf16 and 95 % in e4m3 at the 1.5 GHz that the power cap leaves: 4096
// tokens, 4096 -> 2 x 12288 gated with silu in 586 us (1.41 PFLOP/s) and 320 us
// (2.58 PFLOP/s).  256 rows of 151,936 logits by the memory and the last of 9 rounds
// of tiles: 89 us (4.4 TB/s; 81 into one output that partly stays in L2).  64 x 12288 x
// 4096 in e4m3 by the weight's bytes and about 5 us of launch, first loads, exchange
// and end: 12.8 us (4.0 TB/s), 13.7 with a residual.
//
// Every wait is bounded: one that runs out sets B200_DEV_TIMEOUT, the other
// roles give up too, outstanding copies are awaited and TMEM is freed.
#include "linear.cuh"
#include "once.cuh"
#include "tcgen05.cuh"
#include "words.cuh"

namespace {

using namespace b200;

constexpr int kRows = 128;        // weight rows of a tile (TMEM lanes)
constexpr int kKBytes = 128;      // bytes of K in a panel: one swizzle row
constexpr int kAPanel = kRows * kKBytes;
constexpr int kEpilogueWarps = 16;
constexpr int kSides = kEpilogueWarps / 4;  // warps of a lane quarter
constexpr int kCols = 16;                   // columns they take in turn
static_assert(kSides * kCols >= 64, "the columns a CTA owns at most in a split product");
constexpr int kThreads = (kEpilogueWarps + 3) * 32;
constexpr int kScales = (256 + kSides * kCols - 1) / (kSides * kCols) * kCols;  // of a warp
constexpr int kWeightWarp = kEpilogueWarps;
constexpr int kTokenWarp = kWeightWarp + 1;
constexpr int kMmaWarp = kTokenWarp + 1;
constexpr int kMaxStages = 10;
constexpr int kSmemBudget = 204 * 1024;  // dynamic shared memory of a CTA, at most
constexpr int kGroupTokens = 16;  // token tiles that take turns on the same weight rows
constexpr uint64_t kWaitLimitNs = 1000000000ull;   // 1 s a pipeline wait
constexpr uint64_t kDrainLimitNs = 100000000ull;   // 0.1 s a copy after a give-up

// Panels of a stage.  A stage costs its MMA warp about 400 clocks (the wait, the
// issue, the commit), the MMAs of one panel 64 to 512: the narrow tiles take two.
constexpr int panels(int bn) { return bn <= 128 ? 2 : 1; }

struct __align__(8) Barriers {
  uint64_t full[kMaxStages], empty[kMaxStages];
  uint64_t acc_full[2], acc_empty[2];
  uint32_t tmem_base;
  int32_t error;
};

B200_DEVICE bool wait_or_flag(uint32_t bar, uint32_t parity, Barriers* B, int32_t* dev_status) {
  if (mbar_wait_abortable(bar, parity, dev_status, kWaitLimitNs)) return true;
  if (atomicExch(&B->error, 1) == 0) flag_error(dev_status, B200_DEV_TIMEOUT);
  return false;
}

// The same for a whole warp: true where every lane's wait ended in time.
B200_DEVICE bool warp_wait(uint32_t bar, uint32_t parity, Barriers* B, int32_t* dev_status) {
  return __all_sync(0xffffffffu, wait_or_flag(bar, parity, B, dev_status));
}

// One lane of a converged warp, the same on every call.
B200_DEVICE bool elect_one() {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "elect.sync _|p, 0xffffffff;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}\n"
      : "=r"(r));
  return r != 0;
}

// c format f32, a / b format bf16 (1) of kind::f16 or e4m3 (0) of kind::f8f6f4, both K-major
template <bool FP8>
constexpr uint32_t instruction(uint32_t m, uint32_t n) {
  return (1u << 4) | ((FP8 ? 0u : 1u) << 7) | ((FP8 ? 0u : 1u) << 10) | ((n >> 3) << 17) |
         ((m >> 4) << 24);
}

// PAIR: the two CTAs of a cluster work as one (cta_group::2), rows 0-127 of A
// and the first half of B in the first CTA's shared memory, the rest in the second's
template <bool FP8, bool PAIR>
B200_DEVICE void mma(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  if constexpr (FP8 && PAIR) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
        : "memory");
  } else if constexpr (FP8) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
        : "memory");
  } else if constexpr (PAIR) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
        : "memory");
  } else {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
        : "memory");
  }
}

// every MMA issued so far by this thread is done: an arrival on `bar` (PAIR: on
// the barrier at that place in both CTAs of the pair, the first at rank `leader`)
template <bool PAIR>
B200_DEVICE void commit(uint32_t bar, int leader) {
  if constexpr (PAIR) {
    asm volatile(
        "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 "
        "[%0], %1;" ::"r"(bar),
        "h"(static_cast<uint16_t>(3 << leader))
        : "memory");
  } else {
    umma_commit(bar);
  }
}

// Tiled loads of this GPU's memory into this CTA (no multicast); PAIR: `bar` may lie
// in the other CTA of the pair.
template <bool PAIR>
B200_DEVICE void load_2d(uint32_t dst, const CUtensorMap* map, uint32_t bar, int c0, int c1) {
  if constexpr (PAIR) {
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
        ".cta_group::2 [%0], [%1, {%3, %4}], [%2];" ::"r"(dst),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(c0), "r"(c1)
        : "memory");
  } else {
    tma_load_2d(dst, map, bar, c0, c1);
  }
}
template <bool PAIR>
B200_DEVICE void load_4d(uint32_t dst, const CUtensorMap* map, uint32_t bar, int c0, int c1, int c2,
                         int c3) {
  if constexpr (PAIR) {
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
        ".cta_group::2 [%0], [%1, {%3, %4, %5, %6}], [%2];" ::"r"(dst),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(c0), "r"(c1), "r"(c2), "r"(c3)
        : "memory");
  } else {
    tma_load_4d_nohint(dst, map, bar, c0, c1, c2, c3);
  }
}

B200_DEVICE void prefetch_2d(const CUtensorMap* map, int c0, int c1) {
  asm volatile("cp.async.bulk.prefetch.tensor.2d.L2.global.tile [%0, {%1, %2}];" ::"l"(
                   reinterpret_cast<uint64_t>(map)),
               "r"(c0), "r"(c1)
               : "memory");
}
B200_DEVICE void prefetch_4d(const CUtensorMap* map, int c0, int c1, int c2, int c3) {
  asm volatile("cp.async.bulk.prefetch.tensor.4d.L2.global.tile [%0, {%1, %2, %3, %4}];" ::"l"(
                   reinterpret_cast<uint64_t>(map)),
               "r"(c0), "r"(c1), "r"(c2), "r"(c3)
               : "memory");
}

template <bool PAIR>
B200_DEVICE void tmem_alloc(uint32_t slot, uint32_t cols) {
  if constexpr (PAIR) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(slot),
                 "r"(cols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  } else {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(slot),
                 "r"(cols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
}
template <bool PAIR>
B200_DEVICE void tmem_dealloc(uint32_t tmem, uint32_t cols) {
  if constexpr (PAIR)
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(cols)
                 : "memory");
  else
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(cols)
                 : "memory");
}

B200_DEVICE void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
B200_DEVICE uint32_t remote_smem(uint32_t addr, uint32_t rank) {
  uint32_t r;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
  return r;
}
// an arrival on a barrier of any CTA of the cluster
B200_DEVICE void arrive_remote(uint32_t bar) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}
B200_DEVICE void st_remote(uint32_t addr, const uint32_t* v) {
  asm volatile("st.shared::cluster.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(v[0]), "r"(v[1]),
               "r"(v[2]), "r"(v[3])
               : "memory");
}
B200_DEVICE float4 ld_shared(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
               : "r"(addr)
               : "memory");
  return v;
}

// Where 4 columns (quad) of a row lie in an exchange buffer [from rank][quad][row]
// of 16 bytes: a warp's 32 rows are 512 bytes in one piece, there and back.
// (Rows of own columns, 16 bytes every 4 own, took the network 2.4 times as long.)
B200_DEVICE uint32_t exchange_at(int from, int row, int own, int quad) {
  return static_cast<uint32_t>((from * (own >> 2) + quad) * kRows + row) * 16;
}

struct Tile {
  int token0, n0;
};

// Tiles in groups of kGroupTokens token tiles: within a group the token tiles
// of one weight tile come one after another, so the CTAs at work at a time
// share few weight tiles and few token tiles in L2.
// PAIR: a tile has twice the weight rows, and n0 is its half of this CTA.
template <int BN, bool PAIR>
B200_DEVICE Tile tile_at(const LinearArgs& a, int tile, int half) {
  const int per_group = kGroupTokens * a.n_tiles;
  const int g = tile / per_group;
  const int first = g * kGroupTokens;
  const int rows = min(kGroupTokens, a.m_tiles - first);
  const int rem = tile - g * per_group;
  Tile t;
  t.token0 = (first + rem % rows) * BN;
  const int n_tile = PAIR ? rem / rows * 2 + half : rem / rows;
  t.n0 = n_tile * (a.gated ? kRows / 2 : kRows);
  return t;
}

// Gated: whether the tile's 4 groups of 16 outputs are whole.
B200_DEVICE bool whole_groups(const LinearArgs& a, int n0) { return n0 + kRows / 2 <= (a.n & ~15); }

B200_DEVICE uint32_t even_halves(uint32_t a, uint32_t b) { return __byte_perm(a, b, 0x5410); }
B200_DEVICE uint32_t odd_halves(uint32_t a, uint32_t b) { return __byte_perm(a, b, 0x7632); }

// A lane's share of the epilogue of a tile: turns raw accumulators of this
// lane's row into outputs.  Rows of out that take 16-byte accesses go through a
// buffer of the warp in shared memory ([two tokens][column] words of two bf16,
// 16-byte units swizzled), so a lane stores 8 columns of one token; others take
// 2-byte stores.  (By shuffles instead, at about 6 clocks of the SM each: 4.1
// thousand clocks a 128 x 256 tile with 4-byte stores, 6.5 with 16-byte ones.)
struct Epilogue {
  const LinearArgs& a;
  uint32_t* buf;     // 256 words of this warp
  int lane, row_n;   // output column of this lane
  int base_n;        // first output column of this warp
  bool high;         // upper half-warp
  float w_scale, bias;

  B200_DEVICE Epilogue(const LinearArgs& args, int n0, int warp, int l, uint32_t* b)
      : a(args), buf(b), lane(l) {
    base_n = n0 + (warp & 3) * (a.gated ? 16 : 32);
    row_n = base_n + (a.gated ? l & 15 : l);
    high = l >= 16;
    const int w_row = a.gated && high ? a.n + row_n : row_n;
    const bool live = row_n < a.n;
    w_scale = a.w_scale != nullptr && live ? a.w_scale[w_row] : 1.0f;
    bias = a.bias != nullptr && live ? __bfloat162float(a.bias[w_row]) : 0.0f;
  }

  // the line that holds this warp's columns of a token
  B200_DEVICE void prefetch_residual(int token) const {
    if (base_n < a.n) prefetch_l2(a.residual + token * a.r_row + base_n);
  }

  // Any strides: v[i] is the output of column row_n and token + i * step.
  template <int M>
  B200_DEVICE void put_direct(int token, int step, float (&v)[M]) const {
    const int tokens = row_n < a.n ? (a.m - token + step - 1) / step : 0;  // of this lane
    if (a.residual != nullptr) {
      const __nv_bfloat16* r = a.residual + token * a.r_row + row_n;
#pragma unroll
      for (int i = 0; i < M; ++i, r += step * a.r_row)
        if (i < tokens) v[i] += __bfloat162float(*r);
    }
    __nv_bfloat16* o = a.out + token * a.o_row + row_n;
#pragma unroll
    for (int i = 0; i < M; ++i, o += step * a.o_row)
      if (i < tokens) *o = __float2bfloat16_rn(v[i]);
  }

  // 16-byte unit `unit` of the row of tokens 2 pair, 2 pair + 1 (plain: 32 words a row)
  B200_DEVICE uint4* unit_at(int pair, int unit) const {
    return reinterpret_cast<uint4*>(buf) + pair * 8 + (unit ^ (pair & 1));
  }
  B200_DEVICE uint32_t* word_at(int pair) const {
    return reinterpret_cast<uint32_t*>(unit_at(pair, lane >> 2)) + (lane & 3);
  }

  // Plain: 16 tokens x 32 columns of the warp.  A lane loads and stores tokens
  // 2 pair and 2 pair + 1 of 8 columns, pair = lane / 4.
  struct Piece {
    uint4 even, odd;
  };
  B200_DEVICE void fetch_plain(int token, Piece& p) const {
    const int t = token + (lane >> 2) * 2, n = base_n + (lane & 3) * 8;
    p.even = p.odd = make_uint4(0, 0, 0, 0);
    const __nv_bfloat16* r = a.residual + t * a.r_row + n;
    if (n < a.n && t < a.m) p.even = *reinterpret_cast<const uint4*>(r);
    if (n < a.n && t + 1 < a.m) p.odd = *reinterpret_cast<const uint4*>(r + a.r_row);
  }
  B200_DEVICE void put_plain(int token, float (&v)[16], Piece& res, int next) const {
    const int pair = lane >> 2, unit = (lane & 3) * 2;
    if (a.residual != nullptr) {
      *unit_at(pair, unit) =
          make_uint4(even_halves(res.even.x, res.odd.x), odd_halves(res.even.x, res.odd.x),
                     even_halves(res.even.y, res.odd.y), odd_halves(res.even.y, res.odd.y));
      *unit_at(pair, unit + 1) =
          make_uint4(even_halves(res.even.z, res.odd.z), odd_halves(res.even.z, res.odd.z),
                     even_halves(res.even.w, res.odd.w), odd_halves(res.even.w, res.odd.w));
      __syncwarp();
      if (next >= 0) fetch_plain(next, res);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const uint32_t w = *word_at(i);
        v[2 * i] += bf16_lo(w);
        v[2 * i + 1] += bf16_hi(w);
      }
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) *word_at(i) = pack_bf16x2(v[2 * i], v[2 * i + 1]);
    __syncwarp();
    const uint4 x = *unit_at(pair, unit), y = *unit_at(pair, unit + 1);
    __syncwarp();
    const int t = token + pair * 2, n = base_n + (lane & 3) * 8;
    __nv_bfloat16* o = a.out + t * a.o_row + n;
    if (n < a.n && t < a.m)
      *reinterpret_cast<uint4*>(o) = make_uint4(even_halves(x.x, x.y), even_halves(x.z, x.w),
                                                even_halves(y.x, y.y), even_halves(y.z, y.w));
    if (n < a.n && t + 1 < a.m)
      *reinterpret_cast<uint4*>(o + a.o_row) =
          make_uint4(odd_halves(x.x, x.y), odd_halves(x.z, x.w), odd_halves(y.x, y.y),
                     odd_halves(y.z, y.w));
  }

  // Gated: 16 tokens x 16 columns.  v[j] is column row_n of token 2 j + high; rows
  // of 16 words hold tokens 4 i + high and 4 i + 2 + high, and a lane loads and
  // stores 4 columns of the two tokens of row lane / 4.
  B200_DEVICE void fetch_gated(int token, Piece& p) const {
    const int row = lane >> 2;
    const int t = token + (row >> 1) * 4 + (row & 1), n = base_n + (lane & 3) * 4;
    uint2 x = make_uint2(0, 0), y = make_uint2(0, 0);
    const __nv_bfloat16* r = a.residual + t * a.r_row + n;
    if (n < a.n && t < a.m) x = *reinterpret_cast<const uint2*>(r);
    if (n < a.n && t + 2 < a.m) y = *reinterpret_cast<const uint2*>(r + 2 * a.r_row);
    p.even = make_uint4(even_halves(x.x, y.x), odd_halves(x.x, y.x), even_halves(x.y, y.y),
                        odd_halves(x.y, y.y));
  }
  B200_DEVICE void put_gated(int token, float (&v)[8], Piece& res, int next) const {
    uint32_t* mine = buf + (high ? 16 : 0) + (lane & 15);  // + 32 a row pair
    uint4* piece = reinterpret_cast<uint4*>(buf) + lane;
    if (a.residual != nullptr) {
      *piece = res.even;
      __syncwarp();
      if (next >= 0) fetch_gated(next, res);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        v[2 * i] += bf16_lo(mine[32 * i]);
        v[2 * i + 1] += bf16_hi(mine[32 * i]);
      }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) mine[32 * i] = pack_bf16x2(v[2 * i], v[2 * i + 1]);
    __syncwarp();
    const uint4 x = *piece;
    __syncwarp();
    const int row = lane >> 2;
    const int t = token + (row >> 1) * 4 + (row & 1), n = base_n + (lane & 3) * 4;
    __nv_bfloat16* o = a.out + t * a.o_row + n;
    if (n < a.n && t < a.m)
      *reinterpret_cast<uint2*>(o) = make_uint2(even_halves(x.x, x.y), even_halves(x.z, x.w));
    if (n < a.n && t + 2 < a.m)
      *reinterpret_cast<uint2*>(o + 2 * a.o_row) =
          make_uint2(odd_halves(x.x, x.y), odd_halves(x.z, x.w));
  }

  // Gated: the low half-warp holds gate rows and the high one up rows; each lane
  // gives the other the values of half of the tokens and keeps a gate and an up
  // value of tokens 2 j + high.
  template <int N>
  B200_DEVICE void meet(const float (&v)[N], float (&gate)[N / 2], float (&up)[N / 2]) const {
    if constexpr (N == 16) {
      // 32 bytes a lane through the buffer (units swizzled by 4 lanes)
      const int to = lane * 2, from = (lane ^ 16) * 2, twist = (lane >> 2) & 1;
      uint4* units = reinterpret_cast<uint4*>(buf);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        float s[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) s[j] = high ? v[2 * (4 * h + j)] : v[2 * (4 * h + j) + 1];
        units[(to + h) ^ twist] = make_uint4(__float_as_uint(s[0]), __float_as_uint(s[1]),
                                             __float_as_uint(s[2]), __float_as_uint(s[3]));
      }
      __syncwarp();
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint4 u = units[(from + h) ^ twist];
        const float got[4] = {__uint_as_float(u.x), __uint_as_float(u.y), __uint_as_float(u.z),
                              __uint_as_float(u.w)};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int k = 4 * h + j;
          gate[k] = high ? got[j] : v[2 * k];
          up[k] = high ? v[2 * k + 1] : got[j];
        }
      }
      __syncwarp();
    } else {
#pragma unroll
      for (int i = 0; i < N / 2; ++i) {
        const float got = __shfl_xor_sync(0xffffffffu, high ? v[2 * i] : v[2 * i + 1], 16);
        gate[i] = high ? got : v[2 * i];
        up[i] = high ? v[2 * i + 1] : got;
      }
    }
  }

  // This lane's words of the residual of 16 tokens, where put_columns<16> wants them.
  B200_DEVICE void fetch(int token, Piece& p) const {
    if (!a.wide || a.residual == nullptr) return;
    if (a.gated) fetch_gated(token, p);
    else fetch_plain(token, p);
  }

  // accumulators of the tokens token .. token + N - 1; xs: their scales; res: what
  // fetch() gave for them, and gives for `next` (if any) when it is free; `wait`
  // ends when the accumulators are there
  template <int N, class Wait>
  B200_DEVICE void put_columns(int token, float (&v)[N], const float* xs, Piece& res, int next,
                               Wait&& wait) const {
    wait();
    if (a.w_scale != nullptr) {
#pragma unroll
      for (int i = 0; i < N; i += 4) {
        const float4 s = *reinterpret_cast<const float4*>(xs + i);
        v[i] *= w_scale * s.x;
        v[i + 1] *= w_scale * s.y;
        v[i + 2] *= w_scale * s.z;
        v[i + 3] *= w_scale * s.w;
      }
    }
    if (a.bias != nullptr) {
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] += bias;
    }
    if (a.gated) {
      float gate[N / 2], up[N / 2];
      meet(v, gate, up);
      activate(gate, a.act);
#pragma unroll
      for (int i = 0; i < N / 2; ++i) gate[i] *= up[i];
      if constexpr (N == 16) {
        if (a.wide) {
          put_gated(token, gate, res, next);
          return;
        }
      }
      put_direct(token + (high ? 1 : 0), 2, gate);
    } else {
      activate(v, a.act);
      if constexpr (N == 16) {
        if (a.wide) {
          put_plain(token, v, res, next);
          return;
        }
      }
      put_direct(token, 1, v);
    }
  }
};

// N of the columns of this CTA in a split product: the partials of all ranks in
// rank order, then the epilogue.  The warps of a lane quarter share the columns
// (kSides N of them, at least as many as a CTA owns).
template <int N>
B200_DEVICE void finish_split(const LinearArgs& a, const Epilogue& ep, uint32_t exchange, int own,
                              int token0, int warp, int lane, const float* xs,
                              Epilogue::Piece& res) {
  const int row = (warp & 3) * 32 + lane;
  const int c = (warp >> 2) * N;
  if (c >= own || token0 + c >= a.m) return;
  float v[N];
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = 0.0f;
#pragma unroll 2
  for (int from = 0; from < a.splits; ++from) {
#pragma unroll
    for (int i = 0; i < N; i += 4) {
      const float4 p = ld_shared(exchange + exchange_at(from, row, own, (c + i) >> 2));
      v[i] += p.x;
      v[i + 1] += p.y;
      v[i + 2] += p.z;
      v[i + 3] += p.w;
    }
  }
  ep.put_columns<N>(token0 + c, v, xs, res, -1, [] {});
}

template <int BN, bool FP8, bool PAIR>
__global__ void __launch_bounds__(kThreads, 1)
    linear_kernel(const __grid_constant__ CUtensorMap tm_w, const __grid_constant__ CUtensorMap tm_x,
                  const __grid_constant__ CUtensorMap tm_g, const LinearArgs a) {
  extern __shared__ uint8_t smem_raw[];
  __shared__ Barriers B;
  __shared__ __align__(16) uint32_t turn[kEpilogueWarps][256];  // outputs on their way
  __shared__ __align__(16) float xs[kEpilogueWarps][kScales];  // token scales of a warp's columns
  constexpr int kBRows = PAIR ? BN / 2 : BN;  // tokens in this CTA's shared memory
  constexpr int kPanels = panels(BN);
  constexpr int kBPanel = kBRows * kKBytes;
  constexpr int kABytes = kPanels * kAPanel, kBBytes = kPanels * kBPanel;
  constexpr int kStageBytes = kABytes + kBBytes;
  constexpr int kKElems = FP8 ? 128 : 64;  // of a panel
  constexpr uint32_t kTmemCols = 2 * BN;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  uint8_t* smem = reinterpret_cast<uint8_t*>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  const uint32_t base = smem_u32(smem);
  const uint32_t exchange = base + a.stages * kStageBytes;
  auto full = [&](int s) { return smem_u32(&B.full[s]); };
  auto empty = [&](int s) { return smem_u32(&B.empty[s]); };
  auto acc_full = [&](int b) { return smem_u32(&B.acc_full[b]); };
  auto acc_empty = [&](int b) { return smem_u32(&B.acc_empty[b]); };

  if (threadIdx.x == 0) {
    for (int s = 0; s < a.stages; ++s) {
      mbar_init(full(s), 2);
      mbar_init(empty(s), 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(acc_full(b), 1);
      // PAIR: the first CTA's MMA lane also hears from the second CTA
      mbar_init(acc_empty(b), kEpilogueWarps + (PAIR && blockIdx.x % 2 == 0 ? 1 : 0));
    }
    B.error = 0;
    fence_mbar_init();
    prefetch_tensormap(&tm_w);
    prefetch_tensormap(&tm_x);
    if (a.gated) prefetch_tensormap(&tm_g);
  }
  if (warp == kMmaWarp) {
    tmem_alloc<PAIR>(smem_u32(&B.tmem_base), kTmemCols);
  }
  tc_fence_before();
  if (PAIR || a.splits > 1) cluster_sync();  // every CTA of the cluster runs before any writes to it
  else __syncthreads();
  tc_fence_after();
  const uint32_t tmem = B.tmem_base;
  // a cluster: one tile, its K split among `splits` CTAs (PAIR: pairs of CTAs)
  const int cluster = (PAIR ? 2 : 1) * a.splits;
  const int rank = static_cast<int>(blockIdx.x) % cluster;
  const int half = PAIR ? rank & 1 : 0;
  const int leader = PAIR ? rank & ~1 : 0;
  const int part = PAIR ? rank >> 1 : rank;
  const int first = static_cast<int>(blockIdx.x) / cluster;
  const int stride = static_cast<int>(gridDim.x) / cluster;
  const int kb0 = static_cast<int>(static_cast<int64_t>(a.k_blocks) * part / a.splits);
  const int kb1 = static_cast<int>(static_cast<int64_t>(a.k_blocks) * (part + 1) / a.splits);

  const Tile first_tile = tile_at<BN, PAIR>(a, first, half);
  // a pipeline gave up before this launch: no new work until the host clears the
  // status (read before the wait below: the load would be on every launch's path; once
  // more after it where it is set, since the previous kernel may be the one that clears it;
  // the lanes of a warp agree: its waits are the whole warp's)
  bool aborted = __any_sync(0xffffffffu, timeout_on_record(a.dev_status));
  if (warp == kWeightWarp && lane == 0 && !aborted && first < a.m_tiles * a.n_tiles) {
    // The first weight tiles start towards L2 while the previous kernel drains (a
    // prefetch returns no data: what that kernel still writes is read after the wait).
    for (int p = kb0 * kPanels; p < min(kb1, kb0 + a.stages) * kPanels; ++p) {
      if (!a.gated) prefetch_2d(&tm_w, p * kKElems, first_tile.n0);
      else if (whole_groups(a, first_tile.n0))
        prefetch_4d(&tm_g, p * kKElems, 0, 0, first_tile.n0 / 16);
    }
  }
  pdl_begin();
  if (aborted) aborted = __any_sync(0xffffffffu, timeout_on_record(a.dev_status));
  const int tiles = aborted ? 0 : a.m_tiles * a.n_tiles;

  // The producer and MMA warps run their loops whole and one elected lane issues:
  // in a branch of a single lane every operand of a TMA or MMA instruction takes
  // its own move to the uniform registers (550 clocks a stage, whatever its size).
  if (warp == kWeightWarp || warp == kTokenWarp) {
    const bool elected = elect_one();
    const bool weights = warp == kWeightWarp;
    int stage = 0, issued = 0;
    uint32_t phase = 0;
    bool ok = true;
    for (int tile = first; ok && tile < tiles; tile += stride) {
      const Tile t = tile == first ? first_tile : tile_at<BN, PAIR>(a, tile, half);
      for (int kb = kb0; kb < kb1; ++kb) {
        // (the first use of a stage finds it empty: no wait on the launch's path)
        if (issued >= a.stages && !(ok = warp_wait(empty(stage), phase ^ 1, &B, a.dev_status)))
          break;
        if (elected) {
          // PAIR: both CTAs' copies count on the first CTA's barrier
          const uint32_t bar = PAIR ? remote_smem(full(stage), leader) : full(stage);
          const uint32_t dst = base + stage * kStageBytes;
          if (half == 0)
            mbar_arrive_expect_tx(full(stage), (PAIR ? 2 : 1) * (weights ? kABytes : kBBytes));
#pragma unroll
          for (int p = 0; p < kPanels; ++p) {  // (a panel past K's end arrives as zeros)
            const int k0 = (kb * kPanels + p) * kKElems;
            const uint32_t to = weights ? dst + p * kAPanel : dst + kABytes + p * kBPanel;
            if (!weights) {
              load_2d<PAIR>(to, &tm_x, bar, k0, t.token0 + half * kBRows);
            } else if (a.gated && whole_groups(a, t.n0)) {
              load_4d<PAIR>(to, &tm_g, bar, k0, 0, 0, t.n0 / 16);
            } else if (a.gated) {  // the last groups, or group, of 16
#pragma unroll
              for (int g = 0; g < 4; ++g) {
                load_2d<PAIR>(to + g * 4096, &tm_w, bar, k0, t.n0 + g * 16);
                load_2d<PAIR>(to + g * 4096 + 2048, &tm_w, bar, k0, a.n + t.n0 + g * 16);
              }
            } else {
              load_2d<PAIR>(to, &tm_w, bar, k0, t.n0);
            }
          }
        }
        ++issued;
        if (++stage == a.stages) {
          stage = 0;
          phase ^= 1;
        }
      }
    }
    // After a give-up the copies in flight land before the shared memory goes
    // away (PAIR: the first CTA waits for both CTAs' copies, and the second stays
    // until the cluster barrier at the end).
    if (!ok && half == 0) {
      for (int i = 0; i < min(issued, a.stages); ++i) {
        if (--stage < 0) {
          stage = a.stages - 1;
          phase ^= 1;
        }
        mbar_wait_abortable(full(stage), phase, nullptr, kDrainLimitNs);
      }
    }
  } else if (warp == kMmaWarp && half == 0) {
    constexpr uint32_t idesc = instruction<FP8>(PAIR ? 2 * kRows : kRows, BN);
    const bool elected = elect_one();
    const uint64_t desc0 = smem_desc(base, 16, 1024);  // + 16-byte units
    int stage = 0, count = 0;
    uint32_t phase = 0;
    bool ok = true;
    for (int tile = first; ok && tile < tiles; tile += stride, ++count) {
      const int buf = count & 1;
      if (!(ok = warp_wait(acc_empty(buf), ((count >> 1) & 1) ^ 1, &B, a.dev_status))) break;
      tc_fence_after();
      for (int kb = kb0; kb < kb1; ++kb) {
        if (!(ok = warp_wait(full(stage), phase, &B, a.dev_status))) break;
        tc_fence_after();
        if (elected) {
          const uint64_t da = desc0 + static_cast<uint32_t>(stage * (kStageBytes / 16));
          const uint64_t db = da + kABytes / 16;
#pragma unroll
          for (int j = 0; j < 4 * kPanels; ++j)
            mma<FP8, PAIR>(tmem + buf * BN, da + (j >> 2) * (kAPanel / 16) + 2 * (j & 3),
                           db + (j >> 2) * (kBPanel / 16) + 2 * (j & 3), idesc,
                           kb > kb0 || j > 0 ? 1u : 0u);
          commit<PAIR>(empty(stage), leader);
        }
        if (++stage == a.stages) {
          stage = 0;
          phase ^= 1;
        }
      }
      if (ok && elected) commit<PAIR>(acc_full(buf), leader);
    }
  } else if (PAIR && warp == kMmaWarp && lane == 0 && a.splits == 1) {
    // Second CTA: passes on that its accumulators were read.  From here, not from
    // the epilogue: a release to the cluster waits for the thread's stores.
    int count = 0;
    for (int tile = first; tile < tiles; tile += stride, ++count) {
      const int buf = count & 1;
      if (!wait_or_flag(acc_empty(buf), (count >> 1) & 1, &B, a.dev_status)) break;
      arrive_remote(remote_smem(acc_empty(buf), leader));
    }
  } else if (warp < kEpilogueWarps) {
    const int side = warp >> 2;
    const uint32_t lane0 = static_cast<uint32_t>((warp & 3) * 32) << 16;
    constexpr int kTurn = kSides * kCols;
    int count = 0;
    for (int tile = first; tile < tiles; tile += stride, ++count) {
      const Tile t = tile_at<BN, PAIR>(a, tile, half);
      const int buf = count & 1;
      const uint32_t acc = tmem + lane0 + buf * BN;
      const Epilogue ep(a, t.n0, warp, lane, turn[warp]);
      constexpr int kGroups = (BN + kTurn - 1) / kTurn;  // groups of kCols columns of this warp
      const int cols = min(BN, a.m - t.token0);
      if (a.w_scale != nullptr && a.splits == 1) {
        __syncwarp();
        for (int i = lane; i < kGroups * kCols; i += 32) {
          const int c = side * kCols + i / kCols * kTurn + i % kCols;
          xs[warp][i] = c < cols ? a.x_scale[t.token0 + c] : 0.0f;
        }
        __syncwarp();
      }
      if (a.residual != nullptr) {  // its lines come to L2 while the product runs
        const int from = a.splits == 1 ? 0 : part * (BN / a.splits);
        const int to = a.splits == 1 ? cols : min(cols, from + BN / a.splits);
        for (int c = from + side * 32 + lane; c < to; c += kSides * 32) ep.prefetch_residual(t.token0 + c);
      }
      Epilogue::Piece res;
      if (a.splits == 1 && side * kCols < cols) ep.fetch(t.token0 + side * kCols, res);
      if (!warp_wait(acc_full(buf), (count >> 1) & 1, &B, a.dev_status)) break;
      tc_fence_after();
      if (a.splits == 1) {
#pragma unroll 1
        for (int c = side * kCols, j = 0; c < cols; c += kTurn, j += kCols) {
          float v[kCols];
          tmem_ld16(acc + c, reinterpret_cast<uint32_t*>(v));
          ep.put_columns<kCols>(t.token0 + c, v, &xs[warp][j], res,
                                c + kTurn < cols ? t.token0 + c + kTurn : -1,
                                [&] { tmem_wait_ld16(reinterpret_cast<uint32_t*>(v)); });
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(acc_empty(buf));
      } else {
        // column c belongs to part c / own: into that CTA's exchange buffer
        const int own = BN / a.splits, shift = __ffs(own) - 1;
        const int row = (warp & 3) * 32 + lane;
#pragma unroll 1
        for (int c = side * kCols; c < BN; c += kTurn) {
          uint32_t r[kCols];
          tmem_ld16(acc + c, r);
          tmem_wait_ld16(r);
#pragma unroll
          for (int i = 0; i < kCols; i += 4) {
            const int to = (c + i) >> shift, quad = ((c + i) & (own - 1)) >> 2;
            st_remote(remote_smem(exchange + exchange_at(part, row, own, quad),
                                  PAIR ? 2 * to + half : to), r + i);
          }
        }
      }
    }
  }

  __syncwarp();
  if (a.splits > 1) {  // one tile a cluster
    const bool finishes = warp < kEpilogueWarps && first < tiles;
    const int own = BN / a.splits;
    const int token0 = first_tile.token0 + part * own;
    const int at_once = own >= 32 || (own == 16 && a.wide) ? 16 : own >= 16 ? 8 : 4;
    // scales and bias come while the partials travel
    const Epilogue ep(a, first_tile.n0, warp, lane, turn[finishes ? warp : 0]);
    if (finishes && a.w_scale != nullptr && lane < at_once) {
      const int t = token0 + (warp >> 2) * at_once + lane;
      xs[warp][lane] = t < a.m ? a.x_scale[t] : 0.0f;
    }
    Epilogue::Piece res;
    if (finishes && at_once == 16) ep.fetch(token0 + (warp >> 2) * 16, res);
    cluster_sync();
    if (finishes && B.error == 0) {
      if (at_once == 16) finish_split<16>(a, ep, exchange, own, token0, warp, lane, xs[warp], res);
      else if (at_once == 8) finish_split<8>(a, ep, exchange, own, token0, warp, lane, xs[warp], res);
      else finish_split<4>(a, ep, exchange, own, token0, warp, lane, xs[warp], res);
    }
  }
  tc_fence_before();
  if (PAIR) cluster_sync();  // the other CTA is done with this one's barriers and TMEM
  else __syncthreads();
  tc_fence_after();
  if (warp == kMmaWarp) tmem_dealloc<PAIR>(tmem, kTmemCols);
}

// ------------------------------------------------------------------ host side

b200host::OncePerDevice g_setup;
// CTAs of clusters of 1, 2, 4 and 8 that a device holds at once (clusters do not
// span its GPCs: 8 CTAs a cluster leave some SMs without one)
int g_resident[b200host::OncePerDevice::kDevices][4];

template <int BN, bool FP8, bool PAIR>
cudaError_t set_smem_attr() {
  return cudaFuncSetAttribute(linear_kernel<BN, FP8, PAIR>,
                              cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemBudget + 1024);
}

template <bool FP8>
cudaError_t set_smem_attrs() {
  const cudaError_t es[] = {set_smem_attr<32, FP8, false>(), set_smem_attr<64, FP8, false>(),
                            set_smem_attr<128, FP8, false>(), set_smem_attr<256, FP8, false>(),
                            set_smem_attr<128, FP8, true>(), set_smem_attr<256, FP8, true>()};
  for (cudaError_t e : es)
    if (e != cudaSuccess) return e;
  return cudaSuccess;
}

int set_up(int dev) {
  cudaError_t e = set_smem_attrs<false>();
  if (e == cudaSuccess) e = set_smem_attrs<true>();
  if (e != cudaSuccess) return b200host::status_from_cuda(e);
  g_resident[dev][0] = b200host::sm_count(dev);
  for (int i = 1; i < 4; ++i) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(1u << i);
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = kSmemBudget;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = 1u << i;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    int clusters = 0;
    e = cudaOccupancyMaxActiveClusters(&clusters, linear_kernel<32, false, false>, &cfg);
    if (e != cudaSuccess) return b200host::status_from_cuda(e);
    g_resident[dev][i] = clusters << i;
  }
  return B200_OK;
}

int ensure_set_up(int dev) {
  if (dev < 0 || dev >= b200host::OncePerDevice::kDevices) return B200_ERR_CUDA;
  return g_setup.run(dev, [dev] { return set_up(dev); });
}

// How a product is cut: token tiles of bn, 128 weight rows a CTA or 256 a pair of
// CTAs, and K split among the CTAs or pairs of a cluster.
// The times (us) are fitted to 219 launches of 23 shapes (17 to 2048 tokens, K 300
// to 12,288, both types): 4 for a launch, its first loads and its end; `panel` for
// 128 bytes of K of a tile, or the weight's bytes at 5.6 TB/s where that is more,
// and a third of the other (256 rows of 151,936 logits: 81 us in pairs of 256, 95
// in (128), whose main loops alone would both hide behind the weight);
// `epilogue` for the last tile's, `exchange` for each halving of K.  Over the 23
// shapes the choice is within 2 % of the best cut on average and 10 % at most:
// 64 x 12288 x 4096 in e4m3 takes 13.2 us in (64, split 4) and 16.8 in (64, split
// 2), 512 x 4096 x 4096 18.0 in pairs of 128, 19.0 in (128) and 25 in (64) or
// pairs of 256, 256 x 4096 x 4096 14.7 in (64) and 16.7 in (128, split 2).
struct Cut {
  int bn;
  bool pair;
  int max_log;                        // K is split at most 2^max_log ways
  float panel, epilogue, exchange;
};
constexpr Cut kCuts[] = {
    {32, false, 3, 0.14f, 0.0f, 0.6f},   {64, false, 3, 0.146f, 0.1f, 0.62f},
    {128, false, 2, 0.206f, 0.4f, 3.0f}, {256, false, 0, 0.31f, 1.2f, 0.0f},
    {128, true, 2, 0.15f, 1.6f, 3.1f},   {256, true, 0, 0.25f, 2.1f, 0.0f}};

struct Plan {
  int bn, splits;
  bool pair;
};

// The cut with the least estimated time.
Plan choose(int m, int n_tiles, int k_panels, const int* resident) {
  const float read = static_cast<float>(n_tiles) * k_panels * kAPanel / 5.6e6f;
  Plan best{32, 1, false};
  float least = 3.4e38f;
  for (const Cut& c : kCuts) {
    const int64_t tiles = static_cast<int64_t>((m + c.bn - 1) / c.bn) *
                          (c.pair ? (n_tiles + 1) / 2 : n_tiles);
    for (int log = 0; log <= c.max_log; ++log) {
      const int splits = 1 << log;
      if (splits > 1 && splits * 2 > k_panels) break;
      const int log_ctas = log + (c.pair ? 1 : 0);
      const int64_t room = resident[log_ctas] >> log_ctas;
      if (room == 0) break;
      const float waves = static_cast<float>((tiles + room - 1) / room);
      if (splits > 1 && waves > 1.0f) break;  // clusters that split K do not persist
      const float main = waves * ((k_panels + splits - 1) / splits) * c.panel;
      const float t = 4.0f + (main > read ? main + 0.35f * read : read + 0.35f * main) +
                      c.epilogue + log * c.exchange;
      if (t < least) {
        least = t;
        best = Plan{c.bn, splits, c.pair};
      }
    }
  }
  return best;
}

// rows x k elements of `size` bytes, K innermost
int encode_rows(CUtensorMap* map, const void* base, int64_t rows, int64_t k, int64_t stride,
                bool fp8, int box_rows) {
  const int size = fp8 ? 1 : 2;
  const cuuint64_t dims[2] = {static_cast<cuuint64_t>(k), static_cast<cuuint64_t>(rows)};
  const cuuint64_t strides[1] = {static_cast<cuuint64_t>(stride) * size};
  const cuuint32_t box[2] = {static_cast<cuuint32_t>(kKBytes / size),
                             static_cast<cuuint32_t>(box_rows)};
  const cuuint32_t es[2] = {1, 1};
  return b200host::encode_tiled(map, fp8 ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16,
                                2, const_cast<void*>(base), dims, strides, box, es,
                                CU_TENSOR_MAP_SWIZZLE_128B,
                                CU_TENSOR_MAP_L2_PROMOTION_L2_256B) == CUDA_SUCCESS
             ? B200_OK
             : B200_ERR_TENSOR_MAP;
}

// gate and up rows as (k, 16, gate / up, whole group of 16): a box is a tile's 128 rows
int encode_gated(CUtensorMap* map, const void* base, int64_t n, int64_t k, int64_t stride,
                 bool fp8) {
  const int size = fp8 ? 1 : 2;
  const cuuint64_t row = static_cast<cuuint64_t>(stride) * size;
  const cuuint64_t dims[4] = {static_cast<cuuint64_t>(k), 16u, 2u, static_cast<cuuint64_t>(n / 16)};
  const cuuint64_t strides[3] = {row, row * static_cast<cuuint64_t>(n), row * 16};
  const cuuint32_t box[4] = {static_cast<cuuint32_t>(kKBytes / size), 16, 2, 4};
  const cuuint32_t es[4] = {1, 1, 1, 1};
  return b200host::encode_tiled(map, fp8 ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16,
                                4, const_cast<void*>(base), dims, strides, box, es,
                                CU_TENSOR_MAP_SWIZZLE_128B,
                                CU_TENSOR_MAP_L2_PROMOTION_L2_256B) == CUDA_SUCCESS
             ? B200_OK
             : B200_ERR_TENSOR_MAP;
}

template <int BN, bool FP8, bool PAIR>
cudaError_t launch(const CUtensorMap& tw, const CUtensorMap& tx, const CUtensorMap& tg, LinearArgs a, int sms,
                   cudaStream_t stream) {
  const int stage_bytes = panels(BN) * (kAPanel + (PAIR ? BN / 2 : BN) * kKBytes);
  const int exchange = a.splits > 1 ? BN * kRows * 4 : 0;
  a.stages = (kSmemBudget - exchange) / stage_bytes;
  if (a.stages > kMaxStages) a.stages = kMaxStages;
  const int cluster = (PAIR ? 2 : 1) * a.splits;
  const int64_t ctas = static_cast<int64_t>(a.m_tiles) * a.n_tiles * cluster;
  // without a split of K the CTAs (or pairs) persist and take tiles in turn
  const int resident = PAIR ? g_resident[b200host::current_device()][1] : sms;
  const int grid = static_cast<int>(a.splits > 1 || ctas < resident ? ctas : resident);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(grid));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = a.stages * stage_bytes + exchange + 1024;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = static_cast<unsigned>(cluster);
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = cluster > 1 ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, linear_kernel<BN, FP8, PAIR>, tw, tx, tg, a);
}

template <bool FP8>
cudaError_t launch_bn(int bn, bool pair, const CUtensorMap& tw, const CUtensorMap& tx,
                      const CUtensorMap& tg, const LinearArgs& a, int sms,
                      cudaStream_t stream) {
  if (pair)
    return bn == 128 ? launch<128, FP8, true>(tw, tx, tg, a, sms, stream)
                     : launch<256, FP8, true>(tw, tx, tg, a, sms, stream);
  switch (bn) {
    case 32: return launch<32, FP8, false>(tw, tx, tg, a, sms, stream);
    case 64: return launch<64, FP8, false>(tw, tx, tg, a, sms, stream);
    case 128: return launch<128, FP8, false>(tw, tx, tg, a, sms, stream);
    default: return launch<256, FP8, false>(tw, tx, tg, a, sms, stream);
  }
}

}  // namespace

namespace {

constexpr int kPackAhead = 4;

// dst rows (16-byte aligned, zero to the next multiple of 16 bytes) from src rows
// at any address; a thread takes kPackAhead pieces of 16 bytes of a row
__global__ void __launch_bounds__(256) pack_rows_kernel(const uint8_t* src, int64_t src_stride,
                                                        uint8_t* dst, int64_t dst_stride, int64_t rows,
                                                        int row_bytes) {
  pdl_begin();
  const int64_t row = static_cast<int64_t>(blockIdx.x) * blockDim.y + threadIdx.y;
  if (row >= rows) return;
  const uint8_t* from = src + row * src_stride;
  uint8_t* to = dst + row * dst_stride;
  const int at0 = (blockIdx.y * blockDim.x * kPackAhead + threadIdx.x) * 16;
  Unaligned16 u[kPackAhead];
#pragma unroll
  for (int i = 0; i < kPackAhead; ++i) {
    const int at = at0 + i * blockDim.x * 16;
    if (at + 16 <= row_bytes) u[i] = load_unaligned16(from + at);
  }
#pragma unroll
  for (int i = 0; i < kPackAhead; ++i) {
    const int at = at0 + i * blockDim.x * 16;
    if (at + 16 <= row_bytes) {
      *reinterpret_cast<uint4*>(to + at) = shifted(u[i]);
    } else if (at < row_bytes) {
      uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
      for (int b = 0; b < 15; ++b)
        if (at + b < row_bytes) w[b >> 2] |= static_cast<uint32_t>(from[at + b]) << (8 * (b & 3));
      *reinterpret_cast<uint4*>(to + at) = make_uint4(w[0], w[1], w[2], w[3]);
    }
  }
}

}  // namespace

extern "C" int b200_pack_rows(const void* src, int64_t src_stride, void* dst, int64_t dst_stride,
                              int64_t rows, int row_bytes, void* stream) {
  if (rows < 0 || row_bytes <= 0 || row_bytes > 0x7fffffe0) return B200_ERR_INVALID_ARGUMENT;
  if (rows == 0) return B200_OK;
  const int pieces = (row_bytes + 15) / 16;
  if (!src || !dst || dst_stride < static_cast<int64_t>(pieces) * 16) return B200_ERR_INVALID_ARGUMENT;
  if (!b200host::aligned16(dst) || dst_stride % 16) return B200_ERR_ALIGNMENT;
  int threads = (pieces + kPackAhead - 1) / kPackAhead;
  threads = threads > 128 ? 256 : threads > 64 ? 128 : threads > 32 ? 64 : threads > 16 ? 32 : 16;
  const int columns = (pieces + threads * kPackAhead - 1) / (threads * kPackAhead);
  const int together = 256 / threads;  // rows of a block
  const int64_t blocks = (rows + together - 1) / together;
  if (blocks > 0x7fffffff || columns > 65535) return B200_ERR_INVALID_ARGUMENT;
  return b200host::status_from_cuda(b200host::launch_pdl(
      pack_rows_kernel, dim3(static_cast<unsigned>(blocks), static_cast<unsigned>(columns)),
      dim3(threads, together), 0, static_cast<cudaStream_t>(stream),
      static_cast<const uint8_t*>(src), src_stride, static_cast<uint8_t*>(dst), dst_stride, rows,
      row_bytes));
}

namespace {

int linear_any(const void* x, int64_t x_stride, const float* x_scale, const void* w,
               int64_t w_stride, const float* w_scale, const void* bias,
               const void* residual, int64_t r_stride, void* out, int64_t o_stride,
               int m, int n, int k, int fp8, int gated, int activation,
               int32_t* dev_status, void* stream, bool any_address) {
  // (2 n and the bytes of a row fit an int, and so does the last token tile's end)
  if (m < 0 || n <= 0 || k <= 0 || m > 0x7fffffff - 255 || n > 0x3fffffff || k > 0x1fffffff)
    return B200_ERR_INVALID_ARGUMENT;
  if (activation < B200_ACT_NONE || activation > B200_ACT_GELU_TANH)
    return B200_ERR_INVALID_ARGUMENT;
  if (m == 0) return B200_OK;
  if (!x || !w || !out) return B200_ERR_INVALID_ARGUMENT;
  if (fp8 ? !x_scale || !w_scale : x_scale || w_scale) return B200_ERR_INVALID_ARGUMENT;
  const int64_t unit = fp8 ? 16 : 8;  // elements of 16 bytes
  if (!any_address &&
      (!b200host::aligned16(x) || !b200host::aligned16(w) || x_stride % unit || w_stride % unit))
    return B200_ERR_ALIGNMENT;  // the tensor maps' rule; b200_pack_rows lays rows out
  if (x_stride < k || w_stride < k || o_stride < n || (residual && r_stride < n))
    return B200_ERR_INVALID_ARGUMENT;

  LinearArgs a{};
  a.x_scale = x_scale;
  a.w_scale = w_scale;
  a.bias = static_cast<const __nv_bfloat16*>(bias);
  a.residual = static_cast<const __nv_bfloat16*>(residual);
  a.out = static_cast<__nv_bfloat16*>(out);
  a.r_row = r_stride;
  a.o_row = o_stride;
  a.m = m;
  a.n = n;
  const int per = fp8 ? 128 : 64;
  const int k_panels = (k + per - 1) / per;
  a.gated = gated != 0;
  a.act = activation;
  a.dev_status = dev_status;
  a.wide = n % 8 == 0 && o_stride % 8 == 0 && b200host::aligned16(out) &&
           (residual == nullptr || (r_stride % 8 == 0 && b200host::aligned16(residual)));
  const int dev = b200host::current_device();
  const int sms = b200host::sm_count(dev);
  if (sms <= 0) return B200_ERR_CUDA;
  cudaStream_t cs = static_cast<cudaStream_t>(stream);
  if (b200host::linear_is_small(a, k, fp8 != 0))
    return b200host::status_from_cuda(
        b200host::linear_small(a, x, x_stride, w, w_stride, k, fp8 != 0, sms, cs));
  int st = ensure_set_up(dev);
  if (st != B200_OK) return st;

  const int tile_n = gated ? kRows / 2 : kRows;
  a.n_tiles = (n + tile_n - 1) / tile_n;
  const Plan plan = choose(m, a.n_tiles, k_panels, g_resident[dev]);
  a.k_blocks = (k_panels + panels(plan.bn) - 1) / panels(plan.bn);
  const int bn = plan.bn;
  const bool pair = plan.pair;
  a.m_tiles = (m + bn - 1) / bn;
  a.splits = plan.splits;
  if (pair) a.n_tiles = (a.n_tiles + 1) / 2;
  if (static_cast<int64_t>(a.m_tiles) * a.n_tiles > 0x0fffffff) return B200_ERR_INVALID_ARGUMENT;

  // gated: tw reads single groups of 16 rows, tg whole tiles of gate and up rows
  CUtensorMap tw, tx, tg;
  st = encode_rows(&tw, w, gated ? 2 * static_cast<int64_t>(n) : n, k, w_stride, fp8 != 0,
                   gated ? 16 : kRows);
  const bool whole_tiles = gated && n >= kRows / 2;
  if (st == B200_OK && whole_tiles) st = encode_gated(&tg, w, n, k, w_stride, fp8 != 0);
  if (!whole_tiles) tg = tw;
  if (st == B200_OK) st = encode_rows(&tx, x, m, k, x_stride, fp8 != 0, pair ? bn / 2 : bn);
  if (st != B200_OK) return st;
  return b200host::status_from_cuda(fp8 ? launch_bn<true>(bn, pair, tw, tx, tg, a, sms, cs)
                                        : launch_bn<false>(bn, pair, tw, tx, tg, a, sms, cs));
}

}  // namespace

extern "C" int b200_linear(const void* x, int64_t x_stride, const float* x_scale, const void* w,
                           int64_t w_stride, const float* w_scale, const void* bias,
                           const void* residual, int64_t r_stride, void* out, int64_t o_stride,
                           int m, int n, int k, int fp8, int gated, int activation,
                           int32_t* dev_status, void* stream) {
  return linear_any(x, x_stride, x_scale, w, w_stride, w_scale, bias, residual, r_stride, out,
                    o_stride, m, n, k, fp8, gated, activation, dev_status, stream, false);
}

extern "C" int b200_linear_unaligned(const void* x, int64_t x_stride, const float* x_scale, const void* w,
                                     int64_t w_stride, const float* w_scale, const void* bias,
                                     const void* residual, int64_t r_stride, void* out, int64_t o_stride,
                                     int m, int n, int k, int fp8, int gated, int activation,
                                     int32_t* dev_status, void* stream) {
  if (m > 8) return B200_ERR_UNSUPPORTED;
  return linear_any(x, x_stride, x_scale, w, w_stride, w_scale, bias, residual, r_stride, out,
                    o_stride, m, n, k, fp8, gated, activation, dev_status, stream, true);
}

extern "C" int b200_linear_words(const int64_t* words) {
  if (!words) return B200_ERR_INVALID_ARGUMENT;
  b200host::Words w{words};
  const int m = w.integer(11), n = w.integer(12), k = w.integer(13);
  const int fp8 = w.integer(14), gated = w.integer(15), activation = w.integer(16);
  const bool any_address = w.integer(19) != 0;
  if (!w.fit) return B200_ERR_INVALID_ARGUMENT;
  const auto entry = any_address ? b200_linear_unaligned : b200_linear;
  return entry(w.pointer(0), w.wide(1), w.pointer<float>(2), w.pointer(3), w.wide(4),
               w.pointer<float>(5), w.pointer(6), w.pointer(7), w.wide(8), w.pointer(9), w.wide(10),
               m, n, k, fp8, gated, activation, w.pointer<int32_t>(17), w.pointer(18));
}
