// Attention of many query rows (trees of drafted tokens, large groups) over the
// quantised paged cache, on the 5th-generation tensor cores.
//
// The mathematics, the numbers and the split of the work are kv_attention.cuh's;
// with many rows to a cache head the products and the softmax bound it, not HBM.
//
// One block to an SM, two tiles of 128 query rows, tiles of 128 tokens:
//   warps 0-15  softmax, two threads to a row, 64 columns each: scores from TMEM,
//               probabilities back into the same TMEM columns as f16 (the A operand
//               of P V). One thread to a row left the exponentials, the packing and
//               the TMEM loads of its one warp per scheduler to run one after another
//   warps 16-23 codes and their scales from global memory, decoded to f16 in shared
//               memory (128-byte swizzled rows; keys are K-major, values the same
//               bytes read as MN-major); loads run one tile ahead in registers
//   warp 24     issues tcgen05.mma: S = Q K^T and O += P V of each row tile in turn,
//               so that one row tile's products run under the other's softmax
//   warp 25     what a tile is relative to, which tokens are live and block FP8's key
//               scales. Each of the warps that decode did this for itself before, and
//               had no registers left for the loads ahead (MXFP8 525 -> 420 us)
// TMEM: two score tiles and two output tiles of 128 columns. The codes are decoded
// once for 256 rows, where the register path decodes them for every 32.
//
// Values are relative to one power of two for each of their scales' channel blocks. A tile
// whose scales lie too far apart for that (keys: for one power of two) is walked in several
// passes, each with the tokens that go together and the others hidden; the scales' warp
// says so, and every role walks passes. So the scale of a token does not touch another
// one's bits, whether a row sees it or not.
//
// A row's shift follows its maximum only when 32 probabilities sum to 2^kRise above it
// (the register path's rule, with less room above for more bits below in f16); then the
// softmax threads rescale their row of O in TMEM. The two threads of a row may use
// different shifts within a tile; at its end the lower half's probabilities are scaled.
#pragma once

#include "kv_attention.cuh"
#include "sm100.cuh"

#include <cstddef>

namespace brc {
uint32_t* gemm_status_ptr();  // gemm_sm100.cu: the sticky status word of bounded waits

namespace kvtc {

using namespace kvatt;
using namespace sm100;

constexpr int kTok = 128;
constexpr int kLift = 9;  // log2 of the factor that probabilities carry in f16
constexpr int kRise = 6;  // log2 of how far a sum of 32 of them may pass it
constexpr int kSoftWarps = 16, kLoadWarps = 8;
constexpr int kTcThreads = (kSoftWarps + kLoadWarps + 4) * 32;  // whole warpgroups: two warps idle
// Registers of a thread after setmaxnreg, by warpgroup; 4 x softmax + 2 x codes +
// products are no more than the 7 x 72 that the block was launched with. Block FP8's
// softmax, which holds the keys' scales too, takes them from the other warps (8 trees
// of 64 nodes over 16384 tokens: 480 -> 452 us), and so does NVFP4's (366 -> 355); MXFP8,
// whose codes need theirs, takes longer so (412 -> 427).
template <int KIND>
struct Regs {
  static constexpr bool kMx = KIND == BRC_STE_MXFP8;
  static constexpr uint32_t kSoft = kMx ? 80 : 88, kLoad = kMx ? 64 : 56, kMma = kMx ? 56 : 40;
  static_assert(4 * kSoft + 2 * kLoad + kMma <= 7 * 72, "registers of the launch");
};
// A pass's Meta is written when the scores of the pass two before are done, so that the
// softmax three before is over: a ring of four.
constexpr int kMeta = 4;
constexpr int kBlockBytes = 128 * 128;  // 128 rows of 64 f16, swizzled

struct alignas(16) Meta {
  float sk[kTok];  // block FP8
  int ek;            // MXFP8: what keys are relative to, as E8M0
  uint32_t ev;       // what values are relative to: a biased exponent to each channel block
  uint32_t all;      // every token of the tile is in this pass
  uint32_t more;     // another pass of the tile follows
  uint32_t live[4];  // which are: token 4 i + k, bit i of word k
};

template <int D>
struct alignas(128) Smem {
  uint8_t q[2][D / 64][kBlockBytes];
  uint8_t k[2][D / 64][kBlockBytes];
  uint8_t v[2][D / 64][kBlockBytes];
  Meta meta[kMeta];
  uint64_t meta_full[2], k_full[2], k_empty[2], v_full[2], v_empty[2];
  uint64_t q_full[2], s_full[2], p_full[2], o_full[2], drain;
  Place place;
  uint32_t tmem, abort;
  float pair[2][2][2][128];    // [turn][row tile][half][row]: shifts, then sums
  uint8_t sees[2][2][2][128];  // whether the row sees any of the half's places
  // What a thread's part of a row of O is relative to (a byte to a channel block). It
  // follows the values, where the row sees them, but not so low that O passes 2^100.
  uint32_t refs[2][2][128];
  uint32_t start[4];           // first pass of an item, one slot to an item as of odd
  // Numbers of items whose drafted values are not all finite: one slot to an item, as
  // the loads are at most two items ahead.
  uint32_t odd[4];
};

__device__ __forceinline__ void fence_proxy_smem() {
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
}
// D[tmem] (+)= A[tmem] * B[smem], f16 inputs.
__device__ __forceinline__ void mma_f16_ts(uint32_t d, uint32_t a, uint64_t bdesc, uint32_t idesc,
                                           uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
      "r"(a), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}
// kind::f16 with f16 operands, float32 accumulator; b_mn: B is MN-major.
constexpr uint32_t idesc_f16(uint32_t m, uint32_t n, bool b_mn) {
  return (1u << 4) | (b_mn ? 1u << 16 : 0u) | ((n >> 3) << 17) | ((m >> 4) << 24);
}
__device__ __forceinline__ void tmem_st16(uint32_t addr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
      "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(addr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
      "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
__device__ __forceinline__ void tmem_st_wait() {
  asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
}

// What every role walks through: the items of this block's share.
struct Walk {
  int64_t x, end, seq_start;
  int b, per_seq;
  // current item
  Seq seq;
  int item, head, row0, s_begin, s_end;
  int64_t item_start;
  __device__ __forceinline__ Walk(const Args& a, const Place& p)
      : x((int64_t)blockIdx.x * p.share), end(min(x + p.share, p.total)),
        per_seq(a.c.heads * a.row_blocks) {
    b = p.b;
    seq_start = p.before * per_seq;
  }
  __device__ __forceinline__ bool take(const Args& a) {
    if (x >= end) return false;
    seq = load_seq(a, b);
    item = (int)((x - seq_start) / seq.steps);
    item_start = seq_start + (int64_t)item * seq.steps;
    head = item / a.row_blocks;
    row0 = (item - head * a.row_blocks) * a.rows_per_block;
    s_begin = (int)(x - item_start);
    s_end = (int)min((int64_t)seq.steps, end - item_start);
    return true;
  }
  __device__ __forceinline__ void next() {
    x = item_start + s_end;
    if (s_end == seq.steps && item + 1 == per_seq) {
      seq_start += (int64_t)per_seq * seq.steps;
      ++b;
    }
  }
};

// ------------------------------------------------------------------ loading
// A scale below 2 times the largest code (448 of E4M3, 57344 of E5M2) times 2^this is
// within f16.
template <int FMT>
constexpr int kValueLift = FMT == BRC_FP8_E4M3 ? 6 : -1;

// Zero the codes of a word that stand for something not finite; true if there was one.
template <int FMT>
__device__ __forceinline__ bool clear_odd(uint32_t& w) {
  const uint32_t odd = FMT == BRC_FP8_E4M3 ? ((w & 0x7F7F7F7Fu) + 0x01010101u) & 0x80808080u
                                           : ((w & 0x7C7C7C7Cu) + 0x04040404u) & 0x80808080u;
  w &= ~((odd >> 7) * 0xFFu);
  return odd != 0u;
}

// A warp decodes 16 of a tile's tokens: lane (t, c) reads token 8 g + t, piece 4 i
// + c, for g < 2 and i < kHalves.
template <int KIND, int FMT, int D>
struct Loader {
  using S = Shape<KIND, D>;
  static constexpr int kHalves = S::kRowBytes / 64;
  static_assert(kHalves >= 1, "rows of at least 64 bytes");
  static constexpr int kG = kTok / kLoadWarps / 8;
  uint4 w[kG][kHalves];
  uint32_t s[kG][kHalves];  // scale byte(s) of the piece; values of block FP8: the row's scale

  // VALUES: block FP8 needs the row's scale too
  template <bool VALUES>
  __device__ __forceinline__ void fetch(const uint8_t* data, const void* scale,
                                        const int64_t (&row)[kG], int lane) {
#pragma unroll
    for (int g = 0; g < kG; ++g)
#pragma unroll
      for (int i = 0; i < kHalves; ++i) {
        w[g][i] = make_uint4(0u, 0u, 0u, 0u);
        s[g][i] = 0u;
        if (row[g] >= 0) {
          const int piece = 4 * i + (lane & 3);
          w[g][i] = ldg16(data + row[g] * S::kRowBytes + piece * 16);
          const uint8_t* sp = static_cast<const uint8_t*>(scale) + row[g] * S::kScales;
          if constexpr (KIND == BRC_STE_BLOCK_FP8) {
            if (VALUES)
              s[g][i] = __float_as_uint(__ldg(static_cast<const float*>(scale) + row[g]));
          } else if constexpr (KIND == BRC_STE_MXFP8 && D == 128) {  // one load for both pieces
            s[g][i] = (__ldg(reinterpret_cast<const uint32_t*>(sp)) >> (8 * (piece / 2))) & 0xFFu;
          } else if constexpr (KIND == BRC_STE_MXFP8) {
            s[g][i] = __ldg(sp + piece / 2);
          } else if constexpr (KIND == BRC_STE_NVFP4)
            s[g][i] = __ldg(reinterpret_cast<const uint16_t*>(sp + 2 * piece));
        }
      }
  }
  // Decode into a stage. `first`: token of the warp's first row; `refs`: what each
  // channel block is relative to (a byte); tokens 8 g + lane / 4 of the warp without
  // bit g of `on` become zero. ODD: of drafted tokens (from `drafted` on), what
  // is not finite becomes zero too, code by code or scale by scale; returns whether
  // there was any (the epilogue adds it to the rows that see it). VALUES:
  // of block FP8 times scale * 2^(kValueLift + 127 - ref), which rounds them to f16 once (as
  // the probabilities are). That factor on the probabilities instead, as on the scores,
  // has every softmax thread read every token's from shared memory, 16 bytes to each
  // lane (8 trees of 64 nodes over 16384 tokens: 498 us).
  template <bool ODD, bool VALUES>
  __device__ __forceinline__ bool decode(uint8_t* stage, int first, int lane, uint32_t refs,
                                         uint32_t on, int drafted) {
    bool any = false;
#pragma unroll
    for (int g = 0; g < kG; ++g) {
      const int t = first + 8 * g + (lane >> 2);
#pragma unroll
      for (int i = 0; i < kHalves; ++i) {
        const int piece = 4 * i + (lane & 3);
        uint32_t x[4] = {w[g][i].x, w[g][i].y, w[g][i].z, w[g][i].w};
        bool zero = !((on >> g) & 1u);
        const int ref = (int)((refs >> (8 * (piece / 2))) & 0xFFu);
        if constexpr (ODD) {
          if (t >= drafted && !zero) {
            if constexpr (KIND == BRC_STE_NVFP4) {  // a scale of 16 elements each
#pragma unroll
              for (int y = 0; y < 16; y += 8)
                if (((s[g][i] >> y) & 0x7Fu) == 0x7Fu) {
                  s[g][i] &= 0xFF00u >> y;
                  any = true;
                }
            } else {
              if constexpr (KIND == BRC_STE_MXFP8) zero = s[g][i] == 255u;
              else zero = !isfinite(__uint_as_float(s[g][i]));
              any |= zero;
#pragma unroll
              for (int y = 0; y < 4; ++y) any |= clear_odd<FMT>(x[y]);
            }
          }
        }
        if (zero) x[0] = x[1] = x[2] = x[3] = s[g][i] = 0u;
        uint32_t h[S::kFp4 ? 16 : 8];
        if constexpr (S::kFp4) {
          const uint32_t f0 = fp8x2_to_f16x2<BRC_FP8_E4M3>(__byte_perm(s[g][i], 0, 0x0000));
          const uint32_t f1 = fp8x2_to_f16x2<BRC_FP8_E4M3>(__byte_perm(s[g][i], 0, 0x0011));
#pragma unroll
          for (int y = 0; y < 4; ++y) {
            uint32_t q[4];
            e2m1x8_to_f16x8(x[y], q);
#pragma unroll
            for (int z = 0; z < 4; ++z) h[4 * y + z] = hmul2(q[z], y < 2 ? f0 : f1);
          }
        } else {
#pragma unroll
          for (int y = 0; y < 4; ++y) fp8x4_to_f16x4<FMT>(x[y], h[2 * y], h[2 * y + 1]);
          if constexpr (KIND == BRC_STE_MXFP8) {
            const uint32_t f = half2_pow2<true>((int)s[g][i], (int)s[g][i], ref);
#pragma unroll
            for (int y = 0; y < 8; ++y) h[y] = hmul2(h[y], f);
          } else if constexpr (VALUES) {
            constexpr int kDown = kValueLift<FMT> < 0 ? 2 : 0;  // (the reference may be 254)
            const float f = __uint_as_float(s[g][i]) * (kDown ? 0.25f : 1.f) *
                            __uint_as_float((uint32_t)(254 + kValueLift<FMT> + kDown - (int)(refs & 0xFFu)) << 23);
#pragma unroll
            for (int y = 0; y < 8; ++y) {
              const float2 u = __half22float2(*reinterpret_cast<const __half2*>(&h[y]));
              h[y] = half2_of(u.x * f, u.y * f);
            }
          }
        }
        // a piece is kUnits 16-byte units of a 64-element block's row
        constexpr int kUnits = S::kFp4 ? 4 : 2;
        const int unit = piece * kUnits;
        uint8_t* const dst = stage + (unit >> 3) * kBlockBytes + t * 128;
#pragma unroll
        for (int y = 0; y < kUnits; ++y)
          *reinterpret_cast<uint4*>(dst + ((((unit & 7) + y) ^ (t & 7)) << 4)) =
              make_uint4(h[4 * y], h[4 * y + 1], h[4 * y + 2], h[4 * y + 3]);
      }
    }
    return any;
  }
};

// The scales of a tile's tokens 4 lane .. + 3.
template <int KIND, int D>
struct Scales {
  using S = Shape<KIND, D>;
  uint4 e;

  __device__ __forceinline__ void fetch(const void* scale, int64_t row4) {
    e = make_uint4(0u, 0u, 0u, 0u);
    if (row4 >= 0) {
      if constexpr (KIND == BRC_STE_BLOCK_FP8) {
        e = ldg16(static_cast<const float*>(scale) + row4);
      } else if constexpr (KIND == BRC_STE_MXFP8) {
        const uint8_t* sp = static_cast<const uint8_t*>(scale) + row4 * S::kScales;
        if constexpr (D == 128) {
          e = ldg16(sp);
        } else {
          const uint2 v = __ldg(reinterpret_cast<const uint2*>(sp));
          e.x = v.x;
          e.y = v.y;
        }
      }
    }
  }
  // Token y's biased exponents, a byte to each channel block.
  __device__ __forceinline__ uint32_t bytes(int y) const {
    const uint32_t w[4] = {e.x, e.y, e.z, e.w};
    if constexpr (KIND == BRC_STE_BLOCK_FP8) return (w[y] >> 23) & 0xFFu;
    else if constexpr (D == 128) return w[y];
    else return (w[y / 2] >> (16 * (y & 1))) & 0xFFFFu;
  }
};

// Row of a token in the cache's arrays; -1: no such page.
__device__ __forceinline__ int64_t slot_of(const Args& a, int page, int64_t head_row, int token) {
  return page < 0 || page >= a.c.num_pages
             ? -1
             : (int64_t)((uint64_t)(uint32_t)page * a.page_rows) +
                   (head_row + (token & (a.c.page_size - 1)));
}

template <int KIND, int FMT, int D>
__global__ void __launch_bounds__(kTcThreads, 1) k_attend_tc(Args a, uint32_t* status) {
  using S = Shape<KIND, D>;
  extern __shared__ uint8_t raw[];
  Smem<D>& sm = *reinterpret_cast<Smem<D>*>(
      raw + ((1024u - (smem_u32(raw) & 1023u)) & 1023u));  // swizzled tiles: 1024-byte aligned
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  volatile uint32_t* const abort = &sm.abort;

  if (warp == kSoftWarps + kLoadWarps) {
    tmem_alloc(&sm.tmem, 512);
    tmem_relinquish();
  }
  if (warp == 0) {
    Place p;
    locate(a, a.c.heads * a.row_blocks, gridDim.x, blockIdx.x, -1, p);
    if (lane == 0) {
      sm.place = p;
      sm.abort = 0;
      sm.odd[0] = sm.odd[1] = sm.odd[2] = sm.odd[3] = 0;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        mbar_init(&sm.meta_full[i], 1);
        mbar_init(&sm.k_full[i], kLoadWarps);
        mbar_init(&sm.v_full[i], kLoadWarps);
        mbar_init(&sm.k_empty[i], 1);
        mbar_init(&sm.v_empty[i], 1);
        mbar_init(&sm.q_full[i], kSoftWarps / 2);
        mbar_init(&sm.s_full[i], 1);
        mbar_init(&sm.p_full[i], kSoftWarps / 2);
        mbar_init(&sm.o_full[i], 1);
      }
      mbar_init(&sm.drain, 1);
      fence_mbar_init();
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = sm.tmem;
  const uint32_t s_col[2] = {tmem, tmem + 128}, o_col[2] = {tmem + 256, tmem + 256 + D};
  Walk walk(a, sm.place);

  if (warp < kSoftWarps) {
    // ================================================================ softmax
    regs_inc<Regs<KIND>::kSoft>();
    const int r = warp >> 3, half = (warp >> 2) & 1;  // row tile; half of its columns
    const int mine = (warp & 3) * 32 + lane;
    const uint32_t lanes = (uint32_t)(warp & 3) << 21;  // 32 (warp % 4) lanes, in bits 16 ..
    const uint32_t sc = (r ? s_col[1] : s_col[0]) + lanes + 64 * half;
    const uint32_t oc = (r ? o_col[1] : o_col[0]) + lanes + (D / 2) * half;
    // channel block of this half's 16 columns c (block FP8: the only one)
    auto channel_block = [&](int c) { return KIND == BRC_STE_MXFP8 ? (D / 2 * half + 16 * c) / 32 : 0; };
    // The two warps of 32 rows meet once a pass. A warp that leaves early arrives
    // in its place, and the other one finds the abort flag at its next wait.
    const uint32_t pair_id = 1 + r * 4 + (warp & 3);
    auto meet = [&]() { asm volatile("barrier.cta.sync %0, 64;" ::"r"(pair_id) : "memory"); };
    auto leave = [&]() { asm volatile("barrier.cta.arrive %0, 64;" ::"r"(pair_id) : "memory"); };
    uint32_t pass = 0, number = 0, turn = 0;  // passes and items so far; times met
    uint32_t s_phase = 0, o_phase = 0;
    bool ok = true;
    for (; ok && walk.take(a); walk.next()) {
      ++number;
      const Seq seq = walk.seq;
      const int rows_left = a.rows - walk.row0;
      if (r != 0 && rows_left <= 128) continue;
      const int row = walk.row0 + r * 128 + mine, node = row / a.group;
      const bool valid = row < a.rows && node < seq.drafts;
      const int64_t at_row = ((int64_t)walk.b * a.draft + node) * a.hq + walk.head * a.group +
                             (row - node * a.group);
      // ---- this row of the queries, scaled by a power of two into f16
      float rowf;
      {
        const uint16_t* const src = static_cast<const uint16_t*>(a.q) + at_row * D;
        float top = 0.f;
        if (valid) {
#pragma unroll 4
          for (int i = 0; i < D / 8; ++i) {
            float f[8];
            const uint4 v = ldg16(src + 8 * i);
            if (a.q_f16) unpack<BRC_DTYPE_F16>(v, f);
            else unpack<BRC_DTYPE_BF16>(v, f);
#pragma unroll
            for (int y = 0; y < 8; ++y) top = fmaxf(top, fabsf(f[y]));
          }
        }
        const int k = min(max((int)(__float_as_uint(top) >> 23) - 127, -119), 127);
        // the factor of a score is not negative: its sign goes onto the query
        const float up = copysignf(__uint_as_float((uint32_t)(127 + 7 - k) << 23), a.scale_log2);
        rowf = fabsf(a.scale_log2) * __uint_as_float((uint32_t)(127 + k - 7) << 23);
#pragma unroll 4
        for (int i = half * (D / 16); i < (half + 1) * (D / 16); ++i) {
          uint4 y = make_uint4(0u, 0u, 0u, 0u);
          if (valid) {
            float f[8];
            const uint4 v = ldg16(src + 8 * i);
            if (a.q_f16) unpack<BRC_DTYPE_F16>(v, f);
            else unpack<BRC_DTYPE_BF16>(v, f);
            y = make_uint4(half2_of(f[0] * up, f[1] * up), half2_of(f[2] * up, f[3] * up),
                           half2_of(f[4] * up, f[5] * up), half2_of(f[6] * up, f[7] * up));
          }
          *reinterpret_cast<uint4*>(sm.q[r][i / 8] + mine * 128 + (((i & 7) ^ (mine & 7)) << 4)) = y;
        }
        fence_proxy_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&sm.q_full[r]);
      }
      float m = -INFINITY, l = 0.f;
      bool fresh = true;
      uint32_t& refs = sm.refs[r][half][mine];
      for (int j = walk.s_begin; j < walk.s_end;) {
        if (!(ok = __all_sync(0xFFFFFFFFu, mbar_wait(&sm.s_full[r], s_phase, abort, status, 1u)))) {
          leave();
          break;
        }
        s_phase ^= 1u;
        tc_fence_after();
        if (fresh) pass = sm.start[number & 3u];
        const Meta& meta = sm.meta[pass++ % kMeta];
        const bool more = meta.more;
        const int64_t t0 = (int64_t)j * kTok;
        // (a factor of zero, of a scale of zero or by underflow, would make NaN of the
        // hidden places' minus infinity; a score, below 2^40, times 2^-126 is nothing)
        float f = KIND == BRC_STE_MXFP8 ? rowf * e8m0_value(meta.ek) : rowf;
        if (f < 0x1p-126f) f = 0x1p-126f;
        const bool masked = t0 + kTok > seq.context || !meta.all;
        uint32_t vis[2] = {0xFFFFFFFFu, 0xFFFFFFFFu};
        if (masked) {
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            vis[c] = 0;
            for (int i = 0; i < 32; ++i) {
              const int t = 64 * half + 32 * c + i;
              const int64_t n = t0 + t - seq.context;
              bool see = valid && ((meta.live[t & 3] >> (t >> 2)) & 1u);
              if (see && n >= 0)
                see = a.tree ? a.tree[walk.b * a.tree_stride + (int64_t)node * a.draft + n] != 0
                             : n <= node;
              vis[c] |= (see ? 1u : 0u) << i;
            }
          }
        }
        __syncwarp();
        // 32 scores in units of the row's factor; masked ones -inf
        auto take = [&](const uint32_t (&x)[32], int c, float2 (&u)[16]) {
#pragma unroll
          for (int i = 0; i < 16; ++i)
            u[i] = make_float2(__uint_as_float(x[2 * i]), __uint_as_float(x[2 * i + 1]));
          if constexpr (KIND == BRC_STE_BLOCK_FP8) {
#pragma unroll
            for (int i = 0; i < 16; i += 2) {
              const float4 g = *reinterpret_cast<const float4*>(&meta.sk[64 * half + 32 * c + 2 * i]);
              u[i] = __fmul2_rn(u[i], make_float2(g.x, g.y));
              u[i + 1] = __fmul2_rn(u[i + 1], make_float2(g.z, g.w));
            }
          }
          if (masked) {
            const uint32_t bits = c ? vis[1] : vis[0];
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              if (!((bits >> (2 * i)) & 1u)) u[i].x = -INFINITY;
              if (!((bits >> (2 * i + 1)) & 1u)) u[i].y = -INFINITY;
            }
          }
        };
        // O times g, and relative to `to`; the products up to here are done: S came after
        auto scale_o = [&](float g, uint32_t from, uint32_t to) {
#pragma unroll 1
          for (int c = 0; c < D / 32; ++c) {  // this thread's half of the columns
            uint32_t x[16];
            tmem_ld16(oc + 16 * c, x);
            tmem_ld_wait16(x);
            const int shift = 8 * channel_block(c);
            const int by = (int)((from >> shift) & 0xFFu) - (int)((to >> shift) & 0xFFu);
            // (the two may be further apart than one float32 exponent)
            const int near = max(by, -127);
            const float h = g * kv::pow2i(near - near / 2), h2 = kv::pow2i(near / 2);
#pragma unroll
            for (int i = 0; i < 16; ++i) x[i] = __float_as_uint(__uint_as_float(x[i]) * h * h2);
            tmem_st16(oc + 16 * c, x);
          }
        };
        // `to` no lower than what keeps O times g, relative to `from`, within 2^100. (What a row
        // adds relative to less than its O is then too large by the difference, but O is 2^100,
        // and that at most 2^18 a token.)
        auto low = [&](float g, uint32_t from, uint32_t& to) {
#pragma unroll 1
          for (int c = 0; c < D / 32; ++c) {
            uint32_t x[16];
            tmem_ld16(oc + 16 * c, x);
            tmem_ld_wait16(x);
            float most = 0.f;
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              const float y = fabsf(__uint_as_float(x[i]) * g);
              if (y < INFINITY) most = fmaxf(most, y);
            }
            const int shift = 8 * channel_block(c);
            const int is = (int)((to >> shift) & 0xFFu);
            const int least = (int)((from >> shift) & 0xFFu) + (int)(__float_as_uint(most) >> 23) - 227;
            if (most > 0.f && least > is) to += (uint32_t)(least - is) << shift;
          }
        };
        // This half's shift: the row's, until a score is far above it (and at first the
        // half's maximum). Shifts are whole numbers: less the lift they are exact, so
        // that the row's log-sum-exp does not get their rounding.
        float own = m;
        if (fresh) {
          float top = -INFINITY;
#pragma unroll 1
          for (int c = 0; c < 2; ++c) {
            uint32_t x[32];
            float2 u[16];
            tmem_ld32(sc + 32 * c, x);
            tmem_ld_wait();
            reg_bind32(x);
            take(x, c, u);
#pragma unroll
            for (int i = 0; i < 16; ++i) top = fmaxf(top, fmaxf(u[i].x, u[i].y));
          }
          // A shift beyond 2^18 is a rounded score, and the unrounded product of that score
          // and its factor may be far off it: left to the chunk, which rounds the product
          top = ceilf(top * f);
          if (fabsf(top) < 0x1p18f) own = top;
        }
        // Probabilities carry the factor 2^kLift. Their sum over 32 tokens may pass it by
        // 2^kRise (32 scores at the shift reach 2^5), so that none leaves the range of f16,
        // and the small ones keep the bits that are left. (The values' scales are no part of
        // it: a row's sum does not depend on them.)
        float base = kLift - (own == -INFINITY ? 0.f : own);
        constexpr float most = (float)(1 << (kLift + kRise));
        float2 l2 = make_float2(0.f, 0.f);
        // this tile's probabilities so far (`upto` groups of 32 columns) times g
        auto scale_p = [&](int upto, float g) {
          // (g as f16 would be zero below 2^-25, where large ones are still needed)
          tmem_st_wait();
#pragma unroll 1
          for (int b = 0; b < upto; ++b) {
            uint32_t z[16];
            tmem_ld16(sc + 16 * b, z);
            tmem_ld_wait16(z);
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              const float2 y = __half22float2(*reinterpret_cast<const __half2*>(&z[i]));
              z[i] = half2_of(y.x * g, y.y * g);
            }
            tmem_st16(sc + 16 * b, z);
          }
        };
        auto exps = [&](float2 (&u)[16], float by, float add) {
          float2 t = make_float2(0.f, 0.f);
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            u[i] = __ffma2_rn(u[i], make_float2(by, by), make_float2(add, add));
            u[i] = make_float2(ex2(u[i].x), ex2(u[i].y));
            t = __fadd2_rn(t, u[i]);
          }
          return t;
        };
        // 32 scores to probabilities, into columns that their scores have left
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          uint32_t x[32];
          float2 u[16];
          tmem_ld32(sc + 32 * c, x);
          tmem_ld_wait();
          reg_bind32(x);
          take(x, c, u);
          float2 t;
          float by = f, add = base;
#pragma unroll 1
          for (bool looked = false;; looked = true) {
            t = exps(u, by, add);
            // a score far above the shift shows in the sum; a row that has seen nothing so
            // far has the shift 0, below which its scores may vanish: it always looks
            if (looked || !__any_sync(0xFFFFFFFFu, t.x + t.y > most || own == -INFINITY)) break;
            tmem_ld32(sc + 32 * c, x);
            tmem_ld_wait();
            reg_bind32(x);
            take(x, c, u);
            float top = -INFINITY;
#pragma unroll
            for (int i = 0; i < 16; ++i) top = fmaxf(top, fmaxf(u[i].x, u[i].y));
            top = top == -INFINITY ? top : ceilf(top * f);
            const float nm = fmaxf(own, top), g = nm == own || own == -INFINITY ? 1.f : ex2(own - nm);
            own = nm;
            base = kLift - (own == -INFINITY ? 0.f : own);
            l2 = __fmul2_rn(l2, make_float2(g, g));
            scale_p(c, g);
            // the rounded product (the compiler may join packed operations)
            const float down = own == -INFINITY ? 0.f : -own;
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              u[i].x = __fadd_rn(__fmul_rn(u[i].x, f), down);
              u[i].y = __fadd_rn(__fmul_rn(u[i].y, f), down);
            }
            by = 1.f;
            add = kLift;
          }
          l2 = __fadd2_rn(l2, t);
          uint32_t p[16];
#pragma unroll
          for (int i = 0; i < 16; ++i) p[i] = half2_of(u[i].x, u[i].y);
          tmem_st16(sc + 16 * c, p);
        }
        // ---- the halves agree on the row's shift
        sm.pair[turn][r][half][mine] = own;
        bool sees = !masked || (vis[0] | vis[1]) != 0u;
        if (masked && KIND != BRC_STE_NVFP4) sm.sees[turn][r][half][mine] = sees;
        meet();
        const float nm = fmaxf(own, sm.pair[turn][r][half ^ 1][mine]);
        const bool moved = KIND != BRC_STE_NVFP4 && (fresh || meta.ev != refs);
        float part = (l2.x + l2.y) * (1.f / (1 << kLift));
        if (__any_sync(0xFFFFFFFFu, nm != own || nm != m || moved)) {
          const float gp = nm == own || nm == -INFINITY ? 1.f : ex2(own - nm);
          const float go = nm == m || nm == -INFINITY ? 1.f : ex2(m - nm);
          if (__any_sync(0xFFFFFFFFu, gp != 1.f)) scale_p(2, gp);
          uint32_t from = 0, to = 0;
          if (moved) {
            from = to = refs;
            if (masked) sees |= sm.sees[turn][r][half ^ 1][mine] != 0;
            if (sees || fresh) to = meta.ev;
          }
          if (!fresh && __any_sync(0xFFFFFFFFu, __vsubus4(from, to) & 0xE0E0E0E0u)) low(go, from, to);
          if (moved) refs = to;
          if (!fresh && __any_sync(0xFFFFFFFFu, go != 1.f || to != from)) scale_o(go, from, to);
          part *= gp;
          l *= go;
          m = nm;
        }
        turn ^= 1u;
        l += part;
        tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&sm.p_full[r]);
        fresh = false;
        if (!more) ++j;
      }
      if (!ok) break;
      // ---- the item's output
      if (!(ok = __all_sync(0xFFFFFFFFu, mbar_wait(&sm.o_full[r], o_phase, abort, status, 1u)))) {
        leave();
        break;
      }
      // the row's sum, of both halves (this turn's slots are free: the other half has
      // read them before it met this one last)
      sm.pair[turn][r][half][mine] = l;
      meet();
      l = half ? sm.pair[turn][r][0][mine] + l : l + sm.pair[turn][r][1][mine];
      turn ^= 1u;
      o_phase ^= 1u;
      tc_fence_after();
      const bool whole = walk.s_begin == 0 && walk.s_end == seq.steps;
      const bool none = !valid || l == 0.f;
      const float so = whole ? (none ? 0.f : 1.f / l) : 1.f / kSumUp;
      const bool odd = sm.odd[number & 3u] == number && !none;
      const int64_t slot = 2 * (int64_t)blockIdx.x + (walk.s_begin > 0 ? 0 : 1);
      const int rr = r * 128 + mine;
#pragma unroll 1
      for (int c = 0; c < D / 32; ++c) {
        uint32_t x[16];
        const int col = (D / 2) * half + 16 * c;
        __syncwarp();
        tmem_ld16(oc + 16 * c, x);
        tmem_ld_wait16(x);
        float mul = so * (1.f / (1 << kLift));
        if constexpr (KIND != BRC_STE_NVFP4) {
          constexpr int kOff = KIND == BRC_STE_MXFP8 ? 0 : kValueLift<FMT>;
          mul *= exp2f((float)((int)((refs >> (8 * channel_block(c))) & 0xFFu) - 127 - kOff));
        }
        float o[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) o[i] = none ? 0.f : __uint_as_float(x[i]) * mul;
        if (odd) {  // what was left out of the product, where this row sees it
          const int32_t* const table = a.table + walk.b * a.table_stride;
          for (int64_t t = max((int64_t)walk.s_begin * kTok, (int64_t)seq.context);
               t < min((int64_t)walk.s_end * kTok, (int64_t)seq.total); ++t) {
            const int64_t n = t - seq.context;
            if (!(a.tree ? a.tree[walk.b * a.tree_stride + (int64_t)node * a.draft + n] != 0 : n <= node))
              continue;
            const int64_t page = table[t >> a.page_shift];
            if (page < 0 || page >= a.c.num_pages) continue;
            const int64_t src = page * a.page_rows + (int64_t)walk.head * a.c.page_size +
                                (t & (a.c.page_size - 1));
            for (int i = 0; i < 16; ++i) {
              const float v = value_at<KIND, FMT, D>(a.c, src, col + i);
              if (!isfinite(v)) o[i] += v;
            }
          }
        }
        if (row < a.rows) {
          if (whole) {
            uint32_t y[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              if (a.q_f16) {
                y[i] = half2_of(o[2 * i], o[2 * i + 1]);
              } else {
                const __nv_bfloat162 h = __floats2bfloat162_rn(o[2 * i], o[2 * i + 1]);
                y[i] = *reinterpret_cast<const uint32_t*>(&h);
              }
            }
            uint16_t* const dst = static_cast<uint16_t*>(a.out) + at_row * D + col;
            stg16(dst, make_uint4(y[0], y[1], y[2], y[3]));
            stg16(dst + 8, make_uint4(y[4], y[5], y[6], y[7]));
          } else {
            float* const dst = a.part_o + (slot * a.rows_per_block + rr) * D + col;
#pragma unroll
            for (int i = 0; i < 16; i += 4)
              *reinterpret_cast<float4*>(dst + i) = make_float4(o[i], o[i + 1], o[i + 2], o[i + 3]);
          }
        }
      }
      if (row < a.rows && half == 0) {
        if (whole) {
          if (a.lse) a.lse[at_row] = none ? -INFINITY : (m + log2f(l)) * 0.6931471805599453f;
        } else {
          float* const ml = a.part_ml + (slot * a.rows_per_block + rr) * 2;
          ml[0] = valid ? m : -INFINITY;
          ml[1] = valid ? l : 0.f;
        }
      }
      tc_fence_before();  // O is read before the next item's products overwrite it
    }
  } else if (warp < kSoftWarps + kLoadWarps) {
    // ================================================================ codes
    regs_dec<Regs<KIND>::kLoad>();
    const int lw = warp - kSoftWarps, first = kTok / kLoadWarps * lw;
    uint32_t pass = 0, number = 0;
    bool ok = true;
    for (; ok && walk.take(a); walk.next()) {
      ++number;
      const Seq seq = walk.seq;
      const int32_t* const table = a.table + walk.b * a.table_stride;
      const int64_t head_row = (int64_t)walk.head * a.c.page_size;
      constexpr int kG = Loader<KIND, FMT, D>::kG;
      Loader<KIND, FMT, D> k, v;
      // a tile's pages, fetched a tile before they are needed
      int pages[kG];
      int64_t row[kG];
      auto token = [&](int j, int g) { return j * kTok + first + 8 * g + (lane >> 2); };
      auto pages_of = [&](int j) {
#pragma unroll
        for (int g = 0; g < kG; ++g) {
          const int t = token(j, g);
          pages[g] = j < walk.s_end && t < seq.total ? __ldg(table + (t >> a.page_shift)) : -1;
        }
      };
      auto rows_of = [&](int j) {
#pragma unroll
        for (int g = 0; g < kG; ++g) row[g] = slot_of(a, pages[g], head_row, token(j, g));
      };
      pages_of(walk.s_begin);
      rows_of(walk.s_begin);
      k.template fetch<false>(a.c.k_data, a.c.k_scale, row, lane);
      pages_of(walk.s_begin + 1);
      for (int j = walk.s_begin; j < walk.s_end; ++pass) {
        const uint32_t st = pass & 1u, use = (pass >> 1) & 1u;
        const int64_t t0 = (int64_t)j * kTok;
        const bool drafted = t0 + kTok > seq.context;
        const int from = (int)max((int64_t)0, seq.context - t0);
        v.template fetch<true>(a.c.v_data, a.c.v_scale, row, lane);
        // (the scales' warp has waited for the key stage)
        if (!(ok = __all_sync(0xFFFFFFFFu, mbar_wait(&sm.meta_full[st], use, abort, status, 1u)))) break;
        const Meta& meta = sm.meta[pass % kMeta];
        const uint32_t ek = (uint32_t)meta.ek * 0x01010101u, ev = meta.ev;
        const bool more = meta.more;
        uint32_t on = 0;
#pragma unroll
        for (int g = 0; g < kG; ++g) {
          const int t = first + 8 * g + (lane >> 2);
          on |= ((meta.live[t & 3] >> (t >> 2)) & 1u) << g;
        }
        k.template decode<false, false>(sm.k[st][0], first, lane, ek, on, kTok);
        fence_proxy_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&sm.k_full[st]);
        if (more) {
          k.template fetch<false>(a.c.k_data, a.c.k_scale, row, lane);
        } else if (j + 1 < walk.s_end) {
          rows_of(j + 1);
          k.template fetch<false>(a.c.k_data, a.c.k_scale, row, lane);
          pages_of(j + 2);
        }
        if (!(ok = __all_sync(0xFFFFFFFFu, mbar_wait(&sm.v_empty[st], use ^ 1u, abort, status, 1u)))) break;
        if (drafted) {
          if (v.template decode<true, true>(sm.v[st][0], first, lane, ev, on, from)) sm.odd[number & 3u] = number;
        } else {
          v.template decode<false, true>(sm.v[st][0], first, lane, ev, on, kTok);
        }
        fence_proxy_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&sm.v_full[st]);
        if (!more) ++j;
      }
    }
  } else {
    // ================================================================ products
    regs_dec<Regs<KIND>::kMma>();
    if (warp == kSoftWarps + kLoadWarps) {
    uint32_t pass = 0, q_phase = 0, p_phase[2] = {0, 0}, q_phase1 = 0;
    bool ok = true;
    constexpr uint32_t kIdS = idesc_f16(128, kTok, false), kIdO = idesc_f16(128, D, true);
    const uint64_t hi_k = desc_sw128_hi();
    auto wait = [&](uint64_t* bar, uint32_t parity) {
      return __all_sync(0xFFFFFFFFu, mbar_wait(bar, parity, abort, status, 1u));
    };
    auto scores = [&](int r, uint32_t st) {  // S_r = Q_r K^T
      if (elect_lane()) {
#pragma unroll
        for (int i = 0; i < D / 16; ++i) {
          const uint32_t off = (i / 4) * kBlockBytes + (i % 4) * 32;
          mma_bf16(s_col[r], hi_k | desc_sw128_lo(smem_u32(sm.q[r][0]) + off),
                   hi_k | desc_sw128_lo(smem_u32(sm.k[st][0]) + off), kIdS, i > 0);
        }
        tc_commit(&sm.s_full[r]);
      }
      __syncwarp();
    };
    for (; ok && walk.take(a); walk.next()) {
      const int tiles = a.rows - walk.row0 > 128 ? 2 : 1;
      for (int r = 0; ok && r < tiles; ++r) {
        ok = wait(&sm.q_full[r], r ? q_phase1 : q_phase);
        if (r) q_phase1 ^= 1u;
        else q_phase ^= 1u;
        if (ok && r == 0) ok = wait(&sm.k_full[pass & 1u], (pass >> 1) & 1u);
        tc_fence_after();
        if (ok) scores(r, pass & 1u);
      }
      if (ok && elect_lane()) tc_commit(&sm.k_empty[pass & 1u]);
      __syncwarp();
      bool fresh = true;
      for (int j = walk.s_begin; ok && j < walk.s_end; ++pass, fresh = false) {
        const uint32_t st = pass & 1u, nx = (pass + 1) & 1u;
        if (!sm.meta[pass % kMeta].more) ++j;  // (written before this pass's keys)
        const bool last = j == walk.s_end;
        for (int r = 0; ok && r < tiles; ++r) {
          ok = wait(&sm.p_full[r], p_phase[r]);
          p_phase[r] ^= 1u;
          if (ok && r == 0) ok = wait(&sm.v_full[st], (pass >> 1) & 1u);
          tc_fence_after();
          if (!ok) break;
          if (elect_lane()) {
#pragma unroll
            for (int i = 0; i < kTok / 16; ++i)  // 16 tokens: 8 columns of P (each half's at its own start), 16 rows of V
              mma_f16_ts(o_col[r], s_col[r] + 64 * (i / 4) + 8 * (i % 4),
                         smem_desc(smem_u32(sm.v[st][0]) + 2048 * i, kBlockBytes, 1024, 2), kIdO,
                         !fresh || i > 0);
            if (last) tc_commit(&sm.o_full[r]);
            if (r + 1 == tiles) tc_commit(&sm.v_empty[st]);
          }
          __syncwarp();
          if (!last) {
            if (r == 0) ok = wait(&sm.k_full[nx], ((pass + 1) >> 1) & 1u);
            tc_fence_after();
            if (!ok) break;
            scores(r, nx);
            if (r + 1 == tiles) {
              if (elect_lane()) tc_commit(&sm.k_empty[nx]);
              __syncwarp();
            }
          }
        }
      }
    }
    // all products are done before TMEM is given back (after a timeout too)
    if (elect_lane()) tc_commit(&sm.drain);
    __syncwarp();
    uint32_t none = 0;
    mbar_wait(&sm.drain, 0u, &none, status, 1u);
    } else if (warp == kSoftWarps + kLoadWarps + 1) {
      // ============================================================== scales
      uint32_t pass = 0, number = 0;
      bool ok = true;
      for (; ok && walk.take(a); walk.next()) {
        ++number;
        const Seq seq = walk.seq;
        const int32_t* const table = a.table + walk.b * a.table_stride;
        const int64_t head_row = (int64_t)walk.head * a.c.page_size;
        Scales<KIND, D> k, v;
        // pages a tile before the scales, scales a tile before they are needed
        auto page_of = [&](int j) {
          const int t = j * kTok + 4 * lane;
          return j < walk.s_end && t < seq.total ? __ldg(table + (t >> a.page_shift)) : -1;
        };
        int page = page_of(walk.s_begin);
        int64_t row = slot_of(a, page, head_row, walk.s_begin * kTok + 4 * lane);
        k.fetch(a.c.k_scale, row);
        v.fetch(a.c.v_scale, row);
        page = page_of(walk.s_begin + 1);
        constexpr int kBlocks = kScaleBlocks<KIND, D>;
        // what values are relative to, at first: the lowest
        uint32_t refs[1] = {kSpan<KIND> * (kBlocks == 1 ? 1u : kBlocks == 2 ? 0x0101u : 0x01010101u)};
        bool fresh = true;
        for (int j = walk.s_begin; ok && j < walk.s_end; ++j) {
          const int there = (int)min((int64_t)kTok, seq.total - (int64_t)j * kTok) - 4 * lane;
          const int live4 = row < 0 ? 0 : min(max(there, 0), 4);
          uint32_t left = (1u << live4) - 1u, take, more;
          do {
            take = left;
            int ek = 0;
            if constexpr (KIND != BRC_STE_NVFP4) {
              uint32_t vb[4][1], km[4] = {0u, 0u, 0u, 0u}, hi = 0, lo = 255;
              constexpr uint32_t kFar = kSpan<KIND>;
              const Near<KIND == BRC_STE_MXFP8 ? kFar : 15> near(refs[0]);
              bool off = false;
#pragma unroll
              for (int y = 0; y < 4; ++y) {
                vb[y][0] = v.bytes(y);
                if constexpr (KIND == BRC_STE_MXFP8) km[y] = top_byte(k.bytes(y));
                if ((left >> y) & 1u) {
                  off |= KIND == BRC_STE_MXFP8 ? !near(vb[y][0]) : refs[0] - vb[y][0] > kFar;
                  hi = max(hi, km[y]);
                  lo = min(lo, km[y]);
                }
              }
              if constexpr (KIND == BRC_STE_MXFP8) {
                hi = __reduce_max_sync(0xFFFFFFFFu, hi);
                off |= lo + kFar < hi;
              }
              ek = (int)hi;
              if (__any_sync(0xFFFFFFFFu, off))
                ek = (int)choose<kFar, kFloor<KIND, FMT>, kBlocks>(vb, km, left, take, refs);
            }
            more = __any_sync(0xFFFFFFFFu, (left & ~take) != 0u);
            left &= ~take;
            const uint32_t st = pass & 1u, use = (pass >> 1) & 1u;
            if (!(ok = __all_sync(0xFFFFFFFFu,
                                  mbar_wait(&sm.k_empty[st], use ^ 1u, abort, status, 1u))))
              break;
            Meta& meta = sm.meta[pass % kMeta];
            if constexpr (KIND == BRC_STE_BLOCK_FP8)
              *reinterpret_cast<uint4*>(&meta.sk[4 * lane]) = k.e;
            uint32_t bal[4];
#pragma unroll
            for (int y = 0; y < 4; ++y) bal[y] = __ballot_sync(0xFFFFFFFFu, (take >> y) & 1u);
            if (lane == 0) {
              meta.ek = ek;
              meta.ev = refs[0];
              meta.more = more;
#pragma unroll
              for (int y = 0; y < 4; ++y) meta.live[y] = bal[y];
              meta.all = (bal[0] & bal[1] & bal[2] & bal[3]) == 0xFFFFFFFFu;
              if (fresh) sm.start[number & 3u] = pass;
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(&sm.meta_full[st]);
            ++pass;
            fresh = false;
          } while (more);
          if (!ok) break;
          row = slot_of(a, page, head_row, (j + 1) * kTok + 4 * lane);
          k.fetch(a.c.k_scale, row);
          v.fetch(a.c.v_scale, row);
          page = page_of(j + 2);
        }
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == kSoftWarps + kLoadWarps) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}

static_assert(sizeof(Meta) % 16 == 0 && offsetof(Meta, sk) == 0, "16-byte accesses");
static_assert(offsetof(Smem<128>, meta) % 16 == 0 && offsetof(Smem<128>, k) % 1024 == 0 &&
                  offsetof(Smem<128>, v) % 1024 == 0 && offsetof(Smem<64>, v) % 1024 == 0,
              "swizzled tiles");

template <int KIND, int FMT, int D>
int launch_tc(const Args& a, int blocks, cudaStream_t st) {
  constexpr int bytes = (int)sizeof(Smem<D>) + 1024;
  if (const int rc = check_cuda(cudaFuncSetAttribute(
          k_attend_tc<KIND, FMT, D>, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes)))
    return rc;
  k_attend_tc<KIND, FMT, D><<<blocks, kTcThreads, bytes, st>>>(a, gemm_status_ptr());
  if (const int rc = check_launch()) return rc;
  return launch_join<D>(a, blocks, st);
}

}  // namespace kvtc
}  // namespace brc
