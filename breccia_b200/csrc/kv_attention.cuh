// Attention of a few new tokens (one, or a tree of drafted ones) over the
// quantised paged cache.
//
//   s_ij = scale q_i . k_j,  out_i = sum_j softmax_j(s_ij) v_j  over visible j
//
// The query rows of one sequence and one cache head (draft x hq / heads) share
// every key and value, so the codes are read once for all of them: HBM bounds
// single tokens and small trees. One pass with a running maximum and sum.
//
// Layout. A warp takes 16 tokens at a time straight from global memory into
// the operand fragments of m16n8k16: which head elements stand at which place
// of a fragment is free as long as both operands agree, so a lane's fragment
// words are 16 contiguous bytes of a row, with no shared memory and no
// shuffles between load and product.
//   keys   (B of Q K^T): lane (r, c) holds token r, bytes 64 i + 16 c .. + 15
//   values (B of P V):   lane (r, c) holds tokens 2c, 2c+1, 2c+8, 2c+9, bytes
//                        16 r .. + 15; pairs of tokens are byte permutes
// The score fragment is the probability fragment (A of P V) as it stands.
//
// Numbers. FP8 and FP4 codes are exact in f16. Queries are scaled per row by a
// power of two into f16 (elements below 2^-21 of the row's largest lose bits).
// Key scales: block FP8 multiplies the score; MXFP8's per-block powers of two
// go onto the codes relative to the token's largest, which multiplies the
// score; NVFP4's E4M3 scales times E2M1 codes are exact in f16. Value scales
// likewise, with the largest seen so far by the warp (a power of two) taken
// out, so that f16 holds probability x scale: 11 bits each, against the 8 of a
// bf16 output. Scores, sums, the running maximum and the output are float32.
//
// Work split. The steps of 16 tokens of all (sequence, cache head, row block)
// items are cut into equal shares, one per block, whatever the lengths: the
// lengths stay on the device and ragged batches balance. A block that holds
// only part of an item leaves its sums in the workspace, and a second kernel
// joins the parts in a fixed order.
#pragma once

#include "kv_codec.cuh"
#include "launch.h"

namespace brc {
namespace kvatt {

constexpr int kThreads = 128;
constexpr int kWarps = kThreads / 32;
constexpr float kGrow = 8.f;  // a row's shift follows its maximum when it is this far (log2) behind

struct Args {
  brc_kv_cache c;
  const void* q;
  int q_f16, batch, draft, hq, group, rows;  // rows = draft * group
  const int32_t* table;
  int64_t table_stride;
  int table_pages, page_shift;
  const int32_t* context;
  const int32_t* drafts;
  const uint8_t* tree;
  int64_t tree_stride;
  float scale_log2;
  void* out;
  float* lse;
  float* part_o;   // (2 * blocks, rows per block, d)
  float* part_ml;  // (2 * blocks, rows per block, 2)
  int row_warps, row_blocks, rows_per_block, min_share;
};

struct Seq {
  int context, drafts, total;  // tokens
  int steps;                   // of 16 tokens, at least one
};
__device__ __forceinline__ Seq load_seq(const Args& a, int b) {
  Seq s;
  const int64_t cap = (int64_t)a.table_pages << a.page_shift;
  const int ctx = max(a.context[b], 0);
  s.drafts = a.drafts ? min(max(a.drafts[b], 0), a.draft) : a.draft;
  s.context = (int)min((int64_t)ctx, cap);
  s.total = (int)min((int64_t)ctx + s.drafts, cap);
  s.steps = max((int)(((int64_t)s.total + 15) >> 4), 1);
  return s;
}

// Where a block starts: found by one warp from the lengths.
struct Place {
  int64_t total, share;  // steps over all items, and per block
  int64_t before;        // sum of steps of the sequences before b (per item)
  int b;
};
// The sequence that holds step x of `total` (x < 0: only the total and the
// steps before sequence `want`). Every lane of a warp calls it.
__device__ __forceinline__ void locate(const Args& a, int per_seq, int blocks, int block,
                                       int want, Place& p) {
  const int lane = threadIdx.x & 31;
  const int per = (a.batch + 31) / 32;
  const int b0 = min(lane * per, a.batch), b1 = min(b0 + per, a.batch);
  int64_t mine = 0;
  for (int b = b0; b < b1; ++b) mine += load_seq(a, b).steps;
  int64_t incl = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t v = __shfl_up_sync(0xFFFFFFFFu, incl, o);
    if (lane >= o) incl += v;
  }
  p.total = __shfl_sync(0xFFFFFFFFu, incl, 31) * per_seq;
  p.share = max((p.total + blocks - 1) / blocks, (int64_t)a.min_share);
  const int64_t x = block * p.share;
  const bool holds = want >= 0 ? (want >= b0 && want < b1)
                               : (x >= (incl - mine) * per_seq && x < incl * per_seq);
  const unsigned vote = __ballot_sync(0xFFFFFFFFu, holds);
  int b = b0;
  int64_t before = incl - mine;
  if (holds) {
    for (; b < b1; ++b) {
      const int n = load_seq(a, b).steps;
      if (want >= 0 ? b == want : x < (before + n) * per_seq) break;
      before += n;
    }
  }
  const int src = vote ? __ffs(vote) - 1 : 0;
  p.b = __shfl_sync(0xFFFFFFFFu, b, src);
  p.before = __shfl_sync(0xFFFFFFFFu, before, src);
}

__device__ __forceinline__ void mma(float (&d)[4], const uint4& a, uint32_t b0, uint32_t b1) {
  asm(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
      "{%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a.x), "r"(a.y), "r"(a.z), "r"(a.w), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t hmul2(uint32_t a, uint32_t b) {
  const __half2 r = __hmul2(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&b));
  return *reinterpret_cast<const uint32_t*>(&r);
}
__device__ __forceinline__ uint32_t half2_of(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// 2^-n as f16 bits for n >= 0 (0 below the subnormals); n < 0 stands for infinity.
__device__ __forceinline__ uint32_t half_pow2_neg(int n) {
  if (n < 0) return 0x7C00u;
  return n < 15 ? (uint32_t)(15 - n) << 10 : n < 25 ? 1u << (24 - n) : 0u;
}
// E8M0 byte to float32 (255 as the casts read it: infinity).
__device__ __forceinline__ float e8m0_value(uint32_t e) {
  return e == 0 ? __uint_as_float(0x00400000u) : __uint_as_float(e << 23);
}
template <int N>
__device__ __forceinline__ void ldg_words(const void* p, uint32_t* w) {
  if constexpr (N >= 4) {
#pragma unroll
    for (int i = 0; i < N / 4; ++i) {
      const uint4 v = ldg16(static_cast<const char*>(p) + 16 * i);
      w[4 * i] = v.x; w[4 * i + 1] = v.y; w[4 * i + 2] = v.z; w[4 * i + 3] = v.w;
    }
  } else if constexpr (N == 2) {
    const uint2 v = __ldg(static_cast<const uint2*>(p));
    w[0] = v.x; w[1] = v.y;
  } else {
    w[0] = __ldg(static_cast<const uint32_t*>(p));
  }
}

template <int KIND, int D>
struct Shape {
  static constexpr bool kFp4 = KIND == BRC_STE_NVFP4;
  static constexpr int kRowBytes = kv::row_bytes(KIND, D);
  static constexpr int kScales = kv::row_scales(KIND, D);
  static constexpr int kKeyWords = kRowBytes / 16;    // per lane and token
  static constexpr int kValWords = kRowBytes / 32;    // per lane and token
  static constexpr int kSteps = D / 16;               // products along the head
  static constexpr int kTiles = D / 8;                // output tiles of 8 elements
  static constexpr int kKeyChunk = kKeyWords < 4 ? kKeyWords : 4;  // words loaded together
  static constexpr int kValChunk = kValWords < 4 ? kValWords : 4;
  static constexpr int kKeyScaleWords = KIND == BRC_STE_MXFP8 ? (D + 127) / 128 : 1;
  // head element of output tile j, place n
  __device__ static constexpr int elem(int j, int n) {
    return !kFp4 && D == 256 ? 128 * (j / 16) + 16 * n + j % 16 : n * (D / 8) + j;
  }
};

// One lane's codes and scales of a 16-token step.
template <int KIND, int D>
struct Keys {
  using S = Shape<KIND, D>;
  uint32_t w[2][S::kKeyWords];  // tokens r, r + 8
  uint32_t s[2][2];             // block: the float scales of tokens 2c, 2c+1 (+ 8); else the
                                // scale bytes of tokens r, r + 8
};
template <int KIND, int D>
struct Vals {
  using S = Shape<KIND, D>;
  uint32_t w[4][S::kValWords];  // tokens 2c, 2c+1, 2c+8, 2c+9
  uint32_t s[4][2];             // block: [0..3][0] float scales; else scale bytes per token
};

template <int KIND, int D>
__device__ __forceinline__ void load_keys(const brc_kv_cache& c, int64_t row, int lane,
                                          Keys<KIND, D>& k) {
  using S = Shape<KIND, D>;
  const int r = lane >> 2, q = lane & 3;
#pragma unroll
  for (int n = 0; n < 2; ++n) {
    const uint8_t* p = c.k_data + (row + r + 8 * n) * S::kRowBytes + q * (4 * S::kKeyChunk);
#pragma unroll
    for (int i = 0; i < S::kKeyWords / S::kKeyChunk; ++i)
      ldg_words<S::kKeyChunk>(p + 64 * i, &k.w[n][i * S::kKeyChunk]);
    if constexpr (KIND == BRC_STE_BLOCK_FP8) {
      const uint2 v = __ldg(reinterpret_cast<const uint2*>(
          static_cast<const float*>(c.k_scale) + row + 8 * n + 2 * q));
      k.s[n][0] = v.x;
      k.s[n][1] = v.y;
    } else if constexpr (KIND == BRC_STE_MXFP8) {
      const uint8_t* sp = static_cast<const uint8_t*>(c.k_scale) + (row + r + 8 * n) * S::kScales;
      if constexpr (D == 64) k.s[n][0] = __ldg(reinterpret_cast<const uint16_t*>(sp));
      else ldg_words<D / 128>(sp, k.s[n]);
    } else {
      const uint8_t* sp = static_cast<const uint8_t*>(c.k_scale) + (row + r + 8 * n) * S::kScales;
      if constexpr (D == 64) {
        k.s[n][0] = __ldg(sp + q);
      } else {
#pragma unroll
        for (int i = 0; i < D / 128; ++i)
          k.s[n][i] = __ldg(reinterpret_cast<const uint16_t*>(sp + 8 * i + 2 * q));
      }
    }
  }
}

template <int KIND, int D>
__device__ __forceinline__ void load_vals(const brc_kv_cache& c, int64_t row, int lane,
                                          Vals<KIND, D>& v) {
  using S = Shape<KIND, D>;
  const int r = lane >> 2, q = lane & 3;
#pragma unroll
  for (int t = 0; t < 4; ++t) {
    const int64_t at = row + 2 * q + (t & 1) + 8 * (t >> 1);
    const uint8_t* p = c.v_data + at * S::kRowBytes + r * (4 * S::kValChunk);
#pragma unroll
    for (int i = 0; i < S::kValWords / S::kValChunk; ++i)
      ldg_words<S::kValChunk>(p + 128 * i, &v.w[t][i * S::kValChunk]);
    if constexpr (KIND == BRC_STE_BLOCK_FP8) {
      v.s[t][0] = __ldg(static_cast<const uint32_t*>(c.v_scale) + at);
    } else {
      const uint8_t* sp = static_cast<const uint8_t*>(c.v_scale) + at * S::kScales;
      if constexpr (KIND == BRC_STE_MXFP8) {  // the whole row's bytes: its largest is needed
        if constexpr (D == 64) v.s[t][0] = __ldg(reinterpret_cast<const uint16_t*>(sp));
        else ldg_words<D / 128>(sp, v.s[t]);
      } else if constexpr (D == 256) {
        v.s[t][0] = __ldg(reinterpret_cast<const uint16_t*>(sp + 2 * r));
      } else {
        v.s[t][0] = __ldg(sp + (D == 128 ? r : r >> 1));
      }
    }
  }
}

// Largest byte of a scale row below 255 (255 stands for infinity and never
// becomes the reference).
template <int D>
__device__ __forceinline__ uint32_t top_byte(const uint32_t* s) {
  uint32_t m;
  if constexpr (D == 64) {
    m = s[0];  // two bytes
  } else if constexpr (D == 128) {
    m = s[0];
  } else {
    // 255 must not hide a smaller byte in the same place: taken out first
    const uint32_t a = s[0] & ~__vcmpeq4(s[0], 0xFFFFFFFFu), b = s[1] & ~__vcmpeq4(s[1], 0xFFFFFFFFu);
    m = __vmaxu4(a, b);
  }
  m &= ~__vcmpeq4(m, 0xFFFFFFFFu);
  if constexpr (D != 64) m = __vmaxu4(m, m >> 16);
  return max(m & 0xFFu, (m >> 8) & 0xFFu);
}

// True where a code word or a scale holds something that is not finite.
template <int KIND, int FMT>
__device__ __forceinline__ bool odd_codes(uint32_t w) {
  if constexpr (KIND == BRC_STE_NVFP4) return false;
  else if constexpr (FMT == BRC_FP8_E4M3)
    return (((w & 0x7F7F7F7Fu) + 0x01010101u) & 0x80808080u) != 0;
  else return (((w & 0x7C7C7C7Cu) + 0x04040404u) & 0x80808080u) != 0;
}

template <int KIND, int FMT, int D, int MT>
struct Warp {
  using S = Shape<KIND, D>;
  float o[MT][S::kTiles][4];
  float m[MT][2], l[MT][2];  // shift and sum of rows r, r + 8
  int e;                     // value scales are relative to 2^e

  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int i = 0; i < MT; ++i) {
#pragma unroll
      for (int j = 0; j < S::kTiles; ++j) o[i][j][0] = o[i][j][1] = o[i][j][2] = o[i][j][3] = 0.f;
      m[i][0] = m[i][1] = -INFINITY;
      l[i][0] = l[i][1] = 0.f;
    }
    e = -1000;
  }
  // Raise the reference of the value scales (a power of two) to 2^to, at least 2^-100.
  __device__ __forceinline__ void raise(int to) {
    to = max(to, -100);
    if (to <= e) return;
    const float f = e < -900 ? 1.f : __uint_as_float((uint32_t)max(127 + e - to, 0) << 23);
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int j = 0; j < S::kTiles; ++j)
#pragma unroll
        for (int x = 0; x < 4; ++x) o[i][j][x] *= f;
    e = to;
  }
};

// One value in float32, for the rare step that holds something not finite.
template <int KIND, int FMT, int D>
__device__ __forceinline__ float value_at(const brc_kv_cache& c, int64_t row, int d) {
  using S = Shape<KIND, D>;
  if constexpr (KIND == BRC_STE_NVFP4) {
    const uint32_t b = c.v_data[row * S::kRowBytes + d / 2];
    return dec_e2m1(d & 1 ? b >> 4 : b & 15u) *
           dec_e4m3(static_cast<const uint8_t*>(c.v_scale)[row * S::kScales + d / 16]);
  } else {
    const float v = dec_fp8<FMT>(c.v_data[row * S::kRowBytes + d]);
    if constexpr (KIND == BRC_STE_BLOCK_FP8) return v * static_cast<const float*>(c.v_scale)[row];
    else return v * e8m0_value(static_cast<const uint8_t*>(c.v_scale)[row * S::kScales + d / 32]);
  }
}

template <int KIND, int FMT, int D, int MT>
struct Step {
  using S = Shape<KIND, D>;
  using W = Warp<KIND, FMT, D, MT>;

  // s[mt][n][x]: scores of 16 tokens, not yet scaled by row.
  __device__ static __forceinline__ void scores(const Keys<KIND, D>& k, const uint4* q, int lane,
                                                float (&s)[MT][2][4]) {
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int n = 0; n < 2; ++n) s[i][n][0] = s[i][n][1] = s[i][n][2] = s[i][n][3] = 0.f;
    uint32_t top[2];
    if constexpr (KIND == BRC_STE_MXFP8) {
      top[0] = top_byte<D>(k.s[0]);
      top[1] = top_byte<D>(k.s[1]);
    }
#pragma unroll
    for (int w = 0; w < S::kKeyWords; ++w) {
      uint32_t b[2][S::kFp4 ? 4 : 2];
#pragma unroll
      for (int n = 0; n < 2; ++n) {
        const uint32_t x = k.w[n][w];
        if constexpr (S::kFp4) {
          // 8 codes of one 16-element block; its E4M3 scale is exact in f16
          uint32_t sc;
          if constexpr (D == 64) sc = k.s[n][0] & 0xFFu;
          else sc = (k.s[n][w / 4] >> (8 * ((w % 4) / 2))) & 0xFFu;
          const uint32_t f = fp8x2_to_f16x2<BRC_FP8_E4M3>(sc | (sc << 8));
#pragma unroll
          for (int i = 0; i < 4; ++i) b[n][i] = hmul2(kv::e2m1x2_to_f16x2(x >> (8 * i)), f);
        } else {
          b[n][0] = fp8x2_to_f16x2<FMT>(x);
          b[n][1] = fp8x2_to_f16x2<FMT>(x >> 16);
          if constexpr (KIND == BRC_STE_MXFP8) {
            // chunk w / 4 holds elements 64 (w / 4) + 16 c ..: block 2 (w / 4) + c / 2
            const uint32_t e =
                (k.s[n][w / 8] >> (16 * ((w / 4) % 2) + 8 * ((lane & 3) >> 1))) & 0xFFu;
            const uint32_t h = half_pow2_neg(e == 255 ? -1 : (int)top[n] - (int)e);
            b[n][0] = hmul2(b[n][0], h | (h << 16));
            b[n][1] = hmul2(b[n][1], h | (h << 16));
          }
        }
      }
#pragma unroll
      for (int g = 0; g < (S::kFp4 ? 2 : 1); ++g) {
        const int ks = S::kFp4 ? 2 * w + g : w;
#pragma unroll
        for (int i = 0; i < MT; ++i) {
          const uint4 a = q[(i * S::kSteps + ks) * 32 + lane];
#pragma unroll
          for (int n = 0; n < 2; ++n) mma(s[i][n], a, b[n][2 * g], b[n][2 * g + 1]);
        }
      }
    }
    // the token's own factor
    float f[2][2];
    if constexpr (KIND == BRC_STE_BLOCK_FP8) {
#pragma unroll
      for (int n = 0; n < 2; ++n) {
        f[n][0] = __uint_as_float(k.s[n][0]);
        f[n][1] = __uint_as_float(k.s[n][1]);
      }
    } else if constexpr (KIND == BRC_STE_MXFP8) {
#pragma unroll
      for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int i = 0; i < 2; ++i)
          f[n][i] = e8m0_value(__shfl_sync(0xFFFFFFFFu, top[n], (2 * (lane & 3) + i) * 4));
    }
    if constexpr (KIND != BRC_STE_NVFP4) {
#pragma unroll
      for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
          for (int x = 0; x < 4; ++x) s[i][n][x] *= f[n][x & 1];
    }
  }

  // Running maximum and sum; s becomes the probabilities relative to the shift.
  __device__ static __forceinline__ void softmax(W& w, float (&s)[MT][2][4]) {
    bool grow = false;
    float top[MT][2];
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        top[i][h] = fmaxf(fmaxf(s[i][0][2 * h], s[i][0][2 * h + 1]),
                          fmaxf(s[i][1][2 * h], s[i][1][2 * h + 1]));
        grow |= top[i][h] > w.m[i][h] + kGrow;
      }
    if (__any_sync(0xFFFFFFFFu, grow)) {
#pragma unroll
      for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          float t = top[i][h];
          t = fmaxf(t, __shfl_xor_sync(0xFFFFFFFFu, t, 1));
          t = fmaxf(t, __shfl_xor_sync(0xFFFFFFFFu, t, 2));
          const float m = fmaxf(w.m[i][h], t);
          const float f = m == w.m[i][h] ? 1.f : ex2(w.m[i][h] - m);
          w.m[i][h] = m;
          w.l[i][h] *= f;
#pragma unroll
          for (int j = 0; j < S::kTiles; ++j) {
            w.o[i][j][2 * h] *= f;
            w.o[i][j][2 * h + 1] *= f;
          }
        }
    }
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const float m = w.m[i][h] == -INFINITY ? 0.f : w.m[i][h];
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
          for (int x = 2 * h; x < 2 * h + 2; ++x) {
            s[i][n][x] = ex2(s[i][n][x] - m);
            w.l[i][h] += s[i][n][x];
          }
      }
  }

  // o += p v. Probabilities carry a factor 2^6 (at most 2^8 before it), so that
  // f16 keeps those down to 2^-30 of the largest.
  __device__ static __forceinline__ void values(W& w, const Vals<KIND, D>& v, int lane,
                                                const float (&p)[MT][2][4]) {
    float f[4] = {64.f, 64.f, 64.f, 64.f};
    uint32_t h[2][2];  // [token pair][half of the lane's elements]: f16 pair of value factors
    if constexpr (KIND == BRC_STE_BLOCK_FP8) {
      uint32_t top = 0;
#pragma unroll
      for (int t = 0; t < 4; ++t)
        if (v.s[t][0] < 0x7F800000u) top = max(top, v.s[t][0]);
      if (__any_sync(0xFFFFFFFFu, (int)(top >> 23) - 127 > w.e))
        w.raise((int)(__reduce_max_sync(0xFFFFFFFFu, top) >> 23) - 127);
      const float r = __uint_as_float((uint32_t)(127 - w.e + 6) << 23);
#pragma unroll
      for (int t = 0; t < 4; ++t) f[t] = __uint_as_float(v.s[t][0]) * r;
    } else if constexpr (KIND == BRC_STE_MXFP8) {
      uint32_t top = 0;
#pragma unroll
      for (int t = 0; t < 4; ++t) top = max(top, top_byte<D>(v.s[t]));
      if (__any_sync(0xFFFFFFFFu, (int)top - 127 > w.e))
        w.raise((int)__reduce_max_sync(0xFFFFFFFFu, top) - 127);
#pragma unroll
      for (int i = 0; i < (D == 256 ? 2 : 1); ++i) {
        const int r = lane >> 2, blk = D == 64 ? r >> 2 : 4 * i + (r >> 1);
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          uint32_t x[2];
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            const uint32_t e = (v.s[2 * t + u][i] >> (8 * (blk % 4))) & 0xFFu;
            x[u] = half_pow2_neg(e == 255 ? -1 : w.e + 127 - (int)e);
          }
          h[t][i] = x[0] | (x[1] << 16);
        }
      }
    } else {
      if (w.e < -900) w.e = 0;
#pragma unroll
      for (int i = 0; i < (D == 256 ? 2 : 1); ++i)
#pragma unroll
        for (int t = 0; t < 2; ++t)
          h[t][i] = fp8x2_to_f16x2<BRC_FP8_E4M3>(((v.s[2 * t][0] >> (8 * i)) & 0xFFu) |
                                                 (((v.s[2 * t + 1][0] >> (8 * i)) & 0xFFu) << 8));
    }
    uint4 a[MT];
#pragma unroll
    for (int i = 0; i < MT; ++i) {
      a[i].x = half2_of(p[i][0][0] * f[0], p[i][0][1] * f[1]);
      a[i].y = half2_of(p[i][0][2] * f[0], p[i][0][3] * f[1]);
      a[i].z = half2_of(p[i][1][0] * f[2], p[i][1][1] * f[3]);
      a[i].w = half2_of(p[i][1][2] * f[2], p[i][1][3] * f[3]);
    }
#pragma unroll
    for (int x = 0; x < S::kValWords; ++x) {
      constexpr int kPer = S::kFp4 ? 8 : 4;  // output tiles per word
      uint32_t b[2][kPer];
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const uint32_t u = v.w[2 * t][x], y = v.w[2 * t + 1][x];
        if constexpr (S::kFp4) {
          const uint32_t lo = (u & 0x0F0F0F0Fu) | ((y & 0x0F0F0F0Fu) << 4);
          const uint32_t hi = ((u >> 4) & 0x0F0F0F0Fu) | (y & 0xF0F0F0F0u);
          const uint32_t s = h[t][D == 256 ? x / 2 : 0];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            b[t][2 * i] = hmul2(kv::e2m1x2_to_f16x2(lo >> (8 * i)), s);
            b[t][2 * i + 1] = hmul2(kv::e2m1x2_to_f16x2(hi >> (8 * i)), s);
          }
        } else {
          const uint32_t lo = __byte_perm(u, y, 0x5140), hi = __byte_perm(u, y, 0x7362);
          b[t][0] = fp8x2_to_f16x2<FMT>(lo);
          b[t][1] = fp8x2_to_f16x2<FMT>(lo >> 16);
          b[t][2] = fp8x2_to_f16x2<FMT>(hi);
          b[t][3] = fp8x2_to_f16x2<FMT>(hi >> 16);
          if constexpr (KIND == BRC_STE_MXFP8) {
#pragma unroll
            for (int i = 0; i < 4; ++i) b[t][i] = hmul2(b[t][i], h[t][D == 256 ? x / 4 : 0]);
          }
        }
      }
#pragma unroll
      for (int j = 0; j < kPer; ++j)
#pragma unroll
        for (int i = 0; i < MT; ++i) mma(w.o[i][kPer * x + j], a[i], b[0][j], b[1][j]);
    }
  }

  // The same for a step whose values are not all finite: token by token, only
  // where the row sees the token, so that what it does not see cannot reach it.
  __device__ static __forceinline__ void values_checked(W& w, const brc_kv_cache& c, int64_t row,
                                                        int lane, const float (&p)[MT][2][4],
                                                        uint32_t seen) {
    if (w.e < -900) w.e = 0;
    const float r = 64.f * exp2f((float)-w.e);
    for (int t = 0; t < 16; ++t) {
      const int n = t >> 3, x = t & 1, src = (lane & ~3) | ((t & 7) >> 1);
      float pr[MT][2];
#pragma unroll
      for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const float lo = n ? p[i][1][2 * h] : p[i][0][2 * h];
          const float hi = n ? p[i][1][2 * h + 1] : p[i][0][2 * h + 1];
          pr[i][h] = __shfl_sync(0xFFFFFFFFu, x ? hi : lo, src);
        }
      const uint32_t sees = __shfl_sync(0xFFFFFFFFu, seen, src);
#pragma unroll
      for (int j = 0; j < S::kTiles; ++j)
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const float v = value_at<KIND, FMT, D>(c, row + t, S::elem(j, 2 * (lane & 3) + u));
#pragma unroll
          for (int i = 0; i < MT; ++i)
#pragma unroll
            for (int h = 0; h < 2; ++h)
              if ((sees >> (((i * 2 + h) * 2 + n) * 2 + x)) & 1u) w.o[i][j][2 * h + u] += pr[i][h] * r * v;
        }
    }
  }
};

template <int KIND, int FMT, int D, int MT>
__global__ void __launch_bounds__(kThreads) k_attend(Args a) {
  using S = Shape<KIND, D>;
  using St = Step<KIND, FMT, D, MT>;
  extern __shared__ __align__(16) uint8_t smem[];
  // queries as operand fragments, and (later) the warps' outputs
  uint4* const sq = reinterpret_cast<uint4*>(smem);
  float* const so = reinterpret_cast<float*>(smem);
  __shared__ float s_m[kWarps][16 * MT], s_l[kWarps][16 * MT], s_rowf[kWarps * 16 * MT];
  __shared__ Place s_place;

  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int row_warps = a.row_warps, token_warps = kWarps / row_warps;
  const int rw = warp % row_warps, tw = warp / row_warps;
  const int per_seq = a.c.heads * a.row_blocks;
  if (warp == 0) {
    Place p;
    locate(a, per_seq, gridDim.x, blockIdx.x, -1, p);
    if (lane == 0) s_place = p;
  }
  __syncthreads();
  const int64_t share = s_place.share;
  int64_t x = blockIdx.x * share;
  const int64_t end = min(x + share, s_place.total);
  if (x >= end) return;
  int b = s_place.b;
  int64_t seq_start = s_place.before * per_seq;
  const int rows_per_block = a.rows_per_block;

  while (x < end) {
    const Seq seq = load_seq(a, b);
    const int item = (int)((x - seq_start) / seq.steps);
    const int64_t item_start = seq_start + (int64_t)item * seq.steps;
    const int head = item / a.row_blocks, rb = item - head * a.row_blocks;
    const int s_begin = (int)(x - item_start);
    const int s_end = (int)min((int64_t)seq.steps, end - item_start);
    const int row0 = rb * rows_per_block;

    // ---- queries: scaled per row by a power of two into f16 fragments
    {
      constexpr int LPR = D / 8;
      const int part = tid % LPR, d0 = part * 8;
      for (int rr = tid / LPR; rr < rows_per_block; rr += kThreads / LPR) {
        const int row = row0 + rr, node = row / a.group;
        float f[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) f[i] = 0.f;
        if (row < a.rows && node < seq.drafts) {
          const int64_t at =
              (((int64_t)b * a.draft + node) * a.hq + head * a.group + (row - node * a.group)) * D + d0;
          if (a.q_f16) kv::load8<BRC_DTYPE_F16>(a.q, at, f);
          else kv::load8<BRC_DTYPE_BF16>(a.q, at, f);
        }
        float top = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) top = fmaxf(top, fabsf(f[i]));
#pragma unroll
        for (int o = 1; o < LPR; o <<= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, o));
        // top in [2^k, 2^(k+1)): elements times 2^(7-k)
        const int k = min(max((int)(__float_as_uint(top) >> 23) - 127, -119), 127);
        const float up = __uint_as_float((uint32_t)(127 + 7 - k) << 23);
        if (part == 0) s_rowf[rr] = a.scale_log2 * __uint_as_float((uint32_t)(127 + k - 7) << 23);
        uint32_t* const dst = reinterpret_cast<uint32_t*>(sq);
        const int mt = rr >> 4, r16 = rr & 15;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int d = d0 + 2 * i;  // pair d, d + 1
          int ks, c, j;
          if constexpr (S::kFp4) {
            constexpr int kLane = 8 * S::kKeyChunk;  // elements of a lane's chunk
            const int in = d % (4 * kLane);
            c = in / kLane;
            ks = (d / (4 * kLane)) * (2 * S::kKeyChunk) + (in % kLane) / 4;
            j = d % 4;
          } else {
            c = (d % 64) / 16;
            ks = (d / 64) * 4 + (d % 16) / 4;
            j = d % 4;
          }
          const int reg = (j >> 1) * 2 + (r16 >> 3);
          dst[((mt * S::kSteps + ks) * 32 + (r16 & 7) * 4 + c) * 4 + reg] =
              half2_of(f[2 * i] * up, f[2 * i + 1] * up);
        }
      }
    }
    __syncthreads();

    Warp<KIND, FMT, D, MT> w;
    w.clear();
    const uint4* const q = sq + (int64_t)rw * MT * S::kSteps * 32;
    float rowf[MT][2];
    int node[MT][2];
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int rr = (rw * MT + i) * 16 + (lane >> 2) + 8 * h;
        rowf[i][h] = s_rowf[rr];
        const int row = row0 + rr;
        node[i][h] = row < a.rows ? row / a.group : a.draft;
      }

    const int32_t* const table = a.table + b * a.table_stride;
    const int page_mask = a.c.page_size - 1;
    auto row_at = [&](int s) -> int64_t {  // first cache row of a step, or -1
      const int64_t t = (int64_t)s << 4;
      if (t >= seq.total) return -1;
      const int64_t page = __ldg(table + (t >> a.page_shift));
      if (page < 0 || page >= a.c.num_pages) return -1;
      return (page * a.c.heads + head) * a.c.page_size + (t & page_mask);
    };
    Keys<KIND, D> k;
    Vals<KIND, D> v;
    int s = s_begin + tw;
    int64_t row = s < s_end ? row_at(s) : -1;
    if (row >= 0) {
      load_keys<KIND, D>(a.c, row, lane, k);
      load_vals<KIND, D>(a.c, row, lane, v);
    }
    while (s < s_end) {
      const int sn = s + token_warps;
      const int64_t row_n = sn < s_end ? row_at(sn) : -1;
      if (row >= 0) {
        float p[MT][2][4];
        St::scores(k, q, lane, p);
        if (row_n >= 0) load_keys<KIND, D>(a.c, row_n, lane, k);
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
          for (int n = 0; n < 2; ++n)
#pragma unroll
            for (int y = 0; y < 4; ++y) p[i][n][y] *= rowf[i][y >> 1];
        const int t0 = s << 4;
        uint32_t seen = 0;
        bool checked = false;
        if (t0 + 16 > seq.context) {  // drafted tokens, or past the end
#pragma unroll
          for (int i = 0; i < MT; ++i)
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
              for (int n = 0; n < 2; ++n)
#pragma unroll
                for (int y = 0; y < 2; ++y) {
                  const int t = t0 + n * 8 + 2 * (lane & 3) + y, j = t - seq.context;
                  bool see = t < seq.total && node[i][h] < seq.drafts;
                  if (see && j >= 0)
                    see = a.tree ? a.tree[b * a.tree_stride + (int64_t)node[i][h] * a.draft + j] != 0
                                 : j <= node[i][h];
                  if (see) seen |= 1u << (((i * 2 + h) * 2 + n) * 2 + y);
                  else p[i][n][2 * h + y] = -INFINITY;
                }
          // values past the end count as zero; a drafted value that is not
          // finite must not meet a probability of zero in the product
          bool odd = false;
#pragma unroll
          for (int t = 0; t < 4; ++t) {
            const bool live = t0 + 2 * (lane & 3) + (t & 1) + 8 * (t >> 1) < seq.total;
#pragma unroll
            for (int y = 0; y < S::kValWords; ++y) {
              if (!live) v.w[t][y] = 0;
              odd |= odd_codes<KIND, FMT>(v.w[t][y]);
            }
            if (!live) v.s[t][0] = v.s[t][1] = 0;
            if constexpr (KIND == BRC_STE_BLOCK_FP8) odd |= (v.s[t][0] & 0x7F800000u) == 0x7F800000u;
            else if constexpr (KIND == BRC_STE_NVFP4)
              odd |= (v.s[t][0] & 0x7Fu) == 0x7Fu || (D == 256 && (v.s[t][0] & 0x7F00u) == 0x7F00u);
            else
              odd |= __vcmpeq4(v.s[t][0], 0xFFFFFFFFu) != 0 ||
                     (D == 256 && __vcmpeq4(v.s[t][1], 0xFFFFFFFFu) != 0);
          }
          checked = __any_sync(0xFFFFFFFFu, odd);
        }
        St::softmax(w, p);
        if (checked) St::values_checked(w, a.c, row, lane, p, seen);
        else St::values(w, v, lane, p);
      } else if (row_n >= 0) {
        load_keys<KIND, D>(a.c, row_n, lane, k);
      }
      if (row_n >= 0) load_vals<KIND, D>(a.c, row_n, lane, v);
      row = row_n;
      s = sn;
    }

    // ---- join the warps that share rows
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        float l = w.l[i][h];
        l += __shfl_xor_sync(0xFFFFFFFFu, l, 1);
        l += __shfl_xor_sync(0xFFFFFFFFu, l, 2);
        if ((lane & 3) == 0) {
          const int rr = i * 16 + (lane >> 2) + 8 * h;
          s_m[warp][rr] = w.m[i][h];
          s_l[warp][rr] = l;
        }
      }
    __syncthreads();  // the query fragments are no longer read
    const float scale_o = w.e < -900 ? 1.f : exp2f((float)(w.e - 6));
    constexpr int kPitch = D + 4;
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int j = 0; j < S::kTiles; ++j)
#pragma unroll
        for (int y = 0; y < 4; ++y) {
          const int rr = i * 16 + (lane >> 2) + 8 * (y >> 1);
          so[(warp * 16 * MT + rr) * kPitch + S::elem(j, 2 * (lane & 3) + (y & 1))] =
              w.o[i][j][y] * scale_o;
        }
    __syncthreads();
    const bool whole = s_begin == 0 && s_end == seq.steps;
    const int64_t slot = 2 * (int64_t)blockIdx.x + (s_begin > 0 ? 0 : 1);
    for (int at = tid; at < rows_per_block * (D / 4); at += kThreads) {
      const int rr = at / (D / 4), d = (at - rr * (D / 4)) * 4;
      const int row = row0 + rr;
      if (row >= a.rows) continue;
      const int w0 = rr / (16 * MT), r = rr - w0 * 16 * MT;  // row warp, row in its tile
      float m = -INFINITY;
      for (int t = 0; t < token_warps; ++t) m = fmaxf(m, s_m[t * row_warps + w0][r]);
      float l = 0.f, o[4] = {0.f, 0.f, 0.f, 0.f};
      for (int t = 0; t < token_warps; ++t) {
        const int wi = t * row_warps + w0;
        const float f = m == -INFINITY ? 1.f : ex2(s_m[wi][r] - m);
        l += s_l[wi][r] * f;
        const float4 y = *reinterpret_cast<const float4*>(so + (wi * 16 * MT + r) * kPitch + d);
        o[0] += y.x * f;
        o[1] += y.y * f;
        o[2] += y.z * f;
        o[3] += y.w * f;
      }
      if (whole) {
        const int nd = row / a.group;
        const int64_t at_row =
            ((int64_t)b * a.draft + nd) * a.hq + head * a.group + (row - nd * a.group);
        const bool none = nd >= seq.drafts || l == 0.f;
        const float inv = none ? 0.f : 1.f / l;
        uint2 y;
        if (none) {
          y = make_uint2(0u, 0u);
        } else if (a.q_f16) {
          y = make_uint2(half2_of(o[0] * inv, o[1] * inv), half2_of(o[2] * inv, o[3] * inv));
        } else {
          const __nv_bfloat162 y0 = __floats2bfloat162_rn(o[0] * inv, o[1] * inv);
          const __nv_bfloat162 y1 = __floats2bfloat162_rn(o[2] * inv, o[3] * inv);
          y = make_uint2(*reinterpret_cast<const uint32_t*>(&y0), *reinterpret_cast<const uint32_t*>(&y1));
        }
        *reinterpret_cast<uint2*>(static_cast<uint16_t*>(a.out) + at_row * D + d) = y;
        if (a.lse && d == 0)
          a.lse[at_row] = none ? -INFINITY : (m + log2f(l)) * 0.6931471805599453f;
      } else {
        *reinterpret_cast<float4*>(a.part_o + (slot * rows_per_block + rr) * D + d) =
            make_float4(o[0], o[1], o[2], o[3]);
        if (d == 0) {
          float* const ml = a.part_ml + (slot * rows_per_block + rr) * 2;
          ml[0] = m;
          ml[1] = l;
        }
      }
    }
    __syncthreads();
    x = item_start + s_end;
    if (s_end == seq.steps && item + 1 == per_seq) {
      seq_start += (int64_t)per_seq * seq.steps;
      ++b;
    }
  }
}

// Join the parts of items that several blocks share: one warp to a query row,
// the parts in the order of their tokens.
template <int D>
__global__ void __launch_bounds__(kThreads) k_join(Args a, int blocks) {
  const int lane = threadIdx.x & 31;
  const int64_t id = (int64_t)blockIdx.x * kWarps + (threadIdx.x >> 5);
  const int per_head = a.row_blocks * a.rows_per_block;
  const int64_t per_b = (int64_t)a.c.heads * per_head;
  if (id >= per_b * a.batch) return;
  const int b = (int)(id / per_b);
  const int rest = (int)(id - b * per_b);
  const int head = rest / per_head, row = rest - head * per_head;
  if (row >= a.rows) return;
  const int rb = row / a.rows_per_block, rr = row - rb * a.rows_per_block;
  const int per_seq = a.c.heads * a.row_blocks;
  Place p;
  locate(a, per_seq, blocks, 0, b, p);
  const Seq seq = load_seq(a, b);
  const int64_t start = p.before * per_seq + (int64_t)(head * a.row_blocks + rb) * seq.steps;
  const int64_t c0 = start / p.share, c1 = (start + seq.steps - 1) / p.share;
  if (c0 == c1) return;
  float m = -INFINITY;
  for (int64_t c = c0 + lane; c <= c1; c += 32) {
    const int64_t slot = 2 * c + (c == c0 ? 1 : 0);
    m = fmaxf(m, a.part_ml[(slot * a.rows_per_block + rr) * 2]);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xFFFFFFFFu, m, o));
  constexpr int N = D / 32;
  float l = 0.f, o[N];
#pragma unroll
  for (int i = 0; i < N; ++i) o[i] = 0.f;
  for (int64_t base = c0; base <= c1; base += 32) {
    const int64_t c = base + lane;
    float f = 0.f, lp = 0.f;
    if (c <= c1) {
      const int64_t slot = 2 * c + (c == c0 ? 1 : 0);
      const float2 ml = *reinterpret_cast<const float2*>(a.part_ml + (slot * a.rows_per_block + rr) * 2);
      f = m == -INFINITY ? 1.f : ex2(ml.x - m);
      lp = ml.y * f;
    }
    const int n = (int)min((int64_t)32, c1 - base + 1);
#pragma unroll 4
    for (int i = 0; i < n; ++i) {
      const float fi = __shfl_sync(0xFFFFFFFFu, f, i);
      l += __shfl_sync(0xFFFFFFFFu, lp, i);
      const int64_t ci = base + i, slot = 2 * ci + (ci == c0 ? 1 : 0);
      const float* y = a.part_o + (slot * a.rows_per_block + rr) * D + lane * N;
#pragma unroll
      for (int j = 0; j < N; ++j) o[j] += fi * y[j];
    }
  }
  const int nd = row / a.group;
  const int64_t at = ((int64_t)b * a.draft + nd) * a.hq + head * a.group + (row - nd * a.group);
  const bool none = nd >= seq.drafts || l == 0.f;
  const float inv = none ? 0.f : 1.f / l;
#pragma unroll
  for (int j = 0; j < N; j += 2) {
    uint32_t y = 0;
    if (!none) {
      if (a.q_f16) {
        y = half2_of(o[j] * inv, o[j + 1] * inv);
      } else {
        const __nv_bfloat162 h = __floats2bfloat162_rn(o[j] * inv, o[j + 1] * inv);
        y = *reinterpret_cast<const uint32_t*>(&h);
      }
    }
    *reinterpret_cast<uint32_t*>(static_cast<uint16_t*>(a.out) + at * D + lane * N + j) = y;
  }
  if (a.lse && lane == 0) a.lse[at] = none ? -INFINITY : (m + log2f(l)) * 0.6931471805599453f;
}

// ------------------------------------------------------------------ host
constexpr int smem_bytes(int d, int mt) {
  const int q = kWarps * 16 * mt * d * 2;              // query fragments, most row warps
  const int o = kWarps * 16 * mt * (d + 4) * 4;        // the warps' outputs
  return q > o ? q : o;
}
constexpr int kBlocksPerSm = 4;  // at most; what fits is asked of the driver

template <int KIND, int FMT, int D, int MT>
int launch(Args a, int blocks, cudaStream_t st) {
  constexpr int bytes = smem_bytes(D, MT);
  if (const int rc = check_cuda(cudaFuncSetAttribute(
          k_attend<KIND, FMT, D, MT>, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes)))
    return rc;
  k_attend<KIND, FMT, D, MT><<<blocks, kThreads, bytes, st>>>(a);
  if (const int rc = check_launch()) return rc;
  const int64_t warps = (int64_t)a.batch * a.c.heads * a.row_blocks * a.rows_per_block;
  k_join<D><<<(unsigned)((warps + kWarps - 1) / kWarps), kThreads, 0, st>>>(a, blocks);
  return check_launch();
}

template <int KIND, int FMT>
int by_shape(const Args& a, int mt, int blocks, cudaStream_t st) {
  switch (a.c.head_dim) {
    case 64: return mt == 1 ? launch<KIND, FMT, 64, 1>(a, blocks, st)
                            : launch<KIND, FMT, 64, 2>(a, blocks, st);
    case 128: return mt == 1 ? launch<KIND, FMT, 128, 1>(a, blocks, st)
                             : launch<KIND, FMT, 128, 2>(a, blocks, st);
    default: return launch<KIND, FMT, 256, 1>(a, blocks, st);
  }
}

int attend_block_e4m3(const Args& a, int mt, int blocks, cudaStream_t st);
int attend_block_e5m2(const Args& a, int mt, int blocks, cudaStream_t st);
int attend_mx_e4m3(const Args& a, int mt, int blocks, cudaStream_t st);
int attend_mx_e5m2(const Args& a, int mt, int blocks, cudaStream_t st);
int attend_nvfp4(const Args& a, int mt, int blocks, cudaStream_t st);

}  // namespace kvatt
}  // namespace brc
