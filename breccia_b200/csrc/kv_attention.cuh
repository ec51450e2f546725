// Attention of a few new tokens (one, or a tree of drafted ones) over the
// quantised paged cache.
//
//   s_ij = scale q_i . k_j,  out_i = sum_j softmax_j(s_ij) v_j  over visible j
//
// The query rows of one sequence and one cache head (draft x hq / heads) share
// every key and value, so the codes are read once for all of them: HBM bounds
// single tokens and small trees. One pass with a running maximum and sum.
//
// Layout. A warp takes 16 tokens at a time as the rows of m16n8k16 products, with
// 8 query rows to a product's columns: S^T = K Q^T and O^T = V^T P^T, so a group
// of 8 query heads or fewer wastes nothing and holds half the accumulators of
// the other orientation. Which head elements stand at which place of a fragment
// is free as long as both operands agree, so a lane's words are contiguous bytes
// of a row, read whole:
//   keys    (A of K Q^T):   lane (r, c) reads tokens r, r + 8, bytes 64 i + 16 c .. + 15
//   values  (A of V^T P^T): lane (r, c) reads tokens 2c, 2c+1, 2c+8, 2c+9, bytes
//                           16 r .. + 15; pairs of tokens are byte permutes
// The scores' fragment becomes the probabilities' by two 8 x 8 transposes.
// Codes come through a ring of 16-token stages of each warp's own (asynchronous
// copies, no block barrier).
//
// Numbers. FP8 and FP4 codes are exact in f16. Queries are scaled per row by a
// power of two into f16 (elements below 2^-21 of the row's largest lose bits).
// Key scales: block FP8 multiplies the score; MXFP8's per-block powers of two
// go onto the codes relative to one that the warp's tokens share; NVFP4's E4M3
// scales times E2M1 codes are exact in f16. Value scales likewise, relative to a
// power of two for each channel block (block FP8's go onto the probabilities, so
// that f16 holds probability x scale: 11 bits each, against the 8 of a bf16
// output). These references move with the scales; tokens of a step that do not
// go with one of them are taken in passes of their own ("references" below), so
// that no token's scale touches another one's bits. Scores, sums, the running
// maximum and the output are float32.
//
// Work split. The steps of 16 tokens of all (sequence, cache head, row block)
// items are cut into equal shares, one per block, whatever the lengths: the
// lengths stay on the device and ragged batches balance. A block that holds
// only part of an item leaves its sums in the workspace, and a second kernel
// joins the parts in a fixed order.
//
// Measured on B200, 8 cache heads of 128: 64 tokens of 32 query heads over 8192 tokens
// each (join included) block FP8 191 us (5.8 TB/s), MXFP8 192, NVFP4 158; HBM bounds
// the first, the decoding of codes and scales the other two. Two sequences of 131072
// tokens in NVFP4, 64 query heads: 96 us (3.1 TB/s).
#pragma once

#include "kv_codec.cuh"
#include "launch.h"

namespace brc {
namespace kvatt {

constexpr int kThreads = 128;
constexpr int kWarps = kThreads / 32;
constexpr float kGrow = 8.f;  // a row's shift follows its maximum when it is this far (log2) behind
// Sums of p v carry the factor 2^-kSumDown until they are divided by the sum of p, which
// may be as large as 2^kGrow for each token: values up to the largest float do not overflow.
constexpr int kSumDown = 30;
constexpr float kSumUp = 1 << kSumDown;

struct Args {
  brc_kv_cache c;
  const void* q;
  int q_f16, batch, draft, hq, group, rows;  // rows = draft * group
  const int32_t* table;
  int64_t table_stride;
  int table_pages, page_shift, step_shift;  // 2^step_shift tokens to a step
  uint32_t page_rows;                       // rows from one page to the next: heads * page_size
  const int32_t* context;
  const int32_t* drafts;
  const uint8_t* tree;
  int64_t tree_stride;
  float scale_log2;
  void* out;
  float* lse;
  float* part_o;   // (2 * blocks, rows per block, d): sums of p v
  float* part_ml;  // (2 * blocks, rows per block, 2)
  int row_warps, row_blocks, rows_per_block, min_share;
};

struct Seq {
  int context, drafts, total;  // tokens
  int steps;                   // at least one
};
__device__ __forceinline__ Seq load_seq(const Args& a, int b) {
  Seq s;
  const int64_t cap = (int64_t)a.table_pages << a.page_shift;
  const int ctx = max(a.context[b], 0);
  s.drafts = a.drafts ? min(max(a.drafts[b], 0), a.draft) : a.draft;
  s.context = (int)min((int64_t)ctx, cap);
  s.total = (int)min((int64_t)ctx + s.drafts, cap);
  s.steps = max((int)(((int64_t)s.total + (1 << a.step_shift) - 1) >> a.step_shift), 1);
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
  const int64_t items = (int64_t)a.batch * per_seq;
  p.total = __shfl_sync(0xFFFFFFFFu, incl, 31) * per_seq;
  // small parts cost more to join than they save: at least min_share steps, or an item
  p.share = max((p.total + blocks - 1) / blocks,
                min((int64_t)a.min_share, (p.total + items - 1) / items));
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
// The four codes of a word as two f16 pairs (both halves named to the compiler
// as 16-bit registers: no shift for the upper one).
template <int FMT>
__device__ __forceinline__ void fp8x4_to_f16x4(uint32_t w, uint32_t& lo, uint32_t& hi) {
  if constexpr (FMT == BRC_FP8_E4M3)
    asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, a;\n\t"
        "cvt.rn.f16x2.e4m3x2 %1, b;\n\t}" : "=r"(lo), "=r"(hi) : "r"(w));
  else
    asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %2;\n\tcvt.rn.f16x2.e5m2x2 %0, a;\n\t"
        "cvt.rn.f16x2.e5m2x2 %1, b;\n\t}" : "=r"(lo), "=r"(hi) : "r"(w));
}
// The eight E2M1 codes of a word as four f16 pairs.
__device__ __forceinline__ void e2m1x8_to_f16x8(uint32_t w, uint32_t (&h)[4]) {
  asm("{\n\t.reg .b8 a, b, c, d;\n\tmov.b32 {a, b, c, d}, %4;\n\tcvt.rn.f16x2.e2m1x2 %0, a;\n\t"
      "cvt.rn.f16x2.e2m1x2 %1, b;\n\tcvt.rn.f16x2.e2m1x2 %2, c;\n\tcvt.rn.f16x2.e2m1x2 %3, d;\n\t}"
      : "=r"(h[0]), "=r"(h[1]), "=r"(h[2]), "=r"(h[3])
      : "r"(w));
}
// E8M0 byte to float32 (255 as the casts read it: infinity).
__device__ __forceinline__ float e8m0_value(uint32_t e) {
  return e == 0 ? __uint_as_float(0x00400000u) : __uint_as_float(e << 23);
}
// 2^(e - ref) of two E8M0 bytes as an f16 pair: subnormals and zero below
// 2^-14. INF: a byte of 255 (which never is the reference) gives infinity.
template <bool INF>
__device__ __forceinline__ uint32_t half2_pow2(int e0, int e1, int ref) {
  auto f = [&](int e) {
    int x = max(e - ref + 127, 0);
    if constexpr (INF) x = e == 255 ? 255 : x;
    return __uint_as_float((uint32_t)x << 23);
  };
  return half2_of(f(e0), f(e1));
}

// ------------------------------------------------------------------ references
// What codes are relative to in f16. Scales are taken as biased exponents, a byte to a
// channel block (MXFP8: E8M0 bytes; block FP8: the float32 scale's); 255 is not finite
// and goes with any reference.
//
// Codes whose scale is up to kSpan (log2) below its reference keep their bits: E4M3 codes
// are multiples of 2^-9 and f16 holds multiples of 2^-24 (E5M2's smallest lose what is
// below 2^-25 of their block's largest). Block FP8's scales are multiplied in before the
// rounding to f16, onto the probabilities (here: they then keep what is above 2^-20 of the
// row's largest, as 2^-31 without) or the values (tcgen05: E4M3's smallest codes then just
// are normal numbers). Tokens further apart do not go together, but for scales as the
// casts give them to zeros (kFloor: values below 6e-8, in block FP8 1e-10), which count as
// zero beside larger ones: rows of zeros are common. (MXFP8's E5M2 gives zeros the scale
// of values up to 7e-6, so there only what no cast writes counts.) A reference is set kSlack above the
// scale that asks for it, so that it seldom moves, and not below kSpan, so that scales of
// zero, as a new cache holds them, go together.
template <int KIND>
constexpr int kSpan = KIND == BRC_STE_BLOCK_FP8 ? 11 : 15;
template <int KIND, int FMT>
constexpr uint32_t kFloor = KIND == BRC_STE_MXFP8 ? (FMT == BRC_FP8_E4M3 ? 94 : 93)
                                                  : (FMT == BRC_FP8_E4M3 ? 84 : 77);
constexpr int kSlack = 2;

template <int KIND, int D>
constexpr int kScaleBlocks = KIND == BRC_STE_MXFP8 ? D / 32 : 1;

// Whether up to four bytes lie within SPAN below their references: both as 16-bit
// fields, offset so that the difference does not borrow. Bytes without a block are zero
// on both sides.
template <int SPAN>
struct Near {
  static_assert((SPAN & (SPAN + 1)) == 0, "a mask");
  uint32_t even, odd;
  __device__ __forceinline__ Near() {}
  __device__ __forceinline__ explicit Near(uint32_t refs)
      : even(0x01000100u + SPAN * 0x00010001u - (refs & 0x00FF00FFu)),
        odd(0x01000100u + SPAN * 0x00010001u - ((refs >> 8) & 0x00FF00FFu)) {}
  __device__ __forceinline__ uint32_t refs() const {
    return (0x01000100u + SPAN * 0x00010001u - even) |
           ((0x01000100u + SPAN * 0x00010001u - odd) << 8);
  }
  __device__ __forceinline__ bool operator()(uint32_t x) const {
    const uint32_t a = ((x & 0x00FF00FFu) + even) ^ 0x01000100u;
    const uint32_t b = (((x >> 8) & 0x00FF00FFu) + odd) ^ 0x01000100u;
    return ((a | b) & ~(SPAN * 0x00010001u)) == 0u;
  }
};

// The largest finite byte of up to four.
__device__ __forceinline__ uint32_t top_byte(uint32_t x) {
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 32; i += 8) {
    const uint32_t y = (x >> i) & 0xFFu;
    if (y != 255u) m = max(m, y);
  }
  return m;
}

// Of the tokens in `left` (bit y of each lane: its token y of N), those that go together,
// at least one: block by block, the ones near the largest scale of those that are left.
// W words of four blocks' bytes to a token's values; km: the largest byte of its keys
// (MXFP8). `refs` moves for them where it has to; returns what their keys are relative to.
template <int SPAN, uint32_t FLOOR, int BLOCKS, int N, int W>
__device__ __forceinline__ uint32_t choose(const uint32_t (&v)[N][W], const uint32_t (&km)[N],
                                           uint32_t left, uint32_t& take, uint32_t (&refs)[W]) {
  constexpr uint32_t kTake = SPAN - kSlack;
  take = left;
#pragma unroll
  for (int w = 0; w < W; ++w) {
#pragma unroll 1
    for (int i = 0; i < 8 * (BLOCKS < 4 ? BLOCKS : 4); i += 8) {
      uint32_t top = 0;
#pragma unroll
      for (int y = 0; y < N; ++y) {
        const uint32_t x = (v[y][w] >> i) & 0xFFu;
        if (((take >> y) & 1u) && x != 255u) top = max(top, x);
      }
      top = __reduce_max_sync(0xFFFFFFFFu, top);
      const uint32_t ref = (refs[w] >> i) & 0xFFu;
      bool off = top > ref;
#pragma unroll
      for (int y = 0; y < N; ++y) {
        const uint32_t x = (v[y][w] >> i) & 0xFFu;
        if (x <= FLOOR) continue;  // (its reference is no lower: the largest is not)
        if (x + kTake < top) take &= ~(1u << y);
        else off |= ((take >> y) & 1u) && x + SPAN < ref;
      }
      if (__any_sync(0xFFFFFFFFu, off))
        refs[w] += (min(max(top + kSlack, (uint32_t)SPAN), 254u) - ref) << i;
    }
  }
  uint32_t k = 0;
#pragma unroll
  for (int y = 0; y < N; ++y)
    if ((take >> y) & 1u) k = max(k, km[y]);
  k = __reduce_max_sync(0xFFFFFFFFu, k);
#pragma unroll
  for (int y = 0; y < N; ++y)
    if (km[y] > FLOOR && km[y] + kTake < k) take &= ~(1u << y);
  return k;
}

// A step is two 16-token tiles: two independent chains of products, one set of
// votes and waits for both. Heads of 256 take one, or a ring would not fit.
constexpr __host__ __device__ int subtiles(int d) { return d == 256 ? 1 : 2; }

// One step in shared memory: rows of key codes, rows of value codes, their
// scales. A row's 16-byte pieces are permuted by its number so that the
// operand reads below touch every bank once (64-byte rows: the value reads
// twice).
template <int KIND, int D>
struct Shape {
  static constexpr bool kFp4 = KIND == BRC_STE_NVFP4;
  static constexpr int kRowBytes = kv::row_bytes(KIND, D);
  static constexpr int kPieces = kRowBytes / 16;
  static constexpr int kScales = kv::row_scales(KIND, D);
  static constexpr int kScaleBytes = kScales * (KIND == BRC_STE_BLOCK_FP8 ? 4 : 1);
  static constexpr int kKeyWords = kRowBytes / 16;    // per lane and token
  static constexpr int kValWords = kRowBytes / 32;    // per lane and token
  static constexpr int kKeyRead = kKeyWords < 4 ? kKeyWords : 4;  // words to a read
  static constexpr int kValRead = kValWords < 4 ? kValWords : 4;
  static constexpr int kSteps = D / 16;               // products along the head
  static constexpr int kTiles = D / 16;               // output tiles of 16 elements
  static constexpr int kSub = subtiles(D);
  static constexpr int kRows = 16 * kSub;             // tokens of a step
  static constexpr uint32_t kAll = kSub == 2 ? 0xFFFFFFFFu : 0xFFFFu;
  static constexpr int kTileBytes = kRows * kRowBytes;
  static constexpr int kKeyScales = 2 * kTileBytes;
  static constexpr int kValScales = kKeyScales + kRows * kScaleBytes;
  static constexpr int kStageBytes = kValScales + kRows * kScaleBytes;
  // Where a lane reads: keys, read i of token r (others: constants further on);
  // values, read i of token 2 c.
  __device__ static __forceinline__ int key_offset(int lane, int i) {
    const int r = lane >> 2, c = lane & 3;
    if constexpr (kKeyRead < 4) return r * kRowBytes + c * 8;
    else if constexpr (kPieces >= 8)
      return r * kRowBytes + c * 16 + 64 * ((i & 1) ^ (r & 1)) + 128 * (i >> 1);
    else return r * kRowBytes + c * 16 + 64 * i;
  }
  __device__ static __forceinline__ int val_offset(int lane, int i) {
    const int r = lane >> 2, c = lane & 3;
    if constexpr (kValRead == 4) return 2 * c * kRowBytes + ((r ^ (2 * c)) + 8 * i) * 16;
    else if constexpr (kValRead == 2)
      return 2 * c * kRowBytes + (((r >> 1) ^ ((2 * c) & 2)) * 16) + (r & 1) * 8;
    else return 2 * c * kRowBytes + r * 4;
  }
  __device__ static constexpr int key_piece(int t, int p) {
    return kPieces >= 8 ? p ^ ((t & 1) << 2) : p;
  }
  __device__ static constexpr int val_piece(int t, int p) {
    return kPieces >= 8 ? p ^ (t & 6) : kPieces == 4 ? p ^ (t & 2) : p;
  }
  // head element of a lane's output i (two to a tile), r = lane / 4
  __device__ static constexpr int elem(int i, int r) {
    return !kFp4 && D == 256 ? 128 * (i / 16) + 16 * r + i % 16 : r * (D / 8) + i;
  }
};

__device__ __forceinline__ void cp16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// Start the copy of the 16 rows from `row` on into tile `sub` of a stage (a warp's own).
template <int KIND, int D>
__device__ __forceinline__ void copy_tile(const brc_kv_cache& c, int64_t row, int lane,
                                          uint32_t stage, int sub) {
  using S = Shape<KIND, D>;
  const uint8_t* k = c.k_data + row * S::kRowBytes + lane * 16;
  const uint8_t* v = c.v_data + row * S::kRowBytes + lane * 16;
  const uint32_t at = stage + sub * 16 * S::kRowBytes;
#pragma unroll
  for (int i = 0; i < S::kPieces / 2; ++i) {
    const int id = lane + 32 * i, t = id / S::kPieces, p = id % S::kPieces;
    cp16(at + (t * S::kPieces + S::key_piece(t, p)) * 16, k + 512 * i);
    cp16(at + S::kTileBytes + (t * S::kPieces + S::val_piece(t, p)) * 16, v + 512 * i);
  }
  const int i = lane & 15;
  if (i < S::kScaleBytes) {
    const void* base = lane < 16 ? c.k_scale : c.v_scale;
    cp16(stage + (lane < 16 ? S::kKeyScales : S::kValScales) + (sub * S::kScaleBytes + i) * 16,
         static_cast<const uint8_t*>(base) + row * S::kScaleBytes + i * 16);
  }
}

template <int N>
__device__ __forceinline__ void lds_words(const uint8_t* p, uint32_t* w) {
  if constexpr (N == 4) {
    const uint4 v = *reinterpret_cast<const uint4*>(p);
    w[0] = v.x; w[1] = v.y; w[2] = v.z; w[3] = v.w;
  } else if constexpr (N == 2) {
    const uint2 v = *reinterpret_cast<const uint2*>(p);
    w[0] = v.x; w[1] = v.y;
  } else {
    w[0] = *reinterpret_cast<const uint32_t*>(p);
  }
}

// True where a code word or a scale holds something that is not finite.
template <int KIND, int FMT>
__device__ __forceinline__ bool odd_codes(uint32_t w) {
  if constexpr (KIND == BRC_STE_NVFP4) return false;
  else if constexpr (FMT == BRC_FP8_E4M3)
    return (((w & 0x7F7F7F7Fu) + 0x01010101u) & 0x80808080u) != 0;
  else return (((w & 0x7C7C7C7Cu) + 0x04040404u) & 0x80808080u) != 0;
}

// A warp's notes on an item's steps (in shared memory: they are rare, and registers are not).
struct Later {
  static constexpr int kMost = 13;
  int count, climb, fall;  // steps put off; how far references climbed and fell, in all
  int step[kMost];
};

template <int KIND, int FMT, int D, int NT>
struct Warp {
  using S = Shape<KIND, D>;
  static constexpr int kSpans = kSpan<KIND>;
  static constexpr uint32_t kZero = kFloor<KIND, FMT>;
  static constexpr int kMask = KIND == BRC_STE_MXFP8 ? kSpans : 15;
  static constexpr int kBlocks = kScaleBlocks<KIND, D>;
  static constexpr int kWords = (kBlocks + 3) / 4;
  static constexpr int kOwn = kBlocks == 8 ? 2 : 1;  // channel blocks of a lane's outputs
  float o[NT][S::kTiles][4];  // [elements 2j, 2j + 1][rows 2c, 2c + 1]
  float m[NT][2], l[NT][2];   // shift and (the lane's part of the) sum of rows 2c, 2c + 1
  // What values are relative to: this lane's own (biased exponents), and in MXFP8 all of
  // the warp's as the check wants them, and what keys are relative to
  int e[kOwn];
  Near<kMask> near[kWords];
  uint32_t ke;

  // A lane's outputs are of one block (heads of 256: of two, one in each word of bytes):
  // elements 16 (lane / 4) .. or, in heads of 64, 8 (lane / 4) ..
  __device__ static __forceinline__ int byte_of(int lane) {
    return kBlocks == 1 ? 0 : kBlocks == 2 ? lane >> 4 : lane >> 3;
  }
  __device__ __forceinline__ Warp() {
#pragma unroll
    for (int i = 0; i < NT; ++i) {
#pragma unroll
      for (int j = 0; j < S::kTiles; ++j) o[i][j][0] = o[i][j][1] = o[i][j][2] = o[i][j][3] = 0.f;
      m[i][0] = m[i][1] = -INFINITY;
      l[i][0] = l[i][1] = 0.f;
    }
#pragma unroll
    for (int w = 0; w < kWords; ++w)
      near[w] = Near<kMask>(kSpans * (kBlocks == 1 ? 1u : kBlocks == 2 ? 0x0101u : 0x01010101u));
#pragma unroll
    for (int i = 0; i < kOwn; ++i) e[i] = KIND == BRC_STE_NVFP4 ? 127 : kSpans;
    ke = 0;
  }
  // What the values are relative to becomes `refs`; o is still zero.
  __device__ __forceinline__ void start(const uint32_t (&refs)[kWords], int lane) {
#pragma unroll
    for (int i = 0; i < kWords; ++i) {
      near[i] = Near<kMask>(refs[i]);
      e[i] = (int)((refs[i] >> (8 * byte_of(lane))) & 0xFFu);
    }
  }
  // The same where o is not; not so low that its largest element passes 2^100.
  __device__ __forceinline__ void move(const uint32_t (&refs)[kWords], int lane) {
    uint32_t to[kWords];
#pragma unroll
    for (int i = 0; i < kWords; ++i) {
      float most = 0.f;
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int j = i * (S::kTiles / kOwn); j < (i + 1) * (S::kTiles / kOwn); ++j)
#pragma unroll
          for (int y = 0; y < 4; ++y)
            if (isfinite(o[n][j][y])) most = fmaxf(most, fabsf(o[n][j][y]));
      const int room = 227 - (int)(__float_as_uint(most) >> 23);
      // a lane's bound for its block, then the block's: the largest of its lanes'
      const int own = max((int)((refs[i] >> (8 * byte_of(lane))) & 0xFFu),
                          most == 0.f ? 0 : e[i] - room);
      to[i] = 0;
#pragma unroll
      for (int y = 0; y < (kBlocks < 4 ? kBlocks : 4); ++y)
        to[i] |= __reduce_max_sync(0xFFFFFFFFu, byte_of(lane) == y ? (uint32_t)own : 0u) << (8 * y);
      const int by = max(e[i] - (int)((to[i] >> (8 * byte_of(lane))) & 0xFFu), -127);
      const float f = kv::pow2i(by - by / 2), f2 = kv::pow2i(by / 2);
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int j = i * (S::kTiles / kOwn); j < (i + 1) * (S::kTiles / kOwn); ++j)
#pragma unroll
          for (int y = 0; y < 4; ++y) o[n][j][y] = o[n][j][y] * f * f2;
    }
    start(to, lane);
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

__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
  uint32_t d;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(x));
  return d;
}

template <int KIND, int FMT, int D, int NT>
struct Step {
  using S = Shape<KIND, D>;
  using W = Warp<KIND, FMT, D, NT>;
  static constexpr int kSub = S::kSub;

  // s[u][nt][2 h + x]: score of token 16 u + r + 8 h and row 2c + x, in units of
  // the rows' factors. `live`: the tokens of this pass (the others' scales are not to
  // be looked at). ANY: MXFP8, their scales are not all near the reference.
  template <bool ANY>
  __device__ static __forceinline__ void scores(const W& w, const uint8_t* st, const uint4* q,
                                                int lane, uint32_t live, float (&s)[kSub][NT][4]) {
    const int r = lane >> 2, c = lane & 3;
#pragma unroll
    for (int u = 0; u < kSub; ++u)
#pragma unroll
      for (int i = 0; i < NT; ++i) s[u][i][0] = s[u][i][1] = s[u][i][2] = s[u][i][3] = 0.f;
    constexpr int kReads = S::kKeyWords / S::kKeyRead;
    uint32_t f[kSub][2][kReads];  // scales of a read's codes
    if constexpr (KIND == BRC_STE_MXFP8) {
      int e[kSub][2][kReads];
#pragma unroll
      for (int u = 0; u < kSub; ++u)
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
          for (int i = 0; i < kReads; ++i) {
            // read i holds elements 64 i + 16 c ..: block 2 i + c / 2
            const int t = 16 * u + 8 * n + r;
            e[u][n][i] = st[S::kKeyScales + t * S::kScales + 2 * i + (c >> 1)];
            if (live != S::kAll && !((live >> t) & 1u)) e[u][n][i] = 0;
          }
#pragma unroll
      for (int u = 0; u < kSub; ++u)
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
          for (int i = 0; i < kReads; ++i)
            f[u][n][i] = half2_pow2<ANY>(e[u][n][i], e[u][n][i], (int)w.ke);
    }
#pragma unroll
    for (int i = 0; i < kReads; ++i) {
      uint32_t x[kSub][2][S::kKeyRead];
#pragma unroll
      for (int u = 0; u < kSub; ++u)
#pragma unroll
        for (int n = 0; n < 2; ++n) {
          const int t = 16 * u + 8 * n + r;
          lds_words<S::kKeyRead>(st + (S::key_offset(lane, i) + (16 * u + 8 * n) * S::kRowBytes),
                                 x[u][n]);
          if constexpr (S::kFp4) {
            // a read is one or two 16-element blocks with their scales
            const uint8_t* sp = st + S::kKeyScales + t * S::kScales;
            if constexpr (D == 64) f[u][n][i] = sp[c];
            else f[u][n][i] = *reinterpret_cast<const uint16_t*>(sp + 8 * i + 2 * c);
          }
        }
#pragma unroll
      for (int y = 0; y < S::kKeyRead; ++y) {
        constexpr int kPer = S::kFp4 ? 2 : 1;  // products to a word
        uint4 a[kSub][kPer];
#pragma unroll
        for (int u = 0; u < kSub; ++u) {
          if constexpr (S::kFp4) {
            const uint32_t sel = y < 2 ? 0x0000 : 0x0011;
            const uint32_t g0 = fp8x2_to_f16x2<BRC_FP8_E4M3>(__byte_perm(f[u][0][i], 0, sel));
            const uint32_t g1 = fp8x2_to_f16x2<BRC_FP8_E4M3>(__byte_perm(f[u][1][i], 0, sel));
            uint32_t h0[4], h1[4];
            e2m1x8_to_f16x8(x[u][0][y], h0);
            e2m1x8_to_f16x8(x[u][1][y], h1);
#pragma unroll
            for (int z = 0; z < 2; ++z)
              a[u][z] = make_uint4(hmul2(h0[2 * z], g0), hmul2(h1[2 * z], g1),
                                   hmul2(h0[2 * z + 1], g0), hmul2(h1[2 * z + 1], g1));
          } else {
            fp8x4_to_f16x4<FMT>(x[u][0][y], a[u][0].x, a[u][0].z);
            fp8x4_to_f16x4<FMT>(x[u][1][y], a[u][0].y, a[u][0].w);
            if constexpr (KIND == BRC_STE_MXFP8) {
              a[u][0].x = hmul2(a[u][0].x, f[u][0][i]);
              a[u][0].y = hmul2(a[u][0].y, f[u][1][i]);
              a[u][0].z = hmul2(a[u][0].z, f[u][0][i]);
              a[u][0].w = hmul2(a[u][0].w, f[u][1][i]);
            }
          }
        }
        const int ks = kPer * (S::kKeyRead * i + y);
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          const uint4 b = q[(n * (S::kSteps / 2) + ks / 2) * 32 + lane];
#pragma unroll
          for (int u = 0; u < kSub; ++u) {
            if constexpr (S::kFp4) {
              mma(s[u][n], a[u][0], b.x, b.y);
              mma(s[u][n], a[u][1], b.z, b.w);
            } else {
              if (ks & 1) mma(s[u][n], a[u][0], b.z, b.w);
              else mma(s[u][n], a[u][0], b.x, b.y);
            }
          }
        }
      }
    }
    if constexpr (KIND == BRC_STE_BLOCK_FP8) {  // the token's own factor
#pragma unroll
      for (int u = 0; u < kSub; ++u) {
        const float* g = reinterpret_cast<const float*>(st + S::kKeyScales) + 16 * u + r;
        const float g0 = g[0], g1 = g[8];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          s[u][n][0] *= g0;
          s[u][n][1] *= g0;
          s[u][n][2] *= g1;
          s[u][n][3] *= g1;
        }
      }
    }
  }

  // Running maximum and sum; s becomes the probabilities relative to the shift.
  __device__ static __forceinline__ void softmax(W& w, float (&s)[kSub][NT][4]) {
    bool grow = false;
    float top[NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        top[n][x] = fmaxf(s[0][n][x], s[0][n][2 + x]);
        if constexpr (kSub == 2) top[n][x] = fmaxf(top[n][x], fmaxf(s[kSub - 1][n][x], s[kSub - 1][n][2 + x]));
        grow |= top[n][x] > w.m[n][x] + kGrow;
      }
    if (__any_sync(0xFFFFFFFFu, grow)) {
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          float t = top[n][x];
          t = fmaxf(t, __shfl_xor_sync(0xFFFFFFFFu, t, 4));
          t = fmaxf(t, __shfl_xor_sync(0xFFFFFFFFu, t, 8));
          t = fmaxf(t, __shfl_xor_sync(0xFFFFFFFFu, t, 16));
          const float m = fmaxf(w.m[n][x], t);
          const float f = m == w.m[n][x] ? 1.f : ex2(w.m[n][x] - m);
          w.m[n][x] = m;
          w.l[n][x] *= f;
#pragma unroll
          for (int j = 0; j < S::kTiles; ++j) {
            w.o[n][j][x] *= f;
            w.o[n][j][2 + x] *= f;
          }
        }
    }
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const float m = w.m[n][x] == -INFINITY ? 0.f : w.m[n][x];
#pragma unroll
        for (int u = 0; u < kSub; ++u) {
          s[u][n][x] = ex2(s[u][n][x] - m);
          s[u][n][2 + x] = ex2(s[u][n][2 + x] - m);
          w.l[n][x] += s[u][n][x] + s[u][n][2 + x];
        }
      }
  }

  // o += v^T p. Probabilities carry a factor 2^6 (at most 2^8 before it), so that
  // f16 keeps those down to 2^-30 of the largest. TWO: a second product with
  // what the rounding to f16 left (f16 outputs of few rows: its 2^-11 would
  // show beside the output's own).
  template <bool TWO, bool ANY>
  __device__ static __forceinline__ void values(W& w, const uint8_t* st, int lane, uint32_t live,
                                                const float (&p)[kSub][NT][4]) {
    const int r = lane >> 2, c = lane & 3;
    auto token = [&](int u, int t) { return 16 * u + 2 * c + (t & 1) + 8 * (t >> 1); };
    const bool all = live == S::kAll;
    constexpr int kReads = S::kValWords / S::kValRead;
    float f[kSub][2];        // factor of tokens r, r + 8
    uint32_t h[kSub][2][2];  // [token pair][half of the lane's elements]: f16 pair of value factors
    if constexpr (KIND == BRC_STE_BLOCK_FP8) {
      const float* sp = reinterpret_cast<const float*>(st + S::kValScales);
      const float g = __uint_as_float((uint32_t)(254 + 6 - w.e[0]) << 23);
#pragma unroll
      for (int u = 0; u < kSub; ++u)
#pragma unroll
        for (int n = 0; n < 2; ++n) {
          const int t = 16 * u + 8 * n + r;
          f[u][n] = !all && !((live >> t) & 1u) ? 0.f : sp[t] * g;
        }
    } else if constexpr (KIND == BRC_STE_MXFP8) {
      int e[kSub][4][2];
#pragma unroll
      for (int u = 0; u < kSub; ++u)
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
          for (int i = 0; i < kReads; ++i) {
            const int blk = D == 64 ? r >> 2 : 4 * i + (r >> 1);
            e[u][t][i] = st[S::kValScales + token(u, t) * S::kScales + blk];
            if (!all && !((live >> token(u, t)) & 1u)) e[u][t][i] = 0;
          }
#pragma unroll
      for (int u = 0; u < kSub; ++u)
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          f[u][t] = 64.f;
#pragma unroll
          for (int i = 0; i < kReads; ++i)
            h[u][t][i] = half2_pow2<ANY>(e[u][2 * t][i], e[u][2 * t + 1][i], w.e[i]);
        }
    } else {
#pragma unroll
      for (int u = 0; u < kSub; ++u)
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          f[u][t] = 64.f;
          uint32_t g[2];
#pragma unroll
          for (int y = 0; y < 2; ++y) {
            const int tk = token(u, 2 * t + y);
            const uint8_t* sp = st + S::kValScales + tk * S::kScales;
            if constexpr (D == 256) g[y] = *reinterpret_cast<const uint16_t*>(sp + 2 * r);
            else g[y] = sp[D == 128 ? r : r >> 1];
            if (!all && !((live >> tk) & 1u)) g[y] = 0;
          }
          h[u][t][0] = fp8x2_to_f16x2<BRC_FP8_E4M3>(__byte_perm(g[0], g[1], 0x0040));
          if constexpr (D == 256)
            h[u][t][1] = fp8x2_to_f16x2<BRC_FP8_E4M3>(__byte_perm(g[0], g[1], 0x0051));
        }
    }
    uint32_t b[kSub][NT][2], b2[kSub][NT][2];
#pragma unroll
    for (int u = 0; u < kSub; ++u)
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int y = 0; y < 2; ++y) {
          const float v0 = p[u][n][2 * y] * f[u][y], v1 = p[u][n][2 * y + 1] * f[u][y];
          const uint32_t hi = half2_of(v0, v1);
          b[u][n][y] = transpose8(hi);
          if constexpr (TWO) {
            const float2 g = __half22float2(*reinterpret_cast<const __half2*>(&hi));
            b2[u][n][y] = transpose8(half2_of(v0 - g.x, v1 - g.y));
          }
        }
#pragma unroll
    for (int i = 0; i < kReads; ++i) {
      uint32_t x[kSub][4][S::kValRead];
#pragma unroll
      for (int u = 0; u < kSub; ++u)
#pragma unroll
        for (int t = 0; t < 4; ++t) {
          const uint8_t* q = st + (S::kTileBytes + S::val_offset(lane, i) +
                                   (16 * u + (t & 1) + 8 * (t >> 1)) * S::kRowBytes);
          lds_words<S::kValRead>(q, x[u][t]);
        }
      if (!all) {  // rows without a token hold anything
#pragma unroll
        for (int u = 0; u < kSub; ++u)
#pragma unroll
          for (int t = 0; t < 4; ++t)
#pragma unroll
            for (int y = 0; y < S::kValRead; ++y)
              if (!((live >> token(u, t)) & 1u)) x[u][t][y] = 0;
      }
#pragma unroll
      for (int y = 0; y < S::kValRead; ++y)
#pragma unroll
        for (int u = 0; u < kSub; ++u) {
          constexpr int kPer = S::kFp4 ? 8 : 4;  // elements to a word
          uint32_t a[2][kPer];
#pragma unroll
          for (int t = 0; t < 2; ++t) {
            const uint32_t v0 = x[u][2 * t][y], v1 = x[u][2 * t + 1][y];
            if constexpr (S::kFp4) {
              uint32_t lo[4], hi[4];
              e2m1x8_to_f16x8((v0 & 0x0F0F0F0Fu) | ((v1 & 0x0F0F0F0Fu) << 4), lo);
              e2m1x8_to_f16x8(((v0 >> 4) & 0x0F0F0F0Fu) | (v1 & 0xF0F0F0F0u), hi);
              const uint32_t g = h[u][t][D == 256 ? y / 2 : 0];
#pragma unroll
              for (int z = 0; z < 4; ++z) {
                a[t][2 * z] = hmul2(lo[z], g);
                a[t][2 * z + 1] = hmul2(hi[z], g);
              }
            } else {
              fp8x4_to_f16x4<FMT>(__byte_perm(v0, v1, 0x5140), a[t][0], a[t][1]);
              fp8x4_to_f16x4<FMT>(__byte_perm(v0, v1, 0x7362), a[t][2], a[t][3]);
              if constexpr (KIND == BRC_STE_MXFP8) {
#pragma unroll
                for (int z = 0; z < 4; ++z) a[t][z] = hmul2(a[t][z], h[u][t][i]);
              }
            }
          }
#pragma unroll
          for (int z = 0; z < kPer / 2; ++z) {
            const uint4 av = make_uint4(a[0][2 * z], a[0][2 * z + 1], a[1][2 * z], a[1][2 * z + 1]);
            const int j = kPer / 2 * (S::kValRead * i + y) + z;
#pragma unroll
            for (int n = 0; n < NT; ++n) {
              mma(w.o[n][j], av, b[u][n][0], b[u][n][1]);
              if constexpr (TWO) mma(w.o[n][j], av, b2[u][n][0], b2[u][n][1]);
            }
          }
        }
    }
  }

  // One token to a lane: its scales' bytes.
  struct Token {
    uint32_t k[1][W::kWords], v[1][W::kWords];  // (keys: MXFP8)
    __device__ __forceinline__ Token(const uint8_t* st, int t) {
      if constexpr (KIND == BRC_STE_BLOCK_FP8) {
        v[0][0] = (reinterpret_cast<const uint32_t*>(st + S::kValScales)[t] >> 23) & 0xFFu;
      } else if constexpr (KIND == BRC_STE_MXFP8) {
        const uint8_t* const pk = st + S::kKeyScales + t * S::kScales;
        const uint8_t* const pv = st + S::kValScales + t * S::kScales;
        if constexpr (D == 64) {
          k[0][0] = *reinterpret_cast<const uint16_t*>(pk);
          v[0][0] = *reinterpret_cast<const uint16_t*>(pv);
        } else {
          lds_words<W::kWords>(pk, k[0]);
          lds_words<W::kWords>(pv, v[0]);
        }
      }
    }
    // Whether the references hold it.
    __device__ __forceinline__ bool fits(const W& w) const {
      if constexpr (KIND == BRC_STE_BLOCK_FP8) return w.e[0] - v[0][0] <= (uint32_t)W::kSpans;
      bool in = w.ke - top_key() <= (uint32_t)W::kSpans;
#pragma unroll
      for (int i = 0; i < W::kWords; ++i) in &= w.near[i](v[0][i]);
      return in;
    }
    // The same, scales as of zeros left out.
    __device__ __forceinline__ bool fits_but_zeros(const uint32_t (&refs)[W::kWords],
                                                   uint32_t ke) const {
      bool in = true;
      if constexpr (KIND == BRC_STE_BLOCK_FP8) {
        in = refs[0] - v[0][0] <= (uint32_t)W::kSpans || (v[0][0] <= W::kZero && v[0][0] <= refs[0]);
      } else {
#pragma unroll
        for (int i = 0; i < W::kWords; ++i) {
          const uint32_t zero = __vcmpleu4(v[0][i], __vminu4(refs[i], W::kZero * 0x01010101u));
          in &= Near<W::kMask>(refs[i])((v[0][i] & ~zero) | (refs[i] & zero));
        }
        const uint32_t k = top_key();
        in &= ke - k <= (uint32_t)W::kSpans || (k <= W::kZero && k <= ke);
      }
      return in;
    }
    __device__ __forceinline__ uint32_t top_key() const {
      uint32_t m = 0;
#pragma unroll
      for (int i = 0; i < W::kWords; ++i)
        m = __vmaxu2(m, __vmaxu2(k[0][i] & 0x00FF00FFu, (k[0][i] >> 8) & 0x00FF00FFu));
      return max(m & 0xFFFFu, m >> 16);
    }
  };
  // References that hold the tokens of lanes with `on`, if they go together.
  __device__ static __forceinline__ void around(const Token& mine, bool on,
                                                uint32_t (&refs)[W::kWords], uint32_t& ke) {
#pragma unroll
    for (int i = 0; i < W::kWords; ++i) {
      refs[i] = 0;
#pragma unroll
      for (int y = 0; y < 8 * (W::kBlocks < 4 ? W::kBlocks : 4); y += 8) {
        const uint32_t top = __reduce_max_sync(0xFFFFFFFFu, on ? (mine.v[0][i] >> y) & 0xFFu : 0u);
        refs[i] |= min(max(top + kSlack, (uint32_t)W::kSpans), 254u) << y;
      }
    }
    ke = 0;
    if constexpr (KIND == BRC_STE_MXFP8)
      ke = min(__reduce_max_sync(0xFFFFFFFFu, on ? mine.top_key() : 0u) + kSlack, 254u);
  }
  __device__ static __forceinline__ void first(W& w, const Token& mine, int lane, uint32_t live) {
    uint32_t refs[W::kWords];
    around(mine, (live >> (lane % S::kRows)) & 1u, refs, w.ke);
    w.start(refs, lane);
  }
  // Moves the references to a step that they do not hold. False (and nothing moves) if its
  // tokens do not go together, or if o might leave float32: o falls with references that
  // climb, which only what a row sees may cause, so drafted tokens climb little, and it
  // grows with references that fall.
  __device__ static __forceinline__ bool follow(W& w, const Token& mine, int lane, bool on,
                                                bool drafted, Later& later) {
    uint32_t refs[W::kWords], ke = w.ke;
#pragma unroll
    for (int i = 0; i < W::kWords; ++i)
      refs[i] = KIND == BRC_STE_BLOCK_FP8 ? (uint32_t)w.e[0] : w.near[i].refs();
    if (__all_sync(0xFFFFFFFFu, !on || mine.fits_but_zeros(refs, ke))) return true;
    around(mine, on, refs, ke);
    const bool in = mine.fits_but_zeros(refs, ke);
    int climb = 0, fall = 0, own[W::kOwn];
#pragma unroll
    for (int i = 0; i < W::kWords; ++i) {
      own[i] = (int)((refs[i] >> (8 * W::byte_of(lane))) & 0xFFu);
      climb = max(climb, own[i] - w.e[i]);
      fall = max(fall, w.e[i] - own[i]);
    }
    climb = drafted ? (int)__reduce_max_sync(0xFFFFFFFFu, climb) + later.climb : later.climb;
    fall = (int)__reduce_max_sync(0xFFFFFFFFu, fall) + later.fall;
    if (!__all_sync(0xFFFFFFFFu, !on || in) || climb > 60 || fall > 60) return false;
    __syncwarp();
    if (lane == 0) {
      later.climb = climb;
      later.fall = fall;
    }
#pragma unroll
    for (int i = 0; i < W::kOwn; ++i) {
      const float f = kv::pow2i(max(w.e[i] - own[i], -126));
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int j = i * (S::kTiles / W::kOwn); j < (i + 1) * (S::kTiles / W::kOwn); ++j)
#pragma unroll
          for (int y = 0; y < 4; ++y) w.o[n][j][y] *= f;
    }
    w.start(refs, lane);
    w.ke = ke;
    return true;
  }
  // Takes tokens that go together out of `left`, moves the references to them and
  // returns them; tokens that no row sees (`seen` says) are dropped, whatever they hold.
  template <class Seen>
  __device__ static __forceinline__ uint32_t pick(W& w, const uint8_t* st, int lane, uint32_t& left,
                                                  const Seen& seen) {
    const Token mine(st, lane % S::kRows);
    uint32_t taken = 0;
#pragma unroll 1
    while (left) {  // (choose takes one token at least)
      uint32_t km[1] = {0u}, take, refs[W::kWords];
#pragma unroll
      for (int i = 0; i < W::kWords; ++i) {
        refs[i] = KIND == BRC_STE_BLOCK_FP8 ? (uint32_t)w.e[0] : w.near[i].refs();
        if constexpr (KIND == BRC_STE_MXFP8) km[0] = max(km[0], top_byte(mine.k[0][i]));
      }
      const uint32_t k = choose<W::kSpans, W::kZero, W::kBlocks>(
          mine.v, km, (left >> (lane % S::kRows)) & 1u, take, refs);
      const uint32_t group = __ballot_sync(0xFFFFFFFFu, take != 0u) & S::kAll;
      left &= ~group;
      if (seen(group)) {
        taken = group;
        if constexpr (KIND == BRC_STE_MXFP8) {
          if (__any_sync(0xFFFFFFFFu, k > w.ke || (take && km[0] > W::kZero && km[0] + W::kSpans < w.ke)))
            w.ke = min(k + kSlack, 254u);
        }
        w.move(refs, lane);
        break;
      }
    }
    return taken;
  }

  // Does any value of the step's live rows stand for something not finite?
  __device__ static __forceinline__ bool odd_values(const uint8_t* st, int lane, uint32_t live) {
    bool odd = false;
    constexpr int kLanes = 32 / S::kRows;  // to a row
    const int t = lane / kLanes;
    if ((live >> t) & 1u) {
      constexpr int kWords = S::kRowBytes / 4 / kLanes;
      const uint32_t* p = reinterpret_cast<const uint32_t*>(st + S::kTileBytes + t * S::kRowBytes) +
                          (lane % kLanes) * kWords;
      for (int i = 0; i < kWords; ++i) odd |= odd_codes<KIND, FMT>(p[i]);
      const uint8_t* sp = st + S::kValScales + t * S::kScaleBytes;
      if constexpr (KIND == BRC_STE_BLOCK_FP8) {
        odd |= (*reinterpret_cast<const uint32_t*>(sp) & 0x7F800000u) == 0x7F800000u;
      } else {
        for (int i = 0; i < S::kScales; ++i)
          odd |= KIND == BRC_STE_NVFP4 ? (sp[i] & 0x7F) == 0x7F : sp[i] == 255;
      }
    }
    return __any_sync(0xFFFFFFFFu, odd);
  }

  // The same for a step whose values are not all finite: token by token, only
  // where the row sees the token, so that what it does not see cannot reach it.
  // row[u]: the first cache row of tile u; seen: bits (u, n, h, x) as s.
  __device__ static __forceinline__ void values_checked(W& w, const brc_kv_cache& c,
                                                        const int64_t (&row)[kSub], int lane,
                                                        const float (&p)[kSub][NT][4],
                                                        uint32_t live, uint32_t seen) {
    float f[W::kOwn];
#pragma unroll
    for (int i = 0; i < W::kOwn; ++i) f[i] = 64.f * exp2f((float)(127 - w.e[i]));
#pragma unroll
    for (int u = 0; u < kSub; ++u)
      for (int t = 0; t < 16; ++t) {
        if (!((live >> (16 * u + t)) & 1u)) continue;
        const int half = t >> 3, src = (t & 7) * 4 + (lane & 3);
        float pr[NT][2];
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int x = 0; x < 2; ++x)
            pr[n][x] = __shfl_sync(0xFFFFFFFFu, half ? p[u][n][2 + x] : p[u][n][x], src);
        const uint32_t sees = __shfl_sync(0xFFFFFFFFu, seen, src) >> (4 * NT * u + 2 * half);
#pragma unroll
        for (int j = 0; j < S::kTiles; ++j)
#pragma unroll
          for (int y = 0; y < 2; ++y) {
            const float v = value_at<KIND, FMT, D>(c, row[u] + t, S::elem(2 * j + y, lane >> 2)) *
                            f[j / (S::kTiles / W::kOwn)];
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
              for (int x = 0; x < 2; ++x)
                if ((sees >> (4 * n + x)) & 1u) w.o[n][j][2 * y + x] += pr[n][x] * v;
          }
      }
  }
};

// An item, as the warps of a block walk it.
struct Item {
  Seq seq;
  int b, page_mask;
  uint32_t head_row;
  const int32_t* table;
  // First cache row of the 16-token tile at token t, or -1.
  __device__ __forceinline__ int64_t row_at(const Args& a, int t) const {
    if (t >= seq.total) return -1;
    const int page = __ldg(table + (t >> a.page_shift));
    if (page < 0 || page >= a.c.num_pages) return -1;
    return (int64_t)((uint64_t)(uint32_t)page * a.page_rows) + (head_row + (t & page_mask));
  }
  // The tokens of the step of ROWS at t0, of whose 16-token tiles `bits` are there.
  template <int ROWS>
  __device__ __forceinline__ uint32_t live_of(int t0, uint32_t bits) const {
    uint32_t live = ROWS == 32 ? 0xFFFFFFFFu : 0xFFFFu;
    if (t0 > seq.total - ROWS) live >>= ROWS - (seq.total - t0);
    if (ROWS == 32 && bits != 3) live &= bits == 1 ? 0xFFFFu : 0xFFFF0000u;
    return live;
  }
  // Whether query `node` sees drafted token j (j < 0: a token of the context).
  __device__ __forceinline__ bool sees(const Args& a, int node, int j) const {
    if (j < 0) return true;
    return a.tree ? a.tree[b * a.tree_stride + (int64_t)node * a.draft + j] != 0 : j <= node;
  }
};
template <int NT>
struct Rows {  // rows 2c, 2c + 1 of a lane's tiles: what a score is times, and their nodes
  float factor[NT][2];
  int node[NT][2];
};

// Adds the tokens `live` of the step at t0 in stage st.
template <int KIND, int FMT, int D, int NT, bool ANY>
__device__ __forceinline__ void add_step(Warp<KIND, FMT, D, NT>& w, const Args& a, const Item& it,
                                         const Rows<NT>& rows, const uint8_t* st, const uint4* q,
                                         int lane, int t0, uint32_t live) {
  using S = Shape<KIND, D>;
  using St = Step<KIND, FMT, D, NT>;
  constexpr int kSub = S::kSub;
  constexpr bool kTwo = NT <= 2;
  float p[kSub][NT][4];
  St::template scores<ANY>(w, st, q, lane, live, p);
  const float kf = KIND == BRC_STE_MXFP8 ? e8m0_value(w.ke) : 1.f;
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      const float f = KIND == BRC_STE_MXFP8 ? rows.factor[n][x] * kf : rows.factor[n][x];
#pragma unroll
      for (int u = 0; u < kSub; ++u) {
        p[u][n][x] *= f;
        p[u][n][2 + x] *= f;
      }
    }
  uint32_t seen = 0;
  bool checked = false;
  if (t0 > it.seq.context - S::kRows || live != S::kAll) {  // drafted tokens, or none
#pragma unroll
    for (int u = 0; u < kSub; ++u)
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            const int at = 16 * u + 8 * h + (lane >> 2);
            if (((live >> at) & 1u) && rows.node[n][x] < it.seq.drafts &&
                it.sees(a, rows.node[n][x], t0 - it.seq.context + at))
              seen |= 1u << (4 * (NT * u + n) + 2 * h + x);
            else p[u][n][2 * h + x] = -INFINITY;
          }
    // a drafted value that is not finite must not meet a probability of
    // zero in the product
    checked = St::odd_values(st, lane, live);
  }
  St::softmax(w, p);
  if (checked) {
    int64_t at[kSub];
#pragma unroll
    for (int u = 0; u < kSub; ++u) at[u] = it.row_at(a, t0 + 16 * u);
    St::values_checked(w, a.c, at, lane, p, live, seen);
  } else if constexpr (kTwo) {
    if (a.q_f16) St::template values<true, ANY>(w, st, lane, live, p);
    else St::template values<false, ANY>(w, st, lane, live, p);
  } else {
    St::template values<false, ANY>(w, st, lane, live, p);
  }
}

// The same for the steps that were put off, and those from `s` on, in passes, each with
// tokens that go together. A function of its own, called after the usual steps with the
// warp's state handed over in memory: it is rare, and inlined, or called between them, it
// costs them registers (32 rows of MXFP8: 118 -> 134 us). `ring`: the warp's, free now.
template <int KIND, int FMT, int D, int NT>
struct Passes {
  Warp<KIND, FMT, D, NT> w;
  Item it;
  Rows<NT> rows;
};
template <int KIND, int FMT, int D, int NT>
__device__ __noinline__ void add_in_passes(Passes<KIND, FMT, D, NT>& x, const Args& a,
                                           uint8_t* ring, const uint4* q, int lane,
                                           const Later& later, int s, int s_end, int stride) {
  using S = Shape<KIND, D>;
  using St = Step<KIND, FMT, D, NT>;
  Warp<KIND, FMT, D, NT> w = x.w;
  const uint32_t to = (uint32_t)__cvta_generic_to_shared(ring);
  int put_off = 0;
#pragma unroll 1
  while (true) {
    int t0;
    if (put_off < later.count) {
      t0 = later.step[put_off++] * S::kRows;
    } else if (s < s_end) {
      t0 = s * S::kRows;
      s += stride;
    } else {
      break;
    }
    uint32_t bits = 0;
    for (int u = 0; u < S::kSub; ++u) {
      const int64_t row = x.it.row_at(a, t0 + 16 * u);
      if (row < 0) continue;
      copy_tile<KIND, D>(a.c, row, lane, to, u);
      bits |= 1u << u;
    }
    cp_commit();
    cp_wait<0>();
    __syncwarp();
    uint32_t live = bits ? x.it.template live_of<S::kRows>(t0, bits) : 0u;
    auto seen = [&](uint32_t tokens) {
      if (t0 <= x.it.seq.context - S::kRows) return true;
      bool see = false;
      for (int at = 0; at < S::kRows; ++at) {
        if (!((tokens >> at) & 1u)) continue;
        for (int n = 0; n < NT; ++n)
          for (int i = 0; i < 2; ++i)
            see |= x.rows.node[n][i] < x.it.seq.drafts &&
                   x.it.sees(a, x.rows.node[n][i], t0 - x.it.seq.context + at);
      }
      return __any_sync(0xFFFFFFFFu, see) != 0;
    };
#pragma unroll 1
    for (int pass = 0; pass < S::kRows && live; ++pass) {
      const uint32_t take = St::pick(w, ring, lane, live, seen);
      if (take) add_step<KIND, FMT, D, NT, true>(w, a, x.it, x.rows, ring, q, lane, t0, take);
    }
    __syncwarp();  // the stage is read
  }
  x.w = w;
}

// Blocks that an SM is to hold, as many as the accumulators' registers allow.
constexpr __host__ __device__ int blocks_per_sm(int kind, int d, int nt) {
  if (kind == BRC_STE_NVFP4 && d * nt == 128) return 4;
  // (with the check of the references a third block spills: 16 rows, 8 sequences of 16384
  // tokens, block FP8 76 us with three blocks and 73 with two, MXFP8 83 and 81)
  if (kind != BRC_STE_NVFP4 && d == 128 && nt == 2) return 2;
  return d * nt <= 64 ? 4 : d * nt <= 256 ? 3 : 2;
}
// Stages of a warp's ring: what fits beside the queries in the block's part of
// shared memory, at most 6.
constexpr __host__ __device__ int stage_bytes(int kind, int d) {
  return 2 * 16 * subtiles(d) *
         (kv::row_bytes(kind, d) + kv::row_scales(kind, d) * (kind == BRC_STE_BLOCK_FP8 ? 4 : 1));
}
// Row warps of a block: more than one only with the largest row tile.
constexpr __host__ __device__ int most_tiles(int d) { return d == 256 ? 2 : 4; }
constexpr __host__ __device__ int query_bytes(int d, int nt) {
  return (nt == most_tiles(d) ? kWarps : 1) * 8 * nt * d * 2;
}
constexpr __host__ __device__ int stages(int kind, int d, int nt) {
  const int room = (227 * 1024) / blocks_per_sm(kind, d, nt) - 2048 - query_bytes(d, nt);
  const int n = room / (kWarps * stage_bytes(kind, d));
  return n > 6 ? 6 : n;
}
constexpr __host__ __device__ int ring_bytes(int kind, int d, int nt) {
  const int r = kWarps * stages(kind, d, nt) * stage_bytes(kind, d);
  const int o = kWarps * 8 * nt * (d + 4) * 4;  // the warps' outputs
  return r > o ? r : o;
}

template <int KIND, int FMT, int D, int NT>
__global__ void __launch_bounds__(kThreads, blocks_per_sm(KIND, D, NT))
    k_attend(const __grid_constant__ Args a) {
  using S = Shape<KIND, D>;
  using St = Step<KIND, FMT, D, NT>;
  constexpr int kStages = stages(KIND, D, NT);
  constexpr int kSub = S::kSub;
  extern __shared__ __align__(16) uint8_t smem[];
  // the warps' stages (later: their outputs), then the queries as operand fragments
  uint8_t* const rings = smem;
  float* const so = reinterpret_cast<float*>(smem);
  uint4* const sq = reinterpret_cast<uint4*>(smem + ring_bytes(KIND, D, NT));
  __shared__ float s_m[kWarps][8 * NT], s_l[kWarps][8 * NT], s_rowf[kWarps * 8 * NT];
  __shared__ Place s_place;
  __shared__ Later s_later[kWarps];

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

    // ---- the first stages are on their way while the queries are laid out
    const Item it{seq, b, a.c.page_size - 1, (uint32_t)head * a.c.page_size,
                  a.table + b * a.table_stride};
    // the warp's own ring of stages
    const uint32_t ring = (uint32_t)__cvta_generic_to_shared(rings) + warp * (kStages * S::kStageBytes);
    const uint8_t* const ring_p = rings + warp * (kStages * S::kStageBytes);
    uint32_t there = 0;  // kSub bits to a step, the newest lowest: its tiles that have a page
    int s = s_begin + tw, ahead = s, slot_in = 0, slot_out = 0;
    auto fetch = [&]() {
      uint32_t bits = 0;
      if (ahead < s_end) {
        const int t = ahead * S::kRows;  // (positions fit in 31 bits)
        const uint32_t to = ring + slot_in * S::kStageBytes;
        const int64_t row = it.row_at(a, t);
        if (row >= 0) {
          copy_tile<KIND, D>(a.c, row, lane, to, 0);
          bits = 1;
        }
        if constexpr (kSub == 2) {
          // pages of 32 tokens and more hold the step whole
          const int64_t row1 = a.page_shift > 4 ? (row >= 0 && t + 16 < seq.total ? row + 16 : -1)
                                                : it.row_at(a, t + 16);
          if (row1 >= 0) {
            copy_tile<KIND, D>(a.c, row1, lane, to, 1);
            bits |= 2;
          }
        }
      }
      cp_commit();
      there = there << kSub | bits;
      ahead += token_warps;
      slot_in = slot_in + 1 == kStages ? 0 : slot_in + 1;
    };
#pragma unroll
    for (int i = 0; i < kStages - 1; ++i) fetch();

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
          const uint4 v = ldg16(static_cast<const uint16_t*>(a.q) + at);
          if (a.q_f16) unpack<BRC_DTYPE_F16>(v, f);
          else unpack<BRC_DTYPE_BF16>(v, f);
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
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int d = d0 + 2 * i;  // pair d, d + 1
          int ks, c, j;
          if constexpr (S::kFp4) {
            constexpr int kLane = 8 * S::kKeyRead;  // elements of a lane's chunk
            const int in = d % (4 * kLane);
            c = in / kLane;
            ks = (d / (4 * kLane)) * (2 * S::kKeyRead) + (in % kLane) / 4;
            j = d % 4;
          } else {
            c = (d % 64) / 16;
            ks = (d / 64) * 4 + (d % 16) / 4;
            j = d % 4;
          }
          dst[(((rr >> 3) * (S::kSteps / 2) + ks / 2) * 32 + (rr & 7) * 4 + c) * 4 + (ks & 1) * 2 + (j >> 1)] =
              half2_of(f[2 * i] * up, f[2 * i + 1] * up);
        }
      }
    }
    __syncthreads();

    Warp<KIND, FMT, D, NT> w;
    const uint4* const q = sq + rw * NT * (S::kSteps / 2) * 32;
    Rows<NT> rows;
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const int rr = (rw * NT + n) * 8 + 2 * (lane & 3) + x;
        rows.factor[n][x] = s_rowf[rr];
        const int row = row0 + rr;
        rows.node[n][x] = row < a.rows ? row / a.group : a.draft;
      }

    auto live_of = [&](int t0, uint32_t bits) { return it.template live_of<S::kRows>(t0, bits); };
    if constexpr (KIND != BRC_STE_NVFP4) {
      cp_wait<kStages - 2>();
      __syncwarp();
      const uint32_t bits = there >> ((kStages - 2) * kSub) & ((1u << kSub) - 1);
      if (s < s_end && bits)
        St::first(w, typename St::Token(ring_p, lane % S::kRows), lane, live_of(s * S::kRows, bits));
    }
    Later& later = s_later[warp];
    if (lane == 0) later.count = later.climb = later.fall = 0;
    __syncwarp();
    for (; s < s_end; s += token_warps) {
      cp_wait<kStages - 2>();
      __syncwarp();  // every lane's pieces are there, and the oldest stage is read
      fetch();
      const uint32_t bits = there >> ((kStages - 1) * kSub) & ((1u << kSub) - 1);
      bool now = bits != 0;
      if (now) {
        const uint8_t* const st = ring_p + slot_out * S::kStageBytes;
        const uint32_t live = live_of(s * S::kRows, bits);
        if constexpr (KIND != BRC_STE_NVFP4) {
          const typename St::Token mine(st, lane % S::kRows);
          const bool on = (live >> (lane % S::kRows)) & 1u;
          if (!__all_sync(0xFFFFFFFFu, !on || mine.fits(w))) {
            now = St::follow(w, mine, lane, on, s * S::kRows > seq.context - S::kRows, later);
            if (!now) {
              const int n = later.count;
              if (n == Later::kMost) break;  // the rest of the share, then
              __syncwarp();
              if (lane == 0) {
                later.step[n] = s;
                later.count = n + 1;
              }
              __syncwarp();
            }
          }
        }
        if (now) add_step<KIND, FMT, D, NT, false>(w, a, it, rows, st, q, lane, s * S::kRows, live);
      }
      slot_out = slot_out + 1 == kStages ? 0 : slot_out + 1;
    }
    if constexpr (KIND != BRC_STE_NVFP4) {
      if (later.count || s < s_end) {
        cp_wait<0>();
        __syncwarp();
        Passes<KIND, FMT, D, NT> x{w, it, rows};
        add_in_passes<KIND, FMT, D, NT>(x, a, rings + warp * (kStages * S::kStageBytes), q, lane,
                                        later, s, s_end, token_warps);
        w = x.w;
      }
    }
    cp_wait<0>();

    // ---- join the warps that share rows
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        float l = w.l[n][x];
        l += __shfl_xor_sync(0xFFFFFFFFu, l, 4);
        l += __shfl_xor_sync(0xFFFFFFFFu, l, 8);
        l += __shfl_xor_sync(0xFFFFFFFFu, l, 16);
        if (lane < 4) {
          s_m[warp][8 * n + 2 * lane + x] = w.m[n][x];
          s_l[warp][8 * n + 2 * lane + x] = l;
        }
      }
    __syncthreads();  // the stages are no longer read
    constexpr int kPitch = D + 4;
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int x = 0; x < 2; ++x)
#pragma unroll
        for (int j = 0; j < S::kTiles; j += 2) {
          const float scale_o = exp2f((float)(w.e[j / (S::kTiles / w.kOwn)] - 133 - kSumDown));
          const int rr = 8 * n + 2 * (lane & 3) + x;
          *reinterpret_cast<float4*>(so + (warp * 8 * NT + rr) * kPitch + S::elem(2 * j, lane >> 2)) =
              make_float4(w.o[n][j][x] * scale_o, w.o[n][j][2 + x] * scale_o,
                          w.o[n][j + 1][x] * scale_o, w.o[n][j + 1][2 + x] * scale_o);
        }
    __syncthreads();
    const bool whole = s_begin == 0 && s_end == seq.steps;
    const int64_t slot = 2 * (int64_t)blockIdx.x + (s_begin > 0 ? 0 : 1);
    for (int at = tid; at < rows_per_block * (D / 4); at += kThreads) {
      const int rr = at / (D / 4), d = (at - rr * (D / 4)) * 4;
      const int row = row0 + rr;
      if (row >= a.rows) continue;
      const int w0 = rr / (8 * NT), r = rr - w0 * 8 * NT;  // row warp, row in its tile
      float m = -INFINITY;
      for (int t = 0; t < token_warps; ++t) m = fmaxf(m, s_m[t * row_warps + w0][r]);
      float l = 0.f, o[4] = {0.f, 0.f, 0.f, 0.f};
      for (int t = 0; t < token_warps; ++t) {
        const int wi = t * row_warps + w0;
        const float f = m == -INFINITY ? 1.f : ex2(s_m[wi][r] - m);
        l += s_l[wi][r] * f;
        const float4 y = *reinterpret_cast<const float4*>(so + (wi * 8 * NT + r) * kPitch + d);
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
        const float inv = none ? 0.f : kSumUp / l;
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
    if (x >= end) asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    if (s_end == seq.steps && item + 1 == per_seq) {
      seq_start += (int64_t)per_seq * seq.steps;
      ++b;
    }
  }
}

// Join the parts of items that several blocks share, in the order of their tokens. A
// warp takes the R rows of one block: finding an item's parts takes more instructions
// than adding up a row of them, and the rows' loads are in flight together (8 trees of
// 64 nodes over 16384 tokens, caches cold: one row to a warp 36 us, eight one by one
// 29, eight together 20).
__host__ __device__ __forceinline__ int join_rows(int rows_per_block) {
  return rows_per_block <= 32 ? 1 : rows_per_block / 32;
}

template <int D, int R>
__global__ void __launch_bounds__(kThreads) k_join(Args a, int blocks) {
  const int lane = threadIdx.x & 31;
  const int64_t id = (int64_t)blockIdx.x * kWarps + (threadIdx.x >> 5);
  const int units = a.rows_per_block / R, per_head = a.row_blocks * units;
  const int64_t per_b = (int64_t)a.c.heads * per_head;
  if (id >= per_b * a.batch) return;
  const int b = (int)(id / per_b);
  const int rest = (int)(id - b * per_b);
  const int head = rest / per_head, unit = rest - head * per_head;
  const int rb = unit / units, first = (unit - rb * units) * R;
  const int row0 = rb * a.rows_per_block + first;
  if (row0 >= a.rows) return;
  const int per_seq = a.c.heads * a.row_blocks;
  Place p;
  locate(a, per_seq, blocks, 0, b, p);
  const Seq seq = load_seq(a, b);
  asm volatile("griddepcontrol.wait;" ::: "memory");  // the parts are written
  const int64_t start = p.before * per_seq + (int64_t)(head * a.row_blocks + rb) * seq.steps;
  const int64_t c0 = start / p.share, c1 = (start + seq.steps - 1) / p.share;
  if (c0 == c1) return;
  // (rows past a.rows are read, as there is room for them, and not written)
  auto part = [&](int64_t c) {
    return (2 * c + (c == c0 ? 1 : 0)) * a.rows_per_block + first;
  };
  float m[R];
#pragma unroll
  for (int y = 0; y < R; ++y) m[y] = -INFINITY;
  for (int64_t c = c0 + lane; c <= c1; c += 32) {
    const float* const ml = a.part_ml + part(c) * 2;
#pragma unroll
    for (int y = 0; y < R; ++y) m[y] = fmaxf(m[y], ml[2 * y]);
  }
#pragma unroll
  for (int y = 0; y < R; ++y)
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m[y] = fmaxf(m[y], __shfl_xor_sync(0xFFFFFFFFu, m[y], o));
  constexpr int N = D / 32;
  float l[R], o[R][N];
#pragma unroll
  for (int y = 0; y < R; ++y) {
    l[y] = 0.f;
#pragma unroll
    for (int i = 0; i < N; ++i) o[y][i] = 0.f;
  }
  for (int64_t base = c0; base <= c1; base += 32) {
    const int64_t c = base + lane;
    float f[R], lp[R];
#pragma unroll
    for (int y = 0; y < R; ++y) {
      f[y] = lp[y] = 0.f;
      if (c <= c1) {
        const float2 ml = *reinterpret_cast<const float2*>(a.part_ml + (part(c) + y) * 2);
        f[y] = m[y] == -INFINITY ? 1.f : ex2(ml.x - m[y]);
        lp[y] = ml.y * f[y];
      }
    }
    const int n = (int)min((int64_t)32, c1 - base + 1);
#pragma unroll(R > 2 ? 1 : 4)
    for (int i = 0; i < n; ++i) {
      const float* const x = a.part_o + part(base + i) * D + lane * N;
      float v[R][N];
#pragma unroll
      for (int y = 0; y < R; ++y)
#pragma unroll
        for (int j = 0; j < N; ++j) v[y][j] = x[y * D + j];
#pragma unroll
      for (int y = 0; y < R; ++y) {
        const float fi = __shfl_sync(0xFFFFFFFFu, f[y], i);
        l[y] += __shfl_sync(0xFFFFFFFFu, lp[y], i);
#pragma unroll
        for (int j = 0; j < N; ++j) o[y][j] += fi * v[y][j];
      }
    }
  }
#pragma unroll
  for (int y = 0; y < R; ++y) {
    const int row = row0 + y;
    if (row >= a.rows) return;
    const int nd = row / a.group;
    const int64_t at = ((int64_t)b * a.draft + nd) * a.hq + head * a.group + (row - nd * a.group);
    const bool none = nd >= seq.drafts || l[y] == 0.f;
    const float inv = none ? 0.f : kSumUp / l[y];
#pragma unroll
    for (int j = 0; j < N; j += 2) {
      uint32_t w = 0;
      if (!none) {
        if (a.q_f16) {
          w = half2_of(o[y][j] * inv, o[y][j + 1] * inv);
        } else {
          const __nv_bfloat162 h = __floats2bfloat162_rn(o[y][j] * inv, o[y][j + 1] * inv);
          w = *reinterpret_cast<const uint32_t*>(&h);
        }
      }
      *reinterpret_cast<uint32_t*>(static_cast<uint16_t*>(a.out) + at * D + lane * N + j) = w;
    }
    if (a.lse && lane == 0)
      a.lse[at] = none ? -INFINITY : (m[y] + log2f(l[y])) * 0.6931471805599453f;
  }
}

// ------------------------------------------------------------------ host
// The join's blocks start, and find their places, while the last parts are written.
template <int D, int R>
int launch_join_rows(const Args& a, int blocks, cudaStream_t st) {
  const int64_t warps = (int64_t)a.batch * a.c.heads * a.row_blocks * (a.rows_per_block / R);
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)((warps + kWarps - 1) / kWarps));
  cfg.blockDim = dim3(kThreads);
  cfg.stream = st;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  return check_cuda(cudaLaunchKernelEx(&cfg, k_join<D, R>, a, blocks));
}
template <int D>
int launch_join(const Args& a, int blocks, cudaStream_t st) {
  switch (join_rows(a.rows_per_block)) {
    case 1: return launch_join_rows<D, 1>(a, blocks, st);
    case 2: return launch_join_rows<D, 2>(a, blocks, st);
    case 4: return launch_join_rows<D, 4>(a, blocks, st);
    default: return launch_join_rows<D, 8>(a, blocks, st);
  }
}

template <int KIND, int FMT, int D, int NT>
int launch(const Args& a, int blocks, cudaStream_t st) {
  constexpr int bytes = ring_bytes(KIND, D, NT) + query_bytes(D, NT);
  static_assert(stages(KIND, D, NT) >= 2, "a ring needs two stages");
  if (const int rc = check_cuda(cudaFuncSetAttribute(
          k_attend<KIND, FMT, D, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes)))
    return rc;
  k_attend<KIND, FMT, D, NT><<<blocks, kThreads, bytes, st>>>(a);
  if (const int rc = check_launch()) return rc;
  return launch_join<D>(a, blocks, st);
}

template <int KIND, int FMT>
int by_shape(const Args& a, int nt, int blocks, cudaStream_t st) {
  switch (a.c.head_dim) {
    case 64: return nt == 1 ? launch<KIND, FMT, 64, 1>(a, blocks, st)
                  : nt == 2 ? launch<KIND, FMT, 64, 2>(a, blocks, st)
                            : launch<KIND, FMT, 64, 4>(a, blocks, st);
    case 128: return nt == 1 ? launch<KIND, FMT, 128, 1>(a, blocks, st)
                   : nt == 2 ? launch<KIND, FMT, 128, 2>(a, blocks, st)
                             : launch<KIND, FMT, 128, 4>(a, blocks, st);
    default: return nt == 1 ? launch<KIND, FMT, 256, 1>(a, blocks, st)
                            : launch<KIND, FMT, 256, 2>(a, blocks, st);
  }
}

int attend_block_e4m3(const Args& a, int nt, int blocks, cudaStream_t st);
int attend_block_e5m2(const Args& a, int nt, int blocks, cudaStream_t st);
int attend_mx_e4m3(const Args& a, int nt, int blocks, cudaStream_t st);
int attend_mx_e5m2(const Args& a, int nt, int blocks, cudaStream_t st);
int attend_nvfp4(const Args& a, int nt, int blocks, cudaStream_t st);
// The same with the tcgen05 kernel (kv_attention_tc.cuh): 256 rows to a block,
// steps of 128 tokens; head_dim 128, or 64 with FP8 codes.
int attend_tc_block_e4m3(const Args& a, int blocks, cudaStream_t st);
int attend_tc_block_e5m2(const Args& a, int blocks, cudaStream_t st);
int attend_tc_mx_e4m3(const Args& a, int blocks, cudaStream_t st);
int attend_tc_mx_e5m2(const Args& a, int blocks, cudaStream_t st);
int attend_tc_nvfp4(const Args& a, int blocks, cudaStream_t st);

}  // namespace kvatt
}  // namespace brc
