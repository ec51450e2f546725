// Norm of every query and key head and the position rotation, one pass, with
// the quantised cache write of a serving step fused in, and the gradients.
//
//   r = (mean(x^2) + eps)^-1/2,  z = x r w,  y = R(position) z
//   gz = R^T gy,  gw = sum gz x r,  gx = r (gz w - x r mean(gz w x r))
//
// A stream: HBM bounds it at long prompts, launch latency at single tokens. A
// head lies on LPR = 8, 16 or 32 lanes, eight elements to a lane in two groups
// of four that hold whole rotated pairs (halves: elements 4 p .. and rot / 2 +
// 4 p ..; interleaved: 8 p .. 8 p + 7), so a lane turns its pairs by itself with
// four cosines and sines, and a head's sums are shuffles. A warp takes several
// heads of one token, all queries or all keys: the token's angles and the
// weights are loaded once.
#include "kv_codec.cuh"
#include "launch.h"

namespace brc {
namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;

struct FwdArgs {
  brc_norm_rope a;
  void* q_out;
  // the write
  brc_kv_cache c;
  const void* v;
  int64_t v_token, v_head;
  const void* slots;
  int slots64;
};

__device__ __forceinline__ int64_t load_index(const void* p, int64_t i, int is64) {
  return is64 ? static_cast<const int64_t*>(p)[i] : (int64_t)static_cast<const int32_t*>(p)[i];
}

template <int LPR>
__device__ __forceinline__ float sum_row(float v) {
#pragma unroll
  for (int o = LPR / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, o);
  return v;
}

// Sum of squares of a row; where it passes float32's range the row is taken
// 2^-64 times (x r does not change when eps goes with 2^-128). Every lane of
// the warp calls it. Returns what the row's reciprocal root comes out scaled by.
template <int LPR>
__device__ __forceinline__ float square_sum(float* x, float& ss, float& eps) {
  auto sum = [&]() {
    float v = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) v = __fmaf_rn(x[i], x[i], v);
    return sum_row<LPR>(v);
  };
  ss = sum();
  float by = 1.f;
  if (__any_sync(0xFFFFFFFFu, isinf(ss))) {
    by = isinf(ss) ? 0x1p-64f : 1.f;
    eps *= by * by;
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] *= by;
    ss = sum();
  }
  return by;
}

// ------------------------------------------------------------------ pairs in a lane
// First elements of lane `part`'s two groups of four.
template <bool INTER>
__device__ __forceinline__ void groups(int rot, int part, int& e0, int& e1) {
  if (!INTER && part * 8 < rot) {
    e0 = 4 * part;
    e1 = (rot >> 1) + 4 * part;
  } else {  // whole pairs, or elements that are not rotated
    e0 = 8 * part;
    e1 = e0 + 4;
  }
}
// Four elements as they lie in memory (rows in flight wait in this form: half
// the registers of their float32 values).
template <int DT>
struct Raw {
  uint2 v;
};
template <>
struct Raw<BRC_DTYPE_F32> {
  uint4 v;
};
template <int DT>
__device__ __forceinline__ void load_raw(const void* p, int64_t e, Raw<DT>& r) {
  if constexpr (DT == BRC_DTYPE_F32) r.v = ldg16(static_cast<const char*>(p) + 4 * e);
  else r.v = __ldg(reinterpret_cast<const uint2*>(static_cast<const char*>(p) + 2 * e));
}
template <int DT>
__device__ __forceinline__ void expand(const Raw<DT>& r, float* f) {
  if constexpr (DT == BRC_DTYPE_F32) {
    unpack<DT>(r.v, f);
  } else if constexpr (DT == BRC_DTYPE_BF16) {
    f[0] = __uint_as_float(r.v.x << 16);
    f[1] = __uint_as_float(r.v.x & 0xFFFF0000u);
    f[2] = __uint_as_float(r.v.y << 16);
    f[3] = __uint_as_float(r.v.y & 0xFFFF0000u);
  } else {
    f16x2_to_f32(r.v.x, f[0], f[1]);
    f16x2_to_f32(r.v.y, f[2], f[3]);
  }
}
template <int DT>
__device__ __forceinline__ void load4(const void* p, int64_t e, float* f) {
  Raw<DT> r;
  load_raw<DT>(p, e, r);
  expand<DT>(r, f);
}
template <int DT>
__device__ __forceinline__ void store4(void* p, int64_t e, const float* f) {
  if constexpr (DT == BRC_DTYPE_F32) {
    stg16(static_cast<char*>(p) + 4 * e, make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]),
                                                    __float_as_uint(f[2]), __float_as_uint(f[3])));
  } else {
    uint32_t w[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      if constexpr (DT == BRC_DTYPE_BF16) {
        const __nv_bfloat162 b = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
        w[i] = *reinterpret_cast<const uint32_t*>(&b);
      } else {
        const __half2 h = __floats2half2_rn(f[2 * i], f[2 * i + 1]);
        w[i] = *reinterpret_cast<const uint32_t*>(&h);
      }
    }
    *reinterpret_cast<uint2*>(static_cast<char*>(p) + 2 * e) = make_uint2(w[0], w[1]);
  }
}
__device__ __forceinline__ void load_w4(const void* w, int dtype, int e, float* f) {
  if (dtype == BRC_DTYPE_F32) load4<BRC_DTYPE_F32>(w, e, f);
  else if (dtype == BRC_DTYPE_BF16) load4<BRC_DTYPE_BF16>(w, e, f);
  else load4<BRC_DTYPE_F16>(w, e, f);
}
// The four angles of lane `part`'s pairs; (1, 0) where nothing is rotated; a
// NaN cosine for a position outside the table (not a wrong angle).
__device__ __forceinline__ void load_angles(const brc_norm_rope& a, int64_t token, int part,
                                            float* c, float* s) {
  const int64_t pos = load_index(a.positions, token, a.index64);
  const bool in = pos >= 0 && pos < a.table_rows;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    c[i] = 1.f;
    s[i] = 0.f;
  }
  if (part * 8 < a.rot) {
    const int64_t at = (in ? pos : 0) * (a.rot >> 1) + 4 * part;
    load4<BRC_DTYPE_F32>(a.cos, at, c);
    load4<BRC_DTYPE_F32>(a.sin, at, s);
  }
  if (!in) {
#pragma unroll
    for (int i = 0; i < 4; ++i) c[i] = __uint_as_float(0x7FC00000u);
  }
}
// R z (BACK: R^T z) of the lane's eight elements.
template <bool INTER, bool BACK>
__device__ __forceinline__ void turn_pairs(const float* c, const float* s, float* z) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int x = INTER ? 2 * i : i, y = INTER ? 2 * i + 1 : i + 4;
    const float u = z[x], v = z[y], t = BACK ? -s[i] : s[i];
    z[x] = __fmaf_rn(u, c[i], -__fmul_rn(v, t));
    z[y] = __fmaf_rn(v, c[i], __fmul_rn(u, t));
  }
}

// ------------------------------------------------------------------ forward
// One row, in place; every lane of the warp calls it. Each operation is named,
// so that both kernels below round alike.
template <int LPR, bool INTER>
__device__ __forceinline__ void norm_turn(float* x, const float* w, const float* c, const float* s,
                                          float inv_d, float eps) {
  float ss;
  square_sum<LPR>(x, ss, eps);
  const float r = rsqrtf(__fmaf_rn(ss, inv_d, eps));
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = __fmul_rn(__fmul_rn(x[i], r), w[i]);
  turn_pairs<INTER, false>(c, s, x);
}

// heads in flight per lane (a float32 element takes twice the registers)
constexpr __host__ __device__ int heads_in_flight(int dt) { return dt == BRC_DTYPE_F32 ? 2 : 4; }
constexpr int kHeads = 4;

// blockIdx.y: a chunk of `iters` batches of heads, the queries' first.
template <int DT, int LPR, bool INTER>
__global__ void __launch_bounds__(kThreads, 4) k_fwd(brc_norm_rope a, void* q_out, void* k_out,
                                                  int q_chunks, int iters) {
  constexpr int G = 32 / LPR, kHeads = heads_in_flight(DT);
  const int lane = threadIdx.x & 31, part = lane % LPR;
  const int64_t token = (int64_t)blockIdx.x * kWarps + (threadIdx.x >> 5);
  if (token >= a.tokens) return;
  const bool is_q = (int)blockIdx.y < q_chunks;
  const int heads = is_q ? a.hq : a.hk;
  const int chunk = is_q ? blockIdx.y : blockIdx.y - q_chunks;
  const int64_t hs = is_q ? a.q_head : a.k_head;
  const void* const x = is_q ? a.q : a.k;
  void* const out = is_q ? q_out : k_out;
  const int64_t in0 = token * (is_q ? a.q_token : a.k_token);
  const int64_t out0 = token * heads * a.d;
  const bool on = part * 8 < a.d;
  int e0, e1;
  groups<INTER>(a.rot, part, e0, e1);
  const float inv_d = 1.f / (float)a.d;
  float w[8], c[4], s[4];
#pragma unroll
  for (int i = 0; i < 8; ++i) w[i] = 0.f;
  int h0 = chunk * iters * (kHeads * G) + lane / LPR;
  for (int it = 0; it < iters; ++it, h0 += kHeads * G) {
    Raw<DT> ra[kHeads], rb[kHeads];
#pragma unroll
    for (int u = 0; u < kHeads; ++u) {
      const int h = h0 + u * G;
      ra[u] = rb[u] = Raw<DT>{};
      if (on && h < heads) {
        load_raw<DT>(x, in0 + h * hs + e0, ra[u]);
        load_raw<DT>(x, in0 + h * hs + e1, rb[u]);
      }
    }
    if (it == 0) {
      if (on) {
        load_w4(is_q ? a.wq : a.wk, a.w_dtype, e0, w);
        load_w4(is_q ? a.wq : a.wk, a.w_dtype, e1, w + 4);
      }
      load_angles(a, token, part, c, s);
    }
#pragma unroll
    for (int u = 0; u < kHeads; ++u) {
      const int h = h0 + u * G;
      float f[8];
      expand<DT>(ra[u], f);
      expand<DT>(rb[u], f + 4);
      norm_turn<LPR, INTER>(f, w, c, s, inv_d, a.eps);
      if (on && h < heads) {
        store4<DT>(out, out0 + h * a.d + e0, f);
        store4<DT>(out, out0 + h * a.d + e1, f + 4);
      }
    }
  }
}

// Norm, rotation and the write into a cache. blockIdx.y: a batch of heads of
// queries, of keys or of values. The arithmetic is k_fwd's, operation by
// operation; a key's scales are over elements in a row, so its groups of four
// change lanes (as halves, after their rounding) before they are encoded.
template <int DT, int LPR, bool INTER, int KIND, int FMT>
__global__ void __launch_bounds__(kThreads) k_fwd_write(FwdArgs g, int q_chunks, int k_chunks) {
  constexpr int G = 32 / LPR;
  const brc_norm_rope& a = g.a;
  const int lane = threadIdx.x & 31, part = lane % LPR;
  const int64_t token = (int64_t)blockIdx.x * kWarps + (threadIdx.x >> 5);
  if (token >= a.tokens) return;
  const bool is_q = (int)blockIdx.y < q_chunks, is_v = (int)blockIdx.y >= q_chunks + k_chunks;
  const int heads = is_q ? a.hq : a.hk;
  const int chunk = is_q ? blockIdx.y : blockIdx.y - q_chunks - (is_v ? k_chunks : 0);
  const int h0 = chunk * (kHeads * G) + lane / LPR;
  int64_t slot = load_index(g.slots, token, g.slots64);
  if (slot >= g.c.num_pages * g.c.page_size) slot = -1;
  float f[kHeads][8];
  if (is_v) {
#pragma unroll
    for (int u = 0; u < kHeads; ++u) {
      const int h = h0 + u * G;
#pragma unroll
      for (int i = 0; i < 8; ++i) f[u][i] = 0.f;
      if (h < heads) kv::load8<DT>(g.v, token * g.v_token + h * g.v_head + part * 8, f[u]);
    }
  } else {
    const int64_t hs = is_q ? a.q_head : a.k_head;
    const void* const x = is_q ? a.q : a.k;
    const int64_t in0 = token * (is_q ? a.q_token : a.k_token);
    int e0, e1;
    groups<INTER>(a.rot, part, e0, e1);
#pragma unroll
    for (int u = 0; u < kHeads; ++u) {
      const int h = h0 + u * G;
#pragma unroll
      for (int i = 0; i < 8; ++i) f[u][i] = 0.f;
      if (h < heads) {
        load4<DT>(x, in0 + h * hs + e0, f[u]);
        load4<DT>(x, in0 + h * hs + e1, f[u] + 4);
      }
    }
    float w[8], c[4], s[4];
    load_w4(is_q ? a.wq : a.wk, a.w_dtype, e0, w);
    load_w4(is_q ? a.wq : a.wk, a.w_dtype, e1, w + 4);
    load_angles(a, token, part, c, s);
    const float inv_d = 1.f / (float)a.d;
#pragma unroll
    for (int u = 0; u < kHeads; ++u) {
      norm_turn<LPR, INTER>(f[u], w, c, s, inv_d, a.eps);
      const int h = h0 + u * G;
      if (is_q) {
        if (h < heads) {
          store4<DT>(g.q_out, (token * heads + h) * a.d + e0, f[u]);
          store4<DT>(g.q_out, (token * heads + h) * a.d + e1, f[u] + 4);
        }
      } else {
        // the key as the separate call would have left it, in its own dtype
        uint4 y = kv::pack8<DT>(f[u]);
        if constexpr (!INTER) {
          uint32_t z[4];
#pragma unroll
          for (int i = 0; i < 2; ++i) {  // elements 8 part + 4 i ..
            const int four = 2 * part + i, half = a.rot >> 3;
            const bool turned = four < 2 * half;
            const int from = turned ? (four < half ? four : four - half) : part;
            const bool second = turned ? four >= half : i;
            const uint32_t a0 = __shfl_sync(0xFFFFFFFFu, y.x, from, LPR);
            const uint32_t a1 = __shfl_sync(0xFFFFFFFFu, y.y, from, LPR);
            const uint32_t b0 = __shfl_sync(0xFFFFFFFFu, y.z, from, LPR);
            const uint32_t b1 = __shfl_sync(0xFFFFFFFFu, y.w, from, LPR);
            z[2 * i] = second ? b0 : a0;
            z[2 * i + 1] = second ? b1 : a1;
          }
          y = make_uint4(z[0], z[1], z[2], z[3]);
        }
        unpack<DT>(y, f[u]);
      }
    }
    if (is_q) return;
  }
#pragma unroll
  for (int u = 0; u < kHeads; ++u) {
    const int h = h0 + u * G;
    const bool keep = h < heads && slot >= 0;
    kv::encode_row<KIND, FMT, LPR>(f[u], part, keep, keep ? kv::row_of(g.c, slot, h) : 0,
                                   is_v ? g.c.v_data : g.c.k_data,
                                   is_v ? g.c.v_scale : g.c.k_scale);
  }
}

// ------------------------------------------------------------------ backward
struct BwdArgs {
  brc_norm_rope a;
  const void* g[2];  // gradients of the queries' and keys' outputs
  int64_t g_token[2], g_head[2];
  void* dx[2];
  float* part;      // (blocks, d) sums of the weight gradients
  int q_blocks;     // blocks that take queries; the rest take keys
  int parts_shift;  // a token's heads go to 2^parts_shift warps
};

constexpr int kBwdHeads = 2;
constexpr int kBwdPerSm = 3;

// Persistent: a lane sums the weight gradients of its eight elements over all
// the heads that it takes, so that one row per block is written.
template <int DT, int LPR, bool INTER>
__global__ void __launch_bounds__(kThreads, kBwdPerSm) k_bwd(BwdArgs g) {
  constexpr int G = 32 / LPR;
  const brc_norm_rope& a = g.a;
  const int lane = threadIdx.x & 31, part = lane % LPR;
  const bool is_q = (int)blockIdx.x < g.q_blocks;
  const int side = is_q ? 0 : 1, heads = is_q ? a.hq : a.hk;
  const int block = is_q ? blockIdx.x : blockIdx.x - g.q_blocks;
  const int blocks = is_q ? g.q_blocks : gridDim.x - g.q_blocks;
  const int64_t xt = is_q ? a.q_token : a.k_token, xh = is_q ? a.q_head : a.k_head;
  const int64_t gt = is_q ? g.g_token[0] : g.g_token[1], gh = is_q ? g.g_head[0] : g.g_head[1];
  const void* const px = is_q ? a.q : a.k;
  const void* const pg = is_q ? g.g[0] : g.g[1];
  void* const dx = is_q ? g.dx[0] : g.dx[1];
  const bool on = part * 8 < a.d;
  int e0, e1;
  groups<INTER>(a.rot, part, e0, e1);
  const float inv_d = 1.f / (float)a.d;
  float w[8], dw[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) w[i] = dw[i] = 0.f;
  if (on) {
    load_w4(is_q ? a.wq : a.wk, a.w_dtype, e0, w);
    load_w4(is_q ? a.wq : a.wk, a.w_dtype, e1, w + 4);
  }
  const int n_parts = 1 << g.parts_shift;
  const int per = (heads + n_parts - 1) >> g.parts_shift;  // heads of one warp
  const int64_t units = a.tokens << g.parts_shift;
  for (int64_t unit = (int64_t)block * kWarps + (threadIdx.x >> 5); unit < units;
       unit += (int64_t)blocks * kWarps) {
    const int64_t token = unit >> g.parts_shift;
    const int first = (int)(unit & (n_parts - 1)) * per, last = min(first + per, heads);
    float c[4], s[4];
    load_angles(a, token, part, c, s);
    for (int h0 = first; h0 < last; h0 += kBwdHeads * G) {
      Raw<DT> xa[kBwdHeads], xb[kBwdHeads], ga[kBwdHeads], gb[kBwdHeads];
#pragma unroll
      for (int u = 0; u < kBwdHeads; ++u) {
        const int h = h0 + u * G + lane / LPR;
        xa[u] = xb[u] = ga[u] = gb[u] = Raw<DT>{};
        if (on && h < last) {
          load_raw<DT>(px, token * xt + h * xh + e0, xa[u]);
          load_raw<DT>(px, token * xt + h * xh + e1, xb[u]);
          load_raw<DT>(pg, token * gt + h * gh + e0, ga[u]);
          load_raw<DT>(pg, token * gt + h * gh + e1, gb[u]);
        }
      }
#pragma unroll
      for (int u = 0; u < kBwdHeads; ++u) {
        const int h = h0 + u * G + lane / LPR;
        float x[8], gy[8];
        expand<DT>(xa[u], x);
        expand<DT>(xb[u], x + 4);
        expand<DT>(ga[u], gy);
        expand<DT>(gb[u], gy + 4);
        turn_pairs<INTER, true>(c, s, gy);
        float ss, hx = 0.f, eps = a.eps;
        const float by = square_sum<LPR>(x, ss, eps);
#pragma unroll
        for (int i = 0; i < 8; ++i) hx += gy[i] * w[i] * x[i];
        hx = sum_row<LPR>(hx);
        const float r = rsqrtf(ss * inv_d + eps);
        const float m = hx * r * inv_d;  // mean(gz w x r)
        if (on && h < last) {
          float o[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const float n = x[i] * r;
            dw[i] += gy[i] * n;
            o[i] = r * (gy[i] * w[i] - n * m) * by;
          }
          store4<DT>(dx, (token * heads + h) * a.d + e0, o);
          store4<DT>(dx, (token * heads + h) * a.d + e1, o + 4);
        }
      }
    }
  }
  // lanes of the same elements: G per warp, kWarps warps
  __shared__ float sm[kWarps * G][LPR * 8];
  const int mine = (threadIdx.x >> 5) * G + lane / LPR;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    sm[mine][e0 + i] = dw[i];
    sm[mine][e1 + i] = dw[4 + i];
  }
  __syncthreads();
  for (int i = threadIdx.x; i < a.d; i += kThreads) {
    float t = 0.f;
#pragma unroll
    for (int j = 0; j < kWarps * G; ++j) t += sm[j][i];
    g.part[(int64_t)blockIdx.x * a.d + i] = t;
  }
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}

// Sums of the blocks' rows: 32 columns to a block, 16 row groups, in order.
__global__ void __launch_bounds__(512) k_bwd_weights(const float* part, int q_blocks, int blocks,
                                                     int d, int w_dtype, void* dwq, void* dwk) {
  __shared__ float sm[16][33];
  const int col = blockIdx.x * 32 + (threadIdx.x & 31), grp = threadIdx.x >> 5;
  void* const out = blockIdx.y ? dwk : dwq;
  const int first = blockIdx.y ? q_blocks : 0, last = blockIdx.y ? blocks : q_blocks;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  float s = 0.f;
  if (col < d)
    for (int b = first + grp; b < last; b += 16) s += part[(int64_t)b * d + col];
  sm[grp][threadIdx.x & 31] = s;
  __syncthreads();
  if (grp == 0 && col < d && out) {
#pragma unroll
    for (int j = 1; j < 16; ++j) s += sm[j][threadIdx.x];
    if (w_dtype == BRC_DTYPE_F32) static_cast<float*>(out)[col] = s;
    else if (w_dtype == BRC_DTYPE_BF16)
      static_cast<__nv_bfloat16*>(out)[col] = __float2bfloat16_rn(s);
    else static_cast<__half*>(out)[col] = __float2half_rn(s);
  }
}

// ------------------------------------------------------------------ host
bool bad_stride(int64_t s, int dtype) { return s % (dtype == BRC_DTYPE_F32 ? 4 : 8) != 0; }

int check(const brc_norm_rope* a) {
  if (!a) return BRC_ERR_NULL;
  if (a->dtype < BRC_DTYPE_F32 || a->dtype > BRC_DTYPE_F16 || a->w_dtype < BRC_DTYPE_F32 ||
      a->w_dtype > BRC_DTYPE_F16)
    return BRC_ERR_DTYPE;
  if (a->tokens < 0 || a->hq < 0 || a->hk < 0 || a->table_rows < 0) return BRC_ERR_SHAPE;
  if (a->d < 16 || a->d > 256 || a->d % 16 || a->rot < 16 || a->rot > a->d || a->rot % 16)
    return BRC_ERR_SHAPE;
  if (a->tokens == 0 || a->hq + a->hk == 0) return BRC_OK;
  if ((a->hq && (!a->q || !a->wq)) || (a->hk && (!a->k || !a->wk)) || !a->positions || !a->cos ||
      !a->sin)
    return BRC_ERR_NULL;
  if (a->table_rows == 0) return BRC_ERR_SHAPE;
  if (((uintptr_t)a->q | (uintptr_t)a->k | (uintptr_t)a->wq | (uintptr_t)a->wk |
       (uintptr_t)a->cos | (uintptr_t)a->sin) & 15)
    return BRC_ERR_ALIGN;
  if (bad_stride(a->q_token, a->dtype) || bad_stride(a->q_head, a->dtype) ||
      bad_stride(a->k_token, a->dtype) || bad_stride(a->k_head, a->dtype))
    return BRC_ERR_ALIGN;
  return BRC_OK;
}

int lanes_per_row(int d) { return d <= 64 ? 8 : d <= 128 ? 16 : 32; }

template <int DT, int LPR>
int launch_fwd(const brc_norm_rope& a, void* q_out, void* k_out, cudaStream_t st) {
  const int64_t bx = (a.tokens + kWarps - 1) / kWarps;
  // one batch of heads to a warp while that leaves SMs free, then two (the
  // token's angles and the weights are loaded half as often)
  const int per1 = heads_in_flight(DT) * (32 / LPR);
  const int64_t blocks1 = bx * ((a.hq + per1 - 1) / per1 + (a.hk + per1 - 1) / per1);
  const int iters = blocks1 > 8 * sm_count() ? 2 : 1, per = per1 * iters;
  const int q_chunks = (a.hq + per - 1) / per, chunks = q_chunks + (a.hk + per - 1) / per;
  if (bx > 0x7FFFFFFF || chunks > 65535) return BRC_ERR_RANGE;
  const dim3 grid((unsigned)bx, (unsigned)chunks);
  if (a.interleaved) k_fwd<DT, LPR, true><<<grid, kThreads, 0, st>>>(a, q_out, k_out, q_chunks, iters);
  else k_fwd<DT, LPR, false><<<grid, kThreads, 0, st>>>(a, q_out, k_out, q_chunks, iters);
  return check_launch();
}
template <int DT>
int launch_fwd_any(const brc_norm_rope& a, void* q_out, void* k_out, cudaStream_t st) {
  const int lpr = lanes_per_row(a.d);
  return lpr == 8    ? launch_fwd<DT, 8>(a, q_out, k_out, st)
         : lpr == 16 ? launch_fwd<DT, 16>(a, q_out, k_out, st)
                     : launch_fwd<DT, 32>(a, q_out, k_out, st);
}

template <int DT, int LPR, int KIND, int FMT>
int launch_fwd_write(const FwdArgs& g, cudaStream_t st) {
  const int per = kHeads * (32 / LPR);
  const int64_t bx = (g.a.tokens + kWarps - 1) / kWarps;
  const int q_chunks = (g.a.hq + per - 1) / per, k_chunks = (g.a.hk + per - 1) / per;
  if (bx > 0x7FFFFFFF || q_chunks + 2 * k_chunks > 65535) return BRC_ERR_RANGE;
  const dim3 grid((unsigned)bx, (unsigned)(q_chunks + 2 * k_chunks));
  if (g.a.interleaved)
    k_fwd_write<DT, LPR, true, KIND, FMT><<<grid, kThreads, 0, st>>>(g, q_chunks, k_chunks);
  else k_fwd_write<DT, LPR, false, KIND, FMT><<<grid, kThreads, 0, st>>>(g, q_chunks, k_chunks);
  return check_launch();
}
template <int DT, int KIND, int FMT>
int launch_write_dim(const FwdArgs& g, cudaStream_t st) {
  return g.a.d == 64    ? launch_fwd_write<DT, 8, KIND, FMT>(g, st)
         : g.a.d == 128 ? launch_fwd_write<DT, 16, KIND, FMT>(g, st)
                        : launch_fwd_write<DT, 32, KIND, FMT>(g, st);
}

template <int DT>
int launch_write(const FwdArgs& g, cudaStream_t st) {
  const bool e4 = g.c.fmt == BRC_FP8_E4M3;
  if (g.c.kind == BRC_STE_BLOCK_FP8)
    return e4 ? launch_write_dim<DT, BRC_STE_BLOCK_FP8, BRC_FP8_E4M3>(g, st)
              : launch_write_dim<DT, BRC_STE_BLOCK_FP8, BRC_FP8_E5M2>(g, st);
  if (g.c.kind == BRC_STE_MXFP8)
    return e4 ? launch_write_dim<DT, BRC_STE_MXFP8, BRC_FP8_E4M3>(g, st)
              : launch_write_dim<DT, BRC_STE_MXFP8, BRC_FP8_E5M2>(g, st);
  return launch_write_dim<DT, BRC_STE_NVFP4, BRC_FP8_E4M3>(g, st);
}

template <int DT, int LPR>
void launch_bwd(const BwdArgs& g, int blocks, cudaStream_t st) {
  if (g.a.interleaved) k_bwd<DT, LPR, true><<<blocks, kThreads, 0, st>>>(g);
  else k_bwd<DT, LPR, false><<<blocks, kThreads, 0, st>>>(g);
}
template <int DT>
void launch_bwd_any(const BwdArgs& g, int blocks, cudaStream_t st) {
  const int lpr = lanes_per_row(g.a.d);
  if (lpr == 8) launch_bwd<DT, 8>(g, blocks, st);
  else if (lpr == 16) launch_bwd<DT, 16>(g, blocks, st);
  else launch_bwd<DT, 32>(g, blocks, st);
}

}  // namespace
}  // namespace brc

using namespace brc;

extern "C" {

int brc_qk_norm_rope(const brc_norm_rope* a, void* q_out, void* k_out, void* stream) {
  if (const int rc = check(a)) return rc;
  if (a->tokens == 0 || a->hq + a->hk == 0) return BRC_OK;
  if ((a->hq && !q_out) || (a->hk && !k_out)) return BRC_ERR_NULL;
  if (((uintptr_t)q_out | (uintptr_t)k_out) & 15) return BRC_ERR_ALIGN;
  const cudaStream_t st = (cudaStream_t)stream;
  if (a->dtype == BRC_DTYPE_F32) return launch_fwd_any<BRC_DTYPE_F32>(*a, q_out, k_out, st);
  if (a->dtype == BRC_DTYPE_BF16) return launch_fwd_any<BRC_DTYPE_BF16>(*a, q_out, k_out, st);
  return launch_fwd_any<BRC_DTYPE_F16>(*a, q_out, k_out, st);
}

int brc_qk_norm_rope_write(const brc_norm_rope* a, const void* v, int64_t v_token, int64_t v_head,
                           void* q_out, const brc_kv_cache* c, const void* slots, int slots64,
                           void* stream) {
  if (const int rc = check(a)) return rc;
  if (const int rc = kv::check_cache(c)) return rc;
  if (a->dtype == BRC_DTYPE_F32) return BRC_ERR_DTYPE;
  if (a->hk != c->heads || a->d != c->head_dim) return BRC_ERR_SHAPE;
  if (a->tokens == 0) return BRC_OK;
  if (!v || !slots || (a->hq && !q_out)) return BRC_ERR_NULL;
  if (((uintptr_t)v | (uintptr_t)q_out) & 15) return BRC_ERR_ALIGN;
  if (bad_stride(v_token, a->dtype) || bad_stride(v_head, a->dtype)) return BRC_ERR_ALIGN;
  FwdArgs g{};
  g.a = *a;
  g.q_out = q_out;
  g.c = *c;
  g.v = v;
  g.v_token = v_token;
  g.v_head = v_head;
  g.slots = slots;
  g.slots64 = slots64;
  const cudaStream_t st = (cudaStream_t)stream;
  return a->dtype == BRC_DTYPE_BF16 ? launch_write<BRC_DTYPE_BF16>(g, st)
                                    : launch_write<BRC_DTYPE_F16>(g, st);
}

int64_t brc_qk_norm_rope_bwd_workspace(int d) {
  return d < 16 || d > 256 ? 0 : (int64_t)sm_count() * kBwdPerSm * d * 4;
}

int brc_qk_norm_rope_bwd(const brc_norm_rope* a, const void* gq, const void* gk, int64_t gq_token,
                         int64_t gq_head, int64_t gk_token, int64_t gk_head, void* dq, void* dk,
                         void* dwq, void* dwk, void* workspace, int64_t workspace_bytes,
                         void* stream) {
  if (const int rc = check(a)) return rc;
  if ((a->hq && !dwq) || (a->hk && !dwk) || !workspace) return BRC_ERR_NULL;
  if (workspace_bytes < brc_qk_norm_rope_bwd_workspace(a->d)) return BRC_ERR_SHAPE;
  const cudaStream_t st = (cudaStream_t)stream;
  int blocks = 0, q_blocks = 0;
  if (a->tokens > 0 && a->hq + a->hk > 0) {
    if ((a->hq && (!gq || !dq)) || (a->hk && (!gk || !dk))) return BRC_ERR_NULL;
    if (((uintptr_t)gq | (uintptr_t)gk | (uintptr_t)dq | (uintptr_t)dk | (uintptr_t)workspace) & 15)
      return BRC_ERR_ALIGN;
    if (bad_stride(gq_token, a->dtype) || bad_stride(gq_head, a->dtype) ||
        bad_stride(gk_token, a->dtype) || bad_stride(gk_head, a->dtype))
      return BRC_ERR_ALIGN;
    BwdArgs g{};
    g.a = *a;
    g.g[0] = gq;
    g.g[1] = gk;
    g.g_token[0] = gq_token;
    g.g_token[1] = gk_token;
    g.g_head[0] = gq_head;
    g.g_head[1] = gk_head;
    g.dx[0] = dq;
    g.dx[1] = dk;
    g.part = static_cast<float*>(workspace);
    // enough warps for every SM, none with less than a batch of heads
    const int most = sm_count() * kBwdPerSm, per = kBwdHeads * (32 / lanes_per_row(a->d));
    const int heads = a->hq > a->hk ? a->hq : a->hk;
    while (g.parts_shift < 4 && (a->tokens << g.parts_shift) < 8 * (int64_t)most * kWarps &&
           (heads >> g.parts_shift) > per)
      ++g.parts_shift;
    const int64_t want = ((a->tokens << g.parts_shift) + kWarps - 1) / kWarps;  // of one side
    // the SMs are shared out by the number of heads
    int q_share = a->hk ? (int)((int64_t)most * a->hq / (a->hq + a->hk)) : most;
    if (a->hq && q_share < 1) q_share = 1;
    if (a->hk && q_share > most - 1) q_share = most - 1;
    q_blocks = a->hq ? (int)(want < q_share ? want : q_share) : 0;
    const int k_share = most - q_share;
    blocks = q_blocks + (a->hk ? (int)(want < k_share ? want : k_share) : 0);
    g.q_blocks = q_blocks;
    if (a->dtype == BRC_DTYPE_F32) launch_bwd_any<BRC_DTYPE_F32>(g, blocks, st);
    else if (a->dtype == BRC_DTYPE_BF16) launch_bwd_any<BRC_DTYPE_BF16>(g, blocks, st);
    else launch_bwd_any<BRC_DTYPE_F16>(g, blocks, st);
    if (const int rc = check_launch()) return rc;
  }
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((a->d + 31) / 32, 2);
  cfg.blockDim = dim3(512);
  cfg.stream = st;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  return check_cuda(cudaLaunchKernelEx(&cfg, k_bwd_weights, static_cast<const float*>(workspace),
                                       q_blocks, blocks, a->d, a->w_dtype, dwq, dwk));
}

}  // extern "C"
