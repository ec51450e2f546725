// Norm of every query and key head and the position rotation, one pass, with
// the quantised cache write of a serving step fused in, and the gradients.
//
//   r = (mean(x^2) + eps)^-1/2,  z = x r w,  y = R(position) z
//   gz = R^T gy,  gw = sum gz x r,  gx = r (gz w - x r mean(gz w x r))
//
// A stream: HBM bounds it at long prompts, launch latency at single tokens. A
// head lies on LPR = 8, 16 or 32 lanes, eight elements to a lane, so its loads
// and stores are contiguous, its sums are shuffles, and a rotated pair is two
// lanes' (halves) or one lane's (interleaved) values. A warp takes several
// heads of ONE token, so the token's cosines and sines are loaded once.
#include "kv_codec.cuh"
#include "launch.h"

namespace brc {
namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;

struct FwdArgs {
  brc_norm_rope a;
  void* q_out;
  void* k_out;
  // fused write
  brc_kv_cache c;
  const void* v;
  int64_t v_token, v_head;
  const void* slots;
  int slots64;
};

__device__ __forceinline__ int64_t load_index(const void* p, int64_t i, int is64) {
  return is64 ? static_cast<const int64_t*>(p)[i] : (int64_t)static_cast<const int32_t*>(p)[i];
}

__device__ __forceinline__ void load_w(const void* w, int dtype, int e, float* f) {
  if (dtype == BRC_DTYPE_F32) kv::load8<BRC_DTYPE_F32>(w, e, f);
  else if (dtype == BRC_DTYPE_BF16) kv::load8<BRC_DTYPE_BF16>(w, e, f);
  else kv::load8<BRC_DTYPE_F16>(w, e, f);
}

// The rotation's factors for one lane's eight elements: y_i = z_i c_i + o_i s_i
// with o the pair's other element, s signed. Elements past `rot` get c = 1, s = 0.
struct Turn {
  float c[8], s[8];
  int other;  // lane of the head that holds the other elements (halves)
};

__device__ __forceinline__ void load_turn(const brc_norm_rope& a, int64_t token, int part,
                                          Turn& t) {
  const int64_t pos = load_index(a.positions, token, a.index64);
  const bool in = pos >= 0 && pos < a.table_rows;
  const int half = a.rot >> 1, e = part * 8;
  t.other = part;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    t.c[i] = 1.f;
    t.s[i] = 0.f;
  }
  if (e < a.rot) {
    const int64_t row = (in ? pos : 0) * half;
    if (a.interleaved) {
      const float4 c = *reinterpret_cast<const float4*>(a.cos + row + e / 2);
      const float4 s = *reinterpret_cast<const float4*>(a.sin + row + e / 2);
      const float cc[4] = {c.x, c.y, c.z, c.w}, ss[4] = {s.x, s.y, s.z, s.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        t.c[2 * i] = t.c[2 * i + 1] = cc[i];
        t.s[2 * i] = -ss[i];
        t.s[2 * i + 1] = ss[i];
      }
    } else {
      const bool low = e < half;
      const int at = low ? e : e - half;
      t.other = low ? part + half / 8 : part - half / 8;
      kv::load8<BRC_DTYPE_F32>(a.cos, row + at, t.c);
      kv::load8<BRC_DTYPE_F32>(a.sin, row + at, t.s);
      if (low) {
#pragma unroll
        for (int i = 0; i < 8; ++i) t.s[i] = -t.s[i];
      }
    }
  }
  if (!in) {  // outside the table: NaN, not a wrong angle
#pragma unroll
    for (int i = 0; i < 8; ++i) t.c[i] = __uint_as_float(0x7FC00000u);
  }
}

// R z (or, back, R^T z) of one lane's elements; every lane of the warp calls it.
template <int LPR>
__device__ __forceinline__ void turn8(const Turn& t, bool interleaved, bool back, float* z) {
  float o[8];
  if (interleaved) {
#pragma unroll
    for (int i = 0; i < 8; ++i) o[i] = z[i ^ 1];
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) o[i] = __shfl_sync(0xFFFFFFFFu, z[i], t.other, LPR);
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float b = o[i] * t.s[i];  // R^T: the sines change sign
    z[i] = z[i] * t.c[i] + (back ? -b : b);
  }
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
    for (int i = 0; i < 8; ++i) v += x[i] * x[i];
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

constexpr int kHeads = 4;  // heads in flight per lane

// KIND < 0: norm and rotation only; else the write into a cache of that kind.
template <int DT, int LPR, int KIND, int FMT>
__global__ void __launch_bounds__(kThreads) k_fwd(FwdArgs g) {
  constexpr int G = 32 / LPR;
  constexpr bool kWrite = KIND >= 0;
  const brc_norm_rope& a = g.a;
  const int lane = threadIdx.x & 31, part = lane % LPR, e = part * 8;
  const int64_t token = (int64_t)blockIdx.x * kWarps + (threadIdx.x >> 5);
  if (token >= a.tokens) return;
  const int heads = a.hq + (kWrite ? 2 : 1) * a.hk;
  const int h0 = blockIdx.y * (kHeads * G) + lane / LPR;
  float f[kHeads][8];
#pragma unroll
  for (int u = 0; u < kHeads; ++u) {
    const int h = h0 + u * G;
#pragma unroll
    for (int i = 0; i < 8; ++i) f[u][i] = 0.f;
    if (h < heads && e < a.d) {
      if (h < a.hq) kv::load8<DT>(a.q, token * a.q_token + h * a.q_head + e, f[u]);
      else if (h < a.hq + a.hk)
        kv::load8<DT>(a.k, token * a.k_token + (h - a.hq) * a.k_head + e, f[u]);
      else if constexpr (kWrite)
        kv::load8<DT>(g.v, token * g.v_token + (h - a.hq - a.hk) * g.v_head + e, f[u]);
    }
  }
  Turn t;
  load_turn(a, token, part, t);
  int64_t slot = -1;
  if constexpr (kWrite) {
    slot = load_index(g.slots, token, g.slots64);
    if (slot >= g.c.num_pages * g.c.page_size) slot = -1;
  }
#pragma unroll
  for (int u = 0; u < kHeads; ++u) {
    const int h = h0 + u * G;
    const bool on = h < heads && e < a.d, is_v = h >= a.hq + a.hk;
    float ss, eps = a.eps, x[8], z[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      x[i] = is_v ? 0.f : f[u][i];
      z[i] = 0.f;
    }
    square_sum<LPR>(x, ss, eps);
    const float r = rsqrtf(ss / (float)a.d + eps);
    if (on && !is_v) {
      load_w(h < a.hq ? a.wq : a.wk, a.w_dtype, e, z);
#pragma unroll
      for (int i = 0; i < 8; ++i) z[i] = x[i] * r * z[i];
    }
    turn8<LPR>(t, a.interleaved, false, z);
    if (on && h < a.hq) kv::store8<DT>(g.q_out, (token * a.hq + h) * a.d + e, z);
    if constexpr (!kWrite) {
      if (on && h >= a.hq) kv::store8<DT>(g.k_out, (token * a.hk + h - a.hq) * a.d + e, z);
    } else {
      // the key as the separate call would have left it, in its own dtype
      if (!is_v) unpack<DT>(kv::pack8<DT>(z), f[u]);
      const bool keep = on && h >= a.hq && slot >= 0;
      const int head = is_v ? h - a.hq - a.hk : h - a.hq;
      kv::encode_row<KIND, FMT, LPR>(f[u], part, keep, keep ? kv::row_of(g.c, slot, head) : 0,
                                     is_v ? g.c.v_data : g.c.k_data,
                                     is_v ? g.c.v_scale : g.c.k_scale);
    }
  }
}

// ------------------------------------------------------------------ backward
struct BwdArgs {
  brc_norm_rope a;
  const void* gq;
  const void* gk;
  int64_t gq_token, gq_head, gk_token, gk_head;
  void* dq;
  void* dk;
  float* part;  // (blocks, 2, d) sums of the weight gradients
  int64_t units;  // tokens * chunks
  int chunks;
};

constexpr int kBwdHeads = 2;
constexpr int kBwdBlocksMax = 148 * 4;

// Persistent: a lane sums the weight gradients of its eight elements over all
// the heads that it takes, so that only one row per block is written.
template <int DT, int LPR>
__global__ void __launch_bounds__(kThreads) k_bwd(BwdArgs g) {
  constexpr int G = 32 / LPR;
  const brc_norm_rope& a = g.a;
  const int lane = threadIdx.x & 31, part = lane % LPR, e = part * 8;
  const int heads = a.hq + a.hk;
  float dwq[8], dwk[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) dwq[i] = dwk[i] = 0.f;
  float wq[8], wk[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) wq[i] = wk[i] = 0.f;
  if (e < a.d) {
    if (a.hq) load_w(a.wq, a.w_dtype, e, wq);
    if (a.hk) load_w(a.wk, a.w_dtype, e, wk);
  }
  const int64_t step = (int64_t)gridDim.x * kWarps;
  for (int64_t unit = (int64_t)blockIdx.x * kWarps + (threadIdx.x >> 5); unit < g.units;
       unit += step) {
    const int64_t token = unit / g.chunks;
    const int h0 = (int)(unit - token * g.chunks) * (kBwdHeads * G) + lane / LPR;
    float x[kBwdHeads][8], gy[kBwdHeads][8];
#pragma unroll
    for (int u = 0; u < kBwdHeads; ++u) {
      const int h = h0 + u * G;
#pragma unroll
      for (int i = 0; i < 8; ++i) x[u][i] = gy[u][i] = 0.f;
      if (h < heads && e < a.d) {
        if (h < a.hq) {
          kv::load8<DT>(a.q, token * a.q_token + h * a.q_head + e, x[u]);
          kv::load8<DT>(g.gq, token * g.gq_token + h * g.gq_head + e, gy[u]);
        } else {
          kv::load8<DT>(a.k, token * a.k_token + (h - a.hq) * a.k_head + e, x[u]);
          kv::load8<DT>(g.gk, token * g.gk_token + (h - a.hq) * g.gk_head + e, gy[u]);
        }
      }
    }
    Turn t;
    load_turn(a, token, part, t);
#pragma unroll
    for (int u = 0; u < kBwdHeads; ++u) {
      const int h = h0 + u * G;
      const bool on = h < heads && e < a.d, is_q = h < a.hq;
      turn8<LPR>(t, a.interleaved, true, gy[u]);
      float ss, hx = 0.f, eps = a.eps;
      const float by = square_sum<LPR>(x[u], ss, eps);
#pragma unroll
      for (int i = 0; i < 8; ++i) hx += gy[u][i] * (is_q ? wq[i] : wk[i]) * x[u][i];
      hx = sum_row<LPR>(hx);
      const float r = rsqrtf(ss / (float)a.d + eps);
      const float m = hx * r / (float)a.d;  // mean(gz w x r)
      float o[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float n = x[u][i] * r;
        dwq[i] += on && is_q ? gy[u][i] * n : 0.f;
        dwk[i] += on && !is_q ? gy[u][i] * n : 0.f;
        o[i] = r * (gy[u][i] * (is_q ? wq[i] : wk[i]) - n * m) * by;
      }
      if (on) {
        if (is_q) kv::store8<DT>(g.dq, (token * a.hq + h) * a.d + e, o);
        else kv::store8<DT>(g.dk, (token * a.hk + h - a.hq) * a.d + e, o);
      }
    }
  }
  // lanes of the same elements: G per warp, kWarps warps
  __shared__ float sm[kWarps * G][2][LPR * 8];
  const int mine = (threadIdx.x >> 5) * G + lane / LPR;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    sm[mine][0][e + i] = dwq[i];
    sm[mine][1][e + i] = dwk[i];
  }
  __syncthreads();
  for (int i = threadIdx.x; i < 2 * a.d; i += kThreads) {
    const int side = i >= a.d, at = i - side * a.d;
    float s = 0.f;
#pragma unroll
    for (int j = 0; j < kWarps * G; ++j) s += sm[j][side][at];
    g.part[(int64_t)blockIdx.x * 2 * a.d + i] = s;
  }
}

// Sums of the blocks' rows: 32 columns to a block, 16 row groups.
__global__ void __launch_bounds__(512) k_bwd_weights(const float* part, int blocks, int d,
                                                     int w_dtype, void* dwq, void* dwk) {
  __shared__ float sm[16][33];
  const int col = blockIdx.x * 32 + (threadIdx.x & 31), grp = threadIdx.x >> 5;
  float s = 0.f;
  if (col < 2 * d)
    for (int b = grp; b < blocks; b += 16) s += part[(int64_t)b * 2 * d + col];
  sm[grp][threadIdx.x & 31] = s;
  __syncthreads();
  if (grp == 0 && col < 2 * d) {
#pragma unroll
    for (int j = 1; j < 16; ++j) s += sm[j][threadIdx.x];
    void* out = col < d ? dwq : dwk;
    const int at = col < d ? col : col - d;
    if (out) {
      if (w_dtype == BRC_DTYPE_F32) static_cast<float*>(out)[at] = s;
      else if (w_dtype == BRC_DTYPE_BF16)
        static_cast<__nv_bfloat16*>(out)[at] = __float2bfloat16_rn(s);
      else static_cast<__half*>(out)[at] = __float2half_rn(s);
    }
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

template <int DT, int KIND, int FMT>
int launch_fwd(const FwdArgs& g, cudaStream_t st) {
  const int lpr = lanes_per_row(g.a.d), per = kHeads * (32 / lpr);
  const int heads = g.a.hq + (KIND >= 0 ? 2 : 1) * g.a.hk;
  const int64_t bx = (g.a.tokens + kWarps - 1) / kWarps;
  const int64_t by = (heads + per - 1) / per;
  if (bx > 0x7FFFFFFF || by > 65535) return BRC_ERR_RANGE;
  const dim3 grid((unsigned)bx, (unsigned)by);
  if (lpr == 8) k_fwd<DT, 8, KIND, FMT><<<grid, kThreads, 0, st>>>(g);
  else if (lpr == 16) k_fwd<DT, 16, KIND, FMT><<<grid, kThreads, 0, st>>>(g);
  else k_fwd<DT, 32, KIND, FMT><<<grid, kThreads, 0, st>>>(g);
  return check_launch();
}

template <int DT>
int launch_write(const FwdArgs& g, cudaStream_t st) {
  const bool e4 = g.c.fmt == BRC_FP8_E4M3;
  if (g.c.kind == BRC_STE_BLOCK_FP8)
    return e4 ? launch_fwd<DT, BRC_STE_BLOCK_FP8, BRC_FP8_E4M3>(g, st)
              : launch_fwd<DT, BRC_STE_BLOCK_FP8, BRC_FP8_E5M2>(g, st);
  if (g.c.kind == BRC_STE_MXFP8)
    return e4 ? launch_fwd<DT, BRC_STE_MXFP8, BRC_FP8_E4M3>(g, st)
              : launch_fwd<DT, BRC_STE_MXFP8, BRC_FP8_E5M2>(g, st);
  return launch_fwd<DT, BRC_STE_NVFP4, BRC_FP8_E4M3>(g, st);
}

template <int DT>
void launch_bwd(const BwdArgs& g, int blocks, cudaStream_t st) {
  const int lpr = lanes_per_row(g.a.d);
  if (lpr == 8) k_bwd<DT, 8><<<blocks, kThreads, 0, st>>>(g);
  else if (lpr == 16) k_bwd<DT, 16><<<blocks, kThreads, 0, st>>>(g);
  else k_bwd<DT, 32><<<blocks, kThreads, 0, st>>>(g);
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
  FwdArgs g{};
  g.a = *a;
  g.q_out = q_out;
  g.k_out = k_out;
  const cudaStream_t st = (cudaStream_t)stream;
  if (a->dtype == BRC_DTYPE_F32) return launch_fwd<BRC_DTYPE_F32, -1, 0>(g, st);
  if (a->dtype == BRC_DTYPE_BF16) return launch_fwd<BRC_DTYPE_BF16, -1, 0>(g, st);
  return launch_fwd<BRC_DTYPE_F16, -1, 0>(g, st);
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
  return d < 16 || d > 256 ? 0 : (int64_t)kBwdBlocksMax * 2 * d * 4;
}

int brc_qk_norm_rope_bwd(const brc_norm_rope* a, const void* gq, const void* gk, int64_t gq_token,
                         int64_t gq_head, int64_t gk_token, int64_t gk_head, void* dq, void* dk,
                         void* dwq, void* dwk, void* workspace, int64_t workspace_bytes,
                         void* stream) {
  if (const int rc = check(a)) return rc;
  if ((a->hq && !dwq) || (a->hk && !dwk) || !workspace) return BRC_ERR_NULL;
  if (workspace_bytes < brc_qk_norm_rope_bwd_workspace(a->d)) return BRC_ERR_SHAPE;
  const cudaStream_t st = (cudaStream_t)stream;
  int blocks = 0;
  if (a->tokens > 0 && a->hq + a->hk > 0) {
    if ((a->hq && (!gq || !dq)) || (a->hk && (!gk || !dk))) return BRC_ERR_NULL;
    if (((uintptr_t)gq | (uintptr_t)gk | (uintptr_t)dq | (uintptr_t)dk | (uintptr_t)workspace) & 15)
      return BRC_ERR_ALIGN;
    if (bad_stride(gq_token, a->dtype) || bad_stride(gq_head, a->dtype) ||
        bad_stride(gk_token, a->dtype) || bad_stride(gk_head, a->dtype))
      return BRC_ERR_ALIGN;
    const int per = kBwdHeads * (32 / lanes_per_row(a->d));
    BwdArgs g{*a, gq, gk, gq_token, gq_head, gk_token, gk_head, dq, dk,
              static_cast<float*>(workspace), 0, (a->hq + a->hk + per - 1) / per};
    g.units = a->tokens * g.chunks;
    const int64_t want = (g.units + kWarps - 1) / kWarps;
    blocks = (int)(want < kBwdBlocksMax ? want : kBwdBlocksMax);
    if (a->dtype == BRC_DTYPE_F32) launch_bwd<BRC_DTYPE_F32>(g, blocks, st);
    else if (a->dtype == BRC_DTYPE_BF16) launch_bwd<BRC_DTYPE_BF16>(g, blocks, st);
    else launch_bwd<BRC_DTYPE_F16>(g, blocks, st);
    if (const int rc = check_launch()) return rc;
  }
  k_bwd_weights<<<(2 * a->d + 31) / 32, 512, 0, st>>>(static_cast<const float*>(workspace), blocks,
                                                      a->d, a->w_dtype, dwq, dwk);
  return check_launch();
}

}  // extern "C"
