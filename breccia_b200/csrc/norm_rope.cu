// Norm of every query and key head and the position rotation, one pass, with
// the quantised cache write of a serving step fused in, and the gradients.
//
//   r = (mean(x^2) + eps)^-1/2,  z = x r w,  y = R(position) z
//   gz = R^T gy,  gw = sum gz x r,  gx = r (gz w - x r mean(gz w x r))
//
// A stream: HBM bounds it at long prompts, launch latency at single tokens. A
// head lies on LPR = d / 16 lanes (rounded up to 4, 8 or 16), sixteen elements to a
// lane in two groups of eight that hold whole rotated pairs (halves: elements 8 p
// .. and rot / 2 + 8 p ..; interleaved: 16 p .. 16 p + 15), so a lane turns its
// pairs by itself with eight cosines and sines, and a head's sums are shuffles.
// Eight elements to a lane took 1.6 times the instructions per element and were
// bound by them. A warp takes several heads of one token, all queries or all
// keys: the token's angles and the weights are loaded once. Arithmetic is in
// packed pairs.
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

__device__ __forceinline__ float2 splat(float v) { return make_float2(v, v); }

// Sum of squares of a row; where it passes float32's range the row is taken
// 2^-64 times (x r does not change when eps goes with 2^-128). Every lane of
// the warp calls it. Returns what the row was multiplied by.
template <int LPR>
__device__ __forceinline__ float square_sum(float2* x, float& ss, float& eps) {
  auto sum = [&]() {
    float2 v = make_float2(0.f, 0.f);
#pragma unroll
    for (int i = 0; i < 8; ++i) v = __ffma2_rn(x[i], x[i], v);
    return sum_row<LPR>(__fadd_rn(v.x, v.y));
  };
  ss = sum();
  float by = 1.f;
  if (__any_sync(0xFFFFFFFFu, isinf(ss))) {
    by = isinf(ss) ? 0x1p-64f : 1.f;
    eps *= by * by;
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = __fmul2_rn(x[i], splat(by));
    ss = sum();
  }
  return by;
}

// First elements of lane `part`'s two groups of eight.
template <bool INTER>
__device__ __forceinline__ void groups(int rot, int part, int& e0, int& e1) {
  if (!INTER && part * 16 < rot) {
    e0 = 8 * part;
    e1 = (rot >> 1) + 8 * part;
  } else {  // whole pairs, or elements that are not rotated
    e0 = 16 * part;
    e1 = e0 + 8;
  }
}
template <int DT>
__device__ __forceinline__ void expand(const kv::Raw8<DT>& r, float2* f) {
  float g[8];
  kv::expand8<DT>(r, g);
#pragma unroll
  for (int i = 0; i < 4; ++i) f[i] = make_float2(g[2 * i], g[2 * i + 1]);
}
template <int DT>
__device__ __forceinline__ void store(void* p, int64_t e, const float2* f) {
  float g[8];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    g[2 * i] = f[i].x;
    g[2 * i + 1] = f[i].y;
  }
  kv::store8<DT>(p, e, g);
}
template <int DT>
__device__ __forceinline__ void load_w_as(const void* w, int e, float2* f) {
  kv::Raw8<DT> r;
  kv::load_raw8<DT>(w, e, r);
  expand<DT>(r, f);
}
__device__ __forceinline__ void load_w(const void* w, int dtype, int e, float2* f) {
  if (dtype == BRC_DTYPE_F32) load_w_as<BRC_DTYPE_F32>(w, e, f);
  else if (dtype == BRC_DTYPE_BF16) load_w_as<BRC_DTYPE_BF16>(w, e, f);
  else load_w_as<BRC_DTYPE_F16>(w, e, f);
}
// The eight angles of lane `part`'s pairs; (1, 0) where nothing is rotated; a
// NaN cosine for a position outside the table (not a wrong angle).
__device__ __forceinline__ void load_angles(const brc_norm_rope& a, int64_t token, int part,
                                            float2* c, float2* s) {
  const int64_t pos = load_index(a.positions, token, a.index64);
  const bool in = pos >= 0 && pos < a.table_rows;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    c[i] = splat(1.f);
    s[i] = splat(0.f);
  }
  if (part * 16 < a.rot) {
    const int64_t at = (in ? pos : 0) * (a.rot >> 1) + 8 * part;
    kv::Raw8<BRC_DTYPE_F32> r;
    kv::load_raw8<BRC_DTYPE_F32>(a.cos, at, r);
    expand<BRC_DTYPE_F32>(r, c);
    kv::load_raw8<BRC_DTYPE_F32>(a.sin, at, r);
    expand<BRC_DTYPE_F32>(r, s);
  }
  if (!in) {
#pragma unroll
    for (int i = 0; i < 4; ++i) c[i] = splat(__uint_as_float(0x7FC00000u));
  }
}
// R z (BACK: R^T z) of the lane's sixteen elements. Each operation is named, so
// that every kernel rounds alike.
template <bool INTER, bool BACK>
__device__ __forceinline__ void turn_pairs(const float2* c, const float2* s, float2* z) {
  if constexpr (INTER) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float ci = i & 1 ? c[i / 2].y : c[i / 2].x, si = i & 1 ? s[i / 2].y : s[i / 2].x;
      const float t = BACK ? -si : si;
      z[i] = __ffma2_rn(z[i], splat(ci), __fmul2_rn(make_float2(z[i].y, z[i].x), make_float2(-t, t)));
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 u = z[i], v = z[i + 4], n = make_float2(-s[i].x, -s[i].y);
      z[i] = __ffma2_rn(u, c[i], __fmul2_rn(v, BACK ? s[i] : n));
      z[i + 4] = __ffma2_rn(v, c[i], __fmul2_rn(u, BACK ? n : s[i]));
    }
  }
}

// ------------------------------------------------------------------ forward
// One row, in place; every lane of the warp calls it.
template <int LPR, bool INTER>
__device__ __forceinline__ void norm_turn(float2* x, const float2* w, const float2* c,
                                          const float2* s, float inv_d, float eps) {
  float ss;
  square_sum<LPR>(x, ss, eps);
  const float r = rsqrtf(__fmaf_rn(ss, inv_d, eps));
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = __fmul2_rn(__fmul2_rn(x[i], splat(r)), w[i]);
  turn_pairs<INTER, false>(c, s, x);
}

// ------------------------------------------------------------------ units of a token
// The persistent kernels' work: unit p of a token is a run of its query heads (p
// < q_parts) or key heads. A warp takes every `stride`th unit, in order.
struct Units {
  int64_t tokens;
  int q_parts, parts;   // units of a token
  int q_per, k_per;     // heads of a unit
  int step_p;           // stride % parts
  int64_t step_token;   // stride / parts
};
struct Unit {
  int64_t token;
  int p;
  __device__ __forceinline__ void next(const Units& u) {
    p += u.step_p;
    token += u.step_token;
    if (p >= u.parts) {
      p -= u.parts;
      ++token;
    }
  }
};

// A warp's angles: cosines and sines of two tokens, one in use and one on its
// way (asynchronous copies), so that a new token does not wait for them.
constexpr int kAngles = 128;  // at most d / 2 pairs, padded with (1, 0)
struct Angles {
  float* buf;  // [2][cosines, sines][kAngles]
  int at;
  __device__ __forceinline__ void init(float* b, int rot, int lane) {
    buf = b;
    at = 0;
    for (int i = (rot >> 1) + lane; i < kAngles; i += 32) {
      buf[i] = buf[2 * kAngles + i] = 1.f;
      buf[kAngles + i] = buf[3 * kAngles + i] = 0.f;
    }
  }
  // Start loading a token's angles into the buffer that is not in use. A
  // position outside the table gives NaN cosines (not a wrong angle).
  __device__ __forceinline__ void fetch(const brc_norm_rope& a, int64_t token, int lane) {
    float* const to = buf + (at ^ 1) * 2 * kAngles;
    const int64_t pos = load_index(a.positions, token, a.index64);
    const int half = a.rot >> 1;
    if (pos >= 0 && pos < a.table_rows) {
      for (int i = lane * 4; i < half; i += 128) {
        cp16(to + i, a.cos + pos * half + i);
        cp16(to + kAngles + i, a.sin + pos * half + i);
      }
    } else {
      for (int i = lane; i < kAngles; i += 32) to[i] = __uint_as_float(0x7FC00000u);
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  }
  // The angles last fetched are the ones in use from here on.
  __device__ __forceinline__ void turn(int rot, int lane) {
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    __syncwarp();
    // the other buffer's padding may hold a NaN token's: restore it
    at ^= 1;
    float* const other = buf + (at ^ 1) * 2 * kAngles;
    for (int i = (rot >> 1) + lane; i < kAngles; i += 32) other[i] = 1.f;
    __syncwarp();
  }
  __device__ __forceinline__ const float* cosines() const { return buf + at * 2 * kAngles; }
  static __device__ __forceinline__ void cp16(float* dst, const float* src) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 16;" ::"r"(
                     (uint32_t)__cvta_generic_to_shared(dst)),
                 "l"(src)
                 : "memory");
  }
};
// Eight floats of shared memory as four pairs.
__device__ __forceinline__ void lds8(const float* p, float2* f) {
  const float4 a = *reinterpret_cast<const float4*>(p), b = *reinterpret_cast<const float4*>(p + 4);
  f[0] = make_float2(a.x, a.y);
  f[1] = make_float2(a.z, a.w);
  f[2] = make_float2(b.x, b.y);
  f[3] = make_float2(b.z, b.w);
}
// Both weights as float32 in shared memory, zeros past d: sw[side][LPR * 16].
template <int LPR>
__device__ __forceinline__ void load_weights(const brc_norm_rope& a, float* sw) {
  for (int i = threadIdx.x; i < LPR * 4; i += blockDim.x) {
    const int side = i / (LPR * 2), e = (i % (LPR * 2)) * 8;
    float2 v[4] = {splat(0.f), splat(0.f), splat(0.f), splat(0.f)};
    if (e < a.d && (side ? a.hk : a.hq)) load_w(side ? a.wk : a.wq, a.w_dtype, e, v);
#pragma unroll
    for (int j = 0; j < 4; ++j) *reinterpret_cast<float2*>(sw + side * LPR * 16 + e + 2 * j) = v[j];
  }
}

#ifndef FPS
#define FPS 5
#endif
constexpr int kFwdPerSm = FPS;

// The next rows are on their way while these are worked on.
template <int DT, int LPR, bool INTER>
__global__ void __launch_bounds__(kThreads, kFwdPerSm) k_fwd(brc_norm_rope a, Units us, void* q_out,
                                                             void* k_out) {
  constexpr int G = 32 / LPR;
  __shared__ __align__(16) float sw[2 * LPR * 16];
  __shared__ __align__(16) float sa[kWarps][4 * kAngles];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, part = lane % LPR;
  const bool on = part * 16 < a.d;
  int e0, e1;
  groups<INTER>(a.rot, part, e0, e1);
  Unit u;
  {
    const int64_t first = (int64_t)blockIdx.x * kWarps + warp;
    u.token = first / us.parts;
    u.p = (int)(first - u.token * us.parts);
  }
  Angles an;
  an.init(sa[warp], a.rot, lane);
  kv::Raw8<DT> r0{}, r1{};
  constexpr int kB = DT == BRC_DTYPE_F32 ? 4 : 2;
  // the row that comes next: where it lies, where it goes, heads left to the warp
  // (this lane's is there when more than lane / LPR are left)
  const char* px = nullptr;
  char* po = nullptr;
  int64_t step_x = 0;
  int left = 0;
  bool is_q = true;
  const int mine = on ? lane / LPR : 0x7FFFFFFF;
  const int off = (e1 - e0) * kB;
  auto begin = [&]() {
    is_q = u.p < us.q_parts;
    const int per = is_q ? us.q_per : us.k_per, heads = is_q ? a.hq : a.hk;
    const int first = (is_q ? u.p : u.p - us.q_parts) * per;
    left = min(per, heads - first);
    const int64_t hs = is_q ? a.q_head : a.k_head;
    const int h = first + lane / LPR;
    px = static_cast<const char*>(is_q ? a.q : a.k) +
         (u.token * (is_q ? a.q_token : a.k_token) + h * hs + e0) * kB;
    po = static_cast<char*>(is_q ? q_out : k_out) + ((u.token * heads + h) * a.d + e0) * kB;
    step_x = G * hs * kB;
  };
  auto fetch = [&]() {
    r0 = r1 = kv::Raw8<DT>{};
    if (mine < left) {
      kv::load_raw8<DT>(px, 0, r0);
      kv::load_raw8<DT>(px + off, 0, r1);
    }
  };
  const bool any = u.token < us.tokens;
  if (any) {
    begin();
    fetch();
    an.fetch(a, u.token, lane);
  }
  load_weights<LPR>(a, sw);
  __syncthreads();
  if (!any) return;
  an.turn(a.rot, lane);
  const float inv_d = 1.f / (float)a.d;
  Unit nu = u;
  nu.next(us);
  if (nu.token < us.tokens && nu.token != u.token) an.fetch(a, nu.token, lane);
  while (true) {
    float2 f[8];
    expand<DT>(r0, f);
    expand<DT>(r1, f + 4);
    const int64_t token = u.token;
    const bool there = mine < left;
    char* const out = po;
    const float* const w = sw + (is_q ? 0 : LPR * 16);
    left -= G;
    const bool turn = left <= 0;
    if (turn) {
      u = nu;
      if (u.token < us.tokens) {
        begin();
        fetch();
      }
    } else {
      px += step_x;
      po += G * a.d * kB;
      fetch();
    }
    float ss, eps = a.eps;
    square_sum<LPR>(f, ss, eps);
    const float2 r = splat(rsqrtf(__fmaf_rn(ss, inv_d, eps)));
    float2 t[4], c[4];
    lds8(w + e0, t);
#pragma unroll
    for (int j = 0; j < 4; ++j) f[j] = __fmul2_rn(__fmul2_rn(f[j], r), t[j]);
    lds8(w + e1, t);
#pragma unroll
    for (int j = 0; j < 4; ++j) f[4 + j] = __fmul2_rn(__fmul2_rn(f[4 + j], r), t[j]);
    const float* const cs = an.cosines() + 8 * part;
    lds8(cs, c);
    lds8(cs + kAngles, t);
    turn_pairs<INTER, false>(c, t, f);
    if (there) {
      store<DT>(out, 0, f);
      store<DT>(out + off, 0, f + 4);
    }
    if (turn) {
      if (u.token >= us.tokens) break;
      nu.next(us);
      if (u.token != token) an.turn(a.rot, lane);
      if (nu.token < us.tokens && nu.token != u.token) an.fetch(a, nu.token, lane);
    }
  }
}

// Norm, rotation and the write into a cache. blockIdx.y: a batch of heads of
// queries, of keys or of values. The arithmetic is k_fwd's, operation by
// operation; a key's scales are over elements in a row, so its groups of eight
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
  const int h = chunk * G + lane / LPR;
  const bool on = h < heads;
  int64_t slot = -1;
  if (!is_q) slot = load_index(g.slots, token, g.slots64);
  if (slot >= g.c.num_pages * g.c.page_size) slot = -1;
  kv::Raw8<DT> ra{}, rb{};
  float y[16];
  if (is_v) {
    if (on) {
      kv::load_raw8<DT>(g.v, token * g.v_token + h * g.v_head + part * 16, ra);
      kv::load_raw8<DT>(g.v, token * g.v_token + h * g.v_head + part * 16 + 8, rb);
    }
  } else {
    const int64_t at = is_q ? token * a.q_token + h * a.q_head : token * a.k_token + h * a.k_head;
    int e0, e1;
    groups<INTER>(a.rot, part, e0, e1);
    if (on) {
      kv::load_raw8<DT>(is_q ? a.q : a.k, at + e0, ra);
      kv::load_raw8<DT>(is_q ? a.q : a.k, at + e1, rb);
    }
    float2 w[8], c[4], s[4], f[8];
    load_w(is_q ? a.wq : a.wk, a.w_dtype, e0, w);
    load_w(is_q ? a.wq : a.wk, a.w_dtype, e1, w + 4);
    load_angles(a, token, part, c, s);
    expand<DT>(ra, f);
    expand<DT>(rb, f + 4);
    norm_turn<LPR, INTER>(f, w, c, s, 1.f / (float)a.d, a.eps);
    if (is_q) {
      if (on) {
        store<DT>(g.q_out, (token * heads + h) * a.d + e0, f);
        store<DT>(g.q_out, (token * heads + h) * a.d + e1, f + 4);
      }
      return;
    }
    // the key as the separate call would have left it, in its own dtype
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      y[2 * i] = f[i].x;
      y[2 * i + 1] = f[i].y;
    }
    ra.v = kv::pack8<DT>(y);
    rb.v = kv::pack8<DT>(y + 8);
    if constexpr (!INTER) {
      uint4 z[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {  // elements 16 part + 8 i ..
        const int eight = 2 * part + i, half = a.rot >> 4;
        const bool turned = eight < 2 * half;
        const int from = turned ? (eight < half ? eight : eight - half) : part;
        const bool second = turned ? eight >= half : i;
        auto take = [&](uint32_t u, uint32_t v) {
          u = __shfl_sync(0xFFFFFFFFu, u, from, LPR);
          v = __shfl_sync(0xFFFFFFFFu, v, from, LPR);
          return second ? v : u;
        };
        z[i].x = take(ra.v.x, rb.v.x);
        z[i].y = take(ra.v.y, rb.v.y);
        z[i].z = take(ra.v.z, rb.v.z);
        z[i].w = take(ra.v.w, rb.v.w);
      }
      ra.v = z[0];
      rb.v = z[1];
    }
  }
  kv::expand8<DT>(ra, y);
  kv::expand8<DT>(rb, y + 8);
  const bool keep = on && slot >= 0;
  kv::encode_row<KIND, FMT, LPR>(y, part, keep, keep ? kv::row_of(g.c, slot, h) : 0,
                                 is_v ? g.c.v_data : g.c.k_data,
                                 is_v ? g.c.v_scale : g.c.k_scale);
}

// ------------------------------------------------------------------ backward
struct BwdArgs {
  brc_norm_rope a;
  Units us;  // of one side each: q_parts == parts, or 0
  const void* g[2];  // gradients of the queries' and keys' outputs
  int64_t g_token[2], g_head[2];
  void* dx[2];
  float* part;   // (blocks, d) sums of the weight gradients
  int q_blocks;  // blocks that take queries; the rest take keys
  Units ks;
};

constexpr int kBwdThreads = 128;
constexpr int kBwdWarps = kBwdThreads / 32;
#ifndef BPS
#define BPS 5
#endif
constexpr int kBwdPerSm = BPS;

// A lane sums the weight gradients of its sixteen elements over all the heads
// that it takes (a block takes one side), so that one row per block is written.
template <int DT, int LPR, bool INTER>
__global__ void __launch_bounds__(kBwdThreads, kBwdPerSm) k_bwd(BwdArgs g) {
  constexpr int G = 32 / LPR;
  const brc_norm_rope& a = g.a;
  __shared__ __align__(16) float sw[2 * LPR * 16];
  __shared__ __align__(16) float sa[kBwdWarps][4 * kAngles];
  __shared__ __align__(16) float sm[kBwdWarps * G][LPR * 16];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, part = lane % LPR;
  const bool is_q = (int)blockIdx.x < g.q_blocks;
  const int heads = is_q ? a.hq : a.hk;
  const int block = is_q ? blockIdx.x : blockIdx.x - g.q_blocks;
  const Units& us = is_q ? g.us : g.ks;
  const int64_t xt = is_q ? a.q_token : a.k_token, xh = is_q ? a.q_head : a.k_head;
  const int64_t gt = is_q ? g.g_token[0] : g.g_token[1], gh = is_q ? g.g_head[0] : g.g_head[1];
  const void* const px = is_q ? a.q : a.k;
  const void* const pg = is_q ? g.g[0] : g.g[1];
  void* const dx = is_q ? g.dx[0] : g.dx[1];
  const bool on = part * 16 < a.d;
  int e0, e1;
  groups<INTER>(a.rot, part, e0, e1);
  Unit u;
  {
    const int64_t first = (int64_t)block * kBwdWarps + warp;
    u.token = first / us.parts;
    u.p = (int)(first - u.token * us.parts);
  }
  Angles an;
  an.init(sa[warp], a.rot, lane);
  kv::Raw8<DT> nx0{}, nx1{}, ng0{}, ng1{};
  constexpr int kB = DT == BRC_DTYPE_F32 ? 4 : 2;
  // as in k_fwd
  const char *qx = nullptr, *qg = nullptr;
  char* po = nullptr;
  int left = 0;
  const int mine = on ? lane / LPR : 0x7FFFFFFF;
  const int off = (e1 - e0) * kB;
  auto begin = [&]() {
    const int first = u.p * us.q_per, h = first + lane / LPR;
    left = min(us.q_per, heads - first);
    qx = static_cast<const char*>(px) + (u.token * xt + h * xh + e0) * kB;
    qg = static_cast<const char*>(pg) + (u.token * gt + h * gh + e0) * kB;
    po = static_cast<char*>(dx) + ((u.token * heads + h) * a.d + e0) * kB;
  };
  auto fetch = [&]() {
    nx0 = nx1 = ng0 = ng1 = kv::Raw8<DT>{};
    if (mine < left) {
      kv::load_raw8<DT>(qx, 0, nx0);
      kv::load_raw8<DT>(qx + off, 0, nx1);
      kv::load_raw8<DT>(qg, 0, ng0);
      kv::load_raw8<DT>(qg + off, 0, ng1);
    }
  };
  const bool any = u.token < us.tokens;
  if (any) {
    begin();
    fetch();
    an.fetch(a, u.token, lane);
  }
  load_weights<LPR>(a, sw);
  float2 dw[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) dw[i] = splat(0.f);
  __syncthreads();
  if (any) {
    an.turn(a.rot, lane);
    const float inv_d = 1.f / (float)a.d;
    const float* const w = sw + (is_q ? 0 : LPR * 16);
    Unit nu = u;
    nu.next(us);
    if (nu.token < us.tokens && nu.token != u.token) an.fetch(a, nu.token, lane);
    while (true) {
      float2 x[8], y[8];
      expand<DT>(nx0, x);
      expand<DT>(nx1, x + 4);
      expand<DT>(ng0, y);
      expand<DT>(ng1, y + 4);
      const int64_t token = u.token;
      const bool there = mine < left;
      char* const out = po;
      left -= G;
      const bool turn = left <= 0;
      if (turn) {
        u = nu;
        if (u.token < us.tokens) {
          begin();
          fetch();
        }
      } else {
        qx += G * xh * kB;
        qg += G * gh * kB;
        po += G * a.d * kB;
        fetch();
      }
      {
        const float* const cs = an.cosines() + 8 * part;
        float2 c[4], s[4];
        lds8(cs, c);
        lds8(cs + kAngles, s);
        turn_pairs<INTER, true>(c, s, y);
      }
      float ss, eps = a.eps;
      const float by = square_sum<LPR>(x, ss, eps);
      float2 wt[8], hx2 = splat(0.f);
      lds8(w + e0, wt);
      lds8(w + e1, wt + 4);
#pragma unroll
      for (int i = 0; i < 8; ++i) hx2 = __ffma2_rn(__fmul2_rn(y[i], wt[i]), x[i], hx2);
      const float hx = sum_row<LPR>(__fadd_rn(hx2.x, hx2.y));
      const float r = rsqrtf(__fmaf_rn(ss, inv_d, eps));
      const float m = -(hx * r * inv_d);  // -mean(gz w x r)
      if (there) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float2 n = __fmul2_rn(x[i], splat(r));
          dw[i] = __ffma2_rn(y[i], n, dw[i]);
          x[i] = __fmul2_rn(__ffma2_rn(n, splat(m), __fmul2_rn(y[i], wt[i])), splat(r * by));
        }
        store<DT>(out, 0, x);
        store<DT>(out + off, 0, x + 4);
      }
      if (turn) {
        if (u.token >= us.tokens) break;
        nu.next(us);
        if (u.token != token) an.turn(a.rot, lane);
        if (nu.token < us.tokens && nu.token != u.token) an.fetch(a, nu.token, lane);
      }
    }
  }
  // lanes of the same elements: G per warp
  const int row = warp * G + lane / LPR;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    *reinterpret_cast<float2*>(&sm[row][e0 + 2 * i]) = dw[i];
    *reinterpret_cast<float2*>(&sm[row][e1 + 2 * i]) = dw[4 + i];
  }
  __syncthreads();
  for (int i = threadIdx.x; i < a.d; i += kBwdThreads) {
    float t = 0.f;
#pragma unroll
    for (int j = 0; j < kBwdWarps * G; ++j) t += sm[j][i];
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

int lanes_per_row(int d) { return d <= 64 ? 4 : d <= 128 ? 8 : 16; }

// Split `heads` into runs of whole batches of `batch`: as few as give `want` units
// over all tokens (a token's angles are then loaded once for many heads).
int split_heads(int heads, int batch, int64_t tokens, int64_t want, int& per) {
  if (!heads) {
    per = 1;
    return 0;
  }
  const int most = (heads + batch - 1) / batch;
  int64_t parts = (want + tokens - 1) / tokens;
  if (parts > most) parts = most;
  if (parts < 1) parts = 1;
  per = (int)((most + parts - 1) / parts) * batch;
  return (heads + per - 1) / per;
}
void set_stride(Units& u, int64_t warps) {
  u.step_p = (int)(warps % u.parts);
  u.step_token = warps / u.parts;
}

template <int DT, int LPR>
int launch_fwd(const brc_norm_rope& a, void* q_out, void* k_out, cudaStream_t st) {
  const int64_t most = (int64_t)sm_count() * kFwdPerSm;  // blocks
  Units u{};
  u.tokens = a.tokens;
  const int batch = 32 / LPR;
  u.q_parts = split_heads(a.hq, batch, a.tokens, 8 * most * kWarps, u.q_per);
  u.parts = u.q_parts + split_heads(a.hk, batch, a.tokens, 8 * most * kWarps, u.k_per);
  const int64_t want = (a.tokens * u.parts + kWarps - 1) / kWarps;
  const int blocks = (int)(want < most ? want : most);
  set_stride(u, (int64_t)blocks * kWarps);
  if (a.interleaved) k_fwd<DT, LPR, true><<<blocks, kThreads, 0, st>>>(a, u, q_out, k_out);
  else k_fwd<DT, LPR, false><<<blocks, kThreads, 0, st>>>(a, u, q_out, k_out);
  return check_launch();
}
template <int DT>
int launch_fwd_any(const brc_norm_rope& a, void* q_out, void* k_out, cudaStream_t st) {
  const int lpr = lanes_per_row(a.d);
  return lpr == 4   ? launch_fwd<DT, 4>(a, q_out, k_out, st)
         : lpr == 8 ? launch_fwd<DT, 8>(a, q_out, k_out, st)
                    : launch_fwd<DT, 16>(a, q_out, k_out, st);
}

template <int DT, int LPR, int KIND, int FMT>
int launch_fwd_write(const FwdArgs& g, cudaStream_t st) {
  const int per = 32 / LPR;
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
  return g.a.d == 64    ? launch_fwd_write<DT, 4, KIND, FMT>(g, st)
         : g.a.d == 128 ? launch_fwd_write<DT, 8, KIND, FMT>(g, st)
                        : launch_fwd_write<DT, 16, KIND, FMT>(g, st);
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
  if (g.a.interleaved) k_bwd<DT, LPR, true><<<blocks, kBwdThreads, 0, st>>>(g);
  else k_bwd<DT, LPR, false><<<blocks, kBwdThreads, 0, st>>>(g);
}
template <int DT>
void launch_bwd_any(const BwdArgs& g, int blocks, cudaStream_t st) {
  const int lpr = lanes_per_row(g.a.d);
  if (lpr == 4) launch_bwd<DT, 4>(g, blocks, st);
  else if (lpr == 8) launch_bwd<DT, 8>(g, blocks, st);
  else launch_bwd<DT, 16>(g, blocks, st);
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
    // the SMs are shared out by the number of heads; enough units for every warp
    const int most = sm_count() * kBwdPerSm, batch = 32 / lanes_per_row(a->d);
    int q_share = a->hk ? (int)((int64_t)most * a->hq / (a->hq + a->hk)) : most;
    if (a->hq && q_share < 1) q_share = 1;
    if (a->hk && q_share > most - 1) q_share = most - 1;
    int k_blocks = 0;
    for (int side = 0; side < 2; ++side) {
      Units& u = side ? g.ks : g.us;
      const int heads = side ? a->hk : a->hq, share = side ? most - q_share : q_share;
      u.tokens = a->tokens;
      if (!heads) {
        u.parts = 1;
        continue;
      }
      u.parts = u.q_parts =
          split_heads(heads, batch, a->tokens, 8 * (int64_t)share * kBwdWarps, u.q_per);
      const int64_t want = (a->tokens * u.parts + kBwdWarps - 1) / kBwdWarps;
      const int n = (int)(want < share ? want : share);
      (side ? k_blocks : q_blocks) = n;
      set_stride(u, (int64_t)n * kBwdWarps);
    }
    blocks = q_blocks + k_blocks;
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
