// Norm of every query and key head and the position rotation, one pass, with
// the quantised cache write of a serving step fused in, and the gradients.
//
//   r = (mean(x^2) + eps)^-1/2,  z = x r w,  y = R(position) z
//   gz = R^T gy,  gw = sum gz x r,  gx = r (gz w - x r mean(gz w x r))
//
// A stream: HBM bounds it at long prompts, launch latency at single tokens. A head
// lies on 16 lanes (d <= 64) or 32, four elements to a lane (d > 128: eight) in two
// groups that hold whole rotated pairs (halves: elements 2 p .. and rot / 2 + 2 p
// ..; interleaved: 4 p ..), so a lane turns its pairs by itself and keeps angles
// and weights for all the heads that it works on in ten registers. A warp takes
// up to 8 (16 lanes: 16) heads of a token at once: their sums of squares are
// reduced together, each step of the butterfly halving the rows that a lane
// carries (9 shuffles for 8 rows where one by one takes 40). Sixteen elements to a
// lane needed the angles and weights from shared memory for every head and were
// bound by that (84% of its bandwidth). Measured on B200 (launch included): 16384
// tokens of 32 + 8 heads of 128, forward 64 us bf16 (5.3 TB/s), 102 us float32
// (6.6 TB/s); 8191 tokens, gradients 66 us bf16 (3.8 TB/s), 88 us float32 (5.7).
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

__device__ __forceinline__ float2 splat(float v) { return make_float2(v, v); }

// ------------------------------------------------------------------ layout of a head
// Lanes of a head, pairs of floats to a lane.
constexpr __host__ __device__ int lanes_of(int d) { return d <= 64 ? 16 : 32; }
constexpr __host__ __device__ int pairs_of(int d) { return d <= 128 ? 2 : 4; }
// Heads that a lane works on at once: what their registers allow.
constexpr __host__ __device__ int rows_of(int dt, int np) {
  return (dt == BRC_DTYPE_F32 ? 4 : 8) / (np / 2);
}

// First elements of lane `part`'s two groups of NP.
template <int NP, bool INTER>
__device__ __forceinline__ void groups(int rot, int part, int& e0, int& e1) {
  if (!INTER && part * 2 * NP < rot) {
    e0 = NP * part;
    e1 = (rot >> 1) + NP * part;
  } else {  // whole pairs, or elements that are not rotated
    e0 = 2 * NP * part;
    e1 = e0 + NP;
  }
}

// NP elements as they lie in memory.
template <int BYTES>
struct Raw;
template <>
struct Raw<4> {
  uint32_t v[1];
};
template <>
struct Raw<8> {
  uint32_t v[2];
};
template <>
struct Raw<16> {
  uint32_t v[4];
};
template <int BYTES>
__device__ __forceinline__ void load_raw(const char* p, Raw<BYTES>& r) {
  if constexpr (BYTES == 4) {
    r.v[0] = __ldg(reinterpret_cast<const uint32_t*>(p));
  } else if constexpr (BYTES == 8) {
    const uint2 v = __ldg(reinterpret_cast<const uint2*>(p));
    r.v[0] = v.x;
    r.v[1] = v.y;
  } else {
    const uint4 v = ldg16(p);
    r.v[0] = v.x;
    r.v[1] = v.y;
    r.v[2] = v.z;
    r.v[3] = v.w;
  }
}
template <int BYTES>
__device__ __forceinline__ void store_raw(char* p, const Raw<BYTES>& r) {
  if constexpr (BYTES == 4) *reinterpret_cast<uint32_t*>(p) = r.v[0];
  else if constexpr (BYTES == 8) *reinterpret_cast<uint2*>(p) = make_uint2(r.v[0], r.v[1]);
  else stg16(p, make_uint4(r.v[0], r.v[1], r.v[2], r.v[3]));
}
constexpr __host__ __device__ int bytes_of(int dt) { return dt == BRC_DTYPE_F32 ? 4 : 2; }

template <int DT, int NP>
__device__ __forceinline__ void expand(const Raw<NP * bytes_of(DT)>& r, float2* f) {
#pragma unroll
  for (int i = 0; i < NP / 2; ++i) {
    if constexpr (DT == BRC_DTYPE_F32) {
      f[i] = make_float2(__uint_as_float(r.v[2 * i]), __uint_as_float(r.v[2 * i + 1]));
    } else if constexpr (DT == BRC_DTYPE_BF16) {
      f[i] = make_float2(__uint_as_float(r.v[i] << 16), __uint_as_float(r.v[i] & 0xFFFF0000u));
    } else {
      f16x2_to_f32(r.v[i], f[i].x, f[i].y);
    }
  }
}
template <int DT, int NP>
__device__ __forceinline__ void shrink(const float2* f, Raw<NP * bytes_of(DT)>& r) {
#pragma unroll
  for (int i = 0; i < NP / 2; ++i) {
    if constexpr (DT == BRC_DTYPE_F32) {
      r.v[2 * i] = __float_as_uint(f[i].x);
      r.v[2 * i + 1] = __float_as_uint(f[i].y);
    } else if constexpr (DT == BRC_DTYPE_BF16) {
      const __nv_bfloat162 b = __floats2bfloat162_rn(f[i].x, f[i].y);
      r.v[i] = *reinterpret_cast<const uint32_t*>(&b);
    } else {
      const __half2 h = __floats2half2_rn(f[i].x, f[i].y);
      r.v[i] = *reinterpret_cast<const uint32_t*>(&h);
    }
  }
}
template <int DT, int NP>
__device__ __forceinline__ void load_w_as(const void* w, int e, float2* f) {
  Raw<NP * bytes_of(DT)> r;
  load_raw(static_cast<const char*>(w) + e * bytes_of(DT), r);
  expand<DT, NP>(r, f);
}
// The lane's weights of one side: its two groups.
template <int NP>
__device__ __forceinline__ void load_w(const void* w, int dtype, int e0, int e1, float2* f) {
  if (dtype == BRC_DTYPE_F32) {
    load_w_as<BRC_DTYPE_F32, NP>(w, e0, f);
    load_w_as<BRC_DTYPE_F32, NP>(w, e1, f + NP / 2);
  } else if (dtype == BRC_DTYPE_BF16) {
    load_w_as<BRC_DTYPE_BF16, NP>(w, e0, f);
    load_w_as<BRC_DTYPE_BF16, NP>(w, e1, f + NP / 2);
  } else {
    load_w_as<BRC_DTYPE_F16, NP>(w, e0, f);
    load_w_as<BRC_DTYPE_F16, NP>(w, e1, f + NP / 2);
  }
}
// The angles of lane `part`'s NP pairs; (1, 0) where nothing is rotated; a NaN
// cosine for a position outside the table (not a wrong angle).
template <int NP>
__device__ __forceinline__ void load_angles(const brc_norm_rope& a, int64_t token, int part,
                                            float2* c, float2* s) {
  const int64_t pos = load_index(a.positions, token, a.index64);
  const bool in = pos >= 0 && pos < a.table_rows;
#pragma unroll
  for (int i = 0; i < NP / 2; ++i) {
    c[i] = splat(1.f);
    s[i] = splat(0.f);
  }
  if (part * 2 * NP < a.rot) {
    const int64_t at = (in ? pos : 0) * (a.rot >> 1) + NP * part;
    load_w_as<BRC_DTYPE_F32, NP>(a.cos + at, 0, c);
    load_w_as<BRC_DTYPE_F32, NP>(a.sin + at, 0, s);
  }
  if (!in) {
#pragma unroll
    for (int i = 0; i < NP / 2; ++i) c[i] = splat(__uint_as_float(0x7FC00000u));
  }
}

// R z (BACK: R^T z) of the lane's elements. Each operation is named, so that
// every kernel rounds alike.
template <int NP, bool INTER, bool BACK>
__device__ __forceinline__ void turn_pairs(const float2* c, const float2* s, float2* z) {
  if constexpr (INTER) {
#pragma unroll
    for (int i = 0; i < NP; ++i) {
      const float ci = i & 1 ? c[i / 2].y : c[i / 2].x, si = i & 1 ? s[i / 2].y : s[i / 2].x;
      const float t = BACK ? -si : si;
      z[i] = __ffma2_rn(z[i], splat(ci), __fmul2_rn(make_float2(z[i].y, z[i].x), make_float2(-t, t)));
    }
  } else {
#pragma unroll
    for (int i = 0; i < NP / 2; ++i) {
      const float2 u = z[i], v = z[i + NP / 2], n = make_float2(-s[i].x, -s[i].y);
      z[i] = __ffma2_rn(u, c[i], __fmul2_rn(v, BACK ? s[i] : n));
      z[i + NP / 2] = __ffma2_rn(v, c[i], __fmul2_rn(u, BACK ? n : s[i]));
    }
  }
}

// The same for R rows. Elements that are not rotated have no partner (it may be infinite,
// and zero times it NaN); one branch for all rows (one to a row: 16384 tokens 68 -> 72 us).
template <int R, int NP, bool INTER, bool BACK>
__device__ __forceinline__ void turn_rows(const float2* c, const float2* s, bool rotated,
                                          float2 (&z)[R][NP]) {
  if (rotated) {
#pragma unroll
    for (int i = 0; i < R; ++i) turn_pairs<NP, INTER, BACK>(c, s, z[i]);
  } else {
#pragma unroll
    for (int i = 0; i < R; ++i)
#pragma unroll
      for (int j = 0; j < NP; ++j) z[i][j] = __fmul2_rn(z[i][j], splat(c[0].x));  // 1, or NaN
  }
}

// ------------------------------------------------------------------ sums over a head
// Sums over L lanes of R values each: afterwards the lanes of a head from i *
// (L / R) on hold value i's (R lanes' worth of halving steps, then plain ones).
// Every step adds the same two numbers whichever lane keeps the sum, so a row's
// sum does not depend on which rows are reduced with it.
template <int L, int R>
__device__ __forceinline__ float sum_rows(float (&v)[R]) {
  const int lane = threadIdx.x & 31;
  int o = L / 2;
#pragma unroll
  for (int n = R / 2; n > 0; n >>= 1, o >>= 1) {
    const bool up = lane & o;
#pragma unroll
    for (int i = 0; i < n; ++i) {
      const float give = up ? v[i] : v[i + n], keep = up ? v[i + n] : v[i];
      v[i] = __fadd_rn(keep, __shfl_xor_sync(0xFFFFFFFFu, give, o));
    }
  }
  float t = v[0];
#pragma unroll
  for (int x = L / R / 2; x > 0; x >>= 1) t = __fadd_rn(t, __shfl_xor_sync(0xFFFFFFFFu, t, x));
  return t;
}
// What the lanes that hold value i have, in every lane of the head.
template <int L, int R>
__device__ __forceinline__ float of_row(float v, int i) {
  return __shfl_sync(0xFFFFFFFFu, v, i * (L / R), L);
}
template <int NP>
__device__ __forceinline__ float squares(const float2* x) {
  float2 v = __fmul2_rn(x[0], x[0]);
#pragma unroll
  for (int i = 1; i < NP; ++i) v = __ffma2_rn(x[i], x[i], v);
  return __fadd_rn(v.x, v.y);
}

// ------------------------------------------------------------------ forward
// Rows whose squares pass float32's range are taken kDown times (x r does not change
// when eps goes with its square): elements up to 2^128 then have squares up to 2^56, and
// of 256 that did pass it the largest is 2^60 or more, so that its square does not vanish.
constexpr float kDown = 0x1p-100f;

// R heads of a token in place; every lane of the warp calls it.
template <int L, int NP, int R, bool INTER>
__device__ __forceinline__ void norm_turn(float2 (&x)[R][NP], const float2* w, const float2* c,
                                          const float2* s, bool rotated, float inv_d, float eps) {
  float v[R];
#pragma unroll
  for (int i = 0; i < R; ++i) v[i] = squares<NP>(x[i]);
  float ss = sum_rows<L, R>(v);
  if (__any_sync(0xFFFFFFFFu, isinf(ss))) {
    const float by = isinf(ss) ? kDown : 1.f;
    eps = eps * by * by;
#pragma unroll
    for (int i = 0; i < R; ++i) {
      const float f = of_row<L, R>(by, i);
#pragma unroll
      for (int j = 0; j < NP; ++j) x[i][j] = __fmul2_rn(x[i][j], splat(f));
      v[i] = squares<NP>(x[i]);
    }
    ss = sum_rows<L, R>(v);
  }
  const float r = rsqrtf(__fmaf_rn(ss, inv_d, eps));
#pragma unroll
  for (int i = 0; i < R; ++i) {
    const float2 f = splat(of_row<L, R>(r, i));
#pragma unroll
    for (int j = 0; j < NP; ++j) x[i][j] = __fmul2_rn(__fmul2_rn(x[i][j], f), w[j]);
  }
  turn_rows<R, NP, INTER, false>(c, s, rotated, x);
}

// The persistent kernels' work: unit p of a token is a batch of its query heads
// (p < q_parts) or of its key heads. A warp takes every `stride`th unit.
struct Units {
  int64_t tokens, step_token;  // stride / parts
  int q_parts, parts;          // units of a token
  int step_p;                  // stride % parts
};
struct Unit {
  int64_t token;
  int p;
  __device__ __forceinline__ Unit(const Units& u, int64_t first)
      : token(first / u.parts), p((int)(first - token * u.parts)) {}
  __device__ __forceinline__ void next(const Units& u) {
    p += u.step_p;
    token += u.step_token;
    if (p >= u.parts) {
      p -= u.parts;
      ++token;
    }
  }
};

// Blocks to an SM. The rows of one unit at a time: keeping the next unit's in
// registers too cost more warps than it hid (16384 tokens, bf16: 76 against 64 us).
constexpr __host__ __device__ int fwd_per_sm(int dt, int np) {
  return dt == BRC_DTYPE_F32 || np == 4 ? 3 : 4;
}

template <int DT, int L, int NP, bool INTER>
__global__ void __launch_bounds__(kThreads, fwd_per_sm(DT, NP)) k_fwd(brc_norm_rope a, Units us, void* q_out,
                                                             void* k_out) {
  constexpr int G = 32 / L, R = rows_of(DT, NP), kB = bytes_of(DT);
  const int lane = threadIdx.x & 31, part = lane % L;
  const bool on = part * 2 * NP < a.d;
  int e0, e1;
  groups<NP, INTER>(a.rot, part, e0, e1);
  const int off = (e1 - e0) * kB;
  Unit u(us, (int64_t)blockIdx.x * kWarps + (threadIdx.x >> 5));
  Raw<NP * kB> r0[R], r1[R];
  float2 c[NP / 2], s[NP / 2];
  auto fetch = [&](const Unit& u) {
    const bool is_q = u.p < us.q_parts;
    const int first = (is_q ? u.p : u.p - us.q_parts) * (R * G) + lane / L;
    const int left = (is_q ? a.hq : a.hk) - first;
    const int64_t hs = is_q ? a.q_head : a.k_head;
    const char* p = static_cast<const char*>(is_q ? a.q : a.k) +
                    (u.token * (is_q ? a.q_token : a.k_token) + first * hs + e0) * kB;
#pragma unroll
    for (int i = 0; i < R; ++i, p += G * hs * kB) {
      r0[i] = r1[i] = Raw<NP * kB>{};
      if (on && i * G < left) {
        load_raw(p, r0[i]);
        load_raw(p + off, r1[i]);
      }
    }
  };
  if (u.token >= us.tokens) return;
  fetch(u);
  load_angles<NP>(a, u.token, part, c, s);
  float2 wq[NP], wk[NP];
#pragma unroll
  for (int i = 0; i < NP; ++i) wq[i] = wk[i] = splat(0.f);
  if (on && a.hq) load_w<NP>(a.wq, a.w_dtype, e0, e1, wq);
  if (on && a.hk) load_w<NP>(a.wk, a.w_dtype, e0, e1, wk);
  const float inv_d = 1.f / (float)a.d;
  while (true) {
    float2 x[R][NP], w[NP], nc[NP / 2], ns[NP / 2];
#pragma unroll
    for (int i = 0; i < R; ++i) {
      expand<DT, NP>(r0[i], x[i]);
      expand<DT, NP>(r1[i], x[i] + NP / 2);
    }
    const bool is_q = u.p < us.q_parts;
    const int heads = is_q ? a.hq : a.hk;
    const int first = (is_q ? u.p : u.p - us.q_parts) * (R * G) + lane / L;
    char* out = static_cast<char*>(is_q ? q_out : k_out) +
                ((u.token * heads + first) * a.d + e0) * kB;
    const int left = heads - first;
    u.next(us);
    const bool more = u.token < us.tokens;
#pragma unroll
    for (int i = 0; i < NP; ++i) w[i] = is_q ? wq[i] : wk[i];
    norm_turn<L, NP, R, INTER>(x, w, c, s, part * 2 * NP < a.rot, inv_d, a.eps);
#pragma unroll
    for (int i = 0; i < R; ++i, out += G * a.d * kB) {
      if (on && i * G < left) {
        Raw<NP * kB> y;
        shrink<DT, NP>(x[i], y);
        store_raw(out, y);
        shrink<DT, NP>(x[i] + NP / 2, y);
        store_raw(out + off, y);
      }
    }
    if (!more) break;
    fetch(u);
    load_angles<NP>(a, u.token, part, nc, ns);
#pragma unroll
    for (int i = 0; i < NP / 2; ++i) {
      c[i] = nc[i];
      s[i] = ns[i];
    }
  }
}

// Norm, rotation and the write into a cache. blockIdx.y: a batch of heads of
// queries, of keys or of values. The arithmetic is k_fwd's, operation by
// operation; a key's scales are over elements in a row, so its rows (rounded as
// the separate call rounds them) go through the warp's own shared memory into
// the encoder's order.
template <int DT, int L, int NP, bool INTER, int KIND, int FMT>
__global__ void __launch_bounds__(kThreads) k_fwd_write(FwdArgs g, int q_chunks, int k_chunks) {
  constexpr int G = 32 / L, R = rows_of(DT, NP), D = L * 2 * NP;
  constexpr int LPR = D / 16, kRows = R * G, kPitch = D + 8;
  __shared__ __align__(16) uint16_t rows[kWarps][kRows * kPitch];
  const brc_norm_rope& a = g.a;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, part = lane % L;
  const int64_t token = (int64_t)blockIdx.x * kWarps + warp;
  if (token >= a.tokens) return;
  const bool is_q = (int)blockIdx.y < q_chunks, is_v = (int)blockIdx.y >= q_chunks + k_chunks;
  const int heads = is_q ? a.hq : a.hk;
  const int chunk = is_q ? blockIdx.y : blockIdx.y - q_chunks - (is_v ? k_chunks : 0);
  int64_t slot = -1;
  if (!is_q) slot = load_index(g.slots, token, g.slots64);
  if (slot >= g.c.num_pages * g.c.page_size) slot = -1;
  if (!is_v) {
    const int first = chunk * kRows + lane / L, left = heads - first;
    int e0, e1;
    groups<NP, INTER>(a.rot, part, e0, e1);
    const int off = (e1 - e0) * 2;
    const int64_t hs = is_q ? a.q_head : a.k_head;
    const char* p = static_cast<const char*>(is_q ? a.q : a.k) +
                    (token * (is_q ? a.q_token : a.k_token) + first * hs + e0) * 2;
    Raw<NP * 2> r0[R], r1[R];
#pragma unroll
    for (int i = 0; i < R; ++i, p += G * hs * 2) {
      r0[i] = r1[i] = Raw<NP * 2>{};
      if (i * G < left) {
        load_raw(p, r0[i]);
        load_raw(p + off, r1[i]);
      }
    }
    float2 w[NP], c[NP / 2], s[NP / 2], x[R][NP];
    load_w<NP>(is_q ? a.wq : a.wk, a.w_dtype, e0, e1, w);
    load_angles<NP>(a, token, part, c, s);
#pragma unroll
    for (int i = 0; i < R; ++i) {
      expand<DT, NP>(r0[i], x[i]);
      expand<DT, NP>(r1[i], x[i] + NP / 2);
    }
    norm_turn<L, NP, R, INTER>(x, w, c, s, part * 2 * NP < a.rot, 1.f / (float)a.d, a.eps);
    char* out = is_q ? static_cast<char*>(g.q_out) + ((token * heads + first) * a.d + e0) * 2
                     : reinterpret_cast<char*>(&rows[warp][lane / L * kPitch + e0]);
    const int step = is_q ? G * a.d * 2 : G * kPitch * 2;
#pragma unroll
    for (int i = 0; i < R; ++i, out += step) {
      if (i * G < left) {
        Raw<NP * 2> y;
        shrink<DT, NP>(x[i], y);
        store_raw(out, y);
        shrink<DT, NP>(x[i] + NP / 2, y);
        store_raw(out + off, y);
      }
    }
    if (is_q) return;
    __syncwarp();
  }
  // sixteen elements to a lane, 32 / LPR heads at a time
  const int at = lane % LPR * 16;
#pragma unroll
  for (int i = 0; i < kRows; i += 32 / LPR) {
    const int row = i + lane / LPR, h = chunk * kRows + row;
    const bool there = row < kRows && h < heads;
    kv::Raw8<DT> lo{}, hi{};
    if (there) {
      if (is_v) {
        kv::load_raw8<DT>(g.v, token * g.v_token + h * g.v_head + at, lo);
        kv::load_raw8<DT>(g.v, token * g.v_token + h * g.v_head + at + 8, hi);
      } else {
        lo.v = *reinterpret_cast<const uint4*>(&rows[warp][row * kPitch + at]);
        hi.v = *reinterpret_cast<const uint4*>(&rows[warp][row * kPitch + at + 8]);
      }
    }
    float y[16];
    kv::expand8<DT>(lo, y);
    kv::expand8<DT>(hi, y + 8);
    const bool keep = there && slot >= 0;
    kv::encode_row<KIND, FMT, LPR>(y, lane % LPR, keep, keep ? kv::row_of(g.c, slot, h) : 0,
                                   is_v ? g.c.v_data : g.c.k_data,
                                   is_v ? g.c.v_scale : g.c.k_scale);
  }
}

// ------------------------------------------------------------------ backward
struct BwdArgs {
  brc_norm_rope a;
  Units us[2];       // of one side each
  const void* g[2];  // gradients of the queries' and keys' outputs
  int64_t g_token[2], g_head[2];
  void* dx[2];
  float* part;   // (blocks, d) sums of the weight gradients
  int q_blocks;  // blocks that take queries; the rest take keys
};

constexpr int kBwdThreads = 128;
constexpr int kBwdWarps = kBwdThreads / 32;
constexpr int kBwdPerSm = 6;
constexpr __host__ __device__ int bwd_rows(int dt, int np) { return rows_of(dt, np) / 2; }

// A lane sums the weight gradients of its elements over all the heads that it
// takes (a block takes one side), so that one row per block is written.
template <int DT, int L, int NP, bool INTER>
__global__ void __launch_bounds__(kBwdThreads, kBwdPerSm) k_bwd(BwdArgs g) {
  constexpr int G = 32 / L, R = bwd_rows(DT, NP), kB = bytes_of(DT);
  const brc_norm_rope& a = g.a;
  __shared__ __align__(16) float sm[kBwdWarps * G][L * 2 * NP];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, part = lane % L;
  const bool is_q = (int)blockIdx.x < g.q_blocks;
  const int heads = is_q ? a.hq : a.hk;
  const int block = is_q ? blockIdx.x : blockIdx.x - g.q_blocks;
  const Units& us = is_q ? g.us[0] : g.us[1];
  const int64_t xt = is_q ? a.q_token : a.k_token, xh = is_q ? a.q_head : a.k_head;
  const int64_t gt = is_q ? g.g_token[0] : g.g_token[1], gh = is_q ? g.g_head[0] : g.g_head[1];
  const bool on = part * 2 * NP < a.d;
  int e0, e1;
  groups<NP, INTER>(a.rot, part, e0, e1);
  const int off = (e1 - e0) * kB;
  const char* const px = static_cast<const char*>(is_q ? a.q : a.k) + e0 * kB;
  const char* const pg = static_cast<const char*>(is_q ? g.g[0] : g.g[1]) + e0 * kB;
  char* const dx = static_cast<char*>(is_q ? g.dx[0] : g.dx[1]) + e0 * kB;
  float2 w[NP], dw[NP];
#pragma unroll
  for (int i = 0; i < NP; ++i) w[i] = dw[i] = splat(0.f);
  if (on) load_w<NP>(is_q ? a.wq : a.wk, a.w_dtype, e0, e1, w);
  Raw<NP * kB> x0[R], x1[R], y0[R], y1[R];
  float2 c[NP / 2], s[NP / 2];
  auto fetch = [&](const Unit& u) {
    const int first = u.p * (R * G) + lane / L, left = heads - first;
    const char* p = px + (u.token * xt + first * xh) * kB;
    const char* q = pg + (u.token * gt + first * gh) * kB;
#pragma unroll
    for (int i = 0; i < R; ++i, p += G * xh * kB, q += G * gh * kB) {
      x0[i] = x1[i] = y0[i] = y1[i] = Raw<NP * kB>{};
      if (on && i * G < left) {
        load_raw(p, x0[i]);
        load_raw(p + off, x1[i]);
        load_raw(q, y0[i]);
        load_raw(q + off, y1[i]);
      }
    }
  };
  Unit u(us, (int64_t)block * kBwdWarps + warp);
  const float inv_d = 1.f / (float)a.d;
  if (u.token < us.tokens) {
    fetch(u);
    load_angles<NP>(a, u.token, part, c, s);
    while (true) {
      float2 x[R][NP], y[R][NP];
#pragma unroll
      for (int i = 0; i < R; ++i) {
        expand<DT, NP>(x0[i], x[i]);
        expand<DT, NP>(x1[i], x[i] + NP / 2);
        expand<DT, NP>(y0[i], y[i]);
        expand<DT, NP>(y1[i], y[i] + NP / 2);
      }
      const int first = u.p * (R * G) + lane / L, left = heads - first;
      char* out = dx + (u.token * heads + first) * a.d * kB;
      u.next(us);
      const bool more = u.token < us.tokens;
      float2 nc[NP / 2], ns[NP / 2];
      // sums of x^2 (values 0 .. R - 1) and of gz w x (R .. 2 R - 1) together
      float v[2 * R], by = 1.f, eps = a.eps;
      auto sums = [&]() {
#pragma unroll
        for (int i = 0; i < R; ++i) {
          v[i] = squares<NP>(x[i]);
          float2 t = splat(0.f);
#pragma unroll
          for (int j = 0; j < NP; ++j) t = __ffma2_rn(__fmul2_rn(y[i][j], w[j]), x[i][j], t);
          v[R + i] = __fadd_rn(t.x, t.y);
        }
        return sum_rows<L, 2 * R>(v);
      };
      turn_rows<R, NP, INTER, true>(c, s, part * 2 * NP < a.rot, y);
      float t = sums();
      const bool sq = part < L / 2;  // this lane holds a sum of squares
      if (__any_sync(0xFFFFFFFFu, sq && isinf(t))) {
        by = sq && isinf(t) ? kDown : 1.f;
        eps = eps * by * by;
#pragma unroll
        for (int i = 0; i < R; ++i) {
          const float f = of_row<L, 2 * R>(by, i);
#pragma unroll
          for (int j = 0; j < NP; ++j) x[i][j] = __fmul2_rn(x[i][j], splat(f));
        }
        t = sums();
      }
      const float r = rsqrtf(__fmaf_rn(t, inv_d, eps));  // of lanes with a sum of squares
#pragma unroll
      for (int i = 0; i < R; ++i) {
        const float ri = of_row<L, 2 * R>(r, i), hx = of_row<L, 2 * R>(t, R + i);
        const float bi = of_row<L, 2 * R>(by, i);
        const float2 m = splat(-(hx * ri * inv_d));  // -mean(gz w x r)
        if (on && i * G < left) {
#pragma unroll
          for (int j = 0; j < NP; ++j) {
            const float2 n = __fmul2_rn(x[i][j], splat(ri));
            dw[j] = __ffma2_rn(y[i][j], n, dw[j]);
            x[i][j] = __fmul2_rn(__ffma2_rn(n, m, __fmul2_rn(y[i][j], w[j])), splat(ri * bi));
          }
          Raw<NP * kB> o;
          shrink<DT, NP>(x[i], o);
          store_raw(out, o);
          shrink<DT, NP>(x[i] + NP / 2, o);
          store_raw(out + off, o);
        }
        out += G * a.d * kB;
      }
      if (!more) break;
      fetch(u);
      load_angles<NP>(a, u.token, part, nc, ns);
#pragma unroll
      for (int i = 0; i < NP / 2; ++i) {
        c[i] = nc[i];
        s[i] = ns[i];
      }
    }
  }
  // lanes of the same elements: G per warp
  const int row = warp * G + lane / L;
#pragma unroll
  for (int i = 0; i < NP / 2; ++i) {
    *reinterpret_cast<float2*>(&sm[row][e0 + 2 * i]) = dw[i];
    *reinterpret_cast<float2*>(&sm[row][e1 + 2 * i]) = dw[NP / 2 + i];
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

void set_stride(Units& u, int64_t warps) {
  u.step_p = (int)(warps % u.parts);
  u.step_token = warps / u.parts;
}
int ceil_div(int a, int b) { return (a + b - 1) / b; }

template <int DT, int L, int NP>
int launch_fwd(const brc_norm_rope& a, void* q_out, void* k_out, cudaStream_t st) {
  constexpr int kRows = rows_of(DT, NP) * (32 / L);
  Units u{};
  u.tokens = a.tokens;
  u.q_parts = ceil_div(a.hq, kRows);
  u.parts = u.q_parts + ceil_div(a.hk, kRows);
  const int64_t most = (int64_t)sm_count() * fwd_per_sm(DT, NP);
  const int64_t want = (a.tokens * u.parts + kWarps - 1) / kWarps;
  const int blocks = (int)(want < most ? want : most);
  set_stride(u, (int64_t)blocks * kWarps);
  if (a.interleaved) k_fwd<DT, L, NP, true><<<blocks, kThreads, 0, st>>>(a, u, q_out, k_out);
  else k_fwd<DT, L, NP, false><<<blocks, kThreads, 0, st>>>(a, u, q_out, k_out);
  return check_launch();
}
template <int DT>
int launch_fwd_any(const brc_norm_rope& a, void* q_out, void* k_out, cudaStream_t st) {
  if (a.d <= 64) return launch_fwd<DT, lanes_of(64), pairs_of(64)>(a, q_out, k_out, st);
  if (a.d <= 128) return launch_fwd<DT, lanes_of(128), pairs_of(128)>(a, q_out, k_out, st);
  return launch_fwd<DT, lanes_of(256), pairs_of(256)>(a, q_out, k_out, st);
}

template <int DT, int L, int NP, int KIND, int FMT>
int launch_fwd_write(const FwdArgs& g, cudaStream_t st) {
  constexpr int kRows = rows_of(DT, NP) * (32 / L);
  const int64_t bx = (g.a.tokens + kWarps - 1) / kWarps;
  const int q_chunks = ceil_div(g.a.hq, kRows), k_chunks = ceil_div(g.a.hk, kRows);
  if (bx > 0x7FFFFFFF || q_chunks + 2 * (int64_t)k_chunks > 65535) return BRC_ERR_RANGE;
  const dim3 grid((unsigned)bx, (unsigned)(q_chunks + 2 * k_chunks));
  if (g.a.interleaved)
    k_fwd_write<DT, L, NP, true, KIND, FMT><<<grid, kThreads, 0, st>>>(g, q_chunks, k_chunks);
  else k_fwd_write<DT, L, NP, false, KIND, FMT><<<grid, kThreads, 0, st>>>(g, q_chunks, k_chunks);
  return check_launch();
}
template <int DT, int KIND, int FMT>
int launch_write_dim(const FwdArgs& g, cudaStream_t st) {
  return g.a.d == 64    ? launch_fwd_write<DT, lanes_of(64), pairs_of(64), KIND, FMT>(g, st)
         : g.a.d == 128 ? launch_fwd_write<DT, lanes_of(128), pairs_of(128), KIND, FMT>(g, st)
                        : launch_fwd_write<DT, lanes_of(256), pairs_of(256), KIND, FMT>(g, st);
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

// The blocks: shared out between queries and keys by the number of heads.
template <int DT, int L, int NP>
int launch_bwd(BwdArgs& g, int& blocks, cudaStream_t st) {
  constexpr int kRows = bwd_rows(DT, NP) * (32 / L);
  const int most = sm_count() * kBwdPerSm, hq = g.a.hq, hk = g.a.hk;
  int q_share = hk ? (int)((int64_t)most * hq / (hq + hk)) : most;
  if (hq && q_share < 1) q_share = 1;
  if (hk && q_share > most - 1) q_share = most - 1;
  int n[2] = {0, 0};
  for (int side = 0; side < 2; ++side) {
    Units& u = g.us[side];
    const int heads = side ? hk : hq, share = side ? most - q_share : q_share;
    u.tokens = g.a.tokens;
    u.parts = 1;
    if (!heads) continue;
    u.parts = ceil_div(heads, kRows);
    const int64_t want = (u.tokens * u.parts + kBwdWarps - 1) / kBwdWarps;
    n[side] = (int)(want < share ? want : share);
    set_stride(u, (int64_t)n[side] * kBwdWarps);
  }
  g.q_blocks = n[0];
  blocks = n[0] + n[1];
  if (g.a.interleaved) k_bwd<DT, L, NP, true><<<blocks, kBwdThreads, 0, st>>>(g);
  else k_bwd<DT, L, NP, false><<<blocks, kBwdThreads, 0, st>>>(g);
  return check_launch();
}
template <int DT>
int launch_bwd_any(BwdArgs& g, int& blocks, cudaStream_t st) {
  if (g.a.d <= 64) return launch_bwd<DT, lanes_of(64), pairs_of(64)>(g, blocks, st);
  if (g.a.d <= 128) return launch_bwd<DT, lanes_of(128), pairs_of(128)>(g, blocks, st);
  return launch_bwd<DT, lanes_of(256), pairs_of(256)>(g, blocks, st);
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
    const int rc = a->dtype == BRC_DTYPE_F32    ? launch_bwd_any<BRC_DTYPE_F32>(g, blocks, st)
                   : a->dtype == BRC_DTYPE_BF16 ? launch_bwd_any<BRC_DTYPE_BF16>(g, blocks, st)
                                                : launch_bwd_any<BRC_DTYPE_F16>(g, blocks, st);
    if (rc) return rc;
    q_blocks = g.q_blocks;
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
