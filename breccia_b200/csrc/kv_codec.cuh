// Rows of a quantised key/value cache: the cache's layout, and encoding one
// row (one token, one head) held eight elements to a lane.
//
// Codes and scales are those of the casts of the same rows, bit for bit
// (jvoltci/breccia v0.1.3, src/breccia/kernels/reference/cast.py:384-404 block
// FP8 with block_k = the head dimension, :420-446 MXFP8, :468-496 NVFP4): the
// arithmetic is the casts' own (common.cuh).
#pragma once

#include "common.cuh"
#include "e8m0_thresholds.h"

namespace brc {
namespace kv {

__device__ const uint32_t g_thr[kE8m0Binades] = {BRC_E8M0_THRESHOLDS};

// 2^k for k in [-127, 127] (2^-127 is a float32 subnormal).
__device__ __forceinline__ float pow2i(int k) {
  return k == -127 ? __uint_as_float(0x00400000u) : __uint_as_float((uint32_t)(k + 127) << 23);
}

// Bytes of codes in one row, and number of scales.
__host__ __device__ constexpr int row_bytes(int kind, int d) {
  return kind == BRC_STE_NVFP4 ? d / 2 : d;
}
__host__ __device__ constexpr int row_scales(int kind, int d) {
  return kind == BRC_STE_BLOCK_FP8 ? 1 : kind == BRC_STE_MXFP8 ? d / 32 : d / 16;
}

// Row index of (slot, head) in the (page, head, token) order of the cache; the
// page size is a power of two.
__device__ __forceinline__ int64_t row_of(const brc_kv_cache& c, int64_t slot, int head) {
  const int shift = 31 - __clz(c.page_size);
  return (((slot >> shift) * c.heads + head) << shift) + (slot & (c.page_size - 1));
}

// n / d for 32-bit n and a d fixed at launch, by one multiplication.
struct Divide {
  uint32_t d;
  uint64_t m;  // ceil(2^64 / d); d = 1: unused
  explicit Divide(uint32_t by) : d(by), m(by > 1 ? ~0ull / by + 1 : 0) {}
  __device__ __forceinline__ uint32_t operator()(uint32_t n) const {
    return d == 1 ? n : (uint32_t)__umul64hi(n, m);
  }
};

// A byte of two E2M1 codes (low nibble first) to an f16 pair, exactly.
__device__ __forceinline__ uint32_t e2m1x2_to_f16x2(uint32_t byte) {
  uint32_t d;
  asm("{\n\t.reg .b8 t;\n\tcvt.u8.u32 t, %1;\n\tcvt.rn.f16x2.e2m1x2 %0, t;\n\t}"
      : "=r"(d)
      : "r"(byte));
  return d;
}

template <int DT>
__device__ __forceinline__ uint4 pack8(const float* f) {  // 8 values, one rounding (half types)
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (DT == BRC_DTYPE_BF16) {
      const __nv_bfloat162 b = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
      w[i] = *reinterpret_cast<const uint32_t*>(&b);
    } else {
      const __half2 h = __floats2half2_rn(f[2 * i], f[2 * i + 1]);
      w[i] = *reinterpret_cast<const uint32_t*>(&h);
    }
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// 8 consecutive elements of a row as they lie in memory: rows in flight wait in
// this form (half the registers of their float32 values, for half types).
template <int DT>
struct Raw8 {
  uint4 v;
};
template <>
struct Raw8<BRC_DTYPE_F32> {
  uint4 v, w;
};
template <int DT>
__device__ __forceinline__ void load_raw8(const void* p, int64_t e, Raw8<DT>& r) {
  r.v = ldg16(static_cast<const char*>(p) + (DT == BRC_DTYPE_F32 ? 4 : 2) * e);
  if constexpr (DT == BRC_DTYPE_F32) r.w = ldg16(static_cast<const char*>(p) + 4 * e + 16);
}
template <int DT>
__device__ __forceinline__ void expand8(const Raw8<DT>& r, float* f) {
  unpack<DT>(r.v, f);
  if constexpr (DT == BRC_DTYPE_F32) unpack<DT>(r.w, f + 4);
}
template <int DT>
__device__ __forceinline__ void store8(void* p, int64_t e, const float* f) {
  if constexpr (DT == BRC_DTYPE_F32) {
    char* s = static_cast<char*>(p) + 4 * e;
    stg16(s, make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]),
                        __float_as_uint(f[3])));
    stg16(s + 16, make_uint4(__float_as_uint(f[4]), __float_as_uint(f[5]), __float_as_uint(f[6]),
                             __float_as_uint(f[7])));
  } else {
    stg16(static_cast<char*>(p) + 2 * e, pack8<DT>(f));
  }
}

// Encode one row of LPR * 16 elements, sixteen to a lane (`part` = lane's place in
// the row), into row `row` of a cache side. Every lane of the warp calls it;
// lanes with `on` false only take part in the shuffles.
template <int KIND, int FMT, int LPR>
__device__ __forceinline__ void encode_row(const float* f, int part, bool on, int64_t row,
                                           uint8_t* data, void* scale) {
  constexpr int kBlockLanes = KIND == BRC_STE_BLOCK_FP8 ? LPR : KIND == BRC_STE_MXFP8 ? 2 : 1;
  float am = fmax_nan(fabsf(f[0]), fabsf(f[1]));
#pragma unroll
  for (int i = 2; i < 16; ++i) am = fmax_nan(am, fabsf(f[i]));
#pragma unroll
  for (int o = 1; o < kBlockLanes; o <<= 1)
    am = fmax_nan(am, __shfl_xor_sync(0xFFFFFFFFu, am, o));
  am = fmax_nan(am, 1e-10f);
  if (!on) return;
  constexpr float kMax = FMT == BRC_FP8_E4M3 ? 448.f : 57344.f;
  constexpr float kRcp = FMT == BRC_FP8_E4M3 ? kRcp448 : kRcp57344;
  const bool first = part % kBlockLanes == 0;
  uint32_t w[4];
  if constexpr (KIND == BRC_STE_BLOCK_FP8) {
    const float s = div_const(am, kMax, kRcp);
    if (first) static_cast<float*>(scale)[row] = canon_nan(s);
    if (isfinite(s)) {
      const float r = __frcp_rn(s);
#pragma unroll
      for (int j = 0; j < 4; ++j) w[j] = enc4_div<enc4p_fp8<FMT>>(f + 4 * j, s, r);
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        w[j] = 0;
        for (int i = 0; i < 4; ++i) w[j] |= enc1_fp8<FMT>(div_ieee(f[4 * j + i], s)) << (8 * i);
      }
    }
  } else if constexpr (KIND == BRC_STE_MXFP8) {
    const uint32_t e = e8m0_code(div_const(am, kMax, kRcp), g_thr);
    if (first) static_cast<uint8_t*>(scale)[row * (LPR / 2) + part / 2] = (uint8_t)e;
    if (isfinite(am)) {
      const float r = pow2i(127 - (int)e);  // exact reciprocal of the scale
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float2 a = __fmul2_rn(make_float2(f[4 * j], f[4 * j + 1]), make_float2(r, r));
        const float2 b = __fmul2_rn(make_float2(f[4 * j + 2], f[4 * j + 3]), make_float2(r, r));
        w[j] = enc4p_fp8<FMT>(a.x, a.y, b.x, b.y);
      }
    } else {
      const float s = pow2i((int)e - 127);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        w[j] = 0;
        for (int i = 0; i < 4; ++i) w[j] |= enc1_fp8<FMT>(div_ieee(f[4 * j + i], s)) << (8 * i);
      }
    }
  } else {
    const uint32_t sc = enc1_e4m3(div_const(am, 6.f, kRcp6));
    static_cast<uint8_t*>(scale)[row * LPR + part] = (uint8_t)sc;
    float s = dec_e4m3(sc);
    if (!(s > 0.f)) s = 0x1p-9f;
    if (isfinite(am)) {
      const float r = __frcp_rn(s);
#pragma unroll
      for (int j = 0; j < 4; ++j) w[j] = enc4_div<enc4p_e2m1>(f + 4 * j, s, r);
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        w[j] = 0;
        for (int i = 0; i < 4; ++i) w[j] |= enc1_e2m1(div_ieee(f[4 * j + i], s)) << (8 * i);
      }
    }
  }
  if constexpr (KIND == BRC_STE_NVFP4) {
    // bytes (c0 c1 c2 c3) to nibble pairs: element 2i in the low half
    uint32_t n[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const uint32_t a = w[2 * j] | (w[2 * j] >> 4), b = w[2 * j + 1] | (w[2 * j + 1] >> 4);
      n[j] = __byte_perm(a, b, 0x6420);
    }
    reinterpret_cast<uint2*>(data + row * (LPR * 8))[part] = make_uint2(n[0], n[1]);
  } else {
    stg16(data + row * (LPR * 16) + part * 16, make_uint4(w[0], w[1], w[2], w[3]));
  }
}

// One lane's eight codes of a row and their scale (zeros decode to zeros).
template <int KIND>
struct RowCodes {
  uint32_t w[KIND == BRC_STE_NVFP4 ? 1 : 2];
  uint32_t s;
};
template <int KIND, int LPR>
__device__ __forceinline__ void load_codes(const uint8_t* data, const void* scale, int64_t row,
                                           int part, RowCodes<KIND>& c) {
  if constexpr (KIND == BRC_STE_NVFP4) {
    c.w[0] = __ldg(reinterpret_cast<const uint32_t*>(data + row * (LPR * 4)) + part);
    c.s = __ldg(static_cast<const uint8_t*>(scale) + row * (LPR / 2) + part / 2);
  } else {
    const uint2 w = __ldg(reinterpret_cast<const uint2*>(data + row * (LPR * 8)) + part);
    c.w[0] = w.x;
    c.w[1] = w.y;
    if constexpr (KIND == BRC_STE_BLOCK_FP8) c.s = __ldg(static_cast<const uint32_t*>(scale) + row);
    else c.s = __ldg(static_cast<const uint8_t*>(scale) + row * (LPR / 4) + part / 4);
  }
}
// decode(code) * scale in float32.
template <int KIND, int FMT>
__device__ __forceinline__ void decode_codes(const RowCodes<KIND>& c, float* f) {
  float s;
  if constexpr (KIND == BRC_STE_NVFP4) {
    s = dec_e4m3(c.s);
#pragma unroll
    for (int i = 0; i < 4; ++i)
      f16x2_to_f32(e2m1x2_to_f16x2(c.w[0] >> (8 * i)), f[2 * i], f[2 * i + 1]);
  } else {
    if constexpr (KIND == BRC_STE_BLOCK_FP8) s = __uint_as_float(c.s);
    else s = c.s == 255 ? __uint_as_float(0x7F800000u) : pow2i((int)c.s - 127);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      f16x2_to_f32(fp8x2_to_f16x2<FMT>(c.w[i]), f[4 * i], f[4 * i + 1]);
      f16x2_to_f32(fp8x2_to_f16x2<FMT>(c.w[i] >> 16), f[4 * i + 2], f[4 * i + 3]);
    }
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) f[i] = __fmul_rn(f[i], s);
}

// Host checks shared by the entry points that take a cache.
inline int check_cache(const brc_kv_cache* c) {
  if (!c || !c->k_data || !c->k_scale || !c->v_data || !c->v_scale) return BRC_ERR_NULL;
  if (c->kind != BRC_STE_BLOCK_FP8 && c->kind != BRC_STE_MXFP8 && c->kind != BRC_STE_NVFP4)
    return BRC_ERR_DTYPE;
  if (c->fmt != BRC_FP8_E4M3 && c->fmt != BRC_FP8_E5M2) return BRC_ERR_DTYPE;
  if (c->num_pages <= 0 || c->heads <= 0) return BRC_ERR_SHAPE;
  if (c->page_size < 16 || (c->page_size & (c->page_size - 1))) return BRC_ERR_SHAPE;
  if (c->head_dim != 64 && c->head_dim != 128 && c->head_dim != 256) return BRC_ERR_UNSUPPORTED;
  if (((uintptr_t)c->k_data | (uintptr_t)c->k_scale | (uintptr_t)c->v_data |
       (uintptr_t)c->v_scale) & 15)
    return BRC_ERR_ALIGN;
  return BRC_OK;
}

}  // namespace kv
}  // namespace brc
