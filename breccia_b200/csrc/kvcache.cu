// Quantised key/value cache: rows written as they are produced, and read back.
//
// Both are streams: a row (one token, one head) is read once and written once;
// HBM bounds the read at long prompts, the encoders' integer arithmetic the
// write. To write, a row lies on d / 16 lanes, sixteen elements to a lane, so
// that a scale's block is one or two lanes (block FP8: the row) and what a row
// costs beside its elements is shared by twice as many. To read, it lies on d /
// 8: the 16-byte stores of a warp are then 512 contiguous bytes. Every lane has
// several rows in flight. Measured on B200 (launch included), 8 heads of 128: 16384
// bf16 tokens written as block FP8 25 us (4.0 TB/s; eight elements to a lane 33), 8
// sequences of up to 4096 tokens read from MXFP8 to bf16 39 us (4.9 TB/s).
#include "kv_codec.cuh"
#include "launch.h"

namespace brc {
namespace kv {
namespace {

constexpr int kThreads = 256;
constexpr int kReadRows = 8;  // rows in flight per lane, as they lie in memory
constexpr __host__ __device__ int write_rows(int dt) { return dt == BRC_DTYPE_F32 ? 1 : 2; }

__device__ __forceinline__ int64_t load_index(const void* p, int64_t i, int is64) {
  return is64 ? static_cast<const int64_t*>(p)[i] : (int64_t)static_cast<const int32_t*>(p)[i];
}

struct WriteArgs {
  brc_kv_cache c;
  const void* x[2];  // keys, values
  int64_t token[2], head[2];
  const void* slots;
  int slots64;
  uint32_t rows;  // tokens * heads
  Divide heads;
};

// blockIdx.y: 0 keys, 1 values.
template <int DT, int KIND, int FMT, int LPR>
__global__ void __launch_bounds__(kThreads, 4) k_write(WriteArgs a) {
  constexpr int G = 32 / LPR, kRows = write_rows(DT);
  const int lane = threadIdx.x & 31, part = lane % LPR;
  const int side = blockIdx.y;
  const void* x = side ? a.x[1] : a.x[0];
  const int64_t ts = side ? a.token[1] : a.token[0], hs = side ? a.head[1] : a.head[0];
  uint8_t* data = side ? a.c.v_data : a.c.k_data;
  void* scale = side ? a.c.v_scale : a.c.k_scale;
  const int64_t slots = a.c.num_pages * a.c.page_size;
  const uint32_t first =
      (blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5)) * (kRows * G) + lane / LPR;
  Raw8<DT> lo[kRows], hi[kRows];
  int64_t row[kRows];
#pragma unroll
  for (int u = 0; u < kRows; ++u) {
    const uint32_t r = first + u * G;
    row[u] = -1;
    lo[u] = hi[u] = Raw8<DT>{};
    if (r < a.rows) {
      const uint32_t t = a.heads(r), h = r - t * a.heads.d;
      const int64_t at = t * ts + h * hs + part * 16;
      load_raw8<DT>(x, at, lo[u]);
      load_raw8<DT>(x, at + 8, hi[u]);
      const int64_t slot = load_index(a.slots, t, a.slots64);
      if (slot >= 0 && slot < slots) row[u] = row_of(a.c, slot, (int)h);
    }
  }
#pragma unroll
  for (int u = 0; u < kRows; ++u) {
    float f[16];
    expand8<DT>(lo[u], f);
    expand8<DT>(hi[u], f + 8);
    encode_row<KIND, FMT, LPR>(f, part, row[u] >= 0, row[u], data, scale);
  }
}

struct ReadArgs {
  brc_kv_cache c;
  const int32_t* table;
  const int32_t* lengths;
  int64_t table_stride;
  uint32_t rows;  // batch * length * heads
  int table_pages;
  Divide heads, length;
  void* out[2];
};

template <int DT, int KIND, int FMT, int LPR>
__global__ void __launch_bounds__(kThreads) k_read(ReadArgs a) {
  constexpr int G = 32 / LPR;
  const int lane = threadIdx.x & 31, part = lane % LPR;
  const int side = blockIdx.y;
  const uint8_t* data = side ? a.c.v_data : a.c.k_data;
  const void* scale = side ? a.c.v_scale : a.c.k_scale;
  void* out = side ? a.out[1] : a.out[0];
  const uint32_t first =
      (blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5)) * (kReadRows * G) + lane / LPR;
  const int shift = 31 - __clz(a.c.page_size);
  RowCodes<KIND> w[kReadRows];
#pragma unroll
  for (int u = 0; u < kReadRows; ++u) {
    const uint32_t r = first + u * G;
    w[u] = RowCodes<KIND>{};
    if (r < a.rows) {
      const uint32_t bt = a.heads(r), h = r - bt * a.heads.d;
      const uint32_t b = a.length(bt), t = bt - b * a.length.d;
      const uint32_t p = t >> shift;
      if ((int64_t)t < a.lengths[b] && p < (uint32_t)a.table_pages) {
        const int64_t page = a.table[b * a.table_stride + p];
        if (page >= 0 && page < a.c.num_pages)
          load_codes<KIND, LPR>(data, scale,
                                ((page * a.c.heads + h) << shift) + (t & (a.c.page_size - 1)),
                                part, w[u]);
      }
    }
  }
#pragma unroll
  for (int u = 0; u < kReadRows; ++u) {
    const uint32_t r = first + u * G;
    if (r < a.rows) {
      float f[8];
      decode_codes<KIND, FMT>(w[u], f);
      store8<DT>(out, (int64_t)r * (LPR * 8) + part * 8, f);
    }
  }
}

// Launch gets the head dimension.
template <template <int, int, int, int> class Launch, int DT, int KIND, int FMT, class Args>
int by_dim(int d, const Args& a, dim3 grid, cudaStream_t st) {
  switch (d) {
    case 64: Launch<DT, KIND, FMT, 64>::run(a, grid, st); break;
    case 128: Launch<DT, KIND, FMT, 128>::run(a, grid, st); break;
    default: Launch<DT, KIND, FMT, 256>::run(a, grid, st); break;
  }
  return check_launch();
}
template <template <int, int, int, int> class Launch, int DT, class Args>
int by_kind(const Args& a, dim3 grid, cudaStream_t st) {
  const int d = a.c.head_dim;
  const bool e4 = a.c.fmt == BRC_FP8_E4M3;
  if (a.c.kind == BRC_STE_BLOCK_FP8)
    return e4 ? by_dim<Launch, DT, BRC_STE_BLOCK_FP8, BRC_FP8_E4M3>(d, a, grid, st)
              : by_dim<Launch, DT, BRC_STE_BLOCK_FP8, BRC_FP8_E5M2>(d, a, grid, st);
  if (a.c.kind == BRC_STE_MXFP8)
    return e4 ? by_dim<Launch, DT, BRC_STE_MXFP8, BRC_FP8_E4M3>(d, a, grid, st)
              : by_dim<Launch, DT, BRC_STE_MXFP8, BRC_FP8_E5M2>(d, a, grid, st);
  return by_dim<Launch, DT, BRC_STE_NVFP4, BRC_FP8_E4M3>(d, a, grid, st);
}
template <template <int, int, int, int> class Launch, class Args>
int by_dtype(int dt, const Args& a, dim3 grid, cudaStream_t st) {
  switch (dt) {
    case BRC_DTYPE_F32: return by_kind<Launch, BRC_DTYPE_F32>(a, grid, st);
    case BRC_DTYPE_BF16: return by_kind<Launch, BRC_DTYPE_BF16>(a, grid, st);
    default: return by_kind<Launch, BRC_DTYPE_F16>(a, grid, st);
  }
}
template <int DT, int KIND, int FMT, int D>
struct LaunchWrite {
  static void run(const WriteArgs& a, dim3 grid, cudaStream_t st) {
    k_write<DT, KIND, FMT, D / 16><<<grid, kThreads, 0, st>>>(a);
  }
};
template <int DT, int KIND, int FMT, int D>
struct LaunchRead {
  static void run(const ReadArgs& a, dim3 grid, cudaStream_t st) {
    k_read<DT, KIND, FMT, D / 8><<<grid, kThreads, 0, st>>>(a);
  }
};

// Blocks for `rows` rows, `per_warp` to a warp; 0 where 32 bits do not count them.
int64_t blocks_for(int64_t rows, int per_warp) {
  const int per = (kThreads / 32) * per_warp;
  return rows > 0xFFFFFFFFll - per ? 0 : (rows + per - 1) / per;
}

bool bad_stride(int64_t s, int dtype) { return s % (dtype == BRC_DTYPE_F32 ? 4 : 8) != 0; }

}  // namespace
}  // namespace kv
}  // namespace brc

using namespace brc;
using namespace brc::kv;

extern "C" {

int brc_kv_write(const brc_kv_cache* c, const void* k, const void* v, int dtype, int64_t tokens,
                 int64_t k_token, int64_t k_head, int64_t v_token, int64_t v_head,
                 const void* slots, int slots64, void* stream) {
  if (const int rc = check_cache(c)) return rc;
  if (tokens < 0) return BRC_ERR_SHAPE;
  if (dtype < BRC_DTYPE_F32 || dtype > BRC_DTYPE_F16) return BRC_ERR_DTYPE;
  if (tokens == 0) return BRC_OK;
  if (!k || !v || !slots) return BRC_ERR_NULL;
  if (((uintptr_t)k | (uintptr_t)v) & 15) return BRC_ERR_ALIGN;
  if (bad_stride(k_token, dtype) || bad_stride(k_head, dtype) || bad_stride(v_token, dtype) ||
      bad_stride(v_head, dtype))
    return BRC_ERR_ALIGN;
  if (tokens > 0xFFFFFFFFll) return BRC_ERR_RANGE;
  const int64_t n = blocks_for(tokens * c->heads, write_rows(dtype) * (32 / (c->head_dim / 16)));
  if (n == 0) return BRC_ERR_RANGE;
  WriteArgs a{*c, {k, v}, {k_token, v_token}, {k_head, v_head}, slots, slots64,
              (uint32_t)(tokens * c->heads), Divide((uint32_t)c->heads)};
  return by_dtype<LaunchWrite>(dtype, a, dim3((unsigned)n, 2), (cudaStream_t)stream);
}

int brc_kv_read(const brc_kv_cache* c, const int32_t* table, int64_t table_stride,
                int table_pages, const int32_t* lengths, int batch, int64_t length, void* k_out,
                void* v_out, int out_dtype, void* stream) {
  if (const int rc = check_cache(c)) return rc;
  if (batch < 0 || length < 0 || table_pages < 0 || table_stride < 0) return BRC_ERR_SHAPE;
  if (out_dtype < BRC_DTYPE_F32 || out_dtype > BRC_DTYPE_F16) return BRC_ERR_DTYPE;
  if (batch == 0 || length == 0) return BRC_OK;
  if ((!table && table_pages) || !lengths || !k_out || !v_out) return BRC_ERR_NULL;
  if (((uintptr_t)k_out | (uintptr_t)v_out) & 15) return BRC_ERR_ALIGN;
  if (length > 0x7FFFFFFF || (int64_t)batch * length > 0xFFFFFFFFll) return BRC_ERR_RANGE;
  const int64_t rows = (int64_t)batch * length * c->heads;
  const int64_t n = blocks_for(rows, kReadRows * (32 / (c->head_dim / 8)));
  if (n == 0) return BRC_ERR_RANGE;
  ReadArgs a{*c, table, lengths, table_stride, (uint32_t)rows, table_pages,
             Divide((uint32_t)c->heads), Divide((uint32_t)length), {k_out, v_out}};
  return by_dtype<LaunchRead>(out_dtype, a, dim3((unsigned)n, 2), (cudaStream_t)stream);
}

}  // extern "C"
