// Entry points of the attention over a quantised paged cache: argument checks,
// the split of the query rows, the workspace.
#include "kv_attention.cuh"

using namespace brc;
using namespace brc::kvatt;

namespace {

// Rows of one sequence and cache head: tiles of 8 to a product's columns, up to
// four tiles to a warp (their accumulators take d / 4 registers each: two at d =
// 256), then up to four row warps to a block.
//
// More rows than tc_rows go to the tensor-core kernel: 256 to a block, its time nearly
// the same up to that many. Both sides, 8 cache heads (us, register path / tensor cores,
// caches cold), at the rows of a cache head; 8 sequences of 16384 tokens:
//                        32         48         64         72        128        256
//   block FP8 d 128   114 / 204  181 / 204  187 / 208  321 / 208  337 / 214  599 / 263
//   MXFP8 d 128       122 / 191  200 / 194  206 / 193  353 / 196  370 / 200  663 / 241
//   NVFP4 d 128       112 / 171  183 / 173  189 / 173  325 / 175  343 / 179  611 / 210
//   block FP8 d 64    103 / 165  159 / 165  163 / 167  273 / 167  282 / 169  513 / 206
//   MXFP8 d 64        110 / 155  177 / 155  179 / 157  308 / 157  316 / 159  589 / 193
// one sequence of 16384 tokens, 8 of 1024 and one of 1024, where the two lie closer
// together:
//   block FP8 d 128    52 / 71    67 / 71    71 / 73    93 / 73   107 / 79   134 / 101
//                      42 / 54    54 / 54    58 / 56    71 / 56    85 / 62   107 / 83
//                      36 / 46    44 / 46    46 / 48    54 / 48    65 / 54    69 / 71
//   MXFP8 d 128        56 / 71    71 / 71    75 / 73    99 / 73   112 / 77   144 / 97
//                      44 / 54    56 / 56    60 / 56    75 / 56    87 / 62   112 / 81
//                      38 / 48    44 / 48    50 / 48    56 / 50    67 / 54    71 / 71
// Block FP8 decodes in fewer instructions than the others, so that its register path
// holds out longer.
struct Split {
  bool tc;
  int nt, row_warps, row_blocks, rows_per_block;
};
int tc_rows(const brc_kv_cache* c) { return c->kind == BRC_STE_BLOCK_FP8 ? 64 : 32; }
Split split_rows(int rows, const brc_kv_cache* c) {
  const int d = c->head_dim;
  Split s{};
  s.tc = rows > tc_rows(c) && (d == 128 || (d == 64 && c->kind != BRC_STE_NVFP4));
  if (s.tc) {
    s.rows_per_block = 256;
    s.row_blocks = (rows + 255) / 256;
    return s;
  }
  s.nt = rows <= 8 ? 1 : rows <= 16 ? 2 : most_tiles(d);
  const int tile = 8 * s.nt;
  s.row_warps = rows <= tile ? 1 : rows <= 2 * tile ? 2 : 4;
  s.rows_per_block = tile * s.row_warps;
  s.row_blocks = (rows + s.rows_per_block - 1) / s.rows_per_block;
  return s;
}

int blocks_of(const brc_kv_cache* c, const Split& s) {
  return sm_count() * (s.tc ? 1 : blocks_per_sm(c->kind, c->head_dim, s.nt));
}

int check(const brc_kv_cache* c, int batch, int draft, int hq) {
  if (const int rc = kv::check_cache(c)) return rc;
  if (batch < 0 || draft < 0 || hq <= 0 || hq % c->heads) return BRC_ERR_SHAPE;
  // rows, items and positions are counted in 32 bits
  if ((int64_t)c->heads * c->page_size > 0x40000000) return BRC_ERR_RANGE;
  if ((int64_t)draft * hq > (1 << 24) || (int64_t)batch * c->heads > (1 << 24) ||
      (int64_t)batch * draft * hq > 0x40000000)
    return BRC_ERR_RANGE;
  return BRC_OK;
}

}  // namespace

extern "C" {

int64_t brc_kv_attention_workspace(const brc_kv_cache* c, int batch, int draft, int hq) {
  if (check(c, batch, draft, hq) != BRC_OK) return 0;
  const Split s = split_rows(draft * (hq / c->heads), c);
  return 2 * (int64_t)blocks_of(c, s) * s.rows_per_block * (c->head_dim + 2) * 4;
}

int brc_kv_attention(const brc_kv_cache* c, const void* q, int q_dtype, int batch, int draft,
                     int hq, const int32_t* table, int64_t table_stride, int table_pages,
                     const int32_t* context, const int32_t* drafts, const uint8_t* tree,
                     int64_t tree_stride, float scale, void* out, float* lse, void* workspace,
                     int64_t workspace_bytes, void* stream) {
  if (const int rc = check(c, batch, draft, hq)) return rc;
  if (q_dtype != BRC_DTYPE_BF16 && q_dtype != BRC_DTYPE_F16) return BRC_ERR_DTYPE;
  if (table_pages < 0 || table_stride < 0 || tree_stride < 0) return BRC_ERR_SHAPE;
  if (batch == 0 || draft == 0) return BRC_OK;
  if (!q || !context || !out || !workspace || (!table && table_pages)) return BRC_ERR_NULL;
  if (((uintptr_t)q | (uintptr_t)out | (uintptr_t)workspace) & 15) return BRC_ERR_ALIGN;
  if ((int64_t)table_pages * c->page_size > 0x7FFFFFF0) return BRC_ERR_RANGE;
  const int group = hq / c->heads, rows = draft * group;
  const Split s = split_rows(rows, c);
  const int blocks = blocks_of(c, s);
  if (workspace_bytes < brc_kv_attention_workspace(c, batch, draft, hq)) return BRC_ERR_SHAPE;
  Args a{};
  a.c = *c;
  a.q = q;
  a.q_f16 = q_dtype == BRC_DTYPE_F16;
  a.batch = batch;
  a.draft = draft;
  a.hq = hq;
  a.group = group;
  a.rows = rows;
  a.table = table;
  a.table_stride = table_stride;
  a.table_pages = table_pages;
  for (a.page_shift = 4; (1 << a.page_shift) < c->page_size; ++a.page_shift) {}
  a.step_shift = s.tc ? 7 : subtiles(c->head_dim) == 2 ? 5 : 4;
  a.page_rows = (uint32_t)c->heads * c->page_size;
  a.context = context;
  a.drafts = drafts;
  a.tree = tree;
  a.tree_stride = tree_stride;
  a.scale_log2 = scale * 1.4426950408889634f;
  a.out = out;
  a.lse = lse;
  a.part_o = static_cast<float*>(workspace);
  a.part_ml = a.part_o + 2 * (int64_t)blocks * s.rows_per_block * c->head_dim;
  a.row_warps = s.row_warps;
  a.row_blocks = s.row_blocks;
  a.rows_per_block = s.rows_per_block;
  a.min_share = s.tc ? 2 : 2 * (kWarps / s.row_warps);
  const cudaStream_t st = (cudaStream_t)stream;
  if (s.tc) {
    if (c->kind == BRC_STE_NVFP4) return attend_tc_nvfp4(a, blocks, st);
    if (c->kind == BRC_STE_MXFP8)
      return c->fmt == BRC_FP8_E4M3 ? attend_tc_mx_e4m3(a, blocks, st)
                                    : attend_tc_mx_e5m2(a, blocks, st);
    return c->fmt == BRC_FP8_E4M3 ? attend_tc_block_e4m3(a, blocks, st)
                                  : attend_tc_block_e5m2(a, blocks, st);
  }
  if (c->kind == BRC_STE_NVFP4) return attend_nvfp4(a, s.nt, blocks, st);
  if (c->kind == BRC_STE_MXFP8)
    return c->fmt == BRC_FP8_E4M3 ? attend_mx_e4m3(a, s.nt, blocks, st)
                                  : attend_mx_e5m2(a, s.nt, blocks, st);
  return c->fmt == BRC_FP8_E4M3 ? attend_block_e4m3(a, s.nt, blocks, st)
                                : attend_block_e5m2(a, s.nt, blocks, st);
}

}  // extern "C"
