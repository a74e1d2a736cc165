// Shared by the chunked prefill kernels: launch parameters, the tensor map of a
// pool in the tile layout of the MMA descriptors, and the host-side checks.
#pragma once

#include "decode_common.cuh"

namespace mz {
namespace prefill {

using decode::kTileTok;
using decode::kTimeoutNs;

constexpr int kM = 128;  // query rows per item: 128 / G tokens of a KV head's G query heads

struct PParams {
  void *out;
  int64_t o_st, o_sh;  // out element (row t of the call, head hq, dim d)
  int out_f32;
  const void *q;
  int64_t q_st, q_sh;
  int n_rows;              // rows of q / out
  const int32_t *q_start;  // [B] first row of sequence b in q / out
  const int32_t *q_len;    // [B] query tokens of sequence b
  const int32_t *ctx;      // [B] tokens in the pools, the chunk included
  const int32_t *tables;
  int max_blocks;
  int Hkv, G, bs;
  int64_t n_blocks;
  float scale_log2;
  int sub_log2;      // rows per bulk copy box: gcd(block_size, keys per tile) = 1 << sub_log2
  int32_t *err;
  int n_seqs, qblocks;  // sequences, query blocks per sequence
  ScoreMod mod{};       // modified scores and masks (paged_prefill_mod.cu)
};

// 4-D bulk tensor copy (no multicast): box {64, 8, D / 64, rows / 8} of the
// grouped map at row group `grp`.
__device__ __forceinline__ void tma_load_4d(uint32_t dst, const void *tmap, int grp, uint32_t bar,
                                            uint64_t policy) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes.L2::cache_hint"
      " [%0], [%1, {%2, %2, %2, %3}], [%4], %5;" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(tmap)), "r"(0), "r"(grp), "r"(bar), "l"(policy)
      : "memory");
}

// Pool [rows][D] viewed as 4-D: (64 columns, 8 rows, D / 64 chunks, rows / 8
// groups) with strides (row D*2 B, chunk 128 B, group 8*D*2 B), box {64, 8,
// D / 64, box_rows / 8}, 128-byte swizzle: one copy brings box_rows whole rows
// in the grouped layout the MMA descriptors read.
inline int make_group_map(CUtensorMap *m, const void *base, int64_t rows, int D,
                          CUtensorMapDataType type, int box_rows) {
  auto fn = decode::encode_fn();
  if (!fn) return fail(MZ_ERR_CUDA, "cuTensorMapEncodeTiled is unavailable");
  cuuint64_t dims[4] = {64, 8, static_cast<cuuint64_t>(D / 64), static_cast<cuuint64_t>(rows / 8)};
  cuuint64_t strides[3] = {static_cast<cuuint64_t>(D) * 2, 128, static_cast<cuuint64_t>(D) * 16};
  cuuint32_t box[4] = {64, 8, static_cast<cuuint32_t>(D / 64),
                       static_cast<cuuint32_t>(box_rows / 8)};
  cuuint32_t es[4] = {1, 1, 1, 1};
  CUresult r = fn(m, type, 4, const_cast<void *>(base), dims, strides, box, es,
                  CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                  CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return fail(MZ_ERR_CUDA, "cuTensorMapEncodeTiled (grouped) failed (%d)", (int)r);
  return MZ_OK;
}

// max(a, b, c) in one instruction (three-input max.f32 of sm_100)
__device__ __forceinline__ float fmax3f(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

__device__ __forceinline__ void mbar_arrive(uint32_t bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}

// Checks and fills everything a launch needs; *empty where there is nothing to
// do.  Copy boxes have up to 2^tile_log2 rows.
inline int prepare(PParams *p, CUtensorMap *tk, CUtensorMap *tv, bool *empty, int tile_log2,
                   void *out, int32_t out_dtype, int64_t out_tok_stride, int64_t out_head_stride,
                   const void *q, int64_t q_tok_stride, int64_t q_head_stride, int32_t n_rows,
                   const int32_t *q_start, const int32_t *q_len, int32_t max_q_len,
                   const void *k_pool, const void *v_pool, const int32_t *block_tables,
                   int32_t max_blocks_per_seq, const int32_t *ctx_lens, int32_t n_seqs,
                   int32_t n_heads, int32_t n_kv_heads, int32_t head_dim, int32_t block_size,
                   int64_t n_blocks, float scale, int32_t dtype, int32_t *dev_err,
                   const char *fn) {
  if (dtype != MZ_DTYPE_F16 && dtype != MZ_DTYPE_BF16)
    return fail(MZ_ERR_UNSUPPORTED, "%s: dtype must be F16 or BF16", fn);
  if (out_dtype != dtype && out_dtype != MZ_DTYPE_F32)
    return fail(MZ_ERR_UNSUPPORTED, "%s: out_dtype must equal dtype or be F32", fn);
  if (head_dim != 64 && head_dim != 128)
    return fail(MZ_ERR_UNSUPPORTED, "%s: head_dim %d (supported: 64, 128)", fn, head_dim);
  if (block_size <= 0 || block_size % kTileTok)
    return fail(MZ_ERR_UNSUPPORTED, "%s: block_size %d is not a multiple of 16", fn, block_size);
  if (n_seqs < 0 || n_kv_heads <= 0 || n_heads <= 0 || n_heads % n_kv_heads || max_q_len < 0 ||
      max_blocks_per_seq <= 0 || n_blocks <= 0 || n_rows < 0)
    return fail(MZ_ERR_INVALID_ARG, "%s: bad sizes", fn);
  const int G = n_heads / n_kv_heads;
  if (kM % G)
    return fail(MZ_ERR_UNSUPPORTED, "%s: n_heads / n_kv_heads = %d does not divide %d", fn, G,
                kM);
  if (!std::isfinite(scale) || !(scale > 0.f))
    return fail(MZ_ERR_INVALID_ARG, "%s: scale must be finite and positive", fn);
  *empty = n_seqs == 0 || max_q_len == 0;
  if (*empty) return MZ_OK;
  if (!out || !q || !q_start || !q_len || !k_pool || !v_pool || !block_tables || !ctx_lens)
    return fail(MZ_ERR_INVALID_ARG, "%s: null pointer", fn);
  // rows move as 16-byte vectors: q and out 16-byte aligned, strides whole vectors
  const int oe = out_dtype == MZ_DTYPE_F32 ? 4 : 8;
  if (!aligned(k_pool, 16) || !aligned(v_pool, 16) || !aligned(q, 16) || (q_tok_stride % 8) ||
      (q_head_stride % 8) || !aligned(out, 16) || (out_tok_stride % oe) || (out_head_stride % oe))
    return fail(MZ_ERR_ALIGNMENT,
                "%s: pools, q and out need 16-byte alignment and strides of whole 16-byte "
                "vectors", fn);
  const int64_t rows_total = n_blocks * n_kv_heads * block_size;
  if (rows_total >= (int64_t(1) << 31))
    return fail(MZ_ERR_UNSUPPORTED, "%s: pool has >= 2^31 rows", fn);

  const bool bf16 = dtype == MZ_DTYPE_BF16;
  const auto type = bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  int sub_log2 = 4;  // rows per copy box: gcd(block_size, keys per tile)
  while (sub_log2 < tile_log2 && block_size % (1 << (sub_log2 + 1)) == 0) ++sub_log2;
  if (int rc = make_group_map(tk, k_pool, rows_total, head_dim, type, 1 << sub_log2)) return rc;
  if (int rc = make_group_map(tv, v_pool, rows_total, head_dim, type, 1 << sub_log2)) return rc;

  p->out = out;
  p->o_st = out_tok_stride;
  p->o_sh = out_head_stride;
  p->out_f32 = out_dtype == MZ_DTYPE_F32;
  p->q = q;
  p->q_st = q_tok_stride;
  p->q_sh = q_head_stride;
  p->n_rows = n_rows;
  p->q_start = q_start;
  p->q_len = q_len;
  p->ctx = ctx_lens;
  p->tables = block_tables;
  p->max_blocks = max_blocks_per_seq;
  p->Hkv = n_kv_heads;
  p->G = G;
  p->bs = block_size;
  p->n_blocks = n_blocks;
  p->scale_log2 = static_cast<float>(static_cast<double>(scale) * 1.4426950408889634);
  p->sub_log2 = sub_log2;
  p->err = dev_err;
  if (n_seqs > 65535 || n_kv_heads > 65535)
    return fail(MZ_ERR_UNSUPPORTED, "%s: grid too large", fn);
  const int tpc = kM / G;
  p->n_seqs = n_seqs;
  p->qblocks = (max_q_len - 1) / tpc + 1;  // (any bound up to 2^31 - 1 is taken)
  return MZ_OK;
}

}  // namespace prefill
}  // namespace mz
