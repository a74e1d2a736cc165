// Step metadata on the GPU: block tables, slot maps and positions from the
// requests' lengths, one launch.
//
// With q_b new tokens of sequence b behind ctx_b cached ones, held_b blocks in
// its table already and blocks of bs tokens:
//   need_b  = max(0, ceil((ctx_b + q_b) / bs) - held_b)
//   start_b = q_0 + ... + q_{b-1},  base_b = need_0 + ... + need_{b-1}
//   table[b][held_b + i] = new_ids[base_b + i],            0 <= i < need_b
//   row start_b + i:  pos = ctx_b + i,
//                     slot = table[b][pos / bs] * bs + pos % bs
//
// Latency bounds it: a step of 64 sequences moves a few KB, one of 131072 rows
// 1.6 MB.  So one launch and no second pass: every CTA scans all sequences'
// lengths itself (they sit in L2; 2048 sequences per round of two block
// barriers) instead of waiting for another CTA's prefix, keeps the starts that
// fall into its own 1024 rows, and spreads them over its rows by a running
// maximum.  A new block's id is taken from new_ids where its first row is, so
// no thread reads a table entry that another one writes.  Blocks of a power of
// two are divided by shifts.  64 sequences of one token: 4.5 us between launches
// of a graph; 256 prompts of 131072 rows: 5.1 us (7.4 and 7.6 us with divisions
// and the rows' lengths read again).
#include "common.cuh"

namespace mz {
namespace plan {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kRowsPerThread = 4;
constexpr int kRows = kThreads * kRowsPerThread;  // rows of a CTA
constexpr int kSeqs = 8;                          // most sequences per thread and round

struct PlanParams {
  int32_t *tables;
  int max_blocks;
  const int32_t *ctx, *q, *held, *new_ids;
  int n_new, B, n_rows, bs;
  int bs_log2;  // -1: no power of two
  int64_t n_blocks;
  int32_t *q_start, *positions;
  int64_t *slots;
  int32_t *lengths, *held_out, *n_used;
  int32_t *err;
};

__device__ __forceinline__ int blocks_below(const PlanParams &p, int tokens) {
  return p.bs_log2 >= 0 ? tokens >> p.bs_log2 : tokens / p.bs;
}

// A sequence's checked lengths: q = 0 where they do not fit its table.
struct Seq {
  int ctx, q, held, need;
  bool ok;
};

__device__ __forceinline__ Seq read_seq(const PlanParams &p, int b) {
  Seq s;
  s.ctx = p.ctx[b];
  s.q = p.q[b];
  const int64_t end = (int64_t)s.ctx + s.q;
  s.ok = s.ctx >= 0 && s.q >= 0 && end <= (int64_t)p.max_blocks * p.bs;  // < 2^31
  // ceil(x / bs) = floor((x - 1) / bs) + 1 for x > 0: no sum that could overflow
  s.held = p.held ? p.held[b] : s.ctx > 0 ? blocks_below(p, s.ctx - 1) + 1 : 0;
  s.ok = s.ok && s.held >= 0 && s.held <= p.max_blocks && (int64_t)s.held * p.bs >= s.ctx;
  if (!s.ok) s.q = 0;
  s.need = s.ok && end > 0 ? max(0, blocks_below(p, static_cast<int>(end) - 1) + 1 - s.held) : 0;
  return s;
}

__global__ void __launch_bounds__(kThreads) paged_plan_kernel(const PlanParams p) {
  __shared__ int64_t w_rows[kWarps];
  __shared__ int w_need[kWarps];
  __shared__ int w_mark[kWarps];
  // at a sequence's first row here: the sequence, the position of row 0 of this
  // block in it, its blocks, and where its new ones start
  __shared__ int s_seq[kRows], s_pos[kRows], s_held[kRows], s_base[kRows];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t r0 = (int64_t)blockIdx.x * kRows;
  const int64_t r1 = min(r0 + kRows, (int64_t)p.n_rows);
  for (int i = threadIdx.x; i < kRows; i += kThreads) s_seq[i] = -1;
  __syncthreads();

  int64_t rows0 = 0;  // rows and new blocks of the sequences of earlier rounds
  int need0 = 0;
  const int per = min(kSeqs, (p.B + kThreads - 1) / kThreads);  // sequences per thread
  for (int b0 = 0; b0 < p.B; b0 += kThreads * per) {
    Seq s[kSeqs];
    int64_t rows = 0;
    int need = 0;
    const int bt = b0 + threadIdx.x * per;
#pragma unroll
    for (int k = 0; k < kSeqs; ++k) {
      s[k] = Seq{0, 0, 0, 0, true};
      if (k < per && bt + k < p.B) s[k] = read_seq(p, bt + k);
      rows += s[k].q;
      need += s[k].need;
    }
    int64_t ir = rows;
    int in = need;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t y = __shfl_up_sync(0xffffffffu, ir, o);
      const int z = __shfl_up_sync(0xffffffffu, in, o);
      if (lane >= o) {
        ir += y;
        in += z;
      }
    }
    if (lane == 31) {
      w_rows[warp] = ir;
      w_need[warp] = in;
    }
    __syncthreads();
    int64_t start = rows0 + ir - rows;
    int base = need0 + in - need;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      if (w < warp) {
        start += w_rows[w];
        base += w_need[w];
      }
      rows0 += w_rows[w];
      need0 += w_need[w];
    }
#pragma unroll
    for (int k = 0; k < kSeqs; ++k) {
      const int b = bt + k;
      if (k >= per) break;
      if (b < p.B) {
        const bool fits = start + s[k].q <= p.n_rows;
        const int got = min(s[k].need, max(0, p.n_new - base));
        if (blockIdx.x == 0) {
          p.q_start[b] = static_cast<int>(min(start, (int64_t)p.n_rows));
          p.lengths[b] = s[k].ctx + (fits ? s[k].q : 0);
          p.held_out[b] = s[k].held + (fits ? got : 0);
          if (!s[k].ok) dev_error(p.err, MZ_DEVERR_CONTEXT);
          if (!fits) dev_error(p.err, MZ_DEVERR_ROWS);
          if (got < s[k].need) dev_error(p.err, MZ_DEVERR_BLOCKS);
        }
        // a sequence that does not fit keeps its rows at slot -1
        if (fits && s[k].q > 0 && start < r1 && start + s[k].q > r0) {
          const int i = static_cast<int>(max(start, r0) - r0);
          s_seq[i] = b;
          s_pos[i] = s[k].ctx + static_cast<int>(r0 - start);
          s_held[i] = s[k].held;
          s_base[i] = base;
        } else if (!fits && start >= r0 && start < r1) {
          s_seq[static_cast<int>(start - r0)] = p.B;  // no sequence from here on
        }
      }
      start += s[k].q;
      base += s[k].need;
    }
    __syncthreads();
  }
  if (blockIdx.x == 0 && threadIdx.x == 0) *p.n_used = need0;
  // rows behind the last sequence
  if (threadIdx.x == 0 && rows0 >= r0 && rows0 < r1) s_seq[static_cast<int>(rows0 - r0)] = p.B;
  __syncthreads();

  // running maximum of the marks' places: a row's sequence is the last mark at or before it
  const int i0 = threadIdx.x * kRowsPerThread;
  int mark[kRowsPerThread], m = -1;
#pragma unroll
  for (int k = 0; k < kRowsPerThread; ++k) {
    if (s_seq[i0 + k] >= 0) m = i0 + k;
    mark[k] = m;
  }
  int im = m;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, im, o);
    if (lane >= o) im = max(im, y);
  }
  if (lane == 31) w_mark[warp] = im;
  const int before = __shfl_up_sync(0xffffffffu, im, 1);
  __syncthreads();
  int prev = lane ? before : -1;
  for (int w = 0; w < warp; ++w) prev = max(prev, w_mark[w]);

#pragma unroll
  for (int k = 0; k < kRowsPerThread; ++k) {
    const int i = i0 + k;
    if (r0 + i >= r1) break;
    const int at = max(mark[k], prev);
    int pos = 0;
    int64_t slot = -1;
    const int b = at >= 0 ? s_seq[at] : p.B;
    if (b < p.B) {
      const int held = s_held[at];
      pos = s_pos[at] + i;
      const int j = blocks_below(p, pos), in = pos - j * p.bs;
      int32_t id = -1;
      if (j >= held) {
        const int64_t x = (int64_t)s_base[at] + (j - held);
        if (x < p.n_new) id = p.new_ids[x];
        if (id < 0 || id >= p.n_blocks) {
          if (x < p.n_new) dev_error(p.err, MZ_DEVERR_BLOCK_ID);
          id = -1;
        }
        // the row at a new block's first place in the range writes its entry
        if (in == 0) p.tables[(int64_t)b * p.max_blocks + j] = id;
      } else {
        id = p.tables[(int64_t)b * p.max_blocks + j];
        if (id < 0 || id >= p.n_blocks) {
          dev_error(p.err, MZ_DEVERR_BLOCK_ID);
          id = -1;
        }
      }
      if (id >= 0) slot = (int64_t)id * p.bs + in;
    }
    p.positions[r0 + i] = pos;
    p.slots[r0 + i] = slot;
  }
}

}  // namespace plan
}  // namespace mz

using namespace mz;

extern "C" int mz_paged_plan(int32_t *block_tables, int32_t max_blocks_per_seq,
                             const int32_t *ctx_lens, const int32_t *q_lens, const int32_t *held,
                             const int32_t *new_ids, int32_t n_new_ids, int32_t n_seqs,
                             int32_t n_rows, int32_t block_size, int64_t n_blocks,
                             int32_t *q_start, int32_t *positions, int64_t *slots,
                             int32_t *lengths, int32_t *held_out, int32_t *n_used,
                             int32_t *dev_err, mz_stream_t stream) {
  const char *fn = "mz_paged_plan";
  if (n_seqs < 0 || n_rows < 0 || n_new_ids < 0 || block_size <= 0 || max_blocks_per_seq <= 0 ||
      n_blocks <= 0)
    return fail(MZ_ERR_INVALID_ARG, "%s: bad sizes", fn);
  if ((int64_t)max_blocks_per_seq * block_size >= (int64_t(1) << 31) ||
      (int64_t)n_seqs * max_blocks_per_seq >= (int64_t(1) << 31))
    return fail(MZ_ERR_UNSUPPORTED, "%s: tables span 2^31 or more tokens or entries", fn);
  if (!n_used || (n_rows > 0 && (!positions || !slots)) || (n_new_ids > 0 && !new_ids) ||
      (n_seqs > 0 && (!block_tables || !ctx_lens || !q_lens || !q_start || !lengths || !held_out)))
    return fail(MZ_ERR_INVALID_ARG, "%s: null pointer", fn);
  plan::PlanParams p;
  p.tables = block_tables;
  p.max_blocks = max_blocks_per_seq;
  p.ctx = ctx_lens;
  p.q = q_lens;
  p.held = held;
  p.new_ids = new_ids;
  p.n_new = n_new_ids;
  p.B = n_seqs;
  p.n_rows = n_rows;
  p.bs = block_size;
  p.bs_log2 = -1;
  for (int i = 0; i < 31; ++i)
    if (block_size == 1 << i) p.bs_log2 = i;
  p.n_blocks = n_blocks;
  p.q_start = q_start;
  p.positions = positions;
  p.slots = slots;
  p.lengths = lengths;
  p.held_out = held_out;
  p.n_used = n_used;
  p.err = dev_err;
  const int64_t grid = n_rows > 0 ? ((int64_t)n_rows + plan::kRows - 1) / plan::kRows : 1;
  plan::paged_plan_kernel<<<static_cast<unsigned>(grid), plan::kThreads, 0,
                            static_cast<cudaStream_t>(stream)>>>(p);
  MZ_CHECK_LAUNCH(fn);
  return MZ_OK;
}
