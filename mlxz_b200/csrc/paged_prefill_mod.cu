// Chunked prefill attention over paged KV with modified scores and masks
// (score_mod.cuh), on the tcgen05 tensor cores.
//
// Work comes as items -- (sequence, KV head, block of 128 query rows; row m is
// token q0 + m / G, query head h * G + m % G) -- of which one CTA per SM takes
// two at a time, as two streams that share nothing but the tensor core.  A
// stream is six warps:
//   four softmax warps   one thread per query row: scores of a 64-key tile from
//                        TMEM to registers, masks and modifications, the
//                        running maximum and sum, P back to TMEM, the epilogue
//   a copy warp          streams 64-key K and V tiles through the block table
//                        (bulk tensor copies of gcd(block_size, 64)-row boxes,
//                        128-byte swizzle, no multicast), two slots of each
//   an MMA warp          S_{i+1} = Q.K_{i+1}^T (SS, M = 128, N = 64) into S buffer
//                        (i + 1) % 2, then O += P_i.V_i (TS, N = D)
// What bounds it: a softmax warp's 64 scores a thread take about 1500 cycles a
// tile, in dependent phases (TMEM load, maximum, exponentials, conversion, TMEM
// store), of which the special-function unit needs 512; two warps of two streams
// share a scheduler, and two streams without any order between them fill each
// other's gaps: 4096 new tokens at 16384 with a window of 4096 (32 / 8 heads of
// 128, bf16) take 353 us, 780 TFLOP/s, against 418 us for one stream of 128-key
// tiles whose halves meet at every maximum (409 us launched back to back, where
// the power limit lowers the clock).  The tensor core is the next bound: two tiles
// with P in two bf16 parts take it 2 (8 x 48 + 8 x 64) = 1792 cycles, S at N = 64
// being held up by its operands' shared memory reads, of the 1970 measured.  A cap
// of 50 on 512 new tokens at 3584 of eight sequences: 479 us, 538 TFLOP/s; short
// prompts are bound by an item's latency.  Not kept, each right but slower on
// that case: P.V issued apart from S, by a second warp (533 us) or by one warp
// that polls both streams' barriers (425 us with S first, 482 us with P.V first);
// the MMAs issued by one lane's branch instead of an elected lane (414 us);
// exponentials against the running maximum as it is while the tile's is found,
// redone where it moves (365 us).  P in one bf16 part would give 310 us.
//
// TMEM columns of stream s: O at 128 s, S buffers at 256 + 128 s, 64 each.  P
// takes its scores' place: hi parts in the first 32 columns, lo in the last.
// The running maximum only moves when a row exceeds it by more than 8 (log2
// units); O is rescaled in TMEM on those tiles alone.  An item reads the key
// tiles of the keys that every row sees (prefix and sinks) and those from its
// first row's lowest key on; local tile t is tile t or t + skip of the sequence.
//
// Few items over long contexts would leave SMs idle: then a cluster of up to eight
// CTAs takes one item, its 2 to 16 streams a range of the key tiles each, and they
// join their (m, l, O) through the cluster's shared memory: each stream leaves its
// O there and writes the joined columns that are its share.  No workspace, no
// second launch.  With a cap of 50, 32 tokens at 16384 take 44 us (338 us as whole
// items), 64 at 2000 22 us (51), 32 at 600 19 us (22); 64 behind a window of 4096
// 25 us (73).  Joining costs 3 to 5 us, so clusters
// are no larger than gives two tiles a part of the longest item that the table or
// the window allows (parts of four made 32 tokens at 600 22 us and 1 at 400 17
// instead of 14 us); a shorter item's parts may have one tile, or none.  Not kept: the
// odd last item of a CTA among many shared by its two streams in the same way
// (window 350 against 360 us, but documents 112 against 105, a cap on 256 items of
// 8192 keys 252 against 232: a stream alone runs faster than one of two).
//
// Every wait is bounded; one that gives up sets MZ_DEVERR_TIMEOUT and the abort
// flag, every role leaves its loop, the issuing warps wait (bounded) for their
// copies and MMAs in flight, and the TMEM is freed.
#include <algorithm>
#include <climits>

#include "prefill_common.cuh"
#include "tcgen05.cuh"

namespace mz {
namespace prefill {
namespace two {

constexpr int kN = 64;       // keys per tile
constexpr int kSlots = 2;    // K slots, V slots and S buffers of a stream
constexpr int kStreams = 2;
constexpr int kSoftWarps = 4;  // per stream
constexpr int kPartTiles = 2;  // tiles of a split item's part at least
constexpr int kThreads = 32 * kStreams * (kSoftWarps + 2);
constexpr uint32_t kTmemCols = 512;
constexpr float kRescaleLog2 = 8.f;
static_assert(kSlots == 2, "phases below count tiles by pairs");

template <int D>
struct Cfg {
  // K / V tile: 8 groups of 8 keys, each group the D / 64 column chunks of 8
  // rows x 128 bytes (one swizzle atom per chunk)
  static constexpr int kGroup = 8 * D * 2;
  static constexpr int kTile = (kN / 8) * kGroup;
  static constexpr int kQ = (D / 64) * kM * 128;  // 128 rows x D, chunk-major
  static constexpr int kStream = kQ + 2 * kSlots * kTile;
  static constexpr int kBar = kStreams * kStream;
  // a split item's O (fp32, column by column) in place of Q and K, (m, l) behind it
  static constexpr int kMl = kQ + kSlots * kTile;
  static_assert(kMl == kM * D * 4, "O takes the place of Q and the K slots");
  static constexpr int kSmemBytes = kBar + 256 + 1024;
};

// barriers of a stream (8 bytes each)
constexpr int kBarKFull = 0, kBarVFull = 2, kBarSFull = 4, kBarPFull = 6, kBarPvDone = 8,
              kBarQReady = 10, kBarDrain = 11, kNumBars = 12;
static_assert(8 * kStreams * kNumBars + 8 <= 256, "barrier area");

struct Item {
  int b, h, q0, start, q_hi, kv_len, ntiles;
  // keys [0, prefix) are seen by all rows, [0, head) these and the sinks; lo: no
  // row's other keys start below it; head_tiles, skip: tiles of the head, tiles
  // left out behind them
  int prefix, head, lo, head_tiles, skip;
  int t0;  // first tile of this part, in a split item
  template <bool SPLIT>
  __device__ __forceinline__ int own(int t) const {
    if constexpr (SPLIT) t += t0;
    return t < head_tiles ? t : t + skip;
  }
  // Part i of n, which may be empty.
  __device__ __forceinline__ void cut(int i, int n) {
    const int per = (ntiles + n - 1) / n;
    t0 = min(i * per, ntiles);
    ntiles = min(per, ntiles - t0);
  }
};

// Where a stream's search for its next item stands: sequence b's first item is
// `base`.
struct Walk {
  int b = 0, base = 0;
};

// Item e, whole warps.  Items are the query blocks that the sequences have, a
// sequence's last (longest) ones first and its KV heads in turn, so that
// neighbours in time share K/V through L2 without all reading the same tiles at
// once, and a batch of ragged or empty chunks costs no empty items.  False: none
// is left (*end), or the item's sequence is in error.
__device__ __forceinline__ bool item_at(const PParams &p, Walk &w, int e, Item &it, bool *end) {
  const int lane = threadIdx.x & 31, tpc = kM / p.G;
  int n = 0, blocks = 0;
  for (;; w.b += 32) {
    if (w.b >= p.n_seqs) {
      *end = true;
      return false;
    }
    const int b = w.b + lane;
    n = b < p.n_seqs ? max(0, p.q_len[b]) : 0;
    // (a length near 2^31 must not overflow: its sequence is reported below)
    blocks = min((min(n, INT_MAX - kM) + tpc - 1) / tpc, p.qblocks);
    const int mine = blocks * p.Hkv;
    int incl = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += y;
    }
    const unsigned found = __ballot_sync(0xffffffffu, w.base + incl > e);
    const int from = found ? __ffs(found) - 1 : 31;
    w.base += __shfl_sync(0xffffffffu, found ? incl - mine : incl, from);
    if (found) {
      w.b += from;
      n = __shfl_sync(0xffffffffu, n, from);
      blocks = __shfl_sync(0xffffffffu, blocks, from);
      break;
    }
  }
  it.b = w.b;
  const int r = e - w.base, jr = r / p.Hkv;
  it.h = r - jr * p.Hkv;
  it.q0 = (blocks - 1 - jr) * tpc;
  const int ctx = p.ctx[it.b];
  if (ctx < n || ctx > (int64_t)p.max_blocks * p.bs) {
    if (lane == 0) dev_error(p.err, MZ_DEVERR_CONTEXT);
    return false;
  }
  const int row0 = p.q_start[it.b];
  if (row0 < 0 || (int64_t)row0 + n > p.n_rows) {
    if (lane == 0) dev_error(p.err, MZ_DEVERR_ROWS);
    return false;
  }
  it.start = ctx - n;
  it.q_hi = min(it.q0 + tpc, n);
  const int last = it.start + it.q_hi - 1;  // last causal key of the item
  it.prefix = p.mod.prefix ? max(0, min(p.mod.prefix[it.b], ctx)) : 0;
  it.head = max(it.prefix, p.mod.sink);
  it.lo = 0;
  if (p.mod.first) {
    int lo = INT_MAX;
    for (int t = it.q0 + lane; t < it.q_hi; t += 32) lo = min(lo, p.mod.first[row0 + t]);
    it.lo = max(0, __reduce_min_sync(0xffffffffu, lo));
  }
  if (p.mod.window > 0) it.lo = max(it.lo, it.start + it.q0 - p.mod.window + 1);
  it.kv_len = max(last + 1, it.prefix);
  it.head_tiles = min((it.head + kN - 1) / kN, last / kN + 1);
  // the tile of lo, or the last causal one, is read in any case
  it.skip = max(0, min(it.lo, last) / kN - it.head_tiles);
  it.ntiles = (it.kv_len + kN - 1) / kN - it.skip;
  it.t0 = 0;
  return true;
}

// mbar_wait_bounded that also ends, every so many polls, when a role gave up.
__device__ __forceinline__ bool wait_bounded(uint32_t bar, uint32_t phase,
                                             const volatile int *abort_flag) {
  uint64_t t0 = 0;
  for (uint32_t it = 1;; ++it) {
    if (mbar_try_wait(bar, phase)) return true;
    if ((it & 255u) == 0u) {
      if (*abort_flag) return false;
      const uint64_t now = global_timer_ns();
      if (t0 == 0)
        t0 = now;
      else if (now - t0 > kTimeoutNs)
        return false;
    }
  }
}

__device__ __forceinline__ int cluster_rank() {
  uint32_t r;
  asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return static_cast<int>(r);
}
__device__ __forceinline__ int cluster_size() {
  uint32_t n;
  asm("mov.u32 %0, %%cluster_nctarank;" : "=r"(n));
  return static_cast<int>(n);
}
// All threads of the cluster; what was written before it is seen after it.
__device__ __forceinline__ void cluster_sync() {
  asm volatile(
      "barrier.cluster.arrive.release;\n\t"
      "barrier.cluster.wait.acquire;" ::: "memory");
}
// Shared memory of the cluster's CTA `rank`, at this CTA's address `at`.
__device__ __forceinline__ uint32_t peer_smem(uint32_t at, int rank) {
  uint32_t a;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(at), "r"(rank));
  return a;
}
__device__ __forceinline__ float ld_peer(uint32_t at) {
  float x;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(x) : "r"(at) : "memory");
  return x;
}
__device__ __forceinline__ float2 ld_peer2(uint32_t at) {
  float2 x;
  asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(x.x), "=f"(x.y) : "r"(at) : "memory");
  return x;
}

// Columns [part, part + 1) * D / N of a split item's row, joined from its N parts
// (part j: stream j & 1 of rank j >> 1, at the same place in every CTA; `cta`:
// stream 0's memory here) and written to out at `ob`.
template <int D, bool BF16, int N>
__device__ __forceinline__ void join_parts(const PParams &p, uint32_t cta, int row, int part,
                                           int64_t ob) {
  using C = Cfg<D>;
  constexpr int kCols = D / N, kStep = N < 8 ? 32 / N : 4;  // 32 loads in flight, or more
  static_assert(kCols % kStep == 0, "whole steps");
  uint32_t from[N];
  float2 ml[N];
#pragma unroll
  for (int j = 0; j < N; ++j) {
    from[j] = peer_smem(cta + (j & 1) * C::kStream, j >> 1);
    ml[j] = ld_peer2(from[j] + C::kMl + 8 * row);
  }
  // weights of the parts; none for those without a key of the row, or any tile
  float w[N], top = kNoMax, sum = 0.f;
#pragma unroll
  for (int j = 0; j < N; ++j) top = ml[j].y != 0.f ? fmaxf(top, ml[j].x) : top;
#pragma unroll
  for (int j = 0; j < N; ++j) {
    w[j] = ml[j].y != 0.f ? fast_exp2(ml[j].x - top) : 0.f;
    sum = fmaf(w[j], ml[j].y, sum);
  }
  const float inv = decode::row_inverse(sum);
#pragma unroll 1
  for (int c = part * kCols; c < (part + 1) * kCols; c += kStep) {
    float x[N][kStep], acc[kStep];
#pragma unroll
    for (int j = 0; j < N; ++j)
#pragma unroll
      for (int i = 0; i < kStep; ++i) x[j][i] = ld_peer(from[j] + 4 * ((c + i) * kM + row));
#pragma unroll
    for (int i = 0; i < kStep; ++i) {
      acc[i] = 0.f;
      // (a part of no weight may have left nothing there)
#pragma unroll
      for (int j = 0; j < N; ++j) acc[i] = w[j] != 0.f ? fmaf(w[j], x[j][i], acc[i]) : acc[i];
      acc[i] *= inv;
    }
#pragma unroll
    for (int i = 0; i < kStep; i += 4) {
      if (p.out_f32)
        *reinterpret_cast<float4 *>(static_cast<float *>(p.out) + ob + c + i) =
            make_float4(acc[i], acc[i + 1], acc[i + 2], acc[i + 3]);
      else
        *reinterpret_cast<uint2 *>(static_cast<uint16_t *>(p.out) + ob + c + i) = make_uint2(
            pack2<BF16>(acc[i], acc[i + 1]), pack2<BF16>(acc[i + 2], acc[i + 3]));
    }
  }
}

// MODE 1: masks; 2: masks and the bias by distance; 3: these and capped scores.
// From 2 on the scores take their final form, in log2 units, in registers.
// SPLIT: the cluster's streams share one item, item (block / cluster size).
template <int D, bool BF16, int MODE, bool SPLIT>
__global__ void __launch_bounds__(kThreads, 1)
    paged_prefill_mod_kernel(const __grid_constant__ CUtensorMap tmK,
                             const __grid_constant__ CUtensorMap tmV, const PParams p) {
  using C = Cfg<D>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t *smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  // warps 0-3 and 4-7: softmax of stream 0 and 1; 8, 10: copies; 9, 11: MMAs
  const int st = warp < 8 ? warp >> 2 : (warp - 8) >> 1;
  const bool copies = warp >= 8 && !(warp & 1), mmas = warp >= 8 && (warp & 1);
  const uint32_t sbase = smem_u32(smem) + st * C::kStream;
  const uint32_t qs = sbase;
  auto kst = [&](int s) { return sbase + C::kQ + s * C::kTile; };
  auto vst = [&](int s) { return sbase + C::kQ + (kSlots + s) * C::kTile; };
  const uint32_t bars = smem_u32(smem) + C::kBar + 8 * st * kNumBars;
  auto bar = [&](int i) { return bars + 8 * i; };
  uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(smem + C::kBar + 8 * kStreams * kNumBars);
  volatile int *abort_flag = reinterpret_cast<volatile int *>(tmem_slot + 1);

  if (copies && lane == 0) {
    for (int s = 0; s < kSlots; ++s) {
      mbar_init(bar(kBarKFull + s), 1);
      mbar_init(bar(kBarVFull + s), 1);
      mbar_init(bar(kBarSFull + s), 1);
      mbar_init(bar(kBarPFull + s), kSoftWarps);
      mbar_init(bar(kBarPvDone + s), 1);
    }
    mbar_init(bar(kBarQReady), kSoftWarps);
    mbar_init(bar(kBarDrain), 1);
    if (st == 0) *abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == 9) tc::tmem_alloc(smem_u32(tmem_slot), kTmemCols);
  tc::fence_before_sync();
  __syncthreads();
  tc::fence_after_sync();
  const uint32_t tmem = *tmem_slot;

  // Items go to the streams in turn, all first streams before all second ones:
  // in the last round they spread over the SMs.
  const int ranks = SPLIT ? cluster_size() : 1;
  const int e0 = SPLIT ? blockIdx.x / ranks : st * gridDim.x + blockIdx.x;
  const int e_step = kStreams * gridDim.x;
  Walk walk;
  auto next_item = [&](int &e, Item &it) {
    for (bool end = false;; e += e_step) {
      if (SPLIT && e != e0) return false;
      if (item_at(p, walk, e, it, &end)) return true;
      if (end) return false;
    }
  };
  auto give_up = [&]() {
    dev_error(p.err, MZ_DEVERR_TIMEOUT);
    *abort_flag = 1;
  };
  // whole warp: phase `phase` of barrier b; false when it (or another role) gave up
  auto wait = [&](int b, int phase) {
    if (__all_sync(0xffffffffu, wait_bounded(bar(b), phase & 1, abort_flag))) return true;
    if (lane == 0) give_up();
    return false;
  };
  // two barriers that are mostly both there: one round trip for the two polls
  auto wait2 = [&](int b0, int phase0, int b1, int phase1) {
    const bool x = mbar_try_wait(bar(b0), phase0 & 1), y = mbar_try_wait(bar(b1), phase1 & 1);
    if (__all_sync(0xffffffffu, x && y)) return true;
    return wait(b0, phase0) && wait(b1, phase1);
  };

  Item it;
  int g = 0;  // tiles of this stream so far: slot g % 2, barrier phase g / 2
  int e = e0;
  bool have = next_item(e, it), ok = true;
  const bool found = have;
  const int parts = kStreams * ranks, part = SPLIT ? kStreams * cluster_rank() + st : 0;
  if (SPLIT && have) {
    it.cut(part, parts);
    have = it.ntiles > 0;
  }
  float m_part = kNoMax, l_part = 0.f;  // a split item's

  if (copies) {
    // ---------------- copies: K of tile t, then V of tile t - 1 ----------------
    const uint64_t pol = l2_policy_evict_last();
    const int sub = 1 << p.sub_log2, nst_log2 = 6 - p.sub_log2, nst = 1 << nst_log2;
    const int per = 32 >> nst_log2;  // tiles whose boxes a warp's lanes cover
    int k_issued = 0, v_issued = 0;
    for (; ok && have; e += e_step, have = next_item(e, it)) {
      // lane l holds box l % nst of tile per * x + l / nst; block ids are loaded
      // one such set ahead of their use.  Sets end behind the last tile: the tile
      // next to it stands for all of those, whose keys could pass 2^31.
      auto box_key = [&](int x) {
        const int t = min(per * x + (lane >> nst_log2), it.ntiles);
        return it.template own<SPLIT>(t) * kN + (lane & (nst - 1)) * sub;
      };
      auto ids = [&](int x) -> int32_t {
        const int t = box_key(x);
        return t < it.kv_len ? p.tables[(int64_t)it.b * p.max_blocks + t / p.bs] : 0;
      };
      auto rows = [&](int x, int32_t blk) -> int {
        const int t = box_key(x);
        if (t >= it.kv_len) return 0;
        if (blk < 0 || blk >= p.n_blocks) {
          // a box that no row sees may have lost its block: any block will do
          if (t < it.head || t + sub > it.lo) dev_error(p.err, MZ_DEVERR_BLOCK_ID);
          blk = 0;
        }
        return static_cast<int>(((int64_t)blk * p.Hkv + it.h) * p.bs + t % p.bs);
      };
      auto load = [&](const CUtensorMap *tm, uint32_t dst, uint32_t fbar, int t, int y) {
        const int nsub = min(nst, (it.kv_len - it.template own<SPLIT>(t) * kN + sub - 1) >> p.sub_log2);
        if (lane == 0)
          mbar_arrive_expect_tx(fbar, static_cast<uint32_t>(nsub * sub * D * 2));
        __syncwarp();
        if (lane < nsub) tma_load_4d(dst + lane * (sub / 8) * C::kGroup, tm, y >> 3, fbar, pol);
      };
      int y_prev = 0, y_cur = rows(0, ids(0));
      int32_t id_next = ids(1);
      for (int t = 0; t <= it.ntiles; ++t) {
        if (t > 0 && t % per == 0) {
          y_prev = y_cur;
          y_cur = rows(t / per, id_next);
          id_next = ids(t / per + 1);
        }
        if (t < it.ntiles) {
          const int gt = g + t, s = gt & 1;
          const int y = __shfl_sync(0xffffffffu, y_cur, ((t % per) << nst_log2) + (lane & (nst - 1)));
          // the slot is free once S of tile gt - 2 is computed
          if (gt >= kSlots && !wait(kBarSFull + s, (gt - kSlots) >> 1)) {
            ok = false;
            break;
          }
          load(&tmK, kst(s), bar(kBarKFull + s), t, y);
          k_issued = gt + 1;
        }
        if (t > 0) {
          const int u = t - 1, gu = g + u, s = gu & 1;
          const int y = __shfl_sync(0xffffffffu, u / per == t / per ? y_cur : y_prev,
                                    ((u % per) << nst_log2) + (lane & (nst - 1)));
          // free once P.V of tile gu - 2 is
          if (gu >= kSlots && !wait(kBarPvDone + s, (gu - kSlots) >> 1)) {
            ok = false;
            break;
          }
          load(&tmV, vst(s), bar(kBarVFull + s), u, y);
          v_issued = gu + 1;
        }
      }
      g += it.ntiles;
    }
    // copies still in flight land before the CTA leaves
    if (lane == 0) {
      for (int j = max(0, k_issued - kSlots); j < k_issued; ++j)
        (void)mbar_wait_bounded(bar(kBarKFull + (j & 1)), (j >> 1) & 1, kTimeoutNs);
      for (int j = max(0, v_issued - kSlots); j < v_issued; ++j)
        (void)mbar_wait_bounded(bar(kBarVFull + (j & 1)), (j >> 1) & 1, kTimeoutNs);
    }
    __syncwarp();
  } else if (mmas) {
    // ---------------- MMA issue (whole warp, one elected lane issues) ----------------
    constexpr uint32_t idS = tc::idesc_f16(BF16, kM, kN, false);
    constexpr uint32_t idPV = tc::idesc_f16(BF16, kM, D, true);
    const uint32_t tm = __shfl_sync(0xffffffffu, tmem, 0);
    const uint32_t o_col = tm + 128 * st, s_col = tm + 256 + 128 * st;
    auto issue_s = [&](int j) -> bool {
      const int s = j & 1;
      // K is there; the buffer is free once the P.V that read its P is computed
      if (j < kSlots ? !wait(kBarKFull + s, 0)
                     : !wait2(kBarPvDone + s, (j - kSlots) >> 1, kBarKFull + s, j >> 1))
        return false;
      tc::fence_after_sync();
#pragma unroll
      for (int k = 0; k < D / 16; ++k) {
        const uint32_t ko = (k & 3) * 32;  // 16-column step inside the chunk's atom
        tc::mma_ss_elect(s_col + kN * s, tc::smem_desc_sw128(qs + (k >> 2) * (kM * 128) + ko, 16, 1024),
                         tc::smem_desc_sw128(kst(s) + (k >> 2) * 1024 + ko, 16, C::kGroup), idS,
                         k > 0);
      }
      tc::commit_elect(bar(kBarSFull + s));  // also frees K slot s
      return true;
    };
    for (int nit = 0; ok && have; e += e_step, have = next_item(e, it), ++nit) {
      if (!wait(kBarQReady, nit) || !issue_s(g)) {
        ok = false;
        break;
      }
      for (int i = 0; i < it.ntiles; ++i) {
        if (i + 1 < it.ntiles && !issue_s(g + i + 1)) {
          ok = false;
          break;
        }
        const int j = g + i, s = j & 1;
        // P of an item's first tile is written after the item before's O is read
        if (!wait2(kBarPFull + s, j >> 1, kBarVFull + s, j >> 1)) {
          ok = false;
          break;
        }
        tc::fence_after_sync();
#pragma unroll
        for (int kk = 0; kk < kN / 16; ++kk) {
          const uint32_t pa = s_col + kN * s + 8 * kk;
          const uint64_t dv = tc::smem_desc_sw128(vst(s) + kk * 2 * C::kGroup, 1024, C::kGroup);
          tc::mma_ts_elect(o_col, pa, dv, idPV, (i > 0 || kk > 0) ? 1u : 0u);
          if constexpr (BF16) tc::mma_ts_elect(o_col, pa + 32, dv, idPV, 1u);
        }
        tc::commit_elect(bar(kBarPvDone + s));  // also frees V slot s
      }
      g += it.ntiles;
    }
    // every MMA issued has completed before the TMEM is freed
    tc::commit_elect(bar(kBarDrain));
    (void)mbar_wait_bounded(bar(kBarDrain), 0, kTimeoutNs);
    __syncwarp();
  } else {
    // ---------------- softmax + epilogue ----------------
    const int row = threadIdx.x & (kM - 1);
    const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const uint32_t o_col = tmem + lanes + 128 * st, s_col = tmem + lanes + 256 + 128 * st;
    uint8_t *q_smem = smem + st * C::kStream, *v_smem = q_smem + C::kQ + kSlots * C::kTile;
    // this thread's row of an item: token (rows past the last token repeat it), head
    auto token = [&](const Item &x) { return min(x.q0 + row / p.G, x.q_hi - 1); };
    auto load_q = [&](const Item &x) {
      const int hq = x.h * p.G + row % p.G;
      const bool live = x.q0 + row / p.G < x.q_hi;
      const uint4 *src = reinterpret_cast<const uint4 *>(
          static_cast<const uint16_t *>(p.q) + (int64_t)(p.q_start[x.b] + token(x)) * p.q_st +
          (int64_t)hq * p.q_sh);
#pragma unroll
      for (int u = 0; u < D / 8; ++u) {
        const uint4 v = live ? src[u] : make_uint4(0, 0, 0, 0);
        const int c = u >> 3, uu = u & 7;
        *reinterpret_cast<uint4 *>(q_smem + c * (kM * 128) + row * 128 + ((uu ^ (row & 7)) << 4)) = v;
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(bar(kBarQReady));
    };
    if (have) load_q(it);
    while (ok && have) {
      const int tok = token(it), hq = it.h * p.G + row % p.G;
      const bool live = it.q0 + row / p.G < it.q_hi;
      const int pos = it.start + tok;
      int lo = p.mod.first ? max(0, p.mod.first[p.q_start[it.b] + tok]) : 0;
      if (p.mod.window > 0) lo = max(lo, pos - p.mod.window + 1);
      const int head = max(it.prefix, min(p.mod.sink, pos + 1));
      const float slope = MODE > 1 && p.mod.slopes ? p.mod.slopes[hq] * kLog2e : 0.f;
      float m_used = kNoMax, l = 0.f;
      Item nx;
      int e2 = e + e_step;
      bool have2 = false;
      for (int i = 0; i < it.ntiles; ++i) {
        const int j = g + i, s = j & 1, tile = it.template own<SPLIT>(i);
        if (!wait(kBarSFull + s, j >> 1)) {
          ok = false;
          break;
        }
        tc::fence_after_sync();
        const uint32_t scol = s_col + kN * s;
        float sv[kN];
        {
          uint32_t r[2][32];
          tc::ld32(scol, r[0]);
          tc::ld32(scol + 32, r[1]);
          tc::wait_ld();
#pragma unroll
          for (int x = 0; x < kN; ++x) sv[x] = __uint_as_float(r[x >> 5][x & 31]);
        }
        const int key0 = tile * kN;
        // whether the tile crosses a border of what the row sees, and which of its
        // keys are hidden then
        const bool edge = !((key0 >= lo && key0 + kN - 1 <= pos) || key0 + kN <= head);
        auto hidden = [&](int x) {
          const int key = key0 + x;
          return key >= head && (key > pos || key < lo);
        };
        float top = 0.f;  // MODE 3: no score of the tile is above it
        if constexpr (MODE > 2) {
          float big = fmax3f(fabsf(sv[0]), fabsf(sv[1]), 0.f);
#pragma unroll
          for (int x = 2; x < kN; x += 2) big = fmax3f(big, fabsf(sv[x]), fabsf(sv[x + 1]));
          bool small = __all_sync(0xffffffffu, big <= p.mod.poly_range);
          if (!small) {
            // sixteen scores at a time in TMEM: little code for what few tiles need.
            // Hidden keys may be anything: they must not choose the form.
            big = 0.f;
#pragma unroll 1
            for (int c = 0; c < kN / 16; ++c) {
              uint32_t r[16];
              tc::ld16(scol + 16 * c, r);
              tc::wait_ld();
#pragma unroll
              for (int x = 0; x < 16; ++x) {
                if (edge && hidden(16 * c + x)) r[x] = 0u;
                big = fmaxf(big, fabsf(__uint_as_float(r[x])));
              }
              tc::st16(scol + 16 * c, r);
            }
            tc::wait_st();
            small = __all_sync(0xffffffffu, big <= p.mod.poly_range);
            if (!small) {
#pragma unroll 1
              for (int c = 0; c < kN / 16; ++c) {
                uint32_t r[16];
                tc::ld16(scol + 16 * c, r);
                tc::wait_ld();
#pragma unroll
                for (int x = 0; x < 16; ++x) {
                  const float v = __uint_as_float(r[x]);
                  float y = cap_quick(p.mod, v);
                  // its error grows with the cap: above 1000 for large scores alone
                  if (p.mod.cap_log2 > kQuickCapLog2 && fabsf(v) <= p.mod.poly_range)
                    y = cap_poly(p.mod, v);
                  r[x] = __float_as_uint(y);
                }
                tc::st16(scol + 16 * c, r);
              }
              tc::wait_st();
            }
            uint32_t r[2][32];
            tc::ld32(scol, r[0]);
            tc::ld32(scol + 32, r[1]);
            tc::wait_ld();
#pragma unroll
            for (int x = 0; x < kN; ++x) sv[x] = __uint_as_float(r[x >> 5][x & 31]);
          }
          top = p.mod.cap_log2;
          if (small) {
            top = cap_poly(p.mod, big);
            const uint64_t c0 = f2_pack(p.mod.poly[0], p.mod.poly[0]),
                           c1 = f2_pack(p.mod.poly[1], p.mod.poly[1]),
                           c2 = f2_pack(p.mod.poly[2], p.mod.poly[2]),
                           c3 = f2_pack(p.mod.poly[3], p.mod.poly[3]);
#pragma unroll
            for (int x = 0; x < kN; x += 2) {
              const uint64_t v = f2_pack(sv[x], sv[x + 1]), w = f2_mul(v, v);
              const uint64_t y = f2_fma(f2_fma(f2_fma(w, c3, c2), w, c1), w, c0);
              f2_unpack(f2_mul(y, v), sv[x], sv[x + 1]);
            }
          }
          // (slopes below 0 raise scores with the distance)
          top += fmaxf(0.f, -slope) * fmaxf(fabsf(static_cast<float>(key0 - pos)),
                                            fabsf(static_cast<float>(key0 + kN - 1 - pos)));
        }
        if constexpr (MODE > 1) {
          const float far = static_cast<float>(key0 - pos);
          const float sc = MODE > 2 ? 1.f : p.scale_log2;
          if (key0 + kN - 1 <= pos) {
            const uint64_t s2 = f2_pack(slope, slope), sc2 = f2_pack(sc, sc);
            const float b0 = slope * far;
            const uint64_t b2 = f2_pack(b0, b0);
#pragma unroll
            for (int x = 0; x < kN; x += 2) {
              const uint64_t d = f2_fma(s2, f2_pack(static_cast<float>(x), static_cast<float>(x + 1)), b2);
              const uint64_t v = f2_pack(sv[x], sv[x + 1]);
              f2_unpack(MODE > 2 ? f2_add(v, d) : f2_fma(v, sc2, d), sv[x], sv[x + 1]);
            }
          } else {
#pragma unroll
            for (int x = 0; x < kN; ++x)
              sv[x] = fmaf(-slope, fabsf(far + static_cast<float>(x)), MODE > 2 ? sv[x] : sv[x] * sc);
          }
        }
        if (edge) {
#pragma unroll
          for (int x = 0; x < kN; ++x)
            if (hidden(x)) sv[x] = -INFINITY;
        }
        // the tile's maximum, in four independent chains of three-input maxima; with
        // a cap only where the bound on it exceeds m by more than 8
        bool need = false;
        float m_new = m_used, alpha = 1.f;
        if (MODE < 3 || __any_sync(0xffffffffu, top > m_used + kRescaleLog2)) {
          float m4[4];
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            float m = fmax3f(sv[k], sv[k + 4], sv[k + 8]);
#pragma unroll
            for (int t = 3; t + 1 < kN / 4; t += 2)
              m = fmax3f(m, sv[k + 4 * t], sv[k + 4 * (t + 1)]);
            m4[k] = fmaxf(m, sv[k + kN - 4]);
          }
          float mx = fmax3f(m4[0], m4[1], fmaxf(m4[2], m4[3]));
          if constexpr (MODE < 2) mx *= p.scale_log2;  // scale > 0
          need = mx > m_used + kRescaleLog2;
          m_new = need ? mx : m_used;
          alpha = need ? fast_exp2(m_used - m_new) : 1.f;
        }
        if (i > 0 && __any_sync(0xffffffffu, need)) {
          // O holds P.V up to tile i - 1: S_i was issued after P.V of tile i - 2
          if (!wait(kBarPvDone + ((j - 1) & 1), (j - 1) >> 1)) {
            ok = false;
            break;
          }
          tc::fence_after_sync();
#pragma unroll 1
          for (int c = 0; c < D / 32; ++c) {
            uint32_t r[32];
            tc::ld32(o_col + 32 * c, r);
            tc::wait_ld();
#pragma unroll
            for (int x = 0; x < 32; ++x) r[x] = __float_as_uint(__uint_as_float(r[x]) * alpha);
            tc::st32(o_col + 32 * c, r);
          }
          tc::wait_st();
        }
        m_used = m_new;
        const uint64_t sc2 = f2_pack(p.scale_log2, p.scale_log2), nm2 = f2_pack(-m_used, -m_used);
        uint64_t l2[4] = {0ull, 0ull, 0ull, 0ull};
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          uint32_t hi[16], lo16[16];
#pragma unroll
          for (int w = 0; w < 16; ++w) {
            const uint64_t s2 = f2_pack(sv[32 * c + 2 * w], sv[32 * c + 2 * w + 1]);
            float xa, xe;
            f2_unpack(MODE < 2 ? f2_fma(s2, sc2, nm2) : f2_add(s2, nm2), xa, xe);
            const float a = fast_exp2(xa), z = fast_exp2(xe);
            const uint64_t az = f2_pack(a, z);
            l2[w & 3] = f2_add(l2[w & 3], az);
            hi[w] = pack2<BF16>(a, z);  // fp16 has 11 bits of P in one part, bf16 16 in two
            if constexpr (BF16) {
              // the rest of P, so that P.V carries 16 bits of it
              float ra, rz;
              f2_unpack(f2_sub(az, f2_pack(__uint_as_float(hi[w] << 16),
                                           __uint_as_float(hi[w] & 0xffff0000u))),
                        ra, rz);
              lo16[w] = pack2<BF16>(ra, rz);
            }
          }
          tc::st16(scol + 16 * c, hi);
          if constexpr (BF16) tc::st16(scol + 32 + 16 * c, lo16);
        }
        float l8[8];
#pragma unroll
        for (int k = 0; k < 4; ++k) f2_unpack(l2[k], l8[2 * k], l8[2 * k + 1]);
        l = l * alpha + (((l8[0] + l8[1]) + (l8[2] + l8[3])) + ((l8[4] + l8[5]) + (l8[6] + l8[7])));
        const int nvalid = it.kv_len - key0;
        const bool hole = key0 < it.lo && key0 + kN > it.head;
        if (nvalid < kN || hole) {
          // V of keys past kv_len (stale) and of keys that no row sees may be
          // anything, and 0 * NaN is not 0: they become exact zeros
          if (!wait(kBarVFull + s, j >> 1)) {
            ok = false;
            break;
          }
          for (int x = row; x < kN * (D / 8); x += kM) {
            const int r = x / (D / 8), u = x % (D / 8), key = key0 + r;
            if (key < it.kv_len && (key < it.head || key >= it.lo)) continue;
            const int c = u >> 3, uu = u & 7;
            *reinterpret_cast<uint4 *>(v_smem + s * C::kTile + (r >> 3) * C::kGroup + c * 1024 +
                                       (r & 7) * 128 + ((uu ^ (r & 7)) << 4)) =
                make_uint4(0, 0, 0, 0);
          }
          fence_proxy_async_smem();
        }
        tc::wait_st();
        tc::fence_before_sync();
        __syncwarp();
        if (lane == 0) mbar_arrive(bar(kBarPFull + s));
        if (i + 1 == it.ntiles) {
          // every S of the item is computed: the next item's Q takes its place,
          // so that its first S is computed while this one's O is written out
          have2 = next_item(e2, nx);
          if (have2) load_q(nx);
        }
      }
      if (!ok) break;
      const int jl = g + it.ntiles - 1;
      if (!wait(kBarPvDone + (jl & 1), jl >> 1)) {
        ok = false;
        break;
      }
      tc::fence_after_sync();
      if constexpr (SPLIT) {
        m_part = m_used;
        l_part = l;
        break;
      }
      const float inv = decode::row_inverse(l);
      const int64_t ob = (int64_t)(p.q_start[it.b] + tok) * p.o_st + (int64_t)hq * p.o_sh;
#pragma unroll
      for (int c = 0; c < D / 32; ++c) {
        uint32_t r[32];
        tc::ld32(o_col + 32 * c, r);
        tc::wait_ld();
        if (live) {
          if (p.out_f32) {
            float4 *dst = reinterpret_cast<float4 *>(static_cast<float *>(p.out) + ob + 32 * c);
#pragma unroll
            for (int x = 0; x < 8; ++x)
              dst[x] = make_float4(__uint_as_float(r[4 * x]) * inv, __uint_as_float(r[4 * x + 1]) * inv,
                                   __uint_as_float(r[4 * x + 2]) * inv,
                                   __uint_as_float(r[4 * x + 3]) * inv);
          } else {
            uint4 *dst = reinterpret_cast<uint4 *>(static_cast<uint16_t *>(p.out) + ob + 32 * c);
#pragma unroll
            for (int x = 0; x < 4; ++x)
              dst[x] = make_uint4(pack2<BF16>(__uint_as_float(r[8 * x]) * inv,
                                              __uint_as_float(r[8 * x + 1]) * inv),
                                  pack2<BF16>(__uint_as_float(r[8 * x + 2]) * inv,
                                              __uint_as_float(r[8 * x + 3]) * inv),
                                  pack2<BF16>(__uint_as_float(r[8 * x + 4]) * inv,
                                              __uint_as_float(r[8 * x + 5]) * inv),
                                  pack2<BF16>(__uint_as_float(r[8 * x + 6]) * inv,
                                              __uint_as_float(r[8 * x + 7]) * inv));
          }
        }
      }
      // O has been read: ordered before the next item's first P, which its first
      // P.V waits for
      tc::fence_before_sync();
      g += it.ntiles;
      it = nx;
      e = e2;
      have = have2;
    }
  }

  if constexpr (SPLIT) {
    // Every role comes here, also one that gave up: the barriers end.
    const int row = threadIdx.x & (kM - 1);
    if (warp < 8 && found && ok) {
      if (have) {
        // this stream's copies and products are all complete: O takes the place
        // of its Q and K, neighbouring rows side by side
        float *o = reinterpret_cast<float *>(smem + st * C::kStream) + row;
        const uint32_t o_col = tmem + (static_cast<uint32_t>((warp & 3) * 32) << 16) + 128 * st;
#pragma unroll 1
        for (int c = 0; c < D / 32; ++c) {
          uint32_t r[32];
          tc::ld32(o_col + 32 * c, r);
          tc::wait_ld();
#pragma unroll
          for (int x = 0; x < 32; ++x) o[(32 * c + x) * kM] = __uint_as_float(r[x]);
        }
      }
      *reinterpret_cast<float2 *>(smem + st * C::kStream + C::kMl + 8 * row) =
          make_float2(m_part, l_part);
    }
    cluster_sync();
    if (warp < 8 && found && ok && it.q0 + row / p.G < it.q_hi) {
      const int64_t ob = (int64_t)(p.q_start[it.b] + it.q0 + row / p.G) * p.o_st +
                         (int64_t)(it.h * p.G + row % p.G) * p.o_sh;
      const uint32_t cta = sbase - st * C::kStream;  // stream 0
      if (parts == 2) join_parts<D, BF16, 2>(p, cta, row, part, ob);
      else if (parts == 4) join_parts<D, BF16, 4>(p, cta, row, part, ob);
      else if (parts == 8) join_parts<D, BF16, 8>(p, cta, row, part, ob);
      else join_parts<D, BF16, 16>(p, cta, row, part, ob);
    }
    cluster_sync();  // no CTA leaves while another one reads from it
  }

  tc::fence_before_sync();
  __syncthreads();
  if (warp == 9) {
    tc::fence_after_sync();
    tc::tmem_dealloc(tmem, kTmemCols);
  }
}

template <int D, bool BF16, int MODE, bool SPLIT>
int smem_attr() {
  static DeviceOnce once;
  return smem_optin(paged_prefill_mod_kernel<D, BF16, MODE, SPLIT>, Cfg<D>::kSmemBytes, once,
                    "mz_paged_prefill_mod: shared memory attribute");
}

inline cudaLaunchAttribute cluster_of(int x) {
  cudaLaunchAttribute at{};
  at.id = cudaLaunchAttributeClusterDimension;
  at.val.clusterDim.x = x;
  at.val.clusterDim.y = at.val.clusterDim.z = 1;
  return at;
}

// Clusters of X CTAs that fit the device at once (0: none).
template <int D, bool BF16, int MODE, int X>
int max_clusters(int *n) {
  static DeviceOnce once;
  return device_once(
      once,
      [](int *value) {
        cudaLaunchAttribute at = cluster_of(X);
        cudaLaunchConfig_t cfg{};
        cfg.gridDim = dim3(X);
        cfg.blockDim = dim3(kThreads);
        cfg.dynamicSmemBytes = Cfg<D>::kSmemBytes;
        cfg.attrs = &at;
        cfg.numAttrs = 1;
        return cudaOccupancyMaxActiveClusters(
            value, paged_prefill_mod_kernel<D, BF16, MODE, true>, &cfg);
      },
      n, "mz_paged_prefill_mod: cluster occupancy");
}

// `items` (sequence, head, query block) at most, of up to `tiles` key tiles.
template <int D, bool BF16, int MODE>
int launch(const CUtensorMap &tk, const CUtensorMap &tv, const PParams &p, int64_t items,
           int64_t tiles, int sms, cudaStream_t s) {
  // One item per cluster where all items fit the device at once, in the largest
  // clusters whose streams get kPartTiles tiles each; else whole items.
  int x = 0;
  if (items <= sms && tiles >= kStreams * kPartTiles) {
    if (int rc = smem_attr<D, BF16, MODE, true>()) return rc;
    int n2 = 0, n4 = 0, n8 = 0;
    if (int rc = max_clusters<D, BF16, MODE, 2>(&n2)) return rc;
    if (int rc = max_clusters<D, BF16, MODE, 4>(&n4)) return rc;
    if (int rc = max_clusters<D, BF16, MODE, 8>(&n8)) return rc;
    auto fits = [&](int n, int y) { return items <= n && tiles >= (int64_t)y * kStreams * kPartTiles; };
    x = fits(n8, 8) ? 8 : fits(n4, 4) ? 4 : fits(n2, 2) ? 2 : 1;
  } else if (int rc = smem_attr<D, BF16, MODE, false>()) {
    return rc;
  }
  cudaLaunchAttribute at = cluster_of(x);
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(x ? items * x : std::min<int64_t>(items, sms)));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = Cfg<D>::kSmemBytes;
  cfg.stream = s;
  cfg.attrs = &at;
  cfg.numAttrs = x > 1 ? 1 : 0;
  const cudaError_t e =
      x ? cudaLaunchKernelEx(&cfg, paged_prefill_mod_kernel<D, BF16, MODE, true>, tk, tv, p)
        : cudaLaunchKernelEx(&cfg, paged_prefill_mod_kernel<D, BF16, MODE, false>, tk, tv, p);
  if (e != cudaSuccess) return cuda_fail(e, "mz_paged_prefill_mod");
  return MZ_OK;
}

}  // namespace two
}  // namespace prefill
}  // namespace mz

using namespace mz;
using namespace mz::prefill;

extern "C" int mz_paged_prefill_mod(void *out, int32_t out_dtype, int64_t out_tok_stride,
                                    int64_t out_head_stride, const void *q, int64_t q_tok_stride,
                                    int64_t q_head_stride, int32_t n_rows, const int32_t *q_start,
                                    const int32_t *q_len, int32_t max_q_len, const void *k_pool,
                                    const void *v_pool, const int32_t *block_tables,
                                    int32_t max_blocks_per_seq, const int32_t *ctx_lens,
                                    int32_t n_seqs, int32_t n_heads, int32_t n_kv_heads,
                                    int32_t head_dim, int32_t block_size, int64_t n_blocks,
                                    float scale, const mz_score_mod *mod, int32_t dtype,
                                    int32_t *dev_err, mz_stream_t stream) {
  const char *fn = "mz_paged_prefill_mod";
  CUtensorMap tk, tv;
  PParams p;
  bool empty = false;
  if (int rc = make_score_mod(&p.mod, mod, scale, (int64_t)max_blocks_per_seq * block_size, fn))
    return rc;
  if (int rc = prepare(&p, &tk, &tv, &empty, 6, out, out_dtype, out_tok_stride, out_head_stride, q,
                       q_tok_stride, q_head_stride, n_rows, q_start, q_len, max_q_len, k_pool,
                       v_pool, block_tables, max_blocks_per_seq, ctx_lens, n_seqs, n_heads,
                       n_kv_heads, head_dim, block_size, n_blocks, scale, dtype, dev_err, fn))
    return rc;
  if (empty) return MZ_OK;
  const int64_t items = (int64_t)n_seqs * n_kv_heads * p.qblocks;
  const int sms = sm_count(current_device());
  if (sms <= 0) return fail(MZ_ERR_CUDA, "%s: cannot query the SM count", fn);
  if (items + two::kStreams * (int64_t)sms >= (int64_t(1) << 31))
    return fail(MZ_ERR_UNSUPPORTED, "%s: too many query blocks", fn);
  // key tiles of an item at most: of its table, or of what a window leaves
  const int tpc = kM / p.G;
  int64_t tiles = ((int64_t)max_blocks_per_seq * block_size + two::kN - 1) / two::kN;
  if (p.mod.window > 0 && !p.mod.prefix)
    tiles = std::min(tiles, ((int64_t)p.mod.window + tpc) / two::kN + 2 + p.mod.sink / two::kN);
  const bool bf16 = dtype == MZ_DTYPE_BF16;
  const int mode = p.mod.z_scale != 0.f ? 3 : p.mod.slopes ? 2 : 1;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  int rc = MZ_OK;
#define MZ_TWO(D_, BF_)                                                              \
  rc = mode == 1   ? two::launch<D_, BF_, 1>(tk, tv, p, items, tiles, sms, s)        \
       : mode == 2 ? two::launch<D_, BF_, 2>(tk, tv, p, items, tiles, sms, s)        \
                   : two::launch<D_, BF_, 3>(tk, tv, p, items, tiles, sms, s)
  if (head_dim == 128) {
    if (bf16) MZ_TWO(128, true); else MZ_TWO(128, false);
  } else {
    if (bf16) MZ_TWO(64, true); else MZ_TWO(64, false);
  }
#undef MZ_TWO
  if (rc) return rc;
  MZ_CHECK_LAUNCH(fn);
  return MZ_OK;
}
