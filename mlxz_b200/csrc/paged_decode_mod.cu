// Paged decode attention with modified scores and masks (score_mod.cuh) for
// sm_100a: single tokens, drafted runs, the fused append.
//
// Scheduling, copies and the merge of split pairs are those of the unmodified
// decode (decode_common.cuh): persistent warps over flat lists of 16-token
// tiles, here of the tiles that the mask leaves, a ring of bulk tensor copies
// per warp.
//
// HBM bound by its bytes (4 rows: 2 flop a byte), but with modified scores the
// chain of dependent instructions per tile is what a warp waits for: eight warps
// an SM at 490 instructions a tile ran at 67-77 % of HBM.  So tokens are the
// M = 16 side of mma.sync m16n8k16 here and the grouped query rows the N = 8 side,
// once (up to 8 rows) or twice (up to 16):  S^T = K.Q^T takes 8 products of
// D = 128 where rows as M take 16, O^T += V^T.P^T 8 (16 with bf16's low part of P)
// where they take 16 (32), and Q and O half the registers.  P^T comes from the
// scores' accumulator layout by an 8 x 8 transpose in the warp (movmatrix).
// Measured: a capped, windowed step of 64 sequences up to 8192 tokens (32 / 8
// heads of 128, bf16, 815 MB) 143 us, 5.7 TB/s, 0.88 of the copy rate, 165 us with
// rows as M; four drafted tokens of 32 sequences (16 rows, 462 MB) 103 us, 4.5
// TB/s.  Not kept: three blocks an SM for 16 rows (registers spill, 137 us).
#include <type_traits>

#include "decode_common.cuh"

namespace mz {
namespace decode {

constexpr float kRescaleLog2 = 8.f;

template <int D>
struct ModCfg {
  static constexpr int kStages = D == 64 ? 6 : 3;
  static constexpr int kTileBytes = kTileTok * D * 2;  // one of K or V
  static constexpr int kStageBytes = 2 * kTileBytes;   // K + V
  static constexpr int kSmemTiles = kWarps * kStages * kStageBytes;
  static constexpr int kSmemBars = kWarps * kStages * 8;
  static constexpr int kSmemUnits = kWarps * kUnitQ * static_cast<int>(sizeof(Unit));
  static constexpr int kSmemDefer = kWarps * kMaxDeferred * static_cast<int>(sizeof(Deferred));
  static constexpr int kSmemBytes = kSmemTiles + kSmemBars + kSmemUnits + kSmemDefer + 1024;
};

__device__ __forceinline__ void store_one(const Params &p, int64_t off, float x) {
  if (p.out_f32)
    static_cast<float *>(p.out)[off] = x;
  else if (p.q_bf16)
    static_cast<__nv_bfloat16 *>(p.out)[off] = __float2bfloat16_rn(x);
  else
    static_cast<__half *>(p.out)[off] = __float2half_rn(x);
}

// mma_16816 that the compiler may move: a product of registers alone.
template <bool BF16>
__device__ __forceinline__ void mma_free(float (&d)[4], const uint32_t (&a)[4], uint32_t b0,
                                         uint32_t b1) {
  if constexpr (BF16) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, "
        "{%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  } else {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, "
        "{%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
}

// RG: groups of 8 query rows.
template <int D, bool BF16, int RG>
__global__ void __launch_bounds__(kWarps * 32, 2)
    paged_decode_mod_kernel(const __grid_constant__ CUtensorMap tmK,
                            const __grid_constant__ CUtensorMap tmV, const ModParams p) {
  using C = ModCfg<D>;
  constexpr int S = C::kStages;
  constexpr int KS = D / 16;  // k-steps of K.Q^T, m-tiles of V^T.P^T
  // rows of the weighted merge (with 16 its registers cost the tile loop 3 %)
  constexpr int kMergeRows = RG == 1 ? 8 : 0;

  launch_dependents();
  extern __shared__ uint8_t smem_raw[];
  uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                              ~static_cast<uintptr_t>(1023));
  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const int W = gridDim.x * kWarps;
  const int wid = blockIdx.x * kWarps + warp;

  uint8_t *stages = smem + warp * S * C::kStageBytes;
  uint64_t *bars = reinterpret_cast<uint64_t *>(smem + C::kSmemTiles) + warp * S;
  Unit *uq = reinterpret_cast<Unit *>(smem + C::kSmemTiles + C::kSmemBars) + warp * kUnitQ;
  Deferred *dq = reinterpret_cast<Deferred *>(smem + C::kSmemTiles + C::kSmemBars + C::kSmemUnits) +
                 warp * kMaxDeferred;
  int nd = 0;  // merges this warp owns, run after its tile loop
  const uint32_t bar0 = smem_u32(bars);
  const uint32_t stage0 = smem_u32(stages);

  if (lane == 0) {
    for (int s = 0; s < S; ++s) mbar_init(bar0 + 8 * s, 1);
    fence_mbar_init();
  }
  __syncwarp();

  Sched sch;
  const bool any_work = sch.init(p, lane, wid, W, uq);  // no tiles: no counter is touched

  const uint64_t pol = l2_policy_evict_first();
  auto issue = [&](int s, const Cursor &c) {
    if (lane == 0) {
      const int t = own_tile(p, c.b, c.t, c.n, c.ctx);
      int32_t blk = p.tables[(int64_t)c.b * p.max_blocks + t / p.tpb];
      if (blk < 0 || blk >= p.n_blocks) {
        // the last tile is read even where no row sees it: any block will do then
        const MaskSpan m = mask_span(p, c.b, c.ctx);
        if (p.kn || t * kTileTok < m.head || (t + 1) * kTileTok > m.lo)
          dev_error(p.err, MZ_DEVERR_BLOCK_ID);
        blk = 0;
      }
      const int y = static_cast<int>(((int64_t)blk * p.Hkv + c.h) * p.bs + (t % p.tpb) * kTileTok);
      const uint32_t bar = bar0 + 8 * s;
      const uint32_t dk = stage0 + s * C::kStageBytes;
      mbar_arrive_expect_tx(bar, C::kStageBytes);
#pragma unroll
      for (int c2 = 0; c2 < D / 64; ++c2) {
        tma_load_2d(dk + c2 * 2048, &tmK, c2 * 64, y, bar, pol);
        tma_load_2d(dk + C::kTileBytes + c2 * 2048, &tmV, c2 * 64, y, bar, pol);
      }
    }
  };

  // ldmatrix geometry: K as A (rows = tokens), V^T as A (rows = dims, transposed)
  const int mi = lane >> 3, r8 = lane & 7;
  const int tokK = r8 + 8 * (mi & 1), subK = mi >> 1;
  const int tokV = r8 + 8 * (mi >> 1), subV = mi & 1;
  const int g = lane >> 2, cq = lane & 3;
  // this lane's scores: tokens g, g + 8 of the tile, query rows 8 x + 2 cq, + 1

  uint32_t qb[RG][KS][2];
  float oacc[RG][KS][4];  // dims 16 j + g, + 8; rows 8 x + 2 cq, + 1
  float m[RG][2], l[RG][2];
  MaskSpan span{};
  int skip = 0, p_min = 0, lo_max = 0;
  int pos[RG][2], lo[RG][2];
  float slope[RG][2];

  UnitReader ur;
  bool seg_first = true;

  // Until the launch ahead has completed (programmatic dependent launch) only
  // ctx, the mask's arrays, the tables and the pools are read.
  if (any_work) sch.template prefetch_static<S>(p, issue);
  wait_for_previous_grid();
  zero_empty_outputs<D>(p, wid, W, lane);
  if (!any_work) return;

  sch.template refill<S>(p, 0, issue);
  bool ring_idle = true;
  for (int i = 0; i < sch.issued; ++i) {
    const int s = i % S;
    if (ur.need_pop()) {
      ur.pop(uq);
      seg_first = true;
    }
    const Cursor &cc = ur.cc;

    if (seg_first || cc.t == 0) {
      // New piece: its mask, and the query rows as B fragments.
      seg_first = false;
      span = mask_span(p, cc.b, cc.ctx);
      skip = ntiles_of(cc.ctx) - cc.n;
      p_min = cc.ctx - p.n_q;
      // lower ends rise with the token where the window sets them
      const int first = p.mod.first ? max(0, p.mod.first[cc.b]) : 0;
      lo_max = p.mod.window > 0 ? max(first, cc.ctx - p.mod.window) : first;
#pragma unroll
      for (int x = 0; x < RG; ++x) {
#pragma unroll
        for (int y = 0; y < 2; ++y) {
          const int r = 8 * x + 2 * cq + y;
          m[x][y] = kNoMax;
          l[x][y] = 0.f;
          pos[x][y] = p_min + r / p.G;
          lo[x][y] = p.mod.window > 0 ? max(first, pos[x][y] - p.mod.window + 1) : first;
          slope[x][y] = p.mod.slopes && r < p.rows ? p.mod.slopes[cc.h * p.G + r % p.G] * kLog2e : 0.f;
        }
        const auto *q16 = static_cast<const uint16_t *>(p.q);
        const int r = 8 * x + g;
        const int64_t qo = r < p.rows ? row_offset(p.q_sb, p.q_st, p.q_sh, cc.b, cc.h, r, p.G) : -1;
#pragma unroll
        for (int j = 0; j < KS; ++j) {
          const int d = 16 * j + 2 * cq;
          qb[x][j][0] = qo >= 0 ? *reinterpret_cast<const uint32_t *>(q16 + qo + d) : 0u;
          qb[x][j][1] = qo >= 0 ? *reinterpret_cast<const uint32_t *>(q16 + qo + d + 8) : 0u;
          oacc[x][j][0] = oacc[x][j][1] = oacc[x][j][2] = oacc[x][j][3] = 0.f;
        }
      }
    }

    if (!wait_stage<S>(p, bar0, i, sch.issued, lane)) {
      ring_idle = false;
      break;
    }

    uint8_t *kt = stages + s * C::kStageBytes;
    uint8_t *vt = kt + C::kTileBytes;
    const uint32_t kb = stage0 + s * C::kStageBytes;
    const uint32_t vb = kb + C::kTileBytes;
    const int tile = cc.t >= ntiles_of(span.head) ? cc.t + skip : cc.t;  // own_tile
    const int key0 = tile * kTileTok;
    const bool last_tile = (cc.t == cc.n - 1);
    if (p.kn != nullptr && last_tile) {
      // Fused append: the sequence's new token is its last attended one.  Write
      // it to its pool slot and into the staged tile (which may predate it).
      const int at = cc.ctx - 1;
      constexpr int U = D / 8;  // 16-byte units per row
      if (lane < 2 * U) {
        const bool is_v = lane >= U;
        const int d = (lane - (is_v ? U : 0)) * 8;
        const uint16_t *src =
            (is_v ? p.vn : p.kn) + (int64_t)cc.b * p.kn_sb + (int64_t)cc.h * p.kn_sh + d;
        const uint4 val = *reinterpret_cast<const uint4 *>(src);
        *reinterpret_cast<uint4 *>((is_v ? vt : kt) + swz128(at & (kTileTok - 1), 2 * d)) = val;
        const int32_t blk = p.tables[(int64_t)cc.b * p.max_blocks + at / p.bs];
        if (blk >= 0 && blk < p.n_blocks) {
          uint16_t *dst = (is_v ? p.v_pool : p.k_pool) +
                          ((((int64_t)blk * p.Hkv + cc.h) * p.bs + at % p.bs) * D + d);
          *reinterpret_cast<uint4 *>(dst) = val;
        }
      }
      __syncwarp();
    }
    if (key0 + kTileTok > cc.ctx || (key0 < span.lo && key0 + kTileTok > span.head)) {
      // V of keys past the context (stale) and of keys that no row sees may be
      // anything: exact zeros, so that 0 * V stays 0.
      for (int e = lane; e < kTileTok * (D / 8); e += 32) {
        const int tok = e / (D / 8), d = (e % (D / 8)) * 8, key = key0 + tok;
        if (key >= cc.ctx || (key < span.lo && key >= span.head))
          *reinterpret_cast<uint4 *>(vt + swz128(tok, 2 * d)) = make_uint4(0, 0, 0, 0);
      }
      __syncwarp();
    }

    // S^T = K . Q^T : 16 tokens x rows, even and odd k-steps summed apart.
    float sacc[RG][2][4];
#pragma unroll
    for (int x = 0; x < RG; ++x)
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int e = 0; e < 4; ++e) sacc[x][h][e] = 0.f;
    // (four fragments' loads in flight before the products that use them)
#pragma unroll
    for (int j0 = 0; j0 < KS; j0 += 4) {
      uint32_t a[4][4];
#pragma unroll
      for (int j = 0; j < 4; ++j)
        ldsm_x4(kb + swz128(tokK, 2 * (16 * (j0 + j) + 8 * subK)), a[j][0], a[j][1], a[j][2], a[j][3]);
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int x = 0; x < RG; ++x)
          mma_free<BF16>(sacc[x][j & 1], a[j], qb[x][j0 + j][0], qb[x][j0 + j][1]);
    }
    uint32_t va[4][4];  // the first of V^T, loaded under the softmax
#pragma unroll
    for (int j = 0; j < 4; ++j)
      ldsm_x4_trans(vb + swz128(tokV, 2 * (16 * j + 8 * subV)), va[j][0], va[j][1], va[j][2], va[j][3]);

    // Scores in log2 units, masked; the online softmax of each row.
    const bool all_seen = (key0 >= lo_max && key0 + kTileTok - 1 <= p_min) ||
                          key0 + kTileTok <= span.prefix;
    bool need = false;
#pragma unroll
    for (int x = 0; x < RG; ++x) {
      float(&sc)[4] = sacc[x][0];  // tokens g, g + 8 (e >> 1) of rows 2 cq, + 1 (e & 1)
#pragma unroll
      for (int e = 0; e < 4; ++e) sc[e] += sacc[x][1][e];
      if (p.mod.z_scale == 0.f) {
#pragma unroll
        for (int e = 0; e < 4; ++e) sc[e] *= p.scale_log2;
      } else if (p.mod.cap_log2 <= kQuickCapLog2) {
#pragma unroll
        for (int e = 0; e < 4; ++e) sc[e] = cap_quick(p.mod, sc[e]);
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) sc[e] = p.mod.cap_log2 * tanh_mod(sc[e] * p.mod.z_scale);
      }
      if (p.mod.slopes) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float far = static_cast<float>(pos[x][e & 1] - (key0 + g + 8 * (e >> 1)));
          sc[e] = fmaf(-slope[x][e & 1], fabsf(far), sc[e]);
        }
      }
      if (!all_seen) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int key = key0 + g + 8 * (e >> 1);
          if (!(key < span.prefix ||
                (key <= pos[x][e & 1] && (key >= lo[x][e & 1] || key < p.mod.sink))))
            sc[e] = -INFINITY;
        }
      }
#pragma unroll
      for (int y = 0; y < 2; ++y)
        need |= fmaxf(sc[y], sc[2 + y]) > m[x][y] + kRescaleLog2;
    }
    // m moves, to the largest score so far, only where a row exceeds it by more
    // than 8: most tiles need no maximum across lanes
    if (__any_sync(0xffffffffu, need)) {
#pragma unroll
      for (int x = 0; x < RG; ++x) {
        float alpha[2];
#pragma unroll
        for (int y = 0; y < 2; ++y) {
          float mx = fmaxf(sacc[x][0][y], sacc[x][0][2 + y]);
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
          const float mn = fmaxf(m[x][y], mx);
          alpha[y] = fast_exp2(m[x][y] - mn);
          m[x][y] = mn;
          l[x][y] *= alpha[y];
        }
#pragma unroll
        for (int j = 0; j < KS; ++j) {
          oacc[x][j][0] *= alpha[0];
          oacc[x][j][1] *= alpha[1];
          oacc[x][j][2] *= alpha[0];
          oacc[x][j][3] *= alpha[1];
        }
      }
    }
    // P^T as B fragments: fp16 has 11 bits of P in one part, as in the unmodified
    // kernel (2^-11 of an output, an fp16 output's own rounding, seen in fp32 ones);
    // bf16's 8 are too few for its outputs, so its low part makes them 16
    uint32_t ph[RG][2], pl[RG][2];
#pragma unroll
    for (int x = 0; x < RG; ++x) {
      float(&sc)[4] = sacc[x][0];
#pragma unroll
      for (int e = 0; e < 4; ++e) sc[e] = fast_exp2(sc[e] - m[x][e & 1]);
      l[x][0] += sc[0] + sc[2];
      l[x][1] += sc[1] + sc[3];
      // tokens x rows -> rows x tokens, 8 tokens at a time
      float hi[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) hi[e] = round16<BF16>(sc[e]);
      ph[x][0] = movmatrix_trans(pack2<BF16>(hi[0], hi[1]));
      ph[x][1] = movmatrix_trans(pack2<BF16>(hi[2], hi[3]));
      if constexpr (BF16) {
        pl[x][0] = movmatrix_trans(pack2<BF16>(sc[0] - hi[0], sc[1] - hi[1]));
        pl[x][1] = movmatrix_trans(pack2<BF16>(sc[2] - hi[2], sc[3] - hi[3]));
      }
    }

    // O^T += V^T . P^T
#pragma unroll
    for (int j0 = 0; j0 < KS; j0 += 4) {
      if (j0 > 0) {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          ldsm_x4_trans(vb + swz128(tokV, 2 * (16 * (j0 + j) + 8 * subV)), va[j][0], va[j][1],
                        va[j][2], va[j][3]);
      }
#pragma unroll
      for (int part = 0; part < (BF16 ? 2 : 1); ++part)
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
          for (int x = 0; x < RG; ++x)
            mma_free<BF16>(oacc[x][j0 + j], va[j], part ? pl[x][0] : ph[x][0],
                           part ? pl[x][1] : ph[x][1]);
    }

    // Piece end: last tile of the pair, or last tile of the unit.
    if (last_tile || ur.left == 1) {
      const int bh = cc.b * p.Hkv + cc.h;
      const int pbh = cc.pos - cc.t;  // flat index of tile 0 of this pair
      // units holding the pair's first and last piece (batch-invariant: the
      // pair's pieces are the consecutive units W + fp ...)
      const int uf = p.batch_invariant ? sch.W + ur.fp : sch.unit_of(pbh);
      const int ul = p.batch_invariant ? uf + ur.np - 1 : sch.unit_of(pbh + cc.n - 1);
      const bool whole = uf == ul;
      const int64_t slot = (int64_t)ur.unit + bh;
#pragma unroll
      for (int x = 0; x < RG; ++x)
#pragma unroll
        for (int y = 0; y < 2; ++y) {
          float L = l[x][y];
          L += __shfl_xor_sync(0xffffffffu, L, 4);
          L += __shfl_xor_sync(0xffffffffu, L, 8);
          L += __shfl_xor_sync(0xffffffffu, L, 16);
          const int r = 8 * x + 2 * cq + y;
          if (r < p.rows) {
            if (whole) {
              const float inv = row_inverse(L);
              const int64_t o = row_offset(p.o_sb, p.o_st, p.o_sh, cc.b, cc.h, r, p.G) + g;
#pragma unroll
              for (int j = 0; j < KS; ++j) {
                store_one(p, o + 16 * j, oacc[x][j][y] * inv);
                store_one(p, o + 16 * j + 8, oacc[x][j][2 + y] * inv);
              }
            } else {
              float *pr = p.part + (slot * p.rows + r) * D + g;
#pragma unroll
              for (int j = 0; j < KS; ++j) {
                pr[16 * j] = oacc[x][j][y];
                pr[16 * j + 8] = oacc[x][j][2 + y];
              }
              if (g == 0)
                *reinterpret_cast<float2 *>(p.ml + (slot * p.rows + r) * 2) =
                    make_float2(m[x][y], L);
            }
          }
        }
      if (!whole)
        arrive_or_defer<D, false, kMergeRows>(p, cc, bh, uf, ul - uf + 1, lane, dq, nd,
                                              S * C::kStageBytes);
      seg_first = true;  // the next tile starts a new piece
    }

    __syncwarp();
    --ur.left;
    advance(ur.cc, p);
    sch.template refill<S>(p, i + 1, issue);
  }
  run_deferred<D, false, kMergeRows>(p, dq, nd, stages, S * C::kStageBytes, ring_idle, lane);
}

template <int D, bool BF16, int RG>
static int launch_rows(cudaLaunchConfig_t &cfg, const CUtensorMap &tk, const CUtensorMap &tv,
                       const ModParams &p, const char *fn) {
  static DeviceOnce once;
  if (int rc = smem_optin(paged_decode_mod_kernel<D, BF16, RG>, ModCfg<D>::kSmemBytes, once,
                          "setting the modified-score kernel's shared memory"))
    return rc;
  cfg.dynamicSmemBytes = ModCfg<D>::kSmemBytes;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, paged_decode_mod_kernel<D, BF16, RG>, tk, tv, p);
  if (e != cudaSuccess) return cuda_fail(e, fn);
  MZ_CHECK_LAUNCH(fn);
  return MZ_OK;
}

int launch_mod(cudaLaunchConfig_t &cfg, int D, bool bf16, const CUtensorMap &tk,
               const CUtensorMap &tv, const ModParams &p, const char *fn) {
#define MZ_MOD(D_, BF_)                                                      \
  return p.rows <= 8 ? launch_rows<D_, BF_, 1>(cfg, tk, tv, p, fn)           \
                     : launch_rows<D_, BF_, 2>(cfg, tk, tv, p, fn)
  if (D == 128) {
    if (bf16) MZ_MOD(128, true);
    MZ_MOD(128, false);
  }
  if (bf16) MZ_MOD(64, true);
  MZ_MOD(64, false);
#undef MZ_MOD
}

}  // namespace decode
}  // namespace mz
