// RMS norm of each query and key head, rotation by position, and the write of
// K and V to their cache slots, in one pass.
//
//   y   = x / sqrt(mean(x^2) + eps) * (w + w0)            (over one head; optional)
//   th_i = position[axis_i] * inv_freq_i                  0 <= i < rot_dim / 2
//   (a, b) -> (a cos th_i - b sin th_i, b cos th_i + a sin th_i)
// for the pairs (i, i + rot_dim / 2), or (2 i, 2 i + 1) when interleaved;
// dimensions from rot_dim on are not rotated.  Everything between the load and
// the store is fp32, rounded once.  The angle is formed in fp64 and brought to
// [-1, 1] half turns before it is rounded to fp32: a position of 10^6 leaves
// fp32 angles with 0.06 rad of error.
//
// HBM bound: every head is read once and written once.  A thread keeps one
// head's 16 dimensions -- two 16-byte vectors that hold whole pairs -- and goes
// over the block's tokens, so its weights stay in registers and P = 4, 8 or 16
// neighbouring lanes make a head's sum of squares by shuffles.  The tokens' sines
// and cosines are computed once per block into shared memory, behind the first
// loads.  What costs is latency at 24 warps an SM: more tokens' loads in registers
// cost more in occupancy than they hide, so one token's are, and the two behind it
// are only asked for into L2.  16384 tokens of 32 / 8 heads of 128, bf16, to the
// pools (403 MB): 76 us, 5.3 TB/s, 0.82 of the copy rate; 85 us without the L2
// requests, 91 us as a persistent grid, 90-115 us with a warp per token.
#include <type_traits>

#include "common.cuh"

namespace mz {
namespace rope {

constexpr int kMaxThreads = 384;
constexpr int kTokens = 8;     // most tokens of a block
constexpr int kMaxFreqs = 128;  // head_dim 256 / 2
constexpr int kMaxAxes = 4;

struct RopeParams {
  const void *q, *k, *v;
  int64_t q_ts, q_hs, k_ts, k_hs, v_ts, v_hs;
  void *q_out, *k_out;  // k_out null: K and V go to the pools
  int64_t qo_ts, qo_hs, ko_ts, ko_hs;
  void *k_pool, *v_pool;
  const int64_t *slots;
  int bs;
  int64_t n_slots;
  const int32_t *positions;
  int64_t pos_stride;
  int n_axes;
  const float *inv_freq;
  const int32_t *freq_axes;
  int rot;
  const void *q_weight, *k_weight;
  int w_dtype;
  float w_offset, eps;
  int norm;
  int n_tokens, Hq, Hkv, D;
  int heads, group;  // heads and tokens per block
  int32_t *err;
};

// Eight elements as they lie in memory: one 16-byte vector, or two for fp32.
template <typename T>
struct Raw8 {
  uint4 v[sizeof(T) / 2];
};

template <typename T>
__device__ __forceinline__ Raw8<T> fetch8(const T *src) {
  Raw8<T> r;
#pragma unroll
  for (int i = 0; i < static_cast<int>(sizeof(T) / 2); ++i)
    r.v[i] = reinterpret_cast<const uint4 *>(src)[i];
  return r;
}

// ... widened to fp32, neighbours packed for the two-wide fp32 instructions.
template <typename T>
__device__ __forceinline__ void widen8(const Raw8<T> &r, uint64_t (&x)[4]) {
  const uint32_t w[4] = {r.v[0].x, r.v[0].y, r.v[0].z, r.v[0].w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (sizeof(T) == 4) {
      const uint4 v = r.v[i >> 1];
      x[i] = (i & 1) ? f2_pack(__uint_as_float(v.z), __uint_as_float(v.w))
                     : f2_pack(__uint_as_float(v.x), __uint_as_float(v.y));
    } else if constexpr (std::is_same<T, __nv_bfloat16>::value) {
      x[i] = f2_pack(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xffff0000u));
    } else {
      const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&w[i]));
      x[i] = f2_pack(f.x, f.y);
    }
  }
}

template <typename T>
__device__ __forceinline__ Raw8<T> narrow8(const uint64_t (&x)[4]) {
  Raw8<T> r;
  float f[8];
#pragma unroll
  for (int i = 0; i < 4; ++i) f2_unpack(x[i], f[2 * i], f[2 * i + 1]);
  if constexpr (sizeof(T) == 4) {
    r.v[0] = make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]),
                        __float_as_uint(f[3]));
    r.v[1] = make_uint4(__float_as_uint(f[4]), __float_as_uint(f[5]), __float_as_uint(f[6]),
                        __float_as_uint(f[7]));
  } else {
    constexpr bool BF = std::is_same<T, __nv_bfloat16>::value;
    r.v[0] = make_uint4(pack2<BF>(f[0], f[1]), pack2<BF>(f[2], f[3]), pack2<BF>(f[4], f[5]),
                        pack2<BF>(f[6], f[7]));
  }
  return r;
}

template <typename T>
__device__ __forceinline__ void put8(T *dst, const Raw8<T> &r) {
#pragma unroll
  for (int i = 0; i < static_cast<int>(sizeof(T) / 2); ++i) reinterpret_cast<uint4 *>(dst)[i] = r.v[i];
}

template <typename T>
__device__ __forceinline__ void load8(const T *src, float (&x)[8]) {
  uint64_t y[4];
  widen8<T>(fetch8<T>(src), y);
#pragma unroll
  for (int i = 0; i < 4; ++i) f2_unpack(y[i], x[2 * i], x[2 * i + 1]);
}

// w + w0 at 8 dimensions; w of any of the three types, all ones when null.
__device__ __forceinline__ void load_weight(const void *w, int dtype, float w0, int at,
                                            float (&x)[8]) {
  if (!w) {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = 1.f;
    return;
  }
  if (dtype == MZ_DTYPE_F32)
    load8(static_cast<const float *>(w) + at, x);
  else if (dtype == MZ_DTYPE_BF16)
    load8(static_cast<const __nv_bfloat16 *>(w) + at, x);
  else
    load8(static_cast<const __half *>(w) + at, x);
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] += w0;
}

// Sum of 8 x 2 squares over the P lanes of a head, its norm's factor.
template <int P>
__device__ __forceinline__ float norm_factor(const uint64_t (&a)[4], const uint64_t (&b)[4],
                                             bool act, float inv_d, float eps) {
  uint64_t s2 = 0ull;
#pragma unroll
  for (int i = 0; i < 4; ++i) s2 = f2_fma(a[i], a[i], f2_fma(b[i], b[i], s2));
  float lo, hi;
  f2_unpack(s2, lo, hi);
  float ss = act ? lo + hi : 0.f;
#pragma unroll
  for (int o = 1; o < P; o <<= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
  return rsqrtf(fmaf(ss, inv_d, eps));
}

template <typename T, int P, bool INTER>
__global__ void __launch_bounds__(kMaxThreads, sizeof(T) == 4 ? 1 : 2)
    qk_norm_rope_kernel(const RopeParams p) {
  __shared__ __align__(16) float s_cos[kTokens][kMaxFreqs], s_sin[kTokens][kMaxFreqs];
  __shared__ int64_t s_row[kTokens];  // K / V pool row of head 0, -1: none
  const int64_t t0 = (int64_t)blockIdx.x * p.group;
  const int n_tok = static_cast<int>(min((int64_t)p.group, p.n_tokens - t0));
  const int half = p.rot / 2;

  // this thread's head and its two vectors of 8 dimensions
  const int h = blockIdx.y * p.heads + threadIdx.x / P, u = threadIdx.x % P;
  const int h1 = p.Hq, h2 = p.Hq + p.Hkv, n_heads = h2 + (p.k_out ? 0 : p.Hkv);
  const int kind = h < h1 ? 0 : h < h2 ? 1 : 2;  // q, k, v
  const bool act = threadIdx.x / P < p.heads && h < n_heads && 16 * u < p.D;
  const bool turns = kind < 2 && 16 * u < p.rot;
  const bool wide = 16 * u < p.rot && !INTER;  // the halves' vectors lie rot / 2 apart
  const int d0 = wide ? 8 * u : 16 * u;
  const int dd = wide ? half : 8;
  const int hk = kind == 0 ? h : kind == 1 ? h - h1 : h - h2;

  const T *src = static_cast<const T *>(kind == 0 ? p.q : kind == 1 ? p.k : p.v);
  const int64_t src_ts = kind == 0 ? p.q_ts : kind == 1 ? p.k_ts : p.v_ts;
  src += t0 * src_ts + hk * (kind == 0 ? p.q_hs : kind == 1 ? p.k_hs : p.v_hs) + d0;
  Raw8<T> ra{}, rb{};  // the next token's
  auto fetch = [&](int t) {
    if (act && t < n_tok) {
      ra = fetch8<T>(src + t * src_ts);
      rb = fetch8<T>(src + t * src_ts + dd);
    }
  };
  // ... and those behind it on their way into L2: lane u of a head asks for its
  // u-th 128-byte line
  constexpr int kAhead = 2;
  const bool lines = act && 128 * u < p.D * static_cast<int>(sizeof(T));
  auto ahead = [&](int t) {
    if (lines && t < n_tok)
      asm volatile("prefetch.global.L2 [%0];" ::"l"(
          reinterpret_cast<const char *>(src - d0 + t * src_ts) + 128 * u));
  };
  fetch(0);
#pragma unroll
  for (int t = 1; t <= kAhead; ++t) ahead(t);

  // sines and cosines of the block's tokens, and their slots
  for (int e = threadIdx.x; e < n_tok * half; e += blockDim.x) {
    const int t = e / half, f = e - t * half;
    int ax = p.freq_axes ? p.freq_axes[f] : 0;
    if (ax < 0 || ax >= p.n_axes) {
      dev_error(p.err, MZ_DEVERR_AXIS);
      ax = 0;
    }
    const double th = static_cast<double>(p.positions[ax * p.pos_stride + t0 + t]) *
                      static_cast<double>(p.inv_freq[f]);
    const double turn = th * 0.15915494309189533577;  // 1 / (2 pi)
    sincospif(static_cast<float>(2.0 * (turn - rint(turn))), &s_sin[t][f], &s_cos[t][f]);
  }
  if (!p.k_out && threadIdx.x < n_tok) {
    const int64_t slot = p.slots[t0 + threadIdx.x];
    int64_t row = -1;
    if (slot >= p.n_slots) {
      dev_error(p.err, MZ_DEVERR_SLOT);
    } else if (slot >= 0) {
      const int64_t blk = slot / p.bs;
      row = blk * p.Hkv * p.bs + (slot - blk * p.bs);
    }
    s_row[threadIdx.x] = row;
  }

  // the weights of this thread's dimensions
  uint64_t wa[4], wb[4];
  {
    const void *w = !p.norm || !act || kind == 2 ? nullptr : kind ? p.k_weight : p.q_weight;
    float x[8], y[8];
    load_weight(w, p.w_dtype, p.w_offset, d0, x);
    load_weight(w, p.w_dtype, p.w_offset, d0 + dd, y);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      wa[i] = f2_pack(x[2 * i], x[2 * i + 1]);
      wb[i] = f2_pack(y[2 * i], y[2 * i + 1]);
    }
  }

  // where a token's result goes: q_out and k_out by token, the pools by slot
  const bool pooled = kind > 0 && !p.k_out;
  T *dst;
  int64_t dst_ts = 0;
  if (pooled) {
    dst = static_cast<T *>(kind == 1 ? p.k_pool : p.v_pool) + (int64_t)hk * p.bs * p.D + d0;
  } else if (kind == 0) {
    dst_ts = p.qo_ts;
    dst = static_cast<T *>(p.q_out) + t0 * dst_ts + hk * p.qo_hs + d0;
  } else {
    dst_ts = p.ko_ts;
    dst = static_cast<T *>(p.k_out) + t0 * dst_ts + hk * p.ko_hs + d0;
  }
  __syncthreads();

  const float inv_d = 1.f / static_cast<float>(p.D);
  const bool turned = __any_sync(0xffffffffu, kind < 2);  // a warp of v heads only copies
  for (int t = 0; t < n_tok; ++t) {
    Raw8<T> oa = ra, ob = rb;
    fetch(t + 1);
    ahead(t + 1 + kAhead);
    if (turned) {
      uint64_t a[4], b[4];
      widen8<T>(oa, a);
      widen8<T>(ob, b);
      if (p.norm) {
        const float rs = norm_factor<P>(a, b, act, inv_d, p.eps);
        const uint64_t rs2 = f2_pack(rs, rs);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          a[i] = f2_mul(a[i], f2_mul(wa[i], rs2));
          b[i] = f2_mul(b[i], f2_mul(wb[i], rs2));
        }
      }
      if (turns) {
        const ulonglong2 *cv = reinterpret_cast<const ulonglong2 *>(&s_cos[t][8 * u]);
        const ulonglong2 *sv = reinterpret_cast<const ulonglong2 *>(&s_sin[t][8 * u]);
        const ulonglong2 c01 = cv[0], c23 = cv[1], s01 = sv[0], s23 = sv[1];
        const uint64_t c[4] = {c01.x, c01.y, c23.x, c23.y};
        const uint64_t s[4] = {s01.x, s01.y, s23.x, s23.y};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if constexpr (INTER) {
            // pairs 2 i, 2 i + 1 of the lane: vector a holds pairs 0-3, b 4-7
            uint64_t &v0 = i < 2 ? a[2 * (i & 1)] : b[2 * (i & 1)];
            uint64_t &v1 = i < 2 ? a[2 * (i & 1) + 1] : b[2 * (i & 1) + 1];
            float e0, o0, e1, o1;
            f2_unpack(v0, e0, o0);
            f2_unpack(v1, e1, o1);
            const uint64_t e = f2_pack(e0, e1), o = f2_pack(o0, o1);
            f2_unpack(f2_sub(f2_mul(e, c[i]), f2_mul(o, s[i])), e0, e1);
            f2_unpack(f2_fma(o, c[i], f2_mul(e, s[i])), o0, o1);
            v0 = f2_pack(e0, o0);
            v1 = f2_pack(e1, o1);
          } else {
            const uint64_t e = a[i], o = b[i];
            a[i] = f2_sub(f2_mul(e, c[i]), f2_mul(o, s[i]));
            b[i] = f2_fma(o, c[i], f2_mul(e, s[i]));
          }
        }
      }
      if (kind < 2) {
        oa = narrow8<T>(a);
        ob = narrow8<T>(b);
      }
    }
    if (act) {
      T *to = dst;
      if (pooled) {
        const int64_t row = s_row[t];
        if (row < 0) continue;
        to += row * p.D;
      } else {
        to += t * dst_ts;
      }
      put8(to, oa);
      put8(to + dd, ob);
    }
  }
}

// How a launch is cut: `heads` heads per block, `group` tokens per block.
struct Cut {
  int heads, threads, group;
};

// Blocks of up to kMaxThreads threads over the heads, evenly; kTokens tokens a
// block, fewer while that leaves SMs without a block, and then fewer heads.
inline Cut cut_of(int64_t n_tokens, int n_heads, int P, int sms) {
  Cut c;
  c.group = kTokens;
  int parts = (n_heads * P + kMaxThreads - 1) / kMaxThreads;
  while (c.group > 1 && (n_tokens + c.group - 1) / c.group * parts < 2 * sms) c.group /= 2;
  while (c.group == 1 && n_tokens * parts < sms && n_heads * P > parts * 64) ++parts;
  c.heads = (n_heads + parts - 1) / parts;
  c.threads = (c.heads * P + 31) / 32 * 32;
  return c;
}

template <typename T>
void launch(const RopeParams &p, int P, bool inter, dim3 grid, int threads, cudaStream_t s) {
#define MZ_ROPE(P_)                                                         \
  do {                                                                      \
    if (inter)                                                              \
      qk_norm_rope_kernel<T, P_, true><<<grid, threads, 0, s>>>(p);         \
    else                                                                    \
      qk_norm_rope_kernel<T, P_, false><<<grid, threads, 0, s>>>(p);        \
  } while (0)
  if (P == 4) MZ_ROPE(4);
  else if (P == 8) MZ_ROPE(8);
  else MZ_ROPE(16);
#undef MZ_ROPE
}

}  // namespace rope
}  // namespace mz

using namespace mz;

extern "C" int mz_qk_norm_rope(
    void *q_out, int64_t q_out_tok_stride, int64_t q_out_head_stride, void *k_out,
    int64_t k_out_tok_stride, int64_t k_out_head_stride, const void *q, int64_t q_tok_stride,
    int64_t q_head_stride, const void *k, int64_t k_tok_stride, int64_t k_head_stride,
    const void *v, int64_t v_tok_stride, int64_t v_head_stride, void *k_pool, void *v_pool,
    const int64_t *slot_mapping, int32_t block_size, int64_t n_blocks, const int32_t *positions,
    int64_t pos_axis_stride, int32_t n_axes, const float *inv_freq, const int32_t *freq_axes,
    int32_t rot_dim, int32_t interleaved, const void *q_weight, const void *k_weight,
    int32_t weight_dtype, float weight_offset, float eps, int32_t norm, int32_t n_tokens,
    int32_t n_heads, int32_t n_kv_heads, int32_t head_dim, int32_t dtype, int32_t *dev_err,
    mz_stream_t stream) {
  const char *fn = "mz_qk_norm_rope";
  const int es = dtype_bytes(dtype);
  if (!es) return fail(MZ_ERR_INVALID_ARG, "%s: unknown dtype %d", fn, dtype);
  if (n_tokens < 0 || n_heads <= 0 || n_kv_heads <= 0)
    return fail(MZ_ERR_INVALID_ARG, "%s: bad sizes", fn);
  if (head_dim < 16 || head_dim > 256 || head_dim % 16)
    return fail(MZ_ERR_UNSUPPORTED, "%s: head_dim %d (supported: multiples of 16 up to 256)", fn,
                head_dim);
  if (rot_dim < 0 || rot_dim > head_dim || rot_dim % 16)
    return fail(MZ_ERR_UNSUPPORTED,
                "%s: rotary dimension %d (supported: multiples of 16 up to head_dim)", fn, rot_dim);
  if (n_axes < 1 || n_axes > rope::kMaxAxes || (n_axes > 1 && rot_dim > 0 && !freq_axes))
    return fail(MZ_ERR_INVALID_ARG, "%s: 1..%d position axes, several need freq_axes", fn,
                rope::kMaxAxes);
  if (norm && (!(eps >= 0.f) || !(eps <= 3.4e38f)))
    return fail(MZ_ERR_INVALID_ARG, "%s: eps must be finite and not negative", fn);
  if ((q_weight || k_weight) && !dtype_bytes(weight_dtype))
    return fail(MZ_ERR_INVALID_ARG, "%s: unknown weight dtype %d", fn, weight_dtype);
  if (n_tokens == 0) return MZ_OK;
  const bool append = k_pool || v_pool;
  if (!q || !k || !q_out || (rot_dim > 0 && (!positions || !inv_freq)))
    return fail(MZ_ERR_INVALID_ARG, "%s: null pointer", fn);
  if (append) {
    if (!k_pool || !v_pool || !v || !slot_mapping || k_out)
      return fail(MZ_ERR_INVALID_ARG,
                  "%s: an append needs both pools, v and slots, and no k_out", fn);
    if (block_size <= 0 || n_blocks <= 0)
      return fail(MZ_ERR_INVALID_ARG, "%s: bad pool sizes", fn);
  } else if (!k_out) {
    return fail(MZ_ERR_INVALID_ARG, "%s: neither k_out nor pools", fn);
  }
  const int vec = 16 / es;  // elements of a 16-byte vector
  const void *ptrs[] = {q, k, q_out, append ? v : k_out, append ? k_pool : k, append ? v_pool : k,
                        q_weight, k_weight};
  const int64_t strides[] = {q_tok_stride,  q_head_stride,     k_tok_stride,
                             k_head_stride, q_out_tok_stride,  q_out_head_stride,
                             append ? v_tok_stride : k_out_tok_stride,
                             append ? v_head_stride : k_out_head_stride};
  for (const void *x : ptrs)
    if (!aligned(x, 16)) return fail(MZ_ERR_ALIGNMENT, "%s: tensors need 16-byte alignment", fn);
  for (int64_t x : strides)
    if (x % vec)
      return fail(MZ_ERR_ALIGNMENT, "%s: strides must be whole 16-byte vectors", fn);

  rope::RopeParams p;
  p.q = q;
  p.k = k;
  p.v = v;
  p.q_ts = q_tok_stride;
  p.q_hs = q_head_stride;
  p.k_ts = k_tok_stride;
  p.k_hs = k_head_stride;
  p.v_ts = v_tok_stride;
  p.v_hs = v_head_stride;
  p.q_out = q_out;
  p.k_out = append ? nullptr : k_out;
  p.qo_ts = q_out_tok_stride;
  p.qo_hs = q_out_head_stride;
  p.ko_ts = k_out_tok_stride;
  p.ko_hs = k_out_head_stride;
  p.k_pool = k_pool;
  p.v_pool = v_pool;
  p.slots = slot_mapping;
  p.bs = block_size;
  p.n_slots = append ? n_blocks * block_size : 0;
  p.positions = positions;
  p.pos_stride = pos_axis_stride;
  p.n_axes = n_axes;
  p.inv_freq = inv_freq;
  p.freq_axes = freq_axes;
  p.rot = rot_dim;
  p.q_weight = q_weight;
  p.k_weight = k_weight;
  p.w_dtype = weight_dtype;
  p.w_offset = weight_offset;
  p.eps = eps;
  p.norm = norm ? 1 : 0;
  p.n_tokens = n_tokens;
  p.Hq = n_heads;
  p.Hkv = n_kv_heads;
  p.D = head_dim;
  p.err = dev_err;
  const int sms = sm_count(current_device());
  if (sms <= 0) return fail(MZ_ERR_CUDA, "%s: cannot query the SM count", fn);
  const int P = head_dim <= 64 ? 4 : head_dim <= 128 ? 8 : 16;
  const int64_t heads = (int64_t)n_heads + (append ? 2 : 1) * (int64_t)n_kv_heads;
  if (heads >= (int64_t(1) << 24)) return fail(MZ_ERR_UNSUPPORTED, "%s: too many heads", fn);
  const rope::Cut cut = rope::cut_of(n_tokens, static_cast<int>(heads), P, sms);
  p.heads = cut.heads;
  p.group = cut.group;
  const int64_t gx = ((int64_t)n_tokens + cut.group - 1) / cut.group;
  const int64_t gy = (heads + cut.heads - 1) / cut.heads;
  if (gy > 65535) return fail(MZ_ERR_UNSUPPORTED, "%s: too many heads", fn);
  const dim3 g(static_cast<unsigned>(gx), static_cast<unsigned>(gy));
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const bool inter = interleaved != 0;
  if (dtype == MZ_DTYPE_F32) rope::launch<float>(p, P, inter, g, cut.threads, s);
  else if (dtype == MZ_DTYPE_BF16) rope::launch<__nv_bfloat16>(p, P, inter, g, cut.threads, s);
  else rope::launch<__half>(p, P, inter, g, cut.threads, s);
  MZ_CHECK_LAUNCH(fn);
  return MZ_OK;
}
