// Scores beyond scaled products, and masks beyond the causal one, shared by
// the decode and the prefill attention kernels.
//
// For a token at position p of a sequence and a key at position t,
//   x = scale q.k;   x <- cap tanh(x / cap);   x <- x - slope_h |p - t|
// and the key is seen iff
//   t < prefix_b  or  (t <= p  and  (t >= lo  or  t < sink)),
//   lo = max(first, p - window + 1).
// A row that sees no key has output 0.  The kernels keep x in units of log2 e,
// so that its exponential is one ex2.
#pragma once

#include <cmath>

#include "common.cuh"

namespace mz {

struct ScoreMod {
  const float *slopes;    // [n_heads], null: none
  const int32_t *first;   // per sequence (decode) or per row (prefill), null: 0
  const int32_t *prefix;  // per sequence, null: 0
  int window;             // 0: none
  int sink;
  float z_scale;   // scale / cap; 0: no cap
  float cap_log2;  // cap * log2(e)
  // cap_log2 * tanh(z_scale * s) = s (poly[0] + s^2 (poly[1] + ...)) for raw
  // scores |s| <= poly_range; below 0: no such range
  float poly[4];
  float poly_range;
};

constexpr float kLog2e = 1.4426950408889634f;
// Running maximum of a row that has seen no key yet: finite, so that the
// difference of two of them is 0 and not NaN, and below every score.
constexpr float kNoMax = -3.0e38f;

// tanh to a relative error of about 1e-6: the odd series to z^9 below 0.3 (its
// next term is 5e-8 of z there), 1 - 2 / (e^(2 |z|) + 1) from there on, where
// the subtraction loses no more than two bits.
__device__ __forceinline__ float tanh_mod(float z) {
  const float a = fabsf(z), z2 = z * z;
  float s = fmaf(z2, 2.18694885e-2f, -5.39682540e-2f);
  s = fmaf(s, z2, 1.33333333e-1f);
  s = fmaf(s, z2, -3.33333333e-1f);
  s = fmaf(s * z2, z, z);
  const float e = fast_exp2(a * (2.f * kLog2e));
  const float t = copysignf(1.f - __fdividef(2.f, e + 1.f), z);
  return a < 0.3f ? s : t;
}

// cap_log2 * tanh(z_scale * s): 1 - 2 / (e^(2 z) + 1) is off by 2.4e-7 at most, so
// by less than 2^-12 in the scores up to a cap of 1000.  Decode takes it for every
// score up to that cap (prefill only for tiles with scores beyond half the cap,
// the cubic below for the rest), tanh_mod above it.
__device__ __forceinline__ float rcp_approx(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float cap_quick(const ScoreMod &m, float s) {
  return fmaf(-2.f * m.cap_log2, rcp_approx(fast_exp2(s * (m.z_scale * (2.f * kLog2e))) + 1.f),
              m.cap_log2);
}
__device__ __forceinline__ float cap_poly(const ScoreMod &m, float s) {
  const float w = s * s;
  return fmaf(fmaf(fmaf(w, m.poly[3], m.poly[2]), w, m.poly[1]), w, m.poly[0]) * s;
}
constexpr float kQuickCapLog2 = 1000.f * kLog2e;

// Host side: the fields of mz_score_mod checked and folded with the scale.
// `tokens`: the table's capacity, which bounds what window and sink can mean.
inline int make_score_mod(ScoreMod *m, const mz_score_mod *mod, float scale, int64_t tokens,
                          const char *fn) {
  if (!mod) return fail(MZ_ERR_INVALID_ARG, "%s: mod is null", fn);
  if (!std::isfinite(mod->softcap) || mod->softcap < 0.f ||
      (mod->softcap > 0.f && !std::isfinite(scale / mod->softcap)))
    return fail(MZ_ERR_INVALID_ARG,
                "%s: softcap must be finite, not negative and not so small that scale / softcap "
                "overflows", fn);
  if (tokens >= (int64_t(1) << 31) - 1024)
    return fail(MZ_ERR_UNSUPPORTED, "%s: tables span 2^31 or more tokens", fn);
  if (mod->window < 0 || mod->sink_tokens < 0)
    return fail(MZ_ERR_INVALID_ARG, "%s: window and sink_tokens must not be negative", fn);
  const void *ptrs[] = {mod->alibi_slopes, mod->prefix_lens, mod->first_keys};
  for (const void *x : ptrs)
    if (!aligned(x, 4)) return fail(MZ_ERR_ALIGNMENT, "%s: mod arrays need 4-byte alignment", fn);
  m->slopes = mod->alibi_slopes;
  m->first = mod->first_keys;
  m->prefix = mod->prefix_lens;
  // a window of the whole table hides nothing; no position exceeds it either
  m->window = mod->window >= tokens ? 0 : mod->window;
  m->sink = static_cast<int>(mod->sink_tokens < tokens ? mod->sink_tokens : tokens);
  // a cap of 10^30 leaves every fp32 score as it is; scale / cap would near the
  // smallest fp32 numbers there
  const float cap = mod->softcap < 1e30f ? mod->softcap : 0.f;
  m->z_scale = cap > 0.f ? scale / cap : 0.f;
  const double cap_log2 = static_cast<double>(cap) * 1.4426950408889634;
  m->cap_log2 = static_cast<float>(cap_log2);
  // tanh(z) / z on |z| <= 1/2 by the cubic in z^2 through its values at the four
  // Chebyshev nodes of [0, 1/4]: tanh to 2.5e-7, relative 5.5e-7
  const double tanh_c[4] = {0.999999451, -0.3332628423, 0.1318993943, -0.04439273843};
  double f = cap_log2 * m->z_scale;
  // (up to 1e15, so that s^2 stays finite beside coefficients that vanish)
  m->poly_range = m->z_scale > 0.f ? std::fmin(0.5f / m->z_scale, 1e15f) : -1.f;
  for (int i = 0; i < 4; ++i, f *= static_cast<double>(m->z_scale) * m->z_scale) {
    const double c = tanh_c[i] * f;
    m->poly[i] = static_cast<float>(c);
    if (!(std::fabs(c) < 1e35)) m->poly_range = -1.f;  // a tiny cap: the other form
  }
  return MZ_OK;
}

}  // namespace mz
