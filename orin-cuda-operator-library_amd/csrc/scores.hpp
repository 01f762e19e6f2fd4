#pragma once
// From a dot product to a score, for the attention kernels of language
// models: score = scale * dot, or softcap * tanh(scale * dot / softcap).
//
// The softmax is exp2 of the scores in log2 units. With y = scale * dot / softcap,
//   softcap tanh y = 2 softcap sigma(2 y) - softcap,  sigma(x) = 1 / (1 + e^-x),
// and the constant drops out of a softmax: capped() gives sigma(2 y), one
// v_exp and one v_rcp, and after() = 2 softcap log2 e is its scale. sigma is
// off by 2^-23 at most, a score by softcap / 4e6: up to kSigmaCap below the 2^-11
// by which a probability in fp16 is off.
// kPrecise (fp32, and larger caps): capped() gives tanh y itself and after() softcap log2 e. For
// |y| < 0.625 tanh is the quotient y (945 + 105 y^2 + y^4) / (945 + 420 y^2 +
// 15 y^4), the fifth convergent of Lambert's continued fraction (relative
// error 1e-9 there), as sigma - 1/2 loses the leading digits of a small tanh.

#include "common.hpp"

namespace opl {

constexpr float kSigmaCap = 1024.0f;

struct ScoreRules {
  float scale;       // capped: scale / softcap; else scale * log2 e
  float cap = 0.0f;  // softcap * log2 e; 0: no cap

  static ScoreRules of(float scale, float softcap) {
    ScoreRules r;
    r.scale = softcap > 0.0f ? scale / softcap : scale * kLog2e;
    r.cap = softcap * kLog2e;
    return r;
  }

  bool wide_cap() const { return cap > kSigmaCap * kLog2e; }

  template <bool kPrecise>
  __device__ __forceinline__ float capped(float dot) const {
    const float y = dot * scale;
    if constexpr (!kPrecise) {
      return __builtin_amdgcn_rcpf(1.0f + fast_exp2(dot * (-2.0f * kLog2e * scale)));
    } else {
      const float z = y * y;
      const bool near = z < 0.390625f;
      const float u = fast_exp2(-2.0f * kLog2e * fabsf(y));
      const float n = near ? y * fmaf(z, z + 105.0f, 945.0f) : copysignf(1.0f - u, y);
      const float d = near ? fmaf(z, fmaf(15.0f, z, 420.0f), 945.0f) : 1.0f + u;
      return n * __builtin_amdgcn_rcpf(d);
    }
  }

  // What capped() (or, without a cap, the dot product) is multiplied by.
  template <bool kPrecise>
  __device__ __forceinline__ float after() const {
    return cap == 0.0f ? scale : kPrecise ? cap : 2.0f * cap;
  }

  // The score in log2 units, up to the constant of a capped one.
  template <bool kPrecise>
  __device__ __forceinline__ float log2_score(float dot) const {
    return (cap != 0.0f ? capped<kPrecise>(dot) : dot) * after<kPrecise>();
  }
};

}  // namespace opl
