#pragma once
// From a dot product to a score, for the attention kernels of language
// models: score = scale * dot, or softcap * tanh(scale * dot / softcap), in
// log2 units (times log2 e) so that the softmax is exp2.

#include "common.hpp"

namespace opl {

struct ScoreRules {
  float scale;     // scale * log2 e, or with a cap scale / softcap
  float cap = 0.0f;  // softcap * log2 e; 0: no cap

  static ScoreRules of(float scale, float softcap) {
    ScoreRules r;
    r.scale = softcap > 0.0f ? scale / softcap : scale * kLog2e;
    r.cap = softcap * kLog2e;
    return r;
  }

  // tanh y = 1 - 2 / (1 + e^2y): one v_exp and one v_rcp, absolute error
  // 2e-7. For fp16 inputs that is the error of a score of softcap / 5e6.
  // kPrecise (fp32): for |y| < 0.625 the quotient y (945 + 105 y^2 + y^4) /
  // (945 + 420 y^2 + 15 y^4), the fifth convergent of Lambert's continued
  // fraction (relative error 1e-9 there), since the difference above loses the
  // leading digits of a small tanh.
  template <bool kPrecise>
  __device__ __forceinline__ static float tanh_of(float y) {
    const float far = 1.0f - 2.0f * __builtin_amdgcn_rcpf(1.0f + fast_exp2(2.0f * kLog2e * y));
    if constexpr (!kPrecise) return far;
    const float z = y * y;
    const float near = y * fmaf(z, z + 105.0f, 945.0f) *
                       __builtin_amdgcn_rcpf(fmaf(z, fmaf(15.0f, z, 420.0f), 945.0f));
    return z < 0.390625f ? near : far;
  }

  template <bool kPrecise>
  __device__ __forceinline__ float capped(float dot) const {
    return cap * tanh_of<kPrecise>(dot * scale);
  }

  template <bool kPrecise>
  __device__ __forceinline__ float log2_score(float dot) const {
    return cap != 0.0f ? capped<kPrecise>(dot) : dot * scale;
  }
};

}  // namespace opl
