// The AdamW update of one element, shared by every kernel that steps
// parameters (adamw.hip, adamw_multi.hip), so that they round alike.
#pragma once
#include <cmath>

#include "zk_common.h"

namespace zk {

struct AdamScalars {
  float decay;         // 1 - lr * weight_decay
  float one_minus_b1;  // lerp weight of the first moment
  float b2, one_minus_b2;
  float step_size;     // lr / (1 - b1^t)
  float bc2_sqrt;      // sqrt(1 - b2^t)
  float eps;
};

__device__ __forceinline__ float adam_one(float& p, float g, float& m, float& v,
                                          const AdamScalars& s) {
  p = p * s.decay;
  m = fmaf(s.one_minus_b1, g - m, m);
  v = fmaf(s.one_minus_b2, g * g, v * s.b2);
  const float denom = sqrtf(v) / s.bc2_sqrt + s.eps;
  p = p - s.step_size * (m / denom);
  return p;
}

inline AdamScalars adam_scalars(double lr, double beta1, double beta2, double eps,
                                double weight_decay, int64_t step) {
  AdamScalars s;
  s.decay = static_cast<float>(1.0 - lr * weight_decay);
  s.one_minus_b1 = static_cast<float>(1.0 - beta1);
  s.b2 = static_cast<float>(beta2);
  s.one_minus_b2 = static_cast<float>(1.0 - beta2);
  const double bc1 = 1.0 - std::pow(beta1, static_cast<double>(step));
  const double bc2 = 1.0 - std::pow(beta2, static_cast<double>(step));
  s.step_size = static_cast<float>(lr / bc1);
  s.bc2_sqrt = static_cast<float>(std::sqrt(bc2));
  s.eps = static_cast<float>(eps);
  return s;
}

}  // namespace zk
