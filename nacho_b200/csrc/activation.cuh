// The activations of gated layers.
#pragma once

namespace nb200 {

// act(v) = v s(p(v)) with the logistic function s, p(v) = v, or 2 sqrt(2 / pi) (v + 0.044715 v^3) for the tanh form of gelu. s is computed from
// exp(-|p|), which neither overflows nor loses what is left of it far below zero.
constexpr float GELU1 = 1.5957691216057308f, GELU3 = 0.0713548162726009f;
__device__ __forceinline__ float act_inner(float v, bool gelu) { return gelu ? v * __fmaf_rn(GELU3 * v, v, GELU1) : v; }
__device__ __forceinline__ float logistic(float p, float *small = nullptr) {
    const float t = __expf(-fabsf(p)), part = __fdividef(1.f, 1.f + t);
    if (small) *small = t * part;
    return p < 0.f ? t * part : part;
}

}  // namespace nb200
