// What the files of the gated delta rule share.
#pragma once

#include "common.hpp"

namespace anna {

constexpr int CHUNK = 64;        // tokens of a chunk
constexpr int STEP_TOKENS = 12;  // sequences of at most so many tokens are taken token by token

// A sequence's record in a span's buffer
struct SpanSeq {
  int32_t slot, first, tokens, fresh;
};

// The decay's logarithm and beta of a token and value head, from what the caller gave
struct Gate {
  float g, beta;
};
__device__ __forceinline__ float gate_value(const void* p, int dtype, int64_t i) {
  if (dtype == ANNA_MI_F32) return ((const float*)p)[i];
  const uint16_t h = ((const uint16_t*)p)[i];
  return dtype == ANNA_MI_BF16 ? bf16_bits_to_f32(h) : f16_bits_to_f32(h);
}
__device__ __forceinline__ Gate gate_of(const anna_mi_gated_delta_args& a, int64_t token, int64_t head) {
  Gate r{gate_value(a.decay, a.gates_dtype, token * a.decay_stride + head),
         gate_value(a.beta, a.gates_dtype, token * a.beta_stride + head)};
  if (a.a_log) {
    const float x = r.g + a.dt_bias[head];
    r.g = -expf(a.a_log[head]) * (fmaxf(x, 0.f) + log1pf(expf(-fabsf(x))));  // softplus without overflow
    r.beta = 1.f / (1.f + expf(-r.beta));
  }
  return r;
}

constexpr float NORM_EPS = 1e-6f;

// What the step and chunk files launch, after the checks of anna_mi_gated_delta
int delta_step(const anna_mi_gated_delta_args& a, const anna_mi_state_span& s, hipStream_t stream);

}  // namespace anna
