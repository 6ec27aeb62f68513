// What the files of the gated delta rule share.
#pragma once

#include "common.hpp"

namespace anna {

constexpr int CHUNK = 64;        // tokens of a chunk
// Sequences of at most so many tokens are taken token by token: about where one sequence is as fast both ways.  16 key and
// 32 value heads of 128, bf16: one sequence of 12 tokens takes 13 us by steps and one of 13 takes 16 in chunks; 8
// sequences 21 and 30, 64 sequences 77 and 144 (by steps 16 tokens of one sequence take 19, of eight 28).  More
// sequences cross later; steps hold a sequence's tokens in LDS, which has room for so many.
constexpr int STEP_TOKENS = 12;

// The records of a span's buffer: a sequence, one taken in chunks, a chunk of it
struct SpanSeq {
  int32_t slot, first, tokens, fresh;
};
struct SpanChain {
  SpanSeq seq;
  int32_t first_chunk, pad[3];
};
struct SpanChunk {
  int32_t slot, first, tokens, pad;
};
inline const SpanSeq* span_seqs(const anna_mi_state_span& s) { return (const SpanSeq*)s.buf; }
inline const SpanSeq* span_steps(const anna_mi_state_span& s) { return span_seqs(s) + s.sequences; }
inline const SpanChain* span_chains(const anna_mi_state_span& s) { return (const SpanChain*)(span_steps(s) + s.steps); }
inline const SpanChunk* span_chunks(const anna_mi_state_span& s) { return (const SpanChunk*)(span_chains(s) + s.chains); }
inline const int32_t* span_owners(const anna_mi_state_span& s) { return (const int32_t*)(span_chunks(s) + s.chunks); }

// A call takes a span with a pool of so many slots
int span_take(anna_mi_state_span* span, int64_t slots, const char* what);

// Rows of a tensor, in bytes; and whether those of two share none: of other memory, or other columns of one matrix
struct Rows {
  const void* p;
  int64_t n, stride, bytes;
};
inline bool rows_apart(const Rows& a, const Rows& b) {
  if (!a.p || !b.p || a.n < 1 || b.n < 1) return true;
  const int64_t between = (intptr_t)b.p - (intptr_t)a.p;
  if (between >= (a.n - 1) * a.stride + a.bytes || -between >= (b.n - 1) * b.stride + b.bytes) return true;
  const int64_t stride = a.n > 1 ? a.stride : b.stride;  // a single row may lie between two of the other
  if ((a.n == 1 && b.n == 1) || (b.n > 1 && b.stride != stride) || stride < 1) return false;
  const int64_t column = (between % stride + stride) % stride;
  return column >= a.bytes && column <= stride - b.bytes;
}

// x / (1 + e^-x), off by a few 2^-24 of itself (|x| 2^-24 where x is far below 0)
__device__ __forceinline__ float silu_of(float x) {
  return x * __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(-1.44269504f * x));
}

// The decay's logarithm and beta of a token and value head, from what the caller gave
struct Gate {
  float g, beta;
};
__device__ __forceinline__ float gate_value(const void* p, int dtype, int64_t i) {
  if (dtype == ANNA_MI_F32) return ((const float*)p)[i];
  const uint16_t h = ((const uint16_t*)p)[i];
  return dtype == ANNA_MI_BF16 ? bf16_bits_to_f32(h) : f16_bits_to_f32(h);
}
struct HeadGate {
  bool made;  // from projections
  float rate, bias;
};
__device__ __forceinline__ HeadGate head_gate(const anna_mi_gated_delta_args& a, int64_t head) {
  if (!a.a_log) return {false, 0.f, 0.f};
  return {true, expf(a.a_log[head]), a.dt_bias[head]};
}
__device__ __forceinline__ Gate gate_of(HeadGate h, Gate r) {
  if (h.made) {
    const float x = r.g + h.bias;
    r.g = -h.rate * (fmaxf(x, 0.f) + log1pf(expf(-fabsf(x))));  // softplus without overflow
    r.beta = 1.f / (1.f + expf(-r.beta));
  }
  return r;
}
__device__ __forceinline__ Gate gate_of(const anna_mi_gated_delta_args& a, Gate r, int64_t head) { return gate_of(head_gate(a, head), r); }
__device__ __forceinline__ Gate gate_of(const anna_mi_gated_delta_args& a, int64_t token, int64_t head) {
  return gate_of(a,
                 Gate{gate_value(a.decay, a.gates_dtype, token * a.decay_stride + head),
                      gate_value(a.beta, a.gates_dtype, token * a.beta_stride + head)},
                 head);
}

constexpr float NORM_EPS = 1e-6f;

// What the step and chunk files launch, after the checks of anna_mi_gated_delta
int delta_step(const anna_mi_gated_delta_args& a, const anna_mi_state_span& s, hipStream_t stream);

}  // namespace anna
