// The short causal convolution of a linear-attention layer over packed, ragged sequences, with the last
// width - 1 inputs of every sequence kept in a row of a state pool.
//
//   out[t, c] = act(bias[c] + sum_j weight[c, j] x[t - (width - 1) + j, c]),   x in front of a sequence: its state
//
// A thread takes 4 channels (8 bytes of the 16-bit types) and walks down `tile` tokens with the window in
// registers, so an input is read once, and the width - 1 in front of a tile once more.  The next four tokens' rows are asked
// for in front of a group's stores, and full groups have no branches.  Sums are fp32, rounded to the type once, after
// the activation; the state keeps inputs as they came, so nothing is rounded there.
// The thread that has a sequence's first token also takes the width - 2 tokens behind it, also past its tile:
// it alone reads the state of its channels, and then writes the new one.
//
// Bound by the bytes of x and out.  12787 tokens of 8192 channels in 6 sequences, bf16, width 4 (0.42 GB): 85 us =
// 4.9 TB/s; a copy of 1 GiB runs at 5.2.  8 channels a thread took 165 us (half the waves, so that loads wait for
// stores), groups of four with branches in them 134; rows' addresses by addition and not by product took 284000 tokens of 96
// channels from 29.5 to 27.4.  One token of 64 sequences: 4.0 us, an empty launch takes 3.6.
#include <type_traits>

#include "delta.hpp"

namespace anna {

constexpr int NC = 4;  // channels of a thread

template <int DT>
struct alignas(NC * sizeof(typename Elem<DT>::T)) Vec {
  typename Elem<DT>::T v[NC];
};

template <int DT, int W, bool VEC>
__global__ __launch_bounds__(256) void short_conv_kernel(const typename Elem<DT>::T* __restrict__ x, int64_t x_stride,
                                                         const typename Elem<DT>::T* __restrict__ weight,
                                                         const typename Elem<DT>::T* __restrict__ bias,
                                                         typename Elem<DT>::T* state, uint32_t slots, int64_t state_stride, uint32_t channels,
                                                         int silu, const SpanSeq* __restrict__ seqs,
                                                         const int32_t* __restrict__ owners, int tokens, int tile,
                                                         typename Elem<DT>::T* __restrict__ out, int64_t out_stride) {
  typedef typename Elem<DT>::T T;
  typedef Vec<DT> Row;
  constexpr int FOUR = 4;  // tokens whose loads go together, a group ahead of their use
  const uint32_t groups = (channels + NC - 1) / NC, item = blockIdx.x * 256 + threadIdx.x, c0 = item % groups * NC;
  const int64_t begin = (int64_t)(item / groups) * tile;
  if (begin >= tokens) return;
  const int first = (int)begin, last = (int)min(begin + tile, (int64_t)tokens), n = min((uint32_t)NC, channels - c0);

  auto load = [&](const T* p) {
    Row r;
    if constexpr (VEC) {
      r = *(const Row*)p;
    } else {
#pragma unroll
      for (int e = 0; e < NC; e++) r.v[e] = e < n ? p[e] : (T)0;
    }
    return r;
  };
  auto save = [&](T* p, const Row& r) {
    if constexpr (VEC) {
      *(Row*)p = r;
    } else {
#pragma unroll
      for (int e = 0; e < NC; e++)
        if (e < n) p[e] = r.v[e];
    }
  };

  int s = owners[first];
  SpanSeq seq = seqs[s];
  float w[W][NC], b[NC] = {};
  if constexpr (VEC) {  // the channels' taps lie together
#pragma unroll
    for (int i = 0; i < W; i++) {
      const Row r = load(weight + (int64_t)c0 * W + NC * i);
#pragma unroll
      for (int e = 0; e < NC; e++) w[(NC * i + e) % W][(NC * i + e) / W] = Elem<DT>::to_f32(r.v[e]);
    }
  } else {
#pragma unroll
    for (int e = 0; e < NC; e++)
#pragma unroll
      for (int j = 0; j < W; j++) w[j][e] = e < n ? Elem<DT>::load(weight, (int64_t)(c0 + e) * W + j) : 0.f;
  }
  if (bias)
#pragma unroll
    for (int e = 0; e < NC; e++) b[e] = e < n ? Elem<DT>::load(bias, c0 + e) : 0.f;

  int t = first;
  if (t > seq.first && t < seq.first + W - 1) t = min(seq.first + min(W - 1, seq.tokens), last);  // another thread's
  while (t < last) {
    while (t >= seq.first + seq.tokens) seq = seqs[++s];
    const int pos = t - seq.first, end = seq.first + seq.tokens;
    // to the tile's end, and from a sequence's first token through the width - 2 behind it
    const int stop = min(end, pos == 0 ? max(last, seq.first + W - 1) : last), run = stop - t;
    if ((uint32_t)seq.slot >= slots) {
      Row zeros;
#pragma unroll
      for (int e = 0; e < NC; e++) zeros.v[e] = Elem<DT>::cvt(0.f);
      for (; t < stop; t++) save(out + (int64_t)t * out_stride + c0, zeros);
      continue;
    }
    const T* const from = x + (int64_t)t * x_stride + c0;
    Row next[FOUR], win[W - 1];  // win: the inputs in front of the next one
#pragma unroll
    for (int i = 0; i < FOUR; i++) next[i] = load(from + (int64_t)min(i, run - 1) * x_stride);
#pragma unroll
    for (int j = 0; j < W - 1; j++) {
      const int at = pos - (W - 1) + j;
      if (at >= 0) {
        win[j] = load(x + (int64_t)(seq.first + at) * x_stride + c0);
      } else if (!seq.fresh) {
        win[j] = load(state + seq.slot * state_stride + (int64_t)(W - 1 + at) * channels + c0);
      } else {
#pragma unroll
        for (int e = 0; e < NC; e++) win[j].v[e] = Elem<DT>::cvt(0.f);
      }
    }
    if (pos == 0) {
      // the state after the sequence's tokens: all of the old one that is needed is in the window
      T* to = state + seq.slot * state_stride + c0;
#pragma unroll
      for (int j = 0; j < W - 1; j++) {
        const int at = seq.tokens - (W - 1) + j;
        Row r = win[W - 2];
        if (at >= 0) {
          r = load(x + (int64_t)(seq.first + at) * x_stride + c0);
        } else {
#pragma unroll
          for (int i = 0; i < W - 1; i++)  // window entry i is position i - (W - 1)
            if (i == W - 1 + at) r = win[i];
        }
        save(to + (int64_t)j * channels, r);
      }
    }
    T* to = out + (int64_t)t * out_stride + c0;
    const T* ahead = from + FOUR * x_stride;
    // of `m` tokens from k on; the next ones' rows, which with `all` are all there, are asked for in front of the stores
    auto outputs = [&](int k, int m, auto all) {
      Row rows[W - 1 + FOUR];
#pragma unroll
      for (int j = 0; j < W - 1; j++) rows[j] = win[j];
#pragma unroll
      for (int i = 0; i < FOUR; i++) rows[W - 1 + i] = next[i];
#pragma unroll
      for (int j = 0; j < W - 1; j++) win[j] = rows[FOUR + j];
      if constexpr (all.value) {
#pragma unroll
        for (int i = 0; i < FOUR; i++) next[i] = load(ahead + i * x_stride);
        ahead += FOUR * x_stride;
      } else if (m == FOUR) {
#pragma unroll
        for (int i = 0; i < FOUR; i++) next[i] = load(from + (int64_t)min(k + FOUR + i, run - 1) * x_stride);
      }
      Row y[FOUR];
#pragma unroll
      for (int i = 0; i < FOUR; i++)
#pragma unroll
        for (int e = 0; e < NC; e++) {
          float sum = b[e];
#pragma unroll
          for (int j = 0; j < W; j++) sum = fmaf(Elem<DT>::to_f32(rows[i + j].v[e]), w[j][e], sum);
          y[i].v[e] = Elem<DT>::cvt(silu ? silu_of(sum) : sum);
        }
#pragma unroll
      for (int i = 0; i < FOUR; i++)
        if (i < m) save(to + i * out_stride, y[i]);
      to += FOUR * out_stride;
    };
    int k = 0;
    for (; k + 2 * FOUR <= run; k += FOUR) outputs(k, FOUR, std::true_type());
    if (k + FOUR <= run) {
      outputs(k, FOUR, std::false_type());
      k += FOUR;
    }
    if (k < run) outputs(k, run - k, std::false_type());
    t = stop;
  }
}

template <int DT>
static int launch(const void* x, int64_t channels, int64_t x_stride, const void* weight, int64_t width, const void* bias,
                  void* state, int64_t slots, int64_t state_stride, int activation, const anna_mi_state_span* s, void* out,
                  int64_t out_stride, hipStream_t stream) {
  typedef typename Elem<DT>::T T;
  auto rows = [&](const void* p, int64_t stride) { return (uintptr_t)p % (NC * sizeof(T)) == 0 && stride % NC == 0; };
  const bool vec = channels % NC == 0 && rows(x, x_stride) && rows(out, out_stride) && rows(state, state_stride) && rows(weight, NC);
  // 24 tokens a thread once that fills the chip with 8 waves a compute unit, fewer otherwise.  At 12787 tokens of 8192
  // channels 16 and 48 are within 3% of it; below the limit a call takes as long as one wave's chain of loads.
  const int64_t groups = (channels + NC - 1) / NC;
  int tile = 24;
  while (tile > 1 && groups * ((s->tokens + tile - 1) / tile) < 256 * 8 * 64) tile /= 2;
  const int64_t items = groups * ((s->tokens + tile - 1) / tile), grid = (items + 255) / 256;
  ANNA_CHECK(grid <= INT32_MAX / 256, "causal_conv1d: too many tokens and channels for a launch");
#define ANNA_CONV(W)                                                                                                       \
  case W:                                                                                                                  \
    (vec ? short_conv_kernel<DT, W, true> : short_conv_kernel<DT, W, false>)<<<grid, 256, 0, stream>>>((const T*)x, x_stride, (const T*)weight, (const T*)bias, (T*)state, (uint32_t)slots, \
                                                       state_stride, (uint32_t)channels, activation, span_seqs(*s), span_owners(*s), \
                                                       (int)s->tokens, tile, (T*)out, out_stride);                    \
    break;
  switch (width) {
    ANNA_CONV(2) ANNA_CONV(3) ANNA_CONV(4) ANNA_CONV(5) ANNA_CONV(6) ANNA_CONV(7) ANNA_CONV(8)
    default: set_error("causal_conv1d: width %lld", (long long)width); return ANNA_MI_EINVAL;
  }
#undef ANNA_CONV
  ANNA_LAUNCH_CHECK("causal_conv1d");
  return ANNA_MI_OK;
}

}  // namespace anna

extern "C" int anna_mi_causal_conv1d(const void* x, int dtype, int64_t channels, int64_t x_stride, const void* weight,
                                     int64_t width, const void* bias, void* state, int64_t slots, int64_t state_stride_slot,
                                     int activation, anna_mi_state_span* span, void* out, int64_t out_stride, void* stream) {
  ANNA_CHECK(span != nullptr, "causal_conv1d: null span");
  ANNA_CHECK(anna::valid_dtype(dtype), "causal_conv1d: dtype %d", dtype);
  ANNA_CHECK(width >= 2 && width <= 8, "causal_conv1d: width %lld, 2 to 8 are supported", (long long)width);
  ANNA_CHECK(channels >= 1 && channels <= (1 << 24), "causal_conv1d: %lld channels", (long long)channels);
  ANNA_CHECK(activation == 0 || activation == 1, "causal_conv1d: activation %d", activation);
  ANNA_CHECK(slots >= 0 && slots <= INT32_MAX, "causal_conv1d: %lld slots", (long long)slots);
  ANNA_CHECK(span->max_slot < slots, "causal_conv1d: slot %lld of a state of %lld", (long long)span->max_slot, (long long)slots);
  if (span->tokens == 0) return ANNA_MI_OK;
  ANNA_CHECK(span->tokens <= INT32_MAX && x && weight && out && span->buf && (state || span->max_slot < 0), "causal_conv1d: null pointer");
  ANNA_CHECK(x_stride >= channels || span->tokens == 1, "causal_conv1d: rows of x overlap");
  ANNA_CHECK(out_stride >= channels || span->tokens == 1, "causal_conv1d: rows of out overlap");
  ANNA_CHECK(slots <= 1 || state_stride_slot >= (width - 1) * channels, "causal_conv1d: rows of the state overlap");
  // a state is written while other workgroups still read x
  const int64_t size = dtype == ANNA_MI_F32 ? 4 : 2;
  const anna::Rows states = {state, slots, state_stride_slot * size, (width - 1) * channels * size};
  ANNA_CHECK(anna::rows_apart(states, {x, span->tokens, x_stride * size, channels * size}), "causal_conv1d: the state overlaps x");
  ANNA_CHECK(anna::rows_apart(states, {weight, 1, 0, channels * width * size}), "causal_conv1d: the state overlaps weight");
  ANNA_CHECK(anna::rows_apart(states, {bias, 1, 0, channels * size}), "causal_conv1d: the state overlaps bias");
  if (const int rc = anna::span_take(span, slots, "causal_conv1d")) return rc;
  ANNA_DISPATCH_DTYPE(dtype, DT, return anna::launch<DT>(x, channels, x_stride, weight, width, bias, state, slots, state_stride_slot,
                                                         activation, span, out, out_stride, anna::as_stream(stream)));
}
