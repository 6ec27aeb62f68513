// The short causal convolution of a linear-attention layer over packed, ragged sequences, with the last
// width - 1 inputs of every sequence kept in a row of a state pool.
//
// A thread takes 8 channels (16 bytes of the 16-bit types) and walks down TILE tokens with the window in
// registers, so an input is read once and width - 1 times more at a tile's border.  Bound by the bytes of x and out.
// The thread that has a sequence's first token also takes the width - 2 tokens behind it, also past its tile:
// it alone reads the state of its channels, and then writes the new one.
#include "delta.hpp"

namespace anna {

template <int DT>
struct Vec8 {
  typename Elem<DT>::T v[8];
};

template <int DT, int W>
__global__ __launch_bounds__(256) void short_conv_kernel(const typename Elem<DT>::T* __restrict__ x, int64_t x_stride,
                                                         const typename Elem<DT>::T* __restrict__ weight,
                                                         const typename Elem<DT>::T* __restrict__ bias,
                                                         typename Elem<DT>::T* state, int64_t state_stride, int64_t channels,
                                                         int silu, const SpanSeq* __restrict__ seqs, int sequences, int tokens,
                                                         int tile, int vec, typename Elem<DT>::T* __restrict__ out,
                                                         int64_t out_stride) {
  typedef typename Elem<DT>::T T;
  const int64_t groups = (channels + 7) / 8, item = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int64_t c0 = item % groups * 8;
  const int64_t first = item / groups * tile;
  if (first >= tokens) return;
  const int n = (int)min((int64_t)8, channels - c0), last = (int)min(first + tile, (int64_t)tokens);

  auto load = [&](const T* p, float (&f)[8]) {
    if (vec) {
      const Vec8<DT> v = *(const Vec8<DT>*)__builtin_assume_aligned(p, 16);
#pragma unroll
      for (int e = 0; e < 8; e++) f[e] = Elem<DT>::to_f32(v.v[e]);
    } else {
#pragma unroll
      for (int e = 0; e < 8; e++) f[e] = e < n ? Elem<DT>::load(p, e) : 0.f;
    }
  };
  auto save = [&](T* p, const float (&f)[8]) {
    if (vec) {
      Vec8<DT> v;
#pragma unroll
      for (int e = 0; e < 8; e++) v.v[e] = Elem<DT>::cvt(f[e]);
      *(Vec8<DT>*)__builtin_assume_aligned(p, 16) = v;
    } else {
#pragma unroll
      for (int e = 0; e < 8; e++)
        if (e < n) p[e] = Elem<DT>::cvt(f[e]);
    }
  };

  float w[W][8], b[8] = {};
#pragma unroll
  for (int e = 0; e < 8; e++)
#pragma unroll
    for (int j = 0; j < W; j++) w[j][e] = e < n ? Elem<DT>::load(weight, (c0 + e) * W + j) : 0.f;
  if (bias)
#pragma unroll
    for (int e = 0; e < 8; e++) b[e] = e < n ? Elem<DT>::load(bias, c0 + e) : 0.f;

  // the last sequence that begins at or before the tile and is not empty
  int lo = 0, hi = sequences - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) / 2;
    if (seqs[mid].first <= first) lo = mid;
    else hi = mid - 1;
  }
  int s = lo;
  SpanSeq seq = seqs[s];

  float win[W][8];  // inputs t - W + 1 .. t
  bool begins = true;
  int t = (int)first;
  if (t > seq.first && t < seq.first + W - 1) t = min(seq.first + min(W - 1, seq.tokens), last);  // another thread's
  for (;; t++) {
    if (t >= last && (begins || t >= min(seq.first + W - 1, seq.first + seq.tokens))) break;
    while (t >= seq.first + seq.tokens) {
      seq = seqs[++s];
      begins = true;
    }
    const int pos = t - seq.first;
    if (begins) {
      begins = false;
#pragma unroll
      for (int j = 0; j < W - 1; j++) {
        const int at = pos - (W - 1) + j;
        if (at >= 0) {
          load(x + (int64_t)(seq.first + at) * x_stride + c0, win[j + 1]);
        } else if (seq.slot >= 0 && !seq.fresh) {
          load(state + seq.slot * state_stride + (int64_t)(W - 1 + at) * channels + c0, win[j + 1]);
        } else {
#pragma unroll
          for (int e = 0; e < 8; e++) win[j + 1][e] = 0.f;
        }
      }
      if (pos == 0 && seq.slot >= 0) {
        // the state after the sequence's tokens: all of the old one that is needed is in the window
        T* to = state + seq.slot * state_stride + c0;
#pragma unroll
        for (int j = 0; j < W - 1; j++) {
          const int at = seq.tokens - (W - 1) + j;
          float f[8];
          if (at >= 0) {
            load(x + (int64_t)(seq.first + at) * x_stride + c0, f);
          } else {
#pragma unroll
            for (int i = 0; i < W - 1; i++)  // window entry 1 + i is position i - (W - 1)
              if (i == W - 1 + at)
#pragma unroll
                for (int e = 0; e < 8; e++) f[e] = win[1 + i][e];
          }
          save(to + (int64_t)j * channels, f);
        }
      }
    }
#pragma unroll
    for (int j = 0; j + 1 < W; j++)
#pragma unroll
      for (int e = 0; e < 8; e++) win[j][e] = win[j + 1][e];
    load(x + (int64_t)t * x_stride + c0, win[W - 1]);
    float y[8];
#pragma unroll
    for (int e = 0; e < 8; e++) {
      y[e] = b[e];
#pragma unroll
      for (int j = 0; j < W; j++) y[e] = fmaf(win[j][e], w[j][e], y[e]);
      if (silu) y[e] = y[e] / (1.f + expf(-y[e]));
      if (seq.slot < 0) y[e] = 0.f;
    }
    save(out + (int64_t)t * out_stride + c0, y);
  }
}

template <int DT>
static int launch(const void* x, int64_t channels, int64_t x_stride, const void* weight, int64_t width, const void* bias,
                  void* state, int64_t state_stride, int activation, const anna_mi_state_span* s, void* out,
                  int64_t out_stride, hipStream_t stream) {
  typedef typename Elem<DT>::T T;
  constexpr int64_t unit = 16 / sizeof(T);
  auto rows16 = [&](const void* p, int64_t stride) { return (uintptr_t)p % 16 == 0 && stride % unit == 0; };
  const int vec = channels % 8 == 0 && rows16(x, x_stride) && rows16(out, out_stride) && rows16(state, state_stride);
  // 16 tokens a thread once that fills the chip with 8 waves a compute unit, fewer otherwise
  const int64_t groups = (channels + 7) / 8;
  int tile = 16;
  while (tile > 1 && groups * ((s->tokens + tile - 1) / tile) < 256 * 8 * 64) tile /= 2;
  const int64_t items = groups * ((s->tokens + tile - 1) / tile), grid = (items + 255) / 256;
  ANNA_CHECK(grid <= INT32_MAX / 256, "causal_conv1d: too many tokens and channels for a launch");
#define ANNA_CONV(W)                                                                                                       \
  case W:                                                                                                                  \
    short_conv_kernel<DT, W><<<grid, 256, 0, stream>>>((const T*)x, x_stride, (const T*)weight, (const T*)bias, (T*)state, \
                                                       state_stride, channels, activation, (const SpanSeq*)s->buf,         \
                                                       (int)s->sequences, (int)s->tokens, tile, vec, (T*)out, out_stride); \
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
                                     int activation, const anna_mi_state_span* span, void* out, int64_t out_stride,
                                     void* stream) {
  ANNA_CHECK(span != nullptr, "causal_conv1d: null span");
  ANNA_CHECK(anna::valid_dtype(dtype), "causal_conv1d: dtype %d", dtype);
  ANNA_CHECK(width >= 2 && width <= 8, "causal_conv1d: width %lld, 2 to 8 are supported", (long long)width);
  ANNA_CHECK(channels >= 1 && channels <= (1 << 24), "causal_conv1d: %lld channels", (long long)channels);
  ANNA_CHECK(activation == 0 || activation == 1, "causal_conv1d: activation %d", activation);
  ANNA_CHECK(span->max_slot < slots, "causal_conv1d: slot %lld of a state of %lld", (long long)span->max_slot, (long long)slots);
  if (span->tokens == 0) return ANNA_MI_OK;
  ANNA_CHECK(span->tokens <= INT32_MAX && x && weight && out && span->buf && (state || span->max_slot < 0), "causal_conv1d: null pointer");
  ANNA_CHECK(x_stride >= channels || span->tokens == 1, "causal_conv1d: rows of x overlap");
  ANNA_CHECK(out_stride >= channels || span->tokens == 1, "causal_conv1d: rows of out overlap");
  ANNA_CHECK(slots <= 1 || state_stride_slot >= (width - 1) * channels, "causal_conv1d: rows of the state overlap");
  ANNA_DISPATCH_DTYPE(dtype, DT, return anna::launch<DT>(x, channels, x_stride, weight, width, bias, state, state_stride_slot,
                                                         activation, span, out, out_stride, anna::as_stream(stream)));
}
