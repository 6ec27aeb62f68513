// The gated delta rule token by token, for sequences of one or a few tokens (decode steps, drafts).
//
// A workgroup owns COLS columns of one head's state for all rows, in registers: thread (r, c) the
// columns 4 c .. 4 c + 3 of the rows r, r + RG, ...  Both products of a token with the state are sums over rows,
// and S'^T q = e^g S^T q + (k . q) u with u = beta (v - e^g S^T k), so one round of sums over the old state
// serves both.
//
// It is bound by the state's bytes (key_dim * value_dim * 4 read and written a sequence and head); a
// token's q, k and v are a hundredth of them.
#include "delta.hpp"

namespace anna {

template <int DT, int DK, int COLS>
__global__ __launch_bounds__(256) void delta_step_kernel(const anna_mi_gated_delta_args a, const int32_t* __restrict__ buf,
                                                         int64_t sequences, int slices) {
  typedef typename Elem<DT>::T T;
  constexpr int TC = COLS / 4;     // threads on a row
  constexpr int RG = 256 / TC;     // rows at a time
  constexpr int NR = DK / RG;      // rows of a thread
  constexpr int SUMS = 8;          // S^T k and S^T q of four columns
  __shared__ float part[2][4][TC][SUMS + 1];

  const int tid = threadIdx.x, c = tid % TC, r = tid / TC, wave = tid / 64;
  const uint32_t heads = (uint32_t)a.value_heads, slice = blockIdx.x % (uint32_t)slices, item = blockIdx.x / (uint32_t)slices;
  const uint32_t hv = item % heads, hk = hv / (heads / (uint32_t)a.key_heads);
  const int64_t HV = a.value_heads;
  const int dv = slices * COLS, col = slice * COLS + 4 * c;
  const SpanSeq seq = ((const SpanSeq*)buf)[buf[4 * sequences + item / heads]];

  if (seq.slot < 0) {  // a sequence of nobody
    for (int i = tid; i < seq.tokens * COLS; i += 256)
      ((T*)a.out)[((int64_t)(seq.first + i / COLS) * HV + hv) * dv + slice * COLS + i % COLS] = Elem<DT>::cvt(0.f);
    return;
  }
  float* state = a.state + seq.slot * a.state_stride_slot + hv * DK * dv + col;
  f32x4 S[NR];
#pragma unroll
  for (int i = 0; i < NR; i++) S[i] = seq.fresh ? f32x4{0.f, 0.f, 0.f, 0.f} : *(const f32x4*)(state + (int64_t)(r + RG * i) * dv);

  for (int t = 0; t < seq.tokens; t++) {
    const int64_t token = seq.first + t;
    const T* qp = (const T*)a.query + token * a.query_stride_token + hk * a.query_stride_head;
    const T* kp = (const T*)a.key + token * a.key_stride_token + hk * a.key_stride_head;
    const T* vp = (const T*)a.value + token * a.value_stride_token + hv * a.value_stride_head + col;
    // every wave for itself: |k|^2, |q|^2, k . q
    float kk = 0.f, qq = 0.f, kq = 0.f;
#pragma unroll
    for (int i = 0; i < DK / 64; i++) {
      const float x = Elem<DT>::load(kp, (tid & 63) + 64 * i), y = Elem<DT>::load(qp, (tid & 63) + 64 * i);
      kk = fmaf(x, x, kk);
      qq = fmaf(y, y, qq);
      kq = fmaf(x, y, kq);
    }
    float k[NR], q[NR], v[4], sum[SUMS] = {};
#pragma unroll
    for (int i = 0; i < NR; i++) {
      k[i] = Elem<DT>::load(kp, r + RG * i);
      q[i] = Elem<DT>::load(qp, r + RG * i);
    }
#pragma unroll
    for (int j = 0; j < 4; j++) v[j] = Elem<DT>::load(vp, j);
    const Gate gate = gate_of(a, token, hv);
    const float ck = a.normalize ? rsqrtf(wave_sum_rows(kk) + NORM_EPS) : 1.f;
    const float cq = a.scaling * (a.normalize ? rsqrtf(wave_sum_rows(qq) + NORM_EPS) : 1.f);
    kq = wave_sum_rows(kq) * ck * cq;
#pragma unroll
    for (int i = 0; i < NR; i++) {
      k[i] *= ck;
      q[i] *= cq;
#pragma unroll
      for (int j = 0; j < 4; j++) {
        sum[j] = fmaf(S[i][j], k[i], sum[j]);
        sum[4 + j] = fmaf(S[i][j], q[i], sum[4 + j]);
      }
    }
    // over the row groups: of a wave, then of the four waves
#pragma unroll
    for (int s = 0; s < SUMS; s++) {
      if constexpr (TC <= 8) sum[s] += dpp_move<0x128>(sum[s]);  // row_ror 8: lane ^ 8
      if constexpr (TC <= 16) sum[s] += lane_xor16(sum[s]);
      sum[s] += lane_xor32(sum[s]);
    }
    auto& mine = part[t & 1];
    if ((tid & 63) < TC)
#pragma unroll
      for (int s = 0; s < SUMS; s++) mine[wave][c][s] = sum[s];
    __syncthreads();
#pragma unroll
    for (int s = 0; s < SUMS; s++) sum[s] = (mine[0][c][s] + mine[1][c][s]) + (mine[2][c][s] + mine[3][c][s]);

    const float e = expf(gate.g);
    float u[4];
#pragma unroll
    for (int j = 0; j < 4; j++) u[j] = gate.beta * (v[j] - e * sum[j]);
#pragma unroll
    for (int i = 0; i < NR; i++)
#pragma unroll
      for (int j = 0; j < 4; j++) S[i][j] = fmaf(k[i], u[j], e * S[i][j]);
    if (r == 0) {
      T* out = (T*)a.out + (token * HV + hv) * dv + col;
#pragma unroll
      for (int j = 0; j < 4; j++) out[j] = Elem<DT>::cvt(fmaf(kq, u[j], e * sum[4 + j]));
    }
  }
#pragma unroll
  for (int i = 0; i < NR; i++) *(f32x4*)(state + (int64_t)(r + RG * i) * dv) = S[i];
}

int delta_step(const anna_mi_gated_delta_args& a, const anna_mi_state_span& s, hipStream_t stream) {
  constexpr int COLS = 32;
  const int slices = (int)(a.value_dim / COLS);
  const int64_t grid = s.steps * a.value_heads * slices;
  if (grid == 0) return ANNA_MI_OK;
  ANNA_CHECK(grid <= INT32_MAX / 256, "gated delta rule: too many sequences and heads for a launch");
  ANNA_DISPATCH_DTYPE(a.dtype, DT, {
    if constexpr (DT != ANNA_MI_F32) {
      if (a.key_dim == 64) delta_step_kernel<DT, 64, COLS><<<grid, 256, 0, stream>>>(a, s.buf, s.sequences, slices);
      else delta_step_kernel<DT, 128, COLS><<<grid, 256, 0, stream>>>(a, s.buf, s.sequences, slices);
    }
  });
  ANNA_LAUNCH_CHECK("delta_step");
  return ANNA_MI_OK;
}

}  // namespace anna
