// The gated delta rule token by token, for sequences of one or a few tokens (decode steps, drafts).
//
// A workgroup owns COLS columns of one head's state for all rows, in registers: thread (r, c) the
// columns 4 c .. 4 c + 3 of the rows r, r + RG, ...  Both products of a token with the state are sums over rows,
// and S'^T q = e^g S^T q + (k . q) u with u = beta (v - e^g S^T k), so one round of sums over the old state
// serves both.  While the state is on its way, the waves make the unit vectors and the factors of all tokens, a
// wave a token, in LDS.
//
// It is bound by the state's bytes (key_dim * value_dim * 4 read and written a sequence and head); a
// token's q, k and v are a hundredth of them.  64 sequences' next tokens, 32 value heads of 128 x 128 (0.27 GB): 59 us =
// 4.6 TB/s; a copy of 1 GiB runs at 5.2.  One sequence (4.2 MB): 5.3 us, the loads' latency and a launch.
#pragma once

#include "delta.hpp"

namespace anna {

template <int DK, int COLS> struct StepLds {
  static constexpr int TC = COLS / 4, SUMS = 8;  // threads on a row; S^T k and S^T q of four columns
  float part[2][4][TC][SUMS + 1];
  float ks[STEP_TOKENS][DK], qs[STEP_TOKENS][DK], vs[STEP_TOKENS][COLS];
  float decays[STEP_TOKENS], betas[STEP_TOKENS], kqs[STEP_TOKENS];
};

// Workgroup `block`: a slice of COLS columns of a sequence and value head
template <int DT, int DK, int COLS>
__device__ __forceinline__ void delta_step_block(const anna_mi_gated_delta_args& a, const SpanSeq* __restrict__ steps, int slices,
                                                 uint32_t block, StepLds<DK, COLS>& lds) {
  typedef typename Elem<DT>::T T;
  constexpr int TC = StepLds<DK, COLS>::TC, SUMS = StepLds<DK, COLS>::SUMS;
  constexpr int RG = 256 / TC;  // rows at a time
  constexpr int NR = DK / RG;   // rows of a thread
  auto &part = lds.part;
  auto &ks = lds.ks, &qs = lds.qs;
  auto& vs = lds.vs;
  auto &decays = lds.decays, &betas = lds.betas, &kqs = lds.kqs;

  const int tid = threadIdx.x, c = tid % TC, r = tid / TC, wave = tid / 64, lane = tid % 64;
  const uint32_t heads = (uint32_t)a.value_heads, slice = block % (uint32_t)slices, item = block / (uint32_t)slices;
  const uint32_t hv = item % heads, hk = hv / (heads / (uint32_t)a.key_heads);
  const int64_t HV = a.value_heads;
  const int dv = slices * COLS, col = slice * COLS + 4 * c;
  const SpanSeq seq = steps[item / heads];

  if ((uint32_t)seq.slot >= (uint32_t)a.slots) {  // a sequence of nobody
    for (int i = tid; i < seq.tokens * COLS; i += 256)
      ((T*)a.out)[((int64_t)(seq.first + i / COLS) * HV + hv) * dv + slice * COLS + i % COLS] = Elem<DT>::cvt(0.f);
    return;
  }
  float* state = a.state + seq.slot * a.state_stride_slot + (int64_t)hv * DK * dv + col;
  f32x4 S[NR];
#pragma unroll
  for (int i = 0; i < NR; i++) S[i] = seq.fresh ? f32x4{0.f, 0.f, 0.f, 0.f} : *(const f32x4*)(state + (int64_t)(r + RG * i) * dv);

  for (int t = wave; t < seq.tokens; t += 4) {
    const int64_t token = seq.first + t;
    const T* qp = (const T*)a.query + token * a.query_stride_token + hk * a.query_stride_head;
    const T* kp = (const T*)a.key + token * a.key_stride_token + hk * a.key_stride_head;
    const T* vp = (const T*)a.value + token * a.value_stride_token + hv * a.value_stride_head + slice * COLS;
    float k[DK / 64], q[DK / 64], kk = 0.f, qq = 0.f, kq = 0.f;
#pragma unroll
    for (int i = 0; i < DK / 64; i++) {
      k[i] = Elem<DT>::load(kp, lane + 64 * i);
      q[i] = Elem<DT>::load(qp, lane + 64 * i);
    }
#pragma unroll
    for (int i = 0; i < (COLS + 63) / 64; i++)
      if (lane + 64 * i < COLS) vs[t][lane + 64 * i] = Elem<DT>::load(vp, lane + 64 * i);
    const Gate gate = gate_of(a, token, hv);
#pragma unroll
    for (int i = 0; i < DK / 64; i++) {
      kk = fmaf(k[i], k[i], kk);
      qq = fmaf(q[i], q[i], qq);
      kq = fmaf(k[i], q[i], kq);
    }
    const float ck = a.normalize ? rsqrtf(wave_sum_rows(kk) + NORM_EPS) : 1.f;
    const float cq = a.scaling * (a.normalize ? rsqrtf(wave_sum_rows(qq) + NORM_EPS) : 1.f);
    kq = wave_sum_rows(kq) * ck * cq;
#pragma unroll
    for (int i = 0; i < DK / 64; i++) {
      ks[t][lane + 64 * i] = k[i] * ck;
      qs[t][lane + 64 * i] = q[i] * cq;
    }
    if (lane == 0) {
      decays[t] = expf(gate.g);
      betas[t] = gate.beta;
      kqs[t] = kq;
    }
  }
  __syncthreads();

  for (int t = 0; t < seq.tokens; t++) {
    float k[NR], sum[SUMS] = {};
#pragma unroll
    for (int i = 0; i < NR; i++) {
      k[i] = ks[t][r + RG * i];
      const float q = qs[t][r + RG * i];
#pragma unroll
      for (int j = 0; j < 4; j++) {
        sum[j] = fmaf(S[i][j], k[i], sum[j]);
        sum[4 + j] = fmaf(S[i][j], q, sum[4 + j]);
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
    if (lane < TC)
#pragma unroll
      for (int s = 0; s < SUMS; s++) mine[wave][c][s] = sum[s];
    __syncthreads();
#pragma unroll
    for (int s = 0; s < SUMS; s++) sum[s] = (mine[0][c][s] + mine[1][c][s]) + (mine[2][c][s] + mine[3][c][s]);

    const float e = decays[t], beta = betas[t];
    float u[4];
#pragma unroll
    for (int j = 0; j < 4; j++) u[j] = beta * (vs[t][4 * c + j] - e * sum[j]);
#pragma unroll
    for (int i = 0; i < NR; i++)
#pragma unroll
      for (int j = 0; j < 4; j++) S[i][j] = fmaf(k[i], u[j], e * S[i][j]);
    if (r == 0) {
      const float kq = kqs[t];
      uint32_t w[2];
#pragma unroll
      for (int j = 0; j < 4; j += 2)
        w[j / 2] = (uint32_t)Elem<DT>::cvt(fmaf(kq, u[j], e * sum[4 + j])) |
                   (uint32_t)Elem<DT>::cvt(fmaf(kq, u[j + 1], e * sum[5 + j])) << 16;
      *(uint2*)((T*)a.out + ((seq.first + (int64_t)t) * HV + hv) * dv + col) = make_uint2(w[0], w[1]);
    }
  }
#pragma unroll
  for (int i = 0; i < NR; i++) *(f32x4*)(state + (int64_t)(r + RG * i) * dv) = S[i];
}

}  // namespace anna
