// The gated delta rule in chunks of 64 tokens, for prompts.
//
// Within a chunk, with a_i the sum of the decays' logarithms up to token i and S the state in front of it,
//   u = T' (v - e^a K S),   T' = (1 + A)^-1 diag(beta),   A_ij = beta_i e^{a_i - a_j} k_i . k_j  (j < i)
//   out = e^a Q S + P u,    P_ij = e^{a_i - a_j} q_i . k_j  (j <= i)
//   S'  = e^{a_63} S + (e^{a_63 - a} K)^T u
// Everything that does not need S is computed for all chunks at once (delta_prepare_kernel, a workgroup a chunk and
// value head); the chunks of a sequence then follow each other (delta_chain_kernel), where a wave owns 16 columns of
// one head's state and needs no other wave: columns of S, u and out depend on the same column of v only.
//
// Precision: the state stays fp32.  Products run on the fp16 matrix instructions with fp32 sums; an fp32
// operand x enters as two fp16 values, hi = fp16(x / s) and lo = fp16(x / s - hi), 22 bits of it, with s a power
// of two that brings the largest of its column (of T': of the chunk) to 2^14, so values down to 2^-28 of the
// largest keep all 22 bits.  q and k are exact in one fp16 value once a row's power of two is taken out.
//
// A chunk with a token that is not finite (of the operands that a wave sees) is taken token by token: zeros above
// the diagonals times what is not finite would reach the tokens in front of it.
//
// Operands are held in the order of the matrix instruction's registers: fragment (mt, ks) of an M x K operand
// gives lane (n = lane % 16, g = lane / 16) the 8 values of row (mt, n) at k = 32 ks + 8 g + 0..7.  Rows of tile mt are
// numbered so that the instruction's result, rows 4 g + r of a tile in lane (n, g), is at once the other operand of
// the next product: row m of tile mt stands for index 32 (mt / 2) + 8 (m / 4) + 4 (mt % 2) + m % 4.
#include "delta.hpp"

namespace anna {

__host__ __device__ constexpr int row_of(int mt, int m) { return 32 * (mt / 2) + 8 * (m / 4) + 4 * (mt % 2) + m % 4; }

constexpr int FRAG = 1024;  // bytes of a fragment
constexpr int T_FRAGS = 6;  // of a lower triangular 64 x 64 operand: (0..3, 0), (2, 1), (3, 1)
__device__ __forceinline__ void t_frag(int f, int& mt, int& ks) {
  ks = f >= 4;
  mt = ks ? f - 2 : f;
}

// Factors of a chunk and value head: of K S, of Q S, of u on its way to the state, and {e^{a_63}, scale of T', of P}
struct Factors {
  float decayed_k[CHUNK], decayed_q[CHUNK], to_end[CHUNK];
  float end, t_scale, p_scale;
  int not_finite;  // a q, k, g or beta of the chunk is not
  float pad[60];
};

// The workspace: K, Q and K^T of every chunk and key head, T' (hi, lo), P (hi, and lo for fp16) and the factors
// of every chunk and value head
template <int DK> struct Places {
  static constexpr int64_t MAT = CHUNK * DK * 2;
  char* base;
  int64_t HK, HV, chunks;
  int p_parts;
  __host__ __device__ int64_t head_bytes() const { return T_FRAGS * FRAG * (2 + p_parts) + (int64_t)sizeof(Factors); }
  __host__ __device__ int64_t bytes() const { return chunks * (HK * 3 * MAT + HV * head_bytes()); }
  __device__ char* k(int64_t chunk, int64_t hk) const { return base + (chunk * HK + hk) * 3 * MAT; }
  __device__ char* q(int64_t chunk, int64_t hk) const { return k(chunk, hk) + MAT; }
  __device__ char* kt(int64_t chunk, int64_t hk) const { return k(chunk, hk) + 2 * MAT; }
  __device__ char* t(int64_t chunk, int64_t hv) const { return base + chunks * HK * 3 * MAT + (chunk * HV + hv) * head_bytes(); }
  __device__ char* p(int64_t chunk, int64_t hv) const { return t(chunk, hv) + 2 * T_FRAGS * FRAG; }
  __device__ Factors* factors(int64_t chunk, int64_t hv) const { return (Factors*)(p(chunk, hv) + p_parts * T_FRAGS * FRAG); }
};

// ---------------------------------------------------------------- powers of two

// {2^(14 - e), 2^(e - 14)} for a largest value of exponent e, within fp32's normal range; of 0 the smallest
struct Pow2 {
  float down, up;
};
__device__ __forceinline__ Pow2 pow2_of(float largest) {
  const uint32_t e = min(max((__float_as_uint(largest) >> 23) & 255u, 15u), 254u);
  return {__uint_as_float((268u - e) << 23), __uint_as_float((e - 14u) << 23)};
}

__device__ __forceinline__ f32x4 mfma16(f16x8 a, f16x8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ f32x4 mfma4(float a, float b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0); }

// hi and lo of eight values
__device__ __forceinline__ void split(const float (&x)[8], f16x8& hi, f16x8& lo) {
#pragma unroll
  for (int e = 0; e < 8; e++) {
    hi[e] = (_Float16)x[e];
    lo[e] = (_Float16)(x[e] - (float)hi[e]);
  }
}

// ---------------------------------------------------------------- what needs no state

template <int DT, int DK>
__global__ __launch_bounds__(256) void delta_prepare_kernel(const anna_mi_gated_delta_args a, const int32_t* __restrict__ buf,
                                                            int64_t sequences, const int32_t* __restrict__ chunks,
                                                            const Places<DK> ws) {
  typedef typename Elem<DT>::T T;
  constexpr int LD = DK + 8;    // halves of a row of K and Q in LDS
  constexpr int LF = CHUNK + 4; // floats of a row of A, T and P
  __shared__ _Float16 K[CHUNK][LD], Q[CHUNK][LD];
  __shared__ float A[CHUNK][LF], TI[CHUNK][LF];
  __shared__ double at[CHUNK];  // a
  __shared__ float kf[CHUNK], qf[CHUNK], beta[CHUNK], tops[2][4];
  __shared__ int not_finite;

  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, n = lane & 15, g = lane >> 4;
  const int64_t HV = a.value_heads, chunk = blockIdx.x / HV, hv = blockIdx.x % HV, hk = hv / (HV / a.key_heads);
  const bool writes_k = hv % (HV / a.key_heads) == 0;
  const SpanSeq seq = ((const SpanSeq*)buf)[chunks[2 * chunk]];
  if (seq.slot < 0) return;
  const int64_t first = seq.first + (int64_t)chunks[2 * chunk + 1] * CHUNK;
  const int tokens = min(CHUNK, seq.tokens - chunks[2 * chunk + 1] * CHUNK);
  if (tid == 0) not_finite = 0;
  __syncthreads();

  // rows of K and Q: a power of two taken out of each, what is left to make the unit vector kept as a factor
  constexpr int RL = DK / 8, RR = 256 / RL;  // lanes of a row, rows at a time
  for (int which = 0; which < 2; which++) {
    const T* src = (const T*)(which ? a.query : a.key);
    const int64_t st = which ? a.query_stride_token : a.key_stride_token, sh = which ? a.query_stride_head : a.key_stride_head;
#pragma unroll
    for (int i = 0; i < CHUNK / RR; i++) {
      const int row = tid / RL + RR * i, c = tid % RL * 8;
      float x[8] = {}, ss = 0.f, top = 0.f;
      if (row < tokens) {
        const u32x4 raw = *(const u32x4*)(src + (first + row) * st + hk * sh + c);
        const T* h = (const T*)&raw;
#pragma unroll
        for (int e = 0; e < 8; e++) x[e] = Elem<DT>::to_f32(h[e]);
      }
#pragma unroll
      for (int e = 0; e < 8; e++) {
        ss = fmaf(x[e], x[e], ss);
        top = fmaxf(top, fabsf(x[e]));
      }
#pragma unroll
      for (int off = 1; off < RL; off *= 2) {
        ss += __shfl_xor(ss, off, 64);
        top = fmaxf(top, __shfl_xor(top, off, 64));
      }
      // the largest value goes to 2^8: no sum of 128 products of two rows comes near fp32's limits, and fp16 holds
      // what is 2^-22 of the largest with all its bits
      const int e = top > 0.f && top < INFINITY ? 8 - ilogbf(top) : 0;
      f16x8 h8;
#pragma unroll
      for (int j = 0; j < 8; j++) h8[j] = (_Float16)ldexpf(x[j], e);
      *(f16x8*)&(which ? Q : K)[row][c] = h8;
      if (tid % RL == 0) {
        if (!isfinite(ss)) not_finite = 1;
        const float f = ldexpf(a.normalize ? rsqrtf(ss + NORM_EPS) : 1.f, -e);
        if (which) qf[row] = f * a.scaling;
        else kf[row] = f;
      }
    }
  }
  if (wave == 0) {  // decays: sums of logarithms in 64 bits, as their differences count; -inf stands for e^-10^4 = 0
    Gate gate{0.f, 0.f};
    if (lane < tokens) gate = gate_of(a, first + lane, hv);
    double s = gate.g < -1e4f ? -1e4 : (double)gate.g;
    if (!isfinite(s) || !isfinite(gate.beta)) not_finite = 1;
#pragma unroll
    for (int off = 1; off < 64; off *= 2) {
      const double o = __shfl_up(s, off, 64);
      if (lane >= off) s += o;
    }
    at[lane] = s;
    beta[lane] = gate.beta;
  }
  for (int i = tid; i < CHUNK * LF; i += 256) (&TI[0][0])[i] = 0.f;
  __syncthreads();

  // A and P, 16 rows a wave; P's rows are kept in registers until A has been used up
  f32x4 P[4];
  float p_top = 0.f;
  {
    f16x8 kr[DK / 32], qr[DK / 32];
#pragma unroll
    for (int s = 0; s < DK / 32; s++) {
      kr[s] = *(const f16x8*)&K[16 * wave + n][32 * s + 8 * g];
      qr[s] = *(const f16x8*)&Q[16 * wave + n][32 * s + 8 * g];
    }
#pragma unroll
    for (int ct = 0; ct < 4; ct++) {
      f32x4 kk = {0.f, 0.f, 0.f, 0.f}, qk = {0.f, 0.f, 0.f, 0.f};
      if (ct <= wave) {
#pragma unroll
        for (int s = 0; s < DK / 32; s++) {
          const f16x8 col = *(const f16x8*)&K[16 * ct + n][32 * s + 8 * g];
          kk = mfma16(kr[s], col, kk);
          qk = mfma16(qr[s], col, qk);
        }
      }
      const int j = 16 * ct + n;
      const double aj = at[j];
      const float cj = kf[j];
#pragma unroll
      for (int r = 0; r < 4; r++) {
        const int i = 16 * wave + 4 * g + r;
        const float d = i >= j ? expf((float)(at[i] - aj)) : 0.f;
        A[i][j] = i > j ? beta[i] * d * (kf[i] * kk[r] * cj) : 0.f;
        P[ct][r] = i >= j ? d * (qf[i] * qk[r] * cj) : 0.f;
        p_top = fmaxf(p_top, fabsf(P[ct][r]));
      }
    }
  }
  __syncthreads();

  // (1 + A)^-1: the diagonal blocks by substitution, a lane a column; then larger ones from products,
  // T21 = -T22 (A21 T11)
  if (wave == 0) {
    float x[16];
#pragma unroll
    for (int i = 0; i < 16; i++) {
      float s = i == n ? 1.f : 0.f;
#pragma unroll
      for (int k = 0; k < i; k++) s = fmaf(-A[16 * g + i][16 * g + k], x[k], s);
      x[i] = s;
      TI[16 * g + i][16 * g + n] = s;
    }
  }
  __syncthreads();
  // product of 16 x 16 blocks in LDS; the second form takes a result of the instruction as its right operand: its lane
  // (n, g) holds the rows 4 g + r
  auto block = [&](const float (*L)[LF], int lb, int lc, const float (*R)[LF], int rb, int rc, f32x4 c) {
#pragma unroll
    for (int k = 0; k < 4; k++) c = mfma4(L[16 * lb + n][16 * lc + 4 * g + k], R[16 * rb + 4 * g + k][16 * rc + n], c);
    return c;
  };
  auto times = [&](const float (*L)[LF], int lb, int lc, f32x4 x, f32x4 c) {
#pragma unroll
    for (int k = 0; k < 4; k++) c = mfma4(L[16 * lb + n][16 * lc + 4 * g + k], x[k], c);
    return c;
  };
  const f32x4 zero = {0.f, 0.f, 0.f, 0.f};
  if (wave < 2) {
    const int b = 2 * wave;
    const f32x4 x = block(A, b + 1, b, TI, b, b, zero), y = times(TI, b + 1, b + 1, x, zero);
#pragma unroll
    for (int r = 0; r < 4; r++) TI[16 * (b + 1) + 4 * g + r][16 * b + n] = -y[r];
  }
  __syncthreads();
  {
    const int b = wave & 1, row = 2 + (wave >> 1);  // block column, block row of the result
    f32x4 x2 = zero, x3 = zero;
    for (int c = b; c < 2; c++) {
      x2 = block(A, 2, c, TI, c, b, x2);
      x3 = block(A, 3, c, TI, c, b, x3);
    }
    f32x4 y = times(TI, row, 2, x2, zero);
    if (row == 3) y = times(TI, row, 3, x3, y);
    __syncthreads();  // A and T11, T22 are read
#pragma unroll
    for (int r = 0; r < 4; r++) TI[16 * row + 4 * g + r][16 * b + n] = -y[r];
#pragma unroll
    for (int ct = 0; ct < 4; ct++)
#pragma unroll
      for (int r = 0; r < 4; r++) A[16 * wave + 4 * g + r][16 * ct + n] = P[ct][r];  // P in A's place
  }
  __syncthreads();

  float t_top = 0.f;
  for (int i = tid; i < CHUNK * CHUNK; i += 256) t_top = fmaxf(t_top, fabsf(TI[i / CHUNK][i % CHUNK] * beta[i % CHUNK]));
  t_top = wave_max(t_top);
  p_top = wave_max(p_top);
  if (lane == 0) {
    tops[0][wave] = t_top;
    tops[1][wave] = p_top;
  }
  __syncthreads();
  const Pow2 ts = pow2_of(fmaxf(fmaxf(tops[0][0], tops[0][1]), fmaxf(tops[0][2], tops[0][3])));
  const Pow2 ps = pow2_of(fmaxf(fmaxf(tops[1][0], tops[1][1]), fmaxf(tops[1][2], tops[1][3])));

  char* const t_to = ws.t(chunk, hv);
  char* const p_to = ws.p(chunk, hv);
  for (int f = wave; f < T_FRAGS; f += 4) {
    int mt, ks;
    t_frag(f, mt, ks);
    const int i = row_of(mt, n), j = 32 * ks + 8 * g;
    float x[8], y[8];
#pragma unroll
    for (int e = 0; e < 8; e++) {
      x[e] = TI[i][j + e] * beta[j + e] * ts.down;
      y[e] = A[i][j + e] * ps.down;
    }
    f16x8 hi, lo;
    split(x, hi, lo);
    *(f16x8*)(t_to + (2 * f) * FRAG + 16 * lane) = hi;
    *(f16x8*)(t_to + (2 * f + 1) * FRAG + 16 * lane) = lo;
    split(y, hi, lo);
    *(f16x8*)(p_to + ws.p_parts * f * FRAG + 16 * lane) = hi;
    if (ws.p_parts == 2) *(f16x8*)(p_to + (2 * f + 1) * FRAG + 16 * lane) = lo;
  }
  if (tid < CHUNK) {
    Factors* to = ws.factors(chunk, hv);
    const float e = expf((float)at[tid]);
    to->decayed_k[tid] = e * kf[tid];
    to->decayed_q[tid] = e * qf[tid];
    to->to_end[tid] = expf((float)(at[CHUNK - 1] - at[tid])) * kf[tid];
    if (tid == 0) {
      to->end = expf((float)at[CHUNK - 1]);
      to->t_scale = ts.up;
      to->p_scale = ps.up;
      to->not_finite = not_finite;
    }
  }
  if (!writes_k) return;
  char* const k_to = ws.k(chunk, hk);
  char* const q_to = ws.q(chunk, hk);
  char* const kt_to = ws.kt(chunk, hk);
  for (int f = wave; f < 4 * (DK / 32); f += 4) {
    const int mt = f / (DK / 32), ks = f % (DK / 32), i = row_of(mt, n), d = 32 * ks + 8 * g;
    *(f16x8*)(k_to + f * FRAG + 16 * lane) = *(const f16x8*)&K[i][d];
    *(f16x8*)(q_to + f * FRAG + 16 * lane) = *(const f16x8*)&Q[i][d];
  }
  for (int f = wave; f < DK / 16 * 2; f += 4) {
    const int mt = f / 2, ks = f % 2, d = row_of(mt, n), i = 32 * ks + 8 * g;
    f16x8 h;
#pragma unroll
    for (int e = 0; e < 8; e++) h[e] = K[i + e][d];
    *(f16x8*)(kt_to + f * FRAG + 16 * lane) = h;
  }
}

// ---------------------------------------------------------------- the chain of states

__device__ __forceinline__ f16x8 frag(const char* base, int f, int lane) { return *(const f16x8*)(base + f * FRAG + 16 * lane); }

// Largest of a column, over the four lanes that hold it
__device__ __forceinline__ float column_max(float v) {
  v = fmaxf(v, lane_xor16(v));
  return fmaxf(v, lane_xor32(v));
}
// Tiles 2 s and 2 s + 1 of a product's result as the operand of the next: hi and lo of x * down
__device__ __forceinline__ void operand(f32x4 x, f32x4 y, float down, f16x8& hi, f16x8& lo) {
  const float f[8] = {x[0] * down, x[1] * down, x[2] * down, x[3] * down, y[0] * down, y[1] * down, y[2] * down, y[3] * down};
  split(f, hi, lo);
}
__device__ __forceinline__ float largest(const f32x4& x) { return fmaxf(fmaxf(fabsf(x[0]), fabsf(x[1])), fmaxf(fabsf(x[2]), fabsf(x[3]))); }

// Tokens one after the other, on the chain's layout of the state: lane (n, g) holds rows row_of(t, 4 g + r) of column n
template <int DT, int DK>
__device__ __forceinline__ void delta_tokens(const anna_mi_gated_delta_args& a, int64_t first, int tokens, int64_t hv, int64_t hk,
                                          int64_t col, int g, f32x4 (&S)[DK / 16]) {
  typedef typename Elem<DT>::T T;
  auto total = [](float v) {
    v += lane_xor16(v);
    return v + lane_xor32(v);
  };
  for (int64_t token = first; token < first + tokens; token++) {
    const T* qp = (const T*)a.query + token * a.query_stride_token + hk * a.query_stride_head;
    const T* kp = (const T*)a.key + token * a.key_stride_token + hk * a.key_stride_head;
    const float v = Elem<DT>::load((const T*)a.value, token * a.value_stride_token + hv * a.value_stride_head + col);
    const Gate gate = gate_of(a, token, hv);
    float k[DK / 4], q[DK / 4], kk = 0.f, qq = 0.f, sk = 0.f, sq = 0.f, kq = 0.f;
#pragma unroll
    for (int i = 0; i < DK / 4; i++) {
      k[i] = Elem<DT>::load(kp, row_of(i / 4, 4 * g + i % 4));
      q[i] = Elem<DT>::load(qp, row_of(i / 4, 4 * g + i % 4));
      kk = fmaf(k[i], k[i], kk);
      qq = fmaf(q[i], q[i], qq);
    }
    const float ck = a.normalize ? rsqrtf(total(kk) + NORM_EPS) : 1.f;
    const float cq = a.scaling * (a.normalize ? rsqrtf(total(qq) + NORM_EPS) : 1.f);
#pragma unroll
    for (int i = 0; i < DK / 4; i++) {
      k[i] *= ck;
      q[i] *= cq;
      sk = fmaf(S[i / 4][i % 4], k[i], sk);
      sq = fmaf(S[i / 4][i % 4], q[i], sq);
      kq = fmaf(k[i], q[i], kq);
    }
    const float e = expf(gate.g), u = gate.beta * (v - e * total(sk));
    const float o = fmaf(total(kq), u, e * total(sq));
#pragma unroll
    for (int i = 0; i < DK / 4; i++) S[i / 4][i % 4] = fmaf(k[i], u, e * S[i / 4][i % 4]);
    if (g == 0) ((T*)a.out)[(token * a.value_heads + hv) * a.value_dim + col] = Elem<DT>::cvt(o);
  }
}

template <int DT, int DK>
__global__ __launch_bounds__(64) void delta_chain_kernel(const anna_mi_gated_delta_args a, const int32_t* __restrict__ buf,
                                                         int64_t sequences, const int32_t* __restrict__ chains,
                                                         const Places<DK> ws) {
  typedef typename Elem<DT>::T T;
  constexpr int NT = DK / 16, KS = DK / 32;
  constexpr bool EXACT_OUT = DT == ANNA_MI_F16;  // an fp16 output shows the second parts of its operands
  const int lane = threadIdx.x, n = lane & 15, g = lane >> 4;
  const int64_t HV = a.value_heads, DV = a.value_dim;
  const int slices = (int)(DV / 16);
  const int64_t item = blockIdx.x / slices, hv = item % HV, hk = hv / (HV / a.key_heads);
  const int64_t col = blockIdx.x % slices * 16 + n;
  const int32_t* chain = chains + 2 * (item / HV);
  const SpanSeq seq = ((const SpanSeq*)buf)[chain[0]];
  T* const out = (T*)a.out + hv * DV + col;
  if (seq.slot < 0) {
    for (int t = g; t < seq.tokens; t += 4) out[(seq.first + (int64_t)t) * HV * DV] = Elem<DT>::cvt(0.f);
    return;
  }
  float* const state = a.state + seq.slot * a.state_stride_slot + hv * DK * DV + col;
  f32x4 S[NT];
#pragma unroll
  for (int t = 0; t < NT; t++)
#pragma unroll
    for (int r = 0; r < 4; r++) S[t][r] = seq.fresh ? 0.f : state[row_of(t, 4 * g + r) * DV];

  const f32x4 zero = {0.f, 0.f, 0.f, 0.f};
  const int count = (seq.tokens + CHUNK - 1) / CHUNK;
  for (int c = 0; c < count; c++) {
    const int64_t chunk = chain[1] + (int64_t)c, first = seq.first + (int64_t)c * CHUNK;
    const int tokens = min(CHUNK, seq.tokens - c * CHUNK);
    const char *kf = ws.k(chunk, hk), *qf = ws.q(chunk, hk), *ktf = ws.kt(chunk, hk), *tf = ws.t(chunk, hv), *pf = ws.p(chunk, hv);
    const Factors* fac = ws.factors(chunk, hv);
    float v[4][4], zeros = 0.f;
#pragma unroll
    for (int mt = 0; mt < 4; mt++)
#pragma unroll
      for (int r = 0; r < 4; r++) {
        const int t = row_of(mt, 4 * g + r);
        v[mt][r] = t < tokens ? Elem<DT>::load((const T*)a.value, (first + t) * a.value_stride_token + hv * a.value_stride_head + col) : 0.f;
        zeros = fmaf(v[mt][r], 0.f, zeros);
      }
    if (fac->not_finite || __any(zeros != 0.f)) {  // a NaN differs from 0 too
      delta_tokens<DT, DK>(a, first, tokens, hv, hk, col, g, S);
      continue;
    }

    // K S and Q S
    float top = 0.f;
#pragma unroll
    for (int t = 0; t < NT; t++) top = fmaxf(top, largest(S[t]));
    const Pow2 ss = pow2_of(column_max(top));
    f32x4 ks[4] = {zero, zero, zero, zero}, qs[4] = {zero, zero, zero, zero};
#pragma unroll
    for (int s = 0; s < KS; s++) {
      f16x8 hi, lo;
      operand(S[2 * s], S[2 * s + 1], ss.down, hi, lo);
#pragma unroll
      for (int mt = 0; mt < 4; mt++) {
        const f16x8 k = frag(kf, mt * KS + s, lane), q = frag(qf, mt * KS + s, lane);
        ks[mt] = mfma16(k, hi, ks[mt]);
        ks[mt] = mfma16(k, lo, ks[mt]);
        qs[mt] = mfma16(q, hi, qs[mt]);
        if constexpr (EXACT_OUT) qs[mt] = mfma16(q, lo, qs[mt]);
      }
    }
    // v - e^a K S
    f32x4 x[4];
    top = 0.f;
#pragma unroll
    for (int mt = 0; mt < 4; mt++) {
      const f32x4 f = *(const f32x4*)&fac->decayed_k[row_of(mt, 4 * g)];
#pragma unroll
      for (int r = 0; r < 4; r++) x[mt][r] = fmaf(-f[r] * ss.up, ks[mt][r], v[mt][r]);
      top = fmaxf(top, largest(x[mt]));
    }
    // u = T' x
    const Pow2 xs = pow2_of(column_max(top));
    f32x4 u[4] = {zero, zero, zero, zero};
    {
      f16x8 hi[2], lo[2];
      operand(x[0], x[1], xs.down, hi[0], lo[0]);
      operand(x[2], x[3], xs.down, hi[1], lo[1]);
#pragma unroll
      for (int f = 0; f < T_FRAGS; f++) {
        const int s = f >= 4, mt = s ? f - 2 : f;
        const f16x8 th = frag(tf, 2 * f, lane), tl = frag(tf, 2 * f + 1, lane);
        u[mt] = mfma16(tl, hi[s], u[mt]);
        u[mt] = mfma16(th, lo[s], u[mt]);
        u[mt] = mfma16(th, hi[s], u[mt]);
      }
    }
    const float us = fac->t_scale * xs.up;
    top = 0.f;
#pragma unroll
    for (int mt = 0; mt < 4; mt++) {
#pragma unroll
      for (int r = 0; r < 4; r++) u[mt][r] *= us;
      top = fmaxf(top, largest(u[mt]));
    }
    // out = e^a Q S + P u
    const Pow2 os = pow2_of(column_max(top));
    f32x4 o[4] = {zero, zero, zero, zero};
    {
      f16x8 hi[2], lo[2];
      operand(u[0], u[1], os.down, hi[0], lo[0]);
      operand(u[2], u[3], os.down, hi[1], lo[1]);
#pragma unroll
      for (int f = 0; f < T_FRAGS; f++) {
        const int s = f >= 4, mt = s ? f - 2 : f;
        const f16x8 ph = frag(pf, (EXACT_OUT ? 2 : 1) * f, lane);
        if constexpr (EXACT_OUT) {
          o[mt] = mfma16(frag(pf, 2 * f + 1, lane), hi[s], o[mt]);
          o[mt] = mfma16(ph, lo[s], o[mt]);
        }
        o[mt] = mfma16(ph, hi[s], o[mt]);
      }
    }
    const float ps = fac->p_scale * os.up;
#pragma unroll
    for (int mt = 0; mt < 4; mt++) {
      const f32x4 f = *(const f32x4*)&fac->decayed_q[row_of(mt, 4 * g)];
#pragma unroll
      for (int r = 0; r < 4; r++) {
        const int t = row_of(mt, 4 * g + r);
        if (t < tokens) out[(first + t) * HV * DV] = Elem<DT>::cvt(fmaf(f[r] * ss.up, qs[mt][r], ps * o[mt][r]));
      }
    }
    // S' = e^{a_63} S + K^T (e^{a_63 - a} u)
    top = 0.f;
#pragma unroll
    for (int mt = 0; mt < 4; mt++) {
      u[mt] *= *(const f32x4*)&fac->to_end[row_of(mt, 4 * g)];
      top = fmaxf(top, largest(u[mt]));
    }
    const Pow2 es = pow2_of(column_max(top));
    const float end = fac->end;
    f16x8 hi[2], lo[2];
    operand(u[0], u[1], es.down, hi[0], lo[0]);
    operand(u[2], u[3], es.down, hi[1], lo[1]);
#pragma unroll
    for (int t = 0; t < NT; t++) {
      f32x4 s = zero;
#pragma unroll
      for (int j = 0; j < 2; j++) {
        const f16x8 k = frag(ktf, 2 * t + j, lane);
        s = mfma16(k, lo[j], s);
        s = mfma16(k, hi[j], s);
      }
#pragma unroll
      for (int r = 0; r < 4; r++) S[t][r] = fmaf(s[r], es.up, S[t][r] * end);
    }
  }
#pragma unroll
  for (int t = 0; t < NT; t++)
#pragma unroll
    for (int r = 0; r < 4; r++) state[row_of(t, 4 * g + r) * DV] = S[t][r];
}

// ---------------------------------------------------------------- host

template <int DK> static Places<DK> places(const anna_mi_gated_delta_args& a, const anna_mi_state_span& s) {
  return {(char*)a.workspace, a.key_heads, a.value_heads, s.chunks, a.dtype == ANNA_MI_F16 ? 2 : 1};
}

template <int DT, int DK>
static int delta_chunks(const anna_mi_gated_delta_args& a, const anna_mi_state_span& s, hipStream_t stream) {
  const Places<DK> ws = places<DK>(a, s);
  const int32_t* chains = s.buf + 4 * s.sequences + s.steps;
  const int32_t* chunks = chains + 2 * s.chains;
  const int64_t prepare = s.chunks * a.value_heads, chain = s.chains * a.value_heads * (a.value_dim / 16);
  ANNA_CHECK(prepare <= INT32_MAX / 256 && chain <= INT32_MAX / 64, "gated delta rule: too many tokens and heads for a launch");
  delta_prepare_kernel<DT, DK><<<prepare, 256, 0, stream>>>(a, s.buf, s.sequences, chunks, ws);
  ANNA_LAUNCH_CHECK("delta_prepare");
  delta_chain_kernel<DT, DK><<<chain, 64, 0, stream>>>(a, s.buf, s.sequences, chains, ws);
  ANNA_LAUNCH_CHECK("delta_chain");
  return ANNA_MI_OK;
}

static int check_delta(const anna_mi_gated_delta_args* args, const anna_mi_state_span* span) {
  ANNA_CHECK(args != nullptr && span != nullptr, "gated delta rule: null args or span");
  const anna_mi_gated_delta_args& a = *args;
  ANNA_CHECK(a.dtype == ANNA_MI_BF16 || a.dtype == ANNA_MI_F16, "gated delta rule: dtype %d", a.dtype);
  ANNA_CHECK(valid_dtype(a.gates_dtype), "gated delta rule: gates_dtype %d", a.gates_dtype);
  ANNA_CHECK(a.key_dim == 64 || a.key_dim == 128, "gated delta rule: key_dim %lld, 64 and 128 are supported", (long long)a.key_dim);
  ANNA_CHECK(a.value_dim >= 32 && a.value_dim <= 256 && a.value_dim % 32 == 0,
             "gated delta rule: value_dim %lld, multiples of 32 up to 256 are supported", (long long)a.value_dim);
  ANNA_CHECK(a.key_heads >= 1 && a.value_heads >= a.key_heads && a.value_heads % a.key_heads == 0 && a.value_heads <= 65536,
             "gated delta rule: %lld value heads on %lld key heads", (long long)a.value_heads, (long long)a.key_heads);
  ANNA_CHECK(span->tokens >= 0 && span->tokens <= INT32_MAX, "gated delta rule: %lld tokens", (long long)span->tokens);
  ANNA_CHECK(span->max_slot < a.slots, "gated delta rule: slot %lld of a state of %lld", (long long)span->max_slot, (long long)a.slots);
  return ANNA_MI_OK;
}

}  // namespace anna

extern "C" {

int64_t anna_mi_gated_delta_workspace(const anna_mi_gated_delta_args* args, const anna_mi_state_span* span) {
  if (anna::check_delta(args, span) != ANNA_MI_OK) return 0;
  return args->key_dim == 64 ? anna::places<64>(*args, *span).bytes() : anna::places<128>(*args, *span).bytes();
}

int anna_mi_gated_delta(const anna_mi_gated_delta_args* args, const anna_mi_state_span* span, void* stream) {
  if (const int rc = anna::check_delta(args, span)) return rc;
  const anna_mi_gated_delta_args& a = *args;
  if (span->tokens == 0) return ANNA_MI_OK;
  ANNA_CHECK(a.query && a.key && a.value && a.decay && a.beta && a.out && span->buf && (a.state || span->max_slot < 0),
             "gated delta rule: null pointer");
  ANNA_CHECK(!a.a_log == !a.dt_bias, "gated delta rule: a_log and dt_bias go together");
  auto rows16 = [](const void* p, int64_t st, int64_t sh) { return (uintptr_t)p % 16 == 0 && st % 8 == 0 && sh % 8 == 0; };
  ANNA_CHECK(rows16(a.query, a.query_stride_token, a.query_stride_head) && rows16(a.key, a.key_stride_token, a.key_stride_head) &&
                 rows16(a.value, a.value_stride_token, a.value_stride_head),
             "gated delta rule: rows of query, key and value must be 16-byte aligned");
  ANNA_CHECK((uintptr_t)a.state % 16 == 0 && a.state_stride_slot % 4 == 0, "gated delta rule: states must be 16-byte aligned");
  ANNA_CHECK(a.slots <= 1 || a.state_stride_slot >= a.value_heads * a.key_dim * a.value_dim, "gated delta rule: states overlap");
  ANNA_CHECK(span->chunks == 0 || (a.workspace && (uintptr_t)a.workspace % 256 == 0), "gated delta rule: no workspace, or not 256-byte aligned");
  hipStream_t st = anna::as_stream(stream);
  if (const int rc = anna::delta_step(a, *span, st)) return rc;
  if (span->chains == 0) return ANNA_MI_OK;
  ANNA_DISPATCH_DTYPE(a.dtype, DT, {
    if constexpr (DT != ANNA_MI_F32)
      return a.key_dim == 64 ? anna::delta_chunks<DT, 64>(a, *span, st) : anna::delta_chunks<DT, 128>(a, *span, st);
  });
  return ANNA_MI_OK;
}

}  // extern "C"
