// The gated delta rule in chunks of 64 tokens, for prompts.
//
// Within a chunk, with a_i the sum of the decays' logarithms up to token i and S the state in front of it,
//   u = T' (v - e^a K S),   T' = (1 + A)^-1 diag(beta),   A_ij = beta_i e^{a_i - a_j} k_i . k_j  (j < i)
//   out = e^a Q S + P u,    P_ij = e^{a_i - a_j} q_i . k_j  (j <= i)
//   S'  = e^{a_63} S + (e^{a_63 - a} K)^T u
// Everything that does not need S is computed for all chunks at once (delta_prepare_kernel, a workgroup a chunk and
// key head); the chunks of a sequence then follow each other (delta_chain_kernel), where a wave owns 16 columns of
// one head's state and needs no other wave: columns of S, u and out depend on the same column of v only.
//
// Precision: the state stays fp32.  Products run on the fp16 matrix instructions with fp32 sums; an fp32
// operand x enters as two fp16 values, hi = fp16(x / s) and lo = fp16(2^11 (x / s - hi)), 22 bits of it or 2^-36 where that
// is more, with s a power of two of its column (of T' and P: of the chunk); what lo is a factor of is summed first, and
// brought down by 2^11 in front of the other sums.  q and k are exact in one fp16 value once a row's power of two is
// taken out.
//
// A column's unit s comes from the largest of its state and the chunk's values, which may be far above what a token sees
// of them: an outlier that comes later, a state that a decay has made small.  What a token sees is
//   n_i = max(e^{g_i} n_{i-1}, |k_i| beta_i |v_i|),   n_{-1} the state's largest,
// and 2^-36 of the unit is below the roundings of fp32 sums of that size where n_i is at least 2^-14 units (times
// |k| T', and again |k|, where these are above 1).  A chunk with a smaller n_i is taken token by token, from the state that the wave still has.
// Most columns are fine at a glance: by the old state times the smallest e^a, or the smallest |v| times the smallest |k| beta.
// The loop over n_i runs for the others, for about 1 us: with normal values behind a SiLU and decays of e^-0.06 to e^-2.3 a
// token, in one chunk of a hundred at most, and no chunk goes token by token.  Without the factor 2^11 it would run in
// nearly all of them from e^-0.26 on, and one in five would go token by token at the other end.
//
// Zeros above the diagonals times what is not finite would reach the tokens in front of it.  It also reaches the whole
// of its column's update, where a wave sees it and also takes the chunk token by token.
//
// Operands are held in the order of the matrix instruction's registers: fragment (mt, ks) of an M x K operand
// gives lane (n = lane % 16, g = lane / 16) the 8 values of row (mt, n) at k = 32 ks + 8 g + 0..7.  Rows of tile mt are
// numbered so that the instruction's result, rows 4 g + r of a tile in lane (n, g), is at once the other operand of
// the next product: row m of tile mt stands for index 32 (mt / 2) + 8 (m / 4) + 4 (mt % 2) + m % 4.
//
// What bounds it, 16 key and 32 value heads of 128, bf16.  One sequence of 16384 tokens: preparation 112 us, chain 500.
// The preparation writes 0.3 GB of workspace (58 us at a copy's rate); the rest is latency, about 36000 cycles a
// workgroup of loads, products and the inverse's steps with three workgroups a compute unit to cover for each other (two: 121 us).
// The chain is 256 chunks in a row at 2.0 us each on every compute unit: 82 matrix instructions of the state's
// wave are a quarter of that, some 400 vector instructions that make their operands (splits, scales) a third; the bytes alone
// would take 80 us.  (1.6 us with outputs from one term and terms of one scale, 1.8 with both terms.)
// Eight sequences of 25344 tokens together, fp16: preparation 164 us, chain 390 (350 with terms of one scale). Four waves a
// compute unit there read all operands from LDS, 3.3 to 3.6 us a chunk, vector unit 48% and matrix cores 27% busy, a tenth of
// the cycles with LDS's conflicts.
// Two column groups a wave, which halves what is read, took 650 for 350: the vector unit of half the SIMDs is then too little.
// A wave more for every group's output, with operands in single buffers that the output's waves fill, took 430 for 350.
#include <algorithm>
#include <type_traits>

#include "delta_step.hpp"

namespace anna {

__host__ __device__ constexpr int row_of(int mt, int m) { return 32 * (mt / 2) + 8 * (m / 4) + 4 * (mt % 2) + m % 4; }

constexpr int FRAG = 1024;  // bytes of a fragment
constexpr int T_FRAGS = 6;  // of a lower triangular 64 x 64 operand: (0..3, 0), (2, 1), (3, 1)
__device__ __forceinline__ void t_frag(int f, int& mt, int& ks) {
  ks = f >= 4;
  mt = ks ? f - 2 : f;
}

// Factors of a chunk and value head.  x is taken times 2^11, and down by a power of two where keys are longer than 1: e^a and
// k's with that for K S, and it alone for v; of (T' / its scale) x on its way to the state, with 2^11 for its two terms; e^a for
// Q S; q's for the output (P and Q are without them, so rows of any size keep their bits); e^{a_63}; of P times
// what `U_DOWN` leaves of (T' / its scale) x, which is of x's size whatever beta is.  For the n_i: e^g and |k| beta of
// every token, the smallest of that and of e^a, and what no n_i may be below.  For tokens one by one: K's and Q's factors.
struct Factors {
  float decayed_k[CHUNK], to_end[CHUNK], decay[CHUNK], q[CHUNK], step[CHUNK], weight[CHUNK], k[CHUNK];
  float end, x_down, p_scale, least_weight, least_decay, need, pad[58];
};
constexpr float U_DOWN = 0x1p-15f;  // the largest of T' / its scale is 2^14 to 2^15
constexpr float LO_UP = 0x1p11f, LO_DOWN = 0x1p-11f;

// The workspace: K and Q of every chunk and key head, T' (hi, lo), the factors and P (hi, lo) of every chunk and value head
template <int DK> struct Places {
  static constexpr int64_t MAT = CHUNK * DK * 2;
  char* base;
  int64_t HK, HV, chunks;
  static constexpr int64_t HEAD = 4 * T_FRAGS * FRAG + (int64_t)sizeof(Factors);
  __host__ __device__ int64_t bytes() const { return chunks * (HK * 2 * MAT + HV * HEAD); }
  __device__ char* k(int64_t chunk, int64_t hk) const { return base + (chunk * HK + hk) * 2 * MAT; }
  __device__ char* q(int64_t chunk, int64_t hk) const { return k(chunk, hk) + MAT; }
  __device__ char* t(int64_t chunk, int64_t hv) const { return base + chunks * HK * 2 * MAT + (chunk * HV + hv) * HEAD; }
  __device__ Factors* factors(int64_t chunk, int64_t hv) const { return (Factors*)(t(chunk, hv) + 2 * T_FRAGS * FRAG); }
  __device__ char* p(int64_t chunk, int64_t hv) const { return (char*)(factors(chunk, hv) + 1); }
};

// ---------------------------------------------------------------- powers of two

// {2^(14 - e), 2^(e - 14)} for a largest value of exponent e, so that 2^11 of the first is in fp32's range; of 0 the smallest
struct Pow2 {
  float down, up;
};
__device__ __forceinline__ Pow2 pow2_of(float largest) {
  const uint32_t e = min(max((__float_as_uint(largest) >> 23) & 255u, 26u), 254u);
  return {__uint_as_float((268u - e) << 23), __uint_as_float((e - 14u) << 23)};
}

__device__ __forceinline__ f32x4 mfma16(f16x8 a, f16x8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ f32x4 mfma4(float a, float b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0); }

// hi and lo of eight values x, with UP given as 2^11 x (what made them then has the factor).  The pair of hi
// passes through a register of its own: a value that is a product may be rounded in one step or two, and lo has to be
// what is left of the hi that the matrix instruction gets.  In the constants' registers, which the compiler does not look
// into, a product or sum and its rounding to fp16 are one instruction (v_fma_mix).
template <bool UP = false> __device__ __forceinline__ void split(const float (&x)[8], f16x8& hi, f16x8& lo) {
  typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
  float down = LO_DOWN, up = -LO_UP;
  asm("" : "+s"(up));
  if constexpr (UP) asm("" : "+s"(down));
#pragma unroll
  for (int e = 0; e < 8; e += 2) {
    f16x2 h;
    if constexpr (UP) h = {(_Float16)fmaf(x[e], down, 0.f), (_Float16)fmaf(x[e + 1], down, 0.f)};
    else h = {(_Float16)x[e], (_Float16)x[e + 1]};
    asm("" : "+v"(h));
    hi[e] = h[0];
    hi[e + 1] = h[1];
    lo[e] = (_Float16)fmaf((float)h[0], up, UP ? x[e] : x[e] * LO_UP);
    lo[e + 1] = (_Float16)fmaf((float)h[1], up, UP ? x[e + 1] : x[e + 1] * LO_UP);
  }
}

// ---------------------------------------------------------------- what needs no state

// A sum of logarithms to base 2 in two floats: the difference of two such sums is short of fp32 only by 2^-24 of itself,
// however long the sums are
struct Log2 {
  float hi, lo;
};
__device__ __forceinline__ float exp2_of(Log2 a, Log2 b) { return __builtin_amdgcn_exp2f((a.hi - b.hi) + (a.lo - b.lo)); }
__device__ __forceinline__ float exp2_of(Log2 a) { return __builtin_amdgcn_exp2f(a.hi + a.lo); }

__device__ __forceinline__ float wave_max_rows(float v) {
  v = fmaxf(v, dpp_move<0xB1>(v));
  v = fmaxf(v, dpp_move<0x4E>(v));
  v = fmaxf(v, dpp_move<0x141>(v));
  v = fmaxf(v, dpp_move<0x140>(v));
  v = fmaxf(v, lane_xor16(v));
  return fmaxf(v, lane_xor32(v));
}

// Sums up to and with every lane
template <int SHIFT>
__device__ __forceinline__ double from_lane_before(double v) {  // of the lane SHIFT before in 16 lanes, 0 where there is none
  const uint64_t bits = __builtin_bit_cast(uint64_t, v);
  const uint32_t lo = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)bits, 0x110 + SHIFT, 0xf, 0xf, false);
  const uint32_t hi = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)(bits >> 32), 0x110 + SHIFT, 0xf, 0xf, false);
  return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
__device__ __forceinline__ double lane_value(double v, int lane) {
  const uint64_t bits = __builtin_bit_cast(uint64_t, v);
  const uint32_t lo = __builtin_amdgcn_readlane((int)(uint32_t)bits, lane), hi = __builtin_amdgcn_readlane((int)(uint32_t)(bits >> 32), lane);
  return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
__device__ __forceinline__ double running_sum(double v, int row) {
  v += from_lane_before<1>(v);
  v += from_lane_before<2>(v);
  v += from_lane_before<4>(v);
  v += from_lane_before<8>(v);
  const double t0 = lane_value(v, 15), t1 = lane_value(v, 31), t2 = lane_value(v, 47);
  return v + (row > 2 ? t0 + t1 + t2 : row > 1 ? t0 + t1 : row > 0 ? t0 : 0.);
}

// Of the state's columns in a workgroup of the short sequences here: wide, as latency does not count beside the chunks
// (24 sequences of 4 tokens and one of 2048: 101 us with 128 columns, 107 with 32)
__host__ __device__ inline int step_cols(const anna_mi_gated_delta_args& a) { return a.value_dim % 128 == 0 ? 128 : 32; }

// A workgroup takes a chunk, a key head and `per` of its value heads; those from `blocks` on take short sequences, which
// then cost no launch of their own and run beside work that waits for latency (63 sequences of one token and one of 1024:
// 106 us with a launch for each kind, 97.5 so; one of 1 token and four prompts of 268 to 1500 110 and 105).  A wave has the rows row_of(wave, 0..15) of K and Q,
// which are at once their fragments and the left operands of K K^T and Q K^T.
template <int DT, int DK>
__global__ __launch_bounds__(256, 3) void delta_prepare_kernel(const anna_mi_gated_delta_args a,
                                                               const SpanChunk* __restrict__ chunks, const Places<DK> ws, int per,
                                                               uint32_t blocks, const SpanSeq* __restrict__ steps) {
  typedef typename Elem<DT>::T T;
  constexpr int KS = DK / 32;
  constexpr int LD = DK + 8;     // halves of a row of K in LDS
  constexpr int LF = CHUNK + 4;  // floats of a row of A, then T in its place, then P
  struct Lds {
    _Float16 K[CHUNK][LD];
    float a_rows[CHUNK * LF + 16 * 7];
    Log2 sums[4][CHUNK];  // a / ln 2 of the next four value heads
    float betas[4][CHUNK], kf[CHUNK], qf[CHUNK], kn[CHUNK], tops[2][4];
  };
  __shared__ __attribute__((aligned(16))) union {
    Lds prepare;
    StepLds<DK, 32> narrow;
    StepLds<DK, 128> wide;
  } lds;
  if (blockIdx.x >= blocks) {  // the short sequences beside the chunks
    const int slices = (int)a.value_dim / step_cols(a);
    if (step_cols(a) == 32) delta_step_block<DT, DK, 32>(a, steps, slices, blockIdx.x - blocks, lds.narrow);
    else delta_step_block<DT, DK, 128>(a, steps, slices, blockIdx.x - blocks, lds.wide);
    return;
  }
  auto& K = lds.prepare.K;
  auto& a_rows = lds.prepare.a_rows;
  auto& sums = lds.prepare.sums;
  auto& betas = lds.prepare.betas;
  auto& tops = lds.prepare.tops;
  auto &kf = lds.prepare.kf, &qf = lds.prepare.qf, &kn = lds.prepare.kn;

  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, n = lane & 15, g = lane >> 4;
  // a wave writes rows 8 apart at the same time: every 8 rows 16 banks are left out (107 -> 105 us
  // for 256 chunks of 16 key and 32 value heads)
  auto A = [&](int i, int j) -> float& { return a_rows[i * LF + 16 * (i >> 3) + j]; };
  const uint32_t ratio = (uint32_t)a.value_heads / (uint32_t)a.key_heads, parts = (uint32_t)a.value_heads / (uint32_t)per;
  const uint32_t chunk = blockIdx.x / parts, hv0 = blockIdx.x % parts * per, hk = hv0 / ratio;
  const bool writes_k = hv0 % ratio == 0;
  const SpanChunk here = chunks[chunk];
  if ((uint32_t)here.slot >= (uint32_t)a.slots) return;
  const int64_t first = here.first;
  const int tokens = here.tokens;

  // decays of four value heads, a wave each: sums of logarithms in 64 bits, as their differences count; -inf stands
  // for e^-10^4 = 0
  auto gate_raw = [&](int h) {
    return h < per && lane < tokens ? Gate{gate_value(a.decay, a.gates_dtype, (first + lane) * a.decay_stride + hv0 + h),
                                           gate_value(a.beta, a.gates_dtype, (first + lane) * a.beta_stride + hv0 + h)}
                                    : Gate{0.f, 0.f};
  };
  auto gates = [&](int h, Gate gate) {
    if (h < per) {
      gate = lane < tokens ? gate_of(a, gate, hv0 + h) : Gate{0.f, 0.f};
      const double s = running_sum(gate.g < -1e4f ? -1e4 : (double)gate.g, g) * 1.4426950408889634;
      const float hi = (float)s;
      sums[wave][lane] = {hi, (float)(s - hi)};
      betas[wave][lane] = gate.beta;
    }
  };
  const Gate mine_raw = gate_raw(wave);

  const int mine = row_of(wave, n);
  u32x4 raw[2][KS];
  if (mine < tokens) {
    const T* kp = (const T*)a.key + (first + mine) * a.key_stride_token + hk * a.key_stride_head + 8 * g;
    const T* qp = (const T*)a.query + (first + mine) * a.query_stride_token + hk * a.query_stride_head + 8 * g;
#pragma unroll
    for (int s = 0; s < KS; s++) raw[0][s] = *(const u32x4*)(kp + 32 * s);
#pragma unroll
    for (int s = 0; s < KS; s++) raw[1][s] = *(const u32x4*)(qp + 32 * s);
  } else {
#pragma unroll
    for (int s = 0; s < KS; s++) raw[0][s] = raw[1][s] = u32x4{0, 0, 0, 0};
  }

  gates(wave, mine_raw);

  // a power of two is taken out of every row, and what is left to make the unit vector kept as a factor
  f16x8 kr[KS], qr[KS];
#pragma unroll
  for (int which = 0; which < 2; which++) {
    float ss = 0.f, top = 0.f, x[KS][8];
#pragma unroll
    for (int s = 0; s < KS; s++)
#pragma unroll
      for (int e = 0; e < 8; e++) {
        const uint32_t w = raw[which][s][e / 2];
        x[s][e] = Elem<DT>::to_f32((T)(e & 1 ? w >> 16 : w & 0xffffu));
        ss = fmaf(x[s][e], x[s][e], ss);
        top = fmaxf(top, fabsf(x[s][e]));
      }
    ss += lane_xor16(ss);
    ss += lane_xor32(ss);
    top = fmaxf(top, lane_xor16(top));
    top = fmaxf(top, lane_xor32(top));
    // the largest value goes to 1 .. 2, where what fp16 rounds off the small ones, 2^-25, is below fp32's
    // roundings of the row's products
    const int e = top > 0.f && top < INFINITY ? 1 - __builtin_amdgcn_frexp_expf(top) : 0;
#pragma unroll
    for (int s = 0; s < KS; s++)
#pragma unroll
      for (int j = 0; j < 8; j++) (which ? qr : kr)[s][j] = (_Float16)ldexpf(x[s][j], e);
    const float f = ldexpf(a.normalize ? rsqrtf(ss + NORM_EPS) : 1.f, -e);
    if (which) {
      if (g == 0) qf[mine] = f * a.scaling;
    } else {
      float length = 0.f;  // |k|: of the row without its power of two, so of any size
#pragma unroll
      for (int s = 0; s < KS; s++)
#pragma unroll
        for (int j = 0; j < 8; j++) length = fmaf((float)kr[s][j], (float)kr[s][j], length);
      length += lane_xor16(length);
      length += lane_xor32(length);
      if (g == 0) {
        kf[mine] = f;
        kn[mine] = f * sqrtf(length);
      }
    }
  }
#pragma unroll
  for (int s = 0; s < KS; s++) *(f16x8*)&K[mine][32 * s + 8 * g] = kr[s];
  if (writes_k) {
    char* const k_to = ws.k(chunk, hk) + wave * KS * FRAG + 16 * lane;
    char* const q_to = ws.q(chunk, hk) + wave * KS * FRAG + 16 * lane;
#pragma unroll
    for (int s = 0; s < KS; s++) {
      *(f16x8*)(k_to + s * FRAG) = kr[s];
      *(f16x8*)(q_to + s * FRAG) = qr[s];
    }
  }
  __syncthreads();

  // K K^T and Q K^T of the wave's rows, as far as the tokens that they see: of waves 0 and 1 the first 32
  const int tiles = wave < 2 ? 2 : 4;
  const f32x4 zero = {0.f, 0.f, 0.f, 0.f};
  f32x4 kk[4] = {zero, zero, zero, zero}, qk[4] = {zero, zero, zero, zero};
#pragma unroll
  for (int ct = 0; ct < 4; ct++)
    if (ct < tiles)
#pragma unroll
      for (int s = 0; s < KS; s++) {
        const f16x8 col = *(const f16x8*)&K[16 * ct + n][32 * s + 8 * g];
        kk[ct] = mfma16(kr[s], col, kk[ct]);
        qk[ct] = mfma16(qr[s], col, qk[ct]);
      }
  float ki[4];
#pragma unroll
  for (int r = 0; r < 4; r++) ki[r] = kf[row_of(wave, 4 * g + r)];

  for (int h = 0; h < per; h++) {
    const int64_t hv = hv0 + h;
    if (h > 0) {
      __syncthreads();  // the head before is done with LDS
      if (h % 4 == 0) {
        gates(h + wave, gate_raw(h + wave));
        __syncthreads();
      }
    }
    const Log2* const at = sums[h % 4];
    const float* const beta = betas[h % 4];

    // A and P; P's rows are kept in registers until A's place is free
    f32x4 P[4];
    float p_top = 0.f, t_top = 0.f;
    Log2 ai[4], aj[4];
    float bi[4], cj[4];
#pragma unroll
    for (int r = 0; r < 4; r++) {
      ai[r] = at[row_of(wave, 4 * g + r)];
      bi[r] = beta[row_of(wave, 4 * g + r)];
      aj[r] = at[16 * r + n];
      cj[r] = kf[16 * r + n];
    }
#pragma unroll
    for (int ct = 0; ct < 4; ct++) {
      const int j = 16 * ct + n;
      if (ct < tiles) {
#pragma unroll
        for (int r = 0; r < 4; r++) {  // without branches: tokens that are not seen have a decay of e^-inf
          const int i = row_of(wave, 4 * g + r);
          const float t = (ai[r].hi - aj[ct].hi) + (ai[r].lo - aj[ct].lo), d = __builtin_amdgcn_exp2f(i >= j ? t : -INFINITY) * cj[ct];
          const float x = bi[r] * (ki[r] * kk[ct][r]) * d, y = qk[ct][r] * d;
          A(i, j) = i > j ? x : 0.f;
          P[ct][r] = i >= j ? y : 0.f;
          p_top = fmaxf(p_top, fabsf(P[ct][r]) < INFINITY ? fabsf(P[ct][r]) : 0.f);  // a q that is not finite is its row's affair
        }
      } else {
        P[ct] = zero;
#pragma unroll
        for (int r = 0; r < 4; r++) A(row_of(wave, 4 * g + r), j) = 0.f;
      }
    }
    __syncthreads();

    // T = (1 + A)^-1 in A's place: the diagonal blocks by substitution, a lane a column; then larger ones from
    // products, T21 = -T22 (A21 T11)
    if (wave == 0) {
      float x[16];
      const float b = beta[16 * g + n];
#pragma unroll
      for (int i = 0; i < 16; i++) {
        float s = i == n ? 1.f : 0.f;
#pragma unroll
        for (int k = 0; k < i; k++) s = fmaf(-A(16 * g + i, 16 * g + k), x[k], s);
        x[i] = s;
        t_top = fmaxf(t_top, fabsf(s * b));
      }
#pragma unroll
      for (int i = 0; i < 16; i++) A(16 * g + i, 16 * g + n) = x[i];
    }
    __syncthreads();
    // product of 16 x 16 blocks; the second form takes a result of the instruction as its right operand: its lane
    // (n, g) holds the rows 4 g + r
    auto block = [&](int lb, int lc, int rb, int rc, f32x4 c) {
#pragma unroll
      for (int k = 0; k < 4; k++) c = mfma4(A(16 * lb + n, 16 * lc + 4 * g + k), A(16 * rb + 4 * g + k, 16 * rc + n), c);
      return c;
    };
    auto times = [&](int lb, int lc, f32x4 x, f32x4 c) {
#pragma unroll
      for (int k = 0; k < 4; k++) c = mfma4(A(16 * lb + n, 16 * lc + 4 * g + k), x[k], c);
      return c;
    };
    auto put = [&](int rb, int cb, f32x4 y) {
      const float b = beta[16 * cb + n];
#pragma unroll
      for (int r = 0; r < 4; r++) {
        A(16 * rb + 4 * g + r, 16 * cb + n) = -y[r];
        t_top = fmaxf(t_top, fabsf(y[r] * b));
      }
    };
    if (wave < 2) {
      const int b = 2 * wave;
      const f32x4 y = times(b + 1, b + 1, block(b + 1, b, b, b, zero), zero);
      put(b + 1, b, y);
    }
    __syncthreads();
    {
      const int b = wave & 1, row = 2 + (wave >> 1);  // block column, block row of the result
      f32x4 x2 = zero, x3 = zero;
      for (int c = b; c < 2; c++) {
        x2 = block(2, c, c, b, x2);
        x3 = block(3, c, c, b, x3);
      }
      f32x4 y = times(row, 2, x2, zero);
      if (row == 3) y = times(row, 3, x3, y);
      __syncthreads();  // A21 is read
      put(row, b, y);
    }
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
      float x[8];
#pragma unroll
      for (int e = 0; e < 8; e++) x[e] = A(i, j + e) * beta[j + e] * (ts.down * LO_UP);
      f16x8 hi, lo;
      split<true>(x, hi, lo);
      *(f16x8*)(t_to + (2 * f) * FRAG + 16 * lane) = hi;
      *(f16x8*)(t_to + (2 * f + 1) * FRAG + 16 * lane) = lo;
    }
    if (tid < CHUNK) {
      Factors* to = ws.factors(chunk, hv);
      const float e = exp2_of(at[tid]), weight = tid < tokens ? kn[tid] * fabsf(beta[tid]) : 0.f;
      const float least_weight = -wave_max_rows(tid < tokens ? -weight : -INFINITY), least_decay = -wave_max_rows(-e);
      const float longest = wave_max_rows(tid < tokens ? kn[tid] : 0.f);
      // keys longer than 1 (and a third: unit vectors' lengths are rounded) make x larger than S and v
      const uint32_t longer = min(max((__float_as_uint(0.75f * longest) >> 23) & 255u, 126u), 226u) - 126u;
      const float x_down = __uint_as_float((127u - longer) << 23), x_up = __uint_as_float((127u + longer) << 23);
      to->decayed_k[tid] = e * (kf[tid] * x_down) * LO_UP;
      to->decay[tid] = e;
      to->q[tid] = qf[tid];
      to->to_end[tid] = exp2_of(at[CHUNK - 1], at[tid]) * (kf[tid] * x_up) * ts.up * LO_UP;
      to->step[tid] = tid > 0 ? exp2_of(at[tid], at[tid - 1]) : e;
      to->weight[tid] = weight;
      to->k[tid] = kf[tid];
      if (tid == CHUNK - 1) to->end = e;
      if (tid == 0) {
        const float largest = ts.up / U_DOWN, scale = ps.up * largest * x_up;
        to->p_scale = fminf(scale, 0x1p127f);
        to->x_down = x_down;
        to->least_weight = least_weight;
        to->least_decay = least_decay;
        to->need = scale < 0x1p127f ? 0x1p-14f * fmaxf(1.f, longest * largest * x_up) : INFINITY;
      }
    }
    __syncthreads();
#pragma unroll
    for (int ct = 0; ct < 4; ct++)
#pragma unroll
      for (int r = 0; r < 4; r++) A(row_of(wave, 4 * g + r), 16 * ct + n) = P[ct][r];
    __syncthreads();
    for (int f = wave; f < T_FRAGS; f += 4) {
      int mt, ks;
      t_frag(f, mt, ks);
      const int i = row_of(mt, n), j = 32 * ks + 8 * g;
      float y[8];
#pragma unroll
      for (int e = 0; e < 8; e++) y[e] = A(i, j + e) * (ps.down * LO_UP);
      f16x8 hi, lo;
      split<true>(y, hi, lo);
      *(f16x8*)(p_to + (2 * f) * FRAG + 16 * lane) = hi;
      *(f16x8*)(p_to + (2 * f + 1) * FRAG + 16 * lane) = lo;
    }
  }
}

// ---------------------------------------------------------------- the chain of states

__device__ __forceinline__ f16x8 frag(const char* base, int f, int lane) { return *(const f16x8*)(base + f * FRAG + 16 * lane); }

// Two values rounded to the type, in one register
template <int DT> __device__ __forceinline__ uint32_t pair_of(float x, float y) {
  typedef float f32x2 __attribute__((ext_vector_type(2)));
  typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
  typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
  const f32x2 v = {x, y};
  if constexpr (DT == ANNA_MI_BF16) return __builtin_bit_cast(uint32_t, __builtin_convertvector(v, bf16x2));
  else return __builtin_bit_cast(uint32_t, __builtin_convertvector(v, f16x2));
}

// Largest and smallest size, and the largest of a column over the four lanes that hold it.  A NaN is the answer of all three,
// so that one instruction takes three values as they are.
__device__ __forceinline__ float max_of(float a, float b) { return __builtin_elementwise_maximum(a, b); }
__device__ __forceinline__ float min_of(float a, float b) { return __builtin_elementwise_minimum(a, b); }
__device__ __forceinline__ float column_max(float v) {
  v = max_of(v, lane_xor16(v));
  return max_of(v, lane_xor32(v));
}
// Tiles 2 s and 2 s + 1 of a product's result as the operand of the next
template <bool UP> __device__ __forceinline__ void operand(f32x4 x, f32x4 y, f16x8& hi, f16x8& lo) {
  const float f[8] = {x[0], x[1], x[2], x[3], y[0], y[1], y[2], y[3]};
  split<UP>(f, hi, lo);
}
__device__ __forceinline__ float largest(float top, const f32x4& x) {
  return max_of(max_of(max_of(top, fabsf(x[0])), fabsf(x[1])), max_of(fabsf(x[2]), fabsf(x[3])));
}
__device__ __forceinline__ float smallest(float least, const f32x4& x) {
  return min_of(min_of(min_of(least, fabsf(x[0])), fabsf(x[1])), min_of(fabsf(x[2]), fabsf(x[3])));
}

// A chunk's tokens one after the other, on the chain's layout of the state: lane (n, g) holds rows row_of(t, 4 g + r) of
// column n, which are the 8 values that lane (m, g) has of token (mt, m) in K's and Q's fragments.  `keys`, `values` and the
// factors are in LDS.  All of it is asked for a token ahead.  2048 tokens of 32 heads, one chunk of one group
// of columns this way: 88 -> 136 us (169 with rows from memory when they are needed, and their norms made again).
template <int DT, int DK>
__device__ __forceinline__ void delta_tokens(const anna_mi_gated_delta_args& a, const char* keys, const char* queries, const char* values,
                                             const Factors& fac, int64_t first, int tokens, int64_t hv, int64_t col, int n, int g,
                                             f32x4 (&S)[DK / 16]) {
  typedef typename Elem<DT>::T T;
  constexpr int KS = DK / 32;
  const bool wide = a.gates_dtype == ANNA_MI_F32;
  struct Token {
    f16x8 k[KS], q[KS];
    uint32_t beta;  // as it is: what makes a value of it would wait for all of the loads
    T v;
    float step, kf, qf;
  };
  auto place = [&](int t, int s) {
    const int mt = t / 32 * 2 + t / 4 % 2, m = t % 32 / 8 * 4 + t % 4;
    return (mt * KS + s) * FRAG + 16 * (m + 16 * g);
  };
  auto ask = [&](int t) {
    Token token;
    const int64_t at = (first + t) * a.beta_stride + hv;
    token.beta = wide ? ((const uint32_t*)a.beta)[at] : ((const uint16_t*)a.beta)[at];
#pragma unroll
    for (int s = 0; s < KS; s++) token.q[s] = *(const f16x8*)(queries + place(t, s));
#pragma unroll
    for (int s = 0; s < KS; s++) token.k[s] = *(const f16x8*)(keys + place(t, s));
    token.v = ((const T*)values)[16 * t + n];
    token.step = fac.step[t], token.kf = fac.k[t], token.qf = fac.q[t];
    return token;
  };
  auto total = [](float v) {
    v += lane_xor16(v);
    return v + lane_xor32(v);
  };
  const HeadGate head = head_gate(a, hv);
  Token next = ask(0);
  for (int t = 0; t < tokens; t++) {
    const Token token = next;
    next = ask(min(t + 1, tokens - 1));
    const float v = Elem<DT>::to_f32(token.v), e = token.step, kf = token.kf, qf = token.qf;
    const float bits = wide ? __uint_as_float(token.beta) : a.gates_dtype == ANNA_MI_BF16 ? bf16_bits_to_f32((uint16_t)token.beta) : f16_bits_to_f32((uint16_t)token.beta);
    float k[DK / 4], sk[4] = {}, sq[4] = {};
#pragma unroll
    for (int i = 0; i < DK / 4; i++) {
      k[i] = fmaf((float)token.k[i / 8][i % 8], kf, 0.f);  // one instruction with its conversion
      sk[i % 4] = fmaf(S[i / 4][i % 4], k[i], sk[i % 4]);
    }
    const float u = gate_of(head, Gate{0.f, bits}).beta * (v - e * total((sk[0] + sk[1]) + (sk[2] + sk[3])));
#pragma unroll
    for (int i = 0; i < DK / 4; i++) {
      S[i / 4][i % 4] = fmaf(k[i], u, e * S[i / 4][i % 4]);
      sq[i % 4] = fmaf(S[i / 4][i % 4], fmaf((float)token.q[i / 8][i % 8], qf, 0.f), sq[i % 4]);
    }
    const float o = total((sq[0] + sq[1]) + (sq[2] + sq[3]));
    if (g == 0) ((T*)a.out)[((first + t) * a.value_heads + hv) * a.value_dim + col] = Elem<DT>::cvt(o);
  }
}

typedef __attribute__((address_space(3))) void* lds_ptr;
typedef const __attribute__((address_space(1))) void* global_ptr;
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4* lds_s16x4;

// Four 16-bit values of a column: of every 16 lanes, lane j brings 8 bytes of row j / 4, columns 4 (j % 4) .., and
// takes column j of the four rows
__device__ __forceinline__ s16x4 read_column(const char* p) { return __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4)p); }

// A workgroup of CW groups of 16 columns.  Its LDS: two chunks' operands of the state (K, T', the factors, v), two of
// the output (Q, the factors, P), and with SPLIT what a state's wave hands to the output's.
//   SPLIT: a wave for the state and one for the output of every column group, the output's a chunk behind, and one
//     wave that copies operands from the workspace into LDS a chunk ahead.  For few sequences: the chain of states is
//     all that counts, and what is not in it runs beside it.
//   else: a wave for every column group, that takes the output too, and one for the copies.
template <int DK, int CW, bool SPLIT> struct Stage {
  static constexpr int KS = DK / 32;
  static constexpr int MAT = CHUNK * DK * 2, TS = 2 * T_FRAGS * FRAG, PS = TS, FAC = (int)sizeof(Factors);
  static constexpr int TILE = 16 * (CHUNK * 2 + 8);  // of v [64][16], and of the output's columns [16][64 + 4]
  static constexpr int STATE = MAT + TS + FAC + CW * TILE;  // K, T', factors, v
  static constexpr int OUT = MAT + (SPLIT ? FAC : 0) + PS;  // Q, factors, P
  static constexpr int MAIL = SPLIT ? 2 * (KS + 2) * FRAG + 256 + 64 : 0;  // S, u; their unit a lane; a flag
  static constexpr int MAILS = 2 * STATE + 2 * OUT, TILES = MAILS + 2 * CW * MAIL, TOUCHED = TILES + (SPLIT ? CW * TILE : 0);
  static constexpr int COPIERS = SPLIT && CW == 1 ? 2 : 1, FIRST_COPIER = (SPLIT ? 2 : 1) * CW;
  static constexpr int WAVES = FIRST_COPIER + COPIERS, BYTES = TOUCHED + COPIERS * 256;
};

template <int DT, int DK, int CW, bool SPLIT>
__global__ __launch_bounds__((64 * Stage<DK, CW, SPLIT>::WAVES), 2) void delta_chain_kernel(
    const anna_mi_gated_delta_args a, const SpanChain* __restrict__ chains, const Places<DK> ws, uint32_t units) {
  typedef typename Elem<DT>::T T;
  typedef Stage<DK, CW, SPLIT> St;
  constexpr int NT = DK / 16, KS = DK / 32;
  extern __shared__ __attribute__((aligned(1024))) char lds[];
  const int lane = threadIdx.x & 63, n = lane & 15, g = lane >> 4, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t HV = a.value_heads, DV = a.value_dim;
  // a key head's workgroups on one XCD (workgroup b runs on XCD b % 8), whose L2 then has K and Q once for all of them,
  // and T' and P for a value head's slices
  const uint32_t ratio = (uint32_t)HV / (uint32_t)a.key_heads, slices = (uint32_t)DV / (16 * CW), each = ratio * slices;
  const uint32_t unit_of = blockIdx.x / (8 * each) * 8 + blockIdx.x % 8, part = blockIdx.x / 8 % each;
  if (unit_of >= units) return;
  const uint32_t hk = unit_of % (uint32_t)a.key_heads, hv = hk * ratio + part / slices, col0 = part % slices * (16 * CW);
  const SpanChain chain = chains[unit_of / (uint32_t)a.key_heads];
  const SpanSeq seq = chain.seq;
  const int64_t chunk0 = chain.first_chunk;
  const int count = (seq.tokens + CHUNK - 1) / CHUNK;
  if ((uint32_t)seq.slot >= (uint32_t)a.slots) {
    for (int64_t i = threadIdx.x; i < (int64_t)seq.tokens * 16 * CW; i += 64 * St::WAVES)
      ((T*)a.out)[((seq.first + i / (16 * CW)) * HV + hv) * DV + col0 + i % (16 * CW)] = Elem<DT>::cvt(0.f);
    return;
  }

  // ---- copies of the operands, one piece of FRAG bytes an instruction, the pieces dealt to COPIERS waves
  const int copier = wave - St::FIRST_COPIER;
  auto copy = [&](const char* from, int to, auto bytes) {
    constexpr int N = decltype(bytes)::value / FRAG;
#pragma unroll
    for (int i = 0; i < (N + St::COPIERS - 1) / St::COPIERS; i++) {
      const int at = (St::COPIERS * i + copier) * FRAG;
      if (N % St::COPIERS == 0 || at < N * FRAG)
        __builtin_amdgcn_global_load_lds((global_ptr)(from + at + 16 * lane), (lds_ptr)(lds + to + at), 16, 0, 0);
    }
  };
  auto fetch_state = [&](int c) {
    const int to = (c & 1) * St::STATE;
    copy(ws.k(chunk0 + c, hk), to, std::integral_constant<int, St::MAT>());
    copy(ws.t(chunk0 + c, hv), to + St::MAT, std::integral_constant<int, St::TS + St::FAC>());
    const int tokens = min(CHUNK, seq.tokens - c * CHUNK);
    const T* v = (const T*)a.value + (seq.first + (int64_t)c * CHUNK) * a.value_stride_token + hv * a.value_stride_head + col0;
#pragma unroll
    for (int i = 0; i < 2 * CW / St::COPIERS; i++) {
      // rows behind the last token hold the last one's again; their row of T' is zero
      const int at = St::COPIERS * i + copier, t = min(32 * (at & 1) + lane / 2, tokens - 1);
      __builtin_amdgcn_global_load_lds((global_ptr)(v + t * a.value_stride_token + 16 * (at >> 1) + 8 * (lane & 1)),
                                       (lds_ptr)(lds + to + St::MAT + St::TS + St::FAC + (at >> 1) * St::TILE + (at & 1) * FRAG), 16, 0, 0);
    }
  };
  auto fetch_out = [&](int c) {
    const int to = 2 * St::STATE + (c & 1) * St::OUT;
    copy(ws.q(chunk0 + c, hk), to, std::integral_constant<int, St::MAT>());
    if constexpr (SPLIT) copy((const char*)ws.factors(chunk0 + c, hv), to + St::MAT, std::integral_constant<int, St::FAC + St::PS>());
    else copy(ws.p(chunk0 + c, hv), to + St::MAT, std::integral_constant<int, St::PS>());
  };
  if (wave >= St::FIRST_COPIER) {
    // A chunk's time is short of memory's latency: a word of each line of the chunk after the next is asked for, which
    // brings the line to L2.  A value head's workgroups share its lines among them.  The words go to a corner of LDS that nobody
    // reads.
    constexpr int TOUCHES = CW == 1 ? 1 : CW == 2 ? 2 : 4;
    constexpr int LK = St::MAT / 128, LT = LK + (St::TS + St::FAC) / 128, LQ = LT + St::MAT / 128, LP = LQ + St::PS / 128;
    auto touch = [&](int c) {
      c = min(c, count - 1);
      const char *const k = ws.k(chunk0 + c, hk), *const t = ws.t(chunk0 + c, hv), *const q = ws.q(chunk0 + c, hk), *const p = ws.p(chunk0 + c, hv);
#pragma unroll
      for (int i = 0; i < TOUCHES; i++) {
        const int line = (i * slices + part % slices) * 64 + lane;
        const char* at = line < LK ? k + 128 * line : line < LT ? t + 128 * (line - LK) : line < LQ ? q + 128 * (line - LT) : p + 128 * min(line - LQ, LP - LQ - 1);
        __builtin_amdgcn_global_load_lds((global_ptr)at, (lds_ptr)(lds + St::TOUCHED + 256 * (wave - St::FIRST_COPIER)), 4, 0, 0);
      }
    };
    // the newest are the words, of the first copier alone
    auto wait = [&] {
      if (wave == St::FIRST_COPIER) asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(TOUCHES) : "memory");
      else asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
    };
    fetch_state(0);
    if constexpr (!SPLIT) fetch_out(0);
    if (wave == St::FIRST_COPIER) touch(1);
    for (int c = 0; c < count + SPLIT; c++) {
      wait();
      if (c + 1 < count) {
        fetch_state(c + 1);
        if constexpr (!SPLIT) fetch_out(c + 1);
      }
      if constexpr (SPLIT)
        if (c < count) fetch_out(c);
      if (wave == St::FIRST_COPIER) touch(c + 2);
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // the last words have landed: LDS may go to another workgroup
    return;
  }
  // chunk c (the output's waves: c - 1) is in LDS, and nobody reads the one before any more
  auto meet = [] { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); };

  const int cg = wave % CW;
  const uint32_t col = col0 + 16 * cg + n;
  const f32x4 zero = {0.f, 0.f, 0.f, 0.f};
  // A wave that takes everything has the registers for it if operands are not asked for earlier than this
#define PHASE() __builtin_amdgcn_sched_barrier(0)

  // ---- out = e^a Q S + P u
  auto load_q = [&](const char* at, f16x8 (&Q)[4 * KS]) {
#pragma unroll
    for (int f = 0; f < 4 * KS; f++) Q[f] = frag(at, f, lane);
  };
  auto q_times = [&](const f16x8 (&Q)[4 * KS], const f16x8 (&sh)[KS], const f16x8 (&sl)[KS], f32x4 (&qs)[4]) {
#pragma unroll
    for (int mt = 0; mt < 4; mt++) qs[mt] = zero;
#pragma unroll
    for (int s = 0; s < KS; s++)
#pragma unroll
      for (int mt = 0; mt < 4; mt++) qs[mt] = mfma16(Q[mt * KS + s], sl[s], qs[mt]);
#pragma unroll
    for (int mt = 0; mt < 4; mt++) qs[mt] *= LO_DOWN;
#pragma unroll
    for (int s = 0; s < KS; s++)
#pragma unroll
      for (int mt = 0; mt < 4; mt++) qs[mt] = mfma16(Q[mt * KS + s], sh[s], qs[mt]);
  };
  auto load_p = [&](const char* at, const Factors* fac, f16x8 (&PF)[2 * T_FRAGS], f32x4 (&fd)[4], f32x4 (&fq)[4]) {
#pragma unroll
    for (int f = 0; f < 2 * T_FRAGS; f++) PF[f] = frag(at, f, lane);
#pragma unroll
    for (int mt = 0; mt < 4; mt++) {
      fd[mt] = *(const f32x4*)&fac->decay[row_of(mt, 4 * g)];
      fq[mt] = *(const f32x4*)&fac->q[row_of(mt, 4 * g)];
    }
  };
  auto finish = [&](int c, const f16x8 (&PF)[2 * T_FRAGS], const f32x4 (&fd)[4], const f32x4 (&fq)[4], const f32x4 (&u)[4],
                    const f32x4 (&qs)[4], float unit, float p_scale, char* tile) {
    f16x8 uh[2], ul[2];
#pragma unroll
    for (int s = 0; s < 2; s++) operand<true>(u[2 * s] * (U_DOWN * LO_UP), u[2 * s + 1] * (U_DOWN * LO_UP), uh[s], ul[s]);
    f32x4 o[4] = {zero, zero, zero, zero};
#pragma unroll
    for (int part = 0; part < 3; part++) {
#pragma unroll
      for (int f = 0; f < T_FRAGS; f++) {
        const int s = f >= 4, mt = s ? f - 2 : f;
        o[mt] = mfma16(PF[2 * f + (part == 0)], part == 1 ? ul[s] : uh[s], o[mt]);
      }
      if (part == 1)
#pragma unroll
        for (int mt = 0; mt < 4; mt++) o[mt] *= LO_DOWN;
    }
    // through LDS by columns, so that a lane takes a token's row of 32 bytes
#pragma unroll
    for (int mt = 0; mt < 4; mt++) {
      uint32_t w[2];
#pragma unroll
      for (int r = 0; r < 4; r += 2) {
        const float y0 = fmaf(o[mt][r], p_scale, fd[mt][r] * qs[mt][r]), y1 = fmaf(o[mt][r + 1], p_scale, fd[mt][r + 1] * qs[mt][r + 1]);
        w[r / 2] = pair_of<DT>(y0 * (fq[mt][r] * unit), y1 * (fq[mt][r + 1] * unit));
      }
      *(uint2*)(tile + n * (CHUNK * 2 + 8) + 2 * row_of(mt, 4 * g)) = make_uint2(w[0], w[1]);
    }
    s16x4 row[4];
#pragma unroll
    for (int b = 0; b < 4; b++) row[b] = read_column(tile + (4 * b + n / 4) * (CHUNK * 2 + 8) + 2 * (16 * g + 4 * (n % 4)));
    const int tokens = min(CHUNK, seq.tokens - c * CHUNK);
    if (lane < tokens) {
      T* const to = (T*)a.out + ((seq.first + (int64_t)c * CHUNK + lane) * HV + hv) * DV + col0 + 16 * cg;
      *(u32x4*)to = __builtin_bit_cast(u32x4, __builtin_shufflevector(row[0], row[1], 0, 1, 2, 3, 4, 5, 6, 7));
      *(u32x4*)(to + 8) = __builtin_bit_cast(u32x4, __builtin_shufflevector(row[2], row[3], 0, 1, 2, 3, 4, 5, 6, 7));
    }
  };

  if constexpr (SPLIT) {
    if (wave >= CW) {
      meet();
      for (int c = 0; c < count; c++) {
        meet();
        const char *const st = lds + 2 * St::STATE + (c & 1) * St::OUT, *const mail = lds + St::MAILS + (2 * cg + (c & 1)) * St::MAIL;
        const Factors* const fac = (const Factors*)(st + St::MAT);
        f16x8 sh[KS], sl[KS], Q[4 * KS], PF[2 * T_FRAGS];
        f32x4 qs[4], u[4], fd[4], fq[4];
#pragma unroll
        for (int s = 0; s < KS; s++) {
          sh[s] = frag(mail, s, lane);
          sl[s] = frag(mail, KS + s, lane);
        }
        load_q(st, Q);
#pragma unroll
        for (int mt = 0; mt < 4; mt++) u[mt] = *(const f32x4*)(mail + (2 * KS + mt) * FRAG + 16 * lane);
        const float unit = *(const float*)(mail + 2 * (KS + 2) * FRAG + 4 * lane);
        const int taken = *(const int*)(mail + 2 * (KS + 2) * FRAG + 256);
        load_p(st + St::MAT + St::FAC, fac, PF, fd, fq);
        const float p_scale = fac->p_scale;
        if (taken) continue;  // token by token, by the state's wave
        q_times(Q, sh, sl, qs);
        finish(c, PF, fd, fq, u, qs, unit, p_scale, lds + St::TILES + cg * St::TILE);
      }
      return;
    }
  }

  // ---- the state
  float* const state = a.state + seq.slot * a.state_stride_slot + (int64_t)hv * DK * DV + col;
  f32x4 S[NT];
#pragma unroll
  for (int t = 0; t < NT; t++)
#pragma unroll
    for (int r = 0; r < 4; r++) S[t][r] = seq.fresh ? 0.f : state[row_of(t, 4 * g + r) * DV];
  // S, x and u of a column are held in its unit, a power of two, kept so that the largest of S and v is 2^6 to 2^11:
  // what is computed from them is then short of fp16's upper end
  float unit = 1.f, per_unit = 1.f;
  bool lost = false;  // the column's state is not finite any more

  for (int c = 0; c < count; c++) {
    meet();
    const char* const st = lds + (c & 1) * St::STATE;
    const char* const so = lds + 2 * St::STATE + (c & 1) * St::OUT;
    char* const mail = lds + St::MAILS + (2 * cg + (c & 1)) * St::MAIL;
    const Factors* const fac = (const Factors*)(st + St::MAT + St::TS);
    char* const tile = lds + (c & 1) * St::STATE + St::MAT + St::TS + St::FAC + cg * St::TILE;
    s16x4 v[4];
#pragma unroll
    for (int mt = 0; mt < 4; mt++) v[mt] = read_column(tile + 32 * (row_of(mt, 4 * g) + n / 4) + 8 * (n % 4));
    f16x8 K[4 * KS];
#pragma unroll
    for (int f = 0; f < 4 * KS; f++) K[f] = frag(st, f, lane);
    f32x4 fk[4];
#pragma unroll
    for (int mt = 0; mt < 4; mt++) fk[mt] = *(const f32x4*)&fac->decayed_k[row_of(mt, 4 * g)];
    f32x4 x[4];
    float s_top = 0.f, v_top = 0.f, v_least = INFINITY;
#pragma unroll
    for (int t = 0; t < NT; t++) s_top = largest(s_top, S[t]);
#pragma unroll
    for (int mt = 0; mt < 4; mt++) {
#pragma unroll
      for (int r = 0; r < 4; r++) x[mt][r] = Elem<DT>::to_f32((T)v[mt][r]);
      v_top = largest(v_top, x[mt]);
      v_least = smallest(v_least, x[mt]);
    }
    const float top = column_max(max_of(s_top, v_top * per_unit));
    bool taken = false;  // token by token
    if (__any(top > 2048.f || (top < 64.f && top > 0.f))) {
      const uint32_t e = min(max((__float_as_uint(top) >> 23) & 255u, 10u), 250u);
      const float up = __uint_as_float((e - 9u) << 23), down = __uint_as_float((263u - e) << 23);  // the largest becomes 2^9
      const float s_col = column_max(s_top);
      const bool far = s_col > 0.f && s_col * down < 0x1p-60f;  // the state would lose bits, which the tokens need
      const bool change = ((top > 2048.f && top < INFINITY) || top < 64.f) && unit * up >= 0x1p-100f && unit * up <= 0x1p100f && !far;
      taken = __any(far && !lost);
      unit *= change ? up : 1.f;
      per_unit *= change ? down : 1.f;
      s_top *= change ? down : 1.f;
#pragma unroll
      for (int t = 0; t < NT; t++) S[t] *= change ? down : 1.f;
    }
    // whether every token sees something of the unit's order, at a glance: by the state or by all values
    const uint64_t by_state = __ballot(lost || top == 0.f || s_top * fac->least_decay >= fac->need);
    const uint64_t by_values = __ballot(v_least * per_unit * fac->least_weight >= fac->need);
    const uint64_t sure = by_state | by_state >> 16 | by_state >> 32 | by_state >> 48 | (by_values & by_values >> 16 & by_values >> 32 & by_values >> 48);
    // K S
    f16x8 sh[KS], sl[KS];
#pragma unroll
    for (int s = 0; s < KS; s++) operand<false>(S[2 * s], S[2 * s + 1], sh[s], sl[s]);
    f32x4 ks[4] = {zero, zero, zero, zero}, qs[4];
#pragma unroll
    for (int s = 0; s < KS; s++)
#pragma unroll
      for (int mt = 0; mt < 4; mt++) ks[mt] = mfma16(K[mt * KS + s], sl[s], ks[mt]);
#pragma unroll
    for (int mt = 0; mt < 4; mt++) ks[mt] *= LO_DOWN;
#pragma unroll
    for (int s = 0; s < KS; s++)
#pragma unroll
      for (int mt = 0; mt < 4; mt++) ks[mt] = mfma16(K[mt * KS + s], sh[s], ks[mt]);
    f16x8 TF[2 * T_FRAGS];
    f32x4 fe[4];
    auto load_t = [&] {
#pragma unroll
      for (int f = 0; f < 2 * T_FRAGS; f++) TF[f] = frag(st + St::MAT, f, lane);
#pragma unroll
      for (int mt = 0; mt < 4; mt++) fe[mt] = *(const f32x4*)&fac->to_end[row_of(mt, 4 * g)];
    };
    const float end = fac->end;
    if constexpr (SPLIT) {
      load_t();
#pragma unroll
      for (int s = 0; s < KS; s++) {
        *(f16x8*)(mail + s * FRAG + 16 * lane) = sh[s];
        *(f16x8*)(mail + (KS + s) * FRAG + 16 * lane) = sl[s];
      }
    }
    if constexpr (!SPLIT) {
      PHASE();
      f16x8 Q[4 * KS];
      load_q(so, Q);
      q_times(Q, sh, sl, qs);
      PHASE();
      load_t();
    }
    // x = v - e^a K S, 2^11 of it
    const float x_unit = per_unit * (fac->x_down * LO_UP);
#pragma unroll
    for (int mt = 0; mt < 4; mt++)
#pragma unroll
      for (int r = 0; r < 4; r++) x[mt][r] = fmaf(x[mt][r], x_unit, -(fk[mt][r] * ks[mt][r]));
    f16x8 hi[2], lo[2];
    operand<true>(x[0], x[1], hi[0], lo[0]);
    operand<true>(x[2], x[3], hi[1], lo[1]);
    // K^T: row (t, n) at tokens 32 j + 8 g + 0..7, as columns of K's fragments (2 j and 2 j + 1, t / 2)
    f16x8 KT[2 * NT];
#pragma unroll
    for (int f = 0; f < 2 * NT; f++) {
      const int t = f / 2, j = f % 2;
      s16x4 h[2];
#pragma unroll
      for (int i = 0; i < 2; i++)
        h[i] = read_column(st + ((2 * j + i) * KS + t / 2) * FRAG + (16 * (n % 4) + 4 * g + n / 4) * 16 + 8 * (t % 2));
      KT[f] = __builtin_bit_cast(f16x8, __builtin_shufflevector(h[0], h[1], 0, 1, 2, 3, 4, 5, 6, 7));
    }
    // u = T' x, the small parts first
    f32x4 u[4] = {zero, zero, zero, zero};
#pragma unroll
    for (int part = 0; part < 3; part++) {
#pragma unroll
      for (int f = 0; f < T_FRAGS; f++) {
        const int s = f >= 4, mt = s ? f - 2 : f;
        u[mt] = mfma16(TF[2 * f + (part == 0)], part == 1 ? lo[s] : hi[s], u[mt]);
      }
      if (part == 1)
#pragma unroll
        for (int mt = 0; mt < 4; mt++) u[mt] *= LO_DOWN;
    }
    f32x4 w[4];
#pragma unroll
    for (int mt = 0; mt < 4; mt++) w[mt] = u[mt] * fe[mt];
    operand<true>(w[0], w[1], hi[0], lo[0]);
    operand<true>(w[2], w[3], hi[1], lo[1]);
    const float p_scale = fac->p_scale;
    // S' = e^{a_63} S + K^T (e^{a_63 - a} u)
    f32x4 add[NT];
#pragma unroll
    for (int t = 0; t < NT; t++) add[t] = zero;
#pragma unroll
    for (int j = 0; j < 4; j++) {
#pragma unroll
      for (int t = 0; t < NT; t++) add[t] = mfma16(KT[2 * t + (j & 1)], j < 2 ? lo[j & 1] : hi[j & 1], add[t]);
      if (j == 1)
#pragma unroll
        for (int t = 0; t < NT; t++)
#pragma unroll
          for (int r = 0; r < 4; r++) add[t][r] = fmaf(add[t][r], LO_DOWN, S[t][r] * end);
    }
    // u may overflow where the state's update does not
    float u_top = 0.f;
#pragma unroll
    for (int mt = 0; mt < 4; mt++) u_top = largest(u_top, u[mt]);
    taken = taken || __any(!(fabsf(add[0][0]) < INFINITY && u_top <= 65504.f / U_DOWN) && !lost);
    if ((sure & 0xffff) != 0xffff) {
      float seen = column_max(s_top), least = INFINITY;
      const int tokens = min(CHUNK, seq.tokens - c * CHUNK);
      int column = n;
      asm volatile("" : "+v"(column));  // its address is made here, too
      for (int t = 0; t < tokens; t++) {
        seen = fmaxf(seen * fac->step[t], fac->weight[t] * (fabsf(Elem<DT>::load((const T*)tile, 16 * t + column)) * per_unit));
        least = seen > 0.f ? fminf(least, seen) : least;
      }
      taken = taken || __any(least < fac->need && !lost);
    }
    if constexpr (SPLIT) {
#pragma unroll
      for (int mt = 0; mt < 4; mt++) *(f32x4*)(mail + (2 * KS + mt) * FRAG + 16 * lane) = u[mt];
      *(float*)(mail + 2 * (KS + 2) * FRAG + 4 * lane) = unit;
      *(int*)(mail + 2 * (KS + 2) * FRAG + 256) = taken;
    }
    if (!taken) {
#pragma unroll
      for (int t = 0; t < NT; t++) S[t] = add[t];
      if constexpr (!SPLIT) {
        PHASE();
        f16x8 PF[2 * T_FRAGS];
        f32x4 fd[4], fq[4];
        load_p(so + St::MAT, fac, PF, fd, fq);
        finish(c, PF, fd, fq, u, qs, unit, p_scale, tile);
      }
    } else {
#pragma unroll
      for (int t = 0; t < NT; t++) S[t] *= unit;
      unit = per_unit = 1.f;
      // addresses made from these are made here, and not kept over the chunks
      uint32_t here = col;
      int rows = g;
      asm volatile("" : "+v"(here), "+v"(rows));
      delta_tokens<DT, DK>(a, st, ws.q(chunk0 + c, hk), tile, *fac, seq.first + (int64_t)c * CHUNK, min(CHUNK, seq.tokens - c * CHUNK), hv, here,
                           (int)(here & 15), rows, S);
      // 0, or a NaN where the state is not finite: products that overflow fp16 say nothing about it
      float none = 0.f;
#pragma unroll
      for (int t = 0; t < NT; t++)
#pragma unroll
        for (int r = 0; r < 4; r++) none = fmaf(S[t][r], 0.f, none);
      none += lane_xor16(none);
      none += lane_xor32(none);
      lost = !(none == 0.f);
    }
  }
  if constexpr (SPLIT) meet();
#pragma unroll
  for (int t = 0; t < NT; t++)
#pragma unroll
    for (int r = 0; r < 4; r++) state[row_of(t, 4 * g + r) * DV] = S[t][r] * unit;
}

// ---------------------------------------------------------------- host

template <int DK> static Places<DK> places(const anna_mi_gated_delta_args& a, const anna_mi_state_span& s) {
  return {(char*)a.workspace, a.key_heads, a.value_heads, s.chunks};
}

template <int DT, int DK>
static int delta_chunks(const anna_mi_gated_delta_args& a, const anna_mi_state_span& s, hipStream_t stream) {
  const Places<DK> ws = places<DK>(a, s);
  // a key head's value heads in one workgroup share the products of K, where that still fills the chip: the whole call at 16
  // key heads takes 604 us with both value heads and 629 with one for 256 chunks, 86 and 90 for 32, 52 both ways for 16
  const int64_t ratio = a.value_heads / a.key_heads;
  const int per = s.chunks * a.key_heads >= 512 ? (int)ratio : 1;
  const int64_t steps = s.steps * a.value_heads * (a.value_dim / step_cols(a)), prepare = s.chunks * (a.value_heads / per), groups = s.chains * a.value_heads * (a.value_dim / 16);
  ANNA_CHECK(prepare + steps <= INT32_MAX / 256 && groups <= INT32_MAX / 128, "gated delta rule: too many tokens and heads for a launch");
  delta_prepare_kernel<DT, DK><<<prepare + steps, 256, 0, stream>>>(a, span_chunks(s), ws, per, (uint32_t)prepare, span_steps(s));
  ANNA_LAUNCH_CHECK("delta_prepare");
  const uint32_t units = (uint32_t)(s.chains * a.key_heads);
  hipError_t allowed = hipSuccess;
#define ANNA_CHAIN(CW, SPLIT)                                                                                             \
  {                                                                                                                       \
    typedef Stage<DK, CW, SPLIT> St;                                                                                      \
    static_assert(St::BYTES <= 160 * 1024, "LDS");                                                                        \
    const auto kern = &delta_chain_kernel<DT, DK, CW, SPLIT>;                                                             \
    allowed = hipFuncSetAttribute((const void*)kern, hipFuncAttributeMaxDynamicSharedMemorySize, St::BYTES);              \
    if (allowed == hipSuccess)                                                                                            \
      kern<<<8 * ((units + 7) / 8) * (groups / units / CW), 64 * St::WAVES, St::BYTES, stream>>>(a, span_chains(s), ws, units); \
  }
  constexpr bool SPLIT_TWO = Stage<DK, 2, true>::BYTES <= 160 * 1024;  // at 128 key dims there is no room
  // One workgroup fits a compute unit's LDS in each form.  Its time is the longest chain's or the work's share of 256 compute
  // units, in chunks of 2.0 us with one column group (2.2 where the chip is full), 2.9 with two, 3.1 to 3.6 with four, which
  // share the copies.  bf16, 32 heads of 128, the whole call, one against four: 4000 tokens 161 and 223 us, 4000 + 300
  // 177 and 227, 4000 + 1000 200 and 228, 3000 + 1000 + 200 178 and 180, 4000 + 2000 241 and 235, twice 2048 167 and
  // 135, three times 247 and 147.  Two serve what four do not divide (three times 2048 at 64 key dims, fp16, 96 columns:
  // 173, 201 with one; at 128 dims, bf16, 234 and 243, eight times 395 and 507); at 128 key dims, where the output's wave of
  // its own has no room in LDS, the state's takes the outputs.
  const int64_t work = s.chunks * a.value_heads * (a.value_dim / 16);
  auto share = [&](int cw) { return std::max(256 * s.longest, work / cw); };
  if (a.value_dim % 64 == 0 && 3 * share(1) > 4 * share(4)) ANNA_CHAIN(4, false)
  else if (a.value_dim % 64 != 0 && 6 * share(1) > 7 * share(2)) ANNA_CHAIN(2, SPLIT_TWO)
  else ANNA_CHAIN(1, true)
#undef ANNA_CHAIN
  if (allowed != hipSuccess) return fail_hip(allowed, "delta_chain");
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
  ANNA_CHECK(a.slots >= 0 && a.slots <= INT32_MAX, "gated delta rule: %lld slots", (long long)a.slots);
  ANNA_CHECK(span->max_slot < a.slots, "gated delta rule: slot %lld of a state of %lld", (long long)span->max_slot, (long long)a.slots);
  return ANNA_MI_OK;
}

}  // namespace anna

extern "C" {

int64_t anna_mi_gated_delta_workspace(const anna_mi_gated_delta_args* args, const anna_mi_state_span* span) {
  if (anna::check_delta(args, span) != ANNA_MI_OK) return 0;
  return args->key_dim == 64 ? anna::places<64>(*args, *span).bytes() : anna::places<128>(*args, *span).bytes();
}

int anna_mi_gated_delta(const anna_mi_gated_delta_args* args, anna_mi_state_span* span, void* stream) {
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
  ANNA_CHECK((uintptr_t)a.out % 16 == 0, "gated delta rule: out must be 16-byte aligned");
  ANNA_CHECK((uintptr_t)a.state % 16 == 0 && a.state_stride_slot % 4 == 0, "gated delta rule: states must be 16-byte aligned");
  ANNA_CHECK(a.slots <= 1 || a.state_stride_slot >= a.value_heads * a.key_dim * a.value_dim, "gated delta rule: states overlap");
  ANNA_CHECK(span->chunks == 0 || (a.workspace && (uintptr_t)a.workspace % 256 == 0), "gated delta rule: no workspace, or not 256-byte aligned");
  // a state is written while other workgroups still read the inputs
  const int64_t gate = a.gates_dtype == ANNA_MI_F32 ? 4 : 2;
  const anna::Rows states = {a.state, a.slots, a.state_stride_slot * 4, a.value_heads * a.key_dim * a.value_dim * 4};
  const struct {
    const char* name;
    anna::Rows rows;
  } inputs[] = {{"query", {a.query, span->tokens, a.query_stride_token * 2, ((a.key_heads - 1) * a.query_stride_head + a.key_dim) * 2}},
                {"key", {a.key, span->tokens, a.key_stride_token * 2, ((a.key_heads - 1) * a.key_stride_head + a.key_dim) * 2}},
                {"value", {a.value, span->tokens, a.value_stride_token * 2, ((a.value_heads - 1) * a.value_stride_head + a.value_dim) * 2}},
                {"decay", {a.decay, span->tokens, a.decay_stride * gate, a.value_heads * gate}},
                {"beta", {a.beta, span->tokens, a.beta_stride * gate, a.value_heads * gate}},
                {"a_log", {a.a_log, 1, 0, a.value_heads * 4}},
                {"dt_bias", {a.dt_bias, 1, 0, a.value_heads * 4}}};
  for (const auto& i : inputs) ANNA_CHECK(anna::rows_apart(states, i.rows), "gated delta rule: the state overlaps %s", i.name);
  if (const int rc = anna::span_take(span, a.slots, "gated delta rule")) return rc;
  hipStream_t st = anna::as_stream(stream);
  if (span->chains == 0) return anna::delta_step(a, *span, st);
  ANNA_DISPATCH_DTYPE(a.dtype, DT, {
    if constexpr (DT != ANNA_MI_F32)
      return a.key_dim == 64 ? anna::delta_chunks<DT, 64>(a, *span, st) : anna::delta_chunks<DT, 128>(a, *span, st);
  });
  return ANNA_MI_OK;
}

}  // extern "C"
