// Attention over the paged 4-bit KV cache (page layout in anna_mi.h).
//
// out = softmax(scaling q K^T) V over the tokens up to and with the query's own, K and V held as
// (code + zero) * scale with one scale and zero for 64 values of a token and head.
//
// Split form.  A workgroup takes the query rows of one KV head (R = 16, 32 or 64 rows: tokens times
// query heads of that KV head) and some of the sequence's pages; each of its four waves takes every
// fourth step (a page, or half of one) with an online softmax of its own, and the waves' results are joined at the end.
// Codes go to the matrix cores as whole numbers: 16 + code has the bits 0x4180 | code << 3 in bf16
// (in fp16 0x4C00 | code << 6), so 8 codes cost 8 instructions and no conversion.  With
// o = zero - 16 (the cache's offsets, exact in bf16)
//   q.k   = sum over groups of  scale * (sum_d q_d (16 + code_d) + o * sum_d q_d)
//   p V_d = sum_t ps_t (16 + code_td) + sum_t ps_t o_t,     ps_t = p_t * scale_t rounded to bf16
// where the products with o are matrix instructions too: the first starts the sums (sum_d q_d as three
// bf16 terms, good to 24 bits), the second takes the same rounded ps, so the 16s cancel but for the
// fp32 sums' own roundings.
//   S^T = K Q^T by v_mfma_f32_16x16x32: rows = 16 tokens, columns = 16 query rows; a lane holds four
//   tokens of its query.  O^T = V^T P^T: the lane's eight tokens of two such tiles are its eight k of
//   the second product, so P never leaves the lane; the value codes are stored in that order.
// For fp16 activations ps is split into two bf16 terms: one alone is coarser than the output's type.
// Memory bounds the long contexts: 4 sequences of 100K to 131K tokens (564 MB) take 113 us, 5.0 TB/s, a copy's rate.
// Short ones are bound by the chain of a launch (item, table, first page: ~5 us), two or three steps of ~3 us and the
// merge's launch (5 us): 8 sequences of 1K to 16K (45 MB, head_dim 256) take 23 us, one of 1000 tokens 10 us.
//
// Tile form, for more than 64 query rows of a KV head: further down.
#include <type_traits>

#include "paged.hpp"

namespace anna {
namespace paged {
namespace {

typedef uint16_t u16x4 __attribute__((ext_vector_type(4)));

constexpr float NEG = -INFINITY;
// Probabilities with bf16's exponents stay below 2^-ROOM, in the tile form, whose maximum may lag, 2^-(ROOM - P_SLACK): sums
// of 2^24 of the former, times what stands for a value at most (31 times its scale, and a scale is up to 2^125), and of
// 2^22 of the latter, times the type's largest value, stay within fp32, as the values' mean does.
constexpr float ROOM = 26.0f;

__device__ __forceinline__ f32x4 mfma_bf16(u32x4 a, u32x4 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
template <int DT> __device__ __forceinline__ f32x4 mfma(u32x4 a, u32x4 b, f32x4 c) {
  if constexpr (DT == ANNA_MI_BF16) return mfma_bf16(a, b, c);
  else return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

// The mask of codes16 in a vector register of its own: with it there, a mask and a merge are one instruction
// (v_and_or_b32 takes one operand that is no vector register).
template <int DT> __device__ __forceinline__ uint32_t code_mask() {
  uint32_t mask = DT == ANNA_MI_BF16 ? 0x00780078u : 0x03C003C0u;
  asm volatile("" : "+v"(mask));
  return mask;
}
// 16 + code of the 8 codes of a word, as operand elements of the type.
template <int DT> __device__ __forceinline__ u32x4 codes16(uint32_t w, uint32_t mask) {
  if constexpr (DT == ANNA_MI_BF16)
    return u32x4{((w << 3) & mask) | 0x41804180u, ((w >> 1) & mask) | 0x41804180u, ((w >> 5) & mask) | 0x41804180u,
                 ((w >> 9) & mask) | 0x41804180u};
  else
    return u32x4{((w << 6) & mask) | 0x4C004C00u, ((w << 2) & mask) | 0x4C004C00u, ((w >> 2) & mask) | 0x4C004C00u,
                 ((w >> 6) & mask) | 0x4C004C00u};
}

__device__ __forceinline__ float bf16_lo(uint32_t v) { return __uint_as_float(v << 16); }
__device__ __forceinline__ float bf16_hi(uint32_t v) { return __uint_as_float(v & 0xFFFF0000u); }
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
__device__ __forceinline__ uint32_t pack_bf16(float a, float b) {
  const bf16x2 v = {(__bf16)a, (__bf16)b};
  return __builtin_bit_cast(uint32_t, v);
}

// 2^x of the difference to a running maximum that may still be -inf.
__device__ __forceinline__ float weight(float m, float top) { return m == NEG ? 0.0f : __builtin_amdgcn_exp2f(m - top); }

// A reciprocal within a unit in the last place of fp32, where a division takes ten instructions.
__device__ __forceinline__ float sigmoid(float x) { return __builtin_amdgcn_rcpf(1.0f + __expf(-x)); }

// Four neighbouring gates of an output row, asked for ahead of the sums that they meet.
__device__ __forceinline__ u16x4 gates(const Attend& a, int64_t token, int head, int d) {
  return *(const u16x4*)((const uint16_t*)a.gate + token * a.g_token + head * a.g_head + d);
}

// Four neighbouring values of an output row, gated.
template <int DT>
__device__ __forceinline__ void write_out(const Attend& a, int D, int64_t token, int head, int d, f32x4 v, u16x4 g, int64_t heads) {
  if (a.gate) {
#pragma unroll
    for (int i = 0; i < 4; i++) v[i] *= sigmoid(Elem<DT>::to_f32(g[i]));
  }
  u16x4 o;
#pragma unroll
  for (int i = 0; i < 4; i++) o[i] = Elem<DT>::cvt(v[i]);
  *(u16x4*)((uint16_t*)a.out + (token * heads + head) * D + d) = o;
}

// Tokens of a wave's step: a page, or half of one where a page's registers would leave no room for a second wave.
template <int D, int NQ> constexpr int step_tokens() { return D == 256 || NQ > 1 ? 32 : 64; }

// What a wave holds of a step's tokens in registers.  Lane offsets are unsigned 32-bit numbers, so that the page's
// address stays in scalar registers.
template <int D, int T> struct StepKeys {
  static constexpr int TT = T / 16, NG = D / GROUP, KS = D / 32;
  uint32_t code[TT][KS];
  uint16_t offset[TT][NG];
  uint2 scale[TT][NG];
  __device__ __forceinline__ void load(const uint8_t* page, int half, uint32_t lane) {
    const uint32_t q = lane / 16, r = lane % 16;
    const uint32_t at_code = r * (D / 2) + q * (D / 8), at_scale = K_SCALES * D + q * NG * 8, at_offset = K_OFFSETS * D + r * NG * 2;
#pragma unroll
    for (int t = 0; t < TT; t++) {
      const uint8_t *code_row = page + (2 * half + t) * 8 * D, *scale_row = page + (2 * half + t) * 32 * NG;
      __builtin_memcpy(code[t], __builtin_assume_aligned(code_row + at_code, D / 8 < 16 ? D / 8 : 16), D / 8);
      __builtin_memcpy(scale[t], __builtin_assume_aligned(scale_row + at_scale, NG > 1 ? 16 : 8), NG * 8);
      __builtin_memcpy(offset[t], __builtin_assume_aligned(scale_row + at_offset, NG * 2), NG * 2);
    }
  }
};
template <int D, int T> struct StepValues {
  static constexpr int HALVES = T / 32, NG = D / GROUP;
  u32x4 code[HALVES][NG];
  uint2 scale[HALVES][2][NG], offset[HALVES][2][NG];
  __device__ __forceinline__ void load(const uint8_t* page, int half, uint32_t lane) {
    const uint32_t q = lane / 16;
    const uint32_t at_code = V_CODES * D + lane * 16, at_scale = V_SCALES * D + q * NG * 8, at_offset = V_OFFSETS * D + q * NG * 8;
#pragma unroll
    for (int t = 0; t < HALVES; t++) {
      const uint8_t *code_row = page + (half + t) * 16 * D, *scale_row = page + (half + t) * 64 * NG;
#pragma unroll
      for (int g = 0; g < NG; g++) code[t][g] = *(const u32x4*)(code_row + g * 1024 + at_code);
#pragma unroll
      for (int u = 0; u < 2; u++) {
        __builtin_memcpy(scale[t][u], __builtin_assume_aligned(scale_row + u * 32 * NG + at_scale, NG > 1 ? 16 : 8), NG * 8);
        __builtin_memcpy(offset[t][u], __builtin_assume_aligned(scale_row + u * 32 * NG + at_offset, NG > 1 ? 16 : 8), NG * 8);
      }
    }
  }
};

#define PIN() __builtin_amdgcn_sched_barrier(0)

// NQ: 16-row column tiles of queries.
template <int DT, int D, int NQ>
__global__ __launch_bounds__(256, NQ * D <= 256 ? 2 : 1) void paged_split_kernel(const Attend a) {
  constexpr int NG = D / GROUP, KS = D / 32, DTILES = D / 16, R = 16 * NQ, T = step_tokens<D, NQ>(), TT = T / 16, STEPS = PAGE / T;
  constexpr bool TWO = DT == ANNA_MI_F16;  // ps as two bf16 terms
  __shared__ __align__(16) float joined[4][16][D + 4];
  __shared__ float wave_m[4][16], wave_l[4][16];

  const int H = a.kv_heads, G = a.group;
  const int h = blockIdx.x % H, index = blockIdx.x / H;
  const Item it = a.split[index];
  if (index >= a.header[0]) return;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), lane = threadIdx.x % 64, q = lane / 16, r = lane % 16;
  const int rows = it.count * G;
  const int32_t* table = a.table + it.row * a.width;
  auto page_at = [&](int32_t page) { return a.pool + ((int64_t)page * H + h) * page_bytes(D); };

  // Steps wave, wave + 4, ...  A step's keys are asked for as soon as the last step's are used up, its values
  // likewise: the loads have the other half of the step to arrive in, and need no second set of registers.
  int step = it.page0 * STEPS + wave;
  const int end = it.page1 * STEPS;
  StepKeys<D, T> k;
  StepValues<D, T> v;
  if (step < end) {
    const uint8_t* page = page_at(table[step / STEPS]);
    k.load(page, step % STEPS, lane);
    v.load(page, step % STEPS, lane);
  }
  int32_t next = step + 4 < end ? table[(step + 4) / STEPS] : 0;

  // queries: column r of tile n is row it.tile * R + 16 n + r
  u32x4 qf[NQ][KS];
  uint2 qsum[NQ][NG];  // the groups' sums as three bf16 terms, in k = 0, 1, 2 of the first quarter
  int limit[NQ];             // tokens that the query sees
#pragma unroll
  for (int n = 0; n < NQ; n++) {
    const int row = it.tile * R + 16 * n + r, t = row / G, head = h * G + row % G;
    const bool valid = row < rows;
    limit[n] = valid ? it.start + t + 1 : 0;
    const uint16_t* p = (const uint16_t*)a.query + (int64_t)(it.offset + t) * a.q_token + head * a.q_head + q * 8;
#pragma unroll
    for (int s = 0; s < KS; s++) qf[n][s] = valid ? *(const u32x4*)(p + 32 * s) : u32x4{0, 0, 0, 0};
  }
  PIN();
#pragma unroll
  for (int n = 0; n < NQ; n++)
#pragma unroll
    for (int g = 0; g < NG; g++) {
      float sum = 0;
#pragma unroll
      for (int s = 2 * g; s < 2 * g + 2; s++)
#pragma unroll
        for (int k = 0; k < 4; k++)
          sum += Elem<DT>::to_f32((uint16_t)qf[n][s][k]) + Elem<DT>::to_f32((uint16_t)(qf[n][s][k] >> 16));
      sum += lane_xor16(sum);
      sum += lane_xor32(sum);
      const float hi = bf16_bits_to_f32(f32_to_bf16_bits(sum)), mid = bf16_bits_to_f32(f32_to_bf16_bits(sum - hi));
      qsum[n][g] = q == 0 ? uint2{pack_bf16(hi, mid), pack_bf16(sum - hi - mid, 0.0f)} : uint2{0, 0};
    }

  f32x4 acc[NQ][DTILES], off[NQ][NG];
  float m[NQ], l[NQ];
#pragma unroll
  for (int n = 0; n < NQ; n++) {
    m[n] = NEG, l[n] = 0;
#pragma unroll
    for (int d = 0; d < DTILES; d++) acc[n][d] = f32x4{0, 0, 0, 0};
#pragma unroll
    for (int g = 0; g < NG; g++) off[n][g] = f32x4{0, 0, 0, 0};
  }

  // At 256 dims the queries wait in the wave's own part of LDS: in registers they made the loop reload nine others from
  // memory every step (8 sequences of 1K to 16K: 27.4 us, so 23.3).
  constexpr bool QUERIES_IN_LDS = D == 256;
  u32x4* own = (u32x4*)joined[wave] + lane;
  u32x4* own_sums = (u32x4*)joined[wave] + 64 * KS + lane;
  if (QUERIES_IN_LDS) {
    static_assert(D < 256 || (NQ == 1 && 1024 * (KS + NG) <= (int)sizeof(joined[0])), "the wave's part");
#pragma unroll
    for (int s = 0; s < KS; s++) own[64 * s] = qf[0][s];
#pragma unroll
    for (int g = 0; g < NG; g++) own_sums[64 * g] = u32x4{qsum[0][g].x, qsum[0][g].y, 0, 0};
  }
  const uint32_t vmask = code_mask<ANNA_MI_BF16>(), kmask = DT == ANNA_MI_BF16 ? vmask : code_mask<DT>();
  for (; step < end; step += 4) {
    f32x4 z[NQ][TT];
    if (QUERIES_IN_LDS) {
      asm volatile("" ::: "memory");  // read here, not kept
#pragma unroll
      for (int s = 0; s < KS; s++) qf[0][s] = own[64 * s];
    }
#pragma unroll
    for (int t = 0; t < TT; t++) {
#pragma unroll
      for (int g = 0; g < NG; g++) {
        const uint32_t o = k.offset[t][g] * 0x10001u;
        const uint2 s = k.scale[t][g];
        const u32x4 a0 = codes16<DT>(k.code[t][2 * g], kmask), a1 = codes16<DT>(k.code[t][2 * g + 1], kmask);
#pragma unroll
        for (int n = 0; n < NQ; n++) {
          f32x4 c = mfma_bf16(u32x4{o, o, 0, 0}, QUERIES_IN_LDS ? own_sums[64 * g] : u32x4{qsum[n][g].x, qsum[n][g].y, 0, 0}, f32x4{0, 0, 0, 0});
          c = mfma<DT>(a0, qf[n][2 * g], c);
          c = mfma<DT>(a1, qf[n][2 * g + 1], c);
          if (g == 0) z[n][t] = f32x4{bf16_lo(s.x) * c[0], bf16_hi(s.x) * c[1], bf16_lo(s.y) * c[2], bf16_hi(s.y) * c[3]};
          else {
            z[n][t][0] += bf16_lo(s.x) * c[0];
            z[n][t][1] += bf16_hi(s.x) * c[1];
            z[n][t][2] += bf16_lo(s.y) * c[2];
            z[n][t][3] += bf16_hi(s.y) * c[3];
          }
        }
      }
    }
    PIN();
    const uint8_t* page = page_at(next);
    if (step + 4 < end) k.load(page, (step + 4) % STEPS, lane);
    if (step + 8 < end) next = table[(step + 8) / STEPS];
    PIN();
    // online softmax: a lane holds tokens 16 t + 4 q + i of the query in its column
    const int first = step * T;
#pragma unroll
    for (int n = 0; n < NQ; n++) {
      if (first + T > it.start) {  // only steps with tokens of the span hold any that are not seen
        asm volatile("");          // a branch, not a select for every score of every step
#pragma unroll
        for (int t = 0; t < TT; t++)
#pragma unroll
          for (int i = 0; i < 4; i++)
            if (first + t * 16 + 4 * q + i >= limit[n]) z[n][t][i] = NEG;
      }
      float top = NEG;
#pragma unroll
      for (int t = 0; t < TT; t++)
#pragma unroll
        for (int i = 0; i < 4; i++) top = fmaxf(top, z[n][t][i]);
      top = fmaf(top, a.scale, ROOM);
      top = fmaxf(top, lane_xor16(top));
      top = fmaxf(top, lane_xor32(top));
      top = fmaxf(top, m[n]);
      const float base = top == NEG ? 0.0f : top;
      if (__any(top > m[n])) {
        const float f = weight(m[n], base);
        l[n] *= f;
#pragma unroll
        for (int d = 0; d < DTILES; d++) acc[n][d] *= f;
#pragma unroll
        for (int g = 0; g < NG; g++) off[n][g] *= f;
        m[n] = top;
      }
      float sum = 0;
#pragma unroll
      for (int t = 0; t < TT; t++)
#pragma unroll
        for (int i = 0; i < 4; i++) {
          z[n][t][i] = __builtin_amdgcn_exp2f(fmaf(z[n][t][i], a.scale, -base));
          sum += z[n][t][i];
        }
      l[n] += sum;
    }
#pragma unroll
    for (int half = 0; half < T / 32; half++)
#pragma unroll
      for (int g = 0; g < NG; g++) {
        const uint2 s0 = v.scale[half][0][g], s1 = v.scale[half][1][g], o0 = v.offset[half][0][g], o1 = v.offset[half][1][g];
        u32x4 ps[NQ], rest[NQ];
#pragma unroll
        for (int n = 0; n < NQ; n++) {
          const f32x4 x = z[n][2 * half], y = z[n][2 * half + 1];
          const float u[8] = {x[0] * bf16_lo(s0.x), x[1] * bf16_hi(s0.x), x[2] * bf16_lo(s0.y), x[3] * bf16_hi(s0.y),
                              y[0] * bf16_lo(s1.x), y[1] * bf16_hi(s1.x), y[2] * bf16_lo(s1.y), y[3] * bf16_hi(s1.y)};
#pragma unroll
          for (int e = 0; e < 4; e++) {
            ps[n][e] = pack_bf16(u[2 * e], u[2 * e + 1]);
            if (TWO) rest[n][e] = pack_bf16(u[2 * e] - bf16_lo(ps[n][e]), u[2 * e + 1] - bf16_hi(ps[n][e]));
          }
          const u32x4 o = {o0.x, o0.y, o1.x, o1.y};
          off[n][g] = mfma_bf16(o, ps[n], off[n][g]);
          if (TWO) off[n][g] = mfma_bf16(o, rest[n], off[n][g]);
        }
#pragma unroll
        for (int e = 0; e < 4; e++) {
          const u32x4 av = codes16<ANNA_MI_BF16>(v.code[half][g][e], vmask);
#pragma unroll
          for (int n = 0; n < NQ; n++) {
            acc[n][4 * g + e] = mfma_bf16(av, ps[n], acc[n][4 * g + e]);
            if (TWO) acc[n][4 * g + e] = mfma_bf16(av, rest[n], acc[n][4 * g + e]);
          }
        }
      }
    PIN();
    if (step + 4 < end) v.load(page, (step + 4) % STEPS, lane);
    PIN();
  }

  // the waves' results joined, one column tile at a time
#pragma unroll
  for (int n = 0; n < NQ; n++) {
    float sum = l[n];
    sum += lane_xor16(sum);
    sum += lane_xor32(sum);
    const int c = threadIdx.x / 16, row = it.tile * R + 16 * n + c;
    if (n > 0) __syncthreads();
    if (q == 0) wave_m[wave][r] = m[n], wave_l[wave][r] = sum;
#pragma unroll
    for (int d = 0; d < DTILES; d++) *(f32x4*)&joined[wave][r][16 * d + 4 * q] = acc[n][d] + off[n][d / 4];
    u16x4 gate[D / 64];
#pragma unroll
    for (int k = 0; k < D / 64; k++) {
      gate[k] = u16x4{0, 0, 0, 0};
      if (a.gate && it.part < 0 && row < rows)
        gate[k] = gates(a, it.offset + row / G, h * G + row % G, 64 * k + 4 * (threadIdx.x % 16));
    }
    __syncthreads();
    if (row < rows) {
      const float top = fmaxf(fmaxf(wave_m[0][c], wave_m[1][c]), fmaxf(wave_m[2][c], wave_m[3][c]));
      float f[4], total = 0;
#pragma unroll
      for (int w = 0; w < 4; w++) f[w] = weight(wave_m[w][c], top), total += f[w] * wave_l[w][c];
      const int64_t part = it.part < 0 ? 0 : (int64_t)(it.part + 16 * n + c) * H + h;
      const float inv = it.part < 0 ? 1.0f / total : 1.0f;
#pragma unroll
      for (int k = 0; k < D / 64; k++) {
        const int d = 64 * k + 4 * (threadIdx.x % 16);
        f32x4 v = {0, 0, 0, 0};
#pragma unroll
        for (int w = 0; w < 4; w++) v += f[w] * *(const f32x4*)&joined[w][c][d];
        if (it.part < 0) write_out<DT>(a, D, it.offset + row / G, h * G + row % G, d, v * inv, gate[k], (int64_t)H * G);
        else *(f32x4*)(a.values + part * D + d) = v;
      }
      if (it.part >= 0 && threadIdx.x % 16 == 0) a.stats[2 * part] = top, a.stats[2 * part + 1] = total;
    }
  }
}

// ---------------------------------------------------------------- tile form
// NW waves of 32 query rows each share pages through LDS: every page is turned into dense 16-bit
// operands once for all of them.  S^T = K Q^T and O^T = V^T P^T by v_mfma_f32_32x32x16, in fragment
// order in LDS (64 lanes of 16 bytes: no bank conflicts).  K's rows are permuted so that a lane's
// eight tokens of S^T are, in order, its eight k of the second product and one word of value codes:
// row 16 s + 8 u + e of a half page is token 16 u + 8 s + e.
//
// The operands are fp16 for both types: (code + zero) * scale rounded to 11 bits, probabilities (times 2^8, so
// that small ones stay above fp16's subnormals) too, which keeps the result within a tenth of the output's
// own rounding for bf16.  For fp16 they show beside it: 2.9e-4 in all against 2.1e-4 of the output's alone, from
// the probabilities (a second term for them would give that back for 12% of the time), and up to 5e-4 where single
// channels stand out of the keys, whose values then need more than fp16's bits, as a dense cache's would.
// fp16 holds only so much: from the first page on with scales beyond the limits below an item goes on in bf16 instead, at
// bf16's precision.
//
// The vector unit bounds it: of a page and wave (32 rows, head_dim 128) 32 matrix instructions (1024 cycles) stand against
// ~320 vector ones, 32 of them exponentials, and with two waves a SIMD the two overlap in part.  2048 tokens at the end
// of 32K (32 query heads on 8, head_dim 128): 1119 us, 952 TFLOP/s, 80% of a large product's rate (by the card, up to
// 1200); in bf16 from the first page on 1265.  head_dim 256 has room for one wave a SIMD only (its sums alone are 128
// registers): a page of 128 rows takes 3.9 us, ragged prompts of up to 1500 tokens 116 us (343 TFLOP/s).
// Keys go in times 2^K_BITS, up to 121 scales each: below 2^16.  A scale of K_SCALE_LEAST or more is exact so, and a key's
// subnormal rounding stays below a 2^-8th of a code's step.  Smaller ones are off by up to 2^-25, a key by 121 times that, a
// score (D keys, queries below 2^Q_BITS) by D * 2^-7 of its row's scale: with scales up to 2^-3 / D that moves a probability
// by 2^-10.6 of itself at the very most, and only tiles with rows of larger scales need such keys as bf16 holds them.
// (128 dims, scaling 128^-0.5: queries below 64 do not.)
constexpr float K_SCALE_MOST = 64.0f;
constexpr int K_BITS = 3;
constexpr uint32_t K_SCALE_LEAST = 0x3580;  // bf16's 2^-20
constexpr float V_SCALE_MOST = 256.0f;               // |v| < 2^15
constexpr float V_SCALE_LEAST = 7.62939453125e-6f;   // 2^-17: exact in fp16, subnormal roundings below a 2^-8th of a code's step
constexpr float V_SHRINK = 0.0625f;                  // in bf16: rounded, a group's largest value may be past the type's largest
constexpr int Q_BITS = 11;
constexpr float SCALE_LEAST = 1.1754943508222875e-38f, SCALE_MOST = 3.4028234663852886e38f;  // 2^-126, the largest
constexpr float P_SHIFT = 8.0f, P_SLACK = 4.0f;

// (code + zero) * scale of a pair: the sum is exact, the product rounded once.
__device__ __forceinline__ uint32_t scaled(uint32_t code16, uint32_t offset, uint32_t scale) {
  return __builtin_bit_cast(uint32_t, (__builtin_bit_cast(f16x2, code16) + __builtin_bit_cast(f16x2, offset)) * __builtin_bit_cast(f16x2, scale));
}

template <bool F16> __device__ __forceinline__ f32x16 mfma32(u32x4 a, u32x4 b, f32x16 c) {
  if constexpr (F16) return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  else return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

// What a thread holds of a page until it goes to LDS: the codes of a token's keys (by 16-token quarters of a page)
// and of 16-byte words of values (by halves and groups: UNITS of them a page), with their scales and offsets as
// loaded, and as the pairs that the conversion takes (in the same registers, once the loads are in).
template <int D> struct KeyShare {
  static constexpr int NG = D / GROUP, KW = D / 32;
  uint32_t code[KW];
  uint32_t scale[NG], offset[NG];
  __device__ __forceinline__ void load(const uint8_t* page, int quarter, uint32_t lane) {
    const uint32_t q = lane / 16, r = lane % 16;
    __builtin_memcpy(code, __builtin_assume_aligned(page + quarter * 8 * D + (r * (D / 2) + q * (D / 8)), D / 8 < 16 ? D / 8 : 16), D / 8);
    const uint8_t* row = page + quarter * 32 * NG;
#pragma unroll
    for (int g = 0; g < NG; g++) {
      scale[g] = *(const uint16_t*)(row + (K_SCALES * D + ((r / 4) * NG * 4 + r % 4) * 2) + g * 8);
      offset[g] = *(const uint16_t*)(row + (K_OFFSETS * D + r * NG * 2) + g * 2);
    }
  }
  // The page's tokens from `seen` on become zeros.
  __device__ __forceinline__ void hide_from(int seen, int quarter, uint32_t lane) {
#pragma unroll
    for (int g = 0; g < NG; g++)
      if (16 * quarter + (int)(lane % 16) >= seen) scale[g] = 0;
  }
  // Beyond what fp16 holds; least: bf16 bits of the smallest scale but 0.
  __device__ __forceinline__ bool wide(uint32_t least) const {
    float most = bf16_lo(scale[0]);
    uint32_t smallest = scale[0] - 1;
#pragma unroll
    for (int g = 1; g < NG; g++) most = fmaxf(most, bf16_lo(scale[g])), smallest = min(smallest, scale[g] - 1);
    return most > K_SCALE_MOST || smallest < least - 1;
  }
  __device__ __forceinline__ void convert() {
#pragma unroll
    for (int g = 0; g < NG; g++) {
      const _Float16 s = (_Float16)(bf16_lo(scale[g]) * (1 << K_BITS));
      scale[g] = __builtin_bit_cast(uint32_t, f16x2{s, s});
      offset[g] = __builtin_bit_cast(uint32_t, f16x2{(_Float16)bf16_lo(offset[g]), (_Float16)bf16_lo(offset[g])});
    }
  }
  // Where word 0 goes (the dims 8 q + e of a token); word k (the dims 32 k further) 2 k fragments behind it.  Rows in LDS
  // are permuted as said above.
  static __device__ __forceinline__ int at(int quarter, int lane) {
    const int q = lane / 16, r = lane % 16, row = 16 * (r / 8) + 8 * (quarter & 1) + r % 8;
    return ((quarter / 2) * 2 * KW + q / 2) * 64 + (q & 1) * 32 + row;
  }
  __device__ __forceinline__ void put_f16(u32x4* to, int k, uint32_t mask) const {
    u32x4 c = codes16<ANNA_MI_F16>(code[k], mask);
#pragma unroll
    for (int i = 0; i < 4; i++) c[i] = scaled(c[i], offset[k / 2], scale[k / 2]);
    to[128 * k] = c;
  }
  __device__ __forceinline__ void put_bf16(u32x4* to, int k) const {
    const u32x4 c = codes16<ANNA_MI_BF16>(code[k], 0x00780078u);
    const float s = bf16_lo(scale[k / 2]), o = bf16_lo(offset[k / 2]);
    u32x4 v;
#pragma unroll
    for (int i = 0; i < 4; i++) v[i] = pack_bf16((bf16_lo(c[i]) + o) * s, (bf16_hi(c[i]) + o) * s);
    to[128 * k] = v;
  }
};
template <int D> struct ValueShare {
  static constexpr int NG = D / GROUP;
  u32x4 code;
  uint32_t scale[4], offset[4];  // of the tokens' pairs
  __device__ __forceinline__ void load(const uint8_t* page, int unit, uint32_t lane) {
    const uint32_t q = lane / 16, half = unit / NG, g = unit % NG;
    code = *(const u32x4*)(page + unit * 1024 + (V_CODES * D + lane * 16));
    const uint8_t* row = page + half * 64 * NG + g * 8;
#pragma unroll
    for (int u = 0; u < 2; u++) {
      const uint2 s = *(const uint2*)(row + u * 32 * NG + (V_SCALES * D + q * NG * 8));
      const uint2 o = *(const uint2*)(row + u * 32 * NG + (V_OFFSETS * D + q * NG * 8));
      scale[2 * u] = s.x, scale[2 * u + 1] = s.y, offset[2 * u] = o.x, offset[2 * u + 1] = o.y;
    }
  }
  __device__ __forceinline__ void hide_from(int seen, int unit, uint32_t lane) {
    const int first = unit / NG * 32 + (int)(lane / 16) * 4;
#pragma unroll
    for (int k = 0; k < 4; k++) {
      const int token = first + k / 2 * 16 + k % 2 * 2;
      scale[k] &= (token < seen ? 0xFFFFu : 0u) | (token + 1 < seen ? 0xFFFF0000u : 0u);
    }
  }
  __device__ __forceinline__ bool wide() const {
    // the scales are finite and not negative: their bits are in their order; 0 goes to the end by the 1 taken off
    typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
    u16x2 most = __builtin_bit_cast(u16x2, scale[0]), least = most - (uint16_t)1;
#pragma unroll
    for (int k = 1; k < 4; k++) {
      const u16x2 x = __builtin_bit_cast(u16x2, scale[k]);
      most = __builtin_elementwise_max(most, x);
      least = __builtin_elementwise_min(least, (u16x2)(x - (uint16_t)1));
    }
    constexpr uint32_t MOST = __builtin_bit_cast(uint32_t, V_SCALE_MOST) >> 16, LEAST = (__builtin_bit_cast(uint32_t, V_SCALE_LEAST) >> 16) - 1;
    return (int)(max(most[0], most[1]) > MOST) | (int)(min(least[0], least[1]) < LEAST);
  }
  __device__ __forceinline__ void convert() {
#pragma unroll
    for (int k = 0; k < 4; k++) {
      scale[k] = __builtin_bit_cast(uint32_t, f16x2{(_Float16)bf16_lo(scale[k]), (_Float16)bf16_hi(scale[k])});
      offset[k] = __builtin_bit_cast(uint32_t, f16x2{(_Float16)bf16_lo(offset[k]), (_Float16)bf16_hi(offset[k])});
    }
  }
  // Where word 0 goes (dim r of the group); word w (the dims 16 w further) 16 rows or a dim tile behind it.
  static __device__ __forceinline__ int at(int unit, int lane) {
    const int half = unit / NG, g = unit % NG, q = lane / 16, r = lane % 16;
    return 8 * D + ((half * (D / 32) + 2 * g) * 2 + q / 2) * 64 + (q & 1) * 32 + r;
  }
  __device__ __forceinline__ void put_f16(u32x4* to, int w, uint32_t mask) const {
    u32x4 c = codes16<ANNA_MI_F16>(code[w], mask);
#pragma unroll
    for (int i = 0; i < 4; i++) c[i] = scaled(c[i], offset[i], scale[i]);
    to[128 * (w / 2) + 16 * (w & 1)] = c;
  }
  __device__ __forceinline__ void put_bf16(u32x4* to, int w) const {
    const u32x4 c = codes16<ANNA_MI_BF16>(code[w], 0x00780078u);
    u32x4 v;
#pragma unroll
    for (int i = 0; i < 4; i++)
      v[i] = pack_bf16((bf16_lo(c[i]) + bf16_lo(offset[i])) * (bf16_lo(scale[i]) * V_SHRINK),
                       (bf16_hi(c[i]) + bf16_hi(offset[i])) * (bf16_hi(scale[i]) * V_SHRINK));
    to[128 * (w / 2) + 16 * (w & 1)] = v;
  }
};

// LDS of a buffer: keys then values, 128 * D bytes each.
template <int D> constexpr int buffer_words() { return 2 * 128 * D / 16; }

// On their way out, 32 rows of UNITS four-value units stand in a wave's share of LDS, a row's units turned by the row's
// number, so that neighbouring rows' same unit meets other banks; the turn stays within the row.
template <int UNITS> constexpr int out_unit(int row, int unit) { return row * UNITS + (unit ^ (row & (UNITS < 16 ? UNITS - 1 : 15))); }
template <int UNITS> constexpr bool one_to_one() {
  bool taken[32 * UNITS] = {};
  for (int i = 0; i < 32 * UNITS; i++) {
    const int at = out_unit<UNITS>(i / UNITS, i % UNITS);
    if (at < 0 || at >= 32 * UNITS || taken[at]) return false;
    taken[at] = true;
  }
  return true;
}

// A wave's state: its 32 query rows.
template <int D> struct Rows {
  f32x16 acc[D / 32];
  float m, l;
};

// The running maximum of a lane's query with the scores `top` added, for fp16 less P_SHIFT: P_SHIFT above it the
// probabilities would be 2^P_SHIFT; for bf16 with ROOM instead.  It moves only when it has to, by more than P_SLACK,
// which leaves them within fp16 and spares nearly all rescaling.  Returns the factor of everything summed so far.
template <int D, bool F16> __device__ __forceinline__ bool new_top(Rows<D>& w, float top, float scale, float& factor) {
  top = fmaxf(top, lane_xor32(top));
  top = fmaf(top, scale, F16 ? -P_SHIFT : ROOM);
  const bool moves = top > w.m + P_SLACK;
  factor = 1.0f;
  if (!__any(moves)) return false;
  if (moves) {
    factor = weight(w.m, top);
    w.m = top;
  }
  return true;
}
__device__ __forceinline__ float top_of(const f32x16& z) {
  float top = NEG;
#pragma unroll
  for (int j = 0; j < 16; j++) top = fmaxf(top, z[j]);
  return top;
}
// Token of a half page that row j of a lane's scores stands for.
__device__ __forceinline__ int token_of(int j, int hl) { return 16 * ((j >> 2) & 1) + 8 * (j >> 3) + 4 * hl + (j & 3); }
__device__ __forceinline__ void hide_from(f32x16& z, int half, int hl, int limit) {
#pragma unroll
  for (int j = 0; j < 16; j++)
    if (32 * half + token_of(j, hl) >= limit) z[j] = NEG;
}
// Two neighbouring probabilities of a lane, as a pair of the operand type.
template <bool F16> __device__ __forceinline__ uint32_t probability(const f32x16& z, int j, float scale, float base, float& sum) {
  const float x = __builtin_amdgcn_exp2f(fmaf(z[j], scale, -base)), y = __builtin_amdgcn_exp2f(fmaf(z[j + 1], scale, -base));
  sum += x + y;
  if (!F16) return pack_bf16(x, y);
  return __builtin_bit_cast(uint32_t, f16x2{(_Float16)x, (_Float16)y});
}

// One page in LDS for a wave's rows.  limit: tokens of the page that the lane's query sees; cut: whether any lane's
// is below PAGE.  The two halves of the page go through one behind the other, so that the vector unit's softmax of
// one runs beneath the matrix instructions of the other, and the next page's conversion beneath the rest:
//   scores 0, first(k) | scores 1, softmax 0 | values 0, softmax 1 | values 1, second(k)
// Every step k is a pair of matrix instructions, a pair of fragments AHEAD steps ahead, and a share of the vector
// work; the order is pinned, as the compiler left to itself reads all fragments first and spills.
template <int D, bool F16, int AHEAD, class Q, class A, class B>
__device__ __forceinline__ void take_page(Rows<D>& w, const u32x4* lds, Q query, int limit, bool cut, float scale, int lane, A first,
                                          B second) {
  constexpr int KSTEPS = D / 16, DTILES = D / 32;
  constexpr int KHALF = KSTEPS / 2, VHALF = DTILES, VSTEPS = 2 * DTILES, RING = AHEAD + 1;
  const int hl = lane / 32;
  const u32x4* values = lds + 8 * D;
  f32x16 z[2];
#pragma unroll
  for (int half = 0; half < 2; half++)
#pragma unroll
    for (int j = 0; j < 16; j++) z[half][j] = 0;
  u32x4 f[RING][2], p[4];
  float sum = 0, base = 0, factor[2];
  bool moved[2];
  // step i of the scores: two k steps of half i / KHALF; of the values: two dim tiles of 16 tokens
  auto read = [&](int i) {
#pragma unroll
    for (int u = 0; u < 2; u++) {
      if (i < KSTEPS) f[i % RING][u] = lds[(i / KHALF * KSTEPS + 2 * (i % KHALF) + u) * 64 + lane];
      else if (i < KSTEPS + VSTEPS) {
        const int k = (i - KSTEPS) / (DTILES / 2), d = 2 * ((i - KSTEPS) % (DTILES / 2)) + u;
        f[i % RING][u] = values[(((k / 2) * DTILES + d) * 2 + (k & 1)) * 64 + lane];
      }
    }
  };
  auto reference = [&](int half) {
    if (cut) {
      asm volatile("");  // a branch, not a select for every score of every page
      hide_from(z[half], half, hl, limit);
    }
    moved[half] = new_top<D, F16>(w, top_of(z[half]), scale, factor[half]);
    base = w.m == NEG ? 0.0f : w.m;
  };
  auto rescale = [&](int half) {
    if (moved[half]) {
#pragma unroll
      for (int d = 0; d < DTILES; d++) w.acc[d] *= factor[half];
    }
  };
  // share i of n of a half's eight pairs of probabilities
  auto probabilities = [&](int half, int i, int n) {
#pragma unroll
    for (int k = 8 * i / n; k < 8 * (i + 1) / n; k++) p[2 * half + k / 4][k % 4] = probability<F16>(z[half], 2 * k, scale, base, sum);
  };
#pragma unroll
  for (int i = 0; i < AHEAD; i++) read(i);
#pragma unroll
  for (int i = 0; i < KSTEPS; i++) {
    if (i == KHALF) {
      first(KHALF);
      PIN();
      reference(0);
      w.l *= factor[0];
      rescale(0);
      PIN();
    }
    read(i + AHEAD);
#pragma unroll
    for (int u = 0; u < 2; u++) z[i / KHALF] = mfma32<F16>(f[i % RING][u], query(2 * (i % KHALF) + u), z[i / KHALF]);
    if (i < KHALF) first(i);
    else probabilities(0, i - KHALF, KHALF);
    PIN();
  }
  reference(1);
  PIN();
  const float sum0 = sum;
  sum = 0;
#pragma unroll
  for (int i = 0; i < VSTEPS; i++) {
    if (i == VHALF) {
      w.l = (w.l + sum0) * factor[1] + sum;
      rescale(1);
      PIN();
    }
    read(KSTEPS + i + AHEAD);
#pragma unroll
    for (int u = 0; u < 2; u++) {
      const int d = 2 * (i % (DTILES / 2)) + u;
      w.acc[d] = mfma32<F16>(f[(KSTEPS + i) % RING][u], p[i / (DTILES / 2)], w.acc[d]);
    }
    if (i < VHALF) probabilities(1, i, VHALF);
    else second(i - VHALF);
    PIN();
  }
  second(VHALF);
}

template <int DT, int D, int NW>
__global__ __launch_bounds__(64 * NW) void paged_tile_kernel(const Attend a) {
  constexpr int NG = D / GROUP, KSTEPS = D / 16, KW = D / 32, UNITS = 2 * NG;
  // Waves 0 to 3 turn keys, the last ones values: with 8 waves a wave has one of the two, with 4 all have both.
  constexpr int VALUES = (UNITS + NW - 1) / NW, AHEAD = NW == 4 ? 2 : 1;
  __shared__ __align__(16) u32x4 lds[2 * buffer_words<D>()];
  __shared__ int wide[4];  // by page % 4: a scale is beyond what fp16 holds
  const int H = a.kv_heads, G = a.group;
  const int h = blockIdx.x % H, index = blockIdx.x / H;
  const Item it = a.tile[index];
  if (index >= a.header[1]) return;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), lane = threadIdx.x % 64, hl = lane / 32;
  const int rows = it.count * G, row0 = it.tile * 32 * NW + 32 * wave, row = row0 + lane % 32, t = row / G;
  const bool valid = row < rows;
  const int32_t* table = a.table + it.row * a.width;
  const int head = h * G + row % G;
  auto page_at = [&](int32_t page) { return a.pool + ((int64_t)page * H + h) * page_bytes(D); };

  union Held {  // with 8 waves one of the two
    KeyShare<D> keys;
    ValueShare<D> values;
  };
  struct Both {
    KeyShare<D> keys;
    ValueShare<D> values[VALUES];
  };
  std::conditional_t<NW == 8, Held, Both> held;
  KeyShare<D>& keys = held.keys;
  ValueShare<D>* values;
  if constexpr (NW == 8) values = &held.values;
  else values = held.values;
  const bool has_keys = NW == 4 || wave < 4;
  auto unit_of = [&](int n) { return NW - 1 - wave + n * NW; };
  auto has_unit = [&](int n) { return (n + 1) * NW <= UNITS || unit_of(n) < UNITS; };
  auto load_keys = [&](int32_t id) {
    if (has_keys) keys.load(page_at(id), wave, lane);
  };
  auto load_values = [&](int32_t id) {
#pragma unroll
    for (int n = 0; n < VALUES; n++)
      if (has_unit(n)) values[n].load(page_at(id), unit_of(n), lane);
  };
  auto page_id = [&](int p) { return table[min(p, it.page1 - 1)]; };
  int32_t next = page_id(it.page0);
  load_keys(next);
  load_values(next);
  next = page_id(it.page0 + 1);

  const uint16_t* source = (const uint16_t*)a.query + (int64_t)(it.offset + t) * a.q_token + head * a.q_head + hl * 8;
  auto raw_query = [&](int s) { return valid ? *(const u32x4*)(source + 16 * s) : u32x4{0, 0, 0, 0}; };
  u32x4 qf[KSTEPS];
#pragma unroll
  for (int s = 0; s < KSTEPS; s++) qf[s] = raw_query(s);
  if (threadIdx.x < 4) wide[threadIdx.x] = 0;
  // A row's queries go in times a power of two that brings its largest to 2^(Q_BITS - 1) or above, below 2^Q_BITS, and its
  // scores' scale takes that back: whatever their size, no value that could show is lost, and no row has a say in another's.
  typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
  u16x2 most = {0, 0};
#pragma unroll
  for (int s = 0; s < KSTEPS; s++)
#pragma unroll
    for (int k = 0; k < 4; k++) most = __builtin_elementwise_max(most, __builtin_bit_cast(u16x2, qf[s][k] & 0x7FFF7FFFu));
  int largest = max(most[0], most[1]);
  largest = max(largest, lane_xor32(largest));
  // the exponent of zeros, infinities and NaN is 0
  const int shift = Q_BITS - __builtin_amdgcn_frexp_expf(Elem<DT>::to_f32((uint16_t)largest));
#pragma unroll
  for (int s = 0; s < KSTEPS; s++)
#pragma unroll
    for (int k = 0; k < 4; k++) {
      const float x = ldexpf(Elem<DT>::to_f32((uint16_t)qf[s][k]), shift), y = ldexpf(Elem<DT>::to_f32((uint16_t)(qf[s][k] >> 16)), shift);
      qf[s][k] = __builtin_bit_cast(uint32_t, f16x2{(_Float16)x, (_Float16)y});
    }
  // neither 0 nor infinite, as scores that are not seen are -infinity: beyond these it makes no difference to finite ones
  float scale = __builtin_amdgcn_fmed3f(ldexpf(a.scale, -shift - K_BITS), SCALE_LEAST, SCALE_MOST);
  const bool counts = largest > 0 && largest < (DT == ANNA_MI_BF16 ? 0x7F80 : 0x7C00);  // not for its row alone
  const uint32_t key_least = __syncthreads_or(counts && scale > 0.125f / D) ? K_SCALE_LEAST : 1;
  auto query = [&](int s) { return qf[s]; };

  Rows<D> w;
  w.m = NEG, w.l = 0;
#pragma unroll
  for (int d = 0; d < D / 32; d++)
#pragma unroll
    for (int j = 0; j < 16; j++) w.acc[d][j] = 0;

  // The loads of page p are in: a flag if it is none for fp16, and the scales as fp16.  What no row of the tile sees has no
  // say in that: it is the sequence's later tokens, or what the page held before.
  const int seen_by_any = it.start + (min((it.tile + 1) * 32 * NW, rows) - 1) / G + 1;
  auto not_ahead = [](int x) {  // nothing that follows from it is computed before the loop, to be kept in registers
    asm volatile("" : "+v"(x));
    return x;
  };
  auto convert_keys = [&](int p) {
    if (!has_keys) return;
    if (p * PAGE + PAGE > seen_by_any) keys.hide_from(seen_by_any - p * PAGE, wave & 3, not_ahead(lane));
    if (__any(keys.wide(key_least))) wide[p & 3] = 1;
    keys.convert();
  };
  auto convert_values = [&](int p) {
    bool beyond = false;
#pragma unroll
    for (int n = 0; n < VALUES; n++)
      if (has_unit(n)) {
        if (p * PAGE + PAGE > seen_by_any) values[n].hide_from(seen_by_any - p * PAGE, unit_of(n), not_ahead(lane));
        beyond |= values[n].wide();
        values[n].convert();
      }
    if (__any(beyond)) wide[p & 3] = 1;
  };
  const uint32_t mask = code_mask<ANNA_MI_F16>();
  const int key_at = KeyShare<D>::at(wave & 3, lane);
  int value_at[VALUES];
#pragma unroll
  for (int n = 0; n < VALUES; n++) value_at[n] = ValueShare<D>::at(has_unit(n) ? unit_of(n) : 0, lane);
  auto put_key = [&](u32x4* to, int k) {
    if (has_keys) keys.put_f16(to + key_at, k, mask);
  };
  auto put_value = [&](u32x4* to, int k) {
    if (has_unit(k / 4)) values[k / 4].put_f16(to + value_at[k / 4], k % 4, mask);
  };
  // LDS only: loads of the next page stay in flight
  auto barrier = [] { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); };

  const int seen_by_all = it.start + row0 / G + 1;                                 // tokens that the wave's first row sees
  const int last = row0 < rows ? it.start + min(row0 + 31, rows - 1) / G + 1 : 0;  // and its last
  const int sees = valid ? it.start + t + 1 : 0;

  convert_keys(it.page0);
  convert_values(it.page0);
#pragma unroll
  for (int k = 0; k < KW; k++) put_key(lds, k);
#pragma unroll
  for (int k = 0; k < 4 * VALUES; k++) put_value(lds, k);
  load_keys(next);
  load_values(next);
  next = page_id(it.page0 + 2);
  barrier();
  int p = it.page0;
  // A condition that always holds, but that the compiler takes to differ by lanes: without it, it keeps the two loops' sums
  // apart, in 30 registers more (at 256 dims in memory).
  int on = 1;
  asm volatile("" : "+v"(on));
  for (; p < it.page1 && on && __builtin_amdgcn_readfirstlane(wide[p & 3]) == 0; p++) {
    const int turn = (p - it.page0) & 1;
    u32x4 *now = lds + turn * buffer_words<D>(), *then = lds + (turn ^ 1) * buffer_words<D>();
    if (threadIdx.x == 0) wide[(p + 2) & 3] = 0;
    // The next page's values are converted in the first quarter of this one, its keys in the last; the loads of the
    // page after it follow each, and have a page's time to arrive.  Behind the last page all this goes on with the last
    // one, for nobody: a load that is not always there would have the compiler wait for all of them.
    constexpr int KHALF = KSTEPS / 2, VHALF = D / 32;
    auto first = [&](int i) {
      constexpr int PER = (4 * VALUES + KHALF - 1) / KHALF;
      if (i == 0) convert_values(p + 1);
#pragma unroll
      for (int k = i * PER; k < (i + 1) * PER; k++)
        if (k < 4 * VALUES) put_value(then, k);
      if (i == KHALF) load_values(next);
    };
    auto second = [&](int i) {
      constexpr int PER = (KW + VHALF - 1) / VHALF;
      if (i == 0) convert_keys(p + 1);
#pragma unroll
      for (int k = i * PER; k < (i + 1) * PER; k++)
        if (k < KW) put_key(then, k);
      if (i == VHALF) {
        load_keys(next);
        next = page_id(p + 3);
      }
    };
    if (p * PAGE < last) {
      take_page<D, true, AHEAD>(w, now, query, sees - p * PAGE, p * PAGE + PAGE > seen_by_all, scale, lane, first, second);
    } else {
#pragma unroll
      for (int i = 0; i <= KHALF; i++) first(i);
#pragma unroll
      for (int i = 0; i <= VHALF; i++) second(i);
    }
    barrier();
  }
  // From the first page on that fp16 does not hold, in bf16: one buffer, nothing ahead; the probabilities with ROOM
  // instead of P_SHIFT, the values at V_SHRINK until the end.
  if (p < it.page1) {
    constexpr float LESS = 1.0f / (1ull << (int)(P_SHIFT + ROOM));
    w.m += P_SHIFT + ROOM;
    w.l *= LESS;
    scale = a.scale;
#pragma unroll
    for (int d = 0; d < D / 32; d++) w.acc[d] *= LESS * V_SHRINK;
#pragma unroll
    for (int s = 0; s < KSTEPS; s++) {
      qf[s] = raw_query(s);
      if (DT == ANNA_MI_F16) {
#pragma unroll
        for (int k = 0; k < 4; k++) qf[s][k] = pack_bf16(f16_bits_to_f32((uint16_t)qf[s][k]), f16_bits_to_f32((uint16_t)(qf[s][k] >> 16)));
      }
    }
    for (; p < it.page1; p++) {
      const uint8_t* page = page_at(table[p]);
      if (NW == 4 || wave < 4) {
        KeyShare<D> again;
        again.load(page, wave, lane);
#pragma unroll
        for (int i = 0; i < KW; i++) again.put_bf16(lds + key_at, i);
      }
      for (int k = NW - 1 - wave; k < UNITS; k += NW) {
        ValueShare<D> again;
        again.load(page, k, lane);
#pragma unroll
        for (int i = 0; i < 4; i++) again.put_bf16(lds + ValueShare<D>::at(k, lane), i);
      }
      barrier();
      if (p * PAGE < last)
        take_page<D, false, 1>(w, lds, query, sees - p * PAGE, p * PAGE + PAGE > seen_by_all, scale, lane, [](int) {}, [](int) {});
      barrier();
    }
#pragma unroll
    for (int d = 0; d < D / 32; d++) w.acc[d] *= 1.0f / V_SHRINK;
  }

  // A lane holds, of its query, dims 32 d + 8 b + 4 hl + i.  Through LDS, as fp32, to whole rows: lanes that write 8
  // bytes of 32 rows each took 13 us a workgroup (128 rows of head_dim 256, gated).
  const float total = w.l + lane_xor32(w.l);
  if (it.part >= 0) {
    if (!valid) return;
    const int64_t part = (int64_t)(it.part + 32 * wave + lane % 32) * H + h;
#pragma unroll
    for (int d = 0; d < D / 32; d++)
#pragma unroll
      for (int b = 0; b < 4; b++)
        *(f32x4*)(a.values + part * D + 32 * d + 8 * b + 4 * hl) = f32x4{w.acc[d][4 * b], w.acc[d][4 * b + 1], w.acc[d][4 * b + 2], w.acc[d][4 * b + 3]};
    if (hl == 0) a.stats[2 * part] = w.m, a.stats[2 * part + 1] = total;
    return;
  }
  constexpr int PART = 4 * D / NW, UNITS4 = PART / 4;  // dims of a pass: what the wave's share of LDS holds for 32 rows
  constexpr int LANES = PART / 8, STEP = 64 / LANES, N = 32 / STEP;  // lanes of a row, eight dims each; rows at once
  static_assert(one_to_one<UNITS4>() && NW * 32 * UNITS4 <= 2 * buffer_words<D>(), "a place of its own for every unit");
  f32x4* mine = (f32x4*)lds + wave * 32 * UNITS4;
  const float inv = 1.0f / total;
  const int c = lane % LANES, r0 = lane / LANES, first_row = row0 + r0, step_t = STEP / G, step_h = STEP % G;
  // what a lane writes: rows first_row + i STEP, their tokens and heads without a division each
  auto each_row = [&](auto f) {
    int token = first_row / G, out_head = first_row % G;
#pragma unroll
    for (int i = 0; i < N; i++) {
      f(i, first_row + i * STEP < rows, (int64_t)it.offset + token, h * G + out_head);
      token += step_t;
      out_head += step_h;
      if (out_head >= G) out_head -= G, token++;
    }
  };
#pragma unroll
  for (int pass = 0; pass < D / PART; pass++) {
    const int dim = pass * PART + 8 * c;
    u32x4 gate[N];  // all asked for at once
    if (a.gate)
      each_row([&](int i, bool ours, int64_t token, int head) {
        gate[i] = u32x4{0, 0, 0, 0};
        if (ours) gate[i] = *(const u32x4*)((const uint16_t*)a.gate + token * a.g_token + head * a.g_head + dim);
      });
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // the last pass is read
#pragma unroll
    for (int d = 0; d < PART / 32; d++)
#pragma unroll
      for (int b = 0; b < 4; b++) {
        const f32x16& x = w.acc[pass * (PART / 32) + d];
        const int unit = 8 * d + 2 * b + hl;
        mine[out_unit<UNITS4>(lane % 32, unit)] = f32x4{x[4 * b], x[4 * b + 1], x[4 * b + 2], x[4 * b + 3]} * inv;
      }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    each_row([&](int i, bool ours, int64_t token, int head) {
      const int r = r0 + i * STEP;
      const f32x4 x = mine[out_unit<UNITS4>(r, 2 * c)], y = mine[out_unit<UNITS4>(r, 2 * c + 1)];
      float v[8] = {x[0], x[1], x[2], x[3], y[0], y[1], y[2], y[3]};
      if (a.gate) {
#pragma unroll
        for (int k = 0; k < 4; k++) {
          v[2 * k] *= sigmoid(Elem<DT>::to_f32((uint16_t)gate[i][k]));
          v[2 * k + 1] *= sigmoid(Elem<DT>::to_f32((uint16_t)(gate[i][k] >> 16)));
        }
      }
      u32x4 o;
#pragma unroll
      for (int k = 0; k < 4; k++) o[k] = Elem<DT>::cvt(v[2 * k]) | (uint32_t)Elem<DT>::cvt(v[2 * k + 1]) << 16;
      if (ours) *(u32x4*)((uint16_t*)a.out + (token * H * G + head) * D + dim) = o;
    });
  }
}

// Joins the items of a tile: one workgroup a query row, its eight teams of D / 4 lanes each every eighth item, AHEAD
// of them in flight.  Latency bounds it: with four teams the batch of eight took 6.6 us here, with eight 5.4.
template <int DT, int D>
__global__ __launch_bounds__(2 * D) void paged_merge_kernel(const Attend a) {
  constexpr int LANES = D / 4, TEAMS = 8, AHEAD = 4;
  __shared__ __align__(16) float joined[TEAMS][D];
  __shared__ float team_m[TEAMS], team_l[TEAMS];
  const int H = a.kv_heads, G = a.group, h = blockIdx.x % H, index = blockIdx.x / H;
  const Unit u = a.units[index];
  if (index >= a.header[2]) return;
  const int row = blockIdx.y;
  if (row >= u.rows) return;
  const int team = threadIdx.x / LANES, d = threadIdx.x % LANES * 4;
  const int r = u.row0 + row, head = h * G + r % G;
  const int64_t token = u.offset + r / G;
  u16x4 gate = {0, 0, 0, 0};
  if (a.gate && team == 0) gate = gates(a, token, head, d);
  float top = NEG, total = 0;
  f32x4 v = {0, 0, 0, 0};
  for (int k0 = team; k0 < u.splits; k0 += TEAMS * AHEAD) {
    float m[AHEAD], l[AHEAD];
    f32x4 x[AHEAD];
#pragma unroll
    for (int k = 0; k < AHEAD; k++) {
      m[k] = NEG, l[k] = 0, x[k] = f32x4{0, 0, 0, 0};
      if (k0 + k * TEAMS < u.splits) {
        const int64_t part = (int64_t)(u.part + (k0 + k * TEAMS) * u.rows + row) * H + h;
        m[k] = a.stats[2 * part], l[k] = a.stats[2 * part + 1];
        x[k] = *(const f32x4*)(a.values + part * D + d);
      }
    }
    float next = top;
#pragma unroll
    for (int k = 0; k < AHEAD; k++) next = fmaxf(next, m[k]);
    float f = weight(top, next);
    total *= f;
    v *= f;
#pragma unroll
    for (int k = 0; k < AHEAD; k++) {
      f = weight(m[k], next);
      total += l[k] * f;
      v += x[k] * f;
    }
    top = next;
  }
  *(f32x4*)&joined[team][d] = v;
  if (d == 0) team_m[team] = top, team_l[team] = total;
  __syncthreads();
  if (team != 0) return;
#pragma unroll
  for (int k = 1; k < TEAMS; k++) {
    const float m = team_m[k], next = fmaxf(top, m), f0 = weight(top, next), f1 = weight(m, next);
    total = total * f0 + team_l[k] * f1;
    v = v * f0 + *(const f32x4*)&joined[k][d] * f1;
    top = next;
  }
  write_out<DT>(a, D, token, head, d, v * (1.0f / total), gate, (int64_t)H * G);
}

template <int DT, int D> int launch(const Attend& a, const Grid& g, hipStream_t stream) {
  const unsigned split = (unsigned)(g.split_items * a.kv_heads), tile = (unsigned)(g.tile_items * a.kv_heads);
  if (split > 0) {
    if (g.few_rows == 16) paged_split_kernel<DT, D, 1><<<split, 256, 0, stream>>>(a);
    else if constexpr (D <= 128) {  // 4096 / D rows at most
      if (g.few_rows == 32) paged_split_kernel<DT, D, 2><<<split, 256, 0, stream>>>(a);
      else if constexpr (D == 64) paged_split_kernel<DT, D, 4><<<split, 256, 0, stream>>>(a);
    }
  }
  if (tile > 0) {
    if (g.tile_rows == 128) paged_tile_kernel<DT, D, 4><<<tile, 256, 0, stream>>>(a);
    else if constexpr (D <= 128) paged_tile_kernel<DT, D, 8><<<tile, 512, 0, stream>>>(a);
  }
  if (g.units > 0) paged_merge_kernel<DT, D><<<dim3((unsigned)(g.units * a.kv_heads), (unsigned)g.unit_rows), 2 * D, 0, stream>>>(a);
  ANNA_LAUNCH_CHECK("paged attend");
  return ANNA_MI_OK;
}

}  // namespace

int launch_attend(int dtype, int64_t head_dim, const Attend& a, const Grid& g, hipStream_t stream) {
  if (dtype == ANNA_MI_BF16) {
    if (head_dim == 64) return launch<ANNA_MI_BF16, 64>(a, g, stream);
    if (head_dim == 128) return launch<ANNA_MI_BF16, 128>(a, g, stream);
    return launch<ANNA_MI_BF16, 256>(a, g, stream);
  }
  if (head_dim == 64) return launch<ANNA_MI_F16, 64>(a, g, stream);
  if (head_dim == 128) return launch<ANNA_MI_F16, 128>(a, g, stream);
  return launch<ANNA_MI_F16, 256>(a, g, stream);
}

}  // namespace paged
}  // namespace anna
