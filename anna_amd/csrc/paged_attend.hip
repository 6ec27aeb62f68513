// Attention over the paged 4-bit KV cache (page layout in anna_mi.h).
//
// out = softmax(scaling q K^T) V over the tokens up to and with the query's own, K and V held as
// (code + zero) * scale with one scale and zero for 64 values of a token and head.
//
// Split form.  A workgroup takes the query rows of one KV head (R = 16, 32 or 64 rows: tokens times
// query heads of that KV head) and some of the sequence's pages; each of its four waves takes every
// fourth page with an online softmax of its own, and the waves' results are joined at the end.
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
#include "paged.hpp"

namespace anna {
namespace paged {
namespace {

typedef uint16_t u16x4 __attribute__((ext_vector_type(4)));

constexpr float NEG = -INFINITY;

__device__ __forceinline__ f32x4 mfma_bf16(u32x4 a, u32x4 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
template <int DT> __device__ __forceinline__ f32x4 mfma(u32x4 a, u32x4 b, f32x4 c) {
  if constexpr (DT == ANNA_MI_BF16) return mfma_bf16(a, b, c);
  else return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

// 16 + code of the 8 codes of a word, as operand elements of the type.
template <int DT> __device__ __forceinline__ u32x4 codes16(uint32_t w) {
  if constexpr (DT == ANNA_MI_BF16)
    return u32x4{((w << 3) & 0x00780078u) | 0x41804180u, ((w >> 1) & 0x00780078u) | 0x41804180u,
                 ((w >> 5) & 0x00780078u) | 0x41804180u, ((w >> 9) & 0x00780078u) | 0x41804180u};
  else
    return u32x4{((w << 6) & 0x03C003C0u) | 0x4C004C00u, ((w << 2) & 0x03C003C0u) | 0x4C004C00u,
                 ((w >> 2) & 0x03C003C0u) | 0x4C004C00u, ((w >> 6) & 0x03C003C0u) | 0x4C004C00u};
}

__device__ __forceinline__ float bf16_lo(uint32_t v) { return __uint_as_float(v << 16); }
__device__ __forceinline__ float bf16_hi(uint32_t v) { return __uint_as_float(v & 0xFFFF0000u); }
__device__ __forceinline__ uint32_t pack_bf16(float a, float b) {
  return f32_to_bf16_bits(a) | (uint32_t)f32_to_bf16_bits(b) << 16;
}

// 2^x of the difference to a running maximum that may still be -inf.
__device__ __forceinline__ float weight(float m, float top) { return m == NEG ? 0.0f : __builtin_amdgcn_exp2f(m - top); }

template <int DT> __device__ __forceinline__ float gated(float v, const void* gate, int64_t at) {
  const float g = Elem<DT>::to_f32(((const uint16_t*)gate)[at]);
  return v / (1.0f + __expf(-g));
}

// Four neighbouring values of an output row, gated.
template <int DT>
__device__ __forceinline__ void write_out(const Attend& a, int D, int64_t token, int head, int d, f32x4 v, int64_t heads) {
  if (a.gate) {
#pragma unroll
    for (int i = 0; i < 4; i++) v[i] = gated<DT>(v[i], a.gate, token * a.g_token + head * a.g_head + d + i);
  }
  u16x4 o;
#pragma unroll
  for (int i = 0; i < 4; i++) o[i] = Elem<DT>::cvt(v[i]);
  *(u16x4*)((uint16_t*)a.out + (token * heads + head) * D + d) = o;
}

// NQ: 16-row column tiles of queries.
template <int DT, int D, int NQ>
__global__ __launch_bounds__(256) void paged_split_kernel(const Attend a) {
  constexpr int NG = D / GROUP, KS = D / 32, DTILES = D / 16, R = 16 * NQ;
  constexpr bool TWO = DT == ANNA_MI_F16;  // ps as two bf16 terms
  __shared__ __align__(16) float joined[4][16][D + 4];
  __shared__ float wave_m[4][16], wave_l[4][16];

  const int H = a.kv_heads, G = a.group;
  const int h = blockIdx.x % H, index = blockIdx.x / H;
  if (index >= a.header[0]) return;
  const Item it = a.split[index];
  const int wave = threadIdx.x / 64, lane = threadIdx.x % 64, q = lane / 16, r = lane % 16;
  const int rows = it.count * G;
  const int32_t* table = a.table + it.row * a.width;

  // queries: column r of tile n is row it.tile * R + 16 n + r
  u32x4 qf[NQ][KS];
  u32x4 qsum[NQ][NG];  // the groups' sums as three bf16 terms in k = 0, 1, 2 of the first quarter
  int limit[NQ];       // tokens that the query sees
#pragma unroll
  for (int n = 0; n < NQ; n++) {
    const int row = it.tile * R + 16 * n + r, t = row / G, head = h * G + row % G;
    const bool valid = row < rows;
    limit[n] = valid ? it.start + t + 1 : 0;
    const uint16_t* p = (const uint16_t*)a.query + (int64_t)(it.offset + t) * a.q_token + head * a.q_head + q * 8;
#pragma unroll
    for (int s = 0; s < KS; s++) qf[n][s] = valid ? *(const u32x4*)(p + 32 * s) : u32x4{0, 0, 0, 0};
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
      qsum[n][g] = q == 0 ? u32x4{pack_bf16(hi, mid), pack_bf16(sum - hi - mid, 0.0f), 0, 0} : u32x4{0, 0, 0, 0};
    }
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

  for (int p = it.page0 + wave; p < it.page1; p += 4) {
    const uint8_t* page = a.pool + ((int64_t)table[p] * H + h) * page_bytes(D);
    f32x4 z[NQ][4];
#pragma unroll
    for (int tl = 0; tl < 4; tl++) {
      const uint8_t* kc = page + (tl * 16 + r) * (D / 2) + q * (D / 8);
      uint32_t w[KS];
      __builtin_memcpy(w, __builtin_assume_aligned(kc, D / 8 < 16 ? D / 8 : 16), 4 * KS);
      const uint16_t* ko = (const uint16_t*)(page + K_OFFSETS * D) + (tl * 16 + r) * NG;
      const uint2* ks = (const uint2*)(page + K_SCALES * D) + (tl * 4 + q) * NG;
#pragma unroll
      for (int g = 0; g < NG; g++) {
        const uint32_t o = ko[g] * 0x10001u;
        const uint2 s = ks[g];
        const u32x4 a0 = codes16<DT>(w[2 * g]), a1 = codes16<DT>(w[2 * g + 1]);
#pragma unroll
        for (int n = 0; n < NQ; n++) {
          f32x4 c = mfma_bf16(u32x4{o, o, 0, 0}, qsum[n][g], f32x4{0, 0, 0, 0});
          c = mfma<DT>(a0, qf[n][2 * g], c);
          c = mfma<DT>(a1, qf[n][2 * g + 1], c);
          if (g == 0) z[n][tl] = f32x4{0, 0, 0, 0};
          z[n][tl][0] += bf16_lo(s.x) * c[0];
          z[n][tl][1] += bf16_hi(s.x) * c[1];
          z[n][tl][2] += bf16_lo(s.y) * c[2];
          z[n][tl][3] += bf16_hi(s.y) * c[3];
        }
      }
    }
    // online softmax: a lane holds tokens 16 tl + 4 q + i of the query in its column
#pragma unroll
    for (int n = 0; n < NQ; n++) {
      if (p * PAGE + PAGE > it.start) {  // only pages with tokens of the span hold any that are not seen
#pragma unroll
        for (int tl = 0; tl < 4; tl++)
#pragma unroll
          for (int i = 0; i < 4; i++)
            if (p * PAGE + tl * 16 + 4 * q + i >= limit[n]) z[n][tl][i] = NEG;
      }
      float top = NEG;
#pragma unroll
      for (int tl = 0; tl < 4; tl++)
#pragma unroll
        for (int i = 0; i < 4; i++) top = fmaxf(top, z[n][tl][i]);
      top *= a.scale;
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
      for (int tl = 0; tl < 4; tl++)
#pragma unroll
        for (int i = 0; i < 4; i++) {
          z[n][tl][i] = __builtin_amdgcn_exp2f(fmaf(z[n][tl][i], a.scale, -base));
          sum += z[n][tl][i];
        }
      l[n] += sum;
    }
#pragma unroll
    for (int half = 0; half < 2; half++)
#pragma unroll
      for (int g = 0; g < NG; g++) {
        const int t0 = (half * 8 + q) * NG + g, t1 = (half * 8 + 4 + q) * NG + g;
        const uint2 s0 = ((const uint2*)(page + V_SCALES * D))[t0], s1 = ((const uint2*)(page + V_SCALES * D))[t1];
        const uint2 o0 = ((const uint2*)(page + V_OFFSETS * D))[t0], o1 = ((const uint2*)(page + V_OFFSETS * D))[t1];
        const u32x4 w = ((const u32x4*)(page + V_CODES * D))[(half * NG + g) * 64 + lane];
        u32x4 ps[NQ], rest[NQ];
#pragma unroll
        for (int n = 0; n < NQ; n++) {
          const f32x4 x = z[n][2 * half], y = z[n][2 * half + 1];
          const float v[8] = {x[0] * bf16_lo(s0.x), x[1] * bf16_hi(s0.x), x[2] * bf16_lo(s0.y), x[3] * bf16_hi(s0.y),
                              y[0] * bf16_lo(s1.x), y[1] * bf16_hi(s1.x), y[2] * bf16_lo(s1.y), y[3] * bf16_hi(s1.y)};
#pragma unroll
          for (int k = 0; k < 4; k++) {
            ps[n][k] = pack_bf16(v[2 * k], v[2 * k + 1]);
            if (TWO) rest[n][k] = pack_bf16(v[2 * k] - bf16_lo(ps[n][k]), v[2 * k + 1] - bf16_hi(ps[n][k]));
          }
          const u32x4 o = {o0.x, o0.y, o1.x, o1.y};
          off[n][g] = mfma_bf16(o, ps[n], off[n][g]);
          if (TWO) off[n][g] = mfma_bf16(o, rest[n], off[n][g]);
        }
#pragma unroll
        for (int k = 0; k < 4; k++) {
          const u32x4 av = codes16<ANNA_MI_BF16>(w[k]);
#pragma unroll
          for (int n = 0; n < NQ; n++) {
            acc[n][4 * g + k] = mfma_bf16(av, ps[n], acc[n][4 * g + k]);
            if (TWO) acc[n][4 * g + k] = mfma_bf16(av, rest[n], acc[n][4 * g + k]);
          }
        }
      }
  }

  // the waves' results joined, one column tile at a time
#pragma unroll
  for (int n = 0; n < NQ; n++) {
    float sum = l[n];
    sum += lane_xor16(sum);
    sum += lane_xor32(sum);
    if (n > 0) __syncthreads();
    if (q == 0) wave_m[wave][r] = m[n], wave_l[wave][r] = sum;
#pragma unroll
    for (int d = 0; d < DTILES; d++) *(f32x4*)&joined[wave][r][16 * d + 4 * q] = acc[n][d] + off[n][d / 4];
    __syncthreads();
    const int c = threadIdx.x / 16, row = it.tile * R + 16 * n + c;
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
        if (it.part < 0) write_out<DT>(a, D, it.offset + row / G, h * G + row % G, d, v * inv, (int64_t)H * G);
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
// own rounding.  fp16 holds only so much: a page with scales beyond the limits below, and every page of
// queries above them, is taken in bf16 instead, at bf16's precision.
constexpr float K_SCALE_MOST = 16.0f;                // |k| < 2^11: with |q| <= 2^11 subnormal roundings stay below 2^-14
constexpr float V_SCALE_MOST = 256.0f;               // |v| < 2^15
constexpr float V_SCALE_LEAST = 3.814697265625e-6f;  // 2^-18: subnormal roundings stay below a 2^-7th of a code's step
constexpr float Q_MOST = 2048.0f;
constexpr float P_SHIFT = 8.0f;

typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));

// (code + zero) * scale of a word's 8 codes; offset and scale of each pair of codes.
__device__ __forceinline__ u32x4 dense_f16(uint32_t w, const f16x2* offset, const f16x2* scale, int step) {
  const u32x4 c = codes16<ANNA_MI_F16>(w);
  u32x4 o;
#pragma unroll
  for (int k = 0; k < 4; k++)
    o[k] = __builtin_bit_cast(uint32_t, (__builtin_bit_cast(f16x2, (uint32_t)c[k]) + offset[k * step]) * scale[k * step]);
  return o;
}
__device__ __forceinline__ u32x4 dense_bf16(uint32_t w, const float* offset, const float* scale, int step) {
  const u32x4 c = codes16<ANNA_MI_BF16>(w);
  u32x4 o;
#pragma unroll
  for (int k = 0; k < 4; k++)
    o[k] = pack_bf16((bf16_lo(c[k]) + offset[2 * k * step]) * scale[2 * k * step],
                     (bf16_hi(c[k]) + offset[(2 * k + 1) * step]) * scale[(2 * k + 1) * step]);
  return o;
}
__device__ __forceinline__ f16x2 f16_pair(uint32_t v) { return f16x2{(_Float16)bf16_lo(v), (_Float16)bf16_hi(v)}; }

template <bool F16> __device__ __forceinline__ f32x16 mfma32(u32x4 a, u32x4 b, f32x16 c) {
  if constexpr (F16) return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  else return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

// What a thread holds of a page until it goes to LDS: its share of the codes with their scales and offsets.
// Keys by 16-token quarters of a page, values by 16-byte words of a (half, group): UNITS of each a page.
template <int D> struct Share {
  static constexpr int NG = D / GROUP, KW = D / 32;
  uint32_t kw[KW];
  uint16_t ks[NG], ko[NG];
  u32x4 vw;
  uint2 vs[2], vo[2];
};

template <int D> __device__ __forceinline__ void load_keys(Share<D>& s, const uint8_t* page, int quarter, int lane) {
  constexpr int NG = D / GROUP;
  const int q = lane / 16, r = lane % 16, token = quarter * 16 + r;
  __builtin_memcpy(s.kw, __builtin_assume_aligned(page + token * (D / 2) + q * (D / 8), D / 8 < 16 ? D / 8 : 16), D / 8);
#pragma unroll
  for (int g = 0; g < NG; g++) {
    s.ks[g] = ((const uint16_t*)(page + K_SCALES * D))[((token / 4) * NG + g) * 4 + token % 4];
    s.ko[g] = ((const uint16_t*)(page + K_OFFSETS * D))[token * NG + g];
  }
}
template <int D> __device__ __forceinline__ void load_values(Share<D>& s, const uint8_t* page, int unit, int lane) {
  constexpr int NG = D / GROUP;
  const int half = unit / NG, g = unit % NG, q = lane / 16;
  s.vw = ((const u32x4*)(page + V_CODES * D))[unit * 64 + lane];
#pragma unroll
  for (int u = 0; u < 2; u++) {
    const int at = (half * 8 + 4 * u + q) * NG + g;
    s.vs[u] = ((const uint2*)(page + V_SCALES * D))[at];
    s.vo[u] = ((const uint2*)(page + V_OFFSETS * D))[at];
  }
}

// Whether fp16 holds the operands that these scales make.
template <int D> __device__ __forceinline__ bool keys_wide(const Share<D>& s) {
  bool wide = false;
#pragma unroll
  for (int g = 0; g < D / GROUP; g++) wide |= bf16_bits_to_f32(s.ks[g]) > K_SCALE_MOST;
  return wide;
}
template <int D> __device__ __forceinline__ bool values_wide(const Share<D>& s) {
  const uint32_t sw[4] = {s.vs[0].x, s.vs[0].y, s.vs[1].x, s.vs[1].y};
  bool wide = false;
#pragma unroll
  for (int k = 0; k < 4; k++) {
    const float x = bf16_lo(sw[k]), y = bf16_hi(sw[k]);
    wide |= fmaxf(x, y) > V_SCALE_MOST || (x < V_SCALE_LEAST && x > 0.0f) || (y < V_SCALE_LEAST && y > 0.0f);
  }
  return wide;
}

// Word k of a thread's keys / values to LDS.
template <int D, bool F16> __device__ __forceinline__ void put_key(const Share<D>& s, u32x4* lds, int quarter, int k, int lane) {
  constexpr int KW = D / 32;
  const int q = lane / 16, r = lane % 16, row = 16 * (r / 8) + 8 * (quarter & 1) + r % 8;
  const float scale = bf16_bits_to_f32(s.ks[k / 2]), offset = bf16_bits_to_f32(s.ko[k / 2]);
  const f16x2 s2 = {(_Float16)scale, (_Float16)scale}, o2 = {(_Float16)offset, (_Float16)offset};
  lds[((quarter / 2) * 2 * KW + 2 * k + q / 2) * 64 + (q & 1) * 32 + row] =
      F16 ? dense_f16(s.kw[k], &o2, &s2, 0) : dense_bf16(s.kw[k], &offset, &scale, 0);
}
template <int D, bool F16> __device__ __forceinline__ void put_value(const Share<D>& s, u32x4* lds, int unit, int w, int lane) {
  constexpr int NG = D / GROUP;
  const int half = unit / NG, g = unit % NG, q = lane / 16, r = lane % 16;
  const uint32_t sw[4] = {s.vs[0].x, s.vs[0].y, s.vs[1].x, s.vs[1].y}, ow[4] = {s.vo[0].x, s.vo[0].y, s.vo[1].x, s.vo[1].y};
  float scale[8], offset[8];
  f16x2 s2[4], o2[4];
#pragma unroll
  for (int k = 0; k < 4; k++) {
    scale[2 * k] = bf16_lo(sw[k]), scale[2 * k + 1] = bf16_hi(sw[k]);
    offset[2 * k] = bf16_lo(ow[k]), offset[2 * k + 1] = bf16_hi(ow[k]);
    s2[k] = f16_pair(sw[k]);
    o2[k] = f16_pair(ow[k]);
  }
  lds[((half * (D / 32) + 2 * g + w / 2) * 2 + q / 2) * 64 + (q & 1) * 32 + (w & 1) * 16 + r] =
      F16 ? dense_f16(s.vw[w], o2, s2, 1) : dense_bf16(s.vw[w], offset, scale, 1);
}

// LDS of a buffer: keys then values, 128 * D bytes each.
template <int D> constexpr int buffer_words() { return 2 * 128 * D / 16; }

// A wave's state: its 32 query rows.
template <int D> struct Rows {
  f32x16 acc[D / 32];
  float m, l;
};

// One page in LDS for a wave's rows.  limit: tokens of the page that the lane's query sees; cut: whether any lane's
// is below PAGE.  Fragments are read one step ahead of the matrix instructions that take them, and the order of the
// steps is pinned: left to itself the compiler reads all of them first and spills.  side(k) is work for the vector
// unit that runs beneath step k's matrix instructions.
#define PIN() __builtin_amdgcn_sched_barrier(0)
template <int D, bool F16, class Q, class S>
__device__ __forceinline__ void take_page(Rows<D>& w, const u32x4* lds, Q query, int limit, bool cut, float scale, int lane, S side) {
  constexpr int KSTEPS = D / 16, DTILES = D / 32;
  const int hl = lane / 32;
  const u32x4* values = lds + 8 * D;
  f32x16 z[2];
#pragma unroll
  for (int half = 0; half < 2; half++)
#pragma unroll
    for (int j = 0; j < 16; j++) z[half][j] = 0;
  u32x4 f[2][2];
#pragma unroll
  for (int half = 0; half < 2; half++) f[0][half] = lds[half * KSTEPS * 64 + lane];
#pragma unroll
  for (int s = 0; s < KSTEPS; s++) {
    if (s + 1 < KSTEPS) {
#pragma unroll
      for (int half = 0; half < 2; half++) f[(s + 1) & 1][half] = lds[(half * KSTEPS + s + 1) * 64 + lane];
    }
    const u32x4 q = query(s);
#pragma unroll
    for (int half = 0; half < 2; half++) z[half] = mfma32<F16>(f[s & 1][half], q, z[half]);
    side(s);
    PIN();
  }
  if (cut) {
#pragma unroll
    for (int half = 0; half < 2; half++)
#pragma unroll
      for (int j = 0; j < 16; j++)
        if (32 * half + 16 * ((j >> 2) & 1) + 8 * (j >> 3) + 4 * hl + (j & 3) >= limit) z[half][j] = NEG;
  }
  float top = NEG;
#pragma unroll
  for (int half = 0; half < 2; half++)
#pragma unroll
    for (int j = 0; j < 16; j++) top = fmaxf(top, z[half][j]);
  top = fmaxf(top, lane_xor32(top));
  // the maximum less P_SHIFT, so that probabilities reach 2^P_SHIFT
  top = fmaxf(fmaf(top, scale, -P_SHIFT), w.m);
  const float base = top == NEG ? 0.0f : top;
  if (__any(top > w.m)) {
    const float f = weight(w.m, base);
    w.l *= f;
#pragma unroll
    for (int d = 0; d < DTILES; d++) w.acc[d] *= f;
    w.m = top;
  }
  float sum = 0;
  u32x4 p[4];
#pragma unroll
  for (int k = 0; k < 4; k++)
#pragma unroll
    for (int e = 0; e < 4; e++) {
      const float x = __builtin_amdgcn_exp2f(fmaf(z[k / 2][8 * (k & 1) + 2 * e], scale, -base));
      const float y = __builtin_amdgcn_exp2f(fmaf(z[k / 2][8 * (k & 1) + 2 * e + 1], scale, -base));
      sum += x + y;
      if (F16) {
        const f16x2 h = {(_Float16)x, (_Float16)y};
        p[k][e] = __builtin_bit_cast(uint32_t, h);
      } else p[k][e] = pack_bf16(x, y);
    }
  w.l += sum;
  PIN();
  // steps of two dim tiles
  constexpr int STEPS = 4 * DTILES / 2;
  auto fragment = [&](int step, int u) {
    const int k = step / (DTILES / 2), d = 2 * (step % (DTILES / 2)) + u;
    return values[(((k / 2) * DTILES + d) * 2 + (k & 1)) * 64 + lane];
  };
#pragma unroll
  for (int u = 0; u < 2; u++) f[0][u] = fragment(0, u);
#pragma unroll
  for (int step = 0; step < STEPS; step++) {
    if (step + 1 < STEPS) {
#pragma unroll
      for (int u = 0; u < 2; u++) f[(step + 1) & 1][u] = fragment(step + 1, u);
    }
#pragma unroll
    for (int u = 0; u < 2; u++) {
      const int d = 2 * (step % (DTILES / 2)) + u;
      w.acc[d] = mfma32<F16>(f[step & 1][u], p[step / (DTILES / 2)], w.acc[d]);
    }
    PIN();
  }
}

template <int DT, int D, int NW>
__global__ __launch_bounds__(64 * NW) void paged_tile_kernel(const Attend a) {
  constexpr int NG = D / GROUP, KSTEPS = D / 16, UNITS = 2 * NG;
  constexpr int KEYS = 1, VALUES = (UNITS + NW - 1) / NW, SHARES = VALUES;
  __shared__ __align__(16) u32x4 lds[2 * buffer_words<D>()];
  __shared__ int wide[4];  // by page % 4: a scale is beyond what fp16 holds
  const int H = a.kv_heads, G = a.group;
  const int h = blockIdx.x % H, index = blockIdx.x / H;
  if (index >= a.header[1]) return;
  const Item it = a.tile[index];
  const int wave = threadIdx.x / 64, lane = threadIdx.x % 64, hl = lane / 32;
  const int rows = it.count * G, row0 = it.tile * 32 * NW + 32 * wave, row = row0 + lane % 32, t = row / G;
  const bool valid = row < rows;
  const int32_t* table = a.table + it.row * a.width;
  const int head = h * G + row % G;
  const uint16_t* source = (const uint16_t*)a.query + (int64_t)(it.offset + t) * a.q_token + head * a.q_head + hl * 8;
  auto raw_query = [&](int s) { return valid ? *(const u32x4*)(source + 16 * s) : u32x4{0, 0, 0, 0}; };
  auto page_of = [&](int p) { return a.pool + ((int64_t)table[p] * H + h) * page_bytes(D); };

  if (threadIdx.x < 4) wide[threadIdx.x] = 0;
  u32x4 qf[KSTEPS];
  bool large = false;
  auto too_large = [](float x) { return fabsf(x) > Q_MOST && fabsf(x) < INFINITY; };  // others spoil their own row alone
#pragma unroll
  for (int s = 0; s < KSTEPS; s++) {
    qf[s] = raw_query(s);
    if (DT == ANNA_MI_BF16) {
#pragma unroll
      for (int k = 0; k < 4; k++) {
        large |= too_large(bf16_lo(qf[s][k])) || too_large(bf16_hi(qf[s][k]));
        qf[s][k] = __builtin_bit_cast(uint32_t, f16_pair(qf[s][k]));
      }
    } else {
#pragma unroll
      for (int k = 0; k < 4; k++)
        large |= too_large(f16_bits_to_f32((uint16_t)qf[s][k])) || too_large(f16_bits_to_f32((uint16_t)(qf[s][k] >> 16)));
    }
  }
  const bool all_wide = __syncthreads_or(large) != 0;
  auto fast_query = [&](int s) { return qf[s]; };
  auto slow_query = [&](int s) {
    u32x4 v = raw_query(s);
    if (DT == ANNA_MI_F16) {
#pragma unroll
      for (int k = 0; k < 4; k++) v[k] = pack_bf16(f16_bits_to_f32((uint16_t)v[k]), f16_bits_to_f32((uint16_t)(v[k] >> 16)));
    }
    return v;
  };

  Rows<D> w;
  w.m = NEG, w.l = 0;
#pragma unroll
  for (int d = 0; d < D / 32; d++)
#pragma unroll
    for (int j = 0; j < 16; j++) w.acc[d][j] = 0;

  Share<D> share[SHARES];
  auto load = [&](const uint8_t* page) {
#pragma unroll
    for (int k = 0; k < KEYS; k++)
      if (wave + k * NW < 4) load_keys(share[k], page, wave + k * NW, lane);
#pragma unroll
    for (int k = 0; k < VALUES; k++) {
      const int unit = NW - 1 - wave + k * NW;  // from the last wave on: with 8 waves, other waves than the keys'
      if (unit < UNITS) load_values(share[k], page, unit, lane);
    }
  };
  auto check = [&](int slot) {
    bool beyond = false;
#pragma unroll
    for (int k = 0; k < KEYS; k++)
      if (wave + k * NW < 4) beyond |= keys_wide(share[k]);
#pragma unroll
    for (int k = 0; k < VALUES; k++)
      if (NW - 1 - wave + k * NW < UNITS) beyond |= values_wide(share[k]);
    if (beyond) wide[slot] = 1;
  };
  // word k of this thread's keys and of its values (with 8 waves a wave has only one of the two)
  constexpr int WORDS = NW == 8 ? (D / 32 > 4 ? D / 32 : 4) : D / 32 + 4 * VALUES;
  auto put_word = [&](u32x4* to, int k) {
    if (NW == 8) {
      if (wave < 4) {
        if (k < D / 32) put_key<D, true>(share[0], to, wave, k, lane);
      } else if (k < 4 && NW - 1 - wave < UNITS) put_value<D, true>(share[0], to + 8 * D, NW - 1 - wave, k, lane);
    } else if (k < D / 32) put_key<D, true>(share[0], to, wave, k, lane);
    else {
      const int n = (k - D / 32) / 4, unit = NW - 1 - wave + n * NW;
      if (unit < UNITS) put_value<D, true>(share[n], to + 8 * D, unit, (k - D / 32) % 4, lane);
    }
  };
  // LDS only: loads of the next page stay in flight
  auto barrier = [] { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); };

  const int first = it.start + row0 / G + 1;                            // tokens that the wave's first row sees
  const int last = row0 < rows ? it.start + min(row0 + 31, rows - 1) / G + 1 : 0;  // and its last
  const int sees = valid ? it.start + t + 1 : 0;

  load(page_of(it.page0));
  check(it.page0 & 3);
#pragma unroll
  for (int k = 0; k < WORDS; k++) put_word(lds, k);
  if (it.page0 + 1 < it.page1) load(page_of(it.page0 + 1));
  barrier();
  for (int p = it.page0; p < it.page1; p++) {
    const int turn = (p - it.page0) & 1;
    u32x4 *now = lds + turn * buffer_words<D>(), *then = lds + (turn ^ 1) * buffer_words<D>();
    const bool more = p + 1 < it.page1, slow = all_wide || wide[p & 3] != 0;
    if (threadIdx.x == 0) wide[(p + 2) & 3] = 0;
    if (more) check((p + 1) & 3);
    const int limit = sees - p * PAGE;
    constexpr int PER = (WORDS + KSTEPS - 1) / KSTEPS;
    auto side = [&](int s) {
      if (more) {
#pragma unroll
        for (int k = s * PER; k < (s + 1) * PER; k++)
          if (k < WORDS) put_word(then, k);
      }
    };
    const bool mine = p * PAGE < last;
    if (mine && !slow) {
      take_page<D, true>(w, now, fast_query, limit, p * PAGE + PAGE > first, a.scale, lane, side);
    } else {
#pragma unroll
      for (int s = 0; s < KSTEPS; s++) side(s);
    }
    if (p + 2 < it.page1) load(page_of(p + 2));
    if (slow) {
      // the page again, as bf16
      barrier();
      const uint8_t* page = page_of(p);
      Share<D> again;
      for (int k = wave; k < 4; k += NW) {
        load_keys(again, page, k, lane);
#pragma unroll
        for (int i = 0; i < D / 32; i++) put_key<D, false>(again, now, k, i, lane);
      }
      for (int k = wave; k < UNITS; k += NW) {
        load_values(again, page, k, lane);
#pragma unroll
        for (int i = 0; i < 4; i++) put_value<D, false>(again, now + 8 * D, k, i, lane);
      }
      barrier();
      if (mine) take_page<D, false>(w, now, slow_query, limit, p * PAGE + PAGE > first, a.scale, lane, [](int) {});
    }
    barrier();
  }

  // a lane holds, of its query, dims 32 d + 8 b + 4 hl + i
  const float total = w.l + lane_xor32(w.l);
  if (!valid) return;
  const int64_t part = (int64_t)(it.part + 32 * wave + lane % 32) * H + h;
  const float inv = 1.0f / total;
#pragma unroll
  for (int d = 0; d < D / 32; d++)
#pragma unroll
    for (int b = 0; b < 4; b++) {
      const int dim = 32 * d + 8 * b + 4 * hl;
      const f32x4 v = {w.acc[d][4 * b], w.acc[d][4 * b + 1], w.acc[d][4 * b + 2], w.acc[d][4 * b + 3]};
      if (it.part < 0) write_out<DT>(a, D, it.offset + t, head, dim, v * inv, (int64_t)H * G);
      else *(f32x4*)(a.values + part * D + dim) = v;
    }
  if (it.part >= 0 && hl == 0) a.stats[2 * part] = w.m, a.stats[2 * part + 1] = total;
}

// Joins the items of a tile: one workgroup a query row, its four waves each every fourth item.
template <int DT, int D>
__global__ __launch_bounds__(256) void paged_merge_kernel(const Attend a) {
  constexpr int LANES = D / 4, TEAMS = 256 / LANES;
  __shared__ __align__(16) float joined[TEAMS][D];
  __shared__ float team_m[TEAMS], team_l[TEAMS];
  const int H = a.kv_heads, G = a.group, h = blockIdx.x % H, index = blockIdx.x / H;
  if (index >= a.header[2]) return;
  const Unit u = a.units[index];
  const int row = blockIdx.y;
  if (row >= u.rows) return;
  const int team = threadIdx.x / LANES, d = threadIdx.x % LANES * 4;
  float top = NEG, total = 0;
  f32x4 v = {0, 0, 0, 0};
  for (int k = team; k < u.splits; k += TEAMS) {
    const int64_t part = (int64_t)(u.part + k * u.rows + row) * H + h;
    const float m = a.stats[2 * part], l = a.stats[2 * part + 1];
    const f32x4 x = *(const f32x4*)(a.values + part * D + d);
    const float next = fmaxf(top, m), f0 = weight(top, next), f1 = weight(m, next);
    total = total * f0 + l * f1;
    v = v * f0 + x * f1;
    top = next;
  }
  *(f32x4*)&joined[team][d] = v;
  if (d == 0) team_m[team] = top, team_l[team] = total;
  __syncthreads();
  if (team != 0) return;
  for (int k = 1; k < TEAMS; k++) {
    const float m = team_m[k], next = fmaxf(top, m), f0 = weight(top, next), f1 = weight(m, next);
    total = total * f0 + team_l[k] * f1;
    v = v * f0 + *(const f32x4*)&joined[k][d] * f1;
    top = next;
  }
  const int r = u.row0 + row;
  write_out<DT>(a, D, u.offset + r / G, h * G + r % G, d, v * (1.0f / total), (int64_t)H * G);
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
  if (g.units > 0) paged_merge_kernel<DT, D><<<dim3((unsigned)(g.units * a.kv_heads), (unsigned)g.unit_rows), 256, 0, stream>>>(a);
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
