// Attention over the paged 4-bit KV cache (page layout in anna_mi.h).
//
// out = softmax(scaling q K^T) V over the tokens up to and with the query's own, K and V held as
// (code + zero) * scale with one scale and zero for 64 values of a token and head.
//
// Split form.  A workgroup takes the query rows of one KV head (R = 16, 32 or 64 rows: tokens times
// query heads of that KV head) and some of the sequence's pages; each of its four waves takes every
// fourth page with an online softmax of its own, and the waves' results are joined at the end.
// Codes go to the matrix cores as whole numbers: 128 + code has the bits 0x4300 | code in bf16 (in
// fp16 0x5800 | code << 3), so 8 codes cost 7 or 8 instructions and no conversion.  With
// o = zero - 128 (the cache's offsets, exact in bf16)
//   q.k   = sum over groups of  scale * (sum_d q_d (128 + code_d) + o * sum_d q_d)
//   p V_d = sum_t ps_t (128 + code_td) + sum_t ps_t o_t,     ps_t = p_t * scale_t rounded to bf16
// where the products with o are matrix instructions too: the first starts the sums (sum_d q_d as three
// bf16 terms, good to 24 bits), the second takes the same rounded ps, so the 128s cancel exactly.
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

// 128 + code of the 8 codes of a word, as operand elements of the type.
template <int DT> __device__ __forceinline__ u32x4 codes128(uint32_t w) {
  u32x4 o;
  if constexpr (DT == ANNA_MI_BF16) {
    o[0] = (w & 0x000F000Fu) | 0x43004300u;
    o[1] = ((w >> 4) & 0x000F000Fu) | 0x43004300u;
    o[2] = ((w >> 8) & 0x000F000Fu) | 0x43004300u;
    o[3] = ((w >> 12) & 0x000F000Fu) | 0x43004300u;
  } else {
    o[0] = ((w << 3) & 0x00780078u) | 0x58005800u;
    o[1] = ((w >> 1) & 0x00780078u) | 0x58005800u;
    o[2] = ((w >> 5) & 0x00780078u) | 0x58005800u;
    o[3] = ((w >> 9) & 0x00780078u) | 0x58005800u;
  }
  return o;
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
        const u32x4 a0 = codes128<DT>(w[2 * g]), a1 = codes128<DT>(w[2 * g + 1]);
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
          const u32x4 av = codes128<ANNA_MI_BF16>(w[k]);
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

template <int DT, int D>
int launch(const Attend& a, int64_t split_items, int64_t few_rows, int64_t units, int64_t unit_rows, hipStream_t stream) {
  const unsigned grid = (unsigned)(split_items * a.kv_heads);
  if (grid > 0) {
    if (few_rows == 16) paged_split_kernel<DT, D, 1><<<grid, 256, 0, stream>>>(a);
    else if constexpr (D <= 128) {  // 4096 / D rows at most
      if (few_rows == 32) paged_split_kernel<DT, D, 2><<<grid, 256, 0, stream>>>(a);
      else if constexpr (D == 64) paged_split_kernel<DT, D, 4><<<grid, 256, 0, stream>>>(a);
    }
  }
  if (units > 0) paged_merge_kernel<DT, D><<<dim3((unsigned)(units * a.kv_heads), (unsigned)unit_rows), 256, 0, stream>>>(a);
  ANNA_LAUNCH_CHECK("paged attend");
  return ANNA_MI_OK;
}

}  // namespace

int tile_rows(int64_t head_dim) { return 64; }

int launch_attend(int dtype, int64_t head_dim, const Attend& a, int64_t split_items, int64_t few_rows, int64_t tile_items,
                  int64_t units, int64_t unit_rows, hipStream_t stream) {
  if (dtype == ANNA_MI_BF16) {
    if (head_dim == 64) return launch<ANNA_MI_BF16, 64>(a, split_items, few_rows, units, unit_rows, stream);
    if (head_dim == 128) return launch<ANNA_MI_BF16, 128>(a, split_items, few_rows, units, unit_rows, stream);
    return launch<ANNA_MI_BF16, 256>(a, split_items, few_rows, units, unit_rows, stream);
  }
  if (head_dim == 64) return launch<ANNA_MI_F16, 64>(a, split_items, few_rows, units, unit_rows, stream);
  if (head_dim == 128) return launch<ANNA_MI_F16, 128>(a, split_items, few_rows, units, unit_rows, stream);
  return launch<ANNA_MI_F16, 256>(a, split_items, few_rows, units, unit_rows, stream);
}

}  // namespace paged
}  // namespace anna
