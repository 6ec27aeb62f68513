// Root-mean-square norms of rows: with the residual stream's addition, with a gate, with an e4m3 output.
//
// LANES threads hold a row in registers, VECS vectors of 8 columns each, so that every input is read once;
// rows longer than the registers of a workgroup are read twice.  Sums of squares and the scales are fp32.  The
// sum with the residual is rounded to the type before it is normalised: what is normalised is what the stream
// holds, as in a model that adds and normalises in two steps.  The output is rounded once, from fp32.
//
//   h = x + residual,   y = h / sqrt(mean(h^2) + eps) * (weight + offset) * silu(gate)
//   e4m3: scale = m / 448, code = e4m3(y / scale), m the largest |y| of a group
//
// Bound by the rows' bytes.  8192 rows of 4096 with residual and e4m3 codes (0.24 GB): 49 us = 4.8 TB/s; a copy of
// 1 GiB runs at 5.2 (55 us with a clamp of every code, which branches, and divisions by the group).  262144 rows of 128 with gate (0.2 GB): 41 us = 4.9 TB/s.  64 rows of 2048: 3.1 us, less
// than an empty launch from the host takes.
#include "delta.hpp"

namespace anna {

constexpr float E4M3_MAX = 448.f;
constexpr uint32_t TINY_BITS = (127 - 100) << 23;  // 2^-100: groups below it are held as zeros

template <int DT>
struct Row8 {
  typename Elem<DT>::T v[8];
};

// VEC: eight columns at a time, 16-byte aligned; else `n` of them one by one
template <int DT, bool VEC>
__device__ __forceinline__ Row8<DT> load8(const void* base, int64_t at, int n) {
  const typename Elem<DT>::T* p = (const typename Elem<DT>::T*)base + at;
  if constexpr (VEC) return *(const Row8<DT>*)__builtin_assume_aligned(p, 16);
  Row8<DT> r;
#pragma unroll
  for (int e = 0; e < 8; e++) r.v[e] = e < n ? p[e] : (typename Elem<DT>::T)0;
  return r;
}
// Columns from c on, up to eight; of aligned rows eight or none
template <bool VEC>
__device__ __forceinline__ int columns(int64_t cols, int64_t c) {
  if constexpr (VEC) return c < cols ? 8 : 0;
  return (int)min((int64_t)8, max((int64_t)0, cols - c));
}
template <int DT>
__device__ __forceinline__ void widen(const Row8<DT>& r, float (&f)[8]) {
#pragma unroll
  for (int e = 0; e < 8; e++) f[e] = Elem<DT>::to_f32(r.v[e]);
}
template <int DT, bool VEC>
__device__ __forceinline__ void save8(void* base, int64_t at, int n, const float (&f)[8]) {
  typename Elem<DT>::T* p = (typename Elem<DT>::T*)base + at;
  Row8<DT> r;
#pragma unroll
  for (int e = 0; e < 8; e++) r.v[e] = Elem<DT>::cvt(f[e]);
  if constexpr (VEC) {
    *(Row8<DT>*)__builtin_assume_aligned(p, 16) = r;
  } else {
#pragma unroll
    for (int e = 0; e < 8; e++)
      if (e < n) p[e] = r.v[e];
  }
}

// Sum, and largest bit pattern (of values without sign, so that a NaN is larger than all), over the lanes of a
// row; `part`: a workgroup's exchange for rows of more than a wave
template <int LANES> __device__ __forceinline__ float row_sum(float v, float* part) {
#pragma unroll
  for (int off = 1; off < (LANES < 64 ? LANES : 64); off *= 2) v += __shfl_xor(v, off, 64);
  if constexpr (LANES > 64) {
    if ((threadIdx.x & 63) == 0) part[threadIdx.x / 64] = v;
    __syncthreads();
    v = 0.f;
#pragma unroll
    for (int w = 0; w < LANES / 64; w++) v += part[w];
  }
  return v;
}
template <int LANES> __device__ __forceinline__ uint32_t row_max(uint32_t v, uint32_t* part) {
#pragma unroll
  for (int off = 1; off < (LANES < 64 ? LANES : 64); off *= 2) v = max(v, (uint32_t)__shfl_xor((int)v, off, 64));
  if constexpr (LANES > 64) {
    if ((threadIdx.x & 63) == 0) part[threadIdx.x / 64] = v;
    __syncthreads();
    v = 0;
#pragma unroll
    for (int w = 0; w < LANES / 64; w++) v = max(v, part[w]);
  }
  return v;
}

template <bool VEC>
__device__ __forceinline__ uint32_t abs_max(const float (&y)[8], int n) {
  uint32_t m = 0;
#pragma unroll
  for (int e = 0; e < 8; e++)
    if (VEC || e < n) m = max(m, __float_as_uint(y[e]) & 0x7fffffffu);
  return m;
}
// What divides a group's values: its scale, the same or 0 where it is not finite, and 1 / scale.  With the reciprocal
// rounded once, one step of Markstein's gives the quotient's own rounding: q = y r, q + (y - q scale) r.  A product with 448 / m
// has two, and moves codes whose quotients are halfway between two.
struct Scale {
  float scale, finite, inverse;
};
__device__ __forceinline__ Scale scale_of(uint32_t largest) {
  if (largest < TINY_BITS) return {0.f, 0.f, 0.f};
  const float s = __uint_as_float(largest) / E4M3_MAX;
  return {s, s < INFINITY ? s : 0.f, 1.f / s};
}
__device__ __forceinline__ float quotient(float y, const Scale& s) {
  const float q = y * s.inverse;
  return fmaf(fmaf(-q, s.finite, y), s.inverse, q);
}

// Codes of eight values; a quotient is at most 448 (1 + 2^-23), far from 464, where e4m3 would end
template <bool VEC>
__device__ __forceinline__ void save_codes(uint8_t* p, int n, const float (&y)[8], const Scale& s) {
  uint32_t w[2];
#pragma unroll
  for (int h = 0; h < 2; h++) {
    float c[4];
#pragma unroll
    for (int e = 0; e < 4; e++) c[e] = quotient(y[4 * h + e], s);
    int packed = __builtin_amdgcn_cvt_pk_fp8_f32(c[0], c[1], 0, false);
    w[h] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c[2], c[3], packed, true);
  }
  if constexpr (VEC) {
    *(uint2*)p = make_uint2(w[0], w[1]);
  } else {
#pragma unroll
    for (int e = 0; e < 8; e++)
      if (e < n) p[e] = (uint8_t)(w[e / 4] >> (8 * (e % 4)));
  }
}

// Group of `group` columns in lanes: of a row's LANES threads, group / 8 neighbours
__device__ __forceinline__ uint32_t group_max(uint32_t m, int lanes) {
  for (int off = 1; off < lanes; off *= 2) m = max(m, (uint32_t)__shfl_xor((int)m, off, 64));
  return m;
}

template <int DT, int LANES, int VECS, bool CODES, bool VEC>
__global__ __launch_bounds__(256) void rms_norm_kernel(const anna_mi_rms_norm_args a) {
  constexpr int ROWS = 256 / LANES;
  __shared__ float sums[4];
  __shared__ uint32_t tops[4];
  const int lane = threadIdx.x % LANES;
  int64_t row = (int64_t)blockIdx.x * ROWS + threadIdx.x / LANES;
  const bool live = row < a.rows;
  if (!live) row = a.rows - 1;  // its lanes take part in the exchanges, and store nothing
  const int64_t cols = a.cols;

  // everything is asked for in front of the sum
  Row8<DT> x[VECS], old[VECS], gate[VECS], weight[VECS];
#pragma unroll
  for (int i = 0; i < VECS; i++) {
    const int64_t c = 8 * (int64_t)(lane + LANES * i);
    const int n = columns<VEC>(cols, c);
    if (n == 0) continue;
    x[i] = load8<DT, VEC>(a.x, row * a.x_stride + c, n);
    if (a.residual) old[i] = load8<DT, VEC>(a.residual, row * a.residual_stride + c, n);
    if (a.gate) gate[i] = load8<DT, VEC>(a.gate, row * a.gate_stride + c, n);
    weight[i] = load8<DT, VEC>(a.weight, c, n);
  }
  float h[VECS][8], ss = 0.f;
#pragma unroll
  for (int i = 0; i < VECS; i++) {
    const int64_t c = 8 * (int64_t)(lane + LANES * i);
    const int n = columns<VEC>(cols, c);
    if (n == 0) {
#pragma unroll
      for (int e = 0; e < 8; e++) h[i][e] = 0.f;
      continue;
    }
    widen<DT>(x[i], h[i]);
    if (a.residual) {
      float r[8];
      widen<DT>(old[i], r);
#pragma unroll
      for (int e = 0; e < 8; e++) h[i][e] = Elem<DT>::to_f32(Elem<DT>::cvt(h[i][e] + r[e]));
      if (live) save8<DT, VEC>(a.residual, row * a.residual_stride + c, n, h[i]);
    }
#pragma unroll
    for (int e = 0; e < 8; e++) ss = fmaf(h[i][e], h[i][e], ss);
  }
  const float rs = rsqrtf(row_sum<LANES>(ss, sums) / (float)cols + a.eps);

  uint32_t top = 0;
  const int shift = __builtin_ctz((uint32_t)a.group);  // of groups that are not whole rows
#pragma unroll
  for (int i = 0; i < VECS; i++) {
    const int64_t c = 8 * (int64_t)(lane + LANES * i);
    const int n = columns<VEC>(cols, c);
    if (n > 0) {
      float w[8];
      widen<DT>(weight[i], w);
#pragma unroll
      for (int e = 0; e < 8; e++) h[i][e] = h[i][e] * rs * (w[e] + a.weight_offset);
      if (a.gate) {
        float g[8];
        widen<DT>(gate[i], g);
#pragma unroll
        for (int e = 0; e < 8; e++) h[i][e] *= silu_of(g[e]);
      }
    }
    if constexpr (!CODES) {
      if (live && n > 0) save8<DT, VEC>(a.out, row * a.out_stride + c, n, h[i]);
    } else {
      const uint32_t m = abs_max<VEC>(h[i], n);
      if (a.group == cols) {
        top = max(top, m);
      } else {  // every group lies in neighbouring lanes of one vector row
        const Scale s = scale_of(group_max(m, (int)a.group / 8));
        if (live && n > 0) {
          save_codes<VEC>((uint8_t*)a.out + row * a.out_stride + c, n, h[i], s);
          if ((c & (a.group - 1)) == 0) a.scales[row * (cols >> shift) + (c >> shift)] = s.scale;
        }
      }
    }
  }
  if constexpr (CODES) {
    if (a.group == cols) {
      const Scale s = scale_of(row_max<LANES>(top, tops));
      if (live && lane == 0) a.scales[row] = s.scale;
#pragma unroll
      for (int i = 0; i < VECS; i++) {
        const int64_t c = 8 * (int64_t)(lane + LANES * i);
        const int n = columns<VEC>(cols, c);
        if (live && n > 0) save_codes<VEC>((uint8_t*)a.out + row * a.out_stride + c, n, h[i], s);
      }
    }
  }
}

// Rows of any length: a workgroup a row, read again for every pass (the second from L2)
template <int DT, bool CODES, bool VEC>
__global__ __launch_bounds__(256) void rms_norm_long_kernel(const anna_mi_rms_norm_args a) {
  __shared__ float sums[4];
  __shared__ uint32_t tops[4];
  const int64_t row = blockIdx.x, cols = a.cols;
  const void* src = a.residual ? a.residual : a.x;
  const int64_t src_stride = a.residual ? a.residual_stride : a.x_stride;
  float ss = 0.f;
  for (int64_t c = 8 * (int64_t)threadIdx.x; c < cols; c += 2048) {
    const int n = columns<VEC>(cols, c);
    float h[8];
    widen<DT>(load8<DT, VEC>(a.x, row * a.x_stride + c, n), h);
    if (a.residual) {
      float old[8];
      widen<DT>(load8<DT, VEC>(a.residual, row * a.residual_stride + c, n), old);
#pragma unroll
      for (int e = 0; e < 8; e++) h[e] = Elem<DT>::to_f32(Elem<DT>::cvt(h[e] + old[e]));
      save8<DT, VEC>(a.residual, row * a.residual_stride + c, n, h);  // read again below by the same thread
    }
#pragma unroll
    for (int e = 0; e < 8; e++) ss = fmaf(h[e], h[e], ss);
  }
  const float rs = rsqrtf(row_sum<256>(ss, sums) / (float)cols + a.eps);
  auto value = [&](int64_t c, int n, float (&h)[8]) {
    float w[8];
    widen<DT>(load8<DT, VEC>(src, row * src_stride + c, n), h);
    widen<DT>(load8<DT, VEC>(a.weight, c, n), w);
#pragma unroll
    for (int e = 0; e < 8; e++) h[e] = h[e] * rs * (w[e] + a.weight_offset);
    if (a.gate) {
      float g[8];
      widen<DT>(load8<DT, VEC>(a.gate, row * a.gate_stride + c, n), g);
#pragma unroll
      for (int e = 0; e < 8; e++) h[e] *= silu_of(g[e]);
    }
  };
  const bool by_row = a.group == cols;
  const int shift = __builtin_ctz((uint32_t)a.group);  // of groups that are not whole rows
  Scale s{0.f, 0.f, 0.f};
  if constexpr (CODES) {
    if (by_row) {
      uint32_t top = 0;
      for (int64_t c = 8 * (int64_t)threadIdx.x; c < cols; c += 2048) {
        const int n = columns<VEC>(cols, c);
        float h[8];
        value(c, n, h);
        top = max(top, abs_max<VEC>(h, n));
      }
      s = scale_of(row_max<256>(top, tops));
      if (threadIdx.x == 0) a.scales[row] = s.scale;
    }
  }
  for (int64_t base = 0; base < cols; base += 2048) {  // whole workgroups: a group's lanes meet below
    const int64_t c = base + 8 * (int64_t)threadIdx.x;
    const int n = columns<VEC>(cols, c);
    float h[8] = {};
    if (n > 0) value(c, n, h);
    if constexpr (!CODES) {
      if (n > 0) save8<DT, VEC>(a.out, row * a.out_stride + c, n, h);
    } else {
      if (!by_row) s = scale_of(group_max(abs_max<VEC>(h, n), (int)a.group / 8));
      if (n > 0) {
        save_codes<VEC>((uint8_t*)a.out + row * a.out_stride + c, n, h, s);
        if (!by_row && (c & (a.group - 1)) == 0) a.scales[row * (cols >> shift) + (c >> shift)] = s.scale;
      }
    }
  }
}

template <int DT, bool CODES> static int launch_norm(const anna_mi_rms_norm_args& a, hipStream_t stream) {
  constexpr int64_t unit = 16 / sizeof(typename Elem<DT>::T);
  auto rows16 = [&](const void* p, int64_t stride) { return (uintptr_t)p % 16 == 0 && (a.rows == 1 || stride % unit == 0); };
  const bool vec = a.cols % 8 == 0 && rows16(a.x, a.x_stride) && rows16(a.weight, unit) &&
                   (!a.residual || rows16(a.residual, a.residual_stride)) && (!a.gate || rows16(a.gate, a.gate_stride)) &&
                   (CODES ? (uintptr_t)a.out % 8 == 0 && (a.rows == 1 || a.out_stride % 8 == 0) : rows16(a.out, a.out_stride));
  const int64_t vecs = (a.cols + 7) / 8;
  auto blocks = [&](int rows) { return (a.rows + rows - 1) / rows; };
  const int64_t grid = blocks(vecs <= 8 ? 32 : vecs <= 16 ? 16 : vecs <= 32 ? 8 : vecs <= 64 ? 4 : 1);
  ANNA_CHECK(grid <= INT32_MAX / 256, "rms_norm: %lld rows of %lld columns are too many for a launch", (long long)a.rows, (long long)a.cols);
  // A vector a thread as far as a workgroup reaches, so that a row's loads all go out at once: 8192 rows of 4096 take
  // 55 us with 256 threads a row and 147 with a wave that holds 8 vectors a thread (both before other steps).
#define ANNA_NORM(LANES, VECS)                                                                                          \
  (vec ? rms_norm_kernel<DT, LANES, VECS, CODES, true> : rms_norm_kernel<DT, LANES, VECS, CODES, false>)<<<blocks(256 / LANES), \
                                                                                                           256, 0, stream>>>(a)
  if (vecs <= 8) ANNA_NORM(8, 1);
  else if (vecs <= 16) ANNA_NORM(16, 1);
  else if (vecs <= 32) ANNA_NORM(32, 1);
  else if (vecs <= 64) ANNA_NORM(64, 1);
  else if (vecs <= 256) ANNA_NORM(256, 1);
  else if (vecs <= 512) ANNA_NORM(256, 2);
  else if (vecs <= 1024) ANNA_NORM(256, 4);
  else (vec ? rms_norm_long_kernel<DT, CODES, true> : rms_norm_long_kernel<DT, CODES, false>)<<<a.rows, 256, 0, stream>>>(a);
#undef ANNA_NORM
  ANNA_LAUNCH_CHECK("rms_norm");
  return ANNA_MI_OK;
}

}  // namespace anna

extern "C" int anna_mi_rms_norm(const anna_mi_rms_norm_args* args, void* stream) {
  ANNA_CHECK(args != nullptr, "rms_norm: null args");
  const anna_mi_rms_norm_args& a = *args;
  ANNA_CHECK(anna::valid_dtype(a.dtype), "rms_norm: dtype %d", a.dtype);
  ANNA_CHECK(a.out_format == 0 || a.out_format == 1, "rms_norm: out_format %d", a.out_format);
  ANNA_CHECK(a.rows >= 0 && a.cols >= 1 && a.cols <= (1 << 28), "rms_norm: %lld rows of %lld", (long long)a.rows, (long long)a.cols);
  if (a.rows == 0) return ANNA_MI_OK;
  ANNA_CHECK(a.x && a.weight && a.out && (a.out_format == 0 || a.scales), "rms_norm: null pointer");
  ANNA_CHECK(a.rows == 1 || (a.x_stride >= a.cols && a.out_stride >= a.cols && (!a.residual || a.residual_stride >= a.cols) &&
                             (!a.gate || a.gate_stride >= a.cols)), "rms_norm: rows overlap");
  const int64_t size = a.dtype == ANNA_MI_F32 ? 4 : 2, out_size = a.out_format == 1 ? 1 : size;
  ANNA_CHECK(anna::rows_apart({a.residual, a.rows, a.residual_stride * size, a.cols * size}, {a.out, a.rows, a.out_stride * out_size, a.cols * out_size}),
             "rms_norm: out overlaps the residual");
  if (a.out_format == 1) {
    ANNA_CHECK(a.group == a.cols || ((a.group == 32 || a.group == 64 || a.group == 128) && a.cols % a.group == 0),
               "rms_norm: groups of %lld columns, 32, 64, 128 (a divisor of cols) or whole rows are supported", (long long)a.group);
    ANNA_DISPATCH_DTYPE(a.dtype, DT, return (anna::launch_norm<DT, true>(a, anna::as_stream(stream))));
  }
  ANNA_DISPATCH_DTYPE(a.dtype, DT, return (anna::launch_norm<DT, false>(a, anna::as_stream(stream))));
}
