// Paged 4-bit KV cache: tokens into pages and back, page copies, and the tables' and spans' updates
// (page layout in anna_mi.h).
#include "paged.hpp"

namespace anna {
namespace paged {
namespace {

// ---------------------------------------------------------------- updates
// One workgroup writes what a record says, one 256 table entries, one a whole table row.
__global__ __launch_bounds__(256) void paged_update_kernel(const Update u) {
  const int tid = threadIdx.x;
  int blk = blockIdx.x;
  const int32_t* words = u.words;
  if (blk < u.records) {
    const Record r = reinterpret_cast<const Record*>(words)[blk];
    if (blk == 0 && tid < 4) u.buf[tid] = u.header[tid];
    const int R = r.tiled ? u.tile_rows : u.split_rows, rows = min(R, r.count * u.group - r.tile * R);
    if (r.tile == 0) {
      if (tid == 0) u.buf[u.rows_at + r.index] = r.row;
      const int first = r.start / PAGE, pages = r.count > 0 ? (r.start + r.count - 1) / PAGE - first + 1 : 0;
      Touch* touch = reinterpret_cast<Touch*>(u.buf + u.touch_at) + r.touch0;
      for (int k = tid; k < pages; k += 256) {
        const int p = first + k, t0 = max(r.start, p * PAGE), t1 = min(r.start + r.count, (p + 1) * PAGE);
        touch[k] = Touch{r.row, p, t0 - p * PAGE, t1 - p * PAGE, r.offset + t0 - r.start, {0, 0, 0}};
      }
    }
    Item* items = reinterpret_cast<Item*>(u.buf + (r.tiled ? u.tile_at : u.split_at)) + r.item0;
    for (int k = tid; k < r.splits; k += 256) {
      const int p0 = (int)((int64_t)r.pages * k / r.splits), p1 = (int)((int64_t)r.pages * (k + 1) / r.splits);
      items[k] = Item{r.row, r.start, r.count, r.offset, p0, p1, r.part < 0 ? -1 : r.part + k * rows, r.tile};
    }
    if (r.unit >= 0 && tid == 0)
      reinterpret_cast<Unit*>(u.buf + u.units_at)[r.unit] =
          Unit{r.offset, r.tile * R, rows, r.part, r.splits, {0, 0, 0}};
    return;
  }
  blk -= u.records;
  words += u.records * (int)(sizeof(Record) / 4);
  const int entry_blocks = (u.entries + 255) / 256;
  if (blk < entry_blocks) {
    const int k = blk * 256 + tid;
    if (k < u.entries) u.table[words[2 * k]] = words[2 * k + 1];
    return;
  }
  blk -= entry_blocks;
  words += 2 * u.entries + 3 * blk;
  int32_t* row = u.table + words[0] * u.width;
  const int32_t* source = u.table + words[1] * u.width;
  for (int k = tid; k < u.width; k += 256) {
    if (k >= words[2]) row[k] = 0;
    else if (words[1] >= 0) row[k] = source[k];
  }
}

// ---------------------------------------------------------------- page copies
// One workgroup copies 16 KB of a page of a layer (all KV heads), 64 bytes a thread.
constexpr int COPY_BYTES = 16384;

__global__ __launch_bounds__(256) void paged_copy_kernel(const Copy c) {
  const int source = c.words[2 * blockIdx.y], target = c.words[2 * blockIdx.y + 1];
  const int64_t at = (int64_t)blockIdx.x * COPY_BYTES + threadIdx.x * 16;
  const uint8_t* from = c.from + blockIdx.z * c.from_layer + source * c.page + at;
  uint8_t* to = c.to + blockIdx.z * c.to_layer + target * c.page + at;
  u32x4 v[4];
#pragma unroll
  for (int k = 0; k < 4; k++) {
    v[k] = u32x4{0, 0, 0, 0};
    if (source >= 0 && at + k * 4096 < c.page) v[k] = __builtin_nontemporal_load((const u32x4*)(from + k * 4096));
  }
#pragma unroll
  for (int k = 0; k < 4; k++)
    if (at + k * 4096 < c.page) *(u32x4*)(to + k * 4096) = v[k];
}

// ---------------------------------------------------------------- store and read
__device__ __forceinline__ int code_shift(int e) { return 4 * ((e & 1) * 4 + (e >> 1)); }

template <int DT> __device__ __forceinline__ bool not_finite(u32x4 x) {
  constexpr uint32_t E = DT == ANNA_MI_BF16 ? 0x7F80u : 0x7C00u;
  bool bad = false;
#pragma unroll
  for (int k = 0; k < 4; k++) bad |= (x[k] & E) == E || (x[k] & (E << 16)) == (E << 16);
  return bad;
}

// Minimum / maximum over the 8 lanes that hold a group (64 values, 8 a lane).
__device__ __forceinline__ float group_min(float v) {
  v = fminf(v, dpp_move<0xB1>(v));
  v = fminf(v, dpp_move<0x4E>(v));
  return fminf(v, dpp_move<0x141>(v));
}
__device__ __forceinline__ float group_max(float v) {
  v = fmaxf(v, dpp_move<0xB1>(v));
  v = fmaxf(v, dpp_move<0x4E>(v));
  return fmaxf(v, dpp_move<0x141>(v));
}

// Codes of this lane's 8 values (one a byte), and the group's scale (bf16 bits) and zero.
struct Coded {
  uint32_t lo, hi;
  uint16_t scale;
  int zero;
};
template <int DT> __device__ __forceinline__ Coded quantize(u32x4 raw) {
  float x[8];
#pragma unroll
  for (int k = 0; k < 4; k++) {
    x[2 * k] = Elem<DT>::to_f32((uint16_t)raw[k]);
    x[2 * k + 1] = Elem<DT>::to_f32((uint16_t)(raw[k] >> 16));
  }
  float low = x[0], high = x[0];
#pragma unroll
  for (int k = 1; k < 8; k++) low = fminf(low, x[k]), high = fmaxf(high, x[k]);
  low = group_min(low);
  high = group_max(high);
  // halves, so that a spread of twice the largest value stays finite; the quotients are correctly
  // rounded, so one that lies between two bf16 values stays there and goes to the even one
  const float spread = fmaxf((0.5f * high - 0.5f * low) / 7.5f, fmaxf(fabsf(low), fabsf(high)) / 120.0f);
  Coded c = {0, 0, 0, 0};
  if (!(spread >= 7.888609052210118e-31f)) return c;  // 2^-100
  c.scale = f32_to_bf16_bits(spread);
  const float scale = bf16_bits_to_f32(c.scale);
  const float zero = rintf(low / scale);
  c.zero = (int)zero;
#pragma unroll
  for (int k = 0; k < 8; k++) {
    const float q = fminf(fmaxf(rintf(x[k] / scale) - zero, 0.0f), 15.0f);
    const uint32_t code = (uint32_t)q;
    if (k < 4) c.lo |= code << (8 * k);
    else c.hi |= code << (8 * (k - 4));
  }
  return c;
}

template <int DT, int D>
__global__ __launch_bounds__(256) void paged_store_kernel(uint8_t* __restrict__ pool, const int32_t* __restrict__ table, int64_t width,
                                                          const int32_t* __restrict__ header, const Touch* __restrict__ touch,
                                                          int heads, const uint16_t* __restrict__ keys, int64_t k_token, int64_t k_head,
                                                          const uint16_t* __restrict__ values, int64_t v_token, int64_t v_head) {
  constexpr int NG = D / GROUP, CHUNKS = D / 8, STEPS = PAGE * CHUNKS / 256, PITCH = D + 16;
  __shared__ __align__(16) uint8_t codes[PAGE * PITCH];  // of the values
  __shared__ int bad[PAGE];
  const int tid = threadIdx.x, item = blockIdx.x / heads, h = blockIdx.x % heads;
  if (item >= header[3]) return;
  const Touch t = touch[item];
  uint8_t* page = pool + ((int64_t)table[t.row * width + t.page] * heads + h) * page_bytes(D);
  const int slots = (t.end - t.begin) * CHUNKS;
  if (tid < PAGE) bad[tid] = 0;
  u32x4 kr[STEPS], vr[STEPS];
#pragma unroll
  for (int s = 0; s < STEPS; s++) {
    const int slot = s * 256 + tid, n = slot / CHUNKS, c = slot % CHUNKS;
    if (slot < slots) {
      kr[s] = *(const u32x4*)(keys + (t.token + n) * k_token + h * k_head + c * 8);
      vr[s] = *(const u32x4*)(values + (t.token + n) * v_token + h * v_head + c * 8);
    }
  }
  __syncthreads();
#pragma unroll
  for (int s = 0; s < STEPS; s++) {
    const int slot = s * 256 + tid;
    if (slot < slots && (not_finite<DT>(kr[s]) || not_finite<DT>(vr[s]))) bad[slot / CHUNKS] = 1;
  }
  __syncthreads();
#pragma unroll
  for (int s = 0; s < STEPS; s++) {
    const int slot = s * 256 + tid;
    if (slot >= slots) break;  // whole groups of 8 lanes
    const int n = slot / CHUNKS, c = slot % CHUNKS, token = t.begin + n, g = c / 8;
    const bool lost = bad[n] != 0;
    Coded k = quantize<DT>(kr[s]), v = quantize<DT>(vr[s]);
    if (lost) k = Coded{0, 0, 0x7FC0, 0}, v = Coded{0, 0, 0, 0};
    uint32_t word = 0;
#pragma unroll
    for (int e = 0; e < 8; e++) word |= (((e < 4 ? k.lo : k.hi) >> (8 * (e & 3))) & 15u) << code_shift(e);
    *(uint32_t*)(page + token * (D / 2) + ((c % 4) * (D / 32) + c / 4) * 4) = word;
    *(uint2*)(codes + token * PITCH + c * 8) = uint2{v.lo, v.hi};
    if (c % 8 == 0) {
      const int at = ((token / 4) * NG + g) * 4 + token % 4;
      ((uint16_t*)(page + K_SCALES * D))[at] = k.scale;
      ((uint16_t*)(page + K_OFFSETS * D))[token * NG + g] = f32_to_bf16_bits((float)(k.zero - CODE_BASE));
      ((uint16_t*)(page + V_SCALES * D))[at] = v.scale;
      ((uint16_t*)(page + V_OFFSETS * D))[at] = f32_to_bf16_bits((float)(v.zero - CODE_BASE));
    }
  }
  __syncthreads();
  // value words: 8 tokens of a dim each; those of which the span holds only some keep the others
  for (int unit = tid; unit < 2 * NG * 64; unit += 256) {
    const int half = unit / (NG * 64), g = unit / 64 % NG, lane = unit % 64, q = lane / 16, r = lane % 16;
    uint32_t mask = 0;
#pragma unroll
    for (int e = 0; e < 8; e++) {
      const int token = half * 32 + (e < 4 ? 0 : 12) + 4 * q + e;
      if (token >= t.begin && token < t.end) mask |= 15u << code_shift(e);
    }
    if (mask == 0) continue;
    u32x4 w = {0, 0, 0, 0};
#pragma unroll
    for (int e = 0; e < 8; e++) {
      const int token = half * 32 + (e < 4 ? 0 : 12) + 4 * q + e;
#pragma unroll
      for (int k = 0; k < 4; k++) w[k] |= (codes[token * PITCH + 64 * g + 16 * k + r] & 15u) << code_shift(e);
    }
    u32x4* to = (u32x4*)(page + V_CODES * D) + unit;
    if (mask != 0xFFFFFFFFu) {
      const u32x4 old = *to;
#pragma unroll
      for (int k = 0; k < 4; k++) w[k] = (w[k] & mask) | (old[k] & ~mask);
    }
    *to = w;
  }
}

// 8 codes (bytes) of a group to values of the dense type: exact in fp32, then rounded once.
template <int DT> __device__ __forceinline__ u32x4 expand(uint32_t lo, uint32_t hi, uint16_t scale, uint16_t offset) {
  const float s = bf16_bits_to_f32(scale), z = bf16_bits_to_f32(offset) + (float)CODE_BASE;
  u32x4 out;
#pragma unroll
  for (int k = 0; k < 4; k++) {
    const uint32_t w = k < 2 ? lo >> (16 * k) : hi >> (16 * (k - 2));
    out[k] = Elem<DT>::cvt(((float)(w & 15u) + z) * s) | (uint32_t)Elem<DT>::cvt(((float)((w >> 8) & 15u) + z) * s) << 16;
  }
  return out;
}

template <int DT, int D>
__global__ __launch_bounds__(256) void paged_read_kernel(const uint8_t* __restrict__ pool, const int32_t* __restrict__ table,
                                                         int64_t width, const int32_t* __restrict__ header,
                                                         const Touch* __restrict__ touch, int heads, uint16_t* __restrict__ keys,
                                                         uint16_t* __restrict__ values) {
  constexpr int NG = D / GROUP, CHUNKS = D / 8, PITCH = D + 16;
  __shared__ __align__(16) uint8_t codes[PAGE * PITCH];
  const int tid = threadIdx.x, item = blockIdx.x / heads, h = blockIdx.x % heads;
  if (item >= header[3]) return;
  const Touch t = touch[item];
  const uint8_t* page = pool + ((int64_t)table[t.row * width + t.page] * heads + h) * page_bytes(D);
  for (int unit = tid; unit < 2 * NG * 64; unit += 256) {
    const int half = unit / (NG * 64), g = unit / 64 % NG, lane = unit % 64, q = lane / 16, r = lane % 16;
    const u32x4 w = ((const u32x4*)(page + V_CODES * D))[unit];
#pragma unroll
    for (int e = 0; e < 8; e++) {
      const int token = half * 32 + (e < 4 ? 0 : 12) + 4 * q + e;
#pragma unroll
      for (int k = 0; k < 4; k++) codes[token * PITCH + 64 * g + 16 * k + r] = (w[k] >> code_shift(e)) & 15u;
    }
  }
  __syncthreads();
  for (int slot = tid; slot < (t.end - t.begin) * CHUNKS; slot += 256) {
    const int n = slot / CHUNKS, c = slot % CHUNKS, token = t.begin + n, g = c / 8;
    const uint32_t word = *(const uint32_t*)(page + token * (D / 2) + ((c % 4) * (D / 32) + c / 4) * 4);
    uint32_t lo = 0, hi = 0;
#pragma unroll
    for (int e = 0; e < 8; e++) {
      const uint32_t code = (word >> code_shift(e)) & 15u;
      if (e < 4) lo |= code << (8 * e);
      else hi |= code << (8 * (e - 4));
    }
    const int at = ((token / 4) * NG + g) * 4 + token % 4;
    const int64_t to = ((int64_t)(t.token + n) * heads + h) * D + c * 8;
    *(u32x4*)(keys + to) = expand<DT>(lo, hi, ((const uint16_t*)(page + K_SCALES * D))[at],
                                      ((const uint16_t*)(page + K_OFFSETS * D))[token * NG + g]);
    const uint2 v = *(const uint2*)(codes + token * PITCH + c * 8);
    *(u32x4*)(values + to) = expand<DT>(v.x, v.y, ((const uint16_t*)(page + V_SCALES * D))[at],
                                        ((const uint16_t*)(page + V_OFFSETS * D))[at]);
  }
}

}  // namespace

int launch_update(const Update& u, hipStream_t stream) {
  const int blocks = u.records + (u.entries + 255) / 256 + u.copies;
  if (blocks > 0) paged_update_kernel<<<blocks, 256, 0, stream>>>(u);
  ANNA_LAUNCH_CHECK("paged update");
  return ANNA_MI_OK;
}

int launch_copy(const Copy& c, int64_t layers, hipStream_t stream) {
  if (c.pairs > 0)
    paged_copy_kernel<<<dim3((unsigned)((c.page + COPY_BYTES - 1) / COPY_BYTES), c.pairs, (unsigned)layers), 256, 0, stream>>>(c);
  ANNA_LAUNCH_CHECK("paged copy");
  return ANNA_MI_OK;
}

#define PAGED_DISPATCH(...)                                                                 \
  do {                                                                                      \
    if (dtype == ANNA_MI_BF16) {                                                            \
      constexpr int DT = ANNA_MI_BF16;                                                      \
      if (head_dim == 64) { constexpr int D = 64; __VA_ARGS__; }                            \
      else if (head_dim == 128) { constexpr int D = 128; __VA_ARGS__; }                     \
      else { constexpr int D = 256; __VA_ARGS__; }                                          \
    } else {                                                                                \
      constexpr int DT = ANNA_MI_F16;                                                       \
      if (head_dim == 64) { constexpr int D = 64; __VA_ARGS__; }                            \
      else if (head_dim == 128) { constexpr int D = 128; __VA_ARGS__; }                     \
      else { constexpr int D = 256; __VA_ARGS__; }                                          \
    }                                                                                       \
  } while (0)

int launch_store(int dtype, int64_t head_dim, uint8_t* pool, const int32_t* table, int64_t width, const int32_t* header,
                 const Touch* touch, int64_t touches, int64_t kv_heads, const void* keys, int64_t k_token, int64_t k_head,
                 const void* values, int64_t v_token, int64_t v_head, hipStream_t stream) {
  ANNA_CHECK(touches * kv_heads <= INT32_MAX, "paged_store: too many pages");
  const unsigned grid = (unsigned)(touches * kv_heads);
  PAGED_DISPATCH(paged_store_kernel<DT, D><<<grid, 256, 0, stream>>>(
      pool, table, width, header, touch, (int)kv_heads, (const uint16_t*)keys, k_token, k_head, (const uint16_t*)values, v_token, v_head));
  ANNA_LAUNCH_CHECK("paged store");
  return ANNA_MI_OK;
}

int launch_read(int dtype, int64_t head_dim, const uint8_t* pool, const int32_t* table, int64_t width, const int32_t* header,
                const Touch* touch, int64_t touches, int64_t kv_heads, void* keys, void* values, hipStream_t stream) {
  ANNA_CHECK(touches * kv_heads <= INT32_MAX, "paged_read: too many pages");
  const unsigned grid = (unsigned)(touches * kv_heads);
  PAGED_DISPATCH(paged_read_kernel<DT, D><<<grid, 256, 0, stream>>>(pool, table, width, header, touch, (int)kv_heads, (uint16_t*)keys,
                                                                   (uint16_t*)values));
  ANNA_LAUNCH_CHECK("paged read");
  return ANNA_MI_OK;
}

}  // namespace paged
}  // namespace anna
