// Paged 4-bit KV cache: tokens into pages and back, page copies, and the tables' and spans' updates
// (page layout in anna_mi.h).
#include "paged.hpp"

namespace anna {
namespace paged {
namespace {

// ---------------------------------------------------------------- page copies
// A workgroup copies 16 KB (COPY_BYTES) of a page of a layer (all KV heads), 64 bytes a thread: 94 pages of 32 layers
// (444 MB read and written) take 70 us, 6.3 TB/s, some of it out of the last level's cache; a resize with 408 of them in use
// 349 us, 5.5 TB/s.  Memory bounds it.
__device__ __forceinline__ void copy_chunk(const uint8_t* from, uint8_t* to, int64_t page, int64_t chunk) {
  const int64_t at = chunk * COPY_BYTES + threadIdx.x * 16;
  u32x4 v[4];
#pragma unroll
  for (int k = 0; k < 4; k++) {
    v[k] = u32x4{0, 0, 0, 0};
    if (from && at + k * 4096 < page) v[k] = __builtin_nontemporal_load((const u32x4*)(from + at + k * 4096));
  }
#pragma unroll
  for (int k = 0; k < 4; k++)
    if (at + k * 4096 < page) *(u32x4*)(to + at + k * 4096) = v[k];
}

__global__ __launch_bounds__(256) void paged_copy_kernel(const Copy c) {
  const int source = c.words[2 * blockIdx.y], target = c.words[2 * blockIdx.y + 1];
  copy_chunk(source < 0 ? nullptr : c.from + blockIdx.z * c.from_layer + source * c.page,
             c.to + blockIdx.z * c.to_layer + target * c.page, c.page, blockIdx.x);
}

// ---------------------------------------------------------------- updates
// One workgroup writes what a record says, one 256 table entries, one a whole table row, one copies 16 KB of a page of
// a layer: all that a step needs before its first layer, in one launch.
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
  words += 2 * u.entries;
  if (blk >= u.copies) {
    blk -= u.copies;
    words += 3 * u.copies;
    const int chunks = (int)((u.page + COPY_BYTES - 1) / COPY_BYTES), pair = blk / (chunks * u.layers), layer = blk / chunks % u.layers;
    uint8_t* base = u.pool + layer * u.pool_layer;
    copy_chunk(base + words[2 * pair] * u.page, base + words[2 * pair + 1] * u.page, u.page, blk % chunks);
    return;
  }
  words += 3 * blk;
  int32_t* row = u.table + words[0] * u.width;
  const int32_t* source = u.table + words[1] * u.width;
  for (int k = tid; k < u.width; k += 256) {
    if (k >= words[2]) row[k] = 0;
    else if (words[1] >= 0) row[k] = source[k];
  }
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

// x / y by the (nearly exact) reciprocal of y and one correction: exact where the quotient has few bits, as the halves
// between two codes or two bf16 scales have, and elsewhere far nearer to it than it is to such a half (x and y have 19
// bits between them).  Three instructions, where a division takes ten.
__device__ __forceinline__ float quotient(float x, float y, float reciprocal) {
  const float q = x * reciprocal;
  return fmaf(fmaf(-q, y, x), reciprocal, q);
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
  const float spread = fmaxf(quotient(0.5f * high - 0.5f * low, 7.5f, 1.0f / 7.5f),
                             quotient(fmaxf(fabsf(low), fabsf(high)), 120.0f, 1.0f / 120.0f));
  Coded c = {0, 0, 0, 0};
  if (!(spread >= 7.888609052210118e-31f)) return c;  // 2^-100
  c.scale = f32_to_bf16_bits(spread);
  const float scale = bf16_bits_to_f32(c.scale), inverse = __builtin_amdgcn_rcpf(scale);
  auto steps = [&](float v) { return rintf(quotient(v, scale, inverse)); };
  const float zero = steps(low);
  c.zero = (int)zero;
#pragma unroll
  for (int k = 0; k < 4; k++) {
    c.lo = __builtin_amdgcn_cvt_pk_u8_f32(__builtin_amdgcn_fmed3f(steps(x[k]) - zero, 0.0f, 15.0f), k, c.lo);
    c.hi = __builtin_amdgcn_cvt_pk_u8_f32(__builtin_amdgcn_fmed3f(steps(x[4 + k]) - zero, 0.0f, 15.0f), k, c.hi);
  }
  return c;
}

// Two nibbles a byte: bytes 0 and 2 of x with the next one above each, as 16 bits.
__device__ __forceinline__ uint32_t nibbles(uint32_t x) { return __builtin_amdgcn_perm(0, x | x >> 4, 0x0C0C0200); }
// A word of 8 codes, one a byte: code e at bits 4 * ((e % 2) * 4 + e / 2).
__device__ __forceinline__ uint32_t code_word(uint32_t lo, uint32_t hi) {
  return nibbles(__builtin_amdgcn_perm(hi, lo, 0x06040200)) | nibbles(__builtin_amdgcn_perm(hi, lo, 0x07050301)) << 16;
}

// Tokens of a page and KV head into the page: eight lanes a group, keys straight to their words, values by way of LDS,
// where the codes of eight tokens meet in a word.  Prompts (7957 tokens of 8 heads, 42 MB): 17.6 us, 2.4 TB/s, bound by the
// vector unit (~350 instructions for 16 values of 8 lanes, a third of them rounding) and the chain of a workgroup's
// passes; one token of each of 64 sequences: 5 us, the chain alone.
template <int DT, int D>
__global__ __launch_bounds__(256) void paged_store_kernel(uint8_t* __restrict__ pool, const int32_t* __restrict__ table, int64_t width,
                                                          const int32_t* __restrict__ header, const Touch* __restrict__ touch,
                                                          int heads, const uint16_t* __restrict__ keys, int64_t k_token, int64_t k_head,
                                                          const uint16_t* __restrict__ values, int64_t v_token, int64_t v_head) {
  constexpr int NG = D / GROUP, CHUNKS = D / 8, PITCH = D + 16;
  __shared__ __align__(16) uint8_t codes[PAGE * PITCH];     // of the values
  __shared__ __align__(16) uint8_t image[page_bytes(D)];  // of a page that is written whole, in 16-byte words at the end
  __shared__ int bad[PAGE];
  const int tid = threadIdx.x, item = blockIdx.x / heads, h = blockIdx.x % heads;
  if (item >= header[3]) return;
  const Touch t = touch[item];
  uint8_t* page = pool + ((int64_t)table[t.row * width + t.page] * heads + h) * page_bytes(D);
  const int slots = (t.end - t.begin) * CHUNKS;
  const bool whole = t.end - t.begin == PAGE;
  auto put = [&](int at, auto value) {
    if (whole) *(decltype(value)*)(image + at) = value;
    else *(decltype(value)*)(page + at) = value;
  };
  if (tid < PAGE) bad[tid] = 0;
  const uint16_t *k_from = keys + t.token * k_token + h * k_head, *v_from = values + t.token * v_token + h * v_head;
  auto key = [&](int slot) { return *(const u32x4*)(k_from + slot / CHUNKS * k_token + slot % CHUNKS * 8); };
  auto value = [&](int slot) { return *(const u32x4*)(v_from + slot / CHUNKS * v_token + slot % CHUNKS * 8); };
  // The values go by twice: once for what is not finite, which concerns a token's keys and values, and once, out of
  // the cache, for their codes.  Only the first of a thread's, all that a single token has, stay in registers.
  u32x4 k0 = {0, 0, 0, 0}, v0 = {0, 0, 0, 0};
  if (tid < slots) k0 = key(tid), v0 = value(tid);
  __syncthreads();
  if (tid < slots && (not_finite<DT>(k0) || not_finite<DT>(v0))) bad[tid / CHUNKS] = 1;
  for (int slot = tid + 256; slot < slots; slot += 256)
    if (not_finite<DT>(key(slot)) || not_finite<DT>(value(slot))) bad[slot / CHUNKS] = 1;
  __syncthreads();
  for (int slot = tid; slot < slots; slot += 256) {  // whole groups of 8 lanes
    const u32x4 kr = slot == tid ? k0 : key(slot), vr = slot == tid ? v0 : value(slot);
    const int n = slot / CHUNKS, c = slot % CHUNKS, token = t.begin + n, g = c / 8;
    Coded k = {0, 0, 0x7FC0, 0}, v = {0, 0, 0, 0};
    if (!bad[n]) {
      k = quantize<DT>(kr);
      v = quantize<DT>(vr);
    }
    put(token * (D / 2) + ((c % 4) * (D / 32) + c / 4) * 4, code_word(k.lo, k.hi));
    *(uint2*)(codes + token * PITCH + c * 8) = uint2{v.lo, v.hi};
    if (c % 8 == 0) {
      const int at = 2 * (((token / 4) * NG + g) * 4 + token % 4);
      put(K_SCALES * D + at, k.scale);
      put(K_OFFSETS * D + 2 * (token * NG + g), f32_to_bf16_bits((float)(k.zero - CODE_BASE)));
      put(V_SCALES * D + at, v.scale);
      put(V_OFFSETS * D + at, f32_to_bf16_bits((float)(v.zero - CODE_BASE)));
    }
  }
  __syncthreads();
  // Value words: 8 tokens of a dim each; those of which the span holds only some keep the others.  A thread takes four
  // neighbouring dims: a dword of each token, two tokens to a byte, then the four dims' bytes apart.
  for (int unit = tid; unit < 2 * NG * 64; unit += 256) {
    const int half = unit / (NG * 64), g = unit / 64 % NG, w = unit / 16 % 4, q = unit / 4 % 4, r = unit % 4 * 4;
    const int first = half * 32 + 4 * q;
    uint32_t mask = 0;
#pragma unroll
    for (int e = 0; e < 8; e++) {
      const int token = first + (e < 4 ? e : 12 + e);
      if (token >= t.begin && token < t.end) mask |= 15u << code_shift(e);
    }
    if (mask == 0) continue;
    uint32_t v[8], two[4];
#pragma unroll
    for (int e = 0; e < 8; e++)
      v[e] = *(const uint32_t*)(codes + (first + (e < 4 ? e : 12 + e)) * PITCH + 64 * g + 16 * w + r) & 0x0F0F0F0Fu;
    // nibbles 0 .. 7 of a word are tokens 0, 2, 4, 6, 1, 3, 5, 7
    two[0] = v[0] | v[2] << 4, two[1] = v[4] | v[6] << 4, two[2] = v[1] | v[3] << 4, two[3] = v[5] | v[7] << 4;
    const uint32_t ab = __builtin_amdgcn_perm(two[1], two[0], 0x05010400), AB = __builtin_amdgcn_perm(two[1], two[0], 0x07030602);
    const uint32_t cd = __builtin_amdgcn_perm(two[3], two[2], 0x05010400), CD = __builtin_amdgcn_perm(two[3], two[2], 0x07030602);
    const uint32_t word[4] = {__builtin_amdgcn_perm(cd, ab, 0x05040100), __builtin_amdgcn_perm(cd, ab, 0x07060302),
                              __builtin_amdgcn_perm(CD, AB, 0x05040100), __builtin_amdgcn_perm(CD, AB, 0x07060302)};
    const int at = V_CODES * D + (((half * NG + g) * 64 + q * 16 + r) * 4 + w) * 4;
#pragma unroll
    for (int k = 0; k < 4; k++)
      put(at + 16 * k, mask == 0xFFFFFFFFu ? word[k] : (word[k] & mask) | (*(const uint32_t*)(page + at + 16 * k) & ~mask));
  }
  if (!whole) return;
  __syncthreads();
  for (int at = tid * 16; at < page_bytes(D); at += 256 * 16) *(u32x4*)(page + at) = *(const u32x4*)(image + at);
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

// A page's tokens dense again, values by way of LDS.  7957 tokens of 8 heads (42 MB): 10 us, 4.3 TB/s; memory bounds it.
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
  const int64_t blocks = u.records + (u.entries + 255) / 256 + u.copies +
                         (int64_t)u.pairs * u.layers * ((u.page + COPY_BYTES - 1) / COPY_BYTES);
  ANNA_CHECK(blocks <= INT32_MAX, "paged update: too many pages to copy");
  if (blocks > 0) paged_update_kernel<<<(unsigned)blocks, 256, 0, stream>>>(u);
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
