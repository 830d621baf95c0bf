// The pages of a key-value cache: layout, addresses and the 8- and 4-bit forms, shared by the kernels that write, read and attend to them.
//
// A page holds `page_size` tokens (32, 64, 128 or 256) of every KV head, head-major, so what a wave reads of one head is contiguous.
//   bf16   K (page, head, token, 128)                       a token's row, as the caller has it
//          V (page, head, token / 8, 128, token % 8)        eight tokens of a channel in 16 bytes: the matrix instruction's operand
//                                                           of V^T, loaded from memory into registers without a transposition
//   8 bits K (page, head, token, 128 bytes), V (page, head, token / 8, 128, token % 8 bytes): as in bf16
//          scales of K and V (page, head, token / 32): one byte for the 32 tokens of a tile and head
//   4 bits K (page, head, token, 64 bytes)                  channel 2j in the low half of byte j
//          V (page, head, token / 4, 16, token % 4, 4 bytes) channels 8m .. 8m + 7 of four tokens in 16 bytes
//          scales of K and V (page, head, token / 32, 4, token % 32): one byte a token and group of 32 channels
//
// 4 bits: e2m1 values (0, 0.5, 1, 1.5, 2, 3, 4, 6 and a sign) times 2^e, e + 127 in the byte.  e is the smallest exponent with no
// value of the group above 7 * 2^e: then none is off by more than half the largest step (7 itself becomes 6).  -100 <= e <= 125:
// smaller groups are held as zeros, and 6 * 2^125 is the largest value held.  A group with an infinity or NaN is held as NaN (byte 255).
// 8 bits: e4m3 values (4 bits of precision, up to 448, multiples of 2^-9) times 2^e, e + 127 in the byte.  e is the smallest exponent with no
// finite value of the tile above 448 * 2^e, -100 <= e <= 119; 448 * 2^119 is the largest value held.  An infinity or NaN is held as NaN, by itself.
// The tile's exponent goes up with the tokens that join it, and the codes that are there follow (which rounds those that become less than
// 2^-6 of the scale once more); it starts anew with the tile's first token and never goes down, also where tokens come off the sequence's end.
// Scales are powers of two and the conversions round to nearest even, so what is held follows from the bf16 values alone, to the bit.
#pragma once
#include "pbs_common.h"

constexpr int PAGED_D = 128;
constexpr int PAGED_TILE = 32;   // tokens of a tile: one contraction of the matrix instruction over keys
constexpr int PAGED_MAX_TOKENS = 1 << 30;   // of a sequence: positions stay in 32 bits

struct PagedPool {
  char* k;
  char* v;
  uint8_t* ks;   // scales, 8 and 4 bits only
  uint8_t* vs;
  const int32_t* table;   // (B, max_pages)
  int64_t table_sb;
  int num_pages, max_pages, page_shift, heads;
};

// bytes of one head of a tile of 32 tokens, K or V
template <int BITS>
constexpr int paged_tile_bytes() { return PAGED_TILE * PAGED_D * BITS / 8; }

// The tiles of a pool, counted through pages and heads: tile `t` (of 32 tokens) of a sequence and head; -1 where its page is not in the
// pool or behind the table.
__device__ __forceinline__ int64_t paged_tile_index(const PagedPool& p, int b, int head, int t) {
  const int tiles_shift = p.page_shift - 5, slot = t >> tiles_shift;
  if (slot >= p.max_pages) return -1;
  const int page = p.table[b * p.table_sb + slot];
  if ((unsigned)page >= (unsigned)p.num_pages) return -1;
  return (((int64_t)page * p.heads + head) << tiles_shift) + (t & ((1 << tiles_shift) - 1));
}

// scale byte of a group whose largest magnitude has these bits (bf16, no sign)
__device__ __forceinline__ uint32_t fp4_scale_byte(uint32_t amax) {
  const int e = (int)((amax + 0x1fu) >> 7) - 2;   // the exponent field, one up where the value is above 1.75 * 2^n
  return amax >= 0x7f80u ? 255u : (uint32_t)min(max(e, 27), 252);
}

// 8 bf16 values (two a word) -> 8 codes; `scale` = 2^e.  (Divides by the scale and rounds to nearest even.)
__device__ __forceinline__ uint32_t fp4_codes(u32x4 x, float scale) {
  // (each word by itself: a bit cast of a vector's element takes the vector's first)
  const uint32_t a = x[0], b = x[1], c = x[2], d = x[3];
  uint32_t r = 0;
  r = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(r, __builtin_bit_cast(bf16x2, a), scale, 0);
  r = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(r, __builtin_bit_cast(bf16x2, b), scale, 1);
  r = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(r, __builtin_bit_cast(bf16x2, c), scale, 2);
  r = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(r, __builtin_bit_cast(bf16x2, d), scale, 3);
  return r;
}

// the 8 values of a word of codes, bf16 (exact: a code times a power of two in the range above; NaN where the scale's byte is 255)
__device__ __forceinline__ u32x4 fp4_values(uint32_t codes, float scale) {
  return (u32x4){__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 0)),
                 __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 1)),
                 __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 2)),
                 __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 3))};
}

// ---- 8 bits ----------------------------------------------------------------------------------------------------------------------
typedef __attribute__((ext_vector_type(2))) short s16x2;
typedef __attribute__((ext_vector_type(2))) uint32_t u32x2;
constexpr uint32_t FP8_MOST = 0x7f60u;   // 448 * 2^119 in bf16
__device__ __forceinline__ bool not_finite(uint32_t bf16_bits) { return (bf16_bits & 0x7f80u) == 0x7f80u; }
__device__ __forceinline__ bool fp8_is_nan(uint32_t code) { return (code & 0x7fu) == 0x7fu; }

// scale byte of a tile whose largest finite magnitude has these bits (bf16, no sign)
__device__ __forceinline__ uint32_t fp8_scale_byte(uint32_t amax) {
  return (uint32_t)min(max((int)((amax + 0x1fu) >> 7) - 8, 27), 246);   // the exponent field, one up where the value is above 1.75 * 2^n
}
// two bf16 values with what the conversion does not take mended: infinities become NaN, larger magnitudes 448 * 2^119
__device__ __forceinline__ uint32_t fp8_ready(uint32_t x) {
  auto one = [](uint32_t h) { return not_finite(h) ? h | 0x40u : (h & 0x8000u) | min(h & 0x7fffu, FP8_MOST); };
  return one(x & 0xffffu) | (one(x >> 16) << 16);
}
// 4 bf16 values (two a word) -> 4 codes; `scale` = 2^e.  (Divides by the scale and rounds to nearest even.)
__device__ __forceinline__ uint32_t fp8_codes(uint32_t a, uint32_t b, float scale) {
  s16x2 r = {};
  r = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(r, __builtin_bit_cast(bf16x2, a), scale, 0);
  r = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(r, __builtin_bit_cast(bf16x2, b), scale, 1);
  return __builtin_bit_cast(uint32_t, r);
}
// the values of codes 2 HIGH and 2 HIGH + 1 of a word, bf16 (exact: 4 bits times a power of two in the range above)
template <int HIGH>
__device__ __forceinline__ uint32_t fp8_pair(uint32_t codes, float scale) {
  return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(codes, scale, HIGH));
}

// checks that every entry point on pages makes; fills `p`
int paged_pool(PagedPool* p, const char* what, const void* k_pages, const void* v_pages, const void* k_scale, const void* v_scale,
               const int32_t* page_table, int64_t table_sb, int B, int Hkv, int head_dim, int num_pages, int max_pages, int page_size, int kv_bits);
