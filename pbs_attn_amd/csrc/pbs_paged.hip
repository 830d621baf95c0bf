// Writing new keys and values into a paged cache, with the rotary embedding on the way, and reading a cache back.
#include "pbs_paged.h"
#include "../../include/pbs_hip.h"   // the definitions below are checked against the public declarations

int paged_pool(PagedPool* p, const char* what, const void* k_pages, const void* v_pages, const void* k_scale, const void* v_scale,
               const int32_t* page_table, int64_t table_sb, int B, int Hkv, int head_dim, int num_pages, int max_pages, int page_size, int kv_bits) {
  PBS_REQUIRE(k_pages && v_pages && page_table, "%s: null tensor pointer", what);
  PBS_REQUIRE(head_dim == PAGED_D, "%s: head_dim must be 128, got %d", what, head_dim);
  PBS_REQUIRE(kv_bits == 16 || kv_bits == 4, "%s: a cache of 16 or 4 bits, got %d", what, kv_bits);
  PBS_REQUIRE(kv_bits == 16 || (k_scale && v_scale), "%s: a cache of 4 bits needs its scales", what);
  PBS_REQUIRE(page_size == 32 || page_size == 64 || page_size == 128 || page_size == 256, "%s: pages of 32, 64, 128 or 256 tokens, got %d", what, page_size);
  PBS_REQUIRE(B > 0 && B <= 65535 && Hkv > 0 && Hkv <= 65535, "%s: bad shape", what);
  PBS_REQUIRE(num_pages > 0 && max_pages > 0 && (int64_t)max_pages * page_size <= PAGED_MAX_TOKENS,
              "%s: no pages, or more than 2^30 tokens a sequence", what);
  PBS_REQUIRE((((uintptr_t)k_pages | (uintptr_t)v_pages | (uintptr_t)k_scale | (uintptr_t)v_scale) % 16) == 0,
              "%s: pages and scales must be 16-byte aligned", what);
  p->k = (char*)k_pages; p->v = (char*)v_pages; p->ks = (uint8_t*)k_scale; p->vs = (uint8_t*)v_scale;
  p->table = page_table; p->table_sb = table_sb;
  p->num_pages = num_pages; p->max_pages = max_pages; p->page_shift = __builtin_ctz(page_size); p->heads = Hkv;
  return 0;
}

namespace {

struct AppendArgs {
  PagedPool pool;
  const uint16_t* q;
  const uint16_t* k;
  const uint16_t* v;
  const uint16_t* cos;   // null: no rotation
  const uint16_t* sin;
  uint16_t* q_out;   // (B, Hq, S, 128) contiguous
  uint16_t* k_out;   // (B, Hkv, S, 128) contiguous, or null
  const int32_t* past;
  const int32_t* fresh;   // new tokens of each sequence, null: S
  int B, Hq, Hkv, S;
  int q_heads, q_groups;   // heads of Q that a workgroup goes through with the same cosines, and how many such groups
  int64_t q_sb, q_sh, q_ss, k_sb, k_sh, k_ss, v_sb, v_sh, v_ss, c_sb, c_ss;
};

__device__ __forceinline__ uint32_t largest_bits(u32x4 x) {
  uint32_t m = 0;
#pragma unroll
  for (int e = 0; e < 4; ++e) m = max(m, max(x[e] & 0x7fffu, (x[e] >> 16) & 0x7fffu));
  return m;
}

// x c - y s, x and y c + x s of bf16 pairs: the products are exact in fp32, the sum is rounded once to fp32 and the result once to bf16
__device__ __forceinline__ uint32_t rotate_pair(uint32_t x, uint32_t y, uint32_t c, uint32_t s, float sign) {
  const float lo = __builtin_fmaf(sign * bf16_bits_to_f32(y & 0xffffu), bf16_bits_to_f32(s & 0xffffu), bf16_bits_to_f32(x & 0xffffu) * bf16_bits_to_f32(c & 0xffffu));
  const float hi = __builtin_fmaf(sign * __uint_as_float(y & 0xffff0000u), __uint_as_float(s & 0xffff0000u),
                                  __uint_as_float(x & 0xffff0000u) * __uint_as_float(c & 0xffff0000u));
  return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2){lo, hi}, bf16x2));
}

// Workgroups of 32 tokens (a tile of the cache: its positions, not the call's rows, are aligned) and a few heads of Q, K or V.  Eight lanes
// hold a row, each lane the same 8 channels of both halves, which is what the rotation exchanges; cosines and sines stay in registers over
// the heads.  Bound by memory, each row in and out once: an 8192-token prompt (32 / 8 heads) into bf16 pages 49 us, 4.5 TB/s.  A single token
// takes 3.2 us, two round trips to memory.
template <int BITS>
__global__ __launch_bounds__(256) void append_kernel(AppendArgs a) {
  const int b = blockIdx.z, past = min(max(a.past[b], 0), PAGED_MAX_TOKENS), fresh = a.fresh ? min(max(a.fresh[b], 0), a.S) : a.S;
  const int tile = past / PAGED_TILE + blockIdx.x;
  const int first = tile * PAGED_TILE - past;   // the call's row at the tile's first position: may be negative
  if (first >= a.S) return;
  int group = blockIdx.y;
  const int kind = group < a.q_groups ? 0 : group < a.q_groups + a.Hkv ? 1 : 2;   // Q, K, V
  group -= kind == 0 ? 0 : kind == 1 ? a.q_groups : a.q_groups + a.Hkv;
  const int h0 = kind == 0 ? group * a.q_heads : group, h1 = kind == 0 ? min(h0 + a.q_heads, a.Hq) : h0 + 1;
  if (kind == 2 && first >= fresh) return;
  const int c = threadIdx.x & 7, row = threadIdx.x >> 3, s = first + row;
  const bool in_call = s >= 0 && s < a.S, stored = s >= 0 && s < fresh;

  if (kind == 2 && BITS == 16) {
    // eight tokens of two channels: rows are read whole (a wave reads 256 bytes of each), the cache gets 32 bytes a lane
    const int d = (threadIdx.x & 63) * 2, eight = threadIdx.x >> 6, s0 = first + eight * 8;
    if (s0 + 8 <= 0 || s0 >= fresh) return;
    for (int h = h0; h < h1; ++h) {
      const int64_t at = paged_tile_index(a.pool, b, h, tile);
      if (at < 0) return;
      const uint16_t* src = a.v + b * a.v_sb + h * a.v_sh + d;
      uint16_t* dst = (uint16_t*)(a.pool.v + at * paged_tile_bytes<16>()) + (eight * PAGED_D + d) * 8;
      uint32_t w[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) w[j] = s0 + j >= 0 && s0 + j < fresh ? *(const uint32_t*)(src + (int64_t)(s0 + j) * a.v_ss) : 0;
      if (s0 >= 0 && s0 + 8 <= fresh) {
        u32x4 x, y;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          x[j] = (w[2 * j] & 0xffffu) | (w[2 * j + 1] << 16);
          y[j] = (w[2 * j] >> 16) | (w[2 * j + 1] & 0xffff0000u);
        }
        *(u32x4*)dst = x;
        *(u32x4*)(dst + 8) = y;
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (s0 + j >= 0 && s0 + j < fresh) {
            dst[j] = (uint16_t)w[j];
            dst[8 + j] = (uint16_t)(w[j] >> 16);
          }
      }
    }
    return;
  }

  u32x4 c0 = {}, c1 = {}, s0 = {}, s1 = {};
  if (kind < 2 && a.cos && in_call) {
    const uint16_t* pc = a.cos + b * a.c_sb + (int64_t)s * a.c_ss + c * 8;
    const uint16_t* ps = a.sin + b * a.c_sb + (int64_t)s * a.c_ss + c * 8;
    c0 = *(const u32x4*)pc; c1 = *(const u32x4*)(pc + 64);
    s0 = *(const u32x4*)ps; s1 = *(const u32x4*)(ps + 64);
  }
  for (int h = h0; h < h1; ++h) {
    u32x4 x0 = {}, x1 = {};
    if (in_call) {
      const uint16_t* src = kind == 0   ? a.q + b * a.q_sb + h * a.q_sh + (int64_t)s * a.q_ss
                            : kind == 1 ? a.k + b * a.k_sb + h * a.k_sh + (int64_t)s * a.k_ss
                                        : a.v + b * a.v_sb + h * a.v_sh + (int64_t)s * a.v_ss;
      x0 = *(const u32x4*)(src + c * 8);
      x1 = *(const u32x4*)(src + 64 + c * 8);
    }
    if (kind < 2) {
      if (a.cos) {
        u32x4 y0, y1;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          y0[e] = rotate_pair(x0[e], x1[e], c0[e], s0[e], -1.0f);
          y1[e] = rotate_pair(x1[e], x0[e], c1[e], s1[e], 1.0f);
        }
        x0 = y0; x1 = y1;
      }
      uint16_t* out = kind == 0 ? a.q_out : a.k_out;
      if (out && in_call) {
        out += (((int64_t)b * (kind == 0 ? a.Hq : a.Hkv) + h) * a.S + s) * PAGED_D + c * 8;
        *(u32x4*)out = x0;
        *(u32x4*)(out + 64) = x1;
      }
      if (kind == 0) continue;
    }
    const int64_t at = paged_tile_index(a.pool, b, h, tile);
    if (BITS == 16) {   // K
      if (at >= 0 && stored) {
        uint16_t* dst = (uint16_t*)(a.pool.k + at * paged_tile_bytes<16>()) + row * PAGED_D + c * 8;
        *(u32x4*)dst = x0;
        *(u32x4*)(dst + 64) = x1;
      }
    } else {
      // four lanes hold a group of 32 channels: lanes 0-3 groups 0 and 2, lanes 4-7 groups 1 and 3
      uint32_t m0 = largest_bits(x0), m1 = largest_bits(x1);
      m0 = max(m0, (uint32_t)__shfl_xor((int)m0, 1, 64)); m0 = max(m0, (uint32_t)__shfl_xor((int)m0, 2, 64));
      m1 = max(m1, (uint32_t)__shfl_xor((int)m1, 1, 64)); m1 = max(m1, (uint32_t)__shfl_xor((int)m1, 2, 64));
      const uint32_t e0 = fp4_scale_byte(m0), e1 = fp4_scale_byte(m1);
      const uint32_t w0 = fp4_codes(x0, __uint_as_float(e0 << 23)), w1 = fp4_codes(x1, __uint_as_float(e1 << 23));
      if (at >= 0 && stored) {
        char* dst = (kind == 1 ? a.pool.k : a.pool.v) + at * paged_tile_bytes<4>();
        uint8_t* scale = (kind == 1 ? a.pool.ks : a.pool.vs) + at * 128;
        const int p0 = kind == 1 ? row * 64 + c * 4 : (row >> 2) * 256 + c * 16 + (row & 3) * 4;
        *(uint32_t*)(dst + p0) = w0;
        *(uint32_t*)(dst + p0 + (kind == 1 ? 32 : 128)) = w1;
        if ((c & 3) == 0) {
          scale[(c >> 2) * 32 + row] = (uint8_t)e0;
          scale[(2 + (c >> 2)) * 32 + row] = (uint8_t)e1;
        }
      }
    }
  }
}

struct ReadArgs {
  PagedPool pool;
  const int32_t* lens;
  uint16_t* k_out;   // (B, Hkv, L, 128) contiguous
  uint16_t* v_out;
  int L;
};

// A workgroup per tile of 32 tokens and head, K and V.  Bound by memory (18 000 tokens of 4 heads out of 4 bits: 47 MB in 9 us;
// out of bf16: 74 MB in 13.5 us).
template <int BITS>
__global__ __launch_bounds__(256) void read_kernel(ReadArgs a) {
  const int tile = blockIdx.x, h = blockIdx.y, b = blockIdx.z;
  const int len = min(max(a.lens[b], 0), a.L) - tile * PAGED_TILE;   // tokens of the tile, may be 0 or less
  const int rows = min(PAGED_TILE, a.L - tile * PAGED_TILE);
  const int64_t at = len > 0 ? paged_tile_index(a.pool, b, h, tile) : -1;
  const int64_t out = (((int64_t)b * a.pool.heads + h) * a.L + tile * PAGED_TILE) * PAGED_D;
  const int c = threadIdx.x & 7, row = threadIdx.x >> 3;
  const bool held = at >= 0 && row < len;
  if (BITS == 16) {
    u32x4 x0 = {}, x1 = {};
    if (held) {
      const uint16_t* src = (const uint16_t*)(a.pool.k + at * paged_tile_bytes<16>()) + row * PAGED_D + c * 8;
      x0 = *(const u32x4*)src;
      x1 = *(const u32x4*)(src + 64);
    }
    if (row < rows) {
      uint16_t* dst = a.k_out + out + row * PAGED_D + c * 8;
      *(u32x4*)dst = x0;
      *(u32x4*)(dst + 64) = x1;
    }
    const int d = (threadIdx.x & 63) * 2, eight = threadIdx.x >> 6;   // eight tokens of two channels
    u32x4 y0 = {}, y1 = {};
    if (at >= 0 && eight * 8 < len) {
      const uint16_t* src = (const uint16_t*)(a.pool.v + at * paged_tile_bytes<16>()) + (eight * PAGED_D + d) * 8;
      y0 = *(const u32x4*)src;
      y1 = *(const u32x4*)(src + 8);
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const uint32_t lo = (y0[j / 2] >> (16 * (j & 1))) & 0xffffu, hi = (y1[j / 2] >> (16 * (j & 1))) << 16;
      if (eight * 8 + j < rows) *(uint32_t*)(a.v_out + out + (eight * 8 + j) * PAGED_D + d) = eight * 8 + j < len ? lo | hi : 0u;
    }
  } else {
#pragma unroll
    for (int kv = 0; kv < 2; ++kv) {
      u32x4 x0 = {}, x1 = {};
      if (held) {
        const char* src = (kv == 0 ? a.pool.k : a.pool.v) + at * paged_tile_bytes<4>();
        const uint8_t* scale = (kv == 0 ? a.pool.ks : a.pool.vs) + at * 128;
        const int p0 = kv == 0 ? row * 64 + c * 4 : (row >> 2) * 256 + c * 16 + (row & 3) * 4;
        const float e0 = __uint_as_float((uint32_t)scale[(c >> 2) * 32 + row] << 23), e1 = __uint_as_float((uint32_t)scale[(2 + (c >> 2)) * 32 + row] << 23);
        x0 = fp4_values(*(const uint32_t*)(src + p0), e0);
        x1 = fp4_values(*(const uint32_t*)(src + p0 + (kv == 0 ? 32 : 128)), e1);
      }
      if (row < rows) {
        uint16_t* dst = (kv == 0 ? a.k_out : a.v_out) + out + row * PAGED_D + c * 8;
        *(u32x4*)dst = x0;
        *(u32x4*)(dst + 64) = x1;
      }
    }
  }
}

}  // namespace

extern "C" int pbs_paged_append(const void* q, const void* k, const void* v, const void* cos, const void* sin, void* q_out, void* k_out, void* k_pages,
                                void* v_pages, void* k_scale, void* v_scale, const int32_t* page_table, const int32_t* past_lens,
                                const int32_t* new_lens, int B, int Hq, int Hkv, int S, int head_dim, int num_pages, int max_pages, int page_size,
                                int kv_bits, int64_t q_sb, int64_t q_sh, int64_t q_ss, int64_t k_sb, int64_t k_sh, int64_t k_ss, int64_t v_sb,
                                int64_t v_sh, int64_t v_ss, int64_t c_sb, int64_t c_ss, int64_t table_sb, void* stream) {
  AppendArgs a;
  if (const int rc = paged_pool(&a.pool, "pbs_paged_append", k_pages, v_pages, k_scale, v_scale, page_table, table_sb, B, Hkv, head_dim, num_pages,
                                max_pages, page_size, kv_bits))
    return rc;
  PBS_REQUIRE(k && v && past_lens, "pbs_paged_append: null tensor pointer");
  PBS_REQUIRE(!q == !q_out, "pbs_paged_append: q goes with q_out");
  PBS_REQUIRE(!cos == !sin, "pbs_paged_append: cos goes with sin");
  PBS_REQUIRE(S > 0 && S <= (1 << 26) && Hq >= 0 && Hq <= 65535 && (!q || Hq > 0), "pbs_paged_append: bad shape");
  PBS_REQUIRE(((q_sb | q_sh | q_ss | k_sb | k_sh | k_ss | v_sb | v_sh | v_ss | c_sb | c_ss) % 8) == 0,
              "pbs_paged_append: strides must keep rows 16-byte aligned");
  PBS_REQUIRE((((uintptr_t)q | (uintptr_t)k | (uintptr_t)v | (uintptr_t)cos | (uintptr_t)sin | (uintptr_t)q_out | (uintptr_t)k_out) % 16) == 0,
              "pbs_paged_append: pointers must be 16-byte aligned");
  if (!q) Hq = 0;
  a.q = (const uint16_t*)q; a.k = (const uint16_t*)k; a.v = (const uint16_t*)v; a.cos = (const uint16_t*)cos; a.sin = (const uint16_t*)sin;
  a.q_out = (uint16_t*)q_out; a.k_out = (uint16_t*)k_out;
  a.past = past_lens; a.fresh = new_lens;
  a.B = B; a.Hq = Hq; a.Hkv = Hkv; a.S = S;
  a.q_sb = q_sb; a.q_sh = q_sh; a.q_ss = q_ss; a.k_sb = k_sb; a.k_sh = k_sh; a.k_ss = k_ss; a.v_sb = v_sb; a.v_sh = v_sh; a.v_ss = v_ss;
  a.c_sb = c_sb; a.c_ss = c_ss;
  const int tiles = (S + 2 * PAGED_TILE - 2) / PAGED_TILE;   // whatever the position of the first row in its tile
  // Cosines and sines are twice a row's own bytes: with four heads of Q a workgroup they are read a quarter as often (32 / 8 heads, 8192 tokens
  // into a bf16 cache 57.8 -> 48.7 us), where the chip is full all the same (1024 tokens 7.2 us with one, 7.4 with four, 10.0 with eight).
  a.q_heads = (int64_t)tiles * B * Hq >= 4096 ? 4 : 1;
  a.q_groups = (Hq + a.q_heads - 1) / a.q_heads;
  PBS_REQUIRE(a.q_groups + 2 * Hkv <= 65535, "pbs_paged_append: too many heads");
  const dim3 grid(tiles, a.q_groups + 2 * Hkv, B);
  if (kv_bits == 16) hipLaunchKernelGGL(append_kernel<16>, grid, dim3(256), 0, (hipStream_t)stream, a);
  else hipLaunchKernelGGL(append_kernel<4>, grid, dim3(256), 0, (hipStream_t)stream, a);
  return pbs_check_launch("pbs_paged_append");
}

extern "C" int pbs_paged_read(const void* k_pages, const void* v_pages, const void* k_scale, const void* v_scale, const int32_t* page_table,
                              const int32_t* lens, void* k_out, void* v_out, int B, int Hkv, int max_len, int head_dim, int num_pages, int max_pages,
                              int page_size, int kv_bits, int64_t table_sb, void* stream) {
  ReadArgs a;
  if (const int rc = paged_pool(&a.pool, "pbs_paged_read", k_pages, v_pages, k_scale, v_scale, page_table, table_sb, B, Hkv, head_dim, num_pages,
                                max_pages, page_size, kv_bits))
    return rc;
  PBS_REQUIRE(lens && k_out && v_out, "pbs_paged_read: null tensor pointer");
  PBS_REQUIRE(max_len > 0 && max_len <= (1 << 28), "pbs_paged_read: bad shape");   // (a grid's threads fit 32 bits)
  PBS_REQUIRE((((uintptr_t)k_out | (uintptr_t)v_out) % 16) == 0, "pbs_paged_read: pointers must be 16-byte aligned");
  a.lens = lens; a.k_out = (uint16_t*)k_out; a.v_out = (uint16_t*)v_out; a.L = max_len;
  const dim3 grid((max_len + PAGED_TILE - 1) / PAGED_TILE, Hkv, B);
  if (kv_bits == 16) hipLaunchKernelGGL(read_kernel<16>, grid, dim3(256), 0, (hipStream_t)stream, a);
  else hipLaunchKernelGGL(read_kernel<4>, grid, dim3(256), 0, (hipStream_t)stream, a);
  return pbs_check_launch("pbs_paged_read");
}
