// Attention over a paged cache for prompts behind a filled cache and drafted tokens: 64 or 128 query rows a workgroup.
//
// The mathematics and the row numbering are those of pbs_paged_attn.hip.  Here the waves share the keys and split the rows (16 or 32 each), so
// tiles of 64 keys go through LDS, two buffers: bf16 tiles are copied there asynchronously; values in 4 bits are loaded into registers during
// the tile before and unpacked to bf16 behind it, once for all rows, while keys in 4 bits need no unpacking and go to every wave's registers
// as they are.
//
// A wave's order within a step keeps both units busy: the logits of its second 32 keys beside the weights of the first, the products of the
// first beside the weights of the second.
//
// 500 new tokens of two sequences behind up to 16k (32 / 8 heads) 241 us, 870 TFLOP/s; 1000 behind 32k in 4 bits 582 us, 940 (without the order
// above 671, with the waits for the next tile's copies in front of each step's first product 700).  By the counters neither unit is full: in bf16
// the matrix unit works 49 % of the time and the vector unit 49 %, in 4 bits 43 and 55; two waves a SIMD with 32 rows each overlap them no
// further.
#include "pbs_paged_attn.h"
#include <math.h>

namespace {

constexpr int WAVES = PAGED_WAVES;
constexpr int KEYS = 64;                      // of a step
constexpr int lds_v(int bits) { return bits == 16 ? KEYS * PAGED_D * 2 : 0; }   // V, behind K, in a buffer
constexpr int lds_buffer(int bits) { return lds_v(bits) + KEYS * PAGED_D * 2; }
constexpr int lds_later(int bits) { return 2 * lds_buffer(bits); }
constexpr int lds_share(int bits) { return lds_later(bits) + (int)sizeof(PagedLater); }
constexpr int lds_total(int bits) { return lds_share(bits) + (int)sizeof(PagedShareLds); }

extern __shared__ __attribute__((aligned(16))) char lds[];

// bf16 K: rows of 256 bytes, the 16-byte chunk j of row r in place j ^ (r / 2 % 16): an operand's sixteen lanes read rows 2 n + half.
__device__ __forceinline__ int k_place(int row, int chunk) { return row * 256 + ((chunk ^ ((row >> 1) & 15)) * 16); }

// The next tile of 64 keys on its way into LDS.  A half of 32 keys whose page is not there is read as the pool's first tile, and masked.
template <int BITS>
struct Stage;
template <>
struct Stage<16> {
  uint32_t k_from[4];
  __device__ __forceinline__ void begin(int wave, int lane) {
    // piece i of this wave: rows 16 wave + 4 i .. + 3; lane l fills place l % 16 of row l / 16
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int row = 16 * wave + 4 * i + (lane >> 4);
      k_from[i] = (uint32_t)((row & 31) * 256 + (((lane & 15) ^ ((row >> 1) & 15)) * 16));
    }
  }
  __device__ __forceinline__ void load(const PagedPool& p, int64_t at0, int64_t at1, uint32_t buffer, int wave, int lane) {
    const int64_t at = wave < 2 ? at0 : at1;
    const uint64_t k = uniform64((uint64_t)p.k + at * paged_tile_bytes<16>()), v = uniform64((uint64_t)p.v + at * paged_tile_bytes<16>() + (wave & 1) * 4096);
#pragma unroll
    for (int i = 0; i < 4; ++i) copy_async(k, k_from[i], buffer + (uint32_t)(wave * 4096 + i * 1024));
#pragma unroll
    for (int i = 0; i < 4; ++i) copy_async(v, (uint32_t)(lane * 16 + i * 1024), buffer + (uint32_t)(lds_v(16) + wave * 4096 + i * 1024));
  }
  __device__ __forceinline__ void store(uint32_t buffer, int held0, int held1) {}   // (the copies are awaited by all waves before the barrier)
};
template <>
struct Stage<4> {
  u32x4 v[2];
  u32x2 vs;
  __device__ __forceinline__ void begin(int, int) {}
  __device__ __forceinline__ void load(const PagedPool& p, int64_t at0, int64_t at1, uint32_t, int, int) {
    const int m = threadIdx.x & 15, eight = (threadIdx.x >> 4) & 7;   // eight tokens of channels 8 m .. 8 m + 7, of which a thread unpacks four
    const int64_t at = eight < 4 ? at0 : at1;
    const char* src = p.v + at * paged_tile_bytes<4>() + (eight & 3) * 512 + m * 16;
    v[0] = *(const u32x4*)src;
    v[1] = *(const u32x4*)(src + 256);
    vs = *(const u32x2*)(p.vs + at * 128 + (m >> 2) * 32 + (eight & 3) * 8);
  }
  // `held`: tokens of either half that are there; scales of the others are 2^-127, as they may be NaN and codes are not
  __device__ __forceinline__ void store(uint32_t buffer, int held0, int held1) {
    const int m = threadIdx.x & 15, eight = (threadIdx.x >> 4) & 7, half = threadIdx.x >> 7;
    const int held = (eight < 4 ? held0 : held1) - (eight & 3) * 8;
    bf16x2 x[8][2];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const uint32_t e = j < held ? (vs[j >> 2] >> (8 * (j & 3))) & 0xffu : 0u;
      const uint32_t w = v[j >> 2][j & 3] >> (16 * half);
      x[j][0] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, __uint_as_float(e << 23), 0);
      x[j][1] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, __uint_as_float(e << 23), 1);
    }
    // place 16 d + m holds channel 8 m + d
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      u32x4 lo, hi;
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const uint32_t a = __builtin_bit_cast(uint32_t, x[2 * w][c]), b = __builtin_bit_cast(uint32_t, x[2 * w + 1][c]);
        lo[w] = __builtin_amdgcn_perm(b, a, 0x05040100u);
        hi[w] = __builtin_amdgcn_perm(b, a, 0x07060302u);
      }
      char* dst = lds + buffer + lds_v(4) + (eight * PAGED_D + (4 * half + 2 * c) * 16 + m) * 16;
      *(u32x4*)dst = lo;
      *(u32x4*)(dst + 256) = hi;
    }
  }
};

template <int BITS, int RW>   // RW: 16-row tiles of a wave
__device__ __forceinline__ void work(const PagedAttnArgs& a, const PagedUnit& u, int head, int s0, int steps, float* part) {
  constexpr int ROWS = WAVES * RW * 16;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), n = lane & 15, g = lane >> 4;
  const float c = a.scale_log2;
  PagedLater& later = *(PagedLater*)(lds + lds_later(BITS));
  const bool mixed = u.all_see < u.keys;   // (not with rows of one token)
  if (mixed) later.begin();
  Rows<BITS> q[RW];
  f32x4 o[RW][8];
  float m[RW];
  f32x4 l[RW];   // the weights' sums, as products with ones (every row of the tile the same): 32 bits, on the matrix unit, and no sum over lanes
  int seen[RW];
#pragma unroll
  for (int r = 0; r < RW; ++r) {
    const int row = u.r0 + (wave * RW + r) * 16 + n, token = row / a.G;
    const bool valid = token < u.fresh;
    q[r].load(valid ? a.q + u.b * a.q_sb + (head * a.G + row % a.G) * a.q_sh + (int64_t)token * a.q_ss : nullptr, g);
    seen[r] = valid ? u.past + token + 1 : 0;
    m[r] = -FLT_MAX;
    l[r] = (f32x4){};
#pragma unroll
    for (int d = 0; d < 8; ++d) o[r][d] = (f32x4){};
  }
  const int end = min(s0 + steps, (u.keys + KEYS - 1) / KEYS);
  bf16x8 ones;
#pragma unroll
  for (int j = 0; j < 8; ++j) ones[j] = (__bf16)1.f;
  Stage<BITS> stage;
  stage.begin(wave, lane);
  // tiles of a step: where they are, and how many of their 32 keys (0 where the page is not there)
  auto look_up = [&](int step, int64_t& at0, int64_t& at1, int& held0, int& held1) __attribute__((always_inline)) {
    const int left = u.keys - step * KEYS;
    at0 = paged_tile_index(a.pool, u.b, head, step * 2);
    at1 = left > PAGED_TILE ? paged_tile_index(a.pool, u.b, head, step * 2 + 1) : -1;
    held0 = at0 < 0 ? 0 : min(left, PAGED_TILE);
    held1 = at1 < 0 ? 0 : min(left - PAGED_TILE, PAGED_TILE);
    at0 = max(at0, (int64_t)0);
    at1 = max(at1, (int64_t)0);
  };
  int64_t at0, at1;
  int held0 = 0, held1 = 0, next0 = 0, next1 = 0;
  uint32_t buffer = 0;
  Tile<4> keys[2];   // (4 bits)
  if (s0 < end) {
    look_up(s0, at0, at1, held0, held1);
    stage.load(a.pool, at0, at1, buffer, wave, lane);
    if (BITS == 4) {
      load_k(keys[0], a.pool, at0, n, g);
      load_k(keys[1], a.pool, at1, n, g);
    }
    stage.store(buffer, held0, held1);
  }
  for (int step = s0; step < end; ++step) {
    // this tile's copies have landed, and nobody reads the other buffer any more.  (By the builtin: the compiler sees that the queries have
    // landed too, and does not wait for them behind the next copies, which it does not count.)
    if (BITS == 16) __builtin_amdgcn_s_waitcnt(0x0f70);   // vmcnt(0)
    asm volatile("" ::: "memory");
    __syncthreads();
    if (step + 1 < end) {
      look_up(step + 1, at0, at1, next0, next1);
      stage.load(a.pool, at0, at1, buffer ^ lds_buffer(BITS), wave, lane);
    }
    if (BITS == 16 && held0 + held1 < KEYS) {
      // tokens that are not there hold whatever the page held before: not even times zero
      for (int i = threadIdx.x; i < KEYS / 8 * PAGED_D; i += 256) {
        const int held = (i < 4 * PAGED_D ? held0 : held1) - (i / PAGED_D & 3) * 8;
        u32x4* x = (u32x4*)(lds + buffer + lds_v(BITS)) + i;
        if (held < 8) {
#pragma unroll
          for (int w = 0; w < 4; ++w) (*x)[w] &= held >= 2 * w + 2 ? 0xffffffffu : held == 2 * w + 1 ? 0xffffu : 0u;
        }
      }
      __syncthreads();
    }
    const int k0 = step * KEYS;
    if (mixed && k0 + KEYS > u.all_see) {
#pragma unroll 1
      for (int i = threadIdx.x; i < KEYS / 8 * PAGED_D; i += 256) {
        u32x4* at = (u32x4*)(lds + buffer + lds_v(BITS)) + i;
        const int place = i % PAGED_D, key = k0 + i / PAGED_D * 8;
        u32x4 x = *at;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const uint32_t h = x[j >> 1] >> (16 * (j & 1)) & 0xffffu;
          if (!not_finite(h)) continue;
          later.note(BITS == 16 ? place : (place & 15) * 8 + (place >> 4), key + j, h);
          x[j >> 1] &= j & 1 ? 0xffffu : 0xffff0000u;
        }
        *at = x;
      }
      __syncthreads();
    }
    const char* kt = lds + buffer;
    const char* vt = lds + buffer + lds_v(BITS);
    // Operands are read from LDS two groups of four ahead of the products that take them; the fences keep the compiler from sinking the reads.
    f32x4 s[RW][2][2];
    bf16x8 k[3][4], v[3][4], p[RW][2];
    auto fence = [] __attribute__((always_inline)) { __builtin_amdgcn_sched_barrier(0); };
    auto read_k = [&](int i) __attribute__((always_inline)) {
      // operand row n is token 32 (i / 2) + 2 n + i % 2: a lane ends up with the logits of eight tokens in a row, 32 (i / 2) + 8 g ..
      if (BITS == 16) {
#pragma unroll
        for (int e = 0; e < 4; ++e) k[i % 3][e] = *(const bf16x8*)(kt + k_place(32 * (i >> 1) + 2 * n + (i & 1), e * 4 + g));
      }
    };
    auto read_v = [&](int i) __attribute__((always_inline)) {   // channels 16 d + n, d = 4 (i % 2) .., of tokens 32 (i / 2) + 8 g ..
#pragma unroll
      for (int e = 0; e < 4; ++e) v[i % 3][e] = *(const bf16x8*)(vt + ((4 * (i >> 1) + g) * PAGED_D + (4 * (i & 1) + e) * 16 + n) * 16);
    };
    auto multiply = [&](int i) __attribute__((always_inline)) {
      if constexpr (BITS == 16) {
#pragma unroll
        for (int r = 0; r < RW; ++r) s[r][i >> 1][i & 1] = (f32x4){};
#pragma unroll
        for (int e = 0; e < 4; ++e)
#pragma unroll
          for (int r = 0; r < RW; ++r) s[r][i >> 1][i & 1] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(k[i % 3][e], q[r].q[e], s[r][i >> 1][i & 1], 0, 0, 0);
      } else {
#pragma unroll
        for (int r = 0; r < RW; ++r) s[r][i >> 1][i & 1] = logits(keys[i >> 1], i & 1, q[r]);
      }
    };
    auto weigh = [&](int r, int i) __attribute__((always_inline)) {
      // bf16, as the matrix instruction takes them: half a step is 2^-8 of a weight, above the line and below it
#pragma unroll
      for (int j = 0; j < 8; ++j) p[r][i][j] = (__bf16)__builtin_amdgcn_exp2f(__builtin_fmaf(s[r][i][j & 1][j >> 1], c, -m[r]));
    };
    // 32 keys' masks and maxima.  Where the second 32's grow, the weights of the first, which have not been multiplied yet, are taken again.
    auto look = [&](int i) __attribute__((always_inline)) {
      const int held = i ? held1 : held0, first = k0 + 32 * i;
      if (first + PAGED_TILE > u.all_see || held < PAGED_TILE) {
#pragma unroll
        for (int r = 0; r < RW; ++r) {
          const int there = min(held, seen[r] - first) - 8 * g;
#pragma unroll
          for (int j = 0; j < 8; ++j)
            if (j >= there) s[r][i][j & 1][j >> 1] = -INFINITY;
        }
      }
      float top[RW];
      bool grows = false;
#pragma unroll
      for (int r = 0; r < RW; ++r) {
        top[r] = s[r][i][0][0];
#pragma unroll
        for (int j = 1; j < 8; ++j) top[r] = fmaxf(top[r], s[r][i][j & 1][j >> 1]);
        grows |= __builtin_fmaf(top[r], c, a.room) > m[r];   // (this lane's keys; the row's are looked at where one of them is)
      }
      if (__any(grows)) {
#pragma unroll
        for (int r = 0; r < RW; ++r) {
          const float most = max_over_groups(top[r]) * c;
          const float m_new = most + a.room > m[r] ? most + (a.room + PAGED_SLACK) : m[r], f = __builtin_amdgcn_exp2f(m[r] - m_new);   // (a row goes by its own keys)
          l[r] *= f;
#pragma unroll
          for (int d = 0; d < 8; ++d) o[r][d] *= f;
          m[r] = m_new;
          if (i == 1) weigh(r, 0);
        }
      }
    };
    read_k(0);
    read_k(1);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      fence();
      read_k(i + 2);
      multiply(i);
    }
    fence();
    look(0);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      fence();
      read_v(i);
      multiply(i + 2);
      if (i < RW) {
        weigh(i, 0);
        asm volatile("" : "+v"(p[i][0]));   // (here, and not behind the branch that may take them again)
      }
    }
    fence();
    if (BITS == 4 && step + 1 < end) {
      load_k(keys[0], a.pool, at0, n, g);
      load_k(keys[1], a.pool, at1, n, g);
    }
    look(1);
    // (the wave that multiplies goes before the one that weighs: 246 -> 239 us, in 4 bits 595 -> 580; ahead of the logits' products too 242 and 588)
    __builtin_amdgcn_s_setprio(1);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      fence();
      if (i < 2) read_v(i + 2);
#pragma unroll
      for (int e = 0; e < 4; ++e)
#pragma unroll
        for (int r = 0; r < RW; ++r)
          o[r][4 * (i & 1) + e] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(v[i % 3][e], p[r][i >> 1], o[r][4 * (i & 1) + e], 0, 0, 0);
      if (i < RW) weigh(i, 1);
      if (i & 1) {
#pragma unroll
        for (int r = 0; r < RW; ++r) l[r] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(ones, p[r][i >> 1], l[r], 0, 0, 0);
      }
    }
    __builtin_amdgcn_s_setprio(0);
    fence();
    held0 = next0;
    held1 = next1;
    buffer ^= lds_buffer(BITS);
    if (step + 1 < end) stage.store(buffer, held0, held1);
  }

  const bool noted = mixed && later.is_any();   // (a step's barrier is behind its notes)
#pragma unroll
  for (int r = 0; r < RW; ++r) {
    const float sum = l[r][0];
    const int rr = (wave * RW + r) * 16 + n, row = u.r0 + rr, token = row / a.G;
    if (noted) {
#pragma unroll
      for (int d = 0; d < 8; ++d)
#pragma unroll
        for (int i = 0; i < 4; ++i) o[r][d][i] += later.of(BITS == 16 ? d * 16 + 4 * g + i : (4 * g + i) * 8 + d, u.past + token + 1);
    }
    if (part) {
      if (token >= u.fresh) continue;   // (cleared by the join)
#pragma unroll
      for (int d = 0; d < 8; ++d)
#pragma unroll
        for (int i = 0; i < 4; ++i) part[rr * PAGED_D + (BITS == 16 ? d * 16 + 4 * g + i : (4 * g + i) * 8 + d)] = o[r][d][i];
      if (g == 0) *(f32x2*)(part + ROWS * PAGED_D + rr * 2) = (f32x2){m[r], sum};
    } else if (token < a.S) {
      const float scale = sum == 0.f || token >= u.fresh ? 0.f : 1.f / sum;   // (rows without a token weigh the keys that every row sees)
      uint16_t* dst = a.out + u.b * a.o_sb + (head * a.G + row % a.G) * a.o_sh + (int64_t)token * a.o_ss;
      auto two = [&](float x, float y) __attribute__((always_inline)) {
        return scale == 0.f ? 0u : __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2){x * scale, y * scale}, bf16x2));
      };
      if (BITS == 16) {
#pragma unroll
        for (int d = 0; d < 8; ++d) *(u32x2*)(dst + d * 16 + 4 * g) = (u32x2){two(o[r][d][0], o[r][d][1]), two(o[r][d][2], o[r][d][3])};
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
          *(u32x4*)(dst + (4 * g + i) * 8) = (u32x4){two(o[r][0][i], o[r][1][i]), two(o[r][2][i], o[r][3][i]), two(o[r][4][i], o[r][5][i]), two(o[r][6][i], o[r][7][i])};
      }
    }
  }
  __syncthreads();   // (the next piece's copies go over these buffers)
}

template <int BITS, int RW>
__global__ __launch_bounds__(256, 2) void attn_rows_kernel(PagedAttnArgs a) {
  // Workers that follow each other read the same head's keys at the same time: they go to one of the eight dies and its L2 (workgroups
  // are dealt to them in turn).  Without cuts the heads follow each other, and the row tiles that see the most keys come first.
  const int worker = a.headers ? (int)((blockIdx.x & 7) * (gridDim.x >> 3) + (blockIdx.x >> 3)) : 0;
  paged_go<WAVES * RW * 16, KEYS, 0, WAVES>(a, *(PagedShareLds*)(lds + lds_share(BITS)), worker, true,
                                  [&](const PagedUnit& u, int head, int step, int steps, float* part)
                                  __attribute__((always_inline)) { work<BITS, RW>(a, u, head, step, steps, part); });
}

template <int BITS, int RW>
int launch(const PagedAttnArgs& a, hipStream_t stream) {
  const void* kernel = (const void*)attn_rows_kernel<BITS, RW>;
  if (const int rc = pbs_require_no_static_lds(kernel, "pbs_paged_attn_fwd")) return rc;
  if (const hipError_t e = hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, lds_total(BITS)); e != hipSuccess) {
    pbs_set_error("pbs_paged_attn_fwd: hipFuncSetAttribute: %s", hipGetErrorString(e));
    return (int)e;
  }
  hipLaunchKernelGGL((attn_rows_kernel<BITS, RW>), dim3(a.headers ? a.workers : a.Hkv * a.B * a.row_tiles), dim3(256), lds_total(BITS), stream, a);
  return 0;
}

}  // namespace

int paged_attn_rows(const PagedAttnArgs& a, int kv_bits, int rows, hipStream_t stream) {
  if (kv_bits == 16) return rows == 64 ? launch<16, 1>(a, stream) : launch<16, 2>(a, stream);
  return kv_bits == 8 ? paged_attn_rows8(a, stream) : launch<4, 2>(a, stream);
}
