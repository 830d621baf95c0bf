// Attention over a paged cache in 8 bits for prompts behind a filled cache and drafted tokens: 128 query rows a workgroup.
//
// The mathematics and the row numbering are those of pbs_paged_attn.hip.  As in pbs_paged_rows.hip the waves share the keys and split the rows,
// 32 each, and tiles of 64 keys go through LDS: keys as they are, by asynchronous copies (8 KB, two buffers), values unpacked to bf16 on the
// way, once for all rows (16 KB, two buffers).
//
// A step has 512 cycles of the matrix unit for its logits (the queries are two e4m3 numbers a channel), 576 for its products, and about 1000 of
// the vector unit, half of them exponentials.  So the order is one where each stretch of matrix instructions has vector work beside it that
// does not wait for it, half a tile (32 keys) behind:
//    logits of a tile's second half     beside   weights of its first half
//    products of its first half         beside   maxima of its second half, the next tile's values into LDS
//    (barrier: the next tile is in LDS)
//    logits of the next's first half    beside   weights of the second half
//    products of the second half        beside   maxima of the next's first half
//
// 1000 new tokens behind 32k (32 / 8 heads) 487 us, 1.12 PFLOP/s (with the logits' two parts counted, 1.68), 500 of two sequences behind up to 16k
// 212.  By the counters the matrix unit works 51 % of the time and the vector unit 50 %, at 2.25 GHz: an 8-bit matrix instruction keeps the vector
// unit's issue for about 20 cycles and a bf16 one for 8, so what does run beside them is less than it looks.  With instructions of 32 rows the cycles
// are 3 % fewer and the clock 6 % lower (2.11 GHz): 533 us for 514 at that time.
#include "pbs_paged_attn.h"
#include <math.h>

namespace {

constexpr int WAVES = PAGED_WAVES, RW = 2;   // RW: 16-row tiles of a wave
constexpr int ROWS = WAVES * RW * 16;
constexpr int KEYS = 64;                     // of a step
constexpr int K_BYTES = KEYS * PAGED_D, V_BYTES = KEYS * PAGED_D * 2;
constexpr int LDS_V = 2 * K_BYTES, LDS_LATER = LDS_V + 2 * V_BYTES, LDS_SHARE = LDS_LATER + (int)sizeof(PagedLater);
constexpr int LDS_TOTAL = LDS_SHARE + (int)sizeof(PagedShareLds);

extern __shared__ __attribute__((aligned(16))) char lds[];

// K: rows 2 m and 2 m + 1 are sixteen chunks of 16 bytes, chunk j in place j ^ (m % 16): an operand's sixteen lanes read rows 2 n + half
__device__ __forceinline__ int k_place(int pair, int chunk) { return pair * 256 + ((chunk ^ (pair & 15)) * 16); }
// V: 16 bytes are eight tokens of a channel; place 64 e + m of a group of eight holds channel 2 m + e
__device__ __forceinline__ int channel_at(int place) { return (place & 63) * 2 + (place >> 6); }

// the tile of 64 keys after the one at hand.  A half of 32 keys whose page is not there is read as the pool's first tile of the head, and
// masked.  The page table is read a step ahead; steps behind the last load what is not used.
struct Next {
  int page0, page1;   // of the tile after it
  int held0, held1;   // of their 32 keys (0 and less: not there)
  u32x4 v[2];         // eight tokens of two channels each, of the half that the wave unpacks
  uint32_t ks[2], vs;

  // the pages of a step's two tiles (the keys, and so the first tile of a step that there is, end with the table)
  __device__ __forceinline__ void look_up(const HeadPool& p, int step) {
    const int32_t* row = (const int32_t*)p.row;
    page0 = row[min(step * 2 >> p.tiles_shift, p.last_slot)];
    page1 = row[min((step * 2 + 1) >> p.tiles_shift, p.last_slot)];
  }
  __device__ __forceinline__ void load(const HeadPool& p, int keys, int step, uint32_t k_to, const uint32_t (&k_from)[2], int wave) {
    const int left = keys - step * KEYS, in_page = (1 << p.tiles_shift) - 1;
    const int p0 = __builtin_amdgcn_readfirstlane(page0), p1 = __builtin_amdgcn_readfirstlane(page1);
    const bool there0 = (unsigned)p0 < (unsigned)p.num_pages, there1 = (unsigned)p1 < (unsigned)p.num_pages;
    const uint64_t at0 = (uint64_t)(uint32_t)(there0 ? p0 : 0) * p.page_tiles + (step * 2 & in_page);
    const uint64_t at1 = (uint64_t)(uint32_t)(there1 ? p1 : 0) * p.page_tiles + ((step * 2 + 1) & in_page);
    held0 = there0 ? min(left, PAGED_TILE) : 0;
    held1 = there1 ? min(left - PAGED_TILE, PAGED_TILE) : 0;
    const uint64_t at = wave < 2 ? at0 : at1, k = p.k + at * paged_tile_bytes<8>();
    const char* vp = (const char*)(p.v + at * paged_tile_bytes<8>());
#pragma unroll
    for (int i = 0; i < 2; ++i) copy_async(k, k_from[i], k_to + (uint32_t)(wave * 2048 + i * 1024));
    const uint32_t from = (threadIdx.x & 127) * 16;
    v[0] = *(const u32x4*)(vp + from);
    v[1] = *(const u32x4*)(vp + from + 2048);
    ks[0] = ((const uint8_t*)p.ks)[at0];
    ks[1] = ((const uint8_t*)p.ks)[at1];
    vs = ((const uint8_t*)p.vs)[at];
    look_up(p, step + 1);
  }
  // codes of tokens that are not there become zeros: they may be NaN, and the scale of a half without tokens anything
  __device__ __forceinline__ void hide(int wave) {
    if (held0 + held1 == KEYS) return;
    const int held = wave < 2 ? held0 : held1;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int there = held - (2 * i + (wave & 1)) * 8;
      const uint64_t mask = there >= 8 ? ~0ull : there <= 0 ? 0ull : ~0ull >> (64 - 8 * there);
#pragma unroll
      for (int w = 0; w < 4; ++w) v[i][w] &= (uint32_t)(mask >> (32 * (w & 1)));
    }
    vs = held > 0 ? vs : 127u;
  }
  __device__ __forceinline__ void store(char* to) const {
    const int m = threadIdx.x & 63, eight = (threadIdx.x >> 7) * 4 + ((threadIdx.x >> 6) & 1);
    const float scale = __uint_as_float(vs << 23);
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int e = 0; e < 2; ++e)
        *(u32x4*)(to + ((eight + 2 * i) * PAGED_D + e * 64 + m) * 16) =
            (u32x4){fp8_pair<0>(v[i][2 * e], scale), fp8_pair<1>(v[i][2 * e], scale), fp8_pair<0>(v[i][2 * e + 1], scale), fp8_pair<1>(v[i][2 * e + 1], scale)};
  }
};

__device__ __forceinline__ void fence() { __builtin_amdgcn_sched_barrier(0); }
// The order within a stretch: after each matrix instruction some of the vector unit's (2), of its exponentials (0x400) and reads from LDS (0x100).
// (Left to the compiler the matrix instructions end up behind the vector work: 501 us for 493; five vector instructions behind a product 493, three
// 489.)
__device__ __forceinline__ void beside_logits() {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    __builtin_amdgcn_sched_group_barrier(8, 1, 0);
    __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
    __builtin_amdgcn_sched_group_barrier(2, 3, 0);
    __builtin_amdgcn_sched_group_barrier(0x400, 2, 0);
  }
}
template <int VECTOR>
__device__ __forceinline__ void beside_products() {
#pragma unroll
  for (int i = 0; i < 18; ++i) {
    __builtin_amdgcn_sched_group_barrier(8, 1, 0);
    __builtin_amdgcn_sched_group_barrier(2, VECTOR, 0);
  }
}

__device__ __forceinline__ void work(const PagedAttnArgs& a, const PagedUnit& u, int head, int s0, int steps, float* part) {
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), n = lane & 15, g = lane >> 4;
  const float c = a.scale_log2;
  PagedLater& later = *(PagedLater*)(lds + LDS_LATER);
  const bool mixed = u.all_see < u.keys;   // (not with rows of one token)
  if (mixed) later.begin();
  Rows<8> q[RW];
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
  const int keys = u.keys, all_see = u.all_see;
  const int end = min(s0 + steps, (keys + KEYS - 1) / KEYS);
  bf16x8 ones;
#pragma unroll
  for (int j = 0; j < 8; ++j) ones[j] = (__bf16)1.f;
  // piece i of this wave's K: pairs of rows 8 wave + 4 i .. + 3; lane l fills place l % 16 of pair l / 16
  uint32_t k_from[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int pair = (8 * wave + 4 * i + (lane >> 4)) & 15;
    k_from[i] = (uint32_t)(pair * 256 + (((lane & 15) ^ pair) * 16));
  }

  int k_at = 0, v_at = LDS_V;             // the tile at hand
  int held[2] = {0, 0};
  uint32_t ks[2] = {0, 0};
  f32x4 s[RW][2][2];                      // logits: half, operand row m = token 2 m + its last index
  bf16x8 p[RW], kk[2][2], vv[8];
  Next next;

  auto read_k = [&](int half) __attribute__((always_inline)) {
    // operand row n is token 32 half + 2 n + i: a lane ends up with the logits of eight tokens in a row, 32 half + 8 g ..
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int e = 0; e < 2; ++e) kk[i][e] = *(const bf16x8*)(lds + k_at + k_place(16 * half + n, i * 8 + e * 4 + g));
  };
  auto read_v = [&](int half) __attribute__((always_inline)) {   // places 16 d + n of tokens 32 half + 8 g ..
#pragma unroll
    for (int d = 0; d < 8; ++d) vv[d] = *(const bf16x8*)(lds + v_at + ((4 * half + g) * PAGED_D + d * 16 + n) * 16);
  };
  auto multiply = [&](int half) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const u32x4 x = __builtin_bit_cast(u32x4, kk[i][0]), y = __builtin_bit_cast(u32x4, kk[i][1]);
      const i32x8 k = {(int)x[0], (int)x[1], (int)x[2], (int)x[3], (int)y[0], (int)y[1], (int)y[2], (int)y[3]};
#pragma unroll
      for (int r = 0; r < RW; ++r) s[r][half][i] = logits8(k, ks[half], q[r]);
    }
#pragma unroll
    for (int r = 0; r < RW; ++r) asm volatile("" : "+v"(s[r][half][0]), "+v"(s[r][half][1]));   // (here, and not behind the next branch)
  };
  auto weigh = [&](int half) __attribute__((always_inline)) {
    // bf16, as the matrix instruction takes them: half a step is 2^-8 of a weight, above the line and below it
#pragma unroll
    for (int r = 0; r < RW; ++r)
#pragma unroll
      for (int j = 0; j < 8; ++j) p[r][j] = (__bf16)__builtin_amdgcn_exp2f(__builtin_fmaf(s[r][half][j & 1][j >> 1], c, -m[r]));
#pragma unroll
    for (int r = 0; r < RW; ++r) asm volatile("" : "+v"(p[r]));   // (here, and not behind the next branch)
  };
  auto add = [&]() __attribute__((always_inline)) {
#pragma unroll
    for (int d = 0; d < 8; ++d)
#pragma unroll
      for (int r = 0; r < RW; ++r) o[r][d] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vv[d], p[r], o[r][d], 0, 0, 0);
#pragma unroll
    for (int r = 0; r < RW; ++r) l[r] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(ones, p[r], l[r], 0, 0, 0);
  };
  float top[RW];
  auto hide = [&](int step, int half) __attribute__((always_inline)) {
    const int first = step * KEYS + 32 * half;
    if (first + PAGED_TILE <= all_see && held[half] == PAGED_TILE) return;
#pragma unroll
    for (int r = 0; r < RW; ++r) {
      const int there = min(held[half], seen[r] - first) - 8 * g;
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (j >= there) s[r][half][j & 1][j >> 1] = -INFINITY;
    }
  };
  auto look = [&](int half) __attribute__((always_inline)) {   // whether a maximum grows
    bool grows = false;
#pragma unroll
    for (int r = 0; r < RW; ++r) {
      top[r] = s[r][half][0][0];
#pragma unroll
      for (int j = 1; j < 8; ++j) top[r] = fmaxf(top[r], s[r][half][j & 1][j >> 1]);
      grows |= __builtin_fmaf(top[r], c, a.room) > m[r];   // (this lane's keys; the row's are looked at where one of them is)
    }
    return grows;
  };
  auto grow = [&](bool grows) __attribute__((always_inline)) {
    if (!__any(grows)) return;
#pragma unroll
    for (int r = 0; r < RW; ++r) {
      const float most = max_over_groups(top[r]) * c;
      const float m_new = most + a.room > m[r] ? most + (a.room + PAGED_SLACK) : m[r], f = __builtin_amdgcn_exp2f(m[r] - m_new);   // (a row goes by its own keys)
      l[r] *= f;
#pragma unroll
      for (int d = 0; d < 8; ++d) o[r][d] *= f;
      m[r] = m_new;
    }
  };
  const HeadPool pool(a.pool, u.b, head);
  auto load = [&](int step) __attribute__((always_inline)) { next.load(pool, keys, step, (uint32_t)(k_at ^ K_BYTES), k_from, wave); };
  // The next tile has landed in LDS, and nobody reads the buffers after it any more.
  auto arrive = [&](int step) __attribute__((always_inline)) {
    __builtin_amdgcn_s_waitcnt(0x0f70);   // vmcnt(0): the copies
    asm volatile("" ::: "memory");
    __syncthreads();
    held[0] = next.held0, held[1] = next.held1;
    ks[0] = next.ks[0], ks[1] = next.ks[1];
    if (mixed && step * KEYS + KEYS > all_see) {   // values that are not finite and that some rows do not see
#pragma unroll 1
      for (int i = threadIdx.x; i < KEYS / 8 * PAGED_D; i += 256) {
        u32x4* at = (u32x4*)(lds + v_at) + i;
        u32x4 x = *at;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const uint32_t h = x[j >> 1] >> (16 * (j & 1)) & 0xffffu;
          if (!not_finite(h)) continue;
          later.note(channel_at(i % PAGED_D), step * KEYS + i / PAGED_D * 8 + j, h);
          x[j >> 1] &= j & 1 ? 0xffffu : 0xffff0000u;
        }
        *at = x;
      }
      __syncthreads();
    }
  };
  if (s0 < end) {
    next.look_up(pool, s0);
    k_at = K_BYTES;
    load(s0);
    k_at = 0;
    next.hide(wave);
    next.store(lds + v_at);
    arrive(s0);
    load(s0 + 1);
    read_k(0);
    multiply(0);
    hide(s0, 0);
    grow(look(0));
    read_k(1);
    int step = s0;
    // from a tile whose first half's maxima are known to the next such one
    while (step + 1 < end) {
      fence();
      read_v(0);
      multiply(1);
      weigh(0);
      beside_logits();
      fence();
      next.hide(wave);
      hide(step, 1);
      const int v_next = 2 * LDS_V + V_BYTES - v_at;
      fence();
      __builtin_amdgcn_s_setprio(1);   // (the wave that multiplies values goes before the one that weighs: 517 -> 501 us)
      next.store(lds + v_next);
      add();
      const bool grows = look(1);
      beside_products<3>();
      fence();
      __builtin_amdgcn_s_setprio(0);
      grow(grows);
      read_v(1);     // (the last of this tile)
      k_at ^= K_BYTES;
      v_at = v_next;
      ++step;
      arrive(step);
      read_k(0);
      fence();
      multiply(0);
      load(step + 1);
      weigh(1);
      beside_logits();
      fence();
      hide(step, 0);
      fence();
      __builtin_amdgcn_s_setprio(1);
      read_k(1);
      add();
      const bool grows_next = look(0);
      beside_products<1>();
      fence();
      __builtin_amdgcn_s_setprio(0);
      grow(grows_next);
    }
    read_v(0);
    multiply(1);
    weigh(0);
    add();
    hide(step, 1);
    grow(look(1));
    read_v(1);
    weigh(1);
    add();
  }

  __builtin_amdgcn_s_waitcnt(0x0f70);   // vmcnt(0): copies of a step behind the last
  __syncthreads();   // (the notes are whole, and the next piece's copies go over these buffers)
  const bool noted = mixed && later.is_any();
#pragma unroll
  for (int r = 0; r < RW; ++r) {
    const float sum = l[r][0];
    const int rr = (wave * RW + r) * 16 + n, row = u.r0 + rr, token = row / a.G;
    if (noted) {
#pragma unroll
      for (int d = 0; d < 8; ++d)
#pragma unroll
        for (int i = 0; i < 4; ++i) o[r][d][i] += later.of(channel_at(d * 16 + 4 * g + i), u.past + token + 1);
    }
    if (part) {
      if (token >= u.fresh) continue;   // (cleared by the join)
#pragma unroll
      for (int d = 0; d < 4; ++d)       // channels 32 d + 8 g ..
#pragma unroll
        for (int i = 0; i < 4; i += 2)
          *(f32x4*)(part + rr * PAGED_D + d * 32 + 8 * g + 2 * i) = (f32x4){o[r][d][i], o[r][d + 4][i], o[r][d][i + 1], o[r][d + 4][i + 1]};
      if (g == 0) *(f32x2*)(part + ROWS * PAGED_D + rr * 2) = (f32x2){m[r], sum};
    } else if (token < a.S) {
      const float scale = sum == 0.f || token >= u.fresh ? 0.f : 1.f / sum;   // (rows without a token weigh the keys that every row sees)
      uint16_t* dst = a.out + u.b * a.o_sb + (head * a.G + row % a.G) * a.o_sh + (int64_t)token * a.o_ss;
      auto two = [&](float x, float y) __attribute__((always_inline)) {
        return scale == 0.f ? 0u : __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2){x * scale, y * scale}, bf16x2));
      };
#pragma unroll
      for (int d = 0; d < 4; ++d)
        *(u32x4*)(dst + d * 32 + 8 * g) = (u32x4){two(o[r][d][0], o[r][d + 4][0]), two(o[r][d][1], o[r][d + 4][1]), two(o[r][d][2], o[r][d + 4][2]), two(o[r][d][3], o[r][d + 4][3])};
    }
  }
  __syncthreads();   // (the next piece clears the notes)
}

__global__ __launch_bounds__(256, 2) void attn_rows8_kernel(PagedAttnArgs a) {
  // Workers that follow each other read the same head's keys at the same time: they go to one of the eight dies and its L2 (workgroups
  // are dealt to them in turn).  Without cuts the heads follow each other, and the row tiles that see the most keys come first.
  const int worker = a.headers ? (int)((blockIdx.x & 7) * (gridDim.x >> 3) + (blockIdx.x >> 3)) : 0;
  paged_go<ROWS, KEYS, 0, WAVES>(a, *(PagedShareLds*)(lds + LDS_SHARE), worker, true, [&](const PagedUnit& u, int head, int step, int steps, float* part)
                       __attribute__((always_inline)) { work(a, u, head, step, steps, part); });
}

}  // namespace

int paged_attn_rows8(const PagedAttnArgs& a, hipStream_t stream) {
  const void* kernel = (const void*)attn_rows8_kernel;
  if (const int rc = pbs_require_no_static_lds(kernel, "pbs_paged_attn_fwd")) return rc;
  if (const hipError_t e = hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, LDS_TOTAL); e != hipSuccess) {
    pbs_set_error("pbs_paged_attn_fwd: hipFuncSetAttribute: %s", hipGetErrorString(e));
    return (int)e;
  }
  hipLaunchKernelGGL(attn_rows8_kernel, dim3(a.headers ? a.workers : a.Hkv * a.B * a.row_tiles), dim3(256), LDS_TOTAL, stream, a);
  return 0;
}
