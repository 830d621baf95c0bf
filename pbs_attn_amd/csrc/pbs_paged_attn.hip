// Attention of a batch's new tokens over a paged cache (the tokens themselves are in it already).
//
// For query i of a sequence with `past` tokens before the call: o = sum_j p_j v_j / sum_j p_j, p_j = exp(scale q k_j - m), over the keys
// j <= past + i, m the largest exponent so far (one pass: sums are rescaled where it grows).  All query heads of a KV head and several
// tokens share a tile's rows, row r = (token r / G, head r % G of the group), so a key is read once for all of them.
//
// Here: up to 32 rows of a bf16 cache, up to 64 of an 8- or 4-bit one; pbs_paged_rows.hip and pbs_paged_rows8.hip take more.  Bound by memory, so
// the waves of a workgroup split the keys and each holds all rows: tiles go from memory into registers in the matrix instruction's operand order
// and nothing is shared but the sums at the end.  Sequences of any lengths are cut into 512 equal shares (two workgroups a compute unit; 768 and
// more are slower: more parts; in 8 bits, where few long sequences have one row tile, 256 by workgroups of eight waves), and a second launch joins
// what was cut.  32 / 8 heads behind 128k tokens in bf16 103 us (5.2 TB/s; uncut 2721), 64 sequences of 17 .. 8191 tokens 109 us (5.1), 128 of
// 100 .. 16383 in 4 bits 228 us (5.0).  35 rows in 4 bits are not (60 us, 2.3 TB/s): waves wait for 44 % of their time, one step of loads ahead,
// while the vector unit works 46 % and the matrix unit 28 %.  (Four row tiles in 4 bits, 49 .. 64 rows: 13 registers of a wave go to scratch
// memory, 20 with eight waves.)  In 8 bits 128k tokens take 57 us (5.2 TB/s in this launch, then a join of 5 us; reading as much and nothing else
// 44.5), 128 sequences 366 (5.8), 35 rows of 16 sequences 64 (4.4); 49 .. 64 rows of those 83, with 9 registers of a wave in scratch memory ahead
// of the steps and behind them, none in a step.
#include "pbs_paged_attn.h"
#include "../../include/pbs_hip.h"   // the definitions below are checked against the public declarations
#include <math.h>
#include <algorithm>
#include <type_traits>

namespace {

constexpr int O_PITCH = PAGED_D + 4;

// V^T operands: d's holds eight tokens (8 g ..) of channel 16 d + n, of 8-bit pages of channel 32 (d / 2) + 2 n + d % 2, of 4-bit pages of channel
// 8 n + d; here d = 2 c and 2 c + 1.  `held` of the eight are there.
template <bool TAIL>
__device__ __forceinline__ void values(const Tile<16>& t, int c, int held, bf16x8 (&v)[2]) {
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    u32x4 x = t.v[2 * c + e];
    if (TAIL) {
#pragma unroll
      for (int w = 0; w < 4; ++w) x[w] &= held >= 2 * w + 2 ? 0xffffffffu : held == 2 * w + 1 ? 0xffffu : 0u;
    }
    v[e] = __builtin_bit_cast(bf16x8, x);
  }
}
template <bool TAIL>
__device__ __forceinline__ void values(const Tile<8>& t, int c, int held, bf16x8 (&v)[2]) {
  u32x4 x = t.v[c];
  float scale = __uint_as_float(t.vs << 23);
  if (TAIL) {   // (a tile without tokens has no scale either)
    const uint64_t there = held >= 8 ? ~0ull : held <= 0 ? 0ull : ~0ull >> (64 - 8 * held);
#pragma unroll
    for (int w = 0; w < 4; ++w) x[w] &= (uint32_t)(there >> (32 * (w & 1)));
    scale = held > 0 ? scale : 1.f;
  }
#pragma unroll
  for (int e = 0; e < 2; ++e)
    v[e] = __builtin_bit_cast(bf16x8, (u32x4){fp8_pair<0>(x[2 * e], scale), fp8_pair<1>(x[2 * e], scale), fp8_pair<0>(x[2 * e + 1], scale), fp8_pair<1>(x[2 * e + 1], scale)});
}
template <int C>
__device__ __forceinline__ uint32_t value_pair(uint32_t codes, uint32_t e) {   // channels 2 C and 2 C + 1 of a word
  return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, __uint_as_float(e), C));
}
template <bool TAIL>
__device__ __forceinline__ void values(const Tile<4>& t, int c, int held, bf16x8 (&v)[2]) {
  uint32_t x[8];   // token j: two channels
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    uint32_t e = (t.vs[j >> 2] >> (8 * (j & 3))) & 0xffu;
    if (TAIL) e = j < held ? e : 0u;   // (codes are finite whatever the page held before)
    const uint32_t w = t.v[j >> 2][j & 3];
    x[j] = c == 0 ? value_pair<0>(w, e << 23) : c == 1 ? value_pair<1>(w, e << 23) : c == 2 ? value_pair<2>(w, e << 23) : value_pair<3>(w, e << 23);
  }
  u32x4 lo, hi;
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    lo[w] = __builtin_amdgcn_perm(x[2 * w + 1], x[2 * w], 0x05040100u);
    hi[w] = __builtin_amdgcn_perm(x[2 * w + 1], x[2 * w], 0x07060302u);
  }
  v[0] = __builtin_bit_cast(bf16x8, lo);
  v[1] = __builtin_bit_cast(bf16x8, hi);
}
// infinities and NaN among the values of a lane's first `held` tokens, of which the first is `key`: noted, and out of the tile
__device__ __forceinline__ void set_aside(Tile<16>& t, PagedLater& later, int key, int held, int n) {
#pragma unroll
  for (int d = 0; d < 8; ++d) {
    u32x4 x = t.v[d];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const uint32_t h = x[j >> 1] >> (16 * (j & 1)) & 0xffffu;
      if (!not_finite(h)) continue;
      if (j < held) later.note(d * 16 + n, key + j, h);
      x[j >> 1] &= j & 1 ? 0xffffu : 0xffff0000u;
    }
    t.v[d] = x;
  }
}
__device__ __forceinline__ void set_aside(Tile<8>& t, PagedLater& later, int key, int held, int n) {
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    u32x4 x = t.v[c];
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      if (!fp8_is_nan(x[j >> 2] >> (8 * (j & 3)))) continue;
      if ((j & 7) < held) later.note(c * 32 + n * 2 + (j >> 3), key + (j & 7), 0x7fffu);
      x[j >> 2] &= ~(0xffu << (8 * (j & 3)));
    }
    t.v[c] = x;
  }
}
__device__ __forceinline__ void set_aside(Tile<4>& t, PagedLater& later, int key, int held, int n) {   // (a token's group is NaN or finite)
  u32x2 x = t.vs;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    if ((x[j >> 2] >> (8 * (j & 3)) & 0xffu) != 0xffu) continue;
    if (j < held)
      for (int d = 0; d < 8; ++d) later.note(n * 8 + d, key + j, 0x7fffu);
    x[j >> 2] &= ~(0xffu << (8 * (j & 3)));
  }
  t.vs = x;
}
template <int BITS>
__device__ __forceinline__ int channel_of(int d, int row) { return BITS == 16 ? d * 16 + row : BITS == 8 ? (d >> 1) * 32 + row * 2 + (d & 1) : row * 8 + d; }

// One wave's running softmax over its tiles.  S^T = K Q^T leaves a lane with the logits of tokens 8 g .. 8 g + 7 for query row n, which are
// its share of P^T in O^T += V^T P^T: probabilities never change lanes.
template <int BITS, int R, int NT>
struct Softmax {
  // The queries stay in registers where a wave has one row tile, and in LDS otherwise: 16 registers each (bf16, 35 rows: 256 and 138 spilled)
  Rows<BITS> own;
  RowsLds* lds;
  f32x4 o[R][8];
  float m[R];
  // The weights' sums, in 32 bits: as products with ones on the matrix unit (every row of the tile the same, and no sum over lanes), 8 bits of the
  // lane's own tokens by the vector unit, two at a time: three registers a row tile less (56 rows of 16 sequences 104 -> 93 us; with fewer row
  // tiles the same).
  static constexpr bool LANE_SUMS = BITS == 8;
  typename std::conditional<LANE_SUMS, float, f32x4>::type l[R];
  int seen[R];

  __device__ __forceinline__ void begin(const PagedAttnArgs& a, const PagedUnit& u, int head, int n, int g, int wave, RowsLds* q_lds) {
    lds = q_lds;
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int row = u.r0 + r * 16 + n, token = row / a.G;
      const bool valid = token < u.fresh;
      if (R == 1 || wave == r) {
        own.load(valid ? a.q + u.b * a.q_sb + (head * a.G + row % a.G) * a.q_sh + (int64_t)token * a.q_ss : nullptr, g);
        if (R > 1) own.put(lds[r], g * 16 + n);
      }
      seen[r] = valid ? u.past + token + 1 : 0;
      m[r] = -FLT_MAX;
      l[r] = {};
#pragma unroll
      for (int d = 0; d < 8; ++d) o[r][d] = (f32x4){};
    }
    if (R > 1) __syncthreads();
  }
  // logits of the NT tiles; `k0`: the first one's first key, `keys`: how many there are, bit i of `gone`: tile i's page is not there
  template <bool MASK>
  __device__ __forceinline__ void weigh(const Tile<BITS> (&t)[NT], bf16x8 (&p)[R][NT], int k0, int keys, uint32_t gone, float c, float room, int n, int g) {
    if (R > 1) asm volatile("" ::: "memory");   // (or all queries are read ahead of the loop, into registers)
    // (all row tiles' products first, then one decision: nothing waits for a row tile's maximum)
    float x[R][NT][8], top[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      if (R > 1) own.get(lds[r], g * 16 + n);
#pragma unroll
      for (int i = 0; i < NT; ++i) {
        const f32x4 s0 = logits(t[i], 0, own), s1 = logits(t[i], 1, own);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          x[r][i][j] = (j & 1) ? s1[j >> 1] : s0[j >> 1];
          if (MASK) {
            const int key = k0 + i * PAGED_TILE + 8 * g + j;
            x[r][i][j] = key < min(seen[r], keys) && !(gone >> i & 1) ? x[r][i][j] : -INFINITY;
          }
        }
      }
    }
    bool grows = false;
#pragma unroll
    for (int r = 0; r < R; ++r) {
      top[r] = x[r][0][0];
#pragma unroll
      for (int i = 0; i < NT; ++i)
#pragma unroll
        for (int j = 0; j < 8; ++j) top[r] = fmaxf(top[r], x[r][i][j]);
      grows |= __builtin_fmaf(top[r], c, room) > m[r];   // (this lane's keys; the row's are looked at where one of them is)
    }
    if (__any(grows)) {
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const float most = max_over_groups(top[r]) * c;
        const float m_new = most + room > m[r] ? most + (room + PAGED_SLACK) : m[r], f = __builtin_amdgcn_exp2f(m[r] - m_new);   // (a row goes by its own keys)
        l[r] *= f;
#pragma unroll
        for (int d = 0; d < 8; ++d) o[r][d] *= f;
        m[r] = m_new;
      }
    }
    bf16x8 ones;
#pragma unroll
    for (int j = 0; j < 8; ++j) ones[j] = (__bf16)1.f;
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int i = 0; i < NT; ++i) {
        // bf16, as the matrix instruction takes them: half a step is 2^-8 of a weight, above the line and below it
#pragma unroll
        for (int j = 0; j < 8; ++j) p[r][i][j] = (__bf16)__builtin_amdgcn_exp2f(__builtin_fmaf(x[r][i][j], c, -m[r]));
        if constexpr (LANE_SUMS) {
          const u32x4 w = __builtin_bit_cast(u32x4, p[r][i]);
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const uint32_t two = w[j];
            l[r] = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2, two), (bf16x2){(__bf16)1.f, (__bf16)1.f}, l[r], false);
          }
        } else {
          l[r] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(ones, p[r][i], l[r], 0, 0, 0);
        }
      }
  }
  __device__ __forceinline__ float sum(int r) const {
    if constexpr (LANE_SUMS) {
      TwoOf t = with_lane_xor<16>(__float_as_uint(l[r]));
      const float two = __uint_as_float(t.a) + __uint_as_float(t.b);
      t = with_lane_xor<32>(__float_as_uint(two));
      return __uint_as_float(t.a) + __uint_as_float(t.b);
    } else {
      return l[r][0];
    }
  }
  template <bool TAIL>
  __device__ __forceinline__ void add(const Tile<BITS> (&t)[NT], const bf16x8 (&p)[R][NT], int k0, int keys, uint32_t gone, int g) {
#pragma unroll
    for (int i = 0; i < NT; ++i) {
      // tokens behind the keys hold whatever the page held before: not even times zero
      const int held = gone >> i & 1 ? 0 : keys - k0 - i * PAGED_TILE - 8 * g;
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        bf16x8 v[2];
        values<TAIL>(t[i], c, held, v);
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
          for (int e = 0; e < 2; ++e) o[r][2 * c + e] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(v[e], p[r][i], o[r][2 * c + e], 0, 0, 0);
      }
    }
  }
};

// Steps `s0` .. `s0 + steps - 1` of a unit and head, WAVES * NT tiles a step, NT a wave; then the waves' sums together in LDS, and out, or as a part.
template <int BITS, int R, int NT, int DEPTH, int WAVES>
__device__ __forceinline__ void work(const PagedAttnArgs& a, const PagedUnit& u, int head, int s0, int steps, float* part,
                                     float (&o_lds)[WAVES][16][O_PITCH], float (&ml_lds)[WAVES][16][2], RowsLds* q_lds, PagedLater& later) {
  const int lane = paged_lane(), wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), n = lane & 15, g = lane >> 4;
  const bool mixed = u.all_see < u.keys;   // (never with a single token)
  if (mixed) later.begin();
  Softmax<BITS, R, NT> s;
  s.begin(a, u, head, n, g, wave, q_lds);
  const int tiles = (u.keys + PAGED_TILE - 1) / PAGED_TILE;
  int t = (s0 * WAVES + wave) * NT;                             // this wave's first tile of the step
  const int end = min((s0 + steps) * WAVES * NT, tiles);
  // Loads go out DEPTH steps ahead, a step's K as soon as the K before it in the same registers has been multiplied, its V likewise.  Pages are
  // looked up before that; a tile that is not there is read as the pool's first one, and not used.
  constexpr int STRIDE = WAVES * NT;
  Tile<BITS> tile[DEPTH][NT];
  uint32_t gone[DEPTH] = {};
  int64_t at[NT];
  int step = 0;
  Places<BITS, NT> places(a, u.b, head, STRIDE, tiles);
  if (t < end) {
#pragma unroll
    for (int d = 0; d < DEPTH; ++d) {
      if (t + d * STRIDE >= end) break;
      gone[d] = places.look_up(d, t + d * STRIDE, at);
#pragma unroll
      for (int i = 0; i < NT; ++i) load_k(tile[d][i], places.pool(), at[i], n, g);
#pragma unroll
      for (int i = 0; i < NT; ++i) load_v(tile[d][i], places.pool(), at[i], n, g);
    }
  }
  auto one = [&](auto mask, Tile<BITS> (&tile)[NT], uint32_t& gone) __attribute__((always_inline)) {
    const int next = t + DEPTH * STRIDE, k0 = t * PAGED_TILE;
    // (the older of a compute unit's two workgroups would finish a third earlier and leave the memory half idle: its waves go first in every other
    // step only.  8 bits: 128k tokens of one sequence 58.6 -> 57.3 us, 128 sequences 374 -> 365; a workgroup of eight waves is alone: no difference)
    if (BITS == 8 && R == 1 && WAVES == 4) {
      if ((blockIdx.x >= gridDim.x / 2) == (step & 1)) __builtin_amdgcn_s_setprio(0);
      else __builtin_amdgcn_s_setprio(2);
    }
    // (with several row tiles the loads behind the last step repeat its own: without the branches 35 rows take 68 us for 73; with one row
    // tile the steps are short, and the wait for what nobody uses costs 2 %)
    const bool load = R > 1 || next < end;
    uint32_t gone_next = 0;
    if (load) gone_next = places.look_up(R == 1 || next < end ? step + DEPTH : step, R == 1 || next < end ? next : t, at);
    bf16x8 p[R][NT];
    s.template weigh<mask.value>(tile, p, k0, u.keys, gone, a.scale_log2, a.room, n, g);
    if (load) {
#pragma unroll
      for (int i = 0; i < NT; ++i) load_k(tile[i], places.pool(), at[i], n, g);
    }
    if (mask.value && mixed && k0 + NT * PAGED_TILE > u.all_see) {
#pragma unroll
      for (int i = 0; i < NT; ++i) {
        const int key = k0 + i * PAGED_TILE + 8 * g;
        set_aside(tile[i], later, key, gone >> i & 1 ? 0 : u.keys - key, n);
      }
    }
    __builtin_amdgcn_sched_barrier(0);   // (or the loads sink behind the products: 35 rows 61.2 -> 59.7 us)
    s.template add<mask.value>(tile, p, k0, u.keys, gone, g);
    if (load) {
#pragma unroll
      for (int i = 0; i < NT; ++i) load_v(tile[i], places.pool(), at[i], n, g);
    }
    gone = gone_next;
    t += STRIDE;
    ++step;
  };
  // (tiles that every row sees whole, then the rest: those at the end, and whatever follows a page that is not there)
  const int seen_whole = min(u.all_see, u.keys) / PAGED_TILE - NT;
  auto loop = [&](auto mask) __attribute__((always_inline)) {
    while (t < end) {
      if (!mask.value && (t > seen_whole || gone[0] != 0)) break;
      one(mask, tile[0], gone[0]);
      if (DEPTH == 2) {
        if (t < end && (mask.value || (t <= seen_whole && gone[DEPTH - 1] == 0))) {
          one(mask, tile[DEPTH - 1], gone[DEPTH - 1]);
        } else {   // the buffers change places
#pragma unroll
          for (int i = 0; i < NT; ++i) {
            const Tile<BITS> x = tile[0][i];
            tile[0][i] = tile[DEPTH - 1][i];
            tile[DEPTH - 1][i] = x;
          }
          const uint32_t y = gone[0];
          gone[0] = gone[DEPTH - 1];
          gone[DEPTH - 1] = y;
          break;
        }
      }
    }
  };
  loop(std::false_type{});
  loop(std::true_type{});

  const int lane2 = paged_lane(), n2 = lane2 & 15, g2 = lane2 >> 4;
  bool noted = false;
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const float l = s.sum(r);
    if (r > 0) __syncthreads();   // (the rows before have been read)
    if (g2 == 0) {
      ml_lds[wave][n2][0] = s.m[r];
      ml_lds[wave][n2][1] = l;
    }
    __syncthreads();
    float top = ml_lds[0][n2][0];
#pragma unroll
    for (int w = 1; w < WAVES; ++w) top = fmaxf(top, ml_lds[w][n2][0]);
    const float f = __builtin_amdgcn_exp2f(s.m[r] - top);
    if constexpr (BITS == 8) {   // (a lane's channels lie in eights)
#pragma unroll
      for (int d = 0; d < 8; d += 2)
#pragma unroll
        for (int i = 0; i < 4; i += 2)
          *(f32x4*)&o_lds[wave][n2][channel_of<8>(d, 4 * g2 + i)] =
              (f32x4){s.o[r][d][i] * f, s.o[r][d + 1][i] * f, s.o[r][d][i + 1] * f, s.o[r][d + 1][i + 1] * f};
    } else {
#pragma unroll
      for (int d = 0; d < 8; ++d)
#pragma unroll
        for (int i = 0; i < 4; ++i) o_lds[wave][n2][channel_of<BITS>(d, 4 * g2 + i)] = s.o[r][d][i] * f;
    }
    __syncthreads();
    if (r == 0) noted = mixed && later.is_any();
    // 16 lanes a row, 8 channels a lane
    const int rr = wave * 4 + g2, c = n2 * 8, row = u.r0 + r * 16 + rr, token = row / a.G;
    if (WAVES > 4 && wave >= 4) continue;
    float y[8], row_top = ml_lds[0][rr][0], sum = 0.f;
#pragma unroll
    for (int w = 1; w < WAVES; ++w) row_top = fmaxf(row_top, ml_lds[w][rr][0]);
#pragma unroll
    for (int w = 0; w < WAVES; ++w) sum += ml_lds[w][rr][1] * __builtin_amdgcn_exp2f(ml_lds[w][rr][0] - row_top);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      y[e] = 0.f;
#pragma unroll
      for (int w = 0; w < WAVES; ++w) y[e] += o_lds[w][rr][c + e];
    }
    if (noted) {
#pragma unroll
      for (int e = 0; e < 8; ++e) y[e] += later.of(c + e, u.past + token + 1);
    }
    if (part) {
      if (token >= u.fresh) continue;   // (cleared by the join)
      float* dst = part + (r * 16 + rr) * PAGED_D + c;
      *(f32x4*)dst = (f32x4){y[0], y[1], y[2], y[3]};
      *(f32x4*)(dst + 4) = (f32x4){y[4], y[5], y[6], y[7]};
      if (c == 0) *(f32x2*)(part + R * 16 * PAGED_D + (r * 16 + rr) * 2) = (f32x2){row_top, sum};
    } else if (token < a.S) {
      // (rows without a token weigh the keys that every row sees: their sums are dropped here)
      const float scale = sum == 0.f || token >= u.fresh ? 0.f : 1.f / sum;
      u32x4 w;
#pragma unroll
      for (int e = 0; e < 4; ++e)
        w[e] = scale == 0.f ? 0u : __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2){y[2 * e] * scale, y[2 * e + 1] * scale}, bf16x2));
      *(u32x4*)(a.out + u.b * a.o_sb + (head * a.G + row % a.G) * a.o_sh + (int64_t)token * a.o_ss + c) = w;
    }
  }
  __syncthreads();
}

template <int BITS, int R, int NT, int DEPTH, int WAVES>
__global__ __launch_bounds__(WAVES * 64, 2) void attn_kernel(PagedAttnArgs a) {
  __shared__ __attribute__((aligned(16))) float o_lds[WAVES][16][O_PITCH];
  __shared__ float ml_lds[WAVES][16][2];
  __shared__ PagedShareLds share_lds;
  __shared__ RowsLds q_lds[R > 1 ? R : 1];
  __shared__ PagedLater later;
  // (a worker whose share goes over the end of a unit was the last to finish, by up to a third of its time: 8 bits, five drafted tokens of 16
  // sequences 73.5 -> 63.9 us, 64 sequences of one 61.7 -> 60.1)
  constexpr int EXTRA = BITS == 8 ? (R == 1 ? 1 : 4) : 0;
  paged_go<R * 16, WAVES * NT * PAGED_TILE, EXTRA, WAVES>(a, share_lds, blockIdx.x, false, [&](const PagedUnit& u, int head, int step, int steps, float* part)
                                            __attribute__((always_inline)) { work<BITS, R, NT, DEPTH, WAVES>(a, u, head, step, steps, part, o_lds, ml_lds, q_lds, later); });
}

// Joins the parts of every row tile and head that was cut: its first worker's beginning and the `more` workers' after it.  Sixteen lanes hold a
// row, 8 channels each; the workgroup's sixteen such groups take GROUPS shares of a row's parts and 16 / GROUPS rows.  With few rows there are
// many parts (128k tokens of one sequence: 65), and one group after the other through them all took 35 us.
template <int GROUPS>
__global__ __launch_bounds__(256) void join_kernel(PagedAttnArgs a, int rows) {
  const PagedHeader h = a.headers[blockIdx.x];
  if (h.more == 0) return;
  const int b = h.unit / a.row_tiles, fresh = h.fresh;
  const int lane = threadIdx.x & 15, group = threadIdx.x >> 4, share = group % GROUPS;
  const int rr = blockIdx.y * (16 / GROUPS) + group / GROUPS, row = (h.unit - b * a.row_tiles) * rows + rr, token = row / a.G;
  if (GROUPS == 16 && token >= a.S) return;
  const int slot = paged_slot_floats(rows);
  const float* first = a.parts + ((int64_t)blockIdx.x * 2 + 1) * slot;
  float top = -FLT_MAX, sum = 0.f;
  f32x4 y0 = {}, y1 = {};
  if (token < fresh) {
    // (four parts at a time, all of their loads before the first is used: with 64 parts a row 0.4 us less than a look at the count before each)
    for (int i0 = share; i0 <= h.more; i0 += 4 * GROUPS) {
      f32x2 ml[4];
      f32x4 x0[4], x1[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int i = min(i0 + j * GROUPS, h.more);
        // part i > 0: slot 0 of worker blockIdx.x + i, one slot and i - 1 pairs of slots further on
        const float* p = first + (i == 0 ? 0 : (int64_t)(2 * i - 1) * slot);
        ml[j] = *(const f32x2*)(p + rows * PAGED_D + rr * 2);
        x0[j] = *(const f32x4*)(p + rr * PAGED_D + lane * 8), x1[j] = *(const f32x4*)(p + rr * PAGED_D + lane * 8 + 4);
      }
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if (i0 + j * GROUPS > h.more) break;
        const float m = fmaxf(top, ml[j].x), old = __builtin_amdgcn_exp2f(top - m), now = __builtin_amdgcn_exp2f(ml[j].x - m);
        top = m;
        sum = sum * old + ml[j].y * now;
        y0 = y0 * old + x0[j] * now;
        y1 = y1 * old + x1[j] * now;
      }
    }
  }
  if (GROUPS > 1) {
    __shared__ float y_lds[16][16][8], ml_lds[16][2];
    *(f32x4*)y_lds[group][lane] = y0;
    *(f32x4*)(y_lds[group][lane] + 4) = y1;
    if (lane == 0) {
      ml_lds[group][0] = top;
      ml_lds[group][1] = sum;
    }
    __syncthreads();
    if (share != 0) return;
    for (int w = 0; w < GROUPS; ++w) top = fmaxf(top, ml_lds[group + w][0]);
    sum = 0.f;
    y0 = y1 = (f32x4){};
#pragma unroll
    for (int w = 0; w < GROUPS; ++w) {
      const float f = __builtin_amdgcn_exp2f(ml_lds[group + w][0] - top);
      sum += ml_lds[group + w][1] * f;
      y0 += *(const f32x4*)y_lds[group + w][lane] * f;
      y1 += *(const f32x4*)(y_lds[group + w][lane] + 4) * f;
    }
  }
  if (token >= a.S) return;
  const float scale = sum == 0.f || token >= fresh ? 0.f : 1.f / sum;
  auto two = [&](float x, float y) { return scale == 0.f ? 0u : __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2){x * scale, y * scale}, bf16x2)); };
  *(u32x4*)(a.out + b * a.o_sb + (h.head * a.G + row % a.G) * a.o_sh + (int64_t)token * a.o_ss + lane * 8) =
      (u32x4){two(y0[0], y0[1]), two(y0[2], y0[3]), two(y1[0], y1[1]), two(y1[2], y1[3])};
}

// Keys of a step of a row tile of `rows`, where a workgroup has four waves
constexpr bool through_lds(int rows, int kv_bits) { return rows > (kv_bits == 16 ? 32 : 64); }
constexpr int step_of(int rows, int kv_bits) { return through_lds(rows, kv_bits) ? 64 : (kv_bits == 4 && rows <= 48) || (kv_bits == 8 && rows <= 16) ? 256 : 128; }

struct Plan {
  int rows;      // of a row tile
  int workers;   // 0: sequences are not cut
  int waves;     // of a workgroup
  int step;      // its keys
  size_t bytes;
};
constexpr int row_tile_of(int64_t rows, int kv_bits) { return rows <= 16 ? 16 : rows <= 32 ? 32 : rows <= 48 && kv_bits != 16 ? 48 : rows <= 64 ? 64 : 128; }
constexpr size_t worker_bytes(int rows) { return sizeof(PagedHeader) + 2 * sizeof(float) * paged_slot_floats(rows); }
// lengths up to which no call with row tiles of `rows` is cut
constexpr int never_cut(int kv_bits, int rows) { return kv_bits == 16 ? 640 : kv_bits == 4 ? 1280 : through_lds(rows, 8) ? 950 : 1100; }

Plan plan_of(int B, int Hq, int Hkv, int S, int kv_bits, int max_len) {
  Plan p;
  max_len = std::min(max_len, PAGED_MAX_TOKENS);
  const int64_t rows = (int64_t)S * (Hq / Hkv);
  p.rows = row_tile_of(rows, kv_bits);
  // A cut costs a second launch, 4 us; a workgroup by itself gets 55 GB/s of a bf16 cache.  One sequence, 8 KV heads, uncut against cut: bf16 512
  // tokens 8.7 us against 11.1, 1024 13.3 against 10.2; 4 bits 1024 9.3 against 10.4, 2048 13.0 against 10.7.  Many sequences of 700 tokens in
  // bf16, 1300 in 4 bits: 16 of them 12.4 against 16.1 and 12.6 against 16.2, 32 19.6 against 24.7 and 14.5 against 19.0 (the rule's cut costs them
  // this), 64 37.8 against 37.6 and 30.2 against 27.7, 128 72.9 against 71.2 and 58.4 against 49.4.
  const int64_t units = (int64_t)B * ((rows + p.rows - 1) / p.rows) * Hkv;
  // 8 bits: a cut gains more the longer the units are, and less the more of them there are; the lengths from which it is faster lie near a line for
  // each kernel.  us, uncut against cut, all sequences of that length (in brackets 10 tokens up to it):
  //   16 rows    8 units 1250 11.5, 12.1; 1300 12.4, 11.8     32 1250 11.9, 13.0 (11.8, 11.5); 1400 13.0, 12.9 (12.9, 11.5)
  //              64 1500 15.0, 14.8 (13.2, 11.9); 1800 17.7, 18.2 (15.9, 14.6)     128 2000 19.6, 22.5 (18.0, 19.0); 2400 22.1, 23.5 (20.9, 19.5)
  //              256 2600 30.1, 34.4 (23.5, 25.4); 3300 36.9, 41.2 (27.8, 26.7)     512 2800 59.4, 62.6 (43.4, 43.2); 3300 70.5, 73.6 (47.1, 45.6)
  //   48 rows    32 1100 17.6, 18.4; 1300 19.1, 18.9     64 1600 21.9, 23.8 (20.3, 21.3); 2000 26.0, 24.4     128 2000 26.8, 34.1 (25.4, 25.0);
  //              2400 27.8, 31.3 (26.8, 27.2)     256 3300 43.0, 52.4 (35.9, 38.5); the line costs 4 units of 1000 tokens 2.7: 17.0, 14.3
  //   by LDS     32 units 1000 29, 37; 1200 33, 30     64 1000 31, 40; 1400 40, 34     128 1400 38, 43; 1800 47, 47     176 1600 43, 47; 2000 54, 51
  //              256 1800 55, 58; 2200 63, 63     512 4000 123, 125; the line costs 8 units of 800 tokens 9: 24, 15
  const int64_t least8 = never_cut(8, p.rows) + units * (through_lds(p.rows, 8) ? 5 : 8);
  const int64_t least = kv_bits == 8 ? std::min<int64_t>(least8, 3300) : never_cut(kv_bits, p.rows);
  const bool cut = max_len > least && (!through_lds(p.rows, kv_bits) || units < 4 * PAGED_WORKERS);
  // One worker of eight waves a compute unit instead of two of four: half as many parts, and no older workgroup that goes ahead.  8 bits, with one row
  // tile and few, long units: 128k tokens of one sequence 58.6 -> 55.9 us, 4 KV heads 39.1 -> 35.8, 32 sequences of 8000 tokens 56.3 -> 54.6.  Not
  // where a worker's share is a step or two (one sequence of 4100 tokens 11.1 -> 11.8, of 16000 15.2 -> 16.0), nor where it crosses from unit to
  // unit, as nothing runs beside the end of one (64 sequences of 17 .. 8191 tokens, 4 KV heads 62.2 -> 68.8).
  p.waves = 4, p.step = step_of(p.rows, kv_bits);
  if (kv_bits == 8 && p.rows == 16 && units <= 128 && units * ((max_len + 511) / 512) >= PAGED_WORKERS) p.waves = 8, p.step = 512;
  // (no more workers than there is work for)
  const int64_t steps = units * ((max_len + p.step - 1) / p.step);
  p.workers = cut ? (int)std::min<int64_t>(PAGED_WORKERS * 4 / p.waves, steps + 7) / 8 * 8 : 0;
  // Whole units have eight waves each.  8 bits: only where every compute unit has one at most and four waves would go more than four steps.  us, four
  // against eight: 16 rows, 8 units, 500 tokens 7.0, 7.7, 1000 10.5, 10.7, 1100 11.9, 11.0; 128 units 500 8.9, 9.2, 1000 13.0, 13.2, 1100 14.6, 13.4;
  // 256 units 1000 16.0, 16.1, 1100 17.4, 16.8; 512 units, two of which run beside each other, 1100 26.8, 30.6.  48 rows, 64 units, 500 14.6, 14.6,
  // 700 17.0, 16.4; 256 units 500 17.1, 17.2, 700 19.9, 19.4; 512 units 700 26.4, 36.0.  64 rows, 64 units, 500 16.4, 17.4, 700 19.2, 19.3, 800 20.8,
  // 19.5.
  if (!cut && !through_lds(p.rows, kv_bits)) p.waves = kv_bits == 8 && (units > 256 || max_len <= 4 * step_of(p.rows, 8)) ? 4 : 8;
  p.bytes = p.workers * worker_bytes(p.rows);
  return p;
}

// What holds every call with these heads and at most these sequences, new tokens and lengths: a row tile's rows, the row tiles and the steps of
// four waves grow with each of them, and a plan has no more workers than that, though it may have fewer or none.
size_t workspace_of(int B, int Hq, int Hkv, int S, int kv_bits, int max_len) {
  max_len = std::min(max_len, PAGED_MAX_TOKENS);
  const int64_t rows = (int64_t)S * (Hq / Hkv);
  const int tile = row_tile_of(rows, kv_bits), step = step_of(tile, kv_bits);
  if (max_len <= never_cut(kv_bits, tile)) return 0;
  const int64_t units = std::min<int64_t>(PAGED_WORKERS, (int64_t)B * ((rows + tile - 1) / tile) * Hkv), steps = units * ((max_len + step - 1) / step);
  return std::min<int64_t>(PAGED_WORKERS, (steps + 7) / 8 * 8) * worker_bytes(tile);
}

// NT tiles a wave and step, DEPTH steps ahead; with eight waves several row tiles leave each half the registers.
template <int BITS, int R, int NT, int DEPTH>
void launch(const PagedAttnArgs& a, int waves, hipStream_t stream) {
  const dim3 grid(a.headers ? a.workers : a.Hkv * a.B * a.row_tiles);
  if (waves == 8) hipLaunchKernelGGL((attn_kernel<BITS, R, R == 1 ? NT : 1, R == 1 ? DEPTH : 1, 8>), grid, dim3(512), 0, stream, a);
  else hipLaunchKernelGGL((attn_kernel<BITS, R, NT, DEPTH, 4>), grid, dim3(256), 0, stream, a);
}

}  // namespace

extern "C" size_t pbs_paged_attn_workspace_bytes(int B, int Hq, int Hkv, int S, int head_dim, int kv_bits, int max_len) {
  if (B <= 0 || Hq <= 0 || Hkv <= 0 || S <= 0 || Hq < Hkv || max_len <= 0) return 0;
  return workspace_of(B, Hq, Hkv, S, kv_bits, max_len);
}

extern "C" int pbs_paged_attn_fwd(const void* q, const void* k_pages, const void* v_pages, const void* k_scale, const void* v_scale,
                                  const int32_t* page_table, const int32_t* past_lens, const int32_t* new_lens, void* out, int B, int Hq, int Hkv,
                                  int S, int head_dim, int num_pages, int max_pages, int page_size, int kv_bits, int max_len, int64_t q_sb,
                                  int64_t q_sh, int64_t q_ss, int64_t o_sb, int64_t o_sh, int64_t o_ss, int64_t table_sb, float softmax_scale,
                                  void* workspace, size_t workspace_bytes, void* stream) {
  PagedAttnArgs a;
  if (const int rc = paged_pool(&a.pool, "pbs_paged_attn_fwd", k_pages, v_pages, k_scale, v_scale, page_table, table_sb, B, Hkv, head_dim, num_pages,
                                max_pages, page_size, kv_bits))
    return rc;
  PBS_REQUIRE(q && out && past_lens, "pbs_paged_attn_fwd: null tensor pointer");
  PBS_REQUIRE(S > 0 && S <= (1 << 26) && Hq > 0 && Hq <= 65535 && Hq % Hkv == 0, "pbs_paged_attn_fwd: bad shape");
  PBS_REQUIRE((int64_t)S * (Hq / Hkv) <= (1 << 26), "pbs_paged_attn_fwd: too many query rows");
  PBS_REQUIRE(max_len > 0, "pbs_paged_attn_fwd: max_len must be positive");
  PBS_REQUIRE(softmax_scale > 0.f && softmax_scale <= FLT_MAX, "pbs_paged_attn_fwd: softmax_scale must be positive and finite");
  PBS_REQUIRE(((q_sb | q_sh | q_ss | o_sb | o_sh | o_ss) % 8) == 0, "pbs_paged_attn_fwd: strides must keep rows 16-byte aligned");
  PBS_REQUIRE((((uintptr_t)q | (uintptr_t)out) % 16) == 0, "pbs_paged_attn_fwd: pointers must be 16-byte aligned");
  Plan p = plan_of(B, Hq, Hkv, S, kv_bits, max_len);
  PBS_REQUIRE(p.bytes == 0 || (workspace && ((uintptr_t)workspace % 256) == 0 && workspace_bytes >= p.bytes),
              "pbs_paged_attn_fwd: workspace of %zu bytes, 256-byte aligned, needed", p.bytes);
  a.q = (const uint16_t*)q; a.out = (uint16_t*)out; a.past = past_lens; a.fresh = new_lens;
  a.B = B; a.Hq = Hq; a.Hkv = Hkv; a.S = S; a.G = Hq / Hkv;
  a.q_sb = q_sb; a.q_sh = q_sh; a.q_ss = q_ss; a.o_sb = o_sb; a.o_sh = o_sh; a.o_ss = o_ss;
  a.scale_log2 = softmax_scale * 1.44269504088896340736f;
  a.room = (float)(32 - __builtin_clz((unsigned)(max_pages * page_size - 1)));   // (32 tokens at least)
  a.row_tiles = (S * a.G + p.rows - 1) / p.rows;
  const int64_t units = (int64_t)B * Hkv * a.row_tiles;
  PBS_REQUIRE(units < (1 << 22), "pbs_paged_attn_fwd: too many query rows");   // (a grid's threads fit 32 bits)
  // the line of steps that workers share has to fit 32 bits, whatever the lengths turn out to be: a call that may not is not cut
  if (units * ((int64_t)max_pages * page_size / p.step + 16) > INT32_MAX) p.workers = 0, p.waves = 8;
  a.workers = p.workers;
  a.headers = p.workers ? (PagedHeader*)workspace : nullptr;
  a.parts = p.workers ? (float*)((char*)workspace + p.workers * sizeof(PagedHeader)) : nullptr;
  hipStream_t st = (hipStream_t)stream;
  if (through_lds(p.rows, kv_bits)) {
    if (const int rc = paged_attn_rows(a, kv_bits, p.rows, st)) return rc;
  } else if (kv_bits == 16) {
    if (p.rows == 16) launch<16, 1, 1, 1>(a, p.waves, st);
    else launch<16, 2, 1, 1>(a, p.waves, st);
  } else if (kv_bits == 8) {
    // (one step of one tile a wave, where that is all: 128 sequences of 100 tokens 13.5 -> 12.0 us)
    if (p.rows == 16 && !p.workers && max_len <= 128) launch<8, 1, 1, 1>(a, p.waves, st);
    else if (p.rows == 16) launch<8, 1, 2, 1>(a, p.waves, st);
    else if (p.rows == 32) launch<8, 2, 1, 1>(a, p.waves, st);
    else if (p.rows == 48) launch<8, 3, 1, 1>(a, p.waves, st);
    else launch<8, 4, 1, 1>(a, p.waves, st);
  } else {
    if (p.rows == 16) launch<4, 1, 2, 2>(a, p.waves, st);
    else if (p.rows == 32) launch<4, 2, 2, 1>(a, p.waves, st);
    else if (p.rows == 48) launch<4, 3, 2, 1>(a, p.waves, st);
    else launch<4, 4, 1, 1>(a, p.waves, st);
  }
  if (p.workers) {
    const int rows = (int)std::min<int64_t>(p.rows, (int64_t)S * a.G);
    // (parts of a row, if sequences are alike: with 32 heads' rows of one sequence, 4 KV heads, 128.  Where they are not, a long one's parts are
    // joined by fewer groups than they could be: one of 100000 tokens among 63 of 500, 8 KV heads, bf16 109 us, 4 bits 48, of which the cache
    // takes 109 and 29 at a copy's rate.)
    const int64_t parts = p.workers / units;
    if (parts >= 32) hipLaunchKernelGGL(join_kernel<16>, dim3(p.workers, rows), dim3(256), 0, st, a, p.rows);
    else if (parts >= 4) hipLaunchKernelGGL(join_kernel<4>, dim3(p.workers, (rows + 3) / 4), dim3(256), 0, st, a, p.rows);
    else hipLaunchKernelGGL(join_kernel<1>, dim3(p.workers, (rows + 15) / 16), dim3(256), 0, st, a, p.rows);
  }
  return pbs_check_launch("pbs_paged_attn_fwd");
}
