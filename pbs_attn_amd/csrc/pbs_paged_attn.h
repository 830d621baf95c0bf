// Attention over a paged cache: what its kernels share.  Arguments, the row tiles of a sequence, and how the work is cut.
#pragma once
#include "pbs_paged.h"
#include "pbs_wave.h"
#include <float.h>
#include <limits.h>
#include <math.h>

typedef __attribute__((ext_vector_type(8))) int i32x8;
typedef __attribute__((ext_vector_type(2))) uint32_t u32x2;

constexpr int PAGED_WAVES = 4;       // of a workgroup
constexpr int PAGED_WORKERS = 512;   // workgroups of a launch that cuts sequences, at most: two a compute unit
// A row's exponent m stays `room` .. `room` + PAGED_SLACK (log2) above its largest logit: it is taken up, by the most that it may be, where a logit
// comes nearer, so the sums are rescaled a few times in a sequence rather than with every new maximum.  2^room is as many tokens as the table has
// room for, so the sums of weighted values, which are joined as they are, never pass the largest value that the cache holds, and stay finite as
// their average does (with logits below 2^24; above, the exponent itself is rounded).  It costs the smallest numbers, which come nearer to fp32's
// least, 2^-149: with room for 2^17 tokens weights of less than 2^-101 of the row's largest are zeros, and values below 2^-116 lose bits.
constexpr float PAGED_SLACK = 8.f;

struct PagedHeader {   // of a worker: the piece of work that it began and left to the `more` workers after it
  int unit, head, more, pad;
};

struct PagedAttnArgs {
  PagedPool pool;
  const uint16_t* q;
  uint16_t* out;
  const int32_t* past;
  const int32_t* fresh;   // null: S
  PagedHeader* headers;   // one a worker; null: a workgroup takes a whole row tile of one head
  float* parts;           // two slots a worker: the end of an earlier worker's piece, the beginning of the next one's
  int B, Hq, Hkv, S, G, row_tiles, workers;
  int64_t q_sb, q_sh, q_ss, o_sb, o_sh, o_ss;
  float scale_log2;   // softmax scale times log2(e)
  float room;
};

// a slot: rows of 128 sums, then each row's largest exponent and sum of weights
constexpr int paged_slot_floats(int rows) { return rows * (PAGED_D + 2); }

__device__ __forceinline__ float max_over_groups(float v) {   // lanes l, l ^ 16, l ^ 32, l ^ 48
  TwoOf t = with_lane_xor<16>(__float_as_uint(v));
  v = fmaxf(__uint_as_float(t.a), __uint_as_float(t.b));
  t = with_lane_xor<32>(__float_as_uint(v));
  return fmaxf(__uint_as_float(t.a), __uint_as_float(t.b));
}

// lane id formed where it is asked for: what is derived from it holds no registers elsewhere
__device__ __forceinline__ int paged_lane() {
  int l;
  asm volatile("v_mbcnt_lo_u32_b32 %0, -1, 0\n\tv_mbcnt_hi_u32_b32 %0, -1, %0" : "=v"(l));
  return l;
}

// What a lane holds of a tile of 32 tokens.  n = lane % 16, g = lane / 16.
template <int BITS>
struct Tile;
template <>
struct Tile<16> {
  u32x4 k[8], v[8];
};
template <>
struct Tile<4> {
  u32x4 k[2], v[2];
  uint32_t ks;
  u32x2 vs;
};
__device__ __forceinline__ void load_k(Tile<16>& t, const PagedPool& p, int64_t at, int n, int g) {
  const char* k = p.k + at * paged_tile_bytes<16>() + n * 512 + g * 16;
#pragma unroll
  for (int h = 0; h < 2; ++h)
#pragma unroll
    for (int c = 0; c < 4; ++c) t.k[h * 4 + c] = *(const u32x4*)(k + h * 256 + c * 64);
}
__device__ __forceinline__ void load_v(Tile<16>& t, const PagedPool& p, int64_t at, int n, int g) {
  const char* v = p.v + at * paged_tile_bytes<16>() + g * 2048 + n * 16;
#pragma unroll
  for (int d = 0; d < 8; ++d) t.v[d] = *(const u32x4*)(v + d * 256);
}
__device__ __forceinline__ void load_k(Tile<4>& t, const PagedPool& p, int64_t at, int n, int g) {
  const char* k = p.k + at * paged_tile_bytes<4>() + n * 128 + g * 16;
  t.k[0] = *(const u32x4*)k;
  t.k[1] = *(const u32x4*)(k + 64);
  t.ks = *(const uint16_t*)(p.ks + at * 128 + g * 32 + n * 2);
}
__device__ __forceinline__ void load_v(Tile<4>& t, const PagedPool& p, int64_t at, int n, int g) {
  const char* v = p.v + at * paged_tile_bytes<4>() + g * 512 + n * 16;
  t.v[0] = *(const u32x4*)v;
  t.v[1] = *(const u32x4*)(v + 256);
  t.vs = *(const u32x2*)(p.vs + at * 128 + (n >> 2) * 32 + g * 8);
}

// Values that are not finite, of tokens that some of a row tile's rows do not see (the call's own): not even times zero.  They leave the tile that
// is multiplied, and the rows that see one get it at the end: what a row sees begins with the first token, so the first key is enough.
// (Products of ones that count them instead, in registers, spilled.  Asked for by every row at the end, 35 rows take 64 us; only where one was
// noted, 59.6; without any of it 57.8.)
struct PagedLater {
  int up[PAGED_D], down[PAGED_D];   // by channel: the first key that is an infinity or NaN, for `up` all but -inf, for `down` all but +inf
  int any;

  __device__ __forceinline__ void begin() {
    if (threadIdx.x < PAGED_D) up[threadIdx.x] = down[threadIdx.x] = INT_MAX;
    if (threadIdx.x == 0) any = 0;
    __syncthreads();
  }
  __device__ __forceinline__ void note(int channel, int key, uint32_t bits) {   // (bits of the bf16 value)
    if (bits != 0xff80u) atomicMin(&up[channel], key);
    if (bits != 0x7f80u) atomicMin(&down[channel], key);
    any = 1;
  }
  __device__ __forceinline__ bool is_any() const { return __builtin_amdgcn_readfirstlane(any) != 0; }
  __device__ __forceinline__ float of(int channel, int seen) const {
    return (up[channel] < seen ? INFINITY : 0.f) - (down[channel] < seen ? INFINITY : 0.f);
  }
};
__device__ __forceinline__ bool not_finite(uint32_t bf16_bits) { return (bf16_bits & 0x7f80u) == 0x7f80u; }

// 16 query rows as the matrix instruction's right operand
template <int BITS>
struct Rows;
struct RowsLds {   // of the four waves, lane by lane
  u32x4 q[4][64];
  int scale[64];
};
template <>
struct Rows<16> {
  bf16x8 q[4];
  __device__ __forceinline__ void put(RowsLds& lds, int lane) const {
#pragma unroll
    for (int c = 0; c < 4; ++c) lds.q[c][lane] = __builtin_bit_cast(u32x4, q[c]);
  }
  __device__ __forceinline__ void get(const RowsLds& lds, int lane) {
#pragma unroll
    for (int c = 0; c < 4; ++c) q[c] = __builtin_bit_cast(bf16x8, lds.q[c][lane]);
  }
  __device__ __forceinline__ void load(const uint16_t* row, int g) {
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      u32x4 x = {};
      if (row) x = *(const u32x4*)(row + c * 32 + g * 8);
      q[c] = __builtin_bit_cast(bf16x8, x);
    }
  }
};
// For 4-bit keys the queries are the sum of two e4m3 numbers a channel: the matrix instruction then takes the keys as they lie in memory, with
// their scales.  A bf16 value has 8 bits, e4m3 4: q = 2^e (hi + lo / 32) with hi = e4m3(q / 2^e) and lo the 4 bits that are left, exact down to 2^-21
// of the row's largest channel (below it both halves are subnormal and lo is rounded).
template <>
struct Rows<4> {
  i32x8 hi, lo;
  int scale_hi;
  __device__ __forceinline__ int scale_lo() const { return scale_hi == 255 ? 255 : scale_hi - 5; }
  __device__ __forceinline__ void put(RowsLds& lds, int lane) const {
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      lds.q[c][lane] = (u32x4){(uint32_t)hi[4 * c], (uint32_t)hi[4 * c + 1], (uint32_t)hi[4 * c + 2], (uint32_t)hi[4 * c + 3]};
      lds.q[2 + c][lane] = (u32x4){(uint32_t)lo[4 * c], (uint32_t)lo[4 * c + 1], (uint32_t)lo[4 * c + 2], (uint32_t)lo[4 * c + 3]};
    }
    lds.scale[lane] = scale_hi;
  }
  __device__ __forceinline__ void get(const RowsLds& lds, int lane) {
    const u32x4 a = lds.q[0][lane], b = lds.q[1][lane], c = lds.q[2][lane], d = lds.q[3][lane];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      hi[e] = (int)a[e]; hi[4 + e] = (int)b[e];
      lo[e] = (int)c[e]; lo[4 + e] = (int)d[e];
    }
    scale_hi = lds.scale[lane];
  }
  __device__ __forceinline__ void load(const uint16_t* row, int g) {
    u32x4 x[4] = {};   // channels 16 g .. 16 g + 15 and 64 + 16 g ..: 32 bytes of an 8-bit operand
    if (row) {
      x[0] = *(const u32x4*)(row + g * 16);
      x[1] = *(const u32x4*)(row + g * 16 + 8);
      x[2] = *(const u32x4*)(row + 64 + g * 16);
      x[3] = *(const u32x4*)(row + 64 + g * 16 + 8);
    }
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) top = max(top, max(x[i][e] & 0x7fffu, (x[i][e] >> 16) & 0x7fffu));
    TwoOf t = with_lane_xor<16>(top);
    top = max(t.a, t.b);
    t = with_lane_xor<32>(top);
    top = max(t.a, t.b);
    const int field = max((int)(top >> 7), 20);
    const float up = __uint_as_float((uint32_t)(261 - field) << 23);   // the row's largest magnitude becomes 128 .. 256
#pragma unroll
    for (int w = 0; w < 8; ++w) {
      const uint32_t a = x[w >> 1][(w & 1) * 2], b = x[w >> 1][(w & 1) * 2 + 1];
      const float y0 = bf16_bits_to_f32(a & 0xffffu) * up, y1 = __uint_as_float(a & 0xffff0000u) * up;
      const float y2 = bf16_bits_to_f32(b & 0xffffu) * up, y3 = __uint_as_float(b & 0xffff0000u) * up;
      int h = __builtin_amdgcn_cvt_pk_fp8_f32(y0, y1, 0, false);
      h = __builtin_amdgcn_cvt_pk_fp8_f32(y2, y3, h, true);
      int l = __builtin_amdgcn_cvt_pk_fp8_f32((y0 - __builtin_amdgcn_cvt_f32_fp8(h, 0)) * 32.f, (y1 - __builtin_amdgcn_cvt_f32_fp8(h, 1)) * 32.f, 0, false);
      l = __builtin_amdgcn_cvt_pk_fp8_f32((y2 - __builtin_amdgcn_cvt_f32_fp8(h, 2)) * 32.f, (y3 - __builtin_amdgcn_cvt_f32_fp8(h, 3)) * 32.f, l, true);
      hi[w] = h;
      lo[w] = l;
    }
    scale_hi = field >= 255 ? 255 : field - 7;    // (an infinity or NaN among the queries: NaN)
  }
};

// S^T of one half (16 keys, operand row m = token 2 m + half) and 16 query rows
__device__ __forceinline__ f32x4 logits(const Tile<16>& t, int half, const Rows<16>& r) {
  f32x4 s = {};
#pragma unroll
  for (int c = 0; c < 4; ++c) s = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, t.k[half * 4 + c]), r.q[c], s, 0, 0, 0);
  return s;
}
template <int HALF>
__device__ __forceinline__ f32x4 logits4(const Tile<4>& t, const Rows<4>& r) {
  const i32x8 k = {(int)t.k[HALF][0], (int)t.k[HALF][1], (int)t.k[HALF][2], (int)t.k[HALF][3], 0, 0, 0, 0};
  f32x4 s = {};
  s = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(k, r.lo, s, 4, 0, HALF, (int)t.ks, 0, r.scale_lo());
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(k, r.hi, s, 4, 0, HALF, (int)t.ks, 0, r.scale_hi);
}
__device__ __forceinline__ f32x4 logits(const Tile<4>& t, int half, const Rows<4>& r) { return half ? logits4<1>(t, r) : logits4<0>(t, r); }

// a sequence, and one of its row tiles
struct PagedSeq {
  int b, past, fresh;
  int steps;         // of a row tile with tokens (the last one's: tiles before it see fewer keys, and idle for a while)
  int a_head;        // steps of one head: row tiles without tokens take one, in which their rows are cleared
  int tiles;         // row tiles with tokens
};
template <int ROWS, int STEP>
__device__ __forceinline__ PagedSeq paged_seq(const PagedAttnArgs& a, int b) {
  PagedSeq s;
  s.b = b;
  s.past = min(max(a.past[b], 0), PAGED_MAX_TOKENS);
  s.fresh = a.fresh ? min(max(a.fresh[b], 0), a.S) : a.S;
  s.tiles = (s.fresh * a.G + ROWS - 1) / ROWS;
  s.steps = max((min(s.past + s.fresh, a.pool.max_pages << a.pool.page_shift) + STEP - 1) / STEP, 1);
  s.a_head = s.tiles * s.steps + (a.row_tiles - s.tiles);
  return s;
}
struct PagedUnit {
  int b, r0, past, fresh;
  int keys;      // that its last token sees
  int all_see;   // that its first token sees
};
template <int ROWS>
__device__ __forceinline__ PagedUnit paged_unit(const PagedAttnArgs& a, int b, int past, int fresh, int tile) {
  PagedUnit t;
  t.b = b; t.past = past; t.fresh = fresh;
  t.r0 = tile * ROWS;
  const int first = t.r0 / a.G, last = min(fresh - 1, (t.r0 + ROWS - 1) / a.G);
  t.keys = first < fresh ? min(past + last + 1, a.pool.max_pages << a.pool.page_shift) : 0;
  t.all_see = past + first + 1;
  return t;
}

// Where a workgroup begins, and how many steps are its.  The steps of all sequences lie in one line (sequence, head, row tile, step), cut
// into equal shares, one a worker, so that sequences of any lengths fill the chip.  (The host sees to it that the line's length fits 32 bits.)
struct PagedShare {
  int b, head, tile, step, todo, share;
};
struct PagedShareLds {
  int wave_sums[PAGED_WAVES], left, b;
};
template <int ROWS, int STEP>
__device__ __forceinline__ bool paged_share(const PagedAttnArgs& a, PagedShareLds& lds, int worker, int workers, PagedShare* out) {
  int total = 0, before = 0, mine = 0, from = 0;
  if (a.B == 1) {
    total = a.Hkv * paged_seq<ROWS, STEP>(a, 0).a_head;
  } else {   // running sums over the sequences, a stretch of them a thread
    const int tid = threadIdx.x, stretch = (a.B + 255) / 256, to = min((tid + 1) * stretch, a.B);
    from = min(tid * stretch, a.B);
    for (int i = from; i < to; ++i) mine += a.Hkv * paged_seq<ROWS, STEP>(a, i).a_head;
    before = mine;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const int other = __shfl_up(before, d, 64);
      if ((tid & 63) >= d) before += other;
    }
    if ((tid & 63) == 63) lds.wave_sums[tid >> 6] = before;
    before -= mine;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < PAGED_WAVES; ++w) {
      if (w < (tid >> 6)) before += lds.wave_sums[w];
      total += lds.wave_sums[w];
    }
    total = __builtin_amdgcn_readfirstlane(total);
  }
  const int share = (int)(((unsigned)total + workers - 1) / workers);
  if ((int64_t)share * worker >= total) return false;
  const int start = share * worker;
  out->share = share;
  out->todo = min(share, total - start);
  int b = 0, left = start;
  if (a.B > 1) {
    if (start >= before && start < before + mine) {
      left = start - before;
      for (int i = from;; ++i) {
        const int cost = a.Hkv * paged_seq<ROWS, STEP>(a, i).a_head;
        if (left < cost) {
          lds.b = i;
          lds.left = left;
          break;
        }
        left -= cost;
      }
    }
    __syncthreads();
    b = __builtin_amdgcn_readfirstlane(lds.b);
    left = __builtin_amdgcn_readfirstlane(lds.left);
  }
  const PagedSeq s = paged_seq<ROWS, STEP>(a, b);
  const int full = s.tiles * s.steps;
  out->b = b;
  out->head = left / s.a_head;
  left -= out->head * s.a_head;
  out->tile = left < full ? left / s.steps : s.tiles + (left - full);
  out->step = left < full ? left - out->tile * s.steps : 0;
  return true;
}

// A workgroup's way through its share, or through the one row tile and head that are its without headers: work(unit, head, first step,
// steps, part), part null where the steps are all that the row tile has.
template <int ROWS, int STEP, class Work>
__device__ __forceinline__ void paged_go(const PagedAttnArgs& a, PagedShareLds& lds, int worker, bool last_tile_first, Work&& work) {
  PagedShare at;
  if (a.headers) {
    if (!paged_share<ROWS, STEP>(a, lds, worker, gridDim.x, &at)) {
      if (threadIdx.x == 0) a.headers[worker].more = 0;
      return;
    }
  } else {
    const int unit = blockIdx.x / a.Hkv, tile = unit % a.row_tiles;
    at.b = unit / a.row_tiles; at.head = blockIdx.x % a.Hkv; at.tile = last_tile_first ? a.row_tiles - 1 - tile : tile; at.step = 0;
    at.share = at.todo = INT32_MAX;
  }
  int more = 0;
  PagedSeq s = paged_seq<ROWS, STEP>(a, at.b);
  while (true) {
    const int steps = at.tile < s.tiles ? s.steps : 1, n = min(steps - at.step, at.todo);
    at.todo -= n;
    float* part = nullptr;
    if (n < steps) part = a.parts + ((int64_t)worker * 2 + (at.step == 0)) * paged_slot_floats(ROWS);
    if (at.step == 0 && n < steps) more = (int)((unsigned)(steps - n + at.share - 1) / (unsigned)at.share);
    work(paged_unit<ROWS>(a, s.b, s.past, s.fresh, at.tile), at.head, at.step, n, part);
    if (!a.headers) return;
    if (at.todo == 0) break;
    at.step = 0;
    if (++at.tile == a.row_tiles) {
      at.tile = 0;
      if (++at.head == a.Hkv) {
        at.head = 0;
        s = paged_seq<ROWS, STEP>(a, s.b + 1);
      }
    }
  }
  if (threadIdx.x == 0) a.headers[worker] = {s.b * a.row_tiles + at.tile, at.head, more, 0};
}

// many rows a row tile (csrc/pbs_paged_rows.hip)
int paged_attn_rows(const PagedAttnArgs& a, int kv_bits, int rows, hipStream_t stream);
