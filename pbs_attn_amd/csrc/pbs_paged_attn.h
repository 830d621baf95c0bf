// Attention over a paged cache: what its kernels share.  Arguments, the row tiles of a sequence, and how the work is cut.
#pragma once
#include "pbs_paged.h"
#include "pbs_wave.h"
#include <float.h>

constexpr int PAGED_WAVES = 4;       // of a workgroup
constexpr int PAGED_WORKERS = 512;   // workgroups of a launch that cuts sequences, at most: two a compute unit
// A row's exponent is taken up where a logit is more than this above it (log2): weights stay below 2^8, which costs their sums in fp32 and their
// roundings to bf16 nothing, and the sums are rescaled a few times in a sequence rather than with every new maximum.
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
