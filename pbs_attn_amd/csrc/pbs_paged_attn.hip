// Attention of a batch's new tokens over a paged cache (the tokens themselves are in it already).
//
// For query i of a sequence with `past` tokens before the call: o = sum_j p_j v_j / sum_j p_j, p_j = exp(scale q k_j - m), over the keys
// j <= past + i, m the largest exponent so far (one pass: sums are rescaled where it grows).  All query heads of a KV head and several
// tokens share a tile's rows, row r = (token r / G, head r % G of the group), so a key is read once for all of them.
#include "pbs_paged.h"
#include "pbs_wave.h"
#include "../../include/pbs_hip.h"   // the definitions below are checked against the public declarations
#include <float.h>
#include <math.h>

namespace {

struct AttnArgs {
  PagedPool pool;
  const uint16_t* q;
  uint16_t* out;
  const int32_t* past;
  const int32_t* fresh;   // null: S
  int B, Hq, Hkv, S, G;
  int64_t q_sb, q_sh, q_ss, o_sb, o_sh, o_ss;
  float scale_log2;   // softmax scale times log2(e)
};

constexpr int WAVES = 4;
constexpr int ROWS = 16;
constexpr int O_PITCH = PAGED_D + 4;

__device__ __forceinline__ float max_over_groups(float v) {   // lanes l, l ^ 16, l ^ 32, l ^ 48
  TwoOf t = with_lane_xor<16>(__float_as_uint(v));
  v = fmaxf(__uint_as_float(t.a), __uint_as_float(t.b));
  t = with_lane_xor<32>(__float_as_uint(v));
  return fmaxf(__uint_as_float(t.a), __uint_as_float(t.b));
}
__device__ __forceinline__ float sum_over_groups(float v) {
  TwoOf t = with_lane_xor<16>(__float_as_uint(v));
  v = __uint_as_float(t.a) + __uint_as_float(t.b);
  t = with_lane_xor<32>(__float_as_uint(v));
  return __uint_as_float(t.a) + __uint_as_float(t.b);
}

// Lanes: n = lane % 16, g = lane / 16.  S^T = K Q^T by 16x16x32: operand row m of tile half a is token 2m + a, so that a lane ends up with
// the logits of tokens 8g .. 8g + 7 for query row n, which are its share of P^T in O^T += V^T P^T: probabilities never change lanes.
template <int BITS>
__global__ __launch_bounds__(256) void attn_kernel(AttnArgs a) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, n = lane & 15, g = lane >> 4;
  const int b = blockIdx.z, head = blockIdx.y, r0 = blockIdx.x * ROWS;
  const int past = min(max(a.past[b], 0), PAGED_MAX_TOKENS), fresh = a.fresh ? min(max(a.fresh[b], 0), a.S) : a.S;
  const int row = r0 + n, token = row / a.G, qh = head * a.G + row % a.G;
  const bool valid = token < fresh;
  __shared__ float o_lds[WAVES][ROWS][O_PITCH];
  __shared__ float m_lds[WAVES][ROWS], l_lds[WAVES][ROWS];

  const int seen = valid ? past + token + 1 : 0;                          // keys of this lane's row
  const int last = min(fresh - 1, (r0 + ROWS - 1) / a.G);                 // the tile's last token
  const int keys = min(r0 / a.G < fresh ? past + last + 1 : 0, a.pool.max_pages << a.pool.page_shift);
  const int all_see = past + r0 / a.G + 1;                                // keys that every row sees

  bf16x8 q[4];
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    u32x4 x = {};
    if (valid) x = *(const u32x4*)(a.q + b * a.q_sb + qh * a.q_sh + (int64_t)token * a.q_ss + c * 32 + g * 8);
    q[c] = __builtin_bit_cast(bf16x8, x);
  }
  f32x4 o[8] = {};
  float m = -FLT_MAX, l = 0.f;
  for (int t = wave; t * PAGED_TILE < keys; t += WAVES) {
    const int64_t at = paged_tile_index(a.pool, b, head, t);
    if (at < 0) continue;
    f32x4 st[2] = {};
#pragma unroll
    for (int h = 0; h < 2; ++h) {
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        u32x4 k;
        if (BITS == 16) {
          k = *(const u32x4*)(a.pool.k + at * paged_tile_bytes<16>() + (2 * n + h) * 256 + c * 64 + g * 16);
        } else {
          const uint32_t w = *(const uint32_t*)(a.pool.k + at * paged_tile_bytes<4>() + (2 * n + h) * 64 + c * 16 + g * 4);
          k = fp4_values(w, __uint_as_float((uint32_t)a.pool.ks[at * 128 + c * 32 + 2 * n + h] << 23));
        }
        st[h] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, k), q[c], st[h], 0, 0, 0);
      }
    }
    // st[h][i]: token 8g + 2i + h
    float x[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] = st[j & 1][j >> 1] * a.scale_log2;
    const int k0 = t * PAGED_TILE;
    if (k0 + PAGED_TILE > all_see) {
#pragma unroll
      for (int j = 0; j < 8; ++j) x[j] = k0 + 8 * g + j < seen ? x[j] : -INFINITY;
    }
    float top = x[0];
#pragma unroll
    for (int j = 1; j < 8; ++j) top = fmaxf(top, x[j]);
    const float m_new = fmaxf(m, max_over_groups(top));
    const float scale = exp2f(m - m_new);
    m = m_new;
    l *= scale;
#pragma unroll
    for (int d = 0; d < 8; ++d) o[d] *= scale;
    bf16x8 p;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float e = exp2f(x[j] - m);
      l += e;
      p[j] = (__bf16)e;   // (weights of at most 1, half a step of 2^-8 off: they are summed as they are, and multiply bf16 values)
    }
    // tokens behind the keys hold whatever the page held before: not even times zero
    const int held = keys - k0 - 8 * g;   // of this lane's eight
    u32x4 v[8];
    if (BITS == 16) {
#pragma unroll
      for (int d = 0; d < 8; ++d) {
        v[d] = *(const u32x4*)(a.pool.v + at * paged_tile_bytes<16>() + (g * PAGED_D + d * 16 + n) * 16);
        if (k0 + PAGED_TILE > keys) {
#pragma unroll
          for (int w = 0; w < 4; ++w) v[d][w] &= held >= 2 * w + 2 ? 0xffffffffu : held == 2 * w + 1 ? 0xffffu : 0u;
        }
      }
    } else {
      u32x4 x[8];   // token j: channels 8n .. 8n + 7
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const uint32_t w = *(const uint32_t*)(a.pool.v + at * paged_tile_bytes<4>() + ((2 * g + (j >> 2)) * 16 + n) * 16 + (j & 3) * 4);
        const uint32_t e = a.pool.vs[at * 128 + (n >> 2) * 32 + 8 * g + j];
        x[j] = fp4_values(w, __uint_as_float(e << 23));
        if (j >= held) x[j] = (u32x4){};
      }
#pragma unroll
      for (int c = 0; c < 4; ++c)
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          v[2 * c][w] = __builtin_amdgcn_perm(x[2 * w + 1][c], x[2 * w][c], 0x05040100u);
          v[2 * c + 1][w] = __builtin_amdgcn_perm(x[2 * w + 1][c], x[2 * w][c], 0x07060302u);
        }
    }
#pragma unroll
    for (int d = 0; d < 8; ++d) o[d] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, v[d]), p, o[d], 0, 0, 0);
  }

  l = sum_over_groups(l);
  if (g == 0) { m_lds[wave][n] = m; l_lds[wave][n] = l; }
  __syncthreads();
  float top = m_lds[0][n], sum = 0.f;
#pragma unroll
  for (int w = 1; w < WAVES; ++w) top = fmaxf(top, m_lds[w][n]);
#pragma unroll
  for (int w = 0; w < WAVES; ++w) sum += l_lds[w][n] * exp2f(m_lds[w][n] - top);
  // (rows without a token weigh the keys that every row sees: their sums are dropped here)
  const float f = (sum == 0.f || !valid ? 0.f : 1.f / sum) * exp2f(m - top);
#pragma unroll
  for (int d = 0; d < 8; ++d)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      // operand row 4g + i of tile d: channel 16 d + 4 g + i, of 4-bit pages channel 8 (4 g + i) + d
      const int channel = BITS == 16 ? d * 16 + 4 * g + i : (4 * g + i) * 8 + d;
      o_lds[wave][n][channel] = f == 0.f ? 0.f : o[d][i] * f;
    }
  __syncthreads();
  // 16 lanes a row, 8 channels a lane
  const int rr = threadIdx.x >> 4, c = (threadIdx.x & 15) * 8;
  const int tok = (r0 + rr) / a.G, h = head * a.G + (r0 + rr) % a.G;
  if (tok >= a.S) return;
  u32x4 y;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    f32x2 s = {};
#pragma unroll
    for (int w = 0; w < WAVES; ++w) s += (f32x2){o_lds[w][rr][c + 2 * e], o_lds[w][rr][c + 2 * e + 1]};
    y[e] = __builtin_bit_cast(uint32_t, __builtin_convertvector(s, bf16x2));
  }
  *(u32x4*)(a.out + b * a.o_sb + h * a.o_sh + (int64_t)tok * a.o_ss + c) = y;
}

}  // namespace

extern "C" size_t pbs_paged_attn_workspace_bytes(int B, int Hq, int Hkv, int S, int head_dim, int max_len) { return 0; }

extern "C" int pbs_paged_attn_fwd(const void* q, const void* k_pages, const void* v_pages, const void* k_scale, const void* v_scale,
                                  const int32_t* page_table, const int32_t* past_lens, const int32_t* new_lens, void* out, int B, int Hq, int Hkv,
                                  int S, int head_dim, int num_pages, int max_pages, int page_size, int kv_bits, int max_len, int64_t q_sb,
                                  int64_t q_sh, int64_t q_ss, int64_t o_sb, int64_t o_sh, int64_t o_ss, int64_t table_sb, float softmax_scale,
                                  void* workspace, size_t workspace_bytes, void* stream) {
  AttnArgs a;
  if (const int rc = paged_pool(&a.pool, "pbs_paged_attn_fwd", k_pages, v_pages, k_scale, v_scale, page_table, table_sb, B, Hkv, head_dim, num_pages,
                                max_pages, page_size, kv_bits))
    return rc;
  PBS_REQUIRE(q && out && past_lens, "pbs_paged_attn_fwd: null tensor pointer");
  PBS_REQUIRE(S > 0 && S <= (1 << 26) && Hq > 0 && Hq <= 65535 && Hq % Hkv == 0, "pbs_paged_attn_fwd: bad shape");
  PBS_REQUIRE((int64_t)S * (Hq / Hkv) <= (1 << 26), "pbs_paged_attn_fwd: too many query rows");
  PBS_REQUIRE(softmax_scale > 0.f && softmax_scale <= FLT_MAX, "pbs_paged_attn_fwd: softmax_scale must be positive and finite");
  PBS_REQUIRE(((q_sb | q_sh | q_ss | o_sb | o_sh | o_ss) % 8) == 0, "pbs_paged_attn_fwd: strides must keep rows 16-byte aligned");
  PBS_REQUIRE((((uintptr_t)q | (uintptr_t)out) % 16) == 0, "pbs_paged_attn_fwd: pointers must be 16-byte aligned");
  a.q = (const uint16_t*)q; a.out = (uint16_t*)out; a.past = past_lens; a.fresh = new_lens;
  a.B = B; a.Hq = Hq; a.Hkv = Hkv; a.S = S; a.G = Hq / Hkv;
  a.q_sb = q_sb; a.q_sh = q_sh; a.q_ss = q_ss; a.o_sb = o_sb; a.o_sh = o_sh; a.o_ss = o_ss;
  a.scale_log2 = softmax_scale * 1.44269504088896340736f;
  const dim3 grid((S * a.G + ROWS - 1) / ROWS, Hkv, B);
  if (kv_bits == 16) hipLaunchKernelGGL(attn_kernel<16>, grid, dim3(256), 0, (hipStream_t)stream, a);
  else hipLaunchKernelGGL(attn_kernel<4>, grid, dim3(256), 0, (hipStream_t)stream, a);
  return pbs_check_launch("pbs_paged_attn_fwd");
}
