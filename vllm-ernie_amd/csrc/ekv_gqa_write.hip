// Write side of grouped-query layers:
//
//  * qk_norm_rope   RMS norm of every q / k head and the rotation of a slice of
//                   its channels, one pass.
//  * gqa_append     a call's keys and values into 8-bit pages with a scale per
//                   (page, kv head), and the pages' mean keys.
//  * gqa_prologue   both in one launch.
//
// Built with -ffp-contract=off: the codes, scales and summaries are mirrored
// bit for bit by the CPU oracle.
#include <algorithm>

#include "ekv_gqa.h"
#include "ekv_rows.h"

namespace ekv {

// ---------------------------------------------------------------------------
// qk_norm_rope:  y = rot(x * rsqrt(mean x^2 + eps) * w).
//
// LPR lanes hold a row (8 channels, one 16-byte load, each), so the norm's sum
// and the rotation's partners are shuffles; a lane group takes `batch` heads of
// one token, with the token's cos / sin and the weights in registers.  Bound by
// memory: each row is read once and written once (8,191 tokens of 72 heads of
// 256: 606 MB in 128 us, 4.7 TB/s, a large copy's rate); a decode step's 64
// tokens take 4.4 us, which is the launch and one trip to memory.
// ---------------------------------------------------------------------------
struct NormSide {
  const uint16_t* x;  // bf16 at x + t * tok_stride + h * head_stride
  int64_t tok_stride, head_stride;
  const void* w;      // [D] fp32 or bf16; null: rotation only
  int32_t w_bf16;
  int32_t heads;
  int32_t aligned;    // rows start at 16-byte addresses
  uint16_t* out;      // [T, heads, D]
};

struct NormArgs {
  NormSide side[2];   // q, k
  int32_t num_tokens, dim, batch;
  float eps;
  RopeArgs rope;
  const int64_t* positions;
};

__device__ __forceinline__ void load_row8(const uint16_t* p, bool aligned, float (&v)[8]) {
  if (aligned) {
    unpack_bf16x8(*reinterpret_cast<const uint4*>(p), v);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = bf16_to_f32(p[i]);
  }
}

__device__ __forceinline__ uint4 load_raw8(const uint16_t* p, bool aligned) {
  if (aligned) return *reinterpret_cast<const uint4*>(p);
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) w[i] = p[2 * i] | static_cast<uint32_t>(p[2 * i + 1]) << 16;
  return make_uint4(w[0], w[1], w[2], w[3]);
}

__device__ __forceinline__ float row_max8(uint4 w, float top) {
  float v[8];
  unpack_bf16x8(w, v);
#pragma unroll
  for (int i = 0; i < 8; ++i) top = fmaxf(top, fabsf(v[i]));
  return top;
}

__device__ __forceinline__ void load_weight8(const void* w, int is_bf16, int j, float (&v)[8]) {
  if (is_bf16) {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = bf16_to_f32(static_cast<const uint16_t*>(w)[8 * j + i]);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = static_cast<const float*>(w)[8 * j + i];
  }
}

__host__ __device__ __forceinline__ int64_t norm_units(const NormArgs& a, int s) {
  return static_cast<int64_t>(a.num_tokens) * ((a.side[s].heads + a.batch - 1) / a.batch);
}

// Rows of lane group `unit`; units past the last take part in the shuffles only.
template <int LPR>
__device__ __forceinline__ void norm_unit(const NormArgs& a, int64_t unit, int64_t q_units, int64_t units) {
  const int j = static_cast<int>(threadIdx.x) & (LPR - 1);
  const bool live = unit < units;
  if (!live) unit = units - 1;
  const bool is_k = unit >= q_units;
  const NormSide& s = a.side[is_k];
  if (is_k) unit -= q_units;
  const int per = (s.heads + a.batch - 1) / a.batch;
  const int64_t t = unit / per;
  const int h0 = static_cast<int>(unit - t * per) * a.batch;
  const bool in = live && 8 * j < a.dim;
  float w[8], c[8], sn[8];
  if (s.w && 8 * j < a.dim) load_weight8(s.w, s.w_bf16, j, w);
  rope_factors(a.rope, a.positions[t], j, c, sn);
  // the wave's groups may have different head counts left: all run the same rounds
  for (int b = 0; b < a.batch; ++b) {
    const int h = h0 + b;
    const bool have = in && h < s.heads;
    float v[8] = {};
    if (have) load_row8(s.x + t * s.tok_stride + h * s.head_stride + 8 * j, s.aligned, v);
    if (s.w) row_rms_norm<LPR>(v, w, a.dim, a.eps);
    row_rope<LPR>(v, a.rope, j, c, sn);
    if (have) {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = bf16_to_f32(f32_to_bf16(v[i]));
      *reinterpret_cast<uint4*>(s.out + (t * s.heads + h) * a.dim + 8 * j) = pack_bf16x8(v);
    }
  }
}

template <int LPR>
__global__ void __launch_bounds__(256) qk_norm_rope_kernel(NormArgs a) {
  const int64_t q_units = norm_units(a, 0), units = q_units + norm_units(a, 1);
  norm_unit<LPR>(a, static_cast<int64_t>(blockIdx.x) * (256 / LPR) + threadIdx.x / LPR, q_units, units);
}

// ---------------------------------------------------------------------------
// gqa_append: one workgroup per (sequence, page that the call writes, kv head).
// It owns the page's head, so scales, codes and summary need no other one and
// no order of workgroups shows in the bytes.
//
// Long calls are bound by memory (16 x 8,192 tokens of 8 kv heads of 128 with
// summaries: 808 MB in 180 us, 4.5 TB/s; a large copy 4.7); a decode step by a
// chain of dependent reads (offset, position, page id, scale) and by whole
// 64-byte lines of V for one token's byte in each (64 tokens, 8 kv heads of
// 128: 7.2 us, 8.6 with the key's norm and rotation).
// ---------------------------------------------------------------------------
struct GqaAppendArgs {
  const uint16_t *k, *v;    // bf16 rows at + t * tok_stride + h * head_stride
  int64_t k_tok_stride, k_head_stride, v_tok_stride, v_head_stride;
  int32_t k_aligned, v_aligned;
  int32_t kv_heads, num_tokens;
  const int64_t* positions; // [T]; a sequence's tokens at consecutive positions
  const int32_t* qsl;       // [B + 1]
  int32_t num_seqs, page_slots;  // most pages a sequence's rows touch
  int32_t slots;            // 0: page_slots a sequence; else a sequence's slots follow its tokens
  const int32_t* block_table;
  int64_t bt_stride;
  int32_t bt_width;
  uint8_t* cache;
  int64_t page_stride, num_pages;
  uint8_t* summary;         // null: none
  int64_t summary_stride;
  // key prep (prologue): RMS norm by k_w (null: none) and rotation, rounded to bf16
  int32_t prep;
  const void* k_w;
  int32_t k_w_bf16;
  float eps;
  RopeArgs rope;
};

// Lanes 32 .. 63 of x change places with lanes 0 .. 31 of y.
__device__ __forceinline__ void swap32(uint32_t& x, uint32_t& y) {
  const auto r = __builtin_amdgcn_permlane32_swap(x, y, false, false);
  x = r[0], y = r[1];
}
// Lanes 16 .. 31 (48 .. 63) of x change places with lanes 0 .. 15 (32 .. 47) of y.
__device__ __forceinline__ void swap16(uint32_t& x, uint32_t& y) {
  const auto r = __builtin_amdgcn_permlane16_swap(x, y, false, false);
  x = r[0], y = r[1];
}

// A key row of L lanes with E pieces of 8 channels each: norm and rotation as
// qk_norm_rope has them, sums and products in the same order.
template <int L, int E>
__device__ __forceinline__ void prep_key(float (&v)[E][8], const GqaAppendArgs& a, const float (&w)[E][8], int64_t pos,
                                         int j) {
  if (a.k_w) {
    float s[E];
#pragma unroll
    for (int e = 0; e < E; ++e) {
      s[e] = 0.0f;
#pragma unroll
      for (int i = 0; i < 8; ++i) s[e] = __fmaf_rn(v[e][i], v[e][i], s[e]);
#pragma unroll
      for (int m = L >> 1; m > 0; m >>= 1) s[e] += __shfl_xor(s[e], m, 64);
    }
    const float sum = E == 2 ? s[0] + s[E - 1] : s[0];
    const float r = 1.0f / sqrtf(sum / static_cast<float>(8 * L * E) + a.eps);
#pragma unroll
    for (int e = 0; e < E; ++e) {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[e][i] = v[e][i] * r * w[e][i];
    }
  }
  float c[E][8], s[E][8];
#pragma unroll
  for (int e = 0; e < E; ++e) rope_factors(a.rope, pos, E * j + e, c[e], s[e]);
  if constexpr (E == 1) {
    row_rope<L>(v[0], a.rope, j, c[0], s[0]);
  } else if (a.rope.interleaved) {
#pragma unroll
    for (int e = 0; e < E; ++e) row_rope<L>(v[e], a.rope, E * j + e, c[e], s[e]);
  } else {  // the partner is a piece of this lane or another one
    const int hop = a.rope.rope >> 4, lane = static_cast<int>(threadIdx.x) & 63;
    float y[E][8];
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const int q = E * j + e, at = 8 * q - a.rope.offset;
      const bool in = at >= 0 && at < a.rope.rope, low = at < (a.rope.rope >> 1);
      const int from = in ? (low ? q + hop : q - hop) : q;
      const int src = (lane & ~(L - 1)) + from / E;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float p0 = __shfl(v[0][i], src, 64), p1 = __shfl(v[E - 1][i], src, 64);
        const float p = from % E ? p1 : p0;
        y[e][i] = low ? v[e][i] * c[e][i] - p * s[e][i] : v[e][i] * c[e][i] + p * s[e][i];
      }
    }
#pragma unroll
    for (int e = 0; e < E; ++e) {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[e][i] = y[e][i];
    }
  }
}

// Four dwords of four bytes -> out[k] holds byte k of each.
__device__ __forceinline__ void transpose4(const uint32_t (&a)[4], uint32_t (&out)[4]) {
  const uint32_t l0 = __builtin_amdgcn_perm(a[1], a[0], 0x05010400u), h0 = __builtin_amdgcn_perm(a[1], a[0], 0x07030602u);
  const uint32_t l1 = __builtin_amdgcn_perm(a[3], a[2], 0x05010400u), h1 = __builtin_amdgcn_perm(a[3], a[2], 0x07030602u);
  out[0] = __builtin_amdgcn_perm(l1, l0, 0x05040100u), out[1] = __builtin_amdgcn_perm(l1, l0, 0x07060302u);
  out[2] = __builtin_amdgcn_perm(h1, h0, 0x05040100u), out[3] = __builtin_amdgcn_perm(h1, h0, 0x07060302u);
}

__device__ __forceinline__ uint32_t fp8x4_codes(float a, float b, float c, float d) {
  return f32x2_to_fp8(a, b) | f32x2_to_fp8(c, d) << 16;
}

// Codes times a power of two, coded again.
__device__ __forceinline__ uint32_t fp8x4_scaled(uint32_t w, float r) {
  const f32x4 x = fp8x4_to_f32(w) * r;
  return fp8x4_codes(x[0], x[1], x[2], x[3]);
}

// Lane (i, j) of wave g holds 8 E channels of the tokens 16 t + 4 g + i, t = 0 ..
// 3: V's 16 bytes of (channel, g) lie in the four lanes i of a wave, which hand
// each other dwords by two swaps of half waves and half halves, and turn bytes
// in registers; a whole page's bytes pass through LDS once more, so that they
// leave as whole lines.
template <int D>
struct AppendShape {
  static constexpr int kLanes = D == 64 ? 8 : 16;    // lanes of a row
  static constexpr int kChunks = D == 256 ? 2 : 1;   // 8-channel pieces of a lane
  static constexpr int kThreads = D == 64 ? 128 : 256;
};

template <int D>
__device__ void gqa_append_block(const GqaAppendArgs& a, int block) {
  constexpr int L = AppendShape<D>::kLanes, E = AppendShape<D>::kChunks, kWaves = AppendShape<D>::kThreads / 64;
  __shared__ float red[2][kWaves];
  __shared__ float sums[4][D];
  __shared__ __attribute__((aligned(16))) uint8_t tile[D * kPageTokens];
  const int tid = static_cast<int>(threadIdx.x), lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int j = lane & (L - 1), i = lane >> 4, g = D == 64 ? 2 * wave + ((lane >> 3) & 1) : wave;
  const int h = block % a.kv_heads;
  int slot = block / a.kv_heads, b;
  if (a.slots) {
    // n tokens lie on at most n / 64 + 2 pages
    b = slot_seq(a.qsl, a.num_seqs, a.num_tokens, slot, [](int t, int i) { return t / kPageTokens + 2 * i; }, slot);
    if (b < 0 || slot >= a.page_slots) return;
  } else {
    b = slot / a.page_slots, slot %= a.page_slots;
  }
  const int t0 = a.qsl[b], n = min(a.qsl[b + 1], a.num_tokens) - t0;
  if (t0 < 0 || n <= 0) return;
  const int64_t p0 = a.positions[t0];
  if (p0 < 0) return;
  const int64_t lp = p0 / kPageTokens + slot, base = lp * kPageTokens;
  const int first = static_cast<int>(max(p0 - base, static_cast<int64_t>(0)));
  const int end = static_cast<int>(min(p0 + n - base, static_cast<int64_t>(kPageTokens)));  // rows first .. end - 1
  if (end <= first || lp >= a.bt_width) return;
  const int64_t page = a.block_table[b * a.bt_stride + lp];
  const int64_t tok = t0 + base - p0;  // token of the page's row 0

  // the new rows, asked for beside the page's place; they stay packed
  uint4 kx[4][E], vx[4][E];
#pragma unroll
  for (int t = 0; t < 4; ++t) {
    const int r = 16 * t + 4 * g + i;
    const bool have = r >= first && r < end;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const int c = 8 * (E * j + e);
      kx[t][e] = vx[t][e] = make_uint4(0, 0, 0, 0);
      if (have) {
        kx[t][e] = load_raw8(a.k + (tok + r) * a.k_tok_stride + h * a.k_head_stride + c, a.k_aligned);
        vx[t][e] = load_raw8(a.v + (tok + r) * a.v_tok_stride + h * a.v_head_stride + c, a.v_aligned);
      }
    }
  }
  const bool live = page >= 0 && page < a.num_pages;
  uint8_t* const pg = a.cache + page * a.page_stride;
  uint8_t* const kp = pg + static_cast<int64_t>(h) * kPageTokens * D;
  uint8_t* const vp = pg + static_cast<int64_t>(a.kv_heads + h) * kPageTokens * D;
  float* const ks = reinterpret_cast<float*>(pg + 2ll * a.kv_heads * kPageTokens * D) + h;
  float* const vs = ks + a.kv_heads;
  float kold = 0.0f, vold = 0.0f;
  if (live && first) kold = *ks, vold = *vs;

  if (a.prep) {
    float w[E][8];
    if (a.k_w) {
#pragma unroll
      for (int e = 0; e < E; ++e) load_weight8(a.k_w, a.k_w_bf16, E * j + e, w[e]);
    }
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      const int r = 16 * t + 4 * g + i;
      const bool have = r >= first && r < end;
      if (!__any(have)) continue;  // one token's row is one wave's: 64 tokens, 8 kv heads of 128: 10.9 -> 8.6 us
      float v[E][8];
#pragma unroll
      for (int e = 0; e < E; ++e) unpack_bf16x8(kx[t][e], v[e]);
      prep_key<L, E>(v, a, w, have ? base + r : -1, j);
#pragma unroll
      for (int e = 0; e < E; ++e) {
#pragma unroll
        for (int x = 0; x < 8; ++x) v[e][x] = have ? bf16_to_f32(f32_to_bf16(v[e][x])) : 0.0f;
        kx[t][e] = pack_bf16x8(v[e]);
      }
    }
  }
  float kmax = 0.0f, vmax = 0.0f;
#pragma unroll
  for (int t = 0; t < 4; ++t) {
#pragma unroll
    for (int e = 0; e < E; ++e) kmax = row_max8(kx[t][e], kmax), vmax = row_max8(vx[t][e], vmax);
  }
  kmax = wave_max_xor(kmax, 64);
  vmax = wave_max_xor(vmax, 64);
  if (lane == 0) red[0][wave] = kmax, red[1][wave] = vmax;
  __syncthreads();
  if (!live) return;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) kmax = fmaxf(kmax, red[0][w]), vmax = fmaxf(vmax, red[1][w]);
  const float knew = fmaxf(exp2i(pow2_exponent(kmax, kInv448)), kold);
  const float vnew = fmaxf(exp2i(pow2_exponent(vmax, kInv448)), vold);
  const bool kgrow = first && knew > kold, vgrow = first && vnew > vold;
  const float ki = 1.0f / knew, vi = 1.0f / vnew;  // powers of two: the products below are exact
  const float kr = kold * ki, vr = vold * vi;

  // K: rows as they are; earlier ones again in the larger scale.  sum: of the
  // stored codes' values over this lane's tokens, exact in fp32 in any order
  // (multiples of 2^-9 below 2^15).
  float sum[E][8] = {};
#pragma unroll
  for (int t = 0; t < 4; ++t) {
    const int r = 16 * t + 4 * g + i;
    uint8_t* const dst = kp + r * D + 8 * E * j;
    uint32_t kc[2 * E] = {};
    const bool have = r >= first && r < end, old = r < first && (kgrow || a.summary);
    if (have) {
#pragma unroll
      for (int e = 0; e < E; ++e) {
        float x[8];
        unpack_bf16x8(kx[t][e], x);
        kc[2 * e] = fp8x4_codes(x[0] * ki, x[1] * ki, x[2] * ki, x[3] * ki);
        kc[2 * e + 1] = fp8x4_codes(x[4] * ki, x[5] * ki, x[6] * ki, x[7] * ki);
      }
    } else if (old) {
#pragma unroll
      for (int e = 0; e < 2 * E; ++e) {
        kc[e] = reinterpret_cast<const uint32_t*>(dst)[e];
        if (kgrow) kc[e] = fp8x4_scaled(kc[e], kr);
      }
    }
    if (have || (old && kgrow)) {
      if constexpr (E == 2) *reinterpret_cast<uint4*>(dst) = make_uint4(kc[0], kc[1], kc[2], kc[3]);
      else *reinterpret_cast<uint2*>(dst) = make_uint2(kc[0], kc[1]);
    }
    if (a.summary) {
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const f32x4 lo = fp8x4_to_f32(kc[2 * e]), hi = fp8x4_to_f32(kc[2 * e + 1]);
#pragma unroll
        for (int x = 0; x < 4; ++x) sum[e][x] += lo[x], sum[e][4 + x] += hi[x];
      }
    }
  }

  // V: this lane ends with 4 channels (half of its pieces: i & 1) of the tokens
  // 16 t + 4 g + 0 .. 3 of two t (2 (i >> 1), + 1)
  uint32_t fresh[2], older[2], any = 0;  // bytes of its tokens that are new, or before them
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    fresh[u] = older[u] = 0;
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      const int r = 16 * (2 * (i >> 1) + u) + 4 * g + x;
      fresh[u] |= (r >= first) & (r < end) ? 0xffu << (8 * x) : 0u;
      older[u] |= r < first ? 0xffu << (8 * x) : 0u;
    }
    any |= fresh[u] | (vgrow ? older[u] : 0u);
  }
  const bool all_new = (fresh[0] & fresh[1]) == 0xffffffffu;
  const bool whole = first == 0 && end == kPageTokens;  // uniform
#pragma unroll
  for (int e = 0; e < E; ++e) {
    uint32_t x[4][2];  // [t][half]: four channels of this lane's token
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      float y[8];
      unpack_bf16x8(vx[t][e], y);
      x[t][0] = fp8x4_codes(y[0] * vi, y[1] * vi, y[2] * vi, y[3] * vi);
      x[t][1] = fp8x4_codes(y[4] * vi, y[5] * vi, y[6] * vi, y[7] * vi);
    }
#pragma unroll
    for (int s = 0; s < 2; ++s) {  // lower lanes: t = s from both halves of the wave; upper lanes: t = s + 2
#pragma unroll
      for (int half = 0; half < 2; ++half) swap32(x[s][half], x[s + 2][half]);
    }
    uint32_t y[2][4];  // [t][lane i]
#pragma unroll
    for (int s = 0; s < 2; ++s) {
#pragma unroll
      for (int k = 0; k < 2; ++k) {  // even 16 lanes: half 0 from both, odd ones: half 1
        swap16(x[s + 2 * k][0], x[s + 2 * k][1]);
        y[s][2 * k] = x[s + 2 * k][0], y[s][2 * k + 1] = x[s + 2 * k][1];
      }
    }
    uint32_t z[2][4];
    transpose4(y[0], z[0]);
    transpose4(y[1], z[1]);
    const int c0 = 8 * (E * j + e) + 4 * (i & 1), piece = 2 * g + (i >> 1);  // 8 bytes of a channel's 64
    uint8_t* const dst = vp + c0 * kPageTokens + 8 * piece;
    if (whole) {
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const int at = piece ^ ((c0 >> 3) & 7);  // channels 8 apart share banks
        *reinterpret_cast<uint2*>(tile + (c0 + c) * kPageTokens + 8 * at) = make_uint2(z[0][c], z[1][c]);
      }
    } else if (any) {
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        uint2 out = make_uint2(z[0][c], z[1][c]);
        if (!all_new) {
          uint2 was = *reinterpret_cast<const uint2*>(dst + c * kPageTokens);
          if (vgrow) {
            was.x = (was.x & ~older[0]) | (fp8x4_scaled(was.x, vr) & older[0]);
            was.y = (was.y & ~older[1]) | (fp8x4_scaled(was.y, vr) & older[1]);
          }
          out.x = (out.x & fresh[0]) | (was.x & ~fresh[0]);
          out.y = (out.y & fresh[1]) | (was.y & ~fresh[1]);
        }
        *reinterpret_cast<uint2*>(dst + c * kPageTokens) = out;
      }
    }
  }
  if (whole) {  // a channel's 64 bytes at a time
    __syncthreads();
    for (int u = tid; u < 4 * D; u += AppendShape<D>::kThreads) {
      const int c = u >> 2, s = (c >> 3) & 7;
      const uint4 w = *reinterpret_cast<const uint4*>(tile + c * kPageTokens + 16 * ((u & 3) ^ (s >> 1)));
      *reinterpret_cast<uint4*>(vp + 16 * u) = s & 1 ? make_uint4(w.z, w.w, w.x, w.y) : w;
    }
  }
  if (tid == 0) *ks = knew, *vs = vnew;

  if (a.summary) {  // uniform over the workgroup
#pragma unroll
    for (int e = 0; e < E; ++e) {
#pragma unroll
      for (int x = 0; x < 8; ++x) {
        float s = sum[e][x];
        s += __shfl_xor(s, 16, 64);
        s += __shfl_xor(s, 32, 64);
        if (i == 0) sums[g][8 * (E * j + e) + x] = s;
      }
    }
    __syncthreads();
    float mean = 0.0f;
    if (tid < D) mean = ((sums[0][tid] + sums[1][tid]) + (sums[2][tid] + sums[3][tid])) / static_cast<float>(end);
    float top = wave_max_xor(fabsf(mean), 64);
    if (lane == 0) red[0][wave] = top;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kWaves; ++w) top = fmaxf(top, red[0][w]);
    const float s = exp2i(pow2_exponent(top, kInv127));
    uint8_t* const rec = a.summary + page * a.summary_stride;
    if (tid < D) {
      const float q = fminf(fmaxf(rintf(mean / s), -127.0f), 127.0f);
      reinterpret_cast<int8_t*>(rec)[h * D + tid] = static_cast<int8_t>(q);
    }
    if (tid == 0) reinterpret_cast<float*>(rec + a.kv_heads * D)[h] = s * knew;
  }
}

template <int D>
__global__ void __launch_bounds__(AppendShape<D>::kThreads) gqa_append_kernel(GqaAppendArgs a) {
  gqa_append_block<D>(a, static_cast<int>(blockIdx.x));
}

// The append's workgroups first, whose chain of reads is the longest, then those
// of q's norm and rotation (16 x 8,192 tokens, 32 heads, 8 kv heads of 128:
// 2.96 GB in 700 us, 4.2 TB/s).
template <int D>
__global__ void __launch_bounds__(AppendShape<D>::kThreads) gqa_prologue_kernel(GqaAppendArgs a, NormArgs q, int append_blocks) {
  const int block = static_cast<int>(blockIdx.x);
  if (block < append_blocks) {
    gqa_append_block<D>(a, block);
  } else {
    const int64_t units = norm_units(q, 0);
    constexpr int kRows = AppendShape<D>::kThreads * 8 / D;
    norm_unit<D / 8>(q, static_cast<int64_t>(block - append_blocks) * kRows + threadIdx.x / (D / 8), units, units);
  }
}

// ---------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------
static bool row_aligned(const void* p, int64_t tok_stride, int64_t head_stride) {
  return aligned16(p) && tok_stride % 8 == 0 && head_stride % 8 == 0;
}

static const char* check_rope(const float* cos_sin, int32_t rows, int32_t rope, int32_t offset, int32_t dim) {
  if (!cos_sin && rope) return "cos_sin must not be null";
  if (rows < 0 || rope < 0 || rope % 16 || offset < 0 || offset % 8 || offset + rope > dim)
    return "rope must be a multiple of 16 and rope_offset of 8, inside the head";
  if (!aligned16(cos_sin)) return "cos_sin must be 16-byte aligned";
  return nullptr;
}

// Heads a lane group takes: as many as leave 8 workgroups of 4 waves a CU
// (2048), at most 8 (8,191 tokens of 72 heads of 256: 174 us at 1, 128 at 8, 131
// at 16; 32,768 of 128: 377, 228, 295).
static int norm_batch(int64_t rows, int rows_per_block) {
  int b = 1;
  while (b < 8 && rows / (static_cast<int64_t>(rows_per_block) * 2 * b) >= 2048) b *= 2;
  return b;
}

static int pow2_lanes(int dim) {
  int l = 2;
  while (8 * l < dim) l *= 2;
  return l;
}

template <int D>
static int launch_append_dim(const GqaAppendArgs& a, const NormArgs* q, hipStream_t s) {
  constexpr int kThreads = AppendShape<D>::kThreads, kRows = kThreads * 8 / D;
  const int64_t append = (a.slots ? a.slots : static_cast<int64_t>(a.num_seqs) * a.page_slots) * a.kv_heads;
  const int64_t blocks = append + (q ? (norm_units(*q, 0) + kRows - 1) / kRows : 0);
  EKV_CHECK(blocks * kThreads < (int64_t{1} << 32), "too many rows for one call");
  if (!blocks) return kOk;
  const dim3 grid(static_cast<uint32_t>(blocks));
  if (q) gqa_prologue_kernel<D><<<grid, kThreads, 0, s>>>(a, *q, static_cast<int>(append));
  else gqa_append_kernel<D><<<grid, kThreads, 0, s>>>(a);
  return ekv_launch_status();
}

static int launch_append(const GqaAppendArgs& a, const NormArgs* q, int dim, void* stream) {
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (dim == 64) return launch_append_dim<64>(a, q, s);
  if (dim == 128) return launch_append_dim<128>(a, q, s);
  return launch_append_dim<256>(a, q, s);
}

// Checks and fills what the append and the prologue share; empty calls leave num_seqs 0.
static int append_args(GqaAppendArgs& a, const uint16_t* k, int64_t k_tok_stride, int64_t k_head_stride,
                       const uint16_t* v, int64_t v_tok_stride, int64_t v_head_stride, int32_t num_tokens,
                       int32_t kv_heads, int32_t dim, const int64_t* positions, const int32_t* qsl, int32_t num_seqs,
                       int32_t max_query_len, const int32_t* block_table, int64_t bt_stride, int32_t bt_width,
                       uint8_t* cache, int64_t page_stride, int64_t num_pages, uint8_t* summary,
                       int64_t summary_stride) {
  EKV_CHECK(gqa_dim(dim), "dim must be 64, 128 or 256");
  EKV_CHECK(kv_heads > 0 && num_tokens >= 0 && num_seqs >= 0 && max_query_len >= 0, "negative sizes");
  a = GqaAppendArgs{};
  if (!num_tokens || !num_seqs || !max_query_len) return kOk;
  EKV_CHECK(k && v && positions && qsl && (block_table || !bt_width) && (cache || !num_pages), "null pointer");
  EKV_CHECK(bt_width >= 0 && num_pages >= 0, "negative sizes");
  EKV_CHECK(page_stride >= gqa_page_bytes(kv_heads, dim) && page_stride % 16 == 0 && aligned16(cache),
            "page_stride must be a multiple of 16 of at least kv_heads * (128 * dim + 8) bytes");
  EKV_CHECK(!summary || (summary_stride >= gqa_summary_bytes(kv_heads, dim) && summary_stride % 16 == 0 &&
                         aligned16(summary)),
            "summary_stride must be a multiple of 16 of at least kv_heads * (dim + 4) bytes");
  a.k = k, a.v = v;
  a.k_tok_stride = k_tok_stride, a.k_head_stride = k_head_stride;
  a.v_tok_stride = v_tok_stride, a.v_head_stride = v_head_stride;
  a.k_aligned = row_aligned(k, k_tok_stride, k_head_stride);
  a.v_aligned = row_aligned(v, v_tok_stride, v_head_stride);
  a.kv_heads = kv_heads, a.num_tokens = num_tokens;
  a.positions = positions, a.qsl = qsl, a.num_seqs = num_seqs;
  a.page_slots = (std::min(max_query_len, num_tokens) + kPageTokens - 2) / kPageTokens + 1;
  // Many sequences of unlike lengths: a slot for each page that the rows may
  // touch, not the longest one's for all (256 rows of one token and 8,192 of one
  // sequence, 8 kv heads of 128: 191 -> 42 us).
  const int64_t slots = num_tokens / kPageTokens + int64_t{2} * num_seqs;
  if (static_cast<int64_t>(num_seqs) * a.page_slots > 2 * slots) {
    EKV_CHECK(slots < (int64_t{1} << 31), "too many rows for one call");
    a.slots = static_cast<int32_t>(slots);
  }
  a.block_table = block_table, a.bt_stride = bt_stride, a.bt_width = bt_width;
  a.cache = cache, a.page_stride = page_stride, a.num_pages = num_pages;
  a.summary = summary, a.summary_stride = summary_stride;
  return kOk;
}

}  // namespace ekv

using namespace ekv;

extern "C" int64_t ekv_gqa_page_bytes(int32_t kv_heads, int32_t dim) {
  if (kv_heads <= 0 || !gqa_dim(dim)) return 0;
  return (gqa_page_bytes(kv_heads, dim) + 15) / 16 * 16;
}

extern "C" int64_t ekv_gqa_summary_bytes(int32_t kv_heads, int32_t dim) {
  if (kv_heads <= 0 || !gqa_dim(dim)) return 0;
  return (gqa_summary_bytes(kv_heads, dim) + 15) / 16 * 16;
}

extern "C" int ekv_qk_norm_rope(const uint16_t* q, int64_t q_tok_stride, int64_t q_head_stride, int32_t heads,
                                const uint16_t* k, int64_t k_tok_stride, int64_t k_head_stride, int32_t kv_heads,
                                int32_t num_tokens, int32_t dim, const void* q_w, const void* k_w, int32_t w_is_bf16,
                                float eps, const float* cos_sin, int32_t cos_sin_rows, int32_t rope,
                                int32_t rope_offset, int32_t interleaved, const int64_t* positions, uint16_t* q_out,
                                uint16_t* k_out, void* stream) {
  EKV_CHECK(dim >= 16 && dim <= 512 && dim % 16 == 0, "dim must be a multiple of 16, at most 512");
  EKV_CHECK(heads >= 0 && kv_heads >= 0 && num_tokens >= 0, "negative sizes");
  const char* bad = check_rope(cos_sin, cos_sin_rows, rope, rope_offset, dim);
  EKV_CHECK(!bad, bad);
  const int64_t rows = static_cast<int64_t>(num_tokens) * (static_cast<int64_t>(heads) + kv_heads);
  if (!rows) return kOk;
  EKV_CHECK((!heads || (q && q_out)) && (!kv_heads || (k && k_out)) && positions, "null pointer");
  EKV_CHECK(aligned16(q_out) && aligned16(k_out), "outputs must be 16-byte aligned");
  EKV_CHECK(aligned4(q_w) && aligned4(k_w), "weights must be 4-byte aligned");
  const int lpr = pow2_lanes(dim), per = 256 / lpr;
  NormArgs a{};
  a.side[0] = {q, q_tok_stride, q_head_stride, q_w, w_is_bf16, heads, row_aligned(q, q_tok_stride, q_head_stride), q_out};
  a.side[1] = {k, k_tok_stride, k_head_stride, k_w, w_is_bf16, kv_heads, row_aligned(k, k_tok_stride, k_head_stride),
               k_out};
  a.num_tokens = num_tokens, a.dim = dim, a.eps = eps;
  a.batch = norm_batch(rows, per);
  a.rope = {cos_sin, cos_sin_rows, rope, rope_offset, interleaved};
  a.positions = positions;
  const int64_t units = norm_units(a, 0) + norm_units(a, 1), blocks = (units + per - 1) / per;
  EKV_CHECK(blocks < (int64_t{1} << 24), "too many rows for one call");
  const dim3 grid(static_cast<uint32_t>(blocks));
  hipStream_t s = static_cast<hipStream_t>(stream);
  switch (lpr) {
    case 2: qk_norm_rope_kernel<2><<<grid, 256, 0, s>>>(a); break;
    case 4: qk_norm_rope_kernel<4><<<grid, 256, 0, s>>>(a); break;
    case 8: qk_norm_rope_kernel<8><<<grid, 256, 0, s>>>(a); break;
    case 16: qk_norm_rope_kernel<16><<<grid, 256, 0, s>>>(a); break;
    case 32: qk_norm_rope_kernel<32><<<grid, 256, 0, s>>>(a); break;
    default: qk_norm_rope_kernel<64><<<grid, 256, 0, s>>>(a); break;
  }
  return ekv_launch_status();
}

extern "C" int ekv_gqa_append(const uint16_t* k, int64_t k_tok_stride, int64_t k_head_stride, const uint16_t* v,
                              int64_t v_tok_stride, int64_t v_head_stride, int32_t num_tokens, int32_t kv_heads,
                              int32_t dim, const int64_t* positions, const int32_t* qsl, int32_t num_seqs,
                              int32_t max_query_len, const int32_t* block_table, int64_t bt_stride, int32_t bt_width,
                              uint8_t* cache, int64_t page_stride, int64_t num_pages, uint8_t* summary,
                              int64_t summary_stride, void* stream) {
  GqaAppendArgs a;
  const int rc = append_args(a, k, k_tok_stride, k_head_stride, v, v_tok_stride, v_head_stride, num_tokens, kv_heads,
                             dim, positions, qsl, num_seqs, max_query_len, block_table, bt_stride, bt_width, cache,
                             page_stride, num_pages, summary, summary_stride);
  if (rc || !a.num_seqs) return rc;
  return launch_append(a, nullptr, dim, stream);
}

extern "C" int ekv_gqa_prologue(const uint16_t* q, int64_t q_tok_stride, int64_t q_head_stride, int32_t heads,
                                const uint16_t* k, int64_t k_tok_stride, int64_t k_head_stride, const uint16_t* v,
                                int64_t v_tok_stride, int64_t v_head_stride, int32_t num_tokens, int32_t kv_heads,
                                int32_t dim, const void* q_w, const void* k_w, int32_t w_is_bf16, float eps,
                                const float* cos_sin, int32_t cos_sin_rows, int32_t rope, int32_t rope_offset,
                                int32_t interleaved, const int64_t* positions, const int32_t* qsl, int32_t num_seqs,
                                int32_t max_query_len, const int32_t* block_table, int64_t bt_stride,
                                int32_t bt_width, uint8_t* cache, int64_t page_stride, int64_t num_pages,
                                uint8_t* summary, int64_t summary_stride, uint16_t* q_out, void* stream) {
  GqaAppendArgs a;
  const int rc = append_args(a, k, k_tok_stride, k_head_stride, v, v_tok_stride, v_head_stride, num_tokens, kv_heads,
                             dim, positions, qsl, num_seqs, max_query_len, block_table, bt_stride, bt_width, cache,
                             page_stride, num_pages, summary, summary_stride);
  if (rc) return rc;
  const char* bad = check_rope(cos_sin, cos_sin_rows, rope, rope_offset, dim);
  EKV_CHECK(!bad, bad);
  EKV_CHECK(heads >= 0, "negative sizes");
  EKV_CHECK(aligned4(q_w) && aligned4(k_w), "weights must be 4-byte aligned");
  if (!num_tokens) return kOk;
  EKV_CHECK(positions && (!heads || (q && q_out && aligned16(q_out))), "null pointer or unaligned q_out");
  a.prep = 1, a.k_w = k_w, a.k_w_bf16 = w_is_bf16, a.eps = eps;
  a.rope = {cos_sin, cos_sin_rows, rope, rope_offset, interleaved};
  if (!a.num_seqs) a.kv_heads = 1, a.page_slots = 1;  // no append: q only
  NormArgs n{};
  n.side[0] = {q, q_tok_stride, q_head_stride, q_w, w_is_bf16, heads, row_aligned(q, q_tok_stride, q_head_stride), q_out};
  n.num_tokens = num_tokens, n.dim = dim, n.eps = eps, n.rope = a.rope, n.positions = positions;
  n.batch = norm_batch(static_cast<int64_t>(num_tokens) * heads, 2048 / dim);
  return launch_append(a, &n, dim, stream);
}
