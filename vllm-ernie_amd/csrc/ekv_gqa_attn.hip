// Causal attention of grouped-query layers over 8-bit pages: every page of a
// sequence (gqa_attention) or the pages a row selected (gqa_block_attention).
//
//   out = sum_j exp(s_j) v_j / (sum_j exp(s_j) + exp(sink)),  s_j = scale q . k_j
//   lse = log sum_j exp(s_j)
//
// over the tokens j a row sees: j <= position and, with a window,
// j > position - window.
#include <algorithm>
#include <type_traits>

#include "ekv_gqa.h"

namespace ekv {

constexpr float kLog2e = 0x1.715476p+0f;
constexpr float kLn2 = 0x1.62e430p-1f;
constexpr float kNone = -0x1.fffffep127f;  // reference of a row that has seen no token: no score is below it
// Weights are rounded to fp16 (11 bits, up to 65,504) for the product with V;
// as bf16 their rounding was the largest error of a result (1.4 times that of
// 32-bit weights, for 2% less time at 4,096 rows).  A reference lies 2^kLift
// below the largest score: weights of 2^-19 of the largest keep all bits, those
// down to 2^-30 some, and up to kMoveAt the reference stays (2^9 below it, and so
// moved sooner: 1% more time at 4,096 rows).
constexpr int kLift = 5;
constexpr float kMoveAt = 32768.0f; // weight, or sum of a lane's 16, that moves a row's reference
constexpr int kMaxSplits = 64;

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

struct GqaAttnArgs {
  const uint16_t* q;
  int64_t q_tok_stride, q_head_stride;
  int32_t q_aligned, num_tokens, heads, kv_heads, group;
  const uint8_t* cache;
  int64_t page_stride, num_pages;
  const int32_t* block_table;
  int64_t bt_stride;
  int32_t bt_width, num_seqs;
  const int64_t* positions;
  const int32_t* qsl;       // dense: [B + 1]
  const int32_t* req_ids;   // selected blocks: [T]
  const int32_t* ids;       // selected blocks: [T, kv_heads, n_ids] logical pages, -1 skipped
  int64_t ids_tok_stride, ids_head_stride;
  int32_t n_ids;
  int32_t share;            // neighbouring tokens whose lists a workgroup joins
  int32_t window;           // 0: none
  float scale_log2;
  const float* sinks;
  uint16_t* out;
  int64_t out_tok_stride, out_head_stride;
  float* lse;
  int64_t lse_stride;
  // plan
  int32_t tiles, units, splits, split_pages;  // units: (sequence, kv head, tile)
  int32_t by_rows;          // 1: many rows, `tiles` in all, a sequence's after those of the one before
  int32_t budget;           // 0, or the parts of a (kv head, tile) that its sequences share
  int32_t slots, part_step; // workgroups, and how far apart those of a unit are
  // 0, or of a call that both kernels share: sequences of up to `few` rows are the
  // one's of few rows (kind 0), the others the one's of many (kind 1)
  int32_t few, kind;
  int2* ws_rows;            // [T, heads]: first workgroup, parts | row of its tile << 8 | kind << 16
  float2* ws_ml;            // [slots, rows]: (reference in log2 units, sum)
  float* ws_o;              // [slots, rows, D]
};

// A workgroup's part of a unit.
struct GqaPart {
  int seq, h, tile;
  int part, parts, first;   // first: the workgroup of part 0
  int pages;                // of a part (static), or of the unit as far as known (dynamic)
};

// Which part of what workgroup i takes where up to 64 M sequences share the chip
// by their lengths: every workgroup finds the same smallest Q at which parts of
// Q pages fit the budget.  A sequence's length is taken from its last row, which
// decides the shares only.  Lane i holds the sequences M i .. M i + M - 1.
template <int M>
__device__ __forceinline__ bool find_part(const GqaAttnArgs& a, int i, GqaPart& p) {
  const int lane = static_cast<int>(threadIdx.x) & 63, per = a.kv_heads * a.tiles;
  int w[M];
#pragma unroll
  for (int k = 0; k < M; ++k) {
    const int b = M * lane + k;
    w[k] = 0;
    if (b >= a.num_seqs) continue;
    const int t0 = a.qsl[b], t1 = min(a.qsl[b + 1], a.num_tokens);
    if (t0 >= 0 && t1 > t0 && (!a.few || (t1 - t0) * a.group <= a.few)) {
      const int64_t pos = a.positions[t1 - 1];
      w[k] = static_cast<int>(min(max(pos, static_cast<int64_t>(0)) / kPageTokens + 1, static_cast<int64_t>(max(a.bt_width, 1))));
      if (a.window) w[k] = min(w[k], a.split_pages);  // the most pages a tile sees
    }
  }
  auto sum = [](const int (&v)[M]) {
    int x = v[0];
#pragma unroll
    for (int k = 1; k < M; ++k) x += v[k];
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) x += __shfl_xor(x, m, 64);
    return __builtin_amdgcn_readfirstlane(x);
  };
  const int all = sum(w);
  int q = max((all + a.budget - 1) / a.budget, 4), mine[M];
  if (M > 1) {
    // Nearly equal lengths of sequences that fill a round of the chip by
    // themselves (a budget of two parts each, rounded up) stay whole: 96 of
    // 8,192 tokens, 8 kv heads of 128: 293 -> 283 us, 266 in a grid of equal
    // parts.
    int longest = w[0], some[M];
#pragma unroll
    for (int k = 0; k < M; ++k) longest = max(longest, w[k]), some[k] = w[k] > 0;
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) longest = max(longest, __shfl_xor(longest, m, 64));
    const int count = sum(some);
    if (4ll * longest * count <= 5ll * all && 2 * a.budget < 5 * count) q = max(q, longest);
  }
  while (true) {
    const float inv = 1.0f / static_cast<float>(q);
#pragma unroll
    for (int k = 0; k < M; ++k)
      mine[k] = w[k] ? min(max(static_cast<int>(ceilf(static_cast<float>(w[k]) * inv)), 1), kMaxSplits) : 0;
    if (sum(mine) <= a.budget) break;  // reached: from the longest sequence on there is one part each
    q += (q >> 4) + 1;
  }
  int own = mine[0];
#pragma unroll
  for (int k = 1; k < M; ++k) own += mine[k];
  int upto = own;
#pragma unroll
  for (int m = 1; m < 64; m <<= 1) {
    const int x = __shfl_up(upto, m, 64);
    if (lane >= m) upto += x;
  }
  const int j = i / per, ht = i - j * per;
  const uint64_t at = __ballot(j < upto && j >= upto - own);
  if (!at) return false;
  const int holder = __builtin_ctzll(at);
  int before = __builtin_amdgcn_readlane(upto - own, holder);
#pragma unroll
  for (int k = 0; k < M; ++k) {
    const int parts = __builtin_amdgcn_readlane(mine[k], holder);
    if (j < before + parts) {
      p.seq = M * holder + k;
      p.h = ht % a.kv_heads, p.tile = ht / a.kv_heads;
      p.parts = parts, p.part = j - before, p.first = before * per + ht;
      p.pages = __builtin_amdgcn_readlane(w[k], holder);
      return true;
    }
    before += parts;
  }
  return false;
}

// 8 e4m3fn codes times a power of two -> bf16.
__device__ __forceinline__ bf16x8 fp8x8_to_bf16(uint32_t lo, uint32_t hi, float s) {
  const bf16x2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, s, false);
  const bf16x2 b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, s, true);
  const bf16x2 c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, s, false);
  const bf16x2 d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, s, true);
  return __builtin_bit_cast(bf16x8, make_uint4(__builtin_bit_cast(uint32_t, a), __builtin_bit_cast(uint32_t, b),
                                               __builtin_bit_cast(uint32_t, c), __builtin_bit_cast(uint32_t, d)));
}

// The same as fp16: exact while the power of two is 2^-15 to 2^7.
__device__ __forceinline__ f16x8 fp8x8_to_f16(uint32_t lo, uint32_t hi, float s) {
  const f16x2 a = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, s, false);
  const f16x2 b = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, s, true);
  const f16x2 c = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, s, false);
  const f16x2 d = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, s, true);
  return __builtin_bit_cast(f16x8, make_uint4(__builtin_bit_cast(uint32_t, a), __builtin_bit_cast(uint32_t, b),
                                              __builtin_bit_cast(uint32_t, c), __builtin_bit_cast(uint32_t, d)));
}

// The sums o are held in units of 2^at, in which a page's values are codes times
// 2^-15 to 2^7: most pages' scales are within that of the first one's.  A page
// whose scale is not moves the unit, and the sums with it; `top` is the largest
// scale so far, 2^64 below which no unit goes, as the sums would overflow (values
// of pages whose scale is below 2^-75 of that lose bits).
struct ValueUnit {
  int at = -1000, top = -1000;
};

// The power of two that V's codes of a page with scale vscale (wave-uniform) are
// taken by; a page of scale 0 holds zeros.
template <int NT, int DT>
__device__ __forceinline__ float value_factor(float vscale, ValueUnit& unit, f32x4 (&o)[NT][DT]) {
  const int e = (__builtin_bit_cast(int, vscale) >> 23) - 127;
  if (e == -127) return 0x1p-100f;
  if (e - unit.at < -15 || e - unit.at > 7) {
    unit.top = max(unit.top, e);
    const int to = max(e, unit.top - 64) + 4;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int d = 0; d < DT; ++d) {
#pragma unroll
        for (int i = 0; i < 4; ++i) o[nt][d][i] = __builtin_ldexpf(o[nt][d][i], unit.at - to);
      }
    }
    unit.at = to;
  }
  return exp2i(max(e - unit.at, -100));
}

// Sums and weights' sums as they are without units and lift.
template <int NT, int DT>
__device__ __forceinline__ void plain_units(const ValueUnit& unit, float (&l)[NT], f32x4 (&o)[NT][DT]) {
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    l[nt] *= exp2i(-kLift);
#pragma unroll
    for (int d = 0; d < DT; ++d) {
#pragma unroll
      for (int i = 0; i < 4; ++i) o[nt][d][i] = __builtin_ldexpf(o[nt][d][i], unit.at - kLift);
    }
  }
}

// 16 bytes at a page's scalar base + the lane's offset + a constant: buffer
// loads, so that a page's addresses take one register of a lane.
typedef __amdgpu_buffer_rsrc_t PageRsrc;
__device__ __forceinline__ PageRsrc page_rsrc(const uint8_t* base, uint32_t bytes) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(base), 0, static_cast<int>(bytes), 0x00027000);
}
__device__ __forceinline__ uint4 load16(PageRsrc r, uint32_t lane_at, uint32_t at) {
  return __builtin_bit_cast(uint4, __builtin_amdgcn_raw_buffer_load_b128(r, static_cast<int>(lane_at), static_cast<int>(at), 0));
}

__device__ __forceinline__ float lane_value(float v, int lane) {
  return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), lane));
}

// Result of a row whose weights sum to l around 2^kLift times the reference m: 4 channels.
__device__ __forceinline__ void store_out4(const GqaAttnArgs& a, int64_t t, int hq, int c, f32x4 o, float m, float l,
                                           float sink) {
  float den = l;
  if (a.sinks) den += __builtin_amdgcn_exp2f(sink * kLog2e - m - kLift);
  const float inv = den > 0.0f ? 1.0f / den : (den == den ? 0.0f : den);
  const uint32_t lo = __builtin_bit_cast(uint32_t, bf16x2{static_cast<__bf16>(o[0] * inv), static_cast<__bf16>(o[1] * inv)});
  const uint32_t hi = __builtin_bit_cast(uint32_t, bf16x2{static_cast<__bf16>(o[2] * inv), static_cast<__bf16>(o[3] * inv)});
  uint16_t* p = a.out + t * a.out_tok_stride + hq * a.out_head_stride + c;
  *reinterpret_cast<uint2*>(p) = make_uint2(lo, hi);
}

__device__ __forceinline__ void store_lse(const GqaAttnArgs& a, int64_t t, int hq, float m, float l) {
  if (a.lse) a.lse[t * a.lse_stride + hq] = l == 0.0f ? -__builtin_inff() : (m + (__builtin_amdgcn_logf(l) + kLift)) * kLn2;
}

// Rows of a wave's NT tiles of 16 queries: what each lane's row sees.
template <int NT>
struct RowRange {
  int pos[NT], lo[NT];        // the row sees lo .. pos
  int pmax, pmin, pany;       // of the wave's rows: last token, first of rows that see any, first of all
};

// Scores x (token 16 j + 4 g + i of the page, row n) -> weights around the
// rows' references m, as the B operand of the product with V, and their sums.
// kscale > 0 takes a raw score to log2 units.  A reference is a maximum that the
// row has had, less kLift, and moves only where the page's weights around it grow
// past kMoveAt.  kBySum sees that in their sums, which costs no maximum but the raw
// scores' registers (many rows, where the products bound the kernel: 3% less time
// at 4,096 rows); else in the largest score.  Masks are selects without branches.
template <bool kBySum, int NT, int DT>
__device__ __forceinline__ void softmax_page(f32x4 (&x)[NT][4], float kscale, bool whole, int first, int g,
                                             const RowRange<NT>& r, float (&m)[NT], float (&l)[NT],
                                             f32x4 (&o)[NT][DT], f16x8 (&w)[NT][2]) {
  if (!whole) {
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int from = r.lo[nt] - first - 4 * g, to = r.pos[nt] - first - 4 * g;  // seen: from <= 16 j + i <= to
#pragma unroll
      for (int j = 0; j < 4; ++j) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int at = 16 * j + i;
          x[nt][j][i] = (at >= from) & (at <= to) ? x[nt][j][i] : -__builtin_inff();
        }
      }
    }
  }
  float y[NT][16], s[NT], top[NT], most = 0.0f;
  auto largest = [&](int nt) {
    float t = x[nt][0][0];
#pragma unroll
    for (int i = 1; i < 16; ++i) t = fmaxf(t, x[nt][i >> 2][i & 3]);
    return t * kscale;
  };
  auto weights = [&](int nt) {
#pragma unroll
    for (int i = 0; i < 16; ++i) y[nt][i] = __builtin_amdgcn_exp2f(__builtin_fmaf(x[nt][i >> 2][i & 3], kscale, -m[nt]));
    float t[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) t[i] = y[nt][i] + y[nt][8 + i];
    s[nt] = ((t[0] + t[1]) + (t[2] + t[3])) + ((t[4] + t[5]) + (t[6] + t[7]));
  };
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    if (kBySum) {
      weights(nt);
      most = fmaxf(most, s[nt]);
    } else {
      top[nt] = largest(nt);
      most = fmaxf(most, __builtin_amdgcn_exp2f(top[nt] - m[nt]));
    }
  }
  if (__any(most > kMoveAt)) {  // infinite too: a row's first page, whose reference is none
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      float t = fmaxf((kBySum ? largest(nt) : top[nt]) - kLift, m[nt]);
      t = fmaxf(t, __shfl_xor(t, 16, 64));
      t = fmaxf(t, __shfl_xor(t, 32, 64));
      const float f = __builtin_amdgcn_exp2f(m[nt] - t);
      m[nt] = t;
      l[nt] *= f;
#pragma unroll
      for (int d = 0; d < DT; ++d) o[nt][d] *= f;
      if (kBySum) weights(nt);
    }
  }
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    if (!kBySum) weights(nt);
    l[nt] += s[nt];
#pragma unroll
    for (int i = 0; i < 16; ++i) w[nt][i >> 3][i & 7] = static_cast<_Float16>(y[nt][i]);
  }
}

// The bytes of V group g that belong to tokens low .. last of the page at
// `first`: what lies outside may be anything, NaN codes too.
__device__ __forceinline__ uint4 v_keep(int first, int low, int last, int g) {
  uint32_t keep[4];
#pragma unroll
  for (int t = 0; t < 4; ++t) {
    keep[t] = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int tok = first + 16 * t + 4 * g + i;
      keep[t] |= (tok <= last) & (tok >= low) ? 0xffu << (8 * i) : 0u;
    }
  }
  return make_uint4(keep[0], keep[1], keep[2], keep[3]);
}

__device__ __forceinline__ uint4 and4(uint4 a, uint4 b) { return make_uint4(a.x & b.x, a.y & b.y, a.z & b.z, a.w & b.w); }

// What the rows r0 .. of NT tiles see (flattened (token, head of the group) from
// token t0 on).
template <int NT>
__device__ __forceinline__ void load_ranges(const GqaAttnArgs& a, int t0, int r0, int rows, int n, RowRange<NT>& rr) {
  rr.pmax = -1, rr.pmin = 0x7fffffff, rr.pany = 0x7fffffff;
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    const int r = r0 + 16 * nt + n;
    rr.pos[nt] = 0x7fffffff;  // no row: unmasked zeros, never stored
    if (r < rows) {
      const int p = static_cast<int>(min(max(a.positions[t0 + r / a.group], static_cast<int64_t>(-1)),
                                         static_cast<int64_t>(0x3fffffff)));
      rr.pos[nt] = p;
      rr.pmax = max(rr.pmax, p);
      rr.pany = min(rr.pany, p);
      if (p >= 0) rr.pmin = min(rr.pmin, p);
    }
    rr.lo[nt] = a.window ? rr.pos[nt] - a.window + 1 : 0;
  }
#pragma unroll
  for (int m = 1; m < 16; m <<= 1) {
    rr.pmax = max(rr.pmax, __shfl_xor(rr.pmax, m, 64));
    rr.pmin = min(rr.pmin, __shfl_xor(rr.pmin, m, 64));
    rr.pany = min(rr.pany, __shfl_xor(rr.pany, m, 64));
  }
  rr.pmax = __builtin_amdgcn_readfirstlane(rr.pmax);
  rr.pmin = __builtin_amdgcn_readfirstlane(rr.pmin);
  rr.pany = __builtin_amdgcn_readfirstlane(rr.pany);
}

// Row r's q from channel 16 g on (null where there is no row).  Piece (s, u), a
// lane's part of the B operand, is channels 64 s + 16 g + 8 u .. + 7: K's 16
// bytes of a lane hold the same channels.
__device__ __forceinline__ const uint16_t* q_row(const GqaAttnArgs& a, int t0, int h, int r, int rows, int g) {
  if (r >= rows) return nullptr;
  const int tok = r / a.group, hq = h * a.group + r - tok * a.group;
  return a.q + (t0 + tok) * a.q_tok_stride + hq * a.q_head_stride + 16 * g;
}

template <int S>
__device__ __forceinline__ void load_q(const GqaAttnArgs& a, const uint16_t* row, bf16x8 (&q)[2 * S]) {
#pragma unroll
  for (int f = 0; f < 2 * S; ++f) q[f] = bf16x8{};
  if (!row) return;
  if (a.q_aligned) {
#pragma unroll
    for (int f = 0; f < 2 * S; ++f)
      q[f] = __builtin_bit_cast(bf16x8, *reinterpret_cast<const uint4*>(row + 64 * (f >> 1) + 8 * (f & 1)));
  } else {
#pragma unroll
    for (int f = 0; f < 2 * S; ++f) {
      uint32_t w[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint16_t* p = row + 64 * (f >> 1) + 8 * (f & 1) + 2 * i;
        w[i] = p[0] | static_cast<uint32_t>(p[1]) << 16;
      }
      q[f] = __builtin_bit_cast(bf16x8, make_uint4(w[0], w[1], w[2], w[3]));
    }
  }
}

// The scales of lane i's page (page < 0: none) for head h, K's with the softmax
// scale in log2 units.  K's stays above zero, as a masked score needs it: the
// scale of a page that was never written in a cache of zeros is 0.
__device__ __forceinline__ void page_scales(const GqaAttnArgs& a, int h, int dim, int page, float& ks, float& vs) {
  ks = vs = 0.0f;
  if (page >= 0) {
    const float* sc = reinterpret_cast<const float*>(a.cache + page * a.page_stride +
                                                     2ll * a.kv_heads * kPageTokens * dim) + h;
    ks = fmaxf(sc[0] * a.scale_log2, 0x1p-126f), vs = sc[a.kv_heads];
  }
}

// Rows `from` .. rows - 1 of a sequence, which no workgroup takes (it has more than
// the call said), name no part: what a workspace holds of an earlier call is not
// this one's.
__device__ __forceinline__ void name_no_parts(const GqaAttnArgs& a, int t0, int h, int from, int rows, int step) {
  for (int r = from + static_cast<int>(threadIdx.x); r < rows; r += step)
    a.ws_rows[(t0 + r / a.group) * static_cast<int64_t>(a.heads) + h * a.group + r % a.group] = make_int2(0, a.kind << 16);
}

// ---------------------------------------------------------------------------
// Few rows a kv head: one workgroup per (16 NT rows, kv head, range of pages).
// Each of its W waves takes every W-th page of the range through registers,
// with no LDS in the loop: K as the A operand (16 tokens x 32 channels) against
// q leaves a lane the scores of one row and of the tokens whose V bytes it
// loads, so the weights go straight into the product with V.  The next page's K
// and V are asked for as soon as the products that read their registers are
// issued.  Lists of neighbouring rows may be joined: each page that any of them
// names is read once, and a mask says which rows it counts for.
//
// Bound by the read of the pages (32 rows of 64 heads at 131,072 tokens, 8 kv
// heads of 128: 8.6 GB in 1,412 us, 6.1 TB/s; 13 sequences of 2,000 to 48,000:
// 384 MB in 74 us, 5.2 TB/s); listed pages that rows share by their caches (333
// rows of 32 blocks, 4 kv heads: 698 MB in 73 us, 9.6 TB/s); a short context by
// one page's chain of reads (4,096 tokens: 6.5 us).
// ---------------------------------------------------------------------------
// What a workgroup's rows read: all pages, one token's list, or the joined lists
// of neighbouring tokens.
enum Pages { kDense, kList, kShared };
constexpr int kRange = 2048;     // pages that are joined at a time
constexpr int kShareIds = 256;   // longest lists that are joined

// Waves of a SIMD that the registers allow.
template <int D, int NT>
constexpr int kDecodeWaves = NT * D == 64 ? 4 : NT * D == 128 ? 3 : 2;

template <int D, int NT, int W, Pages P>
__global__ void __launch_bounds__(64 * W, (kDecodeWaves<D, NT>)) gqa_decode_kernel(GqaAttnArgs a) {
  constexpr int S = D / 64, DT = D / 16;
  constexpr bool LIST = P == kList, SHARE = P == kShared;
  __shared__ uint32_t row_mask[SHARE ? kRange : 1];  // of a page: the rows that list it
  __shared__ uint16_t joined[SHARE ? kRange : 1];    // listed pages in order
  __shared__ int counts[SHARE ? kRange / 64 : 1];
  __shared__ float so[W][16][D + 4];
  __shared__ float2 sml[W][16];
  const int tid = static_cast<int>(threadIdx.x), lane = tid & 63, n = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  GqaPart p;
  const bool dynamic = P == kDense && a.budget;
  if (dynamic) {
    if (!(a.num_seqs <= 64 ? find_part<1>(a, static_cast<int>(blockIdx.x), p) : find_part<4>(a, static_cast<int>(blockIdx.x), p)))
      return;
  } else {
    const int unit = static_cast<int>(blockIdx.x) % a.units;
    p.h = unit % a.kv_heads, p.tile = unit / a.kv_heads % a.tiles, p.seq = unit / a.kv_heads / a.tiles;
    p.part = static_cast<int>(blockIdx.x) / a.units, p.parts = a.splits, p.first = unit, p.pages = a.split_pages;
  }
  const int h = p.h, seq = p.seq;

  // the rows: (token, head of the group), flattened
  int t0, rows, b;
  if (LIST) {
    t0 = seq, rows = a.group, b = a.req_ids[seq];
    if (b < 0 || b >= a.num_seqs) return;
  } else if (SHARE) {
    t0 = seq * a.share, rows = min(a.share, a.num_tokens - t0) * a.group, b = 0;
  } else {
    b = seq, t0 = a.qsl[b];
    rows = (min(a.qsl[b + 1], a.num_tokens) - t0) * a.group;
    if (t0 < 0 || (a.few && rows > a.few)) return;
  }
  const int r0 = p.tile * 16 * NT;
  if (r0 >= rows) return;

  // lane i: the wave's i-th page of 64, its logical index and its place (-1:
  // none).  The first ones are asked for before the rows, whose positions and
  // q arrive together with them.
  const int32_t* bt = a.block_table + b * a.bt_stride;
  int base = 0;          // shared lists: first page of the range
  uint32_t listing = 0;  // and lane i's page: its row_mask
  auto list = [&](int e, int end, int& page) {
    int lp = -1;
    if (SHARE) {
      if (e < end) lp = joined[e];
      listing = lp >= 0 ? row_mask[lp] : 0;
      lp += lp >= 0 ? base : 0;
    } else if (e < end) {
      lp = LIST ? a.ids[t0 * a.ids_tok_stride + h * a.ids_head_stride + e] : e;
    }
    page = lp >= 0 && lp < a.bt_width ? bt[lp] : -1;
    return lp;
  };
  const bool early = LIST || (!SHARE && !a.window);
  int share = dynamic ? (p.pages + p.parts - 1) / p.parts : p.pages;
  int pb = p.part * share, pe = LIST ? a.n_ids : dynamic ? p.pages : a.bt_width;
  if (p.part < p.parts - 1) pe = min(pe, pb + share);
  int page, lp;
  if (early) lp = list(pb + wave + W * lane, pe, page);

  // q in registers where they are few, else in LDS (as operand pieces of 64 lanes)
  constexpr bool kQLds = NT * D >= 128;
  __shared__ bf16x8 sq[kQLds ? NT * S * 2 * 64 : 1];
  bf16x8 q[kQLds ? 1 : NT][2 * S];
  if constexpr (kQLds) {
    if (wave < NT) {
      load_q<S>(a, q_row(a, t0, h, r0 + 16 * wave + n, rows, g), q[0]);
#pragma unroll
      for (int f = 0; f < 2 * S; ++f) sq[64 * (wave * 2 * S + f) + lane] = q[0][f];
    }
  } else {
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) load_q<S>(a, q_row(a, t0, h, r0 + 16 * nt + n, rows, g), q[nt]);
  }
  RowRange<NT> rr;
  load_ranges<NT>(a, t0, r0, rows, n, rr);
  if constexpr (kQLds) __syncthreads();
  const int pmax = rr.pmax;
  const int low = a.window && pmax >= 0 ? max(rr.pmin - a.window + 1, 0) : 0;  // first token any row sees
  bool listed = early;
  if (P == kDense) {
    const int last = pmax < 0 ? 0 : min(pmax / kPageTokens + 1, a.bt_width), from = low / kPageTokens;
    if (dynamic) {
      listed = early && last == p.pages;
      share = (max(last - from, 0) + p.parts - 1) / p.parts;
    }
    pb = from + p.part * share;
    pe = p.part == p.parts - 1 ? last : min(pb + share, last);
  }

  f32x4 o[NT][DT] = {};
  float m[NT], l[NT];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) m[nt] = kNone, l[nt] = 0.0f;
  ValueUnit units;

  const uint8_t* const k_base = a.cache + static_cast<int64_t>(h) * kPageTokens * D;
  const uint32_t v_step = static_cast<uint32_t>(a.kv_heads) * kPageTokens * D;
  const uint32_t k_at = n * D + 16 * g, v_at = n * kPageTokens + 16 * g;
  auto load_k = [&](int pg, uint4 (&kr)[4][S]) {
    const PageRsrc r = page_rsrc(k_base + static_cast<int64_t>(pg) * a.page_stride, kPageTokens * D);
#pragma unroll
    for (int s = 0; s < S; ++s) {
#pragma unroll
      for (int j = 0; j < 4; ++j) kr[j][s] = load16(r, k_at + 64 * s, 16 * j * D);
    }
  };
  auto load_v = [&](int pg, uint4 (&vr)[DT]) {
    const PageRsrc r = page_rsrc(k_base + v_step + static_cast<int64_t>(pg) * a.page_stride, kPageTokens * D);
#pragma unroll
    for (int d = 0; d < DT; ++d) vr[d] = load16(r, v_at + 1024 * (d & 3), 4096 * (d >> 2));
  };

  int last_token = pmax;  // that the rows which read these pages see
  auto walk = [&](int pb, int pe) {
    for (int p0 = pb + wave; p0 < pe; p0 += 64 * W) {
      if (!listed || p0 != pb + wave) lp = list(p0 + W * lane, pe, page);
      if (page >= a.num_pages || lp * static_cast<int64_t>(kPageTokens) > last_token) page = -1;
      float ks, vs;
      page_scales(a, h, D, page, ks, vs);
      uint64_t todo = __ballot(page >= 0);
      if (!todo) continue;
      uint4 kr[4][S], vr[DT];
      int at = __builtin_ctzll(todo);
      load_k(__builtin_amdgcn_readlane(page, at), kr);
      load_v(__builtin_amdgcn_readlane(page, at), vr);
      while (true) {
        todo &= todo - 1;
        const int next = todo ? __builtin_ctzll(todo) : -1;
        const int next_page = __builtin_amdgcn_readlane(page, next < 0 ? at : next);
        const int first = __builtin_amdgcn_readlane(lp, at) * kPageTokens;
        const float kscale = lane_value(ks, at), vscale = lane_value(vs, at);

        f32x4 x[NT][4] = {};
#pragma unroll
        for (int s = 0; s < S; ++s) {
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const bf16x8 k0 = fp8x8_to_bf16(kr[j][s].x, kr[j][s].y, 1.0f), k1 = fp8x8_to_bf16(kr[j][s].z, kr[j][s].w, 1.0f);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
              const bf16x8 q0 = kQLds ? sq[64 * (nt * 2 * S + 2 * s) + lane] : q[kQLds ? 0 : nt][2 * s];
              const bf16x8 q1 = kQLds ? sq[64 * (nt * 2 * S + 2 * s + 1) + lane] : q[kQLds ? 0 : nt][2 * s + 1];
              x[nt][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(k0, q0, x[nt][j], 0, 0, 0);
              x[nt][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(k1, q1, x[nt][j], 0, 0, 0);
            }
            if (j & 1) __builtin_amdgcn_sched_barrier(0);  // few converted pieces at a time
          }
        }
        __builtin_amdgcn_sched_barrier(0);  // the next page goes to the registers that the products above read
        if (next >= 0) load_k(next_page, kr);
        __builtin_amdgcn_sched_barrier(0);
        const bool whole = first + kPageTokens - 1 <= rr.pany && (!a.window || first > pmax - a.window);
        if (SHARE) {
          const bool mine = (__builtin_amdgcn_readlane(listing, at) >> n) & 1;
#pragma unroll
          for (int j = 0; j < 4; ++j) {
#pragma unroll
            for (int i = 0; i < 4; ++i) x[0][j][i] = mine ? x[0][j][i] : -__builtin_inff();
          }
        }
        f16x8 w[NT][2];
        softmax_page<false, NT, DT>(x, kscale, whole, first, g, rr, m, l, o, w);
        const float vfactor = value_factor<NT, DT>(vscale, units, o);
        if (!whole) {
          const uint4 keep = v_keep(first, low, last_token, g);
#pragma unroll
          for (int d = 0; d < DT; ++d) vr[d] = and4(vr[d], keep);
        }
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int d = 0; d < DT; ++d) {
          const f16x8 v0 = fp8x8_to_f16(vr[d].x, vr[d].y, vfactor), v1 = fp8x8_to_f16(vr[d].z, vr[d].w, vfactor);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            o[nt][d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v0, w[nt][0], o[nt][d], 0, 0, 0);
            o[nt][d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v1, w[nt][1], o[nt][d], 0, 0, 0);
          }
          if (d & 1) __builtin_amdgcn_sched_barrier(0);
        }
        if (next < 0) break;
        __builtin_amdgcn_sched_barrier(0);
        load_v(next_page, vr);
        at = next;
      }
    }
  };
  if constexpr (!SHARE) {
    walk(pb, pe);
  } else {
    // Runs of tokens of one request, ranges of its pages, and, where a list names
    // a page again, its further mentions: the rows that list each page, and the
    // pages in order.  Every branch around a barrier is the whole workgroup's.
    const int toks = rows / a.group, entries = toks * a.n_ids;
    for (int s0 = 0, s1; s0 < toks; s0 = s1) {
      b = a.req_ids[t0 + s0];
      for (s1 = s0 + 1; s1 < toks && a.req_ids[t0 + s1] == b;) ++s1;
      if (b < 0 || b >= a.num_seqs) continue;
      bt = a.block_table + b * a.bt_stride;
      last_token = -1;  // of this run: what lies behind may be anything, and 0 NaN is no 0
      for (int i = s0; i < s1; ++i) {
        const int64_t last = min(a.positions[t0 + i], static_cast<int64_t>(0x3fffffff));
        last_token = max(last_token, static_cast<int>(max(last, static_cast<int64_t>(-1))));
      }
      const int np = last_token < 0 ? 0 : min(last_token / kPageTokens + 1, a.bt_width);
      for (base = 0; base < np; base += kRange) {
        const int here = min(kRange, np - base), groups = (here + 63) / 64;
        uint32_t left = 0xffffffffu;  // entries of this thread that are not in yet
        while (true) {
          for (int i = tid; i < 64 * groups; i += 64 * W) row_mask[i] = 0;
          __syncthreads();
          for (int i = 0, e = tid; e < entries; ++i, e += 64 * W) {
            const int tok = e / a.n_ids;
            if (!(left >> i & 1) || tok < s0 || tok >= s1) {
              left &= ~(1u << i);
              continue;
            }
            const int id = a.ids[(t0 + tok) * a.ids_tok_stride + h * a.ids_head_stride + e - tok * a.n_ids] - base;
            const uint32_t bits = ((1u << a.group) - 1) << (tok * a.group);
            if (id < 0 || id >= here || !(atomicOr(&row_mask[id], bits) & bits)) left &= ~(1u << i);
          }
          left &= entries > tid ? 0xffffffffu >> (31 - (entries - 1 - tid) / (64 * W)) : 0u;
          const int again = __syncthreads_or(left != 0);
          for (int c = wave; c < groups; c += W) {
            const int some = static_cast<int>(__builtin_popcountll(__ballot(row_mask[64 * c + lane] != 0)));
            if (lane == 0) counts[c] = some;
          }
          __syncthreads();
          int upto = lane < groups ? counts[lane] : 0;
#pragma unroll
          for (int k = 1; k < kRange / 64; k <<= 1) {
            const int v = __shfl_up(upto, k, 64);
            if (lane >= k) upto += v;
          }
          const int total = __builtin_amdgcn_readlane(upto, kRange / 64 - 1);
          for (int c = wave; c < groups; c += W) {
            const bool in = row_mask[64 * c + lane] != 0;
            const uint64_t all = __ballot(in);
            const int before = c ? __builtin_amdgcn_readlane(upto, c - 1) : 0;
            if (in) joined[before + __builtin_popcountll(all & ((1ull << lane) - 1))] = static_cast<uint16_t>(64 * c + lane);
          }
          __syncthreads();
          share = (total + p.parts - 1) / p.parts;
          walk(p.part * share, min((p.part + 1) * share, total));
          __syncthreads();
          if (!again) break;
        }
      }
    }
  }

  // the waves' parts of each row
  plain_units<NT, DT>(units, l, o);
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    l[nt] += __shfl_xor(l[nt], 16, 64);
    l[nt] += __shfl_xor(l[nt], 32, 64);
    if (nt) __syncthreads();
#pragma unroll
    for (int d = 0; d < DT; ++d) *reinterpret_cast<f32x4*>(&so[wave][n][16 * d + 4 * g]) = o[nt][d];
    if (g == 0) sml[wave][n] = make_float2(m[nt], l[nt]);
    __syncthreads();
    const int row = (tid >> 4) & 15, r = r0 + 16 * nt + row;
    if (r >= rows) continue;
    const int64_t t = t0 + r / a.group;
    if (SHARE && (a.req_ids[t] < 0 || a.req_ids[t] >= a.num_seqs)) continue;
    const int hq = h * a.group + r % a.group;
    const float sink = a.sinks ? a.sinks[hq] : 0.0f;
    float top = kNone, sum = 0.0f, f[W];
#pragma unroll
    for (int w = 0; w < W; ++w) top = fmaxf(top, sml[w][row].x);
#pragma unroll
    for (int w = 0; w < W; ++w) {
      f[w] = __builtin_amdgcn_exp2f(sml[w][row].x - top);
      sum += f[w] * sml[w][row].y;
    }
#pragma unroll
    for (int c = 4 * (tid & 15) + 64 * (tid >> 8); c < D; c += 16 * W) {
      f32x4 y = {};
#pragma unroll
      for (int w = 0; w < W; ++w) y += f[w] * *reinterpret_cast<const f32x4*>(&so[w][row][c]);
      if (p.parts == 1) store_out4(a, t, hq, c, y, top, sum, sink);
      else *reinterpret_cast<f32x4*>(a.ws_o + (static_cast<int64_t>(blockIdx.x) * (16 * NT) + 16 * nt + row) * D + c) = y;
    }
    if ((tid & 15) == 0 && tid < 256) {
      if (p.parts == 1) store_lse(a, t, hq, top, sum);
      else a.ws_ml[blockIdx.x * (16 * NT) + 16 * nt + row] = make_float2(top, sum);
      if (a.ws_rows && p.part == 0)
        a.ws_rows[t * a.heads + hq] = make_int2(p.first, p.parts | (16 * nt + row) << 8 | a.kind << 16);
    }
  }
  if (P == kDense && a.ws_rows && p.part == 0 && p.tile == a.tiles - 1) name_no_parts(a, t0, h, r0 + 16 * NT, rows, 64 * W);
}

// ---------------------------------------------------------------------------
// Many rows a kv head: one workgroup per (128 rows, kv head, range of pages).
// Its waves (4 of 32 rows; 8 of 16 at 256 channels, whose sums of 32 would leave
// one wave a SIMD: 1,490 -> 1,100 us at 2,048 rows) share every page: each brings
// its part of it, converted once (K to bf16, as q is, V to fp16, as the weights
// are), into LDS in the order of the operands (1 KB reads of 64 consecutive
// 16-byte pieces, no bank conflicts), while the page before is multiplied.
//
// Bound by the matrix cores and the weights' exponentials, which two waves a
// SIMD overlap in part (4,096 rows of 32 heads of 128 at 32,768 tokens: 1,784 to
// 1,844 us, 1,118 to 1,156 TFLOP/s, matrix cores busy 46% of the cycles; a
// product of 8,192^3 reaches 1,128 on the same card, of 16,384^3 1,350).  At 64
// channels the exponentials are half of the work (2,048 rows of 64 heads at
// 16,384: 810 TFLOP/s), at 256 there are more conversions a product (930).
// ---------------------------------------------------------------------------
template <int D>
struct PrefillShape {
  static constexpr int kWaves = D == 256 ? 8 : 4, kTiles = 8 / kWaves;  // 16-row tiles of a wave
};

template <int D>
__global__ void __launch_bounds__(64 * PrefillShape<D>::kWaves, 2) gqa_prefill_kernel(GqaAttnArgs a) {
  constexpr int W = PrefillShape<D>::kWaves, NT = PrefillShape<D>::kTiles;
  constexpr int S = D / 64, DT = D / 16, KT = 4 * S / W, VT = DT / W;  // pieces of K and V that a wave brings
  constexpr int kHalf = (8 * S + 2 * DT) * 64;  // 16-byte pieces of a page: K, then V
  extern __shared__ __attribute__((aligned(16))) uint8_t smem[];
  bf16x8* const buf = reinterpret_cast<bf16x8*>(smem);
  __shared__ int ranges[W][2];
  const int tid = static_cast<int>(threadIdx.x), lane = tid & 63, n = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int unit = static_cast<int>(blockIdx.x) % a.units, split = static_cast<int>(blockIdx.x) / a.units;
  const int h = unit % a.kv_heads, rest = unit / a.kv_heads;
  int b, tile;  // the longest rows first
  if (a.by_rows) {
    b = slot_seq(a.qsl, a.num_seqs, a.num_tokens, a.tiles - 1 - rest,
                 [&](int t, int i) { return static_cast<int>(static_cast<int64_t>(t) * a.group / 128) + i; }, tile);
    if (b < 0) return;
  } else {
    b = rest % a.num_seqs, tile = a.tiles - 1 - rest / a.num_seqs;
  }
  const int t0 = a.qsl[b];
  const int rows = (min(a.qsl[b + 1], a.num_tokens) - t0) * a.group;
  if (t0 < 0 || tile * 128 >= rows || (a.few && rows <= a.few)) return;
  const int r0 = tile * 128 + 16 * NT * wave;
  RowRange<NT> rr;
  bf16x8 q[NT][2 * S];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) load_q<S>(a, q_row(a, t0, h, r0 + 16 * nt + n, rows, g), q[nt]);
  load_ranges<NT>(a, t0, r0, rows, n, rr);
  if (lane == 0) ranges[wave][0] = rr.pmax, ranges[wave][1] = rr.pmin;
  __syncthreads();
  int pmax = -1, pmin = 0x7fffffff;
#pragma unroll
  for (int w = 0; w < W; ++w) pmax = max(pmax, ranges[w][0]), pmin = min(pmin, ranges[w][1]);
  pmax = __builtin_amdgcn_readfirstlane(pmax);
  pmin = __builtin_amdgcn_readfirstlane(pmin);
  const int low = a.window && pmax >= 0 ? max(pmin - a.window + 1, 0) : 0;
  const int wave_low = a.window && rr.pmax >= 0 ? max(rr.pmin - a.window + 1, 0) : 0;
  const int last = pmax < 0 ? 0 : min(pmax / kPageTokens + 1, a.bt_width);
  const int pb = low / kPageTokens + split * a.split_pages;
  const int pe = split == a.splits - 1 ? last : min(pb + a.split_pages, last);

  f32x4 o[NT][DT] = {};
  float m[NT], l[NT];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) m[nt] = kNone, l[nt] = 0.0f;
  ValueUnit units;

  // this wave's part of a page: pieces KT wave .. of K (S of each 16 tokens),
  // channels D / W wave .. of V
  const uint8_t* const k_base = a.cache + static_cast<int64_t>(h) * kPageTokens * D;
  const uint32_t v_step = static_cast<uint32_t>(a.kv_heads) * kPageTokens * D;
  const uint32_t k_at = (16 * (KT * wave / S) + n) * D + 64 * (KT * wave % S) + 16 * g;
  const uint32_t v_at = (D / W * wave + n) * kPageTokens + 16 * g;
  const int32_t* bt = a.block_table + b * a.bt_stride;
  uint4 kr[KT], vr[VT];

  for (int p0 = pb; p0 < pe; p0 += 64) {
    float ks, vs;
    int page = p0 + lane < pe ? bt[p0 + lane] : -1;
    if (page >= a.num_pages) page = -1;
    page_scales(a, h, D, page, ks, vs);
    uint64_t todo = __ballot(page >= 0);
    if (!todo) continue;
    auto fetch = [&](int at) {
      const uint8_t* pg = k_base + static_cast<int64_t>(__builtin_amdgcn_readlane(page, at)) * a.page_stride;
      const PageRsrc rk = page_rsrc(pg, kPageTokens * D), rv = page_rsrc(pg + v_step, kPageTokens * D);
#pragma unroll
      for (int s = 0; s < KT; ++s) kr[s] = load16(rk, k_at + 64 * s, 0);
#pragma unroll
      for (int i = 0; i < VT; ++i) vr[i] = load16(rv, v_at + 16 * i * kPageTokens, 0);
    };
    auto stage = [&](int at, int half) {
      bf16x8* const dst = buf + half * kHalf + lane;
      const int first = (p0 + at) * kPageTokens;
      const float vfactor = value_factor<NT, DT>(lane_value(vs, at), units, o);
#pragma unroll
      for (int s = 0; s < KT; ++s) {
        dst[((wave * KT + s) * 2) * 64] = fp8x8_to_bf16(kr[s].x, kr[s].y, 1.0f);
        dst[((wave * KT + s) * 2 + 1) * 64] = fp8x8_to_bf16(kr[s].z, kr[s].w, 1.0f);
      }
      if (first + kPageTokens - 1 > pmax || first < low) {
        const uint4 keep = v_keep(first, low, pmax, g);
#pragma unroll
        for (int i = 0; i < VT; ++i) vr[i] = and4(vr[i], keep);
      }
#pragma unroll
      for (int i = 0; i < VT; ++i) {
        dst[(8 * S + (wave * VT + i) * 2) * 64] = __builtin_bit_cast(bf16x8, fp8x8_to_f16(vr[i].x, vr[i].y, vfactor));
        dst[(8 * S + (wave * VT + i) * 2 + 1) * 64] = __builtin_bit_cast(bf16x8, fp8x8_to_f16(vr[i].z, vr[i].w, vfactor));
      }
    };
    int at = __builtin_ctzll(todo), half = 0;
    __syncthreads();  // the buffers of the 64 pages before
    fetch(at);
    stage(at, 0);
    while (at >= 0) {
      todo &= todo - 1;
      const int next = todo ? __builtin_ctzll(todo) : -1;
      __syncthreads();  // page `at` is whole in its half; the other half is read no more
      if (next >= 0) fetch(next);
      const int first = (p0 + at) * kPageTokens;
      if (first <= rr.pmax && first + kPageTokens > wave_low) {
        const bf16x8* const src = buf + half * kHalf + lane;
        f32x4 x[NT][4] = {};
        __builtin_amdgcn_s_setprio(1);
#pragma unroll
        for (int s = 0; s < 2 * S; ++s) {
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const bf16x8 k = src[(j * 2 * S + s) * 64];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
              x[nt][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(k, q[nt][s], x[nt][j], 0, 0, 0);
          }
        }
        __builtin_amdgcn_s_setprio(0);
        const bool whole = first + kPageTokens - 1 <= rr.pany && (!a.window || first > rr.pmax - a.window);
        f16x8 w[NT][2];
        softmax_page<true, NT, DT>(x, lane_value(ks, at), whole, first, g, rr, m, l, o, w);
        __builtin_amdgcn_s_setprio(1);
#pragma unroll
        for (int u = 0; u < 2; ++u) {
#pragma unroll
          for (int d = 0; d < DT; ++d) {
            const f16x8 v = __builtin_bit_cast(f16x8, src[(8 * S + 2 * d + u) * 64]);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
              o[nt][d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v, w[nt][u], o[nt][d], 0, 0, 0);
          }
        }
      }
      __builtin_amdgcn_s_setprio(0);
      if (next >= 0) stage(next, half ^ 1);
      at = next, half ^= 1;
    }
  }

  plain_units<NT, DT>(units, l, o);
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    l[nt] += __shfl_xor(l[nt], 16, 64);
    l[nt] += __shfl_xor(l[nt], 32, 64);
    const int r = r0 + 16 * nt + n;
    if (r >= rows) continue;
    const int64_t t = t0 + r / a.group;
    const int hq = h * a.group + r % a.group;
    const float sink = a.sinks ? a.sinks[hq] : 0.0f;
    const int64_t at = static_cast<int64_t>(blockIdx.x) * 128 + 16 * NT * wave + 16 * nt + n;
#pragma unroll
    for (int d = 0; d < DT; ++d) {
      if (a.splits == 1) store_out4(a, t, hq, 16 * d + 4 * g, o[nt][d], m[nt], l[nt], sink);
      else *reinterpret_cast<f32x4*>(a.ws_o + at * D + 16 * d + 4 * g) = o[nt][d];
    }
    if (g == 0) {
      if (a.splits == 1) store_lse(a, t, hq, m[nt], l[nt]);
      else a.ws_ml[at] = make_float2(m[nt], l[nt]);
      if (a.ws_rows && split == 0)
        a.ws_rows[t * a.heads + hq] = make_int2(unit, a.splits | (16 * (NT * wave + nt) + n) << 8 | a.kind << 16);
    }
  }
  if (a.ws_rows && split == 0 && !a.by_rows && tile == a.tiles - 1) name_no_parts(a, t0, h, (tile + 1) * 128, rows, 64 * W);
}

// Joins a row's parts: out = sum_p e^(m_p - m) o_p / sum_p e^(m_p - m) l_p, one
// wave per (token, head), lane s the s-th part's weight.  Bound by its launch and
// two trips to memory (4 to 6 us).
template <int D, bool LIST>
__global__ void __launch_bounds__(256) gqa_combine_kernel(GqaAttnArgs a, int slot_rows) {
  const int lane = static_cast<int>(threadIdx.x) & 63;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t t = row / a.heads;
  const int hq = static_cast<int>(row - t * a.heads);
  if (t >= a.num_tokens) return;
  const int2 info = a.ws_rows[row];
  const float sink = a.sinks ? a.sinks[hq] : 0.0f;
  const int lo = LIST ? a.req_ids[t] : a.qsl[0], hi = LIST ? a.num_seqs : a.qsl[a.num_seqs];
  if (LIST ? lo < 0 || lo >= hi : t < lo || t >= hi) return;
  const int parts = info.y & 255, at = (info.y >> 8) & 255;
  if (parts < 2 || info.y >> 16 != a.kind) return;  // whole already, no workgroup's, or the other kernel's
  // offsets that do not ascend may leave a row out; whatever the workspace holds, no read leaves it
  if (parts > kMaxSplits || at >= slot_rows || info.x < 0 || info.x + static_cast<int64_t>(parts - 1) * a.part_step >= a.slots)
    return;
  const int64_t first = static_cast<int64_t>(info.x) * slot_rows + at, step = static_cast<int64_t>(a.part_step) * slot_rows;
  float2 ml = make_float2(kNone, 0.0f);
  if (lane < parts) ml = a.ws_ml[first + lane * step];
  float top = ml.x;
#pragma unroll
  for (int m = 1; m < 64; m <<= 1) top = fmaxf(top, __shfl_xor(top, m, 64));
  const float f = __builtin_amdgcn_exp2f(ml.x - top);
  float sum = f * ml.y;
#pragma unroll
  for (int m = 1; m < 64; m <<= 1) sum += __shfl_xor(sum, m, 64);
  // eight parts in flight; the weight of one that saw nothing is 0
  const int c = 4 * (lane & (D / 4 - 1));
  f32x4 y = {};
  for (int s0 = 0; s0 < parts; s0 += 8) {
    f32x4 part[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      part[i] = f32x4{};
      if (s0 + i < parts) part[i] = *reinterpret_cast<const f32x4*>(a.ws_o + (first + (s0 + i) * step) * D + c);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) y += lane_value(f, s0 + i) * part[i];
  }
  if (4 * lane < D) store_out4(a, t, hq, c, y, top, sum, sink);
  if (lane == 0) store_lse(a, t, hq, top, sum);
}

// ---------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------
struct GqaPlan {
  int row_tiles;  // 16-row tiles of a workgroup: 1, 2, 4 in every wave, or 8 over its four (256 channels: eight) waves
  int tiles, splits, split_pages, budget;
  int64_t units, slots;  // slots: workgroups
  bool join, wide, by_rows;
};

// seqs: sequences (dense) or tokens (selected blocks); rows: query rows a kv
// head has in each at most, and in all; pages_of(n): the most pages that n
// consecutive rows see.
template <typename Pages>
static GqaPlan gqa_plan(int64_t seqs, int64_t rows, int64_t all_rows, int kv_heads, int dim, bool list, Pages pages_of,
                        bool whole_rounds = false) {
  GqaPlan p{};
  const int most = dim == 256 ? 1 : dim == 128 ? 2 : 4;
  // The kernel of few rows streams a page once for 16 row_tiles rows, what the
  // registers hold; the one of many rows from there on, in us: 16 sequences of
  // 16,384 tokens, 8 kv heads, 64 rows of 64 channels 62 and 97, of 128 channels
  // 140 and 145 (1 of 32,768: 28 and 35); at 72 rows of 128 184 and 149; at 256
  // channels 32 rows 262 and 268 (1 of 32,768: 37 and 53), 40 rows 331 and 272.
  p.row_tiles = rows <= 16 ? 1 : rows <= 32 ? std::min(2, most) : rows <= (dim == 256 ? 32 : 64) || list ? most : 8;
  p.tiles = static_cast<int>((rows + 16 * p.row_tiles - 1) / (16 * p.row_tiles));
  p.units = seqs * kv_heads * p.tiles;
  // Many sequences of unlike lengths: the tiles that their rows may need, not
  // the longest one's for all (256 rows of one token and 8,192 of one sequence,
  // 64 heads, 8 kv heads of 128: 2,068 -> 1,345 us).
  const int64_t tiles = all_rows / 128 + seqs;
  if (p.row_tiles == 8 && seqs * p.tiles > 2 * tiles && tiles < (int64_t{1} << 31)) {
    p.by_rows = true;
    p.tiles = static_cast<int>(tiles), p.units = kv_heads * tiles;
  }
  const int64_t pages = std::max<int64_t>(pages_of(std::min<int64_t>(rows, 16 * p.row_tiles)), 1);
  const int per_simd = p.row_tiles * dim == 64 ? 4 : p.row_tiles * dim == 128 ? 3 : 2;
  const int wide_waves = 4 * per_simd;
  if (p.row_tiles == 1 && pages > 4 && p.units <= 256 &&
      (pages <= wide_waves || (p.units > 128 && pages <= 6 * wide_waves))) {
    // One workgroup of all the waves that a CU holds to a unit, and no parts to
    // join, where a wave has one page or where units fill most of the chip.
    // 8 kv heads of 128, parts and their join against this, in us: 1 sequence
    // of 8 pages 9.1 and 7.7, of 16 pages 9.2 and 10.3, of 64 pages 10.5 and
    // 25.7; 64 listed pages of 16 tokens 43 and 47, of 17 tokens 49 and 48, of
    // 32 tokens 70 and 63 (with their selection); 32 sequences of 500 to 1,000
    // tokens 20 and 13.5, of 1,500 to 3,000 tokens 41 and 34.
    p.wide = true;
    p.splits = 1, p.split_pages = static_cast<int>(pages), p.slots = p.units;
    return p;
  }
  // workgroups that run at once
  const int64_t round = 256 * (p.row_tiles == 8 ? 2 : per_simd);
  if (!list && p.row_tiles < 8 && seqs > 1 && seqs <= 256 && pages > 8) {
    // Sequences of a dense call differ in length: their parts are shared out on
    // the device, one round of the chip, or as many as leave two parts a unit
    // (13 sequences of 2,000 to 48,000 tokens, 8 kv heads of 128: 82 us with
    // 2,048 equal parts of the longest one, 74 so; 128 of 500 to 32,768 tokens:
    // 482 and 385; 95 of 1,000 and one of 65,536: 411 and 74).
    p.slots = round * std::max<int64_t>((2 * p.units + round - 1) / round, 1);
    p.budget = static_cast<int>(p.slots / (kv_heads * static_cast<int64_t>(p.tiles)));
    p.split_pages = static_cast<int>(std::min<int64_t>(pages, 1 << 30));
    p.splits = 1;
    p.join = true;
    return p;
  }
  // One round of the chip (32 rows of 64 listed pages, 8 kv heads, in parts:
  // 52 us in 768 workgroups, 56 in 2,048).
  // Pages of a part.  Of many rows: 8 where units are fewer than CUs (4 sequences
  // of 4,096 tokens, 16 rows, 8 kv heads of 128: 37 us at 16, 31 at 8), longer
  // ones where each CU has one already (32 of 1,000: 50 us in two parts of 8, 35
  // in one), and 4 while such parts leave each a CU of its own.  At 4 and at 8, in
  // us: 56 units of 128 channels, 16 pages 25 and 29, 20 pages 28 and 28, 40
  // pages 44 and 37; 32 units, 32 pages 26 and 29, 64 pages 31 and 29; 8 units,
  // 128 pages 25 and 29, 256 pages 33 and 30; 16 units of 256 channels, 64 pages
  // 32 and 38, 80 pages 50 and 39; 1 unit of 64, 16 to 80 pages 14 to 16 and 18
  // to 19.  Up to 8 pages stay one part, without a join (56 units of 8: 22 and
  // 20; 8 units: 18 and 20).
  const int64_t least = p.row_tiles < 8 || (pages > 8 && p.units * ((pages + 3) / 4) <= 256) ? 4 : p.units < 256 ? 8 : 32;
  int64_t splits = std::min<int64_t>({(round + (whole_rounds ? 0 : p.units - 1)) / std::max<int64_t>(p.units, 1),
                                      (pages + least - 1) / least, kMaxSplits});
  splits = std::max<int64_t>(splits, 1);
  p.split_pages = static_cast<int>((pages + splits - 1) / splits);
  p.splits = static_cast<int>((pages + p.split_pages - 1) / p.split_pages);
  p.slots = p.units * p.splits;
  p.join = p.splits > 1;
  return p;
}

// A call's launches: `all`, or where chunks may stand beside single rows that see
// many pages, the kernel of few rows, in parts, for sequences of up to few_rows
// and `all` for the others.  Not where the kernel of many rows has parts of fewer
// than 128 pages by itself, whose walk costs about what a second launch does.
// 64 heads, 8 kv heads of 128, `all` against both, in us: 1 row at 131,072 tokens
// and a chunk of 512 2,885 and 191, 3 and four chunks of 512 3,060 and 455; 1 at
// 8,192 and 512 at 1,000 188 and 56; 1 at 8,192 and 512 there too 261 and 264; 1
// at 8,192 and 64 (parts of 16 pages) 55 and 71, 1 at 32,768 and 64 145 and 172.
struct GqaPlans {
  GqaPlan all, few;
  int few_rows;
  bool both;
};

// Rows of the sequences that go to the kernel of few rows: one tile of it, or two
// where a kv head's heads need them, or the mean rows of the others beside one
// chunk.  8 sequences and a chunk of 512, in us: 3 rows of 8 heads at 131,072
// tokens in the kernel of many rows (16 rows here) 1,494, in one tile of 32 515
// (single rows 505 in both); of 16 heads 1,516, in two tiles 434, but single rows
// 330 in one and 401 in two; at 256 channels, 65,536 tokens, 3 rows of 8 heads
// 1,193 and 700, single rows 582 and 722.
static int few_rows(int64_t tokens, int64_t seqs, int64_t max_rows, int group, int dim) {
  const int one = dim == 256 ? 16 : 32;
  const int64_t others = group * std::max<int64_t>((tokens - max_rows + seqs - 2) / std::max<int64_t>(seqs - 1, 1), 1);
  return others > one && others <= 2 * one ? 2 * one : group <= one ? one : group <= 2 * one ? 2 * one : 0;
}

static GqaPlans dense_plans(int64_t tokens, int64_t seqs, int64_t max_rows, int group, int kv_heads, int dim,
                            int64_t max_len, int64_t window) {
  auto pages = [&](int64_t rows) {
    const int64_t all = (max_len + kPageTokens - 1) / kPageTokens;
    const int64_t tokens = (rows + group - 1) / group + 1;  // of a tile that begins inside one
    return window ? std::min(all, (window + tokens - 2) / kPageTokens + 2) : all;
  };
  GqaPlans p{};
  p.all = gqa_plan(seqs, max_rows * group, tokens * group, kv_heads, dim, false, pages);
  p.few_rows = few_rows(tokens, seqs, max_rows, group, dim);
  // some sequence may have as few rows, of those that the call has in all
  const bool some = p.few_rows && tokens <= (seqs - 1) * max_rows + p.few_rows / group;
  p.both = p.all.row_tiles == 8 && some && pages(p.few_rows) >= 128 * p.all.splits;
  if (p.both) p.few = gqa_plan(seqs, p.few_rows, tokens * group, kv_heads, dim, false, pages);
  return p;
}

static GqaPlans block_plans(int64_t num_tokens, int group, int kv_heads, int dim, int64_t num_blocks) {
  GqaPlans p{};
  p.all = gqa_plan(num_tokens, group, num_tokens * group, kv_heads, dim, true, [&](int64_t) { return num_blocks; });
  return p;
}

// Tokens whose lists a workgroup joins: 16 rows of them, where these are four or
// more, their sequences have several such tiles and the tiles fill half of the
// chip.  Lists that agree in nothing but what chance and the forced pages give, 8
// kv heads of 128, apart and joined, with the selection, in us: 290 rows of 32
// pages at 6,000 tokens, 1 head a kv head, 134 and 64; 236 at 14,621, 2 heads, 113
// and 85; 256 at 131,072, 64 pages, 4 heads, 236 and 227.  Below: pairs (8 heads,
// 200 rows at 48,000) 110 and 123; few tiles (70 rows of 1 kv head) 21 and 28; at
// 64 channels a page's read is short against the joining (256 rows of 4 kv heads
// at 20,000, 2 heads) 36 and 44.
static int shared_tokens(int64_t num_tokens, int64_t num_seqs, int kv_heads, int group, int dim, int64_t num_blocks) {
  const int share = 16 / group;
  return share >= 4 && 16 % group == 0 && dim > 64 && num_blocks <= kShareIds &&
                 num_tokens >= std::max<int64_t>(64, 2 * share * num_seqs) && num_tokens / share * kv_heads >= 128
             ? share
             : 1;
}

static GqaPlans shared_plans(int64_t num_tokens, int share, int kv_heads, int dim, int64_t num_blocks) {
  GqaPlans p{};
  p.all = gqa_plan((num_tokens + share - 1) / share, 16, num_tokens, kv_heads, dim, true,
                   [&](int64_t) { return share * num_blocks; }, true);
  return p;
}

static int64_t rows_bytes(int64_t num_tokens, int64_t heads) { return (num_tokens * heads * 8 + 15) / 16 * 16; }

// The parts' sums of a launch.
static int64_t slots_bytes(const GqaPlan& p, int64_t dim) {
  return p.join ? p.slots * 16 * p.row_tiles * (dim + 2) * 4 : 0;
}

static int64_t plan_bytes(const GqaPlans& p, int64_t num_tokens, int64_t heads, int64_t dim) {
  const int64_t n = slots_bytes(p.all, dim) + (p.both ? slots_bytes(p.few, dim) : 0);
  return n ? rows_bytes(num_tokens, heads) + n : 0;
}

// The kernel of a plan.
template <int D, Pages P>
static int launch_parts(const GqaAttnArgs& a, int row_tiles, bool wide, int64_t blocks, hipStream_t s) {
  const dim3 grid(static_cast<uint32_t>(blocks));
  constexpr bool LIST = P != kDense;
  if constexpr (!LIST) {
    if (row_tiles == 8) {
      constexpr int kBytes = 2 * (D / 8 + D / 8) * 64 * 16;
      if (kBytes >= 65536)
        (void)hipFuncSetAttribute(reinterpret_cast<const void*>(gqa_prefill_kernel<D>),
                                  hipFuncAttributeMaxDynamicSharedMemorySize, kBytes);
      gqa_prefill_kernel<D><<<grid, 64 * PrefillShape<D>::kWaves, kBytes, s>>>(a);
    }
  }
  constexpr int kWide = 4 * kDecodeWaves<D, 1>;
  if (row_tiles == 1 && wide) gqa_decode_kernel<D, 1, kWide, P><<<grid, 64 * kWide, 0, s>>>(a);
  else if (row_tiles == 1) gqa_decode_kernel<D, 1, 4, P><<<grid, 256, 0, s>>>(a);
  if constexpr (D <= 128 && P != kShared) {
    if (row_tiles == 2) gqa_decode_kernel<D, 2, 4, P><<<grid, 256, 0, s>>>(a);
  }
  if constexpr (D == 64) {
    if (row_tiles == 4) gqa_decode_kernel<D, 4, 4, P><<<grid, 256, 0, s>>>(a);
  }
  return ekv_launch_status();
}

// The join of its parts.
template <int D, Pages P>
static int launch_join(const GqaAttnArgs& a, int row_tiles, hipStream_t s) {
  const int64_t rows = static_cast<int64_t>(a.num_tokens) * a.heads;
  gqa_combine_kernel<D, P != kDense><<<dim3(static_cast<uint32_t>((rows + 3) / 4)), 256, 0, s>>>(a, 16 * row_tiles);
  return ekv_launch_status();
}

template <Pages P>
static int launch_attn(GqaAttnArgs& a, const GqaPlans& plans, int dim, void* workspace, int64_t workspace_bytes,
                       void* stream) {
  // grids of fewer than 2^32 lanes
  const bool joins = plans.all.join || plans.few.join;
  EKV_CHECK(plans.all.slots < (1 << 23) && plans.few.slots < (1 << 23) &&
                (!joins || static_cast<int64_t>(a.num_tokens) * a.heads < (1 << 26)),
            "too many rows for one call");
  const int64_t need = plan_bytes(plans, a.num_tokens, a.heads, dim);
  if (need > workspace_bytes || (need && !workspace)) {
    set_error("workspace too small");
    return kWorkspaceTooSmall;
  }
  EKV_CHECK(!need || aligned16(workspace), "workspace must be 16-byte aligned");
  if (need) a.ws_rows = static_cast<int2*>(workspace);
  uint8_t* sums = static_cast<uint8_t*>(workspace) + rows_bytes(a.num_tokens, a.heads);
  hipStream_t s = static_cast<hipStream_t>(stream);
  auto by_dim = [&](auto run) {
    if constexpr (P != kShared) {
      if (dim == 64) return run(std::integral_constant<int, 64>{});
    }
    if (dim == 128) return run(std::integral_constant<int, 128>{});
    return run(std::integral_constant<int, 256>{});
  };
  auto parts = [&](const GqaPlan& p) {
    a.tiles = p.tiles, a.units = static_cast<int32_t>(p.units), a.splits = p.splits, a.split_pages = p.split_pages;
    a.budget = p.budget, a.by_rows = p.by_rows;
    if (p.join) {
      a.slots = static_cast<int32_t>(p.slots), a.part_step = p.budget ? a.kv_heads * p.tiles : a.units;
      a.ws_o = reinterpret_cast<float*>(sums);
      a.ws_ml = reinterpret_cast<float2*>(a.ws_o + p.slots * 16 * p.row_tiles * dim);
      sums += slots_bytes(p, dim);
    }
    return by_dim([&](auto d) { return launch_parts<d(), P>(a, p.row_tiles, p.wide, p.slots, s); });
  };
  auto join = [&](const GqaAttnArgs& of, const GqaPlan& p) {
    return p.join ? by_dim([&](auto d) { return launch_join<d(), P>(of, p.row_tiles, s); }) : kOk;
  };
  if (!plans.both) {
    const int rc = parts(plans.all);
    return rc ? rc : join(a, plans.all);
  }
  // joins last: by then each row says which kernel it is of
  a.few = plans.few_rows;
  int rc = parts(plans.few);
  const GqaAttnArgs few = a;
  a.kind = 1;
  if (!rc) rc = parts(plans.all);
  if (!rc) rc = join(few, plans.few);
  return rc ? rc : join(a, plans.all);
}

static int attn_args(GqaAttnArgs& a, const uint16_t* q, int64_t q_tok_stride, int64_t q_head_stride,
                     int32_t num_tokens, int32_t heads, int32_t kv_heads, int32_t dim, const uint8_t* cache,
                     int64_t page_stride, int64_t num_pages, const int32_t* block_table, int64_t bt_stride,
                     int32_t bt_width, const int64_t* positions, int32_t num_seqs, const float* sinks, float scale,
                     uint16_t* out, int64_t out_tok_stride, int64_t out_head_stride, float* lse, int64_t lse_stride) {
  EKV_CHECK(gqa_dim(dim), "dim must be 64, 128 or 256");
  EKV_CHECK(kv_heads > 0 && heads > 0 && heads % kv_heads == 0, "heads must be a multiple of kv_heads");
  EKV_CHECK(num_tokens >= 0 && num_seqs >= 0 && num_pages >= 0 && bt_width >= 0, "negative sizes");
  EKV_CHECK(scale > 0.0f && scale <= 0x1.fffffep127f, "scale must be positive and finite");
  a = GqaAttnArgs{};
  if (!num_tokens || !num_seqs) return kOk;
  EKV_CHECK(q && (cache || !num_pages) && (block_table || !bt_width) && positions && out, "null pointer");
  EKV_CHECK(page_stride >= gqa_page_bytes(kv_heads, dim) && page_stride % 16 == 0 && aligned16(cache),
            "page_stride must be a multiple of 16 of at least kv_heads * (128 * dim + 8) bytes");
  EKV_CHECK(aligned8(out) && out_tok_stride % 4 == 0 && out_head_stride % 4 == 0,
            "out rows must start at 8-byte addresses");
  EKV_CHECK(num_pages < (int64_t{1} << 31) && bt_width <= (1 << 24), "too many pages");
  a.q = q, a.q_tok_stride = q_tok_stride, a.q_head_stride = q_head_stride;
  a.q_aligned = aligned16(q) && q_tok_stride % 8 == 0 && q_head_stride % 8 == 0;
  a.num_tokens = num_tokens, a.heads = heads, a.kv_heads = kv_heads, a.group = heads / kv_heads;
  a.cache = cache, a.page_stride = page_stride, a.num_pages = num_pages;
  a.block_table = block_table, a.bt_stride = bt_stride, a.bt_width = bt_width, a.num_seqs = num_seqs;
  a.positions = positions, a.sinks = sinks, a.scale_log2 = scale * kLog2e;
  a.out = out, a.out_tok_stride = out_tok_stride, a.out_head_stride = out_head_stride;
  a.lse = lse, a.lse_stride = lse_stride;
  return kOk;
}

}  // namespace ekv

using namespace ekv;

extern "C" int64_t ekv_gqa_attention_workspace_size(int32_t num_tokens, int32_t num_seqs, int32_t max_query_len,
                                                    int32_t max_len, int32_t heads, int32_t kv_heads, int32_t dim,
                                                    int32_t window) {
  if (num_tokens <= 0 || num_seqs <= 0 || max_query_len <= 0 || kv_heads <= 0 || heads < kv_heads || !gqa_dim(dim) ||
      window < 0)
    return 0;
  const int64_t rows = std::min(max_query_len, num_tokens);
  return plan_bytes(dense_plans(num_tokens, num_seqs, rows, heads / kv_heads, kv_heads, dim, std::max(max_len, 0), window),
                    num_tokens, heads, dim);
}

extern "C" int ekv_gqa_attention(const uint16_t* q, int64_t q_tok_stride, int64_t q_head_stride, int32_t num_tokens,
                                 int32_t heads, int32_t kv_heads, int32_t dim, const uint8_t* cache,
                                 int64_t page_stride, int64_t num_pages, const int32_t* block_table,
                                 int64_t bt_stride, int32_t bt_width, const int64_t* positions, const int32_t* qsl,
                                 int32_t num_seqs, int32_t max_query_len, int32_t max_len, int32_t window,
                                 const float* sinks, float scale, uint16_t* out, int64_t out_tok_stride,
                                 int64_t out_head_stride, float* lse, int64_t lse_stride, void* workspace,
                                 int64_t workspace_bytes, void* stream) {
  GqaAttnArgs a;
  const int rc = attn_args(a, q, q_tok_stride, q_head_stride, num_tokens, heads, kv_heads, dim, cache, page_stride,
                           num_pages, block_table, bt_stride, bt_width, positions, num_seqs, sinks, scale, out,
                           out_tok_stride, out_head_stride, lse, lse_stride);
  if (rc) return rc;
  EKV_CHECK(max_query_len >= 0 && max_len >= 0 && window >= 0, "negative sizes");
  if (!a.num_tokens || !max_query_len) return kOk;
  EKV_CHECK(qsl, "null pointer");
  a.qsl = qsl, a.window = window;
  const int64_t rows = std::min(max_query_len, num_tokens);
  return launch_attn<kDense>(a, dense_plans(num_tokens, num_seqs, rows, a.group, kv_heads, dim, max_len, window), dim,
                            workspace, workspace_bytes, stream);
}

extern "C" int64_t ekv_gqa_block_attention_workspace_size(int32_t num_tokens, int32_t heads, int32_t kv_heads,
                                                          int32_t dim, int32_t num_blocks) {
  if (num_tokens <= 0 || kv_heads <= 0 || heads < kv_heads || !gqa_dim(dim)) return 0;
  const int group = heads / kv_heads, share = shared_tokens(num_tokens, 1, kv_heads, group, dim, num_blocks);
  const int64_t n = plan_bytes(block_plans(num_tokens, group, kv_heads, dim, num_blocks), num_tokens, heads, dim);
  if (share < 2) return n;
  return std::max(n, plan_bytes(shared_plans(num_tokens, share, kv_heads, dim, num_blocks), num_tokens, heads, dim));
}

extern "C" int ekv_gqa_block_attention(const uint16_t* q, int64_t q_tok_stride, int64_t q_head_stride,
                                       int32_t num_tokens, int32_t heads, int32_t kv_heads, int32_t dim,
                                       const uint8_t* cache, int64_t page_stride, int64_t num_pages,
                                       const int32_t* block_table, int64_t bt_stride, int32_t bt_width,
                                       const int64_t* positions, const int32_t* req_ids, int32_t num_seqs,
                                       const int32_t* blocks, int64_t blocks_tok_stride, int64_t blocks_head_stride,
                                       int32_t num_blocks, const float* sinks, float scale, uint16_t* out,
                                       int64_t out_tok_stride, int64_t out_head_stride, float* lse,
                                       int64_t lse_stride, void* workspace, int64_t workspace_bytes, void* stream) {
  GqaAttnArgs a;
  const int rc = attn_args(a, q, q_tok_stride, q_head_stride, num_tokens, heads, kv_heads, dim, cache, page_stride,
                           num_pages, block_table, bt_stride, bt_width, positions, num_seqs, sinks, scale, out,
                           out_tok_stride, out_head_stride, lse, lse_stride);
  if (rc) return rc;
  EKV_CHECK(num_blocks >= 0 && num_blocks <= (1 << 24), "negative sizes");
  if (!a.num_tokens) return kOk;
  EKV_CHECK(req_ids && (blocks || !num_blocks), "null pointer");
  a.req_ids = req_ids, a.ids = blocks, a.ids_tok_stride = blocks_tok_stride, a.ids_head_stride = blocks_head_stride;
  a.n_ids = num_blocks;
  const int share = shared_tokens(num_tokens, num_seqs, kv_heads, a.group, dim, num_blocks);
  if (share > 1) {
    a.share = share;
    return launch_attn<kShared>(a, shared_plans(num_tokens, share, kv_heads, dim, num_blocks), dim, workspace,
                                workspace_bytes, stream);
  }
  return launch_attn<kList>(a, block_plans(num_tokens, a.group, kv_heads, dim, num_blocks), dim, workspace,
                            workspace_bytes, stream);
}
