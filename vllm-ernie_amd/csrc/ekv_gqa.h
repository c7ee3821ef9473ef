// Grouped-query layers over an 8-bit paged cache: the page, the page summary
// and what their kernels share.
//
// A page holds 64 tokens of kv_heads heads of D channels as e4m3fn codes, with
// one power-of-two scale for each head's 64 x D keys and one for its values:
//   K codes   head h, token r, channel c at (64 h + r) D + c
//   V codes   head h, channel c, token r at 64 D kv_heads + (D h + c) 64 + at(r),
//             at(r) = 16 ((r / 4) % 4) + 4 (r / 16) + r % 4
//   scales    fp32 K scales [kv_heads], then fp32 V scales [kv_heads]
// V is stored by channel, its tokens in the order in which a 16 x 16 product of
// keys and queries leaves a lane its scores: token 16 t + 4 g + i comes out in
// lane group g, so the 16 bytes of group g are the lane's own A operand for the
// product with the weights, loaded without a transpose or a shuffle.
//
// A page's summary is the mean key of each head: D int8 codes a head, then the
// fp32 power-of-two scales [kv_heads].
#pragma once

#include "ekv_common.h"
#include "ekv_internal.h"

namespace ekv {

// Byte of token r within a channel's 64 of V.
__host__ __device__ __forceinline__ constexpr int gqa_v_at(int r) {
  return 16 * ((r >> 2) & 3) + 4 * (r >> 4) + (r & 3);
}

__host__ __device__ __forceinline__ constexpr int64_t gqa_page_bytes(int kv_heads, int dim) {
  return static_cast<int64_t>(kv_heads) * (2 * kPageTokens * dim + 8);
}
__host__ __device__ __forceinline__ constexpr int64_t gqa_summary_bytes(int kv_heads, int dim) {
  return static_cast<int64_t>(kv_heads) * (dim + 4);
}

inline bool gqa_dim(int dim) { return dim == 64 || dim == 128 || dim == 256; }

// Exponent e of the power of two that brings amax to at most `top` codes:
// r = fl32(max(amax, 1e-10) * fl32(1 / top)), e = ceil(log2 r) from r's bits.
// amax up to the largest finite value: an infinity is taken as that.
__device__ __forceinline__ int pow2_exponent(float amax, float inv_top) {
  const float r = fminf(fmaxf(amax, 0x1.b7cdfep-34f), 0x1.fffffep127f) * inv_top;
  const uint32_t u = __float_as_uint(r);
  const int e = static_cast<int>(u >> 23) - 127;
  return (u & 0x7fffffu) ? e + 1 : e;
}
constexpr float kInv448 = 0x1.24924ap-9f;  // fl32(1 / 448)
constexpr float kInv127 = 0x1.020408p-7f;  // fl32(1 / 127)

// Slots (pages to write, tiles of rows) of a call's sequences, one sequence's
// behind the other's: at(token, b) is the first slot of sequence b, whose tokens
// begin at `token`.  Returns the sequence of a slot, `in` its slot among them;
// -1 where there is none.  Each step narrows it down 64 times; offsets that do
// not ascend give some sequence.
template <typename At>
__device__ __forceinline__ int slot_seq(const int32_t* qsl, int num_seqs, int num_tokens, int slot, At at, int& in) {
  const int lane = static_cast<int>(threadIdx.x) & 63;
  int b = 0, step = 1;
  while (64 * step < num_seqs) step *= 64;
  while (true) {
    const int mine = b + step * lane;
    const int first = mine < num_seqs ? at(min(max(qsl[mine], 0), num_tokens), mine) : 0x7fffffff;
    const uint64_t upto = __ballot(first <= slot);
    if (!upto) return -1;
    const int last = 63 - __builtin_clzll(upto);
    b += step * last;
    if (step == 1) {
      in = slot - __builtin_amdgcn_readlane(first, last);
      return b;
    }
    step >>= 6;
  }
}

// ---------------------------------------------------------------------------
// RMS norm of a head and the rotation of a slice of its channels.  A row of D
// channels is held by LPR lanes (a power of two, at least D / 8), 8 channels
// each; lanes past D / 8 hold zeros.
// ---------------------------------------------------------------------------
struct RopeArgs {
  const float* cos_sin;  // [rows, rope]: cos rope / 2 | sin rope / 2
  int32_t rows, rope, offset, interleaved;
};

// y = x * rsqrt(mean x^2 + eps) * w, all in fp32.
template <int LPR>
__device__ __forceinline__ void row_rms_norm(float (&v)[8], const float (&w)[8], int dim, float eps) {
  float s = 0.0f;
#pragma unroll
  for (int i = 0; i < 8; ++i) s = __fmaf_rn(v[i], v[i], s);
#pragma unroll
  for (int m = LPR >> 1; m > 0; m >>= 1) s += __shfl_xor(s, m, 64);
  const float r = 1.0f / sqrtf(s / static_cast<float>(dim) + eps);
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = v[i] * r * w[i];
}

// The 8 (cos, sin) of lane j's channels, each for its own channel; lanes
// outside the slice, and rows outside the table, get the identity.
__device__ __forceinline__ void rope_factors(const RopeArgs& a, int64_t pos, int j, float (&c)[8], float (&s)[8]) {
  const int at = 8 * j - a.offset;  // the lane's first channel within the slice
  const bool in = at >= 0 && at < a.rope && pos >= 0 && pos < a.rows;
  const int half = a.rope >> 1;
#pragma unroll
  for (int i = 0; i < 8; ++i) c[i] = 1.0f, s[i] = 0.0f;
  if (!in) return;
  const float* row = a.cos_sin + pos * a.rope;
  if (a.interleaved) {
    const float4 cv = *reinterpret_cast<const float4*>(row + at / 2);
    const float4 sv = *reinterpret_cast<const float4*>(row + half + at / 2);
    c[0] = c[1] = cv.x, c[2] = c[3] = cv.y, c[4] = c[5] = cv.z, c[6] = c[7] = cv.w;
    s[0] = s[1] = sv.x, s[2] = s[3] = sv.y, s[4] = s[5] = sv.z, s[6] = s[7] = sv.w;
  } else {
    const int k = at < half ? at : at - half;
#pragma unroll
    for (int i = 0; i < 8; i += 4) {
      const float4 cv = *reinterpret_cast<const float4*>(row + k + i);
      const float4 sv = *reinterpret_cast<const float4*>(row + half + k + i);
      c[i] = cv.x, c[i + 1] = cv.y, c[i + 2] = cv.z, c[i + 3] = cv.w;
      s[i] = sv.x, s[i + 1] = sv.y, s[i + 2] = sv.z, s[i + 3] = sv.w;
    }
  }
}

// Turns the pairs of the slice: (a, b) -> (a cos - b sin, b cos + a sin).  The
// partner of channel i is i ^ 1 (interleaved) or half a slice away, which is
// the same 8 channels of another lane.  Every lane of the wave takes part.
template <int LPR>
__device__ __forceinline__ void row_rope(float (&v)[8], const RopeArgs& a, int j, const float (&c)[8],
                                         const float (&s)[8]) {
  if (a.interleaved) {
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
      const float x = v[i], y = v[i + 1];
      v[i] = x * c[i] - y * s[i];
      v[i + 1] = y * c[i] + x * s[i];
    }
  } else {
    const int at = 8 * j - a.offset, hop = a.rope >> 4;
    const bool in = at >= 0 && at < a.rope, low = at < (a.rope >> 1);
    const int lane = static_cast<int>(threadIdx.x) & 63;
    const int from = in ? (low ? lane + hop : lane - hop) : lane;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float p = __shfl(v[i], from, 64);
      v[i] = low ? v[i] * c[i] - p * s[i] : v[i] * c[i] + p * s[i];
    }
  }
}

}  // namespace ekv
