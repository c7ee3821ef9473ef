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
// qk_norm_rope.  LPR lanes hold a row (8 channels each); a lane group takes
// `batch` heads of one token, with the token's cos / sin and the weights in
// registers.
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
// It owns the page's head, so scales, codes and summary need no other one.
// ---------------------------------------------------------------------------
struct GqaAppendArgs {
  const uint16_t *k, *v;    // bf16 rows at + t * tok_stride + h * head_stride
  int64_t k_tok_stride, k_head_stride, v_tok_stride, v_head_stride;
  int32_t k_aligned, v_aligned;
  int32_t kv_heads, num_tokens;
  const int64_t* positions; // [T]; a sequence's tokens at consecutive positions
  const int32_t* qsl;       // [B + 1]
  int32_t num_seqs, page_slots;  // most pages a sequence's rows touch
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

__device__ __forceinline__ float fp8_value(uint32_t byte) {
  return __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(byte), false)[0];
}

template <int D>
__device__ void gqa_append_block(const GqaAppendArgs& a, int block) {
  constexpr int LPR = D / 8, RPP = 256 / LPR, PASSES = kPageTokens / RPP;  // lanes a row, rows a pass
  __shared__ __attribute__((aligned(16))) uint8_t tile[kPageTokens * (D + 16)];
  __shared__ float red[2][4];
  __shared__ float sums[4][D];
  const int tid = static_cast<int>(threadIdx.x), wave = tid >> 6, j = tid & (LPR - 1), r0 = tid / LPR;
  const int h = block % a.kv_heads;
  const int slot = block / a.kv_heads % a.page_slots, b = block / a.kv_heads / a.page_slots;
  const int t0 = a.qsl[b], n = min(a.qsl[b + 1], a.num_tokens) - t0;
  if (t0 < 0 || n <= 0) return;
  const int64_t p0 = a.positions[t0];
  if (p0 < 0) return;
  const int64_t lp = p0 / kPageTokens + slot, base = lp * kPageTokens;
  const int first = static_cast<int>(max(p0 - base, static_cast<int64_t>(0)));
  const int end = static_cast<int>(min(p0 + n - base, static_cast<int64_t>(kPageTokens)));  // rows first .. end - 1
  if (end <= first || lp >= a.bt_width) return;
  const int64_t page = a.block_table[b * a.bt_stride + lp];
  if (page < 0 || page >= a.num_pages) return;
  const int64_t tok = t0 + base - p0;  // token of the page's row 0

  uint8_t* const pg = a.cache + page * a.page_stride;
  uint8_t* const kp = pg + static_cast<int64_t>(h) * kPageTokens * D;
  uint8_t* const vp = pg + static_cast<int64_t>(a.kv_heads + h) * kPageTokens * D;
  float* const ks = reinterpret_cast<float*>(pg + 2ll * a.kv_heads * kPageTokens * D) + h;
  float* const vs = ks + a.kv_heads;

  // the new rows, and their largest values
  float kx[PASSES][8], vx[PASSES][8], kmax = 0.0f, vmax = 0.0f;
  float w[8];
  if (a.prep && a.k_w) load_weight8(a.k_w, a.k_w_bf16, j, w);
#pragma unroll
  for (int i = 0; i < PASSES; ++i) {
    const int r = i * RPP + r0;
    const bool have = r >= first && r < end;
#pragma unroll
    for (int e = 0; e < 8; ++e) kx[i][e] = 0.0f, vx[i][e] = 0.0f;
    if (have) {
      load_row8(a.k + (tok + r) * a.k_tok_stride + h * a.k_head_stride + 8 * j, a.k_aligned, kx[i]);
      load_row8(a.v + (tok + r) * a.v_tok_stride + h * a.v_head_stride + 8 * j, a.v_aligned, vx[i]);
    }
    if (a.prep) {
      float c[8], s[8];
      rope_factors(a.rope, have ? base + r : -1, j, c, s);
      if (a.k_w) row_rms_norm<LPR>(kx[i], w, D, a.eps);
      row_rope<LPR>(kx[i], a.rope, j, c, s);
#pragma unroll
      for (int e = 0; e < 8; ++e) kx[i][e] = have ? bf16_to_f32(f32_to_bf16(kx[i][e])) : 0.0f;
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) kmax = fmaxf(kmax, fabsf(kx[i][e])), vmax = fmaxf(vmax, fabsf(vx[i][e]));
  }
  kmax = wave_max_xor(kmax, 64);
  vmax = wave_max_xor(vmax, 64);
  if ((tid & 63) == 0) red[0][wave] = kmax, red[1][wave] = vmax;
  __syncthreads();
  kmax = fmaxf(fmaxf(red[0][0], red[0][1]), fmaxf(red[0][2], red[0][3]));
  vmax = fmaxf(fmaxf(red[1][0], red[1][1]), fmaxf(red[1][2], red[1][3]));
  const float kold = first ? *ks : 0.0f, vold = first ? *vs : 0.0f;
  const float knew = fmaxf(exp2i(pow2_exponent(kmax, kInv448)), kold);
  const float vnew = fmaxf(exp2i(pow2_exponent(vmax, kInv448)), vold);
  const bool kgrow = first && knew > kold, vgrow = first && vnew > vold;
  const float ki = 1.0f / knew, vi = 1.0f / vnew;  // powers of two: the products below are exact
  const float kr = kold * ki, vr = vold * vi;

  // K codes of the new rows; V codes to LDS, row by row
#pragma unroll
  for (int i = 0; i < PASSES; ++i) {
    const int r = i * RPP + r0;
    if (r >= first && r < end) {
      uint2 kc, vc;
      kc.x = f32x2_to_fp8(kx[i][0] * ki, kx[i][1] * ki) | f32x2_to_fp8(kx[i][2] * ki, kx[i][3] * ki) << 16;
      kc.y = f32x2_to_fp8(kx[i][4] * ki, kx[i][5] * ki) | f32x2_to_fp8(kx[i][6] * ki, kx[i][7] * ki) << 16;
      vc.x = f32x2_to_fp8(vx[i][0] * vi, vx[i][1] * vi) | f32x2_to_fp8(vx[i][2] * vi, vx[i][3] * vi) << 16;
      vc.y = f32x2_to_fp8(vx[i][4] * vi, vx[i][5] * vi) | f32x2_to_fp8(vx[i][6] * vi, vx[i][7] * vi) << 16;
      *reinterpret_cast<uint2*>(kp + r * D + 8 * j) = kc;
      *reinterpret_cast<uint2*>(tile + r * (D + 16) + 8 * j) = vc;
    } else if (r < first && (kgrow || a.summary)) {
      // earlier rows: again in the larger scale
      uint2 kc = *reinterpret_cast<const uint2*>(kp + r * D + 8 * j);
      if (kgrow) {
        const f32x4 lo = fp8x4_to_f32(kc.x) * kr, hi = fp8x4_to_f32(kc.y) * kr;
        kc.x = f32x2_to_fp8(lo[0], lo[1]) | f32x2_to_fp8(lo[2], lo[3]) << 16;
        kc.y = f32x2_to_fp8(hi[0], hi[1]) | f32x2_to_fp8(hi[2], hi[3]) << 16;
        *reinterpret_cast<uint2*>(kp + r * D + 8 * j) = kc;
      }
      if (a.summary) {
        const f32x4 lo = fp8x4_to_f32(kc.x), hi = fp8x4_to_f32(kc.y);
#pragma unroll
        for (int e = 0; e < 4; ++e) kx[i][e] = lo[e] * knew, kx[i][4 + e] = hi[e] * knew;
      }
    }
  }
  __syncthreads();

  // V by channel: 16 bytes at a time, old tokens' bytes requantized, those behind the last row kept
  for (int u = tid; u < 4 * D; u += 256) {
    const int c = u >> 2, g = u & 3;
    uint8_t* const dst = vp + c * kPageTokens + 16 * g;
    const bool whole = first == 0 && end == kPageTokens;
    uint32_t out[4] = {};
    if (!whole) *reinterpret_cast<uint4*>(out) = *reinterpret_cast<const uint4*>(dst);
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      uint32_t word = out[t];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int r = 16 * t + 4 * g + i;
        uint32_t byte = (word >> (8 * i)) & 0xffu;
        if (r >= first && r < end) byte = tile[r * (D + 16) + c];
        else if (r < first && vgrow) byte = f32x2_to_fp8(fp8_value(byte) * vr, 0.0f) & 0xffu;
        word = (word & ~(0xffu << (8 * i))) | byte << (8 * i);
      }
      out[t] = word;
    }
    *reinterpret_cast<uint4*>(dst) = *reinterpret_cast<uint4*>(out);
  }
  if (tid == 0) *ks = knew, *vs = vnew;

  if (a.summary) {  // uniform over the workgroup
    // Sums of codes: multiples of 2^-9 below 2^15, exact in fp32 in any order.
    float sum[8] = {};
#pragma unroll
    for (int i = 0; i < PASSES; ++i) {
      const int r = i * RPP + r0;
      if (r < end) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float y = kx[i][e] * ki;
          sum[e] += r < first ? y : fp8_value(f32x2_to_fp8(y, 0.0f) & 0xffu);
        }
      }
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) {
#pragma unroll
      for (int m = LPR; m < 64; m <<= 1) sum[e] += __shfl_xor(sum[e], m, 64);
    }
    if ((tid & 63) < LPR) {
#pragma unroll
      for (int e = 0; e < 8; ++e) sums[wave][8 * j + e] = sum[e];
    }
    __syncthreads();
    float mean = 0.0f;
    if (tid < D) mean = (((sums[0][tid] + sums[1][tid]) + sums[2][tid]) + sums[3][tid]) / static_cast<float>(end);
    float top = wave_max_xor(fabsf(mean), 64);
    if ((tid & 63) == 0) red[0][wave] = top;
    __syncthreads();
    top = fmaxf(fmaxf(red[0][0], red[0][1]), fmaxf(red[0][2], red[0][3]));
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
__global__ void __launch_bounds__(256) gqa_append_kernel(GqaAppendArgs a) {
  gqa_append_block<D>(a, static_cast<int>(blockIdx.x));
}

// The append's workgroups first, then those of q's norm and rotation.
template <int D>
__global__ void __launch_bounds__(256) gqa_prologue_kernel(GqaAppendArgs a, NormArgs q, int append_blocks) {
  const int block = static_cast<int>(blockIdx.x);
  if (block < append_blocks) {
    gqa_append_block<D>(a, block);
  } else {
    const int64_t units = norm_units(q, 0);
    norm_unit<D / 8>(q, static_cast<int64_t>(block - append_blocks) * (2048 / D) + threadIdx.x / (D / 8), units, units);
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
// (2048), at most 8.
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

static int launch_append(const GqaAppendArgs& a, const NormArgs* q, int dim, void* stream) {
  const int64_t append = static_cast<int64_t>(a.num_seqs) * a.page_slots * a.kv_heads;
  int64_t blocks = append;
  if (q) blocks += (norm_units(*q, 0) + 2048 / dim - 1) / (2048 / dim);
  EKV_CHECK(blocks < (int64_t{1} << 31), "too many rows for one call");
  if (!blocks) return kOk;
  const dim3 grid(static_cast<uint32_t>(blocks));
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (q) {
    if (dim == 64) gqa_prologue_kernel<64><<<grid, 256, 0, s>>>(a, *q, static_cast<int>(append));
    else if (dim == 128) gqa_prologue_kernel<128><<<grid, 256, 0, s>>>(a, *q, static_cast<int>(append));
    else gqa_prologue_kernel<256><<<grid, 256, 0, s>>>(a, *q, static_cast<int>(append));
  } else {
    if (dim == 64) gqa_append_kernel<64><<<grid, 256, 0, s>>>(a);
    else if (dim == 128) gqa_append_kernel<128><<<grid, 256, 0, s>>>(a);
    else gqa_append_kernel<256><<<grid, 256, 0, s>>>(a);
  }
  return ekv_launch_status();
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
  EKV_CHECK(k && v && positions && qsl && block_table && cache, "null pointer");
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
  EKV_CHECK(blocks < (int64_t{1} << 31), "too many rows for one call");
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
