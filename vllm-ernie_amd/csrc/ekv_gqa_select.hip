// Block selection of grouped-query layers: the pages of a sequence that a
// query token attends to, one list for each kv head, by the pages' mean keys.
//
//   score_j = max_g (q_g . m_j) s_j
//
// with q_g the group's heads as int8 codes (one exponent for the group, which
// does not change the order), m_j the page's mean key as int8 codes and s_j its
// power-of-two scale.  The dot products are whole numbers below 2^24, so every
// score is exact in fp32 and the selection depends on no order of summation.
//
// Built with -ffp-contract=off (the quantization of q is mirrored by the oracle).
#include <algorithm>

#include "ekv_gqa.h"

namespace ekv {

constexpr int kSelBins = 2048;
constexpr int kSelMaxBlocks = 32768;  // 16 waves of 32 keys a lane
constexpr int kSelMaxGroup = 64;

struct GqaSelectArgs {
  const uint16_t* q;
  int64_t q_tok_stride, q_head_stride;
  int32_t q_aligned, num_tokens, heads, kv_heads, group;
  const uint8_t* summary;
  int64_t summary_stride, num_pages;
  const int32_t* block_table;
  int64_t bt_stride;
  int32_t bt_width, num_seqs;
  const int64_t* positions;
  const int32_t* req_ids;
  int32_t max_blocks;       // pages that the lanes' keys hold
  int32_t n, keep_first, keep_last;
  int32_t* ids;
  int64_t ids_tok_stride, ids_head_stride;
};

__device__ __forceinline__ void load_q8(const uint16_t* p, bool aligned, float (&v)[8]) {
  if (aligned) {
    const uint4 w = *reinterpret_cast<const uint4*>(p);
    const uint32_t ww[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[2 * i] = __uint_as_float(ww[i] << 16);
      v[2 * i + 1] = __uint_as_float(ww[i] & 0xffff0000u);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = bf16_to_f32(p[i]);
  }
}

// One workgroup per (token, kv head).  Its waves share the pages in order, each
// with the keys of up to KPT chunks of 64, one page a lane; the n-th largest key
// comes from three rounds of a histogram, and the chosen pages are written
// in order by counts of the chunks before.
//
// Bound by the chain of request, table, mean keys and three rounds where rows are
// few (32 rows of 2,048 pages, 8 kv heads of 128: 23 us, of which 69 MB of
// records are 11 at the card's read rate), else by the records' way through the
// caches (333 rows of 750 pages, 4 kv heads: 24 us).
template <int D, int WAVES, int KPT>
__global__ void __launch_bounds__(64 * WAVES) gqa_block_select_kernel(GqaSelectArgs a) {
  constexpr int S = D / 64, kThreads = 64 * WAVES, kRow = D + 16;  // padded rows: 16 of them in 16 bank groups
  constexpr int kPer = kSelBins / kThreads;                        // bins a thread sums
  constexpr bool kAhead = KPT <= 8;                                // pages asked for at entry
  constexpr int kBuf = WAVES == 16 && (KPT > 8 || D == 256) ? 1 : 2;  // chunks of mean keys in registers
  __shared__ __attribute__((aligned(16))) int8_t qc[kSelMaxGroup * kRow];
  __shared__ __attribute__((aligned(16))) uint32_t bins[kSelBins];
  __shared__ uint32_t sums[2][WAVES], found[3];
  __shared__ float red[WAVES];
  const int tid = static_cast<int>(threadIdx.x), lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  // Eight tokens at a time, one an XCD (workgroup i runs on XCD i % 8): the
  // heads of a page's record share cache lines, which its XCD's L2 reads once
  // (32 rows of 2,048 pages, 8 heads of 128: 38 -> 23 us).
  const int block = static_cast<int>(blockIdx.x), eights = a.num_tokens / 8 * 8 * a.kv_heads;
  int h = block % a.kv_heads;
  int64_t t = block / a.kv_heads;
  if (block < eights) h = block / 8 % a.kv_heads, t = block / 8 / a.kv_heads * 8 + block % 8;
  // q is asked for first: nothing of it waits for the request's row of the table
  const int tiles = (a.group + 15) / 16;
  const uint16_t* const q = a.q + t * a.q_tok_stride + static_cast<int64_t>(h) * a.group * a.q_head_stride;
  const bool some = tid < a.group * (D / 8);
  float v[8] = {};
  if (some) load_q8(q + tid / (D / 8) * a.q_head_stride + 8 * (tid % (D / 8)), a.q_aligned, v);
  const int64_t pos = a.positions[t];
  const int b = a.req_ids[t];
  if (b < 0 || b >= a.num_seqs) return;
  int32_t* const out = a.ids + t * a.ids_tok_stride + h * a.ids_head_stride;

  // the wave's pages, asked for before anything waits
  const int32_t* bt = a.block_table + b * a.bt_stride;
  const int each = min((a.max_blocks + 64 * WAVES - 1) / (64 * WAVES), KPT);  // chunks of a wave
  const int base = wave * each * 64;
  auto page_of = [&](int c, int end) {
    const int lp = base + 64 * c + lane;
    return lp < end ? bt[lp] : -1;
  };
  int page[kAhead ? KPT : 1];
  if constexpr (kAhead) {
#pragma unroll
    for (int c = 0; c < KPT; ++c) page[c] = c < each ? page_of(c, min(a.max_blocks, a.bt_width)) : -1;
  }
  const int all = pos < 0 ? 0 : static_cast<int>(min(pos / kPageTokens + 1, static_cast<int64_t>(a.bt_width)));
  const int nb = __builtin_amdgcn_readfirstlane(min(all, a.max_blocks));
  const int chunks = min(max((nb - base + 63) / 64, 0), each);  // of this wave

  // q's codes: one exponent for the group; heads again where a tile has rows left
  float top = 0.0f;
#pragma unroll
  for (int e = 0; e < 8; ++e) top = fmaxf(top, fabsf(v[e]));
  for (int i = tid + kThreads; i < a.group * (D / 8); i += kThreads) {
    load_q8(q + i / (D / 8) * a.q_head_stride + 8 * (i % (D / 8)), a.q_aligned, v);
#pragma unroll
    for (int e = 0; e < 8; ++e) top = fmaxf(top, fabsf(v[e]));
  }
  top = wave_max_xor(top, 64);
  if (lane == 0) red[wave] = top;
  for (int i = tid; i < kSelBins; i += kThreads) bins[i] = 0;
  if (tid == 0) found[1] = 0xffffffffu;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < WAVES; ++w) top = fmaxf(top, red[w]);
  const float qi = 1.0f / exp2i(pow2_exponent(top, kInv127));  // a power of two: products are exact
  for (int i = tid; i < tiles * 16 * (D / 8); i += kThreads) {
    const int row = i / (D / 8), at = 8 * (i % (D / 8));
    load_q8(q + row % a.group * a.q_head_stride + at, a.q_aligned, v);
    uint32_t w[2] = {};
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int code = static_cast<int>(fminf(fmaxf(rintf(v[e] * qi), -127.0f), 127.0f));
      w[e >> 2] |= static_cast<uint32_t>(code & 0xff) << (8 * (e & 3));
    }
    *reinterpret_cast<uint2*>(qc + row * kRow + at) = make_uint2(w[0], w[1]);
  }
  __syncthreads();

  // keys: a chunk is four tiles of 16 pages; the mean keys of the next chunk
  // are on their way while this one is multiplied
  const int m = lane & 15, g = lane >> 4;
  i32x4 qa[S];
#pragma unroll
  for (int s = 0; s < S; ++s) qa[s] = *reinterpret_cast<const i32x4*>(qc + m * kRow + 64 * s + 16 * g);
  i32x4 mk[kBuf][4][S];
  float scale[kBuf];
  bool live[kBuf];
  auto fetch = [&](int c, int buf) {
    int pg = kAhead ? page[kAhead ? c : 0] : page_of(c, nb);
    if (pg >= a.num_pages || base + 64 * c + lane >= nb) pg = -1;
    live[buf] = pg >= 0;
    scale[buf] = 0.0f;
    // 2^-24 of it, which leaves the order: products of up to 2^22 with scales of up to 2^122 stay finite
    if (pg >= 0) scale[buf] = 0x1p-24f * reinterpret_cast<const float*>(a.summary + pg * a.summary_stride + a.kv_heads * D)[h];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int64_t p = __shfl(pg, 16 * u + m, 64);
#pragma unroll
      for (int s = 0; s < S; ++s) {
        mk[buf][u][s] = i32x4{};
        if (p >= 0)
          mk[buf][u][s] = *reinterpret_cast<const i32x4*>(a.summary + p * a.summary_stride + h * D + 64 * s + 16 * g);
      }
    }
  };
  uint32_t key[KPT];
  if (kBuf == 2 && chunks > 0) fetch(0, 0);
#pragma unroll
  for (int c = 0; c < KPT; ++c) {
    key[c] = 0;
    if (c < chunks) {
      if (kBuf == 1) fetch(c, 0);
      else if (c + 1 < KPT && c + 1 < chunks) fetch(c + 1 < KPT ? c + 1 : 0, (c + 1) & 1);
      const int buf = kBuf == 1 ? 0 : c & 1;
      int best = 0;
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        int mx = -0x7fffffff;
        for (int r = 0; r < tiles; ++r) {
          i32x4 acc = {};
#pragma unroll
          for (int s = 0; s < S; ++s) {
            const i32x4 x = r ? *reinterpret_cast<const i32x4*>(qc + (16 * r + m) * kRow + 64 * s + 16 * g) : qa[s];
            acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(x, mk[buf][u][s], acc, 0, 0, 0);
          }
          mx = max(max(mx, max(acc[0], acc[1])), max(acc[2], acc[3]));
        }
        mx = max(mx, __shfl_xor(mx, 16, 64));
        mx = max(mx, __shfl_xor(mx, 32, 64));
        best = g == u ? mx : best;  // page 16 u + m of the chunk: this lane's
      }
      const int lp = base + 64 * c + lane;
      const uint32_t k = lp < a.keep_first || lp >= all - a.keep_last ? 0xffffffffu
                                                                      : score_key(static_cast<float>(best) * scale[buf]);
      key[c] = live[buf] ? k : 0u;
    }
  }

  // The n-th largest key, 11, 11 and 10 bits: the keys above `thr` are taken, and
  // the first `need` of those equal to it.  A bin whose keys are all needed ends
  // the search, as the second round's mostly is.
  uint32_t thr = 0, prefix = 0, mask = 0, need = static_cast<uint32_t>(a.n);
#pragma unroll
  for (int round = 0; round < 3; ++round) {
    const int shift = round == 0 ? 21 : round == 1 ? 10 : 0;
    const uint32_t width = round == 2 ? 1024u : 2048u;
#pragma unroll
    for (int c = 0; c < KPT; ++c) {
      if (c < chunks && key[c] && (key[c] & mask) == prefix) atomicAdd(&bins[(key[c] >> shift) & (width - 1)], 1u);
    }
    __syncthreads();
    uint32_t own[kPer], mine = 0;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      own[i] = bins[kPer * tid + i];
      mine += own[i];
    }
    uint32_t up = mine;  // over the lanes from this one on
#pragma unroll
    for (int k = 1; k < 64; k <<= 1) {
      const uint32_t x = __shfl_down(up, k, 64);
      if (lane + k < 64) up += x;
    }
    if (lane == 0) sums[0][wave] = up;
    __syncthreads();
    uint32_t above = up - mine;  // keys in the bins above this thread's
#pragma unroll
    for (int w = 0; w < WAVES; ++w) above += w > wave ? sums[0][w] : 0u;
    // the bin with fewer than `need` keys above it and at least that many with its own
#pragma unroll
    for (int i = kPer - 1; i >= 0; --i) {
      bins[kPer * tid + i] = 0;  // for the next round
      if (above < need && above + own[i] >= need) found[0] = kPer * tid + i, found[1] = need - above, found[2] = own[i];
      above += own[i];
    }
    __syncthreads();
    const uint32_t bin = found[0], left = found[1], held = found[2];
    if (left == 0xffffffffu) {  // round 0, fewer keys than n: all of them
      need = 0;
      break;
    }
    prefix |= bin << shift;
    mask |= (width - 1) << shift;
    thr = prefix, need = left;
    if (left == held) {
      thr = prefix ? prefix - 1 : 0, need = 0;
      break;
    }
  }

  // in order
  uint32_t gt_sum = 0, eq_sum = 0;
#pragma unroll
  for (int c = 0; c < KPT; ++c) {
    if (c < chunks) {
      gt_sum += static_cast<uint32_t>(__builtin_popcountll(__ballot(key[c] > thr)));
      eq_sum += static_cast<uint32_t>(__builtin_popcountll(__ballot(need && key[c] == thr)));
    }
  }
  __syncthreads();
  if (lane == 0) sums[0][wave] = gt_sum, sums[1][wave] = eq_sum;
  __syncthreads();
  uint32_t gb = 0, eb = 0, total = 0, equal = 0;
#pragma unroll
  for (int w = 0; w < WAVES; ++w) {
    if (w == wave) gb = total, eb = equal;
    total += sums[0][w], equal += sums[1][w];
  }
  total += min(equal, need);
  const uint64_t below = (1ull << lane) - 1;
#pragma unroll
  for (int c = 0; c < KPT; ++c) {
    if (c < chunks) {
      const bool is_gt = key[c] > thr, is_eq = need && key[c] == thr;
      const uint64_t gt = __ballot(is_gt), eq = __ballot(is_eq);
      const uint32_t gr = gb + static_cast<uint32_t>(__builtin_popcountll(gt & below));
      const uint32_t er = eb + static_cast<uint32_t>(__builtin_popcountll(eq & below));
      if (is_gt || (is_eq && er < need)) out[gr + min(er, need)] = base + 64 * c + lane;
      gb += static_cast<uint32_t>(__builtin_popcountll(gt));
      eb += static_cast<uint32_t>(__builtin_popcountll(eq));
    }
  }
  for (uint32_t i = total + tid; i < static_cast<uint32_t>(a.n); i += kThreads) out[i] = -1;
}

template <int D>
static void launch_select(const GqaSelectArgs& a, int64_t grid, hipStream_t s) {
  const dim3 g(static_cast<uint32_t>(grid));
  // 8 kv heads of 128, four waves of 8 chunks against eight of 4: 1 row of 2,048
  // pages 15.1 us and 13.2, 32 rows 20.1 and 19.5, 64 rows 27.3 and 29.8, 512
  // rows 106 and 119.
  if (a.max_blocks <= 2048 && grid >= 512) gqa_block_select_kernel<D, 4, 8><<<g, 256, 0, s>>>(a);
  else if (a.max_blocks <= 2048) gqa_block_select_kernel<D, 8, 4><<<g, 512, 0, s>>>(a);
  else if (a.max_blocks <= 8192) gqa_block_select_kernel<D, 16, 8><<<g, 1024, 0, s>>>(a);
  else gqa_block_select_kernel<D, 16, 32><<<g, 1024, 0, s>>>(a);
}

}  // namespace ekv

using namespace ekv;

extern "C" int ekv_gqa_block_select(const uint16_t* q, int64_t q_tok_stride, int64_t q_head_stride,
                                    int32_t num_tokens, int32_t heads, int32_t kv_heads, int32_t dim,
                                    const uint8_t* summary, int64_t summary_stride, int64_t num_pages,
                                    const int32_t* block_table, int64_t bt_stride, int32_t bt_width,
                                    const int64_t* positions, const int32_t* req_ids, int32_t num_seqs,
                                    int32_t max_len, int32_t keep_first, int32_t keep_last, int32_t* blocks,
                                    int64_t blocks_tok_stride, int64_t blocks_head_stride, int32_t num_blocks,
                                    void* stream) {
  EKV_CHECK(gqa_dim(dim), "dim must be 64, 128 or 256");
  EKV_CHECK(kv_heads > 0 && heads > 0 && heads % kv_heads == 0, "heads must be a multiple of kv_heads");
  EKV_CHECK(heads / kv_heads <= kSelMaxGroup, "at most 64 query heads a kv head");
  EKV_CHECK(num_tokens >= 0 && num_seqs >= 0 && num_pages >= 0 && bt_width >= 0 && max_len >= 0, "negative sizes");
  EKV_CHECK(keep_first >= 0 && keep_last >= 0 && num_blocks >= 0 &&
                static_cast<int64_t>(keep_first) + keep_last <= num_blocks,
            "keep_first + keep_last must be at most num_blocks");
  EKV_CHECK(max_len <= kSelMaxBlocks * kPageTokens, "max_len must be at most 2097152 tokens");
  if (!num_tokens || !num_seqs || !num_blocks) return kOk;
  EKV_CHECK(q && (summary || !num_pages) && (block_table || !bt_width) && positions && req_ids && blocks, "null pointer");
  EKV_CHECK(summary_stride >= gqa_summary_bytes(kv_heads, dim) && summary_stride % 16 == 0 && aligned16(summary),
            "summary_stride must be a multiple of 16 of at least kv_heads * (dim + 4) bytes");
  EKV_CHECK(num_pages < (int64_t{1} << 31), "too many pages");
  const int64_t grid = static_cast<int64_t>(num_tokens) * kv_heads;
  EKV_CHECK(grid < (1 << 22), "too many rows for one call");  // fewer than 2^32 lanes
  GqaSelectArgs a{};
  a.q = q, a.q_tok_stride = q_tok_stride, a.q_head_stride = q_head_stride;
  a.q_aligned = aligned16(q) && q_tok_stride % 8 == 0 && q_head_stride % 8 == 0;
  a.num_tokens = num_tokens, a.heads = heads, a.kv_heads = kv_heads, a.group = heads / kv_heads;
  a.summary = summary, a.summary_stride = summary_stride, a.num_pages = num_pages;
  a.block_table = block_table, a.bt_stride = bt_stride, a.bt_width = bt_width, a.num_seqs = num_seqs;
  a.positions = positions, a.req_ids = req_ids;
  a.max_blocks = (max_len + kPageTokens - 1) / kPageTokens;
  a.n = num_blocks, a.keep_first = keep_first, a.keep_last = keep_last;
  a.ids = blocks, a.ids_tok_stride = blocks_tok_stride, a.ids_head_stride = blocks_head_stride;
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (dim == 64) launch_select<64>(a, grid, s);
  else if (dim == 128) launch_select<128>(a, grid, s);
  else launch_select<256>(a, grid, s);
  return ekv_launch_status();
}
