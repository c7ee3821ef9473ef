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

constexpr int kSelThreads = 1024, kSelWaves = kSelThreads / 64;
constexpr int kSelBins = 2048;
constexpr int kSelMaxBlocks = 32768;  // keys of a row in LDS
constexpr int kSelMaxGroup = 64;

struct GqaSelectArgs {
  const uint16_t* q;
  int64_t q_tok_stride, q_head_stride;
  int32_t num_tokens, heads, kv_heads, group;
  const uint8_t* summary;
  int64_t summary_stride, num_pages;
  const int32_t* block_table;
  int64_t bt_stride;
  int32_t bt_width, num_seqs;
  const int64_t* positions;
  const int32_t* req_ids;
  int32_t max_blocks;       // keys the LDS holds
  int32_t n, keep_first, keep_last;
  int32_t* ids;
  int64_t ids_tok_stride, ids_head_stride;
};

// Counts of a workgroup's threads summed over all threads with a higher id.
__device__ __forceinline__ uint32_t count_above(uint32_t v, uint32_t* tmp) {
  const int lane = static_cast<int>(threadIdx.x) & 63, wave = static_cast<int>(threadIdx.x) >> 6;
  uint32_t s = v;
#pragma unroll
  for (int m = 1; m < 64; m <<= 1) {
    const uint32_t o = __shfl_down(s, m, 64);
    if (lane + m < 64) s += o;
  }
  if (lane == 0) tmp[wave] = s;
  __syncthreads();
  uint32_t above = s - v;
  for (int w = wave + 1; w < kSelWaves; ++w) above += tmp[w];
  __syncthreads();
  return above;
}

// One workgroup per (token, kv head): the keys of all its pages in LDS, then
// the n largest by three rounds of a histogram.
template <int D>
__global__ void __launch_bounds__(kSelThreads) gqa_block_select_kernel(GqaSelectArgs a) {
  constexpr int S = D / 64;
  extern __shared__ __attribute__((aligned(16))) uint32_t keys[];  // [max_blocks rounded up to 64]
  __shared__ __attribute__((aligned(16))) int8_t qc[kSelMaxGroup * D];
  __shared__ uint32_t bins[kSelBins];
  __shared__ uint32_t tmp[kSelWaves], chunk[kSelMaxBlocks / 64 + 1];
  __shared__ uint32_t found[2];
  __shared__ float red[kSelWaves];
  const int tid = static_cast<int>(threadIdx.x), lane = tid & 63, wave = tid >> 6;
  const int h = static_cast<int>(blockIdx.x) % a.kv_heads;
  const int64_t t = blockIdx.x / a.kv_heads;
  const int b = a.req_ids[t];
  if (b < 0 || b >= a.num_seqs) return;
  int32_t* const out = a.ids + t * a.ids_tok_stride + h * a.ids_head_stride;
  const int64_t pos = a.positions[t];
  const int all = pos < 0 ? 0 : static_cast<int>(min(pos / kPageTokens + 1, static_cast<int64_t>(a.bt_width)));
  const int nb = min(all, a.max_blocks);

  // q's codes
  const int tiles = (a.group + 15) / 16;
  float top = 0.0f;
  for (int i = tid; i < a.group * D; i += kSelThreads) {
    const int gh = i / D;
    top = fmaxf(top, fabsf(bf16_to_f32(a.q[t * a.q_tok_stride + (h * a.group + gh) * a.q_head_stride + i % D])));
  }
  top = wave_max_xor(top, 64);
  if (lane == 0) red[wave] = top;
  __syncthreads();
  for (int w = 0; w < kSelWaves; ++w) top = fmaxf(top, red[w]);
  const float qs = exp2i(pow2_exponent(top, kInv127));
  for (int i = tid; i < tiles * 16 * D; i += kSelThreads) {
    const int gh = (i / D) % a.group;  // heads again where a tile has rows left
    const float x = bf16_to_f32(a.q[t * a.q_tok_stride + (h * a.group + gh) * a.q_head_stride + i % D]);
    qc[i] = static_cast<int8_t>(fminf(fmaxf(rintf(x / qs), -127.0f), 127.0f));
  }
  __syncthreads();

  // keys: 64 pages a wave and round, as four tiles of 16
  const int m = lane & 15, g = lane >> 4;
  const int32_t* bt = a.block_table + b * a.bt_stride;
  for (int c = wave; c * 64 < nb; c += kSelWaves) {
    const int lp = 64 * c + lane;
    int64_t page = lp < nb ? bt[lp] : -1;
    if (page >= a.num_pages) page = -1;
    float scale = 0.0f;
    if (page >= 0) scale = reinterpret_cast<const float*>(a.summary + page * a.summary_stride + a.kv_heads * D)[h];
    i32x4 mk[4][S];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int64_t pg = __shfl(static_cast<int>(page), 16 * u + m, 64);
#pragma unroll
      for (int s = 0; s < S; ++s) {
        mk[u][s] = i32x4{};
        if (pg >= 0)
          mk[u][s] = *reinterpret_cast<const i32x4*>(a.summary + pg * a.summary_stride + h * D + 64 * s + 16 * g);
      }
    }
    int best = 0;
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      int mx = -0x7fffffff;
      for (int r = 0; r < tiles; ++r) {
        i32x4 acc = {};
#pragma unroll
        for (int s = 0; s < S; ++s) {
          const i32x4 qa = *reinterpret_cast<const i32x4*>(qc + (16 * r + m) * D + 64 * s + 16 * g);
          acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(qa, mk[u][s], acc, 0, 0, 0);
        }
        mx = max(max(mx, max(acc[0], acc[1])), max(acc[2], acc[3]));
      }
      mx = max(mx, __shfl_xor(mx, 16, 64));
      mx = max(mx, __shfl_xor(mx, 32, 64));
      if (g == u) best = mx;  // page 16 u + m of the chunk: this lane's
    }
    uint32_t key = 0;
    if (page >= 0) {
      key = score_key(static_cast<float>(best) * scale);
      if (lp < a.keep_first || lp >= all - a.keep_last) key = 0xffffffffu;
    }
    keys[64 * c + lane] = key;
  }
  const int chunks = (nb + 63) / 64;

  // the n-th largest key: 11, 11 and 10 bits
  uint32_t prefix = 0, mask = 0, need = static_cast<uint32_t>(a.n);
#pragma unroll
  for (int round = 0; round < 3; ++round) {
    const int shift = round == 0 ? 21 : round == 1 ? 10 : 0;
    const uint32_t width = round == 2 ? 1024u : 2048u;
    for (int i = tid; i < kSelBins; i += kSelThreads) bins[i] = 0;
    if (tid == 0) found[0] = 0, found[1] = 0xffffffffu;
    __syncthreads();
    for (int i = tid; i < chunks * 64; i += kSelThreads) {
      const uint32_t key = keys[i];
      if ((key & mask) == prefix && key) atomicAdd(&bins[(key >> shift) & (width - 1)], 1u);
    }
    __syncthreads();
    const uint32_t lo = bins[2 * tid], hi = bins[2 * tid + 1];
    const uint32_t above = count_above(lo + hi, tmp);
    // the bin with fewer than `need` keys above it and at least that many with its own
    if (above < need && above + hi >= need) found[0] = 2 * tid + 1, found[1] = need - above;
    else if (above + hi < need && above + hi + lo >= need) found[0] = 2 * tid, found[1] = need - above - hi;
    __syncthreads();
    if (found[1] == 0xffffffffu) {  // fewer keys than n: all of them
      prefix = 1, mask = 0xffffffffu, need = 0;
      break;
    }
    prefix |= found[0] << shift;
    mask |= (width - 1) << shift;
    need = found[1];
    __syncthreads();
  }
  // keys above `prefix`, and the first `need` of those equal to it
  for (int c = wave; c < chunks; c += kSelWaves) {
    const uint32_t key = keys[64 * c + lane];
    const uint64_t gt = __ballot(need ? key > prefix : key != 0), eq = __ballot(need && key == prefix);
    if (lane == 0) chunk[c] = static_cast<uint32_t>(__builtin_popcountll(gt)) |
                              static_cast<uint32_t>(__builtin_popcountll(eq)) << 16;
  }
  __syncthreads();
  // sums of the chunks before each, in order; a wave's 64 chunks at a time
  uint32_t gsum = 0, esum = 0;
  if (tid < 512) {
    const uint32_t v = tid < chunks ? chunk[tid] : 0;
    gsum = v & 0xffffu, esum = v >> 16;
#pragma unroll
    for (int k = 1; k < 64; k <<= 1) {
      const uint32_t x = __shfl_up(gsum, k, 64), y = __shfl_up(esum, k, 64);
      if (lane >= k) gsum += x, esum += y;
    }
    if (lane == 63) bins[wave] = gsum, bins[16 + wave] = esum;
    gsum -= v & 0xffffu, esum -= v >> 16;
  }
  __syncthreads();
  uint32_t* const gb = bins + 64;
  uint32_t* const eb = bins + 64 + 512;
  if (tid < 512) {
    for (int w = 0; w < wave; ++w) gsum += bins[w], esum += bins[16 + w];
    gb[tid] = gsum, eb[tid] = esum;
  }
  __syncthreads();
  uint32_t total = 0;
  if (chunks) {
    const uint32_t last = chunk[chunks - 1];
    total = gb[chunks - 1] + (last & 0xffffu) + min(eb[chunks - 1] + (last >> 16), need);
  }
  for (int c = wave; c < chunks; c += kSelWaves) {
    const uint32_t key = keys[64 * c + lane];
    const bool is_gt = need ? key > prefix : key != 0, is_eq = need && key == prefix;
    const uint64_t below = (1ull << lane) - 1;
    const uint32_t gr = gb[c] + static_cast<uint32_t>(__builtin_popcountll(__ballot(is_gt) & below));
    const uint32_t er = eb[c] + static_cast<uint32_t>(__builtin_popcountll(__ballot(is_eq) & below));
    if (is_gt || (is_eq && er < need)) out[gr + min(er, need)] = 64 * c + lane;
  }
  for (uint32_t i = total + tid; i < static_cast<uint32_t>(a.n); i += kSelThreads) out[i] = -1;
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
  EKV_CHECK(q && summary && block_table && positions && req_ids && blocks, "null pointer");
  EKV_CHECK(summary_stride >= gqa_summary_bytes(kv_heads, dim) && summary_stride % 16 == 0 && aligned16(summary),
            "summary_stride must be a multiple of 16 of at least kv_heads * (dim + 4) bytes");
  EKV_CHECK(num_pages < (int64_t{1} << 31), "too many pages");
  const int64_t grid = static_cast<int64_t>(num_tokens) * kv_heads;
  EKV_CHECK(grid < (int64_t{1} << 31), "too many rows for one call");
  GqaSelectArgs a{};
  a.q = q, a.q_tok_stride = q_tok_stride, a.q_head_stride = q_head_stride;
  a.num_tokens = num_tokens, a.heads = heads, a.kv_heads = kv_heads, a.group = heads / kv_heads;
  a.summary = summary, a.summary_stride = summary_stride, a.num_pages = num_pages;
  a.block_table = block_table, a.bt_stride = bt_stride, a.bt_width = bt_width, a.num_seqs = num_seqs;
  a.positions = positions, a.req_ids = req_ids;
  a.max_blocks = (max_len + kPageTokens - 1) / kPageTokens;
  a.n = num_blocks, a.keep_first = keep_first, a.keep_last = keep_last;
  a.ids = blocks, a.ids_tok_stride = blocks_tok_stride, a.ids_head_stride = blocks_head_stride;
  const uint32_t lds = static_cast<uint32_t>((a.max_blocks + 63) / 64 * 64) * 4;
  auto* const kernel = dim == 64 ? gqa_block_select_kernel<64>
                       : dim == 128 ? gqa_block_select_kernel<128> : gqa_block_select_kernel<256>;
  if (lds > 32768)  // over 64 KB with the static part
    (void)hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize,
                              static_cast<int>(lds));
  kernel<<<dim3(static_cast<uint32_t>(grid)), kSelThreads, lds, static_cast<hipStream_t>(stream)>>>(a);
  return ekv_launch_status();
}
