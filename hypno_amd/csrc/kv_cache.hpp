// What the kernels over a paged KV cache share: the cache, the batch of ragged
// sequences that bring new tokens, and how a work-group finds its sequence.
#pragma once

#include <algorithm>

#include "common.hpp"

namespace hypno {

constexpr int kKvFp16 = 0;  // values of HYPNO_HIP_KV_* in include/hypno_hip.h
constexpr int kKvInt8 = 1;
constexpr int kKvFp4 = 2;

// K and V as [pages][kv_heads][page_size][head_dim] (one kv head's tokens of a
// page are one run of memory), fp16, or int8 codes beside [pages][kv_heads][page_size]
// fp32 scales, or 4-bit codes, two a byte, beside [pages][kv_heads][head_dim / 32][page_size]
// fp16 scales.  Page strides are in elements, of 4-bit codes in bytes.
struct KvCache {
  int dtype;
  void* k;
  void* v;
  float* k_scale;
  float* v_scale;
  size_t k_page, v_page, ks_page, vs_page;
  int pages, kv_heads, page_shift, head_dim;  // page_size = 1 << page_shift
};

// Elements of a group of 4-bit codes with one scale.
constexpr int kFp4Group = 32;

// A 4-bit code's value, exact in fp16: its sign, exponent and fraction bit in fp16's
// places have the value times 2^-14 (0.5 of it a subnormal number there too).
__device__ __forceinline__ _Float16 fp4_value(uint32_t code) {
  const uint16_t bits = (uint16_t)((code & 8) << 12 | (code & 7) << 9);
  return __builtin_bit_cast(_Float16, bits) * (_Float16)16384.0f;
}

// Eight 4-bit codes times their scale (twice in a register) -> eight fp16, each rounded
// once.
__device__ __forceinline__ u32x4 fp4_to_f16(uint32_t x, half2v scale) {
  u32x4 r;
  const half2v v[4] = {
      __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(x, 1.0f, 0),
      __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(x, 1.0f, 1),
      __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(x, 1.0f, 2),
      __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(x, 1.0f, 3)};
#pragma unroll
  for (int i = 0; i < 4; i++) r[i] = __builtin_bit_cast(uint32_t, (half2v)(v[i] * scale));
  return r;
}

// The codes of eight finite values: the nearest of 0, 0.5, 1, 1.5, 2, 3, 4, 6 and their
// negatives, halves to the even code (the conversion's own rounding).
__device__ __forceinline__ uint32_t fp4_codes(const float (&y)[8]) {
  uint32_t p = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(0u, y[0], y[1], 1.0f, 0);
  p = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(p, y[2], y[3], 1.0f, 1);
  p = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(p, y[4], y[5], 1.0f, 2);
  return __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(p, y[6], y[7], 1.0f, 3);
}

// Sequence b brings the tokens [cu_q[b], cu_q[b + 1]) of `tokens`, the last ones
// of the kv_lens[b] that it then holds; its page i is page_table[b * width + i].
struct KvBatch {
  const int* cu_q;
  const int* kv_lens;
  const int* page_table;
  int batch, width, tokens;
};

// cu_q[i] as the kernels use it: no value leads out of the token arrays.
__device__ __forceinline__ int cu_at(const KvBatch& b, int i) {
  return min(max(load_global<int>(b.cu_q + i), 0), b.tokens);
}

// The largest i in [0, batch] with cu_q[i] * g / per + i <= slot, or -1: the
// sequence of tile `slot` where sequence i's tiles of `per` rows start at that
// number (g rows a token; a sequence of n tokens has ceil(n * g / per) of them,
// and the numbers between two starts are never fewer).  With g = per = 0: the
// largest i with cu_q[i] <= slot, the sequence of token `slot`.  The whole wave
// reads 64 values at a time and counts, instead of a chain of dependent reads.
__device__ __forceinline__ int find_seq(const KvBatch& b, int slot, int g, int per) {
  const int lane = threadIdx.x & 63;
  int count = 0;
  for (int i0 = 0; i0 <= b.batch; i0 += 64) {
    const int i = i0 + lane;
    bool in = false;
    if (i <= b.batch) {
      const int c = cu_at(b, i);
      in = (per ? (int)((int64_t)c * g / per) + i : c) <= slot;
    }
    count += __popcll(__ballot(in));
  }
  return count - 1;
}

hipError_t launch_append_kv(const KvCache& c, const KvBatch& b, float* q_out, size_t q_out_stride,
                            const float* q, size_t q_stride, int heads, const float* k,
                            size_t k_stride, const float* v, size_t v_stride,
                            const float* inv_freq, int rot, bool pairs, int num_cus,
                            hipStream_t s);

// The keys' bounds of each page and kv head, [pages][kv_heads][2][head_dim] codes (the
// smallest, the largest) beside [pages][kv_heads] fp32 scales.  Page strides are in elements.
struct KeyBounds {
  int8_t* codes;
  float* scale;
  size_t page, s_page;
  int pages, kv_heads, page_shift, head_dim;
};

// The pages that hold a batch's new tokens, numbered over all sequences: where the numbers of
// sequence b begin, whose first token is `first` (n tokens are in floor((n - 1) / page_size) + 2
// pages at most).
__host__ __device__ inline int64_t first_number(int first, int b, int shift) {
  return (first >> shift) + 2 * (int64_t)b;
}

// Which of its pages `number` stands for in sequence b, which brings the tokens [first, end)
// of the kv that it holds; -1: none with a new token and a place in a table of `width`
// pages.  (Where cu_q does not ascend a number may come before the sequence's own.)
__host__ __device__ inline int page_of_number(int64_t number, int b, int first, int end, int kv,
                                              int shift, int width) {
  const int64_t own = number - first_number(first, b, shift), kept = (int64_t)kv - (end - first);
  if (own < 0 || end <= first || kv <= 0) return -1;
  const int64_t at = ((kept > 0 ? kept : 0) >> shift) + own;
  return at <= (kv - 1) >> shift && at < width ? (int)at : -1;
}

// Pages of a sequence that scores are kept of at most (in LDS).
constexpr int kMaxScored = 32768;
// Pages that a token reads at most.
constexpr int kMaxSelected = 1024;

hipError_t launch_key_bounds(const KeyBounds& o, const KvCache& c, const KvBatch& b, int num_cus,
                             hipStream_t s);
// How a call's tokens and pages are split over work-groups, and the workspace that takes.
struct SelectPlan {
  int pages;       // of a sequence
  int pitch, rows, tokens, splits, chunk;
  bool team;
  size_t bytes;
};
// `pages`: of a sequence, at most kMaxScored.
SelectPlan select_plan(int heads, const KeyBounds& k, const KvBatch& b, int pages, int num_cus);
// ws: plan.bytes, or NULL (one kernel then).
hipError_t launch_select_pages(const SelectPlan& p, int* out, int count, int first, int last,
                               const float* q, size_t q_stride, int heads, const KeyBounds& k,
                               const KvBatch& b, void* ws, hipStream_t s);
// How the positions of a tile of rows are split: into ranges of `chunk`, the last
// one of `splits` taking what is left.
struct AttnSplit {
  int splits, chunk;
};

// How a call's rows and positions are split, and the workspace that takes: a place for
// each range of each row that a kernel may have (none where it takes no ranges).
struct AttnPlan {
  int few;        // sequences of at most so many rows go to attn_few_kernel
  int few_waves;  // of its work-groups
  int tile_rows;  // rows of a work-group of attn_tile_kernel
  int cus;
  AttnSplit fs, ts;
  size_t bytes, ml_bytes;
  size_t few_places, tile_places;
  bool by_seq;    // attn_few_kernel's rows are counted by sequence, not by token
};
// The same for a token's selected pages, whose positions are counted page after page.
struct SelectedPlan {
  int waves;  // of a work-group
  AttnSplit fs;
  size_t bytes, ml_bytes;
};
SelectedPlan selected_plan(const KvCache& c, const KvBatch& b, int heads, int count, int num_cus);
hipError_t launch_selected_attention(const SelectedPlan& p, float* out, const float* q,
                                     size_t q_stride, int heads, const KvCache& c,
                                     const KvBatch& b, float scale, const int* selected, int count,
                                     void* ws, hipStream_t s);
AttnPlan attn_plan(const KvCache& c, const KvBatch& b, int heads, int window, int64_t max_kv,
                   int num_cus);
// ws: plan.bytes, 256-byte aligned, or NULL (no range is split then).
hipError_t launch_paged_attention(const AttnPlan& p, float* out, const float* q, size_t q_stride,
                                  int heads, const KvCache& c, const KvBatch& b, float scale,
                                  int window, void* ws, hipStream_t s);

}  // namespace hypno
