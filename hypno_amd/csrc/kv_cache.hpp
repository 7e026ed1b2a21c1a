// What the kernels over a paged KV cache share: the cache, the batch of ragged
// sequences that bring new tokens, and how a work-group finds its sequence.
#pragma once

#include <algorithm>

#include "common.hpp"

namespace hypno {

constexpr int kKvFp16 = 0;  // values of HYPNO_HIP_KV_* in include/hypno_hip.h
constexpr int kKvInt8 = 1;

// K and V as [pages][kv_heads][page_size][head_dim] (one kv head's tokens of a
// page are one run of memory), fp16, or int8 codes beside [pages][kv_heads][page_size]
// fp32 scales.  Page strides are in elements.
struct KvCache {
  int dtype;
  void* k;
  void* v;
  float* k_scale;
  float* v_scale;
  size_t k_page, v_page, ks_page, vs_page;
  int pages, kv_heads, page_shift, head_dim;  // page_size = 1 << page_shift
};

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
AttnPlan attn_plan(const KvCache& c, const KvBatch& b, int heads, int window, int64_t max_kv,
                   int num_cus);
// ws: plan.bytes, 256-byte aligned, or NULL (no range is split then).
hipError_t launch_paged_attention(const AttnPlan& p, float* out, const float* q, size_t q_stride,
                                  int heads, const KvCache& c, const KvBatch& b, float scale,
                                  int window, void* ws, hipStream_t s);

}  // namespace hypno
