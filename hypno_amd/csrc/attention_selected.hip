// Attention of new tokens over pages that were selected for each of them.
#include "attention.hpp"

namespace hypno {

namespace {

// One wave a (token, head).
__global__ void __launch_bounds__(64) selected_rows_kernel(AttnArgs a, const int* selected,
                                                           int count) {
  const int t = blockIdx.x / a.heads, h = blockIdx.x % a.heads;
  const int b = find_seq(a.b, t, 0, 0);
  if (b < 0 || b >= a.b.batch) return;
  const Seq sq = seq_of(a.b, b);
  attn_row(a, sq, t - sq.first, h,
           selected + ((size_t)t * a.c.kv_heads + h / a.group) * count, count);
}

}  // namespace

hipError_t launch_selected_attention(float* out, const float* q, size_t q_stride, int heads,
                                     const KvCache& c, const KvBatch& b, float scale,
                                     const int* selected, int count, hipStream_t s) {
  AttnArgs a = {};
  a.c = c, a.b = b, a.out = out, a.q = q, a.q_stride = q_stride, a.heads = heads;
  a.group = heads / c.kv_heads, a.scale = scale;
  selected_rows_kernel<<<(unsigned)b.tokens * (unsigned)heads, 64, 0, s>>>(a, selected, count);
  return hipGetLastError();
}

}  // namespace hypno
