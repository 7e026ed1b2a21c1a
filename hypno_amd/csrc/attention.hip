// Attention of each sequence's new tokens over its pages of the cache:
//   o = sum_p w_p v_p / sum_p w_p,  w_p = exp(scale q.k_p - m)
// over the positions p that the token sees, in one pass with the running maximum
// m and sum.
#include "kv_cache.hpp"

namespace hypno {

namespace {

struct AttnArgs {
  KvCache c;
  KvBatch b;
  float* out;
  const float* q;
  size_t q_stride;
  int heads, window;
  float scale;
};

// One wave a (token, head).
template <int kType>
__global__ void __launch_bounds__(64) attn_rows_kernel(AttnArgs a) {
  const int t = blockIdx.x, h = blockIdx.y, lane = threadIdx.x;
  const int D = a.c.head_dim, g = h / (a.heads / a.c.kv_heads);
  const int b = find_seq(a.b, t, 0, 0);
  if (b < 0 || b >= a.b.batch) return;
  const int first = cu_at(a.b, b), n = cu_at(a.b, b + 1) - first;
  const int64_t kv = load_global<int>(a.b.kv_lens + b);
  const int64_t pos = kv - n + (t - first);
  const bool past = kv > ((int64_t)a.b.width << a.c.page_shift);
  float q[4], m = -__builtin_inff();
  double o[4] = {}, l = 0.0;  // (20000 additions of one value to an fp32 sum round one way)
  for (int i = 0; i < 4; i++) {
    const int e = lane + 64 * i;
    q[i] = e < D ? a.q[(size_t)t * a.q_stride + (size_t)h * D + e] * a.scale : 0.0f;
  }
  const int64_t lo = a.window ? max(pos - a.window + 1, (int64_t)0) : 0;
  for (int64_t p = lo; p <= pos && !past; p++) {
    const int page = a.b.page_table[(size_t)b * a.b.width + (p >> a.c.page_shift)];
    const bool there = page >= 0 && page < a.c.pages;
    const size_t tok = ((size_t)g << a.c.page_shift) + (p & ((1 << a.c.page_shift) - 1));
    const size_t ki = (size_t)page * a.c.k_page + tok * D, vi = (size_t)page * a.c.v_page + tok * D;
    float s = 0.0f, v[4] = {};
    if (there) {
      for (int i = 0; i < 4; i++) {
        const int e = lane + 64 * i;
        if (e >= D) continue;
        if (kType == kKvFp16) {
          s = fmaf(q[i], (float)((const _Float16*)a.c.k)[ki + e], s);
          v[i] = (float)((const _Float16*)a.c.v)[vi + e];
        } else {
          s = fmaf(q[i], (float)((const int8_t*)a.c.k)[ki + e], s);
          v[i] = (float)((const int8_t*)a.c.v)[vi + e] *
                 a.c.v_scale[(size_t)page * a.c.vs_page + tok];
        }
      }
      s = wave_sum(s);
      if (kType == kKvInt8) s *= a.c.k_scale[(size_t)page * a.c.ks_page + tok];
    } else {
      s = __builtin_nanf("");
    }
    const float mn = fmaxf(m, s);
    const float ref = mn == -__builtin_inff() ? 0.0f : mn;
    const float r = expf(m - ref), w = expf(s - ref);
    m = mn;
    l = l * r + w;
    for (int i = 0; i < 4; i++) o[i] = o[i] * r + (double)w * v[i];
  }
  for (int i = 0; i < 4; i++) {
    const int e = lane + 64 * i;
    if (e < D)
      a.out[((size_t)t * a.heads + h) * D + e] =
          past ? __builtin_nanf("") : l == 0.0 ? 0.0f : (float)(o[i] / l);
  }
}

}  // namespace

hipError_t launch_paged_attention(float* out, const float* q, size_t q_stride, int heads,
                                  const KvCache& c, const KvBatch& b, float scale, int window,
                                  hipStream_t s) {
  const AttnArgs a = {c, b, out, q, q_stride, heads, window, scale};
  const dim3 grid(b.tokens, heads);
  if (c.dtype == kKvFp16)
    attn_rows_kernel<kKvFp16><<<grid, 64, 0, s>>>(a);
  else
    attn_rows_kernel<kKvInt8><<<grid, 64, 0, s>>>(a);
  return hipGetLastError();
}

}  // namespace hypno
