// New tokens' keys and values into a paged cache, keys rotated to their positions
// on the way, and the queries rotated beside them.
//
// Token t, the i-th of its sequence's n new ones, has position p = kv_len - n + i.
// Pair j of a head's first rot elements turns by the angle p * inv_freq[j]:
//   (x0, x1) -> (x0 cos - x1 sin, x1 cos + x0 sin).
// Angles, their sines and the products are in 64 bits: at position 100000 an
// fp32 angle is off by 4e-3, and a key's 8-bit codes are then those of the formula
// but for values within ~1e-16 of a border.  Each result is rounded once to fp32,
// then to the cache's type: fp16 to nearest, or int8 codes
//   s = max|x| / 127 over the head's row, code = round_half_away(x / s)
// with both quotients in fp32 (s = 0 and codes 0 where that underflows; s = NaN
// and codes 0 for a row that holds an infinity or NaN).
//
// Bound: HBM for prompts (2048 tokens, 32/8 heads of 128, 92 MB: 20.6 us, 4.5 TB/s, a
// large copy's 4.9; 999 tokens into an 8-bit cache 9.8, 1.2 TB/s), latency for few tokens (one: 4.2 us, of which an empty kernel is
// about two): the batch's arrays and the page are two dependent reads, and the sines in 64
// bits some hundred operations of one wave.  One work-group a token, so that these are
// computed once for all its heads (a work-group for each 16 of its rows: the prompt takes
// 27 us); the rows are split over several only while the chip is not full.
#include "kv_cache.hpp"

namespace hypno {

namespace {

constexpr int kAppendThreads = 256;
constexpr int kMaxHeadDim = 256;

struct AppendArgs {
  KvCache c;
  KvBatch b;
  float* q_out;
  const float* q;
  const float* k;
  const float* v;
  size_t q_out_stride, q_stride, k_stride, v_stride;
  const float* inv_freq;
  int heads, rot, pairs, vec;
  int lane_shift;  // 1 << lane_shift lanes a row, each with 8 elements
};

__device__ __forceinline__ void load8(float (&x)[8], const float* p, bool vec) {
  if (vec) {
    const float4 a = load_global<float4>(p), b = load_global<float4>(p + 4);
    x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w;
    x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
  } else {
#pragma unroll
    for (int i = 0; i < 8; i++) x[i] = load_global<float>(p + i);
  }
}

// One work-group a token (and row range: blockIdx.y); 8 elements a lane.
template <int kType>
__global__ void __launch_bounds__(kAppendThreads) append_kv_kernel(AppendArgs a) {
  __shared__ double cs[kMaxHeadDim / 2], sn[kMaxHeadDim / 2];
  const int t = blockIdx.x, tid = threadIdx.x, lane = tid & 63;
  const int D = a.c.head_dim, KV = a.c.kv_heads, half = a.rot / 2;
  const int per_wave = 64 >> a.lane_shift;
  const int unit = lane & ((1 << a.lane_shift) - 1), e0 = 8 * unit;
  const int waves = kAppendThreads / 64 * gridDim.y, all = a.heads + 2 * KV;
  int r0 = (blockIdx.y * (kAppendThreads / 64) + tid / 64) * per_wave;
  float x[8], w[8], xn[8], wn[8];  // a lane's elements, the other ones of their pairs
  auto load = [&](float (&x)[8], float (&w)[8], int r0) __attribute__((always_inline)) {
    const int row = r0 + (lane >> a.lane_shift);
#pragma unroll
    for (int i = 0; i < 8; i++) x[i] = w[i] = 0.0f;
    if (row >= all || e0 >= D) return;
    const bool is_q = row < a.heads, is_k = !is_q && row < a.heads + KV;
    const float* src = is_q   ? a.q + (size_t)t * a.q_stride + (size_t)row * D
                       : is_k ? a.k + (size_t)t * a.k_stride + (size_t)(row - a.heads) * D
                              : a.v + (size_t)t * a.v_stride + (size_t)(row - a.heads - KV) * D;
    load8(x, src + e0, a.vec);
    if ((is_q || is_k) && !a.pairs) {
      // Read before anything is written, as a row belongs to one wave (q_out may be q).
      if (half % 8 == 0) {
        if (e0 < a.rot) load8(w, src + (e0 < half ? e0 + half : e0 - half), a.vec);
      } else {
#pragma unroll
        for (int i = 0; i < 8; i++) {
          const int e = e0 + i;
          if (e < a.rot) w[i] = load_global<float>(src + (e < half ? e + half : e - half));
        }
      }
    }
  };
  // The first rows and the frequencies come in while the token's place is looked up.
  load(xn, wn, r0);
  const float freq = tid < half ? load_global<float>(a.inv_freq + tid) : 0.0f;
  const int b = find_seq(a.b, t, 0, 0);
  if (b < 0 || b >= a.b.batch) return;  // a token of no sequence
  const int first = cu_at(a.b, b), n = cu_at(a.b, b + 1) - first;
  const int64_t pos = (int64_t)load_global<int>(a.b.kv_lens + b) - n + (t - first);
  const int64_t at = pos >> a.c.page_shift;
  int page = -1;
  if (pos >= 0 && at < a.b.width)
    page = load_global<int>(a.b.page_table + (size_t)b * a.b.width + at);
  if (tid < half) sincos((double)pos * (double)freq, &sn[tid], &cs[tid]);
  __syncthreads();
  const bool stored = page >= 0 && page < a.c.pages;
  const int slot = (int)(pos & ((1 << a.c.page_shift) - 1));
  for (; r0 < all; r0 += waves * per_wave) {
#pragma unroll
    for (int i = 0; i < 8; i++) x[i] = xn[i], w[i] = wn[i];
    load(xn, wn, r0 + waves * per_wave);
    const int row = r0 + (lane >> a.lane_shift);
    const bool is_q = row < a.heads, is_k = !is_q && row < a.heads + KV;
    const int h = is_q ? row : is_k ? row - a.heads : row - a.heads - KV;
    const bool live = row < all && e0 < D && (is_q || stored);
    if (live && (is_q || is_k)) {
      if (a.pairs) {
#pragma unroll
        for (int i = 0; i < 8; i++) w[i] = x[i ^ 1];
      }
#pragma unroll
      for (int i = 0; i < 8; i++) {
        const int e = e0 + i;
        if (e >= a.rot) continue;
        const bool second = a.pairs ? i & 1 : e >= half;
        const int j = a.pairs ? e / 2 : second ? e - half : e;
        const double s = second ? sn[j] : -sn[j];
        x[i] = (float)fma((double)w[i], s, (double)x[i] * cs[j]);
      }
    }
    if (live && is_q) {
      float* dst = a.q_out + (size_t)t * a.q_out_stride + (size_t)h * D + e0;
      if (a.vec) {
        reinterpret_cast<float4*>(dst)[0] = make_float4(x[0], x[1], x[2], x[3]);
        reinterpret_cast<float4*>(dst)[1] = make_float4(x[4], x[5], x[6], x[7]);
      } else {
#pragma unroll
        for (int i = 0; i < 8; i++) dst[i] = x[i];
      }
    }
    const size_t tok = ((size_t)h << a.c.page_shift) + slot;
    if (kType == kKvFp16) {
      if (live && !is_q) {
        _Float16* dst = (is_k ? (_Float16*)a.c.k + (size_t)page * a.c.k_page
                              : (_Float16*)a.c.v + (size_t)page * a.c.v_page) + tok * D + e0;
        u32x4 p;
#pragma unroll
        for (int i = 0; i < 4; i++)
          p[i] = __builtin_bit_cast(uint16_t, (_Float16)x[2 * i]) |
                 ((uint32_t)__builtin_bit_cast(uint16_t, (_Float16)x[2 * i + 1]) << 16);
        *reinterpret_cast<u32x4*>(dst) = p;
      }
    } else {
      // By bit pattern infinities and NaN are above every finite value.
      uint32_t mb = 0;
#pragma unroll
      for (int i = 0; i < 8; i++) mb = max(mb, __float_as_uint(x[i]) & 0x7FFFFFFFu);
      for (int off = 1 << a.lane_shift >> 1; off > 0; off >>= 1)
        mb = max(mb, (uint32_t)__shfl_xor((int)mb, off, 64));
      if (live && !is_q) {
        const float amax = __uint_as_float(mb);
        const float s = mb < 0x7F800000u ? amax / 127.0f : __builtin_nanf("");
        uint32_t p[2] = {0, 0};
        if (s > 0.0f) {
#pragma unroll
          for (int i = 0; i < 8; i++) {
            const float y = fminf(fmaxf(roundf(x[i] / s), -127.0f), 127.0f);
            p[i / 4] |= ((uint32_t)(int)y & 0xFFu) << 8 * (i % 4);
          }
        }
        int8_t* dst = (is_k ? (int8_t*)a.c.k + (size_t)page * a.c.k_page
                            : (int8_t*)a.c.v + (size_t)page * a.c.v_page) + tok * D + e0;
        *reinterpret_cast<uint2*>(dst) = make_uint2(p[0], p[1]);
        if (unit == 0)
          (is_k ? a.c.k_scale + (size_t)page * a.c.ks_page
                : a.c.v_scale + (size_t)page * a.c.vs_page)[tok] = s;
      }
    }
  }
}

}  // namespace

hipError_t launch_append_kv(const KvCache& c, const KvBatch& b, float* q_out, size_t q_out_stride,
                            const float* q, size_t q_stride, int heads, const float* k,
                            size_t k_stride, const float* v, size_t v_stride,
                            const float* inv_freq, int rot, bool pairs, int num_cus,
                            hipStream_t s) {
  AppendArgs a = {c, b, q_out, q, k, v, q_out_stride, q_stride, k_stride, v_stride,
                  inv_freq, heads, rot, pairs, 0, 0};
  while (8 << a.lane_shift < c.head_dim) a.lane_shift++;
  a.vec = ((((uintptr_t)q | (uintptr_t)q_out | (uintptr_t)k | (uintptr_t)v) & 15) == 0) &&
          ((q_stride | q_out_stride | k_stride | v_stride) & 3) == 0;
  // A token's rows are split over work-groups while the chip is not full.
  const int rows_wg = kAppendThreads / 64 * (64 >> a.lane_shift);
  const int most = (heads + 2 * c.kv_heads + rows_wg - 1) / rows_wg;
  const int split = std::min(most, std::max(1, 4 * num_cus / b.tokens));
  const dim3 grid(b.tokens, split);
  if (c.dtype == kKvFp16)
    append_kv_kernel<kKvFp16><<<grid, kAppendThreads, 0, s>>>(a);
  else
    append_kv_kernel<kKvInt8><<<grid, kAppendThreads, 0, s>>>(a);
  return hipGetLastError();
}

}  // namespace hypno
