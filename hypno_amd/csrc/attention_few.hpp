// What the kernels for few rows share: the pages that were selected for a token, and
// the end, where a work-group's waves add up their parts.
#pragma once

#include "attention.hpp"

namespace hypno {

constexpr int kFewQ = kFewRows;  // rows of a pass: one MFMA's
constexpr int kFewKeys = 32;     // keys of a wave's tile

// Bytes of a wave's part: o of its rows, maxima and sums.
template <int DP>
constexpr int few_part_bytes() {
  return kFewQ * (DP + 4) * 4 + kFewQ * 8;
}

// A selected page: its place in the cache (-1: none of it) and how many of its positions
// are seen (at least one).
struct SeenPage {
  int page, seen;
};

// Fills `list` in LDS with the pages that the `count` numbers at `selected` name and the
// token at `pos` of sequence b sees, in their order; all threads get how many.
__device__ __forceinline__ int seen_pages(const AttnArgs& a, int b, int pos, const int* selected,
                                          SeenPage* list, int* counts) {
  const int tid = threadIdx.x, lane = tid & 63, waves = blockDim.x >> 6;
  const int own = pos < 0 ? -1 : pos >> a.c.page_shift;
  int n = 0;
  for (int e0 = 0; e0 < a.count; e0 += blockDim.x) {
    const int e = e0 + tid, at = e < a.count ? load_global<int>(selected + e) : -1;
    const bool in = at >= 0 && at <= own;
    int page = -1;
    if (in) page = load_global<int>(a.b.page_table + (size_t)b * a.b.width + at);
    if (page >= a.c.pages) page = -1;
    const uint64_t m = __ballot(in);
    if (lane == 0) counts[tid >> 6] = __popcll(m);
    __syncthreads();
    int before = n + __popcll(m & ((1ull << lane) - 1));
    for (int w = 0; w < waves; w++) {
      if (w < tid >> 6) before += counts[w];
      n += counts[w];
    }
    if (in)
      list[before] = {page, (int)min((int64_t)1 << a.c.page_shift,
                                     (int64_t)pos + 1 - ((int64_t)at << a.c.page_shift))};
    __syncthreads();
  }
  return __builtin_amdgcn_readfirstlane(n);
}

// A run of kLen positions in a selected page, or where what is seen of it ends before, its last
// one that is seen: its first slot, and the last of its positions that is seen.
struct SeenRun {
  int page, slot, last;
  int seen;  // positions of the run that was asked for that are seen (0 to kLen)
};
template <int kLen = kRun>
__device__ __forceinline__ SeenRun seen_run(const AttnArgs& a, const SeenPage* list, int p) {
  const SeenPage x = list[p >> a.c.page_shift];
  const int page = __builtin_amdgcn_readfirstlane(x.page);
  const int end = __builtin_amdgcn_readfirstlane(x.seen);
  const int slot = p & ((1 << a.c.page_shift) - 1), start = min(slot, (end - 1) & -kLen);
  return {page, start, min(end - 1 - start, kLen - 1), min(max(end - slot, 0), kLen)};
}

// Bits of the kFewQ rows that wave `wave` computes again, where that is needed.
template <int kWaves>
__device__ __forceinline__ uint32_t again_mask(int wave) {
  return (kWaves == 8 ? 0x0101u : 0x1111u) << wave;
}

// The waves' parts (x, each in kWave bytes of smem) to the output, or the range's place:
// thread (row, piece) takes four elements.  Rows r0 and on of `rows`, kPass of them at most;
// kList: they are the heads of token ti.
template <int DP, int kWaves, int kWave, int kPass, bool kList, typename R>
__device__ __forceinline__ void few_store(const AttnArgs& a, const Seq& sq, int g, int ti, int r0,
                                          int rows, int split, bool past, const R& x,
                                          uint8_t* smem, uint32_t& again) {
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int G = a.group, D = a.c.head_dim, col = lane % kFewQ;
  float* const part = reinterpret_cast<float*>(smem + wave * kWave);
  float2* const ml = reinterpret_cast<float2*>(part + kFewQ * (DP + 4));
#pragma unroll
  for (int k = 0; k < R::kDt; k++)
    *reinterpret_cast<f32x4*>(part + col * (DP + 4) + R::dim(k, 0)) =
        f32x4{x.o[k][0], x.o[k][1], x.o[k][2], x.o[k][3]};
  if (lane < kFewQ) ml[col] = make_float2(x.m, x.l);
  if (tid == 0) again = 0;
  __syncthreads();
  const int or_ = tid / (4 * kWaves), piece = tid % (4 * kWaves);
  float w[kWaves], m = -__builtin_inff(), l = 0.0f;
  auto row_of = [&](int i) {
    return reinterpret_cast<const float*>(smem + i * kWave) + or_ * (DP + 4);
  };
  auto ml_of = [&](int i) {
    return reinterpret_cast<const float2*>(smem + i * kWave + kFewQ * (DP + 4) * 4)[or_];
  };
#pragma unroll
  for (int i = 0; i < kWaves; i++) {
    w[i] = ml_of(i).x;
    m = fmaxf(m, w[i]);
  }
#pragma unroll
  for (int i = 0; i < kWaves; i++) {
    w[i] = w[i] == -__builtin_inff() ? 0.0f : __builtin_amdgcn_exp2f(w[i] - m);
    l += ml_of(i).y * w[i];
  }
  const bool live = or_ < kPass && r0 + or_ < rows;
  const int rr = min(r0 + or_, rows - 1);
  const size_t orow = kList ? (size_t)(sq.first + ti) * a.heads + g * G + rr
                            : (size_t)(sq.first + rr / G) * a.heads + g * G + rr % G;
  const size_t prow = (kList ? orow : few_part(a, sq, g, rr, orow)) * a.fs.splits + split;
  const bool parts = a.fs.splits > 1;
  const float inv = parts ? 1.0f : l == 0.0f ? 0.0f : 1.0f / l;
  float* const dst = parts ? a.fp.o + prow * D : a.out + orow * D;
  float z = l * 0.0f;
  if (live) {
    for (int d = 4 * piece; d < D; d += 16 * kWaves) {
      f32x4 v = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int i = 0; i < kWaves; i++) v += *reinterpret_cast<const f32x4*>(row_of(i) + d) * w[i];
      v *= inv;
#pragma unroll
      for (int j = 0; j < 4; j++) z += v[j] * 0.0f;
      *reinterpret_cast<f32x4*>(dst + d) = v;
    }
    if (parts && piece == 0) a.fp.ml[prow] = make_float2(m, l);
    if (!parts && (!(z == 0.0f) || past)) atomicOr(&again, 1u << or_);
  }
  // (rows again after all that is stored of them)
  if (parts && r0 + kPass >= rows) return;
  __syncthreads();
  if (again) {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    uint32_t left = again & again_mask<kWaves>(wave);
    if (kList) {
      const int* const selected =
          a.selected + ((size_t)(sq.first + ti) * a.c.kv_heads + g) * a.count;
      for (; left; left &= left - 1)
        attn_row(a, sq, ti, g * G + r0 + __ffs(left) - 1, selected, a.count);
    } else {
      attn_rows(a, sq, g, r0, left);
    }
  }
  if (r0 + kPass < rows) __syncthreads();
}

}  // namespace hypno
