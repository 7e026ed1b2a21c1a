// What the attention kernels share: their arguments, the row that is computed
// plainly, and the step of one wave over a tile of keys on MFMA.
//
//   o = sum_p w_p v_p / sum_p w_p,  w_p = exp(scale q.k_p - m)
// over the positions p that a token sees, in one pass with the running maximum m
// and sum.  A row is one (token, head); the rows of a sequence that read one kv
// head, token after token, `group` heads a token, form the columns of the products
//   S^T = K q^T,  O^T = V^T w^T,
// so that a lane holds one row's scores and its part of one row's output, and the
// scores' registers are the second product's operand as they are.
//
// Arithmetic: the cache's values are fp16 or 8-bit codes, both exact as MFMA operands.
// q (scaled by a power of two per row) goes in as two fp16, 22 bits, every product
// twice.  The weights times the values' scale go in as three bf16, all of an fp32, beside
// 8-bit values: a code of 0 beside the largest weight leaves an element to the smallest.
// Beside fp16 values they go in as two fp16: 22 bits down to 2^-15 of the row's largest, and
// steps of 2^-36 of that largest below.  That adds at most 2^-37 of the sum of the |values|
// seen to an element, far less than the heaviest keys' own values round off, but all that
// there is where those are 0 and the rest weighs e^-26.  (fp16 values are no bf16: three
// parts of the weights would take two of the values and three times the products.)
// Sums are fp32.  What this cannot hold (infinities and NaN anywhere in a tile, masked
// places among them, pages that are none) ends in a sum that is no finite number, and
// such a row is computed again by attn_row.
#pragma once

#include "kv_cache.hpp"

namespace hypno {

typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf8 __attribute__((ext_vector_type(8)));
typedef uint32_t uint2_t __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4), aligned(4)));  // (rows at any float)

// What the ranges of rows gave: [row][range], of o [head_dim] each.
struct AttnParts {
  float2* ml;  // maximum (log2), sum
  float* o;
};

// Rows of a sequence that attn_few_kernel takes beside attn_tile_kernel.
constexpr int kFewRows = 16;

struct AttnArgs {
  KvCache c;
  KvBatch b;
  float* out;
  const float* q;
  size_t q_stride;
  int heads, group, window;
  float scale;
  int few;                // sequences of at most so many rows are attn_few_kernel's
  int few_waves;          // of its work-groups (4 or 8)
  int tile_rows;          // rows of a work-group of the other
  AttnSplit fs, ts;       // of attn_few_kernel and attn_tile_kernel
  int cus;
  int by_seq;             // fp's rows: see few_part
  AttnParts fp, tp;       // of the two kernels, where they take ranges
};

// The new tokens of a sequence and what it holds (both at least 0).
struct Seq {
  int b, first, n, kv;
};

// (the same in all lanes)
__device__ __forceinline__ Seq seq_of(const KvBatch& b, int i) {
  const int first = __builtin_amdgcn_readfirstlane(cu_at(b, i));
  const int end = __builtin_amdgcn_readfirstlane(cu_at(b, i + 1));
  const int kv = __builtin_amdgcn_readfirstlane(load_global<int>(b.kv_lens + i));
  return {i, first, max(end - first, 0), max(kv, 0)};
}

// A sequence longer than its table row: its tokens are NaN.
__device__ __forceinline__ bool too_long(const AttnArgs& a, const Seq& s) {
  return s.kv > ((int64_t)a.b.width << a.c.page_shift);
}

// First position that token i of a sequence sees; the last is kv - n + i.
__device__ __forceinline__ int first_seen(const AttnArgs& a, const Seq& s, int i) {
  return a.window ? (int)max((int64_t)s.kv - s.n + i - a.window + 1, (int64_t)0) : 0;
}

// A run of kRun positions from a multiple of it lies in one page, if pages have as many.
constexpr int kRunShift = 4, kRun = 1 << kRunShift;

// Positions that the rows [r0, r1) of a sequence read, from the start of a run (of the
// page's start, where pages are shorter): those before the first that is seen are in its
// page.
struct Span {
  int lo, hi;
};
__device__ __forceinline__ Span span_of(const AttnArgs& a, const Seq& s, int r0, int r1) {
  const int lo = first_seen(a, s, r0 / a.group), hi = s.kv - s.n + (r1 - 1) / a.group + 1;
  if (hi <= lo) return {0, 0};
  return {lo & -(1 << min(a.c.page_shift, kRunShift)), hi};
}

// Ranges that a span is split into (0: nothing is seen).
__device__ __forceinline__ int split_count(const AttnSplit& sp, const Span& x) {
  return x.hi <= x.lo ? 0 : min(sp.splits, (x.hi - x.lo - 1) / sp.chunk + 1);
}

// Row r (of kv head g) of a sequence, `row` of all (token, head), among the rows of fp: by
// sequence kFewRows for each kv head, where both kernels run and that is less than a row
// for each (token, head), which it is otherwise (as in tp).
__device__ __forceinline__ size_t few_part(const AttnArgs& a, const Seq& s, int g, int r,
                                           size_t row) {
  return a.by_seq ? ((size_t)s.b * a.c.kv_heads + g) * kFewRows + r : row;
}

// One row by a wave, plainly, sums in 64 bits.
__device__ __forceinline__ void attn_row(const AttnArgs& a, const Seq& sq, int i, int h) {
  const int lane = threadIdx.x & 63, t = sq.first + i;
  const int D = a.c.head_dim, g = h / a.group;
  const int pos = sq.kv - sq.n + i;
  const bool past = too_long(a, sq);
  float q[4], m = -__builtin_inff();
  double o[4] = {}, l = 0.0;
  for (int j = 0; j < 4; j++) {
    const int e = lane + 64 * j;
    q[j] = e < D ? a.q[(size_t)t * a.q_stride + (size_t)h * D + e] * a.scale : 0.0f;
  }
  for (int p = first_seen(a, sq, i); p <= pos && !past; p++) {
    const int page = a.b.page_table[(size_t)sq.b * a.b.width + (p >> a.c.page_shift)];
    const bool there = page >= 0 && page < a.c.pages;
    const size_t tok = ((size_t)g << a.c.page_shift) + (p & ((1 << a.c.page_shift) - 1));
    const size_t ki = (size_t)page * a.c.k_page + tok * D, vi = (size_t)page * a.c.v_page + tok * D;
    float s = 0.0f, v[4] = {};
    if (there) {
      for (int j = 0; j < 4; j++) {
        const int e = lane + 64 * j;
        if (e >= D) continue;
        if (a.c.dtype == kKvFp16) {
          s = fmaf(q[j], (float)((const _Float16*)a.c.k)[ki + e], s);
          v[j] = (float)((const _Float16*)a.c.v)[vi + e];
        } else {
          s = fmaf(q[j], (float)((const int8_t*)a.c.k)[ki + e], s);
          v[j] = (float)((const int8_t*)a.c.v)[vi + e] *
                 a.c.v_scale[(size_t)page * a.c.vs_page + tok];
        }
      }
      s = wave_sum(s);
      if (a.c.dtype == kKvInt8) s *= a.c.k_scale[(size_t)page * a.c.ks_page + tok];
    } else {
      s = __builtin_nanf("");
    }
    const float mn = fmaxf(m, s);
    const float ref = mn == -__builtin_inff() ? 0.0f : mn;
    const float r = expf(m - ref), w = expf(s - ref);
    m = mn;
    l = l * r + w;
    for (int j = 0; j < 4; j++) o[j] = o[j] * r + (double)w * v[j];
  }
  for (int j = 0; j < 4; j++) {
    const int e = lane + 64 * j;
    if (e < D)
      a.out[((size_t)t * a.heads + h) * D + e] =
          past ? __builtin_nanf("") : l == 0.0 ? 0.0f : (float)(o[j] / l);
  }
}

// Rows r of `seq` (kv head g) whose bit r - r0 is set, one after the other.
__device__ __forceinline__ void attn_rows(const AttnArgs& a, const Seq& s, int g, int r0,
                                          uint64_t rows) {
  while (rows) {
    const int r = r0 + __ffsll((unsigned long long)rows) - 1;
    rows &= rows - 1;
    attn_row(a, s, r / a.group, g * a.group + r % a.group);
  }
}

// --- tiles of K and V in LDS --------------------------------------------------------

// Rows of DP fp16 in 16-byte pieces; piece c of row r lies at c ^ swz(r).  Sixteen
// rows' pieces c, and the 32- or 64-byte parts of four or eight rows that one
// transposing read takes, then lie in different banks.
template <int DP>
struct KvTile {
  static constexpr int kCh = DP / 8, kPitch = DP * 2;
  __device__ static __forceinline__ int swz(int r) {
    const int low = ((r >> 1) & 2) | ((r >> 3) & 1);
    if (kCh % 16 == 0) return ((r & 3) << 2) | low;
    if (kCh % 8 == 0) return ((r >> 1) & 1) << 2 | low;
    return low;
  }
  __device__ static __forceinline__ int at(int r, int c) { return r * kPitch + ((c ^ swz(r)) << 4); }
};

// Lane i's 16 bytes at base + off to lds + 16 i, asynchronously; counted by vmcnt, which
// the caller waits for.  (Not the builtin: the compiler then has every transposing read
// of LDS wait for all such copies, the next tile's too.)  kNt: read once, not kept.
template <bool kNt = false>
__device__ __forceinline__ void dma16(const void* base, uint32_t off, uint8_t* lds) {
#if defined(__HIP_DEVICE_COMPILE__)
  const uint32_t at = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) void*)lds;
  if (kNt)
    asm volatile("s_nop 0\n\tglobal_load_lds_dwordx4 %1, %2 nt"
                 :
                 : "{m0}"(at), "v"(off), "s"(base)
                 : "memory");
  else
    asm volatile("s_nop 0\n\tglobal_load_lds_dwordx4 %1, %2"
                 :
                 : "{m0}"(at), "v"(off), "s"(base)
                 : "memory");
#endif
}
__device__ __forceinline__ void dma16(const void* src, uint8_t* lds) {
#if defined(__HIP_DEVICE_COMPILE__)
  const uint32_t at = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) void*)lds;
  asm volatile("s_nop 0\n\tglobal_load_lds_dwordx4 %1, off"
               :
               : "{m0}"(at), "v"(src)
               : "memory");
#endif
}

__device__ __forceinline__ half8 f16x8(u32x4 x) { return __builtin_bit_cast(half8, x); }
__device__ __forceinline__ bf8 bf16x8(u32x4 x) { return __builtin_bit_cast(bf8, x); }

// Two fp32 -> fp16 each (toward zero), and what these leave in fp16.  `neg`: -1 that
// the compiler does not see (it then takes fp16 and fp32 into one instruction).
__device__ __forceinline__ void split_f16(float x, float y, float neg, uint32_t& h, uint32_t& l) {
  const half2v a = __builtin_bit_cast(half2v, __builtin_amdgcn_cvt_pkrtz(x, y));
  const half2v b = {(_Float16)fmaf((float)a[0], neg, x), (_Float16)fmaf((float)a[1], neg, y)};
  h = __builtin_bit_cast(uint32_t, a);
  l = __builtin_bit_cast(uint32_t, b);
}

// Two fp32 -> three bf16 each, first eight bits first: all 24 bits, fp32's range.
__device__ __forceinline__ void split_bf16(float x, float y, uint32_t& h, uint32_t& l,
                                           uint32_t& r) {
  const float xh = __uint_as_float(__float_as_uint(x) & 0xFFFF0000u), xr = x - xh;
  const float yh = __uint_as_float(__float_as_uint(y) & 0xFFFF0000u), yr = y - yh;
  const float xl = __uint_as_float(__float_as_uint(xr) & 0xFFFF0000u);
  const float yl = __uint_as_float(__float_as_uint(yr) & 0xFFFF0000u);
  h = __builtin_amdgcn_perm(__float_as_uint(y), __float_as_uint(x), 0x07060302u);
  l = __builtin_amdgcn_perm(__float_as_uint(yr), __float_as_uint(xr), 0x07060302u);
  r = __builtin_amdgcn_perm(__float_as_uint(yr - yl), __float_as_uint(xr - xl), 0x07060302u);
}

// Eight 8-bit codes -> eight bf16 (exact).
__device__ __forceinline__ u32x4 codes_to_bf16(uint2 x) {
  u32x4 r;
#pragma unroll
  for (int i = 0; i < 4; i++) {
    const int u = (int)((i < 2 ? x.x : x.y) >> 16 * (i % 2));
    const float a = (float)(int8_t)u, b = (float)(int8_t)(u >> 8);
    r[i] = __builtin_amdgcn_perm(__float_as_uint(b), __float_as_uint(a), 0x07060302u);
  }
  return r;
}

// Eight 8-bit codes -> eight fp16 (exact).
__device__ __forceinline__ u32x4 codes_to_f16(uint2 x) {
  return unpack8_bytes(x.x ^ 0x80808080u, x.y ^ 0x80808080u);
}

__device__ __forceinline__ int page_id(const AttnArgs& a, int b, int p) {
  return load_global<int>(a.b.page_table + (size_t)b * a.b.width + (p >> a.c.page_shift));
}
// The page to read for an entry of the table: 0, with *bad set, where it is none.
__device__ __forceinline__ int page_of(const AttnArgs& a, int id, bool& bad) {
  const bool ok = id >= 0 && id < a.c.pages;
  bad |= !ok;
  return ok ? id : 0;
}

// --- one wave's rows ------------------------------------------------------------------

// NQ rows (16 or 32) a wave, one a lane of each of 64 / NQ groups.
template <int NQ>
struct Mfma;
template <>
struct Mfma<32> {
  typedef float acc __attribute__((ext_vector_type(16)));
  __device__ static __forceinline__ acc mul(half8 a, half8 b, acc c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
  }
  __device__ static __forceinline__ acc mul(bf8 a, bf8 b, acc c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
  }
  // (the maximum, sum) over the lanes of one row
  __device__ static __forceinline__ float max(float x) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false,
                                                    false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
  }
  __device__ static __forceinline__ float sum(float x) { return x + __shfl_xor(x, 32, 64); }
};
template <>
struct Mfma<16> {
  typedef float acc __attribute__((ext_vector_type(4)));
  __device__ static __forceinline__ acc mul(half8 a, half8 b, acc c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
  }
  __device__ static __forceinline__ acc mul(bf8 a, bf8 b, acc c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
  }
  __device__ static __forceinline__ float max(float x) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false,
                                                    false);
    return Mfma<32>::max(fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1])));
  }
  __device__ static __forceinline__ float sum(float x) {
    x += __shfl_xor(x, 16, 64);
    return x + __shfl_xor(x, 32, 64);
  }
};

// The weights go in as 2^kTop at a row's largest score when its reference was last
// moved, and at most as 2^(kTop + kSlack), where fp16 ends (its smallest step is then
// between 2^-36 and 2^-40 of the largest weight).  The more slack, the fewer moves, each
// of which takes o times a factor.

template <int kType, int NQ, int DP, int BK>
struct Rows {
  static constexpr int NG = 64 / NQ;          // lane groups
  static constexpr int kSteps = DP / (8 * NG);  // of a score's sum
  static constexpr int kAcc = NQ * NQ / 64;
  static constexpr int kQuads = BK / (4 * NG);  // of keys a lane holds: 4 NG u + 4 group + 0..3
  static constexpr int kPv = kQuads / 2;      // steps of the second product
  static constexpr int kDt = DP / NQ;
  static constexpr float kTop = kType == kKvFp16 ? 12.0f : 0.0f;
  static constexpr float kSlack = kType == kKvFp16 ? 3.9f : 16.0f;
  typedef typename Mfma<NQ>::acc acc;

  half8 qh[kSteps], ql[kSteps];
  acc o[kDt];
  float m, l;   // reference (log2 units); this lane's part of the sum
  float c;      // scores to log2 units

  // First of the eight elements that a lane holds for step s of a score's sum.  kPairs:
  // two steps' elements side by side, so that 8-bit keys are read sixteen at a time.
  template <bool kPairs>
  __device__ static __forceinline__ int element(int s) {
    const int grp = (threadIdx.x & 63) / NQ;
    return kPairs && s < kSteps / 2 * 2 ? 8 * (NG * (s & ~1) + 2 * grp + (s & 1))
                                        : 8 * (NG * s + grp);
  }

  // `src`: the row's q, or NULL.  Rows are scaled by a power of two to at most 2^15.
  __device__ __forceinline__ void init(const float* src, int D, float scale, bool pairs = false) {
    float x[kSteps][8];
    uint32_t mb = 0;
#pragma unroll
    for (int s = 0; s < kSteps; s++) {
      const int d = pairs ? element<true>(s) : element<false>(s);
#pragma unroll
      for (int j = 0; j < 8; j++) x[s][j] = 0.0f;
      if (src && d < D) {
        const f32x4 u = load_global<f32x4>(src + d), v = load_global<f32x4>(src + d + 4);
#pragma unroll
        for (int j = 0; j < 8; j++) x[s][j] = j < 4 ? u[j] : v[j - 4];
      }
#pragma unroll
      for (int j = 0; j < 8; j++) mb = max(mb, __float_as_uint(x[s][j]) & 0x7FFFFFFFu);
    }
    for (int off = NQ; off < 64; off *= 2) mb = max(mb, (uint32_t)__shfl_xor((int)mb, off, 64));
    int sh = 0;
    if (mb && mb < 0x7F800000u) sh = 15 - __builtin_amdgcn_frexp_expf(__uint_as_float(mb));
#pragma unroll
    for (int s = 0; s < kSteps; s++)
#pragma unroll
      for (int j = 0; j < 8; j++) {
        const float y = ldexpf(scale < 0.0f ? -x[s][j] : x[s][j], sh);
        qh[s][j] = (_Float16)y;
        ql[s][j] = (_Float16)(y - (float)qh[s][j]);
      }
    // A factor of 0 becomes one whose products are as good as 0 (and -inf stays).
    c = ldexpf(fabsf(scale) * 1.4426950408889634f, -sh);
    if (c < 1e-37f) c = 1e-37f;
    m = -__builtin_inff();
    l = 0.0f;
#pragma unroll
    for (int t = 0; t < kDt; t++) o[t] = acc{};
  }

  // Scores of BK keys; key(t, s): the operand of step s for keys NQ t + lane % NQ.  (The
  // scheduling barriers keep a step's reads ahead of the products before it: the
  // compiler puts them right before their use.)
  template <typename F>
  __device__ __forceinline__ void scores(acc (&s)[BK / NQ], F&& key) {
#pragma unroll
    for (int t = 0; t < BK / NQ; t++) s[t] = acc{};
    half8 k[2][BK / NQ];
#pragma unroll
    for (int t = 0; t < BK / NQ; t++) k[0][t] = key(t, 0);
#pragma unroll
    for (int st = 0; st < kSteps; st++) {
      if (st + 1 < kSteps) {
#pragma unroll
        for (int t = 0; t < BK / NQ; t++) k[(st + 1) & 1][t] = key(t, st + 1);
      }
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int t = 0; t < BK / NQ; t++) s[t] = Mfma<NQ>::mul(k[st & 1][t], qh[st], s[t]);
#pragma unroll
      for (int t = 0; t < BK / NQ; t++) s[t] = Mfma<NQ>::mul(k[st & 1][t], ql[st], s[t]);
      __builtin_amdgcn_sched_barrier(0);
    }
  }

  // Scores times the keys' scales (8-bit keys: `ks`, the tile's in LDS), -inf where a
  // key is not seen (kMask: those outside [lo, hi], relative to the tile), and the
  // running maximum; o and the sum go down where it went up.
  template <bool kMask>
  __device__ __forceinline__ void maximum(acc (&s)[BK / NQ], int lo, int hi, const float* ks) {
    constexpr int kPer = kAcc / 4;  // quads of one accumulator
    const int grp = (threadIdx.x & 63) / NQ;
    float mx = -__builtin_inff();
    const int l0 = lo - 4 * grp, h0 = hi - 4 * grp;
#pragma unroll
    for (int u = 0; u < kQuads; u++) {
      f32x4 k4;
      if (kType == kKvInt8) k4 = *reinterpret_cast<const f32x4*>(ks + 4 * NG * u + 4 * grp);
#pragma unroll
      for (int r = 0; r < 4; r++) {
        float x = s[u / kPer][u % kPer * 4 + r];
        if (kType == kKvInt8) x *= k4[r];
        const int key = 4 * NG * u + r;
        if (kMask) x = key < l0 || key > h0 ? -__builtin_inff() : x;
        s[u / kPer][u % kPer * 4 + r] = x;
        mx = fmaxf(mx, x);
      }
    }
    mx = Mfma<NQ>::max(mx) * c;
    if (__any(mx > m + kSlack)) {
      const float n = fmaxf(m, mx);
      const float f = m == -__builtin_inff() ? 0.0f : __builtin_amdgcn_exp2f(m - n);
      m = n;
      l *= f;
#pragma unroll
      for (int t = 0; t < kDt; t++) o[t] *= f;
    }
  }

  // Scores to weights, and o += V^T w over a tile of V rows in LDS (KvTile; fp16, or
  // 8-bit codes as bf16 with the values' scales in `vs`).  While a step's products run,
  // the next step's weights are computed, two at a time.
  __device__ __forceinline__ void values(acc (&s)[BK / NQ], const uint8_t* tile,
                                         const float* vs) {
    constexpr int kPer = kAcc / 4;
    const int lane = threadIdx.x & 63, l16 = lane & 15, grp = lane / NQ;
    const int row0 = 4 * grp + l16 / 4;
    const int col = (NQ == 32 ? (lane >> 4 & 1) * 2 : 0) + (l16 & 3) / 2;
    const float off = kTop - (m == -__builtin_inff() ? 0.0f : m);
    float neg = -1.0f, sum = 0.0f;  // (the tile's sum apart: fewer additions to the long one)
    asm("" : "+s"(neg));
    u32x4 w[2][3];  // the weights' parts of this step and the next, two a register
    auto pair = [&](int p, int i) __attribute__((always_inline)) {
      const int u = 2 * p + i / 2, r = i % 2 * 2;
      float x[2];
#pragma unroll
      for (int j = 0; j < 2; j++)
        x[j] = __builtin_amdgcn_exp2f(fmaf(s[u / kPer][u % kPer * 4 + r + j], c, off));
      sum += x[0] + x[1];
      uint32_t a, b, d = 0;
      if (kType == kKvFp16) {
        split_f16(x[0], x[1], neg, a, b);
      } else {
        const float* v = vs + 4 * NG * u + 4 * grp + r;
        split_bf16(x[0] * v[0], x[1] * v[1], a, b, d);
      }
      w[p & 1][0][i] = a;
      w[p & 1][1][i] = b;
      w[p & 1][2][i] = d;
    };
    auto value = [&](int p, int t) __attribute__((always_inline)) {
      u32x4 v;
#pragma unroll
      for (int q = 0; q < 2; q++) {
        const int row = 4 * NG * (2 * p + q) + row0;
        const uint8_t* src = tile + KvTile<DP>::at(row, NQ / 8 * t + col) + (l16 & 1) * 8;
        typedef short short4v __attribute__((ext_vector_type(4)));
        const auto x = __builtin_bit_cast(
            uint2_t, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                         (__attribute__((address_space(3))) short4v*)src));
        v[2 * q] = x[0];
        v[2 * q + 1] = x[1];
      }
      return v;
    };
    // (two accumulators in turn: a product on the one before it would wait for it)
    constexpr int kGroups = (kDt + 1) / 2;
    u32x4 v[2][2];
    auto values_of = [&](int at) __attribute__((always_inline)) {
#pragma unroll
      for (int j = 0; j < 2; j++)
        if (at % kGroups * 2 + j < kDt) v[at & 1][j] = value(at / kGroups, at % kGroups * 2 + j);
    };
    values_of(0);
#pragma unroll
    for (int i = 0; i < 4; i++) pair(0, i);
#pragma unroll
    for (int p = 0; p < kPv; p++)
#pragma unroll
      for (int g = 0; g < kGroups; g++) {
        const int at = p * kGroups + g;
        if (at + 1 < kPv * kGroups) values_of(at + 1);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int part = 0; part < (kType == kKvFp16 ? 2 : 3); part++)
#pragma unroll
          for (int j = 0; j < 2; j++) {
            const int t = 2 * g + j;
            if (t >= kDt) continue;
            const u32x4 x = v[at & 1][j], y = w[p & 1][part];
            o[t] = kType == kKvFp16 ? Mfma<NQ>::mul(f16x8(x), f16x8(y), o[t])
                                    : Mfma<NQ>::mul(bf16x8(x), bf16x8(y), o[t]);
          }
#pragma unroll
        for (int i = 0; i < 4; i++)
          if (p + 1 < kPv && i * kGroups / 4 == g) pair(p + 1, i);
        __builtin_amdgcn_sched_barrier(0);
      }
    l += sum;
  }

  // Ends the pass: this lane's row sum, NaN where the tiles held pages that are none.
  __device__ __forceinline__ void finish(bool bad) {
    l = bad ? __builtin_nanf("") : Mfma<NQ>::sum(l);
  }

  // d of accumulator register i of tile t (four in a row from 4 * (i / 4)).
  __device__ static __forceinline__ int dim(int t, int i) {
    return NQ * t + 4 * NG * (i / 4) + 4 * ((threadIdx.x & 63) / NQ) + i % 4;
  }
};

// Launchers of the kernels' files.
hipError_t launch_attn_tile(const AttnArgs& a, hipStream_t s);
hipError_t launch_attn_few(const AttnArgs& a, hipStream_t s);

}  // namespace hypno
