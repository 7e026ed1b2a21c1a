// Attention of each sequence's new tokens over its pages of the cache: which kernels
// a call takes, and the sum of what a row's ranges of positions gave (5.6 us for 64 ranges
// of 32 rows, 15 for four of 16384, 42 MB: 2.8 TB/s).
#include <cmath>

#include "attention.hpp"

namespace hypno {

namespace {

// One wave a (token, head): a row over no pages at all.
__global__ void __launch_bounds__(64) attn_rows_kernel(AttnArgs a) {
  const int t = blockIdx.x / a.heads, h = blockIdx.x % a.heads;
  const int b = find_seq(a.b, t, 0, 0);
  if (b < 0 || b >= a.b.batch) return;
  const Seq sq = seq_of(a.b, b);
  attn_row(a, sq, t - sq.first, h);
}

// One (token, head): the maxima, sums and outputs of its ranges, by kWaves waves (one
// where rows are many), each on a part of the ranges.  A lane holds one range's maximum
// and sum, then four elements of the output in every (64 / lanes)th range.
template <int kWaves>
__global__ void __launch_bounds__(256) attn_join_kernel(AttnArgs a) {
  __shared__ f32x4 so[4][64];
  __shared__ float2 sml[4];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int part = wave % kWaves;
  const size_t row = (size_t)blockIdx.x * (4 / kWaves) + wave / kWaves;
  const int t = (int)(row / a.heads), h = (int)(row % a.heads);
  const int D = a.c.head_dim, G = a.group;
  const int b = t < a.b.tokens ? find_seq(a.b, t, 0, 0) : -1;
  if (b < 0 || b >= a.b.batch) return;
  const Seq sq = seq_of(a.b, b);
  const int rows = sq.n * G, r = (t - sq.first) * G + h % G;
  if (r < 0 || r >= rows) return;
  const bool few = rows <= a.few;
  const AttnSplit sp = few ? a.fs : a.ts;
  if (sp.splits <= 1) return;  // written already
  const int per = few ? kFewRows : a.tile_rows, r0 = r / per * per;
  const bool past = too_long(a, sq);
  const int all = past ? 0 : split_count(sp, span_of(a, sq, r0, min(r0 + per, rows)));
  const int first = all * part / kWaves, n = all * (part + 1) / kWaves - first;
  const AttnParts parts = few ? a.fp : a.tp;
  const size_t at0 = (few ? few_part(a, sq, h / G, r, row) : row) * sp.splits + first;
  const float2* ml = parts.ml + at0;
  const int lanes = D <= 64 ? 16 : D <= 128 ? 32 : 64, sub = lane / lanes, d = lane % lanes * 4;
  const float* po = parts.o + at0 * D + d;
  float m = -__builtin_inff(), l = 0.0f;
  f32x4 o = {0.0f, 0.0f, 0.0f, 0.0f};
  for (int i0 = 0; i0 < n; i0 += 64) {
    float2 p = make_float2(-__builtin_inff(), 0.0f);
    if (i0 + lane < n) p = load_global<float2>(ml + i0 + lane);
    float top = fmaxf(m, p.x);
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) top = fmaxf(top, __shfl_xor(top, off, 64));
    const float ref = top == -__builtin_inff() ? 0.0f : top;
    const float f = __builtin_amdgcn_exp2f(m - ref), w = __builtin_amdgcn_exp2f(p.x - ref);
    m = top;
    l = l * f + wave_sum(p.y * w);
    o *= f;
    constexpr int kFly = 8;
    const int cnt = min(64, n - i0), step = 64 / lanes;
    // (all lanes go through every step: a range's weight is read from the lane that has it)
    for (int at = 0; at < cnt; at += kFly * step) {
      const int i = at + sub;
      f32x4 v[kFly];
#pragma unroll
      for (int j = 0; j < kFly; j++)
        if (i + j * step < cnt && d < D)
          v[j] = load_global<f32x4>(po + (size_t)(i0 + i + j * step) * D);
#pragma unroll
      for (int j = 0; j < kFly; j++) {
        // (the lane's number goes modulo 64)
        const float wj = __int_as_float(
            __builtin_amdgcn_ds_bpermute((i + j * step) << 2, __float_as_int(w)));
        if (i + j * step < cnt && d < D) o += v[j] * wj;
      }
    }
  }
  for (int off = lanes; off < 64; off *= 2)
#pragma unroll
    for (int j = 0; j < 4; j++) o[j] += __shfl_xor(o[j], off, 64);
  if (kWaves > 1) {
    so[wave][lane] = o;
    if (lane == 0) sml[wave] = make_float2(m, l);
    __syncthreads();
    if (wave) return;
    float top = m;
    for (int i = 1; i < kWaves; i++) top = fmaxf(top, sml[i].x);
    const float ref = top == -__builtin_inff() ? 0.0f : top;
    l = 0.0f;
    o = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    for (int i = 0; i < kWaves; i++) {
      const float w = __builtin_amdgcn_exp2f(sml[i].x - ref);
      l += sml[i].y * w;
      o += so[i][lane] * w;
    }
  }
  const f32x4 v = o * (l == 0.0f ? 0.0f : 1.0f / l);
  const float z = ((l + v[0]) + (v[1] + v[2]) + v[3]) * 0.0f;
  const bool again = __any(!(z == 0.0f)) || past;
  if (again)
    attn_row(a, sq, t - sq.first, h);
  else if (sub == 0 && d < D)
    *reinterpret_cast<f32x4*>(a.out + row * D + d) = v;
}

// From here on a wave a row, not four.
constexpr unsigned kJoinRows = 1024;

// Bytes of one kernel's ranges at most: a million of them at head_dim 128, where 64
// sequences of 32 heads take 16 to 32 a row and a chunk of 512 tokens four.
constexpr size_t kMaxParts = (size_t)512 << 20;

int up(int64_t a, int64_t b) { return (int)((a + b - 1) / b); }

}  // namespace

AttnPlan attn_plan(const KvCache& c, const KvBatch& b, int heads, int window, int64_t max_kv,
                   int num_cus) {
  AttnPlan p = {};
  p.cus = num_cus;
  const int G = heads / c.kv_heads;
  const int64_t rows = (int64_t)b.tokens * G;
  p.tile_rows = c.head_dim <= 128 ? 128 : 64;
  // Single tokens, or one sequence of few rows: attn_few_kernel alone.  Few sequences, or
  // groups of more than 16: attn_tile_kernel alone, where single tokens run beside the
  // others and not in a second kernel after them.  (us at 32/8 heads of 128, one kernel /
  // both: 333 tokens over 700 / 2000 / 5000 / 16000 beside seven single ones 28 / 39, 50 / 62,
  // 88 / 113, 273 / 305; with 8-bit values 43 / 51, 69 / 76, 134 / 148, 401 / 416; 40 tokens
  // over 2000 beside three 24 / 28 and 30 / 34; a group of 32, 16 sequences, 46 / 48 to 75 /
  // 76.  It costs where no chunk fills the tiles: five tokens beside seven over 16000 116 /
  // 101, with 8-bit values over 2000 and 16000 45 / 29 and 169 / 101; 40 tokens over 16000
  // beside three, 8-bit, 113 / 102.)
  const bool only_few = b.tokens <= b.batch || (b.batch == 1 && rows <= 16);
  const bool only_tile = !only_few && (b.batch <= 8 || G > 16);
  p.few = only_few ? 0x7FFFFFFF : only_tile ? 0 : kFewRows;
  const int64_t room = (int64_t)b.width << c.page_shift;
  const int64_t kv = std::max<int64_t>(1, max_kv ? std::min(max_kv, room) : room);
  // Up to 1024 positions (2048 where sequences and heads alone fill the chip) a
  // work-group takes them all: the kernel that joins ranges costs 4 us and its launch.
  // Beyond, one sequence gets a work-group for each one that the chip holds at a time.
  // Lengths of several may differ, so that the last range to end counts: against the
  // start of a range (about 130 positions' time) the best length grows with the root of
  // all work.  (us at 32/8 heads of 128, ranges of 128 / 256 / 512 / none: one sequence
  // of 3000: 11.1 / 12.0 / 14.1 / -; 8 of up to 6000: 44 / 35 / 32 / -; 64 of up to 2000:
  // - / 67 / 58 / 53.)
  p.fs = {1, 0x7FFFFFFF};
  p.few_waves = 4;
  const size_t token_rows = (size_t)b.tokens * heads, place = (size_t)c.head_dim * 4 + 8;
  const size_t seq_rows = (size_t)b.batch * c.kv_heads * kFewRows;
  p.by_seq = p.few == kFewRows && seq_rows < token_rows;
  const size_t few_rows = p.by_seq ? seq_rows : token_rows;
  const auto most = [&](size_t rows) {  // ranges that kMaxParts has room for
    return std::max<int64_t>(1, (int64_t)std::min<size_t>(kMaxParts / place / rows, 1 << 30));
  };
  if (p.few) {
    const int64_t seen = window ? std::min<int64_t>(kv, (int64_t)window + 16) : kv;
    const int64_t pairs = (int64_t)b.batch * c.kv_heads, slots = 2 * num_cus;
    if (seen > (pairs >= slots ? 2048 : 1024)) {
      const double each = (double)pairs * seen / slots;
      const double best = b.batch > 1 ? std::sqrt(128.0 * each) : each;
      const int64_t least = std::min<int64_t>(std::max<int64_t>(8 * pairs, 128), 512);
      // (whole steps of four waves: a run of positions must not lie across two ranges)
      const int64_t fit = (seen + most(few_rows) - 1) / most(few_rows);
      const int64_t chunk = (std::max({least, (int64_t)best, fit}) + 127) / 128 * 128;
      p.fs.splits = up(seen, chunk);
      p.fs.chunk = (int)std::min<int64_t>(chunk, 0x7FFFFFFF);
    } else if (pairs <= num_cus && seen > 128) {
      p.few_waves = 8;
    }
  }
  // Ranges where they are worth writing and joining their parts: by the time, in us, of a
  // work-group's tiles of 64 positions (1.8 with one work-group a CU and head_dim 128, 1.6
  // times that with two) and of the parts' way through memory.
  p.ts = {1, 0x7FFFFFFF};
  if (p.few != 0x7FFFFFFF) {
    const int64_t seen =
        window ? std::min<int64_t>(kv, (int64_t)window + up(p.tile_rows, G)) : kv;
    const double groups = std::max(1.0, (double)rows / p.tile_rows) * c.kv_heads;
    const double part_us = (double)b.tokens * heads * c.head_dim * 8 / 3.5e6;
    const int dim = c.head_dim <= 64 ? 64 : c.head_dim <= 96 ? 96 : 128;
    const double tile_us = ((c.head_dim > 128 ? 2 : 1) * 0.8 + dim / 128.0) *
                           (c.dtype == kKvInt8 ? 1.2 : 1.0);
    double best = 1e30;
    for (int n = 1; n <= 64; n++) {
      const int64_t chunk = (up(seen, n) + 63) / 64 * 64;
      const int splits = up(seen, chunk);
      if (splits > most(token_rows)) break;
      const double each = groups * splits <= num_cus ? tile_us : 1.6 * tile_us;
      const double us = std::ceil(groups * splits / (2 * num_cus)) * (4.0 + chunk / 64 * each) +
                        (splits > 1 ? 5.0 + part_us * splits : 0.0);
      if (us < best * 0.98) {
        best = us;
        p.ts.splits = splits;
        p.ts.chunk = (int)std::min<int64_t>(chunk, 0x7FFFFFFF);
      }
    }
  }
  p.few_places = p.fs.splits > 1 ? few_rows * p.fs.splits : 0;
  p.tile_places = p.ts.splits > 1 ? token_rows * p.ts.splits : 0;
  p.ml_bytes = ((p.few_places + p.tile_places) * 8 + 255) / 256 * 256;
  p.bytes = p.ml_bytes + (p.few_places + p.tile_places) * c.head_dim * 4;
  return p;
}

hipError_t launch_paged_attention(const AttnPlan& p, float* out, const float* q, size_t q_stride,
                                  int heads, const KvCache& c, const KvBatch& b, float scale,
                                  int window, void* ws, hipStream_t s) {
  AttnArgs a = {c, b, out, q, q_stride, heads, heads / c.kv_heads, window, scale,
                p.few, p.few_waves, p.tile_rows, p.fs, p.ts, p.cus, p.by_seq, {}, {}};
  if (!ws) a.fs = a.ts = {1, 0x7FFFFFFF};
  a.fp.ml = reinterpret_cast<float2*>(ws);
  a.tp.ml = a.fp.ml + p.few_places;
  a.fp.o = reinterpret_cast<float*>((uint8_t*)ws + p.ml_bytes);
  a.tp.o = a.fp.o + p.few_places * c.head_dim;
  const unsigned rows = (unsigned)b.tokens * (unsigned)heads;
  if (c.pages == 0) {
    attn_rows_kernel<<<rows, 64, 0, s>>>(a);
    return hipGetLastError();
  }
  hipError_t e = hipSuccess;
  if (a.few != 0x7FFFFFFF) e = launch_attn_tile(a, s);
  if (e == hipSuccess && a.few) e = launch_attn_few(a, s);
  if (e == hipSuccess && (a.fs.splits > 1 || a.ts.splits > 1)) {
    if (rows < kJoinRows)
      attn_join_kernel<4><<<rows, 256, 0, s>>>(a);
    else
      attn_join_kernel<1><<<(rows + 3) / 4, 256, 0, s>>>(a);
    e = hipGetLastError();
  }
  return e;
}

}  // namespace hypno
