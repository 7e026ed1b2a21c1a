// Pages that a token reads of a long context, by a cheap score of each, and the bounds
// of the keys that the score is made of.
//
// Bounds of a page and kv head: the smallest and largest key in each channel, as codes
//   s = max|k| / 127 over the page's keys, code = round_half_away(k / s)
// with both quotients in fp32 (s = 0 and codes 0 where that underflows; s = NaN and
// codes 0 for a page that holds an infinity or NaN).  For any key of the page
//   q.k <= q+ . hi + q- . lo = sum_d max(q_d lo_d, q_d hi_d),
// q+ and q- the positive and negative part of q: but for the codes' rounding the score
// is the most that any key of the page can give.  With q in 8-bit codes of its own (per
// head, the same rule) that is a product of whole numbers, exact on the matrix cores
// in any order, so that the choice depends on no sum's order:
//   score = bounds' scale * max over the kv head's query heads of q's scale * (whole number)
// with these two products in fp32.
//
// Bound: latency.  Bounds of the 131 pages of 8192 new 4-bit tokens (4.8 MB) 7.6 us, of 64
// sequences' last pages 8.4: a sequence's place, its page and the keys are reads that depend
// on each other, six for 64 sequences (cu_q's end, its values 64 at a time, the sequence's
// own beside its kv_len, the page, the keys).  Pages for one token of 2048 (4.2 MB) 12 us in two kernels, for 512 tokens of
// 512 (their bounds 134 MB out of L2, 8 us of it) 20, for 2048 tokens 67, for 64 tokens of
// 1150 each (151 MB) 46.
#include "kv_cache.hpp"

namespace hypno {

namespace {

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef float f32x4a4 __attribute__((ext_vector_type(4), aligned(4)));

constexpr int kMaxDim = 256;
constexpr int kTeamWaves = 8;

// The code of x with scale s > 0.
__device__ __forceinline__ uint32_t code8(float x, float s) {
  return (uint32_t)(int)fminf(fmaxf(roundf(x / s), -127.0f), 127.0f) & 0xFFu;
}

// --- bounds -------------------------------------------------------------------------------

struct BoundsArgs {
  KvCache c;
  KvBatch b;
  KeyBounds o;
  int lane_shift;  // 1 << lane_shift lanes a key, each with 8 channels
};

// The last sequence whose pages' numbers begin at `number` or before.
__device__ __forceinline__ int seq_of_page(const BoundsArgs& a, int64_t number) {
  const int lane = threadIdx.x & 63;
  int count = 0;
  for (int i0 = 0; i0 <= a.b.batch; i0 += 64) {
    const int i = i0 + lane;
    bool in = false;
    if (i <= a.b.batch) in = first_number(cu_at(a.b, i), i, a.c.page_shift) <= number;
    count += __popcll(__ballot(in));
  }
  return count - 1;
}

template <int kType>
__device__ __forceinline__ void load_keys(float (&x)[8], const BoundsArgs& a, int page, int g,
                                          int slot, int e0) {
  const int D = a.c.head_dim;
  const size_t tok = ((size_t)g << a.c.page_shift) + slot;
  if (kType == kKvFp16) {
    const u32x4 v = load_global<u32x4>((const _Float16*)a.c.k + (size_t)page * a.c.k_page +
                                       tok * D + e0);
#pragma unroll
    for (int i = 0; i < 8; i++)
      x[i] = (float)__builtin_bit_cast(_Float16, (uint16_t)(v[i / 2] >> 16 * (i % 2)));
  } else if (kType == kKvInt8) {
    const uint2 v = load_global<uint2>((const int8_t*)a.c.k + (size_t)page * a.c.k_page + tok * D +
                                       e0);
    const float s = load_global<float>(a.c.k_scale + (size_t)page * a.c.ks_page + tok);
#pragma unroll
    for (int i = 0; i < 8; i++)
      x[i] = (float)(int8_t)((i < 4 ? v.x : v.y) >> 8 * (i % 4)) * s;
  } else {
    const uint32_t v = load_global<uint32_t>((const uint8_t*)a.c.k + (size_t)page * a.c.k_page +
                                             (tok * D + e0) / 2);
    const size_t at = ((size_t)(g * (D / kFp4Group) + e0 / kFp4Group) << a.c.page_shift) + slot;
    const _Float16 s = load_global<_Float16>((const _Float16*)a.c.k_scale +
                                             (size_t)page * a.c.ks_page + at);
    const u32x4 y = fp4_to_f16(v, half2v{s, s});
#pragma unroll
    for (int i = 0; i < 8; i++)
      x[i] = (float)__builtin_bit_cast(_Float16, (uint16_t)(y[i / 2] >> 16 * (i % 2)));
  }
}

// One work-group a (page, kv head) at a time; 8 channels a lane, keys over the rest.
template <int kType>
__global__ void __launch_bounds__(256) key_bounds_kernel(BoundsArgs a) {
  __shared__ float s_lo[4][kMaxDim], s_hi[4][kMaxDim];
  __shared__ uint32_t s_bits[4];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int D = a.c.head_dim, KV = a.c.kv_heads;
  const int unit = tid & ((1 << a.lane_shift) - 1), row = tid >> a.lane_shift;
  const int e0 = 8 * unit, rows = 256 >> a.lane_shift;
  const int64_t numbers = first_number(cu_at(a.b, a.b.batch), a.b.batch, a.c.page_shift);
  for (int64_t w = blockIdx.x; w < numbers * KV; w += gridDim.x) {
    // (all lanes decide the same)
    const int64_t number = w / KV;
    const int g = (int)(w % KV), b = seq_of_page(a, number);
    if (b < 0 || b >= a.b.batch) continue;
    const int kv = load_global<int>(a.b.kv_lens + b);
    const int at = page_of_number(number, b, cu_at(a.b, b), cu_at(a.b, b + 1), kv, a.c.page_shift,
                                  a.b.width);
    if (at < 0) continue;
    const int page = load_global<int>(a.b.page_table + (size_t)b * a.b.width + at);
    if (page < 0 || page >= a.c.pages) continue;
    const int keys = min(1 << a.c.page_shift, kv - (at << a.c.page_shift));
    float lo[8], hi[8];
    uint32_t mb = 0;
#pragma unroll
    for (int i = 0; i < 8; i++) lo[i] = __builtin_inff(), hi[i] = -__builtin_inff();
    if (e0 < D) {
#pragma unroll 4
      for (int r = row; r < keys; r += rows) {
        float x[8];
        load_keys<kType>(x, a, page, g, r, e0);
#pragma unroll
        for (int i = 0; i < 8; i++) {
          lo[i] = fminf(lo[i], x[i]);
          hi[i] = fmaxf(hi[i], x[i]);
          mb = max(mb, __float_as_uint(x[i]) & 0x7FFFFFFFu);
        }
      }
    }
    for (int off = 1 << a.lane_shift; off < 64; off <<= 1)
#pragma unroll
      for (int i = 0; i < 8; i++) {
        lo[i] = fminf(lo[i], __shfl_xor(lo[i], off, 64));
        hi[i] = fmaxf(hi[i], __shfl_xor(hi[i], off, 64));
      }
    for (int off = 32; off > 0; off >>= 1) mb = max(mb, (uint32_t)__shfl_xor((int)mb, off, 64));
    if (lane < 1 << a.lane_shift && e0 < D) {
#pragma unroll
      for (int i = 0; i < 8; i++) s_lo[wave][e0 + i] = lo[i], s_hi[wave][e0 + i] = hi[i];
    }
    if (lane == 0) s_bits[wave] = mb;
    __syncthreads();
    // Two rows of codes, four a lane.
    const int e = 4 * tid % kMaxDim, half = 4 * tid / kMaxDim;
    mb = max(max(s_bits[0], s_bits[1]), max(s_bits[2], s_bits[3]));
    const float s = mb < 0x7F800000u ? __uint_as_float(mb) / 127.0f : __builtin_nanf("");
    if (half < 2 && e < D) {
      uint32_t codes = 0;
#pragma unroll
      for (int i = 0; i < 4; i++) {
        const float x =
            half ? fmaxf(fmaxf(s_hi[0][e + i], s_hi[1][e + i]), fmaxf(s_hi[2][e + i], s_hi[3][e + i]))
                 : fminf(fminf(s_lo[0][e + i], s_lo[1][e + i]), fminf(s_lo[2][e + i], s_lo[3][e + i]));
        if (s > 0.0f) codes |= code8(x, s) << 8 * i;
      }
      *reinterpret_cast<uint32_t*>(a.o.codes + (size_t)page * a.o.page + (size_t)(2 * g + half) * D +
                                   e) = codes;
    }
    if (tid == 0) a.o.scale[(size_t)page * a.o.s_page + g] = s;
    __syncthreads();
  }
}

// --- selection ------------------------------------------------------------------------------

struct SelectArgs {
  KeyBounds k;
  KvBatch b;
  int* out;
  const float* q;
  size_t q_stride;
  int heads, group, count, first, last;
  int rows;    // of a token in a product: 1, 2, 4, 8 or 16, the group's heads or more
  int most;    // pages of a sequence that have a score at most
  int pitch;   // of a token's keys in LDS
  int tokens;  // of a work-group
  int splits, chunk;  // of pages, whose scores a work-group of the first of two kernels takes
  uint32_t* scores;   // [tokens][kv_heads][pitch], between the two
};

// What a launch does: both steps, or one of them.
constexpr int kBoth = 0, kScores = 1, kChoice = 2;

// Scores as whole numbers in their order, from 1 on; 0: no candidate.  (What is no
// number, and infinities, as the largest finite one: below what is always selected.)
__device__ __forceinline__ uint32_t key_of(float x) {
  const float m = 3.4028234663852886e38f;
  const float y = (x == x ? fminf(fmaxf(x, -m), m) : m) + 0.0f;
  const uint32_t u = __float_as_uint(y);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// Orders LDS accesses of a wave's lanes among themselves.
__device__ __forceinline__ void wave_lds_sync() {
#if defined(__HIP_DEVICE_COMPILE__)
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  __builtin_amdgcn_wave_barrier();
#endif
}

// Over the wave's lanes, by moves between neighbours, not through LDS: the sums up to each
// lane, and the largest.
template <int kCtrl, int kRows>
__device__ __forceinline__ uint32_t moved(uint32_t x) {
  return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, kCtrl, kRows, 0xF, false);
}
__device__ __forceinline__ uint32_t wave_scan(uint32_t x) {
  x += moved<0x111, 0xF>(x);  // row_shr:1, 2, 4, 8
  x += moved<0x112, 0xF>(x);
  x += moved<0x114, 0xF>(x);
  x += moved<0x118, 0xF>(x);
  x += moved<0x142, 0xA>(x);  // row_bcast:15, 31
  return x + moved<0x143, 0xC>(x);
}
__device__ __forceinline__ uint32_t wave_max(uint32_t x) {
  x = max(x, moved<0x111, 0xF>(x));
  x = max(x, moved<0x112, 0xF>(x));
  x = max(x, moved<0x114, 0xF>(x));
  x = max(x, moved<0x118, 0xF>(x));
  x = max(x, moved<0x142, 0xA>(x));
  return (uint32_t)__builtin_amdgcn_readlane((int)max(x, moved<0x143, 0xC>(x)), 63);
}

// Wave-wide (the lanes of one) or work-group-wide waits for LDS.
template <bool kTeam>
__device__ __forceinline__ void lds_sync() {
  if (kTeam)
    __syncthreads();
  else
    wave_lds_sync();
}

// One work-group a kv head of up to 16 / rows tokens of a sequence: scores of their pages
// into LDS, 16 rows (token, head) by 16 pages a product, so that a lane has up to four heads
// of a page; then for each token the key of the last page that is taken, eight bits at a time
// from the top by counting.  kTeam: all waves look at one token's keys, else each wave at its
// own tokens'.
//
// Latency is what there is to save: a page's number, its bounds, the counts are reads that
// depend on each other, so that a wave asks for two products' pages at a time, and for the
// next two's numbers with them (four: a third of the waves less, and 5 to 10% longer where
// work-groups fill the chip).  A page's two bounds are one piece of memory, 128 bytes
// of which eight lanes read; lanes that each read of another page, as the product takes
// them, take four times as long (16 us for 2048 pages), so that they change places in LDS.
template <int DP, int kWaves, bool kTeam, int kStep>
__global__ void __launch_bounds__(64 * kWaves, DP > 128 ? 2 : 4)
    select_pages_kernel(SelectArgs a) {
  constexpr int kSteps = 2 * DP / 64, kPitch = 2 * DP + 16, kAtOnce = DP > 128 ? 1 : 2;
  constexpr int kUnits = 2 * DP / 128;  // of 128 bytes of the bounds
  __shared__ __attribute__((aligned(16))) uint8_t codes[16 * kPitch];
  __shared__ __attribute__((aligned(16))) float row_scale[16];
  __shared__ __attribute__((aligned(16))) uint8_t stage[kWaves][16 * 128];
  __shared__ __attribute__((aligned(16))) int hist[kTeam ? 1 : kWaves][256];
  __shared__ uint2 ends[kWaves];
  __shared__ int2 counts[kWaves];
  extern __shared__ uint32_t keys[];  // [tokens][pitch]
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int KV = a.k.kv_heads, G = a.group, D = a.k.head_dim, shift = a.k.page_shift;
  const int slots = gridDim.x / KV / (kStep == kScores ? a.splits : 1);
  const int g = blockIdx.x % KV, slot = blockIdx.x / KV % slots, split = blockIdx.x / KV / slots;
  const int b = find_seq(a.b, slot, 1, a.tokens);
  if (b < 0 || b >= a.b.batch) return;
  const int first = cu_at(a.b, b), n = cu_at(a.b, b + 1) - first;
  const int i0 = (slot - (first / a.tokens + b)) * a.tokens, nt = min(a.tokens, n - i0);
  if (i0 < 0 || nt <= 0) return;
  const int t0 = first + i0;
  // The page of token i of the tile is (pos0 + i) >> shift: -1 and less if it has no place.
  const int64_t pos0 = (int64_t)load_global<int>(a.b.kv_lens + b) - n + i0;
  const int most = min(a.most, a.b.width);
  int top = (int)min((int64_t)most, ((pos0 + nt - 1) >> shift) + 1 - a.last), bottom = a.first;
  if (kStep == kScores) {
    bottom = (int)min((int64_t)a.first + (int64_t)split * a.chunk, (int64_t)max(top, a.first));
    top = (int)min((int64_t)top, (int64_t)bottom + a.chunk);
  }
  // Keys of the tile's token i: [pitch] from `keys_of` on, `keys_step` apart.
  uint32_t* const all_keys = a.scores + ((size_t)t0 * KV + g) * a.pitch;
  uint32_t* const keys_of = kStep == kScores ? all_keys : keys;
  const size_t keys_step = kStep == kScores ? (size_t)KV * a.pitch : a.pitch;
  const int* const table = a.b.page_table + (size_t)b * a.b.width;
  // A wave's pages: 16 kAtOnce in a row, then those 16 kAtOnce kWaves on; a lane looks up
  // lane % 16 of each 16, and reads of lane / 8 and 8 on.
  constexpr int kStride = 16 * kAtOnce * kWaves;
  const int start = bottom + 16 * kAtOnce * wave;
  auto look_up = [&](int (&page)[kAtOnce], int p0) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < kAtOnce; i++) {
      const int p = p0 + 16 * i + lane % 16;
      page[i] = p < top ? load_global<int>(table + p) : -1;
    }
  };
  int page[kAtOnce];
  if (kStep != kChoice) look_up(page, start);

  for (int h0 = 0; kStep != kChoice && h0 < G && top > bottom; h0 += 16) {
    // The rows' codes, [negative part][positive part][zeros]; 16 lanes a row.
    if (wave < 4) {
      const int r = tid / 16, sub = tid % 16;
      // (rows past the group's heads: its first again, which changes no maximum)
      const int tok = r / a.rows, h = h0 + r % a.rows < G ? h0 + r % a.rows : h0;
      const bool live = tok < nt;
      float x[(DP + 127) / 128][8];
      uint32_t mb = 0;
#pragma unroll
      for (int j = 0; j < (DP + 127) / 128; j++) {
        const int e = sub * 8 + 128 * j;
#pragma unroll
        for (int i = 0; i < 8; i++) x[j][i] = 0.0f;
        if (live && e < D) {
          const float* src = a.q + (size_t)(t0 + tok) * a.q_stride + (size_t)(g * G + h) * D + e;
          const f32x4a4 u = load_global<f32x4a4>(src), v = load_global<f32x4a4>(src + 4);
#pragma unroll
          for (int i = 0; i < 8; i++) x[j][i] = i < 4 ? u[i] : v[i - 4];
        }
#pragma unroll
        for (int i = 0; i < 8; i++) mb = max(mb, __float_as_uint(x[j][i]) & 0x7FFFFFFFu);
      }
#pragma unroll
      for (int off = 8; off > 0; off >>= 1) mb = max(mb, (uint32_t)__shfl_xor((int)mb, off, 64));
      const float s = mb < 0x7F800000u ? __uint_as_float(mb) / 127.0f : 0.0f;
#pragma unroll
      for (int j = 0; j < (DP + 127) / 128; j++) {
        const int e = sub * 8 + 128 * j;
        if (e >= DP) continue;
        uint32_t neg[2] = {0, 0}, pos[2] = {0, 0};
        if (s > 0.0f) {
#pragma unroll
          for (int i = 0; i < 8; i++) {
            const uint32_t c = code8(x[j][i], s) << 8 * (i % 4);
            (x[j][i] < 0.0f ? neg : pos)[i / 4] |= c;
          }
        }
        uint8_t* const row = codes + r * kPitch;
        *reinterpret_cast<uint2*>(row + (e < D ? e : 2 * e)) = make_uint2(neg[0], neg[1]);
        *reinterpret_cast<uint2*>(row + (e < D ? D + e : 2 * e + 8)) = make_uint2(pos[0], pos[1]);
      }
      if (sub == 0) row_scale[r] = s;
    }
    __syncthreads();
    i32x4 q[kSteps];
#pragma unroll
    for (int s = 0; s < kSteps; s++)
      q[s] = *reinterpret_cast<const i32x4*>(codes + lane % 16 * kPitch + 64 * s + lane / 16 * 16);
    const f32x4a4 qs = *reinterpret_cast<const f32x4a4*>(row_scale + lane / 16 * 4);
    // The lane's 16 bytes of each unit (past the bounds: their first, which meet zeros), their
    // place in `stage`, and those of the product's: of page lane % 16, of the unit's first half.
    int off[kUnits];
#pragma unroll
    for (int u = 0; u < kUnits; u++) off[u] = 128 * u + lane % 8 * 16 < 2 * D ? 128 * u + lane % 8 * 16 : 0;
    uint8_t* const put = stage[wave] + lane / 8 * 128 + ((lane % 8 ^ lane / 8) << 4);
    const uint8_t* const get = stage[wave] + lane % 16 * 128;
    const int get_at = (lane / 16 ^ lane % 8) << 4;
    if (h0) look_up(page, start);
    for (int p0 = start; p0 < top; p0 += kStride) {
      u32x4 k[kAtOnce][kUnits][2];
      float ks[kAtOnce];
      bool there[kAtOnce];
#pragma unroll
      for (int i = 0; i < kAtOnce; i++) {
        there[i] = page[i] >= 0 && page[i] < a.k.pages;
        const int id = there[i] ? page[i] : 0;
#pragma unroll
        for (int j = 0; j < 2; j++) {
          const int8_t* const src = a.k.codes +
                                    (size_t)__shfl(id, lane / 8 + 8 * j, 64) * a.k.page +
                                    (size_t)2 * g * D;
#pragma unroll
          for (int u = 0; u < kUnits; u++) k[i][u][j] = load_global<u32x4>(src + off[u]);
        }
        ks[i] = load_global<float>(a.k.scale + (size_t)id * a.k.s_page + g);
      }
      look_up(page, p0 + kStride);
#pragma unroll
      for (int i = 0; i < kAtOnce; i++) {
        const int p = p0 + 16 * i + lane % 16;
        i32x4 acc = {0, 0, 0, 0};
#pragma unroll
        for (int u = 0; u < kUnits; u++) {
          // (pages 8 on have the order of the first eight)
          *reinterpret_cast<u32x4*>(put) = k[i][u][0];
          *reinterpret_cast<u32x4*>(put + 8 * 128) = k[i][u][1];
          wave_lds_sync();
          i32x4 x[2];
#pragma unroll
          for (int s = 0; s < 2; s++)
            x[s] = *reinterpret_cast<const i32x4*>(get + (get_at ^ s << 6));
          wave_lds_sync();
#pragma unroll
          for (int s = 0; s < 2; s++)
            acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(q[2 * u + s], x[s], acc, 0, 0, 0);
        }
        // Rows lane / 16 * 4 on of page lane % 16.
        float m[4];
#pragma unroll
        for (int j = 0; j < 4; j++) m[j] = (float)acc[j] * qs[j];
        if (a.rows >= 2) m[0] = fmaxf(m[0], m[1]), m[1] = fmaxf(m[2], m[3]);
        if (a.rows >= 4) m[0] = fmaxf(m[0], m[1]);
        if (a.rows >= 8) m[0] = fmaxf(m[0], __shfl_xor(m[0], 16, 64));
        if (a.rows >= 16) m[0] = fmaxf(m[0], __shfl_xor(m[0], 32, 64));
        const int tokens = a.rows >= 4 ? 1 : 4 / a.rows;  // of a lane
#pragma unroll
        for (int j = 0; j < 4; j++) {
          const int tok = lane / 16 * 4 / a.rows + j;
          if (j >= tokens || tok >= nt || p >= top) continue;
          uint32_t key = key_of(m[j] * ks[i]);
          if (!there[i] || p > ((pos0 + tok) >> shift) - a.last) key = 0;
          uint32_t* const to = keys_of + tok * keys_step + p;
          *to = h0 ? max(*to, key) : key;
        }
      }
    }
    __syncthreads();
  }

  if (kStep == kScores) return;
  if (kStep == kChoice && kTeam) {
    for (int tok = 0; tok < nt; tok++)
      for (int p = bottom + tid; p < top; p += 64 * kWaves)
        keys[(size_t)tok * a.pitch + p] =
            load_global<uint32_t>(all_keys + (size_t)tok * KV * a.pitch + p);
    __syncthreads();
  }

  const int threads = kTeam ? 64 * kWaves : 64, at = kTeam ? tid : lane;
  int* const bins = hist[kTeam ? 0 : wave];
  for (int tok = kTeam ? 0 : wave; tok < nt; tok += kTeam ? 1 : kWaves) {
    const int64_t pos = pos0 + tok;
    const int own = pos < 0 ? -1 : (int)(pos >> shift);
    const int lo = a.first, hi = min(most, own + 1 - a.last);
    const uint32_t* const key = kStep == kChoice && !kTeam ? all_keys + (size_t)tok * KV * a.pitch
                                                           : keys + (size_t)tok * a.pitch;
    // The candidates' keys, some a thread at once (0 past them); all lanes go through it.
    auto each = [&](auto&& f) __attribute__((always_inline)) {
      constexpr int kKeysAtOnce = 8;
      for (int p0 = lo; p0 < hi; p0 += kKeysAtOnce * threads) {
        uint32_t k[kKeysAtOnce];
#pragma unroll
        for (int i = 0; i < kKeysAtOnce; i++) {
          const int p = p0 + i * threads + at;
          k[i] = key[p < hi ? p : lo];
          k[i] = p < hi ? k[i] : 0;
        }
#pragma unroll
        for (int i = 0; i < kKeysAtOnce; i++)
          if (p0 + i * threads < hi) f(k[i]);
      }
    };
    // Candidates, the smallest and largest key, over all threads.
    int all = 0;
    uint32_t low = 0xFFFFFFFFu, high = 0;
    each([&](uint32_t k) __attribute__((always_inline)) {
      all += __popcll(__ballot(k != 0));
      low = min(low, k ? k : 0xFFFFFFFFu);
      high = max(high, k);
    });
    low = ~wave_max(~low);
    high = wave_max(high);
    if (kTeam) {
      if (lane == 0) ends[wave] = make_uint2(low, high), counts[wave].x = all;
      __syncthreads();
      all = 0;
      for (int w = 0; w < kWaves; w++) {
        low = min(low, ends[w].x);
        high = max(high, ends[w].y);
        all += counts[w].x;
      }
    }
    // Keys above `least` are taken, and `ties` of those that are `least`; `left` of the keys
    // that agree with it in the bits from `bits` on are to be.
    const int need = a.count - a.first - a.last;
    uint32_t least = all ? low : 1;
    int ties = 0x7FFFFFFF, left = need;
    if (all > need && need > 0 && high > low) {
      // From the first bit in which keys differ on, up to eight bits at a time.
      int bits = 32 - __clz((int)(high - low));
      uint32_t span = 0xFFFFFFFFu;  // the keys' differences from `from` are at most this
      uint32_t from = low;
      while (true) {
        const int width = min(bits, 8), down = bits - width;
        for (int i = at; i < 256; i += threads) bins[i] = 0;
        lds_sync<kTeam>();
        // (the largest first)
        each([&](uint32_t k) __attribute__((always_inline)) {
          const uint32_t d = k - from;
          if (k >= from && d <= span) atomicAdd(&bins[(d >> down) ^ 255], 1);
        });
        lds_sync<kTeam>();
        // The bin in which the left-th lies; a lane has four.
        const int4 c = *reinterpret_cast<const int4*>(bins + 4 * lane);
        const int upto = (int)wave_scan(c.x + c.y + c.z + c.w);
        const int in = __ffsll((long long)__ballot(upto >= left)) - 1;
        const int c0 = __builtin_amdgcn_readlane(c.x, in), c1 = __builtin_amdgcn_readlane(c.y, in);
        const int c2 = __builtin_amdgcn_readlane(c.z, in), c3 = __builtin_amdgcn_readlane(c.w, in);
        left -= __builtin_amdgcn_readlane(upto, in) - (c0 + c1 + c2 + c3);
        int bin = 4 * in, here = c0;
        if (left > here) left -= here, bin++, here = c1;
        if (left > here) left -= here, bin++, here = c2;
        if (left > here) left -= here, bin++, here = c3;
        from += (uint32_t)(bin ^ 255) << down;
        bits = down;
        lds_sync<kTeam>();
        if (here == left || bits == 0) break;  // (all of the bin, or one key's)
        span = (1u << bits) - 1;
      }
      least = from;
      if (bits == 0) ties = left;
    } else if (all > need) {
      ties = need;
    }
    // In the pages' order; kTeam: each wave a part of them, after how many the others take.
    const int per = kTeam ? (max(hi - lo, 0) + threads - 1) / threads * 64 : max(hi - lo, 0);
    const int p_lo = kTeam ? min(lo + wave * per, max(hi, lo)) : lo;
    const int p_hi = kTeam ? min(p_lo + per, hi) : hi;
    int* const out = a.out + ((size_t)(t0 + tok) * KV + g) * a.count;
    int put = min(a.first, own + 1);
    const int head = put;
    int total = 0;
    if (kTeam) {
      int more = 0, same = 0;
      for (int p0 = p_lo; p0 < p_hi; p0 += 64) {
        const int p = p0 + lane;
        const uint32_t k = p < p_hi ? key[p] : 0;
        more += __popcll(__ballot(k > least));
        same += __popcll(__ballot(k && k == least));
      }
      __syncthreads();
      if (lane == 0) counts[wave] = make_int2(more, same);
      __syncthreads();
      int before = 0;  // that are `least`, in the waves before
      for (int w = 0; w < kWaves; w++) {
        const int2 c = counts[w];
        const int take = need > 0 ? c.x + min(c.y, max(ties - before, 0)) : 0;
        if (w < wave) put += take;
        total += take;
        if (w == wave) same = before;
        before += c.y;
      }
      ties = max(ties - same, 0);
    }
    for (int p0 = p_lo; p0 < p_hi && need > 0; p0 += 64) {
      const int p = p0 + lane;
      const uint32_t k = p < p_hi ? key[p] : 0;
      const uint64_t same = __ballot(k && k == least), before = (1ull << lane) - 1;
      const bool take = k > least || (k && k == least && __popcll(same & before) < ties);
      const uint64_t taken = __ballot(take);
      if (take) out[put + __popcll(taken & before)] = p;
      put += __popcll(taken);
      ties -= min(ties, (int)__popcll(same));
    }
    if (kTeam) put = head + total;
    const int tail = max(own + 1 - a.last, head);
    for (int i = at; i < head; i += threads) out[i] = i;
    for (int p = tail + at; p <= own; p += threads) out[put + p - tail] = p;
    put += own + 1 - tail;
    for (int i = put + at; i < a.count; i += threads) out[i] = -1;
    if (kTeam) __syncthreads();  // (before the next token's counts)
  }
}

template <int DP, int kWaves, bool kTeam, int kStep>
hipError_t run_step(const SelectArgs& a, hipStream_t s) {
  const size_t groups = ((size_t)a.b.tokens / a.tokens + a.b.batch) * a.k.kv_heads;
  const size_t grid = kStep == kScores ? groups * a.splits : groups;
  const size_t lds =
      kStep == kScores || (kStep == kChoice && !kTeam) ? 0 : (size_t)a.tokens * a.pitch * 4;
  if (grid > 0xFFFFFFFFu / (64 * kWaves)) return hipErrorInvalidValue;
  const hipError_t e =
      set_lds_limit((const void*)select_pages_kernel<DP, kWaves, kTeam, kStep>, (int)lds);
  if (e != hipSuccess) return e;
  select_pages_kernel<DP, kWaves, kTeam, kStep><<<(unsigned)grid, 64 * kWaves, lds, s>>>(a);
  return hipGetLastError();
}

template <int DP>
hipError_t run_select(const SelectPlan& p, SelectArgs& a, hipStream_t s) {
  if (a.scores) {
    hipError_t e = run_step<DP, 4, false, kScores>(a, s);
    if (e != hipSuccess) return e;
    a.tokens = p.team ? 1 : 4;
    return p.team ? run_step<64, kTeamWaves, true, kChoice>(a, s)
                  : run_step<64, 4, false, kChoice>(a, s);
  }
  return p.team ? run_step<DP, kTeamWaves, true, kBoth>(a, s) : run_step<DP, 4, false, kBoth>(a, s);
}

}  // namespace

hipError_t launch_key_bounds(const KeyBounds& o, const KvCache& c, const KvBatch& b, int num_cus,
                             hipStream_t s) {
  BoundsArgs a = {c, b, o, 0};
  while (8 << a.lane_shift < c.head_dim) a.lane_shift++;
  // Work-groups for all pages that the batch can have, or as many as the chip holds.
  const size_t slots = std::min((size_t)(b.tokens >> c.page_shift) + 2 * (size_t)b.batch,
                                (size_t)b.batch * ((size_t)b.width + 2));
  const unsigned grid = (unsigned)std::min(slots * c.kv_heads, (size_t)8 * num_cus);
  if (c.dtype == kKvFp16)
    key_bounds_kernel<kKvFp16><<<grid, 256, 0, s>>>(a);
  else if (c.dtype == kKvInt8)
    key_bounds_kernel<kKvInt8><<<grid, 256, 0, s>>>(a);
  else
    key_bounds_kernel<kKvFp4><<<grid, 256, 0, s>>>(a);
  return hipGetLastError();
}

// Bytes of the scores between two kernels at most.
constexpr size_t kMaxScores = (size_t)1 << 30;

SelectPlan select_plan(int heads, const KeyBounds& k, const KvBatch& b, int pages, int num_cus) {
  SelectPlan p = {};
  p.pages = k.pages ? pages : 0;  // (none: nothing has a score)
  p.pitch = (p.pages + 3) / 4 * 4;
  p.rows = 1;
  while (p.rows < 16 && p.rows < heads / k.kv_heads) p.rows *= 2;
  const size_t rows = (size_t)b.tokens * k.kv_heads, most = 16 / p.rows;
  const size_t groups = ((size_t)b.tokens / most + b.batch) * k.kv_heads;
  p.splits = 1;
  p.chunk = (p.pages + 127) / 128 * 128;
  // One kernel, with the scores in LDS, or two and a workspace: where there are few
  // work-groups, so that as many as the chip holds score 128 pages or more each (us, one / two:
  // one token over 2048 pages 19.9 / 12.1, over 4096 32.5 / 13.8), and for chunks whose
  // scores would leave LDS for few waves (512 tokens of 8 kv heads and 4 heads each over 4096
  // pages 250 / 137, of 16 kv heads over 1024 90 / 49; 2048 of the first over 2048, in 32 KB, 236
  // / 248).
  const bool few = p.pages >= 1024 && 2 * groups <= (size_t)num_cus;
  const bool big = b.tokens > b.batch && most * p.pitch * 4 > 40 << 10;
  if (few) {
    const int n = (int)std::min<size_t>((size_t)num_cus / groups, (p.pages + 127) / 128);
    p.chunk = ((p.pages + n - 1) / n + 127) / 128 * 128;
    p.splits = (p.pages + p.chunk - 1) / p.chunk;
  }
  if ((few || big) && rows * p.pitch * 4 <= kMaxScores) {
    p.tokens = (int)most;
    p.team = rows <= 2 * (size_t)num_cus;
    p.bytes = rows * p.pitch * 4;
  }
  return p;
}

// In one kernel, with or for want of a workspace: as many tokens a work-group as a product
// has rows and LDS has room for.  Where these are one or two, or tokens are single, all of
// its waves look for one token's pages.
static void one_kernel(SelectPlan& p, const KvBatch& b) {
  p.splits = 1;
  p.tokens = std::max(1, std::min(16 / p.rows, kMaxScored / std::max(p.pitch, 1)));
  p.team = p.pages > 256 && (p.tokens <= 2 || b.tokens <= b.batch);
}

hipError_t launch_select_pages(const SelectPlan& plan, int* out, int count, int first, int last,
                               const float* q, size_t q_stride, int heads, const KeyBounds& k,
                               const KvBatch& b, void* ws, hipStream_t s) {
  SelectPlan p = plan;
  if (!ws || !p.bytes) one_kernel(p, b);
  SelectArgs a = {};
  a.k = k, a.b = b, a.out = out, a.q = q, a.q_stride = q_stride, a.heads = heads;
  a.group = heads / k.kv_heads, a.count = count, a.first = first, a.last = last;
  a.rows = p.rows, a.most = p.pages, a.pitch = p.pitch, a.tokens = p.tokens;
  a.splits = p.splits, a.chunk = p.chunk, a.scores = p.bytes ? (uint32_t*)ws : nullptr;
  return k.head_dim <= 64    ? run_select<64>(p, a, s)
         : k.head_dim <= 128 ? run_select<128>(p, a, s)
                             : run_select<256>(p, a, s);
}

}  // namespace hypno
