// Attention over 4-bit caches for sequences with few rows, and of single tokens over
// selected pages: the work of attn_few_kernel (a work-group takes one kv head of a
// sequence and a range of its positions, its waves run through tiles of 32 keys on their
// own and add up at the end) on codes that stay 4 bits wide up to the registers.
//
// A run of keys of a kv head in one page is one piece of memory, codes as well as each
// group's scales: whole runs are copied into a wave's own LDS, a tile before they are used
// (two ahead leave LDS for two work-groups a CU, not four, and take 64 sequences of up to 8192
// a quarter longer).  What is copied past the last key is masked, its scales of V set to 0.
// K: lane (key, quarter) reads its quarter of the key's codes as they are, each eight of
// which have one scale; q is held in the same order.  V: the 4-bit transposing read gives a
// lane eight keys' codes of two channels, the scales lie key by key already.  Both become
// fp16 code * scale, rounded once (the values that the cache stands for), two a conversion
// and a product: 128 of some 210 vector operations a tile.
//
// Bound: HBM for long contexts (from 524288 to 1048576 positions of 8 kv heads of 128, 604 MB
// more take 99 us more: 6.1 TB/s); starts, ends and the join for shorter ones.  One token over
// 131072 (151 MB) 33 to 36 us and 5 to join, 64 sequences of up to 8192 (340 MB) 82 to 84 in
// all, 5 to 6 of them to join, and 87.5 with every product twice (kPass 16, three work-groups
// a CU, beside 84).  700 positions of 32/4 heads of 64: 8.0 us, dependent reads of the
// sequence's place, its page and keys, three tiles, the waves' sum.
#include "attention_few.hpp"

namespace hypno {

namespace {

constexpr int kQ = kFewQ, kKeys = kFewKeys;

// kLen: keys of a tile in one page, the whole tile's where pages have as many.
template <int DP, int kLen>
struct Few4 {
  static constexpr int kRuns = kKeys / kLen;
  // Bytes of a run, and instructions that copy them, 16 and 4 bytes a lane.
  static constexpr int kCodes = kLen * DP / 2, kScales = kLen * DP / kFp4Group * 2;
  static constexpr int kCodeCopies = (kCodes + 1023) / 1024, kScaleCopies = (kScales + 255) / 256;
  static constexpr int kTile = 2 * kRuns * (kCodes + kScales);
  // Two tiles; afterwards the wave's part.
  static constexpr int kWave = 2 * kTile > few_part_bytes<DP>() ? 2 * kTile : few_part_bytes<DP>();
};

// Four bytes a lane, as dma16.
__device__ __forceinline__ void dma4(const void* base, uint32_t off, uint8_t* lds) {
#if defined(__HIP_DEVICE_COMPILE__)
  const uint32_t at = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) void*)lds;
  asm volatile("s_nop 0\n\tglobal_load_lds_dword %1, %2"
               :
               : "{m0}"(at), "v"(off), "s"(base)
               : "memory");
#endif
}

// Sum of a lane's value and that of the lane eight columns on.
__device__ __forceinline__ float both_halves(float x) {
  return x + __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), 0x128, 0xF, 0xF,
                                                        false));  // row_ror:8
}

// kPass: rows that go through the tiles together, 16, or 8 whose two parts of q (and of the
// weights) are columns of one product: half the products, and registers for a work-group more
// on a CU.
template <int DP, int kLen, int kPass, int kWaves, bool kList>
__global__ void __launch_bounds__(64 * kWaves, kWaves == 8 ? 2 : DP > 128 ? 2 : kPass == 8 ? 4 : 3)
    attn_few4_kernel(AttnArgs a) {
  typedef Few4<DP, kLen> T;
  constexpr int kRuns = T::kRuns;
  typedef Rows<kKvFp16, kQ, DP, kKeys> R;
  extern __shared__ __attribute__((aligned(16))) uint8_t smem[];
  __shared__ uint32_t again;
  __shared__ int counts[kWaves];
  SeenPage* const list = reinterpret_cast<SeenPage*>(smem + kWaves * T::kWave);
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int KV = a.c.kv_heads, G = a.group, D = a.c.head_dim, B = D / kFp4Group;
  const int col = lane % kQ, grp = lane / kQ, shift = a.c.page_shift;
  // (the order of attn_few_kernel)
  const int units = kList ? a.b.tokens : a.b.batch;
  const int g = blockIdx.x % KV, split = blockIdx.x / KV / units;
  const int unit = blockIdx.x / KV % units, b = kList ? find_seq(a.b, unit, 0, 0) : unit;
  if (kList && (b < 0 || b >= a.b.batch)) return;
  const Seq sq = seq_of(a.b, b);
  const int ti0 = kList ? unit - sq.first : 0;
  if (kList && (ti0 < 0 || ti0 >= sq.n)) return;  // (cu_q that does not ascend)
  const int rows = kList ? G : sq.n * G;
  if (!kList && rows > a.few) return;
  const bool past = too_long(a, sq);
  int seen = 0;
  if (kList && !past) {
    const int* const selected = a.selected + ((size_t)unit * KV + g) * a.count;
    seen = seen_pages(a, b, sq.kv - sq.n + ti0, selected, list, counts) << shift;
  }

  const int mask = (1 << shift) - 1;
  const uint8_t* const kg = (const uint8_t*)a.c.k + (((size_t)g << shift) * D >> 1);
  const uint8_t* const vg = (const uint8_t*)a.c.v + (((size_t)g << shift) * D >> 1);
  const _Float16* const ksg = (const _Float16*)a.c.k_scale + ((size_t)(g * B) << shift);
  const _Float16* const vsg = (const _Float16*)a.c.v_scale + ((size_t)(g * B) << shift);
  uint8_t* const ring = smem + wave * T::kWave;
  // In a tile: K's codes run by run [16][D / 2], V's, K's scales run by run [B][16], V's.
  constexpr int kV = kRuns * T::kCodes, kKs = 2 * kV, kVs = kKs + kRuns * T::kScales;
  const bool same = a.c.k_page == a.c.v_page && a.c.ks_page == a.c.vs_page;
  const int row_bytes = D / 2;
  const int* const table = a.b.page_table + (size_t)b * a.b.width;
  // Where the codes and scales of a tile's first and second 16 keys are.
  auto codes_of = [&](int half) __attribute__((always_inline)) {
    return half * 16 * (kLen == 16 ? DP / 2 : row_bytes);
  };
  auto scales_of = [&](int half) __attribute__((always_inline)) {
    return half * (kLen == 16 ? T::kScales : 32);
  };
  // A lane's first element of step s of a score's sum: quarter by quarter of each 128.
  constexpr int kPart = DP / 4 < 32 ? DP / 4 : 32;
  auto element = [&](int s) __attribute__((always_inline)) {
    return 8 * s / kPart * 4 * kPart + kPart * grp + 8 * s % kPart;
  };

  for (int r0 = 0; r0 < rows; r0 += kPass) {
    const int r1 = min(r0 + kPass, rows), s0 = r0 & -kQ;
    // (the ranges are those of 16 rows, as in the kernel that joins them)
    const Span span = kList ? Span{0, seen} : span_of(a, sq, s0, min(s0 + kQ, rows));
    int lo = past ? 0 : span.lo, hi = past ? 0 : span.hi;
    if (kList) {
      lo = (int)min((int64_t)split * a.fs.chunk, (int64_t)hi);
      hi = (int)min((int64_t)hi, (int64_t)lo + a.fs.chunk);
    } else if (a.fs.splits > 1) {
      const int64_t start = lo + (int64_t)split * a.fs.chunk;
      if (start >= hi && split) continue;
      if (split + 1 < a.fs.splits) hi = (int)min((int64_t)hi, start + a.fs.chunk);
      lo = (int)start;
    }
    const int row = min(r0 + col % kPass, rows - 1);
    const int ti = kList ? ti0 : row / G, h = g * G + (kList ? row : row % G);
    const int t = sq.first + ti;
    const int seen_lo = first_seen(a, sq, ti), seen_hi = min(sq.kv - sq.n + ti, hi - 1);
    const int all_lo = first_seen(a, sq, (r1 - 1) / G);
    const int all_hi = min(sq.kv - sq.n + r0 / G, hi - 1);
    // Run i of a tile: its page (-1: none), first slot, and the positions of it that are there
    // to be seen (0: it is another run again).
    int pid[kRuns] = {}, slot[kRuns] = {};
    uint32_t bad = 0;
    const int tiles = (hi - lo + kKeys - 1) / kKeys;
    const int mine = max(0, (tiles - wave + kWaves - 1) / kWaves);  // this wave's
    auto place = [&](int tile) __attribute__((always_inline)) {
      return lo + (tile * kWaves + wave) * kKeys;
    };
    auto look_up = [&](int tile) __attribute__((always_inline)) {
#pragma unroll
      for (int i = 0; i < kRuns; i++) {
        const int p = min(place(tile) + kLen * i, (hi - 1) & -kLen);
        if (kList) {
          const SeenRun run = seen_run<kLen>(a, list, p);
          pid[i] = run.page, slot[i] = run.slot;
        } else {
          pid[i] = load_const<int>(table + (p >> shift));
          slot[i] = p & mask;
        }
      }
    };
    auto issue = [&](uint8_t* to) __attribute__((always_inline)) {
#pragma unroll
      for (int i = 0; i < kRuns; i++) {
        const bool none = (uint32_t)pid[i] >= (uint32_t)a.c.pages;
        bad |= none;
        const uint32_t pg = none ? 0 : pid[i], first = slot[i] * row_bytes;
        // (strides are below 2^31; K's and V's are mostly the same)
        const uint64_t ko = (uint64_t)pg * (uint32_t)a.c.k_page + first;
        const uint64_t kso = (uint64_t)pg * (uint32_t)a.c.ks_page + slot[i];
        uint64_t vo = ko, vso = kso;
        if (!same) {
          asm volatile("" ::: "memory");  // (not computed on every way)
          vo = (uint64_t)pg * (uint32_t)a.c.v_page + first;
          vso = (uint64_t)pg * (uint32_t)a.c.vs_page + slot[i];
        }
        const uint8_t *const kp = kg + ko, *const vp = vg + vo;
        const _Float16 *const ksp = ksg + kso, *const vsp = vsg + vso;
        to += i * T::kCodes;
#pragma unroll
        for (int c = 0; c < T::kCodeCopies; c++)
          if ((c * 64 + lane) * 16 < kLen * row_bytes) {
            dma16<!kList>(kp, c * 1024 + lane * 16, to + c * 1024);
            dma16<!kList>(vp, c * 1024 + lane * 16, to + kV + c * 1024);
          }
        to -= i * (T::kCodes - T::kScales);
#pragma unroll
        for (int c = 0; c < T::kScaleCopies; c++) {
          const int j = c * 64 + lane, blk = j / (kLen / 2);
          if (blk < B) {
            const uint32_t off = ((blk << shift) + j % (kLen / 2) * 2) * 2;
            dma4(ksp, off, to + kKs + c * 256);
            dma4(vsp, off, to + kVs + c * 256);
          }
        }
        to -= i * T::kScales;
      }
    };

    if (mine > 0) {
      look_up(0);
      issue(ring);
      look_up(1);
    }
    R x;
    x.init_of(r0 + col % kPass < rows ? a.q + (size_t)t * a.q_stride + (size_t)h * D : nullptr, D,
              a.scale, element);
    if (kPass == 8) {
#pragma unroll
      for (int st = 0; st < R::kSteps; st++) x.qh[st] = col < 8 ? x.qh[st] : x.ql[st];
    }
    for (int tile = 0; tile < mine; tile++) {
      const int p0 = place(tile);
      uint8_t* const at = ring + tile % 2 * T::kTile;
      // (this tile's copies, and all reads of the one before)
      asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
      // Positions of the runs that are there to be seen, and the rest's scales of V: 0, as
      // the codes are finite and their weights 0.
      int there[kRuns];
      bool whole = true;
#pragma unroll
      for (int i = 0; i < kRuns; i++) {
        const int p = p0 + kLen * i;
        there[i] = p >= hi ? 0 : kList ? seen_run<kLen>(a, list, p).seen : min(hi - p, kLen);
        whole &= there[i] == kLen;
      }
      if (!whole) {
#pragma unroll
        for (int i = 0; i < kRuns; i++)
          for (int k = lane; k < B * kLen; k += 64)
            if (k % kLen >= there[i])
              *reinterpret_cast<_Float16*>(at + kVs + i * T::kScales + k * 2) = (_Float16)0.0f;
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      }
      // All that this tile needs of LDS is on its way before the copies of a later one.
      constexpr int kQuarters = DP / 4 / kPart;  // of a key's codes in a lane
      typedef uint32_t codes_t __attribute__((ext_vector_type(kPart / 8)));
      codes_t kc[2][kQuarters];
      _Float16 ks[2][kQuarters];
#pragma unroll
      for (int i = 0; i < 2; i++)
#pragma unroll
        for (int c = 0; c < kQuarters; c++) {
          const int e = c * 4 * kPart + kPart * grp, blk = e < D ? e / kFp4Group : 0;
          kc[i][c] = *reinterpret_cast<const codes_t*>(at + codes_of(i) + col * row_bytes +
                                                       (e < D ? e / 2 : 0));
          ks[i][c] = *reinterpret_cast<const _Float16*>(at + kKs + scales_of(i) +
                                                        (blk * kLen + col) * 2);
        }
      if (tile + 1 < mine) {
        issue(ring + (tile + 1) % 2 * T::kTile);
        look_up(tile + 2);
      }
      typename R::acc s[2];
#pragma unroll
      for (int i = 0; i < 2; i++) s[i] = typename R::acc{};
#pragma unroll
      for (int st = 0; st < R::kSteps; st++) {
        const int c = 8 * st / kPart;
        half8 k[2];
#pragma unroll
        for (int i = 0; i < 2; i++)
          k[i] = f16x8(fp4_to_f16(kc[i][c][st % (kPart / 8)], half2v{ks[i][c], ks[i][c]}));
#pragma unroll
        for (int i = 0; i < 2; i++) s[i] = Mfma<kQ>::mul(k[i], x.qh[st], s[i]);
#pragma unroll
        for (int i = 0; i < 2 && kPass == 16; i++) s[i] = Mfma<kQ>::mul(k[i], x.ql[st], s[i]);
        __builtin_amdgcn_sched_barrier(0);
      }
      if (kPass == 8) {
#pragma unroll
        for (int i = 0; i < 2; i++)
#pragma unroll
          for (int r = 0; r < 4; r++) s[i][r] = both_halves(s[i][r]);
      }
      // Keys that a row does not see.  (Apart from the maximum: two ways to that one have the
      // compiler copy all of o.)
      if (kList ? !whole : p0 < all_lo || p0 + kKeys - 1 > all_hi) {
#pragma unroll
        for (int i = 0; i < 2; i++)
#pragma unroll
          for (int r = 0; r < 4; r++) {
            const int key = 16 * i + 4 * grp + r, p = p0 + key;
            if (kList ? key % kLen >= there[i / (kLen / 16)] : p < seen_lo || p > seen_hi)
              s[i][r] = -__builtin_inff();
          }
      }
      x.template maximum<0>(s, 0, 0, nullptr);

      // Weights, two fp16 parts each, in the order of V's keys: run by run four a lane.
      const float off = R::kTop - (x.m == -__builtin_inff() ? 0.0f : x.m);
      float neg = -1.0f, sum = 0.0f;
      asm("" : "+s"(neg));
      u32x4 wh, wl;
#pragma unroll
      for (int i = 0; i < 4; i++) {
        float w[2];
#pragma unroll
        for (int j = 0; j < 2; j++)
          w[j] = __builtin_amdgcn_exp2f(fmaf(s[i / 2][i % 2 * 2 + j], x.c, off));
        sum += w[0] + w[1];
        uint32_t hi16, lo16;
        split_f16(w[0], w[1], neg, hi16, lo16);
        wh[i] = kPass == 16 || col < 8 ? hi16 : lo16, wl[i] = lo16;
      }
      x.l += sum;
      // Channels 32 blk + col and 16 on, of keys 4 grp to 4 grp + 3 of both halves of the tile:
      // row j of the transposed 16 x 16 codes is key j % 4 of half j / 4 % 2, and from j = 8
      // on 16 channels on.
      const uint8_t* const vsrc = at + kV + codes_of(col / 4 % 2) + (4 * grp + col % 4) * row_bytes +
                                  col / 8 * 8;
#pragma unroll
      for (int blk = 0; blk < DP / kFp4Group; blk++) {
        // (past D: whatever is there, for channels that nobody reads)
        typedef int int2v __attribute__((ext_vector_type(2)));
        const auto codes = __builtin_amdgcn_ds_read_tr4_b64_v2i32(
            (__attribute__((address_space(3))) int2v*)(vsrc + blk * 16));
        uint2 sc[2];
#pragma unroll
        for (int i = 0; i < 2; i++)
          sc[i] = *reinterpret_cast<const uint2*>(at + kVs + scales_of(i) +
                                                  (blk * kLen + 4 * grp) * 2);
        const half2v scale[4] = {
            __builtin_bit_cast(half2v, sc[0].x), __builtin_bit_cast(half2v, sc[0].y),
            __builtin_bit_cast(half2v, sc[1].x), __builtin_bit_cast(half2v, sc[1].y)};
#pragma unroll
        for (int half = 0; half < 2; half++) {
          const uint32_t c = (uint32_t)codes[half];
          const half2v v[4] = {__builtin_amdgcn_cvt_scalef32_pk_f16_fp4(c, 1.0f, 0),
                               __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(c, 1.0f, 1),
                               __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(c, 1.0f, 2),
                               __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(c, 1.0f, 3)};
          u32x4 y;
#pragma unroll
          for (int i = 0; i < 4; i++)
            y[i] = __builtin_bit_cast(uint32_t, (half2v)(v[i] * scale[i]));
          const int n = 2 * blk + half;
          x.o[n] = Mfma<kQ>::mul(f16x8(y), f16x8(wh), x.o[n]);
          if (kPass == 16) x.o[n] = Mfma<kQ>::mul(f16x8(y), f16x8(wl), x.o[n]);
        }
      }
    }
    x.finish(bad != 0);
    if (kPass == 8) {
#pragma unroll
      for (int n = 0; n < R::kDt; n++)
#pragma unroll
        for (int r = 0; r < 4; r++) x.o[n][r] = both_halves(x.o[n][r]);
    }
    few_store<DP, kWaves, T::kWave, kPass, kList>(a, sq, g, ti0, r0, rows, split, past, x, smem, again);
  }
}

template <int DP, int kLen, int kPass, int kWaves, bool kList>
hipError_t launch(const AttnArgs& a, hipStream_t s) {
  const int lds = kWaves * Few4<DP, kLen>::kWave + (kList ? a.count * (int)sizeof(SeenPage) : 0);
  const size_t grid = (size_t)(kList ? a.b.tokens : a.b.batch) * a.c.kv_heads * a.fs.splits;
  if (grid > 0xFFFFFF) return hipErrorInvalidValue;
  const hipError_t e = set_lds_limit((const void*)attn_few4_kernel<DP, kLen, kPass, kWaves, kList>, lds);
  if (e != hipSuccess) return e;
  attn_few4_kernel<DP, kLen, kPass, kWaves, kList><<<(unsigned)grid, 64 * kWaves, lds, s>>>(a);
  return hipGetLastError();
}

template <int DP, int kLen, int kPass, int kWaves>
hipError_t run(const AttnArgs& a, hipStream_t s) {
  return a.selected ? launch<DP, kLen, kPass, kWaves, true>(a, s)
                    : launch<DP, kLen, kPass, kWaves, false>(a, s);
}

template <int DP, int kWaves>
hipError_t run(const AttnArgs& a, hipStream_t s) {
  // (a sequence with more rows than a pass goes through its keys once for each.  A call with
  // more tokens than sequences takes 16 rows for all of them: one sequence of two tokens among
  // 64 of up to 8192 87 -> 96 us, of up to 2000 28 -> 39, a launch of the kernel for longer
  // sequences among it)
  const bool one = a.group <= 8 && (a.selected || a.b.tokens <= a.b.batch);
  if (a.c.page_shift > kRunShift)
    return one ? run<DP, 32, 8, kWaves>(a, s) : run<DP, 32, 16, kWaves>(a, s);
  return one ? run<DP, 16, 8, kWaves>(a, s) : run<DP, 16, 16, kWaves>(a, s);
}

}  // namespace

hipError_t launch_attn_few4(const AttnArgs& a, hipStream_t s) {
  const int D = a.c.head_dim;
  if (D > 128) return run<256, 4>(a, s);
  if (a.few_waves == 8) return D <= 64 ? run<64, 8>(a, s) : run<128, 8>(a, s);
  return D <= 64 ? run<64, 4>(a, s) : run<128, 4>(a, s);
}

}  // namespace hypno
