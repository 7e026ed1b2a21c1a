// Attention over 4-bit caches for sequences with few rows, and of single tokens over
// selected pages: the work of attn_few_kernel (a work-group takes one kv head of a
// sequence and a range of its positions, its waves run through tiles of 32 keys on their
// own and add up at the end) on codes that stay 4 bits wide up to the registers.
//
// A run of 16 keys of a kv head is one piece of memory, codes as well as each group's
// scales: whole runs are copied into a wave's own LDS, kAhead tiles before they are used.
// K: lane (key, quarter) reads its quarter of the key's codes, which has one scale or two,
// as they are; q is held in the same order.  V: the 4-bit transposing read gives a lane
// eight keys' codes of two channels, the scales lie key by key already.  Both become fp16
// code * scale, rounded once (the values that the cache stands for), two a conversion and
// a product.
#include "attention_few.hpp"

namespace hypno {

namespace {

constexpr int kQ = kFewQ, kKeys = kFewKeys, kRuns = kKeys / kRun;

template <int DP>
struct Few4 {
  static constexpr int kAhead = DP > 128 ? 2 : 3;
  static constexpr int kCopies = DP > 128 ? 2 : 1;  // instructions of a run's codes
  static constexpr int kCodes = kRun * DP / 2, kScales = kRun * DP / kFp4Group * 2;  // of a run
  static constexpr int kTile = 2 * kRuns * (kCodes + kScales);
  static constexpr int kLoads = 2 * kRuns * (kCopies + 1);
  static constexpr int kStage = (kAhead + 1) * kTile;
  static constexpr int kWave = kStage > few_part_bytes<DP>() ? kStage : few_part_bytes<DP>();
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

template <int kCount>
__device__ __forceinline__ void wait_loads() {
#if defined(__HIP_DEVICE_COMPILE__)
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" : : "n"(kCount) : "memory");
#endif
}

template <int DP, int kWaves, bool kList>
__global__ void __launch_bounds__(64 * kWaves, kWaves == 8 ? 1 : DP > 128 ? 1 : 2)
    attn_few4_kernel(AttnArgs a) {
  typedef Few4<DP> T;
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
  const int pieces = D / 2;  // of 16 bytes, of a run's codes
  const uint32_t scale_off = (((lane / 8) << shift) * 2) + lane % 8 * 4;
  // A lane's first element of step s of a score's sum: quarter by quarter of each 128.
  constexpr int kPart = DP / 4 < 32 ? DP / 4 : 32;
  const auto element = [&](int s) __attribute__((always_inline)) {
    return 8 * s / kPart * 4 * kPart + kPart * grp + 8 * s % kPart;
  };

  for (int r0 = 0; r0 < rows; r0 += kQ) {
    const int r1 = min(r0 + kQ, rows);
    const Span span = kList ? Span{0, seen} : span_of(a, sq, r0, r1);
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
    const int row = min(r0 + col, rows - 1);
    const int ti = kList ? ti0 : row / G, h = g * G + (kList ? row : row % G);
    const int t = sq.first + ti;
    const int seen_lo = first_seen(a, sq, ti), seen_hi = min(sq.kv - sq.n + ti, hi - 1);
    const int all_lo = first_seen(a, sq, (r1 - 1) / G);
    const int all_hi = min(sq.kv - sq.n + r0 / G, hi - 1);
    bool bad = false;
    // Run i of the tile at p0: its page (-1: none), first slot, and the positions of it that
    // are there to be seen (0: it is another run again).
    int pid[kRuns] = {}, slot[kRuns] = {};
    const int tiles = (hi - lo + kKeys - 1) / kKeys;
    const int mine = max(0, (tiles - wave + kWaves - 1) / kWaves);
    auto place = [&](int p0, int i) __attribute__((always_inline)) {
      return lo + (p0 * kWaves + wave) * kKeys + kRun * i;  // (p0: the wave's tile)
    };
    auto look_up = [&](int tile) __attribute__((always_inline)) {
#pragma unroll
      for (int i = 0; i < kRuns; i++) {
        const int p = min(place(tile, i), (hi - 1) & -kRun);
        if (kList) {
          const SeenRun run = seen_run(a, list, p);
          pid[i] = run.page, slot[i] = run.slot;
        } else {
          pid[i] = load_const<int>(a.b.page_table + (size_t)b * a.b.width + (p >> shift));
          slot[i] = p & mask;
        }
      }
    };
    auto issue = [&](uint8_t* to) __attribute__((always_inline)) {
#pragma unroll
      for (int i = 0; i < kRuns; i++) {
        const int pg = __builtin_amdgcn_readfirstlane(page_of(a, pid[i], bad));
        const uint8_t* const kp = kg + (size_t)pg * a.c.k_page + (uint32_t)(slot[i] * pieces);
        const uint8_t* const vp = vg + (size_t)pg * a.c.v_page + (uint32_t)(slot[i] * pieces);
        const _Float16* const ksp = ksg + (size_t)pg * a.c.ks_page + slot[i];
        const _Float16* const vsp = vsg + (size_t)pg * a.c.vs_page + slot[i];
#pragma unroll
        for (int c = 0; c < T::kCopies; c++)
          if (c * 64 + lane < pieces) {
            dma16<!kList>(kp, c * 1024 + lane * 16, to + i * T::kCodes + c * 1024);
            dma16<!kList>(vp, c * 1024 + lane * 16, to + kV + i * T::kCodes + c * 1024);
          }
        if (lane < 8 * B) {
          dma4(ksp, scale_off, to + kKs + i * T::kScales);
          dma4(vsp, scale_off, to + kVs + i * T::kScales);
        }
      }
    };

    uint8_t* to = ring;
    if (mine > 0) {
      look_up(0);
#pragma unroll
      for (int i = 0; i < T::kAhead; i++)
        if (i < mine) {
          issue(to);
          to += T::kTile;
          look_up(i + 1);
        }
    }
    R x;
    x.init_of(r0 + col < rows ? a.q + (size_t)t * a.q_stride + (size_t)h * D : nullptr, D, a.scale,
              element);
    if (mine < T::kAhead) to = ring + T::kAhead * T::kTile;  // (not used)
    const uint8_t* at = ring;
    for (int tile = 0; tile < mine; tile++) {
      const int p0 = place(tile, 0);
      if (tile + T::kAhead <= mine)
        wait_loads<(T::kAhead - 1) * T::kLoads>();
      else
        wait_loads<0>();
      if (tile + T::kAhead < mine) {
        issue(to);
        to = to == ring + T::kAhead * T::kTile ? ring : to + T::kTile;
        look_up(tile + T::kAhead + 1);
      }
      // Positions of the runs that are there to be seen, and the rest's scales of V: 0, as
      // the codes are finite and their weights 0.
      int there[kRuns];
      bool whole = true;
#pragma unroll
      for (int i = 0; i < kRuns; i++) {
        const int p = place(tile, i);
        there[i] = p >= hi ? 0 : kList ? seen_run(a, list, p).seen : min(hi - p, kRun);
        whole &= there[i] == kRun;
      }
      if (!whole) {
#pragma unroll
        for (int i = 0; i < kRuns; i++)
          for (int k = lane; k < B * kRun; k += 64)
            if (k % kRun >= there[i])
              *reinterpret_cast<_Float16*>(const_cast<uint8_t*>(at) + kVs + i * T::kScales + k * 2) =
                  (_Float16)0.0f;
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      }

      typename R::acc s[kRuns];
#pragma unroll
      for (int i = 0; i < kRuns; i++) {
        s[i] = typename R::acc{};
        u32x4 k[R::kSteps];
#pragma unroll
        for (int c = 0; c < DP / 4 / kPart; c++) {
          const int e = c * 4 * kPart + kPart * grp, blk = e < D ? e / kFp4Group : 0;
          const uint8_t* const src = at + i * T::kCodes + col * (D / 2) + (e < D ? e / 2 : 0);
          const _Float16 sc = *reinterpret_cast<const _Float16*>(at + kKs + i * T::kScales +
                                                                 (blk * kRun + col) * 2);
          const half2v two = {sc, sc};
          if constexpr (kPart == 32) {
            const u32x4 codes = *reinterpret_cast<const u32x4*>(src);
#pragma unroll
            for (int j = 0; j < 4; j++) k[c * 4 + j] = fp4_to_f16(codes[j], two);
          } else {
            const uint2 codes = *reinterpret_cast<const uint2*>(src);
            k[0] = fp4_to_f16(codes.x, two);
            k[1] = fp4_to_f16(codes.y, two);
          }
        }
#pragma unroll
        for (int st = 0; st < R::kSteps; st++) s[i] = Mfma<kQ>::mul(f16x8(k[st]), x.qh[st], s[i]);
#pragma unroll
        for (int st = 0; st < R::kSteps; st++) s[i] = Mfma<kQ>::mul(f16x8(k[st]), x.ql[st], s[i]);
      }
      if (kList) {
        if (whole)
          x.template maximum<0>(s, 0, 0, nullptr);
        else
          x.template maximum<2>(s, there[0], there[1], nullptr);
      } else if (p0 < all_lo || p0 + kKeys - 1 > all_hi) {
        x.template maximum<1>(s, seen_lo - p0, seen_hi - p0, nullptr);
      } else {
        x.template maximum<0>(s, 0, 0, nullptr);
      }

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
        wh[i] = hi16, wl[i] = lo16;
      }
      x.l += sum;
      // Channels 32 blk + col and 16 on, of keys 4 grp to 4 grp + 3 of both runs: row j of
      // the transposed 16 x 16 codes is key j % 4 of run j / 4 % 2 and half j / 8.
      const int j = lane % 16;
      const uint8_t* const vsrc = at + kV + j / 4 % 2 * T::kCodes + (4 * grp + j % 4) * (D / 2) +
                                  j / 8 * 8;
#pragma unroll
      for (int blk = 0; blk < DP / kFp4Group; blk++) {
        const int here = blk < B ? blk : 0;
        typedef int int2v __attribute__((ext_vector_type(2)));
        const auto codes = __builtin_amdgcn_ds_read_tr4_b64_v2i32(
            (__attribute__((address_space(3))) int2v*)(vsrc + here * 16));
        uint2 sc[kRuns];
#pragma unroll
        for (int i = 0; i < kRuns; i++)
          sc[i] = *reinterpret_cast<const uint2*>(at + kVs + i * T::kScales +
                                                  (here * kRun + 4 * grp) * 2);
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
          x.o[n] = Mfma<kQ>::mul(f16x8(y), f16x8(wl), x.o[n]);
        }
      }
      at = at == ring + T::kAhead * T::kTile ? ring : at + T::kTile;
    }
    x.finish(__any(bad));
    few_store<DP, kWaves, T::kWave, kList>(a, sq, g, ti0, r0, rows, split, past, x, smem, again);
  }
}

template <int DP, int kWaves, bool kList>
hipError_t launch(const AttnArgs& a, hipStream_t s) {
  const int lds = kWaves * Few4<DP>::kWave + (kList ? a.count * (int)sizeof(SeenPage) : 0);
  const size_t grid = (size_t)(kList ? a.b.tokens : a.b.batch) * a.c.kv_heads * a.fs.splits;
  if (grid > 0xFFFFFF) return hipErrorInvalidValue;
  const hipError_t e = set_lds_limit((const void*)attn_few4_kernel<DP, kWaves, kList>, lds);
  if (e != hipSuccess) return e;
  attn_few4_kernel<DP, kWaves, kList><<<(unsigned)grid, 64 * kWaves, lds, s>>>(a);
  return hipGetLastError();
}

template <int DP, int kWaves>
hipError_t run(const AttnArgs& a, hipStream_t s) {
  return a.selected ? launch<DP, kWaves, true>(a, s) : launch<DP, kWaves, false>(a, s);
}

}  // namespace

hipError_t launch_attn_few4(const AttnArgs& a, hipStream_t s) {
  const int D = a.c.head_dim;
  if (D > 128) return run<256, 4>(a, s);
  if (a.few_waves == 8) return D <= 64 ? run<64, 8>(a, s) : run<128, 8>(a, s);
  return D <= 64 ? run<64, 4>(a, s) : run<128, 4>(a, s);
}

}  // namespace hypno
