// Attention for sequences with few rows (single tokens, drafts): a work-group takes
// one kv head of a sequence and a range of its positions; its waves run through
// tiles of keys on their own, 16 rows at a time, and add up at the end.
//
// Tokens' selected pages go through the same tiles: 16 tokens of 64 pages of 64 (268 MB) 41
// us, 6.5 TB/s; 251 tokens of 31 pages of 32, 8-bit (209 MB, from L2) 57.
//
// Bound: HBM.  One token over 131072 positions (32/8 heads of 128, 537 MB): 78 us, 6.9
// TB/s; 64 sequences of up to 8192 (1.24 GB) 211 us with the sum of their ranges, 5.9; with
// 8-bit values (0.64 GB) 151 us, 4.3: there it is the way through the wave (codes to fp16 and bf16, 310 vector
// operations a tile, 40% of the cycles) at two waves a SIMD, which is what the registers
// allow (three with 42 of them spilt: 357 us; tiles of 64 keys, 15 spilt: 206).
//  * K goes from memory into the MFMA operands' registers, V into LDS, from where it is
//    read transposed; a wave has its own LDS and meets the others only at the end.
//  * Nothing but the next tile is in flight: 16 KB a wave, 128 KB a CU, several times
//    what the memory's latency takes at this rate.
//  * A context of up to 1024 positions is one work-group of eight waves a kv head: 8.0 us
//    for one token over 700 (32/4 heads of 64), most of it latency: the sequence's
//    place, its pages, three tiles one after the other, the waves' sum.

#include "attention_few.hpp"

namespace hypno {

namespace {

constexpr int kQ = kFewQ;
typedef uint32_t u32x4a8 __attribute__((ext_vector_type(4), aligned(8)));

template <int kType, int DP>
struct Few {
  static constexpr int kKeys = kFewKeys;
  static constexpr int kGroups = DP > 128 ? 1 : 2;  // a CU
  static constexpr int kRuns = kKeys / kRun;
  static constexpr int kBytes = kKeys * DP * 2;        // V of one tile in LDS
  static constexpr int kN = kKeys * DP / 8 / 64;       // 16-byte pieces of it a lane
  static constexpr int kBufs = kType == kKvFp16 ? 2 : 1;
  // Per wave: V, 8-bit: scales of K and V; afterwards o of 16 rows, maxima and sums.
  static constexpr int kStage = kBufs * kBytes + (kType == kKvInt8 ? 2 * kKeys * 4 : 0);
  static constexpr int kOut = few_part_bytes<DP>();
  static constexpr int kWave = kStage > kOut ? kStage : kOut;
};

// kOne: pages have kRun positions or more.  kWaves: 4, or 8 where a work-group takes all
// positions and these are few: half the tiles one after the other.  kList: a work-group
// takes one token and the pages selected for it, whose positions it counts page after page.
template <int kType, int DP, bool kOne, int kWaves, bool kList>
__global__ void __launch_bounds__(64 * kWaves, (kWaves == 8 ? 1 : Few<kType, DP>::kGroups))
    attn_few_kernel(AttnArgs a) {
  typedef Few<kType, DP> T;
  constexpr int kKeys = T::kKeys, kRuns = T::kRuns, kVs = T::kN / kRuns;
  typedef KvTile<DP> L;
  typedef Rows<kType, kQ, DP, kKeys> R;
  extern __shared__ __attribute__((aligned(16))) uint8_t smem[];
  __shared__ uint32_t again;
  __shared__ int counts[kWaves];
  static_assert(kOne || !kList, "selected pages have kRun positions or more");
  SeenPage* const list = reinterpret_cast<SeenPage*>(smem + kWaves * T::kWave);
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int KV = a.c.kv_heads, G = a.group, D = a.c.head_dim;
  // The kv head goes fastest and the range slowest: the last ranges, which the shorter
  // sequences do not have, come last.
  const int units = kList ? a.b.tokens : a.b.batch;
  const int g = blockIdx.x % KV, split = blockIdx.x / KV / units;
  const int unit = blockIdx.x / KV % units, b = kList ? find_seq(a.b, unit, 0, 0) : unit;
  if (kList && (b < 0 || b >= a.b.batch)) return;
  const Seq sq = seq_of(a.b, b);
  const int ti0 = kList ? unit - sq.first : 0;  // (the token in its sequence)
  if (kList && (ti0 < 0 || ti0 >= sq.n)) return;  // (cu_q that does not ascend)
  const int rows = kList ? G : sq.n * G;
  if (!kList && rows > a.few) return;
  const bool past = too_long(a, sq);
  const int col = lane % kQ;
  uint8_t* const vbuf = smem + wave * T::kWave;
  float* const ks = reinterpret_cast<float*>(vbuf + T::kBufs * T::kBytes);
  float* const vs = ks + kKeys;

  const int mask = (1 << a.c.page_shift) - 1, item = kType == kKvFp16 ? 2 : 1;
  const uint8_t* const kg = (const uint8_t*)a.c.k + ((size_t)g << a.c.page_shift) * D * item;
  const uint8_t* const vg = (const uint8_t*)a.c.v + ((size_t)g << a.c.page_shift) * D * item;
  // 8-bit keys of head_dim % 16 = 0 are read 16 codes at a time.
  const bool pairs = kType == kKvInt8 && D % 16 == 0;
  // A lane's columns of a K row, and its rows and columns of 16 V rows (those past D: the
  // row's first, whose products are with zeros or not used).
  int kcol[R::kSteps], vrow[kVs], vcol[kVs];
#pragma unroll
  for (int s = 0; s < R::kSteps; s++) {
    const int d = pairs ? R::template element<true>(s) : R::template element<false>(s);
    kcol[s] = d < D ? d : 0;
  }
#pragma unroll
  for (int i = 0; i < kVs; i++) {
    vrow[i] = (i * 64 + lane) / L::kCh;
    const int c = 8 * (((i * 64 + lane) % L::kCh) ^ L::swz(vrow[i]));
    vcol[i] = c < D ? c : 0;
  }

  int seen = 0;  // positions of the pages in `list`
  if (kList && !past) {
    const int* const selected = a.selected + ((size_t)unit * KV + g) * a.count;
    seen = seen_pages(a, b, sq.kv - sq.n + ti0, selected, list, counts) << a.c.page_shift;
  }
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
    // Pages of the next tile's keys: kOne: of its runs; else the lane's.
    int pid[kRuns] = {};
    int now[kRuns] = {}, then[kRuns] = {};  // kList: positions of the runs that are seen
    half8 kf[kRuns][R::kSteps];     // K of the next tile: keys 16 i + col, columns kcol
    uint2 kc[kRuns][R::kSteps], vc[T::kN];  // 8-bit: its codes, and V's
    float kss = 0.0f, vss = 0.0f;
    auto look_up = [&](int p0) __attribute__((always_inline)) {
      if (kList) {
      } else if (kOne) {
#pragma unroll
        for (int i = 0; i < kRuns; i++)
          pid[i] = load_const<int>(a.b.page_table + (size_t)b * a.b.width +
                                   (min(p0 + kRun * i, hi - 1) >> a.c.page_shift));
      } else {
        pid[0] = page_id(a, b, min(p0 + lane % kKeys, hi - 1));
      }
    };
    auto issue = [&](int p0, int buf) __attribute__((always_inline)) {
      int pg[kRuns] = {}, slot0[kRuns], last0[kRuns];
#pragma unroll
      for (int i = 0; i < kRuns; i++) {
        // (kOne: a run past the end is the last one again, rows past it the last row)
        int start = min(p0 + kRun * i, (hi - 1) & -kRun), last = hi - 1 - start;
        if (kList) {
          const SeenRun run = seen_run(a, list, start);
          pid[i] = run.page, slot0[i] = start = run.slot, last0[i] = last = run.last;
          then[i] = p0 + kRun * i < hi ? run.seen : 0;
        }
        if (kOne) pg[i] = __builtin_amdgcn_readfirstlane(page_of(a, pid[i], bad));
        {
          const uint8_t* src;
          uint32_t off;
          if (kOne) {
            src = kg + ((size_t)pg[i] * a.c.k_page + (uint32_t)((start & mask) * D)) * item;
            off = __umul24(min(col, last), D) * item;
          } else {
            src = kg + (size_t)page_of(a, __shfl(pid[0], kQ * i + col, 64), bad) * a.c.k_page *
                           item;
            off = __umul24(min(p0 + kQ * i + col, hi - 1) & mask, D) * item;
          }
          if (kType == kKvFp16) {
#pragma unroll
            for (int s = 0; s < R::kSteps; s++)
              kf[i][s] = load_global<half8>(src + (off + kcol[s] * 2));
          } else if (pairs) {
#pragma unroll
            for (int s = 0; s < R::kSteps; s += 2) {
              if (s + 1 < R::kSteps) {
                const u32x4a8 c = load_global<u32x4a8>(src + (off + kcol[s]));
                kc[i][s] = make_uint2(c[0], c[1]);
                kc[i][s + 1] = make_uint2(c[2], c[3]);
              } else {
                kc[i][s] = load_global<uint2>(src + (off + kcol[s]));
              }
            }
          } else {
#pragma unroll
            for (int s = 0; s < R::kSteps; s++)
              kc[i][s] = load_global<uint2>(src + (off + kcol[s]));
          }
        }
        uint8_t* const dst = vbuf + buf * T::kBytes + i * (T::kBytes / kRuns);
        const uint8_t* vp =
            vg + ((size_t)pg[i] * a.c.v_page + (uint32_t)((start & mask) * D)) * item;
#pragma unroll
        for (int j = 0; j < kVs; j++) {
          uint32_t off = (__umul24(min(vrow[j], last), D) + vcol[j]) * item;
          if (!kOne) {
            const int r = kQ * i + vrow[j];
            vp = vg + (size_t)page_of(a, __shfl(pid[0], r, 64), bad) * a.c.v_page * item;
            off = (__umul24(min(p0 + r, hi - 1) & mask, D) + vcol[j]) * item;
          }
          if (kType == kKvInt8)
            vc[i * kVs + j] = load_global<uint2>(vp + off);
          else if (kOne)
            // (non-temporal; K is not, as each line of it is read by several loads: the 64
            // sequences take 230 us with neither, 217 with both, 211 so; one token over
            // 131072 positions 98, 88 and 88)
            dma16<true>(vp, off, dst + j * 1024);
          else
            dma16(vp + off, dst + j * 1024);
        }
      }
      if (kType == kKvInt8) {
        int page = kOne ? pg[0] : page_of(a, pid[0], bad);
        if (kOne) {
#pragma unroll
          for (int i = 1; i < kRuns; i++) page = lane % kKeys / kRun == i ? pg[i] : page;
        }
        int slot = min(p0 + lane % kKeys, hi - 1) & mask;
        if (kList) {
          slot = slot0[0] + min(lane % kRun, last0[0]);
#pragma unroll
          for (int i = 1; i < kRuns; i++)
            slot = lane % kKeys / kRun == i ? slot0[i] + min(lane % kRun, last0[i]) : slot;
        }
        const size_t tok = ((size_t)g << a.c.page_shift) + slot;
        kss = load_global<float>(a.c.k_scale + (size_t)page * a.c.ks_page + tok);
        vss = load_global<float>(a.c.v_scale + (size_t)page * a.c.vs_page + tok);
      }
    };

    const int step = kWaves * kKeys;
    if (lo + wave * kKeys < hi) {
      look_up(lo + wave * kKeys);
      issue(lo + wave * kKeys, 0);
      look_up(lo + wave * kKeys + step);
    }
    R x;
    x.init(r0 + col < rows ? a.q + (size_t)t * a.q_stride + (size_t)h * D : nullptr, D, a.scale, pairs);
    int buf = 0;
    for (int p0 = lo + wave * kKeys; p0 < hi; p0 += step, buf ^= T::kBufs - 1) {
      typename R::acc s[kRuns];
      auto next = [&]() __attribute__((always_inline)) {
        if (p0 + step < hi) {
          issue(p0 + step, buf ^ (T::kBufs - 1));
          look_up(p0 + 2 * step);
        }
      };
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
#pragma unroll
      for (int i = 0; i < kRuns; i++) now[i] = then[i];
      if (kType == kKvFp16) {
        half8 k[kRuns][R::kSteps];
#pragma unroll
        for (int i = 0; i < kRuns; i++)
#pragma unroll
          for (int st = 0; st < R::kSteps; st++) k[i][st] = kf[i][st];
        next();
        x.scores(s, [&](int i, int st) __attribute__((always_inline)) { return k[i][st]; });
      } else {
        // (the next tile's codes come into the registers of this one's: with a third of
        // the registers less, three work-groups a CU and not two)
#pragma unroll
        for (int i = 0; i < T::kN; i++)
          *reinterpret_cast<u32x4*>(vbuf + (i * 64 + lane) * 16) = codes_to_bf16(vc[i]);
        ks[lane % kKeys] = kss;
        vs[lane % kKeys] = vss;
        x.scores(s, [&](int i, int st) __attribute__((always_inline)) {
          return f16x8(codes_to_f16(kc[i][st]));
        });
        next();
      }
      if (kList) {
        if (now[0] < kRun || now[1] < kRun)
          x.template maximum<2>(s, now[0], now[1], ks);
        else
          x.template maximum<0>(s, 0, 0, ks);
      } else if (p0 < all_lo || p0 + kKeys - 1 > all_hi) {
        x.template maximum<1>(s, seen_lo - p0, seen_hi - p0, ks);
      } else {
        x.template maximum<0>(s, 0, 0, ks);
      }
      x.values(s, vbuf + buf * T::kBytes, vs);
    }
    x.finish(__any(bad));

    few_store<DP, kWaves, T::kWave, kQ, kList>(a, sq, g, ti0, r0, rows, split, past, x, smem, again);
  }
}

template <int kType, int DP, bool kOne, int kWaves, bool kList = false>
hipError_t launch(const AttnArgs& a, hipStream_t s) {
  const int lds = kWaves * Few<kType, DP>::kWave + (kList ? a.count * (int)sizeof(SeenPage) : 0);
  const size_t units = kList ? a.b.tokens : a.b.batch;
  const size_t grid = units * a.c.kv_heads * a.fs.splits;
  if (grid > 0xFFFFFF) return hipErrorInvalidValue;
  const void* kernel = (const void*)attn_few_kernel<kType, DP, kOne, kWaves, kList>;
  const hipError_t e = set_lds_limit(kernel, lds);
  if (e != hipSuccess) return e;
  attn_few_kernel<kType, DP, kOne, kWaves, kList><<<(unsigned)grid, 64 * kWaves, lds, s>>>(a);
  return hipGetLastError();
}

template <int kType, int DP>
hipError_t run(const AttnArgs& a, hipStream_t s) {
  const bool one = a.c.page_shift >= kRunShift;
  if (a.selected) {
    if constexpr (DP <= 128) {
      if (a.few_waves == 8) return launch<kType, DP, true, 8, true>(a, s);
    }
    return launch<kType, DP, true, 4, true>(a, s);
  }
  if constexpr (DP <= 128) {
    if (a.few_waves == 8)
      return one ? launch<kType, DP, true, 8>(a, s) : launch<kType, DP, false, 8>(a, s);
  }
  return one ? launch<kType, DP, true, 4>(a, s) : launch<kType, DP, false, 4>(a, s);
}

}  // namespace

hipError_t launch_attn_few(const AttnArgs& a, hipStream_t s) {
  const int D = a.c.head_dim;
  if (a.c.dtype == kKvFp4) return launch_attn_few4(a, s);
  if (a.c.dtype == kKvFp16)
    return D <= 64    ? run<kKvFp16, 64>(a, s)
           : D <= 96  ? run<kKvFp16, 96>(a, s)
           : D <= 128 ? run<kKvFp16, 128>(a, s)
                      : run<kKvFp16, 256>(a, s);
  return D <= 64    ? run<kKvInt8, 64>(a, s)
         : D <= 96  ? run<kKvInt8, 96>(a, s)
         : D <= 128 ? run<kKvInt8, 128>(a, s)
                    : run<kKvInt8, 256>(a, s);
}

}  // namespace hypno
