// Attention for sequences with many rows (prompts, chunks of them): a work-group
// takes 4 NQ rows of one kv head, NQ a wave, and runs through their positions in
// tiles of BK keys that all four waves read from LDS.
//
// Bound: the matrix cores, at the clock that power leaves them.  Each product goes in
// twice (the two parts of q and of the weights), so that 8192 tokens of 32/8 heads of 128
// (0.55 PFLOP) issue 1.1 PFLOP: 0.94 ms, 1.17 PFLOP/s, where nothing but these MFMAs on
// random data reaches 1.6 (2.46 on zeros: the clock falls) and a large fp16 product of
// the library 1.3.  MFMAs are busy 67% of the cycles, at 1.6 GHz.
//  * 32 rows a wave (32x32x16 MFMA): each piece of K or V that it reads from LDS feeds
//    two MFMAs, and without these reads the whole takes 5% less; 64 rows would need 512
//    registers.  With head_dim above 128, 16 rows: 32 need the registers of two waves for
//    o and q alone.
//  * Tiles of 64 keys twice in LDS (64 KB with head_dim 128): two work-groups a CU, and
//    one's softmax runs beside the other's products.
//  * Rows of one kv head from all of its query heads: K and V are read once for the group,
//    and a causal tile ends after 128 / group tokens.
//  * Work-groups of one kv head share an XCD's L2 (see the order in the kernel).
//  * 4-bit codes become fp16 values on their way into LDS, 64 vector operations a tile for a
//    thread's 32 keys and 32 values: 512 tokens over 16384 266 us, of fp16 ones 254.
// A prompt of 2048: 80 us; its longest work-group's 32 tiles one after the other are 60
// of it, the last of them alone on a CU whose short work-group has ended.  512 tokens over
// 16384: 258 us, 15 of them to join four ranges.

#include <type_traits>

#include "attention.hpp"

namespace hypno {

namespace {

template <int kType, int NQ, int DP, int BK>
struct Tile {
  static constexpr int kRows = 4 * NQ;
  static constexpr int kBytes = BK * DP * 2;          // K or V of one tile
  static constexpr int kN = BK * DP / 8 / 256;        // 16-byte pieces of it a thread
  // 4-bit: groups of 32 codes, 16 bytes, of a wave's BK / 4 rows, and of them a lane.
  static constexpr int kG = BK / 4 * DP / kFp4Group, kNg = (kG + 63) / 64;
  // K and V twice; 8-bit: their scales twice.
  static constexpr int kLds = 4 * kBytes + (kType == kKvInt8 ? 4 * BK * 4 : 0);
};

// kOne: pages have kRun positions or more.
template <int kType, int NQ, int DP, int BK, bool kOne>
__global__ void __launch_bounds__(256, 2) attn_tile_kernel(AttnArgs a) {
  typedef Tile<kType, NQ, DP, BK> T;
  typedef KvTile<DP> L;
  extern __shared__ __attribute__((aligned(16))) uint8_t smem[];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int KV = a.c.kv_heads, G = a.group, D = a.c.head_dim;
  // The kv head goes fastest (work-groups of one head on one XCD, where it has eight),
  // the rows with the most positions first.  Where all work-groups run at once, two a
  // CU, the second half goes up again: a long one beside a short one.
  const int g = blockIdx.x % KV, all = gridDim.x / KV, half = a.cus / KV;
  int at = blockIdx.x / KV;
  if (all - a.b.batch * a.ts.splits <= 2 * half && at >= half) at = all - 1 - (at - half);
  const int split = at % a.ts.splits, slot = (all - 1 - at) / a.ts.splits;
  const int b = find_seq(a.b, slot, G, T::kRows);
  if (b < 0 || b >= a.b.batch) return;
  const Seq sq = seq_of(a.b, b);
  const int rows = sq.n * G;
  const int r0 = (slot - ((int)((int64_t)sq.first * G / T::kRows) + b)) * T::kRows;
  if (r0 < 0 || r0 >= rows || rows <= a.few) return;
  const int r1 = min(r0 + T::kRows, rows);
  const bool past = too_long(a, sq);
  const Span span = span_of(a, sq, r0, r1);
  int lo = past ? 0 : span.lo, hi = past ? 0 : span.hi;
  if (a.ts.splits > 1) {
    const int64_t start = lo + (int64_t)split * a.ts.chunk;
    if (start >= hi && split) return;
    if (split + 1 < a.ts.splits) hi = (int)min((int64_t)hi, start + a.ts.chunk);
    lo = (int)start;
  }

  // This wave's rows: lane % NQ of it, and the positions that it sees.
  typedef Rows<kType == kKvInt8 ? kKvInt8 : kKvFp16, NQ, DP, BK> R;
  const int w0 = r0 + wave * NQ, row = w0 + lane % NQ;
  const bool live = row < rows;
  const int ti = min(row, rows - 1) / G, h = g * G + min(row, rows - 1) % G;
  const int t = sq.first + ti;
  const int seen_lo = first_seen(a, sq, ti), seen_hi = min(sq.kv - sq.n + ti, hi - 1);
  // of the wave's rows: the first and last position that any sees, those that all see
  const int last = min(w0 + NQ, rows) - 1;
  const bool some = w0 < rows;
  const int any_lo = some ? first_seen(a, sq, w0 / G) : 0;
  const int any_hi = some ? min(sq.kv - sq.n + last / G, hi - 1) : -1;
  const int all_lo = some ? first_seen(a, sq, last / G) : 0;
  const int all_hi = some ? min(sq.kv - sq.n + w0 / G, hi - 1) : -1;
  bool bad = false;
  uint8_t* const kbuf = smem;
  uint8_t* const vbuf = smem + 2 * T::kBytes;
  float* const scales = reinterpret_cast<float*>(smem + 4 * T::kBytes);
  // Wave w brings rows BK / 4 w and on of a tile, 16-byte piece by piece.  With
  // kOne these lie in one page, `id`; otherwise each piece's page is in `ids`.
  // (Rows past the end: the last row again, whose weights are 0.)
  constexpr int kMine = BK / 4;
  const int mask = (1 << a.c.page_shift) - 1, item = kType == kKvFp16 ? 2 : 1;
  static_assert(kType != kKvFp4 || kOne, "4-bit pages have kRun positions or more");
  int id = 0, ids[T::kN];  // (with `ids`, id: of the lane's scale)
  uint2 kr[T::kN], vr[T::kN];   // 8-bit codes on their way
  u32x4 kr4[T::kNg], vr4[T::kNg];  // 4-bit: codes and scales on their way
  _Float16 ks4[T::kNg], vs4[T::kNg];
  float sr = 0.0f;
  const int srow = wave * kMine + lane % kMine;
  const bool sk = lane < kMine;
  int rr[T::kN], ch[T::kN];
#pragma unroll
  for (int i = 0; i < T::kN; i++) {
    const int j = (wave * T::kN + i) * 64 + lane;
    rr[i] = j / L::kCh;
    ch[i] = 8 * ((j % L::kCh) ^ L::swz(rr[i]));
    if (ch[i] >= D) ch[i] = 0;  // (columns past D: products with zeros, outputs not used)
  }
  // 4-bit: the row of a wave's group j.  Rows four apart follow each other, as their pieces
  // then lie in different banks when they are stored.
  auto group_row = [&](int j) __attribute__((always_inline)) {
    const int r = j / (DP / kFp4Group);
    return r % (kMine / 4) * 4 + r / (kMine / 4);
  };
  auto look_up = [&](int p0) __attribute__((always_inline)) {
    if (kOne) {
      id = load_const<int>(a.b.page_table + (size_t)b * a.b.width +
                            (min(p0 + wave * kMine, hi - 1) >> a.c.page_shift));
    } else {
#pragma unroll
      for (int i = 0; i < T::kN; i++) ids[i] = page_id(a, b, min(p0 + rr[i], hi - 1));
      if (kType == kKvInt8) id = page_id(a, b, min(p0 + srow, hi - 1));
    }
  };
  const uint8_t* const kg = (const uint8_t*)a.c.k + ((size_t)g << a.c.page_shift) * D * item;
  const uint8_t* const vg = (const uint8_t*)a.c.v + ((size_t)g << a.c.page_shift) * D * item;
  const float* const ksg = a.c.k_scale + ((size_t)g << a.c.page_shift);
  const float* const vsg = a.c.v_scale + ((size_t)g << a.c.page_shift);
  auto issue = [&](int p0, int buf) __attribute__((always_inline)) {
    if constexpr (kType == kKvFp4) {
      const int pg = __builtin_amdgcn_readfirstlane(page_of(a, id, bad)), B = D / kFp4Group;
      const uint8_t* const kp =
          (const uint8_t*)a.c.k + (size_t)pg * a.c.k_page + (((size_t)g << a.c.page_shift) * D >> 1);
      const uint8_t* const vp =
          (const uint8_t*)a.c.v + (size_t)pg * a.c.v_page + (((size_t)g << a.c.page_shift) * D >> 1);
      const _Float16* const ksp = (const _Float16*)a.c.k_scale + (size_t)pg * a.c.ks_page +
                                  ((size_t)(g * B) << a.c.page_shift);
      const _Float16* const vsp = (const _Float16*)a.c.v_scale + (size_t)pg * a.c.vs_page +
                                  ((size_t)(g * B) << a.c.page_shift);
#pragma unroll
      for (int i = 0; i < T::kNg; i++) {
        // (lanes past the groups, and groups past D: the row's first)
        const int j = min(i * 64 + lane, T::kG - 1), blk = j % (DP / kFp4Group);
        const int tok = min(p0 + wave * kMine + group_row(j), hi - 1) & mask;
        const int at = blk < B ? blk : 0;
        const uint32_t off = __umul24(tok, D / 2) + at * 16, so = (at << a.c.page_shift) + tok;
        kr4[i] = load_global<u32x4>(kp + off);
        vr4[i] = load_global<u32x4>(vp + off);
        ks4[i] = load_global<_Float16>(ksp + so);
        vs4[i] = load_global<_Float16>(vsp + so);
      }
      return;
    }
    const int page = kType == kKvInt8 || kOne ? page_of(a, id, bad) : 0;
    uint32_t off[T::kN];
#pragma unroll
    for (int i = 0; i < T::kN; i++)
      off[i] = (__umul24(min(p0 + rr[i], hi - 1) & mask, D) + ch[i]) * item;
    uint8_t* const kd = kbuf + buf * T::kBytes + wave * T::kN * 1024;
    uint8_t* const vd = kd + 2 * T::kBytes;
    if (kOne) {
      const int pg = __builtin_amdgcn_readfirstlane(page);
      const uint8_t* const kp = kg + (size_t)pg * a.c.k_page * item;
      const uint8_t* const vp = vg + (size_t)pg * a.c.v_page * item;
#pragma unroll
      for (int i = 0; i < T::kN; i++) {
        if (kType == kKvFp16) {
          dma16(kp, off[i], kd + i * 1024);
          dma16(vp, off[i], vd + i * 1024);
        } else {
          kr[i] = load_global<uint2>(kp + off[i]);
          vr[i] = load_global<uint2>(vp + off[i]);
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < T::kN; i++) {
        const int pg = page_of(a, ids[i], bad);
        const uint8_t* const kp = kg + (size_t)pg * a.c.k_page * item + off[i];
        const uint8_t* const vp = vg + (size_t)pg * a.c.v_page * item + off[i];
        if (kType == kKvFp16) {
          dma16(kp, kd + i * 1024);
          dma16(vp, vd + i * 1024);
        } else {
          kr[i] = load_global<uint2>(kp);
          vr[i] = load_global<uint2>(vp);
        }
      }
    }
    if (kType == kKvInt8 && lane < 2 * kMine) {
      const int tok = min(p0 + srow, hi - 1) & mask;
      sr = load_global<float>((sk ? ksg + (size_t)page * a.c.ks_page
                                  : vsg + (size_t)page * a.c.vs_page) + tok);
    }
  };
  auto store = [&](int buf) __attribute__((always_inline)) {  // codes: what `issue` loaded
    if constexpr (kType == kKvFp4) {
#pragma unroll
      for (int i = 0; i < T::kNg; i++) {
        const int j = i * 64 + lane, blk = j % (DP / kFp4Group);
        if (T::kG % 64 && j >= T::kG) continue;
        const int r = wave * kMine + group_row(j);
        const half2v ks = {ks4[i], ks4[i]}, vs = {vs4[i], vs4[i]};
#pragma unroll
        for (int c = 0; c < 4; c++) {
          const int at = L::at(r, 4 * blk + c) + buf * T::kBytes;
          *reinterpret_cast<u32x4*>(kbuf + at) = fp4_to_f16(kr4[i][c], ks);
          *reinterpret_cast<u32x4*>(vbuf + at) = fp4_to_f16(vr4[i][c], vs);
        }
      }
      return;
    }
#pragma unroll
    for (int i = 0; i < T::kN; i++) {
      const int at = ((wave * T::kN + i) * 64 + lane) * 16 + buf * T::kBytes;
      *reinterpret_cast<u32x4*>(kbuf + at) = codes_to_f16(kr[i]);
      *reinterpret_cast<u32x4*>(vbuf + at) = codes_to_bf16(vr[i]);
    }
    if (lane < 2 * kMine) scales[(buf * 2 + !sk) * BK + srow] = sr;
  };

  // fp16: tile i + 1 is copied into LDS while tile i is worked on.  Codes: tile i + 1 is
  // stored there (its codes came in during tile i - 1) and the loads of i + 2 begin.
  constexpr int kAhead = kType == kKvFp16 ? 1 : 2;
  const int tiles = (hi - lo + BK - 1) / BK;
  if (tiles > 0) {
    look_up(lo);
    issue(lo, 0);
    if (kType != kKvFp16) {
      store(0);
      look_up(lo + BK);
      if (tiles > 1) issue(lo + BK, 1);
    }
    look_up(lo + kAhead * BK);
  }
  R x;
  x.init(live ? a.q + (size_t)t * a.q_stride + (size_t)h * D : nullptr, D, a.scale);
  if (kType == kKvFp16)
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
  else
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
  // Tiles that all of the wave's rows see whole need no mask; each wave goes through
  // its own runs of the two kinds, tile by tile with the others.
  auto step = [&](auto masked, int i) __attribute__((always_inline)) {
    const int p0 = lo + i * BK, buf = i & 1;
    if (kType != kKvFp16 && i + 1 < tiles) store(buf ^ 1);
    if (i + kAhead < tiles) {
      issue(p0 + kAhead * BK, buf ^ 1);
      look_up(p0 + (kAhead + 1) * BK);
    }
    if (!masked || (p0 <= any_hi && p0 + BK > any_lo)) {
      const uint8_t* kt = kbuf + buf * T::kBytes;
      typename R::acc s[BK / NQ];
      x.scores(s, [&](int kt_i, int st) __attribute__((always_inline)) {
        const int r = NQ * kt_i + lane % NQ;
        return *reinterpret_cast<const half8*>(kt + L::at(r, R::NG * st + lane / NQ));
      });
      const float* ks = scales + buf * 2 * BK;
      x.template maximum<masked ? 1 : 0>(s, seen_lo - p0, seen_hi - p0, ks);
      x.values(s, vbuf + buf * T::kBytes, ks + BK);
    }
    if (kType == kKvFp16)
      asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
    else
      asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
  };
  const int full0 = some ? min(max(all_lo - lo + BK - 1, 0) / BK, tiles) : tiles;
  const int full1 = some ? max(full0, min((all_hi + 1 - lo) / BK, tiles)) : tiles;
  for (int i = 0, run = 0; run < 2; run++) {
    if (run)
      for (; i < full1; i++) step(std::false_type(), i);
    for (const int end = run ? tiles : full0; i < end; i++) step(std::true_type(), i);
  }
  x.finish(__syncthreads_or(bad));

  const size_t orow = (size_t)t * a.heads + h;
  if (a.ts.splits > 1) {
    if (!live) return;
    const size_t part = orow * a.ts.splits + split;
    float* po = a.tp.o + part * D;
#pragma unroll
    for (int k = 0; k < R::kDt; k++)
#pragma unroll
      for (int i = 0; i < R::kAcc; i += 4) {
        const int d = R::dim(k, i);
        if (d < D)
          *reinterpret_cast<f32x4*>(po + d) =
              f32x4{x.o[k][i], x.o[k][i + 1], x.o[k][i + 2], x.o[k][i + 3]};
      }
    if (lane < NQ) a.tp.ml[part] = make_float2(x.m, x.l);
    return;
  }
  const float inv = x.l == 0.0f ? 0.0f : 1.0f / x.l;
  float z = x.l * 0.0f;
#pragma unroll
  for (int k = 0; k < R::kDt; k++)
#pragma unroll
    for (int i = 0; i < R::kAcc; i += 4) {
      const int d = R::dim(k, i);
      f32x4 v;
#pragma unroll
      for (int j = 0; j < 4; j++) {
        z += x.o[k][i + j] * 0.0f;
        v[j] = x.o[k][i + j] * inv;
      }
      if (live && d < D) *reinterpret_cast<f32x4*>(a.out + orow * D + d) = v;
    }
  uint64_t again = __ballot(live && (!(z == 0.0f) || past));
  again |= again >> 32;
  if (NQ == 16) again |= again >> 16;
  // (the stores above, by other lanes, come first)
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  attn_rows(a, sq, g, w0, again & ((1ull << NQ) - 1));
}

template <int kType, int NQ, int DP, int BK, bool kOne>
hipError_t launch(const AttnArgs& a, hipStream_t s) {
  typedef Tile<kType, NQ, DP, BK> T;
  const size_t slots = (size_t)a.b.tokens * a.group / T::kRows + a.b.batch;
  const size_t grid = slots * a.c.kv_heads * a.ts.splits;
  if (grid > 0xFFFFFF) return hipErrorInvalidValue;
  const hipError_t e = set_lds_limit((const void*)attn_tile_kernel<kType, NQ, DP, BK, kOne>, T::kLds);
  if (e != hipSuccess) return e;
  attn_tile_kernel<kType, NQ, DP, BK, kOne><<<(unsigned)grid, 256, T::kLds, s>>>(a);
  return hipGetLastError();
}

template <int kType, int NQ, int DP, int BK>
hipError_t run(const AttnArgs& a, hipStream_t s) {
  return a.c.page_shift >= kRunShift ? launch<kType, NQ, DP, BK, true>(a, s)
                                     : launch<kType, NQ, DP, BK, false>(a, s);
}

}  // namespace

hipError_t launch_attn_tile(const AttnArgs& a, hipStream_t s) {
  const int D = a.c.head_dim;
  if (a.c.dtype == kKvFp4)
    return D <= 64    ? launch<kKvFp4, 32, 64, 64, true>(a, s)
           : D <= 96  ? launch<kKvFp4, 32, 96, 64, true>(a, s)
           : D <= 128 ? launch<kKvFp4, 32, 128, 64, true>(a, s)
                      : launch<kKvFp4, 16, 256, 32, true>(a, s);
  if (a.c.dtype == kKvFp16)
    return D <= 64    ? run<kKvFp16, 32, 64, 64>(a, s)
           : D <= 96  ? run<kKvFp16, 32, 96, 64>(a, s)
           : D <= 128 ? run<kKvFp16, 32, 128, 64>(a, s)
                      : run<kKvFp16, 16, 256, 32>(a, s);
  return D <= 64    ? run<kKvInt8, 32, 64, 64>(a, s)
         : D <= 96  ? run<kKvInt8, 32, 96, 64>(a, s)
         : D <= 128 ? run<kKvInt8, 32, 128, 64>(a, s)
                    : run<kKvInt8, 16, 256, 32>(a, s);
}

}  // namespace hypno
