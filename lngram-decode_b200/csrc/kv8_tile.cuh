// Attention of many rows over the 8-bit cache on the tensor cores: prompts, chunks of prompts, batches of drafts.
//
// kv_tile_kernel's plan (kv_tile.cuh): units of two row tiles of 128 rows against tiles of 64 keys, persistent CTAs, S and P
// and O in TMEM, one row a thread, a warp a row tile that issues its products.  Products are fp16 -- both operands of
// one are of one type, and e4m3 is exact in fp16 -- so between the copies and the products stand
//   warps 12-15  which turn a tile's bytes into the fp16 operand, 16 bytes a step (every eight lanes read and write
//             eight different banks), clear values that no row sees, and bring a unit's queries in: scaled by a power
//             of two a row, as kv8_step_kernel does, and rounded by that to nothing but what lies 2^-39 below the row's
//             largest value (fp16 queries are taken as they are).
// Bytes come through a ring of their own, half as large a tile as the fp16 one.  Exponents go the way of kv8_step.cuh: the
// keys' into the factor of their scores (8 columns at a time, a page's least), the values' into the exponential and
// back out of the sum, and a row's reference lies below its largest score as there.  Weights are rounded to fp16 once, their sum
// is not.
//
// Measured: two prompts of 5001 and 8000 tokens, 28 query and 4 key heads of 128, window of 4096 and 4 sinks: 830 to 865 us by the
// box, 815 to 850 TFLOP/s, about what kv_tile_kernel takes in 16 bits; a key tile takes some 1800 cycles, of which a row's
// thread is busy for 1400 and waits for its scores in the others.  The converters want all four warps on one tile and 96
// registers (two warps for keys and two for values: 5 % more; 88 or 104 registers: 2 %).  64 sequences of 16 drafted tokens
// after 1024 keys, 4 key heads of 64: 50 us (42 us in 16 bits), two waves of units of which one row tile has rows (both row
// tiles on the same rows, the key tiles in turn, their states joined: 62 us).
#pragma once

#include "kv8_step.cuh"
#include "kv_tile.cuh"

namespace lng {

constexpr int K8T_THREADS = 512, K8T_EXPS = 16;  // exponents of so many tiles are kept

template <int HDP>
struct K8tCfg {
  static constexpr uint32_t Q_BYTES = 128 * HDP * 2, Q_HALF = 128 * 128;        // a row tile of queries; 64 columns of it
  static constexpr uint32_t KV_BYTES = KT_BK * HDP * 2, KV_HALF = KT_BK * 128;  // a tile of keys or values in fp16
  static constexpr uint32_t RAW_BYTES = KT_BK * HDP;                            // and as it comes
  static constexpr int SLOTS = HDP == 128 ? 4 : 8, RAW_SLOTS = HDP == 128 ? 6 : 12;
  static constexpr uint32_t TMEM_S = 0, TMEM_O = 256, TMEM_COLS = 512;
  static constexpr uint32_t RING = 2 * Q_BYTES, RAW = RING + SLOTS * KV_BYTES, STAGE = RAW + RAW_SLOTS * RAW_BYTES;
  static constexpr uint32_t EXPS = STAGE + 8 * 4096, SCALES = EXPS + K8T_EXPS * 96, BARS = SCALES + 2 * 256 * 4;
  static constexpr size_t SMEM = BARS + 512 + 1024;
};

struct K8tParams {
  KtParams t;
  KvRows q;
  const int8_t *k_exp, *v_exp;
  int64_t k_exp_page, v_exp_page;
};

// As KtBars, whose names kt_multiply uses: kv_* of the fp16 ring.
template <int HDP>
struct K8tBars {
  static constexpr uint32_t NS = K8tCfg<HDP>::SLOTS, NR = K8tCfg<HDP>::RAW_SLOTS;
  static constexpr uint32_t kv_full = 0, kv_empty = 8 * NS;      // [NS] each; full: four warps, empty: two row tiles
  static constexpr uint32_t raw_full = 16 * NS, raw_empty = raw_full + 8 * NR;  // [NR] each; empty: four warps
  static constexpr uint32_t q_full = raw_empty + 8 * NR, q_empty = q_full + 8;
  static constexpr uint32_t s_full = q_empty + 8, p_full = s_full + 32, pv_done = p_full + 32, o_full = pv_done + 16, idle = o_full + 16;
  static constexpr uint32_t tmem = idle + 16, abort = tmem + 4;
};
static_assert(K8tBars<64>::abort + 4 <= 512 && K8tBars<128>::abort + 4 <= 512, "barriers outgrow their place");

// Two warps, one for keys (and the exponents of both, which the scores' readers need), one for values: every tile's bytes into
// the raw ring, page by page.  A page and then its exponents are looked up for so many tiles at once as the lanes have pieces for: two
// look-ups a tile in a row took longer than the tile's products.  (Exponents of sixteen tiles: a raw slot is given out again when the tile three
// or six before it has been converted, which is behind the products of the tile five or ten before it.)
template <int HDP>
__device__ __forceinline__ void k8t_load(const CUtensorMap* map, const K8tParams& pp, uint32_t bars, uint32_t raw, uint32_t exps,
                                         const uint32_t kv) {
  using Cfg = K8tCfg<HDP>;
  using B = K8tBars<HDP>;
  constexpr uint32_t NR = Cfg::RAW_SLOTS;
  const KtParams& p = pp.t;
  const KvView& c = p.c;
  const int lane = threadIdx.x & 31, box = p.box, boxes = KT_BK / box;
  const int32_t page_mask = (1 << c.page_shift) - 1;
  uint32_t it = kv;
  bool ok = true, there;
  KtWalk walk{};
  KtWork w;
  while (ok && kt_next(p, walk, w, there)) {
    if (!there || w.n == 0) continue;
    const int32_t* row = c.table + w.b * c.table_stride;
    // the unit's next tiles, as many as give every lane a piece: its page (-1: no token sees a key of it) and exponents
    int32_t page = -1, exp_k = 0, exp_v = 0;
    auto look_up = [&](int32_t i) {
      page = -1;
      exp_k = exp_v = 0;
      if (i + lane / boxes >= w.n) return;
      const int32_t key = tile_index(w.tiles, w.j0 + i + lane / boxes) * KT_BK + (lane % boxes) * box;
      if (!any_needed(w.span, key, key + box)) return;
      page = page_of(row, key, c.page_shift, c.num_pages);
      if (page >= 0) {
        if (kv == 0) {
          exp_k = pp.k_exp[page * pp.k_exp_page + w.hk];
          exp_v = pp.v_exp[page * pp.v_exp_page + w.hk];
        }
      } else {
        kv_range_error();
        page = int32_t(c.num_pages);  // behind the last page: the copy fills zeros
      }
    };
#pragma unroll 1
    for (int32_t i = 0; i < w.n; ++i, it += 2) {
      const int lane0 = (i & (32 / boxes - 1)) * boxes;  // of the tile's first piece
      if (lane0 == 0) look_up(i);
      const int32_t slot0 = uniform((tile_index(w.tiles, w.j0 + i) * KT_BK) & page_mask);
      const uint32_t bytes = uint32_t(__popc((__ballot_sync(0xffffffffu, page >= 0) >> lane0) & ((1u << boxes) - 1u))) * uint32_t(box * HDP);
      const uint32_t s = it % NR, bar = bars + B::raw_full + 8 * s, dst = raw + s * Cfg::RAW_BYTES;
      if (it >= NR) ok = __all_sync(0xffffffffu, kt_wait<B>(bars, B::raw_empty + 8 * s, (it / NR - 1) & 1));
      if (!ok) break;
      if (kv == 0) {  // [8] 2^(keys' exponent), [8] values' exponent, [8] 2^-(values' exponent): a number for 8 keys
        const int from = lane0 + ((lane & 7) * 8) / box;
        const int32_t ek = __shfl_sync(0xffffffffu, exp_k, from), ev = __shfl_sync(0xffffffffu, exp_v, from);
        const uint32_t at = exps + (it / 2 % K8T_EXPS) * 96 + (lane & 7) * 4;
        if (lane < 8) {
          sts32(at, __float_as_uint(exp2_whole(ek)));
          sts32(at + 32, __float_as_uint(float(ev)));
          sts32(at + 64, __float_as_uint(exp2_whole(-ev)));
        }
      }
      __syncwarp();
      if (elect_lane()) mbar_expect_at(bar, bytes);
      __syncwarp();
#pragma unroll 1
      for (int r = 0; r < boxes; r += 4) {
        int32_t pg[4];
#pragma unroll
        for (int x = 0; x < 4; ++x) pg[x] = __shfl_sync(0xffffffffu, page, (lane0 + r + x) & 31);
        if (elect_lane()) {
#pragma unroll
          for (int x = 0; x < 4; ++x)
            if (r + x < boxes && pg[x] >= 0) {
              const int32_t slot = (slot0 + (r + x) * box) & page_mask;
              tma_load_4d_at(dst + (r + x) * box * HDP, map, 0, slot, w.hk, pg[x], bar);
            }
        }
        __syncwarp();
      }
    }
  }
  // behind the last copies: they have been converted, or (where a role has given up) have at least landed
  const uint32_t k0 = it >= NR ? it - NR : kv;
  bool used = true;
  for (uint32_t k = k0; k < it; k += 2) used = kt_wait<B>(bars, B::raw_empty + 8 * (k % NR), (k / NR) & 1) && used;
  if (__all_sync(0xffffffffu, used)) return;
  for (uint32_t k = k0; k < it; k += 2) kt_wait<B, true>(bars, B::raw_full + 8 * (k % NR), (k / NR) & 1);
}

// Four warps: a unit's queries, then its tiles of keys and values, into the products' operands.
template <typename T, int HDP>
__device__ __forceinline__ void k8t_convert(const K8tParams& pp, uint32_t bars, uint32_t qs, uint32_t ring, uint32_t raw, uint32_t scales,
                                            int warp) {
  using Cfg = K8tCfg<HDP>;
  using B = K8tBars<HDP>;
  constexpr uint32_t NS = Cfg::SLOTS, NR = Cfg::RAW_SLOTS;
  constexpr int HALVES = HDP / 64, PIECES = HDP / 16;  // 16-byte pieces of a row as it comes
  const KtParams& p = pp.t;
  const int lane = threadIdx.x & 31, group_magic = (65535 + p.group) / p.group;  // r / group = r * magic >> 16 for r < 128
  uint32_t it = 0, units = 0;
  bool ok = true, there;
  KtWalk walk{};
  KtWork w;
  while (ok && kt_next(p, walk, w, there)) {
    if (!there || w.n == 0) continue;
    for (int G = 0; G < (w.tokens1 > 0 ? 2 : 1); ++G) {  // the queries' way from memory begins
      const int r = warp * 32 + lane, tok = (r * group_magic) >> 16;
      const T* src = static_cast<const T*>(pp.q.ptr) + (w.s.first + w.t0 + G * p.tile_tokens + tok) * pp.q.token +
                     int64_t(w.hk * p.group + r - tok * p.group) * pp.q.head;
      if (r < (G ? w.tokens1 : w.tokens0) * p.group)
        for (int x = 0; x < p.c.head_dim; x += 64) asm volatile("prefetch.global.L2 [%0];" ::"l"(src + x));
    }
    if (units > 0) ok = __all_sync(0xffffffffu, kt_wait<B>(bars, B::q_empty, (units - 1) & 1));
    if (!ok) break;
    // queries: eight lanes a row, four rows a step, the loads of as many steps in flight as 16 registers hold
    constexpr int STEPS_Q = 4 / HALVES;
    for (int G = 0; G < (w.tokens1 > 0 ? 2 : 1); ++G) {
      const int32_t rows = (G ? w.tokens1 : w.tokens0) * p.group;
      const int64_t token0 = w.s.first + w.t0 + G * p.tile_tokens;
      const T* const q0 = static_cast<const T*>(pp.q.ptr) + token0 * pp.q.token + int64_t(w.hk) * p.group * pp.q.head;
#pragma unroll 1
      for (int i0 = 0; i0 < 8; i0 += STEPS_Q) {
        const int chunk = lane & 7;
        uint4 x[STEPS_Q][HALVES];
#pragma unroll
        for (int i = 0; i < STEPS_Q; ++i) {
          const int r = warp * 32 + (i0 + i) * 4 + (lane >> 3), tok = (r * group_magic) >> 16;
          const T* src = q0 + tok * pp.q.token + (r - tok * p.group) * pp.q.head + chunk * 8;
#pragma unroll
          for (int hh = 0; hh < HALVES; ++hh)
            x[i][hh] = r < rows && hh * 64 + chunk * 8 < p.c.head_dim ? *reinterpret_cast<const uint4*>(src + hh * 64) : make_uint4(0, 0, 0, 0);
        }
#pragma unroll
        for (int i = 0; i < STEPS_Q; ++i) {
          const int r = warp * 32 + (i0 + i) * 4 + (lane >> 3);
          float down = 1.f, up = 1.f;
          if constexpr (!std::is_same<T, __half>::value) {
            uint32_t two = 0;  // the largest magnitudes, a pair
#pragma unroll
            for (int hh = 0; hh < HALVES; ++hh) {
              const uint32_t words[4] = {x[i][hh].x, x[i][hh].y, x[i][hh].z, x[i][hh].w};
#pragma unroll
              for (int y = 0; y < 4; ++y) {
                const uint32_t v = words[y] & 0x7fff7fffu;
                const __nv_bfloat162 m = __hmax2(*reinterpret_cast<const __nv_bfloat162*>(&two), *reinterpret_cast<const __nv_bfloat162*>(&v));
                two = *reinterpret_cast<const uint32_t*>(&m);
              }
            }
            float most = fmaxf(__uint_as_float(two << 16), __uint_as_float(two & 0xffff0000u));
#pragma unroll
            for (int o = 1; o < 8; o <<= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
            const int32_t e = k8_query_exponent(most);
            down = exp2_whole(-e);
            up = exp2_whole(e);
          }
          if (chunk == 0) sts32(scales + ((units & 1) * 256 + G * 128 + r) * 4, __float_as_uint(p.scale_log2 * up));
#pragma unroll
          for (int hh = 0; hh < HALVES; ++hh)
            sts128(qs + G * Cfg::Q_BYTES + hh * Cfg::Q_HALF + r * 128 + ((chunk ^ (r & 7)) << 4), k8_query<T>(x[i][hh].x, down),
                   k8_query<T>(x[i][hh].y, down), k8_query<T>(x[i][hh].z, down), k8_query<T>(x[i][hh].w, down));
        }
      }
    }
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    __syncwarp();
    if (elect_lane()) mbar_arrive_at(bars + B::q_full);
    __syncwarp();
    ++units;
#pragma unroll 1
    for (int32_t i = 0; i < 2 * w.n && ok; ++i, ++it) {
      const uint32_t rs = it % NR, hs = it % NS;
      const uint32_t from = raw + rs * Cfg::RAW_BYTES, to = ring + hs * Cfg::KV_BYTES;
      ok = kt_wait<B>(bars, B::raw_full + 8 * rs, (it / NR) & 1);
      if (it >= NS) ok = ok && kt_wait<B>(bars, B::kv_empty + 8 * hs, (it / NS - 1) & 1);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      const int32_t key0 = tile_index(w.tiles, w.j0 + (i >> 1)) * KT_BK;
      // values that no row sees may be anything in memory: zero weights must not meet a NaN
      const bool clear = (i & 1) && !all_needed(w.span, key0, key0 + KT_BK);
      // a step: 32 pieces, eight rows by four pieces
      constexpr int STEPS = KT_BK * PIECES / 128;  // a warp's
      uint4 x[STEPS];
#pragma unroll
      for (int y = 0; y < STEPS; ++y) {
        const int step = warp * STEPS + y, r = (step / (PIECES / 4)) * 8 + (lane & 7), piece = (step % (PIECES / 4)) * 4 + (lane >> 3);
        x[y] = k8_lds128(from + k8_at<HDP>(r, piece));
      }
#pragma unroll
      for (int y = 0; y < STEPS; ++y) {
        const int step = warp * STEPS + y, r = (step / (PIECES / 4)) * 8 + (lane & 7), piece = (step % (PIECES / 4)) * 4 + (lane >> 3);
        if (clear && !key_needed(w.span, key0 + r)) x[y] = make_uint4(0, 0, 0, 0);
        const uint32_t at = to + (piece >> 2) * Cfg::KV_HALF + r * 128, c0 = (piece & 3) * 2;
        sts128(at + ((c0 ^ (r & 7)) << 4), k8_unpack(x[y].x & 0xffffu), k8_unpack(x[y].x >> 16), k8_unpack(x[y].y & 0xffffu),
               k8_unpack(x[y].y >> 16));
        sts128(at + (((c0 + 1) ^ (r & 7)) << 4), k8_unpack(x[y].z & 0xffffu), k8_unpack(x[y].z >> 16), k8_unpack(x[y].w & 0xffffu),
               k8_unpack(x[y].w >> 16));
      }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      __syncwarp();
      if (elect_lane()) {
        mbar_arrive_at(bars + B::kv_full + 8 * hs);
        mbar_arrive_at(bars + B::raw_empty + 8 * rs);
      }
      __syncwarp();
    }
  }
  // the last uses of the operands: behind them no product is in flight (else the issuing warps see to that)
  for (uint32_t k = it >= NS ? it - NS : 0; k < it && ok; ++k) ok = kt_wait<B>(bars, B::kv_empty + 8 * (k % NS), (k / NS) & 1);
  if (units > 0 && ok) kt_wait<B>(bars, B::q_empty, (units - 1) & 1);
}

// Weights of a 32-column piece (four runs of 8 columns, whose factors, exponents less the reference, and way back are
// f, add and back) to TMEM column tp.  Otherwise as kt_weights, but with all exponentials on the special-function unit: the
// converters leave no slots on the other pipes (of eight pairs there none, one, two, three, four: 830, 832, 838, 848, 843 us for the
// long prompts above).
__device__ __forceinline__ void k8t_weights(uint32_t (&s)[32], const float (&f)[4], const float (&add)[4], const float (&back)[4],
                                            uint64_t& sum, uint32_t tp) {
  uint64_t v[16];
#pragma unroll
  for (int y = 0; y < 16; ++y)
    v[y] = f2_fma(f2_pack(__uint_as_float(s[2 * y]), __uint_as_float(s[2 * y + 1])), f2_pack(f[y >> 2], f[y >> 2]),
                  f2_pack(add[y >> 2], add[y >> 2]));
  uint32_t w[16];
#pragma unroll
  for (int y = 0; y < 16; ++y) {
    float a, b;
    f2_unpack(v[y], a, b);
    a = exp2_fast(a);
    b = exp2_fast(b);
    v[y] = f2_pack(a, b);
    w[y] = pack2<__half>(a, b);
  }
  tmem_store16(tp, w);
#pragma unroll
  for (int x = 0; x < 4; ++x)
    sum = f2_fma(f2_add(f2_add(v[4 * x], v[4 * x + 1]), f2_add(v[4 * x + 2], v[4 * x + 3])), f2_pack(back[x], back[x]), sum);
}

__device__ __forceinline__ void k8t_lds4(float (&v)[4], uint32_t a) {
  const uint4 w = lds128(a);
  v[0] = __uint_as_float(w.x), v[1] = __uint_as_float(w.y), v[2] = __uint_as_float(w.z), v[3] = __uint_as_float(w.w);
}

// The largest of a 32-column piece's u = score * factor + exponent; NaN if any is.
__device__ __forceinline__ float k8t_max(const uint32_t (&s)[32], const float (&f)[4], const float (&e)[4]) {
  float top = -INFINITY;
#pragma unroll
  for (int x = 0; x < 4; ++x) {
    float m = max_nan(__uint_as_float(s[8 * x]), __uint_as_float(s[8 * x + 1]));
#pragma unroll
    for (int y = 2; y < 8; y += 2) m = max_nan(max_nan(m, __uint_as_float(s[8 * x + y])), __uint_as_float(s[8 * x + y + 1]));
    top = max_nan(top, fmaf(m, f[x], e[x]));
  }
  return top;
}

// The 128 threads of row tile G, one a row (kt_rows, with exponents).
template <typename T, int HDP>
__device__ __forceinline__ void k8t_rows(const K8tParams& pp, uint32_t bars, uint32_t exps, uint32_t scales, uint32_t stage, int warp) {
  using Cfg = K8tCfg<HDP>;
  using B = K8tBars<HDP>;
  const KtParams& p = pp.t;
  const int G = warp >> 2, quad = warp & 3, lane = threadIdx.x & 31, r = quad * 32 + lane;
  const int32_t tok = r / p.group;
  const uint32_t ts = tmem_at(Cfg::TMEM_S + G * 128, quad, 0), to = tmem_at(Cfg::TMEM_O + G * HDP, quad, 0);
  const uint32_t pv_bar = B::pv_done + 8 * G;
  uint32_t base = 0, tile = 0, results = 0, units = 0;  // tiles before this unit, this row tile's tiles and results so far
  bool ok = true, there;
  KtWalk walk{};
  KtWork w;
#pragma unroll 1
  while (kt_next(p, walk, w, there)) {
    if (!there) continue;
    const int32_t cnt = G ? w.cnt1 : w.cnt0;
    const int32_t first = G ? w.pos1 : w.pos0, last = G ? w.last1 : w.last0;
    const int32_t pos = first + tok;
    float m = -INFINITY, l = 0.f, scale = 0.f;
#pragma unroll 1
    for (int32_t i = 0; i < cnt; ++i) {
      const uint32_t t = tile + i;
      const int32_t key0 = tile_index(w.tiles, w.j0 + i) * KT_BK;
      ok = ok && kt_wait<B>(bars, B::s_full + 16 * G + 8 * (t & 1), (t >> 1) & 1);
      __syncwarp();
      tc_fence_after();
      if (i == 0) scale = __uint_as_float(lds32(scales + ((units & 1) * 256 + G * 128 + r) * 4));
      const uint32_t tb = ts + (t & 1) * KT_BK, ex = exps + ((base + i) % K8T_EXPS) * 96;
      uint32_t s0[32], s1[32];
      tmem_ld32(tb, s0);
      tmem_ld32(tb + 32, s1);
      float f0[4], f1[4], e0[4], e1[4];
      k8t_lds4(f0, ex);
      k8t_lds4(f1, ex + 16);
      k8t_lds4(e0, ex + 32);
      k8t_lds4(e1, ex + 48);
#pragma unroll
      for (int x = 0; x < 4; ++x) {  // (never 0: the -inf of a masked column has to stay one)
        f0[x] = fmaxf(f0[x] * scale, 1.1754944e-38f);
        f1[x] = fmaxf(f1[x] * scale, 1.1754944e-38f);
      }
      tmem_wait32(s0);
      tmem_wait32(s1);
      if (!all_visible(key0, key0 + KT_BK, first, last, w.window, w.sinks)) {
        // visible columns of this row: x <= hi and (x > lo or x < sink)
        const int32_t hi = pos - key0, lo = w.window > 0 ? pos - w.window - key0 : -1, sink = w.sinks - key0;
        kt_mask(s0, 0, hi, lo, sink);
        kt_mask(s1, 32, hi, lo, sink);
      }
      // (NaN when one of the row's scores is: it is never a new reference, and makes the sum NaN below)
      const float top = max_nan(k8t_max(s0, f0, e0), k8t_max(s1, f1, e1));
      const bool grow = top > m + K8_TOP || (i == 0 && top > m);
      if (i > 0 && __any_sync(0xffffffffu, grow)) {
        const float f = grow ? (m == -INFINITY ? 0.f : exp2_fast(m - (top - K8_ROOM))) : 1.f;
        l *= f;
        ok = ok && kt_wait<B>(bars, pv_bar, (t - 1) & 1);  // the product before this one is done with O
        __syncwarp();
        tc_fence_after();
#pragma unroll 1
        for (int x = 0; x < HDP; x += 32) {
          uint32_t o[32];
          tmem_ld32(to + x, o);
          tmem_wait32(o);
#pragma unroll
          for (int y = 0; y < 32; ++y) o[y] = __float_as_uint(__uint_as_float(o[y]) * f);
          tmem_store32(to + x, o);
        }
      }
      if (grow) m = top - K8_ROOM;
      const float ref = m == -INFINITY ? 0.f : m;
      uint64_t sum = 0;
      float back[4];
#pragma unroll
      for (int x = 0; x < 4; ++x) e0[x] -= ref, e1[x] -= ref;
      k8t_lds4(back, ex + 64);
      k8t_weights(s0, f0, e0, back, sum, tb);
      k8t_lds4(back, ex + 80);
      k8t_weights(s1, f1, e1, back, sum, tb + 16);
      float a0, a1;
      f2_unpack(sum, a0, a1);
      l += a0 + a1;
      // a NaN score, and one of +inf (inf - inf), makes the row NaN, its sum as well as its weights
      if (!(top < INFINITY)) l = NAN;
      tmem_wait_st();
      tc_fence_before();
      mbar_arrive_at(bars + B::p_full + 16 * G + 8 * (t & 1));
    }
    const bool any = cnt > 0;
    tile += cnt;
    base += w.n;
    if (w.n > 0) ++units;
    if (any) ok = ok && kt_wait<B>(bars, B::o_full + 8 * G, results++ & 1);
    __syncwarp();
    tc_fence_after();
    kt_result<T, HDP>(p, w, to, stage, G, quad, any, __all_sync(0xffffffffu, ok), m, l);
    tc_fence_before();
  }
}

template <typename T, int HDP>
__global__ void __launch_bounds__(K8T_THREADS, 1)
    kv8_tile_kernel(const __grid_constant__ CUtensorMap tmk, const __grid_constant__ CUtensorMap tmv, const __grid_constant__ K8tParams p) {
  using Cfg = K8tCfg<HDP>;
  using B = K8tBars<HDP>;
  extern __shared__ uint8_t kt_smem_raw[];
  const uint32_t qs = (smem_addr(kt_smem_raw) + 1023) & ~1023u, ring = qs + Cfg::RING, raw = qs + Cfg::RAW, stage = qs + Cfg::STAGE;
  const uint32_t exps = qs + Cfg::EXPS, scales = qs + Cfg::SCALES, bars = qs + Cfg::BARS;
  const int warp = uniform(int(threadIdx.x) >> 5);
  if (threadIdx.x == 0) {
    for (int s = 0; s < Cfg::SLOTS; ++s) {
      mbar_init_at(bars + B::kv_full + 8 * s, 4);
      mbar_init_at(bars + B::kv_empty + 8 * s, 2);
    }
    for (int s = 0; s < Cfg::RAW_SLOTS; ++s) {
      mbar_init_at(bars + B::raw_full + 8 * s, 1);
      mbar_init_at(bars + B::raw_empty + 8 * s, 4);
    }
    mbar_init_at(bars + B::q_full, 4);
    mbar_init_at(bars + B::q_empty, 2);
    for (int g = 0; g < 2; ++g) {
      for (int x = 0; x < 16; x += 8) {
        mbar_init_at(bars + B::s_full + 16 * g + x, 1);
        mbar_init_at(bars + B::p_full + 16 * g + x, 128);
      }
      mbar_init_at(bars + B::pv_done + 8 * g, 1);
      mbar_init_at(bars + B::o_full + 8 * g, 1);
      mbar_init_at(bars + B::idle + 8 * g, 1);
    }
    sts32(bars + B::abort, 0u);
    fence_mbar_init();
  }
  if (warp == 8) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(bars + B::tmem), "r"(Cfg::TMEM_COLS)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = lds32(bars + B::tmem);
  // of the launch's 512 x 128 registers a row's thread takes 160, every other 96: 2 x 160 + 2 x 96 = 4 x 128
  if (warp < 8)
    asm volatile("setmaxnreg.inc.sync.aligned.u32 160;" ::: "memory");
  else
    asm volatile("setmaxnreg.dec.sync.aligned.u32 96;" ::: "memory");
  if (warp < 8) {
    k8t_rows<T, HDP>(p, bars, exps, scales, stage + warp * 4096, warp);
  } else if (warp == 8) {
    k8t_load<HDP>(&tmk, p, bars, raw, exps, 0);
  } else if (warp == 9) {
    k8t_load<HDP>(&tmv, p, bars, raw, exps, 1);
  } else if (warp < 12) {
    kt_multiply<__half, HDP, K8tCfg<HDP>, K8tBars<HDP>, true>(p.t, bars, qs, ring, warp - 10);
  } else {
    k8t_convert<T, HDP>(p, bars, qs, ring, raw, scales, warp - 12);
  }
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  tc_fence_before();
  __syncwarp();
  __syncthreads();
  if (warp == 8) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(Cfg::TMEM_COLS));
  }
}

}  // namespace lng
