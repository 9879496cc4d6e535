// Attention of many rows over the paged cache on the tensor cores: prompts, chunks of prompts, batches of
// drafts, and a whole batch against the prefix that it shares.
//
// A unit of work is two tiles of up to 128 (token, head of the key head's group) rows -- the group's heads share
// every key they load -- against the tiles of 64 keys that any of its tokens sees (or one range of them).  One CTA an
// SM takes units in turn, so that a unit's loads and first scores start under the one before.  Roles:
//   warps 0-3, 4-7  a row tile each, one row a thread: S from TMEM, the running maximum and sum in fp32, P, rounded to
//             the cache's type (as the step kernel's weights, and with its errors), over its S's columns;
//   warps 8, 9      load by TMA, page by page, into a ring: queries and keys, values;
//   warps 10, 11    issue a row tile's tcgen05.mma: S = Q K^T (fp32 in TMEM) a key tile ahead, O += P V, P from TMEM.
// TMEM: two S buffers of 64 columns a row tile (P in the same ones) and O of both (2 x head size).
// O is rescaled only when a row's maximum has grown by more than 2^8 (8 in base 2): the old reference stays
// valid, weights reach at most 256, exact in fp32 and in range for fp16, and the quotient is the same.
// Values are the B operand with the head dimension contiguous (MN-major), just as the pages hold them.
//
// What bounds it: at head size 64 a row tile's own softmax, about 1500 of the 1700 cycles that a pair of 64-key tiles
// takes (64 exponentials a thread, with the loads and the maximum before them); at head size 128 what warps 10 and 11
// do in a row, about 2000 cycles (sixteen products, four commits, four waits of a hundred cycles or more).  Key
// tiles of 128 with one S buffer were slower (32 prompts of 2048 tokens, 16 query and 4 key heads of 64: 0.63 against
// 0.55 ms), and so were: scores and products issued by a warp each (0.56 against 0.54 ms; two prompts of 8000
// tokens and 28 heads of 128: 0.75 against 0.76), sixteen row warps, two groups taking a row tile's key tiles in turn
// (0.73 and 0.87 ms), and the next scores loaded while the weights are formed (0.63 and 0.92 ms).
// Measured: 0.534 ms, 515 TFLOP/s, for the former; 0.87 ms, 809 TFLOP/s, for the latter (window of 4096) in a long
// loop, where power sets the clock (0.75 ms, 930 TFLOP/s, in the first few milliseconds).
#pragma once

#include "exp2_poly.cuh"
#include "kv_step.cuh"

namespace lng {

constexpr int KT_BM = 128, KT_BK = 64, KT_THREADS = 384;
// Of eight pairs of exponentials, those on the fma pipe.  None, one, two, three, four (32 prompts of 2048 tokens, heads
// of 64): 571, 559, 551, 533, 555 us; two prompts of 8000 tokens, heads of 128: 736, 727, 761, 755, 754.
constexpr uint32_t KT_FMA_EXP = 0x52;

template <int HDP>
struct KtCfg {
  static constexpr uint32_t Q_BYTES = 128 * HDP * 2, Q_HALF = 128 * 128;        // a row tile of queries; 64 columns of it
  static constexpr uint32_t KV_BYTES = KT_BK * HDP * 2, KV_HALF = KT_BK * 128;  // a tile of keys or values
  static constexpr int SLOTS = HDP == 128 ? 8 : 16;
  static constexpr uint32_t TMEM_S = 0, TMEM_O = 256, TMEM_COLS = 512;
  static constexpr size_t SMEM = size_t(2) * Q_BYTES + size_t(SLOTS) * KV_BYTES + 8 * 4096 + 1024 + 512;
};

struct KtParams {
  KvView c;
  KvRows o;
  int32_t q_heads, group, tile_tokens;  // tile_tokens = 128 / group
  float scale_log2;
  int32_t window, sinks;
  int32_t box;              // keys a TMA copy: min(page size, 64)
  int32_t splits;           // key ranges a unit's tiles are divided into
  int64_t total;            // units
  const int32_t* prefix_table;  // not null: all tokens against the shared prefix, every key visible
  int32_t prefix_len;
  float2* row_ml;           // split or prefix: states to [slot0 + split][row], row = token * q_heads + head
  float* row_o;
  int32_t slot0;
};

// Base of a column range of the CTA's TMEM for the lanes of this warp's quadrant.
__device__ __forceinline__ uint32_t tmem_at(uint32_t tmem, int quadrant, uint32_t col) {
  return tmem + (uint32_t(quadrant * 32) << 16) + col;
}

#define LNG_I8(a, o) "r"((a)[(o)]), "r"((a)[(o) + 1]), "r"((a)[(o) + 2]), "r"((a)[(o) + 3]), "r"((a)[(o) + 4]), \
                     "r"((a)[(o) + 5]), "r"((a)[(o) + 6]), "r"((a)[(o) + 7])
// (tmem_ld32 loads are asynchronous: their registers are only used behind tmem_wait32, which names them, so
// that no use of them can be moved in front of the wait.)
__device__ __forceinline__ void tmem_store32(uint32_t addr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,"
      "%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31};" ::LNG_I8(r, 0),
      LNG_I8(r, 8), LNG_I8(r, 16), LNG_I8(r, 24), "r"(addr)
      : "memory");
}
__device__ __forceinline__ void tmem_store16(uint32_t addr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15};" ::LNG_I8(r, 0),
      LNG_I8(r, 8), "r"(addr)
      : "memory");
}
#undef LNG_I8
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// kind::f16 with A from TMEM (two 16-bit values of a row in a column).
__device__ __forceinline__ void umma_f16_ts(uint32_t tmem_d, uint32_t tmem_a, uint64_t b, uint32_t idesc, uint32_t accum) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(tmem_d),
      "r"(tmem_a), "l"(b), "r"(idesc), "r"(accum)
      : "memory");
}
// A 128-byte swizzled operand, groups of 8 rows 1024 bytes apart: K-major (queries, keys: K contiguous, 16 a
// step of 32 bytes), or with N contiguous (values: one block of 64 columns, 16 rows of K a step of 2048 bytes).
__device__ __forceinline__ uint64_t umma_desc_at(uint32_t tile) {
  uint64_t d = (tile >> 4) & 0x3FFFull;
  d |= uint64_t(1) << 16;  // leading byte offset (unused: one block of 64 columns)
  d |= uint64_t(1024 >> 4) << 32;
  d |= uint64_t(1) << 46;
  d |= uint64_t(2) << 61;
  return d;
}
template <typename T>
__device__ __forceinline__ uint32_t umma_idesc(int M, int N, bool b_mn) {
  const uint32_t f = std::is_same<T, __half>::value ? 0u : 1u;
  return (1u << 4) | (f << 7) | (f << 10) | (uint32_t(b_mn) << 16) | (uint32_t(N >> 3) << 17) | (uint32_t(M >> 4) << 24);
}
__device__ __forceinline__ void tma_load_3d_at(uint32_t dst, const CUtensorMap* map, int32_t x, int32_t y, int32_t z, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(bar)
      : "memory");
}
__device__ __forceinline__ void tma_load_4d_at(uint32_t dst, const CUtensorMap* map, int32_t x, int32_t y, int32_t z, int32_t w,
                                               uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(w), "r"(bar)
      : "memory");
}

// A unit of work: 2 * tile_tokens tokens of one sequence (two row tiles), one key head, one range of the keys.
// Every warp of a CTA walks the CTA's units by itself.
struct KtWork {
  SeqSpan s;
  int64_t b;
  int32_t hk, split;
  int32_t t0, window, sinks;
  int32_t tokens0, tokens1;          // tokens of the two row tiles
  int32_t pos0, pos1, last0, last1;  // first and last position of each row tile
  int32_t cnt0, cnt1;                // key tiles [j0, j0 + cnt) are visited for a row tile
  int32_t j0, n;                     // [j0, j0 + n) for either
  bool shared;
  KeySpan span;
  KeyTiles tiles;
};

// Of the key tiles [j0, j1) those (a leading run) that hold keys up to `last`.
__device__ __forceinline__ int32_t kt_count(const KeyTiles& t, int32_t last, int32_t tokens, int32_t j0, int32_t j1) {
  const int32_t end = last >= 0 && tokens > 0 ? last / KT_BK + 1 : 0;
  int32_t n = end <= t.first ? (end < t.sink_tiles ? end : t.sink_tiles) : t.sink_tiles + end - t.first;
  n = n < j1 ? n : j1;
  return n > j0 ? n - j0 : 0;
}

// a / b for a >= 0 and 0 < b < 2^31 (a 64-bit division takes hundreds of cycles more, of which every unit has two or three).
__device__ __forceinline__ int64_t kt_quotient(int64_t a, int64_t b) {
  return a < (int64_t(1) << 32) ? int64_t(uint32_t(a) / uint32_t(b)) : a / b;
}

__device__ __forceinline__ int32_t uniform(int32_t v) { return __shfl_sync(0xffffffffu, v, 0); }

// The CTA's units: unit i of round k is k * grid + i, every second round backwards, so that each CTA's sum of units
// of falling size evens out.  Steps of equal n: the last units of all sequences, which see the most keys, come
// first.  Ragged steps: the sequences' units in a line, last units first within a sequence; the line is
// searched forward from where the last unit was found.
struct KtWalk {
  int64_t round, b, base;  // base: units of the sequences before b
};

__device__ __forceinline__ bool kt_next(const KtParams& p, KtWalk& walk, KtWork& w, bool& there) {
  const KvView& c = p.c;
  const int64_t grid = gridDim.x, k = walk.round++;
  const int64_t idx = k * grid + (k & 1 ? grid - 1 - int64_t(blockIdx.x) : int64_t(blockIdx.x));
  there = false;
  if (k * grid >= p.total) return false;
  if (idx >= p.total) return true;
  const int32_t inner = c.kv_heads * p.splits;  // (units of the same tokens: at most 65535 * 32)
  const int64_t u = kt_quotient(idx, inner);
  const int32_t rest = int32_t(idx - u * inner);
  w.hk = rest / p.splits;
  w.split = rest - w.hk * p.splits;
  w.shared = p.prefix_table != nullptr;
  const int32_t tt = p.tile_tokens, span = 2 * tt;
  if (w.shared) {  // all tokens of the step are one sequence, standing behind the prefix's last key
    int64_t first = 0, end = c.tokens;
    if (c.cu != nullptr) {
      first = c.cu[0];
      end = c.cu[c.batch];
      if (first < 0 || end < first || end > c.tokens) {
        kv_range_error();
        first = first < 0 ? 0 : first > c.tokens ? c.tokens : first;
        end = end > c.tokens ? c.tokens : end < first ? first : end;
      }
    }
    w.b = 0;
    w.s.first = first;
    w.s.n = int32_t(end - first);
    w.s.len = p.prefix_len;
    if (u * span >= w.s.n) return true;
    w.t0 = int32_t(u * span);
  } else if (c.cu == nullptr) {
    const int64_t per = (c.max_new + span - 1) / span, r = kt_quotient(u, c.batch);
    if (r >= per) return true;
    w.b = u - r * c.batch;
    w.s = kv_span(c, w.b);
    w.t0 = int32_t((per - 1 - r) * span);
  } else {
    const int lane = threadIdx.x & 31;
    for (;;) {  // 32 sequences a step
      if (walk.b >= c.batch) return true;
      const int64_t b = walk.b + lane;
      SeqSpan s{};
      if (b < c.batch) s = kv_span(c, b);
      const int32_t mine = (s.n + span - 1) / span;
      int64_t incl = mine;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int64_t v = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += v;
      }
      incl += walk.base;
      const uint32_t hit = __ballot_sync(0xffffffffu, u >= incl - mine && u < incl);
      if (hit) {
        const int src = __ffs(hit) - 1;
        w.b = walk.b + src;
        w.s.first = __shfl_sync(0xffffffffu, s.first, src);
        w.s.n = __shfl_sync(0xffffffffu, s.n, src);
        w.s.len = __shfl_sync(0xffffffffu, s.len, src);
        w.t0 = __shfl_sync(0xffffffffu, int32_t((incl - 1 - u) * span), src);
        break;
      }
      walk.base = __shfl_sync(0xffffffffu, incl, 31);
      walk.b += 32;
    }
  }
  there = true;
  w.window = w.shared ? 0 : p.window;
  w.sinks = w.shared ? 0 : p.sinks;
  const int32_t left = w.s.n - w.t0;
  w.tokens0 = left < tt ? left : tt;
  w.tokens1 = left <= tt ? 0 : (left < span ? left - tt : tt);
  const int32_t at = w.s.len - w.s.n + w.t0;
  w.pos0 = w.shared ? w.s.len - 1 : at;
  w.last0 = w.shared ? w.s.len - 1 : at + w.tokens0 - 1;
  w.pos1 = w.shared ? w.s.len - 1 : at + tt;
  w.last1 = w.shared ? w.s.len - 1 : at + tt + w.tokens1 - 1;
  w.span = key_span(w.pos0, w.tokens1 > 0 ? w.last1 : w.last0, w.window, w.sinks);
  w.tiles = key_tiles(w.span, KT_BK);
  w.j0 = int32_t(int64_t(w.tiles.count) * w.split / p.splits);
  const int32_t j1 = int32_t(int64_t(w.tiles.count) * (w.split + 1) / p.splits);
  w.cnt0 = uniform(kt_count(w.tiles, w.last0, w.tokens0, w.j0, j1));
  w.cnt1 = uniform(kt_count(w.tiles, w.last1, w.tokens1, w.j0, j1));
  w.n = w.cnt0 > w.cnt1 ? w.cnt0 : w.cnt1;
  return true;
}

// Shared memory behind the tiles, by 32-bit shared addresses (offsets from the block's).
template <int HDP>
struct KtBars {
  static constexpr uint32_t NS = KtCfg<HDP>::SLOTS;
  static constexpr uint32_t kv_full = 0, kv_empty = 8 * NS;  // [NS] each; empty: one arrival a row tile
  static constexpr uint32_t q_full = 16 * NS, q_empty = q_full + 8;  // empty: one arrival a row tile
  static constexpr uint32_t s_full = q_empty + 8;    // [2 row tiles][2]: scores of an even / odd key tile are in TMEM
  static constexpr uint32_t p_full = s_full + 32;   // [2][2], 128 arrivals: the tile's weights are, O is rescaled
  static constexpr uint32_t pv_done = p_full + 32;  // [2] O += P V is done, a phase a tile
  static constexpr uint32_t o_full = pv_done + 16;  // [2] the unit's last one is
  static constexpr uint32_t idle = o_full + 16;     // [2] no product of the row tile is in flight
  static constexpr uint32_t tmem = idle + 16, abort = tmem + 4;
  // A wait names a phase by its parity alone, so a role may only wait for a phase while the barrier can be in that
  // one or the next: every role waits for the phases of its barriers one after the other.
};

__device__ __forceinline__ uint32_t lds32(uint32_t a) {
  uint32_t v;
  asm volatile("ld.volatile.shared.u32 %0, [%1];" : "=r"(v) : "r"(a) : "memory");
  return v;
}
__device__ __forceinline__ void sts32(uint32_t a, uint32_t v) {
  asm volatile("st.volatile.shared.u32 [%0], %1;" ::"r"(a), "r"(v) : "memory");
}
__device__ __forceinline__ void sts128(uint32_t a, uint32_t x, uint32_t y, uint32_t z, uint32_t w) {
  asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(a), "r"(x), "r"(y), "r"(z), "r"(w) : "memory");
}
__device__ __forceinline__ uint4 lds128(uint32_t a) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a) : "memory");
  return v;
}
__device__ __forceinline__ void sts_zero16(uint32_t a) {
  asm volatile("st.shared.v4.u32 [%0], {%1, %1, %1, %1};" ::"r"(a), "r"(0u) : "memory");
}
__device__ __forceinline__ void mbar_init_at(uint32_t bar, uint32_t count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count) : "memory");
}
__device__ __forceinline__ void mbar_arrive_at(uint32_t bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void mbar_expect_at(uint32_t bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
__device__ __forceinline__ void umma_commit_at(uint32_t bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ bool mbar_try_at(uint32_t bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(bar), "r"(parity)
      : "memory");
  return ok != 0;
}
// Wait bounded by time (two seconds; the longest wait of a working kernel is a unit's, milliseconds), which also
// gives up when another role has -- but for the waits (ALONE) with which a role ends: whatever has happened, its own
// copies and products must not outlive the CTA.  An expired wait records the device error.
template <typename B, bool ALONE = false>
__device__ __forceinline__ bool kt_wait(uint32_t bars, uint32_t bar, uint32_t parity) {
  if (mbar_try_at(bars + bar, parity)) return true;
  uint64_t start, now;
  asm volatile("mov.u64 %0, %globaltimer;" : "=l"(start));
  for (uint32_t i = 0;; ++i) {
    if (mbar_try_at(bars + bar, parity)) return true;
    if ((i & 63) != 63) continue;
    if (!ALONE && lds32(bars + B::abort)) return false;
    asm volatile("mov.u64 %0, %globaltimer;" : "=l"(now));
    if (now - start > 2000000000ull) break;
  }
  atomicCAS(&g_error_word, 0u, (unsigned int)DEV_ERR_WAIT_TIMEOUT);
  sts32(bars + B::abort, 1u);
  return false;
}

// -inf in the columns of a 32-column piece (from column `base` of the tile) that the row does not see.
__device__ __forceinline__ void kt_mask(uint32_t (&s)[32], int32_t base, int32_t hi, int32_t lo, int32_t sink) {
#pragma unroll
  for (int x = 0; x < 32; ++x)
    if (base + x > hi) s[x] = 0xff800000u;
  if (base <= lo) {
#pragma unroll
    for (int x = 0; x < 32; ++x)
      if (base + x <= lo && base + x >= sink) s[x] = 0xff800000u;
  }
}
// The larger value, or NaN if either is.
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float kt_max(const uint32_t (&s)[32]) {
  float m0 = __uint_as_float(s[0]), m1 = __uint_as_float(s[1]);
#pragma unroll
  for (int x = 2; x < 30; x += 4) {
    m0 = max_nan(max_nan(m0, __uint_as_float(s[x])), __uint_as_float(s[x + 1]));
    m1 = max_nan(max_nan(m1, __uint_as_float(s[x + 2])), __uint_as_float(s[x + 3]));
  }
  return max_nan(max_nan(max_nan(m0, __uint_as_float(s[30])), __uint_as_float(s[31])), m1);
}
// 2^x of a pair on the fma pipe (exp2_poly.cuh has the steps).  x <= 8 here; below -126, and for the -inf of a masked
// key, the result is 2^-126.  NaN gives 2^-126 too: it is the row's maximum that carries a NaN score.
__device__ __forceinline__ void exp2_fma(uint64_t x2, float& a, float& b) {
  float x0, x1;
  f2_unpack(x2, x0, x1);
  x2 = f2_pack(fmaxf(x0, EXP2_LOW), fmaxf(x1, EXP2_LOW));
  const uint64_t t2 = f2_add(x2, f2_pack(EXP2_ROUND, EXP2_ROUND));
  const uint64_t f2 = f2_fma(f2_add(t2, f2_pack(-EXP2_ROUND, -EXP2_ROUND)), f2_pack(-1.f, -1.f), x2);
  uint64_t r2 = f2_fma(f2, f2_pack(EXP2_C4, EXP2_C4), f2_pack(EXP2_C3, EXP2_C3));
  r2 = f2_fma(r2, f2, f2_pack(EXP2_C2, EXP2_C2));
  r2 = f2_fma(r2, f2, f2_pack(EXP2_C1, EXP2_C1));
  r2 = f2_fma(r2, f2, f2_pack(EXP2_C0, EXP2_C0));
  float t0, t1;
  f2_unpack(t2, t0, t1);
  f2_unpack(r2, a, b);
  a = __int_as_float(__float_as_int(a) + (__float_as_int(t0) << 23));
  b = __int_as_float(__float_as_int(b) + (__float_as_int(t1) << 23));
}

// Weights of a 32-column piece to TMEM column tp: 2^(s * scale - ref), summed in fp32 and packed to the cache's
// type (rounded for the matrix unit; the sum keeps the unrounded weights).  Three of eight pairs go to the fma pipe:
// the special-function unit alone (16 a cycle and SM) would take as long as the products at head size 128 and
// twice as long at 64.
template <typename T>
__device__ __forceinline__ void kt_weights(uint32_t (&s)[32], uint64_t scale2, uint64_t ref2, uint64_t& sum0, uint64_t& sum1,
                                           uint32_t tp) {
  uint64_t v[16];
#pragma unroll
  for (int y = 0; y < 16; ++y) v[y] = f2_fma(f2_pack(__uint_as_float(s[2 * y]), __uint_as_float(s[2 * y + 1])), scale2, ref2);
#pragma unroll
  for (int y = 0; y < 16; ++y) {
    float a, b;
    if (KT_FMA_EXP >> (y & 7) & 1) {
      exp2_fma(v[y], a, b);
    } else {
      f2_unpack(v[y], a, b);
      a = exp2_fast(a);
      b = exp2_fast(b);
    }
    v[y] = f2_pack(a, b);
  }
  uint32_t w[16];
#pragma unroll
  for (int y = 0; y < 16; ++y) {
    float a, b;
    f2_unpack(v[y], a, b);
    w[y] = pack2<T>(a, b);
  }
  tmem_store16(tp, w);
#pragma unroll
  for (int y = 0; y < 16; y += 2) {
    sum0 = f2_add(sum0, v[y]);
    sum1 = f2_add(sum1, v[y + 1]);
  }
}

// Two warps, one for keys (and the units' queries), one for values: every tile's into the ring, page by page.  The
// lanes look up a tile's pages side by side, a tile ahead; one elected lane issues the copies, four pieces in a row
// without anything between (small pages make 16 copies a tile: one at a time they were slower than the products).
template <int HDP>
__device__ __forceinline__ void kt_load(const CUtensorMap* tmq, const CUtensorMap* map, const KtParams& p, uint32_t bars, uint32_t qs,
                                        uint32_t ring, const uint32_t kv) {
  using Cfg = KtCfg<HDP>;
  using B = KtBars<HDP>;
  constexpr uint32_t NS = Cfg::SLOTS;
  const KvView& c = p.c;
  const int lane = threadIdx.x & 31, box = p.box, boxes = KT_BK / box;
  const int32_t page_mask = (1 << c.page_shift) - 1;
  uint32_t it = kv, units = 0;  // this warp's next copy into the ring, units with keys
  bool ok = true, there;
  KtWalk walk{};
  KtWork w;
  while (ok && kt_next(p, walk, w, there)) {
    if (!there || w.n == 0) continue;
    const int32_t* row = w.shared ? p.prefix_table : c.table + w.b * c.table_stride;
    // the page of this lane's piece of a tile (-1: no token sees a key of it)
    auto look_up = [&](int32_t i) -> int32_t {
      const int32_t key = tile_index(w.tiles, w.j0 + i) * KT_BK + lane * box;
      if (lane >= boxes || !any_needed(w.span, key, key + box)) return -1;
      const int32_t page = page_of(row, key, c.page_shift, c.num_pages);
      if (page >= 0) return page;
      kv_range_error();
      return int32_t(c.num_pages);  // behind the last page: the copy fills zeros
    };
    int32_t next = look_up(0);
    if (kv == 0) {
      if (units > 0) ok = __all_sync(0xffffffffu, kt_wait<B>(bars, B::q_empty, (units - 1) & 1));
      if (!ok) break;
      if (elect_lane()) {
        const int32_t tiles_q = w.tokens1 > 0 ? 2 : 1, q0 = int32_t(w.s.first + w.t0);
        mbar_expect_at(bars + B::q_full, uint32_t(p.group * p.tile_tokens) * 128u * (HDP / 64) * tiles_q);
        for (int g = 0; g < tiles_q; ++g)
#pragma unroll
          for (int hh = 0; hh < HDP / 64; ++hh)
            tma_load_3d_at(qs + g * Cfg::Q_BYTES + hh * Cfg::Q_HALF, tmq, hh * 64, w.hk * p.group, q0 + g * p.tile_tokens,
                           bars + B::q_full);
      }
      __syncwarp();
    }
    ++units;
#pragma unroll 1
    for (int32_t i = 0; i < w.n; ++i, it += 2) {
      const int32_t page = next;
      const int32_t slot0 = uniform((tile_index(w.tiles, w.j0 + i) * KT_BK) & page_mask);
      if (i + 1 < w.n) next = look_up(i + 1);
      const uint32_t bytes = uint32_t(__popc(__ballot_sync(0xffffffffu, page >= 0))) * uint32_t(box) * 128u * (HDP / 64);
      const uint32_t s = it % NS, bar = bars + B::kv_full + 8 * s, dst = ring + s * Cfg::KV_BYTES;
      if (it >= NS) ok = __all_sync(0xffffffffu, kt_wait<B>(bars, B::kv_empty + 8 * s, (it / NS - 1) & 1));
      if (!ok) break;
      if (elect_lane()) mbar_expect_at(bar, bytes);
      __syncwarp();
#pragma unroll 1
      for (int r = 0; r < boxes; r += 4) {
        int32_t pg[4];
#pragma unroll
        for (int x = 0; x < 4; ++x) pg[x] = __shfl_sync(0xffffffffu, page, (r + x) & 31);
        if (elect_lane()) {
#pragma unroll
          for (int x = 0; x < 4; ++x)
            if (r + x < boxes && pg[x] >= 0) {
              const int32_t slot = (slot0 + (r + x) * box) & page_mask;
#pragma unroll
              for (int hh = 0; hh < HDP / 64; ++hh)
                tma_load_4d_at(dst + hh * Cfg::KV_HALF + (r + x) * box * 128, map, hh * 64, slot, w.hk, pg[x], bar);
            }
        }
        __syncwarp();
      }
    }
  }
  // the last uses of the ring's slots: behind them no copy and no product is in flight
  const uint32_t k0 = it >= NS ? it - NS : kv;
  bool used = true;
  for (uint32_t k = k0; k < it; k += 2) used = kt_wait<B>(bars, B::kv_empty + 8 * (k % NS), (k / NS) & 1) && used;
  if (kv == 0 && units > 0) used = kt_wait<B>(bars, B::q_empty, (units - 1) & 1) && used;
  if (__all_sync(0xffffffffu, used)) return;
  // (a role has given up: behind the copies themselves)
  for (uint32_t k = k0; k < it; k += 2) kt_wait<B, true>(bars, B::kv_full + 8 * (k % NS), (k / NS) & 1);
  if (kv == 0 && units > 0) kt_wait<B, true>(bars, B::q_full, (units - 1) & 1);
}

// One warp a row tile issues its products: the scores of the next key tile (into the other of two S buffers) ahead
// of O += P V of this one, so that the softmax finds its scores waiting.  P lies over its tile's scores; a product's
// operands are only overwritten once an mbarrier has shown it done (the ISA orders products of unlike operands
// through their completion alone).  APART: the values are waited for when their product is issued, not with the keys (nobody
// touches them in between).
template <typename T, int HDP, typename Cfg = KtCfg<HDP>, typename B = KtBars<HDP>, bool APART = false>
__device__ __forceinline__ void kt_multiply(const KtParams& p, uint32_t bars, uint32_t qs, uint32_t ring, int G) {
  constexpr uint32_t NS = Cfg::SLOTS;
  const uint32_t t_s = Cfg::TMEM_S + G * 128, t_o = Cfg::TMEM_O + G * HDP;  // (all of TMEM is this CTA's: its base is 0)
  const uint32_t pv_bar = B::pv_done + 8 * G;
  uint32_t base = 0, tile = 0, units = 0;  // ring copies before this unit, tiles of this row tile so far, units
  bool ok = true, there;
  // scores of ring copy ik, the row tile's tile t: they go where P of tile t - 2 lay, whose product is done
  auto scores = [&](uint32_t ik, uint32_t t) -> bool {
    const uint32_t sk = ik % NS;
    // (the values too: whoever has seen the scores may touch them)
    const bool good = __all_sync(0xffffffffu, kt_wait<B>(bars, B::kv_full + 8 * sk, (ik / NS) & 1) &&
                                                  (APART || kt_wait<B>(bars, B::kv_full + 8 * ((ik + 1) % NS), ((ik + 1) / NS) & 1)));
    tc_fence_after();
    if (good && elect_lane()) {
      const uint32_t idesc = umma_idesc<T>(KT_BM, KT_BK, false);
      const uint64_t dq = umma_desc_at(qs + G * Cfg::Q_BYTES), dk = umma_desc_at(ring + sk * Cfg::KV_BYTES);
#pragma unroll
      for (int k = 0; k < HDP / 16; ++k)  // (columns behind head_dim are zeros)
        umma_bf16(t_s + (t & 1) * KT_BK, dq + uint64_t((k >> 2) * int(Cfg::Q_HALF >> 4) + (k & 3) * 2),
                  dk + uint64_t((k >> 2) * int(Cfg::KV_HALF >> 4) + (k & 3) * 2), idesc, k > 0 ? 1u : 0u);
      umma_commit_at(bars + B::s_full + 16 * G + 8 * (t & 1));
      umma_commit_at(bars + B::kv_empty + 8 * sk);
    }
    __syncwarp();
    return good;
  };
  KtWalk walk{};
  KtWork w;
  while (ok && kt_next(p, walk, w, there)) {
    if (!there || w.n == 0) continue;
    const int32_t cnt = G ? w.cnt1 : w.cnt0;
    ok = __all_sync(0xffffffffu, kt_wait<B>(bars, B::q_full, units & 1));
    ++units;
    if (cnt > 0 && ok) ok = scores(base, tile);
#pragma unroll 1
    for (int32_t i = 0; i < cnt && ok; ++i) {
      if (tile + i > 0) ok = __all_sync(0xffffffffu, kt_wait<B>(bars, pv_bar, (tile + i - 1) & 1));
      if (i + 1 < cnt) {
        ok = ok && scores(base + 2 * (i + 1), tile + i + 1);
      } else if (elect_lane()) {
        umma_commit_at(bars + B::q_empty);  // behind the unit's last scores
      }
      __syncwarp();
      const uint32_t iv = base + 2 * i + 1, sv = iv % NS, t = tile + i;
      if (APART) ok = ok && kt_wait<B>(bars, B::kv_full + 8 * sv, (iv / NS) & 1);
      ok = __all_sync(0xffffffffu, ok && kt_wait<B>(bars, B::p_full + 16 * G + 8 * (t & 1), (t >> 1) & 1));
      tc_fence_after();
      if (ok && elect_lane()) {
        const uint32_t idesc = umma_idesc<T>(KT_BM, 64, true);
        const uint64_t dv = umma_desc_at(ring + sv * Cfg::KV_BYTES);
#pragma unroll
        for (int k = 0; k < KT_BK / 16; ++k)  // 16 keys: 16 rows of 128 bytes
#pragma unroll
          for (int hh = 0; hh < HDP / 64; ++hh)  // one product per block of 64 columns
            umma_f16_ts(t_o + hh * 64, t_s + (t & 1) * KT_BK + k * 8, dv + uint64_t(k * 128 + hh * int(Cfg::KV_HALF >> 4)), idesc,
                        i > 0 || k > 0 ? 1u : 0u);
        umma_commit_at(bars + pv_bar);
        umma_commit_at(bars + B::kv_empty + 8 * sv);
        if (i + 1 == cnt) umma_commit_at(bars + B::o_full + 8 * G);
      }
      __syncwarp();
    }
    if (cnt == 0 && elect_lane()) mbar_arrive_at(bars + B::q_empty);
    __syncwarp();
    // key tiles that none of this row tile's tokens sees: given back once they are there (not before: the slot's
    // last use by the other row tile may still be going on)
    for (uint32_t k = base + 2 * cnt; k < base + 2 * w.n && ok; ++k) {
      const uint32_t sl = k % NS;
      ok = __all_sync(0xffffffffu, kt_wait<B>(bars, B::kv_full + 8 * sl, (k / NS) & 1));
      if (ok && elect_lane()) mbar_arrive_at(bars + B::kv_empty + 8 * sl);
      __syncwarp();
    }
    base += 2 * w.n;
    tile += cnt;
  }
  // a role has given up: behind this warp's products (else the loading warps have seen the last of them done)
  if (__any_sync(0xffffffffu, !ok || lds32(bars + B::abort) != 0)) {
    if (elect_lane()) umma_commit_at(bars + B::idle + 8 * G);
    __syncwarp();
    kt_wait<B, true>(bars, B::idle + 8 * G, 0);
  }
}

// A warp's 32 rows of a unit's result, from TMEM columns `to` of its lanes: to the output, or with their maximum and
// sum as a state.  Rows pass through 4 KB of shared memory (16-byte pieces swizzled by row), so that eight lanes
// write 128 contiguous bytes of a row.
template <typename T, int HDP>
__device__ __forceinline__ void kt_result(const KtParams& p, const KtWork& w, uint32_t to, uint32_t stage, int G, int quad, bool any,
                                          bool ok, float m, float l) {
  const KvView& c = p.c;
  const int lane = threadIdx.x & 31;
  const int32_t tokens = ok ? (G ? w.tokens1 : w.tokens0) : 0, rows = tokens * p.group;
  const int64_t token0 = w.s.first + w.t0 + G * p.tile_tokens;
  const bool state = p.row_ml != nullptr;
  // no key seen: zeros (weights of masked keys are 2^-126, not 0); a row with a NaN score has l NaN
  const float inv = m == -INFINITY && l == l ? 0.f : 1.f / l;
  auto row_of = [&](int r, int64_t& token, int32_t& head) {
    const int32_t tok = r / p.group;
    token = token0 + tok;
    head = w.hk * p.group + (r - tok * p.group);
  };
  const int64_t state0 = int64_t(p.slot0 + w.split) * c.tokens * p.q_heads;
  if (state && quad * 32 + lane < rows) {
    int64_t token;
    int32_t head;
    row_of(quad * 32 + lane, token, head);
    p.row_ml[state0 + token * p.q_heads + head] = make_float2(l == l ? m : 0.f, l);
  }
  if (state && !any) return;  // (a state of sum 0 is not read)
  const int sub = lane >> 3, piece = lane & 7;
  const uint32_t mine = stage + lane * 128;
#pragma unroll 1
  for (int col = 0; col < HDP; col += 32) {
    uint32_t o[32];
    __syncwarp();
    if (any) {
      tmem_ld32(to + col, o);
      tmem_wait32(o);
    } else {
#pragma unroll
      for (int y = 0; y < 32; ++y) o[y] = 0u;
    }
    if (state) {
#pragma unroll
      for (int y = 0; y < 8; ++y) sts128(mine + ((y ^ (lane & 7)) << 4), o[4 * y], o[4 * y + 1], o[4 * y + 2], o[4 * y + 3]);
    } else {
#pragma unroll
      for (int y = 0; y < 4; ++y) {
        uint32_t w4[4];
#pragma unroll
        for (int z = 0; z < 4; ++z)
          w4[z] = pack2<T>(__uint_as_float(o[8 * y + 2 * z]) * inv, __uint_as_float(o[8 * y + 2 * z + 1]) * inv);
        const int at = (col >> 3 & 4) + y;  // two rounds of 32 columns fill the rows' 128 bytes
        sts128(mine + ((at ^ (lane & 7)) << 4), w4[0], w4[1], w4[2], w4[3]);
      }
      if (!(col & 32)) continue;
    }
    __syncwarp();
#pragma unroll
    for (int x = 0; x < 8; ++x) {
      const int rr = x * 4 + sub, r = quad * 32 + rr;
      if (r >= rows) continue;
      const uint4 v = lds128(stage + rr * 128 + ((piece ^ (rr & 7)) << 4));
      int64_t token;
      int32_t head;
      row_of(r, token, head);
      if (state) {
        const int d = col + piece * 4;
        if (d < c.head_dim) *reinterpret_cast<uint4*>(p.row_o + (state0 + token * p.q_heads + head) * c.head_dim + d) = v;
      } else {
        const int d = col - 32 + piece * 8;
        if (d < c.head_dim) *reinterpret_cast<uint4*>(static_cast<T*>(p.o.ptr) + token * p.o.token + head * p.o.head + d) = v;
      }
    }
  }
  __syncwarp();
}

// The 128 threads of row tile G, one a row: softmax of every key tile's scores, then the unit's result.
template <typename T, int HDP>
__device__ __forceinline__ void kt_rows(const KtParams& p, uint32_t bars, uint32_t ring, uint32_t stage, int warp) {
  using Cfg = KtCfg<HDP>;
  using B = KtBars<HDP>;
  constexpr uint32_t NS = Cfg::SLOTS;
  const int G = warp >> 2, quad = warp & 3, lane = threadIdx.x & 31, r = quad * 32 + lane;
  const int32_t tok = r / p.group;
  const uint32_t ts = tmem_at(Cfg::TMEM_S + G * 128, quad, 0), to = tmem_at(Cfg::TMEM_O + G * HDP, quad, 0);
  const uint32_t pv_bar = B::pv_done + 8 * G;
  const uint64_t scale2 = f2_pack(p.scale_log2, p.scale_log2);
  uint32_t base = 0, tile = 0, results = 0;  // ring copies before this unit, this row tile's tiles and results so far
  bool ok = true, there;
  KtWalk walk{};
  KtWork w;
#pragma unroll 1
  while (kt_next(p, walk, w, there)) {
    if (!there) continue;
    const int32_t cnt = G ? w.cnt1 : w.cnt0;
    const int32_t first = G ? w.pos1 : w.pos0, last = G ? w.last1 : w.last0;
    const int32_t pos = w.shared ? last : first + tok;
    float m = -INFINITY, l = 0.f;
#pragma unroll 1
    for (int32_t i = 0; i < cnt; ++i) {
      const uint32_t t = tile + i;
      const int32_t key0 = tile_index(w.tiles, w.j0 + i) * KT_BK;
      ok = ok && kt_wait<B>(bars, B::s_full + 16 * G + 8 * (t & 1), (t >> 1) & 1);
      if (!all_needed(w.span, key0, key0 + KT_BK)) {
        // slots that no row sees may hold anything: zero weights must not meet a NaN among the values (both row
        // tiles clear them, each before its own product)
        const uint32_t iv = base + 2 * i + 1, sv = iv % NS;
        if (ok && !key_needed(w.span, key0 + (r & 63))) {
          const uint32_t v = ring + sv * Cfg::KV_BYTES + (r & 63) * 128 + (r >> 6) * 64;
#pragma unroll
          for (int hh = 0; hh < HDP / 64; ++hh)
#pragma unroll
            for (int x = 0; x < 4; ++x) sts_zero16(v + hh * Cfg::KV_HALF + x * 16);
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      }
      __syncwarp();
      tc_fence_after();
      const uint32_t tb = ts + (t & 1) * KT_BK;
      uint32_t s0[32], s1[32];
      tmem_ld32(tb, s0);
      tmem_ld32(tb + 32, s1);
      tmem_wait32(s0);
      tmem_wait32(s1);
      if (!all_visible(key0, key0 + KT_BK, first, last, w.window, w.sinks)) {
        // visible columns of this row: x <= hi and (x > lo or x < sink)
        const int32_t hi = pos - key0, lo = w.window > 0 ? pos - w.window - key0 : -1, sink = w.sinks - key0;
        kt_mask(s0, 0, hi, lo, sink);
        kt_mask(s1, 32, hi, lo, sink);
      }
      // (NaN when one of the row's scores is: it is never a new reference, and makes the sum NaN below)
      const float top = max_nan(kt_max(s0), kt_max(s1)) * p.scale_log2;
      const bool grow = top > m + 8.f || (i == 0 && top > m);
      if (i > 0 && __any_sync(0xffffffffu, grow)) {
        const float f = grow ? (m == -INFINITY ? 0.f : exp2_fast(m - top)) : 1.f;
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
      if (grow) m = top;
      const float ref = m == -INFINITY ? 0.f : m;
      const uint64_t ref2 = f2_pack(-ref, -ref);
      uint64_t sum0 = 0, sum1 = 0;
      kt_weights<T>(s0, scale2, ref2, sum0, sum1, tb);
      kt_weights<T>(s1, scale2, ref2, sum0, sum1, tb + 16);
      float a0, a1, b0, b1;
      f2_unpack(sum0, a0, a1);
      f2_unpack(sum1, b0, b1);
      l += (a0 + a1) + (b0 + b1);
      // a NaN score, and one of +inf (inf - inf), makes the row NaN whichever pipe its own weight went through
      if (!(top < INFINITY)) l = NAN;
      tmem_wait_st();
      tc_fence_before();
      mbar_arrive_at(bars + B::p_full + 16 * G + 8 * (t & 1));
    }
    const bool any = cnt > 0;
    tile += cnt;
    base += 2 * w.n;
    if (any) ok = ok && kt_wait<B>(bars, B::o_full + 8 * G, results++ & 1);
    __syncwarp();
    tc_fence_after();
    kt_result<T, HDP>(p, w, to, stage, G, quad, any, __all_sync(0xffffffffu, ok), m, l);
    tc_fence_before();
  }
}

template <typename T, int HDP>
__global__ void __launch_bounds__(KT_THREADS, 1)
    kv_tile_kernel(const __grid_constant__ CUtensorMap tmq, const __grid_constant__ CUtensorMap tmk,
                   const __grid_constant__ CUtensorMap tmv, const __grid_constant__ KtParams p) {
  using Cfg = KtCfg<HDP>;
  using B = KtBars<HDP>;
  extern __shared__ uint8_t kt_smem_raw[];
  const uint32_t qs = (smem_addr(kt_smem_raw) + 1023) & ~1023u, ring = qs + 2 * Cfg::Q_BYTES;
  const uint32_t stage = ring + Cfg::SLOTS * Cfg::KV_BYTES, bars = stage + 8 * 4096;
  const int warp = uniform(int(threadIdx.x) >> 5);
  if (threadIdx.x == 0) {
    for (int s = 0; s < Cfg::SLOTS; ++s) {
      mbar_init_at(bars + B::kv_full + 8 * s, 1);
      mbar_init_at(bars + B::kv_empty + 8 * s, 2);
    }
    mbar_init_at(bars + B::q_full, 1);
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
  if (warp < 8) {
    kt_rows<T, HDP>(p, bars, ring, stage + warp * 4096, warp);
  } else if (warp == 8) {
    kt_load<HDP>(&tmq, &tmk, p, bars, qs, ring, 0);
  } else if (warp == 9) {
    kt_load<HDP>(&tmq, &tmv, p, bars, qs, ring, 1);
  } else {
    kt_multiply<T, HDP>(p, bars, qs, ring, warp - 10);
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

// The sequence whose rows hold `token`, found by a whole warp, which leaves a 32nd of them after each round of
// loads.  (Offsets that do not ascend give some sequence of the batch.)
__device__ __forceinline__ int64_t kt_sequence_of(const KvView& c, int64_t token, int lane) {
  int64_t lo = 0, hi = c.batch;
  while (hi - lo > 1) {
    const int64_t step = (hi - lo + 31) / 32, at = lo + (lane + 1) * step;
    const int found = __popc(__ballot_sync(0xffffffffu, at < hi && c.cu[at] <= token));
    lo += found * step;
    hi = lo + step < hi ? lo + step : hi;
  }
  return lo;
}

// out = the joined states of all slots, a warp a row; rows that belong to no sequence (they have no states, or only
// the prefix's) are left alone.
template <typename T>
__global__ void __launch_bounds__(256)
    kv_rows_join_kernel(const KvView c, int32_t q_heads, const float2* __restrict__ row_ml, const float* __restrict__ row_o,
                        int32_t slots, KvRows out) {
  const int64_t row = (int64_t(blockIdx.x) * blockDim.x + threadIdx.x) >> 5, tokens = c.tokens;
  const int lane = threadIdx.x & 31, col = lane * 4, head_dim = c.head_dim;
  const int64_t token = row / q_heads;
  bool mine = token < tokens;
  if (c.cu != nullptr && mine) {
    const SeqSpan s = kv_span(c, kt_sequence_of(c, token, lane));
    mine = token >= s.first && token < s.first + s.n;
  }
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if (!mine) return;
  const int64_t slot_rows = tokens * q_heads;
  const KsRow x = ks_join_states(
      0, 1, slots, lane, col < head_dim, [&](int i) { return row_ml + i * slot_rows + row; },
      [&](int i) { return row_o + (i * slot_rows + row) * head_dim + col; });
  const int head = int(row - token * q_heads);
  if (col < head_dim) ks_store_row(x, static_cast<T*>(out.ptr) + token * out.token + head * out.head + col);
}

}  // namespace lng
