// Attention of few rows over the paged cache: decoding and the verification of a few drafts, at most 16
// (token, head) rows a key head.
//
// Bound by memory: every key and value is read once for those rows, 4 * 16 flops a 2-byte element at
// most, so the matrix work (mma.sync m16n8k16, the 16 rows = M) stays far below the tensor rate and
// what counts is an unbroken stream of loads.  One CTA an SM; each of its warps owns a ring of three
// stages of 32 keys (keys and values, 48 KB a warp at head size 128) that an elected lane keeps filled by TMA from
// the pages, 16 rows of the tensor map or more a copy, so loads of the next blocks are in flight while a
// block is multiplied, across the borders of sequences too.
//
// The work -- all blocks of 32 visible keys of all (sequence, key head) pairs, in one line -- is cut into
// equal shares, one a warp or (few pairs) one a CTA: whatever the lengths, no SM waits for a longer sequence, and one
// long sequence uses them all.  A pair that lies in one share is finished there; of one that is cut, every share
// stores the softmax state (maximum, sum, unnormalised product, fp32) of its piece, and kv_step_join_kernel
// joins the pieces in order.  A share has at most two pieces (its first and its last pair).
//
// Weights are rounded to the cache's type for the product with the values, since the matrix unit takes both operands
// in one type (more bits would take a second product, with what the rounding left); their sum is not rounded.  Mean error
// against 64 bits, relative to the outputs' size: 0.0023 in bf16 and 0.00028 in fp16, where outputs that are only
// rounded at the end have 0.0017 and 0.00021.
//
// Measured (one token a sequence): 64 sequences of 500 to 16000 keys, 32 query and 8 key heads of 128 (2.24 GB of
// keys and values): 0.37 ms, 6.1 TB/s (0.34 where L2 still holds a twentieth of the keys from the call before); 24
// sequences, window of 4096 and pages of 16: 79 us, 5.1 TB/s (97 with a cold L2); 64 sequences of 300 keys: 31 us, 2.6
// TB/s (a pair's start and end, not its keys); one sequence of 4096 keys, 4 heads of 64: 16 us.
#pragma once

#include <type_traits>

#include "kvcache.cuh"
#include "tc_prims.cuh"

namespace lng {

constexpr int KS_ROWS = 16, KS_STAGES = 3;

template <int HDP>  // head size padded to 64 or 128
struct KsCfg {
  // (blocks of 16 keys on eight warps at head size 128 were slower, 0.46 against 0.39 ms a step of 64 long
  // sequences: what a block costs besides its keys counts twice)
  static constexpr int BK = 32, WARPS = 512 / HDP, THREADS = 32 * WARPS;
  static constexpr uint32_t HALF_BYTES = BK * 128;               // BK keys x 64 values
  static constexpr uint32_t KV_BYTES = HALF_BYTES * (HDP / 64);  // K (or V) of a stage
  static constexpr uint32_t STAGE_BYTES = 2 * KV_BYTES;
  static constexpr uint32_t RING_BYTES = STAGE_BYTES * KS_STAGES;  // one warp's
  static constexpr uint32_t MERGE_BYTES = 4 * KS_ROWS * HDP * 4;  // the products of four warps
  static constexpr size_t SMEM =
      size_t(WARPS) * RING_BYTES + MERGE_BYTES + WARPS * KS_ROWS * 8 + WARPS * KS_STAGES * 8 + 64 + 1024;
};

struct KsParams {
  KvView c;
  KvRows q, o;
  int32_t q_heads, group;
  float scale_log2;  // scale * log2(e): the softmax runs in base 2
  int32_t window, sinks;
  int32_t box;       // keys a TMA copy: min(page size, 32)
  // pieces: slot 2 * share (a pair begun before the share) and 2 * share + 1 (one that goes on behind it)
  float2* piece_ml;  // [2 * shares][piece_rows] (maximum, sum), base 2
  float* piece_o;    // [2 * shares][piece_rows][head_dim]
  int32_t piece_rows;  // room for a pair's rows: 16 here
  int32_t shares;    // into which the line is cut
  // a shared prefix: states of `prefix_slots` ranges of it, [slot][row][..] with row = token * q_heads + head;
  // pairs finished by one CTA then go to slot prefix_slots (null: to o)
  float2* row_ml;
  float* row_o;
  int32_t prefix_slots;
};

// The line of blocks: sequence b's pairs (key heads 0 .. KV - 1) have blocks(b) blocks each.
template <int BK>
__device__ __forceinline__ int32_t ks_blocks(const KvView& c, const SeqSpan& s, int32_t window, int32_t sinks) {
  if (s.n <= 0) return 0;
  return key_tiles(key_span(s.len - s.n, s.len - 1, window, sinks), BK).count;
}

__device__ __forceinline__ int64_t ks_share(int64_t total, int shares) {
  const int64_t per = (total + shares - 1) / shares;
  return per > 0 ? per : 1;
}

// Sums blocks(b) * KV over all sequences and finds, for the CTA's FINDS shares from share0 on, the sequence in which
// the share's first block falls and the line's position where that sequence starts (b = batch behind the line's
// end); returns that of share share0 + mine_of.  All `nthreads` threads take part; thread t sums a contiguous run
// of sequences.
struct KsFound {
  int64_t total, b, start;
};

template <int BK, int FINDS>
__device__ inline KsFound ks_find(const KvView& c, int32_t window, int32_t sinks, int nthreads, int shares, int64_t* warp_tot,
                                  int64_t (*found)[2], int64_t share0, int mine_of) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int64_t run = (c.batch + nthreads - 1) / nthreads;
  const int64_t b0 = tid * run, b1 = b0 + run < c.batch ? b0 + run : c.batch;
  int64_t mine = 0;
  for (int64_t b = b0; b < b1; ++b) mine += int64_t(ks_blocks<BK>(c, kv_span(c, b), window, sinks)) * c.kv_heads;
  int64_t incl = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t v = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += v;
  }
  if (lane == 31) warp_tot[warp] = incl;
  if (tid < FINDS) {
    found[tid][0] = c.batch;
    found[tid][1] = 0;
  }
  __syncthreads();
  int64_t before = 0, total = 0;
  for (int w = 0; w < nthreads / 32; ++w) {
    if (w < warp) before += warp_tot[w];
    total += warp_tot[w];
  }
  const int64_t at = before + incl - mine;
  const int64_t per = ks_share(total, shares);
  for (int f = 0; f < FINDS; ++f) {
    const int64_t want = (share0 + f) * per;
    if (want < at || want >= at + mine) continue;
    int64_t pos = at;
    for (int64_t b = b0; b < b1; ++b) {
      const int64_t n = int64_t(ks_blocks<BK>(c, kv_span(c, b), window, sinks)) * c.kv_heads;
      if (want < pos + n) {
        found[f][0] = b;
        found[f][1] = pos;
        break;
      }
      pos += n;
    }
  }
  __syncthreads();
  return KsFound{total, found[mine_of][0], found[mine_of][1]};
}

__device__ __forceinline__ void tma_load_4d(void* dst, const CUtensorMap* map, int32_t x, int32_t y, int32_t z, int32_t w,
                                            uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(
          smem_addr(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(w), "r"(smem_addr(bar))
      : "memory");
}

template <typename T>
__device__ __forceinline__ void mma_16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (std::is_same<T, __half>::value)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <typename T>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  uint32_t r;
  if constexpr (std::is_same<T, __half>::value)
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  else
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ float exp2_fast(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
// One lane of the (converged) warp.  Copies and products are issued by whole warps with uniform operands and one
// elected lane: operands that the compiler cannot see to be uniform cost a hundred cycles each.
__device__ __forceinline__ bool elect_lane() {
  uint32_t ok;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(ok)::"memory");
  return ok != 0;
}
__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}
__device__ __forceinline__ void ldsm4_t(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}

// A walk along a CTA's share: the current pair, its sequence and the blocks [k0, k1) of it that belong to
// the share.
template <int BK>
struct KsWalk {
  int64_t pos, end;  // in the line
  int64_t b;
  int32_t h, k0, k1, blocks;
  SeqSpan s;
  KeySpan span;
  KeyTiles tiles;
  __device__ __forceinline__ bool done() const { return pos >= end; }
  __device__ __forceinline__ void enter(const KvView& c, int32_t window, int32_t sinks) {
    s = kv_span(c, b);
    span = key_span(s.len - s.n, s.len - 1, window, sinks);
    tiles = key_tiles(span, BK);
    blocks = s.n > 0 ? tiles.count : 0;
  }
  __device__ __forceinline__ void clip() {
    const int64_t left = end - pos;
    k1 = blocks - k0 <= left ? blocks : k0 + int32_t(left);
  }
  __device__ __forceinline__ void start(const KvView& c, int32_t window, int32_t sinks, const KsFound& f, int64_t p0, int64_t p1) {
    pos = p0;
    end = p1;
    if (done()) return;
    b = f.b;
    enter(c, window, sinks);
    const int64_t off = p0 - f.start;
    h = int32_t(off / blocks);
    k0 = int32_t(off - int64_t(h) * blocks);
    clip();
  }
  // to the next pair
  __device__ __forceinline__ void next(const KvView& c, int32_t window, int32_t sinks) {
    pos += k1 - k0;
    if (done()) return;
    k0 = 0;
    if (++h == c.kv_heads) {
      h = 0;
      do {
        ++b;
        enter(c, window, sinks);
      } while (blocks == 0);  // (pos < end: a later sequence has blocks)
    }
    clip();
  }
};

// WS: a share a warp (many pairs: no meeting of warps at each pair's end), else a share a CTA (few pairs: fewer
// pieces a pair).
template <typename T, int HDP, bool WS>
__global__ void __launch_bounds__(KsCfg<HDP>::THREADS, 1)
    kv_step_kernel(const __grid_constant__ CUtensorMap tmk, const __grid_constant__ CUtensorMap tmv, const KsParams p) {
  using Cfg = KsCfg<HDP>;
  constexpr int WARPS = Cfg::WARPS, BK = Cfg::BK, KSTEPS = HDP / 16, NT = HDP / 8, ST = BK / 8;
  extern __shared__ uint8_t ks_smem_raw[];
  uint8_t* base = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(ks_smem_raw) + 1023) & ~uintptr_t(1023));
  float* merge_o = reinterpret_cast<float*>(base + WARPS * Cfg::RING_BYTES);  // [WARPS][16][HDP]
  float2* merge_ml = reinterpret_cast<float2*>(reinterpret_cast<uint8_t*>(merge_o) + Cfg::MERGE_BYTES);  // [WARPS][16]
  uint64_t* bars = reinterpret_cast<uint64_t*>(merge_ml + WARPS * KS_ROWS);   // [WARPS][STAGES]
  __shared__ int64_t warp_tot[WARPS], found[WS ? WARPS : 1][2];
  const KvView& c = p.c;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  uint8_t* ring = base + warp * Cfg::RING_BYTES;
  uint64_t* bar = bars + warp * KS_STAGES;

  if (lane == 0) {
    for (int s = 0; s < KS_STAGES; ++s) mbar_init(&bar[s], 1);
    fence_mbar_init();
    if (warp == 0) {
      tma_prefetch_desc(&tmk);
      tma_prefetch_desc(&tmv);
    }
  }
  // blocks of a pair that are this warp's: all of its share's, or every WARPS-th of the CTA's
  constexpr int STRIDE = WS ? 1 : WARPS;
  const int start = WS ? 0 : warp;
  const int64_t share0 = int64_t(blockIdx.x) * (WS ? WARPS : 1), share = share0 + (WS ? warp : 0);
  const KsFound f = ks_find<BK, WS ? WARPS : 1>(c, p.window, p.sinks, Cfg::THREADS, p.shares, warp_tot, found, share0, WS ? warp : 0);
  const int64_t per = ks_share(f.total, p.shares);
  const int64_t p0 = share * per, p1 = p0 + per < f.total ? p0 + per : f.total;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

  // the loading walk runs KS_STAGES blocks of this warp ahead of the computing walk
  KsWalk<BK> ld, cw;
  ld.start(c, p.window, p.sinks, f, p0, p1);
  cw = ld;
  int32_t ld_k = ld.done() ? 0 : ld.k0 + start;
  uint32_t issued = 0, taken = 0;
  // pages of the warp's next blocks of the pair, a piece (of `box` keys) a lane: looked up together, since a
  // look-up of one block's page takes longer than its copies
  const int boxes = BK / p.box, ahead = 32 / boxes;
  int32_t pages = -1, seen = ahead;  // -1: no row sees a key of the piece; blocks issued out of the looked-up ones
  auto look_up = [&]() {
    const int32_t k = ld_k + (lane / boxes) * STRIDE;
    pages = -1;
    if (k < ld.k1) {
      const int32_t key = tile_index(ld.tiles, k) * BK + (lane % boxes) * p.box;
      if (any_needed(ld.span, key, key + p.box)) {
        pages = page_of(c.table + ld.b * c.table_stride, key, c.page_shift, c.num_pages);
        if (pages < 0) {
          kv_range_error();
          pages = int32_t(c.num_pages);  // behind the last page: the copy fills zeros
        }
      }
    }
    seen = 0;
  };
  auto issue = [&]() {  // the warp's next block into the ring (all lanes keep the walk; an elected one copies)
    while (!ld.done() && ld_k >= ld.k1) {
      ld.next(c, p.window, p.sinks);
      if (!ld.done()) ld_k = ld.k0 + start;
      seen = ahead;
    }
    if (ld.done()) return;
    if (seen == ahead) look_up();
    const uint32_t s = issued % KS_STAGES, mine = boxes == 32 ? 0xffffffffu : ((1u << boxes) - 1u);
    const uint32_t there = (__ballot_sync(0xffffffffu, pages >= 0) >> (seen * boxes)) & mine;
    uint8_t* dk = ring + s * Cfg::STAGE_BYTES;
    uint8_t* dv = dk + Cfg::KV_BYTES;
    const int32_t slot0 = (tile_index(ld.tiles, ld_k) * BK) & ((1 << c.page_shift) - 1);
    if (elect_lane()) mbar_arrive_expect_tx(&bar[s], uint32_t(__popc(there)) * uint32_t(p.box) * 128 * (HDP / 64) * 2);
    __syncwarp();
#pragma unroll 1
    for (int r = 0; r < boxes; r += 2) {  // (two pieces, or the only one, without anything between)
      int32_t pg[2];
#pragma unroll
      for (int x = 0; x < 2; ++x) pg[x] = __shfl_sync(0xffffffffu, pages, (seen * boxes + r + x) & 31);
      if (elect_lane()) {
#pragma unroll
        for (int x = 0; x < 2; ++x)
          if (r + x < boxes && pg[x] >= 0) {
            const int32_t slot = (slot0 + (r + x) * p.box) & ((1 << c.page_shift) - 1);
#pragma unroll
            for (int hh = 0; hh < HDP / 64; ++hh) {
              tma_load_4d(dk + hh * Cfg::HALF_BYTES + (r + x) * p.box * 128, &tmk, hh * 64, slot, ld.h, pg[x], &bar[s]);
              tma_load_4d(dv + hh * Cfg::HALF_BYTES + (r + x) * p.box * 128, &tmv, hh * 64, slot, ld.h, pg[x], &bar[s]);
            }
          }
      }
      __syncwarp();
    }
    ++issued;
    ++seen;
    ld_k += STRIDE;
  };
#pragma unroll 1
  for (int i = 0; i < KS_STAGES; ++i) issue();

  const int g = lane >> 2, t4 = lane & 3;
  const int rows_of_n = p.group;
  bool ok = true;
  for (; !cw.done(); cw.next(c, p.window, p.sinks)) {
    const int32_t rows = rows_of_n * cw.s.n;  // <= 16
    const int32_t pos0 = cw.s.len - cw.s.n;
    // Q fragments (row r = token r / group, head r % group); rows and columns that are not there are zero
    uint32_t qf[KSTEPS][4];
    {
      const T* qa[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int r = g + 8 * i;
        const int tok = r / rows_of_n, hd = r - tok * rows_of_n;
        qa[i] = r < rows ? static_cast<const T*>(p.q.ptr) + (cw.s.first + tok) * p.q.token + (cw.h * p.group + hd) * p.q.head : nullptr;
      }
#pragma unroll
      for (int k = 0; k < KSTEPS; ++k)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int col = k * 16 + (i >> 1) * 8 + t4 * 2;
          const T* src = qa[i & 1];
          qf[k][i] = src && col < c.head_dim ? *reinterpret_cast<const uint32_t*>(src + col) : 0u;
        }
    }
    const int32_t pa = pos0 + g / rows_of_n, pb = pos0 + (g + 8) / rows_of_n;  // the rows' positions
    float oacc[NT][4];
#pragma unroll
    for (int i = 0; i < NT; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) oacc[i][j] = 0.f;
    float ma = -INFINITY, mb = -INFINITY, la = 0.f, lb = 0.f;

    for (int32_t k = cw.k0 + start; k < cw.k1; k += STRIDE) {
      const uint32_t s = taken % KS_STAGES;
      if (ok) ok = mbar_wait_bounded(&bar[s], (taken / KS_STAGES) & 1, &g_error_word, DEV_ERR_WAIT_TIMEOUT);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      uint8_t* sk = ring + s * Cfg::STAGE_BYTES;
      uint8_t* sv = sk + Cfg::KV_BYTES;
      const int32_t key0 = tile_index(cw.tiles, k) * BK;
      const bool whole = all_needed(cw.span, key0, key0 + BK);
      if (!whole) {
        // values of keys that no row sees may be anything in memory: zero weights must not meet a NaN
        constexpr int PARTS = 32 / BK;  // lanes a row
        const int key = lane % BK, part = lane / BK;
        if (!key_needed(cw.span, key0 + key)) {
#pragma unroll
          for (int hh = 0; hh < HDP / 64; ++hh)
#pragma unroll
            for (int i = 0; i < 8 / PARTS; ++i)
              *reinterpret_cast<uint4*>(sv + hh * Cfg::HALF_BYTES + key * 128 + (part * (8 / PARTS) + i) * 16) = make_uint4(0, 0, 0, 0);
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // before the next copy into this stage
        __syncwarp();
      }
      // S = Q K^T: 16 rows x BK keys
      float sacc[ST][4];
#pragma unroll
      for (int i = 0; i < ST; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) sacc[i][j] = 0.f;
      const uint32_t skb = smem_addr(sk), svb = smem_addr(sv);
#pragma unroll
      for (int kk = 0; kk < KSTEPS; ++kk) {
        if (kk * 16 < c.head_dim) {
#pragma unroll
          for (int np = 0; np < ST / 2; ++np) {  // keys 16 np .. + 15
            const int key = np * 16 + (lane & 7) + ((lane >> 4) << 3);
            const int chunk = (kk & 3) * 2 + ((lane >> 3) & 1);
            uint32_t b[4];
            ldsm4(b, skb + (kk >> 2) * Cfg::HALF_BYTES + key * 128 + ((chunk ^ (key & 7)) << 4));
            mma_16816<T>(sacc[2 * np], qf[kk], b[0], b[1]);
            mma_16816<T>(sacc[2 * np + 1], qf[kk], b[2], b[3]);
          }
        }
      }
      if (!all_visible(key0, key0 + BK, pos0, cw.s.len - 1, p.window, p.sinks)) {
#pragma unroll
        for (int n = 0; n < ST; ++n)
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int32_t key = key0 + n * 8 + t4 * 2 + (j & 1);
            if (!key_visible(key, j < 2 ? pa : pb, p.window, p.sinks)) sacc[n][j] = -INFINITY;
          }
      }
      // running maximum and sum of the two rows (base 2)
      float xa = -INFINITY, xb = -INFINITY;
#pragma unroll
      for (int n = 0; n < ST; ++n) {
        xa = fmaxf(xa, fmaxf(sacc[n][0], sacc[n][1]));
        xb = fmaxf(xb, fmaxf(sacc[n][2], sacc[n][3]));
      }
#pragma unroll
      for (int o = 1; o < 4; o <<= 1) {
        xa = fmaxf(xa, __shfl_xor_sync(0xffffffffu, xa, o));
        xb = fmaxf(xb, __shfl_xor_sync(0xffffffffu, xb, o));
      }
      const float na = fmaxf(ma, xa * p.scale_log2), nb = fmaxf(mb, xb * p.scale_log2);
      if (__any_sync(0xffffffffu, na > ma || nb > mb)) {
        const float fa = ma == -INFINITY ? 0.f : exp2_fast(ma - na), fb = mb == -INFINITY ? 0.f : exp2_fast(mb - nb);
        la *= fa;
        lb *= fb;
#pragma unroll
        for (int i = 0; i < NT; ++i) {
          oacc[i][0] *= fa;
          oacc[i][1] *= fa;
          oacc[i][2] *= fb;
          oacc[i][3] *= fb;
        }
        ma = na;
        mb = nb;
      }
      const float ra = ma == -INFINITY ? 0.f : ma, rb = mb == -INFINITY ? 0.f : mb;
#pragma unroll
      for (int n = 0; n < ST; ++n) {
        sacc[n][0] = exp2_fast(sacc[n][0] * p.scale_log2 - ra);
        sacc[n][1] = exp2_fast(sacc[n][1] * p.scale_log2 - ra);
        sacc[n][2] = exp2_fast(sacc[n][2] * p.scale_log2 - rb);
        sacc[n][3] = exp2_fast(sacc[n][3] * p.scale_log2 - rb);
        la += sacc[n][0] + sacc[n][1];
        lb += sacc[n][2] + sacc[n][3];
      }
      // O += P V; the weights are rounded to the cache's type for the matrix unit, their sum is not
#pragma unroll
      for (int kk = 0; kk < BK / 16; ++kk) {
        uint32_t a[4] = {pack2<T>(sacc[2 * kk][0], sacc[2 * kk][1]), pack2<T>(sacc[2 * kk][2], sacc[2 * kk][3]),
                         pack2<T>(sacc[2 * kk + 1][0], sacc[2 * kk + 1][1]), pack2<T>(sacc[2 * kk + 1][2], sacc[2 * kk + 1][3])};
#pragma unroll
        for (int np = 0; np < HDP / 16; ++np) {
          if (np * 16 < c.head_dim) {
            const int key = kk * 16 + (lane & 15);
            const int chunk = (np & 3) * 2 + (lane >> 4);
            uint32_t b[4];
            ldsm4_t(b, svb + (np >> 2) * Cfg::HALF_BYTES + key * 128 + ((chunk ^ (key & 7)) << 4));
            mma_16816<T>(oacc[2 * np], a, b[0], b[1]);
            mma_16816<T>(oacc[2 * np + 1], a, b[2], b[3]);
          }
        }
      }
      ++taken;
      __syncwarp();  // every lane has read the stage
      issue();
    }

#pragma unroll
    for (int o = 1; o < 4; o <<= 1) {
      la += __shfl_xor_sync(0xffffffffu, la, o);
      lb += __shfl_xor_sync(0xffffffffu, lb, o);
    }
    const bool begins = cw.k0 == 0, ends = cw.k1 == cw.blocks, finished = begins && ends;
    const int64_t piece = 2 * share + (begins ? 1 : 0);
    if constexpr (WS) {
      if (!ok) continue;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int r = g + 8 * i;
        if (r >= rows) continue;
        const float m = i ? mb : ma, l = i ? lb : la;
        const int tok = r / rows_of_n, head = cw.h * p.group + (r - tok * rows_of_n);
        const int64_t token = cw.s.first + tok;
        if (finished && p.row_ml == nullptr) {
          const float inv = l == 0.f ? 0.f : 1.f / l;
          T* dst = static_cast<T*>(p.o.ptr) + token * p.o.token + head * p.o.head + t4 * 2;
#pragma unroll
          for (int n = 0; n < NT; ++n)
            if (n * 8 < c.head_dim) *reinterpret_cast<uint32_t*>(dst + n * 8) = pack2<T>(oacc[n][2 * i] * inv, oacc[n][2 * i + 1] * inv);
        } else {
          const int64_t row = int64_t(p.prefix_slots) * c.tokens * p.q_heads + token * p.q_heads + head;
          float2* ml = finished ? p.row_ml + row : p.piece_ml + piece * KS_ROWS + r;
          float* po = (finished ? p.row_o + row * c.head_dim : p.piece_o + (piece * KS_ROWS + r) * c.head_dim) + t4 * 2;
          // (scores that are all NaN leave the maximum at -inf: their NaN sum must not be taken for an empty state)
          if (t4 == 0) *ml = make_float2(l == l ? m : 0.f, l);
#pragma unroll
          for (int n = 0; n < NT; ++n)
            if (n * 8 < c.head_dim) *reinterpret_cast<float2*>(po + n * 8) = make_float2(oacc[n][2 * i], oacc[n][2 * i + 1]);
        }
      }
      continue;
    }
    // the warps' states meet: maximum and sum first, then the products, each scaled to the common maximum
    if (t4 == 0) {
      // (scores that are all NaN leave the maximum at -inf: their NaN sum must not be taken for an empty state)
      merge_ml[warp * KS_ROWS + g] = make_float2(la == la ? ma : 0.f, la);
      merge_ml[warp * KS_ROWS + g + 8] = make_float2(lb == lb ? mb : 0.f, lb);
    }
    // (16-byte vectors swizzled by row, so that the eight rows of a store lie in different banks)
    float* slot_o = merge_o + (warp & 3) * KS_ROWS * HDP;
    auto at = [&](int row, int i) { return slot_o + row * HDP + (((i * 2 + (t4 >> 1)) ^ g) << 2) + (t4 & 1) * 2; };
    if (WARPS == 4 || warp >= 4) {
#pragma unroll
      for (int i = 0; i < NT; ++i) {
        *reinterpret_cast<float2*>(at(g, i)) = make_float2(oacc[i][0], oacc[i][1]);
        *reinterpret_cast<float2*>(at(g + 8, i)) = make_float2(oacc[i][2], oacc[i][3]);
      }
    }
    if constexpr (WARPS > 4) {  // eight warps: the upper four's states join the lower four's
      __syncthreads();
      if (warp < 4) {
        const float2 xa2 = merge_ml[(warp + 4) * KS_ROWS + g], xb2 = merge_ml[(warp + 4) * KS_ROWS + g + 8];
        const float2 ya2 = merge_ml[warp * KS_ROWS + g], yb2 = merge_ml[warp * KS_ROWS + g + 8];
        const float na = fmaxf(xa2.x, ya2.x), nb = fmaxf(xb2.x, yb2.x);
        const float ea = xa2.x == -INFINITY ? 0.f : exp2_fast(xa2.x - na), eb = xb2.x == -INFINITY ? 0.f : exp2_fast(xb2.x - nb);
        const float fa = ya2.x == -INFINITY ? 0.f : exp2_fast(ya2.x - na), fb = yb2.x == -INFINITY ? 0.f : exp2_fast(yb2.x - nb);
#pragma unroll
        for (int i = 0; i < NT; ++i) {
          float2* pa = reinterpret_cast<float2*>(at(g, i));
          float2* pb = reinterpret_cast<float2*>(at(g + 8, i));
          const float2 va = *pa, vb = *pb;
          *pa = make_float2(oacc[i][0] * fa + va.x * ea, oacc[i][1] * fa + va.y * ea);
          *pb = make_float2(oacc[i][2] * fb + vb.x * eb, oacc[i][3] * fb + vb.y * eb);
        }
        __syncwarp();
        if (t4 == 0) {
          merge_ml[warp * KS_ROWS + g] = make_float2(na, ya2.y * fa + xa2.y * ea);
          merge_ml[warp * KS_ROWS + g + 8] = make_float2(nb, yb2.y * fb + xb2.y * eb);
        }
      }
    }
    __syncthreads();
    const int vecs = c.head_dim >> 2;
    for (int it = threadIdx.x; it < rows * vecs; it += Cfg::THREADS) {
      const int r = it / vecs, col = (it - r * vecs) << 2;
      float m = -INFINITY, l = 0.f;
#pragma unroll
      for (int w = 0; w < 4; ++w) m = fmaxf(m, merge_ml[w * KS_ROWS + r].x);
      float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const float2 ml = merge_ml[w * KS_ROWS + r];
        const float e = ml.x == -INFINITY ? 0.f : exp2_fast(ml.x - m);
        const float4 v = *reinterpret_cast<const float4*>(merge_o + (w * KS_ROWS + r) * HDP + (col ^ ((r & 7) << 2)));
        l += e * ml.y;
        o.x += e * v.x;
        o.y += e * v.y;
        o.z += e * v.z;
        o.w += e * v.w;
      }
      const int tok = r / rows_of_n, head = cw.h * p.group + (r - tok * rows_of_n);
      const int64_t token = cw.s.first + tok;
      if (finished && p.row_ml == nullptr) {
        const float inv = l == 0.f ? 0.f : 1.f / l;
        uint2 w2 = make_uint2(pack2<T>(o.x * inv, o.y * inv), pack2<T>(o.z * inv, o.w * inv));
        *reinterpret_cast<uint2*>(static_cast<T*>(p.o.ptr) + token * p.o.token + head * p.o.head + col) = w2;
      } else {
        float2* ml;
        float* po;
        if (finished) {
          const int64_t row = int64_t(p.prefix_slots) * c.tokens * p.q_heads + token * p.q_heads + head;
          ml = p.row_ml + row;
          po = p.row_o + row * c.head_dim;
        } else {
          ml = p.piece_ml + piece * KS_ROWS + r;
          po = p.piece_o + (piece * KS_ROWS + r) * c.head_dim;
        }
        if (col == 0) *ml = make_float2(m, l);
        *reinterpret_cast<float4*>(po + col) = o;
      }
    }
    __syncthreads();
  }
  // a wait has run out: behind this warp's copies in flight, which must not outlive the CTA
  if (!ok)
    for (; taken != issued; ++taken)
      mbar_wait_bounded(&bar[taken % KS_STAGES], (taken / KS_STAGES) & 1, &g_error_word, DEV_ERR_WAIT_TIMEOUT);
  // launched as a dependent of the prefix's kernel, this one must not be complete before it: the join waits for this
  // one only
  asm volatile("griddepcontrol.wait;" ::: "memory");
}

// One row's states, `count` of them, state i at (ml(i), o(i)): the lanes of a warp take a 16-byte vector of the row
// each, the warp every `stride`-th state from `begin`; maximum first, so that the loads of the products do not
// wait for one another.
struct KsRow {
  float m, l;
  float4 o;
};
template <typename ML, typename O>
__device__ __forceinline__ KsRow ks_join_states(int begin, int stride, int count, int lane, bool on, ML ml, O o) {
  KsRow r{-INFINITY, 0.f, make_float4(0.f, 0.f, 0.f, 0.f)};
  for (int i = begin + lane * stride; i < count; i += 32 * stride) r.m = fmaxf(r.m, ml(i)->x);
  r.m = warp_max(r.m);
#pragma unroll 4
  for (int i = begin; i < count; i += stride) {
    const float2 s = *ml(i);
    const bool there = s.x != -INFINITY;
    const float4 v = there && on ? *reinterpret_cast<const float4*>(o(i)) : make_float4(0.f, 0.f, 0.f, 0.f);
    const float e = there ? exp2_fast(s.x - r.m) : 0.f;
    r.l += e * s.y;
    r.o.x += e * v.x;
    r.o.y += e * v.y;
    r.o.z += e * v.z;
    r.o.w += e * v.w;
  }
  return r;
}
__device__ __forceinline__ void ks_join_two(KsRow& a, const KsRow& b) {
  const float n = fmaxf(a.m, b.m);
  const float ea = a.m == -INFINITY ? 0.f : exp2_fast(a.m - n), eb = b.m == -INFINITY ? 0.f : exp2_fast(b.m - n);
  a.m = n;
  a.l = a.l * ea + b.l * eb;
  a.o.x = a.o.x * ea + b.o.x * eb;
  a.o.y = a.o.y * ea + b.o.y * eb;
  a.o.z = a.o.z * ea + b.o.z * eb;
  a.o.w = a.o.w * ea + b.o.w * eb;
}
template <typename T>
__device__ __forceinline__ void ks_store_row(const KsRow& r, T* dst) {
  const float inv = r.l == 0.f ? 0.f : 1.f / r.l;
  *reinterpret_cast<uint2*>(dst) = make_uint2(pack2<T>(r.o.x * inv, r.o.y * inv), pack2<T>(r.o.z * inv, r.o.w * inv));
}

// Joins what the step kernel left in pieces: one CTA a (sequence, key head) pair, its eight warps shared out over
// the pair's rows (several a row when the rows are few).  Rows of pairs without a key become zero (they are
// in nobody's share).  With a prefix every row also takes in the states of the prefix's ranges.
template <typename T, int BK>
__global__ void __launch_bounds__(256) kv_step_join_kernel(const KsParams p) {
  __shared__ int64_t sums[8][2];
  __shared__ KsRow part[8][32];
  const KvView& c = p.c;
  const int64_t b = blockIdx.x / c.kv_heads;
  const int h = int(blockIdx.x - b * c.kv_heads);
  // blocks of all sequences, and of those before b
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  int64_t total = 0, before = 0;
  for (int64_t i = tid; i < c.batch; i += 256) {
    const int64_t n = int64_t(ks_blocks<BK>(c, kv_span(c, i), p.window, p.sinks)) * c.kv_heads;
    total += n;
    if (i < b) before += n;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    total += __shfl_xor_sync(0xffffffffu, total, o);
    before += __shfl_xor_sync(0xffffffffu, before, o);
  }
  if (lane == 0) {
    sums[warp][0] = total;
    sums[warp][1] = before;
  }
  __syncthreads();
  total = before = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    total += sums[i][0];
    before += sums[i][1];
  }
  const SeqSpan s = kv_span(c, b);
  const int32_t blocks = ks_blocks<BK>(c, s, p.window, p.sinks);
  const int64_t per = ks_share(total, p.shares);
  const int64_t first = before + int64_t(h) * blocks;
  const int64_t c0 = first / per, c1 = blocks > 0 ? (first + blocks - 1) / per : c0;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const bool whole = blocks > 0 && c0 == c1;
  if (whole && p.row_ml == nullptr) return;
  const int rows = p.group * s.n;
  if (rows == 0) return;
  const int64_t slot_rows = c.tokens * p.q_heads;
  // states of a row: those of the prefix's ranges, the own one if one CTA finished the pair, else the pieces
  const int shared_n = p.row_ml != nullptr ? p.prefix_slots + (whole ? 1 : 0) : 0;
  const int count = shared_n + (blocks > 0 && !whole ? int(c1 - c0) + 1 : 0);
  int per_row = 1;  // warps a row
  while (per_row * 2 * rows <= 8) per_row *= 2;
  const int at_once = 8 / per_row, sub = warp % per_row, col = lane * 4;
  const bool on = col < c.head_dim;
  for (int r0 = 0; r0 < rows; r0 += at_once) {
    const int r = r0 + warp / per_row;
    const bool live = r < rows;
    const int tok = r / p.group, head = h * p.group + (r - tok * p.group);
    const int64_t token = s.first + tok, row = token * p.q_heads + head;
    auto piece = [&](int i) { return (2 * (c0 + i) + (i == 0 ? 1 : 0)) * p.piece_rows + r; };
    KsRow x{-INFINITY, 0.f, make_float4(0.f, 0.f, 0.f, 0.f)};
    if (live)
      x = ks_join_states(
          sub, per_row, count, lane, on,
          [&](int i) { return i < shared_n ? p.row_ml + i * slot_rows + row : p.piece_ml + piece(i - shared_n); },
          [&](int i) {
            return (i < shared_n ? p.row_o + (i * slot_rows + row) * c.head_dim : p.piece_o + piece(i - shared_n) * c.head_dim) + col;
          });
    if (per_row > 1) {
      part[warp][lane] = x;
      __syncthreads();
      if (sub == 0)
        for (int i = 1; i < per_row; ++i) ks_join_two(x, part[warp + i][lane]);
      __syncthreads();
    }
    if (live && sub == 0 && on) ks_store_row(x, static_cast<T*>(p.o.ptr) + token * p.o.token + head * p.o.head + col);
  }
}

}  // namespace lng
