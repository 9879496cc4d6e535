// Attention of few rows over the 8-bit cache: decoding and the verification of drafts, up to 32 (token, head) rows a key
// head.
//
// kv_step_kernel's plan (kv_step.cuh): all blocks of 32 visible keys in one line, cut into equal shares; each
// warp streams its blocks through a ring of its own that an elected lane fills by TMA; cut pairs are joined by
// kv_step_join_kernel.  What differs is what a block is: half the bytes, and e4m3 under exponents, which makes the
// conversion to the products' type the larger part of the work.
//
// Products in fp16 (mma.sync m16n8k16): e4m3 is exact in it, and a row of queries is scaled by a power of two so that its
// largest value lies in [2^14, 2^15) (fp16 queries are taken as they are).  Keys and values are the A operands,
// S^T = K Q^T and O^T = V^T P^T, so that a converted fragment serves all rows, eight a product: NR = 1, 2 or 4 groups of
// eight.  (With the rows as the A operand, 16 at least, a step of 64 sequences with 4 rows a key head took 208 us; so it
// takes 195.)  P^T, whose keys stand along the wrong axis of the accumulators, is turned by movmatrix.  The
// contraction may run over columns, and over keys, in any order, so fragments are read where they lie: a lane takes 16
// consecutive bytes of a key (its columns of four products), and 16 of a value row for each of its four keys.  Keys are put
// to the products' rows so that eight lanes always meet eight different 16-byte banks (key_of).
//
// Exponents: keys' go into the scores' factor, one a tile of 8 keys (pages hold 8 at least).  Values' go into the
// exponential: with u = score + exponent in base 2, weights 2^(u - M) do not overflow fp16 whatever the pages' exponents, their
// products with the bare e4m3 values need no scaling, and the sum takes 2^-exponent back:
// o = sum w v / sum w 2^-exponent.  M is set K8_ROOM = 7 below the largest u, and follows it only when that has grown past M by
// K8_TOP = 15 (weights reach 2^15 at most), which a vote over the lanes' own values tells: the maximum over the lanes is formed
// only then.  Weights are rounded to fp16 once, their sum is not.  The largest is 2^7 at least, so a key keeps all 11 bits of its
// weight while its u lies up to 21 below the row's largest, loses a bit a power of two below that, and counts
// as zero beside the values from 32 on: it may be as likely as any, if another page's exponent is that much larger.
//
// Measured, one token a sequence: 64 sequences of 500 to 16000 keys, 32 query and 8 key heads of 128 (1.12 GB): 194 us, 5.8 TB/s
// (0.89 of the measured copy rate), now bound by the loads; one sequence of 4096 keys, 4 key heads of 64: 16.5 us, latency.
// With 32 rows the registers do not suffice (heads of 128: 132 and 196 bytes of spill stores in fp16 and bf16, heads of 64: 4); the
// forms for fewer rows keep everything.
#pragma once

#include "kv8.cuh"
#include "kv_step.cuh"

namespace lng {

// HDP: head size padded to 64 or 128; NR: groups of eight rows.
template <int HDP, int NR>
struct K8sCfg {
  static constexpr int BK = 32, ROWS = 8 * NR;
  static constexpr bool Q_REGS = HDP * NR <= 256;  // query fragments in registers, else in shared memory
  static constexpr int WARPS = NR == 1 ? 12 : 8, THREADS = 32 * WARPS;
  static constexpr uint32_t KV_BYTES = BK * HDP, STAGE_BYTES = 2 * KV_BYTES;
  static constexpr int STAGES = (Q_REGS ? 192 : 128) * 1024 / WARPS / STAGE_BYTES;
  static constexpr uint32_t RING_BYTES = STAGE_BYTES * STAGES, Q_BYTES = Q_REGS ? 0 : ROWS * HDP * 2;  // one warp's
  static constexpr uint32_t MERGE_BYTES = NR <= 2 ? 4 * ROWS * HDP * 4 : 0;  // the products of four warps
  static constexpr size_t SMEM = size_t(WARPS) * (RING_BYTES + Q_BYTES) + MERGE_BYTES + WARPS * ROWS * 8 + WARPS * STAGES * 16 + 64 + 1024;
};

struct K8sParams {
  KsParams s;
  const int8_t *k_exp, *v_exp;
  int64_t k_exp_page, v_exp_page;
};

// The key of a tile of 8 that stands in column n of its products.
template <int HDP>
__device__ __forceinline__ int key_of(int n) {
  return HDP == 128 ? n ^ ((n & 1) << 2) : n ^ ((n >> 1) & 1);
}
// Byte offset of 16-byte piece c of row r of a tile as TMA swizzles it.
template <int HDP>
__device__ __forceinline__ uint32_t k8_at(int r, int c) {
  return HDP == 128 ? uint32_t(r * 128 + ((c ^ (r & 7)) << 4)) : uint32_t(r * 64 + ((c ^ ((r >> 1) & 3)) << 4));
}
__device__ __forceinline__ uint4 k8_lds128(uint32_t a) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a) : "memory");
  return v;
}
__device__ __forceinline__ uint2 k8_lds64(uint32_t a) {
  uint2 v;
  asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(a) : "memory");
  return v;
}

// The exponent by which a row of queries is brought down (its largest magnitude is `most`), and two of its values.
__device__ __forceinline__ int32_t k8_query_exponent(float most) {
  const int32_t e = int32_t(__float_as_uint(most) >> 23) - 127 - 14;
  return e < -100 ? -100 : e;  // (a row below 2^-86 keeps fewer bits; its scores are zero to any precision)
}
template <typename T>
__device__ __forceinline__ uint32_t k8_query(uint32_t two, float down) {
  if constexpr (std::is_same<T, __half>::value) return two;
  const float2 f = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&two));
  return pack2<__half>(f.x * down, f.y * down);
}

// The 8 x 8 matrix of 16-bit values of which lane 4 r + c holds row r, columns 2 c and 2 c + 1, turned.
__device__ __forceinline__ uint32_t k8_turn(uint32_t x) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
  return r;
}

// WS: a share a warp (many pairs), else a share a CTA (few pairs; NR up to 2).
template <typename T, int HDP, int NR, bool WS>
__global__ void __launch_bounds__(K8sCfg<HDP, NR>::THREADS, 1)
    kv8_step_kernel(const __grid_constant__ CUtensorMap tmk, const __grid_constant__ CUtensorMap tmv, const K8sParams pp) {
  using Cfg = K8sCfg<HDP, NR>;
  constexpr int WARPS = Cfg::WARPS, BK = Cfg::BK, STAGES = Cfg::STAGES, ROWS = Cfg::ROWS, KSTEPS = HDP / 16, MT = HDP / 16, ST = BK / 8;
  static_assert(WS || NR <= 2, "shares of a CTA: up to 16 rows");
  extern __shared__ uint8_t ks_smem_raw[];
  uint8_t* base = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(ks_smem_raw) + 1023) & ~uintptr_t(1023));
  float* merge_o = reinterpret_cast<float*>(base + WARPS * (Cfg::RING_BYTES + Cfg::Q_BYTES));  // [4][ROWS][HDP]
  float2* merge_ml = reinterpret_cast<float2*>(reinterpret_cast<uint8_t*>(merge_o) + Cfg::MERGE_BYTES);  // [WARPS][ROWS]
  uint64_t* bars = reinterpret_cast<uint64_t*>(merge_ml + WARPS * ROWS);  // [WARPS][STAGES]
  uint64_t* exps_all = bars + WARPS * STAGES;                             // likewise: four tiles' (key, value) exponents
  __shared__ int64_t warp_tot[WARPS], found[WS ? WARPS : 1][2];
  const KsParams& p = pp.s;
  const KvView& c = p.c;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  uint8_t* ring = base + warp * Cfg::RING_BYTES;
  const uint32_t qs = smem_addr(base + WARPS * Cfg::RING_BYTES + warp * Cfg::Q_BYTES);  // [k step][group][lane] fragments
  uint64_t* bar = bars + warp * STAGES;
  uint16_t* exps = reinterpret_cast<uint16_t*>(exps_all + warp * STAGES);

  if (lane == 0) {
    for (int s = 0; s < STAGES; ++s) mbar_init(&bar[s], 1);
    fence_mbar_init();
    if (warp == 0) {
      tma_prefetch_desc(&tmk);
      tma_prefetch_desc(&tmv);
    }
  }
  constexpr int STRIDE = WS ? 1 : WARPS;
  const int start = WS ? 0 : warp;
  const int64_t share0 = int64_t(blockIdx.x) * (WS ? WARPS : 1), share = share0 + (WS ? warp : 0);
  const KsFound f = ks_find<BK, WS ? WARPS : 1>(c, p.window, p.sinks, Cfg::THREADS, p.shares, warp_tot, found, share0, WS ? warp : 0);
  const int64_t per = ks_share(f.total, p.shares);
  const int64_t p0 = share * per, p1 = p0 + per < f.total ? p0 + per : f.total;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

  KsWalk<BK> ld, cw;
  ld.start(c, p.window, p.sinks, f, p0, p1);
  cw = ld;
  int32_t ld_k = ld.done() ? 0 : ld.k0 + start;
  uint32_t issued = 0, taken = 0;
  // pages of the warp's next blocks of the pair, a piece (of `box` keys) a lane, and their exponents: looked up
  // together, since a look-up of one block's page takes longer than its copies
  const int boxes = BK / p.box, ahead = 32 / boxes;
  int32_t pages = -1, seen = ahead;
  uint32_t piece_exps = 0;  // (key, value) exponents of the piece's page, a byte each
  auto look_up = [&]() {
    const int32_t k = ld_k + (lane / boxes) * STRIDE;
    pages = -1;
    piece_exps = 0;
    if (k < ld.k1) {
      const int32_t key = tile_index(ld.tiles, k) * BK + (lane % boxes) * p.box;
      if (any_needed(ld.span, key, key + p.box)) {
        pages = page_of(c.table + ld.b * c.table_stride, key, c.page_shift, c.num_pages);
        if (pages < 0) {
          kv_range_error();
          pages = int32_t(c.num_pages);  // behind the last page: the copy fills zeros
        } else {
          piece_exps = uint8_t(pp.k_exp[pages * pp.k_exp_page + ld.h]) | uint32_t(uint8_t(pp.v_exp[pages * pp.v_exp_page + ld.h])) << 8;
        }
      }
    }
    seen = 0;
  };
  auto issue = [&]() {
    while (!ld.done() && ld_k >= ld.k1) {
      ld.next(c, p.window, p.sinks);
      if (!ld.done()) ld_k = ld.k0 + start;
      seen = ahead;
    }
    if (ld.done()) return;
    if (seen == ahead) look_up();
    const uint32_t s = issued % STAGES, mine = boxes == 32 ? 0xffffffffu : ((1u << boxes) - 1u);
    const uint32_t there = (__ballot_sync(0xffffffffu, pages >= 0) >> (seen * boxes)) & mine;
    uint8_t* dk = ring + s * Cfg::STAGE_BYTES;
    uint8_t* dv = dk + Cfg::KV_BYTES;
    const int32_t slot0 = (tile_index(ld.tiles, ld_k) * BK) & ((1 << c.page_shift) - 1);
    {  // the block's exponents, one a tile of 8 keys
      const uint32_t e = __shfl_sync(0xffffffffu, piece_exps, (seen * boxes + ((lane & (ST - 1)) * 8) / p.box) & 31);
      if (lane < ST) exps[s * ST + lane] = uint16_t(e);
    }
    if (elect_lane()) mbar_arrive_expect_tx(&bar[s], uint32_t(__popc(there)) * uint32_t(p.box) * HDP * 2);
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
            tma_load_4d(dk + (r + x) * p.box * HDP, &tmk, 0, slot, ld.h, pg[x], &bar[s]);
            tma_load_4d(dv + (r + x) * p.box * HDP, &tmv, 0, slot, ld.h, pg[x], &bar[s]);
          }
      }
      __syncwarp();
    }
    ++issued;
    ++seen;
    ld_k += STRIDE;
  };
#pragma unroll 1
  for (int i = 0; i < STAGES; ++i) issue();

  const int g = lane >> 2, t4 = lane & 3;
  const int key_row = key_of<HDP>(g);                                // of a tile of 8: the lane's key
  const int va = key_of<HDP>(2 * t4), vb = key_of<HDP>(2 * t4 + 1);  // and its rows of values
  bool ok = true;
  for (; !cw.done(); cw.next(c, p.window, p.sinks)) {
    const int32_t rows = p.group * cw.s.n;  // <= ROWS; row r = token r / group, head r % group
    const int32_t pos0 = cw.s.len - cw.s.n;
    // Q fragments: lane (g, t4) holds row g of every group of eight, columns col + {0, 1}, {2, 3} of its 16 for product k.
    // Rows and columns that are not there are zero
    uint32_t qf[Cfg::Q_REGS ? KSTEPS : 1][Cfg::Q_REGS ? NR : 1][2];
    float scale[NR][2];  // of the scores of rows 8 n + 2 t4 and the next
#pragma unroll
    for (int n = 0; n < NR; ++n) {
      const int r = 8 * n + g, tok = r / p.group, hd = r - tok * p.group;
      const T* src = r < rows ? static_cast<const T*>(p.q.ptr) + (cw.s.first + tok) * p.q.token + (cw.h * p.group + hd) * p.q.head : nullptr;
      uint32_t w[KSTEPS][2];
#pragma unroll
      for (int k = 0; k < KSTEPS; k += 2) {
        const int col = (k >> 2) * 64 + t4 * 16 + (k & 3) * 4;
        const uint4 v = src && col < c.head_dim ? *reinterpret_cast<const uint4*>(src + col) : make_uint4(0, 0, 0, 0);
        w[k][0] = v.x, w[k][1] = v.y, w[k + 1][0] = v.z, w[k + 1][1] = v.w;
      }
      float mine = p.scale_log2;
      if constexpr (!std::is_same<T, __half>::value) {
        float top = 0.f;
#pragma unroll
        for (int k = 0; k < KSTEPS; ++k)
#pragma unroll
          for (int y = 0; y < 2; ++y) {
            const float2 v = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&w[k][y]));
            top = fmaxf(top, fmaxf(fabsf(v.x), fabsf(v.y)));
          }
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
        const int32_t e = k8_query_exponent(top);
        const float down = exp2_whole(-e);
        mine *= exp2_whole(e);
#pragma unroll
        for (int k = 0; k < KSTEPS; ++k)
#pragma unroll
          for (int y = 0; y < 2; ++y) w[k][y] = k8_query<T>(w[k][y], down);
      }
      scale[n][0] = __shfl_sync(0xffffffffu, mine, 8 * t4);      // (a lane of row 2 t4)
      scale[n][1] = __shfl_sync(0xffffffffu, mine, 8 * t4 + 4);
#pragma unroll
      for (int k = 0; k < KSTEPS; ++k) {
        if constexpr (Cfg::Q_REGS)
          qf[k][n][0] = w[k][0], qf[k][n][1] = w[k][1];
        else
          asm volatile("st.shared.v2.u32 [%0], {%1, %2};" ::"r"(qs + uint32_t(((k * NR + n) * 32 + lane) * 8)), "r"(w[k][0]), "r"(w[k][1]) : "memory");
      }
    }
    __syncwarp();
    float oacc[MT][NR][4];
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int n = 0; n < NR; ++n)
#pragma unroll
        for (int j = 0; j < 4; ++j) oacc[i][n][j] = 0.f;
    float m[NR][2], l[NR][2];  // of rows 8 n + 2 t4 and the next; l: the lane's keys only
#pragma unroll
    for (int n = 0; n < NR; ++n) m[n][0] = m[n][1] = -INFINITY, l[n][0] = l[n][1] = 0.f;

    for (int32_t k = cw.k0 + start; k < cw.k1; k += STRIDE) {
      const uint32_t s = taken % STAGES;
      if (ok) ok = mbar_wait_bounded(&bar[s], (taken / STAGES) & 1, &g_error_word, DEV_ERR_WAIT_TIMEOUT);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      uint8_t* sk = ring + s * Cfg::STAGE_BYTES;
      uint8_t* sv = sk + Cfg::KV_BYTES;
      const int32_t key0 = tile_index(cw.tiles, k) * BK;
      if (!all_needed(cw.span, key0, key0 + BK)) {
        // values of keys that no row sees may be anything in memory: zero weights must not meet a NaN
        if (!key_needed(cw.span, key0 + lane)) {
#pragma unroll
          for (int i = 0; i < HDP / 16; ++i) *reinterpret_cast<uint4*>(sv + lane * HDP + i * 16) = make_uint4(0, 0, 0, 0);
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // before the next copy into this stage
        __syncwarp();
      }
      const uint32_t skb = smem_addr(sk), svb = smem_addr(sv);
      const uint2 packed = k8_lds64(smem_addr(exps + s * ST));
      // S^T: tile pair i holds keys key_row of tiles 2 i (values 0, 1: rows 2 t4 and the next) and 2 i + 1 (values 2, 3)
      float u[2][NR][4];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
#pragma unroll
        for (int n = 0; n < NR; ++n)
#pragma unroll
          for (int j = 0; j < 4; ++j) u[i][n][j] = 0.f;
#pragma unroll
        for (int hh = 0; hh < HDP / 64; ++hh) {
          const uint4 wa = k8_lds128(skb + k8_at<HDP>(16 * i + key_row, hh * 4 + t4)), wb = k8_lds128(skb + k8_at<HDP>(16 * i + 8 + key_row, hh * 4 + t4));
          const uint32_t xa[4] = {wa.x, wa.y, wa.z, wa.w}, xb[4] = {wb.x, wb.y, wb.z, wb.w};
#pragma unroll
          for (int kk = 0; kk < 4; ++kk) {
            const uint32_t a[4] = {k8_unpack(xa[kk] & 0xffffu), k8_unpack(xb[kk] & 0xffffu), k8_unpack(xa[kk] >> 16), k8_unpack(xb[kk] >> 16)};
#pragma unroll
            for (int n = 0; n < NR; ++n) {
              if constexpr (Cfg::Q_REGS) {
                mma_16816<__half>(u[i][n], a, qf[hh * 4 + kk][n][0], qf[hh * 4 + kk][n][1]);
              } else {
                const uint2 b = k8_lds64(qs + uint32_t((((hh * 4 + kk) * NR + n) * 32 + lane) * 8));
                mma_16816<__half>(u[i][n], a, b.x, b.y);
              }
            }
          }
        }
      }
      float back[4];  // 2^-(values' exponent) of the four tiles
      float most[NR][2];
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        const uint32_t e = (x < 2 ? packed.x : packed.y) >> (16 * (x & 1));
        const float fk = exp2_whole(int32_t(int8_t(e & 0xff)));
        const int32_t ev = int32_t(int8_t((e >> 8) & 0xff));
        back[x] = exp2_whole(-ev);
        const float add = float(ev);
#pragma unroll
        for (int n = 0; n < NR; ++n)
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            float& v = u[x >> 1][n][2 * (x & 1) + j];
            v = fmaf(v, scale[n][j] * fk, add);
          }
      }
      if (!all_visible(key0, key0 + BK, pos0, cw.s.len - 1, p.window, p.sinks)) {
#pragma unroll
        for (int n = 0; n < NR; ++n)
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const int32_t pos = pos0 + (8 * n + 2 * t4 + j) / p.group;
#pragma unroll
            for (int x = 0; x < 4; ++x)
              if (!key_visible(key0 + 8 * x + key_row, pos, p.window, p.sinks)) u[x >> 1][n][2 * (x & 1) + j] = -INFINITY;
          }
      }
      bool grow = false;
#pragma unroll
      for (int n = 0; n < NR; ++n)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          most[n][j] = fmaxf(fmaxf(u[0][n][j], u[0][n][2 + j]), fmaxf(u[1][n][j], u[1][n][2 + j]));
          grow = grow || most[n][j] > m[n][j] + K8_TOP;
        }
      if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
        for (int n = 0; n < NR; ++n)
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            float x = most[n][j];
#pragma unroll
            for (int o = 4; o < 32; o <<= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, o));
            x = fmaxf(x - K8_ROOM, m[n][j]);
            const float d = m[n][j] == -INFINITY ? 0.f : exp2_fast(m[n][j] - x);
            m[n][j] = x;
            l[n][j] *= d;
#pragma unroll
            for (int i = 0; i < MT; ++i) {
              oacc[i][n][j] *= d;
              oacc[i][n][2 + j] *= d;
            }
          }
      }
      // weights, and their turned fragments: keys along the products' contraction, a row a lane
      uint32_t pf[2][NR][2];
#pragma unroll
      for (int n = 0; n < NR; ++n) {
        const float ra = m[n][0] == -INFINITY ? 0.f : m[n][0], rb = m[n][1] == -INFINITY ? 0.f : m[n][1];
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          const float wa = exp2_fast(u[x >> 1][n][2 * (x & 1)] - ra), wb = exp2_fast(u[x >> 1][n][2 * (x & 1) + 1] - rb);
          l[n][0] = fmaf(wa, back[x], l[n][0]);
          l[n][1] = fmaf(wb, back[x], l[n][1]);
          pf[x >> 1][n][x & 1] = k8_turn(pack2<__half>(wa, wb));
        }
      }
      // O^T += V^T P^T: product i of the lane's columns 2 i (values 0, 1) and 2 i + 1 (values 2, 3)
#pragma unroll
      for (int kk = 0; kk < 2; ++kk) {
        uint32_t w[4][HDP / 32];  // the lane's columns of its four rows
#pragma unroll
        for (int y = 0; y < 4; ++y) {
          const int r = kk * 16 + (y >> 1) * 8 + ((y & 1) ? vb : va);
          if constexpr (HDP == 128) {
            const uint4 v = k8_lds128(svb + k8_at<HDP>(r, g));
            w[y][0] = v.x, w[y][1] = v.y, w[y][2] = v.z, w[y][3] = v.w;
          } else {
            const uint2 v = k8_lds64(svb + k8_at<HDP>(r, g >> 1) + (g & 1) * 8);
            w[y][0] = v.x, w[y][1] = v.y;
          }
        }
#pragma unroll
        for (int x = 0; x < HDP / 32; ++x) {
          const uint32_t lo0 = __byte_perm(w[0][x], w[1][x], 0x5140), hi0 = __byte_perm(w[0][x], w[1][x], 0x7362);
          const uint32_t lo1 = __byte_perm(w[2][x], w[3][x], 0x5140), hi1 = __byte_perm(w[2][x], w[3][x], 0x7362);
          const uint32_t a0[4] = {k8_unpack(lo0 & 0xffffu), k8_unpack(lo0 >> 16), k8_unpack(lo1 & 0xffffu), k8_unpack(lo1 >> 16)};
          const uint32_t a1[4] = {k8_unpack(hi0 & 0xffffu), k8_unpack(hi0 >> 16), k8_unpack(hi1 & 0xffffu), k8_unpack(hi1 >> 16)};
#pragma unroll
          for (int n = 0; n < NR; ++n) {
            mma_16816<__half>(oacc[2 * x][n], a0, pf[kk][n][0], pf[kk][n][1]);
            mma_16816<__half>(oacc[2 * x + 1][n], a1, pf[kk][n][0], pf[kk][n][1]);
          }
        }
      }
      ++taken;
      __syncwarp();  // every lane has read the stage
      issue();
    }

#pragma unroll
    for (int n = 0; n < NR; ++n)
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) l[n][j] += __shfl_xor_sync(0xffffffffu, l[n][j], o);
    const bool begins = cw.k0 == 0, ends = cw.k1 == cw.blocks, finished = begins && ends;
    const int64_t piece = (2 * share + (begins ? 1 : 0)) * p.piece_rows;
    // of row 8 n + 2 t4 + j the lane holds columns col + [0, HDP / 8): oacc[i][n][j] and [2 + j] are 2 i and 2 i + 1
    const int col = g * (HDP / 8);
    if constexpr (WS) {
      if (!ok) continue;
#pragma unroll
      for (int n = 0; n < NR; ++n)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const int r = 8 * n + 2 * t4 + j;
          if (r >= rows || col >= c.head_dim) continue;
          if (finished) {
            const int tok = r / p.group, head = cw.h * p.group + (r - tok * p.group);
            const float inv = l[n][j] == 0.f ? 0.f : 1.f / l[n][j];
            T* dst = static_cast<T*>(p.o.ptr) + (cw.s.first + tok) * p.o.token + head * p.o.head + col;
#pragma unroll
            for (int i = 0; i < MT; i += 4) {
              uint32_t w[4];
#pragma unroll
              for (int y = 0; y < 4; ++y) w[y] = pack2<T>(oacc[i + y][n][j] * inv, oacc[i + y][n][2 + j] * inv);
              *reinterpret_cast<uint4*>(dst + 2 * i) = make_uint4(w[0], w[1], w[2], w[3]);
            }
          } else {
            // (scores that are all NaN leave the maximum at -inf: their NaN sum must not be taken for an empty state)
            if (g == 0) p.piece_ml[piece + r] = make_float2(l[n][j] == l[n][j] ? m[n][j] : 0.f, l[n][j]);
            float* po = p.piece_o + (piece + r) * c.head_dim + col;
#pragma unroll
            for (int i = 0; i < MT; i += 2)
              *reinterpret_cast<float4*>(po + 2 * i) = make_float4(oacc[i][n][j], oacc[i][n][2 + j], oacc[i + 1][n][j], oacc[i + 1][n][2 + j]);
          }
        }
    } else {
      // the warps' states meet: maxima and sums first, then the products, each scaled to the common maximum, four warps
      // at a time into four slots
#pragma unroll
      for (int n = 0; n < NR; ++n)
#pragma unroll
        for (int j = 0; j < 2; ++j)
          if (g == 0) merge_ml[warp * ROWS + 8 * n + 2 * t4 + j] = make_float2(l[n][j] == l[n][j] ? m[n][j] : 0.f, l[n][j]);
      __syncthreads();
      // (16-byte vectors change places by row and by eight, so that a store's lanes lie in different banks)
      float* slot_o = merge_o + (warp & 3) * ROWS * HDP;
      auto vec_at = [&](int row, int v) { return row * HDP + ((v ^ (row & 7) ^ ((v >> 3) & 7)) << 2); };
#pragma unroll 1
      for (int turn = 0; turn < WARPS / 4; ++turn) {
        if (warp >> 2 == turn) {
#pragma unroll
          for (int n = 0; n < NR; ++n)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              const int r = 8 * n + 2 * t4 + j;
              float top = -INFINITY;
              for (int w = 0; w < WARPS; ++w) top = fmaxf(top, merge_ml[w * ROWS + r].x);
              const float own = merge_ml[warp * ROWS + r].x, e = own == -INFINITY ? 0.f : exp2_fast(own - top);
#pragma unroll
              for (int i = 0; i < MT; i += 2) {
                float4* at = reinterpret_cast<float4*>(slot_o + vec_at(r, (col >> 2) + (i >> 1)));
                float4 v = turn > 0 ? *at : make_float4(0.f, 0.f, 0.f, 0.f);
                v.x += e * oacc[i][n][j];
                v.y += e * oacc[i][n][2 + j];
                v.z += e * oacc[i + 1][n][j];
                v.w += e * oacc[i + 1][n][2 + j];
                *at = v;
              }
            }
        }
        __syncthreads();
      }
      const int vecs = c.head_dim >> 2;
      for (int it = threadIdx.x; it < rows * vecs; it += Cfg::THREADS) {
        const int r = it / vecs, v = it - r * vecs;
        float top = -INFINITY, sum = 0.f;
        for (int w = 0; w < WARPS; ++w) top = fmaxf(top, merge_ml[w * ROWS + r].x);
        for (int w = 0; w < WARPS; ++w) {
          const float2 ml = merge_ml[w * ROWS + r];
          sum += (ml.x == -INFINITY ? 0.f : exp2_fast(ml.x - top)) * ml.y;
        }
        float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          const float4 x = *reinterpret_cast<const float4*>(merge_o + w * ROWS * HDP + vec_at(r, v));
          o.x += x.x;
          o.y += x.y;
          o.z += x.z;
          o.w += x.w;
        }
        if (finished) {
          const int tok = r / p.group, head = cw.h * p.group + (r - tok * p.group);
          const float inv = sum == 0.f ? 0.f : 1.f / sum;
          *reinterpret_cast<uint2*>(static_cast<T*>(p.o.ptr) + (cw.s.first + tok) * p.o.token + head * p.o.head + 4 * v) =
              make_uint2(pack2<T>(o.x * inv, o.y * inv), pack2<T>(o.z * inv, o.w * inv));
        } else {
          if (v == 0) p.piece_ml[piece + r] = make_float2(top, sum);
          *reinterpret_cast<float4*>(p.piece_o + (piece + r) * c.head_dim + 4 * v) = o;
        }
      }
      __syncthreads();
    }
  }
  // a wait has run out: behind this warp's copies in flight, which must not outlive the CTA
  if (!ok)
    for (; taken != issued; ++taken)
      mbar_wait_bounded(&bar[taken % STAGES], (taken / STAGES) & 1, &g_error_word, DEV_ERR_WAIT_TIMEOUT);
}

}  // namespace lng
