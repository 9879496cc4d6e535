// Attention of few rows over the 8-bit cache: decoding and the verification of a few drafts, at most 16
// (token, head) rows a key head.
//
// kv_step_kernel's plan (kv_step.cuh): all blocks of 32 visible keys in one line, cut into equal shares; each
// warp streams its blocks through a ring of its own that an elected lane fills by TMA; cut pairs are joined by
// kv_step_join_kernel.  What differs is what a block is: half the bytes, and e4m3 under exponents.
//
// Products in fp16 (mma.sync m16n8k16): e4m3 is exact in it, and a row of queries is scaled by a power of two so that its
// largest value lies in [2^14, 2^15) (fp16 queries are taken as they are).  The contraction may run over columns, and
// over keys, in any order, so fragments are read where they lie: a lane takes 16 consecutive bytes of a key (its
// columns of four products), 16 of a value row for each of its four keys (a column of sixteen products).  Keys are put
// to the products' columns so that eight lanes always meet eight different 16-byte banks (key_of).
//
// Exponents: keys' go into the scores' factor, one a tile of 8 keys (pages hold 8 at least).  Values' go into the
// exponential: with u = score + exponent in base 2, weights 2^(u - max u) are at most 1 and fit fp16 whatever the
// pages' exponents, their products with the bare e4m3 values need no scaling, and the sum takes 2^-exponent
// back: o = sum w v / sum w 2^-exponent.  Weights are rounded to fp16 once, their sum is not.
#pragma once

#include "kv8.cuh"
#include "kv_step.cuh"

namespace lng {

template <int HDP>  // head size padded to 64 or 128
struct K8sCfg {
  static constexpr int BK = 32, WARPS = 8, THREADS = 32 * WARPS, STAGES = HDP == 128 ? 3 : 6;
  static constexpr uint32_t KV_BYTES = BK * HDP, STAGE_BYTES = 2 * KV_BYTES, RING_BYTES = STAGE_BYTES * STAGES;
  static constexpr uint32_t MERGE_BYTES = 4 * KS_ROWS * HDP * 4;  // the products of four warps
  static constexpr size_t SMEM = size_t(WARPS) * RING_BYTES + MERGE_BYTES + WARPS * KS_ROWS * 8 + WARPS * STAGES * 16 + 64 + 1024;
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

// WS: a share a warp (many pairs), else a share a CTA (few pairs).
template <typename T, int HDP, bool WS>
__global__ void __launch_bounds__(K8sCfg<HDP>::THREADS, 1)
    kv8_step_kernel(const __grid_constant__ CUtensorMap tmk, const __grid_constant__ CUtensorMap tmv, const K8sParams pp) {
  using Cfg = K8sCfg<HDP>;
  constexpr int WARPS = Cfg::WARPS, BK = Cfg::BK, STAGES = Cfg::STAGES, KSTEPS = HDP / 16, NT = HDP / 8, ST = BK / 8;
  extern __shared__ uint8_t ks_smem_raw[];
  uint8_t* base = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(ks_smem_raw) + 1023) & ~uintptr_t(1023));
  float* merge_o = reinterpret_cast<float*>(base + WARPS * Cfg::RING_BYTES);  // [4][16][HDP]
  float2* merge_ml = reinterpret_cast<float2*>(reinterpret_cast<uint8_t*>(merge_o) + Cfg::MERGE_BYTES);  // [WARPS][16]
  uint64_t* bars = reinterpret_cast<uint64_t*>(merge_ml + WARPS * KS_ROWS);   // [WARPS][STAGES]
  uint64_t* exps_all = bars + WARPS * STAGES;                                 // likewise: four tiles' (key, value) exponents
  __shared__ int64_t warp_tot[WARPS], found[WS ? WARPS : 1][2];
  const KsParams& p = pp.s;
  const KvView& c = p.c;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  uint8_t* ring = base + warp * Cfg::RING_BYTES;
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
  const int rows_of_n = p.group;
  const int key_row = key_of<HDP>(g);                                  // of a tile of 8: the lane's key
  const int va = key_of<HDP>(2 * t4), vb = key_of<HDP>(2 * t4 + 1);    // and its rows of values
  bool ok = true;
  for (; !cw.done(); cw.next(c, p.window, p.sinks)) {
    const int32_t rows = rows_of_n * cw.s.n;  // <= 16
    const int32_t pos0 = cw.s.len - cw.s.n;
    // Q fragments (row r = token r / group, head r % group); rows and columns that are not there are zero.  Product kk
    // contracts columns col(kk) + {0, 1} (first halves) and + {2, 3} of every lane's 16
    uint32_t qf[KSTEPS][4];
    float fa = p.scale_log2, fb = p.scale_log2;
    {
      float top[2] = {0.f, 0.f};
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int r = g + 8 * i;
        const int tok = r / rows_of_n, hd = r - tok * rows_of_n;
        const T* src = r < rows ? static_cast<const T*>(p.q.ptr) + (cw.s.first + tok) * p.q.token + (cw.h * p.group + hd) * p.q.head : nullptr;
#pragma unroll
        for (int k = 0; k < KSTEPS; k += 2) {
          const int col = (k >> 2) * 64 + t4 * 16 + (k & 3) * 4;
          const uint4 w = src && col < c.head_dim ? *reinterpret_cast<const uint4*>(src + col) : make_uint4(0, 0, 0, 0);
          qf[k][i] = w.x;
          qf[k][i + 2] = w.y;
          qf[k + 1][i] = w.z;
          qf[k + 1][i + 2] = w.w;
        }
        if constexpr (!std::is_same<T, __half>::value) {
#pragma unroll
          for (int k = 0; k < KSTEPS; ++k)
#pragma unroll
            for (int y = i; y < 4; y += 2) {
              const float2 v = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&qf[k][y]));
              top[i] = fmaxf(top[i], fmaxf(fabsf(v.x), fabsf(v.y)));
            }
          top[i] = fmaxf(top[i], __shfl_xor_sync(0xffffffffu, top[i], 1));
          top[i] = fmaxf(top[i], __shfl_xor_sync(0xffffffffu, top[i], 2));
          const int32_t e = k8_query_exponent(top[i]);
          const float down = exp2_whole(-e);
          (i ? fb : fa) = p.scale_log2 * exp2_whole(e);
#pragma unroll
          for (int k = 0; k < KSTEPS; ++k)
#pragma unroll
            for (int y = i; y < 4; y += 2) qf[k][y] = k8_query<T>(qf[k][y], down);
        }
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
      const uint32_t s = taken % STAGES;
      if (ok) ok = mbar_wait_bounded(&bar[s], (taken / STAGES) & 1, &g_error_word, DEV_ERR_WAIT_TIMEOUT);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      uint8_t* sk = ring + s * Cfg::STAGE_BYTES;
      uint8_t* sv = sk + Cfg::KV_BYTES;
      const int32_t key0 = tile_index(cw.tiles, k) * BK;
      const bool whole = all_needed(cw.span, key0, key0 + BK);
      if (!whole) {
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
      // u = scores in base 2 plus the values' exponents: 16 rows x BK keys
      float sacc[ST][4];
      float back[ST];  // 2^-(values' exponent)
#pragma unroll
      for (int n = 0; n < ST; ++n) {
#pragma unroll
        for (int j = 0; j < 4; ++j) sacc[n][j] = 0.f;
#pragma unroll
        for (int hh = 0; hh < HDP / 64; ++hh) {
          const uint4 w = k8_lds128(skb + k8_at<HDP>(n * 8 + key_row, hh * 4 + t4));
          const uint32_t words[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
          for (int kk = 0; kk < 4; ++kk)
            mma_16816<__half>(sacc[n], qf[hh * 4 + kk], k8_unpack(words[kk] & 0xffffu), k8_unpack(words[kk] >> 16));
        }
        const uint32_t e = (n < 2 ? packed.x : packed.y) >> (16 * (n & 1));
        const float fk = exp2_whole(int32_t(int8_t(e & 0xff)));
        const int32_t ev = int32_t(int8_t((e >> 8) & 0xff));
        back[n] = exp2_whole(-ev);
        const float ga = fa * fk, gb = fb * fk, add = float(ev);
        sacc[n][0] = fmaf(sacc[n][0], ga, add);
        sacc[n][1] = fmaf(sacc[n][1], ga, add);
        sacc[n][2] = fmaf(sacc[n][2], gb, add);
        sacc[n][3] = fmaf(sacc[n][3], gb, add);
      }
      if (!all_visible(key0, key0 + BK, pos0, cw.s.len - 1, p.window, p.sinks)) {
#pragma unroll
        for (int n = 0; n < ST; ++n)
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int32_t key = key0 + n * 8 + ((j & 1) ? vb : va);
            if (!key_visible(key, j < 2 ? pa : pb, p.window, p.sinks)) sacc[n][j] = -INFINITY;
          }
      }
      // running maximum and sum of the two rows
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
      const float na = fmaxf(ma, xa), nb = fmaxf(mb, xb);
      if (__any_sync(0xffffffffu, na > ma || nb > mb)) {
        const float da = ma == -INFINITY ? 0.f : exp2_fast(ma - na), db = mb == -INFINITY ? 0.f : exp2_fast(mb - nb);
        la *= da;
        lb *= db;
#pragma unroll
        for (int i = 0; i < NT; ++i) {
          oacc[i][0] *= da;
          oacc[i][1] *= da;
          oacc[i][2] *= db;
          oacc[i][3] *= db;
        }
        ma = na;
        mb = nb;
      }
      const float ra = ma == -INFINITY ? 0.f : ma, rb = mb == -INFINITY ? 0.f : mb;
#pragma unroll
      for (int n = 0; n < ST; ++n) {
        sacc[n][0] = exp2_fast(sacc[n][0] - ra);
        sacc[n][1] = exp2_fast(sacc[n][1] - ra);
        sacc[n][2] = exp2_fast(sacc[n][2] - rb);
        sacc[n][3] = exp2_fast(sacc[n][3] - rb);
        la = fmaf(sacc[n][0] + sacc[n][1], back[n], la);
        lb = fmaf(sacc[n][2] + sacc[n][3], back[n], lb);
      }
      // O += P V
#pragma unroll
      for (int kk = 0; kk < BK / 16; ++kk) {
        const uint32_t a[4] = {pack2<__half>(sacc[2 * kk][0], sacc[2 * kk][1]), pack2<__half>(sacc[2 * kk][2], sacc[2 * kk][3]),
                               pack2<__half>(sacc[2 * kk + 1][0], sacc[2 * kk + 1][1]), pack2<__half>(sacc[2 * kk + 1][2], sacc[2 * kk + 1][3])};
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
          mma_16816<__half>(oacc[4 * x], a, k8_unpack(lo0 & 0xffffu), k8_unpack(lo1 & 0xffffu));
          mma_16816<__half>(oacc[4 * x + 1], a, k8_unpack(lo0 >> 16), k8_unpack(lo1 >> 16));
          mma_16816<__half>(oacc[4 * x + 2], a, k8_unpack(hi0 & 0xffffu), k8_unpack(hi1 & 0xffffu));
          mma_16816<__half>(oacc[4 * x + 3], a, k8_unpack(hi0 >> 16), k8_unpack(hi1 >> 16));
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
    // of row g (or g + 8) the lane holds columns t4 * NT * 2 + [0, NT) in oacc[.][0] (or [2]) and the NT behind them in the next
    if constexpr (WS) {
      if (!ok) continue;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int r = g + 8 * i;
        if (r >= rows) continue;
        const float m = i ? mb : ma, l = i ? lb : la;
        const int tok = r / rows_of_n, head = cw.h * p.group + (r - tok * rows_of_n);
        const int64_t token = cw.s.first + tok;
        if (finished) {
          const float inv = l == 0.f ? 0.f : 1.f / l;
          T* dst = static_cast<T*>(p.o.ptr) + token * p.o.token + head * p.o.head;
#pragma unroll
          for (int h2 = 0; h2 < 2; ++h2)
#pragma unroll
            for (int n = 0; n < NT; n += 8) {
              const int col = t4 * NT * 2 + h2 * NT + n;
              if (col < c.head_dim) {
                uint32_t w[4];
#pragma unroll
                for (int y = 0; y < 4; ++y)
                  w[y] = pack2<T>(oacc[n + 2 * y][2 * i + h2] * inv, oacc[n + 2 * y + 1][2 * i + h2] * inv);
                *reinterpret_cast<uint4*>(dst + col) = make_uint4(w[0], w[1], w[2], w[3]);
              }
            }
        } else {
          if (t4 == 0) p.piece_ml[piece * KS_ROWS + r] = make_float2(l == l ? m : 0.f, l);
          float* po = p.piece_o + (piece * KS_ROWS + r) * c.head_dim;
#pragma unroll
          for (int h2 = 0; h2 < 2; ++h2)
#pragma unroll
            for (int n = 0; n < NT; n += 4) {
              const int col = t4 * NT * 2 + h2 * NT + n;
              if (col < c.head_dim)
                *reinterpret_cast<float4*>(po + col) =
                    make_float4(oacc[n][2 * i + h2], oacc[n + 1][2 * i + h2], oacc[n + 2][2 * i + h2], oacc[n + 3][2 * i + h2]);
            }
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
    // (16-byte vectors swizzled by row and by eight, so that a store's lanes lie in different banks)
    float* slot_o = merge_o + (warp & 3) * KS_ROWS * HDP;
    auto vec_at = [&](int row, int v) { return row * HDP + (((v & ~7) | ((v ^ row ^ ((v >> 3) << 1)) & 7)) << 2); };
    if (warp >= 4) {
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int h2 = 0; h2 < 2; ++h2)
#pragma unroll
          for (int n = 0; n < NT; n += 4)
            *reinterpret_cast<float4*>(slot_o + vec_at(g + 8 * i, (t4 * NT * 2 + h2 * NT + n) >> 2)) =
                make_float4(oacc[n][2 * i + h2], oacc[n + 1][2 * i + h2], oacc[n + 2][2 * i + h2], oacc[n + 3][2 * i + h2]);
    }
    __syncthreads();
    if (warp < 4) {  // the upper four warps' states join the lower four's
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const float2 x = merge_ml[(warp + 4) * KS_ROWS + g + 8 * i], y = merge_ml[warp * KS_ROWS + g + 8 * i];
        const float n2 = fmaxf(x.x, y.x);
        const float ex = x.x == -INFINITY ? 0.f : exp2_fast(x.x - n2), ey = y.x == -INFINITY ? 0.f : exp2_fast(y.x - n2);
#pragma unroll
        for (int h2 = 0; h2 < 2; ++h2)
#pragma unroll
          for (int n = 0; n < NT; n += 4) {
            float4* at = reinterpret_cast<float4*>(slot_o + vec_at(g + 8 * i, (t4 * NT * 2 + h2 * NT + n) >> 2));
            const float4 v = *at;
            *at = make_float4(oacc[n][2 * i + h2] * ey + v.x * ex, oacc[n + 1][2 * i + h2] * ey + v.y * ex,
                              oacc[n + 2][2 * i + h2] * ey + v.z * ex, oacc[n + 3][2 * i + h2] * ey + v.w * ex);
          }
        __syncwarp();
        if (t4 == 0) merge_ml[warp * KS_ROWS + g + 8 * i] = make_float2(n2, y.y * ey + x.y * ex);
      }
    }
    __syncthreads();
    const int vecs = c.head_dim >> 2;
    for (int it = threadIdx.x; it < rows * vecs; it += Cfg::THREADS) {
      const int r = it / vecs, v = it - r * vecs, col = v << 2;
      float m = -INFINITY, l = 0.f;
#pragma unroll
      for (int w = 0; w < 4; ++w) m = fmaxf(m, merge_ml[w * KS_ROWS + r].x);
      float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const float2 ml = merge_ml[w * KS_ROWS + r];
        const float e = ml.x == -INFINITY ? 0.f : exp2_fast(ml.x - m);
        const float4 x = *reinterpret_cast<const float4*>(merge_o + w * KS_ROWS * HDP + vec_at(r, v));
        l += e * ml.y;
        o.x += e * x.x;
        o.y += e * x.y;
        o.z += e * x.z;
        o.w += e * x.w;
      }
      const int tok = r / rows_of_n, head = cw.h * p.group + (r - tok * rows_of_n);
      const int64_t token = cw.s.first + tok;
      if (finished) {
        const float inv = l == 0.f ? 0.f : 1.f / l;
        *reinterpret_cast<uint2*>(static_cast<T*>(p.o.ptr) + token * p.o.token + head * p.o.head + col) =
            make_uint2(pack2<T>(o.x * inv, o.y * inv), pack2<T>(o.z * inv, o.w * inv));
      } else {
        if (col == 0) p.piece_ml[piece * KS_ROWS + r] = make_float2(m, l);
        *reinterpret_cast<float4*>(p.piece_o + (piece * KS_ROWS + r) * c.head_dim + col) = o;
      }
    }
    __syncthreads();
  }
  // a wait has run out: behind this warp's copies in flight, which must not outlive the CTA
  if (!ok)
    for (; taken != issued; ++taken)
      mbar_wait_bounded(&bar[taken % STAGES], (taken / STAGES) & 1, &g_error_word, DEV_ERR_WAIT_TIMEOUT);
}

}  // namespace lng
