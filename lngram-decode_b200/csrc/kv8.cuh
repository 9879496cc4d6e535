// The paged cache in 8 bits: a slot holds e4m3 values under one exponent for each page and head, an int8 power of
// two.  Appending a step's keys and values, and reading the pages back.
#pragma once

#include "kvcache.cuh"

namespace lng {

constexpr int K8_LEAST = -40, K8_MOST = 40;  // the exponents that a page may have
// Attention's weights in fp16: 2^K8_ROOM for a row's largest score when its reference is set, 2^K8_TOP at most before it is set
// again (fp16 ends below 2^16), so that 7 of the 8 powers of two that nothing else needs lie below the smallest weights.
constexpr float K8_ROOM = 7.f, K8_TOP = 15.f;

// A cache in 8 bits: c's strides count bytes, exponents lie at page * *_exp_page + head.
struct Kv8View {
  KvView c;
  int8_t *k_exp, *v_exp;
  int64_t k_exp_page, v_exp_page;
};

// 2^e for e in [-126, 127].
__device__ __forceinline__ float exp2_whole(int32_t e) { return __int_as_float((e + 127) << 23); }

// The least exponent under which values up to a (finite, not negative) stay within e4m3's 448 = 1.75 * 2^8.
__device__ __forceinline__ int32_t k8_exponent(float a) {
  const uint32_t u = __float_as_uint(a);
  const int32_t e = int32_t(u >> 23) - 127 - ((u & 0x7fffffu) <= 0x600000u ? 8 : 7);
  return e < K8_LEAST ? K8_LEAST : e > K8_MOST ? K8_MOST : e;
}
// Two e4m3 bytes, the first in the lower one.
__device__ __forceinline__ uint32_t k8_pack(float lo, float hi) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
  return r;
}
// Two e4m3 bytes as two fp16 values, exactly.
__device__ __forceinline__ uint32_t k8_unpack(uint32_t two) {
  uint32_t r;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"(uint16_t(two)));
  return r;
}
__device__ __forceinline__ float2 k8_floats(uint32_t two) {
  const uint32_t h = k8_unpack(two);
  return __half22float2(*reinterpret_cast<const __half2*>(&h));
}

// ------------------------------------------------------------------ append
// A page's exponent needs the largest value of all its new tokens before the first of them can be rounded, so a CTA
// takes one page that a sequence writes to, keys or values of some of its heads.  An item is two 16-byte vectors of a row
// as in kv_append_kernel, and cos and sin of a token are formed once for all heads, with angles in 64 bits as there.
// Where a page holds 64 tokens at most (KEEP) so many warps take a head that every lane can keep its items, four at most, in
// registers from the rotation over the search for the maximum to the rounding: all loads of a page are in flight at once.
// (Rotating twice instead, which leaves room for three CTAs an SM, took a quarter more.)  Larger pages, and rotations by halves
// that are no multiple of 8, go through chunks of 64 tokens twice, the second time from L1 or L2, a warp a head.
// Measured, 32 prompts of 2048 tokens in a replayed graph: 4 key heads of 64 (100 MB) 41 us, and 85 us with 16 heads of queries
// (268 MB), where the cache in 16 bits takes 36 and 67 us; bound by the length of a CTA's sequence -- lengths, rows, angles, two
// meetings, stores -- at sixteen warps an SM.  One key head: 28 us.  Pages of 256 keys: 81 us, one key head 56 us, since
// warps without a head are idle.  64 tokens: 4 us.
constexpr int K8A_WARPS = 8, K8A_THREADS = 32 * K8A_WARPS, K8A_CHUNK = 64, K8A_KEEP = 4;

struct K8AppendParams {
  Kv8View v;
  KvRows kr, vr;
  int32_t rotary, interleaved;
  int32_t per;         // pages that a sequence touches at most, without cu
  int32_t head_warps;  // warps a head (KEEP)
  int32_t items;       // of a head: head_dim / 16
  uint32_t items_magic;  // i / items = __umulhi(i, items_magic) where items > 1
  int64_t units;
  const int64_t* positions;
  const float* inv_freq;
};

// Where the units of sequence b begin in the line of a ragged step: no sequence of n tokens touches more than
// ceil((n + 1) / page) + 1 pages, which is what lies between two beginnings at least.
__device__ __forceinline__ int64_t k8_line(const KvView& c, int64_t b) { return (int64_t(c.cu[b]) >> c.page_shift) + 2 * b; }

// Where cos and sin of pair f of the t-th token stand: rows of `half`, in which two neighbours (16 bytes) change places so
// that eight lanes -- eight items of a token, or four of two -- read eight different banks.
__device__ __forceinline__ int k8_angle_at(int t, int f, int half) {
  const int q = f >> 1;
  return t * half + (((half & 7) ? q : q ^ ((q >> 3) & 3) ^ ((t & 1) << 1)) << 1) + (f & 1);
}

// The 16 values of an item's two vectors (columns c0 and c1 on) of the t-th token, rotated: in pairs across the two, or side
// by side.
template <typename T>
__device__ __forceinline__ void k8_values(uint4 w0, uint4 w1, int c0, int c1, int t, int half, bool rot, bool split, const float2* cs, int rotary,
                                          float (&x)[16]) {
  const bool pair = rot && split && c0 < half;  // (items that are not begin behind 2 * half)
  const T *e0 = reinterpret_cast<const T*>(&w0), *e1 = reinterpret_cast<const T*>(&w1);
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    x[e] = to_f32<T>(e0[e]);
    x[8 + e] = to_f32<T>(e1[e]);
  }
  if (pair) {
#pragma unroll
    for (int e = 0; e < 8; e += 2) {
      const float4 r = *reinterpret_cast<const float4*>(cs + k8_angle_at(t, c0 + e, half));
      const float a = x[e], b = x[8 + e], c = x[e + 1], d = x[9 + e];
      x[e] = a * r.x - b * r.y;
      x[8 + e] = b * r.x + a * r.y;
      x[e + 1] = c * r.z - d * r.w;
      x[9 + e] = d * r.z + c * r.w;
    }
  } else if (rot && !split) {
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int e = 0; e < 8; e += 2) {
        const int j = (h ? c1 : c0) + e;
        if (j < rotary) {
          const float2 r = cs[k8_angle_at(t, j >> 1, half)];
          const float a = x[8 * h + e], b = x[8 * h + e + 1];
          x[8 * h + e] = a * r.x - b * r.y;
          x[8 * h + e + 1] = b * r.x + a * r.y;
        }
      }
  }
}

// The 16 values of an item of the t-th token, rotated, and the first columns of its two halves of 8.
template <typename T>
__device__ __forceinline__ void k8_item(const T* src, int item, int t, int half, bool rot, bool split, bool split_vec, const float2* cs,
                                        int rotary, float (&x)[16], int& c0, int& c1) {
  c0 = item * 16;
  c1 = c0 + 8;
  if (rot && split && !split_vec) {  // halves that are no multiple of 8: value by value
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      const int j = c0 + e;
      if (j < half) {
        const float2 r = cs[k8_angle_at(t, j, half)];
        x[e] = to_f32<T>(src[j]) * r.x - to_f32<T>(src[j + half]) * r.y;
      } else if (j < rotary) {
        const float2 r = cs[k8_angle_at(t, j - half, half)];
        x[e] = to_f32<T>(src[j]) * r.x + to_f32<T>(src[j - half]) * r.y;
      } else {
        x[e] = to_f32<T>(src[j]);
      }
    }
    return;
  }
  if (rot && split && item * 8 < half) c0 = item * 8, c1 = c0 + half;
  k8_values<T>(*reinterpret_cast<const uint4*>(src + c0), *reinterpret_cast<const uint4*>(src + c1), c0, c1, t, half, rot, split, cs, rotary, x);
}

// Cos and sin of the tokens [at0, at0 + here) of a page's new ones.
__device__ __forceinline__ void k8_angles(const K8AppendParams& p, float2* cs, int half, int64_t token0, int32_t j0, int at0, int here) {
  for (int x = threadIdx.x; x < here * half; x += K8A_THREADS) {
    const int t = x / half, f = x - t * half;
    const double pos = p.positions ? double(p.positions[token0 + at0 + t]) : double(j0 + at0 + t);
    const double turns = pos * double(p.inv_freq[f]) * 0.15915494309189533577;  // 1 / (2 pi)
    // (what the angle's rounding to fp32 leaves turns sine and cosine once more: of 10^8 rotated values 130 fall on the other
    // side of a border between two e4m3 values, with sine and cosine of 64-bit angles rounded to fp32 135, without this 229)
    const double halves = 2.0 * (turns - rint(turns));
    const float hi = float(halves), lo = float((halves - double(hi)) * 3.14159265358979323846);
    float sn, cn;
    sincospif(hi, &sn, &cn);
    cs[k8_angle_at(t, f, half)] = make_float2(fmaf(-lo, sn, cn), fmaf(lo, cn, sn));
  }
}

// The largest magnitude of 16 values that counts for the exponent: infinities do not, nor NaN.
__device__ __forceinline__ float k8_most(const float (&x)[16]) {
  float top = 0.f;
#pragma unroll
  for (int e = 0; e < 16; ++e) top = fmaxf(top, fabsf(x[e]));
  if (top == INFINITY) {
    top = 0.f;
#pragma unroll
    for (int e = 0; e < 16; ++e) top = fmaxf(top, fabsf(x[e]) < INFINITY ? fabsf(x[e]) : 0.f);
  }
  return top;
}

// 16 values under the exponent whose negative's power of two is `down`, to columns c0 and c1 of a slot.
__device__ __forceinline__ void k8_store(const float (&x)[16], float down, uint8_t* dst, int c0, int c1) {
  uint32_t w[4];
#pragma unroll
  for (int y = 0; y < 4; ++y) {
    // (an infinity must not be taken for the largest value: its byte is NaN's)
    const float a = x[4 * y] * down, b = x[4 * y + 1] * down, c = x[4 * y + 2] * down, d = x[4 * y + 3] * down;
    w[y] = k8_pack(a, b) | (k8_pack(c, d) << 16);
    if (fmaxf(fmaxf(fabsf(a), fabsf(b)), fmaxf(fabsf(c), fabsf(d))) == INFINITY) {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (fabsf(x[4 * y + e]) == INFINITY) w[y] |= 0x7fu << (8 * e);
    }
  }
  *reinterpret_cast<uint2*>(dst + c0) = make_uint2(w[0], w[1]);
  *reinterpret_cast<uint2*>(dst + c1) = make_uint2(w[2], w[3]);
}

// The exponent of a page and head from its new values' largest and, where it holds earlier ones, its old one; the
// earlier slots again where it grew (the lanes of one warp).
__device__ __forceinline__ int32_t k8_settle(float most, int32_t old, bool held, uint8_t* slots, int64_t slot_stride, int32_t count, int vecs,
                                             int lane, bool mine) {
  const int32_t e = k8_exponent(most);
  if (!held) return e;
  if (old >= e) return old;
  if (mine) {
    const float f = exp2_whole(old - e);
    for (int x = lane; x < count * vecs; x += 32) {
      const int t = x / vecs;
      uint4* at = reinterpret_cast<uint4*>(slots + t * slot_stride + (x - t * vecs) * 16);
      uint4 w = *at;
      uint32_t* words = reinterpret_cast<uint32_t*>(&w);
#pragma unroll
      for (int y = 0; y < 4; ++y) {
        const float2 a = k8_floats(words[y] & 0xffffu), d = k8_floats(words[y] >> 16);
        words[y] = k8_pack(a.x * f, a.y * f) | (k8_pack(d.x * f, d.y * f) << 16);
      }
      *at = w;
    }
  }
  return e;
}

template <typename T, bool KEEP>
__device__ __forceinline__ void kv8_append_page(const K8AppendParams& p, float2* cs) {
  __shared__ uint32_t most[K8A_WARPS];
  const KvView& c = p.v.c;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const bool keys = (blockIdx.y & 1) == 0;
  const int per_cta = KEEP ? K8A_WARPS / p.head_warps : K8A_WARPS;  // heads
  const int head = int(blockIdx.y >> 1) * per_cta + (KEEP ? warp / p.head_warps : warp), sub = KEEP ? warp % p.head_warps : 0;
  int64_t b, i;
  if (c.cu == nullptr) {
    b = blockIdx.x / p.per;
    i = blockIdx.x - b * p.per;
  } else {
    int64_t lo = 0, hi = c.batch;
    const int64_t u = blockIdx.x;
    while (hi - lo > 1) {
      const int64_t mid = (lo + hi) >> 1;
      if (k8_line(c, mid) <= u)
        lo = mid;
      else
        hi = mid;
    }
    b = lo;
    i = u - k8_line(c, b);
  }
  if (i < 0) return;
  const SeqSpan s = kv_span(c, b);
  if (s.n <= 0) return;
  // keys outside the sequence's pages go nowhere
  const int64_t lo = s.pos > 0 ? s.pos : 0, hi = s.pos + s.n < c.capacity ? s.pos + s.n : c.capacity;
  if (i == 0 && threadIdx.x == 0 && (s.pos < 0 || s.pos + s.n > c.capacity)) kv_range_error();
  if (lo >= hi) return;
  const int64_t column = (lo >> c.page_shift) + i, from = column << c.page_shift;
  if (from >= hi) return;
  const int32_t j0 = int32_t(from > lo ? from : lo);
  const int32_t j1 = int32_t(hi < from + (1 << c.page_shift) ? hi : from + (1 << c.page_shift));
  const int32_t slot0 = j0 - int32_t(from), count = j1 - j0;
  const int64_t token0 = s.first + (j0 - s.pos);
  const bool on = head < c.kv_heads;
  const KvRows rows = keys ? p.kr : p.vr;
  const T* const src = static_cast<const T*>(rows.ptr) + token0 * rows.token + (on ? head : 0) * rows.head;
  const int half = keys ? p.rotary >> 1 : 0, vecs = c.head_dim >> 4;
  const bool rot = half > 0, split = !p.interleaved, split_vec = (half & 7) == 0;
  uint4 raw[KEEP ? K8A_KEEP : 1][2];
  const int total = on ? count * p.items : 0;
  // item y of the lane: which token, and its columns
  auto place = [&](int y, int& t, int& c0, int& c1) {
    const int it = (y * p.head_warps + sub) * 32 + lane;
    t = p.items > 1 ? int(__umulhi(uint32_t(it), p.items_magic)) : it;
    const int item = it - t * p.items;
    c0 = item * 16;
    c1 = c0 + 8;
    if (rot && split && item * 8 < half) c0 = item * 8, c1 = c0 + half;
    return it < total;
  };
  if constexpr (KEEP) {  // (the rows' way begins before the page is looked up)
    if (threadIdx.x < K8A_WARPS) most[threadIdx.x] = 0u;
#pragma unroll
    for (int y = 0; y < K8A_KEEP; ++y) {
      int t, c0, c1;
      if (place(y, t, c0, c1)) {
        raw[y][0] = __ldcs(reinterpret_cast<const uint4*>(src + t * rows.token + c0));
        raw[y][1] = __ldcs(reinterpret_cast<const uint4*>(src + t * rows.token + c1));
      }
    }
  }
  const int32_t page = page_of(c.table + b * c.table_stride, j0, c.page_shift, c.num_pages);
  if (page < 0) {
    kv_range_error();
    return;
  }
  const int64_t slot_stride = keys ? c.k_slot : c.v_slot;
  uint8_t* const slots = static_cast<uint8_t*>(keys ? c.k : c.v) + page * (keys ? c.k_page : c.v_page) + (on ? head : 0) * (keys ? c.k_head : c.v_head);
  int8_t* const exp = (keys ? p.v.k_exp + page * p.v.k_exp_page : p.v.v_exp + page * p.v.v_exp_page) + (on ? head : 0);
  const int32_t old = slot0 > 0 ? *exp : 0;
  if constexpr (KEEP) {
    if (rot) k8_angles(p, cs, half, token0, j0, 0, count);
    __syncthreads();
    float x[K8A_KEEP][16], top = 0.f;
#pragma unroll
    for (int y = 0; y < K8A_KEEP; ++y) {
      int t, c0, c1;
      if (place(y, t, c0, c1)) {
        k8_values<T>(raw[y][0], raw[y][1], c0, c1, t, half, rot, split, cs, p.rotary, x[y]);
        top = fmaxf(top, k8_most(x[y]));
      }
    }
    top = warp_max(top);
    if (lane == 0) atomicMax(&most[warp / p.head_warps], __float_as_uint(top));  // (not negative: they order as their bits)
    __syncthreads();
    if (!on) return;
    const int32_t e = k8_settle(__uint_as_float(most[warp / p.head_warps]), old, slot0 > 0, slots, slot_stride, slot0, vecs, lane, sub == 0);
    if (sub == 0 && lane == 0) *exp = int8_t(e);
    const float down = exp2_whole(-e);
#pragma unroll
    for (int y = 0; y < K8A_KEEP; ++y) {
      int t, c0, c1;
      if (place(y, t, c0, c1)) k8_store(x[y], down, slots + (slot0 + t) * slot_stride, c0, c1);
    }
  } else {
    // a warp a head; passes over the tokens in chunks: the maximum, then the rounding
    const int chunks = (count + K8A_CHUNK - 1) / K8A_CHUNK;
    float top = 0.f, down = 1.f;
#pragma unroll 1
    for (int pass = 0; pass < 2; ++pass) {
#pragma unroll 1
      for (int ch = 0; ch < chunks; ++ch) {
        const int at0 = ch * K8A_CHUNK, here = min(K8A_CHUNK, count - at0);
        if (rot && (pass == 0 || chunks > 1)) {
          __syncthreads();
          k8_angles(p, cs, half, token0, j0, at0, here);
          __syncthreads();
        }
        for (int it = lane; on && it < here * p.items; it += 32) {
          const int t = it / p.items, item = it - t * p.items;
          float x[16];
          int c0, c1;
          k8_item<T>(src + (at0 + t) * rows.token, item, t, half, rot, split, split_vec, cs, p.rotary, x, c0, c1);
          if (pass == 0)
            top = fmaxf(top, k8_most(x));
          else
            k8_store(x, down, slots + (slot0 + at0 + t) * slot_stride, c0, c1);
        }
      }
      if (pass == 0 && on) {
        const int32_t e = k8_settle(warp_max(top), old, slot0 > 0, slots, slot_stride, slot0, vecs, lane, true);
        __syncwarp();
        if (lane == 0) *exp = int8_t(e);
        down = exp2_whole(-e);
      }
    }
  }
}

template <typename T, bool KEEP>
__global__ void __launch_bounds__(K8A_THREADS, KEEP ? 2 : 4) kv8_append_kernel(const K8AppendParams p) {
  extern __shared__ float2 k8_cs[];  // [tokens][rotary / 2]
  kv8_append_page<T, KEEP>(p, k8_cs);
  // launched beside the queries' kernel, this one must not be complete before it: what follows waits for this one only
  asm volatile("griddepcontrol.wait;" ::: "memory");
}

// ------------------------------------------------------------------ reading back
// Memory bound: a byte in, two out.  A thread takes 16 bytes of a slot; keys (blocks with y = 0) and values in one launch.
struct K8ValuesParams {
  const uint8_t* pages[2];
  int64_t page[2], head[2], slot[2], exp_page[2];
  const int8_t* exps[2];
  uint4* out[2];
  int32_t heads, page_shift, vecs;
  int64_t total;
};
__global__ void __launch_bounds__(256) kv8_values_kernel(const __grid_constant__ K8ValuesParams p) {
  const int which = blockIdx.y;
  const int64_t x = int64_t(blockIdx.x) * 256 + threadIdx.x;
  if (x >= p.total || p.out[which] == nullptr) return;
  const int64_t row = x / p.vecs;  // (page, head, slot)
  const int32_t s = int32_t(row & ((1 << p.page_shift) - 1));
  const int64_t ph = row >> p.page_shift, pg = ph / p.heads;
  const int32_t h = int32_t(ph - pg * p.heads);
  const uint4 w = __ldcs(reinterpret_cast<const uint4*>(p.pages[which] + pg * p.page[which] + h * p.head[which] + s * p.slot[which] +
                                                        (x - row * p.vecs) * 16));
  const float f = exp2_whole(p.exps[which][pg * p.exp_page[which] + h]);
  const uint32_t words[4] = {w.x, w.y, w.z, w.w};
  uint32_t r[8];
#pragma unroll
  for (int y = 0; y < 4; ++y) {
    const float2 a = k8_floats(words[y] & 0xffffu), d = k8_floats(words[y] >> 16);
    const __nv_bfloat162 u = __floats2bfloat162_rn(a.x * f, a.y * f), v = __floats2bfloat162_rn(d.x * f, d.y * f);
    r[2 * y] = *reinterpret_cast<const uint32_t*>(&u);
    r[2 * y + 1] = *reinterpret_cast<const uint32_t*>(&v);
  }
  __stcs(p.out[which] + 2 * x, make_uint4(r[0], r[1], r[2], r[3]));
  __stcs(p.out[which] + 2 * x + 1, make_uint4(r[4], r[5], r[6], r[7]));
}

}  // namespace lng
