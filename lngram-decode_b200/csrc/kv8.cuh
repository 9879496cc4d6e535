// The paged cache in 8 bits: a slot holds e4m3 values under one exponent for each page and head, an int8 power of
// two.  Appending a step's keys and values, and reading the pages back.
#pragma once

#include "kvcache.cuh"

namespace lng {

constexpr int K8_LEAST = -40, K8_MOST = 40;  // the exponents that a page may have

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
// takes one page that a sequence writes to (keys or values of all heads, or of four heads where the step has few
// pages): pass one forms the values and their maximum a head, pass two forms them again (from L1 or L2: the rows are
// read from memory once) and rounds them.  A warp takes a head and meets no other; an item is two 16-byte
// vectors of a row as in kv_append_kernel, and cos and sin of a chunk of tokens are formed once for all heads,
// with angles in 64 bits as there.
constexpr int K8A_THREADS = 128, K8A_CHUNK = 64, K8A_HEADS = 32;

struct K8AppendParams {
  Kv8View v;
  KvRows kr, vr;
  int32_t rotary, interleaved;
  int32_t per;         // pages that a sequence touches at most, without cu
  int32_t head_chunk;  // heads a CTA (at most K8A_HEADS)
  int32_t items;       // of a head: head_dim / 16
  int64_t units;
  const int64_t* positions;
  const float* inv_freq;
};

// Where the units of sequence b begin in the line of a ragged step: no sequence of n tokens touches more than
// ceil((n + 1) / page) + 1 pages, which is what lies between two beginnings at least.
__device__ __forceinline__ int64_t k8_line(const KvView& c, int64_t b) { return (int64_t(c.cu[b]) >> c.page_shift) + 2 * b; }

// The 16 values of an item, rotated, and the first columns of its two halves of 8.
template <typename T>
__device__ __forceinline__ void k8_item(const T* src, int item, int half, bool rot, bool split, bool split_vec, const float2* cs,
                                        int rotary, float (&x)[16], int& c0, int& c1) {
  c0 = item * 16;
  c1 = c0 + 8;
  if (rot && split && !split_vec) {  // halves that are no multiple of 8: value by value
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      const int j = c0 + e;
      if (j < half) {
        const float2 r = cs[j];
        x[e] = to_f32<T>(src[j]) * r.x - to_f32<T>(src[j + half]) * r.y;
      } else if (j < rotary) {
        const float2 r = cs[j - half];
        x[e] = to_f32<T>(src[j]) * r.x + to_f32<T>(src[j - half]) * r.y;
      } else {
        x[e] = to_f32<T>(src[j]);
      }
    }
    return;
  }
  const bool pair = rot && split && item * 8 < half;
  if (pair) c0 = item * 8, c1 = c0 + half;
  const uint4 w0 = *reinterpret_cast<const uint4*>(src + c0), w1 = *reinterpret_cast<const uint4*>(src + c1);
  const T *e0 = reinterpret_cast<const T*>(&w0), *e1 = reinterpret_cast<const T*>(&w1);
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    x[e] = to_f32<T>(e0[e]);
    x[8 + e] = to_f32<T>(e1[e]);
  }
  if (pair) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float2 r = cs[c0 + e];
      const float a = x[e], b = x[8 + e];
      x[e] = a * r.x - b * r.y;
      x[8 + e] = b * r.x + a * r.y;
    }
  } else if (rot && !split) {
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int e = 0; e < 8; e += 2) {
        const int j = (h ? c1 : c0) + e;
        if (j < rotary) {
          const float2 r = cs[j >> 1];
          const float a = x[8 * h + e], b = x[8 * h + e + 1];
          x[8 * h + e] = a * r.x - b * r.y;
          x[8 * h + e + 1] = b * r.x + a * r.y;
        }
      }
  }
}

template <typename T>
__global__ void __launch_bounds__(K8A_THREADS) kv8_append_kernel(const K8AppendParams p) {
  extern __shared__ float2 k8_cs[];  // [chunk][rotary / 2]
  __shared__ float most[K8A_HEADS];
  __shared__ float down[K8A_HEADS];  // 2^-exponent
  const KvView& c = p.v.c;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const bool keys = (blockIdx.y & 1) == 0;
  const int head0 = int(blockIdx.y >> 1) * p.head_chunk, heads = min(p.head_chunk, c.kv_heads - head0);
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
  const int32_t page = page_of(c.table + b * c.table_stride, j0, c.page_shift, c.num_pages);
  if (page < 0) {
    kv_range_error();
    return;
  }
  const int32_t slot0 = j0 - int32_t(from), count = j1 - j0;
  const int64_t token0 = s.first + (j0 - s.pos);
  const KvRows rows = keys ? p.kr : p.vr;
  uint8_t* const pages = static_cast<uint8_t*>(keys ? c.k : c.v) + page * (keys ? c.k_page : c.v_page);
  const int64_t head_stride = keys ? c.k_head : c.v_head, slot_stride = keys ? c.k_slot : c.v_slot;
  int8_t* const exps = (keys ? p.v.k_exp + page * p.v.k_exp_page : p.v.v_exp + page * p.v.v_exp_page) + head0;
  const int half = keys ? p.rotary >> 1 : 0;
  const bool rot = half > 0, split = !p.interleaved, split_vec = (half & 7) == 0;
  if (threadIdx.x < heads) most[threadIdx.x] = 0.f;
  const int chunks = (count + K8A_CHUNK - 1) / K8A_CHUNK;
  auto angles = [&](int ch) {  // cos and sin of a chunk's tokens
    __syncthreads();
    if (rot) {
      const int here = min(K8A_CHUNK, count - ch * K8A_CHUNK);
      for (int x = threadIdx.x; x < here * half; x += K8A_THREADS) {
        const int t = x / half, f = x - t * half, at = ch * K8A_CHUNK + t;
        const double pos = p.positions ? double(p.positions[token0 + at]) : double(j0 + at);
        const double turns = pos * double(p.inv_freq[f]) * 0.15915494309189533577;  // 1 / (2 pi)
        float sn, cn;
        sincospif(float(2.0 * (turns - rint(turns))), &sn, &cn);
        k8_cs[x] = make_float2(cn, sn);
      }
      __syncthreads();
    }
  };
  // pass one: the largest finite value a head
#pragma unroll 1
  for (int ch = 0; ch < chunks; ++ch) {
    angles(ch);
    const int here = min(K8A_CHUNK, count - ch * K8A_CHUNK);
    for (int h = warp; h < heads; h += K8A_THREADS / 32) {
      float top = 0.f;
      for (int it = lane; it < here * p.items; it += 32) {
        const int t = it / p.items, item = it - t * p.items;
        const T* src = static_cast<const T*>(rows.ptr) + (token0 + ch * K8A_CHUNK + t) * rows.token + (head0 + h) * rows.head;
        float x[16];
        int c0, c1;
        k8_item<T>(src, item, half, rot, split, split_vec, k8_cs + t * half, p.rotary, x, c0, c1);
#pragma unroll
        for (int e = 0; e < 16; ++e) top = fmaxf(top, fabsf(x[e]) < INFINITY ? fabsf(x[e]) : 0.f);
      }
      top = warp_max(top);
      if (lane == 0) most[h] = fmaxf(most[h], top);
      __syncwarp();
    }
  }
  // exponents; earlier slots again where one grew
  for (int h = warp; h < heads; h += K8A_THREADS / 32) {
    int32_t e = k8_exponent(most[h]);
    if (slot0 > 0) {
      const int32_t old = exps[h];
      if (old >= e) {
        e = old;
      } else {
        const float f = exp2_whole(old - e);
        const int vecs = c.head_dim >> 4;
        for (int x = lane; x < slot0 * vecs; x += 32) {
          const int t = x / vecs;
          uint4* at = reinterpret_cast<uint4*>(pages + (head0 + h) * head_stride + t * slot_stride + (x - t * vecs) * 16);
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
    }
    __syncwarp();
    if (lane == 0) {
      exps[h] = int8_t(e);
      down[h] = exp2_whole(-e);
    }
    __syncwarp();
  }
  // pass two
#pragma unroll 1
  for (int ch = 0; ch < chunks; ++ch) {
    if (chunks > 1) angles(ch);
    const int here = min(K8A_CHUNK, count - ch * K8A_CHUNK);
    for (int h = warp; h < heads; h += K8A_THREADS / 32) {
      const float f = down[h];
      for (int it = lane; it < here * p.items; it += 32) {
        const int t = it / p.items, item = it - t * p.items, at = ch * K8A_CHUNK + t;
        const T* src = static_cast<const T*>(rows.ptr) + (token0 + at) * rows.token + (head0 + h) * rows.head;
        float x[16];
        int c0, c1;
        k8_item<T>(src, item, half, rot, split, split_vec, k8_cs + t * half, p.rotary, x, c0, c1);
        uint32_t w[4];
#pragma unroll
        for (int y = 0; y < 4; ++y) {
          // (x * 0 makes NaN of an infinity, which must not be taken for the largest value)
#pragma unroll
          for (int e = 0; e < 4; ++e) x[4 * y + e] = fmaf(x[4 * y + e], 0.f, x[4 * y + e] * f);
          w[y] = k8_pack(x[4 * y], x[4 * y + 1]) | (k8_pack(x[4 * y + 2], x[4 * y + 3]) << 16);
        }
        uint8_t* dst = pages + (head0 + h) * head_stride + (slot0 + at) * slot_stride;
        *reinterpret_cast<uint2*>(dst + c0) = make_uint2(w[0], w[1]);
        *reinterpret_cast<uint2*>(dst + c1) = make_uint2(w[2], w[3]);
      }
    }
  }
}

// ------------------------------------------------------------------ reading back
// Memory bound: a byte in, two out.  A thread takes 16 bytes of a slot.
__global__ void __launch_bounds__(256)
    kv8_values_kernel(const uint8_t* __restrict__ pages, int64_t page, int64_t head, int64_t slot, const int8_t* __restrict__ exps,
                      int64_t exp_page, int32_t heads, int32_t page_shift, int32_t vecs, int64_t total, uint4* __restrict__ out) {
  const int64_t x = int64_t(blockIdx.x) * 256 + threadIdx.x;
  if (x >= total) return;
  const int64_t row = x / vecs;  // (page, head, slot)
  const int32_t s = int32_t(row & ((1 << page_shift) - 1));
  const int64_t ph = row >> page_shift, pg = ph / heads;
  const int32_t h = int32_t(ph - pg * heads);
  const uint4 w = __ldcs(reinterpret_cast<const uint4*>(pages + pg * page + h * head + s * slot + (x - row * vecs) * 16));
  const float f = exp2_whole(exps[pg * exp_page + h]);
  const uint32_t words[4] = {w.x, w.y, w.z, w.w};
  uint32_t r[8];
#pragma unroll
  for (int y = 0; y < 4; ++y) {
    const float2 a = k8_floats(words[y] & 0xffffu), d = k8_floats(words[y] >> 16);
    const __nv_bfloat162 u = __floats2bfloat162_rn(a.x * f, a.y * f), v = __floats2bfloat162_rn(d.x * f, d.y * f);
    r[2 * y] = *reinterpret_cast<const uint32_t*>(&u);
    r[2 * y + 1] = *reinterpret_cast<const uint32_t*>(&v);
  }
  __stcs(out + 2 * x, make_uint4(r[0], r[1], r[2], r[3]));
  __stcs(out + 2 * x + 1, make_uint4(r[4], r[5], r[6], r[7]));
}

}  // namespace lng
