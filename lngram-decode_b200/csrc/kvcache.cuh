// The paged key/value cache of a decode loop: appending a step's keys and values with their rotation,
// and causal attention over the pages (sliding window, sinks, a prefix shared by the batch).
#pragma once

#include "address.cuh"
#include "kv_index.cuh"

namespace lng {

// What every kernel of the cache is told (device pointers; strides in elements).
struct KvView {
  void *k, *v;
  int64_t k_page, k_head, k_slot, v_page, v_head, v_slot;
  const int32_t* table;
  int64_t table_stride, num_pages;
  const int32_t* lengths;
  const int32_t* cu;
  int64_t batch, tokens;
  int32_t kv_heads, head_dim, page_shift, capacity, max_new;
};

struct KvRows {
  void* ptr;
  int64_t token, head;
};

__device__ __forceinline__ void kv_range_error() { atomicCAS(&g_error_word, 0u, (unsigned int)DEV_ERR_KV_RANGE); }

__device__ __forceinline__ SeqSpan kv_span(const KvView& c, int64_t b) {
  const SeqSpan s = seq_span(c.cu, c.lengths, b, c.tokens, c.max_new, c.capacity);
  if (s.bad) kv_range_error();
  return s;
}

// The sequence whose rows hold `token`, or -1: division for uniform steps, else a binary search of cu.
__device__ __forceinline__ int64_t kv_sequence_of(const KvView& c, int64_t token) {
  if (c.cu == nullptr)  // (a 64-bit division takes some 40 instructions more)
    return token < (int64_t(1) << 32) ? int64_t(uint32_t(token) / uint32_t(c.max_new)) : token / c.max_new;
  if (token < c.cu[0] || token >= c.cu[c.batch]) return -1;
  int64_t lo = 0, hi = c.batch;  // cu[lo] <= token < cu[hi]
  while (hi - lo > 1) {
    const int64_t mid = (lo + hi) >> 1;
    if (c.cu[mid] <= token)
      lo = mid;
    else
      hi = mid;
  }
  return lo;
}

// ------------------------------------------------------------------ append
// Memory bound: every row is read once and written once.  A warp takes a token (or one of `parts` of it, when
// the step has few tokens) and meets no other: its lanes look up the token's slot, form cos and sin of the token's
// pairs once for all heads, and then move the token's items, an item being two 16-byte vectors of a head -- the two
// halves of eight pairs where pairs are (j, j + half), so rotating q in place is safe.  The angle p * f needs more
// than fp32's 24 bits for far positions (p = 10^6 would leave an error of 0.06 rad): it is formed in turns and
// reduced to the nearest whole one in 64 bits, sine and cosine of the rest fp32.
// What counts is how many warps have loads in flight: CTAs of two warps are replaced as soon as both are through,
// and registers for 48 warps an SM (one item at a time a thread) beat items in pairs.  32 prompts of 2048 tokens, 16
// query and 4 key heads of 64 (403 MB): 8 warps a CTA 86 us, 4 warps 80, 2 warps 77, 1 warp 80; 2 warps with 42
// registers a thread instead of 60: 70 us, 5.8 TB/s.  28 query heads of 128, half rotated: 98 us, 5.4 TB/s.
constexpr int KA_WARPS = 2;
constexpr int KA_MAX_HALF = 64;  // head_dim <= 128

struct KaParams {
  KvView c;
  KvRows kr, vr, qr, qo;
  int32_t q_heads, rotary, interleaved;
  int32_t parts;         // warps a token
  int32_t items;         // of a head: half its vectors, rounded up
  uint32_t items_magic;  // i / items = __umulhi(i, items_magic) where items > 1
  const int64_t* positions;
  const float* inv_freq;
};

template <typename T>
__device__ __forceinline__ void ka_rotate(T& a, T& b, float2 cs) {
  const float x = to_f32<T>(a), y = to_f32<T>(b);
  a = from_f32<T>(x * cs.x - y * cs.y);
  b = from_f32<T>(y * cs.x + x * cs.y);
}

template <typename T>
__global__ void __launch_bounds__(KA_WARPS * 32, 24) kv_append_kernel(const KaParams p) {
  __shared__ __align__(16) float2 cs_all[KA_WARPS][KA_MAX_HALF];
  const KvView& c = p.c;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t w = int64_t(blockIdx.x) * KA_WARPS + warp;
  const int64_t token = p.parts == 1 ? w : int64_t(uint32_t(w) / uint32_t(p.parts));  // (parted only when few)
  if (token >= c.tokens) return;
  const int part = int(w - token * p.parts);
  float2* cs = cs_all[warp];
  const int64_t b = kv_sequence_of(c, token);
  if (b < 0 || b >= c.batch) return;
  const SeqSpan s = kv_span(c, b);
  const int64_t i = token - s.first;
  if (i < 0 || i >= s.n) return;
  // a key outside the sequence's pages (a step past the capacity, say) goes nowhere: every slot there belongs to another
  const int64_t place = s.pos + i;
  const int32_t key = place >= 0 && place < c.capacity ? int32_t(place) : -1;
  const int32_t page = key >= 0 ? page_of(c.table + b * c.table_stride, key, c.page_shift, c.num_pages) : -1;
  if (page < 0) kv_range_error();
  const int32_t slot = key & ((1 << c.page_shift) - 1);
  const int half = p.rotary >> 1;
  if (half > 0) {
    const double pos = p.positions ? double(p.positions[token]) : double(place);
    for (int j = lane; j < half; j += 32) {
      const double turns = pos * double(p.inv_freq[j]) * 0.15915494309189533577;  // 1 / (2 pi)
      float sn, cn;
      sincospif(float(2.0 * (turns - rint(turns))), &sn, &cn);
      cs[j] = make_float2(cn, sn);
    }
    __syncwarp();
  }
  const bool split = !p.interleaved && half > 0, split_vec = split && (half & 7) == 0;
  const int total = (2 * c.kv_heads + p.q_heads) * p.items;
#pragma unroll 1
  for (int it = part * 32 + lane; it < total; it += p.parts * 32) {
    const int h = p.items > 1 ? int(__umulhi(uint32_t(it), p.items_magic)) : it;
    const int item = it - h * p.items;
    const T* src;
    T* dst;
    bool rot = half > 0;
    if (h < c.kv_heads) {
      src = static_cast<const T*>(p.kr.ptr) + token * p.kr.token + h * p.kr.head;
      dst = static_cast<T*>(c.k) + page * c.k_page + slot * c.k_slot + h * c.k_head;
    } else if (h < 2 * c.kv_heads) {
      const int hv = h - c.kv_heads;
      src = static_cast<const T*>(p.vr.ptr) + token * p.vr.token + hv * p.vr.head;
      dst = static_cast<T*>(c.v) + page * c.v_page + slot * c.v_slot + hv * c.v_head;
      rot = false;
    } else {
      const int hq = h - 2 * c.kv_heads;
      src = static_cast<const T*>(p.qr.ptr) + token * p.qr.token + hq * p.qr.head;
      dst = static_cast<T*>(p.qo.ptr) + token * p.qo.token + hq * p.qo.head;
    }
    if (h < 2 * c.kv_heads && page < 0) continue;
    if (rot && split && !split_vec) {  // halves that are no multiple of 8: value by value
      for (int j = item * 16; j < item * 16 + 16 && j < c.head_dim; ++j) {
        if (j < half) {
          T x = src[j], y = src[j + half];
          ka_rotate<T>(x, y, cs[j]);
          dst[j] = x;
          dst[j + half] = y;
        } else if (j >= p.rotary) {
          dst[j] = src[j];
        }
      }
      continue;
    }
    // the item's columns: partners first, then what is not rotated, two vectors each
    int c0 = item * 16, c1 = c0 + 8;
    const bool pair = rot && split && item * 8 < half;
    if (pair) c0 = item * 8, c1 = c0 + half;
    const bool two = c1 < c.head_dim;
    uint4 w0 = __ldcs(reinterpret_cast<const uint4*>(src + c0)), w1 = make_uint4(0, 0, 0, 0);
    if (two) w1 = __ldcs(reinterpret_cast<const uint4*>(src + c1));
    T *e0 = reinterpret_cast<T*>(&w0), *e1 = reinterpret_cast<T*>(&w1);
    if (pair) {
#pragma unroll
      for (int e = 0; e < 8; e += 2) {
        const float4 r = *reinterpret_cast<const float4*>(cs + c0 + e);
        ka_rotate<T>(e0[e], e1[e], make_float2(r.x, r.y));
        ka_rotate<T>(e0[e + 1], e1[e + 1], make_float2(r.z, r.w));
      }
    } else if (rot && p.interleaved) {
#pragma unroll
      for (int e = 0; e < 8; e += 2) {
        if (c0 + e < p.rotary) ka_rotate<T>(e0[e], e0[e + 1], cs[(c0 + e) >> 1]);
        if (c1 + e < p.rotary) ka_rotate<T>(e1[e], e1[e + 1], cs[(c1 + e) >> 1]);
      }
    }
    *reinterpret_cast<uint4*>(dst + c0) = w0;
    if (two) *reinterpret_cast<uint4*>(dst + c1) = w1;
  }
}

}  // namespace lng
