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
  if (c.cu == nullptr) return token / c.max_new;
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
// Memory bound: every row is read once and written once, 16 bytes a thread.  A 256-thread CTA takes TPC
// tokens: first one thread per (token, pair) forms cos and sin -- the angle p * f needs more than fp32's
// 24 bits for far positions (p = 10^6 would leave an error of 0.06 rad), so the product and its reduction
// by 2 pi are 64-bit, once per token and not per head, and sine and cosine of the reduced angle fp32 --
// then the threads walk the tokens' (head, column) vectors.  Pairs (j, j + half) are both handled by the
// thread of column j, so rotating q in place is safe.
template <typename T, int TPC>
__global__ void __launch_bounds__(256)
    kv_append_kernel(KvView c, KvRows kr, KvRows vr, KvRows qr, KvRows qo, int32_t q_heads,
                     const int64_t* __restrict__ positions, const float* __restrict__ inv_freq, int32_t rotary,
                     int32_t interleaved) {
  constexpr int MAX_HALF = 64;  // head_dim <= 128
  __shared__ float2 cs[TPC][MAX_HALF];
  __shared__ int64_t k_base[TPC], v_base[TPC];  // element offsets of the token's slot (head 0), -1: none
  __shared__ int64_t row[TPC];                  // -1: the token belongs to no sequence
  __shared__ double pos[TPC];
  const int half = rotary >> 1, tid = threadIdx.x;
  for (int64_t t0 = int64_t(blockIdx.x) * TPC; t0 < c.tokens; t0 += int64_t(gridDim.x) * TPC) {
    if (tid < TPC) {
      const int64_t t = t0 + tid;
      int64_t kb = -1, vb = -1, rw = -1;
      double p = 0.0;
      const int64_t b = t < c.tokens ? kv_sequence_of(c, t) : -1;
      if (b >= 0 && b < c.batch) {
        const SeqSpan s = kv_span(c, b);
        const int64_t i = t - s.first;
        if (i >= 0 && i < s.n) {
          rw = t;
          const int32_t key = s.len - s.n + int32_t(i);
          p = positions ? double(positions[t]) : double(key);
          const int32_t page = key >= 0 ? page_of(c.table + b * c.table_stride, key, c.page_shift, c.num_pages) : -1;
          if (page >= 0) {
            const int32_t slot = key & ((1 << c.page_shift) - 1);
            kb = page * c.k_page + slot * c.k_slot;
            vb = page * c.v_page + slot * c.v_slot;
          } else {
            kv_range_error();
          }
        }
      }
      k_base[tid] = kb;
      v_base[tid] = vb;
      row[tid] = rw;
      pos[tid] = p;
    }
    __syncthreads();
    for (int i = tid; i < TPC * half; i += 256) {
      const int t = i / half, j = i - t * half;
      const double a = pos[t] * double(inv_freq[j]);
      const float r = float(fma(-rint(a * 0.15915494309189533577), 6.283185307179586476925, a));
      float sn, cn;
      sincosf(r, &sn, &cn);
      cs[t][j] = make_float2(cn, sn);
    }
    __syncthreads();
    // columns of 8 values; in the split form columns of the first half of the rotated part also do
    // their partners, and a half that is no multiple of 8 is rotated value by value
    const int cols = c.head_dim >> 3;
    const bool split_vec = !interleaved && half > 0 && (half & 7) == 0;
    const bool split_any = !interleaved && half > 0 && (half & 7) != 0;
    const int heads = 2 * c.kv_heads + q_heads;
    const int items = TPC * heads * cols;
    for (int it = tid; it < items; it += 256) {
      const int t = it / (heads * cols);
      const int rem = it - t * heads * cols;
      const int h = rem / cols, col = (rem - h * cols) << 3;
      if (row[t] < 0) continue;
      const T* src;
      T* dst;
      bool rot = rotary > 0 && col < rotary;
      if (h < c.kv_heads) {
        if (k_base[t] < 0) continue;
        src = static_cast<const T*>(kr.ptr) + row[t] * kr.token + h * kr.head;
        dst = static_cast<T*>(c.k) + k_base[t] + h * c.k_head;
      } else if (h < 2 * c.kv_heads) {
        if (v_base[t] < 0) continue;
        const int hv = h - c.kv_heads;
        src = static_cast<const T*>(vr.ptr) + row[t] * vr.token + hv * vr.head;
        dst = static_cast<T*>(c.v) + v_base[t] + hv * c.v_head;
        rot = false;
      } else {
        const int hq = h - 2 * c.kv_heads;
        src = static_cast<const T*>(qr.ptr) + row[t] * qr.token + hq * qr.head;
        dst = static_cast<T*>(qo.ptr) + row[t] * qo.token + hq * qo.head;
      }
      if (!rot) {
        *reinterpret_cast<uint4*>(dst + col) = *reinterpret_cast<const uint4*>(src + col);
      } else if (interleaved) {
        uint4 w = *reinterpret_cast<const uint4*>(src + col);
        T* e = reinterpret_cast<T*>(&w);
#pragma unroll
        for (int i = 0; i < 8; i += 2) {
          if (col + i < rotary) {
            const float2 r = cs[t][(col + i) >> 1];
            const float a = to_f32<T>(e[i]), b = to_f32<T>(e[i + 1]);
            e[i] = from_f32<T>(a * r.x - b * r.y);
            e[i + 1] = from_f32<T>(b * r.x + a * r.y);
          }
        }
        *reinterpret_cast<uint4*>(dst + col) = w;
      } else if (split_vec) {
        if (col >= half) continue;  // the partner column does it
        uint4 w0 = *reinterpret_cast<const uint4*>(src + col);
        uint4 w1 = *reinterpret_cast<const uint4*>(src + col + half);
        T* e0 = reinterpret_cast<T*>(&w0);
        T* e1 = reinterpret_cast<T*>(&w1);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float2 r = cs[t][col + i];
          const float a = to_f32<T>(e0[i]), b = to_f32<T>(e1[i]);
          e0[i] = from_f32<T>(a * r.x - b * r.y);
          e1[i] = from_f32<T>(b * r.x + a * r.y);
        }
        *reinterpret_cast<uint4*>(dst + col) = w0;
        *reinterpret_cast<uint4*>(dst + col + half) = w1;
      } else if (split_any) {
        for (int i = 0; i < 8; ++i) {
          const int j = col + i;
          if (j < half) {
            const float2 r = cs[t][j];
            const float a = to_f32<T>(src[j]), b = to_f32<T>(src[j + half]);
            dst[j] = from_f32<T>(a * r.x - b * r.y);
            dst[j + half] = from_f32<T>(b * r.x + a * r.y);
          } else if (j >= rotary) {
            dst[j] = src[j];
          }
        }
      }
    }
    __syncthreads();
  }
}

}  // namespace lng
