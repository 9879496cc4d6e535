// Beam search: the best continuations over a group's beams and the vocabulary, and the states' reordering.
#pragma once

#include "kvcache.cuh"

namespace lng {

// ------------------------------------------------------------------ selection
// One pass over the logits.  Within a row (a beam) candidates rank as their logits do, so a CTA keeps the `width`
// largest logits of its piece of a row beside the piece's maximum and sum of exponentials; a dependent launch, a CTA a
// group, joins the pieces' sums, ranks each row's candidates, and then the rows' against one another by
// score + (logit - log sum), in 64 bits: scores a few ulp of 32 bits apart must not change places.  Ties go to the lower
// index at every step.
constexpr int BS_THREADS = 256, BS_WARPS = 8, BS_MOST = 32;

struct BeamParams {
  const void* logits;
  int64_t row_stride, groups, vocab;
  int32_t beams, width, pieces;
  int64_t piece;  // values of a row that a CTA takes
  const float* scores;
  const uint8_t* done;
  int64_t eos;
  float2* part;   // [rows][pieces] (maximum, sum)
  float* value;   // [rows][pieces][width]
  int32_t* index; // likewise: the token
  float* out_scores;
  int64_t *tokens, *parents;
};

// A list of up to 32 candidates in falling order, one a lane; empty places hold (-inf, INT_MAX).
template <typename F>
struct BeamList {
  F v;
  int32_t i;
  __device__ __forceinline__ void clear() {
    v = F(-INFINITY);
    i = 0x7fffffff;
  }
  // whether (x, id) ranks before what the lane holds
  static __device__ __forceinline__ bool before(F x, int32_t id, F v, int32_t i) { return x > v || (x == v && id < i); }
  // all lanes: the same candidate
  __device__ __forceinline__ void insert(F x, int32_t id) {
    const bool mine = before(x, id, v, i);
    const uint32_t from = __ballot_sync(0xffffffffu, mine);
    const F pv = __shfl_up_sync(0xffffffffu, v, 1);
    const int32_t pi = __shfl_up_sync(0xffffffffu, i, 1);
    if (mine) {
      const bool here = (threadIdx.x & 31) == __ffs(from) - 1;
      v = here ? x : pv;
      i = here ? id : pi;
    }
  }
  // the lanes' own candidates (where `on`), those that rank before the list's place `last`
  __device__ __forceinline__ void offer(bool on, F x, int32_t id, int last) {
    const F lv = __shfl_sync(0xffffffffu, v, last);
    const int32_t li = __shfl_sync(0xffffffffu, i, last);
    uint32_t go = __ballot_sync(0xffffffffu, on && before(x, id, lv, li));
    while (go) {
      const int src = __ffs(go) - 1;
      go &= go - 1;
      insert(__shfl_sync(0xffffffffu, x, src), __shfl_sync(0xffffffffu, id, src));
    }
  }
};

// 16 bytes of values from any address that their type allows: one load, or four or five of a word each (of two-byte
// values at an odd place the first and the last word reach over the values by one).
template <typename T>
__device__ __forceinline__ void beam_vector(const T* src, float (&x)[16 / sizeof(T)]) {
  const uint32_t off = uint32_t(reinterpret_cast<uintptr_t>(src)) & 15u;
  uint32_t w[4];
  if (off == 0) {
    const uint4 v = __ldcs(reinterpret_cast<const uint4*>(src));
    w[0] = v.x, w[1] = v.y, w[2] = v.z, w[3] = v.w;
  } else if ((off & 3u) == 0) {
#pragma unroll
    for (int y = 0; y < 4; ++y) w[y] = reinterpret_cast<const uint32_t*>(src)[y];
  } else {
    const uint32_t* from = reinterpret_cast<const uint32_t*>(reinterpret_cast<uintptr_t>(src) & ~uintptr_t(3));
    uint32_t lo = from[0];
#pragma unroll
    for (int y = 0; y < 4; ++y) {
      const uint32_t hi = from[y + 1];
      w[y] = __funnelshift_r(lo, hi, 16);
      lo = hi;
    }
  }
  const T* e = reinterpret_cast<const T*>(w);
#pragma unroll
  for (int y = 0; y < 16 / int(sizeof(T)); ++y) x[y] = to_f32<T>(e[y]);
}

template <typename T>
__global__ void __launch_bounds__(BS_THREADS) beam_piece_kernel(const BeamParams p) {
  constexpr int N = 16 / sizeof(T);
  __shared__ float2 sums[BS_WARPS];
  __shared__ float lv[BS_WARPS][BS_MOST];
  __shared__ int32_t li[BS_WARPS][BS_MOST];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, last = p.width - 1;
  const int64_t row = blockIdx.x / p.pieces;
  const int32_t piece = int32_t(blockIdx.x - row * p.pieces);
  const T* const src = static_cast<const T*>(p.logits) + row * p.row_stride;
  const int64_t v0 = piece * p.piece, v1 = v0 + p.piece < p.vocab ? v0 + p.piece : p.vocab;
  // vectors begin at the piece's first value wherever that lies, so that equal rows have equal sums and tie; those that
  // reach over the piece's end, or whose words might reach over the logits, are taken value by value
  const int64_t vecs = v1 > v0 ? (v1 - v0 + N - 1) / N : 0;
  const int64_t safe0 = row > 0 ? 0 : 1, safe1 = row + 1 < p.groups * p.beams ? v1 : (v1 < p.vocab ? v1 : v1 - 1);
  const bool odd = (reinterpret_cast<uintptr_t>(src) & 3) != 0;
  BeamList<float> list;
  list.clear();
  float m = -INFINITY, s = 0.f;
  // (all lanes of a warp stay together: the list is the warp's)
  for (int64_t k0 = int64_t(warp) * 32; k0 < vecs; k0 += BS_THREADS) {
    const int64_t k = k0 + lane, at = v0 + k * N;
    float x[N];
    if (at + N <= v1 && (!odd || (at >= safe0 && at + N <= safe1))) {
      beam_vector<T>(src + at, x);
    } else {
#pragma unroll
      for (int y = 0; y < N; ++y) x[y] = at + y < v1 ? to_f32<T>(src[at + y]) : -INFINITY;
    }
    float top = x[0];
#pragma unroll
    for (int y = 1; y < N; ++y) top = fmaxf(top, x[y]);
    if (top > m) {
      s *= m == -INFINITY ? 0.f : __expf(m - top);
      m = top;
    }
    const float ref = m == -INFINITY ? 0.f : m;
#pragma unroll
    for (int y = 0; y < N; ++y) s += __expf(x[y] - ref);
    if (__any_sync(0xffffffffu, top >= __shfl_sync(0xffffffffu, list.v, last))) {
#pragma unroll
      for (int y = 0; y < N; ++y) {
        // (a NaN ranks as -inf; a row that holds one offers nothing in the end)
        list.offer(at + y < v1, x[y] == x[y] ? x[y] : -INFINITY, int32_t(at + y), last);
      }
    }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const float om = __shfl_xor_sync(0xffffffffu, m, o), os = __shfl_xor_sync(0xffffffffu, s, o);
    const float n = fmaxf(m, om), r = n == -INFINITY ? 0.f : n;
    s = s * __expf(m - r) + os * __expf(om - r);
    m = n;
  }
  if (lane == 0) sums[warp] = make_float2(m, s);
  lv[warp][lane] = list.v;
  li[warp][lane] = list.i;
  __syncthreads();
  if (warp > 0) return;
  for (int w = 1; w < BS_WARPS; ++w) list.offer(lane < p.width, lv[w][lane], li[w][lane], last);
  if (lane < p.width) {
    p.value[(row * p.pieces + piece) * p.width + lane] = list.v;
    p.index[(row * p.pieces + piece) * p.width + lane] = list.i;
  }
  if (lane == 0) {
    float n = -INFINITY, t = 0.f;
    for (int w = 0; w < BS_WARPS; ++w) n = fmaxf(n, sums[w].x);
    const float r = n == -INFINITY ? 0.f : n;
    for (int w = 0; w < BS_WARPS; ++w) t += sums[w].y * __expf(sums[w].x - r);
    p.part[row * p.pieces + piece] = make_float2(n, t);
  }
}

__global__ void __launch_bounds__(BS_THREADS) beam_join_kernel(const BeamParams p) {
  __shared__ double cv[BS_MOST][BS_MOST];
  __shared__ int32_t ci[BS_MOST][BS_MOST];
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, last = p.width - 1;
  const int64_t g = blockIdx.x;
  // a warp a row: log of the sum, the row's best
  for (int k = warp; k < p.beams; k += BS_WARPS) {
    const int64_t row = g * p.beams + k;
    const float2* part = p.part + row * p.pieces;
    float m = -INFINITY;
    for (int i = lane; i < p.pieces; i += 32) m = fmaxf(m, part[i].x);
    m = warp_max(m);
    double s = 0.0;
    for (int i = lane; i < p.pieces; i += 32)
      if (part[i].y != 0.f) s += double(part[i].y) * exp(double(part[i].x) - double(m));  // (0: nothing but -inf)
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    const double norm = double(m) + log(s), score = double(p.scores[row]);
    const bool ended = p.done != nullptr && p.done[row] != 0;
    const bool empty = !(norm < INFINITY) || norm == -INFINITY;
    BeamList<float> list;
    list.clear();
    if (!ended && !empty) {
      const int64_t n = int64_t(p.pieces) * p.width;
      const float* value = p.value + row * n;
      const int32_t* index = p.index + row * n;
      for (int64_t i0 = 0; i0 < n; i0 += 32) {
        const bool on = i0 + lane < n;
        list.offer(on, on ? value[i0 + lane] : 0.f, on ? index[i0 + lane] : 0, last);
      }
    }
    double c = score + (double(list.v) - norm);
    int32_t token = list.i;
    if (ended || empty) {  // eos at the beam's score, then the lowest other tokens at -inf; or those alone
      const int32_t eos = int32_t(p.eos);
      token = !ended ? lane : lane == 0 ? eos : lane - 1 < eos ? lane - 1 : lane;
      if (token >= p.vocab) token = 0x7fffffff;
      c = ended && lane == 0 ? score : -INFINITY;
    }
    if (c != c) c = -INFINITY;
    cv[k][lane] = c;
    ci[k][lane] = token;
  }
  __syncthreads();
  if (warp > 0) return;
  BeamList<double> best;
  best.clear();
  int32_t beam = 0;  // (a candidate's place: beam << 5 | place in the beam's list, which orders as beam * vocab + token does among equals)
  for (int k = 0; k < p.beams; ++k) {
    const bool on = lane < p.width && ci[k][lane] != 0x7fffffff;
    best.offer(on, cv[k][lane], (k << 5) | lane, last);
  }
  if (lane < p.width) {
    beam = best.i >> 5;
    const bool there = best.i != 0x7fffffff;
    p.out_scores[g * p.width + lane] = float(best.v);
    p.tokens[g * p.width + lane] = there ? ci[beam][best.i & 31] : 0;
    p.parents[g * p.width + lane] = there ? beam : 0;
  }
}

// ------------------------------------------------------------------ reordering of states
// Memory bound: of each group the rows that are needed are read and the rows that change are written, in place: a
// thread takes one 16-byte column (or, where addresses allow no more, 8, 4, 2 or 1 bytes) of all the group's
// rows, and writes none of them before it has read all that it needs.
constexpr int BR_THREADS = 256, BR_STATES = 8;

struct BeamState {
  uint8_t* ptr;
  int64_t stride, columns;  // columns of `vec` bytes, then `tail` single bytes
  int32_t vec, tail;
  int64_t block0;           // of the grid's x
};
struct BeamReorderParams {
  const int64_t* parents;
  int32_t beams, count;
  BeamState state[BR_STATES];
};

template <int MOST, typename V>
__device__ __forceinline__ void beam_move(uint8_t* at, int64_t stride, const int32_t* from, int32_t beams) {
  V r[MOST];
#pragma unroll
  for (int k = 0; k < MOST; ++k)
    if (k < beams && from[k] != k) r[k] = *reinterpret_cast<const V*>(at + from[k] * stride);
#pragma unroll
  for (int k = 0; k < MOST; ++k)
    if (k < beams && from[k] != k) *reinterpret_cast<V*>(at + k * stride) = r[k];
}

template <int MOST>
__global__ void __launch_bounds__(BR_THREADS) beam_reorder_kernel(const __grid_constant__ BeamReorderParams p) {
  __shared__ int32_t from[BS_MOST];
  const int64_t g = blockIdx.y;
  if (threadIdx.x < p.beams) {
    const int64_t q = p.parents[g * p.beams + threadIdx.x];
    const bool good = q >= 0 && q < p.beams;
    if (!good) kv_range_error();
    from[threadIdx.x] = good ? int32_t(q) : int32_t(threadIdx.x);
  }
  __syncthreads();
  int i = 0;
  while (i + 1 < p.count && blockIdx.x >= p.state[i + 1].block0) ++i;
  const BeamState& s = p.state[i];
  const int64_t x = (int64_t(blockIdx.x) - s.block0) * BR_THREADS + threadIdx.x;
  uint8_t* const base = s.ptr + g * p.beams * s.stride;
  if (x < s.columns) {
    uint8_t* const at = base + x * s.vec;
    switch (s.vec) {
      case 16: beam_move<MOST, uint4>(at, s.stride, from, p.beams); break;
      case 8: beam_move<MOST, uint2>(at, s.stride, from, p.beams); break;
      case 4: beam_move<MOST, uint32_t>(at, s.stride, from, p.beams); break;
      case 2: beam_move<MOST, uint16_t>(at, s.stride, from, p.beams); break;
      default: beam_move<MOST, uint8_t>(at, s.stride, from, p.beams);
    }
  } else if (x < s.columns + s.tail) {
    beam_move<MOST, uint8_t>(base + s.columns * s.vec + (x - s.columns), s.stride, from, p.beams);
  }
}

}  // namespace lng
