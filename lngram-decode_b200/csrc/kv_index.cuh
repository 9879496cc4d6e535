// Index arithmetic of the paged key/value cache: which tokens a sequence adds, which keys they see and
// which tiles of keys a block of queries has to visit.  Plain integer functions without CUDA headers,
// so that the same code also compiles for the host and is checked there against brute force.
#pragma once

#include <stdint.h>

#ifdef __CUDACC__
#define LNG_HD __host__ __device__ __forceinline__
#else
#define LNG_HD inline
#endif

namespace lng {

// The new tokens of sequence b: rows [first, first + n) of the step's tokens, at positions pos .. pos + n - 1 of the
// sequence (its length less its count of tokens, both as given).  `len` is what attention reads: the keys up to the
// last of these rows, so that pos == len - n, or 0 -- no keys -- when the length is out of range.
struct SeqSpan {
  int64_t first, pos;
  int32_t n, len;
  int32_t bad;  // the offsets or the length were out of range
};

// cu (offsets [batch + 1] into `tokens` rows) may be null: every sequence then adds max_new tokens.
// Offsets out of range give an empty or a shorter span, never one outside the caller's rows, and leave every token
// that is kept at its own position; what a length out of range does is said above.
LNG_HD SeqSpan seq_span(const int32_t* cu, const int32_t* lengths, int64_t b, int64_t tokens, int32_t max_new,
                        int32_t capacity) {
  SeqSpan s;
  const int32_t len = lengths[b];
  s.bad = len < 0 || len > capacity;
  s.len = s.bad ? 0 : len;
  if (cu == nullptr) {
    s.first = b * int64_t(max_new);
    s.n = max_new;
    s.pos = int64_t(len) - max_new;
    return s;
  }
  const int64_t begin = cu[b], stop = cu[b + 1];
  int64_t first = begin, end = stop;
  s.pos = int64_t(len) - (end - first);
  if (first < 0 || end < first || end > tokens || end - first > max_new) {
    if (first < 0) first = 0;
    if (first > tokens) first = tokens;
    if (end > tokens) end = tokens;
    if (end < first) end = first;
    if (end - first > max_new) end = first + max_new;
    s.pos += first - begin;
    const int64_t keys = s.pos + (end - first);
    s.len = s.bad || keys < 0 ? 0 : keys < capacity ? int32_t(keys) : capacity;
    s.bad = 1;
  }
  s.first = first;
  s.n = int32_t(end - first);
  return s;
}

// Whether the token at position p sees key j: causal, and with a window > 0 only the window's keys
// (p itself and the window - 1 before it) and the first `sinks`.
LNG_HD bool key_visible(int32_t j, int32_t p, int32_t window, int32_t sinks) {
  return j <= p && (window <= 0 || j > p - window || j < sinks);
}

// The keys that tokens at positions p0 .. p1 (p1 < the length) see between them:
// [0, sink_end) and [lo, hi); empty when hi <= 0.
struct KeySpan {
  int32_t lo, hi, sink_end;
};

LNG_HD KeySpan key_span(int32_t p0, int32_t p1, int32_t window, int32_t sinks) {
  KeySpan k;
  k.hi = p1 + 1 > 0 ? p1 + 1 : 0;
  k.lo = 0;
  k.sink_end = 0;
  if (window > 0 && p0 + 1 > window) {
    k.lo = p0 + 1 - window;
    if (k.lo > k.hi) k.lo = k.hi;
    if (sinks >= k.lo)
      k.lo = 0;
    else
      k.sink_end = sinks > 0 ? sinks : 0;
  }
  return k;
}

LNG_HD bool key_needed(const KeySpan& k, int32_t j) { return j < k.hi && (j >= k.lo || j < k.sink_end); }

// Whether any key of [a, b) is needed / whether all of them are.
LNG_HD bool any_needed(const KeySpan& k, int32_t a, int32_t b) {
  return a < k.sink_end || (a < k.hi && b > k.lo);
}
LNG_HD bool all_needed(const KeySpan& k, int32_t a, int32_t b) {
  return b <= k.sink_end || (a >= k.lo && b <= k.hi);
}
// Whether every one of the keys [a, b) is visible from every position p0 .. p1.
LNG_HD bool all_visible(int32_t a, int32_t b, int32_t p0, int32_t p1, int32_t window, int32_t sinks) {
  return b <= p0 + 1 && (window <= 0 || a > p1 - window || b <= sinks);
}

// The tiles of `bk` keys (aligned to multiples of bk) that hold needed keys, in order: the sinks'
// tiles, then the window's.
struct KeyTiles {
  int32_t sink_tiles, first, count;
};

LNG_HD KeyTiles key_tiles(const KeySpan& k, int32_t bk) {
  KeyTiles t;
  if (k.hi <= 0) {
    t.sink_tiles = t.first = t.count = 0;
    return t;
  }
  t.sink_tiles = (k.sink_end + bk - 1) / bk;
  t.first = k.lo / bk;
  if (t.first < t.sink_tiles) t.first = t.sink_tiles;
  const int32_t end = (k.hi + bk - 1) / bk;
  t.count = t.sink_tiles + (end > t.first ? end - t.first : 0);
  return t;
}
LNG_HD int32_t tile_index(const KeyTiles& t, int32_t j) { return j < t.sink_tiles ? j : t.first + (j - t.sink_tiles); }

// The page that holds key j, or -1 when the table's entry is no page of the cache.
LNG_HD int32_t page_of(const int32_t* table_row, int32_t j, int32_t page_shift, int64_t num_pages) {
  const int32_t p = table_row[j >> page_shift];
  return p >= 0 && int64_t(p) < num_pages ? p : -1;
}

}  // namespace lng
