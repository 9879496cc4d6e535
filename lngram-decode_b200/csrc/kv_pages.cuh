// Tables, slots and reference counts of a paged cache, made on the GPU from the sequences' lengths.
//
// refs[page] counts the table rows that hold a page; 0 is free.  A length below 0 is that of a suspended sequence of
// -1 - length keys.  Everything here is whole numbers, and every choice has one answer: the lowest free pages, in the
// order of sequence and column.
#pragma once

#include <type_traits>

#include "kvcache.cuh"

namespace lng {

constexpr int64_t PG_MOST_BATCH = 8192, PG_MOST_PAGES = int64_t(1) << 22;

struct PgParams {
  KvView c;
  int32_t* table;
  int32_t* lengths;
  int32_t* refs;
  int64_t* slots;
  uint8_t* served;
  int4* copies;
};

__device__ __forceinline__ int32_t pg_real(int32_t length) { return length < 0 ? -1 - length : length; }

// The new tokens of sequence b, rows [first, first + n); offsets out of range add nothing.
__device__ __forceinline__ int32_t pg_new(const KvView& c, int64_t b, int64_t& first) {
  if (c.cu == nullptr) {
    first = b * c.max_new;
    return c.max_new;
  }
  first = c.cu[b];
  const int64_t n = int64_t(c.cu[b + 1]) - first;
  if (first >= 0 && n >= 0 && first + n <= c.tokens && n <= c.max_new) return int32_t(n);
  kv_range_error();
  return 0;
}

__device__ __forceinline__ uint32_t dsmem_u32(const uint32_t* mine, uint32_t rank) {
  uint32_t at, v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(smem_addr(mine)), "r"(rank));
  asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(at) : "memory");
  return v;
}
__device__ __forceinline__ void cluster_meet() {
  asm volatile("barrier.cluster.arrive.aligned;" ::: "memory");
  asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
}

// ------------------------------------------------------------------ extend
// Bound by latency: counts of some thousands to millions of pages, tails of some hundreds of sequences.  One launch:
// a cluster of eight CTAs.  Each takes an eighth of the pages and packs "free" into bits in shared memory; each
// sums the needs of all sequences for itself (they are few), the counts of free pages meet through distributed
// shared memory, and then the r-th free page knows by a search of the needs' running sum whose it is (a lane a page: a
// warp a page took 78 us for 512 forked sequences, whose pages all lie in the first CTA's share).  Nothing is written
// before all CTAs have read what they need.
// Measured: 64 sequences that take 16 tokens each from a pool of 3700 pages: 6 us; 512 forked sequences, 12700 pages: 10 us.
constexpr int PG_CTAS = 8, PG_THREADS = 512, PG_WARPS = PG_THREADS / 32;

__global__ void __cluster_dims__(PG_CTAS, 1, 1) __launch_bounds__(PG_THREADS, 1) kv_pages_extend_kernel(const PgParams p) {
  extern __shared__ int32_t pg_smem[];
  __shared__ int32_t warp_sum_s[PG_WARPS];
  __shared__ uint32_t warp_free[PG_WARPS], cta_free;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");  // (the copies wait for the whole kernel)
  const KvView& c = p.c;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, cta = blockIdx.x;
  const int32_t batch = int32_t(c.batch), page_size = 1 << c.page_shift;
  int32_t* const ends = pg_smem;            // running sum of the needs, a sequence's own counted
  int32_t* const real = ends + batch;       // keys before the step
  int32_t* const tail = real + batch;       // the page that is copied, -1: none, -2: the sequence does not fit its row
  uint32_t* const bits = reinterpret_cast<uint32_t*>(tail + batch);
  const int32_t words = int32_t((c.num_pages + 32 * PG_CTAS - 1) / (32 * PG_CTAS));

  // needs
  const int32_t run = (batch + PG_THREADS - 1) / PG_THREADS;
  const int32_t b0 = min(tid * run, batch), b1 = min(b0 + run, batch);
  int32_t mine = 0;
  for (int32_t b = b0; b < b1; ++b) {
    int64_t first;
    const int32_t len = pg_real(p.lengths[b]), n = pg_new(c, b, first);
    int32_t need = 0, last = -1;
    if (n > 0) {
      if (int64_t(len) + n > c.capacity) {
        last = -2;
      } else {
        const int32_t have = (len + page_size - 1) >> c.page_shift, want = (len + n + page_size - 1) >> c.page_shift;
        need = want - have;
        if (len & (page_size - 1)) {
          const int32_t t = page_of(p.table + b * c.table_stride, len, c.page_shift, c.num_pages);
          if (t >= 0 && p.refs[t] > 1) {
            last = t;
            ++need;
          }
        }
      }
    }
    mine += need;
    ends[b] = need;
    real[b] = len;
    tail[b] = last;
  }
  int32_t incl = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int32_t v = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += v;
  }
  if (lane == 31) warp_sum_s[warp] = incl;

  // free pages of this CTA: a word a round and warp
  uint32_t free_here = 0;
  const int32_t per = (words + PG_WARPS - 1) / PG_WARPS, w0 = min(warp * per, words), w1 = min(w0 + per, words);
  for (int32_t w = w0; w < w1; w += 4) {
    int32_t r[4];
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      const int64_t page = (int64_t(cta) * words + w + x) * 32 + lane;
      r[x] = w + x < w1 && page < c.num_pages ? p.refs[page] : 1;
    }
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      const uint32_t word = __ballot_sync(0xffffffffu, r[x] == 0);
      if (w + x < w1) {
        if (lane == 0) bits[w + x] = word;
        free_here += __popc(word);
      }
    }
  }
  if (lane == 0) warp_free[warp] = free_here;
  __syncthreads();
  int32_t before = incl - mine;
  uint32_t warps_before = 0, total_here = 0;
  for (int w = 0; w < PG_WARPS; ++w) {
    if (w < warp) {
      before += warp_sum_s[w];
      warps_before += warp_free[w];
    }
    total_here += warp_free[w];
  }
  for (int32_t b = b0; b < b1; ++b) ends[b] = before += ends[b];
  if (tid == 0) cta_free = total_here;
  cluster_meet();  // (the barrier's arrive releases, its wait acquires)
  uint32_t rank = warps_before, total = 0;
  for (uint32_t k = 0; k < PG_CTAS; ++k) {
    const uint32_t f = dsmem_u32(&cta_free, k);
    if (k < uint32_t(cta)) rank += f;
    total += f;
  }
  cluster_meet();  // nobody leaves while its count is read; all of refs, table and lengths has been read

  // the first sequence whose running sum is above x
  auto above = [&](uint32_t x) {
    int32_t lo = 0, hi = batch;
    while (lo < hi) {
      const int32_t mid = (lo + hi) >> 1;
      if (uint32_t(ends[mid]) > x)
        hi = mid;
      else
        lo = mid + 1;
    }
    return lo;
  };
  const int32_t cut = above(total);
  const uint32_t taken = cut > 0 ? uint32_t(ends[cut - 1]) : 0u;  // pages that are handed out

  // this warp's free pages: 32 words a round, those that hold one a word a time, a page a lane
  for (int32_t w = w0; w < w1 && rank < taken; w += 32) {
    const uint32_t word = w + lane < w1 ? bits[w + lane] : 0u;
    uint32_t hit = __ballot_sync(0xffffffffu, word != 0);
    while (hit && rank < taken) {
      const int src = __ffs(hit) - 1;
      hit &= hit - 1;
      const uint32_t some = __shfl_sync(0xffffffffu, word, src), r = rank + __popc(some & ((1u << lane) - 1u));
      if ((some >> lane & 1) && r < taken) {
        const int32_t page = int32_t((int64_t(cta) * words + w + src) * 32 + lane);
        const int32_t b = above(r), idx = int32_t(r) - (b > 0 ? ends[b - 1] : 0);
        const int32_t len = real[b], have = (len + page_size - 1) >> c.page_shift, old = tail[b];
        p.table[b * c.table_stride + (old >= 0 ? have - 1 + idx : have + idx)] = page;
        p.refs[page] = 1;
        if (old >= 0 && idx == 0) {
          p.copies[b] = make_int4(old, page, len & (page_size - 1), 0);
          atomicSub(&p.refs[old], 1);
        }
      }
      rank += __popc(some);
    }
  }
  cluster_meet();  // the table is complete
  // a warp a sequence: whether it was served, its length, its tokens' slots
  for (int32_t b = cta * PG_WARPS + warp; b < batch; b += PG_CTAS * PG_WARPS) {
    int64_t first;
    const int32_t n = pg_new(c, b, first), len = real[b], end = ends[b], need = end - (b > 0 ? ends[b - 1] : 0), old = tail[b];
    const bool ok = old != -2 && (need == 0 || uint32_t(end) <= total);
    if (lane == 0) {
      p.served[b] = ok;
      p.lengths[b] = ok ? len + n : -1 - len;
      if (!ok || old < 0) p.copies[b] = make_int4(-1, -1, 0, 0);
    }
    const int32_t* const row = p.table + b * c.table_stride;
    for (int32_t i = lane; i < n; i += 32) {
      int64_t slot = -1;
      if (ok) {
        const int32_t j = len + i, page = page_of(row, j, c.page_shift, c.num_pages);
        if (page >= 0)
          slot = (int64_t(page) << c.page_shift) + (j & (page_size - 1));
        else
          kv_range_error();  // (a last page that is none)
      }
      p.slots[first + i] = slot;
    }
  }
}

// ------------------------------------------------------------------ copies
// Keys (even blocks in y) or values (odd) of the slots that a copied page holds, of a share of the heads.
// Bound by latency: a launch a cache, which for every sequence looks up whether a page is to be copied.  64 sequences, caches of 4
// heads of 64: extend and truncate take 7.5 us for one layer, 35 us for 32; with rows forked before, eight to a page, and 64 pages copied
// 13 us, and for 32 layers 75 us (16 bits) and 86 us (8 bits, where 8-byte vectors make twice as many accesses a byte).
struct PgCopyParams {
  uint8_t *k, *v;
  int64_t k_page, k_head, k_slot, v_page, v_head, v_slot;  // bytes
  int8_t *k_exp, *v_exp;
  int64_t k_exp_page, v_exp_page, num_pages;
  int32_t heads, vecs, page_size;  // 16-byte vectors a slot and head
  const int4* copies;
};

template <int VEC>
__global__ void __launch_bounds__(128) kv_pages_copy_kernel(const PgCopyParams p) {
  using V = typename std::conditional<VEC == 16, uint4, uint2>::type;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int4 m = p.copies[blockIdx.x];
  if (m.y < 0 || m.x < 0 || m.x >= p.num_pages || m.y >= p.num_pages || m.z <= 0 || m.z > p.page_size) return;
  const bool keys = (blockIdx.y & 1) == 0;
  uint8_t* const base = keys ? p.k : p.v;
  const int64_t page = keys ? p.k_page : p.v_page, head = keys ? p.k_head : p.v_head, slot = keys ? p.k_slot : p.v_slot;
  const int shares = gridDim.y >> 1, share = blockIdx.y >> 1;
  int8_t* const exps = keys ? p.k_exp : p.v_exp;
  const int64_t exp_page = keys ? p.k_exp_page : p.v_exp_page;
  for (int h = share; h < p.heads; h += shares) {
    for (int x = threadIdx.x; x < m.z * p.vecs; x += 128) {
      const int s = x / p.vecs;
      const int64_t at = h * head + s * slot + (x - s * p.vecs) * VEC;
      *reinterpret_cast<V*>(base + m.y * page + at) = *reinterpret_cast<const V*>(base + m.x * page + at);
    }
    if (exps && threadIdx.x == 0) exps[m.y * exp_page + h] = exps[m.x * exp_page + h];
  }
}

// ------------------------------------------------------------------ truncate
// A warp a sequence.
__global__ void __launch_bounds__(256) kv_pages_truncate_kernel(const PgParams p, const int32_t* keep, int32_t most) {
  const int lane = threadIdx.x & 31;
  const int64_t b = (int64_t(blockIdx.x) * 256 + threadIdx.x) >> 5;
  const KvView& c = p.c;
  if (b >= c.batch) return;
  const int32_t len = pg_real(p.lengths[b]), asked = keep ? keep[b] : most;
  const int32_t now = min(len, max(asked, 0)), up = (1 << c.page_shift) - 1;
  const int64_t from = (int64_t(now) + up) >> c.page_shift;
  int64_t to = (int64_t(len) + up) >> c.page_shift;
  if (len > c.capacity) {
    kv_range_error();
    to = c.capacity >> c.page_shift;
  }
  int32_t* const row = p.table + b * c.table_stride;
  for (int64_t x = from + lane; x < to; x += 32) {
    const int32_t page = row[x];
    if (page >= 0 && page < c.num_pages && atomicSub(&p.refs[page], 1) <= 0) {
      atomicAdd(&p.refs[page], 1);  // (nobody held it: the caller's counts and table disagree)
      kv_range_error();
    }
    row[x] = -1;
  }
  __syncwarp();
  if (lane == 0) p.lengths[b] = now;
}

// ------------------------------------------------------------------ reorder
// A CTA a group, whose rows only take over one another's: a piece of all its rows at a time goes through shared
// memory, so the table is rewritten in place.  A page of row r gains a holder for every row that takes r over, less
// the one that r was.
constexpr int PG_REORDER_THREADS = 512, PG_REORDER_CELLS = 8192;

__global__ void __launch_bounds__(PG_REORDER_THREADS) kv_pages_reorder_kernel(const PgParams p, const int64_t* parents, int32_t beams) {
  extern __shared__ int32_t pg_rows[];
  int32_t *const from = pg_rows, *const kids = from + beams, *const len = kids + beams, *const cell = len + beams;
  const KvView& c = p.c;
  const int tid = threadIdx.x;
  const int64_t base = int64_t(blockIdx.x) * beams;
  for (int32_t k = tid; k < beams; k += PG_REORDER_THREADS) {
    const int64_t q = parents[base + k];
    const bool good = q >= 0 && q < beams;
    if (!good) kv_range_error();
    from[k] = good ? int32_t(q) : k;
    kids[k] = 0;
    len[k] = p.lengths[base + k];
  }
  __syncthreads();
  int32_t longest = 0;
  for (int32_t k = tid; k < beams; k += PG_REORDER_THREADS) {
    atomicAdd(&kids[from[k]], 1);
    p.lengths[base + k] = len[from[k]];
  }
  __syncthreads();
  const int32_t up = (1 << c.page_shift) - 1, columns = c.capacity >> c.page_shift;
  auto used = [&](int32_t k) {
    const int64_t n = (int64_t(pg_real(len[k])) + up) >> c.page_shift;
    return int32_t(n < columns ? n : columns);
  };
  for (int32_t k = 0; k < beams; ++k) longest = max(longest, used(k));
  const int32_t wide = PG_REORDER_CELLS / beams > 0 ? PG_REORDER_CELLS / beams : 1;  // columns a piece
  for (int32_t c0 = 0; c0 < longest; c0 += wide) {
    const int32_t n = min(wide, longest - c0);
    for (int32_t x = tid; x < beams * n; x += PG_REORDER_THREADS) {
      const int32_t k = x / n, col = c0 + (x - k * n);
      int32_t page = -1;
      if (col < used(k)) {
        page = p.table[(base + k) * c.table_stride + col];
        const int32_t more = kids[k] - 1;
        if (more != 0 && page >= 0 && page < c.num_pages && atomicAdd(&p.refs[page], more) + more < 0) {
          atomicSub(&p.refs[page], more);
          kv_range_error();
        }
      }
      cell[x] = page;
    }
    __syncthreads();
    for (int32_t x = tid; x < beams * n; x += PG_REORDER_THREADS) {
      const int32_t k = x / n, col = c0 + (x - k * n);
      p.table[(base + k) * c.table_stride + col] = cell[from[k] * n + (x - k * n)];
    }
    __syncthreads();
  }
  // behind the longest row's keys
  for (int32_t k = tid >> 5; k < beams; k += PG_REORDER_THREADS / 32)
    for (int32_t col = longest + (tid & 31); col < columns; col += 32) p.table[(base + k) * c.table_stride + col] = -1;
}

}  // namespace lng
