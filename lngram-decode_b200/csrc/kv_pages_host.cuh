// The C ABI's entries of page pools and beams (include/lngram_b200.h).
#pragma once

#include <type_traits>

#include "beam.cuh"
#include "kv_host.cuh"
#include "kv_pages.cuh"

namespace lng {

// What the page calls need of a cache of either kind.
static int check_pool(const lng_kv8_cache* c, const int32_t* refs, const int32_t* cu, int64_t tokens, int64_t max_new) {
  LNG_REQUIRE(c != nullptr, "cache descriptor is NULL");
  if (const int st = check_kv(&c->pages, cu, tokens, max_new)) return st;
  LNG_REQUIRE((c->k_exp == nullptr) == (c->v_exp == nullptr), "k_exp and v_exp go together");
  LNG_REQUIRE(c->pages.batch <= PG_MOST_BATCH, "a pool serves at most 8192 sequences");
  LNG_REQUIRE(c->pages.num_pages <= PG_MOST_PAGES, "a pool holds at most 2^22 pages");
  if (c->pages.batch == 0) return LNG_OK;
  LNG_REQUIRE(refs && c->pages.table && c->pages.lengths, "NULL pointer");
  LNG_REQUIRE(c->pages.max_pages >= 1, "the table has no columns");
  return LNG_OK;
}

static PgParams pg_params(const lng_kv8_cache* c, int32_t* refs, const int32_t* cu, int64_t tokens, int64_t max_new) {
  PgParams p{};
  p.c = kv_view(&c->pages, cu, tokens, max_new);
  p.table = const_cast<int32_t*>(c->pages.table);
  p.lengths = const_cast<int32_t*>(c->pages.lengths);
  p.refs = refs;
  return p;
}

}  // namespace lng

using namespace lng;

// An extend's copies in one cache: a dependent launch, that waits for the whole of the kernel that notes them.
static int launch_pages_copy(const lng_kv8_cache& cache, const int32_t* copies, cudaStream_t stream) {
  const lng_kv_cache& c = cache.pages;
  const int64_t size = cache.k_exp ? 1 : 2;  // bytes a value
  PgCopyParams p{};
  p.k = static_cast<uint8_t*>(c.k), p.v = static_cast<uint8_t*>(c.v);
  p.k_page = c.k_page_stride * size, p.k_head = c.k_head_stride * size, p.k_slot = c.k_slot_stride * size;
  p.v_page = c.v_page_stride * size, p.v_head = c.v_head_stride * size, p.v_slot = c.v_slot_stride * size;
  p.k_exp = cache.k_exp, p.v_exp = cache.v_exp;
  p.k_exp_page = cache.k_exp_stride, p.v_exp_page = cache.v_exp_stride;
  p.num_pages = c.num_pages;
  p.heads = c.num_kv_heads;
  p.page_size = c.page_size;
  p.copies = reinterpret_cast<const int4*>(copies);
  // strides are multiples of 8 values: 16 bytes in 16 bits, 8 bytes in 8
  const int vec = size == 2 ? 16 : 8;
  p.vecs = int32_t(c.head_dim * size / vec);
  const dim3 grid{unsigned(c.batch), unsigned(2 * std::min<int64_t>(8, c.num_kv_heads)), 1u};
  return launch_dependent(vec == 16 ? kv_pages_copy_kernel<16> : kv_pages_copy_kernel<8>, grid, 128u, size_t(0), stream, p);
}

extern "C" int lng_kv_pages_extend(const lng_kv8_cache* caches, int32_t count, int32_t* refs, const int32_t* cu, int64_t tokens,
                                   int64_t max_new, int64_t* slots, uint8_t* served, int32_t* copies, lng_stream_t stream) {
  LNG_REQUIRE(count >= 1 && caches != nullptr, "a pool needs at least one cache");
  for (int32_t i = 0; i < count; ++i) {
    if (const int st = check_pool(&caches[i], refs, cu, tokens, max_new)) return st;
    LNG_REQUIRE(caches[i].pages.k && caches[i].pages.v, "NULL pointer in the cache descriptor");
    LNG_REQUIRE(caches[i].pages.batch == caches[0].pages.batch && caches[i].pages.num_pages == caches[0].pages.num_pages &&
                    caches[i].pages.page_size == caches[0].pages.page_size,
                "a pool's caches must be of one geometry");
  }
  LNG_REQUIRE(caches->pages.batch == 0 || (served && copies), "NULL pointer");
  LNG_REQUIRE(slots || tokens == 0, "slots is NULL");
  LNG_REQUIRE((reinterpret_cast<uintptr_t>(copies) & 15) == 0, "copies must be 16-byte aligned");
  // (rows that belong to no sequence, which without sequences is all of them)
  if (cu && tokens > 0) LNG_CUDA(cudaMemsetAsync(slots, 0xff, size_t(tokens) * 8, S(stream)));
  if (caches->pages.batch == 0) return LNG_OK;
  PgParams p = pg_params(caches, refs, cu, tokens, max_new);
  p.slots = slots;
  p.served = served;
  p.copies = reinterpret_cast<int4*>(copies);
  const int64_t words = ceil_div(p.c.num_pages, 32 * PG_CTAS);
  const size_t smem = size_t(3 * p.c.batch + words) * 4;
  static std::atomic<uint64_t> known{0};
  if (smem > 40 * 1024)
    if (const int st = allow_smem(kv_pages_extend_kernel, 200 * 1024, known)) return st;
  kv_pages_extend_kernel<<<PG_CTAS, PG_THREADS, smem, S(stream)>>>(p);
  LNG_LAUNCHED("kv_pages_extend_kernel");
  for (int32_t i = 0; i < count; ++i)
    if (const int st = launch_pages_copy(caches[i], copies, S(stream))) return st;
  return LNG_OK;
}

extern "C" int lng_kv_pages_truncate(const lng_kv8_cache* cache, int32_t* refs, const int32_t* lengths, int64_t most,
                                     lng_stream_t stream) {
  LNG_REQUIRE(cache != nullptr, "cache descriptor is NULL");
  if (const int st = check_pool(cache, refs, nullptr, cache->pages.batch, 1)) return st;
  LNG_REQUIRE(lengths != nullptr || most >= 0, "most must not be negative");
  if (cache->pages.batch == 0) return LNG_OK;
  const PgParams p = pg_params(cache, refs, nullptr, cache->pages.batch, 1);
  kv_pages_truncate_kernel<<<unsigned(ceil_div(p.c.batch, 8)), 256, 0, S(stream)>>>(p, lengths, int32_t(std::min<int64_t>(most, 1 << 30)));
  LNG_LAUNCHED("kv_pages_truncate_kernel");
  return LNG_OK;
}

extern "C" int lng_kv_pages_reorder(const lng_kv8_cache* cache, int32_t* refs, const int64_t* parents, int64_t groups,
                                    int64_t beams, lng_stream_t stream) {
  LNG_REQUIRE(cache != nullptr, "cache descriptor is NULL");
  if (const int st = check_pool(cache, refs, nullptr, cache->pages.batch, 1)) return st;
  LNG_REQUIRE(groups >= 0 && beams >= 0 && beams <= PG_MOST_BATCH && groups <= PG_MOST_BATCH && groups * beams == cache->pages.batch,
              "groups * beams must be the batch");
  if (cache->pages.batch == 0) return LNG_OK;
  LNG_REQUIRE(parents != nullptr, "parents is NULL");
  const PgParams p = pg_params(cache, refs, nullptr, cache->pages.batch, 1);
  const size_t smem = size_t(3 * beams + std::max<int64_t>(PG_REORDER_CELLS, beams)) * 4;
  static std::atomic<uint64_t> known{0};
  if (smem > 48 * 1024)
    if (const int st = allow_smem(kv_pages_reorder_kernel, 160 * 1024, known)) return st;
  kv_pages_reorder_kernel<<<unsigned(groups), PG_REORDER_THREADS, smem, S(stream)>>>(p, parents, int32_t(beams));
  LNG_LAUNCHED("kv_pages_reorder_kernel");
  return LNG_OK;
}

// ====================================================================== beams
namespace lng {

struct BeamPlan {
  int32_t pieces;
  int64_t piece;
  size_t part, value, index, bytes;
};
// Into how many pieces a row is cut, the same for every row (equal rows tie): what takes the least time when an SM's share
// of the pieces run beside one another, a piece costing its values and as much as 10000 more for its start and end.
static BeamPlan beam_plan(int64_t groups, int64_t beams, int64_t vocab, int64_t width) {
  BeamPlan b{};
  const int64_t rows = groups * beams;
  if (rows <= 0 || vocab <= 0 || width <= 0) return b;
  int64_t pieces = 1;
  double least = 1e300;
  for (int64_t n = 1; n <= 64 && n <= ceil_div(vocab, 2048); ++n) {
    const double cost = double(ceil_div(rows * n, num_sms())) * (double(vocab) / double(n) + 10000.0);
    if (cost < least) {
      least = cost;
      pieces = n;
    }
  }
  b.piece = ceil_div(ceil_div(vocab, pieces), 8) * 8;
  b.pieces = int32_t(ceil_div(vocab, b.piece));
  b.part = 0;
  b.value = al256(size_t(rows) * b.pieces * sizeof(float2));
  b.index = b.value + al256(size_t(rows) * b.pieces * width * 4);
  b.bytes = b.index + al256(size_t(rows) * b.pieces * width * 4);
  return b;
}

}  // namespace lng

extern "C" size_t lng_beam_workspace_bytes(int64_t groups, int64_t beams, int64_t vocab, int64_t width) {
  return beam_plan(groups, beams, vocab, width).bytes;
}

extern "C" int lng_beam_select(const void* logits, int32_t dtype, int64_t row_stride, int64_t groups, int64_t beams, int64_t vocab,
                               const float* scores, const uint8_t* done, int64_t eos, int64_t width, float* out_scores,
                               int64_t* tokens, int64_t* parents, void* workspace, size_t workspace_bytes, lng_stream_t stream) {
  LNG_REQUIRE(is_float_dtype(dtype), "logits must be f32, bf16 or f16");
  LNG_REQUIRE(groups >= 0 && groups < (int64_t(1) << 24), "groups must be in [0, 2^24)");
  LNG_REQUIRE(beams >= 1 && beams <= BS_MOST && width >= 1 && width <= BS_MOST, "beams and width must be in [1, 32]");
  LNG_REQUIRE(vocab >= 1 && vocab < (int64_t(1) << 30), "vocab must be in [1, 2^30)");
  LNG_REQUIRE(width <= beams * vocab, "width must not exceed beams * vocab");
  LNG_REQUIRE(row_stride >= vocab || groups * beams <= 1, "row_stride must be at least vocab");
  LNG_REQUIRE(done == nullptr || (eos >= 0 && eos < vocab), "eos must be a token of the vocabulary");
  if (groups == 0) return LNG_OK;
  LNG_REQUIRE(logits && scores && out_scores && tokens && parents, "NULL pointer");
  LNG_REQUIRE((reinterpret_cast<uintptr_t>(logits) & (dtype_size(dtype) - 1)) == 0, "logits must be aligned to their type");
  const BeamPlan plan = beam_plan(groups, beams, vocab, width);
  LNG_REQUIRE(workspace != nullptr && (reinterpret_cast<uintptr_t>(workspace) & 255) == 0, "workspace must be 256-byte aligned");
  LNG_REQUIRE(workspace_bytes >= plan.bytes, "workspace too small");
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  BeamParams p{};
  p.logits = logits;
  p.row_stride = row_stride;
  p.groups = groups;
  p.vocab = vocab;
  p.beams = int32_t(beams);
  p.width = int32_t(width);
  p.pieces = plan.pieces;
  p.piece = plan.piece;
  p.scores = scores;
  p.done = done;
  p.eos = eos;
  p.part = reinterpret_cast<float2*>(ws + plan.part);
  p.value = reinterpret_cast<float*>(ws + plan.value);
  p.index = reinterpret_cast<int32_t*>(ws + plan.index);
  p.out_scores = out_scores;
  p.tokens = tokens;
  p.parents = parents;
  LNG_REQUIRE(groups * beams * plan.pieces < (int64_t(1) << 31), "too many rows");
  const unsigned grid = unsigned(groups * beams * plan.pieces);
  if (dtype == LNG_F32)
    beam_piece_kernel<float><<<grid, BS_THREADS, 0, S(stream)>>>(p);
  else if (dtype == LNG_BF16)
    beam_piece_kernel<__nv_bfloat16><<<grid, BS_THREADS, 0, S(stream)>>>(p);
  else
    beam_piece_kernel<__half><<<grid, BS_THREADS, 0, S(stream)>>>(p);
  LNG_LAUNCHED("beam_piece_kernel");
  return launch_dependent(beam_join_kernel, unsigned(groups), unsigned(BS_THREADS), size_t(0), S(stream), p);
}

extern "C" int lng_beam_reorder(const int64_t* parents, int64_t groups, int64_t beams, const lng_beam_state* states, int32_t count,
                                lng_stream_t stream) {
  LNG_REQUIRE(groups >= 0 && groups <= 65535, "groups must be in [0, 65535]");
  LNG_REQUIRE(beams >= 1 && beams <= BS_MOST, "beams must be in [1, 32]");
  LNG_REQUIRE(count >= 0 && count <= BR_STATES, "at most 8 states a call");
  if (groups == 0 || count == 0) return LNG_OK;
  LNG_REQUIRE(parents != nullptr && states != nullptr, "NULL pointer");
  BeamReorderParams p{};
  p.parents = parents;
  p.beams = int32_t(beams);
  int64_t blocks = 0;
  for (int32_t i = 0; i < count; ++i) {
    LNG_REQUIRE(states[i].bytes >= 0 && states[i].stride >= states[i].bytes, "a state's rows must not overlap");
    if (states[i].bytes == 0) continue;
    LNG_REQUIRE(states[i].ptr != nullptr, "NULL pointer");
    BeamState& s = p.state[p.count++];
    s.ptr = static_cast<uint8_t*>(states[i].ptr);
    s.stride = states[i].stride;
    const uintptr_t at = reinterpret_cast<uintptr_t>(s.ptr) | uintptr_t(s.stride);
    s.vec = 16;
    while (at & (s.vec - 1)) s.vec >>= 1;
    s.columns = states[i].bytes / s.vec;
    s.tail = int32_t(states[i].bytes - s.columns * s.vec);
    s.block0 = blocks;
    blocks += ceil_div(s.columns + s.tail, BR_THREADS);
  }
  if (p.count == 0) return LNG_OK;
  LNG_REQUIRE(blocks < (int64_t(1) << 31), "the states are too large");
  const dim3 grid{unsigned(blocks), unsigned(groups), 1u};
  if (beams <= 4)
    beam_reorder_kernel<4><<<grid, BR_THREADS, 0, S(stream)>>>(p);
  else if (beams <= 8)
    beam_reorder_kernel<8><<<grid, BR_THREADS, 0, S(stream)>>>(p);
  else
    beam_reorder_kernel<32><<<grid, BR_THREADS, 0, S(stream)>>>(p);
  LNG_LAUNCHED("beam_reorder_kernel");
  return LNG_OK;
}
