// The C ABI's entries of the paged cache in 8 bits (include/lngram_b200.h).
#pragma once

#include "kv8.cuh"
#include "kv8_step.cuh"
#include "kv8_tile.cuh"
#include "kv_host.cuh"

namespace lng {

static int check_kv8(const lng_kv8_cache* c, const int32_t* cu, int64_t tokens, int64_t max_new) {
  LNG_REQUIRE(c != nullptr, "cache descriptor is NULL");
  if (const int st = check_kv(&c->pages, cu, tokens, max_new)) return st;
  LNG_REQUIRE(c->pages.head_dim % 16 == 0, "head_dim of an 8-bit cache must be a multiple of 16");
  LNG_REQUIRE(c->pages.page_size <= 256, "page_size of an 8-bit cache must be at most 256");
  if (tokens == 0 || c->pages.batch == 0) return LNG_OK;
  LNG_REQUIRE(c->k_exp && c->v_exp, "NULL pointer in the cache descriptor");
  LNG_REQUIRE(c->k_exp_stride >= c->pages.num_kv_heads && c->v_exp_stride >= c->pages.num_kv_heads,
              "the exponents' strides must be at least num_kv_heads");
  for (int64_t s : {c->pages.k_page_stride, c->pages.k_head_stride, c->pages.k_slot_stride, c->pages.v_page_stride,
                    c->pages.v_head_stride, c->pages.v_slot_stride})
    LNG_REQUIRE(s % 16 == 0, "strides of an 8-bit cache must be multiples of 16 bytes");
  return LNG_OK;
}

static Kv8View kv8_view(const lng_kv8_cache* c, const int32_t* cu, int64_t tokens, int64_t max_new) {
  return Kv8View{kv_view(&c->pages, cu, tokens, max_new), c->k_exp, c->v_exp, c->k_exp_stride, c->v_exp_stride};
}

// The tensor map of the pages' bytes: one head's slots of one page a copy, the whole head wide (columns behind head_dim
// fill with zeros), rows of 64 or 128 bytes.
static int kv8_page_map(CUtensorMap* map, const lng_kv_cache& c, void* base, int64_t page, int64_t head, int64_t slot, int box) {
  auto enc = tensor_map_encoder();
  if (!enc) return fail(LNG_ERR_CUDA, "cuTensorMapEncodeTiled is unavailable (driver entry point)");
  const bool wide = c.head_dim > 64;
  const cuuint64_t dims[4] = {cuuint64_t(c.head_dim), cuuint64_t(c.page_size), cuuint64_t(c.num_kv_heads), cuuint64_t(c.num_pages)};
  const cuuint64_t strides[3] = {cuuint64_t(slot), cuuint64_t(head), cuuint64_t(page)};
  const cuuint32_t box4[4] = {wide ? 128u : 64u, cuuint32_t(box), 1, 1}, one[4] = {1, 1, 1, 1};
  const CUresult r = enc(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 4, base, dims, strides, box4, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
                         wide ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                         CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return fail(LNG_ERR_CUDA, "cuTensorMapEncodeTiled failed: " + std::to_string(int(r)));
  return LNG_OK;
}
static int kv8_page_maps(CUtensorMap* k, CUtensorMap* v, const lng_kv_cache& c, int box) {
  const int st = kv8_page_map(k, c, c.k, c.k_page_stride, c.k_head_stride, c.k_slot_stride, box);
  return st ? st : kv8_page_map(v, c, c.v, c.v_page_stride, c.v_head_stride, c.v_slot_stride, box);
}

// How an attention call is carried out, and what it needs of the workspace.
struct Kv8Plan {
  int groups;        // by kv8_step_kernel (few rows a key head), of so many groups of eight; 0:
  int shares;        // into which the step kernel's work is cut
  bool warp_shares;  // a share a warp, not a CTA
  int64_t units;     // by kv8_tile_kernel: its units per key head and range of keys
  int splits;        // key ranges, whose states are joined when there are several
  size_t ml, o, bytes;  // states: of the step kernel's pieces, or of the rows in every range
};
static Kv8Plan kv8_plan(const lng_kv8_cache* cache, int64_t tokens, int64_t max_new, int64_t max_len, int32_t q_heads, int32_t window,
                        int32_t sinks) {
  Kv8Plan p{};
  if (!cache || tokens <= 0 || cache->pages.batch <= 0 || cache->pages.num_kv_heads <= 0 || q_heads < cache->pages.num_kv_heads || max_new <= 0)
    return p;
  const lng_kv_cache& c = cache->pages;
  const int64_t group = q_heads / c.num_kv_heads;
  size_t states = 0;
  const int64_t rows = group * max_new, pairs = c.batch * c.num_kv_heads, span = 2 * std::max<int64_t>(1, KT_BM / group);
  int64_t keys = c.max_pages * c.page_size;
  if (max_len > 0) keys = std::min(keys, max_len);
  if (window > 0) keys = std::min(keys, int64_t(window) + sinks + span + KT_BK);
  // Up to four rows the step kernel always, up to 16 unless so few pairs fall into many pieces each (one sequence of 4000
  // keys, 4 key heads of 64, 16 rows: 31 against 19 us by the tile kernel), up to 32 where there are pairs for all SMs: 64
  // sequences of 1024 keys, 4 heads of 64: 45 against 51 us, 8 of 128: 92 against 119, of 8000 keys 349 against 572; but 16
  // sequences of 1024 keys 61 against 33.  (64 rows as two pairs of 32 were no faster than the tile kernel, 51 and 51, 144
  // and 120 us.)
  if (rows <= 4 || (rows <= 16 && pairs * 16 >= num_sms()) || (rows <= 32 && pairs >= num_sms()))
    p.groups = rows <= 8 ? 1 : rows <= 16 ? 2 : 4;
  if (p.groups) {
    // (many pairs: a share a warp; few pairs: a share a CTA, which leaves a twelfth or an eighth of the pieces to join)
    p.warp_shares = pairs >= num_sms() || p.groups > 2;
    const int warps = p.groups == 1 ? K8sCfg<64, 1>::WARPS : K8sCfg<64, 2>::WARPS;
    p.shares = num_sms() * (p.warp_shares ? warps : 1);
    // (no more shares than give every warp of a CTA a block: fewer pieces to join)
    if (!p.warp_shares) p.shares = int(std::max<int64_t>(1, std::min<int64_t>(p.shares, ceil_div(pairs * (ceil_div(keys, 32) + 1), warps))));
    states = size_t(2) * p.shares * 8 * p.groups;
  } else {
    // ragged steps: at most one unit a sequence is not full
    p.units = std::min(c.batch * ceil_div(max_new, span), tokens / span + std::min(c.batch, tokens));
    p.splits = kv_splits(p.units * c.num_kv_heads, std::max<int64_t>(1, ceil_div(keys, KT_BK)));
    if (p.splits > 1) states = size_t(p.splits) * tokens * q_heads;
  }
  p.o = al256(states * 8);
  p.bytes = p.o + al256(states * c.head_dim * 4);
  return p;
}

template <typename T, int HDP, int NR, bool WS>
static int launch_kv8_step(const CUtensorMap& tk, const CUtensorMap& tv, const K8sParams& p, cudaStream_t s) {
  using Cfg = K8sCfg<HDP, NR>;
  auto kern = kv8_step_kernel<T, HDP, NR, WS>;
  static std::atomic<uint64_t> known{0};
  if (const int st = allow_smem(kern, Cfg::SMEM, known)) return st;
  kern<<<unsigned(p.s.shares / (WS ? Cfg::WARPS : 1)), Cfg::THREADS, Cfg::SMEM, s>>>(tk, tv, p);
  LNG_LAUNCHED("kv8_step_kernel");
  return launch_dependent(kv_step_join_kernel<T, Cfg::BK>, unsigned(p.s.c.batch * p.s.c.kv_heads), 256u, size_t(0), s, p.s);
}

template <typename T, int HDP>
static int launch_kv8_tile(const CUtensorMap& tk, const CUtensorMap& tv, const K8tParams& p, cudaStream_t s) {
  using Cfg = K8tCfg<HDP>;
  auto kern = kv8_tile_kernel<T, HDP>;
  static std::atomic<uint64_t> known{0};
  if (const int st = allow_smem(kern, Cfg::SMEM, known)) return st;
  kern<<<unsigned(std::min<int64_t>(p.t.total, num_sms())), K8T_THREADS, Cfg::SMEM, s>>>(tk, tv, p);
  LNG_LAUNCHED("kv8_tile_kernel");
  if (p.t.row_ml == nullptr) return LNG_OK;
  return launch_dependent(kv_rows_join_kernel<T>, unsigned(ceil_div(p.t.c.tokens * p.t.q_heads, 8)), 256u, size_t(0), s, p.t.c,
                          p.t.q_heads, static_cast<const float2*>(p.t.row_ml), static_cast<const float*>(p.t.row_o), p.t.splits, p.t.o);
}

}  // namespace lng

using namespace lng;

extern "C" int lng_kv8_append(const lng_kv8_cache* cache, const int32_t* cu, int64_t tokens, int64_t max_new,
                              const lng_kv_rows* k, const lng_kv_rows* v, const lng_kv_rows* q, const lng_kv_rows* q_out,
                              const int64_t* positions, const float* inv_freq, int32_t rotary_dim, int32_t interleaved,
                              lng_stream_t stream) {
  int st = check_kv8(cache, cu, tokens, max_new);
  if (st) return st;
  const lng_kv_cache& c = cache->pages;
  LNG_REQUIRE(rotary_dim >= 0 && rotary_dim % 2 == 0 && rotary_dim <= c.head_dim, "rotary_dim must be even and at most head_dim");
  LNG_REQUIRE((q == nullptr) == (q_out == nullptr), "q and q_out go together");
  if (tokens == 0 || c.batch == 0) return LNG_OK;
  LNG_REQUIRE(rotary_dim == 0 || inv_freq != nullptr, "inv_freq is NULL");
  if ((st = check_kv_rows(k, c.num_kv_heads, "k")) || (st = check_kv_rows(v, c.num_kv_heads, "v"))) return st;
  if (q && ((st = check_kv_rows(q, 0, "q")) || (st = check_kv_rows(q_out, q->heads, "q_out")))) return st;
  LNG_REQUIRE(!q || q->ptr != q_out->ptr || (q->token_stride == q_out->token_stride && q->head_stride == q_out->head_stride),
              "q_out must be q itself or not overlap it");
  const bool bf16 = c.dtype == LNG_BF16;
  K8AppendParams p{};
  p.v = kv8_view(cache, cu, tokens, max_new);
  p.kr = kv_rows(k), p.vr = kv_rows(v);
  p.rotary = rotary_dim;
  p.interleaved = interleaved;
  p.positions = positions;
  p.inv_freq = inv_freq;
  p.items = c.head_dim / 16;
  p.items_magic = uint32_t((uint64_t(1) << 32) / uint32_t(p.items) + 1);
  p.per = int32_t((max_new + 2 * c.page_size - 2) / c.page_size);  // floor((max_new - 1 + page - 1) / page) + 1
  p.units = cu ? tokens / c.page_size + 2 * c.batch : c.batch * p.per;
  LNG_REQUIRE(p.units < (int64_t(1) << 31), "the step touches too many pages");
  // a page's new tokens in registers: as many warps a head as four items a lane need, or as leave none idle
  const int64_t most = std::min<int64_t>(c.page_size, max_new);
  const bool keep = c.page_size <= K8A_CHUNK && (interleaved || rotary_dim % 16 == 0);
  p.head_warps = 1;
  while (p.head_warps * 32 * K8A_KEEP < most * p.items || (p.head_warps * c.num_kv_heads < K8A_WARPS && p.head_warps * 32 < most * p.items))
    p.head_warps *= 2;
  p.head_warps = std::min(p.head_warps, K8A_WARPS);
  const int64_t per_cta = keep ? K8A_WARPS / p.head_warps : K8A_WARPS;
  const dim3 grid{unsigned(p.units), unsigned(2 * ceil_div(c.num_kv_heads, per_cta)), 1u};
  LNG_REQUIRE(grid.y <= 65535, "too many key heads");
  const size_t smem = size_t(std::min<int64_t>(K8A_CHUNK, most)) * (rotary_dim / 2) * sizeof(float2);
  if (q) {  // the queries: kv_append_kernel without a key head; keys and values are launched beside it
    KaParams a{};
    a.c = p.v.c;
    a.c.kv_heads = 0;
    a.qr = kv_rows(q), a.qo = kv_rows(q_out);
    a.q_heads = q->heads;
    a.rotary = rotary_dim;
    a.interleaved = interleaved;
    a.positions = positions;
    a.inv_freq = inv_freq;
    a.items = (c.head_dim / 8 + 1) / 2;
    a.items_magic = uint32_t((uint64_t(1) << 32) / uint32_t(a.items) + 1);
    const int64_t rounds = ceil_div(int64_t(a.q_heads) * a.items, int64_t(32));
    a.parts = int32_t(std::max<int64_t>(1, std::min<int64_t>(rounds, int64_t(num_sms()) * 8 / tokens)));
    const unsigned blocks = unsigned(ceil_div(tokens * a.parts, int64_t(KA_WARPS)));
    if (bf16)
      kv_append_kernel<__nv_bfloat16><<<blocks, KA_WARPS * 32, 0, S(stream)>>>(a);
    else
      kv_append_kernel<__half><<<blocks, KA_WARPS * 32, 0, S(stream)>>>(a);
    LNG_LAUNCHED("kv_append_kernel");
  }
  auto kern = bf16 ? (keep ? kv8_append_kernel<__nv_bfloat16, true> : kv8_append_kernel<__nv_bfloat16, false>)
                   : (keep ? kv8_append_kernel<__half, true> : kv8_append_kernel<__half, false>);
  if (q) return launch_dependent(kern, grid, unsigned(K8A_THREADS), smem, S(stream), p);
  kern<<<grid, K8A_THREADS, smem, S(stream)>>>(p);
  LNG_LAUNCHED("kv8_append_kernel");
  return LNG_OK;
}

extern "C" int lng_kv8_values(const lng_kv8_cache* cache, void* k_out, void* v_out, lng_stream_t stream) {
  LNG_REQUIRE(cache != nullptr, "cache descriptor is NULL");
  lng_kv8_cache one = *cache;
  one.pages.batch = 1;  // (neither table nor lengths are read)
  one.pages.lengths = reinterpret_cast<const int32_t*>(16);
  one.pages.table = reinterpret_cast<const int32_t*>(16);
  if (const int st = check_kv8(&one, nullptr, 1, 1)) return st;
  LNG_REQUIRE(((reinterpret_cast<uintptr_t>(k_out) | reinterpret_cast<uintptr_t>(v_out)) & 15) == 0, "outputs must be 16-byte aligned");
  const lng_kv_cache& c = cache->pages;
  K8ValuesParams p{};
  while ((1 << p.page_shift) < c.page_size) ++p.page_shift;
  p.pages[0] = static_cast<const uint8_t*>(c.k), p.pages[1] = static_cast<const uint8_t*>(c.v);
  p.page[0] = c.k_page_stride, p.page[1] = c.v_page_stride;
  p.head[0] = c.k_head_stride, p.head[1] = c.v_head_stride;
  p.slot[0] = c.k_slot_stride, p.slot[1] = c.v_slot_stride;
  p.exps[0] = cache->k_exp, p.exps[1] = cache->v_exp;
  p.exp_page[0] = cache->k_exp_stride, p.exp_page[1] = cache->v_exp_stride;
  p.out[0] = static_cast<uint4*>(k_out), p.out[1] = static_cast<uint4*>(v_out);
  p.heads = c.num_kv_heads;
  p.vecs = c.head_dim / 16;
  p.total = c.num_pages * c.num_kv_heads * c.page_size * p.vecs;
  LNG_REQUIRE(ceil_div(p.total, 256) < (int64_t(1) << 31), "the cache is too large");
  const dim3 grid{unsigned(ceil_div(p.total, 256)), 2u, 1u};
  kv8_values_kernel<<<grid, 256, 0, S(stream)>>>(p);
  LNG_LAUNCHED("kv8_values_kernel");
  return LNG_OK;
}

extern "C" size_t lng_kv8_attend_workspace_bytes(const lng_kv8_cache* cache, int64_t tokens, int64_t max_new, int64_t max_len,
                                                 int32_t q_heads, int32_t window, int32_t sinks) {
  return kv8_plan(cache, tokens, max_new, max_len, q_heads, window, sinks).bytes;
}

extern "C" int lng_kv8_attend(const lng_kv8_cache* cache, const int32_t* cu, int64_t tokens, int64_t max_new, int64_t max_len,
                              const lng_kv_rows* q, float scale, int32_t window, int32_t sinks, const lng_kv_rows* out,
                              void* workspace, size_t workspace_bytes, lng_stream_t stream) {
  int st = check_kv8(cache, cu, tokens, max_new);
  if (st) return st;
  const lng_kv_cache& c = cache->pages;
  LNG_REQUIRE(max_len >= 0, "max_len must not be negative");
  LNG_REQUIRE(window >= 0 && sinks >= 0, "window and sinks must not be negative");
  const float scale_log2 = scale * 1.4426950408889634f;
  LNG_REQUIRE(scale > 0.f && std::isfinite(scale_log2), "scale must be positive, and scale * log2(e) finite");
  if (tokens == 0 || c.batch == 0) return LNG_OK;
  if ((st = check_kv_rows(q, 0, "q"))) return st;
  LNG_REQUIRE(q->heads % c.num_kv_heads == 0 && q->heads / c.num_kv_heads <= 128,
              "query heads must be a multiple of the key heads, at most 128 a key head");
  if ((st = check_kv_rows(out, q->heads, "out"))) return st;
  LNG_REQUIRE(out->ptr != q->ptr, "out must not overlap q");
  LNG_REQUIRE(c.batch * c.num_kv_heads < (int64_t(1) << 31), "batch * num_kv_heads must be below 2^31");
  const Kv8Plan plan = kv8_plan(cache, tokens, max_new, max_len, q->heads, window, sinks);
  LNG_REQUIRE(plan.bytes == 0 || (workspace != nullptr && (reinterpret_cast<uintptr_t>(workspace) & 255) == 0),
              "workspace must be 256-byte aligned");
  LNG_REQUIRE(workspace_bytes >= plan.bytes, "workspace too small");
  if (plan.groups) {
    uint8_t* ws = static_cast<uint8_t*>(workspace);
    K8sParams p{};
    p.s.c = kv_view(&c, cu, tokens, max_new);
    p.s.q = kv_rows(q), p.s.o = kv_rows(out);
    p.s.q_heads = q->heads;
    p.s.group = q->heads / c.num_kv_heads;
    p.s.scale_log2 = scale_log2;
    p.s.window = std::min(window, 1 << 30);
    p.s.sinks = std::min(sinks, 1 << 30);
    p.s.box = std::min(c.page_size, K8sCfg<64, 1>::BK);
    p.s.piece_ml = reinterpret_cast<float2*>(ws + plan.ml);
    p.s.piece_o = reinterpret_cast<float*>(ws + plan.o);
    p.s.piece_rows = 8 * plan.groups;
    p.s.shares = plan.shares;
    p.k_exp = cache->k_exp, p.v_exp = cache->v_exp;
    p.k_exp_page = cache->k_exp_stride, p.v_exp_page = cache->v_exp_stride;
    CUtensorMap tk, tv;
    if ((st = kv8_page_maps(&tk, &tv, c, p.s.box))) return st;
    const bool wide = c.head_dim > 64;
    auto launch = [&](auto type) {
      using T = decltype(type);
      const bool ws = plan.warp_shares;
      const cudaStream_t cs = S(stream);
      switch (plan.groups) {
        case 1:
          if (wide) return ws ? launch_kv8_step<T, 128, 1, true>(tk, tv, p, cs) : launch_kv8_step<T, 128, 1, false>(tk, tv, p, cs);
          return ws ? launch_kv8_step<T, 64, 1, true>(tk, tv, p, cs) : launch_kv8_step<T, 64, 1, false>(tk, tv, p, cs);
        case 2:
          if (wide) return ws ? launch_kv8_step<T, 128, 2, true>(tk, tv, p, cs) : launch_kv8_step<T, 128, 2, false>(tk, tv, p, cs);
          return ws ? launch_kv8_step<T, 64, 2, true>(tk, tv, p, cs) : launch_kv8_step<T, 64, 2, false>(tk, tv, p, cs);
        default: return wide ? launch_kv8_step<T, 128, 4, true>(tk, tv, p, cs) : launch_kv8_step<T, 64, 4, true>(tk, tv, p, cs);
      }
    };
    return c.dtype == LNG_BF16 ? launch(__nv_bfloat16()) : launch(__half());
  }
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  K8tParams p{};
  p.t.c = kv_view(&c, cu, tokens, max_new);
  p.t.o = kv_rows(out);
  p.q = kv_rows(q);
  p.t.q_heads = q->heads;
  p.t.group = q->heads / c.num_kv_heads;
  p.t.tile_tokens = KT_BM / p.t.group;
  p.t.scale_log2 = scale_log2;
  p.t.window = std::min(window, 1 << 30);
  p.t.sinks = std::min(sinks, 1 << 30);
  p.t.box = std::min(c.page_size, KT_BK);
  p.t.splits = plan.splits;
  p.t.total = plan.units * c.num_kv_heads * plan.splits;
  if (plan.splits > 1) {
    p.t.row_ml = reinterpret_cast<float2*>(ws + plan.ml);
    p.t.row_o = reinterpret_cast<float*>(ws + plan.o);
  }
  p.k_exp = cache->k_exp, p.v_exp = cache->v_exp;
  p.k_exp_page = cache->k_exp_stride, p.v_exp_page = cache->v_exp_stride;
  CUtensorMap tk, tv;
  if ((st = kv8_page_maps(&tk, &tv, c, p.t.box))) return st;
  const bool wide = c.head_dim > 64;
  auto launch = [&](auto type) {
    using T = decltype(type);
    return wide ? launch_kv8_tile<T, 128>(tk, tv, p, S(stream)) : launch_kv8_tile<T, 64>(tk, tv, p, S(stream));
  };
  return c.dtype == LNG_BF16 ? launch(__nv_bfloat16()) : launch(__half());
}
