// The C ABI's entries of the paged cache in 8 bits (include/lngram_b200.h).
#include "kv8.cuh"
#include "kv_host.cuh"

namespace lng {

int error_word_kv8(int clear) { return error_word_here(clear); }

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
  p.per = int32_t((max_new + 2 * c.page_size - 2) / c.page_size);  // floor((max_new - 1 + page - 1) / page) + 1
  p.units = cu ? tokens / c.page_size + 2 * c.batch : c.batch * p.per;
  LNG_REQUIRE(p.units < (int64_t(1) << 31), "the step touches too many pages");
  p.head_chunk = int32_t(p.units * ceil_div(c.num_kv_heads, K8A_HEADS) * 2 >= 2 * num_sms() ? K8A_HEADS : K8A_THREADS / 32);
  if (p.head_chunk > c.num_kv_heads) p.head_chunk = c.num_kv_heads;
  const dim3 grid(unsigned(p.units), unsigned(2 * ceil_div(c.num_kv_heads, p.head_chunk)));
  LNG_REQUIRE(grid.y <= 65535, "too many key heads");
  const size_t smem = size_t(std::min<int64_t>(K8A_CHUNK, std::min<int64_t>(c.page_size, max_new))) * (rotary_dim / 2) * sizeof(float2);
  if (bf16)
    kv8_append_kernel<__nv_bfloat16><<<grid, K8A_THREADS, smem, S(stream)>>>(p);
  else
    kv8_append_kernel<__half><<<grid, K8A_THREADS, smem, S(stream)>>>(p);
  LNG_LAUNCHED("kv8_append_kernel");
  if (!q) return LNG_OK;
  // the queries: kv_append_kernel without a key head
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
  int shift = 0;
  while ((1 << shift) < c.page_size) ++shift;
  const int vecs = c.head_dim / 16;
  const int64_t total = c.num_pages * c.num_kv_heads * c.page_size * vecs;
  LNG_REQUIRE(ceil_div(total, 256) < (int64_t(1) << 31), "the cache is too large");
  const unsigned grid = unsigned(ceil_div(total, 256));
  if (k_out)
    kv8_values_kernel<<<grid, 256, 0, S(stream)>>>(static_cast<const uint8_t*>(c.k), c.k_page_stride, c.k_head_stride, c.k_slot_stride,
                                                  cache->k_exp, cache->k_exp_stride, c.num_kv_heads, shift, vecs, total,
                                                  static_cast<uint4*>(k_out));
  if (v_out)
    kv8_values_kernel<<<grid, 256, 0, S(stream)>>>(static_cast<const uint8_t*>(c.v), c.v_page_stride, c.v_head_stride, c.v_slot_stride,
                                                  cache->v_exp, cache->v_exp_stride, c.num_kv_heads, shift, vecs, total,
                                                  static_cast<uint4*>(v_out));
  LNG_LAUNCHED("kv8_values_kernel");
  return LNG_OK;
}

extern "C" size_t lng_kv8_attend_workspace_bytes(const lng_kv8_cache* cache, int64_t tokens, int64_t max_new, int64_t max_len,
                                                 int32_t q_heads, int32_t window, int32_t sinks) {
  return 0;
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
  K8RowParams p{};
  p.v = kv8_view(cache, cu, tokens, max_new);
  p.q = kv_rows(q), p.o = kv_rows(out);
  p.q_heads = q->heads;
  p.group = q->heads / c.num_kv_heads;
  p.scale_log2 = scale_log2;
  p.window = std::min(window, 1 << 30);
  p.sinks = std::min(sinks, 1 << 30);
  const unsigned grid = unsigned(ceil_div(tokens * q->heads, 8));
  if (c.dtype == LNG_BF16)
    kv8_row_kernel<__nv_bfloat16><<<grid, 256, 0, S(stream)>>>(p);
  else
    kv8_row_kernel<__half><<<grid, 256, 0, S(stream)>>>(p);
  LNG_LAUNCHED("kv8_row_kernel");
  return LNG_OK;
}
