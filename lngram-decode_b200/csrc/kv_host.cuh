// Host side of the paged caches' entries: what they check, the kernels' view of a cache, launches.
#pragma once

#include <algorithm>
#include <atomic>
#include <cmath>

#include "kvcache.cuh"
#include "tc_prims.cuh"

namespace lng {

static cudaStream_t S(lng_stream_t s) { return reinterpret_cast<cudaStream_t>(s); }

static int check_kv(const lng_kv_cache* c, const int32_t* cu, int64_t tokens, int64_t max_new) {
  LNG_REQUIRE(c != nullptr, "cache descriptor is NULL");
  LNG_REQUIRE(c->dtype == LNG_BF16 || c->dtype == LNG_F16, "cache dtype must be bf16 or f16");
  LNG_REQUIRE(c->page_size >= 8 && c->page_size <= 4096 && (c->page_size & (c->page_size - 1)) == 0,
              "page_size must be a power of two in [8, 4096]");
  LNG_REQUIRE(c->num_pages >= 1 && c->num_pages < (int64_t(1) << 31), "num_pages must be in [1, 2^31)");
  LNG_REQUIRE(c->num_kv_heads >= 1 && c->num_kv_heads <= 65535, "num_kv_heads must be in [1, 65535]");
  LNG_REQUIRE(c->head_dim >= 8 && c->head_dim <= 128 && c->head_dim % 8 == 0, "head_dim must be a multiple of 8 up to 128");
  LNG_REQUIRE(c->batch >= 0 && c->max_pages >= 0, "batch and max_pages must not be negative");
  LNG_REQUIRE(c->max_pages < (int64_t(1) << 30) / c->page_size, "max_pages * page_size must be below 2^30");
  LNG_REQUIRE(c->table_stride >= c->max_pages, "table_stride must be at least max_pages");
  LNG_REQUIRE(max_new >= 0 && max_new < (int64_t(1) << 30), "max_new must be in [0, 2^30)");
  LNG_REQUIRE(tokens >= 0 && tokens < (int64_t(1) << 31), "tokens must be in [0, 2^31)");
  LNG_REQUIRE(cu != nullptr || tokens == c->batch * max_new, "without cu, tokens must be batch * max_new");
  if (tokens == 0 || c->batch == 0) return LNG_OK;
  LNG_REQUIRE(max_new >= 1, "max_new must be positive");
  LNG_REQUIRE(c->k && c->v && c->lengths && (c->table || c->max_pages == 0), "NULL pointer in the cache descriptor");
  LNG_REQUIRE(((reinterpret_cast<uintptr_t>(c->k) | reinterpret_cast<uintptr_t>(c->v)) & 15) == 0,
              "k and v must be 16-byte aligned");
  for (int64_t s : {c->k_page_stride, c->k_head_stride, c->k_slot_stride, c->v_page_stride, c->v_head_stride, c->v_slot_stride})
    LNG_REQUIRE(s > 0 && s % 8 == 0 && s < (int64_t(1) << 38), "cache strides must be positive multiples of 8 elements");
  return LNG_OK;
}

static int check_kv_rows(const lng_kv_rows* r, int64_t heads, const char* what) {
  const std::string w(what);
  LNG_REQUIRE(r != nullptr && r->ptr != nullptr, w + " is NULL");
  LNG_REQUIRE(heads <= 0 || r->heads == heads, w + ": wrong number of heads");
  LNG_REQUIRE(r->heads >= 1 && r->heads <= (1 << 20), w + ": heads must be positive");
  LNG_REQUIRE((reinterpret_cast<uintptr_t>(r->ptr) & 15) == 0, w + " must be 16-byte aligned");
  LNG_REQUIRE(r->token_stride > 0 && r->token_stride % 8 == 0 && r->head_stride > 0 && r->head_stride % 8 == 0 &&
                  r->token_stride < (int64_t(1) << 38) && r->head_stride < (int64_t(1) << 38),
              w + ": strides must be positive multiples of 8 elements");
  return LNG_OK;
}

static KvView kv_view(const lng_kv_cache* c, const int32_t* cu, int64_t tokens, int64_t max_new) {
  KvView v{};
  v.k = c->k;
  v.v = c->v;
  v.k_page = c->k_page_stride;
  v.k_head = c->k_head_stride;
  v.k_slot = c->k_slot_stride;
  v.v_page = c->v_page_stride;
  v.v_head = c->v_head_stride;
  v.v_slot = c->v_slot_stride;
  v.table = c->table;
  v.table_stride = c->table_stride;
  v.num_pages = c->num_pages;
  v.lengths = c->lengths;
  v.cu = cu;
  v.batch = c->batch;
  v.tokens = tokens;
  v.kv_heads = c->num_kv_heads;
  v.head_dim = c->head_dim;
  for (v.page_shift = 0; (1 << v.page_shift) < c->page_size; ++v.page_shift) {
  }
  v.capacity = int32_t(c->max_pages * c->page_size);
  v.max_new = int32_t(max_new);
  return v;
}

static KvRows kv_rows(const lng_kv_rows* r) { return r ? KvRows{r->ptr, r->token_stride, r->head_stride} : KvRows{}; }

// Into how many key ranges units with up to `tiles` key tiles each are divided: one where the units alone fill the
// SMs, else the count with the least estimated time, in tiles -- waves of units (one an SM) times (a range's
// tiles + 8 for a unit's start and its state's way out), plus the join of the states.
static int kv_splits(int64_t units, int64_t tiles) {
  const int64_t sms = num_sms();
  int best = 1;
  if (units >= sms) return best;
  double least = 1e300;
  for (int s = 1; s <= 32 && s <= tiles; ++s) {
    const double cost = double(ceil_div(units * s, sms)) * (ceil_div(tiles, s) + 8) + (s > 1 ? 4 + s * 0.5 : 0.0);
    if (cost < least) {
      least = cost;
      best = s;
    }
  }
  return best;
}

// Lets a kernel use so much dynamic shared memory, once a device (known: a bit for each).
template <typename K>
static int allow_smem(K kern, size_t bytes, std::atomic<uint64_t>& known) {
  int dev = 0;
  LNG_CUDA(cudaGetDevice(&dev));
  const uint64_t bit = dev < 64 ? uint64_t(1) << dev : 0;
  if (known.load(std::memory_order_relaxed) & bit) return LNG_OK;
  LNG_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, int(bytes)));
  known.fetch_or(bit, std::memory_order_relaxed);
  return LNG_OK;
}

// A launch that may start while the kernel before it in the stream still runs (griddepcontrol in both).
template <typename... Params, typename... Args>
static int launch_dependent(void (*kern)(Params...), dim3 grid, unsigned threads, size_t smem, cudaStream_t s, Args... args) {
  cudaLaunchAttribute pdl[1];
  pdl[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  pdl[0].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cfg.attrs = pdl;
  cfg.numAttrs = 1;
  LNG_CUDA(cudaLaunchKernelEx(&cfg, kern, args...));
  return LNG_OK;
}

}  // namespace lng
