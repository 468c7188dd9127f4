// kvs_paged_ops.cpp -- entry points and argument checks of the operators on a paged KV cache
// (include/kvs.h). Nothing here allocates, throws or touches a device before the checks passed.
#include "kvs_paged_ops.cuh"

#include <cuda_runtime.h>

#include <cmath>
#include <cstdarg>
#include <cstdio>

#include "kvs.h"
#include "kvs_kernels.cuh"

namespace {

int fail(int code, const char *fmt, ...) {
  char buf[512];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(buf, sizeof buf, fmt, ap);
  va_end(ap);
  kvs::set_last_error(buf);
  if (code == KVS_E_CUDA) cudaGetLastError();  // reported here, and by no later launch
  return code;
}

#define CHECK(cond, ...)                                   \
  do {                                                     \
    if (!(cond)) return fail(KVS_E_INVAL, __VA_ARGS__);    \
  } while (0)
#define TRY(x)                     \
  do {                             \
    const int rc_ = (x);           \
    if (rc_ != KVS_OK) return rc_; \
  } while (0)
#define CUDA_TRY(x, op)                                                                            \
  do {                                                                                             \
    const cudaError_t e_ = (x);                                                                    \
    if (e_ != cudaSuccess) return fail(KVS_E_CUDA, "%s: %s", op, cudaGetErrorString(e_));          \
  } while (0)

// Makes the tensors' device current for one call.
struct OnDevice {
  int prev = -1, dev;
  explicit OnDevice(int d) : dev(d) {
    cudaGetDevice(&prev);
    if (prev != dev) cudaSetDevice(dev);
  }
  ~OnDevice() {
    if (prev >= 0 && prev != dev) cudaSetDevice(prev);
  }
};

// The device all pointers of a call live on.
struct Where {
  const char *op;
  int device = -1;
  int add(const void *ptr, const char *name) {
    cudaPointerAttributes a{};
    if (!ptr || cudaPointerGetAttributes(&a, ptr) != cudaSuccess || a.type != cudaMemoryTypeDevice) {
      cudaGetLastError();
      return fail(KVS_E_INVAL, "%s: %s must be on device!", op, name);
    }
    CHECK((reinterpret_cast<uintptr_t>(ptr) & 3) == 0, "%s: %s must start on a 4-byte boundary", op, name);
    if (device < 0) device = a.device;
    CHECK(a.device == device, "%s: All tensors must be on the same device!", op);
    return KVS_OK;
  }
};

bool aligned16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }
bool strides16(const int64_t *s, int n) {
  for (int i = 0; i < n; ++i)
    if (s[i] % 16 || s[i] < 0) return false;
  return true;
}

int check_cache(const kvs_paged_cache *c, const char *op, kvs::PagedCache *out) {
  CHECK(c, "%s: the cache is null", op);
  CHECK(c->dtype == KVS_DTYPE_BF16 || c->dtype == KVS_DTYPE_FP16 || c->dtype == KVS_DTYPE_E4M3,
        "%s: cache type %d is not bf16, fp16 or e4m3", op, c->dtype);
  CHECK(c->batch > 0, "%s: page_table must have at least one row", op);
  CHECK(c->batch <= 65535 && c->n_heads <= 65535, "%s: at most 65535 requests and KV heads", op);
  CHECK(c->num_blocks > 0 && c->n_heads > 0 && c->block_size > 0 && c->max_blocks > 0,
        "%s: num_blocks, num_kv_heads, block_size and max_num_blocks_per_seq must be > 0", op);
  CHECK(c->num_blocks <= 0x7FFFFFFFu, "%s: num_blocks must be below 2^31", op);
  const uint32_t step = c->dtype == KVS_DTYPE_E4M3 ? 16 : 8;
  CHECK(c->head_dim > 0 && c->head_dim <= 256 && c->head_dim % step == 0,
        "%s: head_dim (%u) must be a multiple of %u up to 256", op, c->head_dim, step);
  CHECK((uint64_t)c->max_blocks * c->block_size <= 0x7FFFFFFFull,
        "%s: a page-table row must cover fewer than 2^31 tokens", op);
  CHECK(c->k && c->v && c->page_table, "%s: cache_k, cache_v or page_table must be on device!", op);
  CHECK(aligned16(c->k) && aligned16(c->v) && strides16(c->k_strides, 3) && strides16(c->v_strides, 3),
        "%s: cache rows must start on 16-byte boundaries, with strides that are not negative", op);
  CHECK(std::isfinite(c->k_scale) && std::isfinite(c->v_scale) && c->k_scale > 0 && c->v_scale > 0,
        "%s: k_scale and v_scale must be positive and finite", op);
  CHECK(std::isfinite(1.f / c->k_scale) && std::isfinite(1.f / c->v_scale),
        "%s: k_scale and v_scale must have a finite reciprocal", op);
  CHECK(c->dtype == KVS_DTYPE_E4M3 || (c->k_scale == 1.f && c->v_scale == 1.f),
        "%s: k_scale and v_scale belong to an e4m3 cache", op);
  *out = kvs::PagedCache{static_cast<uint8_t *>(c->k), static_cast<uint8_t *>(c->v),
                         c->k_strides[0], c->k_strides[1], c->k_strides[2],
                         c->v_strides[0], c->v_strides[1], c->v_strides[2],
                         c->page_table, c->num_blocks, c->n_heads, c->block_size, c->head_dim, c->batch, c->max_blocks,
                         c->dtype, c->k_scale, c->v_scale};
  return KVS_OK;
}

// Dimensions of what a call writes: none of several elements may have stride 0 (a broadcast view).
bool spread(const int64_t *strides, uint64_t n0, uint64_t n1) { return (n0 <= 1 || strides[0]) && (n1 <= 1 || strides[1]); }
// A sum read and written at one address is read and written by the same strides.
int check_sums(const kvs_paged_cache *c, const float *w, const int64_t *ws, const float *out, const int64_t *os, const char *op) {
  CHECK(w != out || ((c->batch <= 1 || ws[0] == os[0]) && (c->n_heads <= 1 || ws[1] == os[1])),
        "%s: weights_out must be weights itself or not overlap it", op);
  return KVS_OK;
}
int check_written(const kvs_paged_cache *c, const char *op) {
  CHECK(spread(c->k_strides, c->num_blocks, c->n_heads) && spread(c->v_strides, c->num_blocks, c->n_heads) &&
            (c->block_size <= 1 || (c->k_strides[2] && c->v_strides[2])),
        "%s: cache_k and cache_v must not be broadcast", op);
  return KVS_OK;
}

int check_row_type(int32_t dtype, int32_t cache, const char *op) {
  CHECK(dtype == KVS_DTYPE_BF16 || dtype == KVS_DTYPE_FP16, "%s: rows must be bf16 or fp16", op);
  CHECK(cache == KVS_DTYPE_E4M3 || cache == dtype, "%s: rows and cache must have the same type (or the cache e4m3)", op);
  return KVS_OK;
}

int add_cache(Where &w, const kvs_paged_cache *c) {
  TRY(w.add(c->k, "cache_k"));
  TRY(w.add(c->v, "cache_v"));
  return w.add(c->page_table, "page_table");
}

int sms_of(int device, int *sms, const char *op) {
  CUDA_TRY(cudaDeviceGetAttribute(sms, cudaDevAttrMultiProcessorCount, device), op);
  return KVS_OK;
}

int check_decode(const kvs_paged_cache *cache, const kvs_decode_rows *r, const char *op, kvs::PagedCache *c) {
  TRY(check_cache(cache, op, c));
  CHECK(r, "%s: the rows are null", op);
  TRY(check_row_type(r->dtype, cache->dtype, op));
  CHECK(r->q_heads > 0 && r->q_heads % c->n_heads == 0, "%s: q heads (%u) must be a multiple of the KV heads (%u)", op,
        r->q_heads, c->n_heads);
  CHECK(r->q_heads / c->n_heads <= 1024, "%s: at most 1024 query heads per KV head", op);
  return KVS_OK;
}

}  // namespace

extern "C" {

int kvs_qk_norm_rope_fill(const kvs_paged_cache *cache, const kvs_qkv_rows *r, void *stream) {
  const char *op = "qk_norm_rope_fill";
  kvs::QkvFillParams p{};
  TRY(check_cache(cache, op, &p.c));
  CHECK(r, "%s: the rows are null", op);
  TRY(check_row_type(r->dtype, cache->dtype, op));
  CHECK(r->q_heads > 0 && r->q_heads <= 65535, "%s: q heads must be 1 to 65535", op);
  CHECK(r->n_tokens <= 0x7FFFFFFFu / 2, "%s: too many tokens", op);
  CHECK(r->rotary > 0 && r->rotary % 8 == 0 && r->rotary <= cache->head_dim, "%s: rotary (%u) must be a multiple of 8 up to head_dim", op, r->rotary);
  CHECK(r->n_positions > 0, "%s: cos_sin must have at least one row", op);
  CHECK(r->positions ? r->n_axes >= 1 && r->n_axes <= 32 : r->axes == nullptr, "%s: 1 to 32 axes of positions, and axes only with positions", op);
  CHECK(aligned16(r->q) && aligned16(r->k) && aligned16(r->v) && aligned16(r->q_out) && strides16(r->q_strides, 2) &&
            strides16(r->k_strides, 2) && strides16(r->v_strides, 2) && strides16(r->q_out_strides, 2),
        "%s: q, k, v and q_out rows must start on 16-byte boundaries", op);
  CHECK(aligned16(r->cos_sin) && aligned16(r->q_weight) && aligned16(r->k_weight) && aligned16(r->axes),
        "%s: cos_sin, axes and weights must start on 16-byte boundaries", op);
  CHECK(std::isfinite(r->eps) && r->eps >= 0, "%s: eps must be finite and not negative", op);
  TRY(check_written(cache, op));
  CHECK(spread(r->q_out_strides, r->n_tokens, r->q_heads), "%s: q_out must not be broadcast", op);
  if (r->n_tokens == 0) return KVS_OK;
  Where w{op};
  TRY(add_cache(w, cache));
  TRY(w.add(r->q, "q"));
  TRY(w.add(r->k, "k"));
  TRY(w.add(r->v, "v"));
  TRY(w.add(r->q_out, "q_out"));
  TRY(w.add(r->cos_sin, "cos_sin"));
  TRY(w.add(r->cu_seqlens, "cu_seqlens"));
  TRY(w.add(r->start_positions, "start_positions"));
  if (r->positions) TRY(w.add(r->positions, "positions"));
  if (r->axes) TRY(w.add(r->axes, "axes"));
  if (r->q_weight) TRY(w.add(r->q_weight, "q_weight"));
  if (r->k_weight) TRY(w.add(r->k_weight, "k_weight"));
  if (r->out_of_range) TRY(w.add(r->out_of_range, "out_of_range"));
  int sms = 0;
  TRY(sms_of(w.device, &sms, op));
  OnDevice on(w.device);
  p.q = static_cast<const uint8_t *>(r->q);
  p.k = static_cast<const uint8_t *>(r->k);
  p.v = static_cast<const uint8_t *>(r->v);
  p.q_out = static_cast<uint8_t *>(r->q_out);
  p.q_tok = r->q_strides[0], p.q_head = r->q_strides[1];
  p.k_tok = r->k_strides[0], p.k_head = r->k_strides[1];
  p.v_tok = r->v_strides[0], p.v_head = r->v_strides[1];
  p.o_tok = r->q_out_strides[0], p.o_head = r->q_out_strides[1];
  p.cos_sin = r->cos_sin;
  p.cu_seqlens = r->cu_seqlens;
  p.start = r->start_positions;
  p.positions = r->positions;
  p.axes = r->axes;
  p.q_weight = r->q_weight;
  p.k_weight = r->k_weight;
  p.out_of_range = r->out_of_range;
  p.tokens = r->n_tokens;
  p.q_heads = r->q_heads;
  p.rotary = r->rotary;
  p.n_positions = r->n_positions;
  p.n_axes = r->positions ? r->n_axes : 1;
  p.dtype = r->dtype;
  p.eps = r->eps;
  p.interleaved = r->interleaved;
  p.zero_rest = r->zero_rest;
  p.page = kvs::Divisor(p.c.block_size);
  CUDA_TRY(kvs::launch_qkv_fill(p, sms, static_cast<cudaStream_t>(stream)), op);
  return KVS_OK;
}

int kvs_decode_attention_workspace(const kvs_paged_cache *cache, const kvs_decode_rows *r, int32_t device, uint64_t *bytes) {
  const char *op = "decode_attention_workspace";
  kvs::PagedCache c{};
  CHECK(bytes, "%s: null output", op);
  TRY(check_decode(cache, r, op, &c));
  int sms = 0;
  TRY(sms_of(device, &sms, op));
  *bytes = kvs::decode_attention_workspace(c, r->q_heads, r->weights_out != nullptr, sms);
  return KVS_OK;
}

int kvs_paged_decode_attention(const kvs_paged_cache *cache, const kvs_decode_rows *r, void *stream) {
  const char *op = "paged_decode_attention";
  kvs::DecodeAttentionParams p{};
  TRY(check_decode(cache, r, op, &p.c));
  CHECK(aligned16(r->q) && aligned16(r->out) && strides16(r->q_strides, 2) && strides16(r->out_strides, 2),
        "%s: q and out rows must start on 16-byte boundaries", op);
  CHECK(std::isfinite(r->scale), "%s: scale must be finite", op);
  CHECK(spread(r->out_strides, cache->batch, r->q_heads), "%s: out must not be broadcast", op);
  CHECK(!r->weights_out || spread(r->weights_out_strides, cache->batch, cache->n_heads), "%s: weights_out must not be broadcast", op);
  CHECK((r->weights == nullptr) == (r->weights_out == nullptr), "%s: weights and weights_out go together", op);
  CHECK(!r->weights || r->w_len >= (uint64_t)cache->max_blocks * cache->block_size,
        "%s: weights must cover max_num_blocks_per_seq * block_size tokens", op);
  if (r->weights) TRY(check_sums(cache, r->weights, r->weights_strides, r->weights_out, r->weights_out_strides, op));
  CHECK((reinterpret_cast<uintptr_t>(r->workspace) & 255) == 0, "%s: workspace must be 256-byte aligned", op);
  Where w{op};
  TRY(add_cache(w, cache));
  TRY(w.add(r->q, "q"));
  TRY(w.add(r->out, "out"));
  TRY(w.add(r->seq_lens, "seq_lens"));
  TRY(w.add(r->workspace, "workspace"));
  if (r->lse) TRY(w.add(r->lse, "lse"));
  if (r->weights) {
    TRY(w.add(r->weights, "weights"));
    TRY(w.add(r->weights_out, "weights_out"));
  }
  int sms = 0;
  TRY(sms_of(w.device, &sms, op));
  const uint64_t need = kvs::decode_attention_workspace(p.c, r->q_heads, r->weights_out != nullptr, sms);
  CHECK(r->workspace_bytes >= need, "%s: workspace of %llu bytes, %llu are needed", op,
        (unsigned long long)r->workspace_bytes, (unsigned long long)need);
  OnDevice on(w.device);
  p.q = static_cast<const uint8_t *>(r->q);
  p.out = static_cast<uint8_t *>(r->out);
  p.q_req = r->q_strides[0], p.q_head = r->q_strides[1];
  p.o_req = r->out_strides[0], p.o_head = r->out_strides[1];
  p.seq_lens = r->seq_lens;
  p.lse = r->lse;
  p.weights = r->weights;
  p.weights_out = r->weights_out;
  p.w_req = r->weights_strides[0], p.w_head = r->weights_strides[1];
  p.wo_req = r->weights_out_strides[0], p.wo_head = r->weights_out_strides[1];
  p.w_len = r->w_len;
  p.q_heads = r->q_heads;
  p.window = r->window;
  p.dtype = r->dtype;
  p.scale = r->scale;
  p.workspace = static_cast<uint8_t *>(r->workspace);
  CUDA_TRY(kvs::launch_decode_attention(p, sms, static_cast<cudaStream_t>(stream)), op);
  return KVS_OK;
}

int kvs_evict_paged(const kvs_paged_cache *cache, const kvs_evict_rows *r, void *stream) {
  const char *op = "evict_paged";
  kvs::EvictParams p{};
  TRY(check_cache(cache, op, &p.c));
  CHECK(r, "%s: the rows are null", op);
  TRY(check_written(cache, op));
  CHECK(spread(r->weights_out_strides, cache->batch, cache->n_heads), "%s: weights_out must not be broadcast", op);
  CHECK(r->keep > 0 && r->keep <= 0x7FFFFFFFu, "%s: keep must be 1 to 2^31 - 1", op);
  CHECK((uint64_t)r->first + r->recent <= r->keep, "%s: first (%u) + recent (%u) must be <= keep (%u)", op, r->first,
        r->recent, r->keep);
  const uint64_t cap = (uint64_t)cache->max_blocks * cache->block_size;
  CHECK(!r->dst_table || (uint64_t)r->dst_blocks * cache->block_size >= (r->keep < cap ? r->keep : cap),
        "%s: dst_page_table must cover keep (%u) slots", op, r->keep);
  // the page table itself: in place
  const bool in_place = !r->dst_table || r->dst_table == cache->page_table;
  CHECK(!r->dst_table || !in_place || r->dst_blocks == cache->max_blocks || cache->batch == 1,
        "%s: dst_page_table must be page_table itself or name fresh pages", op);
  CHECK(r->w_len >= cap && r->wo_len >= cap, "%s: weights must cover max_num_blocks_per_seq * block_size tokens", op);
  CHECK((uint64_t)cache->batch * cache->n_heads <= 0x7FFFFFFFull / 8, "%s: too many requests and heads", op);
  TRY(check_sums(cache, r->weights, r->weights_strides, r->weights_out, r->weights_out_strides, op));
  Where w{op};
  TRY(add_cache(w, cache));
  TRY(w.add(r->seq_lens, "seq_lens"));
  if (!in_place) TRY(w.add(r->dst_table, "dst_page_table"));
  TRY(w.add(r->weights, "weights"));
  TRY(w.add(r->weights_out, "weights_out"));
  TRY(w.add(r->kept, "kept"));
  TRY(w.add(r->new_lens, "new_lens"));
  if (r->out_of_range) TRY(w.add(r->out_of_range, "out_of_range"));
  int sms = 0;
  TRY(sms_of(w.device, &sms, op));
  OnDevice on(w.device);
  p.seq_lens = r->seq_lens;
  p.dst_table = in_place ? nullptr : r->dst_table;
  p.dst_blocks = r->dst_blocks;
  p.weights = r->weights;
  p.weights_out = r->weights_out;
  p.w_req = r->weights_strides[0], p.w_head = r->weights_strides[1];
  p.wo_req = r->weights_out_strides[0], p.wo_head = r->weights_out_strides[1];
  p.keep = r->keep;
  p.first = r->first;
  p.recent = r->recent;
  p.kept = r->kept;
  p.new_lens = r->new_lens;
  p.out_of_range = r->out_of_range;
  p.page = kvs::Divisor(p.c.block_size);
  p.row_bytes = cache->head_dim * (cache->dtype == KVS_DTYPE_E4M3 ? 1 : 2);
  p.words = kvs::Divisor(p.row_bytes / 16);
  CUDA_TRY(kvs::launch_evict(p, sms, static_cast<cudaStream_t>(stream)), op);
  return KVS_OK;
}

}  // extern "C"
