// kvs_paged_ops.cuh -- parameters and launchers of the operators that compute on a paged KV cache:
//   * qkv_fill (kvs_qkv_fill.cu): norms of queries and keys per head, rotation by the token's
//     position, and the write of K and V rows into the cache;
//   * decode_attention (kvs_decode_attention.cu): attention of one new token per request over the
//     cache, split over its length and joined;
//   * evict (kvs_evict.cu): per request and KV head, the tokens of the largest accumulated weight
//     and the move of their rows to the front of a page table.
// The entry points and their argument checks are in kvs_paged_ops.cpp.
#pragma once

#include <cstdint>
#include <cuda_runtime.h>

namespace kvs {

// Element types of rows (KVS_DTYPE_* of kvs.h).
enum : int32_t { kBf16 = 0, kFp16 = 1, kE4m3 = 2 };

// Division of numbers below 2^31 by one divisor: a product and a shift. For l = ceil(log2 d) and
// m = ceil(2^(31 + l) / d), m < 2^32 and floor(n m / 2^(31 + l)) = floor(n / d) for n < 2^31.
struct Divisor {
  uint32_t d, m, shift;
  Divisor() = default;
  explicit Divisor(uint32_t by) : d(by), m(0), shift(0) {
    uint32_t l = 0;
    while ((1ull << l) < by) ++l;
    if (l == 0) return;  // by one: n itself
    m = (uint32_t)(((1ull << (31 + l)) + by - 1) / by);
    shift = l - 1;
  }
#ifdef __CUDACC__
  __device__ __forceinline__ uint32_t quotient(uint32_t n) const { return d == 1 ? n : __umulhi(n, m) >> shift; }
  __device__ __forceinline__ uint32_t rest(uint32_t n, uint32_t q) const { return n - q * d; }
#endif
};

// A paged cache as the kernels address it: row (page, head, slot) of K starts at
// k + page * k_page + head * k_head + slot * k_row (bytes), so any page layout with contiguous
// rows works. Page-table entries <= 0 hold nothing, entries >= num_blocks are out of range.
struct PagedCache {
  uint8_t *k, *v;
  int64_t k_page, k_head, k_row, v_page, v_head, v_row;
  const int32_t *page_table;  // [batch][max_blocks]
  uint32_t num_blocks, n_heads, block_size, head_dim, batch, max_blocks;
  int32_t dtype;
  float k_scale, v_scale;  // an e4m3 cache holds value / scale
};

#ifdef __CUDACC__
// Page of virtual block `vb` of request `b`: > 0, or 0 (nothing there), or -1 (out of range).
__device__ __forceinline__ int32_t page_of(const PagedCache &c, uint32_t b, uint32_t vb) {
  if (vb >= c.max_blocks) return -1;
  const int32_t p = __ldg(c.page_table + (uint64_t)b * c.max_blocks + vb);
  return p <= 0 ? 0 : ((uint32_t)p < c.num_blocks ? p : -1);
}
#endif

struct QkvFillParams {
  PagedCache c;
  const uint8_t *q, *k, *v;  // [tokens][heads][head_dim], bytes between tokens and heads below
  uint8_t *q_out;
  int64_t q_tok, q_head, k_tok, k_head, v_tok, v_head, o_tok, o_head;
  const float *cos_sin;         // [positions][rotary]: cos of rotary / 2 frequencies, then sin
  const int32_t *cu_seqlens;    // [batch + 1], -1 padded
  const int32_t *start;         // [batch]
  const int32_t *positions;     // [n_axes][tokens], or nullptr: the token's cache position
  const int32_t *axes;          // [rotary / 2]: axis of each frequency, or nullptr: axis 0
  const void *q_weight, *k_weight;  // [head_dim] of the rows' type, or nullptr: no norm
  uint32_t *out_of_range;       // optional counter of tokens that were skipped
  uint32_t tokens, q_heads, rotary, n_positions, n_axes;
  int32_t dtype;                // of q, k, v and q_out
  float eps;
  int interleaved, zero_rest;
  Divisor page;                 // block_size
};
cudaError_t launch_qkv_fill(const QkvFillParams &p, int sms, cudaStream_t stream);

struct DecodeAttentionParams {
  PagedCache c;
  const uint8_t *q;
  uint8_t *out;
  int64_t q_req, q_head, o_req, o_head;  // bytes
  const int32_t *seq_lens;
  float *lse;                 // [batch][q_heads] or nullptr
  const float *weights;       // [batch][n_heads][w_len], w_req / w_head elements apart; or nullptr
  float *weights_out;
  int64_t w_req, w_head, wo_req, wo_head;
  uint32_t w_len;
  uint32_t q_heads, window;   // window 0: every token
  int32_t dtype;              // of q and out
  float scale;                // of the scores, the cache's k_scale not yet in it
  uint8_t *workspace;         // decode_attention_workspace(...) bytes, 256-byte aligned
};
// Bytes of workspace a call needs; the same function lays it out.
uint64_t decode_attention_workspace(const PagedCache &c, uint32_t q_heads, bool weights, int sms);
cudaError_t launch_decode_attention(const DecodeAttentionParams &p, int sms, cudaStream_t stream);

struct EvictParams {
  PagedCache c;
  const int32_t *seq_lens;
  const int32_t *dst_table;   // [batch][dst_blocks], or nullptr: in place
  uint32_t dst_blocks;
  const float *weights;
  float *weights_out;
  int64_t w_req, w_head, wo_req, wo_head;
  uint32_t keep, first, recent;
  int32_t *kept;              // [batch][n_heads][keep]
  int32_t *new_lens;          // [batch]
  uint32_t *out_of_range;
  uint32_t row_bytes;
  Divisor page;               // block_size
  Divisor words;              // 16-byte words of a row
  bool vector_weights;        // rows of weights start on 16-byte boundaries
};
cudaError_t launch_evict(const EvictParams &p, int sms, cudaStream_t stream);

}  // namespace kvs
