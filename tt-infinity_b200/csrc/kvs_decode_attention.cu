// kvs_decode_attention.cu -- attention of one new token per request over a paged KV cache.
//
// For request b, query head g of KV head h and the tokens t that have a page and lie in
// [max(0, L - window), L):
//     s_t = scale * q . k_t      o = sum_t exp(s_t - m) v_t / sum_t exp(s_t - m)      m = max_t s_t
// in one pass over the cache with the running maximum and sum of the softmax.
//
// What bounds it: every valid K and V row is read once; the arithmetic is 2 * group flop per cache
// byte (16-bit cache), far below what the tensor cores do in the time the bytes take, so the kernel
// is built to keep loads in flight and instructions few:
//   * Each warp streams its own 16-token tiles of K and V through a private ring in shared memory
//     (16-byte cp.async, zero-filled where a token is masked, so that nothing a masked slot holds
//     -- infinities, NaN -- reaches the sums). No CTA barrier stands in the main loop, and the loads
//     run ahead of the products across the ends of requests and heads.
//   * The products run with the tokens as the rows of the matrix instruction: S^T = K Q^T
//     (16 tokens x 8 heads) and O^T = V^T P^T (16 elements x 8 heads), so a group of up to 8 heads
//     fills the 8 columns and no instruction works on padding rows; groups up to 16 take two column
//     tiles and larger ones several passes over the cache. (Memory is the bound: the tensor pipe is
//     busy 11 % of the time for a bf16 cache, 18 % for e4m3.)
//   * Work is split by tokens, not by request: the batch's tiles, in units of a few tiles, form one
//     sequence that is cut into equal runs, one per CTA, from lengths that only the device knows.
//     A (request, head) that spans several CTAs leaves partial sums that a second small kernel
//     joins, in the order of the sequence, so results do not depend on timing.
// Device times, with the share of the measured copy rate: 48 contexts up to 16384 tokens, 8 KV heads of
// 128, group 8, bf16: 234 us, 100 %; one of 131071: 88 us, 94 %; 64 up to 12001 from an e4m3 cache: 167 us,
// 81 % (token-major pages of 16: a head's rows are 128 bytes in every 1024), 144 us, 94 % from head-major
// pages.
//
// Scores, maxima, sums and accumulators are 32-bit. The probabilities are rounded to the cache's
// 16-bit type for the second product (fp16 for an e4m3 cache): each is off by at most half a step,
// as the output is once more. fp16 keeps that only down to 2^-14, and a long row's tokens may lie
// further below a first token that takes most of the attention, so fp16 probabilities are held 2^15
// times larger: half a step down to 2^-29 of the largest, 2^-40 of it below. (Rows of 512 tokens, the
// first one 15 / 17 / 19 nats above the others, of value 0: fp16 outputs are off by half a step; unscaled
// by 1.2 / 26 / 26 %. No time is lost to it.) An e4m3 cache is widened to fp16, which holds every e4m3
// value; the queries are scaled by a power of two per head to fit fp16.
#include "kvs_paged_ops.cuh"

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include <atomic>

#include "kvs_kernels.cuh"

namespace kvs {

namespace {

constexpr int kWarps = 4;
constexpr int kThreads = 32 * kWarps;
constexpr uint32_t kTile = 16;  // tokens per warp tile
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
// fp16 probabilities are 2^kLift times as large: at most 2^15 < 65504
constexpr float kLift = 15.f, kUnlift = 1.f / 32768.f;

enum Kind { kKindBf16, kKindFp16, kKindE4m3 };

// How a kernel streams: tiles in a warp's ring, bytes of a CTA's rings and CTAs per SM, by bytes per
// element, padded head_dim and column tiles of 8 heads. Rows of up to 128 bytes carry few bytes per
// instruction, so they get more warps where registers allow: 3 CTAs per SM with 64 KiB each (e4m3,
// head_dim 128, 64 mixed contexts up to 12001 tokens: 168 us against 171 us with 4 CTAs of 48 KiB and
// 172 us with 2 of 96 KiB). Longer rows take 2 CTAs of 96 KiB, and rows of 512 bytes one of 192 KiB,
// three tiles per warp being the least that keeps loads
// in flight while a tile is worked on.
struct Shape {
  int stages, ring, ctas;
};
__host__ __device__ constexpr Shape shape_of(int el, int dp, int nt) {
  Shape s{};
  const bool light = dp * el <= 128 && dp * nt <= 128;
  const int stage = 2 * 16 * dp * el, fit = (light ? 65536 : 98304) / (kWarps * stage);
  s.stages = fit < 3 ? 3 : (fit > 8 ? 8 : fit);
  s.ring = kWarps * s.stages * stage;
  s.ctas = s.ring > 110 * 1024 ? 1 : (light ? 3 : 2);
  return s;
}

template <int kKind, int DP, int NT>
struct Cfg {
  static constexpr int el = kKind == kKindE4m3 ? 1 : 2;
  static constexpr Shape shape = shape_of(el, DP, NT);
  static constexpr int pitch = DP * el;                 // bytes of a row in shared memory
  static constexpr int chunks = pitch / 16;             // 16-byte pieces of a row
  static constexpr int stage = 2 * (int)kTile * pitch;  // K and V of one tile
  static constexpr int stages = shape.stages;
  static constexpr int ring = shape.ring;
  static constexpr int ctas = shape.ctas;
  static constexpr int merge = NT * (DP / 16) * 512;    // one warp's accumulators
  static constexpr int smem = ring + merge + 512;       // the ring starts on a row boundary
  static constexpr int heads = 8 * NT;
};

// A (request, head tile) whose first units this CTA took and that goes on in `followers` more. A CTA
// leaves at most two partials: slot 1 where its last run goes on, slot 0 where its first run continues
// an earlier CTA's. A partial's accumulators lie in the order of the matrix fragments.
struct Join {
  uint32_t b, hh, followers, pad;
};

struct Plan {  // workspace layout
  uint64_t joins, part_o, part_ml, lse2, parts, logits, bytes;
  uint32_t grid, head_tiles, tile_heads, unit_tiles, least_units;
  bool joins_needed, narrow;
};

__host__ __device__ inline uint32_t head_tiles_of(uint32_t group) { return (group + 15) / 16; }

inline uint32_t padded_dim(uint32_t d) { return d <= 64 ? 64 : (d <= 128 ? 128 : 256); }

Plan plan_of(const PagedCache &c, uint32_t q_heads, bool weights, int sms) {
  Plan p{};
  const uint32_t group = q_heads / c.n_heads;
  p.head_tiles = head_tiles_of(group);
  p.tile_heads = group <= 8 ? 8 : 16;
  const uint32_t dp = padded_dim(c.head_dim);
  const uint32_t per_sm = shape_of(c.dtype == kE4m3 ? 1 : 2, dp, p.tile_heads / 8).ctas;
  const uint64_t cap = (uint64_t)c.max_blocks * c.block_size;
  const uint32_t cap_tiles = (uint32_t)((cap + kTile - 1) / kTile);
  // Runs are cut at units of 64 tokens, and a CTA takes 128 tokens at least where requests are at most
  // 2048 tokens long, else 256: shorter runs leave more parts to join (one request, one KV head, 32768
  // tokens: 13.8 us, with 128 tokens at least 19.4 us; one request of 1024 tokens, 8 heads: 9.5 us with
  // 256, 8.5 us with 128). Short requests are not cut at all, which saves the join: 2 requests of up to
  // 193 tokens 7.2 us against 9.1 us, 16 of up to 300 8.0 us against 11.1 us; but one of 500 tokens, 8
  // heads, 9.8 us against 7.7 us, so above 256 tokens only where the GPU has enough of them.
  const uint64_t tiles = (uint64_t)c.batch * c.n_heads * p.head_tiles;
  const bool whole = cap <= 256 || (cap <= 512 && 4 * tiles >= (uint64_t)sms);
  p.unit_tiles = whole ? cap_tiles : 4;
  p.least_units = whole ? 1 : (cap <= 2048 ? 2 : 4);
  const uint64_t units = (cap_tiles + p.unit_tiles - 1) / p.unit_tiles;
  const uint64_t most = (tiles * units + p.least_units - 1) / p.least_units;
  const uint64_t full = (uint64_t)sms * per_sm;
  p.grid = (uint32_t)(most < full ? most : full);
  p.joins_needed = units > 1 && p.grid > 1;
  p.narrow = c.batch <= kThreads && tiles * units < 1ull << 31;
  uint64_t off = 0;
  auto take = [&](uint64_t n) {
    const uint64_t o = off;
    off += (n + 255) & ~255ull;
    return o;
  };
  p.joins = take((uint64_t)p.grid * sizeof(Join));
  p.part_o = take(2ull * p.grid * p.tile_heads * dp * 4);
  p.part_ml = take(2ull * p.grid * p.tile_heads * 8);
  p.lse2 = take(weights ? 4ull * c.batch * q_heads : 0);
  p.parts = take(8ull * c.batch * c.n_heads * p.head_tiles);
  p.logits = take(weights ? 4ull * c.batch * q_heads * cap : 0);
  p.bytes = off;
  return p;
}

struct KernelParams {
  DecodeAttentionParams a;
  Join *joins;
  float *part_o;
  float2 *part_ml;
  float *lse2;    // base-2 log-sum-exp of the rows that were not split, kept for the weights
  float *logits;  // [batch][n_heads][cap][group] scores in base 2, or nullptr
  uint2 *parts;   // [batch][head tiles]: first CTA and how many more hold a part
  uint32_t cap, head_tiles, group, unit_tiles, least_units, join_blocks, pieces, join_parts, weight_chunk;
  bool narrow;   // at most kThreads requests, and all counts of units fit 32 bits
  Divisor page;  // block_size
};

__device__ __forceinline__ uint32_t smem_addr(const void *p) { return (uint32_t)__cvta_generic_to_shared(p); }

__device__ __forceinline__ void cp16(uint32_t dst, const void *src, bool there) {
  // src-size 0 reads nothing and writes zeros
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(there ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp16(uint32_t dst, const void *src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int n>
__device__ __forceinline__ void cp_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(n) : "memory"); }

__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t a) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a) : "memory");
}
__device__ __forceinline__ void ldsm4t(uint32_t (&r)[4], uint32_t a) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a) : "memory");
}
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
template <bool kBf>
__device__ __forceinline__ void mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  if (kBf)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
template <bool kBf>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  if (kBf) {
    const __nv_bfloat162 x = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t *>(&x);
  }
  const __half2 x = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t *>(&x);
}
// Two e4m3 values (the low 16 bits) as fp16.
__device__ __forceinline__ uint32_t widen(uint32_t x) {
  uint32_t y;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(y) : "h"((uint16_t)x));
  return y;
}
__device__ __forceinline__ float2 pair_of(uint32_t x, bool bf) {
  if (bf) return make_float2(__uint_as_float(x << 16), __uint_as_float(x & 0xFFFF0000u));
  return __half22float2(*reinterpret_cast<const __half2 *>(&x));
}
__device__ __forceinline__ void store_elem(uint8_t *row, uint32_t d, float x, int32_t dtype) {
  if (dtype == kBf16) reinterpret_cast<__nv_bfloat16 *>(row)[d] = __float2bfloat16_rn(x);
  else reinterpret_cast<__half *>(row)[d] = __float2half_rn(x);
}

// Tiles of request b: [first, first + count) in units of kTile tokens from the cache's start.
struct Span {
  uint32_t low, len, first, tiles, units;
};
__device__ __forceinline__ Span span_of(const KernelParams &p, uint32_t b) {
  Span s;
  const int32_t n = __ldg(p.a.seq_lens + b);
  s.len = n <= 0 ? 0 : min((uint32_t)n, p.cap);
  // the window ends at the request's last token, also where the table covers fewer tokens
  const uint32_t whole = n <= 0 ? 0 : (uint32_t)n;
  s.low = p.a.window && whole > p.a.window ? whole - p.a.window : 0;
  if (s.low > s.len) s.low = s.len;
  s.first = s.low / kTile;
  s.tiles = s.len > s.low ? (s.len + kTile - 1) / kTile - s.first : 0;
  s.units = max(1u, (s.tiles + p.unit_tiles - 1) / p.unit_tiles);  // an empty row still gets its zeros written
  return s;
}

__device__ __forceinline__ float log2_sum(float m, float l) { return l == 0.f ? -INFINITY : m + __log2f(l); }
__device__ __forceinline__ void store_lse(const KernelParams &p, uint64_t row, float m, float l) {
  const float lse2 = log2_sum(m, l);
  if (p.a.lse) p.a.lse[row] = lse2 * kLn2;
  if (p.lse2) p.lse2[row] = lse2;
}

// Where a CTA is in its run of units: unit `unit` of head tile `hh` of request `b`, `left` units to go.
struct Cursor {
  uint32_t b, hh, unit;
  uint64_t left;
  Span span;
  __device__ __forceinline__ uint32_t take() const { return (uint32_t)min((uint64_t)(span.units - unit), left); }
  __device__ __forceinline__ uint32_t begin(const KernelParams &p) const { return span.first + unit * p.unit_tiles; }
  __device__ __forceinline__ uint32_t end(const KernelParams &p) const { return span.first + min(span.tiles, (unit + take()) * p.unit_tiles); }
  __device__ __forceinline__ void next(const KernelParams &p, uint32_t hh_n) {
    left -= take();
    unit = 0;
    if (++hh == hh_n) {
      hh = 0;
      ++b;
      if (left) span = span_of(p, b);
    }
  }
};

// Factor that brings sums relative to maximum m to maximum M (sums without a token are zero; a NaN
// stays one).
__device__ __forceinline__ float rebase(float m, float l, float M) {
  return m == -INFINITY ? (l == 0.f ? 0.f : 1.f) : exp2_fast(m - M);
}

template <int kKind, int DP, int NT>
__global__ void __launch_bounds__(kThreads, (Cfg<kKind, DP, NT>::ctas)) decode_attention_kernel(const __grid_constant__ KernelParams p) {
  using C = Cfg<kKind, DP, NT>;
  constexpr bool kBf = kKind == kKindBf16;
  constexpr bool k8 = kKind == kKindE4m3;
  constexpr int kSteps = DP / 16;
  extern __shared__ uint8_t smem_raw[];
  uint8_t *const smem = smem_raw + (-smem_addr(smem_raw) & 511);
  __shared__ uint64_t s_scan[kWarps];
  __shared__ Cursor s_at;
  __shared__ uint32_t s_mask[kWarps][C::stages];
  __shared__ float s_m[C::heads], s_l[C::heads];
  const uint32_t tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const PagedCache &c = p.a.c;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

  // ---- this CTA's run of units
  const uint32_t hh_n = c.n_heads * p.head_tiles;
  if (tid == 0) p.joins[blockIdx.x].followers = 0;
  uint64_t quota;
  // The loads run ahead of the products, across the ends of runs: `ahead` is where the loads are.
  Cursor at;
  if (p.narrow) {  // one request per thread and 32-bit counts: one scan
    Span mine{};
    if (tid < c.batch) mine = span_of(p, tid);
    uint32_t incl = mine.units;
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t y = __shfl_up_sync(~0u, incl, o);
      if (lane >= o) incl += y;
    }
    if (lane == 31) s_scan[warp] = incl;
    __syncthreads();
    uint32_t total = 0;
    for (int w = 0; w < kWarps; ++w) {
      if (w < (int)warp) incl += (uint32_t)s_scan[w];
      total += (uint32_t)s_scan[w];
    }
    total *= hh_n;
    const uint32_t share = max(p.least_units, (total + gridDim.x - 1) / gridDim.x), begin = share * blockIdx.x;
    if (begin >= total) return;
    const uint32_t lo = (incl - mine.units) * hh_n;
    if (mine.units && lo <= begin && begin < incl * hh_n) {
      const uint32_t in = begin - lo, hh = in / mine.units;
      s_at = Cursor{tid, hh, in - hh * mine.units, min(share, total - begin), mine};
    }
    __syncthreads();
    at = s_at;
    quota = share;
  } else {
    uint64_t total = 0;
    for (uint32_t base = 0; base < c.batch; base += kThreads) {
      uint64_t x = base + tid < c.batch ? span_of(p, base + tid).units : 0;
      for (int o = 16; o; o >>= 1) x += __shfl_xor_sync(~0u, x, o);
      total += x;
    }
    if (lane == 0) s_scan[warp] = total;
    __syncthreads();
    total = 0;
    for (int w = 0; w < kWarps; ++w) total += s_scan[w];
    total *= hh_n;
    quota = max((uint64_t)p.least_units, (total + gridDim.x - 1) / gridDim.x);
    const uint64_t begin = quota * blockIdx.x;
    if (begin >= total) return;
    // request that holds unit `begin`: the requests' units times hh_n, scanned kThreads at a time
    uint64_t run = 0;
    for (uint32_t base = 0; base < c.batch; base += kThreads) {
      const uint64_t val = base + tid < c.batch ? span_of(p, base + tid).units : 0;
      uint64_t incl = val;
      for (int o = 1; o < 32; o <<= 1) {
        const uint64_t y = __shfl_up_sync(~0u, incl, o);
        if (lane >= o) incl += y;
      }
      __syncthreads();
      if (lane == 31) s_scan[warp] = incl;
      __syncthreads();
      uint64_t before = run, all = 0;
      for (int w = 0; w < kWarps; ++w) {
        if (w < (int)warp) before += s_scan[w];
        all += s_scan[w];
      }
      const uint64_t lo = (before + incl - val) * hh_n, hi = (before + incl) * hh_n;
      if (val && lo <= begin && begin < hi) {
        const uint64_t in = begin - lo;
        s_at = Cursor{base + tid, (uint32_t)(in / val), (uint32_t)(in % val), min(quota, total - begin), span_of(p, base + tid)};
      }
      run += all;
      __syncthreads();
      if (run * hh_n > begin) break;
    }
    at = s_at;
  }
  Cursor ahead = at;

  const uint32_t ring = smem_addr(smem) + warp * C::stages * C::stage;
  const uint32_t row_chunks = (c.head_dim * C::el + 15) / 16;
  const bool one_page = c.block_size % kTile == 0;  // a tile lies in one page
  const float scale2 = p.a.scale * c.k_scale * kLog2e;
  // The pieces of a tile this lane moves: piece lane % chunks of the rows lane / chunks + i * rows_step.
  // In shared memory piece j of row r sits at place j ^ swizzle(r) of the row, so that the eight rows
  // of a matrix load fall on different banks; the swizzle of a sum of disjoint bits is the xor of
  // theirs, which makes all but one term of each address a constant.
  constexpr uint32_t rows_step = 32 / C::chunks;
  static_assert(C::chunks <= 32, "a row is at most 512 bytes");
  const uint32_t my_chunk = lane % C::chunks, my_row = lane / C::chunks;
  auto swizzle = [](uint32_t row) constexpr -> uint32_t { return C::pitch >= 128 ? (row & 7) : ((row >> 1) & 3); };
  const uint32_t my_place = my_row * C::pitch + ((my_chunk ^ swizzle(my_row)) << 4);

  uint32_t bq[kSteps][NT][2];
  // Queries of a run, as they are in memory. The product's index 2j + {0, 1} of a step is element
  // 2j + {0, 1} (and 2j + 8 + {0, 1} eight further on); for an e4m3 cache 4j + {0, 1} (4j + 2 + {0, 1}),
  // the order in which four bytes of a key row come out of a matrix load.
  auto load_queries = [&](const Cursor &of) {
    const uint32_t first_head = of.hh / p.head_tiles * p.group, g_first = of.hh % p.head_tiles * C::heads;
    const uint32_t j = lane & 3;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const uint32_t g = g_first + nt * 8 + (lane >> 2);
      const uint32_t *qr = reinterpret_cast<const uint32_t *>(p.a.q + (int64_t)of.b * p.a.q_req + (int64_t)(first_head + g) * p.a.q_head);
#pragma unroll
      for (int s = 0; s < kSteps; ++s)
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          const uint32_t d = k8 ? 16 * s + 4 * j + 2 * half : 16 * s + 8 * half + 2 * j;
          bq[s][nt][half] = g < p.group && d < c.head_dim ? __ldg(qr + d / 2) : 0u;
        }
    }
  };
  // ---- loads
  uint32_t load_tile_at = ahead.begin(p) + warp, load_end = ahead.end(p);
  int32_t page;            // of the next tile to load; 0: masked
  uint32_t slot;           // this lane's token's (the tile's first token's) slot in its page
  const uint8_t *kh, *vh;  // this KV head's rows; this lane's piece of them where a tile lies in one page
  auto find_head = [&]() {
    const uint32_t h = ahead.hh / p.head_tiles;
    kh = c.k + (int64_t)h * c.k_head + my_chunk * 16;
    vh = c.v + (int64_t)h * c.v_head + my_chunk * 16;
  };
  auto find_page = [&]() {
    page = 0;
    slot = 0;
    if (load_tile_at >= load_end) return;
    // page of this lane's token (of the whole tile, where it lies in one page)
    const uint32_t t = load_tile_at * kTile + (one_page ? 0 : (lane & 15)), vb = p.page.quotient(t);
    slot = p.page.rest(t, vb);
    if (vb >= c.max_blocks) return;
    const int32_t pg = __ldg(c.page_table + (uint64_t)ahead.b * c.max_blocks + vb);
    page = pg > 0 && (uint32_t)pg < c.num_blocks ? pg : 0;
  };
  // to the next tile of this warp, through runs that have none for it
  auto settle = [&]() {
    while (load_tile_at >= load_end && ahead.left) {
      ahead.next(p, hh_n);
      if (!ahead.left) break;
      load_tile_at = ahead.begin(p) + warp;
      load_end = ahead.end(p);
      find_head();
    }
    if (ahead.left) find_page();
  };
  // one tile of K and V into shared memory, and which of its tokens count
  auto load_tile = [&](uint32_t kdst, uint32_t vdst, uint32_t *note) {
    const uint32_t t0 = load_tile_at * kTile;
    uint32_t mask = 0xFFFFu;
    if (t0 + kTile > ahead.span.len) mask = 0xFFFFu >> (t0 + kTile - ahead.span.len);
    if (t0 < ahead.span.low) mask &= 0xFFFFu << (ahead.span.low - t0);
    if (one_page) mask = page ? mask : 0;
    else mask &= __ballot_sync(~0u, page != 0);
    if (lane == 0) *note = mask;
    if (one_page && mask == 0xFFFFu) {
      if (my_chunk >= row_chunks) return;
      const uint8_t *ks = kh + (int64_t)page * c.k_page + (int64_t)(slot + my_row) * c.k_row;
      const uint8_t *vs = vh + (int64_t)page * c.v_page + (int64_t)(slot + my_row) * c.v_row;
      const int64_t kstep = rows_step * c.k_row, vstep = rows_step * c.v_row;
#pragma unroll
      for (uint32_t x = 0; x < kTile / rows_step; ++x) {
        const uint32_t to = (my_place ^ (swizzle(x * rows_step) << 4)) + x * rows_step * C::pitch;
        cp16(kdst + to, ks);
        cp16(vdst + to, vs);
        ks += kstep;
        vs += vstep;
      }
      return;
    }
    const int64_t ko = (int64_t)page * c.k_page + (int64_t)slot * c.k_row;
    const int64_t vo = (int64_t)page * c.v_page + (int64_t)slot * c.v_row;
#pragma unroll
    for (uint32_t x = 0; x < kTile / rows_step; ++x) {
      const uint32_t row = my_row + x * rows_step;
      int64_t kro = one_page ? ko + (int64_t)row * c.k_row : __shfl_sync(~0u, ko, row);
      int64_t vro = one_page ? vo + (int64_t)row * c.v_row : __shfl_sync(~0u, vo, row);
      const bool there = (mask >> row) & 1;
      kro = there ? kro : -(int64_t)my_chunk * 16;  // the address of a piece that is not read stays inside the cache
      vro = there ? vro : -(int64_t)my_chunk * 16;
      if (my_chunk < row_chunks) {
        const uint32_t to = (my_place ^ (swizzle(x * rows_step) << 4)) + x * rows_step * C::pitch;
        cp16(kdst + to, kh + kro, there);
        cp16(vdst + to, vh + vro, there);
      }
    }
  };
  // one tile's loads; past the last one the group is empty, so that groups keep counting
  auto issue = [&](uint32_t stage) {
    if (ahead.left) {
      const uint32_t kdst = ring + stage * C::stage;
      load_tile(kdst, kdst + kTile * C::pitch, &s_mask[warp][stage]);
      load_tile_at += kWarps;
      settle();
    }
    cp_commit();
  };
  // Rows shorter than the padded head_dim: the products run over zeros behind them, which no load
  // overwrites.
  if (row_chunks < C::chunks)
    for (uint32_t row = lane; row < C::stages * 2 * kTile; row += 32)
      for (uint32_t j = row_chunks; j < C::chunks; ++j)
        *reinterpret_cast<uint4 *>(smem + warp * C::stages * C::stage + row * C::pitch + ((j ^ swizzle(row)) << 4)) = make_uint4(0, 0, 0, 0);
  find_head();
  settle();
#pragma unroll
  for (int s = 0; s < C::stages - 1; ++s) issue(s);
  load_queries(at);
  uint32_t stage = 0;
  const uint32_t k_row = (lane & 7) + ((lane >> 3) & 1) * 8, v_row = (lane & 7) + (lane >> 4) * 8;
  const uint32_t k_place = k_row * C::pitch + (((lane >> 4) ^ swizzle(k_row)) << 4);
  const uint32_t v_place = v_row * C::pitch + ((((lane >> 3) & 1) ^ swizzle(v_row)) << 4);

  while (at.left) {
    const uint32_t b = at.b, h = at.hh / p.head_tiles, g0 = (at.hh % p.head_tiles) * C::heads;
    const uint32_t heads = min((uint32_t)C::heads, p.group - g0);
    const uint32_t t_begin = at.begin(p), t_end = at.end(p);

    // ---- queries (loaded before the last run's join): column fragments of Q^T, heads as columns
    float head_scale[NT][2];  // per column of the score tile (heads 2j, 2j + 1)
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      if (!k8) {
        head_scale[nt][0] = head_scale[nt][1] = scale2;
      } else {
        // scaled by a power of two so that the head's largest element is in [1, 2), which fits fp16:
        // elements below 2^-14 of it lose at most 2^-25 of it
        const bool bf = p.a.dtype == kBf16;
        float big = 0.f;
#pragma unroll
        for (int s = 0; s < kSteps; ++s)
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            const float2 x = pair_of(bq[s][nt][half], bf);
            big = fmaxf(big, fmaxf(fabsf(x.x), fabsf(x.y)));
          }
        big = fmaxf(big, __shfl_xor_sync(~0u, big, 1));
        big = fmaxf(big, __shfl_xor_sync(~0u, big, 2));
        // both the factor 2^-e and 2^e have to be normal numbers
        int e = big > 0.f && big < __int_as_float(0x7f800000) ? (int)(__float_as_uint(big) >> 23) - 127 : 0;
        e = max(-126, min(126, e));
        const float down = __uint_as_float((uint32_t)(127 - e) << 23);
        const float up = __uint_as_float((uint32_t)(127 + e) << 23) * scale2;
#pragma unroll
        for (int s = 0; s < kSteps; ++s)
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            const float2 x = pair_of(bq[s][nt][half], bf);
            bq[s][nt][half] = pack2<false>(x.x * down, x.y * down);
          }
        head_scale[nt][0] = __shfl_sync(~0u, up, 8 * (lane & 3));
        head_scale[nt][1] = __shfl_sync(~0u, up, 8 * (lane & 3) + 4);
      }
    }

    float acc[NT][kSteps][4];
    float m[NT][2], l[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      m[nt][0] = m[nt][1] = -INFINITY;
      l[nt][0] = l[nt][1] = 0.f;
#pragma unroll
      for (int s = 0; s < kSteps; ++s)
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[nt][s][i] = 0.f;
    }

    for (uint32_t tile = t_begin + warp; tile < t_end; tile += kWarps) {
      cp_wait<C::stages - 2>();
      __syncwarp();
      issue(stage == 0 ? C::stages - 1 : stage - 1);
      const uint32_t kt = ring + stage * C::stage + k_place, vt = ring + stage * C::stage + kTile * C::pitch + v_place;

      // ---- S^T = K Q^T (two chains of products)
      float sc[NT][4];
      {
        float sd[NT][4];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int i = 0; i < 4; ++i) sc[nt][i] = sd[nt][i] = 0.f;
#pragma unroll
        for (int s = 0; s < kSteps; s += 2) {
          uint32_t a[4];
          if (!k8) {
            ldsm4(a, kt ^ (uint32_t)(s << 5));
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) mma<kBf>(sc[nt], a[0], a[1], a[2], a[3], bq[s][nt][0], bq[s][nt][1]);
            ldsm4(a, kt ^ (uint32_t)((s + 1) << 5));
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) mma<kBf>(sd[nt], a[0], a[1], a[2], a[3], bq[s + 1][nt][0], bq[s + 1][nt][1]);
          } else {
            ldsm4(a, kt ^ (uint32_t)(s << 4));
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              const uint32_t x0 = widen(a[2 * i]), x1 = widen(a[2 * i + 1]), x2 = widen(a[2 * i] >> 16), x3 = widen(a[2 * i + 1] >> 16);
#pragma unroll
              for (int nt = 0; nt < NT; ++nt) mma<false>(i ? sd[nt] : sc[nt], x0, x1, x2, x3, bq[s + i][nt][0], bq[s + i][nt][1]);
            }
          }
        }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int i = 0; i < 4; ++i) sc[nt][i] = (sc[nt][i] + sd[nt][i]) * head_scale[nt][i & 1];
      }

      // ---- running maximum and sum; tokens lane / 4 and lane / 4 + 8, heads 2j and 2j + 1
      const uint32_t mask = s_mask[warp][stage];
      if (mask != 0xFFFFu) {
        const bool in0 = (mask >> (lane >> 2)) & 1, in1 = (mask >> ((lane >> 2) + 8)) & 1;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            if (!in0) sc[nt][i] = -INFINITY;
            if (!in1) sc[nt][2 + i] = -INFINITY;
          }
      }
      bool grew = false;
      float mn[NT][2];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          float x = fmaxf(sc[nt][i], sc[nt][2 + i]);
          x = fmaxf(x, __shfl_xor_sync(~0u, x, 4));
          x = fmaxf(x, __shfl_xor_sync(~0u, x, 8));
          x = fmaxf(x, __shfl_xor_sync(~0u, x, 16));
          mn[nt][i] = fmaxf(m[nt][i], x);
          grew |= mn[nt][i] > m[nt][i];
        }
      if (p.logits) {
        const uint32_t t = tile * kTile + (lane >> 2);
        float *lg = p.logits + (((uint64_t)b * c.n_heads + h) * p.cap + t) * p.group + g0;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const uint32_t g = nt * 8 + 2 * (lane & 3);
            if (t + 8 * i >= at.span.len || g >= heads) continue;
            float *to = lg + 8ull * i * p.group + g;
            if (p.group % 2 == 0) {
              *reinterpret_cast<float2 *>(to) = make_float2(sc[nt][2 * i], sc[nt][2 * i + 1]);
            } else {
              to[0] = sc[nt][2 * i];
              if (g + 1 < heads) to[1] = sc[nt][2 * i + 1];
            }
          }
      }
      if (__any_sync(~0u, grew)) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const float f = mn[nt][i] == -INFINITY ? 0.f : exp2_fast(m[nt][i] - mn[nt][i]);
            m[nt][i] = mn[nt][i];
            l[nt][i] *= f;
#pragma unroll
            for (int s = 0; s < kSteps; ++s) {
              acc[nt][s][i] *= f;
              acc[nt][s][2 + i] *= f;
            }
          }
      }
      uint32_t pb[NT][2];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        float base0 = m[nt][0] == -INFINITY ? 0.f : m[nt][0], base1 = m[nt][1] == -INFINITY ? 0.f : m[nt][1];
        if constexpr (!kBf) base0 -= kLift, base1 -= kLift;
        const float e0 = exp2_fast(sc[nt][0] - base0), e1 = exp2_fast(sc[nt][1] - base1);
        const float e2 = exp2_fast(sc[nt][2] - base0), e3 = exp2_fast(sc[nt][3] - base1);
        l[nt][0] += e0 + e2;
        l[nt][1] += e1 + e3;
        pb[nt][0] = transpose8(pack2<kBf>(e0, e1));
        pb[nt][1] = transpose8(pack2<kBf>(e2, e3));
      }

      // ---- O^T += V^T P^T
      if (!k8) {
#pragma unroll
        for (int s = 0; s < kSteps; ++s) {
          uint32_t a[4];
          ldsm4t(a, vt ^ (uint32_t)(s << 5));
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) mma<kBf>(acc[nt][s], a[0], a[1], a[2], a[3], pb[nt][0], pb[nt][1]);
        }
      } else {
        // a transposed load of byte pairs gives (t0 d0, t0 d1, t1 d0, t1 d1): even elements become
        // rows 0-7 of the 16-element tile, odd ones rows 8-15
#pragma unroll
        for (int s = 0; s < kSteps; s += 2) {
          uint32_t a[4];
          ldsm4t(a, vt ^ (uint32_t)(s << 4));
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const uint32_t lo = __byte_perm(a[i], 0, 0x3120), hi = __byte_perm(a[2 + i], 0, 0x3120);
            const uint32_t x0 = widen(lo), x1 = widen(lo >> 16), x2 = widen(hi), x3 = widen(hi >> 16);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) mma<false>(acc[nt][s + i], x0, x1, x2, x3, pb[nt][0], pb[nt][1]);
          }
        }
      }
      stage = stage + 1 == C::stages ? 0 : stage + 1;
    }
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        l[nt][i] += __shfl_xor_sync(~0u, l[nt][i], 4);
        l[nt][i] += __shfl_xor_sync(~0u, l[nt][i], 8);
        l[nt][i] += __shfl_xor_sync(~0u, l[nt][i], 16);
        if constexpr (!kBf) {
          l[nt][i] *= kUnlift;  // exact: what follows knows nothing of the lift
#pragma unroll
          for (int s = 0; s < kSteps; ++s) {
            acc[nt][s][i] *= kUnlift;
            acc[nt][s][2 + i] *= kUnlift;
          }
        }
      }

    Cursor following = at;
    following.next(p, hh_n);
    if (following.left) load_queries(following);

    // ---- warp 0 takes in the other warps' sums, one after the other (those that had a step)
    float4 *const buf = reinterpret_cast<float4 *>(smem + C::ring);
    for (uint32_t w = 1; w < kWarps; ++w) {
      if (t_begin + w >= t_end) break;
      if (warp == w) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
          for (int s = 0; s < kSteps; ++s)
            buf[(nt * kSteps + s) * 32 + lane] = make_float4(acc[nt][s][0], acc[nt][s][1], acc[nt][s][2], acc[nt][s][3]);
          if (lane < 4) {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              s_m[nt * 8 + 2 * lane + i] = m[nt][i];
              s_l[nt * 8 + 2 * lane + i] = l[nt][i];
            }
          }
        }
      }
      __syncthreads();
      if (warp == 0) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          float f0[2], f1[2];
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const float mw = s_m[nt * 8 + 2 * (lane & 3) + i], lw = s_l[nt * 8 + 2 * (lane & 3) + i];
            const float M = fmaxf(m[nt][i], mw);
            f0[i] = rebase(m[nt][i], l[nt][i], M);
            f1[i] = rebase(mw, lw, M);
            m[nt][i] = M;
            l[nt][i] = l[nt][i] * f0[i] + lw * f1[i];
          }
#pragma unroll
          for (int s = 0; s < kSteps; ++s) {
            const float4 x = buf[(nt * kSteps + s) * 32 + lane];
            acc[nt][s][0] = acc[nt][s][0] * f0[0] + x.x * f1[0];
            acc[nt][s][1] = acc[nt][s][1] * f0[1] + x.y * f1[1];
            acc[nt][s][2] = acc[nt][s][2] * f0[0] + x.z * f1[0];
            acc[nt][s][3] = acc[nt][s][3] * f0[1] + x.w * f1[1];
          }
        }
      }
      __syncthreads();
    }
    if (warp == 0) {
      const bool starts = at.unit == 0, ends = at.unit + at.take() == at.span.units;
      if (starts && ends) {
        const uint32_t r = lane >> 2;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const uint32_t g = nt * 8 + 2 * (lane & 3) + i;
            if (g >= heads) continue;
            const float f = l[nt][i] == 0.f ? 0.f : c.v_scale / l[nt][i];
            uint8_t *o = p.a.out + (int64_t)b * p.a.o_req + (int64_t)(h * p.group + g0 + g) * p.a.o_head;
#pragma unroll
            for (int s = 0; s < kSteps; ++s) {
              const uint32_t d0 = 16 * s + (k8 ? 2 * r : r), d1 = 16 * s + (k8 ? 2 * r + 1 : r + 8);
              if (d0 < c.head_dim) store_elem(o, d0, acc[nt][s][i] * f, p.a.dtype);
              if (d1 < c.head_dim) store_elem(o, d1, acc[nt][s][2 + i] * f, p.a.dtype);
            }
            if (r == 0) store_lse(p, (uint64_t)b * p.a.q_heads + h * p.group + g0 + g, m[nt][i], l[nt][i]);
          }
      } else {
        const uint64_t slot = 2ull * blockIdx.x + (starts ? 1 : 0);
        float4 *po = reinterpret_cast<float4 *>(p.part_o) + slot * NT * kSteps * 32;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
          for (int s = 0; s < kSteps; ++s)
            po[(nt * kSteps + s) * 32 + lane] = make_float4(acc[nt][s][0], acc[nt][s][1], acc[nt][s][2], acc[nt][s][3]);
          if (lane < 4) {
#pragma unroll
            for (int i = 0; i < 2; ++i) p.part_ml[slot * C::heads + nt * 8 + 2 * lane + i] = make_float2(m[nt][i], l[nt][i]);
          }
        }
        // units of this (request, head tile) after the ones taken here, over runs of `quota`
        if (lane == 0 && starts) {
          const uint32_t followers = (uint32_t)((at.span.units - at.take() + quota - 1) / quota);
          p.joins[blockIdx.x] = Join{b, at.hh, followers, 0};
          p.parts[(uint64_t)b * hh_n + at.hh] = make_uint2(blockIdx.x, followers);
        }
      }
      if (lane == 0 && starts && ends) p.parts[(uint64_t)b * hh_n + at.hh] = make_uint2(blockIdx.x, 0);
    }
    at = following;
  }
}

// Joins the partials of a (request, head tile): slot 1 of the CTA that took its first units, then slot 0
// of the CTAs after it. Blocks stand for CTAs or, where there are fewer, for (request, head tile)s. A
// piece is 16 elements of 8 heads (one fragment); a block takes p.pieces of them, each by 8 / p.pieces
// warps that take every so many partials and add up in order.
template <int DP, int NT, bool k8>
__device__ __forceinline__ void join_part(const KernelParams &p, uint32_t block) {
  constexpr int kSteps = DP / 16;
  constexpr uint32_t tile_heads = 8 * NT;
  __shared__ float4 s_sum[8][32];
  __shared__ float s_l[8][8];
  __shared__ float s_top[8][8];
  const uint32_t groups = NT * kSteps / p.pieces, index = block / groups;
  const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const uint32_t piece = block % groups * p.pieces + warp % p.pieces, sub = warp / p.pieces, subs = 8 / p.pieces;
  Join j;
  uint32_t cta = index;
  if (p.join_parts) {
    const uint32_t hh_n = p.a.c.n_heads * p.head_tiles;
    const uint2 part = p.parts[index];
    cta = part.x;
    j = Join{index / hh_n, index % hh_n, part.y, 0};
  } else {
    j = p.joins[cta];
  }
  if (j.followers == 0) return;
  const uint32_t nt = piece / kSteps, s = piece % kSteps;
  const uint32_t g0 = (j.hh % p.head_tiles) * tile_heads + nt * 8, h = j.hh / p.head_tiles;
  const uint32_t n = j.followers + 1;
  auto slot = [&](uint32_t i) -> uint64_t { return i == 0 ? 2ull * cta + 1 : 2ull * (cta + i); };
  // the first partials of each warp are on their way while the maxima are found
  auto sums_of = [&](uint32_t i) {
    return reinterpret_cast<const float4 *>(p.part_o)[(slot(i) * NT * kSteps + nt * kSteps + s) * 32 + lane];
  };
  auto stats_of = [&](uint32_t i) { return *reinterpret_cast<const float4 *>(p.part_ml + slot(i) * tile_heads + nt * 8 + 2 * (lane & 3)); };
  constexpr int kEarly = 4;
  float4 y[kEarly], ml[kEarly];
#pragma unroll
  for (int e = 0; e < kEarly; ++e)
    if (sub + subs * e < n) {
      y[e] = sums_of(sub + subs * e);
      ml[e] = stats_of(sub + subs * e);
    }
  // maximum of each of the eight heads: lane % 8 is the head
  float M = -INFINITY;
#pragma unroll 2
  for (uint32_t i = sub * 4 + lane / 8; i < n; i += 4 * subs) M = fmaxf(M, p.part_ml[slot(i) * tile_heads + nt * 8 + lane % 8].x);
  M = fmaxf(M, __shfl_xor_sync(~0u, M, 8));
  M = fmaxf(M, __shfl_xor_sync(~0u, M, 16));
  if (subs > 1) {
    if (lane < 8) s_top[warp][lane] = M;
    __syncthreads();
    for (uint32_t w = warp % p.pieces; w < 8; w += p.pieces) M = fmaxf(M, s_top[w][lane % 8]);
  }
  const float top[2] = {__shfl_sync(~0u, M, 2 * (lane & 3)), __shfl_sync(~0u, M, 2 * (lane & 3) + 1)};
  float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
  float L[2] = {0.f, 0.f};
  auto add = [&](const float4 &o, const float4 &st) {
    const float f0 = rebase(st.x, st.y, top[0]), f1 = rebase(st.z, st.w, top[1]);
    x.x += f0 * o.x;
    x.y += f1 * o.y;
    x.z += f0 * o.z;
    x.w += f1 * o.w;
    L[0] += f0 * st.y;
    L[1] += f1 * st.w;
  };
#pragma unroll
  for (int e = 0; e < kEarly; ++e)
    if (sub + subs * e < n) add(y[e], ml[e]);
#pragma unroll 4
  for (uint32_t i = sub + subs * kEarly; i < n; i += subs) add(sums_of(i), stats_of(i));
  if (subs > 1) {
    s_sum[warp][lane] = x;
    if (lane < 4) {
      s_l[warp][2 * lane] = L[0];
      s_l[warp][2 * lane + 1] = L[1];
    }
    __syncthreads();
    if (sub) return;
    for (uint32_t w = warp + p.pieces; w < 8; w += p.pieces) {
      const float4 z = s_sum[w][lane];
      x.x += z.x;
      x.y += z.y;
      x.z += z.z;
      x.w += z.w;
      L[0] += s_l[w][2 * (lane & 3)];
      L[1] += s_l[w][2 * (lane & 3) + 1];
    }
  }
  const uint32_t r = lane >> 2;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const uint32_t g = g0 + 2 * (lane & 3) + i;
    if (g >= p.group) continue;
    const uint64_t head = h * p.group + g;
    const float f = L[i] == 0.f ? 0.f : p.a.c.v_scale / L[i];
    uint8_t *o = p.a.out + (int64_t)j.b * p.a.o_req + (int64_t)head * p.a.o_head;
    const uint32_t d0 = 16 * s + (k8 ? 2 * r : r), d1 = 16 * s + (k8 ? 2 * r + 1 : r + 8);
    if (d0 < p.a.c.head_dim) store_elem(o, d0, (i ? x.y : x.x) * f, p.a.dtype);
    if (d1 < p.a.c.head_dim) store_elem(o, d1, (i ? x.w : x.z) * f, p.a.dtype);
    if (s == 0 && r == 0) store_lse(p, (uint64_t)j.b * p.a.q_heads + head, top[i], L[i]);
  }
}

// weights_out[b, h, t] = weights[b, h, t] + sum over the heads of the group of 2^(score - lse), for
// p.weight_chunk tokens. The log-sum-exp of a head that was split is found from its parts here, a warp per
// head, so that this needs no wait for the join.
constexpr uint32_t kWeightTokens = 1024;  // tokens a block looks at at once
template <int NT>
__device__ __forceinline__ void add_weights(const KernelParams &p, uint32_t block) {
  extern __shared__ float s_lse[];
  constexpr uint32_t tile_heads = 8 * NT;
  const uint32_t chunks = (p.cap + p.weight_chunk - 1) / p.weight_chunk, chunk = block % chunks, row = block / chunks;
  const uint32_t h = row % p.a.c.n_heads, b = row / p.a.c.n_heads, lane = threadIdx.x & 31;
  const Span span = span_of(p, b);
  const uint32_t begin = chunk * p.weight_chunk, end = min(min(span.len, p.a.w_len), begin + p.weight_chunk);
  if (begin >= end) return;
  const float *w = p.a.weights + (int64_t)b * p.a.w_req + (int64_t)h * p.a.w_head;
  float *w_out = p.a.weights_out + (int64_t)b * p.a.wo_req + (int64_t)h * p.a.wo_head;
  const float *rows = p.logits + ((uint64_t)b * p.a.c.n_heads + h) * p.cap * p.group;
  constexpr uint32_t per = kWeightTokens / 256;
  const bool fours = p.group % 4 == 0;
  // weights and the scores of four heads of this thread's tokens t0, t0 + 256, ...
  auto load_sums = [&](uint32_t t0, float (&x)[per]) {
#pragma unroll
    for (uint32_t i = 0; i < per; ++i) x[i] = t0 + i * 256 < end ? w[t0 + i * 256] : 0.f;
  };
  auto load_scores = [&](uint32_t t0, uint32_t g, float4 (&y)[per]) {
#pragma unroll
    for (uint32_t i = 0; i < per; ++i) {
      const uint32_t t = t0 + i * 256;
      const bool in = t >= span.low && t < end;
      const float *at = rows + (uint64_t)t * p.group + g;
      y[i] = make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
      if (in && fours) {
        y[i] = *reinterpret_cast<const float4 *>(at);
      } else if (in) {
        y[i].x = at[0];
        if (g + 1 < p.group) y[i].y = at[1];
        if (g + 2 < p.group) y[i].z = at[2];
        if (g + 3 < p.group) y[i].w = at[3];
      }
    }
  };
  float x[per];
  float4 y[per];
  load_sums(begin + threadIdx.x, x);  // on their way while the log-sum-exps are found
  load_scores(begin + threadIdx.x, 0, y);
  for (uint32_t g = threadIdx.x >> 5; g < p.group; g += 8) {
    const uint32_t hh = h * p.head_tiles + g / tile_heads;
    const uint2 part = p.parts[(uint64_t)b * (p.a.c.n_heads * p.head_tiles) + hh];
    float lse2;
    if (part.y == 0) {
      lse2 = p.lse2[(uint64_t)b * p.a.q_heads + h * p.group + g];
    } else {
      auto stats = [&](uint32_t i) { return p.part_ml[(i == 0 ? 2ull * part.x + 1 : 2ull * (part.x + i)) * tile_heads + g % tile_heads]; };
      float M = -INFINITY, L = 0.f;
      for (uint32_t i = lane; i <= part.y; i += 32) M = fmaxf(M, stats(i).x);
      for (int o = 16; o; o >>= 1) M = fmaxf(M, __shfl_xor_sync(~0u, M, o));
      for (uint32_t i = lane; i <= part.y; i += 32) {
        const float2 ml = stats(i);
        L += rebase(ml.x, ml.y, M) * ml.y;
      }
      for (int o = 16; o; o >>= 1) L += __shfl_xor_sync(~0u, L, o);
      lse2 = log2_sum(M, L);
    }
    // a head without a token or a score adds nothing: exp2(-infinity - 0)
    if (lane == 0) s_lse[g] = lse2 == -INFINITY ? 0.f : lse2;
  }
  for (uint32_t g = p.group + threadIdx.x; g < (p.group + 3) / 4 * 4; g += 256) s_lse[g] = 0.f;
  __syncthreads();
  for (uint32_t t0 = begin + threadIdx.x; t0 < end; t0 += kWeightTokens) {
    if (t0 >= begin + kWeightTokens) {
      load_sums(t0, x);
      load_scores(t0, 0, y);
    }
    for (uint32_t g = 0; g < p.group; g += 4) {
      float4 next[per];
      if (g + 4 < p.group) load_scores(t0, g + 4, next);
#pragma unroll
      for (uint32_t i = 0; i < per; ++i) {
        x[i] += (exp2_fast(y[i].x - s_lse[g]) + exp2_fast(y[i].y - s_lse[g + 1])) + (exp2_fast(y[i].z - s_lse[g + 2]) + exp2_fast(y[i].w - s_lse[g + 3]));
        y[i] = next[i];
      }
    }
#pragma unroll
    for (uint32_t i = 0; i < per; ++i)
      if (t0 + i * 256 < end) w_out[t0 + i * 256] = x[i];
  }
}

// What is left to do after all units: the first join_blocks blocks join, the others add up weights.
template <int DP, int NT, bool k8>
__global__ void __launch_bounds__(256, 3) finish_kernel(const __grid_constant__ KernelParams p) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if (blockIdx.x < p.join_blocks) join_part<DP, NT, k8>(p, blockIdx.x);
  else add_weights<NT>(p, blockIdx.x - p.join_blocks);
}

// `after`: starts while the kernel before it drains, and waits for that kernel's results itself.
template <class K>
cudaError_t launch(K kernel, dim3 grid, dim3 block, size_t smem, cudaStream_t stream, const KernelParams &kp, bool after) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = after;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, kp);  // this launch's own error, no earlier call's
  if (e == cudaSuccess) count_launch();
  return e;
}

template <int kKind, int DP, int NT>
cudaError_t run(const KernelParams &kp, const Plan &plan, int sms, cudaStream_t stream) {
  using C = Cfg<kKind, DP, NT>;
  auto kernel = decode_attention_kernel<kKind, DP, NT>;
  static std::atomic<uint64_t> ready{0};  // one bit per device
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  const uint64_t bit = 1ull << (dev & 63);
  if (dev >= 64 || !(ready.load(std::memory_order_acquire) & bit)) {
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, C::smem);
    if (e != cudaSuccess) return e;
    if (dev < 64) ready.fetch_or(bit, std::memory_order_release);
  }
  e = launch(kernel, dim3(plan.grid), dim3(kThreads), C::smem, stream, kp, false);
  if (e != cudaSuccess) return e;
  KernelParams fp = kp;
  // Fragments a joining block takes: up to eight, a warp each, which suits requests of a few parts; where
  // a (request, head) may have many, fewer, with more warps for each.
  const uint64_t tiles = (uint64_t)kp.a.c.batch * kp.a.c.n_heads * kp.head_tiles;
  const uint32_t pieces = NT * (DP / 16), spread = (uint32_t)(plan.grid / tiles);
  fp.pieces = spread >= 16 ? 1 : (spread >= 8 ? 2 : (spread >= 4 ? 4 : 8));
  if (fp.pieces > pieces) fp.pieces = pieces;
  fp.join_parts = tiles < plan.grid;
  fp.join_blocks = plan.joins_needed ? (uint32_t)(fp.join_parts ? tiles : plan.grid) * (pieces / fp.pieces) : 0;
  uint64_t blocks = fp.join_blocks;
  if (kp.logits) {
    // a block finds its heads' log-sum-exps first: chunks long enough that the blocks are few waves
    const uint64_t heads = (uint64_t)kp.a.c.n_heads * kp.a.c.batch;
    uint64_t chunk = kWeightTokens;
    while (chunk < kp.cap && heads * ((kp.cap + chunk - 1) / chunk) > 4ull * sms) chunk *= 2;
    fp.weight_chunk = (uint32_t)chunk;
    blocks += heads * ((kp.cap + chunk - 1) / chunk);
  }
  if (blocks > 0x7FFFFFFFull) return cudaErrorInvalidValue;
  if (blocks)
    e = launch(finish_kernel<DP, NT, kKind == kKindE4m3>, dim3((unsigned)blocks), dim3(256), kp.logits ? 4ull * (kp.group + 3) : 0, stream, fp, true);
  return e;
}

template <int kKind, int DP>
cudaError_t run_group(const KernelParams &kp, const Plan &plan, int sms, cudaStream_t stream) {
  return plan.tile_heads == 8 ? run<kKind, DP, 1>(kp, plan, sms, stream) : run<kKind, DP, 2>(kp, plan, sms, stream);
}

template <int kKind>
cudaError_t run_dim(const KernelParams &kp, const Plan &plan, int sms, cudaStream_t stream) {
  switch (padded_dim(kp.a.c.head_dim)) {
    case 64: return run_group<kKind, 64>(kp, plan, sms, stream);
    case 128: return run_group<kKind, 128>(kp, plan, sms, stream);
    default: return run_group<kKind, 256>(kp, plan, sms, stream);
  }
}

}  // namespace

uint64_t decode_attention_workspace(const PagedCache &c, uint32_t q_heads, bool weights, int sms) {
  return plan_of(c, q_heads, weights, sms).bytes;
}

cudaError_t launch_decode_attention(const DecodeAttentionParams &a, int sms, cudaStream_t stream) {
  const Plan plan = plan_of(a.c, a.q_heads, a.weights_out != nullptr, sms);
  KernelParams kp{};
  kp.a = a;
  kp.joins = reinterpret_cast<Join *>(a.workspace + plan.joins);
  kp.part_o = reinterpret_cast<float *>(a.workspace + plan.part_o);
  kp.part_ml = reinterpret_cast<float2 *>(a.workspace + plan.part_ml);
  kp.parts = reinterpret_cast<uint2 *>(a.workspace + plan.parts);
  kp.cap = a.c.max_blocks * a.c.block_size;
  kp.head_tiles = plan.head_tiles;
  kp.unit_tiles = plan.unit_tiles;
  kp.page = Divisor(a.c.block_size);
  kp.least_units = plan.least_units;
  kp.narrow = plan.narrow;
  kp.group = a.q_heads / a.c.n_heads;
  if (a.weights_out) {
    kp.lse2 = reinterpret_cast<float *>(a.workspace + plan.lse2);
    kp.logits = reinterpret_cast<float *>(a.workspace + plan.logits);
  }
  if (a.c.dtype == kE4m3) return run_dim<kKindE4m3>(kp, plan, sms, stream);
  if (a.c.dtype == kFp16) return run_dim<kKindFp16>(kp, plan, sms, stream);
  return run_dim<kKindBf16>(kp, plan, sms, stream);
}

}  // namespace kvs
