// kvs_decode_attention.cu -- attention of one new token per request over a paged KV cache.
//
// For request b, query head g of KV head h and the tokens t that have a page and lie in
// [max(0, L - window), L):
//     s_t = scale * q . k_t      o = sum_t exp(s_t - m) v_t / sum_t exp(s_t - m)      m = max_t s_t
// in one pass over the cache with the running maximum and sum of the softmax.
//
// What bounds it: every valid K and V row is read once; the arithmetic is 2 * group flop per cache
// byte (16-bit cache), far below what the tensor cores do in the time the bytes take, so the kernel
// is built to keep loads in flight:
//   * Each warp streams its own 16-token tiles of K and V through a private ring in shared memory
//     (16-byte cp.async, zero-filled where a token is masked, so that nothing a masked slot holds
//     -- infinities, NaN -- reaches the sums). No CTA barrier stands in the main loop.
//   * The products run with the tokens as the rows of the matrix instruction: S^T = K Q^T
//     (16 tokens x 8 heads) and O^T = V^T P^T (16 elements x 8 heads), so a group of up to 8 heads
//     fills the 8 columns and no instruction works on padding rows; groups up to 16 take two column
//     tiles and larger ones several passes over the cache.
//   * Work is split by tokens, not by request: the batch's tiles, in units of kUnitTiles, form one
//     sequence that is cut into equal runs, one per CTA, from lengths that only the device knows.
//     A (request, head) that spans several CTAs leaves partial sums that a second small kernel
//     joins, in the order of the sequence, so results do not depend on timing.
//
// Scores, maxima, sums and accumulators are 32-bit. The probabilities are rounded to the cache's
// 16-bit type for the second product (fp16 for an e4m3 cache): each is off by at most half a step,
// as the output is once more. An e4m3 cache is widened to fp16, which holds every e4m3 value; the
// queries are scaled by a power of two per head to fit fp16.
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
constexpr uint32_t kTile = 16;       // tokens per warp tile
constexpr uint32_t kUnitTiles = 16;  // tiles per unit of work: 256 tokens, 4 tiles per warp
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

enum Kind { kKindBf16, kKindFp16, kKindE4m3 };

template <int kKind, int DP, int NT>
struct Cfg {
  static constexpr int el = kKind == kKindE4m3 ? 1 : 2;
  static constexpr int pitch = DP * el;                // bytes of a row in shared memory
  static constexpr int chunks = pitch / 16;            // 16-byte pieces of a row
  static constexpr int stage = 2 * (int)kTile * pitch; // K and V of one tile
  static constexpr int fit = 98304 / (kWarps * stage);
  static constexpr int stages = fit < 3 ? 3 : (fit > 8 ? 8 : fit);
  static constexpr int ring = kWarps * stages * stage;
  static constexpr int ctas = ring > 100 * 1024 ? 1 : 2;  // resident CTAs per SM
  static constexpr int heads = 8 * NT;
  static constexpr int opitch = DP + 4;                // floats of a merged output row: conflict-free
  static_assert(kWarps * heads * opitch * 4 <= ring, "the warps' outputs are merged in the ring");
};

// One head's partial over one CTA's tokens; a CTA leaves at most two (its first run continues an
// earlier CTA's, its last run goes on in the next).
struct Join {
  uint32_t b, hh, followers, pad;
};

struct Plan {  // workspace layout
  uint64_t joins, part_o, part_ml, lse2, logits, bytes;
  uint32_t grid, head_tiles, tile_heads;
};

__host__ __device__ inline uint32_t head_tiles_of(uint32_t group) { return (group + 15) / 16; }

inline uint32_t padded_dim(uint32_t d) { return d <= 64 ? 64 : (d <= 128 ? 128 : 256); }

Plan plan_of(const PagedCache &c, uint32_t q_heads, bool weights, int sms) {
  Plan p{};
  const uint32_t group = q_heads / c.n_heads;
  p.head_tiles = head_tiles_of(group);
  p.tile_heads = group <= 8 ? 8 : 16;
  const uint32_t dp = padded_dim(c.head_dim);
  const uint32_t per_sm = dp == 256 && c.dtype != kE4m3 ? 1 : 2;
  const uint64_t cap = (uint64_t)c.max_blocks * c.block_size;
  const uint64_t units = (cap + kTile * kUnitTiles - 1) / (kTile * kUnitTiles);
  const uint64_t most = (uint64_t)c.batch * c.n_heads * p.head_tiles * units;
  const uint64_t full = (uint64_t)sms * per_sm;
  p.grid = (uint32_t)(most < full ? most : full);
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
  p.logits = take(weights ? 4ull * c.batch * q_heads * cap : 0);
  p.bytes = off;
  return p;
}

struct KernelParams {
  DecodeAttentionParams a;
  Join *joins;
  float *part_o;
  float2 *part_ml;
  float *lse2;    // base-2 log-sum-exp per row, kept for the weights
  float *logits;  // [batch][n_heads][cap][group] scores in base 2, or nullptr
  uint32_t cap, head_tiles, group;
};

__device__ __forceinline__ uint32_t smem_addr(const void *p) { return (uint32_t)__cvta_generic_to_shared(p); }

__device__ __forceinline__ void cp16(uint32_t dst, const void *src, bool there) {
  // src-size 0 reads nothing and writes zeros
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(there ? 16 : 0) : "memory");
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
__device__ __forceinline__ float load_elem(const uint8_t *row, uint32_t d, int32_t dtype) {
  return dtype == kBf16 ? __bfloat162float(reinterpret_cast<const __nv_bfloat16 *>(row)[d])
                        : __half2float(reinterpret_cast<const __half *>(row)[d]);
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
  s.units = max(1u, (s.tiles + kUnitTiles - 1) / kUnitTiles);  // an empty row still gets its zeros written
  return s;
}

template <int kKind, int DP, int NT>
__global__ void __launch_bounds__(kThreads, (Cfg<kKind, DP, NT>::ctas)) decode_attention_kernel(const __grid_constant__ KernelParams p) {
  using C = Cfg<kKind, DP, NT>;
  constexpr bool kBf = kKind == kKindBf16;
  constexpr bool k8 = kKind == kKindE4m3;
  constexpr int kSteps = DP / 16;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ uint64_t s_scan[kWarps + 2];
  __shared__ uint32_t s_where[2];
  __shared__ uint32_t s_mask[kWarps][C::stages];
  __shared__ float s_m[kWarps][C::heads], s_l[kWarps][C::heads], s_f[kWarps][C::heads], s_M[C::heads], s_L[C::heads];
  const uint32_t tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const PagedCache &c = p.a.c;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

  // ---- this CTA's run of units
  const uint32_t hh_n = c.n_heads * p.head_tiles;
  uint64_t total = 0, mine = 0;
  for (uint32_t base = 0; base < c.batch; base += kThreads) {
    mine = base + tid < c.batch ? span_of(p, base + tid).units : 0;
    uint64_t x = mine;
    for (int o = 16; o; o >>= 1) x += __shfl_xor_sync(~0u, x, o);
    total += x;
  }
  if (lane == 0) s_scan[warp] = total;
  __syncthreads();
  total = 0;
  for (int w = 0; w < kWarps; ++w) total += s_scan[w];
  total *= hh_n;
  const uint64_t quota = (total + gridDim.x - 1) / gridDim.x;
  const uint64_t begin = quota * blockIdx.x;
  if (begin >= total) {
    if (tid == 0) p.joins[blockIdx.x].followers = 0;
    return;
  }
  uint64_t left = min(quota, total - begin);
  // request that holds unit `begin`: the requests' units times hh_n, scanned kThreads at a time
  uint64_t run = 0;
  for (uint32_t base = 0; base < c.batch; base += kThreads) {
    const uint64_t val = c.batch <= kThreads ? mine : (base + tid < c.batch ? span_of(p, base + tid).units : 0);
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
      s_where[0] = base + tid;
      s_where[1] = (uint32_t)(in / val);       // head tile
      s_scan[kWarps] = in % val;               // unit within it
    }
    run += all;
    __syncthreads();
    if (run * hh_n > begin) break;
  }
  uint32_t b = s_where[0], hh = s_where[1];
  uint32_t unit = (uint32_t)s_scan[kWarps];
  Span span = span_of(p, b);
  if (tid == 0) p.joins[blockIdx.x].followers = 0;

  const uint32_t ring = smem_addr(smem) + warp * C::stages * C::stage;
  const uint32_t row_chunks = (c.head_dim * C::el + 15) / 16;
  const uint32_t used = k8 ? (c.head_dim + 31) / 32 * 32 : (c.head_dim + 15) / 16 * 16;  // elements the products run over
  const uint32_t used_chunks = used * C::el / 16;
  const bool one_page = c.block_size % kTile == 0;  // a tile lies in one page
  const float scale2 = p.a.scale * c.k_scale * kLog2e;
  // the pieces of a row this lane moves: piece lane % chunks of rows lane / chunks + i * rows_step
  constexpr uint32_t rows_step = C::chunks >= 32 ? 1 : 32 / C::chunks;
  const uint32_t my_chunk = lane % C::chunks, my_row = lane / C::chunks;
  auto swizzle = [](uint32_t row) -> uint32_t { return C::pitch >= 128 ? (row & 7) : ((row >> 1) & 3); };

  while (left) {
    const uint32_t take = (uint32_t)min((uint64_t)(span.units - unit), left);
    const bool starts = unit == 0, ends = unit + take == span.units;
    const uint32_t t_begin = span.first + unit * kUnitTiles;
    const uint32_t t_end = span.first + min(span.tiles, (unit + take) * kUnitTiles);
    const uint32_t h = hh / p.head_tiles, g0 = (hh % p.head_tiles) * C::heads;
    const uint32_t heads = min((uint32_t)C::heads, p.group - g0);
    const uint8_t *kh = c.k + (int64_t)h * c.k_head, *vh = c.v + (int64_t)h * c.v_head;
    const int32_t *table = c.page_table + (uint64_t)b * c.max_blocks;

    // page of this lane's token of a tile (of the tile, where it lies in one page); 0: masked
    auto page_at = [&](uint32_t tile) -> int32_t {
      if (tile >= t_end) return 0;
      const uint32_t t = tile * kTile + (one_page ? 0 : (lane & 15));
      const uint32_t vb = t / c.block_size;
      if (vb >= c.max_blocks) return 0;
      const int32_t pg = __ldg(table + vb);
      return pg > 0 && (uint32_t)pg < c.num_blocks ? pg : 0;
    };
    auto issue = [&](uint32_t tile, uint32_t stage, int32_t page) {
      if (tile < t_end) {
        const uint32_t t0 = tile * kTile;
        const uint32_t kdst = ring + stage * C::stage, vdst = kdst + kTile * C::pitch;
        uint32_t mask = 0xFFFFu;
        if (t0 + kTile > span.len) mask &= 0xFFFFu >> (t0 + kTile - span.len);
        if (t0 < span.low) mask &= 0xFFFFu << (span.low - t0);
        int64_t ko = 0, vo = 0;
        if (one_page) {
          if (page == 0) mask = 0;
          const uint32_t r = t0 % c.block_size;
          ko = (int64_t)page * c.k_page + (int64_t)r * c.k_row;
          vo = (int64_t)page * c.v_page + (int64_t)r * c.v_row;
        } else {
          mask &= __ballot_sync(~0u, page != 0) & 0xFFFFu;
          const uint32_t r = (t0 + (lane & 15)) % c.block_size;
          ko = (int64_t)page * c.k_page + (int64_t)r * c.k_row;
          vo = (int64_t)page * c.v_page + (int64_t)r * c.v_row;
        }
        if (lane == 0) s_mask[warp][stage] = mask;
#pragma unroll
        for (int x = 0; x < C::chunks / 2; ++x) {
          constexpr uint32_t per_row = C::chunks >= 32 ? C::chunks / 32 : 1;  // always 1 for rows up to 512 bytes
          static_assert(per_row == 1, "a row is at most 512 bytes");
          const uint32_t row = my_row + x * rows_step;
          const bool there = (mask >> row) & 1 && my_chunk < row_chunks;
          int64_t kro, vro;
          if (one_page) {
            kro = ko + (int64_t)row * c.k_row;
            vro = vo + (int64_t)row * c.v_row;
          } else {
            kro = __shfl_sync(~0u, ko, row);
            vro = __shfl_sync(~0u, vo, row);
          }
          if (!there) kro = vro = 0;  // the address of a row that is not read stays inside the cache
          if (my_chunk < used_chunks) {
            const uint32_t at = row * C::pitch + ((my_chunk ^ swizzle(row)) << 4);
            const uint32_t src = there ? my_chunk * 16 : 0;
            cp16(kdst + at, kh + kro + src, there);
            cp16(vdst + at, vh + vro + src, there);
          }
        }
      }
      cp_commit();
    };

    // ---- queries: column fragments of Q^T, heads as columns
    uint32_t bq[kSteps][NT][2];
    float head_scale[NT][2];  // per column of the score tile (heads 2j, 2j + 1)
    {
      const uint32_t j = lane & 3, n = lane >> 2;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        const uint32_t g = nt * 8 + n;
        const uint8_t *qr = p.a.q + (int64_t)b * p.a.q_req + (int64_t)(h * p.group + g0 + g) * p.a.q_head;
        const bool live = g < heads;
        if (!k8) {
          head_scale[nt][0] = head_scale[nt][1] = scale2;
#pragma unroll
          for (int s = 0; s < kSteps; ++s)
#pragma unroll
            for (int half = 0; half < 2; ++half) {
              const uint32_t d = 16 * s + 8 * half + 2 * j;
              bq[s][nt][half] = live && d < c.head_dim ? __ldg(reinterpret_cast<const uint32_t *>(qr) + d / 2) : 0u;
            }
        } else {
          // scaled by a power of two so that the head's largest element is in [1, 2): elements
          // below 2^-14 of it lose at most 2^-25 of it
          float big = 0.f;
          for (uint32_t d = j; d < c.head_dim; d += 4)
            if (live) big = fmaxf(big, fabsf(load_elem(qr, d, p.a.dtype)));
          big = fmaxf(big, __shfl_xor_sync(~0u, big, 1));
          big = fmaxf(big, __shfl_xor_sync(~0u, big, 2));
          // both the factor 2^-e and 2^e have to be normal numbers
          int e = big > 0.f && big < __int_as_float(0x7f800000) ? (int)(__float_as_uint(big) >> 23) - 127 : 0;
          e = max(-126, min(126, e));
          const float down = __uint_as_float((uint32_t)(127 - e) << 23);
          const float up = __uint_as_float((uint32_t)(127 + e) << 23) * scale2;
          // k index 2j + {0, 1} of a step is element 4j + {0, 1}, 2j + 8 + {0, 1} is 4j + 2 + {0, 1}: the
          // order in which four bytes of a key row come out of the matrix load
#pragma unroll
          for (int s = 0; s < kSteps; ++s)
#pragma unroll
            for (int half = 0; half < 2; ++half) {
              const uint32_t d = 16 * s + 4 * j + 2 * half;
              const bool in = live && d < c.head_dim;
              bq[s][nt][half] = in ? pack2<false>(load_elem(qr, d, p.a.dtype) * down, load_elem(qr, d + 1, p.a.dtype) * down) : 0u;
            }
          head_scale[nt][0] = __shfl_sync(~0u, up, 8 * j);
          head_scale[nt][1] = __shfl_sync(~0u, up, 8 * j + 4);
        }
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

    uint32_t tile = t_begin + warp;
#pragma unroll
    for (int s = 0; s < C::stages - 1; ++s) issue(tile + s * kWarps, s, page_at(tile + s * kWarps));
    int32_t next_page = page_at(tile + (C::stages - 1) * kWarps);
    uint32_t stage = 0;
    for (; tile < t_end; tile += kWarps) {
      cp_wait<C::stages - 2>();
      __syncwarp();
      {
        const uint32_t fresh = stage == 0 ? C::stages - 1 : stage - 1;
        const uint32_t ahead = tile + (C::stages - 1) * kWarps;
        issue(ahead, fresh, next_page);
        next_page = page_at(ahead + kWarps);
      }
      const uint32_t kt = ring + stage * C::stage, vt = kt + kTile * C::pitch;
      const uint32_t mask = s_mask[warp][stage];

      // ---- S^T = K Q^T
      float sc[NT][4];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) sc[nt][0] = sc[nt][1] = sc[nt][2] = sc[nt][3] = 0.f;
      {
        const uint32_t row = (lane & 7) + ((lane >> 3) & 1) * 8, ch = lane >> 4;
        const uint32_t at = kt + row * C::pitch, sw = swizzle(row);
        if (!k8) {
#pragma unroll
          for (int s = 0; s < kSteps; ++s) {
            if (16 * s >= used) break;
            uint32_t a[4];
            ldsm4(a, at + (((2 * s + ch) ^ sw) << 4));
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) mma<kBf>(sc[nt], a[0], a[1], a[2], a[3], bq[s][nt][0], bq[s][nt][1]);
          }
        } else {
#pragma unroll
          for (int s = 0; s < kSteps; s += 2) {
            if (16 * s >= used) break;
            uint32_t a[4];
            ldsm4(a, at + (((s + ch) ^ sw) << 4));
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              const uint32_t x0 = widen(a[2 * i]), x1 = widen(a[2 * i + 1]), x2 = widen(a[2 * i] >> 16), x3 = widen(a[2 * i + 1] >> 16);
#pragma unroll
              for (int nt = 0; nt < NT; ++nt) mma<false>(sc[nt], x0, x1, x2, x3, bq[s + i][nt][0], bq[s + i][nt][1]);
            }
          }
        }
      }

      // ---- running maximum and sum; tokens lane / 4 and lane / 4 + 8, heads 2j and 2j + 1
      const bool in0 = (mask >> (lane >> 2)) & 1, in1 = (mask >> ((lane >> 2) + 8)) & 1;
      uint32_t pb[NT][2];
      bool grew = false;
      float mn[NT][2];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          sc[nt][i] = in0 ? sc[nt][i] * head_scale[nt][i] : -INFINITY;
          sc[nt][2 + i] = in1 ? sc[nt][2 + i] * head_scale[nt][i] : -INFINITY;
          float x = fmaxf(sc[nt][i], sc[nt][2 + i]);
          x = fmaxf(x, __shfl_xor_sync(~0u, x, 4));
          x = fmaxf(x, __shfl_xor_sync(~0u, x, 8));
          x = fmaxf(x, __shfl_xor_sync(~0u, x, 16));
          mn[nt][i] = fmaxf(m[nt][i], x);
          grew |= mn[nt][i] > m[nt][i];
        }
      if (p.logits) {
        float *lg = p.logits + (((uint64_t)b * c.n_heads + h) * p.cap + (uint64_t)tile * kTile + (lane >> 2)) * p.group + g0;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const uint32_t g = nt * 8 + 2 * (lane & 3) + i;
            const uint32_t t = tile * kTile + (lane >> 2);
            if (g < heads && t < span.len) lg[g] = sc[nt][i];
            if (g < heads && t + 8 < span.len) lg[8ull * p.group + g] = sc[nt][2 + i];
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
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        float e[4];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const float base = m[nt][i] == -INFINITY ? 0.f : m[nt][i];
          e[i] = exp2_fast(sc[nt][i] - base);
          e[2 + i] = exp2_fast(sc[nt][2 + i] - base);
          l[nt][i] += e[i] + e[2 + i];
        }
        pb[nt][0] = transpose8(pack2<kBf>(e[0], e[1]));
        pb[nt][1] = transpose8(pack2<kBf>(e[2], e[3]));
      }

      // ---- O^T += V^T P^T
      {
        const uint32_t row = (lane & 7) + (lane >> 4) * 8, ch = (lane >> 3) & 1;
        const uint32_t at = vt + row * C::pitch, sw = swizzle(row);
        if (!k8) {
#pragma unroll
          for (int s = 0; s < kSteps; ++s) {
            if (16 * s >= used) break;
            uint32_t a[4];
            ldsm4t(a, at + (((2 * s + ch) ^ sw) << 4));
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) mma<kBf>(acc[nt][s], a[0], a[1], a[2], a[3], pb[nt][0], pb[nt][1]);
          }
        } else {
          // a transposed load of byte pairs gives (t0 d0, t0 d1, t1 d0, t1 d1): even elements become
          // rows 0-7 of the 16-element tile, odd ones rows 8-15
#pragma unroll
          for (int s = 0; s < kSteps; s += 2) {
            if (16 * s >= used) break;
            uint32_t a[4];
            ldsm4t(a, at + (((s + ch) ^ sw) << 4));
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              const uint32_t lo = __byte_perm(a[i], 0, 0x3120), hi = __byte_perm(a[2 + i], 0, 0x3120);
              const uint32_t x0 = widen(lo), x1 = widen(lo >> 16), x2 = widen(hi), x3 = widen(hi >> 16);
#pragma unroll
              for (int nt = 0; nt < NT; ++nt) mma<false>(acc[nt][s + i], x0, x1, x2, x3, pb[nt][0], pb[nt][1]);
            }
          }
        }
      }
      stage = stage + 1 == C::stages ? 0 : stage + 1;
    }
    cp_wait<0>();
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        l[nt][i] += __shfl_xor_sync(~0u, l[nt][i], 4);
        l[nt][i] += __shfl_xor_sync(~0u, l[nt][i], 8);
        l[nt][i] += __shfl_xor_sync(~0u, l[nt][i], 16);
      }

    // ---- join the warps
    __syncthreads();  // every warp has read its last tile: the ring becomes the outputs' buffer
    float *so = reinterpret_cast<float *>(smem);
    {
      const uint32_t j = lane & 3, r = lane >> 2;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const uint32_t g = nt * 8 + 2 * j + i;
          float *row = so + (warp * C::heads + g) * C::opitch;
#pragma unroll
          for (int s = 0; s < kSteps; ++s) {
            row[16 * s + (k8 ? 2 * r : r)] = acc[nt][s][i];
            row[16 * s + (k8 ? 2 * r + 1 : r + 8)] = acc[nt][s][2 + i];
          }
          if (r == 0) {
            s_m[warp][g] = m[nt][i];
            s_l[warp][g] = l[nt][i];
          }
        }
      }
    }
    __syncthreads();
    if (tid < C::heads) {
      float M = -INFINITY, L = 0.f;
      for (int w = 0; w < kWarps; ++w) M = fmaxf(M, s_m[w][tid]);
      for (int w = 0; w < kWarps; ++w) {
        const float f = s_m[w][tid] == -INFINITY ? (s_l[w][tid] == 0.f ? 0.f : 1.f) : exp2_fast(s_m[w][tid] - M);
        s_f[w][tid] = f;
        L += f * s_l[w][tid];
      }
      s_M[tid] = M;
      s_L[tid] = L;
    }
    __syncthreads();
    const bool whole = starts && ends;
    const uint32_t slot = 2 * blockIdx.x + (starts ? 1 : 0);
    for (uint32_t e = tid; e < heads * DP; e += kThreads) {
      const uint32_t g = e / DP, d = e % DP;
      if (d >= c.head_dim) continue;
      float x = 0.f;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) x += s_f[w][g] * so[(w * C::heads + g) * C::opitch + d];
      if (whole) {
        const float L = s_L[g];
        store_elem(p.a.out + (int64_t)b * p.a.o_req + (int64_t)(h * p.group + g0 + g) * p.a.o_head, d, L == 0.f ? 0.f : x / L * c.v_scale, p.a.dtype);
      } else {
        p.part_o[((uint64_t)slot * C::heads + g) * DP + d] = x;
      }
    }
    if (tid < heads) {
      if (whole) {
        const float lse2 = s_L[tid] == 0.f ? -INFINITY : s_M[tid] + __log2f(s_L[tid]);
        const uint64_t at = (uint64_t)b * p.a.q_heads + h * p.group + g0 + tid;
        if (p.a.lse) p.a.lse[at] = lse2 * kLn2;
        if (p.lse2) p.lse2[at] = lse2;
      } else {
        p.part_ml[(uint64_t)slot * C::heads + tid] = make_float2(s_M[tid], s_L[tid]);
      }
    }
    if (tid == 0 && starts && !ends) {
      // units of this (request, head tile) after the ones taken here, over runs of `quota`
      const uint64_t rest = span.units - take;
      p.joins[blockIdx.x] = Join{b, hh, (uint32_t)((rest + quota - 1) / quota), 0};
    }
    left -= take;
    unit = 0;
    if (++hh == hh_n && left) {
      hh = 0;
      ++b;
      span = span_of(p, b);
    }
    __syncthreads();  // the buffer is a ring again
  }
}

// Joins the partials of the (request, head tile) whose first units CTA blockIdx.x took: slot 1 of
// that CTA, then slot 0 of the CTAs after it. One block per head.
template <int DP>
__global__ void __launch_bounds__(256) join_kernel(const __grid_constant__ KernelParams p, uint32_t tile_heads) {
  extern __shared__ float s_fac[];
  __shared__ float s_red[8];
  __shared__ float s_out[256];
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const Join j = p.joins[blockIdx.x];
  if (j.followers == 0) return;
  const uint32_t g = blockIdx.y, g0 = (j.hh % p.head_tiles) * tile_heads, h = j.hh / p.head_tiles;
  if (g0 + g >= p.group) return;
  const uint32_t n = j.followers + 1, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  auto slot = [&](uint32_t i) -> uint64_t { return i == 0 ? 2ull * blockIdx.x + 1 : 2ull * (blockIdx.x + i); };
  float M = -INFINITY;
  for (uint32_t i = tid; i < n; i += 256) M = fmaxf(M, p.part_ml[slot(i) * tile_heads + g].x);
  for (int o = 16; o; o >>= 1) M = fmaxf(M, __shfl_xor_sync(~0u, M, o));
  if (lane == 0) s_red[warp] = M;
  __syncthreads();
  for (int w = 0; w < 8; ++w) M = fmaxf(M, s_red[w]);
  __syncthreads();
  float L = 0.f;
  for (uint32_t i = tid; i < n; i += 256) {
    const float2 ml = p.part_ml[slot(i) * tile_heads + g];
    const float f = ml.x == -INFINITY ? (ml.y == 0.f ? 0.f : 1.f) : exp2_fast(ml.x - M);
    s_fac[i] = f;
    L += f * ml.y;
  }
  for (int o = 16; o; o >>= 1) L += __shfl_xor_sync(~0u, L, o);
  if (lane == 0) s_red[warp] = L;
  __syncthreads();
  L = 0.f;
  for (int w = 0; w < 8; ++w) L += s_red[w];
  // 256 / DP groups of threads take every (256 / DP)-th partial of an element
  constexpr uint32_t parts = 256 / DP;
  const uint32_t d = tid % DP, part = tid / DP;
  float x = 0.f;
  if (d < p.a.c.head_dim) {
#pragma unroll 4
    for (uint32_t i = part; i < n; i += parts) x += s_fac[i] * p.part_o[(slot(i) * tile_heads + g) * DP + d];
  }
  s_out[tid] = x;
  __syncthreads();
  const uint64_t head = h * p.group + g0 + g;
  if (part == 0 && d < p.a.c.head_dim) {
#pragma unroll
    for (uint32_t i = 1; i < parts; ++i) x += s_out[i * DP + d];
    store_elem(p.a.out + (int64_t)j.b * p.a.o_req + (int64_t)head * p.a.o_head, d, L == 0.f ? 0.f : x / L * p.a.c.v_scale, p.a.dtype);
  }
  if (tid == 0) {
    const float lse2 = L == 0.f ? -INFINITY : M + __log2f(L);
    if (p.a.lse) p.a.lse[(uint64_t)j.b * p.a.q_heads + head] = lse2 * kLn2;
    if (p.lse2) p.lse2[(uint64_t)j.b * p.a.q_heads + head] = lse2;
  }
}

// weights_out[b, h, t] = weights[b, h, t] + sum over the heads of the group of 2^(score - lse).
__global__ void __launch_bounds__(256) add_weights_kernel(const __grid_constant__ KernelParams p) {
  extern __shared__ float s_lse[];
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const uint32_t h = blockIdx.y, b = blockIdx.z;
  const Span span = span_of(p, b);
  const uint32_t t = blockIdx.x * 256 + threadIdx.x;
  if (blockIdx.x * 256 >= min(span.len, p.a.w_len)) return;
  for (uint32_t g = threadIdx.x; g < p.group; g += 256) s_lse[g] = p.lse2[(uint64_t)b * p.a.q_heads + h * p.group + g];
  __syncthreads();
  if (t >= min(span.len, p.a.w_len)) return;
  float x = 0.f;
  if (t >= span.low) {
    const float *lg = p.logits + (((uint64_t)b * p.a.c.n_heads + h) * p.cap + t) * p.group;
    for (uint32_t g = 0; g < p.group; ++g) x += s_lse[g] == -INFINITY ? 0.f : exp2_fast(lg[g] - s_lse[g]);
  }
  p.a.weights_out[(int64_t)b * p.a.wo_req + (int64_t)h * p.a.wo_head + t] =
      p.a.weights[(int64_t)b * p.a.w_req + (int64_t)h * p.a.w_head + t] + x;
}

template <class K, class... Args>
cudaError_t launch_after(K kernel, dim3 grid, dim3 block, size_t smem, cudaStream_t stream, Args... args) {
  // starts while the kernel before it drains; it waits for that kernel's results itself
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  count_launch();
  return cudaLaunchKernelEx(&cfg, kernel, args...);
}

template <int kKind, int DP, int NT>
cudaError_t run(const KernelParams &kp, const Plan &plan, cudaStream_t stream) {
  using C = Cfg<kKind, DP, NT>;
  auto kernel = decode_attention_kernel<kKind, DP, NT>;
  static std::atomic<uint64_t> ready{0};  // one bit per device
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  const uint64_t bit = 1ull << (dev & 63);
  if (dev >= 64 || !(ready.load(std::memory_order_acquire) & bit)) {
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, C::ring);
    if (e != cudaSuccess) return e;
    if (dev < 64) ready.fetch_or(bit, std::memory_order_release);
  }
  kernel<<<plan.grid, kThreads, C::ring, stream>>>(kp);
  count_launch();
  e = cudaGetLastError();
  if (e != cudaSuccess) return e;
  // a request of one unit is never split
  if (kp.cap > kTile * kUnitTiles && plan.grid > 1) {
    const uint32_t heads = kp.group < (uint32_t)C::heads ? kp.group : (uint32_t)C::heads;
    e = launch_after(join_kernel<DP>, dim3(plan.grid, heads), dim3(256), 4ull * (plan.grid + 1), stream, kp, (uint32_t)C::heads);
    if (e != cudaSuccess) return e;
  }
  if (kp.logits) {
    const dim3 grid((kp.cap + 255) / 256, kp.a.c.n_heads, kp.a.c.batch);
    e = launch_after(add_weights_kernel, grid, dim3(256), 4ull * kp.group, stream, kp);
  }
  return e;
}

template <int kKind, int DP>
cudaError_t run_group(const KernelParams &kp, const Plan &plan, cudaStream_t stream) {
  return plan.tile_heads == 8 ? run<kKind, DP, 1>(kp, plan, stream) : run<kKind, DP, 2>(kp, plan, stream);
}

template <int kKind>
cudaError_t run_dim(const KernelParams &kp, const Plan &plan, cudaStream_t stream) {
  switch (padded_dim(kp.a.c.head_dim)) {
    case 64: return run_group<kKind, 64>(kp, plan, stream);
    case 128: return run_group<kKind, 128>(kp, plan, stream);
    default: return run_group<kKind, 256>(kp, plan, stream);
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
  kp.cap = a.c.max_blocks * a.c.block_size;
  kp.head_tiles = plan.head_tiles;
  kp.group = a.q_heads / a.c.n_heads;
  if (a.weights_out) {
    kp.lse2 = reinterpret_cast<float *>(a.workspace + plan.lse2);
    kp.logits = reinterpret_cast<float *>(a.workspace + plan.logits);
  }
  if (a.c.dtype == kE4m3) return run_dim<kKindE4m3>(kp, plan, stream);
  if (a.c.dtype == kFp16) return run_dim<kKindFp16>(kp, plan, stream);
  return run_dim<kKindBf16>(kp, plan, stream);
}

}  // namespace kvs
