// kvs_evict.cu -- eviction from a paged KV cache by accumulated attention weight.
//
// Per (request, KV head): of the tokens that have a page, the first `first` and the last `recent`
// positions stay, and of the others those of the largest weight (equal weights: the lowest
// position), `keep` in all. Their rows move, in order, to slots 0, 1, ... of the destination.
//
// Choosing: weights become 32-bit keys that sort as the weights do (0: no token, the largest: a
// token that stays), and the keep-th largest key is found by its digits of 10, 8, 8 and 6 bits, most
// significant first: a histogram of the keys that share the digits found so far, then the bin in
// which the count from above reaches what is left. Once few keys share the digits, they are ranked
// against one another instead. A cluster of up to 8 CTAs shares a row; the keys stay in shared memory
// between the passes, so the weights are read from memory once, and the CTAs add up one another's
// histograms there (digits of 12, 10 and 10 bits took longer: the exchange grows with the bins). What
// bounds it is latency for a few rows (counting, exchange, scan: about 9 us for 4200 tokens) and
// instructions for many (28 us for 3.1 M weights). Chosen tokens are ranked by counting from the row's
// start, so the result does not depend on timing.
//
// Moving: a second kernel. To fresh pages, 64 ranks per CTA (12 prompts of up to 32768 tokens, 8 heads,
// trimmed to 4096: 57 us of 87 us in all, the measured copy rate for 370 MB; moving in the first kernel,
// by the CTA that chose the rows, took as long for many rows and longer for few). In place, one CTA per
// 64-byte column of K or V of one (request, head), a batch of ranks at a time: a kept token's rank is at
// most its position, so writing ranks [i, i + n) only overwrites positions whose own rows have been read
// by then.
#include "kvs_paged_ops.cuh"

#include <cooperative_groups.h>

#include <atomic>

#include "kvs_kernels.cuh"

namespace kvs {

namespace {

namespace cg = cooperative_groups;

constexpr int kSelThreads = 256;
constexpr int kSelWarps = kSelThreads / 32;
constexpr uint32_t kStays = 0xFFFFFFFFu;
constexpr uint32_t kMaxCached = 49152;  // keys a CTA holds in shared memory (192 KiB beside its histograms)

// Keys sort as the weights: NaN above +inf, -0 equal to 0, never 0 and never kStays.
__device__ __forceinline__ uint32_t key_of(float w) {
  if (w != w) return 0xFFC00000u;
  if (w == 0.f) w = 0.f;  // one zero
  const uint32_t u = __float_as_uint(w);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

__device__ __forceinline__ uint32_t length_of(const EvictParams &p, uint32_t b) {
  const int32_t n = __ldg(p.seq_lens + b);
  return n <= 0 ? 0 : min((uint32_t)n, p.c.max_blocks * p.c.block_size);
}

// digits of the keys, most significant first: 10, 8, 8 and 6 bits
constexpr uint32_t kAllBins = 1024 + 256 + 256 + 64;
constexpr uint32_t kNoBin = 0xFFFFFFFFu;
constexpr uint32_t kFew = kSelThreads;  // keys that are ranked against one another, one per thread

struct Found {
  uint32_t bin, left, count, total;  // count: keys in the bin
};

// Exclusive prefix of `mine` over the threads' warps (what the warps before this one hold) and the sum
// over all: `mine` is the warp's total, the same in every lane.
__device__ __forceinline__ uint2 over_warps(uint32_t mine, uint32_t *s_warp) {
  const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  if (lane == 0) s_warp[warp] = mine;
  __syncthreads();
  const uint32_t x = lane < kSelWarps ? s_warp[lane] : 0;
  return make_uint2(__reduce_add_sync(~0u, lane < warp ? x : 0), __reduce_add_sync(~0u, x));
}

// Adds up the cluster's histograms (`hist` in each CTA's shared memory), scans them from the largest
// bin down and finds the one in which the count reaches min(want, total). Same result in every CTA and
// thread; bin stays kNoBin where everything is wanted.
template <uint32_t BINS>
__device__ Found find_bin(cg::cluster_group &cluster, uint32_t *hist, uint32_t want, uint32_t *s_warp, uint32_t *s_out) {
  constexpr uint32_t per = BINS <= kSelThreads ? 1 : BINS / kSelThreads;
  static_assert(per == 1 || per == 2 || per == 4, "one access per thread");
  const uint32_t tid = threadIdx.x, lane = tid & 31;
  const uint32_t low = BINS - (tid + 1) * per;  // this thread's lowest bin
  const uint32_t ctas = cluster.num_blocks();
  uint32_t bins[per] = {};
  auto add = [&](const uint32_t *from) {
    if (per == 4) {
      const uint4 x = *reinterpret_cast<const uint4 *>(from + low);
      bins[0] += x.x, bins[1 % per] += x.y, bins[2 % per] += x.z, bins[3 % per] += x.w;
    } else if (per == 2) {
      const uint2 x = *reinterpret_cast<const uint2 *>(from + low);
      bins[0] += x.x, bins[1 % per] += x.y;
    } else {
      bins[0] += from[low];
    }
  };
  const bool mine = tid * per < BINS;
  if (mine) add(hist);
  const uint32_t me = cluster.block_rank();
#pragma unroll
  for (uint32_t r = 1; r < 8; ++r)
    if (r < ctas && mine) add(cluster.map_shared_rank(hist, (me + r) & (ctas - 1)));
  uint32_t sum = 0;
#pragma unroll
  for (uint32_t i = 0; i < per; ++i) sum += bins[i];
  uint32_t incl = sum;
  for (int o = 1; o < 32; o <<= 1) {
    const uint32_t y = __shfl_up_sync(~0u, incl, o);
    if (lane >= o) incl += y;
  }
  const uint2 w = over_warps(__shfl_sync(~0u, incl, 31), s_warp);
  incl += w.x;
  const uint32_t goal = min(want, w.y);
  uint32_t above = incl - sum;
  if (goal < w.y && above < goal && goal <= incl) {
#pragma unroll
    for (uint32_t i = per; i-- > 0;) {
      if (above < goal && goal <= above + bins[i]) {
        s_out[0] = low + i;
        s_out[1] = goal - above;
        s_out[2] = bins[i];
      }
      above += bins[i];
    }
  }
  __syncthreads();
  return Found{s_out[0], s_out[1], s_out[2], w.y};
}

// Chooses the tokens of one (request, KV head) per cluster and moves their weights.
__global__ void __launch_bounds__(kSelThreads) select_kernel(const __grid_constant__ EvictParams p, uint32_t cached_keys) {
  extern __shared__ __align__(16) uint32_t s_keys[];
  __shared__ __align__(16) uint32_t s_hist[kAllBins];
  __shared__ uint32_t s_count[2];           // above the threshold, equal to it
  __shared__ uint32_t s_warp[6][kSelWarps];
  __shared__ uint32_t s_out[5][3];
  __shared__ __align__(16) uint32_t s_all[kFew];
  __shared__ uint32_t s_few[kFew], s_few_count;
  cg::cluster_group cluster = cg::this_cluster();
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const uint32_t ctas = cluster.num_blocks(), rank = cluster.block_rank();
  auto sync_all = [&]() {  // a cluster's barrier costs several times a block's
    if (ctas > 1) cluster.sync();
    else __syncthreads();
  };
  const uint32_t row = blockIdx.x / ctas, b = row / p.c.n_heads, h = row % p.c.n_heads;
  const uint32_t tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const uint32_t len = length_of(p, b);
  const uint32_t piece = ((len + ctas - 1) / ctas + 3) / 4 * 4;  // tokens are taken four at a time
  const uint32_t t0 = min(len, rank * piece), n = min(len - t0, piece);
  const float *w = p.weights + (int64_t)b * p.w_req + (int64_t)h * p.w_head;
  const bool cached = piece <= cached_keys;

  const int32_t *table = p.c.page_table + (uint64_t)b * p.c.max_blocks;
  const uint32_t quads = (n + 3) / 4;
  // four weights, and their pages (one, where four tokens never lie in two): loads only
  auto load_quad = [&](uint32_t q, float4 &x, int4 &page) {
    const uint32_t t = t0 + 4 * q;
    if (p.vector_weights && 4 * q + 3 < n) {
      x = __ldg(reinterpret_cast<const float4 *>(w + t));
    } else {
      x.x = __ldg(w + t);
      x.y = __ldg(w + min(t + 1, len - 1));
      x.z = __ldg(w + min(t + 2, len - 1));
      x.w = __ldg(w + min(t + 3, len - 1));
    }
    page.x = __ldg(table + p.page.quotient(t));
    if (p.c.block_size % 4 == 0) {
      page.y = page.z = page.w = page.x;
    } else {
      page.y = __ldg(table + p.page.quotient(min(t + 1, len - 1)));
      page.z = __ldg(table + p.page.quotient(min(t + 2, len - 1)));
      page.w = __ldg(table + p.page.quotient(min(t + 3, len - 1)));
    }
  };
  auto keys_of = [&](uint32_t q, const float4 &x, const int4 &page) -> uint4 {
    auto key = [&](uint32_t i, float y, int32_t pg) -> uint32_t {
      const uint32_t t = t0 + i;
      const bool there = pg > 0 && (uint32_t)pg < p.c.num_blocks && i < n;
      return !there ? 0u : (t < p.first || t + p.recent >= len ? kStays : key_of(y));
    };
    return make_uint4(key(4 * q, x.x, page.x), key(4 * q + 1, x.y, page.y), key(4 * q + 2, x.z, page.z), key(4 * q + 3, x.w, page.w));
  };
  auto quad_at = [&](uint32_t q) -> uint4 {
    if (cached) return reinterpret_cast<const uint4 *>(s_keys)[q];
    float4 x;
    int4 page;
    load_quad(q, x, page);
    return keys_of(q, x, page);
  };

  for (uint32_t i = tid; i < kAllBins; i += kSelThreads) s_hist[i] = 0;
  if (tid < 5) s_out[tid][0] = kNoBin;
  if (tid == 0) s_few_count = 0;
  __syncthreads();
  constexpr uint32_t kAhead = 4;
  for (uint32_t base = tid; base < quads; base += kSelThreads * kAhead) {
    float4 x[kAhead];
    int4 page[kAhead];
#pragma unroll
    for (uint32_t u = 0; u < kAhead; ++u)  // all on their way before the first is looked at
      load_quad(min(base + u * kSelThreads, quads - 1), x[u], page[u]);
#pragma unroll
    for (uint32_t u = 0; u < kAhead; ++u) {
      const uint32_t q = base + u * kSelThreads;
      if (q >= quads) break;
      const uint4 k = keys_of(q, x[u], page[u]);
      if (cached) reinterpret_cast<uint4 *>(s_keys)[q] = k;
      if (k.x) atomicAdd(&s_hist[k.x >> 22], 1u);
      if (k.y) atomicAdd(&s_hist[k.y >> 22], 1u);
      if (k.z) atomicAdd(&s_hist[k.z >> 22], 1u);
      if (k.w) atomicAdd(&s_hist[k.w >> 22], 1u);
    }
  }
  sync_all();
  Found f = find_bin<1024>(cluster, s_hist, p.keep, s_warp[0], s_out[0]);
  const uint32_t want = min(f.total, p.keep);
  // keys above `found` are chosen, and the first `left` equal to it; where all keys of a bin are
  // wanted, its lowest key is as good a threshold as any (and with no bin at all the lowest key, 1)
  uint32_t found = 0, left = kNoBin;
  // (no key below 2^22 but 0 has a token, so keys that share the first digit are tokens' keys)
  auto next_digit = [&](uint32_t *hist, uint32_t shift, uint32_t bits) {
    auto count = [&](uint32_t key) {
      if ((key ^ found) >> (shift + bits) == 0) atomicAdd(&hist[key >> shift & ((1u << bits) - 1)], 1u);
    };
#pragma unroll 2
    for (uint32_t q = tid; q < quads; q += kSelThreads) {
      const uint4 k = quad_at(q);
      count(k.x), count(k.y), count(k.z), count(k.w);
    }
    sync_all();
  };
  // Few keys share the digits found: every CTA collects them all and ranks each against the others.
  auto rank_few = [&](uint32_t low, uint32_t wanted, uint32_t total) {
    auto collect = [&](uint32_t key) {
      if ((key ^ found) >> low == 0) s_few[atomicAdd(&s_few_count, 1u)] = key;
    };
#pragma unroll 2
    for (uint32_t q = tid; q < quads; q += kSelThreads) {
      const uint4 k = quad_at(q);
      collect(k.x), collect(k.y), collect(k.z), collect(k.w);
    }
    sync_all();
    const uint32_t theirs = lane < ctas ? *cluster.map_shared_rank(&s_few_count, lane) : 0;
    uint32_t before = 0, mine = 0;
    bool here = false;
    for (uint32_t r = 0; r < ctas; ++r) {
      const uint32_t count = __shfl_sync(~0u, theirs, r);
      if (tid >= before && tid < before + count) {
        mine = cluster.map_shared_rank(s_few, r)[tid - before];
        here = true;
      }
      before += count;
    }
    s_all[tid] = here ? mine : 0;  // zeros behind the last one count for nothing
    __syncthreads();
    if (here) {
      uint32_t larger = 0, same = 0;
#pragma unroll 4
      for (uint32_t i = 0; i < total; i += 4) {
        const uint4 x = *reinterpret_cast<const uint4 *>(s_all + i);
        larger += (x.x > mine) + (x.y > mine) + (x.z > mine) + (x.w > mine);
        same += (x.x == mine) + (x.y == mine) + (x.z == mine) + (x.w == mine);
      }
      if (larger < wanted && wanted <= larger + same) {
        s_out[4][0] = mine;
        s_out[4][1] = wanted - larger;
      }
    }
    __syncthreads();
    found = s_out[4][0];
    left = s_out[4][1];
  };
  if (f.bin != kNoBin) {
    found = f.bin << 22;
    if (f.count <= kFew) {
      rank_few(22, f.left, f.count);
    } else {
      next_digit(s_hist + 1024, 14, 8);
      f = find_bin<256>(cluster, s_hist + 1024, f.left, s_warp[1], s_out[1]);
      if (f.bin != kNoBin) {
        found |= f.bin << 14;
        if (f.count <= kFew) {
          rank_few(14, f.left, f.count);
        } else {
          next_digit(s_hist + 1280, 6, 8);
          f = find_bin<256>(cluster, s_hist + 1280, f.left, s_warp[2], s_out[2]);
          if (f.bin != kNoBin) {
            found |= f.bin << 6;
            next_digit(s_hist + 1536, 0, 6);
            f = find_bin<64>(cluster, s_hist + 1536, f.left, s_warp[3], s_out[3]);
            if (f.bin != kNoBin) {
              found |= f.bin;
              left = f.left;
            }
          }
        }
      }
    }
  }
  found = max(found, 1u);
  // chosen: keys above `found`, and the first `left` keys equal to it
  const uint32_t share = ((quads + kSelWarps - 1) / kSelWarps + 31) / 32 * 32;  // quads of a warp
  const uint32_t q0 = min(quads, warp * share), q1 = min(quads, q0 + share);
  auto above_in = [&](const uint4 &k) { return (uint32_t)(k.x > found) + (k.y > found) + (k.z > found) + (k.w > found); };
  auto equal_in = [&](const uint4 &k) { return (uint32_t)(k.x == found) + (k.y == found) + (k.z == found) + (k.w == found); };
  uint32_t above = 0, equal = 0;
  for (uint32_t q = q0 + lane; q < q1; q += 32) {
    const uint4 k = quad_at(q);
    above += above_in(k);
    equal += equal_in(k);
  }
  above = __reduce_add_sync(~0u, above);
  equal = __reduce_add_sync(~0u, equal);
  const uint2 of_above = over_warps(above, s_warp[4]), of_equal = over_warps(equal, s_warp[5]);
  uint32_t cta_above = 0, cta_equal = 0;  // in the CTAs before this one
  if (ctas > 1) {
    if (tid == 0) {
      s_count[0] = of_above.y;
      s_count[1] = of_equal.y;
    }
    sync_all();
    // lane r: the counts of CTA r, where it comes before this one
    const bool before = lane < rank;
    const uint32_t a = before ? *cluster.map_shared_rank(&s_count[0], lane) : 0, e = before ? *cluster.map_shared_rank(&s_count[1], lane) : 0;
    cta_above = __reduce_add_sync(~0u, a);
    cta_equal = __reduce_add_sync(~0u, e);
  }
  above = cta_above + of_above.x;
  equal = cta_equal + of_equal.x;
  int32_t *kept = p.kept + (uint64_t)row * p.keep;
  for (uint32_t base = q0; base < q1; base += 32) {  // the warp's quads in order
    const uint32_t q = base + lane;
    const uint4 k = q < q1 ? quad_at(q) : make_uint4(0, 0, 0, 0);
    const uint32_t own = above_in(k) | equal_in(k) << 16;
    uint32_t incl = own;
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t y = __shfl_up_sync(~0u, incl, o);
      if (lane >= o) incl += y;
    }
    uint32_t a = above + ((incl - own) & 0xFFFFu), e = equal + ((incl - own) >> 16);
    auto place = [&](uint32_t key, uint32_t i) {
      if (key > found) {
        kept[a + min(e, left)] = (int32_t)(t0 + i);
        ++a;
      } else if (key == found) {
        if (e < left) kept[a + e] = (int32_t)(t0 + i);
        ++e;
      }
    };
    place(k.x, 4 * q), place(k.y, 4 * q + 1), place(k.z, 4 * q + 2), place(k.w, 4 * q + 3);
    const uint32_t all = __shfl_sync(~0u, incl, 31);
    above += all & 0xFFFFu;
    equal += all >> 16;
  }
  for (uint32_t i = want + rank * kSelThreads + tid; i < p.keep; i += ctas * kSelThreads) kept[i] = -1;
  if (h == 0 && rank == 0 && tid == 0) p.new_lens[b] = (int32_t)want;
  // the ranks of this CTA's tokens
  const uint32_t begin = cta_above + min(cta_equal, left), end = cta_above + of_above.y + min(cta_equal + of_equal.y, left);
  float *w_out = p.weights_out + (int64_t)b * p.wo_req + (int64_t)h * p.wo_head;
  const bool in_turn = w_out == w;  // then every weight of the row is read before one is written
  __syncthreads();
  // the weights of ranks base, base + kSelThreads, ...: positions first, so that their loads overlap
  constexpr uint32_t kRanks = 4;
  auto weights_of = [&](uint32_t base, float (&x)[kRanks]) {
    int32_t t[kRanks];
#pragma unroll
    for (uint32_t u = 0; u < kRanks; ++u) t[u] = base + u * kSelThreads < end ? kept[base + u * kSelThreads] : 0;
#pragma unroll
    for (uint32_t u = 0; u < kRanks; ++u) x[u] = base + u * kSelThreads < end ? w[t[u]] : 0.f;
  };
  if (in_turn && cached)
    for (uint32_t i = begin + tid; i < end; i += kSelThreads * kRanks) {
      float x[kRanks];
      weights_of(i, x);
#pragma unroll
      for (uint32_t u = 0; u < kRanks; ++u)
        if (i + u * kSelThreads < end) s_keys[i + u * kSelThreads - begin] = __float_as_uint(x[u]);
    }
  sync_all();  // and no CTA leaves while another reads its counts
  if (!in_turn || cached) {
    for (uint32_t i = begin + tid; i < end; i += kSelThreads * kRanks) {
      float x[kRanks];
      if (!in_turn) weights_of(i, x);
#pragma unroll
      for (uint32_t u = 0; u < kRanks; ++u)
        if (i + u * kSelThreads < end) w_out[i + u * kSelThreads] = in_turn ? __uint_as_float(s_keys[i + u * kSelThreads - begin]) : x[u];
    }
    for (uint32_t i = want + rank * kSelThreads + tid; i < len; i += ctas * kSelThreads) w_out[i] = 0.f;
  }
}

constexpr int kMoveThreads = 256;

// Weights of the kept tokens to the front of weights_out (which is weights) and zeros behind them, for
// rows longer than the selection's CTAs hold: a batch of ranks is read before any of it is written.
__global__ void __launch_bounds__(kMoveThreads) move_weights_kernel(const __grid_constant__ EvictParams p) {
  constexpr uint32_t per = 8;
  const uint32_t h = blockIdx.x, b = blockIdx.y;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const float *w = p.weights + (int64_t)b * p.w_req + (int64_t)h * p.w_head;
  float *o = p.weights_out + (int64_t)b * p.wo_req + (int64_t)h * p.wo_head;
  const int32_t *kept = p.kept + ((uint64_t)b * p.c.n_heads + h) * p.keep;
  const uint32_t n = (uint32_t)p.new_lens[b], len = length_of(p, b);
  for (uint32_t base = 0; base < n; base += kMoveThreads * per) {
    float x[per];
#pragma unroll
    for (uint32_t u = 0; u < per; ++u) {
      const uint32_t i = base + u * kMoveThreads + threadIdx.x;
      if (i < n) x[u] = w[kept[i]];
    }
    __syncthreads();
#pragma unroll
    for (uint32_t u = 0; u < per; ++u) {
      const uint32_t i = base + u * kMoveThreads + threadIdx.x;
      if (i < n) o[i] = x[u];
    }
  }
  __syncthreads();
  for (uint32_t i = n + threadIdx.x; i < len; i += kMoveThreads) o[i] = 0.f;
}

// Page of slot i of request b's destination, or -1.
__device__ __forceinline__ int32_t dst_page(const EvictParams &p, uint32_t b, uint32_t vb) {
  if (vb >= p.dst_blocks) return -1;
  const int32_t pg = __ldg(p.dst_table + (uint64_t)b * p.dst_blocks + vb);
  return pg > 0 && (uint32_t)pg < p.c.num_blocks ? pg : -1;
}

// To fresh pages: kMoveRows ranks of one (request, head) per CTA.
constexpr uint32_t kMoveRows = 64;
__global__ void __launch_bounds__(kMoveThreads) move_kernel(const __grid_constant__ EvictParams p) {
  __shared__ struct {
    int64_t k_src[kMoveRows], v_src[kMoveRows], k_dst[kMoveRows], v_dst[kMoveRows];  // byte offsets; -1: nowhere
  } s;
  const uint32_t h = blockIdx.y, b = blockIdx.z, tid = threadIdx.x, words = p.row_bytes / 16;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const uint32_t n = (uint32_t)p.new_lens[b], base = blockIdx.x * kMoveRows;
  if (base >= n) return;
  const uint32_t rows = min(kMoveRows, n - base);
  if (tid < rows) {
    const uint32_t i = base + tid, t = (uint32_t)p.kept[((uint64_t)b * p.c.n_heads + h) * p.keep + i];
    const uint32_t sb = p.page.quotient(t), db = p.page.quotient(i), sr = p.page.rest(t, sb), dr = p.page.rest(i, db);
    const int32_t sp = page_of(p.c, b, sb), dp = dst_page(p, b, db);
    s.k_src[tid] = (int64_t)sp * p.c.k_page + (int64_t)h * p.c.k_head + (int64_t)sr * p.c.k_row;
    s.v_src[tid] = (int64_t)sp * p.c.v_page + (int64_t)h * p.c.v_head + (int64_t)sr * p.c.v_row;
    s.k_dst[tid] = dp < 0 ? -1 : (int64_t)dp * p.c.k_page + (int64_t)h * p.c.k_head + (int64_t)dr * p.c.k_row;
    s.v_dst[tid] = dp < 0 ? -1 : (int64_t)dp * p.c.v_page + (int64_t)h * p.c.v_head + (int64_t)dr * p.c.v_row;
    if (dp < 0 && h == 0 && p.out_of_range) atomicAdd(p.out_of_range, 1u);
  }
  __syncthreads();
  const uint32_t side = rows * words;
  constexpr int kAhead = 4;  // words in flight per thread, of K and of V
  for (uint32_t at = tid; at < side; at += kMoveThreads * kAhead) {
    int4 x[kAhead], y[kAhead];
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const uint32_t e = at + u * kMoveThreads, r = p.words.quotient(e), q = p.words.rest(e, r);
      if (e < side) {
        x[u] = *reinterpret_cast<const int4 *>(p.c.k + s.k_src[r] + 16 * q);
        y[u] = *reinterpret_cast<const int4 *>(p.c.v + s.v_src[r] + 16 * q);
      }
    }
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const uint32_t e = at + u * kMoveThreads, r = p.words.quotient(e), q = p.words.rest(e, r);
      if (e < side && s.k_dst[r] >= 0) {
        *reinterpret_cast<int4 *>(p.c.k + s.k_dst[r] + 16 * q) = x[u];
        *reinterpret_cast<int4 *>(p.c.v + s.v_dst[r] + 16 * q) = y[u];
      }
    }
  }
}

// In place: one CTA moves a 64-byte column of K (even blockIdx.x) or V of one (request, head),
// kColumnRows ranks at a time.
constexpr int kColumnUnroll = 8;
constexpr uint32_t kColumnRows = kMoveThreads / 4 * kColumnUnroll;
__global__ void __launch_bounds__(kMoveThreads) move_in_place_kernel(const __grid_constant__ EvictParams p) {
  const uint32_t h = blockIdx.y, b = blockIdx.z, tid = threadIdx.x;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const uint32_t is_v = blockIdx.x & 1, word = (blockIdx.x >> 1) * 4 + (tid & 3);
  const bool live = word < p.row_bytes / 16;
  uint8_t *cache = (is_v ? p.c.v : p.c.k) + (int64_t)h * (is_v ? p.c.v_head : p.c.k_head) + 16 * word;
  const int64_t page_b = is_v ? p.c.v_page : p.c.k_page, row_b = is_v ? p.c.v_row : p.c.k_row;
  const uint32_t n = (uint32_t)p.new_lens[b];
  const int32_t *kept = p.kept + ((uint64_t)b * p.c.n_heads + h) * p.keep;
  for (uint32_t base = 0; base < n; base += kColumnRows) {
    int4 x[kColumnUnroll];
    int64_t to[kColumnUnroll];
#pragma unroll
    for (int u = 0; u < kColumnUnroll; ++u) {
      const uint32_t i = base + u * (kMoveThreads / 4) + tid / 4;
      to[u] = -1;
      if (i < n && live) {
        const uint32_t t = (uint32_t)kept[i];
        const int32_t dp = page_of(p.c, b, i / p.c.block_size);
        if (dp <= 0) {
          if (h == 0 && blockIdx.x == 0 && (tid & 3) == 0 && p.out_of_range) atomicAdd(p.out_of_range, 1u);
        } else if (t != i) {
          const int32_t sp = page_of(p.c, b, t / p.c.block_size);
          x[u] = *reinterpret_cast<const int4 *>(cache + (int64_t)sp * page_b + (int64_t)(t % p.c.block_size) * row_b);
          to[u] = (int64_t)dp * page_b + (int64_t)(i % p.c.block_size) * row_b;
        }
      }
    }
    __syncthreads();
#pragma unroll
    for (int u = 0; u < kColumnUnroll; ++u)
      if (to[u] >= 0) *reinterpret_cast<int4 *>(cache + to[u]) = x[u];
  }
}

}  // namespace

cudaError_t launch_evict(const EvictParams &p, int sms, cudaStream_t stream) {
  if (p.c.batch == 0) return cudaSuccess;
  const uint64_t cap = (uint64_t)p.c.max_blocks * p.c.block_size;
  // CTAs per row: pieces of 1024 tokens while SMs are left, of 8192 otherwise. 8 rows of 16000 tokens:
  // 16 us against 38 us with a CTA per row; 64 rows of up to 8000: 36 us with four CTAs per row, 38 us
  // with eight, 45 us with one; 96 rows of up to 32768: 87 us with four, 95 us with eight, 118 us with two.
  const uint64_t rows = (uint64_t)p.c.batch * p.c.n_heads;
  uint32_t ctas = 1;
  while (ctas < 8 && cap > 1024ull * ctas && (rows * ctas < 1ull * sms || cap > 8192ull * ctas)) ctas *= 2;
  const uint64_t piece = ((cap + ctas - 1) / ctas + 3) / 4 * 4;
  const uint32_t cached = piece <= kMaxCached ? (uint32_t)piece : 0;
  const size_t smem = 4ull * cached;
  static std::atomic<uint64_t> ready{0};  // one bit per device
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  const uint64_t bit = 1ull << (dev & 63);
  if (dev >= 64 || !(ready.load(std::memory_order_acquire) & bit)) {
    e = cudaFuncSetAttribute(select_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 4 * kMaxCached);
    if (e != cudaSuccess) return e;
    if (dev < 64) ready.fetch_or(bit, std::memory_order_release);
  }
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(p.c.batch * p.c.n_heads * ctas);
  cfg.blockDim = dim3(kSelThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim = {ctas, 1, 1};
  cfg.attrs = at;
  cfg.numAttrs = 1;
  EvictParams q = p;
  q.vector_weights = (reinterpret_cast<uintptr_t>(p.weights) & 15) == 0 && p.w_req % 4 == 0 && p.w_head % 4 == 0;
  e = cudaLaunchKernelEx(&cfg, select_kernel, q, cached);
  if (e != cudaSuccess) return e;
  count_launch();
  // the move starts while the selection drains and waits for its results itself
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.blockDim = dim3(kMoveThreads);
  cfg.dynamicSmemBytes = 0;
  if (p.dst_table) {
    const uint64_t most = cap < p.keep ? cap : p.keep;
    cfg.gridDim = dim3((unsigned)((most + kMoveRows - 1) / kMoveRows), p.c.n_heads, p.c.batch);
    e = cudaLaunchKernelEx(&cfg, move_kernel, p);
    if (e != cudaSuccess) return e;
    count_launch();
  }
  if (!p.dst_table) {
    cfg.gridDim = dim3(2 * ((p.row_bytes + 63) / 64), p.c.n_heads, p.c.batch);
    e = cudaLaunchKernelEx(&cfg, move_in_place_kernel, p);
    if (e != cudaSuccess) return e;
    count_launch();
  }
  if (!cached && p.weights == p.weights_out) {
    cfg.gridDim = dim3(p.c.n_heads, p.c.batch);
    e = cudaLaunchKernelEx(&cfg, move_weights_kernel, p);
    if (e == cudaSuccess) count_launch();
  }
  return e;
}

}  // namespace kvs
