// kvs_evict.cu -- eviction from a paged KV cache by accumulated attention weight.
//
// Per (request, KV head): of the tokens that have a page, the first `first` and the last `recent`
// positions stay, and of the others those of the largest weight (equal weights: the lowest
// position), `keep` in all. Their rows move, in order, to slots 0, 1, ... of the destination.
//
// Choosing: weights become 32-bit keys that sort as the weights do (0: no token, the largest: a
// token that stays), and the keep-th largest key is found by its digits of 12, 10 and 10 bits, most
// significant first: a histogram of the keys that share the digits found so far, then the bin in
// which the count from above reaches what is left. (Twelve bits first: sign, exponent and three bits
// more, so that weights of like size do not all count in a few bins.) A cluster of up to 8 CTAs
// shares a row; the keys stay in shared memory between the passes, so the weights are read from memory
// once, and the CTAs add up one another's histograms there. What bounds it is latency: three rounds of
// counting, exchange and scan. Chosen tokens are ranked by counting from the row's start, so the
// result does not depend on timing.
//
// Moving: to fresh pages, rows are copied by as many CTAs as there are rows for. In place, the rows
// of one (request, head) are moved by one CTA per 64-byte column of K or V, a batch of ranks at a
// time: a kept token's rank is at most its position, so writing ranks [i, i + n) only overwrites
// positions whose own rows have been read by then.
#include "kvs_paged_ops.cuh"

#include <cooperative_groups.h>

#include <atomic>

#include "kvs_kernels.cuh"

namespace kvs {

namespace {

namespace cg = cooperative_groups;

constexpr int kSelThreads = 512;
constexpr int kSelWarps = kSelThreads / 32;
constexpr uint32_t kStays = 0xFFFFFFFFu;
constexpr uint32_t kMaxCached = 49152;  // keys a CTA holds in shared memory (192 KiB beside its histograms)

// Keys sort as the weights: NaN above +inf, -0 equal to 0, never 0 and never kStays.
__device__ __forceinline__ uint32_t key_of(float w) {
  if (w != w) return 0xFFC00000u;
  if (w == 0.f) w = 0.f;  // one zero
  const uint32_t u = __float_as_uint(w);
  return u == 0x80000000u ? 0x80000000u : (u & 0x80000000u ? ~u : u | 0x80000000u);
}

__device__ __forceinline__ uint32_t length_of(const EvictParams &p, uint32_t b) {
  const int32_t n = __ldg(p.seq_lens + b);
  return n <= 0 ? 0 : min((uint32_t)n, p.c.max_blocks * p.c.block_size);
}

constexpr uint32_t kBins[3] = {4096, 1024, 1024};
constexpr uint32_t kAllBins = 4096 + 1024 + 1024;

struct Found {
  uint32_t bin, left, total;
};

// Adds up the cluster's histograms (`hist` in each CTA's shared memory), scans them from the largest
// bin down and finds the one in which the count reaches `want` of all that was counted (`all`: of
// min(total, want)). Same result in every CTA and thread; bin is BINS where everything is wanted.
template <uint32_t BINS>
__device__ Found find_bin(cg::cluster_group &cluster, uint32_t *hist, uint32_t want, uint32_t *s_warp, uint32_t *s_out) {
  constexpr uint32_t per = BINS / kSelThreads;
  static_assert(per == 2 || per == 8, "whole vectors per thread");
  const uint32_t tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const uint32_t low = BINS - (tid + 1) * per;  // this thread's lowest bin
  uint32_t bins[per];
#pragma unroll
  for (uint32_t i = 0; i < per; ++i) bins[i] = 0;
  for (uint32_t r = 0; r < cluster.num_blocks(); ++r) {
    const uint32_t *from = cluster.map_shared_rank(hist, r) + low;
    if (per == 8) {
#pragma unroll
      for (uint32_t i = 0; i < per; i += 4) {
        const uint4 x = *reinterpret_cast<const uint4 *>(from + i);
        bins[i] += x.x, bins[(i + 1) % per] += x.y, bins[(i + 2) % per] += x.z, bins[(i + 3) % per] += x.w;
      }
    } else {
      const uint2 x = *reinterpret_cast<const uint2 *>(from);
      bins[0] += x.x, bins[1] += x.y;
    }
  }
  uint32_t sum = 0;
#pragma unroll
  for (uint32_t i = 0; i < per; ++i) sum += bins[i];
  uint32_t incl = sum;
  for (int o = 1; o < 32; o <<= 1) {
    const uint32_t y = __shfl_up_sync(~0u, incl, o);
    if (lane >= o) incl += y;
  }
  if (lane == 31) s_warp[warp] = incl;
  __syncthreads();
  uint32_t before = 0, total = 0;
  for (uint32_t i = 0; i < kSelWarps; ++i) {
    if (i < warp) before += s_warp[i];
    total += s_warp[i];
  }
  incl += before;
  const uint32_t goal = min(want, total);
  if (tid == 0) {
    s_out[0] = BINS;
    s_out[1] = 0;
  }
  __syncthreads();
  uint32_t above = incl - sum;
  if (goal < total && above < goal && goal <= incl) {
#pragma unroll
    for (uint32_t i = per; i-- > 0;) {
      if (above < goal && goal <= above + bins[i]) {
        s_out[0] = low + i;
        s_out[1] = goal - above;
      }
      above += bins[i];
    }
  }
  __syncthreads();
  return Found{s_out[0], s_out[1], total};
}

__global__ void __launch_bounds__(kSelThreads) select_kernel(const __grid_constant__ EvictParams p, uint32_t cached_keys) {
  extern __shared__ __align__(16) uint32_t s_keys[];
  __shared__ __align__(16) uint32_t s_hist[kAllBins];
  __shared__ uint32_t s_count[2];           // above the threshold, equal to it
  __shared__ uint32_t s_warp[2][kSelWarps];
  __shared__ uint32_t s_out[2];
  cg::cluster_group cluster = cg::this_cluster();
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const uint32_t ctas = cluster.num_blocks(), rank = cluster.block_rank();
  const uint32_t row = blockIdx.x / ctas, b = row / p.c.n_heads, h = row % p.c.n_heads;
  const uint32_t tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const uint32_t len = length_of(p, b);
  const uint32_t piece = (len + ctas - 1) / ctas;
  const uint32_t t0 = min(len, rank * piece), n = min(len - t0, piece);
  const float *w = p.weights + (int64_t)b * p.w_req + (int64_t)h * p.w_head;
  const bool cached = piece <= cached_keys;

  auto compute = [&](uint32_t i) -> uint32_t {
    const uint32_t t = t0 + i;
    const float x = __ldg(w + t);
    if (page_of(p.c, b, p.page.quotient(t)) <= 0) return 0u;
    return t < p.first || t + p.recent >= len ? kStays : key_of(x);
  };
  auto key_at = [&](uint32_t i) -> uint32_t { return cached ? s_keys[i] : compute(i); };

  for (uint32_t i = tid; i < kAllBins; i += kSelThreads) s_hist[i] = 0;
  __syncthreads();
  constexpr uint32_t kAhead = 8;
  for (uint32_t base = tid; base < n; base += kSelThreads * kAhead) {
    uint32_t key[kAhead];
#pragma unroll
    for (uint32_t u = 0; u < kAhead; ++u) {
      const uint32_t i = base + u * kSelThreads;
      key[u] = i < n ? compute(i) : 0;
    }
#pragma unroll
    for (uint32_t u = 0; u < kAhead; ++u) {
      const uint32_t i = base + u * kSelThreads;
      if (cached && i < n) s_keys[i] = key[u];
      if (key[u]) atomicAdd(&s_hist[key[u] >> 20], 1u);
    }
  }
  cluster.sync();
  Found f = find_bin<4096>(cluster, s_hist, p.keep, s_warp[0], s_out);
  const uint32_t want = min(f.total, p.keep);
  uint32_t found = 1, left = 0xFFFFFFFFu;  // every token there is (keys are 1 or more)
  if (f.bin < 4096) {
    found = f.bin << 20;
    for (uint32_t i = tid; i < n; i += kSelThreads) {
      const uint32_t key = key_at(i);
      if (key && key >> 20 == f.bin) atomicAdd(&s_hist[4096 + (key >> 10 & 1023)], 1u);
    }
    cluster.sync();
    // where all of a bin is wanted, its lowest key is as good a threshold as any
    Found g = find_bin<1024>(cluster, s_hist + 4096, f.left, s_warp[0], s_out);
    left = g.left;
    if (g.bin < 1024) {
      found |= g.bin << 10;
      for (uint32_t i = tid; i < n; i += kSelThreads) {
        const uint32_t key = key_at(i);
        if (key && key >> 10 == found >> 10) atomicAdd(&s_hist[5120 + (key & 1023)], 1u);
      }
      cluster.sync();
      g = find_bin<1024>(cluster, s_hist + 5120, g.left, s_warp[0], s_out);
      left = g.left;
      if (g.bin < 1024) found |= g.bin;
      else left = 0xFFFFFFFFu;
    } else {
      left = 0xFFFFFFFFu;
    }
    found = max(found, 1u);
  }
  // chosen: keys above `found`, and the first `left` keys equal to it
  const uint32_t share = ((n + kSelWarps - 1) / kSelWarps + 31) / 32 * 32;
  const uint32_t i0 = min(n, warp * share), i1 = min(n, i0 + share);
  uint32_t above = 0, equal = 0;
  for (uint32_t i = i0; i < i1; i += 32) {
    const uint32_t key = i + lane < i1 ? key_at(i + lane) : 0;
    above += __popc(__ballot_sync(~0u, key > found));
    equal += __popc(__ballot_sync(~0u, key == found));
  }
  __syncthreads();  // s_warp is read no more
  if (lane == 0) {
    s_warp[0][warp] = above;
    s_warp[1][warp] = equal;
  }
  __syncthreads();
  if (tid < 2) {
    uint32_t sum = 0;
    for (int i = 0; i < kSelWarps; ++i) sum += s_warp[tid][i];
    s_count[tid] = sum;
  }
  cluster.sync();
  above = equal = 0;
  for (uint32_t r = 0; r < rank; ++r) {
    above += *cluster.map_shared_rank(&s_count[0], r);
    equal += *cluster.map_shared_rank(&s_count[1], r);
  }
  for (uint32_t i = 0; i < warp; ++i) {
    above += s_warp[0][i];
    equal += s_warp[1][i];
  }
  int32_t *kept = p.kept + (uint64_t)row * p.keep;
  for (uint32_t i = i0; i < i1; i += 32) {
    const uint32_t key = i + lane < i1 ? key_at(i + lane) : 0;
    const uint32_t ba = __ballot_sync(~0u, key > found), be = __ballot_sync(~0u, key == found);
    const uint32_t below = (1u << lane) - 1;
    const uint32_t a = above + __popc(ba & below), e = equal + __popc(be & below);
    if (key > found || (key == found && e < left)) kept[a + min(e, left)] = (int32_t)(t0 + i + lane);
    above += __popc(ba);
    equal += __popc(be);
  }
  for (uint32_t i = want + rank * kSelThreads + tid; i < p.keep; i += ctas * kSelThreads) kept[i] = -1;
  if (h == 0 && rank == 0 && tid == 0) p.new_lens[b] = (int32_t)want;
  cluster.sync();  // no CTA leaves while another reads its counts
}

constexpr int kMoveThreads = 256;
constexpr uint32_t kMoveRows = 64;

// Weights of the kept tokens to the front of weights_out, zeros behind them up to the old length;
// weights_out may be weights: a batch of ranks is read before any of it is written.
__device__ void move_weights(const EvictParams &p, uint32_t b, uint32_t h) {
  constexpr uint32_t per = 8;
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

__device__ __forceinline__ int32_t dst_page(const EvictParams &p, uint32_t b, uint32_t i) {
  const uint32_t vb = i / p.c.block_size;
  if (vb >= p.dst_blocks) return -1;
  const int32_t pg = __ldg(p.dst_table + (uint64_t)b * p.dst_blocks + vb);
  return pg > 0 && (uint32_t)pg < p.c.num_blocks ? pg : -1;
}

// To fresh pages: kMoveRows ranks of one (request, head) per CTA; the last x block moves weights.
__global__ void __launch_bounds__(kMoveThreads) move_kernel(const __grid_constant__ EvictParams p) {
  __shared__ int64_t s_src[2][kMoveRows], s_dst[2][kMoveRows];
  const uint32_t h = blockIdx.y, b = blockIdx.z, tid = threadIdx.x;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if (blockIdx.x == gridDim.x - 1) {
    move_weights(p, b, h);
    return;
  }
  const uint32_t n = (uint32_t)p.new_lens[b], base = blockIdx.x * kMoveRows;
  if (base >= n) return;
  const uint32_t rows = min(kMoveRows, n - base);
  if (tid < rows) {
    const uint32_t i = base + tid;
    const uint32_t t = (uint32_t)p.kept[((uint64_t)b * p.c.n_heads + h) * p.keep + i];
    const int32_t sp = page_of(p.c, b, t / p.c.block_size), dp = dst_page(p, b, i);
    const uint32_t sr = t % p.c.block_size, dr = i % p.c.block_size;
    s_src[0][tid] = (int64_t)sp * p.c.k_page + (int64_t)h * p.c.k_head + (int64_t)sr * p.c.k_row;
    s_src[1][tid] = (int64_t)sp * p.c.v_page + (int64_t)h * p.c.v_head + (int64_t)sr * p.c.v_row;
    s_dst[0][tid] = dp < 0 ? -1 : (int64_t)dp * p.c.k_page + (int64_t)h * p.c.k_head + (int64_t)dr * p.c.k_row;
    s_dst[1][tid] = dp < 0 ? -1 : (int64_t)dp * p.c.v_page + (int64_t)h * p.c.v_head + (int64_t)dr * p.c.v_row;
    if (dp < 0 && h == 0 && p.out_of_range) atomicAdd(p.out_of_range, 1u);
  }
  __syncthreads();
  const uint32_t words = p.row_bytes / 16, side = rows * words, total = 2 * side;
  constexpr int kUnroll = 8;
  for (uint32_t at = tid; at < total; at += kMoveThreads * kUnroll) {
    int4 x[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const uint32_t e = at + u * kMoveThreads;
      if (e < total) {
        const uint32_t s = e >= side, in = e - s * side, r = in / words, q = in % words;
        x[u] = *reinterpret_cast<const int4 *>((s ? p.c.v : p.c.k) + s_src[s][r] + 16 * q);
      }
    }
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const uint32_t e = at + u * kMoveThreads;
      if (e < total) {
        const uint32_t s = e >= side, in = e - s * side, r = in / words, q = in % words;
        if (s_dst[s][r] >= 0) *reinterpret_cast<int4 *>((s ? p.c.v : p.c.k) + s_dst[s][r] + 16 * q) = x[u];
      }
    }
  }
}

// In place: one CTA moves a 64-byte column of K (even blockIdx.x) or V of one (request, head),
// kColumnRows ranks at a time; the last x block moves the weights.
constexpr int kColumnUnroll = 8;
constexpr uint32_t kColumnRows = kMoveThreads / 4 * kColumnUnroll;
__global__ void __launch_bounds__(kMoveThreads) move_in_place_kernel(const __grid_constant__ EvictParams p) {
  const uint32_t h = blockIdx.y, b = blockIdx.z, tid = threadIdx.x;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if (blockIdx.x == gridDim.x - 1) {
    move_weights(p, b, h);
    return;
  }
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
  // CTAs per row: pieces of 1024 tokens while the GPU has room for more CTAs, of 8192 otherwise
  const uint64_t rows = (uint64_t)p.c.batch * p.c.n_heads;
  uint32_t ctas = 1;
  while (ctas < 8 && cap > 1024ull * ctas && (rows * ctas < 2ull * sms || cap > 8192ull * ctas)) ctas *= 2;
  const uint64_t piece = (cap + ctas - 1) / ctas;
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
  e = cudaLaunchKernelEx(&cfg, select_kernel, p, cached);
  if (e != cudaSuccess) return e;
  count_launch();
  // the move starts while the selection drains and waits for its results itself
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.blockDim = dim3(kMoveThreads);
  cfg.dynamicSmemBytes = 0;
  const uint64_t most = cap < p.keep ? cap : p.keep;
  if (p.dst_table) {
    cfg.gridDim = dim3((unsigned)((most + kMoveRows - 1) / kMoveRows + 1), p.c.n_heads, p.c.batch);
    e = cudaLaunchKernelEx(&cfg, move_kernel, p);
  } else {
    cfg.gridDim = dim3(2 * ((p.row_bytes + 63) / 64) + 1, p.c.n_heads, p.c.batch);
    e = cudaLaunchKernelEx(&cfg, move_in_place_kernel, p);
  }
  if (e == cudaSuccess) count_launch();
  return e;
}

}  // namespace kvs
