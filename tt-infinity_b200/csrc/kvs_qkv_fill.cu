// kvs_qkv_fill.cu -- norms of queries and keys per head, rotation by the token's position, and the
// write of K and V rows into a paged cache, in one pass.
//
// For a row x of head_dim elements (a head of one token):
//     y = x * w / sqrt(mean(x^2) + eps)        (queries and keys, where a weight is given)
//     (a, b) -> (a cos - b sin, a sin + b cos) on the pairs (i, i + rotary / 2), or (2i, 2i + 1),
// with the cosine and sine of frequency i at the token's position (on the frequency's axis), in
// 32 bits, rounded once on the way out. Values are only copied (and scaled for an e4m3 cache).
//
// What bounds it: each row is read once and written once; a token step of a few tokens is bound by
// the chain of lookups (request, start, page, cosines) ahead of the first row. A group of
// head_dim / 8 lanes owns a row, each lane the same four pairs of every row: a pair's two elements
// sit in one lane (two 8-byte accesses, or one of 16 bytes), so the rotation needs no exchange, the
// norm one reduction, and cosines, sines and weights stay in registers over a token's rows.
#include "kvs_paged_ops.cuh"

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include "kvs_kernels.cuh"

namespace kvs {

namespace {

constexpr int kWarps = 4;
constexpr int kUnroll = 4;  // rows in flight per lane

template <bool kBf>
__device__ __forceinline__ float2 widen2(uint32_t x) {
  if (kBf) return make_float2(__uint_as_float(x << 16), __uint_as_float(x & 0xFFFF0000u));
  return __half22float2(*reinterpret_cast<const __half2 *>(&x));
}
template <bool kBf>
__device__ __forceinline__ uint32_t narrow2(float lo, float hi) {
  if (kBf) {
    const __nv_bfloat162 y = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t *>(&y);
  }
  const __half2 y = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t *>(&y);
}
__device__ __forceinline__ uint32_t narrow4_e4m3(float a, float b, float c, float d) {
  const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
  const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(c, d), __NV_SATFINITE, __NV_E4M3);
  return lo | hi << 16;
}

// Number of entries of cu_seqlens (non-decreasing, -1 padding last and largest) that are <= t.
__device__ __forceinline__ uint32_t entries_up_to(const int32_t *cu, uint32_t n, uint32_t t, uint32_t lane) {
  uint32_t lo = 0;
  while (n) {
    const uint32_t step = (n + 31) / 32, i = (lane + 1) * step - 1;
    const uint32_t v = i < n ? (uint32_t)__ldg(cu + lo + i) : 0xFFFFFFFFu;
    const uint32_t hit = __popc(__ballot_sync(~0u, v <= t));
    lo += hit * step;
    n = min(step - 1, n - hit * step);
  }
  return lo;
}

// kLanes lanes own a row. Each warp takes one token and `rows_per` of its rows.
template <bool kBf, int kLanes>
__global__ void __launch_bounds__(32 * kWarps) qkv_fill_kernel(const __grid_constant__ QkvFillParams p, uint32_t parts, uint32_t rows_per) {
  constexpr uint32_t rows_at_once = 32 / kLanes;
  const uint32_t lane = threadIdx.x & 31;
  const uint64_t item = (uint64_t)blockIdx.x * kWarps + (threadIdx.x >> 5);
  const uint32_t t = (uint32_t)(item / parts), part = (uint32_t)(item % parts);
  if (t >= p.tokens) return;
  const PagedCache &c = p.c;
  const uint32_t rows = p.q_heads + 2 * c.n_heads;
  const uint32_t r0 = part * rows_per, r1 = min(rows, r0 + rows_per);
  const uint32_t l = lane % kLanes, sub = lane / kLanes;
  const uint32_t pair = 4 * l, half = p.rotary / 2, rest = (c.head_dim - p.rotary) / 2;
  const bool mine = 2 * pair < c.head_dim;
  const bool turns = pair < half;
  // the first elements of this lane's pairs, and how far the second ones are (halves layout)
  const uint32_t e0 = p.interleaved ? 2 * pair : (turns ? pair : pair + half);
  const uint32_t e1 = p.interleaved ? 2 * pair + 4 : (turns ? pair + half : pair + half + rest);

  // ---- the token: its request, its slot in the cache and its position
  const uint32_t upto = entries_up_to(p.cu_seqlens, c.batch + 1, t, lane);
  const bool inside = upto >= 1 && upto <= c.batch && (uint32_t)__ldg(p.cu_seqlens + upto) != 0xFFFFFFFFu;
  if (!inside) {  // behind the last sequence
    if (p.zero_rest && mine)
      for (uint32_t r = r0 + sub; r < min(r1, p.q_heads); r += rows_at_once) {
        uint8_t *o = p.q_out + (int64_t)t * p.o_tok + (int64_t)r * p.o_head;
        *reinterpret_cast<uint2 *>(o + 2 * e0) = make_uint2(0, 0);
        *reinterpret_cast<uint2 *>(o + 2 * e1) = make_uint2(0, 0);
      }
    return;
  }
  const uint32_t req = upto - 1;
  const uint32_t slot = t - (uint32_t)__ldg(p.cu_seqlens + req) + (uint32_t)__ldg(p.start + req);
  const int32_t page = page_of(c, req, slot / c.block_size);
  uint32_t pos = slot;
  if (p.positions) pos = lane < p.n_axes ? (uint32_t)__ldg(p.positions + (uint64_t)lane * p.tokens + t) : 0;
  const bool bad = __any_sync(~0u, pos >= p.n_positions);
  if ((bad || page < 0) && part == 0 && lane == 0 && p.out_of_range) atomicAdd(p.out_of_range, 1u);
  float cs[4], sn[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    uint32_t at = pos;
    if (p.positions) {
      const uint32_t axis = p.axes && turns ? (uint32_t)__ldg(p.axes + pair + i) : 0u;
      at = __shfl_sync(~0u, pos, min(axis, p.n_axes - 1));
    }
    cs[i] = 1.f;
    sn[i] = 0.f;
    if (turns && !bad) {
      cs[i] = __ldg(p.cos_sin + (uint64_t)at * p.rotary + pair + i);
      sn[i] = __ldg(p.cos_sin + (uint64_t)at * p.rotary + half + pair + i);
    }
  }
  const int64_t k_at = (int64_t)page * c.k_page + (int64_t)(slot % c.block_size) * c.k_row;
  const int64_t v_at = (int64_t)page * c.v_page + (int64_t)(slot % c.block_size) * c.v_row;
  const bool store = page > 0 && !bad;
  const float inv_dim = 1.f / (float)c.head_dim;
  const float k_inv = 1.f / c.k_scale, v_inv = 1.f / c.v_scale;

  // a row's eight elements of this lane as (first, second) elements of its pairs
  auto split = [&](uint2 lo, uint2 hi, float (&a)[4], float (&b)[4]) {
    const float2 x0 = widen2<kBf>(lo.x), x1 = widen2<kBf>(lo.y), x2 = widen2<kBf>(hi.x), x3 = widen2<kBf>(hi.y);
    if (p.interleaved) {
      a[0] = x0.x; b[0] = x0.y; a[1] = x1.x; b[1] = x1.y; a[2] = x2.x; b[2] = x2.y; a[3] = x3.x; b[3] = x3.y;
    } else {
      a[0] = x0.x; a[1] = x0.y; a[2] = x1.x; a[3] = x1.y; b[0] = x2.x; b[1] = x2.y; b[2] = x3.x; b[3] = x3.y;
    }
  };
  auto weight_of = [&](const void *w, float (&a)[4], float (&b)[4]) {
    if (!w || !mine) return;
    const uint8_t *x = static_cast<const uint8_t *>(w);
    split(__ldg(reinterpret_cast<const uint2 *>(x + 2 * e0)), __ldg(reinterpret_cast<const uint2 *>(x + 2 * e1)), a, b);
  };
  float qa[4] = {1.f, 1.f, 1.f, 1.f}, qb[4] = {1.f, 1.f, 1.f, 1.f}, ka[4] = {1.f, 1.f, 1.f, 1.f}, kb[4] = {1.f, 1.f, 1.f, 1.f};
  weight_of(p.q_weight, qa, qb);
  weight_of(p.k_weight, ka, kb);

  for (uint32_t base = r0; base < r1; base += kUnroll * rows_at_once) {
    uint2 lo[kUnroll], hi[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const uint32_t r = base + u * rows_at_once + sub;
      lo[u] = hi[u] = make_uint2(0, 0);
      if (r < r1 && mine) {
        const uint8_t *x = r < p.q_heads ? p.q + (int64_t)t * p.q_tok + (int64_t)r * p.q_head
                           : r < p.q_heads + c.n_heads ? p.k + (int64_t)t * p.k_tok + (int64_t)(r - p.q_heads) * p.k_head
                                                       : p.v + (int64_t)t * p.v_tok + (int64_t)(r - p.q_heads - c.n_heads) * p.v_head;
        lo[u] = *reinterpret_cast<const uint2 *>(x + 2 * e0);
        hi[u] = *reinterpret_cast<const uint2 *>(x + 2 * e1);
      }
    }
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const uint32_t r = base + u * rows_at_once + sub;
      const bool is_q = r < p.q_heads, is_k = !is_q && r < p.q_heads + c.n_heads;
      float a[4], b[4];
      split(lo[u], hi[u], a, b);
      float ss = 0.f;
#pragma unroll
      for (int i = 0; i < 4; ++i) ss += a[i] * a[i] + b[i] * b[i];
#pragma unroll
      for (int o = kLanes / 2; o; o >>= 1) ss += __shfl_xor_sync(~0u, ss, o);
      if (is_q || is_k) {
        const bool normed = is_q ? p.q_weight != nullptr : p.k_weight != nullptr;
        const float f = normed ? rsqrtf(ss * inv_dim + p.eps) : 1.f;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float x = a[i] * f * (is_q ? qa[i] : ka[i]), y = b[i] * f * (is_q ? qb[i] : kb[i]);
          a[i] = turns ? x * cs[i] - y * sn[i] : x;
          b[i] = turns ? x * sn[i] + y * cs[i] : y;
        }
      }
      if (r >= r1 || !mine) continue;
      uint8_t *o;
      if (is_q) {
        o = p.q_out + (int64_t)t * p.o_tok + (int64_t)r * p.o_head;
        if (bad) {
#pragma unroll
          for (int i = 0; i < 4; ++i) a[i] = b[i] = 0.f;
        }
      } else {
        if (!store) continue;
        o = is_k ? c.k + k_at + (int64_t)(r - p.q_heads) * c.k_head : c.v + v_at + (int64_t)(r - p.q_heads - c.n_heads) * c.v_head;
        if (c.dtype == kE4m3) {
          const float f = is_k ? k_inv : v_inv;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            a[i] *= f;
            b[i] *= f;
          }
          if (p.interleaved) {
            *reinterpret_cast<uint32_t *>(o + e0) = narrow4_e4m3(a[0], b[0], a[1], b[1]);
            *reinterpret_cast<uint32_t *>(o + e1) = narrow4_e4m3(a[2], b[2], a[3], b[3]);
          } else {
            *reinterpret_cast<uint32_t *>(o + e0) = narrow4_e4m3(a[0], a[1], a[2], a[3]);
            *reinterpret_cast<uint32_t *>(o + e1) = narrow4_e4m3(b[0], b[1], b[2], b[3]);
          }
          continue;
        }
      }
      if (p.interleaved) {
        *reinterpret_cast<uint2 *>(o + 2 * e0) = make_uint2(narrow2<kBf>(a[0], b[0]), narrow2<kBf>(a[1], b[1]));
        *reinterpret_cast<uint2 *>(o + 2 * e1) = make_uint2(narrow2<kBf>(a[2], b[2]), narrow2<kBf>(a[3], b[3]));
      } else {
        *reinterpret_cast<uint2 *>(o + 2 * e0) = make_uint2(narrow2<kBf>(a[0], a[1]), narrow2<kBf>(a[2], a[3]));
        *reinterpret_cast<uint2 *>(o + 2 * e1) = make_uint2(narrow2<kBf>(b[0], b[1]), narrow2<kBf>(b[2], b[3]));
      }
    }
  }
}

}  // namespace

cudaError_t launch_qkv_fill(const QkvFillParams &p, cudaStream_t stream) {
  if (p.tokens == 0) return cudaSuccess;
  const uint32_t rows = p.q_heads + 2 * p.c.n_heads;
  const int lanes = p.c.head_dim <= 64 ? 8 : (p.c.head_dim <= 128 ? 16 : 32);
  const uint32_t step = kUnroll * (32 / lanes);
  const uint32_t parts = (rows + step - 1) / step;
  const uint64_t items = (uint64_t)p.tokens * parts;
  const dim3 grid((unsigned)((items + kWarps - 1) / kWarps));
  const bool bf = p.dtype == kBf16;
#define KVS_FILL(kBf, kLanes) qkv_fill_kernel<kBf, kLanes><<<grid, 32 * kWarps, 0, stream>>>(p, parts, step)
  if (bf && lanes == 8) KVS_FILL(true, 8);
  else if (bf && lanes == 16) KVS_FILL(true, 16);
  else if (bf) KVS_FILL(true, 32);
  else if (lanes == 8) KVS_FILL(false, 8);
  else if (lanes == 16) KVS_FILL(false, 16);
  else KVS_FILL(false, 32);
#undef KVS_FILL
  count_launch();
  return cudaGetLastError();
}

}  // namespace kvs
