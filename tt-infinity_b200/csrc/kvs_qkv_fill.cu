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
// the chain of lookups (request, start, page, cosines), which the first rows' loads do not wait for.
// A warp takes one token and some of its rows of one kind (q, k or v). A few lanes own a row, each the
// same pairs of every row: a pair's two elements sit in one lane, so the rotation needs no exchange and
// the norm one reduction over the row's lanes. Norm weight, cosine and sine of a pair are four
// coefficients that stay in registers over the warp's rows:
//     (a, b) -> (a A + b B, a C + b D) / sqrt(mean + eps)    A = wa cos, B = -wb sin, C = wa sin, D = wb cos
// and the next rows are loaded while these are computed. Blocks of one warp: warps of a token differ in
// length (queries, keys and values), and a block holds its registers until its last warp is done (72 us
// against 60 us with blocks of two). 8192 tokens of 64 + 2 x 8 heads of 128: 57 us, 93 % of the measured
// copy rate.
#include "kvs_paged_ops.cuh"

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include "kvs_kernels.cuh"

namespace kvs {

namespace {

constexpr int kUnroll = 2;  // rows in flight per lane

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

// PP pairs of 16-bit elements: half of a lane's elements of a row, one access.
template <int PP>
struct Half;
template <>
struct Half<4> {
  using type = uint2;
};
template <>
struct Half<8> {
  using type = uint4;
};

// PP pairs per lane, kLanes lanes per row (32 / kLanes rows at once).
template <bool kBf, bool kInter, int PP, int kLanes>
struct Rows {
  using H = typename Half<PP>::type;
  static constexpr uint32_t at_once = 32 / kLanes;
  static constexpr uint32_t step = kUnroll * at_once;

  // Where the halves of this lane's pairs lie in a row, and whether the pairs are rotated.
  struct Place {
    uint32_t e0, e1, pair, sub;
    bool mine, turns;
  };
  __device__ static __forceinline__ Place place(const QkvFillParams &p, uint32_t lane) {
    Place w;
    const uint32_t half = p.rotary / 2;
    w.pair = PP * (lane % kLanes);
    w.sub = lane / kLanes;
    w.mine = 2 * w.pair < p.c.head_dim;
    w.turns = w.pair < half;
    w.e0 = kInter ? 2 * w.pair : (w.turns ? w.pair : w.pair + half);
    w.e1 = kInter ? 2 * w.pair + PP : w.e0 + (w.turns ? half : (p.c.head_dim - p.rotary) / 2);
    return w;
  }
  // a row's elements of this lane as first and second elements of its pairs
  __device__ static __forceinline__ void split(const H &lo, const H &hi, float (&a)[PP], float (&b)[PP]) {
    const uint32_t *x = reinterpret_cast<const uint32_t *>(&lo), *y = reinterpret_cast<const uint32_t *>(&hi);
#pragma unroll
    for (int i = 0; i < PP / 2; ++i) {
      const float2 u = widen2<kBf>(x[i]), v = widen2<kBf>(y[i]);
      if (kInter) {
        a[i] = u.x, b[i] = u.y;
        a[PP / 2 + i] = v.x, b[PP / 2 + i] = v.y;
      } else {
        a[2 * i] = u.x, a[2 * i + 1] = u.y;
        b[2 * i] = v.x, b[2 * i + 1] = v.y;
      }
    }
  }
  // two halves in the order of memory
  __device__ static __forceinline__ void unsplit(const float (&a)[PP], const float (&b)[PP], float (&x)[2 * PP]) {
#pragma unroll
    for (int i = 0; i < PP; ++i) {
      x[i] = kInter ? (i & 1 ? b[i / 2] : a[i / 2]) : a[i];
      x[PP + i] = kInter ? (i & 1 ? b[PP / 2 + i / 2] : a[PP / 2 + i / 2]) : b[i];
    }
  }
  __device__ static __forceinline__ void store16(uint8_t *o, const Place &w, const float (&x)[2 * PP]) {
    H h[2];
    uint32_t *y = reinterpret_cast<uint32_t *>(h);
#pragma unroll
    for (int i = 0; i < PP; ++i) y[i] = narrow2<kBf>(x[2 * i], x[2 * i + 1]);
    *reinterpret_cast<H *>(o + 2 * w.e0) = h[0];
    *reinterpret_cast<H *>(o + 2 * w.e1) = h[1];
  }
  __device__ static __forceinline__ void store8(uint8_t *o, const Place &w, const float (&x)[2 * PP], float f) {
    uint32_t y[PP / 2];
#pragma unroll
    for (int i = 0; i < PP / 2; ++i) y[i] = narrow4_e4m3(x[4 * i] * f, x[4 * i + 1] * f, x[4 * i + 2] * f, x[4 * i + 3] * f);
    if (PP == 8) {
      *reinterpret_cast<uint2 *>(o + w.e0) = make_uint2(y[0], y[1]);
      *reinterpret_cast<uint2 *>(o + w.e1) = make_uint2(y[PP / 4], y[PP / 4 + 1]);
    } else {
      *reinterpret_cast<uint32_t *>(o + w.e0) = y[0];
      *reinterpret_cast<uint32_t *>(o + w.e1) = y[1];
    }
  }
  // rows [row, row + step) below `end`, `stride` bytes apart
  __device__ static __forceinline__ void load(const uint8_t *x, int64_t stride, uint32_t row, uint32_t end, const Place &w, H (&lo)[kUnroll], H (&hi)[kUnroll]) {
    const uint8_t *at = x + (int64_t)(row + w.sub) * stride;
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      if (row + u * at_once + w.sub < end && w.mine) {
        lo[u] = *reinterpret_cast<const H *>(at + 2 * w.e0);
        hi[u] = *reinterpret_cast<const H *>(at + 2 * w.e1);
      }
      at += at_once * stride;
    }
  }

  // Norm and rotation of the rows [row, end) (the first `step` of them already loaded): `coef` as above.
  template <bool k8>
  __device__ static __forceinline__ void turn(const QkvFillParams &p, const Place &w, const uint8_t *x, int64_t in, uint8_t *o, int64_t out, uint32_t row,
                                              uint32_t end, H (&lo)[kUnroll], H (&hi)[kUnroll], const float (&coef)[4][PP], bool normed, float scale) {
    const float inv_dim = 1.f / (float)p.c.head_dim;
    for (; row < end; row += step) {
      H next_lo[kUnroll], next_hi[kUnroll];
      load(x, in, row + step, end, w, next_lo, next_hi);
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) {
        float a[PP], b[PP], r[2 * PP];
        split(lo[u], hi[u], a, b);
        float f = 1.f;
        if (normed) {
          float ss = 0.f;
#pragma unroll
          for (int i = 0; i < PP; ++i) ss += a[i] * a[i] + b[i] * b[i];
          if (!w.mine) ss = 0.f;
#pragma unroll
          for (int k = kLanes / 2; k; k >>= 1) ss += __shfl_xor_sync(~0u, ss, k);
          f = rsqrtf(ss * inv_dim + p.eps);
        }
        float y[PP], z[PP];
#pragma unroll
        for (int i = 0; i < PP; ++i) {
          y[i] = a[i] * coef[0][i];
          z[i] = b[i] * coef[3][i];
          if (w.turns) {
            y[i] += b[i] * coef[1][i];
            z[i] += a[i] * coef[2][i];
          }
          y[i] *= f;
          z[i] *= f;
        }
        const uint32_t q = row + u * at_once + w.sub;
        if (q < end && w.mine) {
          unsplit(y, z, r);
          if (k8) store8(o + (int64_t)q * out, w, r, scale);
          else store16(o + (int64_t)q * out, w, r);
        }
      }
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) {
        lo[u] = next_lo[u];
        hi[u] = next_hi[u];
      }
    }
  }
};

// Jobs of a token: q_parts warps for its queries, then warps for its keys and values, each `per` rows
// (of both).
template <bool kBf, bool kInter, int PP, int kLanes>
__global__ void __launch_bounds__(32) qkv_fill_kernel(const __grid_constant__ QkvFillParams p, uint32_t q_parts, uint32_t per) {
  using R = Rows<kBf, kInter, PP, kLanes>;
  const uint32_t lane = threadIdx.x, t = blockIdx.x;
  const PagedCache &c = p.c;
  const bool is_q = blockIdx.y < q_parts;
  const uint32_t row0 = (is_q ? blockIdx.y : blockIdx.y - q_parts) * per, end = min(is_q ? p.q_heads : c.n_heads, row0 + per);
  const typename R::Place w = R::place(p, lane);
  const uint8_t *x = is_q ? p.q + (int64_t)t * p.q_tok : p.k + (int64_t)t * p.k_tok;
  const uint8_t *v = p.v + (int64_t)t * p.v_tok;
  const int64_t in = is_q ? p.q_head : p.k_head;
  typename R::H lo[kUnroll], hi[kUnroll], v_lo[kUnroll], v_hi[kUnroll];
  // the first rows are on their way while the token's place is looked up
  R::load(x, in, row0, end, w, lo, hi);
  if (!is_q) R::load(v, p.v_head, row0, end, w, v_lo, v_hi);
  // and so is what does not depend on that place
  uint32_t pos = p.positions && lane < p.n_axes ? (uint32_t)__ldg(p.positions + (uint64_t)lane * p.tokens + t) : 0;
  int4 axis[PP / 4] = {};
  if (p.axes && w.turns)
#pragma unroll
    for (int i = 0; i < PP / 4; ++i) axis[i] = __ldg(reinterpret_cast<const int4 *>(p.axes + w.pair) + i);
  const void *weight = is_q ? p.q_weight : p.k_weight;
  typename R::H weight_lo, weight_hi;
  if (weight && w.mine) {
    weight_lo = __ldg(reinterpret_cast<const typename R::H *>(static_cast<const uint8_t *>(weight) + 2 * w.e0));
    weight_hi = __ldg(reinterpret_cast<const typename R::H *>(static_cast<const uint8_t *>(weight) + 2 * w.e1));
  }

  // ---- the token: its request, its slot in the cache and its position
  const uint32_t upto = entries_up_to(p.cu_seqlens, c.batch + 1, t, lane);
  const bool inside = upto >= 1 && upto <= c.batch && (uint32_t)__ldg(p.cu_seqlens + upto) != 0xFFFFFFFFu;
  bool bad = false;
  uint32_t slot = 0, vb = 0;
  int32_t page = 0;
  if (inside) {
    const uint32_t req = upto - 1;
    slot = t - (uint32_t)__ldg(p.cu_seqlens + req) + (uint32_t)__ldg(p.start + req);
    vb = slot < 0x80000000u ? p.page.quotient(slot) : c.max_blocks;
    page = page_of(c, req, vb);
    if (!p.positions) pos = slot;
    bad = __any_sync(~0u, pos >= p.n_positions);
    if ((bad || page < 0) && blockIdx.y == 0 && lane == 0 && p.out_of_range) atomicAdd(p.out_of_range, 1u);
  }
  if (is_q && (!inside || bad)) {
    if ((bad || p.zero_rest) && w.mine)  // rows behind the last sequence stay as they are unless asked for
      for (uint32_t r = row0 + w.sub; r < end; r += R::at_once) {
        uint8_t *o = p.q_out + (int64_t)t * p.o_tok + (int64_t)r * p.o_head;
        *reinterpret_cast<typename R::H *>(o + 2 * w.e0) = typename R::H{};
        *reinterpret_cast<typename R::H *>(o + 2 * w.e1) = typename R::H{};
      }
    return;
  }
  if (!is_q && (!inside || bad || page <= 0)) return;
  const uint32_t in_page = slot - vb * c.block_size;

  if (!is_q) {
    uint8_t *o = c.v + (int64_t)page * c.v_page + (int64_t)in_page * c.v_row;
    const float f = 1.f / c.v_scale;
    for (uint32_t row = row0; row < end; row += R::step) {
      if (row != row0) R::load(v, p.v_head, row, end, w, v_lo, v_hi);
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) {
        const uint32_t r = row + u * R::at_once + w.sub;
        if (r >= end || !w.mine) continue;
        uint8_t *to = o + (int64_t)r * c.v_head;
        if (c.dtype == kE4m3) {
          float a[PP], b[PP], y[2 * PP];
          R::split(v_lo[u], v_hi[u], a, b);
          R::unsplit(a, b, y);
          R::store8(to, w, y, f);
        } else {
          *reinterpret_cast<typename R::H *>(to + 2 * w.e0) = v_lo[u];
          *reinterpret_cast<typename R::H *>(to + 2 * w.e1) = v_hi[u];
        }
      }
    }
  }

  // ---- coefficients of this lane's pairs
  float coef[4][PP];
  float wa[PP], wb[PP];
#pragma unroll
  for (int i = 0; i < PP; ++i) wa[i] = wb[i] = 1.f;
  if (weight && w.mine) R::split(weight_lo, weight_hi, wa, wb);
  const uint32_t half = p.rotary / 2;
#pragma unroll
  for (int i = 0; i < PP; i += 4) {
    float4 cs = make_float4(1.f, 1.f, 1.f, 1.f), sn = make_float4(0.f, 0.f, 0.f, 0.f);
    if (p.axes) {
      const uint32_t of[4] = {(uint32_t)axis[i / 4].x, (uint32_t)axis[i / 4].y, (uint32_t)axis[i / 4].z, (uint32_t)axis[i / 4].w};
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const uint32_t at = __shfl_sync(~0u, pos, min(of[k], p.n_axes - 1));
        if (w.turns) {
          (&cs.x)[k] = __ldg(p.cos_sin + (uint64_t)at * p.rotary + w.pair + i + k);
          (&sn.x)[k] = __ldg(p.cos_sin + (uint64_t)at * p.rotary + half + w.pair + i + k);
        }
      }
    } else {
      const uint32_t at = p.positions ? __shfl_sync(~0u, pos, 0) : pos;
      if (w.turns) {
        cs = __ldg(reinterpret_cast<const float4 *>(p.cos_sin + (uint64_t)at * p.rotary + w.pair + i));
        sn = __ldg(reinterpret_cast<const float4 *>(p.cos_sin + (uint64_t)at * p.rotary + half + w.pair + i));
      }
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      // the pairs of an interleaved lane come as (first half, second half) of its elements: in order
      coef[0][i + k] = wa[i + k] * (&cs.x)[k];
      coef[1][i + k] = -wb[i + k] * (&sn.x)[k];
      coef[2][i + k] = wa[i + k] * (&sn.x)[k];
      coef[3][i + k] = wb[i + k] * (&cs.x)[k];
    }
  }
  const bool normed = weight != nullptr;
  if (is_q)
    R::template turn<false>(p, w, x, in, p.q_out + (int64_t)t * p.o_tok, p.o_head, row0, end, lo, hi, coef, normed, 1.f);
  else {
    uint8_t *o = c.k + (int64_t)page * c.k_page + (int64_t)in_page * c.k_row;
    if (c.dtype == kE4m3) R::template turn<true>(p, w, x, in, o, c.k_head, row0, end, lo, hi, coef, normed, 1.f / c.k_scale);
    else R::template turn<false>(p, w, x, in, o, c.k_head, row0, end, lo, hi, coef, normed, 1.f);
  }
}

template <bool kBf, bool kInter, int PP, int kLanes>
cudaError_t run(const QkvFillParams &p, int sms, cudaStream_t stream) {
  using R = Rows<kBf, kInter, PP, kLanes>;
  // Rows per warp: many share one lookup and one set of coefficients, as long as 16 warps per SM are left.
  // 8192 tokens of 64 + 2 x 8 heads: 57 us with up to 64 rows per warp, 63 us with 16.
  const uint32_t steps = (p.q_heads + R::step - 1) / R::step;
  uint32_t per = 8;
  while (per > 1 && (uint64_t)p.tokens * ((steps + per - 1) / per) < 16ull * sms) per /= 2;
  const uint32_t q_parts = (steps + per - 1) / per, kv_parts = (p.c.n_heads + per * R::step - 1) / (per * R::step);
  const dim3 grid(p.tokens, q_parts + kv_parts);
  if (grid.y > 65535) return cudaErrorInvalidValue;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(32);
  cfg.stream = stream;
  // this launch's own error, no earlier call's
  const cudaError_t e = cudaLaunchKernelEx(&cfg, qkv_fill_kernel<kBf, kInter, PP, kLanes>, p, q_parts, per * R::step);
  if (e == cudaSuccess) count_launch();
  return e;
}

template <bool kBf, bool kInter>
cudaError_t run_dim(const QkvFillParams &p, int sms, cudaStream_t stream) {
  const uint32_t d = p.c.head_dim;
  // 16-byte halves where both the rotated part and the rest split into eights of pairs
  if (p.rotary % 16 == 0 && d % 16 == 0) {
    if (d <= 64) return run<kBf, kInter, 8, 4>(p, sms, stream);
    if (d <= 128) return run<kBf, kInter, 8, 8>(p, sms, stream);
    return run<kBf, kInter, 8, 16>(p, sms, stream);
  }
  if (d <= 64) return run<kBf, kInter, 4, 8>(p, sms, stream);
  if (d <= 128) return run<kBf, kInter, 4, 16>(p, sms, stream);
  return run<kBf, kInter, 4, 32>(p, sms, stream);
}

}  // namespace

cudaError_t launch_qkv_fill(const QkvFillParams &p, int sms, cudaStream_t stream) {
  if (p.tokens == 0) return cudaSuccess;
  if (p.interleaved) return p.dtype == kBf16 ? run_dim<true, true>(p, sms, stream) : run_dim<false, true>(p, sms, stream);
  return p.dtype == kBf16 ? run_dim<true, false>(p, sms, stream) : run_dim<false, false>(p, sms, stream);
}

}  // namespace kvs
