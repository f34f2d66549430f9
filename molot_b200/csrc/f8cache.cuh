// The 8-bit block-scaled paged cache (MOLOT_KV_F8B): writing rows into it,
// decode attention over it, and eviction from it by accumulated attention
// weight.
//
// Format.  K and V pools are [num_pages][nkv][page_size][d] FP8 E4M3 codes;
// each block of 16 slots of a head has one FP32 scale, a power of two, in
// [num_pages][nkv][page_size / 16]: value = code * scale.  With s = 2^e the
// rule is the smallest e in [-64, 120] whose range covers the block,
// amax <= 448 * 2^e, amax the largest finite magnitude.  Because s is a
// power of two, dividing by it is exact, every code is the correctly rounded
// E4M3 value of x / s, and moving a code to another scale changes it only
// where it becomes subnormal: a block whose scale grows re-encodes its older
// rows without a second rounding of normal values.  E4M3's own exponent
// keeps the relative step (2^-4) over 2^15 of range, so the power of two
// costs no accuracy against amax / 448.  Infinities saturate, NaN stays NaN.
#pragma once

#include <cuda_fp8.h>
#include <cuda_runtime.h>
#include <math_constants.h>

#include <cstdint>

#include "act.cuh"
#include "ptx.cuh"

namespace molot {

constexpr int kF8Blk = 16;  // slots per scale

// One sequence of a plan (device array): 32 bytes, loaded as two int4.
struct alignas(16) F8Seq {
  int n;         // slots
  int first;     // first visible slot
  int lo;        // first slot of the window (>= first)
  int sink_end;  // slots [first, sink_end) stay visible whatever the window
  int a0, na;    // blocks of the sink range before the window's: [a0, a0 + na)
  int b0;        // the window's first block
  int nblk;      // blocks to visit in all: na + the window's
};

// A pool's device pointers (one layer).
struct F8Pool {
  uint8_t* k;
  uint8_t* v;
  float* k_scale;
  float* v_scale;
  const int* bt;  // [B][max_pages]
  int max_pages, page_size, nkv, d;
};

__device__ __forceinline__ float f8_exp2i(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }

// Scale of a block whose largest finite magnitude is amax: 448 = 1.75 * 2^8,
// so e is amax's exponent minus 8, one more when its mantissa exceeds 1.75.
__device__ __forceinline__ float f8_block_scale(float amax) {
  const int e = (int)((__float_as_uint(amax) + 0x1fffffu) >> 23) - 127 - 8;
  return f8_exp2i(min(max(e, -64), 120));
}

__device__ __forceinline__ float f8_inv_pow2(float s) {  // 1 / s for s = 2^e, exact
  return __uint_as_float((254u << 23) - __float_as_uint(s));
}

__device__ __forceinline__ float f8_decode(uint8_t c) {
  return __half2float(__half(__nv_cvt_fp8_to_halfraw(c, __NV_E4M3)));
}

// Four values, already divided by their scale -> four codes.
__device__ __forceinline__ uint32_t f8_encode4(float x, float y, float z, float w) {
  const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(x, y), __NV_SATFINITE, __NV_E4M3);
  const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(z, w), __NV_SATFINITE, __NV_E4M3);
  return lo | (hi << 16);
}
__device__ __forceinline__ void f8_decode4(uint32_t c, float s, float* x) {
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const __half2 h(__nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(c >> (16 * i)), __NV_E4M3));
    const float2 f = __half22float2(h);
    x[2 * i] = f.x * s;
    x[2 * i + 1] = f.y * s;
  }
}

// ------------------------------------------------------------------ write
struct F8WriteArgs {
  F8Pool pool;
  const void* k;  // row r, head h: k + r * k_stride + h * d (elements)
  const void* v;
  long long k_stride, v_stride;
  const int* n0;      // [B] slots before the new rows
  const int* len;     // [B] slots with them
  const int* row;     // [B + 1] prefix of new rows
  const int* blk;     // [B + 1] prefix of touched blocks
  float* weight;      // counters of the new slots become 0, or NULL
  int B, nitems;
};

// A warp per touched block, head and pool: the new rows' magnitude, the
// block's scale, the codes.  Bound by bytes.  The older rows of a partly
// filled block are read only when its scale grows.
template <class T, int D>
__global__ void __launch_bounds__(128) f8_write_kernel(const __grid_constant__ F8WriteArgs a) {
  constexpr int EPL = Act<T>::EPL, NC = kF8Blk * D / EPL / 32;
  const int lane = threadIdx.x & 31;
  const int item = blockIdx.x * 4 + (threadIdx.x >> 5);
  if (item >= a.nitems) return;
  const int nkv = a.pool.nkv;
  const int kv = item & 1, h = (item >> 1) % nkv, x = (item >> 1) / nkv;
  const int b = warp_find(a.blk, a.B, x);
  const int n0 = a.n0[b], n = a.len[b];
  const int blk = n0 / kF8Blk + (x - a.blk[b]);
  const int t0 = blk * kF8Blk;  // first slot of the block
  const int ps = a.pool.page_size;
  const long long page = a.pool.bt[(long long)b * a.pool.max_pages + t0 / ps];
  const long long hp = page * nkv + h;
  uint8_t* codes = (kv ? a.pool.v : a.pool.k) + (hp * ps + t0 % ps) * D;
  float* scale = (kv ? a.pool.v_scale : a.pool.k_scale) + hp * (ps / kF8Blk) + (t0 % ps) / kF8Blk;
  const T* rows = static_cast<const T*>(kv ? a.v : a.k) + (long long)h * D;
  const long long stride = kv ? a.v_stride : a.k_stride;
  const long long r0 = (long long)a.row[b] - n0 + t0;  // row of the block's slot 0
  float val[NC][EPL];
  float amax = 0.f;
#pragma unroll
  for (int i = 0; i < NC; ++i) {
    const int e = (lane + 32 * i) * EPL, r = e / D, c = e % D;
    const int t = t0 + r;
#pragma unroll
    for (int j = 0; j < EPL; ++j) val[i][j] = 0.f;
    if (t >= n0 && t < n) Act<T>::load(rows + (r0 + r) * stride + c, val[i]);
  }
#pragma unroll
  for (int i = 0; i < NC; ++i)
#pragma unroll
    for (int j = 0; j < EPL; ++j) amax = fmaxf(amax, finite_abs(val[i][j]));
  float s = f8_block_scale(warp_max(amax));
  bool recode = false;  // older rows under a grown scale
  float s_old = s;
  if (t0 < n0) {
    s_old = *scale;
    recode = s > s_old;
    s = fmaxf(s, s_old);
  }
  const float inv = f8_inv_pow2(s);
#pragma unroll
  for (int i = 0; i < NC; ++i) {
    const int e = (lane + 32 * i) * EPL, r = e / D;
    const int t = t0 + r;
    const bool fresh = t >= n0 && t < n;
    if (!fresh && !(recode && t < n0)) continue;
#pragma unroll
    for (int j = 0; j < EPL; j += 4) {
      float* v = &val[i][j];
      if (!fresh) f8_decode4(*reinterpret_cast<const uint32_t*>(codes + e + j), s_old, v);
      *reinterpret_cast<uint32_t*>(codes + e + j) =
          f8_encode4(v[0] * inv, v[1] * inv, v[2] * inv, v[3] * inv);
    }
  }
  __syncwarp();
  if (lane == 0) *scale = s;
  if (kv == 0 && a.weight && lane < kF8Blk && t0 + lane >= n0 && t0 + lane < n)
    a.weight[hp * ps + t0 % ps + lane] = 0.f;
}

// ----------------------------------------------------------------- decode
struct F8DecodeArgs {
  F8Pool pool;
  const F8Seq* seqs;
  const int* prefix;  // [B + 1] block visits (a block once for every kv head)
  const void* q;      // sequence b, head h: q + b * q_stride + h * d
  void* o;            // [B][nq][d]
  float* lse;         // [B][nq] or NULL
  float* score;       // [prefix[B]][16][G] base-2 scores (accumulation), or NULL
  float* lse2;        // [B][nq] base-2 log-sum-exp (accumulation), or NULL
  const float* slopes;
  long long q_stride;
  int B, nq, G;
  float scale, cap;
};

// A CTA per query head and sequence, a warp per slot.
template <class T, int D>
__global__ void __launch_bounds__(128) f8_decode_kernel(const __grid_constant__ F8DecodeArgs a) {
  constexpr int E = D / 32;
  const int h = blockIdx.x, b = blockIdx.y, g = h / a.G;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const F8Seq sq = a.seqs[b];
  const int ps = a.pool.page_size, nkv = a.pool.nkv;
  const float slope = a.slopes ? a.slopes[h] : 0.f;
  float q[E], o[E], m = -CUDART_INF_F, l = 0.f;
#pragma unroll
  for (int i = 0; i < E; ++i) {
    q[i] = Act<T>::one(static_cast<const T*>(a.q) + b * a.q_stride + (long long)h * D + lane * E + i);
    o[i] = 0.f;
  }
  for (int i = 0; i < sq.nblk; ++i) {
    const int blk = i < sq.na ? sq.a0 + i : sq.b0 + i - sq.na;
    const int t0 = blk * kF8Blk;
    const long long hp = (long long)a.pool.bt[(long long)b * a.pool.max_pages + t0 / ps] * nkv + g;
    const long long row = (hp * ps + t0 % ps) * D + lane * E;
    const float ks = a.pool.k_scale[hp * (ps / kF8Blk) + (t0 % ps) / kF8Blk];
    const float vs = a.pool.v_scale[hp * (ps / kF8Blk) + (t0 % ps) / kF8Blk];
    for (int r = warp; r < kF8Blk; r += 4) {
      const int t = t0 + r;
      const bool see = t >= sq.first && t < sq.n && (t >= sq.lo || t < sq.sink_end);
      float s = 0.f;
      if (see) {
#pragma unroll
        for (int j = 0; j < E; ++j) s += q[j] * f8_decode(a.pool.k[row + (long long)r * D + j]);
#pragma unroll
        for (int x = 16; x; x >>= 1) s += __shfl_xor_sync(0xffffffffu, s, x);
      }
      s = see ? score_logit(s * ks * a.scale, a.cap, slope, (float)(sq.n - 1 - t)) : -CUDART_INF_F;
      if (a.score && lane == 0)
        a.score[(((long long)a.prefix[b] + (long long)g * sq.nblk + i) * kF8Blk + r) * a.G + h % a.G] = s;
      if (!see) continue;
      const float mn = fmaxf(m, s), al = ex2(m - mn), p = ex2(s - mn);
      m = mn;
      l = l * al + p;
#pragma unroll
      for (int j = 0; j < E; ++j)
        o[j] = o[j] * al + p * vs * f8_decode(a.pool.v[row + (long long)r * D + j]);
    }
  }
  __shared__ float sm[4], sl[4], so[4][D];
  if (lane == 0) sm[warp] = m, sl[warp] = l;
#pragma unroll
  for (int i = 0; i < E; ++i) so[warp][lane * E + i] = o[i];
  __syncthreads();
  const float mx = fmaxf(fmaxf(sm[0], sm[1]), fmaxf(sm[2], sm[3]));
  float w[4], lt = 0.f;
  for (int i = 0; i < 4; ++i) {
    w[i] = sm[i] == -CUDART_INF_F ? 0.f : ex2(sm[i] - mx);
    lt += w[i] * sl[i];
  }
  const float inv = sq.nblk > 0 && lt > 0.f ? 1.f / lt : 0.f;
  for (int i = threadIdx.x; i < D; i += 128)
    Act<T>::store(static_cast<T*>(a.o) + ((long long)b * a.nq + h) * D + i,
                  inv * (w[0] * so[0][i] + w[1] * so[1][i] + w[2] * so[2][i] + w[3] * so[3][i]));
  if (threadIdx.x == 0) {
    const float z = lt > 0.f ? mx + log2f(lt) : -CUDART_INF_F;
    if (a.lse) a.lse[(long long)b * a.nq + h] = z * kLn2;
    if (a.lse2) a.lse2[(long long)b * a.nq + h] = z;
  }
}

struct F8WeightArgs {
  F8Pool pool;
  const F8Seq* seqs;
  const int* prefix;
  const float* score;
  const float* lse2;
  const float* win;  // [num_pages][nkv][page_size]
  float* wout;       // may be win
  int nq, G;
};

// Counters: wout = win + the slot's weights summed over the kv head's group,
// from the scores that the decode left.  A thread per slot; heads in order,
// so the sum does not depend on the launch.
__global__ void __launch_bounds__(128) f8_weight_kernel(const __grid_constant__ F8WeightArgs a) {
  const int g = blockIdx.y, b = blockIdx.z;
  const F8Seq sq = a.seqs[b];
  const int t = blockIdx.x * 128 + threadIdx.x;
  if (t >= sq.n) return;
  const int ps = a.pool.page_size;
  const long long hp =
      (long long)a.pool.bt[(long long)b * a.pool.max_pages + t / ps] * a.pool.nkv + g;
  const int blk = t / kF8Blk;
  const bool inA = blk >= sq.a0 && blk < sq.a0 + sq.na;
  const int i = inA ? blk - sq.a0 : blk - sq.b0 + sq.na;
  float p = 0.f;
  if (inA || (blk >= sq.b0 && i < sq.nblk)) {
    const float* s = a.score +
                     (((long long)a.prefix[b] + (long long)g * sq.nblk + i) * kF8Blk + t % kF8Blk) * a.G;
    const float* z = a.lse2 + (long long)b * a.nq + (long long)g * a.G;
    for (int j = 0; j < a.G; ++j)
      if (s[j] != -CUDART_INF_F) p += ex2(s[j] - z[j]);
  }
  a.wout[hp * ps + t % ps] = a.win[hp * ps + t % ps] + p;
}

// ------------------------------------------------------------------ evict
struct F8EvictArgs {
  F8Pool src, dst;
  const float* win;
  float* wout;
  int* kept;  // [B][nkv][budget]
  const F8Seq* seqs;
  int B, budget, recent;
};

// Order-preserving unsigned key of a counter; NaN below everything.
__device__ __forceinline__ uint32_t f8_key(float w) {
  const uint32_t u = __float_as_uint(w == 0.f ? 0.f : w);  // -0 ties with 0
  if (w != w) return 0u;
  return (u >> 31) ? ~u : u | 0x80000000u;
}

constexpr int kF8SelThreads = 1024;

// The slots to keep of one sequence and kv head, ascending: a radix select
// of the (budget - recent)-th largest key over slots [0, n - recent), 8 bits
// a pass, then an ordered compaction: keys above the threshold, and the
// lowest slots among those equal to it.
__global__ void __launch_bounds__(kF8SelThreads) f8_select_kernel(const __grid_constant__ F8EvictArgs a) {
  const int g = blockIdx.x, b = blockIdx.y;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int n = a.seqs[b].n, nkv = a.src.nkv, ps = a.src.page_size;
  int* kept = a.kept + ((long long)b * nkv + g) * a.budget;
  if (n <= a.budget) {
    for (int i = tid; i < a.budget; i += kF8SelThreads) kept[i] = i < n ? i : -1;
    return;
  }
  const int old = n - a.recent, want = a.budget - a.recent;
  const int* bt = a.src.bt + (long long)b * a.src.max_pages;
  auto key = [&](int t) {
    return f8_key(a.win[((long long)bt[t / ps] * nkv + g) * ps + t % ps]);
  };
  __shared__ int hist[256];
  __shared__ int s_digit, s_left;
  uint32_t pre = 0, mask = 0;
  int left = want;  // still to take among the keys that match the prefix
  for (int shift = 24; shift >= 0 && want > 0; shift -= 8) {
    if (tid < 256) hist[tid] = 0;
    __syncthreads();
    for (int t = tid; t < old; t += kF8SelThreads) {
      const uint32_t k = key(t);
      if ((k & mask) == pre) atomicAdd(&hist[(k >> shift) & 255], 1);
    }
    __syncthreads();
    if (tid == 0) {
      int r = left, dgt = 255;
      while (dgt > 0 && hist[dgt] < r) r -= hist[dgt--];
      s_digit = dgt;
      s_left = r;
    }
    __syncthreads();
    pre |= (uint32_t)s_digit << shift;
    mask |= 255u << shift;
    left = s_left;
    __syncthreads();
  }
  // Warp w compacts the contiguous slots [w * per, (w + 1) * per).
  const int per = ((old + 31) / 32 + 31) / 32 * 32;
  const int t_lo = min(old, warp * per), t_hi = min(old, t_lo + per);
  __shared__ int s_gt[32], s_eq[32];
  int gt = 0, eq = 0;
  for (int t = t_lo + lane; t - lane < t_hi; t += 32) {
    const uint32_t k = t < t_hi && want > 0 ? key(t) : 0u;
    const bool in = t < t_hi && want > 0;
    gt += __popc(__ballot_sync(0xffffffffu, in && k > pre));
    eq += __popc(__ballot_sync(0xffffffffu, in && k == pre));
  }
  if (lane == 0) s_gt[warp] = gt, s_eq[warp] = eq;
  __syncthreads();
  int eq0 = 0, at = 0;  // equal keys and kept slots before this warp's
  for (int w = 0; w < warp; ++w) {
    at += s_gt[w] + min(s_eq[w], max(0, left - eq0));
    eq0 += s_eq[w];
  }
  for (int t = t_lo + lane; t - lane < t_hi; t += 32) {
    const bool in = t < t_hi && want > 0;
    const uint32_t k = in ? key(t) : 0u;
    const unsigned below = (1u << lane) - 1u;
    const unsigned me = __ballot_sync(0xffffffffu, in && k == pre);
    const bool take = in && (k > pre || (k == pre && eq0 + __popc(me & below) < left));
    const unsigned mt = __ballot_sync(0xffffffffu, take);
    if (take) kept[at + __popc(mt & below)] = t;
    at += __popc(mt);
    eq0 += __popc(me);
  }
  for (int i = tid; i < a.recent; i += kF8SelThreads) kept[want + i] = old + i;
}

// A warp per destination block, head and pool: 16 kept rows from anywhere in
// the sequence, their common scale, their codes.  Bound by bytes.
template <int D>
__global__ void __launch_bounds__(128) f8_move_kernel(const __grid_constant__ F8EvictArgs a) {
  constexpr int NC = kF8Blk * D / 16 / 32;  // 16-byte chunks per lane
  const int lane = threadIdx.x & 31;
  const int item = blockIdx.x * 4 + (threadIdx.x >> 5);
  const int nkv = a.src.nkv, b = blockIdx.y;
  const int kv = item & 1, h = (item >> 1) % nkv, blk = (item >> 1) / nkv;
  const int m = min(a.seqs[b].n, a.budget);
  const int j0 = blk * kF8Blk;
  if (j0 >= m) return;
  const int* kept = a.kept + ((long long)b * nkv + h) * a.budget + j0;
  const int ps = a.src.page_size, pd = a.dst.page_size;
  // lane r (< 16) holds where destination row r comes from
  long long src = 0;
  float sscale = 0.f;
  const int* bt = a.src.bt + (long long)b * a.src.max_pages;
  const long long dhp = (long long)a.dst.bt[(long long)b * a.dst.max_pages + j0 / pd] * nkv + h;
  if (lane < kF8Blk && j0 + lane < m) {
    const int t = kept[lane];
    const long long hp = (long long)bt[t / ps] * nkv + h;
    src = hp * ps + t % ps;
    sscale = (kv ? a.src.v_scale : a.src.k_scale)[hp * (ps / kF8Blk) + (t % ps) / kF8Blk];
    if (kv == 0 && a.win) a.wout[dhp * pd + j0 % pd + lane] = a.win[src];
  }
  const uint8_t* pool = kv ? a.src.v : a.src.k;
  uint4 c[NC];
  float sc[NC], amax = 0.f;
#pragma unroll
  for (int i = 0; i < NC; ++i) {
    const int e = (lane + 32 * i) * 16, r = e / D;
    const long long row = __shfl_sync(0xffffffffu, src, r);
    sc[i] = __shfl_sync(0xffffffffu, sscale, r);
    c[i] = make_uint4(0, 0, 0, 0);
    if (j0 + r < m) c[i] = *reinterpret_cast<const uint4*>(pool + row * D + e % D);
  }
#pragma unroll
  for (int i = 0; i < NC; ++i) {
    const uint32_t w[4] = {c[i].x, c[i].y, c[i].z, c[i].w};
    float x[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      f8_decode4(w[j], sc[i], x);
#pragma unroll
      for (int q = 0; q < 4; ++q) amax = fmaxf(amax, finite_abs(x[q]));
    }
  }
  const float s = f8_block_scale(warp_max(amax)), inv = f8_inv_pow2(s);
  uint8_t* out = (kv ? a.dst.v : a.dst.k) + (dhp * pd + j0 % pd) * D;
#pragma unroll
  for (int i = 0; i < NC; ++i) {
    const int e = (lane + 32 * i) * 16, r = e / D;
    if (j0 + r >= m) continue;
    uint32_t w[4] = {c[i].x, c[i].y, c[i].z, c[i].w};
    float x[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      f8_decode4(w[j], sc[i], x);
      w[j] = f8_encode4(x[0] * inv, x[1] * inv, x[2] * inv, x[3] * inv);
    }
    *reinterpret_cast<uint4*>(out + e) = make_uint4(w[0], w[1], w[2], w[3]);
  }
  if (lane == 0)
    (kv ? a.dst.v_scale : a.dst.k_scale)[dhp * (pd / kF8Blk) + (j0 % pd) / kF8Blk] = s;
}

}  // namespace molot
