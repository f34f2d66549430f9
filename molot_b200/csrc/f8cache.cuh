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
#include <type_traits>

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
// One query per sequence and head over the visible blocks, split along the
// slots over the whole GPU.
//
// Work.  An item is one 16-slot block of one kv head for up to 8 of its
// query heads (a head group; nq / nkv above 8 makes several).  Items are
// numbered sequence by sequence, segment by segment (sequence, kv head, head
// group) and block by block, and every CTA takes an equal contiguous range,
// whatever the raggedness.  A warp takes one block at a time.  A segment
// inside one CTA is finished there; one that several share leaves a record
// per CTA (reference, sum, unnormalised output), merged by the last CTA to
// finish, in CTA order.
//
// Mathematics.  The products run on the tensor cores with the slots in the
// rows: S^T [16 slots x 8 heads] = K Q^T and O^T [d x 8 heads] += V^T P^T by
// mma.m16n8k16, FP16 operands, FP32 sums.  E4M3 codes are exact in FP16, so
// the block scales stay outside: K's multiplies the scores, V's the weights.
// A query row is scaled by a power of two into FP16's range; FP32 queries,
// and the weights of FP32 outputs, are split in a high and a low FP16 part
// (22 bits); for 16-bit types the query is exact in one part, and one FP16
// part of the weights is 4 bits finer than BF16.  The dims of a K row and
// the slots and dims of V are numbered so that a lane's 16-byte loads are
// its matrix operands: nothing passes through shared memory.
//
// Softmax in base 2 with one reference M per head, raised only when a
// score passes it by 2^8.  What must not overflow FP16 is the weight times
// the scale 2^ev of the block's V, so M follows s + ev: P = 2^(s - M + 6 + ev)
// <= 2^14 multiplies the codes, while l adds 2^(s - M + 38), which stays
// within FP32 for every ev in [-64, 120].  O = sum(P * code) * 2^32 / l.
//
// Bound by the bytes of the cache: a warp keeps one block of K and of V in
// flight (4 KB at d = 128), 16 warps an SM.
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
  float* rec;    // [2 * grid] records
  int* tickets;  // [B * nkv * head groups], zero between launches
  long long q_stride;
  long long items;
  int B, nq, G, HG;  // HG head groups of up to 8 per kv head
  int has_empty;     // some sequence sees nothing
  float scale, cap;
};

constexpr int kF8Warps = 8;

template <class T, int D>
struct F8Dec {
  static constexpr bool kSplit = std::is_same<T, float>::value;
  static constexpr int KS = D / 16;            // k steps of S, and m tiles of O
  static constexpr int CH = D / 64;            // 16-byte chunks of a K row per lane
  static constexpr int VB = D >= 128 ? 16 : 8;  // bytes of a V row's chunk per lane
  static constexpr int VC = D / 8 / VB;        // chunks
  static constexpr int kCtas = D == 256 ? 1 : 2;
  static constexpr int kFrag = KS * 32 * 4;      // floats of O in fragment order
  static constexpr int kRec = kFrag + 16;        // + M[8], l[8]
  static constexpr int kQ = KS * 32 * 8;         // bytes of one FP16 part of Q
  static constexpr int kSmem = kF8Warps * kRec * 4 + 2 * kQ + 64;
};

__device__ __forceinline__ uint4 ldg_stream(const void* p) {
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "l"(p));
  return v;
}
__device__ __forceinline__ uint2 ldg_stream2(const void* p) {
  uint2 v;
  asm volatile("ld.global.nc.L1::no_allocate.v2.u32 {%0, %1}, [%2];"
               : "=r"(v.x), "=r"(v.y)
               : "l"(p));
  return v;
}
__device__ __forceinline__ void cvt4(uint32_t w, uint32_t& lo, uint32_t& hi) {
  asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %2;\n\t"
      "cvt.rn.f16x2.e4m3x2 %0, a;\n\tcvt.rn.f16x2.e4m3x2 %1, b;\n\t}"
      : "=r"(lo), "=r"(hi)
      : "r"(w));
}
__device__ __forceinline__ void mma16816(float* c, uint32_t a0, uint32_t a1, uint32_t a2,
                                         uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
      "{%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t movmatrix_trans(uint32_t a) {
  uint32_t d;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
  return d;
}
__device__ __forceinline__ uint32_t pack_h2(float x, float y) {
  const __half2 h = __floats2half2_rn(x, y);
  return *reinterpret_cast<const uint32_t*>(&h);
}
// x - fp16(x), per half of the packed pair
__device__ __forceinline__ uint32_t pack_h2_rest(uint32_t hi, float x, float y) {
  const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&hi));
  return pack_h2(x - f.x, y - f.y);
}

template <class T, int D>
__global__ void __launch_bounds__(kF8Warps * 32, F8Dec<T, D>::kCtas)
    f8_decode_kernel(const __grid_constant__ F8DecodeArgs a) {
  using F = F8Dec<T, D>;
  constexpr int KS = F::KS, CH = F::CH, VC = F::VC;
  extern __shared__ __align__(16) unsigned char smem[];
  float* recs = reinterpret_cast<float*>(smem);                     // [warps][kRec]
  unsigned char* qs = smem + kF8Warps * F::kRec * 4;                // high part, then low
  float* qinv = reinterpret_cast<float*>(qs + 2 * F::kQ);           // [8]
  __shared__ int s_last;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int g = lane >> 2, t4 = lane & 3;  // fragment row group, column pair
  const int nkv = a.pool.nkv, ps = a.pool.page_size, bpp = ps / kF8Blk;
  const long long grid = gridDim.x;
  const long long x0 = blockIdx.x * a.items / grid, x1 = (blockIdx.x + 1) * a.items / grid;

  for (long long x = x0; x < x1;) {
    // the item's segment
    const int b = warp_find(a.prefix, a.B, (int)(x / a.HG));
    const F8Seq sq = a.seqs[b];
    const long long base = (long long)a.prefix[b] * a.HG;
    const int seg = (int)((x - base) / sq.nblk);
    const int i0 = (int)((x - base) % sq.nblk);
    const int i1 = (int)min((long long)sq.nblk, i0 + (x1 - x));
    const int h = seg / a.HG, hg = seg % a.HG;
    const int head0 = h * a.G + hg * 8, nh = min(8, a.G - hg * 8);
    const int* bt = a.pool.bt + (long long)b * a.pool.max_pages;
    x += i1 - i0;

    // Q in operand order, a warp per head
    {
      float v[D / 32], am = 0.f;
#pragma unroll
      for (int i = 0; i < D / 32; ++i) {
        v[i] = warp < nh ? Act<T>::one(static_cast<const T*>(a.q) + b * a.q_stride +
                                       (long long)(head0 + warp) * D + lane + 32 * i)
                         : 0.f;
        am = fmaxf(am, finite_abs(v[i]));
      }
      am = warp_max(am);
      // 2^e brings the largest magnitude into [2^13, 2^14)
      const int ex = (int)(__float_as_uint(am) >> 23);
      const int e = am > 0.f ? min(max(140 - ex, -126), 126) : 0;
      const float up = f8_exp2i(e);
#pragma unroll
      for (int i = 0; i < D / 32; ++i) {
        const int dd = lane + 32 * i;
        const int j = (dd >> 6) * 4 + ((dd & 15) >> 2), tt = (dd & 63) >> 4, r = dd & 3;
        const int at = (j * 32 + warp * 4 + tt) * 4 + r;
        const __half hi = __float2half_rn(v[i] * up);
        reinterpret_cast<__half*>(qs)[at] = hi;
        if (F::kSplit)
          reinterpret_cast<__half*>(qs + F::kQ)[at] =
              __float2half_rn(v[i] * up - __half2float(hi));
      }
      if (lane == 0) qinv[warp] = f8_exp2i(-e);
    }
    __syncthreads();
    uint2 qh[KS];
#pragma unroll
    for (int j = 0; j < KS; ++j) qh[j] = reinterpret_cast<const uint2*>(qs)[j * 32 + lane];
    const float sc0 = a.scale * qinv[2 * t4], sc1 = a.scale * qinv[2 * t4 + 1];
    float slope0 = 0.f, slope1 = 0.f;
    if (a.slopes) {
      if (2 * t4 < nh) slope0 = a.slopes[head0 + 2 * t4];
      if (2 * t4 + 1 < nh) slope1 = a.slopes[head0 + 2 * t4 + 1];
    }

    float o[KS][4], m0 = -CUDART_INF_F, m1 = -CUDART_INF_F, l0 = 0.f, l1 = 0.f;
#pragma unroll
    for (int i = 0; i < KS; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;

    auto block_of = [&](int i) { return i < sq.na ? sq.a0 + i : sq.b0 + i - sq.na; };
    uint4 ka[CH], kb[CH];
    uint4 vr[4][VC];  // slots 2t, 2t + 1, 2t + 8, 2t + 9 (VB = 8: the low halves)
    float ks = 0.f, vs = 0.f;
    long long nrow = 0;  // row index (times d: byte offset) of the block being fetched
    int pages = 0;       // lane l: page of block i + 8 l of the current run
    auto locate = [&](int i) {  // of block i, page from the run's lane
      const int k = ((i - i0) / kF8Warps) & 31;
      if (k == 0) {
        const int bi = i + lane * kF8Warps;
        pages = bi < i1 ? bt[block_of(bi) / bpp] : 0;
      }
      const long long page = __shfl_sync(0xffffffffu, pages, k);
      return ((page * nkv + h) * bpp + block_of(i) % bpp);
    };
    auto load_k = [&](long long blk) {
      ks = __ldg(a.pool.k_scale + blk);
      const uint8_t* p = a.pool.k + blk * (kF8Blk * D) + g * D + t4 * 16;
#pragma unroll
      for (int c = 0; c < CH; ++c) {
        ka[c] = ldg_stream(p + c * 64);
        kb[c] = ldg_stream(p + 8 * D + c * 64);
      }
    };
    auto load_v = [&](long long blk) {
      vs = __ldg(a.pool.v_scale + blk);
#pragma unroll
      for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int c = 0; c < VC; ++c) {
          const uint8_t* p = a.pool.v + blk * (kF8Blk * D) +
                             (2 * t4 + (r & 1) + (r & 2) * 4) * D + c * 128 + g * F::VB;
          if (F::VB == 16) {
            vr[r][c] = ldg_stream(p);
          } else {
            const uint2 w = ldg_stream2(p);
            vr[r][c] = make_uint4(w.x, w.y, 0, 0);
          }
        }
    };
    int i = i0 + warp;
    if (i < i1) {
      nrow = locate(i);
      load_k(nrow);
      load_v(nrow);
    }
    for (; i < i1; i += kF8Warps) {
      // S^T: two chains, so that a product need not wait for the last one
      float s[2][4] = {};
#pragma unroll
      for (int c = 0; c < CH; ++c) {
        const uint32_t wa[4] = {ka[c].x, ka[c].y, ka[c].z, ka[c].w};
        const uint32_t wb[4] = {kb[c].x, kb[c].y, kb[c].z, kb[c].w};
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          const int j = c * 4 + w;
          uint32_t a0, a1, a2, a3;
          cvt4(wa[w], a0, a2);
          cvt4(wb[w], a1, a3);
          mma16816(s[w & 1], a0, a1, a2, a3, qh[j].x, qh[j].y);
          if (F::kSplit) {
            const uint2 ql = reinterpret_cast<const uint2*>(qs + F::kQ)[j * 32 + lane];
            mma16816(s[(w & 1) ^ 1], a0, a1, a2, a3, ql.x, ql.y);
          }
        }
      }
      const float ksc = ks, vsc = vs;
      const int blk_t = block_of(i) * kF8Blk;
      const bool more = i + kF8Warps < i1;
      if (more) {
        nrow = locate(i + kF8Warps);
        load_k(nrow);
      }
      // base-2 scores: [0..1] slot g, [2..3] slot g + 8; heads 2t, 2t + 1
      float z[4];
      {
        const float c0 = ksc * sc0, c1 = ksc * sc1;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const float dist = (float)(sq.n - 1 - (blk_t + g + (r >> 1) * 8));
          z[r] = score_logit((s[0][r] + s[1][r]) * (r & 1 ? c1 : c0), a.cap,
                             r & 1 ? slope1 : slope0, dist);
        }
      }
      const bool edge = blk_t < sq.first || blk_t + kF8Blk > sq.n ||
                        (blk_t < sq.lo && blk_t + kF8Blk > sq.sink_end);
      if (edge) {  // mask slots, and zero V where a code may be NaN
        auto see = [&](int t) {
          return t >= sq.first && t < sq.n && (t >= sq.lo || t < sq.sink_end);
        };
        if (!see(blk_t + g)) z[0] = z[1] = -CUDART_INF_F;
        if (!see(blk_t + g + 8)) z[2] = z[3] = -CUDART_INF_F;
#pragma unroll
        for (int r = 0; r < 4; ++r)
          if (!see(blk_t + 2 * t4 + (r & 1) + (r & 2) * 4)) {
#pragma unroll
            for (int c = 0; c < VC; ++c) vr[r][c] = make_uint4(0, 0, 0, 0);
          }
      }
      if (a.score) {
        float* sp = a.score + (((long long)a.prefix[b] + (long long)h * sq.nblk + i) * kF8Blk + g) *
                                  a.G + hg * 8 + 2 * t4;
        if (2 * t4 < nh) sp[0] = z[0], sp[8 * a.G] = z[2];
        if (2 * t4 + 1 < nh) sp[1] = z[1], sp[8 * a.G + 1] = z[3];
      }
      const float ev = (float)((int)(__float_as_uint(vsc) >> 23) - 127);
      const float q0 = fmaxf(z[0], z[2]) + ev, q1 = fmaxf(z[1], z[3]) + ev;
      if (__any_sync(0xffffffffu, q0 > m0 + 8.f || q1 > m1 + 8.f)) {
        float n0 = q0, n1 = q1;
#pragma unroll
        for (int k = 4; k < 32; k <<= 1) {
          n0 = fmaxf(n0, __shfl_xor_sync(0xffffffffu, n0, k));
          n1 = fmaxf(n1, __shfl_xor_sync(0xffffffffu, n1, k));
        }
        n0 = fmaxf(n0, m0);
        n1 = fmaxf(n1, m1);
        const float f0 = n0 == m0 ? 1.f : ex2(m0 - n0), f1 = n1 == m1 ? 1.f : ex2(m1 - n1);
        m0 = n0, m1 = n1;
        l0 *= f0, l1 *= f1;
#pragma unroll
        for (int k = 0; k < KS; ++k) {
          o[k][0] *= f0, o[k][2] *= f0;
          o[k][1] *= f1, o[k][3] *= f1;
        }
      }
      const float r0 = 38.f - m0, r1 = 38.f - m1;
      const float up = vsc * 0x1p-32f;  // 2^(ev - 32)
      float p[4];
#pragma unroll
      for (int r = 0; r < 4; ++r)
        p[r] = z[r] == -CUDART_INF_F ? 0.f : ex2(z[r] + (r & 1 ? r1 : r0));
      l0 += p[0] + p[2];
      l1 += p[1] + p[3];
#pragma unroll
      for (int r = 0; r < 4; ++r) p[r] *= up;
      const uint32_t h0 = pack_h2(p[0], p[1]), h1 = pack_h2(p[2], p[3]);
      const uint32_t b0 = movmatrix_trans(h0), b1 = movmatrix_trans(h1);
      uint32_t e0 = 0, e1 = 0;
      if (F::kSplit) {
        e0 = movmatrix_trans(pack_h2_rest(h0, p[0], p[1]));
        e1 = movmatrix_trans(pack_h2_rest(h1, p[2], p[3]));
      }
#pragma unroll
      for (int c = 0; c < VC; ++c) {
#pragma unroll
        for (int w = 0; w < F::VB / 4; ++w) {
          const uint32_t* x0w = &vr[0][c].x;
          const uint32_t* x1w = &vr[1][c].x;
          const uint32_t* x2w = &vr[2][c].x;
          const uint32_t* x3w = &vr[3][c].x;
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            const uint32_t sel = u ? 0x7362 : 0x5140;
            uint32_t a0, a1, a2, a3;
            cvt4(__byte_perm(x0w[w], x1w[w], sel), a0, a1);
            cvt4(__byte_perm(x2w[w], x3w[w], sel), a2, a3);
            const int k = c * (F::VB / 2) + 2 * w + u;
            mma16816(o[k], a0, a1, a2, a3, b0, b1);
            if (F::kSplit) mma16816(o[k], a0, a1, a2, a3, e0, e1);
          }
        }
      }
      if (more) load_v(nrow);
    }

    // merge the warps: records in fragment order, then one sum per position
#pragma unroll
    for (int k = 4; k < 32; k <<= 1) {
      l0 += __shfl_xor_sync(0xffffffffu, l0, k);
      l1 += __shfl_xor_sync(0xffffffffu, l1, k);
    }
    {
      float* r = recs + warp * F::kRec;
#pragma unroll
      for (int k = 0; k < KS; ++k)
        reinterpret_cast<float4*>(r)[k * 32 + lane] = make_float4(o[k][0], o[k][1], o[k][2], o[k][3]);
      if (g == 0) {
        r[F::kFrag + 2 * t4] = m0, r[F::kFrag + 2 * t4 + 1] = m1;
        r[F::kFrag + 8 + 2 * t4] = l0, r[F::kFrag + 9 + 2 * t4] = l1;
      }
    }
    __syncthreads();

    // Sums of n records (stride st floats) at fragment position f4 for heads
    // 2t, 2t + 1; M and l of the heads along with it.
    auto gather = [&](const float* r, int n, long long st, int f4, float4& acc, float2& mm,
                      float2& ll) {
      const int hh = 2 * (f4 & 3);
      mm = make_float2(-CUDART_INF_F, -CUDART_INF_F);
#pragma unroll 8
      for (int k = 0; k < n; ++k) {
        const float2 v = *reinterpret_cast<const float2*>(r + k * st + F::kFrag + hh);
        mm.x = fmaxf(mm.x, v.x), mm.y = fmaxf(mm.y, v.y);
      }
      acc = make_float4(0.f, 0.f, 0.f, 0.f);
      ll = make_float2(0.f, 0.f);
#pragma unroll 8
      for (int k = 0; k < n; ++k) {
        const float* rk = r + k * st;
        const float2 mv = *reinterpret_cast<const float2*>(rk + F::kFrag + hh);
        const float2 lv = *reinterpret_cast<const float2*>(rk + F::kFrag + 8 + hh);
        const float4 v = reinterpret_cast<const float4*>(rk)[f4];
        const float fx = mv.x == -CUDART_INF_F ? 0.f : ex2(mv.x - mm.x);
        const float fy = mv.y == -CUDART_INF_F ? 0.f : ex2(mv.y - mm.y);
        ll.x += fx * lv.x, ll.y += fy * lv.y;
        acc.x += fx * v.x, acc.z += fx * v.z;
        acc.y += fy * v.y, acc.w += fy * v.w;
      }
    };
    // O, log-sum-exp of position f4: dims dim, dim + 1 of heads 2t, 2t + 1
    auto finish = [&](int f4, const float4& acc, const float2& mm, const float2& ll) {
      const int k = f4 >> 5, gg = (f4 >> 2) & 7, hh = 2 * (f4 & 3);
      constexpr int KC = F::VB / 2;  // m tiles per chunk
      const int dim = (k / KC) * 128 + gg * F::VB + 2 * (k % KC);
#pragma unroll
      for (int y = 0; y < 2; ++y) {
        if (hh + y >= nh) continue;
        const float l = y ? ll.y : ll.x;
        const float inv = l > 0.f || l != l ? 0x1p32f / l : 0.f;
        const long long row = (long long)b * a.nq + head0 + hh + y;
        T* op = static_cast<T*>(a.o) + row * D + dim;
        Act<T>::store(op, (y ? acc.y : acc.x) * inv);
        Act<T>::store(op + 1, (y ? acc.w : acc.z) * inv);
        if (k == 0 && gg == 0) {
          const float z = l == 0.f ? -CUDART_INF_F : (y ? mm.y : mm.x) - 38.f + log2f(l);
          if (a.lse) a.lse[row] = z * kLn2;
          if (a.lse2) a.lse2[row] = z;
        }
      }
    };
    const bool whole = i0 == 0 && i1 == sq.nblk;
    float* rec = nullptr;
    if (!whole) rec = a.rec + (2 * (long long)blockIdx.x + (x - (i1 - i0) == x0 ? 0 : 1)) * F::kRec;
    for (int f4 = tid; f4 < KS * 32; f4 += kF8Warps * 32) {
      float4 acc;
      float2 mm, ll;
      gather(recs, kF8Warps, F::kRec, f4, acc, mm, ll);
      if (whole) {
        finish(f4, acc, mm, ll);
      } else {
        reinterpret_cast<float4*>(rec)[f4] = acc;
        if (f4 < 4) {
          *reinterpret_cast<float2*>(rec + F::kFrag + 2 * f4) = mm;
          *reinterpret_cast<float2*>(rec + F::kFrag + 8 + 2 * f4) = ll;
        }
      }
    }
    if (!whole) {
      // CTAs [c0, c1] share the segment's items [y0, y1]
      const long long y0 = base + (long long)seg * sq.nblk, y1 = y0 + sq.nblk - 1;
      const long long c0 = ((y0 + 1) * grid + a.items - 1) / a.items - 1;
      const long long c1 = ((y1 + 1) * grid + a.items - 1) / a.items - 1;
      __threadfence();
      __syncthreads();
      if (tid == 0) {
        int* tk = a.tickets + ((long long)b * nkv + h) * a.HG + hg;
        const bool last = ptx::atom_add_acq_rel_gpu(tk, 1) == (int)(c1 - c0);
        if (last) *tk = 0;
        s_last = last;
      }
      __syncthreads();
      if (s_last) {
        __threadfence();
        // the first CTA's record is its first one when the segment starts
        // its range, else its last; the others' ranges start inside
        const long long first = 2 * c0 + (c0 * a.items / grid == y0 ? 0 : 1);
        const int n = (int)(c1 - c0);
        for (int f4 = tid; f4 < KS * 32; f4 += kF8Warps * 32) {
          float4 acc, acc1;
          float2 mm, ll, mm1, ll1;
          gather(a.rec + first * F::kRec, 1, 0, f4, acc1, mm1, ll1);
          gather(a.rec + 2 * (c0 + 1) * F::kRec, n, 2 * F::kRec, f4, acc, mm, ll);
          const float nx = fmaxf(mm.x, mm1.x), ny = fmaxf(mm.y, mm1.y);
          const float ax = mm1.x == -CUDART_INF_F ? 0.f : ex2(mm1.x - nx);
          const float ay = mm1.y == -CUDART_INF_F ? 0.f : ex2(mm1.y - ny);
          const float bx = mm.x == -CUDART_INF_F ? 0.f : ex2(mm.x - nx);
          const float by = mm.y == -CUDART_INF_F ? 0.f : ex2(mm.y - ny);
          acc = make_float4(acc1.x * ax + acc.x * bx, acc1.y * ay + acc.y * by,
                            acc1.z * ax + acc.z * bx, acc1.w * ay + acc.w * by);
          ll = make_float2(ll1.x * ax + ll.x * bx, ll1.y * ay + ll.y * by);
          finish(f4, acc, make_float2(nx, ny), ll);
        }
      }
    }
    __syncthreads();  // shared memory is free for the next segment
  }
  if (a.has_empty)
    for (int b = blockIdx.x; b < a.B; b += gridDim.x) {
      if (a.seqs[b].nblk > 0) continue;
      for (int i = tid; i < a.nq * D; i += kF8Warps * 32)
        Act<T>::store(static_cast<T*>(a.o) + (long long)b * a.nq * D + i, 0.f);
      for (int i = tid; i < a.nq; i += kF8Warps * 32) {
        if (a.lse) a.lse[(long long)b * a.nq + i] = -CUDART_INF_F;
        if (a.lse2) a.lse2[(long long)b * a.nq + i] = -CUDART_INF_F;
      }
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
