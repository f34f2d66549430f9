// Prefill attention over packed documents with modified scores: a cap by
// tanh, a bias that grows with distance, a sliding window, and a prefix that
// every row of its document sees.  BF16 or FP16 operands on the 5th-generation
// tensor cores (tcgen05), FP32 scores, statistics and output sums.
//
// Rows.  A matrix row is a (position, query head) pair: row r of a tile is
// position r / G, head r % G of one kv head's group, so K and V are read once
// for the whole group and a short document still fills a tile.  A CTA takes
// one work item: 128 * kTiles rows of one document and one kv head (two
// 128-row tiles for d <= 128, one for d = 256, which tensor memory's 512
// columns allow), and streams the visible key tiles past them.
//
// Per key tile j and row tile s:  S_s = Q_s K_j^T (tcgen05.mma, both operands
// in shared memory, brought by TMA with the 128-byte swizzle);  the row
// tile's warpgroup reads its rows of S (a thread per row, so maxima and sums
// never leave the thread), applies cap, bias and mask, and writes
// P = 2^(x - m) in the operands' type over S's columns;  O_s += P V_j with P
// from tensor memory and V as an MN-major operand, straight as TMA brought it.
// m is raised, and O rescaled, only when a score passes it by 2^8: the
// weights stay below 2^8, which costs nothing in BF16 and stays far inside
// FP16's range.  P's rounding to 16 bits is what the tensor cores take; the
// sum l is taken of the weights before it, in FP32.
//
// The issuing thread orders  PV_s(j), QK_s(j + 1)  for s = 0, 1, so one row
// tile's products run while the other's softmax does, and the commit of
// QK_s(j + 1) also tells that PV_s(j) is done: O and S may be touched.
//
// Masked keys.  Scores are replaced, so K may hold anything there.  V
// multiplies weights of zero, and 0 * NaN is NaN, so on key tiles that some
// row does not see entirely two warps look V over in shared memory, put
// zeros in the place of infinities and NaN, and name the keys; a row that
// does see such a key becomes NaN.
//
// Warps: 0-3 (4-7) softmax of row tile 0 (1), epilogue; then one that issues
// TMA copies, one that issues MMAs, two that look over V.  Every wait is
// bounded; one that runs out records a status code and ends the CTA.
#pragma once

#include <cuda.h>

#include <type_traits>

#include "act.cuh"
#include "ptx.cuh"

namespace molot {

// A plan's work item (device array).
struct alignas(16) PackedItem {
  int q0;      // packed row of the document's first query
  int m0;      // first position row of the item, within the document's queries
  int m_rows;  // the document's query rows
  int k0, nk;  // packed key rows [k0, k0 + nk)
  int prefix;  // keys [0, prefix) of the document are seen by all its rows
  int pad[2];
};

struct PackedArgs {
  void* o;     // [T][nq][d]
  float* lse;  // [T][nq] or NULL
  const float* slopes;
  const PackedItem* items;
  int* status;
  int nq, nkv, G, BP, window;  // BP positions per row tile
  float scale, cap;
  unsigned long long timeout_ns;
};

template <int D>
struct PackedShape {
  static constexpr int kTiles = D == 256 ? 1 : 2;   // row tiles of a CTA
  static constexpr int BN = D == 256 ? 64 : 128;    // keys of a tile
  static constexpr int kBufs = 2;                   // S buffers in all
  // K / V ring, K and V in turn; at d = 64 long enough that no second CTA,
  // which would wait for tensor memory, fits the SM
  static constexpr int kSlots = D == 64 ? 8 : 4;
  static constexpr int kVSlots = kSlots / 2;
  static constexpr int kQ = 128 * D * 2;            // bytes of a Q tile
  static constexpr int kKV = BN * D * 2;            // bytes of a ring slot
  static constexpr int kBar = kTiles * kQ + kSlots * kKV;
  static constexpr int kSmem = kBar + 512 + 1024;   // + alignment
  static constexpr uint32_t kS = 0, kO = kBufs * BN;  // tensor-memory columns
  static constexpr int kSoft = 128 * kTiles;        // softmax threads
  static constexpr int kThreads = kSoft + 128;
  static_assert(kO + kTiles * D <= 512, "tensor memory");
  static_assert(kSmem <= 227 * 1024, "shared memory");
};

namespace pk {

// Shared-memory matrix descriptor, 128-byte swizzle (type 2), version 1.
// K-major: sbo = bytes between groups of 8 rows (lbo unused).  MN-major: sbo =
// bytes between groups of 8 k, lbo = bytes between groups of 64 columns.
__device__ __forceinline__ uint64_t desc128(uint32_t addr, uint32_t lbo, uint32_t sbo) {
  return (uint64_t)((addr >> 4) & 0x3fff) | ((uint64_t)((lbo >> 4) & 0x3fff) << 16) |
         ((uint64_t)((sbo >> 4) & 0x3fff) << 32) | (1ull << 46) | (2ull << 61);
}
// F32 sums of 16-bit products (bf: BF16, else FP16), M = 128; mn: B is MN-major.
__host__ __device__ constexpr uint32_t idesc(bool bf, int n, bool mn) {
  return (1u << 4) | ((bf ? 1u : 0u) << 7) | ((bf ? 1u : 0u) << 10) | ((mn ? 1u : 0u) << 16) |
         ((uint32_t)(n >> 3) << 17) | (8u << 24);
}
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t id, int acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
      "l"(a), "l"(b), "r"(id), "r"(acc)
      : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t id, int acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
      "r"(a), "l"(b), "r"(id), "r"(acc)
      : "memory");
}
__device__ __forceinline__ void commit(uint64_t* bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(
                   ptx::smem_u32(bar))
               : "memory");
}
__device__ __forceinline__ void fence_before() {
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
}
__device__ __forceinline__ void fence_after() {
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
}
#define PK_R8(r, o) "r"(r[o]), "r"(r[o + 1]), "r"(r[o + 2]), "r"(r[o + 3]), "r"(r[o + 4]), \
                    "r"(r[o + 5]), "r"(r[o + 6]), "r"(r[o + 7])
#define PK_O8(r, o) "=r"(r[o]), "=r"(r[o + 1]), "=r"(r[o + 2]), "=r"(r[o + 3]), "=r"(r[o + 4]), \
                    "=r"(r[o + 5]), "=r"(r[o + 6]), "=r"(r[o + 7])
#define PK_IO8(r, o) "+r"(r[o]), "+r"(r[o + 1]), "+r"(r[o + 2]), "+r"(r[o + 3]), "+r"(r[o + 4]), \
                     "+r"(r[o + 5]), "+r"(r[o + 6]), "+r"(r[o + 7])
// 32 columns of this thread's lane; the values are there after wait_ld.
__device__ __forceinline__ void ld32(uint32_t addr, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,"
      "%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : PK_O8(r, 0), PK_O8(r, 8), PK_O8(r, 16), PK_O8(r, 24)
      : "r"(addr));
}
__device__ __forceinline__ void wait_ld(uint32_t* r) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : PK_IO8(r, 0), PK_IO8(r, 8), PK_IO8(r, 16), PK_IO8(r, 24)::"memory");
}
__device__ __forceinline__ void st32(uint32_t addr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,"
      "%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(addr),
      PK_R8(r, 0), PK_R8(r, 8), PK_R8(r, 16), PK_R8(r, 24)
      : "memory");
}
__device__ __forceinline__ void wait_st() {
  asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
}
// TMA: box at (x, y, z) of a three-dimensional tensor; x a multiple of 64.
__device__ __forceinline__ void tma3(void* dst, const CUtensorMap* map, int x, int y, int z,
                                     uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cta.global.tile.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(ptx::smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(ptx::smem_u32(bar))
      : "memory");
}

template <class T>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  uint32_t r;
  if (std::is_same<T, __half>::value)
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  else
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
// Bits [lo, hi) of 32.
__device__ __forceinline__ uint32_t bits(int lo, int hi) {
  lo = min(max(lo, 0), 32), hi = min(max(hi, 0), 32);
  const uint32_t h = hi == 32 ? 0xffffffffu : (1u << hi) - 1u;
  const uint32_t l = lo == 32 ? 0xffffffffu : (1u << lo) - 1u;
  return h & ~l;
}

}  // namespace pk

// kMode: kPlain takes scale >= 0 and no score changes; kBias adds the
// distance bias (and takes any scale); kCap caps, with a bias that may be 0.
enum PackedMode { kPlain = 0, kBias = 1, kCap = 2 };

template <class T, int D, int kMode>
__global__ void __launch_bounds__(PackedShape<D>::kThreads, 1)
    packed_kernel(const __grid_constant__ CUtensorMap mq, const __grid_constant__ CUtensorMap mk,
                  const __grid_constant__ CUtensorMap mv, const __grid_constant__ PackedArgs a) {
  using S = PackedShape<D>;
  constexpr int BN = S::BN, NT = S::kTiles;
  constexpr bool kBf = std::is_same<T, __nv_bfloat16>::value;
  extern __shared__ unsigned char smem_raw[];
  unsigned char* smem = smem_raw + ((1024 - (ptx::smem_u32(smem_raw) & 1023)) & 1023);
  unsigned char* kv = smem + NT * S::kQ;
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + S::kBar);
  uint64_t* full = bars;                  // [kSlots]
  uint64_t* empty = bars + S::kSlots;     // [kSlots]
  uint64_t* s_full = empty + S::kSlots;   // [2]
  uint64_t* p_full = s_full + 2;          // [2]
  uint64_t* o_full = p_full + 2;
  uint64_t* q_full = o_full + 1;
  uint64_t* pv_done = q_full + 1;  // one row tile: P V of a key tile
  uint64_t* v_ok = pv_done + 1;    // [kVSlots]
  uint32_t* bad = reinterpret_cast<uint32_t*>(v_ok + S::kVSlots);  // [kVSlots][4] keys
  volatile uint32_t* tmem_sm = bad + 4 * S::kVSlots;
  volatile int* abort_flag = reinterpret_cast<volatile int*>(bad + 4 * S::kVSlots + 1);

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  constexpr int kTmaWarp = S::kSoft / 32, kMmaWarp = kTmaWarp + 1;
  const int g = blockIdx.x % a.nkv;
  const PackedItem it = a.items[blockIdx.x / a.nkv];
  // positions of the item's rows, and the key tiles they see
  const int pos0 = it.nk - it.m_rows + it.m0;
  const int pos_last = it.nk - it.m_rows + min(it.m0 + NT * a.BP, it.m_rows) - 1;
  const int lo = a.window > 0 ? max(0, pos0 - a.window + 1) : 0;
  const int hi = max(pos_last + 1, it.prefix);  // <= nk
  const int pre_t = (it.prefix + BN - 1) / BN;  // tiles [0, pre_t) hold the prefix
  const int win_t = lo / BN;                    // tiles from win_t on hold the window
  const int skip = max(0, win_t - pre_t);       // tiles between them, not visited
  const int n1 = skip > 0 ? pre_t : 0x7fffffff;
  const int ntiles = max(0, (hi + BN - 1) / BN - skip);
  auto tile_of = [&](int j) { return j < n1 ? j : j + skip; };
  // every row of the item sees every key of the tile at t0
  auto whole = [&](int t0) {
    return t0 + BN <= it.prefix ||
           (t0 + BN - 1 <= pos0 && (a.window <= 0 || pos_last - t0 < a.window));
  };
  auto wait = [&](uint64_t* bar, uint32_t par, int code) {
    if (*abort_flag) return;
    if (!ptx::mbar_wait_bounded(bar, par, a.timeout_ns)) {
      *abort_flag = 1;
      atomicCAS(a.status, 0, code);
    }
  };

  if (tid == 0) {
    for (int i = 0; i < S::kSlots; ++i) {
      ptx::mbar_init(full + i, 1);
      ptx::mbar_init(empty + i, 1);
    }
    for (int i = 0; i < 2; ++i) {
      ptx::mbar_init(s_full + i, 1);
      ptx::mbar_init(p_full + i, 128);
    }
    ptx::mbar_init(o_full, 1);
    ptx::mbar_init(q_full, 1);
    ptx::mbar_init(pv_done, 1);
    for (int i = 0; i < S::kVSlots; ++i) ptx::mbar_init(v_ok + i, 64);
    *abort_flag = 0;
    ptx::fence_mbar_init();
  }
  if (warp == kMmaWarp) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                     ptx::smem_u32(const_cast<uint32_t*>(tmem_sm))),
                 "r"(512));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  pk::fence_before();
  __syncthreads();
  pk::fence_after();
  const uint32_t tm = *tmem_sm;

  if (warp < kTmaWarp) {
    // ------------------------------------------------------------- softmax
    // 384 threads x 168 registers: 256 x 224 + 128 x 56
    if constexpr (NT == 2) ptx::setmaxnreg_inc<224>();
    const int tile = warp >> 2;
    const int r = tid & 127;
    const uint32_t lane_base = tm + ((uint32_t)((warp & 3) * 32) << 16);
    const uint32_t o_col = lane_base + S::kO + tile * D;
    const int pl = r / a.G, hd = r - pl * a.G;
    const int m = it.m0 + tile * a.BP + pl;
    const bool valid = pl < a.BP && m < it.m_rows;
    const int pos = it.nk - it.m_rows + m;
    const int head = g * a.G + hd;
    const int r_hi = valid ? pos + 1 : 0, r_lo = a.window > 0 ? pos - a.window + 1 : 0;
    const int r_pre = valid ? it.prefix : 0;
    const float sl = a.scale * kLog2e;
    const float slope = kMode != kPlain && a.slopes && valid ? a.slopes[head] * kLog2e : 0.f;
    const float cap2 = a.cap * kLog2e, in = kMode == kCap ? a.scale / a.cap : 0.f;
    // kPlain: m and the scores are in units of raw products, sl brings them
    // to base 2; else they are base-2 already.
    const float unit = kMode == kPlain ? sl : 1.f;
    float mx = -CUDART_INF_F, l = 0.f;
    for (int j = 0; j < ntiles; ++j) {
      const int buf = NT == 2 ? tile : j & 1;
      const uint32_t s_col = lane_base + S::kS + buf * BN;
      wait(s_full + buf, (NT == 2 ? j : j >> 1) & 1, 1);
      __syncwarp();
      pk::fence_after();
      uint32_t s[BN];
#pragma unroll
      for (int c = 0; c < BN; c += 32) pk::ld32(s_col + c, s + c);
#pragma unroll
      for (int c = 0; c < BN; c += 32) pk::wait_ld(s + c);
      const int t0 = tile_of(j) * BN;
      if (kMode != kPlain) {
        const float d0 = (float)(t0 - pos);
#pragma unroll
        for (int i = 0; i < BN; ++i) {
          float x = __uint_as_float(s[i]);
          if (kMode == kCap) {
            x = fmaf(-slope, fabsf(d0 + i), cap2 * tanhf(x * in));
          } else {
            x = fmaf(x, sl, -slope * fabsf(d0 + i));
          }
          s[i] = __float_as_uint(x);
        }
      }
      if (!whole(t0)) {
        // on a tile whose V was looked over: a row that sees a bad key is NaN
        const int slot = j % S::kVSlots;
        wait(v_ok + slot, (j / S::kVSlots) & 1, 2);
#pragma unroll
        for (int c = 0; c < BN; c += 32) {
          const uint32_t see =
              pk::bits(r_lo - t0 - c, r_hi - t0 - c) | pk::bits(0, r_pre - t0 - c);
#pragma unroll
          for (int i = 0; i < 32; ++i)
            if (!((see >> i) & 1)) s[c + i] = 0xff800000u;
          if (bad[slot * 4 + c / 32] & see) l = CUDART_NAN_F;
        }
      }
      float mc4[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) mc4[k] = __uint_as_float(s[k]);
#pragma unroll
      for (int i = 4; i < BN; i += 4)
#pragma unroll
        for (int k = 0; k < 4; ++k) mc4[k] = fmaxf(mc4[k], __uint_as_float(s[i + k]));
      const float mc = fmaxf(fmaxf(mc4[0], mc4[1]), fmaxf(mc4[2], mc4[3]));
      const bool raise = (mc - mx) * unit > 8.f || (mx == -CUDART_INF_F && mc > mx);
      const bool resc = raise && mx != -CUDART_INF_F;
      const float alpha = resc ? ex2((mx - mc) * unit) : 1.f;
      if (raise) mx = mc;
      l *= alpha;
      if (__any_sync(0xffffffffu, resc)) {
        if (NT == 1) {  // Q K of this tile was issued before P V of the last
          wait(pv_done, (j - 1) & 1, 2);
          __syncwarp();
          pk::fence_after();
        }
#pragma unroll 1
        for (int c = 0; c < D; c += 32) {
          uint32_t o[32];
          pk::ld32(o_col + c, o);
          pk::wait_ld(o);
#pragma unroll
          for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * alpha);
          pk::st32(o_col + c, o);
        }
      }
      // (s - m) * unit, not s * unit - m * unit: the subtraction is exact near
      // the maximum, however large the scores
      const float neg = mx == -CUDART_INF_F ? 0.f : -mx;
      float2 sum[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
#pragma unroll
      for (int c = 0; c < BN; c += 64) {
        uint32_t p[32];
#pragma unroll
        for (int i = 0; i < 32; ++i) {
          float2 z = __fadd2_rn(make_float2(__uint_as_float(s[c + 2 * i]),
                                            __uint_as_float(s[c + 2 * i + 1])),
                                make_float2(neg, neg));
          if (kMode == kPlain) z = __fmul2_rn(z, make_float2(unit, unit));
          const float x = ex2(z.x), y = ex2(z.y);
          sum[i & 1] = __fadd2_rn(sum[i & 1], make_float2(x, y));
          p[i] = pk::pack2<T>(x, y);
        }
        pk::st32(s_col + c / 2, p);
      }
      l += (sum[0].x + sum[0].y) + (sum[1].x + sum[1].y);
      pk::wait_st();
      pk::fence_before();
      ptx::mbar_arrive(p_full + buf);
    }
    // epilogue
    if (ntiles > 0) {
      wait(o_full, 0, 3);
      __syncwarp();
      pk::fence_after();
    }
    const float inv = l > 0.f || l != l ? 1.f / l : 0.f;
    const long long row = ((long long)it.q0 + m) * a.nq + head;
    T* op = static_cast<T*>(a.o) + row * D;
#pragma unroll 1
    for (int c = 0; c < D; c += 32) {
      uint32_t o[32];
      if (ntiles > 0) {
        pk::ld32(o_col + c, o);
        pk::wait_ld(o);
      }
      if (valid) {
#pragma unroll
        for (int i = 0; i < 32; i += 8) {
          uint32_t w[4];
#pragma unroll
          for (int k = 0; k < 4; ++k)
            w[k] = ntiles > 0 ? pk::pack2<T>(__uint_as_float(o[i + 2 * k]) * inv,
                                             __uint_as_float(o[i + 2 * k + 1]) * inv)
                              : 0u;
          *reinterpret_cast<uint4*>(op + c + i) = make_uint4(w[0], w[1], w[2], w[3]);
        }
      }
    }
    if (valid && a.lse)
      a.lse[row] = l == 0.f ? -CUDART_INF_F : (mx * unit + log2f(l)) * kLn2;
    pk::fence_before();
  } else {
    if constexpr (NT == 2) ptx::setmaxnreg_dec<56>();
    if (warp == kTmaWarp) {
      // ---------------------------------------------------------- copies
      if (lane == 0 && ntiles > 0) {
        ptx::mbar_arrive_expect_tx(q_full, NT * a.G * a.BP * D * 2);
        for (int i = 0; i < NT; ++i)
          for (int c = 0; c < D / 64; ++c)
            pk::tma3(smem + i * S::kQ + c * 128 * 128, &mq, c * 64, g * a.G,
                     it.q0 + it.m0 + i * a.BP, q_full);
        const int n = 2 * ntiles;
        int k = 0;
        for (; k < n && !*abort_flag; ++k) {
          const int slot = k % S::kSlots;
          if (k >= S::kSlots) wait(empty + slot, (k / S::kSlots - 1) & 1, 4);
          if (*abort_flag) break;
          ptx::mbar_arrive_expect_tx(full + slot, S::kKV);
          for (int c = 0; c < D / 64; ++c)
            pk::tma3(kv + slot * S::kKV + c * BN * 128, k & 1 ? &mv : &mk, c * 64, g,
                     it.k0 + tile_of(k >> 1) * BN, full + slot);
        }
        // copies in flight end before the CTA does
        if (*abort_flag) {
          ptx::mbar_wait_bounded(q_full, 0, a.timeout_ns);
          for (int i = max(0, k - S::kSlots); i < k; ++i)
            ptx::mbar_wait_bounded(full + i % S::kSlots, (i / S::kSlots) & 1, a.timeout_ns);
        }
      }
    } else if (warp == kMmaWarp) {
      // -------------------------------------------------------- products
      if (lane == 0 && ntiles > 0) {
        constexpr uint32_t id_s = pk::idesc(kBf, BN, false), id_o = pk::idesc(kBf, D, true);
        const uint32_t q_addr = ptx::smem_u32(smem), kv_addr = ptx::smem_u32(kv);
        auto qk = [&](int tile, int j) {  // S = Q K_j^T
          const uint32_t q = q_addr + tile * S::kQ, k = kv_addr + (2 * j) % S::kSlots * S::kKV;
          const uint32_t d = tm + S::kS + (NT == 2 ? tile : j & 1) * BN;
#pragma unroll
          for (int c = 0; c < D / 16; ++c)
            pk::mma_ss(d, pk::desc128(q + (c >> 2) * 128 * 128 + (c & 3) * 32, 0, 1024),
                       pk::desc128(k + (c >> 2) * BN * 128 + (c & 3) * 32, 0, 1024), id_s, c > 0);
        };
        auto pv = [&](int tile, int j) {  // O += P V_j
          const uint32_t v = kv_addr + (2 * j + 1) % S::kSlots * S::kKV;
          const uint32_t p = tm + S::kS + (NT == 2 ? tile : j & 1) * BN;
#pragma unroll
          for (int c = 0; c < BN / 16; ++c)
            pk::mma_ts(tm + S::kO + tile * D, p + c * 8,
                       pk::desc128(v + c * 2048, BN * 128, 1024), id_o, j > 0 || c > 0);
        };
        auto full_of = [&](int k) { wait(full + k % S::kSlots, (k / S::kSlots) & 1, 5); };
        wait(q_full, 0, 6);
        full_of(0);
        pk::fence_after();
        for (int i = 0; i < NT && !*abort_flag; ++i) {
          qk(i, 0);
          pk::commit(s_full + i);
        }
        if (!*abort_flag) pk::commit(empty);  // K_0's slot
        for (int j = 0; j < ntiles; ++j) {
          const bool next = j + 1 < ntiles;
          if (next) full_of(2 * j + 2);
          if (NT == 1 && next && !*abort_flag) {  // the other S buffer
            pk::fence_after();
            qk(0, j + 1);
            pk::commit(s_full + ((j + 1) & 1));
          }
          full_of(2 * j + 1);
          if (!whole(tile_of(j) * BN)) wait(v_ok + j % S::kVSlots, (j / S::kVSlots) & 1, 2);
          for (int i = 0; i < NT; ++i) {
            const int buf = NT == 2 ? i : j & 1;
            wait(p_full + buf, (NT == 2 ? j : j >> 1) & 1, 7);
            if (*abort_flag) break;
            pk::fence_after();
            pv(i, j);
            if (NT == 1) pk::commit(pv_done);
            if (NT == 2 && next) {
              qk(i, j + 1);
              pk::commit(s_full + i);
            }
          }
          if (*abort_flag) break;
          pk::commit(empty + (2 * j + 1) % S::kSlots);
          if (next) pk::commit(empty + (2 * j + 2) % S::kSlots);
        }
        pk::commit(o_full);
        // the products in flight end before tensor memory is freed
        if (*abort_flag) ptx::mbar_wait_bounded(o_full, 0, a.timeout_ns);
      }
    } else {
      // ------------------------------------------------- V's masked rows
      const int w = (warp - kMmaWarp - 1) * 32 + lane;  // keys w, w + 64
      for (int j = 0; j < ntiles; ++j) {
        const int k = 2 * j + 1, slot = k % S::kSlots, vs = j % S::kVSlots;
        wait(full + slot, (k / S::kSlots) & 1, 8);
        if (whole(tile_of(j) * BN)) {
          ptx::mbar_arrive(v_ok + vs);
          continue;
        }
        bool any_fix = false;
        for (int key = w; key < BN; key += 64) {
          bool found = false;
          if (!*abort_flag) {
            for (int c = 0; c < D / 64; ++c) {
#pragma unroll
              for (int i = 0; i < 8; ++i) {
                // 16-byte pieces of the row, in whatever order the swizzle put them
                uint4* p = reinterpret_cast<uint4*>(kv + slot * S::kKV + c * BN * 128 + key * 128 +
                                                    i * 16);
                uint4 x = *p;
                uint32_t* xw = &x.x;
                bool hit = false;
                constexpr uint32_t e = kBf ? 0x7f80u : 0x7c00u;
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                  const bool b0 = (xw[q] & e) == e, b1 = (xw[q] & (e << 16)) == (e << 16);
                  if (b0) xw[q] &= 0xffff0000u;
                  if (b1) xw[q] &= 0x0000ffffu;
                  hit |= b0 || b1;
                }
                if (hit) *p = x;
                found |= hit;
              }
            }
          }
          const uint32_t word = __ballot_sync(0xffffffffu, found);
          if (lane == 0) bad[vs * 4 + key / 32] = word;
          any_fix |= found;
        }
        if (any_fix) asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
        ptx::mbar_arrive(v_ok + vs);
      }
    }
  }
  __syncthreads();
  if (warp == kMmaWarp) {
    pk::fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tm), "r"(512));
  }
}

}  // namespace molot
