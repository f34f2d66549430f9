// Prefill attention over packed documents with modified scores: a cap by
// tanh, a bias that grows with distance, a sliding window, and a prefix that
// every row of its document sees.
#pragma once

#include "act.cuh"

namespace molot {

// A plan's document (device array).
struct alignas(16) PackedDoc {
  int q0, nq_rows;  // packed query rows [q0, q0 + nq_rows)
  int k0, nk;       // packed key rows [k0, k0 + nk)
  int prefix;       // keys [0, prefix) of the document are seen by all its rows
  int pad[3];
};

struct PackedArgs {
  const void* q;
  const void* k;
  const void* v;
  void* o;     // [T][nq][d]
  float* lse;  // [T][nq] or NULL
  const float* slopes;
  const PackedDoc* docs;
  const int* row0;  // [ndocs + 1] prefix of query rows
  long long q_stride, k_stride, v_stride;
  int ndocs, nq, G, window;
  float scale, cap;
};

// A CTA per query row and head, a warp per key.
template <class T, int D>
__global__ void __launch_bounds__(128) packed_simple_kernel(const __grid_constant__ PackedArgs a) {
  constexpr int E = D / 32;
  const int h = blockIdx.y, x = blockIdx.x, g = h / a.G;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const PackedDoc doc = a.docs[warp_find(a.row0, a.ndocs, x)];
  const int pos = doc.nk - doc.nq_rows + (x - doc.q0);  // position in the document
  const float slope = a.slopes ? a.slopes[h] : 0.f;
  const int lo = a.window > 0 ? max(0, pos - a.window + 1) : 0;
  const int pre = min(doc.prefix, doc.nk);
  float q[E], o[E], m = -CUDART_INF_F, l = 0.f;
#pragma unroll
  for (int i = 0; i < E; ++i) {
    q[i] = Act<T>::one(static_cast<const T*>(a.q) + x * a.q_stride + (long long)h * D + lane * E + i);
    o[i] = 0.f;
  }
  for (int t = warp; t < max(pos + 1, pre); t += 4) {
    if (!(t < pre || (t >= lo && t <= pos))) continue;
    const T* kr = static_cast<const T*>(a.k) + (doc.k0 + t) * a.k_stride + (long long)g * D + lane * E;
    const T* vr = static_cast<const T*>(a.v) + (doc.k0 + t) * a.v_stride + (long long)g * D + lane * E;
    float s = 0.f;
#pragma unroll
    for (int j = 0; j < E; ++j) s += q[j] * Act<T>::one(kr + j);
#pragma unroll
    for (int i = 16; i; i >>= 1) s += __shfl_xor_sync(0xffffffffu, s, i);
    s = score_logit(s * a.scale, a.cap, slope, (float)abs(pos - t));
    const float mn = fmaxf(m, s), al = ex2(m - mn), p = ex2(s - mn);
    m = mn;
    l = l * al + p;
#pragma unroll
    for (int j = 0; j < E; ++j) o[j] = o[j] * al + p * Act<T>::one(vr + j);
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
  const float inv = lt > 0.f ? 1.f / lt : 0.f;
  for (int i = threadIdx.x; i < D; i += 128)
    Act<T>::store(static_cast<T*>(a.o) + ((long long)x * a.nq + h) * D + i,
                  inv * (w[0] * so[0][i] + w[1] * so[1][i] + w[2] * so[2][i] + w[3] * so[3][i]));
  if (threadIdx.x == 0 && a.lse)
    a.lse[(long long)x * a.nq + h] = lt > 0.f ? (mx + log2f(lt)) * kLn2 : -CUDART_INF_F;
}

}  // namespace molot
