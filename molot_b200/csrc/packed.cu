// C ABI of packed-document prefill attention (molot_packed_*).
#include "packed.cuh"

#include <algorithm>
#include <cstdio>
#include <cstring>
#include <exception>
#include <new>
#include <vector>

#include "molot_b200.h"

namespace molot {
int set_last_error(int code, const char* msg);

namespace {

int pk_fail(int code, const char* msg) { return set_last_error(code, msg); }

int pk_cuda(cudaError_t e, const char* what) {
  if (e == cudaSuccess) return MOLOT_OK;
  char buf[256];
  snprintf(buf, sizeof buf, "%s: %s", what, cudaGetErrorString(e));
  return set_last_error(e == cudaErrorMemoryAllocation ? MOLOT_ERR_NOMEM : MOLOT_ERR_CUDA, buf);
}

#define PK_CUDA(call)                                  \
  do {                                                 \
    if (int rc_ = pk_cuda((call), #call)) return rc_;  \
  } while (0)

}  // namespace
}  // namespace molot

using namespace molot;

struct molot_packed_plan {
  int device = -1;
  bool built = false;
  int ndocs = 0, nq = 0, nkv = 0, d = 0, window = 0;
  int rows = 0, keys = 0;
  int* h_buf = nullptr;
  int* d_buf = nullptr;
  size_t h_cap = 0, d_cap = 0, o_row = 0;
  cudaEvent_t uploaded = nullptr;
};

namespace molot {
namespace {

int pk_build(molot_packed_plan* p, int ndocs, const int* q_lens, const int* k_lens,
             const int* prefix, int window, int nq, int nkv, int d, cudaStream_t st) {
  std::vector<PackedDoc> docs(ndocs);
  std::vector<int> row(ndocs + 1);
  long long q0 = 0, k0 = 0;
  for (int i = 0; i < ndocs; ++i) {
    const int ql = q_lens[i], kl = k_lens ? k_lens[i] : ql, pre = prefix ? prefix[i] : 0;
    if (ql < 0 || kl < 0 || pre < 0) return pk_fail(MOLOT_ERR_INVALID, "negative length or prefix");
    docs[i] = PackedDoc{(int)q0, ql, (int)k0, kl, std::min(pre, kl), {0, 0, 0}};
    row[i] = (int)q0;
    q0 += ql;
    k0 += kl;
    if (q0 > (1 << 30) || k0 > (1 << 30)) return pk_fail(MOLOT_ERR_INVALID, "batch too large");
  }
  row[ndocs] = (int)q0;
  const size_t o_row = (size_t)ndocs * (sizeof(PackedDoc) / 4), total = o_row + ndocs + 1;
  if (p->built) PK_CUDA(cudaEventSynchronize(p->uploaded));
  p->built = false;
  if (p->h_cap < total) {
    cudaFreeHost(p->h_buf);
    p->h_buf = nullptr;
    p->h_cap = 0;
    PK_CUDA(cudaMallocHost(&p->h_buf, total * sizeof(int)));
    p->h_cap = total;
  }
  if (p->d_cap < total) {
    PK_CUDA(cudaDeviceSynchronize());
    cudaFree(p->d_buf);
    p->d_buf = nullptr;
    p->d_cap = 0;
    const size_t cap = std::max<size_t>(total, 1024);
    PK_CUDA(cudaMalloc(&p->d_buf, cap * sizeof(int)));
    p->d_cap = cap;
  }
  std::memcpy(p->h_buf, docs.data(), ndocs * sizeof(PackedDoc));
  std::memcpy(p->h_buf + o_row, row.data(), (ndocs + 1) * sizeof(int));
  PK_CUDA(cudaMemcpyAsync(p->d_buf, p->h_buf, total * sizeof(int), cudaMemcpyHostToDevice, st));
  PK_CUDA(cudaEventRecord(p->uploaded, st));
  p->o_row = o_row;
  p->ndocs = ndocs;
  p->nq = nq;
  p->nkv = nkv;
  p->d = d;
  p->window = window;
  p->rows = (int)q0;
  p->keys = (int)k0;
  p->built = true;
  return MOLOT_OK;
}

template <class T>
int pk_launch(const molot_packed_plan* p, const PackedArgs& a, cudaStream_t st) {
  const dim3 grid(p->rows, p->nq);
  switch (p->d) {
    case 64: packed_simple_kernel<T, 64><<<grid, 128, 0, st>>>(a); break;
    case 128: packed_simple_kernel<T, 128><<<grid, 128, 0, st>>>(a); break;
    default: packed_simple_kernel<T, 256><<<grid, 128, 0, st>>>(a); break;
  }
  return pk_cuda(cudaGetLastError(), "packed attention launch");
}

}  // namespace
}  // namespace molot

extern "C" {

int molot_packed_plan_create(molot_packed_plan** out) {
  if (!out) return pk_fail(MOLOT_ERR_INVALID, "null out");
  *out = nullptr;
  int n = 0, dev = 0;
  if (cudaGetDeviceCount(&n) != cudaSuccess || n == 0)
    return pk_fail(MOLOT_ERR_NO_DEVICE, "no CUDA device visible");
  PK_CUDA(cudaGetDevice(&dev));
  auto* p = new (std::nothrow) molot_packed_plan();
  if (!p) return pk_fail(MOLOT_ERR_NOMEM, "plan");
  p->device = dev;
  if (int rc = pk_cuda(cudaEventCreateWithFlags(&p->uploaded, cudaEventDisableTiming),
                       "cudaEventCreate")) {
    delete p;
    return rc;
  }
  *out = p;
  return MOLOT_OK;
}

void molot_packed_plan_destroy(molot_packed_plan* p) {
  if (!p) return;
  int prev = -1;
  cudaGetDevice(&prev);
  cudaSetDevice(p->device);
  cudaDeviceSynchronize();
  cudaFreeHost(p->h_buf);
  cudaFree(p->d_buf);
  cudaEventDestroy(p->uploaded);
  if (prev >= 0) cudaSetDevice(prev);
  delete p;
}

int molot_packed_plan_build(molot_packed_plan* p, int ndocs, int nq, int nkv, int d,
                            const int* q_lens, const int* k_lens, const int* prefix, int window,
                            void* stream) {
  if (!p || !q_lens || ndocs <= 0) return pk_fail(MOLOT_ERR_INVALID, "bad plan arguments");
  if (nq <= 0 || nkv <= 0 || nq > 65535 || nq % nkv)
    return pk_fail(MOLOT_ERR_INVALID, "nq must be a multiple of nkv");
  if (d != 64 && d != 128 && d != 256)
    return pk_fail(MOLOT_ERR_UNSUPPORTED, "head_dim must be 64, 128 or 256");
  int dev = -1;
  PK_CUDA(cudaGetDevice(&dev));
  if (dev != p->device) return pk_fail(MOLOT_ERR_INVALID, "plan used on another device");
  try {
    return pk_build(p, ndocs, q_lens, k_lens, prefix, window, nq, nkv, d, (cudaStream_t)stream);
  } catch (const std::exception&) {
    return pk_fail(MOLOT_ERR_NOMEM, "plan arrays");
  }
}

int molot_packed_attend(molot_packed_plan* p, const void* q, const void* k, const void* v, void* o,
                        float* lse, int act_dtype, long long q_stride, long long k_stride,
                        long long v_stride, float scale, float softcap, const float* slopes,
                        void* stream) {
  if (!p || !p->built) return pk_fail(MOLOT_ERR_INVALID, "plan not built");
  if (act_dtype == MOLOT_ACT_F32)
    return pk_fail(MOLOT_ERR_UNSUPPORTED, "packed attention takes MOLOT_ACT_BF16 or MOLOT_ACT_F16");
  if (act_dtype != MOLOT_ACT_BF16 && act_dtype != MOLOT_ACT_F16)
    return pk_fail(MOLOT_ERR_INVALID, "unknown act_dtype");
  if (p->rows == 0) return MOLOT_OK;
  if (!q || !o || (p->keys > 0 && (!k || !v))) return pk_fail(MOLOT_ERR_INVALID, "null pointer");
  const long long hq = (long long)p->nq * p->d, hk = (long long)p->nkv * p->d;
  auto bad = [](const void* x, long long s) {
    return (reinterpret_cast<uintptr_t>(x) & 15) != 0 || s % 8 != 0;
  };
  if (q_stride < hq || k_stride < hk || v_stride < hk || bad(q, q_stride) || bad(k, k_stride) ||
      bad(v, v_stride) || bad(o, 0))
    return pk_fail(MOLOT_ERR_INVALID,
                   "rows must be 16-byte aligned and at least heads * d elements apart");
  if (!(softcap >= 0.f) || softcap > 3e38f || !(scale == scale))
    return pk_fail(MOLOT_ERR_INVALID, "softcap must be finite and not negative");
  int dev = -1;
  PK_CUDA(cudaGetDevice(&dev));
  if (dev != p->device) return pk_fail(MOLOT_ERR_INVALID, "plan used on another device");
  const PackedArgs a{q, k, v, o, lse, slopes, reinterpret_cast<const PackedDoc*>(p->d_buf),
                     p->d_buf + p->o_row, q_stride, k_stride, v_stride, p->ndocs, p->nq,
                     p->nq / p->nkv, p->window, scale, softcap};
  return act_dtype == MOLOT_ACT_BF16 ? pk_launch<__nv_bfloat16>(p, a, (cudaStream_t)stream)
                                     : pk_launch<__half>(p, a, (cudaStream_t)stream);
}

}  // extern "C"
