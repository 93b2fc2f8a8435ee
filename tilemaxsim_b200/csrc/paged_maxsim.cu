// paged_maxsim.cu -- MaxSim over a paged 8-bit corpus (see paged.cu for the pages):
//
//   score[q, doc] = sum_i max over the document's pages p of  scale_p * max_j <Q[q,i,:], code_pj>
//
// The scale of a page is not negative, so it is applied once to the page's maximum. Rows behind a
// document's last token repeat that token: maxima run over whole pages.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include "tms_device.cuh"
#include "tms_internal.h"

namespace tms {
namespace {

struct PagedArgs {
  const void* Q;
  int q_bf16;
  int64_t n_queries;
  int nq, d, page_shift;
  const uint8_t* codes;
  const float* scales;
  int64_t n_pages;
  const int64_t* page_offsets;
  const int32_t* page_ids;
  int64_t n_docs, page_cap;
  float* out;
};

// A maximum that a NaN survives.
__device__ __forceinline__ float max_nan(float x, float y) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(x), "f"(y));
  return r;
}

constexpr int kSimpleThreads = 128;

// One CTA for each (query, document): a thread takes a page row and walks the query's rows.
__global__ void __launch_bounds__(kSimpleThreads) paged_simple_kernel(const PagedArgs a) {
  extern __shared__ float q[];  // (nq, d), then (4, ) warp maxima
  float* const part = q + a.nq * a.d;
  const int64_t doc = blockIdx.x;
  const int64_t query = blockIdx.y;
  for (int i = threadIdx.x; i < a.nq * a.d; i += kSimpleThreads) {
    const int64_t at = query * a.nq * a.d + i;
    q[i] = a.q_bf16 ? __bfloat162float(static_cast<const __nv_bfloat16*>(a.Q)[at])
                    : __half2float(static_cast<const __half*>(a.Q)[at]);
  }
  __syncthreads();
  int64_t lo = a.page_offsets[doc], hi = a.page_offsets[doc + 1];
  lo = lo < 0 ? 0 : lo;
  hi = hi > a.page_cap ? a.page_cap : hi;
  float score = hi > lo ? 0.f : -__builtin_huge_valf();
  for (int i = 0; i < a.nq && hi > lo; ++i) {
    float best = -__builtin_huge_valf();
    for (int64_t r = (lo << a.page_shift) + threadIdx.x; r < (hi << a.page_shift); r += kSimpleThreads) {
      const int64_t id = a.page_ids[r >> a.page_shift];
      if (id < 0 || id >= a.n_pages) continue;
      const uint8_t* c = a.codes + ((id << a.page_shift) + (r & ((1 << a.page_shift) - 1))) * a.d;
      float s = 0.f;
      for (int e = 0; e < a.d; ++e)
        s += q[i * a.d + e] * __half2float(__half(__nv_cvt_fp8_to_halfraw(c[e], __NV_E4M3)));
      best = max_nan(best, s * a.scales[id]);
    }
    for (int o = 16; o > 0; o >>= 1) best = max_nan(best, __shfl_xor_sync(0xffffffffu, best, o));
    if (lane_id() == 0) part[threadIdx.x >> 5] = best;
    __syncthreads();
    for (int w = 0; w < kSimpleThreads / 32; ++w)
      best = max_nan(best, part[w]);
    __syncthreads();
    score += best;
  }
  if (threadIdx.x == 0) a.out[query * a.n_docs + doc] = score;
}

}  // namespace
}  // namespace tms

using namespace tms;

extern "C" size_t tms_paged_workspace_size(int64_t n_queries, int64_t nq, int64_t n_docs) {
  if (n_queries <= 0 || nq <= 32 || n_docs <= 0) return 0;
  return static_cast<size_t>(n_queries * ((nq + 31) / 32) * n_docs) * sizeof(float);
}

extern "C" int tms_paged_maxsim(const void* Q, int q_dtype, int64_t n_queries, int64_t nq,
                                int64_t d, const void* codes, const float* scales, int64_t n_pages,
                                int64_t page_size, const int64_t* page_offsets,
                                const int32_t* page_ids, const int32_t* page_docs, int64_t n_docs,
                                int64_t page_capacity, float* out, void* workspace,
                                size_t workspace_bytes, void* stream) {
  NvtxRange nvtx_range("tms_paged_maxsim");
  if (q_dtype != TMS_F16 && q_dtype != TMS_BF16) return TMS_ERR_INVALID;
  if (n_queries < 0 || nq < 0 || d <= 0 || n_docs < 0 || n_pages < 0 || page_capacity < 0)
    return TMS_ERR_INVALID;
  if (page_size != 16 && page_size != 32 && page_size != 64 && page_size != 128) return TMS_ERR_UNSUPPORTED;
  if (d % 16 != 0 || d > TMS_PAGED_MAX_D) return TMS_ERR_UNSUPPORTED;
  if (n_queries == 0 || n_docs == 0) return TMS_OK;
  if (nq == 0) return TMS_ERR_INVALID;
  if (n_docs >= (int64_t(1) << 31) || page_capacity >= (int64_t(1) << 31) ||
      n_pages * page_size >= (int64_t(1) << 31))
    return TMS_ERR_UNSUPPORTED;
  if (!Q || !out || !page_offsets || (page_capacity > 0 && (!page_ids || !page_docs)) ||
      (n_pages > 0 && (!codes || !scales)))
    return TMS_ERR_INVALID;
  if ((reinterpret_cast<uintptr_t>(Q) & 15) || (reinterpret_cast<uintptr_t>(codes) & 15)) return TMS_ERR_INVALID;
  const size_t need = tms_paged_workspace_size(n_queries, nq, n_docs);
  if (need && (!workspace || workspace_bytes < need)) return TMS_ERR_WORKSPACE;
  int shift = 4;
  while ((int64_t(1) << shift) < page_size) ++shift;
  const PagedArgs a{Q, q_dtype == TMS_BF16, n_queries, static_cast<int>(nq), static_cast<int>(d), shift,
                    static_cast<const uint8_t*>(codes), scales, n_pages, page_offsets, page_ids, n_docs,
                    page_capacity, out};
  const size_t smem = (nq * d + 8) * sizeof(float);
  if (cudaFuncSetAttribute(paged_simple_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                           static_cast<int>(smem)) != cudaSuccess)
    return TMS_ERR_CUDA;
  paged_simple_kernel<<<dim3(static_cast<unsigned>(n_docs), static_cast<unsigned>(n_queries)), kSimpleThreads,
                        smem, static_cast<cudaStream_t>(stream)>>>(a);
  return cuda_status(cudaGetLastError());
}
