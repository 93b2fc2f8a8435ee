// paged.cu -- the paged 8-bit corpus: page tables, writing tokens into pages, reading them back.
// (The scoring kernel over such a corpus is in paged_maxsim.cu.)
//
// A pool holds n_pages pages of `page_size` token rows of d e4m3 values, with one fp32 scale for
// each page: token value = scale * code. A document owns ceil(length / page_size) pages, listed in
// order in a CSR table (page_offsets, page_ids); page_docs names the owner of every table entry.
// Rows behind a document's last token repeat that token, so a maximum over whole pages equals the
// maximum over the document's tokens and no reader needs the lengths.
//
// No counterpart in the reference, whose corpora are fixed tensors (src/flash_maxsim_kernel.py:248-273).
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include "tms_device.cuh"
#include "tms_internal.h"

namespace tms {
namespace {

// ------------------------------------------------------------------------------------------------
// page tables
// ------------------------------------------------------------------------------------------------
struct TableArgs {
  const int64_t* lengths;      // (n_lengths,)
  int64_t n_lengths;
  const int64_t* doc_ids;      // (n_docs,) or nullptr: document i is lengths[i]
  int64_t n_docs;
  const int64_t* src_offsets;  // (n_lengths + 1,) or nullptr: pages are taken in order
  const int32_t* pages;
  int64_t n_src;
  int page_shift;
  int64_t* page_offsets;   // (n_docs + 1,)
  int64_t* token_offsets;  // (n_docs + 1,)
  int32_t* page_ids;       // (page_cap,)
  int32_t* page_docs;      // (page_cap,)
  int64_t page_cap;
  int64_t* slots;          // (token_cap,) or nullptr
  int64_t token_cap;
  int64_t* tile_sums;      // workspace: (tiles, 2) pages and tokens of each tile of documents
};

constexpr int kTableThreads = 256;
constexpr int kTileDocs = 1024;  // documents of one tile (four for each thread)

// Document i's length; an id outside the store has none, a negative length counts as zero, and one
// of 2^31 or more, which no pool holds, as 2^31 - 1 (so that no sum of lengths overflows).
__device__ __forceinline__ int64_t table_length(const TableArgs& a, int64_t i) {
  int64_t id = i;
  if (a.doc_ids) {
    id = __ldg(a.doc_ids + i);
    if (id < 0 || id >= a.n_lengths) return 0;
  }
  const int64_t len = __ldg(a.lengths + id);
  return len < 0 ? 0 : len > 0x7fffffff ? 0x7fffffff : len;
}

__device__ __forceinline__ int64_t warp_inclusive(int64_t v) {
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t y = __shfl_up_sync(0xffffffffu, v, o);
    if (lane_id() >= static_cast<uint32_t>(o)) v += y;
  }
  return v;
}

// Block-wide exclusive scan of (pages, tokens), one pair a thread; totals come back in *tp and *tt.
__device__ __forceinline__ void block_scan2(int64_t& p, int64_t& t, int64_t* tp, int64_t* tt,
                                            int64_t (*sh)[2]) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t ip = warp_inclusive(p), it = warp_inclusive(t);
  if (lane == 31) {
    sh[warp][0] = ip;
    sh[warp][1] = it;
  }
  __syncthreads();
  int64_t bp = 0, bt = 0, sp = 0, st = 0;
  for (int w = 0; w < static_cast<int>(blockDim.x >> 5); ++w) {
    if (w == warp) {
      bp = sp;
      bt = st;
    }
    sp += sh[w][0];
    st += sh[w][1];
  }
  __syncthreads();
  *tp = sp;
  *tt = st;
  p = bp + ip - p;
  t = bt + it - t;
}

// Sums of one tile of documents.
__global__ void __launch_bounds__(kTableThreads) table_sums_kernel(const TableArgs a) {
  __shared__ int64_t sh[kTableThreads / 32][2];
  const int64_t i0 = static_cast<int64_t>(blockIdx.x) * kTileDocs;
  const int64_t round = (int64_t(1) << a.page_shift) - 1;
  int64_t p = 0, t = 0, tp, tt;
  for (int j = 0; j < kTileDocs / kTableThreads; ++j) {
    const int64_t i = i0 + j * kTableThreads + threadIdx.x;
    const int64_t len = i < a.n_docs ? table_length(a, i) : 0;
    p += (len + round) >> a.page_shift;
    t += len;
  }
  block_scan2(p, t, &tp, &tt, sh);
  if (threadIdx.x == 0) {
    a.tile_sums[2 * blockIdx.x] = tp;
    a.tile_sums[2 * blockIdx.x + 1] = tt;
  }
}

// Both offset arrays: one CTA a tile, its base the sum of the tiles before it.
__global__ void __launch_bounds__(kTableThreads) table_offsets_kernel(const TableArgs a) {
  __shared__ int64_t sh[kTableThreads / 32][2];
  const int64_t i0 = static_cast<int64_t>(blockIdx.x) * kTileDocs;
  const int64_t round = (int64_t(1) << a.page_shift) - 1;
  int64_t p = 0, t = 0, bp, bt;
  for (int64_t w = threadIdx.x; w < blockIdx.x; w += kTableThreads) {
    p += a.tile_sums[2 * w];
    t += a.tile_sums[2 * w + 1];
  }
  block_scan2(p, t, &bp, &bt, sh);
  for (int j = 0; j < kTileDocs / kTableThreads; ++j) {
    const int64_t i = i0 + j * kTableThreads + threadIdx.x;
    const int64_t len = i < a.n_docs ? table_length(a, i) : 0;
    int64_t tp, tt;
    p = (len + round) >> a.page_shift;
    t = len;
    block_scan2(p, t, &tp, &tt, sh);
    if (i < a.n_docs) {
      a.page_offsets[i] = bp + p;
      a.token_offsets[i] = bt + t;
    }
    bp += tp;
    bt += tt;
  }
  if (threadIdx.x == 0 && i0 + kTileDocs >= a.n_docs) {
    a.page_offsets[a.n_docs] = bp;
    a.token_offsets[a.n_docs] = bt;
  }
}

// The last document d in [0, n_docs) with page_offsets[d] <= k (k lies below the total).
__device__ __forceinline__ int64_t owner_of(const int64_t* page_offsets, int64_t n_docs, int64_t k) {
  int64_t lo = 0, hi = n_docs;  // the first offset above k is in (lo, hi]
  while (hi - lo > 1) {
    const int64_t mid = (lo + hi) >> 1;
    if (page_offsets[mid] <= k) lo = mid;
    else hi = mid;
  }
  return lo;
}

// Page ids, owners and token slots: a warp takes 32 consecutive table entries, finds their owners
// (a lane for each) and then writes the slots of one page after the other.
__global__ void __launch_bounds__(kTableThreads) table_fill_kernel(const TableArgs a) {
  const int lane = threadIdx.x & 31;
  const int64_t warps = static_cast<int64_t>(gridDim.x) * (kTableThreads / 32);
  const int64_t warp = static_cast<int64_t>(blockIdx.x) * (kTableThreads / 32) + (threadIdx.x >> 5);
  const int64_t total = a.page_offsets[a.n_docs];
  const int64_t page = int64_t(1) << a.page_shift;
  for (int64_t k0 = warp * 32; k0 < a.page_cap; k0 += warps * 32) {
    const int64_t k = k0 + lane;
    int64_t tok = 0, id = -1, doc = -1;
    int count = 0;
    if (k < total && k < a.page_cap) {
      doc = owner_of(a.page_offsets, a.n_docs, k);
      const int64_t nth = k - a.page_offsets[doc];
      const int64_t t0 = a.token_offsets[doc], t1 = a.token_offsets[doc + 1];
      int64_t src = k;
      if (a.src_offsets) src = __ldg(a.src_offsets + (a.doc_ids ? __ldg(a.doc_ids + doc) : doc)) + nth;
      if (src >= 0 && src < a.n_src) id = __ldg(a.pages + src);
      tok = t0 + nth * page;
      count = static_cast<int>(t1 - tok < page ? t1 - tok : page);
    }
    if (k < a.page_cap) {
      a.page_ids[k] = static_cast<int32_t>(id);
      a.page_docs[k] = static_cast<int32_t>(doc);
    }
    if (!a.slots) continue;
    for (int l = 0; l < 32; ++l) {
      const int n = __shfl_sync(0xffffffffu, count, l);
      const int64_t t = __shfl_sync(0xffffffffu, tok, l);
      const int64_t pid = __shfl_sync(0xffffffffu, id, l);
      for (int j = lane; j < n; j += 32)
        if (t + j < a.token_cap) a.slots[t + j] = pid < 0 ? -1 : (pid << a.page_shift) + j;
    }
  }
  if (!a.slots) return;
  int64_t rest = a.token_offsets[a.n_docs];  // tokens from here on have no table entry
  if (total > a.page_cap) {
    const int64_t doc = owner_of(a.page_offsets, a.n_docs, a.page_cap);
    rest = a.token_offsets[doc] + ((a.page_cap - a.page_offsets[doc]) << a.page_shift);
  }
  for (int64_t t = rest + warp * 32 + lane; t < a.token_cap; t += warps * 32) a.slots[t] = -1;
}

// ------------------------------------------------------------------------------------------------
// writing tokens into pages
// ------------------------------------------------------------------------------------------------
constexpr float kE4m3Max = 448.f;

struct WriteArgs {
  const void* x;
  const void* residual;  // nullptr, or laid out as x
  const void* weight;    // (d,) or nullptr
  int64_t stride_doc;    // padded input: elements from one document to the next
  int64_t stride_tok;    // elements from one token row to the next
  int64_t n_rows;        // ragged: rows of x; padded: rows of each document
  int padded;
  int norm;
  float eps;
  int d, page_shift;
  const int64_t* page_offsets;
  const int64_t* token_offsets;
  const int32_t* page_ids;
  const int32_t* page_docs;
  int64_t n_docs, page_cap;
  uint8_t* codes;
  float* scales;
  int64_t n_pages;
};

// Eight consecutive elements of a row.
template <typename T>
__device__ __forceinline__ void load8(const T* p, float (&v)[8]) {
  if constexpr (sizeof(T) == 4) {
    const float4 lo = *reinterpret_cast<const float4*>(p), hi = *reinterpret_cast<const float4*>(p + 4);
    v[0] = lo.x, v[1] = lo.y, v[2] = lo.z, v[3] = lo.w;
    v[4] = hi.x, v[5] = hi.y, v[6] = hi.z, v[7] = hi.w;
  } else {
    const uint4 u = *reinterpret_cast<const uint4*>(p);
    const T* e = reinterpret_cast<const T*>(&u);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = static_cast<float>(e[i]);
  }
}

__device__ __forceinline__ bool finite(double v) { return fabs(v) <= 1.7e308; }

// e4m3 of a double, rounded once: to odd on the way to fp32 (24 bits, more than e4m3's 4 + 2), then
// to nearest. Larger magnitudes give 448.
__device__ __forceinline__ uint8_t e4m3_of_double(double t) {
  float f = __double2float_rz(t);
  if (static_cast<double>(f) != t) f = __uint_as_float(__float_as_uint(f) | 1u);
  return static_cast<uint8_t>(__nv_cvt_float_to_fp8(f, __NV_SATFINITE, __NV_E4M3));
}

constexpr int kWriteThreads = 128;

// One CTA a page. Pass one: each row's sum of squares and largest magnitude, then the page's
// largest normalised magnitude and its scale. Pass two: the codes. A group of lanes holds a row,
// eight elements a lane.
template <typename T>
__global__ void __launch_bounds__(kWriteThreads) page_write_kernel(const WriteArgs a) {
  __shared__ double row_factor[128];
  __shared__ double warp_max[kWriteThreads / 32];
  __shared__ int bad_any;
  const int page = 1 << a.page_shift;
  const int vecs = a.d >> 3;
  int group = 2;  // lanes of a row: a power of two, at most 32
  while (group < vecs) group <<= 1;
  const int sub = threadIdx.x % group, row0 = threadIdx.x / group, rows_step = kWriteThreads / group;
  const bool in_row = sub < vecs;
  const int64_t total_all = a.page_offsets[a.n_docs];
  const int64_t total = total_all < a.page_cap ? total_all : a.page_cap;
  double w[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) w[i] = 1.0;
  if (a.weight && in_row) {
    float wf[8];
    load8(static_cast<const T*>(a.weight) + sub * 8, wf);
#pragma unroll
    for (int i = 0; i < 8; ++i) w[i] = wf[i];
  }
  for (int64_t k = blockIdx.x; k < total; k += gridDim.x) {
    const int64_t doc = a.page_docs[k], id = a.page_ids[k];
    if (doc < 0 || doc >= a.n_docs || id < 0 || id >= a.n_pages) continue;
    const int64_t nth = k - a.page_offsets[doc];
    const int64_t t0 = a.token_offsets[doc];
    if (nth < 0 || nth > k || t0 < 0 || (!a.padded && t0 > a.n_rows)) continue;  // malformed tables
    const int64_t first = nth << a.page_shift;
    const int64_t left = a.token_offsets[doc + 1] - t0 - first;
    if (left < 1) continue;
    const int count = left < page ? static_cast<int>(left) : page;
    // rows [first, first + count) of the document; rows outside x read as zeros
    const int64_t doc_off = a.padded ? doc * a.stride_doc : t0 * a.stride_tok;
    const int64_t limit = a.padded ? a.n_rows - first : a.n_rows - t0 - first;
    const T* const x = static_cast<const T*>(a.x) + doc_off + first * a.stride_tok;
    const T* const res =
        a.residual ? static_cast<const T*>(a.residual) + doc_off + first * a.stride_tok : nullptr;
    auto load = [&](int r, double (&h)[8]) {
      float v[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) h[i] = 0.0;
      if (!in_row || r >= limit) return;
      load8(x + r * a.stride_tok + sub * 8, v);
#pragma unroll
      for (int i = 0; i < 8; ++i) h[i] = v[i];
      if (res) {
        load8(res + r * a.stride_tok + sub * 8, v);
#pragma unroll
        for (int i = 0; i < 8; ++i) h[i] += v[i];
      }
    };
    if (threadIdx.x == 0) bad_any = 0;
    __syncthreads();
    double best = 0.0;
    bool bad = false;
    for (int r0 = 0; r0 < page; r0 += rows_step) {
      const int r = r0 + row0;
      double h[8], s = 0.0, m = 0.0;
      const bool on = r < count;
      if (on) load(r, h);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        if (!on) h[i] = 0.0;
        s += h[i] * h[i];
        const double y = fabs(h[i] * w[i]);
        if (!(y <= m) && m == m) m = y;  // a NaN stays
      }
      for (int o = group >> 1; o > 0; o >>= 1) {
        s += __shfl_xor_sync(0xffffffffu, s, o);
        const double y = __shfl_xor_sync(0xffffffffu, m, o);
        if (!(y <= m) && m == m) m = y;
      }
      double f = 1.0;
      if (a.norm == TMS_NORM_L2) {
        const double n = sqrt(s);
        f = 1.0 / (n > a.eps ? n : static_cast<double>(a.eps));
      } else if (a.norm == TMS_NORM_RMS) {
        f = 1.0 / sqrt(s / a.d + a.eps);
      }
      if (on && sub == 0) row_factor[r] = f;
      const double y = m * f;
      bad |= on && !(finite(s) && finite(y));
      if (on && y > best) best = y;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const double y = __shfl_xor_sync(0xffffffffu, best, o);
      if (y > best) best = y;
    }
    if (lane_id() == 0) warp_max[threadIdx.x >> 5] = best;
    if (bad) bad_any = 1;
    __syncthreads();
    best = warp_max[0];
    for (int i = 1; i < kWriteThreads / 32; ++i)
      if (warp_max[i] > best) best = warp_max[i];
    const bool poison = bad_any != 0;
    const float scale = poison ? __int_as_float(0x7fffffff) : static_cast<float>(best / kE4m3Max);
    for (int r0 = 0; r0 < page; r0 += rows_step) {
      const int r = r0 + row0;
      const int src = r < count ? r : count - 1;
      if (r < page && in_row) {
        double h[8];
        load(src, h);
        const double f = row_factor[src];
        alignas(8) uint8_t c[8];
#pragma unroll
        for (int i = 0; i < 8; ++i)
          c[i] = poison ? 0x7f : scale > 0.f ? e4m3_of_double(h[i] * w[i] * f / scale) : 0;
        *reinterpret_cast<uint2*>(a.codes + ((id << a.page_shift) + r) * a.d + sub * 8) =
            *reinterpret_cast<const uint2*>(c);
      }
    }
    if (threadIdx.x == 0) a.scales[id] = scale;
    __syncthreads();
  }
}

// ------------------------------------------------------------------------------------------------
// reading tokens back
// ------------------------------------------------------------------------------------------------
struct ReadArgs {
  const uint8_t* codes;
  const float* scales;
  int64_t n_pages;
  int page_shift, d;
  const int64_t* slots;
  int64_t n_slots;
  void* out;
};

// out[t] = scale * code of slot t; a slot outside the pool gives a row of zeros. A thread takes
// eight elements. One multiplication in fp32, then one rounding to the output type.
template <typename T>
__global__ void page_read_kernel(const ReadArgs a) {
  const int vecs = a.d >> 3;
  const int64_t n = a.n_slots * vecs;
  for (int64_t e = blockIdx.x * static_cast<int64_t>(blockDim.x) + threadIdx.x; e < n;
       e += static_cast<int64_t>(gridDim.x) * blockDim.x) {
    const int64_t t = e / vecs;
    const int sub = static_cast<int>(e - t * vecs);
    const int64_t slot = a.slots[t];
    alignas(16) T v[8];
    if (slot >= 0 && (slot >> a.page_shift) < a.n_pages) {
      const uint2 c = *reinterpret_cast<const uint2*>(a.codes + slot * a.d + sub * 8);
      const float s = a.scales[slot >> a.page_shift];
      const uint8_t* b = reinterpret_cast<const uint8_t*>(&c);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const __half_raw h = __nv_cvt_fp8_to_halfraw(b[i], __NV_E4M3);
        v[i] = static_cast<T>(__half2float(__half(h)) * s);
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = static_cast<T>(0.f);
    }
    T* const o = static_cast<T*>(a.out) + t * a.d + sub * 8;
#pragma unroll
    for (int i = 0; i < static_cast<int>(sizeof(T)) / 2; ++i)
      reinterpret_cast<uint4*>(o)[i] = reinterpret_cast<const uint4*>(v)[i];
  }
}

int page_shift_of(int64_t page_size) {
  for (int s = 4; s <= 7; ++s)
    if (page_size == (int64_t(1) << s)) return s;
  return -1;
}

bool misaligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) != 0; }

}  // namespace
}  // namespace tms

using namespace tms;

extern "C" size_t tms_page_tables_workspace_size(int64_t n_docs) {
  if (n_docs <= 0) return 0;
  return static_cast<size_t>((n_docs + kTileDocs - 1) / kTileDocs) * 16;
}

extern "C" int tms_page_tables(const int64_t* lengths, int64_t n_lengths, const int64_t* doc_ids,
                               int64_t n_docs, const int64_t* src_offsets, const int32_t* pages,
                               int64_t n_src_pages, int64_t page_size, int64_t* page_offsets,
                               int64_t* token_offsets, int32_t* page_ids, int32_t* page_docs,
                               int64_t page_capacity, int64_t* slots, int64_t token_capacity,
                               void* workspace, size_t workspace_bytes, void* stream) {
  NvtxRange nvtx_range("tms_page_tables");
  const int shift = page_shift_of(page_size);
  if (shift < 0) return TMS_ERR_UNSUPPORTED;
  if (n_lengths < 0 || n_docs < 0 || n_src_pages < 0 || page_capacity < 0 || token_capacity < 0)
    return TMS_ERR_INVALID;
  if (!doc_ids && n_docs > n_lengths) return TMS_ERR_INVALID;
  if (n_docs >= (int64_t(1) << 31) || page_capacity >= (int64_t(1) << 31)) return TMS_ERR_UNSUPPORTED;
  if (!page_offsets || !token_offsets || (n_lengths > 0 && !lengths) || (n_src_pages > 0 && !pages) ||
      (page_capacity > 0 && (!page_ids || !page_docs)))
    return TMS_ERR_INVALID;
  if (n_docs > 0 && (!workspace || workspace_bytes < tms_page_tables_workspace_size(n_docs)))
    return TMS_ERR_WORKSPACE;
  if (reinterpret_cast<uintptr_t>(workspace) & 7) return TMS_ERR_INVALID;
  int status = TMS_OK;
  const DeviceInfo* dev = current_device_info(&status);
  if (!dev) return status;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const TableArgs a{lengths, n_lengths, doc_ids, n_docs, src_offsets, pages, n_src_pages, shift, page_offsets,
                    token_offsets, page_ids, page_docs, page_capacity, slots, slots ? token_capacity : 0,
                    static_cast<int64_t*>(workspace)};
  const int64_t tiles = n_docs > 0 ? (n_docs + kTileDocs - 1) / kTileDocs : 1;
  if (tiles > 1) table_sums_kernel<<<static_cast<unsigned>(tiles), kTableThreads, 0, st>>>(a);
  table_offsets_kernel<<<static_cast<unsigned>(tiles), kTableThreads, 0, st>>>(a);
  int64_t blocks = (page_capacity + kTableThreads - 1) / kTableThreads;
  const int64_t most = static_cast<int64_t>(dev->num_sms) * 8;
  blocks = blocks < 1 ? 1 : blocks > most ? most : blocks;
  table_fill_kernel<<<static_cast<unsigned>(blocks), kTableThreads, 0, st>>>(a);
  return cuda_status(cudaGetLastError());
}

extern "C" int tms_page_write(const void* x, int dtype, int64_t n_rows, int64_t stride_doc,
                              int64_t stride_token, int padded, const void* residual,
                              const void* weight, int norm, float eps, int64_t d,
                              int64_t page_size, const int64_t* page_offsets,
                              const int64_t* token_offsets, const int32_t* page_ids,
                              const int32_t* page_docs, int64_t n_docs, int64_t page_capacity,
                              void* codes, float* scales, int64_t n_pages, void* stream) {
  NvtxRange nvtx_range("tms_page_write");
  if (dtype != TMS_F16 && dtype != TMS_BF16 && dtype != TMS_F32) return TMS_ERR_INVALID;
  if (norm != TMS_NORM_NONE && norm != TMS_NORM_L2 && norm != TMS_NORM_RMS) return TMS_ERR_INVALID;
  if (weight && norm != TMS_NORM_RMS) return TMS_ERR_INVALID;
  if (!(eps >= 0.f)) return TMS_ERR_INVALID;
  if (n_rows < 0 || d <= 0 || n_docs < 0 || page_capacity < 0 || n_pages < 0) return TMS_ERR_INVALID;
  const int shift = page_shift_of(page_size);
  if (shift < 0 || d % 16 != 0 || d > TMS_PAGED_MAX_D) return TMS_ERR_UNSUPPORTED;
  if (n_docs == 0 || page_capacity == 0 || n_pages == 0) return TMS_OK;
  const int64_t esize = dtype == TMS_F32 ? 4 : 2;
  if ((stride_doc * esize) % 16 || (stride_token * esize) % 16) return TMS_ERR_INVALID;
  if (!page_offsets || !token_offsets || !page_ids || !page_docs || !codes || !scales || (n_rows > 0 && !x))
    return TMS_ERR_INVALID;
  if (misaligned16(x) || misaligned16(residual) || misaligned16(weight) || misaligned16(codes))
    return TMS_ERR_INVALID;
  int status = TMS_OK;
  const DeviceInfo* dev = current_device_info(&status);
  if (!dev) return status;
  const WriteArgs a{x, residual, weight, stride_doc, stride_token, n_rows, padded, norm, eps,
                    static_cast<int>(d), shift, page_offsets, token_offsets, page_ids, page_docs, n_docs,
                    page_capacity, static_cast<uint8_t*>(codes), scales, n_pages};
  const int64_t most = static_cast<int64_t>(dev->num_sms) * 12;
  const unsigned blocks = static_cast<unsigned>(page_capacity < most ? page_capacity : most);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (dtype == TMS_F16) page_write_kernel<__half><<<blocks, kWriteThreads, 0, st>>>(a);
  else if (dtype == TMS_BF16) page_write_kernel<__nv_bfloat16><<<blocks, kWriteThreads, 0, st>>>(a);
  else page_write_kernel<float><<<blocks, kWriteThreads, 0, st>>>(a);
  return cuda_status(cudaGetLastError());
}

extern "C" int tms_page_read(const void* codes, const float* scales, int64_t n_pages,
                             int64_t page_size, int64_t d, const int64_t* slots, int64_t n_slots,
                             void* out, int out_dtype, void* stream) {
  NvtxRange nvtx_range("tms_page_read");
  if (out_dtype != TMS_F16 && out_dtype != TMS_BF16 && out_dtype != TMS_F32) return TMS_ERR_INVALID;
  if (n_pages < 0 || d <= 0 || n_slots < 0) return TMS_ERR_INVALID;
  const int shift = page_shift_of(page_size);
  if (shift < 0 || d % 16 != 0 || d > TMS_PAGED_MAX_D) return TMS_ERR_UNSUPPORTED;
  if (n_slots == 0) return TMS_OK;
  if (!slots || !out || (n_pages > 0 && (!codes || !scales))) return TMS_ERR_INVALID;
  if (misaligned16(codes) || misaligned16(out)) return TMS_ERR_INVALID;
  int status = TMS_OK;
  const DeviceInfo* dev = current_device_info(&status);
  if (!dev) return status;
  const ReadArgs a{static_cast<const uint8_t*>(codes), scales, n_pages, shift, static_cast<int>(d), slots,
                   n_slots, out};
  int64_t blocks = (n_slots * (d / 8) + 255) / 256;
  const int64_t most = static_cast<int64_t>(dev->num_sms) * 16;
  if (blocks > most) blocks = most;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (out_dtype == TMS_F16) page_read_kernel<__half><<<static_cast<unsigned>(blocks), 256, 0, st>>>(a);
  else if (out_dtype == TMS_BF16) page_read_kernel<__nv_bfloat16><<<static_cast<unsigned>(blocks), 256, 0, st>>>(a);
  else page_read_kernel<float><<<static_cast<unsigned>(blocks), 256, 0, st>>>(a);
  return cuda_status(cudaGetLastError());
}
