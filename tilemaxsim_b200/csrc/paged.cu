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
#include <type_traits>

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
  int64_t* tile_sums;      // workspace: (tiles, 2) pages and tokens of each tile of documents,
  int32_t* owners;         // and the document that owns each 32nd table entry
};

constexpr int kTableThreads = 256;
constexpr int kTileDocs = 1024;  // documents of one tile (four for each thread)
constexpr int kFewDocs = 2048;   // documents whose offsets a CTA works out for itself

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
      // the entries 32 b of this document
      const int64_t end = bp + p + ((len + round) >> a.page_shift), most = a.page_cap;
      for (int64_t b = (bp + p + 31) >> 5; (b << 5) < (end < most ? end : most); ++b) a.owners[b] = static_cast<int32_t>(i);
    }
    bp += tp;
    bt += tt;
  }
  if (threadIdx.x == 0 && i0 + kTileDocs >= a.n_docs) {
    a.page_offsets[a.n_docs] = bp;
    a.token_offsets[a.n_docs] = bt;
  }
}

// The last document d in [lo, hi) with page_offsets[d] <= k, which page_offsets[lo] is.
__device__ __forceinline__ int64_t owner_of(const int64_t* page_offsets, int64_t lo, int64_t hi, int64_t k) {
  while (hi - lo > 1) {
    const int64_t mid = (lo + hi) >> 1;
    if (page_offsets[mid] <= k) lo = mid;
    else hi = mid;
  }
  return lo;
}

// 400,000 documents (72.8M slots, 582 MB) take 126 us here and 12 us for their offsets; a plain fill
// of the slots takes 81 us. Issue slots are 58% busy; the rest is waits for the entries' loads and for
// shuffles. A slot at a time with its own bounds checks took 219 us.
//
// Page ids, owners and slots of the 32 table entries from k0 on, by one warp: a lane for each entry
// (`doc` owns it, where it lies below the total), then the entries' slots one after the other. The
// entries' tokens follow one another, so one base and 32-bit distances from it place them.
__device__ __forceinline__ void fill_entries(const TableArgs& a, int64_t k0, int64_t total, int64_t doc,
                                             int64_t doc_page, int64_t doc_token, int64_t doc_end) {
  constexpr uint32_t kAllWarp = 0xffffffffu;
  const int lane = threadIdx.x & 31;
  const int page = 1 << a.page_shift;
  const int64_t k = k0 + lane;
  const bool used = k < total && k < a.page_cap;
  int64_t tok = 0;
  int id = -1, count = 0;
  if (used) {
    const int64_t nth = k - doc_page;
    int64_t src = k;
    if (a.src_offsets) src = __ldg(a.src_offsets + (a.doc_ids ? __ldg(a.doc_ids + doc) : doc)) + nth;
    if (src >= 0 && src < a.n_src) id = __ldg(a.pages + src);
    tok = doc_token + (nth << a.page_shift);
    count = static_cast<int>(doc_end - tok < page ? doc_end - tok : page);
  }
  if (k < a.page_cap) {
    a.page_ids[k] = id;
    a.page_docs[k] = used ? static_cast<int32_t>(doc) : -1;
  }
  if (!a.slots) return;
  const int64_t base = __shfl_sync(kAllWarp, tok, 0);
  const int at = static_cast<int>(tok - base);
  int64_t* const to = a.slots + base;
  const int64_t room = a.token_cap - base;
  const int entries = __popc(__ballot_sync(kAllWarp, used));
  const int last_at = __shfl_sync(kAllWarp, at + count, entries > 0 ? entries - 1 : 0);
  const bool fits = last_at <= room;
  const int place = at << 8 | count;  // at most 4,064 and 128
  if (fits && !__any_sync(kAllWarp, used && id < 0)) {
    // every slot is there: 32 of them an instruction, of one page or of two
    const int each = page < 32 ? 32 >> a.page_shift : 1, j = page < 32 ? lane & (page - 1) : lane;
    const int sub = page < 32 ? lane >> a.page_shift : 0;
    for (int from = 0; from < page; from += page < 32 ? page : 32)
#pragma unroll 8
      for (int l = 0; l < 32; l += each) {
        const int w = __shfl_sync(kAllWarp, place, l + sub), p = __shfl_sync(kAllWarp, id, l + sub);
        if (from + j < (w & 0xff)) to[(w >> 8) + from + j] = (static_cast<int64_t>(p) << a.page_shift) + from + j;
      }
    return;
  }
  for (int l = 0; l < entries; ++l) {
    const int w = __shfl_sync(kAllWarp, place, l), p = __shfl_sync(kAllWarp, id, l);
    for (int j = lane; j < (w & 0xff); j += 32)
      if ((w >> 8) + j < room) to[(w >> 8) + j] = p < 0 ? -1 : (static_cast<int64_t>(p) << a.page_shift) + j;
  }
}

// Slots that no entry covers, from token `rest` on.
__device__ __forceinline__ void fill_rest(const TableArgs& a, int64_t rest) {
  if (!a.slots) return;
  const int64_t step = static_cast<int64_t>(gridDim.x) * blockDim.x;
  for (int64_t t = rest + static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x; t < a.token_cap; t += step)
    a.slots[t] = -1;
}

// A warp takes 32 consecutive table entries at a time. Its first entry's owner is in the workspace,
// the others' are among the next documents, whose offsets a lane each loads at once.
__global__ void __launch_bounds__(kTableThreads) table_fill_kernel(const TableArgs a) {
  constexpr uint32_t kAllWarp = 0xffffffffu;
  const int lane = threadIdx.x & 31;
  const int64_t warps = static_cast<int64_t>(gridDim.x) * (kTableThreads / 32);
  const int64_t warp = static_cast<int64_t>(blockIdx.x) * (kTableThreads / 32) + (threadIdx.x >> 5);
  const int64_t total = a.page_offsets[a.n_docs];
  for (int64_t k0 = warp * 32; k0 < a.page_cap; k0 += warps * 32) {
    const int64_t k = k0 + lane;
    int64_t doc = 0, doc_page = 0, doc_token = 0, doc_end = 0;
    if (k0 < total) {
      const int64_t lo = a.owners[k0 >> 5];
      const int64_t next = lo + 1 + lane;
      const int64_t starts = a.page_offsets[next < a.n_docs ? next : a.n_docs];  // where document `next` starts
      int d = 0;  // documents after lo that start at or before k
#pragma unroll
      for (int w = 16; w > 0; w >>= 1)
        if (__shfl_sync(kAllWarp, starts, d + w - 1) <= k) d += w;
      const int64_t last = __shfl_sync(kAllWarp, starts, 31);  // all lanes take part, before any is left out
      const bool beyond = d == 31 && last <= k;
      doc = lo + d;
      if (beyond && k < total) doc = owner_of(a.page_offsets, lo, a.n_docs, k);  // many empty documents
      if (k < total) {
        doc_page = a.page_offsets[doc];
        doc_token = a.token_offsets[doc];
        doc_end = a.token_offsets[doc + 1];
      }
    }
    fill_entries(a, k0, total, doc, doc_page, doc_token, doc_end);
  }
  int64_t rest = a.token_offsets[a.n_docs];  // tokens from here on have no table entry
  if (total > a.page_cap) {
    const int64_t doc = owner_of(a.page_offsets, 0, a.n_docs, a.page_cap);
    rest = a.token_offsets[doc] + ((a.page_cap - a.page_offsets[doc]) << a.page_shift);
  }
  fill_rest(a, rest);
}

// Few documents, in one launch: every CTA works out all offsets in shared memory (eight documents
// a thread) and fills its part of the tables; the first one also writes the offsets.
__global__ void __launch_bounds__(kTableThreads) table_few_kernel(const TableArgs a) {
  __shared__ int64_t pages[kFewDocs + 1], tokens[kFewDocs + 1];
  __shared__ int64_t sh[kTableThreads / 32][2];
  constexpr int kEach = kFewDocs / kTableThreads;
  const int lane = threadIdx.x & 31;
  const int n = static_cast<int>(a.n_docs);
  const int64_t round = (int64_t(1) << a.page_shift) - 1;
  const int each = (n + kTableThreads - 1) / kTableThreads;  // documents of a thread
  const int i0 = threadIdx.x * each;
  int64_t len[kEach], p = 0, t = 0, total, total_tokens;
#pragma unroll
  for (int j = 0; j < kEach; ++j) {
    len[j] = j < each && i0 + j < n ? table_length(a, i0 + j) : 0;
    p += (len[j] + round) >> a.page_shift;
    t += len[j];
  }
  block_scan2(p, t, &total, &total_tokens, sh);
#pragma unroll
  for (int j = 0; j < kEach; ++j) {
    if (j >= each || i0 + j >= n) break;
    pages[i0 + j] = p;
    tokens[i0 + j] = t;
    p += (len[j] + round) >> a.page_shift;
    t += len[j];
  }
  if (threadIdx.x == 0) {
    pages[n] = total;
    tokens[n] = total_tokens;
  }
  __syncthreads();
  if (blockIdx.x == 0)
    for (int i = threadIdx.x; i <= n; i += kTableThreads) {
      a.page_offsets[i] = pages[i];
      a.token_offsets[i] = tokens[i];
    }
  const int64_t warps = static_cast<int64_t>(gridDim.x) * (kTableThreads / 32);
  const int64_t warp = static_cast<int64_t>(blockIdx.x) * (kTableThreads / 32) + (threadIdx.x >> 5);
  for (int64_t k0 = warp * 32; k0 < a.page_cap; k0 += warps * 32) {
    const int64_t k = k0 + lane;
    int64_t doc = 0, doc_page = 0, doc_token = 0, doc_end = 0;
    if (k < total) {
      doc = owner_of(pages, 0, n, k);
      doc_page = pages[doc];
      doc_token = tokens[doc];
      doc_end = tokens[doc + 1];
    }
    fill_entries(a, k0, total, doc, doc_page, doc_token, doc_end);
  }
  int64_t rest = total_tokens;
  if (total > a.page_cap) {
    const int64_t doc = owner_of(pages, 0, n, a.page_cap);
    rest = tokens[doc] + ((a.page_cap - pages[doc]) << a.page_shift);
  }
  fill_rest(a, rest);
}

// ------------------------------------------------------------------------------------------------
// writing tokens into pages
// ------------------------------------------------------------------------------------------------
constexpr float kE4m3Max = 448.f;

// Four fp32 values as e4m3, to nearest, ties to even; larger magnitudes give 448, a NaN 0x7f.
__device__ __forceinline__ uint32_t e4m3x4(float2 lo, float2 hi) {
  uint32_t r;
  asm("{\n\t.reg .b16 p, q;\n\t"
      "cvt.rn.satfinite.e4m3x2.f32 p, %2, %1;\n\t"
      "cvt.rn.satfinite.e4m3x2.f32 q, %4, %3;\n\t"
      "mov.b32 %0, {p, q};\n\t}\n"
      : "=r"(r)
      : "f"(lo.x), "f"(lo.y), "f"(hi.x), "f"(hi.y));
  return r;
}

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

__device__ __forceinline__ bool finite(double v) { return fabs(v) <= 1.7e308; }

// e4m3 of a double, rounded once: to odd on the way to fp32 (24 bits, more than e4m3's 4 + 2), then
// to nearest. Larger magnitudes give 448.
__device__ __forceinline__ uint8_t e4m3_of_double(double t) {
  float f = __double2float_rz(t);
  if (static_cast<double>(f) != t) f = __uint_as_float(__float_as_uint(f) | 1u);
  return static_cast<uint8_t>(e4m3x4(make_float2(f, 0.f), make_float2(0.f, 0.f)) & 0xffu);
}

// Eight consecutive elements of a row, as they are stored.
template <typename T>
struct Eight {
  uint4 v[sizeof(T) / 2];
  __device__ __forceinline__ void load(const T* p) {
#pragma unroll
    for (int i = 0; i < static_cast<int>(sizeof(T)) / 2; ++i) v[i] = __ldg(reinterpret_cast<const uint4*>(p) + i);
  }
  __device__ __forceinline__ void take(const T* p) {  // from shared memory
#pragma unroll
    for (int i = 0; i < static_cast<int>(sizeof(T)) / 2; ++i) v[i] = reinterpret_cast<const uint4*>(p)[i];
  }
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int i = 0; i < static_cast<int>(sizeof(T)) / 2; ++i) v[i] = make_uint4(0, 0, 0, 0);
  }
  // The largest magnitude of 16-bit values, two at a time: their bits without the sign are ordered
  // as they are (a NaN's above infinity's).
  __device__ __forceinline__ float top() const {
    const uint32_t m = __vmaxu2(__vmaxu2(v[0].x & 0x7fff7fffu, v[0].y & 0x7fff7fffu),
                                __vmaxu2(v[0].z & 0x7fff7fffu, v[0].w & 0x7fff7fffu));
    const uint32_t w = max(m & 0xffffu, m >> 16);
    if constexpr (std::is_same<T, __nv_bfloat16>::value) return __uint_as_float(w << 16);
    else return __half2float(__ushort_as_half(static_cast<unsigned short>(w)));
  }
  __device__ __forceinline__ float at(int i) const {
    const uint4& q = v[sizeof(T) == 4 ? i >> 2 : 0];
    const int j = sizeof(T) == 4 ? i & 3 : i >> 1;
    const uint32_t w = j == 0 ? q.x : j == 1 ? q.y : j == 2 ? q.z : q.w;
    if constexpr (sizeof(T) == 4) return __uint_as_float(w);
    else if constexpr (std::is_same<T, __nv_bfloat16>::value)
      return __uint_as_float(i & 1 ? w & 0xffff0000u : w << 16);
    else
      return __half2float(__ushort_as_half(static_cast<unsigned short>(i & 1 ? w >> 16 : w)));
  }
};

// One page at a time a CTA of one, two or four warps, the next page on its way into shared memory (cp.async)
// meanwhile; a group of 2 to 32 lanes takes a row, eight elements a lane. The input is read from
// memory once and the codes are written once. Pages of more than kStageBytes of input are read twice
// instead, the second time from the caches (3.64M tokens of 128 bf16 values in pages of 128: 825 us).
//
// The scale is the fp32 rounding, and every code the e4m3 rounding, of what 64 bits give, at little
// more than fp32's cost. fp32 gives every row's factor to 2^-21. Only rows whose largest magnitude
// comes within 2^-19 of the page's can set the scale: they (one, as a rule) are summed again in
// fp64, which brings their factors to 2^-41, and have fp64's own root where that leaves the scale
// open. A code is that of t = h * w * factor / scale: where t * (1 - 2^-20) and t * (1 + 2^-20)
// round to the same one, fp32 is sure of it; the others (about one of 4,000 groups of eight
// elements) are done again in fp64, with its root and a division: whole numbers of a rational length
// have exact ties, which a factor 2^-42 off would break to one side. Where nothing is normalised,
// added or weighted, ties are common and exact, and one fp32 division with its remainder decides them
// (5,000 documents: 164 us; fp64's took a quarter more). Pages that hold a magnitude or a sum of
// squares outside [1e-30, 1e30], zeros apart, go through fp64 altogether; NaN and infinities are found
// there.
//
// 20,000 documents (3.6M tokens, 128 bf16 values, unit length) take 454 us, 3.1 TB/s. Neither memory nor
// issue slots (62% busy) are full: with 21 warps an SM, a warp waits for its CTA's barriers, for fixed
// latencies and for shared memory, in about equal parts. Fewer instructions help all the same: with the
// width as a constant of the kernel where it is 128 (D) that took a sixth less, and 1,600 pages with a
// residual 14.9 us against 17; the page size as a constant too would give 2% more. The look whether the
// scale is open takes 3 us (20 of 1,050 at d = 256). Before, rows held in registers took 770 us (few warps
// fit), all sums in fp64 600-820, sixteen elements a lane 546, fp64 roots for all rows that can set the
// scale 830.
__device__ __forceinline__ double max_keep_nan(double x, double y) { return y <= x || x != x ? x : y; }
__device__ __forceinline__ bool usual(float v) { return v >= 1e-30f && v <= 1e30f; }

// Threads of a CTA: 32 where a page's input is 4 KB at most, 64 up to 8 KB, else 128: as many CTAs as
// shared memory has stages for then have warps enough, and few warps a page wait for one another
// little. 3.64M tokens of bf16, before the look at open scales: d = 64 288 us with 32 threads, 342 with 64; pages of 16 468 and 572;
// pages of 32 515 with 32, 452 with 64, 548 with 128; pages of 64 538 with 64, 456 with 128; d = 256
// 1,232 and 1,030. 1,024 documents with a residual (16 KB a page): 52 us with 64, 45 with 128.
constexpr int write_threads(int input) { return input <= 4096 ? 32 : input <= 8192 ? 64 : 128; }
constexpr int kStaticBytes = 2048;       // a CTA's other shared memory, at most
constexpr int kStageBytes = 24 * 1024;  // most input of a page (x and residual) that is staged

// h / scale to fp32, moved off a midpoint between two codes to the side of the true quotient, where
// that is not the midpoint itself. Codes are 2^-3 of the leading power of two apart, 2^-9 below 2^-6:
// there 2^-6 is added to look, which has the same spacing. A midpoint ends in 0x80000.
__device__ __forceinline__ float off_midpoint(float h, float scale) {
  const float q = __fdiv_rn(h, scale), m = fabsf(q);
  const float level = m < 0.015625f ? m + 0.015625f : m;
  if ((__float_as_uint(level) & 0xfffffu) != 0x80000u) return q;
  if (m < 0.015625f && level - 0.015625f != m) return q;  // beside a midpoint, lost in the sum
  const float rest = fmaf(-q, scale, h);  // exact
  if (rest == 0.f) return q;
  return __uint_as_float(__float_as_uint(q) + ((rest > 0.f) == (q > 0.f) ? 1u : 0xffffffffu));
}

__device__ __forceinline__ double scale_of(double y) { return y * (1.0 / kE4m3Max); }
// Whether scale_of(y), y off by 2^-41 at most, rounds to fp32 for certain: its 29 bits below fp32's are not
// within 2^13 of the middle, and fp32 has it as a normal number.
__device__ __forceinline__ bool sure_scale(double y) {
  const double s = scale_of(y);
  const int below = __double2loint(s) & 0x1fffffff;
  return abs(below - 0x10000000) > 0x2000 && s > 1.2e-38;
}

struct Entry {    // where a table entry's rows come from
  int64_t at;     // element offset of its first row
  int64_t id;
  int limit;      // rows of x from there on, up to a page
  int count;      // 0: the entry is skipped
};

template <typename T, bool SUM, bool WEIGHT, bool STAGED, int D>
struct PageRows {
  const WriteArgs& a;
  const T* stage;  // x's rows, then the residual's
  int sub, group, d;
  bool in_row;
  // Eight elements of row src (of the page) of x, and of the residual.
  __device__ __forceinline__ void load(const Entry& e, int src, Eight<T>& x, Eight<T>& r) const {
    if (!in_row || (!STAGED && src >= e.limit)) {
      x.zero();
      if constexpr (SUM) r.zero();
      return;
    }
    if constexpr (STAGED) {
      const T* const p = stage + src * d + sub * 8;
      x.take(p);
      if constexpr (SUM) r.take(p + (d << a.page_shift));
    } else {
      const int64_t at = e.at + src * a.stride_tok + sub * 8;
      x.load(static_cast<const T*>(a.x) + at);
      if constexpr (SUM) r.load(static_cast<const T*>(a.residual) + at);
    }
  }
};

// A row in fp64, by the lanes that hold it: its eight elements a lane (times the weights), its
// largest magnitude, and what both are to be divided by: fp64's own root, where `full`, or the inverse of a
// factor that a Newton step, which squares fp32's 2^-21, gives (`factor`; cheaper, but off a tie).
struct ExactRow {
  double h[8], factor, norm, top;
  bool bad;
};
template <typename T, bool SUM, bool WEIGHT, bool STAGED, int D>
__device__ __forceinline__ void exact_row(const PageRows<T, SUM, WEIGHT, STAGED, D>& rows, const Entry& e, int src,
                                          float near, bool full, ExactRow& o) {
  const WriteArgs& a = rows.a;
  Eight<T> x, r;
  rows.load(e, src, x, r);
  double s = 0.0;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    o.h[j] = x.at(j);
    if constexpr (SUM) o.h[j] += static_cast<double>(r.at(j));
    s = fma(o.h[j], o.h[j], s);
  }
  if constexpr (WEIGHT) {
    Eight<T> w;
    w.zero();
    if (rows.in_row) w.load(static_cast<const T*>(a.weight) + rows.sub * 8);
#pragma unroll
    for (int j = 0; j < 8; ++j) o.h[j] *= static_cast<double>(w.at(j));
  }
  for (int m = rows.group >> 1; m > 0; m >>= 1) s += __shfl_xor_sync(0xffffffffu, s, m);
  o.top = 0.0;
  if (SUM || (WEIGHT && sizeof(T) == 4) || full) {
#pragma unroll
    for (int j = 0; j < 8; ++j) o.top = max_keep_nan(o.top, fabs(o.h[j]));
    for (int m = rows.group >> 1; m > 0; m >>= 1) o.top = max_keep_nan(o.top, __shfl_xor_sync(0xffffffffu, o.top, m));
  } else {  // the magnitudes are exact in fp32
    float top = 0.f;
#pragma unroll
    for (int j = 0; j < 8; ++j) top = fmaxf(top, fabsf(static_cast<float>(o.h[j])));
    for (int m = rows.group >> 1; m > 0; m >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, m));
    o.top = top;
  }
  o.factor = o.norm = 1.0;
  o.bad = false;
  if (!full) {
    const double f = near, v = a.norm == TMS_NORM_RMS ? s * (1.0 / rows.d) + a.eps : s;
    if (a.norm != TMS_NORM_NONE) o.factor = f + 0.5 * f * (1.0 - v * f * f);
    return;
  }
  if (a.norm == TMS_NORM_L2) {
    const double n = sqrt(s);
    o.norm = n > a.eps ? n : static_cast<double>(a.eps);
  } else if (a.norm == TMS_NORM_RMS) {
    o.norm = sqrt(s / rows.d + a.eps);
  }
  o.bad = !(finite(s) && finite(o.top / o.norm));
}

template <typename T, bool SUM, bool WEIGHT, bool STAGED, int D, int kWriteThreads>
__global__ void __launch_bounds__(kWriteThreads, 768 / kWriteThreads)
page_write_kernel(const WriteArgs a, int lanes) {
  const int d = D > 0 ? D : a.d, group = D > 0 ? D / 8 : lanes;
  constexpr uint32_t kAllWarp = 0xffffffffu;
  constexpr int kWarps = kWriteThreads / 32;
  extern __shared__ __align__(16) uint8_t stage_bytes[];
  __shared__ Entry entries[3];
  __shared__ float row_factor[128], row_top[128];
  __shared__ float warp_top[kWarps];
  __shared__ double warp_best[kWarps];
  __shared__ int warp_odd[kWarps], warp_bad[kWarps];
  const int page = 1 << a.page_shift;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int sub = threadIdx.x & (group - 1), step = kWriteThreads / group, row0 = threadIdx.x / group;
  const bool in_row = sub < (d >> 3);
  T* const stages = reinterpret_cast<T*>(stage_bytes);
  const int stage_elems = (d << a.page_shift) * (SUM ? 2 : 1);
  Eight<T> wt;
  wt.zero();
  bool odd_weight = false;
  if (WEIGHT && in_row) {
    wt.load(static_cast<const T*>(a.weight) + sub * 8);
#pragma unroll
    for (int j = 0; j < 8; ++j) odd_weight |= !(fabsf(wt.at(j)) <= 1e30f);
  }
  const float per_d = 1.f / d;
  // After the sums below a lane has those of `held` of its four rows, from row number `mine` on.
  const int held = group == 2 ? 2 : 1;
  const int mine = group == 2 ? (sub & 1) * 2 : (sub & 1) * 2 + (sub >> 1 & 1);

  const int64_t total_all = a.page_offsets[a.n_docs];
  const int64_t total = total_all < a.page_cap ? total_all : a.page_cap;
  auto find = [&](int64_t k) {
    Entry e = {0, 0, 0, 0};
    if (k >= total) return e;
    const int64_t doc = __ldg(a.page_docs + k);
    e.id = __ldg(a.page_ids + k);
    if (doc < 0 || doc >= a.n_docs || e.id < 0 || e.id >= a.n_pages) return e;
    const int64_t nth = k - __ldg(a.page_offsets + doc);
    const int64_t t0 = __ldg(a.token_offsets + doc), t1 = __ldg(a.token_offsets + doc + 1);
    if (nth < 0 || nth > k || t0 < 0 || (!a.padded && t0 > a.n_rows)) return e;  // malformed tables
    const int64_t first = nth << a.page_shift;
    const int64_t left = t1 - t0 - first;
    const int64_t limit = a.padded ? a.n_rows - first : a.n_rows - t0 - first;
    e.at = (a.padded ? doc * a.stride_doc : t0 * a.stride_tok) + first * a.stride_tok;
    e.limit = limit < 0 ? 0 : limit < page ? static_cast<int>(limit) : page;
    e.count = left < 1 ? 0 : left < page ? static_cast<int>(left) : page;
    return e;
  };
  // This thread's part of every row it takes: the same lanes copy a row that read it.
  const int64_t row_jump = step * a.stride_tok, my_from = row0 * a.stride_tok + sub * 8;
  const uint32_t my_to = smem_u32(stage_bytes) + (row0 * d + sub * 8) * static_cast<uint32_t>(sizeof(T));
  const uint32_t to_jump = step * d * static_cast<uint32_t>(sizeof(T));
  auto fetch = [&](const Entry& e, int which) {  // the entry's rows into a stage
    const int count = e.count < e.limit ? e.count : e.limit;
    uint32_t to = my_to + which * stage_elems * static_cast<uint32_t>(sizeof(T));
    const T* from = static_cast<const T*>(a.x) + e.at + my_from;
    const T* from_res = static_cast<const T*>(a.residual) + e.at + my_from;
    const uint32_t res = (d << a.page_shift) * static_cast<uint32_t>(sizeof(T));
    if (!in_row) return;
    for (int row = row0 + (count - row0 + step - 1) / step * step; row < e.count; row += step) {  // rows x does not have
      if (row < count) continue;
      T* const p = stages + which * stage_elems + row * d + sub * 8;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        p[i] = T(0.f);
        if constexpr (SUM) p[(d << a.page_shift) + i] = T(0.f);
      }
    }
    for (int row = row0; row < count; row += step, to += to_jump, from += row_jump) {
#pragma unroll
      for (int i = 0; i < static_cast<int>(sizeof(T)) / 2; ++i) cp_async16(to + 16 * i, from + i * (16 / sizeof(T)));
      if constexpr (SUM) {
#pragma unroll
        for (int i = 0; i < static_cast<int>(sizeof(T)) / 2; ++i)
          cp_async16(to + res + 16 * i, from_res + i * (16 / sizeof(T)));
        from_res += row_jump;
      }
    }
  };

  if (threadIdx.x == 0) entries[0] = find(blockIdx.x);
  __syncthreads();
  if constexpr (STAGED) fetch(entries[0], 0);
  int now = 0, at = 0;  // the stage, and the place among the entries, of this page
  for (int64_t k = blockIdx.x; k < total; k += gridDim.x, now ^= 1, at = at == 2 ? 0 : at + 1) {
    const int after = at == 2 ? 0 : at + 1;
    if (threadIdx.x == 0) entries[after] = find(k + gridDim.x);
    if constexpr (STAGED) cp_async_wait_all();
    __syncthreads();  // this page's rows are there, the next entry is known, the page before is done
    if constexpr (STAGED) fetch(entries[after], now ^ 1);
    const Entry e = entries[at];
    if (e.count == 0) continue;  // the same for the whole CTA
    const PageRows<T, SUM, WEIGHT, STAGED, D> rows{a, stages + now * stage_elems, sub, group, d, in_row};

    float top = 0.f;
    bool odd = odd_weight;
    for (int r0 = row0, b = 0; b < page; r0 += 4 * step, b += 4 * step) {  // the same turns for all lanes
      float sums[4], tops[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        sums[i] = tops[i] = 0.f;
        const int row = r0 + i * step;
        if (row >= e.count) continue;
        Eight<T> x, r;
        rows.load(e, row, x, r);
        uint64_t s2 = 0;
#pragma unroll
        for (int j = 0; j < 8; j += 2) {
          float h0 = x.at(j), h1 = x.at(j + 1);
          if constexpr (SUM) h0 += r.at(j), h1 += r.at(j + 1);
          const uint64_t h2 = f2_pack(h0, h1);
          s2 = f2_fma(h2, h2, s2);
          if constexpr (SUM || WEIGHT || sizeof(T) == 4) {
            if constexpr (WEIGHT) h0 *= wt.at(j), h1 *= wt.at(j + 1);
            tops[i] = fmaxf(tops[i], fmaxf(fabsf(h0), fabsf(h1)));  // a NaN shows in the sum
          }
        }
        const float2 two = f2_unpack(s2);
        sums[i] = two.x + two.y;
        if constexpr (!(SUM || WEIGHT || sizeof(T) == 4)) tops[i] = x.top();
      }
      // Over the lanes of a group: while a lane has more than one row, it hands half of them to its
      // partner and takes the other half's partial results; then plain exchanges.
      {
        const bool upper = sub & 1;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const float s = __shfl_xor_sync(kAllWarp, upper ? sums[i] : sums[i + 2], 1);
          const float t = __shfl_xor_sync(kAllWarp, upper ? tops[i] : tops[i + 2], 1);
          sums[i] = (upper ? sums[i + 2] : sums[i]) + s;
          tops[i] = fmaxf(upper ? tops[i + 2] : tops[i], t);
        }
      }
      if (group > 2) {
        const bool upper = sub & 2;
        const float s = __shfl_xor_sync(kAllWarp, upper ? sums[0] : sums[1], 2);
        const float t = __shfl_xor_sync(kAllWarp, upper ? tops[0] : tops[1], 2);
        sums[0] = (upper ? sums[1] : sums[0]) + s;
        tops[0] = fmaxf(upper ? tops[1] : tops[0], t);
        for (int o = 4; o < group; o <<= 1) {
          sums[0] += __shfl_xor_sync(kAllWarp, sums[0], o);
          tops[0] = fmaxf(tops[0], __shfl_xor_sync(kAllWarp, tops[0], o));
        }
      }
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int row = r0 + (mine + i) * step;
        if (i >= held || row >= e.count) break;
        float f = 1.f;
        odd |= !(usual(tops[i]) && usual(sums[i])) && !(sums[i] == 0.f && tops[i] == 0.f);
        if (a.norm != TMS_NORM_NONE) {
          if (a.norm == TMS_NORM_L2) {
            f = sums[i] > 0.f ? rsqrtf(sums[i]) : 1.f;
            odd |= sums[i] > 0.f ? !(f * a.eps < 0.999f) : a.eps == 0.f;  // at or under eps; 0 / 0
          } else {
            f = rsqrtf(fmaf(sums[i], per_d, a.eps));
          }
          odd |= !usual(f);
        }
        const float t = tops[i] * f;
        row_factor[row] = f;
        row_top[row] = t;
        top = fmaxf(top, t);
      }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(kAllWarp, top, o));
    odd = __any_sync(kAllWarp, odd);
    if (lane == 0) {
      warp_top[warp] = top;
      warp_odd[warp] = odd;
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kWarps; ++i) {
      top = fmaxf(top, warp_top[i]);
      odd |= warp_odd[i] != 0;
    }
    // Rows that can set the scale, a warp for each 32 rows.
    double best = 0.0;
    bool bad = false;
    for (int base = warp * 32; base < page; base += kWriteThreads) {
      const int row = base + lane;
      uint32_t might = __ballot_sync(kAllWarp, row < e.count && (odd || row_top[row] >= top * (1.f - 0x1p-19f)));
      while (might) {
        const int r = base + __ffs(might) - 1;
        might &= might - 1;
        ExactRow exact;
        double y;
        for (bool full = odd;; full = true) {  // the same for all lanes
          exact_row(rows, e, r, row_factor[r], full, exact);
          y = full ? exact.top / exact.norm : exact.top * exact.factor;
          if (full || sure_scale(y)) break;
        }
        bad |= exact.bad;
        if (y > best) best = y;
      }
    }
    if (lane == 0) {
      warp_best[warp] = best;
      warp_bad[warp] = bad;
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kWarps; ++i) {
      if (warp_best[i] > best) best = warp_best[i];
      bad |= warp_bad[i] != 0;
    }
    const float scale = bad ? __int_as_float(0x7fffffff) : static_cast<float>(scale_of(best));
    const bool plain = !odd && usual(scale);
    const float inverse = __frcp_rn(scale);
    if (threadIdx.x == 0) a.scales[e.id] = scale;
    uint8_t* const out = a.codes + (e.id << a.page_shift) * d + sub * 8;
    for (int r0 = row0, b = 0; b < page; r0 += 4 * step, b += 4 * step) {  // the same turns for all lanes
      uint32_t unsure = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int row = r0 + i * step;
        if (row >= page) break;
        const int src = row < e.count ? row : e.count - 1;  // behind the last token: that token again
        Eight<T> x, r;
        rows.load(e, src, x, r);
        const float g = row_factor[src] * inverse;
        const float under = g * (1.f - 0x1p-20f), over = g * (1.f + 0x1p-20f);
        uint32_t word[2], other[2];
#pragma unroll
        for (int j = 0; j < 8; j += 4) {
          float h[4];
#pragma unroll
          for (int l = 0; l < 4; ++l) {
            h[l] = x.at(j + l);
            if constexpr (SUM) h[l] += r.at(j + l);
            if constexpr (WEIGHT) h[l] *= wt.at(j + l);
          }
          const uint64_t p0 = f2_pack(h[0], h[1]), p1 = f2_pack(h[2], h[3]);
          const uint64_t lo2 = f2_pack(under, under), hi2 = f2_pack(over, over);
          word[j >> 2] = e4m3x4(f2_unpack(f2_mul(p0, lo2)), f2_unpack(f2_mul(p1, lo2)));
          other[j >> 2] = e4m3x4(f2_unpack(f2_mul(p0, hi2)), f2_unpack(f2_mul(p1, hi2)));
        }
        if (!plain || !usual(g)) {
          unsure |= 1u << i;
        } else if ((word[0] ^ other[0]) | (word[1] ^ other[1])) {
          if (!SUM && !WEIGHT && a.norm == TMS_NORM_NONE) {  // h is exact, and so is the remainder of h / scale
#pragma unroll
            for (int j = 0; j < 8; j += 4)
              word[j >> 2] = e4m3x4(make_float2(off_midpoint(x.at(j), scale), off_midpoint(x.at(j + 1), scale)),
                                    make_float2(off_midpoint(x.at(j + 2), scale), off_midpoint(x.at(j + 3), scale)));
          } else {
            unsure |= 1u << i;
          }
        }
        if (in_row) *reinterpret_cast<uint2*>(out + row * d) = make_uint2(word[0], word[1]);
      }
      // Rows that fp32 is not sure of, again.
      uint32_t again = __reduce_or_sync(kAllWarp, unsure);
      while (again) {
        const int i = __ffs(again) - 1;
        again &= again - 1;
        const int row = r0 + i * step;
        const int src = row < e.count ? row : e.count - 1;
        ExactRow exact;
        exact_row(rows, e, src, 0.f, true, exact);
        if (!(unsure >> i & 1u) || row >= page || !in_row) continue;
        uint32_t word[2] = {0, 0};
        const double by = exact.norm * scale;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const uint32_t code = bad ? 0x7fu : scale > 0.f ? e4m3_of_double(exact.h[j] / by) : 0u;
          word[j >> 2] |= code << (8 * (j & 3));
        }
        *reinterpret_cast<uint2*>(out + row * d) = make_uint2(word[0], word[1]);
      }
    }
  }
  if constexpr (STAGED) cp_async_wait_all();
}

template <typename T, bool SUM, bool WEIGHT, int D, int THREADS>
cudaError_t launch_staged(const WriteArgs& a, int group, unsigned blocks, int input, cudaStream_t st) {
  // A constant width has pages of 16 rows at least: fewer threads than those take are not reached.
  if constexpr (D > 0 && THREADS < write_threads(D * 16 * static_cast<int>(sizeof(T)) * (SUM ? 2 : 1))) {
    return cudaErrorInvalidValue;
  } else {
    auto kern = page_write_kernel<T, SUM, WEIGHT, true, D, THREADS>;
    if (2 * input + kStaticBytes > 48 * 1024) {  // more than a launch may have unasked
      const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, 2 * kStageBytes);
      if (e != cudaSuccess) return e;
    }
    kern<<<blocks, THREADS, 2 * input, st>>>(a, group);
    return cudaGetLastError();
  }
}

template <typename T, bool SUM, bool WEIGHT>
cudaError_t launch_write_as(const WriteArgs& a, const DeviceInfo* dev, cudaStream_t st) {
  int group = 2;  // lanes of a row
  while (group * 8 < a.d) group <<= 1;
  const int input = (a.d << a.page_shift) * static_cast<int>(sizeof(T)) * (SUM ? 2 : 1);
  const bool staged = input <= kStageBytes;
  const int threads = staged ? write_threads(input) : 128;
  // As many CTAs as fit at a time: each then has its next page on the way while it works on one.
  const int fit = staged ? dev->max_smem_optin / (2 * input + kStaticBytes) : 16, room = staged ? 768 / threads : 16;
  const int64_t most = static_cast<int64_t>(dev->num_sms) * (fit < room ? fit : room);
  const unsigned blocks = static_cast<unsigned>(a.page_cap < most ? a.page_cap : most);
  if (!staged) {
    page_write_kernel<T, SUM, WEIGHT, false, 0, 128><<<blocks, 128, 0, st>>>(a, group);
    return cudaGetLastError();
  }
  if (a.d == 128) {  // a constant width where it is the usual one: see the kernel's figures
    return threads == 32   ? launch_staged<T, SUM, WEIGHT, 128, 32>(a, group, blocks, input, st)
           : threads == 64 ? launch_staged<T, SUM, WEIGHT, 128, 64>(a, group, blocks, input, st)
                           : launch_staged<T, SUM, WEIGHT, 128, 128>(a, group, blocks, input, st);
  }
  return threads == 32   ? launch_staged<T, SUM, WEIGHT, 0, 32>(a, group, blocks, input, st)
         : threads == 64 ? launch_staged<T, SUM, WEIGHT, 0, 64>(a, group, blocks, input, st)
                         : launch_staged<T, SUM, WEIGHT, 0, 128>(a, group, blocks, input, st);
}

template <typename T>
cudaError_t launch_write(const WriteArgs& a, const DeviceInfo* dev, cudaStream_t st) {
  if (a.residual) return a.weight ? launch_write_as<T, true, true>(a, dev, st) : launch_write_as<T, true, false>(a, dev, st);
  return a.weight ? launch_write_as<T, false, true>(a, dev, st) : launch_write_as<T, false, false>(a, dev, st);
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

// out[t] = scale * code of slot t; a slot outside the pool gives a row of zeros. One multiplication
// in fp32, then one rounding to the output type. A group of lanes takes a row, sixteen elements a
// lane (one 16-byte load), and a thread ROWS rows, whose loads are all in flight before the first
// store: what bounds it is memory. The output is written past the caches' working set. 3.6M rows of
// 128 to bf16 take 299 us with two rows and 266 us with four (5.3 TB/s), 182 thousand to fp16 15.5 us
// with either: four where that makes 32 CTAs an SM and more, two, which start sooner, below.

template <typename T>
__device__ __forceinline__ uint32_t two_as(float x, float y) {
  if constexpr (std::is_same<T, __half>::value) {
    const __half2 h = __floats2half2_rn(x, y);
    return *reinterpret_cast<const uint32_t*>(&h);
  } else {
    const __nv_bfloat162 h = __floats2bfloat162_rn(x, y);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
}
__device__ __forceinline__ float2 e4m3x2_value(uint32_t two) {
  uint32_t h;
  asm("{\n\t.reg .b16 p;\n\tcvt.u16.u32 p, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, p;\n\t}\n" : "=r"(h) : "r"(two));
  return __half22float2(*reinterpret_cast<const __half2*>(&h));
}

template <typename T, int ROWS>
__global__ void __launch_bounds__(256) page_read_kernel(const ReadArgs a, int group) {
  const int sub = threadIdx.x & (group - 1);
  const int64_t rows = 256 / group;  // of a CTA at a time
  const bool in_row = sub * 16 < a.d;
  for (int64_t t0 = blockIdx.x * rows * ROWS + threadIdx.x / group; t0 < a.n_slots;
       t0 += gridDim.x * rows * ROWS) {
    int64_t slot[ROWS];
    uint4 c[ROWS];
    float scale[ROWS];
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
      const int64_t t = t0 + i * rows;
      slot[i] = t < a.n_slots ? __ldg(a.slots + t) : -1;
    }
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
      c[i] = make_uint4(0, 0, 0, 0);
      scale[i] = 0.f;
      if (slot[i] >= 0 && (slot[i] >> a.page_shift) < a.n_pages && in_row) {
        c[i] = __ldg(reinterpret_cast<const uint4*>(a.codes + slot[i] * a.d + sub * 16));
        scale[i] = __ldg(a.scales + (slot[i] >> a.page_shift));
      }
    }
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
      const int64_t t = t0 + i * rows;
      if (t >= a.n_slots || !in_row) continue;
      const uint32_t w[4] = {c[i].x, c[i].y, c[i].z, c[i].w};
      float v[16];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float2 f = e4m3x2_value(w[j >> 1] >> (16 * (j & 1)) & 0xffffu);
        v[2 * j] = f.x * scale[i];
        v[2 * j + 1] = f.y * scale[i];
      }
      uint4* const o = reinterpret_cast<uint4*>(static_cast<T*>(a.out) + t * a.d + sub * 16);
      if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int q = 0; q < 4; ++q)
          __stcs(o + q, make_uint4(__float_as_uint(v[4 * q]), __float_as_uint(v[4 * q + 1]),
                                   __float_as_uint(v[4 * q + 2]), __float_as_uint(v[4 * q + 3])));
      } else {
#pragma unroll
        for (int q = 0; q < 2; ++q)
          __stcs(o + q, make_uint4(two_as<T>(v[8 * q], v[8 * q + 1]), two_as<T>(v[8 * q + 2], v[8 * q + 3]),
                                   two_as<T>(v[8 * q + 4], v[8 * q + 5]), two_as<T>(v[8 * q + 6], v[8 * q + 7])));
      }
    }
  }
}

template <typename T>
void launch_read(const ReadArgs& a, const DeviceInfo* dev, cudaStream_t st) {
  int group = 1;  // lanes of a row
  while (group * 16 < a.d) group <<= 1;
  const int64_t rows = 256 / group, most = static_cast<int64_t>(dev->num_sms) * 16;
  const bool many = a.n_slots >= rows * 4 * dev->num_sms * 32;
  const int64_t each = rows * (many ? 4 : 2);
  const int64_t blocks = (a.n_slots + each - 1) / each;
  const unsigned grid = static_cast<unsigned>(blocks < most ? blocks : most);
  if (many) page_read_kernel<T, 4><<<grid, 256, 0, st>>>(a, group);
  else page_read_kernel<T, 2><<<grid, 256, 0, st>>>(a, group);
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

extern "C" size_t tms_page_tables_workspace_size(int64_t n_docs, int64_t page_capacity) {
  if (n_docs <= kFewDocs || page_capacity < 0) return 0;
  return static_cast<size_t>((n_docs + kTileDocs - 1) / kTileDocs) * 16 +
         align_up(static_cast<size_t>(page_capacity / 32 + 1) * 4, 16);
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
  const size_t need = tms_page_tables_workspace_size(n_docs, page_capacity);
  if (need && (!workspace || workspace_bytes < need)) return TMS_ERR_WORKSPACE;
  if (reinterpret_cast<uintptr_t>(workspace) & 7) return TMS_ERR_INVALID;
  int status = TMS_OK;
  const DeviceInfo* dev = current_device_info(&status);
  if (!dev) return status;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const int64_t tiles = (n_docs + kTileDocs - 1) / kTileDocs;
  int64_t* const sums = static_cast<int64_t*>(workspace);
  const TableArgs a{lengths, n_lengths, doc_ids, n_docs, src_offsets, pages, n_src_pages, shift, page_offsets,
                    token_offsets, page_ids, page_docs, page_capacity, slots, slots ? token_capacity : 0,
                    sums, reinterpret_cast<int32_t*>(sums + 2 * tiles)};
  int64_t blocks = (page_capacity + kTableThreads - 1) / kTableThreads;
  const int64_t most = static_cast<int64_t>(dev->num_sms) * 8;
  blocks = blocks < 1 ? 1 : blocks > most ? most : blocks;
  if (n_docs <= kFewDocs) {
    if (blocks > dev->num_sms) blocks = dev->num_sms;  // each CTA works out the offsets
    table_few_kernel<<<static_cast<unsigned>(blocks), kTableThreads, 0, st>>>(a);
  } else {
    table_sums_kernel<<<static_cast<unsigned>(tiles), kTableThreads, 0, st>>>(a);
    table_offsets_kernel<<<static_cast<unsigned>(tiles), kTableThreads, 0, st>>>(a);
    table_fill_kernel<<<static_cast<unsigned>(blocks), kTableThreads, 0, st>>>(a);
  }
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
  if (!(eps >= 0.f && eps <= 3.4028235e38f)) return TMS_ERR_INVALID;
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
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return cuda_status(dtype == TMS_F16    ? launch_write<__half>(a, dev, st)
                     : dtype == TMS_BF16 ? launch_write<__nv_bfloat16>(a, dev, st)
                                         : launch_write<float>(a, dev, st));
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
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (out_dtype == TMS_F16) launch_read<__half>(a, dev, st);
  else if (out_dtype == TMS_BF16) launch_read<__nv_bfloat16>(a, dev, st);
  else launch_read<float>(a, dev, st);
  return cuda_status(cudaGetLastError());
}
