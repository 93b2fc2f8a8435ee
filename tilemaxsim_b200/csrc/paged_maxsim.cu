// paged_maxsim.cu -- MaxSim over a paged 8-bit corpus (see paged.cu for the pages):
//
//   score[q, doc] = sum_i max over the document's pages p of  scale_p * max_j <Q[q,i,:], code_pj>
//
// The scale of a page is not negative, so it is applied once to the page's maximum. Rows behind a
// document's last token repeat that token: maxima run over whole pages, and nothing is masked.
//
// The codes go to the tensor cores as they are stored (tcgen05 kind::f8f6f4, fp32 accumulators).
// A 16-bit query element does not fit e4m3's four significant bits, so each query row is scaled by
// a power of two (its largest magnitude lands in [128, 256)) and split into terms, each the rounding
// of what the terms before it left, e4m3 ones and an e5m2 one last: two terms hold bf16's eight bits,
// three hold fp16's eleven, the last three of them at most in the last term. The terms are laid side by
// side along K against the same tokens, so one accumulator holds the whole product. What is lost lies
// under e5m2's three bits of what e4m3's smallest step, 2^-9, leaves: an element below 2^-13 (bf16) or
// 2^-10 (fp16) of its row's largest is off by at most 2^-21 of that largest. (With an e4m3 term last it
// was 2^-17 of it, at the same speed.)
//
// Work split. The table entries (pages) are cut into ranges at document boundaries, one a CTA, and
// each range evenly into S streams. A tile is 256 token columns: W = 256 / S of each stream's next
// pages. Query rows are the MMA's M dimension, 32 rows (a "chunk") to a TMEM lane quarter. Up to
// four chunks at a time use M = 128; one or two use the weight-stationary MMA with M = 32 or 64,
// which repeats the rows over the lane quarters and gives each quarter its own columns (a scan of
// 100k documents took 549 us with the rows repeated by hand at M = 128). Either way each of
// the eight epilogue warps reads one chunk's rows against one stream's columns and keeps each row's
// running maximum. A document cut by a stream boundary is joined from the streams' partial maxima
// when the CTA is done. Few long documents would leave ranges uneven: they are cut evenly instead, and
// what a document has in several ranges is joined by a kernel of its own. No atomics, and the sums
// run in one order: results do not depend on the launch.
//
// For one or two chunks, tokens of d = 64 lie two to a row of 128 bytes, in memory as in a stage, which
// halves the rows that the TMA brings and the stage's bytes: the MMAs take N = 128 rows twice, their first
// 64 bytes and their second, into the two halves of the columns.
//
// What bounds it (in a few passes, and in passes without end, which run into the power cap and other inputs).
// One query over 100k documents (18.2M tokens, 2.53 GB of pages): memory, 402 and 443 us, 6.3 and 5.7
// TB/s. 64 queries over 4,000 documents: the tensor cores, 252 and 298 us, 1,510 and 1,280 TFLOP/s of the
// query's own products, which the two terms double. 5 queries of 77 rows at d = 256 in fp16 (three
// terms): the tensor cores, 221 and 259 us. Few chunks of narrow tokens: the instructions that a warp's
// own loop takes for a tile, where each waits for the one before. 18.2M tokens of d = 64: 265 us, the
// MMA warp (397 us with loops and 64-bit descriptors around its 8 MMAs and one wait after the other).
// d = 64, pages of 16, 5.1M tokens, 3 queries: 123 and 136 us, the epilogue, the MMA warp and the 16 boxes
// a tile. Copying the pages by cp.async in place of the TMA: 154 us with four warps, 181-228 with two.
//
// Warp roles (320 threads, one CTA an SM): warp 0 loads pages by TMA (a lane for each box of up to
// 32 rows), warp 1 owns TMEM and issues the MMAs, warps 2-9 are the epilogue. A document that ends
// puts its 32 row maxima into a queue in shared memory; up to sixteen documents are summed at a time
// (two lanes each), which takes the 5-step shuffle sum per document out of the loop.
#include <type_traits>

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include "tms_device.cuh"
#include "tms_internal.h"

namespace tms {
namespace {

constexpr int kThreads = 320;
constexpr int kEpiWarp0 = 2;
constexpr int kReadyBarrier = 1;  // named barrier: warp 0 arrives (streams, barriers), warps 1-9 wait
constexpr int kJoinBarrier = 2;   // named barrier of the epilogue warps: the streams are done
constexpr int kTile = 256;        // token columns of a tile
constexpr int kStages = 6, kSlots = 4;  // at most
constexpr uint32_t kRow = 128;          // bytes of a row in one K chunk
// Bytes of a stage, which holds one K chunk of a tile; in pairs, two tokens share a row.
constexpr uint32_t stage_bytes(bool pair) { return kTile * kRow / (pair ? 2 : 1); }
constexpr int kQueue = 16;        // documents of an epilogue warp's queue
constexpr int kQueueStride = 33;  // floats; the odd stride keeps both accesses conflict-free
constexpr int kMostMt = 4;        // most M tiles of a CTA
constexpr float kNegInf = -__builtin_huge_valf();
// What a range begins with: nothing of its own, a document's first page, or a page inside a document
// that goes on behind the range.
constexpr int kRangeEmpty = -3, kRangeClean = -2, kRangeInside = -1;
// Ranges cut documents whose mean length is this or more, as far as the host knows it: by the capacity of the
// tables, which for a selection is a bound (its results do not depend on it; a needless join takes 2 us).
constexpr int kSplitTokens = 1024;
constexpr int kSplitDocs = 16;      // and of which there are fewer than this for each range
constexpr int kMostSms = 160;       // CTAs that the workspace has parts for

struct PagedArgs {
  const void* Q;
  int q_bf16;
  int terms;
  int nq, nchunk;      // query rows; 32-row chunks of a query
  int n_chunks;        // over all queries
  int n_mtiles, mt, groups, ranges;
  int d, kc;           // kc: 128-byte K chunks
  int stages;
  int page_shift, unit_shift;  // log2 of the page rows, and of the units (boxes) in a page
  const uint8_t* packed;       // the packed query tiles, or nullptr: the CTA packs its own
  const float* packed_factor;
  const float* scales;
  int64_t n_pages;
  const int64_t* page_offsets;
  const int32_t* page_ids;
  const int32_t* page_docs;
  int64_t n_docs, page_cap;
  float* out;          // (n_chunks, n_docs)
  // Where ranges may cut documents: (ranges, 2, 4 n_mtiles, 32) row maxima of the document that a
  // range begins in the middle of, and of the one that it ends in the middle of; and (ranges, 2)
  // which document the first one is (kRange...) and whether there is a second one. Else nullptr.
  float* parts;
  int* part_docs;
  uint32_t* err;
  uint64_t timeout_ns;
  int debug_flags;
};

struct Stream {  // what one stream of a CTA covers
  int32_t first, units;  // first table entry; boxes
  int32_t open;          // whether its first document began in the stream before
  int32_t end;           // the last table entry + 1 that a document can reach
};
struct SmemLayout {
  uint32_t q, q_bytes, stage, queue, best, head, factor, bars, streams, misc, total;
};

__host__ __device__ inline SmemLayout smem_layout(int nc, int mt, int terms, int kc, int stages, bool pair) {
  SmemLayout L;
  L.q = 0;
  L.q_bytes = static_cast<uint32_t>(terms * kc * nc * 32) * kRow;  // of one M tile
  L.stage = static_cast<uint32_t>(mt) * L.q_bytes;
  L.queue = L.stage + static_cast<uint32_t>(stages) * stage_bytes(pair);
  L.best = L.queue + 8u * kQueue * kQueueStride * 4u;
  L.head = L.best + 8u * static_cast<uint32_t>(mt) * 128u;
  L.factor = L.head + 8u * static_cast<uint32_t>(mt) * 128u;
  L.bars = L.factor + static_cast<uint32_t>(mt * nc) * 128u;
  L.streams = L.bars + (2u * kStages + 2u * kSlots + 2u) * 8u;
  L.misc = L.streams + 8u * static_cast<uint32_t>(sizeof(Stream));
  L.total = L.misc + 64u;
  return L;
}

// Maxima that a NaN survives.
__device__ __forceinline__ float max_nan(float x, float y) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(x), "f"(y));
  return r;
}
__device__ __forceinline__ float max3_nan(float x, float y, float z) {
  float r;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(x), "f"(y), "f"(z));
  return r;
}
// The maximum of N (16 or 32) accumulator columns.
template <int N>
__device__ __forceinline__ float max_columns(const uint32_t* r) {
  float m[5];
#pragma unroll
  for (int i = 0; i < 5; ++i)
    m[i] = max3_nan(__uint_as_float(r[3 * i]), __uint_as_float(r[3 * i + 1]), __uint_as_float(r[3 * i + 2]));
  float rest = __uint_as_float(r[15]);
  if constexpr (N == 32) {
#pragma unroll
    for (int i = 0; i < 5; ++i)
      m[i] = max3_nan(m[i], __uint_as_float(r[16 + 2 * i]), __uint_as_float(r[17 + 2 * i]));
#pragma unroll
    for (int i = 0; i < 3; ++i)
      m[i] = max3_nan(m[i], __uint_as_float(r[26 + 2 * i]), __uint_as_float(r[27 + 2 * i]));
  }
  return max3_nan(max3_nan(m[0], m[1], m[2]), max_nan(m[3], m[4]), rest);
}

// The same of 16 columns in two groups of eight, 16 columns apart.
__device__ __forceinline__ float max_columns_pair(const uint32_t* r) {
  const float a = max3_nan(__uint_as_float(r[0]), __uint_as_float(r[1]), __uint_as_float(r[2]));
  const float b = max3_nan(__uint_as_float(r[3]), __uint_as_float(r[4]), __uint_as_float(r[5]));
  const float c = max3_nan(__uint_as_float(r[6]), __uint_as_float(r[7]), __uint_as_float(r[16]));
  const float d = max3_nan(__uint_as_float(r[17]), __uint_as_float(r[18]), __uint_as_float(r[19]));
  const float e = max3_nan(__uint_as_float(r[20]), __uint_as_float(r[21]), __uint_as_float(r[22]));
  return max3_nan(max3_nan(a, b, c), max_nan(d, e), __uint_as_float(r[23]));
}
// 32 lanes x 16 columns, asynchronous, into r[0..15]; valid after tmem_wait_ld32.
__device__ __forceinline__ void tmem_ld16_async(uint32_t taddr, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr)
      : "memory");
}

// One lane of a converged warp.
__device__ __forceinline__ uint32_t elect_one() {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "elect.sync _|p, 0xffffffff;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}\n"
      : "=r"(r));
  return r;
}
// D(tmem) (+)= A * B^T, both K-major 8-bit in shared memory, fp32 accumulation, issued by the lane
// whose `leader` is set. The whole warp runs the loop around it: the descriptors then stay in
// uniform registers (64 queries, 4k documents: 423 us under "lane == 0", 324 us so at the time).
__device__ __forceinline__ void mma_f8(uint32_t d_tmem, uint64_t adesc, uint64_t bdesc, uint32_t idesc,
                                       uint32_t accumulate, uint32_t leader) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "setp.ne.b32 q, %5, 0;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(d_tmem),
      "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate), "r"(leader)
      : "memory");
}
// The weight-stationary form for M = 32 or 64 rows: the rows come out repeated over the lane
// quarters, each with its own share of the columns. B stays in the tensor core's buffer over the
// query terms that multiply it: KEEP 0 fills the buffer, 1 uses it, 2 uses it for the last time.
template <int KEEP>
__device__ __forceinline__ void mma_f8_ws(uint32_t d_tmem, uint64_t adesc, uint64_t bdesc, uint32_t idesc,
                                          uint32_t accumulate, uint32_t leader) {
#define TMS_MMA_WS(usage)                                                                            \
  asm volatile(                                                                                      \
      "{\n\t.reg .pred p, q;\n\t"                                                                    \
      "setp.ne.b32 p, %4, 0;\n\t"                                                                    \
      "setp.ne.b32 q, %5, 0;\n\t"                                                                    \
      "@q tcgen05.mma.ws.cta_group::1.kind::f8f6f4.collector::b0::" usage " [%0], %1, %2, %3, p;\n\t}\n" ::"r"(d_tmem), \
      "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate), "r"(leader)                               \
      : "memory")
  if constexpr (KEEP == 0) TMS_MMA_WS("fill");
  else if constexpr (KEEP == 1) TMS_MMA_WS("use");
  else TMS_MMA_WS("lastuse");
#undef TMS_MMA_WS
}
// mbar_wait by a converged warp.
__device__ __forceinline__ bool warp_wait(uint32_t bar, uint32_t parity, volatile int* abort, uint64_t timeout_ns,
                                          uint32_t* err, uint32_t site) {
  if (__all_sync(0xffffffffu, mbar_try_wait(bar, parity))) return true;
  return __all_sync(0xffffffffu, mbar_wait(bar, parity, abort, timeout_ns, err, site));
}
// Arrives on `bar` when the MMAs issued so far by the leader are done.
__device__ __forceinline__ void commit(uint32_t bar, uint32_t leader) {
  asm volatile(
      "{\n\t.reg .pred q;\n\t"
      "setp.ne.b32 q, %1, 0;\n\t"
      "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}\n" ::"r"(bar),
      "r"(leader)
      : "memory");
}
// tma_load_2d by the lane whose `leader` is set; all lanes of a converged warp run it alike.
__device__ __forceinline__ void box_load(uint32_t dst, const CUtensorMap* map, uint32_t bar, int32_t x, int32_t y,
                                         uint64_t policy, uint32_t leader) {
  asm volatile(
      "{\n\t.reg .pred q;\n\t"
      "setp.ne.b32 q, %6, 0;\n\t"
      "@q cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.L2::cache_hint"
      " [%0], [%1, {%3, %4}], [%2], %5;\n\t}\n" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(x), "r"(y), "l"(policy), "r"(leader)
      : "memory");
}
__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst),
               "l"(reinterpret_cast<uint64_t>(src)), "r"(bytes), "r"(bar)
               : "memory");
}
// The packed queries come from the launch before this one, which this one does not wait to end.
__device__ __forceinline__ void wait_for_packed() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

// A value that is the same in all lanes, told to the compiler.
__device__ __forceinline__ int uniform(int v) { return __shfl_sync(0xffffffffu, v, 0); }

// First table entry of part j of `parts`: an even cut, moved up to the next document's first entry.
__device__ __forceinline__ int64_t cut_at(const PagedArgs& a, int64_t total, int64_t j, int64_t parts) {
  const int64_t c = total * j / parts;
  if (c <= 0) return 0;
  if (c >= total) return total;
  const int64_t doc = __ldg(a.page_docs + c);
  if (doc < 0 || doc >= a.n_docs) return c;
  if (__ldg(a.page_offsets + doc) >= c) return c;
  const int64_t next = __ldg(a.page_offsets + doc + 1);
  return next < c ? c : next > total ? total : next;
}

__device__ __forceinline__ int64_t clamp_entry(const PagedArgs& a, int64_t v) {
  return v < 0 ? 0 : v > a.page_cap ? a.page_cap : v;
}

// Rows [r0, r0 + kPackRows) of an M tile (32 * nc rows) as e4m3 and e5m2 terms in the 128-byte-swizzle layout
// (16-byte unit u of row r at u ^ (r % 8); tiles [term][K chunk][row]) at `tile`, and for each row
// the power of two to undo at `factor`. One warp, a lane four elements of each 128-byte chunk.
constexpr int kPackRows = 4;

__device__ __forceinline__ void pack_rows(const PagedArgs& a, int nc, int m, int r0, uint8_t* tile, float* factor) {
  const int lane = lane_id();
  uint2 u[kPackRows][2];
#pragma unroll
  for (int i = 0; i < kPackRows; ++i) {
    const int r = r0 + i;
    const int chunk = m * 4 + (r >> 5);
    const int query = chunk / a.nchunk;
    const int row = (chunk - query * a.nchunk) * 32 + (r & 31);
    const bool real = chunk < a.n_chunks && row < a.nq;
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      const int e = c * 128 + lane * 4;
      u[i][c] = make_uint2(0, 0);
      if (real && e < a.d)
        u[i][c] = __ldg(reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(a.Q) +
                                                       (static_cast<int64_t>(query) * a.nq + row) * a.d + e));
    }
  }
#pragma unroll
  for (int i = 0; i < kPackRows; ++i) {
    const int r = r0 + i;
    float v[8];
    float big = 0.f;
#pragma unroll
    for (int h = 0; h < 4; ++h) {
      const uint32_t w = h & 2 ? (h & 1 ? u[i][1].y : u[i][1].x) : (h & 1 ? u[i][0].y : u[i][0].x);
      if (a.q_bf16) {
        v[2 * h] = __uint_as_float(w << 16);
        v[2 * h + 1] = __uint_as_float(w & 0xffff0000u);
      } else {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w));
        v[2 * h] = f.x;
        v[2 * h + 1] = f.y;
      }
      big = max3_nan(big, fabsf(v[2 * h]), fabsf(v[2 * h + 1]));
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) big = max_nan(big, __shfl_xor_sync(0xffffffffu, big, o));
    // big * 2^up lies in [128, 256). 2^up and 2^-up can leave fp32's normal range, so both are
    // applied as two factors; a row of zeros takes up = 0.
    const bool finite = big <= 3.4028235e38f;
    const bool small = big < 1.1754944e-38f;  // a subnormal magnitude: find its exponent after 2^64
    const uint32_t bits = __float_as_uint(small ? big * 18446744073709551616.f : big);
    const int exp = static_cast<int>(bits >> 23) - 127 - (small ? 64 : 0);
    const int up = finite && big > 0.f ? 7 - exp : 0;  // -120 .. 140
    const int half = up >> 1;
    const float s1 = __uint_as_float(static_cast<uint32_t>(127 + half) << 23);
    const float s2 = __uint_as_float(static_cast<uint32_t>(127 + up - half) << 23);
    if (lane == 0)
      factor[r] = finite ? __uint_as_float(static_cast<uint32_t>(127 - half) << 23) *
                               __uint_as_float(static_cast<uint32_t>(127 - (up - half)) << 23)
                         : __int_as_float(0x7fffffff);
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      if (c >= a.kc) break;
      float rest[4];
#pragma unroll
      for (int h = 0; h < 4; ++h) rest[h] = finite ? v[c * 4 + h] * s1 * s2 : 0.f;
      uint8_t* at = tile + static_cast<uint32_t>(c * 32 * nc + r) * kRow + (((lane >> 2) ^ (r & 7)) << 4) + (lane & 3) * 4;
      for (int t = 0; t < a.terms; ++t) {
        uint32_t word = 0;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const float2 now = make_float2(rest[2 * h], rest[2 * h + 1]);
          __nv_fp8x2_storage_t two;
          if (t == a.terms - 1) {
            two = __nv_cvt_float2_to_fp8x2(now, __NV_SATFINITE, __NV_E5M2);
          } else {
            two = __nv_cvt_float2_to_fp8x2(now, __NV_SATFINITE, __NV_E4M3);
            const float2 back = __half22float2(__half2(__nv_cvt_fp8x2_to_halfraw2(two, __NV_E4M3)));
            rest[2 * h] -= back.x;
            rest[2 * h + 1] -= back.y;
          }
          word |= static_cast<uint32_t>(two) << (16 * h);
        }
        *reinterpret_cast<uint32_t*>(at) = word;
        at += static_cast<uint32_t>(a.kc * 32 * nc) * kRow;
      }
    }
  }
}

// All M tiles (of four chunks) of a call, packed once, not by each CTA: 128 rows took a CTA 7 us. The
// scoring kernel's CTAs start meanwhile and find their streams.
__global__ void __launch_bounds__(256) paged_pack_kernel(const PagedArgs a, uint8_t* packed, float* factor) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int64_t row = (static_cast<int64_t>(blockIdx.x) * 8 + (threadIdx.x >> 5)) * kPackRows;
  const int m = static_cast<int>(row >> 7);
  if (m < a.n_mtiles)
    pack_rows(a, 4, m, static_cast<int>(row & 127), packed + static_cast<int64_t>(m) * a.terms * a.kc * 128 * kRow,
              factor + static_cast<int64_t>(m) * 128);
}

// NC: chunks of an M tile (1, 2 or 4); U: tokens of a box (16 or 32); PAIR: d = 64, and two tokens to a
// row of 128 bytes, in memory and in a stage.
template <int NC, int U, bool PAIR>
__global__ void __launch_bounds__(kThreads, 1)
paged_mma_kernel(const __grid_constant__ CUtensorMap codes_map, const __grid_constant__ PagedArgs a) {
  constexpr int kStreams = 8 / NC;
  constexpr int W = kTile / kStreams;     // columns of a stream in a tile
  constexpr int kUnits = W / U;           // boxes of a stream in a tile
  constexpr int kCols = kTile * NC / 4;   // TMEM columns of an accumulator: the columns of a lane quarter
  constexpr int kAcc = 512 / kCols < kSlots ? 512 / kCols : kSlots;  // accumulators
  constexpr uint32_t kAllWarp = 0xffffffffu;
  static_assert(kCols == 2 * W && 32 % kUnits == 0 && 2 * kUnits <= kQueue, "two warps a lane quarter");
  extern __shared__ __align__(1024) uint8_t smem[];
  constexpr int kBoxRows = PAIR ? U / 2 : U;
  constexpr uint32_t kStageBytes = stage_bytes(PAIR);
  const SmemLayout L = smem_layout(NC, a.mt, a.terms, a.kc, a.stages, PAIR);
  const int warp = uniform(threadIdx.x >> 5), lane = lane_id();
  const int group = blockIdx.x % a.groups, range = blockIdx.x / a.groups;
  const int m_first = group * a.mt;
  const int mt = a.n_mtiles - m_first < a.mt ? a.n_mtiles - m_first : a.mt;

  uint32_t* const tmem_slot = reinterpret_cast<uint32_t*>(smem + L.misc);
  int* const tiles = reinterpret_cast<int*>(smem + L.misc + 4);
  int* const goes_on = reinterpret_cast<int*>(smem + L.misc + 48);
  volatile int* const abort_flag = reinterpret_cast<volatile int*>(smem + L.misc + 8);
  volatile int* const never_flag = reinterpret_cast<volatile int*>(smem + L.misc + 12);
  int* const head_docs = reinterpret_cast<int*>(smem + L.misc + 16);  // 8: an epilogue warp's head document
  Stream* const streams = reinterpret_cast<Stream*>(smem + L.streams);
  const uint32_t base = smem_u32(smem);
  const uint32_t bars = base + L.bars;
  auto full_bar = [&](int s) { return bars + 8u * s; };
  auto empty_bar = [&](int s) { return bars + 8u * (kStages + s); };
  auto accf_bar = [&](int s) { return bars + 8u * (2 * kStages + s); };
  auto acce_bar = [&](int s) { return bars + 8u * (2 * kStages + kSlots + s); };
  const uint32_t done_bar = bars + 8u * (2 * kStages + 2 * kSlots), query_bar = done_bar + 8u;
  int n_tiles = 0;
  bool dead;
  if (warp == 0) {
    // Barriers and streams. Every decision of the CTA goes by what this warp read of the tables.
    if (lane == 0) {
      *abort_flag = (base & 1023u) ? 1 : 0;
      *never_flag = 0;
      if (*abort_flag) atomicCAS(a.err, 0u, kDevErrTimeout | 40u);
      for (int s = 0; s < a.stages; ++s) {
        mbar_init(full_bar(s), 1);
        mbar_init(empty_bar(s), 1);
      }
      for (int s = 0; s < kAcc; ++s) {
        mbar_init(accf_bar(s), 1);
        mbar_init(acce_bar(s), 8);
      }
      mbar_init(done_bar, 1);
      mbar_init(query_bar, 1);
      fence_mbar_init();
    }
    const int64_t total = clamp_entry(a, __ldg(a.page_offsets + a.n_docs));
    const int64_t cut = lane >= 2   ? 0
                        : a.parts ? total * (range + lane) / a.ranges
                                  : cut_at(a, total, range + lane, a.ranges);
    const int64_t lo = __shfl_sync(kAllWarp, cut, 0);
    int64_t hi = __shfl_sync(kAllWarp, cut, 1);
    hi = hi < lo ? lo : hi;
    const int64_t first = lo + (hi - lo) * lane / kStreams;  // of stream `lane`
    const int64_t next = lo + (hi - lo) * (lane + 1) / kStreams;
    const int units = lane < kStreams ? static_cast<int>((next - first) << a.unit_shift) : 0;  // below 2^30 (host)
    if (lane < kStreams) {
      const bool open = units > 0 && first > (a.parts ? 0 : lo) && __ldg(a.page_docs + first) == __ldg(a.page_docs + first - 1);
      streams[lane] = Stream{static_cast<int32_t>(first), units, open, static_cast<int32_t>(a.parts ? total : hi)};
    }
    n_tiles = (units + kUnits - 1) / kUnits;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const int y = __shfl_xor_sync(kAllWarp, n_tiles, o);
      n_tiles = y > n_tiles ? y : n_tiles;
    }
    if (lane == 0) {
      *tiles = n_tiles;
      // whether the last document goes on in the next range
      *goes_on = a.parts && hi > lo && hi < total && __ldg(a.page_docs + hi) == __ldg(a.page_docs + hi - 1);
    }
    __syncwarp();
    dead = *abort_flag != 0;
    asm volatile("barrier.arrive %0, %1;" ::"r"(kReadyBarrier), "r"(kThreads) : "memory");
    if (a.packed && !dead && n_tiles > 0) {
      if (lane == 0) {
        wait_for_packed();
        mbar_arrive_expect_tx(query_bar, static_cast<uint32_t>(mt) * L.q_bytes);
        for (int m = 0; m < mt; ++m)
          bulk_load(base + L.q + static_cast<uint32_t>(m) * L.q_bytes,
                    a.packed + static_cast<int64_t>(m_first + m) * L.q_bytes, L.q_bytes, query_bar);
      }
      __syncwarp();
    }
  } else {
    if (warp == 1) {
      tmem_alloc(smem_u32(tmem_slot), 512);
      tmem_relinquish();
    }
    float* const factor = reinterpret_cast<float*>(smem + L.factor);
    if (a.packed) {
      wait_for_packed();
      for (int i = threadIdx.x - 32; i < mt * 128; i += kThreads - 32) factor[i] = a.packed_factor[m_first * 128 + i];
    } else {  // one or two chunks
      for (int r0 = (warp - 1) * kPackRows; r0 < 32 * NC; r0 += 9 * kPackRows)
        pack_rows(a, NC, m_first, r0, smem + L.q, factor);
      fence_proxy_async_smem();  // the tensor core reads what the packing wrote
    }
    tc_fence_before();
    asm volatile("barrier.sync %0, %1;" ::"r"(kReadyBarrier), "r"(kThreads) : "memory");
    tc_fence_after();
    n_tiles = *tiles;
    dead = *abort_flag != 0;
  }
  n_tiles = uniform(n_tiles);

  // Documents without a table entry: this CTA's share of them, done by the epilogue warps while the
  // first tile is on its way.
  auto write_empty = [&]() {
    const int64_t lo = a.n_docs * range / a.ranges, hi = a.n_docs * (range + 1) / a.ranges;
    for (int64_t doc = lo + threadIdx.x - kEpiWarp0 * 32; doc < hi; doc += kThreads - kEpiWarp0 * 32) {
      if (clamp_entry(a, __ldg(a.page_offsets + doc)) < clamp_entry(a, __ldg(a.page_offsets + doc + 1))) continue;
      for (int c = m_first * 4; c < (m_first + mt) * 4 && c < a.n_chunks; ++c) a.out[c * a.n_docs + doc] = kNegInf;
    }
  };
  if (dead) {
    // no role runs: misaligned shared memory
  } else if (n_tiles == 0) {
    if (warp >= kEpiWarp0) write_empty();
    if (a.parts && threadIdx.x == 32) a.part_docs[2 * range] = kRangeEmpty;
  } else if (warp == 0) {
    // ------------------------------------------------------------------ loads: a lane for each box
    static_assert(kTile / U <= 32, "a lane for each box");
    const int stream = lane / kUnits, nth = lane % kUnits;
    const Stream mine = stream < kStreams ? streams[stream] : Stream{0, 0, 0, 0};
    const uint64_t policy = a.groups > 1 ? policy_evict_normal() : policy_evict_first();
    const int half_mask = (1 << a.unit_shift) - 1;
    auto page_of = [&](int unit) -> int64_t {
      return unit < mine.units ? __ldg(a.page_ids + mine.first + (unit >> a.unit_shift)) : -1;
    };
    // Page ids are fetched kAhead tiles ahead: one tile ahead, the wait for them paced the loop.
    constexpr int kAhead = 4;
    int64_t ids[kAhead];
#pragma unroll
    for (int i = 0; i < kAhead; ++i) ids[i] = page_of(i * kUnits + nth);
    int s = 0;
    uint32_t ph = 0, armed = 0, armed_par = 0;
    const uint32_t leader = elect_one();
    bool ok = !(a.debug_flags & 1);
    for (int t0 = 0; ok && t0 < n_tiles; t0 += kAhead) {
#pragma unroll
     for (int i = 0; i < kAhead; ++i) {
      const int t = t0 + i;
      if (!ok || t >= n_tiles) break;
      const int unit = t * kUnits + nth;
      const int64_t id = ids[i];
      ids[i] = page_of(unit + kAhead * kUnits);
      const bool load = id >= 0 && id < a.n_pages;
      const uint32_t mask = __ballot_sync(kAllWarp, load), boxes = __popc(mask);
      const int32_t y = static_cast<int32_t>(id << (a.page_shift - PAIR)) + (unit & half_mask) * kBoxRows;
      int32_t rows[kTile / U];  // of all boxes, before the first load: a shuffle between loads holds them up
#pragma unroll
      for (int b = 0; b < kTile / U; ++b) rows[b] = __shfl_sync(kAllWarp, y, b);
      for (int c = 0; c < a.kc; ++c) {
        ok = warp_wait(empty_bar(s), ph ^ 1u, abort_flag, a.timeout_ns, a.err, 41);
        if (!ok) break;
        if (lane == 0) mbar_arrive_expect_tx(full_bar(s), boxes * static_cast<uint32_t>(kBoxRows * kRow));
        armed |= 1u << s;
        armed_par = (armed_par & ~(1u << s)) | (ph << s);
        __syncwarp();
        auto load_box = [&](int b) {
          box_load(base + L.stage + static_cast<uint32_t>(s) * kStageBytes + b * kBoxRows * kRow, &codes_map,
                   full_bar(s), c * 128, rows[b], policy, leader);
        };
        if (boxes == kTile / U) {  // without a branch for each (137 against 132 us with sixteen)
#pragma unroll
          for (int b = 0; b < kTile / U; ++b) load_box(b);
        } else {
#pragma unroll
          for (int b = 0; b < kTile / U; ++b)
            if (mask >> b & 1u) load_box(b);
        }
        if (++s == a.stages) { s = 0; ph ^= 1u; }
      }
     }
    }
    // every copy lands before the CTA ends, also where a wait of another role gave up
    for (int i = 0; i < a.stages; ++i)
      if (armed & (1u << i)) mbar_wait(full_bar(i), (armed_par >> i) & 1u, never_flag, a.timeout_ns, a.err, 42);
    if (a.packed) mbar_wait(query_bar, 0, never_flag, a.timeout_ns, a.err, 47);
  } else {
    const uint32_t tmem = static_cast<uint32_t>(uniform(static_cast<int>(*tmem_slot)));
    if (warp == 1) {
      // ---------------------------------------------------------------- MMA issue
      constexpr uint32_t idesc = make_idesc(32 * NC, PAIR ? kTile / 2 : kTile, 0);  // e4m3 operands, fp32 accumulator
      constexpr uint32_t idesc_last = idesc | 1u << 7;  // the last term: A is e5m2
      const uint32_t leader = elect_one();
      const uint64_t desc0 = sw128_kmajor_desc(0);
      auto desc = [&](uint32_t lo) { return desc0 & ~0xffffffffull | lo; };  // steps stay in the low word
      const uint32_t a0 = static_cast<uint32_t>(sw128_kmajor_desc(base + L.q));
      const uint32_t b0 = static_cast<uint32_t>(sw128_kmajor_desc(base + L.stage));
      const uint32_t term_step = static_cast<uint32_t>(a.kc * 32 * NC) * kRow >> 4;  // in descriptor units
      const int terms = a.terms, kc = a.kc, stages = a.stages;
      const int last_steps = (a.d - (kc - 1) * 128 + 31) / 32;  // 32-element steps of the last chunk
      int s = 0;
      uint32_t ph = 0, slot = 0, acc_ph = 1;
      bool ok = true;
      if (a.packed) ok = __all_sync(kAllWarp, mbar_wait(query_bar, 0, abort_flag, a.timeout_ns, a.err, 48));
      for (int t = 0; ok && t < n_tiles; ++t) {
        for (int m = 0; m < mt; ++m) {
          // An accumulator and the tile's first stage, looked at together.
          const bool both = mbar_try_wait(acce_bar(slot), acc_ph) & (m > 0 || mbar_try_wait(full_bar(s), ph));
          if (!__all_sync(kAllWarp, both)) {
            ok = warp_wait(acce_bar(slot), acc_ph, abort_flag, a.timeout_ns, a.err, 44);
            if (ok && m == 0) ok = warp_wait(full_bar(s), ph, abort_flag, a.timeout_ns, a.err, 43);
            if (!ok) break;
          }
          tc_fence_after();
          for (int c = 0; c < kc; ++c) {  // kc > 1 comes with one M tile
            if (c > 0) {
              ok = warp_wait(full_bar(s), ph, abort_flag, a.timeout_ns, a.err, 43);
              if (!ok) break;
              tc_fence_after();
            }
            const int steps = c == kc - 1 ? last_steps : 4;
            const uint32_t a_lo = a0 + static_cast<uint32_t>(m * L.q_bytes + c * 32 * NC * kRow) / 16;
            const uint32_t b_lo = b0 + static_cast<uint32_t>(s) * (kStageBytes / 16);
            const uint32_t to = tmem + slot * kCols;
            auto step = [&](auto three, uint32_t to, uint32_t at, uint32_t bt, uint32_t acc) {  // 32 elements of K
              if constexpr (NC == 4) {
                mma_f8(to, desc(at), desc(bt), idesc, acc, leader);
                if constexpr (three.value) mma_f8(to, desc(at + term_step), desc(bt), idesc, 1, leader);
                mma_f8(to, desc(at + (three.value ? 2 : 1) * term_step), desc(bt), idesc_last, 1, leader);
              } else {
                mma_f8_ws<0>(to, desc(at), desc(bt), idesc, acc, leader);
                if constexpr (three.value) mma_f8_ws<1>(to, desc(at + term_step), desc(bt), idesc, 1, leader);
                mma_f8_ws<2>(to, desc(at + (three.value ? 2 : 1) * term_step), desc(bt), idesc_last, 1, leader);
              }
            };
            // The issuing warp's own instructions count: one warp alone takes several clocks for each.
            auto all_steps = [&](auto three) {
              if constexpr (PAIR) {
                // first the rows' first tokens, then their second ones, 64 bytes on, into columns of their own
#pragma unroll
                for (int k = 0; k < 4; ++k) step(three, to + (k >> 1) * W, a_lo + 2 * (k & 1), b_lo + 2 * k, k & 1);
              } else if (steps == 4) {
#pragma unroll
                for (int k = 0; k < 4; ++k) step(three, to, a_lo + 2 * k, b_lo + 2 * k, k > 0 || c > 0);
              } else {
                for (int k = 0; k < steps; ++k) step(three, to, a_lo + 2 * k, b_lo + 2 * k, k > 0 || c > 0);
              }
            };
            if (terms == 3) all_steps(std::true_type());
            else all_steps(std::false_type());
            if (m == mt - 1) {
              commit(empty_bar(s), leader);
              if (++s == stages) { s = 0; ph ^= 1u; }
            }
          }
          if (!ok) break;
          commit(accf_bar(slot), leader);
          if (++slot == kAcc) { slot = 0; acc_ph ^= 1u; }
        }
      }
      commit(done_bar, leader);  // nothing is in flight when the CTA ends
      mbar_wait(done_bar, 0, never_flag, a.timeout_ns, a.err, 45);
    } else {
      // ---------------------------------------------------------------- epilogue
      const int quarter = warp & 3, half = (warp - kEpiWarp0) >> 2;
      const int chunk = quarter % NC;
      const int stream = quarter / NC * 2 + half;
      const int me = half * 4 + quarter;  // this warp's place in the shared arrays
      const int my_first = streams[stream].first, my_units = streams[stream].units, cta_end = streams[stream].end;
      const int half_mask = (1 << a.unit_shift) - 1;
      float* const queue = reinterpret_cast<float*>(smem + L.queue) + me * kQueue * kQueueStride;
      float* const bests = reinterpret_cast<float*>(smem + L.best) + me * a.mt * 32 + lane;  // [m], running
      float* const heads = reinterpret_cast<float*>(smem + L.head) + me * a.mt * 32 + lane;  // [m]
      const float* const factor = reinterpret_cast<const float*>(smem + L.factor) + chunk * 32 + lane;
      const int first_chunk = m_first * 4 + chunk;
      int queued = 0;
      int64_t my_dest = 0;
      auto push = [&](int m, int doc, float v) {
        const int c = first_chunk + m * 4;
        if (c >= a.n_chunks) return;
        queue[queued * kQueueStride + lane] = v * factor[m * 32 * NC];
        if (lane == queued) my_dest = c * a.n_docs + doc;
        ++queued;
      };
      auto flush = [&]() {
        __syncwarp();
        const float* const row = queue + (lane & 15) * kQueueStride + (lane >> 4) * 16;
        float sum = row[0];
#pragma unroll
        for (int i = 1; i < 16; ++i) sum += row[i];
        sum += __shfl_xor_sync(kAllWarp, sum, 16);
        if (lane < queued) a.out[my_dest] = sum;
        __syncwarp();
        queued = 0;
      };
      // What the epilogue needs of 32 boxes, a lane for each: the page's scale (-1: no page there) and
      // the document that ends with the box (-1: none does). Table entries are loaded 64 boxes ahead and
      // looked at 32 boxes ahead, when the scale is loaded: no load is waited for where it is issued.
      float cur_scale = 0.f, next_scale = 0.f;
      int cur_ends = -1, next_ends = -1;
      int entry_id = -1, entry_doc = -1, entry_after = -1;  // page, document, the next entry's document
      uint32_t end_mask = 0;  // a bit for each of the 32 boxes with which a document ends
      uint32_t odd_mask = 0;  // and for each that is not a plain page inside a document
      auto entries = [&](int u0) {
        const int u = u0 + lane;
        entry_id = entry_doc = entry_after = -1;
        if (u < my_units) {
          const int v = my_first + (u >> a.unit_shift);
          entry_id = __ldg(a.page_ids + v);
          if ((u & half_mask) == half_mask) {
            entry_doc = __ldg(a.page_docs + v);
            if (v + 1 < cta_end) entry_after = __ldg(a.page_docs + v + 1);
          }
        }
      };
      auto fetch = [&](int u0) {
        next_scale = -1.f;
        if (entry_id >= 0 && entry_id < a.n_pages) next_scale = __ldg(a.scales + entry_id);
        next_ends = entry_doc >= 0 && entry_doc < a.n_docs && entry_after != entry_doc ? entry_doc : -1;
        entries(u0 + 32);
      };
      entries(0);
      fetch(0);
      write_empty();
      for (int m = 0; m < mt; ++m) bests[m * 32] = kNegInf;
      bool open = streams[stream].open;  // the document in hand began in the stream before
      if (lane == 0) head_docs[me] = -1;
      int slot = 0;
      uint32_t acc_ph = 0;
      bool ok = true;
      for (int t = 0; ok && t < n_tiles; ++t) {
        const int unit0 = t * kUnits;
        if ((unit0 & 31) == 0) {
          cur_scale = next_scale;
          cur_ends = next_ends;
          end_mask = __ballot_sync(kAllWarp, cur_ends >= 0);
          odd_mask = __ballot_sync(kAllWarp, cur_ends >= 0 || cur_scale < 0.f);
          fetch(unit0 + 32);  // also past the stream's end: another stream may go on
        }
        float scales[kUnits];
#pragma unroll
        for (int i = 0; i < kUnits; ++i) scales[i] = __shfl_sync(kAllWarp, cur_scale, (unit0 + i) & 31);
        const uint32_t ends_here = end_mask >> (unit0 & 31);
        const uint32_t odd_here = odd_mask >> (unit0 & 31);
        bool still_open = open;
        for (int m = 0; m < mt; ++m) {
          float best = bests[m * 32];
          ok = warp_wait(accf_bar(slot), acc_ph, abort_flag, a.timeout_ns, a.err, 46);
          if (!ok) break;
          tc_fence_after();
          // In pairs, a stream's first tokens of rows lie in one half of the columns, the second ones in the other.
          const uint32_t at = tmem + slot * kCols + half * (PAIR ? W / 2 : W) + (static_cast<uint32_t>(quarter * 32) << 16);
          auto load = [&](int b, uint32_t(&r)[32]) {  // 32 tokens' columns
            if constexpr (PAIR) {
              tmem_ld16_async(at + 16 * b, r);
              tmem_ld16_async(at + W + 16 * b, r + 16);
            } else {
              tmem_ld32_async(at + 32 * b, r);
            }
          };
          still_open = open;
          auto one = [&](int i, float v) {  // box i of the tile is done
            if (!(scales[i] < 0.f)) best = max_nan(best, v * scales[i]);
            if (ends_here >> i & 1u) {
              const int ends = __shfl_sync(kAllWarp, cur_ends, (unit0 + i) & 31);
              if (still_open) {  // joined with the streams before at the end
                heads[m * 32] = best;
                if (lane == 0) head_docs[me] = ends;
                still_open = false;
              } else {
                push(m, ends, best);
              }
              best = kNegInf;
            }
          };
          uint32_t ra[32], rb[32];
          load(0, ra);
#pragma unroll
          for (int b = 0; b < W / 32; ++b) {
            uint32_t(&cur)[32] = (b & 1) ? rb : ra;
            uint32_t(&nxt)[32] = (b & 1) ? ra : rb;
            tmem_wait_ld32(cur);
            if (b + 1 < W / 32) {
              load(b + 1, nxt);
            } else {  // the accumulator goes back before its last columns are reduced
              tc_fence_before();
              __syncwarp();
              if (lane == 0) mbar_arrive(acce_bar(slot));
            }
            if constexpr (U == 32) {
              const float v = max_columns<32>(cur);
              if (!(odd_here >> b & 1u)) best = max_nan(best, v * scales[b]);
              else one(b, v);
            } else {
              const float v = PAIR ? max_columns_pair(cur) : max_columns<16>(cur);
              const float w = PAIR ? max_columns_pair(cur + 8) : max_columns<16>(cur + 16);
              if (!(odd_here >> 2 * b & 3u)) {
                best = max3_nan(best, v * scales[2 * b], w * scales[2 * b + 1]);
              } else {
                one(2 * b, v);
                one(2 * b + 1, w);
              }
            }
          }
          bests[m * 32] = best;
          if (queued > kQueue - kUnits) flush();
          if (++slot == kAcc) { slot = 0; acc_ph ^= 1u; }
        }
        open = still_open;
      }
      // Documents that streams share: the chunk's first stream's warp walks the streams in order.
      asm volatile("barrier.sync %0, %1;" ::"r"(kJoinBarrier), "r"(256) : "memory");
      if (ok && quarter < NC && half == 0) {
        int begins = kRangeClean;
        for (int m = 0; m < mt; ++m) {
          float* const part = a.parts + (static_cast<int64_t>(range) * 8 * a.n_mtiles + first_chunk + m * 4) * 32 + lane;
          const float f = factor[m * 32 * NC];
          float run = kNegInf;
          bool first = true, inside = false;  // inside: still in the document that the range began in the middle of
          for (int s = 0; s < kStreams; ++s) {
            if (streams[s].units == 0) continue;
            const int at = (s & 1) * 4 + (s >> 1) * NC + chunk;
            const float tail = reinterpret_cast<const float*>(smem + L.best)[(at * a.mt + m) * 32 + lane];
            if (first) inside = streams[s].open;
            first = false;
            if (streams[s].open && head_docs[at] < 0) {  // inside one document from end to end
              run = max_nan(run, tail);
              continue;
            }
            if (streams[s].open) {
              const float v = max_nan(run, reinterpret_cast<const float*>(smem + L.head)[(at * a.mt + m) * 32 + lane]);
              if (inside) {
                part[0] = v * f;
                begins = head_docs[at];
                inside = false;
              } else {
                push(m, head_docs[at], v);
                if (queued == kQueue) flush();
              }
            }
            run = tail;
          }
          if (inside) begins = kRangeInside;
          if (*goes_on) part[4 * a.n_mtiles * 32] = run * f;
        }
        if (a.parts && chunk == 0 && lane == 0) {
          a.part_docs[2 * range] = begins;
          a.part_docs[2 * range + 1] = *goes_on;
        }
      }
      if (queued) flush();
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(*tmem_slot, 512);
  }
}

// Documents that several ranges have parts of: a warp for each range that one begins in, and chunk.
// The sum runs as the scoring kernel's: rows 0-15, rows 16-31, then both.
__global__ void __launch_bounds__(256) paged_join_kernel(const PagedArgs a) {
  const int lane = lane_id();
  const int64_t w = static_cast<int64_t>(blockIdx.x) * 8 + (threadIdx.x >> 5);
  const int r = static_cast<int>(w / a.n_chunks), chunk = static_cast<int>(w % a.n_chunks);
  if (r >= a.ranges) return;
  const int64_t step = static_cast<int64_t>(4) * a.n_mtiles * 32;  // from a range's first part to its second
  const float* const at = a.parts + static_cast<int64_t>(chunk) * 32 + lane;
  const int begins = a.part_docs[2 * r];
  if (begins == kRangeEmpty || begins == kRangeInside || !a.part_docs[2 * r + 1]) return;
  float v = at[(2 * r + 1) * step];
  for (int e = r + 1; e < a.ranges; ++e) {
    const int doc = a.part_docs[2 * e];
    if (doc == kRangeEmpty) continue;
    if (doc == kRangeInside) {
      v = max_nan(v, at[(2 * e + 1) * step]);
      continue;
    }
    if (doc < 0 || doc >= a.n_docs) return;
    v = max_nan(v, at[2 * e * step]);
    float lo = __shfl_sync(0xffffffffu, v, 0), hi = __shfl_sync(0xffffffffu, v, 16);
    for (int i = 1; i < 16; ++i) {
      lo += __shfl_sync(0xffffffffu, v, i);
      hi += __shfl_sync(0xffffffffu, v, 16 + i);
    }
    if (lane == 0) a.out[chunk * a.n_docs + doc] = lo + hi;
    return;
  }
}

// out[q, doc] = the sum of the query's chunks, in order.
__global__ void paged_sum_kernel(const float* __restrict__ part, float* __restrict__ out, int64_t n_queries,
                                 int64_t n_docs, int nchunk) {
  const int64_t total = n_queries * n_docs;
  for (int64_t i = blockIdx.x * static_cast<int64_t>(blockDim.x) + threadIdx.x; i < total;
       i += static_cast<int64_t>(gridDim.x) * blockDim.x) {
    const int64_t q = i / n_docs, doc = i - q * n_docs;
    float s = 0.f;
    for (int p = 0; p < nchunk; ++p) s += part[(q * nchunk + p) * n_docs + doc];
    out[i] = s;
  }
}

__global__ void paged_fill_kernel(float* out, int64_t n) {
  for (int64_t i = blockIdx.x * static_cast<int64_t>(blockDim.x) + threadIdx.x; i < n;
       i += static_cast<int64_t>(gridDim.x) * blockDim.x)
    out[i] = kNegInf;
}

int blocks_for(int64_t work, const DeviceInfo* dev) {
  const int64_t b = (work + 255) / 256, most = static_cast<int64_t>(dev->num_sms) * 8;
  return static_cast<int>(b < 1 ? 1 : b > most ? most : b);
}

template <int NC, int U, bool PAIR>
int launch(const CUtensorMap& map, const PagedArgs& a, cudaStream_t st) {
  auto kern = paged_mma_kernel<NC, U, PAIR>;
  const uint32_t smem = smem_layout(NC, a.mt, a.terms, a.kc, a.stages, PAIR).total;
  if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem)) != cudaSuccess)
    return TMS_ERR_CUDA;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(a.groups * a.ranges));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute early = {};
  early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  early.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &early;
  cfg.numAttrs = a.packed ? 1 : 0;  // the packing kernel is the launch before
  return cuda_status(cudaLaunchKernelEx(&cfg, kern, map, a));
}

// Workspace: the chunks' scores of queries of more than 32 rows, then the packed query tiles and
// their factors when there are more than two chunks, then the parts of documents cut by ranges.
struct Workspace {
  size_t chunks, packed, factor, parts, part_docs;
  size_t total() const { return chunks + packed + factor + parts + part_docs; }
};
Workspace workspace_of(int64_t n_queries, int64_t nq, int64_t d, int64_t n_docs, int64_t page_size, int64_t page_cap) {
  Workspace w = {};
  const int64_t nchunk = (nq + 31) / 32, mtiles = (n_queries * nchunk + 3) / 4;
  if (nchunk > 1) w.chunks = align_up(static_cast<size_t>(n_queries * nchunk * n_docs) * sizeof(float), 128);
  if (n_queries * nchunk > 2) {
    w.packed = static_cast<size_t>(mtiles * 3 * ((d + 127) / 128) * 128) * kRow;
    w.factor = static_cast<size_t>(mtiles) * 128 * sizeof(float);
  }
  // Mean lengths by the table's capacity. Ranges times M tiles are at
  // most 4 for each SM (a CTA holds up to four M tiles).
  if (mtiles <= 2 * kMostSms && page_cap * page_size >= n_docs * kSplitTokens && n_docs < kSplitDocs * kMostSms) {
    w.parts = static_cast<size_t>(4 * kMostSms + mtiles) * 8 * 32 * sizeof(float);
    w.part_docs = 2 * kMostSms * sizeof(int);
  }
  return w;
}

}  // namespace
}  // namespace tms

using namespace tms;

extern "C" size_t tms_paged_workspace_size(int64_t n_queries, int64_t nq, int64_t d, int64_t n_docs,
                                           int64_t page_size, int64_t page_capacity) {
  if (n_queries <= 0 || nq <= 0 || d <= 0 || n_docs <= 0 || page_size <= 0 || page_capacity <= 0) return 0;
  return workspace_of(n_queries, nq, d, n_docs, page_size, page_capacity).total();
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
  const int64_t nchunk = (nq + 31) / 32;
  if (page_capacity >= (int64_t(1) << 30) || page_capacity * ((page_size + 31) / 32) >= (int64_t(1) << 30) ||
      n_docs >= (int64_t(1) << 31) || n_pages >= (int64_t(1) << 27) ||
      n_pages * page_size >= (int64_t(1) << 31) || nq >= (int64_t(1) << 24) ||
      n_queries >= (int64_t(1) << 24) || n_queries * nchunk >= (int64_t(1) << 24))
    return TMS_ERR_UNSUPPORTED;
  if (!Q || !out || !page_offsets || (page_capacity > 0 && (!page_ids || !page_docs)) ||
      (n_pages > 0 && (!codes || !scales)))
    return TMS_ERR_INVALID;
  if ((reinterpret_cast<uintptr_t>(Q) & 15) || (reinterpret_cast<uintptr_t>(codes) & 15) ||
      (reinterpret_cast<uintptr_t>(workspace) & 127))
    return TMS_ERR_INVALID;
  const Workspace w =
      page_capacity > 0 ? workspace_of(n_queries, nq, d, n_docs, page_size, page_capacity) : Workspace{};
  const size_t need = w.total();
  if (need && (!workspace || workspace_bytes < need)) return TMS_ERR_WORKSPACE;
  int status = TMS_OK;
  const DeviceInfo* dev = current_device_info(&status);
  if (!dev) return status;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (n_pages == 0 || page_capacity == 0) {  // every document is empty
    paged_fill_kernel<<<blocks_for(n_queries * n_docs, dev), 256, 0, st>>>(out, n_queries * n_docs);
    return cuda_status(cudaGetLastError());
  }

  PagedArgs a = {};
  a.Q = Q;
  a.q_bf16 = q_dtype == TMS_BF16;
  a.terms = a.q_bf16 ? 2 : 3;
  a.nq = static_cast<int>(nq);
  a.nchunk = static_cast<int>(nchunk);
  a.n_chunks = static_cast<int>(n_queries * nchunk);
  a.n_mtiles = (a.n_chunks + 3) / 4;
  a.d = static_cast<int>(d);
  a.kc = (a.d + 127) / 128;
  a.page_shift = 4;
  while ((int64_t(1) << a.page_shift) < page_size) ++a.page_shift;
  const int U = page_size == 16 ? 16 : 32;
  a.unit_shift = a.page_shift - (U == 16 ? 4 : 5);
  a.scales = scales;
  a.n_pages = n_pages;
  a.page_offsets = page_offsets;
  a.page_ids = page_ids;
  a.page_docs = page_docs;
  a.n_docs = n_docs;
  a.page_cap = page_capacity;
  a.out = nchunk > 1 ? static_cast<float*>(workspace) : out;
  a.err = dev->err_word;
  a.timeout_ns = wait_timeout_ns();
  a.debug_flags = debug_flags();

  const int nc = a.n_chunks < 3 ? a.n_chunks : 4;
  // Two tokens of d = 64 to a row, for one or two chunks: 18.2M tokens 260 us against 328 (pages of 16 rows
  // 278 against 388), two chunks over 5.1M 96 against 114. With four, the epilogue's twice as many loads
  // cost more than the TMA gains: 114 against 111, 64 queries 192 against 189.
  const bool pair = d == 64 && nc < 4;
  const uint32_t room = static_cast<uint32_t>(dev->max_smem_optin);
  // As many M tiles a CTA as leave two stages: each tile of tokens is then loaded and held for all
  // of them. With two K chunks a tile's stages pass one by one, so there is one M tile.
  a.mt = a.kc > 1 ? 1 : a.n_mtiles < kMostMt ? a.n_mtiles : kMostMt;
  while (a.mt > 1 && smem_layout(nc, a.mt, a.terms, a.kc, 2, pair).total > room) --a.mt;
  a.groups = (a.n_mtiles + a.mt - 1) / a.mt;
  a.mt = (a.n_mtiles + a.groups - 1) / a.groups;
  a.stages = 2;
  while (a.stages < kStages && smem_layout(nc, a.mt, a.terms, a.kc, a.stages + 1, pair).total <= room) ++a.stages;
  int64_t ranges = dev->num_sms / a.groups;
  if (ranges > page_capacity) ranges = page_capacity;
  a.ranges = static_cast<int>(ranges < 1 ? 1 : ranges);

  uint8_t* const packed = static_cast<uint8_t*>(workspace) + w.chunks;
  float* const factor = reinterpret_cast<float*>(packed + w.packed);
  if (w.parts && ranges > 1 && dev->num_sms <= kMostSms && n_docs < kSplitDocs * ranges) {
    a.parts = factor + w.factor / sizeof(float);
    a.part_docs = reinterpret_cast<int*>(a.parts + w.parts / sizeof(float));
  }
  if (nc == 4) {
    paged_pack_kernel<<<static_cast<unsigned>((a.n_mtiles * 128 + 8 * kPackRows - 1) / (8 * kPackRows)), 256, 0, st>>>(
        a, packed, factor);
    if (cudaGetLastError() != cudaSuccess) return TMS_ERR_CUDA;
    a.packed = packed;
    a.packed_factor = factor;
  }
  CUtensorMap map;
  const int64_t row = pair ? 2 * d : d, rows = n_pages * page_size / (pair ? 2 : 1);
  int rc = encode_tmap_2d(&map, CU_TENSOR_MAP_DATA_TYPE_UINT8, codes, static_cast<uint64_t>(row),
                          static_cast<uint64_t>(rows), static_cast<uint64_t>(row), 128,
                          static_cast<uint32_t>(pair ? U / 2 : U));
  if (rc != TMS_OK) return rc;
  if (U == 16) {
    rc = nc == 4   ? launch<4, 16, false>(map, a, st)
         : nc == 2 ? (pair ? launch<2, 16, true>(map, a, st) : launch<2, 16, false>(map, a, st))
                   : (pair ? launch<1, 16, true>(map, a, st) : launch<1, 16, false>(map, a, st));
  } else {
    rc = nc == 4   ? launch<4, 32, false>(map, a, st)
         : nc == 2 ? (pair ? launch<2, 32, true>(map, a, st) : launch<2, 32, false>(map, a, st))
                   : (pair ? launch<1, 32, true>(map, a, st) : launch<1, 32, false>(map, a, st));
  }
  if (rc != TMS_OK) return rc;
  if (a.parts) {
    paged_join_kernel<<<static_cast<unsigned>((static_cast<int64_t>(a.ranges) * a.n_chunks + 7) / 8), 256, 0, st>>>(a);
    if (cudaGetLastError() != cudaSuccess) return TMS_ERR_CUDA;
  }
  if (nchunk == 1) return TMS_OK;
  paged_sum_kernel<<<blocks_for(n_queries * n_docs, dev), 256, 0, st>>>(a.out, out, n_queries, n_docs, a.nchunk);
  return cuda_status(cudaGetLastError());
}
