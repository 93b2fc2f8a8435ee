// paged_maxsim.cu -- MaxSim over a paged 8-bit corpus (see paged.cu for the pages):
//
//   score[q, doc] = sum_i max over the document's pages p of  scale_p * max_j <Q[q,i,:], code_pj>
//
// The scale of a page is not negative, so it is applied once to the page's maximum. Rows behind a
// document's last token repeat that token: maxima run over whole pages, and nothing is masked.
//
// The codes go to the tensor cores as they are stored (tcgen05 kind::f8f6f4, fp32 accumulators).
// A 16-bit query element does not fit e4m3's four significant bits, so each query row is scaled by
// a power of two (its largest magnitude lands in [128, 256)) and split into e4m3 terms, each the
// rounding of what the terms before it left: two terms hold bf16's eight bits, three hold fp16's
// eleven. The terms are laid side by side along K against the same tokens, so one accumulator
// holds the whole product. What is lost lies under e4m3's smallest step: an element below 2^-9
// (bf16) or 2^-6 (fp16) of its row's largest is off by at most 2^-17 of that largest.
//
// Work split. The table entries (pages) are cut into ranges, one a CTA, and each range into S
// streams, all at document boundaries: no document straddles two streams, so there is no merge
// between CTAs or warps, no atomic, and results do not depend on the launch. A tile is TN token
// columns: W = TN / S of each stream's next pages. Query rows sit on the 128 TMEM lanes, 32 rows (a
// "chunk") to a lane quarter; with one or two chunks they are repeated over the quarters, so that
// all eight epilogue warps have a stream of their own: a warp always reads one chunk's rows
// against one stream's columns, and keeps each row's running maximum in a register.
//
// Warp roles (320 threads, one CTA an SM): warp 0 loads pages by TMA (a lane for each box of up to
// 32 rows), warp 1 owns TMEM and issues the MMAs, warps 2-9 are the epilogue. A document that ends
// puts its 32 row maxima into a queue in shared memory; sixteen documents are summed at a time (two
// lanes each), which takes the 5-step shuffle sum per document out of the loop.
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
constexpr uint32_t kChunkTile = 128 * 128;  // 128 rows of one 128-byte K chunk
constexpr int kQueue = 16;                  // documents of an epilogue warp's queue
constexpr int kQueueStride = 33;            // floats; the odd stride keeps both accesses conflict-free
constexpr float kNegInf = -__builtin_huge_valf();

struct PagedArgs {
  const void* Q;
  int q_bf16;
  int terms;
  int nq, nchunk;      // query rows; 32-row chunks of a query
  int64_t n_queries;
  int n_chunks;        // over all queries
  int n_mtiles, mt, groups, ranges;
  int d, kc;           // kc: 128-byte K chunks
  int stages;
  int page_shift, unit_shift;  // log2 of the page rows, and of the units (boxes) in a page
  const float* scales;
  int64_t n_pages;
  const int64_t* page_offsets;
  const int32_t* page_ids;
  const int32_t* page_docs;
  int64_t n_docs, page_cap;
  float* out;          // (n_chunks, n_docs)
  uint32_t* err;
  uint64_t timeout_ns;
  int debug_flags;
};

struct SmemLayout {
  uint32_t q, stage, stage_bytes, queue, factor, bars, streams, misc, total;
};
struct Stream {  // what one stream of a CTA covers
  int32_t first, units;  // first table entry; boxes
};
constexpr int kMaxStages = 8;

__host__ __device__ inline SmemLayout smem_layout(int TN, int mt, int terms, int kc, int stages) {
  SmemLayout L;
  L.q = 0;
  L.stage = static_cast<uint32_t>(mt * terms * kc) * kChunkTile;
  L.stage_bytes = static_cast<uint32_t>(kc * TN) * 128u;
  L.queue = L.stage + static_cast<uint32_t>(stages) * L.stage_bytes;
  L.factor = L.queue + 8u * kQueue * kQueueStride * 4u;
  L.bars = L.factor + static_cast<uint32_t>(mt) * 128u * 4u;
  L.streams = L.bars + (2u * kMaxStages + 2u * 4u + 1u) * 8u;
  L.misc = L.streams + 8u * static_cast<uint32_t>(sizeof(Stream));
  L.total = L.misc + 24u;
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
// D(tmem) (+)= A * B^T, both K-major e4m3 in shared memory, fp32 accumulation, issued by the lane
// whose `leader` is set. The whole warp runs the loop around it: the descriptors then stay in
// uniform registers (an issue loop under "lane == 0" cost about 600 clocks a K chunk).
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
__device__ __forceinline__ void commit(uint32_t bar, uint32_t leader) {
  asm volatile(
      "{\n\t.reg .pred q;\n\t"
      "setp.ne.b32 q, %1, 0;\n\t"
      "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}\n" ::"r"(bar),
      "r"(leader)
      : "memory");
}

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

// Query rows of this CTA's M tiles -> e4m3 terms in the 128-byte-swizzle layout (16-byte unit u of
// row r at u ^ (r % 8)), and each row's power of two to undo. Warps 1-9; a warp takes four rows at
// a time, a lane four elements of each 128-byte chunk.
template <int NC>
__device__ void pack_queries(const PagedArgs& a, const SmemLayout& L, uint8_t* smem, int m_first, int mt) {
  const int lane = lane_id(), warp = (threadIdx.x >> 5) - 1;
  constexpr int kWarps = 9, kRows = 4;
  const int rows = mt * 32 * NC;  // distinct rows; NC < 4 repeats them over the lane quarters
  float* const factor = reinterpret_cast<float*>(smem + L.factor);
  for (int r0 = warp * kRows; r0 < rows; r0 += kWarps * kRows) {
    float v[kRows][8];
    float big[kRows];
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
      const int r = r0 + i;
      const int64_t chunk = static_cast<int64_t>(m_first) * 4 + (r >> 5);
      const int64_t query = chunk / a.nchunk;
      const int row = static_cast<int>(chunk - query * a.nchunk) * 32 + (r & 31);
      const bool real = r < rows && chunk < a.n_chunks && row < a.nq;
      big[i] = 0.f;
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const int e = c * 128 + lane * 4;
        uint2 u = make_uint2(0, 0);
        if (real && e < a.d)
          u = __ldg(reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(a.Q) +
                                                   (query * a.nq + row) * a.d + e));
        const uint32_t w[2] = {u.x, u.y};
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          if (a.q_bf16) {
            v[i][c * 4 + h * 2] = __uint_as_float(w[h] << 16);
            v[i][c * 4 + h * 2 + 1] = __uint_as_float(w[h] & 0xffff0000u);
          } else {
            const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[h]));
            v[i][c * 4 + h * 2] = f.x;
            v[i][c * 4 + h * 2 + 1] = f.y;
          }
        }
#pragma unroll
        for (int h = 0; h < 4; ++h) big[i] = max_nan(big[i], fabsf(v[i][c * 4 + h]));
      }
    }
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) big[i] = max_nan(big[i], __shfl_xor_sync(0xffffffffu, big[i], o));
      const int r = r0 + i;
      if (r >= rows) continue;
      // big * 2^up in [128, 256), in two steps because 2^up alone can leave fp32's range
      int exp = 0;
      const bool finite = big[i] <= 3.4028235e38f;
      if (finite && big[i] > 0.f) frexpf(big[i], &exp);
      const int up = big[i] > 0.f && finite ? 8 - exp : 0;
      const int up1 = up > 100 ? 100 : up;
      const float s1 = ldexpf(1.f, up1), s2 = ldexpf(1.f, up - up1);
      const int m = r / (32 * NC), q_row = r - m * 32 * NC;
      if (lane < 4 / NC)
        factor[m * 128 + lane * 32 * NC + q_row] = finite ? ldexpf(1.f, -up) : __int_as_float(0x7fffffff);
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        if (c >= a.kc) break;
        float rest[4];
#pragma unroll
        for (int h = 0; h < 4; ++h) rest[h] = finite ? v[i][c * 4 + h] * s1 * s2 : 0.f;
        for (int t = 0; t < a.terms; ++t) {
          uint32_t word = 0;
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const __nv_fp8x2_storage_t two =
                __nv_cvt_float2_to_fp8x2(make_float2(rest[2 * h], rest[2 * h + 1]), __NV_SATFINITE, __NV_E4M3);
            const float2 back = __half22float2(__half2(__nv_cvt_fp8x2_to_halfraw2(two, __NV_E4M3)));
            rest[2 * h] -= back.x;
            rest[2 * h + 1] -= back.y;
            word |= static_cast<uint32_t>(two) << (16 * h);
          }
          uint8_t* const tile = smem + L.q + static_cast<uint32_t>((m * a.terms + t) * a.kc + c) * kChunkTile;
#pragma unroll
          for (int copy = 0; copy < 4 / NC; ++copy) {
            const int row = copy * 32 * NC + q_row;
            *reinterpret_cast<uint32_t*>(tile + row * 128 + (((lane >> 2) ^ (row & 7)) << 4) + (lane & 3) * 4) = word;
          }
        }
      }
    }
  }
}

// NC: chunks of an M tile (1, 2 or 4); U: rows of a box (16 or 32); MT: most M tiles of a CTA.
template <int TN, int NC, int U, int MT>
__global__ void __launch_bounds__(kThreads, 1)
paged_mma_kernel(const __grid_constant__ CUtensorMap codes_map, const PagedArgs a) {
  constexpr int kStreams = (8 / NC < TN / 32) ? 8 / NC : TN / 32;
  constexpr int W = TN / kStreams;      // columns of a stream in a tile
  constexpr int kUnits = W / U;         // boxes of a stream in a tile
  constexpr int kSlots = 512 / TN;      // accumulators in TMEM
  constexpr int kActive = NC * kStreams;  // epilogue warps that read
  constexpr uint32_t kAllWarp = 0xffffffffu;
  static_assert(kActive <= 8 && 32 % kUnits == 0, "one stream a warp");
  extern __shared__ __align__(1024) uint8_t smem[];
  const SmemLayout L = smem_layout(TN, a.mt, a.terms, a.kc, a.stages);
  const int warp = threadIdx.x >> 5, lane = lane_id();
  const int group = blockIdx.x % a.groups, range = blockIdx.x / a.groups;
  const int m_first = group * a.mt;
  const int mt = a.n_mtiles - m_first < a.mt ? a.n_mtiles - m_first : a.mt;

  uint32_t* const tmem_slot = reinterpret_cast<uint32_t*>(smem + L.misc);
  volatile int* const abort_flag = reinterpret_cast<volatile int*>(smem + L.misc + 8);
  volatile int* const never_flag = reinterpret_cast<volatile int*>(smem + L.misc + 16);
  const uint32_t bars = smem_u32(smem + L.bars);
  auto full_bar = [&](int s) { return bars + 8u * s; };
  auto empty_bar = [&](int s) { return bars + 8u * (kMaxStages + s); };
  auto accf_bar = [&](int s) { return bars + 8u * (2 * kMaxStages + s); };
  auto acce_bar = [&](int s) { return bars + 8u * (2 * kMaxStages + 4 + s); };
  const uint32_t done_bar = bars + 8u * (2 * kMaxStages + 8);
  Stream* const streams = reinterpret_cast<Stream*>(smem + L.streams);
  int* const tiles = reinterpret_cast<int*>(smem + L.misc + 4);
  int n_tiles = 0;
  bool dead;
  if (warp == 0) {
    // Barriers and streams. Every decision of the CTA goes by what this warp read of the tables.
    if (lane == 0) {
      *abort_flag = (smem_u32(smem) & 1023u) ? 1 : 0;
      *never_flag = 0;
      if (*abort_flag) atomicCAS(a.err, 0u, kDevErrTimeout | 40u);
      for (int s = 0; s < a.stages; ++s) {
        mbar_init(full_bar(s), 1);
        mbar_init(empty_bar(s), 1);
      }
      for (int s = 0; s < kSlots; ++s) {
        mbar_init(accf_bar(s), 1);
        mbar_init(acce_bar(s), kActive);
      }
      mbar_init(done_bar, 1);
      fence_mbar_init();
    }
    const int64_t total = clamp_entry(a, __ldg(a.page_offsets + a.n_docs));
    int64_t first = 0;  // lane s: the first entry of stream s
    if (lane <= kStreams)
      first = cut_at(a, total, static_cast<int64_t>(range) * kStreams + lane, static_cast<int64_t>(a.ranges) * kStreams);
    int64_t len = __shfl_down_sync(kAllWarp, first, 1) - first;
    if (lane >= kStreams || len < 0) len = 0;
    const int units = static_cast<int>(len << a.unit_shift);  // below 2^30 (checked on the host)
    if (lane < kStreams) streams[lane] = Stream{static_cast<int32_t>(first), units};
    n_tiles = (units + kUnits - 1) / kUnits;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const int y = __shfl_xor_sync(kAllWarp, n_tiles, o);
      n_tiles = y > n_tiles ? y : n_tiles;
    }
    if (lane == 0) *tiles = n_tiles;
    __syncwarp();
    dead = *abort_flag != 0;
    asm volatile("barrier.arrive %0, %1;" ::"r"(kReadyBarrier), "r"(kThreads) : "memory");
  } else {
    if (warp == 1) {
      tmem_alloc(smem_u32(tmem_slot), 512);
      tmem_relinquish();
    }
    pack_queries<NC>(a, L, smem, m_first, mt);
    fence_proxy_async_smem();  // the tensor core reads what the packing wrote
    tc_fence_before();
    asm volatile("barrier.sync %0, %1;" ::"r"(kReadyBarrier), "r"(kThreads) : "memory");
    tc_fence_after();
    n_tiles = *tiles;
    dead = *abort_flag != 0;
  }

  if (dead || n_tiles == 0) {
    // no role runs (misaligned shared memory, or nothing to score)
  } else if (warp == 0) {
    // ------------------------------------------------------------------ loads: a lane for each box
    static_assert(TN / U <= 32, "a lane for each box");
    const int stream = lane / kUnits, nth = lane % kUnits;
    const Stream mine = stream < kStreams ? streams[stream] : Stream{0, 0};
    const uint64_t policy = a.groups > 1 ? policy_evict_normal() : policy_evict_first();
    const int half_mask = (1 << a.unit_shift) - 1;
    auto page_of = [&](int unit) -> int64_t {
      return unit < mine.units ? __ldg(a.page_ids + mine.first + (unit >> a.unit_shift)) : -1;
    };
    int64_t next = page_of(nth);
    int s = 0;
    uint32_t ph = 0, armed = 0, armed_par = 0;
    bool ok = !(a.debug_flags & 1);
    for (int t = 0; ok && t < n_tiles; ++t) {
      const int unit = t * kUnits + nth;
      const int64_t id = next;
      if (t + 1 < n_tiles) next = page_of(unit + kUnits);
      ok = mbar_wait(empty_bar(s), ph ^ 1u, abort_flag, a.timeout_ns, a.err, 41);
      ok = __all_sync(kAllWarp, ok);
      if (!ok) break;
      const bool load = id >= 0 && id < a.n_pages;
      const uint32_t boxes = __popc(__ballot_sync(kAllWarp, load));
      if (lane == 0) mbar_arrive_expect_tx(full_bar(s), boxes * static_cast<uint32_t>(a.kc * U * 128));
      armed |= 1u << s;
      armed_par = (armed_par & ~(1u << s)) | (ph << s);
      __syncwarp();
      if (load) {
        const uint32_t dst = smem_u32(smem) + L.stage + static_cast<uint32_t>(s) * L.stage_bytes + lane * U * 128;
        const int32_t y = static_cast<int32_t>(id << a.page_shift) + (unit & half_mask) * U;
        for (int c = 0; c < a.kc; ++c)
          tma_load_2d(dst + static_cast<uint32_t>(c * TN * 128), &codes_map, full_bar(s), c * 128, y, policy);
      }
      if (++s == a.stages) { s = 0; ph ^= 1u; }
    }
    // every copy lands before the CTA ends, also where a wait of another role gave up
    for (int i = 0; i < a.stages; ++i)
      if (armed & (1u << i)) mbar_wait(full_bar(i), (armed_par >> i) & 1u, never_flag, a.timeout_ns, a.err, 42);
  } else {
    const uint32_t tmem = *tmem_slot;
    if (warp == 1) {
      // ---------------------------------------------------------------- MMA issue
      constexpr uint32_t idesc = make_idesc(128, TN, 0);  // e4m3 operands, fp32 accumulator
      const uint32_t leader = elect_one();
      const uint32_t q0 = smem_u32(smem) + L.q, d0 = smem_u32(smem) + L.stage;
      int s = 0;
      uint32_t ph = 0, u = 0;
      bool ok = true;
      for (int t = 0; ok && t < n_tiles; ++t) {
        ok = mbar_wait(full_bar(s), ph, abort_flag, a.timeout_ns, a.err, 43);
        ok = __all_sync(kAllWarp, ok);
        if (!ok) break;
        tc_fence_after();
        const uint32_t b0 = d0 + static_cast<uint32_t>(s) * L.stage_bytes;
        for (int m = 0; m < mt; ++m, ++u) {
          const uint32_t slot = u % kSlots;
          ok = mbar_wait(acce_bar(slot), ((u / kSlots) & 1u) ^ 1u, abort_flag, a.timeout_ns, a.err, 44);
          ok = __all_sync(kAllWarp, ok);
          if (!ok) break;
          tc_fence_after();
          uint32_t acc = 0;
          for (int term = 0; term < a.terms; ++term)
            for (int c = 0; c < a.kc; ++c) {
              const int left = a.d - c * 128;
              const uint64_t ad = sw128_kmajor_desc(q0 + static_cast<uint32_t>((m * a.terms + term) * a.kc + c) * kChunkTile);
              const uint64_t bd = sw128_kmajor_desc(b0 + static_cast<uint32_t>(c * TN * 128));
#pragma unroll
              for (int k = 0; k < 4; ++k) {
                if (k * 32 >= left) break;
                mma_f8(tmem + slot * TN, ad + 2 * k, bd + 2 * k, idesc, acc, leader);
                acc = 1;
              }
            }
          commit(accf_bar(slot), leader);
        }
        if (ok) commit(empty_bar(s), leader);
        if (++s == a.stages) { s = 0; ph ^= 1u; }
      }
      commit(done_bar, leader);  // nothing is in flight when the CTA ends
      mbar_wait(done_bar, 0, never_flag, a.timeout_ns, a.err, 45);
    } else {
      // ---------------------------------------------------------------- epilogue
      const int quarter = warp & 3, half = (warp - kEpiWarp0) >> 2;
      const int chunk = quarter % NC;
      const int stream = quarter / NC + (4 / NC) * half;
      if (stream < kStreams) {
        const int64_t my_first = streams[stream].first;
        const int my_units = streams[stream].units;
        const int64_t my_end = my_first + (my_units >> a.unit_shift);
        const int half_mask = (1 << a.unit_shift) - 1;
        float* const queue = reinterpret_cast<float*>(smem + L.queue) + (warp - kEpiWarp0) * kQueue * kQueueStride;
        const float* const factor = reinterpret_cast<const float*>(smem + L.factor) + quarter * 32 + lane;
        int queued = 0;
        int64_t my_dest = 0;
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
        // What the epilogue needs of 32 boxes, a lane for each, fetched 32 boxes ahead: the page's
        // scale (-1: no page there) and the document that ends with the box (-1: none does).
        float cur_scale = 0.f, next_scale = 0.f;
        int cur_ends = -1, next_ends = -1;
        auto fetch = [&](int u0) {
          const int u = u0 + lane;
          next_scale = -1.f;
          next_ends = -1;
          if (u < my_units) {
            const int64_t v = my_first + (u >> a.unit_shift);
            const int64_t id = __ldg(a.page_ids + v);
            const int doc = __ldg(a.page_docs + v);
            if (id >= 0 && id < a.n_pages) next_scale = __ldg(a.scales + id);
            if ((u & half_mask) == half_mask && doc >= 0 && doc < a.n_docs &&
                (v + 1 >= my_end || __ldg(a.page_docs + v + 1) != doc))
              next_ends = doc;
          }
        };
        fetch(0);
        float best[MT];
#pragma unroll
        for (int m = 0; m < MT; ++m) best[m] = kNegInf;
        uint32_t u = 0;
        bool ok = true;
        for (int t = 0; ok && t < n_tiles; ++t) {
          const int unit0 = t * kUnits;
          if ((unit0 & 31) == 0) {
            cur_scale = next_scale;
            cur_ends = next_ends;
            fetch(unit0 + 32);  // also past the stream's end: another stream may go on
          }
#pragma unroll
          for (int m = 0; m < MT; ++m) {
            if (m >= mt) break;
            const uint32_t slot = u % kSlots;
            ok = mbar_wait(accf_bar(slot), (u / kSlots) & 1u, abort_flag, a.timeout_ns, a.err, 46);
            ok = __all_sync(kAllWarp, ok);
            if (!ok) break;
            ++u;
            tc_fence_after();
            const uint32_t at = tmem + slot * TN + stream * W + (static_cast<uint32_t>(quarter * 32) << 16);
            const int64_t global_chunk = static_cast<int64_t>(m_first + m) * 4 + chunk;
            auto one = [&](int i, float v) {  // box i of the tile is done
              const int from = (unit0 + i) & 31;
              const float scale = __shfl_sync(kAllWarp, cur_scale, from);
              const int ends = __shfl_sync(kAllWarp, cur_ends, from);
              if (!(scale < 0.f)) best[m] = max_nan(best[m], v * scale);
              if (ends >= 0) {
                if (global_chunk < a.n_chunks) {
                  queue[queued * kQueueStride + lane] = best[m] * factor[m * 128];
                  if (lane == queued) my_dest = global_chunk * a.n_docs + ends;
                  if (++queued == kQueue) flush();
                }
                best[m] = kNegInf;
              }
            };
            uint32_t ra[32], rb[32];
            tmem_ld32_async(at, ra);
#pragma unroll
            for (int b = 0; b < W / 32; ++b) {
              uint32_t(&cur)[32] = (b & 1) ? rb : ra;
              uint32_t(&nxt)[32] = (b & 1) ? ra : rb;
              tmem_wait_ld32(cur);
              if (b + 1 < W / 32) {
                tmem_ld32_async(at + 32 * (b + 1), nxt);
              } else {  // the accumulator goes back before its last columns are reduced
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(acce_bar(slot));
              }
              if constexpr (U == 32) {
                one(b, max_columns<32>(cur));
              } else {
                one(2 * b, max_columns<16>(cur));
                one(2 * b + 1, max_columns<16>(cur + 16));
              }
            }
          }
        }
        if (queued) flush();
      }
    }
  }

  // Documents without a table entry: this CTA's share of them.
  const int64_t lo = a.n_docs * range / a.ranges, hi = a.n_docs * (range + 1) / a.ranges;
  for (int64_t doc = lo + threadIdx.x; doc < hi; doc += kThreads) {
    if (clamp_entry(a, __ldg(a.page_offsets + doc)) < clamp_entry(a, __ldg(a.page_offsets + doc + 1))) continue;
    for (int c = m_first * 4; c < (m_first + mt) * 4 && c < a.n_chunks; ++c) a.out[c * a.n_docs + doc] = kNegInf;
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(*tmem_slot, 512);
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

template <int TN, int NC, int U, int MT>
int launch(const CUtensorMap& map, const PagedArgs& a, cudaStream_t st) {
  auto kern = paged_mma_kernel<TN, NC, U, MT>;
  const uint32_t smem = smem_layout(TN, a.mt, a.terms, a.kc, a.stages).total;
  if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem)) != cudaSuccess)
    return TMS_ERR_CUDA;
  kern<<<static_cast<unsigned>(a.groups * a.ranges), kThreads, smem, st>>>(map, a);
  return cuda_status(cudaGetLastError());
}

template <int TN, int U>
int launch_nc(const CUtensorMap& map, const PagedArgs& a, cudaStream_t st) {
  if (a.n_chunks == 1) return launch<TN, 1, U, 1>(map, a, st);
  if (a.n_chunks == 2) return launch<TN, 2, U, 1>(map, a, st);
  if (a.mt == 1) return launch<TN, 4, U, 1>(map, a, st);
  return launch<TN, 4, U, 4>(map, a, st);
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
  const int64_t nchunk = (nq + 31) / 32;
  if (page_capacity * ((page_size + 31) / 32) >= (int64_t(1) << 30)) return TMS_ERR_UNSUPPORTED;
  if (n_docs >= (int64_t(1) << 31) || n_pages >= (int64_t(1) << 27) ||
      n_pages * page_size >= (int64_t(1) << 31) || nq >= (int64_t(1) << 24) ||
      n_queries >= (int64_t(1) << 24) || n_queries * nchunk >= (int64_t(1) << 24))
    return TMS_ERR_UNSUPPORTED;
  if (!Q || !out || !page_offsets || (page_capacity > 0 && (!page_ids || !page_docs)) ||
      (n_pages > 0 && (!codes || !scales)))
    return TMS_ERR_INVALID;
  if ((reinterpret_cast<uintptr_t>(Q) & 15) || (reinterpret_cast<uintptr_t>(codes) & 15)) return TMS_ERR_INVALID;
  const size_t need = tms_paged_workspace_size(n_queries, nq, n_docs);
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
  a.n_queries = n_queries;
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
  a.out = need ? static_cast<float*>(workspace) : out;
  a.err = dev->err_word;
  a.timeout_ns = wait_timeout_ns();
  a.debug_flags = debug_flags();

  // Tiles of 256 tokens keep the MMA's operand reads (A again for every tile) under the
  // shared-memory port's rate; with two K chunks only 128 leave room for the query terms.
  const int TN = a.kc == 1 ? 256 : 128;
  const int most_mt = a.n_mtiles < 4 ? a.n_mtiles : 4;
  const uint32_t room = static_cast<uint32_t>(dev->max_smem_optin);
  for (a.mt = most_mt; a.mt > 1; --a.mt)
    if (smem_layout(TN, a.mt, a.terms, a.kc, 2).total <= room) break;
  a.groups = (a.n_mtiles + a.mt - 1) / a.mt;
  a.mt = (a.n_mtiles + a.groups - 1) / a.groups;
  a.stages = 2;
  while (a.stages < kMaxStages && smem_layout(TN, a.mt, a.terms, a.kc, a.stages + 1).total <= room) ++a.stages;
  int64_t ranges = dev->num_sms / a.groups;
  if (ranges > page_capacity) ranges = page_capacity;
  a.ranges = static_cast<int>(ranges < 1 ? 1 : ranges);

  CUtensorMap map;
  int rc = encode_tmap_2d(&map, CU_TENSOR_MAP_DATA_TYPE_UINT8, codes, static_cast<uint64_t>(d),
                          static_cast<uint64_t>(n_pages * page_size), static_cast<uint64_t>(d), 128,
                          static_cast<uint32_t>(U));
  if (rc != TMS_OK) return rc;
  if (TN == 256) rc = U == 16 ? launch_nc<256, 16>(map, a, st) : launch_nc<256, 32>(map, a, st);
  else rc = U == 16 ? launch_nc<128, 16>(map, a, st) : launch_nc<128, 32>(map, a, st);
  if (rc != TMS_OK || nchunk == 1) return rc;
  paged_sum_kernel<<<blocks_for(n_queries * n_docs, dev), 256, 0, st>>>(a.out, out, n_queries, n_docs, a.nchunk);
  return cuda_status(cudaGetLastError());
}
