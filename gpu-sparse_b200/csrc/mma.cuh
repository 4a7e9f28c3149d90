// Matrix products on the fifth-generation tensor cores (sm_100a) for the vocabulary head.
//
//   acc[m, n] = sum over k of A[m, k] * B[n, k]      (16-bit operands, fp32 accumulators)
//
// A pair of CTAs (one cluster, two SMs) works on one output tile of 256 x 256 at a time: each
// CTA holds half of A's rows and half of B's and computes its 128 rows of the tile against all
// of B (tcgen05 cta_group::2), so every operand byte that reaches an SM feeds twice the products
// it would feed alone.  Pairs are persistent and walk a list of tiles; what happens to a finished
// tile is the job's epilogue, which reads the accumulators from tensor memory and reduces or
// stores them, so no product has to be written out to be used.  Warp roles:
//   warp 0      TMA producer: one lane streams this CTA's operand halves of every 64-deep step
//               through a ring of shared-memory stages; the copies of both CTAs signal the
//               first CTA's barrier
//   warp 1      MMA issuer (first CTA of the pair only): one lane issues four 16-deep
//               tcgen05.mma per stage for both CTAs
//   warp 2      owns the tensor memory (two accumulators of 128 x 256 per CTA, so that the
//               products of a tile run while the epilogue drains the one before)
//   warps 4-11  epilogue: thread i of each group of four warps owns accumulator row i (tensor-
//               memory lane i), the first group the lower half of the columns, the second the
//               upper; two warps per scheduler hide each other's latencies
// An operand is either K-major (rows of A or B contiguous along k) or MN-major (contiguous
// along m or n); both are read in place with 128-byte swizzled boxes, so no transposed copy
// is ever made.
//
// What bounds it (B200, D = 768): with an epilogue that does nothing 4096 x 30522 logits take
// 117 us, 1.64 PFLOP/s; the library's large products reach 1.67 in a burst.  In steps of
// milliseconds the power limit takes the clock down (library: 1.39).  Operands come
// from L2 at 10 TB/s; the logits of 16384 rows took 3.4 % less with half of A's loads left out and
// 5.7 % less with all of them.
//
// Every wait is bounded.  A role whose wait runs out raises its CTA's fault flag and stops; the
// epilogue then sees NaN accumulators for that and all later tiles of the CTA, so the results
// show it.  Before a pair ends, its CTAs tell each other how far they came, and whatever is still
// on its way to one of them (copies, arrivals) is waited for there (wind_down).
//
// A job type provides
//   kStages, kScratch            depth of the operand ring, bytes of epilogue scratch
//   Walk walk(pair, pairs)       per-thread view of a pair's tile list
//   Walk::next(Tile&)            the next tile, false past the end
//   Epi epi()                    per-thread epilogue state; per tile, begin() is called while its
//                                products run (loads that they hide) and tile() when they are done
#pragma once
#include "common.cuh"

#include <cuda.h>

namespace gsp {
namespace mm {

constexpr int kRows = 128;               // rows of A per CTA
constexpr int kBM = 2 * kRows;           // rows of A per tile
constexpr int kBN = 256;                 // most rows of B per tile
constexpr int kBK = 64;                  // depth of one stage: 128 bytes of a 16-bit operand
constexpr int kEpiWarp0 = 4;             // first epilogue warp (a multiple of 4: warp % 4 is
                                         // the tensor-memory quarter it may read)
constexpr int kEpiWarps = 8;
constexpr int kThreads = 32 * (kEpiWarp0 + kEpiWarps);
constexpr int kABytes = kRows * kBK * 2;
constexpr int kBBytes = kBN / 2 * kBK * 2;
constexpr int kStageBytes = kABytes + kBBytes;
constexpr int kTmemCols = 2 * kBN;
constexpr int32_t kTailPolls = 1 << 24;  // of the waits for what has been issued already
template <class Job>
constexpr int smem_bytes() {
  return Job::kStages * kStageBytes + Job::kScratch + 256 + 1024;   // + barriers, alignment slack
}

// One output tile.  a/b select the operand maps; a0/b0 are the tile's first row (m or n) of
// each operand, ak/bk the first k of it.
struct Tile {
  int32_t a, b;          // operand map indices
  int32_t a0, b0;
  int32_t ak, bk;
  int32_t nk;            // 64-deep steps; 0: the product is zero
  bool a_mn, b_mn;       // operand is MN-major
  bool b_cut;            // an MN-major B whose rows are no whole blocks of 64 (2D map, a copy per
                         // block; else, and for A, a 3D map [block][k][64] and one copy)
  bool a_stream;         // A passes through L2 (B, and else A, is kept there)
  int32_t a_rows;        // rows of a K-major A's boxes, at most kRows; fewer: A has no more, they
                         // are the first CTA's, and the other rows of the tile are not read
  int32_t bn;            // rows of B of this tile (a K-major B's map has boxes of half of it)
  int32_t x, y, flags;   // the job's own coordinates
};

// ---- PTX ---------------------------------------------------------------------------------
// Returns once the kernel before this one in the stream has finished and its writes are visible
// (see launch() in vocab.cuh); only then may the kernel after this one be set up, so that no more
// than two of a chain are in flight.
__device__ __forceinline__ void after_previous() {
  asm volatile("griddepcontrol.wait;\n\tgriddepcontrol.launch_dependents;" ::: "memory");
}
__device__ __forceinline__ uint32_t su32(const void* p) { return uint32_t(__cvta_generic_to_shared(p)); }
__device__ __forceinline__ void bar_init(uint64_t* b, uint32_t n) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(su32(b)), "r"(n));
}
__device__ __forceinline__ void bar_expect(uint64_t* b, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(su32(b)), "r"(bytes) : "memory");
}
__device__ __forceinline__ void bar_arrive(uint64_t* b) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(su32(b)) : "memory");
}
__device__ __forceinline__ bool bar_test(uint64_t* b, uint32_t parity) {
  uint32_t ok;
  asm volatile("{ .reg .pred p; mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2; selp.u32 %0, 1, 0, p; }"
               : "=r"(ok)
               : "r"(su32(b)), "r"(parity)
               : "memory");
  return ok != 0;
}
// false if `limit` polls ran out or the CTA has faulted
__device__ __forceinline__ bool bar_wait(uint64_t* b, uint32_t parity, int32_t limit, volatile int32_t* fault) {
  for (int32_t i = 0; i <= limit; ++i) {
    if (bar_test(b, parity)) return true;
    if ((i & 63) == 63 && *fault) return false;
  }
  return false;
}
// waits for what is on its way already (a bound of its own: the caller's limit may be 0)
__device__ __forceinline__ void bar_land(uint64_t* b, uint32_t parity) {
  for (int32_t i = 0; i < kTailPolls; ++i) {
    if (bar_test(b, parity)) return;
    __nanosleep(32);
  }
}
// the last `depth` of `count` phases of a ring of barriers (phase i is barrier i % depth's
// (i / depth)-th)
__device__ __forceinline__ void bars_land(uint64_t* ring, int32_t depth, int32_t count) {
  for (int32_t i = count > depth ? count - depth : 0; i < count; ++i) bar_land(ring + i % depth, uint32_t(i / depth) & 1);
}
// counts bytes at a barrier that no copy brings
__device__ __forceinline__ void bar_complete(uint64_t* b, uint32_t bytes) {
  asm volatile("mbarrier.complete_tx.relaxed.cta.shared::cta.b64 [%0], %1;" ::"r"(su32(b)), "r"(bytes) : "memory");
}
// the address of a CTA's copy of a shared-memory object of this CTA
__device__ __forceinline__ uint32_t in_cta(const void* p, int32_t rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(su32(p)), "r"(rank));
  return r;
}
__device__ __forceinline__ uint32_t in_first_cta(const void* p) { return in_cta(p, 0); }
__device__ __forceinline__ void store_remote(uint32_t cluster_addr, int32_t v) {
  asm volatile("st.shared::cluster.b32 [%0], %1;" ::"r"(cluster_addr), "r"(v) : "memory");
}
__device__ __forceinline__ uint32_t cta_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release;\n\tbarrier.cluster.wait.acquire;" ::: "memory");
}
// relaxed: what it orders is tensor memory (the tcgen05 fences do that); a release would wait for
// all stores in flight, which measured 14 % of the logits' gradient
__device__ __forceinline__ void arrive_remote(uint32_t cluster_addr) {
  asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(cluster_addr) : "memory");
}
// L2 policies of an operand's reads: kept (weights and states, read over and over) or first to
// go (a matrix that streams through)
__device__ __forceinline__ uint64_t l2_policy(bool keep) {
  uint64_t p;
  if (keep) {
    asm("createpolicy.fractional.L2::evict_last.b64 %0, 1.0;" : "=l"(p));
  } else {
    asm("createpolicy.fractional.L2::evict_first.b64 %0, 1.0;" : "=l"(p));
  }
  return p;
}
// this CTA's copy of a box, counted at the barrier `bar` (a cluster address, in either CTA)
__device__ __forceinline__ void tma_2d(void* dst, const CUtensorMap* map, int32_t x, int32_t y, uint32_t bar, uint64_t policy) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes.cta_group::2.L2::cache_hint [%0], "
      "[%1, {%2, %3}], [%4], %5;" ::"r"(su32(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(bar), "l"(policy)
      : "memory");
}
__device__ __forceinline__ void tma_3d(void* dst, const CUtensorMap* map, int32_t x, int32_t y, int32_t z, uint32_t bar,
                                       uint64_t policy) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes.cta_group::2.L2::cache_hint [%0], "
      "[%1, {%2, %3, %4}], [%5], %6;" ::"r"(su32(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(bar), "l"(policy)
      : "memory");
}
// Stores a box of shared memory (128-byte swizzled rows) where the map says; the executing
// thread owns the copy's group.
__device__ __forceinline__ void tma_store_2d(const CUtensorMap* map, const void* src, int32_t x, int32_t y) {
  asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%1, %2}], [%3];" ::"l"(
                   reinterpret_cast<uint64_t>(map)),
               "r"(x), "r"(y), "r"(su32(src))
               : "memory");
  asm volatile("cp.async.bulk.commit_group;" ::: "memory");
}
__device__ __forceinline__ void tma_store_wait_read() { asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory"); }
__device__ __forceinline__ void tma_store_wait() { asm volatile("cp.async.bulk.wait_group 0;" ::: "memory"); }
// this thread's shared-memory writes before it become visible to bulk copies after it
__device__ __forceinline__ void fence_async() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
// arrives once the products issued so far are done, at this CTA's barrier or at both CTAs'
__device__ __forceinline__ void commit_own(uint64_t* bar) {
  asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(su32(bar)) : "memory");
}
__device__ __forceinline__ void commit_both(uint64_t* bar) {
  asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(
                   su32(bar)),
               "h"(uint16_t(3))
               : "memory");
}
__device__ __forceinline__ void mma_f16(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{ .reg .pred p; setp.ne.b32 p, %4, 0; tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p; }" ::"r"(d), "l"(a),
      "l"(b), "r"(idesc), "r"(acc));
}
// thread i of the warp gets columns c .. c+31 of tensor-memory lane (quarter base + i)
__device__ __forceinline__ void tmem_ld32(uint32_t addr, float (&v)[32]) {
  uint32_t r[32];
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
        "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(addr));
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
  for (int j = 0; j < 32; ++j) v[j] = __uint_as_float(r[j]);
}

// Shared-memory matrix descriptors (128-byte swizzle, offsets in 16-byte units, version bit
// 46).  K-major: a box is rows of 64 k (128 bytes), 8-row groups 1024 bytes apart; a 16-deep
// step advances 32 bytes.  MN-major: a box is 64 k-rows of 64 m/n (128 bytes), boxes of 64
// m/n 8192 bytes apart (leading offset), 8-k groups 1024 bytes apart (stride offset); a
// 16-deep step advances 2048 bytes.
__device__ __forceinline__ uint64_t desc(uint32_t addr, bool mn) {
  const uint64_t lead = mn ? (8192 >> 4) : 1;
  return uint64_t((addr >> 4) & 0x3FFF) | (lead << 16) | (uint64_t(1024 >> 4) << 32) | (1ull << 46) | (2ull << 61);
}
// fp32 accumulators, A and B both bf16 or both fp16
__device__ __forceinline__ uint32_t inst_desc(bool bf16, bool a_mn, bool b_mn, int32_t bn) {
  const uint32_t ty = bf16 ? 1u : 0u;
  return (1u << 4) | (ty << 7) | (ty << 10) | (uint32_t(a_mn) << 15) | (uint32_t(b_mn) << 16) |
         (uint32_t(bn >> 3) << 17) | (uint32_t(kBM >> 4) << 24);
}

// A finished tile's accumulators as an epilogue warp sees them: row `row` of the tile's A, and
// of the columns [c_lo, c_hi).
struct Acc {
  uint32_t taddr;        // this warp's quarter of the tile's tensor-memory columns
  uint32_t free_bar;     // counts the warps that are done with the accumulators
  bool zero, bad;        // nk == 0; a wait ran out
  unsigned char* scratch;
  int warp, lane;        // epilogue warp 0..7
  int half, lane_row;    // column half; row of this CTA's 128
  int buf;               // alternates from tile to tile
  int32_t rank, row, c_lo, c_hi;
  __device__ __forceinline__ void ld32(int32_t c, float (&v)[32]) const {
    if (bad || zero) {
      const float f = bad ? __uint_as_float(0x7FC00000u) : 0.0f;
#pragma unroll
      for (int j = 0; j < 32; ++j) v[j] = f;
    } else {
      __syncwarp();          // the load is a warp's: lanes may have parted since the last one
      tmem_ld32(taddr + uint32_t(c), v);
    }
  }
  // every epilogue warp, once per tile, after its last ld32: the accumulators may be overwritten
  __device__ __forceinline__ void release() const {
    fence_before();
    __syncwarp();
    if (lane == 0) arrive_remote(free_bar);
  }
  // this CTA's epilogue warps
  __device__ __forceinline__ void sync() const {
    __syncwarp();
    asm volatile("bar.sync 1, %0;" ::"n"(32 * kEpiWarps) : "memory");
  }
};

// How far a CTA came: stages its producer asked for, stages and tiles whose products were issued
// (the first CTA's; counted as they are issued: counters kept for the end of the loop cost it 2 %,
// 628 instead of 613 us for 64 documents), and whether one of its waits ran out.
struct Progress {
  int32_t issued, fed, tiles, fault;
};

// After a wait has run out in either CTA, by one thread of each: returns once nothing is on its way
// to this CTA's shared memory any more.  A stage is asked for only when the products have read what
// its slot held, so the CTAs are at most kStages apart.  The copies of both count at the first CTA's
// barriers: for a stage that only one of them asked for it makes up the other's part.
template <int kStages>
__device__ __noinline__ void wind_down(uint64_t* full, uint64_t* empty, uint64_t* acc_full, const Progress* progress, int32_t rank,
                                       const Tile& t) {
  const Progress own = progress[0], peer = progress[1], first = progress[rank];
  if (rank == 0) {
    // the second CTA's bytes of a stage: the same for all tiles of a job
    const uint32_t second = uint32_t((!t.a_mn && t.a_rows < kRows ? 0 : kRows) + (t.b_mn ? kBN / 2 : t.bn / 2)) * (kBK * 2);
    for (int32_t i = peer.issued; i < own.issued; ++i) bar_complete(full + i % kStages, second);
    for (int32_t i = own.issued; i < peer.issued; ++i) bar_expect(full + i % kStages, second);
    bars_land(full, kStages, own.issued > peer.issued ? own.issued : peer.issued);
  }
  bars_land(empty, kStages, first.fed);
  bars_land(acc_full, 2, first.tiles);
}

template <class Job>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads, 1) mma_kernel(const __grid_constant__ Job job) {
  constexpr int kStages = Job::kStages;
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  unsigned char* smem =
      reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  unsigned char* scratch = smem + kStages * kStageBytes;
  uint64_t* full = reinterpret_cast<uint64_t*>(scratch + Job::kScratch);   // [kStages], used in the first CTA
  uint64_t* empty = full + kStages;                                        // [kStages]
  uint64_t* acc_full = empty + kStages;                                    // [2]
  uint64_t* acc_empty = acc_full + 2;                                      // [2], used in the first CTA
  uint64_t* drain = acc_empty + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 1);
  Progress* progress = reinterpret_cast<Progress*>(tmem_slot + 2);         // [2], own and the other CTA's
  volatile int32_t *fault = &progress->fault, *fed = &progress->fed, *tiles = &progress->tiles;
  const int wid = threadIdx.x >> 5, lane = lane_id();
  const int32_t limit = job.wait_limit;
  const int32_t rank = int32_t(cta_rank());
  const int32_t pair = int32_t(blockIdx.x) >> 1, pairs = int32_t(gridDim.x) >> 1;

  if (threadIdx.x == 0) {
    for (int i = 0; i < kStages; ++i) {
      bar_init(full + i, 1);
      bar_init(empty + i, 1);
    }
    for (int i = 0; i < 2; ++i) {
      bar_init(acc_full + i, 1);
      bar_init(acc_empty + i, 2 * kEpiWarps);
    }
    bar_init(drain, 1);
    progress[0] = Progress{0, 0, 0, 0};
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (wid == 2) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(su32(tmem_slot)),
                 "r"(kTmemCols));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
  }
  fence_before();
  __syncthreads();
  cluster_sync();
  fence_after();
  after_previous();
  const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(tmem_slot);

  if (wid == 0) {
    if (lane == 0) {
      auto walk = job.walk(pair, pairs);
      const uint64_t keep = l2_policy(true), stream = l2_policy(false);
      Tile t;
      uint32_t it = 0;
      bool ok = true;
      while (ok && walk.next(t)) {
        const uint64_t pol_a = t.a_stream ? stream : keep;
        const CUtensorMap* ma = &job.maps[t.a];
        const CUtensorMap* mb = &job.maps[t.b];
        const int32_t nb = t.bn / 2, a0 = t.a0 + rank * kRows, b0 = t.b0 + rank * nb;
        const bool few = !t.a_mn && t.a_rows < kRows;
        // (an MN-major B is always read 128 rows wide: past D there are zeros)
        const uint32_t bytes = uint32_t((few ? t.a_rows : 2 * kRows) + (t.b_mn ? kBN : 2 * nb)) * (kBK * 2);
        for (int32_t k = 0; k < t.nk; ++k, ++it) {
          const uint32_t s = it % kStages, n = it / kStages;
          if (n > 0) ok = bar_wait(empty + s, (n - 1) & 1, limit, fault);
          if (!ok) break;
          unsigned char* as = smem + s * kStageBytes;
          unsigned char* bs = as + kABytes;
          const uint32_t bar = in_first_cta(full + s);
          if (rank == 0) bar_expect(full + s, bytes);
          if (!t.a_mn) {
            if (!few || rank == 0) tma_2d(as, ma, t.ak + k * kBK, a0, bar, pol_a);
          } else {
            tma_3d(as, ma, 0, t.ak + k * kBK, a0 / 64, bar, pol_a);
          }
          if (!t.b_mn) {
            tma_2d(bs, mb, t.bk + k * kBK, b0, bar, keep);
          } else if (!t.b_cut) {
            tma_3d(bs, mb, 0, t.bk + k * kBK, b0 / 64, bar, keep);
          } else {
            for (int32_t j = 0; j < kBN / 128; ++j) tma_2d(bs + j * 8192, mb, b0 + j * 64, t.bk + k * kBK, bar, keep);
          }
        }
      }
      progress->issued = int32_t(it);
      // the last stages are handed back too: their copies have landed then, and the arrivals that
      // say so find this CTA's barriers still there
      for (uint32_t i = it > uint32_t(kStages) ? it - kStages : 0; ok && i < it; ++i)
        ok = bar_wait(empty + i % kStages, (i / kStages) & 1, kTailPolls, fault);
      if (!ok) *fault = 1;
    }
  } else if (wid == 1) {
    if (lane == 0 && rank == 0) {
      auto walk = job.walk(pair, pairs);
      Tile t;
      uint32_t it = 0;
      bool ok = true;
      for (int32_t i = 0; ok && walk.next(t); ++i) {
        const int32_t buf = i & 1, use = i >> 1;
        if (use > 0) ok = bar_wait(acc_empty + buf, (use - 1) & 1, limit, fault);
        if (!ok) break;
        fence_after();
        const uint32_t d = tmem + uint32_t(buf * kBN);
        const uint32_t id = inst_desc(job.bf16 != 0, t.a_mn, t.b_mn, t.bn);
        const uint64_t step_a = t.a_mn ? (2048 >> 4) : (32 >> 4), step_b = t.b_mn ? (2048 >> 4) : (32 >> 4);
        for (int32_t k = 0; k < t.nk; ++k, ++it) {
          const uint32_t s = it % kStages, n = it / kStages;
          ok = bar_wait(full + s, n & 1, limit, fault);
          if (!ok) break;
          fence_after();
          const uint32_t as = su32(smem + s * kStageBytes);
          const uint64_t da = desc(as, t.a_mn), db = desc(as + kABytes, t.b_mn);
#pragma unroll
          for (int q = 0; q < kBK / 16; ++q) mma_f16(d, da + q * step_a, db + q * step_b, id, (k > 0 || q > 0) ? 1u : 0u);
          commit_both(empty + s);
          *fed = int32_t(it) + 1;
        }
        if (!ok) break;
        commit_both(acc_full + buf);
        *tiles = i + 1;
      }
      if (!ok) *fault = 1;
      commit_own(drain);          // every product issued has finished before the memory is given back
      bar_land(drain, 0);
    }
  } else if (wid >= kEpiWarp0) {
    auto walk = job.walk(pair, pairs);
    auto epi = job.epi();
    Tile t;
    Acc acc;
    acc.warp = wid - kEpiWarp0;
    acc.lane = lane;
    acc.half = acc.warp >> 2;
    acc.lane_row = (acc.warp & 3) * 32 + lane;
    acc.rank = rank;
    acc.scratch = scratch;
    bool ok = true;
    for (int32_t i = 0; walk.next(t); ++i) {
      const int32_t buf = i & 1, use = i >> 1;
      acc.buf = buf;
      acc.row = t.a0 + rank * kRows + acc.lane_row;
      acc.c_lo = acc.half * (t.bn / 2);
      acc.c_hi = acc.c_lo + t.bn / 2;
      epi.begin(job, t, acc);
      if (ok) {
        ok = bar_wait(acc_full + buf, use & 1, limit, fault);
        if (!ok) *fault = 1;
        ok = __all_sync(FULL, ok);
      }
      fence_after();
      acc.taddr = tmem + (uint32_t(32 * (acc.warp & 3)) << 16) + uint32_t(buf * kBN);
      acc.free_bar = in_first_cta(acc_empty + buf);
      acc.zero = t.nk == 0;
      acc.bad = !ok;
      epi.tile(job, t, acc);
    }
  }
  __syncwarp();
  fence_before();
  __syncthreads();
  if (threadIdx.x == 0) {
    const uint32_t to = in_cta(progress + 1, rank ^ 1);
    store_remote(to, progress->issued);
    store_remote(to + 4, progress->fed);
    store_remote(to + 8, progress->tiles);
    store_remote(to + 12, progress->fault);
  }
  cluster_sync();         // neither CTA's memory goes away while the other may still use it
  if (progress[0].fault | progress[1].fault) {      // both CTAs see both
    if (threadIdx.x == 0) {
      auto walk = job.walk(pair, pairs);
      Tile t;
      if (walk.next(t)) wind_down<kStages>(full, empty, acc_full, progress, rank, t);
    }
    __syncwarp();
    cluster_sync();
  }
  if (wid == 2) {
    fence_after();
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kTmemCols));
  }
}

// CTAs of a launch: all pairs of SMs
inline int pair_ctas() { return num_sms() & ~1; }

}  // namespace mm
}  // namespace gsp
