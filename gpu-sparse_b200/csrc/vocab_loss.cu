// Softmax losses over the vocabulary without its logits: cross entropy and distillation from
// a teacher's top scores.
//
// For a row t with logits s[v] and target distribution q (one entry for cross entropy, the
// teacher's entries for distillation), with c = log2(e) / tau and z = c s:
//   lse2 = log2 sum_v 2^z[v],   loss = tau^2 (sum_j q_j log q_j + ln 2 (lse2 - sum_j q_j z_j))
//   dloss/ds[v] = tau (2^(z[v] - lse2) - q[v])
//
// Forward.  The tiles (256 rows x 256 vocabulary rows) of all rows are one long list, row
// block by row block, cut into equal shares, one per pair of CTAs, so every SM has the same work
// whatever the sizes.  The two epilogue threads that own a row (a column half each) carry its
// running maximum, sum and target dot product in registers along the share and write them once
// per row block; a second kernel joins the partial results (in share order) and sums the losses.
// Bound by the products (V = 30522, D = 768: 16384 rows 528 us, 1.45 PFLOP/s; one row 15 us, of
// which 7 are W's bytes).  With a small D it is the epilogue: 64 us for 4096 rows at D = 64, where
// the exponentials alone are 27 (16 a cycle and SM); the rest is the latency of two epilogue warps
// per scheduler.  The sums take ex2.approx (2^-22 relative), which leaves a loss off by 3e-7.
//
// Backward.  Per piece of the vocabulary: the logits' tiles again, whose epilogue turns them
// into P = gradient of the logits, rounded once to 16 bits, then the two products of
// vocab.cu.  A piece is as large as 512 MiB of P allow, since the products' tile lists want
// to be long; P makes one trip through memory, which the products' arithmetic hides.  The logits'
// pass is bound by its epilogue: 624 us for 16384 rows (P leaves by TMA: 711 instead of 771 us
// with plain stores at that step), and with D = 64 still 130 of the 164 us that 4096 rows take
// with D = 768.  d_bias sums the unrounded P (a warp's 32 x 32 block through shared memory, then
// the row blocks).
//   P is scaled so that the largest row coefficient is 1 in bf16, where a target's softmax - 1 is
// then -1 or close and rounds to next to nothing, and 2^14 in fp16, whose range would lose
// gradients of 1e-8; the products' epilogue takes the scale out in fp32.  Rounding P to 16 bits is
// what lets the products run at the 16-bit rate; gradients of 4096 distilled rows are off by 0.0023
// of their norm in bf16 and those of 500 rows by 0.00029 in fp16, where rounding the exact ones
// costs 0.0017 and 0.00021.  For up to 128 rows P is held in two parts (see low_rows).
#include "vocab.cuh"

namespace gsp {
namespace vocab {
namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr int kFirst = 1, kLast = 2;

struct Lists {             // target entries
  const int32_t* tgt;      // cross entropy: one per packed row
  const int4* hit;         // distillation (see State)
  const int32_t* off;
  float* pz;               // distillation, forward (see Teacher)
  int64_t K, buckets;
  int32_t shift;
};
Lists lists_of(const State& s, bool list, float* pz) {
  return list ? Lists{nullptr, s.hit, s.off, pz, s.K, s.buckets, s.bucket_shift} : Lists{s.tgt, nullptr, nullptr, nullptr, 0, 0, 0};
}
// A teacher's rows while the forward pass works on them (null for cross entropy).
struct Teacher {
  int32_t* cnt;       // [T] entries of every row
  float* ent;         // [T] sum p log p
  int2* entry;        // [T, K] (id, probability's bits), ids distinct
  float* pz;          // [Tp, K] by packed row: probability x logit of every entry
  uint8_t* flag;      // [T] row takes part
};

// ---- distillation: a teacher row's probabilities, ids listed twice joined -----------------
// A CTA per row.  The ids go into a hash table in shared memory (linear probing, at most half
// full); an id belongs to the first entry that lists it, which adds up the others' probabilities
// in the order they are listed.  Bound by latency: 4096 rows of 100 entries 25 us, 500 rows of
// 1000 17 us.
constexpr int kTeacherThreads = 512;      // a thread per entry, if possible: the work is latency
struct TeacherSlot {
  int32_t id, first, times;
};
__global__ void __launch_bounds__(kTeacherThreads)
teacher_kernel(const float* __restrict__ scores, const int64_t* __restrict__ in_ids, int32_t K, int32_t log_slots, int64_t V,
               float inv_tau, const Teacher s) {
  mm::after_previous();
  extern __shared__ TeacherSlot slot[];          // [1 << log_slots], then ids [K], p [K]
  const int32_t slots = 1 << log_slots;
  int32_t* id = reinterpret_cast<int32_t*>(slot + slots);      // then the entry's slot; -1: left out
  float* p = reinterpret_cast<float*>(id + K);
  __shared__ float red[kTeacherThreads / 32];
  __shared__ int32_t wcount[kTeacherThreads / 32];
  const int64_t t = blockIdx.x;
  const int threads = blockDim.x, warps = threads >> 5, tid = threadIdx.x, wid = tid >> 5, lane = tid & 31;
  auto reduce = [&](float v, bool is_max) {
    for (int o = 16; o > 0; o >>= 1) {
      const float u = __shfl_xor_sync(FULL, v, o);
      v = is_max ? fmaxf(v, u) : v + u;
    }
    __syncthreads();
    if (lane == 0) red[wid] = v;
    __syncthreads();
    v = red[0];
    for (int i = 1; i < warps; ++i) v = is_max ? fmaxf(v, red[i]) : v + red[i];
    return v;
  };
  for (int32_t i = tid; i < slots; i += threads) slot[i] = TeacherSlot{-1, kNoId, 0};
  float mx = neg_inf();
  for (int32_t j = tid; j < K; j += threads) {
    const int64_t v = in_ids[t * K + j];
    const float x = scores[t * K + j];
    const bool in = v >= 0 && v < V && x != neg_inf();
    id[j] = in ? int32_t(v) : -1;
    p[j] = x;
    if (in) mx = fmaxf(mx, x);
  }
  mx = reduce(mx, true);
  float sum = 0.0f;
  for (int32_t j = tid; j < K; j += threads) {
    if (id[j] < 0) continue;
    const float e = expf((p[j] - mx) * inv_tau);
    p[j] = e;
    sum += e;
    uint32_t h = uint32_t(id[j]) * 2654435761u >> (32 - log_slots);
    for (;;) {                           // ends: there are more slots than entries
      const int32_t was = atomicCAS(&slot[h].id, -1, id[j]);
      if (was == -1 || was == id[j]) break;
      h = (h + 1) & (slots - 1);
    }
    atomicMin(&slot[h].first, j);
    atomicAdd(&slot[h].times, 1);
    id[j] = int32_t(h);                  // from here on the slot, which has the id
  }
  sum = reduce(sum, false);              // (also makes the table visible)
  int32_t n = 0;
  float ent = 0.0f;
  for (int32_t j0 = 0; j0 < K; j0 += threads) {
    const int32_t j = j0 + tid;
    bool head = false;
    float q = 0.0f;
    if (j < K && id[j] >= 0) {
      const TeacherSlot& own = slot[id[j]];
      head = own.first == j;
      if (head) {
        q = p[j];
        if (own.times > 1) {
          for (int32_t i = j + 1; i < K; ++i) q += id[i] == id[j] ? p[i] : 0.0f;
        }
        q /= sum;
        head = q != 0.0f;                // an entry whose probability underflowed adds nothing
        if (head) ent += q * logf(q);
      }
    }
    const uint32_t w = __ballot_sync(FULL, head);
    if (lane == 0) wcount[wid] = __popc(w);
    __syncthreads();
    int32_t at = n;
    for (int i = 0; i < warps; ++i) {
      if (i < wid) at += wcount[i];
      n += wcount[i];
    }
    __syncthreads();
    if (head) s.entry[t * K + at + __popc(w & lanemask_lt())] = make_int2(slot[id[j]].id, __float_as_int(q));
  }
  ent = reduce(ent, false);
  if (tid == 0) {
    s.cnt[t] = n;
    s.ent[t] = ent;
    s.flag[t] = n > 0;
  }
}

// The entries of 32 packed rows (one epilogue warp's) sorted into buckets of the vocabulary (32
// columns), so that the warp finds those of its block side by side, however they are spread over
// the rows.  gridDim.y CTAs per 32 rows: each reads all entries, counts those before its share of
// the buckets and places its own.  The order inside a bucket is the atomics' and shows nowhere:
// every entry has a place of its own in pz and in P.  4096 rows of 100 entries take 8 us, 500 of
// 1000 13 us (22 with one CTA per 32 rows).
constexpr int kBucketThreads = 1024, kBucketAhead = 8, kBucketSplits = 8;
__global__ void __launch_bounds__(kBucketThreads) bucket_kernel(const State s, const Teacher tc) {
  mm::after_previous();
  extern __shared__ int32_t count[];           // [this CTA's buckets]
  __shared__ int32_t part[32];
  const int32_t n = s.head[0], r0 = int32_t(blockIdx.x) * 32;
  if (r0 >= n) return;
  const int32_t all_b = int32_t(s.buckets), tid = threadIdx.x, wid = tid >> 5, lane = tid & 31;
  const int32_t b_lo = share_lo(all_b, gridDim.y, blockIdx.y), nb = share_lo(all_b, gridDim.y, blockIdx.y + 1) - b_lo;
  for (int32_t b = tid; b < nb; b += kBucketThreads) count[b] = 0;
  __syncthreads();
  // a warp per row, kBucketAhead entries per lane in flight
  const bool live = r0 + wid < n;
  const int64_t orig = live ? s.map[r0 + wid] : 0;
  const int32_t c = live ? tc.cnt[orig] : 0;
  const int2* entry = tc.entry + orig * s.K;
  int32_t before_mine = 0;
  for (int32_t i0 = lane; i0 < c; i0 += 32 * kBucketAhead) {
    int32_t id[kBucketAhead];
#pragma unroll
    for (int k = 0; k < kBucketAhead; ++k) id[k] = i0 + 32 * k < c ? entry[i0 + 32 * k].x : -1;
#pragma unroll
    for (int k = 0; k < kBucketAhead; ++k) {
      const int32_t b = (id[k] >> s.bucket_shift) - b_lo;
      if (id[k] >= 0 && b < 0) ++before_mine;
      if (id[k] >= 0 && b >= 0 && b < nb) atomicAdd(count + b, 1);
    }
  }
  before_mine = __reduce_add_sync(FULL, before_mine);
  if (lane == 0) part[wid] = before_mine;
  __syncthreads();
  int32_t base = __reduce_add_sync(FULL, part[lane]);
  __syncthreads();
  // exclusive scan
  int32_t* off = s.off + int64_t(blockIdx.x) * (all_b + 1) + b_lo;
  for (int32_t b0 = 0; b0 < nb; b0 += kBucketThreads) {
    const int32_t b = b0 + tid;
    const int32_t v = b < nb ? count[b] : 0;
    int32_t x = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int32_t u = __shfl_up_sync(FULL, x, o);
      if (lane >= o) x += u;
    }
    if (lane == 31) part[wid] = x;
    __syncthreads();
    const int32_t w = part[lane];
    const int32_t before = __reduce_add_sync(FULL, lane < wid ? w : 0), all = __reduce_add_sync(FULL, w);
    if (b < nb) off[b] = count[b] = base + before + x - v;
    base += all;
    __syncthreads();
  }
  if (tid == 0 && blockIdx.y == gridDim.y - 1) off[nb] = base;
  int4* hit = s.hit + int64_t(r0) * s.K;
  for (int32_t i0 = lane; i0 < c; i0 += 32 * kBucketAhead) {
    int2 e[kBucketAhead];
#pragma unroll
    for (int k = 0; k < kBucketAhead; ++k) e[k] = i0 + 32 * k < c ? entry[i0 + 32 * k] : make_int2(-1, 0);
#pragma unroll
    for (int k = 0; k < kBucketAhead; ++k) {
      const int32_t b = (e[k].x >> s.bucket_shift) - b_lo;
      if (e[k].x >= 0 && b >= 0 && b < nb) hit[atomicAdd(count + b, 1)] = make_int4(e[k].x, wid, e[k].y, i0 + 32 * k);
    }
  }
}

// The entries of a warp's 32 rows x half a tile, 32 at a time in registers, one per lane: the first
// (usually all) loaded while products run, others when a block of 32 columns gets to them.  (With
// one bucket per half tile, looked through for every 32 columns, the logits' gradient of 500 rows
// of 1000 entries over 100000 words took 84 us instead of 75, their forward pass 64 instead of 54.)
struct Hits {
  const int4* first;
  int32_t edge;         // lane i: where the half's i-th bucket begins
  int32_t at;           // the 32 that e holds
  int32_t v_half, shift;
  int4 e;
  __device__ void load(const Lists& l, int32_t row0, int32_t rows, int32_t v0, int lane) {
    edge = at = 0;
    v_half = v0;
    shift = l.shift;
    e.x = kNoId;
    if (row0 >= rows) return;
    const int32_t b = v0 >> l.shift;
    if (lane < 5) edge = (l.off + int64_t(row0 / 32) * (l.buckets + 1))[min(b + lane, int32_t(l.buckets))];
    const int32_t begin = __shfl_sync(FULL, edge, 0);
    edge -= begin;
    first = l.hit + int64_t(row0) * l.K + begin;
    fetch(0, lane);
  }
  __device__ void fetch(int32_t i, int lane) {
    const int32_t n = __shfl_sync(FULL, edge, 4);
    at = i;
    e.x = kNoId;
    if (i + lane < n) e = first[i + lane];
  }
  // f(entry, live) for every 32 entries that have some in [v0, v0 + 32): every lane calls it
  template <typename F>
  __device__ void each(int32_t v0, int lane, F&& f) {
    const int b = (v0 >> shift) - (v_half >> shift);
    const int32_t lo = __shfl_sync(FULL, edge, b), hi = __shfl_sync(FULL, edge, b + 1);
    for (int32_t i = lo & ~31; i < hi; i += 32) {
      if (i != at) fetch(i, lane);
      const bool in = e.x >= v0 && e.x < v0 + 32;
      if (__any_sync(FULL, in)) f(e, in);
    }
  }
};

// This tile's share of bias2 for one warp: loaded by begin() while the products run (a float4
// per lane, the 128 columns of a half), spread to all lanes through shared memory.
struct BiasTile {
  static constexpr int kBytes = mm::kBN / 2 * 4;
  static __device__ void load(const float* bias2, unsigned char* smem, int lane) {
    const float4 b = __ldg(reinterpret_cast<const float4*>(bias2) + lane);
    __syncwarp();
    reinterpret_cast<float4*>(smem)[lane] = b;
    __syncwarp();
  }
};
// z = c s + bias2 of 32 consecutive vocabulary rows
__device__ __forceinline__ void to_z(const float (&v)[32], F2 c, const float* bias, F2 (&z)[16]) {
#pragma unroll
  for (int q = 0; q < 8; ++q) {
    const float4 x = *reinterpret_cast<const float4*>(bias + 4 * q);
    z[2 * q] = fma2(f2(v[4 * q], v[4 * q + 1]), c, f2(x.x, x.y));
    z[2 * q + 1] = fma2(f2(v[4 * q + 2], v[4 * q + 3]), c, f2(x.z, x.w));
  }
}

// ---- forward -----------------------------------------------------------------------------
// Partial results of a (share, row block): [2 column halves][maximum, sum of 2^(z - m),
// sum q z][kBM rows], at index share + row block (which no two of them have in common, since
// along the list one of the two always grows).
constexpr int kPart = 2 * 3 * mm::kBM;
constexpr int kBiasScratch = mm::kEpiWarps * BiasTile::kBytes;
constexpr int kListScratch = mm::kEpiWarps * kBlockBytes;      // a 32 x 32 block per warp

template <bool kList>
struct LossJob {
  static constexpr int kStages = kList ? 5 : 6, kScratch = kBiasScratch + (kList ? kListScratch : 0);
  CUtensorMap maps[2];      // H, W (K-major)
  int32_t wait_limit, bf16;
  const int32_t* head;
  int32_t nt, nk;           // tiles along the vocabulary, steps along D
  int32_t a_rows;
  float c;
  const float* bias2;
  Lists lists;
  float* part;              // [pairs + row blocks][kPart]

  struct Walk {
    int32_t lo, x, hi, nt, nk, a_rows;
    __device__ bool next(mm::Tile& t) {
      if (x >= hi) return false;
      t.a_rows = a_rows;
      t.x = x / nt;
      t.y = x - t.x * nt;
      t.a = 0, t.b = 1;
      t.a0 = t.x * mm::kBM;
      t.b0 = t.y * mm::kBN;
      t.ak = t.bk = 0;
      t.nk = nk;
      t.a_mn = t.b_mn = t.b_cut = t.a_stream = false;
      t.bn = mm::kBN;
      t.flags = (x == lo || t.y == 0 ? kFirst : 0) | (x == hi - 1 || t.y == nt - 1 ? kLast : 0);
      ++x;
      return true;
    }
  };
  __device__ Walk walk(int32_t pair, int32_t pairs) const {
    const int32_t tot = (head[0] + mm::kBM - 1) / mm::kBM * nt, lo = share_lo(tot, pairs, pair);
    return Walk{lo, lo, share_lo(tot, pairs, pair + 1), nt, nk, a_rows};
  }

  struct Epi {
    float m, l, dot;
    int32_t tgt;
    Hits hits;
    __device__ float* bias(const mm::Acc& a) { return reinterpret_cast<float*>(a.scratch + a.warp * BiasTile::kBytes); }
    __device__ void begin(const LossJob& j, const mm::Tile& t, const mm::Acc& a) {
      const int32_t v0 = t.y * mm::kBN + a.c_lo;
      BiasTile::load(j.bias2 + v0, reinterpret_cast<unsigned char*>(bias(a)), a.lane);
      if (t.flags & kFirst) {
        m = neg_inf();
        l = dot = 0.0f;
        if constexpr (!kList) tgt = a.row < j.head[0] ? j.lists.tgt[a.row] : -1;
      }
      if constexpr (kList) hits.load(j.lists, a.row - a.lane, j.head[0], v0, a.lane);
    }
    __device__ void tile(const LossJob& j, const mm::Tile& t, const mm::Acc& a) {
      const float* b = bias(a) - a.c_lo;
      const F2 c2 = f2(j.c, j.c);
#pragma unroll 1
      for (int32_t c0 = a.c_lo; c0 < a.c_hi; c0 += 32) {
        float z[32];
        a.ld32(c0, z);
        if (c0 + 32 == a.c_hi) a.release();
        F2 z2[16];
        to_z(z, c2, b + c0, z2);
#pragma unroll
        for (int k = 0; k < 16; ++k) split(z2[k], z[2 * k], z[2 * k + 1]);
        const int32_t v0 = t.y * mm::kBN + c0;
        if constexpr (kList) {
          float* block = reinterpret_cast<float*>(a.scratch + kBiasScratch + a.warp * kBlockBytes);
          float* pz = j.lists.pz + int64_t(a.row - a.lane) * j.lists.K;
          bool put = false;
          hits.each(v0, a.lane, [&](const int4& e, bool in) {
            if (!put) {
              __syncwarp();
              block_put(block, z, a.lane);
              __syncwarp();
              put = true;
            }
            if (in) pz[e.y * j.lists.K + e.w] = __int_as_float(e.z) * block[e.y * kBlockLd + e.x - v0];
          });
        } else {
          const int32_t d = tgt - v0;
          if (d >= 0 && d < 32) {
#pragma unroll
            for (int k = 0; k < 32; ++k) {
              if (k == d) dot = z[k];
            }
          }
        }
        float x[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) x[k] = max3(z[4 * k], z[4 * k + 1], fmaxf(z[4 * k + 2], z[4 * k + 3]));
        const float cm = fmaxf(max3(x[0], x[1], x[2]), max3(x[3], x[4], max3(x[5], x[6], x[7])));
        if (cm > m) {
          l *= ex2(m - cm);
          m = cm;
        }
        const float base = m == neg_inf() ? 0.0f : -m;
        const F2 base2 = f2(base, base);
        F2 e0 = f2(0.0f, 0.0f), e1 = e0;
#pragma unroll
        for (int k = 0; k < 16; k += 2) {
          float p, q;
          split(add2(z2[k], base2), p, q);
          e0 = add2(e0, f2(ex2(p), ex2(q)));
          split(add2(z2[k + 1], base2), p, q);
          e1 = add2(e1, f2(ex2(p), ex2(q)));
        }
        float p, q;
        split(add2(e0, e1), p, q);
        l += p + q;
      }
      if (t.flags & kLast) {
        float* o = j.part + (int64_t(blockIdx.x >> 1) + t.x) * kPart + a.half * 3 * mm::kBM + a.rank * mm::kRows + a.lane_row;
        o[0] = m;
        o[mm::kBM] = l;
        o[2 * mm::kBM] = dot;
      }
    }
  };
  __device__ Epi epi() const { return Epi{}; }
};

// Joins a row's partial results and sums the losses.  A warp per row, a lane per partial result
// (a single row has two from every pair), joined in a fixed tree.  The blocks' sums are added by
// whichever block finishes last, in block order.
constexpr int kJoinRows = 8;
struct RowSum {
  float m, l, dot;
  __device__ void add(float pm, float pl, float pd) {
    const float nm = fmaxf(m, pm), base = nm == neg_inf() ? 0.0f : nm;
    l = l * ex2(m - base) + pl * ex2(pm - base);
    m = nm;
    dot += pd;
  }
};
__global__ void __launch_bounds__(32 * kJoinRows)
join_kernel(int32_t* head, const int32_t* map, const float* part, int32_t nt, int32_t pairs, const Teacher tc, int64_t K,
            float tau2, int32_t reduction, float* lse2, double* sums, float* loss) {
  mm::after_previous();
  __shared__ double red[kJoinRows];
  __shared__ bool last;
  const int32_t n = head[0], wid = threadIdx.x >> 5, lane = lane_id();
  const int32_t r = int32_t(blockIdx.x) * kJoinRows + wid, mb = r / mm::kBM;
  double mine = 0.0;
  if (r < n) {
    const int32_t tot = (n + mm::kBM - 1) / mm::kBM * nt;
    const int32_t c0 = share_of(tot, pairs, mb * nt), parts = 2 * (share_of(tot, pairs, (mb + 1) * nt - 1) + 1 - c0);
    const int32_t orig = map[r];
    RowSum t{neg_inf(), 0.0f, 0.0f};
    if (tc.pz) {
      const int32_t c = tc.cnt[orig];
      for (int32_t i = lane; i < c; i += 32) t.dot += tc.pz[int64_t(r) * K + i];
    }
    for (int32_t i0 = 0; i0 < parts; i0 += 160) {        // five loads of each kind in flight
      float pm[5], pl[5], pd[5];
#pragma unroll
      for (int k = 0; k < 5; ++k) {
        const int32_t i = i0 + 32 * k + lane;
        const float* o = part + int64_t(c0 + (i >> 1) + mb) * kPart + (i & 1) * 3 * mm::kBM + r % mm::kBM;
        const bool in = i < parts;
        pm[k] = in ? o[0] : neg_inf();
        pl[k] = in ? o[mm::kBM] : 0.0f;
        pd[k] = in ? o[2 * mm::kBM] : 0.0f;
      }
#pragma unroll
      for (int k = 0; k < 5; ++k) t.add(pm[k], pl[k], pd[k]);
    }
#pragma unroll
    for (int o = 1; o < 32; o <<= 1)
      t.add(__shfl_xor_sync(FULL, t.m, o), __shfl_xor_sync(FULL, t.l, o), __shfl_xor_sync(FULL, t.dot, o));
    const float z = t.m + log2f(t.l);
    const float v = tau2 * fmaf(z - t.dot, kLn2, tc.pz ? tc.ent[orig] : 0.0f);
    if (lane == 0) {
      lse2[r] = z;
      if (reduction == GSP_REDUCE_NONE) loss[orig] = v;
    }
    mine = double(v);
  }
  if (reduction == GSP_REDUCE_NONE) return;
  if (lane == 0) red[wid] = mine;
  __syncthreads();
  if (threadIdx.x == 0) {
    double s = 0.0;
    for (int i = 0; i < kJoinRows; ++i) s += red[i];
    sums[blockIdx.x] = s;
    __threadfence();
    last = atomicAdd(head + 1, 1) == int32_t(gridDim.x) - 1;
  }
  __syncthreads();
  if (!last) return;
  __threadfence();
  double v = 0.0;
  for (int32_t i = threadIdx.x; i < int32_t(gridDim.x); i += 32 * kJoinRows) v += *reinterpret_cast<volatile double*>(sums + i);
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(FULL, v, o);
  if (lane == 0) red[wid] = v;
  __syncthreads();
  if (threadIdx.x == 0) {
    v = 0.0;
    for (int i = 0; i < kJoinRows; ++i) v += red[i];
    *loss = float(reduction == GSP_REDUCE_MEAN ? v / (n > 0 ? n : 1) : v);
  }
}

// ---- backward ----------------------------------------------------------------------------
// The packed rows a second time from row `low` on (see low_rows); the rows between and up to the
// next 64, which the products read, zero.
__device__ void low_parts(const State& s, int32_t low, int32_t n) {
  const int32_t per = int32_t(s.Dp / 8), end = (low + n + 63) / 64 * 64;
  uint4* h = reinterpret_cast<uint4*>(s.h);
#pragma unroll 4
  for (int32_t i = n * per + threadIdx.x; i < end * per; i += 1024)
    h[i] = i >= low * per && i < (low + n) * per ? h[i - low * per] : make_uint4(0, 0, 0, 0);
}

// Row coefficients of P: ga[r] = tau * grad_loss (divided by the rows of a mean) over their
// largest finite size; lse2 of the padding rows +inf, so that their P is 0.  One CTA; the others
// zero d_hidden.
__global__ void __launch_bounds__(1024)
grad_rows_kernel(State s, const float* grad_loss, int32_t reduction, float tau, int32_t bf16, int32_t low, float* ga,
                 float* scale, void* d_hidden, int64_t hidden_bytes) {
  mm::after_previous();
  __shared__ float red[32];
  if (blockIdx.x > 0) {
    zero_share(d_hidden, hidden_bytes, int64_t(blockIdx.x) - 1, int64_t(gridDim.x) - 1);
    return;
  }
  const int32_t n = s.head[0];
  if (low > 0) low_parts(s, low, n);
  const int32_t np = (n + kRowPad - 1) / kRowPad * kRowPad;
  const float mul = tau / float(reduction == GSP_REDUCE_MEAN ? (n > 0 ? n : 1) : 1);
  float gmax = 0.0f;
  if (reduction == GSP_REDUCE_NONE) {
    for (int32_t r = threadIdx.x; r < n; r += 1024) {
      const float g = fabsf(grad_loss[s.map[r]] * mul);
      if (g < __uint_as_float(0x7F800000u)) gmax = fmaxf(gmax, g);
    }
    for (int o = 16; o > 0; o >>= 1) gmax = fmaxf(gmax, __shfl_xor_sync(FULL, gmax, o));
    if (lane_id() == 0) red[threadIdx.x >> 5] = gmax;
    __syncthreads();
    gmax = red[lane_id()];
    for (int o = 16; o > 0; o >>= 1) gmax = fmaxf(gmax, __shfl_xor_sync(FULL, gmax, o));
  } else {
    const float g = fabsf(*grad_loss * mul);
    if (g < __uint_as_float(0x7F800000u)) gmax = g;
  }
  if (gmax == 0.0f) gmax = 1.0f;
  const float top = bf16 ? 1.0f : 16384.0f;
  if (threadIdx.x == 0) *scale = gmax / top;
  for (int32_t r = threadIdx.x; r < np; r += 1024) {
    if (r < n) {
      ga[r] = (reduction == GSP_REDUCE_NONE ? grad_loss[s.map[r]] : *grad_loss) * mul / gmax * top;
    } else {
      ga[r] = 0.0f;
      s.lse2[r] = __uint_as_float(0x7F800000u);
    }
  }
  if (low == 0) zero_tail_rows(s.h, s.Dp, n);
}

template <bool kList>
struct LogitGradJob {
  // scratch: per warp 32 rows x 64 columns of P on their way out; bias2 of the tile; a 32 x 32
  // block per warp; column sums of 8 x 16 rows (two buffers)
  static constexpr int kOutBytes = 32 * 128, kBiasOff = mm::kEpiWarps * kOutBytes, kBlockOff = kBiasOff + kBiasScratch;
  static constexpr int kColOff = kBlockOff + mm::kEpiWarps * kBlockBytes;
  static constexpr int kStages = 4, kScratch = kColOff + 2 * 8 * mm::kBN * 4;
  CUtensorMap maps[3];      // H, W (K-major); P as 32 x 64 boxes
  int32_t wait_limit, bf16;
  const int32_t* head;
  int32_t nk, v0, nt;       // the piece's first vocabulary row and 256-wide tiles
  int32_t a_rows;
  int32_t low;              // see low_rows
  float c;
  const float *bias2, *lse2, *ga;
  Lists lists;
  int64_t pitch;            // of P and colpart
  float* colpart;           // [128-row blocks][pitch], or null

  // shares along the vocabulary, as in the forward pass: a row's coefficients are read once per
  // share (its entries are found by bucket, tile by tile)
  struct Walk {
    int32_t lo, x, hi, nt, nk, v0, a_rows;
    __device__ bool next(mm::Tile& t) {
      if (x >= hi) return false;
      t.a_rows = a_rows;
      t.x = x / nt;
      t.y = x - t.x * nt;
      t.a = 0, t.b = 1;
      t.a0 = t.x * mm::kBM;
      t.b0 = v0 + t.y * mm::kBN;
      t.ak = t.bk = 0;
      t.nk = nk;
      t.a_mn = t.b_mn = t.b_cut = t.a_stream = false;
      t.bn = mm::kBN;
      t.flags = (x == lo || t.y == 0 ? kFirst : 0) | (x == hi - 1 ? kLast : 0);
      ++x;
      return true;
    }
  };
  __device__ Walk walk(int32_t pair, int32_t pairs) const {
    const int32_t tot = (head[0] + mm::kBM - 1) / mm::kBM * nt, lo = share_lo(tot, pairs, pair);
    return Walk{lo, lo, share_lo(tot, pairs, pair + 1), nt, nk, v0, a_rows};
  }

  struct Epi {
    float lse, ga;
    int32_t tgt;
    bool live, rest;        // rest: this warp's rows hold what the rounding of others left
    Hits hits;
    __device__ float* bias(const mm::Acc& a) { return reinterpret_cast<float*>(a.scratch + kBiasOff + a.warp * BiasTile::kBytes); }
    __device__ void begin(const LogitGradJob& j, const mm::Tile& t, const mm::Acc& a) {
      const int32_t v0 = t.b0 + a.c_lo;
      BiasTile::load(j.bias2 + v0, reinterpret_cast<unsigned char*>(bias(a)), a.lane);
      rest = j.low > 0 && a.row >= j.low;
      const int32_t row = rest ? a.row - j.low : a.row;
      if (t.flags & kFirst) {
        live = row < j.head[0];
        lse = j.lse2[row];
        ga = j.ga[row];
        if constexpr (!kList) tgt = live ? j.lists.tgt[row] : -1;
      }
      if constexpr (kList) hits.load(j.lists, row - a.lane, j.head[0], v0, a.lane);
    }
    __device__ void tile(const LogitGradJob& j, const mm::Tile& t, const mm::Acc& a) {
      unsigned char* out = a.scratch + a.warp * kOutBytes;
      const float* b = bias(a) - a.c_lo;
      float* block = reinterpret_cast<float*>(a.scratch + kBlockOff + a.warp * kBlockBytes);
      // partial column sums: two rows per warp of 32 rows
      float* cols = reinterpret_cast<float*>(a.scratch + kColOff) + (a.buf * 8 + (a.warp & 3) * 2 + ((a.lane >> 3) & 1)) * mm::kBN +
                    4 * (a.lane & 7);
      const F2 c2 = f2(j.c, j.c), lse2 = f2(-lse, -lse), ga2 = f2(ga, ga);
#pragma unroll 1
      for (int32_t c0 = a.c_lo; c0 < a.c_hi; c0 += 32) {
        // the column sums of the block before this one: loaded here, added up after this block's
        // arithmetic, which covers their latency
        ColLoads before;
        if (j.colpart && c0 > a.c_lo) block_load(before, block, a.lane);
        float z[32];
        a.ld32(c0, z);
        if (c0 + 32 == a.c_hi) a.release();
        const int32_t v0 = t.b0 + c0;
        {
          F2 z2[16];
          to_z(z, c2, b + c0, z2);
#pragma unroll
          for (int k = 0; k < 16; ++k) {
            float p, q;
            split(add2(z2[k], lse2), p, q);
            split(mul2(f2(ex2(p), ex2(q)), ga2), z[2 * k], z[2 * k + 1]);
          }
        }
        if (!live) {        // padding rows: 0 whatever their hidden states hold
#pragma unroll
          for (int k = 0; k < 32; ++k) z[k] = 0.0f;
        }
        bool staged = false;
        if constexpr (kList) {
          hits.each(v0, a.lane, [&](const int4& e, bool in) {
            if (!staged) {
              __syncwarp();       // the column sums of the block before have been read
              block_put(block, z, a.lane);
              staged = true;
            }
            const float g = __shfl_sync(FULL, ga, e.y & 31);
            __syncwarp();
            float* at = block + (e.y & 31) * kBlockLd + (e.x - v0);
            if (in) *at = fmaf(-g, __int_as_float(e.z), *at);
          });
          if (staged) {
            __syncwarp();
            const float* mine = block + a.lane * kBlockLd;
#pragma unroll
            for (int q = 0; q < 8; ++q) {
              const float4 x = *reinterpret_cast<const float4*>(mine + 4 * q);
              z[4 * q] = x.x, z[4 * q + 1] = x.y, z[4 * q + 2] = x.z, z[4 * q + 3] = x.w;
            }
          }
        } else {
          const int32_t d = tgt - v0;
          if (d >= 0 && d < 32) {
#pragma unroll
            for (int k = 0; k < 32; ++k) {
              if (k == d) z[k] -= ga;
            }
          }
        }
        uint32_t w[16];
        pack32(z, w, j.bf16 != 0);
        if (rest) {
          unpack_rest(z, w, j.bf16 != 0);
          pack32(z, w, j.bf16 != 0);
#pragma unroll
          for (int k = 0; k < 32; ++k) z[k] = 0.0f;      // no part of the column sums
          __syncwarp();
          staged = false;
        }
        // half a 128-byte row at a time, 16-byte pieces swizzled as the map wants them
        if ((c0 & 32) == 0) {
          if (a.lane == 0) mm::tma_store_wait_read();
          __syncwarp();
        }
#pragma unroll
        for (int q = 0; q < 4; ++q)
          reinterpret_cast<uint4*>(out + a.lane * 128)[(((c0 & 32) >> 3) + q) ^ (a.lane & 7)] =
              make_uint4(w[4 * q], w[4 * q + 1], w[4 * q + 2], w[4 * q + 3]);
        if (c0 & 32) {
          mm::fence_async();
          __syncwarp();
          if (a.lane == 0) mm::tma_store_2d(&j.maps[2], out, t.y * mm::kBN + c0 - 32, a.row);
        }
        if (j.colpart) {
          if (c0 > a.c_lo) {
            const float4 x = block_sums(before);
            if (a.lane < 16) *reinterpret_cast<float4*>(cols + c0 - 32) = x;
          }
          if (!staged) {
            __syncwarp();
            block_put(block, z, a.lane);
          }
          __syncwarp();
        }
      }
      if (j.colpart) {
        ColLoads last;
        block_load(last, block, a.lane);
        const float4 x = block_sums(last);
        if (a.lane < 16) *reinterpret_cast<float4*>(cols + a.c_hi - 32) = x;
      }
      if ((t.flags & kLast) && a.lane == 0) mm::tma_store_wait();
      if (j.colpart) {
        a.sync();
        const int c = a.warp * 32 + a.lane;
        const float* q = reinterpret_cast<const float*>(a.scratch + kColOff) + a.buf * 8 * mm::kBN + c;
        float x = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; ++i) x += q[i * mm::kBN];
        j.colpart[int64_t(t.x * 2 + a.rank) * j.pitch + t.y * mm::kBN + c] = x;
      }
    }
  };
  __device__ Epi epi() const { return Epi{}; }
};

// ---- host --------------------------------------------------------------------------------
struct Fwd {
  int32_t* counts;
  float* part;
  double* sums;
  Teacher tc;
  int64_t bytes;
};
Fwd carve_fwd(void* base, const gsp_vocab_view* vw, int64_t K) {
  Fwd f{};
  Carver c{static_cast<char*>(base)};
  f.counts = c.take<int32_t>(pack_counts(vw->T));
  f.part = c.take<float>((mm::pair_ctas() / 2 + pad_rows(vw->T) / mm::kBM) * kPart);
  f.sums = c.take<double>(pad_rows(vw->T) / kJoinRows);
  if (K > 0) {
    f.tc.cnt = c.take<int32_t>(vw->T);
    f.tc.ent = c.take<float>(vw->T);
    f.tc.entry = c.take<int2>(vw->T * K);
    f.tc.pz = c.take<float>(pad_rows(vw->T) * K);
    f.tc.flag = c.take<uint8_t>(vw->T);
  }
  f.bytes = c.off;
  return f;
}
struct Bwd {
  float *ga, *scale, *colpart;
  GradScratch grad;
  uint16_t* P;
  int64_t pitch, bytes;
};
Bwd carve_bwd(void* base, const gsp_vocab_view* vw) {
  Bwd b{};
  Carver c{static_cast<char*>(base)};
  const int64_t Tp = pad_rows(vw->T);
  b.pitch = piece_cols(Tp, vw->V);
  b.ga = c.take<float>(Tp);
  b.scale = c.take<float>(1);
  b.colpart = c.take<float>(Tp / mm::kRows * b.pitch);
  b.grad = carve_grad(c, vw, Tp, b.pitch);
  b.P = c.take<uint16_t>(Tp * b.pitch);
  b.bytes = c.off;
  return b;
}

// Rows of a box of H: up to 128 tokens no more than there are (a single token's product would
// else spend as long on rows of nothing as on the vocabulary)
int32_t box_rows(int64_t T) { return int32_t(T >= mm::kRows ? mm::kRows : up(T, 8)); }

// tau^2 scales the losses and 1 / tau the logits: both stay normal numbers
int check_temperature(float tau, const char* what) {
  const float t2 = tau * tau;
  GSP_REQUIRE(tau > 0.0f && t2 >= 0x1p-126f && t2 < __builtin_inff(), GSP_ERR_ARG,
              "%s: temperature must be positive, from 1.1e-19 to 1.8e19, got %g", what, double(tau));
  return GSP_OK;
}

int check_reduction(int32_t reduction, const char* what) {
  GSP_REQUIRE(reduction >= GSP_REDUCE_NONE && reduction <= GSP_REDUCE_MEAN, GSP_ERR_ARG, "%s: unknown reduction %d", what,
              reduction);
  return GSP_OK;
}

template <bool kList>
int run_forward(const gsp_vocab_view* vw, const State& s, const Fwd& f, float tau, int32_t reduction, float* loss,
                cudaStream_t st) {
  const Weight w = weight_rows(vw, s);
  int rc;
  LossJob<kList> j{};
  const bool bf = is_bf16(vw);
  j.a_rows = box_rows(vw->T);
  if ((rc = make_map(&j.maps[0], bf, s.h, s.Dp, s.Tp, s.Dp, j.a_rows))) return rc;
  if ((rc = make_map(&j.maps[1], bf, w.w, vw->D, vw->V, w.ld, mm::kBN / 2))) return rc;
  j.wait_limit = gsp_get_wait_limit();
  j.bf16 = bf;
  j.head = s.head;
  j.nt = int32_t(s.Vp / mm::kBN);
  j.nk = int32_t((vw->D + mm::kBK - 1) / mm::kBK);
  j.c = kLog2e / tau;
  j.bias2 = s.bias2;
  j.lists = lists_of(s, kList, f.tc.pz);
  j.part = f.part;
  if ((rc = launch_mma(j, st))) return rc;
  if (reduction == GSP_REDUCE_NONE) GSP_CUDA(cudaMemsetAsync(loss, 0, size_t(vw->T) * sizeof(float), st));
  return launch(join_kernel, dim3(unsigned((vw->T + kJoinRows - 1) / kJoinRows)), 32 * kJoinRows, 0, st, s.head, s.map, f.part,
                j.nt, mm::pair_ctas() / 2, f.tc, s.K, tau * tau, reduction, s.lse2, f.sums, loss);
}

template <bool kList>
int run_backward(const gsp_vocab_view* vw, const State& s, const Bwd& b, float tau, void* d_hidden, void* d_weight,
                 float* d_bias, cudaStream_t st) {
  const Weight w = weight_rows(vw, s);
  int rc;
  LogitGradJob<kList> j{};
  const bool bf = is_bf16(vw);
  j.low = low_rows(vw);
  j.a_rows = box_rows(j.low + vw->T);
  if ((rc = make_map(&j.maps[0], bf, s.h, s.Dp, s.Tp, s.Dp, j.a_rows))) return rc;
  if ((rc = make_map(&j.maps[1], bf, w.w, vw->D, vw->V, w.ld, mm::kBN / 2))) return rc;
  j.wait_limit = gsp_get_wait_limit();
  j.bf16 = bf;
  j.head = s.head;
  j.nk = int32_t((vw->D + mm::kBK - 1) / mm::kBK);
  j.c = kLog2e / tau;
  j.bias2 = s.bias2;
  j.lse2 = s.lse2;
  j.ga = b.ga;
  j.lists = lists_of(s, kList, nullptr);
  if ((rc = make_map(&j.maps[2], bf, b.P, b.pitch, s.Tp, b.pitch, 32))) return rc;
  j.pitch = b.pitch;
  j.colpart = d_bias ? b.colpart : nullptr;
  for (int64_t v0 = 0; v0 < vw->V; v0 += b.pitch) {
    const int64_t cols = min64(b.pitch, vw->V - v0);
    j.v0 = int32_t(v0);
    j.nt = int32_t((cols + mm::kBN - 1) / mm::kBN);
    if ((rc = launch_mma(j, st))) return rc;
    const GradPiece pc{b.P, b.pitch, v0, cols, v0 == 0, v0 + cols >= vw->V, Sparse{}, j.low};
    if ((rc = grad_products(vw, s, w.w, w.ld, pc, b.grad, BiasSums{b.colpart, b.pitch, d_bias ? d_bias + v0 : nullptr}, b.scale, d_hidden, d_weight, st))) return rc;
  }
  return GSP_OK;
}

}  // namespace

int64_t loss_ws_bytes(const gsp_vocab_view* vw, int64_t K, bool backward) {
  return backward ? carve_bwd(nullptr, vw).bytes : carve_fwd(nullptr, vw, K).bytes;
}

}  // namespace vocab
}  // namespace gsp

using namespace gsp;
using namespace gsp::vocab;

extern "C" int gsp_vocab_ce(const gsp_vocab_view* vw, const int64_t* targets, int64_t ignore_index, int32_t reduction,
                            float* loss, void* state, int64_t state_bytes, void* ws, int64_t ws_bytes, void* stream) {
  int rc = check_view(vw, "vocab_cross_entropy");
  if (rc) return rc;
  if ((rc = check_reduction(reduction, "vocab_cross_entropy"))) return rc;
  cudaStream_t st = as_stream(stream);
  GSP_REQUIRE(loss || (vw->T == 0 && reduction == GSP_REDUCE_NONE), GSP_ERR_ARG, "vocab_cross_entropy: null loss");
  const State s = carve_state(state, vw, 0, 0);
  const Fwd f = carve_fwd(ws, vw, 0);
  if ((rc = check_buffers(state, state_bytes, s.bytes, ws, ws_bytes, f.bytes, "vocab_cross_entropy"))) return rc;
  if (vw->T == 0) {
    if (reduction != GSP_REDUCE_NONE) GSP_CUDA(cudaMemsetAsync(loss, 0, sizeof(float), st));
    return GSP_OK;
  }
  GSP_REQUIRE(targets && vw->hidden && vw->weight, GSP_ERR_ARG, "vocab_cross_entropy: null input");
  if ((rc = pack_rows(vw, targets, ignore_index, nullptr, kLog2e, Texts{}, s, f.counts, st))) return rc;
  return run_forward<false>(vw, s, f, 1.0f, reduction, loss, st);
}

extern "C" int gsp_vocab_distill(const gsp_vocab_view* vw, const float* scores, const int64_t* ids, int64_t K, float tau,
                                 int32_t reduction, float* loss, void* state, int64_t state_bytes, void* ws,
                                 int64_t ws_bytes, void* stream) {
  int rc = check_view(vw, "topk_distillation");
  if (rc) return rc;
  if ((rc = check_reduction(reduction, "topk_distillation"))) return rc;
  cudaStream_t st = as_stream(stream);
  GSP_REQUIRE(K >= 1 && K <= GSP_DISTILL_MAX_K, GSP_ERR_ARG, "topk_distillation: %lld teacher entries, 1 to %d are supported",
              (long long)K, GSP_DISTILL_MAX_K);
  if ((rc = check_temperature(tau, "topk_distillation"))) return rc;
  GSP_REQUIRE(loss || (vw->T == 0 && reduction == GSP_REDUCE_NONE), GSP_ERR_ARG, "topk_distillation: null loss");
  const State s = carve_state(state, vw, K, 0);
  const Fwd f = carve_fwd(ws, vw, K);
  if ((rc = check_buffers(state, state_bytes, s.bytes, ws, ws_bytes, f.bytes, "topk_distillation"))) return rc;
  if (vw->T == 0) {
    if (reduction != GSP_REDUCE_NONE) GSP_CUDA(cudaMemsetAsync(loss, 0, sizeof(float), st));
    return GSP_OK;
  }
  GSP_REQUIRE(scores && ids && vw->hidden && vw->weight, GSP_ERR_ARG, "topk_distillation: null input");
  int32_t log_slots = 5;
  while ((1 << log_slots) < 2 * K) ++log_slots;
  const size_t teacher_bytes = (size_t(1) << log_slots) * sizeof(TeacherSlot) + size_t(K) * 8;
  const int threads = K >= kTeacherThreads ? kTeacherThreads : int(up(K, 32));
  rc = launch(teacher_kernel, dim3(unsigned(vw->T)), threads, teacher_bytes, st, scores, ids, int32_t(K), log_slots, vw->V,
              1.0f / tau, f.tc);
  if (rc) return rc;
  if ((rc = pack_rows(vw, nullptr, 0, f.tc.flag, kLog2e / tau, Texts{}, s, f.counts, st))) return rc;
  // few rows: several CTAs for each 32 of them
  const int64_t groups = (vw->T + 31) / 32, wide = num_sms() / groups;
  const unsigned splits = unsigned(wide < 1 ? 1 : min64(wide, kBucketSplits));
  const int bucket_bytes = int((s.buckets + splits - 1) / splits * 4);
  if ((rc = ensure_smem(reinterpret_cast<const void*>(&bucket_kernel), bucket_bytes))) return rc;
  if ((rc = launch(bucket_kernel, dim3(unsigned(groups), splits), kBucketThreads, size_t(bucket_bytes), st, s, f.tc))) return rc;
  return run_forward<true>(vw, s, f, tau, reduction, loss, st);
}

extern "C" int gsp_vocab_loss_backward(const gsp_vocab_view* vw, int32_t kind, int64_t K, float tau, int32_t reduction,
                                       const float* grad_loss, void* d_hidden, void* d_weight,
                                       float* d_bias, void* state, int64_t state_bytes, void* ws, int64_t ws_bytes,
                                       void* stream) {
  int rc = check_view(vw, "vocab loss backward");
  if (rc) return rc;
  if ((rc = check_reduction(reduction, "vocab loss backward"))) return rc;
  if ((rc = check_grads(vw, d_hidden, d_weight, "vocab loss backward"))) return rc;
  GSP_REQUIRE(kind == GSP_VOCAB_CE || kind == GSP_VOCAB_DISTILL, GSP_ERR_ARG, "vocab loss backward: unknown kind %d", kind);
  const bool list = kind == GSP_VOCAB_DISTILL;
  GSP_REQUIRE(!list || (K >= 1 && K <= GSP_DISTILL_MAX_K), GSP_ERR_ARG, "vocab loss backward: bad teacher entries");
  if (list && (rc = check_temperature(tau, "vocab loss backward"))) return rc;
  cudaStream_t st = as_stream(stream);
  const State s = carve_state(state, vw, list ? K : 0, 0);
  const Bwd b = carve_bwd(ws, vw);
  if ((rc = check_buffers(state, state_bytes, s.bytes, ws, ws_bytes, b.bytes, "vocab loss backward"))) return rc;
  const size_t VD = size_t(vw->V) * size_t(vw->D);
  if (vw->T == 0) {
    if (d_weight) GSP_CUDA(cudaMemsetAsync(d_weight, 0, VD * 2, st));
    if (d_bias) GSP_CUDA(cudaMemsetAsync(d_bias, 0, size_t(vw->V) * sizeof(float), st));
    return GSP_OK;
  }
  GSP_REQUIRE(grad_loss && vw->weight, GSP_ERR_ARG, "vocab loss backward: null input");
  if (!list) tau = 1.0f;
  const int64_t hidden_bytes = vw->T * vw->D * 2;
  const int64_t zero_blocks = d_hidden ? min64((hidden_bytes + 65535) / 65536, num_sms()) : 0;
  rc = launch(grad_rows_kernel, dim3(unsigned(1 + zero_blocks)), 1024, 0, st, s, grad_loss, reduction, tau, int32_t(is_bf16(vw)),
              low_rows(vw), b.ga, b.scale, d_hidden, hidden_bytes);
  if (rc) return rc;
  return list ? run_backward<true>(vw, s, b, tau, d_hidden, d_weight, d_bias, st)
              : run_backward<false>(vw, s, b, tau, d_hidden, d_weight, d_bias, st);
}
