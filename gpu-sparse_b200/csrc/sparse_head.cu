// The sparse head: y[b, v] = log1p(relu(max over the tokens t of text b of H[t] . W[v] + bias[v])),
// the term weights an index is built from, and its gradient.
//
// Forward.  The product is taken as W H^T, vocabulary rows in the tensor memory's lanes and
// packed tokens in its columns, so that the maximum over a text's tokens runs along one
// thread's registers: one compare per logit, no exchange between threads, and log1p only on
// the maximum (it is monotone).  Tiles are ordered tokens-fastest and cut into equal shares,
// one per pair of CTAs.  The texts open at the end of a column half are carried to the thread
// that has the same vocabulary row in the next half (shared memory, a named barrier in each
// direction), and a text that a share's border cuts leaves its partial maxima for a joining
// kernel.  Texts may so have any length, and no work is lost to their padding.  Bound by the
// products (V = 30522, D = 768): 64 texts of up to 512 tokens take 510 us, 1.66 PFLOP/s, 500
// short queries 342 us, 1.21 PFLOP/s, their ends costing the epilogue more; one query 13 us, of
// which 7 are W's bytes.
//
// Backward.  Each (text, term) with y > 0 (or NaN) sends ds = dy exp(-y) to its winning token:
//   dH[win] += ds W[v],   dW[v] += ds H[win],   d_bias[v] += ds.
// Term weights are sparse (a trained head keeps hundreds of 30522 terms), so these are sums of
// few rows of W and H, gathered from L2 in a fixed order, fp32 throughout: dW takes a term's
// texts one after the other, dH a list of the entries sorted by token (a counting sort that keeps
// the order of the terms).  While a head is still dense over short texts (more than one entry in
// kGatherWeight of tokens x vocabulary) the gathers would cost more than products: then P
// [tokens, V] with one entry per (text, term) goes through the losses' two products.  The
// entries are counted on the GPU and the kernels of the other way return at once.
//   The products take P rounded once to 16 bits, the gathers take ds in fp32, so the number of
// entries decides on the precision too: fp16 gradients are off by 0.0003 of their norm as products,
// by 0.00021 gathered, which is their own rounding (bf16: 0.0024 and 0.0017).
//   The gathers move 585 MB in 102 us for dW and 571 MB in 91 us for dH (32 texts of 256 tokens, one
// entry in 671): 5.7 and 6.3 TB/s, where the products read L2 at 9 to 10.6.  At 0.4 to 0.5
// instructions a cycle with four rows in flight for each of 16 warps they are bound by the latency
// of these loads and by the additions.
#include "vocab.cuh"

namespace gsp {
namespace vocab {
namespace {

constexpr int kFirst = 1, kLast = 2;      // of a share along one row of tiles
constexpr int kBegin = 4, kEnd = 8;       // of a share

// Whether z takes the maximum over from m: it is larger, or the first NaN.  A NaN has a winner like
// any other maximum, so that its gradient is NaN too.
__device__ __forceinline__ bool takes(float z, float m) { return !(z <= m) && m == m; }
__device__ __forceinline__ bool is_nan(float x) { return x != x; }

template <bool kWin>
struct HeadJob {
  // scratch: per warp 16 finished maxima and tokens per lane; per column half the carry
  static constexpr int kSlots = 16;
  static constexpr int kSlotBytes = kSlots * 32 * 4 * 2;
  static constexpr int kCarryOff = mm::kEpiWarps * kSlotBytes;
  static constexpr int kStages = 5, kScratch = kCarryOff + 2 * (mm::kRows * 8 + 16);
  CUtensorMap maps[2];      // W, H (K-major)
  int32_t wait_limit, bf16;
  const int32_t* head;
  const int32_t* map;
  int32_t L, V, nvt, nk, bn;
  const float* bias;
  float* y;
  int32_t* win;
  float* part_m;            // [pairs][2: begun elsewhere, open at the end][kBM]
  int32_t* part_i;

  struct Walk {
    int32_t lo, x, hi, ntt, nk, bn;
    __device__ bool next(mm::Tile& t) {
      if (x >= hi) return false;
      t.x = x / ntt;
      t.y = x - t.x * ntt;
      t.a = 0, t.b = 1;
      t.a0 = t.x * mm::kBM;
      t.b0 = t.y * bn;
      t.ak = t.bk = 0;
      t.nk = nk;
      t.a_mn = t.b_mn = t.b_cut = t.a_stream = false;
      t.bn = bn;
      t.a_rows = mm::kRows;
      t.flags = (x == lo || t.y == 0 ? kFirst : 0) | (x == hi - 1 || t.y == ntt - 1 ? kLast : 0) | (x == lo ? kBegin : 0) |
                (x == hi - 1 ? kEnd : 0);
      ++x;
      return true;
    }
  };
  __device__ Walk walk(int32_t pair, int32_t pairs) const {
    const int32_t ntt = (head[0] + bn - 1) / bn, tot = ntt * nvt, lo = share_lo(tot, pairs, pair);
    return Walk{lo, lo, share_lo(tot, pairs, pair + 1), ntt, nk, bn};
  }

  struct Epi {
    // (a NaN that no token won, -inf plus a bias of +inf, is given to the row)
    __device__ static void put(const HeadJob& j, int32_t row, int32_t v, float bias, float m, int32_t idx) {
      if (v >= j.V) return;
      const float x = m + bias;
      const int64_t o = int64_t(j.map[row] / j.L) * j.V + v;
      j.y[o] = x > 0.0f ? log1pf(x) : (is_nan(x) ? x : 0.0f);
      if (kWin) j.win[o] = x <= 0.0f ? -1 : (idx >= 0 ? idx : row);
    }
    __device__ static void part(const HeadJob& j, const mm::Acc& a, int which, float m, int32_t idx) {
      const int64_t o = (int64_t(blockIdx.x >> 1) * 2 + which) * mm::kBM + a.rank * mm::kRows + a.lane_row;
      j.part_m[o] = m;
      if (kWin) j.part_i[o] = idx;
    }
    uint32_t ends[4];      // which of this half's columns end a text
    bool cut;              // the text open at the half's start began in an earlier share
    __device__ void begin(const HeadJob& j, const mm::Tile& t, const mm::Acc& a) {
      const int32_t n = j.head[0], r_lo = t.b0 + a.c_lo, r_hi = min(t.b0 + a.c_hi, n);
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const int32_t r = r_lo + 32 * w + a.lane;
        bool e = false;
        if (r < r_hi) e = r + 1 == n || j.map[r] / j.L != j.map[r + 1] / j.L;
        ends[w] = __ballot_sync(FULL, e);
      }
      if ((t.flags & kFirst) && a.half == 0) cut = t.b0 > 0 && j.map[t.b0 - 1] / j.L == j.map[t.b0] / j.L;
    }
    __device__ void tile(const HeadJob& j, const mm::Tile& t, const mm::Acc& a) {
      const int32_t n = j.head[0], v = a.row;
      const float bias = j.bias && v < j.V ? __ldg(j.bias + v) : 0.0f;
      const int32_t r_lo = t.b0 + a.c_lo, r_hi = min(t.b0 + a.c_hi, n);
      float* slot_m = reinterpret_cast<float*>(a.scratch + a.warp * kSlotBytes) + a.lane;
      int32_t* slot_i = reinterpret_cast<int32_t*>(slot_m + kSlots * 32);
      float m = neg_inf(), head_m = neg_inf();
      int32_t idx = -1, head_i = -1, head_row = -1;     // head: the first text that ends here
#pragma unroll 1
      for (int w = 0; w < 4; ++w) {
        const int32_t r0 = r_lo + 32 * w;
        if (r0 >= r_hi) break;
        float z[32];
        a.ld32(a.c_lo + 32 * w, z);
        if (r0 + 32 >= r_hi) a.release();
        const uint32_t word = w < 2 ? (w == 0 ? ends[0] : ends[1]) : (w == 2 ? ends[2] : ends[3]);
        // 16 columns at a time; columns past the last row are past the last text's end
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          uint32_t bits = (word >> (16 * h)) & 0xFFFFu;
          const int32_t rb = r0 + 16 * h;
          int32_t won = -1;
          if (bits == 0) {
            const float before = m;
#pragma unroll
            for (int k = 0; k < 16; ++k) {
              if (kWin) won = z[16 * h + k] > m ? k : won;
              asm("max.NaN.f32 %0, %0, %1;" : "+f"(m) : "f"(z[16 * h + k]));
            }
            if (kWin && is_nan(m) && !is_nan(before)) {
#pragma unroll
              for (int k = 15; k >= 0; --k) won = is_nan(z[16 * h + k]) ? k : won;
            }
            if (kWin && won >= 0) idx = rb + won;
          } else {
            int32_t e = 0;
#pragma unroll
            for (int k = 0; k < 16; ++k) {
              if (kWin) idx = takes(z[16 * h + k], m) ? rb + k : idx;
              asm("max.NaN.f32 %0, %0, %1;" : "+f"(m) : "f"(z[16 * h + k]));
              if ((bits >> k) & 1) {
                slot_m[e * 32] = m;
                if (kWin) slot_i[e * 32] = idx;
                ++e;
                m = neg_inf();
                idx = -1;
              }
            }
            for (int32_t q = 0; q < e; ++q) {
              const int32_t row = rb + __ffs(bits) - 1;
              bits &= bits - 1;
              const float x = slot_m[q * 32];
              const int32_t xi = kWin ? slot_i[q * 32] : 0;
              if (head_row < 0) {
                head_row = row;
                head_m = x;
                head_i = xi;
              } else {
                put(j, row, v, bias, x, xi);
              }
            }
          }
        }
      }
      if (r_lo >= r_hi) a.release();
      // the text open at this half's start: what the halves before it in the share found
      unsigned char* carry = a.scratch + kCarryOff;
      constexpr int kCarryBytes = mm::kRows * 8 + 16;
      float* in_m = reinterpret_cast<float*>(carry + (1 - a.half) * kCarryBytes) + a.lane_row;
      float* out_m = reinterpret_cast<float*>(carry + a.half * kCarryBytes) + a.lane_row;
      int32_t* in_cut = reinterpret_cast<int32_t*>(carry + (1 - a.half) * kCarryBytes + mm::kRows * 8);
      int32_t* out_cut = reinterpret_cast<int32_t*>(carry + a.half * kCarryBytes + mm::kRows * 8);
      float cm = neg_inf();
      int32_t ci = -1;
      // the two halves' threads take turns over all of the share, so neither overtakes the other
      __syncwarp();
      if (a.half == 1 || !(t.flags & kBegin)) asm volatile("bar.sync %0, 256;" ::"r"(3 - a.half) : "memory");
      if (!(t.flags & kFirst) || a.half == 1) {
        cm = in_m[0];
        if (kWin) ci = reinterpret_cast<int32_t*>(in_m)[mm::kRows];
        cut = *in_cut != 0;
      }
      float open_m = m;
      int32_t open_i = idx;
      if (head_row >= 0) {
        const int32_t hi = kWin && takes(head_m, cm) ? head_i : ci;
        asm("max.NaN.f32 %0, %0, %1;" : "+f"(head_m) : "f"(cm));
        if (cut) part(j, a, 0, head_m, hi);
        else put(j, head_row, v, bias, head_m, hi);
        cut = false;
      } else {
        if (kWin) open_i = takes(m, cm) ? idx : ci;
        asm("max.NaN.f32 %0, %0, %1;" : "+f"(open_m) : "f"(cm));
      }
      if ((t.flags & kLast) && a.half == 1) {
        const int32_t end = min(t.b0 + t.bn, n);
        if (end < n && j.map[end] / j.L == j.map[end - 1] / j.L) part(j, a, 1, open_m, open_i);
      } else {
        out_m[0] = open_m;
        if (kWin) reinterpret_cast<int32_t*>(out_m)[mm::kRows] = open_i;
        if (a.lane_row == 0) *out_cut = cut;
      }
      __syncwarp();
      if (a.half == 0 || !(t.flags & kEnd)) asm volatile("bar.arrive %0, 256;" ::"r"(2 + a.half) : "memory");
    }
  };
  __device__ Epi epi() const { return Epi{}; }
};

struct JoinParams {
  const int32_t *head, *map;
  int32_t L, bn, pairs, nvt;
  int64_t V;
  const float* bias;
  const float* part_m;
  const int32_t* part_i;
  float* y;
  int32_t* win;
};

// A block per share: a text that began in an earlier share and ends in this one is joined from
// the shares it crosses, in order.
__global__ void __launch_bounds__(mm::kBM) head_join_kernel(const JoinParams p) {
  mm::after_previous();
  const int32_t n = p.head[0];
  const int32_t ntt = (n + p.bn - 1) / p.bn, tot = ntt * p.nvt, c = blockIdx.x;
  const int32_t lo = share_lo(tot, p.pairs, c), hi = share_lo(tot, p.pairs, c + 1);
  if (lo >= hi) return;
  const int32_t vt = lo / ntt, r0 = (lo - vt * ntt) * p.bn;
  if (r0 == 0) return;
  const int32_t text = p.map[r0] / p.L;
  if (p.map[r0 - 1] / p.L != text) return;
  // does it end inside this share?
  const int64_t row_end = min64(n, int64_t(min(hi, (vt + 1) * ntt) - vt * ntt) * p.bn);
  if (row_end < n && p.map[row_end] / p.L == text) return;
  int32_t first = c - 1;
  for (;; --first) {
    const int64_t at = int64_t(share_lo(tot, p.pairs, first) - vt * ntt) * p.bn;   // its first row along this tile row
    if (at <= 0 || p.map[at - 1] / p.L != text) break;
  }
  float m = neg_inf();
  int32_t idx = -1;
  for (int32_t s = first; s <= c; ++s) {
    const int64_t o = (int64_t(s) * 2 + (s == c ? 0 : 1)) * mm::kBM + threadIdx.x;
    const float x = p.part_m[o];
    if (p.win && takes(x, m)) idx = p.part_i[o];
    asm("max.NaN.f32 %0, %0, %1;" : "+f"(m) : "f"(x));
  }
  const int64_t v = int64_t(vt) * mm::kBM + threadIdx.x;
  if (v >= p.V) return;
  const float x = m + (p.bias ? p.bias[v] : 0.0f);
  p.y[text * p.V + v] = x > 0.0f ? log1pf(x) : (is_nan(x) ? x : 0.0f);
  if (p.win) p.win[text * p.V + v] = x <= 0.0f ? -1 : (idx >= 0 ? idx : r0);
}

// ---- backward ----------------------------------------------------------------------------
struct Survey {
  int64_t nnz;            // entries: (text, term) pairs with a gradient
  uint32_t absmax;        // largest finite |dy| of them (an upper bound of |ds|, which scales fp16's P)
  uint32_t pad_;
};

// ds of (text, term) pairs o[k] (negative: none) and their tokens' packed rows (-1: no gradient; a
// NaN weight has one, NaN, even where dy is 0); all loads are issued before the first is used
template <int N>
__device__ __forceinline__ void entry_grads(const float* y, const int32_t* win, const float* dy, const int64_t (&o)[N],
                                            int32_t (&row)[N], float (&ds)[N]) {
  float d[N], v[N];
#pragma unroll
  for (int k = 0; k < N; ++k) {
    row[k] = o[k] >= 0 ? win[o[k]] : -1;
    d[k] = o[k] >= 0 ? dy[o[k]] : 0.0f;
    v[k] = o[k] >= 0 ? y[o[k]] : 0.0f;
  }
#pragma unroll
  for (int k = 0; k < N; ++k) {
    if (d[k] == 0.0f && !is_nan(v[k])) row[k] = -1;
    ds[k] = row[k] >= 0 ? d[k] * expf(-v[k]) : 0.0f;
  }
}

// The counting sort.  A warp takes one of kSegs runs of a text's terms and keeps a counter per
// token of the text in shared memory; the counts [packed row][run] are scanned in that order, so
// that a token's entries end up side by side in the order of their terms.
constexpr int kSegs = 64;
constexpr int kSortSmem = 48 * 1024;
struct SortParams {
  const int32_t *head, *text;
  const float *y, *dy;
  const int32_t* win;
  int64_t B, V;
  int32_t L;               // counters per warp; 0: the survey alone
  int32_t* count;          // [packed rows][kSegs]
  const int64_t* offset;   // their exclusive scan
  int2* list;              // (term, ds)
  Sparse sparse;
};
inline int sort_warps(int64_t L) { return int(L * 4 * 8 <= kSortSmem ? 8 : kSortSmem / (L * 4)); }

// Counts; also the survey, d_hidden's zeroes and the packed rows' tail.  (Survey and counts are
// zeroed before.)
__global__ void __launch_bounds__(256)
survey_kernel(State s, const SortParams p, Survey* out, void* d_hidden, int64_t hidden_bytes) {
  mm::after_previous();
  extern __shared__ int32_t counters[];
  const int lane = lane_id(), wid = threadIdx.x >> 5, warps = blockDim.x >> 5;
  const int64_t job = int64_t(blockIdx.x) * warps + wid, b = job / kSegs;
  const int32_t seg = int32_t(job % kSegs);
  if (b < p.B) {
    const int32_t first = p.text[b], len = p.text[b + 1] - first;
    const bool sort = p.L > 0;
    int32_t* mine = counters + wid * p.L;
    if (sort) {
      for (int32_t i = lane; i < len; i += 32) mine[i] = 0;
      __syncwarp();
    }
    const int64_t per = (p.V + kSegs - 1) / kSegs, lo = seg * per, hi = min64(p.V, lo + per);
    uint32_t c = 0;
    float m = 0.0f;
    for (int64_t t0 = lo; t0 < hi; t0 += 256) {
      int32_t r[8];
      float d[8];
      // (volatile: loads of both in flight.  Left to itself the compiler asks for d only where r >= 0,
      // after r has come: a training step on 32 texts took 375 us instead of 365)
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const int64_t t = t0 + 32 * k + lane;
        r[k] = -1;
        d[k] = 0.0f;
        if (t < hi) {
          asm volatile("ld.global.b32 %0, [%1];" : "=r"(r[k]) : "l"(p.win + b * p.V + t));
          asm volatile("ld.global.f32 %0, [%1];" : "=f"(d[k]) : "l"(p.dy + b * p.V + t));
        }
      }
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const float a = fabsf(d[k]);
        if (r[k] >= 0 && a < __uint_as_float(0x7F800000u)) m = fmaxf(m, a);
        if (r[k] >= 0 && d[k] == 0.0f && !is_nan(p.y[b * p.V + t0 + 32 * k + lane])) r[k] = -1;
        c += r[k] >= 0;
      }
      if (sort) {
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          if (r[k] >= 0) atomicAdd(mine + (r[k] - first), 1);
        }
      }
    }
    if (sort) {
      __syncwarp();
      for (int32_t i = lane; i < len; i += 32) p.count[int64_t(first + i) * kSegs + seg] = mine[i];
    }
    c = __reduce_add_sync(FULL, c);
    const uint32_t w = __reduce_max_sync(FULL, __float_as_uint(m));
    if (lane == 0) {
      if (c) atomicAdd(reinterpret_cast<unsigned long long*>(&out->nnz), static_cast<unsigned long long>(c));
      if (w) atomicMax(&out->absmax, w);
    }
  }
  if (d_hidden) zero_share(d_hidden, hidden_bytes, blockIdx.x, gridDim.x);
  if (blockIdx.x == 0) zero_tail_rows(s.h, s.Dp, s.head[0]);
}

// The list: every warp places its run's entries where the scan says.
__global__ void __launch_bounds__(256) place_kernel(const SortParams p) {
  mm::after_previous();
  extern __shared__ int32_t counters[];
  const int lane = lane_id(), wid = threadIdx.x >> 5, warps = blockDim.x >> 5;
  const int64_t job = int64_t(blockIdx.x) * warps + wid, b = job / kSegs;
  const int32_t seg = int32_t(job % kSegs);
  if (b >= p.B || !p.sparse.gather(p.head[0], p.V)) return;
  const int32_t first = p.text[b], len = p.text[b + 1] - first;
  int32_t* next = counters + wid * p.L;
  for (int32_t i = lane; i < len; i += 32) next[i] = int32_t(p.offset[int64_t(first + i) * kSegs + seg]);
  __syncwarp();
  const int64_t per = (p.V + kSegs - 1) / kSegs, lo = seg * per, hi = min64(p.V, lo + per);
  for (int64_t t0 = lo; t0 < hi; t0 += 256) {
    int64_t o[8];
    int32_t r[8];
    float g[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) o[k] = t0 + 32 * k + lane < hi ? b * p.V + t0 + 32 * k + lane : -1;
    entry_grads(p.y, p.win, p.dy, o, r, g);
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      if (!__any_sync(FULL, r[k] >= 0)) continue;
      const uint32_t same = __match_any_sync(FULL, r[k]);
      int32_t at = 0;
      if (r[k] >= 0) at = next[r[k] - first];
      __syncwarp();
      if (r[k] >= 0) {
        p.list[at + __popc(same & lanemask_lt())] = make_int2(int32_t(t0 + 32 * k + lane), __float_as_int(g[k]));
        if (lane == __ffs(same) - 1) next[r[k] - first] = at + __popc(same);
      }
      __syncwarp();
    }
  }
}

struct GatherParams {
  const int32_t *head, *map;
  Sparse sparse;
  const int64_t* offset;   // of the list, by packed row x kSegs
  const int2* list;
  const float *y, *dy;
  const int32_t* win;
  const uint16_t *h, *w;
  int64_t Dp, ldw, B, V, D;
  int32_t bf16;
  uint16_t *dh, *dw;
  float* db;
};

// 8 columns of every 256 from d0 of a row, zeros from column `end` on; rows start on 16-byte
// boundaries, and the 16 bytes that hold its last column belong to it or to nobody
template <int kCols>
__device__ __forceinline__ void load_row(const uint16_t* from, int64_t d0, int64_t end, int lane, uint4 (&x)[kCols]) {
#pragma unroll
  for (int q = 0; q < kCols; ++q) {
    const int64_t c = d0 + q * 256 + lane * 8;
    x[q] = c < end ? __ldg(reinterpret_cast<const uint4*>(from + c)) : make_uint4(0, 0, 0, 0);
  }
}
// acc += g x
template <int kCols>
__device__ __forceinline__ void add_row(float (&acc)[kCols][8], const uint4 (&x)[kCols], float g, bool bf) {
#pragma unroll
  for (int q = 0; q < kCols; ++q) {
    const uint32_t u[4] = {x[q].x, x[q].y, x[q].z, x[q].w};
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const float2 f = unpack2(u[k], bf);
      acc[q][2 * k] = fmaf(g, f.x, acc[q][2 * k]);
      acc[q][2 * k + 1] = fmaf(g, f.y, acc[q][2 * k + 1]);
    }
  }
}
// 8 columns (or the last n of a row) at any address
__device__ __forceinline__ void store8(uint16_t* out, int n, const float (&v)[8], bool bf) {
  uint32_t u[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) u[k] = pack2(v[2 * k], v[2 * k + 1], bf);
  if (n == 8 && (reinterpret_cast<uintptr_t>(out) & 15) == 0) {
    *reinterpret_cast<uint4*>(out) = make_uint4(u[0], u[1], u[2], u[3]);
  } else {
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      if (k < n) out[k] = uint16_t(u[k >> 1] >> (16 * (k & 1)));
    }
  }
}

// dW and d_bias: a warp per term, eight terms per CTA.  The warp takes the texts in order, 256 at
// a time through shared memory (whose loads are then whole sectors), and adds the winners' rows;
// a lane has 8 columns of every 256, up to 1024 columns at a time.
constexpr int kTexts = 256;
template <int kCols>
__global__ void __launch_bounds__(256, 2) gather_weight_kernel(const GatherParams p) {
  mm::after_previous();
  __shared__ int32_t row[kTexts][9];
  __shared__ float grad[kTexts][9];
  const bool gather = p.sparse.gather(p.head[0], p.V) && p.dw;
  if (!gather && !p.db) return;
  const int64_t v0 = int64_t(blockIdx.x) * 8, v = v0 + (threadIdx.x >> 5);
  const int wid = threadIdx.x >> 5, lane = lane_id();
  const bool bf = p.bf16 != 0;
  float db = 0.0f;
  for (int64_t d0 = 0; d0 < (gather ? p.D : 1); d0 += 256 * kCols) {
    float acc[kCols][8];
#pragma unroll
    for (int q = 0; q < kCols; ++q) {
#pragma unroll
      for (int k = 0; k < 8; ++k) acc[q][k] = 0.0f;
    }
    for (int64_t b0 = 0; b0 < p.B; b0 += kTexts) {
      __syncthreads();
      int64_t o[kTexts * 8 / 256];
      int32_t r[kTexts * 8 / 256];
      float g[kTexts * 8 / 256];
#pragma unroll
      for (int i = 0; i < kTexts * 8 / 256; ++i) {
        const int e = i * 256 + threadIdx.x, b = e >> 3, c = e & 7;
        o[i] = b0 + b < p.B && v0 + c < p.V ? (b0 + b) * p.V + v0 + c : -1;
      }
      entry_grads(p.y, p.win, p.dy, o, r, g);
#pragma unroll
      for (int i = 0; i < kTexts * 8 / 256; ++i) {
        const int e = i * 256 + threadIdx.x;
        row[e >> 3][e & 7] = r[i];
        grad[e >> 3][e & 7] = g[i];
      }
      __syncthreads();
      const int texts = int(min64(kTexts, p.B - b0));
      for (int q32 = 0; q32 < texts; q32 += 32) {
        const int32_t r = row[q32 + lane][wid];
        const float g = grad[q32 + lane][wid];
        if (d0 == 0) db += g;
        uint32_t live = __ballot_sync(FULL, r >= 0);
        if (!gather) continue;
        while (live) {
          uint4 x[4][kCols];         // four rows in flight
          float gs[4];
#pragma unroll
          for (int t = 0; t < 4; ++t) {
            const int src = live ? __ffs(live) - 1 : 0;
            const int32_t rs = __shfl_sync(FULL, r, src);
            gs[t] = live ? __shfl_sync(FULL, g, src) : 0.0f;
            load_row(p.h + int64_t(live ? rs : 0) * p.Dp, d0, live ? p.Dp : 0, lane, x[t]);
            live &= live - 1;
          }
#pragma unroll
          for (int t = 0; t < 4; ++t) add_row(acc, x[t], gs[t], bf);
        }
      }
    }
    if (!gather || v >= p.V) continue;
#pragma unroll
    for (int q = 0; q < kCols; ++q) {
      const int64_t c = d0 + q * 256 + lane * 8;
      if (c < p.D) store8(p.dw + v * p.D + c, int(min64(8, p.D - c)), acc[q], bf);
    }
  }
  if (p.db) {
    for (int o = 16; o > 0; o >>= 1) db += __shfl_xor_sync(FULL, db, o);
    if (lane == 0 && v < p.V) p.db[v] = db;
  }
}

// dH: a warp per packed row, eight rows per CTA; a lane has 8 columns of every 256 (up to 1024
// columns; blockIdx.y goes on).  A row with more than kHeavy entries (a token may have won most
// of the vocabulary) is shared by the CTA's warps afterwards, whose sums are added in order.
constexpr int kHeavy = 256;
template <int kCols>
__device__ __forceinline__ void gather_run(const GatherParams& p, int32_t lo, int32_t hi, int64_t d0, int lane, bool bf,
                                           float (&acc)[kCols][8]) {
#pragma unroll
  for (int q = 0; q < kCols; ++q) {
#pragma unroll
    for (int k = 0; k < 8; ++k) acc[q][k] = 0.0f;
  }
  for (int32_t i0 = lo; i0 < hi; i0 += 32) {
    int2 e = make_int2(0, 0);
    if (i0 + lane < hi) e = p.list[i0 + lane];
    const int32_t m = min(32, hi - i0);
    for (int32_t i = 0; i < m; i += 4) {
      uint4 x[4][kCols];
      float g[4];
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        const int32_t v = __shfl_sync(FULL, e.x, i + t);
        g[t] = __int_as_float(__shfl_sync(FULL, e.y, i + t));      // 0 past the last entry
        load_row(p.w + int64_t(v) * p.ldw, d0, i + t < m ? p.D : 0, lane, x[t]);
      }
#pragma unroll
      for (int t = 0; t < 4; ++t) add_row(acc, x[t], g[t], bf);
    }
  }
}
template <int kCols>
__global__ void __launch_bounds__(256, 2) gather_hidden_kernel(const GatherParams p) {
  mm::after_previous();
  __shared__ float4 sums[7][2][32];
  const int32_t n = p.head[0], r0 = blockIdx.x * 8;
  if (r0 >= n || !p.sparse.gather(n, p.V)) return;
  const int wid = threadIdx.x >> 5, lane = lane_id();
  const bool bf = p.bf16 != 0;
  const int64_t d0 = int64_t(blockIdx.y) * 256 * kCols;
  float acc[kCols][8];
  const int32_t r = r0 + wid;
  int32_t e0 = 0, e1 = 0;
  if (r < n) {
    e0 = int32_t(p.offset[int64_t(r) * kSegs]);
    e1 = int32_t(p.offset[int64_t(r + 1) * kSegs]);
  }
  if (e1 > e0 && e1 - e0 <= kHeavy) {              // (a row without entries is zero already)
    gather_run(p, e0, e1, d0, lane, bf, acc);
    uint16_t* out = p.dh + int64_t(p.map[r]) * p.D;
#pragma unroll
    for (int q = 0; q < kCols; ++q) {
      const int64_t c = d0 + q * 256 + lane * 8;
      if (c < p.D) store8(out + c, int(min64(8, p.D - c)), acc[q], bf);
    }
  }
  if (!__syncthreads_or(e1 - e0 > kHeavy)) return;
  for (int32_t h = r0; h < min(n, r0 + 8); ++h) {
    e0 = int32_t(p.offset[int64_t(h) * kSegs]);
    e1 = int32_t(p.offset[int64_t(h + 1) * kSegs]);
    if (e1 - e0 <= kHeavy) continue;
    const int32_t per = (e1 - e0 + 7) / 8, lo = min(e0 + wid * per, e1);
    gather_run(p, lo, min(lo + per, e1), d0, lane, bf, acc);
#pragma unroll
    for (int q = 0; q < kCols; ++q) {
      const int64_t c0 = d0 + q * 256, c = c0 + lane * 8;
      if (c0 >= p.D) break;
      __syncthreads();
      if (wid > 0) {
        sums[wid - 1][0][lane] = make_float4(acc[q][0], acc[q][1], acc[q][2], acc[q][3]);
        sums[wid - 1][1][lane] = make_float4(acc[q][4], acc[q][5], acc[q][6], acc[q][7]);
      }
      __syncthreads();
      if (wid > 0 || c >= p.D) continue;
#pragma unroll
      for (int w = 0; w < 7; ++w) {
        const float4 a = sums[w][0][lane], b = sums[w][1][lane];
        acc[q][0] += a.x, acc[q][1] += a.y, acc[q][2] += a.z, acc[q][3] += a.w;
        acc[q][4] += b.x, acc[q][5] += b.y, acc[q][6] += b.z, acc[q][7] += b.w;
      }
      store8(p.dh + int64_t(p.map[h]) * p.D + c, int(min64(8, p.D - c)), acc[q], bf);
    }
  }
}

struct SpreadParams {
  const int32_t *head, *text;
  const float *y, *dy;
  const int32_t* win;
  const Survey* survey;
  Sparse sparse;
  float* scale;
  uint16_t* P;
  int64_t pitch, v0, cols, V, B;
  int32_t bf16;
};
// P = ds * this, at most 2^100: the quotient leaves fp32 for |dy| below 5e-35, and the gradients of
// entries that 2^100 lifts to no more than 2^14 are far below fp16's smallest numbers anyway
__device__ __forceinline__ float p_scale(const Survey* s, bool bf16) {
  const float m = bf16 ? 0.0f : __uint_as_float(s->absmax);
  return m > 0.0f ? fminf(16384.0f / m, 0x1p100f) : 1.0f;
}
constexpr int kSpreadRows = 64;
// P of a piece: a thread owns 8 columns of one text and writes them for kSpreadRows of its rows
// (of every gridDim.z x kSpreadRows, for texts longer than a grid is deep); the blocks of text B
// zero the rows past the packed ones.
__global__ void __launch_bounds__(256) spread_kernel(const SpreadParams p) {
  mm::after_previous();
  const int32_t n = p.head[0];
  if (p.sparse.gather(n, p.V)) return;
  const int64_t c = (int64_t(blockIdx.x) * 256 + threadIdx.x) * 8;
  const int64_t b = blockIdx.y;
  const float up_by = p_scale(p.survey, p.bf16 != 0);
  if (blockIdx.x == 0 && b == 0 && blockIdx.z == 0 && threadIdx.x == 0) *p.scale = 1.0f / up_by;
  const int32_t r0 = (b < p.B ? p.text[b] : n) + blockIdx.z * kSpreadRows;
  const int32_t end = b < p.B ? p.text[b + 1] : (n + mm::kBM - 1) / mm::kBM * mm::kBM;
  if (r0 >= end || c >= p.pitch) return;
  int32_t w[8];
  float ds[8];
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    const int64_t v = p.v0 + c + k;
    w[k] = -1;
    ds[k] = 0.0f;
    if (b < p.B && c + k < p.cols) {
      w[k] = p.win[b * p.V + v];
      if (w[k] >= 0) ds[k] = p.dy[b * p.V + v] * expf(-p.y[b * p.V + v]) * up_by;
    }
  }
  for (int64_t rz = r0; rz < end; rz += int64_t(gridDim.z) * kSpreadRows) {
    const int32_t r1 = int32_t(min64(end, rz + kSpreadRows));
    for (int32_t r = int32_t(rz); r < r1; ++r) {
      uint4 o;
      uint32_t* u = &o.x;
#pragma unroll
      for (int k = 0; k < 4; ++k)
        u[k] = pack2(w[2 * k] == r ? ds[2 * k] : 0.0f, w[2 * k + 1] == r ? ds[2 * k + 1] : 0.0f, p.bf16 != 0);
      *reinterpret_cast<uint4*>(p.P + int64_t(r) * p.pitch + c) = o;
    }
  }
}

// ---- dense rows -> CSR -------------------------------------------------------------------
__global__ void __launch_bounds__(1024) rows_count_kernel(const float* y, int64_t V, float min_weight, int32_t* nnz) {
  mm::after_previous();
  __shared__ int32_t part[32];
  const float* row = y + int64_t(blockIdx.x) * V;
  int32_t n = 0;
  for (int64_t v = threadIdx.x; v < V; v += 1024) n += row[v] > min_weight;
  n = __reduce_add_sync(FULL, n);
  if (lane_id() == 0) part[threadIdx.x >> 5] = n;
  __syncthreads();
  if (threadIdx.x < 32) {
    n = __reduce_add_sync(FULL, part[threadIdx.x]);
    if (threadIdx.x == 0) nnz[blockIdx.x] = n;
  }
}
__global__ void __launch_bounds__(1024)
rows_fill_kernel(const float* y, int64_t V, float min_weight, const int64_t* indptr, int32_t* indices, float* data) {
  mm::after_previous();
  __shared__ int32_t part[32];
  const float* row = y + int64_t(blockIdx.x) * V;
  const int wid = threadIdx.x >> 5, lane = lane_id();
  int64_t at = indptr[blockIdx.x];
  const int64_t end = indptr[blockIdx.x + 1];
  for (int64_t v0 = 0; v0 < V; v0 += 1024) {
    const int64_t v = v0 + threadIdx.x;
    const float x = v < V ? row[v] : 0.0f;
    const bool keep = v < V && x > min_weight;
    const uint32_t w = __ballot_sync(FULL, keep);
    if (lane == 0) part[wid] = __popc(w);
    __syncthreads();
    const int32_t mine = part[lane];
    const int32_t before = __reduce_add_sync(FULL, lane < wid ? mine : 0), all = __reduce_add_sync(FULL, mine);
    __syncthreads();
    const int64_t o = at + before + __popc(w & lanemask_lt());
    if (keep && o < end) {       // never past the counted entries
      indices[o] = int32_t(v);
      data[o] = x;
    }
    at += all;
  }
}

// ---- host --------------------------------------------------------------------------------
struct Fwd {
  int32_t *counts, *part_i;
  float* part_m;
  int64_t bytes;
};
Fwd carve_fwd(void* base, const gsp_vocab_view* vw) {
  Fwd f{};
  Carver c{static_cast<char*>(base)};
  f.counts = c.take<int32_t>(pack_counts(vw->T));
  f.part_m = c.take<float>(int64_t(mm::pair_ctas()) * mm::kBM);
  f.part_i = c.take<int32_t>(int64_t(mm::pair_ctas()) * mm::kBM);
  f.bytes = c.off;
  return f;
}
struct Bwd {
  Survey* survey;
  int32_t* count;
  int64_t* offset;
  void* scan;
  float* scale;
  GradScratch grad;
  uint16_t* P;        // or the list
  int64_t zeroed, scan_bytes, room;
  int64_t pitch, bytes;
};
Bwd carve_bwd(void* base, const gsp_vocab_view* vw) {
  Bwd b{};
  Carver c{static_cast<char*>(base)};
  const int64_t Tp = pad_rows(vw->T);
  b.pitch = piece_cols(Tp, vw->V);
  b.survey = c.take<Survey>(1);
  b.count = c.take<int32_t>(vw->T * kSegs);
  b.zeroed = c.off;
  b.offset = c.take<int64_t>(vw->T * kSegs + 1);
  b.scan_bytes = gsp_scan_ws_bytes(vw->T * kSegs);
  b.scan = c.take<char>(b.scan_bytes);
  b.scale = c.take<float>(1);
  b.grad = carve_grad(c, vw, Tp, b.pitch);
  b.P = c.take<uint16_t>(Tp * b.pitch);
  // (positions in the list are 32-bit)
  b.room = min64(Tp * b.pitch * 2 / int64_t(sizeof(int2)), (int64_t(1) << 31) - 64);
  b.bytes = c.off;
  return b;
}

template <bool kWin>
int run_head(const gsp_vocab_view* vw, const State& s, const Fwd& f, int32_t L, int32_t bn, float* y, int32_t* win,
             cudaStream_t st) {
  const Weight w = weight_rows(vw, s);
  HeadJob<kWin> j{};
  j.wait_limit = gsp_get_wait_limit();
  j.bf16 = is_bf16(vw);
  j.head = s.head;
  j.map = s.map;
  j.L = L;
  j.V = int32_t(vw->V);
  j.nvt = int32_t((vw->V + mm::kBM - 1) / mm::kBM);
  j.nk = int32_t((vw->D + mm::kBK - 1) / mm::kBK);
  j.bn = bn;
  j.bias = vw->bias;
  j.y = y;
  j.win = win;
  j.part_m = f.part_m;
  j.part_i = f.part_i;
  const bool bf = is_bf16(vw);
  int rc;
  if ((rc = make_map(&j.maps[0], bf, w.w, vw->D, vw->V, w.ld, mm::kRows))) return rc;
  if ((rc = make_map(&j.maps[1], bf, s.h, s.Dp, vw->T, s.Dp, bn / 2))) return rc;
  return launch_mma(j, st);
}

// blocks of 256 columns that a lane of the gathering kernels holds
int gather_cols(int64_t D) { return D > 768 ? 4 : int((D + 255) / 256); }

int check_texts(const gsp_vocab_view* vw, int64_t L, const char* what) {
  const int rc = check_view(vw, what);
  if (rc) return rc;
  GSP_REQUIRE(L >= 1 && vw->T % L == 0, GSP_ERR_ARG, "%s: %lld tokens are not whole texts of %lld", what, (long long)vw->T,
              (long long)L);
  GSP_REQUIRE(vw->T / L <= 65534, GSP_ERR_ARG, "%s: more than 65534 texts in one call", what);
  return GSP_OK;
}

}  // namespace

int64_t head_ws_bytes(const gsp_vocab_view* vw, bool backward) {
  return backward ? carve_bwd(nullptr, vw).bytes : carve_fwd(nullptr, vw).bytes;
}
int64_t loss_ws_bytes(const gsp_vocab_view* vw, int64_t K, bool backward);

}  // namespace vocab
}  // namespace gsp

using namespace gsp;
using namespace gsp::vocab;

extern "C" int64_t gsp_vocab_ws_bytes(const gsp_vocab_view* vw, int64_t K, int32_t kind, int32_t backward) {
  const int rc = check_view(vw, "gsp_vocab_ws_bytes");
  if (rc) return -rc;
  if (kind < GSP_VOCAB_CE || kind > GSP_VOCAB_HEAD || K < 0) {
    set_error("gsp_vocab_ws_bytes: bad arguments");
    return -GSP_ERR_ARG;
  }
  return kind == GSP_VOCAB_HEAD ? head_ws_bytes(vw, backward != 0) : loss_ws_bytes(vw, kind == GSP_VOCAB_DISTILL ? K : 0, backward != 0);
}

extern "C" int gsp_sparse_head(const gsp_vocab_view* vw, int64_t L, const uint8_t* mask, float* y, int32_t* win, void* state,
                               int64_t state_bytes, void* ws, int64_t ws_bytes, void* stream) {
  int rc = check_texts(vw, L, "sparse_head");
  if (rc) return rc;
  const State s = carve_state(state, vw, 0, vw->T > 0 ? vw->T : 1);
  const Fwd f = carve_fwd(ws, vw);
  if ((rc = check_buffers(state, state_bytes, s.bytes, ws, ws_bytes, f.bytes, "sparse_head"))) return rc;
  if (vw->T == 0) return GSP_OK;
  GSP_REQUIRE(vw->hidden && vw->weight && y, GSP_ERR_ARG, "sparse_head: null input or output");
  cudaStream_t st = as_stream(stream);
  if ((rc = pack_rows(vw, nullptr, 0, mask, 0.0f, Texts{L, y, win}, s, f.counts, st))) return rc;
  // columns of a tile: no more than the tokens need (a single query's product is then as short
  // as reading W allows)
  const int32_t bn = int32_t(vw->T >= mm::kBN ? mm::kBN : up(vw->T, 64));
  rc = win ? run_head<true>(vw, s, f, int32_t(L), bn, y, win, st)
           : run_head<false>(vw, s, f, int32_t(L), bn, y, win, st);
  if (rc || vw->T <= bn) return rc;      // one tile of tokens: no share cuts a text
  JoinParams p{};
  p.head = s.head;
  p.map = s.map;
  p.L = int32_t(L);
  p.bn = bn;
  p.pairs = mm::pair_ctas() / 2;
  p.V = vw->V;
  p.nvt = int32_t((vw->V + mm::kBM - 1) / mm::kBM);
  p.bias = vw->bias;
  p.part_m = f.part_m;
  p.part_i = f.part_i;
  p.y = y;
  p.win = win;
  return launch(head_join_kernel, dim3(unsigned(p.pairs)), mm::kBM, 0, st, p);
}

extern "C" int gsp_sparse_head_backward(const gsp_vocab_view* vw, int64_t L, const float* y, const int32_t* win,
                                        const float* dy, void* d_hidden, void* d_weight, float* d_bias, void* state,
                                        int64_t state_bytes, void* ws, int64_t ws_bytes, void* stream) {
  int rc = check_texts(vw, L, "sparse_head backward");
  if (rc) return rc;
  if ((rc = check_grads(vw, d_hidden, d_weight, "sparse_head backward"))) return rc;
  const State s = carve_state(state, vw, 0, vw->T > 0 ? vw->T : 1);
  const Bwd b = carve_bwd(ws, vw);
  if ((rc = check_buffers(state, state_bytes, s.bytes, ws, ws_bytes, b.bytes, "sparse_head backward"))) return rc;
  cudaStream_t st = as_stream(stream);
  if (vw->T == 0) {
    if (d_weight) GSP_CUDA(cudaMemsetAsync(d_weight, 0, size_t(vw->V) * size_t(vw->D) * 2, st));
    if (d_bias) GSP_CUDA(cudaMemsetAsync(d_bias, 0, size_t(vw->V) * sizeof(float), st));
    return GSP_OK;
  }
  GSP_REQUIRE(y && win && dy && vw->weight, GSP_ERR_ARG, "sparse_head backward: null input");
  const int64_t B = vw->T / L;
  const bool bf = is_bf16(vw);
  const Weight w = weight_rows(vw, s);
  // longer texts than the sort has counters for take the products
  const bool sort = d_hidden && L * 4 <= kSortSmem, may = !d_hidden || sort;
  GSP_CUDA(cudaMemsetAsync(b.survey, 0, size_t(sort ? b.zeroed : int64_t(sizeof(Survey))), st));
  SortParams q{};
  q.head = s.head;
  q.text = s.text;
  q.y = y;
  q.dy = dy;
  q.win = win;
  q.B = B;
  q.V = vw->V;
  q.L = sort ? int32_t(L) : 0;
  q.count = b.count;
  q.offset = b.offset;
  q.list = reinterpret_cast<int2*>(b.P);
  q.sparse = Sparse{may ? &b.survey->nnz : nullptr, b.room};
  const int warps = sort ? sort_warps(L) : 8;
  const unsigned sort_blocks = unsigned((B * kSegs + warps - 1) / warps);
  const size_t sort_bytes = sort ? size_t(warps) * size_t(L) * 4 : 0;
  rc = launch(survey_kernel, dim3(sort_blocks), 32 * warps, sort_bytes, st, s, q, b.survey, d_hidden, vw->T * vw->D * 2);
  if (rc) return rc;
  if (sort) {
    if ((rc = gsp_scan_i32(b.count, vw->T * kSegs, b.offset, b.scan, b.scan_bytes, stream))) return rc;
    if ((rc = launch(place_kernel, dim3(sort_blocks), 32 * warps, sort_bytes, st, q))) return rc;
  }
  GatherParams g{};
  g.head = s.head;
  g.map = s.map;
  g.sparse = q.sparse;
  g.offset = b.offset;
  g.list = q.list;
  g.y = y;
  g.dy = dy;
  g.win = win;
  g.h = s.h;
  g.w = w.w;
  g.Dp = s.Dp;
  g.ldw = w.ld;
  g.B = B;
  g.V = vw->V;
  g.D = vw->D;
  g.bf16 = bf;
  g.dh = static_cast<uint16_t*>(d_hidden);
  g.dw = static_cast<uint16_t*>(d_weight);
  g.db = d_bias;
  if (d_weight || d_bias) {
    const unsigned blocks = unsigned((vw->V + 7) / 8);
    const int cols = gather_cols(vw->D);
    const auto kernel = cols == 1   ? gather_weight_kernel<1>
                        : cols == 2 ? gather_weight_kernel<2>
                        : cols == 3 ? gather_weight_kernel<3>
                                    : gather_weight_kernel<4>;
    if ((rc = launch(kernel, dim3(blocks), 256, 0, st, g))) return rc;
  }
  if (sort) {
    const dim3 blocks(unsigned((vw->T + 7) / 8), unsigned((vw->D + 1023) / 1024));
    const int cols = gather_cols(vw->D);
    const auto kernel = cols == 1   ? gather_hidden_kernel<1>
                        : cols == 2 ? gather_hidden_kernel<2>
                        : cols == 3 ? gather_hidden_kernel<3>
                                    : gather_hidden_kernel<4>;
    if ((rc = launch(kernel, blocks, 256, 0, st, g))) return rc;
  }
  if (!d_hidden && !d_weight) return GSP_OK;
  SpreadParams p{};
  p.head = s.head;
  p.text = s.text;
  p.y = y;
  p.dy = dy;
  p.win = win;
  p.survey = b.survey;
  p.sparse = q.sparse;
  p.scale = b.scale;
  p.P = b.P;
  p.pitch = b.pitch;
  p.V = vw->V;
  p.B = B;
  p.bf16 = bf;
  const int64_t zs = min64(((L < mm::kBM ? mm::kBM : L) + kSpreadRows - 1) / kSpreadRows, 65535);
  for (int64_t v0 = 0; v0 < vw->V; v0 += b.pitch) {
    p.v0 = v0;
    p.cols = min64(b.pitch, vw->V - v0);
    rc = launch(spread_kernel, dim3(unsigned((b.pitch / 8 + 255) / 256), unsigned(B + 1), unsigned(zs)), 256, 0, st, p);
    if (rc) return rc;
    const GradPiece pc{b.P, b.pitch, v0, p.cols, v0 == 0, v0 + p.cols >= vw->V, q.sparse};
    if ((rc = grad_products(vw, s, w.w, w.ld, pc, b.grad, BiasSums{}, b.scale, d_hidden, d_weight, st))) return rc;
  }
  return GSP_OK;
}

extern "C" int gsp_dense_rows_count(const float* y, int64_t B, int64_t V, float min_weight, int32_t* nnz, void* stream) {
  GSP_REQUIRE(B >= 0 && V >= 1 && (B == 0 || (y && nnz)), GSP_ERR_ARG, "gsp_dense_rows_count: bad arguments");
  if (B == 0) return GSP_OK;
  return launch(rows_count_kernel, dim3(unsigned(B)), 1024, 0, as_stream(stream), y, V, min_weight, nnz);
}

extern "C" int gsp_dense_rows_fill(const float* y, int64_t B, int64_t V, float min_weight, const int64_t* indptr,
                                   int32_t* indices, float* data, void* stream) {
  GSP_REQUIRE(B >= 0 && V >= 1 && (B == 0 || (y && indptr)), GSP_ERR_ARG, "gsp_dense_rows_fill: bad arguments");
  if (B == 0) return GSP_OK;
  return launch(rows_fill_kernel, dim3(unsigned(B)), 1024, 0, as_stream(stream), y, V, min_weight, indptr, indices, data);
}
