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
// kernel.  Texts may so have any length, and no work is lost to their padding.
//
// Backward.  Each (text, term) with y > 0 sends ds = dy exp(-y) to its winning token; as a
// matrix P [tokens, V] with one entry per (text, term) this is the shape of the losses'
// gradient, and the same two products finish it.
#include "vocab.cuh"

namespace gsp {
namespace vocab {
namespace {

constexpr int kFirst = 1, kLast = 2;      // of a share along one row of tiles
constexpr int kBegin = 4, kEnd = 8;       // of a share

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
      t.a_mn = t.b_mn = t.a_stream = false;
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
    __device__ static void put(const HeadJob& j, int32_t row, int32_t v, float bias, float m, int32_t idx) {
      if (v >= j.V) return;
      const float x = m + bias;
      const int64_t o = int64_t(j.map[row] / j.L) * j.V + v;
      j.y[o] = x > 0.0f ? log1pf(x) : (x != x ? x : 0.0f);
      if (kWin) j.win[o] = x > 0.0f ? idx : -1;
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
#pragma unroll
            for (int k = 0; k < 16; ++k) {
              if (kWin) won = z[16 * h + k] > m ? k : won;
              asm("max.NaN.f32 %0, %0, %1;" : "+f"(m) : "f"(z[16 * h + k]));
            }
            if (kWin && won >= 0) idx = rb + won;
          } else {
            int32_t e = 0;
#pragma unroll
            for (int k = 0; k < 16; ++k) {
              if (kWin) idx = z[16 * h + k] > m ? rb + k : idx;
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
        const int32_t hi = kWin && head_m > cm ? head_i : ci;
        asm("max.NaN.f32 %0, %0, %1;" : "+f"(head_m) : "f"(cm));
        if (cut) part(j, a, 0, head_m, hi);
        else put(j, head_row, v, bias, head_m, hi);
        cut = false;
      } else {
        if (kWin) open_i = m > cm ? idx : ci;
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
  const uint8_t* mask;
  int32_t L, bn, pairs, nvt;
  int64_t B, V;
  const float* bias;
  const float* part_m;
  const int32_t* part_i;
  float* y;
  int32_t* win;
};

// Blocks [0, pairs): a text that began in an earlier share and ends in this one is joined from
// the shares it crosses, in order.  Blocks past them: texts without tokens get zero rows.
__global__ void __launch_bounds__(mm::kBM) head_join_kernel(const JoinParams p) {
  const int32_t n = p.head[0];
  if (int32_t(blockIdx.x) >= p.pairs) {
    const int64_t b = int64_t(blockIdx.x) - p.pairs;
    bool any = false;
    for (int64_t t = threadIdx.x; t < p.L; t += mm::kBM) any |= p.mask[b * p.L + t] != 0;
    if (__syncthreads_or(any)) return;
    for (int64_t v = threadIdx.x; v < p.V; v += mm::kBM) {
      p.y[b * p.V + v] = 0.0f;
      if (p.win) p.win[b * p.V + v] = -1;
    }
    return;
  }
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
    if (p.win && x > m) idx = p.part_i[o];
    asm("max.NaN.f32 %0, %0, %1;" : "+f"(m) : "f"(x));
  }
  const int64_t v = int64_t(vt) * mm::kBM + threadIdx.x;
  if (v >= p.V) return;
  const float x = m + (p.bias ? p.bias[v] : 0.0f);
  p.y[text * p.V + v] = x > 0.0f ? log1pf(x) : (x != x ? x : 0.0f);
  if (p.win) p.win[text * p.V + v] = x > 0.0f ? idx : -1;
}

// ---- backward ----------------------------------------------------------------------------
// largest finite |dy| (fp16: an upper bound of |ds|, which scales P)
__global__ void __launch_bounds__(256) absmax_kernel(const float* dy, int64_t n, uint32_t* out) {
  float m = 0.0f;
  for (int64_t i = int64_t(blockIdx.x) * 256 + threadIdx.x; i < n; i += int64_t(gridDim.x) * 256) {
    const float a = fabsf(dy[i]);
    if (a < __uint_as_float(0x7F800000u)) m = fmaxf(m, a);
  }
  const uint32_t w = __reduce_max_sync(FULL, __float_as_uint(m));
  if (lane_id() == 0 && w) atomicMax(out, w);
}

__global__ void __launch_bounds__(1024) tail_kernel(State s) { zero_tail_rows(s.h, s.Dp, s.head[0]); }

struct SpreadParams {
  const int32_t *head, *map;
  const float *y, *dy;
  const int32_t* win;
  const uint32_t* absmax;       // fp16 only
  float* scale;
  uint16_t* P;
  int64_t pitch, v0, cols, V, B;
  int32_t L, bf16;
};
__device__ __forceinline__ float p_scale(const uint32_t* absmax) {     // P = ds * this
  const float m = absmax ? __uint_as_float(*absmax) : 0.0f;
  return m > 0.0f ? 16384.0f / m : 1.0f;
}
__device__ __forceinline__ int32_t lower_row(const int32_t* map, int32_t n, int64_t key) {
  int32_t lo = 0, hi = n;
  while (lo < hi) {
    const int32_t mid = (lo + hi) >> 1;
    if (map[mid] < key) lo = mid + 1;
    else hi = mid;
  }
  return lo;
}
constexpr int kSpreadRows = 64;
// P of a piece: a thread owns 8 columns of one text and writes them for up to kSpreadRows of
// its rows; the blocks of text B zero the rows past the packed ones.
__global__ void __launch_bounds__(256) spread_kernel(const SpreadParams p) {
  const int32_t n = p.head[0];
  const int64_t c = (int64_t(blockIdx.x) * 256 + threadIdx.x) * 8;
  const int64_t b = blockIdx.y;
  const float up_by = p_scale(p.absmax);
  if (blockIdx.x == 0 && b == 0 && blockIdx.z == 0 && threadIdx.x == 0) *p.scale = 1.0f / up_by;
  int32_t r0, r1;
  if (b < p.B) {
    r0 = lower_row(p.map, n, b * p.L) + blockIdx.z * kSpreadRows;
    r1 = min(lower_row(p.map, n, (b + 1) * p.L), r0 + kSpreadRows);
  } else {
    r0 = n + blockIdx.z * kSpreadRows;
    r1 = min((n + mm::kBM - 1) / mm::kBM * mm::kBM, r0 + kSpreadRows);
  }
  if (r0 >= r1 || c >= p.pitch) return;
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
  for (int32_t r = r0; r < r1; ++r) {
    uint4 o;
    uint32_t* u = &o.x;
#pragma unroll
    for (int k = 0; k < 4; ++k)
      u[k] = pack2(w[2 * k] == r ? ds[2 * k] : 0.0f, w[2 * k + 1] == r ? ds[2 * k + 1] : 0.0f, p.bf16 != 0);
    *reinterpret_cast<uint4*>(p.P + int64_t(r) * p.pitch + c) = o;
  }
}

__global__ void __launch_bounds__(256) head_bias_kernel(const float* y, const int32_t* win, const float* dy, int64_t B, int64_t V,
                                                        float* d_bias) {
  const int64_t v = int64_t(blockIdx.x) * 256 + threadIdx.x;
  if (v >= V) return;
  float s = 0.0f;
  for (int64_t b = 0; b < B; ++b) {
    if (win[b * V + v] >= 0) s += dy[b * V + v] * expf(-y[b * V + v]);
  }
  d_bias[v] = s;
}

// ---- dense rows -> CSR -------------------------------------------------------------------
__global__ void __launch_bounds__(1024) rows_count_kernel(const float* y, int64_t V, float min_weight, int32_t* nnz) {
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
  void* wcopy;
  int64_t bytes;
};
Fwd carve_fwd(void* base, const gsp_vocab_view* vw) {
  Fwd f{};
  Carver c{static_cast<char*>(base)};
  f.counts = c.take<int32_t>(pack_counts(vw->T));
  f.part_m = c.take<float>(int64_t(mm::pair_ctas()) * mm::kBM);
  f.part_i = c.take<int32_t>(int64_t(mm::pair_ctas()) * mm::kBM);
  f.wcopy = c.take<char>(weight_copy_bytes(vw));
  f.bytes = c.off;
  return f;
}
struct Bwd {
  uint32_t* absmax;
  float* scale;
  GradScratch grad;
  uint16_t* P;
  void* wcopy;
  int64_t pitch, bytes;
};
Bwd carve_bwd(void* base, const gsp_vocab_view* vw) {
  Bwd b{};
  Carver c{static_cast<char*>(base)};
  const int64_t Tp = pad_rows(vw->T);
  b.pitch = piece_cols(Tp, vw->V);
  b.absmax = c.take<uint32_t>(1);
  b.scale = c.take<float>(1);
  b.grad = carve_grad(c, vw, Tp, b.pitch);
  b.P = c.take<uint16_t>(Tp * b.pitch);
  b.wcopy = c.take<char>(weight_copy_bytes(vw));
  b.bytes = c.off;
  return b;
}

template <bool kWin>
int run_head(const gsp_vocab_view* vw, const State& s, const Fwd& f, int32_t L, int32_t bn, float* y, int32_t* win,
             const uint16_t* w, int64_t ldw, cudaStream_t st) {
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
  if ((rc = make_map(&j.maps[0], bf, w, vw->D, vw->V, ldw, mm::kRows))) return rc;
  if ((rc = make_map(&j.maps[1], bf, s.h, s.Dp, vw->T, s.Dp, bn / 2))) return rc;
  return mm::launch(j, st);
}

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
  const State s = carve_state(state, vw->T, vw->V, vw->D, 0, false);
  const Fwd f = carve_fwd(ws, vw);
  GSP_REQUIRE(state && state_bytes >= s.bytes && ws && ws_bytes >= f.bytes, GSP_ERR_ARG,
              "sparse_head: state or workspace too small");
  if (vw->T == 0) return GSP_OK;
  GSP_REQUIRE(vw->hidden && vw->weight && y, GSP_ERR_ARG, "sparse_head: null input or output");
  cudaStream_t st = as_stream(stream);
  if ((rc = pack_rows(vw, nullptr, 0, mask, 0.0f, s, f.counts, st))) return rc;
  const uint16_t* w;
  int64_t ldw;
  if ((rc = weight_rows(vw, f.wcopy, &w, &ldw, st))) return rc;
  // columns of a tile: no more than the tokens need (a single query's product is then as short
  // as reading W allows)
  const int32_t bn = int32_t(vw->T >= mm::kBN ? mm::kBN : up(vw->T, 64));
  rc = win ? run_head<true>(vw, s, f, int32_t(L), bn, y, win, w, ldw, st)
           : run_head<false>(vw, s, f, int32_t(L), bn, y, win, w, ldw, st);
  if (rc) return rc;
  JoinParams p{};
  p.head = s.head;
  p.map = s.map;
  p.mask = mask;
  p.L = int32_t(L);
  p.bn = bn;
  p.pairs = mm::pair_ctas() / 2;
  p.B = vw->T / L;
  p.V = vw->V;
  p.nvt = int32_t((vw->V + mm::kBM - 1) / mm::kBM);
  p.bias = vw->bias;
  p.part_m = f.part_m;
  p.part_i = f.part_i;
  p.y = y;
  p.win = win;
  head_join_kernel<<<unsigned(p.pairs + (mask ? p.B : 0)), mm::kBM, 0, st>>>(p);
  GSP_CHECK_LAUNCH();
  return GSP_OK;
}

extern "C" int gsp_sparse_head_backward(const gsp_vocab_view* vw, int64_t L, const float* y, const int32_t* win,
                                        const float* dy, void* d_hidden, void* d_weight, float* d_bias, void* state,
                                        int64_t state_bytes, void* ws, int64_t ws_bytes, void* stream) {
  int rc = check_texts(vw, L, "sparse_head backward");
  if (rc) return rc;
  if ((rc = check_grads(vw, d_hidden, d_weight, "sparse_head backward"))) return rc;
  const State s = carve_state(state, vw->T, vw->V, vw->D, 0, false);
  const Bwd b = carve_bwd(ws, vw);
  GSP_REQUIRE(state && state_bytes >= s.bytes && ws && ws_bytes >= b.bytes, GSP_ERR_ARG,
              "sparse_head backward: state or workspace too small");
  cudaStream_t st = as_stream(stream);
  if (vw->T == 0) {
    if (d_weight) GSP_CUDA(cudaMemsetAsync(d_weight, 0, size_t(vw->V) * size_t(vw->D) * 2, st));
    if (d_bias) GSP_CUDA(cudaMemsetAsync(d_bias, 0, size_t(vw->V) * sizeof(float), st));
    return GSP_OK;
  }
  GSP_REQUIRE(y && win && dy && vw->weight, GSP_ERR_ARG, "sparse_head backward: null input");
  const int64_t B = vw->T / L;
  if (d_bias) {
    head_bias_kernel<<<unsigned((vw->V + 255) / 256), 256, 0, st>>>(y, win, dy, B, vw->V, d_bias);
    GSP_CHECK_LAUNCH();
  }
  if (!d_hidden && !d_weight) return GSP_OK;
  if (d_hidden) GSP_CUDA(cudaMemsetAsync(d_hidden, 0, size_t(vw->T) * size_t(vw->D) * 2, st));
  const bool bf = is_bf16(vw);
  if (!bf) {
    GSP_CUDA(cudaMemsetAsync(b.absmax, 0, sizeof(uint32_t), st));
    absmax_kernel<<<num_sms() * 4, 256, 0, st>>>(dy, B * vw->V, b.absmax);
    GSP_CHECK_LAUNCH();
  }
  tail_kernel<<<1, 1024, 0, st>>>(s);
  GSP_CHECK_LAUNCH();
  const uint16_t* w;
  int64_t ldw;
  if ((rc = weight_rows(vw, b.wcopy, &w, &ldw, st))) return rc;
  SpreadParams p{};
  p.head = s.head;
  p.map = s.map;
  p.y = y;
  p.dy = dy;
  p.win = win;
  p.absmax = bf ? nullptr : b.absmax;
  p.scale = b.scale;
  p.P = b.P;
  p.pitch = b.pitch;
  p.V = vw->V;
  p.B = B;
  p.L = int32_t(L);
  p.bf16 = bf;
  const int64_t zs = ((L < mm::kBM ? mm::kBM : L) + kSpreadRows - 1) / kSpreadRows;
  GSP_REQUIRE(zs <= 65535, GSP_ERR_ARG, "sparse_head backward: texts of %lld tokens are too long", (long long)L);
  for (int64_t v0 = 0; v0 < vw->V; v0 += b.pitch) {
    p.v0 = v0;
    p.cols = min64(b.pitch, vw->V - v0);
    spread_kernel<<<dim3(unsigned((b.pitch / 8 + 255) / 256), unsigned(B + 1), unsigned(zs)), 256, 0, st>>>(p);
    GSP_CHECK_LAUNCH();
    const GradPiece pc{b.P, b.pitch, v0, p.cols, v0 == 0, v0 + p.cols >= vw->V};
    if ((rc = grad_products(vw, s, w, ldw, pc, b.grad, BiasSums{}, b.scale, d_hidden, d_weight, st))) return rc;
  }
  return GSP_OK;
}

extern "C" int gsp_dense_rows_count(const float* y, int64_t B, int64_t V, float min_weight, int32_t* nnz, void* stream) {
  GSP_REQUIRE(B >= 0 && V >= 1 && (B == 0 || (y && nnz)), GSP_ERR_ARG, "gsp_dense_rows_count: bad arguments");
  if (B == 0) return GSP_OK;
  rows_count_kernel<<<unsigned(B), 1024, 0, as_stream(stream)>>>(y, V, min_weight, nnz);
  GSP_CHECK_LAUNCH();
  return GSP_OK;
}

extern "C" int gsp_dense_rows_fill(const float* y, int64_t B, int64_t V, float min_weight, const int64_t* indptr,
                                   int32_t* indices, float* data, void* stream) {
  GSP_REQUIRE(B >= 0 && V >= 1 && (B == 0 || (y && indptr)), GSP_ERR_ARG, "gsp_dense_rows_fill: bad arguments");
  if (B == 0) return GSP_OK;
  rows_fill_kernel<<<unsigned(B), 1024, 0, as_stream(stream)>>>(y, V, min_weight, indptr, indices, data);
  GSP_CHECK_LAUNCH();
  return GSP_OK;
}
