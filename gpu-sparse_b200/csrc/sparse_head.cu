// The sparse head: y[b, v] = log1p(relu(max over the tokens t of text b of H[t] . W[v] + bias[v])),
// the term weights an index is built from, and its gradient.
//
// Forward.  The product is taken as W H^T, vocabulary rows in the tensor memory's lanes and
// packed tokens in its columns, so that the maximum over a text's tokens runs along one
// thread's registers: one compare per logit, no exchange between threads, and log1p only on
// the maximum (it is monotone).  Tiles are ordered tokens-fastest and cut into equal shares,
// one per CTA; the running maximum is carried from tile to tile, and a text that a share's
// border cuts leaves its partial maxima for a joining kernel.  Texts may so have any length,
// and no work is lost to their padding.
//
// Backward.  Each (text, term) with y > 0 sends ds = dy exp(-y) to its winning token; as a
// matrix P [tokens, V] with one entry per (text, term) this is the shape of the losses'
// gradient, and the same two products finish it.
#include "vocab.cuh"

namespace gsp {
namespace vocab {
namespace {

constexpr int kFirst = 1, kLast = 2;

template <bool kWin>
struct HeadJob {
  CUtensorMap maps[2];      // W, H (K-major)
  int32_t wait_limit, bf16;
  const int32_t* head;
  const int32_t* map;
  int32_t L, V, nvt, nk, bn;
  const float* bias;
  float* y;
  int32_t* win;
  float* part_m;            // [ctas][2][128]
  int32_t* part_i;

  struct Walk {
    int64_t lo, hi;
    int32_t ntt, nk, bn;
    __device__ bool get(int32_t i, mm::Tile& t) const {
      const int64_t x = lo + i;
      if (x >= hi) return false;
      t.x = int32_t(x / ntt);
      t.y = int32_t(x - int64_t(t.x) * ntt);
      t.a = 0, t.b = 1;
      t.a0 = t.x * mm::kBM;
      t.b0 = t.y * bn;
      t.ak = t.bk = 0;
      t.nk = nk;
      t.a_mn = t.b_mn = false;
      t.bn = bn;
      t.flags = (i == 0 || t.y == 0 ? kFirst : 0) | (x == hi - 1 || t.y == ntt - 1 ? kLast : 0);
      return true;
    }
  };
  __device__ Walk walk() const {
    const int32_t ntt = (head[0] + bn - 1) / bn;
    const int64_t tot = int64_t(ntt) * nvt;
    return Walk{share_lo(tot, gridDim.x, blockIdx.x), share_lo(tot, gridDim.x, blockIdx.x + 1), ntt, nk, bn};
  }

  struct Epi {
    float m;
    int32_t idx;
    bool cut;            // the open text began before this share
    __device__ void flush(const HeadJob& j, int32_t text, int32_t v, float bias, int slot_row) {
      if (cut) {
        const int64_t o = int64_t(blockIdx.x) * 2 * mm::kBM + slot_row;
        j.part_m[o] = m;
        if (kWin) j.part_i[o] = idx;
      } else if (v < j.V) {
        const float x = m + bias;
        const int64_t o = int64_t(text) * j.V + v;
        j.y[o] = x > 0.0f ? log1pf(x) : (x != x ? x : 0.0f);
        if (kWin) j.win[o] = x > 0.0f ? idx : -1;
      }
      cut = false;
      m = neg_inf();
      idx = -1;
    }
    __device__ void tile(const HeadJob& j, const mm::Tile& t, const mm::Acc& a) {
      const int32_t n = j.head[0];
      if (t.flags & kFirst) {
        m = neg_inf();
        idx = -1;
        cut = t.b0 > 0 && j.map[t.b0 - 1] / j.L == j.map[t.b0] / j.L;
      }
      const int slot_row = a.warp * 32 + a.lane;
      const int32_t v = t.a0 + slot_row;
      const float bias = j.bias && v < j.V ? __ldg(j.bias + v) : 0.0f;
      bool open = false;
      for (int32_t c0 = 0; c0 < t.bn; c0 += 32) {
        const int32_t r0 = t.b0 + c0;
        if (r0 >= n) break;
        float z[32];
        a.ld32(c0, z);
        // text of every column, and which columns end one
        const int32_t r = r0 + a.lane;
        const int32_t text = r < n ? j.map[r] / j.L : -1;
        const int32_t after = r + 1 < n ? j.map[r + 1] / j.L : -1;
        const uint32_t ends = __ballot_sync(FULL, r < n && text != after);
        int32_t won = -1;
        if (ends == 0) {
          // whole block inside a text
#pragma unroll
          for (int k = 0; k < 32; ++k) {
            if (kWin) won = z[k] > m ? k : won;
            asm("max.NaN.f32 %0, %0, %1;" : "+f"(m) : "f"(z[k]));
          }
          if (kWin && won >= 0) idx = r0 + won;
          open = true;
        } else {
          const int32_t live = min(32, n - r0);
#pragma unroll
          for (int k = 0; k < 32; ++k) {
            if (k < live) {
              if (kWin) idx = z[k] > m ? r0 + k : idx;
              asm("max.NaN.f32 %0, %0, %1;" : "+f"(m) : "f"(z[k]));
              if ((ends >> k) & 1) flush(j, __shfl_sync(FULL, text, k), v, bias, slot_row);
            }
          }
          open = !((ends >> (live - 1)) & 1);
        }
      }
      if ((t.flags & kLast) && open) {
        const int64_t o = (int64_t(blockIdx.x) * 2 + 1) * mm::kBM + slot_row;
        j.part_m[o] = m;
        if (kWin) j.part_i[o] = idx;
      }
    }
  };
  __device__ Epi epi() const { return Epi{}; }
};

struct JoinParams {
  const int32_t *head, *map;
  const uint8_t* mask;
  int32_t L, bn, ctas;
  int64_t B, V, nvt;
  const float* bias;
  const float* part_m;
  const int32_t* part_i;
  float* y;
  int32_t* win;
};

// Blocks [0, ctas): a text that began in an earlier share and ends in this one is joined from
// the shares it crosses, in order.  Blocks past them: texts without tokens get zero rows.
__global__ void __launch_bounds__(mm::kBM) head_join_kernel(const JoinParams p) {
  const int32_t n = p.head[0];
  if (int32_t(blockIdx.x) >= p.ctas) {
    const int64_t b = int64_t(blockIdx.x) - p.ctas;
    bool any = p.mask == nullptr && p.L > 0;
    if (p.mask) {
      for (int64_t t = threadIdx.x; t < p.L; t += mm::kBM) any |= p.mask[b * p.L + t] != 0;
    }
    if (__syncthreads_or(any)) return;
    for (int64_t v = threadIdx.x; v < p.V; v += mm::kBM) {
      p.y[b * p.V + v] = 0.0f;
      if (p.win) p.win[b * p.V + v] = -1;
    }
    return;
  }
  const int32_t ntt = (n + p.bn - 1) / p.bn;
  const int64_t tot = int64_t(ntt) * p.nvt, c = blockIdx.x;
  const int64_t lo = share_lo(tot, p.ctas, c), hi = share_lo(tot, p.ctas, c + 1);
  if (lo >= hi) return;
  const int64_t vt = lo / ntt, t0 = lo - vt * ntt;
  if (t0 == 0) return;
  const int64_t r0 = t0 * p.bn;
  const int32_t text = p.map[r0] / p.L;
  if (p.map[r0 - 1] / p.L != text) return;
  // does it end inside this share?
  const int64_t row_end = min64(n, (min64(hi, (vt + 1) * ntt) - vt * ntt) * p.bn);
  if (row_end < n && p.map[row_end] / p.L == text) return;
  int64_t first = c - 1;
  for (;; --first) {
    const int64_t l0 = share_lo(tot, p.ctas, first);
    if (l0 == share_lo(tot, p.ctas, first + 1)) continue;      // an empty share
    const int64_t at = (l0 - vt * ntt) * p.bn;                 // its first row for this tile row
    if (at <= 0 || p.map[at - 1] / p.L != text) break;
  }
  float m = neg_inf();
  int32_t idx = -1;
  for (int64_t s = first; s <= c; ++s) {
    if (share_lo(tot, p.ctas, s) == share_lo(tot, p.ctas, s + 1)) continue;
    const int64_t o = (s * 2 + (s == c ? 0 : 1)) * mm::kBM + threadIdx.x;
    const float x = p.part_m[o];
    if (p.win && x > m) idx = p.part_i[o];
    asm("max.NaN.f32 %0, %0, %1;" : "+f"(m) : "f"(x));
  }
  const int64_t v = vt * mm::kBM + threadIdx.x;
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
  f.part_m = c.take<float>(int64_t(num_sms()) * 2 * mm::kBM);
  f.part_i = c.take<int32_t>(int64_t(num_sms()) * 2 * mm::kBM);
  f.wcopy = c.take<char>(weight_copy_bytes(vw));
  f.bytes = c.off;
  return f;
}
struct Bwd {
  uint32_t* absmax;
  float *scale, *dh_acc;
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
  b.dh_acc = c.take<float>(b.pitch < vw->V ? Tp * up(vw->D, 32) : 0);
  b.P = c.take<uint16_t>(Tp * b.pitch);
  b.wcopy = c.take<char>(weight_copy_bytes(vw));
  b.bytes = c.off;
  return b;
}

template <bool kWin>
int launch_head(const gsp_vocab_view* vw, HeadJob<kWin>& j, const State& s, const uint16_t* w, int64_t ldw, cudaStream_t st) {
  const bool bf = is_bf16(vw);
  int rc;
  if ((rc = make_map(&j.maps[0], bf, w, vw->D, vw->V, ldw, mm::kBM))) return rc;
  if ((rc = make_map(&j.maps[1], bf, s.h, s.Dp, s.Tp, s.Dp, j.bn))) return rc;
  if ((rc = ensure_smem(reinterpret_cast<const void*>(&mm::mma_kernel<HeadJob<kWin>>), mm::kSmem))) return rc;
  mm::mma_kernel<HeadJob<kWin>><<<num_sms(), mm::kThreads, mm::kSmem, st>>>(j);
  GSP_CHECK_LAUNCH();
  return GSP_OK;
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
  return launch_head<kWin>(vw, j, s, w, ldw, st);
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
int64_t loss_ws_bytes(const gsp_vocab_view* vw, bool backward);

}  // namespace vocab
}  // namespace gsp

using namespace gsp;
using namespace gsp::vocab;

extern "C" int64_t gsp_vocab_ws_bytes(const gsp_vocab_view* vw, int32_t kind, int32_t backward) {
  const int rc = check_view(vw, "gsp_vocab_ws_bytes");
  if (rc) return -rc;
  if (kind < GSP_VOCAB_CE || kind > GSP_VOCAB_HEAD) {
    set_error("gsp_vocab_ws_bytes: unknown kind %d", kind);
    return -GSP_ERR_ARG;
  }
  return kind == GSP_VOCAB_HEAD ? head_ws_bytes(vw, backward != 0) : loss_ws_bytes(vw, backward != 0);
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
  const int32_t bn = int32_t(vw->T >= mm::kBN ? mm::kBN : up(vw->T, 32));
  rc = win ? run_head<true>(vw, s, f, int32_t(L), bn, y, win, w, ldw, st)
           : run_head<false>(vw, s, f, int32_t(L), bn, y, win, w, ldw, st);
  if (rc) return rc;
  JoinParams p{};
  p.head = s.head;
  p.map = s.map;
  p.mask = mask;
  p.L = int32_t(L);
  p.bn = bn;
  p.ctas = num_sms();
  p.B = vw->T / L;
  p.V = vw->V;
  p.nvt = (vw->V + mm::kBM - 1) / mm::kBM;
  p.bias = vw->bias;
  p.part_m = f.part_m;
  p.part_i = f.part_i;
  p.y = y;
  p.win = win;
  head_join_kernel<<<unsigned(p.ctas + (mask ? p.B : 0)), mm::kBM, 0, st>>>(p);
  GSP_CHECK_LAUNCH();
  return GSP_OK;
}

extern "C" int gsp_sparse_head_backward(const gsp_vocab_view* vw, int64_t L, const float* y, const int32_t* win,
                                        const float* dy, void* d_hidden, void* d_weight, float* d_bias, void* state,
                                        int64_t state_bytes, void* ws, int64_t ws_bytes, void* stream) {
  int rc = check_texts(vw, L, "sparse_head backward");
  if (rc) return rc;
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
    if ((rc = grad_products(vw, s, w, ldw, pc, b.dh_acc, b.scale, d_hidden, d_weight, st))) return rc;
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
