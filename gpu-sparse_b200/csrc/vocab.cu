// Shared parts of the vocabulary head's operators: packing, operand maps, backward products.
#include "vocab.cuh"

#include <cudaTypedefs.h>

namespace gsp {
namespace vocab {

namespace {

PFN_cuTensorMapEncodeTiled_v12000 tma_encoder() {
  static PFN_cuTensorMapEncodeTiled_v12000 fn = [] {
    void* f = nullptr;
    cudaDriverEntryPointQueryResult q = cudaDriverEntryPointSymbolNotFound;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &q) != cudaSuccess ||
        q != cudaDriverEntryPointSuccess) {
      (void)cudaGetLastError();
      f = nullptr;
    }
    return reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(f);
  }();
  return fn;
}

__device__ __forceinline__ bool row_valid(const int64_t* targets, int64_t ignore, const uint8_t* flag, int64_t V, int64_t r) {
  if (targets) {
    const int64_t t = targets[r];
    return t >= 0 && t < V && t != ignore;
  }
  return flag ? flag[r] != 0 : true;
}

__global__ void __launch_bounds__(256) count_kernel(const int64_t* targets, int64_t ignore, const uint8_t* flag, int64_t V,
                                                    int64_t T, int32_t* counts) {
  mm::after_previous();
  const int64_t r = int64_t(blockIdx.x) * 256 + threadIdx.x;
  const int n = __syncthreads_count(r < T && row_valid(targets, ignore, flag, V, r));
  if (threadIdx.x == 0) counts[blockIdx.x] = n;
}

// copies `cols` 16-bit values and zeroes the rest of the row up to `pad` (a multiple of 8);
// one warp per row
__device__ __forceinline__ void copy_row(const uint16_t* src, uint16_t* dst, int64_t cols, int64_t pad, int lane) {
  if (((reinterpret_cast<uintptr_t>(src) | reinterpret_cast<uintptr_t>(dst)) & 15) == 0 && cols % 8 == 0) {
    const uint4* s = reinterpret_cast<const uint4*>(src);
    uint4* d = reinterpret_cast<uint4*>(dst);
    for (int64_t i = lane; i < cols / 8; i += 32) d[i] = __ldg(s + i);
    for (int64_t i = cols + lane; i < pad; i += 32) dst[i] = 0;
  } else {
#pragma unroll 8
    for (int64_t i = lane; i < pad; i += 32) dst[i] = i < cols ? src[i] : uint16_t(0);
  }
}

struct PackParams {
  const uint16_t* hidden;
  int64_t T, ldh, D, Dp, V, Vp;
  const int64_t* targets;
  int64_t ignore;
  const uint8_t* flag;
  const int32_t* counts;    // valid rows of every 256; null: count them here
  const float* bias;
  float bias_scale;         // 0: no bias2
  float* bias2;
  uint16_t* h;
  int32_t *map, *head, *tgt, *text;
  int32_t L;                // > 0: texts of L rows
  float* y;
  int32_t* win;
  const uint16_t* weight;   // to copy, or null
  int64_t ldw, Dw;
  uint16_t* w;
  int32_t per, pack_blocks, text_blocks;      // rows per block; blocks of each kind, W's copy last
};

// Blocks of p.per (at most 32) rows: their packed position is the number of valid rows before
// them.  Then a block per text that may be empty, and blocks of 8 rows of W's copy.
__global__ void __launch_bounds__(256) pack_kernel(const PackParams p) {
  __shared__ int32_t part[8];
  __shared__ uint32_t word;
  const int wid = threadIdx.x >> 5, lane = lane_id();
  mm::after_previous();
  if (int32_t(blockIdx.x) >= p.pack_blocks) {
    const int64_t b = int32_t(blockIdx.x) - p.pack_blocks;
    if (b < p.text_blocks) {
      bool any = false;
      for (int64_t t = threadIdx.x; t < p.L; t += 256) any |= p.flag[b * p.L + t] != 0;
      if (__syncthreads_or(any)) return;
      for (int64_t v = threadIdx.x; v < p.V; v += 256) {
        p.y[b * p.V + v] = 0.0f;
        if (p.win) p.win[b * p.V + v] = -1;
      }
    } else {
      const int64_t r = (b - p.text_blocks) * 8 + wid;
      if (r < p.V) copy_row(p.weight + r * p.ldw, p.w + r * p.Dw, p.D, p.Dw, lane);
    }
    return;
  }
  const int64_t r0 = int64_t(blockIdx.x) * p.per;
  if (p.bias_scale != 0.0f) {
    for (int64_t v = int64_t(blockIdx.x) * 256 + threadIdx.x; v < p.Vp; v += int64_t(p.pack_blocks) * 256)
      p.bias2[v] = v < p.V ? (p.bias ? p.bias[v] * p.bias_scale : 0.0f) : neg_inf();
  }
  if (r0 >= p.T) return;
  int32_t mine = 0;
  const int64_t b0 = r0 & ~int64_t(255);
  if (p.counts) {
    for (int64_t i = threadIdx.x; i < b0 / 256; i += 256) mine += p.counts[i];
    if (b0 + threadIdx.x < r0 && row_valid(p.targets, p.ignore, p.flag, p.V, b0 + threadIdx.x)) ++mine;
  } else {
    for (int64_t r = threadIdx.x; r < r0; r += 256) mine += row_valid(p.targets, p.ignore, p.flag, p.V, r);
  }
  mine = __reduce_add_sync(FULL, mine);
  if (lane == 0) part[wid] = mine;
  if (wid == 0) {
    const uint32_t w = __ballot_sync(FULL, lane < p.per && r0 + lane < p.T && row_valid(p.targets, p.ignore, p.flag, p.V, r0 + lane));
    if (lane == 0) word = w;
  }
  __syncthreads();
  int32_t base = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) base += part[i];
  const uint32_t w = word;
  for (int i = wid; i < p.per; i += 8) {
    if (!((w >> i) & 1)) continue;
    const int32_t d = base + __popc(w & ((1u << i) - 1));
    copy_row(p.hidden + (r0 + i) * p.ldh, p.h + int64_t(d) * p.Dp, p.D, p.Dp, lane);
    if (lane == 0) {
      p.map[d] = int32_t(r0 + i);
      if (p.targets) p.tgt[d] = int32_t(p.targets[r0 + i]);
    }
  }
  if (p.L > 0 && wid == 0) {
    const int64_t r = r0 + lane;
    if (lane < p.per && r < p.T && r % p.L == 0) p.text[r / p.L] = base + __popc(w & lanemask_lt());
  }
  if (r0 + p.per >= p.T && threadIdx.x == 0) {
    if (p.L > 0) p.text[p.T / p.L] = base + __popc(w);
    p.head[0] = base + __popc(w);
    p.head[1] = 0;
  }
}

// ---- backward products -------------------------------------------------------------------
// Both products' tiles form one list, first dH's (256 rows x 256 of D, k along the piece's
// vocabulary), then dW's (256 vocabulary rows x 256 of D, k along the rows).  Tile counts and
// depths differ by orders of magnitude with the sizes (32 rows: 3 dH tiles of 477 steps, 360 dW
// tiles of one), so the list is cut by steps and not by tiles: every pair of CTAs gets the same
// number of steps, and a tile cut by a border is finished from its fp32 fragments by
// finish_kernel, in list order.  Pairs are dealt to the 256-wide tiles of D in turn, so that the
// pairs that read the same rows of P run side by side.  Bound by the matrix pipe (74 % active) and
// L2, 10 TB/s: 1.33 PFLOP/s for 4096 rows, 1.31 for 16384 (V = 30522, D = 768).
constexpr int kOutBytes = 32 * 128;    // a warp's 32 rows x 64 columns of dW on their way out
constexpr int kFinishRows = 16;
// Steps an epilogue counts for in the cut: with 1, 3, 6 and 10 the products of one row take 39,
// 28, 29 and 36 us, of 1229 rows 102, 96, 102 and 110.
constexpr int kTileCost = 3;

struct GradList {
  int32_t nh, nw, nkh, nkw;       // tiles of each kind along this D tile, steps of each
  __device__ int64_t total() const { return int64_t(nh) * (nkh + kTileCost) + int64_t(nw) * (nkw + kTileCost); }
  // tile of position x, its first position, its steps
  __device__ void at(int64_t x, bool* is_h, int32_t* blk, int64_t* start, int32_t* nk) const {
    const int64_t lh = nkh + kTileCost, lw = nkw + kTileCost, h_end = nh * lh;
    if (x < h_end) {
      *is_h = true, *nk = nkh;
      *blk = int32_t(x / lh);
      *start = *blk * lh;
    } else {
      *is_h = false, *nk = nkw;
      *blk = int32_t((x - h_end) / lw);
      *start = h_end + *blk * lw;
    }
  }
};

struct GradJob {
  static constexpr int kStages = 6, kScratch = mm::kEpiWarps * kOutBytes;
  CUtensorMap maps[5];       // P K-major, P MN-major, W MN-major, H MN-major; dW as 32 x 64 boxes
  int32_t wait_limit, bf16;
  const int32_t* n_rows;
  Sparse sparse;             // see GradPiece
  const int32_t* map;
  int32_t D, nbs;            // 256-wide tiles of D
  int32_t v0, cols, V;
  int32_t first, last;
  int32_t low;               // first row of P's low parts, or 0
  bool want_h, want_w, w_cut;
  int64_t ld_out;            // of dh and dw
  float* dh_acc;
  int32_t ld_acc;
  float* frag;               // [pairs][2: begun elsewhere, ends elsewhere][2 CTAs][128][256]
  const float* scale;        // null: 1
  uint16_t *dh, *dw;

  __device__ int32_t rows() const {       // of P, low parts among them
    const int32_t n = *n_rows;
    return low && n > 0 ? low + n : n;
  }
  __device__ GradList list() const {
    const int32_t n = rows();
    if (sparse.gather(n, V)) return GradList{0, 0, 0, 0};
    return GradList{want_h ? (n + mm::kBM - 1) / mm::kBM : 0, want_w ? (cols + mm::kBM - 1) / mm::kBM : 0, (cols + 63) / 64,
                    (n + 63) / 64};
  }
  // shares per D tile: pairs past groups * nbs stay idle, and no share is empty
  __device__ int32_t groups(int32_t pairs, int64_t tot) const { return int32_t(min64(pairs / nbs, tot)); }
  __device__ float* fragment(int32_t pair, bool ends_elsewhere, int32_t rank) const {
    return frag + ((int64_t(pair) * 2 + ends_elsewhere) * 2 + rank) * mm::kRows * mm::kBN;
  }

  static constexpr int kIsH = 1, kFrag = 2, kEndsElsewhere = 4, kEnd = 8;
  struct Walk {
    GradList l;
    int64_t x, x1;
    int32_t nb, nb_step, nbs, D, v0;
    bool w_cut, low;
    __device__ bool next(mm::Tile& t) {
      for (;;) {
        if (x >= x1) {             // with more D tiles than pairs a pair takes several, whole
          nb += nb_step;
          if (nb >= nbs) return false;
          x = 0;
          continue;
        }
        bool is_h;
        int32_t blk, nk;
        int64_t start;
        l.at(x, &is_h, &blk, &start, &nk);
        const int64_t end = start + nk + kTileCost, y = x1 < end ? x1 : end;
        const int32_t k0 = int32_t(min64(x - start, nk)), k1 = int32_t(min64(y - start, nk));
        const bool whole_zero = nk == 0 && x == start;
        x = y;
        if (k0 >= k1 && !whole_zero) continue;      // only the tail of a tile's cost
        t.b0 = nb * mm::kBN;
        t.bn = D - t.b0 > 128 ? 256 : 128;
        t.a0 = blk * mm::kBM;
        t.ak = k0 * mm::kBK;
        t.a_rows = mm::kRows;
        t.b_mn = true;
        t.b_cut = is_h && w_cut;
        t.a = is_h ? 0 : 1;
        t.b = is_h ? 2 : 3;
        t.a_mn = !is_h;
        t.a_stream = true;
        t.bk = (is_h ? v0 : 0) + k0 * mm::kBK;
        t.nk = k1 - k0;
        t.x = blk;
        t.y = nb;
        t.flags = (is_h ? kIsH : 0) | (k0 > 0 || k1 < nk || (is_h && low) ? kFrag : 0) | (k1 < nk && k0 == 0 ? kEndsElsewhere : 0) |
                  (x >= x1 && nb + nb_step >= nbs ? kEnd : 0);
        return true;
      }
    }
  };
  __device__ Walk walk(int32_t pair, int32_t pairs) const {
    const GradList l = list();
    const int64_t tot = l.total();
    if (nbs > pairs) return Walk{l, tot > 0 ? 0 : 1, tot, pair, tot > 0 ? pairs : nbs, nbs, D, v0, w_cut, false};
    const int32_t groups = this->groups(pairs, tot), g = pair / nbs;
    if (g >= groups) return Walk{l, 0, 0, 0, nbs, nbs, D, v0, w_cut, false};
    return Walk{l, g * tot / groups, (g + 1) * tot / groups, pair % nbs, nbs, nbs, D, v0, w_cut, low > 0};
  }

  // 8 columns from c of a finished row: r a packed row (dH) or a vocabulary row of the piece (dW)
  __device__ void finish8(bool is_h, int32_t r, int32_t c, float (&v)[8]) const {
    uint16_t* out;
    const float sc = scale ? *scale : 1.0f;
    if (is_h) {
      float* acc = dh_acc + int64_t(r) * ld_acc + c;
      if (!first) {
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] += acc[k];
      }
      if (!last) {
#pragma unroll
        for (int k = 0; k < 8; ++k) acc[k] = v[k];
        return;
      }
      out = dh + int64_t(map ? map[r] : r) * ld_out + c;
    } else {
      out = dw + int64_t(v0 + r) * ld_out + c;
    }
    const bool bf = bf16 != 0;
    *reinterpret_cast<uint4*>(out) = make_uint4(pack2(v[0] * sc, v[1] * sc, bf), pack2(v[2] * sc, v[3] * sc, bf),
                                                pack2(v[4] * sc, v[5] * sc, bf), pack2(v[6] * sc, v[7] * sc, bf));
  }

  struct Epi {
    bool is_h, live;
    uint16_t* row;         // of dH
    float sc;
    __device__ void begin(const GradJob& j, const mm::Tile& t, const mm::Acc& a) {
      is_h = t.flags & kIsH;
      live = is_h ? a.row < j.rows() : a.row < j.cols;
      row = nullptr;
      if (live && is_h && !j.low) row = j.dh + int64_t(j.map ? j.map[a.row] : a.row) * j.ld_out;
      sc = j.scale ? *j.scale : 1.0f;
    }
    __device__ void tile(const GradJob& j, const mm::Tile& t, const mm::Acc& a) {
      const bool bf = j.bf16 != 0;
      float* acc = j.dh_acc + int64_t(a.row) * j.ld_acc;
      float* frag = j.fragment(int32_t(blockIdx.x) >> 1, (t.flags & kEndsElsewhere) != 0, a.rank) + a.lane_row * mm::kBN;
      unsigned char* out = a.scratch + a.warp * kOutBytes;
      for (int32_t c = a.c_lo; c < a.c_hi; c += 32) {
        float v[32];
        a.ld32(c, v);
        if (c + 32 == a.c_hi) a.release();
        uint32_t* u = reinterpret_cast<uint32_t*>(v);
        const int32_t d0 = t.b0 + c;
        if (t.flags & kFrag) {
          if (live && d0 < j.D) {
#pragma unroll
            for (int q = 0; q < 4; ++q) st256(frag + c + 8 * q, u + 8 * q);
          }
        } else if (is_h) {
          if (!live || d0 >= j.D) continue;
          if (!j.first) {
#pragma unroll
            for (int q = 0; q < 4; ++q) {
              uint32_t o[8];
              ld256(acc + d0 + 8 * q, o);
#pragma unroll
              for (int k = 0; k < 8; ++k) v[8 * q + k] += __uint_as_float(o[k]);
            }
          }
          if (!j.last) {
#pragma unroll
            for (int q = 0; q < 4; ++q) st256(acc + d0 + 8 * q, u + 8 * q);
            continue;
          }
#pragma unroll
          for (int k = 0; k < 32; ++k) v[k] *= sc;
          store_row16(row, d0, int32_t(j.ld_out), v, bf);
        } else {
          // half a 128-byte row at a time, 16-byte pieces swizzled as the map wants them; the
          // map cuts off what lies past dW's rows and columns
          if ((c & 32) == 0) {
            if (a.lane == 0) mm::tma_store_wait_read();
            __syncwarp();
          }
#pragma unroll
          for (int q = 0; q < 4; ++q)
            reinterpret_cast<uint4*>(out + a.lane * 128)[(((c & 32) >> 3) + q) ^ (a.lane & 7)] =
                make_uint4(pack2(v[8 * q] * sc, v[8 * q + 1] * sc, bf), pack2(v[8 * q + 2] * sc, v[8 * q + 3] * sc, bf),
                           pack2(v[8 * q + 4] * sc, v[8 * q + 5] * sc, bf), pack2(v[8 * q + 6] * sc, v[8 * q + 7] * sc, bf));
          if (c & 32) {
            mm::fence_async();
            __syncwarp();
            const int32_t x = d0 - 32, y = j.v0 + a.row;
            if (a.lane == 0 && x < j.D && y < j.V) mm::tma_store_2d(&j.maps[4], out, x, y);
          }
        }
      }
      if ((t.flags & kEnd) && a.lane == 0) mm::tma_store_wait();
    }
  };
  __device__ Epi epi() const { return Epi{}; }
};

// d_bias of a piece: the column sums of P that the logits' epilogue left for every 128 rows.  8
// warps share the row blocks of 32 columns; their sums are added in order.
__device__ void bias_grad(const BiasSums& b, int32_t n, int32_t cols, const float* scale, int64_t block) {
  __shared__ float got[8][32];
  const int wid = threadIdx.x >> 5, lane = lane_id();
  const int64_t c = block * 32 + lane;
  const int32_t blocks = (n + mm::kRows - 1) / mm::kRows;
  float s = 0.0f;
  if (c < cols) {
#pragma unroll 4
    for (int32_t i = wid; i < blocks; i += 8) s += b.part[int64_t(i) * b.pitch + c];
  }
  got[wid][lane] = s;
  __syncthreads();
  if (wid > 0 || c >= cols) return;
#pragma unroll
  for (int w = 1; w < 8; ++w) s += got[w][lane];
  b.out[c] = s * *scale;
}

// Finishes the tiles that a border between two shares cuts: the pair whose share holds a tile's
// last step adds the fragments in list order.  With low parts it finishes dH's tile even uncut,
// whose rows are then sums of two.  Block (pair, CTA of the pair, 16 rows): two rows per
// warp, 8 columns per lane.  The blocks past them finish d_bias.
__global__ void __launch_bounds__(256)
finish_kernel(const __grid_constant__ GradJob j, int32_t pairs, int32_t frag_blocks, const BiasSums b) {
  mm::after_previous();
  if (int32_t(blockIdx.x) >= frag_blocks) {
    bias_grad(b, *j.n_rows, j.cols, j.scale, int64_t(blockIdx.x) - frag_blocks);
    return;
  }
  const GradList l = j.list();
  const int64_t tot = l.total();
  const int32_t pair = blockIdx.x / (2 * mm::kRows / kFinishRows), sub = blockIdx.x % (2 * mm::kRows / kFinishRows);
  const int32_t groups = j.groups(pairs, tot);
  const int32_t g = pair / j.nbs, nb = pair % j.nbs;
  if (g >= groups) return;
  const int64_t x0 = g * tot / groups, x1 = (g + 1) * tot / groups;
  bool is_h;
  int32_t blk, nk;
  int64_t start;
  l.at(x0, &is_h, &blk, &start, &nk);
  const bool two = is_h && j.low > 0;
  // begins here and is finished, or ends elsewhere
  if ((x0 == start && !two) || x0 - start >= nk || x1 - start < nk) return;
  const int32_t first = int32_t(((start + 1) * groups - 1) / tot);   // the share that holds the tile's first step
  const int32_t rank = sub & 1, c = lane_id() * 8;
  if (nb * mm::kBN + c >= j.D) return;
#pragma unroll
  for (int i = 0; i < kFinishRows / 8; ++i) {
    const int32_t row = (sub >> 1) * kFinishRows + i * 8 + (threadIdx.x >> 5), r = blk * mm::kBM + rank * mm::kRows + row;
    if (r >= (is_h ? *j.n_rows : j.cols)) return;
    float v[8] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
    auto add = [&](int32_t s, int32_t in_tile) {
      uint32_t o[8];
      ld256(j.fragment(s * j.nbs + nb, s == first && s < g, in_tile / mm::kRows) + in_tile % mm::kRows * mm::kBN + c, o);
#pragma unroll
      for (int k = 0; k < 8; ++k) v[k] += __uint_as_float(o[k]);
    };
    const int32_t in_tile = rank * mm::kRows + row;
#pragma unroll 4
    for (int32_t s = first; s <= g; ++s) add(s, in_tile);
    if (two) {
#pragma unroll 4
      for (int32_t s = first; s <= g; ++s) add(s, in_tile + j.low);
    }
    j.finish8(is_h, r, nb * mm::kBN + c, v);
  }
}

}  // namespace

State carve_state(void* base, const gsp_vocab_view* vw, int64_t K, int64_t texts) {
  const int64_t T = vw->T, V = vw->V, D = vw->D;
  State s{};
  Carver c{static_cast<char*>(base)};
  s.Tp = pad_rows(T);
  s.Dp = up(D, 64);
  s.Vp = up(V, kRowPad);
  s.head = c.take<int32_t>(16);
  s.map = c.take<int32_t>(s.Tp);
  s.h = c.take<uint16_t>(s.Tp * s.Dp);
  if (texts > 0) {
    s.text = c.take<int32_t>(texts + 1);
  } else {
    s.bias2 = c.take<float>(s.Vp);
    s.lse2 = c.take<float>(s.Tp);
    s.tgt = c.take<int32_t>(K > 0 ? 0 : s.Tp);
  }
  if (K > 0) {
    s.K = K;
    s.hit = c.take<int4>(s.Tp * K);
    // 32 columns (an epilogue's step) per bucket, more where that would be more buckets than the
    // sort has counters for
    s.bucket_shift = 5;
    while ((s.Vp >> s.bucket_shift) > 8192) ++s.bucket_shift;
    s.buckets = (s.Vp + (int64_t(1) << s.bucket_shift) - 1) >> s.bucket_shift;
    s.off = c.take<int32_t>(s.Tp / 32 * (s.buckets + 1));
  }
  if (!weight_direct(vw)) s.w = c.take<uint16_t>(V * up(D, 8));
  s.bytes = c.off;
  return s;
}

int check_view(const gsp_vocab_view* vw, const char* what) {
  GSP_REQUIRE(vw, GSP_ERR_ARG, "%s: null view", what);
  GSP_REQUIRE(vw->dtype == GSP_W_BF16 || vw->dtype == GSP_W_F16, GSP_ERR_ARG, "%s: dtype must be bf16 or fp16", what);
  GSP_REQUIRE(vw->T >= 0 && vw->T <= (int64_t(1) << 30), GSP_ERR_ARG, "%s: %lld tokens out of range", what, (long long)vw->T);
  GSP_REQUIRE(vw->V >= 1 && vw->V <= (int64_t(1) << 30), GSP_ERR_ARG, "%s: %lld vocabulary rows out of range", what,
              (long long)vw->V);
  GSP_REQUIRE(vw->D >= 1 && vw->D <= (int64_t(1) << 20), GSP_ERR_ARG, "%s: width %lld out of range", what, (long long)vw->D);
  GSP_REQUIRE(up256(vw->T) / 256 * (up256(vw->V) / 256) < (int64_t(1) << 31), GSP_ERR_ARG,
              "%s: %lld tokens x %lld vocabulary rows are too many for one call", what, (long long)vw->T, (long long)vw->V);
  GSP_REQUIRE(vw->ld_hidden >= vw->D && vw->ld_weight >= vw->D, GSP_ERR_ARG, "%s: row stride smaller than the width", what);
  return GSP_OK;
}

int check_buffers(const void* state, int64_t state_bytes, int64_t state_need, const void* ws, int64_t ws_bytes,
                  int64_t ws_need, const char* what) {
  GSP_REQUIRE(state && state_bytes >= state_need && ws && ws_bytes >= ws_need, GSP_ERR_ARG, "%s: state or workspace too small",
              what);
  GSP_REQUIRE(((reinterpret_cast<uintptr_t>(state) | reinterpret_cast<uintptr_t>(ws)) & 255) == 0, GSP_ERR_ARG,
              "%s: state and workspace must start on 256-byte boundaries", what);
  return GSP_OK;
}

int make_map(CUtensorMap* m, bool bf16, const void* base, int64_t cols, int64_t rows, int64_t ld, int box_rows) {
  PFN_cuTensorMapEncodeTiled_v12000 enc = tma_encoder();
  GSP_REQUIRE(enc, GSP_ERR_CUDA, "vocabulary head: cuTensorMapEncodeTiled is not available");
  const cuuint64_t dims[2] = {cuuint64_t(cols), cuuint64_t(rows)};
  const cuuint64_t strides[1] = {cuuint64_t(ld) * 2};
  const cuuint32_t box[2] = {mm::kBK, cuuint32_t(box_rows)};
  const cuuint32_t es[2] = {1, 1};
  const CUresult r = enc(m, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2,
                         const_cast<void*>(base), dims, strides, box, es, CU_TENSOR_MAP_INTERLEAVE_NONE,
                         CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  GSP_REQUIRE(r == CUDA_SUCCESS, GSP_ERR_CUDA, "vocabulary head: tensor map failed (%d)", int(r));
  return GSP_OK;
}

int make_map_mn(CUtensorMap* m, bool bf16, const void* base, int64_t cols, int64_t rows, int64_t ld) {
  PFN_cuTensorMapEncodeTiled_v12000 enc = tma_encoder();
  GSP_REQUIRE(enc, GSP_ERR_CUDA, "vocabulary head: cuTensorMapEncodeTiled is not available");
  const cuuint64_t dims[3] = {64, cuuint64_t(rows), cuuint64_t(cols / 64)};
  const cuuint64_t strides[2] = {cuuint64_t(ld) * 2, 128};
  const cuuint32_t box[3] = {64, mm::kBK, 2};
  const cuuint32_t es[3] = {1, 1, 1};
  const CUresult r = enc(m, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3,
                         const_cast<void*>(base), dims, strides, box, es, CU_TENSOR_MAP_INTERLEAVE_NONE,
                         CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  GSP_REQUIRE(r == CUDA_SUCCESS, GSP_ERR_CUDA, "vocabulary head: tensor map failed (%d)", int(r));
  return GSP_OK;
}

int pack_rows(const gsp_vocab_view* vw, const int64_t* targets, int64_t ignore, const uint8_t* flag, float bias_scale,
              const Texts& texts, const State& s, int32_t* counts, cudaStream_t st) {
  const int64_t T = vw->T;
  int rc;
  // up to 2048 rows every CTA counts the rows before its own itself (at most 8 loads a
  // thread), which saves the launch of the counting pass
  const bool pre = T > 2048;
  if (pre) {
    rc = launch(count_kernel, dim3(unsigned((T + 255) / 256)), 256, 0, st, targets, ignore, flag, vw->V, T, counts);
    if (rc) return rc;
  }
  PackParams p{};
  p.hidden = static_cast<const uint16_t*>(vw->hidden);
  p.T = T;
  p.ldh = vw->ld_hidden;
  p.D = vw->D;
  p.Dp = s.Dp;
  p.V = vw->V;
  p.Vp = s.Vp;
  p.targets = targets;
  p.ignore = ignore;
  p.flag = flag;
  p.counts = pre ? counts : nullptr;
  p.bias = vw->bias;
  p.bias_scale = bias_scale;
  p.bias2 = s.bias2;
  p.h = s.h;
  p.map = s.map;
  p.head = s.head;
  p.tgt = s.tgt;
  p.text = s.text;
  p.L = int32_t(texts.L);
  p.y = texts.y;
  p.win = texts.win;
  p.weight = static_cast<const uint16_t*>(vw->weight);
  p.ldw = vw->ld_weight;
  p.Dw = up(vw->D, 8);
  p.w = s.w;
  p.per = T <= 4096 ? 8 : 32;      // few rows: more CTAs, a row per warp
  const int64_t blocks = (T + p.per - 1) / p.per;
  p.pack_blocks = int32_t(blocks < 32 ? 32 : blocks);
  p.text_blocks = int32_t(texts.L > 0 && flag ? T / texts.L : 0);
  const int64_t copy_blocks = s.w ? (vw->V + 7) / 8 : 0;
  return launch(pack_kernel, dim3(unsigned(p.pack_blocks + p.text_blocks + copy_blocks)), 256, 0, st, p);
}

int64_t piece_cols(int64_t Tp, int64_t V) {
  int64_t c = kPieceBytes / (2 * Tp) / kRowPad * kRowPad;
  if (c < kRowPad) c = kRowPad;
  const int64_t all = up(V, kRowPad);
  if (c >= all) return all;
  const int64_t pieces = (all + c - 1) / c;          // pieces of about equal size
  return up((all + pieces - 1) / pieces, kRowPad);
}

// Gradient rows are stored in whole 32-byte pieces; rows of any other width are made in a padded
// copy, which one more kernel unpacks.
int check_grads(const gsp_vocab_view* vw, const void* d_hidden, const void* d_weight, const char* what) {
  GSP_REQUIRE(vw->D % 16 != 0 || ((reinterpret_cast<uintptr_t>(d_hidden) | reinterpret_cast<uintptr_t>(d_weight)) & 31) == 0,
              GSP_ERR_ARG, "%s: d_hidden and d_weight must start on 32-byte boundaries", what);
  return GSP_OK;
}

GradScratch carve_grad(Carver& c, const gsp_vocab_view* vw, int64_t Tp, int64_t pitch) {
  GradScratch g{};
  const int64_t ld = up(vw->D, 16);
  g.dh_acc = c.take<float>(pitch < vw->V ? Tp * up(vw->D, 32) : 0);
  g.frag = c.take<float>(int64_t(mm::pair_ctas()) * 2 * mm::kRows * mm::kBN);
  g.dh = c.take<uint16_t>(vw->D % 16 ? Tp * ld : 0);
  g.dw = c.take<uint16_t>(vw->D % 16 ? vw->V * ld : 0);
  return g;
}

// rows of ld 16-bit values -> rows of D at out (map: where each row goes); a warp per row
__global__ void __launch_bounds__(256)
unpad_kernel(const uint16_t* dh, const int32_t* n_rows, const int32_t* map, uint16_t* out_h, int64_t h_blocks,
             const uint16_t* dw, int64_t V, uint16_t* out_w, int64_t ld, int64_t D, Sparse sparse) {
  mm::after_previous();
  if (sparse.gather(*n_rows, V)) return;
  const int lane = lane_id();
  const int64_t warp = int64_t(blockIdx.x) * 8 + (threadIdx.x >> 5);
  const uint16_t* src;
  uint16_t* dst;
  if (blockIdx.x < h_blocks) {
    if (warp >= *n_rows) return;
    src = dh + warp * ld;
    dst = out_h + int64_t(map[warp]) * D;
  } else {
    const int64_t r = warp - h_blocks * 8;
    if (r >= V) return;
    src = dw + r * ld;
    dst = out_w + r * D;
  }
#pragma unroll 8
  for (int64_t i = lane; i < D; i += 32) dst[i] = src[i];
}

int grad_products(const gsp_vocab_view* vw, const State& s, const uint16_t* w, int64_t ldw, const GradPiece& pc,
                  const GradScratch& g, const BiasSums& bias, const float* scale, void* d_hidden, void* d_weight,
                  cudaStream_t st) {
  GradJob j{};
  const bool bf = is_bf16(vw);
  int rc;
  const bool padded = vw->D % 16 != 0;
  uint16_t* dh = padded && d_hidden ? g.dh : static_cast<uint16_t*>(d_hidden);
  uint16_t* dw = padded && d_weight ? g.dw : static_cast<uint16_t*>(d_weight);
  j.ld_out = up(vw->D, 16);
  if (dw && (rc = make_map(&j.maps[4], bf, dw, j.ld_out, vw->V, j.ld_out, 32))) return rc;
  if ((rc = make_map(&j.maps[0], bf, pc.P, pc.pitch, s.Tp, pc.pitch, mm::kRows))) return rc;
  if ((rc = make_map_mn(&j.maps[1], bf, pc.P, pc.pitch, s.Tp, pc.pitch))) return rc;
  j.w_cut = vw->D % 64 != 0;
  if ((rc = j.w_cut ? make_map(&j.maps[2], bf, w, vw->D, vw->V, ldw, mm::kBK)
                    : make_map_mn(&j.maps[2], bf, w, vw->D, vw->V, ldw)))
    return rc;
  if ((rc = make_map_mn(&j.maps[3], bf, s.h, s.Dp, pc.low ? s.Tp : vw->T, s.Dp))) return rc;
  j.wait_limit = gsp_get_wait_limit();
  j.bf16 = bf;
  j.n_rows = s.head;
  j.sparse = pc.sparse;
  j.map = padded ? nullptr : s.map;
  j.D = int32_t(vw->D);
  j.nbs = int32_t((vw->D + mm::kBN - 1) / mm::kBN);
  j.v0 = int32_t(pc.v0);
  j.cols = int32_t(pc.cols);
  j.V = int32_t(vw->V);
  j.first = pc.first;
  j.low = pc.low;
  j.last = pc.last;
  j.want_h = d_hidden != nullptr;
  j.want_w = d_weight != nullptr;
  j.dh_acc = g.dh_acc;
  j.ld_acc = int32_t(up(vw->D, 32));
  j.frag = g.frag;
  j.scale = scale;
  j.dh = dh;
  j.dw = dw;
  if ((d_hidden || d_weight) && (rc = launch_mma(j, st))) return rc;
  const int32_t pairs = mm::pair_ctas() / 2;
  // with more D tiles than pairs no tile is cut
  const int32_t frag_blocks = (d_hidden || d_weight) && j.nbs <= pairs ? pairs * (2 * mm::kRows / kFinishRows) : 0;
  const int32_t blocks = frag_blocks + (bias.out ? int32_t((pc.cols + 31) / 32) : 0);
  if (blocks > 0) {
    if ((rc = launch(finish_kernel, dim3(unsigned(blocks)), 256, 0, st, j, pairs, frag_blocks, bias))) return rc;
  }
  if (padded && pc.last && (d_hidden || d_weight)) {
    const int64_t hb = d_hidden ? (vw->T + 7) / 8 : 0, wb = d_weight ? (vw->V + 7) / 8 : 0;
    rc = launch(unpad_kernel, dim3(unsigned(hb + wb)), 256, 0, st, dh, s.head, s.map, static_cast<uint16_t*>(d_hidden), hb, dw,
                vw->V, static_cast<uint16_t*>(d_weight), j.ld_out, vw->D, pc.sparse);
    if (rc) return rc;
  }
  return GSP_OK;
}

}  // namespace vocab
}  // namespace gsp

extern "C" int64_t gsp_vocab_state_bytes(const gsp_vocab_view* vw, int64_t K, int32_t kind) {
  const int rc = gsp::vocab::check_view(vw, "gsp_vocab_state_bytes");
  if (rc) return -rc;
  if (K < 0 || kind < GSP_VOCAB_CE || kind > GSP_VOCAB_HEAD) {
    gsp::set_error("gsp_vocab_state_bytes: bad arguments");
    return -GSP_ERR_ARG;
  }
  // the sparse head's texts: at most one per token
  return gsp::vocab::carve_state(nullptr, vw, kind == GSP_VOCAB_DISTILL ? K : 0,
                                 kind == GSP_VOCAB_HEAD ? (vw->T > 0 ? vw->T : 1) : 0).bytes;
}
