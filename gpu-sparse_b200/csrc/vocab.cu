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
  int32_t *map, *head, *tgt;
};

// 32 rows per CTA: their packed position is the number of valid rows before them.
__global__ void __launch_bounds__(256) pack_kernel(const PackParams p) {
  __shared__ int32_t part[8];
  __shared__ uint32_t word;
  const int64_t r0 = int64_t(blockIdx.x) * 32;
  const int wid = threadIdx.x >> 5, lane = lane_id();
  if (p.bias_scale != 0.0f) {
    for (int64_t v = int64_t(blockIdx.x) * 256 + threadIdx.x; v < p.Vp; v += int64_t(gridDim.x) * 256)
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
    const uint32_t w = __ballot_sync(FULL, r0 + lane < p.T && row_valid(p.targets, p.ignore, p.flag, p.V, r0 + lane));
    if (lane == 0) word = w;
  }
  __syncthreads();
  int32_t base = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) base += part[i];
  const uint32_t w = word;
  for (int i = wid; i < 32; i += 8) {
    if (!((w >> i) & 1)) continue;
    const int32_t d = base + __popc(w & ((1u << i) - 1));
    copy_row(p.hidden + (r0 + i) * p.ldh, p.h + int64_t(d) * p.Dp, p.D, p.Dp, lane);
    if (lane == 0) {
      p.map[d] = int32_t(r0 + i);
      if (p.targets) p.tgt[d] = int32_t(p.targets[r0 + i]);
    }
  }
  if (r0 + 32 >= p.T && threadIdx.x == 0) {
    p.head[0] = base + __popc(w);
    p.head[1] = 0;
  }
}

__global__ void __launch_bounds__(256) copy_weight_kernel(const uint16_t* w, int64_t ldw, int64_t V, int64_t D, int64_t Dp,
                                                          uint16_t* out) {
  const int64_t r = int64_t(blockIdx.x) * 8 + (threadIdx.x >> 5);
  if (r < V) copy_row(w + r * ldw, out + r * Dp, D, Dp, lane_id());
}

// ---- backward products -------------------------------------------------------------------
struct GradJob {
  CUtensorMap maps[4];       // P K-major, P MN-major, W MN-major, H MN-major
  int32_t wait_limit, bf16;
  const int32_t* n_rows;
  const int32_t* map;
  int32_t D, nbs;            // 256-wide tiles of D
  int32_t v0, cols, V;
  int32_t first, last;
  bool want_h, want_w, vec_h, vec_w;
  float* dh_acc;
  int32_t ld_acc;
  const float* scale;        // null: 1
  uint16_t *dh, *dw;

  struct Walk {
    int32_t nh, nw, rows, cols, v0, nbs, D;
    bool h_first;
    __device__ bool get(int32_t i, mm::Tile& t) const {
      int64_t x = int64_t(i) * gridDim.x + blockIdx.x;
      if (x >= nh + nw) return false;
      // tiles with the longer sums first, so that the last ones to start are short
      bool is_h = h_first ? x < nh : x >= nw;
      if (h_first ? !is_h : is_h) x -= h_first ? nh : nw;
      const int32_t blk = int32_t(x / nbs), nb = int32_t(x - int64_t(blk) * nbs);
      t.b0 = nb * mm::kBN;
      t.bn = min(mm::kBN, (D - t.b0 + 63) / 64 * 64);
      t.a0 = blk * mm::kBM;
      t.ak = 0;
      t.b_mn = true;
      if (is_h) {
        t.a = 0, t.b = 2, t.a_mn = false, t.bk = v0, t.nk = (cols + 63) / 64;
      } else {
        t.a = 1, t.b = 3, t.a_mn = true, t.bk = 0, t.nk = (rows + 63) / 64;
      }
      t.x = blk;
      t.y = nb;
      t.flags = is_h;
      return true;
    }
  };
  __device__ Walk walk() const {
    const int32_t n = *n_rows;
    const int32_t nh = want_h ? (n + mm::kBM - 1) / mm::kBM * nbs : 0;
    const int32_t nw = want_w ? (cols + mm::kBM - 1) / mm::kBM * nbs : 0;
    return Walk{nh, nw, n, cols, v0, nbs, D, cols >= n};
  }

  struct Epi {
    __device__ void tile(const GradJob& j, const mm::Tile& t, const mm::Acc& a) {
      const int32_t r = t.a0 + a.warp * 32 + a.lane;
      const float sc = j.scale ? *j.scale : 1.0f;
      const bool bf = j.bf16 != 0;
      if (t.flags) {
        const bool live = r < *j.n_rows;
        uint16_t* row = live && j.last ? j.dh + int64_t(j.map[r]) * j.D : nullptr;
        float* acc = j.dh_acc + int64_t(r) * j.ld_acc;
        for (int32_t c = 0; c < t.bn; c += 32) {
          float v[32];
          a.ld32(c, v);
          if (!live || t.b0 + c >= j.ld_acc) continue;
          uint32_t* u = reinterpret_cast<uint32_t*>(v);
          if (!j.first) {
#pragma unroll
            for (int q = 0; q < 4; ++q) {
              uint32_t o[8];
              ld256(acc + t.b0 + c + 8 * q, o);
#pragma unroll
              for (int k = 0; k < 8; ++k) v[8 * q + k] += __uint_as_float(o[k]);
            }
          }
          if (j.last) {
#pragma unroll
            for (int k = 0; k < 32; ++k) v[k] *= sc;
            store_row16(row, t.b0 + c, j.D, v, bf, j.vec_h);
          } else {
#pragma unroll
            for (int q = 0; q < 4; ++q) st256(acc + t.b0 + c + 8 * q, u + 8 * q);
          }
        }
      } else {
        const int32_t v_row = j.v0 + r;
        const bool live = r < j.cols && v_row < j.V;
        uint16_t* row = j.dw + int64_t(v_row) * j.D;
        for (int32_t c = 0; c < t.bn; c += 32) {
          float v[32];
          a.ld32(c, v);
          if (!live) continue;
#pragma unroll
          for (int k = 0; k < 32; ++k) v[k] *= sc;
          store_row16(row, t.b0 + c, j.D, v, bf, j.vec_w);
        }
      }
    }
  };
  __device__ Epi epi() const { return Epi{}; }
};

}  // namespace

State carve_state(void* base, int64_t T, int64_t V, int64_t D, int64_t K, bool loss) {
  State s{};
  Carver c{static_cast<char*>(base)};
  s.Tp = pad_rows(T);
  s.Dp = up(D, 8);
  s.Vp = up(V, kRowPad);
  s.head = c.take<int32_t>(16);
  s.map = c.take<int32_t>(s.Tp);
  s.h = c.take<uint16_t>(s.Tp * s.Dp);
  if (loss) {
    s.bias2 = c.take<float>(s.Vp);
    s.lse2 = c.take<float>(s.Tp);
    s.tgt = c.take<int32_t>(K > 0 ? 0 : s.Tp);
  }
  if (K > 0) {
    s.cnt = c.take<int32_t>(T);
    s.ent = c.take<float>(T);
    s.ids = c.take<int32_t>(T * K);
    s.p = c.take<float>(T * K);
    s.flag = c.take<uint8_t>(T);
  }
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
  GSP_REQUIRE(vw->ld_hidden >= vw->D && vw->ld_weight >= vw->D, GSP_ERR_ARG, "%s: row stride smaller than the width", what);
  return GSP_OK;
}

int64_t weight_copy_bytes(const gsp_vocab_view* vw) {
  const bool direct = vw->ld_weight % 8 == 0 && (reinterpret_cast<uintptr_t>(vw->weight) & 15) == 0 && vw->ld_weight < (int64_t(1) << 38);
  return direct ? 0 : up256(vw->V * up(vw->D, 8) * 2);
}

int weight_rows(const gsp_vocab_view* vw, void* scratch, const uint16_t** w, int64_t* ld, cudaStream_t st) {
  if (weight_copy_bytes(vw) == 0) {
    *w = static_cast<const uint16_t*>(vw->weight);
    *ld = vw->ld_weight;
    return GSP_OK;
  }
  const int64_t Dp = up(vw->D, 8);
  copy_weight_kernel<<<unsigned((vw->V + 7) / 8), 256, 0, st>>>(static_cast<const uint16_t*>(vw->weight), vw->ld_weight, vw->V,
                                                              vw->D, Dp, static_cast<uint16_t*>(scratch));
  GSP_CHECK_LAUNCH();
  *w = static_cast<const uint16_t*>(scratch);
  *ld = Dp;
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

int pack_rows(const gsp_vocab_view* vw, const int64_t* targets, int64_t ignore, const uint8_t* flag, float bias_scale,
              const State& s, int32_t* counts, cudaStream_t st) {
  const int64_t T = vw->T;
  // up to 2048 rows every CTA counts the rows before its own itself (at most 8 loads a
  // thread), which saves the launch of the counting pass
  const bool pre = T > 2048;
  if (pre) {
    count_kernel<<<unsigned((T + 255) / 256), 256, 0, st>>>(targets, ignore, flag, vw->V, T, counts);
    GSP_CHECK_LAUNCH();
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
  const int64_t blocks = (T + 31) / 32;
  pack_kernel<<<unsigned(blocks < 32 ? 32 : blocks), 256, 0, st>>>(p);
  GSP_CHECK_LAUNCH();
  return GSP_OK;
}

int64_t piece_cols(int64_t Tp, int64_t V) {
  int64_t c = kPieceBytes / (2 * Tp) / kRowPad * kRowPad;
  if (c < kRowPad) c = kRowPad;
  const int64_t all = up(V, kRowPad);
  if (c >= all) return all;
  const int64_t pieces = (all + c - 1) / c;          // pieces of about equal size
  return up((all + pieces - 1) / pieces, kRowPad);
}

int grad_products(const gsp_vocab_view* vw, const State& s, const uint16_t* w, int64_t ldw, const GradPiece& pc,
                  float* dh_acc, const float* scale, void* d_hidden, void* d_weight, cudaStream_t st) {
  if (!d_hidden && !d_weight) return GSP_OK;
  GradJob j{};
  const bool bf = is_bf16(vw);
  int rc;
  if ((rc = make_map(&j.maps[0], bf, pc.P, pc.pitch, s.Tp, pc.pitch, mm::kBM))) return rc;
  if ((rc = make_map(&j.maps[1], bf, pc.P, pc.pitch, s.Tp, pc.pitch, mm::kBK))) return rc;
  if ((rc = make_map(&j.maps[2], bf, w, vw->D, vw->V, ldw, mm::kBK))) return rc;
  if ((rc = make_map(&j.maps[3], bf, s.h, s.Dp, s.Tp, s.Dp, mm::kBK))) return rc;
  j.wait_limit = gsp_get_wait_limit();
  j.bf16 = bf;
  j.n_rows = s.head;
  j.map = s.map;
  j.D = int32_t(vw->D);
  j.nbs = int32_t((vw->D + mm::kBN - 1) / mm::kBN);
  j.v0 = int32_t(pc.v0);
  j.cols = int32_t(pc.cols);
  j.V = int32_t(vw->V);
  j.first = pc.first;
  j.last = pc.last;
  j.want_h = d_hidden != nullptr;
  j.want_w = d_weight != nullptr;
  j.vec_h = vw->D % 16 == 0 && (reinterpret_cast<uintptr_t>(d_hidden) & 31) == 0;
  j.vec_w = vw->D % 16 == 0 && (reinterpret_cast<uintptr_t>(d_weight) & 31) == 0;
  j.dh_acc = dh_acc;
  j.ld_acc = int32_t(up(vw->D, 32));
  j.scale = scale;
  j.dh = static_cast<uint16_t*>(d_hidden);
  j.dw = static_cast<uint16_t*>(d_weight);
  if ((rc = ensure_smem(reinterpret_cast<const void*>(&mm::mma_kernel<GradJob>), mm::kSmem))) return rc;
  mm::mma_kernel<GradJob><<<num_sms(), mm::kThreads, mm::kSmem, st>>>(j);
  GSP_CHECK_LAUNCH();
  return GSP_OK;
}

}  // namespace vocab
}  // namespace gsp

extern "C" int64_t gsp_vocab_state_bytes(int64_t T, int64_t V, int64_t D, int64_t K, int32_t kind) {
  if (T < 0 || V < 1 || D < 1 || K < 0 || kind < GSP_VOCAB_CE || kind > GSP_VOCAB_HEAD) {
    gsp::set_error("gsp_vocab_state_bytes: bad arguments");
    return -GSP_ERR_ARG;
  }
  return gsp::vocab::carve_state(nullptr, T, V, D, kind == GSP_VOCAB_DISTILL ? K : 0, kind != GSP_VOCAB_HEAD).bytes;
}
