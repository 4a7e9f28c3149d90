// Shared parts of the vocabulary head's operators (vocab_loss.cu, sparse_head.cu): tokens
// packed to the valid ones, operand maps, and the two products every backward pass ends in.
//
// Notation: H [T, D] hidden states, W [V, D] vocabulary projection (both bf16 or both fp16),
// s = H W^T + bias the logits, of which no more than a tile ever exists.
#pragma once
#include "mma.cuh"

namespace gsp {
namespace vocab {

constexpr int kRowPad = 256;     // packed rows and vocabulary columns are allocated in these
inline int64_t up(int64_t x, int64_t m) { return (x + m - 1) / m * m; }
inline int64_t up256(int64_t x) { return up(x, 256); }
inline int64_t pad_rows(int64_t T) { return T > 0 ? up(T, kRowPad) : kRowPad; }

// Carves a caller's buffer; with a null base it only counts.
struct Carver {
  char* base;
  int64_t off = 0;
  template <typename T>
  T* take(int64_t n) {
    T* p = base ? reinterpret_cast<T*>(base + off) : nullptr;
    off = up256(off + n * int64_t(sizeof(T)));
    return p;
  }
};

// What the forward pass leaves for the backward pass, in a buffer of the caller's.
struct State {
  int32_t* head;      // [0] packed rows, [1] ticket of the reducing kernels
  int32_t* map;       // [Tp] original row of every packed row, ascending
  uint16_t* h;        // [Tp, Dp] packed hidden states
  int32_t* text;      // [texts + 1] first packed row of every text (sparse head)
  float* bias2;       // [Vp] bias in units of the exponent's base 2, -inf past V (losses)
  float* lse2;        // [Tp] log2 of the softmax's denominator (losses)
  int32_t* tgt;       // [Tp] target of every packed row (cross entropy)
  int4* hit;          // a teacher's entries of every 32 packed rows by vocabulary bucket: (id, row
                      // of the 32, probability's bits, entry of the row), 32 K a group
  int32_t* off;       // [Tp / 32, buckets + 1] first hit of every bucket
  uint16_t* w;        // [V, up(D, 8)] copy of a projection whose rows a TMA map cannot describe
  int64_t Tp, Dp, Vp, K, buckets, bytes;
  int32_t bucket_shift;      // log2 of a bucket's vocabulary rows
};
constexpr int32_t kNoId = 0x7FFFFFFF;
// loss: texts is 0; sparse head: K is 0
State carve_state(void* base, const gsp_vocab_view* vw, int64_t K, int64_t texts);

int check_view(const gsp_vocab_view* vw, const char* what);
// state and workspace: large enough and on 256-byte boundaries, which all parts of them rely on
int check_buffers(const void* state, int64_t state_bytes, int64_t state_need, const void* ws, int64_t ws_bytes,
                  int64_t ws_need, const char* what);
int check_grads(const gsp_vocab_view* vw, const void* d_hidden, const void* d_weight, const char* what);
inline bool is_bf16(const gsp_vocab_view* vw) { return vw->dtype == GSP_W_BF16; }
// whether a TMA map can describe W's rows as they are (else the forward call copies them)
inline bool weight_direct(const gsp_vocab_view* vw) {
  return vw->ld_weight % 8 == 0 && (reinterpret_cast<uintptr_t>(vw->weight) & 15) == 0 && vw->ld_weight < (int64_t(1) << 38);
}
// W as a TMA map can describe it
struct Weight {
  const uint16_t* w;
  int64_t ld;
};
inline Weight weight_rows(const gsp_vocab_view* vw, const State& s) {
  if (s.w) return Weight{s.w, up(vw->D, 8)};
  return Weight{static_cast<const uint16_t*>(vw->weight), vw->ld_weight};
}

// 2D map of a row-major 16-bit matrix: boxes of 64 columns x box_rows rows, 128-byte swizzle,
// zeros outside
int make_map(CUtensorMap* m, bool bf16, const void* base, int64_t cols, int64_t rows, int64_t ld, int box_rows);
// The same matrix (cols a multiple of 64) as [cols / 64][rows][64] for an MN-major operand: boxes
// of 2 x 64 x 64
int make_map_mn(CUtensorMap* m, bool bf16, const void* base, int64_t cols, int64_t rows, int64_t ld);

// Packs the rows that take part (targets: id in [0, V) and != ignore; else flag != 0) to the
// front of st.h, keeping their order, and writes st.map, st.head[0] and st.w; bias2 when
// bias_scale != 0.  Texts (texts.L > 0): st.text, and zero rows of y (and -1 in win) for those
// without tokens.
struct Texts {
  int64_t L;
  float* y;
  int32_t* win;
};
int pack_rows(const gsp_vocab_view* vw, const int64_t* targets, int64_t ignore, const uint8_t* flag, float bias_scale,
              const Texts& texts, const State& s, int32_t* counts, cudaStream_t st);
inline int64_t pack_counts(int64_t T) { return (T + 255) / 256 + 1; }

// How sparse the gradient of the logits is: with so few of n x V entries nonzero that gathering
// rows for them costs less than the products (and with room for a list of them), they are
// gathered.  Both sides at V = 30522, D = 768, in us: 32 texts of 256 tokens, one entry in 671 of
// n x V: 237 gathered, 729 as products; one in 256: 385 and 729; 500 texts of 32, one in 5500: 369
// and 1443; one in 61: 3493 and 1547.  They cross near one entry in 150.
constexpr int64_t kGatherWeight = 160;
struct Sparse {
  const int64_t* nnz;      // entries, or null: always the products
  int64_t room;
  __device__ __forceinline__ bool gather(int64_t n, int64_t V) const {
    return nnz && *nnz <= room && *nnz * kGatherWeight <= n * V;
  }
};

// Backward products over a piece of the vocabulary [v0, v0 + cols): P [Tp, pitch] is the
// gradient of the piece's logits,
//   dH (+)= P W[v0 : v0 + cols],   dW[v0 : v0 + cols] = P^T H   (each where asked for),
// in one launch, and a second that finishes them.  Between pieces dH is carried in fp32.
struct GradPiece {
  const uint16_t* P;
  int64_t pitch, v0, cols;
  bool first, last;
  Sparse sparse;           // few enough entries in P and the call does nothing
  int32_t low;             // see low_rows
};
struct GradScratch {
  float* dh_acc;      // [Tp, up(D, 32)], or null when there is one piece
  float* frag;        // partial tiles
  uint16_t *dh, *dw;  // gradient rows padded to 16 columns, when D is not a multiple of 16
};
GradScratch carve_grad(Carver& c, const gsp_vocab_view* vw, int64_t Tp, int64_t pitch);
// Up to 128 rows fill half a tile of P; the other half, from this row on, then holds what rounding
// P to 16 bits left over (the packed rows stand there a second time), and the products add both:
// with few rows few entries of P decide a gradient, and their roundings would not average out.
// Distilling 32 rows of 10 entries, d_weight is off by 0.0017 of its norm (its own rounding) instead
// of 0.0025; the backward pass of 32 rows takes 2 us more in the logits and 4 in the finish.
// 0: more rows, P rounded once.  (More tiles along D than pairs finish no tile from fragments.)
inline int32_t low_rows(const gsp_vocab_view* vw) {
  const bool few = vw->T <= mm::kRows && (vw->D + mm::kBN - 1) / mm::kBN <= mm::pair_ctas() / 2;
  return few ? int32_t((vw->T + 63) / 64 * 64) : 0;
}
// column sums of the piece's unrounded P for every 128 rows [row blocks][pitch], and where
// their total goes (null: nowhere)
struct BiasSums {
  const float* part;
  int64_t pitch;
  float* out;
};
int grad_products(const gsp_vocab_view* vw, const State& s, const uint16_t* w, int64_t ldw, const GradPiece& pc,
                  const GradScratch& g, const BiasSums& bias, const float* scale, void* d_hidden, void* d_weight,
                  cudaStream_t st);
// Columns of one piece: P takes at most kPieceBytes (or 256 columns).  A training step on 16384
// rows takes 3.33 ms with pieces of 64 MiB, which stay in L2 but make short tile lists and carry
// dH more often, 3.04 with 128, 2.86 with 256, 2.80 with 512 and 2.92 with 1024; on 8192 rows
// 1.58, 1.44, 1.38, 1.40 and 1.40.
constexpr int64_t kPieceBytes = int64_t(512) << 20;
int64_t piece_cols(int64_t Tp, int64_t V);
// Zeroes the packed rows past the n taking part that the products' last 64-deep step reads:
// their P is 0, and 0 times whatever was there must be 0.  All threads of one CTA.
__device__ __forceinline__ void zero_tail_rows(uint16_t* h, int64_t Dp, int32_t n) {
  const int64_t end = (int64_t(n) + 63) / 64 * 64;
  uint4* p = reinterpret_cast<uint4*>(h + int64_t(n) * Dp);
  for (int64_t i = threadIdx.x; i < (end - n) * Dp / 8; i += blockDim.x) p[i] = make_uint4(0, 0, 0, 0);
}
// Zeroes this block's share of d_hidden's rows: the products write only those that took part.
__device__ __forceinline__ void zero_share(void* d, int64_t bytes, int64_t block, int64_t blocks) {
  const int64_t head = min64((16 - int64_t(reinterpret_cast<uintptr_t>(d) & 15)) & 15, bytes), n = (bytes - head) / 16;
  char* c = static_cast<char*>(d);
  if (block == 0) {
    for (int64_t i = threadIdx.x; i < head; i += blockDim.x) c[i] = 0;
    for (int64_t i = head + n * 16 + threadIdx.x; i < bytes; i += blockDim.x) c[i] = 0;
  }
  uint4* p = reinterpret_cast<uint4*>(c + head);
  for (int64_t i = block * blockDim.x + threadIdx.x; i < n; i += blocks * blockDim.x) p[i] = make_uint4(0, 0, 0, 0);
}

// ---- launches ----------------------------------------------------------------------------
// Every kernel of a call is launched so that it may start while the one before it in the stream
// still runs, and begins with after_previous(), which returns once that one has finished and its
// writes are visible: what is hidden is the launch itself and, in the products, the set-up of
// barriers and tensor memory.
template <class... P, class... A>
int launch(void (*kernel)(P...), dim3 grid, int threads, size_t smem, cudaStream_t st, A... args) {
  cudaLaunchConfig_t c{};
  c.gridDim = grid;
  c.blockDim = dim3(unsigned(threads));
  c.dynamicSmemBytes = smem;
  c.stream = st;
  cudaLaunchAttribute at{};
  at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at.val.programmaticStreamSerializationAllowed = 1;
  c.attrs = &at;
  c.numAttrs = 1;
  GSP_CUDA(cudaLaunchKernelEx(&c, kernel, P(args)...));
  return GSP_OK;
}
template <class Job>
int launch_mma(const Job& job, cudaStream_t st) {
  const int rc = ensure_smem(reinterpret_cast<const void*>(&mm::mma_kernel<Job>), mm::smem_bytes<Job>());
  if (rc) return rc;
  return launch(mm::mma_kernel<Job>, dim3(unsigned(mm::pair_ctas())), mm::kThreads, size_t(mm::smem_bytes<Job>()), st, job);
}

// ---- device helpers ----------------------------------------------------------------------
// (relative error up to 2^-22; results below 2^-126 are 0)
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float neg_inf() { return __uint_as_float(0xFF800000u); }
// two floats rounded to nearest even into one 32-bit word, `lo` in the low half
__device__ __forceinline__ uint32_t pack2(float lo, float hi, bool bf16) {
  uint32_t r;
  if (bf16) {
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  } else {
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  }
  return r;
}
__device__ __forceinline__ float2 unpack2(uint32_t x, bool bf16) {
  if (bf16) return make_float2(__uint_as_float(x << 16), __uint_as_float(x & 0xFFFF0000u));
  float2 r;
  asm("{ .reg .b16 a, b; mov.b32 {a, b}, %2; cvt.f32.f16 %0, a; cvt.f32.f16 %1, b; }" : "=f"(r.x), "=f"(r.y) : "r"(x));
  return r;
}
// 32 of them (one branch on the type)
__device__ __forceinline__ void pack32(const float (&v)[32], uint32_t (&w)[16], bool bf16) {
  if (bf16) {
#pragma unroll
    for (int k = 0; k < 16; ++k) w[k] = pack2(v[2 * k], v[2 * k + 1], true);
  } else {
#pragma unroll
    for (int k = 0; k < 16; ++k) w[k] = pack2(v[2 * k], v[2 * k + 1], false);
  }
}
// v = what pack32 (w) lost of it; 0 where that is not finite
__device__ __forceinline__ void unpack_rest(float (&v)[32], const uint32_t (&w)[16], bool bf16) {
#pragma unroll
  for (int k = 0; k < 16; ++k) {
    const float2 f = unpack2(w[k], bf16);
    v[2 * k] -= f.x;
    v[2 * k + 1] -= f.y;
  }
#pragma unroll
  for (int k = 0; k < 32; ++k) v[k] = fabsf(v[k]) < __uint_as_float(0x7F800000u) ? v[k] : 0.0f;
}
// 32-byte accesses of global memory (sm_100a), p a multiple of 32 bytes
__device__ __forceinline__ void st256(void* p, const uint32_t* r) {
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(r[0]), "r"(r[1]), "r"(r[2]),
               "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
               : "memory");
}
__device__ __forceinline__ void ld256(const void* p, uint32_t* r) {
  asm volatile("ld.global.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
               : "l"(p)
               : "memory");
}
// 32 accumulators of one row -> 16-bit, columns c0 .. min(c0 + 32, ld); the row starts on a
// 32-byte boundary and ld is a multiple of 16
__device__ __forceinline__ void store_row16(uint16_t* row, int32_t c0, int32_t ld, const float (&v)[32], bool bf16) {
  uint32_t w[16];
  pack32(v, w, bf16);
  st256(row + c0, w);
  if (c0 + 16 < ld) st256(row + c0 + 16, w + 8);
}
// two fp32 operations per instruction (sm_100a)
struct F2 {
  uint64_t v;
};
__device__ __forceinline__ F2 f2(float a, float b) {
  F2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r.v) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void split(F2 x, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(x.v)); }
__device__ __forceinline__ F2 fma2(F2 a, F2 b, F2 c) {
  F2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
  return r;
}
__device__ __forceinline__ F2 add2(F2 a, F2 b) {
  F2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ F2 mul2(F2 a, F2 b) {
  F2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
// A warp's 32 x 32 block (lane = row) through shared memory (32 rows of kBlockLd floats, which
// keeps 16-byte accesses free of bank conflicts).
constexpr int kBlockLd = 36;
constexpr int kBlockBytes = 32 * kBlockLd * 4;
__device__ __forceinline__ void block_put(float* block, const float (&v)[32], int lane) {
  float4* o = reinterpret_cast<float4*>(block + lane * kBlockLd);
#pragma unroll
  for (int q = 0; q < 8; ++q) o[q] = make_float4(v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3]);
}
// Column sums of the block in two steps, so that other work can stand between the loads and the
// sums: lane l loads columns 4 (l % 8) .. + 3 of the rows l / 8 + 4 i; lanes 0-15 receive the sums
// over those rows and the rows of lane l + 16 (two partial sums per column).
struct ColLoads {
  float4 x[8];
};
__device__ __forceinline__ void block_load(ColLoads& c, const float* block, int lane) {
  const float* p = block + (lane >> 3) * kBlockLd + (lane & 7) * 4;
#pragma unroll
  for (int i = 0; i < 8; ++i) c.x[i] = *reinterpret_cast<const float4*>(p + 4 * i * kBlockLd);
}
__device__ __forceinline__ float4 block_sums(const ColLoads& c) {
  F2 a = f2(0.0f, 0.0f), b = a;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    a = add2(a, f2(c.x[i].x, c.x[i].y));
    b = add2(b, f2(c.x[i].z, c.x[i].w));
  }
  float4 s;
  split(a, s.x, s.y);
  split(b, s.z, s.w);
  s.x += __shfl_xor_sync(FULL, s.x, 16);
  s.y += __shfl_xor_sync(FULL, s.y, 16);
  s.z += __shfl_xor_sync(FULL, s.z, 16);
  s.w += __shfl_xor_sync(FULL, s.w, 16);
  return s;
}

// A list of `tot` tiles in equal consecutive shares: share c is [share_lo(c), share_lo(c + 1)),
// tile x lies in share share_of(x).  No share is empty unless all later ones are.
__host__ __device__ __forceinline__ int32_t share_lo(int32_t tot, int32_t shares, int32_t c) {
  return tot <= shares ? (c < tot ? c : tot) : int32_t(uint64_t(c) * uint32_t(tot) / uint32_t(shares));
}
__host__ __device__ __forceinline__ int32_t share_of(int32_t tot, int32_t shares, int32_t x) {
  return tot <= shares ? x : int32_t(((uint64_t(x) + 1) * uint32_t(shares) - 1) / uint32_t(tot));
}

}  // namespace vocab
}  // namespace gsp
