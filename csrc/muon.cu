// Orthogonalising an update by Newton-Schulz products, and the Muon step
// around it (Jordan et al. 2024):
//
//   X <- U / (|U|_F + eps)
//   repeat:  A = X X^T,  B = b A + c A A,  X <- a X + B X        (rows <= cols;
//            A = X^T X and X B otherwise: the Gram matrix of the shorter side)
//
// and, in the step form, m <- mu m + g, U = g + mu m (or m), W <- W (1 - lr wd)
// - lr k X, all over a batch of equally shaped matrices.
//
// Numerics.  The operands of the products are fp16 at 2^12 times their value
// (|X|, |A|, |B| stay below 3, so nothing overflows, and an entry of a
// 4096-wide X is far above the subnormals); accumulators are fp32.  X itself is
// carried as a pair of fp16, high and low (22 bits), and the a X term adds
// both: rounding X would put noise under every small singular value, which
// five steps multiply by up to 480, while a product's rounding is confined to
// the directions of the large ones.  One product of high parts per matrix then
// leaves X within about 1e-3 of exact (bf16 operands, the usual choice:
// 3e-2 to 1e-1 on gradients of decaying spectrum), below a bf16 answer's own
// rounding of 1.7e-3.  `split` keeps low parts of A and B too and adds the two
// cross products: three times the work, an fp32 answer.
//
// Work per step with s the shorter and l the longer side: s^2 l + s^3 for the
// two symmetric products (only tiles that touch the lower triangle are
// computed, and written twice) and 2 s^2 l: bound by the tensor cores, except
// a few small matrices, which are bound by the latency of 15 dependent launches.
//
// One persistent warp-specialised kernel does every product: TMA loads, one
// tcgen05.mma issuer, accumulators double-buffered in TMEM so that a tile's
// epilogue runs under the next one's products.  A tile is 256 x 256 on a pair
// of SMs (cta_group::2) or 128 x 128 on one, by the longest SM's work, or, where
// that leaves SMs idle, 128 x 64; where SMs are idle all the same, a cluster
// shares the K of each tile and adds the parts up over distributed shared memory.
//
// Measured (B200; cuBLAS bf16 1634 TFLOP/s in bursts, 1395 sustained under the
// power cap), useful operations, symmetric ones counted once: 4096 x 4096, five
// steps, 1.09 ms = 1260 TFLOP/s in bursts, 1.32 ms = 1040 sustained (tensor pipe
// active 76 to 82 % of the time; the rest is the last wave of 256 tiles on 74
// pairs).  12 x 2304 x 768 with momentum and weights 470 us = 579 TFLOP/s: K is 768,
// so a tile brings 512 KB of addend and result to 768 KB of operands (tensor pipe
// 59 % active in X^T X, 40 % in the update).  768 x 768 89 us: 17 launches of 5.3 us,
// each a chain of launch, first load, 12 blocks of K (410 cycles each: 60 bytes of
// operands a cycle and SM) and epilogue, on 42 to 72 of the SMs.
#include <cuda_fp16.h>
#include <cudaTypedefs.h>

#include <iterator>
#include <type_traits>

#include "md_sm100.cuh"

constexpr int kMuonBatch = 64;  // matrices per call

// Mirrored field for field by minidist/ops/muon.py.
struct MdMuonParams {
  int count, rows, cols;
  int dtype;                // of src and out: 0 bf16, 1 fp16, 2 fp32
  int step;                 // 0: out = orthogonal(src); 1: Muon step (everything fp32)
  int split;                // 1: three products
  int iterations;
  float a, b, c, eps;
  // step form: src = gradients, m = momenta, out = weights, shadow = bf16 copies (or null entries)
  float momentum;
  int nesterov;
  float decay;              // W <- decay W - rate X
  float rate;
  const float* lr;          // null, or device learning rate: decay and rate are then per unit of it (1 - lr decay, lr rate)
  const float* inv_scale;   // null, or device factor on the gradients
  const float* skip;        // null, or device flag: nonzero leaves everything as it is
  void* workspace;
  long long workspace_bytes;
  int tile;                 // 0 choose, 1: 128 x 128 tiles, 2: 256 x 256 tiles on SM pairs, 3: 128 x 64
  md::Status* status;
  const void* src[kMuonBatch];
  float* m[kMuonBatch];
  void* out[kMuonBatch];
  __nv_bfloat16* shadow[kMuonBatch];
};

namespace md {
namespace muon {

constexpr float kScale = 4096.f;  // fp16 operands hold kScale times the value
constexpr int kChunk = 8192;      // elements per block of the norm and conversion passes
constexpr int kThreads = 256;

template <typename T> __device__ __forceinline__ float to_f(T v);
template <> __device__ __forceinline__ float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }
template <> __device__ __forceinline__ float to_f(__half v) { return __half2float(v); }
template <> __device__ __forceinline__ float to_f(float v) { return v; }

template <typename T>
struct alignas(sizeof(T) * 4) Four {
  T v[4];
};

__device__ __forceinline__ float block_sum(float v) {
  __shared__ float part[kThreads / 32];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, o);
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = v;
  __syncthreads();
  float t = 0.f;
#pragma unroll
  for (int i = 0; i < kThreads / 32; ++i) t += part[i];
  return t;
}

// What the first two kernels need (an argument's bytes count in a launch of a few us).
template <bool STEP>
struct Source {
  int rows, cols, nesterov;
  float momentum, eps;
  const float *inv_scale, *skip;
  const void* src[kMuonBatch];
  float* m[STEP ? kMuonBatch : 1];
};

// Momentum (step form) and the chunk's share of |U|^2.  grid (chunks, count).
template <typename T, bool STEP>
__global__ void __launch_bounds__(kThreads) norm_kernel(const __grid_constant__ Source<STEP> p,
                                                        float* __restrict__ partial) {
  pdl_trigger();
  pdl_wait();
  const int which = blockIdx.y;
  const long long n = static_cast<long long>(p.rows) * p.cols;
  const long long lo = static_cast<long long>(blockIdx.x) * kChunk;
  const long long hi = lo + kChunk < n ? lo + kChunk : n;
  const T* g = static_cast<const T*>(p.src[which]);
  float* m = STEP ? p.m[which] : nullptr;
  if (STEP && p.skip != nullptr && *p.skip != 0.f) return;
  const float gs = STEP && p.inv_scale != nullptr ? *p.inv_scale : 1.f;
  float sum = 0.f;
  auto one = [&](float gv, float mv, float& m_new) {
    if (!STEP) return gv;
    gv *= gs;
    m_new = fmaf(p.momentum, mv, gv);
    return p.nesterov ? fmaf(p.momentum, m_new, gv) : m_new;
  };
  const bool vec = (reinterpret_cast<uintptr_t>(g) % (4 * sizeof(T))) == 0 && (reinterpret_cast<uintptr_t>(m) & 15u) == 0;
  const long long nv = vec ? (hi - lo) / 4 : 0;
#pragma unroll 4
  for (long long i = threadIdx.x; i < nv; i += kThreads) {
    const Four<T> gv = *reinterpret_cast<const Four<T>*>(g + lo + 4 * i);
    Four<float> mv = {};
    if (STEP) mv = *reinterpret_cast<const Four<float>*>(m + lo + 4 * i);
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const float u = one(to_f(gv.v[q]), mv.v[q], mv.v[q]);
      sum = fmaf(u, u, sum);
    }
    if (STEP) *reinterpret_cast<Four<float>*>(m + lo + 4 * i) = mv;
  }
  for (long long k = lo + 4 * nv + threadIdx.x; k < hi; k += kThreads) {
    float mv = STEP ? m[k] : 0.f;
    const float u = one(to_f(g[k]), mv, mv);
    sum = fmaf(u, u, sum);
    if (STEP) m[k] = mv;
  }
  sum = block_sum(sum);
  if (threadIdx.x == 0) partial[static_cast<long long>(which) * gridDim.x + blockIdx.x] = sum;
}

__device__ __forceinline__ void split_half(float v, __half& hi, __half& lo) {
  hi = __float2half_rn(v);
  lo = __float2half_rn(v - __half2float(hi));
}

// X = U kScale / (|U| + eps) as high and low fp16 of row stride ldx.  grid (chunks, count).
template <typename T, bool STEP>
__global__ void __launch_bounds__(kThreads) convert_kernel(const __grid_constant__ Source<STEP> p,
                                                           const float* __restrict__ partial, __half* __restrict__ xh,
                                                           __half* __restrict__ xl, int ldx) {
  pdl_trigger();
  pdl_wait();
  const int which = blockIdx.y;
  // The chunks' shares in a fixed order (the same in every block of the matrix).
  float total = 0.f;
  for (int i = threadIdx.x; i < static_cast<int>(gridDim.x); i += kThreads)
    total += partial[static_cast<long long>(which) * gridDim.x + i];
  total = block_sum(total);
  const float inv = kScale / (sqrtf(total) + p.eps);
  const long long n = static_cast<long long>(p.rows) * p.cols;
  const long long lo = static_cast<long long>(blockIdx.x) * kChunk;
  const long long hi = lo + kChunk < n ? lo + kChunk : n;
  const T* g = static_cast<const T*>(p.src[which]);
  const float* m = STEP ? p.m[which] : nullptr;
  const float gs = STEP && p.inv_scale != nullptr ? *p.inv_scale : 1.f;
  // Position of the chunk's first element; inside the chunk 32-bit division is enough.
  const long long row_lo = lo / p.cols;
  const uint32_t col_lo = static_cast<uint32_t>(lo - row_lo * p.cols), cols = static_cast<uint32_t>(p.cols);
  const long long base = (static_cast<long long>(which) * p.rows + row_lo) * ldx;
  auto place = [&](uint32_t i) {  // of element lo + i
    const uint32_t e = col_lo + i, r = e / cols;
    return base + static_cast<long long>(r) * ldx + (e - r * cols);
  };
  auto value = [&](float gv, float mv) {
    if (!STEP) return gv * inv;
    return (p.nesterov ? fmaf(p.momentum, mv, gv * gs) : mv) * inv;
  };
  const bool vec = p.cols % 4 == 0 && (reinterpret_cast<uintptr_t>(g) % (4 * sizeof(T))) == 0 &&
                   (reinterpret_cast<uintptr_t>(m) & 15u) == 0;
  const long long nv = vec ? (hi - lo) / 4 : 0;  // (four columns never straddle rows; chunks are whole vectors)
#pragma unroll 4
  for (long long i = threadIdx.x; i < nv; i += kThreads) {
    const long long k = lo + 4 * i;
    const Four<T> gv = *reinterpret_cast<const Four<T>*>(g + k);
    Four<float> mv = {};
    if (STEP) mv = *reinterpret_cast<const Four<float>*>(m + k);
    const long long o = place(static_cast<uint32_t>(4 * i));
    Four<__half> h, l;
#pragma unroll
    for (int q = 0; q < 4; ++q) split_half(value(to_f(gv.v[q]), mv.v[q]), h.v[q], l.v[q]);
    *reinterpret_cast<Four<__half>*>(xh + o) = h;
    *reinterpret_cast<Four<__half>*>(xl + o) = l;
  }
  for (long long k = lo + 4 * nv + threadIdx.x; k < hi; k += kThreads) {
    const long long o = place(static_cast<uint32_t>(k - lo));
    split_half(value(to_f(g[k]), STEP ? m[k] : 0.f), xh[o], xl[o]);
  }
}

// ---------------------------------------------------------------------------
// The products
// ---------------------------------------------------------------------------
constexpr int BM = 128;   // rows of A per CTA and stage
constexpr int BK = 64;
constexpr int kShort = 128;  // K up to this: split products fill an accumulator for every 16 of it
constexpr int kOperand = BM * BK * 2;  // 16 KB
constexpr int kRing = 10 * kOperand;   // shared memory for the stages (and the partial sums of a shared K)
constexpr int kEpiWarps = 8;
constexpr int kChunkBytes = 32 * 32 * 2;       // an epilogue chunk of fp16: 32 rows x 64 bytes
constexpr int kWarpBytes = 4 * kChunkBytes;    // a warp's staging
constexpr int kPartBytes = 32 * 32 * 4;        // partial sums of a chunk
constexpr int kSmemBytes = 1024 + kRing + kEpiWarps * kWarpBytes + 512;
constexpr int kGemmThreads = 64 + 32 * kEpiWarps;

enum Mode : int { kGram = 0, kPoly = 1, kNext = 2, kLast = 3 };

struct GemmParams {
  int M, N, K;
  int tiles_m, tiles_n, per_batch, units, k_blocks, splits;
  int runs;  // accumulators that a block of K fills (split products of a short K: one for each 16)
  float alpha, beta;
  // kLast: what leaves
  int dtype, step;
  float decay, rate;
  const float* lr;
  const float* skip;
  Status* status;
};
struct LastParams : GemmParams {  // (1 KB of pointers, which the other launches need not carry)
  void* out[kMuonBatch];
  __nv_bfloat16* shadow[kMuonBatch];
};
template <int MODE>
using Params = std::conditional_t<MODE == kLast, LastParams, GemmParams>;

// kind::f16 with f16 operands, fp32 accumulators.
constexpr uint32_t idesc_f16(int M, int N, bool a_mn, bool b_mn) {
  return (1u << 4) | ((a_mn ? 1u : 0u) << 15) | ((b_mn ? 1u : 0u) << 16) | (static_cast<uint32_t>(N >> 3) << 17) |
         (static_cast<uint32_t>(M >> 4) << 24);
}

__device__ __forceinline__ uint32_t cluster_ctarank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ uint32_t map_to_cta(uint32_t smem_addr, uint32_t cta) {
  uint32_t out;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(out) : "r"(smem_addr), "r"(cta));
  return out;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// By every warp, its lanes together again: what was written to the others' shared memory is there.
__device__ __forceinline__ void cluster_join() {
  __syncwarp();
  cluster_sync();
}

// Tile load whose bytes are counted on `bar`: this CTA's barrier, or with CG = 2 the pair
// leader's (cluster address).  By a whole warp, one elected lane issues: addresses and
// coordinates stay in uniform registers.
template <int CG>
__device__ __forceinline__ void load_tile(const CUtensorMap* map, uint32_t bar, const uint8_t* dst, int x, int y, int z) {
  if constexpr (CG == 2) {
    asm volatile(
        "{\n\t.reg .pred e;\n\t.reg .b32 r;\n\t"
        "elect.sync r|e, 0xffffffff;\n\t"
        "@e cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes"
        " [%0], [%1, {%3, %4, %5}], [%2];\n\t}\n" ::"r"(smem_u32(dst)),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(x), "r"(y), "r"(z)
        : "memory");
  } else {
    asm volatile(
        "{\n\t.reg .pred e;\n\t.reg .b32 r;\n\t"
        "elect.sync r|e, 0xffffffff;\n\t"
        "@e cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
        " [%0], [%1, {%3, %4, %5}], [%2];\n\t}\n" ::"r"(smem_u32(dst)),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(x), "r"(y), "r"(z)
        : "memory");
  }
}
__device__ __forceinline__ void expect_elect(uint64_t* bar, uint32_t bytes) {
  asm volatile(
      "{\n\t.reg .pred e;\n\t.reg .b32 r;\n\t"
      "elect.sync r|e, 0xffffffff;\n\t"
      "@e mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;\n\t}\n" ::"r"(smem_u32(bar)), "r"(bytes)
      : "memory");
}
// A bounded wait by a whole warp: its lanes go on, or give up, together, as the elections and barriers that
// follow need them to.
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, Status* st, uint32_t where,
                                          volatile int* abort_flag) {
  return __all_sync(0xFFFFFFFFu, mbar_wait(bar, parity, st, where, abort_flag));
}
// The four MMAs of a block of K (their descriptors are a step of 16 of K apart), by one elected lane.
template <int CG, int kStepA, int kStepB>
__device__ __forceinline__ void mma_block(uint32_t tmem_d, uint64_t adesc, uint64_t bdesc, uint32_t idesc,
                                          uint32_t accumulate) {
  static_assert(BK == 64);
  if constexpr (CG == 2) {
    asm volatile(
        "{\n\t.reg .pred p, t, e;\n\t.reg .b32 r;\n\t.reg .b64 a1, a2, a3, b1, b2, b3;\n\t"
        "add.s64 a1, %1, %5;\n\tadd.s64 a2, a1, %5;\n\tadd.s64 a3, a2, %5;\n\t"
        "add.s64 b1, %2, %6;\n\tadd.s64 b2, b1, %6;\n\tadd.s64 b3, b2, %6;\n\t"
        "setp.ne.b32 p, %4, 0;\n\tsetp.eq.b32 t, %4, %4;\n\t"
        "elect.sync r|e, 0xffffffff;\n\t"
        "@e tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t"
        "@e tcgen05.mma.cta_group::2.kind::f16 [%0], a1, b1, %3, t;\n\t"
        "@e tcgen05.mma.cta_group::2.kind::f16 [%0], a2, b2, %3, t;\n\t"
        "@e tcgen05.mma.cta_group::2.kind::f16 [%0], a3, b3, %3, t;\n\t}\n" ::"r"(tmem_d),
        "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate), "n"(kStepA), "n"(kStepB)
        : "memory");
  } else {
    asm volatile(
        "{\n\t.reg .pred p, t, e;\n\t.reg .b32 r;\n\t.reg .b64 a1, a2, a3, b1, b2, b3;\n\t"
        "add.s64 a1, %1, %5;\n\tadd.s64 a2, a1, %5;\n\tadd.s64 a3, a2, %5;\n\t"
        "add.s64 b1, %2, %6;\n\tadd.s64 b2, b1, %6;\n\tadd.s64 b3, b2, %6;\n\t"
        "setp.ne.b32 p, %4, 0;\n\tsetp.eq.b32 t, %4, %4;\n\t"
        "elect.sync r|e, 0xffffffff;\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], a1, b1, %3, t;\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], a2, b2, %3, t;\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], a3, b3, %3, t;\n\t}\n" ::"r"(tmem_d),
        "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate), "n"(kStepA), "n"(kStepB)
        : "memory");
  }
}
// One MMA (16 of K), by one elected lane.
template <int CG>
__device__ __forceinline__ void mma_step(uint32_t tmem_d, uint64_t adesc, uint64_t bdesc, uint32_t idesc,
                                         uint32_t accumulate) {
  static_assert(CG == 1);
  asm volatile(
      "{\n\t.reg .pred p, e;\n\t.reg .b32 r;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "elect.sync r|e, 0xffffffff;\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(tmem_d),
      "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}
// Arrive on `bar` in every CTA of the pair once the MMAs issued so far are complete.
template <int CG>
__device__ __forceinline__ void commit_all(uint64_t* bar) {
  if constexpr (CG == 2) {
    const uint16_t mask = 0x3;
    asm volatile(
        "{\n\t.reg .pred e;\n\t.reg .b32 r;\n\t"
        "elect.sync r|e, 0xffffffff;\n\t"
        "@e tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;\n\t}\n" ::"r"(
            smem_u32(bar)),
        "h"(mask)
        : "memory");
  } else {
    umma_commit_elect(bar);
  }
}
template <int CG>
__device__ __forceinline__ void commit_own(uint64_t* bar) {
  if constexpr (CG == 2) {
    asm volatile(
        "{\n\t.reg .pred e;\n\t.reg .b32 r;\n\t"
        "elect.sync r|e, 0xffffffff;\n\t"
        "@e tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}\n" ::"r"(smem_u32(bar))
        : "memory");
  } else {
    umma_commit_elect(bar);
  }
}

// An epilogue chunk in and out (shared-memory addresses).
__device__ __forceinline__ void tma_load_3d_at(const CUtensorMap* map, uint64_t* bar, uint32_t dst, int x, int y, int z) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(smem_u32(bar)), "r"(x), "r"(y), "r"(z)
      : "memory");
}
__device__ __forceinline__ void tma_store_3d_at(const CUtensorMap* map, uint32_t src, int x, int y, int z) {
  asm volatile("cp.async.bulk.tensor.3d.global.shared::cta.bulk_group [%0, {%2, %3, %4}], [%1];" ::"l"(
                   reinterpret_cast<uint64_t>(map)),
               "r"(src), "r"(x), "r"(y), "r"(z)
               : "memory");
}

// Unit -> (matrix, tile row, tile column).  The symmetric products enumerate the tiles that reach the
// diagonal or lie below it only: R (tile rows over tile columns) more in every tile row.
template <bool SYM, int R>
__device__ __forceinline__ void decode(const GemmParams& p, int u, int& b, int& tm, int& tn) {
  b = u / p.per_batch;
  const int t = u - b * p.per_batch;
  if (SYM) {
    tm = static_cast<int>((sqrtf(8.f / R * static_cast<float>(t) + 1.f) - 1.f) * 0.5f);
    while (R * (tm + 1) * (tm + 2) / 2 <= t) ++tm;
    while (R * tm * (tm + 1) / 2 > t) --tm;
    tn = t - R * tm * (tm + 1) / 2;
  } else {
    tm = t / p.tiles_n;
    tn = t - tm * p.tiles_n;
  }
}

// Byte offset of a 16-byte piece in a chunk of 64-byte rows under the 64-byte TMA swizzle.
__device__ __forceinline__ uint32_t sw64_off(int row, int piece) {
  return static_cast<uint32_t>(row * 64 + ((piece ^ ((row >> 1) & 3)) << 4));
}

// f += the lane's row of a staged fp16 chunk times `by`.
__device__ __forceinline__ void add_staged(uint32_t chunk, int lane, float by, float (&f)[32]) {
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    uint32_t w[4];
    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3])
                 : "r"(chunk + sw64_off(lane, q)));
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const float2 v = __half22float2(*reinterpret_cast<const __half2*>(&w[k]));
      f[8 * q + 2 * k] = fmaf(by, v.x, f[8 * q + 2 * k]);
      f[8 * q + 2 * k + 1] = fmaf(by, v.y, f[8 * q + 2 * k + 1]);
    }
  }
}

// The lane's row of a chunk, packed in pairs.
__device__ __forceinline__ void stage(uint32_t chunk, int lane, const uint32_t (&w)[16]) {
#pragma unroll
  for (int q = 0; q < 4; ++q)
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(chunk + sw64_off(lane, q)), "r"(w[4 * q]),
                 "r"(w[4 * q + 1]), "r"(w[4 * q + 2]), "r"(w[4 * q + 3])
                 : "memory");
}
// ... and its transpose: the lane's row becomes a column.
__device__ __forceinline__ void stage_mirrored(uint32_t chunk, int lane, const uint32_t (&w)[16]) {
#pragma unroll
  for (int j = 0; j < 32; ++j)
    asm volatile("st.shared.b16 [%0], %1;" ::"r"(chunk + sw64_off(j, lane >> 3) + (lane & 7) * 2),
                 "h"(static_cast<uint16_t>(j & 1 ? w[j / 2] >> 16 : w[j / 2]))
                 : "memory");
}

// High and low fp16 parts of 32 values, packed in pairs (low parts only if asked for).
template <bool LOW>
__device__ __forceinline__ void split32(const float (&v)[32], uint32_t (&h)[16], uint32_t (&l)[16]) {
#pragma unroll
  for (int q = 0; q < 16; ++q) {
    const __half2 a = __floats2half2_rn(v[2 * q], v[2 * q + 1]);
    h[q] = *reinterpret_cast<const uint32_t*>(&a);
    if (LOW) {
      const float2 b = __half22float2(a);
      const __half2 c = __floats2half2_rn(v[2 * q] - b.x, v[2 * q + 1] - b.y);
      l[q] = *reinterpret_cast<const uint32_t*>(&c);
    }
  }
}

// What leaves: 32 x 32 fp32 values (kScale times X) staged in 128-byte rows, 16-byte pieces swizzled
// by the row.  A lane takes four neighbouring columns of every fourth row, so that a warp's access is
// four whole 128-byte lines; the weights to update are asked for one chunk ahead (`old`), because the
// products' operand loads keep the L2 busy and a load issued at its use waits 3000 cycles.
struct Out {
  float rate, decay;
  bool idle, wide;  // nothing to write; rows and addresses allow whole pieces
};
__device__ __forceinline__ void load_old(const LastParams& p, const Out& o, int b, int row0, int n0, int lane, float4 (&old)[8]) {
  const int col = n0 + (lane & 7) * 4;
  if (!p.step || !o.wide || o.idle || col >= p.N) return;
  const float* w = static_cast<const float*>(p.out[b]) + static_cast<long long>(row0 + (lane >> 3)) * p.N + col;
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (row0 + 4 * i + (lane >> 3) < p.M) old[i] = *reinterpret_cast<const float4*>(w + 4ll * i * p.N);
}
__device__ __forceinline__ void write_out(const LastParams& p, const Out& o, uint32_t staged, int b, int row0, int n0,
                                          int lane, const float4 (&old)[8]) {
  if (o.idle) return;
  const int col = n0 + (lane & 7) * 4;
  const int left = min(4, p.N - col);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int r = 4 * i + (lane >> 3);
    if (row0 + r >= p.M || left <= 0) continue;
    float4 v;
    asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];"
                 : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
                 : "r"(staged + r * 128 + (((lane & 7) ^ (r & 7)) << 4)));
    const long long at = static_cast<long long>(row0 + r) * p.N + col;
    if (o.wide) {
      if (p.step) {
        v.x = fmaf(old[i].x, o.decay, o.rate * v.x), v.y = fmaf(old[i].y, o.decay, o.rate * v.y);
        v.z = fmaf(old[i].z, o.decay, o.rate * v.z), v.w = fmaf(old[i].w, o.decay, o.rate * v.w);
      } else {
        v.x *= o.rate, v.y *= o.rate, v.z *= o.rate, v.w *= o.rate;
      }
      if (p.dtype == 2) {
        *reinterpret_cast<float4*>(static_cast<float*>(p.out[b]) + at) = v;
        if (p.shadow[b] != nullptr)
          *reinterpret_cast<uint2*>(p.shadow[b] + at) = make_uint2(pack_bf16x2(v.x, v.y), pack_bf16x2(v.z, v.w));
      } else if (p.dtype == 0) {
        *reinterpret_cast<uint2*>(static_cast<__nv_bfloat16*>(p.out[b]) + at) =
            make_uint2(pack_bf16x2(v.x, v.y), pack_bf16x2(v.z, v.w));
      } else {
        const __half2 x = __floats2half2_rn(v.x, v.y), y = __floats2half2_rn(v.z, v.w);
        *reinterpret_cast<uint2*>(static_cast<__half*>(p.out[b]) + at) =
            make_uint2(*reinterpret_cast<const uint32_t*>(&x), *reinterpret_cast<const uint32_t*>(&y));
      }
    } else {
      const float f[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if (j >= left) break;
        if (p.step) {
          float* w = static_cast<float*>(p.out[b]) + at + j;
          const float t = fmaf(*w, o.decay, o.rate * f[j]);
          *w = t;
          if (p.shadow[b] != nullptr) p.shadow[b][at + j] = __float2bfloat16_rn(t);
        } else if (p.dtype == 0) {
          static_cast<__nv_bfloat16*>(p.out[b])[at + j] = __float2bfloat16_rn(f[j] * o.rate);
        } else if (p.dtype == 1) {
          static_cast<__half*>(p.out[b])[at + j] = __float2half_rn(f[j] * o.rate);
        } else {
          static_cast<float*>(p.out[b])[at + j] = f[j] * o.rate;
        }
      }
    }
  }
}

// 32 x 32 fp32 in 128-byte rows, 16-byte pieces swizzled by the row: the lane's row in and out.
__device__ __forceinline__ void put_staged(uint32_t staged, int lane, const float (&v)[32]) {
#pragma unroll
  for (int q = 0; q < 8; ++q)
    asm volatile("st.shared.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(staged + lane * 128 + ((q ^ (lane & 7)) << 4)),
                 "f"(v[4 * q]), "f"(v[4 * q + 1]), "f"(v[4 * q + 2]), "f"(v[4 * q + 3])
                 : "memory");
}
__device__ __forceinline__ void get_staged(uint32_t staged, int lane, float (&v)[32]) {
#pragma unroll
  for (int q = 0; q < 8; ++q)
    asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];"
                 : "=f"(v[4 * q]), "=f"(v[4 * q + 1]), "=f"(v[4 * q + 2]), "=f"(v[4 * q + 3])
                 : "r"(staged + lane * 128 + ((q ^ (lane & 7)) << 4))
                 : "memory");
}

// The parts that a product reads and writes: X is a pair throughout, A and B with split products only.
template <bool SPLIT, int MODE>
struct Parts {
  static constexpr bool kAddend = MODE != kGram;
  static constexpr bool kAddLow = SPLIT || MODE == kNext || MODE == kLast;  // the addend is a pair
  static constexpr bool kLow = SPLIT || MODE == kNext;  // the result is a pair
};
template <bool SPLIT, int MODE>
struct Maps {  // high and low parts: operands, addend, result
  using P = Parts<SPLIT, MODE>;
  CUtensorMap a[SPLIT ? 2 : 1], b[SPLIT ? 2 : 1], d[P::kLow ? 2 : 1], c[P::kAddend && P::kAddLow ? 2 : 1];
};

// SPLIT: a stage holds both parts of both operands, loaded once for the three products of a block of K:
// low x high and high x low first, then high x high.  The tensor core truncates as it accumulates, always
// towards zero, which over a long K would cost a few bits of the 22, so every block's sum is added up in
// fp32 registers (errors after five steps: 1.0e-6 at 1000 x 3000, 2.4e-6 at 600 x 5000, as fp32's own
// products; 1.3e-5 at 1100 x 1030 when each product was one accumulation over K).  A short K has too few
// sums for fp32's own roundings to be worse than a block's four truncations, so there every 16 of K
// have an accumulator (63 x 1317: 1.7e-6, by blocks of 64 3.5e-6, fp32's own 1.5e-6; 54 x 297 1.4e-6,
// 2.5e-6 and 1.6e-6; 94 us and 98, nine of 65 x 2810 184 us and 175), which a long K would pay for and
// not need (1600 x 6400: 1.31 ms, by blocks 1.04 ms, and 1.0e-6 either way).
// KS (CG = 1): the blocks of K are shared by a cluster of `splits` CTAs, which sum their accumulators over
// distributed shared memory and finish a share of the tile each.
template <int CG, int BN, bool KS, bool SPLIT, bool A_MN, bool B_MN, int MODE>
__global__ void __launch_bounds__(kGemmThreads, 1)
    product_kernel(const __grid_constant__ Maps<SPLIT, MODE> maps, const __grid_constant__ Params<MODE> p) {
  constexpr bool SYM = MODE == kGram || MODE == kPoly;
  constexpr int R = CG * BM / BN;     // a tile is R times as high as wide
  constexpr int kCols = BN / CG;      // columns of the tile whose operand rows this CTA loads
  constexpr int kOperandB = kCols * BK * 2;
  constexpr int kAcc = SPLIT ? 4 : 2;  // accumulators in TMEM
  constexpr int kTmemCols = kAcc * BN;
  constexpr int kParts = SPLIT ? 2 : 1;
  constexpr int kStage = kParts * (kOperand + kOperandB);
  constexpr int kSums = KS ? BN / 32 * 4 * kPartBytes : 0;
  constexpr int kSt = (kRing - kSums) / kStage > 6 ? 6 : (kRing - kSums) / kStage;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sA = smem;
  uint8_t* sB = smem + kSt * kParts * kOperand;
  uint8_t* sRed = smem + kSt * kStage;  // KS: partial sums of this CTA's share of the tile
  uint8_t* sEpi = smem + kRing;
  uint64_t* bars = reinterpret_cast<uint64_t*>(sEpi + kEpiWarps * kWarpBytes);
  uint64_t* full_bar = bars;
  uint64_t* empty_bar = bars + kSt;
  uint64_t* tfull_bar = bars + 2 * kSt;
  uint64_t* tempty_bar = tfull_bar + kAcc;
  uint64_t* drain_bar = tempty_bar + kAcc;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain_bar + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(drain_bar + 2);
  uint64_t* c_bar = drain_bar + 3;  // two per epilogue warp
  static_assert((2 * kSt + 2 * kAcc + 3 + 2 * kEpiWarps) * 8 <= 512);

  // (Through a shuffle: the compiler then knows that a warp's role is the same for all its lanes, and
  // keeps the issuing loops' addresses and descriptors in uniform registers.)
  const int warp = __shfl_sync(0xFFFFFFFFu, static_cast<int>(threadIdx.x) >> 5, 0), lane = threadIdx.x & 31;
  const uint32_t crank = CG == 2 ? cluster_ctarank() : 0u;
  const int part = KS ? static_cast<int>(cluster_ctarank()) : 0;
  const bool leader = crank == 0;
  const int group = KS ? p.splits : CG;  // CTAs that share a tile
  const int first = static_cast<int>(blockIdx.x) / group, stride = static_cast<int>(gridDim.x) / group;

  if (threadIdx.x == 0) {
    for (int s = 0; s < kSt; ++s) {
      mbar_init(&full_bar[s], 1);
      mbar_init(&empty_bar[s], 1);
    }
    for (int a = 0; a < kAcc; ++a) {
      mbar_init(&tfull_bar[a], 1);
      mbar_init(&tempty_bar[a], CG * kEpiWarps);
    }
    mbar_init(drain_bar, 1);
    for (int i = 0; i < 2 * kEpiWarps; ++i) mbar_init(&c_bar[i], 1);
    *abort_flag = 0;
    fence_mbar_init();
    tma_prefetch_desc(&maps.a[0]);
    tma_prefetch_desc(&maps.b[0]);
  }
  if (warp == 1) {
    if constexpr (CG == 2) {
      asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)),
                   "r"(kTmemCols) : "memory");
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    } else {
      tmem_alloc(tmem_slot, kTmemCols);
      tmem_relinquish();
    }
  }
  tc_fence_before();
  __syncthreads();
  if constexpr (CG == 2 || KS) cluster_sync();  // the others run, and their barriers exist, before anything reaches them
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  pdl_trigger();
  pdl_wait();

  const int lo = KS ? p.k_blocks * part / p.splits : 0, hi = KS ? p.k_blocks * (part + 1) / p.splits : p.k_blocks;
  const int run = SPLIT ? 1 : p.k_blocks;  // blocks that one accumulator adds up
  // A tile on the diagonal of X X^T or A A: this CTA's rows of B are among its rows of A, loaded once.
  auto same = [&](int tm, int tn) { return SYM && tn / R == tm; };
  if (warp == 0) {
    // ---------------------------------------------------------- producer (whole warp, elected lane issues)
    int stage = 0;
    uint32_t phase = 0;
    int armed[kSt];
    for (int s = 0; s < kSt; ++s) armed[s] = -1;
    bool ok = true;
    for (int u = first; u < p.units && ok; u += stride) {
      int b, tm, tn;
      decode<SYM, R>(p, u, b, tm, tn);
      const int row = tm * (CG * BM) + static_cast<int>(crank) * BM;
      const int col = tn * BN + static_cast<int>(crank) * kCols;
      for (int i = lo; i < hi; ++i) {
        const int k = i * BK;
        if (!warp_wait(&empty_bar[stage], phase ^ 1u, p.status, 420, abort_flag)) {
          ok = false;
          break;
        }
        uint32_t bar = smem_u32(&full_bar[stage]);
        if constexpr (CG == 2) bar = map_to_cta(bar, 0);
        const bool once = same(tm, tn);
        if (leader) expect_elect(&full_bar[stage], CG * kParts * (kOperand + (once ? 0 : kOperandB)));
        armed[stage] = static_cast<int>(phase);
#pragma unroll
        for (int w = 0; w < kParts; ++w) {
          uint8_t* da = sA + (stage * kParts + w) * kOperand;
          uint8_t* db = sB + (stage * kParts + w) * kOperandB;
          if (A_MN) {
            load_tile<CG>(&maps.a[w], bar, da, row, k, b);
            load_tile<CG>(&maps.a[w], bar, da + kOperand / 2, row + 64, k, b);
          } else {
            load_tile<CG>(&maps.a[w], bar, da, k, row, b);
          }
          if (once) continue;
          if (B_MN) {
#pragma unroll
            for (int c = 0; c < kCols / 64; ++c)
              load_tile<CG>(&maps.b[w], bar, db + c * (kOperand / 2), col + c * 64, k, b);
          } else {
            load_tile<CG>(&maps.b[w], bar, db, k, col, b);
          }
        }
        if (++stage == kSt) {
          stage = 0;
          phase ^= 1u;
        }
      }
    }
    // No copy into this pair's shared memory may be in flight at exit (the follower's are counted
    // on the leader's barriers, which the leader's MMA has consumed before the last cluster barrier).
    if (leader)
      for (int s = 0; s < kSt; ++s)
        if (armed[s] >= 0) mbar_wait(&full_bar[s], static_cast<uint32_t>(armed[s]), p.status, 421, nullptr);
  } else if (warp == 1 && leader) {
    // ---------------------------------------------------------- MMA issuer
    constexpr uint32_t idesc = idesc_f16(CG * BM, BN, A_MN, B_MN);
    constexpr uint32_t kHalfTile = kOperand / 2;  // 64 MN-elements of 64 K-rows
    const uint64_t a_base = sdesc_sw128(smem_u32(sA), A_MN ? kHalfTile : 16, 1024);
    const uint64_t b_base = sdesc_sw128(smem_u32(sB), B_MN ? kHalfTile : 16, 1024);
    int stage = 0, acc = 0;
    uint32_t phase = 0, acc_phase = 0;
    // A wait that ran out is noted, and the warp goes on to where it hands its sums over: the lanes stay
    // together without a vote for every block of K (which cost 3 % at 768 x 768).
    bool ok = true;
    for (int u = first; u < p.units && ok; u += stride) {
      int b, tm, tn;
      decode<SYM, R>(p, u, b, tm, tn);
      for (int i0 = lo; i0 < hi; i0 += run) {
        ok &= mbar_wait(&tempty_bar[acc], acc_phase ^ 1u, p.status, 422, abort_flag);
        tc_fence_after();
        const uint32_t d_tmem = tmem_base + static_cast<uint32_t>(acc * BN);
        const int i1 = min(hi, i0 + run);
        for (int i = i0; i < i1; ++i) {
          ok &= mbar_wait(&full_bar[stage], phase, p.status, 423, abort_flag);
          tc_fence_after();
          const uint64_t a_st = a_base + static_cast<uint32_t>(stage * kParts * kOperand >> 4);
          // (64 rows of a stage, in either order, are half an operand on)
          const bool once = same(tm, tn);
          const uint64_t b_st = once ? a_st + static_cast<uint32_t>((tn % R) * (kOperand / 2) >> 4)
                                     : b_base + static_cast<uint32_t>(stage * kParts * kOperandB >> 4);
          const uint32_t a_low = static_cast<uint32_t>(kOperand >> 4);
          const uint32_t b_low = static_cast<uint32_t>((once ? kOperand : kOperandB) >> 4);
          constexpr uint32_t kStepA = A_MN ? 128 : 2, kStepB = B_MN ? 128 : 2;  // 16 of K on
          bool whole = true;  // the block is one accumulator's
          if constexpr (SPLIT) whole = p.runs == 1;
          if (whole) {
#pragma unroll
            for (int t = SPLIT ? 0 : 2; t < 3; ++t) {  // low x high, high x low, high x high
              const uint64_t at = a_st + (t == 0 ? a_low : 0u);
              const uint64_t bt = b_st + (t == 1 ? b_low : 0u);
              mma_block<CG, kStepA, kStepB>(d_tmem, at, bt, idesc, (i > i0 || (SPLIT && t > 0)) ? 1u : 0u);
            }
          }
          if constexpr (SPLIT) {
            if (!whole) {  // an accumulator for every 16 of K
#pragma unroll 1
              for (int r = 0; r < BK / 16; ++r) {
                const uint32_t d = tmem_base + static_cast<uint32_t>(acc * BN);
                mma_step<CG>(d, a_st + a_low + r * kStepA, b_st + r * kStepB, idesc, 0u);
                mma_step<CG>(d, a_st + r * kStepA, b_st + b_low + r * kStepB, idesc, 1u);
                mma_step<CG>(d, a_st + r * kStepA, b_st + r * kStepB, idesc, 1u);
                ok = __all_sync(0xFFFFFFFFu, ok);
                if (!ok || r + 1 == BK / 16) break;  // (handed over below)
                commit_all<CG>(&tfull_bar[acc]);
                if (++acc == kAcc) {
                  acc = 0;
                  acc_phase ^= 1u;
                }
                ok &= mbar_wait(&tempty_bar[acc], acc_phase ^ 1u, p.status, 422, abort_flag);
                tc_fence_after();
              }
            }
          }
          commit_all<CG>(&empty_bar[stage]);
          if (++stage == kSt) {
            stage = 0;
            phase ^= 1u;
          }
        }
        ok = __all_sync(0xFFFFFFFFu, ok);
        if (!ok) break;  // (not handed over)
        commit_all<CG>(&tfull_bar[acc]);
        if (++acc == kAcc) {
          acc = 0;
          acc_phase ^= 1u;
        }
      }
    }
    commit_own<CG>(drain_bar);  // every MMA is complete before TMEM is given back
    mbar_wait(drain_bar, 0, p.status, 424, nullptr);
  } else if (warp >= 2) {
    // ---------------------------------------------------------- epilogue
    const int quarter = warp & 3;          // the TMEM lanes this warp may read
    const int half = (warp - 2) / 4;       // two warps per quarter share the columns
    constexpr int kChunks = BN / 64;       // 32-column chunks per warp
    int acc = 0;
    uint32_t acc_phase = 0;
    uint32_t tempty[2] = {smem_u32(&tempty_bar[0]), smem_u32(&tempty_bar[1])};  // (CG = 2: the leader's)
    if constexpr (CG == 2) {
      static_assert(kAcc == 2);
      tempty[0] = map_to_cta(tempty[0], 0);
      tempty[1] = map_to_cta(tempty[1], 0);
    }
    auto release = [&]() {
      tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        if constexpr (CG == 2)
          asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(tempty[acc]) : "memory");
        else
          mbar_arrive(&tempty_bar[acc]);
      }
      if (++acc == kAcc) {
        acc = 0;
        acc_phase ^= 1u;
      }
    };
    // Staging: slot = the addend's chunk (high, low) on arrival, the result's on departure.  Two slots,
    // so that the next addend arrives under this chunk's arithmetic; one where a result with its
    // mirror image needs both.
    constexpr bool kAddend = Parts<SPLIT, MODE>::kAddend, kAddLow = Parts<SPLIT, MODE>::kAddLow,
                   kLow = Parts<SPLIT, MODE>::kLow;
    constexpr int kSlots = SPLIT && SYM ? 1 : 2;
    const uint32_t base = smem_u32(sEpi) + (warp - 2) * kWarpBytes;
    uint64_t* cb = c_bar + (warp - 2) * 2;
    int ctr = 0;           // chunks done
    int coming = 0;        // addends on their way, into the slots from ctr on
    // Slot `i` may be overwritten: its own accesses are done (fence, warp barrier), its result has been read.
    auto acquire = [&]() {
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) bulk_wait_read_all();
      __syncwarp();
    };
    auto fetch = [&](int i, int b, int row0, int n0) {
      acquire();
      ++coming;
      if (lane == 0) {
        uint64_t* bar = &cb[i % kSlots];
        const uint32_t dst = base + (i % kSlots) * (kWarpBytes / 2);
        mbar_arrive_expect_tx(bar, kAddLow ? 2 * kChunkBytes : kChunkBytes);
        tma_load_3d_at(&maps.c[0], bar, dst, n0, row0, b);
        if constexpr (kAddLow) tma_load_3d_at(&maps.c[1], bar, dst + kChunkBytes, n0, row0, b);
      }
    };
    bool ok = true;
    Out out;
    float4 old[8];
    auto prepare_out = [&](int b, int row0, int n0) {
      if constexpr (MODE == kLast) {
        const float lr = p.lr != nullptr ? *p.lr : 1.f;
        out.rate = p.step ? -p.rate * lr * (1.f / kScale) : 1.f / kScale;
        out.decay = p.lr != nullptr ? 1.f - lr * p.decay : p.decay;
        out.idle = p.step && p.skip != nullptr && *p.skip != 0.f;
        const unsigned long long piece = p.dtype == 2 ? 15u : 7u;
        out.wide = p.N % 4 == 0 && (reinterpret_cast<uintptr_t>(p.out[b]) & piece) == 0 &&
                   (reinterpret_cast<uintptr_t>(p.shadow[b]) & 7u) == 0;
        load_old(p, out, b, row0, n0, lane, old);
      }
    };
    auto load_acc = [&](int c, float (&v)[32]) {  // this warp's chunk c of the current accumulator
      uint32_t r[32];
      tmem_ld_32x32b_x32(tmem_base + (static_cast<uint32_t>(quarter * 32) << 16) +
                             static_cast<uint32_t>(acc * BN + (half * kChunks + c) * 32), r);
      tmem_ld_wait();
#pragma unroll
      for (int j = 0; j < 32; ++j) v[j] = __uint_as_float(r[j]);
    };
    // Split products: the runs of this warp's columns, added up in registers.
    auto add_runs = [&](float (&sum)[kChunks * 32]) {
#pragma unroll
      for (int j = 0; j < kChunks * 32; ++j) sum[j] = 0.f;
      for (int r = (hi - lo) * p.runs; r > 0; --r) {
        if (!warp_wait(&tfull_bar[acc], acc_phase, p.status, 425, abort_flag)) {
          ok = false;
          return;
        }
        tc_fence_after();
#pragma unroll
        for (int c = 0; c < kChunks; ++c) {
          float v[32];
          load_acc(c, v);
#pragma unroll
          for (int j = 0; j < 32; ++j) sum[c * 32 + j] += v[j];
        }
        release();
      }
    };
    // A chunk of products, from here to memory.  `more`: another one of this tile follows on its right.
    auto finish = [&](float (&v)[32], int b, int row0, int n0, bool more) {
      const uint32_t slot = base + (ctr % kSlots) * (kWarpBytes / 2);
#pragma unroll
      for (int j = 0; j < 32; ++j) v[j] *= p.alpha;
      if constexpr (kAddend) {
        if (kSlots == 2 && more) fetch(ctr + 1, b, row0, n0 + 32);
        if (!warp_wait(&cb[ctr % kSlots], static_cast<uint32_t>(ctr / kSlots) & 1u, p.status, 426, abort_flag)) {
          ok = false;
          return;
        }
        add_staged(slot, lane, p.beta, v);
        if (kAddLow) add_staged(slot + kChunkBytes, lane, p.beta, v);
        --coming;
        __syncwarp();  // the whole chunk has been read
      } else {
        // (the other slot's result may still be leaving; this one's has to be out)
        if (lane == 0) {
          if (kSlots == 2) asm volatile("cp.async.bulk.wait_group.read 1;" ::: "memory");
          else bulk_wait_read_all();
        }
        __syncwarp();
      }
      if constexpr (MODE == kLast) {
        put_staged(slot, lane, v);
        __syncwarp();
        write_out(p, out, slot, b, row0, n0, lane, old);
        if (more) load_old(p, out, b, row0, n0 + 32, lane, old);
      } else {
        const bool mirrored = SYM && n0 < row0;  // (the block on the diagonal is its own mirror image)
        uint32_t h[16], l[16];
        split32<kLow>(v, h, l);
        stage(slot, lane, h);
        if (kLow) stage(slot + kChunkBytes, lane, l);
        constexpr uint32_t kMirror = kLow ? 2 * kChunkBytes : kChunkBytes;
        if (SYM && mirrored) {
          stage_mirrored(slot + kMirror, lane, h);
          if (kLow) stage_mirrored(slot + kMirror + kChunkBytes, lane, l);
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) {
          tma_store_3d_at(&maps.d[0], slot, n0, row0, b);
          if constexpr (kLow) tma_store_3d_at(&maps.d[1], slot + kChunkBytes, n0, row0, b);
          if (SYM && mirrored) {
            tma_store_3d_at(&maps.d[0], slot + kMirror, row0, n0, b);
            if constexpr (kLow) tma_store_3d_at(&maps.d[1], slot + kMirror + kChunkBytes, row0, n0, b);
          }
          bulk_commit_group();
        }
      }
      ++ctr;
      if (kAddend && kSlots == 1 && more) fetch(ctr, b, row0, n0 + 32);
    };
    // Whether the 32 x 32 chunk at (row0, n0) is to be computed.
    auto wanted = [&](int row0, int n0) { return row0 < p.M && n0 < p.N && (!SYM || n0 <= row0); };

    if constexpr (KS) {
      // The tile's chunks are dealt to the CTAs: chunk t (columns t / 4, rows t % 4) belongs to CTA
      // t / per, warp t % per there.
      int b, tm, tn;
      decode<SYM, R>(p, first, b, tm, tn);
      const int per = BN / 32 * 4 / p.splits, mine = part * per + (warp - 2);
      const int row0 = tm * BM + (mine & 3) * 32, n0 = tn * BN + (mine >> 2) * 32;
      const bool has = warp - 2 < per && wanted(row0, n0);
      if (kAddend && has) fetch(ctr, b, row0, n0);
      if constexpr (MODE == kLast)
        if (has) prepare_out(b, row0, n0);
      auto send = [&](int c, float (&v)[32]) {
        const int column = half * kChunks + c, t = column * 4 + quarter;
        if (!wanted(tm * BM + quarter * 32, tn * BN + column * 32)) return;
        const uint32_t to = map_to_cta(smem_u32(sRed) + ((t % per) * p.splits + part) * kPartBytes, t / per);
#pragma unroll
        for (int q = 0; q < 8; ++q)
          asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(to + lane * 128 + ((q ^ (lane & 7)) << 4)),
                       "f"(v[4 * q]), "f"(v[4 * q + 1]), "f"(v[4 * q + 2]), "f"(v[4 * q + 3])
                       : "memory");
      };
      if constexpr (SPLIT) {
        float sum[kChunks * 32];
        add_runs(sum);
        if (ok) {
#pragma unroll
          for (int c = 0; c < kChunks; ++c) {
            float v[32];
#pragma unroll
            for (int j = 0; j < 32; ++j) v[j] = sum[c * 32 + j];
            send(c, v);
          }
        }
      } else {
        ok = warp_wait(&tfull_bar[acc], acc_phase, p.status, 425, abort_flag);
        if (ok) {
          tc_fence_after();
#pragma unroll 1
          for (int c = 0; c < kChunks; ++c) {
            float v[32];
            load_acc(c, v);
            send(c, v);
          }
        }
      }
      cluster_join();
      if (ok && has) {
        float v[32];
        const uint32_t from = smem_u32(sRed) + (warp - 2) * p.splits * kPartBytes;
        get_staged(from, lane, v);
#pragma unroll 1
        for (int s = 1; s < p.splits; ++s) {
          float w[32];
          get_staged(from + s * kPartBytes, lane, w);
#pragma unroll
          for (int j = 0; j < 32; ++j) v[j] += w[j];
        }
        finish(v, b, row0, n0, false);
      }
    } else {
      for (int u = first; u < p.units && ok; u += stride) {
        int b, tm, tn;
        decode<SYM, R>(p, u, b, tm, tn);
        const int row0 = tm * (CG * BM) + static_cast<int>(crank) * BM + quarter * 32;
        const int col0 = tn * BN + half * kChunks * 32;
        int chunks = 0;  // (those wanted come first)
        while (chunks < kChunks && wanted(row0, col0 + chunks * 32)) ++chunks;
        if (kAddend && chunks > 0) fetch(ctr, b, row0, col0);
        // (Split products of narrow tiles ask for the old weights after their sums: together they spill.)
        constexpr bool kLate = SPLIT && BN == 64;
        if constexpr (MODE == kLast && !kLate)
          if (chunks > 0) prepare_out(b, row0, col0);
        if constexpr (SPLIT) {
          float sum[kChunks * 32];
          add_runs(sum);
          if constexpr (MODE == kLast && kLate)
            if (chunks > 0) prepare_out(b, row0, col0);
          // (unrolled, so that the sums stay in registers)
#pragma unroll
          for (int c = 0; c < kChunks; ++c)
            if (c < chunks && ok) {
              float v[32];
#pragma unroll
              for (int j = 0; j < 32; ++j) v[j] = sum[c * 32 + j];
              finish(v, b, row0, col0 + c * 32, c + 1 < chunks);
            }
        } else {
          if (!warp_wait(&tfull_bar[acc], acc_phase, p.status, 425, abort_flag)) break;
          tc_fence_after();
#pragma unroll 1
          for (int c = 0; c < chunks && ok; ++c) {
            float v[32];
            load_acc(c, v);
            finish(v, b, row0, col0 + c * 32, c + 1 < chunks);
          }
          release();
        }
      }
    }
    // Nothing may be in flight into or out of shared memory at exit.
    for (; coming > 0; --coming, ++ctr)
      mbar_wait(&cb[ctr % kSlots], static_cast<uint32_t>(ctr / kSlots) & 1u, p.status, 427, nullptr);
    if (lane == 0) bulk_wait_all();
  }
  if constexpr (KS)
    if (warp < 2) cluster_join();
  tc_fence_before();
  __syncthreads();
  if constexpr (CG == 2) cluster_sync();
  tc_fence_after();
  if (warp == 1) {
    if constexpr (CG == 2)
      asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(kTmemCols) : "memory");
    else
      tmem_dealloc(tmem_base, kTmemCols);
  }
}

// ---------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------
PFN_cuTensorMapEncodeTiled_v12000 g_encode_muon = nullptr;

bool get_encoder() {
  if (g_encode_muon != nullptr) return true;
  void* fn = nullptr;
  cudaDriverEntryPointQueryResult q;
  if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &fn, cudaEnableDefault, &q) != cudaSuccess ||
      q != cudaDriverEntryPointSuccess || fn == nullptr)
    return false;
  g_encode_muon = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(fn);
  return true;
}

// A stack of fp16 matrices and its tensor maps: operand tiles of 64 columns x 128 rows (K-major) or
// 64 columns x 64 rows (K-major for narrow tiles, MN-major), and epilogue chunks of 32 x 32.
// Columns and rows past the matrix read as zero and are not written.
struct Stack {
  CUtensorMap by_128, by_64, chunk;
  bool make(void* ptr, int rows, int cols, int count) {
    return encode(&by_128, ptr, rows, cols, count, 64, 128) && encode(&by_64, ptr, rows, cols, count, 64, 64) &&
           encode(&chunk, ptr, rows, cols, count, 32, 32);
  }
  static bool encode(CUtensorMap* map, void* ptr, int rows, int cols, int count, cuuint32_t box_cols, cuuint32_t box_rows) {
    const cuuint64_t ld = static_cast<cuuint64_t>(cols + 7) / 8 * 16;
    cuuint64_t dims[3] = {static_cast<cuuint64_t>(cols), static_cast<cuuint64_t>(rows), static_cast<cuuint64_t>(count)};
    cuuint64_t strides[2] = {ld, ld * rows};
    cuuint32_t box[3] = {box_cols, box_rows, 1};
    cuuint32_t estr[3] = {1, 1, 1};
    return g_encode_muon(map, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, ptr, dims, strides, box, estr,
                         CU_TENSOR_MAP_INTERLEAVE_NONE,
                         box_cols == 64 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B,
                         CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
  }
};
// High and low parts.
struct Pair {
  Stack part[2];
};

int tiles(int n, int t) { return (n + t - 1) / t; }
// Tiles of height x width that a product computes per matrix: all, or those that reach the diagonal.
long long tiles_of(bool sym, int rows, int cols, int height, int width) {
  const long long m = tiles(rows, height), n = tiles(cols, width), r = height / width;
  return sym ? r * m * (m - 1) / 2 + n : m * n;
}

int sms() {
  static int n = 0;
  if (n == 0) {
    int dev = 0;
    cudaGetDevice(&dev);
    cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev);
  }
  return n;
}

template <int CG, int BN, bool KS, bool SPLIT, bool A_MN, bool B_MN, int MODE>
cudaError_t launch_product(const Pair& a, const Pair& b, const Pair& c, const Pair& d, LastParams& p, int count,
                           cudaStream_t stream) {
  constexpr bool SYM = MODE == kGram || MODE == kPoly;
  p.tiles_m = tiles(p.M, BM * CG);
  p.tiles_n = tiles(p.N, BN);
  p.per_batch = static_cast<int>(tiles_of(SYM, p.M, p.N, BM * CG, BN));
  p.units = p.per_batch * count;
  p.k_blocks = (p.K + BK - 1) / BK;
  p.runs = p.K <= kShort ? BK / 16 : 1;
  auto kern = product_kernel<CG, BN, KS, SPLIT, A_MN, B_MN, MODE>;
  static int done[64] = {0};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev >= 64 || !done[dev]) {
    const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemBytes);
    if (e != cudaSuccess) return e;
    if (dev < 64) done[dev] = 1;
  }
  const int slots = sms() / CG, group = KS ? p.splits : CG;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(group * (KS || p.units < slots ? p.units : slots)));
  cfg.blockDim = dim3(kGemmThreads);
  cfg.dynamicSmemBytes = kSmemBytes;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  cfg.attrs = attr;
  cfg.numAttrs = 0;
  if (CG == 2 || KS) {
    attr[cfg.numAttrs].id = cudaLaunchAttributeClusterDimension;
    attr[cfg.numAttrs].val.clusterDim.x = group;
    attr[cfg.numAttrs].val.clusterDim.y = 1;
    attr[cfg.numAttrs].val.clusterDim.z = 1;
    ++cfg.numAttrs;
  }
  if (pdl_enabled()) {
    attr[cfg.numAttrs].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[cfg.numAttrs].val.programmaticStreamSerializationAllowed = 1;
    ++cfg.numAttrs;
  }
  Maps<SPLIT, MODE> maps;
  for (int i = 0; i < static_cast<int>(std::size(maps.a)); ++i) {
    maps.a[i] = A_MN ? a.part[i].by_64 : a.part[i].by_128;
    maps.b[i] = B_MN || BN / CG == 64 ? b.part[i].by_64 : b.part[i].by_128;
  }
  for (int i = 0; i < static_cast<int>(std::size(maps.c)); ++i) maps.c[i] = c.part[i].chunk;
  for (int i = 0; i < static_cast<int>(std::size(maps.d)); ++i) maps.d[i] = d.part[i].chunk;
  return cudaLaunchKernelEx(&cfg, kern, maps, static_cast<const Params<MODE>&>(p));
}

// How a product is cut.  `tile`: 0 choose, 1: 128 x 128 tiles, 2: 256 x 256 tiles on SM pairs
// (not split products), 3: 128 x 64.
template <bool A_MN, bool B_MN, int MODE>
cudaError_t product(int tile, bool split, const Pair& a, const Pair& b, const Pair& c, const Pair& d, LastParams& p,
                    int count, cudaStream_t s) {
  constexpr bool SYM = MODE == kGram || MODE == kPoly;
  auto units = [&](int height, int width) { return tiles_of(SYM, p.M, p.N, height, width) * count; };
  p.splits = 1;
  if (tile == 3 || (tile == 0 && units(BM, 64) <= sms())) {
    // Few tiles: narrow ones (768 x 768: 89 us, with 128 x 128 106; fp32 2 x 203 x 1001: 134 and 186), and K
    // shared by as many CTAs as fit the SMs together and have enough blocks each to pay for the exchange:
    // 8 of single products (256 x 4096: 84 us, by twos 89; 512 x 512, not shared, 81, by twos 93), of split
    // products one (fp32 2 x 203 x 1001: 110 us, not shared 134; 600 x 5000 278 and 444).
    const int blocks = tiles(p.K, BK), least = split ? 1 : 8;
    while (p.splits < 8 && units(BM, 64) * 2 * p.splits <= sms() && blocks >= 2 * least * p.splits) p.splits *= 2;
    if (p.splits > 1)
      return split ? launch_product<1, 64, true, true, A_MN, B_MN, MODE>(a, b, c, d, p, count, s)
                   : launch_product<1, 64, true, false, A_MN, B_MN, MODE>(a, b, c, d, p, count, s);
    return split ? launch_product<1, 64, false, true, A_MN, B_MN, MODE>(a, b, c, d, p, count, s)
                 : launch_product<1, 64, false, false, A_MN, B_MN, MODE>(a, b, c, d, p, count, s);
  }
  if (split) return launch_product<1, 128, false, true, A_MN, B_MN, MODE>(a, b, c, d, p, count, s);
  // 128 x 128 tiles on one SM or 256 x 256 on a pair: whichever should take less time, counted in blocks
  // of K on a pair (512 cycles).  A chain is the first tile's products, then for every further tile the
  // longer of its products and its epilogue, then the last epilogue; a small tile has half the products
  // and epilogue at 0.8 and 0.57 of the time (its operands are loaded 1.5 times as often), a pair 5
  // blocks more to begin and end.  The constants are fitted to 24 shapes (profiles/operators.md).  One /
  // pairs / the rule, us for five steps: 12 x 768 x 768 199 / 223 / 200, 4 x 1024 x 1024 165 / 223 / 151,
  // 12 x 2304 x 768 434 / 425 / 419, 1600 x 6400 408 / 467 / 362, 2500 x 2500 711 / 485 / 485, 4096 x 4096
  // 1312 / 1119 / 1127; it errs most, by 3 %, at 5 x 1500 x 1700 (649 / 530 / 544).
  auto chain = [](long long waves, float main, float epilogue) {
    return main + static_cast<float>(waves - 1) * fmaxf(main, epilogue) + epilogue;
  };
  constexpr int kPieces = MODE == kGram ? 2 : MODE == kPoly ? 3 : 4;  // 16-bit parts in and out, mirror images too
  const float blocks = static_cast<float>(tiles(p.K, BK)), epilogue = 6.f * kPieces;
  const int pairs = sms() / 2;
  const float on_pairs = chain((units(2 * BM, 2 * BM) + pairs - 1) / pairs, blocks, epilogue) + 5.f;
  const float on_one = chain((units(BM, BM) + sms() - 1) / sms(), 0.8f * blocks, 0.57f * epilogue);
  if (tile == 2 || (tile == 0 && on_pairs <= on_one))
    return launch_product<2, 256, false, false, A_MN, B_MN, MODE>(a, b, c, d, p, count, s);
  return launch_product<1, 128, false, false, A_MN, B_MN, MODE>(a, b, c, d, p, count, s);
}

struct Layout {  // byte offsets in the workspace (each 256-byte aligned)
  long long x[2][2], a[2], f[2], partial, total;
};
Layout layout(int count, int rows, int cols, bool split) {
  const int s = rows < cols ? rows : cols;
  const long long x = static_cast<long long>(count) * rows * ((cols + 7) / 8 * 8) * 2;
  const long long g = static_cast<long long>(count) * s * ((s + 7) / 8 * 8) * 2;
  const long long chunks = (static_cast<long long>(rows) * cols + kChunk - 1) / kChunk;
  Layout l{};
  long long at = 0;
  auto take = [&](long long bytes) {
    const long long o = at;
    at += (bytes + 255) / 256 * 256;
    return o;
  };
  for (int i = 0; i < 2; ++i)
    for (int w = 0; w < 2; ++w) l.x[i][w] = take(x);
  for (int w = 0; w <= static_cast<int>(split); ++w) {
    l.a[w] = take(g);
    l.f[w] = take(g);
  }
  l.partial = take(chunks * count * 4);
  l.total = at;
  return l;
}

template <typename T, bool STEP>
cudaError_t prepare(const MdMuonParams& p, const Layout& l, int chunks, cudaStream_t s) {
  uint8_t* ws = static_cast<uint8_t*>(p.workspace);
  float* partial = reinterpret_cast<float*>(ws + l.partial);
  Source<STEP> from{p.rows, p.cols, p.nesterov, p.momentum, p.eps, p.inv_scale, p.skip};
  for (int i = 0; i < p.count; ++i) {
    from.src[i] = p.src[i];
    if (STEP) from.m[i] = p.m[i];
  }
  const dim3 grid(chunks, p.count), block(kThreads);
  cudaError_t e = launch_pdl(norm_kernel<T, STEP>, grid, block, 0, s, from, partial);
  if (e != cudaSuccess) return e;
  return launch_pdl(convert_kernel<T, STEP>, grid, block, 0, s, from, static_cast<const float*>(partial),
                    reinterpret_cast<__half*>(ws + l.x[0][0]), reinterpret_cast<__half*>(ws + l.x[0][1]),
                    (p.cols + 7) / 8 * 8);
}

}  // namespace muon
}  // namespace md

// Bytes of workspace that md_muon needs.
extern "C" long long md_muon_workspace(int count, int rows, int cols, int split) {
  if (count <= 0 || rows <= 0 || cols <= 0) return 0;
  return md::muon::layout(count, rows, cols, split != 0).total;
}

// 0 ok; negative: refused (nothing launched); positive: CUDA error of a launch.
extern "C" int md_muon(const MdMuonParams* prm, cudaStream_t stream) {
  using namespace md::muon;
  if (prm == nullptr) return -1;
  const MdMuonParams& p = *prm;
  if (p.count <= 0 || p.count > kMuonBatch || p.rows <= 0 || p.cols <= 0 || p.iterations < 1) return -2;
  if (p.dtype < 0 || p.dtype > 2 || (p.step && p.dtype != 2)) return -3;
  for (int i = 0; i < p.count; ++i)
    if (p.src[i] == nullptr || p.out[i] == nullptr || (p.step && p.m[i] == nullptr)) return -4;
  const Layout l = layout(p.count, p.rows, p.cols, p.split != 0);
  if (p.workspace == nullptr || (reinterpret_cast<uintptr_t>(p.workspace) & 255u) || p.workspace_bytes < l.total) return -5;
  if (!get_encoder()) return -6;
  const long long chunks = (static_cast<long long>(p.rows) * p.cols + kChunk - 1) / kChunk;
  if (chunks > 0x7fffffffll) return -7;

  uint8_t* ws = static_cast<uint8_t*>(p.workspace);
  const int small = p.rows < p.cols ? p.rows : p.cols;
  const bool tall = p.rows > p.cols, split = p.split != 0;
  Pair x[2], a{}, f{};
  bool ok = true;
  for (int i = 0; i < 2; ++i)
    for (int w = 0; w < 2; ++w) ok = ok && x[i].part[w].make(ws + l.x[i][w], p.rows, p.cols, p.count);
  for (int w = 0; w <= static_cast<int>(split); ++w)
    ok = ok && a.part[w].make(ws + l.a[w], small, small, p.count) &&
         f.part[w].make(ws + l.f[w], small, small, p.count);
  if (!ok) return -8;

  cudaError_t e = p.step           ? prepare<float, true>(p, l, static_cast<int>(chunks), stream)
                  : p.dtype == 0   ? prepare<__nv_bfloat16, false>(p, l, static_cast<int>(chunks), stream)
                  : p.dtype == 1   ? prepare<__half, false>(p, l, static_cast<int>(chunks), stream)
                                   : prepare<float, false>(p, l, static_cast<int>(chunks), stream);
  if (e != cudaSuccess) return static_cast<int>(e);

  LastParams g{};
  g.status = p.status;
  g.dtype = p.dtype, g.step = p.step;
  g.decay = p.decay, g.rate = p.rate, g.lr = p.lr, g.skip = p.skip;
  for (int i = 0; i < p.count; ++i) g.out[i] = p.out[i], g.shadow[i] = p.step ? p.shadow[i] : nullptr;
  const float per = 1.f / kScale;
  for (int it = 0; it < p.iterations && e == cudaSuccess; ++it) {
    const bool last = it + 1 == p.iterations;
    const Pair &xs = x[it & 1], &xn = x[~it & 1];
    // A = X X^T (X^T X)
    g.M = g.N = small, g.K = tall ? p.rows : p.cols;
    g.alpha = per, g.beta = 0.f;
    e = tall ? product<true, true, kGram>(p.tile, split, xs, xs, a, a, g, p.count, stream)
             : product<false, false, kGram>(p.tile, split, xs, xs, a, a, g, p.count, stream);
    if (e != cudaSuccess) break;
    // B = b A + c A A
    g.K = small;
    g.alpha = p.c * per, g.beta = p.b;
    e = product<false, false, kPoly>(p.tile, split, a, a, a, f, g, p.count, stream);
    if (e != cudaSuccess) break;
    // X <- a X + B X (X B)
    g.M = p.rows, g.N = p.cols;
    g.alpha = per, g.beta = p.a;
    if (last)
      e = tall ? product<false, false, kLast>(p.tile, split, xs, f, xs, xn, g, p.count, stream)
               : product<false, true, kLast>(p.tile, split, f, xs, xs, xn, g, p.count, stream);
    else
      e = tall ? product<false, false, kNext>(p.tile, split, xs, f, xs, xn, g, p.count, stream)
               : product<false, true, kNext>(p.tile, split, f, xs, xs, xn, g, p.count, stream);
  }
  return static_cast<int>(e);
}
