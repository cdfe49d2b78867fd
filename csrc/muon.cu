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
// of SMs (cta_group::2) or 128 x 128 on one.
#include <cuda_fp16.h>
#include <cudaTypedefs.h>

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
  int tile;                 // 0 choose, 1: 128 x 128 tiles, 2: 256 x 256 tiles on SM pairs
  md::Status* status;
  const void* src[kMuonBatch];
  float* m[kMuonBatch];
  void* out[kMuonBatch];
  __nv_bfloat16* shadow[kMuonBatch];
};

namespace md {
namespace muon {

constexpr float kScale = 4096.f;  // fp16 operands hold kScale times the value
constexpr int kChunk = 16384;     // elements per block of the norm and conversion passes
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

// Momentum (step form) and the chunk's share of |U|^2.  grid (chunks, count).
template <typename T, bool STEP>
__global__ void __launch_bounds__(kThreads) norm_kernel(const __grid_constant__ MdMuonParams p, float* __restrict__ partial) {
  pdl_trigger();
  pdl_wait();
  const long long n = static_cast<long long>(p.rows) * p.cols;
  const long long lo = static_cast<long long>(blockIdx.x) * kChunk;
  const long long hi = lo + kChunk < n ? lo + kChunk : n;
  const T* g = static_cast<const T*>(p.src[blockIdx.y]);
  float* m = p.m[blockIdx.y];
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
  if (threadIdx.x == 0) partial[static_cast<long long>(blockIdx.y) * gridDim.x + blockIdx.x] = sum;
}

__device__ __forceinline__ void split_half(float v, __half& hi, __half& lo) {
  hi = __float2half_rn(v);
  lo = __float2half_rn(v - __half2float(hi));
}

// X = U kScale / (|U| + eps) as high and low fp16 of row stride ldx.  grid (chunks, count).
template <typename T, bool STEP>
__global__ void __launch_bounds__(kThreads) convert_kernel(const __grid_constant__ MdMuonParams p,
                                                           const float* __restrict__ partial, __half* __restrict__ xh,
                                                           __half* __restrict__ xl, int ldx) {
  pdl_trigger();
  pdl_wait();
  // The chunks' shares in a fixed order (the same in every block of the matrix).
  float total = 0.f;
  for (int i = threadIdx.x; i < static_cast<int>(gridDim.x); i += kThreads)
    total += partial[static_cast<long long>(blockIdx.y) * gridDim.x + i];
  total = block_sum(total);
  const float inv = kScale / (sqrtf(total) + p.eps);
  const long long n = static_cast<long long>(p.rows) * p.cols;
  const long long lo = static_cast<long long>(blockIdx.x) * kChunk;
  const long long hi = lo + kChunk < n ? lo + kChunk : n;
  const T* g = static_cast<const T*>(p.src[blockIdx.y]);
  const float* m = p.m[blockIdx.y];
  const float gs = STEP && p.inv_scale != nullptr ? *p.inv_scale : 1.f;
  const long long base = static_cast<long long>(blockIdx.y) * p.rows * ldx;
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
    const long long r = k / p.cols, o = base + r * ldx + (k - r * p.cols);
    Four<__half> h, l;
#pragma unroll
    for (int q = 0; q < 4; ++q) split_half(value(to_f(gv.v[q]), mv.v[q]), h.v[q], l.v[q]);
    *reinterpret_cast<Four<__half>*>(xh + o) = h;
    *reinterpret_cast<Four<__half>*>(xl + o) = l;
  }
  for (long long k = lo + 4 * nv + threadIdx.x; k < hi; k += kThreads) {
    const long long r = k / p.cols, o = base + r * ldx + (k - r * p.cols);
    split_half(value(to_f(g[k]), STEP ? m[k] : 0.f), xh[o], xl[o]);
  }
}

// ---------------------------------------------------------------------------
// The products
// ---------------------------------------------------------------------------
constexpr int BM = 128;   // rows of A and of B per CTA and stage
constexpr int BK = 64;
constexpr int kOperand = BM * BK * 2;  // 16 KB
constexpr int kStages = 6;
constexpr int kEpiWarps = 8;
constexpr int kSmemBytes = 1024 + kStages * 2 * kOperand + 256;
constexpr int kGemmThreads = 64 + 32 * kEpiWarps;

// Split products: the tensor core truncates as it accumulates, which over a long K costs a few bits of
// the 22.  After this many blocks of K the accumulator is added to fp32 registers and starts again
// (measured error of a 1100 x 1030 answer: 1.3e-5 in one accumulation).
constexpr int kSplitRun = 2;

enum Mode : int { kGram = 0, kPoly = 1, kNext = 2, kLast = 3 };

struct GemmParams {
  int M, N, K;
  int tiles_m, tiles_n, per_batch, units, k_blocks;
  float alpha, beta;
  const __half* c[2];       // kPoly: A, kNext / kLast: X (high, low or null)
  __half* d[2];             // high, low or null
  long long ldc, ldd, batch_c, batch_d;
  // kLast: what leaves
  int dtype, step;
  float decay, rate;
  const float* lr;
  const float* skip;
  Status* status;
  void* out[kMuonBatch];
  __nv_bfloat16* shadow[kMuonBatch];
};

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

// Tile load whose bytes are counted on `bar`: this CTA's barrier, or with CG = 2 the pair
// leader's (cluster address).
template <int CG>
__device__ __forceinline__ void load_tile(const CUtensorMap* map, uint32_t bar, void* dst, int x, int y, int z) {
  if constexpr (CG == 2) {
    asm volatile(
        "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes"
        " [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(smem_u32(dst)),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(x), "r"(y), "r"(z)
        : "memory");
  } else {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
        " [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(smem_u32(dst)),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(x), "r"(y), "r"(z)
        : "memory");
  }
}
template <int CG>
__device__ __forceinline__ void mma(uint32_t tmem_d, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
  if constexpr (CG == 2) {
    asm volatile(
        "{\n\t.reg .pred p, e;\n\t.reg .b32 r;\n\t"
        "elect.sync r|e, 0xffffffff;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "@e tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(tmem_d),
        "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
        : "memory");
  } else {
    umma_bf16_ss_elect(tmem_d, adesc, bdesc, idesc, accumulate);  // (the element type is in idesc)
  }
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

// Unit -> (matrix, tile row, tile column).  The symmetric products enumerate the tiles on and below
// the diagonal only.
template <bool SYM>
__device__ __forceinline__ void decode(const GemmParams& p, int u, int& b, int& tm, int& tn) {
  b = u / p.per_batch;
  const int t = u - b * p.per_batch;
  if (SYM) {
    tm = static_cast<int>((sqrtf(8.f * static_cast<float>(t) + 1.f) - 1.f) * 0.5f);
    while ((tm + 1) * (tm + 2) / 2 <= t) ++tm;
    while (tm * (tm + 1) / 2 > t) --tm;
    tn = t - tm * (tm + 1) / 2;
  } else {
    tm = t / p.tiles_n;
    tn = t - tm * p.tiles_n;
  }
}

__device__ __forceinline__ void load32(const __half* src, bool full, int left, float (&f)[32]) {
  if (full) {
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const uint4 w = *reinterpret_cast<const uint4*>(src + 8 * q);
      const uint32_t ws[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const float2 v = __half22float2(*reinterpret_cast<const __half2*>(&ws[k]));
        f[8 * q + 2 * k] = v.x;
        f[8 * q + 2 * k + 1] = v.y;
      }
    }
  } else {
#pragma unroll
    for (int j = 0; j < 32; ++j) f[j] = j < left ? __half2float(src[j]) : 0.f;
  }
}

// One accumulator row of a thread, 32 columns from n0: the epilogue of one chunk.  `acc` is in TMEM
// (its load is issued here, ahead of C's) or, with split products, already in registers.
template <int MODE, bool SPLIT>
__device__ __forceinline__ void epilogue_chunk(const GemmParams& p, int b, int row0, int lane, int n0, uint32_t taddr,
                                               const float* sum) {
  const int row = row0 + lane;
  const bool row_ok = row < p.M;
  const bool full = n0 + 32 <= p.N;
  const int left = p.N - n0;
  constexpr bool SYM = MODE == kGram || MODE == kPoly;
  if (SYM && n0 > row0 + 31) return;  // above the diagonal (warp-uniform)
  uint32_t r[32];
  if constexpr (!SPLIT) tmem_ld_32x32b_x32(taddr, r);
  float cf[32], cl[32];
  constexpr bool has_low = SPLIT || MODE == kNext || MODE == kLast;  // X is always a pair, A with split products
  if (MODE != kGram && row_ok) {
    const long long o = b * p.batch_c + row * p.ldc + n0;
    load32(p.c[0] + o, full, left, cf);
    if (has_low) load32(p.c[1] + o, full, left, cl);
  }
  if constexpr (!SPLIT) tmem_ld_wait();
  if (!row_ok) return;  // (nothing warp-collective below)
  float v[32];
#pragma unroll
  for (int j = 0; j < 32; ++j) {
    v[j] = (SPLIT ? sum[j] : __uint_as_float(r[j])) * p.alpha;
    if (MODE != kGram) v[j] = fmaf(p.beta, has_low ? cf[j] + cl[j] : cf[j], v[j]);
  }
  if constexpr (MODE == kLast) {
    if (p.step) {
      if (p.skip != nullptr && *p.skip != 0.f) return;
      const float lr = p.lr != nullptr ? *p.lr : 1.f;
      const float rate = p.rate * lr * (1.f / kScale), decay = p.lr != nullptr ? 1.f - lr * p.decay : p.decay;
      float* w = static_cast<float*>(p.out[b]) + static_cast<long long>(row) * p.N + n0;
      __nv_bfloat16* sh = p.shadow[b];
      if (sh != nullptr) sh += static_cast<long long>(row) * p.N + n0;
      if (full && (reinterpret_cast<uintptr_t>(w) & 15u) == 0 && (reinterpret_cast<uintptr_t>(sh) & 7u) == 0) {
#pragma unroll
        for (int q = 0; q < 8; ++q) {
          float4 t = *reinterpret_cast<const float4*>(w + 4 * q);
          t.x = fmaf(t.x, decay, -rate * v[4 * q]);
          t.y = fmaf(t.y, decay, -rate * v[4 * q + 1]);
          t.z = fmaf(t.z, decay, -rate * v[4 * q + 2]);
          t.w = fmaf(t.w, decay, -rate * v[4 * q + 3]);
          *reinterpret_cast<float4*>(w + 4 * q) = t;
          if (sh != nullptr) *reinterpret_cast<uint2*>(sh + 4 * q) = make_uint2(pack_bf16x2(t.x, t.y), pack_bf16x2(t.z, t.w));
        }
      } else {
#pragma unroll
        for (int j = 0; j < 32; ++j)
          if (j < left) {
            const float t = fmaf(w[j], decay, -rate * v[j]);
            w[j] = t;
            if (sh != nullptr) sh[j] = __float2bfloat16_rn(t);
          }
      }
    } else {
#pragma unroll
      for (int j = 0; j < 32; ++j) v[j] *= 1.f / kScale;
      const long long o = static_cast<long long>(row) * p.N + n0;
      if (p.dtype == 2) {
        float* w = static_cast<float*>(p.out[b]) + o;
        if (full && (reinterpret_cast<uintptr_t>(w) & 15u) == 0) {
#pragma unroll
          for (int q = 0; q < 8; ++q)
            *reinterpret_cast<float4*>(w + 4 * q) = make_float4(v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3]);
        } else {
#pragma unroll
          for (int j = 0; j < 32; ++j)
            if (j < left) w[j] = v[j];
        }
      } else {
        uint32_t pk[16];
#pragma unroll
        for (int q = 0; q < 16; ++q) {
          if (p.dtype == 0) {
            pk[q] = pack_bf16x2(v[2 * q], v[2 * q + 1]);
          } else {
            const __half2 h = __floats2half2_rn(v[2 * q], v[2 * q + 1]);
            pk[q] = *reinterpret_cast<const uint32_t*>(&h);
          }
        }
        uint16_t* w = static_cast<uint16_t*>(p.out[b]) + o;
        if (full && (reinterpret_cast<uintptr_t>(w) & 15u) == 0) {
#pragma unroll
          for (int q = 0; q < 4; ++q)
            *reinterpret_cast<uint4*>(w + 8 * q) = make_uint4(pk[4 * q], pk[4 * q + 1], pk[4 * q + 2], pk[4 * q + 3]);
        } else {
#pragma unroll
          for (int j = 0; j < 32; ++j)
            if (j < left) w[j] = static_cast<uint16_t>(j & 1 ? pk[j / 2] >> 16 : pk[j / 2]);
        }
      }
    }
    return;
  } else {
    __align__(16) __half h[32];
    __align__(16) __half l[32];
#pragma unroll
    for (int j = 0; j < 32; ++j) split_half(v[j], h[j], l[j]);
    const bool below = !SYM || n0 + 31 <= row0;  // warp-uniform: no column above the diagonal
#pragma unroll
    for (int w = 0; w < (SPLIT || MODE == kNext ? 2 : 1); ++w) {
      __half* d = p.d[w] + b * p.batch_d;
      const __half* x = w == 0 ? h : l;
      __half* dst = d + row * p.ldd + n0;
      if (below && full) {
#pragma unroll
        for (int q = 0; q < 4; ++q) *reinterpret_cast<uint4*>(dst + 8 * q) = *reinterpret_cast<const uint4*>(x + 8 * q);
      } else {
#pragma unroll
        for (int j = 0; j < 32; ++j)
          if (j < left && (!SYM || n0 + j <= row)) dst[j] = x[j];
      }
      if (SYM) {  // the mirrored half: 32 lanes write 32 neighbours of a row
        __half* t = d + static_cast<long long>(n0) * p.ldd + row;
#pragma unroll
        for (int j = 0; j < 32; ++j)
          if (j < left && (below || n0 + j < row)) t[j * p.ldd] = x[j];
      }
    }
  }
}

template <int CG, bool SPLIT, bool A_MN, bool B_MN, int MODE>
__global__ void __launch_bounds__(kGemmThreads, 1)
    product_kernel(const __grid_constant__ CUtensorMap ah, const __grid_constant__ CUtensorMap al,
                   const __grid_constant__ CUtensorMap bh, const __grid_constant__ CUtensorMap bl,
                   const __grid_constant__ GemmParams p) {
  constexpr bool SYM = MODE == kGram || MODE == kPoly;
  constexpr int BN = BM * CG;  // tile columns (and rows of the pair's tile)
  constexpr int kTmemCols = 2 * BN;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sA = smem;
  uint8_t* sB = smem + kStages * kOperand;
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + 2 * kStages * kOperand);
  uint64_t* full_bar = bars;
  uint64_t* empty_bar = bars + kStages;
  uint64_t* tfull_bar = bars + 2 * kStages;
  uint64_t* tempty_bar = bars + 2 * kStages + 2;
  uint64_t* drain_bar = bars + 2 * kStages + 4;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 2 * kStages + 5);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(bars + 2 * kStages + 6);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t crank = CG == 2 ? cluster_ctarank() : 0u;
  const bool leader = crank == 0;
  const int first = CG == 2 ? static_cast<int>(blockIdx.x >> 1) : static_cast<int>(blockIdx.x);
  const int stride = CG == 2 ? static_cast<int>(gridDim.x >> 1) : static_cast<int>(gridDim.x);

  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; ++s) {
      mbar_init(&full_bar[s], 1);
      mbar_init(&empty_bar[s], 1);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(&tfull_bar[a], 1);
      mbar_init(&tempty_bar[a], CG * kEpiWarps);
    }
    mbar_init(drain_bar, 1);
    *abort_flag = 0;
    fence_mbar_init();
    tma_prefetch_desc(&ah);
    tma_prefetch_desc(&bh);
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
  if constexpr (CG == 2) cluster_sync();  // the peer's barriers exist before anything arrives on them
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  pdl_trigger();
  pdl_wait();

  const int blocks = p.k_blocks * (SPLIT ? 3 : 1);
  const int run = SPLIT ? kSplitRun : blocks;  // blocks that one accumulator adds up
  if (warp == 0 && lane == 0) {
    // ---------------------------------------------------------- producer
    int stage = 0;
    uint32_t phase = 0;
    int armed[kStages];
    for (int s = 0; s < kStages; ++s) armed[s] = -1;
    bool ok = true;
    for (int u = first; u < p.units && ok; u += stride) {
      int b, tm, tn;
      decode<SYM>(p, u, b, tm, tn);
      const int row = tm * (CG * BM) + static_cast<int>(crank) * BM;
      const int col = tn * BN + static_cast<int>(crank) * BM;
      for (int i = 0; i < blocks; ++i) {
        // high x high, high x low, low x high
        const int which = i / p.k_blocks, k = (i - which * p.k_blocks) * BK;
        const CUtensorMap* ta = which == 2 ? &al : &ah;
        const CUtensorMap* tb = which == 1 ? &bl : &bh;
        if (!mbar_wait(&empty_bar[stage], phase ^ 1u, p.status, 420, abort_flag)) {
          ok = false;
          break;
        }
        uint32_t bar = smem_u32(&full_bar[stage]);
        if constexpr (CG == 2) bar = map_to_cta(bar, 0);
        if (leader) mbar_arrive_expect_tx(&full_bar[stage], CG * 2 * kOperand);
        armed[stage] = static_cast<int>(phase);
        uint8_t* da = sA + stage * kOperand;
        uint8_t* db = sB + stage * kOperand;
        if (A_MN) {
          load_tile<CG>(ta, bar, da, row, k, b);
          load_tile<CG>(ta, bar, da + kOperand / 2, row + 64, k, b);
        } else {
          load_tile<CG>(ta, bar, da, k, row, b);
        }
        if (B_MN) {
          load_tile<CG>(tb, bar, db, col, k, b);
          load_tile<CG>(tb, bar, db + kOperand / 2, col + 64, k, b);
        } else {
          load_tile<CG>(tb, bar, db, k, col, b);
        }
        if (++stage == kStages) {
          stage = 0;
          phase ^= 1u;
        }
      }
    }
    // No copy into this pair's shared memory may be in flight at exit (the follower's are counted
    // on the leader's barriers, which the leader's MMA has consumed before the last cluster barrier).
    if (leader)
      for (int s = 0; s < kStages; ++s)
        if (armed[s] >= 0) mbar_wait(&full_bar[s], static_cast<uint32_t>(armed[s]), p.status, 421, nullptr);
  } else if (warp == 1 && leader) {
    // ---------------------------------------------------------- MMA issuer
    constexpr uint32_t idesc = idesc_f16(CG * BM, BN, A_MN, B_MN);
    constexpr uint32_t kHalfTile = kOperand / 2;  // 64 MN-elements of 64 K-rows
    const uint64_t a_base = sdesc_sw128(smem_u32(sA), A_MN ? kHalfTile : 16, 1024);
    const uint64_t b_base = sdesc_sw128(smem_u32(sB), B_MN ? kHalfTile : 16, 1024);
    int stage = 0, acc = 0;
    uint32_t phase = 0, acc_phase = 0;
    bool ok = true;
    for (int u = first; u < p.units && ok; u += stride) {
      for (int i0 = 0; i0 < blocks; i0 += run) {
        if (!mbar_wait(&tempty_bar[acc], acc_phase ^ 1u, p.status, 422, abort_flag)) {
          ok = false;
          break;
        }
        tc_fence_after();
        const uint32_t d_tmem = tmem_base + static_cast<uint32_t>(acc * BN);
        const int i1 = min(blocks, i0 + run);
        for (int i = i0; i < i1; ++i) {
          if (!mbar_wait(&full_bar[stage], phase, p.status, 423, abort_flag)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint64_t a_st = a_base + static_cast<uint32_t>(stage * kOperand >> 4);
          const uint64_t b_st = b_base + static_cast<uint32_t>(stage * kOperand >> 4);
#pragma unroll
          for (int k = 0; k < BK / 16; ++k)
            mma<CG>(d_tmem, a_st + (A_MN ? k * (2048 >> 4) : k * (32 >> 4)), b_st + (B_MN ? k * (2048 >> 4) : k * (32 >> 4)),
                    idesc, (i > i0 || k > 0) ? 1u : 0u);
          commit_all<CG>(&empty_bar[stage]);
          if (++stage == kStages) {
            stage = 0;
            phase ^= 1u;
          }
        }
        if (!ok) break;
        commit_all<CG>(&tfull_bar[acc]);
        if (++acc == 2) {
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
    uint32_t tempty[2] = {smem_u32(&tempty_bar[0]), smem_u32(&tempty_bar[1])};
    if constexpr (CG == 2) {
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
      if (++acc == 2) {
        acc = 0;
        acc_phase ^= 1u;
      }
    };
    bool ok = true;
    for (int u = first; u < p.units && ok; u += stride) {
      int b, tm, tn;
      decode<SYM>(p, u, b, tm, tn);
      const int row0 = tm * (CG * BM) + static_cast<int>(crank) * BM + quarter * 32;
      auto t_row = [&]() {
        return tmem_base + (static_cast<uint32_t>(quarter * 32) << 16) + static_cast<uint32_t>(acc * BN);
      };
      float sum[SPLIT ? kChunks * 32 : 1];
      if constexpr (SPLIT) {
#pragma unroll
        for (int j = 0; j < kChunks * 32; ++j) sum[j] = 0.f;
        for (int i0 = 0; i0 < blocks; i0 += run) {
          if (!mbar_wait(&tfull_bar[acc], acc_phase, p.status, 425, abort_flag)) {
            ok = false;
            break;
          }
          tc_fence_after();
#pragma unroll
          for (int c = 0; c < kChunks; ++c) {
            uint32_t r[32];
            tmem_ld_32x32b_x32(t_row() + (half * kChunks + c) * 32, r);
            tmem_ld_wait();
#pragma unroll
            for (int j = 0; j < 32; ++j) sum[c * 32 + j] += __uint_as_float(r[j]);
          }
          release();
        }
        if (!ok) break;
      } else {
        if (!mbar_wait(&tfull_bar[acc], acc_phase, p.status, 425, abort_flag)) break;
        tc_fence_after();
      }
#pragma unroll(SPLIT ? kChunks : 1)
      for (int c = 0; c < kChunks; ++c) {
        const int n0 = tn * BN + (half * kChunks + c) * 32;
        if (n0 >= p.N || row0 >= p.M) break;  // warp-uniform
        epilogue_chunk<MODE, SPLIT>(p, b, row0, lane, n0, SPLIT ? 0u : t_row() + (half * kChunks + c) * 32,
                                    SPLIT ? sum + c * 32 : nullptr);
        __syncwarp();
      }
      if constexpr (!SPLIT) release();
    }
  }
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

// A stack of fp16 matrices and its two tensor maps: 64 columns x 128 rows (K-major operand) and
// 64 columns x 64 rows (MN-major).  Columns past the matrix read as zero.
struct Stack {
  __half* data;
  int rows, cols, ld;
  long long batch;
  CUtensorMap k_major, mn_major;
  bool make(__half* ptr, int r, int c, int count) {
    data = ptr;
    rows = r, cols = c, ld = (c + 7) / 8 * 8;
    batch = static_cast<long long>(rows) * ld;
    return encode(&k_major, count, 128) && encode(&mn_major, count, 64);
  }
  bool encode(CUtensorMap* map, int count, cuuint32_t box_rows) {
    cuuint64_t dims[3] = {static_cast<cuuint64_t>(cols), static_cast<cuuint64_t>(rows), static_cast<cuuint64_t>(count)};
    cuuint64_t strides[2] = {static_cast<cuuint64_t>(ld) * 2, static_cast<cuuint64_t>(batch) * 2};
    cuuint32_t box[3] = {64, box_rows, 1};
    cuuint32_t estr[3] = {1, 1, 1};
    return g_encode_muon(map, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, data, dims, strides, box, estr,
                         CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                         CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
  }
};

int sms() {
  static int n = 0;
  if (n == 0) {
    int dev = 0;
    cudaGetDevice(&dev);
    cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev);
  }
  return n;
}

template <int CG, bool SPLIT, bool A_MN, bool B_MN, int MODE>
cudaError_t launch_product(const Stack* const (&a)[2], const Stack* const (&b)[2], GemmParams& p, int count,
                           cudaStream_t stream) {
  constexpr bool SYM = MODE == kGram || MODE == kPoly;
  constexpr int tile = BM * CG;
  p.tiles_m = (p.M + tile - 1) / tile;
  p.tiles_n = (p.N + tile - 1) / tile;
  p.per_batch = SYM ? p.tiles_m * (p.tiles_m + 1) / 2 : p.tiles_m * p.tiles_n;
  p.units = p.per_batch * count;
  p.k_blocks = (p.K + BK - 1) / BK;
  auto kern = product_kernel<CG, SPLIT, A_MN, B_MN, MODE>;
  static int done[64] = {0};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev >= 64 || !done[dev]) {
    const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemBytes);
    if (e != cudaSuccess) return e;
    if (dev < 64) done[dev] = 1;
  }
  const int slots = sms() / CG;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(CG * (p.units < slots ? p.units : slots)));
  cfg.blockDim = dim3(kGemmThreads);
  cfg.dynamicSmemBytes = kSmemBytes;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  cfg.attrs = attr;
  cfg.numAttrs = 0;
  if (CG == 2) {
    attr[cfg.numAttrs].id = cudaLaunchAttributeClusterDimension;
    attr[cfg.numAttrs].val.clusterDim.x = 2;
    attr[cfg.numAttrs].val.clusterDim.y = 1;
    attr[cfg.numAttrs].val.clusterDim.z = 1;
    ++cfg.numAttrs;
  }
  if (pdl_enabled()) {
    attr[cfg.numAttrs].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[cfg.numAttrs].val.programmaticStreamSerializationAllowed = 1;
    ++cfg.numAttrs;
  }
  auto map = [](const Stack* s, bool mn) -> const CUtensorMap& { return mn ? s->mn_major : s->k_major; };
  return cudaLaunchKernelEx(&cfg, kern, map(a[0], A_MN), map(a[1], A_MN), map(b[0], B_MN), map(b[1], B_MN), p);
}

template <bool A_MN, bool B_MN, int MODE>
cudaError_t product(int tile, bool split, const Stack* const (&a)[2], const Stack* const (&b)[2], GemmParams& p, int count,
                    cudaStream_t s) {
  if (split) return launch_product<1, true, A_MN, B_MN, MODE>(a, b, p, count, s);
  return tile == 2 ? launch_product<2, false, A_MN, B_MN, MODE>(a, b, p, count, s)
                   : launch_product<1, false, A_MN, B_MN, MODE>(a, b, p, count, s);
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
  const dim3 grid(chunks, p.count), block(kThreads);
  cudaError_t e = launch_pdl(norm_kernel<T, STEP>, grid, block, 0, s, p, partial);
  if (e != cudaSuccess) return e;
  return launch_pdl(convert_kernel<T, STEP>, grid, block, 0, s, p, static_cast<const float*>(partial),
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
  Stack x[2][2], a[2], f[2];
  bool ok = true;
  for (int i = 0; i < 2; ++i)
    for (int w = 0; w < 2; ++w)
      ok = ok && x[i][w].make(reinterpret_cast<__half*>(ws + l.x[i][w]), p.rows, p.cols, p.count);
  for (int w = 0; w <= static_cast<int>(split); ++w)
    ok = ok && a[w].make(reinterpret_cast<__half*>(ws + l.a[w]), small, small, p.count) &&
         f[w].make(reinterpret_cast<__half*>(ws + l.f[w]), small, small, p.count);
  if (!ok) return -8;

  cudaError_t e = p.step           ? prepare<float, true>(p, l, static_cast<int>(chunks), stream)
                  : p.dtype == 0   ? prepare<__nv_bfloat16, false>(p, l, static_cast<int>(chunks), stream)
                  : p.dtype == 1   ? prepare<__half, false>(p, l, static_cast<int>(chunks), stream)
                                   : prepare<float, false>(p, l, static_cast<int>(chunks), stream);
  if (e != cudaSuccess) return static_cast<int>(e);

  // Pairs of SMs where their larger tiles still occupy most of the SMs.
  const auto tiles = [](long long n, int t) { return (n + t - 1) / t; };
  const long long sym = tiles(small, 256) * (tiles(small, 256) + 1) / 2 * p.count;
  const long long all = tiles(p.rows, 256) * tiles(p.cols, 256) * p.count;
  const int tile_sym = p.tile ? p.tile : (sym >= sms() / 4 ? 2 : 1);
  const int tile_all = p.tile ? p.tile : (all >= sms() / 4 ? 2 : 1);

  GemmParams g{};
  g.status = p.status;
  g.dtype = p.dtype, g.step = p.step;
  g.decay = p.decay, g.rate = p.rate, g.lr = p.lr, g.skip = p.skip;
  for (int i = 0; i < p.count; ++i) g.out[i] = p.out[i], g.shadow[i] = p.step ? p.shadow[i] : nullptr;
  const float per = 1.f / kScale;
  const Stack* as[2] = {&a[0], split ? &a[1] : &a[0]};
  const Stack* fs[2] = {&f[0], split ? &f[1] : &f[0]};
  auto put = [](const Stack& hi, const Stack* lo, __half* (&d)[2], long long& ld, long long& batch) {
    d[0] = hi.data, d[1] = lo != nullptr ? lo->data : nullptr, ld = hi.ld, batch = hi.batch;
  };
  auto from = [](const Stack& hi, const Stack* lo, const __half* (&c)[2], long long& ld, long long& batch) {
    c[0] = hi.data, c[1] = lo != nullptr ? lo->data : nullptr, ld = hi.ld, batch = hi.batch;
  };
  for (int it = 0; it < p.iterations && e == cudaSuccess; ++it) {
    const bool last = it + 1 == p.iterations;
    const Stack* xs[2] = {&x[it & 1][0], &x[it & 1][1]};
    // A = X X^T (X^T X)
    g.M = g.N = small, g.K = tall ? p.rows : p.cols;
    g.alpha = per, g.beta = 0.f;
    put(a[0], split ? &a[1] : nullptr, g.d, g.ldd, g.batch_d);
    e = tall ? product<true, true, kGram>(tile_sym, split, xs, xs, g, p.count, stream)
             : product<false, false, kGram>(tile_sym, split, xs, xs, g, p.count, stream);
    if (e != cudaSuccess) break;
    // B = b A + c A A
    g.K = small;
    g.alpha = p.c * per, g.beta = p.b;
    from(a[0], split ? &a[1] : nullptr, g.c, g.ldc, g.batch_c);
    put(f[0], split ? &f[1] : nullptr, g.d, g.ldd, g.batch_d);
    e = product<false, false, kPoly>(tile_sym, split, as, as, g, p.count, stream);
    if (e != cudaSuccess) break;
    // X <- a X + B X (X B)
    g.M = p.rows, g.N = p.cols;
    g.alpha = per, g.beta = p.a;
    from(*xs[0], xs[1], g.c, g.ldc, g.batch_c);
    put(x[~it & 1][0], &x[~it & 1][1], g.d, g.ldd, g.batch_d);
    if (last)
      e = tall ? product<false, false, kLast>(tile_all, split, xs, fs, g, p.count, stream)
               : product<false, true, kLast>(tile_all, split, fs, xs, g, p.count, stream);
    else
      e = tall ? product<false, false, kNext>(tile_all, split, xs, fs, g, p.count, stream)
               : product<false, true, kNext>(tile_all, split, fs, xs, g, p.count, stream);
  }
  return static_cast<int>(e);
}
