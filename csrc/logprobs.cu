// Log probabilities of given tokens, with entropy and the best alternatives,
// and their gradient, over rows of logits z:
//
//   log p_j = (z_j - m) / T - log S,   S = sum_j exp((z_j - m) / T),   m = max_j z_j
//   H       = log S - (1 / S) sum_j exp((z_j - m) / T) (z_j - m) / T
//   dz_j    = (sum_i g_i ([j = t_i] - p_j) - g_H p_j (log p_j + H)) / T
//
// with one g_i for the given token and one for each alternative.  The row is
// read once forward (m, S and the entropy's sum are carried together and
// rescaled when the maximum moves) and once backward, where p is recomputed
// from z, m and log S; no [rows, V] float is ever stored.
//
// A row with no logit above -inf has no distribution: log p = -inf for every
// token, H = 0, gradient 0, alternatives the lowest indices.  A NaN or +inf
// logit makes the row's numbers NaN.
//
// Alternatives are ordered by value, ties by the lower index: a 64-bit key
// (order-preserving bits of the value, ~index) makes every logit different, so the
// selection does not depend on the order in which threads meet.  Each lane keeps
// the maxima of four interleaved parts of what it reads, at one instruction per
// vector.  A lower bound for the k-th best logit comes from the lanes' maxima: each
// of the block's 4 warps puts forward its k/4 + 4 largest, and the k-th of those is
// the bound; for a warp that has a row to itself it is the k-th largest of its 128
// parts, by a bitwise search with ballots.  Only the parts that reach it, about k
// of 512, are looked at again (from L2), what is not below the bound is collected
// and ranked by counting.
//
// A row belongs to a warp, a block or a cluster of up to 8 blocks, the fewest that
// keep the SMs full.  Bound by DRAM (2 or 4 bytes a logit, read once), with the
// issue slots close behind: nine instructions a logit after pairing the fp32
// arithmetic (twelve before), two thirds of the slots.
//
// Measured (B200, copy rate 6.55 TB/s), 50257 logits a row, bf16: 8192 rows with
// entropy 138 us forward (6.0 TB/s) and 269 us backward (6.1 TB/s); 4096 rows
// without entropy 72 us (5.7 TB/s), with entropy and 20 alternatives 102 us
// (4.0 TB/s: the selection's chain of dependent steps, about 2 us a row, is only
// partly hidden by the other blocks of the SM).  fp32, 5 alternatives: 5.5 TB/s.
// One row of fp32 with 5 alternatives: 8 us, most of it the latency of a cluster's
// launch, first loads and joins.
#include <cuda_fp16.h>

#include "md_sm100.cuh"

struct MdLogprobsParams {
  const void* logits;
  long long ld;            // row stride in elements
  int dtype;               // 0 bf16, 1 fp16, 2 fp32
  int rows, vocab;
  const long long* tokens;
  long long ignore;        // rows with this token: log p = 0 and no gradient through it
  float inv_t;             // 1 / temperature
  int top;
  int want_entropy;
  float* logprob;          // [rows]
  float* entropy;          // [rows] or null
  float* top_logprob;      // [rows, top]
  long long* top_token;    // [rows, top]
  float* row_max;          // [rows] m, or null when no gradient will be asked for
  float* row_log;          // [rows] log S, or null
  // Backward: gradients of the outputs (null: none) and the result.
  const float* g_logprob;
  const float* g_entropy;
  const float* g_top;
  void* dlogits;
  long long ldd;
  md::Status* status;
};

namespace md {
namespace logprobs {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr int kMaxTop = 64;
constexpr int kWarps = 4;      // of a block, forward: many small blocks, whose tails run under each other's reads
constexpr int kThreads = 32 * kWarps;
constexpr int kBackWarps = 8;  // ... and backward, which has no tail
constexpr int kFillWarps = 64;  // warps per SM that keep DRAM busy
constexpr int kShortRow = 512;  // vectors: rows below this have a warp each when alternatives are asked for
constexpr int kParts = 4;      // interleaved parts of a lane, each with a maximum of its own
constexpr int kFound = 256;    // logits not below the bound that are collected at once (more: the bound is raised)
// exp2 of anything below is 0 in fp32; keeps 0 * log 0 at 0.
constexpr float kFloor = -200.f;

template <typename T> __device__ __forceinline__ float to_f(T v);
template <> __device__ __forceinline__ float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }
template <> __device__ __forceinline__ float to_f(__half v) { return __half2float(v); }
template <> __device__ __forceinline__ float to_f(float v) { return v; }
template <typename T> __device__ __forceinline__ T from_f(float v);
template <> __device__ __forceinline__ __nv_bfloat16 from_f(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half from_f(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ float from_f(float v) { return v; }

// Terms of sums that hold a 1 (the row's maximum), and p itself: 2 ulp, and 0 below 2^-126, are under
// what a lane's hundreds of additions at 2^-24 each may cost, and this is one instruction where the
// exact function is several, in a loop whose issue slots are two thirds full.
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Pairs of fp32 in one register pair: one instruction for two additions, products or both.
using Two = unsigned long long;
__device__ __forceinline__ Two two(float a, float b) {
  Two v;
  asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(a), "f"(b));
  return v;
}
__device__ __forceinline__ float2 both(Two v) {
  float2 f;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(f.x), "=f"(f.y) : "l"(v));
  return f;
}
__device__ __forceinline__ Two add2(Two a, Two b) {
  Two v;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(v) : "l"(a), "l"(b));
  return v;
}
__device__ __forceinline__ Two mul2(Two a, Two b) {
  Two v;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(v) : "l"(a), "l"(b));
  return v;
}
__device__ __forceinline__ Two fma2(Two a, Two b, Two c) {
  Two v;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(v) : "l"(a), "l"(b), "l"(c));
  return v;
}

template <typename T> struct Pack;  // 16 bytes of logits
template <> struct Pack<__nv_bfloat16> {
  static constexpr int N = 8;
  static constexpr int kZeros = 16;  // low bits of the fp32 value that are always zero, or not worth searching
  static __device__ __forceinline__ float max(const uint4& w) {  // NaN only where all are
    uint32_t a, b;
    asm("max.bf16x2 %0, %1, %2;" : "=r"(a) : "r"(w.x), "r"(w.y));
    asm("max.bf16x2 %0, %1, %2;" : "=r"(b) : "r"(w.z), "r"(w.w));
    asm("max.bf16x2 %0, %1, %2;" : "=r"(a) : "r"(a), "r"(b));
    return fmaxf(__uint_as_float(a << 16), __uint_as_float(a & 0xFFFF0000u));
  }
  static __device__ __forceinline__ void get(const uint4& w, float (&f)[8]) {
    const uint32_t ws[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      f[2 * q] = __uint_as_float(ws[q] << 16);
      f[2 * q + 1] = __uint_as_float(ws[q] & 0xFFFF0000u);
    }
  }
  static __device__ __forceinline__ uint4 put(const float (&f)[8]) {
    return make_uint4(pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]), pack_bf16x2(f[4], f[5]),
                      pack_bf16x2(f[6], f[7]));
  }
};
template <> struct Pack<__half> {
  static constexpr int N = 8;
  static constexpr int kZeros = 13;
  static __device__ __forceinline__ float max(const uint4& w) {
    uint32_t a, b;
    asm("max.f16x2 %0, %1, %2;" : "=r"(a) : "r"(w.x), "r"(w.y));
    asm("max.f16x2 %0, %1, %2;" : "=r"(b) : "r"(w.z), "r"(w.w));
    asm("max.f16x2 %0, %1, %2;" : "=r"(a) : "r"(a), "r"(b));
    const float2 v = __half22float2(*reinterpret_cast<const __half2*>(&a));
    return fmaxf(v.x, v.y);
  }
  static __device__ __forceinline__ void get(const uint4& w, float (&f)[8]) {
    const uint32_t ws[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const float2 v = __half22float2(*reinterpret_cast<const __half2*>(&ws[q]));
      f[2 * q] = v.x, f[2 * q + 1] = v.y;
    }
  }
  static __device__ __forceinline__ uint4 put(const float (&f)[8]) {
    uint32_t o[4];
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const __half2 h = __floats2half2_rn(f[2 * q], f[2 * q + 1]);
      o[q] = *reinterpret_cast<const uint32_t*>(&h);
    }
    return make_uint4(o[0], o[1], o[2], o[3]);
  }
};
template <> struct Pack<float> {
  static constexpr int N = 4;
  static constexpr int kZeros = 12;
  static __device__ __forceinline__ float max(const uint4& w) {
    return fmaxf(fmaxf(__uint_as_float(w.x), __uint_as_float(w.y)), fmaxf(__uint_as_float(w.z), __uint_as_float(w.w)));
  }
  static __device__ __forceinline__ void get(const uint4& w, float (&f)[4]) {
    f[0] = __uint_as_float(w.x), f[1] = __uint_as_float(w.y), f[2] = __uint_as_float(w.z), f[3] = __uint_as_float(w.w);
  }
  static __device__ __forceinline__ uint4 put(const float (&f)[4]) {
    return make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
  }
};

// Order-preserving bits of a value: NaN counts as -inf (its row has no order), -0 as +0.  0 is below
// every value.
__device__ __forceinline__ uint32_t order_of(float v) {
  if (!(v == v)) v = -INFINITY;
  const uint32_t b = __float_as_uint(v + 0.f);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
// Larger value first, then lower index: different for every logit of a row.
__device__ __forceinline__ unsigned long long key_of(uint32_t order, int index) {
  return static_cast<unsigned long long>(order) << 32 | static_cast<uint32_t>(~index);
}
__device__ __forceinline__ float key_value(unsigned long long k) {
  const uint32_t o = static_cast<uint32_t>(k >> 32);
  return __uint_as_float(o & 0x80000000u ? o & 0x7FFFFFFFu : ~o);
}
__device__ __forceinline__ int key_index(unsigned long long k) { return static_cast<int>(~static_cast<uint32_t>(k)); }

// Running maximum m, s = sum exp2((z - m) L), e = sum exp2((z - m) L) (z - m) L.
struct Stats {
  float m, s, e;
};
__device__ __forceinline__ void rescale(Stats& a, float m, float L) {  // m >= a.m
  if (a.m == m) return;
  if (a.m == -INFINITY) {  // nothing above -inf so far: its terms were all zero
    a.s = a.s != a.s ? a.s : 0.f;
    a.e = 0.f;
  } else {
    const float d = (a.m - m) * L, c = ex2(d);
    a.e = c * fmaf(fmaxf(d, kFloor), a.s, a.e);
    a.s *= c;
  }
  a.m = m;
}
__device__ __forceinline__ Stats join(Stats a, Stats b, float L) {
  const float m = fmaxf(a.m, b.m);
  rescale(a, m, L);
  rescale(b, m, L);
  a.s += b.s;
  a.e += b.e;
  return a;
}

__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
__device__ __forceinline__ uint32_t in_first(const void* smem) {  // the same place in the cluster's CTA 0
  uint32_t out;
  asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(out) : "r"(smem_u32(smem)));
  return out;
}

// The share of a row that one warp reads: `head` single logits up to the first 16-byte boundary (the
// first warp, a lane each), vectors [v0, v1), and the single logits from `tail` after the last whole
// vector (the last warp).
template <typename T>
struct Share {
  const T* row;
  const uint4* vec;
  int head, v0, v1, tail, vocab;  // head = 0 / tail = vocab where the singles are another warp's
  int base;                       // index of vector 0's first logit
  __device__ __forceinline__ Share(const T* r, int V, int part, int parts) : row(r), vocab(V) {
    constexpr int N = Pack<T>::N;
    const int mis = static_cast<int>((reinterpret_cast<uintptr_t>(r) & 15u) / sizeof(T));
    base = mis ? min(V, N - mis) : 0;
    const int nv = (V - base) / N;
    vec = reinterpret_cast<const uint4*>(r + base);
    v0 = static_cast<int>(static_cast<long long>(nv) * part / parts);
    v1 = static_cast<int>(static_cast<long long>(nv) * (part + 1) / parts);
    head = part == 0 ? base : 0;
    tail = part == parts - 1 ? base + nv * N : V;
  }
};

struct Selection {                    // of one row in one block
  unsigned long long found[kFound];
  unsigned long long best[kMaxTop];   // in order; 0: none
  unsigned long long bound;
  int count;
};
// (Rows that have a warp each need a selection per warp.)
template <bool TOP>
struct BlockMem {
  Stats stats[kWarps];
  Stats meet_stats[8];
  uint32_t put[TOP ? kThreads : 1];
  uint8_t part[TOP ? kWarps : 1][32 * kParts];    // the parts that a warp looks at again
  unsigned long long meet[8][TOP ? kMaxTop : 1];  // of the cluster's blocks, in block 0
};

// How many keys of 8 descending lists of k are larger than `key` (the searches side by side).
__device__ __forceinline__ int larger_in(const unsigned long long (&lists)[8][kMaxTop], int n, int k, unsigned long long key) {
  int lo[8];
#pragma unroll
  for (int x = 0; x < 8; ++x) lo[x] = 0;
  for (int step = kMaxTop; step > 0; step >>= 1) {
#pragma unroll
    for (int x = 0; x < 8; ++x) {
      const int at = lo[x] + step;  // lists[x][0 .. at) all larger?
      if (x < n && at <= k && lists[x][at - 1] > key) lo[x] = at;
    }
  }
  int sum = 0;
#pragma unroll
  for (int x = 0; x < 8; ++x) sum += lo[x];
  return sum;
}

// The largest bound (to Pack<T>::kZeros bits) that `k` of the warp's parts reach; 0 if fewer hold anything.
template <typename T>
__device__ __forceinline__ uint32_t reached_by(const uint32_t (&o)[kParts], int k) {
  uint32_t bound = 0;
#pragma unroll 1
  for (int bit = 31; bit >= Pack<T>::kZeros; --bit) {
    const uint32_t c = bound | 1u << bit;
    int n = 0;
#pragma unroll
    for (int q = 0; q < kParts; ++q) n += __popc(__ballot_sync(0xFFFFFFFFu, o[q] >= c));
    if (n >= k) bound = c;
  }
  return bound;
}

// The k best of a row (or of a block's part of one) into sel.best.  top[q]: maximum of this lane's
// part q.  Called by the warps that share it: one (SOLO) or all of the block.
template <typename T, bool SOLO, bool TOP>
__device__ __forceinline__ void select(const Share<T>& sh, const float (&top)[kParts], int k, BlockMem<TOP>& sm, Selection& sel) {
  constexpr int N = Pack<T>::N;
  constexpr int kTeam = SOLO ? 32 : kThreads;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, me = SOLO ? lane : static_cast<int>(threadIdx.x);
  auto sync = [] {
    if (SOLO) __syncwarp();
    else __syncthreads();
  };
  uint32_t o[kParts], mine = 0;
#pragma unroll
  for (int q = 0; q < kParts; ++q) {
    const bool any = sh.v0 + q * 32 + lane < sh.v1 || (q == 0 && (lane < sh.head || sh.tail + lane < sh.vocab));
    o[q] = any ? order_of(top[q]) : 0u;
    mine = max(mine, o[q]);
  }
  if (SOLO) {
    const uint32_t b = reached_by<T>(o, k);
    if (lane == 0) sel.bound = static_cast<unsigned long long>(b) << 32, sel.count = 0;
  } else {
    const int each = min(32, k / kWarps + 4), all = each * kWarps;
    for (int i = 0; i < each; ++i) {
      const uint32_t largest = __reduce_max_sync(0xFFFFFFFFu, mine);
      if (lane == __ffs(__ballot_sync(0xFFFFFFFFu, mine == largest)) - 1) mine = 0;
      if (lane == 0) sm.put[warp * each + i] = largest;
    }
    if (me == 0) sel.count = 0;
    sync();
    if (me < all) {
      const uint32_t own = sm.put[me];
      int rank = 0;
#pragma unroll 8
      for (int j = 0; j < all; ++j) rank += sm.put[j] > own || (sm.put[j] == own && j < me);
      if (rank == k - 1) sel.bound = static_cast<unsigned long long>(own) << 32;
    }
  }
  sync();
  int n;
  for (;;) {
    const unsigned long long bound = sel.bound;
    const uint32_t least = static_cast<uint32_t>(bound >> 32);
    auto offer = [&](float z, int index) {
      const unsigned long long key = key_of(order_of(z), index);
      if (key < bound) return;
      const int at = atomicAdd(&sel.count, 1);
      if (at < kFound) sel.found[at] = key;
    };
    int parts = 0;
#pragma unroll
    for (int q = 0; q < kParts; ++q) {
      const unsigned in = __ballot_sync(0xFFFFFFFFu, o[q] != 0u && o[q] >= least);
      if (in >> lane & 1u) sm.part[warp][parts + __popc(in & ((1u << lane) - 1u))] = static_cast<uint8_t>(q * 32 + lane);
      parts += __popc(in);
    }
    __syncwarp();
    // Lowest indices first, so that among equal logits those that count are found before the list is
    // full, and once it is, there is no need to go on.
    if (lane < sh.head) offer(to_f(sh.row[lane]), lane);
    const int rounds = (sh.v1 - sh.v0 + 32 * kParts - 1) / (32 * kParts);
    for (int t = lane; t < parts * rounds; t += 32) {
      if (*static_cast<volatile int*>(&sel.count) > kFound) break;
      const int round = t / parts, v = sh.v0 + round * 32 * kParts + sm.part[warp][t - round * parts];
      if (v >= sh.v1) continue;
      float f[N];
      Pack<T>::get(__ldg(sh.vec + v), f);
#pragma unroll
      for (int j = 0; j < N; ++j)
        if (order_of(f[j]) >= least) offer(f[j], sh.base + v * N + j);
    }
    if (sh.tail + lane < sh.vocab) offer(to_f(sh.row[sh.tail + lane]), sh.tail + lane);
    sync();
    n = sel.count;
    if (n <= kFound) break;
    // More than fit: the k-th of those that did is a higher bound.
    for (int i = me; i < kFound; i += kTeam) {
      const unsigned long long key = sel.found[i];
      int rank = 0;
      for (int j = 0; j < kFound; ++j) rank += sel.found[j] > key;
      if (rank == k - 1) sel.bound = key;
    }
    sync();
    if (me == 0) sel.count = 0;
    sync();
  }
  for (int i = me; i < n; i += kTeam) {
    const unsigned long long key = sel.found[i];
    int rank = 0;
#pragma unroll 4
    for (int j = 0; j < n; ++j) rank += sel.found[j] > key;
    if (rank < k) sel.best[rank] = key;
  }
  for (int i = n + me; i < k; i += kTeam) sel.best[i] = 0ull;
  sync();
}

// Blocks per SM that the registers are cut for: ten (48 registers), eight (64) for fp32 logits with
// alternatives, which at 48 spill 164 bytes in the loop (2048 x 50257, top 5: 78 us with eight, 80 with
// nine, 83 with ten; without entropy 77, 80, 90).
template <typename T, bool TOP>
constexpr int kBlocksPerSm = TOP && sizeof(T) == 4 ? 8 : 10;

// `share` warps per row (1, 2 or 4), or with ctas > 1 whole blocks of a cluster.
template <typename T, bool ENT, bool TOP>
__global__ void __launch_bounds__(kThreads, kBlocksPerSm<T, TOP>) forward_kernel(const __grid_constant__ MdLogprobsParams p, int share, int ctas) {
  constexpr int N = Pack<T>::N;
  constexpr uint32_t kFull = 0xFFFFFFFFu;
  extern __shared__ __align__(16) uint8_t smem_raw[];
  BlockMem<TOP>& sm = *reinterpret_cast<BlockMem<TOP>*>(smem_raw);
  Selection* selections = reinterpret_cast<Selection*>(smem_raw + sizeof(BlockMem<TOP>));
  if (ctas > 1) cluster_arrive();
  pdl_trigger();
  pdl_wait();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int rank = ctas > 1 ? static_cast<int>(cluster_rank()) : 0;
  const long long r = ctas > 1 ? blockIdx.x / ctas : static_cast<long long>(blockIdx.x) * (kWarps / share) + warp / share;
  const bool live = r < p.rows;
  const T* row = static_cast<const T*>(p.logits) + (live ? r : 0) * p.ld;
  const float L = p.inv_t * kLog2e;
  Stats st = {-INFINITY, 0.f, 0.f};
  if (live) {
    const Share<T> sh(row, p.vocab, rank * share + warp % share, share * ctas);
    float top[kParts];
#pragma unroll
    for (int q = 0; q < kParts; ++q) top[q] = -INFINITY;
    // This lane's sums, even and odd logits apart; shift = -m, or 0 while the maximum is still -inf
    // (every logit is then -inf or NaN, and adding 0 keeps both).
    float m = -INFINITY;
    Two s2 = two(0.f, 0.f), e2 = s2, shift = s2;
    const Two L2 = two(L, L);
    auto raise = [&](float to) {  // the maximum grows to `to`
      if (m == -INFINITY) {  // all terms so far were zero, or NaN
        e2 = two(0.f, 0.f);
      } else {
        const float d = (m - to) * L, c = ex2(d), least = fmaxf(d, kFloor);
        if (ENT) e2 = mul2(two(c, c), fma2(two(least, least), s2, e2));
        s2 = mul2(two(c, c), s2);
      }
      m = to;
      shift = two(-to, -to);
    };
    auto add = [&](Two z) {
      const Two d2 = mul2(add2(z, shift), L2);
      const float2 d = both(d2);
      const Two x = two(ex2(d.x), ex2(d.y));
      s2 = add2(s2, x);
      if (ENT) e2 = fma2(x, two(fmaxf(d.x, kFloor), fmaxf(d.y, kFloor)), e2);
    };
    auto single = [&](int j) {
      const float z = to_f(row[j]);
      if (TOP) top[0] = fmaxf(top[0], z);
      if (z > m) raise(z);
      add(two(z, -INFINITY));
    };
    if (lane < sh.head) single(lane);
    // Four vectors at a time, their maximum first: a warp steps aside for a new maximum whenever one
    // of its lanes has one, which in a short share is nearly every time it looks.
    auto vectors = [&](const uint4 (&w)[kParts], int n) {
      float mx[kParts], all = m;
#pragma unroll
      for (int q = 0; q < kParts; ++q) {
        if (q >= n) break;
        mx[q] = Pack<T>::max(w[q]);
        if (TOP) top[q] = fmaxf(top[q], mx[q]);
        all = fmaxf(all, mx[q]);
      }
      if (all > m) raise(all);
#pragma unroll
      for (int q = 0; q < kParts; ++q) {
        if (q >= n) break;
        float f[N];
        Pack<T>::get(w[q], f);
#pragma unroll
        for (int j = 0; j < N; j += 2) add(two(f[j], f[j + 1]));
      }
    };
    uint4 w[kParts];
    int v = sh.v0 + lane;
    for (; v + (kParts - 1) * 32 < sh.v1; v += kParts * 32) {
#pragma unroll
      for (int q = 0; q < kParts; ++q) w[q] = __ldg(sh.vec + v + q * 32);
      vectors(w, kParts);
    }
    const int rest = (sh.v1 - v + 31) / 32;  // (0 or less: none)
    if (rest > 0) {
#pragma unroll
      for (int q = 0; q < kParts; ++q)
        if (q < rest) w[q] = __ldg(sh.vec + v + q * 32);
      vectors(w, rest);
    }
    if (sh.tail + lane < sh.vocab) single(sh.tail + lane);
    st = {m, both(s2).x + both(s2).y, both(e2).x + both(e2).y};

    __syncwarp();
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      Stats b;
      b.m = __shfl_xor_sync(kFull, st.m, o);
      b.s = __shfl_xor_sync(kFull, st.s, o);
      b.e = ENT ? __shfl_xor_sync(kFull, st.e, o) : 0.f;
      st = join(st, b, L);
    }
    // (A block that shares a row with alternatives has no other row: all its warps are here.)
    if (TOP && share == 1) select<T, true>(sh, top, p.top, sm, selections[warp]);
    if (TOP && share == kWarps) select<T, false>(sh, top, p.top, sm, selections[0]);
  }

  // ---- the warps of a row, then the blocks of a cluster
  const int k = TOP ? p.top : 0;
  int threads = 32, me = lane;  // that finish the row
  if (share > 1) {
    if (lane == 0) sm.stats[warp] = st;
    __syncthreads();
    const int w0 = warp / share * share;
    st = sm.stats[w0];
    for (int w = 1; w < share; ++w) st = join(st, sm.stats[w0 + w], L);
    threads = 32 * share, me = tid - w0 * 32;
  }
  const unsigned long long* best = selections[share == 1 ? warp : 0].best;
  if (ctas > 1) {
    cluster_wait();  // every block of the cluster runs: its shared memory can be written
    if (tid == 0) {
      const uint32_t d = in_first(&sm.meet_stats[rank]);
      asm volatile("st.shared::cluster.f32 [%0], %1;\n\tst.shared::cluster.f32 [%0+4], %2;\n\t"
                   "st.shared::cluster.f32 [%0+8], %3;" ::"r"(d), "f"(st.m), "f"(st.s), "f"(st.e) : "memory");
    }
    for (int i = tid; i < k; i += kThreads)
      asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(in_first(&sm.meet[rank][i])), "l"(best[i]) : "memory");
    __syncwarp();
    cluster_arrive();
    cluster_wait();
    if (rank != 0) return;
    st = sm.meet_stats[0];
    for (int c = 1; c < ctas; ++c) st = join(st, sm.meet_stats[c], L);
    if constexpr (TOP) {
      // Merge of sorted lists: a key's place is how many are larger.
      for (int i = tid; i < ctas * k; i += kThreads) {
        const unsigned long long key = sm.meet[i / k][i % k];
        const int place = larger_in(sm.meet, ctas, k, key);
        if (key != 0ull && place < k) selections[0].best[place] = key;
      }
      __syncthreads();
    }
  }
  if (!live) return;

  // ---- the row's results
  const bool empty = st.m == -INFINITY && st.s == 0.f;
  const float log_s = logf(st.s);
  auto logp = [&](float z) { return empty ? -INFINITY : (z - st.m) * p.inv_t - log_s; };
  if (me == 0) {
    const long long t = p.tokens[r];
    float lp = 0.f;
    if (t != p.ignore) {
      if (t >= 0 && t < p.vocab) {
        lp = logp(to_f(row[t]));
      } else {
        report(p.status, kBadArgument, 410, static_cast<uint32_t>(t));
        lp = __int_as_float(0x7fffffff);
      }
    }
    p.logprob[r] = lp;
    if (ENT) p.entropy[r] = empty ? 0.f : log_s - st.e / st.s * kLn2;
    if (p.row_max != nullptr) {
      p.row_max[r] = st.m;
      p.row_log[r] = log_s;
    }
  }
  for (int i = me; i < k; i += threads) {
    p.top_logprob[r * k + i] = logp(key_value(best[i]));
    p.top_token[r * k + i] = key_index(best[i]);
  }
}

// dz, `share` warps per row (a power of two), or `slices` whole blocks.
template <typename T, bool ENT>
__global__ void __launch_bounds__(32 * kBackWarps) backward_kernel(const __grid_constant__ MdLogprobsParams p, int share, int slices) {
  constexpr int N = Pack<T>::N;
  constexpr int kAhead = 2;
  pdl_trigger();
  pdl_wait();
  const int warp = threadIdx.x >> 5, threads = 32 * share, me = static_cast<int>(threadIdx.x) & (threads - 1);
  const long long r = slices > 1 ? blockIdx.x / slices : static_cast<long long>(blockIdx.x) * (kBackWarps / share) + warp / share;
  const int slice = slices > 1 ? static_cast<int>(blockIdx.x % slices) : 0;
  const bool live = r < p.rows;
  const T* z = static_cast<const T*>(p.logits) + (live ? r : 0) * p.ld;
  T* dz = static_cast<T*>(p.dlogits) + (live ? r : 0) * p.ldd;
  const float L = p.inv_t * kLog2e;
  const float m = live ? p.row_max[r] : 0.f, log_s = live ? p.row_log[r] : 0.f;
  const bool empty = m == -INFINITY && log_s == -INFINITY;
  const long long t = live ? p.tokens[r] : p.ignore;
  const bool scored = t != p.ignore;
  const float g = scored && p.g_logprob != nullptr ? p.g_logprob[r] : 0.f;
  const int k = live && p.g_top != nullptr ? p.top : 0;
  float all = g;
  for (int i = 0; i < k; ++i) all += p.g_top[r * k + i];
  // dz_j = -p_j (A + B log2 p_j) + ..., A = (all + g_H H) / T, B = g_H ln 2 / T
  const float gh = ENT && live ? p.g_entropy[r] : 0.f;
  const float A = (ENT && live ? fmaf(gh, p.entropy[r], all) : all) * p.inv_t;
  const float B = gh * kLn2 * p.inv_t;
  const float shift = log_s * kLog2e;
  auto smooth = [&](float f) {  // the part of dz that every logit has
    const float d = fmaf(f - m, L, -shift);
    const float x = ex2(d);
    return -x * (ENT ? fmaf(B, fmaxf(d, kFloor), A) : A);
  };

  const Share<T> sh(z, p.vocab, slice, slices);
  if (live && empty) {
    for (int j = sh.base + sh.v0 * N + me; j < sh.base + sh.v1 * N; j += threads) dz[j] = from_f<T>(0.f);
    if (me < sh.head) dz[me] = from_f<T>(0.f);
    if (sh.tail + me < p.vocab) dz[sh.tail + me] = from_f<T>(0.f);
  } else if (live) {
    uint4* dv = reinterpret_cast<uint4*>(dz + sh.base);
    auto vector = [&](const uint4& w, int v) {
      float f[N];
      Pack<T>::get(w, f);
#pragma unroll
      for (int j = 0; j < N; ++j) f[j] = smooth(f[j]);
      dv[v] = Pack<T>::put(f);
    };
    int v = sh.v0 + me;
    for (; v + (kAhead - 1) * threads < sh.v1; v += kAhead * threads) {
      uint4 w[kAhead];
#pragma unroll
      for (int i = 0; i < kAhead; ++i) w[i] = __ldg(sh.vec + v + i * threads);
#pragma unroll
      for (int i = 0; i < kAhead; ++i) vector(w[i], v + i * threads);
    }
    for (; v < sh.v1; v += threads) vector(__ldg(sh.vec + v), v);
    if (me < sh.head) dz[me] = from_f<T>(smooth(to_f(z[me])));
    if (sh.tail + me < p.vocab) dz[sh.tail + me] = from_f<T>(smooth(to_f(z[sh.tail + me])));
  }
  // The logits that a gradient names: written again, with every term that names them, by the block
  // that wrote them (an index named twice gets the same value twice).
  __syncthreads();
  if (!live || empty) return;
  const int lo = slice == 0 ? 0 : sh.base + sh.v0 * N, hi = slice == slices - 1 ? p.vocab : sh.base + sh.v1 * N;
  for (int i = me; i <= k; i += threads) {
    const long long j = i < k ? p.top_token[r * k + i] : (scored ? t : -1);
    if (j < lo || j >= hi) continue;
    float named = j == t ? g : 0.f;
    for (int q = 0; q < k; ++q) named += p.top_token[r * k + q] == j ? p.g_top[r * k + q] : 0.f;
    dz[j] = from_f<T>(fmaf(named, p.inv_t, smooth(to_f(z[j]))));
  }
}

// Warps per row (a power of two up to the block's) and, of whole blocks, blocks per row: more than one
// while there are fewer than `fill` and every lane keeps a few vectors.
struct Split {
  int share, ctas;
  unsigned blocks;
};
Split split_rows(int rows, int nv, int share, int warps, int most_ctas, int fill) {
  Split s{share, 1, 0};
  if (share == warps)
    while (s.ctas < most_ctas && static_cast<long long>(rows) * s.ctas < fill && nv / (64 * warps * s.ctas) >= 2) s.ctas *= 2;
  s.blocks = s.ctas > 1 ? static_cast<unsigned>(rows) * s.ctas
                        : static_cast<unsigned>((static_cast<long long>(rows) * share + warps - 1) / warps);
  return s;
}

template <typename T, bool ENT, bool TOP>
cudaError_t launch_forward(const MdLogprobsParams& p, cudaStream_t stream) {
  const int nv = p.vocab / Pack<T>::N;
  // Sums alone: the fewest warps per row that keep the SMs full (a warp's joins and tail cost less
  // the longer its share; 8192 rows of 50257 bf16: 147 us with one warp each, 138 with two, as here,
  // 142 with four; 6000 rows 127, 111, 108; 8192 rows of 8192 29, 31, 40).  With
  // alternatives a block, whose selection runs under the reads of the others on its SM, or a warp for
  // rows too short for that (2000 rows of 8192, top 32: 23 us with blocks, 26 us with warps; 8192
  // rows of 1000, top 5: 19 us with warps, 51 us with blocks).
  int share = 1;
  if (TOP) share = nv >= kShortRow ? kWarps : 1;
  else while (share < kWarps && static_cast<long long>(p.rows) * share < 148 * kFillWarps && nv / (2 * share) >= 64) share *= 2;
  const Split s = split_rows(p.rows, nv, share, kWarps, 8, 148);
  auto kern = forward_kernel<T, ENT, TOP>;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(s.blocks);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = sizeof(BlockMem<TOP>) + (TOP ? (share == 1 ? kWarps : 1) * sizeof(Selection) : 0);
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  cfg.attrs = attr;
  cfg.numAttrs = 0;
  if (s.ctas > 1) {
    attr[cfg.numAttrs].id = cudaLaunchAttributeClusterDimension;
    attr[cfg.numAttrs].val.clusterDim.x = s.ctas;
    attr[cfg.numAttrs].val.clusterDim.y = 1;
    attr[cfg.numAttrs].val.clusterDim.z = 1;
    ++cfg.numAttrs;
  }
  if (pdl_enabled()) {
    attr[cfg.numAttrs].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[cfg.numAttrs].val.programmaticStreamSerializationAllowed = 1;
    ++cfg.numAttrs;
  }
  return cudaLaunchKernelEx(&cfg, kern, p, s.share, s.ctas);
}

template <typename T>
cudaError_t forward(const MdLogprobsParams& p, cudaStream_t s) {
  if (p.want_entropy) return p.top > 0 ? launch_forward<T, true, true>(p, s) : launch_forward<T, true, false>(p, s);
  return p.top > 0 ? launch_forward<T, false, true>(p, s) : launch_forward<T, false, false>(p, s);
}

template <typename T>
cudaError_t backward(const MdLogprobsParams& p, cudaStream_t s) {
  // The most warps per row that leave each lane several vectors.
  const int nv = p.vocab / Pack<T>::N;
  int share = 1;
  while (share < kBackWarps && nv / (32 * 2 * share) >= 4) share *= 2;
  const Split sp = split_rows(p.rows, nv, share, kBackWarps, 64, 148 * 4);
  const dim3 grid(sp.blocks), block(32 * kBackWarps);
  return p.g_entropy != nullptr ? launch_pdl(backward_kernel<T, true>, grid, block, 0, s, p, sp.share, sp.ctas)
                                : launch_pdl(backward_kernel<T, false>, grid, block, 0, s, p, sp.share, sp.ctas);
}

int check(const MdLogprobsParams& p) {
  if (p.rows < 0 || p.vocab <= 0 || p.ld < p.vocab || p.dtype < 0 || p.dtype > 2) return -2;
  if (p.rows > (1 << 27)) return -3;
  if (!(p.inv_t > 0.f) || p.top < 0 || p.top > kMaxTop || p.top > p.vocab) return -4;
  return 0;
}

}  // namespace logprobs
}  // namespace md

// 0 ok; negative: refused (nothing launched); positive: CUDA error of the launch.
extern "C" int md_logprobs(const MdLogprobsParams* prm, cudaStream_t s) {
  using namespace md::logprobs;
  if (prm == nullptr) return -1;
  const MdLogprobsParams& p = *prm;
  if (int rc = check(p)) return rc;
  if (p.rows == 0) return 0;
  if (p.logits == nullptr || p.tokens == nullptr || p.logprob == nullptr || (p.want_entropy && p.entropy == nullptr) ||
      (p.top > 0 && (p.top_logprob == nullptr || p.top_token == nullptr)) ||
      (p.row_max == nullptr) != (p.row_log == nullptr))
    return -5;
  return static_cast<int>(p.dtype == 0   ? forward<__nv_bfloat16>(p, s)
                          : p.dtype == 1 ? forward<__half>(p, s)
                                         : forward<float>(p, s));
}

extern "C" int md_logprobs_backward(const MdLogprobsParams* prm, cudaStream_t s) {
  using namespace md::logprobs;
  if (prm == nullptr) return -1;
  const MdLogprobsParams& p = *prm;
  if (int rc = check(p)) return rc;
  if (p.rows == 0) return 0;
  if (p.logits == nullptr || p.tokens == nullptr || p.dlogits == nullptr || p.ldd < p.vocab || p.row_max == nullptr ||
      p.row_log == nullptr || (p.g_entropy != nullptr && p.entropy == nullptr) ||
      (p.g_top != nullptr && (p.top <= 0 || p.top_token == nullptr)))
    return -5;
  // A vector has to start at the same distance from a 16-byte boundary in z and dz, in every row.
  const long long es = p.dtype == 2 ? 4 : 2;
  if (((reinterpret_cast<uintptr_t>(p.logits) ^ reinterpret_cast<uintptr_t>(p.dlogits)) & 15u) || (p.ld - p.ldd) * es % 16)
    return -6;
  return static_cast<int>(p.dtype == 0   ? backward<__nv_bfloat16>(p, s)
                          : p.dtype == 1 ? backward<__half>(p, s)
                                         : backward<float>(p, s));
}
