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
// (value's order-preserving bits, ~index) makes every key different, so the
// selection does not depend on the order in which threads meet.  Each of 128
// lane groups keeps the largest key it has seen (a by-product of the running
// maximum); the k-th largest of those 128 is a lower bound for the k-th best
// logit, and only the k groups above it can hold one, so the second look at
// the row reads 1/128 of it for each alternative instead of all of it.
//
// Bound by DRAM (2 or 4 bytes a logit; one exp2 each is about 3/4 of that
// time at bf16).  Few rows: a cluster of up to 8 CTAs shares a row and the
// partial results meet in the first one's shared memory.
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
constexpr int kGroups = 128;   // lane groups that keep a maximum of their own
constexpr int kKeys = 1024;    // candidates kept at once
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

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

template <typename T> struct Pack;  // 16 bytes of logits
template <> struct Pack<__nv_bfloat16> {
  static constexpr int N = 8;
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
  static __device__ __forceinline__ void get(const uint4& w, float (&f)[4]) {
    f[0] = __uint_as_float(w.x), f[1] = __uint_as_float(w.y), f[2] = __uint_as_float(w.z), f[3] = __uint_as_float(w.w);
  }
  static __device__ __forceinline__ uint4 put(const float (&f)[4]) {
    return make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
  }
};

// Order-preserving key: larger value first, then lower index.  NaN counts as
// -inf (its row has no order), -0 as +0.
__device__ __forceinline__ unsigned long long key_of(float v, int index) {
  if (!(v == v)) v = -INFINITY;
  const uint32_t b = __float_as_uint(v + 0.f);
  const uint32_t o = b & 0x80000000u ? ~b : b | 0x80000000u;
  return static_cast<unsigned long long>(o) << 32 | static_cast<uint32_t>(~index);
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

// The part of a row that one CTA of the cluster reads: `head` single logits up
// to the first 16-byte boundary (CTA 0), vectors [v0, v1), `tail` single
// logits after the last whole vector (the last CTA).
template <typename T>
struct Part {
  const T* row;
  const uint4* vec;
  int head, v0, v1, tail0, vocab;
  bool first, last;
  __device__ __forceinline__ Part(const T* r, int V, int rank, int ctas) : row(r), vocab(V) {
    constexpr int N = Pack<T>::N;
    const int mis = static_cast<int>((reinterpret_cast<uintptr_t>(r) & 15u) / sizeof(T));
    head = mis ? min(V, N - mis) : 0;
    const int nv = (V - head) / N;
    vec = reinterpret_cast<const uint4*>(r + head);
    v0 = static_cast<int>(static_cast<long long>(nv) * rank / ctas);
    v1 = static_cast<int>(static_cast<long long>(nv) * (rank + 1) / ctas);
    tail0 = head + nv * N;
    first = rank == 0;
    last = rank == ctas - 1;
  }
};

template <int THREADS, bool TOP>
struct Smem {
  unsigned long long group_key[TOP ? kGroups : 1];
  unsigned long long keys[TOP ? kKeys : 1];
  unsigned long long meet[TOP ? 8 * kMaxTop : 1];  // the cluster's best keys, in CTA 0
  Stats meet_stats[8];
  Stats warp_stats[THREADS / 32];
  unsigned long long bound;
  int owner[TOP ? kMaxTop : 1];
  int owners, count;
};

// Rank of every key of a list = how many are larger; write(i, rank) for each.
template <int THREADS, typename F>
__device__ __forceinline__ void by_rank(const unsigned long long* keys, int n, F write) {
  for (int i = threadIdx.x; i < n; i += THREADS) {
    const unsigned long long k = keys[i];
    int rank = 0;
    for (int j = 0; j < n; ++j) rank += keys[j] > k;
    write(i, rank);
  }
}

template <typename T, int THREADS, bool ENT, bool TOP>
__global__ void __launch_bounds__(THREADS) forward_kernel(const __grid_constant__ MdLogprobsParams p, int ctas) {
  constexpr int N = Pack<T>::N;
  constexpr int kWidth = THREADS / kGroups;  // lanes of a group
  constexpr int kAhead = 4;                  // vectors in flight per thread
  extern __shared__ __align__(16) uint8_t smem_raw[];
  using S = Smem<THREADS, TOP>;
  S& sm = *reinterpret_cast<S*>(smem_raw);
  if (ctas > 1) cluster_arrive();
  pdl_trigger();
  pdl_wait();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int rank = ctas > 1 ? static_cast<int>(cluster_rank()) : 0;
  const long long r = blockIdx.x / ctas;
  const Part<T> part(static_cast<const T*>(p.logits) + r * p.ld, p.vocab, rank, ctas);
  const float L = p.inv_t * kLog2e;

  // ---- one pass: maximum, sums, and the place of this thread's maximum
  Stats st = {-INFINITY, 0.f, 0.f};
  int at = -1;
  auto single = [&](int j) {
    const float z = to_f(part.row[j]);
    if (TOP && at < 0) at = j;
    if (z > st.m) {
      rescale(st, z, L);
      at = j;
    }
    const float d = st.m == -INFINITY ? (z != z ? z : -INFINITY) : (z - st.m) * L;
    const float x = ex2(d);
    st.s += x;
    if (ENT) st.e = fmaf(x, fmaxf(d, kFloor), st.e);
  };
  if (part.first && tid < part.head) single(tid);
  auto vector = [&](const uint4& w, int v) {
    float f[N];
    Pack<T>::get(w, f);
    float mx = f[0];
#pragma unroll
    for (int j = 1; j < N; ++j) mx = fmaxf(mx, f[j]);
    if (TOP && at < 0) at = part.head + v * N;
    if (mx > st.m) {
      rescale(st, mx, L);
      if (TOP) {
        int o = N - 1;
#pragma unroll
        for (int j = N - 2; j >= 0; --j) o = f[j] == mx ? j : o;
        at = part.head + v * N + o;
      }
    }
    // (While the maximum is still -inf every logit is -inf or NaN: subtracting 0 keeps both.)
    const float m = st.m == -INFINITY ? 0.f : st.m;
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const float d = (f[j] - m) * L;
      const float x = ex2(d);
      st.s += x;
      if (ENT) st.e = fmaf(x, fmaxf(d, kFloor), st.e);
    }
  };
  int v = part.v0 + tid;
  for (; v + (kAhead - 1) * THREADS < part.v1; v += kAhead * THREADS) {
    uint4 w[kAhead];
#pragma unroll
    for (int i = 0; i < kAhead; ++i) w[i] = __ldg(part.vec + v + i * THREADS);
#pragma unroll
    for (int i = 0; i < kAhead; ++i) vector(w[i], v + i * THREADS);
  }
  for (; v < part.v1; v += THREADS) vector(__ldg(part.vec + v), v);
  if (part.last && part.tail0 + tid < part.vocab) single(part.tail0 + tid);

  // ---- alternatives: this thread's best key, then its group's
  unsigned long long best = TOP && at >= 0 ? key_of(st.m, at) : 0ull;

  // ---- sums of the CTA
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    Stats b;
    b.m = __shfl_xor_sync(0xFFFFFFFFu, st.m, o);
    b.s = __shfl_xor_sync(0xFFFFFFFFu, st.s, o);
    b.e = ENT ? __shfl_xor_sync(0xFFFFFFFFu, st.e, o) : 0.f;
    st = join(st, b, L);
  }
  if (lane == 0) sm.warp_stats[warp] = st;
  if (TOP) {
#pragma unroll
    for (int o = 1; o < kWidth; o <<= 1) {
      const unsigned long long other = __shfl_xor_sync(0xFFFFFFFFu, best, o);
      best = other > best ? other : best;
    }
    if (tid % kWidth == 0) sm.group_key[tid / kWidth] = best;
    if (tid == 0) {
      sm.bound = 0ull;
      sm.count = 0;
      sm.owners = 0;
    }
  }
  __syncthreads();
  if (ctas > 1) cluster_wait();  // every CTA of the cluster runs: its shared memory can be written
  if (warp == 0) {
    Stats a = lane < THREADS / 32 ? sm.warp_stats[lane] : Stats{-INFINITY, 0.f, 0.f};
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      Stats b;
      b.m = __shfl_xor_sync(0xFFFFFFFFu, a.m, o);
      b.s = __shfl_xor_sync(0xFFFFFFFFu, a.s, o);
      b.e = ENT ? __shfl_xor_sync(0xFFFFFFFFu, a.e, o) : 0.f;
      a = join(a, b, L);
    }
    if (lane == 0) {
      if (ctas == 1) sm.meet_stats[0] = a;
      else {
        const uint32_t d = in_first(&sm.meet_stats[rank]);
        asm volatile("st.shared::cluster.f32 [%0], %1;\n\tst.shared::cluster.f32 [%0+4], %2;\n\t"
                     "st.shared::cluster.f32 [%0+8], %3;" ::"r"(d), "f"(a.m), "f"(a.s), "f"(a.e) : "memory");
      }
    }
  }

  if (TOP) {
    const int k = p.top;
    {  // Rank of each group's best key (a share of the comparisons per lane of the group).
      const int g = tid / kWidth, sub = tid % kWidth;
      const unsigned long long mine = sm.group_key[g];
      int larger = 0;
#pragma unroll 8
      for (int j = sub; j < kGroups; j += kWidth) larger += sm.group_key[j] > mine;
#pragma unroll
      for (int o = 1; o < kWidth; o <<= 1) larger += __shfl_xor_sync(0xFFFFFFFFu, larger, o);
      if (sub == 0 && mine != 0ull && larger < k) {
        sm.owner[larger] = g;
        atomicAdd(&sm.owners, 1);
        if (larger == k - 1) sm.bound = mine;
      }
    }
    __syncthreads();
    // Every logit of the k best groups that is not below the bound.  If they do not all fit, the
    // k-th best of those that did is a higher bound, and the look is repeated with it.
    const int owners = sm.owners;
    int n;
    for (;;) {
      const unsigned long long bound = sm.bound;
      auto offer = [&](float z, int j) {
        const unsigned long long key = key_of(z, j);
        if (key >= bound) {
          const int c = atomicAdd(&sm.count, 1);
          if (c < kKeys) sm.keys[c] = key;
        }
      };
      for (int o = warp; o < owners; o += THREADS / 32) {
        const int g = sm.owner[o];
        // The group's vectors: kWidth neighbours out of every THREADS.
        for (int q = lane;; q += 32) {
          const int vi = part.v0 + (q / kWidth) * THREADS + g * kWidth + q % kWidth;
          if (part.v0 + (q / kWidth) * THREADS >= part.v1) break;
          if (vi < part.v1) {
            float f[N];
            Pack<T>::get(__ldg(part.vec + vi), f);
#pragma unroll
            for (int j = 0; j < N; ++j) offer(f[j], part.head + vi * N + j);
          }
        }
        const int t = g * kWidth + lane;  // ... and its single logits
        if (lane < kWidth) {
          if (part.first && t < part.head) offer(to_f(part.row[t]), t);
          if (part.last && part.tail0 + t < part.vocab) offer(to_f(part.row[part.tail0 + t]), part.tail0 + t);
        }
      }
      __syncthreads();
      n = sm.count;
      if (n <= kKeys) break;
      by_rank<THREADS>(sm.keys, kKeys, [&](int i, int rk) { if (rk == k - 1) sm.bound = sm.keys[i]; });
      __syncthreads();
      if (tid == 0) sm.count = 0;
      __syncthreads();
    }
    // This CTA's best k, in order; with a cluster they meet in CTA 0.
    by_rank<THREADS>(sm.keys, n, [&](int i, int rk) {
      if (rk < k) {
        if (ctas == 1) sm.meet[rk] = sm.keys[i];
        else {
          const uint32_t d = in_first(&sm.meet[rank * kMaxTop + rk]);
          asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(d), "l"(sm.keys[i]) : "memory");
        }
      }
    });
    for (int i = n + tid; i < k; i += THREADS) {  // fewer logits here than alternatives
      if (ctas == 1) sm.meet[i] = 0ull;
      else {
        const uint32_t d = in_first(&sm.meet[rank * kMaxTop + i]);
        asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(d), "l"(0ull) : "memory");
      }
    }
  }
  if (ctas > 1) {
    __syncwarp();
    cluster_arrive();
    cluster_wait();
    if (rank != 0) return;
  } else {
    __syncthreads();
  }

  // ---- the row's results
  Stats a = sm.meet_stats[0];
  for (int c = 1; c < ctas; ++c) a = join(a, sm.meet_stats[c], L);
  const bool empty = a.m == -INFINITY && a.s == 0.f;
  const float log_s = logf(a.s);
  auto logp = [&](float z) { return empty ? -INFINITY : (z - a.m) * p.inv_t - log_s; };
  if (tid == 0) {
    const long long t = p.tokens[r];
    float lp = 0.f;
    if (t != p.ignore) {
      if (t >= 0 && t < p.vocab) {
        lp = logp(to_f(part.row[t]));
      } else {
        report(p.status, kBadArgument, 410, static_cast<uint32_t>(t));
        lp = __int_as_float(0x7fffffff);
      }
    }
    p.logprob[r] = lp;
    if (ENT) p.entropy[r] = empty ? 0.f : log_s - a.e / a.s * kLn2;
    if (p.row_max != nullptr) {
      p.row_max[r] = a.m;
      p.row_log[r] = log_s;
    }
  }
  if (TOP) {
    const int k = p.top;
    auto put = [&](unsigned long long key, int rk) {
      p.top_logprob[r * k + rk] = logp(key_value(key));
      p.top_token[r * k + rk] = key_index(key);
    };
    if (ctas == 1) {
      for (int i = tid; i < k; i += THREADS) put(sm.meet[i], i);
    } else {
      for (int i = tid; i < ctas * k; i += THREADS) {
        const unsigned long long key = sm.meet[(i / k) * kMaxTop + i % k];
        if (key == 0ull) continue;
        int rk = 0;
        for (int c = 0; c < ctas; ++c)
          for (int j = 0; j < k; ++j) rk += sm.meet[c * kMaxTop + j] > key;
        if (rk < k) put(key, rk);
      }
    }
  }
}

// dz for a slice of a row: blockIdx.x = row * slices + slice.
template <typename T, bool ENT>
__global__ void __launch_bounds__(256) backward_kernel(const __grid_constant__ MdLogprobsParams p, int slices) {
  constexpr int N = Pack<T>::N;
  constexpr int kAhead = 2;
  pdl_trigger();
  pdl_wait();
  const int tid = threadIdx.x;
  const long long r = blockIdx.x / slices;
  const int slice = blockIdx.x % slices;
  const T* z = static_cast<const T*>(p.logits) + r * p.ld;
  T* dz = static_cast<T*>(p.dlogits) + r * p.ldd;
  const float L = p.inv_t * kLog2e;
  const float m = p.row_max[r], log_s = p.row_log[r];
  const bool empty = m == -INFINITY && log_s == -INFINITY;
  const long long t = p.tokens[r];
  const bool scored = t != p.ignore;
  const float g = scored && p.g_logprob != nullptr ? p.g_logprob[r] : 0.f;
  const int k = p.g_top != nullptr ? p.top : 0;
  float all = g;
  for (int i = 0; i < k; ++i) all += p.g_top[r * k + i];
  // dz_j = -p_j (A + B log2 p_j) + ..., A = (all + g_H H) / T, B = g_H ln 2 / T
  const float gh = ENT ? p.g_entropy[r] : 0.f;
  const float A = (ENT ? fmaf(gh, p.entropy[r], all) : all) * p.inv_t;
  const float B = gh * kLn2 * p.inv_t;
  const float shift = log_s * kLog2e;
  auto smooth = [&](float f) {  // the part of dz that every logit has
    const float d = (f - m) * L - shift;
    const float x = ex2(d);
    return -x * (ENT ? fmaf(B, fmaxf(d, kFloor), A) : A);
  };

  const int mis = static_cast<int>((reinterpret_cast<uintptr_t>(z) & 15u) / sizeof(T));
  const int head = mis ? min(p.vocab, N - mis) : 0;
  const int nv = (p.vocab - head) / N;
  const int v0 = static_cast<int>(static_cast<long long>(nv) * slice / slices);
  const int v1 = static_cast<int>(static_cast<long long>(nv) * (slice + 1) / slices);
  const int tail0 = head + nv * N;
  if (empty) {
    for (int j = head + v0 * N + tid; j < head + v1 * N; j += 256) dz[j] = from_f<T>(0.f);
    if (slice == 0 && tid < head) dz[tid] = from_f<T>(0.f);
    if (slice == slices - 1 && tail0 + tid < p.vocab) dz[tail0 + tid] = from_f<T>(0.f);
    return;
  }
  const uint4* zv = reinterpret_cast<const uint4*>(z + head);
  uint4* dv = reinterpret_cast<uint4*>(dz + head);
  auto vector = [&](const uint4& w, int v) {
    float f[N];
    Pack<T>::get(w, f);
#pragma unroll
    for (int j = 0; j < N; ++j) f[j] = smooth(f[j]);
    dv[v] = Pack<T>::put(f);
  };
  int v = v0 + tid;
  for (; v + (kAhead - 1) * 256 < v1; v += kAhead * 256) {
    uint4 w[kAhead];
#pragma unroll
    for (int i = 0; i < kAhead; ++i) w[i] = __ldg(zv + v + i * 256);
#pragma unroll
    for (int i = 0; i < kAhead; ++i) vector(w[i], v + i * 256);
  }
  for (; v < v1; v += 256) vector(__ldg(zv + v), v);
  if (slice == 0 && tid < head) dz[tid] = from_f<T>(smooth(to_f(z[tid])));
  if (slice == slices - 1 && tail0 + tid < p.vocab) dz[tail0 + tid] = from_f<T>(smooth(to_f(z[tail0 + tid])));

  // The logits that a gradient names: written again, with every term that names them, by the CTA
  // that wrote them (an index named twice gets the same value twice).
  const int lo = slice == 0 ? 0 : head + v0 * N, hi = slice == slices - 1 ? p.vocab : head + v1 * N;
  __syncthreads();
  for (int i = tid; i <= k; i += 256) {
    const long long j = i < k ? p.top_token[r * k + i] : (scored ? t : -1);
    if (j < lo || j >= hi) continue;
    float named = j == t ? g : 0.f;
    for (int q = 0; q < k; ++q) named += p.top_token[r * k + q] == j ? p.g_top[r * k + q] : 0.f;
    dz[j] = from_f<T>(fmaf(named, p.inv_t, smooth(to_f(z[j]))));
  }
}

template <typename T, int THREADS, bool ENT, bool TOP>
cudaError_t launch_forward(const MdLogprobsParams& p, int ctas, cudaStream_t stream) {
  auto kern = forward_kernel<T, THREADS, ENT, TOP>;
  const size_t smem = sizeof(Smem<THREADS, TOP>);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(p.rows) * ctas);
  cfg.blockDim = dim3(THREADS);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  cfg.attrs = attr;
  cfg.numAttrs = 0;
  if (ctas > 1) {
    attr[cfg.numAttrs].id = cudaLaunchAttributeClusterDimension;
    attr[cfg.numAttrs].val.clusterDim.x = ctas;
    attr[cfg.numAttrs].val.clusterDim.y = 1;
    attr[cfg.numAttrs].val.clusterDim.z = 1;
    ++cfg.numAttrs;
  }
  if (pdl_enabled()) {
    attr[cfg.numAttrs].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[cfg.numAttrs].val.programmaticStreamSerializationAllowed = 1;
    ++cfg.numAttrs;
  }
  return cudaLaunchKernelEx(&cfg, kern, p, ctas);
}

template <typename T, int THREADS>
cudaError_t pick_forward(const MdLogprobsParams& p, int ctas, cudaStream_t s) {
  if (p.want_entropy)
    return p.top > 0 ? launch_forward<T, THREADS, true, true>(p, ctas, s) : launch_forward<T, THREADS, true, false>(p, ctas, s);
  return p.top > 0 ? launch_forward<T, THREADS, false, true>(p, ctas, s) : launch_forward<T, THREADS, false, false>(p, ctas, s);
}

template <typename T>
cudaError_t forward(const MdLogprobsParams& p, cudaStream_t s) {
  const int nv = p.vocab / Pack<T>::N;
  // Rows that do not fill the SMs are shared by a cluster while each CTA keeps a few vectors per
  // thread; short rows take fewer threads, so that a thread still has several vectors.
  int ctas = 1;
  while (ctas < 8 && static_cast<long long>(p.rows) * ctas < 148 && nv / (2 * ctas) >= 512) ctas *= 2;
  const int mine = nv / ctas;
  if (mine >= 2048) return pick_forward<T, 512>(p, ctas, s);
  return mine >= 512 ? pick_forward<T, 256>(p, ctas, s) : pick_forward<T, 128>(p, ctas, s);
}

template <typename T>
cudaError_t backward(const MdLogprobsParams& p, cudaStream_t s) {
  constexpr int N = Pack<T>::N;
  const int nv = p.vocab / N;
  int slices = 1;  // enough CTAs for the SMs, several vectors per thread
  while (static_cast<long long>(p.rows) * slices < 148 * 4 && nv / (2 * slices) >= 256) slices *= 2;
  const dim3 grid(static_cast<unsigned>(p.rows) * slices), block(256);
  return p.g_entropy != nullptr ? launch_pdl(backward_kernel<T, true>, grid, block, 0, s, p, slices)
                                : launch_pdl(backward_kernel<T, false>, grid, block, 0, s, p, slices);
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
