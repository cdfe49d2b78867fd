// Rotary positions: each pair (a, b) of a head's first R channels is turned by
// the angle pos * f_i of its frequency,
//
//   a' = a cos - b sin,   b' = b cos + a sin,
//
// and the remaining D - R channels pass through.  Pairs are neighbours
// (2i, 2i+1) in the interleaved layout and (i, i + R/2) in the half layout.
// cos and sin come from an fp32 table [positions, R/2] of (cos, sin) computed
// once in 64 bits, so no angle is reduced on the device and a long context
// loses nothing; a factor on both (YaRN's attention scale) is part of the
// table.  The gradient is the transpose: the same kernel with sin negated.
//
// q and k go through one launch, each read once and written once, in place or
// into another tensor, at any batch / token / head stride, so q and k are
// turned where the QKV projection left them.
//
// DRAM-bound: 2 bytes in and out per channel against three flops.  A thread
// owns one vector (interleaved) or one pair of vectors R/2 apart (half) of a
// token and walks up to kHeads heads with it, so a table entry is loaded once
// for all of them and the loads of kHeads heads are in flight together.
#include <cuda_fp16.h>

#include "md_sm100.cuh"

struct MdRotaryParams {
  const void* x[2];        // q, k (k null: none)
  void* y[2];
  long long xs[2][3];      // element strides of batch, token, head
  long long ys[2][3];
  int heads[2];
  const float* table;      // [positions, R/2, 2]
  long long table_rows;
  const void* positions;   // null: the token's index in its sequence
  int positions64;         // 1: int64, 0: int32
  long long ps[2];         // element strides of batch, token
  int batch, seq, dim, rotary;
  int interleaved;
  int inverse;             // 1: turn back (the gradient)
  int dtype;               // 0 bf16, 1 fp16, 2 fp32
  md::Status* status;
};

namespace md {
namespace rotary {

template <typename T> __device__ __forceinline__ float to_f(T v);
template <> __device__ __forceinline__ float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }
template <> __device__ __forceinline__ float to_f(__half v) { return __half2float(v); }
template <> __device__ __forceinline__ float to_f(float v) { return v; }
template <typename T> __device__ __forceinline__ T from_f(float v);
template <> __device__ __forceinline__ __nv_bfloat16 from_f(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half from_f(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ float from_f(float v) { return v; }

template <typename T, int VEC>
struct alignas(sizeof(T) * VEC) Vec {
  T v[VEC];
};

// One thread: unit `u` of a token, heads h0, h0 + 1, .. h0 + HEADS - 1 (q's heads first, then k's).
// PAIRED: the unit is two vectors of VEC channels that turn together (the half layout; the
// interleaved layout with VEC = 1); otherwise one vector of VEC / 2 interleaved pairs.
template <typename T, int VEC, bool HALF, int HEADS>
__global__ void __launch_bounds__(256) rotary_kernel(const __grid_constant__ MdRotaryParams p, int units, int rot_units,
                                                     int head_groups, long long total) {
  constexpr bool PAIRED = HALF || VEC == 1;
  constexpr int NCS = PAIRED ? VEC : VEC / 2;  // (cos, sin) entries a unit needs
  using V = Vec<T, VEC>;
  pdl_trigger();
  pdl_wait();
  const long long id = blockIdx.x * 256ll + threadIdx.x;
  if (id >= total) return;
  const long long tg = id / units;
  const int u = static_cast<int>(id - tg * units);
  const long long token = tg / head_groups;
  const int h0 = static_cast<int>(tg - token * head_groups) * HEADS;
  const int b = static_cast<int>(token / p.seq), s = static_cast<int>(token - static_cast<long long>(b) * p.seq);
  const int all = p.heads[0] + p.heads[1];
  const bool turns = u < rot_units;

  int c0, c1;  // first channel of the unit's vectors
  if (!turns) c0 = c1 = p.rotary + (u - rot_units) * VEC;
  else if (HALF) c0 = u * VEC, c1 = p.rotary / 2 + u * VEC;
  else if (VEC == 1) c0 = 2 * u, c1 = 2 * u + 1;
  else c0 = c1 = u * VEC;

  V x0[HEADS], x1[HEADS];
  const T* src[HEADS];
  T* dst[HEADS];
#pragma unroll
  for (int i = 0; i < HEADS; ++i) {
    const int hh = h0 + i;
    const int w = hh >= p.heads[0] ? 1 : 0;
    const int h = hh - (w ? p.heads[0] : 0);
    src[i] = static_cast<const T*>(w ? p.x[1] : p.x[0]) + b * (w ? p.xs[1][0] : p.xs[0][0]) +
             s * (w ? p.xs[1][1] : p.xs[0][1]) + h * (w ? p.xs[1][2] : p.xs[0][2]);
    dst[i] = static_cast<T*>(w ? p.y[1] : p.y[0]) + b * (w ? p.ys[1][0] : p.ys[0][0]) +
             s * (w ? p.ys[1][1] : p.ys[0][1]) + h * (w ? p.ys[1][2] : p.ys[0][2]);
    if (hh < all) {
      x0[i] = *reinterpret_cast<const V*>(src[i] + c0);
      if (PAIRED && turns) x1[i] = *reinterpret_cast<const V*>(src[i] + c1);
    }
  }
  if (!turns) {
#pragma unroll
    for (int i = 0; i < HEADS; ++i)
      if (h0 + i < all) *reinterpret_cast<V*>(dst[i] + c0) = x0[i];
    return;
  }

  long long pos = s;
  if (p.positions != nullptr) {
    const long long o = b * p.ps[0] + s * p.ps[1];
    pos = p.positions64 ? static_cast<const long long*>(p.positions)[o] : static_cast<const int*>(p.positions)[o];
  }
  float cs[2 * NCS];
  if (pos >= 0 && pos < p.table_rows) {
    const float* t = p.table + (pos * (p.rotary / 2) + (PAIRED ? u * (HALF ? VEC : 1) : u * (VEC / 2))) * 2;
    if (NCS % 2 == 0) {  // two entries at a time: such a vector width divides R/2, so rows are whole
#pragma unroll
      for (int q = 0; q < NCS / 2; ++q) {
        const float4 f = __ldg(reinterpret_cast<const float4*>(t) + q);
        cs[4 * q] = f.x, cs[4 * q + 1] = f.y, cs[4 * q + 2] = f.z, cs[4 * q + 3] = f.w;
      }
    } else {
#pragma unroll
      for (int q = 0; q < NCS; ++q) {
        const float2 f = __ldg(reinterpret_cast<const float2*>(t) + q);
        cs[2 * q] = f.x, cs[2 * q + 1] = f.y;
      }
    }
  } else {  // outside the table: reported, and visible in the result
    if (u == 0) report(p.status, kBadArgument, 400, static_cast<uint32_t>(pos));
#pragma unroll
    for (int q = 0; q < 2 * NCS; ++q) cs[q] = __int_as_float(0x7fffffff);
  }
  if (p.inverse) {
#pragma unroll
    for (int q = 0; q < NCS; ++q) cs[2 * q + 1] = -cs[2 * q + 1];
  }
#pragma unroll
  for (int i = 0; i < HEADS; ++i) {
    if (h0 + i >= all) break;
    if (PAIRED) {
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        const float a = to_f(x0[i].v[j]), c = to_f(x1[i].v[j]);
        x0[i].v[j] = from_f<T>(a * cs[2 * j] - c * cs[2 * j + 1]);
        x1[i].v[j] = from_f<T>(c * cs[2 * j] + a * cs[2 * j + 1]);
      }
      *reinterpret_cast<V*>(dst[i] + c0) = x0[i];
      *reinterpret_cast<V*>(dst[i] + c1) = x1[i];
    } else {
#pragma unroll
      for (int j = 0; j < VEC / 2; ++j) {
        const float a = to_f(x0[i].v[2 * j]), c = to_f(x0[i].v[2 * j + 1]);
        x0[i].v[2 * j] = from_f<T>(a * cs[2 * j] - c * cs[2 * j + 1]);
        x0[i].v[2 * j + 1] = from_f<T>(c * cs[2 * j] + a * cs[2 * j + 1]);
      }
      *reinterpret_cast<V*>(dst[i] + c0) = x0[i];
    }
  }
}

constexpr int kHeads = 4;

template <typename T, int VEC, bool HALF>
cudaError_t launch(const MdRotaryParams& p, bool in_place, cudaStream_t stream) {
  constexpr bool PAIRED = HALF || VEC == 1;
  const int rot_units = PAIRED ? p.rotary / 2 / VEC : p.rotary / VEC;
  const int units = rot_units + (in_place ? 0 : (p.dim - p.rotary) / VEC);
  const long long tokens = static_cast<long long>(p.batch) * p.seq;
  const int all = p.heads[0] + p.heads[1];
  // One head per thread while that leaves SMs without work, four once the grid is larger.
  const bool few = tokens * units * all < 148ll * 2048;
  const int per = few ? 1 : kHeads;
  const int groups = (all + per - 1) / per;
  const long long total = tokens * groups * units;
  const long long blocks = (total + 255) / 256;
  if (blocks > 0x7fffffffll) return cudaErrorInvalidConfiguration;
  const dim3 grid(static_cast<unsigned>(blocks));
  return few ? launch_pdl(rotary_kernel<T, VEC, HALF, 1>, grid, dim3(256), 0, stream, p, units, rot_units, groups, total)
             : launch_pdl(rotary_kernel<T, VEC, HALF, kHeads>, grid, dim3(256), 0, stream, p, units, rot_units, groups, total);
}

template <typename T, int VEC>
cudaError_t pick_layout(const MdRotaryParams& p, bool in_place, cudaStream_t s) {
  return p.interleaved ? launch<T, VEC, false>(p, in_place, s) : launch<T, VEC, true>(p, in_place, s);
}

}  // namespace rotary
}  // namespace md

// 0 ok; negative: refused (nothing launched); positive: CUDA error of the launch.
extern "C" int md_rotary(const MdRotaryParams* prm, cudaStream_t stream) {
  using namespace md::rotary;
  if (prm == nullptr) return -1;
  const MdRotaryParams& p = *prm;
  if (p.batch < 0 || p.seq < 0 || p.heads[0] < 0 || p.heads[1] < 0 || p.dim <= 0) return -2;
  if (p.rotary <= 0 || p.rotary % 2 || p.rotary > p.dim || p.table == nullptr || p.table_rows < 0) return -3;
  if (reinterpret_cast<uintptr_t>(p.table) & 15u) return -4;
  if (p.dtype < 0 || p.dtype > 2) return -5;
  if (p.batch == 0 || p.seq == 0 || p.heads[0] + p.heads[1] == 0) return 0;
  const int es = p.dtype == 2 ? 4 : 2;
  // The widest vector that divides every offset a vector can start at: the tensors' addresses
  // and strides, the head, its rotary part and, for the half layout, half of that.
  unsigned long long bits = static_cast<unsigned long long>(p.dim) * es | static_cast<unsigned long long>(p.rotary) * es;
  if (!p.interleaved) bits |= static_cast<unsigned long long>(p.rotary / 2) * es;
  bool in_place = true;
  for (int w = 0; w < 2; ++w) {
    if (p.heads[w] == 0) continue;
    if (p.x[w] == nullptr || p.y[w] == nullptr) return -6;
    bits |= reinterpret_cast<uintptr_t>(p.x[w]) | reinterpret_cast<uintptr_t>(p.y[w]);
    in_place = in_place && p.x[w] == p.y[w];
    for (int i = 0; i < 3; ++i) {
      bits |= static_cast<unsigned long long>(p.xs[w][i]) * es | static_cast<unsigned long long>(p.ys[w][i]) * es;
      if (p.xs[w][i] != p.ys[w][i]) in_place = false;
    }
  }
  int vec = 1;
  while (vec * es < 16 && bits % (2ull * vec * es) == 0) vec *= 2;
  cudaError_t e;
  if (p.dtype == 0) {
    e = vec == 8   ? pick_layout<__nv_bfloat16, 8>(p, in_place, stream)
        : vec == 4 ? pick_layout<__nv_bfloat16, 4>(p, in_place, stream)
        : vec == 2 ? pick_layout<__nv_bfloat16, 2>(p, in_place, stream)
                   : pick_layout<__nv_bfloat16, 1>(p, in_place, stream);
  } else if (p.dtype == 1) {
    e = vec == 8   ? pick_layout<__half, 8>(p, in_place, stream)
        : vec == 4 ? pick_layout<__half, 4>(p, in_place, stream)
        : vec == 2 ? pick_layout<__half, 2>(p, in_place, stream)
                   : pick_layout<__half, 1>(p, in_place, stream);
  } else {
    e = vec == 4   ? pick_layout<float, 4>(p, in_place, stream)
        : vec == 2 ? pick_layout<float, 2>(p, in_place, stream)
                   : pick_layout<float, 1>(p, in_place, stream);
  }
  return static_cast<int>(e);
}
