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
// DRAM-bound: 2 bytes in and out per channel against three flops, so what counts is
// few instructions per byte and enough loads in flight.  A thread owns one unit of
// a token (a vector, in the half layout the two vectors that turn together) for
// four heads: cos and sin are loaded once for all four, the index arithmetic
// (multiplications instead of divisions) is paid once, and the channels that pass
// through are copied by the same threads in vectors of their own width.
//
// Measured (B200, copy rate 6.55 TB/s): 20011 tokens of 32 + 32 heads of 80, 40 of
// them turned, bf16: 76 us, 5.4 TB/s (a loop over vectors with divisions and single
// conversions: 190 us, of which 45 % was issuing instructions); 16 x 1024 tokens of
// 12 + 12 heads of 64 in a packed projection: 20 us, 5.0 TB/s, a third of it start
// and end of so short a launch; fp32 heads of 128: 6.4 TB/s; one token for each of
// 32 sequences: 1.9 us.  An odd R/2 in the half layout, or odd strides, go by single
// channels: the prompt with 50 of 80 turned 129 us (interleaved, by pairs, 104).
// Two heads per thread instead of four measured the same within 5 % on paired layouts
// and 15 % slower on interleaved ones.
#include <cuda_fp16.h>

#include <type_traits>

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

template <int BYTES> struct RawOf;
template <> struct RawOf<16> { using type = uint4; };
template <> struct RawOf<8> { using type = uint2; };
template <> struct RawOf<4> { using type = uint32_t; };
template <> struct RawOf<2> { using type = uint16_t; };

// VEC channels as loaded, and as fp32 (pairs are converted together).
template <typename T, int VEC>
struct Vec {
  using Raw = typename RawOf<sizeof(T) * VEC>::type;
  static __device__ __forceinline__ void get(const Raw& raw, float (&f)[VEC]) {
    const T* t = reinterpret_cast<const T*>(&raw);
    if constexpr (sizeof(T) == 2 && VEC >= 2) {
      const uint32_t* w = reinterpret_cast<const uint32_t*>(&raw);
#pragma unroll
      for (int q = 0; q < VEC / 2; ++q) {
        float2 v;
        if constexpr (std::is_same<T, __nv_bfloat16>::value) v = unpack_bf16x2(w[q]);
        else v = __half22float2(*reinterpret_cast<const __half2*>(w + q));
        f[2 * q] = v.x, f[2 * q + 1] = v.y;
      }
    } else {
#pragma unroll
      for (int j = 0; j < VEC; ++j) f[j] = to_f(t[j]);
    }
  }
  static __device__ __forceinline__ Raw put(const float (&f)[VEC]) {
    Raw raw;
    if constexpr (sizeof(T) == 2 && VEC >= 2) {
      uint32_t* w = reinterpret_cast<uint32_t*>(&raw);
#pragma unroll
      for (int q = 0; q < VEC / 2; ++q) {
        if constexpr (std::is_same<T, __nv_bfloat16>::value) {
          w[q] = pack_bf16x2(f[2 * q], f[2 * q + 1]);
        } else {
          const __half2 h = __floats2half2_rn(f[2 * q], f[2 * q + 1]);
          w[q] = *reinterpret_cast<const uint32_t*>(&h);
        }
      }
    } else {
      T* t = reinterpret_cast<T*>(&raw);
#pragma unroll
      for (int j = 0; j < VEC; ++j) t[j] = from_f<T>(f[j]);
    }
    return raw;
  }
};

// n / d and n mod d for n < 2^31 by one multiplication (d from the host; Granlund & Montgomery 1994).
struct Divide {
  unsigned d, mul, shift;
  static Divide by(unsigned d) {
    Divide v{d, 0, 0};
    while ((1ull << v.shift) < d) ++v.shift;
    v.mul = static_cast<unsigned>(((1ull << 32) * ((1ull << v.shift) - d)) / d + 1);
    return v;
  }
  __device__ __forceinline__ unsigned operator()(unsigned n) const { return (__umulhi(n, mul) + n) >> shift; }
};

constexpr int kHeads = 4;  // heads per thread

struct Shape {
  unsigned total[2];   // threads with work, for q and for k
  Divide units;        // units of a head
  Divide groups[2];    // groups of kHeads heads, or single heads when there are few threads
  Divide seq;
  int per;             // heads of a group (kHeads or 1)
  int pass_bytes;      // width of the pass-through vectors (16, 8, 4 or 2)
  int pass;            // pass-through vectors of a head (0: in place)
};

template <typename W>
__device__ __forceinline__ void copy_pass(const char* x, char* y, long long xs, long long ys, int n, int u, int units, int pass) {
  for (int v = u; v < pass; v += units) {
    W w[kHeads];
#pragma unroll
    for (int i = 0; i < kHeads; ++i)
      if (i < n) w[i] = *reinterpret_cast<const W*>(x + i * xs + v * sizeof(W));
#pragma unroll
    for (int i = 0; i < kHeads; ++i)
      if (i < n) *reinterpret_cast<W*>(y + i * ys + v * sizeof(W)) = w[i];
  }
}

// PAIRED: a unit is two vectors of VEC channels that turn together (the half layout; the
// interleaved layout with VEC = 1); otherwise one vector of VEC / 2 interleaved pairs.
template <typename T, int VEC, bool HALF>
__global__ void __launch_bounds__(256, 3) rotary_kernel(const __grid_constant__ MdRotaryParams p,
                                                     const __grid_constant__ Shape sh) {
  constexpr bool PAIRED = HALF || VEC == 1;
  constexpr int NCS = PAIRED ? VEC : VEC / 2;  // (cos, sin) entries a unit needs
  using V = Vec<T, VEC>;
  using Raw = typename V::Raw;
  pdl_trigger();
  pdl_wait();
  const int w = blockIdx.y;  // q or k
  const unsigned id = blockIdx.x * 256u + threadIdx.x;
  if (id >= sh.total[w]) return;
  const unsigned rest = sh.units(id);
  const int u = static_cast<int>(id - rest * sh.units.d);
  const unsigned token = sh.groups[w](rest);
  const int h0 = static_cast<int>(rest - token * sh.groups[w].d) * sh.per;
  const unsigned b = sh.seq(token);
  const int s = static_cast<int>(token - b * sh.seq.d);
  const int n = min(sh.per, p.heads[w] - h0);
  const long long xs = p.xs[w][2], ys = p.ys[w][2];
  const T* x = static_cast<const T*>(p.x[w]) + b * p.xs[w][0] + s * p.xs[w][1] + h0 * xs;
  T* y = static_cast<T*>(p.y[w]) + b * p.ys[w][0] + s * p.ys[w][1] + h0 * ys;
  // First channels of the unit's vectors.
  const int c0 = HALF ? u * VEC : PAIRED ? 2 * u : u * VEC;
  const int c1 = HALF ? p.rotary / 2 + u * VEC : PAIRED ? 2 * u + 1 : 0;
  Raw r0[kHeads], r1[kHeads];
#pragma unroll
  for (int i = 0; i < kHeads; ++i) {
    if (i < n) {
      r0[i] = *reinterpret_cast<const Raw*>(x + i * xs + c0);
      if (PAIRED) r1[i] = *reinterpret_cast<const Raw*>(x + i * xs + c1);
    }
  }

  long long pos = s;
  if (p.positions != nullptr) {
    const long long o = b * p.ps[0] + s * p.ps[1];
    pos = p.positions64 ? static_cast<const long long*>(p.positions)[o] : static_cast<const int*>(p.positions)[o];
  }
  float cs[2 * NCS];
  if (pos >= 0 && pos < p.table_rows) {
    const float* t = p.table + (pos * (p.rotary / 2) + (PAIRED ? u * (HALF ? VEC : 1) : u * (VEC / 2))) * 2;
    if (NCS % 2 == 0) {  // two entries at a time: such a width divides R/2, so rows are whole and aligned
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
  for (int i = 0; i < kHeads; ++i) {
    if (i >= n) break;
    T* dst = y + i * ys;
    float a[VEC], c[VEC], o[VEC];
    V::get(r0[i], a);
    if (PAIRED) {
      V::get(r1[i], c);
#pragma unroll
      for (int j = 0; j < VEC; ++j) o[j] = a[j] * cs[2 * j] - c[j] * cs[2 * j + 1];
      *reinterpret_cast<Raw*>(dst + c0) = V::put(o);
#pragma unroll
      for (int j = 0; j < VEC; ++j) o[j] = c[j] * cs[2 * j] + a[j] * cs[2 * j + 1];
      *reinterpret_cast<Raw*>(dst + c1) = V::put(o);
    } else {
#pragma unroll
      for (int j = 0; j < VEC / 2; ++j) {
        o[2 * j] = a[2 * j] * cs[2 * j] - a[2 * j + 1] * cs[2 * j + 1];
        o[2 * j + 1] = a[2 * j + 1] * cs[2 * j] + a[2 * j] * cs[2 * j + 1];
      }
      *reinterpret_cast<Raw*>(dst + c0) = V::put(o);
    }
  }
  if (sh.pass > 0) {
    const char* px = reinterpret_cast<const char*>(x + p.rotary);
    char* py = reinterpret_cast<char*>(y + p.rotary);
    const long long xb = xs * static_cast<long long>(sizeof(T)), yb = ys * static_cast<long long>(sizeof(T));
    const int units = static_cast<int>(sh.units.d);
    if (sh.pass_bytes == 16) copy_pass<uint4>(px, py, xb, yb, n, u, units, sh.pass);
    else if (sh.pass_bytes == 8) copy_pass<uint2>(px, py, xb, yb, n, u, units, sh.pass);
    else if (sh.pass_bytes == 4) copy_pass<uint32_t>(px, py, xb, yb, n, u, units, sh.pass);
    else copy_pass<uint16_t>(px, py, xb, yb, n, u, units, sh.pass);
  }
}

template <typename T, int VEC, bool HALF>
cudaError_t launch(const MdRotaryParams& p, bool in_place, int pass_bytes, cudaStream_t stream) {
  constexpr bool PAIRED = HALF || VEC == 1;
  const int units = PAIRED ? p.rotary / 2 / VEC : p.rotary / VEC;
  Shape sh;
  sh.units = Divide::by(units);
  sh.seq = Divide::by(p.seq);
  sh.pass_bytes = pass_bytes;
  sh.pass = in_place ? 0 : (p.dim - p.rotary) * static_cast<int>(sizeof(T)) / pass_bytes;
  const long long tokens = static_cast<long long>(p.batch) * p.seq;
  // One head per thread while that leaves SMs without work, four once the grid is larger.
  sh.per = tokens * units * (p.heads[0] + p.heads[1]) < 148ll * 2048 ? 1 : kHeads;
  long long most = 0;
  for (int w = 0; w < 2; ++w) {
    const int groups = (p.heads[w] + sh.per - 1) / sh.per;
    const long long total = tokens * groups * units;
    if (total > 0x7fffff00ll) return cudaErrorInvalidConfiguration;
    sh.groups[w] = Divide::by(groups > 0 ? groups : 1);
    sh.total[w] = static_cast<unsigned>(total);
    if (total > most) most = total;
  }
  const dim3 grid(static_cast<unsigned>((most + 255) / 256), p.heads[1] > 0 ? 2 : 1);
  return launch_pdl(rotary_kernel<T, VEC, HALF>, grid, dim3(256), 0, stream, p, sh);
}

template <typename T, int VEC>
cudaError_t pick_layout(const MdRotaryParams& p, bool in_place, int pass_bytes, cudaStream_t s) {
  return p.interleaved ? launch<T, VEC, false>(p, in_place, pass_bytes, s) : launch<T, VEC, true>(p, in_place, pass_bytes, s);
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
  // Two entries at a time are read where a row holds an even number of them, one at a time elsewhere
  // (an odd R/2 leaves units of one entry), so a table may start at any of its rows.
  if (reinterpret_cast<uintptr_t>(p.table) & (p.rotary % 4 == 0 ? 15u : 7u)) return -4;
  if (p.dtype < 0 || p.dtype > 2) return -5;
  if (p.batch == 0 || p.seq == 0 || p.heads[0] + p.heads[1] == 0) return 0;
  const int es = p.dtype == 2 ? 4 : 2;
  // The widest vectors that divide every offset one can start at: the tensors' addresses and strides,
  // and the rotary part (half of it in the half layout) or, passing through, its end and the head's.
  unsigned long long bits = 0;
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
  auto widest = [](unsigned long long offsets, int from) {
    int w = from;
    while (w < 16 && offsets % (2ull * w) == 0) w *= 2;
    return w;
  };
  const unsigned long long turned = static_cast<unsigned long long>(p.interleaved ? p.rotary : p.rotary / 2) * es;
  const int vec = widest(bits | turned, es) / es;
  const int pass = widest(bits | static_cast<unsigned long long>(p.rotary) * es | static_cast<unsigned long long>(p.dim) * es, es);
  cudaError_t e;
  if (p.dtype == 0) {
    e = vec == 8   ? pick_layout<__nv_bfloat16, 8>(p, in_place, pass, stream)
        : vec == 4 ? pick_layout<__nv_bfloat16, 4>(p, in_place, pass, stream)
        : vec == 2 ? pick_layout<__nv_bfloat16, 2>(p, in_place, pass, stream)
                   : pick_layout<__nv_bfloat16, 1>(p, in_place, pass, stream);
  } else if (p.dtype == 1) {
    e = vec == 8   ? pick_layout<__half, 8>(p, in_place, pass, stream)
        : vec == 4 ? pick_layout<__half, 4>(p, in_place, pass, stream)
        : vec == 2 ? pick_layout<__half, 2>(p, in_place, pass, stream)
                   : pick_layout<__half, 1>(p, in_place, pass, stream);
  } else {
    e = vec == 4   ? pick_layout<float, 4>(p, in_place, pass, stream)
        : vec == 2 ? pick_layout<float, 2>(p, in_place, pass, stream)
                   : pick_layout<float, 1>(p, in_place, pass, stream);
  }
  return static_cast<int>(e);
}
