// norm.hip — the residual update around a block with the norms on its two
// sides, on gfx950.
//
//   u = y * rsqrt(mean(y^2) + eps) * (post + offset)    (u = y without post)
//   h = x + scale * gate * u                            (gate 1 without one)
//   n = h * rsqrt(mean(h^2) + eps) * (pre + offset)     (of h before its rounding)
//
// over rows of H elements.  All in 32 bits; h and n are rounded once each.
// HBM-bound: x, y and the gate are read once, h and n written once.  A workgroup
// takes a row and holds it in registers, 8 elements (one or two 16-byte loads)
// a lane and vector, so nothing is read twice; all loads, the weights' too, are
// issued before the first sum, so a single row waits for memory once (1 x 4096:
// 5.0 us, the launch's own time; 2047 x 2880 with a gate and both norms: 14.8 us,
// 4.0 TB/s of its 59 MB).
#include <hip/hip_runtime.h>

#include <type_traits>

#include "common.hpp"
#include "kernels.hpp"
#include "wave.hpp"

namespace mlxq {

namespace {

typedef uint32_t u32x4_e __attribute__((ext_vector_type(4), aligned(2)));

// 8 elements of a row as they lie in memory
template <int XT>
struct Raw {
  u32x4 w[XT == GEN_F32 ? 2 : 1];
  __device__ __forceinline__ float operator[](int e) const {
    if constexpr (XT == GEN_F32) return __uint_as_float(w[e / 4][e % 4]);
    else if constexpr (XT == GEN_BF16) return __uint_as_float(e & 1 ? w[0][e / 2] & 0xFFFF0000u : w[0][e / 2] << 16);
    else return xt_to_f32<1>(e & 1 ? w[0][e / 2] >> 16 : w[0][e / 2] & 0xFFFFu);
  }
};

// Elements i .. i + 7 of a row of H at p, zeros past its end.
template <int XT>
__device__ __forceinline__ Raw<XT> load8(const void* p, int i, int H) {
  constexpr int ES = XT == GEN_F32 ? 4 : 2;
  Raw<XT> r;
  const char* q = static_cast<const char*>(p) + (int64_t)i * ES;
  if (i + 8 <= H) {
#pragma unroll
    for (int k = 0; k < ES / 2; k++) {
      const u32x4_e v = reinterpret_cast<const u32x4_e*>(q)[k];
      r.w[k] = u32x4{v[0], v[1], v[2], v[3]};
    }
  } else {
#pragma unroll
    for (int k = 0; k < ES / 2; k++) r.w[k] = u32x4{0u, 0u, 0u, 0u};
#pragma unroll
    for (int e = 0; e < 8; e++) {  // the row's last elements
      if (i + e >= H) continue;
      if constexpr (ES == 4) r.w[e / 4][e % 4] = reinterpret_cast<const uint32_t*>(q)[e];
      else r.w[0][e / 2] |= (uint32_t)reinterpret_cast<const uint16_t*>(q)[e] << (16 * (e & 1));
    }
  }
  return r;
}

template <int XT>
__device__ __forceinline__ void store8(void* p, int i, int H, const float (&v)[8]) {
  constexpr int ES = XT == GEN_F32 ? 4 : 2;
  char* q = static_cast<char*>(p) + (int64_t)i * ES;
  Raw<XT> r;
  if constexpr (ES == 4) {
#pragma unroll
    for (int e = 0; e < 8; e++) r.w[e / 4][e % 4] = __float_as_uint(v[e]);
  } else {
#pragma unroll
    for (int e = 0; e < 8; e += 2)
      r.w[0][e / 2] = f32_to_xt<XT == GEN_F16 ? 1 : 0>(v[e]) | f32_to_xt<XT == GEN_F16 ? 1 : 0>(v[e + 1]) << 16;
  }
  if (i + 8 <= H) {
#pragma unroll
    for (int k = 0; k < ES / 2; k++) reinterpret_cast<u32x4_e*>(q)[k] = r.w[k];
  } else {
#pragma unroll
    for (int e = 0; e < 8; e++) {
      if (i + e >= H) continue;
      if constexpr (ES == 4) reinterpret_cast<uint32_t*>(q)[e] = r.w[e / 4][e % 4];
      else reinterpret_cast<uint16_t*>(q)[e] = (uint16_t)(r.w[0][e / 2] >> (16 * (e & 1)));
    }
  }
}

// 8 weights: of the row's type as they lie in memory, or (W32) any type in 32 bits
template <int XT, bool W32>
__device__ __forceinline__ Raw<W32 ? GEN_F32 : XT> load_weight(const void* p, int type, int i, int H) {
  if constexpr (W32) {
    if (type == GEN_F32) return load8<GEN_F32>(p, i, H);
    const Raw<XT> r = load8<XT>(p, i, H);
    Raw<GEN_F32> w;
#pragma unroll
    for (int e = 0; e < 8; e++) w.w[e / 4][e % 4] = __float_as_uint(r[e]);
    return w;
  } else {
    return load8<XT>(p, i, H);
  }
}

// Sum over the workgroup, the same in each thread; lds: 16 words of this sum.
__device__ __forceinline__ float block_sum(float v, float* lds) {
  v = wave_sum(v, threadIdx.x & 63);
  const int waves = blockDim.x >> 6;
  if (waves == 1) return v;
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
  __syncthreads();
  float s = 0.f;
  for (int w = 0; w < waves; w++) s += lds[w];
  return s;
}

// NV vectors of 8 elements a lane: vector v of lane t is elements 8 (v threads + t) on.
template <int XT, int NV, bool W32>
__global__ __launch_bounds__(1024) void residual_norm_kernel(const ResidualNormArgs a) {
  constexpr int ES = XT == GEN_F32 ? 4 : 2;
  __shared__ float sums[2][16];
  const int64_t t = blockIdx.x, gr = t / a.gate_div;
  const char* x = static_cast<const char*>(a.x) + t * a.x_row * ES;
  const char* y = static_cast<const char*>(a.y) + t * a.y_row * ES;
  const char* g = static_cast<const char*>(a.gate) + gr * a.gate_row * ES;
  const int step = 8 * blockDim.x, i0 = 8 * threadIdx.x;
  Raw<XT> rx[NV], ry[NV], rg[NV];
  Raw<W32 ? GEN_F32 : XT> wp[NV], wn[NV];
#pragma unroll
  for (int v = 0; v < NV; v++) ry[v] = load8<XT>(y, i0 + v * step, a.H);
#pragma unroll
  for (int v = 0; v < NV; v++) rx[v] = load8<XT>(x, i0 + v * step, a.H);
  float gate = a.scale;
  if (a.gate) {
    if (a.gate_col) {
#pragma unroll
      for (int v = 0; v < NV; v++) rg[v] = load8<XT>(g, i0 + v * step, a.H);
    } else {
      gate *= XT == GEN_F32 ? *reinterpret_cast<const float*>(g)
                            : xt_to_f32<XT == GEN_F16 ? 1 : 0>(*reinterpret_cast<const uint16_t*>(g));
    }
  }
  if (a.post) {
#pragma unroll
    for (int v = 0; v < NV; v++) wp[v] = load_weight<XT, W32>(a.post, a.post_type, i0 + v * step, a.H);
  }
  if (a.pre) {
#pragma unroll
    for (int v = 0; v < NV; v++) wn[v] = load_weight<XT, W32>(a.pre, a.pre_type, i0 + v * step, a.H);
  }
  float f = 1.f;
  if (a.post) {
    float s = 0.f;
#pragma unroll
    for (int v = 0; v < NV; v++)
#pragma unroll
      for (int e = 0; e < 8; e++) s += ry[v][e] * ry[v][e];
    f = rsqrtf(block_sum(s, sums[0]) / (float)a.H + a.eps);
  }
  float h[NV][8], s = 0.f;
  const bool gates = a.gate && a.gate_col;
#pragma unroll
  for (int v = 0; v < NV; v++) {
#pragma unroll
    for (int e = 0; e < 8; e++) {
      float u = ry[v][e];
      if (a.post) u = u * f * (wp[v][e] + a.offset);
      if (gates) u *= rg[v][e];
      h[v][e] = rx[v][e] + gate * u;
      s += h[v][e] * h[v][e];
    }
    store8<XT>(static_cast<char*>(a.h) + t * a.H * ES, i0 + v * step, a.H, h[v]);
  }
  if (!a.pre) return;
  f = rsqrtf(block_sum(s, sums[1]) / (float)a.H + a.eps);
#pragma unroll
  for (int v = 0; v < NV; v++) {
#pragma unroll
    for (int e = 0; e < 8; e++) h[v][e] = h[v][e] * f * (wn[v][e] + a.offset);
    store8<XT>(static_cast<char*>(a.n) + t * a.H * ES, i0 + v * step, a.H, h[v]);
  }
}

template <int XT>
hipError_t launch(const ResidualNormArgs& a, hipStream_t stream) {
  const int vecs = (a.H + 7) / 8;
  // One vector a lane while all rows' waves are resident (256 CUs of 32), two
  // past that: 2047 rows of 2880 15.4 us with two and 17.3 with one, 1400 of 8192
  // 21.0 and 23.6 (float32 43.5 and 41.4); 700 rows of 2880 8.8 and 8.2, 4096 of
  // 64 9.1 and 5.5.
  int nv = a.T * ((vecs + 63) / 64) > 8192 ? 2 : 1;
  while ((vecs + nv - 1) / nv > 1024) nv *= 2;
  const dim3 grid((unsigned)a.T), block((unsigned)(((vecs + nv - 1) / nv + 63) / 64 * 64));
  const bool w32 = XT != GEN_F32 && ((a.post && a.post_type != XT) || (a.pre && a.pre_type != XT));
  auto run = [&](auto w) {
    constexpr bool W32 = decltype(w)::value;
    if (nv == 1) hipLaunchKernelGGL((residual_norm_kernel<XT, 1, W32>), grid, block, 0, stream, a);
    else if (nv == 2) hipLaunchKernelGGL((residual_norm_kernel<XT, 2, W32>), grid, block, 0, stream, a);
    else hipLaunchKernelGGL((residual_norm_kernel<XT, 4, W32>), grid, block, 0, stream, a);
  };
  if constexpr (XT != GEN_F32) {
    if (w32) {
      run(std::true_type{});
      return hipGetLastError();
    }
  }
  run(std::false_type{});
  return hipGetLastError();
}

}  // namespace

hipError_t launch_residual_norm(const ResidualNormArgs& a, hipStream_t stream) {
  if (a.T == 0 || a.H == 0) return hipSuccess;
  if (a.H > kNormMaxH || a.T > 0x7FFFFFFF || a.gate_div < 1) return hipErrorInvalidValue;
  if (a.type == GEN_BF16) return launch<GEN_BF16>(a, stream);
  if (a.type == GEN_F16) return launch<GEN_F16>(a, stream);
  return launch<GEN_F32>(a, stream);
}

}  // namespace mlxq
