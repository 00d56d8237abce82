// norm.hip — the residual update around a block with the norms on its two
// sides, on gfx950.
//
//   u = y * rsqrt(mean(y^2) + eps) * (post + offset)    (u = y without post)
//   h = x + scale * gate * u                            (gate 1 without one)
//   n = h * rsqrt(mean(h^2) + eps) * (pre + offset)     (of h before its rounding)
//
// over rows of H elements.  All in 32 bits; h and n are rounded once each.
// HBM-bound: x, y and the gate are read once, h and n written once.
#include <hip/hip_runtime.h>

#include "common.hpp"
#include "kernels.hpp"

namespace mlxq {

namespace {

__device__ __forceinline__ float load(const void* p, int64_t i, int type) {
  if (type == GEN_F32) return static_cast<const float*>(p)[i];
  const uint32_t w = static_cast<const uint16_t*>(p)[i];
  return type == GEN_BF16 ? xt_to_f32<0>(w) : xt_to_f32<1>(w);
}

__device__ __forceinline__ void store(void* p, int64_t i, float v, int type) {
  if (type == GEN_F32) static_cast<float*>(p)[i] = v;
  else static_cast<uint16_t*>(p)[i] = (uint16_t)(type == GEN_BF16 ? f32_to_xt<0>(v) : f32_to_xt<1>(v));
}

// sum over the workgroup's 256 threads, the same in each
__device__ __forceinline__ float block_sum(float v, float* lds) {
#pragma unroll
  for (int s = 32; s; s >>= 1) v += __shfl_xor(v, s);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
  __syncthreads();
  return (lds[0] + lds[1]) + (lds[2] + lds[3]);
}

__global__ __launch_bounds__(256) void residual_norm_kernel(const ResidualNormArgs a) {
  extern __shared__ float row[];  // [4] sums, then h in 32 bits
  float* hs = row + 4;
  const int64_t t = blockIdx.x;
  const int64_t xr = t * a.x_row, yr = t * a.y_row, gr = (t / a.gate_div) * a.gate_row;
  float f = 1.f;
  if (a.post) {
    float s = 0.f;
    for (int i = threadIdx.x; i < a.H; i += 256) {
      const float y = load(a.y, yr + i, a.type);
      s += y * y;
    }
    f = rsqrtf(block_sum(s, row) / (float)a.H + a.eps);
  }
  float s = 0.f;
  for (int i = threadIdx.x; i < a.H; i += 256) {
    float u = load(a.y, yr + i, a.type);
    if (a.post) u = u * f * (load(a.post, i, a.post_type) + a.offset);
    if (a.gate) u *= load(a.gate, gr + i * a.gate_col, a.type);
    const float h = load(a.x, xr + i, a.type) + a.scale * u;
    hs[i] = h;
    s += h * h;
  }
  const float fn = rsqrtf(block_sum(s, row) / (float)a.H + a.eps);
  for (int i = threadIdx.x; i < a.H; i += 256) {
    store(a.h, t * a.H + i, hs[i], a.type);
    if (a.pre) store(a.n, t * a.H + i, hs[i] * fn * (load(a.pre, i, a.pre_type) + a.offset), a.type);
  }
}

}  // namespace

hipError_t launch_residual_norm(const ResidualNormArgs& a, hipStream_t stream) {
  if (a.T == 0 || a.H == 0) return hipSuccess;
  if (a.H > kNormMaxH || a.T > 0x7FFFFFFF || a.gate_div < 1) return hipErrorInvalidValue;
  hipLaunchKernelGGL(residual_norm_kernel, dim3((unsigned)a.T), dim3(256), (4 + a.H) * sizeof(float), stream, a);
  return hipGetLastError();
}

}  // namespace mlxq
