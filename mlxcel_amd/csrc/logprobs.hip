// logprobs.hip — log probabilities of given tokens, the entropy and the most
// probable tokens of rows of logits, on gfx950.
//
//   z_i = scale * (x_i - max x),  S = sum_i exp(z_i)
//   log p_i = z_i - log S,  entropy = log S - (sum_i exp(z_i) z_i) / S
//
// in 32 bits; terms of x_i = -inf are 0.  The alternatives are the k largest
// x_i (scale > 0 keeps their order), equal ones by the lower index; -0 equals
// 0, NaN is above everything.  A row of -inf alone gives every token -inf and
// the entropy 0; a row with NaN or +inf gives NaN.
#include <hip/hip_runtime.h>

#include "common.hpp"
#include "kernels.hpp"

namespace mlxq {

namespace {

template <int XT>
__device__ __forceinline__ float load(const void* p, int64_t i) {
  if constexpr (XT == GEN_F32) return static_cast<const float*>(p)[i];
  else return xt_to_f32<XT == GEN_F16 ? 1 : 0>(static_cast<const uint16_t*>(p)[i]);
}

// The order of the alternatives as one unsigned number: the value's order,
// then the lower index.
__device__ __forceinline__ uint64_t order_key(float x, uint32_t i) {
  uint32_t u = __float_as_uint(x + 0.f);  // -0 becomes 0
  u = x != x ? 0xFF800001u : (u & 0x80000000u) ? ~u : u | 0x80000000u;
  return ((uint64_t)u << 32) | (uint32_t)~i;
}
__device__ __forceinline__ float key_value(uint64_t k) {
  const uint32_t u = (uint32_t)(k >> 32);
  return __uint_as_float(u & 0x80000000u ? u & 0x7FFFFFFFu : ~u);
}

template <int XT>
__global__ __launch_bounds__(256) void token_logprobs_kernel(const LogprobArgs a) {
  __shared__ uint64_t best[4];
  __shared__ float sums[8];
  const int tid = threadIdx.x, wave = tid >> 6;
  const int64_t t = blockIdx.x, row = t * a.row;
  // the largest key below `below`
  auto largest = [&](uint64_t below) -> uint64_t {
    uint64_t k = 0;
    for (int i = tid; i < a.V; i += 256) {
      const uint64_t v = order_key(load<XT>(a.logits, row + i), i);
      if (v < below && v > k) k = v;
    }
#pragma unroll
    for (int s = 32; s; s >>= 1) {
      const uint64_t o = __shfl_xor((unsigned long long)k, s);
      k = o > k ? o : k;
    }
    __syncthreads();
    if ((tid & 63) == 0) best[wave] = k;
    __syncthreads();
    for (int w = 0; w < 4; w++) k = best[w] > k ? best[w] : k;
    return k;
  };
  uint64_t key = largest(~0ull);
  const float m = key_value(key);
  float s = 0.f, e = 0.f;
  for (int i = tid; i < a.V; i += 256) {
    const float x = load<XT>(a.logits, row + i);
    const float z = x == m ? 0.f : a.scale * (x - m);
    if (x != -INFINITY) {
      const float p = expf(z);
      s += p;
      e += p == 0.f ? 0.f : p * z;
    }
  }
#pragma unroll
  for (int d = 32; d; d >>= 1) {
    s += __shfl_xor(s, d);
    e += __shfl_xor(e, d);
  }
  if ((tid & 63) == 0) {
    sums[wave] = s;
    sums[4 + wave] = e;
  }
  __syncthreads();
  s = (sums[0] + sums[1]) + (sums[2] + sums[3]);
  e = (sums[4] + sums[5]) + (sums[6] + sums[7]);
  const bool nothing = m == -INFINITY, bad = !(m < INFINITY);
  const float ls = logf(s);
  auto logprob = [&](float x) -> float {
    return bad ? NAN : x == -INFINITY ? -INFINITY : (x == m ? 0.f : a.scale * (x - m)) - ls;
  };
  for (int j = tid; j < a.n_tok; j += 256) {
    const int tok = a.tokens[t * a.n_tok + j];
    a.given[t * a.n_tok + j] = tok >= 0 && tok < a.V ? logprob(load<XT>(a.logits, row + tok)) : NAN;
  }
  if (tid == 0) a.entropy[t] = bad ? NAN : nothing ? 0.f : ls - e / s;
  for (int j = 0; j < a.k; j++) {
    if (j) key = largest(key);
    if (tid == 0) {
      a.top[t * a.k + j] = logprob(key_value(key));
      a.ids[t * a.k + j] = (int32_t)~(uint32_t)key;
    }
  }
}

}  // namespace

hipError_t launch_token_logprobs(const LogprobArgs& a, hipStream_t stream) {
  if (a.T == 0) return hipSuccess;
  if (a.V < 1 || a.k < 0 || a.k > kTopMax || a.k > a.V || a.T > 0x7FFFFFFF) return hipErrorInvalidValue;
  const dim3 grid((unsigned)a.T), block(256);
  if (a.type == GEN_BF16) hipLaunchKernelGGL(token_logprobs_kernel<GEN_BF16>, grid, block, 0, stream, a);
  else if (a.type == GEN_F16) hipLaunchKernelGGL(token_logprobs_kernel<GEN_F16>, grid, block, 0, stream, a);
  else hipLaunchKernelGGL(token_logprobs_kernel<GEN_F32>, grid, block, 0, stream, a);
  return hipGetLastError();
}

}  // namespace mlxq
