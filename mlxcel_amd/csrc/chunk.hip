// chunk.hip — attention of several new tokens per sequence over a paged
// key-value cache on gfx950.
//
//   s_j = cap(q_i . k_j * scale)   over the keys j that token i sees: (p - window, p], p = length - new + i
//   o_i = sum_j exp(s_j - m) v_j / (sum_j exp(s_j - m) + exp(sink - m))
//
// One wave a token and query head: a lane scores one of 64 keys at a time, then
// holds some columns of the result while the 64 probabilities go round.
#include <hip/hip_runtime.h>

#include "common.hpp"
#include "kernels.hpp"
#include "wave.hpp"

namespace mlxq {

namespace {

constexpr float kLog2e = 1.44269504088896340736f;

template <int XT>
__device__ __forceinline__ float element(const void* p, int64_t i) {
  if constexpr (XT == GEN_F32) return static_cast<const float*>(p)[i];
  else return xt_to_f32<XT == GEN_F16 ? 1 : 0>(static_cast<const uint16_t*>(p)[i]);
}
template <int XT>
__device__ __forceinline__ void store_element(void* p, int64_t i, float v) {
  if constexpr (XT == GEN_F32) static_cast<float*>(p)[i] = v;
  else static_cast<uint16_t*>(p)[i] = (uint16_t)f32_to_xt<XT == GEN_F16 ? 1 : 0>(v);
}
__device__ __forceinline__ float exp2_diff(float a, float b) {
  return __builtin_amdgcn_exp2f(a - (b == -INFINITY ? 0.f : b));
}

template <int XT>
__global__ __launch_bounds__(256) void chunk_attention_kernel(const ChunkAttnArgs a) {
  __shared__ float qs[4][256];
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int64_t unit = (int64_t)blockIdx.x * 4 + wave;
  const bool mine = unit < (int64_t)a.T * a.Hq;
  const int t = mine ? (int)(unit / a.Hq) : 0, h = mine ? (int)(unit % a.Hq) : 0;
  for (int d = lane; d < a.D; d += 64) qs[wave][d] = element<XT>(a.q, t * a.q_tok + h * a.q_head + d);
  __syncthreads();
  if (!mine) return;
  // the last sequence that starts at or before t
  int lo = 0, hi = a.B;
  while (lo < hi) {
    const int mid = (lo + hi) / 2;
    if (a.starts[mid] <= t) lo = mid + 1;
    else hi = mid;
  }
  const int b = lo - 1;
  if (b < 0 || t >= a.starts[b + 1]) return;
  const int64_t cap = (int64_t)a.width * a.page;
  const int len = (int)min((int64_t)max(a.lengths[b], 0), cap);
  const int p = len - (a.starts[b + 1] - t), k1 = p + 1, k0 = a.window > 0 ? max(0, k1 - a.window) : 0;
  const int kh = h / (a.Hq / a.Hkv);
  float m = -INFINITY, l = 0.f, o[4] = {0.f, 0.f, 0.f, 0.f};
  for (int k = k0; k < k1; k += 64) {
    const int key = min(k + lane, k1 - 1);
    const int pid = min(max(a.table[b * a.table_row + key / a.page], 0), a.pages - 1), off = key % a.page;
    float s = 0.f;
    for (int d = 0; d < a.D; d++)
      s = fmaf(qs[wave][d], element<XT>(a.k, pid * a.k_page + kh * a.k_head + off * a.k_tok + d), s);
    s *= a.scale;
    if (a.softcap > 0.f) s = a.softcap * tanhf(s / a.softcap);
    s = k + lane < k1 ? s * kLog2e : -INFINITY;
    const float M = fmaxf(m, wave_max(s, lane)), f = exp2_diff(m, M), e = exp2_diff(s, M);
    m = M;
    l = l * f + wave_sum(e, lane);
    for (int i = 0; i < 4; i++) o[i] *= f;
    for (int j = 0; j < min(64, k1 - k); j++) {
      const float w = __shfl(e, j);
      const int vp = __shfl(pid, j), vo = __shfl(off, j);
      for (int i = 0; i < 4; i++)
        if (lane + 64 * i < a.D)
          o[i] = fmaf(w, element<XT>(a.v, vp * a.v_page + kh * a.v_head + vo * a.v_tok + lane + 64 * i), o[i]);
    }
  }
  if (a.sinks && k1 > k0) {
    const float sink = a.sinks[h] * kLog2e, M = fmaxf(m, sink), f = exp2_diff(m, M);
    l = l * f + exp2_diff(sink, M);
    for (int i = 0; i < 4; i++) o[i] *= f;
  }
  for (int i = 0; i < 4; i++)
    if (lane + 64 * i < a.D)
      store_element<XT>(a.out, ((int64_t)t * a.Hq + h) * a.D + lane + 64 * i, k1 > k0 ? o[i] / l : 0.f);
}

}  // namespace

hipError_t launch_chunk_attention(const ChunkAttnArgs& a, hipStream_t stream) {
  if (a.T == 0 || a.B == 0) return hipSuccess;
  if (a.D < 8 || a.D > 256 || a.D % 8 || a.pages < 1 || a.page < 1) return hipErrorInvalidValue;
  const int64_t wgs = ((int64_t)a.T * a.Hq + 3) / 4;
  if (wgs > kMaxGroups) return hipErrorInvalidValue;
  auto run = [&](auto kernel) { hipLaunchKernelGGL(kernel, dim3((unsigned)wgs), dim3(256), 0, stream, a); };
  if (a.type == GEN_BF16) run(chunk_attention_kernel<GEN_BF16>);
  else if (a.type == GEN_F16) run(chunk_attention_kernel<GEN_F16>);
  else run(chunk_attention_kernel<GEN_F32>);
  return hipGetLastError();
}

}  // namespace mlxq
