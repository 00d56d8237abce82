// rotary.hip — the position rotation of attention heads, alone or on the way
// into a paged key-value cache, on gfx950.
//
//   (a, b) -> factor (a cos t - b sin t, b cos t + a sin t),  t = position * inv_freq[i]
//
// for pairs i < n of a head: elements (i, n + i), or (2 i, 2 i + 1) interleaved;
// the elements from 2 n on are copied.  An element is read and written once,
// which is the bound; a workgroup takes one token's heads, so a token's n
// angles are worked out once for all of them and shared through LDS, while 16 bytes (32 of
// a pair of halves) a thread are on their way: 8191 tokens of 32 heads of 96 in 16 bits
// (101 MB) 23.3 us a launch among others, 4.3 TB/s (24.6 traced); with the loads behind the
// angles 24.0.  A thread for two (four) heads, so half (a quarter) of the angles and
// workgroups: 1.05 (1.4) times as long.
//
// The angle of a far position needs more than 32 bits (2^20 * 1.0f is off by
// whole steps of 1/16): it is taken in turns in 64 bits, whole turns and
// quarters of one come off exactly, and what is left, at most an eighth of a
// turn, goes through the power series of sine and cosine in 32 bits (terms up to
// x^9 and x^10: the next is below 2^-28).
#include <hip/hip_runtime.h>

#include "common.hpp"
#include "kernels.hpp"

namespace mlxq {

namespace {

// cos and sin of `turns` turns
__device__ __forceinline__ float2 cos_sin(double turns) {
  turns -= rint(turns);
  const double quarter = rint(4.0 * turns);
  const float x = (float)((turns - 0.25 * quarter) * 6.283185307179586476925), y = x * x;
  float s = 1.f / 362880, c = -1.f / 3628800;
  s = fmaf(s, y, -1.f / 5040);
  s = fmaf(s, y, 1.f / 120);
  s = fmaf(s, y, -1.f / 6);
  s = fmaf(s * y, x, x);
  c = fmaf(c, y, 1.f / 40320);
  c = fmaf(c, y, -1.f / 720);
  c = fmaf(c, y, 1.f / 24);
  c = fmaf(c, y, -0.5f);
  c = fmaf(c, y, 1.f);
  const int q = (int)quarter & 3;
  const float cs = q & 1 ? s : c, sn = q & 1 ? c : s;
  return float2{q == 1 || q == 2 ? -cs : cs, q & 2 ? -sn : sn};
}

template <int XT>
struct Element {
  using T = uint16_t;
  static __device__ float up(T v) { return xt_to_f32<XT == GEN_F16 ? 1 : 0>(v); }
  static __device__ T down(float v) { return (T)f32_to_xt<XT == GEN_F16 ? 1 : 0>(v); }
};
template <>
struct Element<GEN_F32> {
  using T = float;
  static __device__ float up(T v) { return v; }
  static __device__ T down(float v) { return v; }
};

// A head's units of 16 bytes: those of its pairs (half layout: W pairs, two
// vectors; interleaved: W / 2 pairs, one vector), then those of the rest; the
// last of each may be part full.  Rows of any stride: 16 bytes of element alignment.
__host__ __device__ inline int rotary_units(const RotaryArgs& a, int W) {
  return ((a.interleaved ? 2 * a.n : a.n) + W - 1) / W + (a.D - 2 * a.n + W - 1) / W;
}

template <int XT, bool INTER>
__global__ __launch_bounds__(256) void rotary_kernel(const RotaryArgs a) {
  using E = Element<XT>;
  using T = typename E::T;
  constexpr int W = 16 / sizeof(T);
  typedef T Vec __attribute__((ext_vector_type(W), aligned(sizeof(T))));
  extern __shared__ float2 turn[];  // [n] factor * (cos, sin)
  const int tid = threadIdx.x, unit = tid & ((1 << a.unit_shift) - 1);
  const int pairs = INTER ? 2 * a.n : a.n, rot = (pairs + W - 1) / W, units = rotary_units(a, W);
  const int at = blockIdx.y * (256 >> a.unit_shift) + (tid >> a.unit_shift), heads = a.Hq + 2 * a.Hkv;
  const float freq = tid < a.n ? a.inv_freq[tid] : 0.f;
  // first element of unit u, and whether all of it is there
  auto first_of = [&](int u) -> int { return u < rot ? u * W : 2 * a.n + (u - rot) * W; };
  auto whole = [&](int u) -> bool { return (u < rot ? pairs : a.D) - first_of(u) >= W; };
  // tokens without a sign: the step past the last of 2^31 - 1 stays below 2^32
  for (uint32_t t = blockIdx.x; t < (uint32_t)a.T; t += gridDim.x) {
    const int pos = a.positions[t];
    // where the token's keys and values go (-1: nowhere)
    int pid = -1, off = 0;
    if (a.Hkv > 0) {
      const int row = a.rows[t];
      if (row >= 0 && row < a.table_rows && pos >= 0 && pos / a.page < a.width && !(a.lengths && pos >= a.lengths[row])) {
        pid = a.table[row * a.table_row + pos / a.page];
        off = pos % a.page;
        if (pid >= a.pages) pid = -1;
      }
    }
    const int kind = at < a.Hq ? 0 : at < a.Hq + a.Hkv ? 1 : 2, h = at - (kind == 0 ? 0 : kind == 1 ? a.Hq : a.Hq + a.Hkv);
    const T* src = static_cast<const T*>(kind == 0 ? a.q : kind == 1 ? a.k : a.v) +
                   (kind == 0 ? t * a.q_tok + h * a.q_head : kind == 1 ? t * a.k_tok + h * a.k_head : t * a.v_tok + h * a.v_head);
    Vec v, w;
    auto load = [&](int u) {
      v = *reinterpret_cast<const Vec*>(src + first_of(u));
      if (!INTER && u < rot) w = *reinterpret_cast<const Vec*>(src + a.n + first_of(u));
    };
    // a thread's first unit is on its way while the angles are worked out
    if (at < heads && unit < units && whole(unit)) load(unit);
    for (int i = tid; i < a.n; i += 256) {
      const float2 r = cos_sin((double)pos * ((double)(i == tid ? freq : a.inv_freq[i]) * 0.15915494309189533577));
      turn[i] = float2{r.x * a.factor, r.y * a.factor};
    }
    __syncthreads();
    auto rotate = [&](T& x, T& y, int i) {
      const float2 r = turn[i];
      const float p = E::up(x), q = E::up(y);
      x = E::down(p * r.x - q * r.y);
      y = E::down(q * r.x + p * r.y);
    };
    if (at < heads && (kind == 0 || pid >= 0)) {
      T* dst = static_cast<T*>(kind == 0 ? a.out : kind == 1 ? a.kp : a.vp) +
               (kind == 0   ? t * a.out_tok + h * a.out_head
                : kind == 1 ? pid * a.kp_page + h * a.kp_head + off * a.kp_tok
                            : pid * a.vp_page + h * a.vp_head + off * a.vp_tok);
      const bool turned = kind < 2;
      for (int u = unit; u < units; u += 1 << a.unit_shift) {
        const int e0 = first_of(u);
        if (whole(u)) {
          if (u != unit) load(u);
          if (turned && u < rot) {
#pragma unroll
            for (int e = 0; e < W; e += INTER ? 2 : 1) {
              T x = v[e], y = INTER ? v[e + 1] : w[e];
              rotate(x, y, INTER ? (e0 + e) / 2 : e0 + e);
              v[e] = x;
              if constexpr (INTER) v[e + 1] = y;
              else w[e] = y;
            }
          }
          *reinterpret_cast<Vec*>(dst + e0) = v;
          if (!INTER && u < rot) *reinterpret_cast<Vec*>(dst + a.n + e0) = w;
        } else if (u >= rot) {
          for (int e = e0; e < a.D; e++) dst[e] = src[e];
        } else {
          for (int e = e0; e < pairs; e += INTER ? 2 : 1) {
            const int other = INTER ? e + 1 : a.n + e;
            T x = src[e], y = src[other];
            if (turned) rotate(x, y, INTER ? e / 2 : e);
            dst[e] = x;
            dst[other] = y;
          }
        }
      }
    }
    __syncthreads();  // the angles are free again
  }
}

template <int XT>
void launch(RotaryArgs a, hipStream_t stream) {
  a.unit_shift = 0;
  while (a.unit_shift < 8 && (1 << a.unit_shift) < rotary_units(a, XT == GEN_F32 ? 4 : 8)) a.unit_shift++;
  const int heads = a.Hq + 2 * a.Hkv, per = 256 >> a.unit_shift;
  const dim3 grid((unsigned)(a.T < (1 << 20) ? a.T : 1 << 20), (unsigned)((heads + per - 1) / per));
  const size_t lds = (size_t)a.n * sizeof(float2);
  if (a.interleaved) hipLaunchKernelGGL((rotary_kernel<XT, true>), grid, dim3(256), lds, stream, a);
  else hipLaunchKernelGGL((rotary_kernel<XT, false>), grid, dim3(256), lds, stream, a);
}

}  // namespace

hipError_t launch_rotary(const RotaryArgs& a, hipStream_t stream) {
  if (a.T == 0 || a.D == 0 || a.Hq + a.Hkv == 0) return hipSuccess;
  if (a.n < 0 || 2 * a.n > a.D || a.D > kRotaryMaxD || a.Hq + 2 * a.Hkv > kRotaryMaxHeads) return hipErrorInvalidValue;
  if (a.Hkv > 0 && (a.pages < 1 || a.page < 1)) return hipErrorInvalidValue;
  if (a.type == GEN_BF16) launch<GEN_BF16>(a, stream);
  else if (a.type == GEN_F16) launch<GEN_F16>(a, stream);
  else launch<GEN_F32>(a, stream);
  return hipGetLastError();
}

}  // namespace mlxq
