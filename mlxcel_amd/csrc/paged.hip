// paged.hip — attention of one new token per sequence over a paged key-value
// cache on gfx950.
//
//   s_t = cap(q . k_t * scale)   over the sequence's keys t in [lo, hi)
//   o   = sum_t exp(s_t - m) v_t / (sum_t exp(s_t - m) + exp(sink - m))
//
// with hi the length, lo = hi - window (0 without one), cap(s) = s or
// c tanh(s / c), m the largest s_t (and sink).  Each key and value is read
// once; that read is the bound (4 D operations a byte pair and query head stay
// far under the matrix rate).
//
// One workgroup takes one sequence and key head; its waves take tiles of 16
// keys in turn, each with a running maximum and sum of its own, and join them
// in LDS at the end.  Both products run on MFMA with the layouts chosen so that
// nothing moves between them:
//   S^T[key][head] = K Q^T: lane (c, g) = (lane % 16, lane / 16) loads 16 bytes
//     of key c, so the tile's keys are read in 16 rows of 64 contiguous bytes;
//     it ends with the scores of keys 4 g + r (r < 4) of head c.
//   O^T[d][head] += V^T P^T in 32-bit MFMAs of 4 keys: step r takes keys
//     4 g + r, for which lane (c, g) already holds P of head c; it loads V of
//     key 4 g + r, columns VE c .. VE c + VE - 1, so a key's row is read as one
//     contiguous run.  Accumulator j is column VE c + j, rows 4 g + r' of
//     O^T: d = VE (4 g + r') + j, head c, the lane whose maximum rescales it.
// P stays in 32 bits (no rounding of probabilities); the 32-bit MFMAs cost
// 64 cycles a key of 128 columns on one SIMD where the read of a key takes a
// CU 64 cycles, a quarter of the four SIMDs' time.
#include <hip/hip_runtime.h>

#include "common.hpp"
#include "kernels.hpp"

namespace mlxq {

namespace {

constexpr int kWaves = 4;
constexpr float kLog2e = 1.44269504088896340736f;

// 16- and 8-byte loads of element alignment (rows of any stride)
typedef uint32_t u32x4_e __attribute__((ext_vector_type(4), aligned(2)));
typedef uint32_t u32x2_e __attribute__((ext_vector_type(2), aligned(2)));

// XT: GEN_BF16 / GEN_F16 / GEN_F32.  DP: head width rounded up.
template <int XT, int DP>
struct Geo {
  static constexpr bool F32 = XT == GEN_F32;
  static constexpr int ES = F32 ? 4 : 2;
  static constexpr int KE = 16 / ES;               // elements of a 16-byte load
  static constexpr int KC = DP / (4 * KE);         // K loads of a lane: d = 4 KE c + KE g
  static constexpr int VE = F32 || DP <= 64 ? 4 : 8;
  static constexpr int NB = (DP + 16 * VE - 1) / (16 * VE);  // V loads of a lane and key
  static constexpr int VW = VE * ES / 4;           // words of one
  static constexpr int LD = DP + 4;                // LDS row of O (floats)
};

template <int XT>
__device__ __forceinline__ float element(uint32_t w, int hi) {
  if constexpr (XT == GEN_BF16) return __uint_as_float(hi ? w & 0xFFFF0000u : w << 16);
  else if constexpr (XT == GEN_F16) return (float)__builtin_bit_cast(_Float16, (uint16_t)(hi ? w >> 16 : w & 0xFFFFu));
  else return __uint_as_float(w);
}

template <int XT>
__device__ __forceinline__ void store_element(void* p, int64_t i, float v) {
  if constexpr (XT == GEN_F32) static_cast<float*>(p)[i] = v;
  else static_cast<uint16_t*>(p)[i] = (uint16_t)f32_to_xt<XT == GEN_F16 ? 1 : 0>(v);
}

// exp2(a - b), 0 where a is -inf (also where b is)
__device__ __forceinline__ float exp2_diff(float a, float b) {
  return __builtin_amdgcn_exp2f(a - (b == -INFINITY ? 0.f : b));
}

template <int XT, int DP>
__global__ __launch_bounds__(256) void paged_attention_kernel(const PagedAttnArgs a) {
  using G = Geo<XT, DP>;
  extern __shared__ float lds[];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, c = lane & 15, g = lane >> 4;
  const int per = a.Hq / a.Hkv, tiles_h = (per + 15) / 16;
  int id = blockIdx.x;
  const int ht = id % tiles_h;
  id /= tiles_h;
  const int hk = id % a.Hkv, b = id / a.Hkv;
  const int heads = min(16, per - 16 * ht);  // of this workgroup
  const int head0 = hk * per + 16 * ht;
  const int64_t cap = (int64_t)a.width * a.page;
  const int hi = (int)min((int64_t)max(a.lengths[b], 0), cap);
  const int lo = a.window > 0 ? max(0, hi - a.window) : 0;

  // Q of head c: B operand, the d order of the K loads
  uint32_t q[G::KC][4];
  {
    const char* qp = static_cast<const char*>(a.q) + (b * a.q_b + (head0 + min(c, heads - 1)) * a.q_h) * G::ES;
#pragma unroll
    for (int i = 0; i < G::KC; i++) {
      const int d = 4 * G::KE * i + G::KE * g;
      const u32x4_e w = *reinterpret_cast<const u32x4_e*>(qp + (d < a.D ? d : 0) * G::ES);
#pragma unroll
      for (int e = 0; e < 4; e++) q[i][e] = d < a.D ? w[e] : 0u;
    }
  }
  const int32_t* table = a.table + b * a.table_row;
  const char* kb = static_cast<const char*>(a.k) + hk * a.k_head * G::ES;
  const char* vb = static_cast<const char*>(a.v) + hk * a.v_head * G::ES;

  f32x4 o[G::NB][G::VE];
#pragma unroll
  for (int i = 0; i < G::NB; i++)
#pragma unroll
    for (int j = 0; j < G::VE; j++) o[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
  float m = -INFINITY, l = 0.f;

  const int t1 = (hi + 15) / 16;
  for (int t = lo / 16 + wave; t < t1; t += kWaves) {
    // the lane's key, inside the sequence (rows past its ends are never read)
    const int key = min(max(16 * t + c, lo), hi - 1);
    const int slot = key / a.page, off = key - slot * a.page;
    const int pid = min(max(table[slot], 0), a.pages - 1);
    const char* kp = kb + (pid * a.k_page + off * a.k_tok) * G::ES;
    uint32_t kr[G::KC][4];
#pragma unroll
    for (int i = 0; i < G::KC; i++) {
      const int d = 4 * G::KE * i + G::KE * g;
      const u32x4_e w = *reinterpret_cast<const u32x4_e*>(kp + (d < a.D ? d : 0) * G::ES);
#pragma unroll
      for (int e = 0; e < 4; e++) kr[i][e] = w[e];
      if (DP != a.D) {  // columns past the head are zero on both sides
#pragma unroll
        for (int e = 0; e < 4; e++) kr[i][e] = d < a.D ? kr[i][e] : 0u;
      }
    }
    const bool whole = 16 * t >= lo && 16 * t + 16 <= hi;
    uint32_t vr[4][G::NB][G::VW];
#pragma unroll
    for (int r = 0; r < 4; r++) {
      const int vpid = __shfl(pid, 4 * g + r), voff = __shfl(off, 4 * g + r);
      const char* vp = vb + (vpid * a.v_page + voff * a.v_tok) * G::ES;
      const int vkey = 16 * t + 4 * g + r;
      const bool live = whole || (vkey >= lo && vkey < hi);
#pragma unroll
      for (int i = 0; i < G::NB; i++) {
        const int d = 16 * G::VE * i + G::VE * c;
        const char* p = vp + (d < a.D ? d : 0) * G::ES;  // columns past the head are dropped at the end
        if constexpr (G::VW == 4) {
          const u32x4_e w = *reinterpret_cast<const u32x4_e*>(p);
#pragma unroll
          for (int e = 0; e < 4; e++) vr[r][i][e] = live ? w[e] : 0u;
        } else {
          const u32x2_e w = *reinterpret_cast<const u32x2_e*>(p);
#pragma unroll
          for (int e = 0; e < 2; e++) vr[r][i][e] = live ? w[e] : 0u;
        }
      }
    }

    f32x4 s = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < G::KC; i++) {
      if constexpr (G::F32) {
#pragma unroll
        for (int e = 0; e < 4; e++)
          s = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(kr[i][e]), __uint_as_float(q[i][e]), s, 0, 0, 0);
      } else {
        s = mfma16x16x32_xt<XT == GEN_F16 ? 1 : 0>(u32x4{kr[i][0], kr[i][1], kr[i][2], kr[i][3]},
                                                   u32x4{q[i][0], q[i][1], q[i][2], q[i][3]}, s);
      }
    }
    float mt = m;
#pragma unroll
    for (int r = 0; r < 4; r++) {
      float x = s[r] * a.scale;
      if (a.softcap > 0.f) x = a.softcap * tanhf(x / a.softcap);
      x *= kLog2e;
      const int sk = 16 * t + 4 * g + r;
      s[r] = whole || (sk >= lo && sk < hi) ? x : -INFINITY;
      mt = fmaxf(mt, s[r]);
    }
    mt = fmaxf(mt, __shfl_xor(mt, 16));
    mt = fmaxf(mt, __shfl_xor(mt, 32));
    const float f = exp2_diff(m, mt);
    m = mt;
    l *= f;
#pragma unroll
    for (int i = 0; i < G::NB; i++)
#pragma unroll
      for (int j = 0; j < G::VE; j++)
#pragma unroll
        for (int r = 0; r < 4; r++) o[i][j][r] *= f;
#pragma unroll
    for (int r = 0; r < 4; r++) {
      const float p = exp2_diff(s[r], m);
      l += p;
#pragma unroll
      for (int i = 0; i < G::NB; i++)
#pragma unroll
        for (int j = 0; j < G::VE; j++) {
          const float v = element<XT>(vr[r][i][G::F32 ? j : j >> 1], j & 1);
          o[i][j] = __builtin_amdgcn_mfma_f32_16x16x4f32(v, p, o[i][j], 0, 0, 0);
        }
    }
  }
  l += __shfl_xor(l, 16);
  l += __shfl_xor(l, 32);

  // join the waves: O rows [wave][head][LD], then (m, l) [wave][16][2]
  float* ml = lds + kWaves * heads * G::LD;
  if (c < heads) {
    float* row = lds + (wave * heads + c) * G::LD;
#pragma unroll
    for (int i = 0; i < G::NB; i++)
#pragma unroll
      for (int r = 0; r < 4; r++) {
        const int d = 16 * G::VE * i + G::VE * (4 * g + r);
        if (d < DP) {
#pragma unroll
          for (int j = 0; j < G::VE; j++) row[d + j] = o[i][j][r];
        }
      }
    if (g == 0) {
      ml[(wave * 16 + c) * 2] = m;
      ml[(wave * 16 + c) * 2 + 1] = l;
    }
  }
  __syncthreads();
  for (int e = threadIdx.x; e < heads * a.D; e += 256) {
    const int h = e / a.D, d = e - h * a.D;
    float M = -INFINITY, L = 0.f, acc = 0.f;
#pragma unroll
    for (int w = 0; w < kWaves; w++) M = fmaxf(M, ml[(w * 16 + h) * 2]);
    const float sink = a.sinks ? a.sinks[head0 + h] * kLog2e : -INFINITY;
    M = fmaxf(M, sink);
#pragma unroll
    for (int w = 0; w < kWaves; w++) {
      const float f = exp2_diff(ml[(w * 16 + h) * 2], M);
      L += f * ml[(w * 16 + h) * 2 + 1];
      acc += f * lds[(w * heads + h) * G::LD + d];
    }
    if (a.sinks) L += exp2_diff(sink, M);
    store_element<XT>(a.out, ((int64_t)b * a.Hq + head0 + h) * a.D + d, L == 0.f ? 0.f : acc / L);
  }
}

template <int XT, int DP>
hipError_t launch(const PagedAttnArgs& a, hipStream_t stream) {
  const int per = a.Hq / a.Hkv, heads = per < 16 ? per : 16;
  const int64_t wgs = (int64_t)a.B * a.Hkv * ((per + 15) / 16);
  if (wgs > 0x7FFFFFFF) return hipErrorInvalidValue;
  const size_t bytes = (size_t)(kWaves * heads * Geo<XT, DP>::LD + kWaves * 32) * sizeof(float);
  hipLaunchKernelGGL((paged_attention_kernel<XT, DP>), dim3((unsigned)wgs), dim3(256), bytes, stream, a);
  return hipGetLastError();
}

template <int XT>
hipError_t launch_width(const PagedAttnArgs& a, hipStream_t stream) {
  if (a.D <= 64) return launch<XT, 64>(a, stream);
  if (a.D <= 96) return launch<XT, 96>(a, stream);
  if (a.D <= 128) return launch<XT, 128>(a, stream);
  if (a.D <= 192) return launch<XT, 192>(a, stream);
  return launch<XT, 256>(a, stream);
}

}  // namespace

hipError_t launch_paged_attention(const PagedAttnArgs& a, hipStream_t stream) {
  if (a.B == 0) return hipSuccess;
  if (a.D < 8 || a.D > 256 || a.D % 8 || a.pages < 1 || a.page < 1) return hipErrorInvalidValue;
  if (a.type == GEN_BF16) return launch_width<GEN_BF16>(a, stream);
  if (a.type == GEN_F16) return launch_width<GEN_F16>(a, stream);
  return launch_width<GEN_F32>(a, stream);
}

}  // namespace mlxq
