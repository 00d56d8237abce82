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
// The work is cut evenly whatever the lengths: with a sequence's keys counted
// in steps of 64 for each key head (and each 16 of its query heads), workgroup w
// takes steps [w n, (w + 1) n) of them all.  The lengths are on the device, so
// each workgroup finds its first step from a scan over them.  A sequence's head
// that crosses a workgroup's end leaves its sum, maximum and output so far in
// scratch; the last of its workgroups to arrive joins them, in the order of the
// keys, so the result does not depend on who came last.
//
// In a step each wave takes 16 keys, with a running maximum and sum of its own;
// the waves are joined in LDS at a head's end.  The next 16 keys are loaded
// right after the product that used up these ones' registers, and their page
// numbers one step before that, so a wave keeps 4 to 8 KiB in flight (D = 128,
// 16 bits).  Both products run on MFMA with the layouts chosen so that nothing
// moves between them:
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

#include <algorithm>
#include <type_traits>

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
  // Workgroups a CU holds: by registers (K, V, Q and O of a lane)
  static constexpr int WGS = DP * ES <= 128 ? 4 : DP * ES <= 256 ? 3 : DP * ES <= 512 ? 2 : 1;
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

constexpr int kStep = 16 * kWaves;  // keys of a step

// First 16-key tile and number of steps of a sequence.
__device__ __forceinline__ int steps_of(int len, int64_t cap, int window, int& lo, int& hi) {
  hi = (int)min((int64_t)max(len, 0), cap);
  lo = window > 0 ? max(0, hi - window) : 0;
  const int tiles = (hi + 15) / 16 - lo / 16;
  return (tiles + kWaves - 1) / kWaves;
}

// Words of one partial result: O [heads][DP], then (m, l) [heads][2].
constexpr int part_words(int heads, int DP) { return heads * (DP + 2); }

template <int XT, int DP>
__global__ __launch_bounds__(256, (Geo<XT, DP>::WGS)) void paged_attention_kernel(const PagedAttnArgs a) {
  using G = Geo<XT, DP>;
  extern __shared__ __align__(16) float lds[];
  __shared__ u32x4 qs[G::KC * 64];
  __shared__ int64_t scan[kWaves];
  __shared__ int64_t first_off;  // of this workgroup's first step in its sequence
  __shared__ int first_b;
  __shared__ uint32_t arrived;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int c = lane & 15, g = lane >> 4;
  const int per = a.Hq / a.Hkv, tiles_h = (per + 15) / 16;
  const int64_t cap = (int64_t)a.width * a.page;
  const int heads_b = a.Hkv * tiles_h;  // (key head, 16 query heads) of a sequence

  // the sequences' steps: thread i sums those of its share
  int64_t total, n, at, end;
  {
    const int share = (a.B + 255) / 256, b0 = min(tid * share, a.B), b1 = min(b0 + share, a.B);
    int64_t mine = 0;
    int lo, hi;
    for (int b = b0; b < b1; b++) mine += (int64_t)heads_b * steps_of(a.lengths[b], cap, a.window, lo, hi);
    int64_t sum = mine;
#pragma unroll
    for (int s = 1; s < 64; s <<= 1) {
      const int64_t o = __shfl_up((long long)sum, s);
      if (lane >= s) sum += o;
    }
    if (lane == 63) scan[wave] = sum;
    __syncthreads();
    int64_t before = sum - mine;
    total = 0;
#pragma unroll
    for (int w = 0; w < kWaves; w++) {
      if (w < wave) before += scan[w];
      total += scan[w];
    }
    n = max((total + a.wgs - 1) / a.wgs, (int64_t)a.least);
    at = blockIdx.x * n;
    end = min(at + n, total);
    if (at < end && before <= at && at < before + mine) {
      int64_t off = at - before;
      int b = b0;
      for (;; b++) {
        const int64_t s = (int64_t)heads_b * steps_of(a.lengths[b], cap, a.window, lo, hi);
        if (off < s) break;
        off -= s;
      }
      first_b = b;
      first_off = off;
    }
    __syncthreads();
  }
  // a sequence without keys has no steps: its output is zeros
  for (int b = blockIdx.x; b < a.B; b += a.wgs) {
    int lo, hi;
    if (steps_of(a.lengths[b], cap, a.window, lo, hi) == 0)
      for (int i = tid; i < a.Hq * a.D; i += 256) store_element<XT>(a.out, (int64_t)b * a.Hq * a.D + i, 0.f);
  }
  if (at >= end) return;
  int b = __builtin_amdgcn_readfirstlane(first_b);
  int64_t off = first_off;
  const __amdgpu_buffer_rsrc_t parts = buffer_rsrc(a.part, (uint32_t)((int64_t)2 * a.wgs * part_words(min(per, 16), DP) * 4));

  while (at < end) {
    int lo, hi;
    const int steps = steps_of(a.lengths[b], cap, a.window, lo, hi);
    if (steps == 0 || off >= (int64_t)steps * heads_b) {
      b++;
      off = 0;
      continue;
    }
    const int hh = (int)(off / steps), s0 = (int)(off - (int64_t)hh * steps);
    const int s1 = (int)min((int64_t)steps, s0 + (end - at));
    const int hk = hh / tiles_h, ht = hh - hk * tiles_h;
    const int heads = min(16, per - 16 * ht), head0 = hk * per + 16 * ht;

    // Q of head c in LDS, a lane's 16 bytes after the other: B operand, the d
    // order of the K loads
    for (int i = wave; i < G::KC; i += kWaves) {
      const char* qp = static_cast<const char*>(a.q) + (b * a.q_b + (head0 + min(c, heads - 1)) * a.q_h) * G::ES;
      const int d = 4 * G::KE * i + G::KE * g;
      const u32x4_e w = *reinterpret_cast<const u32x4_e*>(qp + (d < a.D ? d : 0) * G::ES);
      qs[i * 64 + lane] = d < a.D ? u32x4{w[0], w[1], w[2], w[3]} : u32x4{0u, 0u, 0u, 0u};
    }
    __syncthreads();
    const int32_t* table = a.table + b * a.table_row;
    const char* kb = static_cast<const char*>(a.k) + hk * a.k_head * G::ES;
    const char* vb = static_cast<const char*>(a.v) + hk * a.v_head * G::ES;

    f32x4 o[G::NB][G::VE];
#pragma unroll
    for (int i = 0; i < G::NB; i++)
#pragma unroll
      for (int j = 0; j < G::VE; j++) o[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    float m = -INFINITY, l = 0.f;
    uint32_t kr[G::KC][4], vr[4][G::NB][G::VW];
    int pid = 0, pid_next = 0, key_off = 0;

    // the lane's key of tile t, inside the sequence (rows past its ends are never read)
    auto page_of = [&](int t, int& in_page) -> int {
      const int key = min(max(16 * t + c, lo), hi - 1);
      const int slot = (int)(((uint64_t)(uint32_t)key * a.page_mul) >> a.page_shift);
      in_page = key - slot * a.page;
      return slot;
    };
    auto load_k = [&]() {
      const char* kp = kb + (pid * a.k_page + key_off * a.k_tok) * G::ES;
#pragma unroll
      for (int i = 0; i < G::KC; i++) {
        const int d = 4 * G::KE * i + G::KE * g;
        const u32x4_e w = *reinterpret_cast<const u32x4_e*>(kp + (d < a.D ? d : 0) * G::ES);
#pragma unroll
        for (int e = 0; e < 4; e++) kr[i][e] = w[e];
      }
    };
    auto load_v = [&]() {
#pragma unroll
      for (int r = 0; r < 4; r++) {
        const int vpid = __shfl(pid, 4 * g + r), voff = __shfl(key_off, 4 * g + r);
        const char* vp = vb + (vpid * a.v_page + voff * a.v_tok) * G::ES;
#pragma unroll
        for (int i = 0; i < G::NB; i++) {
          const int d = 16 * G::VE * i + G::VE * c;
          const char* p = vp + (d < a.D ? d : 0) * G::ES;  // columns past the head are dropped at the end
          if constexpr (G::VW == 4) {
            const u32x4_e w = *reinterpret_cast<const u32x4_e*>(p);
#pragma unroll
            for (int e = 0; e < 4; e++) vr[r][i][e] = w[e];
          } else {
            const u32x2_e w = *reinterpret_cast<const u32x2_e*>(p);
#pragma unroll
            for (int e = 0; e < 2; e++) vr[r][i][e] = w[e];
          }
        }
      }
    };
    auto page_id = [&](int slot) { return min(max(table[slot], 0), a.pages - 1); };

    // this wave's tiles of the segment
    const int t0 = lo / 16 + s0 * kWaves + wave, t1 = min((hi + 15) / 16, lo / 16 + s1 * kWaves);
    if (t0 < t1) {
      const int slot = page_of(t0, key_off);
      int unused;
      const int slot2 = t0 + kWaves < t1 ? page_of(t0 + kWaves, unused) : slot;
      pid = page_id(slot);
      pid_next = page_id(slot2);
      load_k();
      load_v();
    }
    for (int t = t0; t < t1; t += kWaves) {
      const bool whole = 16 * t >= lo && 16 * t + 16 <= hi, more = t + kWaves < t1;
      if (DP != a.D) {  // columns past the head are zero on both sides
#pragma unroll
        for (int i = 0; i < G::KC; i++)
#pragma unroll
          for (int e = 0; e < 4; e++) kr[i][e] = 4 * G::KE * i + G::KE * g < a.D ? kr[i][e] : 0u;
      }
      f32x4 s = {0.f, 0.f, 0.f, 0.f};
      asm volatile("" ::: "memory");  // Q is read again each tile, not kept in registers
#pragma unroll
      for (int i = 0; i < G::KC; i++) {
        const u32x4 q = qs[i * 64 + lane];
        if constexpr (G::F32) {
#pragma unroll
          for (int e = 0; e < 4; e++)
            s = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(kr[i][e]), __uint_as_float(q[e]), s, 0, 0, 0);
        } else {
          s = mfma16x16x32_xt<XT == GEN_F16 ? 1 : 0>(u32x4{kr[i][0], kr[i][1], kr[i][2], kr[i][3]}, q, s);
        }
      }
      if (more) {
        pid = pid_next;
        page_of(t + kWaves, key_off);
        if (t + 2 * kWaves < t1) {
          int unused;
          pid_next = page_id(page_of(t + 2 * kWaves, unused));
        }
        load_k();
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
      if (__any(mt > m)) {
        const float f = exp2_diff(m, mt);
        m = mt;
        l *= f;
#pragma unroll
        for (int i = 0; i < G::NB; i++)
#pragma unroll
          for (int j = 0; j < G::VE; j++)
#pragma unroll
            for (int r = 0; r < 4; r++) o[i][j][r] *= f;
      }
      if (!whole) {  // the values of keys outside count as zero, also where they are not numbers
#pragma unroll
        for (int r = 0; r < 4; r++) {
          const int vk = 16 * t + 4 * g + r;
          const bool live = vk >= lo && vk < hi;
#pragma unroll
          for (int i = 0; i < G::NB; i++)
#pragma unroll
            for (int e = 0; e < G::VW; e++) vr[r][i][e] = live ? vr[r][i][e] : 0u;
        }
      }
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
      if (more) load_v();
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
            for (int j = 0; j < G::VE; j += 4)
              *reinterpret_cast<f32x4*>(row + d + j) = f32x4{o[i][j][r], o[i][j + 1][r], o[i][j + 2][r], o[i][j + 3][r]};
          }
        }
      if (g == 0) {
        ml[(wave * 16 + c) * 2] = m;
        ml[(wave * 16 + c) * 2 + 1] = l;
      }
    }
    __syncthreads();
    const int64_t u0 = at - s0, u1 = u0 + steps;  // the head's steps among all
    const int w0 = (int)(u0 / n), w1 = (int)((u1 - 1) / n);
    const int words = part_words(heads, DP);
    auto part_at = [&](int w) -> uint32_t {  // bytes; a workgroup's first head that began before it, or its last
      return (uint32_t)((2 * w + (w == w0)) * part_words(min(per, 16), DP)) * 4u;
    };
    auto finish = [&](int h, int d, float M, float L, float acc) {
      if (a.sinks) {
        const float sink = a.sinks[head0 + h] * kLog2e, M2 = fmaxf(M, sink), f = exp2_diff(M, M2);
        L = L * f + exp2_diff(sink, M2);
        acc *= f;
      }
      store_element<XT>(a.out, ((int64_t)b * a.Hq + head0 + h) * a.D + d, L == 0.f ? 0.f : acc / L);
    };
    for (int e = tid; e < heads * DP; e += 256) {
      const int h = e / DP, d = e - h * DP;
      float M = -INFINITY, L = 0.f, acc = 0.f;
#pragma unroll
      for (int w = 0; w < kWaves; w++) M = fmaxf(M, ml[(w * 16 + h) * 2]);
#pragma unroll
      for (int w = 0; w < kWaves; w++) {
        const float f = exp2_diff(ml[(w * 16 + h) * 2], M);
        L += f * ml[(w * 16 + h) * 2 + 1];
        acc += f * lds[(w * heads + h) * G::LD + d];
      }
      if (w0 == w1) {
        if (d < a.D) finish(h, d, M, L, acc);
      } else {
        const uint32_t p = part_at(blockIdx.x);
        __builtin_amdgcn_raw_buffer_store_b32(__float_as_uint(acc), parts, p + e * 4, 0, kAgentScope);
        if (d == 0) {
          __builtin_amdgcn_raw_buffer_store_b32(__float_as_uint(M), parts, p + (heads * DP + 2 * h) * 4, 0, kAgentScope);
          __builtin_amdgcn_raw_buffer_store_b32(__float_as_uint(L), parts, p + (heads * DP + 2 * h + 1) * 4, 0,
                                                kAgentScope);
        }
      }
    }
    if (w0 != w1) {
      __builtin_amdgcn_s_waitcnt(0);  // this thread's partial stores have completed
      __syncthreads();
      if (tid == 0) arrived = __hip_atomic_fetch_add(a.cnt + w0, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      __syncthreads();
      if (arrived == (uint32_t)(w1 - w0)) {  // the last one joins, in the order of the keys
        if (tid == 0) __hip_atomic_store(a.cnt + w0, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        for (int e = tid; e < heads * DP; e += 256) {
          const int h = e / DP, d = e - h * DP;
          float M = -INFINITY, L = 0.f, acc = 0.f;
          for (int w = w0; w <= w1; w++) {
            const uint32_t p = part_at(w), pm = p + (heads * DP + 2 * h) * 4;
            const float mw = __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(parts, pm, 0, kAgentScope));
            const float lw = __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(parts, pm + 4, 0, kAgentScope));
            const float ow = __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(parts, p + e * 4, 0, kAgentScope));
            const float M2 = fmaxf(M, mw), f = exp2_diff(M, M2), fw = exp2_diff(mw, M2);
            M = M2;
            L = L * f + lw * fw;
            acc = acc * f + ow * fw;
          }
          if (d < a.D) finish(h, d, M, L, acc);
        }
      }
    }
    __syncthreads();  // the LDS rows are free again
    off += s1 - s0;
    at += s1 - s0;
  }
}

template <int XT, int DP>
hipError_t launch(const PagedAttnArgs& a, hipStream_t stream) {
  const int per = a.Hq / a.Hkv, heads = per < 16 ? per : 16;
  const size_t bytes = (size_t)(kWaves * heads * Geo<XT, DP>::LD + kWaves * 32) * sizeof(float);
  hipLaunchKernelGGL((paged_attention_kernel<XT, DP>), dim3((unsigned)a.wgs), dim3(256), bytes, stream, a);
  return hipGetLastError();
}

// f(type, width of the kernel)
template <typename F>
auto with_kernel(const PagedAttnArgs& a, F&& f) {
  auto width = [&](auto xt) {
    constexpr int XT = decltype(xt)::value;
    if (a.D <= 64) return f(xt, std::integral_constant<int, 64>{});
    if (a.D <= 96) return f(xt, std::integral_constant<int, 96>{});
    if (a.D <= 128) return f(xt, std::integral_constant<int, 128>{});
    if (a.D <= 192) return f(xt, std::integral_constant<int, 192>{});
    return f(xt, std::integral_constant<int, 256>{});
  };
  if (a.type == GEN_BF16) return width(std::integral_constant<int, GEN_BF16>{});
  if (a.type == GEN_F16) return width(std::integral_constant<int, GEN_F16>{});
  return width(std::integral_constant<int, GEN_F32>{});
}

}  // namespace

// Steps a workgroup takes at least: below that, joining costs more than it saves.
constexpr int kLeastSteps = 4;

void paged_attention_plan(PagedAttnArgs& a, int cus, int64_t* part_bytes) {
  a.page_shift = 30;
  while (((int64_t)1 << (a.page_shift - 30)) < a.page) a.page_shift++;
  // exact for keys below 2^30: the error of page_mul, below page <= 2^(shift - 30), times the key stays below 2^shift
  a.page_mul = (uint32_t)((((uint64_t)1 << a.page_shift) + a.page - 1) / a.page);
  const int per = a.Hq / a.Hkv;
  const int64_t keys = a.window > 0 ? std::min<int64_t>(a.window + 15, (int64_t)a.width * a.page) : (int64_t)a.width * a.page;
  const int64_t most = (int64_t)a.B * a.Hkv * ((per + 15) / 16) * ((keys + 15 + kStep - 1) / kStep);
  a.least = kLeastSteps;
  const int resident = with_kernel(a, [](auto xt, auto dp) { return Geo<decltype(xt)::value, decltype(dp)::value>::WGS; });
  a.wgs = (int)std::max<int64_t>(1, std::min<int64_t>((most + a.least - 1) / a.least, (int64_t)cus * resident));
  const int words = with_kernel(a, [&](auto, auto dp) { return part_words(std::min(per, 16), decltype(dp)::value); });
  *part_bytes = (int64_t)2 * a.wgs * words * 4;
}

hipError_t launch_paged_attention(const PagedAttnArgs& a, hipStream_t stream) {
  if (a.B == 0) return hipSuccess;
  if (a.D < 8 || a.D > 256 || a.D % 8 || a.pages < 1 || a.page < 1 || a.wgs < 1 || a.wgs > kSplitCounters)
    return hipErrorInvalidValue;
  return with_kernel(a, [&](auto xt, auto dp) { return launch<decltype(xt)::value, decltype(dp)::value>(a, stream); });
}

}  // namespace mlxq
