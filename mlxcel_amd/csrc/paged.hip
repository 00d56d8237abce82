// paged.hip — attention of one new token per sequence over a paged key-value
// cache on gfx950.
//
//   s_t = cap(q . k_t * scale)   over the sequence's keys t in [lo, hi)
//   o   = sum_t exp(s_t - m) v_t / (sum_t exp(s_t - m) + exp(sink - m))
//
// with hi the length, lo = hi - window (0 without one), cap(s) = s or
// c tanh(s / c), m the largest s_t (and sink).  Each key and value is read
// once for each 16 query heads of its key head; that read is the bound (4 D
// operations a byte pair and query head stay far under the matrix rate).
//
// The work is cut evenly whatever the lengths: with a sequence's keys counted
// in steps of 128 (of 64 with wide 32-bit heads) for each key head and each 16 of
// its query heads, and two more for what a head's start and end cost, workgroup w
// takes [w n, (w + 1) n) of them all.  The lengths are on the device, so each
// workgroup finds its first step from a scan over them.  A sequence's head that
// crosses a workgroup's end leaves its sum, maximum and output so far in scratch;
// the last of its workgroups to arrive joins them, in the order of the keys, so
// the result does not depend on who came last.
//
// In a step each wave takes 32 (16) keys, with a running maximum and sum of its
// own; the waves are joined in LDS at a head's end.  Its next keys are loaded
// right after the product that used up these ones' registers, and their page
// numbers one step before that, so a wave keeps 8 to 16 KiB in flight (D = 128,
// 16 bits).  Both products run on MFMA with the layouts chosen so that nothing
// moves between them:
//   S^T[key][head] = K Q^T: lane (c, g) = (lane % 16, lane / 16) loads 16 bytes
//     of key c, so the tile's keys are read in 16 rows of 64 contiguous bytes;
//     it ends with the scores of keys 4 g + r (r < 4) of head c.
//   O^T[d][head] += V^T P^T: lane (c, g) loads V of keys 4 g + r (r < 4), columns
//     VE c .. VE c + VE - 1, so a key's row is read as one contiguous run and the
//     lane holds P of the same keys for head c.  Accumulator j is column VE c + j,
//     rows 4 g + r' of O^T: d = VE (4 g + r') + j, head c, the lane whose maximum
//     rescales it.  16-bit pools: one MFMA of 32 keys, slot 4 t + r of group g key
//     4 g + r of tile t; a column's keys are put side by side with byte permutes,
//     and P goes in as the sum of three bfloat16 or two float16 numbers, which
//     leave at most 2^-24 of it out, what a 32-bit number would: three MFMAs of 16
//     cycles a column instead of the 256 cycles of 32-bit ones.  With two bfloat16
//     numbers (2^-17 left out) 258 of 131072 results of 32 ragged sequences were not
//     the 64-bit ones rounded, with three 15, at 41.5 and 41.6 us (width 256 38.9 and
//     39.3).  A part may be 0 or below it, so an infinite value may give NaN.  32-bit
//     pools: MFMAs of 4 keys, step r taking keys 4 g + r.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cfloat>
#include <type_traits>

#include "common.hpp"
#include "kernels.hpp"
#include "wave.hpp"

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
  // 16-key tiles a wave takes at a time: 16-bit products of 32 keys; 32-bit
  // ones have no shape to fill and take two tiles where they fit the registers
  static constexpr int KT = !F32 || DP <= 64 ? 2 : 1;
  static constexpr int KEYS = 16 * KT * 4;         // keys of a step (4 waves)
  // Workgroups a CU holds: by registers (K, V and O of a lane)
  static constexpr int WGS = DP * ES * KT <= 256 ? 4 : DP * ES * KT <= 512 ? 2 : 1;
};

// Two 32-bit values as a pair of 16-bit ones, rounded to nearest.
template <int XT>
__device__ __forceinline__ uint32_t pack(float lo, float hi) {
  if constexpr (XT == GEN_BF16) {
    typedef float f32x2 __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2{lo, hi}, bf16x2));
  } else {
    typedef _Float16 h2 __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(uint32_t, h2{(_Float16)lo, (_Float16)hi});
  }
}
template <int XT>
__device__ __forceinline__ float half(uint32_t w, int hi) {
  return xt_to_f32<XT == GEN_F16 ? 1 : 0>(hi ? w >> 16 : w & 0xFFFFu);
}

template <int XT>
__device__ __forceinline__ void store_element(void* p, int64_t i, float v) {
  if constexpr (XT == GEN_F32) static_cast<float*>(p)[i] = v;
  else static_cast<uint16_t*>(p)[i] = (uint16_t)f32_to_xt<XT == GEN_F16 ? 1 : 0>(v);
}

template <int XT>
__device__ __forceinline__ void store4(void* p, int64_t i, f32x4 v) {
#pragma unroll
  for (int e = 0; e < 4; e++) store_element<XT>(p, i + e, v[e]);
}

// Probabilities are held as 2^lift p: in float16 their largest is then 2^14, and
// those down to 2^-28 of it keep all their bits (smaller ones differ by 2^-39 of it).
template <int XT>
constexpr float kLift = XT == GEN_F16 ? 14.f : 0.f;

// A load that leaves the caches to others (ONCE), or an ordinary one.
template <bool ONCE, typename T>
__device__ __forceinline__ T load(const char* p) {
  if constexpr (ONCE) return __builtin_nontemporal_load(reinterpret_cast<const T*>(p));
  else return *reinterpret_cast<const T*>(p);
}

// exp2(a - b), 0 where a is -inf (also where b is)
__device__ __forceinline__ float exp2_diff(float a, float b) {
  return __builtin_amdgcn_exp2f(a - (b == -INFINITY ? 0.f : b));
}

// Keys [lo, hi) of a sequence, and its steps.
template <int KEYS>
__device__ __forceinline__ int steps_of(int len, int64_t cap, int window, int& lo, int& hi) {
  hi = (int)min((int64_t)max(len, 0), cap);
  lo = window > 0 ? max(0, hi - window) : 0;
  return (hi - lo + KEYS - 1) / KEYS;
}

// Steps of a head that is not cut: taking them one after the other costs about
// what a join costs (one sequence of 1000 keys, 8 steps a head: 11.1 us cut, 24.8
// whole; 200 sequences of 1 to 4 steps: 15.5 us whole, 16.5 cut at every step).
constexpr int kWholeSteps = 4;

// What a head's start and end cost, in steps: with 0 32 ragged sequences took
// 45.8 us, with 2 42.0, with 4 44.9 (16 ragged ones of width 256 44.6, 36.5, 39.7).
constexpr int kAround = 2;

constexpr int64_t kLastCache = (int64_t)256 << 20;

// Workgroups whose results one of them joins, and how many are read at a time.
// Joins of 8, 16 and 32: one sequence of 8000 keys on 8 heads 18.3, 20.0 and 23.7 us,
// of 40000 keys on one head 20.8, 20.3 and 24.2, 32 ragged sequences 41.8, 40.9 and
// 40.7.  4, 8 and 16 at a time (more than the registers hold): 19.8, 20.0 and 31.2;
// 19.9, 20.3 and 31.9; 40.8, 40.9 and 50.8.
constexpr int kJoin = 16, kFlight = 8;

// Words of one partial result: O [heads][DP], then (m, l) [heads][2].
constexpr int part_words(int heads, int DP) { return heads * (DP + 2); }

template <int XT, int DP>
__global__ __launch_bounds__(256, (Geo<XT, DP>::WGS)) void paged_attention_kernel(const PagedAttnArgs a) {
  using G = Geo<XT, DP>;
  extern __shared__ __align__(16) float lds[];
  __shared__ u32x4 qs[G::KC * 64];
  __shared__ uint32_t arrived;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int c = lane & 15, g = lane >> 4;
  const int per = a.Hq / a.Hkv, tiles_h = (per + 15) / 16;
  const int64_t cap = (int64_t)a.width * a.page;
  const int heads_b = a.Hkv * tiles_h;  // (key head, 16 query heads) of a sequence

  // Where this workgroup's units begin and end: unit among all, unit in its
  // sequence, sequence, its length.
  struct Bound {
    int unit, off, b, len;
  };
  auto steps_in = [&](int len) {
    int lo, hi;
    return steps_of<G::KEYS>(len, cap, a.window, lo, hi);
  };
  auto units_in = [&](int len) {  // of one head
    const int s = steps_in(len);
    return s ? kAround + s : 0;
  };
  // Unit p, `off` into sequence b, unless it cuts a head of few steps: that one
  // belongs to the workgroup of its first step.
  auto bound_at = [&](int p, int off, int b, int len) -> Bound {
    const int u = units_in(len), up = steps_in(len) <= kWholeSteps && off % u > kAround ? u - off % u : 0;
    return Bound{p + up, off + up, b, len};
  };
  auto clear = [&](int b) {  // a sequence without keys has no steps: its output is zeros
    for (int i = tid; i < a.Hq * a.D; i += 256) store_element<XT>(a.out, (int64_t)b * a.Hq * a.D + i, 0.f);
  };
  int n, total;
  Bound first, last;
  if (a.B <= 64) {  // each wave finds them by itself, sequence i in lane i
    const int len = lane < a.B ? a.lengths[lane] : 0, units = units_in(len), mine = heads_b * units;
    int sum = mine;
#pragma unroll
    for (int s = 1; s < 64; s <<= 1) {
      const int o = __shfl_up(sum, s);
      if (lane >= s) sum += o;
    }
    total = __builtin_amdgcn_readlane(sum, 63);
    n = (total + a.wgs - 1) / a.wgs;
    auto find = [&](int p) -> Bound {
      if (p >= total) return Bound{total, 0, 0, 0};
      const int i = __builtin_ctzll(__ballot(sum - mine <= p && p < sum));
      return bound_at(p, p - __builtin_amdgcn_readlane(sum - mine, i), i, __builtin_amdgcn_readlane(len, i));
    };
    first = find(blockIdx.x * n);
    last = find((blockIdx.x + 1) * n);
    for (uint64_t none = __ballot(lane < a.B && units == 0); none; none &= none - 1)
      if (__builtin_ctzll(none) % a.wgs == (int)blockIdx.x) clear(__builtin_ctzll(none));
  } else {  // thread i sums those of its share
    __shared__ int scan[kWaves];
    __shared__ Bound bound[2];
    const int share = (a.B + 255) / 256, b0 = min(tid * share, a.B), b1 = min(b0 + share, a.B);
    int mine = 0;
    for (int b = b0; b < b1; b++) mine += heads_b * units_in(a.lengths[b]);
    int sum = mine;
#pragma unroll
    for (int s = 1; s < 64; s <<= 1) {
      const int o = __shfl_up(sum, s);
      if (lane >= s) sum += o;
    }
    if (lane == 63) scan[wave] = sum;
    __syncthreads();
    int before = sum - mine;
    total = 0;
#pragma unroll
    for (int w = 0; w < kWaves; w++) {
      if (w < wave) before += scan[w];
      total += scan[w];
    }
    n = (total + a.wgs - 1) / a.wgs;
#pragma unroll
    for (int i = 0; i < 2; i++) {
      const int p = ((int)blockIdx.x + i) * n;
      if (p >= total) {
        if (tid == 0) bound[i] = Bound{total, 0, 0, 0};
      } else if (before <= p && p < before + mine) {
        int off = p - before, b = b0;
        while (b + 1 < b1 && off >= heads_b * units_in(a.lengths[b])) off -= heads_b * units_in(a.lengths[b++]);
        bound[i] = bound_at(p, off, b, a.lengths[b]);
      }
    }
    for (int b = blockIdx.x; b < a.B; b += a.wgs)
      if (steps_in(a.lengths[b]) == 0) clear(b);
    __syncthreads();
    first = bound[0];
    last = bound[1];
  }
  int at = __builtin_amdgcn_readfirstlane(first.unit);
  const int end = __builtin_amdgcn_readfirstlane(last.unit);
  if (at >= end) return;
  int off = __builtin_amdgcn_readfirstlane(first.off), b = __builtin_amdgcn_readfirstlane(first.b);
  int len = __builtin_amdgcn_readfirstlane(first.len);
  // More keys and values than the last cache holds beside others' are not kept
  // there for the next call: 2.1 GB 360 -> 325 us, 174 MB among other work 46 -> 44.5 us
  // (read again and again by itself 37 -> 44 us).
  const bool once =
      ((int64_t)total - (int64_t)kAround * heads_b * a.B) * (G::KEYS * 2 * G::ES) * a.D > kLastCache / 2;
  // scores in units of log2 e
  const float scale = a.softcap > 0.f ? a.scale / a.softcap : a.scale * kLog2e, cap_log2e = a.softcap * kLog2e;
  const int slot_words = part_words(min(per, 16), DP);
  const __amdgpu_buffer_rsrc_t parts = buffer_rsrc(a.part, (uint32_t)((int64_t)4 * a.wgs * slot_words * 4));

  auto run = [&](auto ONCE) {
    while (at < end) {
      int lo, hi;
      const int steps = steps_of<G::KEYS>(len, cap, a.window, lo, hi), units = units_in(len);
      if (off >= units * heads_b) {
        if (++b >= a.B) break;
        len = __builtin_amdgcn_readfirstlane(a.lengths[b]);
        off = 0;
        continue;
      }
      const int hh = off / units, skip = max(kAround - (off - hh * units), 0);
      if (at + skip >= end) break;  // its steps begin in the next workgroup
      at += skip;
      off += skip;
      const int s0 = off - hh * units - kAround, s1 = min(steps, s0 + (end - at));
      const int hk = hh / tiles_h, ht = hh - hk * tiles_h;
      const int heads = min(16, per - 16 * ht), head0 = hk * per + 16 * ht;

      const int32_t* table = a.table + b * a.table_row;
      const char* kb = static_cast<const char*>(a.k) + hk * a.k_head * G::ES;
      const char* vb = static_cast<const char*>(a.v) + hk * a.v_head * G::ES;

      f32x4 o[G::NB][G::VE];
#pragma unroll
      for (int i = 0; i < G::NB; i++)
#pragma unroll
        for (int j = 0; j < G::VE; j++) o[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
      float m = -INFINITY, l = 0.f;
      uint32_t kr[G::KT][G::KC][4], vr[G::KT][4][G::NB][G::VW];
      int pid[G::KT], entry[G::KT], key_off[G::KT];  // pages of the keys in hand, table entries of the next ones
      // this wave's keys of the segment: 16 KT from k0 on, every KEYS
      const int k0 = lo + s0 * G::KEYS + wave * (16 * G::KT), k1 = min(hi, lo + s1 * G::KEYS);

      // The lane's key of the tile from `from` on.  Past the segment it is the
      // segment's last key: rows outside the sequence are never read, and loads
      // past the end need no branch (they ask for one row, which is at hand).
      auto page_of = [&](int from, int& in_page) -> int {
        const int key = min(from + c, k1 - 1);
        const int slot = (int)(((uint64_t)(uint32_t)key * a.page_mul) >> a.page_shift);
        in_page = key - slot * a.page;
        return slot;
      };
      auto load_k = [&](auto ONCE, int t) {
        const char* kp = kb + (pid[t] * a.k_page + key_off[t] * a.k_tok) * G::ES;
#pragma unroll
        for (int i = 0; i < G::KC; i++) {
          const int d = 4 * G::KE * i + G::KE * g;
          const u32x4_e w = load<decltype(ONCE)::value, u32x4_e>(kp + (d < a.D ? d : 0) * G::ES);
#pragma unroll
          for (int e = 0; e < 4; e++) kr[t][i][e] = w[e];
        }
      };
      auto load_v = [&](auto ONCE, int t) {
#pragma unroll
        for (int r = 0; r < 4; r++) {
          const int vpid = __shfl(pid[t], 4 * g + r), voff = __shfl(key_off[t], 4 * g + r);
          const char* vp = vb + (vpid * a.v_page + voff * a.v_tok) * G::ES;
#pragma unroll
          for (int i = 0; i < G::NB; i++) {
            const int d = 16 * G::VE * i + G::VE * c;
            const char* p = vp + (d < a.D ? d : 0) * G::ES;  // columns past the head are dropped at the end
            if constexpr (G::VW == 4) {
              const u32x4_e w = load<decltype(ONCE)::value, u32x4_e>(p);
#pragma unroll
              for (int e = 0; e < 4; e++) vr[t][r][i][e] = w[e];
            } else {
              const u32x2_e w = load<decltype(ONCE)::value, u32x2_e>(p);
#pragma unroll
              for (int e = 0; e < 2; e++) vr[t][r][i][e] = w[e];
            }
          }
        }
      };
      // the keys in hand become those from `from` on; the ones after them have their table entries loaded
      auto advance = [&](int from) {
#pragma unroll
        for (int t = 0; t < G::KT; t++) {
          int unused;
          pid[t] = min(max(entry[t], 0), a.pages - 1);
          page_of(from + 16 * t, key_off[t]);
          entry[t] = table[page_of(from + G::KEYS + 16 * t, unused)];
        }
      };

      // Q of head c in LDS, a lane's 16 bytes after the other: B operand, the d
      // order of the K loads
      u32x4 q0[(G::KC + kWaves - 1) / kWaves];
#pragma unroll
      for (int i = wave, j = 0; j < (G::KC + kWaves - 1) / kWaves; i += kWaves, j++) {
        const int d = 4 * G::KE * i + G::KE * g;
        const char* qp = static_cast<const char*>(a.q) + (b * a.q_b + (head0 + min(c, heads - 1)) * a.q_h) * G::ES;
        const u32x4_e w = *reinterpret_cast<const u32x4_e*>(qp + (d < a.D ? d : 0) * G::ES);
        q0[j] = d < a.D ? u32x4{w[0], w[1], w[2], w[3]} : u32x4{0u, 0u, 0u, 0u};
      }
      if (k0 < k1) {
#pragma unroll
        for (int t = 0; t < G::KT; t++) entry[t] = table[page_of(k0 + 16 * t, key_off[t])];
        advance(k0);
#pragma unroll
        for (int t = 0; t < G::KT; t++) load_k(ONCE, t);
#pragma unroll
        for (int t = 0; t < G::KT; t++) load_v(ONCE, t);
      }
#pragma unroll
      for (int i = wave, j = 0; j < (G::KC + kWaves - 1) / kWaves; i += kWaves, j++)
        if (i < G::KC) qs[i * 64 + lane] = q0[j];
      __syncthreads();
      for (int k = k0; k < k1; k += G::KEYS) {
        if (DP != a.D) {  // columns past the head are zero on both sides
#pragma unroll
          for (int t = 0; t < G::KT; t++)
#pragma unroll
            for (int i = 0; i < G::KC; i++)
#pragma unroll
              for (int e = 0; e < 4; e++) kr[t][i][e] = 4 * G::KE * i + G::KE * g < a.D ? kr[t][i][e] : 0u;
        }
        f32x4 s[G::KT];
#pragma unroll
        for (int t = 0; t < G::KT; t++) s[t] = f32x4{0.f, 0.f, 0.f, 0.f};
        asm volatile("" ::: "memory");  // Q is read again each time, not kept in registers
#pragma unroll
        for (int i = 0; i < G::KC; i++) {
          const u32x4 q = qs[i * 64 + lane];
#pragma unroll
          for (int t = 0; t < G::KT; t++) {
            if constexpr (G::F32) {
#pragma unroll
              for (int e = 0; e < 4; e++)
                s[t] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(kr[t][i][e]), __uint_as_float(q[e]), s[t], 0,
                                                            0, 0);
            } else {
              s[t] = mfma16x16x32_xt<XT == GEN_F16 ? 1 : 0>(
                  u32x4{kr[t][i][0], kr[t][i][1], kr[t][i][2], kr[t][i][3]}, q, s[t]);
            }
          }
        }
        advance(k + G::KEYS);
#pragma unroll
        for (int t = 0; t < G::KT; t++) load_k(ONCE, t);
        if (a.softcap > 0.f) {
#pragma unroll
          for (int t = 0; t < G::KT; t++)
#pragma unroll
            for (int r = 0; r < 4; r++) s[t][r] = cap_log2e * tanhf(s[t][r] * scale);
        } else {
#pragma unroll
          for (int t = 0; t < G::KT; t++)
#pragma unroll
            for (int r = 0; r < 4; r++) s[t][r] *= scale;
        }
        float mt = m;
#pragma unroll
        for (int t = 0; t < G::KT; t++)
#pragma unroll
          for (int r = 0; r < 4; r++) {
            s[t][r] = k + 16 * t + 4 * g + r < k1 ? s[t][r] : -INFINITY;
            mt = fmaxf(mt, s[t][r]);
          }
        mt = fmaxf(mt, lane_xor<16>(mt, lane));
        mt = fmaxf(mt, lane_xor<32>(mt, lane));
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
        if (k + 16 * G::KT > k1) {
          // past the segment p is 0, and the row read in its place has to count as 0 also where it is not finite
#pragma unroll
          for (int t = 0; t < G::KT; t++)
#pragma unroll
            for (int r = 0; r < 4; r++)
#pragma unroll
              for (int i = 0; i < G::NB; i++)
#pragma unroll
                for (int e = 0; e < G::VW; e++) vr[t][r][i][e] = k + 16 * t + 4 * g + r < k1 ? vr[t][r][i][e] : 0u;
        }
#pragma unroll
        for (int t = 0; t < G::KT; t++)
#pragma unroll
          for (int r = 0; r < 4; r++) {
            s[t][r] = exp2_diff(s[t][r] + kLift<XT>, m);
            l += s[t][r];
          }
        if constexpr (G::F32) {
#pragma unroll
          for (int t = 0; t < G::KT; t++)
#pragma unroll
            for (int r = 0; r < 4; r++)
#pragma unroll
              for (int i = 0; i < G::NB; i++)
#pragma unroll
                for (int j = 0; j < G::VE; j++)
                  o[i][j] =
                      __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(vr[t][r][i][j]), s[t][r], o[i][j], 0, 0, 0);
        } else {
          // P as a sum of 16-bit numbers, each what the ones before it leave of it
          constexpr int TERMS = XT == GEN_BF16 ? 3 : 2;
          u32x4 pt[TERMS];
#pragma unroll
          for (int t = 0; t < 2; t++)
#pragma unroll
            for (int r = 0; r < 4; r += 2) {
              float lo = s[t][r], hi = s[t][r + 1];
#pragma unroll
              for (int n = 0; n < TERMS; n++) {
                const uint32_t w = pack<XT>(lo, hi);
                pt[n][2 * t + r / 2] = w;
                lo -= half<XT>(w, 0);
                hi -= half<XT>(w, 1);
              }
            }
#pragma unroll
          for (int i = 0; i < G::NB; i++)
#pragma unroll
            for (int j = 0; j < G::VE; j++) {
              const uint32_t sel = j & 1 ? 0x07060302u : 0x05040100u;
              u32x4 v;
#pragma unroll
              for (int t = 0; t < 2; t++)
#pragma unroll
                for (int r = 0; r < 4; r += 2)
                  v[2 * t + r / 2] = __builtin_amdgcn_perm(vr[t][r + 1][i][j / 2], vr[t][r][i][j / 2], sel);
#pragma unroll
              for (int n = 0; n < TERMS; n++) o[i][j] = mfma16x16x32_xt<XT == GEN_F16 ? 1 : 0>(v, pt[n], o[i][j]);
            }
        }
#pragma unroll
        for (int t = 0; t < G::KT; t++) load_v(ONCE, t);
      }
      l += lane_xor<16>(l, lane);
      l += lane_xor<32>(l, lane);

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
                *reinterpret_cast<f32x4*>(row + d + j) =
                    f32x4{o[i][j][r], o[i][j + 1][r], o[i][j + 2][r], o[i][j + 3][r]};
            }
          }
        if (g == 0) {
          ml[(wave * 16 + c) * 2] = m - kLift<XT>;
          ml[(wave * 16 + c) * 2 + 1] = l;
        }
      }
      __syncthreads();
      const int w0 = (at - s0) / n, w1 = steps <= kWholeSteps ? w0 : (at - s0 + steps - 1) / n;
      // bytes of a workgroup's partial result: of its last head (slot 1), or of one that began before it (slot 0)
      auto part_at = [&](int w) -> uint32_t { return (uint32_t)((2 * w + (w == w0)) * slot_words) * 4u; };
      // and of the neighbours that it leads, in a place of its own: others of the joining threads may still read the first
      const uint32_t joined = (uint32_t)(2 * a.wgs * slot_words) * 4u;
      auto put = [&](uint32_t p, int e, float M, float L, f32x4 acc) {
        __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, acc), parts, p + e * 16, 0, kAgentScope);
        if (e % (DP / 4) == 0)
          __builtin_amdgcn_raw_buffer_store_b64(u32x2{__float_as_uint(M), __float_as_uint(L)}, parts,
                                                p + (heads * DP + 2 * (e / (DP / 4))) * 4, 0, kAgentScope);
      };
      auto finish = [&](int h, int d, float M, float L, f32x4 acc) {
        float f = 1.f;
        if (a.sinks) {
          const float x = a.sinks[head0 + h];
          // the largest finite sinks stay finite in the other base
          const float sink = isinf(x) ? x : fminf(fmaxf(x * kLog2e, -FLT_MAX), FLT_MAX), M2 = fmaxf(M, sink);
          f = exp2_diff(M, M2);
          L = L * f + exp2_diff(sink, M2);
        }
        const float r = f / L;  // scores and sink all -inf: 0 / 0, not a number as the definition says
        if (d < a.D) store4<XT>(a.out, ((int64_t)b * a.Hq + head0 + h) * a.D + d, acc * r);
      };
      for (int e = tid; e < heads * (DP / 4); e += 256) {
        const int h = e / (DP / 4), d = 4 * (e - h * (DP / 4));
        float M = -INFINITY, L = 0.f;
        f32x4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < kWaves; w++) M = fmaxf(M, ml[(w * 16 + h) * 2]);
#pragma unroll
        for (int w = 0; w < kWaves; w++) {
          const float f = exp2_diff(ml[(w * 16 + h) * 2], M);
          L += f * ml[(w * 16 + h) * 2 + 1];
          acc += f * *reinterpret_cast<const f32x4*>(lds + (w * heads + h) * G::LD + d);
        }
        if (w0 == w1) {
          finish(h, d, M, L, acc);
        } else {
          put(part_at(blockIdx.x), e, M, L, acc);
        }
      }
      if (w0 != w1) {
        // The last of up to kJoin neighbours to arrive joins them; of more, the
        // last to have joined its neighbours joins the results.
        auto last_of = [&](uint32_t* cnt, int of) -> bool {
          __builtin_amdgcn_s_waitcnt(0);  // this thread's partial stores have completed
          __syncthreads();
          if (tid == 0) {
            const uint32_t old = __hip_atomic_fetch_add(cnt, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            arrived = old == (uint32_t)(of - 1);
            if (arrived) __hip_atomic_store(cnt, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
          }
          __syncthreads();
          return arrived != 0;
        };
        // sum of the results, from byte `from` on, of workgroups w, w + by, .. (of them), in the order of the keys
        auto join = [&](uint32_t from, int w, int by, int of, int e, float& M, float& L, f32x4& acc) {
          const int h = e / (DP / 4);
          M = -INFINITY, L = 0.f, acc = f32x4{0.f, 0.f, 0.f, 0.f};
          for (int i0 = 0; i0 < of; i0 += kFlight) {
            u32x4 ow[kFlight];
            u32x2 mw[kFlight];
#pragma unroll
            for (int i = 0; i < kFlight; i++) {
              const uint32_t p = from + part_at(w + by * min(i0 + i, of - 1));
              mw[i] = __builtin_bit_cast(u32x2, __builtin_amdgcn_raw_buffer_load_b64(parts, p + (heads * DP + 2 * h) * 4,
                                                                                     0, kAgentScope));
              ow[i] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(parts, p + e * 16, 0, kAgentScope));
            }
#pragma unroll
            for (int i = 0; i < kFlight; i++) {
              if (i0 + i >= of) break;
              const float mi = __uint_as_float(mw[i][0]), M2 = fmaxf(M, mi);
              const float f = exp2_diff(M, M2), fi = exp2_diff(mi, M2);
              M = M2;
              L = L * f + __uint_as_float(mw[i][1]) * fi;
              acc = acc * f + __builtin_bit_cast(f32x4, ow[i]) * fi;
            }
          }
        };
        const int of = w1 - w0 + 1, mine = ((int)blockIdx.x - w0) / kJoin * kJoin, near = min(kJoin, of - mine);
        // a workgroup may lead neighbours of a head that began before it and of its last one
        if (last_of(a.cnt + 2 * (w0 + mine) + (mine == 0), near)) {
          for (int e = tid; e < heads * (DP / 4); e += 256) {
            const int h = e / (DP / 4), d = 4 * (e - h * (DP / 4));
            float M, L;
            f32x4 acc;
            join(0, w0 + mine, 1, near, e, M, L, acc);
            if (of <= kJoin) finish(h, d, M, L, acc);
            else put(joined + part_at(w0 + mine), e, M, L, acc);
          }
          const int groups = (of + kJoin - 1) / kJoin;
          if (of > kJoin && last_of(a.cnt + 2 * a.wgs + w0, groups)) {
            for (int e = tid; e < heads * (DP / 4); e += 256) {
              const int h = e / (DP / 4), d = 4 * (e - h * (DP / 4));
              float M, L;
              f32x4 acc;
              join(joined, w0, kJoin, groups, e, M, L, acc);
              finish(h, d, M, L, acc);
            }
          }
        }
      }
      __syncthreads();  // the LDS rows are free again
      off += s1 - s0;
      at += s1 - s0;
    }
  };
  if (once) run(std::true_type{});
  else run(std::false_type{});
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

bool paged_attention_plan(PagedAttnArgs& a, int cus, int64_t* part_bytes) {
  a.page_shift = 30;
  while (((int64_t)1 << (a.page_shift - 30)) < a.page) a.page_shift++;
  // exact for keys below 2^30: the error of page_mul, below page <= 2^(shift - 30), times the key stays below 2^shift
  a.page_mul = (uint32_t)((((uint64_t)1 << a.page_shift) + a.page - 1) / a.page);
  const int per = a.Hq / a.Hkv;
  const int64_t cap = (int64_t)a.width * a.page, keys = a.window > 0 ? std::min<int64_t>(a.window, cap) : cap;
  int step = 0, resident = 0;
  with_kernel(a, [&](auto xt, auto dp) {
    step = Geo<decltype(xt)::value, decltype(dp)::value>::KEYS;
    resident = Geo<decltype(xt)::value, decltype(dp)::value>::WGS;
    return 0;
  });
  const int64_t heads = (int64_t)a.B * a.Hkv * ((per + 15) / 16), most = heads * ((keys + step - 1) / step);
  a.wgs = (int)std::max<int64_t>(1, std::min<int64_t>(most, (int64_t)cus * resident));
  const int words = with_kernel(a, [&](auto, auto dp) { return part_words(std::min(per, 16), decltype(dp)::value); });
  *part_bytes = (int64_t)4 * a.wgs * words * 4;
  return most + kAround * heads <= (1 << 30);
}

hipError_t launch_paged_attention(const PagedAttnArgs& a, hipStream_t stream) {
  if (a.B == 0) return hipSuccess;
  if (a.D < 8 || a.D > 256 || a.D % 8 || a.pages < 1 || a.page < 1 || a.wgs < 1 || 3 * a.wgs > kSplitCounters)
    return hipErrorInvalidValue;
  return with_kernel(a, [&](auto xt, auto dp) { return launch<decltype(xt)::value, decltype(dp)::value>(a, stream); });
}

}  // namespace mlxq
