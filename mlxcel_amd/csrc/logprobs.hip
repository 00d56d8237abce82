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
//
// HBM-bound: each logit is read once.  A row is cut over `split` workgroups
// where there are few rows; in each, a wave takes chunks of 64 lanes x 16 values
// in turn.  A lane keeps a running maximum with S and sum_i exp(z_i) z_i relative
// to it, rescaled once a chunk.  Alternatives are picked in the same pass.  If
// each of the workgroup's A waves has ceil(k / A) lanes whose maxima reach f, k
// values do, and only values that reach f can be among the k largest; each wave
// sorts its lanes' maxima after its 1st, 2nd, 4th, .. chunk, and the least of the
// waves' ceil(k / A)-th ones is f.  Few values of a chunk pass (k / 4 or so of the
// first 1024 a wave, then fewer): they are collected in LDS as numbers that order
// (value, index) pairs and merged 64 at a time into the wave's 64 largest, sorted
// over its lanes.  The waves' and workgroups' lists and sums are joined at the
// end, the last workgroup of a row to arrive joining the row's.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdlib>

#include "common.hpp"
#include "kernels.hpp"

namespace mlxq {

namespace {

constexpr int kWaves = 4, kChunk = 1024;  // values of a wave's chunk
constexpr int kRowWgs = 4;                // workgroups a CU is given where rows are cut
constexpr float kLog2e = 1.44269504088896340736f, kLn2 = 0.69314718055994530942f;

typedef uint32_t u32x4_e __attribute__((ext_vector_type(4), aligned(2)));

template <int XT>
__device__ __forceinline__ float load(const void* p, int64_t i) {
  if constexpr (XT == GEN_F32) return static_cast<const float*>(p)[i];
  else return xt_to_f32<XT == GEN_F16 ? 1 : 0>(static_cast<const uint16_t*>(p)[i]);
}

// The order of the alternatives as one unsigned number: the value's order,
// then the lower index.  0 is no value.
__device__ __forceinline__ uint64_t order_key(float x, uint32_t i) {
  uint32_t u = __float_as_uint(x + 0.f);  // -0 becomes 0
  u = x != x ? 0xFF800001u : (u & 0x80000000u) ? ~u : u | 0x80000000u;
  return ((uint64_t)u << 32) | (uint32_t)~i;
}
__device__ __forceinline__ float key_value(uint64_t k) {
  const uint32_t u = (uint32_t)(k >> 32);
  return __uint_as_float(u & 0x80000000u ? u & 0x7FFFFFFFu : ~u);
}

// ---- sorted lists of 64 keys, one a lane --------------------------------------

// The value of the lane whose number differs in bit J: vector operations only
// (4 is 3 then 7; halves and rows of 16 are swapped between two registers).
template <int J>
__device__ __forceinline__ uint32_t lane_xor(uint32_t v, int lane) {
  if constexpr (J == 1) return __builtin_amdgcn_mov_dpp(v, 0xB1, 0xF, 0xF, false);
  else if constexpr (J == 2) return __builtin_amdgcn_mov_dpp(v, 0x4E, 0xF, 0xF, false);
  else if constexpr (J == 4)
    return __builtin_amdgcn_mov_dpp(__builtin_amdgcn_mov_dpp(v, 0x1B, 0xF, 0xF, false), 0x141, 0xF, 0xF, false);
  else if constexpr (J == 8) return __builtin_amdgcn_mov_dpp(v, 0x128, 0xF, 0xF, false);
  else if constexpr (J == 16) {
    const auto r = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    return lane & 16 ? r[0] : r[1];
  } else {
    const auto r = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    return lane & 32 ? r[0] : r[1];
  }
}
template <int J>
__device__ __forceinline__ uint64_t lane_xor64(uint64_t v, int lane) {
  return ((uint64_t)lane_xor<J>((uint32_t)(v >> 32), lane) << 32) | lane_xor<J>((uint32_t)v, lane);
}

// One step of a bitonic network: lanes J apart, the larger to the lower lane
// where `down`.
template <int J>
__device__ __forceinline__ void exchange(uint64_t& v, int lane, bool down) {
  const uint64_t o = lane_xor64<J>(v, lane);
  const bool larger = ((lane & J) == 0) == down;
  v = (o > v) == larger ? o : v;
}
template <int SIZE, int J>
__device__ __forceinline__ void bitonic(uint64_t& v, int lane) {
  exchange<J>(v, lane, SIZE == 64 || (lane & SIZE) == 0);
  if constexpr (J > 1) bitonic<SIZE, J / 2>(v, lane);
}
// Largest first, where lanes from n on hold 0.
__device__ __forceinline__ void sort64(uint64_t& v, int lane, int n) {
  bitonic<2, 1>(v, lane);
  bitonic<4, 2>(v, lane);
  bitonic<8, 4>(v, lane);
  bitonic<16, 8>(v, lane);
  if (n > 16) bitonic<32, 16>(v, lane);
  if (n > 32) bitonic<64, 32>(v, lane);
}
// Largest first.
template <int SIZE, int J>
__device__ __forceinline__ void bitonic_values(float& v, int lane) {
  const float o = __uint_as_float(lane_xor<J>(__float_as_uint(v), lane));
  v = ((lane & J) == 0) == (SIZE == 64 || (lane & SIZE) == 0) ? fmaxf(v, o) : fminf(v, o);
  if constexpr (J > 1) bitonic_values<SIZE, J / 2>(v, lane);
}
__device__ __forceinline__ float sorted_values(float v, int lane) {
  bitonic_values<2, 1>(v, lane);
  bitonic_values<4, 2>(v, lane);
  bitonic_values<8, 4>(v, lane);
  bitonic_values<16, 8>(v, lane);
  bitonic_values<32, 16>(v, lane);
  bitonic_values<64, 32>(v, lane);
  return v;
}

// The next value below (not a number below -inf; -0 is 0).
__device__ __forceinline__ float below(float f) {
  if (f == -INFINITY) return NAN;
  const uint32_t u = __float_as_uint(f);
  return __uint_as_float(f == 0.f ? 0x80000001u : f > 0.f ? u - 1 : u + 1);
}

// The 64 largest of two sorted lists, sorted.
__device__ __forceinline__ void merge64(uint64_t& v, uint64_t o, int lane) {
  o = __shfl((unsigned long long)o, 63 - lane);
  v = o > v ? o : v;
  bitonic<64, 32>(v, lane);
}

// ---- sums ------------------------------------------------------------------------

// Of a set of logits: their maximum m, s = sum 2^w and e = sum 2^w w with
// w = a (x - m), a = scale log2 e.
struct Sums {
  float m, s, e;
};
// The same with maximum M >= m.
__device__ __forceinline__ Sums rebase(Sums v, float M, float a) {
  const float d = v.m == M ? 0.f : v.m == -INFINITY ? -INFINITY : a * (v.m - M);
  const float f = __builtin_amdgcn_exp2f(d);
  return Sums{M, v.s * f, f == 0.f ? v.s * 0.f : f * (v.e + v.s * d)};
}
__device__ __forceinline__ Sums add(Sums x, Sums y, float a) {
  const float M = fmaxf(x.m, y.m);
  x = rebase(x, M, a);
  y = rebase(y, M, a);
  return Sums{M, x.s + y.s, x.e + y.e};
}

template <int XT>
__global__ __launch_bounds__(256, 5) void token_logprobs_kernel(const LogprobArgs a) {
  constexpr int PER = XT == GEN_F32 ? 4 : 8;  // values of a 16-byte load
  constexpr int NL = 16 / PER;                // loads of a lane and chunk
  __shared__ uint64_t cand[kWaves][128], lists[kWaves][64];
  __shared__ Sums sums[kWaves];
  __shared__ float reached[kWaves];
  __shared__ uint32_t arrived;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int64_t t = blockIdx.x / a.split;
  const int part = blockIdx.x - (int)t * a.split;  // of the row
  const char* row = static_cast<const char*>(a.logits) + t * a.row * (16 / PER);
  const float sc = a.scale * kLog2e;
  const int chunks = (a.V + kChunk - 1) / kChunk;
  const int step = a.split * kWaves;

  Sums mine = {-INFINITY, 0.f, 0.f};
  uint64_t list = 0, floor = 0;  // keys up to `floor` cannot be among the k largest
  float floor_value = NAN;       // their value; not a number: there are none
  int waiting = 0;               // candidates in LDS
  auto merge = [&](int n) {  // the first n <= 64 candidates
    __builtin_amdgcn_wave_barrier();
    uint64_t v = lane < n ? cand[wave][lane] : 0;
    const uint64_t rest = cand[wave][64 + lane];
    sort64(v, lane, n);
    merge64(list, v, lane);
    if (waiting > 64) cand[wave][lane] = rest;
    waiting -= n;
    __builtin_amdgcn_wave_barrier();
    const uint64_t kth = __shfl((unsigned long long)list, a.k - 1);
    if (kth > floor) {
      floor = kth;
      floor_value = key_value(kth);
    }
  };

  auto load_chunk = [&](int c, u32x4 (&w)[NL]) {
#pragma unroll
    for (int j = 0; j < NL; j++) {
      const int i = c * kChunk + (j * 64 + lane) * PER;
      if (i + PER <= a.V) {
        const u32x4_e v = *reinterpret_cast<const u32x4_e*>(row + (int64_t)i * (16 / PER));
        w[j] = u32x4{v[0], v[1], v[2], v[3]};
      } else {
#pragma unroll
        for (int e = 0; e < 4; e++) {
          w[j][e] = XT == GEN_F32 ? 0xFF800000u : XT == GEN_F16 ? 0xFC00FC00u : 0xFF80FF80u;  // -inf
          if constexpr (XT == GEN_F32) {
            if (i + e < a.V) w[j][e] = reinterpret_cast<const uint32_t*>(row)[i + e];
          } else {
            const uint16_t* p = reinterpret_cast<const uint16_t*>(row);
            if (i + 2 * e < a.V) w[j][e] = (w[j][e] & 0xFFFF0000u) | p[i + 2 * e];
            if (i + 2 * e + 1 < a.V) w[j][e] = (w[j][e] & 0xFFFFu) | (uint32_t)p[i + 2 * e + 1] << 16;
          }
        }
      }
    }
  };
  auto value = [&](const u32x4 (&w)[NL], int v) -> float {  // value v of the lane's 16
    if constexpr (XT == GEN_F32) return __uint_as_float(w[v / 4][v % 4]);
    else {
      const uint32_t u = w[v / 8][v % 8 / 2];
      if constexpr (XT == GEN_BF16) return __uint_as_float(v & 1 ? u & 0xFFFF0000u : u << 16);
      else return xt_to_f32<1>(v & 1 ? u >> 16 : u & 0xFFFFu);
    }
  };

  auto add_chunk = [&](const u32x4 (&w)[NL]) -> float {  // the lane's largest value of it
    float top = value(w, 0);
#pragma unroll
    for (int v = 1; v < 16; v++) top = fmaxf(top, value(w, v));
    if (top > mine.m) mine = rebase(mine, top, sc);
    const float m = mine.m == -INFINITY ? 0.f : mine.m;
#pragma unroll
    for (int v = 0; v < 16; v++) {
      const float z = (value(w, v) - m) * sc, p = __builtin_amdgcn_exp2f(z);
      mine.s += p;
      mine.e += p * fmaxf(z, -1000.f);  // 2^-1000 is 0, and so is its product with z
    }
    return top;
  };
  // waves of this workgroup that have values; what they all reach
  const int active = min(kWaves, chunks - part * kWaves), each = (a.k + active - 1) / active;
  auto post = [&]() {
    const float v = sorted_values(mine.m, lane);
    if (lane == each - 1) __hip_atomic_store(&reached[wave], v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
  };
  auto collect = [&](int c, const u32x4 (&w)[NL], float top) {
    float f = INFINITY;
#pragma unroll
    for (int i = 0; i < kWaves; i++)
      f = fminf(f, __hip_atomic_load(&reached[i], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP));
    // Values equal to f count; those equal to the list's floor come later and
    // lose to it.  A sum that is not a number may hide one among the values.
    const float above = fmaxf(floor_value, below(f));
    if (!__any(!(top <= above) || mine.s != mine.s)) return;
    auto index = [&](int v) { return c * kChunk + ((v / PER) * 64 + lane) * PER + v % PER; };
    uint32_t left = 0;  // the lane's values that pass, taken one a lane at a time
#pragma unroll
    for (int v = 0; v < 16; v++) left |= !(value(w, v) <= above) ? 1u << v : 0u;
    while (__any(left)) {
      const int v = left ? __builtin_ctz(left) : 0;
      constexpr int W = 4 * NL;
      uint32_t word[W];
#pragma unroll
      for (int i = 0; i < W; i++) word[i] = w[i / 4][i % 4];
      const int wi = XT == GEN_F32 ? v : v / 2;
#pragma unroll
      for (int bit = W / 2; bit; bit /= 2)
#pragma unroll
        for (int i = 0; i < bit; i++) word[i] = wi & bit ? word[i + bit] : word[i];
      float x;
      if constexpr (XT == GEN_F32) x = __uint_as_float(word[0]);
      else x = xt_to_f32<XT == GEN_F16 ? 1 : 0>(v & 1 ? word[0] >> 16 : word[0] & 0xFFFFu);
      const uint64_t kv = left && index(v) < a.V ? order_key(x, (uint32_t)index(v)) : 0;
      const uint64_t hits = __ballot(kv > floor);
      if (kv > floor) cand[wave][waiting + __popcll(hits & ((1ull << lane) - 1))] = kv;
      waiting += __popcll(hits);
      left &= left - 1;
      if (waiting >= 64) merge(64);
    }
  };

  u32x4 next[NL], w[NL];
  int c = part * kWaves + wave;
  if (c < chunks) {
    load_chunk(c, w);
    if (c + step < chunks) load_chunk(c + step, next);
    const float top = add_chunk(w);
    if (a.k > 0) {
      post();
      __syncthreads();
      collect(c, w, top);
    }
  } else if (a.k > 0) {
    if (lane == 0) reached[wave] = INFINITY;
    __syncthreads();
  }
  c += step;
  for (int n = 2; c < chunks; c += step, n++) {
#pragma unroll
    for (int j = 0; j < NL; j++) w[j] = next[j];
    if (c + step < chunks) load_chunk(c + step, next);
    const float top = add_chunk(w);
    if (a.k == 0) continue;
    if ((n & (n - 1)) == 0) post();
    collect(c, w, top);
  }
  if (waiting > 0) merge(waiting);

  // join the workgroup
#pragma unroll
  for (int d = 32; d; d >>= 1) mine = add(mine, Sums{__shfl_xor(mine.m, d), __shfl_xor(mine.s, d), __shfl_xor(mine.e, d)}, sc);
  if (lane == 0) sums[wave] = mine;
  lists[wave][lane] = list;
  __syncthreads();
  Sums all = sums[0];
#pragma unroll
  for (int w = 1; w < kWaves; w++) all = add(all, sums[w], sc);
  if (wave == 0 && a.k > 0) {
#pragma unroll
    for (int w = 1; w < kWaves; w++) merge64(list, lists[w][lane], lane);
  }

  // and the row's workgroups: (m, s, e, 0), then 64 keys of each
  if (a.split > 1) {
    constexpr int WORDS = 4 + 128;
    const __amdgpu_buffer_rsrc_t parts = buffer_rsrc(a.part, (uint32_t)(a.T * a.split * WORDS * 4));
    auto part_at = [&](int i) -> uint32_t { return (uint32_t)((t * a.split + i) * WORDS * 4); };
    if (wave == 0) {
      const uint32_t p = part_at(part);
      if (lane == 0)
        __builtin_amdgcn_raw_buffer_store_b128(
            u32x4{__float_as_uint(all.m), __float_as_uint(all.s), __float_as_uint(all.e), 0u}, parts, p, 0, kAgentScope);
      if (a.k > 0)
        __builtin_amdgcn_raw_buffer_store_b64(u32x2{(uint32_t)list, (uint32_t)(list >> 32)}, parts, p + 16 + lane * 8, 0,
                                              kAgentScope);
    }
    __builtin_amdgcn_s_waitcnt(0);  // the stores have completed
    __syncthreads();
    if (tid == 0) {
      const uint32_t old = __hip_atomic_fetch_add(a.cnt + t, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      arrived = old == (uint32_t)(a.split - 1);
      if (arrived) __hip_atomic_store(a.cnt + t, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    __syncthreads();
    if (!arrived) return;
    // wave w joins parts w, w + 4, .. in order, then the waves as before
    mine = Sums{-INFINITY, 0.f, 0.f};
    list = 0;
    constexpr int U = 8;  // parts in flight
    for (int i0 = wave; i0 < a.split; i0 += kWaves * U) {
      u32x4 v[U];
      u32x2 o[U];
#pragma unroll
      for (int u = 0; u < U; u++) {
        const uint32_t p = part_at(min(i0 + u * kWaves, a.split - 1));
        v[u] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(parts, p, 0, kAgentScope));
        if (a.k > 0)
          o[u] = __builtin_bit_cast(u32x2, __builtin_amdgcn_raw_buffer_load_b64(parts, p + 16 + lane * 8, 0, kAgentScope));
      }
#pragma unroll
      for (int u = 0; u < U; u++) {
        if (i0 + u * kWaves >= a.split) break;
        mine = add(mine, Sums{__uint_as_float(v[u][0]), __uint_as_float(v[u][1]), __uint_as_float(v[u][2])}, sc);
        if (a.k > 0) merge64(list, ((uint64_t)o[u][1] << 32) | o[u][0], lane);
      }
    }
    __syncthreads();
    if (lane == 0) sums[wave] = mine;
    lists[wave][lane] = list;
    __syncthreads();
    all = sums[0];
#pragma unroll
    for (int w = 1; w < kWaves; w++) all = add(all, sums[w], sc);
    if (wave == 0 && a.k > 0) {
#pragma unroll
      for (int w = 1; w < kWaves; w++) merge64(list, lists[w][lane], lane);
    }
  }

  const bool bad = all.s != all.s, nothing = all.m == -INFINITY;
  const float ls = logf(all.s);
  auto logprob = [&](float x) -> float {
    return bad ? NAN : x == -INFINITY ? -INFINITY : a.scale * (x - all.m) - ls;
  };
  for (int j = tid; j < a.n_tok; j += 256) {
    const int tok = a.tokens[t * a.n_tok + j];
    a.given[t * a.n_tok + j] = tok >= 0 && tok < a.V ? logprob(load<XT>(row, tok)) : NAN;
  }
  if (tid == 0) a.entropy[t] = bad ? NAN : nothing ? 0.f : ls - kLn2 * (all.e / all.s);
  if (tid < a.k) {
    a.top[t * a.k + tid] = logprob(key_value(list));
    a.ids[t * a.k + tid] = (int32_t)~(uint32_t)list;
  }
}

}  // namespace

void token_logprobs_plan(LogprobArgs& a, int cus, int64_t* part_bytes) {
  const int cpw = getenv("LP_CPW") ? atoi(getenv("LP_CPW")) : 1;
  const int chunks = (a.V + kChunk - 1) / kChunk, most = (chunks + kWaves * cpw - 1) / (kWaves * cpw);
  const int rw = getenv("LP_RW") ? atoi(getenv("LP_RW")) : kRowWgs;
  const int64_t want = ((int64_t)cus * rw + a.T - 1) / std::max<int64_t>(a.T, 1);
  a.split = (int)std::max<int64_t>(1, std::min<int64_t>(most, want));
  *part_bytes = a.split > 1 ? a.T * a.split * (4 + 128) * 4 : 0;
}

hipError_t launch_token_logprobs(const LogprobArgs& a, hipStream_t stream) {
  if (a.T == 0) return hipSuccess;
  if (a.V < 1 || a.k < 0 || a.k > kTopMax || a.k > a.V || a.split < 1 || (a.split > 1 && a.T > kSplitCounters) ||
      a.T * a.split > 0x7FFFFFFF)
    return hipErrorInvalidValue;
  const dim3 grid((unsigned)(a.T * a.split)), block(256);
  if (a.type == GEN_BF16) hipLaunchKernelGGL(token_logprobs_kernel<GEN_BF16>, grid, block, 0, stream, a);
  else if (a.type == GEN_F16) hipLaunchKernelGGL(token_logprobs_kernel<GEN_F16>, grid, block, 0, stream, a);
  else hipLaunchKernelGGL(token_logprobs_kernel<GEN_F32>, grid, block, 0, stream, a);
  return hipGetLastError();
}

}  // namespace mlxq
