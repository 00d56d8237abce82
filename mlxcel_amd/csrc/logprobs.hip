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
// to it, rescaled once a chunk.
//
// The alternatives are found in the same pass.  If each of the workgroup's A
// waves has ceil(k / A) lanes whose maxima so far reach f, or one wave k of them,
// then k values reach f and no lower one is among the k largest.  Each wave
// sorts its lanes' maxima after its 2nd, 8th, 32nd, .. chunk, which gives the
// workgroup its f.  A lane whose 16 values of a chunk reach f notes the chunk and
// its largest (a few instructions where none does); the notes are weighed against
// the last f at the end, when all but about k of them fall away, and the rest's
// values are read again, as numbers that order (value, index) pairs.  Mostly a
// few more than k reach f, and are sorted at once.  Where there are more than 256
// (many equal values), they are merged 64 at a time into sorted lists of the 64
// largest, one a wave.  The last workgroup of a row to arrive joins the row's in the same way.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <type_traits>

#include "common.hpp"
#include "kernels.hpp"
#include "wave.hpp"

namespace mlxq {

namespace {

constexpr int kWaves = 4, kChunk = 1024;  // values of a wave's chunk
// Values that a workgroup sorts at once, one a thread.  With 64 alternatives, 256
// against 128 and 64 (what is above goes through the lists): 64 rows of 50257 16.4 us,
// 32.1 and 29.6, 2000 of 3000 21.0, 33.8 and 42.7; with 20 all the same.
constexpr int kFew = 256;
// Workgroups a CU is given where rows are cut, each of at least two chunks a
// wave: each pays for its own start and end.  Rows of 100003 with 20 alternatives,
// 2 against 3 of them: float32 100 rows 20.8 and 23.4 us, 300 31.7 and 33.4, 600
// 47.8 and 65.0, bfloat16 300 30.3 and 30.1, 600 40.2 and 46.1; with 4,
// 300 rows of 151936 float32 logits 50.5 against 40.9.  8 rows of 262144 take
// 16 us, 21 with one chunk a wave.
constexpr int kRowWgs = 2;
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
  const float o = lane_xor<J>(v, lane);
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

// Over the wave's lanes, the same in each.
__device__ __forceinline__ Sums wave_sums(Sums v, float a, int lane) {
  const float M = wave_max(v.m, lane);
  v = rebase(v, M, a);
  return Sums{M, wave_sum(v.s, lane), wave_sum(v.e, lane)};
}

// ONCE: the logits are not kept in the caches.
template <int XT, bool ONCE>
__global__ __launch_bounds__(256, 4) void token_logprobs_kernel(const LogprobArgs a) {
  constexpr int PER = XT == GEN_F32 ? 4 : 8;  // values of a 16-byte load
  constexpr int NL = 16 / PER;                // loads of a lane and chunk
  constexpr uint32_t kNone = XT == GEN_F32 ? 0xFF800000u : XT == GEN_F16 ? 0xFC00FC00u : 0xFF80FF80u;  // -inf
  __shared__ uint64_t notes[kWaves][128], cand[kWaves][128], lists[kWaves][64];
  __shared__ uint64_t few[kFew], marked[kFew];
  __shared__ Sums sums[kWaves];
  __shared__ float reached[3][kWaves];
  __shared__ uint32_t arrived;
  __shared__ int count[2];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int64_t t = blockIdx.x / a.split;
  const int part = blockIdx.x - (int)t * a.split;  // of the row
  const char* row = static_cast<const char*>(a.logits) + t * a.row * (16 / PER);
  const float sc = a.scale * kLog2e;
  const int chunks = (a.V + kChunk - 1) / kChunk;
  const int step = a.split * kWaves;

  Sums mine = {-INFINITY, 0.f, 0.f};
  uint64_t list = 0, floor = 0;  // of values that were too many; keys up to `floor` cannot be among the k largest
  float floor_value = NAN;       // their value; not a number: there are none
  int waiting = 0, noted = 0;    // candidates, notes in LDS
  auto merge = [&](int n) __attribute__((always_inline)) {      // the first n <= 64 candidates
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

  // First value loaded for a chunk: the last chunk reaches back into the one
  // before it, whose values are then left out, so that every load is whole.
  auto start = [&](int c) { return min(c * kChunk, max(a.V - kChunk, 0)); };
  // Past the row's chunks its last one again: loads that need no branch.
  auto load_chunk = [&](int c, u32x4 (&w)[NL]) {
    c = min(c, chunks - 1);
    if (a.V >= kChunk) {
      const char* p = row + ((int64_t)start(c) + lane * PER) * (16 / PER);
#pragma unroll
      for (int j = 0; j < NL; j++) {
        const u32x4_e* q = reinterpret_cast<const u32x4_e*>(p + j * 1024);
        const u32x4_e v = ONCE ? __builtin_nontemporal_load(q) : *q;
        w[j] = u32x4{v[0], v[1], v[2], v[3]};
      }
      return;
    }
#pragma unroll
    for (int j = 0; j < NL; j++) {  // a short row, -inf past its end
      const int i = (j * 64 + lane) * PER;
#pragma unroll
      for (int e = 0; e < 4; e++) {
        w[j][e] = kNone;
        if constexpr (XT == GEN_F32) {
          if (i + e < a.V) w[j][e] = reinterpret_cast<const uint32_t*>(row)[i + e];
        } else {
          const uint16_t* p = reinterpret_cast<const uint16_t*>(row);
          if (i + 2 * e < a.V) w[j][e] = (w[j][e] & 0xFFFF0000u) | p[i + 2 * e];
          if (i + 2 * e + 1 < a.V) w[j][e] = (w[j][e] & 0xFFFFu) | (uint32_t)p[i + 2 * e + 1] << 16;
        }
      }
    }
  };
  auto index = [&](int c, int v) { return start(c) + ((v / PER) * 64 + lane) * PER + v % PER; };
  auto counts = [&](int c, int i) { return i >= c * kChunk && i < a.V; };
  auto value = [&](const u32x4 (&w)[NL], int v) -> float {  // value v of the lane's 16
    if constexpr (XT == GEN_F32) return __uint_as_float(w[v / 4][v % 4]);
    else {
      const uint32_t u = w[v / 8][v % 8 / 2];
      if constexpr (XT == GEN_BF16) return __uint_as_float(v & 1 ? u & 0xFFFF0000u : u << 16);
      else return xt_to_f32<1>(v & 1 ? u >> 16 : u & 0xFFFFu);
    }
  };

  auto add_chunk = [&](int c, u32x4 (&w)[NL]) -> float {  // the lane's largest value of it
    if (start(c) != c * kChunk) {
#pragma unroll
      for (int j = 0; j < NL; j++)
#pragma unroll
        for (int e = 0; e < 4; e++) {
          const int v = j * PER + e * (PER / 4);
          if (!counts(c, index(c, v))) w[j][e] = PER == 4 ? kNone : (w[j][e] & 0xFFFF0000u) | (kNone & 0xFFFFu);
          if (PER == 8 && !counts(c, index(c, v + 1))) w[j][e] = (w[j][e] & 0xFFFFu) | (kNone & 0xFFFF0000u);
        }
    }
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
  // waves of this workgroup that have values
  const int active = min(kWaves, chunks - part * kWaves), each = (a.k + active - 1) / active;
  auto post = [&]() __attribute__((always_inline)) {
    const float v = sorted_values(mine.m, lane);
    auto put = [&](int i, int r) {
      if (lane == r - 1) __hip_atomic_store(&reached[i][wave], v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
    };
    put(0, each);
    put(1, min(2 * each, a.k));
    put(2, a.k);
  };
  // What k values of the workgroup reach: `each` of every wave, twice as many of
  // two waves, or k of one.
  auto reach = [&]() -> float {
    float f = INFINITY, m1 = -INFINITY, m2 = -INFINITY, m3 = -INFINITY;
#pragma unroll
    for (int i = 0; i < kWaves; i++) {
      auto get = [&](int r) { return __hip_atomic_load(&reached[r][i], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP); };
      f = fminf(f, get(0));
      const float x = get(1);
      m2 = fmaxf(m2, fminf(m1, x));
      m1 = fmaxf(m1, x);
      m3 = fmaxf(m3, get(2));
    }
    return fmaxf(f, fmaxf(m2, m3));
  };
  // Value v of the 16 that lane l has of chunk c, its key (0: none).
  auto key_at = [&](uint32_t c, uint32_t l, int v) -> uint64_t {
    const int i = start(c) + ((v / PER) * 64 + (int)l) * PER + v % PER;
    return counts(c, i) ? order_key(load<XT>(row, i), (uint32_t)i) : 0;
  };
  // Notes: the largest value's order above the chunk and lane.
  auto note = [&](int c, float top) __attribute__((always_inline)) {
    // Values equal to f count; those equal to the list's floor come later and
    // lose to it.  A sum that is not a number may hide one among the values.
    const float above = fmaxf(floor_value, below(reach()));
    const bool hit = !(top <= above) || mine.s != mine.s;
    const uint64_t hits = __ballot(hit);
    if (hits == 0) return;
    if (hit)
      notes[wave][noted + __popcll(hits & ((1ull << lane) - 1))] =
          (order_key(mine.s != mine.s ? INFINITY : top, 0) & ~0xFFFFFFFFull) | (uint32_t)(c * 64 + lane);
    noted += __popcll(hits);
    if (noted < 64) return;
    // room: those that f has left behind go first
    post();
    const uint64_t least = order_key(reach(), 0xFFFFFFFFu);
    __builtin_amdgcn_wave_barrier();
    const uint64_t n0 = notes[wave][lane], n1 = lane + 64 < noted ? notes[wave][lane + 64] : 0;
    const uint64_t k0 = __ballot(n0 >= least), k1 = __ballot(n1 >= least);
    __builtin_amdgcn_wave_barrier();
    if (n0 >= least) notes[wave][__popcll(k0 & ((1ull << lane) - 1))] = n0;
    if (n1 >= least) notes[wave][__popcll(k0) + __popcll(k1 & ((1ull << lane) - 1))] = n1;
    noted = __popcll(k0) + __popcll(k1);
    while (noted >= 64) {  // too many reach it: their values go through the list
      __builtin_amdgcn_wave_barrier();
      noted -= 64;
      const uint32_t at = (uint32_t)notes[wave][noted + lane];
      for (int v = 0; v < 16; v++) {
        const uint64_t kv = key_at(at / 64, at % 64, v);
        const uint64_t h = __ballot(kv > floor);
        if (kv > floor) cand[wave][waiting + __popcll(h & ((1ull << lane) - 1))] = kv;
        waiting += __popcll(h);
        if (waiting >= 64) merge(64);
      }
      if (waiting > 0) merge(waiting);
    }
  };

  // two chunks at a time, the next two on their way
  u32x4 w0[NL], w1[NL];
  int c = part * kWaves + wave;
  load_chunk(c, w0);
  load_chunk(c + step, w1);
  if (tid < 2) count[tid] = 0;
  // the first given tokens' logits, needed at the end
  const int token = tid < a.n_tok ? a.tokens[t * a.n_tok + tid] : -1;
  const float token_logit = token >= 0 && token < a.V ? load<XT>(row, token) : NAN;
  bool posted = true;  // this wave's maxima as they stand
  if (c >= chunks) {
    if (lane == 0) {
      reached[0][wave] = INFINITY;
      reached[1][wave] = reached[2][wave] = -INFINITY;
    }
    __syncthreads();
  }
  for (int n = 1; c < chunks; n++, c += 2 * step) {
    float top0 = add_chunk(c, w0), top1 = -INFINITY;
    load_chunk(c + 2 * step, w0);
    const bool two = c + step < chunks;
    if (two) top1 = add_chunk(c + step, w1);
    load_chunk(c + 3 * step, w1);
    // after 2, 8, 32, .. chunks: 300 rows of 151936 float32 with 5 alternatives 42.2 us,
    // bfloat16 with 20 39.2; after 2, 4, 8, .. 43.5 and 40.5, after each two 45.7 and
    // 45.2, after the first two alone 42.8 and 40.1
    posted = a.k == 0 || ((n & (n - 1)) == 0 && (n & 0x55555555));
    if (posted && a.k > 0) post();
    if (n == 1) __syncthreads();  // the first maxima are shared before any value is noted
    if (a.k > 0) {
#pragma unroll 1
      for (int h = 0; h <= two; h++) note(c + h * step, h ? top1 : top0);
    }
  }

  if (!posted) post();
  mine = wave_sums(mine, sc, lane);
  if (lane == 0) sums[wave] = mine;
  // Puts the lanes' N keys of at least `least` into `to`, while it has room, and counts them.
  auto pick = [&](auto& key, uint64_t least, uint64_t* to, int* n) __attribute__((always_inline)) {
    constexpr int N = sizeof(key) / sizeof(key[0]);
    uint64_t hits[N];
    int total = 0;
#pragma unroll
    for (int i = 0; i < N; i++) {
      hits[i] = __ballot(key[i] != 0 && key[i] >= least);
      total += __popcll(hits[i]);
    }
    if (total == 0) return;
    int at = 0;
    if (lane == 0) at = atomicAdd(n, total);
    at = __builtin_amdgcn_readfirstlane(at);
#pragma unroll
    for (int i = 0; i < N; i++) {
      const int mine = at + __popcll(hits[i] & ((1ull << lane) - 1));
      if ((hits[i] >> lane & 1) && mine < kFew) to[mine] = key[i];
      at += __popcll(hits[i]);
    }
  };
  auto merge_lists = [&]() {
    lists[wave][lane] = list;
    __syncthreads();
    if (wave == 0) {
#pragma unroll
      for (int w = 1; w < kWaves; w++) merge64(list, lists[w][lane], lane);
    }
  };
  // The 64 largest of n <= kFew of `few`, sorted in wave 0's lanes.
  auto sort_few = [&](int n) {
    list = tid < n ? few[tid] : 0;
    if (wave * 64 < n) sort64(list, lane, n - wave * 64);
    if (n > 64) merge_lists();
  };
  __syncthreads();
  Sums all = sums[0];
#pragma unroll
  for (int w = 1; w < kWaves; w++) all = add(all, sums[w], sc);
  if (a.k > 0) {
    const uint64_t least = order_key(reach(), 0xFFFFFFFFu);
    uint64_t held[1] = {lane < noted ? notes[wave][lane] : 0}, listed[1] = {list};
    pick(held, least, marked, &count[0]);
    pick(listed, least, few, &count[1]);
    __syncthreads();
    if (count[0] <= kFew) {  // four lanes a note
      for (int i0 = 0; i0 < count[0]; i0 += 64) {
        const int i = i0 + tid / 4;
        const uint32_t at = i < count[0] ? (uint32_t)marked[i] : 0;
        uint64_t kv[4];
#pragma unroll
        for (int v = 0; v < 4; v++) kv[v] = i < count[0] ? key_at(at / 64, at % 64, 4 * (tid % 4) + v) : 0;
        pick(kv, least, few, &count[1]);
      }
      __syncthreads();
    }
    if (count[0] <= kFew && count[1] <= kFew) {
      sort_few(count[1]);
    } else {
      for (int n = 0; n < noted; n++) {  // a note at a time, its values in 16 lanes
        const uint32_t at = (uint32_t)notes[wave][n];
        const uint64_t kv = lane < 16 ? key_at(at / 64, at % 64, lane) : 0;
        const uint64_t h = __ballot(kv > floor);
        if (kv > floor) cand[wave][waiting + __popcll(h & ((1ull << lane) - 1))] = kv;
        waiting += __popcll(h);
        if (waiting >= 64) merge(64);
      }
      if (waiting > 0) merge(waiting);
      merge_lists();
    }
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
    // the sums in order, wave w those of parts w, w + 4, ..
    mine = Sums{-INFINITY, 0.f, 0.f};
    list = 0;
    auto load_list = [&](int i) -> uint64_t {
      const u32x2 o = __builtin_bit_cast(
          u32x2, __builtin_amdgcn_raw_buffer_load_b64(parts, part_at(i) + 16 + lane * 8, 0, kAgentScope));
      return ((uint64_t)o[1] << 32) | o[0];
    };
    constexpr int U = 8;  // parts of a wave in flight
    u32x4 v[U];
    uint64_t o[U];
    auto load_parts = [&](int i0) {
#pragma unroll
      for (int u = 0; u < U; u++) {
        const int i = min(i0 + u * kWaves, a.split - 1);
        v[u] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(parts, part_at(i), 0, kAgentScope));
        if (a.k > 0) o[u] = load_list(i);
      }
    };
    // What k keys reach: of the first 64 parts the ceil(k / r)-th largest of
    // their r-th keys, r about twice what each part has of the k.
    uint64_t least = 0, head = 0;
    const int n = min(a.split, 64), r = min(2 * ((a.k + n - 1) / n), a.k);
    if (a.k > 0) {
      const u32x2 h = __builtin_bit_cast(
          u32x2, __builtin_amdgcn_raw_buffer_load_b64(parts, part_at(min(lane, n - 1)) + 16 + (r - 1) * 8, 0, kAgentScope));
      head = lane < n ? ((uint64_t)h[1] << 32) | h[0] : 0;
    }
    load_parts(wave);
    if (tid == 0) count[1] = 0;
    if (a.k > 0) {
      sort64(head, lane, n);
      least = __shfl((unsigned long long)head, (a.k + r - 1) / r - 1);
    }
    __syncthreads();
    for (int i0 = wave; i0 < a.split; i0 += kWaves * U) {
      if (i0 != wave) load_parts(i0);
#pragma unroll
      for (int u = 0; u < U; u++) {
        if (i0 + u * kWaves < a.split)
          mine = add(mine, Sums{__uint_as_float(v[u][0]), __uint_as_float(v[u][1]), __uint_as_float(v[u][2])}, sc);
        else o[u] = 0;
      }
      if (a.k > 0) pick(o, least, few, &count[1]);
    }
    if (lane == 0) sums[wave] = mine;
    __syncthreads();
    all = sums[0];
#pragma unroll
    for (int w = 1; w < kWaves; w++) all = add(all, sums[w], sc);
    if (a.k > 0) {
      if (count[1] <= kFew) {
        sort_few(count[1]);
      } else {
        for (int i = wave; i < a.split; i += kWaves) merge64(list, load_list(i), lane);
        merge_lists();
      }
    }
  }

  const bool bad = all.s != all.s, nothing = all.m == -INFINITY;
  const float ls = logf(all.s);
  auto logprob = [&](float x) -> float {
    return bad || x != x ? NAN : x == -INFINITY ? -INFINITY : a.scale * (x - all.m) - ls;
  };
  for (int j = tid; j < a.n_tok; j += 256) {
    float x = token_logit;
    if (j >= 256) {
      const int other = a.tokens[t * a.n_tok + j];
      x = other >= 0 && other < a.V ? load<XT>(row, other) : NAN;
    }
    a.given[t * a.n_tok + j] = logprob(x);
  }
  if (tid == 0) a.entropy[t] = bad ? NAN : nothing ? 0.f : ls - kLn2 * (all.e / all.s);
  if (tid < a.k) {
    a.top[t * a.k + tid] = logprob(key_value(list));
    a.ids[t * a.k + tid] = (int32_t)~(uint32_t)list;
  }
}

}  // namespace

void token_logprobs_plan(LogprobArgs& a, int cus, int64_t* part_bytes) {
  const int chunks = (a.V + kChunk - 1) / kChunk, most = (chunks + 2 * kWaves - 1) / (2 * kWaves);
  const int64_t want = ((int64_t)cus * kRowWgs + a.T - 1) / std::max<int64_t>(a.T, 1);
  a.split = (int)std::max<int64_t>(1, std::min<int64_t>(most, want));
  *part_bytes = a.split > 1 ? a.T * a.split * (4 + 128) * 4 : 0;
}

hipError_t launch_token_logprobs(const LogprobArgs& a, hipStream_t stream) {
  if (a.T == 0) return hipSuccess;
  if (a.V < 1 || a.k < 0 || a.k > kTopMax || a.k > a.V || a.split < 1 || (a.split > 1 && a.T > kSplitCounters) ||
      a.T * a.split > 0x7FFFFFFF)
    return hipErrorInvalidValue;
  const dim3 grid((unsigned)(a.T * a.split)), block(256);
  // more logits than the caches would still hold for the next reader are not
  // kept there: 300 x 151936 float32 43.4 -> 40.5 us, bfloat16 (91 MB) 37.3 and 37.7
  const bool once = a.T * a.V * (a.type == GEN_F32 ? 4 : 2) > ((int64_t)128 << 20);
  auto run = [&](auto xt) {
    constexpr int XT = decltype(xt)::value;
    if (once) hipLaunchKernelGGL((token_logprobs_kernel<XT, true>), grid, block, 0, stream, a);
    else hipLaunchKernelGGL((token_logprobs_kernel<XT, false>), grid, block, 0, stream, a);
  };
  if (a.type == GEN_BF16) run(std::integral_constant<int, GEN_BF16>{});
  else if (a.type == GEN_F16) run(std::integral_constant<int, GEN_F16>{});
  else run(std::integral_constant<int, GEN_F32>{});
  return hipGetLastError();
}

}  // namespace mlxq
