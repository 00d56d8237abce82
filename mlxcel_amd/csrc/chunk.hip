// chunk.hip — attention of several new tokens per sequence over a paged
// key-value cache on gfx950.
//
//   s_j = cap(q_i . k_j * scale)   over the keys j that token i sees: (p - window, p], p = length - new + i
//   o_i = sum_j exp(s_j - m) v_j / (sum_j exp(s_j - m) + exp(sink - m))
//
// A tile is up to 128 rows, (token, query head) pairs of one key head, over the
// keys that any of them sees.  Its workgroup takes 64 keys a step (32 of wide
// 32-bit heads): the step's K and V rows go to LDS directly while the step before
// is worked on, in the order of their keys, whatever pages they come from.  K is
// 32 keys ahead of V, so that the scores of 32 keys are worked out beside the
// values of the 32 before.  Each of the four waves has 32 rows, with O, the
// running maximum and the running sum in registers.  Both
// products are 32x32 MFMAs whose operands need no exchange between lanes:
//   S^T[key][row] = K Q^T: lane (c, g) = (lane % 32, lane / 32) ends with keys
//     8 i + 4 g + e (i, e < 4) of row c, so a row's maximum and sum are taken
//     within a lane and its neighbour lane ^ 32;
//   O^T[d][row] += V^T P^T: the lane's keys are those it holds P of; V comes out
//     of LDS transposed (16-bit types: four keys of a column a read).
// 16-bit products take P as the sum of two 16-bit numbers: bfloat16 ones leave
// out at most 2^-17 of it, float16 ones 2^-23 or 2^-39 of the largest.  One number
// would leave out 2^-9, as much as the result's own rounding, for a third of the
// matrix work.
//
// Values that are not finite would reach the rows that do not see their key (0 inf), and scores past
// 2^25 would take probabilities out of their type: a tile whose results are not all finite, or one of whose rows has
// a largest probability far from 1, is worked out again, where exponents are exact and 32 keys with such a value
// are taken one at a time, each for the rows that see it.
//
// Many new tokens are bound by the matrix instructions, at the clock that the
// card keeps under them: 2048 tokens of 32768 of 32 heads of 128 (8 key heads) in
// bfloat16 1400 us (1385 to 1470 by the card), that is 762 TFLOP/s or, with P's second number
// counted, 1144 (the matrix instructions alone: 1170 us).  Few are bound by HBM
// and by the join of what was cut: 16 sequences of 5 tokens over 43000 keys of 4
// key heads 42 us for 88 MB.  Short tiles (a window of 128 tokens) are bound by their vector
// operations and by what a tile's start waits for: five prompts of 1500 tokens of 64 heads of 64, 83 us.
//
// The work is cut evenly whatever the lengths: a tile counts its keys and kAround
// more, and workgroup w takes [w n, (w + 1) n) of all tiles laid end to end,
// rounded to whole steps.  Lengths and starts are on the device, so each workgroup
// finds its first tile from a scan over the sequences and, among the tiles of
// one, from the closed form of their sum.  A tile that crosses a workgroup's end
// leaves its sum, maximum and output so far in scratch; the last of its workgroups
// to arrive joins them, in the order of the keys, so the result does not depend on
// who came last.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cfloat>
#include <type_traits>

#include "common.hpp"
#include "kernels.hpp"
#include "wave.hpp"

namespace mlxq {

namespace {

constexpr int kWaves = 4, kRows = 32 * kWaves;
constexpr float kLog2e = 1.44269504088896340736f;

// What a tile's start and end cost, in keys.
constexpr int kAround = 192;
// Keys of a tile that is not cut, and the least units that a workgroup takes.
constexpr int kWhole = 256, kLeast = 128;

// Results of other workgroups that are read at a time, and how many times 16 bytes of each lane.
constexpr int kFlight = 8, kUnits = 4;

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
// 16-byte loads of element alignment (rows of any stride)
typedef uint32_t u32x4_e __attribute__((ext_vector_type(4), aligned(2)));

// XT: GEN_BF16 / GEN_F16 / GEN_F32.  DP: head width rounded up.
template <int XT, int DP>
struct Geo {
  static constexpr bool F32 = XT == GEN_F32;
  static constexpr int ES = F32 ? 4 : 2;
  static constexpr int CE = 16 / ES;            // elements of 16 bytes
  static constexpr int C = DP / CE;             // 16-byte chunks of a row
  static constexpr int NC = (C + 7) / 8;        // blocks of 8 chunks
  static constexpr int DT = DP / 32;            // 32-column tiles of O
  static constexpr int KEYS = DP * ES <= (F32 ? 256 : 512) ? 64 : 32;  // of a step
  static constexpr int KT = KEYS / 32;
  // A step in LDS: K, then V; each in blocks [8 chunks of the row][KEYS rows][128 bytes],
  // so that a wave's 64 lanes fill 8 rows of a block in their order.
  static constexpr int TILE = NC * KEYS * 128;
  // Workgroups a CU holds: by registers.  16-bit heads of 64, 2 instead of 3: short tiles (five
  // prompts of 1500 with a window of 128) take 101 us instead of 83, 5 tokens of each of 16 sequences
  // 28.2 instead of 27.0, long ones (2048 tokens of 32768) 899 either way.  float32 heads of 96 (128), 64
  // keys a step and one workgroup instead of 32 keys and two: 300 tokens of 14636 537 (681) us
  // instead of 472 (630), 5 new ones of each of 16 sequences 112 (141) instead of 98 (135).
  static constexpr int WGS = DP * ES <= 128 ? 3 : DP * ES <= (F32 ? 512 : 256) ? 2 : 1;
};
// Chunk p of row r of a block lies at place p ^ swizzle(r).  K is read one chunk
// of 16 rows at a time, which then hit all banks; V four rows of 64 bytes.
__device__ __forceinline__ int swizzle_k(int r) { return (r >> 1) & 7; }
__device__ __forceinline__ int swizzle_v(int r) { return (r >> 1 & 1) * 4; }

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

// v less the low (high) half of w, exact where w holds v rounded; one instruction.  minus
// is in a register.  bfloat16: -1 in that half, 0 in the other (the compiler writes a low
// bfloat16 -1 as the inline constant -1.0, whose bits are in the high half).  float16: -1 in
// 32 bits (of a subtraction the compiler makes a conversion more).
template <int XT, int HI>
__device__ __forceinline__ float less(float v, uint32_t w, uint32_t minus) {
  if constexpr (XT == GEN_BF16)
    return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2, w), __builtin_bit_cast(bf16x2, minus), v, false);
  else return fmaf((float)__builtin_bit_cast(_Float16, (uint16_t)(HI ? w >> 16 : w)), __uint_as_float(minus), v);
}

template <int XT>
__device__ __forceinline__ f32x16 mfma32(u32x4 a, u32x4 b, f32x16 c) {
  if constexpr (XT == GEN_BF16)
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

// LDS by pointers of its own: 32 bits, and what is constant goes into the instruction.
typedef __attribute__((address_space(3))) char Lds;
template <typename T>
__device__ __forceinline__ T lds_read(const Lds* p) {
  return *(const __attribute__((address_space(3))) T*)p;
}
template <typename T>
__device__ __forceinline__ void lds_write(Lds* p, T v) {
  *(__attribute__((address_space(3))) T*)p = v;
}

// Four rows of the lane's column: row i of the 16 lanes' 4 x 16 elements is read
// by lanes 4 i .. 4 i + 3, lane j gets column j.
__device__ __forceinline__ u32x2 read_transposed(const Lds* p) {
  return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)p));
}

// 16 bytes a lane to LDS, in the order of the lanes.
__device__ __forceinline__ void to_lds(const char* from, Lds* to) {
  __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)from,
                                   (__attribute__((address_space(3))) void*)to, 16, 0, 0);
}

// All waves' loads to LDS have arrived, and all have read what is filled next.
__device__ __forceinline__ void step_barrier() {
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
}

// Four values to consecutive places.
template <int XT>
__device__ __forceinline__ void store4(void* p, int64_t i, f32x4 v) {
  if constexpr (XT == GEN_F32) {
    typedef float f32x4_e __attribute__((ext_vector_type(4), aligned(4)));
    *reinterpret_cast<f32x4_e*>(static_cast<float*>(p) + i) = f32x4_e{v[0], v[1], v[2], v[3]};
  } else {
    typedef uint32_t u32x2_e __attribute__((ext_vector_type(2), aligned(2)));
    uint32_t h[4];
#pragma unroll
    for (int e = 0; e < 4; e++) h[e] = f32_to_xt<XT == GEN_F16 ? 1 : 0>(v[e]);
    *reinterpret_cast<u32x2_e*>(static_cast<uint16_t*>(p) + i) = u32x2_e{h[0] | h[1] << 16, h[2] | h[3] << 16};
  }
}

// Two values as a pair of 16-bit results, rounded as store4 does.
template <int XT>
__device__ __forceinline__ uint32_t pack_out(float lo, float hi) {
  return f32_to_xt<XT == GEN_F16 ? 1 : 0>(lo) | f32_to_xt<XT == GEN_F16 ? 1 : 0>(hi) << 16;
}

// Probabilities are held as 2^lift p: in float16 their largest is then 2^14, and
// those down to 2^-28 of it keep all their bits (smaller ones differ by 2^-39 of it).
template <int XT>
constexpr float kLift = XT == GEN_F16 ? 14.f : 0.f;

// exp2(a - b), 0 where a is -inf (also where b is)
__device__ __forceinline__ float exp2_diff(float a, float b) {
  return __builtin_amdgcn_exp2f(a - (b == -INFINITY ? 0.f : b));
}

// The new tokens of a sequence that have a position, and its tiles.
struct Seq {
  int first, n, p0;  // row of the first of n tokens, its position
  int tiles;         // of a head: tile_tokens tokens each
  int late;          // tiles up to this one see key 0
  int skip;          // rows before `first` without a position
};
__device__ __forceinline__ Seq seq_of(const ChunkAttnArgs& a, int start, int end, int length) {
  const int st = min(max(start, 0), a.T), all = min(max(end, st), a.T) - st;
  const int len = (int)min((int64_t)max(length, 0), (int64_t)a.width * a.page);
  Seq s;
  s.skip = max(all - len, 0);
  s.n = all - s.skip;
  s.first = st + s.skip;
  s.p0 = len - s.n;
  // v / tile_tokens: (v + 1/2) / tile_tokens is no nearer to a whole number than 1/2 of one
  s.tiles = (int)((s.n + a.tile_tokens - 0.5) * a.inv_tile_tokens);
  const int lo = s.p0 - a.window + 1;
  s.late = a.window == 0 ? s.tiles : lo > 0 ? 0 : (int)((0.5 - lo) * a.inv_tile_tokens) + 1;
  return s;
}
__device__ __forceinline__ int tile_lo(const ChunkAttnArgs& a, const Seq& s, int j) {
  return a.window > 0 ? max(0, s.p0 + j * a.tile_tokens - a.window + 1) : 0;
}
__device__ __forceinline__ int tile_hi(const ChunkAttnArgs& a, const Seq& s, int j) {
  return s.p0 + min(s.n, (j + 1) * a.tile_tokens);
}
// The units of a tile are its keys and kAround more.  All counts of units are whole
// numbers below 2^52, held as doubles: their products and sums cost a fraction of 64-bit ones.
// sum over tiles i < j of kAround + tile_hi(i) - tile_lo(i)
__device__ __forceinline__ double before(const ChunkAttnArgs& a, const Seq& s, int j) {
  const double tt = a.tile_tokens, J = j, L = s.late;
  double sum = J * (kAround + s.p0) + tt * (J * (J + 1) * 0.5);
  if (j == s.tiles) sum -= J * tt - s.n;
  if (j > s.late) sum -= (J - L) * (s.p0 - a.window + 1) + tt * ((J * (J - 1) - L * (L - 1)) * 0.5);
  return sum;
}
// The tiles of a head are taken shortest, longest, second shortest, ..: tile number q
// in that order, and the units of those before it.  Two neighbours together then cost
// about the same everywhere, so that workgroups begin near the same key of their tiles
// and find each other's keys in L2 (2048 tokens of 32768: 6% of the requests missed it
// instead of 66%).
__device__ __forceinline__ int tile_at(const Seq& s, int q) { return q & 1 ? s.tiles - 1 - q / 2 : q / 2; }
__device__ __forceinline__ double units_before(const ChunkAttnArgs& a, const Seq& s, double head, int q) {
  return before(a, s, (q + 1) / 2) + (q > 1 ? head - before(a, s, s.tiles - q / 2) : 0.0);
}
// v / d, whole
__device__ __forceinline__ double divide(double v, double d) {
  double q = floor(v / d);
  if (q * d > v) q -= 1.0;
  if ((q + 1.0) * d <= v) q += 1.0;
  return q;
}

__device__ __forceinline__ double lane_value(double v, int from) {
  const uint64_t u = __builtin_bit_cast(uint64_t, v);
  const uint32_t lo = __builtin_amdgcn_readlane((uint32_t)u, from), hi = __builtin_amdgcn_readlane((uint32_t)(u >> 32), from);
  return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
__device__ __forceinline__ Seq lane_value(const Seq& s, int from) {
  return Seq{(int)__builtin_amdgcn_readlane(s.first, from), (int)__builtin_amdgcn_readlane(s.n, from),
             (int)__builtin_amdgcn_readlane(s.p0, from),    (int)__builtin_amdgcn_readlane(s.tiles, from),
             (int)__builtin_amdgcn_readlane(s.late, from),  (int)__builtin_amdgcn_readlane(s.skip, from)};
}

// Words of one partial result: O as the registers of `waves` waves hold it, 16 bytes of
// each lane after the other, then (m, l) of their rows.
constexpr int part_words(int waves, int DP) { return waves * (32 * DP + 64); }

template <int XT, int DP>
__global__ __launch_bounds__(256, (Geo<XT, DP>::WGS)) void chunk_attention_kernel(const ChunkAttnArgs a) {
  using G = Geo<XT, DP>;
  constexpr int kKeys = G::KEYS;
  // Keys and values of two steps.  Objects of their own, with one sum from each to what is
  // read of it, so that the compiler sees that what is being filled is not what is read and
  // does not wait for it (it did, at 1700 us for 2048 tokens of 32768).
  __shared__ __align__(16) char k_obj0[G::TILE], v_obj0[G::TILE], k_obj1[G::TILE], v_obj1[G::TILE];
  Lds *const k_lds0 = (Lds*)k_obj0, *const v_lds0 = (Lds*)v_obj0, *const k_lds1 = (Lds*)k_obj1, *const v_lds1 = (Lds*)v_obj1;
  __shared__ uint32_t arrived, odd;  // odd: the tile has to be worked out again
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int c = lane & 31, g = lane >> 5;
  // neighbours in the order of the keys on one XCD
  const int w = a.wgs % 8 == 0 ? (int)(blockIdx.x % 8) * (a.wgs / 8) + (int)(blockIdx.x / 8) : (int)blockIdx.x;
  const int per = a.Hq / a.Hkv, hp = a.tile_heads, tiles_h = (per + hp - 1) / hp, heads_b = a.Hkv * tiles_h;

  // Where this workgroup's work begins and ends: head and tile number of sequence b (past
  // the last: the next one's first), key of its range.
  struct Bound {
    int b, hh, nth, key;
    double base;  // of the sequence, among all units
    __device__ __forceinline__ bool ahead_of(const Bound& o) const {
      return b != o.b ? b < o.b : hh != o.hh ? hh < o.hh : nth != o.nth ? nth < o.nth : key < o.key;
    }
  };
  auto load_seq = [&](int b) __attribute__((always_inline)) -> Seq {
    const int s = __builtin_amdgcn_readfirstlane(a.starts[b]), e = __builtin_amdgcn_readfirstlane(a.starts[b + 1]);
    return lane_value(seq_of(a, s, e, __builtin_amdgcn_readfirstlane(a.lengths[b])), 0);
  };
  auto bound_at = [&](double off, int b, const Seq& s, double base) __attribute__((always_inline)) -> Bound {
    const double head = before(a, s, s.tiles), hh = divide(off, head);
    off -= hh * head;
    int lo = 0, hi = s.tiles;  // the last tile that begins at or before off: a lane looks at each
    while (hi - lo > 1) {
      const int by = (hi - lo + 63) >> 6, q = lo + lane * by;
      const int n = __popcll(__ballot(q < hi && units_before(a, s, head, q) <= off));
      hi = min(hi, lo + n * by);
      lo += (n - 1) * by;
    }
    off -= units_before(a, s, head, lo);
    const int j = tile_at(s, lo), keys = tile_hi(a, s, j) - tile_lo(a, s, j), r = (int)off - kAround;
    // a tile that is not cut belongs to the workgroup that begins it
    const bool past = keys <= kWhole && off > 0.0;
    return Bound{b, (int)__builtin_amdgcn_readfirstlane((int)hh), (int)__builtin_amdgcn_readfirstlane(lo + past),
                 (int)__builtin_amdgcn_readfirstlane(past || r <= 0 ? 0 : r / kKeys * kKeys), base};
  };
  auto clear = [&](const Seq& s) __attribute__((always_inline)) {  // rows without a position
    const int64_t from = (int64_t)(s.first - s.skip) * a.Hq * a.D, n = (int64_t)s.skip * a.Hq * a.D;
    for (int64_t i = 4 * tid; i < n; i += 1024) store4<XT>(a.out, from + i, f32x4{0.f, 0.f, 0.f, 0.f});
  };
  double total, n;
  Bound at, end;
  Seq sq{};  // sequence at.b
  {
    auto units_of = [&](const Seq& s) __attribute__((always_inline)) { return heads_b * before(a, s, s.tiles); };
    auto per_group = [&]() __attribute__((always_inline)) { return fmax(floor(total * a.inv_wgs) + 1.0, (double)kLeast); };
    double sum, mine;
    auto scan = [&](int lanes) __attribute__((always_inline)) {
      for (int s = 1; s < lanes; s <<= 1) {
        const double o = __shfl_up(sum, s);
        if (lane >= s) sum += o;
      }
    };
    if (a.B <= 64) {  // each wave finds them by itself, sequence i in lane i
      const Seq s = lane < a.B ? seq_of(a, a.starts[lane], a.starts[lane + 1], a.lengths[lane]) : Seq{};
      sum = mine = units_of(s);
      scan(a.B);
      total = lane_value(sum, a.B - 1);
      n = lane_value(per_group(), 0);
      end = Bound{a.B, 0, 0, 0, total};
#pragma unroll 1
      for (int i = 0; i < 2; i++) {
        at = end;
        const double p = (w + 1 - i) * n;
        end = Bound{a.B, 0, 0, 0, total};
        if (p < total) {
          const int b = __builtin_ctzll(__ballot(sum - mine <= p && p < sum));
          const double base = lane_value(sum - mine, b);
          sq = lane_value(s, b);
          end = bound_at(p - base, b, sq, base);
        }
      }
      const Bound first = end;  // the second round looked for the beginning
      end = at;
      at = first;
      for (uint64_t none = __ballot(s.skip > 0); none; none &= none - 1) {
        const int b = __builtin_ctzll(none);
        if (b % a.wgs == w) clear(lane_value(s, b));
      }
    } else {  // thread i sums those of its share
      double* sums = reinterpret_cast<double*>(k_obj0);
      Bound* bound = reinterpret_cast<Bound*>(k_obj0 + 64);
      const int share = (a.B + 255) / 256, b0 = min(tid * share, a.B), b1 = min(b0 + share, a.B);
      mine = 0.0;
      for (int b = b0; b < b1; b++) mine += units_of(seq_of(a, a.starts[b], a.starts[b + 1], a.lengths[b]));
      sum = mine;
      scan(64);
      if (lane == 63) sums[wave] = sum;
      __syncthreads();
      double ahead = sum - mine;
      total = 0.0;
#pragma unroll
      for (int i = 0; i < kWaves; i++) {
        if (i < wave) ahead += sums[i];
        total += sums[i];
      }
      total = lane_value(total, 0);
      n = lane_value(per_group(), 0);
#pragma unroll 1
      for (int i = 0; i < 2; i++) {
        const double p = (w + i) * n;
        if (p >= total) {
          if (tid == 0) bound[i] = Bound{a.B, 0, 0, 0, total};
        } else if (ahead <= p && p < ahead + mine) {
          double base = ahead;
          for (int b = b0; b < b1; b++) {
            const double u = units_of(seq_of(a, a.starts[b], a.starts[b + 1], a.lengths[b]));
            if (p < base + u) {
              bound[i] = Bound{b, 0, 0, 0, base};
              break;
            }
            base += u;
          }
        }
      }
      for (int b = w; b < a.B; b += a.wgs) {
        const Seq s = load_seq(b);
        if (s.skip > 0) clear(s);
      }
      __syncthreads();
#pragma unroll 1
      for (int i = 1; i >= 0; i--) {
        end = at;
        at.b = __builtin_amdgcn_readfirstlane(bound[i].b);
        at.hh = at.nth = at.key = 0;
        at.base = lane_value(bound[i].base, 0);
        if (at.b < a.B) {
          sq = load_seq(at.b);
          at = bound_at((w + i) * n - at.base, at.b, sq, at.base);
        }
      }
      __syncthreads();  // the LDS is free again
    }
  }
  if (!at.ahead_of(end)) return;

  // Of two workgroups of a CU the older one's waves go first, and it is done at 3/4 of the
  // time (205 of 270 us); so the younger one goes first in every other step (three prompts of 1000 tokens
  // beside 61 single tokens 254 us instead of 258, 2048 tokens of 32768 1390 instead of 1411).
  const bool later = blockIdx.x >= gridDim.x / 2;
  uint32_t minus_lo = XT == GEN_F16 ? 0xBF800000u : 0x0000BF80u, minus_hi = 0xBF800000u;
  asm volatile("" : "+s"(minus_lo), "+s"(minus_hi));
  // A thread brings place lane % 8 of every block of rows 8 wave + lane / 8 (+ 32) of a step.
  const int my_row8 = 8 * wave + (lane >> 3), k_chunk = (lane & 7) ^ swizzle_k(my_row8), v_chunk = (lane & 7) ^ swizzle_v(my_row8);
  const int chunks = a.D / G::CE;
  // What a lane reads of a block: chunk 2 i + g of K's row c, i < 4; the row and the 8 bytes of
  // V's 32 columns, even and odd ones of two.  One sum each, which the compiler leaves alone: of
  // the parts it would make pointers that it no longer knows to be V's.
  int k_lane[4], v_lane[2];
  {
    const int i16 = lane & 15, r = 4 * g + (i16 >> 2), ch = 2 * ((lane >> 4) & 1) + ((i16 >> 1) & 1);
#pragma unroll
    for (int i = 0; i < 4; i++) k_lane[i] = c * 128 + ((2 * i + g) ^ swizzle_k(c)) * 16;
#pragma unroll
    for (int i = 0; i < 2; i++) {
      // of one block past the head the last chunk of the head instead
      const int at = DP == 64 ? min(4 * i + ch, a.D / G::CE - 1) : 4 * i + ch;
      v_lane[i] = r * 128 + (at ^ swizzle_v(r)) * 16 + (i16 & 1) * 8;
    }
    asm volatile("" : "+v"(k_lane[0]), "+v"(k_lane[1]), "+v"(k_lane[2]), "+v"(k_lane[3]), "+v"(v_lane[0]), "+v"(v_lane[1]));
  }
  // The chunks past the head are zero and stay so: K's count in the scores, and values that are not finite, whatever
  // lay there, would send every tile the slow way.  (V's of a kernel of one block, where results go through, are not read.)
  if (DP != a.D) {
    for (int i = tid; i < G::TILE / 16; i += 256) {
      for (char* p : {k_obj0, v_obj0, k_obj1, v_obj1}) reinterpret_cast<u32x4*>(p)[i] = u32x4{0u, 0u, 0u, 0u};
    }
  }
  // Scores in units of log2 e are `scale` times the product (the tanh of a soft
  // cap); a negative scale's sign goes to Q, so that the largest product is the largest score.
  // A scale of 0 is the smallest number instead: scores then do not differ either, and -inf stays what it is.
  const float scale = fmaxf((a.softcap > 0.f ? a.softcap : fabsf(a.scale)) * kLog2e, FLT_MIN);
  const float cap_in = a.softcap > 0.f ? fminf(2.f * kLog2e * fabsf(a.scale) / a.softcap, FLT_MAX) : 0.f;
  const __amdgpu_buffer_rsrc_t parts = buffer_rsrc(a.part, (uint32_t)((int64_t)4 * a.wgs * a.slot_words * 4));

  double head_units = lane_value(before(a, sq, sq.tiles), 0);
  while (at.ahead_of(end)) {
    if (at.nth >= sq.tiles) {
      at.nth = at.key = 0;
      if (++at.hh >= heads_b || sq.tiles == 0) {
        at.hh = 0;
        at.base = lane_value(at.base + heads_b * head_units, 0);
        if (++at.b >= a.B) break;
        sq = load_seq(at.b);
        head_units = lane_value(before(a, sq, sq.tiles), 0);
      }
      continue;
    }
    const int j = tile_at(sq, at.nth), hk = tiles_h == 1 ? at.hh : at.hh / tiles_h, ht = at.hh - hk * tiles_h;
    const int heads = min(hp, per - hp * ht), head0 = hk * per + hp * ht;
    const int tok0 = j * a.tile_tokens, toks = min(a.tile_tokens, sq.n - tok0), rows = toks * heads;
    const int lo = tile_lo(a, sq, j), hi = tile_hi(a, sq, j);
    const bool ends = at.b == end.b && at.hh == end.hh && at.nth == end.nth;
    const int k0 = lo + at.key, k1 = ends ? min(hi, lo + end.key) : hi;
    // the tile's workgroups
    int w0 = w, w1 = w;
    if (k0 > lo || k1 < hi) {
      const double p0 = at.base + at.hh * head_units + units_before(a, sq, head_units, at.nth) + kAround;
      w0 = __builtin_amdgcn_readfirstlane((int)divide(p0 + kKeys + n - 1.0, n)) - 1;
      w1 = __builtin_amdgcn_readfirstlane((int)divide(p0 + (hi - lo) + n - 1.0, n)) - 1;
    }

    // this wave's rows, and the keys that any of them sees
    // row / heads for rows below 128 and at most 128 heads
    const uint32_t inv_heads = heads == hp ? a.inv_tile_heads : (65536 + heads - 1) / heads;
    auto token_of = [&](int row) __attribute__((always_inline)) -> int { return (int)(row * inv_heads >> 16); };
    const int r0 = 32 * wave, my_row = min(r0 + c, rows - 1), my_tok = token_of(my_row);
    const int pos = sq.p0 + tok0 + my_tok;
    const bool busy = r0 < rows;
    const int see1 = min(pos + 1, k1), see0 = a.window > 0 ? max(0, pos + 1 - a.window) : 0;
    const int wave_hi = sq.p0 + tok0 + token_of(min(r0 + 31, rows - 1)) + 1, first_hi = sq.p0 + tok0 + token_of(min(r0, rows - 1)) + 1;
    const int wave_lo = a.window > 0 ? max(0, first_hi - a.window) : 0, last_lo = a.window > 0 ? max(0, wave_hi - a.window) : 0;

    const char* qp = static_cast<const char*>(a.q) +
                     ((int64_t)(sq.first + tok0 + my_tok) * a.q_tok + (head0 + my_row - my_tok * heads) * a.q_head) * G::ES;
    u32x4 qf[G::C / 2];
    // Q is asked for behind the first K and looked at when that is there (before it: short tiles 81.9 us
    // instead of 83.0, prompts beside single tokens 255 instead of 254)
    auto load_q = [&]() __attribute__((always_inline)) {
#pragma unroll
      for (int i = 0; i < G::C / 2; i++) {
        const int d = (2 * i + g) * G::CE;
        const u32x4_e v = *reinterpret_cast<const u32x4_e*>(qp + (DP == a.D || d < a.D ? d : 0) * G::ES);
        qf[i] = u32x4{v[0], v[1], v[2], v[3]};
      }
    };
    auto finish_q = [&]() __attribute__((always_inline)) {
      if (DP != a.D) {
#pragma unroll
        for (int i = 0; i < G::C / 2; i++) qf[i] = (2 * i + g) * G::CE < a.D ? qf[i] : u32x4{0u, 0u, 0u, 0u};
      }
      if (a.scale < 0.f) {
#pragma unroll
        for (int i = 0; i < G::C / 2; i++) qf[i] ^= G::F32 ? 0x80000000u : 0x80008000u;
      }
    };
    f32x16 o[G::DT];
    float m, l, off;  // off: what is added to a score before its exponential is taken

    const int32_t* table = a.table + at.b * a.table_row;
    const char* kb = static_cast<const char*>(a.k) + hk * a.k_head + k_chunk * 16;
    const char* vb = static_cast<const char*>(a.v) + hk * a.v_head + v_chunk * 16;
    // A thread's rows of a step from key k on are k + my_row8 (+ 32) of V and 32 keys more of K:
    // the scores of 32 keys are worked out beside the values of the 32 before them.
    int entry[G::KT + 1], in_page[G::KT + 1];
    int64_t v_off = 0;  // bytes to the V row that comes next
    // table entries of keys from + my_row8 (+ 32); past the range they are the last key's
    auto look_row = [&](int from, int t) __attribute__((always_inline)) {
      const uint32_t key = min(from + my_row8, hi - 1);
      const uint32_t slot = __umulhi(key << 2, a.page_mul) >> (a.page_shift - 30);
      in_page[t] = key - slot * a.page;
      entry[t] = table[slot];
    };
    auto look = [&](int from) __attribute__((always_inline)) {
#pragma unroll
      for (int t = 0; t < G::KT; t++) look_row(from + 32 * t, t);
    };
    // bytes to the looked-up row t in a pool of these strides
    auto place = [&](int t, int64_t page_bytes, int64_t tok_bytes) __attribute__((always_inline)) -> int64_t {
      const int pid = min(max(entry[t], 0), a.pages - 1);
      if (a.direct) return (int64_t)((uint64_t)(uint32_t)pid * (uint32_t)page_bytes + (uint64_t)(uint32_t)in_page[t] * (uint32_t)tok_bytes);
      return pid * page_bytes + in_page[t] * tok_bytes;
    };
    // Of a row only the last block may be part full.  It is looked at where the kernel's width has a part
    // full one anyway, or the head is narrower (heads of 128 take the same with a look in every step: 2048
    // tokens of 32768 1383 and 1388 us).
    constexpr bool kLook = G::C % 8 != 0;
    // a row to LDS without passing through registers
    auto rows_to_lds = [&](const char* from, int chunk, Lds* to, int row) __attribute__((always_inline)) {
#pragma unroll
      for (int i = 0; i < G::NC; i++)
        if (8 * i + 8 <= G::C || 8 * i + chunk < chunks) to_lds(from + i * 128, to + (i * kKeys + row + 8 * wave) * 128);
    };
    // a row to LDS, rows `row` on of the blocks
    auto bring_row = [&](const char* from, int chunk, Lds* to, int row) __attribute__((always_inline)) {
      if (a.direct) {  // 16-byte aligned, strides of 32 bits
        if (kLook || DP == a.D) {
          rows_to_lds(from, chunk, to, row);
        } else {
#pragma unroll
          for (int i = 0; i < G::NC; i++)
            if (8 * i + chunk < chunks) to_lds(from + i * 128, to + (i * kKeys + row + 8 * wave) * 128);
        }
      } else {
#pragma unroll
        for (int i = 0; i < G::NC; i++)
          if (8 * i + chunk < chunks) {
            const u32x4_e x = *reinterpret_cast<const u32x4_e*>(from + i * 128);
            lds_write(to + ((i * kKeys + row + my_row8) * 128 + (lane & 7) * 16), u32x4{x[0], x[1], x[2], x[3]});
          }
      }
    };
    // K of looked-up row t, V of the one before
    auto bring_k = [&](int t, Lds* to, int row) __attribute__((always_inline)) {
      const int64_t off = place(t, a.k_page, a.k_tok);
      bring_row(kb + off, k_chunk, to, row);
      v_off = a.same ? off : place(t, a.v_page, a.v_tok);
    };
    auto bring_v = [&](Lds* to, int row) __attribute__((always_inline)) { bring_row(vb + v_off, v_chunk, to, row); };
    // a step to LDS
    auto bring = [&](Lds* ks, Lds* vs) __attribute__((always_inline)) {
#pragma unroll
      for (int t = 0; t < G::KT; t++) {
        bring_v(vs, 32 * t);
        bring_k(t, ks, 32 * t);
      }
    };

    f32x16 s;  // scores of 32 keys
    float mt;  // and their largest
    auto read_k = [&](const Lds* ks, int row, int i) __attribute__((always_inline)) -> u32x4 {
      return lds_read<u32x4>(ks + k_lane[i & 3] + (i / 4 * kKeys + row) * 128);
    };
    // 16 u + the lane's eight keys of column 32 dt + c
    auto read_v = [&](const Lds* vs, int row, int u, int dt) __attribute__((always_inline)) -> u32x4 {
      const Lds* p = vs + v_lane[dt & 1] + (dt / 2 * kKeys + row + 16 * u) * 128;
      const u32x2 x = read_transposed(p), y = read_transposed(p + 8 * 128);
      return u32x4{x[0], x[1], y[0], y[1]};
    };
    // the lane's e-th key of that column, 32-bit types
    auto read_v32 = [&](const Lds* vs, int row, int e, int dt) __attribute__((always_inline)) -> float {
      const int key = 8 * (e / 4) + 4 * g + e % 4;
      return lds_read<float>(vs + ((dt * kKeys + row + key) * 128 + ((c >> 2) ^ swizzle_v(e)) * 16 + (c & 3) * 4));
    };
    auto products = [&](const Lds* ks, int row) __attribute__((always_inline)) -> f32x16 {
      f32x16 r;
#pragma unroll
      for (int e = 0; e < 16; e++) r[e] = 0.f;
      if constexpr (G::F32) {
        u32x4 kf = read_k(ks, row, 0);
#pragma unroll
        for (int i = 0; i < G::C / 2; i++) {
          const u32x4 next = read_k(ks, row, min(i + 1, G::C / 2 - 1));
#pragma unroll
          for (int e = 0; e < 4; e++)
            r = __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(kf[e]), __uint_as_float(qf[i][e]), r, 0, 0, 0);
          kf = next;
          // One read ahead: all of them would take the registers of Q (300 tokens of 14636, 32 heads
          // of 192: 995 us instead of 984; of 64 and 128 within 1%; of 256 1391 instead of 1410).
          __builtin_amdgcn_sched_barrier(0);
        }
      } else {
#pragma unroll
        for (int i = 0; i < G::C / 2; i++) r = mfma32<XT>(read_k(ks, row, i), qf[i], r);
      }
      return r;
    };
    auto largest = [&]() __attribute__((always_inline)) {
      mt = s[0];
#pragma unroll
      for (int e = 1; e < 16; e++) mt = fmaxf(mt, s[e]);
      mt = fmaxf(mt, lane_xor<32>(mt, lane)) * scale;
    };
    // soft cap and mask of the scores of the keys from k on
    auto special = [&](int k) __attribute__((always_inline)) {
      const bool hidden = k + 32 > first_hi || k < last_lo;  // some key from some row of this wave
      if (a.softcap > 0.f) {
        // tanh x = 1 - 2 / (e^2x + 1), where that is off by 7 roundings of the result at most, infinite x included; below
        // 1/2, where it would be off by as many of 1, x + x^3 P(x^2) with P fitted over that range (off by 2^-26 of the
        // result).  t is 2 x log2 e.
        float edge = kLog2e, lead = 0.01724145f;
        asm volatile("" : "+s"(edge), "+s"(lead));  // or they would be in registers all through the steps
#pragma unroll
        for (int e = 0; e < 16; e++) {
          const float t = s[e] * cap_in, x = t * 0.346573590f, y = x * x;
          const float p = fmaf(fmaf(fmaf(lead, y, -0.05304547f), y, 0.13325879f), y, -0.33333144f);
          const float far = 1.f - 2.f * __builtin_amdgcn_rcpf(__builtin_amdgcn_exp2f(t) + 1.f);
          s[e] = fabsf(t) < edge ? fmaf(x * y, p, x) : far;
        }
      }
      if (hidden) {
        const int from = see0 - k - 4 * g, to = see1 - k - 4 * g;
#pragma unroll
        for (int e = 0; e < 16; e++) {
          const int key = 8 * (e / 4) + e % 4;  // after k + 4 g
          s[e] = key >= from && key < to ? s[e] : -INFINITY;
        }
      }
      if (a.softcap > 0.f || hidden) largest();
    };
    auto seen = [&](int k) __attribute__((always_inline)) -> bool { return busy && k < k1 && k < wave_hi && k + 32 > wave_lo; };
    auto grow = [&]() __attribute__((always_inline)) {  // the running maximum
      if (__any(mt > m)) {
        const float to = fmaxf(mt, m), f = exp2_diff(m, to);
        m = to;
        off = kLift<XT> - (m == -INFINITY ? 0.f : m);
        l *= f;
#pragma unroll
        for (int i = 0; i < G::DT; i++)
#pragma unroll
          for (int e = 0; e < 16; e++) o[i][e] *= f;
      }
    };
    // probabilities in place of the scores
    auto exponentials = [&]() __attribute__((always_inline)) {
      float sum = 0.f;
#pragma unroll
      for (int e = 0; e < 16; e++) {
        s[e] = __builtin_amdgcn_exp2f(fmaf(s[e], scale, off));
        sum += s[e];
      }
      l += sum;
    };
    // The same with the product of large scores rounded as the maximum was: the largest exponent is kLift itself.
    // exponentials() takes the product as it is, and the exponents of a row are off by half a step of its maximum
    // (2^22: 1/4), all by the same.
    auto exponentials_safe = [&]() __attribute__((always_inline)) {
      const float from = m == -INFINITY ? 0.f : m;
      float sum = 0.f;
#pragma unroll
      for (int e = 0; e < 16; e++) {
        float x = s[e] * scale;
        asm volatile("" : "+v"(x));  // or the product and the difference are one operation again
        s[e] = __builtin_amdgcn_exp2f(fabsf(from) < 4194304.f ? fmaf(s[e], scale, off) : (x - from) + kLift<XT>);
        sum += s[e];
      }
      l += sum;
    };
    auto values = [&](const Lds* vs, int row) __attribute__((always_inline)) {
      if constexpr (G::F32) {
        auto read = [&](int e, int dt) __attribute__((always_inline)) -> float { return read_v32(vs, row, e, dt); };
        float v[G::DT], next[G::DT];
#pragma unroll
        for (int dt = 0; dt < G::DT; dt++) v[dt] = read(0, dt);
#pragma unroll
        for (int e = 0; e < 16; e++) {
#pragma unroll
          for (int dt = 0; dt < G::DT; dt++) next[dt] = read(min(e + 1, 15), dt);
#pragma unroll
          for (int dt = 0; dt < G::DT; dt++) {
            o[dt] = __builtin_amdgcn_mfma_f32_32x32x2f32(v[dt], s[e], o[dt], 0, 0, 0);
            v[dt] = next[dt];
          }
          __builtin_amdgcn_sched_barrier(0);
        }
      } else {
#pragma unroll
        for (int u = 0; u < 2; u++) {
          u32x4 p0, p1;  // 16 keys: P as the sum of two numbers
#pragma unroll
          for (int e = 0; e < 4; e++) {
            const float x = s[8 * u + 2 * e], y = s[8 * u + 2 * e + 1];
            p0[e] = pack<XT>(x, y);
            if constexpr (XT == GEN_F16) asm volatile("" : "+v"(p0[e]));  // or it is converted again
            p1[e] = pack<XT>(less<XT, 0>(x, p0[e], minus_lo), less<XT, 1>(y, p0[e], minus_hi));
          }
          u32x4 vf[G::DT];
#pragma unroll
          for (int dt = 0; dt < G::DT; dt++) vf[dt] = read_v(vs, row, u, dt);
#pragma unroll
          for (int dt = 0; dt < G::DT; dt++) o[dt] = mfma32<XT>(vf[dt], p0, o[dt]);
#pragma unroll
          for (int dt = 0; dt < G::DT; dt++) o[dt] = mfma32<XT>(vf[dt], p1, o[dt]);
        }
      }
    };
    // The same where values that are not finite must count only for the rows that see their key (bit e of `see`:
    // the lane's e-th key): one key at a time, and 32 columns after the other (registers would be taken from the steps).
    auto values_safe = [&](const Lds* vs, int g, uint32_t see) __attribute__((always_inline)) {
      const uint32_t see_other = lane_xor<32>(see, lane);
#pragma unroll
      for (int dt = 0; dt < G::DT; dt++) {
        f32x16 ps = s;
#pragma unroll 1
        for (int i = 0; i < 16; i++) {
          const float other = lane_xor<32>(ps[0], lane);
#pragma unroll 1
          for (int gg = 0; gg < 2; gg++) {
            const int key = 8 * (i / 4) + 4 * gg + i % 4;
            const float p = gg == g ? ps[0] : other;
            const bool sees = (gg == g ? see : see_other) >> i & 1u;
            int at = (key * 128 + g * 4 * G::ES) ^ (swizzle_v(key) * 16);
            asm volatile("" : "+v"(at));
#pragma unroll
            for (int q = 0; q < 4; q++) {  // columns 32 dt + 8 q + 4 g and the three after it
              const int ch = (32 * dt + 8 * q) / G::CE;
              const Lds* vp = vs + ((at ^ (ch & 7) * 16) + (32 * dt + 8 * q) / (8 * G::CE) * kKeys * 128);
              float v[4];
              if constexpr (G::F32) {
                const f32x4 w = lds_read<f32x4>(vp);
#pragma unroll
                for (int e = 0; e < 4; e++) v[e] = w[e];
              } else {
                const u32x2 w = lds_read<u32x2>(vp);
#pragma unroll
                for (int e = 0; e < 4; e++) v[e] = half<XT>(w[e / 2], e % 2);
              }
#pragma unroll
              for (int e = 0; e < 4; e++) o[dt][4 * q + e] = sees ? fmaf(p, v[e], o[dt][4 * q + e]) : o[dt][4 * q + e];
            }
          }
#pragma unroll
          for (int e = 0; e < 15; e++) ps[e] = ps[e + 1];
        }
      }
    };
    // Whether some of the 32 V rows' values is not finite, each looked at by the lane that multiplies it.
    auto wild = [&](const Lds* vs, int c) __attribute__((always_inline)) -> bool {
      uint32_t kExp = G::F32 ? 0x7F800000u : XT == GEN_BF16 ? 0x7F80u : 0x7C00u;
      int head = a.D - c;
      asm volatile("" : "+s"(kExp), "+v"(head));  // or they would be in registers all through the steps
      bool found = false;
#pragma unroll
      for (int dt = 0; dt < G::DT; dt++) {
        bool here = false;
        if constexpr (G::F32) {
#pragma unroll
          for (int e = 0; e < 16; e++) here |= (__float_as_uint(read_v32(vs, 0, e, dt)) & kExp) == kExp;
        } else {
#pragma unroll
          for (int u = 0; u < 2; u++) {
            const u32x4 w = read_v(vs, 0, u, dt);
#pragma unroll
            for (int e = 0; e < 4; e++) here |= (w[e] & kExp) == kExp || (w[e] >> 16 & kExp) == kExp;
          }
        }
        found |= here && 32 * dt < head;
      }
      return __any(found);
    };
    auto reset = [&]() __attribute__((always_inline)) {
#pragma unroll
      for (int i = 0; i < G::DT; i++)
#pragma unroll
        for (int e = 0; e < 16; e++) o[i][e] = 0.f;
      m = -INFINITY, l = 0.f, off = kLift<XT>;
      look_row(k0, G::KT);
      look(k0 + 32);
      __syncthreads();  // the last tile's steps have been read
      if (tid == 0) odd = 0u;
      bring_k(G::KT, k_lds1, 0);
    };
    // The values of 32 keys and the scores of the 32 after them, for 16-bit types in an order
    // that gives each matrix instruction vector operations to run beside: the score products
    // take the exponentials and the split of the first 16 keys, their values the split of the
    // others, theirs the next maximum.  extra(i), i < 3 N: what else there is to do behind
    // the i-th of them.
    auto overlapped = [&](const Lds* ks, const Lds* vs, int row, auto&& extra) __attribute__((always_inline)) {
      constexpr int N = G::DT * 2, AHEAD = 4;  // K reads on their way
      grow();
      u32x4 kf[N], vf[2][G::DT], pt[2][2];
      auto split = [&](int u, int e) __attribute__((always_inline)) {
        const float x = s[8 * u + 2 * e], y = s[8 * u + 2 * e + 1];
        pt[u][0][e] = pack<XT>(x, y);
        if constexpr (XT == GEN_F16) asm volatile("" : "+v"(pt[u][0][e]));  // or it is converted again
        pt[u][1][e] = pack<XT>(less<XT, 0>(x, pt[u][0][e], minus_lo), less<XT, 1>(y, pt[u][0][e], minus_hi));
        asm volatile("" : "+v"(pt[u][0][e]), "+v"(pt[u][1][e]));  // here, not where it is used
      };
#pragma unroll
      for (int i = 0; i < AHEAD; i++) kf[i] = read_k(ks, row, i);
      f32x16 next;
#pragma unroll
      for (int e = 0; e < 16; e++) next[e] = 0.f;
      float sum = 0.f;
      auto exponential = [&](int e) __attribute__((always_inline)) {
        s[e] = __builtin_amdgcn_exp2f(fmaf(s[e], scale, off));
        sum += s[e];
      };
      // some before the first product, whose operand is on its way
#pragma unroll
      for (int e = 0; e < 4; e++) exponential(e);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int i = 0; i < N; i++) {
        next = mfma32<XT>(kf[i], qf[i], next);
        if (i + AHEAD < N) kf[i + AHEAD] = read_k(ks, row, i + AHEAD);
#pragma unroll
        for (int dt = 0; dt < G::DT; dt++)
          if (i == N / 2 + dt % (N / 2)) vf[0][dt] = read_v(vs, row, 0, dt);
#pragma unroll
        for (int e = 4 + 12 * i / N; e < 4 + 12 * (i + 1) / N; e++) exponential(e);
        if (i >= N / 2) {
#pragma unroll
          for (int e = 4 * (i - N / 2) / (N - N / 2); e < 4 * (i + 1 - N / 2) / (N - N / 2); e++) split(0, e);
        }
        extra(i);
        __builtin_amdgcn_sched_barrier(0);
      }
      l += sum;
      mt = next[0];
#pragma unroll
      for (int u = 0; u < 2; u++)
#pragma unroll
        for (int i = 0; i < N; i++) {
          o[i % G::DT] = mfma32<XT>(vf[u][i % G::DT], pt[u][i / G::DT], o[i % G::DT]);
          if (u == 0) {
#pragma unroll
            for (int dt = 0; dt < G::DT; dt++)
              if (i == dt) vf[1][dt] = read_v(vs, row, 1, dt);
#pragma unroll
            for (int e = 4 * i / N; e < 4 * (i + 1) / N; e++) split(1, e);
          } else {
#pragma unroll
            for (int e = 16 * i / N; e < 16 * (i + 1) / N; e++) mt = fmaxf(mt, next[e]);
          }
          extra((u + 1) * N + i);
          __builtin_amdgcn_sched_barrier(0);
        }
      mt = fmaxf(mt, lane_xor<32>(mt, lane)) * scale;
      s = next;
    };
    // 32 keys from k on: their values, and the scores of the 32 after them (K and V rows of one step)
    auto half_step = [&](const Lds* ks, const Lds* vs, int row, int k) __attribute__((always_inline)) {
      if (seen(k)) {
        if constexpr (G::F32) {
          grow();
          const f32x16 next = products(ks, row);
          exponentials();
          values(vs, row);
          s = next;
          largest();
        } else {
          overlapped(ks, vs, row, [](int) {});
        }
      } else if (seen(k + 32)) {
        s = products(ks, row);
        largest();
      }
      if (seen(k + 32)) special(k + 32);
    };
    auto step = [&](const Lds* ks, const Lds* vs, int k) __attribute__((always_inline)) {
#pragma unroll
      for (int t = 0; t < G::KT; t++) half_step(ks, vs, 32 * t, k + 32 * t);
    };
    reset();
    load_q();
    bring(k_lds0, v_lds0);
    look(k0 + 32 + kKeys);
    step_barrier();
    finish_q();
    if (seen(k0)) {
      s = products(k_lds1, 0);
      largest();
      special(k0);
    }
    step_barrier();
    // Steps whose keys, and the 32 after them, are all seen by every row of the tile, with others
    // behind them: no masks, nothing to decide.
    const int all_hi = min(k1, sq.p0 + tok0 + 1), all_lo = a.window > 0 ? max(0, hi - a.window) : 0;
    const bool easy = !G::F32 && a.direct && a.same && (kLook || a.D == DP) && a.softcap == 0.f;
    auto easy_step = [&](const Lds* ks, const Lds* vs, Lds* k_next, Lds* v_next, int k) __attribute__((always_inline)) {
      if constexpr (!G::F32) {
        int64_t k_off = 0;
        auto rest = [&](int i) __attribute__((always_inline)) {  // brings the next step, a piece at a time
#pragma unroll
          for (int t = 0; t < G::KT; t++) {
            if (i == 3 * t) k_off = (int64_t)((uint64_t)(uint32_t)min(max(entry[t], 0), a.pages - 1) * (uint32_t)a.k_page +
                                              (uint64_t)(uint32_t)in_page[t] * (uint32_t)a.k_tok);
            if (i == 3 * t + 1) rows_to_lds(vb + v_off, v_chunk, v_next, 32 * t);
            if (i == 3 * t + 2) {
              rows_to_lds(kb + k_off, k_chunk, k_next, 32 * t);
              v_off = k_off;
            }
          }
          if (i == 3 * G::KT) look(k + 32 + 2 * kKeys);
        };
        if (busy) {
          overlapped(ks, vs, 0, rest);
          if constexpr (G::KT > 1) overlapped(ks, vs, 32, [](int) {});
        } else {
#pragma unroll
          for (int i = 0; i <= 3 * G::KT; i++) rest(i);
        }
        step_barrier();
      }
    };
    // while a step is worked on the next is brought, and the one after it looked up
    for (int k = k0; k < k1; k += 2 * kKeys) {
      if (easy && k + 32 >= all_lo && k + 3 * kKeys + 32 <= all_hi) {
        do {
          if (G::WGS == 2 && later) __builtin_amdgcn_s_setprio(1);
          easy_step(k_lds0, v_lds0, k_lds1, v_lds1, k);
          if (G::WGS == 2 && later) __builtin_amdgcn_s_setprio(0);
          easy_step(k_lds1, v_lds1, k_lds0, v_lds0, k + kKeys);
          k += 2 * kKeys;
        } while (k + 3 * kKeys + 32 <= all_hi);
      }
      if (k + kKeys < k1) {
        bring(k_lds1, v_lds1);
        look(k + 32 + 2 * kKeys);
      }
      step(k_lds0, v_lds0, k);
      step_barrier();
      if (k + kKeys >= k1) break;
      if (k + 2 * kKeys < k1) {
        bring(k_lds0, v_lds0);
        look(k + 32 + 3 * kKeys);
      }
      step(k_lds1, v_lds1, k + kKeys);
      step_barrier();
    }
    l += lane_xor<32>(l, lane);
    float x = l;  // not finite where some value is not
#pragma unroll
    for (int i = 0; i < G::DT; i++)
#pragma unroll
      for (int e = 0; e < 16; e++) x = fmaf(o[i][e], 0.f, x);
    // A row's largest probability is 2^kLift, more or less by a factor of 2 while scores are below 2^25 (in
    // base 2).  Of larger ones it may have left the type: upwards it is found in x, downwards here.
    const float least = kLift<XT> == 0.f ? 0.25f : 4096.f;
    if (r0 + c < rows && (!isfinite(x) || (l < least && m != -INFINITY))) odd = 1u;
    __syncthreads();
    if (__builtin_expect(__builtin_amdgcn_readfirstlane(odd), 0)) {
      // again, 32 keys at a time
      reset();
      int g_safe = g, c_safe = c;
      asm volatile("" : "+v"(g_safe), "+v"(c_safe));
      for (int k = k0; k < k1; k += 32) {
        if (k > k0) {
          bring_k(0, k_lds1, 0);
          look(k + 32);
        }
        bring_v(v_lds1, 0);
        step_barrier();
        if (seen(k)) {
          s = products(k_lds1, 0);
          largest();
          special(k);
          grow();
          uint32_t see = 0u;  // a score of -inf is a key that is not seen, or one that has no part
#pragma unroll
          for (int e = 15; e >= 0; e--) see = 2 * see + (s[e] != -INFINITY ? 1u : 0u);
          exponentials_safe();
          if (wild(v_lds1, c_safe)) values_safe(v_lds1, g_safe, see);
          else values(v_lds1, 0);
        }
        step_barrier();
      }
      l += lane_xor<32>(l, lane);
    }

    // From here on by another copy of the lane's number: addresses worked out from the first
    // would be kept in registers all through the steps, which do not have them.
    int lane2 = lane;
    asm volatile("" : "+v"(lane2));
    const int c2 = lane2 & 31, g2 = lane2 >> 5;
    // A row's result is its sum times finish(row, M, L); where it lies.
    auto finish = [&](int r, float M, float L) __attribute__((always_inline)) -> float {
      float f = 1.f;
      if (a.sinks) {
        const float x = a.sinks[head0 + r - token_of(r) * heads];
        // the largest finite sinks stay finite in the other base
        const float sink = isinf(x) ? x : fminf(fmaxf(x * kLog2e, -FLT_MAX), FLT_MAX), M2 = fmaxf(M, sink);
        f = exp2_diff(M, M2);
        L = L * f + exp2_diff(sink, M2);
      }
      return f / L;
    };
    auto out_at = [&](int r) __attribute__((always_inline)) -> int64_t {
      const int tok = token_of(r);
      return ((int64_t)(sq.first + tok0 + tok) * a.Hq + head0 + r - tok * heads) * a.D;
    };
    if (w0 == w1) {
      if (busy) {
        const int row2 = min(r0 + c2, rows - 1);
        const float f = finish(row2, m - kLift<XT>, l);
        if constexpr (G::F32) {
          const int64_t to = out_at(row2);
          if (r0 + c2 < rows) {
#pragma unroll
            for (int dt = 0; dt < G::DT; dt++)
#pragma unroll
              for (int e = 0; e < 16; e += 4) {
                const int d = 32 * dt + 2 * e + 4 * g2;
                if (d < a.D) store4<XT>(a.out, to + d, f32x4{o[dt][e], o[dt][e + 1], o[dt][e + 2], o[dt][e + 3]} * f);
              }
          }
        } else {
          // through LDS, so that whole rows are written: chunk i of row r at place i ^ swizzle(r); the step's rows have
          // been read.  In blocks that the head fills: what lies past it stays.
          constexpr int LOW = (G::C & -G::C) < 8 ? (G::C & -G::C) : 8;
          static_assert(DP == 64 || 32 * G::C * 16 <= (G::NC - 1) * kKeys * 128, "");
          Lds* mine = DP == 64 ? (wave < 2 ? v_lds0 : v_lds1) + (wave & 1) * (32 * G::C * 16)
                               : wave < 2 ? (wave == 0 ? v_lds0 : v_lds1) : (wave == 2 ? k_lds0 : k_lds1);
#pragma unroll
          for (int dt = 0; dt < G::DT; dt++)
#pragma unroll
            for (int q = 0; q < 4; q++)
              lds_write(mine + ((c2 * G::C + ((4 * dt + q) ^ (c2 & (LOW - 1)))) * 16 + g2 * 8),
                        u32x2{pack_out<XT>(o[dt][4 * q] * f, o[dt][4 * q + 1] * f), pack_out<XT>(o[dt][4 * q + 2] * f, o[dt][4 * q + 3] * f)});
          const int live = min(32, rows - r0);
#pragma unroll
          for (int i = 0; i < G::C / 2; i++) {
            const int at16 = i * 64 + lane2, r = at16 / G::C, ch = at16 - r * G::C;
            const u32x4 v = lds_read<u32x4>(mine + (r * G::C + (ch ^ (r & (LOW - 1)))) * 16);
            if (r < live && ch < chunks)
              *reinterpret_cast<u32x4_e*>(static_cast<uint16_t*>(a.out) + out_at(r0 + r) + ch * 8) = u32x4_e{v[0], v[1], v[2], v[3]};
          }
        }
      }
    } else {
      // bytes of a workgroup's partial result: of its last tile (slot 1), or of one that began before it (slot 0)
      auto part_at = [&](int v) __attribute__((always_inline)) -> uint32_t { return (uint32_t)((2 * v + (v == w0)) * a.slot_words) * 4u; };
      // and of the neighbours that it leads, in a place of its own: others of the joining threads may still read the first
      const uint32_t joined = (uint32_t)(2 * a.wgs * a.slot_words) * 4u;
      const int waves = (rows + 31) >> 5;
      // of wave v: 16 bytes of each lane, i-th of 4 DT; its rows' maxima and sums
      auto sum_at = [&](int v, int i) __attribute__((always_inline)) -> uint32_t { return (uint32_t)((v * 4 * G::DT + i) * 64 + lane2) * 16u; };
      auto ml_at = [&](int v) __attribute__((always_inline)) -> uint32_t { return (uint32_t)(waves * 32 * DP + (v * 32 + c2) * 2) * 4u; };
      auto put = [&](uint32_t p, int v, int i, f32x4 acc) __attribute__((always_inline)) {
        __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, acc), parts, p + sum_at(v, i), 0, kAgentScope);
      };
      auto put_ml = [&](uint32_t p, int v, float M, float L) __attribute__((always_inline)) {
        if (g2 == 0)
          __builtin_amdgcn_raw_buffer_store_b64(u32x2{__float_as_uint(M), __float_as_uint(L)}, parts, p + ml_at(v), 0, kAgentScope);
      };
      if (busy) {
#pragma unroll
        for (int dt = 0; dt < G::DT; dt++)
#pragma unroll
          for (int q = 0; q < 4; q++)
            put(part_at(w), wave, 4 * dt + q, f32x4{o[dt][4 * q], o[dt][4 * q + 1], o[dt][4 * q + 2], o[dt][4 * q + 3]});
        put_ml(part_at(w), wave, m - kLift<XT>, l);
      }
      // The last of up to kFlight neighbours to arrive joins them; more are joined in two steps, the
      // root of their number at a time (16 sequences of 5 tokens over 43000 keys in all: 42.1 us, with
      // up to 16 in the first step 46.8).
      auto last_of = [&](uint32_t* cnt, int of) __attribute__((always_inline)) -> bool {
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
      // Sums the results, from byte `from` on, of workgroups v, v + by, .. (of them), in the
      // order of the keys: a wave takes kUnits times 16 bytes of each lane at a time.
      auto join = [&](uint32_t from, int v, int by, int of, bool last) __attribute__((always_inline)) {
#pragma unroll 1
        for (int u0 = wave * kUnits; u0 < waves * 4 * G::DT; u0 += kWaves * kUnits) {
          const int bw = u0 / (4 * G::DT), i = u0 - bw * (4 * G::DT);
          float M = -INFINITY, L = 0.f;
          f32x4 acc[kUnits];
#pragma unroll
          for (int q = 0; q < kUnits; q++) acc[q] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll 1
          for (int i0 = 0; i0 < of; i0 += kFlight) {
            u32x4 ow[kFlight][kUnits];
            u32x2 mw[kFlight];
#pragma unroll
            for (int k = 0; k < kFlight; k++) {
              const uint32_t p = from + part_at(v + by * min(i0 + k, of - 1));
              mw[k] = __builtin_bit_cast(u32x2, __builtin_amdgcn_raw_buffer_load_b64(parts, p + ml_at(bw), 0, kAgentScope));
#pragma unroll
              for (int q = 0; q < kUnits; q++)
                ow[k][q] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(parts, p + sum_at(bw, i + q), 0, kAgentScope));
            }
#pragma unroll
            for (int k = 0; k < kFlight; k++) {
              if (i0 + k >= of) break;
              const float mi = __uint_as_float(mw[k][0]), M2 = fmaxf(M, mi);
              const float f = exp2_diff(M, M2), fi = exp2_diff(mi, M2);
              M = M2;
              L = L * f + __uint_as_float(mw[k][1]) * fi;
#pragma unroll
              for (int q = 0; q < kUnits; q++) acc[q] = acc[q] * f + __builtin_bit_cast(f32x4, ow[k][q]) * fi;
            }
          }
          if (last) {
            const int r = 32 * bw + c2;
            const float by_row = finish(min(r, rows - 1), M, L);
            const int64_t to = out_at(min(r, rows - 1));
#pragma unroll
            for (int q = 0; q < kUnits; q++) {
              const int d = 8 * (i + q) + 4 * g2;  // 32 (i / 4) + 8 (i % 4)
              if (r < rows && d < a.D) store4<XT>(a.out, to + d, acc[q] * by_row);
            }
          } else {
#pragma unroll
            for (int q = 0; q < kUnits; q++) put(joined + part_at(v), bw, i + q, acc[q]);
            if (i == 0) put_ml(joined + part_at(v), bw, M, L);
          }
        }
      };
      const int of = w1 - w0 + 1, by = of <= kFlight ? of : (int)ceilf(__builtin_amdgcn_sqrtf((float)of));
      const int lead = (w - w0) / by * by, near = min(by, of - lead);
      // a workgroup may lead neighbours of a tile that began before it and of its last one
      if (last_of(a.cnt + 2 * (w0 + lead) + (lead == 0), near)) {
        join(0, w0 + lead, 1, near, of <= by);
        if (of > by) {
          const int groups = (of + by - 1) / by;
          if (last_of(a.cnt + 2 * a.wgs + w0, groups)) join(joined, w0, by, groups, true);
        }
      }
    }
    at.nth++;
    at.key = 0;
  }
}

// f(type, width of the kernel)
template <typename F>
auto with_kernel(const ChunkAttnArgs& a, F&& f) {
  auto width = [&](auto xt) {
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

bool chunk_attention_plan(ChunkAttnArgs& a, int cus, int64_t* part_bytes) {
  a.page_shift = 30;
  while (((int64_t)1 << (a.page_shift - 30)) < a.page) a.page_shift++;
  // exact for keys below 2^30: the error of page_mul, below page <= 2^(shift - 30), times the key stays below 2^shift
  a.page_mul = (uint32_t)((((uint64_t)1 << a.page_shift) + a.page - 1) / a.page);
  const int esz = a.type == GEN_F32 ? 4 : 2;
  uint64_t bits = reinterpret_cast<uintptr_t>(a.k) | reinterpret_cast<uintptr_t>(a.v);
  a.direct = 1;
  for (int64_t* st : {&a.k_page, &a.k_head, &a.k_tok, &a.v_page, &a.v_head, &a.v_tok}) {
    *st *= esz;
    bits |= (uint64_t)*st;
    if (*st < 0 || *st > 0xFFFFFFFFll) a.direct = 0;
  }
  if (bits & 15) a.direct = 0;
  a.same = a.k_page == a.v_page && a.k_tok == a.v_tok;
  const int per = a.Hq / a.Hkv;
  a.tile_heads = std::min(per, kRows);
  a.tile_tokens = kRows / a.tile_heads;
  a.inv_tile_heads = (65536 + a.tile_heads - 1) / a.tile_heads;
  a.inv_tile_tokens = 1.0 / a.tile_tokens;
  const int64_t cap = (int64_t)a.width * a.page;
  const int64_t keys = a.window > 0 ? std::min<int64_t>(cap, (int64_t)a.window + a.tile_tokens) : cap;
  const int64_t heads = (int64_t)a.Hkv * ((per + a.tile_heads - 1) / a.tile_heads);
  const int64_t tiles = heads * (((int64_t)a.T + a.tile_tokens - 1) / a.tile_tokens + std::min(a.B, a.T));
  const int resident = with_kernel(a, [](auto xt, auto dp) { return Geo<decltype(xt)::value, decltype(dp)::value>::WGS; });
  // tiles of a sequence are counted in 32 bits, keys of all of them, without a window, below 2^52
  if (tiles > (1 << 30) || tiles * (double)(cap + kAround) > 4e15) return false;
  a.wgs = (int)std::max<int64_t>(1, std::min<int64_t>((tiles * (keys + kAround) + kLeast - 1) / kLeast, (int64_t)cus * resident));
  a.inv_wgs = 1.0 / a.wgs;
  const int waves = (int)((std::min<int64_t>(kRows, (int64_t)a.T * a.tile_heads) + 31) / 32);
  a.slot_words = with_kernel(a, [&](auto, auto dp) { return part_words(waves, decltype(dp)::value); });
  *part_bytes = (int64_t)4 * a.wgs * a.slot_words * 4;
  return *part_bytes < ((int64_t)1 << 32);
}

hipError_t launch_chunk_attention(const ChunkAttnArgs& a, hipStream_t stream) {
  if (a.T == 0 || a.B == 0) return hipSuccess;
  if (a.D < 8 || a.D > 256 || a.D % 8 || a.pages < 1 || a.page < 1 || a.wgs < 1 || 3 * a.wgs > kSplitCounters)
    return hipErrorInvalidValue;
  return with_kernel(a, [&](auto xt, auto dp) {
    constexpr int XT = decltype(xt)::value, DP = decltype(dp)::value;
    hipLaunchKernelGGL((chunk_attention_kernel<XT, DP>), dim3((unsigned)a.wgs), dim3(256), 0, stream, a);
    return hipGetLastError();
  });
}

}  // namespace mlxq
