// adjust.hip — penalties for the tokens of a history, biases of single tokens
// and a grammar's mask on logits, on gfx950.
//
//   x' = x / r where x > 0, else x r             for tokens in the history
//   x' -= presence + frequency * times           for those in it `times` > 0 times after the prompt
//   x' += bias                                   for tokens with one
//   x' = -inf                                    for tokens whose bit of the mask is 0
//
// A logit is read and written once, which is the floor; beyond that it takes
// looking through the history.  A workgroup takes 16 bytes of one
// row a thread and counts the history's tokens that fall into them in LDS, a word a
// token: whole numbers, so the order of the atomic operations does not matter.  Of
// several biases of one token the last in the list counts: LDS keeps the largest
// place.  Whoever finds a token first puts it on a list; a thread for each of the list
// works out its logit and leaves it in the word.
#include <hip/hip_runtime.h>

#include <type_traits>

#include "common.hpp"
#include "kernels.hpp"

namespace mlxq {

namespace {

constexpr uint32_t kSeen = 0x80000000u;  // in the prompt; the bits below count the places after it

typedef uint32_t u32x4_e __attribute__((ext_vector_type(4), aligned(2)));
typedef int32_t i32x4_e __attribute__((ext_vector_type(4), aligned(4)));

// Biases that a thread asks for before anything else, beside four tokens of the history.
constexpr int kAhead = 2;

constexpr int kThreads = 256;

template <int XT>
constexpr int kChunk = kThreads * (XT == GEN_F32 ? 4 : 8);

// One workgroup: logits [first, first + CHUNK) of row t, 16 bytes a thread.  All that does not
// depend on something else is asked for first: the logits, the mask, the beginning of the
// history and of the biases, the row's numbers.  128 rows of 151936 in bfloat16 with 4000 tokens
// of history, 300 biases and a mask: 27 us a launch among others (81 MB; 27.6 traced), of which 11
// are the history past its first 1024 tokens, a dozen vector operations and a wait for LDS each
// in every workgroup of a row.  Others, where this took 28.3: every thread working out its own
// logits instead of a list, in which most lanes wait for the few that have one, 35; the list made
// from the words afterwards 29.8; the whole history asked for ahead 28.5, but a mask alone then
// takes 5.3 instead of 4.7; workgroups of 512 (1024) threads, half (a quarter) of the looking
// through the history, 30.3 (39.7); two (four) times 16 bytes a thread 40 (67), the tables leave
// too few waves.
template <int XT>
__global__ __launch_bounds__(kThreads) void adjust_logits_kernel(const AdjustArgs a) {
  constexpr int ES = XT == GEN_F32 ? 4 : 2, W = 16 / ES, CHUNK = kChunk<XT>;
  extern __shared__ __align__(16) uint32_t lds[];
  const int tid = threadIdx.x, chunks = (a.V + CHUNK - 1) / CHUNK, t = blockIdx.x / chunks;
  const int first = (blockIdx.x - t * chunks) * CHUNK;
  const char* src = static_cast<const char*>(a.x) + (t * a.x_row + first) * ES;
  char* dst = static_cast<char*>(a.out) + (t * a.out_row + first) * ES;
  const bool edits = a.n > 0 || a.m > 0;
  const int32_t *h = a.history + t * a.history_row, *ids = a.bias_ids + t * a.bias_ids_row;
  const float* values = a.bias + t * a.bias_row;
  // entries 4 i .. 4 i + 3 of the history, -1 past its end
  auto four = [&](int i) -> i32x4_e {
    i32x4_e r = {-1, -1, -1, -1};
    if (4 * i + 3 < a.n) {
      r = *reinterpret_cast<const i32x4_e*>(h + 4 * i);
    } else {
#pragma unroll
      for (int q = 0; q < 3; q++)
        if (4 * i + q < a.n) r[q] = h[4 * i + q];
    }
    return r;
  };
  i32x4_e early = four(tid);
  int32_t early_id[kAhead];
#pragma unroll
  for (int k = 0; k < kAhead; k++) early_id[k] = k * kThreads + tid < a.m ? ids[k * kThreads + tid] : -1;
  int n = a.n, prompt = 0;
  float rep = 1.f, pres = 0.f, freq = 0.f;
  if (a.n > 0) {
    if (a.history_lengths) n = min(max(a.history_lengths[t], 0), a.n);
    if (a.prompts) prompt = a.prompts[t];
    if (a.repetition) rep = a.repetition[t];
    if (a.presence) pres = a.presence[t];
    if (a.frequency) freq = a.frequency[t];
  }
  const int e = tid * W;
  u32x4 v = {0u, 0u, 0u, 0u};
  const bool whole = first + e + W <= a.V;
  const uint32_t bits = a.mask && first + e < a.V ? a.mask[t * a.mask_row + (first + e) / 32] >> ((first + e) & 31) : 0u;
  if (whole) {
    const u32x4_e w = *reinterpret_cast<const u32x4_e*>(src + e * ES);
    v = u32x4{w[0], w[1], w[2], w[3]};
  } else {
#pragma unroll
    for (int i = 0; i < W; i++)
      if (first + e + i < a.V) {
        if constexpr (ES == 4) v[i] = reinterpret_cast<const uint32_t*>(src)[e + i];
        else v[i / 2] |= (uint32_t)reinterpret_cast<const uint16_t*>(src)[e + i] << (16 * (i & 1));
      }
  }
  if (edits) {
    // A word a token: how often the history has it, then the bits of its new logit, made other than 0; its last
    // place among the biases (-1: none).  The history's tokens, each once.
    uint32_t* times = lds;
    int* place = reinterpret_cast<int*>(lds + CHUNK);
    uint16_t* list = reinterpret_cast<uint16_t*>(lds + (a.m > 0 ? 2 : 1) * CHUNK);
    __shared__ uint32_t listed;
    const uint32_t here = (uint32_t)min(CHUNK, a.V - first);  // tokens past the row's end count for nothing
    if (tid == 0) listed = 0u;
#pragma unroll
    for (int i = 0; i < CHUNK / (4 * kThreads); i++) reinterpret_cast<u32x4*>(times)[i * kThreads + tid] = u32x4{0u, 0u, 0u, 0u};
    if (a.m > 0) {
#pragma unroll
      for (int i = 0; i < CHUNK / (4 * kThreads); i++) reinterpret_cast<u32x4*>(place)[i * kThreads + tid] = u32x4{~0u, ~0u, ~0u, ~0u};
    }
    __syncthreads();
    auto count = [&](int i, int32_t token) {
      const uint32_t at = (uint32_t)token - (uint32_t)first;
      if (i < n && at < here) {
        const uint32_t had = i < prompt ? atomicOr(times + at, kSeen) : atomicAdd(times + at, 1u);
        if (had == 0u) list[atomicAdd(&listed, 1u)] = (uint16_t)at;
      }
    };
    auto mark = [&](int i, int32_t token) {
      const uint32_t at = (uint32_t)token - (uint32_t)first;
      if (i < a.m && at < here) atomicMax(place + at, i);
    };
    for (int i = tid; 4 * (i - tid) < n; i += kThreads) {
      if (i != tid) early = four(i);
#pragma unroll
      for (int q = 0; q < 4; q++) count(4 * i + q, early[q]);
    }
    if (a.m > 0) {
#pragma unroll
      for (int k = 0; k < kAhead; k++) mark(k * kThreads + tid, early_id[k]);
      for (int i = kAhead * kThreads + tid; i < a.m; i += kThreads) mark(i, ids[i]);
    }
    __syncthreads();
    auto logit = [&](uint32_t at) -> float {
      if constexpr (ES == 4) return reinterpret_cast<const float*>(src)[at];
      else return xt_to_f32<XT == GEN_F16 ? 1 : 0>(reinterpret_cast<const uint16_t*>(src)[at]);
    };
    auto leave = [&](uint32_t at, float x) {
      if constexpr (ES == 4) times[at] = ~(x == x ? __float_as_uint(x) : 0x7FC00000u);
      else times[at] = 0x10000u | f32_to_xt<XT == GEN_F16 ? 1 : 0>(x);
    };
    for (uint32_t i = tid; i < listed; i += kThreads) {
      const uint32_t at = list[i], c = times[at];
      const int p = a.m > 0 ? place[at] : -1;
      float x = logit(at);
      x = x > 0.f ? x / rep : x * rep;
      if (c & ~kSeen) x -= pres + freq * (float)(c & ~kSeen);
      if (p >= 0) x += values[p];
      leave(at, x);
    }
    // tokens with a bias alone
    auto alone = [&](int i, int32_t token) {
      const uint32_t at = (uint32_t)token - (uint32_t)first;
      if (i < a.m && at < here && place[at] == i && times[at] == 0u) leave(at, logit(at) + values[i]);
    };
    if (a.m > 0) {
#pragma unroll
      for (int k = 0; k < kAhead; k++) alone(k * kThreads + tid, early_id[k]);
      for (int i = kAhead * kThreads + tid; i < a.m; i += kThreads) alone(i, ids[i]);
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < W; i += 4) {
      const u32x4 r = *reinterpret_cast<const u32x4*>(times + e + i);
      if constexpr (ES == 4) {
#pragma unroll
        for (int q = 0; q < 4; q++) v[q] = r[q] ? ~r[q] : v[q];
      } else {
#pragma unroll
        for (int q = 0; q < 4; q += 2) {
          const uint32_t both = r[q] ? (v[(i + q) / 2] & 0xFFFF0000u) | (r[q] & 0xFFFFu) : v[(i + q) / 2];
          v[(i + q) / 2] = r[q + 1] ? (both & 0xFFFFu) | r[q + 1] << 16 : both;
        }
      }
    }
  }
  constexpr uint32_t kNone = XT == GEN_F32 ? 0xFF800000u : XT == GEN_F16 ? 0xFC00u : 0xFF80u;  // -inf
  if (first + e >= a.V) return;
  if (a.mask) {
#pragma unroll
    for (int i = 0; i < W; i++) {
      const bool keep = bits >> i & 1u;
      if constexpr (ES == 4) v[i] = keep ? v[i] : kNone;
      else v[i / 2] = keep ? v[i / 2] : (v[i / 2] & (i & 1 ? 0x0000FFFFu : 0xFFFF0000u)) | kNone << (16 * (i & 1));
    }
  }
  if (whole) {
    *reinterpret_cast<u32x4_e*>(dst + e * ES) = u32x4_e{v[0], v[1], v[2], v[3]};
  } else {
#pragma unroll
    for (int i = 0; i < W; i++)
      if (first + e + i < a.V) {
        if constexpr (ES == 4) reinterpret_cast<uint32_t*>(dst)[e + i] = v[i];
        else reinterpret_cast<uint16_t*>(dst)[e + i] = (uint16_t)(v[i / 2] >> (16 * (i & 1)));
      }
  }
}

// f(type)
template <typename F>
auto with_kernel(const AdjustArgs& a, F&& f) {
  if (a.type == GEN_BF16) return f(std::integral_constant<int, GEN_BF16>{});
  if (a.type == GEN_F16) return f(std::integral_constant<int, GEN_F16>{});
  return f(std::integral_constant<int, GEN_F32>{});
}

}  // namespace

int64_t adjust_logits_groups(const AdjustArgs& a) {
  const int chunk = with_kernel(a, [](auto xt) { return kChunk<decltype(xt)::value>; });
  return (int64_t)((a.V + chunk - 1) / chunk) * a.T;
}

hipError_t launch_adjust_logits(const AdjustArgs& a, hipStream_t stream) {
  if (a.T == 0 || a.V == 0) return hipSuccess;
  const int64_t groups = adjust_logits_groups(a);
  if (groups > kMaxGroups) return hipErrorInvalidValue;
  return with_kernel(a, [&](auto xt) {
    constexpr int XT = decltype(xt)::value;
    const size_t bytes = a.n > 0 || a.m > 0 ? (size_t)kChunk<XT> * (4 + (a.m > 0 ? 4 : 0) + (a.n > 0 ? 2 : 0)) : 0;
    hipLaunchKernelGGL((adjust_logits_kernel<XT>), dim3((unsigned)groups), dim3(kThreads), bytes, stream, a);
    return hipGetLastError();
  });
}

}  // namespace mlxq
