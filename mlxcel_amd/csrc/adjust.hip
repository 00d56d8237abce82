// adjust.hip — penalties for the tokens of a history, biases of single tokens
// and a grammar's mask on logits, on gfx950.
//
//   x' = x / r where x > 0, else x r             for tokens in the history
//   x' -= presence + frequency * times           for those in it `times` > 0 times after the prompt
//   x' += bias                                   for tokens with one
//   x' = -inf                                    for tokens whose bit of the mask is 0
//
// A logit is read and written once, which is the bound.  A workgroup takes 16 bytes of one
// row a thread and counts the history's tokens that fall into them in LDS, a word a
// token: whole numbers, so the order of the atomic operations does not matter.  Of
// several biases of one token the last in the list counts: LDS keeps the largest
// place, which then makes way for the value.
#include <hip/hip_runtime.h>

#include <type_traits>

#include "common.hpp"
#include "kernels.hpp"

namespace mlxq {

namespace {

constexpr uint32_t kNoBias = 0xFFFFFFFFu;  // -1 as a place, a NaN that is not written as a value
constexpr uint32_t kSeen = 0x80000000u;  // in the prompt; the bits below count the places after it

typedef uint32_t u32x4_e __attribute__((ext_vector_type(4), aligned(2)));

// Entries of the history and of the biases that a thread asks for before anything else.
constexpr int kAhead = 4;

template <int XT>
constexpr int kChunk = 256 * (XT == GEN_F32 ? 4 : 8);

// One workgroup: logits [first, first + 256 W) of row t, W in 16 bytes.  All that does not
// depend on something else is asked for first: the logits, the mask, the beginning of the
// history and of the biases, the row's numbers.  128 rows of 151936 with 2 (4) times as many
// logits a workgroup, so half as many of them: 40 (67) us instead of 33.5; one row 6.8 (12.3) instead of 5.1.
template <int XT>
__global__ __launch_bounds__(256) void adjust_logits_kernel(const AdjustArgs a) {
  constexpr int ES = XT == GEN_F32 ? 4 : 2, W = 16 / ES, CHUNK = kChunk<XT>;
  extern __shared__ __align__(16) uint32_t lds[];
  const int tid = threadIdx.x, chunks = (a.V + CHUNK - 1) / CHUNK, t = blockIdx.x / chunks;
  const int first = (blockIdx.x - t * chunks) * CHUNK;
  const char* src = static_cast<const char*>(a.x) + (t * a.x_row + first) * ES;
  char* dst = static_cast<char*>(a.out) + (t * a.out_row + first) * ES;
  const bool edits = a.n > 0 || a.m > 0;
  const int32_t *h = a.history + t * a.history_row, *ids = a.bias_ids + t * a.bias_ids_row;
  const float* values = a.bias + t * a.bias_row;
  int32_t early[kAhead], early_id[kAhead];
  float early_bias[kAhead];
#pragma unroll
  for (int k = 0; k < kAhead; k++) {
    early[k] = k * 256 + tid < a.n ? h[k * 256 + tid] : -1;
    early_id[k] = k * 256 + tid < a.m ? ids[k * 256 + tid] : -1;
    early_bias[k] = k * 256 + tid < a.m ? values[k * 256 + tid] : 0.f;
  }
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
  // a word a token: how often the history has it; its last place among the biases, then the bias (kNoBias: none)
  uint32_t *times = lds, *place = lds + (a.n > 0 ? CHUNK : 0);
  if (edits) {
    if (a.n > 0) {
#pragma unroll
      for (int i = 0; i < CHUNK / 1024; i++) reinterpret_cast<u32x4*>(times)[i * 256 + tid] = u32x4{0u, 0u, 0u, 0u};
    }
    if (a.m > 0) {
#pragma unroll
      for (int i = 0; i < CHUNK / 1024; i++)
        reinterpret_cast<u32x4*>(place)[i * 256 + tid] = u32x4{kNoBias, kNoBias, kNoBias, kNoBias};
    }
    __syncthreads();
    auto count = [&](int i, int32_t token) {
      const uint32_t at = (uint32_t)token - (uint32_t)first;
      if (i < n && at < (uint32_t)CHUNK) {  // past the row's end it counts for nothing
        if (i < prompt) atomicOr(times + at, kSeen);
        else atomicAdd(times + at, 1u);
      }
    };
    auto mark = [&](int i, int32_t token) {
      const uint32_t at = (uint32_t)token - (uint32_t)first;
      if (i < a.m && at < (uint32_t)CHUNK) atomicMax(reinterpret_cast<int*>(place) + at, i);
    };
    if (a.n > 0) {
#pragma unroll
      for (int k = 0; k < kAhead; k++) count(k * 256 + tid, early[k]);
      for (int i0 = kAhead * 256; i0 < n; i0 += kAhead * 256) {
#pragma unroll
        for (int k = 0; k < kAhead; k++) early[k] = i0 + k * 256 + tid < n ? h[i0 + k * 256 + tid] : -1;
#pragma unroll
        for (int k = 0; k < kAhead; k++) count(i0 + k * 256 + tid, early[k]);
      }
    }
    if (a.m > 0) {
#pragma unroll
      for (int k = 0; k < kAhead; k++) mark(k * 256 + tid, early_id[k]);
      for (int i = kAhead * 256 + tid; i < a.m; i += 256) mark(i, ids[i]);
      __syncthreads();
      // A value whose bits are a place that is looked for later would be taken for one: past the
      // first kAhead * 256 places values stay in memory (places are what is left in LDS).
      if (a.m <= kAhead * 256) {
        bool mine[kAhead];
#pragma unroll
        for (int k = 0; k < kAhead; k++) {
          const uint32_t at = (uint32_t)early_id[k] - (uint32_t)first;
          mine[k] = k * 256 + tid < a.m && at < (uint32_t)CHUNK && place[at] == (uint32_t)(k * 256 + tid);
        }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < kAhead; k++)
          if (mine[k]) place[early_id[k] - first] = early_bias[k] == early_bias[k] ? __float_as_uint(early_bias[k]) : 0x7FC00000u;
      }
    }
    __syncthreads();
  }
  auto get = [&](const u32x4& w, int i) -> float {
    if constexpr (ES == 4) return __uint_as_float(w[i]);
    else return xt_to_f32<XT == GEN_F16 ? 1 : 0>((w[i / 2] >> (16 * (i & 1))) & 0xFFFFu);
  };
  auto put = [&](u32x4& w, int i, float x) {
    if constexpr (ES == 4) w[i] = __float_as_uint(x);
    else w[i / 2] = (w[i / 2] & (i & 1 ? 0x0000FFFFu : 0xFFFF0000u)) | f32_to_xt<XT == GEN_F16 ? 1 : 0>(x) << (16 * (i & 1));
  };
  constexpr uint32_t kNone = XT == GEN_F32 ? 0xFF800000u : XT == GEN_F16 ? 0xFC00u : 0xFF80u;  // -inf
  if (first + e >= a.V) return;
  if (edits) {
    uint32_t c[W], p[W];
    bool any = false;
#pragma unroll
    for (int i = 0; i < W; i++) {
      c[i] = a.n > 0 ? times[e + i] : 0u;
      p[i] = a.m > 0 ? place[e + i] : kNoBias;
      any |= c[i] != 0u || p[i] != kNoBias;
    }
    if (any) {
#pragma unroll
      for (int i = 0; i < W; i++) {
        if (c[i] == 0u && p[i] == kNoBias) continue;
        float x = get(v, i);
        if (c[i]) {
          x = x > 0.f ? x / rep : x * rep;
          if (c[i] & ~kSeen) x -= pres + freq * (float)(c[i] & ~kSeen);
        }
        if (p[i] != kNoBias) x += a.m <= kAhead * 256 ? __uint_as_float(p[i]) : values[p[i]];
        put(v, i, x);
      }
    }
  }
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
    const size_t bytes = (size_t)((a.n > 0) + (a.m > 0)) * kChunk<XT> * 4;
    hipLaunchKernelGGL((adjust_logits_kernel<XT>), dim3((unsigned)groups), dim3(256), bytes, stream, a);
    return hipGetLastError();
  });
}

}  // namespace mlxq
