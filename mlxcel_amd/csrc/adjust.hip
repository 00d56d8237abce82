// adjust.hip — penalties for the tokens of a history, biases of single tokens
// and a grammar's mask on logits, on gfx950.
//
//   x' = x / r where x > 0, else x r             for tokens in the history
//   x' -= presence + frequency * times           for those in it `times` > 0 times after the prompt
//   x' += bias                                   for tokens with one
//   x' = -inf                                    for tokens whose bit of the mask is 0
//
// A logit is read and written once, which is the bound.  A workgroup takes a
// stretch of one row, loads it, and counts the history's tokens that fall into it
// in LDS, a word a token: whole numbers, so the order of the atomic operations
// does not matter.  Of several biases of one token the last in the list counts:
// LDS keeps the largest place.
#include <hip/hip_runtime.h>

#include <type_traits>

#include "common.hpp"
#include "kernels.hpp"

namespace mlxq {

namespace {

constexpr uint32_t kSeen = 0x80000000u;  // in the prompt; the bits below count the places after it

typedef uint32_t u32x4_e __attribute__((ext_vector_type(4), aligned(2)));

// One workgroup: logits [first, first + 256 U W) of row t, W in 16 bytes.
template <int XT, int U>
__global__ __launch_bounds__(256) void adjust_logits_kernel(const AdjustArgs a) {
  constexpr int ES = XT == GEN_F32 ? 4 : 2, W = 16 / ES, CHUNK = 256 * U * W;
  extern __shared__ __align__(16) uint32_t lds[];
  const int tid = threadIdx.x, chunks = (a.V + CHUNK - 1) / CHUNK, t = blockIdx.x / chunks;
  const int first = (blockIdx.x - t * chunks) * CHUNK;
  const char* src = static_cast<const char*>(a.x) + (t * a.x_row + first) * ES;
  char* dst = static_cast<char*>(a.out) + (t * a.out_row + first) * ES;
  u32x4 v[U];
#pragma unroll
  for (int u = 0; u < U; u++) {
    const int e = (u * 256 + tid) * W;
    if (first + e + W <= a.V) {
      const u32x4_e w = *reinterpret_cast<const u32x4_e*>(src + e * ES);
      v[u] = u32x4{w[0], w[1], w[2], w[3]};
    } else {
      uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
      for (int i = 0; i < W; i++)
        if (first + e + i < a.V) {
          if constexpr (ES == 4) w[i] = reinterpret_cast<const uint32_t*>(src)[e + i];
          else w[i / 2] |= (uint32_t)reinterpret_cast<const uint16_t*>(src)[e + i] << (16 * (i & 1));
        }
      v[u] = u32x4{w[0], w[1], w[2], w[3]};
    }
  }
  const bool edits = a.n > 0 || a.m > 0;
  uint32_t *times = lds, *place = lds + (a.n > 0 ? CHUNK : 0);
  if (edits) {
    for (int i = tid; i < ((a.n > 0) + (a.m > 0)) * CHUNK / 4; i += 256) reinterpret_cast<u32x4*>(lds)[i] = u32x4{0, 0, 0, 0};
    __syncthreads();
    if (a.n > 0) {
      const int n = a.history_lengths ? min(max(a.history_lengths[t], 0), a.n) : a.n;
      const int prompt = a.prompts ? a.prompts[t] : 0;
      const int32_t* h = a.history + t * a.history_row;
      for (int i = tid; i < n; i += 256) {
        const uint32_t at = (uint32_t)h[i] - (uint32_t)first;
        if (at < (uint32_t)CHUNK) {  // past the row's end it counts for nothing
          if (i < prompt) atomicOr(times + at, kSeen);
          else atomicAdd(times + at, 1u);
        }
      }
    }
    if (a.m > 0) {
      const int32_t* ids = a.bias_ids + t * a.bias_ids_row;
      for (int i = tid; i < a.m; i += 256) {
        const uint32_t at = (uint32_t)ids[i] - (uint32_t)first;
        if (at < (uint32_t)CHUNK) atomicMax(place + at, (uint32_t)i + 1u);
      }
    }
    __syncthreads();
  }
  const float rep = a.repetition ? a.repetition[t] : 1.f, pres = a.presence ? a.presence[t] : 0.f;
  const float freq = a.frequency ? a.frequency[t] : 0.f;
  auto get = [&](const u32x4& w, int i) -> float {
    if constexpr (ES == 4) return __uint_as_float(w[i]);
    else return xt_to_f32<XT == GEN_F16 ? 1 : 0>((w[i / 2] >> (16 * (i & 1))) & 0xFFFFu);
  };
  auto put = [&](u32x4& w, int i, float x) {
    if constexpr (ES == 4) w[i] = __float_as_uint(x);
    else w[i / 2] = (w[i / 2] & (i & 1 ? 0x0000FFFFu : 0xFFFF0000u)) | f32_to_xt<XT == GEN_F16 ? 1 : 0>(x) << (16 * (i & 1));
  };
#pragma unroll
  for (int u = 0; u < U; u++) {
    const int e = (u * 256 + tid) * W;
    if (first + e >= a.V) continue;
    if (edits) {
#pragma unroll
      for (int i = 0; i < W; i++) {
        const uint32_t c = a.n > 0 ? times[e + i] : 0u, p = a.m > 0 ? place[e + i] : 0u;
        if ((c | p) == 0u) continue;
        float x = get(v[u], i);
        if (c) {
          x = x > 0.f ? x / rep : x * rep;
          if (c & ~kSeen) x -= pres + freq * (float)(c & ~kSeen);
        }
        if (p) x += a.bias[t * a.bias_row + (p - 1)];
        put(v[u], i, x);
      }
    }
    if (a.mask) {
      const uint32_t bits = a.mask[t * a.mask_row + (first + e) / 32] >> ((first + e) & 31);
#pragma unroll
      for (int i = 0; i < W; i++)
        if (!(bits >> i & 1u)) put(v[u], i, -INFINITY);
    }
    if (first + e + W <= a.V) {
      *reinterpret_cast<u32x4_e*>(dst + e * ES) = u32x4_e{v[u][0], v[u][1], v[u][2], v[u][3]};
    } else {
#pragma unroll
      for (int i = 0; i < W; i++)
        if (first + e + i < a.V) {
          if constexpr (ES == 4) reinterpret_cast<uint32_t*>(dst)[e + i] = v[u][i];
          else reinterpret_cast<uint16_t*>(dst)[e + i] = (uint16_t)(v[u][i / 2] >> (16 * (i & 1)));
        }
    }
  }
}

// f(type, vectors a thread)
template <typename F>
auto with_kernel(const AdjustArgs& a, F&& f) {
  auto vectors = [&](auto xt) { return f(xt, std::integral_constant<int, 2>{}); };
  if (a.type == GEN_BF16) return vectors(std::integral_constant<int, GEN_BF16>{});
  if (a.type == GEN_F16) return vectors(std::integral_constant<int, GEN_F16>{});
  return vectors(std::integral_constant<int, GEN_F32>{});
}
template <int XT, int U>
constexpr int kChunk = 256 * U * (XT == GEN_F32 ? 4 : 8);

}  // namespace

int64_t adjust_logits_groups(const AdjustArgs& a) {
  const int chunk = with_kernel(a, [](auto xt, auto u) { return kChunk<decltype(xt)::value, decltype(u)::value>; });
  return (int64_t)((a.V + chunk - 1) / chunk) * a.T;
}

hipError_t launch_adjust_logits(const AdjustArgs& a, hipStream_t stream) {
  if (a.T == 0 || a.V == 0) return hipSuccess;
  const int64_t groups = adjust_logits_groups(a);
  if (groups > kMaxGroups) return hipErrorInvalidValue;
  return with_kernel(a, [&](auto xt, auto u) {
    constexpr int XT = decltype(xt)::value, U = decltype(u)::value;
    const size_t bytes = (size_t)((a.n > 0) + (a.m > 0)) * kChunk<XT, U> * 4;
    hipLaunchKernelGGL((adjust_logits_kernel<XT, U>), dim3((unsigned)groups), dim3(256), bytes, stream, a);
    return hipGetLastError();
  });
}

}  // namespace mlxq
