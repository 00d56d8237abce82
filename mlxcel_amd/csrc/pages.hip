// pages.hip — the pages of a paged key-value cache on gfx950: reserving them
// for new tokens, writing the tokens' keys and values, sharing them between
// sequences, freeing them and moving them together.
//
// A sequence (a row of the table) of n tokens holds the first
// ceil(n / page) entries of its row; refs counts the sequences that hold a
// page, 0 for a free one.  Free pages are given out in ascending order and
// requests served in their order, so every result is one fixed function of the
// inputs.  The bookkeeping is a few thousand words and runs in one workgroup
// (launch latency and its barriers bound it); the copies of pages run on the
// whole card and are bound by HBM.
//
// Page numbers out of range are never followed; such an entry is copied or
// kept as it stands.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "common.hpp"
#include "kernels.hpp"

namespace mlxq {

namespace {

constexpr int kPlanThreads = 1024, kPlanWaves = kPlanThreads / 64;
constexpr int kBlock = 4 * kPlanThreads;  // pages looked at together, four a thread
constexpr int kNear = 4096;               // free pages listed in LDS

typedef int32_t i32x4_e __attribute__((ext_vector_type(4), aligned(4)));

// Sums over the workgroup's kPlanThreads threads; two sets of words in turn, so
// that one barrier a sum is enough.
template <typename T>
struct Scan {
  T (*words)[kPlanWaves];
  int turn = 0;
  // exclusive, and the total
  __device__ __forceinline__ T operator()(T v, T& total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    T x = v;
#pragma unroll
    for (int s = 1; s < 64; s <<= 1) {
      const T o = __shfl_up(x, s);
      if (lane >= s) x += o;
    }
    T* w = words[turn ^= 1];
    if (lane == 63) w[wave] = x;
    __syncthreads();
    T before = 0;
    total = 0;
#pragma unroll
    for (int i = 0; i < kPlanWaves; i++) {
      if (i < wave) before += w[i];
      total += w[i];
    }
    return before + x - v;
  }
};

__device__ __forceinline__ int pages_of(int64_t tokens, int page) { return (int)((tokens + page - 1) / page); }

// refs of pages 4 tid .. 4 tid + 3 of the block from `at` on (past the end: held)
__device__ __forceinline__ i32x4_e load_refs(const int32_t* refs, int pages, int at) {
  const int p = at + 4 * (int)threadIdx.x;
  if (p <= pages - 4) return *reinterpret_cast<const i32x4_e*>(refs + p);
  i32x4_e r;
#pragma unroll
  for (int e = 0; e < 4; e++) r[e] = p < pages - e ? refs[p + e] : 1;
  return r;
}

// The free pages in ascending order, found as they are asked for: the first
// kNear in LDS, the others in scratch.  All members are the same in every thread.
struct FreeList {
  const int32_t* refs;
  int pages;
  int32_t *near, *far;
  i32x4_e block;  // refs at `at`, on their way
  int at = 0;
  int have = 0;
  __device__ __forceinline__ int32_t get(int i) const { return i < kNear ? near[i] : far[i]; }
  // until there are `want` or refs is at its end
  __device__ void extend(int64_t want, Scan<int>& scan) {
    while (have < want && at < pages) {
      const i32x4_e next = load_refs(refs, pages, at + kBlock);
      int n = 0, total;
#pragma unroll
      for (int e = 0; e < 4; e++) n += block[e] == 0;
      int r = have + scan(n, total);
#pragma unroll
      for (int e = 0; e < 4; e++)
        if (block[e] == 0) {
          (r < kNear ? near : far)[r] = at + 4 * (int)threadIdx.x + e;
          r++;
        }
      have += total;
      at += kBlock;
      block = next;
    }
    __syncthreads();  // the list's new entries are read by other threads
  }
};

// The last of n ascending numbers that is at most v.
__device__ __forceinline__ int owner_of(const int64_t* first, int n, int64_t v) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) / 2;
    if (first[mid] <= v) lo = mid;
    else hi = mid;
  }
  return lo;
}

__global__ __launch_bounds__(kPlanThreads) void cache_reserve_kernel(const CacheBook b, const int32_t* counts,
                                                                     int32_t* granted, int32_t* far) {
  __shared__ int64_t sums[2][kPlanWaves];
  __shared__ int flags[2][kPlanWaves];
  __shared__ int32_t near[kNear];
  __shared__ int64_t first[kPlanThreads];
  __shared__ int32_t need_s[kPlanThreads];
  __shared__ int64_t taken_s;
  const int tid = threadIdx.x;
  Scan<int64_t> scan{sums};
  Scan<int> count{flags};
  FreeList free{b.refs, b.pages, near, far, load_refs(b.refs, b.pages, 0)};
  int64_t used = 0;
  for (int r0 = 0; r0 < b.rows; r0 += kPlanThreads) {
    const int r = r0 + tid, n = min(kPlanThreads, b.rows - r0);
    int64_t len = 0, cnt = 0;
    int had = 0, need = 0;
    bool ok = false;
    if (r < b.rows) {
      len = b.lengths[r];
      cnt = counts[r];
      // a row that cannot hold its tokens, or counts below zero, are refused
      ok = len >= 0 && cnt >= 0 && len + cnt <= (int64_t)b.width * b.page;
      if (ok) {
        had = pages_of(len, b.page);
        need = pages_of(len + cnt, b.page) - had;
      }
    }
    int64_t total;
    int64_t before = scan(need, total);
    if (total > 0) {
      free.extend(used + total, count);
      if (free.have - used < total) {
        // too few pages: row by row, each that still fits
        need_s[tid] = need;
        __syncthreads();
        if (tid == 0) {
          int64_t left = free.have - used, sum = 0;
          for (int i = 0; i < n; i++) {
            first[i] = sum;
            if (need_s[i] > left) need_s[i] = -1;
            else {
              left -= need_s[i];
              sum += need_s[i];
            }
          }
          taken_s = sum;
        }
        __syncthreads();
        if (need_s[tid] < 0) {
          ok = false;
          need = 0;
        }
        before = first[tid];
        total = taken_s;
        __syncthreads();
      }
      first[tid] = r < b.rows ? before : INT64_MAX;
      need_s[tid] = had;
      __syncthreads();
      for (int64_t i = tid; i < total; i += kPlanThreads) {
        const int o = owner_of(first, n, i);
        const int32_t p = free.get((int)(used + i));
        b.table[(int64_t)(r0 + o) * b.table_row + need_s[o] + (i - first[o])] = p;
        b.refs[p] = 1;
      }
      used += total;
      __syncthreads();
    }
    if (r < b.rows) {
      granted[r] = ok;
      if (ok) b.lengths[r] = (int32_t)(len + cnt);
    }
  }
}

// ---- append ------------------------------------------------------------------

// One workgroup a token; the token's page number is the same for all its
// elements.  W: 16 bytes where everything is aligned to them, else one element.
template <typename W>
__global__ __launch_bounds__(256) void cache_append_kernel(const CacheAppendArgs a) {
  const int t = blockIdx.x, row = a.rows[t], pos = a.positions[t];
  if (row < 0 || row >= a.table_rows || pos < 0 || pos / a.page >= a.width) return;
  if (a.lengths && pos >= a.lengths[row]) return;
  const int pid = a.table[row * a.table_row + pos / a.page], off = pos % a.page;
  if (pid < 0 || pid >= a.pages) return;
  const int per = a.D * a.esz / (int)sizeof(W);  // words of a head
  for (int i = threadIdx.x; i < 2 * a.Hkv * per; i += 256) {
    const int v = i >= a.Hkv * per, j = v ? i - a.Hkv * per : i, h = j / per, w = j - h * per;
    const char* src = static_cast<const char*>(v ? a.v : a.k) +
                      (v ? t * a.v_tok + h * a.v_head : t * a.k_tok + h * a.k_head) * a.esz;
    char* dst = static_cast<char*>(v ? a.vp : a.kp) +
                (v ? pid * a.vp_page + h * a.vp_head + off * a.vp_tok
                   : pid * a.kp_page + h * a.kp_head + off * a.kp_tok) * a.esz;
    reinterpret_cast<W*>(dst)[w] = reinterpret_cast<const W*>(src)[w];
  }
}

// ---- copies of pages -----------------------------------------------------------

// One page by one workgroup, four words a thread on their way.  What is written
// is not kept in the caches, nor, where it is copied ONCE, what is read: fork of
// 4 into 32 over 72 pools 30.9 -> 27.7 us (36.6 with both), compact of 16 pools
// 71.4 -> 66.3 us (inputs in turn).
template <bool ONCE, typename W>
__device__ __forceinline__ void copy_page(char* base, int64_t stride, int64_t bytes, int from, int to) {
  const W* s = reinterpret_cast<const W*>(base + from * stride);
  W* d = reinterpret_cast<W*>(base + to * stride);
  const int64_t n = bytes / (int64_t)sizeof(W);
  int64_t i = threadIdx.x;
  for (; i + 3 * 256 < n; i += 4 * 256) {
    W v[4];
#pragma unroll
    for (int u = 0; u < 4; u++) v[u] = ONCE ? __builtin_nontemporal_load(s + i + u * 256) : s[i + u * 256];
#pragma unroll
    for (int u = 0; u < 4; u++) __builtin_nontemporal_store(v[u], d + i + u * 256);
  }
  for (; i < n; i += 256) d[i] = s[i];
}

// ---- fork ----------------------------------------------------------------------

// scratch: the list of free pages, then per pair {tokens or -1, fresh page or -1}
__global__ __launch_bounds__(kPlanThreads) void cache_fork_plan_kernel(const CacheBook b, const int32_t* src,
                                                                       const int32_t* dst, int n, int32_t* granted,
                                                                       int32_t* far, int32_t* pair) {
  __shared__ int sums[2][kPlanWaves], flags[2][kPlanWaves];
  __shared__ int32_t near[kNear], dst_s[kPlanThreads];
  const int tid = threadIdx.x;
  Scan<int> scan{sums}, count{flags};
  FreeList free{b.refs, b.pages, near, far, load_refs(b.refs, b.pages, 0)};
  int used = 0;
  for (int i0 = 0; i0 < n; i0 += kPlanThreads) {
    const int i = i0 + tid;
    const int s = i < n ? src[i] : -1, d = i < n ? dst[i] : -1;
    bool ok = s >= 0 && s < b.rows && d >= 0 && d < b.rows;
    const int64_t len = ok ? b.lengths[s] : 0;
    ok = ok && len >= 0 && len <= (int64_t)b.width * b.page && b.lengths[d] == 0;
    dst_s[tid] = d;
    __syncthreads();
    // the first pair of a row takes it
    for (int j = 0; ok && j < i0; j++) ok = dst[j] != d;
    for (int j = 0; ok && j < tid; j += 8) {
#pragma unroll
      for (int e = 0; e < 8; e++) ok = ok && (j + e >= tid || dst_s[j + e] != d);
    }
    const int part = ok && len % b.page != 0;
    int total;
    const int r = used + scan(part, total);
    if (total > 0) free.extend(used + total, count);
    int fresh = -1;
    if (part) {
      if (r < free.have) {
        fresh = free.get(r);
        b.refs[fresh] = 1;
      } else {
        ok = false;
      }
    }
    if (i < n) {
      granted[i] = ok;
      pair[2 * i] = ok ? (int32_t)len : -1;
      pair[2 * i + 1] = fresh;
    }
    used = min(used + total, free.have);
    __syncthreads();
  }
}

// Workgroups count pools first, in eights: those of one pool then run on one XCD
// whatever their pair, and a page that is copied several times is read into that
// XCD's L2 once.  Past the pools, and where `book`, one more a pair for its row
// of the table.
template <typename W>
__global__ __launch_bounds__(256) void cache_fork_copy_kernel(const CacheBook b, const int32_t* src, const int32_t* dst,
                                                              const int32_t* pair, const PoolList pools, int columns,
                                                              bool book) {
  const int i = blockIdx.x / columns, q = blockIdx.x - i * columns;
  const int len = pair[2 * i], fresh = pair[2 * i + 1];
  if (len < 0 || (q >= pools.n && (q > pools.n || !book))) return;
  const int full = len / b.page;
  const int32_t* from = b.table + src[i] * b.table_row;
  if (q == pools.n) {
    int32_t* to = b.table + dst[i] * b.table_row;
    for (int j = threadIdx.x; j < full; j += 256) {
      const int32_t p = from[j];
      to[j] = p;
      if (p >= 0 && p < b.pages) atomicAdd(b.refs + p, 1);
    }
    if (threadIdx.x == 0) {
      if (fresh >= 0) to[full] = fresh;
      b.lengths[dst[i]] = len;
    }
    return;
  }
  if (fresh < 0) return;
  const int old = from[full];
  if (old < 0 || old >= b.pages) return;
  copy_page<false, W>(pools.base[q], pools.stride, pools.bytes, old, fresh);
}

// ---- free ------------------------------------------------------------------------

__global__ __launch_bounds__(256) void cache_free_kernel(const CacheBook b, const int32_t* rows) {
  __shared__ int len_s;
  const int row = rows[blockIdx.x];
  if (row < 0 || row >= b.rows) return;
  // of several requests for one row one gets its length; the first entries of
  // the table are read meanwhile
  const int32_t* t = b.table + row * b.table_row;
  int32_t p = (int)threadIdx.x < b.width ? t[threadIdx.x] : -1;
  if (threadIdx.x == 0) len_s = atomicExch(b.lengths + row, 0);
  __syncthreads();
  const int64_t len = min((int64_t)max(len_s, 0), (int64_t)b.width * b.page);
  const int held = pages_of(len, b.page);
  for (int j = threadIdx.x; j < held; j += 256) {
    if (j >= 256) p = t[j];
    if (p >= 0 && p < b.pages) atomicSub(b.refs + p, 1);
  }
}

// ---- compact ---------------------------------------------------------------------

// scratch: the number of moves (16 words), to[pages], holes[pages], movers[pages]
__global__ __launch_bounds__(kPlanThreads) void cache_compact_plan_kernel(const CacheBook b, int32_t* live_out,
                                                                          int32_t* moves, int32_t* to, int32_t* holes,
                                                                          int32_t* movers) {
  __shared__ int sums[2][kPlanWaves];
  const int tid = threadIdx.x;
  Scan<int> scan{sums};
  i32x4_e block = load_refs(b.refs, b.pages, 0);
  auto held_at = [&](const i32x4_e& r, int at, int e) { return at + 4 * tid + e < b.pages && r[e] > 0; };
  int live = 0, n;
  for (int at = 0; at < b.pages; at += 4 * kBlock) {  // four blocks on their way
    i32x4_e r[4];
#pragma unroll
    for (int k = 0; k < 4; k++) r[k] = load_refs(b.refs, b.pages, at + k * kBlock);
#pragma unroll
    for (int k = 0; k < 4; k++)
#pragma unroll
      for (int e = 0; e < 4; e++) live += held_at(r[k], at + k * kBlock, e);
  }
  scan(live, n);
  // holes are the free pages below n, movers the held ones from n on: as many
  int nh = 0, nm = 0;
  for (int at = 0; at < b.pages; at += kBlock) {
    const i32x4_e r = block;
    block = load_refs(b.refs, b.pages, at + kBlock);
    const int p = at + 4 * tid;
    int mine = 0, total;  // holes and movers, 16 bits each
#pragma unroll
    for (int e = 0; e < 4; e++) mine += held_at(r, at, e) ? (p + e >= n ? 1 << 16 : 0) : (p + e < n);
    const int before = scan(mine, total);
    int h = nh + (before & 0xFFFF), m = nm + (before >> 16);
#pragma unroll
    for (int e = 0; e < 4; e++) {
      if (p + e >= b.pages) break;
      to[p + e] = p + e;
      if (held_at(r, at, e)) {
        if (p + e >= n) movers[m++] = p + e;
      } else if (p + e < n) {
        holes[h++] = p + e;
      }
    }
    nh += total & 0xFFFF;
    nm += total >> 16;
  }
  __syncthreads();
  for (int i = tid; i < nm; i += kPlanThreads) {
    const int h = holes[i], m = movers[i];
    to[m] = h;
    b.refs[h] = b.refs[m];
    b.refs[m] = 0;
  }
  if (tid == 0) {
    moves[0] = (int)nm;
    live_out[0] = n;
  }
}

// Workgroups take (move, pool) pairs in turn; the last `rows` workgroups
// rewrite a row of the table each.
template <typename W>
__global__ __launch_bounds__(256) void cache_compact_copy_kernel(const CacheBook b, const int32_t* moves,
                                                                 const int32_t* to, const int32_t* holes,
                                                                 const int32_t* movers, const PoolList pools,
                                                                 int movers_wgs) {
  if ((int)blockIdx.x >= movers_wgs) {
    const int row = blockIdx.x - movers_wgs;
    const int64_t len = min((int64_t)max(b.lengths[row], 0), (int64_t)b.width * b.page);
    int32_t* t = b.table + row * b.table_row;
    for (int j = threadIdx.x; j < pages_of(len, b.page); j += blockDim.x) {
      const int32_t p = t[j];
      if (p >= 0 && p < b.pages) t[j] = to[p];
    }
    return;
  }
  const int64_t n = (int64_t)moves[0] * pools.n;
  for (int64_t i = blockIdx.x; i < n; i += movers_wgs) {
    const int m = (int)(i / pools.n), q = (int)(i - (int64_t)m * pools.n);
    copy_page<true, W>(pools.base[q], pools.stride, pools.bytes, movers[m], holes[m]);
  }
}

// The widest of 16-, 2- and 1-byte words that every page of every pool allows:
// f(word).
template <typename F>
void with_word(const PoolList& p, F&& f) {
  uintptr_t v = (uintptr_t)p.bytes | (uintptr_t)p.stride;
  for (int i = 0; i < p.n; i++) v |= reinterpret_cast<uintptr_t>(p.base[i]);
  if ((v & 15) == 0) f(u32x4{});
  else if ((v & 1) == 0) f(uint16_t{});
  else f(uint8_t{});
}

}  // namespace

hipError_t launch_cache_reserve(const CacheBook& b, const int32_t* counts, int32_t* granted, int32_t* scratch,
                                hipStream_t stream) {
  if (b.rows == 0) return hipSuccess;
  hipLaunchKernelGGL(cache_reserve_kernel, dim3(1), dim3(kPlanThreads), 0, stream, b, counts, granted, scratch);
  return hipGetLastError();
}

hipError_t launch_cache_append(const CacheAppendArgs& a, hipStream_t stream) {
  if (a.T == 0 || a.Hkv == 0 || a.D == 0) return hipSuccess;
  if (a.pages < 1 || a.page < 1) return hipErrorInvalidValue;
  uintptr_t v = reinterpret_cast<uintptr_t>(a.k) | reinterpret_cast<uintptr_t>(a.v) |
                reinterpret_cast<uintptr_t>(a.kp) | reinterpret_cast<uintptr_t>(a.vp);
  const int64_t st[] = {a.k_tok, a.k_head, a.v_tok, a.v_head, a.kp_page, a.kp_head, a.kp_tok,
                        a.vp_page, a.vp_head, a.vp_tok, (int64_t)a.D};
  for (int64_t s : st) v |= (uintptr_t)(s * a.esz);
  const dim3 grid((unsigned)a.T), block(256);
  if ((v & 15) == 0) hipLaunchKernelGGL(cache_append_kernel<u32x4>, grid, block, 0, stream, a);
  else if (a.esz == 2) hipLaunchKernelGGL(cache_append_kernel<uint16_t>, grid, block, 0, stream, a);
  else hipLaunchKernelGGL(cache_append_kernel<uint32_t>, grid, block, 0, stream, a);
  return hipGetLastError();
}

int64_t cache_fork_words(int pages, int n) { return (int64_t)pages + 2 * (int64_t)n; }
int64_t cache_compact_words(int pages) { return 16 + 3 * (int64_t)pages; }

hipError_t launch_cache_fork_plan(const CacheBook& b, const int32_t* src, const int32_t* dst, int n, int32_t* granted,
                                  int32_t* scratch, hipStream_t stream) {
  if (n == 0) return hipSuccess;
  hipLaunchKernelGGL(cache_fork_plan_kernel, dim3(1), dim3(kPlanThreads), 0, stream, b, src, dst, n, granted, scratch,
                     scratch + b.pages);
  return hipGetLastError();
}

hipError_t launch_cache_fork_copy(const CacheBook& b, const int32_t* src, const int32_t* dst, int n,
                                  const int32_t* scratch, const PoolList& pools, bool book, hipStream_t stream) {
  if (n == 0) return hipSuccess;
  const int columns = (int)cache_fork_columns(book ? pools.n : pools.n - 1);
  if (columns == 0) return hipSuccess;
  if (n * (int64_t)columns > kMaxGroups) return hipErrorInvalidValue;
  const dim3 grid((unsigned)(n * columns)), block(256);
  const int32_t* pair = scratch + b.pages;
  with_word(pools, [&](auto w) {
    hipLaunchKernelGGL(cache_fork_copy_kernel<decltype(w)>, grid, block, 0, stream, b, src, dst, pair, pools, columns,
                       book);
  });
  return hipGetLastError();
}

hipError_t launch_cache_free(const CacheBook& b, const int32_t* rows, int n, hipStream_t stream) {
  if (n == 0 || b.rows == 0) return hipSuccess;
  hipLaunchKernelGGL(cache_free_kernel, dim3((unsigned)n), dim3(256), 0, stream, b, rows);
  return hipGetLastError();
}

hipError_t launch_cache_compact_plan(const CacheBook& b, int32_t* live, int32_t* scratch, hipStream_t stream) {
  int32_t* to = scratch + 16;
  hipLaunchKernelGGL(cache_compact_plan_kernel, dim3(1), dim3(kPlanThreads), 0, stream, b, live, scratch, to,
                     to + b.pages, to + 2 * (int64_t)b.pages);
  return hipGetLastError();
}

hipError_t launch_cache_compact_copy(const CacheBook& b, const int32_t* scratch, const PoolList& pools, bool book,
                                     int cus, hipStream_t stream) {
  // 2, 4, 8, 16 and 32 workgroups a CU: 16 pools of 32 KiB pages 65.0, 67.6, 67.2, 66.2
  // and 65.0 us, 48 pools of 4 KiB pages 36.1, 30.5, 28.6, 29.5 and 27.7
  const int wgs = pools.n > 0 && b.pages > 0 ? std::min(cus * 8, kCompactGroups) : 0;
  const int64_t grid = (int64_t)wgs + (book ? b.rows : 0);
  if (grid == 0) return hipSuccess;
  if (grid > kMaxGroups) return hipErrorInvalidValue;
  const int32_t* to = scratch + 16;
  const int32_t *holes = to + b.pages, *movers = to + 2 * (int64_t)b.pages;
  with_word(pools, [&](auto w) {
    hipLaunchKernelGGL(cache_compact_copy_kernel<decltype(w)>, dim3((unsigned)grid), dim3(256), 0, stream, b, scratch, to,
                       holes, movers, pools, wgs);
  });
  return hipGetLastError();
}

}  // namespace mlxq
