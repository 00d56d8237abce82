// host.hpp — what the C ABI's host files share (api.cpp, api_decode.cpp):
// errors and their status codes, dtype facts, views of mlxq_array, and the
// per-stream workspaces (defined in api.cpp).
#pragma once

#include <hip/hip_runtime.h>

#include <algorithm>
#include <exception>
#include <mutex>
#include <sstream>
#include <string>
#include <vector>

#include "../../include/mlxq.h"

namespace mlxq {
namespace host {

using Shape = std::vector<int64_t>;

// message of the last failing call on this thread
inline thread_local std::string g_last_error;

struct Error {
  mlxq_status code;
  std::string msg;
};

[[noreturn]] inline void fail(mlxq_status code, const std::string& msg) { throw Error{code, msg}; }
[[noreturn]] inline void invalid(const std::ostringstream& os) { fail(MLXQ_EINVAL, os.str()); }
[[noreturn]] inline void unsupported(const std::string& msg) { fail(MLXQ_EUNSUPPORTED, "[mlxq] " + msg); }

inline void hip_check(hipError_t e, const char* what) {
  if (e != hipSuccess) fail(MLXQ_EHIP, std::string("[mlxq] ") + what + ": " + hipGetErrorString(e));
}

template <typename F>
mlxq_status guarded(F&& f) {
  try {
    f();
    g_last_error.clear();
    return MLXQ_OK;
  } catch (const Error& e) {
    g_last_error = e.msg;
    return e.code;
  } catch (const std::exception& e) {
    g_last_error = std::string("[mlxq] internal error: ") + e.what();
    return MLXQ_EHIP;
  }
}

// ---- dtype facts (mlx::core::Dtype order) ----------------------------------

inline const char* dtype_name(int d) {
  static const char* names[] = {"bool",  "uint8",   "uint16",  "uint32",  "uint64",
                                "int8",  "int16",   "int32",   "int64",   "float16",
                                "float32", "float64", "bfloat16", "complex64"};
  return (d >= 0 && d <= 13) ? names[d] : "unknown";
}
inline bool is_floating(int d) { return d == MLXQ_FLOAT16 || d == MLXQ_FLOAT32 || d == MLXQ_FLOAT64 || d == MLXQ_BFLOAT16; }
inline bool is_integral(int d) { return d >= MLXQ_BOOL + 1 && d <= MLXQ_INT64; }
inline int dtype_size(int d) {
  static const int sz[] = {1, 1, 2, 4, 8, 1, 2, 4, 8, 2, 4, 8, 2, 8};
  return (d >= 0 && d <= 13) ? sz[d] : 0;
}

// Upstream MLX promote_types for the floating types this op layer meets
// (jax-style lattice: f16+bf16 -> f32, anything with f32/f64 -> the wider).
inline int promote(int a, int b) {
  if (a == b) return a;
  if (!is_floating(a) && !is_floating(b)) return a < b ? b : a;  // stays integral
  if (a == MLXQ_FLOAT64 || b == MLXQ_FLOAT64) return MLXQ_FLOAT64;
  if (is_floating(a) && !is_floating(b)) return a;
  if (is_floating(b) && !is_floating(a)) return b;
  return MLXQ_FLOAT32;  // f16/bf16/f32 mixes
}

// ---- array views -------------------------------------------------------------

struct View {
  const mlxq_array* a = nullptr;
  int64_t dim(int i) const { return a->shape[i < 0 ? i + a->ndim : i]; }
  int ndim() const { return a->ndim; }
  Shape shape() const { return Shape(a->shape, a->shape + a->ndim); }
  int dtype() const { return a->dtype; }
  int64_t size() const {
    int64_t s = 1;
    for (int i = 0; i < a->ndim; i++) s *= a->shape[i];
    return s;
  }
  bool row_contiguous() const {
    int64_t st = 1;
    for (int i = a->ndim - 1; i >= 0; i--) {
      if (a->shape[i] != 1 && a->strides[i] != st) return false;
      st *= a->shape[i];
    }
    return true;
  }
};

inline std::string fmt_shape(const Shape& s) {
  std::ostringstream os;
  os << "(";
  for (size_t i = 0; i < s.size(); i++) os << s[i] << (i + 1 == s.size() ? "" : ",");
  os << ")";
  return os.str();
}

inline void check_array(const mlxq_array* a, const char* name) {
  if (!a) fail(MLXQ_EINVAL, std::string("[mlxq] ") + name + " must not be NULL");
  if (a->ndim < 0 || a->ndim > MLXQ_MAX_DIMS)
    fail(MLXQ_EINVAL, std::string("[mlxq] ") + name + " has an invalid ndim");
  for (int i = 0; i < a->ndim; i++)
    if (a->shape[i] < 0) fail(MLXQ_EINVAL, std::string("[mlxq] ") + name + " has a negative dimension");
}

// ---- workspaces (api.cpp) ------------------------------------------------------

// Slots of a stream's workspace: 0 kernel scratch, 1 the row-contiguous copies
// of strided operands, 2 the flat index lists of gathers run in chunks, 3 the
// counters of launches that join partial results, 4 the page lists of the
// cache operators.
int current_device();
int device_cus(int dev);
// At least `bytes` of the stream's slot (grown unless the stream is being
// captured, which is an error).
void* stream_workspace(int dev, hipStream_t stream, size_t bytes, int slot);
// kSplitCounters words, all zero between launches; null where they would have
// to be allocated under a capture.
uint32_t* stream_counters(int dev, hipStream_t stream);
// The launches of one call that takes a stream's workspaces follow each other on
// the stream: held while it issues them, so that no call of another thread uses
// the same buffers between them.
class StreamTurn {
  std::lock_guard<std::mutex> lk_;

 public:
  explicit StreamTurn(hipStream_t stream);
};
bool needs_staging(const mlxq_array* a);
mlxq_array contiguous_like(const mlxq_array* a, void* data);
void copy_view(const mlxq_array* src, const mlxq_array* dst, hipStream_t stream);
void check_out(const mlxq_array* out, const Shape& shape, int dtype, const char* tag);

}  // namespace host
}  // namespace mlxq
