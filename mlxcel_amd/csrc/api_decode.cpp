// api_decode.cpp — the C ABI of the serving operators around the quantized
// projections (include/mlxq.h): attention over a paged cache, the cache's
// pages, residual norms, token log probabilities.  Arguments are checked here
// and the kernels launched; nothing waits for the device.
#include <hip/hip_runtime.h>

#include <cmath>

#include "host.hpp"
#include "kernels.hpp"

namespace {

using namespace mlxq::host;
using mlxq::CacheBook;

// [tag] message
struct Refusal {
  std::ostringstream os;
  explicit Refusal(const char* tag) { os << "[" << tag << "] "; }
  template <typename T>
  Refusal& operator<<(const T& v) {
    os << v;
    return *this;
  }
  [[noreturn]] void invalid() { mlxq::host::invalid(os); }
  [[noreturn]] void unsupported() { fail(MLXQ_EUNSUPPORTED, os.str()); }
};

// An operand with ndim axes (any number: -1) of type dtype (any: -1).
View operand(const mlxq_array* a, const char* tag, const char* name, int ndim, int dtype) {
  check_array(a, name);
  if (ndim >= 0 && a->ndim != ndim)
    (Refusal(tag) << name << " must have " << ndim << " dimensions but has shape " << fmt_shape(View{a}.shape()) << ".")
        .invalid();
  if (dtype >= 0 && a->dtype != dtype)
    (Refusal(tag) << name << " must be " << dtype_name(dtype) << " but is " << dtype_name(a->dtype) << ".").invalid();
  const int sz = dtype_size(a->dtype);
  if (sz == 0) (Refusal(tag) << name << " has an unknown dtype.").invalid();
  if (View{a}.size() > 0) {
    if (!a->data) (Refusal(tag) << name << " has no data.").invalid();
    if (reinterpret_cast<uintptr_t>(a->data) % sz) (Refusal(tag) << name << " is not aligned to its elements.").invalid();
  }
  return View{a};
}

void same_shape(View a, const Shape& s, const char* tag, const char* name) {
  if (a.shape() != s)
    (Refusal(tag) << name << " must have shape " << fmt_shape(s) << " but has shape " << fmt_shape(a.shape()) << ".")
        .invalid();
}

int float_type(View a, const char* tag, const char* name) {
  switch (a.dtype()) {
    case MLXQ_BFLOAT16: return mlxq::GEN_BF16;
    case MLXQ_FLOAT16: return mlxq::GEN_F16;
    case MLXQ_FLOAT32: return mlxq::GEN_F32;
    default:
      (Refusal(tag) << name << " must be bfloat16, float16 or float32 but is " << dtype_name(a.dtype()) << ".").invalid();
  }
}

bool unit_last(View a) { return a.ndim() == 0 || a.dim(-1) <= 1 || a.a->strides[a.ndim() - 1] == 1; }

int fits_int(int64_t v, const char* tag, const char* what) {
  if (v > 0x7FFFFFFF) (Refusal(tag) << what << " is too large (" << v << ").").unsupported();
  return (int)v;
}

// an int32 vector, dense
View vec32(const mlxq_array* a, const char* tag, const char* name) {
  View v = operand(a, tag, name, 1, MLXQ_INT32);
  if (!unit_last(v)) (Refusal(tag) << name << " must be contiguous.").unsupported();
  fits_int(v.dim(0), tag, name);
  return v;
}

View table32(const mlxq_array* a, const char* tag) {
  View t = operand(a, tag, "table", 2, MLXQ_INT32);
  if (!unit_last(t)) (Refusal(tag) << "table's rows must be contiguous.").unsupported();
  fits_int(t.dim(0), tag, "table");
  return t;
}

// Tokens a row of the table can hold: kernels count them in 32 bits.
void check_capacity(int64_t width, int64_t page, const char* tag) {
  if (page > 0 && width > ((int64_t)1 << 30) / page)
    (Refusal(tag) << "a table of " << width << " pages of " << page << " tokens is too wide.").unsupported();
}

CacheBook book(const mlxq_array* table, const mlxq_array* lengths, const mlxq_array* refs, int64_t page,
               const char* tag) {
  View t = table32(table, tag), l = vec32(lengths, tag, "lengths"), r = vec32(refs, tag, "refs");
  if (l.dim(0) != t.dim(0))
    (Refusal(tag) << "table and lengths must have as many rows but have shapes " << fmt_shape(t.shape()) << " and "
                  << fmt_shape(l.shape()) << ".").invalid();
  if (r.dim(0) > (1 << 30)) (Refusal(tag) << "refs has too many pages (" << r.dim(0) << ").").unsupported();
  if (page < 1) (Refusal(tag) << "a page must hold at least one token but holds " << page << ".").invalid();
  check_capacity(t.dim(1), page, tag);
  CacheBook b{};
  b.table = static_cast<int32_t*>(table->data);
  b.lengths = static_cast<int32_t*>(lengths->data);
  b.refs = static_cast<int32_t*>(refs->data);
  b.table_row = table->strides[0];
  b.rows = (int)t.dim(0);
  b.width = (int)t.dim(1);
  b.pages = (int)r.dim(0);
  b.page = (int)page;
  return b;
}

// Whether one page (every axis but the first) is a dense block in any order of
// its axes: then its bytes can be moved as they lie.
bool dense_page(View p) {
  bool used[MLXQ_MAX_DIMS] = {};
  int64_t next = 1;
  for (int n = 1; n < p.ndim(); n++) {
    int at = -1;
    for (int i = 1; i < p.ndim(); i++)
      if (!used[i] && (p.dim(i) == 1 || p.a->strides[i] == next) && (at < 0 || p.dim(at) != 1)) at = i;
    if (at < 0) return false;
    used[at] = true;
    next *= p.dim(at);
  }
  return true;
}

// The pools of one call: same type, shape and strides, pages that can be moved
// whole.  Returns the number of tokens of a page.
int64_t check_pools(int32_t n, const mlxq_array* const* pools, int64_t pages, const char* tag) {
  if (n < 1 || !pools) (Refusal(tag) << "at least one pool is needed.").invalid();
  View first = operand(pools[0], tag, "pools[0]", 4, -1);
  for (int i = 0; i < n; i++) {
    View p = operand(pools[i], tag, "pools", 4, -1);
    if (p.shape() != first.shape() || p.dtype() != first.dtype())
      (Refusal(tag) << "pools must have one shape and type but pools[" << i << "] is " << dtype_name(p.dtype()) << " "
                    << fmt_shape(p.shape()) << " and pools[0] " << dtype_name(first.dtype()) << " "
                    << fmt_shape(first.shape()) << ".").invalid();
    for (int d = 0; d < 4; d++)
      if (p.dim(d) > 1 && p.a->strides[d] != first.a->strides[d])
        (Refusal(tag) << "pools must have the same strides.").unsupported();
  }
  if (!dense_page(first)) (Refusal(tag) << "each page of a pool must be a dense block of memory.").unsupported();
  if (first.dim(0) != pages)
    (Refusal(tag) << "refs must have one entry a page but has " << pages << " and the pools have " << first.dim(0)
                  << " pages.").invalid();
  return first.dim(2);
}

// Runs f over the pools, at most kPoolsPerLaunch of them at a time.
template <typename F>
void each_pools(int32_t n, const mlxq_array* const* pools, F&& f) {
  View first{pools[0]};
  const int sz = dtype_size(first.dtype());
  mlxq::PoolList l{};
  l.bytes = first.dim(0) > 0 ? first.size() / first.dim(0) * sz : 0;
  l.stride = (first.dim(0) > 1 ? first.a->strides[0] : 0) * sz;
  for (int i = 0; i < n; i += mlxq::kPoolsPerLaunch) {
    l.n = l.bytes > 0 ? std::min(n - i, mlxq::kPoolsPerLaunch) : 0;
    for (int j = 0; j < l.n; j++) l.base[j] = static_cast<char*>(pools[i + j]->data);
    f(l, i == 0);
  }
}

int32_t* page_lists(hipStream_t stream, int64_t words) {
  return static_cast<int32_t*>(stream_workspace(current_device(), stream, (size_t)words * sizeof(int32_t), 4));
}

uint32_t* counters(int dev, hipStream_t stream, const char* tag) {
  uint32_t* c = stream_counters(dev, stream);
  if (!c)
    fail(MLXQ_ENOMEM, std::string("[") + tag + "] this stream has no counters yet and is being captured; run the call "
                      "once before the capture or reserve with mlxq_workspace_reserve");
  return c;
}

// Bytes of an operand's row-contiguous copy in the staging workspace.
size_t padded(View v) { return ((size_t)v.size() * dtype_size(v.dtype()) + 255) & ~(size_t)255; }

// x's rows as a matrix [rows][last axis]: the stride of a row where one number
// says it and the last axis is dense
bool matrix_rows(View x, int64_t& row) {
  if (!unit_last(x)) return false;
  row = x.ndim() > 0 ? x.dim(-1) : 1;
  int64_t want = -1;
  for (int i = x.ndim() - 2; i >= 0; i--) {
    if (x.dim(i) == 1) continue;
    if (want < 0) row = x.a->strides[i];
    else if (x.a->strides[i] != want) return false;
    want = x.a->strides[i] * x.dim(i);
  }
  return true;
}

}  // namespace

extern "C" {

mlxq_status mlxq_paged_attention(const mlxq_array* q, const mlxq_array* k_pool, const mlxq_array* v_pool,
                                 const mlxq_array* table, const mlxq_array* lengths, const mlxq_array* sinks,
                                 float scale, float softcap, int32_t window, mlxq_array* out, void* stream_) {
  return guarded([&] {
    const char* tag = "paged_attention";
    View x = operand(q, tag, "q", 3, -1);
    mlxq::PagedAttnArgs a{};
    a.type = float_type(x, tag, "q");
    View k = operand(k_pool, tag, "k_pool", 4, x.dtype()), v = operand(v_pool, tag, "v_pool", 4, x.dtype());
    same_shape(v, k.shape(), tag, "v_pool");
    View t = table32(table, tag), l = vec32(lengths, tag, "lengths");
    a.B = fits_int(x.dim(0), tag, "q");
    a.Hq = fits_int(x.dim(1), tag, "q");
    a.Hkv = fits_int(k.dim(1), tag, "k_pool");
    if (x.dim(2) != k.dim(3))
      (Refusal(tag) << "q and the pools must have one head width but have " << x.dim(2) << " and " << k.dim(3) << ".")
          .invalid();
    if (a.Hkv < 1 || a.Hq % a.Hkv)
      (Refusal(tag) << "query heads (" << a.Hq << ") must be a multiple of the pools' heads (" << a.Hkv << ").").invalid();
    if (t.dim(0) != a.B || l.dim(0) != a.B)
      (Refusal(tag) << "table and lengths must have one row a sequence (" << a.B << ") but have shapes "
                    << fmt_shape(t.shape()) << " and " << fmt_shape(l.shape()) << ".").invalid();
    if (!std::isfinite(scale)) (Refusal(tag) << "scale must be finite.").invalid();
    if (!std::isfinite(softcap) || softcap < 0.f)
      (Refusal(tag) << "softcap must be finite and not negative but is " << softcap << ".").invalid();
    if (window < 0) (Refusal(tag) << "window must not be negative but is " << window << ".").invalid();
    if (sinks) {
      View s = operand(sinks, tag, "sinks", 1, MLXQ_FLOAT32);
      same_shape(s, Shape{a.Hq}, tag, "sinks");
      if (!unit_last(s)) (Refusal(tag) << "sinks must be contiguous.").unsupported();
      a.sinks = static_cast<const float*>(sinks->data);
    }
    check_out(out, x.shape(), x.dtype(), tag);
    operand(out, tag, "out", 3, -1);
    if (x.size() == 0) return;
    if (x.dim(2) % 8 || x.dim(2) > 256)
      (Refusal(tag) << "head widths up to 256 that are a multiple of 8 are implemented, not " << x.dim(2) << ".")
          .unsupported();
    if (!unit_last(k) || !unit_last(v))
      (Refusal(tag) << "the pools' last axis must be contiguous.").unsupported();
    if (k.dim(0) < 1 || k.dim(2) < 1) (Refusal(tag) << "the pools have no pages.").invalid();
    check_capacity(t.dim(1), k.dim(2), tag);
    a.D = (int)x.dim(2);
    a.pages = fits_int(k.dim(0), tag, "k_pool");
    a.page = fits_int(k.dim(2), tag, "k_pool");
    a.width = (int)t.dim(1);
    a.window = window;
    a.scale = scale;
    a.softcap = softcap;
    a.k = k_pool->data;
    a.v = v_pool->data;
    a.k_page = k_pool->strides[0], a.k_head = k_pool->strides[1], a.k_tok = k_pool->strides[2];
    a.v_page = v_pool->strides[0], a.v_head = v_pool->strides[1], a.v_tok = v_pool->strides[2];
    a.table = static_cast<const int32_t*>(table->data);
    a.table_row = table->strides[0];
    a.lengths = static_cast<const int32_t*>(lengths->data);
    hipStream_t stream = reinterpret_cast<hipStream_t>(stream_);
    const StreamTurn turn(stream);
    mlxq_array qc = *q, oc = *out;
    const bool stage_q = !unit_last(x), stage_out = !View{out}.row_contiguous();
    if (stage_q || stage_out) {
      char* p = static_cast<char*>(
          stream_workspace(current_device(), stream, ((int)stage_q + (int)stage_out) * padded(x), 1));
      if (stage_q) {
        qc = contiguous_like(q, p);
        copy_view(q, &qc, stream);
        p += padded(x);
      }
      if (stage_out) oc = contiguous_like(out, p);
    }
    a.q = qc.data;
    a.q_b = qc.strides[0];
    a.q_h = qc.strides[1];
    a.out = oc.data;
    const int dev = current_device();
    int64_t part_bytes = 0;
    if (!mlxq::paged_attention_plan(a, device_cus(dev), &part_bytes))
      (Refusal(tag) << "a table of " << a.B << " rows of " << t.dim(1) << " pages holds too many keys for one call.")
          .unsupported();
    a.part = static_cast<float*>(stream_workspace(dev, stream, part_bytes, 0));
    a.cnt = counters(dev, stream, tag);
    hip_check(mlxq::launch_paged_attention(a, stream), "paged attention launch");
    if (stage_out) copy_view(&oc, out, stream);
  });
}

mlxq_status mlxq_cache_reserve(const mlxq_array* table, const mlxq_array* lengths, const mlxq_array* refs,
                               const mlxq_array* counts, int32_t page, mlxq_array* granted, void* stream_) {
  return guarded([&] {
    const char* tag = "cache_reserve";
    const CacheBook b = book(table, lengths, refs, page, tag);
    same_shape(vec32(counts, tag, "counts"), Shape{b.rows}, tag, "counts");
    same_shape(vec32(granted, tag, "granted"), Shape{b.rows}, tag, "granted");
    if (b.rows == 0) return;
    hipStream_t stream = reinterpret_cast<hipStream_t>(stream_);
    const StreamTurn turn(stream);
    hip_check(mlxq::launch_cache_reserve(b, static_cast<const int32_t*>(counts->data),
                                         static_cast<int32_t*>(granted->data), page_lists(stream, b.pages), stream),
              "cache reserve launch");
  });
}

mlxq_status mlxq_cache_append(const mlxq_array* k, const mlxq_array* v, const mlxq_array* k_pool,
                              const mlxq_array* v_pool, const mlxq_array* table, const mlxq_array* positions,
                              const mlxq_array* rows, const mlxq_array* lengths, void* stream_) {
  return guarded([&] {
    const char* tag = "cache_append";
    View kv = operand(k, tag, "k", 3, -1);
    float_type(kv, tag, "k");
    View vv = operand(v, tag, "v", 3, kv.dtype());
    same_shape(vv, kv.shape(), tag, "v");
    View kp = operand(k_pool, tag, "k_pool", 4, kv.dtype()), vp = operand(v_pool, tag, "v_pool", 4, kv.dtype());
    same_shape(vp, kp.shape(), tag, "v_pool");
    if (kp.dim(1) != kv.dim(1) || kp.dim(3) != kv.dim(2))
      (Refusal(tag) << "k and the pools must have the same heads and width but have shapes " << fmt_shape(kv.shape())
                    << " and " << fmt_shape(kp.shape()) << ".").invalid();
    View t = table32(table, tag);
    same_shape(vec32(positions, tag, "positions"), Shape{kv.dim(0)}, tag, "positions");
    same_shape(vec32(rows, tag, "rows"), Shape{kv.dim(0)}, tag, "rows");
    if (lengths) same_shape(vec32(lengths, tag, "lengths"), Shape{t.dim(0)}, tag, "lengths");
    if (kv.size() == 0 || t.size() == 0) return;
    if (!unit_last(kv) || !unit_last(vv) || !unit_last(kp) || !unit_last(vp))
      (Refusal(tag) << "the last axis of k, v and the pools must be contiguous.").unsupported();
    if (kp.dim(0) < 1 || kp.dim(2) < 1) (Refusal(tag) << "the pools have no pages.").invalid();
    check_capacity(t.dim(1), kp.dim(2), tag);
    fits_int(2 * kv.dim(1) * kv.dim(2) * dtype_size(kv.dtype()), tag, "a token");
    mlxq::CacheAppendArgs a{};
    a.k = k->data, a.v = v->data, a.kp = k_pool->data, a.vp = v_pool->data;
    a.k_tok = k->strides[0], a.k_head = k->strides[1], a.v_tok = v->strides[0], a.v_head = v->strides[1];
    a.kp_page = k_pool->strides[0], a.kp_head = k_pool->strides[1], a.kp_tok = k_pool->strides[2];
    a.vp_page = v_pool->strides[0], a.vp_head = v_pool->strides[1], a.vp_tok = v_pool->strides[2];
    a.table = static_cast<const int32_t*>(table->data);
    a.table_row = table->strides[0];
    a.positions = static_cast<const int32_t*>(positions->data);
    a.rows = static_cast<const int32_t*>(rows->data);
    a.lengths = lengths ? static_cast<const int32_t*>(lengths->data) : nullptr;
    a.T = fits_int(kv.dim(0), tag, "k");
    a.Hkv = (int)kv.dim(1);
    a.D = (int)kv.dim(2);
    a.esz = dtype_size(kv.dtype());
    a.table_rows = (int)t.dim(0);
    a.width = (int)t.dim(1);
    a.pages = fits_int(kp.dim(0), tag, "k_pool");
    a.page = fits_int(kp.dim(2), tag, "k_pool");
    hip_check(mlxq::launch_cache_append(a, reinterpret_cast<hipStream_t>(stream_)), "cache append launch");
  });
}

mlxq_status mlxq_cache_fork(int32_t n, const mlxq_array* const* pools, const mlxq_array* table,
                            const mlxq_array* lengths, const mlxq_array* refs, const mlxq_array* src,
                            const mlxq_array* dst, mlxq_array* granted, void* stream_) {
  return guarded([&] {
    const char* tag = "cache_fork";
    View r = vec32(refs, tag, "refs");
    const int64_t page = check_pools(n, pools, r.dim(0), tag);
    const CacheBook b = book(table, lengths, refs, page, tag);
    View s = vec32(src, tag, "src");
    same_shape(vec32(dst, tag, "dst"), s.shape(), tag, "dst");
    same_shape(vec32(granted, tag, "granted"), s.shape(), tag, "granted");
    const int pairs = (int)s.dim(0);
    if (pairs == 0) return;
    // before the plan, which changes the book
    if (pairs * mlxq::cache_fork_columns(std::min(n, mlxq::kPoolsPerLaunch)) > mlxq::kMaxGroups)
      (Refusal(tag) << "too many pairs (" << pairs << ") for one call.").unsupported();
    hipStream_t stream = reinterpret_cast<hipStream_t>(stream_);
    const int32_t *sp = static_cast<const int32_t*>(src->data), *dp = static_cast<const int32_t*>(dst->data);
    const StreamTurn turn(stream);
    int32_t* ws = page_lists(stream, mlxq::cache_fork_words(b.pages, pairs));
    hip_check(mlxq::launch_cache_fork_plan(b, sp, dp, pairs, static_cast<int32_t*>(granted->data), ws, stream),
              "cache fork launch");
    each_pools(n, pools, [&](const mlxq::PoolList& l, bool first) {
      hip_check(mlxq::launch_cache_fork_copy(b, sp, dp, pairs, ws, l, first, stream), "cache fork launch");
    });
  });
}

mlxq_status mlxq_cache_free(const mlxq_array* table, const mlxq_array* lengths, const mlxq_array* refs,
                            const mlxq_array* rows, int32_t page, void* stream_) {
  return guarded([&] {
    const char* tag = "cache_free";
    const CacheBook b = book(table, lengths, refs, page, tag);
    View r = vec32(rows, tag, "rows");
    hip_check(mlxq::launch_cache_free(b, static_cast<const int32_t*>(rows->data), (int)r.dim(0),
                                      reinterpret_cast<hipStream_t>(stream_)),
              "cache free launch");
  });
}

mlxq_status mlxq_cache_compact(int32_t n, const mlxq_array* const* pools, const mlxq_array* table,
                               const mlxq_array* lengths, const mlxq_array* refs, mlxq_array* live, void* stream_) {
  return guarded([&] {
    const char* tag = "cache_compact";
    View r = vec32(refs, tag, "refs");
    const int64_t page = check_pools(n, pools, r.dim(0), tag);
    const CacheBook b = book(table, lengths, refs, page, tag);
    same_shape(vec32(live, tag, "live"), Shape{1}, tag, "live");
    if (b.rows > mlxq::kMaxGroups - mlxq::kCompactGroups)
      (Refusal(tag) << "a table of " << b.rows << " rows is too long.").unsupported();
    hipStream_t stream = reinterpret_cast<hipStream_t>(stream_);
    const int cus = device_cus(current_device());
    const StreamTurn turn(stream);
    int32_t* ws = page_lists(stream, mlxq::cache_compact_words(b.pages));
    hip_check(mlxq::launch_cache_compact_plan(b, static_cast<int32_t*>(live->data), ws, stream),
              "cache compact launch");
    each_pools(n, pools, [&](const mlxq::PoolList& l, bool first) {
      hip_check(mlxq::launch_cache_compact_copy(b, ws, l, first, cus, stream), "cache compact launch");
    });
  });
}

mlxq_status mlxq_residual_norm(const mlxq_array* x, const mlxq_array* y, const mlxq_array* post_weight,
                               const mlxq_array* gate, float scale, const mlxq_array* pre_weight, float eps,
                               float weight_offset, mlxq_array* h, mlxq_array* n, void* stream_) {
  return guarded([&] {
    const char* tag = "residual_norm";
    View xv = operand(x, tag, "x", -1, -1);
    mlxq::ResidualNormArgs a{};
    a.type = float_type(xv, tag, "x");
    if (xv.ndim() < 1) (Refusal(tag) << "x must have at least one dimension.").invalid();
    const Shape shape = xv.shape();
    const int64_t H = shape.back();
    View yv = operand(y, tag, "y", -1, xv.dtype());
    same_shape(yv, shape, tag, "y");
    auto weight = [&](const mlxq_array* w, const char* name, int& type) -> const void* {
      if (!w) return nullptr;
      View v = operand(w, tag, name, 1, -1);
      same_shape(v, Shape{H}, tag, name);
      if (v.dtype() != xv.dtype() && v.dtype() != MLXQ_FLOAT32)
        (Refusal(tag) << name << " must have x's type (" << dtype_name(xv.dtype()) << ") or float32 but is "
                      << dtype_name(v.dtype()) << ".").invalid();
      if (!unit_last(v)) (Refusal(tag) << name << " must be contiguous.").unsupported();
      type = float_type(v, tag, name);
      return w->data;
    };
    a.post = weight(post_weight, "post_weight", a.post_type);
    a.pre = weight(pre_weight, "pre_weight", a.pre_type);
    if (!std::isfinite(scale)) (Refusal(tag) << "scale must be finite.").invalid();
    if (!std::isfinite(eps) || eps < 0.f) (Refusal(tag) << "eps must be finite and not negative.").invalid();
    if (!std::isfinite(weight_offset)) (Refusal(tag) << "weight_offset must be finite.").invalid();
    a.T = H > 0 ? xv.size() / H : 0;
    a.gate_div = 1;
    mlxq_array gc{};
    if (gate) {
      // The gate broadcasts against x: over the last axis, over all rows, or
      // over the last of the axes before it (one gate a batch entry).
      View g = operand(gate, tag, "gate", -1, xv.dtype());
      gc = *gate;
      if (g.ndim() < 1) (Refusal(tag) << "gate must have at least one dimension.").invalid();
      if (g.ndim() > xv.ndim()) (Refusal(tag) << "gate has more dimensions than x.").invalid();
      Shape gs = g.shape();
      while ((int)gs.size() < xv.ndim()) gs.insert(gs.begin(), 1);
      int64_t inner = 1;  // rows that share a gate row
      bool ones = true;   // of the axes seen so far, from the last
      for (int i = xv.ndim() - 2; i >= 0; i--) {
        if (gs[i] != shape[i] && gs[i] != 1)
          (Refusal(tag) << "gate with shape " << fmt_shape(g.shape()) << " does not broadcast to " << fmt_shape(shape)
                        << ".").invalid();
        if (gs[i] != shape[i]) {  // broadcast
          if (!ones)
            (Refusal(tag) << "a gate that is broadcast over an axis before one that it has is not implemented.")
                .unsupported();
          inner *= shape[i];
        } else if (shape[i] != 1) {
          ones = false;
        }
      }
      if (gs.back() != H && gs.back() != 1)
        (Refusal(tag) << "gate with shape " << fmt_shape(g.shape()) << " does not broadcast to " << fmt_shape(shape)
                      << ".").invalid();
      a.gate_div = std::max<int64_t>(inner, 1);
      a.gate_col = gs.back() == 1 && H != 1 ? 0 : 1;
    }
    check_out(h, shape, xv.dtype(), tag);
    operand(h, tag, "h", -1, -1);
    if ((n != nullptr) != (pre_weight != nullptr))
      (Refusal(tag) << "n is given where pre_weight is, and only there.").invalid();
    if (n) {
      check_out(n, shape, xv.dtype(), tag);
      operand(n, tag, "n", -1, -1);
    }
    if (xv.size() == 0) return;
    if (H > mlxq::kNormMaxH)
      (Refusal(tag) << "rows of at most " << mlxq::kNormMaxH << " elements are implemented, not " << H << ".")
          .unsupported();
    fits_int(a.T, tag, "x");
    a.H = (int)H;
    a.scale = scale, a.eps = eps, a.offset = weight_offset;
    // operands whose rows one stride does not describe go through a dense copy
    hipStream_t stream = reinterpret_cast<hipStream_t>(stream_);
    const StreamTurn turn(stream);
    mlxq_array xc = *x, yc = *y, hc = *h, nc = n ? *n : mlxq_array{};
    const bool sx = !matrix_rows(xv, a.x_row), sy = !matrix_rows(yv, a.y_row);
    const bool sg = gate && !matrix_rows(View{gate}, a.gate_row);
    const bool sh = !View{h}.row_contiguous(), sn = n && !View{n}.row_contiguous();
    if (sx || sy || sg || sh || sn) {
      const size_t bytes = ((int)sx + (int)sy + (int)sh + (int)sn) * padded(xv) + (sg ? padded(View{gate}) : 0);
      char* p = static_cast<char*>(stream_workspace(current_device(), stream, bytes, 1));
      auto in = [&](const mlxq_array* from, mlxq_array& c, int64_t& row) {
        c = contiguous_like(from, p);
        copy_view(from, &c, stream);
        row = View{from}.dim(-1);
        p += padded(View{from});
      };
      auto result = [&](const mlxq_array* to, mlxq_array& c) {
        c = contiguous_like(to, p);
        p += padded(View{to});
      };
      if (sx) in(x, xc, a.x_row);
      if (sy) in(y, yc, a.y_row);
      if (sg) in(gate, gc, a.gate_row);
      if (sh) result(h, hc);
      if (sn) result(n, nc);
    }
    if (gate && View{gate}.size() == View{gate}.dim(-1)) a.gate_row = 0;  // one row for all
    a.x = xc.data, a.y = yc.data, a.gate = gate ? gc.data : nullptr, a.h = hc.data, a.n = n ? nc.data : nullptr;
    hip_check(mlxq::launch_residual_norm(a, stream), "residual norm launch");
    if (sh) copy_view(&hc, h, stream);
    if (sn) copy_view(&nc, n, stream);
  });
}

mlxq_status mlxq_token_logprobs(const mlxq_array* logits, const mlxq_array* tokens, int32_t top_k, float scale,
                                mlxq_array* logprobs, mlxq_array* entropy, mlxq_array* top_logprobs,
                                mlxq_array* top_ids, void* stream_) {
  return guarded([&] {
    const char* tag = "token_logprobs";
    View x = operand(logits, tag, "logits", 2, -1);
    mlxq::LogprobArgs a{};
    a.type = float_type(x, tag, "logits");
    View t = operand(tokens, tag, "tokens", 2, MLXQ_INT32);
    if (t.dim(0) != x.dim(0))
      (Refusal(tag) << "tokens must have one row a row of logits (" << x.dim(0) << ") but have shape "
                    << fmt_shape(t.shape()) << ".").invalid();
    if (!(scale > 0.f) || !std::isfinite(scale))
      (Refusal(tag) << "scale must be finite and above zero but is " << scale << ".").invalid();
    if (top_k < 0 || top_k > x.dim(1))
      (Refusal(tag) << "top_k must be between 0 and the number of tokens (" << x.dim(1) << ") but is " << top_k << ".")
          .invalid();
    const Shape top{x.dim(0), top_k};
    check_out(logprobs, t.shape(), MLXQ_FLOAT32, tag);
    check_out(entropy, Shape{x.dim(0)}, MLXQ_FLOAT32, tag);
    if (top_k > 0) {
      check_out(top_logprobs, top, MLXQ_FLOAT32, tag);
      check_out(top_ids, top, MLXQ_INT32, tag);
    }
    auto dense = [&](const mlxq_array* r, const char* name) {
      View v = operand(r, tag, name, -1, -1);
      if (v.size() > 0 && !v.row_contiguous()) (Refusal(tag) << name << " must be contiguous.").unsupported();
      return r->data;
    };
    a.tokens = static_cast<const int32_t*>(dense(tokens, "tokens"));
    a.given = static_cast<float*>(dense(logprobs, "logprobs"));
    a.entropy = static_cast<float*>(dense(entropy, "entropy"));
    if (top_k > 0) {
      a.top = static_cast<float*>(dense(top_logprobs, "top_logprobs"));
      a.ids = static_cast<int32_t*>(dense(top_ids, "top_ids"));
    }
    if (x.dim(0) == 0) return;
    if (x.dim(1) == 0) (Refusal(tag) << "logits have no tokens.").invalid();
    if (top_k > mlxq::kTopMax)
      (Refusal(tag) << "at most " << mlxq::kTopMax << " alternatives are implemented, not " << top_k << ".").unsupported();
    if (x.dim(1) > ((int64_t)1 << 30)) (Refusal(tag) << "rows of " << x.dim(1) << " logits are too long.").unsupported();
    a.T = fits_int(x.dim(0), tag, "logits");
    a.V = (int)x.dim(1);
    a.n_tok = fits_int(t.dim(1), tag, "tokens");
    a.k = top_k;
    a.scale = scale;
    hipStream_t stream = reinterpret_cast<hipStream_t>(stream_);
    const StreamTurn turn(stream);
    mlxq_array xc = *logits;
    if (!unit_last(x)) {
      xc = contiguous_like(logits, stream_workspace(current_device(), stream, padded(x), 1));
      copy_view(logits, &xc, stream);
    }
    a.logits = xc.data;
    a.row = xc.strides[0];
    const int dev = current_device();
    int64_t part_bytes = 0;
    mlxq::token_logprobs_plan(a, device_cus(dev), &part_bytes);
    if (part_bytes > 0) {
      a.part = static_cast<float*>(stream_workspace(dev, stream, part_bytes, 0));
      a.cnt = counters(dev, stream, tag);
    }
    hip_check(mlxq::launch_token_logprobs(a, stream), "token log probabilities launch");
  });
}

}  // extern "C"
