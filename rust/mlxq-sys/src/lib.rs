//! Rust bindings to `libmlxq.so` (`include/mlxq.h`): the MI355X quantized
//! matmul library that stands in for MLX's `quantized_matmul`, `gather_qmm`,
//! `dequantize`, `quantize`, `quantized_linear_forward` and the fused decode
//! MoE kernels behind mlxcel's `cxx` bridge.
//!
//! `sys` holds the raw `extern "C"` declarations, one per symbol of the
//! header.  The safe layer mirrors the reference's bridge functions
//! (`src/lib/mlxcel-core/src/lib.rs:1374-1416` `gather_qmm` /
//! `quantized_matmul` / `dequantize`, `:697-707` `quantized_linear_forward`,
//! `:2336-2380` `fused_moe_expert_kernel` / `fused_moe_geglu_kernel`,
//! `:2666` `clear_memory_cache`, `:2720` `get_cache_memory`, `:2925-2940`
//! `quantized_matmul_matches_dense_gemm`): same argument order and meaning,
//! nullable arrays as `Option`, and a `Result` whose error carries the
//! library's status and message (the reference's `std::invalid_argument`
//! text for argument errors).  The library is eager: callers pass device
//! views of already-allocated arrays and a HIP stream; the output shape and
//! dtype come from the `*_shape` queries.

#![allow(clippy::too_many_arguments)]

use std::ffi::{CStr, CString};
use std::fmt;
use std::os::raw::c_void;

/// Raw declarations of `include/mlxq.h`.
pub mod sys {
    #![allow(non_camel_case_types)]
    use std::os::raw::{c_char, c_void};

    pub const MLXQ_MAX_DIMS: usize = 8;

    pub const MLXQ_OK: i32 = 0;
    pub const MLXQ_EINVAL: i32 = 1;
    pub const MLXQ_EUNSUPPORTED: i32 = 2;
    pub const MLXQ_EHIP: i32 = 3;
    pub const MLXQ_ENOMEM: i32 = 4;

    /// A strided view of device memory (strides in elements).
    #[repr(C)]
    #[derive(Clone, Copy, Debug)]
    pub struct mlxq_array {
        pub data: *mut c_void,
        pub dtype: i32,
        pub ndim: i32,
        pub shape: [i64; MLXQ_MAX_DIMS],
        pub strides: [i64; MLXQ_MAX_DIMS],
    }

    extern "C" {
        pub fn mlxq_last_error() -> *const c_char;
        pub fn mlxq_version() -> *const c_char;
        pub fn mlxq_workspace_reserve(bytes: usize, stream: *mut c_void) -> i32;
        pub fn mlxq_get_cache_memory() -> usize;
        pub fn mlxq_clear_cache() -> i32;
        pub fn mlxq_reload_options();

        pub fn mlxq_quantized_matmul(
            x: *const mlxq_array, w: *const mlxq_array, scales: *const mlxq_array, biases: *const mlxq_array,
            transpose: bool, group_size: i32, bits: i32, mode: *const c_char, out: *mut mlxq_array,
            stream: *mut c_void,
        ) -> i32;
        pub fn mlxq_quantized_matmul_noalloc(
            x: *const mlxq_array, w: *const mlxq_array, scales: *const mlxq_array, biases: *const mlxq_array,
            transpose: bool, group_size: i32, bits: i32, mode: *const c_char, out: *mut mlxq_array,
            stream: *mut c_void,
        ) -> i32;
        pub fn mlxq_quantized_linear(
            x: *const mlxq_array, w: *const mlxq_array, scales: *const mlxq_array, biases: *const mlxq_array,
            linear_bias: *const mlxq_array, group_size: i32, bits: i32, mode: *const c_char,
            out: *mut mlxq_array, stream: *mut c_void,
        ) -> i32;
        pub fn mlxq_quantized_matmul_matches_dense_gemm(
            x: *const mlxq_array, w: *const mlxq_array, scales: *const mlxq_array, biases: *const mlxq_array,
            group_size: i32, bits: i32,
        ) -> i32;
        pub fn mlxq_quantized_matmul_multi(
            x: *const mlxq_array, n: i32, w: *const *const mlxq_array, scales: *const *const mlxq_array,
            biases: *const *const mlxq_array, group_size: i32, bits: i32, mode: *const c_char,
            out: *const *mut mlxq_array, stream: *mut c_void,
        ) -> i32;
        pub fn mlxq_quantized_matmul_shape(
            x: *const mlxq_array, w: *const mlxq_array, scales: *const mlxq_array, biases: *const mlxq_array,
            transpose: bool, group_size: i32, bits: i32, mode: *const c_char, out_ndim: *mut i32,
            out_shape: *mut i64, out_dtype: *mut i32,
        ) -> i32;
        pub fn mlxq_gather_qmm(
            x: *const mlxq_array, w: *const mlxq_array, scales: *const mlxq_array, biases: *const mlxq_array,
            lhs_indices: *const mlxq_array, rhs_indices: *const mlxq_array, transpose: bool, group_size: i32,
            bits: i32, sorted_indices: bool, mode: *const c_char, global_scale: *const mlxq_array,
            out: *mut mlxq_array, stream: *mut c_void,
        ) -> i32;
        pub fn mlxq_gather_qmm_shape(
            x: *const mlxq_array, w: *const mlxq_array, scales: *const mlxq_array, biases: *const mlxq_array,
            lhs_indices: *const mlxq_array, rhs_indices: *const mlxq_array, transpose: bool, group_size: i32,
            bits: i32, mode: *const c_char, out_ndim: *mut i32, out_shape: *mut i64, out_dtype: *mut i32,
        ) -> i32;
        pub fn mlxq_dequantize(
            w: *const mlxq_array, scales: *const mlxq_array, biases: *const mlxq_array, group_size: i32,
            bits: i32, mode: *const c_char, dtype: i32, out: *mut mlxq_array, stream: *mut c_void,
        ) -> i32;
        pub fn mlxq_quantize(
            w: *const mlxq_array, group_size: i32, bits: i32, mode: *const c_char, wq_out: *mut mlxq_array,
            scales_out: *mut mlxq_array, biases_out: *mut mlxq_array, stream: *mut c_void,
        ) -> i32;
        pub fn mlxq_fused_moe_expert(
            x: *const mlxq_array, indices: *const mlxq_array, gate_w: *const mlxq_array,
            gate_s: *const mlxq_array, gate_b: *const mlxq_array, up_w: *const mlxq_array,
            up_s: *const mlxq_array, up_b: *const mlxq_array, down_w: *const mlxq_array,
            down_s: *const mlxq_array, down_b: *const mlxq_array, scores: *const mlxq_array, din: i32,
            dff: i32, k: i32, gu_bits: i32, d_bits: i32, group_size: i32, out: *mut mlxq_array,
            stream: *mut c_void,
        ) -> i32;
        pub fn mlxq_fused_moe_geglu(
            x: *const mlxq_array, indices: *const mlxq_array, gate_w: *const mlxq_array,
            gate_s: *const mlxq_array, gate_b: *const mlxq_array, up_w: *const mlxq_array,
            up_s: *const mlxq_array, up_b: *const mlxq_array, down_w: *const mlxq_array,
            down_s: *const mlxq_array, down_b: *const mlxq_array, scores: *const mlxq_array, din: i32,
            dff: i32, k: i32, gu_bits: i32, d_bits: i32, group_size: i32, out: *mut mlxq_array,
            stream: *mut c_void,
        ) -> i32;
        pub fn mlxq_paged_attention(
            q: *const mlxq_array, k_pool: *const mlxq_array, v_pool: *const mlxq_array, table: *const mlxq_array,
            lengths: *const mlxq_array, sinks: *const mlxq_array, scale: f32, softcap: f32, window: i32,
            out: *mut mlxq_array, stream: *mut c_void,
        ) -> i32;
        pub fn mlxq_cache_reserve(
            table: *const mlxq_array, lengths: *const mlxq_array, refs: *const mlxq_array,
            counts: *const mlxq_array, page: i32, granted: *mut mlxq_array, stream: *mut c_void,
        ) -> i32;
        pub fn mlxq_cache_append(
            k: *const mlxq_array, v: *const mlxq_array, k_pool: *const mlxq_array, v_pool: *const mlxq_array,
            table: *const mlxq_array, positions: *const mlxq_array, rows: *const mlxq_array,
            lengths: *const mlxq_array, stream: *mut c_void,
        ) -> i32;
        pub fn mlxq_cache_fork(
            n: i32, pools: *const *const mlxq_array, table: *const mlxq_array, lengths: *const mlxq_array,
            refs: *const mlxq_array, src: *const mlxq_array, dst: *const mlxq_array, granted: *mut mlxq_array,
            stream: *mut c_void,
        ) -> i32;
        pub fn mlxq_cache_free(
            table: *const mlxq_array, lengths: *const mlxq_array, refs: *const mlxq_array,
            rows: *const mlxq_array, page: i32, stream: *mut c_void,
        ) -> i32;
        pub fn mlxq_cache_compact(
            n: i32, pools: *const *const mlxq_array, table: *const mlxq_array, lengths: *const mlxq_array,
            refs: *const mlxq_array, live: *mut mlxq_array, stream: *mut c_void,
        ) -> i32;
        pub fn mlxq_residual_norm(
            x: *const mlxq_array, y: *const mlxq_array, post_weight: *const mlxq_array, gate: *const mlxq_array,
            scale: f32, pre_weight: *const mlxq_array, eps: f32, weight_offset: f32, h: *mut mlxq_array,
            n: *mut mlxq_array, stream: *mut c_void,
        ) -> i32;
        pub fn mlxq_token_logprobs(
            logits: *const mlxq_array, tokens: *const mlxq_array, top_k: i32, scale: f32,
            logprobs: *mut mlxq_array, entropy: *mut mlxq_array, top_logprobs: *mut mlxq_array,
            top_ids: *mut mlxq_array, stream: *mut c_void,
        ) -> i32;
        pub fn mlxq_paged_attention_chunk(
            q: *const mlxq_array, k_pool: *const mlxq_array, v_pool: *const mlxq_array, table: *const mlxq_array,
            lengths: *const mlxq_array, starts: *const mlxq_array, sinks: *const mlxq_array, scale: f32, softcap: f32,
            window: i32, out: *mut mlxq_array, stream: *mut c_void,
        ) -> i32;
        pub fn mlxq_rotary_frequencies(
            dims: i32, base: f64, scaling: i32, factor: f64, original: f64, low: f64, high: f64, inv_freq: *mut f32,
            attention_factor: *mut f32,
        ) -> i32;
        pub fn mlxq_rotary(
            x: *const mlxq_array, positions: *const mlxq_array, inv_freq: *const mlxq_array, interleaved: bool,
            factor: f32, out: *mut mlxq_array, stream: *mut c_void,
        ) -> i32;
        pub fn mlxq_rotary_append(
            q: *const mlxq_array, k: *const mlxq_array, v: *const mlxq_array, k_pool: *const mlxq_array,
            v_pool: *const mlxq_array, table: *const mlxq_array, positions: *const mlxq_array,
            rows: *const mlxq_array, lengths: *const mlxq_array, inv_freq: *const mlxq_array, interleaved: bool,
            factor: f32, out: *mut mlxq_array, stream: *mut c_void,
        ) -> i32;
        pub fn mlxq_adjust_logits(
            logits: *const mlxq_array, history: *const mlxq_array, history_lengths: *const mlxq_array,
            prompts: *const mlxq_array, repetition: *const mlxq_array, presence: *const mlxq_array,
            frequency: *const mlxq_array, bias_ids: *const mlxq_array, bias: *const mlxq_array,
            mask: *const mlxq_array, out: *mut mlxq_array, stream: *mut c_void,
        ) -> i32;
    }
}

pub use sys::MLXQ_MAX_DIMS;

/// Element types, numbered as `mlx::core::Dtype::Val` (`include/mlxq.h`).
#[repr(i32)]
#[derive(Clone, Copy, Debug, PartialEq, Eq)]
pub enum Dtype {
    Bool = 0,
    Uint8 = 1,
    Uint16 = 2,
    Uint32 = 3,
    Uint64 = 4,
    Int8 = 5,
    Int16 = 6,
    Int32 = 7,
    Int64 = 8,
    Float16 = 9,
    Float32 = 10,
    Float64 = 11,
    Bfloat16 = 12,
    Complex64 = 13,
}

impl Dtype {
    pub fn from_code(code: i32) -> Option<Dtype> {
        use Dtype::*;
        Some(match code {
            0 => Bool,
            1 => Uint8,
            2 => Uint16,
            3 => Uint32,
            4 => Uint64,
            5 => Int8,
            6 => Int16,
            7 => Int32,
            8 => Int64,
            9 => Float16,
            10 => Float32,
            11 => Float64,
            12 => Bfloat16,
            13 => Complex64,
            _ => return None,
        })
    }
}

/// What a failing call returned.  `Invalid` carries the reference's
/// exception text (rethrow it as MLX would); `Unsupported` means "fall back
/// to MLX"; `Hip` and `NoMem` are execution failures.
#[derive(Clone, Debug, PartialEq, Eq)]
pub enum Error {
    Invalid(String),
    Unsupported(String),
    Hip(String),
    NoMem(String),
    Other(i32, String),
}

impl fmt::Display for Error {
    fn fmt(&self, f: &mut fmt::Formatter<'_>) -> fmt::Result {
        match self {
            Error::Invalid(m) | Error::Unsupported(m) | Error::Hip(m) | Error::NoMem(m) => f.write_str(m),
            Error::Other(code, m) => write!(f, "mlxq status {code}: {m}"),
        }
    }
}

impl std::error::Error for Error {}

pub type Result<T> = std::result::Result<T, Error>;

fn last_error() -> String {
    // SAFETY: the library returns a NUL-terminated, thread-local string.
    unsafe {
        let p = sys::mlxq_last_error();
        if p.is_null() {
            String::new()
        } else {
            CStr::from_ptr(p).to_string_lossy().into_owned()
        }
    }
}

/// Maps a status code to `Ok(())` or the error with the thread's message.
pub fn check(status: i32) -> Result<()> {
    match status {
        sys::MLXQ_OK => Ok(()),
        sys::MLXQ_EINVAL => Err(Error::Invalid(last_error())),
        sys::MLXQ_EUNSUPPORTED => Err(Error::Unsupported(last_error())),
        sys::MLXQ_EHIP => Err(Error::Hip(last_error())),
        sys::MLXQ_ENOMEM => Err(Error::NoMem(last_error())),
        code => Err(Error::Other(code, last_error())),
    }
}

/// A strided view of device memory: what mlxcel's bridge builds from an
/// evaluated `mlx::core::array` (its data pointer, dtype, shape and strides
/// in elements).
#[derive(Clone, Copy, Debug)]
pub struct ArrayView {
    raw: sys::mlxq_array,
}

impl ArrayView {
    /// Row-contiguous view of `shape`.
    ///
    /// # Safety
    /// `data` must be a device pointer of the current HIP device holding the
    /// whole view, alive until the stream has run the calls that use it.
    pub unsafe fn contiguous(data: *mut c_void, dtype: Dtype, shape: &[i64]) -> ArrayView {
        let mut strides = vec![0i64; shape.len()];
        let mut st = 1i64;
        for i in (0..shape.len()).rev() {
            strides[i] = st;
            st *= shape[i];
        }
        ArrayView::strided(data, dtype, shape, &strides)
    }

    /// View with explicit strides (in elements).
    ///
    /// # Safety
    /// As `contiguous`; every element the strides reach must lie inside the
    /// allocation.
    pub unsafe fn strided(data: *mut c_void, dtype: Dtype, shape: &[i64], strides: &[i64]) -> ArrayView {
        assert!(shape.len() <= MLXQ_MAX_DIMS && strides.len() == shape.len(), "at most 8 dimensions");
        let mut raw = sys::mlxq_array {
            data,
            dtype: dtype as i32,
            ndim: shape.len() as i32,
            shape: [0; MLXQ_MAX_DIMS],
            strides: [0; MLXQ_MAX_DIMS],
        };
        raw.shape[..shape.len()].copy_from_slice(shape);
        raw.strides[..strides.len()].copy_from_slice(strides);
        ArrayView { raw }
    }

    pub fn shape(&self) -> &[i64] {
        &self.raw.shape[..self.raw.ndim as usize]
    }

    pub fn dtype(&self) -> Option<Dtype> {
        Dtype::from_code(self.raw.dtype)
    }

    pub fn as_raw(&self) -> *const sys::mlxq_array {
        &self.raw
    }

    fn as_raw_mut(&mut self) -> *mut sys::mlxq_array {
        &mut self.raw
    }
}

fn opt(a: Option<&ArrayView>) -> *const sys::mlxq_array {
    a.map_or(std::ptr::null(), |v| v.as_raw())
}

fn cmode(mode: &str) -> CString {
    // a mode with an interior NUL cannot name a valid mode; the library
    // rejects the empty string with the reference's message
    CString::new(mode).unwrap_or_default()
}

/// Output shape and dtype of a call, from a `*_shape` query.
#[derive(Clone, Debug, PartialEq, Eq)]
pub struct OutSpec {
    pub shape: Vec<i64>,
    pub dtype: Dtype,
}

fn out_spec(ndim: i32, shape: &[i64; MLXQ_MAX_DIMS], dtype: i32) -> Result<OutSpec> {
    let dtype = Dtype::from_code(dtype).ok_or_else(|| Error::Other(-1, format!("unknown dtype code {dtype}")))?;
    Ok(OutSpec { shape: shape[..ndim as usize].to_vec(), dtype })
}

/// The library's version string.
pub fn version() -> String {
    // SAFETY: a static NUL-terminated string.
    unsafe { CStr::from_ptr(sys::mlxq_version()).to_string_lossy().into_owned() }
}

/// Shape and dtype `quantized_matmul` would produce (the reference's
/// validation and messages, no device work).
pub fn quantized_matmul_shape(
    x: &ArrayView, w: &ArrayView, scales: &ArrayView, biases: Option<&ArrayView>, transpose: bool,
    group_size: i32, bits: i32, mode: &str,
) -> Result<OutSpec> {
    let m = cmode(mode);
    let (mut nd, mut sh, mut dt) = (0i32, [0i64; MLXQ_MAX_DIMS], 0i32);
    // SAFETY: the views are plain structs; no device memory is touched.
    check(unsafe {
        sys::mlxq_quantized_matmul_shape(
            x.as_raw(), w.as_raw(), scales.as_raw(), opt(biases), transpose, group_size, bits, m.as_ptr(),
            &mut nd, sh.as_mut_ptr(), &mut dt,
        )
    })?;
    out_spec(nd, &sh, dt)
}

/// `y = x @ dequantize(w, scales, biases)^T` (transpose) or without the
/// transpose, as the reference's `ffi::quantized_matmul`, into `out`.
///
/// # Safety
/// Every view must describe live device memory of the current device;
/// `stream` is a `hipStream_t` (null: the default stream).
pub unsafe fn quantized_matmul(
    x: &ArrayView, w: &ArrayView, scales: &ArrayView, biases: Option<&ArrayView>, transpose: bool,
    group_size: i32, bits: i32, mode: &str, out: &mut ArrayView, stream: *mut c_void,
) -> Result<()> {
    let m = cmode(mode);
    check(sys::mlxq_quantized_matmul(
        x.as_raw(), w.as_raw(), scales.as_raw(), opt(biases), transpose, group_size, bits, m.as_ptr(),
        out.as_raw_mut(), stream,
    ))
}

/// `quantized_matmul` with its scratch in the library's fixed per-GPU array:
/// for callers that cannot allocate (HIP-graph capture, serving loops).
/// Calls that overlap on one GPU race on that array.
///
/// # Safety
/// As `quantized_matmul`.
pub unsafe fn quantized_matmul_noalloc(
    x: &ArrayView, w: &ArrayView, scales: &ArrayView, biases: Option<&ArrayView>, transpose: bool,
    group_size: i32, bits: i32, mode: &str, out: &mut ArrayView, stream: *mut c_void,
) -> Result<()> {
    let m = cmode(mode);
    check(sys::mlxq_quantized_matmul_noalloc(
        x.as_raw(), w.as_raw(), scales.as_raw(), opt(biases), transpose, group_size, bits, m.as_ptr(),
        out.as_raw_mut(), stream,
    ))
}

/// The reference's `quantized_linear_forward`: `x @ W^T + linear_bias`.
///
/// # Safety
/// As `quantized_matmul`.
pub unsafe fn quantized_linear_forward(
    x: &ArrayView, weight: &ArrayView, scales: &ArrayView, biases: Option<&ArrayView>,
    linear_bias: Option<&ArrayView>, group_size: i32, bits: i32, mode: &str, out: &mut ArrayView,
    stream: *mut c_void,
) -> Result<()> {
    let m = cmode(mode);
    check(sys::mlxq_quantized_linear(
        x.as_raw(), weight.as_raw(), scales.as_raw(), opt(biases), opt(linear_bias), group_size, bits,
        m.as_ptr(), out.as_raw_mut(), stream,
    ))
}

/// The reference's `quantized_matmul_matches_dense_gemm`: false here for
/// every input (no call returns the bytes of dequantize + a dense GEMM).
pub fn quantized_matmul_matches_dense_gemm(
    x: &ArrayView, weight: &ArrayView, scales: &ArrayView, biases: Option<&ArrayView>, group_size: i32,
    bits: i32,
) -> bool {
    // SAFETY: host-only predicate.
    unsafe {
        sys::mlxq_quantized_matmul_matches_dense_gemm(
            x.as_raw(), weight.as_raw(), scales.as_raw(), opt(biases), group_size, bits,
        ) != 0
    }
}

/// Several projections of one activation (q/k/v, gate/up): bit for bit the
/// separate `quantized_matmul` calls, one launch at decode row counts.
///
/// # Safety
/// As `quantized_matmul`; the slices have equal lengths (1 to 4).
pub unsafe fn quantized_matmul_multi(
    x: &ArrayView, w: &[&ArrayView], scales: &[&ArrayView], biases: Option<&[&ArrayView]>, group_size: i32,
    bits: i32, mode: &str, out: &mut [&mut ArrayView], stream: *mut c_void,
) -> Result<()> {
    let n = w.len();
    assert!(scales.len() == n && out.len() == n && biases.map_or(true, |b| b.len() == n));
    let m = cmode(mode);
    let wp: Vec<*const sys::mlxq_array> = w.iter().map(|v| v.as_raw()).collect();
    let sp: Vec<*const sys::mlxq_array> = scales.iter().map(|v| v.as_raw()).collect();
    let bp: Option<Vec<*const sys::mlxq_array>> = biases.map(|b| b.iter().map(|v| v.as_raw()).collect());
    let op: Vec<*mut sys::mlxq_array> = out.iter_mut().map(|v| v.as_raw_mut()).collect();
    check(sys::mlxq_quantized_matmul_multi(
        x.as_raw(), n as i32, wp.as_ptr(), sp.as_ptr(), bp.as_ref().map_or(std::ptr::null(), |b| b.as_ptr()),
        group_size, bits, m.as_ptr(), op.as_ptr(), stream,
    ))
}

/// Shape and dtype `gather_qmm` would produce.
pub fn gather_qmm_shape(
    x: &ArrayView, w: &ArrayView, scales: &ArrayView, biases: Option<&ArrayView>,
    lhs_indices: Option<&ArrayView>, rhs_indices: Option<&ArrayView>, transpose: bool, group_size: i32,
    bits: i32, mode: &str,
) -> Result<OutSpec> {
    let m = cmode(mode);
    let (mut nd, mut sh, mut dt) = (0i32, [0i64; MLXQ_MAX_DIMS], 0i32);
    // SAFETY: host-only query.
    check(unsafe {
        sys::mlxq_gather_qmm_shape(
            x.as_raw(), w.as_raw(), scales.as_raw(), opt(biases), opt(lhs_indices), opt(rhs_indices), transpose,
            group_size, bits, m.as_ptr(), &mut nd, sh.as_mut_ptr(), &mut dt,
        )
    })?;
    out_spec(nd, &sh, dt)
}

/// The reference's `ffi::gather_qmm`, into `out`.
///
/// # Safety
/// As `quantized_matmul`.
pub unsafe fn gather_qmm(
    x: &ArrayView, w: &ArrayView, scales: &ArrayView, biases: Option<&ArrayView>,
    lhs_indices: Option<&ArrayView>, rhs_indices: Option<&ArrayView>, transpose: bool, group_size: i32,
    bits: i32, sorted_indices: bool, mode: &str, global_scale: Option<&ArrayView>, out: &mut ArrayView,
    stream: *mut c_void,
) -> Result<()> {
    let m = cmode(mode);
    check(sys::mlxq_gather_qmm(
        x.as_raw(), w.as_raw(), scales.as_raw(), opt(biases), opt(lhs_indices), opt(rhs_indices), transpose,
        group_size, bits, sorted_indices, m.as_ptr(), opt(global_scale), out.as_raw_mut(), stream,
    ))
}

/// The reference's `ffi::dequantize` (`dtype`: None = the reference
/// default), into `out`.
///
/// # Safety
/// As `quantized_matmul`.
pub unsafe fn dequantize(
    w: &ArrayView, scales: &ArrayView, biases: Option<&ArrayView>, group_size: i32, bits: i32, mode: &str,
    dtype: Option<Dtype>, out: &mut ArrayView, stream: *mut c_void,
) -> Result<()> {
    let m = cmode(mode);
    check(sys::mlxq_dequantize(
        w.as_raw(), scales.as_raw(), opt(biases), group_size, bits, m.as_ptr(), dtype.map_or(-1, |d| d as i32),
        out.as_raw_mut(), stream,
    ))
}

/// `mlx::core::quantize` into caller-allocated outputs (`biases_out` for
/// affine only).
///
/// # Safety
/// As `quantized_matmul`.
pub unsafe fn quantize(
    w: &ArrayView, group_size: i32, bits: i32, mode: &str, wq_out: &mut ArrayView, scales_out: &mut ArrayView,
    biases_out: Option<&mut ArrayView>, stream: *mut c_void,
) -> Result<()> {
    let m = cmode(mode);
    let b = biases_out.map_or(std::ptr::null_mut(), |v| v.as_raw_mut());
    check(sys::mlxq_quantize(
        w.as_raw(), group_size, bits, m.as_ptr(), wq_out.as_raw_mut(), scales_out.as_raw_mut(), b, stream,
    ))
}

/// The twelve arrays of one fused decode-MoE call, in the reference's order.
pub struct MoeArrays<'a> {
    pub x: &'a ArrayView,
    pub indices: &'a ArrayView,
    pub gate_w: &'a ArrayView,
    pub gate_s: &'a ArrayView,
    pub gate_b: &'a ArrayView,
    pub up_w: &'a ArrayView,
    pub up_s: &'a ArrayView,
    pub up_b: &'a ArrayView,
    pub down_w: &'a ArrayView,
    pub down_s: &'a ArrayView,
    pub down_b: &'a ArrayView,
    pub scores: &'a ArrayView,
}

/// The reference's `fused_moe_expert_kernel` (SwiGLU experts).  `Err(
/// Unsupported)` for configurations without a kernel: the caller takes its
/// `gather_qmm` route, as it does for the reference's `Err`.
///
/// # Safety
/// As `quantized_matmul`.
pub unsafe fn fused_moe_expert_kernel(
    a: &MoeArrays, din: i32, dff: i32, k: i32, gu_bits: i32, d_bits: i32, group_size: i32, out: &mut ArrayView,
    stream: *mut c_void,
) -> Result<()> {
    check(sys::mlxq_fused_moe_expert(
        a.x.as_raw(), a.indices.as_raw(), a.gate_w.as_raw(), a.gate_s.as_raw(), a.gate_b.as_raw(),
        a.up_w.as_raw(), a.up_s.as_raw(), a.up_b.as_raw(), a.down_w.as_raw(), a.down_s.as_raw(),
        a.down_b.as_raw(), a.scores.as_raw(), din, dff, k, gu_bits, d_bits, group_size, out.as_raw_mut(), stream,
    ))
}

/// The reference's `fused_moe_geglu_kernel` (GeGLU experts).
///
/// # Safety
/// As `quantized_matmul`.
pub unsafe fn fused_moe_geglu_kernel(
    a: &MoeArrays, din: i32, dff: i32, k: i32, gu_bits: i32, d_bits: i32, group_size: i32, out: &mut ArrayView,
    stream: *mut c_void,
) -> Result<()> {
    check(sys::mlxq_fused_moe_geglu(
        a.x.as_raw(), a.indices.as_raw(), a.gate_w.as_raw(), a.gate_s.as_raw(), a.gate_b.as_raw(),
        a.up_w.as_raw(), a.up_s.as_raw(), a.up_b.as_raw(), a.down_w.as_raw(), a.down_s.as_raw(),
        a.down_b.as_raw(), a.scores.as_raw(), din, dff, k, gu_bits, d_bits, group_size, out.as_raw_mut(), stream,
    ))
}

/// Attention of one query token per sequence over a paged cache (`q`, `out`
/// `[B, query heads, width]`, pools `[pages, kv heads, page, width]`, `table`
/// `[B, n]` and `lengths` `[B]` int32).  `softcap` and `window` 0: none.
///
/// # Safety
/// The views must describe device memory that is valid for the call's work on `stream`.
pub unsafe fn paged_attention(
    q: &ArrayView, k_pool: &ArrayView, v_pool: &ArrayView, table: &ArrayView, lengths: &ArrayView,
    sinks: Option<&ArrayView>, scale: f32, softcap: f32, window: i32, out: &mut ArrayView, stream: *mut c_void,
) -> Result<()> {
    check(sys::mlxq_paged_attention(
        q.as_raw(), k_pool.as_raw(), v_pool.as_raw(), table.as_raw(), lengths.as_raw(), opt(sinks), scale, softcap,
        window, out.as_raw_mut(), stream,
    ))
}

/// The book of a paged cache: `table` `[rows, n]`, `lengths` `[rows]` and `refs`
/// `[pages]`, int32, updated in place by the functions below.
pub struct CacheBook<'a> {
    pub table: &'a ArrayView,
    pub lengths: &'a ArrayView,
    pub refs: &'a ArrayView,
}

/// Pages for `counts[r]` more tokens of every row; `granted[r]` is 0 for a row that they do not hold.
///
/// # Safety
/// As [`paged_attention`].
pub unsafe fn cache_reserve(
    book: &CacheBook, counts: &ArrayView, page: i32, granted: &mut ArrayView, stream: *mut c_void,
) -> Result<()> {
    check(sys::mlxq_cache_reserve(
        book.table.as_raw(), book.lengths.as_raw(), book.refs.as_raw(), counts.as_raw(), page, granted.as_raw_mut(),
        stream,
    ))
}

/// Writes tokens' keys and values `[T, kv heads, width]` to their rows' pages.
///
/// # Safety
/// As [`paged_attention`].
pub unsafe fn cache_append(
    k: &ArrayView, v: &ArrayView, k_pool: &ArrayView, v_pool: &ArrayView, table: &ArrayView, positions: &ArrayView,
    rows: &ArrayView, lengths: Option<&ArrayView>, stream: *mut c_void,
) -> Result<()> {
    check(sys::mlxq_cache_append(
        k.as_raw(), v.as_raw(), k_pool.as_raw(), v_pool.as_raw(), table.as_raw(), positions.as_raw(), rows.as_raw(),
        opt(lengths), stream,
    ))
}

fn raw_list(pools: &[&ArrayView]) -> Vec<*const sys::mlxq_array> {
    pools.iter().map(|p| p.as_raw()).collect()
}

/// Makes the empty rows `dst[i]` copies of rows `src[i]`, sharing full pages.
///
/// # Safety
/// As [`paged_attention`].
pub unsafe fn cache_fork(
    pools: &[&ArrayView], book: &CacheBook, src: &ArrayView, dst: &ArrayView, granted: &mut ArrayView,
    stream: *mut c_void,
) -> Result<()> {
    let p = raw_list(pools);
    check(sys::mlxq_cache_fork(
        p.len() as i32, p.as_ptr(), book.table.as_raw(), book.lengths.as_raw(), book.refs.as_raw(), src.as_raw(),
        dst.as_raw(), granted.as_raw_mut(), stream,
    ))
}

/// Empties rows.
///
/// # Safety
/// As [`paged_attention`].
pub unsafe fn cache_free(book: &CacheBook, rows: &ArrayView, page: i32, stream: *mut c_void) -> Result<()> {
    check(sys::mlxq_cache_free(
        book.table.as_raw(), book.lengths.as_raw(), book.refs.as_raw(), rows.as_raw(), page, stream,
    ))
}

/// Moves the held pages to the front of every pool; `live` `[1]` gets their number.
///
/// # Safety
/// As [`paged_attention`].
pub unsafe fn cache_compact(
    pools: &[&ArrayView], book: &CacheBook, live: &mut ArrayView, stream: *mut c_void,
) -> Result<()> {
    let p = raw_list(pools);
    check(sys::mlxq_cache_compact(
        p.len() as i32, p.as_ptr(), book.table.as_raw(), book.lengths.as_raw(), book.refs.as_raw(), live.as_raw_mut(),
        stream,
    ))
}

/// `h = x + scale * gate * post(y)`, `n = pre(h)`; `n` exactly where `pre_weight` is.
///
/// # Safety
/// As [`paged_attention`].
pub unsafe fn residual_norm(
    x: &ArrayView, y: &ArrayView, post_weight: Option<&ArrayView>, gate: Option<&ArrayView>, scale: f32,
    pre_weight: Option<&ArrayView>, eps: f32, weight_offset: f32, h: &mut ArrayView, n: Option<&mut ArrayView>,
    stream: *mut c_void,
) -> Result<()> {
    let n = n.map_or(std::ptr::null_mut(), |v| v.as_raw_mut());
    check(sys::mlxq_residual_norm(
        x.as_raw(), y.as_raw(), opt(post_weight), opt(gate), scale, opt(pre_weight), eps, weight_offset,
        h.as_raw_mut(), n, stream,
    ))
}

/// Log probabilities of `tokens` `[T, m]`, the entropy `[T]` and, where `top` is
/// given, the most probable tokens (log probabilities and ids, `[T, k]`).
///
/// # Safety
/// As [`paged_attention`].
pub unsafe fn token_logprobs(
    logits: &ArrayView, tokens: &ArrayView, scale: f32, logprobs: &mut ArrayView, entropy: &mut ArrayView,
    top: Option<(i32, &mut ArrayView, &mut ArrayView)>, stream: *mut c_void,
) -> Result<()> {
    let (k, lp, ids) = match top {
        Some((k, lp, ids)) => (k, lp.as_raw_mut(), ids.as_raw_mut()),
        None => (0, std::ptr::null_mut(), std::ptr::null_mut()),
    };
    check(sys::mlxq_token_logprobs(
        logits.as_raw(), tokens.as_raw(), k, scale, logprobs.as_raw_mut(), entropy.as_raw_mut(), lp, ids, stream,
    ))
}

/// Attention of several new tokens per sequence: rows `starts[b] .. starts[b + 1]`
/// of `q` `[T, query heads, width]` are the last of `lengths[b]` tokens.  Rows of
/// no sequence are left as they were in `out`.
///
/// # Safety
/// As [`paged_attention`].
pub unsafe fn paged_attention_chunk(
    q: &ArrayView, k_pool: &ArrayView, v_pool: &ArrayView, table: &ArrayView, lengths: &ArrayView, starts: &ArrayView,
    sinks: Option<&ArrayView>, scale: f32, softcap: f32, window: i32, out: &mut ArrayView, stream: *mut c_void,
) -> Result<()> {
    check(sys::mlxq_paged_attention_chunk(
        q.as_raw(), k_pool.as_raw(), v_pool.as_raw(), table.as_raw(), lengths.as_raw(), starts.as_raw(), opt(sinks),
        scale, softcap, window, out.as_raw_mut(), stream,
    ))
}

/// How [`rotary_frequencies`] scales for contexts `factor` times `original` tokens
/// (`mlxq_rotary_scaling` in `include/mlxq.h`).
#[derive(Clone, Copy, Debug, PartialEq)]
pub enum RotaryScaling {
    Plain,
    Linear { factor: f64 },
    Base { factor: f64 },
    Bands { factor: f64, original: f64, low: f64, high: f64 },
    Ramp { factor: f64, original: f64, low: f64, high: f64 },
}

/// The `dims / 2` frequencies of [`rotary`] and its factor, worked out on the host.
pub fn rotary_frequencies(dims: i32, base: f64, scaling: RotaryScaling) -> Result<(Vec<f32>, f32)> {
    let (kind, factor, original, low, high) = match scaling {
        RotaryScaling::Plain => (0, 1.0, 0.0, 0.0, 0.0),
        RotaryScaling::Linear { factor } => (1, factor, 0.0, 0.0, 0.0),
        RotaryScaling::Base { factor } => (2, factor, 0.0, 0.0, 0.0),
        RotaryScaling::Bands { factor, original, low, high } => (3, factor, original, low, high),
        RotaryScaling::Ramp { factor, original, low, high } => (4, factor, original, low, high),
    };
    let mut inv_freq = vec![0f32; (dims.max(2) / 2) as usize];
    let mut by = 1f32;
    // SAFETY: writes dims / 2 floats and one to host memory.
    check(unsafe {
        sys::mlxq_rotary_frequencies(dims, base, kind, factor, original, low, high, inv_freq.as_mut_ptr(), &mut by)
    })?;
    Ok((inv_freq, by))
}

/// Rotates the first `2 n` elements of the heads of `x` `[T, heads, width]` by
/// `positions` `[T]` times `inv_freq` `[n]` (device memory), times `factor`.
///
/// # Safety
/// As [`paged_attention`].
pub unsafe fn rotary(
    x: &ArrayView, positions: &ArrayView, inv_freq: &ArrayView, interleaved: bool, factor: f32, out: &mut ArrayView,
    stream: *mut c_void,
) -> Result<()> {
    check(sys::mlxq_rotary(
        x.as_raw(), positions.as_raw(), inv_freq.as_raw(), interleaved, factor, out.as_raw_mut(), stream,
    ))
}

/// [`rotary`] of `q` to `out` and of `k` on its way into the pages, with `v` beside
/// it: [`cache_append`] of the rotated keys in one launch.
///
/// # Safety
/// As [`paged_attention`].
pub unsafe fn rotary_append(
    q: &ArrayView, k: &ArrayView, v: &ArrayView, k_pool: &ArrayView, v_pool: &ArrayView, table: &ArrayView,
    positions: &ArrayView, rows: &ArrayView, lengths: Option<&ArrayView>, inv_freq: &ArrayView, interleaved: bool,
    factor: f32, out: &mut ArrayView, stream: *mut c_void,
) -> Result<()> {
    check(sys::mlxq_rotary_append(
        q.as_raw(), k.as_raw(), v.as_raw(), k_pool.as_raw(), v_pool.as_raw(), table.as_raw(), positions.as_raw(),
        rows.as_raw(), opt(lengths), inv_freq.as_raw(), interleaved, factor, out.as_raw_mut(), stream,
    ))
}

/// The parts of [`adjust_logits`]; what is `None` is left out.
#[derive(Default)]
pub struct LogitAdjustments<'a> {
    pub history: Option<&'a ArrayView>,
    pub history_lengths: Option<&'a ArrayView>,
    pub prompts: Option<&'a ArrayView>,
    pub repetition: Option<&'a ArrayView>,
    pub presence: Option<&'a ArrayView>,
    pub frequency: Option<&'a ArrayView>,
    pub bias_ids: Option<&'a ArrayView>,
    pub bias: Option<&'a ArrayView>,
    pub mask: Option<&'a ArrayView>,
}

/// Penalties, biases and a grammar's mask on `logits` `[T, V]`.
///
/// # Safety
/// As [`paged_attention`].
pub unsafe fn adjust_logits(
    logits: &ArrayView, a: &LogitAdjustments, out: &mut ArrayView, stream: *mut c_void,
) -> Result<()> {
    check(sys::mlxq_adjust_logits(
        logits.as_raw(), opt(a.history), opt(a.history_lengths), opt(a.prompts), opt(a.repetition), opt(a.presence),
        opt(a.frequency), opt(a.bias_ids), opt(a.bias), opt(a.mask), out.as_raw_mut(), stream,
    ))
}

/// Grows `stream`'s workspace (so later calls, e.g. under graph capture,
/// need not allocate).
pub fn workspace_reserve(bytes: usize, stream: *mut c_void) -> Result<()> {
    // SAFETY: allocates on the current device; `stream` is a hipStream_t.
    check(unsafe { sys::mlxq_workspace_reserve(bytes, stream) })
}

/// The reference's `get_cache_memory`: bytes the library's workspaces hold.
pub fn get_cache_memory() -> usize {
    // SAFETY: reads the library's bookkeeping only.
    unsafe { sys::mlxq_get_cache_memory() }
}

/// The reference's `clear_memory_cache`: synchronizes and frees every
/// workspace (graphs captured earlier must not be replayed afterwards).
pub fn clear_memory_cache() -> Result<()> {
    // SAFETY: synchronizes the devices that hold a workspace first.
    check(unsafe { sys::mlxq_clear_cache() })
}

/// Re-reads the `MLXQ_*` environment switches (A/B measurement only).
pub fn reload_options() {
    // SAFETY: swaps an immutable snapshot.
    unsafe { sys::mlxq_reload_options() }
}

#[cfg(test)]
mod tests {
    use super::*;

    fn view(dtype: Dtype, shape: &[i64]) -> ArrayView {
        // shape queries never dereference the data pointer
        unsafe { ArrayView::contiguous(std::ptr::null_mut(), dtype, shape) }
    }

    #[test]
    fn version_names_the_target() {
        assert!(version().contains("gfx950"));
    }

    #[test]
    fn shape_query_follows_the_reference() {
        let x = view(Dtype::Bfloat16, &[3, 4096]);
        let w = view(Dtype::Uint32, &[14336, 512]);
        let s = view(Dtype::Bfloat16, &[14336, 64]);
        let spec = quantized_matmul_shape(&x, &w, &s, Some(&s), true, 64, 4, "affine").unwrap();
        assert_eq!(spec, OutSpec { shape: vec![3, 14336], dtype: Dtype::Bfloat16 });
    }

    #[test]
    fn argument_errors_carry_the_reference_text() {
        let x = view(Dtype::Bfloat16, &[3, 4096]);
        let w = view(Dtype::Uint32, &[14336, 512]);
        let s = view(Dtype::Bfloat16, &[14336, 64]);
        match quantized_matmul_shape(&x, &w, &s, None, true, 64, 4, "affine") {
            Err(Error::Invalid(m)) => assert!(m.contains("Biases must be provided")),
            other => panic!("{other:?}"),
        }
    }

    #[test]
    fn strides_default_to_row_major() {
        let v = view(Dtype::Float16, &[2, 3, 4]);
        assert_eq!(v.raw.strides[..3], [12, 4, 1]);
        assert_eq!(v.shape(), &[2, 3, 4]);
        assert_eq!(v.dtype(), Some(Dtype::Float16));
    }
}
