"""MLX-style quantized ops over torch device tensors, backed by ``libmlxq.so``.

Mirrors the reference operator interface (the MLX ops mlxcel binds through
``ffi::quantized_matmul`` / ``ffi::gather_qmm`` / ``ffi::dequantize`` /
``ffi::quantize_weights_*``; src/lib/mlxcel-core/src/lib.rs:1374-1416,
overlays/rocm/mlx/ops.cpp:4955-5008, 5454-5492, 5753-5805, 5841-5948): same
names, argument meaning, defaults and output shapes/dtypes.  Errors follow
MLX's Python binding: argument errors raise ``ValueError`` with the
reference's message; combinations this library does not implement raise
``NotImplementedError``.

Torch is used only for device memory and the current HIP stream; all
arithmetic happens in the HIP kernels.

Each wrapper hands its arguments to the native module first (csrc/pyext.cpp:
exact torch tensors on a HIP device, plain Python numbers); where that returns
None, or the module is missing or was built for another torch, the call takes
the ctypes binding below, which also reports the errors.
"""
from __future__ import annotations

import ctypes
import os
import warnings
from typing import Optional, Sequence

import torch

from . import _lib


class _ctypes_only:
    """Stands in for the native module: every call takes the ctypes binding."""
    quantized_matmul = quantized_matmul_multi = gather_qmm = staticmethod(lambda *a: None)
    dequantize = quantize = fused_moe = staticmethod(lambda *a: None)
    paged_attention = residual_norm = token_logprobs = staticmethod(lambda *a: None)
    cache_reserve = cache_append = cache_fork = cache_free = cache_compact = staticmethod(lambda *a: None)
    paged_attention_chunk = rotary = rotary_append = adjust_logits = staticmethod(lambda *a: None)


def _load_native():
    """The native module where it is there and was built for this torch."""
    if not os.path.exists(_lib.NATIVE_PATH):
        return _ctypes_only
    try:
        from . import _mlxq_native as native

        built_for = getattr(native, "torch_version", "(unknown)")
        if built_for == torch.__version__:
            return native
        why = f"it was built for torch {built_for}, this is {torch.__version__}"
    except ImportError as e:  # another torch or Python, or no libmlxq.so beside it
        why = str(e)
    warnings.warn(f"{_lib.NATIVE_PATH} is not used, calls go through ctypes: {why}")
    return _ctypes_only


_native = _load_native()

_TORCH_TO_MLXQ = {
    torch.bool: _lib.BOOL,
    torch.uint8: _lib.UINT8,
    torch.uint16: _lib.UINT16,
    torch.uint32: _lib.UINT32,
    torch.uint64: _lib.UINT64,
    torch.int8: _lib.INT8,
    torch.int16: _lib.INT16,
    torch.int32: _lib.INT32,
    torch.int64: _lib.INT64,
    torch.float16: _lib.FLOAT16,
    torch.float32: _lib.FLOAT32,
    torch.float64: _lib.FLOAT64,
    torch.bfloat16: _lib.BFLOAT16,
}
_MLXQ_TO_TORCH = {v: k for k, v in _TORCH_TO_MLXQ.items()}


class QuantizedOpError(RuntimeError):
    pass


def _arr(t: Optional[torch.Tensor]):
    if t is None:
        return None
    if t.dim() > _lib.MAX_DIMS:
        raise ValueError(f"[mlxq] at most {_lib.MAX_DIMS} dimensions are supported")
    a = _lib.MlxqArray()
    a.data = t.data_ptr() if t.numel() > 0 else None
    a.dtype = _TORCH_TO_MLXQ.get(t.dtype, -1)
    if a.dtype < 0:
        raise ValueError(f"[mlxq] unsupported tensor dtype {t.dtype}")
    a.ndim = t.dim()
    for i, (s, st) in enumerate(zip(t.shape, t.stride())):
        a.shape[i] = s
        a.strides[i] = st
    return ctypes.byref(a), a  # keep `a` alive with the reference


def _ref(pair):
    return None if pair is None else pair[0]


def _raise(status: int) -> None:
    msg = _lib.last_error()
    if status == _lib.EINVAL:
        raise ValueError(msg)
    if status == _lib.EUNSUPPORTED:
        raise NotImplementedError(msg)
    raise QuantizedOpError(f"status {status}: {msg}")


def _done(r):
    """The native module's result, or the error of its status code."""
    if type(r) is int:
        _raise(r)
    return r


def _stream(device: torch.device) -> ctypes.c_void_p:
    return ctypes.c_void_p(torch.cuda.current_stream(device).cuda_stream)


def _opt(v: Optional[int]) -> int:
    return -1 if v is None else int(v)


def _mode(mode: str) -> bytes:
    return mode.encode() if isinstance(mode, str) else bytes(mode)


def _empty(ndim, shape, dtype, device) -> torch.Tensor:
    return torch.empty(tuple(shape[: ndim.value]), dtype=_MLXQ_TO_TORCH[dtype.value], device=device)


def _device_of(x: torch.Tensor) -> torch.device:
    if x.device.type != "cuda":
        raise ValueError("[mlxq] tensors must live on a HIP device (torch 'cuda' device)")
    return x.device


def quantized_matmul(x: torch.Tensor, w: torch.Tensor, scales: torch.Tensor,
                     biases: Optional[torch.Tensor] = None, transpose: bool = True,
                     group_size: Optional[int] = None, bits: Optional[int] = None,
                     mode: str = "affine", *, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``x @ dequantize(w, scales, biases).T`` (``transpose=True``), as ``mx.quantized_matmul``."""
    r = _native.quantized_matmul(x, w, scales, biases, None, False, transpose, group_size, bits, mode, out)
    if r is not None:
        return _done(r)
    lib = _lib.load()
    ax, aw, as_, ab = _arr(x), _arr(w), _arr(scales), _arr(biases)
    gs, b = _opt(group_size), _opt(bits)
    if out is None:
        nd, sh, dt = ctypes.c_int32(), (ctypes.c_int64 * _lib.MAX_DIMS)(), ctypes.c_int32()
        st = lib.mlxq_quantized_matmul_shape(_ref(ax), _ref(aw), _ref(as_), _ref(ab), transpose, gs, b,
                                             _mode(mode), ctypes.byref(nd), sh, ctypes.byref(dt))
        if st:
            _raise(st)
        out = _empty(nd, sh, dt, _device_of(x))
    ao = _arr(out)
    dev = _device_of(x)
    with torch.cuda.device(dev):
        st = lib.mlxq_quantized_matmul(_ref(ax), _ref(aw), _ref(as_), _ref(ab), transpose, gs, b,
                                       _mode(mode), _ref(ao), _stream(dev))
    if st:
        _raise(st)
    return out


def quantized_linear(x: torch.Tensor, w: torch.Tensor, scales: torch.Tensor, biases: Optional[torch.Tensor] = None,
                     linear_bias: Optional[torch.Tensor] = None, group_size: Optional[int] = None,
                     bits: Optional[int] = None, mode: str = "affine", *,
                     out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """The reference's ``quantized_linear_forward``: ``x @ W^T + linear_bias``."""
    r = _native.quantized_matmul(x, w, scales, biases, linear_bias, True, True, group_size, bits, mode, out)
    if r is not None:
        return _done(r)
    lib = _lib.load()
    gs, b = _opt(group_size), _opt(bits)
    ax, aw, as_, ab, alb = _arr(x), _arr(w), _arr(scales), _arr(biases), _arr(linear_bias)
    if out is None:
        nd, sh, dt = ctypes.c_int32(), (ctypes.c_int64 * _lib.MAX_DIMS)(), ctypes.c_int32()
        st = lib.mlxq_quantized_matmul_shape(_ref(ax), _ref(aw), _ref(as_), _ref(ab), True, gs, b, _mode(mode),
                                             ctypes.byref(nd), sh, ctypes.byref(dt))
        if st:
            _raise(st)
        out = _empty(nd, sh, dt, _device_of(x))
    ao = _arr(out)
    dev = _device_of(x)
    with torch.cuda.device(dev):
        st = lib.mlxq_quantized_linear(_ref(ax), _ref(aw), _ref(as_), _ref(ab), _ref(alb), gs, b, _mode(mode),
                                       _ref(ao), _stream(dev))
    if st:
        _raise(st)
    return out


def quantized_matmul_matches_dense_gemm(x: torch.Tensor, w: torch.Tensor, scales: torch.Tensor,
                                        biases: Optional[torch.Tensor] = None, group_size: int = 64,
                                        bits: int = 4) -> bool:
    """The reference's predicate of the same name (no device work)."""
    lib = _lib.load()
    return bool(lib.mlxq_quantized_matmul_matches_dense_gemm(_ref(_arr(x)), _ref(_arr(w)), _ref(_arr(scales)),
                                                             _ref(_arr(biases)), group_size, bits))


def quantized_matmul_multi(x: torch.Tensor, ws: Sequence[torch.Tensor], scales: Sequence[torch.Tensor],
                           biases: Optional[Sequence[Optional[torch.Tensor]]] = None,
                           group_size: Optional[int] = None, bits: Optional[int] = None, mode: str = "affine", *,
                           out: Optional[Sequence[torch.Tensor]] = None) -> list:
    """``[quantized_matmul(x, w_i, s_i, b_i) for i]`` (transpose=True) in one
    call; at decode sizes one launch that reads x once (q/k/v, gate/up)."""
    r = _native.quantized_matmul_multi(x, ws, scales, biases, group_size, bits, mode, out)
    if r is not None:
        return _done(r)
    lib = _lib.load()
    n = len(ws)
    gs, b = _opt(group_size), _opt(bits)
    dev = _device_of(x)
    if out is None:
        out = []
        for w_, s_, b_ in zip(ws, scales, biases if biases is not None else [None] * n):
            nd, sh, dt = ctypes.c_int32(), (ctypes.c_int64 * _lib.MAX_DIMS)(), ctypes.c_int32()
            st = lib.mlxq_quantized_matmul_shape(_ref(_arr(x)), _ref(_arr(w_)), _ref(_arr(s_)), _ref(_arr(b_)),
                                                 True, gs, b, _mode(mode), ctypes.byref(nd), sh, ctypes.byref(dt))
            if st:
                _raise(st)
            out.append(_empty(nd, sh, dt, dev))
    P = ctypes.POINTER(_lib.MlxqArray)

    def ptrs(ts):  # (pointer array, the structs it points to: kept alive by the caller)
        structs = [_arr(t)[1] if t is not None else None for t in ts]
        return (P * n)(*[ctypes.pointer(v) if v is not None else None for v in structs]), structs

    pw, kw = ptrs(ws)
    ps, ks = ptrs(scales)
    po, ko = ptrs(out)
    pb, kb = ptrs(biases) if biases is not None else (None, None)
    ax = _arr(x)
    with torch.cuda.device(dev):
        st = lib.mlxq_quantized_matmul_multi(_ref(ax), n, pw, ps, pb, gs, b, _mode(mode), po, _stream(dev))
    if st:
        _raise(st)
    return list(out)


def gather_qmm(x: torch.Tensor, w: torch.Tensor, scales: torch.Tensor,
               biases: Optional[torch.Tensor] = None, lhs_indices: Optional[torch.Tensor] = None,
               rhs_indices: Optional[torch.Tensor] = None, transpose: bool = True,
               group_size: Optional[int] = None, bits: Optional[int] = None, mode: str = "affine",
               sorted_indices: bool = False, *, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``out[i] = x[lhs[i]] @ dequantize(w[rhs[i]]).T``, as ``mx.gather_qmm``."""
    r = _native.gather_qmm(x, w, scales, biases, lhs_indices, rhs_indices, transpose, group_size, bits, mode,
                           sorted_indices, out)
    if r is not None:
        return _done(r)
    lib = _lib.load()
    ax, aw, as_, ab = _arr(x), _arr(w), _arr(scales), _arr(biases)
    al, ar = _arr(lhs_indices), _arr(rhs_indices)
    gs, b = _opt(group_size), _opt(bits)
    if out is None:
        nd, sh, dt = ctypes.c_int32(), (ctypes.c_int64 * _lib.MAX_DIMS)(), ctypes.c_int32()
        st = lib.mlxq_gather_qmm_shape(_ref(ax), _ref(aw), _ref(as_), _ref(ab), _ref(al), _ref(ar), transpose,
                                       gs, b, _mode(mode), ctypes.byref(nd), sh, ctypes.byref(dt))
        if st:
            _raise(st)
        out = _empty(nd, sh, dt, _device_of(x))
    ao = _arr(out)
    dev = _device_of(x)
    with torch.cuda.device(dev):
        st = lib.mlxq_gather_qmm(_ref(ax), _ref(aw), _ref(as_), _ref(ab), _ref(al), _ref(ar), transpose, gs, b,
                                 sorted_indices, _mode(mode), None, _ref(ao), _stream(dev))
    if st:
        _raise(st)
    return out


def _default_gs_bits(mode: str, group_size, bits):
    d = {"affine": (64, 4), "mxfp4": (32, 4), "nvfp4": (16, 4), "mxfp8": (32, 8)}.get(mode, (64, 4))
    return (d[0] if group_size is None else group_size), (d[1] if bits is None else bits)


def dequantize(w: torch.Tensor, scales: torch.Tensor, biases: Optional[torch.Tensor] = None,
               group_size: Optional[int] = None, bits: Optional[int] = None, mode: str = "affine",
               dtype: Optional[torch.dtype] = None, *, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``mx.dequantize``; affine output is bit-exact to MLX's CPU graph."""
    lib = _lib.load()
    gs, b = _default_gs_bits(mode, group_size, bits)
    dcode = -1 if dtype is None else _TORCH_TO_MLXQ[dtype]
    if out is None:
        if b <= 0:
            raise ValueError(f"[dequantize] Invalid value for bits: {b}")
        if w.dim() < 1:
            raise ValueError("[dequantize] The matrix to be dequantized must have at least 2 dimension "
                             f"but it has only {w.dim()}.")
        shape = list(w.shape)
        shape[-1] = shape[-1] * 32 // b
        odt = dtype if dtype is not None else (scales.dtype if mode == "affine" else torch.bfloat16)
        out = torch.empty(shape, dtype=odt, device=_device_of(w))
    r = _native.dequantize(w, scales, biases, gs, b, mode, dcode, out)
    if r is not None:
        return _done(r)
    aw, as_, ab, ao = _arr(w), _arr(scales), _arr(biases), _arr(out)
    dev = _device_of(w)
    with torch.cuda.device(dev):
        st = lib.mlxq_dequantize(_ref(aw), _ref(as_), _ref(ab), gs, b, _mode(mode), dcode, _ref(ao),
                                 _stream(dev))
    if st:
        _raise(st)
    return out


def quantize(w: torch.Tensor, group_size: Optional[int] = None, bits: Optional[int] = None,
             mode: str = "affine") -> Sequence[torch.Tensor]:
    """``mx.quantize``: returns ``(wq, scales, biases)`` (affine) or ``(wq, scales)``."""
    lib = _lib.load()
    gs, b = _default_gs_bits(mode, group_size, bits)
    dev = _device_of(w)
    if w.dim() < 2 or gs <= 0 or b <= 0 or w.shape[-1] % gs or (w.shape[-1] * b) % 32:
        # let the library produce the reference's message
        wq = scales = biases = w.new_empty((0,))
    else:
        qshape = list(w.shape)
        qshape[-1] = w.shape[-1] * b // 32
        sshape = list(w.shape)
        sshape[-1] = w.shape[-1] // gs
        wq = torch.empty(qshape, dtype=torch.uint32, device=dev)
        if mode == "affine":
            scales = torch.empty(sshape, dtype=w.dtype, device=dev)
            biases = torch.empty(sshape, dtype=w.dtype, device=dev)
        else:
            scales = torch.empty(sshape, dtype=torch.uint8, device=dev)
            biases = None
    r = _native.quantize(w, group_size, bits, mode, wq, scales, biases)
    if r is not None:
        if r is not True:
            _raise(r)
        return (wq, scales, biases) if mode == "affine" else (wq, scales)
    aw, aq, as_, ab = _arr(w), _arr(wq), _arr(scales), _arr(biases)
    with torch.cuda.device(dev):
        st = lib.mlxq_quantize(_ref(aw), _opt(group_size), _opt(bits), _mode(mode), _ref(aq), _ref(as_),
                               _ref(ab), _stream(dev))
    if st:
        _raise(st)
    return (wq, scales, biases) if mode == "affine" else (wq, scales)


def _fused_moe(fn_name: str, x, indices, gate_w, gate_s, gate_b, up_w, up_s, up_b, down_w, down_s, down_b,
               scores, din: int, dff: int, k: int, gu_bits: int, d_bits: int, group_size: int,
               out: Optional[torch.Tensor]) -> torch.Tensor:
    r = _native.fused_moe(fn_name == "mlxq_fused_moe_geglu", x, indices, gate_w, gate_s, gate_b, up_w, up_s, up_b,
                          down_w, down_s, down_b, scores, din, dff, k, gu_bits, d_bits, group_size, out)
    if r is not None:
        return _done(r)
    lib = _lib.load()
    dev = _device_of(x)
    if out is None:
        out = torch.empty(max(int(din), 0), dtype=x.dtype, device=dev)
    arrs = [_arr(t) for t in (x, indices, gate_w, gate_s, gate_b, up_w, up_s, up_b, down_w, down_s, down_b,
                              scores, out)]
    with torch.cuda.device(dev):
        st = getattr(lib, fn_name)(*[_ref(a) for a in arrs[:12]], din, dff, k, gu_bits, d_bits, group_size,
                                   _ref(arrs[12]), _stream(dev))
    if st:
        _raise(st)
    return out


def fused_moe_expert(x, indices, gate_w, gate_s, gate_b, up_w, up_s, up_b, down_w, down_s, down_b, scores,
                     din: int, dff: int, k: int, gu_bits: int, d_bits: int, group_size: int, *,
                     out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """The reference's ``fused_moe_expert_kernel`` (SwiGLU experts, one decode
    token): ``sum_j scores[j] * down_e(silu(gate_e(x)) * up_e(x))`` over
    ``e = indices[j]``; returns a ``(din,)`` tensor in x's dtype."""
    return _fused_moe("mlxq_fused_moe_expert", x, indices, gate_w, gate_s, gate_b, up_w, up_s, up_b, down_w,
                      down_s, down_b, scores, din, dff, k, gu_bits, d_bits, group_size, out)


def fused_moe_geglu(x, indices, gate_w, gate_s, gate_b, up_w, up_s, up_b, down_w, down_s, down_b, scores,
                    din: int, dff: int, k: int, gu_bits: int, d_bits: int, group_size: int, *,
                    out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """The reference's ``fused_moe_geglu_kernel`` (GeGLU experts: tanh-approximated
    GELU of the gate times up)."""
    return _fused_moe("mlxq_fused_moe_geglu", x, indices, gate_w, gate_s, gate_b, up_w, up_s, up_b, down_w,
                      down_s, down_b, scores, din, dff, k, gu_bits, d_bits, group_size, out)


def _together(*tensors: Optional[torch.Tensor]) -> torch.device:
    """The device of the call's tensors, which must be one HIP device."""
    dev = _device_of(tensors[0])
    for t in tensors[1:]:
        if t is not None and t.device != dev:
            raise ValueError(f"[mlxq] tensors must live on one device but are on {dev} and {t.device}")
    return dev


def _run(name: str, dev: torch.device, *args) -> None:
    """One C call on the device's current stream: tensors (or None) and numbers."""
    arrs = [_arr(a) if isinstance(a, torch.Tensor) else None for a in args]
    with torch.cuda.device(dev):
        st = getattr(_lib.load(), name)(*[a if r is None else _ref(r) for a, r in zip(args, arrs)], _stream(dev))
    if st:
        _raise(st)


def _pointers(pools: Sequence[torch.Tensor]):
    """An array of pointers to the pools' structs (kept alive by it)."""
    P = ctypes.POINTER(_lib.MlxqArray)
    return (P * len(pools))(*[ctypes.pointer(_arr(t)[1]) for t in pools])


def paged_attention(q: torch.Tensor, k_pool: torch.Tensor, v_pool: torch.Tensor, table: torch.Tensor,
                    lengths: torch.Tensor, *, window: int = 0, softcap: float = 0.0,
                    sinks: Optional[torch.Tensor] = None, scale: Optional[float] = None,
                    out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Attention of one query token per sequence over a paged cache.

    ``q`` (B, query heads, width); ``k_pool``, ``v_pool`` (pages, kv heads, page,
    width) of q's type (bfloat16, float16, float32) with a contiguous last axis;
    ``table`` (B, n) and ``lengths`` (B) int32: sequence b's tokens are
    ``lengths[b]`` ones on the pages ``table[b]``, the last of them the query's own.  A
    length of 0 gives zeros.  ``scale`` is ``width ** -0.5`` by default;
    ``softcap`` c > 0 makes a score s ``c tanh(s / c)``; ``window`` w > 0 keeps
    the last w tokens; ``sinks`` (query heads) float32 join each head's softmax
    sum."""
    if scale is None:
        scale = q.shape[-1] ** -0.5 if q.dim() and q.shape[-1] else 1.0
    r = _native.paged_attention(q, k_pool, v_pool, table, lengths, sinks, scale, softcap, window, out)
    if r is not None:
        return _done(r)
    dev = _together(q, k_pool, v_pool, table, lengths, sinks, out)
    if out is None:
        out = torch.empty(q.shape, dtype=q.dtype, device=dev)
    _run("mlxq_paged_attention", dev, q, k_pool, v_pool, table, lengths, sinks, scale, softcap, window, out)
    return out


def cache_reserve(table: torch.Tensor, lengths: torch.Tensor, refs: torch.Tensor, counts: torch.Tensor,
                  page: int) -> torch.Tensor:
    """Pages for ``counts[r]`` more tokens of every row, the lowest free pages
    first; updates ``table`` (rows, n), ``lengths`` (rows) and ``refs`` (pages),
    all int32, in place.  Returns int32 flags: 0 for a row that the free pages or
    the table do not hold, which stays as it was."""
    r = _native.cache_reserve(table, lengths, refs, counts, page)
    if r is not None:
        return _done(r)
    dev = _together(table, lengths, refs, counts)
    granted = torch.empty(counts.shape, dtype=torch.int32, device=dev)
    _run("mlxq_cache_reserve", dev, table, lengths, refs, counts, int(page), granted)
    return granted


def cache_append(k: torch.Tensor, v: torch.Tensor, k_pool: torch.Tensor, v_pool: torch.Tensor, table: torch.Tensor,
                 positions: torch.Tensor, rows: torch.Tensor, *, lengths: Optional[torch.Tensor] = None) -> None:
    """Writes the keys and values of tokens, ``k`` and ``v`` (T, kv heads,
    width), to position ``positions[t]`` of sequence ``rows[t]`` (int32).  Where a
    reservation may have been refused pass ``lengths``: tokens at or past their
    sequence's length are then left out, like those whose row, position or page
    is out of range."""
    r = _native.cache_append(k, v, k_pool, v_pool, table, positions, rows, lengths)
    if r is not None:
        return None if r is True else _raise(r)
    dev = _together(k, v, k_pool, v_pool, table, positions, rows, lengths)
    _run("mlxq_cache_append", dev, k, v, k_pool, v_pool, table, positions, rows, lengths)


def cache_fork(pools: Sequence[torch.Tensor], table: torch.Tensor, lengths: torch.Tensor, refs: torch.Tensor,
               src: torch.Tensor, dst: torch.Tensor) -> torch.Tensor:
    """Makes each empty row ``dst[i]`` a copy of row ``src[i]``: full pages are
    shared, a part-full last page is copied in every pool to the lowest free
    page.  Returns int32 flags: 0 for a pair that could not be served."""
    pools = list(pools)
    r = _native.cache_fork(pools, table, lengths, refs, src, dst)
    if r is not None:
        return _done(r)
    dev = _together(table, lengths, refs, src, dst, *pools)
    granted = torch.empty(src.shape, dtype=torch.int32, device=dev)
    _run("mlxq_cache_fork", dev, len(pools), _pointers(pools), table, lengths, refs, src, dst, granted)
    return granted


def cache_free(table: torch.Tensor, lengths: torch.Tensor, refs: torch.Tensor, rows: torch.Tensor,
               page: int) -> None:
    """Empties the sequences ``rows``: their pages lose a reference, their
    lengths become 0."""
    r = _native.cache_free(table, lengths, refs, rows, page)
    if r is not None:
        return None if r is True else _raise(r)
    _run("mlxq_cache_free", _together(table, lengths, refs, rows), table, lengths, refs, rows, int(page))


def cache_compact(pools: Sequence[torch.Tensor], table: torch.Tensor, lengths: torch.Tensor,
                  refs: torch.Tensor) -> torch.Tensor:
    """Moves the held pages to the front of every pool, with their refs and the
    table's entries; returns their number, int32 (1)."""
    pools = list(pools)
    r = _native.cache_compact(pools, table, lengths, refs)
    if r is not None:
        return _done(r)
    dev = _together(table, lengths, refs, *pools)
    live = torch.empty(1, dtype=torch.int32, device=dev)
    _run("mlxq_cache_compact", dev, len(pools), _pointers(pools), table, lengths, refs, live)
    return live


def residual_norm(x: torch.Tensor, y: torch.Tensor, *, post_weight: Optional[torch.Tensor] = None,
                  gate: Optional[torch.Tensor] = None, scale: float = 1.0,
                  pre_weight: Optional[torch.Tensor] = None, eps: float = 1e-6, weight_offset: float = 0.0):
    """The residual update of a block and the norms on its sides:
    ``h = x + scale * gate * rms(y, post_weight)``, ``n = rms(h, pre_weight)`` with
    ``rms(t, w) = t * rsqrt(mean(t**2) + eps) * (w + weight_offset)``.  Returns
    ``(h, n)``; without ``post_weight`` y is taken as it is, without ``pre_weight`` n
    is None.  ``gate`` broadcasts over the last axis, all rows, or the rows of a
    batch entry."""
    r = _native.residual_norm(x, y, post_weight, gate, scale, pre_weight, eps, weight_offset)
    if r is not None:
        return _done(r)
    dev = _together(x, y, post_weight, gate, pre_weight)
    h = torch.empty(x.shape, dtype=x.dtype, device=dev)
    n = None if pre_weight is None else torch.empty_like(h)
    _run("mlxq_residual_norm", dev, x, y, post_weight, gate, scale, pre_weight, eps, weight_offset, h, n)
    return h, n


def token_logprobs(logits: torch.Tensor, tokens: torch.Tensor, *, top_k: int = 0, scale: float = 1.0):
    """Of each row of ``logits`` (T, V), under ``log_softmax(scale * logits)``:
    the log probabilities of ``tokens`` (T, m) int32, the entropy (T), and the
    ``top_k`` <= 64 most probable tokens with theirs (equal logits by the lower
    token).  Returns ``(logprobs, entropy, top_logprobs, top_ids)``, float32 and
    int32, the last two None for ``top_k`` 0."""
    r = _native.token_logprobs(logits, tokens, top_k, scale)
    if r is not None:
        return _done(r)
    dev = _together(logits, tokens)
    rows = logits.shape[0] if logits.dim() else 0
    f32 = dict(dtype=torch.float32, device=dev)
    out = [torch.empty(tokens.shape, **f32), torch.empty(rows, **f32), None, None]
    if top_k > 0:
        out[2] = torch.empty(rows, top_k, **f32)
        out[3] = torch.empty(rows, top_k, dtype=torch.int32, device=dev)
    _run("mlxq_token_logprobs", dev, logits, tokens, int(top_k), scale, *out)
    return tuple(out)


def paged_attention_chunk(q: torch.Tensor, k_pool: torch.Tensor, v_pool: torch.Tensor, table: torch.Tensor,
                          lengths: torch.Tensor, starts: torch.Tensor, *, window: int = 0, softcap: float = 0.0,
                          sinks: Optional[torch.Tensor] = None, scale: Optional[float] = None,
                          out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``paged_attention`` for several new tokens per sequence: rows ``starts[b]``
    to ``starts[b + 1] - 1`` of ``q`` (T, query heads, width) are the last of
    sequence b's ``lengths[b]`` tokens, whose keys and values are in the pages
    already; each sees the keys up to its own (the last ``window`` of them).
    ``starts`` (B + 1) int32, ascending.  Rows of no sequence are left as they were
    in ``out`` (undefined in a new one), which may be q; tokens before a sequence's
    first give zeros."""
    if scale is None:
        scale = q.shape[-1] ** -0.5 if q.dim() and q.shape[-1] else 1.0
    r = _native.paged_attention_chunk(q, k_pool, v_pool, table, lengths, starts, sinks, scale, softcap, window, out)
    if r is not None:
        return _done(r)
    dev = _together(q, k_pool, v_pool, table, lengths, starts, sinks, out)
    if out is None:
        out = torch.empty(q.shape, dtype=q.dtype, device=dev)
    _run("mlxq_paged_attention_chunk", dev, q, k_pool, v_pool, table, lengths, starts, sinks, scale, softcap, window, out)
    return out


_ROTARY_SCALING = {None: 0, "linear": 1, "base": 2, "bands": 3, "ramp": 4}


def rotary_frequencies(dims: int, base: float = 10000.0, *, scaling: Optional[str] = None, factor: float = 1.0,
                       original: float = 0.0, low: Optional[float] = None, high: Optional[float] = None, device="cuda"):
    """``(inv_freq, attention_factor)`` for ``rotary``: ``base ** (-2 i / dims)``
    for the ``dims / 2`` pairs, float32, and a float.  ``scaling`` for contexts
    ``factor`` times the ``original`` tokens: "linear" divides all by factor;
    "base" grows the base by ``factor ** (dims / (dims - 2))``; "bands" divides
    those that turn at most ``low`` (1) times over the original tokens, keeps
    those that turn ``high`` (4) times or more and takes the ones between in
    proportion; "ramp" is that in proportion to the pair's number, between
    ``high`` (32) and ``low`` (1) turns, with an attention factor of
    ``0.1 ln(factor) + 1``."""
    if scaling not in _ROTARY_SCALING:
        raise ValueError(f"[rotary_frequencies] scaling must be one of {list(_ROTARY_SCALING)} but is {scaling!r}.")
    low = 1.0 if low is None else low
    high = (32.0 if scaling == "ramp" else 4.0) if high is None else high
    inv, by = (ctypes.c_float * max(int(dims) // 2, 1))(), ctypes.c_float()
    st = _lib.load().mlxq_rotary_frequencies(int(dims), base, _ROTARY_SCALING[scaling], factor, original, low, high, inv,
                                             ctypes.byref(by))
    if st:
        _raise(st)
    return torch.tensor(list(inv), dtype=torch.float32, device=device), by.value


def rotary(x: torch.Tensor, positions: torch.Tensor, inv_freq: torch.Tensor, *, interleaved: bool = False,
           factor: float = 1.0, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Rotates the first ``2 n`` elements of every head of ``x`` (T, heads, width)
    by its token's position: pair i, elements ``(i, n + i)`` or, interleaved,
    ``(2 i, 2 i + 1)``, by ``positions[t] * inv_freq[i]``, times ``factor``; the rest
    is copied.  ``positions`` (T) int32, ``inv_freq`` (n) float32
    (``rotary_frequencies``).  ``-positions`` give the gradient for x.  ``out`` may be
    x."""
    r = _native.rotary(x, positions, inv_freq, interleaved, factor, out)
    if r is not None:
        return _done(r)
    dev = _together(x, positions, inv_freq, out)
    if out is None:
        out = torch.empty(x.shape, dtype=x.dtype, device=dev)
    _run("mlxq_rotary", dev, x, positions, inv_freq, bool(interleaved), factor, out)
    return out


def rotary_append(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, k_pool: torch.Tensor, v_pool: torch.Tensor,
                  table: torch.Tensor, positions: torch.Tensor, rows: torch.Tensor, inv_freq: torch.Tensor, *,
                  lengths: Optional[torch.Tensor] = None, interleaved: bool = False, factor: float = 1.0,
                  out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``rotary`` of ``q`` (T, query heads, width), which it returns, and of ``k`` (T,
    kv heads, width) on its way into the pages, with ``v`` beside it:
    ``cache_append`` of the rotated keys in one launch.  Tokens that have no place
    in the cache (a row, position or page out of range, at or past ``lengths``) are
    left out of it; their queries are rotated all the same."""
    r = _native.rotary_append(q, k, v, k_pool, v_pool, table, positions, rows, lengths, inv_freq, interleaved, factor, out)
    if r is not None:
        return _done(r)
    dev = _together(q, k, v, k_pool, v_pool, table, positions, rows, lengths, inv_freq, out)
    if out is None:
        out = torch.empty(q.shape, dtype=q.dtype, device=dev)
    _run("mlxq_rotary_append", dev, q, k, v, k_pool, v_pool, table, positions, rows, lengths, inv_freq, bool(interleaved),
         factor, out)
    return out


def adjust_logits(logits: torch.Tensor, *, history: Optional[torch.Tensor] = None,
                  history_lengths: Optional[torch.Tensor] = None, prompts: Optional[torch.Tensor] = None,
                  repetition: Optional[torch.Tensor] = None, presence: Optional[torch.Tensor] = None,
                  frequency: Optional[torch.Tensor] = None, bias_ids: Optional[torch.Tensor] = None,
                  bias: Optional[torch.Tensor] = None, mask: Optional[torch.Tensor] = None,
                  out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Penalties, biases and a grammar's mask on ``logits`` (T, V), in this order:
    tokens among the first ``history_lengths[t]`` of ``history`` (T, n) are divided
    by ``repetition[t]`` where positive and multiplied by it elsewhere; those at
    place ``prompts[t]`` or later lose ``presence[t] + frequency[t] * times``;
    ``bias[t, j]`` is added to token ``bias_ids[t, j]`` (of equal ids the last
    counts); tokens whose bit of ``mask`` (T, ceil(V / 32)) is 0 (bit ``v % 32`` of
    word ``v // 32``) become -inf.  int32 and float32; steps that are not given are
    left out.  ``out`` may be ``logits``."""
    args = (history, history_lengths, prompts, repetition, presence, frequency, bias_ids, bias, mask)
    r = _native.adjust_logits(logits, *args, out)
    if r is not None:
        return _done(r)
    dev = _together(logits, *args, out)
    if out is None:
        out = torch.empty(logits.shape, dtype=logits.dtype, device=dev)
    _run("mlxq_adjust_logits", dev, logits, *args, out)
    return out


def workspace_reserve(nbytes: int, device: Optional[torch.device] = None) -> None:
    """Grow the current stream's workspace to ``nbytes`` before a HIP-graph
    capture (a call under capture never allocates; it fails instead)."""
    lib = _lib.load()
    dev = torch.device("cuda", torch.cuda.current_device()) if device is None else device
    with torch.cuda.device(dev):
        st = lib.mlxq_workspace_reserve(int(nbytes), _stream(dev))
    if st:
        _raise(st)


def get_cache_memory() -> int:
    """Device bytes held by the library's workspaces (``get_cache_memory``)."""
    return int(_lib.load().mlxq_get_cache_memory())


def clear_cache() -> None:
    """Free every workspace after synchronizing (``clear_memory_cache``)."""
    st = _lib.load().mlxq_clear_cache()
    if st:
        _raise(st)
