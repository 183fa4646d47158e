"""Host-side mirror of the reference's operator interface, over the C ABI.

  fp8_mm(a, b, as, bs, c)      src/mix_gemm/hip_mix_gemm_kernel.cpp:508-516
  int8_mm / bf16_mm            the stubs in src/gemm/sm80_gemm_kernel.cu:4-22
  int8_mm_block                int8 operands with the 128-block scales of fp8_mm (no counterpart in the reference)
  matrix_transpose(in, out)    src/transpose/transpose.cu:60-74
  gemm(...)                    GEMM_kernel_v*<In, Out> of include/gemm.h:25-66
  quantize(x, ...)             the Q_A / Q_B of README.md:1 (the reference has no quantiser)
  layer_norm(x, ...), layer_norm_backward(dy, x, ...), checkpoint(x, ...), restore(q, scales, ...), weight_gradient(dy, q, scales, ...)
                               training around the products: a layer norm, activations kept in 8 bits, the gradients computed
                               from them (no counterpart in the reference)
  rms_norm(x, ...), rms_norm_backward(dy, h, ...), group_rows(ids, ...), add_adapters(y, x, ...), add_adapters_backward(dy, x, ...),
  log_probabilities(logits, tokens, ...), log_probabilities_backward(logits, tokens, ...)
                               beside the products of a language model: its norm, low-rank adapters of many requests at once, what its
                               last product says of tokens (no counterpart in the reference)

Tensors are torch CUDA(HIP) tensors; only their data pointers and the current
stream cross the boundary."""
import ctypes as C
import os
import warnings

import torch

from .lib import check, load_library, load_torch_extension

DT_F32, DT_BF16, DT_F16, DT_I8, DT_F8E4M3, DT_I32 = 0, 1, 2, 3, 4, 5
B_KN, B_NK = 0, 1
SCALE_PER_MATRIX, SCALE_BLOCK128 = 1, 2
LAYOUT_K_CONTIGUOUS, LAYOUT_REFERENCE = 0, 1
QUANT_PER_MATRIX, QUANT_BLOCK_1x128, QUANT_BLOCK_128x128 = 1, 2, 3

_TORCH_DT = {
    torch.float32: DT_F32, torch.bfloat16: DT_BF16, torch.float16: DT_F16, torch.int8: DT_I8,
    torch.int32: DT_I32, torch.float8_e4m3fn: DT_F8E4M3,
}


_native_module = None
_NATIVE_ENTRIES = ("ops_gemm", "ops_scaled_gemm", "ops_transpose", "ops_quantize", "ops_layer_norm", "ops_layer_norm_backward", "ops_checkpoint",
                   "ops_restore", "ops_weight_gradient", "ops_rms_norm", "ops_rms_norm_backward", "ops_group_rows", "ops_add_adapters",
                   "ops_add_adapters_backward", "ops_log_probabilities", "ops_log_probabilities_backward")


def _native():
    """The extension module that reads the tensors and calls the library in one step, or False: QGEMM_LIBRARY names a library
    it is not linked to, or it cannot be used (not built for this Python, or built before it had what is called here), which
    is said once.  The functions below then go through ctypes, to the same entries.
    (Host time of quantise and multiply, 1 x 2048 x 1024: 11.6 + 8.4 us through ctypes, 4.1 + 3.8 us through the module.)"""
    global _native_module
    if _native_module is None:
        _native_module = False
        if not os.environ.get("QGEMM_LIBRARY"):
            load_library()                      # (its absence is an error, not a reason to go another way)
            try:
                module = load_torch_extension()
                missing = [f for f in _NATIVE_ENTRIES if not hasattr(module, f)]
                if missing:
                    raise ImportError(f"{getattr(module, '__file__', 'qgemm_python')} has no {', '.join(missing)}: build it again")
                _native_module = module
            except ImportError as e:
                warnings.warn(f"calls go through ctypes, at twice the host time: {e}", RuntimeWarning, stacklevel=3)
    return _native_module


def _dt(t, fp8_as_uint8=False):
    if t.dtype == torch.uint8 and fp8_as_uint8:
        return DT_F8E4M3
    try:
        return _TORCH_DT[t.dtype]
    except KeyError:
        raise TypeError(f"unsupported tensor dtype {t.dtype}") from None


def _stream():
    return C.c_void_p(torch.cuda.current_stream().cuda_stream)


def _need_gpu(*ts):
    for t in ts:
        if t is not None and not t.is_cuda:
            raise ValueError("qgemm operates on device tensors only (there is no CPU path)")


def set_option(key, value):
    check(load_library().qgemm_set_option(key.encode(), int(value)))


def force_config(name=None):
    """Pin the row `name` of the variant tables for the GEMM calls that follow (None: back to the heuristic)."""
    check(load_library().qgemm_force_config(name.encode() if name else None))


def variant_names(in_dtype, scale_mode=0, k_major=0):
    """Names of the rows of the family that serves (in_dtype, scale_mode, k_major); arguments as for plan()."""
    lib = load_library()
    out = []
    for i in range(lib.qgemm_variant_count(in_dtype, scale_mode, k_major)):
        buf = C.create_string_buffer(64)
        check(lib.qgemm_variant_name(in_dtype, scale_mode, k_major, i, buf, 64))
        out.append(buf.value.decode())
    return out


def plan(in_dtype, scale_mode, k_major, M, N, K, out_dtype=DT_BF16):
    """Name of the kernel configuration the library would choose (no launch, no device needed)."""
    buf = C.create_string_buffer(128)
    check(load_library().qgemm_plan_out(in_dtype, out_dtype, scale_mode, k_major, M, N, K, buf, 128))
    return buf.value.decode()


def last_config():
    buf = C.create_string_buffer(128)
    check(load_library().qgemm_last_config(buf, 128))
    return buf.value.decode()


def last_any_kernel():
    """Which kernel the last product with last_config() "strided_any_shape" ran."""
    buf = C.create_string_buffer(64)
    check(load_library().qgemm_last_any_kernel(buf, 64))
    return buf.value.decode()


def selftest_layouts():
    """-> (ok, report)"""
    buf = C.create_string_buffer(4096)
    st = load_library().qgemm_selftest_layouts(buf, 4096)
    return st == 0, buf.value.decode()


def tile_map(wg, tiles_m, tiles_n, group_m):
    tm, tn = C.c_uint32(), C.c_uint32()
    check(load_library().qgemm_tile_map(wg, tiles_m, tiles_n, group_m, C.byref(tm), C.byref(tn)))
    return tm.value, tn.value


def gemm(A, B, C_out, layout_b="nk", M=None, N=None, K=None, ldA=None, ldB=None, ldC=None):
    """C[M,N] = A[M,K] @ B.  layout_b "kn": B is [K,N] (GEMM_kernel_v1..v5);
    "nk": B is [N,K] (GEMM_kernel_v3_1 / v4_1)."""
    native = _native()
    if native and (layout_b == "nk" or layout_b == "kn"):
        st = native.ops_gemm(A, B, C_out, layout_b == "kn", M, N, K, ldA, ldB, ldC)
        if st == 0:
            return C_out
        if st > 0:
            check(st)
    _need_gpu(A, B, C_out)
    lb = {"kn": B_KN, "nk": B_NK}[layout_b]
    M = A.shape[0] if M is None else M
    K = A.shape[1] if K is None else K
    N = (B.shape[1] if lb == B_KN else B.shape[0]) if N is None else N
    ldA = A.stride(0) if ldA is None else ldA
    ldB = B.stride(0) if ldB is None else ldB
    ldC = C_out.stride(0) if ldC is None else ldC
    check(load_library().qgemm_gemm(_dt(A, True), _dt(C_out), lb, A.data_ptr(), ldA, B.data_ptr(), ldB,
                                    C_out.data_ptr(), ldC, M, N, K, _stream()))
    return C_out


def scaled_gemm(A, B, a_scale, b_scale, C_out, M, N, K, scale_mode, layout=LAYOUT_K_CONTIGUOUS, split_k=0,
                in_dtype=None, ldC=None):
    native = _native()
    if native:
        st = native.ops_scaled_gemm(A, B, a_scale, b_scale, C_out, M, N, K, scale_mode, layout, split_k, in_dtype, ldC)
        if st == 0:
            return C_out
        if st > 0:
            check(st)
    _need_gpu(A, B, a_scale, b_scale, C_out)
    in_dtype = _dt(A, True) if in_dtype is None else in_dtype
    ldC = C_out.stride(0) if ldC is None else ldC
    check(load_library().qgemm_scaled_gemm(
        in_dtype, _dt(C_out), scale_mode, layout, A.data_ptr(), B.data_ptr(),
        a_scale.data_ptr() if a_scale is not None else None, b_scale.data_ptr() if b_scale is not None else None,
        C_out.data_ptr(), ldC, M, N, K, split_k, _stream()))
    return C_out


def _need_fp8(*ts):
    """The kernels decode OCP e4m3 (torch.float8_e4m3fn, or its raw codes as uint8).  The gfx942 "fnuz" encoding
    the reference's fp8_mm names has another bias and another NaN: refuse it rather than compute with every value
    doubled."""
    for t in ts:
        if t.dtype not in (torch.float8_e4m3fn, torch.uint8):
            raise TypeError(f"fp8 operands must be torch.float8_e4m3fn (OCP e4m3) or uint8 codes, got {t.dtype}")


def _need_out(c, m, n):
    if c.dim() != 2 or tuple(c.shape) != (m, n) or c.stride(1) != 1 or (m > 1 and c.stride(0) < n):
        raise ValueError(f"c must be [{m}, {n}] with unit inner stride, got shape {tuple(c.shape)} strides {c.stride()}")


def fp8_mm(a, b, a_scale, b_scale, c):
    """The reference entry (hip_mix_gemm_kernel.cpp:425-439, 508-516):
      a        [m, k] fp8, column-major  (storage a[i + j*m])
      b        [n, k] fp8, column-major  (storage b[n + k*n_total], i.e. [k, n] row-major)
      a_scale  [m, k/128] fp32, column-major;  b_scale [n/128, k/128] fp32, column-major
      c        [m, n] bf16, row-major
    m = a.size(0), n = b.size(0), k = a.size(1) exactly as the reference reads them."""
    m, n, k = a.size(0), b.size(0), a.size(1)
    _need_fp8(a, b)
    _need_out(c, m, n)
    return scaled_gemm(a, b, a_scale, b_scale, c, m, n, k, SCALE_BLOCK128, LAYOUT_REFERENCE, in_dtype=DT_F8E4M3,
                       ldC=c.stride(0))


def int8_mm(a, b, a_scale, b_scale, c, split_k=0):
    """Per-matrix scaled int8 GEMM: a [m,k] int8, b [n,k] int8 (both K-contiguous), one fp32 scale each,
    c [m,n] fp32 / bf16 / fp16, or int32 for the raw accumulators."""
    m, k = a.shape
    n = b.shape[0]
    if a.dtype != torch.int8 or b.dtype != torch.int8:
        raise TypeError(f"int8_mm takes int8 operands, got {a.dtype} and {b.dtype}")
    _need_out(c, m, n)
    return scaled_gemm(a, b, a_scale, b_scale, c, m, n, k, SCALE_PER_MATRIX, split_k=split_k, in_dtype=DT_I8,
                       ldC=c.stride(0))


def int8_mm_block(a, b, a_scale, b_scale, c, split_k=0):
    """int8 GEMM with 128-block scales, the int8 twin of fp8_mm's arithmetic (hip_mix_gemm_kernel.cpp:231-244) on
    K-contiguous operands: a [m,k] int8, b [n,k] int8, a_scale [m, ceil(k/128)] and b_scale [ceil(n/128), ceil(k/128)]
    fp32 row-major, c [m,n] fp32 / bf16 / fp16.  Every 128-wide K block's exact int32 partial is folded into an fp32
    sum with a_scale[m, kb] * b_scale[n // 128, kb]."""
    m, k = a.shape
    n = b.shape[0]
    if a.dtype != torch.int8 or b.dtype != torch.int8:
        raise TypeError(f"int8_mm_block takes int8 operands, got {a.dtype} and {b.dtype}")
    _need_out(c, m, n)
    return scaled_gemm(a, b, a_scale, b_scale, c, m, n, k, SCALE_BLOCK128, split_k=split_k, in_dtype=DT_I8, ldC=c.stride(0))


def bf16_mm(a, b, c):
    """a [m,k], b [n,k] (K-contiguous), c [m,n]; plain GEMM with fp32 accumulation."""
    return gemm(a, b, c, "nk")


def matrix_transpose(idata, odata, M=None, N=None):
    """odata[N, M] = idata[M, N]^T for 1-, 2- or 4-byte elements."""
    native = _native()
    if native:
        st = native.ops_transpose(idata, odata, M, N)
        if st == 0:
            return odata
        if st > 0:
            check(st)
    _need_gpu(idata, odata)
    M = idata.shape[0] if M is None else M
    N = idata.shape[1] if N is None else N
    check(load_library().qgemm_transpose(idata.element_size(), idata.data_ptr(), odata.data_ptr(), M, N, _stream()))
    return odata


def quantize(x, out_dtype=torch.float8_e4m3fn, mode=QUANT_PER_MATRIX, rows_contiguous_scales=False):
    """q, scales = quantise(x): x [rows, cols] fp32 / bf16 / fp16 (row stride free), q [rows, cols] int8 or
    fp8-e4m3.  scales: [1] for QUANT_PER_MATRIX; [rows, ceil(cols/128)] for QUANT_BLOCK_1x128 (or its
    transpose, storage [ceil(cols/128), rows], with rows_contiguous_scales: the a_scale arrangement of the
    reference layout); [ceil(rows/128), ceil(cols/128)] for QUANT_BLOCK_128x128 (transposed likewise)."""
    native = _native()
    if native:
        st, q, scales = native.ops_quantize(x, out_dtype, mode, rows_contiguous_scales)
        if st == 0:
            return q, scales
        if st > 0:
            check(st)
    _need_gpu(x)
    assert x.dim() == 2 and x.stride(1) == 1
    rows, cols = x.shape
    q = torch.empty((rows, cols), dtype=out_dtype, device=x.device)
    if mode == QUANT_PER_MATRIX:
        scales = torch.empty(1, dtype=torch.float32, device=x.device)
        rs = cs = 0
    else:
        nbr = rows if mode == QUANT_BLOCK_1x128 else (rows + 127) // 128
        nbc = (cols + 127) // 128
        if rows_contiguous_scales:
            scales = torch.empty((nbc, nbr), dtype=torch.float32, device=x.device)
            rs, cs = 1, nbr
        else:
            scales = torch.empty((nbr, nbc), dtype=torch.float32, device=x.device)
            rs, cs = nbc, 1
    ld = x.stride(0) if rows > 1 else max(cols, 1)          # the stride of a single row is arbitrary
    check(load_library().qgemm_quantize(_dt(x), _dt(q, True), mode, x.data_ptr(), ld, rows, cols, q.data_ptr(),
                                        cols, scales.data_ptr(), rs, cs, _stream()))
    return q, scales


# ---- layer norm, activations in 8 bits, weight gradients.  Tensors of any number of dimensions are rows of their last one; the rows have to lie
# evenly spaced, their elements side by side.
_FLOATS = (torch.float32, torch.bfloat16, torch.float16)
_CODES = (torch.int8, torch.float8_e4m3fn)


def _rows_of(t, name):
    """(rows, cols, ld) of a tensor as rows of its last dimension."""
    _need_gpu(t)
    if t.dim() < 1 or t.shape[-1] < 1:
        raise ValueError(f"{name} must have a last dimension of one or more elements, got shape {tuple(t.shape)}")
    cols, rows, step, even = t.shape[-1], 1, 0, t.shape[-1] == 1 or t.stride(-1) == 1
    for n, stride in reversed(list(zip(t.shape[:-1], t.stride()[:-1]))):
        if n == 1:
            continue
        if rows == 1:
            step = stride
        even = even and (rows == 1 or stride == rows * step)
        rows *= n
    if rows == 0:
        return 0, cols, cols
    ld = step if rows > 1 else cols
    if not even or ld < cols:
        raise ValueError(f"{name} must be rows of contiguous elements, evenly spaced, got shape {tuple(t.shape)} strides {t.stride()}")
    return rows, cols, ld


def _need_type(t, types, name):
    dtype = t if isinstance(t, torch.dtype) else t.dtype
    if dtype not in types:
        raise TypeError(f"{name} must be one of {', '.join(str(x) for x in types)}, got {dtype}")


def _need_floats(t, n, name):
    _need_gpu(t)
    _need_type(t, (torch.float32,), name)
    if t.numel() != n or not t.is_contiguous():
        raise ValueError(f"{name} must hold {n} contiguous values, got shape {tuple(t.shape)}")
    return t.data_ptr()


def _parameters(weight, bias, cols):
    """(type, pointer, pointer) of a layer norm's parameters, one of which or both may be None."""
    if weight is None:
        if bias is not None:
            raise ValueError("a bias needs a weight")
        return DT_F32, None, None
    for t, name in ((weight, "weight"), (bias, "bias")):
        if t is None:
            continue
        _need_gpu(t)
        _need_type(t, _FLOATS, name)
        if t.numel() != cols or not t.is_contiguous() or t.dtype != weight.dtype:
            raise ValueError(f"{name} must hold {cols} contiguous values of {weight.dtype}, got {t.dtype} {tuple(t.shape)}")
    return _dt(weight), weight.data_ptr(), None if bias is None else bias.data_ptr()


def _scales_like(t, cols):
    return torch.empty((*t.shape[:-1], -(-cols // 128)), dtype=torch.float32, device=t.device)


def layer_norm(x, weight=None, bias=None, eps=1e-5, out_dtype=None, keep=None):
    """y, mean, rstd = layer norm of the rows of x [..., cols], fp32 / bf16 / fp16: y = xhat * weight + bias with xhat = (x - mean) * rstd,
    rstd = 1 / sqrt(var + eps); weight and bias [cols], fp32 / bf16 / fp16, or None.  y has x's type, or out_dtype; mean and rstd are fp32.
    keep (torch.int8 or torch.float8_e4m3fn): y, mean, rstd, q, scales, where q and scales are xhat in 8 bits as checkpoint() gives it: what
    layer_norm_backward and weight_gradient need of this layer's activations."""
    native = _native()
    if native:
        st, *out = native.ops_layer_norm(x, weight, bias, eps, out_dtype, keep)
        if st == 0:
            return tuple(out) if keep is not None else tuple(out[:3])
        if st > 0:
            check(st)
    rows, cols, ld = _rows_of(x, "x")
    out_dtype = x.dtype if out_dtype is None else out_dtype
    _need_type(x, _FLOATS, "x")
    _need_type(out_dtype, _FLOATS, "out_dtype")
    params, w, b = _parameters(weight, bias, cols)
    y = torch.empty(x.shape, dtype=out_dtype, device=x.device)
    mean, rstd = (torch.empty(x.shape[:-1], dtype=torch.float32, device=x.device) for _ in range(2))
    q = scales = None
    if keep is not None:
        _need_type(keep, _CODES, "keep")
        q, scales = torch.empty(x.shape, dtype=keep, device=x.device), _scales_like(x, cols)
    check(load_library().qgemm_layer_norm(
        _dt(x), _dt(y), params, DT_I8 if q is None else _dt(q), x.data_ptr(), ld, w, b, eps, y.data_ptr(), cols, mean.data_ptr(), rstd.data_ptr(),
        None if q is None else q.data_ptr(), cols, None if q is None else scales.data_ptr(), rows, cols, _stream()))
    return (y, mean, rstd) if keep is None else (y, mean, rstd, q, scales)


def layer_norm_backward(dy, x, mean, rstd, weight=None, scales=None, bias=True, out_dtype=None):
    """dx, dweight, dbias of layer_norm: dy [..., cols]; x is the norm's input, with its mean and rstd, or the codes q that
    layer_norm(..., keep=...) gave, with their scales (mean may be None then).  dx has dy's type, or out_dtype; dweight and dbias have weight's, and
    are None where weight is (dbias also with bias=False)."""
    native = _native()
    if native:
        st, *out = native.ops_layer_norm_backward(dy, x, mean, rstd, weight, scales, bias, out_dtype)
        if st == 0:
            return tuple(out)
        if st > 0:
            check(st)
    rows, cols, lddy = _rows_of(dy, "dy")
    xrows, xcols, ldx = _rows_of(x, "x")
    if (rows, cols) != (xrows, xcols):
        raise ValueError(f"dy and x must have the same rows, got {tuple(dy.shape)} and {tuple(x.shape)}")
    out_dtype = dy.dtype if out_dtype is None else out_dtype
    _need_type(dy, _FLOATS, "dy")
    _need_type(out_dtype, _FLOATS, "out_dtype")
    _need_type(x, _FLOATS + _CODES, "x")
    params, w, _ = _parameters(weight, None, cols)
    if x.dtype in _CODES:
        if scales is None:
            raise ValueError("codes need their scales")
        s, m = _need_floats(scales, rows * -(-cols // 128), "scales"), None
    else:
        if mean is None or scales is not None:
            raise ValueError("x that is not in 8 bits needs its mean, and has no scales")
        s, m = None, _need_floats(mean, rows, "mean")
    r = _need_floats(rstd, rows, "rstd")
    dx = torch.empty(dy.shape, dtype=out_dtype, device=dy.device)
    dw = None if weight is None else torch.empty_like(weight)
    db = None if weight is None or not bias else torch.empty_like(weight)
    check(load_library().qgemm_layer_norm_backward(
        _dt(dy), _dt(x), _dt(dx), params, dy.data_ptr(), lddy, x.data_ptr(), ldx, s, m, r, w, dx.data_ptr(), cols,
        None if dw is None else dw.data_ptr(), None if db is None else db.data_ptr(), rows, cols, _stream()))
    return dx, dw, db


def checkpoint(x, dtype=torch.int8):
    """q, scales = an activation x [..., cols], fp32 / bf16 / fp16, in 8 bits for the backward pass: codes (torch.int8 or torch.float8_e4m3fn) and
    one power of two for the 128 columns of a block, scales [..., ceil(cols/128)].  q * scale is exact in bf16
    (float8_e4m3fn: under scales of 2^-124 and more)."""
    native = _native()
    if native:
        st, q, scales = native.ops_checkpoint(x, dtype)
        if st == 0:
            return q, scales
        if st > 0:
            check(st)
    rows, cols, ld = _rows_of(x, "x")
    _need_type(x, _FLOATS, "x")
    _need_type(dtype, _CODES, "dtype")
    q, scales = torch.empty(x.shape, dtype=dtype, device=x.device), _scales_like(x, cols)
    check(load_library().qgemm_checkpoint(_dt(x), _dt(q), x.data_ptr(), ld, rows, cols, q.data_ptr(), cols, scales.data_ptr(), _stream()))
    return q, scales


def restore(q, scales, dtype=torch.bfloat16):
    """The values that codes of checkpoint(), layer_norm(..., keep=...) or quantize(x, ..., QUANT_BLOCK_1x128) stand for."""
    native = _native()
    if native:
        st, x = native.ops_restore(q, scales, dtype)
        if st == 0:
            return x
        if st > 0:
            check(st)
    rows, cols, ld = _rows_of(q, "q")
    _need_type(q, _CODES, "q")
    _need_type(dtype, _FLOATS, "dtype")
    s = _need_floats(scales, rows * -(-cols // 128), "scales")
    x = torch.empty(q.shape, dtype=dtype, device=q.device)
    check(load_library().qgemm_restore(_dt(q), _dt(x), q.data_ptr(), ld, s, rows, cols, x.data_ptr(), cols, _stream()))
    return x


def weight_gradient(dy, q, scales, weight=None, bias=None, out_dtype=torch.float32):
    """dw [n, cols], db [n] (fp32) = the gradients of a linear layer z = v W^T + c: dw = dy^T v, db = the sums of dy over its rows.  dy [..., n] bf16 or fp16;
    v is the layer's input in 8 bits, q [..., cols] and its scales.  With weight (and bias) q holds a layer norm's xhat, and
    v = xhat * weight + bias is meant."""
    native = _native()
    if native:
        st, dw, db = native.ops_weight_gradient(dy, q, scales, weight, bias, out_dtype)
        if st == 0:
            return dw, db
        if st > 0:
            check(st)
    rows, n, lddy = _rows_of(dy, "dy")
    qrows, cols, ldq = _rows_of(q, "q")
    if rows != qrows:
        raise ValueError(f"dy and q must have the same rows, got {tuple(dy.shape)} and {tuple(q.shape)}")
    _need_type(dy, _FLOATS[1:], "dy")
    _need_type(q, _CODES, "q")
    _need_type(out_dtype, _FLOATS, "out_dtype")
    params, w, b = _parameters(weight, bias, cols)
    s = _need_floats(scales, rows * -(-cols // 128), "scales")
    dw, db = torch.empty((n, cols), dtype=out_dtype, device=dy.device), torch.empty(n, dtype=torch.float32, device=dy.device)
    check(load_library().qgemm_weight_gradient(_dt(dy), _dt(q), _dt(dw), params, dy.data_ptr(), lddy, q.data_ptr(), ldq, s, w, b, dw.data_ptr(), cols,
                                               db.data_ptr(), rows, n, cols, _stream()))
    return dw, db


# ---- beside the products of a language model.  Tensors are rows of their last dimension, as above; all of them on the current device.
def _need_here(*ts):
    _need_gpu(*ts)
    here = torch.cuda.current_device()
    for t in ts:
        if t is not None and t.device.index != here:
            raise ValueError(f"tensors must be on the current device, cuda:{here}, got one on {t.device}")


def _weight(weight, cols):
    """(type, pointer) of a norm's weight, which may be None."""
    params, w, _ = _parameters(weight, None, cols)
    return params, w


def _like(t, other, name, dtypes=None):
    """ld of a tensor that has to have the rows of `other`, (rows, cols)."""
    rows, cols, ld = _rows_of(t, name)
    if (rows, cols) != other:
        raise ValueError(f"{name} must be {other[0]} rows of {other[1]}, got shape {tuple(t.shape)}")
    if dtypes is not None:
        _need_type(t, dtypes, name)
    return ld


def rms_norm(x, weight=None, eps=1e-6, residual=None, out_dtype=None, codes=None, store_y=True):
    """y, h, rstd = root-mean-square norm of the rows of x [..., cols], fp32 / bf16 / fp16: y = h * rstd * weight, rstd = 1 / sqrt(mean h^2 + eps), h = x, or with a
    residual (x's shape) h = x + residual in the residual's type, the residual stream's next value; the norm is that of what h stores.  weight [cols] or
    None.  y has x's type, or out_dtype; rstd is fp32.
    codes (torch.int8 or torch.float8_e4m3fn): y, h, rstd, q, scales, where q and scales are y in 8 bits, as quantize(y, codes, QUANT_BLOCK_1x128) of the fp32 y
    gives it: an operand of the block-scaled products.  store_y=False: y is None, and only its codes are written."""
    native = _native()
    if native:
        st, *out = native.ops_rms_norm(x, weight, eps, residual, out_dtype, codes, store_y)
        if st == 0:
            return tuple(out) if codes is not None else tuple(out[:3])
        if st > 0:
            check(st)
    _need_here(x, weight, residual)
    rows, cols, ld = _rows_of(x, "x")
    out_dtype = x.dtype if out_dtype is None else out_dtype
    _need_type(x, _FLOATS, "x")
    _need_type(out_dtype, _FLOATS, "out_dtype")
    params, w = _weight(weight, cols)
    if not store_y and codes is None:
        raise ValueError("nothing is asked for: neither y nor codes")
    h, ldr = x, 0
    if residual is not None:
        ldr = _like(residual, (rows, cols), "residual", _FLOATS)
        h = torch.empty(x.shape, dtype=residual.dtype, device=x.device)
    y = torch.empty(x.shape, dtype=out_dtype, device=x.device) if store_y else None
    rstd = torch.empty(x.shape[:-1], dtype=torch.float32, device=x.device)
    q = scales = None
    if codes is not None:
        _need_type(codes, _CODES, "codes")
        q, scales = torch.empty(x.shape, dtype=codes, device=x.device), _scales_like(x, cols)
    at = lambda t: None if t is None else t.data_ptr()  # noqa: E731
    check(load_library().qgemm_rms_norm(
        _dt(x), _dt(h), _TORCH_DT[out_dtype], params, DT_I8 if q is None else _dt(q), x.data_ptr(), ld, at(residual), ldr, w, eps,
        None if residual is None else h.data_ptr(), cols, at(y), cols, rstd.data_ptr(), at(q), cols, at(scales), rows, cols, _stream()))
    return (y, h, rstd) if codes is None else (y, h, rstd, q, scales)


def rms_norm_backward(dy, h, rstd, weight=None, dh=None, out_dtype=None):
    """dx, dweight of rms_norm: dy [..., cols], h and rstd as rms_norm gave them; dh: the gradient that arrives along the residual stream (of h), which is added: dx is
    then the gradient of x and of the residual.  dx has dy's type, or out_dtype; dweight has weight's, and is None where weight is."""
    native = _native()
    if native:
        st, *out = native.ops_rms_norm_backward(dy, h, rstd, weight, dh, out_dtype)
        if st == 0:
            return tuple(out)
        if st > 0:
            check(st)
    _need_here(dy, h, rstd, weight, dh)
    rows, cols, lddy = _rows_of(dy, "dy")
    out_dtype = dy.dtype if out_dtype is None else out_dtype
    _need_type(dy, _FLOATS, "dy")
    _need_type(out_dtype, _FLOATS, "out_dtype")
    ldh = _like(h, (rows, cols), "h", _FLOATS)
    lddh = 0 if dh is None else _like(dh, (rows, cols), "dh", _FLOATS)
    params, w = _weight(weight, cols)
    r = _need_floats(rstd, rows, "rstd")
    dx = torch.empty(dy.shape, dtype=out_dtype, device=dy.device)
    dw = None if weight is None else torch.empty_like(weight)
    check(load_library().qgemm_rms_norm_backward(
        _dt(dy), _dt(h), DT_F32 if dh is None else _dt(dh), _dt(dx), params, dy.data_ptr(), lddy, h.data_ptr(), ldh, r, w, None if dh is None else dh.data_ptr(), lddh,
        dx.data_ptr(), cols, None if dw is None else dw.data_ptr(), rows, cols, _stream()))
    return dx, dw


class RowGroups:
    """Rows grouped by their adapters: what group_rows() gives and the adapters' products take.  `words` is the library's own."""
    __slots__ = ("rows", "adapters", "words")

    def __init__(self, rows, adapters, words):
        self.rows, self.adapters, self.words = rows, adapters, words


def group_rows(ids, adapters):
    """RowGroups of the rows whose adapters are ids [rows], int32 or int64 on the device: 0 .. adapters - 1, any other number means none.  Made once, it serves every
    add_adapters and add_adapters_backward whose rows have these adapters."""
    native = _native()
    if native:
        st, words = native.ops_group_rows(ids, adapters)
        if st == 0:
            return RowGroups(ids.numel(), adapters, words)
        if st > 0:
            check(st)
    _need_here(ids)
    _need_type(ids, (torch.int32, torch.int64), "ids")
    if not ids.is_contiguous():
        raise ValueError(f"ids must be contiguous, got strides {ids.stride()}")
    rows, n = ids.numel(), C.c_size_t()
    check(load_library().qgemm_group_rows_words(rows, _size(adapters, "adapters"), C.byref(n)))
    words = torch.empty(n.value, dtype=torch.int32, device=ids.device)
    check(load_library().qgemm_group_rows(ids.element_size(), ids.data_ptr(), rows, adapters, words.data_ptr(), _stream()))
    return RowGroups(rows, adapters, words)


def _size(n, name):
    if n < 0:
        raise ValueError(f"{name} must not be negative, got {n}")
    return n


def _adapters(x, A, B, groups, scaling):
    """rows, k, ldx, rank, n and the pointer of the scaling, of operands that fit together."""
    if not isinstance(groups, RowGroups):
        raise TypeError(f"groups must be what group_rows() gives, got {type(groups).__name__}")
    _need_here(x, A, B, groups.words, scaling)
    n = C.c_size_t()
    check(load_library().qgemm_group_rows_words(groups.rows, groups.adapters, C.byref(n)))
    _need_type(groups.words, (torch.int32,), "groups")
    if groups.words.numel() != n.value or not groups.words.is_contiguous():
        raise ValueError(f"groups must be what group_rows() gives for {groups.rows} rows and {groups.adapters} adapters")
    rows, k, ldx = _rows_of(x, "x")
    _need_type(x, _FLOATS[1:], "x")
    for t, name in ((A, "A"), (B, "B")):
        _need_type(t, (x.dtype,), name)
        if t.dim() != 3 or not t.is_contiguous() or min(t.shape) < 1:
            raise ValueError(f"{name} must be contiguous [adapters, rank, columns], got shape {tuple(t.shape)} strides {t.stride()}")
    if A.shape[0] != groups.adapters or A.shape[:2] != B.shape[:2] or A.shape[2] != k or rows != groups.rows:
        raise ValueError(f"x {tuple(x.shape)}, A {tuple(A.shape)}, B {tuple(B.shape)} and groups of {groups.rows} rows and {groups.adapters} adapters do not fit together")
    return rows, k, ldx, A.shape[1], B.shape[2], None if scaling is None else _need_floats(scaling, groups.adapters, "scaling")


def add_adapters(y, x, A, B, groups, scaling=None, out=None, keep=False):
    """out[t] = y[t] + scaling[i] * (x[t] A[i]^T) B[i] for every row t and its adapter i (group_rows); y[t] for a row of none.  x [..., k] bf16 or fp16; A [adapters, rank, k] and
    B [adapters, rank, n] of x's type, the rank (up to 128) as rows of both; scaling [adapters] fp32 or None; y [..., n] is the result of the product that the adapters stand
    beside, fp32 / bf16 / fp16.  out: a tensor like y, which may be y itself; None: a new one.
    keep: out, u, where u [..., rank] fp32 is x A^T, what the backward pass needs."""
    native = _native()
    if native and isinstance(groups, RowGroups):
        st, res, u = native.ops_add_adapters(y, x, A, B, groups.words, groups.rows, groups.adapters, scaling, out, keep)
        if st == 0:
            return (res, u) if keep else res
        if st > 0:
            check(st)
    rows, k, ldx, rank, n, s = _adapters(x, A, B, groups, scaling)
    _need_here(y, out)
    ldy = _like(y, (rows, n), "y", _FLOATS)
    if out is None:
        out = torch.empty(y.shape, dtype=y.dtype, device=y.device)
    if out.shape != y.shape:
        raise ValueError(f"out must have y's shape, {tuple(y.shape)}, got {tuple(out.shape)}")
    ldo = _like(out, (rows, n), "out", (y.dtype,))
    u = torch.empty((*x.shape[:-1], rank), dtype=torch.float32, device=x.device) if keep else None
    check(load_library().qgemm_add_adapters(
        _dt(x), _dt(y), y.data_ptr(), ldy, x.data_ptr(), ldx, A.data_ptr(), B.data_ptr(), s, groups.words.data_ptr(), out.data_ptr(), ldo,
        None if u is None else u.data_ptr(), rows, groups.adapters, rank, k, n, _stream()))
    return (out, u) if keep else out


def add_adapters_backward(dy, x, u, A, B, groups, scaling=None, dx=None, grad_dtype=torch.float32):
    """dx, dA, dB of add_adapters: dy [..., n] of x's type, u as add_adapters(..., keep=True) gave it.  dx: the gradient of x that arrives from the product beside the adapters, fp32 / bf16 /
    fp16, to which theirs is added in a new tensor of its type; None: theirs alone, of x's type.  dA and dB have grad_dtype; zeros for adapters without rows.  (The gradient of
    y is dy.)"""
    native = _native()
    if native and isinstance(groups, RowGroups):
        st, *out = native.ops_add_adapters_backward(dy, x, u, A, B, groups.words, groups.rows, groups.adapters, scaling, dx, grad_dtype)
        if st == 0:
            return tuple(out)
        if st > 0:
            check(st)
    rows, k, ldx, rank, n, s = _adapters(x, A, B, groups, scaling)
    _need_here(dy, u, dx)
    lddy = _like(dy, (rows, n), "dy", (x.dtype,))
    _need_type(grad_dtype, _FLOATS, "grad_dtype")
    up = _need_floats(u, rows * rank, "u")
    ld0 = k if dx is None else _like(dx, (rows, k), "dx", _FLOATS)
    res = torch.empty(x.shape, dtype=x.dtype if dx is None else dx.dtype, device=x.device)
    dA, dB = (torch.empty(t.shape, dtype=grad_dtype, device=x.device) for t in (A, B))
    check(load_library().qgemm_add_adapters_backward(
        _dt(x), _dt(res), _dt(dA), dy.data_ptr(), lddy, x.data_ptr(), ldx, up, A.data_ptr(), B.data_ptr(), s, groups.words.data_ptr(),
        None if dx is None else dx.data_ptr(), ld0, res.data_ptr(), k, dA.data_ptr(), dB.data_ptr(), rows, groups.adapters, rank, k, n, _stream()))
    return res, dA, dB


def _tokens(tokens, rows):
    _need_here(tokens)
    _need_type(tokens, (torch.int32, torch.int64), "tokens")
    if tokens.numel() != rows or not tokens.is_contiguous():
        raise ValueError(f"tokens must hold {rows} contiguous numbers, got shape {tuple(tokens.shape)}")
    return tokens.data_ptr()


def log_probabilities(logits, tokens, top=0):
    """logp, entropy, lse [...] fp32 of logits [..., vocabulary], fp32 / bf16 / fp16, and tokens [...], int32 or int64: log softmax at the token, the softmax's entropy, log sum
    exp.  A token outside the vocabulary (-100) asks for nothing, its logp is 0.  -inf is a token that cannot be; a row of nothing else has lse = logp = -inf
    and entropy 0.
    top (up to 32): logp, entropy, lse, values, indices [..., top], the most probable tokens (int64) and their log probabilities, equal ones in the order of their numbers."""
    native = _native()
    if native:
        st, *out = native.ops_log_probabilities(logits, tokens, top)
        if st == 0:
            return tuple(out) if top else tuple(out[:3])
        if st > 0:
            check(st)
    _need_here(logits)
    rows, cols, ld = _rows_of(logits, "logits")
    _need_type(logits, _FLOATS, "logits")
    t = _tokens(tokens, rows)
    lead = logits.shape[:-1]
    logp, entropy, lse = (torch.empty(lead, dtype=torch.float32, device=logits.device) for _ in range(3))
    values, indices = (torch.empty((*lead, _size(top, "top")), dtype=d, device=logits.device) for d in (torch.float32, torch.int64))
    check(load_library().qgemm_log_probabilities(_dt(logits), tokens.element_size(), logits.data_ptr(), ld, t, top, logp.data_ptr(), entropy.data_ptr(),
                                                 lse.data_ptr(), values.data_ptr(), indices.data_ptr(), rows, cols, _stream()))
    return (logp, entropy, lse, values, indices) if top else (logp, entropy, lse)


def log_probabilities_backward(logits, tokens, lse, entropy, dlogp, dentropy=None, out_dtype=None):
    """dlogits = dlogp * ([token] - p) - dentropy * p * (log p + entropy), of logits' type or out_dtype: the gradient of the logits out of those of log_probabilities' logp and
    entropy (None: zeros); lse and entropy as it gave them."""
    native = _native()
    if native:
        st, out = native.ops_log_probabilities_backward(logits, tokens, lse, entropy, dlogp, dentropy, out_dtype)
        if st == 0:
            return out
        if st > 0:
            check(st)
    _need_here(logits, lse, entropy, dlogp, dentropy)
    rows, cols, ld = _rows_of(logits, "logits")
    out_dtype = logits.dtype if out_dtype is None else out_dtype
    _need_type(logits, _FLOATS, "logits")
    _need_type(out_dtype, _FLOATS, "out_dtype")
    t = _tokens(tokens, rows)
    at = [None if v is None else _need_floats(v, rows, name) for v, name in ((lse, "lse"), (entropy, "entropy"), (dlogp, "dlogp"), (dentropy, "dentropy"))]
    out = torch.empty(logits.shape, dtype=out_dtype, device=logits.device)
    check(load_library().qgemm_log_probabilities_backward(_dt(logits), _dt(out), tokens.element_size(), logits.data_ptr(), ld, t, *at, out.data_ptr(), cols, rows, cols,
                                                          _stream()))
    return out
