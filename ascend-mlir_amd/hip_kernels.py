"""ctypes binding of the fused-kernel C ABI (include/afir_hip_kernels.h).

Tensors are torch CUDA(ROCm) tensors used purely as device buffers; every
function launches on torch's current stream unless `stream` (a raw
hipStream_t value) is given, and returns the output tensor.  Nothing here
computes on the host.
"""
from __future__ import annotations

import ctypes
import os
import struct

from . import KERNELS_LIB

_HERE = os.path.dirname(os.path.abspath(__file__))


class AfirHipError(RuntimeError):
    pass


class _KernelInfo(ctypes.Structure):
    _fields_ = [("name", ctypes.c_char_p), ("symbol", ctypes.c_char_p),
                ("num_inputs", ctypes.c_int), ("num_outputs", ctypes.c_int),
                ("num_tiling_fields", ctypes.c_int),
                ("tiling_fields", ctypes.POINTER(ctypes.c_char_p)),
                ("signature", ctypes.c_char_p)]


EXPORTED_SYMBOLS = [
    "afir_hip_last_error",
    "afir_hip_launch_fused_add_mul",
    "afir_hip_launch_broadcast_add_reducesum",
    "afir_hip_launch_broadcast_add_reducesum_noalloc",
    "afir_hip_launch_relu_broadcast_add_transpose",
    "afir_hip_launch_gather_scale_shift",
    "afir_hip_launch_matmul_add_leakyrelu",
    "afir_hip_launch_mxfp4_quantize",
    "afir_hip_launch_mxfp4_matmul_add_leakyrelu",
    "afir_hip_mxfp4_matmul_workspace_bytes",
    "afir_hip_launch_norm_gate_residual",
    "afir_hip_launch_norm_gate_residual_backward",
    "afir_hip_norm_gate_residual_backward_workspace_bytes",
    "afir_hip_kernel_count",
    "afir_hip_kernel_info",
    "afir_hip_find_kernel",
    "afir_hip_launch",
    "afir_hip_argument_bytes",
    "afir_hip_region_register",
    "afir_hip_region_unregister",
    "afir_hip_region_info",
    "afir_hip_region_tiling_field",
    "afir_hip_region_kernel",
    "afir_hip_region_route",
    "afir_hip_region_emit_source",
    "afir_hip_region_attach_code_object",
    "afir_hip_region_compile",
    "afir_hip_region_load",
    "afir_hip_region_prefer_code_object",
    "afir_hip_region_argument_bytes",
    "afir_hip_launch_region",
    "afir_hip_last_launch",
]

_lib = None


def load():
    """dlopen the kernel library; raises if it has not been built."""
    global _lib
    if _lib is not None:
        return _lib
    if not os.path.exists(KERNELS_LIB):
        raise AfirHipError(
            f"{KERNELS_LIB} is missing: build it with "
            "`python ascend-mlir_amd/build.py` (there is no CPU fallback)")
    L = ctypes.CDLL(KERNELS_LIB)
    vp, u32 = ctypes.c_void_p, ctypes.c_uint32
    L.afir_hip_last_error.restype = ctypes.c_char_p
    L.afir_hip_last_launch.restype = ctypes.c_char_p
    L.afir_hip_last_launch.argtypes = [ctypes.POINTER(u32), ctypes.POINTER(u32)]
    for name, nptr in [("afir_hip_launch_fused_add_mul", 5),
                       ("afir_hip_launch_broadcast_add_reducesum", 5),
                       ("afir_hip_launch_broadcast_add_reducesum_noalloc", 5),
                       ("afir_hip_launch_relu_broadcast_add_transpose", 5),
                       ("afir_hip_launch_gather_scale_shift", 7),
                       ("afir_hip_launch_matmul_add_leakyrelu", 6),
                       ("afir_hip_launch_mxfp4_quantize", 6),
                       ("afir_hip_launch_mxfp4_matmul_add_leakyrelu", 8),
                       ("afir_hip_launch_norm_gate_residual", 9),
                       ("afir_hip_launch_norm_gate_residual_backward", 14)]:
        fn = getattr(L, name)
        fn.restype = u32
        fn.argtypes = [u32, vp] + [vp] * nptr
    for name in ("afir_hip_mxfp4_matmul_workspace_bytes", "afir_hip_norm_gate_residual_backward_workspace_bytes"):
        getattr(L, name).restype = ctypes.c_size_t
        getattr(L, name).argtypes = [vp]
    L.afir_hip_kernel_count.restype = ctypes.c_int
    L.afir_hip_kernel_info.restype = ctypes.POINTER(_KernelInfo)
    L.afir_hip_kernel_info.argtypes = [ctypes.c_int]
    L.afir_hip_find_kernel.restype = ctypes.POINTER(_KernelInfo)
    L.afir_hip_find_kernel.argtypes = [ctypes.c_char_p]
    L.afir_hip_launch.restype = u32
    L.afir_hip_launch.argtypes = [ctypes.c_char_p, u32, vp, ctypes.c_int,
                                  ctypes.POINTER(vp), vp, vp, ctypes.c_size_t]
    _lib = L
    return L


def last_launch() -> dict:
    """The kernel this thread launched last through the library, and its grid."""
    wg, th = ctypes.c_uint32(0), ctypes.c_uint32(0)
    name = load().afir_hip_last_launch(ctypes.byref(wg), ctypes.byref(th))
    return {"kernel": (name or b"").decode(), "workgroups": wg.value, "threads": th.value}


def kernel_table():
    L = load()
    out = []
    for i in range(L.afir_hip_kernel_count()):
        k = L.afir_hip_kernel_info(i).contents
        out.append({
            "name": k.name.decode(), "symbol": k.symbol.decode(),
            "num_inputs": k.num_inputs, "num_outputs": k.num_outputs,
            "tiling_fields": [k.tiling_fields[j].decode()
                              for j in range(k.num_tiling_fields)],
            "signature": k.signature.decode()})
    return out


def pack_tiling(*fields) -> bytes:
    return struct.pack("<%dq" % len(fields), *[int(f) for f in fields])


def f32_bits(x: float) -> int:
    return struct.unpack("<I", struct.pack("<f", x))[0]


def _check(rc):
    if rc != 0:
        raise AfirHipError(f"rc={rc}: {load().afir_hip_last_error().decode()}")


def _stream(stream):
    if stream is not None:
        return ctypes.c_void_p(stream)
    import torch
    return ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)


def _ptr(t):
    return ctypes.c_void_p(t.data_ptr())


def _dev(t, dtype, what):
    import torch
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise AfirHipError(f"{what}: expected a device tensor")
    if t.dtype != dtype:
        raise AfirHipError(f"{what}: expected {dtype}, got {t.dtype}")
    if not t.is_contiguous():
        raise AfirHipError(f"{what}: expected a contiguous tensor")
    return t


def launch_raw(symbol: str, block_dim: int, stream, ptrs, tiling: bytes):
    """Call a launcher symbol with raw device addresses (ints)."""
    L = load()
    fn = getattr(L, symbol)
    buf = ctypes.create_string_buffer(tiling, len(tiling))
    args = [ctypes.c_void_p(p) for p in ptrs]
    return fn(ctypes.c_uint32(block_dim), _stream(stream), *args,
              ctypes.cast(buf, ctypes.c_void_p))


def fused_add_mul(a, b, out=None, block_dim=0, stream=None):
    import torch
    _dev(a, torch.float32, "a"); _dev(b, torch.float32, "b")
    if a.shape != b.shape:
        raise AfirHipError("fused_add_mul: a and b must have the same shape")
    if out is None:
        out = torch.empty_like(a)
    _dev(out, torch.float32, "out")
    rows = a.shape[0] if a.dim() > 0 else 1
    cols = a.numel() // rows if rows else 0
    _check(launch_raw("afir_hip_launch_fused_add_mul", block_dim, stream,
                      [a.data_ptr(), b.data_ptr(), out.data_ptr(), 0],
                      pack_tiling(rows, cols)))
    return out


def broadcast_add_reducesum(x, bias, out=None, block_dim=0, stream=None):
    import torch
    _dev(x, torch.float32, "x"); _dev(bias, torch.float32, "bias")
    m, n = x.shape
    if bias.shape != (n,):
        raise AfirHipError("broadcast_add_reducesum: bias must have shape [N]")
    if out is None:
        out = torch.empty((m,), dtype=torch.float32, device=x.device)
    _dev(out, torch.float32, "out")
    _check(launch_raw("afir_hip_launch_broadcast_add_reducesum", block_dim, stream,
                      [x.data_ptr(), bias.data_ptr(), out.data_ptr(), 0],
                      pack_tiling(m, n)))
    return out


def relu_broadcast_add_transpose(x, c, out=None, block_dim=0, stream=None):
    import torch
    _dev(x, torch.float16, "x"); _dev(c, torch.float16, "c")
    b, m, n = x.shape
    if c.shape != (n,):
        raise AfirHipError("relu_broadcast_add_transpose: c must have shape [N]")
    if out is None:
        out = torch.empty((b, n, m), dtype=torch.float16, device=x.device)
    _dev(out, torch.float16, "out")
    _check(launch_raw("afir_hip_launch_relu_broadcast_add_transpose", block_dim, stream,
                      [x.data_ptr(), c.data_ptr(), out.data_ptr(), 0],
                      pack_tiling(b, m, n)))
    return out


def gather_scale_shift(table, indices, scale, shift, out=None, workspace=None,
                       block_dim=0, stream=None):
    import torch
    _dev(table, torch.float16, "table"); _dev(indices, torch.int32, "indices")
    _dev(scale, torch.float16, "scale"); _dev(shift, torch.float16, "shift")
    v, d = table.shape
    (r,) = indices.shape
    if scale.shape != (d,) or shift.shape != (d,):
        raise AfirHipError("gather_scale_shift: scale/shift must have shape [D]")
    if out is None:
        out = torch.empty((r, d), dtype=torch.float16, device=table.device)
    _dev(out, torch.float16, "out")
    ws = workspace.data_ptr() if workspace is not None else 0
    _check(launch_raw("afir_hip_launch_gather_scale_shift", block_dim, stream,
                      [table.data_ptr(), indices.data_ptr(), scale.data_ptr(),
                       shift.data_ptr(), out.data_ptr(), ws],
                      pack_tiling(v, d, r)))
    return out


def matmul_add_leakyrelu(a, b, bias, alpha=0.01, out=None, block_dim=0, stream=None):
    import torch
    _dev(a, torch.bfloat16, "a"); _dev(b, torch.bfloat16, "b")
    _dev(bias, torch.bfloat16, "bias")
    m, k = a.shape
    k2, n = b.shape
    if k != k2 or bias.shape != (n,):
        raise AfirHipError("matmul_add_leakyrelu: shape mismatch")
    if out is None:
        out = torch.empty((m, n), dtype=torch.bfloat16, device=a.device)
    _dev(out, torch.bfloat16, "out")
    _check(launch_raw("afir_hip_launch_matmul_add_leakyrelu", block_dim, stream,
                      [a.data_ptr(), b.data_ptr(), bias.data_ptr(), out.data_ptr(), 0],
                      pack_tiling(m, k, n, f32_bits(alpha))))
    return out


# ---- four-bit block products, and the norms around a residual block ------------
#
# Unlike the families above these take tensors of any of the three float types and rows
# with a stride, launch on the device of their tensors, and check every tensor against the
# others before they launch.  They are called once per layer and token, so the checks are
# one expression per tensor; only a tensor that fails it is looked at closely.  Autograd does
# not see them: results carry no graph, also where an input requires a gradient.

_ELEM_TYPES = {}
_entries = {}


def _elem_type(dtype, what):
    if not _ELEM_TYPES:
        import torch
        _ELEM_TYPES.update({torch.float32: 0, torch.float16: 1, torch.bfloat16: 2})
    code = _ELEM_TYPES.get(dtype)
    if code is None:
        raise AfirHipError(f"{what}: expected float32, float16 or bfloat16, got {dtype}")
    return code


def _device_of(t, what):
    """Index of the device of a call's first tensor."""
    try:
        index = t.get_device()
    except AttributeError:
        index = -1
    if index < 0:
        raise AfirHipError(f"{what}: expected a device tensor")
    return index


def _explain(t, shape, dtype, index, what):
    """Raises for the first thing about t that is not as it has to be."""
    import torch
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise AfirHipError(f"{what}: expected a device tensor")
    if t.get_device() != index:
        raise AfirHipError(f"{what}: on {t.device}, the call's first tensor is on device {index}")
    if t.dtype != dtype:
        raise AfirHipError(f"{what}: expected {dtype}, got {t.dtype}")
    if t.shape != shape:
        raise AfirHipError(f"{what}: expected shape {tuple(shape)}, got {tuple(t.shape)}")


def _dense(t, shape, dtype, index, what):
    try:
        if t.is_contiguous() and t.shape == shape and t.dtype is dtype and t.get_device() == index:
            return
    except AttributeError:
        pass
    _explain(t, shape, dtype, index, what)
    raise AfirHipError(f"{what}: expected a contiguous tensor")


def _rows(t, shape, dtype, index, what):
    """A matrix of rows that may have a stride; returns the stride in elements."""
    try:
        if t.is_contiguous() and t.shape == shape and t.dtype is dtype and t.get_device() == index:
            return shape[1]
    except AttributeError:
        pass
    _explain(t, shape, dtype, index, what)
    ld, unit = t.stride()
    if unit != 1 and shape[1] > 1:
        raise AfirHipError(f"{what}: the numbers of a row must be adjacent")
    if ld < shape[1]:
        if shape[0] > 1:
            raise AfirHipError(f"{what}: rows must not overlap")
        return shape[1]   # one row: its stride means nothing
    return ld


def _given_stream(stream, index):
    """The caller's stream as the current one, for a call's results and scratch as well: memory
    from another stream's pool may still be in use by work that is under way there.  0 is the
    default stream's handle (ExternalStream would take it for "any stream of the pool", which
    waits for nothing that the caller has issued)."""
    import torch
    given = torch.cuda.ExternalStream(stream, device=index) if stream else torch.cuda.default_stream(index)
    return torch.cuda.stream(given)


def _launch_on(index, symbol, block_dim, tiling, workspace, *tensors):
    """Launch on the current stream of device `index`; tensors may be None."""
    import torch
    fn = _entries.get(symbol)
    if fn is None:
        fn = _entries[symbol] = getattr(load(), symbol)
    ptrs = [None if t is None else t.data_ptr() for t in tensors]
    if torch.cuda.current_device() != index:
        with torch.cuda.device(index):
            rc = fn(block_dim, torch._C._cuda_getCurrentRawStream(index), *ptrs, workspace, tiling)
    else:
        # (the raw handle: building a Stream object takes as long as the rest of the call)
        rc = fn(block_dim, torch._C._cuda_getCurrentRawStream(index), *ptrs, workspace, tiling)
    if rc:
        _check(rc)


def _like(t):
    """A dense tensor of t's shape and type.  (An allocation is a tenth of a call: empty_like takes 1.2 us,
    new_empty 1.7 and empty with a type and a device 2.2.)"""
    import torch
    return torch.empty_like(t) if t.is_contiguous() else t.new_empty(t.shape)


def _workspace(query, tiling, like):
    """Scratch of the size that the library asks for, from torch's allocator, which hands it
    out again only to work that follows on the current stream, that of this call."""
    fn = _entries.get(query)
    if fn is None:
        fn = _entries[query] = getattr(load(), query)
    size = fn(tiling)
    if not size:
        return None
    import torch
    return like.new_empty((size,), dtype=torch.uint8)


_PACK5, _PACK11, _PACK13 = (struct.Struct(f"<{count}q").pack for count in (5, 11, 13))


def mxfp4_quantize(x, axis=-1, codes=None, scales=None, values=None, return_values=False,
                   block_dim=0, stream=None):
    """x -> MXFP4 along `axis`: blocks of 32 numbers share a power of two, numbers are e2m1.

    axis -1 (or 1): x is [R, K].  axis 0: x is [K, R], a weight kept input-major, say; codes
    and scales are laid out as for its transpose.  Rows of x may have a stride.  Returns
    (codes uint8 [R, ceil(K/32)*16], scales float8_e8m0fnu [R, ceil(K/32)]), and with
    return_values (or values=) also the numbers they stand for, in x's shape and type.
    Blocks that hold an infinity or a NaN read as NaN throughout."""
    import torch
    index = _device_of(x, "x")
    if stream is not None:
        with _given_stream(stream, index):
            return mxfp4_quantize(x, axis, codes, scales, values, return_values, block_dim)
    if x.dim() != 2:
        raise AfirHipError("mxfp4_quantize: x must have two dimensions")
    if axis not in (-1, 0, 1):
        raise AfirHipError("mxfp4_quantize: axis must be 0 or 1 (or -1)")
    shape, dtype = x.shape, x.dtype
    kind = _elem_type(dtype, "x")
    ld = _rows(x, shape, dtype, index, "x")
    k, r = shape if axis == 0 else (shape[1], shape[0])
    kb = (k + 31) // 32
    if codes is None:
        codes = x.new_empty((r, kb * 16), dtype=torch.uint8)
    else:
        _dense(codes, (r, kb * 16), torch.uint8, index, "codes")
    if scales is None:
        scales = x.new_empty((r, kb), dtype=torch.float8_e8m0fnu)
    else:
        _dense(scales, (r, kb), torch.float8_e8m0fnu, index, "scales")
    if values is not None:
        _dense(values, shape, dtype, index, "values")
    elif return_values:
        values = _like(x)
    _launch_on(index, "afir_hip_launch_mxfp4_quantize", block_dim,
               _PACK5(shape[0], shape[1], ld, 0 if axis == 0 else 1, kind), None, x, codes, scales, values)
    return (codes, scales) if values is None else (codes, scales, values)


def mxfp4_matmul_add_leakyrelu(a, a_scales, b, b_scales, bias=None, alpha=0.01, out=None, out_dtype=None, k=None,
                               block_dim=0, stream=None):
    """out [M, N] = leakyrelu(A @ B^T + bias, alpha) with A [M, K] and B [N, K] in MXFP4, as
    mxfp4_quantize gives them; alpha=1 leaves the sum as it is.  out_dtype (bfloat16 unless
    out is given) is the type of bias and out.  k: K itself, where it is not a multiple of
    32 (only checked against the codes)."""
    import torch
    index = _device_of(a, "a")
    if stream is not None:
        with _given_stream(stream, index):
            return mxfp4_matmul_add_leakyrelu(a, a_scales, b, b_scales, bias, alpha, out, out_dtype, k, block_dim)
    try:
        (m, row), (n, _) = a.shape, b.shape
    except (AttributeError, ValueError):
        raise AfirHipError("mxfp4_matmul_add_leakyrelu: codes must be tensors of two dimensions") from None
    kb = row // 16
    if row % 16:
        raise AfirHipError("mxfp4_matmul_add_leakyrelu: code rows must be whole blocks of 16 bytes")
    if k is None:
        k = kb * 32
    elif (k + 31) // 32 != kb:
        raise AfirHipError(f"mxfp4_matmul_add_leakyrelu: k = {k} does not have {kb} blocks")
    _dense(a, (m, row), torch.uint8, index, "a")
    _dense(b, (n, row), torch.uint8, index, "b")
    _dense(a_scales, (m, kb), torch.float8_e8m0fnu, index, "a_scales")
    _dense(b_scales, (n, kb), torch.float8_e8m0fnu, index, "b_scales")
    if out is None:
        dtype = torch.bfloat16 if out_dtype is None else out_dtype
        kind = _elem_type(dtype, "out")
        out = a.new_empty((m, n), dtype=dtype)
    else:
        dtype = out.dtype if out_dtype is None else out_dtype
        kind = _elem_type(dtype, "out")
        _dense(out, (m, n), dtype, index, "out")
    if bias is not None:
        _dense(bias, (n,), dtype, index, "bias")
    tiling = _PACK5(m, k, n, f32_bits(alpha), kind)
    ws = _workspace("afir_hip_mxfp4_matmul_workspace_bytes", tiling, a)
    _launch_on(index, "afir_hip_launch_mxfp4_matmul_add_leakyrelu", block_dim, tiling,
               None if ws is None else ws.data_ptr(), a, a_scales, b, b_scales, bias, out)
    return out


def _gate_rows(gate, m, n, rows_per_gate, dtype, index):
    """(rows_per_gate, row stride) of a gate [G, N] or [N] for m rows."""
    if gate is None:
        return max(m, 1), n
    if _device_of(gate, "gate") != index:
        _explain(gate, None, None, index, "gate")
    if gate.dim() == 1:
        gate = gate.unsqueeze(0)
    if gate.dim() != 2:
        raise AfirHipError("gate: expected one or two dimensions")
    g = gate.shape[0]
    if rows_per_gate is None:
        rows_per_gate = max(m, 1) if g == 1 else 1
    # (a batch of no rows needs no gate row, and may come with the one learned row of every batch)
    if rows_per_gate < 1 or (-(-m // rows_per_gate) != g and (m, g) != (0, 1)):
        raise AfirHipError(f"gate: {g} rows of {rows_per_gate} do not cover {m} rows")
    return rows_per_gate, _rows(gate, (g, n), dtype, index, "gate")


def norm_gate_residual(x, f=None, post_weight=None, gate=None, pre_weight=None, residual_scale=1.0, eps=1e-6,
                       rows_per_gate=None, y=None, h=None, block_dim=0, stream=None):
    """The end of one residual block and the start of the next, in one pass:

        y = residual_scale * x + gate * rmsnorm(f) * post_weight        h = rmsnorm(y) * pre_weight

    x, f [M, N] (rows may have a stride), weights [N], gate [G, N] or [N]: row i takes gate
    row i // rows_per_gate (None: one gate row for all rows, or one each).  Without f, y is x
    (the norm ahead of the first block); without pre_weight there is no h.  Returns (y, h).
    y=x and h=f work in place; y and h must not overlap.  The results carry no autograd graph:
    norm_gate_residual_backward gives the gradients."""
    index = _device_of(x, "x")
    if stream is not None:
        with _given_stream(stream, index):
            return norm_gate_residual(x, f, post_weight, gate, pre_weight, residual_scale, eps, rows_per_gate, y, h,
                                      block_dim)
    if x.dim() != 2:
        raise AfirHipError("norm_gate_residual: x must have two dimensions")
    dtype = x.dtype
    kind = _elem_type(dtype, "x")
    m, n = shape = x.shape
    ld_x = _rows(x, shape, dtype, index, "x")
    ld_f = ld_gate = ld_y = ld_h = n
    if f is None:
        if post_weight is not None or gate is not None or y is not None or pre_weight is None:
            raise AfirHipError("norm_gate_residual: without f only x and pre_weight are used")
        rows_per_gate = max(m, 1)
    else:
        ld_f = _rows(f, shape, dtype, index, "f")
        _dense(post_weight, (n,), dtype, index, "post_weight")
        rows_per_gate, ld_gate = _gate_rows(gate, m, n, rows_per_gate, dtype, index)
        if y is None:
            y = _like(x)
        ld_y = _rows(y, shape, dtype, index, "y")
    if pre_weight is not None:
        _dense(pre_weight, (n,), dtype, index, "pre_weight")
        if h is None:
            h = _like(x)
        elif h is y:
            raise AfirHipError("norm_gate_residual: y and h are two results")
        ld_h = _rows(h, shape, dtype, index, "h")
    elif h is not None:
        raise AfirHipError("norm_gate_residual: h needs pre_weight")
    _launch_on(index, "afir_hip_launch_norm_gate_residual", block_dim,
               _PACK11(m, n, rows_per_gate, ld_x, ld_f, ld_gate, ld_y, ld_h, f32_bits(residual_scale), f32_bits(eps), kind),
               None, x, f, post_weight, gate, pre_weight, y, h)
    return (x if f is None else y), h


def norm_gate_residual_backward(dy, dh, y, f=None, post_weight=None, gate=None, pre_weight=None, residual_scale=1.0,
                                eps=1e-6, rows_per_gate=None, block_dim=0, stream=None):
    """The gradients (dx, df, dpost_weight, dgate, dpre_weight) of norm_gate_residual from
    those of its results and the y it returned; None where it had no such input.  dy None:
    zero.  dh, pre_weight None: the call had no h (y is not read then).  An empty y is refused:
    there are no rows to sum the weights' gradients over."""
    index = _device_of(y, "y")
    if stream is not None:
        with _given_stream(stream, index):
            return norm_gate_residual_backward(dy, dh, y, f, post_weight, gate, pre_weight, residual_scale, eps,
                                               rows_per_gate, block_dim)
    if y.dim() != 2:
        raise AfirHipError("norm_gate_residual_backward: y must have two dimensions")
    dtype = y.dtype
    kind = _elem_type(dtype, "y")
    m, n = shape = y.shape
    if m == 0 or n == 0:
        raise AfirHipError("norm_gate_residual_backward: empty tensors have no gradients to write")
    ld_y = _rows(y, shape, dtype, index, "y")
    ld_dy = ld_dh = ld_f = ld_gate = n
    if (dh is None) != (pre_weight is None):
        raise AfirHipError("norm_gate_residual_backward: dh and pre_weight go together")
    if dh is None and dy is None:
        raise AfirHipError("norm_gate_residual_backward: dy or dh is needed")
    if dh is None and f is None:
        raise AfirHipError("norm_gate_residual_backward: f or dh is needed")
    if dy is not None:
        ld_dy = _rows(dy, shape, dtype, index, "dy")
    df = dpost = dgate = dpre = None
    if dh is not None:
        ld_dh = _rows(dh, shape, dtype, index, "dh")
        _dense(pre_weight, (n,), dtype, index, "pre_weight")
        dpre = _like(pre_weight)
    if f is None:
        if post_weight is not None or gate is not None:
            raise AfirHipError("norm_gate_residual_backward: post_weight and gate need f")
        rows_per_gate = m
    else:
        ld_f = _rows(f, shape, dtype, index, "f")
        _dense(post_weight, (n,), dtype, index, "post_weight")
        rows_per_gate, ld_gate = _gate_rows(gate, m, n, rows_per_gate, dtype, index)
        df = _like(y)
        dpost = _like(post_weight)
        if gate is not None:
            dgate = _like(gate)
    dx = _like(y)
    tiling = _PACK13(m, n, rows_per_gate, ld_dy, ld_dh, ld_y, ld_f, ld_gate, n, n,
                     f32_bits(residual_scale), f32_bits(eps), kind)
    ws = _workspace("afir_hip_norm_gate_residual_backward_workspace_bytes", tiling, y)
    _launch_on(index, "afir_hip_launch_norm_gate_residual_backward", block_dim, tiling, ws.data_ptr(),
               dy, dh, None if dh is None else y, f, post_weight, gate, pre_weight, dx, df, dpost, dgate, dpre)
    return dx, df, dpost, dgate, dpre


def prepare(symbol: str, ptrs, tiling: bytes, block_dim: int = 0, stream=None):
    """Pre-marshal one launch; returns a zero-argument callable that issues it
    (used by tight loops such as the benchmark to keep host overhead down).
    The stream is captured now."""
    L = load()
    fn = getattr(L, symbol)
    buf = ctypes.create_string_buffer(tiling, len(tiling))
    args = [ctypes.c_uint32(block_dim), _stream(stream)]
    args += [ctypes.c_void_p(p) for p in ptrs]
    args.append(ctypes.cast(buf, ctypes.c_void_p))

    def call(_fn=fn, _args=tuple(args), _keep=buf):
        rc = _fn(*_args)
        if rc:
            _check(rc)
    return call


# ---- fused-region programs ---------------------------------------------------

_TORCH_TYPES = None


def _torch_type(name):
    global _TORCH_TYPES
    import torch
    if _TORCH_TYPES is None:
        _TORCH_TYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32,
                        "i32": torch.int32, "i64": torch.int64, "i16": torch.int16}
    return _TORCH_TYPES[name]


HIPCC_REGION_FLAGS = ["--genco", "--offload-arch=gfx950", "-O3", "-nogpuinc", "-ffp-contract=off",
                      "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops"]


def compile_region_source(source: str, cache_dir: str = None) -> bytes:
    """HIP source of a region (Region.emit_source, afir-translate
    --emit-hip-source) -> code object bytes.  Raises AfirHipError when hipcc is
    missing or rejects the source."""
    import hashlib
    import shutil
    import subprocess
    import tempfile
    cache_dir = cache_dir or os.path.join(_HERE, "lib", "region_cache")
    key = hashlib.sha256(("\n".join(HIPCC_REGION_FLAGS) + "\n" + source).encode()).hexdigest()[:24]
    path = os.path.join(cache_dir, key + ".hsaco")
    if os.path.exists(path):
        with open(path, "rb") as f:
            return f.read()
    hipcc = shutil.which("hipcc") or "/opt/rocm/bin/hipcc"
    if not os.path.exists(hipcc):
        raise AfirHipError("hipcc not found: cannot compile a region kernel")
    os.makedirs(cache_dir, exist_ok=True)
    with tempfile.TemporaryDirectory() as tmp:
        src = os.path.join(tmp, "region.hip")
        obj = os.path.join(tmp, "region.hsaco")
        with open(src, "w") as f:
            f.write(source)
        p = subprocess.run([hipcc, *HIPCC_REGION_FLAGS, "-o", obj, src], capture_output=True, text=True)
        if p.returncode != 0:
            raise AfirHipError("hipcc rejected the region source:\n" + p.stderr[-2000:])
        with open(obj, "rb") as f:
            image = f.read()
    tmp_path = path + f".{os.getpid()}.tmp"
    with open(tmp_path, "wb") as f:
        f.write(image)
    os.replace(tmp_path, path)
    return image


class Region:
    """A registered fused-region program (afir_hip_region_register)."""

    def __init__(self, text: str):
        L = load()
        u64 = ctypes.c_uint64
        L.afir_hip_region_register.restype = ctypes.c_uint32
        L.afir_hip_region_register.argtypes = [ctypes.c_char_p, ctypes.c_size_t, ctypes.POINTER(u64)]
        L.afir_hip_region_unregister.argtypes = [u64]
        L.afir_hip_region_info.argtypes = [u64] + [ctypes.POINTER(ctypes.c_int)] * 3
        L.afir_hip_region_tiling_field.restype = ctypes.c_char_p
        L.afir_hip_region_tiling_field.argtypes = [u64, ctypes.c_int]
        L.afir_hip_region_argument_bytes.argtypes = [u64, ctypes.c_void_p, ctypes.c_size_t,
                                                    ctypes.POINTER(ctypes.c_size_t), ctypes.c_int]
        L.afir_hip_launch_region.restype = ctypes.c_uint32
        L.afir_hip_launch_region.argtypes = [u64, ctypes.c_uint32, ctypes.c_void_p, ctypes.c_int,
                                             ctypes.POINTER(ctypes.c_void_p), ctypes.c_void_p,
                                             ctypes.c_void_p, ctypes.c_size_t]
        data = text.encode()
        h = u64(0)
        _check(L.afir_hip_region_register(data, len(data), ctypes.byref(h)))
        self.handle = h.value
        ni, no, nf = ctypes.c_int(), ctypes.c_int(), ctypes.c_int()
        _check(L.afir_hip_region_info(u64(self.handle), ctypes.byref(ni), ctypes.byref(no), ctypes.byref(nf)))
        self.num_inputs, self.num_outputs = ni.value, no.value
        self.tiling_fields = [L.afir_hip_region_tiling_field(u64(self.handle), i).decode()
                              for i in range(nf.value)]
        L.afir_hip_region_kernel.restype = ctypes.c_char_p
        L.afir_hip_region_kernel.argtypes = [u64]
        self.kernel = L.afir_hip_region_kernel(u64(self.handle)).decode()
        self.arg_types = [l.split()[2] for l in text.splitlines() if l.split()[:1] == ["arg"]]

    # ---- kernels compiled for this program ----

    def emit_source(self) -> str:
        """HIP source of the kernels specialised for this program."""
        L = load()
        L.afir_hip_region_emit_source.argtypes = [ctypes.c_uint64, ctypes.c_char_p, ctypes.c_size_t,
                                                  ctypes.POINTER(ctypes.c_size_t)]
        n = ctypes.c_size_t(0)
        _check(L.afir_hip_region_emit_source(ctypes.c_uint64(self.handle), None, 0, ctypes.byref(n)))
        buf = ctypes.create_string_buffer(n.value + 1)
        _check(L.afir_hip_region_emit_source(ctypes.c_uint64(self.handle), buf, n.value + 1, ctypes.byref(n)))
        return buf.value.decode()

    def attach_code_object(self, image: bytes):
        L = load()
        L.afir_hip_region_attach_code_object.argtypes = [ctypes.c_uint64, ctypes.c_char_p, ctypes.c_size_t]
        _check(L.afir_hip_region_attach_code_object(ctypes.c_uint64(self.handle), image, len(image)))
        L.afir_hip_region_kernel.restype = ctypes.c_char_p
        self.kernel = L.afir_hip_region_kernel(ctypes.c_uint64(self.handle)).decode()

    def prefer_code_object(self, prefer: bool = True):
        """Run the attached code object even where a hand-tuned family matches."""
        L = load()
        L.afir_hip_region_prefer_code_object.argtypes = [ctypes.c_uint64, ctypes.c_int]
        _check(L.afir_hip_region_prefer_code_object(ctypes.c_uint64(self.handle), 1 if prefer else 0))
        L.afir_hip_region_kernel.restype = ctypes.c_char_p
        self.kernel = L.afir_hip_region_kernel(ctypes.c_uint64(self.handle)).decode()
        return self

    def compile(self, cache_dir: str = None, in_process: bool = None):
        """Emit, compile and attach.  With hipcc (the default where it exists) the code
        object is kept in `cache_dir` (default: lib/region_cache beside the libraries)
        under the hash of its source, so a program is compiled once.  in_process=True, or
        no hipcc on this host: compiled inside the process by the HIP runtime's own
        compiler library (afir_hip_region_compile), nothing cached."""
        import shutil
        if in_process is None:
            in_process = not (shutil.which("hipcc") or os.path.exists("/opt/rocm/bin/hipcc"))
        if in_process:
            L = load()
            L.afir_hip_region_compile.restype = ctypes.c_uint32
            L.afir_hip_region_compile.argtypes = [ctypes.c_uint64, ctypes.c_void_p, ctypes.c_size_t,
                                                  ctypes.POINTER(ctypes.c_size_t)]
            n = ctypes.c_size_t(0)
            _check(L.afir_hip_region_compile(ctypes.c_uint64(self.handle), None, 0, ctypes.byref(n)))
            self.kernel = L.afir_hip_region_kernel(ctypes.c_uint64(self.handle)).decode()
            return self
        source = self.emit_source()
        self.attach_code_object(compile_region_source(source, cache_dir))
        return self

    def close(self):
        if self.handle:
            load().afir_hip_region_unregister(ctypes.c_uint64(self.handle))
            self.handle = 0

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def route(self, tiling: bytes) -> str:
        """"family", "compiled" or "interpreter": the kernels a launch with these
        shapes runs on (host only)."""
        L = load()
        L.afir_hip_region_route.restype = ctypes.c_char_p
        L.afir_hip_region_route.argtypes = [ctypes.c_uint64, ctypes.c_void_p, ctypes.c_size_t]
        buf = ctypes.create_string_buffer(tiling, len(tiling))
        got = L.afir_hip_region_route(ctypes.c_uint64(self.handle), buf, len(tiling)).decode()
        if not got:
            raise AfirHipError(L.afir_hip_last_error().decode())
        return got

    def argument_bytes(self, tiling: bytes):
        n = self.num_inputs + self.num_outputs
        out = (ctypes.c_size_t * n)()
        buf = ctypes.create_string_buffer(tiling, len(tiling))
        _check(load().afir_hip_region_argument_bytes(ctypes.c_uint64(self.handle), buf, len(tiling), out, n))
        return list(out)

    def launch_raw(self, ptrs, tiling: bytes, workspace=0, block_dim=0, stream=None):
        arr = (ctypes.c_void_p * len(ptrs))(*[ctypes.c_void_p(p) for p in ptrs])
        buf = ctypes.create_string_buffer(tiling, len(tiling))
        return load().afir_hip_launch_region(ctypes.c_uint64(self.handle), block_dim, _stream(stream),
                                             len(ptrs), arr, ctypes.c_void_p(workspace), buf, len(tiling))

    def prepare(self, ptrs, tiling: bytes, workspace=0, block_dim=0, stream=None):
        """Pre-marshal one launch; returns a zero-argument callable."""
        L = load()
        arr = (ctypes.c_void_p * len(ptrs))(*[ctypes.c_void_p(p) for p in ptrs])
        buf = ctypes.create_string_buffer(tiling, len(tiling))
        args = (ctypes.c_uint64(self.handle), ctypes.c_uint32(block_dim), _stream(stream), len(ptrs),
                arr, ctypes.c_void_p(workspace), ctypes.cast(buf, ctypes.c_void_p), len(tiling))

        def call(_fn=L.afir_hip_launch_region, _args=args, _keep=(arr, buf)):
            rc = _fn(*_args)
            if rc:
                _check(rc)
        return call

    def __call__(self, *inputs, out_shape, workspace=None, block_dim=0, stream=None):
        """inputs: device tensors in argument order; returns the output tensor."""
        import torch
        if len(inputs) != self.num_inputs:
            raise AfirHipError(f"region expects {self.num_inputs} inputs, got {len(inputs)}")
        for i, t in enumerate(inputs):
            _dev(t, _torch_type(self.arg_types[i]), f"region input {i}")
        out = torch.empty(tuple(out_shape), dtype=_torch_type(self.arg_types[-1]), device=inputs[0].device)
        dims = [d for t in inputs for d in t.shape] + list(out.shape)
        tiling = pack_tiling(*dims)
        ws = workspace.data_ptr() if workspace is not None else 0
        _check(self.launch_raw([t.data_ptr() for t in inputs] + [out.data_ptr()], tiling, ws,
                               block_dim, stream))
        return out
