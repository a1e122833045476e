"""ctypes binding of the C ABI in include/catlass_b200.h.

Used by the tests and the benchmark to call the library exactly as a C caller would: PODs, raw device
pointers, a stream handle.  Loading fails loudly when the shared object is missing; nothing here computes.
"""
import ctypes
import os

from . import build as _build

SUCCESS, INVALID, CUDA_ERROR, DEVICE_TIMEOUT, SCRATCH_TOO_SMALL = 0, 1, 2, 3, 4
ROW_MAJOR, COLUMN_MAJOR, ZN = 0, 1, 2
GROUP_LIST_INT64, GROUP_LIST_INT32 = 0, 1
DTYPE_F32, DTYPE_BF16, DTYPE_F16, DTYPE_F32_IN_U64 = 0, 1, 2, 3
FLAG_STATIC_WEIGHTS = 2
QUANT_PER_TENSOR, QUANT_PER_CHANNEL = 0, 1

_u32, _u64, _vp = ctypes.c_uint32, ctypes.c_uint64, ctypes.c_void_p


class QuantMatmulArgs(ctypes.Structure):
    _fields_ = [
        ("m", _u32), ("n", _u32), ("k", _u32), ("layout_a", _u32), ("layout_b", _u32),
        ("a", _vp), ("b", _vp), ("scale", _vp), ("per_token_scale", _vp), ("d", _vp), ("acc", _vp),
        ("workspace", _vp), ("workspace_bytes", _u64), ("block_num", _u32), ("flags", _u32),
        ("scale_type", _u32), ("d_type", _u32),
    ]


class GroupedQuantMatmulArgs(ctypes.Structure):
    _fields_ = [
        ("m", _u32), ("n", _u32), ("k", _u32), ("group_count", _u32), ("layout_b", _u32),
        ("group_list_type", _u32),
        ("a", _vp), ("b", _vp), ("group_list", _vp), ("scale", _vp), ("per_token_scale", _vp), ("d", _vp),
        ("acc", _vp), ("workspace", _vp), ("workspace_bytes", _u64), ("block_num", _u32), ("flags", _u32),
        ("scale_type", _u32), ("d_type", _u32),
    ]


class GroupedSliceKArgs(ctypes.Structure):
    _fields_ = [
        ("m", _u32), ("n", _u32), ("k", _u32), ("group_count", _u32), ("group_list_type", _u32), ("scale_type", _u32),
        ("a", _vp), ("b", _vp), ("group_list", _vp), ("scale", _vp), ("per_token_scale", _vp), ("d", _vp),
        ("acc", _vp), ("workspace", _vp), ("workspace_bytes", _u64), ("block_num", _u32), ("d_type", _u32),
    ]


class GroupedFixpipeDequantArgs(ctypes.Structure):
    _fields_ = [
        ("m", _u32), ("n", _u32), ("k", _u32), ("group_count", _u32), ("layout_b", _u32),
        ("group_list_type", _u32), ("quant_mode", _u32), ("scale_per_tensor", ctypes.c_float),
        ("a", _vp), ("b", _vp), ("group_list", _vp), ("per_channel_scale", _vp), ("d", _vp), ("acc", _vp),
        ("workspace", _vp), ("workspace_bytes", _u64), ("block_num", _u32), ("per_channel_scale_type", _u32),
        ("d_type", _u32), ("flags", _u32),
    ]


class GroupedQuantMatmulHostArgs(ctypes.Structure):
    _fields_ = [
        ("m", _u32), ("n", _u32), ("k", _u32), ("group_count", _u32), ("layout_b", _u32), ("chunks", _u32),
        ("a_host", _vp), ("group_list_host", _vp), ("per_token_host", _vp), ("d_host", _vp),
        ("b", _vp), ("scale", _vp), ("workspace", _vp), ("workspace_bytes", _u64),
    ]


class W4A8MatmulArgs(ctypes.Structure):
    _fields_ = [
        ("m", _u32), ("n", _u32), ("k", _u32), ("group_size", _u32),
        ("a", _vp), ("w_packed", _vp), ("weight_scale", _vp), ("per_token_scale", _vp), ("d", _vp),
        ("workspace", _vp), ("workspace_bytes", _u64), ("block_num", _u32), ("flags", _u32),
        ("d_type", _u32), ("pack_axis", _u32),
    ]


class MxMatmulArgs(ctypes.Structure):
    _fields_ = [
        ("m", _u32), ("n", _u32), ("k", _u32), ("format", _u32), ("layout_a", _u32), ("layout_b", _u32),
        ("a", _vp), ("b", _vp), ("scale_a", _vp), ("scale_b", _vp), ("d", _vp),
        ("workspace", _vp), ("workspace_bytes", _u64), ("block_num", _u32), ("flags", _u32),
    ]


class MxGroupedMatmulArgs(ctypes.Structure):
    _fields_ = [
        ("m", _u32), ("n", _u32), ("k", _u32), ("group_count", _u32), ("format", _u32), ("layout_b", _u32),
        ("group_list_type", _u32), ("group_list_kind", _u32),
        ("a", _vp), ("b", _vp), ("group_list", _vp), ("scale_a", _vp), ("scale_b", _vp), ("d", _vp),
        ("workspace", _vp), ("workspace_bytes", _u64), ("block_num", _u32), ("flags", _u32),
    ]


GROUP_LIST_SIZES, GROUP_LIST_PREFIX_SUMS = 0, 1


class MxGroupedSwigluQuantArgs(ctypes.Structure):
    _fields_ = [
        ("m", _u32), ("n", _u32), ("k", _u32), ("group_count", _u32), ("layout_b", _u32),
        ("group_list_type", _u32), ("group_list_kind", _u32), ("flags", _u32),
        ("a", _vp), ("b", _vp), ("group_list", _vp), ("scale_a", _vp), ("scale_b", _vp), ("q", _vp), ("q_scale", _vp),
        ("workspace", _vp), ("workspace_bytes", _u64), ("block_num", _u32), ("reserved", _u32),
    ]


class QuantizeInt8Args(ctypes.Structure):
    _fields_ = [("rows", _u32), ("k", _u32), ("x_type", _u32), ("reserved", _u32), ("x_pitch", _u64), ("x", _vp),
                ("q", _vp), ("scale", _vp)]


class MxQuantizeArgs(ctypes.Structure):
    _fields_ = [
        ("rows", _u32), ("k", _u32), ("format", _u32), ("x_type", _u32), ("x_pitch", _u64),
        ("x", _vp), ("q", _vp), ("scale", _vp),
    ]


class MxGroupedFinalizeRoutingArgs(ctypes.Structure):
    _fields_ = [
        ("m", _u32), ("n", _u32), ("k", _u32), ("group_count", _u32), ("layout_b", _u32),
        ("group_list_type", _u32), ("group_list_kind", _u32), ("row_index_type", _u32), ("batch", _u32),
        ("shared_rows", _u32), ("shared_offset", _u32), ("shared_weight", ctypes.c_float),
        ("a", _vp), ("b", _vp), ("group_list", _vp), ("scale_a", _vp), ("scale_b", _vp), ("logit", _vp),
        ("row_index", _vp), ("bias", _vp), ("shared_input", _vp), ("out", _vp),
        ("workspace", _vp), ("workspace_bytes", _u64), ("block_num", _u32), ("flags", _u32),
    ]


MX_E4M3, MX_E2M1 = 0, 1
MX_OUT_F32 = 1
W4_PACKED_ALONG_K, W4_PACKED_ALONG_N = 0, 1

_lib = None


def library_path():
    return _build.LIB_PATH


def load():
    """The loaded shared library. Raises if it has not been built (python -m catlass_b200.build)."""
    global _lib
    if _lib is not None:
        return _lib
    path = library_path()
    if not os.path.exists(path):
        raise RuntimeError(
            f"{path} is missing: build it with `python -m catlass_b200.build` (needs nvcc). "
            "There is no fallback path.")
    lib = ctypes.CDLL(path)
    for name, args_t in (("cb200_quant_matmul", QuantMatmulArgs),
                         ("cb200_grouped_quant_matmul_slice_m", GroupedQuantMatmulArgs),
                         ("cb200_grouped_matmul_slice_m_fixpipe_dequant", GroupedFixpipeDequantArgs),
                         ("cb200_grouped_quant_matmul_slice_k", GroupedSliceKArgs),
                         ("cb200_w4a8_matmul", W4A8MatmulArgs),
                         ("cb200_mx_matmul", MxMatmulArgs),
                         ("cb200_mx_grouped_matmul_slice_m", MxGroupedMatmulArgs),
                         ("cb200_mx_grouped_matmul_slice_m_swiglu_mx_quant", MxGroupedSwigluQuantArgs),
                         ("cb200_mx_grouped_matmul_finalize_routing", MxGroupedFinalizeRoutingArgs)):
        getattr(lib, name + "_can_implement").argtypes = [ctypes.POINTER(args_t)]
        getattr(lib, name + "_can_implement").restype = ctypes.c_int
        getattr(lib, name + "_workspace_size").argtypes = [ctypes.POINTER(args_t)]
        getattr(lib, name + "_workspace_size").restype = _u64
        getattr(lib, name).argtypes = [ctypes.POINTER(args_t), _vp]
        getattr(lib, name).restype = ctypes.c_int
    lib.cb200_grouped_quant_matmul_slice_m_host.argtypes = [ctypes.POINTER(GroupedQuantMatmulHostArgs), _vp]
    lib.cb200_grouped_quant_matmul_slice_m_host.restype = ctypes.c_int
    lib.cb200_grouped_quant_matmul_slice_m_host_workspace_size.argtypes = [ctypes.POINTER(GroupedQuantMatmulHostArgs)]
    lib.cb200_grouped_quant_matmul_slice_m_host_workspace_size.restype = _u64
    lib.cb200_mx_quantize.argtypes = [ctypes.POINTER(MxQuantizeArgs), _vp]
    lib.cb200_mx_quantize.restype = ctypes.c_int
    lib.cb200_mx_quantize_can_implement.argtypes = [ctypes.POINTER(MxQuantizeArgs)]
    lib.cb200_mx_quantize_can_implement.restype = ctypes.c_int
    lib.cb200_quantize_per_token_int8.argtypes = [ctypes.POINTER(QuantizeInt8Args), _vp]
    lib.cb200_quantize_per_token_int8.restype = ctypes.c_int
    lib.cb200_quantize_per_token_int8_can_implement.argtypes = [ctypes.POINTER(QuantizeInt8Args)]
    lib.cb200_quantize_per_token_int8_can_implement.restype = ctypes.c_int
    lib.cb200_mx_matmul_static.argtypes = [ctypes.POINTER(MxMatmulArgs), _vp]
    lib.cb200_mx_matmul_static.restype = ctypes.c_int
    lib.cb200_mx_matmul_static_scratch_bytes.restype = _u64
    lib.cb200_selftest_wait_timeout.argtypes = [_u32, _vp]
    lib.cb200_selftest_wait_timeout.restype = ctypes.c_int
    lib.cb200_device_status.argtypes = [ctypes.POINTER(_u32)]
    lib.cb200_device_status.restype = ctypes.c_int
    lib.cb200_last_cuda_error.restype = ctypes.c_int
    lib.cb200_launch_count.restype = _u64
    lib.cb200_version.restype = ctypes.c_char_p
    _lib = lib
    return lib


class CallError(RuntimeError):
    def __init__(self, what, status):
        super().__init__(f"{what} returned status {status} (cuda error {load().cb200_last_cuda_error()})")
        self.status = status


def _check(what, status):
    if status != SUCCESS:
        raise CallError(what, status)


def device_status():
    """(status, code): synchronises the device and reads the kernels' status word."""
    code = _u32(0)
    st = load().cb200_device_status(ctypes.byref(code))
    return st, code.value


def launch_count():
    return int(load().cb200_launch_count())


def _p(t):
    return None if t is None else ctypes.c_void_p(t.data_ptr())


def _stream(stream):
    if stream is None:
        import torch
        stream = torch.cuda.current_stream()
    return ctypes.c_void_p(stream.cuda_stream)


def quant_matmul(a, b, scale, per_token, d, m, n, k, layout_b=COLUMN_MAJOR, acc=None, stream=None,
                 block_num=0, layout_a=ROW_MAJOR, scale_type=DTYPE_F32, d_type=DTYPE_BF16, static_weights=False):
    """Enqueue the dense W8A8 dequant matmul. Arguments are torch CUDA tensors used as raw buffers."""
    args = QuantMatmulArgs(m=m, n=n, k=k, layout_a=layout_a, layout_b=layout_b, a=_p(a), b=_p(b),
                           scale=_p(scale), per_token_scale=_p(per_token), d=_p(d), acc=_p(acc),
                           workspace=None, workspace_bytes=0, block_num=block_num,
                           flags=FLAG_STATIC_WEIGHTS if static_weights else 0, scale_type=scale_type, d_type=d_type)
    _check("cb200_quant_matmul", load().cb200_quant_matmul(ctypes.byref(args), _stream(stream)))


def grouped_quant_matmul(a, b, group_list, scale, per_token, d, m, n, k, group_count, layout_b=ROW_MAJOR,
                         acc=None, stream=None, block_num=0, group_list_type=GROUP_LIST_INT64,
                         scale_type=DTYPE_F32, d_type=DTYPE_BF16):
    args = GroupedQuantMatmulArgs(m=m, n=n, k=k, group_count=group_count, layout_b=layout_b,
                                  group_list_type=group_list_type, a=_p(a), b=_p(b),
                                  group_list=_p(group_list), scale=_p(scale), per_token_scale=_p(per_token),
                                  d=_p(d), acc=_p(acc), workspace=None, workspace_bytes=0,
                                  block_num=block_num, flags=0, scale_type=scale_type, d_type=d_type)
    _check("cb200_grouped_quant_matmul_slice_m",
           load().cb200_grouped_quant_matmul_slice_m(ctypes.byref(args), _stream(stream)))


def grouped_fixpipe_dequant(a, b, group_list, d, m, n, k, group_count, quant_mode, scale_per_tensor=1.0,
                            per_channel_scale=None, per_channel_scale_type=DTYPE_F32, layout_b=ROW_MAJOR,
                            d_type=DTYPE_F16, acc=None, stream=None, group_list_type=GROUP_LIST_INT64):
    """Grouped slice-M W8A8 with per-tensor (quant_mode 0) or per-channel (1) dequant, no per-token factor."""
    args = GroupedFixpipeDequantArgs(m=m, n=n, k=k, group_count=group_count, layout_b=layout_b,
                                     group_list_type=group_list_type, quant_mode=quant_mode,
                                     scale_per_tensor=scale_per_tensor, a=_p(a), b=_p(b), group_list=_p(group_list),
                                     per_channel_scale=_p(per_channel_scale), d=_p(d), acc=_p(acc), workspace=None,
                                     workspace_bytes=0, block_num=0, per_channel_scale_type=per_channel_scale_type,
                                     d_type=d_type, flags=0)
    _check("cb200_grouped_matmul_slice_m_fixpipe_dequant",
           load().cb200_grouped_matmul_slice_m_fixpipe_dequant(ctypes.byref(args), _stream(stream)))


def grouped_quant_matmul_slice_k_workspace_size(m, n, k, group_count):
    args = GroupedSliceKArgs(m=m, n=n, k=k, group_count=group_count, a=256, b=256, group_list=256, scale=256,
                             per_token_scale=256, d=256)
    return int(load().cb200_grouped_quant_matmul_slice_k_workspace_size(ctypes.byref(args)))


def grouped_quant_matmul_slice_k(a, b, group_list, scale, per_token, d, m, n, k, group_count, workspace, acc=None,
                                 stream=None, group_list_type=GROUP_LIST_INT64, scale_type=DTYPE_F32,
                                 d_type=DTYPE_BF16, block_num=0):
    """Grouped slice-K W8A8: a [k][m] (A column-major), b [k][n], group_list prefix sums over K, scale [G][n],
    per_token [G][m], d [G][m][n]."""
    args = GroupedSliceKArgs(m=m, n=n, k=k, group_count=group_count, group_list_type=group_list_type,
                             scale_type=scale_type, a=_p(a), b=_p(b), group_list=_p(group_list), scale=_p(scale),
                             per_token_scale=_p(per_token), d=_p(d), acc=_p(acc), workspace=_p(workspace),
                             workspace_bytes=0 if workspace is None else workspace.numel() * workspace.element_size(),
                             block_num=block_num, d_type=d_type)
    _check("cb200_grouped_quant_matmul_slice_k",
           load().cb200_grouped_quant_matmul_slice_k(ctypes.byref(args), _stream(stream)))


W4A8_SPLIT_K = 1  # flags: split the K range over a CTA cluster (faster, fp32 sums reassociated)


def _w4a8_args(a, w_packed, weight_scale, per_token, d, m, n, k, group_size, flags, d_type, pack_axis, workspace):
    return W4A8MatmulArgs(m=m, n=n, k=k, group_size=group_size, a=_p(a), w_packed=_p(w_packed),
                          weight_scale=_p(weight_scale), per_token_scale=_p(per_token), d=_p(d),
                          workspace=_p(workspace),
                          workspace_bytes=0 if workspace is None else workspace.numel() * workspace.element_size(),
                          block_num=0, flags=flags, d_type=d_type, pack_axis=pack_axis)


def w4a8_matmul_workspace_size(m, n, k, group_size, pack_axis=W4_PACKED_ALONG_K, aligned=True):
    """Bytes the call needs (0 on the fast path). `aligned`: the operand pointers are 16-byte aligned."""
    ptr = 256 if aligned else 257
    args = W4A8MatmulArgs(m=m, n=n, k=k, group_size=group_size, a=ptr, w_packed=ptr, weight_scale=256,
                          per_token_scale=256, d=256, pack_axis=pack_axis)
    return int(load().cb200_w4a8_matmul_workspace_size(ctypes.byref(args)))


def w4a8_matmul(a, w_packed, weight_scale, per_token, d, m, n, k, group_size, stream=None, split_k=False,
                static_weights=False, d_type=DTYPE_BF16, pack_axis=W4_PACKED_ALONG_K, workspace=None):
    flags = (W4A8_SPLIT_K if split_k else 0) | (FLAG_STATIC_WEIGHTS if static_weights else 0)
    args = _w4a8_args(a, w_packed, weight_scale, per_token, d, m, n, k, group_size, flags, d_type, pack_axis, workspace)
    _check("cb200_w4a8_matmul", load().cb200_w4a8_matmul(ctypes.byref(args), _stream(stream)))


def _mx_args(a, b, scale_a, scale_b, d, m, n, k, fmt, workspace, layout_a, layout_b, out_f32):
    return MxMatmulArgs(m=m, n=n, k=k, format=fmt, layout_a=layout_a, layout_b=layout_b, a=_p(a), b=_p(b),
                        scale_a=_p(scale_a), scale_b=_p(scale_b), d=_p(d), workspace=_p(workspace),
                        workspace_bytes=0 if workspace is None else workspace.numel() * workspace.element_size(),
                        block_num=0, flags=MX_OUT_F32 if out_f32 else 0)


def mx_matmul_workspace_size(m, n, k, fmt, layout_a=ROW_MAJOR, layout_b=COLUMN_MAJOR):
    args = MxMatmulArgs(m=m, n=n, k=k, format=fmt, layout_a=layout_a, layout_b=layout_b, a=256, b=256,
                        scale_a=256, scale_b=256, d=256)
    return int(load().cb200_mx_matmul_workspace_size(ctypes.byref(args)))


def mx_matmul(a, b, scale_a, scale_b, d, m, n, k, fmt, workspace, stream=None, layout_a=ROW_MAJOR,
              layout_b=COLUMN_MAJOR, out_f32=False):
    """a: [m][k] elements, or [k][m] with layout_a = COLUMN_MAJOR; b: [n][k] (column-major B), or [k][n] with
    layout_b = ROW_MAJOR; E2M1: two elements per byte along the contiguous axis.  Scales follow the operand:
    [rows][KS] bytes, or [KS/2][rows][2] for an operand stored with k first (KS = even number of 32-blocks).
    workspace: a CUDA byte tensor of at least mx_matmul_workspace_size bytes."""
    args = _mx_args(a, b, scale_a, scale_b, d, m, n, k, fmt, workspace, layout_a, layout_b, out_f32)
    _check("cb200_mx_matmul", load().cb200_mx_matmul(ctypes.byref(args), _stream(stream)))


def mx_matmul_static(a, b, scale_a, scale_b, d, m, n, k, fmt, stream=None, layout_a=ROW_MAJOR,
                     layout_b=COLUMN_MAJOR, out_f32=False):
    """cb200_mx_matmul_static: as mx_matmul, scratch inside the library image, no workspace argument."""
    args = _mx_args(a, b, scale_a, scale_b, d, m, n, k, fmt, None, layout_a, layout_b, out_f32)
    _check("cb200_mx_matmul_static", load().cb200_mx_matmul_static(ctypes.byref(args), _stream(stream)))


def _mx_grouped_args(a, b, group_list, scale_a, scale_b, d, m, n, k, group_count, fmt, workspace, layout_b,
                     group_list_type, group_list_kind, out_f32):
    return MxGroupedMatmulArgs(m=m, n=n, k=k, group_count=group_count, format=fmt, layout_b=layout_b,
                               group_list_type=group_list_type, group_list_kind=group_list_kind, a=_p(a), b=_p(b),
                               group_list=_p(group_list), scale_a=_p(scale_a), scale_b=_p(scale_b), d=_p(d),
                               workspace=_p(workspace),
                               workspace_bytes=0 if workspace is None else workspace.numel() * workspace.element_size(),
                               block_num=0, flags=MX_OUT_F32 if out_f32 else 0)


def mx_grouped_matmul_workspace_size(m, n, k, group_count, fmt, layout_b=COLUMN_MAJOR):
    args = MxGroupedMatmulArgs(m=m, n=n, k=k, group_count=group_count, format=fmt, layout_b=layout_b, a=256, b=256,
                               group_list=256, scale_a=256, scale_b=256, d=256)
    return int(load().cb200_mx_grouped_matmul_slice_m_workspace_size(ctypes.byref(args)))


def mx_grouped_matmul(a, b, group_list, scale_a, scale_b, d, m, n, k, group_count, fmt, workspace, stream=None,
                      layout_b=COLUMN_MAJOR, group_list_type=GROUP_LIST_INT64, group_list_kind=GROUP_LIST_SIZES,
                      out_f32=False):
    """Grouped slice-M MX matmul: a [m][k], b [G][n][k] (or [G][k][n] with layout_b = ROW_MAJOR), group_list the
    groups' row counts (or prefix sums), scales as for mx_matmul with a leading group axis on scale_b."""
    args = _mx_grouped_args(a, b, group_list, scale_a, scale_b, d, m, n, k, group_count, fmt, workspace, layout_b,
                            group_list_type, group_list_kind, out_f32)
    _check("cb200_mx_grouped_matmul_slice_m",
           load().cb200_mx_grouped_matmul_slice_m(ctypes.byref(args), _stream(stream)))


def mx_grouped_swiglu_quant_workspace_size(m, n, k, group_count, layout_b=COLUMN_MAJOR):
    args = MxGroupedSwigluQuantArgs(m=m, n=n, k=k, group_count=group_count, layout_b=layout_b, a=256, b=256,
                                    group_list=256, scale_a=256, scale_b=256, q=256, q_scale=256)
    return int(load().cb200_mx_grouped_matmul_slice_m_swiglu_mx_quant_workspace_size(ctypes.byref(args)))


def mx_grouped_swiglu_quant(a, b, group_list, scale_a, scale_b, q, q_scale, m, n, k, group_count, workspace,
                            stream=None, layout_b=COLUMN_MAJOR, group_list_type=GROUP_LIST_INT64,
                            group_list_kind=GROUP_LIST_SIZES):
    """Grouped slice-M MXFP8 matmul + SwiGLU + MX quantisation: q [m][n/2] E4M3 bytes, q_scale [m][n/64] E8M0."""
    args = MxGroupedSwigluQuantArgs(
        m=m, n=n, k=k, group_count=group_count, layout_b=layout_b, group_list_type=group_list_type,
        group_list_kind=group_list_kind, flags=0, a=_p(a), b=_p(b), group_list=_p(group_list), scale_a=_p(scale_a),
        scale_b=_p(scale_b), q=_p(q), q_scale=_p(q_scale), workspace=_p(workspace),
        workspace_bytes=0 if workspace is None else workspace.numel() * workspace.element_size(), block_num=0)
    _check("cb200_mx_grouped_matmul_slice_m_swiglu_mx_quant",
           load().cb200_mx_grouped_matmul_slice_m_swiglu_mx_quant(ctypes.byref(args), _stream(stream)))


ROUTING_DETERMINISTIC = 1


def mx_grouped_finalize_routing_workspace_size(m, n, k, group_count, batch, layout_b=COLUMN_MAJOR, deterministic=False):
    args = MxGroupedFinalizeRoutingArgs(m=m, n=n, k=k, group_count=group_count, layout_b=layout_b, batch=batch, a=256,
                                        b=256, group_list=256, scale_a=256, scale_b=256, logit=256, row_index=256,
                                        out=256, flags=ROUTING_DETERMINISTIC if deterministic else 0)
    return int(load().cb200_mx_grouped_matmul_finalize_routing_workspace_size(ctypes.byref(args)))


def mx_grouped_finalize_routing(a, b, group_list, scale_a, scale_b, logit, row_index, out, m, n, k, group_count, batch,
                                workspace, bias=None, shared_input=None, shared_rows=0, shared_offset=0,
                                shared_weight=0.0, stream=None, layout_b=COLUMN_MAJOR,
                                group_list_type=GROUP_LIST_INT64, group_list_kind=GROUP_LIST_SIZES,
                                row_index_type=GROUP_LIST_INT64, deterministic=False):
    """Grouped slice-M MXFP8 matmul + finalize routing: out [batch][n] fp32 = shared contribution +
    sum over rows p of logit[p] * (C[p] + bias[group]) at row row_index[p]."""
    args = MxGroupedFinalizeRoutingArgs(
        m=m, n=n, k=k, group_count=group_count, layout_b=layout_b, group_list_type=group_list_type,
        group_list_kind=group_list_kind, row_index_type=row_index_type, batch=batch, shared_rows=shared_rows,
        shared_offset=shared_offset, shared_weight=shared_weight, a=_p(a), b=_p(b), group_list=_p(group_list),
        scale_a=_p(scale_a), scale_b=_p(scale_b), logit=_p(logit), row_index=_p(row_index), bias=_p(bias),
        shared_input=_p(shared_input), out=_p(out), workspace=_p(workspace),
        workspace_bytes=0 if workspace is None else workspace.numel() * workspace.element_size(), block_num=0,
        flags=ROUTING_DETERMINISTIC if deterministic else 0)
    _check("cb200_mx_grouped_matmul_finalize_routing",
           load().cb200_mx_grouped_matmul_finalize_routing(ctypes.byref(args), _stream(stream)))


def mx_quantize(x, q, scale, rows, k, fmt, x_type=DTYPE_F32, x_pitch=0, stream=None):
    """x: fp32 / bf16 [rows][k] -> q codes ([rows][k] bytes, E2M1 [rows][ceil(k/2)]) and scale [rows][KS] bytes."""
    args = MxQuantizeArgs(rows=rows, k=k, format=fmt, x_type=x_type, x_pitch=x_pitch, x=_p(x), q=_p(q), scale=_p(scale))
    _check("cb200_mx_quantize", load().cb200_mx_quantize(ctypes.byref(args), _stream(stream)))


def _host_args(a_host, group_list_host, per_token_host, d_host, b, scale, m, n, k, group_count, layout_b, chunks,
               workspace):
    return GroupedQuantMatmulHostArgs(
        m=m, n=n, k=k, group_count=group_count, layout_b=layout_b, chunks=chunks, a_host=_p(a_host),
        group_list_host=_p(group_list_host), per_token_host=_p(per_token_host), d_host=_p(d_host), b=_p(b),
        scale=_p(scale), workspace=_p(workspace),
        workspace_bytes=0 if workspace is None else workspace.numel() * workspace.element_size())


def grouped_quant_matmul_host_workspace_size(m, n, k, group_count, chunks=0):
    args = GroupedQuantMatmulHostArgs(m=m, n=n, k=k, group_count=group_count, layout_b=ROW_MAJOR, chunks=chunks)
    return int(load().cb200_grouped_quant_matmul_slice_m_host_workspace_size(ctypes.byref(args)))


def grouped_quant_matmul_host(a_host, group_list_host, per_token_host, d_host, b, scale, m, n, k, group_count,
                              workspace, layout_b=ROW_MAJOR, chunks=0, stream=None):
    """Host-resident A / per-token scales / int64 group list / D (CPU tensors, pinned for overlap); b, scale and
    workspace are CUDA tensors."""
    args = _host_args(a_host, group_list_host, per_token_host, d_host, b, scale, m, n, k, group_count, layout_b,
                      chunks, workspace)
    _check("cb200_grouped_quant_matmul_slice_m_host",
           load().cb200_grouped_quant_matmul_slice_m_host(ctypes.byref(args), _stream(stream)))


def quantize_per_token_int8(x, q, scale, rows, k, x_type=DTYPE_F32, x_pitch=0, stream=None):
    """x: fp32 / bf16 [rows][k] -> q int8 [rows][k] and scale fp32 [rows] (amax / 127), the A operand and the
    per-token scale of the W8A8 entry points."""
    args = QuantizeInt8Args(rows=rows, k=k, x_type=x_type, reserved=0, x_pitch=x_pitch, x=_p(x), q=_p(q), scale=_p(scale))
    _check("cb200_quantize_per_token_int8", load().cb200_quantize_per_token_int8(ctypes.byref(args), _stream(stream)))



# ---- routing, dispatch, combine and the NVFP4 format
ROUTE_SOFTMAX, ROUTE_SIGMOID = 0, 1
ROUTE_GROUP_MAX, ROUTE_GROUP_TOP2_SUM = 0, 1
ROUTE_RENORMALIZE = 1
DISPATCH_INDEX, DISPATCH_COPY, DISPATCH_INT8, DISPATCH_MX_E4M3, DISPATCH_NVFP4 = 0, 1, 2, 3, 4
NVFP4_SCALES_ROWS, NVFP4_SCALES_TILED = 0, 1
NVFP4_SWIGLU = 1
_FLOAT_BYTES = {DTYPE_F32: 4, DTYPE_BF16: 2, DTYPE_F16: 2}


class MoeRouteArgs(ctypes.Structure):
    _fields_ = [
        ("tokens", _u32), ("experts", _u32), ("top_k", _u32), ("score", _u32), ("groups", _u32), ("groups_kept", _u32),
        ("group_score", _u32), ("flags", _u32), ("logits_type", _u32), ("scaling", ctypes.c_float),
        ("logits_pitch", _u64), ("logits", _vp), ("bias", _vp), ("token_count", _vp), ("weights", _vp), ("ids", _vp),
    ]


class MoeDispatchArgs(ctypes.Structure):
    _fields_ = [
        ("tokens", _u32), ("experts", _u32), ("top_k", _u32), ("k", _u32), ("format", _u32), ("x_type", _u32),
        ("expert_begin", ctypes.c_int32), ("group_list_type", _u32), ("group_list_kind", _u32),
        ("row_index_type", _u32), ("x_pitch", _u64), ("x", _vp), ("ids", _vp), ("weights", _vp), ("tensor_scale", _vp),
        ("q", _vp), ("scale", _vp), ("group_list", _vp), ("position", _vp), ("row_index", _vp), ("row_weight", _vp),
        ("workspace", _vp), ("workspace_bytes", _u64),
    ]


class MoeCombineArgs(ctypes.Structure):
    _fields_ = [
        ("tokens", _u32), ("top_k", _u32), ("n", _u32), ("rows", _u32), ("d_type", _u32), ("out_type", _u32),
        ("shared_weight", ctypes.c_float), ("reserved", _u32), ("d", _vp), ("position", _vp), ("weights", _vp),
        ("shared", _vp), ("out", _vp),
    ]


class Nvfp4QuantizeArgs(ctypes.Structure):
    _fields_ = [
        ("rows", _u32), ("k", _u32), ("x_type", _u32), ("scale_layout", _u32), ("flags", _u32),
        ("row_count_type", _u32), ("x_pitch", _u64), ("x", _vp), ("tensor_scale", _vp), ("row_count", _vp), ("q", _vp),
        ("scale", _vp),
    ]


class Nvfp4MatmulArgs(ctypes.Structure):
    _fields_ = [
        ("m", _u32), ("n", _u32), ("k", _u32), ("scale_a_layout", _u32), ("scale_b_layout", _u32), ("d_type", _u32),
        ("a", _vp), ("b", _vp), ("scale_a", _vp), ("scale_b", _vp), ("alpha", _vp), ("d", _vp), ("workspace", _vp),
        ("workspace_bytes", _u64), ("block_num", _u32), ("flags", _u32),
    ]


class Nvfp4GroupedMatmulArgs(ctypes.Structure):
    _fields_ = [
        ("m", _u32), ("n", _u32), ("k", _u32), ("group_count", _u32), ("scale_b_layout", _u32), ("group_list_type", _u32),
        ("group_list_kind", _u32), ("d_type", _u32), ("a", _vp), ("b", _vp), ("group_list", _vp), ("scale_a", _vp),
        ("scale_b", _vp), ("alpha", _vp), ("d", _vp), ("workspace", _vp), ("workspace_bytes", _u64), ("block_num", _u32),
        ("flags", _u32),
    ]


_prepared = {}


def _function(name, args_t, result=ctypes.c_int):
    """The library's function `name` with its argument types set (looked up once)."""
    fn = _prepared.get(name)
    if fn is None:
        fn = getattr(load(), name)
        fn.argtypes = [ctypes.POINTER(args_t)] + ([_vp] if result is ctypes.c_int and not name.endswith("_can_implement") else [])
        fn.restype = result
        _prepared[name] = fn
    return fn


def _device(t, what):
    """Index of the device of a CUDA tensor."""
    if t is None or t.get_device() < 0:
        raise ValueError(f"{what} must be a CUDA tensor")
    return t.get_device()


def _sizes(bits, *values):
    """Refuses sizes that the library's 32-bit fields would not hold as they are; bits: the values' bitwise or, which has
    a sign or a bit from 31 up when one of them has."""
    if bits >> 31:
        raise ValueError(f"sizes must lie in [0, 2^31), got {values}")


def _buffer(t, nbytes, what, device, itemsize=0):
    """Address of a tensor of that device used as a raw buffer of at least `nbytes` bytes; None stays None.  With an
    itemsize, a buffer of another size has to have elements of that many bytes (or one: raw bytes), which refuses a tensor
    of the right shape and the wrong type."""
    if t is None:
        return None
    if t.get_device() != device or not t.is_contiguous():
        raise ValueError(f"{what} must be a contiguous tensor of device {device}")
    have = t.nbytes
    if have != nbytes:
        if have < nbytes:
            raise ValueError(f"{what} holds {have} bytes, {nbytes} are needed")
        if itemsize and t.itemsize != itemsize and t.itemsize != 1:
            raise ValueError(f"{what} must have elements of {itemsize} bytes, not {t.dtype}")
    return t.data_ptr()


def _rows(t, rows, width, pitch, elem, what, device):
    """As _buffer, for `rows` rows of `width` elements with `pitch` elements between them (a view with strided rows is
    taken: only the storage behind its first element has to be long enough)."""
    if not pitch:
        return _buffer(t, rows * width * elem, what, device, elem)
    if t is None:
        return None
    if t.get_device() != device:
        raise ValueError(f"{what} must be a tensor of device {device}")
    if t.itemsize != elem and t.itemsize != 1:
        raise ValueError(f"{what} must have elements of {elem} bytes, not {t.dtype}")
    need = ((rows - 1) * pitch + width) * elem if rows and width else 0
    have = t.untyped_storage().nbytes() - t.storage_offset() * t.itemsize
    if have < need:
        raise ValueError(f"{what} holds {have} bytes, {need} are needed")
    return t.data_ptr()


def _enqueue(name, args, device, stream):
    """Calls the library on that device, on `stream` or the device's current stream."""
    import torch
    fn = _prepared.get(name) or _function(name, type(args))
    handle = torch._C._cuda_getCurrentRawStream(device) if stream is None else stream.cuda_stream
    if torch.cuda.current_device() == device:
        _check(name, fn(ctypes.byref(args), handle))
    else:
        with torch.cuda.device(device):
            _check(name, fn(ctypes.byref(args), handle))


def _float_bytes(type_code, what):
    if type_code not in _FLOAT_BYTES:
        raise ValueError(f"{what} must be DTYPE_F32, DTYPE_BF16 or DTYPE_F16")
    return _FLOAT_BYTES[type_code]


def moe_route(logits, weights, ids, tokens, experts, top_k, score=ROUTE_SOFTMAX, bias=None, groups=1, groups_kept=None,
              group_score=ROUTE_GROUP_MAX, renormalize=True, scaling=1.0, logits_type=DTYPE_F32, logits_pitch=0,
              token_count=None, stream=None):
    """logits [tokens][experts] -> weights fp32 and ids int32 [tokens][top_k], the experts with the largest scores (plus
    bias) of the best groups, ties to the lower index; id -1 and weight 0 where no expert is left."""
    dev = _device(logits, "logits")
    _sizes(tokens | experts | top_k | groups | logits_pitch, tokens, experts, top_k, groups, logits_pitch)
    out = tokens * top_k * 4
    args = MoeRouteArgs(tokens, experts, top_k, score, groups, groups if groups_kept is None else groups_kept,
                        group_score, ROUTE_RENORMALIZE if renormalize else 0, logits_type, scaling, logits_pitch,
                        _rows(logits, tokens, experts, logits_pitch, _float_bytes(logits_type, "logits_type"), "logits",
                              dev),
                        _buffer(bias, experts * 4, "bias", dev, 4), _buffer(token_count, 4, "token_count", dev, 4),
                        _buffer(weights, out, "weights", dev, 4), _buffer(ids, out, "ids", dev, 4))
    _enqueue("cb200_moe_route", args, dev, stream)


def moe_dispatch_workspace_size(tokens, experts, top_k):
    args = MoeDispatchArgs(tokens=tokens, experts=experts, top_k=top_k, format=DISPATCH_INDEX, ids=256, position=256,
                           group_list=256)
    return int(_function("cb200_moe_dispatch_workspace_size", MoeDispatchArgs, _u64)(ctypes.byref(args)))


def _dispatch_sizes(rows, k, fmt, x_bytes):
    """Bytes of q and of scale that `rows` dispatched rows take."""
    if fmt == DISPATCH_COPY:
        return rows * k * x_bytes, 0
    if fmt == DISPATCH_INT8:
        return rows * k, rows * 4
    if fmt == DISPATCH_MX_E4M3:
        return rows * k, rows * ((k // 32 + 1) // 2 * 2)
    if fmt == DISPATCH_NVFP4:
        return rows * (k // 2), rows * (k // 16)
    return 0, 0


def moe_dispatch(x, ids, weights, group_list, position, tokens, experts, top_k, k, fmt, q=None, scale=None,
                 row_index=None, row_weight=None, x_type=DTYPE_BF16, x_pitch=0, tensor_scale=None, workspace=None,
                 expert_begin=0, group_list_type=GROUP_LIST_INT64, group_list_kind=GROUP_LIST_PREFIX_SUMS,
                 row_index_type=GROUP_LIST_INT32, stream=None):
    """ids, weights [tokens][top_k] of a router -> rows sorted by expert: group_list [experts], position [tokens][top_k]
    (row of each pair, -1 when dropped), row_index / row_weight [tokens * top_k], and x [tokens][k] written to its rows
    of q / scale in the format `fmt`.  workspace: moe_dispatch_workspace_size bytes."""
    dev = _device(ids, "ids")
    _sizes(tokens | experts | top_k | k | x_pitch, tokens, experts, top_k, k, x_pitch)
    rows = tokens * top_k
    x_bytes = _float_bytes(x_type, "x_type")
    q_bytes, scale_bytes = _dispatch_sizes(rows, k, fmt, x_bytes)
    index_bytes = 8 if row_index_type == GROUP_LIST_INT64 else 4
    list_bytes = 8 if group_list_type == GROUP_LIST_INT64 else 4
    args = MoeDispatchArgs(
        tokens, experts, top_k, k, fmt, x_type, expert_begin, group_list_type, group_list_kind, row_index_type, x_pitch,
        None if fmt == DISPATCH_INDEX else _rows(x, tokens, k, x_pitch, x_bytes, "x", dev),
        _buffer(ids, rows * 4, "ids", dev, 4), _buffer(weights, rows * 4, "weights", dev, 4),
        _buffer(tensor_scale, 4, "tensor_scale", dev), _buffer(q, q_bytes, "q", dev),
        _buffer(scale, scale_bytes, "scale", dev),
        _buffer(group_list, experts * list_bytes, "group_list", dev, list_bytes),
        _buffer(position, rows * 4, "position", dev, 4),
        _buffer(row_index, rows * index_bytes, "row_index", dev, index_bytes),
        _buffer(row_weight, rows * 4, "row_weight", dev, 4), _buffer(workspace, 0, "workspace", dev),
        0 if workspace is None else workspace.nbytes)
    _enqueue("cb200_moe_dispatch", args, dev, stream)


def moe_combine(d, position, weights, out, tokens, n, top_k, rows=None, d_type=DTYPE_BF16, out_type=DTYPE_BF16,
                shared=None, shared_weight=1.0, stream=None):
    """out[t] = shared_weight * shared[t] + sum_j weights[t][j] * d[position[t][j]], d [rows][n] (rows: tokens * top_k
    unless given), slots with a negative position skipped."""
    dev = _device(d, "d")
    rows = tokens * top_k if rows is None else rows
    _sizes(tokens | n | top_k | rows, tokens, n, top_k, rows)
    d_elem, out_elem = _float_bytes(d_type, "d_type"), _float_bytes(out_type, "out_type")
    out_bytes = tokens * n * out_elem
    args = MoeCombineArgs(tokens, top_k, n, rows, d_type, out_type, shared_weight, 0,
                          _buffer(d, rows * n * d_elem, "d", dev, d_elem),
                          _buffer(position, tokens * top_k * 4, "position", dev, 4),
                          _buffer(weights, tokens * top_k * 4, "weights", dev, 4),
                          _buffer(shared, out_bytes, "shared", dev, out_elem),
                          _buffer(out, out_bytes, "out", dev, out_elem))
    _enqueue("cb200_moe_combine", args, dev, stream)


def nvfp4_tiled_scale_bytes(rows, k):
    """Bytes of a tiled scale array of rows x k elements."""
    return (rows + 127) // 128 * ((k + 63) // 64) * 512


def nvfp4_quantize(x, q, scale, rows, k, tensor_scale, x_type=DTYPE_BF16, x_pitch=0, scale_layout=NVFP4_SCALES_ROWS,
                   swiglu=False, row_count=None, row_count_type=GROUP_LIST_INT64, stream=None):
    """x [rows][k] (with swiglu [rows][2k]: act next to gate) -> q [rows][k/2] bytes and E4M3 scales by rows ([rows][k/16]
    bytes) or tiled (nvfp4_tiled_scale_bytes bytes), in units of the device scalar tensor_scale."""
    dev = _device(x, "x")
    _sizes(rows | k | x_pitch, rows, k, x_pitch)
    width = 2 * k if swiglu else k
    count_bytes = 8 if row_count_type == GROUP_LIST_INT64 else 4
    scale_bytes = nvfp4_tiled_scale_bytes(rows, k) if scale_layout == NVFP4_SCALES_TILED else rows * (k // 16)
    args = Nvfp4QuantizeArgs(
        rows, k, x_type, scale_layout, NVFP4_SWIGLU if swiglu else 0, row_count_type, x_pitch,
        _rows(x, rows, width, x_pitch, _float_bytes(x_type, "x_type"), "x", dev),
        _buffer(tensor_scale, 4, "tensor_scale", dev),
        _buffer(row_count, count_bytes, "row_count", dev, count_bytes),
        _buffer(q, rows * (k // 2), "q", dev), _buffer(scale, scale_bytes, "scale", dev))
    _enqueue("cb200_nvfp4_quantize", args, dev, stream)


def _nvfp4_scale_bytes(rows, k, layout):
    return nvfp4_tiled_scale_bytes(rows, k) if layout == NVFP4_SCALES_TILED else rows * (k // 16)


def nvfp4_matmul_workspace_size(m, n, k, scale_a_layout=NVFP4_SCALES_ROWS, scale_b_layout=NVFP4_SCALES_ROWS):
    args = Nvfp4MatmulArgs(m=m, n=n, k=k, scale_a_layout=scale_a_layout, scale_b_layout=scale_b_layout, a=256, b=256,
                           scale_a=256, scale_b=256, d=256)
    return int(_function("cb200_nvfp4_matmul_workspace_size", Nvfp4MatmulArgs, _u64)(ctypes.byref(args)))


def nvfp4_matmul(a, b, scale_a, scale_b, d, m, n, k, workspace=None, alpha=None, scale_a_layout=NVFP4_SCALES_ROWS,
                 scale_b_layout=NVFP4_SCALES_ROWS, d_type=DTYPE_BF16, stream=None, block_num=0):
    """a [m][k/2], b [n][k/2] packed E2M1 with E4M3 scales by rows or tiled -> d [m][n] = alpha * a @ b^T.  alpha: device
    scalar (the product of the tensor scales); workspace: nvfp4_matmul_workspace_size bytes."""
    dev = _device(a, "a")
    _sizes(m | n | k | block_num, m, n, k, block_num)
    elem = _float_bytes(d_type, "d_type")
    args = Nvfp4MatmulArgs(
        m, n, k, scale_a_layout, scale_b_layout, d_type, _buffer(a, m * (k // 2), "a", dev), _buffer(b, n * (k // 2), "b", dev),
        _buffer(scale_a, _nvfp4_scale_bytes(m, k, scale_a_layout), "scale_a", dev),
        _buffer(scale_b, _nvfp4_scale_bytes(n, k, scale_b_layout), "scale_b", dev), _buffer(alpha, 4, "alpha", dev, 4),
        _buffer(d, m * n * elem, "d", dev, elem), _buffer(workspace, 0, "workspace", dev),
        0 if workspace is None else workspace.nbytes, block_num, 0)
    _enqueue("cb200_nvfp4_matmul", args, dev, stream)


def nvfp4_grouped_matmul_workspace_size(m, n, k, group_count, scale_b_layout=NVFP4_SCALES_ROWS):
    args = Nvfp4GroupedMatmulArgs(m=m, n=n, k=k, group_count=group_count, scale_b_layout=scale_b_layout, a=256, b=256,
                                  group_list=256, scale_a=256, scale_b=256, d=256)
    return int(_function("cb200_nvfp4_grouped_matmul_slice_m_workspace_size", Nvfp4GroupedMatmulArgs, _u64)(
        ctypes.byref(args)))


def nvfp4_grouped_matmul(a, b, group_list, scale_a, scale_b, d, m, n, k, group_count, workspace, alpha=None,
                         scale_b_layout=NVFP4_SCALES_ROWS, d_type=DTYPE_BF16, group_list_type=GROUP_LIST_INT64,
                         group_list_kind=GROUP_LIST_SIZES, stream=None, block_num=0):
    """Grouped slice-M NVFP4 matmul: a [m][k/2], b [G][n][k/2], scale_a by rows, scale_b by rows or tiled per group,
    alpha [G] on the device; rows past the last group are not written."""
    dev = _device(a, "a")
    _sizes(m | n | k | group_count | block_num, m, n, k, group_count, block_num)
    elem = _float_bytes(d_type, "d_type")
    list_bytes = 8 if group_list_type == GROUP_LIST_INT64 else 4
    args = Nvfp4GroupedMatmulArgs(
        m, n, k, group_count, scale_b_layout, group_list_type, group_list_kind, d_type, _buffer(a, m * (k // 2), "a", dev),
        _buffer(b, group_count * n * (k // 2), "b", dev),
        _buffer(group_list, group_count * list_bytes, "group_list", dev, list_bytes),
        _buffer(scale_a, m * (k // 16), "scale_a", dev),
        _buffer(scale_b, group_count * _nvfp4_scale_bytes(n, k, scale_b_layout), "scale_b", dev),
        _buffer(alpha, group_count * 4, "alpha", dev, 4), _buffer(d, m * n * elem, "d", dev, elem),
        _buffer(workspace, 0, "workspace", dev), 0 if workspace is None else workspace.nbytes, block_num, 0)
    _enqueue("cb200_nvfp4_grouped_matmul_slice_m", args, dev, stream)
