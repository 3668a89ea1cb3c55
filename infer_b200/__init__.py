"""infer_b200 — B200 (sm_100a) backend for Feather's quantized-linear hot path.

The product is ``libfth_b200.so`` (hand-written CUDA behind the C ABI declared in ``include/fth_b200.h``)
plus the C++17 adapter under ``infer_b200/adapter`` that registers it with Feather's ``KernelDispatcher``.
This module is the thin Python host side used by the tests and the benchmark: ctypes mirrors of the C
structs and helpers that take device pointers from torch tensors.  torch is used for device memory and
streams only.  There is no CPU path: if the library is missing, loading raises.
"""
from __future__ import annotations

import ctypes as C
import os

_HERE = os.path.dirname(os.path.abspath(__file__))
# FTH_B200_LIBRARY names another build of the same library (an instrumented or experimental one); default: the in-tree build
LIB_PATH = os.environ.get("FTH_B200_LIBRARY") or os.path.join(_HERE, "libfth_b200.so")

INT8, FP16, FP32, INT32, BF16, E4M3, E5M2 = 1, 3, 4, 5, 11, 12, 13
OP_FC, OP_MATMUL, OP_GEMM = 0, 1, 2
BIAS_NONE, BIAS_VECTOR, BIAS_MATRIX = 0, 1, 2
VARIANT_AUTO, VARIANT_SIMT, VARIANT_SKINNY, VARIANT_TCGEN05, VARIANT_STREAM = 0, 1, 2, 3, 4
OK, ERR_INVALID, ERR_UNSUPPORTED, ERR_CUDA, ERR_OVERFLOW, ERR_TIMEOUT, ERR_SCRATCH_LIMIT = 0, -1, -2, -3, -4, -5, -6

EXPORTS = [
    "fth_b200_abi_version", "fth_b200_last_variant", "fth_b200_launch_count", "fth_b200_reset_launch_count",
    "fth_b200_fp8_linear", "fth_b200_fp8_linear_supported", "fth_b200_fp8_linear_workspace_bytes",
    "fth_b200_device_status", "fth_b200_fp8_linear_noalloc", "fth_b200_noalloc_scratch_bytes",
    "fth_b200_int8_linear", "fth_b200_int8_linear_supported", "fth_b200_int8_linear_workspace_bytes",
    "fth_b200_int8_conv2d", "fth_b200_int8_conv2d_supported", "fth_b200_int8_conv2d_workspace_bytes",
    "fth_b200_int8_conv2d_packed_weight_bytes", "fth_b200_int8_conv2d_pack_weights",
    "fth_b200_int8_relu_table", "fth_b200_int8_lookup",
    "fth_b200_quantize_linear", "fth_b200_dequantize_linear", "fth_b200_cast",
    "fth_b200_quantize_linear_axis", "fth_b200_dequantize_linear_axis", "fth_b200_small_copy",
    "fth_b200_plan_create_fp8_linear", "fth_b200_plan_create_int8_linear", "fth_b200_plan_create_int8_conv2d",
    "fth_b200_plan_run", "fth_b200_plan_launch", "fth_b200_plan_input_bytes", "fth_b200_plan_output_bytes",
    "fth_b200_plan_destroy",
    "fth_b200_peer_buffer_create", "fth_b200_peer_buffer_open", "fth_b200_peer_buffer_close", "fth_b200_peer_buffer_destroy",
    "fth_b200_gather_sync", "fth_b200_gather_wait", "fth_b200_fp8_linear_argmax",
    "fth_b200_fp8_lm_head_argmax", "fth_b200_fp8_linear_fused", "fth_b200_fp8_linear_fused_supported", "fth_b200_qwen_rms_norm", "fth_b200_binary", "fth_b200_silu", "fth_b200_silu_mul",
    "fth_b200_rope_turns", "fth_b200_rope", "fth_b200_kv4_assign", "fth_b200_kv4_release", "fth_b200_kv4_append", "fth_b200_kv4_gather",
    "fth_b200_kv4_attention", "fth_b200_kv4_attention_supported", "fth_b200_kv4_attention_workspace_bytes",
]
BINARY_ADD, BINARY_MUL = 0, 1
ROPE_HALF, ROPE_INTERLEAVED = 0, 1
ROPE_SCALINGS = {"none": 0, "linear": 1, "ntk": 2, "yarn": 3, "banded": 4}
KV4_OK, KV4_NO_BLOCKS, KV4_TABLE_FULL, KV4_TOO_MANY_TOKENS, KV4_BAD_LENGTH, KV4_BAD_BLOCK = 0, 1, 2, 3, 4, 5


class Fp8LinearDesc(C.Structure):
    _fields_ = [
        ("dtype", C.c_int32), ("op", C.c_int32), ("m", C.c_int64), ("k", C.c_int64), ("n", C.c_int64),
        ("trans_b", C.c_int32), ("a_dtype", C.c_int32), ("out_dtype", C.c_int32), ("bias_mode", C.c_int32),
        ("a", C.c_void_p), ("w", C.c_void_p), ("bias", C.c_void_p), ("out", C.c_void_p), ("ldo", C.c_int64),
        ("a_scale", C.c_float), ("w_scale", C.c_float), ("bias_scale", C.c_float), ("out_scale", C.c_float),
        ("w_channel_scales", C.c_void_p), ("alpha", C.c_float), ("beta", C.c_float),
        ("workspace", C.c_void_p), ("workspace_bytes", C.c_size_t), ("variant", C.c_int32), ("weights_static", C.c_int32),
        ("gather_peers", C.c_int32), ("gather_out", C.c_void_p * 7),
        ("gather_world", C.c_int32), ("gather_rank", C.c_int32), ("gather_flags", C.c_void_p * 8), ("gather_multicast_out", C.c_void_p),
    ]


class Fp8LinearFusion(C.Structure):
    _fields_ = [
        ("prologue", C.c_int32), ("norm_weight_dtype", C.c_int32), ("norm_weight", C.c_void_p), ("norm_weight_offset", C.c_float),
        ("norm_epsilon", C.c_float), ("a2", C.c_void_p), ("residual", C.c_void_p), ("w2", C.c_void_p), ("w2_scale", C.c_float),
        ("out2", C.c_void_p), ("n2", C.c_int64), ("ldo2", C.c_int64), ("epilogue", C.c_int32), ("out_codes_scale", C.c_float),
        ("out_codes", C.c_void_p), ("ldo_codes", C.c_int64),
    ]


FUSE_NONE, FUSE_RMS_NORM, FUSE_SILU_MUL = 0, 1, 2
FUSE_OUT_NONE, FUSE_OUT_SILU_MUL = 0, 1


class Int8LinearDesc(C.Structure):
    _fields_ = [
        ("op", C.c_int32), ("m", C.c_int64), ("k", C.c_int64), ("n", C.c_int64), ("trans_b", C.c_int32),
        ("a_dtype", C.c_int32), ("out_dtype", C.c_int32), ("bias_mode", C.c_int32),
        ("a", C.c_void_p), ("w", C.c_void_p), ("bias", C.c_void_p), ("out", C.c_void_p), ("ldo", C.c_int64),
        ("a_scale", C.c_float), ("a_zp", C.c_int32), ("w_scales", C.c_void_p), ("w_zps", C.c_void_p),
        ("w_params", C.c_int64), ("w_zp_max_abs", C.c_int32), ("out_scale", C.c_float), ("out_zp", C.c_int32),
        ("alpha", C.c_float), ("beta", C.c_float), ("bias_max_abs", C.c_int64),
        ("workspace", C.c_void_p), ("workspace_bytes", C.c_size_t), ("variant", C.c_int32), ("weights_static", C.c_int32),
        ("gather_peers", C.c_int32), ("gather_out", C.c_void_p * 7),
        ("gather_world", C.c_int32), ("gather_rank", C.c_int32), ("gather_flags", C.c_void_p * 8), ("gather_multicast_out", C.c_void_p),
    ]


class Int8Conv2dDesc(C.Structure):
    _fields_ = [
        ("batch", C.c_int64), ("ic", C.c_int64), ("ih", C.c_int64), ("iw", C.c_int64), ("oc", C.c_int64),
        ("kh", C.c_int64), ("kw", C.c_int64),
        ("stride_h", C.c_int32), ("stride_w", C.c_int32), ("pad_h", C.c_int32), ("pad_w", C.c_int32),
        ("dilation_h", C.c_int32), ("dilation_w", C.c_int32), ("group", C.c_int32),
        ("x", C.c_void_p), ("w", C.c_void_p), ("bias", C.c_void_p), ("out", C.c_void_p),
        ("x_scale", C.c_float), ("x_zp", C.c_int32), ("w_scales", C.c_void_p), ("w_zps", C.c_void_p),
        ("w_params", C.c_int64), ("w_zp_max_abs", C.c_int32), ("out_scale", C.c_float), ("out_zp", C.c_int32),
        ("relu_lut", C.c_void_p), ("bias_max_abs", C.c_int64), ("workspace", C.c_void_p),
        ("workspace_bytes", C.c_size_t), ("weights_packed", C.c_int32), ("variant", C.c_int32), ("packed_w", C.c_void_p),
    ]


class RopeScaling(C.Structure):
    _fields_ = [("rotary_dim", C.c_int32), ("scaling", C.c_int32), ("base", C.c_double), ("factor", C.c_double), ("original", C.c_double),
                ("fast", C.c_double), ("slow", C.c_double)]


class RopeDesc(C.Structure):
    _fields_ = [
        ("dtype", C.c_int32), ("layout", C.c_int32), ("tokens", C.c_int64), ("head_dim", C.c_int32), ("rotary_dim", C.c_int32),
        ("q_heads", C.c_int32), ("k_heads", C.c_int32), ("q", C.c_void_p), ("q_out", C.c_void_p), ("k", C.c_void_p), ("k_out", C.c_void_p),
        ("ldq", C.c_int64), ("ldq_out", C.c_int64), ("ldk", C.c_int64), ("ldk_out", C.c_int64), ("positions", C.c_void_p),
        ("turns", C.c_void_p), ("amplitude", C.c_float),
    ]


class Kv4Cache(C.Structure):
    _fields_ = [("k_codes", C.c_void_p), ("v_codes", C.c_void_p), ("k_params", C.c_void_p), ("v_params", C.c_void_p), ("blocks", C.c_int64),
                ("block_size", C.c_int32), ("kv_heads", C.c_int32), ("head_dim", C.c_int32)]


class Kv4AssignDesc(C.Structure):
    _fields_ = [
        ("requests", C.c_int32), ("max_blocks", C.c_int32), ("block_size", C.c_int32), ("blocks", C.c_int64), ("tokens", C.c_int64),
        ("cached_lens", C.c_void_p), ("new_lens", C.c_void_p), ("free_blocks", C.c_void_p), ("free_count", C.c_void_p),
        ("free_count_out", C.c_void_p), ("block_table", C.c_void_p), ("total_lens", C.c_void_p), ("query_start", C.c_void_p),
        ("slots", C.c_void_p), ("positions", C.c_void_p), ("status", C.c_void_p),
    ]


class Kv4ReleaseDesc(C.Structure):
    _fields_ = [
        ("requests", C.c_int32), ("max_blocks", C.c_int32), ("block_size", C.c_int32), ("blocks", C.c_int64), ("lens", C.c_void_p),
        ("keep_lens", C.c_void_p), ("free_blocks", C.c_void_p), ("free_count", C.c_void_p), ("free_count_out", C.c_void_p),
        ("block_table", C.c_void_p), ("lens_out", C.c_void_p), ("status", C.c_void_p),
    ]


class Kv4AppendDesc(C.Structure):
    _fields_ = [("cache", Kv4Cache), ("dtype", C.c_int32), ("tokens", C.c_int64), ("k", C.c_void_p), ("v", C.c_void_p), ("ldk", C.c_int64),
                ("ldv", C.c_int64), ("slots", C.c_void_p), ("rope", C.c_void_p)]


class Kv4GatherDesc(C.Structure):
    _fields_ = [("cache", Kv4Cache), ("dtype", C.c_int32), ("tokens", C.c_int64), ("slots", C.c_void_p), ("k_out", C.c_void_p),
                ("v_out", C.c_void_p), ("ldk", C.c_int64), ("ldv", C.c_int64)]


class Kv4AttentionDesc(C.Structure):
    _fields_ = [
        ("cache", Kv4Cache), ("dtype", C.c_int32), ("requests", C.c_int32), ("tokens", C.c_int64), ("q_heads", C.c_int32),
        ("max_blocks", C.c_int32), ("max_query", C.c_int32), ("causal", C.c_int32), ("window", C.c_int32), ("scale", C.c_float),
        ("q", C.c_void_p), ("out", C.c_void_p), ("ldq", C.c_int64), ("ldo", C.c_int64), ("lse", C.c_void_p), ("block_table", C.c_void_p),
        ("total_lens", C.c_void_p), ("query_start", C.c_void_p), ("workspace", C.c_void_p), ("workspace_bytes", C.c_size_t),
    ]


_lib = None


def lib():
    """Loads libfth_b200.so; raises if it has not been built (there is no fallback)."""
    global _lib
    if _lib is None:
        if not os.path.exists(LIB_PATH):
            raise RuntimeError(
                f"{LIB_PATH} is missing: build it with `python -m infer_b200.build` (needs nvcc); "
                "this backend has no CPU or library fallback")
        handle = C.CDLL(LIB_PATH)
        handle.fth_b200_last_variant.restype = C.c_char_p
        handle.fth_b200_launch_count.restype = C.c_int64
        handle.fth_b200_int8_conv2d_workspace_bytes.restype = C.c_size_t
        handle.fth_b200_int8_conv2d_packed_weight_bytes.restype = C.c_size_t
        handle.fth_b200_fp8_linear_workspace_bytes.restype = C.c_size_t
        handle.fth_b200_int8_linear_workspace_bytes.restype = C.c_size_t
        handle.fth_b200_noalloc_scratch_bytes.restype = C.c_size_t
        handle.fth_b200_kv4_attention_workspace_bytes.restype = C.c_size_t
        handle.fth_b200_plan_input_bytes.restype = C.c_int64
        handle.fth_b200_plan_output_bytes.restype = C.c_int64
        handle.fth_b200_plan_input_bytes.argtypes = [C.c_void_p]
        handle.fth_b200_plan_output_bytes.argtypes = [C.c_void_p]
        handle.fth_b200_plan_destroy.argtypes = [C.c_void_p]
        handle.fth_b200_plan_destroy.restype = None
        handle.fth_b200_gather_sync.argtypes = [C.c_void_p, C.c_int32, C.c_int32, C.c_uint32, C.c_void_p]
        handle.fth_b200_gather_wait.argtypes = [C.c_void_p, C.c_int32, C.c_int32, C.c_void_p]
        handle.fth_b200_plan_run.argtypes = [C.c_void_p, C.c_void_p, C.c_void_p, C.c_void_p]
        handle.fth_b200_plan_launch.argtypes = [C.c_void_p, C.c_void_p, C.c_void_p, C.c_void_p]
        _lib = handle
    return _lib


class B200Error(RuntimeError):
    def __init__(self, code: int, what: str):
        super().__init__(f"{what} failed with status {code}")
        self.code = code


def check(code: int, what: str) -> None:
    if code != OK:
        raise B200Error(code, what)


def last_variant() -> str:
    return lib().fth_b200_last_variant().decode()


def ptr(t):
    """Device (or host) address of a torch tensor / numpy array / int / None."""
    if t is None:
        return None
    if isinstance(t, int):
        return t
    if hasattr(t, "data_ptr"):
        return t.data_ptr()
    return t.ctypes.data


def current_stream():
    import torch
    return C.c_void_p(torch.cuda.current_stream().cuda_stream)


def fp8_linear_desc(*, dtype, op, m, k, n, a, w, out, a_scale, w_scale, out_scale, trans_b=False, bias=None,
                    bias_mode=BIAS_NONE, bias_scale=1.0, alpha=1.0, beta=1.0, a_dtype=0, out_dtype=0, ldo=0,
                    w_channel_scales=None, workspace=None, workspace_bytes=0,
                    variant=VARIANT_AUTO, weights_static=False) -> Fp8LinearDesc:
    d = Fp8LinearDesc()
    d.dtype, d.op, d.m, d.k, d.n, d.trans_b = dtype, op, m, k, n, int(trans_b)
    d.a_dtype, d.out_dtype, d.bias_mode = a_dtype, out_dtype, bias_mode
    d.a, d.w, d.bias, d.out, d.ldo = ptr(a), ptr(w), ptr(bias), ptr(out), ldo
    d.a_scale, d.w_scale, d.bias_scale, d.out_scale = a_scale, w_scale, bias_scale, out_scale
    d.w_channel_scales = ptr(w_channel_scales)
    d.alpha, d.beta, d.variant, d.weights_static = alpha, beta, variant, int(weights_static)
    d.workspace, d.workspace_bytes = ptr(workspace), workspace_bytes
    return d


def int8_linear_desc(*, op, m, k, n, a, w, out, a_scale, a_zp, w_scales, w_zps, w_params, out_scale, out_zp,
                     trans_b=False, bias=None, bias_mode=BIAS_NONE, alpha=1.0, beta=1.0, a_dtype=0, out_dtype=0,
                     ldo=0, w_zp_max_abs=0, bias_max_abs=0, workspace=None, workspace_bytes=0,
                     variant=VARIANT_AUTO, weights_static=False) -> Int8LinearDesc:
    d = Int8LinearDesc()
    d.op, d.m, d.k, d.n, d.trans_b = op, m, k, n, int(trans_b)
    d.a_dtype, d.out_dtype, d.bias_mode = a_dtype, out_dtype, bias_mode
    d.a, d.w, d.bias, d.out, d.ldo = ptr(a), ptr(w), ptr(bias), ptr(out), ldo
    d.a_scale, d.a_zp, d.w_scales, d.w_zps, d.w_params = a_scale, a_zp, ptr(w_scales), ptr(w_zps), w_params
    d.w_zp_max_abs, d.out_scale, d.out_zp = w_zp_max_abs, out_scale, out_zp
    d.alpha, d.beta, d.bias_max_abs, d.variant = alpha, beta, bias_max_abs, variant
    d.weights_static = int(weights_static)
    d.workspace, d.workspace_bytes = ptr(workspace), workspace_bytes
    return d


def int8_conv2d_desc(*, batch, ic, ih, iw, oc, kh, kw, x, w, out, x_scale, x_zp, w_scales, w_zps, w_params,
                     out_scale, out_zp, bias=None, stride=(1, 1), pad=(1, 1), dil=(1, 1), group=1, relu_lut=None,
                     w_zp_max_abs=0, bias_max_abs=0, workspace=None, workspace_bytes=0, weights_packed=0,
                     variant=VARIANT_AUTO) -> Int8Conv2dDesc:
    d = Int8Conv2dDesc()
    d.batch, d.ic, d.ih, d.iw, d.oc, d.kh, d.kw = batch, ic, ih, iw, oc, kh, kw
    d.stride_h, d.stride_w, d.pad_h, d.pad_w = stride[0], stride[1], pad[0], pad[1]
    d.dilation_h, d.dilation_w, d.group = dil[0], dil[1], group
    d.x, d.w, d.bias, d.out = ptr(x), ptr(w), ptr(bias), ptr(out)
    d.x_scale, d.x_zp, d.w_scales, d.w_zps, d.w_params = x_scale, x_zp, ptr(w_scales), ptr(w_zps), w_params
    d.w_zp_max_abs, d.out_scale, d.out_zp = w_zp_max_abs, out_scale, out_zp
    d.relu_lut, d.bias_max_abs = ptr(relu_lut), bias_max_abs
    d.workspace, d.workspace_bytes, d.weights_packed, d.variant = ptr(workspace), workspace_bytes, weights_packed, variant
    return d


def fp8_linear(desc: Fp8LinearDesc, stream=None) -> None:
    check(lib().fth_b200_fp8_linear(C.byref(desc), stream or current_stream()), "fth_b200_fp8_linear")


def fp8_linear_fusion(*, prologue=FUSE_NONE, norm_weight=None, norm_weight_dtype=BF16, norm_weight_offset=0.0, norm_epsilon=1e-6, a2=None,
                      residual=None, w2=None, w2_scale=1.0, out2=None, n2=0, ldo2=0, epilogue=FUSE_OUT_NONE, out_codes=None,
                      out_codes_scale=1.0, ldo_codes=0) -> Fp8LinearFusion:
    f = Fp8LinearFusion()
    f.prologue, f.norm_weight_dtype, f.norm_weight = prologue, norm_weight_dtype, ptr(norm_weight)
    f.norm_weight_offset, f.norm_epsilon = norm_weight_offset, norm_epsilon
    f.a2, f.residual, f.w2, f.w2_scale, f.out2, f.n2, f.ldo2 = ptr(a2), ptr(residual), ptr(w2), w2_scale, ptr(out2), n2, ldo2
    f.epilogue = epilogue
    f.out_codes, f.out_codes_scale, f.ldo_codes = ptr(out_codes), out_codes_scale, ldo_codes
    return f


def fp8_linear_fused(desc: Fp8LinearDesc, fusion: Fp8LinearFusion, stream=None) -> None:
    check(lib().fth_b200_fp8_linear_fused(C.byref(desc), C.byref(fusion), stream or current_stream()), "fth_b200_fp8_linear_fused")


def int8_linear(desc: Int8LinearDesc, stream=None) -> None:
    check(lib().fth_b200_int8_linear(C.byref(desc), stream or current_stream()), "fth_b200_int8_linear")


def int8_conv2d(desc: Int8Conv2dDesc, stream=None) -> None:
    check(lib().fth_b200_int8_conv2d(C.byref(desc), stream or current_stream()), "fth_b200_int8_conv2d")


def cast(in_dtype, x, in_scale, out_dtype, out, out_scale, count, stream=None) -> None:
    check(lib().fth_b200_cast(C.c_int32(in_dtype), C.c_void_p(ptr(x)), C.c_float(in_scale), C.c_int32(out_dtype),
                              C.c_void_p(ptr(out)), C.c_float(out_scale), C.c_int64(count),
                              stream or current_stream()), "fth_b200_cast")


def quantize_linear(x_dtype, x, scales, zps, params, out, rows, channels, stream=None, inner=1) -> None:
    """x is [rows, channels, inner]; the parameters run along `channels` (inner = 1: the last axis)."""
    check(lib().fth_b200_quantize_linear_axis(C.c_int32(x_dtype), C.c_void_p(ptr(x)), C.c_void_p(ptr(scales)),
                                              C.c_void_p(ptr(zps)), C.c_int64(params), C.c_void_p(ptr(out)),
                                              C.c_int64(rows), C.c_int64(channels), C.c_int64(inner), stream or current_stream()),
          "fth_b200_quantize_linear_axis")


def dequantize_linear(x, scales, zps, params, out, to_dtype, rows, channels, stream=None, inner=1) -> None:
    check(lib().fth_b200_dequantize_linear_axis(C.c_void_p(ptr(x)), C.c_void_p(ptr(scales)), C.c_void_p(ptr(zps)),
                                                C.c_int64(params), C.c_void_p(ptr(out)), C.c_int32(to_dtype),
                                                C.c_int64(rows), C.c_int64(channels), C.c_int64(inner), stream or current_stream()),
          "fth_b200_dequantize_linear_axis")


def small_copy(dst, src, nbytes, stream=None) -> None:
    """A few KB between a page-locked host buffer and device memory, copied by the SMs on the stream."""
    check(lib().fth_b200_small_copy(C.c_void_p(ptr(dst)), C.c_void_p(ptr(src)), C.c_int64(nbytes), stream or current_stream()),
          "fth_b200_small_copy")


def int8_lookup(x, out, count, lut, stream=None) -> None:
    check(lib().fth_b200_int8_lookup(C.c_void_p(ptr(x)), C.c_void_p(ptr(out)), C.c_int64(count),
                                     C.c_void_p(ptr(lut)), stream or current_stream()), "fth_b200_int8_lookup")


def int8_relu_table(in_scale, in_zp, out_scale, out_zp):
    import numpy as np
    lut = np.empty(256, np.int8)
    check(lib().fth_b200_int8_relu_table(C.c_float(in_scale), C.c_int32(in_zp), C.c_float(out_scale),
                                         C.c_int32(out_zp), C.c_void_p(lut.ctypes.data)), "fth_b200_int8_relu_table")
    return lut


def qwen_rms_norm(x_dtype, x, weight_dtype, weight, weight_offset, epsilon, out_dtype, out, rows, hidden, stream=None) -> None:
    check(lib().fth_b200_qwen_rms_norm(C.c_int32(x_dtype), C.c_void_p(ptr(x)), C.c_int32(weight_dtype), C.c_void_p(ptr(weight)),
                                       C.c_float(weight_offset), C.c_float(epsilon), C.c_int32(out_dtype), C.c_void_p(ptr(out)),
                                       C.c_int64(rows), C.c_int64(hidden), stream or current_stream()), "fth_b200_qwen_rms_norm")


def binary(op, dtype, lhs, rhs, out, count, rhs_count=0, stream=None) -> None:
    check(lib().fth_b200_binary(C.c_int32(op), C.c_int32(dtype), C.c_void_p(ptr(lhs)), C.c_void_p(ptr(rhs)), C.c_void_p(ptr(out)),
                                C.c_int64(count), C.c_int64(rhs_count), stream or current_stream()), "fth_b200_binary")


def silu(dtype, x, out, count, stream=None) -> None:
    check(lib().fth_b200_silu(C.c_int32(dtype), C.c_void_p(ptr(x)), C.c_void_p(ptr(out)), C.c_int64(count),
                              stream or current_stream()), "fth_b200_silu")


def silu_mul(dtype, gate, up, out, count, stream=None) -> None:
    check(lib().fth_b200_silu_mul(C.c_int32(dtype), C.c_void_p(ptr(gate)), C.c_void_p(ptr(up)), C.c_void_p(ptr(out)), C.c_int64(count),
                                  stream or current_stream()), "fth_b200_silu_mul")


# ---- rotary positions, the 4-bit cache and its attention (include/fth_b200.h) -------------------------------------------
# The *_desc functions take torch tensors or device addresses.  A tensor must live on a GPU, the same one for all tensors of
# a descriptor; its row stride is taken from it unless a stride is given.  The calls run on that GPU, on its current stream
# unless one is given.

def _tensors(desc, **tensors):
    """Stores the addresses in the descriptor's fields, checks where the tensors are, and keeps them alive with it."""
    keep, device = [], None
    for name, t in tensors.items():
        if hasattr(t, "data_ptr"):
            if not t.is_cuda:
                raise ValueError(f"{name} is not on a GPU")
            if device is not None and t.device.index != device:
                raise ValueError(f"{name} is on cuda:{t.device.index}, other tensors on cuda:{device}")
            device = t.device.index
        keep.append(t)
        setattr(desc, name, ptr(t))
    desc._keep = getattr(desc, "_keep", []) + keep
    if device is not None:
        if getattr(desc, "_device", device) != device:
            raise ValueError(f"tensors on cuda:{device} and cuda:{desc._device}")
        desc._device = device
    return desc


def _dense(**tensors):
    for name, t in tensors.items():
        if hasattr(t, "is_contiguous") and not t.is_contiguous():
            raise ValueError(f"{name} is not contiguous")


_SIZES = {FP32: 4, FP16: 2, BF16: 2}
_NAMES = {FP32: "torch.float32", FP16: "torch.float16", BF16: "torch.bfloat16"}


def _rows(name, t, dtype, tokens, heads, head_dim, ld):
    """Row stride of [tokens, heads, head_dim] (or [tokens, heads * head_dim], or elements in a row); the rows lie inside the tensor.
    Bits held in integers may be of any type."""
    if t is None or not hasattr(t, "stride"):
        return ld
    if t.element_size() != _SIZES.get(dtype, t.element_size()):
        raise ValueError(f"{name} has {t.element_size()}-byte elements")
    if t.is_floating_point() and str(t.dtype) != _NAMES.get(dtype, str(t.dtype)):
        raise ValueError(f"{name} is {t.dtype}, not {_NAMES[dtype]}")
    row = heads * head_dim
    if ld == 0 and t.dim() >= 2:
        inner = t.stride(-1) == 1 or t.shape[-1] == 1
        if t.dim() == 3:
            inner = inner and (t.stride(1) == head_dim or t.shape[1] == 1) and t.shape[1] * t.shape[2] == row
        else:
            inner = inner and t.dim() == 2 and t.shape[1] == row
        if not inner or t.shape[0] < tokens or (tokens > 1 and t.stride(0) == 0):
            raise ValueError(f"{name}: expected [{tokens}, {heads}, {head_dim}] with heads {head_dim} apart, got {tuple(t.shape)}, strides {t.stride()}")
        if t.shape[0] > 1:
            ld = t.stride(0)
    span = 1 + sum((n - 1) * step for n, step in zip(t.shape, t.stride())) if t.numel() else 0
    need = (tokens - 1) * (ld or row) + row if tokens > 0 else 0
    if span < need:
        raise ValueError(f"{name}: {tokens} rows of {row}, {ld or row} apart, take {need} elements, the tensor holds {span}")
    return ld


def _count(name, t, count):
    if hasattr(t, "numel") and t.numel() < count:
        raise ValueError(f"{name} has {t.numel()} elements, needs {count}")
    if hasattr(t, "element_size") and t.element_size() != 4:
        raise ValueError(f"{name} has {t.element_size()}-byte elements, needs 4")


def _call(name, desc, stream):
    """Runs an entry point with the descriptor's GPU current."""
    call = getattr(desc, "_call", None)
    if call is None:  # what every call of the descriptor needs, looked up once
        import torch
        fn = getattr(lib(), name)
        fn.argtypes = [C.c_void_p, C.c_void_p]
        # the current stream's handle without a Stream object, which costs as much as the launch
        raw = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda device: torch.cuda.current_stream(device).cuda_stream)
        call = desc._call = (fn, C.byref(desc), torch.cuda, raw)
    fn, arg, cuda, raw = call
    device, now = getattr(desc, "_device", None), cuda.current_device()
    if device is None or now == device:
        code = fn(arg, stream or raw(now))
    else:
        with cuda.device(device):
            code = fn(arg, stream or raw(device))
    if code != OK:
        raise B200Error(code, name)


def rope_turns(rotary_dim, base=10000.0, scaling="none", factor=1.0, original=0.0, fast=0.0, slow=0.0):
    """Host table of turns per position (float64, [rotary_dim / 2]) and the amplitude; see fth_b200_rope_turns."""
    import numpy as np
    if scaling not in ROPE_SCALINGS:
        raise ValueError(f"scaling {scaling!r}: one of {sorted(ROPE_SCALINGS)}")
    s = RopeScaling(rotary_dim, ROPE_SCALINGS[scaling], base, factor, original, fast, slow)
    turns, amplitude = np.empty(max(rotary_dim // 2, 0), np.float64), C.c_float()
    check(lib().fth_b200_rope_turns(C.byref(s), C.c_void_p(turns.ctypes.data), C.byref(amplitude)), "fth_b200_rope_turns")
    return turns, amplitude.value


def rope_desc(*, dtype, layout, tokens, head_dim, rotary_dim, positions, turns, amplitude=1.0, q=None, q_out=None, q_heads=0, k=None,
              k_out=None, k_heads=0, ldq=0, ldq_out=0, ldk=0, ldk_out=0) -> RopeDesc:
    d = RopeDesc()
    d.dtype, d.layout, d.tokens, d.head_dim, d.rotary_dim = dtype, layout, tokens, head_dim, rotary_dim
    d.q_heads, d.k_heads, d.amplitude = q_heads, k_heads, amplitude
    d.ldq, d.ldq_out = _rows("q", q, dtype, tokens, q_heads, head_dim, ldq), _rows("q_out", q_out, dtype, tokens, q_heads, head_dim, ldq_out)
    d.ldk, d.ldk_out = _rows("k", k, dtype, tokens, k_heads, head_dim, ldk), _rows("k_out", k_out, dtype, tokens, k_heads, head_dim, ldk_out)
    _dense(positions=positions, turns=turns)
    _count("positions", positions, tokens)
    if hasattr(turns, "element_size") and (turns.element_size() != 8 or turns.numel() < rotary_dim // 2):
        raise ValueError(f"turns: needs {rotary_dim // 2} float64")
    return _tensors(d, q=q, q_out=q_out, k=k, k_out=k_out, positions=positions, turns=turns)


def rope(desc: RopeDesc, stream=None) -> None:
    _call("fth_b200_rope", desc, stream)


def kv4_cache(*, k_codes, v_codes, k_params, v_params, blocks, block_size, kv_heads, head_dim) -> Kv4Cache:
    c = Kv4Cache()
    c.blocks, c.block_size, c.kv_heads, c.head_dim = blocks, block_size, kv_heads, head_dim
    tensors = dict(k_codes=k_codes, v_codes=v_codes, k_params=k_params, v_params=v_params)
    _dense(**tensors)
    tokens = blocks * kv_heads * block_size
    for name, t in tensors.items():
        need = tokens * (head_dim // 2 if "codes" in name else 4)
        if hasattr(t, "numel") and t.numel() * t.element_size() < need:
            raise ValueError(f"{name} has {t.numel() * t.element_size()} bytes, needs {need}")
    return _tensors(c, **tensors)


def kv4_new_cache(torch, *, blocks, block_size, kv_heads, head_dim, device="cuda") -> Kv4Cache:
    """Allocates one layer's cache (its contents are arbitrary until they are written)."""
    codes, params = (blocks, kv_heads, block_size, head_dim // 2), (blocks, kv_heads, block_size)
    make = lambda shape, dtype: torch.zeros(shape, dtype=dtype, device=device)  # noqa: E731
    return kv4_cache(k_codes=make(codes, torch.uint8), v_codes=make(codes, torch.uint8), k_params=make(params, torch.int32),
                     v_params=make(params, torch.int32), blocks=blocks, block_size=block_size, kv_heads=kv_heads, head_dim=head_dim)


def _with_cache(d, cache):
    d.cache = cache
    d._keep = [cache]
    if hasattr(cache, "_device"):
        d._device = cache._device
    return d


def kv4_assign_desc(*, requests, max_blocks, block_size, blocks, tokens, cached_lens, new_lens, free_blocks, free_count, free_count_out,
                    block_table, total_lens, query_start, slots, positions, status) -> Kv4AssignDesc:
    d = Kv4AssignDesc()
    d.requests, d.max_blocks, d.block_size, d.blocks, d.tokens = requests, max_blocks, block_size, blocks, tokens
    t = dict(cached_lens=cached_lens, new_lens=new_lens, free_blocks=free_blocks, free_count=free_count, free_count_out=free_count_out,
             block_table=block_table, total_lens=total_lens, query_start=query_start, slots=slots, positions=positions, status=status)
    need = dict(cached_lens=requests, new_lens=requests, free_blocks=blocks, free_count=1, free_count_out=1, block_table=requests * max_blocks,
                total_lens=requests, query_start=requests + 1, slots=tokens, positions=tokens, status=2)
    _dense(**t)
    for name in t:
        _count(name, t[name], need[name])
    return _tensors(d, **t)


def kv4_assign(desc: Kv4AssignDesc, stream=None) -> None:
    _call("fth_b200_kv4_assign", desc, stream)


def kv4_release_desc(*, requests, max_blocks, block_size, blocks, lens, keep_lens, free_blocks, free_count, free_count_out, block_table,
                     lens_out, status) -> Kv4ReleaseDesc:
    d = Kv4ReleaseDesc()
    d.requests, d.max_blocks, d.block_size, d.blocks = requests, max_blocks, block_size, blocks
    t = dict(lens=lens, keep_lens=keep_lens, free_blocks=free_blocks, free_count=free_count, free_count_out=free_count_out,
             block_table=block_table, lens_out=lens_out, status=status)
    need = dict(lens=requests, keep_lens=requests, free_blocks=blocks, free_count=1, free_count_out=1, block_table=requests * max_blocks,
                lens_out=requests, status=2)
    _dense(**t)
    for name in t:
        _count(name, t[name], need[name])
    return _tensors(d, **t)


def kv4_release(desc: Kv4ReleaseDesc, stream=None) -> None:
    _call("fth_b200_kv4_release", desc, stream)


def kv4_append_desc(*, cache, dtype, tokens, k, v, slots, ldk=0, ldv=0, rope=None) -> Kv4AppendDesc:
    """rope: a rope_desc of the same k with k_out=None (its q is turned in the same launch)."""
    d = _with_cache(Kv4AppendDesc(), cache)
    d.dtype, d.tokens = dtype, tokens
    d.ldk, d.ldv = _rows("k", k, dtype, tokens, cache.kv_heads, cache.head_dim, ldk), _rows("v", v, dtype, tokens, cache.kv_heads, cache.head_dim, ldv)
    _dense(slots=slots)
    _count("slots", slots, tokens)
    if rope is not None:
        if getattr(rope, "_device", getattr(d, "_device", None)) != getattr(d, "_device", None):
            raise ValueError("rope tensors and cache are on different GPUs")
        d._keep.append(rope)
        d.rope = C.addressof(rope)
    return _tensors(d, k=k, v=v, slots=slots)


def kv4_append(desc: Kv4AppendDesc, stream=None) -> None:
    _call("fth_b200_kv4_append", desc, stream)


def kv4_gather_desc(*, cache, dtype, tokens, slots, k_out=None, v_out=None, ldk=0, ldv=0) -> Kv4GatherDesc:
    d = _with_cache(Kv4GatherDesc(), cache)
    d.dtype, d.tokens = dtype, tokens
    d.ldk = _rows("k_out", k_out, dtype, tokens, cache.kv_heads, cache.head_dim, ldk)
    d.ldv = _rows("v_out", v_out, dtype, tokens, cache.kv_heads, cache.head_dim, ldv)
    _dense(slots=slots)
    _count("slots", slots, tokens)
    return _tensors(d, slots=slots, k_out=k_out, v_out=v_out)


def kv4_gather(desc: Kv4GatherDesc, stream=None) -> None:
    _call("fth_b200_kv4_gather", desc, stream)


def kv4_attention_desc(*, cache, dtype, requests, tokens, q_heads, q, out, block_table, max_blocks, total_lens, scale, query_start=None,
                       max_query=1, causal=True, window=0, lse=None, ldq=0, ldo=0, workspace=None, workspace_bytes=0) -> Kv4AttentionDesc:
    d = _with_cache(Kv4AttentionDesc(), cache)
    d.dtype, d.requests, d.tokens, d.q_heads, d.max_blocks, d.max_query = dtype, requests, tokens, q_heads, max_blocks, max_query
    d.causal, d.window, d.scale, d.workspace_bytes = int(causal), window, scale, workspace_bytes
    d.ldq, d.ldo = _rows("q", q, dtype, tokens, q_heads, cache.head_dim, ldq), _rows("out", out, dtype, tokens, q_heads, cache.head_dim, ldo)
    _dense(block_table=block_table, total_lens=total_lens, query_start=query_start, lse=lse)
    _count("block_table", block_table, requests * max_blocks)
    _count("total_lens", total_lens, requests)
    _count("query_start", query_start, requests + 1)
    _count("lse", lse, tokens * q_heads)
    if hasattr(workspace, "numel") and workspace.numel() * workspace.element_size() < workspace_bytes:
        raise ValueError(f"workspace has {workspace.numel() * workspace.element_size()} bytes, not {workspace_bytes}")
    return _tensors(d, q=q, out=out, lse=lse, block_table=block_table, total_lens=total_lens, query_start=query_start, workspace=workspace)


def kv4_attention_workspace(torch, desc: Kv4AttentionDesc):
    """Allocates and zero-fills the scratch an attention descriptor needs and attaches it; returns the tensor."""
    need = lib().fth_b200_kv4_attention_workspace_bytes(C.byref(desc))
    if not need:
        check(lib().fth_b200_kv4_attention_supported(C.byref(desc)), "fth_b200_kv4_attention_supported")
        return None
    ws = torch.zeros(need, dtype=torch.uint8, device=f"cuda:{desc._device}" if getattr(desc, "_device", None) is not None else "cuda")
    _tensors(desc, workspace=ws)
    desc.workspace_bytes = need
    return ws


def kv4_attention(desc: Kv4AttentionDesc, stream=None) -> None:
    _call("fth_b200_kv4_attention", desc, stream)


def device_status() -> int:
    return lib().fth_b200_device_status()


def linear_workspace(torch, desc):
    """Allocates and zero-fills the scratch a linear descriptor may use and attaches it; returns the tensor."""
    fn = lib().fth_b200_fp8_linear_workspace_bytes if isinstance(desc, Fp8LinearDesc) else lib().fth_b200_int8_linear_workspace_bytes
    fn.restype = C.c_size_t
    need = fn(C.byref(desc))
    if not need:
        return None
    ws = torch.zeros(need, dtype=torch.uint8, device="cuda")
    desc.workspace, desc.workspace_bytes = ws.data_ptr(), need
    return ws


class Plan:
    """Host-buffer plan (Prepare once, compute many): see fth_b200_plan_* in include/fth_b200.h."""

    def __init__(self, desc, keepalive=()):
        self._h = C.c_void_p()
        self._keep = keepalive
        if isinstance(desc, Fp8LinearDesc):
            fn = lib().fth_b200_plan_create_fp8_linear
        elif isinstance(desc, Int8LinearDesc):
            fn = lib().fth_b200_plan_create_int8_linear
        else:
            fn = lib().fth_b200_plan_create_int8_conv2d
        check(fn(C.byref(desc), C.byref(self._h)), "fth_b200_plan_create")

    @property
    def input_bytes(self) -> int:
        return lib().fth_b200_plan_input_bytes(self._h)

    @property
    def output_bytes(self) -> int:
        return lib().fth_b200_plan_output_bytes(self._h)

    def run(self, host_in, host_out, stream=None) -> None:
        check(lib().fth_b200_plan_run(self._h, C.c_void_p(ptr(host_in)), C.c_void_p(ptr(host_out)),
                                      stream or current_stream()), "fth_b200_plan_run")

    def launch(self, device_in, device_out, stream=None) -> None:
        check(lib().fth_b200_plan_launch(self._h, C.c_void_p(ptr(device_in)), C.c_void_p(ptr(device_out)),
                                         stream or current_stream()), "fth_b200_plan_launch")

    def close(self) -> None:
        if self._h:
            lib().fth_b200_plan_destroy(self._h)
            self._h = C.c_void_p()

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass
