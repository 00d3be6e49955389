"""ctypes binding of liblaya_b200.so, the sm_100a execution library (include/laya_b200.h).

The library is built in-tree next to this file (see build.py).  There is no fallback: if the
library is missing, importing the runtime raises, so a run never silently executes elsewhere.
"""
import ctypes as ct
from pathlib import Path

LIB_NAME = "liblaya_b200.so"
LIB_PATH = Path(__file__).with_name(LIB_NAME)

OK, ERR_INVALID, ERR_CUDA, ERR_DEVICE, ERR_STATE, ERR_NO_DEVICE = range(6)
DTYPE_F32, DTYPE_F16, DTYPE_BF16, DTYPE_MX8 = 0, 1, 2, 3
ROTARY_NONE, ROTARY_LINEAR, ROTARY_NTK, ROTARY_PARTS = 0, 1, 2, 3
ACT_NONE, ACT_RELU, ACT_GELU, ACT_SILU = 0, 1, 2, 3
PRECISION_BF16, PRECISION_F16 = 0, 1

# Every symbol declared in include/laya_b200.h.
EXPORTS = (
    "laya_create", "laya_load_tensor", "laya_load_checkpoint", "laya_scan_checkpoint", "laya_finalize", "laya_predict", "laya_submit", "laya_collect",
    "laya_shape_class",
    "laya_forward_device", "laya_packed_ints", "laya_pack", "laya_reserve", "laya_stream", "laya_set_profiling",
    "laya_profile_read", "laya_read_tensor", "laya_cached_shapes", "laya_pool_bytes", "laya_destroy",
    "laya_last_error", "laya_set_launch_options", "laya_current_device", "laya_op_gemm", "laya_op_gemm_ln", "laya_interleave_geglu", "laya_op_attention", "laya_op_attention_gathered",
    "laya_attention_tiles", "laya_op_embed_norm", "laya_op_head_tail", "laya_op_norm", "laya_op_gemm_residual_static",
    "laya_mx8_scale_bytes", "laya_op_mx8_quantize", "laya_op_mx8_dequantize", "laya_op_rms_norm_mx8", "laya_op_mx8_linear",
    "laya_op_rotary", "laya_op_attend",
)
STATIC_SCRATCH_FLOATS = 4 * 1024 * 1024


class Config(ct.Structure):
    _fields_ = [("vocab", ct.c_int32), ("width", ct.c_int32), ("heads", ct.c_int32), ("layers", ct.c_int32),
                ("intermediate", ct.c_int32), ("global_every", ct.c_int32), ("window", ct.c_int32),
                ("theta_global", ct.c_float), ("theta_local", ct.c_float), ("eps", ct.c_float),
                ("max_len", ct.c_int32), ("head_layers", ct.c_int32), ("n_act", ct.c_int32),
                ("precision", ct.c_int32)]


class Metrics(ct.Structure):
    _fields_ = [("gpu_ms", ct.c_float), ("rows", ct.c_int32), ("batch", ct.c_int32), ("options", ct.c_int32),
                ("cache_miss", ct.c_int32), ("graph_capture", ct.c_int32), ("graph_replay", ct.c_int32),
                ("kernel_launches", ct.c_int32), ("owned_gpu_bytes", ct.c_uint64)]


class Mx8Convert(ct.Structure):
    _fields_ = [("rows", ct.c_int32), ("cols", ct.c_int32), ("dtype", ct.c_int32),
                ("values", ct.c_void_p), ("scales", ct.c_void_p), ("ldv", ct.c_int64),
                ("data", ct.c_void_p), ("ld", ct.c_int64)]


class RmsNormMx8(ct.Structure):
    _fields_ = [("rows", ct.c_int32), ("cols", ct.c_int32), ("dtype", ct.c_int32), ("residual_dtype", ct.c_int32),
                ("x", ct.c_void_p), ("ldx", ct.c_int64), ("residual", ct.c_void_p), ("ldr", ct.c_int64),
                ("sum_out", ct.c_void_p), ("lds", ct.c_int64), ("weight", ct.c_void_p),
                ("values", ct.c_void_p), ("scales", ct.c_void_p), ("ldv", ct.c_int64), ("eps", ct.c_float)]


class Mx8Linear(ct.Structure):
    _fields_ = [("rows", ct.c_int32), ("features", ct.c_int32), ("cols", ct.c_int32), ("activation", ct.c_int32),
                ("x", ct.c_void_p), ("x_scales", ct.c_void_p), ("ldx", ct.c_int64),
                ("w", ct.c_void_p), ("w_scales", ct.c_void_p), ("ldw", ct.c_int64),
                ("gate", ct.c_void_p), ("gate_scales", ct.c_void_p), ("ldg", ct.c_int64),
                ("bias", ct.c_void_p), ("gate_bias", ct.c_void_p),
                ("residual", ct.c_void_p), ("ldr", ct.c_int64),
                ("out", ct.c_void_p), ("out_scales", ct.c_void_p), ("ldo", ct.c_int64),
                ("residual_dtype", ct.c_int32), ("out_dtype", ct.c_int32)]


class Heads(ct.Structure):
    _fields_ = [("x", ct.c_void_p), ("x_token", ct.c_int64), ("x_head", ct.c_int64),
                ("out", ct.c_void_p), ("out_token", ct.c_int64), ("out_head", ct.c_int64),
                ("heads", ct.c_int32), ("reserved", ct.c_int32)]


class Rotary(ct.Structure):
    _fields_ = [("tokens", ct.c_int32), ("head_dim", ct.c_int32), ("dims", ct.c_int32), ("dtype", ct.c_int32),
                ("part", Heads * 2), ("positions", ct.c_void_p), ("positions_64", ct.c_int32), ("interleaved", ct.c_int32),
                ("backward", ct.c_int32), ("scaling", ct.c_int32),
                ("theta", ct.c_double), ("factor", ct.c_double), ("length", ct.c_double), ("low", ct.c_double), ("high", ct.c_double),
                ("magnitude", ct.c_float)]


class Attend(ct.Structure):
    _fields_ = [(name, ct.c_int32) for name in ("sequences", "heads", "kv_heads", "head_dim", "dtype", "q_tokens", "k_tokens",
                                                "max_queries", "max_keys")]
    for _name in ("q", "k", "v", "out"):
        _fields_ += [(_name, ct.c_void_p), (_name + "_token", ct.c_int64), (_name + "_head", ct.c_int64)]
    _fields_ += [(_name, ct.c_void_p) for _name in ("lse", "starts", "lengths", "k_starts", "k_lengths")]
    _fields_ += [("scale", ct.c_float), ("cap", ct.c_float), ("causal", ct.c_int32), ("window_left", ct.c_int32),
                 ("window_right", ct.c_int32)]
    _fields_ += [(_name, ct.c_void_p) for _name in ("prefix", "documents", "k_documents", "slopes", "distance_bias")]
    _fields_ += [("reach", ct.c_int32), ("reserved", ct.c_int32)]


_lib = None


def load():
    """Loads the library once and declares its signatures."""
    global _lib
    if _lib is not None:
        return _lib
    if not LIB_PATH.is_file():
        raise RuntimeError(f"{LIB_PATH} is missing: build it with `python -m laya_cuda.build` "
                           "(nvcc, sm_100a); there is no CPU fallback")
    lib = ct.CDLL(str(LIB_PATH))
    p, i, i32p, i64p, f32p = ct.c_void_p, ct.c_int, ct.POINTER(ct.c_int32), ct.POINTER(ct.c_int64), ct.POINTER(ct.c_float)
    sig = {
        "laya_create": (i, [ct.POINTER(Config), i, i, ct.POINTER(p)]),
        "laya_load_tensor": (i, [p, ct.c_char_p, i, i64p, i, p]),
        "laya_load_checkpoint": (i, [p, ct.c_char_p]),
        "laya_scan_checkpoint": (i, [ct.c_char_p, i64p, i64p]),
        "laya_finalize": (i, [p]),
        "laya_predict": (i, [p, p, p, p, p, p, i, i, p, p, ct.POINTER(Metrics)]),
        "laya_submit": (i, [p, p, p, p, p, p, i, i, i64p]),
        "laya_collect": (i, [p, ct.c_int64, p, p, ct.POINTER(Metrics)]),
        "laya_shape_class": (i, [p, p, i, i32p, i32p, i32p]),
        "laya_forward_device": (i, [p, p, i, i, i, i, p, p]),
        "laya_packed_ints": (ct.c_int64, [i, i, i]),
        "laya_pack": (i, [p, p, p, p, p, i, i, i, i, i, p]),
        "laya_reserve": (i, [p, i, i, i]),
        "laya_stream": (p, [p]),
        "laya_set_profiling": (i, [p, i]),
        "laya_profile_read": (i, [p, i, ct.POINTER(ct.c_double), i64p, ct.POINTER(ct.c_double)]),
        "laya_read_tensor": (i, [p, ct.c_char_p, f32p, ct.c_int64]),
        "laya_cached_shapes": (i, [p, i32p]),
        "laya_pool_bytes": (i, [p, ct.POINTER(ct.c_uint64), ct.POINTER(ct.c_uint64)]),
        "laya_destroy": (i, [p]),
        "laya_last_error": (ct.c_char_p, [p]),
        "laya_set_launch_options": (i, [i, ct.c_uint64]),
        "laya_current_device": (i, [ct.POINTER(i)]),
        "laya_op_gemm": (i, [i, i, p, p, i, i, i, p, i, p, i, p, i, p, i, p, i, i, p, p]),
        "laya_op_gemm_ln": (i, [i, p, p, i, i, i, p, i, p, p, p, ct.c_float, p, i, p, p]),
        "laya_interleave_geglu": (i, [p, p, i, i]),
        "laya_op_attention": (i, [i, i, p, p, p, i, p, p, i, i, i, p, p]),
        "laya_op_attention_gathered": (i, [i, p, p, p, i, p, p, i, i, i, p, p]),
        "laya_attention_tiles": (i, [p, p, i, i, i, p, i]),
        "laya_op_embed_norm": (i, [i, p, p, p, ct.c_float, i, i, i, p, p, p, p]),
        "laya_op_norm": (i, [i, p, p, i, p, p, ct.c_float, p, i, i, p]),
        "laya_op_head_tail": (i, [i, p, p, p, i, i, i, p, p, p, p, p, p, i, p, p, p, p, p, p]),
        "laya_op_gemm_residual_static": (i, [i, p, p, i, i, i, i, p, p, p, p]),
    }
    sig |= {
        "laya_mx8_scale_bytes": (ct.c_int64, [i, i]),
        "laya_op_mx8_quantize": (i, [p, p]),
        "laya_op_mx8_dequantize": (i, [p, p]),
        "laya_op_rms_norm_mx8": (i, [p, p]),
        "laya_op_mx8_linear": (i, [p, p, p]),
        "laya_op_rotary": (i, [p, p]),
        "laya_op_attend": (i, [p, p, p]),
    }
    for name, (res, args) in sig.items():
        fn = getattr(lib, name)
        fn.restype, fn.argtypes = res, args
    _lib = lib
    return lib


def check(code, handle=None):
    """Maps a status code to the reference's exception types (ValueError / RuntimeError)."""
    if code == OK:
        return
    message = load().laya_last_error(handle).decode(errors="replace")
    if code == ERR_INVALID:
        raise ValueError(message)
    raise RuntimeError(message or f"laya_b200 error {code}")
