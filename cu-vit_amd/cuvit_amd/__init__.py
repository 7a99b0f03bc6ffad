"""Python binding of libcuvit_amd.so, the MI355X (gfx950) layer-kernel library.

The library's interface is the C ABI in include/cuvit/capi.h; this module binds
it with ctypes, and the launchers' plain case with the native module beside it
(_native.so), so programs can drive the HIP kernels on device tensors that
PyTorch allocates. PyTorch provides device memory and the stream
handle only; every computation runs in the library's own HIP kernels. There is
no fallback: if the library is not built, loading raises.

Launcher functions mirror the reference's kernels.hpp (names, argument order,
error behaviour): an invalid argument raises InvalidArgument (a ValueError, the
counterpart of std::invalid_argument), an oversized launch raises LengthError,
and a failed launch raises HipError.
"""

from __future__ import annotations

import ctypes
import os
import sys
import threading
from typing import Optional

__all__ = [
    "CuvitError", "InvalidArgument", "LengthError", "HipError", "OutOfRange",
    "GemmProblem", "VitConfig", "library", "library_path", "check", "stream_handle",
    "gemm", "layer_norm", "softmax", "gelu", "extract_patches", "extract_patches_f32_to_bf16",
    "add", "add_broadcast",
    "broadcast", "convert_to_bf16", "convert_to_f32", "attention", "attention_supported",
    "gemm_problem", "WeightWriter", "WeightFile", "VisionTransformer",
    "NO_TRANSPOSE", "TRANSPOSED", "PRECISION_F32", "PRECISION_BF16",
    "Preprocessing", "RgbImage", "load_ppm", "preprocess", "preprocess_image", "cli_path",
    "RotaryProblem", "QkNormProblem", "GatedProblem", "rotary_problem", "qk_norm_problem", "gated_problem",
    "rotary", "qk_norm_rotary", "qk_norm_rotary_backward", "qk_norm_rotary_workspace",
    "gated_gemm", "gated_backward",
    "gated_checkpoint_gemm", "gated_checkpoint_backward", "gated_checkpoint_scales",
    "PackedAttentionProblem", "packed_attention_problem", "packed_attention", "packed_attention_workspace",
    "packed_attention_backward", "packed_attention_backward_workspace",
    "ROTARY_HALVES", "ROTARY_ADJACENT", "NORM_RMS", "NORM_LAYER",
    "GATE_SILU", "GATE_GELU", "GATE_GELU_TANH",
]

_HERE = os.path.dirname(os.path.abspath(__file__))
_DEFAULT_LIB = os.path.join(os.path.dirname(_HERE), "lib", "libcuvit_amd.so")

NO_TRANSPOSE = 0
TRANSPOSED = 1

PRECISION_F32 = 0
PRECISION_BF16 = 1

ROTARY_HALVES = 0
ROTARY_ADJACENT = 1

NORM_RMS = 0
NORM_LAYER = 1

GATE_SILU = 0
GATE_GELU = 1
GATE_GELU_TANH = 2

OK = 0
ERROR_INVALID_ARGUMENT = 1
ERROR_LENGTH = 2
ERROR_HIP = 3
ERROR_RUNTIME = 4
ERROR_OUT_OF_RANGE = 5


class CuvitError(RuntimeError):
    """Base of the errors a C-ABI status turns into."""

    def __init__(self, status: int, message: str):
        super().__init__(message)
        self.status = status


class InvalidArgument(CuvitError, ValueError):
    """CUVIT_ERROR_INVALID_ARGUMENT (std::invalid_argument in the reference)."""


class LengthError(CuvitError):
    """CUVIT_ERROR_LENGTH (std::length_error)."""


class HipError(CuvitError):
    """CUVIT_ERROR_HIP (CudaError in the reference); .hip_code is the hipError_t."""

    def __init__(self, status: int, message: str, hip_code: int):
        super().__init__(status, message)
        self.hip_code = hip_code


class OutOfRange(CuvitError, IndexError):
    """CUVIT_ERROR_OUT_OF_RANGE (std::out_of_range)."""


class GemmBatch(ctypes.Structure):
    _fields_ = [
        ("count", ctypes.c_int),
        ("stride_a", ctypes.c_int64),
        ("stride_b", ctypes.c_int64),
        ("stride_c", ctypes.c_int64),
        ("inner", ctypes.c_int),
        ("outer_stride_a", ctypes.c_int64),
        ("outer_stride_b", ctypes.c_int64),
        ("outer_stride_c", ctypes.c_int64),
    ]


class GemmEpilogue(ctypes.Structure):
    _fields_ = [("accumulate", ctypes.c_uint8), ("gelu", ctypes.c_uint8)]


class GemmProblem(ctypes.Structure):
    """cuvit_gemm_problem / cuvit::GemmProblem (reference kernels.hpp:74-85)."""

    _fields_ = [
        ("m", ctypes.c_int),
        ("n", ctypes.c_int),
        ("k", ctypes.c_int),
        ("layout", ctypes.c_int32),
        ("alpha", ctypes.c_float),
        ("lda", ctypes.c_int),
        ("ldb", ctypes.c_int),
        ("ldc", ctypes.c_int),
        ("batch", GemmBatch),
        ("epilogue", GemmEpilogue),
    ]


class VitConfig(ctypes.Structure):
    """cuvit_vit_config / cuvit::VitConfig (reference vit.hpp:15-35)."""

    _fields_ = [
        ("image_size", ctypes.c_int),
        ("patch_size", ctypes.c_int),
        ("channels", ctypes.c_int),
        ("embed_dim", ctypes.c_int),
        ("depth", ctypes.c_int),
        ("heads", ctypes.c_int),
        ("mlp_hidden", ctypes.c_int),
        ("classes", ctypes.c_int),
        ("layer_norm_epsilon", ctypes.c_float),
    ]

    def patches_per_side(self) -> int:
        return self.image_size // self.patch_size

    def patch_count(self) -> int:
        return self.patches_per_side() ** 2

    def token_count(self) -> int:
        return self.patch_count() + 1

    def head_dim(self) -> int:
        return self.embed_dim // self.heads

    def patch_elements(self) -> int:
        return self.channels * self.patch_size * self.patch_size


class Preprocessing(ctypes.Structure):
    """cuvit_preprocessing / cuvit::Preprocessing (reference image.hpp:30-38),
    with the reference's defaults: size 224, crop fraction 0.9, mean and
    stddev 0.5 per channel."""

    _fields_ = [
        ("size", ctypes.c_int),
        ("crop_fraction", ctypes.c_float),
        ("mean", ctypes.c_float * 3),
        ("stddev", ctypes.c_float * 3),
    ]

    def __init__(self, size: int = 224, crop_fraction: float = 0.9,
                 mean=(0.5, 0.5, 0.5), stddev=(0.5, 0.5, 0.5)):
        super().__init__(size, crop_fraction, (ctypes.c_float * 3)(*mean),
                         (ctypes.c_float * 3)(*stddev))


class Rotation(ctypes.Structure):
    """cuvit_rotation: how a head's values pair up, how many pairs each axis
    owns, and the floats from one image's positions to the next (0: shared)."""

    _fields_ = [
        ("pairing", ctypes.c_int32),
        ("axes", ctypes.c_int),
        ("pairs", ctypes.c_int * 3),
        ("position_stride", ctypes.c_int64),
    ]


class HeadStrides(ctypes.Structure):
    """cuvit_head_strides: elements from one image, token and head to the next;
    0 selects the packed [images, tokens, heads, head_dim] one."""

    _fields_ = [("image", ctypes.c_int64), ("token", ctypes.c_int64), ("head", ctypes.c_int64)]


class RotaryProblem(ctypes.Structure):
    """cuvit_rotary_problem."""

    _fields_ = [
        ("images", ctypes.c_int),
        ("tokens", ctypes.c_int),
        ("heads", ctypes.c_int),
        ("head_dim", ctypes.c_int),
        ("rotation", Rotation),
        ("inverse", ctypes.c_uint8),
        ("input", HeadStrides),
        ("output", HeadStrides),
    ]


class QkNormProblem(ctypes.Structure):
    """cuvit_qk_norm_problem."""

    _fields_ = [
        ("images", ctypes.c_int),
        ("tokens", ctypes.c_int),
        ("heads", ctypes.c_int),
        ("kv_heads", ctypes.c_int),
        ("head_dim", ctypes.c_int),
        ("norm", ctypes.c_int32),
        ("epsilon", ctypes.c_float),
        ("rotation", Rotation),
    ]


class GatedProblem(ctypes.Structure):
    """cuvit_gated_problem."""

    _fields_ = [
        ("m", ctypes.c_int),
        ("n", ctypes.c_int),
        ("k", ctypes.c_int),
        ("activation", ctypes.c_int32),
        ("lda", ctypes.c_int),
        ("ldb", ctypes.c_int),
        ("ldc", ctypes.c_int),
        ("ld_preactivations", ctypes.c_int),
    ]


class TokenStrides(ctypes.Structure):
    """cuvit_token_strides: elements from one token and head to the next; 0
    selects the packed [tokens, heads, head_dim] one."""

    _fields_ = [("token", ctypes.c_int64), ("head", ctypes.c_int64)]


class PackedAttentionProblem(ctypes.Structure):
    """cuvit_packed_attention_problem."""

    _fields_ = [
        ("sequences", ctypes.c_int),
        ("tokens", ctypes.c_int),
        ("kv_tokens", ctypes.c_int),
        ("heads", ctypes.c_int),
        ("kv_heads", ctypes.c_int),
        ("head_dim", ctypes.c_int),
        ("scale", ctypes.c_float),
        ("causal", ctypes.c_uint8),
        ("q", TokenStrides),
        ("k", TokenStrides),
        ("v", TokenStrides),
        ("out", TokenStrides),
    ]


_P = ctypes.c_void_p
_I = ctypes.c_int
_L = ctypes.c_int64
_F = ctypes.c_float
_SIGNATURES = {
    "cuvit_last_error": (ctypes.c_char_p, []),
    "cuvit_last_hip_error": (_I, []),
    "cuvit_version": (_I, []),
    "cuvit_gemm_problem_init": (None, [ctypes.POINTER(GemmProblem), _I, _I, _I, _I]),
    "cuvit_gemm_f32": (_I, [_P, _P, _P, _P, ctypes.POINTER(GemmProblem), _P]),
    "cuvit_gemm_bf16": (_I, [_P, _P, _P, _P, ctypes.POINTER(GemmProblem), _P]),
    "cuvit_layer_norm_f32": (_I, [_P, _P, _P, _P, _I, _I, _F, _P]),
    "cuvit_layer_norm_bf16": (_I, [_P, _P, _P, _P, _I, _I, _F, _P]),
    "cuvit_gelu_f32": (_I, [_P, _P, _L, _P]),
    "cuvit_gelu_bf16": (_I, [_P, _P, _L, _P]),
    "cuvit_softmax_f32": (_I, [_P, _P, _I, _I, _P]),
    "cuvit_softmax_bf16": (_I, [_P, _P, _I, _I, _P]),
    "cuvit_extract_patches_f32": (_I, [_P, _P, _I, _I, _I, _I, _I, _P]),
    "cuvit_extract_patches_bf16": (_I, [_P, _P, _I, _I, _I, _I, _I, _P]),
    "cuvit_extract_patches_f32_to_bf16": (_I, [_P, _P, _I, _I, _I, _I, _I, _P]),
    "cuvit_add_f32": (_I, [_P, _P, _L, _P]),
    "cuvit_add_broadcast_f32": (_I, [_P, _P, _L, _I, _P]),
    "cuvit_broadcast_f32": (_I, [_P, _P, _L, _L, _I, _P]),
    "cuvit_broadcast_bf16": (_I, [_P, _P, _L, _L, _I, _P]),
    "cuvit_convert_f32_to_bf16": (_I, [_P, _P, _L, _P]),
    "cuvit_convert_bf16_to_f32": (_I, [_P, _P, _L, _P]),
    "cuvit_attention_supported": (_I, [_I, _I]),
    "cuvit_attention_f32": (_I, [_P, _P, _I, _I, _I, _I, _P]),
    "cuvit_attention_bf16": (_I, [_P, _P, _I, _I, _I, _I, _P]),
    "cuvit_rotary_problem_init": (None, [ctypes.POINTER(RotaryProblem), _I, _I, _I, _I, _I, ctypes.POINTER(_I), _I]),
    "cuvit_rotary_f32": (_I, [_P, _P, _P, _P, ctypes.POINTER(RotaryProblem), _P]),
    "cuvit_rotary_bf16": (_I, [_P, _P, _P, _P, ctypes.POINTER(RotaryProblem), _P]),
    "cuvit_qk_norm_problem_init": (None, [ctypes.POINTER(QkNormProblem), _I, _I, _I, _I, _I,
                                          ctypes.POINTER(_I), _I, _I]),
    "cuvit_qk_norm_rotary_f32": (_I, [_P] * 8 + [ctypes.POINTER(QkNormProblem), _P]),
    "cuvit_qk_norm_rotary_bf16": (_I, [_P] * 8 + [ctypes.POINTER(QkNormProblem), _P]),
    "cuvit_qk_norm_rotary_workspace": (_L, [ctypes.POINTER(QkNormProblem)]),
    "cuvit_qk_norm_rotary_backward_f32": (_I, [_P] * 12 + [_L, ctypes.POINTER(QkNormProblem), _P]),
    "cuvit_qk_norm_rotary_backward_bf16": (_I, [_P] * 12 + [_L, ctypes.POINTER(QkNormProblem), _P]),
    "cuvit_gated_problem_init": (None, [ctypes.POINTER(GatedProblem), _I, _I, _I, _I]),
    "cuvit_gated_gemm_f32": (_I, [_P, _P, _P, _P, _P, ctypes.POINTER(GatedProblem), _P]),
    "cuvit_gated_gemm_bf16": (_I, [_P, _P, _P, _P, _P, ctypes.POINTER(GatedProblem), _P]),
    "cuvit_gated_backward_f32": (_I, [_P, _P, _P, ctypes.POINTER(GatedProblem), _P]),
    "cuvit_gated_backward_bf16": (_I, [_P, _P, _P, ctypes.POINTER(GatedProblem), _P]),
    "cuvit_gated_checkpoint_scales": (_L, [ctypes.POINTER(GatedProblem)]),
    "cuvit_gated_checkpoint_gemm_f32": (_I, [_P] * 6 + [ctypes.POINTER(GatedProblem), _P]),
    "cuvit_gated_checkpoint_gemm_bf16": (_I, [_P] * 6 + [ctypes.POINTER(GatedProblem), _P]),
    "cuvit_gated_checkpoint_backward_f32": (_I, [_P] * 5 + [ctypes.POINTER(GatedProblem), _P]),
    "cuvit_gated_checkpoint_backward_bf16": (_I, [_P] * 5 + [ctypes.POINTER(GatedProblem), _P]),
    "cuvit_packed_attention_problem_init": (None, [ctypes.POINTER(PackedAttentionProblem), _I, _I, _I, _I]),
    "cuvit_packed_attention_problem_projection": (None, [ctypes.POINTER(PackedAttentionProblem)]),
    "cuvit_packed_attention_workspace": (_L, [ctypes.POINTER(PackedAttentionProblem)]),
    "cuvit_packed_attention_f32": (_I, [_P] * 9 + [_L, ctypes.POINTER(PackedAttentionProblem), _P]),
    "cuvit_packed_attention_bf16": (_I, [_P] * 9 + [_L, ctypes.POINTER(PackedAttentionProblem), _P]),
    "cuvit_packed_attention_backward_workspace": (_L, [ctypes.POINTER(PackedAttentionProblem)]),
    "cuvit_packed_attention_backward_f32": (_I, [_P] * 13 + [_L, ctypes.POINTER(PackedAttentionProblem), _P]),
    "cuvit_packed_attention_backward_bf16": (_I, [_P] * 13 + [_L, ctypes.POINTER(PackedAttentionProblem), _P]),
    "cuvit_weight_writer_create": (_I, [ctypes.POINTER(_P)]),
    "cuvit_weight_writer_add": (_I, [_P, ctypes.c_char_p, _I, ctypes.POINTER(_L), _P]),
    "cuvit_weight_writer_add_bf16": (_I, [_P, ctypes.c_char_p, _I, ctypes.POINTER(_L), _P]),
    "cuvit_weight_writer_write": (_I, [_P, ctypes.c_char_p]),
    "cuvit_weight_writer_destroy": (None, [_P]),
    "cuvit_weight_file_load": (_I, [ctypes.c_char_p, ctypes.POINTER(_P)]),
    "cuvit_weight_file_size": (_L, [_P]),
    "cuvit_weight_file_contains": (_I, [_P, ctypes.c_char_p]),
    "cuvit_weight_file_float_data": (_I, [_P, ctypes.c_char_p, _I, ctypes.POINTER(_L), ctypes.POINTER(_P)]),
    "cuvit_weight_file_bf16_data": (_I, [_P, ctypes.c_char_p, _I, ctypes.POINTER(_L), ctypes.POINTER(_P)]),
    "cuvit_weight_file_version": (_I, [_P]),
    "cuvit_weight_file_type": (_I, [_P, ctypes.c_char_p]),
    "cuvit_weight_file_entry_name": (ctypes.c_char_p, [_P, _L]),
    "cuvit_weight_file_payload_bytes": (ctypes.c_uint64, [_P]),
    "cuvit_weight_file_destroy": (None, [_P]),
    "cuvit_vit_config_default": (None, [ctypes.POINTER(VitConfig)]),
    "cuvit_vit_config_validate": (_I, [ctypes.POINTER(VitConfig)]),
    "cuvit_vit_create": (_I, [ctypes.POINTER(VitConfig), _P, _I, ctypes.POINTER(_P)]),
    "cuvit_vit_create_ex": (_I, [ctypes.POINTER(VitConfig), _P, _I, _I, ctypes.POINTER(_P)]),
    "cuvit_vit_precision": (_I, [_P]),
    "cuvit_vit_forward": (_I, [_P, _P, _P, _I, _P]),
    "cuvit_vit_weight_bytes": (ctypes.c_uint64, [_P]),
    "cuvit_vit_activation_bytes": (ctypes.c_uint64, [_P]),
    "cuvit_vit_destroy": (None, [_P]),
    "cuvit_image_load_ppm": (_I, [ctypes.c_char_p, ctypes.POINTER(_P)]),
    "cuvit_image_width": (_I, [_P]),
    "cuvit_image_height": (_I, [_P]),
    "cuvit_image_pixels": (_P, [_P]),
    "cuvit_image_destroy": (None, [_P]),
    "cuvit_preprocessing_default": (None, [ctypes.POINTER(Preprocessing)]),
    "cuvit_preprocess_u8": (_I, [_P, _I, _I, _I, ctypes.POINTER(Preprocessing), _P, _P]),
}

_lib: Optional[ctypes.CDLL] = None


def library_path() -> str:
    return os.environ.get("CUVIT_AMD_LIBRARY", _DEFAULT_LIB)


def library() -> ctypes.CDLL:
    """The loaded libcuvit_amd.so. Raises if it has not been built."""
    global _lib
    if _lib is None:
        path = library_path()
        if not os.path.exists(path):
            raise RuntimeError(
                f"libcuvit_amd.so not found at {path}: build it first "
                "(python -c 'import __graft_entry__ as g; g.build()' or make -C cu-vit_amd)")
        lib = ctypes.CDLL(path)
        for name, (restype, argtypes) in _SIGNATURES.items():
            fn = getattr(lib, name)
            fn.restype = restype
            fn.argtypes = argtypes
        _lib = lib
    return _lib


_NATIVE_FUNCTIONS = (
    "cuvit_layer_norm_f32", "cuvit_layer_norm_bf16", "cuvit_softmax_f32", "cuvit_softmax_bf16",
    "cuvit_extract_patches_f32", "cuvit_extract_patches_bf16", "cuvit_gemm_f32", "cuvit_gemm_bf16",
    "cuvit_attention_f32", "cuvit_attention_bf16", "cuvit_preprocess_u8", "cuvit_vit_forward",
    "cuvit_rotary_f32", "cuvit_rotary_bf16", "cuvit_qk_norm_rotary_f32", "cuvit_qk_norm_rotary_bf16",
    "cuvit_qk_norm_rotary_backward_f32", "cuvit_qk_norm_rotary_backward_bf16", "cuvit_qk_norm_rotary_workspace",
    "cuvit_gated_gemm_f32", "cuvit_gated_gemm_bf16", "cuvit_gated_backward_f32", "cuvit_gated_backward_bf16",
    "cuvit_packed_attention_f32", "cuvit_packed_attention_bf16", "cuvit_packed_attention_workspace",
    "cuvit_packed_attention_backward_f32", "cuvit_packed_attention_backward_bf16",
    "cuvit_packed_attention_backward_workspace", "cuvit_gated_checkpoint_gemm_f32",
    "cuvit_gated_checkpoint_gemm_bf16", "cuvit_gated_checkpoint_backward_f32",
    "cuvit_gated_checkpoint_backward_bf16", "cuvit_gated_checkpoint_scales",
)


_NATIVE_CALLS = ("layer_norm", "softmax", "extract_patches", "gemm", "attention", "preprocess", "vit_forward",
                 "rotary", "qk_norm_rotary", "qk_norm_rotary_backward", "gated_gemm", "gated_backward",
                 "packed_attention", "packed_attention_backward", "gated_checkpoint_gemm",
                 "gated_checkpoint_backward")


def _not_plain(*arguments) -> int:
    return -1


def _native_module(torch):
    """The native module, or None (with a warning) where it is not built or was
    built for another PyTorch or Python, whose tensors it would misread."""
    import warnings

    try:
        from . import _native
    except ImportError as error:
        reason = str(error)
    else:
        here = (torch.__version__.split("+")[0], *sys.version_info[:2])
        if getattr(_native, "built_for", None) == here:
            return _native
        reason = f"it was built for {getattr(_native, 'built_for', 'an older binding')}, this is {here}"
    warnings.warn(f"cuvit_amd: no native binding ({reason}); calls take the slower ctypes path. "
                  "Build it with `make python` in cu-vit_amd.", RuntimeWarning, stacklevel=4)
    return None


class _NativeCalls:
    """The launchers' plain case in native code (csrc/binding/native.cpp): each
    takes a launcher's arguments and returns the library's status, or -1 where
    they are not plain GPU tensors and whole numbers that pass every check; the
    Python code then takes the call, as it does every call without the module.
    The module is loaded with the first launcher that can be given a tensor:
    a program without torch has none. A LayerNorm call of 197 rows takes 4.0 us
    of a stream of calls so, 10.4 through the Python code."""

    def __init__(self):
        self._lock = threading.Lock()

    def __getattr__(self, name):
        if name not in _NATIVE_CALLS:
            raise AttributeError(name)
        torch = sys.modules.get("torch")
        if torch is None:
            return _not_plain
        with self._lock:
            if name not in self.__dict__:
                native = _native_module(torch)
                if native is not None:
                    lib = library()
                    native.bind(GemmProblem, Preprocessing, RotaryProblem, QkNormProblem, GatedProblem,
                                PackedAttentionProblem, *(ctypes.cast(getattr(lib, f), _P).value for f in _NATIVE_FUNCTIONS))
                for call in _NATIVE_CALLS:
                    setattr(self, call, getattr(native, call) if native is not None else _not_plain)
        return self.__dict__[name]


_native_calls = _NativeCalls()


def check(status: int) -> None:
    """Raises the exception matching a C-ABI status."""
    if status == OK:
        return
    lib = library()
    message = (lib.cuvit_last_error() or b"").decode()
    if status == ERROR_INVALID_ARGUMENT:
        raise InvalidArgument(status, message)
    if status == ERROR_LENGTH:
        raise LengthError(status, message)
    if status == ERROR_HIP:
        raise HipError(status, message, lib.cuvit_last_hip_error())
    if status == ERROR_OUT_OF_RANGE:
        raise OutOfRange(status, message)
    raise CuvitError(status, message)


def _ptr(x) -> Optional[int]:
    """Device address of a torch tensor, an int address, or None (NULL)."""
    if x is None:
        return None
    if isinstance(x, int):
        return x
    return x.data_ptr()


def _operand(x, name: str, dtype: str, elements: int) -> Optional[int]:
    """The address of operand @p x after checking that the kernel may touch
    @p elements of it: a torch tensor must live on the GPU, hold @p dtype
    ("float32", "bfloat16", "uint8" and the like), be contiguous and have at least that
    many elements; anything else would be a device access outside the
    tensor or a host address read by the GPU. Raw int addresses and None go
    through unchecked, as in the C API (None becomes NULL, which the library
    rejects with its own message)."""
    if x is None or isinstance(x, int):
        return x
    if x.device.type != "cuda":
        raise InvalidArgument(ERROR_INVALID_ARGUMENT, f"{name} is not a GPU tensor ({x.device})")
    if str(x.dtype) != "torch." + dtype:
        raise InvalidArgument(ERROR_INVALID_ARGUMENT,
                              f"{name} holds {x.dtype}; this launch needs torch.{dtype}")
    if not x.is_contiguous():
        raise InvalidArgument(ERROR_INVALID_ARGUMENT, f"{name} is not contiguous")
    if x.numel() < elements:
        raise InvalidArgument(ERROR_INVALID_ARGUMENT,
                              f"{name} holds {x.numel()} elements; the launch touches {elements}")
    return x.data_ptr()


def _positive(*extents) -> bool:
    """True when every extent is positive: only then are the operand checks
    applied, so that zero and negative extents reach the library's own
    checks in the reference's order (a zero extent returns first, even with
    null pointers; a negative one is InvalidArgument)."""
    return all(int(e) > 0 for e in extents)


def _storage(bf16: bool) -> str:
    return "bfloat16" if bf16 else "float32"


def _offset_range(count: int, inner: int, stride: int, outer_stride: int):
    """Smallest and largest element offset of a batch entry's operand
    (split batches: entry i sits at (i / inner) * outer_stride + (i % inner)
    * stride; flat ones at i * stride)."""
    if 0 < inner < count:
        outer_span = (count // inner - 1) * outer_stride
        inner_span = (inner - 1) * stride
        return (min(0, outer_span) + min(0, inner_span), max(0, outer_span) + max(0, inner_span))
    span = (count - 1) * stride
    return min(0, span), max(0, span)


def _gemm_operands(a, b, bias, c, problem: "GemmProblem", bf16: bool):
    p = problem
    if not _positive(p.m, p.n, p.batch.count) or p.k < 0:
        return _ptr(a), _ptr(b), _ptr(bias), _ptr(c)
    transposed = p.layout == TRANSPOSED
    lda = p.lda or p.k
    ldb = p.ldb or (p.k if transposed else p.n)
    ldc = p.ldc or p.n
    if lda < p.k or ldc < p.n or ldb < (p.k if transposed else p.n):
        return _ptr(a), _ptr(b), _ptr(bias), _ptr(c)  # the library names the bad ld
    count, inner = p.batch.count, p.batch.inner

    def span(rows: int, ld: int, cols: int, stride: int, outer_stride: int, name: str) -> int:
        if rows <= 0 or cols <= 0:
            return 0
        low, high = _offset_range(count, inner, stride, outer_stride)
        if low < 0:
            raise InvalidArgument(ERROR_INVALID_ARGUMENT,
                                  f"{name}: a batch entry starts before the tensor")
        return high + (rows - 1) * ld + cols

    t = _storage(bf16)
    a_rows, a_cols = p.m, p.k
    b_rows, b_cols = (p.n, p.k) if transposed else (p.k, p.n)
    return (_operand(a, "A", t, span(a_rows, lda, a_cols, p.batch.stride_a,
                                     p.batch.outer_stride_a, "A")),
            _operand(b, "B", t, span(b_rows, ldb, b_cols, p.batch.stride_b,
                                     p.batch.outer_stride_b, "B")),
            _operand(bias, "bias", "float32", p.n),
            _operand(c, "C", t, span(p.m, ldc, p.n, p.batch.stride_c, p.batch.outer_stride_c, "C")))


def stream_handle(stream=None) -> Optional[int]:
    """hipStream_t of a torch stream (default: torch's current stream)."""
    import torch

    if stream is None:
        if not torch.cuda.is_available():
            return None  # host-only use: argument validation never reaches a stream
        stream = torch.cuda.current_stream()
    return stream.cuda_stream or None


def _bf16(x) -> bool:
    if x is None or isinstance(x, int):
        return False
    import torch

    return x.dtype == torch.bfloat16


def gemm_problem(m: int, n: int, k: int, layout: int = NO_TRANSPOSE) -> GemmProblem:
    """The reference's gemm_problem() (kernels.hpp:89-96)."""
    problem = GemmProblem()
    library().cuvit_gemm_problem_init(ctypes.byref(problem), m, n, k, layout)
    return problem


def gemm(a, b, bias, c, problem: GemmProblem, stream=None, bf16: Optional[bool] = None) -> None:
    status = _native_calls.gemm(a, b, bias, c, problem, stream, bf16)
    if status >= 0:
        return check(status)
    bf16 = bf16 if bf16 is not None else _bf16(a)
    fn = library().cuvit_gemm_bf16 if bf16 else library().cuvit_gemm_f32
    pa, pb, pbias, pc = _gemm_operands(a, b, bias, c, problem, bf16)
    check(fn(pa, pb, pbias, pc, ctypes.byref(problem), stream_handle(stream)))


def layer_norm(x, gamma, beta, out, rows: int, columns: int, epsilon: float = 1.0e-6,
               stream=None, bf16: Optional[bool] = None) -> None:
    status = _native_calls.layer_norm(x, gamma, beta, out, rows, columns, epsilon, stream, bf16)
    if status >= 0:
        return check(status)
    bf16 = bf16 if bf16 is not None else _bf16(x)
    fn = library().cuvit_layer_norm_bf16 if bf16 else library().cuvit_layer_norm_f32
    if _positive(rows, columns):
        t, n = _storage(bf16), rows * columns
        x, out = _operand(x, "x", t, n), _operand(out, "out", t, n)
        gamma = _operand(gamma, "gamma", "float32", columns)
        beta = _operand(beta, "beta", "float32", columns)
    check(fn(_ptr(x), _ptr(gamma), _ptr(beta), _ptr(out), rows, columns, epsilon,
             stream_handle(stream)))


def softmax(x, out, rows: int, columns: int, stream=None, bf16: Optional[bool] = None) -> None:
    status = _native_calls.softmax(x, out, rows, columns, stream, bf16)
    if status >= 0:
        return check(status)
    bf16 = bf16 if bf16 is not None else _bf16(x)
    fn = library().cuvit_softmax_bf16 if bf16 else library().cuvit_softmax_f32
    if _positive(rows, columns):
        t, n = _storage(bf16), rows * columns
        x, out = _operand(x, "x", t, n), _operand(out, "out", t, n)
    check(fn(_ptr(x), _ptr(out), rows, columns, stream_handle(stream)))


def gelu(x, out, count: int, stream=None, bf16: Optional[bool] = None) -> None:
    bf16 = bf16 if bf16 is not None else _bf16(x)
    fn = library().cuvit_gelu_bf16 if bf16 else library().cuvit_gelu_f32
    if _positive(count):
        x, out = _operand(x, "x", _storage(bf16), count), _operand(out, "out", _storage(bf16), count)
    check(fn(_ptr(x), _ptr(out), count, stream_handle(stream)))


def extract_patches(images, patches, batch: int, channels: int, height: int, width: int,
                    patch: int, stream=None, bf16: Optional[bool] = None) -> None:
    status = _native_calls.extract_patches(images, patches, batch, channels, height, width, patch,
                                            stream, bf16)
    if status >= 0:
        return check(status)
    bf16 = bf16 if bf16 is not None else _bf16(images)
    fn = library().cuvit_extract_patches_bf16 if bf16 else library().cuvit_extract_patches_f32
    if _positive(batch, channels, height, width, patch):
        n = batch * channels * height * width
        images = _operand(images, "images", _storage(bf16), n)
        patches = _operand(patches, "patches", _storage(bf16), n)
    check(fn(_ptr(images), _ptr(patches), batch, channels, height, width, patch,
             stream_handle(stream)))


def extract_patches_f32_to_bf16(images, patches, batch: int, channels: int, height: int,
                                width: int, patch: int, stream=None) -> None:
    """fp32 images into bf16 patch rows in one pass (bitwise the conversion
    then the bf16 gather)."""
    if _positive(batch, channels, height, width, patch):
        n = batch * channels * height * width
        images = _operand(images, "images", "float32", n)
        patches = _operand(patches, "patches", _storage(True), n)
    check(library().cuvit_extract_patches_f32_to_bf16(_ptr(images), _ptr(patches), batch, channels,
                                                      height, width, patch, stream_handle(stream)))


def add(accumulator, addend, count: int, stream=None) -> None:
    if _positive(count):
        accumulator = _operand(accumulator, "accumulator", "float32", count)
        addend = _operand(addend, "addend", "float32", count)
    check(library().cuvit_add_f32(_ptr(accumulator), _ptr(addend), count, stream_handle(stream)))


def add_broadcast(accumulator, addend, count: int, batch: int, stream=None) -> None:
    if _positive(count, batch):
        accumulator = _operand(accumulator, "accumulator", "float32", count * batch)
        addend = _operand(addend, "addend", "float32", count)
    check(library().cuvit_add_broadcast_f32(_ptr(accumulator), _ptr(addend), count, batch,
                                            stream_handle(stream)))


def broadcast(destination, source, count: int, destination_stride: int, batch: int,
              stream=None, bf16: Optional[bool] = None) -> None:
    bf16 = bf16 if bf16 is not None else _bf16(destination)
    fn = library().cuvit_broadcast_bf16 if bf16 else library().cuvit_broadcast_f32
    if _positive(count, batch) and destination_stride >= count:
        destination = _operand(destination, "destination", _storage(bf16),
                               (batch - 1) * destination_stride + count)
        source = _operand(source, "source", _storage(bf16), count)
    check(fn(_ptr(destination), _ptr(source), count, destination_stride, batch,
             stream_handle(stream)))


def convert_to_bf16(x, out, count: int, stream=None) -> None:
    """fp32 -> bf16, round to nearest-even (an extension)."""
    if _positive(count):
        x, out = _operand(x, "x", "float32", count), _operand(out, "out", "bfloat16", count)
    check(library().cuvit_convert_f32_to_bf16(_ptr(x), _ptr(out), count, stream_handle(stream)))


def convert_to_f32(x, out, count: int, stream=None) -> None:
    """bf16 -> fp32, exact (an extension)."""
    if _positive(count):
        x, out = _operand(x, "x", "bfloat16", count), _operand(out, "out", "float32", count)
    check(library().cuvit_convert_bf16_to_f32(_ptr(x), _ptr(out), count, stream_handle(stream)))


def attention_supported(tokens: int, head_dim: int) -> bool:
    """True when the fused attention kernel covers (tokens, head_dim)."""
    return bool(library().cuvit_attention_supported(tokens, head_dim))


def attention(qkv, context, images: int, heads: int, tokens: int, head_dim: int,
              stream=None) -> None:
    """Fused softmax(Q.K^T / sqrt(head_dim)).V from the packed
    [images, tokens, 3, heads, head_dim] projection into
    [images, tokens, heads, head_dim]; an extension replacing the reference's
    three attention launches (vit.cu:205-245) with bitwise the same result."""
    status = _native_calls.attention(qkv, context, images, heads, tokens, head_dim, stream)
    if status >= 0:
        return check(status)
    bf16 = _bf16(qkv)
    fn = library().cuvit_attention_bf16 if bf16 else library().cuvit_attention_f32
    if _positive(images, heads, tokens, head_dim):
        n = images * tokens * heads * head_dim
        qkv = _operand(qkv, "qkv", _storage(bf16), 3 * n)
        context = _operand(context, "context", _storage(bf16), n)
    check(fn(_ptr(qkv), _ptr(context), images, heads, tokens, head_dim, stream_handle(stream)))


def _launch_device(stream, *operands) -> None:
    """Refuses operands that are on another GPU than the launch: a kernel there
    would reach into this one's memory, or fault."""
    tensors = [x for x in operands if x is not None and not isinstance(x, int) and x.device.type == "cuda"]
    if not tensors:
        return
    import torch

    index = stream.device.index if stream is not None else torch.cuda.current_device()
    for x in tensors:
        if x.device.index != index:
            raise InvalidArgument(ERROR_INVALID_ARGUMENT,
                                  f"an operand is on {x.device}, the launch on cuda:{index}")


def _pair_counts(pairs):
    counts = [int(p) for p in pairs]
    return len(counts), (ctypes.c_int * max(len(counts), 1))(*counts)


def rotary_problem(images: int, tokens: int, heads: int, head_dim: int, pairs,
                   pairing: int = ROTARY_HALVES) -> RotaryProblem:
    """The rotation of packed [images, tokens, heads, head_dim] heads, ``pairs``
    counting each axis' pairs (at most three axes; head_dim // 2 pairs in all
    turn whole heads). A ladder of frequencies for an axis of n pairs is
    ``base ** (-i / n)``, i from 0."""
    problem = RotaryProblem()
    axes, counts = _pair_counts(pairs)
    library().cuvit_rotary_problem_init(ctypes.byref(problem), images, tokens, heads, head_dim, axes, counts, pairing)
    return problem


def qk_norm_problem(images: int, tokens: int, heads: int, head_dim: int, pairs=(),
                    pairing: int = ROTARY_HALVES, norm: int = NORM_RMS, epsilon: float = 1.0e-6,
                    kv_heads: Optional[int] = None) -> QkNormProblem:
    """The norm (and rotation, if there are pairs) of a packed projection
    [images, tokens, heads + 2 kv_heads, head_dim]; kv_heads as many as heads
    unless given."""
    problem = QkNormProblem()
    axes, counts = _pair_counts(pairs)
    library().cuvit_qk_norm_problem_init(ctypes.byref(problem), images, tokens, heads, head_dim, axes, counts,
                                         pairing, norm)
    problem.epsilon = epsilon
    if kv_heads is not None:
        problem.kv_heads = kv_heads
    return problem


def gated_problem(m: int, n: int, k: int, activation: int = GATE_SILU) -> GatedProblem:
    """A gated product of packed operands: A [m, k], B [2 n, k], C [m, n]."""
    problem = GatedProblem()
    library().cuvit_gated_problem_init(ctypes.byref(problem), m, n, k, activation)
    return problem


def _rotation_operands(rotation: Rotation, images: int, tokens: int, positions, frequencies):
    if not 0 <= rotation.axes <= 3 or rotation.position_stride < 0:
        return _ptr(positions), _ptr(frequencies)  # the library names what is wrong
    total = sum(rotation.pairs[:rotation.axes])
    if total <= 0 or min(rotation.pairs[:rotation.axes]) < 0:
        return _ptr(positions), _ptr(frequencies)
    reach = (images - 1) * rotation.position_stride + tokens * rotation.axes
    return (_operand(positions, "positions", "float32", reach),
            _operand(frequencies, "frequencies", "float32", total))


def rotary(x, positions, frequencies, out, problem: RotaryProblem, stream=None, bf16: Optional[bool] = None) -> None:
    """Rotates heads by their tokens' positions on up to three axes (row and
    column of a patch; time too): pair i of a token turns by
    ``positions[token, axis of i] * frequencies[i]`` radians, the angle taken in
    64 bits. x and out are [images, tokens, heads, head_dim], or as the problem's
    strides say; out may be x. ``problem.inverse`` turns back, which is also the
    gradient: grad_x is the inverse rotation of grad_out. An extension."""
    status = _native_calls.rotary(x, positions, frequencies, out, problem, stream, bf16)
    if status >= 0:
        return check(status)
    bf16 = bf16 if bf16 is not None else _bf16(x)
    fn = library().cuvit_rotary_bf16 if bf16 else library().cuvit_rotary_f32
    p = problem
    if _positive(p.images, p.tokens, p.heads, p.head_dim):
        _launch_device(stream, x, positions, frequencies, out)

        def reach(s: HeadStrides) -> int:
            return ((p.images - 1) * (s.image or p.tokens * p.heads * p.head_dim)
                    + (p.tokens - 1) * (s.token or p.heads * p.head_dim)
                    + (p.heads - 1) * (s.head or p.head_dim) + p.head_dim)

        positions, frequencies = _rotation_operands(p.rotation, p.images, p.tokens, positions, frequencies)
        x = _operand(x, "x", _storage(bf16), reach(p.input))
        out = _operand(out, "out", _storage(bf16), reach(p.output))
    check(fn(_ptr(x), _ptr(positions), _ptr(frequencies), _ptr(out), ctypes.byref(problem), stream_handle(stream)))


def _qk_norm_operands(p: QkNormProblem, bf16: bool, packed, weights, positions, frequencies):
    values = p.images * p.tokens * (p.heads + 2 * p.kv_heads) * p.head_dim
    positions, frequencies = _rotation_operands(p.rotation, p.images, p.tokens, positions, frequencies)
    return ([_operand(x, name, _storage(bf16), values) for name, x in packed.items()],
            [_operand(x, name, "float32", p.head_dim) for name, x in weights.items()], positions, frequencies)


def qk_norm_rotary(qkv, q_gamma, k_gamma, positions, frequencies, out, problem: QkNormProblem, q_beta=None,
                   k_beta=None, stream=None, bf16: Optional[bool] = None) -> None:
    """Normalises each query and key head of a packed projection
    [images, tokens, heads + 2 kv_heads, head_dim], scales (gamma), shifts (beta)
    and rotates it, in one pass. out may be qkv: the value heads then stay, else
    they are copied. With kv_heads = heads the result is attention()'s qkv.
    gamma and beta are [head_dim] fp32, None for 1 and 0. An extension."""
    status = _native_calls.qk_norm_rotary(qkv, q_gamma, k_gamma, positions, frequencies, out, problem, q_beta,
                                          k_beta, stream, bf16)
    if status >= 0:
        return check(status)
    bf16 = bf16 if bf16 is not None else _bf16(qkv)
    fn = library().cuvit_qk_norm_rotary_bf16 if bf16 else library().cuvit_qk_norm_rotary_f32
    p = problem
    if _positive(p.images, p.tokens, p.heads, p.kv_heads, p.head_dim):
        _launch_device(stream, qkv, q_gamma, k_gamma, positions, frequencies, out, q_beta, k_beta)
        (qkv, out), (q_gamma, k_gamma, q_beta, k_beta), positions, frequencies = _qk_norm_operands(
            p, bf16, {"qkv": qkv, "out": out},
            {"q_gamma": q_gamma, "k_gamma": k_gamma, "q_beta": q_beta, "k_beta": k_beta}, positions, frequencies)
    check(fn(_ptr(qkv), _ptr(q_gamma), _ptr(q_beta), _ptr(k_gamma), _ptr(k_beta), _ptr(positions),
             _ptr(frequencies), _ptr(out), ctypes.byref(problem), stream_handle(stream)))


def qk_norm_rotary_workspace(problem: QkNormProblem) -> int:
    """Bytes of the workspace that qk_norm_rotary_backward() sums in."""
    return library().cuvit_qk_norm_rotary_workspace(ctypes.byref(problem))


def qk_norm_rotary_backward(qkv, q_gamma, k_gamma, positions, frequencies, grad_out, grad_qkv,
                            problem: QkNormProblem, workspace=None, grad_q_gamma=None, grad_k_gamma=None,
                            grad_q_beta=None, grad_k_beta=None, stream=None, bf16: Optional[bool] = None) -> None:
    """The gradients of qk_norm_rotary() from its input qkv and the gradient of
    its whole packed output; grad_qkv may be grad_out. The gradients of gamma and
    beta ([head_dim] fp32, overwritten, None: not computed) are summed in
    ``workspace``, a uint8 tensor of qk_norm_rotary_workspace() bytes that one
    call uses at a time: calls on several streams, and captured graphs that may
    overlap, take one each."""
    status = _native_calls.qk_norm_rotary_backward(qkv, q_gamma, k_gamma, positions, frequencies, grad_out, grad_qkv,
                                                   problem, workspace, grad_q_gamma, grad_k_gamma, grad_q_beta,
                                                   grad_k_beta, stream, bf16)
    if status >= 0:
        return check(status)
    bf16 = bf16 if bf16 is not None else _bf16(qkv)
    fn = library().cuvit_qk_norm_rotary_backward_bf16 if bf16 else library().cuvit_qk_norm_rotary_backward_f32
    p = problem
    nbytes = qk_norm_rotary_workspace(p)
    if _positive(p.images, p.tokens, p.heads, p.kv_heads, p.head_dim):
        _launch_device(stream, qkv, q_gamma, k_gamma, positions, frequencies, grad_out, grad_qkv, workspace,
                       grad_q_gamma, grad_k_gamma, grad_q_beta, grad_k_beta)
        packed, weights, positions, frequencies = _qk_norm_operands(
            p, bf16, {"qkv": qkv, "grad_out": grad_out, "grad_qkv": grad_qkv},
            {"q_gamma": q_gamma, "k_gamma": k_gamma, "grad_q_gamma": grad_q_gamma, "grad_k_gamma": grad_k_gamma,
             "grad_q_beta": grad_q_beta, "grad_k_beta": grad_k_beta}, positions, frequencies)
        qkv, grad_out, grad_qkv = packed
        q_gamma, k_gamma, grad_q_gamma, grad_k_gamma, grad_q_beta, grad_k_beta = weights
        workspace = _operand(workspace, "workspace", "uint8", nbytes)
    elif _positive(p.heads, p.head_dim):  # no tokens: the gradients are zeros
        _launch_device(stream, grad_q_gamma, grad_k_gamma, grad_q_beta, grad_k_beta)
        grad_q_gamma, grad_k_gamma, grad_q_beta, grad_k_beta = (
            _operand(x, name, "float32", p.head_dim) for name, x in
            (("grad_q_gamma", grad_q_gamma), ("grad_k_gamma", grad_k_gamma), ("grad_q_beta", grad_q_beta),
             ("grad_k_beta", grad_k_beta)))
    check(fn(_ptr(qkv), _ptr(q_gamma), _ptr(k_gamma), _ptr(positions), _ptr(frequencies), _ptr(grad_out),
             _ptr(grad_qkv), _ptr(grad_q_gamma), _ptr(grad_q_beta), _ptr(grad_k_gamma), _ptr(grad_k_beta),
             _ptr(workspace), nbytes, ctypes.byref(problem), stream_handle(stream)))


def _gated_reach(p: GatedProblem):
    """Elements that C and the preactivations reach, or None where a leading
    dimension is too small (the library names it)."""
    ldc, ld_pre = p.ldc or p.n, p.ld_preactivations or 2 * p.n
    if ldc < p.n or ld_pre < 2 * p.n:
        return None
    return (p.m - 1) * ldc + p.n, (p.m - 1) * ld_pre + 2 * p.n


def gated_gemm(a, b, bias, c, problem: GatedProblem, preactivations=None, stream=None,
               bf16: Optional[bool] = None) -> None:
    """C = activation(gate) * value with [gate, value] = A.B^T + bias: a gated
    MLP's first product. B is a Linear layer's weight [2 n, k], the gate's n rows
    first, bias [2 n] fp32 or None. A ``preactivations`` tensor [m, 2 n] receives
    [gate, value], for gated_backward(). An extension."""
    status = _native_calls.gated_gemm(a, b, bias, c, problem, preactivations, stream, bf16)
    if status >= 0:
        return check(status)
    bf16 = bf16 if bf16 is not None else _bf16(a)
    fn = library().cuvit_gated_gemm_bf16 if bf16 else library().cuvit_gated_gemm_f32
    p = problem
    if _positive(p.m, p.n) and p.k >= 0:
        _launch_device(stream, a, b, bias, c, preactivations)
        reach = _gated_reach(p)
        lda, ldb = p.lda or p.k, p.ldb or p.k
        if reach is not None and lda >= p.k and ldb >= p.k:
            t = _storage(bf16)
            a = _operand(a, "A", t, (p.m - 1) * lda + p.k)
            b = _operand(b, "B", t, (2 * p.n - 1) * ldb + p.k)
            bias = _operand(bias, "bias", "float32", 2 * p.n)
            c = _operand(c, "C", t, reach[0])
            preactivations = _operand(preactivations, "preactivations", t, reach[1])
    check(fn(_ptr(a), _ptr(b), _ptr(bias), _ptr(c), _ptr(preactivations), ctypes.byref(problem),
             stream_handle(stream)))


def gated_backward(preactivations, grad, grad_preactivations, problem: GatedProblem, stream=None,
                   bf16: Optional[bool] = None) -> None:
    """The gate's gradient: from the preactivations [m, 2 n] that gated_gemm()
    kept and the gradient [m, n] of its result, the gradient of the
    preactivations (which may take their place). The gradients of A and of the
    weight are plain products with it. An extension."""
    status = _native_calls.gated_backward(preactivations, grad, grad_preactivations, problem, stream, bf16)
    if status >= 0:
        return check(status)
    bf16 = bf16 if bf16 is not None else _bf16(preactivations)
    fn = library().cuvit_gated_backward_bf16 if bf16 else library().cuvit_gated_backward_f32
    p = problem
    if _positive(p.m, p.n):
        _launch_device(stream, preactivations, grad, grad_preactivations)
        reach = _gated_reach(p)
        if reach is not None:
            t = _storage(bf16)
            preactivations = _operand(preactivations, "preactivations", t, reach[1])
            grad = _operand(grad, "grad", t, reach[0])
            grad_preactivations = _operand(grad_preactivations, "grad_preactivations", t, reach[1])
    check(fn(_ptr(preactivations), _ptr(grad), _ptr(grad_preactivations), ctypes.byref(problem),
             stream_handle(stream)))


def gated_checkpoint_scales(problem: GatedProblem) -> int:
    """How many scales a gated product's codes have: 2 ceil(n / 32) a row."""
    return library().cuvit_gated_checkpoint_scales(ctypes.byref(problem))


def gated_checkpoint_gemm(a, b, bias, c, codes, scales, problem: GatedProblem, stream=None,
                          bf16: Optional[bool] = None) -> None:
    """gated_gemm() that keeps [gate, value] in 8 bits, for
    gated_checkpoint_backward(): ``codes`` [m, 2 n] float8_e4m3fn and ``scales``
    [m, 2 ceil(n / 32)] float8_e8m0fnu, a power of two for every 32 columns of a
    half. Values are rounded once, from their fp32 sums; infinities and NaN become
    NaN. An extension."""
    status = _native_calls.gated_checkpoint_gemm(a, b, bias, c, codes, scales, problem, stream, bf16)
    if status >= 0:
        return check(status)
    bf16 = bf16 if bf16 is not None else _bf16(a)
    fn = library().cuvit_gated_checkpoint_gemm_bf16 if bf16 else library().cuvit_gated_checkpoint_gemm_f32
    p = problem
    if _positive(p.m, p.n) and p.k >= 0:
        _launch_device(stream, a, b, bias, c, codes, scales)
        reach = _gated_reach(p)
        lda, ldb = p.lda or p.k, p.ldb or p.k
        if reach is not None and lda >= p.k and ldb >= p.k:
            t = _storage(bf16)
            a = _operand(a, "A", t, (p.m - 1) * lda + p.k)
            b = _operand(b, "B", t, (2 * p.n - 1) * ldb + p.k)
            bias = _operand(bias, "bias", "float32", 2 * p.n)
            c = _operand(c, "C", t, reach[0])
            codes = _operand(codes, "codes", "float8_e4m3fn", reach[1])
            scales = _operand(scales, "scales", "float8_e8m0fnu", gated_checkpoint_scales(p))
    check(fn(_ptr(a), _ptr(b), _ptr(bias), _ptr(c), _ptr(codes), _ptr(scales), ctypes.byref(problem),
             stream_handle(stream)))


def gated_checkpoint_backward(codes, scales, grad, grad_preactivations, problem: GatedProblem, hidden=None,
                              stream=None, bf16: Optional[bool] = None) -> None:
    """gated_backward() from the codes and scales that gated_checkpoint_gemm()
    kept. A ``hidden`` tensor [m, n] receives activation(gate) * value again, as
    the codes have them, for the gradient of the weight behind the product; it may
    be ``grad``. An extension."""
    status = _native_calls.gated_checkpoint_backward(codes, scales, grad, grad_preactivations, problem, hidden,
                                                     stream, bf16)
    if status >= 0:
        return check(status)
    bf16 = bf16 if bf16 is not None else _bf16(grad)
    fn = library().cuvit_gated_checkpoint_backward_bf16 if bf16 else library().cuvit_gated_checkpoint_backward_f32
    p = problem
    if _positive(p.m, p.n):
        _launch_device(stream, codes, scales, grad, grad_preactivations, hidden)
        reach = _gated_reach(p)
        if reach is not None:
            t = _storage(bf16)
            codes = _operand(codes, "codes", "float8_e4m3fn", reach[1])
            scales = _operand(scales, "scales", "float8_e8m0fnu", gated_checkpoint_scales(p))
            grad = _operand(grad, "grad", t, reach[0])
            grad_preactivations = _operand(grad_preactivations, "grad_preactivations", t, reach[1])
            hidden = _operand(hidden, "hidden", t, reach[0])
    check(fn(_ptr(codes), _ptr(scales), _ptr(grad), _ptr(grad_preactivations), _ptr(hidden), ctypes.byref(problem),
             stream_handle(stream)))


def packed_attention_problem(sequences: int, tokens: int, heads: int, head_dim: int, kv_heads: Optional[int] = None,
                             kv_tokens: Optional[int] = None, causal: bool = False, scale: float = 0.0,
                             projection: bool = False) -> PackedAttentionProblem:
    """Attention over ``sequences`` packed ones: q and out [tokens, heads,
    head_dim], k and v [kv_tokens, kv_heads, head_dim] (kv_tokens as many as
    tokens, kv_heads as heads unless given), or with ``projection`` all three
    within one [tokens, heads + 2 kv_heads, head_dim], as qk_norm_rotary() leaves
    it. Causal: the last query sees the last key. scale 0 is 1 / sqrt(head_dim)."""
    problem = PackedAttentionProblem()
    library().cuvit_packed_attention_problem_init(ctypes.byref(problem), sequences, tokens, heads, head_dim)
    if kv_heads is not None:
        problem.kv_heads = kv_heads
    if kv_tokens is not None:
        problem.kv_tokens = kv_tokens
    problem.causal = int(causal)
    problem.scale = scale
    if projection:
        library().cuvit_packed_attention_problem_projection(ctypes.byref(problem))
    return problem


def packed_attention_workspace(problem: PackedAttentionProblem) -> int:
    """Bytes of the workspace that packed_attention() needs, 0 for none."""
    return library().cuvit_packed_attention_workspace(ctypes.byref(problem))


def packed_attention_backward_workspace(problem: PackedAttentionProblem) -> int:
    """Bytes of the workspace that packed_attention_backward() needs."""
    return library().cuvit_packed_attention_backward_workspace(ctypes.byref(problem))


def _packed_reach(tokens: int, heads: int, head_dim: int, strides: TokenStrides) -> int:
    if tokens == 0:
        return 0
    return ((tokens - 1) * (strides.token or heads * head_dim) + (heads - 1) * (strides.head or head_dim) + head_dim)


def _packed_operands(p: PackedAttentionProblem, names, q, k, v, bf16: bool):
    """Addresses of q, k and v, or of the projection q where k and v are None."""
    t, size = _storage(bf16), 2 if bf16 else 4
    shared = (p.kv_tokens, p.kv_heads, p.head_dim)
    if k is None and v is None and q is not None and p.kv_tokens > 0:
        if p.kv_tokens != p.tokens:
            raise InvalidArgument(ERROR_INVALID_ARGUMENT, f"{names[0]} without {names[1]} and {names[2]} is a "
                                  "projection, which holds as many keys as queries")
        to_k, to_v = p.heads * p.head_dim, (p.heads + p.kv_heads) * p.head_dim
        reach = max(_packed_reach(p.tokens, p.heads, p.head_dim, p.q), to_k + _packed_reach(*shared, p.k),
                    to_v + _packed_reach(*shared, p.v))
        slots = (p.heads + 2 * p.kv_heads) * p.head_dim
        if any(s.token < slots or s.head not in (0, p.head_dim) for s in (p.q, p.k, p.v)):
            raise InvalidArgument(ERROR_INVALID_ARGUMENT, f"{names[0]} without {names[1]} and {names[2]} is a "
                                  "projection; the problem's strides are not one's (projection=True)")
        q = _operand(q, names[0], t, reach)
        return q, q + to_k * size, q + to_v * size
    return (_operand(q, names[0], t, _packed_reach(p.tokens, p.heads, p.head_dim, p.q)),
            _operand(k, names[1], t, _packed_reach(*shared, p.k)),
            _operand(v, names[2], t, _packed_reach(*shared, p.v)))


def _packed_plain(p: PackedAttentionProblem) -> bool:
    """Whether the operands' sizes follow from the problem; else the library
    names what is wrong, or has nothing to do."""
    return (_positive(p.sequences, p.heads, p.kv_heads, p.head_dim) and p.tokens >= 0 and p.kv_tokens >= 0
            and all(s.token >= 0 and s.head >= 0 for s in (p.q, p.k, p.v, p.out)))


def _packed_starts(p: PackedAttentionProblem, starts, kv_starts, kv_lengths):
    return (_operand(starts, "starts", "int32", p.sequences + 1),
            _operand(kv_starts, "kv_starts", "int32", p.sequences + 1),
            _operand(kv_lengths, "kv_lengths", "int32", p.sequences))


def packed_attention(q, k, v, starts, out, problem: PackedAttentionProblem, kv_starts=None, kv_lengths=None, lse=None,
                     workspace=None, stream=None, bf16: Optional[bool] = None) -> None:
    """out = softmax(scale q.k^T).v within each of the packed sequences: sequence s
    has the queries starts[s] to starts[s + 1] - 1 and the keys kv_starts[s] to
    kv_starts[s + 1] - 1 (kv_starts None: starts), of which with kv_lengths the
    first kv_lengths[s] are filled; all int32 GPU tensors. With k and v None, q is
    a whole projection [tokens, heads + 2 kv_heads, head_dim]. lse, [tokens, heads]
    fp32 or None, receives each row's log-sum-exp, which the gradients need.
    ``workspace``: a uint8 tensor of packed_attention_workspace() bytes (None for
    0) that one call uses at a time. Rows outside every sequence stay as they
    were. An extension."""
    status = _native_calls.packed_attention(q, k, v, starts, out, problem, kv_starts, kv_lengths, lse, workspace,
                                            stream, bf16)
    if status >= 0:
        return check(status)
    bf16 = bf16 if bf16 is not None else _bf16(q)
    fn = library().cuvit_packed_attention_bf16 if bf16 else library().cuvit_packed_attention_f32
    p = problem
    nbytes = packed_attention_workspace(p)
    if _packed_plain(p) and p.tokens > 0:
        _launch_device(stream, q, k, v, starts, out, kv_starts, kv_lengths, lse, workspace)
        q, k, v = _packed_operands(p, ("q", "k", "v"), q, k, v, bf16)
        starts, kv_starts, kv_lengths = _packed_starts(p, starts, kv_starts, kv_lengths)
        out = _operand(out, "out", _storage(bf16), _packed_reach(p.tokens, p.heads, p.head_dim, p.out))
        lse = _operand(lse, "lse", "float32", p.tokens * p.heads)
        workspace = _operand(workspace, "workspace", "uint8", nbytes)
    check(fn(_ptr(q), _ptr(k), _ptr(v), _ptr(starts), _ptr(kv_starts), _ptr(kv_lengths), _ptr(out), _ptr(lse),
             _ptr(workspace), nbytes, ctypes.byref(problem), stream_handle(stream)))


def packed_attention_backward(q, k, v, starts, out, lse, grad_out, grad_q, grad_k, grad_v,
                              problem: PackedAttentionProblem, kv_starts=None, kv_lengths=None, workspace=None,
                              stream=None, bf16: Optional[bool] = None) -> None:
    """The gradients of packed_attention() from its operands, its out and lse and
    the gradient of out. grad_q, grad_k and grad_v are overwritten within the
    sequences; with k and v None, grad_q is the whole projection's gradient and
    grad_k and grad_v are None. ``workspace``: a uint8 tensor of
    packed_attention_backward_workspace() bytes that one call uses at a time:
    calls on several streams, and captured graphs that may overlap, take one
    each. An extension."""
    status = _native_calls.packed_attention_backward(q, k, v, starts, out, lse, grad_out, grad_q, grad_k, grad_v,
                                                     problem, kv_starts, kv_lengths, workspace, stream, bf16)
    if status >= 0:
        return check(status)
    bf16 = bf16 if bf16 is not None else _bf16(q)
    fn = library().cuvit_packed_attention_backward_bf16 if bf16 else library().cuvit_packed_attention_backward_f32
    p = problem
    nbytes = packed_attention_backward_workspace(p)
    if _packed_plain(p) and p.tokens + p.kv_tokens > 0:
        _launch_device(stream, q, k, v, starts, out, lse, grad_out, grad_q, grad_k, grad_v, kv_starts, kv_lengths,
                       workspace)
        if (k is None and v is None) != (grad_k is None and grad_v is None):
            raise InvalidArgument(ERROR_INVALID_ARGUMENT, "a projection's gradient is one tensor, as it is")
        q, k, v = _packed_operands(p, ("q", "k", "v"), q, k, v, bf16)
        grad_q, grad_k, grad_v = _packed_operands(p, ("grad_q", "grad_k", "grad_v"), grad_q, grad_k, grad_v, bf16)
        starts, kv_starts, kv_lengths = _packed_starts(p, starts, kv_starts, kv_lengths)
        reach = _packed_reach(p.tokens, p.heads, p.head_dim, p.out)
        out = _operand(out, "out", _storage(bf16), reach)
        grad_out = _operand(grad_out, "grad_out", _storage(bf16), reach)
        lse = _operand(lse, "lse", "float32", p.tokens * p.heads)
        workspace = _operand(workspace, "workspace", "uint8", nbytes)
    check(fn(_ptr(q), _ptr(k), _ptr(v), _ptr(starts), _ptr(kv_starts), _ptr(kv_lengths), _ptr(out), _ptr(lse),
             _ptr(grad_out), _ptr(grad_q), _ptr(grad_k), _ptr(grad_v), _ptr(workspace), nbytes, ctypes.byref(problem),
             stream_handle(stream)))


class WeightWriter:
    """WeightFileWriter (reference weights.hpp:78-92) over the C ABI."""

    def __init__(self):
        handle = ctypes.c_void_p()
        check(library().cuvit_weight_writer_create(ctypes.byref(handle)))
        self._handle = handle

    def add(self, name: str, array) -> None:
        import numpy as np

        data = np.ascontiguousarray(array, dtype=np.float32)
        extents = (ctypes.c_int64 * max(data.ndim, 1))(*data.shape)
        check(library().cuvit_weight_writer_add(self._handle, name.encode(), data.ndim, extents,
                                                data.ctypes.data))

    def add_bf16(self, name: str, bits) -> None:
        """A bfloat16 tensor from its bit patterns (uint16); the file becomes version 2."""
        import numpy as np

        data = np.ascontiguousarray(bits, dtype=np.uint16)
        extents = (ctypes.c_int64 * max(data.ndim, 1))(*data.shape)
        check(library().cuvit_weight_writer_add_bf16(self._handle, name.encode(), data.ndim,
                                                     extents, data.ctypes.data))

    def write(self, path: str) -> None:
        check(library().cuvit_weight_writer_write(self._handle, os.fsencode(path)))

    def close(self) -> None:
        if getattr(self, "_handle", None):
            library().cuvit_weight_writer_destroy(self._handle)
            self._handle = None

    def __del__(self):
        self.close()


class WeightFile:
    """WeightFile (reference weights.hpp:45-74) over the C ABI."""

    def __init__(self, path: str):
        handle = ctypes.c_void_p()
        check(library().cuvit_weight_file_load(os.fsencode(path), ctypes.byref(handle)))
        self._handle = handle

    @property
    def handle(self):
        return self._handle

    def __len__(self) -> int:
        return library().cuvit_weight_file_size(self._handle)

    def contains(self, name: str) -> bool:
        return bool(library().cuvit_weight_file_contains(self._handle, name.encode()))

    def names(self):
        lib = library()
        return [lib.cuvit_weight_file_entry_name(self._handle, i).decode() for i in range(len(self))]

    def payload_bytes(self) -> int:
        return library().cuvit_weight_file_payload_bytes(self._handle)

    def float_data(self, name: str, shape):
        import numpy as np

        extents = (ctypes.c_int64 * max(len(shape), 1))(*shape)
        pointer = ctypes.c_void_p()
        check(library().cuvit_weight_file_float_data(self._handle, name.encode(), len(shape),
                                                     extents, ctypes.byref(pointer)))
        count = int(np.prod(shape)) if len(shape) else 1
        buffer = (ctypes.c_float * count).from_address(pointer.value) if count else []
        return np.array(np.frombuffer(buffer, dtype=np.float32, count=count)).reshape(shape)

    def bf16_data(self, name: str, shape):
        """The bfloat16 payload's bit patterns (uint16)."""
        import numpy as np

        extents = (ctypes.c_int64 * max(len(shape), 1))(*shape)
        pointer = ctypes.c_void_p()
        check(library().cuvit_weight_file_bf16_data(self._handle, name.encode(), len(shape),
                                                    extents, ctypes.byref(pointer)))
        count = int(np.prod(shape)) if len(shape) else 1
        buffer = (ctypes.c_uint16 * count).from_address(pointer.value) if count else []
        return np.array(np.frombuffer(buffer, dtype=np.uint16, count=count)).reshape(shape)

    @property
    def version(self) -> int:
        return library().cuvit_weight_file_version(self._handle)

    def dtype(self, name: str) -> int:
        """1 for float32, 2 for bfloat16, 0 when absent."""
        return library().cuvit_weight_file_type(self._handle, name.encode())

    def close(self) -> None:
        if getattr(self, "_handle", None):
            library().cuvit_weight_file_destroy(self._handle)
            self._handle = None

    def __del__(self):
        self.close()


def default_config() -> VitConfig:
    config = VitConfig()
    library().cuvit_vit_config_default(ctypes.byref(config))
    return config


def validate_config(config: VitConfig) -> None:
    check(library().cuvit_vit_config_validate(ctypes.byref(config)))


class VisionTransformer:
    """VisionTransformer (reference vit.hpp:53-120) over the C ABI."""

    def __init__(self, config: VitConfig, weights: WeightFile, max_batch: int = 1,
                 precision: int = 0):
        """precision: PRECISION_F32 (the reference's) or PRECISION_BF16 (an extension)."""
        handle = ctypes.c_void_p()
        check(library().cuvit_vit_create_ex(ctypes.byref(config), weights.handle, max_batch,
                                            precision, ctypes.byref(handle)))
        self._handle = handle
        self.config = config
        self.max_batch = max_batch

    @property
    def precision(self) -> int:
        return library().cuvit_vit_precision(self._handle)

    def forward(self, images, logits, batch: int, stream=None) -> None:
        c = self.config
        status = _native_calls.vit_forward(self._handle.value if self._handle else None, images, logits, batch,
                                           c.channels * c.image_size * c.image_size, c.classes, stream)
        if status >= 0:
            return check(status)
        if _positive(batch):
            images = _operand(images, "images", "float32",
                              batch * c.channels * c.image_size * c.image_size)
            logits = _operand(logits, "logits", "float32", batch * c.classes)
        check(library().cuvit_vit_forward(self._handle, _ptr(images), _ptr(logits), batch,
                                          stream_handle(stream)))

    def weight_bytes(self) -> int:
        return library().cuvit_vit_weight_bytes(self._handle)

    def activation_bytes(self) -> int:
        return library().cuvit_vit_activation_bytes(self._handle)

    def close(self) -> None:
        if getattr(self, "_handle", None):
            library().cuvit_vit_destroy(self._handle)
            self._handle = None

    def __del__(self):
        self.close()


def expected_tensor_names(config: VitConfig):
    """VisionTransformer::expected_tensor_names (reference vit.cu:49-63), with shapes."""
    e, t, h = config.embed_dim, config.token_count(), config.mlp_hidden
    names = [("cls_token", (1, 1, e)), ("pos_embed", (1, t, e)),
             ("patch_embed.proj.weight", (e, config.channels, config.patch_size, config.patch_size)),
             ("patch_embed.proj.bias", (e,))]
    for i in range(config.depth):
        p = f"blocks.{i}."
        names += [(p + "norm1.weight", (e,)), (p + "norm1.bias", (e,)),
                  (p + "attn.qkv.weight", (3 * e, e)), (p + "attn.qkv.bias", (3 * e,)),
                  (p + "attn.proj.weight", (e, e)), (p + "attn.proj.bias", (e,)),
                  (p + "norm2.weight", (e,)), (p + "norm2.bias", (e,)),
                  (p + "mlp.fc1.weight", (h, e)), (p + "mlp.fc1.bias", (h,)),
                  (p + "mlp.fc2.weight", (e, h)), (p + "mlp.fc2.bias", (e,))]
    names += [("norm.weight", (e,)), ("norm.bias", (e,)),
              ("head.weight", (config.classes, e)), ("head.bias", (config.classes,))]
    return names


class RgbImage:
    """cuvit::RgbImage (reference image.hpp:12-19): .pixels is a uint8 numpy
    array of shape [height, width, 3], interleaved RGB."""

    def __init__(self, width: int, height: int, pixels):
        self.width = width
        self.height = height
        self.pixels = pixels

    def empty(self) -> bool:
        return self.pixels is None or self.pixels.size == 0


def load_ppm(path: str) -> RgbImage:
    """load_ppm (reference image.cpp:57-93) through the C ABI; a malformed or
    missing file raises CuvitError with the reference's message."""
    import numpy as np

    lib = library()
    handle = ctypes.c_void_p()
    check(lib.cuvit_image_load_ppm(os.fsencode(path), ctypes.byref(handle)))
    try:
        width, height = lib.cuvit_image_width(handle), lib.cuvit_image_height(handle)
        count = width * height * 3
        buffer = (ctypes.c_uint8 * count).from_address(lib.cuvit_image_pixels(handle))
        pixels = np.frombuffer(buffer, dtype=np.uint8).reshape(height, width, 3).copy()
    finally:
        lib.cuvit_image_destroy(handle)
    return RgbImage(width, height, pixels)


def preprocess(pixels, tensor, batch: int, width: int, height: int,
               settings: Optional[Preprocessing] = None, stream=None) -> None:
    """cuvit_preprocess_u8: @p batch device images [batch, height, width, 3]
    uint8 into the device tensor [batch, 3, size, size] float (the reference's
    preprocess, image.cpp:95-135, batched on the GPU)."""
    settings = settings if settings is not None else Preprocessing()
    status = _native_calls.preprocess(pixels, tensor, batch, width, height, settings, stream)
    if status >= 0:
        return check(status)
    if _positive(batch, width, height, settings.size):
        pixels = _operand(pixels, "pixels", "uint8", batch * height * width * 3)
        tensor = _operand(tensor, "tensor", "float32", batch * 3 * settings.size * settings.size)
    check(library().cuvit_preprocess_u8(_ptr(pixels), batch, width, height,
                                        ctypes.byref(settings), _ptr(tensor),
                                        stream_handle(stream)))


def preprocess_image(image: RgbImage, settings: Optional[Preprocessing] = None):
    """The reference's preprocess(image, settings) -> [3, size, size] numpy
    float32, computed on cuda:0 by the library's kernel."""
    import numpy as np
    import torch

    settings = settings if settings is not None else Preprocessing()
    if image.empty():
        raise InvalidArgument(ERROR_INVALID_ARGUMENT, "Cannot preprocess an empty image")
    device = torch.device("cuda:0")
    pixels = torch.from_numpy(np.ascontiguousarray(image.pixels, dtype=np.uint8)).to(device)
    size = settings.size
    tensor = torch.empty(3 * max(size, 0) * max(size, 0), dtype=torch.float32, device=device)
    preprocess(pixels, tensor, 1, image.width, image.height, settings)
    torch.cuda.synchronize()
    return tensor.cpu().numpy().reshape(3, size, size)


def cli_path() -> str:
    """The cu-vit command-line program built beside the library."""
    return os.path.join(os.path.dirname(_HERE), "bin", "cu-vit")
