"""ctypes binding of libfattn.so (include/fattn.h).

The library is the only compute path: if it is missing or fails to load, every call raises
FusedAttentionError -- there is no CPU or composed fallback.
"""
from __future__ import annotations

import ctypes
import importlib.machinery
import importlib.util
from pathlib import Path

import torch  # noqa: F401  -- loaded first, so libfattn binds to torch's HIP runtime

LIB_PATH = Path(__file__).resolve().parent.parent / "lib" / "libfattn.so"
OPERATORS_PATH = LIB_PATH.with_name("torch_operators.so")

# Return codes (include/fattn.h).
FATTN_EINVAL = -1
FATTN_EHEADDIM = -2
FATTN_EALIGN = -3
FATTN_ERANGE = -4
FATTN_EWORKSPACE = -5

# Element types.
DTYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
FP4 = 3  # (of a cache: uint8 tensors)

# Every entry point include/fattn.h declares.
EXPORTS = (
    "fattn_fwd_f32",
    "fattn_bwd_workspace_bytes",
    "fattn_bwd_workspace_min_bytes",
    "fattn_bwd_workspace_split_bytes",
    "fattn_bwd_prep_f32",
    "fattn_bwd_main_f32",
    "fattn_bwd_dq_f32",
    "fattn_bwd_f32",
    "fattn_bwd_f32_noalloc",
    "fattn_fwd_f32_d64",
    "fattn_bwd_prep_f32_d64",
    "fattn_bwd_main_f32_d64",
    "fattn_bwd_dq_f32_d64",
    "fattn_bwd_f32_d64",
    "fattn_qkv_forward",
    "fattn_qkv_backward",
    "fattn_forward",
    "fattn_backward",
    "fattn_rotary",
    "fattn_paged_append",
    "fattn_paged_attention_workspace_bytes",
    "fattn_paged_attention",
    "fattn_paged_scored_attention",
    "fattn_paged_read",
    "fattn_cross_workspace_bytes",
    "fattn_cross_forward",
    "fattn_cross_backward_workspace_bytes",
    "fattn_cross_backward",
    "fattn_scored_workspace_bytes",
    "fattn_scored_forward",
    "fattn_scored_backward_workspace_bytes",
    "fattn_scored_backward",
    "fattn_last_error",
    "fattn_version",
    "fattn_bwd_status",
)


class FusedAttentionError(RuntimeError):
    """An error of the fused attention op; the message carries the reference's prefix
    (`fused_attention:` or `fused_attention_qkv:`), and `code` the C-ABI return code."""

    def __init__(self, msg: str, code: int = 0):
        super().__init__(msg)
        self.code = code


_lib = None
_operators = None

I64 = ctypes.c_int64
P = ctypes.c_void_p
A3 = ctypes.POINTER(ctypes.c_int64)
C_INT = ctypes.c_int
C_FLOAT = ctypes.c_float
C_DOUBLE = ctypes.c_double
SIZE = ctypes.c_size_t


def _declare(L: ctypes.CDLL) -> None:
    L.fattn_last_error.argtypes = []
    L.fattn_last_error.restype = ctypes.c_char_p
    L.fattn_version.argtypes = []
    L.fattn_version.restype = ctypes.c_char_p
    for name in ("fattn_bwd_workspace_bytes", "fattn_bwd_workspace_min_bytes",
                 "fattn_bwd_workspace_split_bytes"):
        getattr(L, name).argtypes = [I64, I64, I64, I64]
        getattr(L, name).restype = SIZE
    for sfx in ("", "_d64"):
        getattr(L, "fattn_fwd_f32" + sfx).argtypes = [P, P, P, P, P, I64, I64, I64, I64, C_FLOAT,
                                                      C_INT, A3, A3, A3, P]
        getattr(L, "fattn_bwd_prep_f32" + sfx).argtypes = [P, P, A3, P, SIZE, I64, I64, I64, I64,
                                                           P]
        getattr(L, "fattn_bwd_main_f32" + sfx).argtypes = [P, P, P, P, P, P, P, P, SIZE, I64,
                                                           I64, I64, I64, C_FLOAT, C_INT, A3, A3,
                                                           A3, A3, P]
        getattr(L, "fattn_bwd_dq_f32" + sfx).argtypes = [P, P, SIZE, I64, I64, I64, I64, C_FLOAT,
                                                         C_INT, P]
        getattr(L, "fattn_bwd_f32" + sfx).argtypes = [P, P, P, P, P, P, P, P, SIZE, I64, I64, I64,
                                                      I64, C_FLOAT, C_INT, A3, A3, A3, A3, P]
    L.fattn_bwd_f32_noalloc.argtypes = [P, P, P, P, P, P, P, I64, I64, I64, I64, C_FLOAT, C_INT,
                                        A3, A3, A3, A3, P]
    L.fattn_qkv_forward.argtypes = [P, I64, A3, A3, I64, C_FLOAT, C_INT, P, P, P]
    L.fattn_qkv_backward.argtypes = [P, I64, A3, A3, I64, C_FLOAT, C_INT, P, P, P, I64, A3, A3,
                                     P, P, SIZE, P]
    L.fattn_forward.argtypes = [P, I64, A3, A3, P, I64, A3, A3, P, I64, A3, A3, C_FLOAT, C_INT,
                                P, P, P]
    L.fattn_backward.argtypes = [P, I64, A3, A3, P, I64, A3, A3, P, I64, A3, A3, C_FLOAT, C_INT,
                                 P, P, P, I64, A3, A3, P, P, SIZE, P]
    # (The operators around self-attention, which torch_operators.so calls: arrays by their addresses.)
    L.fattn_rotary.argtypes = [C_INT, I64, I64, I64, P, P, P, P, P, C_INT, P, C_INT, P, P, I64, C_INT,
                               C_DOUBLE, C_INT, P]
    L.fattn_paged_append.argtypes = [C_INT, C_INT, I64, I64, I64, I64, I64, P, P, P, P, P, P, P, P, P,
                                     P, P, P, I64, I64, P, I64, I64, P, P, P, I64, C_INT, C_DOUBLE, P]
    L.fattn_paged_attention_workspace_bytes.argtypes = [I64, I64, I64, I64, I64]
    L.fattn_paged_attention_workspace_bytes.restype = SIZE
    L.fattn_paged_attention.argtypes = [C_INT, C_INT, I64, I64, I64, I64, P, P, P, P, P, P, P, I64, I64,
                                        P, I64, I64, P, C_FLOAT, P, SIZE, P]
    L.fattn_paged_scored_attention.argtypes = [C_INT, C_INT, I64, I64, I64, I64, P, P, P, P, P, P, P, I64, I64,
                                               P, I64, I64, P, C_FLOAT, C_FLOAT, P, P, SIZE, P]
    L.fattn_paged_read.argtypes = [C_INT, C_INT, I64, I64, I64, I64, P, P, P, P, I64, I64, P, I64, I64, P,
                                   P, P, P, P]
    L.fattn_scored_backward_workspace_bytes.argtypes = [I64, I64, I64, I64, I64, I64, C_INT]
    L.fattn_scored_backward_workspace_bytes.restype = SIZE
    for name in ("fattn_cross_workspace_bytes", "fattn_cross_backward_workspace_bytes",
                 "fattn_scored_workspace_bytes"):
        getattr(L, name).argtypes = [I64, I64, I64, I64, I64, I64]
        getattr(L, name).restype = SIZE
    L.fattn_cross_forward.argtypes = [P, P, P, P, P, P, I64, I64, I64, I64, I64, I64, P, C_FLOAT, P, P,
                                      P, SIZE, P]
    L.fattn_cross_backward.argtypes = [P, P, P, P, P, P, I64, I64, I64, I64, I64, I64, P, C_FLOAT, P, P,
                                       P, P, P, P, P, SIZE, P]
    scored = [P, P, P, P, P, P, I64, I64, I64, I64, I64, I64, C_FLOAT, C_INT, C_FLOAT, P, P, I64, P]
    L.fattn_scored_forward.argtypes = [*scored, P, P, P, SIZE, P]
    L.fattn_scored_backward.argtypes = [*scored, P, P, P, P, P, P, P, SIZE, P]
    L.fattn_bwd_status.argtypes = [P, SIZE, I64, I64, I64, P, ctypes.POINTER(C_INT)]
    for name in EXPORTS:
        if name not in ("fattn_last_error", "fattn_version") and "workspace" not in name:
            getattr(L, name).restype = C_INT


def lib() -> ctypes.CDLL:
    """The loaded libfattn.so; raises FusedAttentionError if it is not built."""
    global _lib
    if _lib is None:
        if not LIB_PATH.exists():
            raise FusedAttentionError(
                f"fused_attention: {LIB_PATH} is not built (run __graft_entry__.build() or "
                "python candle-fused-attn_amd/build.py); there is no fallback path")
        try:
            L = ctypes.CDLL(str(LIB_PATH))
        except OSError as e:
            raise FusedAttentionError(f"fused_attention: cannot load {LIB_PATH}: {e}") from e
        _declare(L)
        _lib = L
    return _lib


def operators():
    """The loaded torch_operators.so (torch tensors to libfattn's operators around self-attention);
    raises FusedAttentionError if it is not built."""
    global _operators
    if _operators is None:
        lib()
        if not OPERATORS_PATH.exists():
            raise FusedAttentionError(
                f"fused_attention: {OPERATORS_PATH} is not built (run __graft_entry__.build() or "
                "python candle-fused-attn_amd/build.py); there is no fallback path")
        loader = importlib.machinery.ExtensionFileLoader("torch_operators", str(OPERATORS_PATH))
        try:
            module = importlib.util.module_from_spec(
                importlib.util.spec_from_loader("torch_operators", loader))
        except ImportError as e:
            raise FusedAttentionError(f"fused_attention: cannot load {OPERATORS_PATH}: {e}") from e
        _operators = module
    return _operators


def last_error() -> str:
    msg = lib().fattn_last_error()
    return msg.decode() if msg else ""


def check(rc: int) -> None:
    if rc != 0:
        raise FusedAttentionError(last_error() or f"fused_attention: error {rc}", rc)


def arr(values) -> ctypes.Array:
    vals = [int(x) for x in values]
    return (ctypes.c_int64 * len(vals))(*vals)


def version() -> str:
    return lib().fattn_version().decode()
