"""ctypes binding of ``libpace_kv_hip.so`` (declared in ``include/pace_kv_hip.h``).

The library is the only implementation of the hot path: if it is missing or a
symbol cannot be resolved this module raises, it never substitutes another path.
"""
from __future__ import annotations

import ctypes
import os
from ctypes import POINTER, Structure, c_char_p, c_float, c_int32, c_int64, c_size_t, c_void_p
from typing import Optional

_LIB_PATH = os.path.join(os.path.dirname(os.path.abspath(__file__)), "_lib", "libpace_kv_hip.so")

BLOCK_TOKENS = 16
DTYPE_F32, DTYPE_BF16 = 0, 1
ABI_VERSION = 15
STATIC_SCRATCH_BYTES = 32 << 20  # PACE_PAGED_ATTN_STATIC_SCRATCH_BYTES
ELEM_Q4 = 1  # PACE_KV_ELEM_Q4: pools of 4-bit rows, strides in bytes
HEAD_DIMS = (64, 96, 128, 256)  # head sizes the pool kernels are built for

EXPORTED_SYMBOLS = (
    "pace_kv_last_error",
    "pace_kv_abi_version",
    "pace_kv_append",
    "pace_kv_append_paged",
    "pace_kv_append_paged_at",
    "pace_kv_gather",
    "pace_kv_gather_packed",
    "pace_kv_gather_live",
    "pace_kv_copy_blocks",
    "pace_rope_apply",
    "pace_rope_apply_f32",
    "pace_rope_append_paged",
    "pace_paged_attn_partition_tokens",
    "pace_paged_attn_plan",
    "pace_paged_attn_kernel_name",
    "pace_kv_plan_compaction",
    "pace_kv_apply_moves",
    "pace_kv_apply_moves_tracked",
    "pace_kv_plan_compaction_flags",
    "pace_paged_attn_workspace_bytes",
    "pace_paged_attn_workspace_bytes_for_parts",
    "pace_paged_attn_workspace_for",
    "pace_paged_attn_decode",
    "pace_paged_attn_verify",
    "pace_paged_attn_verify_static",
    "pace_kv_compact_blocks",
    "pace_attn_dense",
    "pace_attn_dense_ws",
    "pace_attn_dense_workspace_bytes",
)


class PoolDesc(Structure):
    """``pace_kv_pool_t``."""

    _fields_ = [
        ("k", c_void_p),
        ("v", c_void_p),
        ("k_block_stride", c_int64),
        ("k_head_stride", c_int64),
        ("v_block_stride", c_int64),
        ("v_head_stride", c_int64),
        ("num_blocks", c_int32),
        ("num_kv_heads", c_int32),
        ("head_dim", c_int32),
        ("block_size", c_int32),
        ("elem_bytes", c_int32),  # 0 / 2: bf16 slabs, 4: fp32 rows, ELEM_Q4: 4-bit rows
        ("reserved", c_int32),
    ]


class RopeDesc(Structure):
    """``pace_rope_t``."""

    _fields_ = [
        ("cos", c_void_p),
        ("sin", c_void_p),
        ("table_dtype", c_int32),
        ("table_rows", c_int32),
        ("rotary_dim", c_int32),
        ("interleaved", c_int32),
        ("positions", c_void_p),
        ("pos_stride_b", c_int32),
    ]


class PagedAttnArgs(Structure):
    """``pace_paged_attn_args_t``."""

    _fields_ = [
        ("q", c_void_p),
        ("q_stride_b", c_int64),
        ("q_stride_h", c_int64),
        ("q_stride_s", c_int64),
        ("out", c_void_p),
        ("o_stride_b", c_int64),
        ("o_stride_h", c_int64),
        ("o_stride_s", c_int64),
        ("block_table", c_void_p),
        ("table_stride", c_int32),
        ("seq_lens", c_void_p),
        ("kv_start", c_void_p),
        ("mask", c_void_p),
        ("mask_dtype", c_int32),
        ("mask_len", c_int32),
        ("mask_stride_b", c_int64),
        ("mask_stride_s", c_int64),
        ("batch", c_int32),
        ("num_q_heads", c_int32),
        ("q_len", c_int32),
        ("causal", c_int32),
        ("max_seq_len", c_int32),
        ("partition_tokens", c_int32),
        ("scale", c_float),
        ("workspace", c_void_p),
        ("workspace_bytes", c_size_t),
        ("k_new", c_void_p),
        ("v_new", c_void_p),
        ("new_stride_b", c_int64),
        ("new_stride_h", c_int64),
        ("new_stride_t", c_int64),
        ("n_new", c_int32),
        ("work_items", c_void_p),
        ("n_work_items", c_int32),
        ("seq_parts", c_void_p),
        ("max_parts", c_int32),
        ("seq_len_bias", c_int32),
        ("rope", POINTER(RopeDesc)),
        ("seq_len_bias_ptr", c_void_p),
        ("window", c_int32),
        ("sinks", c_int32),
    ]


class AttnPlan(Structure):
    """``pace_attn_plan_t``."""

    _fields_ = [
        ("n_work_items", c_int32),
        ("max_parts", c_int32),
        ("partition_tokens", c_int32),
        ("reserved", c_int32),
        ("workspace_bytes", c_size_t),
    ]


WORK_INTS = 16  # PACE_ATTN_WORK_INTS: int32 per work descriptor


class NativeError(RuntimeError):
    """A C-ABI entry point returned a failure code."""


_lib: Optional[ctypes.CDLL] = None


def library_path() -> str:
    return _LIB_PATH


def load() -> ctypes.CDLL:
    """Load the shared library once and declare every prototype."""
    global _lib
    if _lib is not None:
        return _lib
    if not os.path.exists(_LIB_PATH):
        raise ImportError(
            f"{_LIB_PATH} is missing: build it with `python amd-pace_amd/build.py` "
            "(hipcc, gfx950). There is no other implementation of this path."
        )
    lib = ctypes.CDLL(_LIB_PATH)
    P = POINTER(PoolDesc)
    lib.pace_kv_last_error.restype = c_char_p
    lib.pace_kv_last_error.argtypes = []
    lib.pace_kv_abi_version.restype = c_int32
    lib.pace_kv_abi_version.argtypes = []
    lib.pace_kv_append.restype = ctypes.c_int
    lib.pace_kv_append.argtypes = [P, c_void_p, c_void_p, c_int64, c_int64, c_int64, c_int32, c_int32, c_void_p, c_void_p]
    lib.pace_kv_append_paged.restype = ctypes.c_int
    lib.pace_kv_append_paged.argtypes = [
        P, c_void_p, c_void_p, c_int64, c_int64, c_int64, c_int32, c_int32,
        c_void_p, c_int32, c_void_p, c_int32, c_void_p,
    ]
    lib.pace_kv_append_paged_at.restype = ctypes.c_int
    lib.pace_kv_append_paged_at.argtypes = [
        P, c_void_p, c_void_p, c_int64, c_int64, c_int64, c_int32, c_int32,
        c_void_p, c_int32, c_void_p, c_int32, c_void_p, c_void_p,
    ]
    lib.pace_kv_gather.restype = ctypes.c_int
    lib.pace_kv_gather.argtypes = [
        P, c_void_p, c_int32, c_void_p, c_int32, c_int32, c_int32, c_void_p, c_void_p, c_int64, c_int64, c_int32, c_int32, c_void_p,
    ]
    lib.pace_kv_gather_packed.restype = ctypes.c_int
    lib.pace_kv_gather_packed.argtypes = [
        P, c_void_p, c_int32, c_void_p, c_int32, c_void_p, c_int32, c_int32, c_void_p, c_void_p, c_int32, c_void_p,
    ]
    lib.pace_kv_gather_live.restype = ctypes.c_int
    lib.pace_kv_gather_live.argtypes = [
        P, c_void_p, c_int32, c_void_p, c_int32, c_void_p, c_int32, c_int32, c_void_p, c_void_p, c_int64, c_int64, c_int32, c_int32, c_void_p,
    ]
    lib.pace_kv_copy_blocks.restype = ctypes.c_int
    lib.pace_kv_copy_blocks.argtypes = [P, P, c_void_p, c_int32, c_void_p]
    R = POINTER(RopeDesc)
    rows = [c_void_p, c_void_p, c_int64, c_int64, c_int64, c_int32]  # in, out, strides b/h/t, heads
    lib.pace_rope_apply.restype = ctypes.c_int
    lib.pace_rope_apply.argtypes = [R] + rows + rows + [c_int32, c_int32, c_int32, c_void_p]
    lib.pace_rope_apply_f32.restype = ctypes.c_int
    lib.pace_rope_apply_f32.argtypes = [R] + rows + rows + [c_int32, c_int32, c_int32, c_void_p]
    lib.pace_rope_append_paged.restype = ctypes.c_int
    lib.pace_rope_append_paged.argtypes = (
        [P, R] + rows + [c_void_p, c_void_p, c_int64, c_int64, c_int64, c_int32, c_int32]
        + [c_void_p, c_int32, c_void_p, c_int32, c_void_p]
    )
    lib.pace_paged_attn_partition_tokens.restype = c_int32
    lib.pace_paged_attn_partition_tokens.argtypes = [c_int32] * 7
    lib.pace_paged_attn_plan.restype = ctypes.c_int
    lib.pace_paged_attn_plan.argtypes = [c_void_p, c_void_p] + [c_int32] * 8 + [c_void_p, c_int32, c_void_p, POINTER(AttnPlan)]
    lib.pace_paged_attn_kernel_name.restype = ctypes.c_int
    lib.pace_paged_attn_kernel_name.argtypes = [P, POINTER(PagedAttnArgs), ctypes.c_char_p, c_size_t]
    lib.pace_kv_plan_compaction.restype = c_int32
    lib.pace_kv_plan_compaction.argtypes = [c_void_p, c_int32, c_void_p, c_int32, c_int32, c_void_p, c_int32, c_int32, c_void_p]
    lib.pace_kv_apply_moves.restype = ctypes.c_int
    lib.pace_kv_apply_moves.argtypes = [c_void_p, c_int32, c_void_p, c_int32, c_int32, c_void_p, c_int32, c_void_p]
    lib.pace_paged_attn_workspace_bytes.restype = c_size_t
    lib.pace_paged_attn_workspace_bytes.argtypes = [c_int32] * 7
    lib.pace_paged_attn_workspace_bytes_for_parts.restype = c_size_t
    lib.pace_paged_attn_workspace_bytes_for_parts.argtypes = [c_int32] * 5
    A = POINTER(PagedAttnArgs)
    lib.pace_paged_attn_workspace_for.restype = c_size_t
    lib.pace_paged_attn_workspace_for.argtypes = [P, A]
    lib.pace_paged_attn_decode.restype = ctypes.c_int
    lib.pace_paged_attn_decode.argtypes = [P, A, c_void_p]
    lib.pace_paged_attn_verify.restype = ctypes.c_int
    lib.pace_paged_attn_verify.argtypes = [P, A, c_void_p]
    lib.pace_paged_attn_verify_static.restype = ctypes.c_int
    lib.pace_paged_attn_verify_static.argtypes = [P, A, c_void_p]
    lib.pace_attn_dense.restype = ctypes.c_int
    lib.pace_attn_dense.argtypes = [
        c_void_p, c_void_p, c_void_p, c_void_p, c_int32, c_int32, c_int32, c_int32, c_int32, c_int32,
        c_void_p, c_int32, c_int32, c_int32, c_int32, c_void_p,
    ]
    lib.pace_kv_compact_blocks.restype = c_int32
    lib.pace_kv_compact_blocks.argtypes = [c_void_p, c_int32, c_void_p, c_int32, c_void_p, c_int32, c_void_p, c_void_p, c_int32, c_void_p,
                                           c_void_p]
    lib.pace_kv_plan_compaction_flags.restype = c_int32
    lib.pace_kv_plan_compaction_flags.argtypes = [c_void_p, c_int32, c_void_p, c_int32]
    lib.pace_kv_apply_moves_tracked.restype = ctypes.c_int
    lib.pace_kv_apply_moves_tracked.argtypes = [c_void_p, c_int32, c_void_p, c_int32, c_int32, c_void_p, c_int32, c_void_p, c_void_p, c_void_p,
                                                c_void_p]
    lib.pace_attn_dense_ws.restype = ctypes.c_int
    lib.pace_attn_dense_ws.argtypes = [
        c_void_p, c_void_p, c_void_p, c_void_p, c_int32, c_int32, c_int32, c_int32, c_int32, c_int32,
        c_void_p, c_int32, c_int32, c_int32, c_int32, c_void_p, ctypes.c_size_t, c_void_p,
    ]
    lib.pace_attn_dense_workspace_bytes.restype = ctypes.c_size_t
    lib.pace_attn_dense_workspace_bytes.argtypes = [c_int32] * 7
    got = int(lib.pace_kv_abi_version())
    if got != ABI_VERSION:
        raise ImportError(f"{_LIB_PATH} has ABI version {got}, this package needs {ABI_VERSION}: rebuild it")
    _lib = lib
    return lib


def kernel_name(pool_desc: PoolDesc, args: PagedAttnArgs) -> str:
    """The kernel instantiation an attention call with these arguments launches (nothing is launched)."""
    buf = ctypes.create_string_buffer(256)
    check(load().pace_paged_attn_kernel_name(ctypes.byref(pool_desc), ctypes.byref(args), buf, len(buf)))
    return buf.value.decode()


def check(rc: int) -> None:
    """Raise ``NativeError`` carrying the library's message when ``rc`` is a failure."""
    if rc != 0:
        msg = load().pace_kv_last_error().decode("utf-8", "replace")
        raise NativeError(f"[{rc}] {msg}")


def current_stream_ptr() -> int:
    """Raw ``hipStream_t`` of torch's current stream on the current device."""
    import torch

    raw = getattr(torch._C, "_cuda_getCurrentRawStream", None)
    if raw is not None:  # one C call instead of building a Stream object
        return int(raw(torch.cuda.current_device()))
    return int(torch.cuda.current_stream().cuda_stream)
