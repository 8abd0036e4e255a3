"""ctypes binding of ``libnvamd.so`` (the C ABI in ``include/nvamd.h``).

The wrappers take torch tensors, check shapes the way the reference's Python
layers do (ValueError on a shape mismatch), pass raw device pointers and the
current HIP stream, and raise if the library reports an error.  There is no
fallback: if the library is missing, every call raises, so a test or bench that
passes has run the HIP kernels.
"""
from __future__ import annotations

import ctypes
import importlib
import os
import warnings
from pathlib import Path
from typing import NamedTuple

import torch

LIB_PATH = Path(__file__).resolve().parent / "libnvamd.so"

NVAMD_OK = 0
_ERRORS = {-1: "invalid argument", -2: "unsupported configuration", -3: "workspace missing or too small",
           -4: "needs more than the library's static scratch (NVAMD_DECODE_SCRATCH_BYTES)",
           -5: "first use of the static scratch on this device made while the stream is captured; make one "
               "call outside graph capture first"}
DECODE_SCRATCH_BYTES = 64 * 1024 * 1024  # NVAMD_DECODE_SCRATCH_BYTES

_c_int = ctypes.c_int
_c_i64 = ctypes.c_int64
_c_ptr = ctypes.c_void_p
_c_size = ctypes.c_size_t
_c_float = ctypes.c_float

# name -> (restype, argtypes)
_SIGNATURES = {
    "nvamd_version": (_c_int, []),
    "nvamd_errors_fetch": (_c_int, [_c_ptr, _c_ptr]),
    "nvamd_errors_clear": (_c_int, [_c_ptr]),
    "nvamd_paged_decode_workspace_size": (_c_size, [_c_int, _c_int, _c_int, _c_int]),
    "nvamd_paged_decode": (
        _c_int,
        [_c_ptr, _c_i64, _c_ptr, _c_i64, _c_ptr, _c_ptr, _c_int, _c_int, _c_ptr, _c_int, _c_int, _c_ptr,
         _c_int, _c_int, _c_int, _c_int, _c_float, _c_int, _c_ptr, _c_size, _c_ptr],
    ),
    "nvamd_paged_decode_noalloc": (
        _c_int,
        [_c_ptr, _c_i64, _c_ptr, _c_i64, _c_ptr, _c_ptr, _c_int, _c_int, _c_ptr, _c_int, _c_int, _c_ptr,
         _c_int, _c_int, _c_int, _c_int, _c_float, _c_int, _c_ptr],
    ),
    "nvamd_paged_decode_fused": (
        _c_int,
        [_c_ptr, _c_i64, _c_ptr, _c_i64, _c_ptr, _c_i64, _c_ptr, _c_i64, _c_ptr, _c_ptr, _c_ptr, _c_ptr, _c_int,
         _c_float, _c_ptr, _c_ptr, _c_int, _c_int, _c_ptr, _c_ptr, _c_int, _c_int, _c_ptr, _c_int, _c_int, _c_int,
         _c_int, _c_float, _c_int, _c_ptr, _c_size, _c_ptr],
    ),
    "nvamd_kv_cache_write": (
        _c_int,
        [_c_ptr, _c_i64, _c_ptr, _c_i64, _c_ptr, _c_ptr, _c_ptr, _c_int, _c_int, _c_int, _c_i64, _c_ptr],
    ),
    "nvamd_pack_batch": (
        _c_int,
        [_c_ptr, _c_int, _c_ptr, _c_int, _c_ptr, _c_ptr, _c_int, _c_int, _c_int, _c_ptr, _c_int, _c_int, _c_ptr,
         _c_ptr, _c_ptr, _c_ptr, _c_ptr, _c_ptr, _c_ptr],
    ),
    "nvamd_varlen_prefill": (
        _c_int,
        [_c_ptr, _c_i64, _c_ptr, _c_i64, _c_ptr, _c_i64, _c_ptr, _c_i64, _c_ptr, _c_int, _c_int, _c_int, _c_int,
         _c_int, _c_float, _c_ptr],
    ),
    "nvamd_paged_prefill": (
        _c_int,
        [_c_ptr, _c_i64, _c_ptr, _c_i64, _c_ptr, _c_ptr, _c_int, _c_int, _c_ptr, _c_int, _c_int, _c_ptr, _c_ptr,
         _c_int, _c_int, _c_int, _c_int, _c_int, _c_float, _c_ptr],
    ),
    "nvamd_add_rms_norm": (_c_int, [_c_ptr, _c_ptr, _c_ptr, _c_ptr, _c_int, _c_int, _c_float, _c_ptr]),
    "nvamd_rms_norm_tiled": (_c_int, [_c_ptr, _c_i64, _c_ptr, _c_ptr, _c_int, _c_int, _c_float, _c_ptr]),
    "nvamd_silu_mul": (_c_int, [_c_ptr, _c_i64, _c_ptr, _c_i64, _c_int, _c_int, _c_ptr]),
    "nvamd_argmax_rows": (_c_int, [_c_ptr, _c_i64, _c_int, _c_int, _c_ptr, _c_ptr]),
    "nvamd_skinny_linear_workspace_size": (_c_size, [_c_int, _c_int, _c_int]),
    "nvamd_skinny_linear": (
        _c_int,
        [_c_ptr, _c_i64, _c_ptr, _c_ptr, _c_float, _c_ptr, _c_ptr, _c_i64, _c_ptr, _c_int, _c_int, _c_int, _c_int,
         _c_int, _c_ptr, _c_size, _c_ptr]),
    "nvamd_skinny_linear_rows": (
        _c_int,
        [_c_ptr, _c_i64, _c_ptr, _c_ptr, _c_i64, _c_ptr, _c_int, _c_int, _c_int, _c_int, _c_int, _c_ptr, _c_size,
         _c_ptr]),
    "nvamd_embed_rows": (
        _c_int, [_c_ptr, _c_ptr, _c_i64, _c_int, _c_ptr, _c_i64, _c_int, _c_ptr, _c_int, _c_int, _c_ptr]),
    "nvamd_kv_cache_write_fp4": (
        _c_int,
        [_c_ptr, _c_i64, _c_ptr, _c_i64, _c_ptr, _c_ptr, _c_ptr, _c_ptr, _c_int, _c_int, _c_ptr, _c_int, _c_int,
         _c_int, _c_ptr],
    ),
    "nvamd_kv_cache_read_fp4": (
        _c_int,
        [_c_ptr, _c_i64, _c_ptr, _c_i64, _c_ptr, _c_ptr, _c_ptr, _c_ptr, _c_int, _c_int, _c_ptr, _c_int, _c_int,
         _c_int, _c_ptr],
    ),
    "nvamd_qk_norm_rope_fp4": (
        _c_int,
        [_c_ptr, _c_i64, _c_ptr, _c_i64, _c_ptr, _c_i64, _c_ptr, _c_i64, _c_ptr, _c_i64, _c_ptr, _c_ptr, _c_ptr,
         _c_ptr, _c_int, _c_ptr, _c_ptr, _c_ptr, _c_ptr, _c_int, _c_int, _c_ptr, _c_int, _c_int, _c_int, _c_int,
         _c_float, _c_ptr],
    ),
    "nvamd_paged_decode_fp4": (
        _c_int,
        [_c_ptr, _c_i64, _c_ptr, _c_i64, _c_ptr, _c_ptr, _c_ptr, _c_ptr, _c_int, _c_int, _c_ptr, _c_int, _c_int,
         _c_ptr, _c_int, _c_int, _c_int, _c_int, _c_float, _c_int, _c_ptr, _c_size, _c_ptr],
    ),
    "nvamd_paged_decode_fused_fp4": (
        _c_int,
        [_c_ptr, _c_i64, _c_ptr, _c_i64, _c_ptr, _c_i64, _c_ptr, _c_i64, _c_ptr, _c_ptr, _c_ptr, _c_ptr, _c_int,
         _c_float, _c_ptr, _c_ptr, _c_ptr, _c_ptr, _c_int, _c_int, _c_ptr, _c_ptr, _c_int, _c_int, _c_ptr, _c_int,
         _c_int, _c_int, _c_int, _c_float, _c_int, _c_ptr, _c_size, _c_ptr],
    ),
    "nvamd_paged_prefill_fp4": (
        _c_int,
        [_c_ptr, _c_i64, _c_ptr, _c_i64, _c_ptr, _c_ptr, _c_ptr, _c_ptr, _c_int, _c_int, _c_ptr, _c_int, _c_int,
         _c_ptr, _c_ptr, _c_int, _c_int, _c_int, _c_int, _c_int, _c_int, _c_float, _c_ptr, _c_size, _c_ptr],
    ),
    "nvamd_paged_prefill_fp4_workspace_size": (_c_size, [_c_int, _c_int, _c_int, _c_int, _c_int, _c_int]),
    "nvamd_kv_cache_write_fp8": (
        _c_int,
        [_c_ptr, _c_i64, _c_ptr, _c_i64, _c_ptr, _c_ptr, _c_ptr, _c_ptr, _c_int, _c_int, _c_ptr, _c_int, _c_int,
         _c_int, _c_ptr],
    ),
    "nvamd_kv_cache_read_fp8": (
        _c_int,
        [_c_ptr, _c_i64, _c_ptr, _c_i64, _c_ptr, _c_ptr, _c_ptr, _c_ptr, _c_int, _c_int, _c_ptr, _c_int, _c_int,
         _c_int, _c_ptr],
    ),
    "nvamd_kv_cache_kept_size_fp8": (_c_size, [_c_int, _c_int, _c_int]),
    "nvamd_kv_cache_keep_fp8": (
        _c_int,
        [_c_ptr, _c_size, _c_ptr, _c_ptr, _c_ptr, _c_ptr, _c_int, _c_int, _c_int, _c_ptr, _c_int, _c_int, _c_int, _c_ptr],
    ),
    "nvamd_kv_cache_restore_fp8": (
        _c_int,
        [_c_ptr, _c_size, _c_ptr, _c_ptr, _c_ptr, _c_ptr, _c_int, _c_int, _c_int, _c_int, _c_int, _c_int, _c_ptr],
    ),
    "nvamd_qk_norm_rope_fp8": (
        _c_int,
        [_c_ptr, _c_i64, _c_ptr, _c_i64, _c_ptr, _c_i64, _c_ptr, _c_i64, _c_ptr, _c_i64, _c_ptr, _c_ptr, _c_ptr,
         _c_ptr, _c_int, _c_ptr, _c_ptr, _c_ptr, _c_ptr, _c_int, _c_int, _c_ptr, _c_int, _c_int, _c_int, _c_int,
         _c_float, _c_ptr],
    ),
    "nvamd_paged_decode_fp8": (
        _c_int,
        [_c_ptr, _c_i64, _c_ptr, _c_i64, _c_ptr, _c_ptr, _c_ptr, _c_ptr, _c_int, _c_int, _c_ptr, _c_int, _c_int,
         _c_ptr, _c_int, _c_int, _c_int, _c_int, _c_float, _c_int, _c_ptr, _c_size, _c_ptr],
    ),
    "nvamd_paged_decode_fused_fp8": (
        _c_int,
        [_c_ptr, _c_i64, _c_ptr, _c_i64, _c_ptr, _c_i64, _c_ptr, _c_i64, _c_ptr, _c_ptr, _c_ptr, _c_ptr, _c_int,
         _c_float, _c_ptr, _c_ptr, _c_ptr, _c_ptr, _c_int, _c_int, _c_ptr, _c_ptr, _c_int, _c_int, _c_ptr, _c_int,
         _c_int, _c_int, _c_int, _c_float, _c_int, _c_ptr, _c_size, _c_ptr],
    ),
    "nvamd_paged_prefill_fp8": (
        _c_int,
        [_c_ptr, _c_i64, _c_ptr, _c_i64, _c_ptr, _c_ptr, _c_ptr, _c_ptr, _c_int, _c_int, _c_ptr, _c_int, _c_int,
         _c_ptr, _c_ptr, _c_int, _c_int, _c_int, _c_int, _c_int, _c_int, _c_float, _c_ptr, _c_size, _c_ptr],
    ),
    "nvamd_paged_prefill_fp8_workspace_size": (_c_size, [_c_int, _c_int, _c_int, _c_int, _c_int, _c_int]),
    "nvamd_copy_blocks": (
        _c_int, [_c_ptr, _c_ptr, _c_int, _c_int, _c_int, _c_ptr, _c_ptr, _c_int, _c_ptr]),
    "nvamd_qk_norm_rope": (
        _c_int,
        [_c_ptr, _c_i64, _c_ptr, _c_i64, _c_ptr, _c_i64, _c_ptr, _c_ptr, _c_ptr, _c_ptr, _c_int, _c_ptr,
         _c_ptr, _c_ptr, _c_i64, _c_int, _c_int, _c_int, _c_int, _c_float, _c_ptr],
    ),
}

_lib: ctypes.CDLL | None = None


def exported_symbols() -> list[str]:
    """Names the binding expects the library to export."""
    return sorted(_SIGNATURES)


def load() -> ctypes.CDLL:
    """Load the library once; raise RuntimeError if it has not been built."""
    global _lib
    if _lib is not None:
        return _lib
    if not LIB_PATH.exists():
        raise RuntimeError(
            f"{LIB_PATH} is missing: build it with `python -m nano_vllm_ascend_amd.build` "
            "(or __graft_entry__.build()); there is no CPU fallback"
        )
    lib = ctypes.CDLL(os.fspath(LIB_PATH))
    for name, (restype, argtypes) in _SIGNATURES.items():
        fn = getattr(lib, name)
        fn.restype = restype
        fn.argtypes = argtypes
    _bind_calls(lib)
    _lib = lib
    return lib


_calls = None  # csrc/calls.cpp: eager calls of the quantised caches and of copies, checked and made in one step; None: not usable


def _bind_calls(lib: ctypes.CDLL) -> None:
    """The library needs nothing of torch, the extension is tied to the torch that it was built with: without it the calls
    go through the checks in this file, with the same results."""
    global _calls
    try:
        calls = importlib.import_module("._calls", __package__)
        if calls.ABI_VERSION != lib.nvamd_version():
            raise ImportError(f"built for version {calls.ABI_VERSION} of the C ABI, the library has {lib.nvamd_version()}")
    except ImportError as e:
        _calls = None
        warnings.warn(f"eager calls of a quantised KV cache take some 5 us more each: {LIB_PATH.with_name('_calls.so')} cannot "
                      f"be used ({e}); `python -m nano_vllm_ascend_amd.build` builds it", RuntimeWarning, stacklevel=3)
        return
    for index, kind in enumerate((_FP4, _FP8)):
        functions = (kind.write, kind.read, kind.norm_rope, kind.decode, kind.decode_fused, kind.prefill,
                     kind.prefill_workspace)
        calls.bind(index, kind.pages, *(ctypes.cast(getattr(lib, f), ctypes.c_void_p).value for f in functions))
    calls.bind_copy(ctypes.cast(lib.nvamd_copy_blocks, ctypes.c_void_p).value)
    _calls = calls


def _check(status: int, name: str) -> None:
    if status == NVAMD_OK:
        return
    if status < 0:
        raise ValueError(f"{name}: {_ERRORS.get(status, 'error')} (status {status})")
    raise RuntimeError(f"{name}: HIP launch failed with hipError_t {status}")


_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)


def _stream() -> int:
    """hipStream_t of torch's current stream on the current device (the same handle as
    torch.cuda.current_stream().cuda_stream, also under a side stream or graph capture, looked up
    in ~0.3 us instead of ~2.8 us: it is asked for on every eager launch)."""
    if _raw_stream is not None:
        return _raw_stream(torch.cuda.current_device())
    return torch.cuda.current_stream().cuda_stream


def _ptr(t: torch.Tensor | None) -> int | None:
    return None if t is None else t.data_ptr()


def _require(cond: bool, msg) -> None:
    """Raise ValueError(msg) unless cond; msg may be a callable that builds the message, so a
    passing check formats nothing (these checks run on every eager launch)."""
    if not cond:
        raise ValueError(msg() if callable(msg) else msg)


def _row_stride(t: torch.Tensor) -> int:
    """Element stride between tokens of a [T, heads, D] (or [T, heads*D]) view whose rows are dense."""
    if t.dim() == 3:
        _require(t.stride(2) == 1 and t.stride(1) == t.shape[2], lambda: f"rows of {tuple(t.shape)} are not dense")
    else:
        _require(t.stride(-1) == 1, lambda: f"rows of {tuple(t.shape)} are not dense")
    return t.stride(0)


def _bf16_cuda(name: str, t: torch.Tensor) -> None:
    _require(t.dtype == torch.bfloat16, lambda: f"{name} must be bfloat16, got {t.dtype}")
    _require(t.is_cuda, lambda: f"{name} must be on the GPU")


def version() -> int:
    return int(load().nvamd_version())


# ------------------------------------------------------------------ index errors (device error word)
# Where the reference's indexing raises IndexError (index_copy_ into the KV cache, the RoPE cache
# lookup, the block-table gather), the kernels skip or clamp the access and set a bit in a
# per-device error word.  The runner copies the word to the host with each step's tokens (no extra
# synchronisation) and raises IndexError there.
ERR_SLOT, ERR_POSITION, ERR_CONTEXT, ERR_BLOCK, ERR_ORDER = 1, 2, 4, 8, 16  # NVAMD_ERR_*
_ERR_TEXT = {
    ERR_SLOT: "a slot_mapping entry outside the KV cache (index_copy_, nv/npu/paged_kv_cache.py:68-69)",
    ERR_POSITION: "a position outside the RoPE table (nv/layers/rotary_embedding.py:49-50)",
    ERR_CONTEXT: "a context length its block-table row or the launch's bound cannot hold",
    ERR_BLOCK: "a block-table entry outside the block pool",
    ERR_ORDER: "rows of a 16-slot tile of an 8-bit cache that do not follow one another in the order of their slots",
}


def describe_index_errors(bits: int) -> str:
    parts = [text for bit, text in _ERR_TEXT.items() if bits & bit]
    unknown = bits & ~sum(_ERR_TEXT)
    if unknown:
        parts.append(f"unknown bits {unknown:#x}")
    return "; ".join(parts)


def clear_index_errors() -> None:
    """Zero the current device's error word (a kernel on the current stream)."""
    _check(load().nvamd_errors_clear(_stream()), "nvamd_errors_clear")


class IndexErrorWord:
    """A host copy of the device's index-error word, fetched on the current stream beside a step's
    other results (pinned memory, so the copy is asynchronous) and checked once they have landed."""

    def __init__(self, host: torch.Tensor | None = None):
        self.host = host if host is not None else torch.zeros(1, dtype=torch.int32, pin_memory=True)

    def fetch(self) -> None:
        _check(load().nvamd_errors_fetch(self.host.data_ptr(), _stream()), "nvamd_errors_fetch")

    def raise_if_set(self) -> None:
        """Call after the copy has landed (the step's tokens were read)."""
        bits = int(self.host[0])
        if bits:
            self.host.zero_()
            clear_index_errors()
            raise IndexError(f"index out of range in the step's kernels: {describe_index_errors(bits)} "
                             f"(error word {bits:#x})")


def index_errors() -> int:
    """The current device's error word, read synchronously (tests and debugging)."""
    word = IndexErrorWord()
    word.fetch()
    torch.cuda.current_stream().synchronize()
    return int(word.host[0])


# ------------------------------------------------------------------ optional host-side range checks
# The kernels never read or write outside their buffers, but where the reference's torch indexing
# (index_select of the RoPE cache, index_copy_ into the KV cache, the block-table gather) would
# raise on an index out of range they clamp, skip or truncate instead.  With range checks on
# (set_range_checks(True), or NVAMD_CHECK_RANGES=1 in the environment) the eager wrappers read the
# indices back to the host and raise IndexError first.  That costs a device-to-host copy per call,
# so it is a debugging aid, off by default; calls made while a graph is being captured are not
# checked (a capture cannot synchronise).
_range_checks = os.environ.get("NVAMD_CHECK_RANGES", "") not in ("", "0")


def set_range_checks(enabled: bool) -> bool:
    """Turn the host-side range checks on or off; returns the previous setting."""
    global _range_checks
    prev, _range_checks = _range_checks, bool(enabled)
    return prev


def _checking() -> bool:
    return _range_checks and not (torch.cuda.is_available() and torch.cuda.is_current_stream_capturing())


def check_positions(positions: torch.Tensor, max_positions: int) -> None:
    """RoPE rows are index_select-ed by position (nv/layers/rotary_embedding.py:44-55)."""
    pos = positions.detach().reshape(-1).cpu()
    if pos.numel() and (int(pos.min()) < 0 or int(pos.max()) >= max_positions):
        raise IndexError(f"position out of range [0, {max_positions}) of the RoPE table: "
                         f"min {int(pos.min())}, max {int(pos.max())}")


def check_slots(slot_mapping: torch.Tensor, num_slots: int) -> None:
    """K/V rows are index_copy_-ed at their slots (nv/npu/paged_kv_cache.py:68-69); -1 marks a padding
    row that is not stored (an extension the reference never emits)."""
    sl = slot_mapping.detach().reshape(-1).cpu()
    if sl.numel() and (int(sl.min()) < -1 or int(sl.max()) >= num_slots):
        raise IndexError(f"slot out of range [0, {num_slots}) (or -1 for padding): "
                         f"min {int(sl.min())}, max {int(sl.max())}")


def check_paged_context(block_tables: torch.Tensor, context_lens: torch.Tensor, num_blocks: int, block_size: int,
                        max_context_len: int | None = None) -> None:
    """Every context fits its bound and its block-table row, and the entries it reads name pool blocks
    (the reference gathers K/V through the table, nv/layers/npu_paged_attention.py:89-99)."""
    ctx = context_lens.detach().reshape(-1).cpu().long()
    bt = block_tables.detach().cpu().long()
    width = bt.shape[1] * block_size
    for i, c in enumerate(ctx.tolist()):
        if c < 0 or c > width or (max_context_len is not None and c > max_context_len):
            raise IndexError(f"context length {c} of row {i} is outside [0, min({width}, "
                             f"{max_context_len if max_context_len is not None else width})]")
        used = bt[i, : -(-c // block_size)]
        if used.numel() and (int(used.min()) < 0 or int(used.max()) >= num_blocks):
            raise IndexError(f"block-table row {i} names a block outside [0, {num_blocks}): {used.tolist()}")


def paged_decode_workspace_size(max_batch: int, num_heads: int, num_kv_heads: int, max_context_len: int) -> int:
    return int(load().nvamd_paged_decode_workspace_size(max_batch, num_heads, num_kv_heads, max_context_len))


def alloc_paged_decode_workspace(max_batch: int, num_heads: int, num_kv_heads: int, max_context_len: int,
                                 device) -> torch.Tensor:
    """Zero-filled workspace (the kernel keeps its counters at zero between calls)."""
    nbytes = paged_decode_workspace_size(max_batch, num_heads, num_kv_heads, max_context_len)
    return torch.zeros(nbytes, dtype=torch.uint8, device=device)


def paged_decode(out: torch.Tensor, q: torch.Tensor, key_cache: torch.Tensor, value_cache: torch.Tensor,
                 block_tables: torch.Tensor, context_lens: torch.Tensor, scale: float, max_context_len: int,
                 workspace: torch.Tensor) -> torch.Tensor:
    """out[i,h] = softmax(q[i,h] K^T * scale) V over the paged context of sequence i.

    q/out: [B, Hq, 128] bf16 (dense rows, any token stride); caches
    [NB, block_size, Hkv, 128] bf16; block_tables int32 [B, W]; context_lens
    int32 [B] on the device; max_context_len bounds every context_lens entry.
    """
    lib = load()
    args = _decode_args(out, q, key_cache, value_cache, block_tables, context_lens, scale, max_context_len)
    status = lib.nvamd_paged_decode(*args, workspace.data_ptr(), workspace.numel() * workspace.element_size(),
                                    _stream())
    _check(status, "nvamd_paged_decode")
    return out


def paged_decode_noalloc(out: torch.Tensor, q: torch.Tensor, key_cache: torch.Tensor, value_cache: torch.Tensor,
                         block_tables: torch.Tensor, context_lens: torch.Tensor, scale: float,
                         max_context_len: int) -> torch.Tensor:
    """``paged_decode`` without a workspace: the library's static per-GPU scratch serves as one.

    Raises ValueError when the call needs more than DECODE_SCRATCH_BYTES
    (paged_decode_workspace_size of its sizes), or when the first call on a device is made under
    graph capture (the first call clears the scratch's counters, which capture would only record).
    Calls that overlap on one GPU share the scratch and race.
    """
    lib = load()
    args = _decode_args(out, q, key_cache, value_cache, block_tables, context_lens, scale, max_context_len)
    _check(lib.nvamd_paged_decode_noalloc(*args, _stream()), "nvamd_paged_decode_noalloc")
    return out


def _decode_args(out, q, key_cache, value_cache, block_tables, context_lens, scale, max_context_len) -> tuple:
    """Checked arguments of the decode entry points, up to the workspace.  The checks are written out (a small
    batch's eager decode is bound by the host: 4.7 us of a 15 us call went to them as helper calls)."""
    for name, t in (("q", q), ("out", out), ("key_cache", key_cache), ("value_cache", value_cache)):
        if t.dtype is not torch.bfloat16 or not t.is_cuda:
            _bf16_cuda(name, t)  # raises
    q_shape, kv_shape = q.shape, key_cache.shape
    if len(q_shape) != 3 or out.shape != q_shape:
        raise ValueError(f"q/out shape mismatch: {tuple(q_shape)} vs {tuple(out.shape)}")
    if len(kv_shape) != 4 or value_cache.shape != kv_shape:
        raise ValueError("key/value cache shape mismatch")
    if not (key_cache.is_contiguous() and value_cache.is_contiguous()):
        raise ValueError("caches must be contiguous")
    nb, bs, hkv, d = kv_shape
    b, hq, dq = q_shape
    if dq != d:
        raise ValueError(f"head_dim mismatch {dq} vs {d}")
    bt_shape, bt_stride = block_tables.shape, block_tables.stride()
    if block_tables.dtype is not torch.int32 or len(bt_shape) != 2 or bt_shape[0] != b:
        raise ValueError("block_tables must be int32 [B, W]")
    if bt_stride[1] != 1:
        raise ValueError("block_tables rows must be dense")
    if context_lens.dtype is not torch.int32 or context_lens.numel() != b or not context_lens.is_cuda:
        raise ValueError("context_lens must be int32 [B] on the device")
    if not context_lens.is_contiguous():
        raise ValueError("context_lens must be contiguous")
    q_stride, out_stride = q.stride(), out.stride()
    for t, st in ((q, q_stride), (out, out_stride)):
        if st[2] != 1 or st[1] != d:
            raise ValueError(f"rows of {tuple(t.shape)} are not dense")
    if _range_checks and _checking():
        check_paged_context(block_tables, context_lens, nb, bs, int(max_context_len))
    return (out.data_ptr(), out_stride[0], q.data_ptr(), q_stride[0], key_cache.data_ptr(),
            value_cache.data_ptr(), nb, bs, block_tables.data_ptr(), bt_stride[0], bt_shape[1],
            context_lens.data_ptr(), b, hq, hkv, d, float(scale), int(max_context_len))


def paged_decode_fused(out: torch.Tensor, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor,
                       q_weight: torch.Tensor, k_weight: torch.Tensor, positions: torch.Tensor,
                       cos_sin: torch.Tensor, eps: float, key_cache: torch.Tensor, value_cache: torch.Tensor,
                       slot_mapping: torch.Tensor, block_tables: torch.Tensor, context_lens: torch.Tensor,
                       scale: float, max_context_len: int, workspace: torch.Tensor) -> torch.Tensor:
    """One decode step of attention: qk_norm_rope (with the KV store) then paged_decode, in one launch.

    q: raw [B, Hq, 128] and k, v: raw [B, Hkv, 128] rows of the new tokens (views into the
    projection output are fine; they are not modified).  Writes out and the caches only.
    slot_mapping[i] must be the cache slot of row positions[i] of sequence i (decode metadata).
    """
    lib = load()
    args = _decode_args(out, q, key_cache, value_cache, block_tables, context_lens, scale, max_context_len)
    for name, t in (("k", k), ("v", v)):
        if t.dtype is not torch.bfloat16 or not t.is_cuda:
            _bf16_cuda(name, t)  # raises
    b, hkv, d = q.shape[0], key_cache.shape[2], key_cache.shape[3]
    if k.shape != v.shape or k.shape != (b, hkv, d):
        raise ValueError(f"k/v must be [B, Hkv, D] = {(b, hkv, d)}, got {tuple(k.shape)} and {tuple(v.shape)}")
    if q_weight.dtype is not torch.bfloat16 or k_weight.dtype is not torch.bfloat16:
        raise ValueError("norm weights must be bf16")
    if q_weight.numel() != d or k_weight.numel() != d:
        raise ValueError("norm weights must have head_dim elements")
    if not (q_weight.is_contiguous() and k_weight.is_contiguous()):
        raise ValueError("norm weights must be contiguous")
    if positions.dtype is not torch.int64 or positions.numel() != b or not positions.is_cuda:
        raise ValueError("positions must be int64 [B] on the device")
    table = cos_sin.shape
    if (cos_sin.dtype is not torch.float32 or len(table) != 2 or table[1] != d or not cos_sin.is_cuda
            or not cos_sin.is_contiguous()):
        raise ValueError("cos_sin must be contiguous fp32 [max_positions, head_dim]")
    if slot_mapping.dtype is not torch.int64 or slot_mapping.numel() != b or not slot_mapping.is_cuda:
        raise ValueError("slot_mapping must be int64 [B] on the device")
    if _range_checks and _checking():
        check_positions(positions, table[0])
        check_slots(slot_mapping, key_cache.shape[0] * key_cache.shape[1])
    status = lib.nvamd_paged_decode_fused(
        *args[:4], k.data_ptr(), _row_stride(k), v.data_ptr(), _row_stride(v), q_weight.data_ptr(),
        k_weight.data_ptr(), positions.contiguous().data_ptr(), cos_sin.data_ptr(), table[0], float(eps), *args[4:8],
        slot_mapping.contiguous().data_ptr(), *args[8:], workspace.data_ptr(),
        workspace.numel() * workspace.element_size(), _stream())
    _check(status, "nvamd_paged_decode_fused")
    return out


def kv_cache_write(key_states: torch.Tensor, value_states: torch.Tensor, key_cache: torch.Tensor,
                   value_cache: torch.Tensor, slot_mapping: torch.Tensor) -> None:
    """cache_flat[slot_mapping[t]] = kv[t] for the K and the V cache of one layer."""
    lib = load()
    _bf16_cuda("key_states", key_states)
    _bf16_cuda("value_states", value_states)
    _require(key_states.shape == value_states.shape and key_states.dim() == 3, "k/v shape mismatch")
    t, hkv, d = key_states.shape
    _require(key_cache.is_contiguous() and value_cache.is_contiguous(), "caches must be contiguous")
    _require(key_cache.shape[-2:] == (hkv, d), lambda: f"kv shape mismatch: got {tuple(key_states.shape)}")
    _require(slot_mapping.dtype == torch.int64 and slot_mapping.numel() == t and slot_mapping.is_cuda,
             f"slot_mapping numel {slot_mapping.numel()} != total_tokens {t}")
    num_slots = key_cache.numel() // (hkv * d)
    if _checking():
        check_slots(slot_mapping, num_slots)
    status = lib.nvamd_kv_cache_write(
        key_states.data_ptr(), _row_stride(key_states), value_states.data_ptr(), _row_stride(value_states),
        key_cache.data_ptr(), value_cache.data_ptr(), slot_mapping.contiguous().data_ptr(), t, hkv, d, num_slots,
        _stream(),
    )
    _check(status, "nvamd_kv_cache_write")


def qk_norm_rope(q: torch.Tensor, k: torch.Tensor, q_weight: torch.Tensor, k_weight: torch.Tensor,
                 positions: torch.Tensor, cos_sin: torch.Tensor, eps: float,
                 v: torch.Tensor | None = None, key_cache: torch.Tensor | None = None,
                 value_cache: torch.Tensor | None = None, slot_mapping: torch.Tensor | None = None) -> None:
    """In place: q, k <- RoPE(RMSNorm_head(x) * w); optionally store post-RoPE k and v in the caches."""
    lib = load()
    _bf16_cuda("q", q)
    _bf16_cuda("k", k)
    _require(q.dim() == 3 and k.dim() == 3 and q.shape[0] == k.shape[0], "q/k must be [T, heads, D]")
    t, hq, d = q.shape
    hkv = k.shape[1]
    _require(k.shape[2] == d, "q/k head_dim mismatch")
    _require(q_weight.dtype == torch.bfloat16 and k_weight.dtype == torch.bfloat16, "norm weights must be bf16")
    _require(q_weight.numel() == d and k_weight.numel() == d, "norm weights must have head_dim elements")
    _require(positions.dtype == torch.int64 and positions.numel() == t and positions.is_cuda,
             "positions must be int64 [T] on the device")
    _require(cos_sin.dtype == torch.float32 and cos_sin.dim() == 2 and cos_sin.shape[1] == d and cos_sin.is_cuda,
             "cos_sin must be fp32 [max_positions, head_dim]")
    store = key_cache is not None
    num_slots = 0
    if store:
        _require(v is not None and value_cache is not None and slot_mapping is not None, "store needs v, caches, slots")
        _bf16_cuda("v", v)
        _require(v.shape == k.shape, "k/v shape mismatch")
        _require(key_cache.is_contiguous() and value_cache.is_contiguous(), "caches must be contiguous")
        _require(slot_mapping.dtype == torch.int64 and slot_mapping.numel() == t, "slot_mapping must be int64 [T]")
        num_slots = key_cache.numel() // (hkv * d)
    if _checking():
        check_positions(positions, cos_sin.shape[0])
        if store:
            check_slots(slot_mapping, num_slots)
    status = lib.nvamd_qk_norm_rope(
        q.data_ptr(), _row_stride(q), k.data_ptr(), _row_stride(k), _ptr(v), _row_stride(v) if store else 0,
        q_weight.data_ptr(), k_weight.data_ptr(), positions.data_ptr(), cos_sin.data_ptr(), cos_sin.shape[0],
        _ptr(key_cache), _ptr(value_cache), _ptr(slot_mapping.contiguous()) if store else None, num_slots,
        t, hq, hkv, d, float(eps), _stream(),
    )
    _check(status, "nvamd_qk_norm_rope")


def pack_batch(desc: torch.Tensor, batch: int, updates: torch.Tensor | None, num_updates: int,
               token_ids: torch.Tensor | None, mirror: torch.Tensor, block_size: int,
               block_tables: torch.Tensor | None = None, context_lens: torch.Tensor | None = None,
               slot_mapping: torch.Tensor | None = None, positions: torch.Tensor | None = None,
               cu_seqlens: torch.Tensor | None = None, last_token_indices: torch.Tensor | None = None,
               input_ids: torch.Tensor | None = None) -> None:
    """Expand per-sequence descriptors into the packed-batch metadata on the GPU (see nvamd.h)."""
    lib = load()
    _require(desc.dtype == torch.int32 and desc.is_cuda and desc.numel() >= 5 * batch, "desc must be int32 [5, B]")
    _require(mirror.dtype == torch.int32 and mirror.dim() == 2 and mirror.is_contiguous(), "mirror must be int32 2-D")
    if block_tables is not None:
        _require(block_tables.dtype == torch.int32 and block_tables.stride(1) == 1 and block_tables.shape[0] >= batch,
                 "block_tables must be int32 [B, W] with dense rows")
    for name, t, dt in (("context_lens", context_lens, torch.int32), ("slot_mapping", slot_mapping, torch.int64),
                        ("positions", positions, torch.int64), ("cu_seqlens", cu_seqlens, torch.int32),
                        ("last_token_indices", last_token_indices, torch.int64),
                        ("input_ids", input_ids, torch.int64)):
        if t is not None:
            _require(t.dtype == dt and t.is_cuda and t.is_contiguous(),
                     lambda: f"{name} must be a contiguous {dt} GPU tensor")
    status = lib.nvamd_pack_batch(
        desc.data_ptr(), batch, _ptr(updates), num_updates, _ptr(token_ids), mirror.data_ptr(), mirror.shape[1],
        mirror.shape[0], block_size, _ptr(block_tables), block_tables.stride(0) if block_tables is not None else 0,
        block_tables.shape[1] if block_tables is not None else 0, _ptr(context_lens), _ptr(slot_mapping),
        _ptr(positions), _ptr(cu_seqlens), _ptr(last_token_indices), _ptr(input_ids), _stream(),
    )
    _check(status, "nvamd_pack_batch")


def varlen_prefill(out: torch.Tensor, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cu_seqlens_q: torch.Tensor,
                   max_q_len: int, scale: float) -> torch.Tensor:
    """Dense causal varlen attention: q/out [T, Hq, 128], k/v [T, Hkv, 128], cu_seqlens_q int32 [B+1] (device)."""
    lib = load()
    for name, t in (("q", q), ("k", k), ("v", v), ("out", out)):
        _bf16_cuda(name, t)
        _require(t.dim() == 3, lambda: f"{name} must be [T, heads, D]")
    _require(out.shape == q.shape, "q/out shape mismatch")
    _require(k.shape == v.shape and k.shape[0] == q.shape[0], lambda: f"k/v token mismatch: q={tuple(q.shape)} "
             f"k={tuple(k.shape)} v={tuple(v.shape)}")
    _require(cu_seqlens_q.dtype == torch.int32 and cu_seqlens_q.is_cuda and cu_seqlens_q.is_contiguous(),
             "cu_seqlens_q must be int32 on the device")
    n_seqs = cu_seqlens_q.numel() - 1
    status = lib.nvamd_varlen_prefill(
        out.data_ptr(), _row_stride(out), q.data_ptr(), _row_stride(q), k.data_ptr(), _row_stride(k),
        v.data_ptr(), _row_stride(v), cu_seqlens_q.data_ptr(), n_seqs, int(max_q_len), q.shape[1], k.shape[1],
        q.shape[2], float(scale), _stream(),
    )
    _check(status, "nvamd_varlen_prefill")
    return out


def paged_prefill(out: torch.Tensor, q: torch.Tensor, key_cache: torch.Tensor, value_cache: torch.Tensor,
                  block_tables: torch.Tensor, cu_seqlens_q: torch.Tensor, kv_lens: torch.Tensor, max_q_len: int,
                  scale: float) -> torch.Tensor:
    """Prefix-hit prefill: queries are the last q_len of kv_len positions, keys read through the cache pages."""
    lib = load()
    for name, t in (("q", q), ("out", out), ("key_cache", key_cache), ("value_cache", value_cache)):
        _bf16_cuda(name, t)
    _require(out.shape == q.shape and q.dim() == 3, "q/out shape mismatch")
    _require(key_cache.dim() == 4 and key_cache.shape == value_cache.shape, "key/value cache shape mismatch")
    _require(key_cache.is_contiguous() and value_cache.is_contiguous(), "caches must be contiguous")
    _require(block_tables.dtype == torch.int32 and block_tables.stride(1) == 1, "block_tables must be int32 [B, W]")
    _require(cu_seqlens_q.dtype == torch.int32 and kv_lens.dtype == torch.int32 and kv_lens.is_cuda,
             "cu_seqlens_q / kv_lens must be int32 on the device")
    nb, bs, hkv, d = key_cache.shape
    n_seqs = cu_seqlens_q.numel() - 1
    _require(kv_lens.numel() >= n_seqs and block_tables.shape[0] >= n_seqs, "per-sequence metadata too short")
    if _checking():
        check_paged_context(block_tables[:n_seqs], kv_lens[:n_seqs], nb, bs)
    status = lib.nvamd_paged_prefill(
        out.data_ptr(), _row_stride(out), q.data_ptr(), _row_stride(q), key_cache.data_ptr(), value_cache.data_ptr(),
        nb, bs, block_tables.data_ptr(), block_tables.stride(0), block_tables.shape[1], cu_seqlens_q.data_ptr(),
        kv_lens.data_ptr(), n_seqs, int(max_q_len), q.shape[1], hkv, d, float(scale), _stream(),
    )
    _check(status, "nvamd_paged_prefill")
    return out


# ------------------------------------------------------------------ KV caches held in 4 and in 8 bits
# The same path over pages of FP4 codes with a power-of-two scale per 32 dims, or of e4m3 codes with one per tile of 16
# tokens (formats and layouts: nvamd.h).
FP4_ROW_BYTES, FP4_ROW_SCALES = 64, 4  # of a head vector
FP8_ROW_BYTES, FP8_TILE = 128, 16      # of a head vector; tokens that share a scale


class Fp4Pages(NamedTuple):
    """The keys or the values of one layer in 4 bits: ``codes`` uint8 [blocks, kv heads, block_size, 64] and ``scales``
    uint8 [blocks, kv heads, block_size, 4], contiguous.  Pages are opaque (``kv_cache_read_fp4`` gives their values)."""

    codes: torch.Tensor
    scales: torch.Tensor

    @property
    def shape(self) -> tuple[int, int, int, int]:
        """[blocks, block_size, kv heads, head_dim], as a bf16 cache of these pages has it."""
        nb, hkv, bs, width = self.codes.shape
        return nb, bs, hkv, 2 * width


class Fp8Pages(NamedTuple):
    """The keys or the values of one layer in 8 bits: ``codes`` uint8 [blocks, kv heads, block_size, 128] and ``scales``
    uint8 [blocks, kv heads, block_size / 16], contiguous.  Pages are opaque (``kv_cache_read_fp8`` gives their values)."""

    codes: torch.Tensor
    scales: torch.Tensor

    @property
    def shape(self) -> tuple[int, int, int, int]:
        """[blocks, block_size, kv heads, head_dim], as a bf16 cache of these pages has it."""
        nb, hkv, bs, width = self.codes.shape
        return nb, bs, hkv, width


class _Kind:
    """A quantised cache: its pages, the bytes of a head vector's codes, the names of its entry points (put together here: in
    a call they would take 0.1 us of its 4)."""

    def __init__(self, name: str, pages: type, row_bytes: int):
        self.name, self.pages, self.row_bytes = name, pages, row_bytes
        self.write, self.read = f"nvamd_kv_cache_write_{name}", f"nvamd_kv_cache_read_{name}"
        self.norm_rope = f"nvamd_qk_norm_rope_{name}"
        self.decode, self.decode_fused = f"nvamd_paged_decode_{name}", f"nvamd_paged_decode_fused_{name}"
        self.prefill, self.prefill_workspace = (f"nvamd_paged_prefill_{name}{s}" for s in ("", "_workspace_size"))

    def scales(self, nb: int, hkv: int, bs: int) -> tuple[int, ...]:
        return (nb, hkv, bs, FP4_ROW_SCALES) if self.pages is Fp4Pages else (nb, hkv, bs // FP8_TILE)


_FP4 = _Kind("fp4", Fp4Pages, FP4_ROW_BYTES)
_FP8 = _Kind("fp8", Fp8Pages, FP8_ROW_BYTES)
_HEAD_DIM = 128


def _checked_pages(kind: _Kind, key_pages, value_pages):
    """Checks the pages of a layer; returns blocks, block_size, kv heads, their addresses and their device."""
    if type(key_pages) is not kind.pages or type(value_pages) is not kind.pages:
        raise ValueError(f"key and value pages must be {kind.pages.__name__}")
    kc, ks = key_pages
    vc, vs = value_pages
    shape = kc.shape
    if len(shape) != 4 or shape[3] != kind.row_bytes or vc.shape != shape:
        raise ValueError(f"codes must be [blocks, kv heads, block_size, {kind.row_bytes}] for keys and values, got "
                         f"{tuple(shape)} and {tuple(vc.shape)}")
    nb, hkv, bs, _ = shape
    scales = kind.scales(nb, hkv, bs)
    if ks.shape != scales or vs.shape != scales:
        raise ValueError(f"scales must be {scales}, got {tuple(ks.shape)} and {tuple(vs.shape)}")
    u8 = torch.uint8
    if not (kc.dtype is u8 and ks.dtype is u8 and vc.dtype is u8 and vs.dtype is u8 and kc.is_contiguous()
            and ks.is_contiguous() and vc.is_contiguous() and vs.is_contiguous()):
        raise ValueError("pages must be contiguous uint8 tensors")
    device = kc.get_device()
    if not device == ks.get_device() == vc.get_device() == vs.get_device():
        raise ValueError("the pages of a layer must be on one device")
    return nb, bs, hkv, (kc.data_ptr(), ks.data_ptr(), vc.data_ptr(), vs.data_ptr()), device


def _stream_of(device: int, *tensors: torch.Tensor) -> int:
    """The current stream, which every launch goes to: the tensors and the pages have to be on its device."""
    for t in tensors:
        if t.get_device() != device:
            raise ValueError(f"every tensor must be on the GPU of the pages (device {device}), one is on {t.device}")
    if device < 0:
        raise ValueError("every tensor must be on the GPU")
    if device != torch.cuda.current_device():
        raise ValueError(f"the tensors are on device {device}, the current device is {torch.cuda.current_device()}")
    return _raw_stream(device) if _raw_stream is not None else _stream()


def _int32(name: str, value) -> int:
    """An int argument of the C ABI (ctypes would keep the lower half of a larger number)."""
    value = int(value)
    if not -(1 << 31) <= value < 1 << 31:
        raise ValueError(f"{name} {value} is past 32 bits")
    return value


def _heads(name: str, t: torch.Tensor, rows: int, heads: int, d: int) -> int:
    """Checks a [T, heads, D] bf16 view of dense rows; returns its row stride."""
    if t.shape != (rows, heads, d):
        raise ValueError(f"{name} must be {(rows, heads, d)}, got {tuple(t.shape)}")
    if t.dtype is not torch.bfloat16:
        raise ValueError(f"{name} must be bfloat16, got {t.dtype}")
    row, head, unit = t.stride()
    if (unit != 1 or (head != d and heads > 1)) and rows:
        raise ValueError(f"rows of {name} {tuple(t.shape)} are not dense")
    return row if rows > 1 else max(row, heads * d)  # a single row's stride says nothing


def check_tile_order(slot_mapping: torch.Tensor) -> None:
    """Rows that go to one tile of the 8-bit cache follow one another, in the order of their slots, with no padding row
    between them."""
    sl = slot_mapping.detach().reshape(-1).cpu()
    begins = sl >= 0
    begins[1:] &= (sl[1:] != sl[:-1] + 1) | (sl[1:] % FP8_TILE == 0)
    tiles = sl[begins] // FP8_TILE
    if tiles.numel() != tiles.unique().numel():
        raise IndexError("rows of a tile of 16 slots do not follow one another in the call, in the order of their slots")


def _page_slots(slot_mapping: torch.Tensor, rows: int, num_slots: int, writes: _Kind | None = None) -> int:
    if (slot_mapping.dtype is not torch.int64 or slot_mapping.shape != (rows,) or not slot_mapping.is_contiguous()):
        raise ValueError(f"slot_mapping must be contiguous int64 [{rows}], got {slot_mapping.dtype} "
                         f"{tuple(slot_mapping.shape)}")
    if _range_checks and _checking():
        check_slots(slot_mapping, num_slots)
        if writes is _FP8:
            check_tile_order(slot_mapping)
    return slot_mapping.data_ptr()


def _made(answer, name: str) -> bool:
    """Whether csrc/calls.cpp has made the call, as it does if every argument is plainly right; raises for what the library
    answered.  If not, and with range checks on, the checks of the functions below name what is wrong, or they call."""
    if answer is None:
        return False
    if type(answer) is int:
        _check(answer, name)
    return True


def _write(kind: _Kind, key_states, value_states, key_pages, value_pages, slot_mapping) -> None:
    lib, name = _lib or load(), kind.write
    if _calls and not _range_checks and type(key_pages) is kind.pages:
        made = _calls.write(key_states, value_states, key_pages, value_pages, slot_mapping)
        if made is True or _made(made, name):
            return
    nb, bs, hkv, pages, device = _checked_pages(kind, key_pages, value_pages)
    t, d = key_states.shape[0], _HEAD_DIM
    k_stride, v_stride = _heads("key_states", key_states, t, hkv, d), _heads("value_states", value_states, t, hkv, d)
    slots = _page_slots(slot_mapping, t, nb * bs, kind)
    status = getattr(lib, name)(
        key_states.data_ptr(), k_stride, value_states.data_ptr(), v_stride, *pages, nb, bs, slots, t, hkv, d,
        _stream_of(device, key_states, value_states, slot_mapping))
    if status:
        _check(status, name)


def _read(kind: _Kind, key_pages, value_pages, slot_mapping, k_out, v_out) -> tuple[torch.Tensor, torch.Tensor]:
    lib, name = _lib or load(), kind.read
    if _calls and not _range_checks and k_out is None and v_out is None and type(key_pages) is kind.pages:
        rows = _calls.read(key_pages, value_pages, slot_mapping)
        if type(rows) is tuple or _made(rows, name):
            return rows
    nb, bs, hkv, pages, device = _checked_pages(kind, key_pages, value_pages)
    t, d = slot_mapping.shape[0], _HEAD_DIM
    slots = _page_slots(slot_mapping, t, nb * bs)
    k_stride = v_stride = hkv * d
    if k_out is None:
        k_out = torch.empty((t, hkv, d), dtype=torch.bfloat16, device=key_pages.codes.device)
    else:
        k_stride = _heads("k_out", k_out, t, hkv, d)
    if v_out is None:
        v_out = torch.empty((t, hkv, d), dtype=torch.bfloat16, device=key_pages.codes.device)
    else:
        v_stride = _heads("v_out", v_out, t, hkv, d)
    status = getattr(lib, name)(k_out.data_ptr(), k_stride, v_out.data_ptr(), v_stride, *pages, nb, bs, slots,
                                t, hkv, d, _stream_of(device, k_out, v_out, slot_mapping))
    if status:
        _check(status, name)
    return k_out, v_out


def _rope_args(q_weight, k_weight, positions, cos_sin, t: int, d: int) -> None:
    for name, w in (("q_weight", q_weight), ("k_weight", k_weight)):
        if w.dtype is not torch.bfloat16 or w.shape != (d,) or not w.is_contiguous():
            raise ValueError(f"{name} must be contiguous bf16 [{d}]")
    if positions.dtype is not torch.int64 or positions.shape != (t,) or not positions.is_contiguous():
        raise ValueError(f"positions must be contiguous int64 [{t}]")
    table = cos_sin.shape
    if cos_sin.dtype is not torch.float32 or len(table) != 2 or table[1] != d or not cos_sin.is_contiguous():
        raise ValueError("cos_sin must be contiguous fp32 [max_positions, head_dim]")


def _norm_rope(kind: _Kind, q, k, v, q_weight, k_weight, positions, cos_sin, eps, key_pages, value_pages, slot_mapping,
               q_out, k_out) -> torch.Tensor:
    lib, name = _lib or load(), kind.norm_rope
    if _calls and not _range_checks and type(key_pages) is kind.pages:
        rotated = _calls.rope(q, k, v, q_weight, k_weight, positions, cos_sin, eps, key_pages, value_pages, slot_mapping,
                              q_out, k_out)
        if type(rotated) is torch.Tensor or _made(rotated, name):
            return rotated
    nb, bs, hkv, pages, device = _checked_pages(kind, key_pages, value_pages)
    d = _HEAD_DIM
    if q.dim() != 3:
        raise ValueError(f"q must be [T, heads, D], got {tuple(q.shape)}")
    t, hq, _ = q.shape
    q_stride, k_stride, v_stride = _heads("q", q, t, hq, d), _heads("k", k, t, hkv, d), _heads("v", v, t, hkv, d)
    if q_out is None:
        q_out, qo_stride = torch.empty((t, hq, d), dtype=torch.bfloat16, device=q.device), hq * d
    else:
        qo_stride = _heads("q_out", q_out, t, hq, d)
    q_ptr, k_ptr, qo_ptr, ko_ptr, ko_stride = q.data_ptr(), k.data_ptr(), q_out.data_ptr(), None, 0
    if k_out is not None:
        ko_stride, ko_ptr = _heads("k_out", k_out, t, hkv, d), k_out.data_ptr()
    if (qo_ptr == q_ptr and qo_stride != q_stride) or (ko_ptr == k_ptr and ko_stride != k_stride):
        raise ValueError("an output in place of its input must have the input's row stride")
    _rope_args(q_weight, k_weight, positions, cos_sin, t, d)
    slots = _page_slots(slot_mapping, t, nb * bs, kind)
    if _range_checks and _checking():
        check_positions(positions, cos_sin.shape[0])
    status = getattr(lib, name)(
        qo_ptr, qo_stride, ko_ptr, ko_stride, q_ptr, q_stride, k_ptr, k_stride, v.data_ptr(), v_stride,
        q_weight.data_ptr(), k_weight.data_ptr(), positions.data_ptr(), cos_sin.data_ptr(), cos_sin.shape[0], *pages, nb,
        bs, slots, t, hq, hkv, d, float(eps),
        _stream_of(device, q, k, v, q_out, q if k_out is None else k_out, q_weight, k_weight, positions, cos_sin,
                   slot_mapping))
    if status:
        _check(status, name)
    return q_out


def _attention_args(kind: _Kind, out, q, key_pages, value_pages, block_tables, seqs: int):
    """Checked arguments that decode and prefill share, up to the block tables; [heads, kv heads, head_dim]; the device."""
    nb, bs, hkv, pages, device = _checked_pages(kind, key_pages, value_pages)
    d = _HEAD_DIM
    shape = q.shape
    if len(shape) != 3 or out.shape != shape:
        raise ValueError(f"q/out shape mismatch: {tuple(shape)} vs {tuple(out.shape)}")
    t, hq, dq = shape
    if dq != d:
        raise ValueError(f"head_dim mismatch {dq} vs {d}")
    if q.dtype is not torch.bfloat16 or out.dtype is not torch.bfloat16:
        raise ValueError(f"q and out must be bfloat16, got {q.dtype} and {out.dtype}")
    q_stride, out_stride = q.stride(), out.stride()
    for name, st in (("q", q_stride), ("out", out_stride)):
        if t and (st[2] != 1 or (hq > 1 and st[1] != d)):
            raise ValueError(f"rows of {name} {tuple(shape)} are not dense")
    tables, bt_stride = block_tables.shape, block_tables.stride()
    if block_tables.dtype is not torch.int32 or len(tables) != 2 or tables[0] < seqs:
        raise ValueError(f"block_tables must be int32 [{seqs}, W]")
    width = tables[1]
    if bt_stride[1] != 1 and width > 1:
        raise ValueError("block_tables rows must be dense")
    if tables[0] > 1 and bt_stride[0] < width:
        raise ValueError(f"rows of block_tables overlap: {tuple(tables)} with a row stride of {bt_stride[0]}")
    bt_row = _int32("the row stride of block_tables", bt_stride[0] if tables[0] > 1 else width)
    least = hq * d  # a single row's stride says nothing
    return (out.data_ptr(), out_stride[0] if t > 1 else max(out_stride[0], least), q.data_ptr(),
            q_stride[0] if t > 1 else max(q_stride[0], least), *pages, nb, bs, block_tables.data_ptr(),
            bt_row, width), (hq, hkv, d), device


def _step_args(block_tables, context_lens, workspace, b: int) -> None:
    if block_tables.shape[0] != b:
        raise ValueError(f"block_tables must be int32 [{b}, W]")
    if context_lens.dtype is not torch.int32 or context_lens.shape != (b,) or not context_lens.is_contiguous():
        raise ValueError(f"context_lens must be contiguous int32 [{b}]")
    if not workspace.is_contiguous():
        raise ValueError("workspace must be contiguous")


def _decode(kind: _Kind, out, q, key_pages, value_pages, block_tables, context_lens, scale, max_context_len,
            workspace) -> torch.Tensor:
    lib, name = _lib or load(), kind.decode
    if _calls and not _range_checks and type(key_pages) is kind.pages:
        made = _calls.decode(out, q, key_pages, value_pages, block_tables, context_lens, scale, max_context_len, workspace)
        if type(made) is torch.Tensor or _made(made, name):
            return made
    if out is None:
        out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    b = q.shape[0]
    args, heads, device = _attention_args(kind, out, q, key_pages, value_pages, block_tables, b)
    _step_args(block_tables, context_lens, workspace, b)
    max_context_len = _int32("max_context_len", max_context_len)
    if _range_checks and _checking():
        check_paged_context(block_tables, context_lens, args[8], args[9], max_context_len)
    status = getattr(lib, name)(*args, context_lens.data_ptr(), b, *heads, float(scale), max_context_len,
                                workspace.data_ptr(), workspace.nbytes,
                                _stream_of(device, q, out, block_tables, context_lens, workspace))
    if status:
        _check(status, name)
    return out


def _decode_fused(kind: _Kind, out, q, k, v, q_weight, k_weight, positions, cos_sin, eps, key_pages, value_pages,
                  slot_mapping, block_tables, context_lens, scale, max_context_len, workspace) -> torch.Tensor:
    lib, name = _lib or load(), kind.decode_fused
    if _calls and not _range_checks and type(key_pages) is kind.pages:
        made = _calls.decode_fused(out, q, k, v, q_weight, k_weight, positions, cos_sin, eps, key_pages, value_pages,
                                   slot_mapping, block_tables, context_lens, scale, max_context_len, workspace)
        if type(made) is torch.Tensor or _made(made, name):
            return made
    if out is None:
        out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    b = q.shape[0]
    args, heads, device = _attention_args(kind, out, q, key_pages, value_pages, block_tables, b)
    _step_args(block_tables, context_lens, workspace, b)
    max_context_len = _int32("max_context_len", max_context_len)
    nb, bs, (hq, hkv, d) = args[8], args[9], heads
    k_stride, v_stride = _heads("k", k, b, hkv, d), _heads("v", v, b, hkv, d)
    _rope_args(q_weight, k_weight, positions, cos_sin, b, d)
    slots = _page_slots(slot_mapping, b, nb * bs, kind)
    if _range_checks and _checking():
        check_positions(positions, cos_sin.shape[0])
        check_paged_context(block_tables, context_lens, nb, bs, max_context_len)
    status = getattr(lib, name)(
        *args[:4], k.data_ptr(), k_stride, v.data_ptr(), v_stride, q_weight.data_ptr(), k_weight.data_ptr(),
        positions.data_ptr(), cos_sin.data_ptr(), cos_sin.shape[0], float(eps), *args[4:10], slots,
        *args[10:], context_lens.data_ptr(), b, hq, hkv, d, float(scale), max_context_len, workspace.data_ptr(),
        workspace.nbytes,
        _stream_of(device, q, k, v, out, q_weight, k_weight, positions, cos_sin, slot_mapping, block_tables,
                   context_lens, workspace))
    if status:
        _check(status, name)
    return out


def _prefill(kind: _Kind, out, q, key_pages, value_pages, block_tables, cu_seqlens_q, kv_lens, max_q_len,
             scale) -> torch.Tensor:
    lib, name = _lib or load(), kind.prefill
    if _calls and not _range_checks and type(key_pages) is kind.pages:
        made = _calls.prefill(out, q, key_pages, value_pages, block_tables, cu_seqlens_q, kv_lens, max_q_len, scale)
        if made is out or _made(made, name):
            return out
    if cu_seqlens_q.dtype is not torch.int32 or cu_seqlens_q.dim() != 1 or not cu_seqlens_q.is_contiguous():
        raise ValueError("cu_seqlens_q must be contiguous int32 [n + 1]")
    n = cu_seqlens_q.numel() - 1
    args, heads, device = _attention_args(kind, out, q, key_pages, value_pages, block_tables, n)
    if n < 0 or kv_lens.dtype is not torch.int32 or kv_lens.numel() < n or not kv_lens.is_contiguous():
        raise ValueError("kv_lens must be contiguous int32, one per sequence")
    max_q_len = _int32("max_q_len", max_q_len)
    if _range_checks and _checking():
        check_paged_context(block_tables[:n], kv_lens[:n], args[8], args[9])
    stream = _stream_of(device, q, out, block_tables, cu_seqlens_q, kv_lens)
    need = getattr(lib, kind.prefill_workspace)(n, max_q_len, heads[0], heads[1], args[9], args[12])
    space = torch.empty(need, dtype=torch.uint8, device=q.device) if need else None  # freed behind the call
    status = getattr(lib, name)(*args, cu_seqlens_q.data_ptr(), kv_lens.data_ptr(), n, q.shape[0], max_q_len,
                                *heads, float(scale), space.data_ptr() if need else None, need, stream)
    if status:
        _check(status, name)
    return out


def kv_cache_write_fp4(key_states: torch.Tensor, value_states: torch.Tensor, key_pages: Fp4Pages,
                       value_pages: Fp4Pages, slot_mapping: torch.Tensor) -> None:
    """Rows [T, Hkv, 128] of bf16 keys and values, quantised into the pages at their slots (-1: padding, skipped; no slot
    twice in a call)."""
    _write(_FP4, key_states, value_states, key_pages, value_pages, slot_mapping)


def kv_cache_write_fp8(key_states: torch.Tensor, value_states: torch.Tensor, key_pages: Fp8Pages,
                       value_pages: Fp8Pages, slot_mapping: torch.Tensor) -> None:
    """Rows [T, Hkv, 128] of bf16 keys and values, quantised into the pages at their slots (-1: padding, skipped).

    The rows of a tile of 16 slots follow one another, in the order of their slots, as a sequence's tokens do; tiles come
    in any order.  Rows in the tile of one of the 32 before them that do not follow it are not stored and reported
    (``ERR_ORDER`` in the error word); ``set_range_checks(True)`` refuses all other orders, too.  Rows that begin a tile set its scale and start it anew, others raise it where they need to and keep
    what the tile holds."""
    _write(_FP8, key_states, value_states, key_pages, value_pages, slot_mapping)


def kv_cache_read_fp4(key_pages: Fp4Pages, value_pages: Fp4Pages, slot_mapping: torch.Tensor,
                      k_out: torch.Tensor | None = None,
                      v_out: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """The bf16 keys and values [T, Hkv, 128] that the pages hold at the slots (zeros for -1)."""
    return _read(_FP4, key_pages, value_pages, slot_mapping, k_out, v_out)


def kv_cache_read_fp8(key_pages: Fp8Pages, value_pages: Fp8Pages, slot_mapping: torch.Tensor,
                      k_out: torch.Tensor | None = None,
                      v_out: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """``kv_cache_read_fp4`` of pages of 8 bits (slots in any order)."""
    return _read(_FP8, key_pages, value_pages, slot_mapping, k_out, v_out)


def _layers_fp8(pools):
    """Checks the tensors of a cache of 8 bits [layers, ...]; layers, blocks, block_size, kv heads, addresses, device."""
    kc, ks, vc, vs = pools
    if any(t.dim() < 2 or t.shape[0] != kc.shape[0] or t.shape[0] == 0 or not t.is_contiguous() for t in pools):
        raise ValueError("codes and scales must be contiguous tensors of as many layers")
    nb, bs, hkv, _, device = _checked_pages(_FP8, Fp8Pages(kc[0], ks[0]), Fp8Pages(vc[0], vs[0]))
    return kc.shape[0], nb, bs, hkv, [t.data_ptr() for t in pools], device


def kv_cache_keep_fp8(pools, slot_mapping: torch.Tensor) -> torch.Tensor:
    """The tiles of 16 slots, of every layer, that rows at these slots would go behind, as they are now.

    ``pools``: key codes, key scales, value codes and value scales of an ``Fp8PagedKVCache`` [layers, ...].  Such rows may
    raise a tile's scale, which rounds the codes of the others again; ``kv_cache_restore_fp8`` undoes it."""
    lib = _lib or load()
    layers, nb, bs, hkv, at, device = _layers_fp8(pools)
    t = slot_mapping.shape[0] if slot_mapping.dim() == 1 else -1
    slots = _page_slots(slot_mapping, t, nb * bs)
    stream = _stream_of(device, slot_mapping)
    kept = torch.empty((t, lib.nvamd_kv_cache_kept_size_fp8(layers, 1, hkv)), dtype=torch.uint8, device=pools[0].device)
    _check(lib.nvamd_kv_cache_keep_fp8(kept.data_ptr(), kept.nbytes, *at, layers, nb, bs, slots, t, hkv, _HEAD_DIM, stream),
           "nvamd_kv_cache_keep_fp8")
    return kept


def kv_cache_restore_fp8(pools, kept: torch.Tensor) -> None:
    """Puts back what ``kv_cache_keep_fp8`` kept: the tokens before those rows are again as they were."""
    lib = _lib or load()
    layers, nb, bs, hkv, at, device = _layers_fp8(pools)
    if (kept.dtype is not torch.uint8 or kept.dim() != 2 or not kept.is_contiguous()
            or kept.shape[1] != lib.nvamd_kv_cache_kept_size_fp8(layers, 1, hkv)):
        raise ValueError(f"kept must be what was kept of {layers} layers of {hkv} heads, got {tuple(kept.shape)}")
    _check(lib.nvamd_kv_cache_restore_fp8(kept.data_ptr(), kept.nbytes, *at, layers, nb, bs, kept.shape[0], hkv, _HEAD_DIM,
                                          _stream_of(device, kept)), "nvamd_kv_cache_restore_fp8")


def qk_norm_rope_fp4(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, q_weight: torch.Tensor,
                     k_weight: torch.Tensor, positions: torch.Tensor, cos_sin: torch.Tensor, eps: float,
                     key_pages: Fp4Pages, value_pages: Fp4Pages, slot_mapping: torch.Tensor, *,
                     q_out: torch.Tensor | None = None, k_out: torch.Tensor | None = None) -> torch.Tensor:
    """RoPE(RMSNorm_head(x) * w) of q and k in one pass that also stores the rotated k and the raw v in the pages.

    Returns the rotated q: ``q_out``, which may be q itself, or a new tensor.  The rotated k is written
    only to the pages unless ``k_out`` (which may be k itself) asks for it.  64-bit arithmetic, one rounding to bf16."""
    return _norm_rope(_FP4, q, k, v, q_weight, k_weight, positions, cos_sin, eps, key_pages, value_pages, slot_mapping,
                      q_out, k_out)


def qk_norm_rope_fp8(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, q_weight: torch.Tensor,
                     k_weight: torch.Tensor, positions: torch.Tensor, cos_sin: torch.Tensor, eps: float,
                     key_pages: Fp8Pages, value_pages: Fp8Pages, slot_mapping: torch.Tensor, *,
                     q_out: torch.Tensor | None = None, k_out: torch.Tensor | None = None) -> torch.Tensor:
    """``qk_norm_rope_fp4`` into pages of 8 bits (rows in the order that ``kv_cache_write_fp8`` asks for)."""
    return _norm_rope(_FP8, q, k, v, q_weight, k_weight, positions, cos_sin, eps, key_pages, value_pages, slot_mapping,
                      q_out, k_out)


def paged_decode_fp4(out: torch.Tensor | None, q: torch.Tensor, key_pages: Fp4Pages, value_pages: Fp4Pages,
                     block_tables: torch.Tensor, context_lens: torch.Tensor, scale: float, max_context_len: int,
                     workspace: torch.Tensor) -> torch.Tensor:
    """``paged_decode`` over pages of 4 bits; the workspace is the same (``alloc_paged_decode_workspace``).  Without
    ``out`` the result is a new tensor."""
    return _decode(_FP4, out, q, key_pages, value_pages, block_tables, context_lens, scale, max_context_len, workspace)


def paged_decode_fp8(out: torch.Tensor | None, q: torch.Tensor, key_pages: Fp8Pages, value_pages: Fp8Pages,
                     block_tables: torch.Tensor, context_lens: torch.Tensor, scale: float, max_context_len: int,
                     workspace: torch.Tensor) -> torch.Tensor:
    """``paged_decode_fp4`` over pages of 8 bits."""
    return _decode(_FP8, out, q, key_pages, value_pages, block_tables, context_lens, scale, max_context_len, workspace)


def paged_decode_fused_fp4(out: torch.Tensor | None, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor,
                           q_weight: torch.Tensor, k_weight: torch.Tensor, positions: torch.Tensor,
                           cos_sin: torch.Tensor, eps: float, key_pages: Fp4Pages, value_pages: Fp4Pages,
                           slot_mapping: torch.Tensor, block_tables: torch.Tensor, context_lens: torch.Tensor,
                           scale: float, max_context_len: int, workspace: torch.Tensor) -> torch.Tensor:
    """``qk_norm_rope_fp4`` and ``paged_decode_fp4`` in one launch, with the same bits: the step's k and v go to the slots
    of their sequences' last positions (-1: not stored), q, k and v stay as they are."""
    return _decode_fused(_FP4, out, q, k, v, q_weight, k_weight, positions, cos_sin, eps, key_pages, value_pages,
                         slot_mapping, block_tables, context_lens, scale, max_context_len, workspace)


def paged_decode_fused_fp8(out: torch.Tensor | None, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor,
                           q_weight: torch.Tensor, k_weight: torch.Tensor, positions: torch.Tensor,
                           cos_sin: torch.Tensor, eps: float, key_pages: Fp8Pages, value_pages: Fp8Pages,
                           slot_mapping: torch.Tensor, block_tables: torch.Tensor, context_lens: torch.Tensor,
                           scale: float, max_context_len: int, workspace: torch.Tensor) -> torch.Tensor:
    """``qk_norm_rope_fp8`` and ``paged_decode_fp8`` in one launch, with the same bits: the step's k and v go to the slots
    of their sequences' last positions (-1: not stored), q, k and v stay as they are."""
    return _decode_fused(_FP8, out, q, k, v, q_weight, k_weight, positions, cos_sin, eps, key_pages, value_pages,
                         slot_mapping, block_tables, context_lens, scale, max_context_len, workspace)


def paged_prefill_fp4(out: torch.Tensor, q: torch.Tensor, key_pages: Fp4Pages, value_pages: Fp4Pages,
                      block_tables: torch.Tensor, cu_seqlens_q: torch.Tensor, kv_lens: torch.Tensor, max_q_len: int,
                      scale: float) -> torch.Tensor:
    """``paged_prefill`` over pages of 4 bits: queries are the last q_len of kv_len positions, all keys in the cache."""
    return _prefill(_FP4, out, q, key_pages, value_pages, block_tables, cu_seqlens_q, kv_lens, max_q_len, scale)


def paged_prefill_fp8(out: torch.Tensor, q: torch.Tensor, key_pages: Fp8Pages, value_pages: Fp8Pages,
                      block_tables: torch.Tensor, cu_seqlens_q: torch.Tensor, kv_lens: torch.Tensor, max_q_len: int,
                      scale: float) -> torch.Tensor:
    """``paged_prefill`` over pages of 8 bits: queries are the last q_len of kv_len positions, all keys in the cache."""
    return _prefill(_FP8, out, q, key_pages, value_pages, block_tables, cu_seqlens_q, kv_lens, max_q_len, scale)


# ------------------------------------------------------------------ blocks of a cache
COPY_MAX_POOLS = 8


def check_block_pairs(sources: torch.Tensor, targets: torch.Tensor, num_blocks: int) -> None:
    """Blocks of the pool, no target twice, none that another pair reads."""
    src, dst = sources.detach().cpu().tolist(), targets.detach().cpu().tolist()
    if any(not 0 <= b < num_blocks for b in src + dst):
        raise IndexError(f"a block outside [0, {num_blocks}): {src} -> {dst}")
    read = {s for s, d in zip(src, dst) if s != d}
    if len(set(dst)) != len(dst) or read & set(dst):
        raise IndexError(f"a block is a target twice, or a target and a source: {src} -> {dst}")


def copy_blocks(pools, sources: torch.Tensor, targets: torch.Tensor) -> None:
    """pool[:, targets[i]] = pool[:, sources[i]] of every pool, in one launch.

    ``pools``: up to 8 contiguous tensors [layers, blocks, ...] of any type, with the same layers and blocks; sources and
    targets: int32 [n] on the device.  No block is a target twice, or a target and another pair's source."""
    lib = _lib or load()
    if _calls and not _range_checks and _made(_calls.copy(pools, sources, targets), "nvamd_copy_blocks"):
        return
    pools = list(pools)
    if not 0 < len(pools) <= COPY_MAX_POOLS:
        raise ValueError(f"1 to {COPY_MAX_POOLS} pools, got {len(pools)}")
    layers, blocks = pools[0].shape[:2] if pools[0].dim() > 2 else (0, 0)
    device = pools[0].get_device()
    for p in pools:
        if p.dim() < 3 or p.shape[:2] != (layers, blocks) or not p.is_contiguous() or p.numel() == 0:
            raise ValueError(f"pools must be contiguous [{layers}, {blocks}, ...] tensors, one is {tuple(p.shape)}")
    n = sources.shape[0] if sources.dim() == 1 else -1
    for name, t in (("sources", sources), ("targets", targets)):
        if t.dtype is not torch.int32 or t.shape != (n,) or not t.is_contiguous():
            raise ValueError(f"{name} must be contiguous int32 [n], got {t.dtype} {tuple(t.shape)}")
    if _range_checks and _checking():
        check_block_pairs(sources, targets, blocks)
    stream = _stream_of(device, sources, targets, *pools)
    at = (ctypes.c_void_p * len(pools))(*(p.data_ptr() for p in pools))
    sizes = (ctypes.c_int64 * len(pools))(*(p.nbytes // (layers * blocks) for p in pools))
    status = lib.nvamd_copy_blocks(at, sizes, len(pools), layers, blocks, sources.data_ptr(), targets.data_ptr(), n,
                                   stream)
    if status:
        _check(status, "nvamd_copy_blocks")


def add_rms_norm(delta: torch.Tensor | None, residual: torch.Tensor, weight: torch.Tensor, out: torch.Tensor,
                 eps: float) -> torch.Tensor:
    """residual += delta (if given); out = RMSNorm(residual) * weight.  Rows of any multiple of 8 bf16
    elements."""
    lib = load()
    _bf16_cuda("residual", residual)
    _bf16_cuda("out", out)
    _require(residual.is_contiguous() and out.is_contiguous() and out.shape == residual.shape, "rows must be dense")
    _require(weight.dtype == torch.bfloat16 and weight.numel() == residual.shape[-1], "weight must be bf16 [hidden]")
    if delta is not None:
        _require(delta.shape == residual.shape and delta.is_contiguous() and delta.dtype == torch.bfloat16,
                 "delta must match residual")
    hidden = residual.shape[-1]
    status = lib.nvamd_add_rms_norm(_ptr(delta), residual.data_ptr(), weight.data_ptr(), out.data_ptr(),
                                    residual.numel() // hidden, hidden, float(eps), _stream())
    _check(status, "nvamd_add_rms_norm")
    return out


def silu_mul(gate_up: torch.Tensor, out: torch.Tensor | None = None) -> torch.Tensor:
    """silu(gate_up[:, :I]) * gate_up[:, I:] for a [T, 2I] bf16 projection output."""
    lib = load()
    _bf16_cuda("gate_up", gate_up)
    t, two_i = gate_up.shape
    inter = two_i // 2
    out = torch.empty((t, inter), dtype=gate_up.dtype, device=gate_up.device) if out is None else out
    status = lib.nvamd_silu_mul(gate_up.data_ptr(), _row_stride(gate_up), out.data_ptr(), _row_stride(out), t, inter,
                                _stream())
    _check(status, "nvamd_silu_mul")
    return out


def argmax_rows(logits: torch.Tensor, out: torch.Tensor | None = None) -> torch.Tensor:
    """First index of each row's maximum (int64 [rows]) of a bf16 [rows, vocab] tensor."""
    lib = load()
    _bf16_cuda("logits", logits)
    rows, vocab = logits.shape
    out = torch.empty(rows, dtype=torch.int64, device=logits.device) if out is None else out
    _require(out.dtype == torch.int64 and out.numel() >= rows, "out must be int64 [rows]")
    status = lib.nvamd_argmax_rows(logits.data_ptr(), _row_stride(logits), rows, vocab, out.data_ptr(), _stream())
    _check(status, "nvamd_argmax_rows")
    return out


SKINNY_MAX_ROWS = 128  # rows the skinny projection kernels take (decode batches)
EPI_STORE, EPI_SILU, EPI_RESID = 0, 1, 2


def skinny_linear_workspace_size(n: int, k: int, epilogue: int = EPI_STORE) -> int:
    """Bytes of zero-filled workspace a skinny projection of this shape needs (0: none)."""
    return int(load().nvamd_skinny_linear_workspace_size(n, k, epilogue))


_SKINNY_COUNTER_BYTES = 16384  # arrival counters at the front of the workspace: the only part that has to be zero


def alloc_skinny_workspace(shapes, device) -> torch.Tensor:
    """A workspace for skinny projections of the given (n, k, epilogue) shapes, called one after another."""
    need = max([skinny_linear_workspace_size(*s) for s in shapes] + [16])
    ws = torch.empty(need, dtype=torch.uint8, device=device)
    ws[:_SKINNY_COUNTER_BYTES].zero_()
    return ws


GEMM_X_TILED = 1
GEMM_Y_TILED = 2


def is_tiled(t: torch.Tensor) -> bool:
    """A tiled matrix is a contiguous [rows/16, cols/32, 512] tensor (the skinny GEMM's operand order)."""
    return t.dim() == 3 and t.shape[2] == 512


def tile(a: torch.Tensor) -> torch.Tensor:
    """Row-major [R, C] (C % 32 == 0) -> tiled [ceil(R/16), C/32, 512]: 16 x 32 tiles, row-tile major,
    element (r, c) of a tile at 128 * (c // 8) + 8 * r + c % 8.  Padding rows are zero."""
    _require(a.dim() == 2 and a.shape[1] % 32 == 0, "tile() takes [R, C] with C % 32 == 0")
    r, c = a.shape
    rp = -(-r // 16) * 16
    if rp != r:
        a = torch.cat([a, a.new_zeros(rp - r, c)])
    return a.reshape(rp // 16, 16, c // 32, 4, 8).permute(0, 2, 3, 1, 4).reshape(rp // 16, c // 32, 512).contiguous()


def untile(t: torch.Tensor, rows: int | None = None) -> torch.Tensor:
    """Tiled [R/16, C/32, 512] -> row-major [rows, C] (a copy; rows defaults to R)."""
    _require(is_tiled(t), "untile() takes a tiled [R/16, C/32, 512] tensor")
    rt, ct, _ = t.shape
    a = t.reshape(rt, ct, 4, 16, 8).permute(0, 3, 1, 2, 4).reshape(rt * 16, ct * 32)
    return (a if rows is None else a[:rows]).contiguous()


def tiled_empty(rows: int, cols: int, device, dtype=torch.bfloat16) -> torch.Tensor:
    """Uninitialised tiled storage for a [rows, cols] matrix (rows padded to a multiple of 16)."""
    return torch.empty((-(-rows // 16), cols // 32, 512), dtype=dtype, device=device)


def skinny_linear(x: torch.Tensor, w: torch.Tensor, out: torch.Tensor | None = None, *, epilogue: int = EPI_STORE,
                  x_ssq: torch.Tensor | None = None, norm_weight: torch.Tensor | None = None, eps: float = 1e-6,
                  y_ssq: torch.Tensor | None = None, workspace: torch.Tensor | None = None, m: int | None = None,
                  y_tiled: bool = False, w_rows: bool = False) -> torch.Tensor:
    """Decode-batch projection x[M, K] @ W^T (M <= 128) with an optional RMSNorm prologue and a store,
    SiLU*mul or residual-add epilogue (one HIP launch).  Returns the output (the residual for EPI_RESID).

    w is the weight tiled (``tile(W)``; SILU: the fused [2I, K] gate/up weight), or with ``w_rows`` the
    contiguous [N, K] weight itself (no norm prologue).  x is row-major
    [M, K] or tiled (then ``m`` gives the valid rows); with ``y_tiled`` the output (the residual
    for EPI_RESID) is tiled with 16 * ceil(M/16) rows."""
    lib = load()
    _bf16_cuda("x", x)
    _bf16_cuda("w", w)
    if w_rows:
        _require(w.dim() == 2 and w.is_contiguous(), "w must be a contiguous [N, K] matrix")
        _require(x_ssq is None, "a row-major weight takes no norm prologue")
        wn, wk = w.shape
    else:
        _require(is_tiled(w), "w must be tiled: tile(W)")
        wn, wk = 16 * w.shape[0], 32 * w.shape[1]
    x_tiled = is_tiled(x)
    if x_tiled:
        _require(m is not None and 0 <= m <= 16 * x.shape[0], "a tiled x needs m <= its padded rows")
        _require(m <= 16 or x.shape[0] >= 2, "a tiled x of more than 16 rows holds 32")
        k = 32 * x.shape[1]
    else:
        m, k = x.shape
    _require(wk == k, "w must be [N, K], tiled [N/16, K/32, 512]")
    n = wn // 2 if epilogue == EPI_SILU else wn
    if epilogue == EPI_RESID:
        _require(out is not None, "the residual epilogue updates `out` in place")
        _require(y_ssq is not None and y_ssq.dtype == torch.float32 and y_ssq.is_contiguous()
                 and y_ssq.numel() >= m * (n // 32), "y_ssq must be fp32 [M, N/32]")
    if y_tiled:
        out = tiled_empty(max(m, 1), n, x.device) if out is None else out
        _require(is_tiled(out) and out.dtype == torch.bfloat16 and out.shape[1] * 32 == n
                 and 16 * out.shape[0] >= m and (m <= 16 or out.shape[0] >= 2), "out must be tiled bf16 [M, N]")
    else:
        out = torch.empty((m, n), dtype=x.dtype, device=x.device) if out is None else out
        _require(out.shape == (m, n) and out.dtype == torch.bfloat16 and out.stride(1) == 1,
                 "out must be bf16 [M, N]")
    if x_ssq is not None:
        _require(norm_weight is not None and norm_weight.dtype == torch.bfloat16 and norm_weight.numel() == k,
                 "norm_weight must be bf16 [K]")
        _require(x_ssq.dtype == torch.float32 and x_ssq.is_contiguous() and x_ssq.numel() >= m * (k // 32),
                 "x_ssq must be fp32 [M, K/32]")
    need = skinny_linear_workspace_size(n, k, epilogue) if n % 32 == 0 and k % 256 == 0 else 0
    if need and workspace is None:
        workspace = torch.zeros(need, dtype=torch.uint8, device=x.device)
    flags = (GEMM_X_TILED if x_tiled else 0) | (GEMM_Y_TILED if y_tiled else 0)
    tail = (out.data_ptr(), 0 if y_tiled else out.stride(0), _ptr(y_ssq), int(epilogue), flags, m, n, k,
            _ptr(workspace), workspace.numel() if workspace is not None else 0, _stream())
    x_args = (x.data_ptr(), 0 if x_tiled else _row_stride(x))
    if w_rows:
        status = lib.nvamd_skinny_linear_rows(*x_args, w.data_ptr(), *tail)
    else:
        status = lib.nvamd_skinny_linear(*x_args, _ptr(x_ssq), _ptr(norm_weight), float(eps), w.data_ptr(), *tail)
    _check(status, "nvamd_skinny_linear")
    return out


def rms_norm_tiled(x: torch.Tensor, weight: torch.Tensor, eps: float, out: torch.Tensor | None = None) -> torch.Tensor:
    """RMSNorm of row-major [M, H] (H % 32 == 0, H <= 8192), written tiled: the operand of ``skinny_linear`` where
    H is no width of its norm prologue.  Rounds like ``add_rms_norm``."""
    lib = load()
    _bf16_cuda("x", x)
    _bf16_cuda("weight", weight)
    _require(x.dim() == 2 and x.stride(1) == 1, "x must be [M, H] with dense rows")
    rows, hidden = x.shape
    _require(weight.numel() == hidden and weight.is_contiguous(), "weight must be [H]")
    out = tiled_empty(max(rows, 1), hidden, x.device) if out is None else out
    _require(is_tiled(out) and out.dtype == torch.bfloat16 and out.is_contiguous() and out.shape[1] * 32 == hidden
             and 16 * out.shape[0] >= rows, "out must be tiled bf16 [M, H]")
    status = lib.nvamd_rms_norm_tiled(x.data_ptr(), x.stride(0), weight.data_ptr(), out.data_ptr(), rows, hidden,
                                      float(eps), _stream())
    _check(status, "nvamd_rms_norm_tiled")
    return out


def linear(x: torch.Tensor, w_tiled: torch.Tensor, out: torch.Tensor | None = None,
           workspace: torch.Tensor | None = None) -> torch.Tensor:
    """x[M, K] @ W[N, K]^T in bf16 for M <= 128 (HIP skinny GEMM; w_tiled = tile(W))."""
    return skinny_linear(x, w_tiled, out, workspace=workspace)


def linear_silu_mul(x: torch.Tensor, w_gate_up_tiled: torch.Tensor, out: torch.Tensor | None = None,
                    workspace: torch.Tensor | None = None) -> torch.Tensor:
    """silu(x @ W[:I]^T) * (x @ W[I:]^T) in bf16 for M <= 128 (one HIP launch; W the [2I, K] gate/up
    weight, passed as tile(W))."""
    _require(w_gate_up_tiled.shape[0] % 2 == 0, "the gate/up weight must be [2I, K]")
    return skinny_linear(x, w_gate_up_tiled, out, epilogue=EPI_SILU, workspace=workspace)


def embed_rows(ids: torch.Tensor, table: torch.Tensor, out: torch.Tensor | None = None,
               ssq: torch.Tensor | None = None, out_tiled: bool = False) -> torch.Tensor:
    """table[ids] (zero rows for ids outside the vocab) and, if given, per-32-column sums of squares.
    With ``out_tiled`` the rows are written tiled (16 * ceil(rows/16) padded rows, padding untouched)."""
    lib = load()
    _bf16_cuda("table", table)
    _require(ids.dtype == torch.int64 and ids.is_cuda and ids.is_contiguous(), "ids must be int64 on the GPU")
    rows = ids.numel()
    vocab, hidden = table.shape
    if out_tiled:
        out = tiled_empty(max(rows, 1), hidden, table.device) if out is None else out
        _require(is_tiled(out) and out.dtype == torch.bfloat16 and out.shape[1] * 32 == hidden
                 and 16 * out.shape[0] >= rows, "out must be tiled bf16 [rows, hidden]")
    else:
        out = torch.empty((rows, hidden), dtype=table.dtype, device=table.device) if out is None else out
        _require(out.shape == (rows, hidden) and out.dtype == torch.bfloat16, "out must be bf16 [rows, hidden]")
    if ssq is not None:
        _require(ssq.dtype == torch.float32 and ssq.is_contiguous() and ssq.numel() >= rows * (hidden // 32),
                 "ssq must be fp32 [rows, hidden/32]")
    status = lib.nvamd_embed_rows(ids.data_ptr(), table.data_ptr(), _row_stride(table), vocab, out.data_ptr(),
                                  0 if out_tiled else _row_stride(out), int(out_tiled), _ptr(ssq), rows, hidden,
                                  _stream())
    _check(status, "nvamd_embed_rows")
    return out
