"""ctypes bridge to libm4_bridge.so -- the MI355X quantization-router prefill path.

Mirrors the reference's Python bridge (core/bridge/m4_bridge.py:18-280): the
same class and module-level names, format ints, M/K/N inference, non-zero
status -> RuntimeError mapping, deferred NaN/Inf tripwire at synchronize(),
and in-flight buffer retention until synchronize().  Buffers are torch-ROCm
tensors (device pointers, zero-copy) or numpy arrays (host memory, staged by
the library).  There is no fallback: if the shared library is missing the
constructor raises.
"""
from __future__ import annotations

import ctypes
import os
from enum import IntEnum
from pathlib import Path
from typing import Any, Optional, Union


class QuantFormat(IntEnum):
    """core/bridge/m4_bridge.py:18-24 (ids 0..5 are dispatchable)."""
    QUANT_Q4_0 = 0
    QUANT_MLX_4BIT = 1
    QUANT_Q4_K = 2
    QUANT_TERNARY_1_58 = 3
    QUANT_VAR_RATE_AFFINE = 4
    QUANT_EXL3 = 5
    # beyond the reference's dispatchable range (kernel-name entry points only)
    QUANT_Q8_0 = 6
    QUANT_PRISM_Q2_0 = 7
    QUANT_MLX_4BIT_G64 = 8  # MLX's native 64-element groups (36 B / 64)


LIB_NAME = "libm4_bridge.so"


def _find_library_path() -> Path:
    """Library location: $M4_BRIDGE_LIB_PATH (or the reference's
    $M4_BRIDGE_DYLIB_PATH), then next to this file, then the cwd
    (core/bridge/m4_bridge.py:27-44)."""
    for var in ("M4_BRIDGE_LIB_PATH", "M4_BRIDGE_DYLIB_PATH"):
        env = os.environ.get(var)
        if env and Path(env).is_file():
            return Path(env)
    here = Path(__file__).resolve().parent
    candidates = [here / LIB_NAME, here.parent / LIB_NAME, Path.cwd() / LIB_NAME]
    for cand in candidates:
        if cand.is_file():
            return cand
    raise FileNotFoundError(
        f"Could not locate {LIB_NAME}. Checked: {[str(c) for c in candidates]}. "
        "Build it with `python m4-prefill-engine_amd/build.py` or set M4_BRIDGE_LIB_PATH."
    )


_VP, _SZ, _I, _U32, _F = ctypes.c_void_p, ctypes.c_size_t, ctypes.c_int, ctypes.c_uint32, ctypes.c_float

# name -> (argtypes, restype); every symbol declared in include/m4_mlx_bridge.h
SIGNATURES = {
    "m4_bridge_init": ([ctypes.c_char_p], ctypes.c_bool),
    "m4_bridge_get_expected_weight_bytes": ([_I, _U32, _U32], _SZ),
    "m4_bridge_dispatch_gemm": ([_VP, _SZ, _VP, _SZ, _VP, _SZ, _I, _U32, _U32, _U32], _I),
    "m4_bridge_dispatch_gemv": ([_VP, _SZ, _VP, _SZ, _VP, _SZ, _I, _U32, _U32], _I),
    "m4_bridge_synchronize": ([], None),
    "m4_bridge_get_uma_footprint_mb": ([], ctypes.c_double),
    "m4_bridge_is_initialized": ([], ctypes.c_bool),
    "m4_bridge_shutdown": ([], None),
    "m4_bridge_validate_gemm": ([_VP, _SZ, _VP, _SZ, _VP, _SZ, _I, _U32, _U32, _U32], _I),
    "m4_bridge_dispatch_gemm_noalloc": ([_VP, _SZ, _VP, _SZ, _VP, _SZ, _I, _U32, _U32, _U32], _I),
    "m4_bridge_projection_plan": ([_I, _U32, _U32, ctypes.POINTER(_U32), _U32, _I, _VP], _I),
    "m4_bridge_dispatch_router_gemm": ([_VP, _SZ, _VP, _SZ, _VP, _SZ, _I, _U32, _U32, _U32], _I),
    "m4_bridge_dispatch_head_gemm": ([_VP, _SZ, _VP, _SZ, _VP, _SZ, _I, _U32, _U32, _U32, _U32], _I),
    "m4_bridge_dispatch_router_kernel": ([ctypes.c_char_p, _VP, _SZ, _VP, _SZ, _VP, _SZ,
                                          ctypes.POINTER(ctypes.c_uint32), _U32], _I),
    "m4_bridge_dispatch_gemm_residual": ([_VP, _SZ, _VP, _SZ, _VP, _SZ, _VP, _SZ, _I, _U32, _U32, _U32], _I),
    "m4_bridge_dispatch_swiglu": ([_VP, _SZ, _VP, _SZ, _VP, _SZ, _VP, _SZ, _I, _U32, _U32, _U32], _I),
    "m4_bridge_quantize_kv_q8_0": ([_VP, _SZ, _VP, _SZ, ctypes.c_uint64], _I),
    "m4_bridge_dispatch_flash_attn_q8_0": ([_VP, _SZ, _VP, _SZ, _VP, _SZ, _VP, _SZ, _U32, _U32, _U32, _F, _I], _I),
    "m4_bridge_prefill_layer": ([_VP] * 9 + [_I, _U32, _U32, _U32, _U32, _U32, _F], _I),
    "m4_bridge_dispatch_flash_attn_q8_0_gqa": ([_VP, _SZ, _VP, _SZ, _VP, _SZ, _VP, _SZ, _U32, _U32, _U32, _U32, _F,
                                                _I], _I),
    "m4_bridge_rmsnorm": ([_VP, _SZ, _VP, _SZ, _VP, _SZ, _U32, _U32, _F, _I], _I),
    "m4_bridge_rope": ([_VP, _SZ, _U32, _U32, _U32, _F, _U32, _I], _I),
    "m4_bridge_prefill_layer_ex": ([_VP] * 11 + [_I, _U32, _U32, _U32, _U32, _U32, _U32, _F, _I, _F, _I, _F, _U32,
                                                 _I], _I),
    "m4_bridge_prefill_layer_ex_kv": ([_VP] * 13 + [_I, _U32, _U32, _U32, _U32, _U32, _U32, _F, _I, _F, _I, _F,
                                                    _U32, _I], _I),
    "m4_bridge_dequantize": ([_VP, _SZ, _VP, _SZ, _I, _U32, _U32], _I),
    "m4_bridge_kv_cache_bytes": ([_I, _U32, _U32, _U32, _U32], _SZ),
    "m4_bridge_rope_axes_table": ([_VP, _VP, _U32, _U32, _VP], _I),
    "m4_bridge_rope_axes": ([_VP, _VP, _U32, _VP, _VP, _U32, _U32, _U32], _I),
    "m4_bridge_kv_cache_append": ([_VP, _VP, _U32, _VP, _VP, _VP, _VP, _U32, _VP, _VP, _U32], _I),
    "m4_bridge_kv_cache_read": ([_VP, _VP, _U32, _VP, _VP], _I),
    "m4_bridge_paged_attn_workspace": ([_VP, _VP, _U32, _U32, _U32], _SZ),
    "m4_bridge_dispatch_paged_attn": ([_VP, _VP, _U32, _VP, _VP, _U32, _F, _U32, _VP, _SZ], _I),
    "m4_bridge_draft_tree": ([_VP, _U32, _VP, _VP], _I),
    "m4_bridge_dispatch_paged_attn_tree": ([_VP, _VP, _U32, _VP, _VP, _U32, _F, _U32, _VP, _VP, _VP, _SZ], _I),
    "m4_bridge_tree_accept": ([_VP, _U32] + [_VP] * 6, _I),
    "m4_bridge_kv_cache_keep": ([_VP, _VP, _U32, _VP, _VP, _VP], _I),
    "m4_bridge_kv_cache_weigh": ([_VP, _VP, _U32, _VP, _VP, _U32, _F, _U32, _VP, _SZ], _I),
    "m4_bridge_kv_cache_evict": ([_VP, _VP, _VP, _SZ, _VP, _U32, _U32, _U32, _U32, _U32, _VP, _SZ, _VP, _VP, _SZ], _I),
    "m4_bridge_kv_evict_workspace": ([_VP, _VP], _SZ),
    "m4_bridge_paged_layer": ([_VP] * 13 + [_U32, _VP, _VP, _U32, _I, _U32, _U32, _U32, _F, _U32, _I, _F], _I),
    "m4_bridge_validate_rope_axes": ([_VP, _VP, _U32, _VP, _VP, _U32, _U32, _U32], _I),
    "m4_bridge_validate_kv_cache_append": ([_VP, _VP, _U32, _VP, _VP, _VP, _VP, _U32, _VP, _VP, _U32], _I),
    "m4_bridge_validate_kv_cache_read": ([_VP, _VP, _U32, _VP, _VP], _I),
    "m4_bridge_validate_paged_attn": ([_VP, _VP, _U32, _VP, _VP, _U32, _F, _U32, _VP, _SZ], _I),
    "m4_bridge_validate_draft_tree": ([_VP, _U32, _VP, _VP], _I),
    "m4_bridge_validate_paged_attn_tree": ([_VP, _VP, _U32, _VP, _VP, _U32, _F, _U32, _VP, _VP, _VP, _SZ], _I),
    "m4_bridge_validate_tree_accept": ([_VP, _U32] + [_VP] * 6, _I),
    "m4_bridge_validate_kv_cache_keep": ([_VP, _VP, _U32, _VP, _VP, _VP], _I),
    "m4_bridge_validate_kv_cache_weigh": ([_VP, _VP, _U32, _VP, _VP, _U32, _F, _U32, _VP, _SZ], _I),
    "m4_bridge_validate_kv_cache_evict": ([_VP, _VP, _VP, _SZ, _VP, _U32, _U32, _U32, _U32, _U32, _VP, _SZ, _VP, _VP, _SZ], _I),
    "m4_bridge_set_stream": ([_VP], _I),
    "m4_bridge_get_stream": ([], _VP),
    "m4_bridge_last_error": ([], ctypes.c_char_p),
    "m4_probe_hbm_bandwidth": ([_SZ, _I, ctypes.POINTER(ctypes.c_double), ctypes.POINTER(ctypes.c_double)], _I),
    "m4_probe_mfma_f16": ([_U32, _I, ctypes.POINTER(ctypes.c_double), ctypes.POINTER(ctypes.c_double)], _I),
    "m4_probe_mfma_f16_random": ([_U32, _I, ctypes.POINTER(ctypes.c_double), ctypes.POINTER(ctypes.c_double)], _I),
    "m4_registry_get": ([_I, _VP], _I),
    "m4_registry_get_by_name": ([ctypes.c_char_p], _I),
    "m4_registry_available_formats": ([ctypes.POINTER(_I), _I], _I),
    "m4_registry_compute_weight_bytes": ([_I, ctypes.c_uint64], ctypes.c_uint64),
    "m4_registry_has_format": ([_I], ctypes.c_bool),
    "m4_registry_register_codec": ([_VP], _I),
}


class CodecInfo(ctypes.Structure):
    """m4_quant_codec_info (include/m4_mlx_bridge.h)."""
    _fields_ = [
        ("format", ctypes.c_int),
        ("name", ctypes.c_char_p),
        ("description", ctypes.c_char_p),
        ("block_size", ctypes.c_uint32),
        ("struct_size", ctypes.c_uint64),
        ("bits_per_weight", ctypes.c_double),
        ("gemm_kernel_name", ctypes.c_char_p),
        ("head_gemm_kernel_name", ctypes.c_char_p),
    ]


class ProjectionPlan(ctypes.Structure):
    """m4_projection_plan_t (include/m4_mlx_bridge.h)."""
    _fields_ = [("kernel", ctypes.c_int), ("tile_rows", _U32), ("tile_cols", _U32), ("k_groups", _U32),
                ("k_splits", _U32)]

    KERNELS = ("few_rows", "small_m", "tiled", "wide")

    @property
    def kernel_name(self) -> str:
        return self.KERNELS[self.kernel]

    def astuple(self) -> tuple:
        return (self.kernel_name, self.tile_rows, self.tile_cols, self.k_groups, self.k_splits)


def projection_plan(lib: ctypes.CDLL, format_id: int, M: int, K: int, *N: int, swiglu: bool = False) -> ProjectionPlan:
    """The kernel that [M, K] x [N, K]^T in a format runs (several N: projections
    launched together), from the library's own choice; no GPU needed."""
    plan = ProjectionPlan()
    rc = lib.m4_bridge_projection_plan(int(format_id), M, K, (_U32 * len(N))(*N), len(N), int(swiglu),
                                       ctypes.byref(plan))
    if rc:
        raise ValueError(f"m4_bridge_projection_plan failed with status code {rc}")
    return plan


_torch: Any = None  # the module, once a library is loaded


class KVCacheStruct(ctypes.Structure):
    """m4_kv_cache_t (include/m4_mlx_bridge.h)."""
    _fields_ = [("pages", _VP), ("bytes", _SZ), ("format", _I), ("num_pages", _U32), ("page_size", _U32),
                ("Hkv", _U32), ("D", _U32)]


class KVBatchStruct(ctypes.Structure):
    """m4_kv_batch_t (include/m4_mlx_bridge.h)."""
    _fields_ = [("B", _U32), ("q_start", _VP), ("kv_len", _VP), ("page_table", _VP),
                ("table_pages", _U32), ("table_stride", _U32), ("max_new", _U32), ("max_kv", _U32)]


class RowsStruct(ctypes.Structure):
    """m4_rows_t (include/m4_mlx_bridge.h)."""
    _fields_ = [("ptr", _VP), ("bytes", _SZ), ("token_stride", ctypes.c_int64), ("head_stride", ctypes.c_int64)]


_ROWS = ctypes.sizeof(RowsStruct)
# two and four m4_rows_t as words: one object a call is made faster than one for each
_ROWS2, _ROWS4 = ctypes.c_uint64 * 8, ctypes.c_uint64 * 16


class RopeAxesStruct(ctypes.Structure):
    """m4_rope_axes_t (include/m4_mlx_bridge.h)."""
    MAX_PAIRS, PAIR_BYTES = 128, 12
    _fields_ = [("pairs", _U32), ("axes", _U32), ("traditional", _I), ("table", _VP), ("table_bytes", _SZ)]


def _int32(name: str, t: Any, dims: int) -> Any:
    import torch

    if not isinstance(t, torch.Tensor) or t.dtype != torch.int32 or t.dim() != dims:
        raise ValueError(f"{name} must be an int32 tensor with {dims} dimension(s)")
    if t.numel() and t.stride(-1) != 1:
        raise ValueError(f"{name} must be contiguous along its last dimension")
    return t


class PagedKVCache:
    """One layer's paged, quantized KV cache (m4_kv_cache_t): `num_pages` pages of
    `page_size` tokens (16, 32, 64, 128 or 256), `Hkv` heads of `D` (64 or 128) dims, in
    format Q8_0 or Q4_0.  `pages` is its memory, a uint8 tensor of any shape (made
    here when it is None)."""

    def __init__(self, format: Union[int, QuantFormat], num_pages: int, page_size: int, Hkv: int, D: int, pages=None,
                 device: str = "cuda") -> None:
        import torch

        self.format, self.num_pages, self.page_size, self.Hkv, self.D = int(format), num_pages, page_size, Hkv, D
        need = self.nbytes(format, num_pages, page_size, Hkv, D)
        if need == 0:
            raise ValueError(f"no paged cache of format {int(format)}, {num_pages} pages of {page_size} tokens, "
                             f"{Hkv} heads of {D}")
        if pages is None:
            pages = torch.zeros(need, dtype=torch.uint8, device=device)
        if not isinstance(pages, torch.Tensor) or pages.dtype != torch.uint8 or not pages.is_contiguous():
            raise ValueError("pages must be a contiguous uint8 tensor")
        if pages.numel() < need:
            raise ValueError(f"pages holds {pages.numel()} bytes, {need} are needed")
        self.pages = pages
        self.struct = KVCacheStruct(pages.data_ptr(), pages.numel(), self.format, num_pages, page_size, Hkv, D)
        self.ref = ctypes.addressof(self.struct)

    @staticmethod
    def nbytes(format: Union[int, QuantFormat], num_pages: int, page_size: int, Hkv: int, D: int) -> int:
        dims = (num_pages, page_size, Hkv, D)
        if not all(0 <= d < 1 << 32 for d in dims):
            return 0
        return int(HIPBridge.get_instance().lib.m4_bridge_kv_cache_bytes(int(format), *dims))


class KVBatch:
    """The sequences of a call (m4_kv_batch_t).  q_start [B + 1], kv_len [B] and
    page_table [B, pages] are int32 device tensors that the kernels read when they
    run, so a captured graph follows what is written to them.  The rows
    q_start[b] .. q_start[b + 1] of a call are the last keys of sequence b, which has
    kv_len[b] keys with them.  max_new and max_kv: what to expect of the longest
    sequence (None reads them from the device, which waits for it); they choose
    kernels and the workspace, results hold for any lengths."""

    def __init__(self, q_start, kv_len, page_table, max_new: Optional[int] = None, max_kv: Optional[int] = None) -> None:
        self.q_start, self.kv_len = _int32("q_start", q_start, 1), _int32("kv_len", kv_len, 1)
        self.page_table = _int32("page_table", page_table, 2)
        B = kv_len.shape[0]
        if q_start.shape[0] != B + 1 or page_table.shape[0] != B:
            raise ValueError(f"q_start, kv_len and page_table disagree: {q_start.shape[0]}, {B} and "
                             f"{page_table.shape[0]} rows (B + 1, B, B)")
        if max_new is None:
            max_new = int(q_start.diff().max().item()) if B else 0
        if max_kv is None:
            max_kv = int(kv_len.max().item()) if B else 0
        self.B = B
        self.struct = KVBatchStruct(B, q_start.data_ptr(), kv_len.data_ptr(), page_table.data_ptr(),
                                    page_table.shape[1], page_table.stride(0), max(int(max_new), 0), max(int(max_kv), 0))
        self.ref = ctypes.addressof(self.struct)


class RotaryAxes:
    """Rotary embedding of the first `dims` dims of a head (m4_rope_axes_t): pair i turns
    by positions[pair_axes[i]] * inv_freq[i], inv_freq theta^(-2i / dims) unless given.
    `sections`: pairs per axis, in runs (time, height, width); `pair_axes`: the axis
    of each pair, for any other order; neither: one axis.  Pairs are dims
    (i, i + dims / 2), or (2i, 2i + 1) when traditional."""

    def __init__(self, dims: int, theta: float = 10000.0, sections=None, pair_axes=None, inv_freq=None,
                 traditional: bool = False) -> None:
        import torch

        pairs = dims // 2
        if dims <= 0 or dims % 16 or pairs > RopeAxesStruct.MAX_PAIRS:
            raise ValueError(f"dims={dims} must be a positive multiple of 16, at most {2 * RopeAxesStruct.MAX_PAIRS}")
        if sections is not None and pair_axes is not None:
            raise ValueError("give sections or pair_axes, not both")
        if sections is not None:
            pair_axes = [a for a, n in enumerate(sections) for _ in range(n)]
        if pair_axes is None:
            pair_axes = [0] * pairs
        pair_axes = [int(a) for a in pair_axes]
        if len(pair_axes) != pairs or min(pair_axes) < 0 or max(pair_axes) > 255:
            raise ValueError(f"{pairs} pairs need an axis each, got {len(pair_axes)}")
        if inv_freq is None:
            if not theta > 0:
                raise ValueError(f"theta={theta} must be positive")
            inv_freq = [float(theta) ** (-i / pairs) for i in range(pairs)]
        inv_freq = [float(f) for f in inv_freq]
        if len(inv_freq) != pairs:
            raise ValueError(f"{pairs} pairs need a frequency each, got {len(inv_freq)}")
        axes = max(pair_axes) + 1 if sections is None else max(len(sections), 1)
        self.dims, self.axes, self.traditional = dims, axes, bool(traditional)
        self._table = (ctypes.c_uint8 * (pairs * RopeAxesStruct.PAIR_BYTES))()
        rc = HIPBridge.get_instance().lib.m4_bridge_rope_axes_table((ctypes.c_double * pairs)(*inv_freq),
                                                                    (ctypes.c_uint8 * pairs)(*pair_axes), pairs, axes,
                                                                    self._table)
        if rc:
            raise ValueError(f"m4_bridge_rope_axes_table failed with status code {rc}")
        self._on: dict = {}  # device -> (table, struct, its address)
        if torch.cuda.is_available():
            self.on(torch.device("cuda", torch.cuda.current_device()))

    def on(self, device) -> int:
        """Address of the struct for a device, whose copy of the table is made on first use (the current device's with
        the object; another's before a capture)."""
        held = self._on.get(device)
        if held is None:
            import torch

            t = torch.frombuffer(bytearray(self._table), dtype=torch.uint8).to(device)
            struct = RopeAxesStruct(self.dims // 2, self.axes, int(self.traditional), t.data_ptr(), t.numel())
            held = self._on[device] = (t, struct, ctypes.addressof(struct))
        return held[2]


class DraftTreeStruct(ctypes.Structure):
    """m4_draft_tree_t (include/m4_mlx_bridge.h)."""
    _fields_ = [("mask", _VP), ("mask_bytes", _SZ), ("positions", _VP), ("positions_bytes", _SZ), ("words", _U32)]


class DraftTree:
    """What each of a call's T rows sees of its sequence's new tokens (m4_draft_tree_t): bit j % 32 of mask[row][j // 32]
    (int32 [T, words]) for the j-th of them, and each row's position (int32 [T]; None where no window is used).  Any
    mask will do; HIPBridge.draft_tree fills both from the nodes' parents."""

    def __init__(self, mask, positions=None) -> None:
        import torch

        if not isinstance(mask, torch.Tensor) or mask.dtype != torch.int32 or mask.dim() != 2 or not mask.is_contiguous():
            raise ValueError("mask must be a contiguous int32 tensor [T, words]")
        if mask.shape[1] == 0:
            raise ValueError("a mask needs a word a row at least")
        if positions is not None:
            _int32("positions", positions, 1)
            if positions.shape[0] != mask.shape[0]:
                raise ValueError(f"mask has {mask.shape[0]} rows, positions {positions.shape[0]}")
        self.mask, self.positions = mask, positions
        self.T, self.words = mask.shape
        self.struct = DraftTreeStruct(mask.data_ptr(), mask.nbytes, positions.data_ptr() if positions is not None else None,
                                      positions.nbytes if positions is not None else 0, self.words)
        self.ref = ctypes.addressof(self.struct)

    @classmethod
    def empty(cls, T: int, max_nodes: int, device="cuda") -> "DraftTree":
        """For T rows of trees with at most `max_nodes` nodes, to be filled."""
        import torch

        return cls(torch.empty(T, max(1, -(-max_nodes // 32)), dtype=torch.int32, device=device),
                   torch.empty(T, dtype=torch.int32, device=device))


def load_library(path: Optional[Union[str, Path]] = None) -> ctypes.CDLL:
    # One HIP runtime per process: torch-ROCm ships its own libamdhip64.so.7.
    # Importing torch first makes the library bind to that already-loaded
    # runtime (same SONAME) instead of loading /opt/rocm's beside it, which
    # would leave torch without a usable device.
    global _torch
    try:
        import torch as _torch
    except ImportError:
        pass
    lib = ctypes.CDLL(str(Path(path) if path else _find_library_path()))
    for name, (args, res) in SIGNATURES.items():
        fn = getattr(lib, name)
        fn.argtypes = args
        fn.restype = res
    return lib


def _is_torch(x: Any) -> bool:
    return type(x).__module__.startswith("torch")


def _current_stream(device: int) -> int:
    """Handle of torch's current stream on a device.  The raw getter returns it
    without building a Stream object (0.2 instead of 2.0 us, of ~8 us that an
    eager call takes on the host)."""
    global _raw_stream
    if _raw_stream is None:
        import torch

        _raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (
            lambda d: torch.cuda.current_stream(d).cuda_stream)
    return _raw_stream(device)


_raw_stream: Any = None


class HIPBridge:
    """Counterpart of the reference's MetalUMABridge (core/bridge/m4_bridge.py:47-242)."""

    _instance: Optional["HIPBridge"] = None
    _retained_contig: list = []

    def __init__(self, lib_path: Optional[Union[str, Path]] = None) -> None:
        self._lib = load_library(lib_path)
        self._in_flight_tensors: list[tuple] = []
        self._pending_finite_checks: list = []

    @property
    def lib(self) -> ctypes.CDLL:
        return self._lib

    @classmethod
    def get_instance(cls, lib_path: Optional[Union[str, Path]] = None) -> "HIPBridge":
        if cls._instance is None:
            cls._instance = cls(lib_path)
        return cls._instance

    # -- buffers ------------------------------------------------------------
    @classmethod
    def extract_buffer_address_and_size(cls, arr: Any) -> tuple[int, int]:
        """(address, nbytes) of a torch tensor or numpy array; non-contiguous
        inputs are made contiguous and retained until synchronize()
        (core/bridge/m4_bridge.py:110-127)."""
        if _is_torch(arr):
            if not arr.is_contiguous():
                arr = arr.contiguous()
                cls._retained_contig.append(arr)
            return arr.data_ptr(), arr.nbytes
        import numpy as np

        a = arr
        if not isinstance(a, np.ndarray):
            raise TypeError(f"unsupported buffer type {type(arr)!r}")
        if not a.flags["C_CONTIGUOUS"]:
            a = np.ascontiguousarray(a)
            cls._retained_contig.append(a)
        return int(a.ctypes.data), int(a.nbytes)

    def _bind_stream(self, *bufs: Any) -> None:
        """Issue on torch's current stream when any buffer is a CUDA tensor, so
        the kernels are ordered after the work that produced the inputs."""
        for b in bufs:
            if _is_torch(b) and b.is_cuda:
                self._lib.m4_bridge_set_stream(_current_stream(b.get_device()))
                return

    def _check(self, name: str, ret: int) -> int:
        if ret != 0:
            raise RuntimeError(f"{name} failed with status code {ret}")
        return ret

    # -- reference API ------------------------------------------------------
    def init(self, metallib_path: Optional[str] = None) -> bool:
        c_path = metallib_path.encode("utf-8") if metallib_path else None
        return bool(self._lib.m4_bridge_init(c_path))

    def is_initialized(self) -> bool:
        return bool(self._lib.m4_bridge_is_initialized())

    def get_expected_weight_bytes(self, format: Union[int, QuantFormat], K: int, N: int) -> int:
        return int(self._lib.m4_bridge_get_expected_weight_bytes(int(format), K, N))

    def dispatch_gemm(self, X, W, Y, format, M=None, K=None, N=None, check_finite: bool = False) -> int:
        """Y[M,N] = X[M,K] . W^T (core/bridge/m4_bridge.py:136-179)."""
        x_ptr, x_bytes = self.extract_buffer_address_and_size(X)
        w_ptr, w_bytes = self.extract_buffer_address_and_size(W)
        y_ptr, y_bytes = self.extract_buffer_address_and_size(Y)
        if M is None:
            M = X.shape[0] if len(X.shape) >= 2 else 1
        if K is None:
            K = X.shape[1] if len(X.shape) >= 2 else X.shape[0]
        if N is None:
            N = Y.shape[1] if len(Y.shape) >= 2 else Y.shape[0]
        self._bind_stream(X, W, Y)
        ret = self._lib.m4_bridge_dispatch_gemm(x_ptr, x_bytes, w_ptr, w_bytes, y_ptr, y_bytes, int(format),
                                                int(M), int(K), int(N))
        self._check("m4_bridge_dispatch_gemm", ret)
        self._in_flight_tensors.append((X, W, Y))
        if check_finite:
            self._pending_finite_checks.append(Y)
        return ret

    def dispatch_gemv(self, x, W, y, format, K=None, N=None, check_finite: bool = False) -> int:
        """y[N] = W . x (core/bridge/m4_bridge.py:181-220)."""
        x_ptr, x_bytes = self.extract_buffer_address_and_size(x)
        w_ptr, w_bytes = self.extract_buffer_address_and_size(W)
        y_ptr, y_bytes = self.extract_buffer_address_and_size(y)
        if K is None:
            K = x.shape[-1]
        if N is None:
            N = y.shape[-1]
        self._bind_stream(x, W, y)
        ret = self._lib.m4_bridge_dispatch_gemv(x_ptr, x_bytes, w_ptr, w_bytes, y_ptr, y_bytes, int(format),
                                                int(K), int(N))
        self._check("m4_bridge_dispatch_gemv", ret)
        self._in_flight_tensors.append((x, W, y))
        if check_finite:
            self._pending_finite_checks.append(y)
        return ret

    def synchronize(self) -> None:
        """Waits for the issued work, releases retained buffers, then runs the
        deferred NaN/Inf tripwire (core/bridge/m4_bridge.py:222-233)."""
        self._lib.m4_bridge_synchronize()
        self._in_flight_tensors.clear()
        self._retained_contig.clear()
        if self._pending_finite_checks:
            checks = list(self._pending_finite_checks)
            self._pending_finite_checks.clear()
            for t in checks:
                if not _all_finite(t):
                    raise FloatingPointError(
                        "Tripwire assertion failed: Non-finite values (NaN/Inf) detected in output tensor.")

    def get_uma_footprint_mb(self) -> float:
        return float(self._lib.m4_bridge_get_uma_footprint_mb())

    def shutdown(self) -> None:
        self._in_flight_tensors.clear()
        self._retained_contig.clear()
        self._pending_finite_checks.clear()
        self._lib.m4_bridge_shutdown()

    # -- router extensions ----------------------------------------------------
    def dispatch_router_gemm(self, X, W, Y, format, M=None, K=None, N=None, check_finite: bool = False) -> int:
        """Y = X . W^T for every format with a kernel, PRISM_Q2_0 and Q8_0 weights
        included (quant_router_gemm_<fmt>_64x64, quant_router_kernels.metal:588-750)."""
        x_ptr, x_bytes = self.extract_buffer_address_and_size(X)
        w_ptr, w_bytes = self.extract_buffer_address_and_size(W)
        y_ptr, y_bytes = self.extract_buffer_address_and_size(Y)
        M = X.shape[0] if M is None else M
        K = X.shape[1] if K is None else K
        N = Y.shape[1] if N is None else N
        self._bind_stream(X, W, Y)
        ret = self._lib.m4_bridge_dispatch_router_gemm(x_ptr, x_bytes, w_ptr, w_bytes, y_ptr, y_bytes, int(format),
                                                       int(M), int(K), int(N))
        self._check("m4_bridge_dispatch_router_gemm", ret)
        self._in_flight_tensors.append((X, W, Y))
        if check_finite:
            self._pending_finite_checks.append(Y)
        return ret

    def dispatch_head_gemm(self, X, W, Y, format, M, H, D, K, check_finite: bool = False) -> int:
        """Direct-head projection: Y [H, M, D] (quant_router_kernels.metal:754-927)."""
        a = [self.extract_buffer_address_and_size(t) for t in (X, W, Y)]
        self._bind_stream(X, W, Y)
        ret = self._lib.m4_bridge_dispatch_head_gemm(a[0][0], a[0][1], a[1][0], a[1][1], a[2][0], a[2][1],
                                                     int(format), M, H, D, K)
        self._check("m4_bridge_dispatch_head_gemm", ret)
        self._in_flight_tensors.append((X, W, Y))
        if check_finite:
            self._pending_finite_checks.append(Y)
        return ret

    def dispatch_router_kernel(self, kernel_name: str, X, W, Y, *dims, check_finite: bool = False) -> int:
        """A router kernel by its Metal pipeline name with that kernel's slots:
        buffers A = X, B = W, C = Y, then the constants -- (M, N, K) for
        quant_router_gemm_<fmt>_64x64, (M, H, D, K) for the head kernels
        (quant_router_kernels.metal:588-927).  The vector-ALU ternary names
        quant_router_{,head_}gemm_ternary_1_58_vec (:934-1201) compute the same
        projection on the matrix-core path."""
        a = [self.extract_buffer_address_and_size(t) for t in (X, W, Y)]
        self._bind_stream(X, W, Y)
        arr = (ctypes.c_uint32 * max(len(dims), 1))(*[int(d) for d in dims])
        ret = self._lib.m4_bridge_dispatch_router_kernel(kernel_name.encode(), a[0][0], a[0][1], a[1][0], a[1][1],
                                                         a[2][0], a[2][1], arr, len(dims))
        self._check("m4_bridge_dispatch_router_kernel", ret)
        self._in_flight_tensors.append((X, W, Y))
        if check_finite:
            self._pending_finite_checks.append(Y)
        return ret

    def dispatch_gemm_residual(self, X, W, R, Y, format, M, K, N) -> int:
        a = [self.extract_buffer_address_and_size(t) for t in (X, W, R, Y)]
        self._bind_stream(X, W, R, Y)
        ret = self._lib.m4_bridge_dispatch_gemm_residual(a[0][0], a[0][1], a[1][0], a[1][1], a[2][0], a[2][1],
                                                         a[3][0], a[3][1], int(format), M, K, N)
        self._check("m4_bridge_dispatch_gemm_residual", ret)
        self._in_flight_tensors.append((X, W, R, Y))
        return ret

    def dispatch_swiglu(self, X, Wg, Wu, Out, format, M, N_mlp, K) -> int:
        """Out = silu(X . Wg^T) * (X . Wu^T) (brick3_swiglu_kernels.metal:428-698)."""
        a = [self.extract_buffer_address_and_size(t) for t in (X, Wg, Wu, Out)]
        self._bind_stream(X, Wg, Wu, Out)
        ret = self._lib.m4_bridge_dispatch_swiglu(a[0][0], a[0][1], a[1][0], a[1][1], a[2][0], a[2][1],
                                                  a[3][0], a[3][1], int(format), M, N_mlp, K)
        self._check("m4_bridge_dispatch_swiglu", ret)
        self._in_flight_tensors.append((X, Wg, Wu, Out))
        return ret

    def quantize_kv_q8_0(self, src, dst, num_blocks: Optional[int] = None) -> int:
        """fp16 -> Q8_0 blocks (unified_kernels.metal:118-145)."""
        s = self.extract_buffer_address_and_size(src)
        d = self.extract_buffer_address_and_size(dst)
        nb = s[1] // 64 if num_blocks is None else num_blocks
        self._bind_stream(src, dst)
        ret = self._lib.m4_bridge_quantize_kv_q8_0(s[0], s[1], d[0], d[1], nb)
        self._check("m4_bridge_quantize_kv_q8_0", ret)
        self._in_flight_tensors.append((src, dst))
        return ret

    def dispatch_flash_attn_q8_0(self, Q, Kq, Vq, O, H, M, D, scale, o_token_major: bool = False) -> int:
        """Causal attention over a Q8_0 KV cache (brick4_attn_kernels.metal:572-911)."""
        a = [self.extract_buffer_address_and_size(t) for t in (Q, Kq, Vq, O)]
        self._bind_stream(Q, Kq, Vq, O)
        ret = self._lib.m4_bridge_dispatch_flash_attn_q8_0(a[0][0], a[0][1], a[1][0], a[1][1], a[2][0], a[2][1],
                                                           a[3][0], a[3][1], H, M, D, float(scale),
                                                           int(bool(o_token_major)))
        self._check("m4_bridge_dispatch_flash_attn_q8_0", ret)
        self._in_flight_tensors.append((Q, Kq, Vq, O))
        return ret

    def prefill_layer(self, X, Wq, Wk, Wv, Wo, Wg, Wu, Wd, X_out, format, M, d_model, H, D, N_mlp,
                      attn_scale) -> int:
        """One prefill layer (models/transformer_layer.mm:75-218) over device tensors."""
        bufs = (X, Wq, Wk, Wv, Wo, Wg, Wu, Wd, X_out)
        ptrs = [self.extract_buffer_address_and_size(t)[0] for t in bufs]
        self._bind_stream(*bufs)
        ret = self._lib.m4_bridge_prefill_layer(*ptrs, int(format), M, d_model, H, D, N_mlp, float(attn_scale))
        self._check("m4_bridge_prefill_layer", ret)
        self._in_flight_tensors.append(bufs)
        return ret

    def dispatch_flash_attn_q8_0_gqa(self, Q, Kq, Vq, O, H, Hkv, M, D, scale, o_token_major: bool = False) -> int:
        """Grouped-query causal attention: K/V hold Hkv heads (src/engine/model.py:234-236)."""
        a = [self.extract_buffer_address_and_size(t) for t in (Q, Kq, Vq, O)]
        self._bind_stream(Q, Kq, Vq, O)
        ret = self._lib.m4_bridge_dispatch_flash_attn_q8_0_gqa(a[0][0], a[0][1], a[1][0], a[1][1], a[2][0], a[2][1],
                                                               a[3][0], a[3][1], H, Hkv, M, D, float(scale),
                                                               int(bool(o_token_major)))
        self._check("m4_bridge_dispatch_flash_attn_q8_0_gqa", ret)
        self._in_flight_tensors.append((Q, Kq, Vq, O))
        return ret

    def rmsnorm(self, X, w, Y, eps: float = 1e-5, norm_type: int = 1) -> int:
        """RMSNorm over the rows of X [M, D] (src/engine/model.py:39-48); norm_type 2 = gemma_add_one."""
        a = [self.extract_buffer_address_and_size(t) for t in (X, w, Y)]
        M, D = X.shape
        self._bind_stream(X, w, Y)
        ret = self._lib.m4_bridge_rmsnorm(a[0][0], a[0][1], a[1][0], a[1][1], a[2][0], a[2][1], M, D, float(eps),
                                          int(norm_type))
        self._check("m4_bridge_rmsnorm", ret)
        self._in_flight_tensors.append((X, w, Y))
        return ret

    def rope(self, T, theta: float = 10000.0, offset: int = 0, traditional: bool = False) -> int:
        """RoPE in place on T [H, M, D] (nn.RoPE, src/engine/model.py:112-116)."""
        ptr, nbytes = self.extract_buffer_address_and_size(T)
        H, M, D = T.shape
        self._bind_stream(T)
        ret = self._lib.m4_bridge_rope(ptr, nbytes, H, M, D, float(theta), int(offset), int(bool(traditional)))
        self._check("m4_bridge_rope", ret)
        self._in_flight_tensors.append((T,))
        return ret

    def prefill_layer_ex(self, X, w_attn, Wq, Wk, Wv, Wo, w_ffn, Wg, Wu, Wd, X_out, format, M, d_model, Hq, Hkv, D,
                         N_mlp, attn_scale, norm_type: int = 1, norm_eps: float = 1e-5, rope: bool = True,
                         rope_theta: float = 10000.0, rope_offset: int = 0, rope_traditional: bool = False) -> int:
        """The MLX transformer block on the router's kernels (src/engine/model.py:181-265)."""
        bufs = (X, w_attn, Wq, Wk, Wv, Wo, w_ffn, Wg, Wu, Wd, X_out)
        ptrs = [None if t is None else self.extract_buffer_address_and_size(t)[0] for t in bufs]
        self._bind_stream(*[t for t in bufs if t is not None])
        ret = self._lib.m4_bridge_prefill_layer_ex(*ptrs, int(format), M, d_model, Hq, Hkv, D, N_mlp,
                                                   float(attn_scale), int(norm_type), float(norm_eps), int(bool(rope)),
                                                   float(rope_theta), int(rope_offset), int(bool(rope_traditional)))
        self._check("m4_bridge_prefill_layer_ex", ret)
        self._in_flight_tensors.append(bufs)
        return ret

    def prefill_layer_ex_kv(self, X, w_attn, Wq, Wk, Wv, Wo, w_ffn, Wg, Wu, Wd, X_out, Kq_out, Vq_out, format, M,
                            d_model, Hq, Hkv, D, N_mlp, attn_scale, norm_type: int = 1, norm_eps: float = 1e-5,
                            rope: bool = True, rope_theta: float = 10000.0, rope_offset: int = 0,
                            rope_traditional: bool = False) -> int:
        """prefill_layer_ex that also writes the layer's Q8_0 K / V cache
        (unified_prefill_engine.mm:548-572) to Kq_out / Vq_out."""
        bufs = (X, w_attn, Wq, Wk, Wv, Wo, w_ffn, Wg, Wu, Wd, X_out, Kq_out, Vq_out)
        ptrs = [None if t is None else self.extract_buffer_address_and_size(t)[0] for t in bufs]
        self._bind_stream(*[t for t in bufs if t is not None])
        ret = self._lib.m4_bridge_prefill_layer_ex_kv(*ptrs, int(format), M, d_model, Hq, Hkv, D, N_mlp,
                                                      float(attn_scale), int(norm_type), float(norm_eps),
                                                      int(bool(rope)), float(rope_theta), int(rope_offset),
                                                      int(bool(rope_traditional)))
        self._check("m4_bridge_prefill_layer_ex_kv", ret)
        self._in_flight_tensors.append(bufs)
        return ret

    # -- serving over a paged KV cache -----------------------------------------
    def _rows(self, name: str, t: Any, token_major: bool, heads: Optional[int], D: Optional[int], out: bool) -> tuple:
        """(m4_rows_t's four words, T, heads, tensor) of fp16 rows [heads, T, D], or [T, heads, D] when token_major.
        Any strides that keep 8 elements together are taken as they are; other inputs
        are copied (and retained until synchronize())."""
        if not isinstance(t, _torch.Tensor) or t.dtype is not _torch.float16 or len(t.shape) != 3:
            raise ValueError(f"{name} must be an fp16 tensor with 3 dimensions")
        a, b, d = t.shape
        T, H = (a, b) if token_major else (b, a)
        if (heads is not None and H != heads) or (D is not None and d != D):
            raise ValueError(f"{name} has {H} heads of {d}, expected {heads} of {D}")
        sa, sb, sd = t.stride()
        ptr = t.data_ptr()
        if sd != 1 or (sa | sb) & 7 or ptr & 15:
            if t.numel() and out:
                raise ValueError(f"{name} must be contiguous along its last dimension, 16-byte aligned, with strides "
                                 f"that are multiples of 8")
            t = t.clone(memory_format=_torch.contiguous_format)
            self._retained_contig.append(t)
            sa, sb, sd = t.stride()
            ptr = t.data_ptr()
        ts, hs = (sa, sb) if token_major else (sb, sa)
        held = ((T - 1) * ts + (H - 1) * hs + d) * 2 if T and H else 0
        return (ptr, held, ts, hs), T, H, t

    def _positions(self, positions: Any, rope: "RotaryAxes", T: int) -> tuple:
        """(pointer, stride) of int32 positions [T] or [axes, T], expanded over the axes (stride 0) included."""
        if positions is None:
            return None, 0
        shape = positions.shape
        if positions.dtype is not _torch.int32 or len(shape) not in (1, 2) or (T and positions.stride(-1) != 1):
            raise ValueError("positions must be int32 [T] or [axes, T], contiguous along T")
        if shape[-1] != T or (shape[0] if len(shape) == 2 else 1) < rope.axes:
            raise ValueError(f"positions {tuple(shape)} do not give {rope.axes} axes of {T} tokens")
        return positions.data_ptr(), (positions.stride(0) if len(shape) == 2 else T)

    def _on_stream_of(self, t: Any) -> None:
        device = t.get_device()
        if device >= 0:
            self._lib.m4_bridge_set_stream(_current_stream(device))

    def rope_axes(self, X, Y, rope: RotaryAxes, positions, token_major: bool = False) -> int:
        """Y = X [H, T, D] (or [T, H, D]) turned by positions [T] or [axes, T]; Y may be X."""
        x, T, H, X = self._rows("X", X, token_major, None, None, False)
        y, Ty, _, _ = self._rows("Y", Y, token_major, H, X.shape[2], True)
        if positions is None or Ty != T:
            raise ValueError("X and Y need the same rows, and positions")
        pos, stride = self._positions(positions, rope, T)
        self._on_stream_of(X)
        rows = _ROWS2(*x, *y)
        at = ctypes.addressof(rows)
        ret = self._lib.m4_bridge_rope_axes(rope.on(X.device), pos, stride, at, at + _ROWS, T, H, X.shape[2])
        self._check("m4_bridge_rope_axes", ret)
        self._in_flight_tensors.append((X, Y, rope, positions))
        return ret

    def kv_cache_append(self, cache: PagedKVCache, batch: KVBatch, K, V, rope: Optional[RotaryAxes] = None,
                        positions=None, Q=None, Q_out=None, token_major: bool = False) -> int:
        """Writes the batch's rows of K, V [Hkv, T, D] (or [T, Hkv, D]) to the cache, K turned by `rope` first; Q
        [H, T, D] is turned into Q_out (Q itself when None) by the same launch.  positions
        None: each token's place in its sequence."""
        k, T, _, K = self._rows("K", K, token_major, cache.Hkv, cache.D, False)
        v, Tv, _, V = self._rows("V", V, token_major, cache.Hkv, cache.D, False)
        if Tv != T:
            raise ValueError(f"K has {T} rows, V {Tv}")
        if Q is None and Q_out is not None:
            raise ValueError("Q_out without Q")
        if Q is not None and rope is None:
            raise ValueError("Q is turned by rope: give both or neither")
        pos, stride = self._positions(positions, rope, T) if rope is not None else (None, 0)
        q = qo = (0, 0, 0, 0)
        H = 0
        if Q is not None:
            Q_out = Q if Q_out is None else Q_out
            qo, To, H, _ = self._rows("Q_out", Q_out, token_major, None, cache.D, True)
            q, Tq, _, Q = (qo, To, H, Q) if Q is Q_out else self._rows("Q", Q, token_major, H, cache.D, False)
            if Tq != T or To != T:
                raise ValueError(f"K has {T} rows, Q {Tq} and Q_out {To}")
        self._on_stream_of(K)
        rows = _ROWS4(*k, *v, *q, *qo)
        at = ctypes.addressof(rows)
        at_q, at_qo = (at + 2 * _ROWS, at + 3 * _ROWS) if Q is not None else (None, None)
        ret = self._lib.m4_bridge_kv_cache_append(cache.ref, batch.ref, T, at, at + _ROWS,
                                                  rope.on(K.device) if rope is not None else None, pos, stride, at_q,
                                                  at_qo, H)
        self._check("m4_bridge_kv_cache_append", ret)
        self._in_flight_tensors.append((cache, batch, K, V, rope, Q, Q_out, positions))
        return ret

    def kv_cache_read(self, cache: PagedKVCache, batch: KVBatch, K, V, token_major: bool = False) -> int:
        """The cached values of the batch's rows into K, V [Hkv, T, D] (or [T, Hkv, D])."""
        k, T, _, _ = self._rows("K", K, token_major, cache.Hkv, cache.D, True)
        v, Tv, _, _ = self._rows("V", V, token_major, cache.Hkv, cache.D, True)
        if Tv != T:
            raise ValueError(f"K has {T} rows, V {Tv}")
        self._on_stream_of(K)
        rows = _ROWS2(*k, *v)
        at = ctypes.addressof(rows)
        ret = self._lib.m4_bridge_kv_cache_read(cache.ref, batch.ref, T, at, at + _ROWS)
        self._check("m4_bridge_kv_cache_read", ret)
        self._in_flight_tensors.append((cache, batch, K, V))
        return ret

    def paged_attn_workspace(self, cache: PagedKVCache, batch: KVBatch, H: int, T: int, window: int = 0) -> int:
        """Bytes of workspace that dispatch_paged_attn needs for T rows of H heads."""
        return int(self._lib.m4_bridge_paged_attn_workspace(cache.ref, batch.ref, T, H, window))

    def _lse(self, lse: Any, H: int, T: int, out: bool) -> tuple:
        """m4_rows_t's words for fp32 [H, T], any strides."""
        if not isinstance(lse, _torch.Tensor) or lse.dtype is not _torch.float32 or lse.shape != (H, T):
            raise ValueError(f"lse must be an fp32 tensor [{H}, {T}]")
        hs, ts = lse.stride()
        if out and T * H and ((T > 1 and ts == 0) or (H > 1 and hs == 0)):
            raise ValueError("lse has values that share their memory")
        return lse.data_ptr(), ((T - 1) * ts + (H - 1) * hs + 1) * 4 if T and H else 0, ts, hs

    def _tree(self, tree: "DraftTree", T: int) -> int:
        if tree.T != T:
            raise ValueError(f"the tree has {tree.T} rows, the call {T}")
        return tree.ref

    def _ids(self, name: str, t: Any, n: int) -> int:
        if not isinstance(t, _torch.Tensor) or t.dtype is not _torch.int32 or t.shape != (n,) or not t.is_contiguous():
            raise ValueError(f"{name} must be a contiguous int32 tensor [{n}]")
        return t.data_ptr()

    def draft_tree(self, batch: KVBatch, parents, tree: DraftTree) -> int:
        """Fills `tree` for the batch's rows from their parents, int32 [T]: node numbers within the sequence, -1 for
        none.  Once a step, for all layers; kv_cache_append takes tree.positions."""
        if tree.positions is None:
            raise ValueError("the tree has no positions to fill")
        at = self._ids("parents", parents, tree.T)
        self._on_stream_of(parents)
        ret = self._lib.m4_bridge_draft_tree(batch.ref, tree.T, at, tree.ref)
        self._check("m4_bridge_draft_tree", ret)
        self._in_flight_tensors.append((batch, parents, tree))
        return ret

    def tree_accept(self, batch: KVBatch, parents, tokens, targets, path, count, next_token) -> int:
        """The model's path down each tree: from node 0 on, the first node behind whose token is the model's choice
        (`targets`).  All int32: parents, tokens, targets, path [T]; count, next_token [B]."""
        T, B = parents.shape[0], batch.B
        ptrs = [self._ids(n, t, T) for n, t in (("parents", parents), ("tokens", tokens), ("targets", targets), ("path", path))]
        ptrs += [self._ids(n, t, B) for n, t in (("count", count), ("next_token", next_token))]
        self._on_stream_of(parents)
        ret = self._lib.m4_bridge_tree_accept(batch.ref, T, *ptrs)
        self._check("m4_bridge_tree_accept", ret)
        self._in_flight_tensors.append((batch, parents, tokens, targets, path, count, next_token))
        return ret

    def kv_cache_keep(self, cache: PagedKVCache, batch: KVBatch, keep, count, kv_len_out=None) -> int:
        """Of each sequence's new tokens the count[b] that its rows of `keep` [T] name (rising, as tree_accept's path)
        move to the places of the first; kv_len_out [B] (may be batch.kv_len): what the sequences then hold."""
        T = keep.shape[0]
        ptrs = [self._ids("keep", keep, T), self._ids("count", count, batch.B),
                self._ids("kv_len_out", kv_len_out, batch.B) if kv_len_out is not None else None]
        self._on_stream_of(keep)
        ret = self._lib.m4_bridge_kv_cache_keep(cache.ref, batch.ref, T, *ptrs)
        self._check("m4_bridge_kv_cache_keep", ret)
        self._in_flight_tensors.append((cache, batch, keep, count, kv_len_out))
        return ret

    def _sums(self, cache: PagedKVCache, sums: Any) -> tuple:
        shape = (cache.num_pages, cache.Hkv, cache.page_size)
        if not isinstance(sums, _torch.Tensor) or sums.dtype is not _torch.float32 or sums.shape != shape or not sums.is_contiguous():
            raise ValueError(f"sums must be a contiguous fp32 tensor {list(shape)}")
        return sums.data_ptr(), sums.nbytes

    def kv_cache_weigh(self, cache: PagedKVCache, batch: KVBatch, Q, lse, sums, scale: float, token_major: bool = False,
                       window: int = 0) -> int:
        """Adds to sums [num_pages, Hkv, page_size] (fp32) the weight that the batch's rows Q [H, T, D] (or [T, H, D]) give
        each key they see, for the batch's own tokens in place of what was there; lse [H, T] (fp32, any strides) as
        dispatch_paged_attn writes it for the same rows, scale and window."""
        q, T, H, Q = self._rows("Q", Q, token_major, None, cache.D, False)
        z = self._lse(lse, H, T, False)
        at_sums, held = self._sums(cache, sums)
        if not 0 <= window < 1 << 32:
            raise ValueError(f"window={window}")
        self._on_stream_of(Q)
        rows = _ROWS2(*q, *z)
        at = ctypes.addressof(rows)
        ret = self._lib.m4_bridge_kv_cache_weigh(cache.ref, batch.ref, T, at, at + _ROWS, H, float(scale), window, at_sums, held)
        self._check("m4_bridge_kv_cache_weigh", ret)
        self._in_flight_tensors.append((cache, batch, Q, lse, sums))
        return ret

    def kv_evict_workspace(self, cache: PagedKVCache, batch: KVBatch) -> int:
        """Bytes of workspace that kv_cache_evict needs; 0 for many or short sequences."""
        return int(self._lib.m4_bridge_kv_evict_workspace(cache.ref, batch.ref))

    def kv_cache_evict(self, cache: PagedKVCache, batch: KVBatch, sums, table_out, kv_len_out, budget: int, sinks: int = 0,
                       recent: int = 0, kept=None, workspace=None) -> int:
        """Copies of each sequence and KV head the first `sinks`, the last `recent` and the heaviest other keys by `sums`,
        `budget` together, to the pages of table_out (int32 [B, pages]), in their order and with their sums.
        kv_len_out int32 [B]: how many; kept int32 [B, Hkv, budget]: the places that they had, then -1 (None: not
        wanted).  `workspace`: a uint8 device tensor of kv_evict_workspace bytes, where these are any, as
        dispatch_paged_attn's.  The caller goes on with table_out and kv_len_out and has the old pages back."""
        B = batch.B
        _int32("table_out", table_out, 2)
        if table_out.shape[0] != B:
            raise ValueError(f"table_out has {table_out.shape[0]} rows, the batch {B}")
        for name, v in (("budget", budget), ("sinks", sinks), ("recent", recent)):
            if not 0 <= v < 1 << 32:
                raise ValueError(f"{name}={v}")
        at_sums, held = self._sums(cache, sums)
        at_len = self._ids("kv_len_out", kv_len_out, B)
        given = kept  # one made here goes back to the stream that the kernels are on, behind them
        if kept is None:
            kept = _torch.empty(B, cache.Hkv, budget, dtype=_torch.int32, device=sums.device)
        elif kept.dtype is not _torch.int32 or kept.shape != (B, cache.Hkv, budget) or not kept.is_contiguous():
            raise ValueError(f"kept must be a contiguous int32 tensor [{B}, {cache.Hkv}, {budget}]")
        if workspace is not None and not (isinstance(workspace, _torch.Tensor) and workspace.is_contiguous()):
            raise ValueError("workspace must be a contiguous tensor")
        self._on_stream_of(sums)
        given_ws = workspace
        if workspace is None:
            need = self.kv_evict_workspace(cache, batch)
            workspace = _torch.empty(need, dtype=_torch.uint8, device=sums.device) if need else None
        ret = self._lib.m4_bridge_kv_cache_evict(cache.ref, batch.ref, at_sums, held, table_out.data_ptr(), table_out.shape[1],
                                                 table_out.stride(0), budget, sinks, recent, kept.data_ptr(), kept.nbytes,
                                                 at_len, workspace.data_ptr() if workspace is not None else None,
                                                 workspace.nbytes if workspace is not None else 0)
        self._check("m4_bridge_kv_cache_evict", ret)
        self._in_flight_tensors.append((cache, batch, sums, table_out, kv_len_out, given, given_ws))
        return ret

    def dispatch_paged_attn(self, cache: PagedKVCache, batch: KVBatch, Q, O, scale: float, token_major: bool = False,
                            o_token_major: bool = False, window: int = 0, workspace=None,
                            tree: Optional[DraftTree] = None, lse=None) -> int:
        """Causal attention of the batch's rows Q [H, T, D] (or [T, H, D]) over their sequences' cached keys (append
        first); O [H, T, D], or [T, H, D] when o_token_major.  `workspace`: a uint8 device tensor of
        paged_attn_workspace bytes, not shared with a call that may run at the same time (None: from torch's
        allocator, on the current stream).  `tree`: which of its sequence's new tokens a row sees, in place of those up
        to itself; `lse` [H, T] (fp32, any strides): receives the logarithm of each row's sum of exponentials."""
        q, T, H, Q = self._rows("Q", Q, token_major, None, cache.D, False)
        o, To, _, _ = self._rows("O", O, o_token_major, H, cache.D, True)
        if To != T:
            raise ValueError(f"Q has {T} rows, O {To}")
        if not 0 <= window < 1 << 32:
            raise ValueError(f"window={window}")
        if workspace is not None and not (isinstance(workspace, _torch.Tensor) and workspace.is_contiguous()):
            raise ValueError("workspace must be a contiguous tensor")  # its bytes are counted from its address on
        at_tree = self._tree(tree, T) if tree is not None else None
        if tree is not None and window and tree.positions is None:
            raise ValueError("a window needs the tree's positions")
        z = self._lse(lse, H, T, True) if lse is not None else None
        self._on_stream_of(Q)
        given = workspace  # one made here goes back to the stream that the kernels are on, behind them
        if workspace is None:
            workspace = _torch.empty(self.paged_attn_workspace(cache, batch, H, T, window), dtype=_torch.uint8,
                                     device=Q.device)
        if tree is None and lse is None:
            rows = _ROWS2(*q, *o)
            at = ctypes.addressof(rows)
            ret = self._lib.m4_bridge_dispatch_paged_attn(cache.ref, batch.ref, T, at, at + _ROWS, H, float(scale), window,
                                                          workspace.data_ptr(), workspace.nbytes)
            self._check("m4_bridge_dispatch_paged_attn", ret)
            self._in_flight_tensors.append((cache, batch, Q, O, given))
            return ret
        rows = _ROWS4(*q, *o, *(z or (0, 0, 0, 0)), 0, 0, 0, 0)
        at = ctypes.addressof(rows)
        ret = self._lib.m4_bridge_dispatch_paged_attn_tree(cache.ref, batch.ref, T, at, at + _ROWS, H, float(scale), window,
                                                           at_tree, at + 2 * _ROWS if z else None, workspace.data_ptr(),
                                                           workspace.nbytes)
        self._check("m4_bridge_dispatch_paged_attn_tree", ret)
        self._in_flight_tensors.append((cache, batch, Q, O, given, tree, lse))
        return ret

    def paged_layer(self, X, w_attn, Wq, Wk, Wv, Wo, w_ffn, Wg, Wu, Wd, X_out, format, d_model, Hq, N_mlp, attn_scale,
                    cache: PagedKVCache, batch: KVBatch, rope: Optional[RotaryAxes] = None, positions=None,
                    norm_type: int = 1, norm_eps: float = 1e-5, window: int = 0) -> int:
        """prefill_layer_ex over a paged cache: X, X_out [T, d_model] are the batch's rows, whose keys are appended and
        whose queries see their sequences' (positions None: each token's place)."""
        bufs = (X, w_attn, Wq, Wk, Wv, Wo, w_ffn, Wg, Wu, Wd, X_out)
        T = X.shape[0]
        if not 0 <= window < 1 << 32:
            raise ValueError(f"window={window}")
        for name, t in (("X", X), ("X_out", X_out)):
            if t.dtype is not _torch.float16 or tuple(t.shape) != (T, d_model) or not t.is_contiguous():
                raise ValueError(f"{name} must be contiguous fp16 [{T}, {d_model}]")
        ptrs = [None if t is None else self.extract_buffer_address_and_size(t)[0] for t in bufs]
        pos, stride = self._positions(positions, rope, T) if rope is not None else (None, 0)
        self._on_stream_of(X)
        ret = self._lib.m4_bridge_paged_layer(*ptrs, cache.ref, batch.ref, T,
                                              rope.on(X.device) if rope is not None else None, pos, stride, int(format),
                                              d_model, Hq, N_mlp, float(attn_scale), window, int(norm_type),
                                              float(norm_eps))
        self._check("m4_bridge_paged_layer", ret)
        self._in_flight_tensors.append((*bufs, cache, batch, rope, positions))
        return ret

    def dequantize(self, W, out, format, K, N) -> int:
        a = [self.extract_buffer_address_and_size(t) for t in (W, out)]
        self._bind_stream(W, out)
        ret = self._lib.m4_bridge_dequantize(a[0][0], a[0][1], a[1][0], a[1][1], int(format), K, N)
        self._check("m4_bridge_dequantize", ret)
        self._in_flight_tensors.append((W, out))
        return ret

    def last_error(self) -> str:
        return (self._lib.m4_bridge_last_error() or b"").decode()


# The reference's class name, for callers written against it.
MetalUMABridge = HIPBridge


def _all_finite(t: Any) -> bool:
    if _is_torch(t):
        import torch

        return bool(torch.isfinite(t).all().item())
    import numpy as np

    a = np.asarray(t)
    if a.dtype == np.uint16:
        a = a.view(np.float16)
    return bool(np.isfinite(a).all())


# Module-level convenience functions matching the C-ABI (core/bridge/m4_bridge.py:245-280)
def m4_bridge_init(metallib_path: Optional[str] = None) -> bool:
    return HIPBridge.get_instance().init(metallib_path)


def m4_bridge_dispatch_gemm(X, W, Y, format, M=None, K=None, N=None, check_finite: bool = False) -> int:
    return HIPBridge.get_instance().dispatch_gemm(X, W, Y, format, M, K, N, check_finite=check_finite)


def m4_bridge_dispatch_gemv(x, W, y, format, K=None, N=None, check_finite: bool = False) -> int:
    return HIPBridge.get_instance().dispatch_gemv(x, W, y, format, K, N, check_finite=check_finite)


def m4_bridge_synchronize() -> None:
    HIPBridge.get_instance().synchronize()


def m4_bridge_get_uma_footprint_mb() -> float:
    return HIPBridge.get_instance().get_uma_footprint_mb()
