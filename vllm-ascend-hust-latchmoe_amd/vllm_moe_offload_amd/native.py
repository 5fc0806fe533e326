"""ctypes binding of liblatchmoe_hip.so (the gfx950 hot-path kernels).

Every wrapper takes torch tensors that already live on the GPU, checks shape,
dtype and contiguity on the host, and launches on the current torch stream
(or the stream given).  Nothing here falls back to a CPU or PyTorch
implementation: if the library is missing the import of a wrapper raises.

The C declarations live in include/latchmoe.h; `EXPORTED_SYMBOLS` lists them.
"""

from __future__ import annotations

import atexit
import contextlib
import ctypes
import os
from dataclasses import dataclass
from pathlib import Path

import torch

from vllm_moe_offload_amd import mxfp4

LIB_PATH = Path(__file__).resolve().parent / "lib" / "liblatchmoe_hip.so"

LMOE_SCORING_SOFTMAX = 0
LMOE_SCORING_SIGMOID = 1
LMOE_PATH_AUTO = 0
LMOE_PATH_GEMV = 1
LMOE_PATH_MFMA = 2
LMOE_PATH_STREAM = 3
LMOE_ERR_ARG = 1000
LMOE_ERR_SHAPE = 1001
META_ACTIVE, META_PAIRS, META_ERRORS, META_TILES = 0, 1, 2, 3
META_GEN, META_ROUTER_TIMEOUT = 4, 6
ROUTER_SYNC_WORDS = 64 + 2 * 16 * 256  # LMOE_ROUTER_SYNC_WORDS: arrival count, then the tagged logit words
META_COUNT = 64  # LMOE_META_COUNT
FLAG_UNPLACED, FLAG_ROUTER_TIMEOUT, FLAG_COUNT = 0, 1, 4  # lmoe_device_flags words
MFMA_BLOCK_M = 256  # row-tile height of the prefill MFMA GEMM (tile table of lmoe_permute)
STREAM_BLOCK_M = 96  # row tiles of the weight-streaming MFMA kernel (few pairs per slot)
PART_BLOCK_M = 320  # row tiles of the one-workgroup-per-CU prefill GEMM (lmoe_grouped_mlp)
FUSED_DECODE_MAX_PAIRS = 1024
SKIP_KEEP_ROWS = 2  # LMOE_SKIP_KEEP_ROWS: lmoe_permute mode of the later passes of a multi-pass layer
GEMV_MAX_I = 4096  # the decode GEMV kernels hold at most 16 chunks of 256 act columns
TWO_PASS_MAX_COLS = 4096  # lmoe_decode_mlp_two_passes: the row-per-wave GEMVs only
PERMUTE_TWO_MAX_PAIRS = 1024  # lmoe_permute_two_tables: one workgroup per table

EXPORTED_SYMBOLS = (
    "lmoe_status_string",
    "lmoe_abi_version",
    "lmoe_device_flags",
    "lmoe_router_gate",
    "lmoe_router_topk",
    "lmoe_router_topk_permute",
    "lmoe_router_gate_topk_permute",
    "lmoe_router_gate_topk_pairs",
    "lmoe_permute_workspace_bytes",
    "lmoe_permute",
    "lmoe_permute_two_tables",
    "lmoe_gather_rows",
    "lmoe_grouped_mlp",
    "lmoe_grouped_mlp_pass",
    "lmoe_gateup_silu",
    "lmoe_down",
    "lmoe_decode_mlp_two_passes",
    "lmoe_stream_mlp_two_passes",
    "lmoe_combine",
    "lmoe_combine_f32",
    "lmoe_add_rms_norm",
    "lmoe_rows_to_mx8",
    "lmoe_mx4_bytes",
    "lmoe_mx4_gateup_silu",
    "lmoe_mx4_down",
    "lmoe_mx4_fused_moe",
    "lmoe_mx4_decode_few",
    "lmoe_mx4_decode_one",
    "lmoe_fused_moe_decode",
    "lmoe_fused_moe_decode_noalloc",
    "lmoe_down_combine",
    "lmoe_stage_copy",
    "lmoe_stage_gather",
    "lmoe_table_update",
    "lmoe_slot_plan",
    "lmoe_wave_plan_bytes",
    "lmoe_wave_plan",
    "lmoe_wave_stage",
)

_vp = ctypes.c_void_p
_i = ctypes.c_int
_f = ctypes.c_float
_sz = ctypes.c_size_t

_SIGNATURES = {
    "lmoe_status_string": (ctypes.c_char_p, [_i]),
    "lmoe_abi_version": (_i, []),
    "lmoe_device_flags": (_i, [_vp, _i, _vp]),
    "lmoe_router_gate": (_i, [_vp, _vp, _i, _i, _i, _vp, _i, _vp]),
    "lmoe_router_topk": (
        _i,
        [_vp, _i, _i, _i, _i, _i, _i, _vp, _vp, _i, _i, _i, _f, _vp, _vp, _vp, _vp],
    ),
    "lmoe_router_topk_permute": (
        _i,
        [_vp, _i, _i, _i, _i, _i, _i, _vp, _vp, _i, _i, _i, _f, _vp, _vp, _vp,
         _vp, _i, _i, _i, _i, _vp, _vp, _vp, _vp, _vp, _vp, _vp, _vp],
    ),
    "lmoe_router_gate_topk_permute": (
        _i,
        [_vp, _vp, _i, _i, _i, _vp, _i, _i, _i, _i, _vp, _vp, _i, _i, _i, _f, _vp, _vp, _vp,
         _vp, _i, _i, _i, _i, _vp, _vp, _vp, _vp, _vp, _vp, _vp, _vp, _vp],
    ),
    "lmoe_router_gate_topk_pairs": (
        _i,
        [_vp, _vp, _i, _i, _vp, _i, _i, _i, _i, _vp, _vp, _i, _i, _i, _f, _vp, _vp, _vp, _vp, _i, _i, _i,
         _vp, _vp, _vp, _vp, _vp, _vp],
    ),
    "lmoe_permute_workspace_bytes": (_sz, [_i, _i]),
    "lmoe_permute": (
        _i,
        [_vp, _i, _vp, _i, _i, _i, _i, _vp, _vp, _vp, _vp, _vp, _vp, _vp, _vp, _sz, _vp],
    ),
    "lmoe_permute_two_tables": (
        _i,
        [_vp, _i, _i, _vp, _vp, _i, _i, _vp, _vp, _vp, _vp, _vp, _vp, _vp, _i, _i, _vp, _vp, _vp, _vp, _vp,
         _vp, _vp],
    ),
    "lmoe_gather_rows": (_i, [_vp, _i, _i, _vp, _vp, _i, _vp, _vp]),
    "lmoe_grouped_mlp": (
        _i,
        [_vp, _i, _i, _i, _i, _vp, _vp, _i, _vp, _vp, _vp, _vp, _vp, _i, _i, _i, _vp, _vp, _vp],
    ),
    "lmoe_grouped_mlp_pass": (
        _i,
        [_vp, _i, _i, _i, _i, _vp, _vp, _i, _vp, _vp, _vp, _vp, _vp, _i, _i, _i, _i, _vp, _vp, _vp],
    ),
    "lmoe_gateup_silu": (
        _i,
        [_vp, _i, _i, _i, _i, _vp, _i, _vp, _vp, _vp, _vp, _vp, _i, _i, _i, _vp, _vp],
    ),
    "lmoe_down": (_i, [_vp, _i, _i, _vp, _i, _vp, _vp, _vp, _vp, _vp, _i, _i, _i, _vp, _vp]),
    "lmoe_decode_mlp_two_passes": (
        _i,
        [_vp, _i, _i, _i, _i, _vp, _vp, _i, _vp, _vp, _vp, _vp, _vp, _vp, _i, _vp, _vp, _vp, _i, _vp,
         _vp, _vp],
    ),
    "lmoe_stream_mlp_two_passes": (
        _i,
        [_vp, _i, _i, _i, _i, _vp, _vp, _i, _vp, _vp, _vp, _vp, _vp, _vp, _i, _vp, _vp, _vp, _vp, _i, _i,
         _vp, _vp, _vp],
    ),
    "lmoe_combine": (_i, [_vp, _vp, _vp, _i, _i, _i, _vp, _vp, _vp]),
    "lmoe_combine_f32": (_i, [_vp, _vp, _vp, _i, _i, _i, _vp, _vp, _vp]),
    "lmoe_add_rms_norm": (_i, [_vp, _i, _i, _vp, _i, _vp, _i, _f, _vp, _vp, _vp, _vp, _vp]),
    "lmoe_rows_to_mx8": (_i, [_vp, _i, _i, _vp, _vp, _vp]),
    "lmoe_mx4_bytes": (ctypes.c_longlong, [_i, _i]),
    "lmoe_mx4_gateup_silu": (
        _i,
        [_vp, _vp, _i, _i, _i, _i, _vp, _i, _vp, _vp, _vp, _vp, _vp, _i, _i, _i, _vp, _vp, _i, _vp],
    ),
    "lmoe_mx4_down": (
        _i,
        [_vp, _vp, _i, _i, _i, _vp, _i, _vp, _vp, _vp, _vp, _vp, _i, _i, _i, _vp, _i, _vp],
    ),
    "lmoe_mx4_fused_moe": (
        _i,
        [_vp, _vp, _i, _i, _i, _i, _vp, _vp, _i, _vp, _vp, _vp, _i, _i, _i, _vp, _vp, _vp, _vp],
    ),
    "lmoe_mx4_decode_few": (
        _i,
        [_vp, _vp, _i, _i, _i, _i, _vp, _vp, _i, _vp, _vp, _vp, _i, _vp, _vp, _vp, _vp, _vp, _vp],
    ),
    "lmoe_mx4_decode_one": (
        _i,
        [_vp, _vp, _i, _i, _i, _vp, _vp, _i, _vp, _vp, _vp, _i, _vp, _vp, _i, _vp, _i, _vp, _vp, _vp, _vp, _vp],
    ),
    "lmoe_fused_moe_decode": (
        _i,
        [_vp, _i, _i, _i, _i, _vp, _vp, _i, _vp, _vp, _vp, _vp, _vp, _vp, _vp, _vp, _vp, _vp,
         _i, _vp],
    ),
    "lmoe_fused_moe_decode_noalloc": (
        _i,
        [_vp, _i, _i, _i, _i, _vp, _vp, _i, _vp, _vp, _vp, _vp, _vp, _vp, _vp, _vp, _i, _vp],
    ),
    "lmoe_down_combine": (_i, [_vp, _i, _i, _i, _i, _vp, _i, _vp, _vp, _vp, _vp, _vp, _vp, _vp, _vp]),
    "lmoe_stage_copy": (_i, [_vp, _vp, _vp, _i, _vp, _vp, _vp]),
    "lmoe_stage_gather": (_i, [_vp, _vp, _vp, _i, _vp, _i, _vp, _vp, _i, _i, _vp, _vp, _vp]),
    "lmoe_slot_plan": (_i, [_vp, _vp, _vp, _vp, _i, _vp, _i, _vp, _i, ctypes.c_int64, _vp, _vp]),
    "lmoe_table_update": (_i, [_vp, _i, _vp, _vp, _i, _vp]),
    "lmoe_wave_plan_bytes": (ctypes.c_longlong, [_i, _i, _i]),
    "lmoe_wave_plan": (_i, [_vp, _i, _i, _i, _i, _i, _vp, _vp]),
    "lmoe_wave_stage": (
        _i,
        [_vp, _i, _i, _i, _i, _vp, _vp, _vp, _vp, _i, _vp, _vp, _vp, _vp, ctypes.c_longlong, ctypes.c_longlong,
         _vp, _i, _i, _i, _vp],
    ),
}

_LIB: ctypes.CDLL | None = None


class NativeLibraryMissing(RuntimeError):
    """liblatchmoe_hip.so is not built; there is no fallback path."""


def library_path() -> Path:
    override = os.environ.get("LATCHMOE_HIP_LIB")
    return Path(override) if override else LIB_PATH


def load_library() -> ctypes.CDLL:
    """Load (once) and return the HIP kernel library, raising if absent."""
    global _LIB
    if _LIB is not None:
        return _LIB
    path = library_path()
    if not path.exists():
        raise NativeLibraryMissing(
            f"{path} is missing: build it with "
            "`python vllm-ascend-hust-latchmoe_amd/build_native.py` "
            "(the slot-indexed MoE path has no CPU or PyTorch fallback)"
        )
    lib = ctypes.CDLL(str(path))
    for name, (restype, argtypes) in _SIGNATURES.items():
        fn = getattr(lib, name)
        fn.restype = restype
        fn.argtypes = argtypes
    _LIB = lib
    atexit.register(release_device_resources)
    return lib


def release_device_resources() -> dict:
    """Drop every device and page-locked buffer this package holds and
    return them to the HIP runtime while it is fully up: the workspace and
    constant caches, the runtime singleton (slot banks, stage banks, host
    store, events), then torch's device cache and its page-locked host cache.
    Registered with atexit when the library loads, so it runs at the start of
    interpreter shutdown: a page-locked block still cached there would be
    freed only by torch's allocator destructor during C++ static teardown,
    after tools attached to the runtime (a profiler's memory-copy tracing) may
    already have shut down.  Returns torch's host-allocator statistics after
    the release (empty when unavailable).  Safe to call more than once."""
    import gc

    from vllm_moe_offload_amd import fused_moe, layer
    from vllm_moe_offload_amd.moe_offload import runtime

    fused_moe.clear_workspaces()
    layer.clear_constants()
    runtime.reset_moe_offload_runtime()
    gc.collect()
    stats: dict = {}
    try:
        if torch.cuda.is_available() and torch.cuda.is_initialized():
            torch.cuda.synchronize()
            torch.cuda.empty_cache()
            empty_host = getattr(torch._C, "_host_emptyCache", None)
            if empty_host is not None:
                empty_host()
            host_stats = getattr(torch.cuda, "host_memory_stats", None)
            if host_stats is not None:
                stats = dict(host_stats())
    except RuntimeError:
        pass  # a device that already failed has nothing left to return
    return stats


def _check(status: int, fn: str) -> None:
    if status != 0:
        msg = load_library().lmoe_status_string(int(status))
        raise RuntimeError(f"{fn} failed with status {status}: {msg.decode()}")


def device_flags(*, clear: bool = True, stream=None) -> list[int]:
    """The current device's status words (lmoe_device_flags: pairs a masked
    combine dropped, one-launch router waits that gave up), summed over the
    library's kernels since the last clear.  Synchronizes the stream."""
    lib = load_library()
    buf = (ctypes.c_int32 * FLAG_COUNT)()
    _check(lib.lmoe_device_flags(ctypes.cast(buf, ctypes.c_void_p), int(bool(clear)), _stream(stream)),
           "lmoe_device_flags")
    return [int(v) for v in buf]


def _ptr(t: torch.Tensor | None) -> int | None:
    return None if t is None else int(t.data_ptr())


# The current stream's handle without a Stream object around it, where torch has
# the call (a few microseconds less of host time in every wrapper).
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)
_device_index = getattr(torch._C, "_cuda_getDevice", None) or torch.cuda.current_device


def _stream(stream: torch.cuda.Stream | None) -> int:
    if stream is None and _raw_stream is not None:
        return _raw_stream(_device_index())
    s = stream if stream is not None else torch.cuda.current_stream()
    return int(s.cuda_stream)


def current_stream_handle(device_index: int) -> int:
    """The raw handle of a device's current stream (0: the default stream)."""
    if _raw_stream is not None:
        return _raw_stream(device_index)
    return int(torch.cuda.current_stream(device_index).cuda_stream)


def _on(stream: torch.cuda.Stream | None):
    """Outputs that a call makes come from the pool of the stream that writes them:
    memory of the current stream's pool may still be in use by its queued work."""
    return contextlib.nullcontext() if stream is None else torch.cuda.stream(stream)


def _new(shape, dtype: torch.dtype, device, stream: torch.cuda.Stream | None) -> torch.Tensor:
    if stream is None:
        return torch.empty(shape, dtype=dtype, device=device)
    with _on(stream):
        return torch.empty(shape, dtype=dtype, device=device)


def _need(t: torch.Tensor, name: str, dtype: torch.dtype, shape: tuple | None = None) -> None:
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a tensor")
    if t.device.type != "cuda":
        raise ValueError(f"{name} must be a device tensor, got {t.device}")
    if t.dtype != dtype:
        raise ValueError(f"{name} must be {dtype}, got {t.dtype}")
    if not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous")
    if shape is not None and tuple(t.shape) != tuple(shape):
        raise ValueError(f"{name} has shape {tuple(t.shape)}, expected {tuple(shape)}")


# ---------------------------------------------------------------------------
# 8-bit rows and the norm in front of a MoE layer
# ---------------------------------------------------------------------------
@dataclass(frozen=True)
class Mx8Rows:
    """Rows in 8 bits: e4m3 values, one power-of-two scale per 32 columns
    (value[r, c] = q[r, c] * 2^(scale[r, c // 32] - 127); 255: NaN)."""

    q: torch.Tensor      # [R, K] float8_e4m3fn
    scale: torch.Tensor  # [R, K / 32] uint8

    @classmethod
    def allocate(cls, rows: int, columns: int, device) -> "Mx8Rows":
        if int(columns) <= 0 or int(columns) % mxfp4.GROUP:
            raise ValueError(f"8-bit rows are multiples of {mxfp4.GROUP} columns, got {columns}")
        return cls(torch.empty((int(rows), int(columns)), dtype=torch.float8_e4m3fn, device=device),
                   torch.empty((int(rows), int(columns) // mxfp4.GROUP), dtype=torch.uint8, device=device))

    @property
    def shape(self) -> torch.Size:
        return self.q.shape

    @property
    def device(self) -> torch.device:
        return self.q.device

    @property
    def dtype(self) -> torch.dtype:
        return self.q.dtype

    def __getitem__(self, rows: slice) -> "Mx8Rows":
        if not isinstance(rows, slice):
            raise TypeError("8-bit rows are sliced by rows")
        return Mx8Rows(self.q[rows], self.scale[rows])

    def float(self) -> torch.Tensor:
        """The f32 values that the rows stand for (checks and exports)."""
        s = mxfp4.scale_values(self.scale)
        return (self.q.float().unflatten(-1, (-1, mxfp4.GROUP)) * s.unsqueeze(-1)).flatten(-2)


def _is(t, dtype: torch.dtype, shape: tuple) -> bool:
    """What _need checks, without its words: for calls whose host time counts.
    (_need then says what is wrong.)"""
    return isinstance(t, torch.Tensor) and t.dtype is dtype and t.is_cuda and t.shape == shape and t.is_contiguous()


def _need_mx8(rows, name: str, shape: tuple | None = None) -> None:
    if not isinstance(rows, Mx8Rows):
        raise TypeError(f"{name} must be Mx8Rows")
    if shape is not None and _is(rows.q, torch.float8_e4m3fn, shape) and shape[1] % mxfp4.GROUP == 0 and \
            _is(rows.scale, torch.uint8, (shape[0], shape[1] // mxfp4.GROUP)):
        return
    _need(rows.q, f"{name}.q", torch.float8_e4m3fn, shape)
    if rows.q.dim() != 2 or rows.q.shape[1] % mxfp4.GROUP:
        raise ValueError(f"{name} must be [R, K], K a multiple of {mxfp4.GROUP}, got {tuple(rows.q.shape)}")
    _need(rows.scale, f"{name}.scale", torch.uint8, (rows.q.shape[0], rows.q.shape[1] // mxfp4.GROUP))


def _same_device(*tensors) -> None:
    """Every operand on the current device: a launch goes to its stream."""
    here = torch.cuda.current_device()
    for t in tensors:
        if t is not None and t.get_device() != here:
            raise ValueError(f"operand on {t.device}, the current device is cuda:{here}")


def _fits(t: torch.Tensor, dtype: torch.dtype, shape, here: int) -> bool:
    """_is on device here; _refuse says what is wrong."""
    return t.dtype is dtype and t.get_device() == here and t.shape == shape and t.is_contiguous()


def _take_mx8(rows, name: str, shape, here: int) -> tuple[torch.Tensor, torch.Tensor]:
    """(values, scales) of 8-bit rows [T, K] on device here."""
    q, scale = rows.q, rows.scale
    if not (shape[1] % 32 == 0 and _fits(q, torch.float8_e4m3fn, shape, here) and
            _fits(scale, torch.uint8, (shape[0], shape[1] // 32), here)):
        _need_mx8(rows, name, tuple(shape))
        _same_device(q, scale)
    return q, scale


def _refuse(t, name: str, dtype: torch.dtype, shape: tuple | None = None) -> None:
    _need(t, name, dtype, shape)
    _same_device(t)


def add_rms_norm(
    x: torch.Tensor,
    weight: torch.Tensor,
    *,
    residual: torch.Tensor | None = None,
    residual_out: torch.Tensor | None = None,
    out: torch.Tensor | None = None,
    mx8: Mx8Rows | None = None,
    eps: float = 1e-6,
    stream=None,
):
    """r = x + residual; y = r / sqrt(mean(r^2) + eps) * weight.

    y goes to out (bf16: the router gate, bf16 experts), to mx8 (4-bit experts'
    8-bit rows) or to both; with neither given a bf16 out is made.  r goes to
    residual_out, in place of residual if that is not given.  x [T, H] bf16,
    residual bf16 or f32, weight [H] bf16 or f32; r is kept in f32 between the
    sum and the outputs, the squares are summed in f32.  residual_out may be x,
    out may be x, or residual if residual_out is another buffer (where an f32
    residual is not one of them); outputs that overlap anything otherwise are
    refused.  H a multiple of 8 (of 32 with mx8) up to 32768.  Returns (out, mx8,
    residual_out), None for what was not asked for."""
    lib = load_library()
    bf16, f32 = torch.bfloat16, torch.float32
    if not isinstance(x, torch.Tensor) or x.dim() != 2:
        raise ValueError("x must be a [T, H] tensor")
    here = _device_index()
    shape = x.shape
    T, H = shape
    if not _fits(x, bf16, shape, here):
        _refuse(x, "x", bf16)
    wdt = f32 if weight.dtype is f32 else bf16
    if not _fits(weight, wdt, (H,), here):
        _refuse(weight, "weight", wdt, (H,))
    rdt = bf16
    if residual is not None:
        rdt = f32 if residual.dtype is f32 else bf16
        if not _fits(residual, rdt, shape, here):
            _refuse(residual, "residual", rdt, shape)
        if residual_out is None:
            residual_out = residual
        elif not _fits(residual_out, rdt, shape, here):
            _refuse(residual_out, "residual_out", rdt, shape)
    elif residual_out is not None:
        raise ValueError("residual_out needs a residual")
    if not eps >= 0.0:
        raise ValueError(f"eps must not be negative, got {eps}")
    if out is None and mx8 is None:
        out = _new(shape, bf16, x.device, stream)
    elif out is not None and not _fits(out, bf16, shape, here):
        _refuse(out, "out", bf16, shape)
    q = scale = None
    if mx8 is not None:
        if not isinstance(mx8, Mx8Rows):
            raise TypeError("mx8 must be Mx8Rows")
        q, scale = _take_mx8(mx8, "mx8", shape, here)
    px, po = x.data_ptr(), None if out is None else out.data_ptr()
    pr = pro = None
    if residual is not None:
        pr, pro = residual.data_ptr(), residual_out.data_ptr()
        if T:
            if po == pro:
                raise ValueError("out and residual_out must be two buffers")
            if rdt is f32 and (po == pr or pro == px):
                raise ValueError("rows of two types cannot share a buffer")
    status = lib.lmoe_add_rms_norm(px, T, H, pr, rdt is f32, weight.data_ptr(), wdt is f32, eps, pro, po, _ptr(q),
                                   _ptr(scale), _stream(stream))
    if status:
        _refuse_overlap(status, H)
        _check(status, "lmoe_add_rms_norm")
    return out, mx8, residual_out


def _refuse_overlap(status: int, H: int) -> None:
    """What LMOE_ERR_ARG means where the operands have been checked."""
    if status == LMOE_ERR_ARG and H > 0:
        raise ValueError("operands overlap: an output over another one, or over an input other than row for row")


def rows_to_mx8(x: torch.Tensor, mx8: Mx8Rows | None = None, *, stream=None) -> Mx8Rows:
    """bf16 rows x [T, H] in 8 bits (rows that were normed elsewhere)."""
    lib = load_library()
    _need(x, "x", torch.bfloat16)
    if x.dim() != 2:
        raise ValueError(f"x must be [T, H], got {tuple(x.shape)}")
    if mx8 is None:
        with _on(stream):
            mx8 = Mx8Rows.allocate(x.shape[0], x.shape[1], x.device)
    _need_mx8(mx8, "mx8", tuple(x.shape))
    _same_device(x, mx8.q, mx8.scale)
    status = lib.lmoe_rows_to_mx8(_ptr(x), x.shape[0], x.shape[1], _ptr(mx8.q), _ptr(mx8.scale), _stream(stream))
    _refuse_overlap(status, x.shape[1])
    _check(status, "lmoe_rows_to_mx8")
    return mx8


# ---------------------------------------------------------------------------
# router
# ---------------------------------------------------------------------------
def _check_biases(bias: torch.Tensor | None, logit_bias: torch.Tensor | None, E: int) -> None:
    if bias is not None:
        _need(bias, "e_score_correction_bias", torch.float32, (E,))
    if logit_bias is not None:
        _need(logit_bias, "logit_bias", torch.float32, (E,))


def router_gate(x: torch.Tensor, wg: torch.Tensor, logits: torch.Tensor, *, stream=None) -> torch.Tensor:
    """logits = x . wg^T with f32 accumulation (bf16 or f32 output)."""
    lib = load_library()
    T, H = x.shape
    E = wg.shape[0]
    _need(x, "x", torch.bfloat16)
    _need(wg, "wg", torch.bfloat16, (E, H))
    if logits.dtype not in (torch.bfloat16, torch.float32):
        raise ValueError("logits must be bf16 or f32")
    _need(logits, "logits", logits.dtype, (T, E))
    _check(
        lib.lmoe_router_gate(_ptr(x), _ptr(wg), T, H, E, _ptr(logits),
                             int(logits.dtype == torch.float32), _stream(stream)),
        "lmoe_router_gate",
    )
    return logits


def router_topk(
    logits: torch.Tensor,
    top_k: int,
    *,
    scoring: str = "softmax",
    bias: torch.Tensor | None = None,
    logit_bias: torch.Tensor | None = None,
    num_expert_group: int = 1,
    topk_group: int = 1,
    renormalize: bool = True,
    routed_scaling_factor: float = 1.0,
    n_shared: int = 0,
    w_bf16: torch.Tensor | None = None,
    ids: torch.Tensor | None = None,
    w_f32: torch.Tensor | None = None,
    stream=None,
) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor | None]:
    """Select top_k experts per token (bias: e_score_correction_bias, for
    selection only; logit_bias: added to the logits before scoring).
    Returns (w_bf16 [T,k+S], ids int32 [T,k+S], w_f32) with S = n_shared
    columns of the pinned shared-expert suffix (ids E, E+1, ..., weight 1)
    after the routed ones."""
    lib = load_library()
    if logits.dtype not in (torch.bfloat16, torch.float32):
        raise ValueError("logits must be bf16 or f32")
    _need(logits, "logits", logits.dtype)
    T, E = logits.shape
    if scoring == "softmax":
        mode = LMOE_SCORING_SOFTMAX
    elif scoring == "sigmoid":
        mode = LMOE_SCORING_SIGMOID
    else:
        raise ValueError(f"unsupported scoring function {scoring!r}")
    _check_biases(bias, logit_bias, E)
    dev = logits.device
    kw = int(top_k) + int(n_shared)
    if w_bf16 is None:
        w_bf16 = _new((T, kw), torch.bfloat16, dev, stream)
    if ids is None:
        ids = _new((T, kw), torch.int32, dev, stream)
    _need(w_bf16, "topk_weights", torch.bfloat16, (T, kw))
    _need(ids, "topk_ids", torch.int32, (T, kw))
    if w_f32 is not None:
        _need(w_f32, "w_f32", torch.float32, (T, kw))
    _check(
        lib.lmoe_router_topk(
            _ptr(logits), int(logits.dtype == torch.float32), T, E, int(top_k), int(n_shared), mode,
            _ptr(bias), _ptr(logit_bias), int(num_expert_group or 1), int(topk_group or 1),
            int(bool(renormalize)), float(routed_scaling_factor),
            _ptr(w_f32), _ptr(w_bf16), _ptr(ids), _stream(stream),
        ),
        "lmoe_router_topk",
    )
    return w_bf16, ids, w_f32


def router_topk_permute(
    logits: torch.Tensor,
    top_k: int,
    perm: "Permutation",
    *,
    log2phy: torch.Tensor | None = None,
    skip_unmapped: bool = False,
    block_m: int | None = None,
    scoring: str = "softmax",
    bias: torch.Tensor | None = None,
    logit_bias: torch.Tensor | None = None,
    num_expert_group: int = 1,
    topk_group: int = 1,
    renormalize: bool = True,
    routed_scaling_factor: float = 1.0,
    n_shared: int = 0,
    w_bf16: torch.Tensor | None = None,
    ids: torch.Tensor | None = None,
    w_f32: torch.Tensor | None = None,
    second: "tuple[Permutation, torch.Tensor] | None" = None,
    stream=None,
) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor | None]:
    """router_topk then permute into perm, in one launch when the shape allows
    it (T <= 16, E <= 256); otherwise the two launches.  For a slot table
    (log2phy) that is final before the router runs.  second = (permutation,
    table) of a later pass over the same ids (the decode overflow stage
    buffer; perm is then built with skip_unmapped): built after perm in skip
    mode 2 on perm.row_idx, in the same launch as perm when the selection
    runs on its own (permute_two_tables)."""
    lib = load_library()
    if logits.dtype not in (torch.bfloat16, torch.float32):
        raise ValueError("logits must be bf16 or f32")
    _need(logits, "logits", logits.dtype)
    T, E = logits.shape
    mode = {"softmax": LMOE_SCORING_SOFTMAX, "sigmoid": LMOE_SCORING_SIGMOID}.get(scoring)
    if mode is None:
        raise ValueError(f"unsupported scoring function {scoring!r}")
    _check_biases(bias, logit_bias, E)
    dev = logits.device
    kw = int(top_k) + int(n_shared)
    if w_bf16 is None:
        w_bf16 = _new((T, kw), torch.bfloat16, dev, stream)
    if ids is None:
        ids = _new((T, kw), torch.int32, dev, stream)
    _need(w_bf16, "topk_weights", torch.bfloat16, (T, kw))
    _need(ids, "topk_ids", torch.int32, (T, kw))
    if w_f32 is not None:
        _need(w_f32, "w_f32", torch.float32, (T, kw))
    if T * kw != perm.n_pairs:
        raise ValueError(f"permutation buffers sized for {perm.n_pairs} pairs, got {T * kw}")
    n_table = 0
    if log2phy is not None:
        _need(log2phy, "log2phy", torch.int32)
        n_table = int(log2phy.numel())
    if second is not None and (log2phy is None or not skip_unmapped):
        raise ValueError("a second pass needs the first pass's table with skip_unmapped")
    bm = MFMA_BLOCK_M if block_m is None else int(block_m)
    status = lib.lmoe_router_topk_permute(
        _ptr(logits), int(logits.dtype == torch.float32), T, E, int(top_k), int(n_shared), mode,
        _ptr(bias), _ptr(logit_bias), int(num_expert_group or 1), int(topk_group or 1),
        int(bool(renormalize)), float(routed_scaling_factor),
        _ptr(w_f32), _ptr(w_bf16), _ptr(ids),
        _ptr(log2phy), n_table, perm.n_slots, int(bool(skip_unmapped)), bm,
        _ptr(perm.counts), _ptr(perm.offsets), _ptr(perm.sorted_pairs), _ptr(perm.row_idx),
        _ptr(perm.active), _ptr(perm.tile_off), _ptr(perm.meta), _stream(stream),
    )
    if status == LMOE_ERR_SHAPE:
        router_topk(logits, top_k, scoring=scoring, bias=bias, logit_bias=logit_bias,
                    num_expert_group=num_expert_group,
                    topk_group=topk_group, renormalize=renormalize,
                    routed_scaling_factor=routed_scaling_factor, n_shared=n_shared, w_bf16=w_bf16, ids=ids,
                    w_f32=w_f32, stream=stream)
        if second is not None:
            permute_two_tables(ids, perm, log2phy, second[0], second[1], block_m=bm, stream=stream)
        else:
            permute(ids, perm, log2phy=log2phy, skip_unmapped=skip_unmapped, block_m=bm, stream=stream)
        return w_bf16, ids, w_f32
    _check(status, "lmoe_router_topk_permute")
    perm.builds += 1
    perm.block_m = bm
    if second is not None:
        permute(ids, second[0], log2phy=second[1], keep_rows=True, row_idx=perm.row_idx, block_m=bm,
                stream=stream)
    return w_bf16, ids, w_f32


def router_gate_topk_permute(
    x: torch.Tensor,
    wg: torch.Tensor,
    logits: torch.Tensor,
    top_k: int,
    perm: "Permutation",
    *,
    log2phy: torch.Tensor | None = None,
    skip_unmapped: bool = False,
    block_m: int | None = None,
    scoring: str = "softmax",
    bias: torch.Tensor | None = None,
    logit_bias: torch.Tensor | None = None,
    num_expert_group: int = 1,
    topk_group: int = 1,
    renormalize: bool = True,
    routed_scaling_factor: float = 1.0,
    n_shared: int = 0,
    w_bf16: torch.Tensor | None = None,
    ids: torch.Tensor | None = None,
    w_f32: torch.Tensor | None = None,
    stream=None,
) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor | None]:
    """router_gate, router_topk and permute into perm in one launch when the
    shape allows it (T <= 16, E <= 256, H <= 8192); otherwise router_gate and
    router_topk_permute.  Same outputs bit for bit; logits is written too.
    Uses perm.sync (arrival count and tagged logit words): calls that may run concurrently
    need separate Permutation buffers."""
    lib = load_library()
    T, H = x.shape
    E = wg.shape[0]
    _need(x, "x", torch.bfloat16)
    _need(wg, "wg", torch.bfloat16, (E, H))
    if logits.dtype not in (torch.bfloat16, torch.float32):
        raise ValueError("logits must be bf16 or f32")
    _need(logits, "logits", logits.dtype, (T, E))
    mode = {"softmax": LMOE_SCORING_SOFTMAX, "sigmoid": LMOE_SCORING_SIGMOID}.get(scoring)
    if mode is None:
        raise ValueError(f"unsupported scoring function {scoring!r}")
    _check_biases(bias, logit_bias, E)
    dev = x.device
    kw = int(top_k) + int(n_shared)
    if w_bf16 is None:
        w_bf16 = _new((T, kw), torch.bfloat16, dev, stream)
    if ids is None:
        ids = _new((T, kw), torch.int32, dev, stream)
    _need(w_bf16, "topk_weights", torch.bfloat16, (T, kw))
    _need(ids, "topk_ids", torch.int32, (T, kw))
    if w_f32 is not None:
        _need(w_f32, "w_f32", torch.float32, (T, kw))
    if T * kw != perm.n_pairs:
        raise ValueError(f"permutation buffers sized for {perm.n_pairs} pairs, got {T * kw}")
    n_table = 0
    if log2phy is not None:
        _need(log2phy, "log2phy", torch.int32)
        n_table = int(log2phy.numel())
    bm = MFMA_BLOCK_M if block_m is None else int(block_m)
    status = lib.lmoe_router_gate_topk_permute(
        _ptr(x), _ptr(wg), T, H, E, _ptr(logits), int(logits.dtype == torch.float32), int(top_k),
        int(n_shared), mode, _ptr(bias), _ptr(logit_bias), int(num_expert_group or 1),
        int(topk_group or 1),
        int(bool(renormalize)), float(routed_scaling_factor),
        _ptr(w_f32), _ptr(w_bf16), _ptr(ids),
        _ptr(log2phy), n_table, perm.n_slots, int(bool(skip_unmapped)), bm,
        _ptr(perm.counts), _ptr(perm.offsets), _ptr(perm.sorted_pairs), _ptr(perm.row_idx),
        _ptr(perm.active), _ptr(perm.tile_off), _ptr(perm.meta), _ptr(perm.sync), _stream(stream),
    )
    if status == LMOE_ERR_SHAPE:
        router_gate(x, wg, logits, stream=stream)
        return router_topk_permute(
            logits, top_k, perm, log2phy=log2phy, skip_unmapped=skip_unmapped, block_m=bm,
            scoring=scoring, bias=bias, logit_bias=logit_bias, num_expert_group=num_expert_group,
            topk_group=topk_group,
            renormalize=renormalize, routed_scaling_factor=routed_scaling_factor, n_shared=n_shared,
            w_bf16=w_bf16, ids=ids, w_f32=w_f32, stream=stream,
        )
    _check(status, "lmoe_router_gate_topk_permute")
    perm.builds += 1
    perm.block_m = bm
    return w_bf16, ids, w_f32


def router_gate_topk_pairs(
    x: torch.Tensor,
    wg: torch.Tensor,
    logits: torch.Tensor,
    top_k: int,
    perm: "Permutation",
    *,
    log2phy: torch.Tensor | None = None,
    skip_unmapped: bool = False,
    scoring: str = "softmax",
    bias: torch.Tensor | None = None,
    logit_bias: torch.Tensor | None = None,
    num_expert_group: int = 1,
    topk_group: int = 1,
    renormalize: bool = True,
    routed_scaling_factor: float = 1.0,
    n_shared: int = 0,
    w_bf16: torch.Tensor | None = None,
    ids: torch.Tensor | None = None,
    w_f32: torch.Tensor | None = None,
    stream=None,
) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor | None]:
    """One token: router_gate_topk_permute's gate and selection (the same
    bits) with perm in the one-token pair order (lmoe_router_gate_topk_pairs:
    the placed pairs at positions 0, 1, ... in pair order, active[pos] their
    slots; counts, offsets and tile_off are not written), the form
    fused_moe_decode(distinct_slots=True) reads.  Falls back to
    router_gate_topk_permute (the sorted permutation, which that call reads
    the same way) where the one launch does not take the shape."""
    lib = load_library()
    T, H = x.shape
    E = wg.shape[0]
    if T != 1:
        raise ValueError("the pair-order router serves one token")
    _need(x, "x", torch.bfloat16)
    _need(wg, "wg", torch.bfloat16, (E, H))
    if logits.dtype not in (torch.bfloat16, torch.float32):
        raise ValueError("logits must be bf16 or f32")
    _need(logits, "logits", logits.dtype, (T, E))
    mode = {"softmax": LMOE_SCORING_SOFTMAX, "sigmoid": LMOE_SCORING_SIGMOID}.get(scoring)
    if mode is None:
        raise ValueError(f"unsupported scoring function {scoring!r}")
    _check_biases(bias, logit_bias, E)
    dev = x.device
    kw = int(top_k) + int(n_shared)
    if w_bf16 is None:
        w_bf16 = _new((T, kw), torch.bfloat16, dev, stream)
    if ids is None:
        ids = _new((T, kw), torch.int32, dev, stream)
    _need(w_bf16, "topk_weights", torch.bfloat16, (T, kw))
    _need(ids, "topk_ids", torch.int32, (T, kw))
    if w_f32 is not None:
        _need(w_f32, "w_f32", torch.float32, (T, kw))
    if kw != perm.n_pairs:
        raise ValueError(f"permutation buffers sized for {perm.n_pairs} pairs, got {kw}")
    n_table = 0
    if log2phy is not None:
        _need(log2phy, "log2phy", torch.int32)
        n_table = int(log2phy.numel())
    status = lib.lmoe_router_gate_topk_pairs(
        _ptr(x), _ptr(wg), H, E, _ptr(logits), int(logits.dtype == torch.float32), int(top_k),
        int(n_shared), mode, _ptr(bias), _ptr(logit_bias), int(num_expert_group or 1), int(topk_group or 1),
        int(bool(renormalize)), float(routed_scaling_factor), _ptr(w_f32), _ptr(w_bf16), _ptr(ids),
        _ptr(log2phy), n_table, perm.n_slots, int(bool(skip_unmapped)),
        _ptr(perm.sorted_pairs), _ptr(perm.row_idx), _ptr(perm.active), _ptr(perm.meta), _ptr(perm.sync),
        _stream(stream),
    )
    if status == LMOE_ERR_SHAPE:
        return router_gate_topk_permute(
            x, wg, logits, top_k, perm, log2phy=log2phy, skip_unmapped=skip_unmapped, scoring=scoring,
            bias=bias, logit_bias=logit_bias, num_expert_group=num_expert_group, topk_group=topk_group,
            renormalize=renormalize, routed_scaling_factor=routed_scaling_factor, n_shared=n_shared,
            w_bf16=w_bf16, ids=ids, w_f32=w_f32, stream=stream,
        )
    _check(status, "lmoe_router_gate_topk_pairs")
    perm.builds += 1
    return w_bf16, ids, w_f32


# ---------------------------------------------------------------------------
# permutation
# ---------------------------------------------------------------------------
_CU_COUNT: dict[int, int] = {}


def _cu_count(device) -> int:
    idx = torch.device(device).index
    idx = torch.cuda.current_device() if idx is None else idx
    if idx not in _CU_COUNT:
        _CU_COUNT[idx] = int(torch.cuda.get_device_properties(idx).multi_processor_count)
    return _CU_COUNT[idx]


_OFFSET32_LIMIT = 2**31 - 1


# The decode GEMVs take a layer of up to this many tokens, and past it one of
# few pairs per expert; the rest goes to the weight-streaming MFMA kernel.  A
# GEMV pays ~70 vector instructions per row pair and token, the MFMA kernel has
# fewer bytes in flight per wave and a longer chain before its first weight
# load, so the line lies at a number of pairs per expert, higher where the
# GEMVs' rows fill the chunks that they are compiled for (GEMV_WHOLE_HIDDEN,
# GEMV_WHOLE_INTERMEDIATE).  A layer's experts, GEMV / streaming, us, every
# expert as likely (H, I, experts, top k):
#   2048, 768, 128, 8     33 tokens 166 / 176, 40: 177 / 184, 44: 182 / 183, 64: 212 / 195
#   2048, 768, 128, 4     33: 130 / 141, 64: 165 / 177, 80: 178 / 184
#   2048, 1024, 128, 8    33: 220 / 239, 44: 243 / 247, 48: 248 / 250, 56: 265 / 255
#   2048, 512, 256, 8     33: 166 / 183, 64: 224 / 238, 80: 246 / 253
#   1024, 512, 128, 8     33: 67 / 74, 44: 71 / 76, 56: 77 / 78
#   4096, 768, 128, 8     33: 326 / 340, 40: 352 / 351, 48: 372 / 356
#   2048, 1408, 60, 4     28: 143 / 143, 33: 151 / 149, 48: 174 / 162
#   2048, 1408, 160, 4    33: 243 / 259, 64: 329 / 344
#   4096, 1536, 64, 4     33: 333 / 345, 40: 347 / 347, 64: 417 / 363
#   5120, 1536, 256, 8    33: 1138 / 1131, 64: 1609 / 1527
#   7168, 2048, 257, 9    8 tokens 712 / 718, 32: 2115 / 2099, 110: 3566 / 3134
# Skewed routing has fewer experts at work and moves the line down, but is not
# known when the layer is launched: with the Zipf(1.1) rank bias the first of
# these takes 107 / 100 at 33 tokens (whole step) and 128 / 109 at 44.
DECODE_GEMV_MAX_TOKENS = 32
GEMV_MAX_PAIRS_PER_EXPERT = 2.1
GEMV_MAX_PAIRS_PER_EXPERT_WHOLE = 2.75
GEMV_WHOLE_HIDDEN = (1024, 2048, 4096)
GEMV_WHOLE_INTERMEDIATE = (512, 768, 1024, 2048, 4096)
# Most pairs per slot, on average, of a pass on STREAM_BLOCK_M-row tiles: past
# one tile per slot the second one costs as much as the wider tiles do.  A
# layer's experts, streaming / 320-row tiles, us (tokens, pairs per slot):
#   Qwen3 shape   no rank bias  300 (19) 211 / 242, 1024 (64) 254 / 271, 1200 (75) 270 / 278, 1300 (81) 302 / 281
#                 half of it    300 228 / 260, 800 (50) 262 / 321, 1200 307 / 348, 1300 329 / 351
#                 Zipf(1.1)     300 216 / 287, 600 (38) 245 / 287, 1200 316 / 362
#   Qwen1.5-MoE   no rank bias  300 (20) 195 / 217, 800 (53) 212 / 234, 1100 (73) 244 / 243
#                 half of it    400 (27) 207 / 257, 800 252 / 269, 1100 281 / 288
#                 Zipf(1.1)     800 259 / 284, 1100 294 / 301
#   DeepSeek-V3   no rank bias  700 (25) 3522 / 3997, 1024 (36) 3803 / 4241, 2048 (72) 4331 / 4761
#                 half of it    1100 (39) 4048 / 4399, 2048 4772 / 4737
#                 Zipf(1.1)     1100 4018 / 4262, 2048 4867 / 5033
# The average is all that the host knows.  Where the routing leaves most slots
# without a pair the others hold more than it says and the wide tiles would be
# faster: 1100 tokens of the Qwen3 shape on 32 of its 128 experts (275 pairs
# each) 199 / 138, on 64 of them 252 / 205; 600 tokens on 32 125 / 112.
STREAM_MAX_PAIRS_PER_SLOT = 75


def aligned16(*tensors: torch.Tensor) -> bool:
    """Whether every tensor starts on a 16-byte boundary."""
    return all(t.data_ptr() % 16 == 0 for t in tensors)


def layer_path(tokens: int, top_k: int, hidden: int, intermediate: int, n_experts: int | None = None, *,
               aligned: bool = True) -> int:
    """The MLP path of a layer of `tokens` tokens with top_k pairs each over
    n_experts experts (all of the layer's, also where a pass holds fewer): the
    decode GEMVs for a few tokens or few pairs per expert, the streaming MFMA kernel with partial sums
    (LMOE_PATH_STREAM, accumulation as accurate as the GEMVs') up to
    FUSED_DECODE_MAX_PAIRS pairs, the MFMA kernels past that.  The paths round
    differently, so the choice depends on nothing that changes when a layer is
    split into passes (slots, waves, routing).  The streaming kernel needs
    hidden % 64 == 0 and hidden states and gate-up weights that start on 16-byte
    boundaries (aligned); without them the GEMVs serve all of their range."""
    if tokens * top_k > FUSED_DECODE_MAX_PAIRS or intermediate > GEMV_MAX_I:
        return LMOE_PATH_MFMA
    if tokens <= DECODE_GEMV_MAX_TOKENS or hidden % 64 != 0 or not aligned:
        return LMOE_PATH_GEMV
    if n_experts is not None and hidden in GEMV_WHOLE_HIDDEN:
        most = GEMV_MAX_PAIRS_PER_EXPERT_WHOLE if intermediate in GEMV_WHOLE_INTERMEDIATE else GEMV_MAX_PAIRS_PER_EXPERT
        if tokens * top_k < most * n_experts:
            return LMOE_PATH_GEMV
    return LMOE_PATH_STREAM


def prefill_block_m(n_experts: int, hidden: int, intermediate: int, device="cuda",
                    cu_count: int | None = None, n_pairs: int | None = None,
                    pass_pairs: int | None = None) -> int:
    """Row-tile height for the prefill GEMMs of one pass over n_experts slots
    (the block_m to build the permutation with).  n_pairs is the layer's pair
    count, pass_pairs the pass's own where that is one wave of the layer.

    STREAM_BLOCK_M selects the weight-streaming kernel, for passes of few pairs
    per slot (pass_pairs over n_experts, when n_pairs is given).

    320 selects the kernel with one workgroup per CU: a slot of up to 320
    pairs is one row tile, and each CU runs an equal number of units (a row
    tile's 128 gate-up columns).  With n_experts * ceil(I / 128) units it
    takes one round when they fit on the CUs, and balanced rounds when there
    are many.  Just past one round (a 43-slot wave on 256 CUs: 258 units) the
    last units would run alone, and the 256-row tile grid finishes first
    (measured 136 + 64 us against 166 + 74 us for gate_up + down); there 256
    is returned.  Needs hidden % 64 == 0 (else 256), and activation operands
    below 2^31 elements (the 320-row kernel's offsets are 32-bit: n_pairs
    rows of max(hidden, intermediate) bounds both GEMMs; else 256, whose
    offsets are 64-bit).  cu_count defaults to the device's."""
    if hidden % 64 != 0:
        return MFMA_BLOCK_M
    if n_pairs is not None and int(n_pairs) * max(int(hidden), int(intermediate)) > _OFFSET32_LIMIT:
        return MFMA_BLOCK_M
    if n_pairs is not None:
        if int(n_pairs if pass_pairs is None else pass_pairs) <= STREAM_MAX_PAIRS_PER_SLOT * int(n_experts):
            return STREAM_BLOCK_M
    cus = int(cu_count) if cu_count is not None else _cu_count(device)
    units = int(n_experts) * ((int(intermediate) + 127) // 128)
    if cus < units <= cus + cus // 4:
        return MFMA_BLOCK_M
    return PART_BLOCK_M


MX4_BLOCK_M = (32, 64, 128)  # row-tile heights of the 4-bit experts' prefill kernel
# Up to this many pairs per expert the split-K kernel, row tiles past it: bf16 rows, 8-bit
# rows.  Time of the captured layer, split-K over 32-row tiles (H, I, experts, top k):
#   pairs per expert     3           4           6           8
#   2048, 768, 128, 8    .98; .96    1.02; .98   1.13; 1.04
#   2048, 1408, 60, 4    .96; .93    .95; .93    1.07; .95   1.18; 1.00
#   4096, 1024, 16, 2                .83; .82    .88; .83    1.07; 1.02
#   2048, 512, 16, 2                 .86; .89    .90; .89    1.08; 1.09
#   7168, 2048, 32, 8    1.02; 1.00  1.02; .98   .99; .99    1.07; 1.01
#   4096, 2048, 64, 4    .94; .90    .97; .90    1.12; 1.00  1.18; .98
#   1024, 512, 64, 4     1.03; .97   1.08; .99   1.26; 1.13
# One number for each kind of rows is a compromise: of bf16 rows it costs 8% at 4 pairs
# (1024 x 512 x 64) and 12% at 6 (4096 x 1024 x 16), of 8-bit rows 13% at 6 (1024 x 512).
MX4_FEW_PAIRS_PER_EXPERT = 4
MX4_FEW_PAIRS_PER_EXPERT_MX8 = 6


# The longest 8-bit rows of a tile of each height: the tile keeps all their scales in LDS
# (160 KiB, less two stages of rows and the pairs).  The split-K kernel takes any.
MX4_MAX_COLUMNS_MX8 = {32: 147200, 64: 73600, 128: 32640}


def mx4_path(n_pairs: int, n_experts: int, mx8: bool = False, columns: int = 0) -> int:
    """The path of a layer of 4-bit experts, for every pass of it: the split-K
    kernel for few pairs per expert (mx8: of 8-bit rows) and for 8-bit rows too
    long for any row tile (columns: the longer of x's and act's), row tiles past that."""
    few = MX4_FEW_PAIRS_PER_EXPERT_MX8 if mx8 else MX4_FEW_PAIRS_PER_EXPERT
    if n_pairs <= few * n_experts or (mx8 and columns > MX4_MAX_COLUMNS_MX8[MX4_BLOCK_M[0]]):
        return LMOE_PATH_GEMV
    return LMOE_PATH_MFMA


# Row-tile heights but the last, with the most pairs per slot, on average, and the most
# gate-up workgroups (tiles of that height by 128 columns) that each is used up to: the
# shorter tiles, while they do not fill the card.  us of the captured layer, 32 / 64 / 128
# rows (bf16 rows; 8-bit rows; workgroups at 32 rows):
#   4096, 1024, 8, 2     48 pairs per slot  48 / 65 / 96;  42 / 49 / 64 (160)
#                        192                75 / 76 / 104; 59 / 64 / 70 (448)
#   2048, 1024, 16, 2    96                 50 / 57 / 73;  44 / 47 / 52 (512)
#                        192                72 / 69 / 77;  59 / 54 / 55 (896)
#   4096, 1408, 16, 4    48                 73 / 78 / 105; 70 / 71 / 76 (440)
#                        96                 97 / 98 / 117; 87 / 80 / 83 (704)
#   2048, 768, 32, 4     48                 52 / 56 / 72;  50 / 51 / 55 (480)
#   1024, 512, 64, 4     48                 43 / 47 / 57;  40 / 40 / 46 (640)
# and, gate-up and down alone,
#   2048, 768, 128, 8    25                 80 / 82 / 99;    76 / 78 / 81
#                        64                 126 / 116 / 136; 109 / 95 / 96
#                        100                170 / 148 / 169; 144 / 117 / 115
#                        256                380 / 321 / 311; 290 / 254 / 209
#   7168, 2048, 32, 8    50                 225 / 183 / 203 (8-bit rows)
#                        100                325 / 262 / 247
MX4_HEIGHTS = ((32, 32, 640), (64, 100, 1024))


def mx4_block_m(n_pairs: int, n_experts: int, intermediate: int = 1024, mx8_columns: int = 0) -> int:
    """Row-tile height of 4-bit experts' products (the permutation's block_m) for
    n_pairs pairs over n_experts slots of experts intermediate wide.  mx8_columns:
    the longer of x's and act's rows, where they are in 8 bits."""
    best = MX4_BLOCK_M[-1]
    for bm, pairs, groups in MX4_HEIGHTS:
        if n_pairs <= pairs * n_experts or (n_pairs // bm + n_experts) * -(-intermediate // 128) <= groups:
            best = bm
            break
    while mx8_columns > MX4_MAX_COLUMNS_MX8[best] and best > MX4_BLOCK_M[0]:
        best //= 2
    return best


@dataclass
class Permutation:
    """Device outputs of lmoe_permute for one (n_pairs, n_slots) shape.

    Buffers are allocated once and reused (fixed addresses, graph safe).
    """

    n_pairs: int
    n_slots: int
    counts: torch.Tensor        # [P] i32 histogram (expert_tokens, count type)
    offsets: torch.Tensor       # [P+1] i32
    sorted_pairs: torch.Tensor  # [N] i32 flat pair at each sorted position
    row_idx: torch.Tensor       # [N] i32 sorted position of each pair (expanded_row_idx) or -1
    active: torch.Tensor        # [P] i32 slots with count > 0: heavy slots first (by count), then ascending
    tile_off: torch.Tensor      # [P+1] i32 MFMA tile prefix
    meta: torch.Tensor          # [4] i32
    workspace: torch.Tensor     # int8 scratch for the multi-block path
    sync: torch.Tensor          # [ROUTER_SYNC_WORDS] i32: the one-launch router's arrival count (kept at 0) and tagged logit words
    block_m: int = MFMA_BLOCK_M  # tile height tile_off was last built with
    builds: int = 0  # lmoe_permute builds issued on these buffers

    @classmethod
    def allocate(cls, n_pairs: int, n_slots: int, device, *, cleared: bool = True) -> "Permutation":
        """cleared: the buffers start as zeros, as the router calls that build the
        permutation need; lmoe_permute does not."""
        lib = load_library()
        new = torch.zeros if cleared else torch.empty
        ws = int(lib.lmoe_permute_workspace_bytes(int(n_pairs), int(n_slots)))
        i32 = dict(dtype=torch.int32, device=device)
        return cls(
            n_pairs=int(n_pairs),
            n_slots=int(n_slots),
            counts=new(n_slots, **i32),
            offsets=new(n_slots + 1, **i32),
            sorted_pairs=new(max(1, n_pairs), **i32),
            row_idx=new(max(1, n_pairs), **i32),
            active=new(n_slots, **i32),
            tile_off=new(n_slots + 1, **i32),
            meta=new(META_COUNT, **i32),
            workspace=torch.empty(max(ws, 1), dtype=torch.int8, device=device),
            sync=new(ROUTER_SYNC_WORDS, **i32),
        )


def permute(
    ids: torch.Tensor,
    perm: Permutation,
    *,
    log2phy: torch.Tensor | None = None,
    skip_unmapped: bool = False,
    keep_rows: bool = False,
    row_idx: torch.Tensor | None = None,
    table_len: int | None = None,
    block_m: int = MFMA_BLOCK_M,
    stream=None,
) -> Permutation:
    """Remap ids through log2phy and stable-sort the flat pairs by slot.

    table_len (<= log2phy.numel()) limits the ids the table covers; with
    skip_unmapped, ids past it are left to another pass.  keep_rows (a later
    pass of a multi-pass layer; implies skip_unmapped) leaves the row_idx of
    the pairs this pass does not place as an earlier pass wrote it, so the
    layer's single combine masks exactly the pairs no pass placed.  row_idx
    replaces perm.row_idx as the output (the first pass's permutation when
    the passes build separate permutations)."""
    lib = load_library()
    if not _is(ids, torch.int32, getattr(ids, "shape", ())):
        _need(ids, "topk_ids", torch.int32)
    n = ids.numel()
    if n != perm.n_pairs:
        raise ValueError(f"permutation buffers sized for {perm.n_pairs} pairs, got {n}")
    rows = perm.row_idx if row_idx is None else row_idx
    if row_idx is not None:
        _need(row_idx, "row_idx", torch.int32)
        if int(row_idx.numel()) < max(1, n):
            raise ValueError("row_idx has fewer entries than pairs")
    mode = SKIP_KEEP_ROWS if keep_rows else int(bool(skip_unmapped))
    n_table = 0
    if log2phy is not None:
        _need(log2phy, "log2phy", torch.int32)
        n_table = int(log2phy.numel()) if table_len is None else min(int(table_len), int(log2phy.numel()))
    _check(
        lib.lmoe_permute(
            ids.data_ptr(), n, _ptr(log2phy), n_table,
            perm.n_slots, mode, int(block_m),
            perm.counts.data_ptr(), perm.offsets.data_ptr(), perm.sorted_pairs.data_ptr(),
            rows.data_ptr(), perm.active.data_ptr(), perm.tile_off.data_ptr(), perm.meta.data_ptr(),
            perm.workspace.data_ptr(), perm.workspace.numel(), _stream(stream),
        ),
        "lmoe_permute",
    )
    perm.block_m = int(block_m)
    perm.builds += 1
    return perm


def permute_two_tables(
    ids: torch.Tensor,
    perm: Permutation,
    log2phy: torch.Tensor,
    second: Permutation,
    second_log2phy: torch.Tensor,
    *,
    block_m: int = MFMA_BLOCK_M,
    stream=None,
) -> tuple[Permutation, Permutation]:
    """permute(ids, perm, log2phy, skip_unmapped=True) followed by
    permute(ids, second, second_log2phy, keep_rows=True, row_idx=perm.row_idx)
    (the bank and overflow-table builds of a decode overflow layer), in one
    launch up to PERMUTE_TWO_MAX_PAIRS pairs, as the two calls past that."""
    lib = load_library()
    _need(ids, "topk_ids", torch.int32)
    _need(log2phy, "log2phy", torch.int32)
    _need(second_log2phy, "second_log2phy", torch.int32)
    n = int(ids.numel())
    if n != perm.n_pairs or n != second.n_pairs:
        raise ValueError(f"permutation buffers sized for {perm.n_pairs} / {second.n_pairs} pairs, got {n}")
    if n > PERMUTE_TWO_MAX_PAIRS:
        permute(ids, perm, log2phy=log2phy, skip_unmapped=True, block_m=block_m, stream=stream)
        permute(ids, second, log2phy=second_log2phy, keep_rows=True, row_idx=perm.row_idx, block_m=block_m,
                stream=stream)
        return perm, second
    _check(
        lib.lmoe_permute_two_tables(
            _ptr(ids), n, int(block_m), _ptr(perm.row_idx),
            _ptr(log2phy), int(log2phy.numel()), perm.n_slots, _ptr(perm.counts), _ptr(perm.offsets),
            _ptr(perm.sorted_pairs), _ptr(perm.active), _ptr(perm.tile_off), _ptr(perm.meta),
            _ptr(second_log2phy), int(second_log2phy.numel()), second.n_slots, _ptr(second.counts),
            _ptr(second.offsets), _ptr(second.sorted_pairs), _ptr(second.active), _ptr(second.tile_off),
            _ptr(second.meta), _stream(stream),
        ),
        "lmoe_permute_two_tables",
    )
    for p in (perm, second):
        p.block_m = int(block_m)
        p.builds += 1
    return perm, second


def gather_rows(x: torch.Tensor, top_k: int, perm: Permutation, out: torch.Tensor | None = None,
                *, stream=None) -> torch.Tensor:
    """expanded_x: out[pos] = x[sorted_pairs[pos] // top_k]."""
    lib = load_library()
    _need(x, "x", torch.bfloat16)
    H = x.shape[1]
    if out is None:
        out = _new((perm.n_pairs, H), torch.bfloat16, x.device, stream)
    _need(out, "x_sorted", torch.bfloat16, (perm.n_pairs, H))
    _check(
        lib.lmoe_gather_rows(_ptr(x), H, int(top_k), _ptr(perm.sorted_pairs), _ptr(perm.meta),
                             perm.n_pairs, _ptr(out), _stream(stream)),
        "lmoe_gather_rows",
    )
    return out


# ---------------------------------------------------------------------------
# expert MLP and combine
# ---------------------------------------------------------------------------
def _check_bank(w13: torch.Tensor, w2: torch.Tensor, H: int) -> tuple[int, int]:
    _need(w13, "w13_slots", torch.bfloat16)
    _need(w2, "w2_slots", torch.bfloat16)
    if w13.dim() != 3 or w2.dim() != 3:
        raise ValueError("slot banks must be [P, 2I, H] and [P, H, I]")
    P, two_i, h = w13.shape
    if h != H or two_i % 2 != 0:
        raise ValueError(f"w13_slots shape {tuple(w13.shape)} does not match H={H}")
    I = two_i // 2
    if tuple(w2.shape) != (P, H, I):
        raise ValueError(f"w2_slots shape {tuple(w2.shape)} != {(P, H, I)}")
    return P, I


def grouped_mlp(
    x: torch.Tensor,
    top_k: int,
    w13_slots: torch.Tensor,
    w2_slots: torch.Tensor,
    perm: Permutation,
    act: torch.Tensor,
    y: torch.Tensor,
    *,
    path: int = LMOE_PATH_AUTO,
    pass_pairs: int | None = None,
    stream=None,
) -> torch.Tensor:
    """y[pair] = W2_s . (silu(W13_s[:I] x) * W13_s[I:] x) for the placed pairs.
    pass_pairs: how many of the pairs the pass is expected to place, where it
    is one wave of its layer (chooses the kernel's form, not its bits).
    4-bit banks (mxfp4.pack_experts; uint8): x and act are both bf16 or both
    Mx8Rows, y is bf16 or f32, perm is built with block_m=mx4_block_m(..) (where
    row tiles run, another height is refused).  On path LMOE_PATH_GEMV (which AUTO then is) a
    bf16 act may be [N, 2, I]: rows in two parts whose sum is the value, so that
    its rounding does not show in batches of few tokens."""
    if mxfp4.is_mx4(w13_slots) or mxfp4.is_mx4(w2_slots):
        if x.shape[1] != w2_slots.shape[1]:
            raise ValueError(f"rows of {x.shape[1]} columns, w2_slots of {w2_slots.shape[1]} rows")
        gateup_silu(x, top_k, w13_slots, perm, act, path=path, stream=stream)
        return down(act, w2_slots, perm, y, path=path, stream=stream)
    lib = load_library()
    _need(x, "x", torch.bfloat16)
    T, H = x.shape
    P, I = _check_bank(w13_slots, w2_slots, H)
    if P != perm.n_slots:
        raise ValueError(f"slot bank has {P} slots, permutation {perm.n_slots}")
    if perm.n_pairs != T * top_k:
        raise ValueError("permutation does not match T * top_k pairs")
    _need(act, "act", torch.bfloat16, (perm.n_pairs, I))
    _need(y, "y", torch.bfloat16, (perm.n_pairs, H))
    _check(
        lib.lmoe_grouped_mlp_pass(
            _ptr(x), T, H, I, int(top_k), _ptr(w13_slots), _ptr(w2_slots), P,
            _ptr(perm.offsets), _ptr(perm.sorted_pairs), _ptr(perm.active), _ptr(perm.tile_off),
            _ptr(perm.meta), perm.n_pairs, perm.n_pairs if pass_pairs is None else int(pass_pairs), perm.block_m,
            int(path), _ptr(act), _ptr(y), _stream(stream),
        ),
        "lmoe_grouped_mlp_pass",
    )
    return y


def gateup_silu(x: torch.Tensor, top_k: int, w13_slots: torch.Tensor, perm: Permutation, act: torch.Tensor,
                *, path: int = LMOE_PATH_AUTO, stream=None) -> torch.Tensor:
    """act[pos] = silu(W13_s[:I] x) * (W13_s[I:] x) for the placed pairs (GMM1 + SwiGLU)."""
    if mxfp4.is_mx4(w13_slots):
        return _mx4_gateup_silu(x, top_k, w13_slots, perm, act, path=path, stream=stream)
    lib = load_library()
    _need(x, "x", torch.bfloat16)
    _need(w13_slots, "w13_slots", torch.bfloat16)
    T, H = x.shape
    P, two_i, h = w13_slots.shape
    if h != H or P != perm.n_slots:
        raise ValueError("w13_slots does not match x or the permutation")
    I = two_i // 2
    _need(act, "act", torch.bfloat16, (perm.n_pairs, I))
    _check(
        lib.lmoe_gateup_silu(
            _ptr(x), T, H, I, int(top_k), _ptr(w13_slots), P, _ptr(perm.offsets), _ptr(perm.sorted_pairs),
            _ptr(perm.active), _ptr(perm.tile_off), _ptr(perm.meta), perm.n_pairs, perm.block_m, int(path),
            _ptr(act), _stream(stream),
        ),
        "lmoe_gateup_silu",
    )
    return act


def down(act: torch.Tensor, w2_slots: torch.Tensor, perm: Permutation, y: torch.Tensor,
         *, path: int = LMOE_PATH_AUTO, stream=None) -> torch.Tensor:
    """y[pair] = W2_s act[pos] for the placed pairs (GMM2)."""
    if mxfp4.is_mx4(w2_slots):
        return _mx4_down(act, w2_slots, perm, y, path=path, stream=stream)
    lib = load_library()
    _need(w2_slots, "w2_slots", torch.bfloat16)
    P, H, I = w2_slots.shape
    if P != perm.n_slots:
        raise ValueError("w2_slots does not match the permutation")
    _need(act, "act", torch.bfloat16, (perm.n_pairs, I))
    _need(y, "y", torch.bfloat16, (perm.n_pairs, H))
    _check(
        lib.lmoe_down(
            _ptr(act), H, I, _ptr(w2_slots), P, _ptr(perm.offsets), _ptr(perm.sorted_pairs), _ptr(perm.active),
            _ptr(perm.tile_off), _ptr(perm.meta), perm.n_pairs, perm.block_m, int(path), _ptr(y), _stream(stream),
        ),
        "lmoe_down",
    )
    return y


def _need_mx4(bank: torch.Tensor, name: str, perm: Permutation, K: int, rows: int | None = None) -> int:
    """Check a 4-bit bank of K columns; returns its rows per expert."""
    width = mxfp4.row_bytes(K)
    if rows is not None and _is(bank, torch.uint8, (perm.n_slots, rows, width)):
        return rows
    _need(bank, name, torch.uint8)
    if bank.dim() != 3 or bank.shape[0] != perm.n_slots:
        raise ValueError(f"{name} has shape {tuple(bank.shape)}, the permutation {perm.n_slots} slots")
    if int(bank.shape[2]) != width:
        raise ValueError(f"{name} rows of {int(bank.shape[2])} bytes do not hold {K} columns in 4 bits")
    if rows is not None and int(bank.shape[1]) != rows:
        raise ValueError(f"{name} has {int(bank.shape[1])} rows per expert, not {rows}")
    return int(bank.shape[1])


def _need_rows(rows, name: str, shape: tuple | None = None) -> tuple[torch.Tensor, torch.Tensor | None]:
    """bf16 rows or Mx8Rows, [R, K]: (values, scales or None)."""
    if isinstance(rows, Mx8Rows):
        _need_mx8(rows, name, shape)
        return rows.q, rows.scale
    if shape is None or not _is(rows, torch.bfloat16, shape):
        _need(rows, name, torch.bfloat16, shape)
    if rows.dim() != 2:
        raise ValueError(f"{name} must be [R, K], got {tuple(rows.shape)}")
    return rows, None


def _need_act(act, n: int) -> tuple[torch.Tensor, torch.Tensor | None, bool]:
    """act rows of n pairs: (values, scales or None, bf16 in two parts)."""
    split = not isinstance(act, Mx8Rows) and act.dim() == 3
    if not split:
        return *_need_rows(act, "act", (n, act.shape[-1])), False
    if not _is(act, torch.bfloat16, (n, 2, act.shape[-1])):
        _need(act, "act", torch.bfloat16, (n, 2, act.shape[-1]))
    return act, None, True


def _need_y(y, shape: tuple) -> bool:
    """bf16 or f32 rows by pair; whether they are f32."""
    if not isinstance(y, torch.Tensor) or y.dtype not in (torch.bfloat16, torch.float32):
        raise ValueError("y must be bf16 or f32")
    if not _is(y, y.dtype, shape):
        _need(y, "y", y.dtype, shape)
    return y.dtype is torch.float32


def _check_products(status: int, fn: str, perm: Permutation) -> None:
    if status == LMOE_ERR_SHAPE and perm.block_m not in MX4_BLOCK_M:
        raise ValueError(f"{fn}: unsupported shape; the permutation was built with block_m {perm.block_m}, row tiles "
                         f"of 4-bit experts have {MX4_BLOCK_M} rows (mx4_block_m)")
    _check(status, fn)


def _mx4_gateup_silu(x, top_k: int, w13_slots: torch.Tensor, perm: Permutation, act, *, path: int, stream):
    xq, xs = _need_rows(x, "x", tuple(x.shape))
    T, H = xq.shape
    n = perm.n_pairs
    if n != T * top_k:
        raise ValueError("permutation does not match T * top_k pairs")
    aq, as_, split = _need_act(act, n)
    I = aq.shape[-1]
    if (xs is None) != (as_ is None):
        raise ValueError("x and act must both be bf16 or both be Mx8Rows")
    _need_mx4(w13_slots, "w13_slots", perm, H, 2 * I)
    _same_device(xq, xs, w13_slots, perm.offsets, aq, as_)
    p = perm
    _check_products(
        load_library().lmoe_mx4_gateup_silu(
            xq.data_ptr(), _ptr(xs), T, H, I, top_k, w13_slots.data_ptr(), p.n_slots, p.offsets.data_ptr(),
            p.sorted_pairs.data_ptr(), p.active.data_ptr(), p.tile_off.data_ptr(), p.meta.data_ptr(), n, p.block_m, path,
            aq.data_ptr(), _ptr(as_), split, _stream(stream),
        ),
        "lmoe_mx4_gateup_silu", p,
    )
    return act


def _mx4_down(act, w2_slots: torch.Tensor, perm: Permutation, y: torch.Tensor, *, path: int, stream):
    n = perm.n_pairs
    aq, as_, split = _need_act(act, n)
    I = aq.shape[-1]
    H = _need_mx4(w2_slots, "w2_slots", perm, I, w2_slots.shape[1] if w2_slots.dim() == 3 else None)
    y_f32 = _need_y(y, (n, H))
    _same_device(aq, as_, w2_slots, perm.offsets, y)
    p = perm
    _check_products(
        load_library().lmoe_mx4_down(
            aq.data_ptr(), _ptr(as_), split, H, I, w2_slots.data_ptr(), p.n_slots, p.offsets.data_ptr(),
            p.sorted_pairs.data_ptr(), p.active.data_ptr(), p.tile_off.data_ptr(), p.meta.data_ptr(), n, p.block_m, path,
            y.data_ptr(), y_f32, _stream(stream),
        ),
        "lmoe_mx4_down", p,
    )
    return y


class _Mx4Workspace(ctypes.Structure):
    """lmoe_mx4_workspace."""

    _fields_ = [(n, _vp) for n in ("counts", "offsets", "sorted_pairs", "row_idx", "active", "tile_off", "meta",
                                   "permute_workspace")] + \
               [("permute_workspace_bytes", _sz), ("act", _vp), ("act_scale", _vp), ("y", _vp), ("y_f32", ctypes.c_int32),
                ("act_split", ctypes.c_int32)]


class Mx4Buffers:
    """The buffers of a layer of 4-bit experts (lmoe_mx4_workspace): a permutation,
    act (bf16 or Mx8Rows, [N, I]; bf16 [N, 2, I]: rows in two parts, where the
    split-K kernel runs) and y (bf16 or f32, [N, H]), checked once."""

    def __init__(self, perm: Permutation, act, y: torch.Tensor) -> None:
        aq, as_, self.split = _need_act(act, act.shape[0])
        if y.dtype not in (torch.bfloat16, torch.float32):
            raise ValueError("y must be bf16 or f32")
        _need(y, "y", y.dtype)
        if y.dim() != 2:
            raise ValueError(f"y must be [N, H], got {tuple(y.shape)}")
        if aq.shape[0] < perm.n_pairs or y.shape[0] < perm.n_pairs:
            raise ValueError("act and y need a row for every pair")
        self.perm, self.act, self.y = perm, act, y
        self.device_index = y.get_device()
        for t in (aq, as_, perm.counts, perm.offsets, perm.sorted_pairs, perm.row_idx, perm.active, perm.tile_off,
                  perm.meta, perm.workspace):
            if t is not None and t.get_device() != self.device_index:
                raise ValueError(f"a buffer on {t.device}, y on {y.device}")
        self.hidden, self.intermediate = int(y.shape[1]), int(aq.shape[-1])
        self.mx8 = as_ is not None
        H, I, P = self.hidden, self.intermediate, perm.n_slots
        self.w13_shape, self.w2_shape = (P, 2 * I, mxfp4.row_bytes(H)), (P, H, mxfp4.row_bytes(I))
        self.act_ptr, self.act_scale_ptr = _ptr(aq), _ptr(as_)
        p = perm
        self._struct = _Mx4Workspace(
            _ptr(p.counts), _ptr(p.offsets), _ptr(p.sorted_pairs), _ptr(p.row_idx), _ptr(p.active), _ptr(p.tile_off),
            _ptr(p.meta), _ptr(p.workspace), int(p.workspace.numel()), _ptr(aq), _ptr(as_), _ptr(y),
            int(y.dtype == torch.float32), int(self.split))
        self.address = ctypes.addressof(self._struct)


def _mx4_layer_args(x, topk_weights, topk_ids, w13_slots, w2_slots, log2phy, bufs: Mx4Buffers, out, add):
    """Check a layer call over 4-bit banks; (x values, scales, T, k, table length)."""
    bf16, i32, u8 = torch.bfloat16, torch.int32, torch.uint8
    here = _device_index()
    if bufs.device_index != here:
        raise ValueError(f"buffers on cuda:{bufs.device_index}, the current device is cuda:{here}")
    pairs = topk_ids.shape
    T, k = pairs
    rows = (T, bufs.hidden)
    mx8 = isinstance(x, Mx8Rows)
    if mx8:
        xq, xs = _take_mx8(x, "x", rows, here)
    else:
        xq, xs = x, None
        if not _fits(x, bf16, rows, here):
            _refuse(x, "x", bf16, rows)
    if mx8 != bufs.mx8:
        raise ValueError("x and act must both be bf16 or both be Mx8Rows")
    if T * k != bufs.perm.n_pairs:
        raise ValueError(f"buffers for {bufs.perm.n_pairs} pairs, got {T * k}")
    if not _fits(topk_weights, bf16, pairs, here):
        _refuse(topk_weights, "topk_weights", bf16, pairs)
    if not _fits(topk_ids, i32, pairs, here):
        _refuse(topk_ids, "topk_ids", i32, pairs)
    if not _fits(w13_slots, u8, bufs.w13_shape, here):
        _refuse(w13_slots, "w13_slots", u8, bufs.w13_shape)
    if not _fits(w2_slots, u8, bufs.w2_shape, here):
        _refuse(w2_slots, "w2_slots", u8, bufs.w2_shape)
    if not _fits(out, bf16, rows, here):
        _refuse(out, "out", bf16, rows)
    if add is not None and not _fits(add, bf16, rows, here):
        _refuse(add, "add", bf16, rows)
    n_table = 0
    if log2phy is not None:
        n_table = log2phy.numel()
        if not _fits(log2phy, i32, (n_table,), here):
            _refuse(log2phy, "log2phy", i32)
    return xq, xs, T, k, n_table


def mx4_fused_moe(x, topk_weights: torch.Tensor, topk_ids: torch.Tensor, w13_slots: torch.Tensor,
                  w2_slots: torch.Tensor, log2phy: torch.Tensor | None, bufs: Mx4Buffers, out: torch.Tensor, *,
                  add: torch.Tensor | None = None, path: int = LMOE_PATH_AUTO, block_m: int, stream=None) -> torch.Tensor:
    """permute, gateup_silu, down and combine over 4-bit banks, in one call."""
    lib = load_library()
    xq, xs, T, k, n_table = _mx4_layer_args(x, topk_weights, topk_ids, w13_slots, w2_slots, log2phy, bufs, out, add)
    _check(
        lib.lmoe_mx4_fused_moe(
            xq.data_ptr(), _ptr(xs), T, bufs.hidden, bufs.intermediate, k, w13_slots.data_ptr(), w2_slots.data_ptr(),
            bufs.perm.n_slots, topk_weights.data_ptr(), topk_ids.data_ptr(), _ptr(log2phy), n_table, path, block_m,
            bufs.address, _ptr(add), out.data_ptr(), _stream(stream),
        ),
        "lmoe_mx4_fused_moe",
    )
    bufs.perm.block_m = block_m
    bufs.perm.builds += 1
    return out


# Up to this many pairs fused_experts goes straight from the ids (mx4_decode_few takes
# 64), past it through the permutation, whose order starts the heavy slots first.  us of
# the captured layer, permutation / ids (H, I, experts, top k; tokens):
#   2048, 768, 128, 8    2: 26.0 / 23.0, 3: 27.3 / 25.9, 4: 28.0 / 27.5, 6: 31.0 / 30.8, 8: 32.9 / 32.5
#   2048, 1408, 60, 4    2: 26.8 / 23.1, 4: 28.0 / 25.4, 8: 32.7 / 31.2
#   7168, 2048, 64, 8    2: 71.9 / 69.0, 3: 83.7 / 80.9, 4: 97.7 / 96.2, 6: 109.2 / 111.0, 8: 114.4 / 118.5 (8-bit rows)
MX4_DIRECT_PAIRS = 32


def mx4_decode_few(x, topk_weights: torch.Tensor, topk_ids: torch.Tensor, w13_slots: torch.Tensor,
                   w2_slots: torch.Tensor, log2phy: torch.Tensor | None, bufs: Mx4Buffers, out: torch.Tensor, *,
                   add: torch.Tensor | None = None, stream=None) -> torch.Tensor:
    """Few tokens over 4-bit banks, straight from their ids (bufs.perm is left as
    it was; act and y rows lie by pair), with mx4_fused_moe's bits on path
    LMOE_PATH_GEMV.  At most 64 pairs; y is f32, a bf16 act in two parts."""
    lib = load_library()
    xq, xs, T, k, n_table = _mx4_layer_args(x, topk_weights, topk_ids, w13_slots, w2_slots, log2phy, bufs, out, add)
    if bufs.y.dtype is not torch.float32 or (xs is None and not bufs.split):
        raise ValueError("few tokens' y rows are f32, their bf16 act rows in two parts, [N, 2, I]")
    _check(
        lib.lmoe_mx4_decode_few(
            xq.data_ptr(), _ptr(xs), T, bufs.hidden, bufs.intermediate, k, w13_slots.data_ptr(), w2_slots.data_ptr(),
            bufs.perm.n_slots, topk_weights.data_ptr(), topk_ids.data_ptr(), _ptr(log2phy), n_table, _ptr(add),
            bufs.act_ptr, bufs.act_scale_ptr, bufs.y.data_ptr(), out.data_ptr(), _stream(stream),
        ),
        "lmoe_mx4_decode_few",
    )
    return out


def mx4_decode_one(x, topk_weights: torch.Tensor, topk_ids: torch.Tensor, w13_slots: torch.Tensor,
                   w2_slots: torch.Tensor, log2phy: torch.Tensor | None, bufs: Mx4Buffers, out: torch.Tensor, *,
                   add: torch.Tensor | None = None, second: tuple | None = None, stream=None) -> torch.Tensor:
    """One token over 4-bit banks, straight from its ids (no permutation is built:
    bufs.perm is left as it was).  The sums over K are cut otherwise than
    mx4_fused_moe's, so out may be off that form's by a rounding; one token taken
    in waves over fewer slots than it has experts has that form.  second = (w13,
    w2, log2phy) of another bank, for experts that log2phy leaves out (the decode
    overflow buffer)."""
    lib = load_library()
    xq, xs, T, k, n_table = _mx4_layer_args(x, topk_weights, topk_ids, w13_slots, w2_slots, log2phy, bufs, out, add)
    if T != 1:
        raise ValueError(f"one token, got {T}")
    if xs is None and not bufs.split:
        raise ValueError("one token's bf16 act rows are in two parts, [k, 2, I]")
    b13 = b2 = tab = None
    n_slots_b = n_table_b = 0
    if second is not None:
        if log2phy is None:
            raise ValueError("a second bank needs the first one's table")
        b13, b2, tab = second
        n_slots_b, n_table_b = b13.shape[0], tab.numel()
        _need(b13, "second w13", torch.uint8, (n_slots_b, *w13_slots.shape[1:]))
        _need(b2, "second w2", torch.uint8, (n_slots_b, *w2_slots.shape[1:]))
        _need(tab, "second log2phy", torch.int32)
        _same_device(b13, b2, tab)
    _check(
        lib.lmoe_mx4_decode_one(
            xq.data_ptr(), _ptr(xs), bufs.hidden, bufs.intermediate, k, w13_slots.data_ptr(), w2_slots.data_ptr(),
            bufs.perm.n_slots, topk_weights.data_ptr(), topk_ids.data_ptr(), _ptr(log2phy), n_table,
            _ptr(b13), _ptr(b2), n_slots_b, _ptr(tab), n_table_b, _ptr(add), bufs.act_ptr, bufs.act_scale_ptr, out.data_ptr(), _stream(stream),
        ),
        "lmoe_mx4_decode_one",
    )
    return out


def decode_mlp_two_passes(
    x: torch.Tensor,
    top_k: int,
    w13_a: torch.Tensor,
    w2_a: torch.Tensor,
    perm_a: Permutation,
    w13_b: torch.Tensor,
    w2_b: torch.Tensor,
    perm_b: Permutation,
    act: torch.Tensor,
    y: torch.Tensor,
    *,
    stream=None,
) -> torch.Tensor:
    """The decode GEMVs of both passes of an overflow layer (bank a, overflow
    stage buffer b, each with its own permutation over the same ids) in one
    gate_up and one down launch; y[pair] as grouped_mlp(path=GEMV) writes it
    for either pass.  The tables must map disjoint experts.  Rows up to
    TWO_PASS_MAX_COLS columns (H and I): past that, run the passes one by
    one (grouped_mlp)."""
    lib = load_library()
    _need(x, "x", torch.bfloat16)
    T, H = x.shape
    Pa, I = _check_bank(w13_a, w2_a, H)
    Pb, Ib = _check_bank(w13_b, w2_b, H)
    if Ib != I:
        raise ValueError("the two passes' banks have different intermediate sizes")
    if H > TWO_PASS_MAX_COLS or I > TWO_PASS_MAX_COLS:
        raise ValueError(f"rows past {TWO_PASS_MAX_COLS} columns: run the passes one by one")
    if Pa != perm_a.n_slots or Pb != perm_b.n_slots:
        raise ValueError("a slot bank does not match its permutation")
    if perm_a.n_pairs != T * top_k or perm_b.n_pairs != T * top_k:
        raise ValueError("permutations do not match T * top_k pairs")
    _need(act, "act", torch.bfloat16, (perm_a.n_pairs, I))
    _need(y, "y", torch.bfloat16, (perm_a.n_pairs, H))
    _check(
        lib.lmoe_decode_mlp_two_passes(
            _ptr(x), T, H, I, int(top_k), _ptr(w13_a), _ptr(w2_a), Pa, _ptr(perm_a.offsets),
            _ptr(perm_a.sorted_pairs), _ptr(perm_a.active), _ptr(perm_a.meta), _ptr(w13_b), _ptr(w2_b), Pb,
            _ptr(perm_b.offsets), _ptr(perm_b.sorted_pairs), _ptr(perm_b.active), perm_a.n_pairs, _ptr(act),
            _ptr(y), _stream(stream),
        ),
        "lmoe_decode_mlp_two_passes",
    )
    return y


def stream_mlp_two_passes(
    x: torch.Tensor,
    top_k: int,
    w13_a: torch.Tensor,
    w2_a: torch.Tensor,
    perm_a: Permutation,
    w13_b: torch.Tensor,
    w2_b: torch.Tensor,
    perm_b: Permutation,
    act: torch.Tensor,
    y: torch.Tensor,
    *,
    path: int = LMOE_PATH_STREAM,
    stream=None,
) -> torch.Tensor:
    """decode_mlp_two_passes on the weight-streaming MFMA kernel: y[pair] as
    grouped_mlp(path) writes it for either pass (path STREAM or MFMA).  Both
    permutations are built with block_m STREAM_BLOCK_M; the tables must map disjoint
    experts; H % 64 == 0."""
    lib = load_library()
    _need(x, "x", torch.bfloat16)
    T, H = x.shape
    Pa, I = _check_bank(w13_a, w2_a, H)
    Pb, Ib = _check_bank(w13_b, w2_b, H)
    if Ib != I:
        raise ValueError("the two passes' banks have different intermediate sizes")
    if Pa != perm_a.n_slots or Pb != perm_b.n_slots:
        raise ValueError("a slot bank does not match its permutation")
    if perm_a.n_pairs != T * top_k or perm_b.n_pairs != T * top_k:
        raise ValueError("permutations do not match T * top_k pairs")
    if perm_a.block_m != STREAM_BLOCK_M or perm_b.block_m != STREAM_BLOCK_M:
        raise ValueError(f"both permutations need block_m={STREAM_BLOCK_M}")
    _need(act, "act", torch.bfloat16, (perm_a.n_pairs, I))
    _need(y, "y", torch.bfloat16, (perm_a.n_pairs, H))
    _check(
        lib.lmoe_stream_mlp_two_passes(
            _ptr(x), T, H, I, int(top_k), _ptr(w13_a), _ptr(w2_a), Pa, _ptr(perm_a.offsets),
            _ptr(perm_a.sorted_pairs), _ptr(perm_a.tile_off), _ptr(perm_a.meta), _ptr(w13_b), _ptr(w2_b), Pb,
            _ptr(perm_b.offsets), _ptr(perm_b.sorted_pairs), _ptr(perm_b.tile_off), _ptr(perm_b.meta),
            perm_a.n_pairs, int(path), _ptr(act), _ptr(y), _stream(stream),
        ),
        "lmoe_stream_mlp_two_passes",
    )
    return y


def combine(
    y: torch.Tensor,
    topk_weights: torch.Tensor,
    out: torch.Tensor,
    *,
    row_mask: torch.Tensor | None = None,
    add: torch.Tensor | None = None,
    stream=None,
) -> torch.Tensor:
    """out[t] = add[t] + sum_j w[t,j] * y[t*k+j] (pairs with row_mask < 0
    skipped); y bf16, or f32 (4-bit experts' rows of a few tokens)."""
    lib = load_library()
    _need(topk_weights, "topk_weights", torch.bfloat16)
    T, k = topk_weights.shape
    if y.dtype not in (torch.bfloat16, torch.float32):
        raise ValueError(f"y must be bf16 or f32, got {y.dtype}")
    _need(y, "y", y.dtype)
    H = y.shape[1]
    if y.shape[0] < T * k:
        raise ValueError("y has fewer rows than pairs")
    _need(out, "out", torch.bfloat16, (T, H))
    if row_mask is not None:
        _need(row_mask, "row_mask", torch.int32)
    if add is not None:
        _need(add, "add", torch.bfloat16, (T, H))
    fn = "lmoe_combine_f32" if y.dtype == torch.float32 else "lmoe_combine"
    _check(
        getattr(lib, fn)(_ptr(y), _ptr(row_mask), _ptr(topk_weights), T, k, H, _ptr(add),
                         _ptr(out), _stream(stream)),
        fn,
    )
    return out


def fused_moe_decode(
    x: torch.Tensor,
    topk_weights: torch.Tensor,
    w13_slots: torch.Tensor,
    w2_slots: torch.Tensor,
    perm: Permutation,
    act: torch.Tensor,
    out: torch.Tensor,
    *,
    add: torch.Tensor | None = None,
    y: torch.Tensor | None = None,
    distinct_slots: bool = False,
    stream=None,
) -> torch.Tensor:
    """Decode layer body: gate_up GEMV, then down GEMV fused with the combine
    (up to 16 pairs, no y, or up to 256 pairs where H gives about one workgroup
    per CU), or with a [T*k, H] bf16 workspace y and more pairs the down GEMV
    per (row block, slot) into y and the combine; same out either way.  The
    GEMVs at every token count (fused_moe.fused_experts leaves them where
    layer_path does).  distinct_slots: the caller promises that no slot serves
    two pairs of one token (router-fed ids through a slot table); with one
    token it selects the faster one-pair-per-slot kernels."""
    lib = load_library()
    _need(x, "x", torch.bfloat16)
    T, H = x.shape
    _need(topk_weights, "topk_weights", torch.bfloat16)
    k = topk_weights.shape[1]
    P, I = _check_bank(w13_slots, w2_slots, H)
    if perm.n_pairs != T * k or perm.n_slots != P:
        raise ValueError("permutation does not match the batch or the slot bank")
    if T * k > FUSED_DECODE_MAX_PAIRS:
        raise ValueError(f"fused decode supports at most {FUSED_DECODE_MAX_PAIRS} pairs")
    _need(act, "act", torch.bfloat16, (perm.n_pairs, I))
    _need(out, "out", torch.bfloat16, (T, H))
    if add is not None:
        _need(add, "add", torch.bfloat16, (T, H))
    if y is not None:
        _need(y, "y", torch.bfloat16, (perm.n_pairs, H))
    _check(
        lib.lmoe_fused_moe_decode(
            _ptr(x), T, H, I, k, _ptr(w13_slots), _ptr(w2_slots), P, _ptr(topk_weights),
            _ptr(perm.offsets), _ptr(perm.sorted_pairs), _ptr(perm.row_idx), _ptr(perm.active),
            _ptr(perm.meta), _ptr(add), _ptr(act), _ptr(y), _ptr(out), int(bool(distinct_slots)),
            _stream(stream),
        ),
        "lmoe_fused_moe_decode",
    )
    return out


NOALLOC_SCRATCH_BYTES = 8 << 20  # LMOE_NOALLOC_SCRATCH_BYTES


def fused_moe_decode_noalloc(
    x: torch.Tensor,
    topk_weights: torch.Tensor,
    w13_slots: torch.Tensor,
    w2_slots: torch.Tensor,
    perm: Permutation,
    out: torch.Tensor,
    *,
    add: torch.Tensor | None = None,
    distinct_slots: bool = False,
    stream=None,
) -> torch.Tensor:
    """fused_moe_decode with act / y in the library's per-GPU scratch array
    (nothing is allocated; calls that overlap on one GPU race)."""
    lib = load_library()
    _need(x, "x", torch.bfloat16)
    T, H = x.shape
    _need(topk_weights, "topk_weights", torch.bfloat16)
    k = topk_weights.shape[1]
    P, I = _check_bank(w13_slots, w2_slots, H)
    if perm.n_pairs != T * k or perm.n_slots != P:
        raise ValueError("permutation does not match the batch or the slot bank")
    _need(out, "out", torch.bfloat16, (T, H))
    if add is not None:
        _need(add, "add", torch.bfloat16, (T, H))
    _check(
        lib.lmoe_fused_moe_decode_noalloc(
            _ptr(x), T, H, I, k, _ptr(w13_slots), _ptr(w2_slots), P, _ptr(topk_weights),
            _ptr(perm.offsets), _ptr(perm.sorted_pairs), _ptr(perm.row_idx), _ptr(perm.active),
            _ptr(perm.meta), _ptr(add), _ptr(out), int(bool(distinct_slots)), _stream(stream),
        ),
        "lmoe_fused_moe_decode_noalloc",
    )
    return out


def down_combine(
    act: torch.Tensor,
    topk_weights: torch.Tensor,
    w2_slots: torch.Tensor,
    perm: Permutation,
    out: torch.Tensor,
    *,
    add: torch.Tensor | None = None,
    stream=None,
) -> torch.Tensor:
    """Second half of fused_moe_decode: down GEMV fused with the combine."""
    lib = load_library()
    _need(topk_weights, "topk_weights", torch.bfloat16)
    T, k = topk_weights.shape
    _need(w2_slots, "w2_slots", torch.bfloat16)
    P, H, I = w2_slots.shape
    if perm.n_pairs != T * k or perm.n_slots != P:
        raise ValueError("permutation does not match the batch or the slot bank")
    _need(act, "act", torch.bfloat16, (perm.n_pairs, I))
    _need(out, "out", torch.bfloat16, (T, H))
    if add is not None:
        _need(add, "add", torch.bfloat16, (T, H))
    _check(
        lib.lmoe_down_combine(
            _ptr(act), T, H, I, k, _ptr(w2_slots), P, _ptr(topk_weights), _ptr(perm.offsets),
            _ptr(perm.row_idx), _ptr(perm.active), _ptr(perm.meta), _ptr(add), _ptr(out), _stream(stream),
        ),
        "lmoe_down_combine",
    )
    return out


# ---------------------------------------------------------------------------
# staging
# ---------------------------------------------------------------------------
def _table_pairs(table_update):
    """(table, idx tuple, val tuple, fill) of a table_update argument."""
    table, idx, val = table_update[:3]
    fill = bool(table_update[3]) if len(table_update) > 3 else False
    return table, tuple(int(i) for i in idx), tuple(int(v) for v in val), fill


def stage_copy(
    copies: list[tuple[int, int, int]],
    transfer_stream: torch.cuda.Stream,
    *,
    wait_event: torch.cuda.Event | None = None,
    done_event: torch.cuda.Event | None = None,
    table_update: tuple | None = None,
) -> None:
    """Queue (dst_ptr, src_ptr, nbytes) copies on transfer_stream with one
    hipMemcpyAsync each (any host memory, pageable included).

    The stream first waits for wait_event (slot release) and done_event is
    recorded after the batch; both are torch events, ordered through torch so
    their lazily created handles stay valid.  table_update = (table,
    indices, values[, fill]) writes those int32 entries after the copies
    (fill: every other entry becomes -1), inside the same done_event."""
    lib = load_library()
    if wait_event is not None:
        transfer_stream.wait_event(wait_event)
    n = len(copies)
    dst = (ctypes.c_void_p * max(n, 1))(*[c[0] for c in copies])
    src = (ctypes.c_void_p * max(n, 1))(*[c[1] for c in copies])
    nbytes = (ctypes.c_size_t * max(n, 1))(*[c[2] for c in copies])
    _check(
        lib.lmoe_stage_copy(dst, src, nbytes, n, int(transfer_stream.cuda_stream), None, None),
        "lmoe_stage_copy",
    )
    if table_update is not None:
        table, idx, val, fill = _table_pairs(table_update)
        if fill:
            full = dict.fromkeys(range(int(table.numel())), -1)
            full.update(zip(idx, val))
            idx, val = tuple(full), tuple(full.values())
        table_update_entries(table, idx, val, stream=transfer_stream)
    if done_event is not None:
        done_event.record(transfer_stream)


def stage_gather(
    copies: list[tuple[int, int, int]],
    transfer_stream: torch.cuda.Stream,
    *,
    table_update: tuple | None = None,
) -> bool:
    """Queue (dst_ptr, src_ptr, nbytes) copies as gather-copy kernel launches
    on transfer_stream, with the table_update = (table, indices, values[,
    fill]) entries written by the same launch.  Sources must be page-locked
    host memory or device memory; the library checks every range and refuses
    (returns False, nothing queued) what the device cannot read or what is
    not 16-byte aligned, so the caller can take stage_copy."""
    lib = load_library()
    n = len(copies)
    dst = (ctypes.c_void_p * max(n, 1))(*[c[0] for c in copies])
    src = (ctypes.c_void_p * max(n, 1))(*[c[1] for c in copies])
    nbytes = (ctypes.c_size_t * max(n, 1))(*[c[2] for c in copies])
    table = None
    n_table = n_tab = fill = 0
    ia = va = None
    if table_update is not None:
        table, idx, val, fill_b = _table_pairs(table_update)
        _need(table, "table", torch.int32)
        n_table, n_tab, fill = int(table.numel()), len(idx), int(fill_b)
        ia = (ctypes.c_int32 * max(n_tab, 1))(*idx)
        va = (ctypes.c_int32 * max(n_tab, 1))(*val)
    status = lib.lmoe_stage_gather(dst, src, nbytes, n, _ptr(table), n_table, ia, va, n_tab, fill,
                                   int(transfer_stream.cuda_stream), None, None)
    if status in (LMOE_ERR_ARG, LMOE_ERR_SHAPE):
        return False
    _check(status, "lmoe_stage_gather")
    return True


def table_update_entries(table: torch.Tensor, idx, val, *, stream=None) -> None:
    """table[idx[i]] = val[i] (distinct int indices) with one small kernel
    whose arguments carry the pairs: no staging tensor, no copy."""
    lib = load_library()
    _need(table, "table", torch.int32)
    n = len(idx)
    if n != len(val):
        raise ValueError(f"indices and values differ in length: {n} != {len(val)}")
    if n == 0:
        return
    ia = (ctypes.c_int32 * n)(*[int(i) for i in idx])
    va = (ctypes.c_int32 * n)(*[int(v) for v in val])
    _check(lib.lmoe_table_update(_ptr(table), int(table.numel()), ia, va, n, _stream(stream)),
           "lmoe_table_update")


# ---------------------------------------------------------------------------
# device-side capacity waves (lmoe_wave_plan / lmoe_wave_stage)
# ---------------------------------------------------------------------------
WAVE_PLAN_MAX_EXPERTS = 1024
WAVE_PLAN_MAX_SLOTS = 1024
WAVE_PLAN_MAX_WAVES = 256


class WavePlan:
    """Device buffer of one layer shape's wave plan (fixed address, graph safe)."""

    HEADER = 4

    def __init__(self, n_routed: int, n_slots: int, max_waves: int, device) -> None:
        n = int(load_library().lmoe_wave_plan_bytes(int(n_routed), int(n_slots), int(max_waves)))
        if n < 0:
            raise ValueError(f"device wave plan supports <= {WAVE_PLAN_MAX_EXPERTS} experts, "
                             f"<= {WAVE_PLAN_MAX_SLOTS} slots and <= {WAVE_PLAN_MAX_WAVES} waves; got "
                             f"{n_routed}, {n_slots}, {max_waves}")
        self.n_routed, self.n_slots, self.max_waves = int(n_routed), int(n_slots), int(max_waves)
        self.buf = torch.zeros(n // 4, dtype=torch.int32, device=device)

    # host views (tests and evidence; each reads the device buffer)
    def to_host(self) -> dict:
        b = self.buf.cpu().tolist()
        E, W, P, h = self.n_routed, self.max_waves, self.n_slots, self.HEADER
        counts = b[h:h + E]
        wave_of = b[h + E:h + 2 * E]
        slot_of = b[h + 2 * E:h + 3 * E]
        size = b[h + 3 * E:h + 3 * E + W]
        members = b[h + 3 * E + W:]
        n_waves = b[0]
        waves = tuple(tuple(members[w * P:w * P + size[w]]) for w in range(max(n_waves, 0)))
        return {"n_waves": n_waves, "n_active": b[1], "invalid": b[2], "counts": counts, "wave_of": wave_of,
                "slot_of": slot_of, "size": size, "waves": waves}


def wave_plan(ids: torch.Tensor, plan: WavePlan, *, n_total: int | None = None, stream=None) -> WavePlan:
    lib = load_library()
    _need(ids, "topk_ids", torch.int32)
    n_total = plan.n_routed if n_total is None else int(n_total)
    _check(lib.lmoe_wave_plan(_ptr(ids), int(ids.numel()), plan.n_routed, n_total, plan.n_slots, plan.max_waves,
                              _ptr(plan.buf), _stream(stream)), "lmoe_wave_plan")
    return plan


def wave_stage(plan: WavePlan, wave: int, *, main_table: torch.Tensor, main_owner: torch.Tensor,
               main_w13: torch.Tensor,
               main_w2: torch.Tensor, main_slots: int, host_w13: torch.Tensor, host_w2: torch.Tensor,
               stage_w13: torch.Tensor, stage_w2: torch.Tensor, stage_table: torch.Tensor,
               n_pinned: int = 0, stream=None) -> None:
    """Copy wave `wave`'s experts into the stage buffer and write its table.
    host_w13 / host_w2 must be page-locked [n_routed, ...] blocks."""
    lib = load_library()
    for name, t in (("main_w13", main_w13), ("main_w2", main_w2), ("stage_w13", stage_w13),
                    ("stage_w2", stage_w2), ("host_w13", host_w13), ("host_w2", host_w2)):
        if t.dtype not in (torch.bfloat16, torch.uint8) or t.dtype != main_w13.dtype or not t.is_contiguous():
            raise ValueError(f"{name} must be a contiguous bf16 tensor (or all of them 4-bit, uint8)")
    if not (host_w13.is_pinned() and host_w2.is_pinned()):
        raise ValueError("device wave staging reads the host store directly: it must be page-locked")
    if int(host_w13.shape[0]) < plan.n_routed or int(main_table.numel()) < plan.n_routed:
        raise ValueError("host store or main table does not cover the routed experts")
    if int(stage_w13.shape[0]) < plan.n_slots + int(n_pinned) or int(main_w13.shape[0]) < int(main_slots):
        raise ValueError("stage buffer or main bank is smaller than its slot count")
    _need(main_table, "main_table", torch.int32)
    _need(main_owner, "main_owner", torch.int32)
    if int(main_owner.numel()) < int(main_slots):
        raise ValueError("main_owner must hold one entry per main slot")
    _need(stage_table, "stage_table", torch.int32)
    size = int(host_w13.element_size())
    b13 = int(host_w13[0].numel()) * size
    b2 = int(host_w2[0].numel()) * size
    if int(stage_w13[0].numel()) * size != b13 or int(stage_w2[0].numel()) * size != b2 or \
            int(main_w13[0].numel()) * size != b13 or int(main_w2[0].numel()) * size != b2:
        raise ValueError("expert row sizes differ between host store, main bank and stage buffer")
    _check(lib.lmoe_wave_stage(
        _ptr(plan.buf), plan.n_routed, plan.n_slots, plan.max_waves, int(wave), _ptr(main_table),
        _ptr(main_owner), _ptr(main_w13), _ptr(main_w2), int(main_slots), _ptr(host_w13), _ptr(host_w2), _ptr(stage_w13),
        _ptr(stage_w2), b13, b2, _ptr(stage_table), int(stage_table.numel()), int(n_pinned), plan.n_slots,
        _stream(stream)), "lmoe_wave_stage")
