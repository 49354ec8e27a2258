"""ctypes binding of libf8b200.so (the C-ABI kernel library, `include/f8b200.h`).

There is no fallback: if the library is missing or a call fails the caller gets an
exception.  Nothing here runs on the CPU.
"""
from __future__ import annotations

import ctypes
import functools
import os
from array import array
from typing import Optional, Sequence

import torch

_LIB_PATH = os.path.join(os.path.dirname(os.path.abspath(__file__)), "lib", "libf8b200.so")
_lib: Optional[ctypes.CDLL] = None

BF16, FP16, FP32 = 0, 1, 2
E4M3, E5M2 = 0, 1

_HP_CODE = {torch.bfloat16: BF16, torch.float16: FP16, torch.float32: FP32}
_FP8_CODE = {torch.float8_e4m3fn: E4M3, torch.float8_e5m2: E5M2}
FP8_DTYPE = {E4M3: torch.float8_e4m3fn, E5M2: torch.float8_e5m2}

# every symbol include/f8b200.h declares
EXPORTS = (
    "f8b200_status_string",
    "f8b200_device_check",
    "f8b200_last_cuda_error",
    "f8b200_amax",
    "f8b200_multi_amax",
    "f8b200_amax_to_scale",
    "f8b200_cast",
    "f8b200_cast_dynamic",
    "f8b200_cast_scatter",
    "f8b200_multi_cast",
    "f8b200_transpose_u8",
    "f8b200_delayed_sync",
    "f8b200_gemm_fp8",
    "f8b200_gemm_fp8_ws",
    "f8b200_gemm_fp8_static_scratch",
    "f8b200_gemm_kernel_choice",
    "f8b200_gemm_fp8_scatter_rows",
    "f8b200_sum_slots",
    "f8b200_rmsnorm_amax",
    "f8b200_rmsnorm_cast",
    "f8b200_swiglu_amax",
    "f8b200_swiglu_amax_approx",
    "f8b200_swiglu_cast",
    "f8b200_rmsnorm_bwd_workspace_bytes",
    "f8b200_rmsnorm_bwd",
    "f8b200_swiglu_bwd",
    "f8b200_swiglu_bwd_approx",
    "f8b200_block_exponent_bytes",
    "f8b200_cast_blockwise",
    "f8b200_uncast_blockwise",
    "f8b200_gemm_blockwise",
    "f8b200_layer_norm",
    "f8b200_layer_norm_bwd_workspace_bytes",
    "f8b200_layer_norm_bwd",
    "f8b200_multi_norm_workspace_bytes",
    "f8b200_multi_norm",
    "f8b200_multi_clip",
    "f8b200_read_device_error",
    "f8b200_check_device_error",
)


ERR_BAD_ARG = -1


class F8B200Error(RuntimeError):
    status = 0  # of the entry point that returned it


def lib_path() -> str:
    return _LIB_PATH


def load() -> ctypes.CDLL:
    """Loads the kernel library once; raises if it has not been built."""
    global _lib
    if _lib is not None:
        return _lib
    if not os.path.exists(_LIB_PATH):
        raise F8B200Error(
            f"{_LIB_PATH} is missing: build it with `python -m float8_experimental_b200.csrc.build` "
            "(there is no CPU or PyTorch fallback for these kernels)"
        )
    lib = ctypes.CDLL(_LIB_PATH)
    vp, i64, i32 = ctypes.c_void_p, ctypes.c_int64, ctypes.c_int
    lib.f8b200_status_string.restype = ctypes.c_char_p
    lib.f8b200_status_string.argtypes = [i32]
    lib.f8b200_last_cuda_error.restype = ctypes.c_char_p
    lib.f8b200_last_cuda_error.argtypes = []
    lib.f8b200_device_check.argtypes = []
    lib.f8b200_amax.argtypes = [vp, i32, i64, vp, vp]
    lib.f8b200_multi_amax.argtypes = [ctypes.POINTER(vp), ctypes.POINTER(i64), i32, i32, vp, vp]
    lib.f8b200_amax_to_scale.argtypes = [vp, i64, i32, i32, i32, vp, vp]
    lib.f8b200_cast.argtypes = [vp, i32, i64, i64, i64, i32, vp, vp, i32, i32, vp, i64, vp, i64, vp, i32, vp]
    lib.f8b200_cast_scatter.argtypes = [vp, i32, i64, i64, i64, i32, vp, vp, i32, i32, ctypes.POINTER(vp), i32, i64,
                                        vp]
    lib.f8b200_cast_dynamic.argtypes = [vp, i32, i64, i64, i32, vp, vp, vp, vp]
    lib.f8b200_multi_cast.argtypes = [ctypes.POINTER(vp), ctypes.POINTER(i64), i32, i32, vp, i32, i32, ctypes.POINTER(vp), vp]
    lib.f8b200_transpose_u8.argtypes = [vp, i64, i64, i64, vp, i64, vp]
    lib.f8b200_delayed_sync.argtypes = [vp, vp, i64, i64, i32, i64, i32, vp, vp, i64, vp]
    lib.f8b200_gemm_fp8.argtypes = [vp, i32, i64, vp, i32, i64, vp, vp, vp, i32, vp, i64, i64, i64, i64, i32, vp]
    lib.f8b200_gemm_fp8_static_scratch.argtypes = lib.f8b200_gemm_fp8.argtypes
    lib.f8b200_gemm_fp8_ws.argtypes = [vp, i32, i32, i64, vp, i32, i32, i64, vp, vp, vp, i32, vp, i64, i64, i64, i64,
                                       i32, vp, i64, vp]
    lib.f8b200_rmsnorm_amax.argtypes = [vp, i32, i64, i64, i64, vp, ctypes.c_float, vp, vp, vp]
    lib.f8b200_rmsnorm_cast.argtypes = [vp, i32, i64, i64, i64, vp, vp, vp, i32, vp, vp, i64, vp]
    lib.f8b200_swiglu_amax.argtypes = [vp, vp, i32, i64, i64, i64, i64, vp, i64, vp, vp]
    lib.f8b200_swiglu_amax_approx.argtypes = [vp, vp, i32, i64, i64, i64, i64, vp, i64, vp, vp]
    lib.f8b200_swiglu_cast.argtypes = [vp, vp, i32, i64, i64, i64, i64, vp, i32, vp, vp, i64, vp]
    lib.f8b200_rmsnorm_bwd_workspace_bytes.argtypes = [i64]
    lib.f8b200_rmsnorm_bwd_workspace_bytes.restype = i64
    lib.f8b200_rmsnorm_bwd.argtypes = [vp, vp, i32, i64, i64, i64, i64, vp, vp, vp, i64, vp, vp, i64, vp]
    lib.f8b200_swiglu_bwd.argtypes = [vp, vp, vp, i32, i64, i64, i64, i64, i64, vp, vp, i64, vp]
    lib.f8b200_swiglu_bwd_approx.argtypes = [vp, vp, vp, i32, i64, i64, i64, i64, i64, vp, vp, i64, vp]
    lib.f8b200_read_device_error.argtypes = [ctypes.POINTER(ctypes.c_uint32)]
    lib.f8b200_check_device_error.argtypes = []
    lib.f8b200_gemm_kernel_choice.argtypes = [i64, i64, i64]
    lib.f8b200_gemm_fp8_scatter_rows.argtypes = [vp, i32, i32, i64, vp, i32, i32, i64, vp, vp, vp, i32, ctypes.POINTER(vp),
                                                 i32, i64, i64, i64, i64, i64, vp, i64, vp]
    lib.f8b200_sum_slots.argtypes = [vp, i32, i64, i32, i64, vp, vp]
    lib.f8b200_cast_blockwise.argtypes = [vp, i32, i64, i64, i64, i32, i32, vp, i64, vp, i64, vp, vp, i64, vp, i64, vp, vp]
    lib.f8b200_block_exponent_bytes.argtypes = [i64, i64]
    lib.f8b200_block_exponent_bytes.restype = i64
    lib.f8b200_uncast_blockwise.argtypes = [vp, i32, i64, i64, i64, vp, i64, i64, i32, i32, i32, vp, i64, vp]
    lib.f8b200_gemm_blockwise.argtypes = [vp, i32, i32, i64, vp, i64, i64, i32, vp, vp, i32, i32, i64, vp, i64, i64, i32, vp,
                                          vp, i32, vp, i64, i64, i64, i64, vp, i64, vp]
    lib.f8b200_layer_norm.argtypes = [vp, i32, i64, i64, i64, vp, vp, i32, ctypes.c_float, vp, i64, vp, vp, vp]
    lib.f8b200_layer_norm_bwd_workspace_bytes.argtypes = [i64]
    lib.f8b200_layer_norm_bwd_workspace_bytes.restype = i64
    lib.f8b200_layer_norm_bwd.argtypes = [vp, vp, i32, i64, i64, i64, i64, vp, i32, vp, vp, vp, i64, vp, vp, vp, i64, vp]
    lib.f8b200_multi_norm_workspace_bytes.argtypes = [ctypes.POINTER(i64), i32]
    lib.f8b200_multi_norm_workspace_bytes.restype = i64
    lib.f8b200_multi_norm.argtypes = [ctypes.POINTER(vp), ctypes.POINTER(i64), ctypes.POINTER(i32), i32, i32, i32, vp, vp,
                                      i64, vp]
    lib.f8b200_multi_clip.argtypes = [ctypes.POINTER(vp), ctypes.POINTER(i64), ctypes.POINTER(i32), i32, vp, ctypes.c_float,
                                      vp]
    for name in EXPORTS:
        fn = getattr(lib, name)
        if fn.restype is not ctypes.c_char_p and fn.restype is not i64:
            fn.restype = i32
    _lib = lib
    return lib


def _check(status: int, what: str) -> None:
    if status == 0:
        return
    lib = load()
    msg = lib.f8b200_status_string(status).decode()
    detail = lib.f8b200_last_cuda_error().decode() if status == -4 else ""
    error = F8B200Error(f"{what}: {msg}" + (f" [{detail}]" if detail else ""))
    error.status = status
    raise error


def hp_code(dtype: torch.dtype) -> int:
    try:
        return _HP_CODE[dtype]
    except KeyError:
        raise F8B200Error(f"unsupported high-precision dtype {dtype}") from None


def fp8_code(dtype: torch.dtype) -> int:
    try:
        return _FP8_CODE[dtype]
    except KeyError:
        raise F8B200Error(f"unsupported float8 dtype {dtype}") from None


def _stream(t: torch.Tensor) -> int:
    # the handle alone: torch.cuda.current_stream builds a Stream object around it, 3 us of host time per launch
    return torch._C._cuda_getCurrentRawStream(t.get_device())


def _require_cuda(*tensors: Optional[torch.Tensor]) -> None:
    for t in tensors:
        if t is not None and not t.is_cuda:
            raise F8B200Error("f8b200 kernels run on CUDA tensors only (no CPU path exists)")


def _ptr(t: Optional[torch.Tensor]) -> Optional[int]:
    return None if t is None else t.data_ptr()


# ---------------------------------------------------------------------------
# instrumentation for the benchmark: kernel launch count and, on request, CUDA events
# around every launch (recorded on the launching stream)
# ---------------------------------------------------------------------------
_launches = 0
_events_on = False
_events = {}


def reset_counters() -> None:
    global _launches
    _launches = 0
    _events.clear()


def launch_count() -> int:
    return _launches


def enable_kernel_events(on: bool) -> None:
    global _events_on
    _events_on = bool(on)


def kernel_event_totals():
    """{kind: (total_ms, launches)} of the launches recorded since reset_counters()."""
    torch.cuda.synchronize()
    return {k: (sum(a.elapsed_time(b) for a, b in v), len(v)) for k, v in _events.items()}


@functools.lru_cache(maxsize=None)
def _sm_pairs(device: int) -> int:
    return torch.cuda.get_device_properties(device).multi_processor_count // 2


class _Launch:
    """Context manager around one kernel launch on `device`: makes that device current
    (only if it is not already), counts the launch, optionally times it."""

    __slots__ = ("kind", "n", "start", "guard")

    def __init__(self, kind: str, device: torch.device, n: int = 1):
        self.kind, self.n, self.start = kind, n, None
        idx = device.index
        # the tensor at hand has initialised CUDA, which torch.cuda.current_device would see to first
        self.guard = None if (idx is None or idx == torch._C._cuda_getDevice()) else torch.cuda.device(idx)

    def __enter__(self):
        global _launches
        _launches += self.n
        if self.guard is not None:
            self.guard.__enter__()
        if _events_on:
            self.start = torch.cuda.Event(enable_timing=True)
            self.start.record()
        return self

    def __exit__(self, *exc):
        if self.start is not None:
            end = torch.cuda.Event(enable_timing=True)
            end.record()
            _events.setdefault(self.kind, []).append((self.start, end))
        if self.guard is not None:
            self.guard.__exit__(*exc)
        return False


# ---------------------------------------------------------------------------
# thin tensor-level wrappers (each sets the device of its first argument)
# ---------------------------------------------------------------------------
def amax(x: torch.Tensor, out: torch.Tensor) -> None:
    _require_cuda(x, out)
    with _Launch("amax", x.device):
        _check(load().f8b200_amax(x.data_ptr(), hp_code(x.dtype), x.numel(), out.data_ptr(), _stream(x)), "f8b200_amax")


def multi_amax(xs: Sequence[torch.Tensor], out: torch.Tensor) -> None:
    n = len(xs)
    if n == 0:
        return
    _require_cuda(out, *xs)
    dt = xs[0].dtype
    if any(t.dtype != dt for t in xs):
        raise F8B200Error("multi_amax needs tensors of one dtype")
    ptrs = (ctypes.c_void_p * n)(*[t.data_ptr() for t in xs])
    numels = (ctypes.c_int64 * n)(*[t.numel() for t in xs])
    with _Launch("amax", out.device, (n + 127) // 128):
        _check(load().f8b200_multi_amax(ptrs, numels, n, hp_code(dt), out.data_ptr(), _stream(out)), "f8b200_multi_amax")


def amax_to_scale(amax_t: torch.Tensor, fp8_kind: int, amax_dtype: int, orig_dtype: int, out: torch.Tensor) -> None:
    _require_cuda(amax_t, out)
    with _Launch("scale", out.device):
        _check(
            load().f8b200_amax_to_scale(amax_t.data_ptr(), amax_t.numel(), fp8_kind, amax_dtype, orig_dtype,
                                        out.data_ptr(), _stream(out)),
            "f8b200_amax_to_scale",
        )


def cast(x: torch.Tensor, rows: int, cols: int, ld_x: int, scale_src: int, scale_in: torch.Tensor,
         scale_out: Optional[torch.Tensor], product_fp32: bool, fp8_kind: int, out: Optional[torch.Tensor],
         ld_out: int, out_t: Optional[torch.Tensor], ld_out_t: int, amax_out: Optional[torch.Tensor],
         reverse: bool) -> None:
    _require_cuda(x, scale_in, scale_out, out, out_t, amax_out)
    with _Launch("cast", x.device):
        _check(
            load().f8b200_cast(x.data_ptr(), hp_code(x.dtype), rows, cols, ld_x, scale_src, scale_in.data_ptr(),
                               _ptr(scale_out), int(product_fp32), fp8_kind, _ptr(out), ld_out, _ptr(out_t),
                               ld_out_t, _ptr(amax_out), int(reverse), _stream(x)),
            "f8b200_cast",
        )


def cast_dynamic(x: torch.Tensor, rows: int, cols: int, fp8_kind: int, amax_out: torch.Tensor, scale_out: torch.Tensor,
                 out: torch.Tensor) -> None:
    """`f8b200_cast_dynamic`: amax + cast of a contiguous matrix in one host call (two launches)."""
    _require_cuda(x, amax_out, scale_out, out)
    with _Launch("cast", x.device, 2):
        _check(load().f8b200_cast_dynamic(x.data_ptr(), hp_code(x.dtype), rows, cols, fp8_kind, amax_out.data_ptr(),
                                          scale_out.data_ptr(), out.data_ptr(), _stream(x)), "f8b200_cast_dynamic")


def multi_cast(xs: Sequence[torch.Tensor], scales: torch.Tensor, product_fp32: bool, fp8_kind: int,
               outs: Sequence[torch.Tensor]) -> None:
    """`f8b200_multi_cast`: every contiguous tensor of `xs` cast with its own scale (`scales[i]`) into
    `outs[i]`, one launch per 96 tensors."""
    n = len(xs)
    if n == 0:
        return
    _require_cuda(scales, *xs, *outs)
    dt = xs[0].dtype
    if any(t.dtype != dt for t in xs):
        raise F8B200Error("multi_cast needs tensors of one dtype")
    ptrs = (ctypes.c_void_p * n)(*[t.data_ptr() for t in xs])
    optrs = (ctypes.c_void_p * n)(*[t.data_ptr() for t in outs])
    numels = (ctypes.c_int64 * n)(*[t.numel() for t in xs])
    with _Launch("cast", scales.device, (n + 95) // 96):
        _check(load().f8b200_multi_cast(ptrs, numels, n, hp_code(dt), scales.data_ptr(), int(product_fp32), fp8_kind,
                                        optrs, _stream(scales)), "f8b200_multi_cast")


def transpose_u8(src: torch.Tensor, rows: int, cols: int, ld_in: int, dst: torch.Tensor, ld_out: int) -> None:
    _require_cuda(src, dst)
    with _Launch("transpose", src.device):
        _check(load().f8b200_transpose_u8(src.data_ptr(), rows, cols, ld_in, dst.data_ptr(), ld_out, _stream(src)),
               "f8b200_transpose_u8")


def delayed_sync(amax_t: torch.Tensor, hist: torch.Tensor, n_e4m3: int, orig_dtype: int, scale_out: torch.Tensor,
                 hist_out: Optional[torch.Tensor]) -> None:
    _require_cuda(amax_t, hist, scale_out, hist_out)
    rows, hist_len = hist.shape
    with _Launch("sync", hist.device):
        _check(
            load().f8b200_delayed_sync(amax_t.data_ptr(), hist.data_ptr(), hist.stride(0), rows, hist_len, n_e4m3,
                                       orig_dtype, scale_out.data_ptr(), _ptr(hist_out),
                                       hist_out.stride(0) if hist_out is not None else 0, _stream(hist)),
            "f8b200_delayed_sync",
        )


# ---------------------------------------------------------------------------
# optional single-GPU library: the cluster-multicast GEMM (csrc/gemm_mc.cu).  Runs on several GPUs
# ship without it; everything then goes through libf8b200.so.
# ---------------------------------------------------------------------------
_MC_LIB_PATH = os.path.join(os.path.dirname(_LIB_PATH), "libf8b200_mc.so")
_mc_lib = None
_mc_tried = False


def load_mc():
    """The multicast GEMM library, or None when it was not built / not shipped."""
    global _mc_lib, _mc_tried
    if not _mc_tried:
        _mc_tried = True
        if os.path.exists(_MC_LIB_PATH):
            lib = ctypes.CDLL(_MC_LIB_PATH)
            vp, i64, i32 = ctypes.c_void_p, ctypes.c_int64, ctypes.c_int
            lib.f8b200_mc_gemm_fp8.argtypes = [vp, i32, i32, i64, vp, i32, i32, i64, vp, vp, vp, i32, vp, i64, i64, i64,
                                               i64, i32, i32, vp, i64, vp]
            lib.f8b200_mc_gemm_fp8.restype = i32
            lib.f8b200_mc_read_device_error.argtypes = [ctypes.POINTER(ctypes.c_uint32)]
            lib.f8b200_mc_read_device_error.restype = i32
            _mc_lib = lib
    return _mc_lib


def _single_gpu_job() -> bool:
    """True only when this process can be sure it belongs to a job that uses ONE GPU: exactly one
    CUDA device is visible, no launcher announced more than one rank (WORLD_SIZE /
    LOCAL_WORLD_SIZE, which are set before `init_process_group` runs), and no process group with
    more than one rank exists.  The multicast GEMM may run in such jobs only: its TMA loads must
    never be handed memory of another GPU."""
    if torch.cuda.device_count() != 1:
        return False
    for var in ("WORLD_SIZE", "LOCAL_WORLD_SIZE"):
        try:
            if int(os.environ.get(var, "1")) > 1:
                return False
        except ValueError:
            return False
    if torch.distributed.is_available() and torch.distributed.is_initialized() and torch.distributed.get_world_size() > 1:
        return False
    return True


def _mc_cluster(m: int, n: int, k: int):
    """Cluster shape (tiles along M, along N) of the multicast GEMM for this product, or None
    to use the kernels of libf8b200.so.  Opt-in: F8B200_GEMM_MC=21 / 22 / 41 select 2 x 1 or
    2 x 2 clusters of 256x256 tiles, or two CTA pairs sharing B; by default (and with
    F8B200_GEMM_MC=0, or when F8B200_GEMM_MODE forces a kernel) nothing uses it, because the
    512x256 pair kernel of libf8b200.so measured faster on every product.  Only jobs on a single
    GPU may use it at all (`_single_gpu_job`; the C entry point checks on its side that every
    pointer is the current device's own memory)."""
    mode = os.environ.get("F8B200_GEMM_MC", "0")
    if mode not in ("21", "22", "41") or not _single_gpu_job() or load_mc() is None:
        return None
    if os.environ.get("F8B200_GEMM_MODE", "")[:1] in ("1", "2", "w", "p"):
        return None
    return {"21": (2, 1), "22": (2, 2), "41": (4, 1)}[mode]


GEMM_WORKSPACE_BYTES = 256  # F8B200_GEMM_WORKSPACE_BYTES in include/f8b200.h
_gemm_workspaces: dict = {}


def _gemm_workspace(device: torch.device, stream: int) -> torch.Tensor:
    """Scheduling workspace of the GEMMs issued on `stream` of `device`: one small buffer per
    stream, kept for the life of the process, because GEMMs that may overlap must not share one."""
    key = (device.index, stream)
    ws = _gemm_workspaces.get(key)
    if ws is None:
        ws = torch.empty(GEMM_WORKSPACE_BYTES, dtype=torch.uint8, device=device)
        _gemm_workspaces[key] = ws
    return ws


def gemm_fp8(a: torch.Tensor, lda: int, b: torch.Tensor, ldb: int, scale_a: torch.Tensor, scale_b: torch.Tensor,
             bias: Optional[torch.Tensor], out: torch.Tensor, ldo: int, m: int, n: int, k: int,
             use_fast_accum: bool, a_mn_major: bool = False, b_mn_major: bool = False) -> None:
    """`f8b200_gemm_fp8_ws` with this stream's workspace (dynamic tile scheduling).  `a` is the
    [m, k] operand stored K-contiguous, or with `a_mn_major` its transpose stored [k, m]; likewise
    `b` ([n, k], or [k, n] with `b_mn_major`).  F8B200_GEMM_WS=0 in the environment selects the
    workspace-free `f8b200_gemm_fp8` (K-major operands only)."""
    _require_cuda(a, b, scale_a, scale_b, bias, out)
    stream = _stream(a)
    cluster = _mc_cluster(m, n, k)
    with _Launch("gemm", a.device):
        if cluster is not None:
            ws = _gemm_workspace(a.device, stream)
            rc = _mc_lib.f8b200_mc_gemm_fp8(a.data_ptr(), fp8_code(a.dtype), int(a_mn_major), lda, b.data_ptr(),
                                            fp8_code(b.dtype), int(b_mn_major), ldb, scale_a.data_ptr(),
                                            scale_b.data_ptr(), _ptr(bias), hp_code(out.dtype), out.data_ptr(), ldo,
                                            m, n, k, cluster[0], cluster[1], ws.data_ptr(), ws.numel(), stream)
            if rc != -6:  # F8B200_ERR_UNSUPPORTED: such clusters cannot be scheduled here / layout not covered
                if rc != 0:
                    raise F8B200Error(f"f8b200_mc_gemm_fp8: {load().f8b200_status_string(rc).decode()}")
                return
        if os.environ.get("F8B200_GEMM_WS", "1") == "0" and not (a_mn_major or b_mn_major):
            _check(
                load().f8b200_gemm_fp8(a.data_ptr(), fp8_code(a.dtype), lda, b.data_ptr(), fp8_code(b.dtype), ldb,
                                       scale_a.data_ptr(), scale_b.data_ptr(), _ptr(bias), hp_code(out.dtype),
                                       out.data_ptr(), ldo, m, n, k, int(use_fast_accum), stream),
                "f8b200_gemm_fp8",
            )
        else:
            ws = _gemm_workspace(a.device, stream)
            _check(
                load().f8b200_gemm_fp8_ws(a.data_ptr(), fp8_code(a.dtype), int(a_mn_major), lda, b.data_ptr(),
                                          fp8_code(b.dtype), int(b_mn_major), ldb, scale_a.data_ptr(),
                                          scale_b.data_ptr(), _ptr(bias), hp_code(out.dtype), out.data_ptr(), ldo, m,
                                          n, k, int(use_fast_accum), ws.data_ptr(), ws.numel(), stream),
                "f8b200_gemm_fp8_ws",
            )


def gemm_fp8_scatter_rows(a: torch.Tensor, lda: int, b: torch.Tensor, ldb: int, scale_a: torch.Tensor,
                          scale_b: torch.Tensor, out_dtype: torch.dtype, out_ptrs: Sequence[int], rows_per_block: int,
                          ldo: int, m: int, n: int, k: int, a_mn_major: bool = False, b_mn_major: bool = False) -> None:
    """`f8b200_gemm_fp8_scatter_rows`: the GEMM whose output row blocks go round-robin to the
    addresses in `out_ptrs` (this device's own buffer and peer-mapped buffers of other devices)."""
    _require_cuda(a, b, scale_a, scale_b)
    stream = _stream(a)
    ws = _gemm_workspace(a.device, stream)
    arr = (ctypes.c_void_p * len(out_ptrs))(*[ctypes.c_void_p(p) for p in out_ptrs])
    with _Launch("gemm", a.device):
        _check(
            load().f8b200_gemm_fp8_scatter_rows(a.data_ptr(), fp8_code(a.dtype), int(a_mn_major), lda, b.data_ptr(),
                                                fp8_code(b.dtype), int(b_mn_major), ldb, scale_a.data_ptr(),
                                                scale_b.data_ptr(), None, hp_code(out_dtype), arr, len(out_ptrs),
                                                rows_per_block, ldo, m, n, k, ws.data_ptr(), ws.numel(), stream),
            "f8b200_gemm_fp8_scatter_rows",
        )


def sum_slots(slots: torch.Tensor, n_slots: int, slot_stride: int, numel: int, out: torch.Tensor) -> None:
    """`f8b200_sum_slots`: out = sum of the first `n_slots` slots of `slots` (fp32 accumulation)."""
    _require_cuda(slots, out)
    with _Launch("sum_slots", out.device):
        _check(
            load().f8b200_sum_slots(slots.data_ptr(), n_slots, slot_stride, hp_code(out.dtype), numel, out.data_ptr(),
                                    _stream(out)),
            "f8b200_sum_slots",
        )


def gemm_kernel_choice(m: int, n: int, k: int) -> int:
    """Code of the kernel the library would run for this product (see include/f8b200.h)."""
    return int(load().f8b200_gemm_kernel_choice(m, n, k))


def gemm_fp8_static_scratch(a: torch.Tensor, lda: int, b: torch.Tensor, ldb: int, scale_a: torch.Tensor,
                            scale_b: torch.Tensor, bias: Optional[torch.Tensor], out: torch.Tensor, ldo: int, m: int,
                            n: int, k: int, use_fast_accum: bool) -> None:
    """`f8b200_gemm_fp8_static_scratch`: dynamic tile scheduling with the scheduling words in the
    library's own static device array (at most 16 streams per device)."""
    _require_cuda(a, b, scale_a, scale_b, bias, out)
    with _Launch("gemm", a.device):
        _check(
            load().f8b200_gemm_fp8_static_scratch(a.data_ptr(), fp8_code(a.dtype), lda, b.data_ptr(),
                                                  fp8_code(b.dtype), ldb, scale_a.data_ptr(), scale_b.data_ptr(),
                                                  _ptr(bias), hp_code(out.dtype), out.data_ptr(), ldo, m, n, k,
                                                  int(use_fast_accum), _stream(a)),
            "f8b200_gemm_fp8_static_scratch",
        )


def rmsnorm_amax(x: torch.Tensor, rows: int, cols: int, ld: int, weight: torch.Tensor, eps: float,
                 rstd_out: torch.Tensor, amax_out: torch.Tensor) -> None:
    _require_cuda(x, weight, rstd_out, amax_out)
    with _Launch("norm_amax", x.device):
        _check(
            load().f8b200_rmsnorm_amax(x.data_ptr(), hp_code(x.dtype), rows, cols, ld, weight.data_ptr(), float(eps),
                                       rstd_out.data_ptr(), amax_out.data_ptr(), _stream(x)),
            "f8b200_rmsnorm_amax",
        )


def rmsnorm_cast(x: torch.Tensor, rows: int, cols: int, ld: int, weight: torch.Tensor, rstd: torch.Tensor,
                 amax: torch.Tensor, scale_out: Optional[torch.Tensor], out: torch.Tensor, ld_out: int) -> None:
    _require_cuda(x, weight, rstd, amax, scale_out, out)
    with _Launch("norm_cast", x.device):
        _check(
            load().f8b200_rmsnorm_cast(x.data_ptr(), hp_code(x.dtype), rows, cols, ld, weight.data_ptr(),
                                       rstd.data_ptr(), amax.data_ptr(), fp8_code(out.dtype), _ptr(scale_out),
                                       out.data_ptr(), ld_out, _stream(x)),
            "f8b200_rmsnorm_cast",
        )


def swiglu_amax(a: torch.Tensor, b: torch.Tensor, rows: int, cols: int, ld_a: int, ld_b: int,
                y_out: Optional[torch.Tensor], ld_y: int, amax_out: torch.Tensor, approx: bool = False) -> None:
    _require_cuda(a, b, y_out, amax_out)
    args = (a.data_ptr(), b.data_ptr(), hp_code(a.dtype), rows, cols, ld_a, ld_b, _ptr(y_out), ld_y,
            amax_out.data_ptr(), _stream(a))
    with _Launch("glu_amax", a.device):
        if approx:
            _check(load().f8b200_swiglu_amax_approx(*args), "f8b200_swiglu_amax_approx")
        else:
            _check(load().f8b200_swiglu_amax(*args), "f8b200_swiglu_amax")


def swiglu_cast(a: torch.Tensor, b: torch.Tensor, rows: int, cols: int, ld_a: int, ld_b: int, amax: torch.Tensor,
                scale_out: Optional[torch.Tensor], out: torch.Tensor, ld_out: int) -> None:
    _require_cuda(a, b, amax, scale_out, out)
    with _Launch("glu_cast", a.device):
        _check(
            load().f8b200_swiglu_cast(a.data_ptr(), b.data_ptr(), hp_code(a.dtype), rows, cols, ld_a, ld_b,
                                      amax.data_ptr(), fp8_code(out.dtype), _ptr(scale_out), out.data_ptr(), ld_out,
                                      _stream(a)),
            "f8b200_swiglu_cast",
        )


def cast_scatter(x: torch.Tensor, rows: int, cols: int, ld_x: int, amax: torch.Tensor, scale_out: torch.Tensor,
                 fp8_kind: int, out_ptrs: Sequence[int], ld_out: int) -> None:
    """Dynamic cast of `x` whose row-major bytes go to every address in `out_ptrs` (this
    device's own buffer and peer-mapped buffers of other devices)."""
    _require_cuda(x, amax, scale_out)
    arr = (ctypes.c_void_p * len(out_ptrs))(*[ctypes.c_void_p(p) for p in out_ptrs])
    with _Launch("cast", x.device):
        _check(
            load().f8b200_cast_scatter(x.data_ptr(), hp_code(x.dtype), rows, cols, ld_x, 1, amax.data_ptr(),
                                       scale_out.data_ptr(), 0, fp8_kind, arr, len(out_ptrs), ld_out, _stream(x)),
            "f8b200_cast_scatter",
        )


def rmsnorm_bwd(x: torch.Tensor, g: torch.Tensor, rows: int, cols: int, ld_x: int, ld_g: int, weight: torch.Tensor,
                rstd: torch.Tensor, dx: torch.Tensor, dweight: torch.Tensor) -> None:
    _require_cuda(x, g, weight, rstd, dx, dweight)
    nbytes = int(load().f8b200_rmsnorm_bwd_workspace_bytes(cols))
    ws = torch.empty(nbytes, dtype=torch.uint8, device=x.device)
    with _Launch("norm_bwd", x.device, 2):
        _check(
            load().f8b200_rmsnorm_bwd(x.data_ptr(), g.data_ptr(), hp_code(x.dtype), rows, cols, ld_x, ld_g,
                                      weight.data_ptr(), rstd.data_ptr(), dx.data_ptr(), cols, dweight.data_ptr(),
                                      ws.data_ptr(), nbytes, _stream(x)),
            "f8b200_rmsnorm_bwd",
        )


def swiglu_bwd(a: torch.Tensor, b: torch.Tensor, g: torch.Tensor, rows: int, cols: int, ld_a: int, ld_b: int,
               ld_g: int, da: torch.Tensor, db: torch.Tensor, approx: bool = False) -> None:
    _require_cuda(a, b, g, da, db)
    args = (a.data_ptr(), b.data_ptr(), g.data_ptr(), hp_code(a.dtype), rows, cols, ld_a, ld_b, ld_g, da.data_ptr(),
            db.data_ptr(), cols, _stream(a))
    with _Launch("glu_bwd", a.device):
        if approx:
            _check(load().f8b200_swiglu_bwd_approx(*args), "f8b200_swiglu_bwd_approx")
        else:
            _check(load().f8b200_swiglu_bwd(*args), "f8b200_swiglu_bwd")


def cast_blockwise(x: torch.Tensor, rows: int, cols: int, ld_x: int, fp8_kind: int, by_square: bool,
                   out_r: Optional[torch.Tensor], ld_r: int, scale_r: Optional[torch.Tensor], ld_scale_r: int,
                   exp_r: Optional[torch.Tensor], out_c: Optional[torch.Tensor], ld_c: int,
                   scale_c: Optional[torch.Tensor], ld_scale_c: int, exp_c: Optional[torch.Tensor]) -> None:
    _require_cuda(x, out_r, scale_r, exp_r, out_c, scale_c, exp_c)
    with _Launch("cast_block", x.device):
        _check(
            load().f8b200_cast_blockwise(x.data_ptr(), hp_code(x.dtype), rows, cols, ld_x, fp8_kind, int(by_square),
                                         _ptr(out_r), ld_r, _ptr(scale_r), ld_scale_r, _ptr(exp_r), _ptr(out_c), ld_c,
                                         _ptr(scale_c), ld_scale_c, _ptr(exp_c), _stream(x)),
            "f8b200_cast_blockwise",
        )


def uncast_blockwise(q: torch.Tensor, rows: int, cols: int, ld_q: int, scale: torch.Tensor, block_rows: int,
                     block_cols: int, y: torch.Tensor, ld_y: int) -> None:
    _require_cuda(q, scale, y)
    with _Launch("uncast_block", q.device):
        _check(
            load().f8b200_uncast_blockwise(q.data_ptr(), fp8_code(q.dtype), rows, cols, ld_q, scale.data_ptr(),
                                           scale.stride(0), scale.stride(1), block_rows, block_cols, hp_code(y.dtype),
                                           y.data_ptr(), ld_y, _stream(q)),
            "f8b200_uncast_blockwise",
        )


def gemm_blockwise(a: torch.Tensor, lda: int, a_mn_major: bool, scale_a: torch.Tensor, a_block_rows: int,
                   exp_a: Optional[torch.Tensor], b: torch.Tensor, ldb: int, b_mn_major: bool, scale_b: torch.Tensor,
                   b_block_rows: int, exp_b: Optional[torch.Tensor], bias: Optional[torch.Tensor], out: torch.Tensor, ldo: int, m: int, n: int, k: int) -> None:
    _require_cuda(a, b, scale_a, scale_b, exp_a, exp_b, bias, out)
    # more 256 x 256 tiles than CTA pairs are handed out through a word of memory; it belongs to this launch alone (a word per
    # stream would be shared by graphs captured on it that are replayed at the same time)
    ws = None
    if exp_a is not None and exp_b is not None and -(-m // 256) * -(-n // 256) > _sm_pairs(a.get_device()):
        ws = torch.empty(GEMM_WORKSPACE_BYTES, dtype=torch.uint8, device=a.device)
    with _Launch("gemm_block", a.device):
        _check(
            load().f8b200_gemm_blockwise(a.data_ptr(), fp8_code(a.dtype), int(a_mn_major), lda, scale_a.data_ptr(),
                                         scale_a.stride(0), scale_a.stride(1), a_block_rows, _ptr(exp_a), b.data_ptr(),
                                         fp8_code(b.dtype), int(b_mn_major), ldb, scale_b.data_ptr(), scale_b.stride(0),
                                         scale_b.stride(1), b_block_rows, _ptr(exp_b), _ptr(bias), hp_code(out.dtype), out.data_ptr(),
                                         ldo, m, n, k, _ptr(ws), GEMM_WORKSPACE_BYTES if ws is not None else 0,
                                         _stream(a)),
            "f8b200_gemm_blockwise",
        )


class BlockForm:
    """One form of a block-scaled cast at an address inside a caller's buffer: the fp8 bytes of [rows, cols], their factors
    and exponent bytes.  `by` is "row", "col" or "square"; as in `f8b200_cast_blockwise`.

    A training step holds nine of these tensors; as tensors of their own they would cost more host time than its
    launches."""

    __slots__ = ("rows", "cols", "by", "pitch", "data", "scale", "exps", "exps_t", "nbytes")

    def __init__(self, rows: int, cols: int, by: str):
        self.rows, self.cols, self.by, self.pitch = rows, cols, by, -(-cols // 16) * 16
        kb, rb = -(-cols // 128), -(-rows // 128)
        factors = kb * rows if by == "row" else rb * cols if by == "col" else rb * kb
        self.data = 0
        self.scale = -(-rows * self.pitch // 256) * 256
        at = self.scale + -(-4 * factors // 256) * 256
        as_rows, as_cols = -(-rows // 256) * 1024 * -(-cols // 512), -(-cols // 256) * 1024 * -(-rows // 512)
        self.exps = self.exps_t = None  # of the matrix and of its transpose, as operands
        if by != "col":
            self.exps, at = at, at + as_rows
        if by != "row":
            self.exps_t, at = at, at + as_cols
        self.nbytes = at  # a multiple of 256

    def at(self, base: int) -> "BlockForm":
        self.data, self.scale = base, self.scale + base
        self.exps = None if self.exps is None else self.exps + base
        self.exps_t = None if self.exps_t is None else self.exps_t + base
        return self

    def tensors(self, buf: torch.Tensor, start: int):
        """The form as tensors, views of the buffer `buf` (uint8) in which it lies from byte `start` on: (bytes, factors,
        exponent bytes as an operand by columns or transposed, otherwise by rows)."""
        kb, rb = -(-self.cols // 128), -(-self.rows // 128)
        shape = {"row": (kb, self.rows), "col": (rb, self.cols), "square": (rb, kb)}[self.by]
        exps, nbytes = (self.exps, -(-self.rows // 256) * 1024 * -(-self.cols // 512)) if self.by == "row" else \
            (self.exps_t, -(-self.cols // 256) * 1024 * -(-self.rows // 512))
        scale_at, exps_at = start + self.scale - self.data, start + exps - self.data
        data = buf[start:start + self.rows * self.pitch].view(self.rows, self.pitch)[:, : self.cols].view(torch.float8_e4m3fn)
        scale = buf[scale_at:scale_at + 4 * shape[0] * shape[1]].view(torch.float32).view(shape)
        return data, scale.t() if self.by == "row" else scale, buf[exps_at:exps_at + nbytes]

    def operand(self, transposed: bool = False):
        """(address, MN-major, pitch, factors, row stride, k-block stride, rows per factor, exponents) for the GEMM."""
        if self.by == "square":
            strides = (1, -(-self.cols // 128)) if transposed else (-(-self.cols // 128), 1)
            return (self.data, int(transposed), self.pitch, self.scale, *strides, 128, self.exps_t if transposed else self.exps)
        if transposed != (self.by == "col"):
            raise F8B200Error(f"a cast by {self.by} serves the {'matrix' if transposed else 'transpose'} only")
        return (self.data, int(transposed), self.pitch, self.scale, 1, self.cols if transposed else self.rows, 1,
                self.exps_t if transposed else self.exps)


def block_cast_into(x: torch.Tensor, ld_x: int, row: Optional[BlockForm], col: Optional[BlockForm]) -> None:
    """`f8b200_cast_blockwise` of the e4m3 forms `row` (or a square one) and `col` of one matrix."""
    first = row or col
    square = first.by == "square"
    r = (row.data, row.pitch, row.scale, -(-row.cols // 128) if square else row.rows, row.exps) if row else (None, 0, None, 0, None)
    c = (col.data, col.pitch, col.scale, col.cols, col.exps_t) if col else (None, 0, None, 0, row.exps_t if square else None)
    _require_cuda(x)
    with _Launch("cast_block", x.device):
        _check(
            load().f8b200_cast_blockwise(x.data_ptr(), hp_code(x.dtype), first.rows, first.cols, ld_x, E4M3, int(square), *r, *c,
                                         _stream(x)),
            "f8b200_cast_blockwise",
        )


def block_gemm_into(a, b, bias: Optional[torch.Tensor], out: torch.Tensor, m: int, n: int, k: int, ws: int) -> None:
    """`f8b200_gemm_blockwise` of two e4m3 `BlockForm.operand`s; `ws`: the address of a scheduling word or 0."""
    _require_cuda(bias, out)
    with _Launch("gemm_block", out.device):
        _check(
            load().f8b200_gemm_blockwise(a[0], E4M3, a[1], a[2], a[3], a[4], a[5], a[6], a[7], b[0], E4M3, b[1], b[2], b[3], b[4],
                                         b[5], b[6], b[7], _ptr(bias), hp_code(out.dtype), out.data_ptr(), n, m, n, k,
                                         ws or None, GEMM_WORKSPACE_BYTES if ws else 0, _stream(out)),
            "f8b200_gemm_blockwise",
        )


def linear_blockwise(x: torch.Tensor, m: int, k: int, ld_x: int, weight: torch.Tensor, ldw: int, w_mn_major: bool,
                     weight_scale: torch.Tensor, bias: Optional[torch.Tensor], out: torch.Tensor, n: int) -> None:
    """out [m, n] = x [m, k] cast by rows, times the transpose of an fp8 weight with one factor per 128 x 128: the cast
    and the product (`f8b200_cast_blockwise`, `f8b200_gemm_blockwise`) with the cast's bytes and factors in one
    scratch buffer.  Few rows leave the GPU waiting for the host, so this is as little host work as the two need."""
    _require_cuda(x, weight, weight_scale, bias, out)
    pitch = -(-k // 16) * 16
    data_bytes = -(-m * pitch // 16) * 16
    scratch = torch.empty(data_bytes + 4 * m * -(-k // 128), dtype=torch.uint8, device=x.device)
    data, stream = scratch.data_ptr(), _stream(x)
    scale = data + data_bytes  # [k-block][row]
    lib = load()
    with _Launch("gemm_block", x.device, 2):
        _check(lib.f8b200_cast_blockwise(x.data_ptr(), hp_code(x.dtype), m, k, ld_x, E4M3, 0, data, pitch, scale, m, None,
                                         None, 0, None, 0, None, stream), "f8b200_cast_blockwise")
        _check(lib.f8b200_gemm_blockwise(data, E4M3, 0, pitch, scale, 1, m, 1, None, weight.data_ptr(),
                                         fp8_code(weight.dtype), int(w_mn_major), ldw, weight_scale.data_ptr(),
                                         weight_scale.stride(0), weight_scale.stride(1), 128, None, _ptr(bias),
                                         hp_code(out.dtype), out.data_ptr(), n, m, n, k, None, 0, stream),
               "f8b200_gemm_blockwise")


def layer_norm(x: torch.Tensor, rows: int, cols: int, ld_x: int, weight: Optional[torch.Tensor],
               bias: Optional[torch.Tensor], affine_dtype: torch.dtype, eps: float, y: torch.Tensor,
               mean: Optional[torch.Tensor], rstd: Optional[torch.Tensor]) -> None:
    _require_cuda(x, weight, bias, y, mean, rstd)
    with _Launch("layer_norm", x.device):
        _check(
            load().f8b200_layer_norm(x.data_ptr(), hp_code(x.dtype), rows, cols, ld_x, _ptr(weight), _ptr(bias),
                                     hp_code(affine_dtype), float(eps), y.data_ptr(), cols, _ptr(mean), _ptr(rstd),
                                     _stream(x)),
            "f8b200_layer_norm",
        )


def layer_norm_bwd(x: torch.Tensor, g: torch.Tensor, rows: int, cols: int, ld_x: int, ld_g: int,
                   weight: Optional[torch.Tensor], affine_dtype: torch.dtype, mean: torch.Tensor, rstd: torch.Tensor,
                   dx: Optional[torch.Tensor], dw: Optional[torch.Tensor], db: Optional[torch.Tensor]) -> None:
    _require_cuda(x, g, weight, mean, rstd, dx, dw, db)
    nbytes = int(load().f8b200_layer_norm_bwd_workspace_bytes(cols)) if dw is not None or db is not None else 0
    ws = torch.empty(nbytes, dtype=torch.uint8, device=x.device) if nbytes else None
    with _Launch("layer_norm_bwd", x.device, (1 if dx is not None else 0) + (2 if nbytes else 0)):
        _check(
            load().f8b200_layer_norm_bwd(x.data_ptr(), g.data_ptr(), hp_code(x.dtype), rows, cols, ld_x, ld_g,
                                         _ptr(weight), hp_code(affine_dtype), mean.data_ptr(), rstd.data_ptr(), _ptr(dx),
                                         cols, _ptr(dw), _ptr(db), _ptr(ws), nbytes, _stream(x)),
            "f8b200_layer_norm_bwd",
        )


class TensorArrays:
    """Addresses, sizes and types of dense CUDA tensors of one device as the multi-tensor entry points take them."""

    __slots__ = ("n", "ptrs", "numels", "codes", "device")

    def __init__(self, xs: Sequence[torch.Tensor]):
        # hundreds of tensors per call: every pass over them is a C-level map
        n = self.n = len(xs)
        T = torch.Tensor
        devices = set(map(T.get_device, xs))
        if len(devices) > 1:
            raise F8B200Error(f"tensors on different devices ({', '.join(sorted({str(t.device) for t in xs}))})")
        if -1 in devices:
            raise F8B200Error("f8b200 kernels run on CUDA tensors only (no CPU path exists)")
        self.device = xs[0].device if n else None
        dtypes = [t.dtype for t in xs]
        codes = {dtype: hp_code(dtype) for dtype in set(dtypes)}
        self.ptrs = (ctypes.c_void_p * n).from_buffer(array("Q", map(T.data_ptr, xs))) if n else None
        self.numels = (ctypes.c_int64 * n).from_buffer(array("q", map(T.numel, xs))) if n else None
        self.codes = (ctypes.c_int * n).from_buffer(array("i", map(codes.__getitem__, dtypes))) if n else None


MULTI_TENSORS_PER_LAUNCH = 1024  # tensors whose addresses fit one launch's parameters (csrc/grad_clip.cu)


def multi_norm(xs: TensorArrays, kind: int, root: bool, out: torch.Tensor) -> None:
    """`f8b200_multi_norm` over dense tensors of one device, each taken as its storage lies."""
    n = xs.n
    _require_cuda(out)
    nbytes = int(load().f8b200_multi_norm_workspace_bytes(xs.numels, n))
    ws = torch.empty(nbytes, dtype=torch.uint8, device=out.device) if nbytes else None
    with _Launch("multi_norm", out.device, 1 + -(-n // MULTI_TENSORS_PER_LAUNCH)):
        _check(load().f8b200_multi_norm(xs.ptrs, xs.numels, xs.codes, n, kind, int(root), out.data_ptr(), _ptr(ws), nbytes,
                                        _stream(out)), "f8b200_multi_norm")


def multi_clip(xs: TensorArrays, total_norm: torch.Tensor, max_norm: float) -> None:
    n = xs.n
    _require_cuda(total_norm)
    with _Launch("multi_clip", total_norm.device, -(-n // MULTI_TENSORS_PER_LAUNCH)):
        try:
            _check(load().f8b200_multi_clip(xs.ptrs, xs.numels, xs.codes, n, total_norm.data_ptr(), float(max_norm),
                                            _stream(total_norm)), "f8b200_multi_clip")
        except F8B200Error as e:
            if e.status != ERR_BAD_ARG:
                raise
            # the only bad argument that tensors can be
            raise F8B200Error("f8b200_multi_clip: tensors that overlap in memory cannot be scaled together") from None


def check_device_error() -> None:
    """Raises F8B200Error (F8B200_ERR_TIMEOUT) when a bounded wait inside a GEMM kernel gave up
    since the last poll: the outputs of those launches are undefined.  Synchronises the device, so
    call it where the program synchronises anyway (the end of a step, a benchmark's timed region).
    With F8B200_POLL_ERRORS=1 in the environment `sync_float8_amax_and_scale_history` and
    `precompute_float8_dynamic_scale_for_fsdp` poll it once per call."""
    flags = read_device_error()
    if flags != 0:
        raise F8B200Error(f"device error word {flags:#x}: " + load().f8b200_status_string(-7).decode())


def poll_errors_if_enabled() -> None:
    if os.environ.get("F8B200_POLL_ERRORS", "0") == "1" and torch.cuda.is_available():
        check_device_error()


def read_device_error() -> int:
    v = ctypes.c_uint32(0)
    _check(load().f8b200_read_device_error(ctypes.byref(v)), "f8b200_read_device_error")
    flags = int(v.value)
    if _mc_lib is not None:  # the multicast library keeps an error word of its own
        w = ctypes.c_uint32(0)
        if _mc_lib.f8b200_mc_read_device_error(ctypes.byref(w)) == 0:
            flags |= int(w.value)
    return flags
