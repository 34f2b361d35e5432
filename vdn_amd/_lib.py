"""ctypes binding of libvdnmi.so, the C-ABI library of hand-written gfx950 kernels.

torch is imported first on purpose: its bundled HIP runtime carries the same SONAME
(libamdhip64.so.7) that libvdnmi.so links against, so the library binds to the runtime
that owns torch's device memory and streams.

There is no fallback. A missing or stale library raises RuntimeError, and every nonzero
status from the library raises RuntimeError with the library's own message.
"""
from __future__ import annotations

import ctypes
import os
import threading

import torch
import numpy as np

LIBRARY_PATH = os.path.join(os.path.dirname(os.path.abspath(__file__)), "libvdnmi.so")

_i64 = ctypes.c_int64
_i32 = ctypes.c_int
_f32 = ctypes.c_float
_ptr = ctypes.c_void_p

# name -> argtypes; every entry point returns int status.
SIGNATURES = {
    "vdn_mxfp8_quantize": [_ptr, _i64, _i64, _i64, _ptr, _ptr, _ptr, _ptr],
    "vdn_mxfp8_act_quantize": [_ptr, _i64, _i64, _i64, _i32, _ptr, _ptr, _ptr, _ptr, _ptr],
    "vdn_mxfp8_prenorm_quantize": [_ptr, _i64, _i64, _i64, _ptr, _f32, _ptr, _i64, _ptr, _i64,
                                   _ptr, _i32, _ptr, _ptr, _ptr, _ptr, _ptr],
    "vdn_mxfp8_gemm": [_ptr, _ptr, _i64, _ptr, _ptr, _i64, _i64, _ptr, _ptr, _i64, _ptr, _i64,
                       _ptr, _ptr, _i64, _i64, _i64, _ptr, _ptr],
    "vdn_mxfp8_gemm_act_quantize": [_ptr, _ptr, _i64, _ptr, _ptr, _i64, _i64, _ptr, _i32, _ptr,
                                    _ptr, _i64, _i64, _ptr, _ptr],
    "vdn_mxfp8_gemm_ws": [_ptr, _ptr, _i64, _ptr, _ptr, _i64, _i64, _ptr, _ptr, _i64, _ptr, _i64,
                          _ptr, _ptr, _i64, _i64, _i64, _ptr, _ptr, _i64, _ptr],
    "vdn_mxfp8_gemm_act_quantize_ws": [_ptr, _ptr, _i64, _ptr, _ptr, _i64, _i64, _ptr, _i32, _ptr,
                                       _ptr, _i64, _i64, _ptr, _ptr, _i64, _ptr],
    "vdn_mxfp8_gemm_workspace": [_i64, _i64, _i64, _i32, _ptr],
    "vdn_mxfp8_gemm_plan": [_i64, _i64, _i64, _i32, _ptr, _ptr],
    "vdn_vda_prepare": [_ptr, _i64, _i32, _i64, _i64, _i32, _i32, _i32, _i32, _ptr, _ptr],
    "vdn_vda_conv_prepare": [_ptr, _i32, _i64, _i64, _i32, _i32, _i32, _ptr, _ptr, _i32, _ptr,
                             _ptr],
    "vdn_vda_statistics": [_ptr, _i64, _i64, _i64, _ptr, _i64, _i64, _i64, _ptr, _i64, _i64, _i64,
                           _i32, _i32, _i32, _i32, _i32, _ptr, _ptr, _ptr],
    "vdn_vda_factors": [_ptr, _ptr, _ptr, _i64, _ptr, _ptr, _ptr],
    "vdn_vda_compose": [_ptr, _ptr, _i32, _ptr, _ptr, _i32, _ptr, _ptr, _ptr],
    "vdn_vda_scan": [_ptr, _ptr, _ptr, _i32, _i32, _i32, _ptr, _ptr],
    "vdn_vda_chunk_scan": [_ptr, _ptr, _ptr, _i32, _i32, _ptr, _ptr, _i32, _ptr, _ptr],
    "vdn_vda_log_prefix": [_ptr, _i32, _i32, _ptr, _ptr],
    "vdn_vda_gather": [_ptr, _ptr, _ptr, _ptr, _ptr, _ptr, _ptr, _ptr, _ptr, _ptr, _i32, _i32,
                       _i32, _i32, _ptr, _ptr],
    "vdn_vda_readout": [_ptr, _i64, _i64, _i64, _i32, _ptr, _ptr, _i32, _f32, _ptr, _i64, _i64,
                        _i64, _ptr, _i64, _i64, _i64, _i32, _i32, _i32, _i32, _ptr],
    "vdn_vda_epilogue": [_ptr, _ptr, _i32, _f32, _ptr, _i64, _i64, _i64, _ptr, _i64, _i64, _i64,
                         _i32, _i32, _i32, _i32, _ptr],
    "vdn_qk_rmsnorm_rope": [_ptr, _i64, _i64, _i64, _ptr, _i64, _i64, _i64, _ptr, _i64, _ptr,
                            _i64, _f32, _ptr, _i64, _i64, _ptr, _i64, _i64, _i32, _i32, _i64,
                            _i32, _i32, _ptr, _ptr, _ptr],
    "vdn_rotary": [_ptr, _i64, _i64, _ptr, _i64, _i64, _ptr, _ptr, _i32, _f32, _ptr, _i32, _ptr,
                   _i32, _i32, _f32, _i64, _i32, _i32, _i32, _i32, _ptr, _i64, _i64, _ptr, _i64,
                   _i64, _ptr],
    "vdn_window_attention": [_ptr, _i64, _i64, _ptr, _i64, _i64, _ptr, _i64, _i64, _ptr, _i32,
                             _ptr, _ptr, _i32, _i32, _i32, _f32, _ptr, _i64, _i64, _ptr, _i64,
                             _i64, _ptr, _i64, _i64, _ptr],
    "vdn_window_attention_mxfp8": [_ptr, _i64, _i64, _ptr, _i64, _i64, _ptr, _i64, _i64, _ptr,
                                   _i32, _ptr, _ptr, _i32, _f32, _ptr, _i64, _i64, _ptr, _f32,
                                   _ptr, _ptr, _i64, _i32, _ptr],
    "vdn_causal_attention": [_ptr, _i64, _i64, _ptr, _i64, _i64, _ptr, _i64, _i64, _ptr, _i32,
                             _i32, _i32, _i32, _i32, _i32, _f32, _ptr, _i64, _i64, _ptr, _i64,
                             _i64, _ptr],
    "vdn_cache_write": [_ptr, _ptr, _ptr, _ptr, _ptr, _i32, _i32, _i32, _i32, _ptr, _i64, _i32,
                        _i32, _ptr, _ptr, _ptr, _i64, _i64, _ptr, _i64, _i64, _i32, _i32, _ptr],
    "vdn_cache_read": [_ptr, _ptr, _ptr, _ptr, _ptr, _i32, _i32, _i32, _i32, _ptr, _i64, _i32,
                       _i32, _ptr, _ptr, _ptr, _i64, _i64, _ptr, _i64, _i64, _i32, _i32, _ptr],
    "vdn_cache_attention": [_ptr, _i64, _i64, _i64, _ptr, _ptr, _ptr, _ptr, _ptr, _i32, _i32,
                            _i32, _i32, _ptr, _i64, _i32, _i32, _ptr, _i32, _i32, _i32, _f32,
                            _ptr, _i64, _i64, _i64, _ptr, _ptr, _i64, _ptr],
    "vdn_cache_attention_workspace": [_i32, _i32, _i32, _ptr],
    "vdn_cache_attention_heads": [_ptr, _i64, _i64, _ptr, _ptr, _ptr, _ptr, _ptr, _i32, _i32, _i32,
                                  _i32, _ptr, _i64, _i64, _i32, _i32, _ptr, _i32, _i32, _f32, _ptr,
                                  _i64, _i64, _ptr, _ptr, _i64, _ptr],
    "vdn_cache_means": [_ptr, _ptr, _ptr, _i32, _i32, _i32, _i32, _ptr, _i64, _i32, _i32, _ptr,
                        _ptr, _ptr, _ptr],
    "vdn_cache_select": [_ptr, _i64, _i64, _i64, _ptr, _ptr, _i32, _i32, _i32, _i32, _ptr, _i64,
                         _i32, _i32, _ptr, _i32, _i32, _i32, _i32, _i32, _i32, _ptr, _ptr, _ptr,
                         _i64, _ptr],
    "vdn_cache_select_workspace": [_i32, _i32, _i32, _i32, _ptr],
    "vdn_prefix_attention": [_ptr, _i64, _i64, _i64, _ptr, _ptr, _ptr, _ptr, _ptr, _i32, _i32, _i32,
                             _i32, _ptr, _i64, _i32, _ptr, _i32, _i32, _ptr, _ptr, _i64, _i32, _i32, _ptr,
                             _i32, _i32, _i32, _f32, _ptr, _i64, _i64, _i64, _ptr, _ptr, _i64, _ptr],
    "vdn_prefix_attention_workspace": [_i32, _i32, _i32, _i32, _i32, _i32, _i32, _i32, _ptr],
    "vdn_vda_readout_mxfp8": [_ptr, _i64, _i64, _i64, _i32, _ptr, _ptr, _i32, _f32, _ptr, _i64,
                              _i64, _i64, _ptr, _ptr, _i64, _i32, _i32, _i32, _i32, _ptr],
    "vdn_vda_readout_gated": [_ptr, _i64, _i64, _i64, _i32, _ptr, _ptr, _i32, _f32, _ptr, _i64,
                              _ptr, _ptr, _ptr, _i64, _i64, _i64, _ptr, _ptr, _i64, _i32, _i32,
                              _i32, _i32, _ptr],
    "vdn_gate_projection": [_ptr, _i64, _i64, _ptr, _i32, _i32, _i32, _ptr, _ptr, _ptr, _ptr,
                            _ptr, _ptr],
    "vdn_frame_alpha": [_ptr, _i32, _i32, _ptr, _ptr, _ptr, _i32, _i32, _ptr, _ptr],
    "vdn_adaln_tables": [_ptr, _i32, _i64, _i32, _i64, _ptr, _ptr, _i64, _ptr, _i64, _ptr],
}

_LOCK = threading.Lock()
_LIB = None


def load() -> ctypes.CDLL:
    """Loads libvdnmi.so once; raises RuntimeError when it has not been built."""
    global _LIB
    if _LIB is not None:
        return _LIB
    with _LOCK:
        if _LIB is None:
            if not os.path.exists(LIBRARY_PATH):
                raise RuntimeError(
                    f"{LIBRARY_PATH} is missing: build it with `python -c 'import __graft_entry__ "
                    "as g; g.build()'` (hipcc, gfx950). There is no non-HIP fallback.")
            lib = ctypes.CDLL(LIBRARY_PATH)
            lib.vdn_last_error.restype = ctypes.c_char_p
            lib.vdn_last_error.argtypes = []
            lib.vdn_abi_version.restype = ctypes.c_int
            for name, args in SIGNATURES.items():
                fn = getattr(lib, name)
                fn.argtypes = args
                fn.restype = ctypes.c_int
            _LIB = lib
    return _LIB


def exported_symbols() -> list[str]:
    return ["vdn_last_error", "vdn_abi_version", *SIGNATURES]


class LaunchTimer:
    """Records a pair of timing events around every call of the named entry points while
    active (`with LaunchTimer({...}) as t:`). The events go on the caller's current stream,
    the stream every entry point launches on, so each pair brackets that launch; the stream's
    handle is kept with them."""

    def __init__(self, names):
        self.names = set(names)
        self.records = []

    def __enter__(self):
        _TIMERS.append(self)
        return self

    def __exit__(self, *exc):
        _TIMERS.remove(self)

    def durations(self):
        """[(name, args, milliseconds, stream handle)] after synchronising the device."""
        torch.cuda.synchronize()
        return [(n, a, s.elapsed_time(e), h) for n, a, s, e, h in self.records]


_TIMERS: list[LaunchTimer] = []


def call(name: str, *args) -> None:
    lib = load()
    timers = [t for t in _TIMERS if name in t.names] if _TIMERS else None
    if timers:
        start = torch.cuda.Event(enable_timing=True)
        start.record()
    status = getattr(lib, name)(*args)
    if status != 0:
        raise RuntimeError(f"{name} failed ({status}): {lib.vdn_last_error().decode()}")
    if timers:
        end = torch.cuda.Event(enable_timing=True)
        end.record()
        handle = torch.cuda.current_stream().cuda_stream
        for t in timers:
            t.records.append((name, args, start, end, handle))


def ptr(t: torch.Tensor | None) -> int | None:
    return None if t is None else t.data_ptr()


def stream(device: torch.device) -> int:
    """The caller's current HIP stream on `device` (launches never go to a private stream)."""
    if device.type != "cuda":
        raise ValueError(f"expected a CUDA (HIP) device, but got {device}")
    index = device.index
    return torch._C._cuda_getCurrentRawStream(torch.cuda.current_device() if index is None
                                              else index)


def call_on(device_index: int, name: str, *args) -> None:
    """call() with device `device_index` as the current one: a launch goes to the current device,
    whatever its stream's is."""
    if device_index != torch._C._cuda_getDevice():
        with torch.cuda.device(device_index):
            return call(name, *args)
    if _TIMERS:
        return call(name, *args)
    lib = _LIB or load()
    status = getattr(lib, name)(*args)
    if status != 0:
        raise RuntimeError(f"{name} failed ({status}): {lib.vdn_last_error().decode()}")


def raw_stream(device_index: int) -> int:
    """stream() by device index."""
    return torch._C._cuda_getCurrentRawStream(device_index)


def require_gpu(t: torch.Tensor, what: str) -> None:
    if t.device.type != "cuda":
        raise ValueError(f"{what} must be a CUDA (HIP) tensor")


def _reach(t: torch.Tensor, first_dim: int = 0) -> int:
    """Elements from a view's first one up to behind its last one, of its dimensions from first_dim on."""
    return 1 + sum((n - 1) * s for n, s in zip(t.shape[first_dim:], t.stride()[first_dim:]))


def _starts(t: torch.Tensor, dims) -> np.ndarray:
    """Where the runs of a view's last dimension begin, over the given dimensions."""
    at = np.zeros(1, dtype=np.int64)
    for i in dims:
        at = (at[:, None] + t.stride(i) * np.arange(t.shape[i])).ravel()
    return at


def overlaps_itself(t: torch.Tensor) -> bool:
    """Whether elements of a view (unit last stride) share memory."""
    reach = 1
    for s, n in sorted((s, n) for n, s in zip(t.shape, t.stride()) if n > 1):
        if s < reach:       # its dimensions do not nest, as those of slices of a dense tensor do
            return bool((np.diff(np.sort(_starts(t, range(t.ndim - 1)))) < t.shape[-1]).any())
        reach += (n - 1) * s
    return False


def overlap(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether two views of rows (unit last stride, as long in both) share memory. Where that would be
    long to tell (rows of different strides in ranges that cross, rows of very many interleaved
    runs) they are taken not to."""
    if a.numel() == 0 or b.numel() == 0:
        return False
    apart = (b.data_ptr() - a.data_ptr()) // a.element_size()
    if apart >= _reach(a) or -apart >= _reach(b):
        return False
    row = a.stride(0)
    if b.stride(0) != row or row == 0:
        return False
    wide_a, wide_b, column = _reach(a, 1), _reach(b, 1), apart % row
    if column >= wide_a and column + wide_b <= row:     # slices beside each other
        return False
    # runs that lie less than a run's length apart, in some row of a and the k-th one behind it in b
    dims = range(1, a.ndim - 1)
    if a[0].numel() * b[0].numel() > a.shape[-1] ** 2 << 20:
        return False
    delta = apart + _starts(b, dims)[None] - _starts(a, dims)[:, None]
    k = -((delta + a.shape[-1] - 1) // row)             # the least k with delta + k row > -length
    k = np.maximum(k, 1 - a.shape[0])
    return bool(((delta + k * row < a.shape[-1]) & (k < b.shape[0])).any())


def check_attention_out(out: torch.Tensor, query: torch.Tensor, *sources: torch.Tensor) -> None:
    """Refuses a caller's `out` whose elements share memory, or that lies over what other workgroups
    still read: the sources, or the query unless it is the query itself (a workgroup writes the
    rows that it has read)."""
    if not out.is_contiguous() and overlaps_itself(out):
        raise ValueError("out must not overlap itself")
    storage = out.untyped_storage().data_ptr()
    for x in sources:
        if x.untyped_storage().data_ptr() == storage and overlap(out, x):
            raise ValueError("out must not overlap key or value")
    if query.untyped_storage().data_ptr() == storage \
            and (out.data_ptr() != query.data_ptr() or out.stride() != query.stride()) \
            and overlap(out, query):
        raise ValueError("out may be the query itself, but must not overlap it otherwise")
