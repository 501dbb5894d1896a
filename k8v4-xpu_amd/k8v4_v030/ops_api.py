"""ctypes boundary into the gfx950 HIP library (``libk8v4_hip.so``).

``ops()`` returns an object whose methods carry the names and argument orders
of the reference's ``torch.ops.xe2_kv`` ops (k8v4_v030/ops_api.py:14-25,
native/xe2_kv_ops.cpp:1779-1822), so callers written against the reference
keep working.  Each method validates its tensors the way the reference's
``TORCH_CHECK``s do (dtypes, ranks, within-page strides, the 2-or-4 head
rule, with the same messages) and then passes raw device pointers, sizes and
the current HIP stream to the C ABI declared in ``include/k8v4_abi.h``.
Errors come back as ``RuntimeError``.  There is no fallback: a missing
library raises ``FileNotFoundError`` and a CPU tensor raises.
"""
from __future__ import annotations

import ctypes
import os
from pathlib import Path

import torch

from .layout import GQA, PAGE

_DEFAULT_LIB = Path(__file__).resolve().parent / "libk8v4_hip.so"
_LIB = None
_LOADED: str | None = None
_OPS = None

F16, BF16, F32 = 0, 1, 2
_DTYPE_CODE = {torch.float16: F16, torch.bfloat16: BF16, torch.float32: F32}

_i64 = ctypes.c_int64
_i32 = ctypes.c_int
_vp = ctypes.c_void_p


def library_path() -> str:
    """``K8V4_HIP_LIB`` if set, else the in-tree build."""
    return os.environ.get("K8V4_HIP_LIB", str(_DEFAULT_LIB))


def _declare(lib: ctypes.CDLL) -> None:
    lib.k8v4_abi_version.restype = _i32
    lib.k8v4_abi_version.argtypes = []
    lib.k8v4_last_error.restype = ctypes.c_char_p
    lib.k8v4_last_error.argtypes = []
    lib.k8v4_kv_store_paged.restype = _i32
    lib.k8v4_kv_store_paged.argtypes = [
        _vp, _vp, _i32, _i64, _i64, _vp, _i64, _i32, _i32,
        _vp, _vp, _vp, _vp, _vp,
        _i64, _i64, _i64, _i64, _i64, _i64, _vp,
    ]
    for name, argtypes, restype in _EXTRA_SYMBOLS:
        fn = getattr(lib, name)
        fn.argtypes = argtypes
        fn.restype = restype


# Entry points beyond the store: (name, argtypes, restype).
_EXTRA_SYMBOLS: list[tuple[str, list, object]] = [
    (
        "k8v4_attn_batch",
        [_vp, _i32, _i64, _vp, _vp, _vp, _vp, _vp, _i64, _i64, _i64, _i64, _i64, _i64,
         _vp, _i64, _i64, _i32, _vp, _vp, _i64, _i64, _i32, _i32, _i32,
         _vp, _i32, _i64, _vp, _i64, _i32, _vp],
        _i32,
    ),
    ("k8v4_attn_workspace_bytes", [_i64, _i64, _i32, _i32, _i32, _i32, _i32], _i64),
]
_EXTRA_SYMBOLS.append(("k8v4_attn_batch_profiled", _EXTRA_SYMBOLS[0][1] + [_vp, _i32], _i32))
_EXTRA_SYMBOLS.append((
    "k8v4_prefill_paged",
    [_vp, _i32, _i64, _vp, _vp, _vp, _vp, _vp, _i64, _i64, _i64, _i64, _i64, _i64,
     _vp, _i64, _i32, _i64, _i64, _i32, _i32, ctypes.c_float, _vp, _i32, _i64, _vp, _i64, _vp],
    _i32,
))
_EXTRA_SYMBOLS.append(("k8v4_prefill_workspace_bytes", [_i64, _i64, _i32, _i32], _i64))
_EXTRA_SYMBOLS.append(("k8v4_prefill_uses_tiles", [_i64, _i64, _i32, _i32], _i32))
_EXTRA_SYMBOLS.append((
    "k8v4_prefill_paged_batch",
    [_vp, _i32, _i64, _vp, _vp, _vp, _vp, _vp, _i64, _i64, _i64, _i64, _i64, _i64,
     _vp, _i64, _i64, _i32, _i32, _vp, _vp, _vp, _vp, _i32, _i32, ctypes.c_float, _vp, _i32, _i64, _vp, _i64, _vp],
    _i32,
))
_EXTRA_SYMBOLS.append(("k8v4_prefill_batch_workspace_bytes", [_i32, _i32], _i64))
_EXTRA_SYMBOLS.append(("k8v4_k_store_paged", [_vp, _i32, _i64, _vp, _i64, _i32, _i32, _vp, _vp, _i64, _i64, _i64, _vp],
                       _i32))
_EXTRA_SYMBOLS.append(("k8v4_v_store_paged",
                       [_vp, _i32, _i64, _vp, _i64, _i32, _i32, _vp, _vp, _vp, _i64, _i64, _i64, _i64, _vp], _i32))
_EXTRA_SYMBOLS.append(("k8v4_q_quant", [_vp, _i32, _i32, _i64, _i64, _i32, _i32, _vp, _vp, _vp], _i32))
_EXTRA_SYMBOLS.append((
    "k8v4_attn_batch_q8",
    [_vp, _vp, _i64, _i64, _vp, _vp, _vp, _vp, _vp, _i64, _i64, _i64, _i64, _i64, _i64,
     _vp, _i64, _i64, _i32, _vp, _vp, _i64, _i64, _i32, _i32, _i32,
     _vp, _i32, _i64, _vp, _i64, _i32, _vp],
    _i32,
))
_EXTRA_SYMBOLS.append(("k8v4_attn_batch_noalloc", _EXTRA_SYMBOLS[0][1][:28] + [_i32, _vp], _i32))
_EXTRA_SYMBOLS.append(("k8v4_attn_noalloc_max_bytes", [], _i64))
_EXTRA_SYMBOLS.append(("k8v4_decode_fault_count", [], _i64))
_EXTRA_SYMBOLS.append((
    "k8v4_kv_load_paged",
    [_vp, _vp, _vp, _vp, _vp, _i64, _i64, _i64, _i64, _i64, _i64,
     _vp, _i64, _i64, _i32, _vp, _vp, _i64, _i32, _i32, _vp, _vp, _i32, _i64, _i64, _i64, _vp],
    _i32,
))
_EXTRA_SYMBOLS.append((
    "k8v4_attn_shared",
    [_vp, _i32, _i64, _vp, _vp, _vp, _vp, _vp, _i64, _i64, _i64, _i64, _i64, _i64,
     _vp, _i64, _i64, _vp, _i64, _i64, _i32, _vp, _i64, _i32, _i32, _i32, _vp, _i32, _i64, _vp, _i64, _vp],
    _i32,
))
_EXTRA_SYMBOLS.append(("k8v4_attn_shared_workspace_bytes", [_i64, _i32, _i32, _i32], _i64))
_EXTRA_SYMBOLS.append(("k8v4_attn_shared_many_rows", [_i64, _i32, _i32, _i32, _i64], _i32))
_EXTRA_SYMBOLS.append((
    "k8v4_verify_drafts",
    [_vp, _i32, _i64, _i64, _vp, _i64, _i64, _vp, _i32, _i64, _vp, _vp, _i64, _vp, _vp,
     _i64, _i32, _i64, _vp, _i64, _vp, _vp, _vp, _i64, _vp],
    _i32,
))
_EXTRA_SYMBOLS.append(("k8v4_verify_drafts_workspace_bytes", [_i64, _i64], _i64))
_CACHE = [_vp, _vp, _vp, _vp, _vp, _i64, _i64, _i64, _i64, _i64, _i64]
_EXTRA_SYMBOLS.append((
    "k8v4_rope_kv_store_paged",
    [_vp, _vp, _vp, _i32, _i64, _i64, _i64, _vp, _i32, _vp, _i32, _i64, _i64, _i32, _i32, _vp, _i64, _i32, _i32,
     *_CACHE, _vp, _i64, _vp],
    _i32,
))
_EXTRA_SYMBOLS.append((
    "k8v4_attn_tree",
    [_vp, _i32, _i64, *_CACHE, _vp, _i64, _i64, _i32, _vp, _vp, _i64, _i64, _i32, _i32, _i32, _vp, _i32, _i64,
     _vp, _i64, _vp],
    _i32,
))
_EXTRA_SYMBOLS.append(("k8v4_attn_tree_workspace_bytes", [_i64, _i32, _i32, _i32], _i64))
_EXTRA_SYMBOLS.append((
    "k8v4_accept_tree",
    [_vp, _i32, _i64, _vp, _i64, _vp, _vp, _i64, _vp, _i64, _i32, _i32, _vp, _i64, _vp, _i64, _vp, _vp, _vp],
    _i32,
))
_EXTRA_SYMBOLS.append((
    "k8v4_kv_keep_paged",
    [*_CACHE, _vp, _i64, _i64, _i32, _vp, _vp, _i64, _i32, _vp, _i64, _i32, _i32, _vp],
    _i32,
))
_EXTRA_SYMBOLS.append((
    "k8v4_token_logprobs",
    [_vp, _i32, _i64, _vp, _i32, _i64, _i64, _i32, _vp, _vp, _vp, _vp, _i64, _vp, _i64, _vp, _i64, _vp],
    _i32,
))
_EXTRA_SYMBOLS.append(("k8v4_token_logprobs_workspace_bytes", [_i64, _i64, _i32], _i64))
Q_TOKENS, Q_PADDED = 0, 1


def load_library():
    """Load the shared library once per process (path from :func:`library_path`)."""
    global _LIB, _LOADED
    path = library_path()
    if _LOADED != path:
        if not os.path.isfile(path):
            raise FileNotFoundError("K8/V4 library is not at %s" % path)
        lib = ctypes.CDLL(path)
        _declare(lib)
        _LIB, _LOADED = lib, path
    return _LIB


def _check(rc: int, lib) -> None:
    if rc != 0:
        raise RuntimeError(lib.k8v4_last_error().decode("utf-8", "replace"))


def _require(cond: bool, message: str, *parts) -> None:
    """Raise with ``message`` (``parts`` put into it only then) unless ``cond``."""
    if not cond:
        raise RuntimeError(message % parts if parts else message)


def _checked_hkv(hkv: int) -> int:
    _require(hkv in (2, 4), "unsupported per-GPU KV head count %d (this library serves 2 or 4)" % hkv)
    return hkv


# The checks below run on every eager call (a short decode step is bound by
# them, not by its kernels), so the usual case formats no message and compares
# whole shapes and strides: one token over 2,048, store and attention, 36.3 ->
# 26.0 us a step; a store of a few tokens 16.5 -> 10.6.


def _on_gpu(*tensors: torch.Tensor) -> torch.device:
    dev = tensors[0].device
    index = tensors[0].get_device()
    if dev.type == "cuda" and all(t.get_device() == index for t in tensors):
        return dev
    for t in tensors:
        _require(t.is_cuda, "K8/V4 ops need GPU tensors, got a %s tensor" % t.device.type)
        _require(t.device == dev, "K8/V4 op tensors are on different devices")
    return dev


# The raw handle of torch.cuda.current_stream(dev), without building the Python
# stream object around it: a private function, so where a torch lacks it the
# public call serves.
_RAW_STREAM = getattr(torch._C, "_cuda_getCurrentRawStream", None)


def _stream(dev: torch.device) -> int:
    if _RAW_STREAM is None:
        return int(torch.cuda.current_stream(dev).cuda_stream)
    return _RAW_STREAM(dev.index)


def _ptr(t: torch.Tensor) -> int:
    return int(t.data_ptr())


def check_paged_k(k_cache: torch.Tensor, k_scale: torch.Tensor, hkv: int, head_dim: int) -> None:
    """Shape and within-page stride rules of the K views (xe2_kv_ops.cpp:1333-1349)."""
    if not (
        k_cache.dtype == torch.int8 and k_scale.dtype == torch.float32
        and k_cache.shape[1:] == (PAGE, hkv, head_dim) and k_scale.shape == (k_cache.shape[0], PAGE, hkv)
        and k_cache.stride()[1:] == (hkv * head_dim, head_dim, 1) and k_scale.stride()[1:] == (hkv, 1)
    ):
        _reject_paged_k(k_cache, k_scale, hkv, head_dim)


def _reject_paged_k(k_cache, k_scale, hkv: int, head_dim: int) -> None:
    _require(k_cache.dtype == torch.int8, "k_cache int8")
    _require(k_scale.dtype == torch.float32, "k_scale float32")
    _require(
        k_cache.dim() == 4 and tuple(k_cache.shape[1:]) == (PAGE, hkv, head_dim),
        "k_cache [num_blocks,64,%d,%d] NHD" % (hkv, head_dim),
    )
    _require(
        k_scale.dim() == 3 and tuple(k_scale.shape) == (k_cache.shape[0], PAGE, hkv),
        "k_scale [num_blocks,64,%d]" % hkv,
    )
    _require(k_cache.stride()[1:] == (hkv * head_dim, head_dim, 1), "k_cache within-page strides")
    _require(k_scale.stride()[1:] == (hkv, 1), "k_scale within-page strides")


def check_paged_v(v_cache, v_scale, v_zero, hkv: int, head_dim: int) -> None:
    """Shape and within-page stride rules of the V views (xe2_kv_ops.cpp:1352-1370)."""
    cols = head_dim // 2
    plane = (v_cache.shape[0] if v_cache.dim() else -1, PAGE, hkv)
    if not (
        v_cache.dtype == torch.uint8 and v_scale.dtype == torch.float32 and v_zero.dtype == torch.float32
        and v_cache.shape[1:] == (PAGE, hkv, cols) and v_scale.shape == plane and v_zero.shape == plane
        and v_cache.stride()[1:] == (hkv * cols, cols, 1)
        and v_scale.stride()[1:] == (hkv, 1) and v_zero.stride()[1:] == (hkv, 1)
    ):
        _reject_paged_v(v_cache, v_scale, v_zero, hkv, head_dim)


def _reject_paged_v(v_cache, v_scale, v_zero, hkv: int, head_dim: int) -> None:
    cols = head_dim // 2
    _require(v_cache.dtype == torch.uint8, "v_cache uint8 packed int4")
    _require(v_scale.dtype == torch.float32 and v_zero.dtype == torch.float32, "v scale/zero float32")
    _require(
        v_cache.dim() == 4 and tuple(v_cache.shape[1:]) == (PAGE, hkv, cols),
        "v_cache [num_blocks,64,%d,%d] NHD packed" % (hkv, cols),
    )
    _require(v_scale.shape == v_zero.shape, "v_scale/v_zero shape")
    _require(
        v_scale.dim() == 3 and tuple(v_scale.shape) == (v_cache.shape[0], PAGE, hkv),
        "v_scale [num_blocks,64,%d]" % hkv,
    )
    _require(v_cache.stride()[1:] == (hkv * cols, cols, 1), "v_cache within-page strides")
    _require(v_scale.stride()[1:] == (hkv, 1), "v_scale within-page")
    _require(v_zero.stride()[1:] == (hkv, 1), "v_zero within-page")


def cache_args(k_cache, k_scale, v_cache, v_scale, v_zero) -> list[int]:
    """Pointers and byte page strides of the five region views, in ABI order."""
    return [
        k_cache.data_ptr(), k_scale.data_ptr(), v_cache.data_ptr(), v_scale.data_ptr(), v_zero.data_ptr(),
        k_cache.shape[0],
        k_cache.stride(0),
        k_scale.stride(0) * 4,
        v_cache.stride(0),
        v_scale.stride(0) * 4,
        v_zero.stride(0) * 4,
    ]


def _checked_cache(k_cache, k_scale, v_cache, v_scale, v_zero):
    """``(hkv, head_dim, cache_args)`` of five region views, each tensor's shape and
    strides fetched once (the checks and messages of :func:`check_paged_k` and
    :func:`check_paged_v`, to which anything unusual goes)."""
    shape, ks = k_cache.shape, k_cache.stride()
    if len(shape) == 4:
        pages, rows, hkv, dim = shape
        plane, cols = (pages, rows, hkv), dim // 2
        s1, vs, s2, s3 = k_scale.stride(), v_cache.stride(), v_scale.stride(), v_zero.stride()
        if (
            rows == PAGE and hkv in (2, 4) and dim in (128, 256)
            and k_cache.dtype == torch.int8 and v_cache.dtype == torch.uint8
            and k_scale.dtype == v_scale.dtype == v_zero.dtype == torch.float32
            and k_scale.shape == v_scale.shape == v_zero.shape == plane and v_cache.shape == (pages, rows, hkv, cols)
            and ks[1:] == (hkv * dim, dim, 1) and vs[1:] == (hkv * cols, cols, 1)
            and s1[1:] == s2[1:] == s3[1:] == (hkv, 1)
        ):
            return hkv, dim, (
                k_cache.data_ptr(), k_scale.data_ptr(), v_cache.data_ptr(), v_scale.data_ptr(), v_zero.data_ptr(),
                pages, ks[0], s1[0] * 4, vs[0], s2[0] * 4, s3[0] * 4,
            )
    _require(k_cache.dim() == 4 and v_cache.dim() == 4, "k_cache [num_blocks,64,HKV,D] NHD")
    hkv, dim = _checked_hkv(int(k_cache.shape[2])), int(k_cache.shape[3])
    _require(dim in (128, 256), "k_cache head dim must be 128 or 256")
    check_paged_k(k_cache, k_scale, hkv, dim)
    check_paged_v(v_cache, v_scale, v_zero, hkv, dim)
    _require(k_cache.shape[0] == v_cache.shape[0], "k/v num_blocks")
    return hkv, dim, tuple(cache_args(k_cache, k_scale, v_cache, v_scale, v_zero))


def _src_rows(t: torch.Tensor, name: str, hkv: int, head_dim: int) -> int:
    """Validate a ``[T, hkv, D]`` 16-bit source; returns its token stride in elements."""
    if not (
        t.dtype in (torch.float16, torch.bfloat16) and t.shape[1:] == (hkv, head_dim)
        and t.stride()[1:] == (head_dim, 1)
    ):
        _reject_src_rows(t, name, hkv, head_dim)
    return t.stride(0) if t.shape[0] > 1 else hkv * head_dim


def _reject_src_rows(t: torch.Tensor, name: str, hkv: int, head_dim: int) -> None:
    _require(t.dtype in (torch.float16, torch.bfloat16), "%s must be float16 or bfloat16" % name)
    _require(t.dim() == 3 and t.shape[2] == head_dim, "%s [T,HKV,%d]" % (name, head_dim))
    _require(t.shape[1] == hkv, "%s heads" % name)
    _require(t.stride(2) == 1 and t.stride(1) == head_dim, "%s head/dim strides must be (%d, 1)" % (name, head_dim))


class BoundCall:
    """One validated op call: the C entry point plus its argument list.

    Calling it enqueues the op on the current stream of the call's device;
    the tensors it was bound with are kept alive with it.
    """

    __slots__ = ("_lib", "_fn", "_profiled", "_args", "_dev", "_keep")

    def __init__(self, lib, fn, args, dev, keep, profiled=None):
        self._lib, self._fn, self._profiled = lib, fn, profiled
        self._args, self._dev, self._keep = tuple(args), dev, keep

    def __call__(self, split_done_event=None, stages: int = 3) -> None:
        stream = _stream(self._dev)
        if split_done_event is None and stages == 3:
            rc = self._fn(*self._args, stream)
        else:
            _require(self._profiled is not None, "this op has no staged variant")
            rc = self._profiled(*self._args, stream, int(split_done_event or 0), int(stages))
        _check(rc, self._lib)


class DeviceCall(BoundCall):
    """A :class:`BoundCall` that launches on its tensors' device, whichever is current."""

    __slots__ = ()

    def __call__(self) -> None:
        if torch.cuda.current_device() == self._dev.index:
            _check(self._fn(*self._args, _stream(self._dev)), self._lib)
            return
        with torch.cuda.device(self._dev):
            _check(self._fn(*self._args, _stream(self._dev)), self._lib)


class _Ops:
    """Methods named after the reference's ``torch.ops.xe2_kv`` schemas."""

    def __init__(self, lib):
        self._lib = lib
        self._legacy_ws: dict[torch.device, torch.Tensor] = {}

    # -- quantize-and-write ------------------------------------------------
    def kv_store_paged(self, k_fp16, v_fp16, slot_mapping, k_cache, k_scale, v_cache, v_scale, v_zero):
        """Quantize K/V ``[T, HKV, D]`` into the paged cache at ``slot_mapping`` (int64 ``[T]``)."""
        bound = self.bind_kv_store_paged(k_fp16, v_fp16, slot_mapping, k_cache, k_scale, v_cache, v_scale, v_zero)
        if bound is not None:
            bound()

    def bind_kv_store_paged(self, k_fp16, v_fp16, slot_mapping, k_cache, k_scale, v_cache, v_scale, v_zero):
        """Validate a store once; returns a :class:`BoundCall` (None when there are no tokens)."""
        _require(k_fp16.dim() == 3, "k_fp16 [T,HKV,D]")
        head_dim = int(k_fp16.shape[2])
        _require(head_dim in (128, 256), "k_fp16 [T,HKV,D] with D in (128, 256)")
        _require(k_fp16.dtype == v_fp16.dtype, "k/v_fp16 dtypes differ")
        _require(v_fp16.shape == k_fp16.shape, "v_fp16 must match k_fp16")
        _require(slot_mapping.dtype == torch.int64, "slot_mapping int64")
        _require(slot_mapping.is_contiguous(), "slot_mapping must be contiguous")
        hkv = _checked_hkv(int(k_fp16.shape[1]))
        check_paged_k(k_cache, k_scale, hkv, head_dim)
        check_paged_v(v_cache, v_scale, v_zero, hkv, head_dim)
        _require(k_cache.shape[0] == v_cache.shape[0], "k/v num_blocks")
        _require(slot_mapping.numel() == k_fp16.shape[0], "slot_mapping [T]")
        ks = _src_rows(k_fp16, "k_fp16", hkv, head_dim)
        vs = _src_rows(v_fp16, "v_fp16", hkv, head_dim)
        ntok = int(k_fp16.shape[0])
        if ntok == 0:
            return None
        tensors = (k_fp16, v_fp16, slot_mapping, k_cache, k_scale, v_cache, v_scale, v_zero)
        dev = _on_gpu(*tensors)
        args = [
            _ptr(k_fp16), _ptr(v_fp16), _DTYPE_CODE[k_fp16.dtype], ks, vs,
            _ptr(slot_mapping), ntok, hkv, head_dim,
            *cache_args(k_cache, k_scale, v_cache, v_scale, v_zero),
        ]
        return BoundCall(self._lib, self._lib.k8v4_kv_store_paged, args, dev, tensors)

    # -- quantize-and-write with the rotation ----------------------------------
    def rope_kv_store_paged(self, q_fp16, k_fp16, v_fp16, positions, cos_sin, neox, slot_mapping, k_cache, k_scale,
                            v_cache, v_scale, v_zero, q_out):
        """:meth:`kv_store_paged` with the keys rotated by their positions on the way, and
        the queries rotated.

        ``q_fp16`` ``[T, HQ, D]`` and ``q_out`` of its shape and dtype (may be ``q_fp16``;
        both None: no queries); ``positions`` int32 or int64 ``[T]``; ``cos_sin``
        ``[P, R]`` (fp16, bf16 or fp32), row p the R / 2 cosines, then the sines of
        position p, R a multiple of 16 up to D; ``neox``: pairs are dims (i, i + R / 2),
        else (2 i, 2 i + 1).  Keys are quantized from the unrounded rotation.  Slots
        are distinct; a token without one (negative, or past the last page) stores nothing;
        one whose position lies outside the table neither, and its query rows become
        zeros."""
        bound = self.bind_rope_kv_store_paged(q_fp16, k_fp16, v_fp16, positions, cos_sin, neox, slot_mapping, k_cache,
                                              k_scale, v_cache, v_scale, v_zero, q_out)
        if bound is not None:
            bound()

    def bind_rope_kv_store_paged(self, q_fp16, k_fp16, v_fp16, positions, cos_sin, neox, slot_mapping, k_cache,
                                 k_scale, v_cache, v_scale, v_zero, q_out):
        """Validate a rotated store once; returns a :class:`DeviceCall` (None when there are no tokens)."""
        _require(k_fp16.dim() == 3, "k_fp16 [T,HKV,D]")
        ntok, hkv, head_dim = k_fp16.shape
        _require(head_dim in (128, 256), "k_fp16 [T,HKV,D] with D in (128, 256)")
        _checked_hkv(hkv)
        _require(k_fp16.dtype == v_fp16.dtype, "k/v_fp16 dtypes differ")
        _require(v_fp16.shape == k_fp16.shape, "v_fp16 must match k_fp16")
        _require(slot_mapping.dtype == torch.int64 and slot_mapping.is_contiguous(), "slot_mapping int64")
        chkv, cdim, cache = _checked_cache(k_cache, k_scale, v_cache, v_scale, v_zero)
        _require(chkv == hkv and cdim == head_dim, "k_cache [num_blocks,64,%d,%d] NHD", hkv, head_dim)
        _require(slot_mapping.shape == (ntok,), "slot_mapping [T]")
        _require(positions.dtype in (torch.int32, torch.int64) and positions.shape == (ntok,)
                 and positions.is_contiguous(), "positions must be a contiguous int32 or int64 [T]")
        _require(cos_sin.dtype in _DTYPE_CODE and cos_sin.dim() == 2, "cos_sin float16, bfloat16 or float32 [P,R]")
        table_rows, rot = cos_sin.shape
        _require(rot % 16 == 0 and 16 <= rot <= head_dim and table_rows >= 1,
                 "cos_sin [P,R] with R a multiple of 16 up to the head dim")
        _require(cos_sin.stride(1) == 1, "cos_sin rows must be contiguous")
        ks = _src_rows(k_fp16, "k_fp16", hkv, head_dim)
        vs = _src_rows(v_fp16, "v_fp16", hkv, head_dim)
        _require((q_fp16 is None) == (q_out is None), "q_fp16 and q_out go together")
        tensors = (k_fp16, v_fp16, positions, cos_sin, slot_mapping, k_cache, k_scale, v_cache, v_scale, v_zero)
        heads = GQA * hkv
        q_ptr = out_ptr = 0
        qs = qos = heads * head_dim
        if q_fp16 is not None:
            _require(q_fp16.shape == (ntok, heads, head_dim), "q_fp16 [T,HQ,D] with HQ = 6 * HKV")
            _require(q_fp16.dtype == k_fp16.dtype, "q/k_fp16 dtypes differ")
            _require(q_out.shape == q_fp16.shape and q_out.dtype == q_fp16.dtype, "q_out must match q_fp16")
            qs = _src_rows(q_fp16, "q_fp16", heads, head_dim)
            qos = _src_rows(q_out, "q_out", heads, head_dim)
            q_ptr, out_ptr = q_fp16.data_ptr(), q_out.data_ptr()
            _require(q_ptr != out_ptr or qs == qos, "q_out may be q_fp16 itself, not another view of its rows")
            tensors += (q_fp16, q_out)
        if ntok == 0:
            return None
        dev = _on_gpu(*tensors)
        args = (
            q_ptr, k_fp16.data_ptr(), v_fp16.data_ptr(), _DTYPE_CODE[k_fp16.dtype], qs, ks, vs,
            positions.data_ptr(), int(positions.dtype == torch.int64), cos_sin.data_ptr(), _DTYPE_CODE[cos_sin.dtype],
            table_rows, cos_sin.stride(0) if table_rows > 1 else rot, rot, int(bool(neox)),
            slot_mapping.data_ptr(), ntok, hkv, head_dim, *cache, out_ptr, qos,
        )
        return DeviceCall(self._lib, self._lib.k8v4_rope_kv_store_paged, args, dev, tensors)

    # -- decode / MTP verify ----------------------------------------------
    def attn_workspace_bytes(self, batch: int, table_width: int, pages_per_block: int, q_len: int,
                             hkv: int, head_dim: int, num_splits: int = 0) -> int:
        """Scratch bytes :meth:`int8k_int4v_attn_batch` needs for this shape."""
        n = int(self._lib.k8v4_attn_workspace_bytes(batch, table_width, pages_per_block, q_len, hkv,
                                                    head_dim, num_splits))
        _require(n > 0, "bad shape for the decode workspace")
        return n

    def int8k_int4v_attn_batch(self, q_fp16, q8, q_scale, k_cache, k_scale, v_cache, v_scale, v_zero,
                               block_table, seq_lens, visible_lens, partials_ws, m_ws, l_ws, merged_ws,
                               out, q_len, pages_per_block, num_splits: int = 0, split_done_event=None,
                               stages: int = 3):
        """One uniform-q_len decode batch (argument order of the reference op).

        Validates and launches; :meth:`bind_int8k_int4v_attn_batch` takes the
        same arguments and returns the validated call for repeated launches.

        ``q8``, ``q_scale``, ``m_ws``, ``l_ws`` and ``merged_ws`` are accepted for
        signature compatibility and left untouched: Q is quantized inside the
        kernel and the split-K state lives in the bytes of ``partials_ws``.
        ``visible_lens`` is None, an empty tensor (derive causal ends from
        ``seq_lens``) or int32 ``[B, >= 1 + q_len]``.

        Timing hooks (no effect on results): ``split_done_event`` is a raw
        hipEvent_t handle recorded after the split-K kernel; ``stages`` = 1 runs
        only the split-K kernel, 2 only the merge (over the workspace a
        ``stages=1`` call with the same arguments filled), 3 both.
        """
        self.bind_int8k_int4v_attn_batch(
            q_fp16, q8, q_scale, k_cache, k_scale, v_cache, v_scale, v_zero, block_table, seq_lens,
            visible_lens, partials_ws, m_ws, l_ws, merged_ws, out, q_len, pages_per_block, num_splits,
        )(split_done_event=split_done_event, stages=stages)

    def bind_int8k_int4v_attn_batch(self, q_fp16, q8, q_scale, k_cache, k_scale, v_cache, v_scale, v_zero,
                                    block_table, seq_lens, visible_lens, partials_ws, m_ws, l_ws, merged_ws,
                                    out, q_len, pages_per_block, num_splits: int = 0):
        """Validate one decode call; returns a :class:`BoundCall` that launches it.

        The call keeps the tensors' device addresses: their contents may change
        between launches (new queries, lengths, tables), their storage may not.
        """
        del q8, q_scale, m_ws, l_ws, merged_ws
        q_len = int(q_len)
        pages_per_block = int(pages_per_block)
        _require(pages_per_block >= 1, "pages_per_block")
        _require(q_len > 0 and q_len * GQA <= PAGE, "q_len*GQA exceeds BM")
        _require(q_fp16.dim() == 3, "q_fp16 [T,HQ,D]")
        head_dim = int(q_fp16.shape[2])
        _require(head_dim in (128, 256), "q_fp16 [T,HQ,D] with D in (128, 256)")
        _require(q_fp16.shape[1] % GQA == 0, "q_fp16 heads must be a multiple of GQA=6")
        hkv = _checked_hkv(int(q_fp16.shape[1]) // GQA)
        _require(q_fp16.dtype in (torch.float16, torch.bfloat16), "q_fp16 must be float16 or bfloat16")
        _require(q_fp16.stride(2) == 1 and q_fp16.stride(1) == head_dim, "q_fp16 head/dim strides")
        _require(out.shape == q_fp16.shape, "out shape")
        _require(out.dtype in (torch.float16, torch.bfloat16, torch.float32), "out float16, bfloat16 or float32")
        _require(out.stride(2) == 1 and out.stride(1) == head_dim, "out head/dim strides")
        _require(q_fp16.shape[0] % q_len == 0, "T must be B*q_len")
        batch = int(q_fp16.shape[0]) // q_len
        _require(batch >= 1, "empty batch")
        check_paged_k(k_cache, k_scale, hkv, head_dim)
        check_paged_v(v_cache, v_scale, v_zero, hkv, head_dim)
        _require(k_cache.shape[0] == v_cache.shape[0], "k/v num_blocks")
        _require(block_table.dtype == torch.int32, "block_table int32")
        _require(block_table.dim() == 2 and block_table.shape[0] == batch, "block_table [B, splits]")
        _require(block_table.stride(1) == 1, "block_table rows must be contiguous")
        _require(int(block_table.shape[1]) > 0, "block_table n_splits")
        _require(seq_lens.dtype == torch.int32 and seq_lens.numel() >= batch, "seq_lens [B]")
        _require(seq_lens.is_contiguous(), "seq_lens XPU contig (graph input)")
        vis_ptr, vis_stride = 0, 0
        if visible_lens is not None and visible_lens.numel() > 0:
            _require(visible_lens.dtype == torch.int32, "visible_lens int32")
            _require(visible_lens.dim() == 2 and visible_lens.shape[0] == batch
                     and visible_lens.shape[1] >= q_len + 1, "visible_lens [B, 1+q_len]")
            _require(visible_lens.stride(1) == 1, "visible_lens rows must be contiguous")
            vis_ptr, vis_stride = _ptr(visible_lens), int(visible_lens.stride(0))
        _require(partials_ws is not None and partials_ws.is_contiguous(), "partials_ws must be a contiguous buffer")
        tensors = (q_fp16, k_cache, k_scale, v_cache, v_scale, v_zero, block_table, seq_lens, out, partials_ws)
        dev = _on_gpu(*tensors)
        ws_bytes = int(partials_ws.numel()) * partials_ws.element_size()
        args = [
            _ptr(q_fp16), _DTYPE_CODE[q_fp16.dtype], int(q_fp16.stride(0)),
            *cache_args(k_cache, k_scale, v_cache, v_scale, v_zero),
            _ptr(block_table), int(block_table.stride(0)), int(block_table.shape[1]), pages_per_block,
            _ptr(seq_lens), vis_ptr, vis_stride, batch, q_len, hkv, head_dim,
            _ptr(out), _DTYPE_CODE[out.dtype], int(out.stride(0)),
            _ptr(partials_ws), ws_bytes, int(num_splits),
        ]
        keep = tensors + ((visible_lens,) if vis_ptr else ())
        return BoundCall(self._lib, self._lib.k8v4_attn_batch, args, dev, keep,
                         profiled=self._lib.k8v4_attn_batch_profiled)

    # -- decode / MTP verify over a shared prefix -----------------------------
    def attn_shared_workspace_bytes(self, batch: int, q_len: int, hkv: int, head_dim: int) -> int:
        """Scratch bytes :meth:`int8k_int4v_attn_shared` needs (any prefix and lengths)."""
        n = int(self._lib.k8v4_attn_shared_workspace_bytes(int(batch), int(q_len), int(hkv), int(head_dim)))
        _require(n > 0, "bad shape for the shared-prefix workspace")
        return n

    def attn_shared_many_rows(self, batch: int, q_len: int, hkv: int, head_dim: int, prefix_len: int) -> bool:
        """Whether :meth:`int8k_int4v_attn_shared` attends to this prefix by the kernel that
        holds many query rows (False: eight tokens at a time, or no page is shared)."""
        n = int(self._lib.k8v4_attn_shared_many_rows(int(batch), int(q_len), int(hkv), int(head_dim), int(prefix_len)))
        _require(n >= 0, "bad shape for the shared-prefix plan")
        return n == 1

    def int8k_int4v_attn_shared(self, q_fp16, k_cache, k_scale, v_cache, v_scale, v_zero, prefix_table, prefix_len,
                                block_table, seq_lens, workspace, out, q_len, pages_per_block):
        """:meth:`int8k_int4v_attn_batch` for sequences that begin with the same cached
        pages, those read once for all of them.

        ``prefix_table`` (int32 ``[W']``, for instance ``block_table[0]``) names the
        pages of the first ``prefix_len`` tokens, all of them stored; its whole pages
        (``prefix_len // 64``) stand for those of every sequence, whatever the
        sequences' own rows of ``block_table`` (int32 ``[B, W]``) hold there, and the
        tokens behind them come from those rows.  ``seq_lens`` (int32 ``[B]``) counts all of a sequence's
        tokens, the prefix included; a row whose causal end lies inside the prefix
        sees the prefix up to there, one that sees nothing gives zeros.  The other
        arguments and the numerics are the batch op's; ``workspace`` holds
        :meth:`attn_shared_workspace_bytes` bytes."""
        self.bind_int8k_int4v_attn_shared(q_fp16, k_cache, k_scale, v_cache, v_scale, v_zero, prefix_table,
                                          prefix_len, block_table, seq_lens, workspace, out, q_len,
                                          pages_per_block)()

    def bind_int8k_int4v_attn_shared(self, q_fp16, k_cache, k_scale, v_cache, v_scale, v_zero, prefix_table,
                                     prefix_len, block_table, seq_lens, workspace, out, q_len, pages_per_block):
        """Validate one shared-prefix call; returns a :class:`DeviceCall` that launches it.

        Lengths, tables and queries may change between launches, ``prefix_len`` may not."""
        q_len, prefix_len, pages_per_block = int(q_len), int(prefix_len), int(pages_per_block)
        _require(pages_per_block >= 1, "pages_per_block")
        _require(prefix_len >= 0, "negative prefix length")
        _require(q_len > 0 and q_len * GQA <= PAGE, "q_len*GQA exceeds BM")
        _require(q_fp16.dim() == 3, "q_fp16 [T,HQ,D]")
        tokens, heads, head_dim = (int(x) for x in q_fp16.shape)
        _require(head_dim in (128, 256), "q_fp16 [T,HQ,D] with D in (128, 256)")
        _require(heads % GQA == 0, "q_fp16 heads must be a multiple of GQA=6")
        hkv = _checked_hkv(heads // GQA)
        _require(q_fp16.dtype in (torch.float16, torch.bfloat16), "q_fp16 must be float16 or bfloat16")
        _require(q_fp16.stride()[1:] == (head_dim, 1), "q_fp16 head/dim strides")
        _require(out.shape == q_fp16.shape, "out shape")
        _require(out.dtype in (torch.float16, torch.bfloat16, torch.float32), "out float16, bfloat16 or float32")
        _require(out.stride()[1:] == (head_dim, 1), "out head/dim strides")
        _require(tokens % q_len == 0, "T must be B*q_len")
        batch = tokens // q_len
        _require(batch >= 1, "empty batch")
        check_paged_k(k_cache, k_scale, hkv, head_dim)
        check_paged_v(v_cache, v_scale, v_zero, hkv, head_dim)
        _require(k_cache.shape[0] == v_cache.shape[0], "k/v num_blocks")
        _require(block_table.dtype == torch.int32 and block_table.dim() == 2 and block_table.shape[0] == batch,
                 "block_table int32 [B, splits]")
        _require(int(block_table.shape[1]) > 0, "block_table n_splits")
        _require(block_table.stride(1) == 1, "block_table rows must be contiguous")
        _require(seq_lens.dtype == torch.int32 and seq_lens.numel() >= batch and seq_lens.is_contiguous(),
                 "seq_lens must be a contiguous int32 [B]")
        _require(workspace.is_contiguous(), "workspace must be a contiguous buffer")
        tensors = (q_fp16, k_cache, k_scale, v_cache, v_scale, v_zero, block_table, seq_lens, out, workspace)
        prefix_width = 0
        if prefix_len >= PAGE:
            _require(prefix_table is not None and prefix_table.dtype == torch.int32 and prefix_table.dim() == 1
                     and (prefix_table.shape[0] < 2 or prefix_table.stride(0) == 1),
                     "prefix_table must be a contiguous int32 row")
            prefix_width = int(prefix_table.shape[0])
            tensors += (prefix_table,)
        dev = _on_gpu(*tensors)
        row = heads * head_dim
        args = [
            _ptr(q_fp16), _DTYPE_CODE[q_fp16.dtype], int(q_fp16.stride(0)) if tokens > 1 else row,
            *cache_args(k_cache, k_scale, v_cache, v_scale, v_zero),
            _ptr(prefix_table) if prefix_width else 0, prefix_width, prefix_len,
            _ptr(block_table), int(block_table.stride(0)) if batch > 1 else int(block_table.shape[1]),
            int(block_table.shape[1]), pages_per_block, _ptr(seq_lens), batch, q_len, hkv, head_dim,
            _ptr(out), _DTYPE_CODE[out.dtype], int(out.stride(0)) if tokens > 1 else row,
            _ptr(workspace), int(workspace.numel()) * workspace.element_size(),
        ]
        return DeviceCall(self._lib, self._lib.k8v4_attn_shared, args, dev, tensors)

    # -- decode of drafted trees ------------------------------------------------
    def attn_tree_workspace_bytes(self, batch: int, nodes: int, hkv: int, head_dim: int) -> int:
        """Scratch bytes :meth:`int8k_int4v_attn_tree` needs (any lengths)."""
        n = int(self._lib.k8v4_attn_tree_workspace_bytes(int(batch), int(nodes), int(hkv), int(head_dim)))
        _require(n > 0, "bad shape for the tree workspace")
        return n

    def int8k_int4v_attn_tree(self, q_fp16, k_cache, k_scale, v_cache, v_scale, v_zero, block_table, seq_lens,
                              tree_masks, workspace, out, nodes, pages_per_block):
        """:meth:`int8k_int4v_attn_batch` for trees of drafted tokens.

        Each sequence has ``nodes`` (up to 64) query tokens, stored as its last tokens
        (``seq_lens`` counts them): node j lies at position ``seq_len - nodes + j`` and
        attends to the tokens ahead of the tree and to every node i whose bit i is set in
        ``tree_masks[b, j]`` (int64 ``[B, nodes]``; a row expanded over the batch is one
        tree for all; :func:`k8v4_v030.plan.tree_masks` makes them from parents).  The
        other arguments and the numerics are the batch op's; ``workspace`` holds
        :meth:`attn_tree_workspace_bytes` bytes.  The kernel is chosen by the table's
        width: short contexts are served best with no wider a table than they need."""
        self.bind_int8k_int4v_attn_tree(q_fp16, k_cache, k_scale, v_cache, v_scale, v_zero, block_table, seq_lens,
                                        tree_masks, workspace, out, nodes, pages_per_block)()

    def bind_int8k_int4v_attn_tree(self, q_fp16, k_cache, k_scale, v_cache, v_scale, v_zero, block_table, seq_lens,
                                   tree_masks, workspace, out, nodes, pages_per_block):
        """Validate one tree call; returns a :class:`DeviceCall` that launches it.

        Lengths, tables, masks and queries may change between launches."""
        nodes, pages_per_block = int(nodes), int(pages_per_block)
        _require(pages_per_block >= 1, "pages_per_block")
        _require(1 <= nodes <= 64, "1 to 64 nodes a tree")
        _require(q_fp16.dim() == 3, "q_fp16 [T,HQ,D]")
        tokens, heads, head_dim = q_fp16.shape
        _require(head_dim in (128, 256), "q_fp16 [T,HQ,D] with D in (128, 256)")
        _require(heads % GQA == 0, "q_fp16 heads must be a multiple of GQA=6")
        hkv = _checked_hkv(heads // GQA)
        _require(q_fp16.dtype in (torch.float16, torch.bfloat16), "q_fp16 must be float16 or bfloat16")
        _require(q_fp16.stride()[1:] == (head_dim, 1), "q_fp16 head/dim strides")
        _require(out.shape == q_fp16.shape, "out shape")
        _require(out.dtype in (torch.float16, torch.bfloat16, torch.float32), "out float16, bfloat16 or float32")
        _require(out.stride()[1:] == (head_dim, 1), "out head/dim strides")
        _require(tokens % nodes == 0, "T must be B*nodes")
        batch = tokens // nodes
        _require(batch >= 1, "empty batch")
        chkv, cdim, cache = _checked_cache(k_cache, k_scale, v_cache, v_scale, v_zero)
        _require(chkv == hkv and cdim == head_dim, "k_cache [num_blocks,64,%d,%d] NHD", hkv, head_dim)
        _require(block_table.dtype == torch.int32 and block_table.dim() == 2 and block_table.shape[0] == batch,
                 "block_table int32 [B, splits]")
        _require(int(block_table.shape[1]) > 0, "block_table n_splits")
        _require(block_table.stride(1) == 1, "block_table rows must be contiguous")
        _require(seq_lens.dtype == torch.int32 and seq_lens.numel() >= batch and seq_lens.is_contiguous(),
                 "seq_lens must be a contiguous int32 [B]")
        _require(tree_masks.dtype == torch.int64 and tree_masks.shape == (batch, nodes)
                 and (nodes == 1 or tree_masks.stride(1) == 1), "tree_masks int64 [B,nodes] with contiguous rows")
        _require(workspace.is_contiguous(), "workspace must be a contiguous buffer")
        tensors = (q_fp16, k_cache, k_scale, v_cache, v_scale, v_zero, block_table, seq_lens, tree_masks, out, workspace)
        dev = _on_gpu(*tensors)
        row, width = heads * head_dim, block_table.shape[1]
        args = (
            q_fp16.data_ptr(), _DTYPE_CODE[q_fp16.dtype], q_fp16.stride(0) if tokens > 1 else row,
            *cache, block_table.data_ptr(), block_table.stride(0) if batch > 1 else width, width, pages_per_block,
            seq_lens.data_ptr(), tree_masks.data_ptr(), tree_masks.stride(0) if batch > 1 else nodes, batch, nodes,
            hkv, head_dim, out.data_ptr(), _DTYPE_CODE[out.dtype], out.stride(0) if tokens > 1 else row,
            workspace.data_ptr(), workspace.numel() * workspace.element_size(),
        )
        return DeviceCall(self._lib, self._lib.k8v4_attn_tree, args, dev, tensors)

    # -- chunked prefill ----------------------------------------------------
    def prefill_workspace_bytes(self, seq_len: int, q_len: int, hkv: int, head_dim: int) -> int:
        """Scratch bytes :meth:`prefill_paged` needs for this shape."""
        n = int(self._lib.k8v4_prefill_workspace_bytes(int(seq_len), int(q_len), int(hkv), int(head_dim)))
        _require(n >= 0, "bad shape for the prefill workspace")
        return n

    def prefill_uses_tiles(self, seq_len: int, q_len: int, hkv: int, head_dim: int) -> bool:
        """Whether :meth:`prefill_paged` always serves this shape from per-KV-head
        tile images (each page dequantized once per head), which its workspace
        then has to hold.  False: it does so only where the workspace has room
        and that is faster, and may convert pages in place."""
        n = int(self._lib.k8v4_prefill_uses_tiles(int(seq_len), int(q_len), int(hkv), int(head_dim)))
        _require(n >= 0, "bad shape for the prefill plan")
        return n == 1

    def prefill_paged(self, q, k_cache, k_scale, v_cache, v_scale, v_zero, block_row, seq_len: int,
                      pages_per_block: int, scale: float, out, workspace=None):
        """Bottom-right causal attention of ``q [q_len, HQ, D]`` over one sequence's pages into ``out``."""
        call = self.bind_prefill_paged(q, k_cache, k_scale, v_cache, v_scale, v_zero, block_row, seq_len,
                                       pages_per_block, scale, out, workspace)
        if call is not None:
            call()

    def bind_prefill_paged(self, q, k_cache, k_scale, v_cache, v_scale, v_zero, block_row, seq_len: int,
                           pages_per_block: int, scale: float, out, workspace=None):
        """Validate one prefill; returns a :class:`BoundCall` (None when ``q_len`` is 0).

        ``workspace`` is a device buffer of at least :meth:`prefill_workspace_bytes`
        bytes; None allocates one (the prefill path is not graph-captured)."""
        _require(q.dim() == 3, "query [T,HQ,D]")
        head_dim = int(q.shape[2])
        _require(head_dim in (128, 256), "query [T,HQ,D] with D in (128, 256)")
        hkv = int(k_cache.shape[2]) if k_cache.dim() == 4 else -1
        _require(int(q.shape[1]) == GQA * hkv,
                 "query has %d heads, the K8/V4 cache holds %d (needs %d)" % (int(q.shape[1]), hkv, GQA * hkv))
        _checked_hkv(hkv)
        check_paged_k(k_cache, k_scale, hkv, head_dim)
        check_paged_v(v_cache, v_scale, v_zero, hkv, head_dim)
        q_len, seq_len = int(q.shape[0]), int(seq_len)
        if q_len > seq_len:
            raise RuntimeError("query longer than the KV sequence")
        if q_len == 0:
            return None
        _require(q.dtype in (torch.float16, torch.bfloat16), "query must be float16 or bfloat16")
        _require(q.stride(2) == 1 and q.stride(1) == head_dim, "query head/dim strides")
        _require(out.shape == q.shape, "out shape")
        _require(out.dtype in (torch.float16, torch.bfloat16, torch.float32), "out float16, bfloat16 or float32")
        _require(out.stride(2) == 1 and out.stride(1) == head_dim, "out head/dim strides")
        _require(block_row.dtype == torch.int32 and block_row.dim() == 1 and block_row.stride(0) == 1,
                 "block_row must be a contiguous int32 [width] row")
        _require(int(pages_per_block) >= 1, "pages_per_block")
        tensors = (q, k_cache, k_scale, v_cache, v_scale, v_zero, block_row, out)
        dev = _on_gpu(*tensors)
        need = self.prefill_workspace_bytes(seq_len, q_len, hkv, head_dim)
        if workspace is None:
            workspace = torch.empty(max(need, 16) // 4 + 4, dtype=torch.float32, device=dev)
        _require(workspace.is_contiguous() and workspace.device == dev, "prefill workspace must be a contiguous "
                 "buffer on the query's device")
        tensors = tensors + (workspace,)
        args = [
            _ptr(q), _DTYPE_CODE[q.dtype], int(q.stride(0)) if q_len > 1 else GQA * hkv * head_dim,
            *cache_args(k_cache, k_scale, v_cache, v_scale, v_zero),
            _ptr(block_row), int(block_row.shape[0]), int(pages_per_block), seq_len, q_len, hkv, head_dim,
            float(scale), _ptr(out), _DTYPE_CODE[out.dtype],
            int(out.stride(0)) if q_len > 1 else GQA * hkv * head_dim,
            _ptr(workspace), int(workspace.numel()) * workspace.element_size(),
        ]
        return BoundCall(self._lib, self._lib.k8v4_prefill_paged, args, dev, tensors)

    def prefill_batch_workspace_bytes(self, hkv: int, head_dim: int) -> int:
        """Scratch bytes :meth:`prefill_paged_batch` needs (any sequences)."""
        n = int(self._lib.k8v4_prefill_batch_workspace_bytes(int(hkv), int(head_dim)))
        _require(n >= 0, "bad shape for the prefill workspace")
        return n

    def prefill_paged_batch(self, q, k_cache, k_scale, v_cache, v_scale, v_zero, block_table, tok0, q_lens,
                            seq_lens, rows, pages_per_block: int, scale: float, out, workspace=None):
        """Several sequences' prefill in one call (the chunks of one step).

        Sequence i: query rows ``q[tok0[i] : tok0[i] + q_lens[i]]`` (bottom-right
        causal over its ``seq_lens[i]`` keys) into the same rows of ``out``, its
        pages in ``block_table[rows[i]]``.  ``tok0``, ``q_lens``, ``seq_lens`` and
        ``rows`` are Python integer sequences of one length.  Same numerics as
        :meth:`prefill_paged` per sequence."""
        _require(q.dim() == 3, "query [T,HQ,D]")
        head_dim = int(q.shape[2])
        _require(head_dim in (128, 256), "query [T,HQ,D] with D in (128, 256)")
        hkv = int(k_cache.shape[2]) if k_cache.dim() == 4 else -1
        _require(int(q.shape[1]) == GQA * hkv,
                 "query has %d heads, the K8/V4 cache holds %d (needs %d)" % (int(q.shape[1]), hkv, GQA * hkv))
        _checked_hkv(hkv)
        check_paged_k(k_cache, k_scale, hkv, head_dim)
        check_paged_v(v_cache, v_scale, v_zero, hkv, head_dim)
        tok0, q_lens, seq_lens, rows = ([int(x) for x in v] for v in (tok0, q_lens, seq_lens, rows))
        n = len(tok0)
        _require(len(q_lens) == n and len(seq_lens) == n and len(rows) == n,
                 "tok0, q_lens, seq_lens and rows must have one length")
        _require(block_table.dtype == torch.int32 and block_table.dim() == 2 and block_table.stride(1) == 1,
                 "block_table must be int32 [B, W] with unit column stride")
        tokens = int(q.shape[0])
        for t0, ql, sl, r in zip(tok0, q_lens, seq_lens, rows):
            if ql > sl:
                raise RuntimeError("query longer than the KV sequence")
            _require(ql >= 0 and t0 >= 0 and t0 + ql <= tokens, "sequence rows outside the query")
            _require(0 <= r < int(block_table.shape[0]), "block table row out of range")
        if n == 0 or max(q_lens) == 0:
            return
        _require(q.dtype in (torch.float16, torch.bfloat16), "query must be float16 or bfloat16")
        _require(q.stride(2) == 1 and q.stride(1) == head_dim, "query head/dim strides")
        _require(out.shape == q.shape, "out shape")
        _require(out.dtype in (torch.float16, torch.bfloat16, torch.float32), "out float16, bfloat16 or float32")
        _require(out.stride(2) == 1 and out.stride(1) == head_dim, "out head/dim strides")
        _require(int(pages_per_block) >= 1, "pages_per_block")
        tensors = (q, k_cache, k_scale, v_cache, v_scale, v_zero, block_table, out)
        dev = _on_gpu(*tensors)
        need = self.prefill_batch_workspace_bytes(hkv, head_dim)
        if workspace is None:
            workspace = torch.empty(max(need, 16) // 4 + 4, dtype=torch.float32, device=dev)
        _require(workspace.is_contiguous() and workspace.device == dev, "prefill workspace must be a contiguous "
                 "buffer on the query's device")
        arrays = [(ctypes.c_int64 * n)(*v) for v in (tok0, q_lens, seq_lens, rows)]
        row_stride = GQA * hkv * head_dim
        rc = self._lib.k8v4_prefill_paged_batch(
            _ptr(q), _DTYPE_CODE[q.dtype], int(q.stride(0)) if tokens > 1 else row_stride,
            *cache_args(k_cache, k_scale, v_cache, v_scale, v_zero),
            _ptr(block_table), int(block_table.stride(0)), int(block_table.shape[1]), int(pages_per_block), n,
            *[ctypes.cast(x, ctypes.c_void_p) for x in arrays], hkv, head_dim, float(scale),
            _ptr(out), _DTYPE_CODE[out.dtype], int(out.stride(0)) if tokens > 1 else row_stride,
            _ptr(workspace), int(workspace.numel()) * workspace.element_size(), _stream(dev))
        _check(rc, self._lib)

    # -- K-only / V-only stores ----------------------------------------------
    def k_store_paged(self, k_fp16, slot_mapping, k_cache, k_scale):
        """The K half of :meth:`kv_store_paged` (xe2_kv_ops.cpp:1371-1389)."""
        _require(k_fp16.dim() == 3 and int(k_fp16.shape[2]) in (128, 256), "k_fp16 [T,HKV,D] with D in (128, 256)")
        head_dim = int(k_fp16.shape[2])
        _require(slot_mapping.dtype == torch.int64 and slot_mapping.is_contiguous(), "slot_mapping int64")
        hkv = _checked_hkv(int(k_fp16.shape[1]))
        check_paged_k(k_cache, k_scale, hkv, head_dim)
        _require(slot_mapping.numel() == k_fp16.shape[0], "slot_mapping [T]")
        ks = _src_rows(k_fp16, "k_fp16", hkv, head_dim)
        if k_fp16.shape[0] == 0:
            return
        dev = _on_gpu(k_fp16, slot_mapping, k_cache, k_scale)
        rc = self._lib.k8v4_k_store_paged(_ptr(k_fp16), _DTYPE_CODE[k_fp16.dtype], ks, _ptr(slot_mapping),
                                          int(k_fp16.shape[0]), hkv, head_dim, _ptr(k_cache), _ptr(k_scale),
                                          int(k_cache.shape[0]), int(k_cache.stride(0)), int(k_scale.stride(0)) * 4,
                                          _stream(dev))
        _check(rc, self._lib)

    def v_store_paged(self, v_fp16, slot_mapping, v_cache, v_scale, v_zero):
        """The V half of :meth:`kv_store_paged` (xe2_kv_ops.cpp:1391-1409)."""
        _require(v_fp16.dim() == 3 and int(v_fp16.shape[2]) in (128, 256), "v_fp16 [T,HKV,D] with D in (128, 256)")
        head_dim = int(v_fp16.shape[2])
        _require(slot_mapping.dtype == torch.int64 and slot_mapping.is_contiguous(), "slot_mapping int64")
        hkv = _checked_hkv(int(v_fp16.shape[1]))
        check_paged_v(v_cache, v_scale, v_zero, hkv, head_dim)
        _require(slot_mapping.numel() == v_fp16.shape[0], "slot_mapping [T]")
        vs = _src_rows(v_fp16, "v_fp16", hkv, head_dim)
        if v_fp16.shape[0] == 0:
            return
        dev = _on_gpu(v_fp16, slot_mapping, v_cache, v_scale, v_zero)
        rc = self._lib.k8v4_v_store_paged(_ptr(v_fp16), _DTYPE_CODE[v_fp16.dtype], vs, _ptr(slot_mapping),
                                          int(v_fp16.shape[0]), hkv, head_dim, _ptr(v_cache), _ptr(v_scale),
                                          _ptr(v_zero), int(v_cache.shape[0]), int(v_cache.stride(0)),
                                          int(v_scale.stride(0)) * 4, int(v_zero.stride(0)) * 4, _stream(dev))
        _check(rc, self._lib)

    # -- reading the cache back ----------------------------------------------
    def kv_load_paged(self, k_cache, k_scale, v_cache, v_scale, v_zero, block_table, seq_starts, row_starts,
                      pages_per_block, k_out, v_out):
        """The inverse of :meth:`kv_store_paged`: cached K/V rows of a ragged batch, dequantized.

        Sequence b's tokens from ``seq_starts[b]`` (int32 ``[B]``; None: 0) on go to
        rows ``row_starts[b] .. row_starts[b + 1] - 1`` (int32 ``[B + 1]``, not
        decreasing) of ``k_out`` / ``v_out`` ``[N, HKV, D]`` (fp16, bf16 or fp32;
        either may be None), its pages in ``block_table[b]``.  A token outside its
        table row or on a page outside the cache gives zeros; rows that belong to
        no sequence are left as they were."""
        bound = self.bind_kv_load_paged(k_cache, k_scale, v_cache, v_scale, v_zero, block_table, seq_starts,
                                        row_starts, pages_per_block, k_out, v_out)
        if bound is not None:
            bound()

    def bind_kv_load_paged(self, k_cache, k_scale, v_cache, v_scale, v_zero, block_table, seq_starts, row_starts,
                           pages_per_block, k_out, v_out):
        """Validate a read once; returns a :class:`DeviceCall` (None when there are no rows)."""
        out = v_out if k_out is None else k_out
        _require(out is not None, "k_out or v_out")
        hkv, head_dim, cache = _checked_cache(k_cache, k_scale, v_cache, v_scale, v_zero)
        _require(block_table.dtype == torch.int32 and block_table.dim() == 2 and block_table.stride(1) == 1,
                 "block_table must be int32 [B, W] with unit column stride")
        batch, width = block_table.shape
        _require(row_starts.dtype == torch.int32 and row_starts.shape == (batch + 1,) and row_starts.is_contiguous(),
                 "row_starts must be a contiguous int32 [B + 1]")
        if seq_starts is not None:
            _require(seq_starts.dtype == torch.int32 and seq_starts.shape == (batch,) and seq_starts.is_contiguous(),
                     "seq_starts must be a contiguous int32 [B]")
        _require(int(pages_per_block) >= 1, "pages_per_block")
        rows, dtype = out.shape[0] if out.dim() else -1, out.dtype
        _require(dtype in _DTYPE_CODE, "k/v_out float16, bfloat16 or float32")
        for x in (k_out, v_out):
            if x is not None and not (
                x.dtype == dtype and x.shape == (rows, hkv, head_dim) and x.stride()[1:] == (head_dim, 1)
            ):
                _require(x.dtype == dtype, "k/v_out dtypes differ")
                _require(x.shape == (rows, hkv, head_dim), "k/v_out [N,%d,%d]" % (hkv, head_dim))
                _require(False, "k/v_out head/dim strides")
        if rows == 0 or batch == 0:
            return None
        _require(width > 0, "block_table width")
        tensors = (k_cache, k_scale, v_cache, v_scale, v_zero, block_table, row_starts)
        tensors += tuple(x for x in (k_out, v_out, seq_starts) if x is not None)
        dev = _on_gpu(*tensors)
        row = hkv * head_dim
        args = (
            *cache, block_table.data_ptr(), block_table.stride(0), width, int(pages_per_block),
            0 if seq_starts is None else seq_starts.data_ptr(), row_starts.data_ptr(), batch, hkv, head_dim,
            0 if k_out is None else k_out.data_ptr(), 0 if v_out is None else v_out.data_ptr(), _DTYPE_CODE[dtype],
            row if k_out is None or rows == 1 else k_out.stride(0),
            row if v_out is None or rows == 1 else v_out.stride(0), rows,
        )
        return DeviceCall(self._lib, self._lib.k8v4_kv_load_paged, args, dev, tensors)

    # -- verification of drafted tokens ----------------------------------------
    def verify_drafts_workspace_bytes(self, batch: int, vocab: int) -> int:
        """Scratch bytes :meth:`verify_drafts` needs (any number of drafts)."""
        n = int(self._lib.k8v4_verify_drafts_workspace_bytes(int(batch), int(vocab)))
        _require(n >= 0, "bad shape for the verify workspace")
        return n

    def verify_drafts(self, target_probs, draft_probs, draft_tokens, num_drafts, accept_uniform, sample_uniform,
                      seq_lens, workspace, out_tokens, accepted, next_lens):
        """Accept or refuse a step's drafted tokens and sample the token after them.

        ``target_probs`` ``[B, K + 1, V]`` and ``draft_probs`` ``[B, K, V]`` (None: the
        drafts were chosen outright) of one dtype (fp16, bf16, fp32); ``draft_tokens``
        int32 or int64 ``[B, K]``; ``num_drafts`` int32 ``[B]`` (None: K each);
        ``accept_uniform`` fp32 ``[B, K]`` and ``sample_uniform`` fp32 ``[B]`` in [0, 1).
        Draft i is accepted iff ``u_i q_i(x_i) < p_i(x_i)``; behind the first refusal
        (or the last draft) one token is drawn from ``max(p - q, 0)`` (or ``p``).
        ``out_tokens`` int64 ``[B, K + 1]``: the accepted drafts, the drawn token, then
        -1; ``accepted`` int32 ``[B]``; ``next_lens`` int32 ``[B]`` (None: not wanted;
        may be ``seq_lens``): ``seq_lens + accepted + 1``, what the next step's
        attention takes.  A row without any positive probability draws -1."""
        bound = self.bind_verify_drafts(target_probs, draft_probs, draft_tokens, num_drafts, accept_uniform,
                                        sample_uniform, seq_lens, workspace, out_tokens, accepted, next_lens)
        if bound is not None:
            bound()

    def bind_verify_drafts(self, target_probs, draft_probs, draft_tokens, num_drafts, accept_uniform,
                           sample_uniform, seq_lens, workspace, out_tokens, accepted, next_lens):
        """Validate a verification once; returns a :class:`DeviceCall` (None for an empty batch)."""
        _require(target_probs.dim() == 3, "target_probs [B,K+1,V]")
        _require(target_probs.dtype in (torch.float16, torch.bfloat16, torch.float32),
                 "target_probs float16, bfloat16 or float32")
        batch, drafts, vocab = int(target_probs.shape[0]), int(target_probs.shape[1]) - 1, int(target_probs.shape[2])
        _require(drafts >= 0 and vocab >= 1, "target_probs [B,K+1,V]")
        _require(target_probs.stride(2) == 1 or vocab == 1, "target_probs rows must be contiguous")
        tensors = (target_probs, draft_tokens, accept_uniform, sample_uniform, workspace, out_tokens, accepted)
        if draft_probs is not None:
            _require(draft_probs.shape == (batch, drafts, vocab), "draft_probs [B,K,V]")
            _require(draft_probs.dtype == target_probs.dtype, "target/draft_probs dtypes differ")
            _require(draft_probs.stride(2) == 1 or vocab == 1, "draft_probs rows must be contiguous")
            tensors += (draft_probs,)
        _require(draft_tokens.dtype in (torch.int32, torch.int64) and draft_tokens.shape == (batch, drafts),
                 "draft_tokens int32 or int64 [B,K]")
        _require(drafts <= 1 or draft_tokens.stride(1) == 1, "draft_tokens rows must be contiguous")
        _require(accept_uniform.dtype == torch.float32 and accept_uniform.shape == (batch, drafts),
                 "accept_uniform float32 [B,K]")
        _require(drafts <= 1 or accept_uniform.stride(1) == 1, "accept_uniform rows must be contiguous")
        _require(sample_uniform.dtype == torch.float32 and sample_uniform.shape == (batch,)
                 and sample_uniform.is_contiguous(), "sample_uniform must be a contiguous float32 [B]")
        _require(out_tokens.dtype == torch.int64 and out_tokens.shape == (batch, drafts + 1)
                 and (drafts == 0 or out_tokens.stride(1) == 1), "out_tokens int64 [B,K+1] with contiguous rows")
        _require(next_lens is None or seq_lens is not None, "next_lens needs seq_lens")
        for name, x in (("num_drafts", num_drafts), ("seq_lens", seq_lens), ("accepted", accepted),
                        ("next_lens", next_lens)):
            if x is not None or name == "accepted":
                _require(x is not None and x.dtype == torch.int32 and x.shape == (batch,) and x.is_contiguous(),
                         "%s must be a contiguous int32 [B]" % name)
                if name != "accepted":
                    tensors += (x,)
        _require(workspace.is_contiguous(), "verify workspace must be a contiguous buffer")
        if batch == 0:
            return None
        dev = _on_gpu(*tensors)
        many = batch > 1
        has_q = draft_probs is not None
        args = [
            _ptr(target_probs), _DTYPE_CODE[target_probs.dtype],
            int(target_probs.stride(0)) if many else vocab * (drafts + 1),
            int(target_probs.stride(1)) if drafts else vocab,
            _ptr(draft_probs) if has_q else 0,
            int(draft_probs.stride(0)) if has_q and many else vocab * max(drafts, 1),
            int(draft_probs.stride(1)) if has_q and drafts > 1 else vocab,
            _ptr(draft_tokens), int(draft_tokens.dtype == torch.int64),
            int(draft_tokens.stride(0)) if many else drafts,
            0 if num_drafts is None else _ptr(num_drafts),
            _ptr(accept_uniform), int(accept_uniform.stride(0)) if many else drafts, _ptr(sample_uniform),
            0 if seq_lens is None else _ptr(seq_lens), batch, drafts, vocab,
            _ptr(out_tokens), int(out_tokens.stride(0)) if many else drafts + 1, _ptr(accepted),
            0 if next_lens is None else _ptr(next_lens),
            _ptr(workspace), int(workspace.numel()) * workspace.element_size(),
        ]
        return DeviceCall(self._lib, self._lib.k8v4_verify_drafts, args, dev, tensors)

    # -- the accepted branch of a drafted tree ------------------------------------
    def accept_tree(self, draft_tokens, parents, target_tokens, seq_lens, path, out_tokens, accepted, next_lens,
                    num_nodes=None):
        """The branch of each drafted tree that the target's tokens confirm.

        ``draft_tokens`` int32 or int64 ``[B, N]`` (N up to 64; node 0 is the sequence's
        last token, its draft is not read); ``parents`` int32 ``[B, N]`` (a row expanded
        over the batch: one tree for all), ``parents[i] < i``; ``target_tokens`` int64
        ``[B, N]``: what the target chose after each node; ``num_nodes`` int32 ``[B]``
        (None: N each).  From node 0 the walk goes to the lowest child whose draft is the
        token chosen at its parent, over at most ``path.shape[1]`` nodes.  ``path`` int32
        ``[B, W]``: its nodes, then -1; ``out_tokens`` int64 ``[B, W]``: the token chosen at
        each, then -1; ``accepted`` int32 ``[B]``: its nodes behind node 0; ``next_lens``
        int32 ``[B]`` (None: not wanted; may be ``seq_lens``): ``seq_lens + accepted + 1``."""
        bound = self.bind_accept_tree(draft_tokens, parents, target_tokens, seq_lens, path, out_tokens, accepted,
                                      next_lens, num_nodes)
        if bound is not None:
            bound()

    def bind_accept_tree(self, draft_tokens, parents, target_tokens, seq_lens, path, out_tokens, accepted, next_lens,
                         num_nodes=None):
        """Validate one acceptance; returns a :class:`DeviceCall` (None for an empty batch)."""
        shape, walk = draft_tokens.shape, path.shape
        whole = seq_lens is not None and next_lens is not None and num_nodes is None
        # The usual call in one condition; any other goes through the checks one by one.
        if not (
            whole and len(shape) == 2 and 1 <= shape[1] <= 64 and draft_tokens.dtype in (torch.int32, torch.int64)
            and parents.dtype == path.dtype == accepted.dtype == seq_lens.dtype == next_lens.dtype == torch.int32
            and target_tokens.dtype == out_tokens.dtype == torch.int64
            and parents.shape == target_tokens.shape == shape and out_tokens.shape == walk and len(walk) == 2
            and walk[0] == shape[0] and 1 <= walk[1] <= shape[1]
            and accepted.shape == seq_lens.shape == next_lens.shape == shape[:1]
            and draft_tokens.is_contiguous() and parents.is_contiguous() and target_tokens.is_contiguous()
            and path.is_contiguous() and out_tokens.is_contiguous() and accepted.is_contiguous()
            and seq_lens.is_contiguous() and next_lens.is_contiguous()
        ):
            self._check_accept(draft_tokens, parents, target_tokens, seq_lens, path, out_tokens, accepted, next_lens,
                               num_nodes)
        batch, nodes = shape
        width = walk[1]
        if batch == 0:
            return None
        tensors = (draft_tokens, parents, target_tokens, path, out_tokens, accepted)
        tensors += tuple(x for x in (seq_lens, next_lens, num_nodes) if x is not None)
        dev = _on_gpu(*tensors)
        many = batch > 1
        args = (
            draft_tokens.data_ptr(), int(draft_tokens.dtype == torch.int64), draft_tokens.stride(0) if many else nodes,
            parents.data_ptr(), parents.stride(0) if many else nodes, 0 if num_nodes is None else num_nodes.data_ptr(),
            target_tokens.data_ptr(), target_tokens.stride(0) if many else nodes,
            0 if seq_lens is None else seq_lens.data_ptr(), batch, nodes, width,
            path.data_ptr(), path.stride(0) if many else width, out_tokens.data_ptr(),
            out_tokens.stride(0) if many else width, accepted.data_ptr(),
            0 if next_lens is None else next_lens.data_ptr(),
        )
        return DeviceCall(self._lib, self._lib.k8v4_accept_tree, args, dev, tensors)

    @staticmethod
    def _check_accept(draft_tokens, parents, target_tokens, seq_lens, path, out_tokens, accepted, next_lens, num_nodes):
        _require(draft_tokens.dim() == 2 and draft_tokens.dtype in (torch.int32, torch.int64),
                 "draft_tokens int32 or int64 [B,N]")
        batch, nodes = (int(x) for x in draft_tokens.shape)
        _require(1 <= nodes <= 64, "1 to 64 nodes a tree")
        _require(parents.dtype == torch.int32 and parents.shape == (batch, nodes), "parents int32 [B,N]")
        _require(target_tokens.dtype == torch.int64 and target_tokens.shape == (batch, nodes), "target_tokens int64 [B,N]")
        _require(path.dtype == torch.int32 and path.dim() == 2 and path.shape[0] == batch, "path int32 [B,W]")
        width = int(path.shape[1])
        _require(1 <= width <= nodes, "path [B,W] with W of 1 .. N")
        _require(out_tokens.dtype == torch.int64 and out_tokens.shape == (batch, width), "out_tokens int64 [B,W]")
        for name, x in (("draft_tokens", draft_tokens), ("parents", parents), ("target_tokens", target_tokens),
                        ("path", path), ("out_tokens", out_tokens)):
            _require(x.shape[1] == 1 or x.stride(1) == 1, "%s rows must be contiguous" % name)
        _require(next_lens is None or seq_lens is not None, "next_lens needs seq_lens")
        for name, x in (("accepted", accepted), ("seq_lens", seq_lens), ("next_lens", next_lens),
                        ("num_nodes", num_nodes)):
            if x is not None or name == "accepted":
                _require(x is not None and x.dtype == torch.int32 and x.shape == (batch,) and x.is_contiguous(),
                         "%s must be a contiguous int32 [B]" % name)

    def kv_keep_paged(self, k_cache, k_scale, v_cache, v_scale, v_zero, block_table, seq_starts, path, accepted,
                      pages_per_block):
        """The cache rows of each accepted branch moved to the places of a linear sequence.

        The tree of sequence b lies in the cache from token ``seq_starts[b]`` (int32
        ``[B]``) on; token ``seq_starts[b] + path[b, i]`` is copied to ``seq_starts[b] + i``
        for i up to ``accepted[b]`` (:meth:`accept_tree` gives ``path`` int32 ``[B, W]`` and
        ``accepted`` int32 ``[B]``), codes and planes unchanged.  Once per layer.  Entries
        ``path[b, i] <= i`` or outside the table or cache move nothing; sequences must not
        share the pages that their trees lie on."""
        bound = self.bind_kv_keep_paged(k_cache, k_scale, v_cache, v_scale, v_zero, block_table, seq_starts, path,
                                        accepted, pages_per_block)
        if bound is not None:
            bound()

    def bind_kv_keep_paged(self, k_cache, k_scale, v_cache, v_scale, v_zero, block_table, seq_starts, path, accepted,
                           pages_per_block):
        """Validate one move; returns a :class:`DeviceCall` (None where there is nothing to move)."""
        hkv, head_dim, cache = _checked_cache(k_cache, k_scale, v_cache, v_scale, v_zero)
        table = block_table.shape
        if not (
            len(table) == 2 and path.dim() == 2 and path.shape[0] == table[0]
            and block_table.dtype == seq_starts.dtype == path.dtype == accepted.dtype == torch.int32
            and seq_starts.shape == accepted.shape == table[:1] and block_table.is_contiguous()
            and path.is_contiguous() and seq_starts.is_contiguous() and accepted.is_contiguous()
        ):
            _require(block_table.dtype == torch.int32 and block_table.dim() == 2 and block_table.stride(1) == 1,
                     "block_table must be int32 [B, W] with unit column stride")
            for name, x in (("seq_starts", seq_starts), ("accepted", accepted)):
                _require(x.dtype == torch.int32 and x.shape == table[:1] and x.is_contiguous(),
                         "%s must be a contiguous int32 [B]" % name)
            _require(path.dtype == torch.int32 and path.dim() == 2 and path.shape[0] == table[0], "path int32 [B,W]")
            _require(path.shape[1] <= 1 or path.stride(1) == 1, "path rows must be contiguous")
        batch, width = path.shape
        _require(int(pages_per_block) >= 1, "pages_per_block")
        if batch == 0 or width == 0:
            return None
        _require(table[1] > 0, "block_table width")
        tensors = (k_cache, k_scale, v_cache, v_scale, v_zero, block_table, seq_starts, path, accepted)
        dev = _on_gpu(*tensors)
        args = (
            *cache, block_table.data_ptr(), block_table.stride(0) if batch > 1 else table[1], table[1], int(pages_per_block),
            seq_starts.data_ptr(), path.data_ptr(), path.stride(0) if batch > 1 else width, width,
            accepted.data_ptr(), batch, hkv, head_dim,
        )
        return DeviceCall(self._lib, self._lib.k8v4_kv_keep_paged, args, dev, tensors)

    # -- log probabilities ---------------------------------------------------------
    def token_logprobs_workspace_bytes(self, rows: int, vocab: int, top: int) -> int:
        """Scratch bytes :meth:`token_logprobs` needs (may be 0)."""
        n = int(self._lib.k8v4_token_logprobs_workspace_bytes(int(rows), int(vocab), int(top)))
        _require(n >= 0, "bad shape for the log probability workspace")
        return n

    def token_logprobs(self, logits, tokens, workspace, logprobs, ranks, entropy, top_ids, top_logprobs):
        """Log probabilities, ranks, entropies and likeliest tokens of rows of logits.

        ``logits`` ``[N, V]`` (fp16, bf16 or fp32, rows of any stride); ``tokens`` int32 or
        int64 ``[N]`` with ``logprobs`` fp32 ``[N]`` and ``ranks`` int32 ``[N]`` (all three
        None: not wanted); ``entropy`` fp32 ``[N]`` (None: not wanted), in nats; ``top_ids``
        int64 and ``top_logprobs`` fp32 ``[N, K]`` (K up to 64; both None: not wanted), the K
        likeliest tokens, of equal logits the lower index first.  Rank 1 is the likeliest
        token.  Logits of minus infinity or NaN have no probability: rank 0, -inf; where a row
        has fewer than K others, ids -1 and -inf.  ``workspace`` holds
        :meth:`token_logprobs_workspace_bytes` bytes (None where that is 0)."""
        bound = self.bind_token_logprobs(logits, tokens, workspace, logprobs, ranks, entropy, top_ids, top_logprobs)
        if bound is not None:
            bound()

    def bind_token_logprobs(self, logits, tokens, workspace, logprobs, ranks, entropy, top_ids, top_logprobs):
        """Validate one call; returns a :class:`DeviceCall` (None for no rows)."""
        shape = logits.shape
        whole = tokens is not None and entropy is not None and top_ids is not None and workspace is not None
        # The usual call in one condition; any other goes through the checks one by one.
        if not (
            whole and len(shape) == 2 and shape[1] >= 1 and logits.dtype in _DTYPE_CODE and logits.stride(1) == 1
            and logprobs is not None and ranks is not None and top_logprobs is not None
            and tokens.dtype in (torch.int32, torch.int64) and ranks.dtype == torch.int32
            and logprobs.dtype == entropy.dtype == top_logprobs.dtype == torch.float32 and top_ids.dtype == torch.int64
            and tokens.shape == logprobs.shape == ranks.shape == entropy.shape == shape[:1]
            and top_ids.dim() == 2 and top_ids.shape[0] == shape[0] and top_ids.shape[1] <= 64
            and top_logprobs.shape == top_ids.shape
            and tokens.is_contiguous() and logprobs.is_contiguous() and ranks.is_contiguous()
            and entropy.is_contiguous() and top_ids.is_contiguous() and top_logprobs.is_contiguous()
            and workspace.is_contiguous()
        ):
            self._check_logprobs(logits, tokens, workspace, logprobs, ranks, entropy, top_ids, top_logprobs)
        rows, vocab = shape
        if rows == 0:
            return None
        top = 0 if top_ids is None else top_ids.shape[1]
        tensors = (logits, tokens, logprobs, ranks, entropy, workspace) + ((top_ids, top_logprobs) if top else ())
        if not whole:
            tensors = tuple(x for x in tensors if x is not None)
        dev = _on_gpu(*tensors)
        many = rows > 1
        args = (
            logits.data_ptr(), _DTYPE_CODE[logits.dtype], logits.stride(0) if many else vocab,
            0 if tokens is None else tokens.data_ptr(), int(tokens is not None and tokens.dtype == torch.int64),
            rows, vocab, top, 0 if tokens is None else logprobs.data_ptr(), 0 if tokens is None else ranks.data_ptr(),
            0 if entropy is None else entropy.data_ptr(),
            top_ids.data_ptr() if top else 0, top_ids.stride(0) if top and many else top,
            top_logprobs.data_ptr() if top else 0, top_logprobs.stride(0) if top and many else top,
            0 if workspace is None else workspace.data_ptr(),
            0 if workspace is None else workspace.numel() * workspace.element_size(),
        )
        return DeviceCall(self._lib, self._lib.k8v4_token_logprobs, args, dev, tensors)

    @staticmethod
    def _check_logprobs(logits, tokens, workspace, logprobs, ranks, entropy, top_ids, top_logprobs):
        _require(logits.dim() == 2 and logits.dtype in _DTYPE_CODE, "logits float16, bfloat16 or float32 [N,V]")
        rows, vocab = logits.shape
        _require(vocab >= 1 and (vocab == 1 or logits.stride(1) == 1), "logits rows must be contiguous")
        _require((tokens is None) == (logprobs is None) and (tokens is None) == (ranks is None),
                 "tokens, logprobs and ranks go together")
        if tokens is not None:
            _require(tokens.dtype in (torch.int32, torch.int64) and tokens.shape == (rows,) and tokens.is_contiguous(),
                     "tokens must be a contiguous int32 or int64 [N]")
            _require(ranks.dtype == torch.int32 and ranks.shape == (rows,) and ranks.is_contiguous(),
                     "ranks must be a contiguous int32 [N]")
        for name, x in (("logprobs", logprobs), ("entropy", entropy)):
            if x is not None:
                _require(x.dtype == torch.float32 and x.shape == (rows,) and x.is_contiguous(),
                         "%s must be a contiguous float32 [N]" % name)
        _require((top_ids is None) == (top_logprobs is None), "top_ids and top_logprobs go together")
        if top_ids is not None:
            _require(top_ids.dtype == torch.int64 and top_ids.dim() == 2 and top_ids.shape[0] == rows, "top_ids int64 [N,K]")
            _require(top_ids.shape[1] <= 64, "0 to 64 likeliest tokens")
            _require(top_logprobs.dtype == torch.float32 and top_logprobs.shape == top_ids.shape, "top_logprobs float32 [N,K]")
            _require(top_ids.shape[1] <= 1 or (top_ids.stride(1) == 1 and top_logprobs.stride(1) == 1),
                     "top_ids/top_logprobs rows must be contiguous")
        if workspace is not None:
            _require(workspace.is_contiguous(), "log probability workspace must be a contiguous buffer")

    # -- the Q-once tile and the ops that read it ----------------------------
    def q_quant_once(self, q_fp16, q8, q_scale):
        """Quantize the padded query tile ``[HKV, 64, D]`` into ``q8`` / ``q_scale`` (xe2_kv_ops.cpp:1248-1265)."""
        _require(q_fp16.dtype in (torch.float16, torch.bfloat16), "q_fp16 must be float16 or bfloat16")
        _require(q_fp16.dim() == 3 and q_fp16.shape[1] == PAGE and int(q_fp16.shape[2]) in (128, 256),
                 "q_fp16 shape [HKV,64,D]")
        _require(q_fp16.is_contiguous(), "q_fp16 must be contiguous")
        hkv = _checked_hkv(int(q_fp16.shape[0]))
        self._quantize_tile(q_fp16, Q_PADDED, 0, 0, hkv, int(q_fp16.shape[2]), q8, q_scale)

    def _quantize_tile(self, q, layout, tok_stride, ntok, hkv, head_dim, q8, q_scale):
        _require(q8.dtype == torch.int8, "q8 must be int8")
        _require(q_scale.dtype == torch.float32, "q_scale must be float32")
        _require(q8.is_contiguous() and q8.numel() == hkv * PAGE * head_dim, "q8 numel [HKV,64,D]")
        _require(q_scale.is_contiguous() and q_scale.numel() == hkv * PAGE, "q_scale numel [HKV,64]")
        dev = _on_gpu(q, q8, q_scale)
        rc = self._lib.k8v4_q_quant(_ptr(q), _DTYPE_CODE[q.dtype], layout, tok_stride, ntok, hkv, head_dim,
                                    _ptr(q8), _ptr(q_scale), _stream(dev))
        _check(rc, self._lib)

    def int8k_int4v_s1_paged(self, q8, q_scale, k_cache, k_scale, v_cache, v_scale, v_zero, block_table, seq_lens,
                             out):
        """One sequence over the paged cache from a Q-once tile, workspace owned by
        the library (the reference's legacy op, xe2_kv_ops.cpp:1628-1639)."""
        self.int8k_int4v_s1_varlen_paged(q8, q_scale, k_cache, k_scale, v_cache, v_scale, v_zero, block_table,
                                         seq_lens, None, None, None, None, None, out, 1)

    def int8k_int4v_s1_varlen_paged(self, q8, q_scale, k_cache, k_scale, v_cache, v_scale, v_zero, block_table,
                                    seq_lens, visible_lens, partials_ws, m_ws, l_ws, merged_ws, out,
                                    pages_per_block: int = 1):
        """One sequence from a Q-once tile with optional explicit causal ends and a
        caller workspace (xe2_kv_ops.cpp:1641-1660).  ``out`` is ``[Tq, HQ, D]``;
        Tq is the query length.  ``m_ws``, ``l_ws`` and ``merged_ws`` are accepted
        and unused; ``partials_ws`` holds the split states (None: the library's
        own buffer, as the reference's legacy op keeps one)."""
        del m_ws, l_ws, merged_ws
        _require(q8.dtype == torch.int8, "q8 int8")
        _require(q_scale.dtype == torch.float32, "q_scale float32")
        _require(k_cache.dim() == 4, "k_cache [num_blocks,64,HKV,D] NHD")
        hkv = _checked_hkv(int(k_cache.shape[2]))
        head_dim = int(k_cache.shape[3])
        _require(head_dim in (128, 256), "k_cache head dim must be 128 or 256")
        check_paged_k(k_cache, k_scale, hkv, head_dim)
        check_paged_v(v_cache, v_scale, v_zero, hkv, head_dim)
        _require(k_cache.shape[0] == v_cache.shape[0], "k/v num_blocks")
        _require(q8.is_contiguous() and q8.numel() == hkv * PAGE * head_dim, "q8 unique [HKV,64,D]")
        _require(q_scale.is_contiguous() and q_scale.numel() == hkv * PAGE, "q_scale numel [HKV,64]")
        _require(block_table.dtype == torch.int32, "block_table int32")
        row = block_table if block_table.dim() == 1 else block_table.reshape(-1, block_table.shape[-1])[0]
        _require(row.numel() > 0 and row.is_contiguous(), "block_table n_splits")
        _require(seq_lens.dtype == torch.int32 and seq_lens.numel() >= 1 and seq_lens.is_contiguous(),
                 "seq_lens int32")
        _require(out.dim() == 3 and out.shape[1] == GQA * hkv and out.shape[2] == head_dim, "out [Tq,HQ,D]")
        _require(out.dtype in (torch.float16, torch.bfloat16, torch.float32), "out float32 or float16")
        _require(out.stride(2) == 1 and out.stride(1) == head_dim, "out head/dim strides")
        tq = int(out.shape[0])
        _require(tq > 0 and tq * GQA <= PAGE, "Tq*GQA must fit BM=64 pad")
        vis_ptr, vis_stride = 0, 0
        if visible_lens is not None and visible_lens.numel() > 0:
            _require(visible_lens.dtype == torch.int32 and visible_lens.numel() >= tq + 1 and
                     visible_lens.is_contiguous(), "visible_lens int32 [1+Tq]")
            vis_ptr, vis_stride = _ptr(visible_lens), tq + 1
        ppb = max(1, int(pages_per_block))
        dev = _on_gpu(q8, q_scale, k_cache, k_scale, v_cache, v_scale, v_zero, row, seq_lens, out)
        need = self.attn_workspace_bytes(1, int(row.numel()), ppb, tq, hkv, head_dim)
        if partials_ws is None:
            ws = self._own_workspace(dev, need)
        else:
            _require(partials_ws.is_contiguous() and partials_ws.device == dev, "partials_ws must be a contiguous "
                     "buffer on the cache's device")
            ws = partials_ws
        rc = self._lib.k8v4_attn_batch_q8(
            _ptr(q8), _ptr(q_scale), hkv * PAGE * head_dim, hkv * PAGE,
            *cache_args(k_cache, k_scale, v_cache, v_scale, v_zero),
            _ptr(row), int(row.numel()), int(row.numel()), ppb, _ptr(seq_lens), vis_ptr, vis_stride, 1, tq, hkv,
            head_dim, _ptr(out), _DTYPE_CODE[out.dtype], int(out.stride(0)) if tq > 1 else GQA * hkv * head_dim,
            _ptr(ws), int(ws.numel()) * ws.element_size(), 0, _stream(dev))
        _check(rc, self._lib)

    def _own_workspace(self, dev, nbytes: int) -> torch.Tensor:
        """The library-owned split-state buffer of the workspace-free legacy op (grows on demand)."""
        have = self._legacy_ws.get(dev)
        if have is None or have.numel() * 4 < nbytes:
            have = self._legacy_ws[dev] = torch.empty(max(4, -(-nbytes // 4)), dtype=torch.int32, device=dev)
        return have

    def int8k_int4v_s1_varlen_from_q(self, q_fp16, q8, q_scale, k_cache, k_scale, v_cache, v_scale, v_zero,
                                     block_table, seq_lens, visible_lens, partials_ws, m_ws, l_ws, merged_ws, out,
                                     pages_per_block: int = 1):
        """Quantize ``q_fp16`` into the Q-once tile (token rows ``[T, HQ, D]`` are
        packed, a padded ``[HKV, 64, D]`` tile is quantized as is), then
        :meth:`int8k_int4v_s1_varlen_paged` (xe2_kv_ops.cpp:1663-1712)."""
        _require(q_fp16.dtype in (torch.float16, torch.bfloat16), "q_fp16 must be float16 or bfloat16")
        _require(k_cache.dim() == 4, "k_cache [num_blocks,64,HKV,D] NHD")
        hkv = _checked_hkv(int(k_cache.shape[2]))
        head_dim = int(k_cache.shape[3])
        if q_fp16.dim() == 3 and q_fp16.shape[1] == GQA * hkv and q_fp16.shape[2] == head_dim:
            tq = int(q_fp16.shape[0])
            _require(tq > 0 and tq * GQA <= PAGE, "tq*GQA exceeds BM")
            _require(q_fp16.stride(2) == 1 and q_fp16.stride(1) == head_dim, "q_fp16 head/dim strides")
            self._quantize_tile(q_fp16, Q_TOKENS, int(q_fp16.stride(0)) if tq > 1 else GQA * hkv * head_dim, tq,
                                hkv, head_dim, q8, q_scale)
        else:
            _require(q_fp16.numel() == hkv * PAGE * head_dim and q_fp16.is_contiguous(), "q_fp16 numel")
            self._quantize_tile(q_fp16, Q_PADDED, 0, 0, hkv, head_dim, q8, q_scale)
        self.int8k_int4v_s1_varlen_paged(q8, q_scale, k_cache, k_scale, v_cache, v_scale, v_zero, block_table,
                                         seq_lens, visible_lens, partials_ws, m_ws, l_ws, merged_ws, out,
                                         pages_per_block)

    def int8k_int4v_decode_step(self, q_fp16, k_fp16, v_fp16, slot_mapping, q8, q_scale, k_cache, k_scale, v_cache,
                                v_scale, v_zero, block_table, seq_lens, visible_lens, partials_ws, m_ws, l_ws,
                                merged_ws, out):
        """One decode step of one sequence: store the new K/V, then attend
        (xe2_kv_ops.cpp:1716-1731)."""
        self.kv_store_paged(k_fp16, v_fp16, slot_mapping, k_cache, k_scale, v_cache, v_scale, v_zero)
        self.int8k_int4v_s1_varlen_from_q(q_fp16, q8, q_scale, k_cache, k_scale, v_cache, v_scale, v_zero,
                                          block_table, seq_lens, visible_lens, partials_ws, m_ws, l_ws, merged_ws,
                                          out)

    # -- the reference's unpaged single-page stage tests ---------------------
    _UNPAGED = ("%s: the reference's unpaged single-page op (contiguous [64, 256] K/V rows, per-page partial "
                "outputs) is a stage test of its own kernels and is not part of this library; use %s")

    def k_store(self, *args, **kwargs):
        raise RuntimeError(self._UNPAGED % ("k_store", "k_store_paged or kv_store_paged"))

    def v_store(self, *args, **kwargs):
        raise RuntimeError(self._UNPAGED % ("v_store", "v_store_paged or kv_store_paged"))

    def int8k_int4v_s1(self, *args, **kwargs):
        raise RuntimeError(self._UNPAGED % ("int8k_int4v_s1", "int8k_int4v_s1_paged"))


def ops() -> _Ops:
    """The op table, after loading the library named by :func:`library_path`."""
    global _OPS
    lib = load_library()
    if _OPS is None or _OPS._lib is not lib:
        _OPS = _Ops(lib)
    return _OPS


__all__ = ["BoundCall", "GQA", "PAGE", "library_path", "load_library", "ops", "check_paged_k", "check_paged_v"]
