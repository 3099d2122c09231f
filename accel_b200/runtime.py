"""Direct dispatch of the sm_100a kernels on torch-owned device memory.

torch supplies device memory and streams; every computation is one `ab_launch` through the C ABI.
The binding order, the lengths block and the std140 uniform bytes are the reference's
(internal/kernels/accel_kernels.go codecs; specs/061-ptx-target.md:152-159)."""
from __future__ import annotations

import ctypes as C
import functools
import struct
from typing import List, Optional, Sequence

import torch

from . import _lib

# ---------------------------------------------------------------- std140 uniform blocks


def gemm_dims(M: int, N: int, K: int) -> bytes:                 # GEMMDims, gemm.go:11
    return struct.pack("<IIII", M, N, K, 0)


def attn_dims(q_heads, kv_heads, head_dim, scale) -> bytes:     # AttnDims
    return struct.pack("<IIIf", q_heads, kv_heads, head_dim, scale)


def paged_dims(q_heads, kv_heads, head_dim, block, scale) -> bytes:     # PagedDims, paged.go:16
    return struct.pack("<IIIIfIII", q_heads, kv_heads, head_dim, block, scale, 0, 0, 0)


def batched_dims(batch, q_heads, kv_heads, head_dim, block, max_pages, scale) -> bytes:
    # BatchedDims / RaggedDims, batched.go:13, ragged.go:17
    return struct.pack("<IIIIIIfI", batch, q_heads, kv_heads, head_dim, block, max_pages, scale, 0)


def prefill_dims(q_heads, kv_heads, head_dim, q_seq, base, scale) -> bytes:         # PrefillDims, prefill.go:18
    return struct.pack("<IIIIIfII", q_heads, kv_heads, head_dim, q_seq, base, scale, 0, 0)


def paged_prefill_dims(q_heads, kv_heads, head_dim, q_seq, base, block, scale) -> bytes:
    # PagedPrefillDims, prefill.go:368
    return struct.pack("<IIIIIIfI", q_heads, kv_heads, head_dim, q_seq, base, block, scale, 0)


_window_dims = struct.Struct("<IIIIIIfIIIII").pack


def window_dims(batch, q_heads, kv_heads, head_dim, block, max_pages, scale, window, sinks, capacity, q_seq, base) -> bytes:
    # WindowDims: the window forms' own block
    return _window_dims(batch, q_heads, kv_heads, head_dim, block, max_pages, scale, window, sinks,
                       capacity, q_seq, base)


def logprob_dims(vocab, rows, targets, top) -> bytes:
    return struct.pack("<IIII", vocab, rows, targets, top)


def grouped_dims(experts, K, N) -> bytes:                       # GroupedDims, grouped.go:10
    return struct.pack("<IIII", experts, K, N, 0)


def grouped_tiled_dims(experts, tokens, K, N) -> bytes:         # GroupedTiledDims
    return struct.pack("<IIII", experts, tokens, K, N)


def segment_dims(rows) -> bytes:                                # SegmentDims, segment.go
    return struct.pack("<IIII", rows, 0, 0, 0)


def row_params(rows, width, capacity) -> bytes:                 # RowParams, elementwise.go
    return struct.pack("<IIII", rows, width, capacity, 0)


def row_dims(rows, width, eps) -> bytes:                        # RowDims, norm.go
    return struct.pack("<IIfI", rows, width, eps, 0)


def rope_params(rows, width, rotary_dim, base) -> bytes:        # RoPEParams, elementwise.go
    return struct.pack("<IIIf", rows, width, rotary_dim, base)


def sample_dims(vocab, rows) -> bytes:                          # SampleDims, sample.go
    return struct.pack("<IIII", vocab, rows, 0, 0)


def row_sample_dims(vocab, rows, history=0, slots=0) -> bytes:  # RowSampleDims, rowsample.go:25
    return struct.pack("<IIII", vocab, rows, history, slots)


def top_dims(vocab, k=0, p=0.0) -> bytes:                        # TopDims, topk.go:10
    return struct.pack("<IIfI", vocab, k, p, 0)


def penalty_dims(vocab, history, count, repetition, presence, frequency) -> bytes:   # PenaltyDims, penalty.go:15
    return struct.pack("<IIIfffII", vocab, history, count, repetition, presence, frequency, 0, 0)


# ---------------------------------------------------------------- launch
_workspaces: dict = {}


def kernel_names():
    L = _lib.lib()
    return [L.ab_kernel_name(i).decode() for i in range(L.ab_kernel_count())]


def workspace_bytes(name: str, lengths: Sequence[int], uniform: Optional[bytes]) -> int:
    L = _lib.lib()
    lens = (C.c_uint32 * len(lengths))(*lengths)
    out = C.c_size_t(0)
    ub = uniform or b""
    _lib.check(L.ab_workspace_bytes(name.encode(), lens, len(lengths), ub if ub else None,
                                    len(ub), C.byref(out)))
    return out.value


def _workspace(device: torch.device, need: int) -> Optional[torch.Tensor]:
    if need == 0:
        return None
    key = (device.index, torch.cuda.current_stream(device).cuda_stream)
    ws = _workspaces.get(key)
    if ws is None or ws.numel() < need:
        ws = torch.empty(max(need, 1 << 20), dtype=torch.uint8, device=device)
        _workspaces[key] = ws
    return ws


def launch(name: str, bindings: Sequence[torch.Tensor], uniform: Optional[bytes] = None,
           lengths: Optional[Sequence[int]] = None, workspace: Optional[torch.Tensor] = None):
    """One dispatch of reference kernel `name` on the current stream of the tensors' device.
    `lengths` defaults to each tensor's element count."""
    L = _lib.lib()
    if not bindings:
        raise ValueError("no bindings")
    dev = bindings[0].device
    if dev.type != "cuda":
        raise _lib.AccelError(_lib.AB_ERR_NO_DEVICE, f"{name}: bindings live on {dev}; this backend "
                              "runs on a CUDA device and has no CPU path")
    for t in bindings:
        if t.device != dev or not t.is_contiguous():
            raise ValueError(f"{name}: every binding is a contiguous tensor on {dev}")
    lens = list(lengths) if lengths is not None else [t.numel() for t in bindings]
    ub = uniform or b""
    if workspace is None:
        workspace = _workspace(dev, workspace_bytes(name, lens, uniform))
    ptrs = (C.c_void_p * len(bindings))(*[t.data_ptr() for t in bindings])
    clens = (C.c_uint32 * len(lens))(*lens)
    with torch.cuda.device(dev):
        stream = torch.cuda.current_stream(dev).cuda_stream
        rc = L.ab_launch(name.encode(), C.c_void_p(stream), ptrs, clens, len(bindings),
                         ub if ub else None, len(ub),
                         C.c_void_p(workspace.data_ptr()) if workspace is not None else None,
                         workspace.numel() if workspace is not None else 0)
    _lib.check(rc)


# the current stream's handle without the Stream object around it, where torch offers that
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda i: torch.cuda.current_stream(i).cuda_stream)


_encoded = functools.lru_cache(None)(str.encode)


# a call's pointers and lengths as the bytes of C arrays, by how many there are
_pointers = [struct.Struct(f"{n}Q").pack for n in range(16)]
_counts = [struct.Struct(f"{n}I").pack for n in range(16)]


# the current device's number, where torch offers it without a look at whether CUDA is up
_current_device = getattr(torch._C, "_cuda_getDevice", None) or torch.cuda.current_device


def launch_own(name: str, bindings: Sequence[Optional[torch.Tensor]], uniform: bytes, scratch: bool = False,
               lens: Optional[List[int]] = None):
    """`launch` for the operators whose scratch memory (scratch: they may need some) is the call's own:
    it comes from torch's allocator, so a call captured into a CUDA graph keeps it in that graph's pool
    and two graphs, or two streams, never share it.  The bindings are contiguous: the caller has seen to
    that, and the first is a tensor on a device.  A caller that knows how many elements each has says so (lens).  A binding of
    None is empty; one of more elements than 32 bits count is passed as 0xffffffff, which those kernels read as that many or
    more."""
    index = bindings[0].get_device()
    if index < 0:
        raise _lib.AccelError(_lib.AB_ERR_NO_DEVICE, f"{name}: bindings live on {bindings[0].device}; this backend "
                              "runs on a CUDA device and has no CPU path")
    if index != _current_device():
        with torch.cuda.device(index):
            return launch_own(name, bindings, uniform, scratch, lens)
    if lens is None:
        lens = [0 if t is None else min(t.numel(), 0xffffffff) for t in bindings]
    ptrs = []
    for t, n in zip(bindings, lens):
        if n == 0:
            ptrs.append(0)
            continue
        if t.get_device() != index:
            raise ValueError(f"{name}: every binding is a contiguous tensor on {bindings[0].device}")
        ptrs.append(t.data_ptr())
    count, counts, ws, ws_bytes = len(ptrs), _counts[len(ptrs)](*lens), None, 0
    if scratch:
        need = C.c_size_t(0)
        rc = _lib.lib().ab_workspace_bytes(_encoded(name), counts, count, uniform, len(uniform), C.byref(need))
        if rc:
            _lib.check(rc)
        ws_bytes = need.value
        if ws_bytes:
            ws = bindings[0].new_empty(ws_bytes, dtype=torch.uint8)
    rc = _lib.lib().ab_launch(_encoded(name), _raw_stream(index), _pointers[count](*ptrs), counts, count, uniform, len(uniform),
                              ws.data_ptr() if ws is not None else None, ws_bytes)
    if rc:
        _lib.check(rc)


def copy_pages(caches: Sequence[torch.Tensor], pointers: Sequence[int], src: Sequence[int], dst: Sequence[int], block: int):
    """ab_cache_copy_pages on the current stream of the caches' device; pointers: the caches' addresses."""
    t, n = caches[0], len(src)
    dev = t.device
    if dev.type != "cuda":
        raise _lib.AccelError(_lib.AB_ERR_NO_DEVICE, f"copy_pages: the caches live on {dev}; this backend runs on a CUDA "
                              "device and has no CPU path")
    if dev.index != _current_device():
        with torch.cuda.device(dev):
            return copy_pages(caches, pointers, src, dst, block)
    page_bytes = t.numel() // t.shape[0] * t.element_size() * block if t.numel() else 0
    if page_bytes == 0:
        if n:
            raise _lib.AccelError(_lib.AB_ERR_INVALID, "copy_pages: the caches are empty")
        return
    try:
        s, d = struct.pack(f"{n}I", *src), struct.pack(f"{n}I", *dst)
    except struct.error as e:
        raise _lib.AccelError(_lib.AB_ERR_INVALID, f"copy_pages: a page id is u32: {e}") from None
    rc = _lib.lib().ab_cache_copy_pages(_raw_stream(dev.index), struct.pack(f"{len(pointers)}Q", *pointers), len(pointers),
                                        page_bytes, t.shape[0] // block, s, d, n)
    if rc:
        _lib.check(rc)


def attention_error():
    """Raises once a bounded device-side wait of a windowed prefill has run out (synchronous; sticky)."""
    _lib.check(_lib.lib().ab_attention_error())


def last_selection() -> str:
    return _lib.lib().ab_last_selection().decode()


def launch_count() -> int:
    """Kernels this library has launched (or recorded into a capture) so far in this process."""
    return int(_lib.lib().ab_launch_count())
