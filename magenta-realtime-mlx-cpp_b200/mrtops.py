"""Python bindings of the operators on device buffers (include/mrtdf.h,
"operators") for torch CUDA tensors, in the same library as mrtdf.py. The
calls go through lib/_mrtops.so (bind/mrtops_torch.cpp).

``tree_attention`` attends a tree of drafted tokens (or one token) over a KV
cache, ``cache_mass`` collects each cached row's attention weight,
``cache_commit`` appends an accepted path, ``cache_evict`` drops the rows with
the least weight, ``q4_quantize`` / ``q4_linear`` multiply by 4-bit weights.
``stream_cache`` shows a decoding stream's own KV cache as tensors.

Every call queues its kernels on the current torch stream of the tensors'
device and returns without waiting; it may be captured into a CUDA graph.
Outputs that are not given are new tensors, workspaces come from torch's
allocator per call, so calls on several streams do not share any. float32 and
bfloat16; the operators have no gradients (an input that requires one is
refused while gradients are on, one with a forward-mode tangent while those
are). Errors raise ``mrtdf.MrtdfError``.
"""
from __future__ import annotations

import ctypes
import importlib.util
import os
import struct
from typing import Optional, Tuple

import torch

import mrtdf

# sizeof-exact layouts of C structures (native alignment).
_CACHE = struct.Struct("@QQQ4q7iQQQ")
_PACK = struct.Struct("@QQQQQq5i0Q")

_DTYPES = {torch.float32: mrtdf.DTYPE_FP32, torch.bfloat16: mrtdf.DTYPE_BF16}
MAX_NODES = 64
MAX_Q4_ROWS = 64

_L = None


def lib() -> ctypes.CDLL:
    global _L
    if _L is None:
        L = mrtdf.lib()
        L.mrtdf_q4_quantize.argtypes = [ctypes.c_char_p, ctypes.c_void_p]
        L.mrtdf_stream_cache.argtypes = [ctypes.c_void_p, ctypes.c_int, ctypes.c_int, ctypes.c_char_p,
                                         ctypes.POINTER(ctypes.c_int)]
        _L = L
    return _L


def _load():
    """The extension module lib/_mrtops.so (bind/mrtops_torch.cpp)."""
    path = os.path.join(mrtdf.HERE, "lib", "_mrtops.so")
    if not os.path.exists(path):
        raise mrtdf.MrtdfError(-1, f"{path} is missing: run magenta-realtime-mlx-cpp_b200/build.py")
    spec = importlib.util.spec_from_file_location("_mrtops", path)
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    m.set_error(mrtdf.MrtdfError)
    return m


_ops = _load()


def _invalid(msg: str):
    raise mrtdf.MrtdfError(1, msg)


def _check(rc: int) -> None:
    if rc:
        mrtdf._check(rc)


def tree_attention(q: torch.Tensor, k_new: torch.Tensor, v_new: torch.Tensor, k_cache: torch.Tensor,
                   v_cache: torch.Tensor, lens: torch.Tensor, parents: Optional[torch.Tensor] = None, *,
                   scale: float = 1.0, rel_bias: Optional[torch.Tensor] = None, pos: Optional[torch.Tensor] = None,
                   next_pos: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None,
                   lse: Optional[torch.Tensor] = None,
                   workspace: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """Attention of ``nodes`` drafted tokens over a KV cache (mrtdf_tree_attention).

    q (batch, heads, nodes, head_dim); k_new, v_new (batch, kv_heads, nodes,
    head_dim): any strides with contiguous rows, so views of a fused projection
    do. k_cache, v_cache (batch, kv_heads, capacity, head_dim); lens (batch)
    int32 rows in use. parents (batch, nodes) int32: the node above, -1 for the
    last cached token, anything else outside [-1, i) for a padded node; None is
    a chain (and a plain decode step for one node). rel_bias (heads, rel_len)
    float32 is added at the clamped distance; pos (batch, kv_heads, capacity)
    and next_pos (batch) int32 are positions where rows do not lie in order.
    Returns (out, lse): out like q (contiguous unless given), lse (batch, heads,
    nodes) float32. ``workspace``: a byte tensor to use instead of a new one."""
    return _ops.tree_attention(q, k_new, v_new, k_cache, v_cache, lens, parents, scale, rel_bias, pos, next_pos, out, lse,
                               workspace)


def cache_mass(q: torch.Tensor, lse: torch.Tensor, k_new: torch.Tensor, k_cache: torch.Tensor, lens: torch.Tensor,
               path: torch.Tensor, mass: torch.Tensor, *, scale: float = 1.0, rel_bias: Optional[torch.Tensor] = None,
               pos: Optional[torch.Tensor] = None, next_pos: Optional[torch.Tensor] = None, decay: float = 1.0,
               mass_out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Adds the attention weight that the accepted path gives to each row
    (mrtdf_cache_mass): mass_out = decay * mass + sum over path rows and query
    heads of exp(x - lse) for rows in use, and the sums alone for the rows that
    cache_commit will append. q, lse, k_new as in the verification, with the
    layers in front where the cache has them; path (batch, path_len) int32 ended
    by -1; mass (..., batch, kv_heads, capacity) float32. In place unless
    mass_out is given; returns mass_out."""
    return _ops.cache_mass(q, lse, k_new, k_cache, lens, path, mass, scale, rel_bias, pos, next_pos, decay, mass_out)


def cache_commit(k_new: torch.Tensor, v_new: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                 lens: torch.Tensor, path: torch.Tensor, *, pos: Optional[torch.Tensor] = None,
                 next_pos: Optional[torch.Tensor] = None, lens_out: Optional[torch.Tensor] = None,
                 next_pos_out: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """Appends the accepted path's rows to the cache of every layer, in place
    (mrtdf_cache_commit); pos, where given, gets the rows' positions. Returns
    (lens_out, next_pos_out), new tensors unless given (next_pos_out is None
    without next_pos)."""
    return _ops.cache_commit(k_new, v_new, k_cache, v_cache, lens, path, pos, next_pos, lens_out, next_pos_out)


def cache_evict(k_cache: torch.Tensor, v_cache: torch.Tensor, lens: torch.Tensor, mass: torch.Tensor,
                pos: torch.Tensor, next_pos: torch.Tensor, *, budget: int, recent: int = 0, sinks: int = 0,
                mass_out: Optional[torch.Tensor] = None, pos_out: Optional[torch.Tensor] = None,
                lens_out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Drops all but ``budget`` rows of every longer sequence, per layer and kv
    head (mrtdf_cache_evict): positions of the last ``recent`` tokens and the
    first ``sinks`` stay, then the rows with the largest mass. Moves K, V, mass
    and pos in place (mass and pos to mass_out and pos_out where given); returns
    lens_out, a new tensor unless given."""
    return _ops.cache_evict(k_cache, v_cache, lens, mass, pos, next_pos, budget, recent, sinks, mass_out, pos_out, lens_out)


def q4_linear(x: torch.Tensor, packed: torch.Tensor, scales: torch.Tensor, biases: torch.Tensor, *,
              out: Optional[torch.Tensor] = None, out_dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """x (m, k) times 4-bit weights (n, k) (mrtdf_q4_linear): packed (n, k / 2)
    uint8, scales and biases (n, k / group) of x's dtype. out (m, n) of
    out_dtype (x's, or float32)."""
    if out_dtype is not None and (out_dtype not in _DTYPES or (out is not None and out.dtype != out_dtype)):
        _invalid("out_dtype must be float32 or bfloat16, and that of out")
    if out is None and out_dtype is torch.bfloat16 and x.dtype is not torch.bfloat16:
        _invalid("float32 x gives float32 out")
    return _ops.q4_linear(x, packed, scales, biases, out, out_dtype is torch.float32)


def q4_quantize(w: torch.Tensor, group: int = 64) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """(packed, scales, biases) of float32 or bfloat16 weights (n, k), as
    q4_linear takes them (mrtdf_q4_quantize)."""
    if w.requires_grad and torch.is_grad_enabled():
        _invalid("w requires a gradient, which the operators do not give")
    if torch.autograd.forward_ad.unpack_dual(w).tangent is not None:
        _invalid("w has a forward-mode tangent, which the operators do not carry on")
    if w.dim() != 2 or w.stride(1) != 1:
        _invalid("w must be (n, k) with contiguous rows")
    n, k = w.shape
    if group not in (32, 64, 128) or n < 1 or k < 1 or k % group:
        _invalid("group must be 32, 64 or 128 and divide k")
    code = _DTYPES.get(w.dtype)
    if code is None or not w.is_cuda:
        _invalid(f"w must be float32 or bfloat16 on a CUDA device, is {w.dtype} on {w.device}")
    dev = w.device
    packed = torch.empty((n, k // 2), dtype=torch.uint8, device=dev)
    scales = torch.empty((n, k // group), dtype=w.dtype, device=dev)
    biases = torch.empty_like(scales)
    _check(lib().mrtdf_q4_quantize(_PACK.pack(_PACK.size, w.data_ptr(), packed.data_ptr(), scales.data_ptr(),
                                              biases.data_ptr(), w.stride(0), n, k, group, code, dev.index),
                                   torch.cuda.current_stream(dev).cuda_stream))
    return packed, scales, biases


class _Borrowed:
    """Device memory of a stream, as the CUDA array interface shows it (16-bit
    elements as whole numbers). Keeps the stream alive."""

    def __init__(self, owner, ptr: int, shape, esize: int):
        self._owner = owner
        self.__cuda_array_interface__ = {"shape": shape, "typestr": "<f4" if esize == 4 else "<i2", "data": (ptr, False),
                                         "version": 3, "strides": None, "stream": None}


def stream_cache(stream: mrtdf.Stream, kind: int) -> Tuple[torch.Tensor, torch.Tensor, int]:
    """(k, v, rows in use) of a decoding stream's KV cache (mrtdf_stream_cache):
    kind 0 temporal self, 1 depth self, 2 cross attention; k and v are
    (layers, rows, heads, capacity, 64) tensors over the stream's own memory,
    valid until ``stream.close()``. The stream's kernels run on its own CUDA
    stream: wait for it (``stream.sync()``) before reading here."""
    raw, n = ctypes.create_string_buffer(_CACHE.size), ctypes.c_int()
    _check(lib().mrtdf_stream_cache(stream.h, kind, -1, raw, ctypes.byref(n)))
    f = _CACHE.unpack(raw.raw)
    shape, dtype, dev = tuple(f[7:12]), f[12], f[13]
    esize = 4 if dtype == mrtdf.DTYPE_FP32 else 2
    pair = []
    for ptr in f[1:3]:
        t = torch.as_tensor(_Borrowed(stream, ptr, shape, esize), device=f"cuda:{dev}")
        pair.append(t if esize == 4 else t.view(torch.bfloat16))
    return pair[0], pair[1], n.value
