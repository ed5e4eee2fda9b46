"""Python bindings of the operators on device buffers (include/mrtdf.h,
"operators") over ctypes, for torch CUDA tensors, in the same library as
mrtdf.py.

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
refused while gradients are on). Errors raise ``mrtdf.MrtdfError``.
"""
from __future__ import annotations

import ctypes
import struct
from typing import Optional, Tuple

import torch

import mrtdf

# sizeof-exact layouts of the C structures (native alignment).
_CACHE = struct.Struct("@QQQ4q7iQQQ")
_TREE = struct.Struct("@Q" + "Q4q" * 4 + "QQQQQiiif0Q")
_MASS = struct.Struct("@Q" + "Q4q" * 2 + "QQQQQiiiiff0Q")
_COMMIT = struct.Struct("@Q" + "Q4q" * 2 + "QQQii0Q")
_EVICT = struct.Struct("@QQQQQiii0Q")
_Q4 = struct.Struct("@QQQQQQqq7i0Q")
_PACK = struct.Struct("@QQQQQq5i0Q")

_DTYPES = {torch.float32: mrtdf.DTYPE_FP32, torch.bfloat16: mrtdf.DTYPE_BF16}
MAX_NODES = 64
MAX_Q4_ROWS = 64

_L = None
_workspace_bytes: dict = {}


def lib() -> ctypes.CDLL:
    global _L
    if _L is None:
        L = mrtdf.lib()
        two = [ctypes.c_char_p, ctypes.c_char_p, ctypes.c_void_p]
        for n in ("tree_attention", "cache_mass", "cache_commit", "cache_evict"):
            getattr(L, "mrtdf_" + n).argtypes = two
        L.mrtdf_tree_attention_workspace.argtypes = [ctypes.c_char_p, ctypes.c_char_p, ctypes.POINTER(ctypes.c_size_t)]
        L.mrtdf_q4_linear.argtypes = [ctypes.c_char_p, ctypes.c_void_p]
        L.mrtdf_q4_quantize.argtypes = [ctypes.c_char_p, ctypes.c_void_p]
        L.mrtdf_stream_cache.argtypes = [ctypes.c_void_p, ctypes.c_int, ctypes.c_int, ctypes.c_char_p,
                                         ctypes.POINTER(ctypes.c_int)]
        _L = L
    return _L


def _invalid(msg: str):
    raise mrtdf.MrtdfError(1, msg)


def _rows(t: torch.Tensor, shape, like: torch.Tensor, name: str):
    """(pointer, four strides) of a (..., n, head_dim) tensor."""
    if t.shape != shape:
        _invalid(f"{name} must be {tuple(shape)}, is {tuple(t.shape)}")
    if t.dtype != like.dtype or t.device != like.device:
        _invalid(f"{name} must be {like.dtype} on {like.device}, is {t.dtype} on {t.device}")
    if t.requires_grad and torch.is_grad_enabled():
        _invalid(f"{name} requires a gradient, which the operators do not give")
    st = t.stride()
    if st[-1] != 1:
        _invalid(f"{name}: elements of a row must lie next to each other")
    return (t.data_ptr(), 0, *st[:-1]) if len(st) == 4 else (t.data_ptr(), *st[:-1])


def _flat(t: Optional[torch.Tensor], shape, dtype, device, name: str) -> int:
    """Pointer of a contiguous tensor (0 for None)."""
    if t is None:
        return 0
    if t.shape != shape or t.dtype != dtype or t.device != device:
        _invalid(f"{name} must be {dtype} {tuple(shape)} on {device}, is {t.dtype} {tuple(t.shape)} on {t.device}")
    if not t.is_contiguous():
        _invalid(f"{name} must be contiguous")
    if t.requires_grad and torch.is_grad_enabled():
        _invalid(f"{name} requires a gradient, which the operators do not give")
    return t.data_ptr()


def _cache(k: torch.Tensor, v: Optional[torch.Tensor], lens, pos, next_pos, layered: bool) -> Tuple[bytes, tuple]:
    """The packed mrtdf_cache of a (layers, batch, kv_heads, capacity, head_dim)
    cache, or of one layer's four dimensions."""
    shape, st = k.shape, k.stride()
    if len(shape) == 4:
        dims, strides = (1, *shape), (0, *st)
    elif len(shape) == 5 and layered:
        dims, strides = tuple(shape), st
    else:
        _invalid("the cache must be (batch, kv_heads, capacity, head_dim)" +
                 (", with the layers in front where there are several" if layered else ""))
    if not k.is_cuda:
        _invalid("the cache must be on a CUDA device")
    code = _DTYPES.get(k.dtype)
    if code is None:
        _invalid(f"the cache must be float32 or bfloat16, is {k.dtype}")
    if strides[4] != 1:
        _invalid("the cache: elements of a row must lie next to each other")
    vp = 0
    if v is not None:
        if v.shape != shape or v.dtype != k.dtype or v.device != k.device:
            _invalid("k_cache and v_cache must have the same shape, dtype and device")
        if v.stride() != st:
            _invalid("k_cache and v_cache must have the same strides")
        vp = v.data_ptr()
    if k.requires_grad and torch.is_grad_enabled():
        _invalid("the cache requires a gradient, which the operators do not give")
    dev = k.device
    batch = dims[1]
    packed = _CACHE.pack(_CACHE.size, k.data_ptr(), vp, *strides[:4], *dims, code, dev.index,
                         _flat(lens, (batch,), torch.int32, dev, "lens"),
                         _flat(pos, shape[:-1], torch.int32, dev, "pos"),
                         _flat(next_pos, (batch,), torch.int32, dev, "next_pos"))
    return packed, dims


def _stream(device: torch.device) -> int:
    return torch._C._cuda_getCurrentRawStream(device.index)


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
    cache, (_, batch, kv, cap, d) = _cache(k_cache, v_cache, lens, pos, next_pos, False)
    if q.dim() != 4:
        _invalid("q must be (batch, heads, nodes, head_dim)")
    _, heads, nodes, _ = q.shape
    dev = k_cache.device
    shape, new = (batch, heads, nodes, d), (batch, kv, nodes, d)
    if out is None:
        out = torch.empty(shape, dtype=q.dtype, device=dev)
    if lse is None:
        lse = torch.empty(shape[:3], dtype=torch.float32, device=dev)
    rel_len = 0
    if rel_bias is not None:
        if rel_bias.dim() != 2:
            _invalid("rel_bias must be (heads, rel_len)")
        rel_len = rel_bias.shape[1]
    body = (_TREE.size, *_rows(q, shape, k_cache, "q"), *_rows(k_new, new, k_cache, "k_new"),
            *_rows(v_new, new, k_cache, "v_new"), *_rows(out, shape, k_cache, "out"),
            _flat(lse, shape[:3], torch.float32, dev, "lse"),
            _flat(parents, (batch, nodes), torch.int32, dev, "parents"),
            _flat(rel_bias, (heads, rel_len), torch.float32, dev, "rel_bias"))
    tail = (heads, nodes, rel_len, scale)
    key = (batch, kv, cap, d, q.dtype, dev.index, heads, nodes)
    need = _workspace_bytes.get(key)
    if need is None:
        size = ctypes.c_size_t()
        _check(lib().mrtdf_tree_attention_workspace(cache, _TREE.pack(*body, 0, 0, *tail), ctypes.byref(size)))
        need = size.value
        if len(_workspace_bytes) > 4096:
            _workspace_bytes.clear()
        _workspace_bytes[key] = need
    ws = 0
    if need:
        if workspace is None:
            workspace = torch.empty(need, dtype=torch.uint8, device=dev)
        elif workspace.device != dev or not workspace.is_contiguous():
            _invalid("workspace must be contiguous and on the cache's device")
        ws, need = workspace.data_ptr(), workspace.numel() * workspace.element_size()
    _check(lib().mrtdf_tree_attention(cache, _TREE.pack(*body, ws, need, *tail), _stream(dev)))
    return out, lse


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
    cache, (layers, batch, kv, cap, d) = _cache(k_cache, None, lens, pos, next_pos, True)
    if q.dim() != k_cache.dim():
        _invalid("q must have the cache's number of dimensions")
    heads, nodes = q.shape[-3], q.shape[-2]
    lead, dev = tuple(k_cache.shape[:-3]), k_cache.device
    if mass_out is None:
        mass_out = mass
    if path.dim() != 2:
        _invalid("path must be (batch, path_len)")
    rel_len = 0
    if rel_bias is not None:
        if rel_bias.dim() != 2:
            _invalid("rel_bias must be (heads, rel_len)")
        rel_len = rel_bias.shape[1]
    f32, i32 = torch.float32, torch.int32
    _check(lib().mrtdf_cache_mass(cache, _MASS.pack(
        _MASS.size, *_rows(q, (*lead, heads, nodes, d), k_cache, "q"), *_rows(k_new, (*lead, kv, nodes, d), k_cache, "k_new"),
        _flat(lse, (*lead, heads, nodes), f32, dev, "lse"), _flat(path, (batch, path.shape[1]), i32, dev, "path"),
        _flat(rel_bias, (heads, rel_len), f32, dev, "rel_bias"), _flat(mass, (*lead, kv, cap), f32, dev, "mass"),
        _flat(mass_out, (*lead, kv, cap), f32, dev, "mass_out"), heads, nodes, path.shape[1], rel_len, scale, decay),
        _stream(dev)))
    return mass_out


def cache_commit(k_new: torch.Tensor, v_new: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                 lens: torch.Tensor, path: torch.Tensor, *, pos: Optional[torch.Tensor] = None,
                 next_pos: Optional[torch.Tensor] = None, lens_out: Optional[torch.Tensor] = None,
                 next_pos_out: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """Appends the accepted path's rows to the cache of every layer, in place
    (mrtdf_cache_commit); pos, where given, gets the rows' positions. Returns
    (lens_out, next_pos_out), new tensors unless given (next_pos_out is None
    without next_pos)."""
    cache, (layers, batch, kv, cap, d) = _cache(k_cache, v_cache, lens, pos, next_pos, True)
    if k_new.dim() != k_cache.dim():
        _invalid("k_new must have the cache's number of dimensions")
    if path.dim() != 2:
        _invalid("path must be (batch, path_len)")
    lead, dev, nodes = tuple(k_cache.shape[:-3]), k_cache.device, k_new.shape[-2]
    if lens_out is None:
        lens_out = torch.empty_like(lens)
    if next_pos_out is None and next_pos is not None:
        next_pos_out = torch.empty_like(next_pos)
    new, i32 = (*lead, kv, nodes, d), torch.int32
    _check(lib().mrtdf_cache_commit(cache, _COMMIT.pack(
        _COMMIT.size, *_rows(k_new, new, k_cache, "k_new"), *_rows(v_new, new, k_cache, "v_new"),
        _flat(path, (batch, path.shape[1]), i32, dev, "path"), _flat(lens_out, (batch,), i32, dev, "lens_out"),
        _flat(next_pos_out, (batch,), i32, dev, "next_pos_out"), nodes, path.shape[1]), _stream(dev)))
    return lens_out, next_pos_out


def cache_evict(k_cache: torch.Tensor, v_cache: torch.Tensor, lens: torch.Tensor, mass: torch.Tensor,
                pos: torch.Tensor, next_pos: torch.Tensor, *, budget: int, recent: int = 0, sinks: int = 0,
                mass_out: Optional[torch.Tensor] = None, pos_out: Optional[torch.Tensor] = None,
                lens_out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Drops all but ``budget`` rows of every longer sequence, per layer and kv
    head (mrtdf_cache_evict): positions of the last ``recent`` tokens and the
    first ``sinks`` stay, then the rows with the largest mass. Moves K, V, mass
    and pos in place (mass and pos to mass_out and pos_out where given); returns
    lens_out, a new tensor unless given."""
    cache, (layers, batch, kv, cap, d) = _cache(k_cache, v_cache, lens, pos, next_pos, True)
    dev, shape = k_cache.device, k_cache.shape[:-1]
    if lens_out is None:
        lens_out = torch.empty_like(lens)
    _check(lib().mrtdf_cache_evict(cache, _EVICT.pack(
        _EVICT.size, _flat(mass, shape, torch.float32, dev, "mass"),
        _flat(mass if mass_out is None else mass_out, shape, torch.float32, dev, "mass_out"),
        _flat(pos if pos_out is None else pos_out, shape, torch.int32, dev, "pos_out"),
        _flat(lens_out, (batch,), torch.int32, dev, "lens_out"), budget, recent, sinks), _stream(dev)))
    return lens_out


def q4_linear(x: torch.Tensor, packed: torch.Tensor, scales: torch.Tensor, biases: torch.Tensor, *,
              out: Optional[torch.Tensor] = None, out_dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """x (m, k) times 4-bit weights (n, k) (mrtdf_q4_linear): packed (n, k / 2)
    uint8, scales and biases (n, k / group) of x's dtype. out (m, n) of
    out_dtype (x's, or float32)."""
    if x.dim() != 2 or packed.dim() != 2 or scales.dim() != 2:
        _invalid("x, packed, scales and biases must have two dimensions")
    m, k = x.shape
    n, groups = scales.shape
    dev = x.device
    code = _DTYPES.get(x.dtype)
    if code is None or not x.is_cuda:
        _invalid(f"x must be float32 or bfloat16 on a CUDA device, is {x.dtype} on {dev}")
    if x.requires_grad and torch.is_grad_enabled():
        _invalid("x requires a gradient, which the operators do not give")
    if m < 1 or k < 1 or groups < 1 or k % groups:
        _invalid("k must be a multiple of the number of groups")
    xs = x.stride()
    if xs[1] != 1:
        _invalid("x: elements of a row must lie next to each other")
    if out is None:
        out = torch.empty((m, n), dtype=out_dtype or x.dtype, device=dev)
    elif out_dtype is not None and out.dtype != out_dtype:
        _invalid("out and out_dtype do not agree")
    if out.shape != (m, n) or out.device != dev or out.dtype not in _DTYPES or (n > 1 and out.stride(1) != 1):
        _invalid(f"out must be float32 or bfloat16 {(m, n)} on {dev} with contiguous rows")
    _check(lib().mrtdf_q4_linear(_Q4.pack(
        _Q4.size, x.data_ptr(), _flat(packed, (n, k // 2), torch.uint8, dev, "packed"),
        _flat(scales, (n, groups), x.dtype, dev, "scales"), _flat(biases, (n, groups), x.dtype, dev, "biases"),
        out.data_ptr(), xs[0], out.stride(0), m, n, k, k // groups, code, _DTYPES[out.dtype], dev.index), _stream(dev)))
    return out


def q4_quantize(w: torch.Tensor, group: int = 64) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """(packed, scales, biases) of float32 or bfloat16 weights (n, k), as
    q4_linear takes them (mrtdf_q4_quantize)."""
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
                                              biases.data_ptr(), w.stride(0), n, k, group, code, dev.index), _stream(dev)))
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
