"""Operators whose device waits run out: the call ends, its context stays usable.
The waits look once and give up (mrtdf_check_*_wait), no copy is left out and
nothing is broken: most of what they wait for is still on its way then."""
from __future__ import annotations

import ctypes
import time

import pytest

torch = pytest.importorskip("torch")

from test_ops_gpu import BF, DEV, F32, check_q4, check_tree, ints, normal, ops, q4_case, tree_inputs  # noqa: E402,F401
from test_ops_host import _CACHE, _Q4, _TREE  # noqa: E402

pytestmark = pytest.mark.gpu


def hurried_tree(ops, q, kn, vn, k, v, lens, rel_bias=None):
    """(out, lse) of mrtdf_check_tree_attention_wait on contiguous tensors."""
    L = ops.lib()
    B, H, N, D = q.shape
    KV, cap = k.shape[1], k.shape[2]
    out, lse = torch.zeros_like(q), torch.zeros(B, H, N, device=DEV)

    def rows(t):
        return t.data_ptr(), 0, *t.stride()[:3]

    cache = _CACHE.pack(_CACHE.size, k.data_ptr(), v.data_ptr(), 0, *k.stride()[:3], 1, B, KV, cap, D, 1, 0, lens.data_ptr(), 0, 0)
    bias = (rel_bias.data_ptr(), rel_bias.shape[1]) if rel_bias is not None else (0, 0)

    def args(ws, size):
        return _TREE.pack(_TREE.size, *rows(q), *rows(kn), *rows(vn), *rows(out), lse.data_ptr(), 0, bias[0], ws, size, H, N, bias[1], 0.125)

    need = ctypes.c_size_t()
    L.mrtdf_tree_attention_workspace.argtypes = [ctypes.c_char_p, ctypes.c_char_p, ctypes.POINTER(ctypes.c_size_t)]
    L.mrtdf_check_tree_attention_wait.argtypes = [ctypes.c_char_p, ctypes.c_char_p, ctypes.c_void_p]
    assert L.mrtdf_tree_attention_workspace(cache, args(0, 0), ctypes.byref(need)) == 0, L.mrtdf_last_error()
    ws = torch.zeros(max(16, need.value), dtype=torch.uint8, device=DEV)
    rc = L.mrtdf_check_tree_attention_wait(cache, args(ws.data_ptr(), need.value), torch.cuda.current_stream().cuda_stream)
    assert rc == 0, L.mrtdf_last_error()
    torch.cuda.synchronize()
    return out, lse


# Items of many CTAs and CTAs of many items, one block of rows and several.
TREES = [(1, 16, 1, 8, 6000), (64, 8, 1, 16, 700), (3, 16, 2, 40, 3000)]


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("bias", [0, 32])
@pytest.mark.parametrize("B,H,KV,N,cap", TREES)
def test_tree_ends_when_waits_run_out(ops, D, bias, B, H, KV, N, cap):
    x = tree_inputs(1, BF, B, H, KV, N, D, cap)
    lens = ints([cap - 3 * b for b in range(B)])
    kw = dict(rel_bias=normal(2, H, bias)) if bias else {}
    ops.tree_attention(*x, lens, **kw)
    torch.cuda.synchronize()
    begin = time.perf_counter()
    hurried_tree(ops, *x, lens, **kw)
    assert time.perf_counter() - begin < 0.4  # less than one wait's limit
    small = [t[:1] for t in x]
    check_tree(ops, small, lens[:1], None, scale=0.125, **kw)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("bias", [0, 32])
@pytest.mark.parametrize("B,H,KV,N,cap", TREES)
def test_tree_rows_whose_waits_ran_out_are_nan(ops, D, bias, B, H, KV, N, cap):
    """In whole items and in those that several CTAs share: a row is NaN, its lse
    too, or as without the hurry. None is zeros or a softmax over a part."""
    x = tree_inputs(1, BF, B, H, KV, N, D, cap)
    lens = ints([cap - 3 * b for b in range(B)])
    kw = dict(rel_bias=normal(2, H, bias)) if bias else {}
    want, want_lse = ops.tree_attention(*x, lens, scale=0.125, **kw)
    failed = 0
    for _ in range(3):
        out, lse = hurried_tree(ops, *x, lens, **kw)
        gone = torch.isnan(lse)
        assert torch.equal(torch.isnan(out), gone[..., None].expand_as(out))
        assert torch.equal(out[~gone], want[~gone]) and torch.equal(lse[~gone], want_lse[~gone])
        failed += int(gone.sum())
    assert failed


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("m,n,k,group", [(8, 10000, 8192, 128), (33, 20000, 4096, 32), (16, 700, 131072, 64)])
def test_q4_ends_and_shows_waits_that_ran_out(ops, dtype, m, n, k, group):
    """Row blocks that one CTA has and those that several share; more stages per CTA
    than its ring holds, so that its copies have to wait for a free place."""
    x, packed, scales, biases = q4_case(m, dtype, m, n, k, group)
    want = ops.q4_linear(x, packed, scales, biases, out_dtype=F32)
    L, need = ops.lib(), ctypes.c_size_t()
    L.mrtdf_q4_linear_workspace.argtypes = [ctypes.c_char_p, ctypes.POINTER(ctypes.c_size_t)]
    L.mrtdf_check_q4_linear_wait.argtypes = [ctypes.c_char_p, ctypes.c_void_p]
    out = torch.zeros(m, n, device=DEV)

    def args(ws, size):
        return _Q4.pack(_Q4.size, x.data_ptr(), packed.data_ptr(), scales.data_ptr(), biases.data_ptr(), out.data_ptr(), ws, size,
                        k, n, m, n, k, group, int(dtype is BF), 0, 0)

    assert L.mrtdf_q4_linear_workspace(args(0, 0), ctypes.byref(need)) == 0 and need.value
    ws = torch.zeros(need.value, dtype=torch.uint8, device=DEV)
    failed = 0
    for _ in range(3):
        torch.cuda.synchronize()
        begin = time.perf_counter()
        rc = L.mrtdf_check_q4_linear_wait(args(ws.data_ptr(), need.value), torch.cuda.current_stream().cuda_stream)
        assert rc == 0, L.mrtdf_last_error()
        torch.cuda.synchronize()
        assert time.perf_counter() - begin < 2.0
        gone = torch.isnan(out)
        assert torch.equal(out[~gone], want[~gone])
        failed += int(gone.sum())
    assert failed
    assert torch.equal(check_q4(ops, x, packed, scales, biases, out_dtype=F32), want)
