"""What the operators on device buffers (mrtops.py) owe to torch's autograd: they
have no gradients, so they refuse tensors that want one."""
from __future__ import annotations

import pytest

torch = pytest.importorskip("torch")

from test_ops_gpu import DEV, F32, ints, normal, q4_case, tree_inputs  # noqa: E402


@pytest.fixture(scope="module")
def ops(mrtdf):
    import mrtops

    return mrtops


def test_q4_quantize_refuses_weights_that_require_a_gradient(ops, mrtdf):
    w = torch.zeros(4, 64).requires_grad_()
    with pytest.raises(mrtdf.MrtdfError, match="gradient"):
        ops.q4_quantize(w)
    with torch.no_grad(), pytest.raises(mrtdf.MrtdfError, match="CUDA"):
        ops.q4_quantize(w)


@pytest.mark.gpu
def test_q4_quantize_takes_parameters_without_gradients(ops):
    w = torch.randn(4, 64, device="cuda").requires_grad_()
    with torch.no_grad():
        a = ops.q4_quantize(w)
    b = ops.q4_quantize(w.detach())
    assert all(torch.equal(x, y) for x, y in zip(a, b))


@pytest.mark.gpu
def test_forward_mode_tangents_are_refused(ops, mrtdf):
    from torch.autograd import forward_ad

    x, packed, scales, biases = q4_case(5, F32, 2, 10, 128, 64)
    q, kn, vn, k, v = tree_inputs(1, F32, 1, 1, 1, 1, 64, 8)
    with forward_ad.dual_level():
        for f in (lambda: ops.q4_linear(forward_ad.make_dual(x, torch.ones_like(x)), packed, scales, biases),
                  lambda: ops.q4_quantize(forward_ad.make_dual(x, torch.ones_like(x))),
                  lambda: ops.tree_attention(forward_ad.make_dual(q, torch.ones_like(q)), kn, vn, k, v, ints([4])),
                  lambda: ops.tree_attention(q, kn, vn, k, forward_ad.make_dual(v, torch.ones_like(v)), ints([4]))):
            with pytest.raises(mrtdf.MrtdfError, match="tangent"):
                f()
        with forward_ad._set_fwd_grad_enabled(False):
            ops.q4_linear(forward_ad.make_dual(x, torch.ones_like(x)), packed, scales, biases)


@pytest.mark.gpu
def test_a_saved_cache_does_not_change_unnoticed(ops):
    w = normal(0, 1, 2, 20, 64).requires_grad_()
    k, v, kn = normal(1, 1, 2, 20, 64), normal(2, 1, 2, 20, 64), normal(3, 1, 2, 4, 64)
    loss = (w * k).sum()
    ops.cache_commit(kn, kn, k, v, ints([3]), ints([[0, 1]]))
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()


@pytest.mark.gpu
def test_every_written_tensor_raises_its_version(ops):
    def rises(f, *written):
        before = [t._version for t in written]
        f()
        assert all(t._version > b for t, b in zip(written, before))

    q, kn, vn, k, v = tree_inputs(1, F32, 1, 2, 1, 3, 64, 2000)
    out, lse, ws = torch.empty_like(q), torch.empty(1, 2, 3, device=DEV), torch.empty(1 << 24, dtype=torch.uint8, device=DEV)
    lens, path = ints([9]), ints([[0, 1]])
    rises(lambda: ops.tree_attention(q, kn, vn, k, v, lens, out=out, lse=lse, workspace=ws), out, lse, ws)
    mass, mass_out = torch.ones(1, 1, 2000, device=DEV), torch.zeros(1, 1, 2000, device=DEV)
    pos, pos_out = (torch.zeros(1, 1, 2000, dtype=torch.int32, device=DEV) for _ in range(2))
    lens_out, next_out = ints([0]), ints([0])
    rises(lambda: ops.cache_mass(q, lse, kn, k, lens, path, mass), mass)
    rises(lambda: ops.cache_mass(q, lse, kn, k, lens, path, mass, mass_out=mass_out), mass_out)
    rises(lambda: ops.cache_commit(kn, vn, k, v, lens, path, pos=pos, next_pos=lens, lens_out=lens_out, next_pos_out=next_out),
          k, v, pos, lens_out, next_out)
    rises(lambda: ops.cache_evict(k, v, lens, mass, pos, lens, budget=4, mass_out=mass_out, pos_out=pos_out, lens_out=lens_out),
          k, v, mass_out, pos_out, lens_out)
    rises(lambda: ops.cache_evict(k, v, lens, mass, pos, lens, budget=4), k, v, mass, pos)
    x, packed, scales, biases = q4_case(5, F32, 2, 10, 128, 64)
    y = torch.empty(2, 10, device=DEV)
    rises(lambda: ops.q4_linear(x, packed, scales, biases, out=y), y)


@pytest.mark.gpu
def test_tensors_of_inference_mode_are_taken(ops):
    """They have no version."""
    with torch.inference_mode():
        q, kn, vn, k, v = (t.clone() for t in tree_inputs(1, F32, 1, 2, 1, 3, 64, 20))
        out, _ = ops.tree_attention(q, kn, vn, k, v, ints([9]))
        ops.cache_commit(kn, vn, k, v, ints([9]), ints([[0, 1]]))
    assert out.is_inference() and k.is_inference() and torch.equal(k[:, :, 9:11], kn[:, :, :2])
    ops.cache_commit(kn, vn, k, v, ints([11]), ints([[0, 1]]))
    assert torch.equal(k[:, :, 11:13], kn[:, :, :2])
