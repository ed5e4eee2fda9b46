"""What the operators on device buffers (mrtops.py) owe to torch's autograd: they
have no gradients, so they refuse tensors that want one."""
from __future__ import annotations

import pytest

torch = pytest.importorskip("torch")

from test_ops_gpu import F32, ints, q4_case, tree_inputs  # noqa: E402


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
