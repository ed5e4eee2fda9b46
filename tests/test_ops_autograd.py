"""What the operators on device buffers (mrtops.py) owe to torch's autograd: they
have no gradients, so they refuse tensors that want one."""
from __future__ import annotations

import pytest

torch = pytest.importorskip("torch")


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
