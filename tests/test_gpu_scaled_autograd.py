"""The tensor calls of the block-scaled operators beside torch's record of gradients."""
import pytest
import torch

from accessor_universal_test_b200 import scaled

pytestmark = pytest.mark.gpu


def tensors():
    g = torch.Generator(device="cuda").manual_seed(3)
    return [torch.randn(s, generator=g, device="cuda") for s in ((6, 256), (6, 256), (256,))]


@pytest.mark.parametrize("which", range(3))
def test_a_tensor_that_requires_a_gradient_is_refused(ws, which):
    args = tensors()
    before = args[1].clone()
    args[which].requires_grad_()
    x, residual, gain = args
    with pytest.raises(ValueError, match="requires a gradient"):
        scaled.rms_norm(ws, x, gain, residual=residual)
    assert torch.equal(residual, before)
    with torch.no_grad():
        a, _ = scaled.rms_norm(ws, x, gain, residual=residual)
    assert torch.isfinite(a.scales).all() and not a.scales.requires_grad
    if which == 0:
        with pytest.raises(ValueError, match="requires a gradient"):
            scaled.encode(ws, x)


def test_a_result_that_requires_a_gradient_is_refused(ws):
    x, _, _ = tensors()
    a, b = scaled.encode(ws, x), scaled.encode(ws, x, block_rows=128)
    out = torch.zeros(6, 6, device="cuda", requires_grad=True)
    with pytest.raises(ValueError, match="requires a gradient"):
        scaled.matmul(ws, a, b, out=out)
    with torch.no_grad():
        scaled.matmul(ws, a, b, out=out)
    assert (out != 0).any()


def test_what_is_written_in_place_counts_as_changed(ws):
    """A backward pass that saved the old residual, or result, does not go on with
    the new one."""
    x, residual, gain = tensors()
    factor = torch.ones(256, device="cuda", requires_grad=True)
    saved = (residual * factor).sum()
    scaled.rms_norm(ws, x, gain, residual=residual)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        saved.backward()
    a, b = scaled.encode(ws, x), scaled.encode(ws, x, block_rows=128)
    out = scaled.matmul(ws, a, b, dtype=torch.float32)
    saved = (out * torch.ones(6, device="cuda", requires_grad=True)).sum()
    scaled.matmul(ws, a, b, out=out)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        saved.backward()
    versions = a.storage._version, a.scales._version
    scaled.encode(ws, x, out=a)
    assert a.storage._version > versions[0] and a.scales._version > versions[1]


def test_calls_in_inference_mode(ws):
    with torch.inference_mode():
        x, residual, gain = tensors()
        a, stream = scaled.rms_norm(ws, x, gain, residual=residual)
        b = scaled.encode(ws, x, block_rows=128)
        out = scaled.matmul(ws, a, b, dtype=torch.float32)
        torch.testing.assert_close(out, a.decoded() @ b.decoded().t(), rtol=1e-4, atol=1e-3)
    again = scaled.matmul(ws, a, b, out=out)
    assert again is out
