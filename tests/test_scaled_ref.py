"""The 64-bit forms of the block-scaled operators against torch's 8-bit
floats, and the refusals of the C entry points that need no GPU."""
import numpy as np
import pytest
import torch

import scaled_ref as ref

TORCH = {ref.E4M3: torch.float8_e4m3fn, ref.E5M2: torch.float8_e5m2}


@pytest.mark.parametrize("code", [ref.E4M3, ref.E5M2])
def test_code_values(code):
    want = torch.arange(256, dtype=torch.int16).to(torch.uint8).view(TORCH[code]).double().numpy()
    np.testing.assert_array_equal(ref.code_values(code), want)


@pytest.mark.parametrize("code", [ref.E4M3, ref.E5M2])
def test_rounding(code):
    v = ref.code_values(code)
    v = np.unique(v[np.isfinite(v)])
    ties = (v[1:] + v[:-1]) / 2
    x = np.concatenate([v, ties, np.nextafter(ties.astype(np.float32), np.float32(np.inf)),
                        np.random.default_rng(3).standard_normal(4096) * 20])
    x = x.astype(np.float32)
    want = torch.from_numpy(x).clamp(-ref.LARGEST[code], ref.LARGEST[code]).to(TORCH[code])
    np.testing.assert_array_equal(ref.round_to_code(x, code), want.double().numpy())


def test_scale_layout():
    x = np.ones((130, 300), np.float32)
    x[129, 299] = 448 * 4
    s = ref.scales_of(x, ref.E4M3, 128)
    assert s.shape == (3, 2) and s[2, 1] == 4 and s[2, 0] == np.float32(1) / np.float32(448)
    assert ref.spread(s, 130, 300, 128)[129, 299] == 4


def test_entry_points_refuse_a_missing_workspace(autlib):
    from accessor_universal_test_b200 import _lib
    bad = _lib.AUT_ERR_INVALID_ARGUMENT
    assert autlib.aut_encode_scaled(None, 0, 0, 1, None, 0, 0, 0, None, 0, None, 0, None) == bad
    assert autlib.aut_rms_norm_scaled(None, 0, 0, None, 0, None, None, 0, None, 0.0, 0, 0, None,
                                      0, None, 0, None) == bad
    assert autlib.aut_gemm_scaled(None, 0, 0, 0, None, 0, None, 0, None, 0, None, 0, 0, 0, 0,
                                  None, 0, None) == bad
    assert b"workspace" in autlib.aut_last_error()


def test_tensor_calls_refuse_what_does_not_fit():
    """scaled.* check their tensors before anything is launched."""
    from accessor_universal_test_b200 import scaled

    class Handle:  # a workspace's device is all the checks look at
        device = 0

    ws = Handle()
    x = torch.zeros(4, 256)
    with pytest.raises(ValueError, match="workspace on cuda:0"):
        scaled.encode(ws, x)
    with pytest.raises(ValueError, match="two dimensions"):
        scaled.encode(ws, x[0])
    with pytest.raises(ValueError, match="two dimensions"):
        scaled.rms_norm(ws, x[0])
    with pytest.raises(ValueError, match="block_rows"):
        scaled.Scaled(4, 256, block_rows=2)
    with pytest.raises(ValueError, match="code"):
        scaled.Scaled(4, 256, code=7)
    a, b = scaled.Scaled(4, 256), scaled.Scaled(300, 256, block_rows=128)
    assert a.scales.shape == (2, 4) and b.scales.shape == (2, 3)
    assert scaled.Scaled(3, 100).storage.shape == (3, 112)
    with pytest.raises(ValueError, match="scales by rows"):
        scaled.matmul(ws, b, b)
    with pytest.raises(ValueError, match="columns"):
        scaled.matmul(ws, a, scaled.Scaled(300, 128, block_rows=128))
    with pytest.raises(ValueError, match="workspace on cuda:0"):
        scaled.matmul(ws, a, b)


def test_tensor_calls_refuse_to_drop_a_gradient():
    """Refused before anything else where gradients are recorded, and only there."""
    from accessor_universal_test_b200 import scaled

    class Handle:
        device = 0

    ws = Handle()
    grad = torch.zeros(4, 256, requires_grad=True)
    for call in (lambda: scaled.encode(ws, grad), lambda: scaled.rms_norm(ws, grad),
                 lambda: scaled.encode(ws, grad * 2)):
        with pytest.raises(ValueError, match="requires a gradient"):
            call()
    with torch.no_grad(), pytest.raises(ValueError, match="workspace on cuda:0"):
        scaled.encode(ws, grad)
    with pytest.raises(ValueError, match="workspace on cuda:0"):
        scaled.encode(ws, grad.detach())
