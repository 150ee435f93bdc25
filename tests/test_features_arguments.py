"""How the layers' Python entries read their arrays, on the host: stand-ins with a
tensor's shape, strides and type."""

import pytest
import torch

from mojogp_amd import features


def _rows(t):
    class Device:  # the tensor, but for its device
        dtype, shape, requires_grad = t.dtype, t.shape, t.requires_grad

        def stride(self):
            return t.stride()

        def get_device(self):
            return 0

        def data_ptr(self):
            return t.data_ptr()

    return features._rows(Device(), "x", t.dtype, 0)[1:]


@pytest.mark.parametrize("shape", [(2, 0, 24), (0, 3, 24), (2, 3, 0, 5, 24), (0, 0, 24), (2, 3, 0, 24)])
def test_empty_arrays_have_no_rows(shape):
    t = torch.empty(shape)
    assert _rows(t) == (0, 24, 24)
    if len(shape) == 3:
        assert _rows(t.transpose(0, 1)) == (0, 24, 24)


def test_rows_of_more_dimensions():
    t = torch.empty(2, 3, 5, 40)
    assert _rows(t) == (30, 40, 40)
    assert _rows(t[..., :24]) == (30, 24, 40)
    assert _rows(t[:, :1, :, :24][:1]) == (5, 24, 40)
    with pytest.raises(ValueError, match="collapse"):
        _rows(t[:, :, :4])


def test_arrays_that_require_a_gradient_are_refused():
    """No graph is recorded through these calls, so none may end in them unnoticed."""
    x, w = torch.zeros(4, 8), torch.zeros(8, requires_grad=True)
    with pytest.raises(ValueError, match="x requires a gradient"):
        features.layer_norm(x.clone().requires_grad_())
    with pytest.raises(ValueError, match="weight requires a gradient"):
        features._vector(w, "weight", 8, torch.float32, -1)
    with torch.no_grad():
        assert features._vector(w, "weight", 8, torch.float32, -1) == w.data_ptr()
        with pytest.raises(ValueError, match="device tensor"):  # the next check
            features.layer_norm(x.clone().requires_grad_())
    assert features._vector(w.detach(), "weight", 8, torch.float32, -1) == w.data_ptr()
