"""Results beside and in place of what the layers read: columns of one table, and
the in-place forms."""

import numpy as np
import pytest
import torch

from mojogp_amd import _lib, features

pytestmark = pytest.mark.gpu

TYPES = (torch.float32, torch.bfloat16, torch.float16)


def _table(rows, width, kind):
    rng = np.random.default_rng(rows + width)
    return torch.from_numpy(rng.normal(size=(rows, width))).to("cuda", kind)


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("rows, width", [(5, 3), (40, 33), (300, 256), (1500, 771), (9, 1030),
                                         (700, 4099), (3, 9001)])
def test_layer_norm_in_place(kind, rows, width):
    """Narrow, ragged and wide rows, also as columns of a wider table."""
    x = _table(rows, width, kind)
    want = features.layer_norm(x)
    wide = torch.zeros(rows, width + 11, device="cuda", dtype=kind)
    view = wide[:, 3:3 + width]
    view.copy_(x)
    assert features.layer_norm(view, out=view) is view
    assert torch.equal(view, want) and not wide[:, :3].any() and not wide[:, 3 + width:].any()
    assert torch.equal(features.layer_norm(x, out=x), want)


@pytest.mark.parametrize("kind", TYPES)
def test_columns_of_one_table(kind):
    """Inputs and results side by side share no memory and are served."""
    t = _table(70, 96, kind)
    x, w = t[:, :24].clone(), _table(24, 24, kind)
    want = (features.layer_norm(x), features.gated_layer(x, w, w), features.dropout(x, 0.3, 5))
    features.layer_norm(t[:, :24], out=t[:, 24:48])
    features.gated_layer(t[:, :24], w, w, out=t[:, 48:72])
    features.dropout(t[:, :24], 0.3, 5, out=t[:, 72:])
    assert torch.equal(t[:, :24], x)
    for k, a in enumerate(want):
        assert torch.equal(t[:, 24 * (k + 1):24 * (k + 2)], a)
    rows = _table(40, 24, kind)
    even = rows[::2].clone()
    features.layer_norm(rows[::2], out=rows[1::2])
    assert torch.equal(rows[::2], even) and torch.equal(rows[1::2], features.layer_norm(even))


def test_shared_memory_is_refused():
    t, w = _table(50, 40, torch.float32), _table(24, 24, torch.float32)
    for out in (t[:, 1:25], t[:, :24]):
        with pytest.raises(_lib.NativeCallError, match="shares memory"):
            features.gated_layer(t[:, :24], w, w, out=out)
    for call in (features.layer_norm, lambda x, out: features.dropout(x, 0.2, 1, out=out)):
        with pytest.raises(_lib.NativeCallError, match="shares memory"):
            call(t[:, :24], out=t[:, 1:25])
        with pytest.raises(_lib.NativeCallError, match="shares memory"):
            call(t[:-1, :24], out=t[1:, :24])
