"""The float64 AdamW and its 8-bit format, pinned on their own."""

import numpy as np
import pytest
import torch

from oracle import optim as oo


def test_means_are_an_ocp_format():
    codes = torch.arange(127, dtype=torch.uint8)
    assert np.array_equal(codes.view(torch.float8_e4m3fn).double().numpy(), oo.TABLE_M)
    assert oo.TABLE_M[-1] == oo.TOP_M and oo.TABLE_V[-1] == oo.TOP_V
    assert oo.TABLE_V[1] == 2.0 ** -33 and (np.diff(oo.TABLE_V) > 0).all()


@pytest.mark.parametrize("signed", [True, False])
def test_encoding_keeps_the_formats_values_and_the_mean(signed, rng):
    values = oo.TABLE_M if signed else oo.TABLE_V
    x = np.zeros(256)
    x[:len(values)] = values
    for draw in (0, 65535):  # what the format has is not moved
        code, scale = oo.encode(x, np.full(256, draw), signed)
        assert scale[0] == 1.0 and np.array_equal(oo.decode(code, scale, signed), x)
    a = rng.uniform(0, 1, 256) ** 4
    a[0] = 1.0
    draws = (np.arange(4096)[:, None] * 16 + 8).repeat(256, axis=1)  # every probability
    mean = np.mean([oo.decode(*oo.encode(a, d, signed), signed) for d in draws], axis=0)
    gap = np.gradient(values).max() / values[-1]
    # evenly spread draws reach every share to 1 / 4096 of a step
    assert np.abs(mean - a).max() <= gap / 4096 + 1e-7


def test_step_is_torch_s(rng):
    """Ten steps of torch.optim.AdamW in float64."""
    p = rng.normal(size=50)
    t = torch.from_numpy(p.copy()).requires_grad_()
    opt = torch.optim.AdamW([t], lr=3e-3, betas=(0.8, 0.95), eps=1e-6, weight_decay=0.1)
    m = v = np.zeros(50)
    for step in range(1, 11):
        g = rng.normal(size=50)
        t.grad = torch.from_numpy(g)
        opt.step()
        m, v = oo.moments(m, v, g, (0.8, 0.95))
        p = oo.update(p, m, v, 3e-3, step, (0.8, 0.95), 1e-6, 0.1)
        assert np.allclose(p, t.detach().numpy(), rtol=1e-12, atol=1e-14)
