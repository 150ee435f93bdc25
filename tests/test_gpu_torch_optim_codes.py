"""The 8-bit states on the device: every scale and every code is that of the quotients
in 64 bits, the largest value over the format's and a value over its block's scale.
Means of no memory (both decay rates zero) are the gradients and their squares
themselves, which fp32 gradients reach to within 2^-23 of where a draw begins to
round them up; a factor held in fp32 moves codes there."""

import numpy as np
import pytest
import torch

from mojogp_amd import optim
from oracle import optim as oo

pytestmark = pytest.mark.gpu

SEED = (1 << 63) + 9


def _check(opt, m, v, step):
    word = oo.words(SEED, step, len(m))
    for x, draw, signed, codes, scales in ((m, word & 0xFFFF, True, opt.exp_avg, opt.exp_avg_scale),
                                           (v, word >> 16, False, opt.exp_avg_sq,
                                            opt.exp_avg_sq_scale)):
        code, scale = oo.encode(x, draw, signed)
        got = codes.cpu().numpy().astype(np.int64)
        if signed:  # a rounded-off negative value keeps its sign
            code, got = (np.where(c == 128, 0, c) for c in (code, got))
        assert np.array_equal(scales.cpu().numpy(), scale)
        assert np.array_equal(got, code)


@pytest.mark.parametrize("squares", [False, True])
def test_values_next_to_their_borders(squares):
    rng = np.random.default_rng(21)
    blocks, step = 64, 7
    table, top = (oo.TABLE_V, oo.TOP_V) if squares else (oo.TABLE_M, oo.TOP_M)
    word = oo.words(SEED, step, blocks * 256).reshape(blocks, 256)
    draw = word >> 16 if squares else word & 0xFFFF
    most = (rng.uniform(1, 2, blocks) * 2.0 ** rng.integers(-30, 15, blocks)).astype(np.float32)
    size = most.astype(np.float64) ** 2 if squares else most.astype(np.float64)
    scale = (size / top).astype(np.float32).astype(np.float64)[:, None]
    code = rng.integers(len(table) // 2, len(table) - 2, draw.shape)
    at = scale * (table[code] + (table[code + 1] - table[code]) * (1 - (draw + 0.5) / 65536))
    g = (np.sqrt(at) if squares else at).astype(np.float32)
    g = np.where(rng.random(g.shape) < 0.5, np.nextafter(g, np.float32(0)), g)
    g = np.minimum(g, np.nextafter(most, np.float32(0))[:, None])  # the largest stays what it is
    g[:, 100] = most
    g *= rng.choice([-1, 1], g.shape).astype(np.float32)
    p = torch.zeros(g.size, device="cuda")
    opt = optim.AdamW([p], bits=8, betas=(0.0, 0.0), seed=SEED)
    opt.step([torch.from_numpy(g.ravel()).cuda()], 0.0, step)
    m = g.ravel().astype(np.float64)
    _check(opt, m, m * m, step)


def test_millions_of_values():
    """Sixteen million of them, from states of steps before and clipped gradients."""
    rng = np.random.default_rng(22)
    n, betas = 1 << 22, (0.9, 0.999)
    size = np.exp(rng.normal(size=(n // 256, 1))) * np.exp(0.7 * rng.normal(size=(n // 256, 256)))
    p = torch.zeros(n, device="cuda")
    opt = optim.AdamW([p], bits=8, betas=betas, seed=SEED)
    for step in range(1, 5):
        g = (1e-3 * size * rng.normal(size=size.shape)).astype(np.float32).ravel()
        m = oo.decode(opt.exp_avg.cpu().numpy(), opt.exp_avg_scale.cpu().numpy(), True)
        v = oo.decode(opt.exp_avg_sq.cpu().numpy(), opt.exp_avg_sq_scale.cpu().numpy(), False)
        opt.step([torch.from_numpy(g).cuda()], 1e-3, step, grad_scale=0.7)
        _check(opt, *oo.moments(m, v, 0.7 * g.astype(np.float64), betas), step)


@pytest.mark.parametrize("largest", [2.0 ** -120, 1.5 * 2.0 ** -120, 2.0 ** -119, 2.0 ** -117])
def test_the_smallest_blocks(largest):
    """Zeros stay zeros in blocks whose scale is below fp32's normal range."""
    g = np.zeros(512, np.float32)
    g[:4] = largest, -largest, largest / 2, -largest / 3
    g[256:260] = np.float32(0.99) * g[:4]
    p = torch.zeros(512, device="cuda")
    opt = optim.AdamW([p], bits=8, betas=(0.0, 0.0), eps=1e-30, seed=SEED)
    opt.step([torch.from_numpy(g).cuda()], 0.0, 3)
    m = g.astype(np.float64)
    _check(opt, m, m * m, 3)
    got = opt.values()["exp_avg"]
    assert not got[4:256].any() and not got[260:].any()
    assert float(opt.exp_avg_scale[0]) > 0


@pytest.mark.parametrize("bad", [float("inf"), -float("inf"), float("nan"), -float("nan"), 1e30])
def test_blocks_that_are_not_in_float32(bad):
    """Every value of the block is NaN, of no other; of a finite gradient whose square
    passes float32, the squares alone."""
    p = torch.zeros(768, device="cuda")
    g = torch.linspace(-1.0, 1.0, 768, device="cuda")
    g[300] = bad
    opt = optim.AdamW([p], bits=8, seed=SEED)
    opt.step([g], 0.0, 1)
    spoilt = torch.zeros(768, dtype=torch.bool, device="cuda")
    spoilt[256:512] = True
    got = opt.values()
    assert torch.equal(torch.isnan(got["exp_avg_sq"]), spoilt)
    assert torch.equal(torch.isnan(got["exp_avg"]), spoilt & (not np.isfinite(bad)))
    assert torch.isfinite(got["exp_avg"][~spoilt]).all()
