"""How calls of the input gradient share a handle: graphs, threads, errors."""

import numpy as np
import pytest
import torch

from mojogp_amd import _lib
from mojogp_amd._provider import NativeProvider

pytestmark = pytest.mark.gpu


def _inputs(n, d, t, seed=0):
    rng = np.random.default_rng([n, d, t, seed])
    X = rng.normal(size=(n, d)).astype(np.float32)
    params = np.append(np.sqrt(d) * rng.uniform(0.6, 1.2, size=d), 1.3).astype(np.float32)
    return X, params, *(rng.normal(size=(t, n)).astype(np.float32) for _ in range(2))


def test_a_stream_in_capture_is_refused():
    """The handle's buffers and events have no place in a graph; the refusal comes
    before either is touched, so that the handle works on."""
    X, params, L, R = _inputs(500, 3, 4)
    p = NativeProvider("rbf", True, X, params, 0.1)
    l, r = torch.from_numpy(L).cuda(), torch.from_numpy(R).cuda()
    out = torch.empty(500, 3, device="cuda")
    try:
        for used in (False, True):  # before the first call, and after one
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                l2 = l * 2.0
                with pytest.raises(_lib.NativeCallError, match="recorded into a graph"):
                    p.input_gradient_device(l, r, out=out)
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(l2, l * 2.0)
            want = p.input_gradient(L, R)
            got = p.input_gradient_device(l, r, out=out)
            assert np.array_equal(got.cpu().numpy(), want)
        p.update_params(params * np.float32(1.5))
        assert np.array_equal(p.input_gradient_device(l, r).cpu().numpy(), p.input_gradient(L, R))
    finally:
        p.close()
