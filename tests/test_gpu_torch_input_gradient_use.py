"""How calls of the input gradient share a handle: graphs, threads, errors."""

import threading

import numpy as np
import pytest
import torch

from mojogp_amd import _lib
from mojogp_amd._provider import NativeProvider
from test_zz_no_alloc import _hip

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


def test_threads_of_one_handle():
    """Calls from several threads, each on a stream of its own and of another size,
    share the work buffers one after another."""
    X, params, L, R = _inputs(6000, 4, 20)
    p = NativeProvider("matern52", True, X, params, 0.1)
    l, r = torch.from_numpy(L).cuda(), torch.from_numpy(R).cuda()
    columns = (1, 5, 16, 20)
    want = [p.input_gradient(L[:t], R[:t]) for t in columns]
    torch.cuda.synchronize()
    got, errors = [[] for _ in columns], []
    start = threading.Barrier(len(columns))

    def work(k):
        try:
            stream = torch.cuda.Stream()
            start.wait()
            with torch.cuda.stream(stream):
                for _ in range(25):
                    got[k].append(p.input_gradient_device(l[:columns[k]], r[:columns[k]]))
            stream.synchronize()
        except Exception as e:  # noqa: BLE001 - reported below
            errors.append(e)

    threads = [threading.Thread(target=work, args=(k,)) for k in range(len(columns))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    p.close()
    assert not errors
    for k in range(len(columns)):
        assert all(np.array_equal(g.cpu().numpy(), want[k]) for g in got[k])


def test_a_call_that_fails_after_its_launches_is_waited_for():
    """An error that the runtime still held from elsewhere ends the call once its
    kernels run: a change of the parameters waits for them all the same, and the
    next calls are right."""
    X, params, L, R = _inputs(20000, 8, 16)
    p = NativeProvider("matern52", True, X, params, 0.1)
    l, r = torch.from_numpy(L).cuda(), torch.from_numpy(R).cuda()
    out = torch.zeros(20000, 8, device="cuda")
    try:
        want = p.input_gradient(L, R)
        torch.cuda.synchronize()
        assert _hip().hipSetDevice(10 ** 6) != 0  # no such device
        with pytest.raises(_lib.NativeCallError):
            p.input_gradient_device(l, r, out=out)
        p.update_params(params * np.float32(2.0))
        torch.cuda.synchronize()
        assert np.array_equal(out.cpu().numpy(), want)
        assert np.array_equal(p.input_gradient_device(l, r).cpu().numpy(), p.input_gradient(L, R))
    finally:
        p.close()
