"""Contexts over torch's streams while torch captures them.  Run as a program (tests/test_gpu_scoring_edges.py does): torch has to be
loaded before the library, so that both use one HIP runtime."""
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

import numpy as np  # noqa: E402

from snekmer_amd import _hip, apply, engine  # noqa: E402


def raises(kind, says, call):
    try:
        call()
    except kind as e:
        assert says in str(e), e
        return
    raise AssertionError(f"{says}: nothing was raised")


def a_graph_that_outlives_its_context():
    """Forward and backward captured by torch; the context goes, another takes over what it held; replays give NaN for wrong labels and
    report nothing to the other context, and what they compute is what eager calls give."""
    s = torch.cuda.Stream()
    own = _hip.Context(0, stream=s.cuda_stream)
    n, a = 40, 300
    with torch.cuda.stream(s):
        g = torch.Generator(device="cuda")
        g.manual_seed(2)
        scores = torch.randn(n, a, generator=g, device="cuda")
        labels = torch.randint(0, a, (n,), generator=g, device="cuda", dtype=torch.int32)
        d_logp = torch.randn(n, generator=g, device="cuda")
        logp, entropy = torch.empty(n, device="cuda"), torch.empty(n, device="cuda")
        stats, grad = torch.empty(n, 2, device="cuda"), torch.empty(n, a, device="cuda")
        out = apply.LogProbabilities(logp=logp, entropy=entropy, stats=stats)

        def step(ctx):
            apply.log_probabilities(ctx, scores, labels, out=out)
            apply.log_probabilities_backward(ctx, scores, labels, out, d_logp=d_logp, out=grad)

        step(own)
        s.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            step(own)
        own.sync()
        own.close()
        other = _hip.Context(0, stream=s.cuda_stream)
        for wrong in (a, -7, a + 1, 5):
            labels[3] = wrong
            logp.zero_()
            grad.zero_()
            graph.replay()
            other.sync()
            replayed = [logp.clone(), grad.clone()]
            bad = wrong != 5
            assert bool(torch.isnan(logp[3])) == bad and bool(torch.isnan(grad[3]).all()) == bad
            assert bool(torch.isfinite(logp[4:]).all()) and bool(torch.isfinite(grad[:3]).all())
            step(other)
            if bad:
                raises(_hip.HipError, "label outside", other.sync)  # (an eager call still says so)
            for x, y in zip(replayed, (logp, grad)):
                assert torch.equal(torch.nan_to_num(x, 7.0), torch.nan_to_num(y, 7.0))
        other.sync()
        other.close()


def calls_that_would_end_a_capture():
    """Inside torch's capture: waits, copies that wait, fills, replays and the context's end are refused, timing records nothing, arrays may
    go; the capture ends well and its replays are right, and so is the context."""
    s = torch.cuda.Stream()
    own = _hip.Context(0, stream=s.cuda_stream)
    with torch.cuda.stream(s):
        x = torch.ones(500, 64, dtype=torch.bfloat16, device="cuda")
        w = torch.ones(300, 64, dtype=torch.bfloat16, device="cuda")
        y, z = (torch.empty(500, 300, dtype=torch.bfloat16, device="cuda") for _ in range(2))
        engine.linear(own, x, w, out=z)  # (whatever the call needs at first)
        own.graph_begin()
        engine.linear(own, x, w, out=z)
        recorded = own.graph_end()
        kept, going = own.to_device(np.arange(100, dtype=np.float32)), own.to_device(np.arange(100, dtype=np.float32))
        pinned = own.host_alloc(64)
        csr = [own.to_device(np.array(v, t)) for v, t in (([0, 1, 3], np.int64), ([2, 0, 3], np.uint32), ([1, 5, 2], np.uint32))]
        dense = engine.csr_to_dense(own, 2, *csr, 4, dtype=np.float32)
        own.profile_enable(True)
        s.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            engine.linear(own, x, w, out=y)
            for call in (own.sync, kept.download, lambda: kept.upload(np.zeros(100, np.float32)), lambda: own.profile_read("k_linear"), own.profile_reset, own.profile_dump,
                         recorded.launch, own.close, lambda: engine.csr_to_dense(own, 2, *csr, 4, dtype=np.float32, out=dense), lambda: own.call("skm_memset", kept.ptr, 0, 400)):
                raises(_hip.HipError, "captures", call)
            assert own.lib.skm_graph_destroy(own.handle, recorded.handle) == _hip.UNSUPPORTED
            del going
        own.profile_enable(False)
        for value in (2.0, 1.0, 3.0):
            x.fill_(value)
            y.zero_()
            z.zero_()
            g.replay()
            recorded.launch()
            own.sync()
            assert bool((y == 64 * value).all()) and bool((z == 64 * value).all())
        assert own.profile_read("k_linear")[0] == 0
        assert np.array_equal(kept.download(), np.arange(100, dtype=np.float32))
        assert np.array_equal(dense.download(), [[0, 0, 1, 0], [5, 0, 0, 2]])
        pinned[:] = 7
        recorded.close()
    own.close()


for check in (a_graph_that_outlives_its_context, calls_that_would_end_a_capture):
    print(check.__name__, flush=True)
    check()
print("all passed", flush=True)
