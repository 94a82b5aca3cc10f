"""The scoring operators on torch's arrays and streams.  Run as a program (tests/test_gpu_scoring.py does): torch has to be loaded
before the library, so that both use one HIP runtime."""
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


def streams():
    """No wait between the two libraries' work: the stream that both use orders it."""
    for stream in (torch.cuda.default_stream(), torch.cuda.Stream()):
        own = _hip.Context(0, stream=stream.cuda_stream)
        with torch.cuda.stream(stream):
            g = torch.Generator(device="cuda")
            g.manual_seed(1)
            x = torch.randint(-3, 4, (4000, 512), generator=g, device="cuda").to(torch.bfloat16)
            w = torch.randint(-3, 4, (700, 512), generator=g, device="cuda").to(torch.bfloat16)
            y = torch.empty(4000, 700, dtype=torch.bfloat16, device="cuda")
            for i in range(4):
                xi = x + i
                engine.linear(own, xi, w, out=y)
                copy = y.clone()
                y.fill_(-1.0)  # whole numbers below 2^24: exact before the one rounding
                assert torch.equal(copy, (xi.float() @ w.float().t()).to(torch.bfloat16))
            labels = torch.randint(0, 700, (4000,), generator=g, device="cuda")
            out = apply.log_probabilities(own, copy, labels, k=1)
            best = torch.as_tensor(out.top_index, device="cuda").long()
            assert torch.equal(copy.float().gather(1, best)[:, 0], copy.float().amax(dim=1))
            logp = torch.as_tensor(out.logp, device="cuda").double()
            want = torch.log_softmax(copy.double(), dim=1).gather(1, labels[:, None])[:, 0]
            assert float((logp - want).abs().max()) <= 2.0 ** -24 * 200 * (1 + float(want.abs().max()))
            # columns of a wider array, transposed rows, a tensor that wants a gradient, one on the host
            wide = torch.cat([x, x], dim=1)
            engine.linear(own, wide[:, 512:], w, out=y)
            assert torch.equal(y, (x.float() @ w.float().t()).to(torch.bfloat16))
            raises(ValueError, "next to each other", lambda: engine.linear(own, x.t(), w))
            raises(TypeError, "on the device", lambda: engine.linear(own, x.cpu(), w))
            raises(Exception, "grad", lambda: engine.linear(own, x.float().requires_grad_(), w.float()))
        stream.synchronize()
        own.close()


def captures():
    """Inside torch's own capture calls without scratch are recorded; those with scratch, and allocations, are refused."""
    s = torch.cuda.Stream()
    own = _hip.Context(0, stream=s.cuda_stream)
    with torch.cuda.stream(s):
        x, odd = (torch.ones(20000, k, dtype=torch.bfloat16, device="cuda") for k in (64, 63))
        w = torch.ones(300, 64, dtype=torch.bfloat16, device="cuda")
        narrow = w[:, :63]
        y = torch.empty(20000, 300, dtype=torch.bfloat16, device="cuda")
        engine.linear(own, x, w, out=y)
        s.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            engine.linear(own, x, w, out=y)
            raises(_hip.HipError, "captures", lambda: engine.linear(own, odd, narrow, out=y))
            raises(_hip.HipError, "captures", lambda: own.empty(5, np.float32))
        for value in (2.0, 1.0, 3.0):
            x.fill_(value)
            y.zero_()
            g.replay()
            s.synchronize()
            assert bool((y == 64 * value).all())
            engine.linear(own, odd, narrow, out=y)
            assert bool((y == 63).all())
    own.close()


for check in (streams, captures):
    print(check.__name__, flush=True)
    check()
print("all passed", flush=True)
