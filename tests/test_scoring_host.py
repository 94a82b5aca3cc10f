"""Parts of the scoring operators that can be checked without a device: index arithmetic of the kernels compiled for the host, and
what the library's sources and Python layer promise about streams, devices and arguments."""
import os
import re
import shutil
import subprocess

import pytest

from snekmer_amd import _hip, apply, engine
from test_scoring import CTX, LABELS, Fake, NoDevice, S, _stats

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "snekmer_amd", "csrc")


def run_on_host(tmp_path, source):
    """Compiles a program against the kernels' headers and runs it: its output."""
    if shutil.which("g++") is None:
        pytest.skip("no g++ here")
    path = tmp_path / "check.cpp"
    path.write_text(source)
    program = str(tmp_path / "check")
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", f"-I{CSRC}", str(path), "-o", program], check=True)
    return subprocess.run([program], capture_output=True, text=True, check=True, timeout=60).stdout


def test_a_labels_entry_is_inside_its_row(tmp_path):
    """Every tile of rows of 1 .. 2100 classes, labels from below 0 to a tile behind the row and far ones: a label that is a class is
    found in exactly one tile, at its place; one that is not is found in none, so that nothing is read at it."""
    out = run_on_host(tmp_path, r"""
#include <algorithm>
#include <cstdio>
#include "skm_logprob.h"
int main()
{
    const int64_t tile = 1024, far[] = {INT64_MIN, INT64_MIN + 1, -(1LL << 40), -2, 1LL << 31, 1LL << 32, (1LL << 32) + 5, 1LL << 40, INT64_MAX};
    long looked = 0;
    for (int64_t cols = 1; cols <= 2100; cols += cols < 40 || (cols > 990 && cols < 1060) || cols > 2030 ? 1 : 37) {
        auto check = [&](int64_t y) {
            int found = 0;
            for (int64_t base = 0; base < cols; base += tile) {
                const int off = lp_entry_of(y, base, (int)std::min(tile, cols - base));
                if (off < 0)
                    continue;
                ++found;
                if (base + off != y || y >= cols)
                    return false;
            }
            ++looked;
            return found == (y >= 0 && y < cols);
        };
        for (int64_t y = -3; y < cols + tile + 3; ++y)
            if (!check(y))
                return std::printf("label %lld of %lld\n", (long long)y, (long long)cols), 1;
        for (int64_t y : far)
            if (!check(y))
                return std::printf("label %lld of %lld\n", (long long)y, (long long)cols), 1;
    }
    std::printf("looked at %ld\n", looked);
}
""")
    assert int(out.split()[-1]) > 100000


@pytest.mark.parametrize("T", [1e-31, 1e-30, 1e30, 1e31, -1.0])
def test_temperatures_that_the_library_does_not_take(T):
    """Both layers refuse the same ones; the Python layer says so as it says it of any other argument."""
    for call in (lambda: apply.log_probabilities(CTX, S, LABELS, temperature=T),
                 lambda: apply.log_probabilities_backward(CTX, S, LABELS, _stats(), d_logp=Fake((4,)), temperature=T)):
        with pytest.raises(ValueError, match="temperature.*between"):
            call()


class HostTensor:
    """A tensor of a library whose type has the array interface, on the host: an error is behind it."""

    is_cuda = False

    def __init__(self, values):
        self.values = values

    @property
    def __cuda_array_interface__(self):
        raise AttributeError("the tensor is on the host")

    def __array__(self, dtype=None, copy=None):
        import numpy as np

        return np.asarray(self.values, dtype=dtype)


def test_labels_in_another_librarys_host_memory():
    """Labels may lie on the host, in whatever reads as an array there; they are looked at and copied like a list."""
    uploads, calls = [], []

    class Recorder(NoDevice):
        def to_device(self, host):
            uploads.append(host.tolist())
            return Fake(host.shape, "<i4")

        def call(self, name, *args):
            calls.append(name)

    apply.log_probabilities(Recorder(), S, HostTensor([0, 5, -1, 2]))
    assert uploads == [[0, 5, -1, 2]] and calls == ["skm_log_probabilities"]
    with pytest.raises(ValueError, match="labels: outside"):
        apply.log_probabilities(Recorder(), S, HostTensor([0, 6, -1, 2]))
    with pytest.raises(TypeError, match="on the device"):  # scores may not
        apply.log_probabilities(Recorder(), HostTensor([[1.0, 2.0]]), [0])


def test_views_of_negated_values_are_refused():
    """torch's imag of conj: the words in memory have the other sign.  Elements two apart are refused as such; one column has none."""

    class Negated(Fake):
        def is_neg(self):
            return True

    for view, ndim in ((Negated((3, 1), strides=(8, 8)), 2), (Negated((1,)), 1)):
        with pytest.raises(ValueError, match="x: a view of negated"):
            _hip.array_view(CTX, view, "x", ndim, _hip.FLOAT_TYPES)
    Negated.is_neg = lambda self: False
    assert _hip.array_view(CTX, Negated((3, 1), strides=(8, 8)), "x", 2, _hip.FLOAT_TYPES)[2] == 2


# ---------------------------------------------------------------------------- contexts over a caller's stream, as the sources handle them
def functions_of_the_library():
    """(file, name, parameters, body) of every function at file scope in the library's sources."""
    for name in sorted(os.listdir(CSRC)):
        if not name.endswith(".hip"):
            continue
        text = open(os.path.join(CSRC, name)).read()
        for m in re.finditer(r'^(?:extern "C" |static |template <[^>]*>\s*)*(?:int|bool|void)\s+(\w+)\(([^)]*)\)\s*\{', text, re.M):
            end = text.index("\n}\n", m.end())
            yield name, m.group(1), m.group(2), text[m.end():end]


def test_every_call_on_a_contexts_stream_is_on_its_device():
    """The null stream, which a context may be over, is the CURRENT device's, and launches want the stream's device to be the current one:
    whatever uses a context's stream makes its device current first.  (One device here: the calls' sources are looked at.)"""
    scopes = ("SKM_ON_DEVICE(", "SKM_ON_STREAM(", "skm_device_scope scope(")
    # its stream is never the null stream; swaps two contexts' streams of one device and calls what is looked at here
    exempt = {"skm_graph_end", "skm_cosine_csr_phase"}
    looked = 0
    for file, name, parameters, body in functions_of_the_library():
        if "skm_ctx" not in parameters or name in exempt:
            continue
        # entry points, and what they call behind the scope of another function
        if name.startswith("skm_") and not name.endswith("_async") and name not in ("skm_ws", "skm_pool_alloc", "skm_pool_free", "skm_foreign_capture"):
            use = re.search(r"(hip[A-Z]\w+\([^;]*|<<<[^;]*|hipStream_t \w+ = )ctx->stream", body)
            if use is None:
                continue
            looked += 1
            first = min((body.index(s) for s in scopes if s in body), default=None)
            assert first is not None and first < use.start(), f"{file}: {name}"
        assert "hipSetDevice" not in body, f"{file}: {name}"  # (the scopes give the caller's device back)
    assert looked > 60


ASKS = ("SKM_NOT_WHILE_CAPTURED(", "skm_ws(", "skm_foreign_capture(")


def test_nothing_waits_for_a_stream_that_its_owner_captures():
    """A wait inside the owner's capture ends the capture: every function that waits has asked first, by itself or by asking for scratch
    memory, which is refused then."""
    asks = ASKS
    # waits of the pool (for streams that it has asked about) and at the end of the process
    exempt = {"park_locked", "quiesce_locked", "skm_stream_release", "shutdown_at_exit"}
    looked = 0
    for file, name, parameters, body in functions_of_the_library():
        wait = re.search(r"hip(Stream|Event)Synchronize\(", body)
        if wait is None or name in exempt:
            continue
        looked += 1
        first = min((body.index(a) for a in asks if a in body), default=None)
        assert first is not None and first < wait.start(), f"{file}: {name}"
    assert looked > 20


def test_no_fill_is_recorded_into_an_owners_capture():
    """Fills that a stream capture records have given wrong results on replays after the first: whoever fills has asked, too."""
    exempt = {"skm_count_stage_async"}  # (behind skm_count_csr and skm_vectorize_csr)
    looked = 0
    for file, name, parameters, body in functions_of_the_library():
        fill = re.search(r"hipMemsetAsync\(", body)
        if fill is None or name in exempt:
            continue
        looked += 1
        first = min((body.index(a) for a in ASKS if a in body), default=None)
        assert first is not None and first < fill.start(), f"{file}: {name}"
    assert looked > 15
