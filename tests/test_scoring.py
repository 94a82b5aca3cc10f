"""Refusals of the scoring operators (engine.linear, apply.log_probabilities and their backward passes) and the conversions
beside them.  No kernel is launched here: every call has to raise before it reaches the library."""
import numpy as np
import pytest

from snekmer_amd import _hip, apply, engine


class NoDevice:
    """A context whose library must not be reached."""

    device = 0
    handle = 1

    @property
    def lib(self):
        return _hip.load_library()

    def call(self, name, *args):
        raise AssertionError(f"{name} was reached")

    def empty(self, shape, dtype):
        shape = shape if isinstance(shape, tuple) else (shape,)
        return Fake(shape, {np.dtype(np.float32): "<f4", np.dtype(np.float16): "<f2", np.dtype(np.int32): "<i4", _hip.bfloat16: "<V2"}[np.dtype(dtype)])


class Device:
    def __init__(self, index):
        self.index = index


class Fake:
    """The array interface of an array that is not there."""

    def __init__(self, shape, typestr="<f4", strides=None, device=0, readonly=False, mask=None):
        self.shape = shape
        self.__dict__["iface"] = {"shape": shape, "typestr": typestr, "data": (0x7000000000, readonly), "strides": strides, "version": 2}
        if mask is not None:
            self.iface["mask"] = mask
        self.device = Device(device)

    @property
    def __cuda_array_interface__(self):
        return self.iface


CTX = NoDevice()


def test_bfloat16_words_round_to_nearest_even_and_come_back():
    values = np.array([0.0, -0.0, 1.0, 1.00390625, 1.01171875, 3.4e38, -3.4e38, np.inf, -np.inf, 1e-40, 65280.0], dtype=np.float32)
    back = _hip.from_bfloat16(_hip.to_bfloat16(values))
    want = [0.0, -0.0, 1.0, 1.0, 1.015625, np.inf, -np.inf, np.inf, -np.inf, back[9], 65280.0]  # halfway cases go to the even word
    assert np.array_equal(back, np.array(want, dtype=np.float32))
    assert abs(back[9] - 1e-40) <= 2.0 ** -134  # subnormal words are 2^-133 apart
    assert np.isnan(_hip.from_bfloat16(_hip.to_bfloat16(np.array([np.nan, -np.nan], dtype=np.float32)))).all()
    words = np.arange(1 << 16, dtype=np.uint16)
    finite = _hip.from_bfloat16(words.view(_hip.bfloat16))
    ok = ~np.isnan(finite)
    assert np.array_equal(_hip.to_bfloat16(finite)[ok].view(np.uint16), words[ok])
    assert _hip.to_bfloat16(np.zeros((3, 5), np.float32)).shape == (3, 5)


@pytest.mark.parametrize("make, error, says", [
    (lambda: np.zeros((2, 3), np.float32), TypeError, "on the device"),
    (lambda: [[1.0]], TypeError, "on the device"),
    (lambda: Fake((2, 3), "<f8"), TypeError, "type <f8"),
    (lambda: Fake((2, 3), device=1), ValueError, "device 1"),
    (lambda: Fake((6,)), ValueError, "1 dimensions"),
    (lambda: Fake((2, 3), strides=(12, 8)), ValueError, "next to each other"),
    (lambda: Fake((2, 3), strides=(8, 4)), ValueError, "overlap"),
    (lambda: Fake((2, 3), strides=(0, 4)), ValueError, "overlap"),
    (lambda: Fake((2, 3), strides=(-12, 4)), ValueError, "overlap"),
    (lambda: Fake((2, 3), strides=(14, 4)), ValueError, "between elements"),
    (lambda: Fake((2, 3), mask=object()), ValueError, "masked"),
])
def test_arrays_that_the_operators_do_not_take(make, error, says):
    with pytest.raises(error, match=says):
        _hip.array_view(CTX, make(), "x", 2, _hip.FLOAT_TYPES)


def test_views_of_strided_rows():
    assert _hip.array_view(CTX, Fake((2, 3)), "x", 2, _hip.FLOAT_TYPES)[1:] == ((2, 3), 3, "<f4")
    assert _hip.array_view(CTX, Fake((2, 3), "<V2", strides=(16, 2)), "x", 2, _hip.FLOAT_TYPES)[1:] == ((2, 3), 8, "<V2")
    assert _hip.array_view(CTX, Fake((1, 3), strides=(2, 4)), "x", 2, _hip.FLOAT_TYPES)[2] == 3  # one row: its stride is never used
    assert _hip.array_view(CTX, Fake((4, 1), strides=(8, 100)), "x", 2, _hip.FLOAT_TYPES)[2] == 2  # one column: only rows have a stride
    with pytest.raises(ValueError, match="read-only"):
        _hip.array_view(CTX, Fake((2, 3), readonly=True), "x", 2, _hip.FLOAT_TYPES, writable=True)


X, W = Fake((4, 6)), Fake((5, 6))


@pytest.mark.parametrize("call, error, says", [
    (lambda: engine.linear(CTX, X, Fake((5, 7))), ValueError, "w: shape"),
    (lambda: engine.linear(CTX, X, Fake((5, 6), "<f2")), TypeError, "w: elements"),
    (lambda: engine.linear(CTX, X, W, bias=Fake((4,))), ValueError, "bias: shape"),
    (lambda: engine.linear(CTX, X, W, residual=Fake((4, 6))), ValueError, "residual: shape"),
    (lambda: engine.linear(CTX, X, W, preact=Fake((5, 4))), ValueError, "preact: shape"),
    (lambda: engine.linear(CTX, X, W, out=Fake((4, 5), "<V2")), TypeError, "out: elements"),
    (lambda: engine.linear(CTX, X, W, out=Fake((4, 5), readonly=True)), ValueError, "out: the array is read-only"),
    (lambda: engine.linear(CTX, X, W, activation="swish"), ValueError, "activation"),
    (lambda: engine.linear(CTX, X, W, activation=["relu"]), ValueError, "activation"),
    (lambda: engine.linear_backward(CTX, Fake((4, 5)), X, W, activation="gelu"), ValueError, "preact"),
    (lambda: engine.linear_backward(CTX, Fake((4, 5)), X, None), ValueError, "w: dx"),
    (lambda: engine.linear_backward(CTX, Fake((4, 5)), None, W), ValueError, "x: dw"),
    (lambda: engine.linear_backward(CTX, Fake((3, 5)), X, W), ValueError, "x: shape"),
    (lambda: engine.linear_backward(CTX, Fake((4, 5)), X, Fake((5, 7))), ValueError, "w: shape"),
    (lambda: engine.linear_backward(CTX, Fake((4, 5)), X, W, dx=Fake((4, 7))), ValueError, "dx: shape"),
    (lambda: engine.linear_backward(CTX, Fake((4, 5)), X, W, dbias=Fake((5,), "<f2")), TypeError, "dbias: elements"),
])
def test_linear_refuses(call, error, says):
    with pytest.raises(error, match=says):
        call()


S = Fake((4, 6))
LABELS = Fake((4,), "<i4")


def _stats(**more):
    return apply.LogProbabilities(stats=Fake((4, 2)), **more)


@pytest.mark.parametrize("call, error, says", [
    (lambda: apply.log_probabilities(CTX, S, LABELS, k=17), ValueError, "k: 17"),
    (lambda: apply.log_probabilities(CTX, S, LABELS, k=-1), ValueError, "k: -1"),
    (lambda: apply.log_probabilities(CTX, S, LABELS, temperature=0.0), ValueError, "temperature"),
    (lambda: apply.log_probabilities(CTX, S, LABELS, temperature=float("nan")), ValueError, "temperature"),
    (lambda: apply.log_probabilities(CTX, S, LABELS, temperature=float("inf")), ValueError, "temperature"),
    (lambda: apply.log_probabilities(CTX, S, LABELS, ncols=7), ValueError, "ncols"),
    (lambda: apply.log_probabilities(CTX, S, LABELS, ncols=0), ValueError, "ncols"),
    (lambda: apply.log_probabilities(CTX, Fake((4, 0)), LABELS), ValueError, "no classes"),
    (lambda: apply.log_probabilities(CTX, S, Fake((5,), "<i4")), ValueError, "labels: shape"),
    (lambda: apply.log_probabilities(CTX, S, Fake((4,), "<f4")), TypeError, "labels: elements"),
    (lambda: apply.log_probabilities(CTX, S, [0.5, 1, 2, 3]), TypeError, "labels"),
    (lambda: apply.log_probabilities(CTX, S, [0, 1, 2, 6]), ValueError, "labels: outside"),
    (lambda: apply.log_probabilities(CTX, S, [0, 1, -2, 3]), ValueError, "labels: outside"),
    (lambda: apply.log_probabilities(CTX, S, LABELS, mask=Fake((4, 5), "|u1")), ValueError, "mask: shape"),
    (lambda: apply.log_probabilities(CTX, S, LABELS, mask=Fake((4,), "|u1")), ValueError, "mask: shape"),
    (lambda: apply.log_probabilities(CTX, S, LABELS, mask=Fake((4, 6), "<i4")), TypeError, "mask: elements"),
    (lambda: apply.log_probabilities(CTX, S, None, out=apply.LogProbabilities(logp=Fake((4,)))), ValueError, "labels"),
    (lambda: apply.log_probabilities(CTX, S, LABELS, out=apply.LogProbabilities(top_index=Fake((4, 1), "<i4"))), ValueError, "k is 0"),
    (lambda: apply.log_probabilities(CTX, S, LABELS, k=2, out=apply.LogProbabilities(top_index=Fake((4, 3), "<i4"))), ValueError, "top_index: shape"),
    (lambda: apply.log_probabilities(CTX, S, LABELS, k=2, out=apply.LogProbabilities(top_logp=Fake((4, 2), strides=(12, 4)))), ValueError, "top_logp: rows"),
    (lambda: apply.log_probabilities(CTX, S, LABELS, out=apply.LogProbabilities(entropy=Fake((4,), strides=(8,)))), ValueError, "entropy"),
    (lambda: apply.log_probabilities_backward(CTX, S, LABELS, _stats()), ValueError, "d_logp, d_entropy"),
    (lambda: apply.log_probabilities_backward(CTX, S, None, _stats(), d_logp=Fake((4,))), ValueError, "labels"),
    (lambda: apply.log_probabilities_backward(CTX, S, LABELS, apply.LogProbabilities(), d_logp=Fake((4,))), ValueError, "forward"),
    (lambda: apply.log_probabilities_backward(CTX, S, LABELS, _stats(), d_entropy=Fake((4,))), ValueError, "forward"),
    (lambda: apply.log_probabilities_backward(CTX, S, LABELS, _stats(), d_logp=Fake((4, 1))), ValueError, "d_logp"),
    (lambda: apply.log_probabilities_backward(CTX, S, LABELS, _stats(), d_logp=Fake((4,)), out=Fake((4, 7))), ValueError, "out: shape"),
    (lambda: apply.log_probabilities_backward(CTX, S, LABELS, _stats(), d_logp=Fake((4,)), out=Fake((4, 6), "<f2")), TypeError, "out: elements"),
])
def test_log_probabilities_refuse(call, error, says):
    with pytest.raises(error, match=says):
        call()


def test_a_context_is_confined_or_on_the_callers_stream():
    with pytest.raises(ValueError, match="caller's stream"):
        _hip.Context(0, cu_groups=(0, 3), stream=0)


def test_the_library_refuses_a_null_context():
    lib = _hip.load_library()
    null = [None] * 4
    assert lib.skm_linear(None, 0, 0, 1, 1, 1, None, 1, None, 1, *null[:2], 1, None, 1, None, 1) == -1
    assert lib.skm_linear_backward(None, 0, 0, 1, 1, 1, None, 1, None, 1, None, 1, None, 1, None, 1, None, 1, None) == -1
    assert lib.skm_log_probabilities(None, 0, 1, 1, None, 1, None, 0, None, 32, 0, 1.0, None, None, None, None, None) == -1
    assert lib.skm_log_probabilities_backward(None, 0, 1, 1, None, 1, None, 0, None, 32, 1.0, None, None, None, None, None, 1) == -1
