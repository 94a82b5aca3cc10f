"""The scoring operators at the ends of what their documentation allows: labels that are no class, gradients and scores of extreme
size, several errors at once, arrays without cells, other libraries' captures."""
import math
import os
import subprocess
import sys

import numpy as np
import pytest

from snekmer_amd import _hip, apply, engine
from test_gpu_scoring import HALF_STEP, SMALLEST, U, block, check_logp, plain_logp, rounded, values, whole_numbers

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    c = _hip.Context(0)
    yield c
    c.close()


# ---------------------------------------------------------------------------- labels that are no class
@pytest.mark.parametrize("dt", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("masked", [False, True])
@pytest.mark.parametrize("a", [1, 50, 1023, 1025, 2500])
def test_gradient_of_rows_with_wrong_labels(ctx, a, masked, dt):
    """Labels from the row's end to the end of its last tile and far behind it, in every row and the last one: NaN for the row's classes,
    0 where a class is not allowed, the other rows as without them."""
    rng = np.random.default_rng(a)
    end = -(-a // 1024) * 1024
    wrong = [a, a + 1, end - 1, end, end + 7, -2, 2 ** 31 - 1, 2 ** 32 + 3, 2 ** 62]
    labels = np.concatenate([[v, i % a] for i, v in enumerate(wrong)] + [[a]]).astype(np.int64)
    n = labels.size
    words, s = rounded(block("normal", n, a, a), dt)
    mask = (rng.random((n, a)) < 0.7).astype(np.uint8) if masked else None
    right = np.where((labels >= 0) & (labels < a), labels, -1)
    d, dm = ctx.to_device(words), None if mask is None else ctx.to_device(mask)
    ones = ctx.to_device(np.ones(n, np.float32))
    fwd = apply.log_probabilities(ctx, d, right, mask=dm)
    want = values(apply.log_probabilities_backward(ctx, d, right, fwd, d_logp=ones, mask=dm).download(), dt)
    got = apply.log_probabilities_backward(ctx, d, ctx.to_device(labels), fwd, d_logp=ones, mask=dm)
    with pytest.raises(_hip.HipError, match="label outside"):
        ctx.sync()
    got = values(got.download(), dt)
    allowed = np.ones((n, a), bool) if mask is None else mask != 0
    bad = right != labels
    assert np.isnan(got[bad][allowed[bad]]).all() and (got[bad][~allowed[bad]] == 0).all()
    assert np.array_equal(got[~bad], want[~bad])


# ---------------------------------------------------------------------------- gradients and scores of extreme size
def exact_gradient(want, labels, gl, gh, T):
    """[gl ((j == y) - p_j) - gh p_j (z_j + H)] / T in 64 bits; p z is 0 where p is."""
    z, p, h = np.where(want["p"] > 0, want["z"], 0.0), want["p"], want["entropy"][:, None]
    known = labels >= 0
    g = np.where(known, gl, 0.0)
    out = -g[:, None] * p - gh[:, None] * p * (z + h)
    at = np.flatnonzero(known), labels[known]
    out[at] += g[known] * (p[at] - np.expm1(want["z"][at]))
    return out / T


@pytest.mark.parametrize("dt", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("T", [0.05, 1.0])
def test_entropy_gradient_of_large_size_beside_classes_at_the_types_lowest_value(ctx, dt, T):
    """Classes that a mask filled with the type's lowest value have p = 0 in any precision, and no part in the gradient, however large the
    gradient that comes in (2^25: a scaled loss; 2^80); the label may be one of them.  p is off by (4 |d| + 4 l + 8) u relative, d the scaled
    difference below 2^8 here where p is not 0, plus what l and H are off: 2^-13 of the terms covers them.  p below 2^-126 may be 0."""
    lowest = {"f32": np.finfo(np.float32).min, "f16": -65504.0, "bf16": -3.3895313892515355e38}[dt]
    rng = np.random.default_rng(5)
    n, a = 6, 1500
    s = rng.normal(size=(n, a))
    s[rng.random((n, a)) < 0.5] = lowest
    s[3] = lowest
    s[3, 700] = 1.0  # one class is left
    s[4] = lowest    # all of them alike
    words, s = rounded(s, dt)
    labels = np.array([0, -1, 1499, 700, 3, 5])
    labels[5] = np.flatnonzero(s[5] == s[5].min())[0]  # (a class that the mask filled)
    want = plain_logp(s, labels, 0, T)
    d = ctx.to_device(words)
    fwd = apply.log_probabilities(ctx, d, labels, temperature=T)
    for size in (2.0 ** 25, 2.0 ** 80) if dt != "f16" else (2.0 ** 7,):
        gl, gh = rng.normal(size=n).astype(np.float32), (size * rng.normal(size=n)).astype(np.float32)
        for use_l in (True, False):
            g = gl.astype(np.float64) * use_l
            got = values(apply.log_probabilities_backward(ctx, d, labels, fwd, d_logp=ctx.to_device(gl) if use_l else None, d_entropy=ctx.to_device(gh),
                                                          temperature=T).download(), dt)
            exact = exact_gradient(want, labels, g, gh.astype(np.float64), T)
            z = np.where(want["p"] > 0, want["z"], 0.0)
            weight = (np.abs(g)[:, None] + np.abs(gh.astype(np.float64))[:, None] * (np.abs(z) + want["entropy"][:, None] + 1.0)) / T
            terms = want["p"] * weight + np.abs(g)[:, None] * (np.arange(a) == labels[:, None]) / T
            assert (np.abs(got - exact) <= 2.0 ** -13 * terms + 2.0 ** -125 * weight + HALF_STEP[dt] * np.abs(exact) * 1.01 + SMALLEST[dt]).all()
            gone = (want["p"] == 0) & (np.arange(a) != labels[:, None])
            assert gone[:4].any() and (got[gone] == 0).all()


@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("T", [1e-20, 1e-29])
def test_gradients_at_temperatures_near_nothing(ctx, dt, T):
    """Everything is on the largest score: H = 0 and p is 0 or 1, so the entropy's gradient is 0 and the label's is +-gl / T (two roundings
    of float32: 1 / T and the product)."""
    rng = np.random.default_rng(8)
    words, s = rounded(np.stack([rng.permutation(700) / 64.0 - 3.0 for _ in range(5)]), dt)  # (steps of 1 / 64: distinct in float32)
    if dt == "bf16":
        s[:, 0], words[:, 0] = 20.0, rounded(np.full(5, 20.0), dt)[0]  # (the largest one, once)
    labels = np.array([3, -1, 0, 699, 5])
    labels[4] = s[4].argmax()
    gl, gh = rng.normal(size=5).astype(np.float32), rng.normal(size=5).astype(np.float32)
    d = ctx.to_device(words)
    fwd = apply.log_probabilities(ctx, d, labels, temperature=T)
    assert (fwd.entropy.download() == 0).all()
    got = values(apply.log_probabilities_backward(ctx, d, labels, fwd, d_logp=ctx.to_device(gl), d_entropy=ctx.to_device(gh), temperature=T).download(), dt)
    exact = np.zeros((5, 700))
    for i, y in enumerate(labels):
        if y >= 0:
            exact[i, y] += gl[i] / T
            exact[i, s[i].argmax()] -= gl[i] / T
    assert (np.abs(got - exact) <= (4 * U + HALF_STEP[dt] * 1.01) * np.abs(exact)).all()


# ---------------------------------------------------------------------------- activations, relative to themselves
def one_term(ctx, z, name, dt):
    """(y, slope) of an activation at the values z of type dt, as float64: the product x z with x = 1 is exact, so is the one of dz."""
    words, zt = rounded(np.asarray(z)[:, None], dt)
    one = ctx.to_device(rounded(np.ones((1, 1)), dt)[0])
    y, pre = engine.linear(ctx, ctx.to_device(words), one, activation=name, preact=True)
    g = ctx.to_device(rounded(np.ones_like(words, dtype=np.float32) if dt != "bf16" else np.ones(words.shape, np.float32), dt)[0])
    dx, _, _ = engine.linear_backward(ctx, g, None, one, activation=name, preact=pre, dw=None, dbias=None)
    return zt[:, 0], values(y.download(), dt)[:, 0], values(dx.download(), dt)[:, 0]


@pytest.mark.parametrize("dt", ["f32", "f16", "bf16"])
def test_sigmoids_slope_relative_to_itself(ctx, dt):
    """e / (1 + e)^2 with e = exp(-|z|): the exponential's argument has one rounding and the instruction's own ulp, (|z| + 2) 2^-23, the rest
    (the sum, a reciprocal of one ulp twice, two products) below 8 u; half a step of the type follows, of its smallest numbers too."""
    z, _, got = one_term(ctx, np.concatenate([np.linspace(-80, 80, 641), [12.0, 15.0, 17.0, 20.0]]), "sigmoid", dt)
    e = np.exp(-np.abs(z))
    want = e / (1 + e) ** 2
    room = (np.abs(z) + 2) * 2.0 ** -23 + 8 * U + HALF_STEP[dt] * 1.01
    assert (np.abs(got - want) <= room * want + SMALLEST[dt]).all()
    assert (got[np.abs(z) < 10] > 0).all() and np.array_equal(got[:641], got[:641][::-1])  # (an even function)


def test_float32_activations_relative_to_themselves(ctx):
    """Roundings of float32, u = 2^-24 each.  exp(-|z|): what the argument's rounding loses is put back; the instruction's ulp (2 u) and a
    rounding, squared, and the square's: 8 u.  sigmoid: 8 + 1 (sum) + 2 (reciprocal) + 1: 16 u covers it.  silu: one more.  gelu: the
    polynomial 5 u, its argument 3 u, the exponential 8, two products: 32 u.  gelu_tanh: the argument 2 u of the exponential has six
    roundings, each the argument's size in the result.  Below 2^-126 half a step of the smallest numbers, times z where z multiplies."""
    z, y, slope = one_term(ctx, np.concatenate([np.linspace(-103, 87, 3801), -(2.0 ** np.arange(-20, 6.5, 0.5))]), "sigmoid", "f32")
    e = np.exp(-np.abs(z))
    want = np.where(z > 0, 1 / (1 + e), e / (1 + e))
    tiny = 2.0 ** -148
    assert (np.abs(y - want) <= 16 * U * want + tiny).all()
    want = e / (1 + e) ** 2
    assert (np.abs(slope - want) <= 20 * U * want + tiny).all()  # (the reciprocal twice)
    z, y, slope = one_term(ctx, z, "silu", "f32")
    want = z * np.where(z > 0, 1, e) / (1 + e)
    assert (np.abs(y - want) <= 17 * U * np.abs(want) + tiny * np.abs(z)).all()
    low = z < -3  # the slope s (1 + z (1 - s)) has its root at -1.28; here z / (1 + z) is below 1.5
    s = e / (1 + e)
    want = (s * (1 + z * (1 - s)))[low]
    assert (np.abs(slope[low] - want) <= 32 * U * np.abs(want) + tiny * np.abs(z[low])).all()
    z, y, _ = one_term(ctx, -np.linspace(1e-3, 13.0, 2001), "gelu", "f32")
    want = z * 0.5 * np.vectorize(math.erfc)(-z / math.sqrt(2.0))
    assert (np.abs(y - want) <= 32 * U * np.abs(want) + tiny * np.abs(z)).all()
    z, y, _ = one_term(ctx, np.linspace(-10.2, 10.0, 2001), "gelu_tanh", "f32")
    two_u = 2 * math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3)
    want = z / (1 + np.exp(-two_u))
    assert (np.abs(y - want) <= (6 * np.abs(two_u) + 20) * U * np.abs(want) + tiny * np.abs(z)).all()


@pytest.mark.parametrize("dt", ["f16", "bf16"])
@pytest.mark.parametrize("name, low", [("sigmoid", -80.0), ("silu", -80.0), ("gelu", -12.0), ("gelu_tanh", -9.0)])
def test_activations_of_16_bits_relative_to_themselves(ctx, name, low, dt):
    """The plain exponential is off by its argument's rounding, the argument times 2^-23 covers it (below 110: 2^-16), a dozen roundings of
    float32 around it; half a step of the type follows."""
    z, y, _ = one_term(ctx, np.linspace(low, 20.0, 1601), name, dt)
    if name == "gelu":
        want = z * 0.5 * np.vectorize(math.erfc)(-z / math.sqrt(2.0))
    else:
        u = 2 * math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3) if name == "gelu_tanh" else z
        e = np.exp(-np.abs(u))
        want = (1.0 if name == "sigmoid" else z) * np.where(u > 0, 1.0, e) / (1 + e)
    assert (np.abs(y - want) <= (2.0 ** -15 + HALF_STEP[dt] * 1.01) * np.abs(want) + SMALLEST[dt]).all()


@pytest.mark.parametrize("name", ["gelu", "gelu_tanh", "silu", "sigmoid"])
def test_float32_activations_keep_nan_and_reach_their_limits(ctx, name):
    z, y, slope = one_term(ctx, [np.nan, 300.0, -300.0, 2.0 ** 127, -2.0 ** 127, 0.0, -0.0], name, "f32")
    assert np.isnan(y[0]) and np.isnan(slope[0])
    up = np.ones(2) if name == "sigmoid" else z[[1, 3]]
    assert np.array_equal(y[[1, 3]], up) and np.array_equal(y[[2, 4]], [0, 0])
    assert np.array_equal(slope[1:5], [0, 0, 0, 0] if name == "sigmoid" else [1, 0, 1, 0])
    half = 0.5 if name != "sigmoid" else 0.25
    assert np.allclose(y[5:], 0.5 if name == "sigmoid" else 0.0, rtol=32 * U, atol=0) and np.allclose(slope[5:], half, rtol=32 * U)


# ---------------------------------------------------------------------------- errors that only the device sees
@pytest.mark.parametrize("first", ["sequence", "label"])
def test_two_errors_at_once_are_both_reported(ctx, first):
    """A bound that a sequence exceeds and a label that is no class, neither waited for in between: one report names both, once."""
    from snekmer_amd import alphabet

    own = _hip.Context(0)
    lut = alphabet.build_lut("hydro")
    batch = engine.SeqBatch.from_strings(own, ["MKVLAAGIWMKVLAAGIW", "MKVL"])
    batch.max_len = 6
    s = own.to_device(whole_numbers((3, 20), 1))
    labels = own.to_device(np.array([0, 20, 1], np.int32))
    calls = [lambda: engine.vectorize_fused(own, batch, lut, 4), lambda: apply.log_probabilities(own, s, labels)]
    kept = [call() for call in (calls if first == "sequence" else calls[::-1])]
    with pytest.raises(_hip.HipError, match="EMPTY") as e:
        own.sync()
    assert e.value.code == -1 and "label outside" in str(e.value)
    own.sync()
    del kept
    own.close()


class At:
    """An array of another library at any address."""

    def __init__(self, base, shape, typestr, offset):
        self.base, self.shape = base, shape
        self.interface = {"shape": shape, "typestr": typestr, "data": (base.ptr + offset, False), "strides": None, "version": 2}

    @property
    def __cuda_array_interface__(self):
        return self.interface


def test_vectors_between_addresses_of_their_type_are_refused(ctx):
    """The rows' vectors are read and written as whole elements (scores, as documented, need no more than their own type's alignment)."""
    s = ctx.to_device(whole_numbers((4, 10), 1))
    room = ctx.zeros(400, np.uint8)
    labels = ctx.to_device(np.arange(4, dtype=np.int32))
    fwd = apply.log_probabilities(ctx, s, labels)
    ones = ctx.to_device(np.ones(4, np.float32))
    f, i = "<f4", "<i4"
    for name, out in (("logp", At(room, (4,), f, 2)), ("entropy", At(room, (4,), f, 1)), ("stats", At(room, (4, 2), f, 6)), ("top_index", At(room, (4, 2), i, 2)),
                      ("top_logp", At(room, (4, 2), f, 3))):
        with pytest.raises(_hip.HipError, match=f"{name} is not aligned"):
            apply.log_probabilities(ctx, s, labels, k=2, out=apply.LogProbabilities(**{name: out}))
    for wrong in (At(room, (4,), i, 2), At(room, (4,), "<i8", 4)):
        with pytest.raises(_hip.HipError, match="labels is not aligned"):
            apply.log_probabilities(ctx, s, wrong)
    backward = lambda **more: apply.log_probabilities_backward(ctx, s, more.pop("labels", labels), more.pop("forward", fwd), **more)
    for name, call in (("labels", lambda: backward(labels=At(room, (4,), "<i8", 4), d_logp=ones)), ("grad_logp", lambda: backward(d_logp=At(room, (4,), f, 2))),
                       ("grad_entropy", lambda: backward(d_entropy=At(room, (4,), f, 2))),
                       ("stats", lambda: backward(d_logp=ones, forward=apply.LogProbabilities(stats=At(room, (4, 2), f, 2)))),
                       ("entropy", lambda: backward(d_entropy=ones, forward=apply.LogProbabilities(stats=fwd.stats, entropy=At(room, (4,), f, 2))))):
        with pytest.raises(_hip.HipError, match=f"{name} is not aligned"):
            call()
    four = apply.log_probabilities(ctx, s, At(room, (4,), "<i8", 8), out=apply.LogProbabilities(logp=At(room, (4,), f, 100), stats=At(room, (4, 2), f, 204)))
    ctx.sync()
    assert four.host() == {}  # (on their own addresses they are taken)


# ---------------------------------------------------------------------------- arrays without cells
class Nowhere:
    """An array without cells, as other libraries hold it: at address 0."""

    def __init__(self, shape, typestr="<f4"):
        assert 0 in shape
        self.shape = shape
        self.interface = {"shape": shape, "typestr": typestr, "data": (0, False), "strides": None, "version": 2}

    @property
    def __cuda_array_interface__(self):
        return self.interface


def test_arrays_without_cells_need_no_address(ctx):
    f = np.float32
    w, x = ctx.to_device(whole_numbers((4, 5), 1)), ctx.to_device(whole_numbers((3, 5), 2))
    engine.linear(ctx, Nowhere((0, 5)), w, residual=Nowhere((0, 4)), preact=Nowhere((0, 4)), out=Nowhere((0, 4)))
    y = engine.linear(ctx, Nowhere((3, 0)), Nowhere((4, 0)), bias=ctx.to_device(np.ones(4, f)))
    assert (y.download() == 1).all()
    # no rows: dx has no cells, dw and dbias are empty sums
    dx = Nowhere((0, 5))
    assert engine.linear_backward(ctx, Nowhere((0, 4)), None, w, dx=dx, dw=None, dbias=None)[0] is dx
    _, dw, db = engine.linear_backward(ctx, Nowhere((0, 4)), Nowhere((0, 5)), w, dx=dx)
    assert (dw.download() == 0).all() and (db.download() == 0).all()
    # no outputs, no features
    dx, dw, db = engine.linear_backward(ctx, Nowhere((3, 0)), x, Nowhere((0, 5)), dw=Nowhere((0, 5)), dbias=Nowhere((0,)))
    assert (dx.download() == 0).all()
    engine.linear_backward(ctx, ctx.to_device(whole_numbers((3, 4), 3)), Nowhere((3, 0)), Nowhere((4, 0)), dx=Nowhere((3, 0)), dw=Nowhere((4, 0)), dbias=None)
    _, _, db = engine.linear_backward(ctx, ctx.to_device(np.ones((3, 4), f)), Nowhere((3, 0)), Nowhere((4, 0)), dx=Nowhere((3, 0)), dw=Nowhere((4, 0)))
    assert (db.download() == 3).all()
    # no score rows
    s, one = Nowhere((0, 7)), Nowhere((0,))
    out = apply.LogProbabilities(logp=one, entropy=Nowhere((0,)), stats=Nowhere((0, 2)), top_index=Nowhere((0, 3), "<i4"), top_logp=Nowhere((0, 3)))
    apply.log_probabilities(ctx, s, Nowhere((0,), "<i8"), k=3, out=out)
    for more in (dict(d_logp=one), dict(d_entropy=one), dict(d_logp=one, d_entropy=one)):
        apply.log_probabilities_backward(ctx, s, Nowhere((0,), "<i4"), out, out=s, **more)
    with pytest.raises(_hip.HipError, match="no gradient is asked for"):
        engine.linear_backward(ctx, ctx.to_device(whole_numbers((3, 4), 3)), x, w, dx=None, dw=None, dbias=None)
    ctx.sync()


# ---------------------------------------------------------------------------- beside other libraries
@pytest.mark.parametrize("guard", ["0", "1"])
def test_while_torch_captures(guard):
    """tests/torch_interop_edges.py, in a process that loads torch first; with and without the bytes that guard the ends of arrays."""
    run = subprocess.run([sys.executable, "-u", os.path.join(os.path.dirname(__file__), "torch_interop_edges.py")], capture_output=True, text=True, timeout=110,
                         env=dict(os.environ, SKM_GUARD=guard))
    assert run.returncode == 0 and run.stdout.rstrip().endswith("all passed"), run.stdout + run.stderr


# ---------------------------------------------------------------------------- as they are used together
@pytest.mark.parametrize("alpha, k, full", [("solvacc", 6, True), ("red6", 5, False), ("hydro", 7, True)])
def test_a_head_over_the_counts_of_sequences(ctx, alpha, k, full):
    """Sequences -> k-mer counts -> dense rows (the whole basis, or the one that was observed) -> scores of a head -> log probabilities of the
    families -> gradients, all on the device; each step against float64 from what the step before it left, the gradient against the formula."""
    from helpers import ensure_red6
    from snekmer_amd import alphabet
    from snekmer_amd.synth import synth_families

    ensure_red6()
    lut = alphabet.build_lut(alpha)
    n, a = 300, 15
    res, off, _ = synth_families(n, 90, family=20, seed=4)
    batch = engine.SeqBatch(ctx, res, off)
    csr = engine.count_csr(ctx, batch, lut, k)
    if full:
        width = lut.nsym ** k
        x = engine.csr_to_dense(ctx, n, csr.rowptr, csr.codes, csr.counts, width, dtype=np.float32)
    else:
        basis = engine.build_basis(ctx, csr, lut.nsym, k)
        width = basis.ncols
        x = engine.csr_to_dense(ctx, n, csr.rowptr, csr.colidx, csr.counts, width, dtype=np.float32)
    rowptr, counts = csr.rowptr.download(n + 1), csr.counts.download(csr.nnz)
    columns = (csr.codes if full else csr.colidx).download(csr.nnz).astype(np.int64)
    dense = np.zeros((n, width))
    dense[np.repeat(np.arange(n), np.diff(rowptr)), columns] = counts
    assert np.array_equal(x.download(), dense) and dense.sum() > 50 * n
    rng = np.random.default_rng(k)
    w, b = (rng.normal(size=(a, width)) / 8).astype(np.float32), rng.normal(size=a).astype(np.float32)
    groups = np.arange(n) // 20
    dw_, db_ = ctx.to_device(w), ctx.to_device(b)
    z = engine.linear(ctx, x, dw_, bias=db_)
    w64, z32 = w.astype(np.float64), z.download().astype(np.float64)
    room = (width + 2) * U * (dense @ np.abs(w64).T + np.abs(b))
    assert (np.abs(z32 - (dense @ w64.T + b)) <= room).all()
    T = 0.8
    lp = apply.log_probabilities(ctx, z, groups, k=3, temperature=T)
    want = plain_logp(z32, groups, 3, T)
    check_logp(lp.host(), want, a, T, 3)
    ds = apply.log_probabilities_backward(ctx, z, groups, lp, d_logp=ctx.to_device(np.full(n, -1.0 / n, np.float32)), temperature=T)
    g = ds.download().astype(np.float64)
    exact = exact_gradient(want, groups, np.full(n, -1.0 / n), np.zeros(n), T)
    # p: (4 |d| + 4 l + 8) u and what l is off, (16 + 90 + 4 l) u: all |d| below 2^7 here
    assert (np.abs(g - exact) <= 2.0 ** -13 * (want["p"] + (np.arange(a) == groups[:, None])) / (n * T)).all()
    dx, dw, db = (v.download().astype(np.float64) for v in engine.linear_backward(ctx, ds, x, dw_))
    for got, left, right, length in ((dx, g, w64, a), (dw, g.T, dense, n), (db[None], np.ones((1, n)), g, n)):
        assert (np.abs(got - left @ right) <= (length + 2) * U * (np.abs(left) @ np.abs(right)) + 2.0 ** -140).all()
