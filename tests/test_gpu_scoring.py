"""The scoring operators on the device against plain float64 restatements: engine.linear, apply.log_probabilities and their
backward passes.

Tolerances count roundings.  u = 2^-24 is half a step of float32; an output in a narrower type adds half a step of that type
relative to its value (float16 2^-11, bfloat16 2^-8) and half of the smallest step it has."""
import math
import os
import subprocess
import sys

import numpy as np
import pytest

from snekmer_amd import _hip, apply, engine

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
TYPES = {"f32": np.float32, "f16": np.float16, "bf16": _hip.bfloat16}
HALF_STEP = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}
SMALLEST = {"f32": 2.0 ** -149, "f16": 2.0 ** -25, "bf16": 2.0 ** -134}


@pytest.fixture(scope="module")
def ctx():
    c = _hip.Context(0)
    yield c
    c.close()


def rounded(a, dt):
    """(device words, the float64 values they stand for)."""
    a = np.ascontiguousarray(a, dtype=np.float32)
    if dt == "bf16":
        w = _hip.to_bfloat16(a)
        return w, _hip.from_bfloat16(w).astype(np.float64)
    w = a.astype(TYPES[dt])
    return w, w.astype(np.float64)


def values(words, dt):
    return _hip.from_bfloat16(words).astype(np.float64) if dt == "bf16" else np.asarray(words).astype(np.float64)


def padded(ctx, words, pad, fill, lead=0):
    """The matrix inside longer rows (`pad` more columns, `lead` elements in front of the first): (interface object, whole)."""
    rows, cols = words.shape
    whole = np.full(lead + rows * (cols + pad), fill, dtype=words.dtype) if words.dtype != _hip.bfloat16 else \
        _hip.to_bfloat16(np.full(lead + rows * (cols + pad), fill, dtype=np.float32))
    inner = whole[lead:].reshape(rows, cols + pad)
    inner[:, :cols] = words
    d = ctx.to_device(whole)
    return Strided(d, (rows, cols), cols + pad, lead), d


class Strided:
    """A block of a DeviceArray's memory, as another library would name it."""

    def __init__(self, base, shape, ld, lead=0):
        size = base.dtype.itemsize
        typestr = "<V2" if base.dtype == _hip.bfloat16 else base.dtype.str
        self.base, self.shape = base, shape
        self.__cuda_array_interface = {"shape": shape, "typestr": typestr, "data": (base.ptr + lead * size, False), "strides": (ld * size, size), "version": 2}

    @property
    def __cuda_array_interface__(self):
        return self.__cuda_array_interface

    def download(self):
        size = self.base.dtype.itemsize
        lead = (self.__cuda_array_interface["data"][0] - self.base.ptr) // size
        ld = self.__cuda_array_interface["strides"][0] // size
        flat = self.base.download().ravel()
        rows, cols = self.shape
        return np.stack([flat[lead + i * ld:lead + i * ld + cols] for i in range(rows)]) if rows else flat[:0].reshape(0, cols)


# ---------------------------------------------------------------------------- log probabilities
def plain_logp(s, labels, k, T, mask=None):
    """From the definition in 64 bits; indices by a stable sort."""
    s = s.copy()
    if mask is not None:
        s[np.broadcast_to(mask, s.shape) == 0] = -np.inf
    n, a = s.shape
    out = {"logp": np.zeros(n), "entropy": np.zeros(n), "stats": np.full((n, 2), -np.inf), "top_index": np.full((n, k), -1), "top_logp": np.full((n, k), -np.inf),
           "spread": np.zeros((n, 3)), "p": np.zeros((n, a)), "z": np.full((n, a), -np.inf)}
    for i in range(n):
        allowed = s[i] > -np.inf
        if np.isnan(s[i]).any() or (s[i] == np.inf).any():
            for name in ("logp", "entropy", "stats", "top_logp"):
                out[name][i] = np.nan
            out["p"][i] = out["z"][i] = np.nan
            out["p"][i][s[i] == -np.inf] = 0.0
            if labels is not None and labels[i] == -1:
                out["logp"][i] = 0.0
            continue
        if not allowed.any():
            if labels is not None and labels[i] >= 0:
                out["logp"][i] = -np.inf
            continue
        m = s[i].max()
        with np.errstate(over="ignore"):
            d = (s[i] - m) / T
        e = np.where(d < 0, np.exp(d), 0.0)
        ties = int((d == 0).sum())
        l = math.log1p(e.sum() + ties - 1)
        z = d - l
        p = np.exp(z)
        live = p > 0
        out["stats"][i] = m, l
        out["p"][i], out["z"][i] = p, np.where(allowed, z, -np.inf)
        out["entropy"][i] = -(p[live] * z[live]).sum()
        out["spread"][i] = (p[live] * -d[live]).sum(), (p[live] * d[live] ** 2).sum(), l
        if labels is not None and labels[i] >= 0:
            out["logp"][i] = z[labels[i]] if allowed[labels[i]] else -np.inf
        order = np.argsort(-(s[i] + 0.0), kind="stable")[:k]
        order = order[s[i][order] > -np.inf]
        out["top_index"][i, :order.size] = order
        out["top_logp"][i, :order.size] = z[order]
    return out


def logp_bounds(want, cols, T):
    """Bounds on |l|, entropy and log p errors.  t = (s - m) * c2 has three roundings (difference, constant, product): 2^t is off by
    3u |d| + 2u relative; a lane adds 16 terms a tile, 6 levels of the wave and up to 16 + 64 states follow: a sum of positive terms
    is off by (16 tiles + 90) u relative; log1p by 2u.  Weighted by p these become the two moments of d in `spread`."""
    depth = 16 * math.ceil(cols / 1024) + 90
    ed, ed2, l = want["spread"].T
    on_l = U * (3 * ed + 2 + depth + 4 * l)
    on_h = on_l + U * (3 * ed2 + (8 + 2 * depth) * (ed + 0.01)) + 2 * U * want["entropy"] if want["entropy"].size else on_l
    return on_l, on_h


def check_logp(got, want, cols, T, k):
    on_l, on_h = logp_bounds(want, cols, T)
    assert np.array_equal(got["stats"][:, 0].astype(np.float64), want["stats"][:, 0], equal_nan=True)

    def near(a, b, bound):
        a = a.astype(np.float64)
        with np.errstate(over="ignore"):
            b = np.where(np.isinf(b.astype(np.float32)), b.astype(np.float32), b)  # what float32 cannot hold rounds to an infinity
        fine = np.isfinite(b)
        assert np.array_equal(np.isnan(a), np.isnan(b)) and np.array_equal(a[~fine], b[~fine], equal_nan=True)
        bound = np.broadcast_to(bound, b.shape)
        bad = np.abs(a[fine] - b[fine]) > bound[fine] + 2 * U * np.abs(b[fine])
        assert not bad.any(), (a[fine][bad][:4], b[fine][bad][:4], bound[fine][bad][:4])

    near(got["stats"][:, 1], want["stats"][:, 1], on_l)
    near(got["entropy"], want["entropy"], np.nan_to_num(on_h, posinf=0, neginf=0))
    if "logp" in got:
        near(got["logp"], want["logp"], on_l + 4 * U * np.abs(np.nan_to_num(want["logp"], neginf=0) + np.nan_to_num(want["stats"][:, 1], neginf=0)))
    if k:
        assert np.array_equal(got["top_index"], want["top_index"])
        l = np.nan_to_num(want["stats"][:, 1], neginf=0)[:, None]
        near(got["top_logp"], want["top_logp"], on_l[:, None] + 4 * U * np.abs(np.nan_to_num(want["top_logp"], neginf=0) + l))


def block(kind, n, a, seed):
    rng = np.random.default_rng(seed)
    if kind == "cosine":  # most families share no k-mer with a query: zeros, and ties among them
        s = np.where(rng.random((n, a)) < 0.9, 0.0, rng.random((n, a)))
        s[::5] = 0.0
        s[1::7] = np.round(s[1::7], 1)
    elif kind == "ascending":
        s = np.tile(np.linspace(-3, 3, a), (n, 1))
    elif kind == "peaked":  # one class holds nearly everything
        s = rng.normal(size=(n, a)) * 0.1
        s[np.arange(n), rng.integers(0, a, n)] += 12.0
    else:
        s = 3.0 * rng.normal(size=(n, a))
    return s


# one class to several tiles of 1024; one wave, four, sixteen, and several workgroups a row
SHAPES = [(1, 1), (3, 2), (5, 7), (2, 64), (7, 255), (4, 1000), (9, 1024), (3, 1025), (2, 2049), (5, 4097), (2, 16385), (1, 33001), (1, 70003)]


@pytest.mark.parametrize("kind", ["cosine", "normal", "ascending", "peaked"])
@pytest.mark.parametrize("dt", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("n, a", SHAPES)
def test_log_probabilities_by_shape(ctx, n, a, dt, kind):
    words, s = rounded(block(kind, n, a, n * 1000 + a), dt)
    labels = np.random.default_rng(a).integers(0, a, n)
    labels[n // 2 + 1::3] = -1
    k = [0, 1, 5, 16][(n + a) % 4]
    T = [1.0, 0.05, 0.7][a % 3]
    got = apply.log_probabilities(ctx, ctx.to_device(words), labels, k=k, temperature=T).host()
    check_logp(got, plain_logp(s, labels, k, T), a, T, k)


@pytest.mark.parametrize("n, a", [(4500, 40), (2500, 1000), (2100, 1500), (700, 3000)])
def test_log_probabilities_of_many_rows(ctx, n, a):
    words, s = rounded(block("cosine", n, a, 3), "f32")
    labels = np.random.default_rng(5).integers(-1, a, n)
    got = apply.log_probabilities(ctx, ctx.to_device(words), labels, k=10, temperature=0.1).host()
    check_logp(got, plain_logp(s, labels, 10, 0.1), a, 0.1, 10)


@pytest.mark.parametrize("dt", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("shared", [True, False])
@pytest.mark.parametrize("n, a", [(6, 9), (7, 1023), (5, 5000), (3, 40001)])
def test_masks_and_what_lies_under_them(ctx, n, a, shared, dt):
    rng = np.random.default_rng(a)
    words, s = rounded(block("normal", n, a, a), dt)
    mask = (rng.random(a if shared else (n, a)) < 0.6).astype(np.uint8) * rng.integers(1, 255, a if shared else (n, a)).astype(np.uint8)
    if not shared:
        mask[1] = 0          # nothing left
        mask[2] = 0
        mask[2, a - 1] = 1   # one class left, the last
    words, s = words.copy(), s.copy()
    hidden = np.broadcast_to(mask, (n, a)) == 0
    for j, bad in enumerate((np.nan, np.inf, -np.inf)):
        w, v = rounded(np.full(1, bad), dt)
        at = hidden & (rng.random((n, a)) < 0.2)
        words[at], s[at] = w[0], v[0]
    labels = rng.integers(0, a, n)
    d = ctx.to_device(words)
    dm = ctx.to_device(mask)
    fwd = apply.log_probabilities(ctx, d, labels, k=8, temperature=0.5, mask=dm)
    want = plain_logp(s, labels, 8, 0.5, mask)
    check_logp(fwd.host(), want, a, 0.5, 8)
    g = values(apply.log_probabilities_backward(ctx, d, labels, fwd, d_logp=ctx.to_device(np.ones(n, np.float32)), d_entropy=ctx.to_device(np.ones(n, np.float32)),
                                                temperature=0.5, mask=dm).download(), dt)
    assert (g[hidden] == 0).all() and np.isfinite(g).all()


@pytest.mark.parametrize("dt", ["f32", "f16", "bf16"])
def test_rows_without_a_distribution_and_scores_at_the_types_ends(ctx, dt):
    top = {"f32": np.finfo(np.float32).max, "f16": 65504.0, "bf16": 3.3895313892515355e38}[dt]
    rows = np.zeros((9, 1100), dtype=np.float32)
    rows[0, 1050] = np.nan
    rows[1, 3] = np.inf
    rows[2] = -np.inf
    rows[3] = -top            # every class at the lowest value: a uniform distribution
    rows[4] = -top
    rows[4, 7] = top          # the difference overflows: one class holds everything
    rows[5, :] = -np.inf
    rows[5, 1099] = 1.0
    rows[6, ::2] = -0.0       # equal to 0
    rows[7, 0] = np.nan
    rows[7, 1] = -np.inf
    rows[8, :5] = np.inf
    words, s = rounded(rows, dt)
    labels = np.array([2, 3, 0, 9, 7, 0, 1, -1, 4])
    d = ctx.to_device(words)
    for T in (1.0, 0.25):
        fwd = apply.log_probabilities(ctx, d, labels, k=4, temperature=T)
        want = plain_logp(s, labels, 4, T)
        want["spread"][4] = 0.0  # (one class: every sum is exact)
        check_logp(fwd.host(), want, 1100, T, 4)
        g = values(apply.log_probabilities_backward(ctx, d, labels, fwd, d_logp=ctx.to_device(np.ones(9, np.float32)), temperature=T).download(), dt)
        assert np.isnan(g[0]).all() and (g[2] == 0).all() and np.isnan(g[1]).all()
        assert np.isfinite(g[3:7]).all() and (g[4] == 0).all()
        # the label of row 5 is not allowed: the formula's (0 - p) is left, here at the one class that is
        assert (g[5, :1099] == 0).all() and g[5, 1099] == -1.0 / T
        assert g[7, 1] == 0 and np.isnan(g[7, 2:]).all()


@pytest.mark.parametrize("dt", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("pad, lead", [(0, 1), (1, 0), (3, 1), (24, 2)])
def test_rows_of_any_stride_and_alignment(ctx, dt, pad, lead):
    n, a = 6, 1403
    words, s = rounded(block("normal", n, a, pad), dt)
    view, _ = padded(ctx, words, pad, np.nan, lead)
    labels = np.arange(n) * 200
    fwd = apply.log_probabilities(ctx, view, labels, k=6)
    check_logp(fwd.host(), plain_logp(s, labels, 6, 1.0), a, 1.0, 6)
    out, whole = padded(ctx, words, pad, 77.0, lead)
    gl = ctx.to_device(np.linspace(-1, 1, n).astype(np.float32))
    apply.log_probabilities_backward(ctx, view, labels, fwd, d_logp=gl, out=out)
    again = apply.log_probabilities_backward(ctx, ctx.to_device(words), labels, fwd, d_logp=gl)
    assert np.array_equal(out.download().view(np.uint8), again.download().view(np.uint8))
    flat = values(whole.download(), dt)
    inner = flat[lead:].reshape(n, a + pad)
    assert (flat[:lead] == 77.0).all() and (inner[:, a:] == 77.0).all()  # what lies around the rows stays as it was


def test_columns_of_a_wider_block(ctx):
    words, s = rounded(block("cosine", 12, 104, 1), "f32")
    d = ctx.to_device(words)
    labels = np.arange(12)
    fwd = apply.log_probabilities(ctx, d, labels, k=3, ncols=101)
    check_logp(fwd.host(), plain_logp(s[:, :101], labels, 3, 1.0), 101, 1.0, 3)
    g = apply.log_probabilities_backward(ctx, d, labels, fwd, d_logp=ctx.to_device(np.ones(12, np.float32)), ncols=101, out=d)
    got = d.download()
    assert g is d and np.array_equal(got[:, 101:], words[:, 101:])
    assert np.allclose(got[:, :101].sum(axis=1), 0.0, atol=101 * 8 * U)  # a row's gradient of log p sums to nothing


def test_labels_of_both_widths_and_wrong_ones(ctx):
    words, s = rounded(block("normal", 5, 50, 2), "f32")
    d = ctx.to_device(words)
    labels = np.array([0, 49, -1, 7, 7])
    want = apply.log_probabilities(ctx, d, labels).host()["logp"]
    for t in (np.int32, np.int64):
        assert np.array_equal(apply.log_probabilities(ctx, d, ctx.to_device(labels.astype(t))).host()["logp"], want)
    for bad in (50, -2, 2 ** 40):
        wrong = ctx.to_device(np.array([0, 49, bad, 7, 7], dtype=np.int64))
        fwd = apply.log_probabilities(ctx, d, wrong)
        with pytest.raises(_hip.HipError, match="label outside"):
            ctx.sync()
        got = fwd.logp.download()
        assert np.isnan(got[2]) and np.array_equal(np.delete(got, 2), np.delete(want, 2))
        g = apply.log_probabilities_backward(ctx, d, wrong, fwd, d_logp=ctx.to_device(np.ones(5, np.float32)))
        with pytest.raises(_hip.HipError, match="label outside"):
            ctx.sync()
        got = g.download()
        assert np.isnan(got[2]).all() and np.isfinite(np.delete(got, 2, axis=0)).all()


def test_only_what_is_asked_for_and_no_rows(ctx):
    words, s = rounded(block("normal", 6, 300, 4), "bf16")
    d = ctx.to_device(words)
    want = plain_logp(s, None, 5, 1.0)
    only = apply.LogProbabilities(top_index=ctx.empty((6, 5), np.int32))
    assert apply.log_probabilities(ctx, d, k=5, out=only) is only
    assert np.array_equal(only.top_index.download(), want["top_index"]) and list(only.host()) == ["top_index"]
    none = apply.log_probabilities(ctx, ctx.empty((0, 300), np.float32), [], k=2).host()
    assert none["logp"].shape == (0,) and none["top_index"].shape == (0, 2)


def gradient_bound(want, s, labels, gl, gh, T, cols, dt):
    """p: the exponent has a difference, two constants, a product, l and one fma: 4u(|d| + l) + 4u relative, and the forward pass's l
    moves it by its own error; z + H and the sums around it: 6u of their terms; the whole is scaled and rounded three times."""
    on_l, on_h = logp_bounds(want, cols, T)
    z, p, l, h = want["z"], want["p"], want["stats"][:, 1:], want["entropy"][:, None]
    z0 = np.where(p > 0, z, 0.0)
    d = np.abs(z0 + l)
    rel = U * (4 * d + 4 * l + 8) + on_l[:, None]
    size = np.abs(gl)[:, None] + np.abs(gh)[:, None] * np.abs(z0 + h)
    b = p * (rel * size + np.abs(gh)[:, None] * (6 * U * (np.abs(z0) + l + h) + on_l[:, None] + on_h[:, None]) + 4 * U * size)
    known = labels >= 0
    at = np.flatnonzero(known), labels[known]
    b[at] += (8 * U + rel[at]) * np.abs(gl)[known]
    return b / T


def test_more_rows_than_one_launch_holds(ctx):
    """2^26 and some rows of two classes: a launch takes 2^26 of them.  Rows repeat with a period that no power of two divides."""
    n, period = (1 << 26) + 37, 1009
    rng = np.random.default_rng(6)
    w, s = rounded(rng.normal(size=(period, 2)), "bf16")
    labels = rng.integers(0, 2, period)
    times = n // period + 1
    out = apply.log_probabilities(ctx, ctx.to_device(np.tile(w, (times, 1))[:n]), ctx.to_device(np.tile(labels.astype(np.int32), times)[:n]), k=0)
    logp = out.logp.download()
    want = plain_logp(s, labels, 1, 1.0)["logp"]
    assert np.abs(logp[:period] - want).max() < 16 * U * (1 + np.abs(want).max())
    assert np.array_equal(logp, np.tile(logp[:period], times)[:n])


def test_the_longest_row(ctx):
    """2^31 - 1 equal classes: every one has the same log probability, the first ones are the best."""
    a = (1 << 31) - 1
    s = ctx.zeros((1, a), _hip.bfloat16)
    out = apply.log_probabilities(ctx, s, [a - 1], k=3).host()
    want = -math.log(a)
    assert np.array_equal(out["top_index"], [[0, 1, 2]])
    for got in (out["logp"], out["top_logp"], -out["entropy"]):
        assert np.abs(got - want).max() <= 8 * U * abs(want)


@pytest.mark.parametrize("dt", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("n, a, kind", [(1, 1, "normal"), (4, 5, "normal"), (6, 1000, "cosine"), (5, 2500, "peaked"), (2, 9000, "normal")])
def test_gradient_against_the_formula(ctx, n, a, kind, dt):
    words, s = rounded(block(kind, n, a, a + 7), dt)
    rng = np.random.default_rng(a)
    labels = rng.integers(0, a, n)
    if kind == "peaked":
        labels = s.argmax(axis=1)  # the label holds nearly all of the mass: 1 - p has to keep its digits
    if n > 3:
        labels[3] = -1
    T = 0.5
    gl, gh = rng.normal(size=n).astype(np.float32), rng.normal(size=n).astype(np.float32)
    d = ctx.to_device(words)
    fwd = apply.log_probabilities(ctx, d, labels, temperature=T)
    want = plain_logp(s, labels, 1, T)
    z, p, h = want["z"], want["p"], want["entropy"][:, None]
    for use_l, use_h in ((True, True), (True, False), (False, True)):
        a_l, a_h = gl.astype(np.float64) * use_l, gh.astype(np.float64) * use_h
        got = apply.log_probabilities_backward(ctx, d, labels, fwd, d_logp=ctx.to_device(gl) if use_l else None, d_entropy=ctx.to_device(gh) if use_h else None, temperature=T)
        known = labels >= 0
        a_l = np.where(known, a_l, 0.0)
        exact = -a_l[:, None] * p - a_h[:, None] * p * (z + h)
        at = np.flatnonzero(known), labels[known]
        exact[at] += a_l[known] * p[at] - a_l[known] * np.expm1(z[at])
        exact /= T
        bound = gradient_bound(want, s, labels, a_l, a_h, T, a, dt)
        err = np.abs(values(got.download(), dt) - exact)
        assert (err <= bound + HALF_STEP[dt] * np.abs(exact) * 1.01 + SMALLEST[dt] + 1e-37).all(), float((err - bound).max())


def test_gradient_against_differences(ctx):
    n, a, T = 4, 37, 0.8
    words, s = rounded(block("normal", n, a, 11), "f32")
    labels = np.array([3, -1, 0, 36])
    gl, gh = np.array([1.0, 0.5, -2.0, 0.7], np.float32), np.array([0.3, -1.0, 0.0, 2.0], np.float32)
    d = ctx.to_device(words)
    fwd = apply.log_probabilities(ctx, d, labels, temperature=T)
    got = apply.log_probabilities_backward(ctx, d, labels, fwd, d_logp=ctx.to_device(gl), d_entropy=ctx.to_device(gh), temperature=T).download()

    def total(x):
        w = plain_logp(x, labels, 1, T)
        return float((gl * w["logp"] + gh * w["entropy"]).sum())

    step = 1e-5
    for i, j in [(0, 3), (0, 4), (1, 0), (2, 0), (2, 9), (3, 36), (3, 1)]:
        up, down = s.copy(), s.copy()
        up[i, j] += step
        down[i, j] -= step
        # the third derivative is below 20 here: step^2 * 20 / 6, and 64-bit noise over the step
        assert abs(got[i, j] - (total(up) - total(down)) / (2 * step)) < 1e-9 + 1e-9 + 64 * U * 4


# ---------------------------------------------------------------------------- the matrix product
def act_plain(name, z):
    if name == "relu":
        return np.maximum(z, 0.0)
    if name == "gelu":
        return 0.5 * z * (1.0 + np.vectorize(math.erf)(z / math.sqrt(2.0)))
    if name == "gelu_tanh":
        return 0.5 * z * (1.0 + np.tanh(math.sqrt(2.0 / math.pi) * (z + 0.044715 * z ** 3)))
    if name == "silu":
        return z / (1.0 + np.exp(-z))
    if name == "sigmoid":
        return 1.0 / (1.0 + np.exp(-z))
    return z


def slope_plain(name, z):
    if name == "relu":
        return (z > 0).astype(np.float64)
    if name == "gelu":
        return 0.5 * (1.0 + np.vectorize(math.erf)(z / math.sqrt(2.0))) + z * np.exp(-0.5 * z * z) / math.sqrt(2.0 * math.pi)
    if name == "gelu_tanh":
        c = math.sqrt(2.0 / math.pi)
        t = np.tanh(c * (z + 0.044715 * z ** 3))
        return 0.5 * (1.0 + t) + 0.5 * z * (1.0 - t * t) * c * (1.0 + 3 * 0.044715 * z * z)
    g = 1.0 / (1.0 + np.exp(-z))
    if name == "silu":
        return g * (1.0 + z * (1.0 - g))
    if name == "sigmoid":
        return g * (1.0 - g)
    return np.ones_like(z)


def whole_numbers(shape, seed, most=4):
    return np.random.default_rng(seed).integers(-most, most + 1, shape).astype(np.float32)


def as_type(exact, dt):
    """Whole numbers below 2^24 are exact in float32: what an output of this type has to hold, bit for bit."""
    f = exact.astype(np.float32)
    assert (f == exact).all()
    with np.errstate(over="ignore"):
        return values(_hip.to_bfloat16(f) if dt == "bf16" else f.astype(TYPES[dt]), dt)


# one row to several tiles, sizes next to the tiles' and the contraction steps' ends, sums in parts (few tiles, long rows)
PRODUCTS = [(1, 1, 1), (1, 5, 3), (3, 1, 64), (2, 31, 33), (33, 65, 17), (17, 16, 127), (127, 129, 64), (128, 128, 128), (130, 260, 72), (1, 1000, 4096), (16, 100, 2048),
            (5, 300, 6561), (64, 7, 5000), (257, 511, 200), (300, 1000, 1031)]


@pytest.mark.parametrize("dt", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("m, n, k", PRODUCTS)
def test_products_of_whole_numbers_are_exact(ctx, m, n, k, dt):
    x, w, b, r = whole_numbers((m, k), 1), whole_numbers((n, k), 2), whole_numbers(n, 3, 20), whole_numbers((m, n), 4, 100)
    dx, dw, db, dr = (ctx.to_device(rounded(v, dt)[0]) for v in (x, w, b, r))
    z = x.astype(np.float64) @ w.T.astype(np.float64)
    assert np.array_equal(values(engine.linear(ctx, dx, dw).download(), dt), as_type(z, dt))
    y, pre = engine.linear(ctx, dx, dw, bias=db, activation="relu", residual=dr, preact=True)
    assert np.array_equal(values(pre.download(), dt), as_type(z + b, dt))
    assert np.array_equal(values(y.download(), dt), as_type(np.maximum(z + b, 0) + r, dt))


@pytest.mark.parametrize("dt", ["f32", "f16", "bf16"])
def test_a_chip_full_of_tiles_is_exact(ctx, dt):
    """Enough outputs for the largest tiles, and a contraction that ends inside a step."""
    x, w = whole_numbers((4100, 296), 1, 3), whole_numbers((4230, 296), 2, 3)
    y = engine.linear(ctx, ctx.to_device(rounded(x, dt)[0]), ctx.to_device(rounded(w, dt)[0]))
    assert np.array_equal(values(y.download(), dt), as_type((x @ w.T).astype(np.float64), dt))  # (below 2^24: exact in float32)


@pytest.mark.parametrize("dt", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("m, n, k", [(1, 1, 1), (2, 31, 33), (33, 65, 17), (130, 260, 72), (300, 70, 1031), (5, 300, 700), (1, 64, 2000), (1025, 40, 24)])
def test_gradients_of_whole_numbers_are_exact(ctx, m, n, k, dt):
    x, w, g = whole_numbers((m, k), 1), whole_numbers((n, k), 2), whole_numbers((m, n), 3)
    d = [ctx.to_device(rounded(v, dt)[0]) for v in (g, x, w)]
    dx, dw, db = engine.linear_backward(ctx, *d)
    g64, x64, w64 = (v.astype(np.float64) for v in (g, x, w))
    assert np.array_equal(values(dx.download(), dt), as_type(g64 @ w64, dt))
    assert np.array_equal(values(dw.download(), dt), as_type(g64.T @ x64, dt))
    assert np.array_equal(values(db.download(), dt), as_type(g64.sum(axis=0), dt))
    z = whole_numbers((m, n), 5)
    dx, dw, db = engine.linear_backward(ctx, *d, activation="relu", preact=ctx.to_device(rounded(z, dt)[0]))
    dz = g64 * (z > 0)
    assert np.array_equal(values(dx.download(), dt), as_type(dz @ w64, dt))
    assert np.array_equal(values(dw.download(), dt), as_type(dz.T @ x64, dt))
    assert np.array_equal(values(db.download(), dt), as_type(dz.sum(axis=0), dt))


@pytest.mark.parametrize("dt", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("name", ["none", "relu", "gelu", "gelu_tanh", "silu", "sigmoid"])
def test_activations_and_their_slopes(ctx, name, dt):
    """z comes from a product of one term (x z, w = 1), so it is exact; act and slope then have a few roundings of float32: the
    exponential's argument is below 2^5 in size (|z| + 2 roundings of it matter less than s (1 - s) |z| < 0.3), a sigmoid and two or three
    products: 2^-21 (1 + |z|) covers them, half a step of the type follows."""
    grid = np.concatenate([np.linspace(-9, 9, 399), [0.0, -0.0, 1e-6, -1e-6, 30.0, -30.0, 80.0, -80.0, 100.0, -100.0]])
    words, z = rounded(grid[:, None], dt)
    one = ctx.to_device(rounded(np.ones((1, 1)), dt)[0])
    y, pre = engine.linear(ctx, ctx.to_device(words), one, activation=name, preact=True)
    assert np.array_equal(values(pre.download(), dt), z)
    with np.errstate(over="ignore"):
        want, slope = act_plain(name, z), slope_plain(name, z)
    room = 2.0 ** -21 * (1 + np.minimum(np.abs(z), 10))
    assert (np.abs(values(y.download(), dt) - want) <= room + HALF_STEP[dt] * np.abs(want) * 1.01 + SMALLEST[dt]).all()
    g = ctx.to_device(rounded(np.ones_like(grid[:, None]), dt)[0])
    dx, _, _ = engine.linear_backward(ctx, g, None, one, activation=name, preact=pre, dw=None, dbias=None)
    # (dz is rounded once, the product with 1 is exact)
    assert (np.abs(values(dx.download(), dt) - slope) <= room + HALF_STEP[dt] * np.abs(slope) * 1.01 + SMALLEST[dt]).all()


@pytest.mark.parametrize("dt", ["f32", "f16", "bf16"])
def test_a_layer_of_ordinary_numbers(ctx, dt):
    """Sums of k products in float32: at most (k + 2) u sum |x w| off, whatever the order; the activation and the residual as above.
    Backward: dz is off by half a step of the type, the sums by (length + 2) u."""
    m, n, k = 200, 150, 333
    rng = np.random.default_rng(9)
    xw, x = rounded(rng.normal(size=(m, k)), dt)
    ww, w = rounded(rng.normal(size=(n, k)) / math.sqrt(k), dt)
    bw, b = rounded(rng.normal(size=n), dt)
    rw, r = rounded(rng.normal(size=(m, n)), dt)
    gw, g = rounded(rng.normal(size=(m, n)), dt)
    dxv, dwv, dbv, drv, dgv = (ctx.to_device(v) for v in (xw, ww, bw, rw, gw))
    h = HALF_STEP[dt]
    for name in ("silu", "gelu"):
        y, pre = engine.linear(ctx, dxv, dwv, bias=dbv, activation=name, residual=drv, preact=True)
        z = x @ w.T + b
        room = (k + 2) * U * (np.abs(x) @ np.abs(w).T + np.abs(b))
        zt = values(pre.download(), dt)
        assert (np.abs(zt - z) <= room + h * np.abs(z) * 1.01).all()
        want = act_plain(name, z) + r
        assert (np.abs(values(y.download(), dt) - want) <= 1.2 * room + 2.0 ** -20 * (1 + np.abs(z)) + h * np.abs(want) * 1.01).all()
        gx, gwt, gb = (values(v.download(), dt) for v in engine.linear_backward(ctx, dgv, dxv, dwv, activation=name, preact=pre))
        dz = g * slope_plain(name, zt)
        off = h * np.abs(dz) + 2.0 ** -21 * np.abs(g) * (1 + np.abs(zt))
        for got, a, ao, c, length in ((gx, dz, off, w, n), (gwt, dz.T, off.T, x, m)):
            exact = a @ c
            assert (np.abs(got - exact) <= ao @ np.abs(c) + (length + 2) * U * (np.abs(a) @ np.abs(c)) * 1.01 + h * np.abs(exact) * 1.01).all()
        exact = dz.sum(axis=0)
        assert (np.abs(gb - exact) <= (2.0 ** -21 * np.abs(g) * (1 + np.abs(zt)) + (m + 2) * U * np.abs(dz)).sum(axis=0) + h * np.abs(exact) * 1.01).all()


@pytest.mark.parametrize("dt", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("pad, lead", [(1, 0), (3, 1), (8, 0), (16, 1)])
def test_matrices_of_any_stride_and_alignment(ctx, dt, pad, lead):
    m, n, k = 70, 45, 136
    x, w, r, g = whole_numbers((m, k), 1), whole_numbers((n, k), 2), whole_numbers((m, n), 3), whole_numbers((m, n), 4)
    (xv, _), (wv, _), (rv, _), (gv, _) = (padded(ctx, rounded(v, dt)[0], pad, np.nan, lead) for v in (x, w, r, g))
    yv, whole = padded(ctx, rounded(np.zeros((m, n)), dt)[0], pad, 77.0, lead)
    zv, wholez = padded(ctx, rounded(np.zeros((m, n)), dt)[0], pad, 77.0, lead)
    engine.linear(ctx, xv, wv, residual=rv, preact=zv, out=yv)
    z = x.astype(np.float64) @ w.T
    assert np.array_equal(values(yv.download(), dt), as_type(z + r, dt)) and np.array_equal(values(zv.download(), dt), as_type(z, dt))
    for flat in (whole, wholez):
        flat = values(flat.download(), dt)
        assert (flat[:lead] == 77.0).all() and (flat[lead:].reshape(m, n + pad)[:, n:] == 77.0).all()
    dxv, wholex = padded(ctx, rounded(np.zeros((m, k)), dt)[0], pad, 77.0, lead)
    dwv, wholew = padded(ctx, rounded(np.zeros((n, k)), dt)[0], pad, 77.0, lead)
    engine.linear_backward(ctx, gv, xv, wv, activation="relu", preact=rv, dx=dxv, dw=dwv, dbias=False)
    dz = g * (r > 0)
    assert np.array_equal(values(dxv.download(), dt), as_type(dz.astype(np.float64) @ w, dt)) and np.array_equal(values(dwv.download(), dt), as_type(dz.T.astype(np.float64) @ x, dt))
    for flat, rows, cols in ((wholex, m, k), (wholew, n, k)):
        flat = values(flat.download(), dt)
        assert (flat[:lead] == 77.0).all() and (flat[lead:].reshape(rows, cols + pad)[:, cols:] == 77.0).all()


# outputs m x n, contraction k: together they take every tile, whole contractions and contractions in parts, for both widths of types
TILES = [(70, 74, 72), (70, 74, 2056), (8200, 72, 74), (2050, 1032, 130), (70, 2056, 4102), (1030, 4102, 72), (8200, 72, 4106), (2050, 2054, 522), (4096, 2048, 2080), (4094, 4096, 1034)]


@pytest.mark.parametrize("dt", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("m, n, k", TILES)
def test_every_tile_in_every_orientation(ctx, m, n, k, dt):
    """One product three times: forward, as a gradient of inputs (b across the contraction) and as a gradient of weights (both across)."""
    a, b = whole_numbers((m, k), 1, 2), whole_numbers((n, k), 2, 2)
    want = as_type(a @ b.T, dt)  # (sums below 2^24: exact in float32)
    da, db, dat, dbt = (ctx.to_device(rounded(v, dt)[0]) for v in (a, b, a.T, b.T))
    assert np.array_equal(values(engine.linear(ctx, da, db).download(), dt), want)
    dx, _, _ = engine.linear_backward(ctx, da, None, dbt, dw=None, dbias=None)
    assert np.array_equal(values(dx.download(), dt), want)
    _, dw, dbias = engine.linear_backward(ctx, dat, dbt, None, dx=None)
    assert np.array_equal(values(dw.download(), dt), want)
    assert np.array_equal(values(dbias.download(), dt), as_type(a.sum(axis=1, dtype=np.float64), dt))


@pytest.mark.parametrize("dt", ["f32", "bf16"])
def test_rows_that_lie_megabytes_apart(ctx, dt):
    """Rows 2^24 bytes apart and more, 300 of them: offsets inside a tile pass 32 bits.  Written and read back by products with the identity."""
    m, n, k = 300, 72, 88
    size = np.dtype(TYPES[dt]).itemsize
    ld = (1 << 24) // size + 8
    x, w, eye = whole_numbers((m, k), 1), whole_numbers((n, k), 2), np.eye(k, dtype=np.float32)
    g = whole_numbers((m, n), 3)
    dx, dw, dg, deye, deyen = (ctx.to_device(rounded(v, dt)[0]) for v in (x, w, g, eye, np.eye(n, dtype=np.float32)))
    far = ctx.empty(m * ld, TYPES[dt])
    xf, yf, gf = (Strided(far, (m, c), ld, lead) for c, lead in ((k, 0), (n, 4096), (n, 8192)))
    engine.linear(ctx, dx, deye, out=xf)
    engine.linear(ctx, dg, deyen, out=gf)
    engine.linear(ctx, xf, dw, residual=gf, out=yf)
    want = x @ w.T + g
    assert np.array_equal(values(engine.linear(ctx, yf, deyen).download(), dt), as_type(want, dt))
    gx, gw, gb = engine.linear_backward(ctx, gf, xf, dw)
    assert np.array_equal(values(gx.download(), dt), as_type(g @ w, dt))
    assert np.array_equal(values(gw.download(), dt), as_type(g.T @ x, dt))
    assert np.array_equal(values(gb.download(), dt), as_type(g.sum(axis=0), dt))
    # weights that far apart: few rows, many rows, and across the contraction
    engine.linear(ctx, dw, deye, out=Strided(far, (n, k), ld))
    wf = Strided(far, (n, k), ld)
    assert np.array_equal(values(engine.linear(ctx, dx, wf).download(), dt), as_type(x @ w.T, dt))
    few = ctx.to_device(rounded(x[:3], dt)[0])
    assert np.array_equal(values(engine.linear(ctx, few, wf).download(), dt), as_type(x[:3] @ w.T, dt))
    gx, _, _ = engine.linear_backward(ctx, dg, None, wf, dw=None, dbias=None)
    assert np.array_equal(values(gx.download(), dt), as_type(g @ w, dt))


def test_more_than_two_to_the_31_outputs(ctx):
    """66000 x 33000 outputs, looked at by columns and rows at the ends (a product with the identity copies them out)."""
    m, n, k = 66000, 33000, 8
    x, w = whole_numbers((m, k), 1), whole_numbers((n, k), 2)
    y = engine.linear(ctx, ctx.to_device(rounded(x, "bf16")[0]), ctx.to_device(rounded(w, "bf16")[0]))
    eye = ctx.to_device(rounded(np.eye(64, dtype=np.float32), "bf16")[0])
    for i, j in ((0, 0), (m - 5, 0), (0, n - 64), (m - 5, n - 64), (65100, 32768)):
        block = engine.linear(ctx, Strided(y, (5, 64), n, i * n + j), eye)
        assert np.array_equal(values(block.download(), "bf16"), as_type(x[i:i + 5] @ w[j:j + 64].T, "bf16"))


@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("name", ["none", "relu", "gelu", "gelu_tanh", "silu", "sigmoid"])
def test_slopes_far_from_zero(ctx, name, dt):
    """Past |z| = 2^7 every activation is a constant or the identity to float32: slopes of 0 or 1, also where z z is past the type's largest value."""
    z = np.array([[200.0], [-200.0], [1e10], [-1e10], [1e20], [-1e20], [2.0 ** 126], [-2.0 ** 126]], np.float32)
    one = rounded(np.ones((1, 1), np.float32), dt)[0]
    _, _, db = engine.linear_backward(ctx, *(ctx.to_device(v) for v in (rounded(np.ones((1, 8), np.float32), dt)[0],)), None, None, activation=name,
                                      preact=ctx.to_device(rounded(z.reshape(1, 8), dt)[0]), dx=None, dw=None)
    up = {"none": 1.0, "sigmoid": 0.0}.get(name, 1.0)
    down = 1.0 if name == "none" else 0.0
    assert np.array_equal(values(db.download(), dt), np.tile([up, down], 4))
    y = engine.linear(ctx, ctx.to_device(rounded(z, dt)[0]), ctx.to_device(one), activation=name).download()
    zt = rounded(z, dt)[1][:, 0]
    want = {"none": zt, "sigmoid": (zt > 0).astype(float)}.get(name, np.maximum(zt, 0))
    assert np.array_equal(values(y, dt)[:, 0], want)


def test_gelu_keeps_its_precision_in_the_tail(ctx):
    """z Phi(z) for z down to -12, relative to itself: the exponential's argument z z / 2 <= 72 has two roundings, 72 * 2^-23 in all; a
    dozen more of float32 around it: below 2^-16."""
    z = -np.linspace(0.5, 12.0, 301).astype(np.float32)
    one = ctx.to_device(np.ones((1, 1), np.float32))
    y = engine.linear(ctx, ctx.to_device(z[:, None]), one, activation="gelu").download()[:, 0].astype(np.float64)
    z = z.astype(np.float64)
    want = z * 0.5 * np.vectorize(math.erfc)(-z / math.sqrt(2.0))
    assert np.abs(y / want - 1).max() < 2.0 ** -16


def test_infinities_and_nan_stay_in_their_rows(ctx):
    x, w = whole_numbers((40, 90), 1), whole_numbers((50, 90), 2)
    w[w == 0] = 1
    x[7, 3], x[8, 5] = np.nan, np.inf
    y = engine.linear(ctx, ctx.to_device(x), ctx.to_device(w)).download()
    assert np.isnan(y[7]).all() and np.isinf(y[8]).all()
    rest = np.delete(np.arange(40), [7, 8])
    assert np.array_equal(y[rest].astype(np.float64), x[rest].astype(np.float64) @ w.T)


def test_empty_sizes(ctx):
    f = np.float32
    assert engine.linear(ctx, ctx.empty((0, 5), f), ctx.empty((4, 5), f)).shape == (0, 4)
    b = ctx.to_device(np.arange(4, dtype=f))
    y = engine.linear(ctx, ctx.empty((3, 0), f), ctx.empty((4, 0), f), bias=b, activation="relu").download()
    assert np.array_equal(y, np.tile(np.arange(4, dtype=f), (3, 1)))  # an empty sum
    dx, dw, db = engine.linear_backward(ctx, ctx.empty((0, 4), f), ctx.empty((0, 5), f), ctx.to_device(whole_numbers((4, 5), 1)))
    assert dx.shape == (0, 5) and (dw.download() == 0).all() and (db.download() == 0).all()
    dx, dw, db = engine.linear_backward(ctx, ctx.empty((3, 0), f), ctx.to_device(whole_numbers((3, 5), 1)), ctx.empty((0, 5), f))
    assert (dx.download() == 0).all() and dw.shape == (0, 5) and db.shape == (0,)


def test_memory_shared_between_arguments(ctx):
    x, w = ctx.to_device(whole_numbers((64, 64), 1)), ctx.to_device(whole_numbers((64, 64), 2))
    for bad in (dict(out=x), dict(out=w), dict(preact=x), dict(residual=x, out=Strided(x, (63, 64), 64, 64))):
        with pytest.raises((_hip.HipError, ValueError)):
            engine.linear(ctx, x, w, **bad)
    y = ctx.empty((64, 64), np.float32)
    with pytest.raises(_hip.HipError, match="share"):
        engine.linear(ctx, x, w, preact=y, out=y)
    with pytest.raises(_hip.HipError, match="shares memory"):
        engine.linear_backward(ctx, y, x, w, dx=y)
    same = ctx.empty((64, 64), np.float32)
    with pytest.raises(_hip.HipError, match="two gradients"):
        engine.linear_backward(ctx, y, x, w, dx=same, dw=same)
    # the residual itself may be the output, and column blocks of one matrix interleave
    r = ctx.to_device(whole_numbers((64, 64), 3))
    want = whole_numbers((64, 64), 1).astype(np.float64) @ whole_numbers((64, 64), 2).T + whole_numbers((64, 64), 3)
    engine.linear(ctx, x, w, residual=r, out=r)
    assert np.array_equal(r.download().astype(np.float64), want)
    both = ctx.to_device(np.concatenate([whole_numbers((64, 64), 1), np.zeros((64, 64), np.float32)], axis=1))
    engine.linear(ctx, Strided(both, (64, 64), 128), w, out=Strided(both, (64, 64), 128, 64))
    assert np.array_equal(both.download()[:, 64:].astype(np.float64), want - whole_numbers((64, 64), 3))
    s = ctx.to_device(whole_numbers((4, 100), 1))
    fwd = apply.log_probabilities(ctx, s, [0, 1, 2, 3])
    with pytest.raises(_hip.HipError, match="shares memory"):
        apply.log_probabilities_backward(ctx, Strided(s, (3, 100), 100), [0, 1, 2], apply.LogProbabilities(stats=ctx.to_device(fwd.stats.download()[:3])),
                                         d_logp=ctx.to_device(np.ones(3, np.float32)), out=Strided(s, (3, 100), 100, 100))


def test_log_probabilities_that_share_memory(ctx):
    s = ctx.to_device(whole_numbers((8, 100), 1))
    labels = ctx.to_device(np.arange(8, dtype=np.int32))
    row = ctx.empty(8, np.float32)
    for out in (dict(logp=row, entropy=row), dict(logp=Flat(s, 8, s.ptr + 160)), dict(logp=row, entropy=Flat(labels, 8, labels.ptr)), dict(stats=Strided(s, (8, 2), 2, 784), logp=row)):
        with pytest.raises(_hip.HipError, match="share"):
            apply.log_probabilities(ctx, s, labels, out=apply.LogProbabilities(**out))
    wider = ctx.to_device(np.zeros((8, 104), np.float32))  # the columns behind the scores are free to use
    out = Strided(wider, (8, 100), 104)
    fwd = apply.log_probabilities(ctx, s, labels)
    with pytest.raises(_hip.HipError, match="another input"):
        apply.log_probabilities_backward(ctx, s, labels, fwd, d_logp=Flat(wider, 8, wider.ptr), out=out)
    with pytest.raises(TypeError):
        apply.log_probabilities(ctx, s, labels, mask=[1] * 100)


class Flat:
    """n float32 values at an address inside a DeviceArray's memory."""

    def __init__(self, base, n, ptr):
        self.base, self.shape = base, (n,)
        self.interface = {"shape": (n,), "typestr": "<f4", "data": (ptr, False), "strides": None, "version": 2}

    @property
    def __cuda_array_interface__(self):
        return self.interface


# ---------------------------------------------------------------------------- streams, captures, other libraries' arrays
def test_beside_torch():
    """Contexts over torch's streams, torch's arrays, its captures: tests/torch_interop.py, in a process that loads torch first
    (loaded second, torch brings a HIP runtime of its own that finds no device)."""
    run = subprocess.run([sys.executable, "-u", os.path.join(os.path.dirname(__file__), "torch_interop.py")], capture_output=True, text=True, timeout=110)
    assert run.returncode == 0 and run.stdout.rstrip().endswith("all passed"), run.stdout + run.stderr


def test_a_recorded_step_replays(ctx):
    """Forward and backward of a head in one graph: every replay, with eager work and waits between, gives the eager result."""
    own = _hip.Context(0)
    m, n, k = 300, 130, 1031
    rng = np.random.default_rng(3)
    x, w = (own.to_device(rounded(rng.normal(size=s), "bf16")[0]) for s in ((m, k), (n, k)))
    labels = own.to_device(rng.integers(0, n, m).astype(np.int32))
    ones = own.to_device(np.ones(m, np.float32))
    y, pre, ds = (own.empty((m, n), _hip.bfloat16) for _ in range(3))
    dw = own.empty((n, k), _hip.bfloat16)
    out = apply.LogProbabilities(own.empty(m, np.float32), own.empty(m, np.float32), own.empty((m, 2), np.float32), own.empty((m, 3), np.int32), own.empty((m, 3), np.float32))

    def step():
        engine.linear(own, x, w, activation="gelu", preact=pre, out=y)
        apply.log_probabilities(own, y, labels, k=3, out=out)
        apply.log_probabilities_backward(own, y, labels, out, d_logp=ones, out=ds)
        engine.linear_backward(own, ds, x, w, activation="gelu", preact=pre, dx=None, dw=dw, dbias=None)

    def result():
        return [a.download().tobytes() for a in (y, out.logp, out.top_index, ds, dw)]

    step()
    step()
    own.graph_begin()
    step()
    graph = own.graph_end()
    other = rounded(rng.normal(size=(m, k)), "bf16")[0]
    first = x.download()
    for i in range(4):
        x.upload(first if i % 2 else other)
        graph.launch()
        own.sync()
        replayed = result()
        step()
        assert result() == replayed, i
    # two graphs of one context share its scratch: their replays follow each other on its stream
    own.graph_begin()
    engine.linear_backward(own, ds, x, w, activation="gelu", preact=pre, dx=None, dw=dw, dbias=None)
    second = own.graph_end()
    graph.launch()
    second.launch()
    assert result() == replayed
    graph.close()
    second.close()
    own.close()


def test_the_null_stream_is_not_captured():
    null = _hip.Context(0, stream=0)
    with pytest.raises(_hip.HipError, match="null stream"):
        null.graph_begin()
    null.close()


def test_results_do_not_change_from_call_to_call(ctx):
    rng = np.random.default_rng(0)
    x, w, g = (ctx.to_device(rounded(rng.normal(size=s), "bf16")[0]) for s in ((500, 3001), (90, 3001), (500, 90)))
    s = ctx.to_device(rng.normal(size=(3, 50000)).astype(np.float32))
    first = None
    for _ in range(3):
        got = [engine.linear(ctx, x, w).download().tobytes()] + [a.download().tobytes() for a in engine.linear_backward(ctx, g, x, w)]
        got += [a.tobytes() for a in apply.log_probabilities(ctx, s, [1, 2, 3], k=9).host().values()]
        first = first or got
        assert got == first


def test_two_threads_with_a_context_each():
    """Each thread's forward and backward give what they give alone (contexts share no scratch)."""
    import threading

    def work(own, seed, rounds):
        rng = np.random.default_rng(seed)
        x, w = (own.to_device(rounded(rng.normal(size=sh), "bf16")[0]) for sh in ((400, 2001), (150, 2001)))
        labels, ones = own.to_device(rng.integers(0, 150, 400).astype(np.int32)), own.to_device(np.ones(400, np.float32))
        got = []
        for _ in range(rounds):
            y, pre = engine.linear(own, x, w, activation="silu", preact=True)
            fwd = apply.log_probabilities(own, y, labels, k=4)
            ds = apply.log_probabilities_backward(own, y, labels, fwd, d_logp=ones)
            dx, dw, db = engine.linear_backward(own, ds, x, w, activation="silu", preact=pre)
            got.append([v.download().tobytes() for v in (y, fwd.logp, fwd.top_index, dx, dw, db)])
        return got

    contexts = [_hip.Context(0) for _ in range(2)]
    alone = [work(c, i, 1)[0] for i, c in enumerate(contexts)]
    results = [None, None]

    def thread(i):
        results[i] = work(contexts[i], i, 25)

    threads = [threading.Thread(target=thread, args=(i,)) for i in range(2)]
    for th in threads:
        th.start()
    for th in threads:
        th.join(60)
    for i in range(2):
        assert results[i] is not None and all(r == alone[i] for r in results[i])
        contexts[i].close()


# ---------------------------------------------------------------------------- as they are used together
def test_self_evaluation_of_learned_annotations(ctx):
    """learn_apply's materialised block read as a distribution: its best alternative is the prediction, its log probability of the
    sequence's own annotation agrees with the float64 softmax of the block."""
    from helpers import ensure_red6
    from snekmer_amd import alphabet
    from snekmer_amd.synth import synth_families

    ensure_red6()
    lut = alphabet.build_lut("red6")
    res, off, _ = synth_families(400, 120, family=20, seed=3)
    batch = engine.SeqBatch(ctx, res, off)
    csr = engine.count_csr(ctx, batch, lut, 8)
    basis = engine.build_basis(ctx, csr, lut.nsym, 8)
    groups = np.arange(400) // 20
    out = apply.learn_apply(ctx, csr, basis.ncols, groups, 20, materialize=True, basis=basis, alternatives=5, temperature=0.1)
    lp = out["log_probabilities"].host()
    block64 = out["scores"].download().reshape(-1, out["ld"])[:400, :20].astype(np.float64)
    check_logp(lp, plain_logp(block64, groups, 5, 0.1), 20, 0.1, 5)
    clear = block64.max(axis=1) - np.sort(block64, axis=1)[:, -2] > 1e-6  # (float32 block, float64 top-2)
    assert np.array_equal(lp["top_index"][clear, 0], out["top2_index"][clear, 0].astype(np.int32))


def test_a_head_over_kmer_counts_and_its_gradient(ctx):
    """Counts of a full basis -> linear head -> log probabilities of the annotations -> gradient of the mean loss with respect to the
    weights, against differences of the float64 loss."""
    rng = np.random.default_rng(1)
    n, k, a = 60, 81, 7
    counts = rng.poisson(0.5, size=(n, k)).astype(np.float32)
    weights = (rng.normal(size=(a, k)) / 9).astype(np.float32)
    bias = rng.normal(size=a).astype(np.float32)
    labels = rng.integers(0, a, n)
    x, w, b = ctx.to_device(counts), ctx.to_device(weights), ctx.to_device(bias)
    s = engine.linear(ctx, x, w, bias=b)
    fwd = apply.log_probabilities(ctx, s, labels, k=2)
    ds = apply.log_probabilities_backward(ctx, s, labels, fwd, d_logp=ctx.to_device(np.full(n, -1.0 / n, np.float32)))
    dx, dw, db = (v.download() for v in engine.linear_backward(ctx, ds, x, w))

    def loss(wt, bs):
        z = counts.astype(np.float64) @ wt.T + bs
        return -plain_logp(z, labels, 1, 1.0)["logp"].mean()

    w64, b64, h = weights.astype(np.float64), bias.astype(np.float64), 1e-5
    for i, j in [(0, 0), (3, 40), (6, 80)]:
        up, down = w64.copy(), w64.copy()
        up[i, j] += h
        down[i, j] -= h
        # float32 scores of up to 81 terms: p is off by about 100 u, counts are below 6; h^2 times a third derivative below 6^3
        assert abs(dw[i, j] - (loss(up, b64) - loss(down, b64)) / (2 * h)) < 100 * U * 6 + 6 ** 3 * h * h + 1e-9
    for i in (0, 6):
        up, down = b64.copy(), b64.copy()
        up[i] += h
        down[i] -= h
        assert abs(db[i] - (loss(w64, up) - loss(w64, down)) / (2 * h)) < 100 * U + h * h + 1e-9
    assert np.abs(db.sum()) < 1e-6 and dx.shape == (n, k)
