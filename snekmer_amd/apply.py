"""apply: the counts -> family totals -> cosine -> top-2 chain of ``snekmer learn`` / ``snekmer apply``
on the device, and the log probabilities of annotations under such scores.

Reference code replaced (all per sequence / per basis k-mer in Python + pandas):
  per-annotation sums of count rows      snekmer/rules/learn.smk:385-408
  cosine_similarity(totals, counts).T    snekmer/rules/apply.smk:278-289, rules/learn.smk:811-829
  top-2 scores, prediction, delta        snekmer/rules/apply.smk:312-328, rules/learn.smk:831-849

The CSV/confidence-table bookkeeping around these steps stays with the caller.
"""
import ctypes as C
from typing import Optional, Sequence, Tuple

import numpy as np

from . import _hip, engine

_p = C.c_void_p
_i64 = C.c_int64


class ColumnTotals:
    """The family-total matrix by column (skm_group_postings): colptr uint32[ncols+1], post uint64 = family | total << 32
    (families ascending inside a column), normsq uint64[families] (exact squared norms of the total rows).  The layout
    skm_apply_top2 reads; `group_sum` hangs it on the CSR it returns so that `apply_top2` does not sort the totals again."""

    def __init__(self, n, ncols, nnz, colptr, post, normsq):
        self.n, self.ncols, self.nnz, self.colptr, self.post, self.normsq = n, ncols, nnz, colptr, post, normsq


def group_totals(ctx, csr: engine.CountsCSR, groups: Sequence[int], ngroups: int, basis=None, ncols: Optional[int] = None) -> ColumnTotals:
    """Per-annotation sums of the count rows (snekmer/rules/learn.smk:385-408) BY COLUMN.  `basis`: the engine.Basis of
    `csr` with its postings (engine.build_basis / the vectorize stage leave the count matrix by column: no sort is needed
    then); without it the CSR is transposed first (skm_csr_transpose; `ncols` or one look at the column ids)."""
    if csr.colidx is None:
        raise ValueError("group_sum needs column ids: call engine.build_basis first")
    if getattr(csr, "elided", False):
        raise ValueError("group_sum needs real column ids: build the basis without elide_singletons "
                         "(0xFFFFFFFF marks k-mers of one row only and is not a column)")
    g = np.ascontiguousarray(groups, dtype=np.uint32)
    if g.size != csr.n:
        raise ValueError("one group id per row is required")
    if g.size and int(g.max()) >= ngroups:
        raise ValueError("group id out of range")
    d_g = ctx.to_device(g if g.size else np.zeros(1, np.uint32))
    nnz = csr.nnz
    if basis is not None and basis.colptr is not None and basis.post is not None and basis.post_bits == 64:
        ncols, colptr, post = basis.ncols, basis.colptr, basis.post
    else:
        if ncols is None:
            if basis is not None:
                ncols = basis.ncols
            else:
                ncols = (int(csr.colidx.download(nnz).max()) + 1) if nnz else 0
        colptr, post = engine.transpose(ctx, csr.n, nnz, ncols, csr.rowptr, csr.colidx, csr.counts)
    out_colptr = ctx.empty(ncols + 1, np.uint32)
    out_post = ctx.empty(max(nnz, 1), np.uint64)
    normsq = ctx.empty(max(ngroups, 1), np.uint64)
    got = _i64(0)
    ctx.call("skm_group_postings", _i64(csr.n), _i64(ncols), _p(colptr.ptr), _p(post.ptr), _i64(nnz), _p(d_g.ptr), _i64(ngroups),
             _p(out_colptr.ptr), _p(out_post.ptr), _p(normsq.ptr), _p(None), C.byref(got))
    return ColumnTotals(ngroups, ncols, int(got.value), out_colptr, out_post, normsq)


def group_sum(ctx, csr: engine.CountsCSR, groups: Sequence[int], ngroups: int, basis=None, ncols: Optional[int] = None) -> engine.CountsCSR:
    """Sum the count rows of each group.  `csr.colidx` must be set (engine.build_basis); the
    result is a CountsCSR over the same column space whose `colidx` (ascending per row) and
    `counts` are filled and whose `codes` are unused.  Its `columns` attribute holds the same totals by column
    (ColumnTotals), which `apply_top2` uses as they are.  `basis` (with postings): see `group_totals`."""
    cols = group_totals(ctx, csr, groups, ngroups, basis=basis, ncols=ncols)
    cap = max(cols.nnz, 1)
    out = engine.CountsCSR(ctx, ngroups, cols.nnz, 32, ctx.empty(ngroups + 1, np.int64), ctx.empty(1, np.uint32),
                           ctx.empty(cap, np.uint32), None)
    out.colidx = ctx.empty(cap, np.uint32)
    ctx.call("skm_postings_to_csr", _i64(cols.ncols), _i64(cols.nnz), _p(cols.colptr.ptr), _p(cols.post.ptr), _i64(ngroups),
             _p(out.rowptr.ptr), _p(out.colidx.ptr), _p(out.counts.ptr))
    out.columns = cols
    return out


def cosine_rows_vs_totals(ctx, csr: engine.CountsCSR, ncols: int, totals: engine.CountsCSR, mode: int = 0):
    """cosine_similarity(totals, counts).T of the reference: float32 [csr.n x totals.n] on the
    device, both operands over the same `ncols` columns."""
    if getattr(csr, "elided", False) or getattr(totals, "elided", False):
        raise ValueError("rectangular cosine needs real column ids on both sides (no elide_singletons)")
    xr = engine.row_norms(ctx, csr.n, csr.rowptr, csr.counts)
    yr = engine.row_norms(ctx, totals.n, totals.rowptr, totals.counts)
    colptr, post = engine.transpose(ctx, totals.n, totals.nnz, ncols, totals.rowptr, totals.colidx, totals.counts)
    ld = (totals.n + 3) // 4 * 4
    return engine.cosine_matrix(ctx, csr, xr, totals.n, ncols, colptr, post, yr, mode=mode, ld=ld), ld


def row_top2(ctx, scores, n: int, m: int, ld: int) -> Tuple[np.ndarray, np.ndarray]:
    """(indices [n,2] uint32, values [n,2] float32): np.argsort(-S, axis=1)[:, :2] and the scores
    there, ties towards the lower column."""
    idx = ctx.empty(max(2 * n, 1), np.uint32)
    val = ctx.empty(max(2 * n, 1), np.float32)
    ctx.call("skm_row_top2", _i64(n), _i64(m), _p(scores.ptr), _i64(ld), _p(idx.ptr), _p(val.ptr))
    return idx.download(2 * n).reshape(n, 2), val.download(2 * n).reshape(n, 2)


def apply_top2(ctx, csr: engine.CountsCSR, ncols: int, totals: engine.CountsCSR,
               row0: int = 0, row1: Optional[int] = None, order: Optional[Sequence[int]] = None):
    """The apply epilogue fused with the cosine (skm_apply_top2): for every query row the two
    best-scoring rows of `totals`, without materialising the N x A score block of
    rules/apply.smk:282-289.  Returns (idx uint32[rows,2], score float64[rows,2], dot int64[rows,2]);
    scores are formed in float64 from the exact integer dot products and squared norms, so
    ``round(score[:,0] - score[:,1], 2)`` is the reference's ``delta`` (apply.smk:320-325).
    `order`: a permutation of the rows [0, row1 - row0) in which to PROCESS them (results stay in row order): rows that
    share k-mers next to each other - e.g. ``np.argsort(labels, kind="stable")`` in learn.smk's self-evaluation - make the
    kernel's one random access per entry hit in L2."""
    row1 = csr.n if row1 is None else row1
    rows = row1 - row0
    d_order = None
    if order is not None:
        order = np.ascontiguousarray(order, dtype=np.uint32)
        if order.size != rows or (rows and not (np.sort(order) == np.arange(rows, dtype=np.uint32)).all()):
            raise ValueError("order must be a permutation of the rows")
        d_order = ctx.to_device(order if rows else np.zeros(1, np.uint32))
    if getattr(csr, "elided", False) or getattr(totals, "elided", False):
        raise ValueError("apply_top2 needs real column ids on both sides (no elide_singletons)")
    xsq = engine.row_normsq(ctx, csr.n, csr.rowptr, csr.counts)
    cols = totals if isinstance(totals, ColumnTotals) else getattr(totals, "columns", None)
    if cols is not None and cols.ncols == ncols:  # the totals by column already (group_sum / group_totals): nothing to sort
        colptr, post, ysq, m = cols.colptr, cols.post, cols.normsq, cols.n
    else:
        ysq = engine.row_normsq(ctx, totals.n, totals.rowptr, totals.counts)
        colptr, post = engine.transpose(ctx, totals.n, totals.nnz, ncols, totals.rowptr, totals.colidx, totals.counts)
        m = totals.n
    idx = ctx.empty(max(2 * rows, 1), np.uint32)
    score = ctx.empty(max(2 * rows, 1), np.float64)
    dot = ctx.empty(max(2 * rows, 1), np.int64)
    ctx.call("skm_apply_top2", _i64(csr.n), _p(csr.rowptr.ptr), _p(csr.colidx.ptr), _p(csr.counts.ptr), _p(xsq.ptr),
             _i64(m), _i64(ncols), _p(colptr.ptr), _p(post.ptr), _p(ysq.ptr), _i64(row0), _i64(row1),
             _p(d_order.ptr if d_order is not None else None), _p(idx.ptr), _p(score.ptr), _p(dot.ptr))
    return (idx.download(2 * rows).reshape(rows, 2), score.download(2 * rows).reshape(rows, 2),
            dot.download(2 * rows).reshape(rows, 2))


class LogProbabilities:
    """What `log_probabilities` computes, as device arrays (float32; top_index int32), one row per score row: `logp` [n] of the
    given labels, `entropy` [n] in nats, `stats` [n, 2] (largest allowed score m, l with log p(j) = (score_j - m) / T - l; the
    backward pass reads them), `top_index` / `top_logp` [n, k] of the best classes.  Members that are None are not computed."""

    __slots__ = ("logp", "entropy", "stats", "top_index", "top_logp")

    def __init__(self, logp=None, entropy=None, stats=None, top_index=None, top_logp=None):
        self.logp, self.entropy, self.stats, self.top_index, self.top_logp = logp, entropy, stats, top_index, top_logp

    def host(self) -> dict:
        """The members that are DeviceArrays, as numpy arrays by name."""
        got = {name: getattr(self, name) for name in self.__slots__}
        return {name: a.download() for name, a in got.items() if isinstance(a, _hip.DeviceArray)}


_LABEL_TYPES = {"<i4": 32, "<i8": 64}
MAX_ALTERNATIVES = 16


def _score_arguments(ctx, scores, labels, mask, ncols, temperature):
    """The arguments that both passes share, checked: (dtype code, rows, cols, scores, ld, mask, ldmask, labels, label_bits)
    and what has to live until the call has been queued."""
    sp, (rows, cols), ld, t = _hip.array_view(ctx, scores, "scores", 2, _hip.FLOAT_TYPES)
    if ncols is not None:
        if not 0 < int(ncols) <= cols:
            raise ValueError(f"ncols: {ncols} of {cols} columns")
        cols = int(ncols)
    if cols < 1:
        raise ValueError("scores: no classes")
    if not 1e-30 < float(temperature) < 1e30:  # (what the library takes: 1 / T and log2(e) / T stay ordinary float32 numbers)
        raise ValueError(f"temperature: {temperature} (want a positive number between 1e-30 and 1e30)")
    mp, ldmask = None, 0
    if mask is not None:
        two = len(getattr(mask, "shape", ())) == 2
        mp, ms, ldmask, _ = _hip.array_view(ctx, mask, "mask", 2 if two else 1, ("|u1", "|b1"))
        engine._expect("mask", ms, (rows, cols) if two else (cols,))
        ldmask = ldmask if two else 0
    lp, bits, keep = None, 32, None
    if labels is not None:
        if not _hip.is_device_array(labels):
            host = np.asarray(labels)
            if host.dtype.kind not in "iu" and host.size:
                raise TypeError(f"labels: {host.dtype} (want integers)")
            if host.size and (host.min() < -1 or host.max() >= cols):
                raise ValueError(f"labels: outside -1 .. {cols - 1}")
            labels = keep = ctx.to_device(host.astype(np.int32).reshape(host.shape))
        lp, ls, _, lt = _hip.array_view(ctx, labels, "labels", 1, _LABEL_TYPES)
        engine._expect("labels", ls, (rows,))
        bits = _LABEL_TYPES[lt]
    return (_hip.FLOAT_TYPES[t], rows, cols, sp, ld, mp, ldmask, lp, bits), keep


def _packed(ctx, x, name, shape, types, writable=False):
    """Pointer of an array of this shape whose elements all lie next to each other, None for None."""
    if x is None:
        return None
    ptr, got, ld, _ = _hip.array_view(ctx, x, name, len(shape), types, writable=writable)
    engine._expect(name, got, shape)
    if len(shape) == 2 and ld != shape[1]:
        raise ValueError(f"{name}: rows must lie next to each other")
    return ptr


def log_probabilities(ctx, scores, labels=None, k: int = 0, temperature: float = 1.0, mask=None, ncols: Optional[int] = None,
                      out: Optional[LogProbabilities] = None) -> LogProbabilities:
    """softmax(scores / temperature) by rows, of a score block resident on the device (skm_log_probabilities): the log
    probability of each row's given label, the entropy, and the k best classes, ties towards the lower column as in
    `row_top2`.  What `learn_apply(materialize=True)` / `cosine_rows_vs_totals` / `engine.linear` produce, read as a
    distribution over annotations: where the reference maps the difference of the two best scores to a confidence
    (snekmer/rules/apply.smk:320-326), this says how likely each annotation is under the scores.

    `scores` [n, ld] float32, float16 or `_hip.bfloat16`, of which the first `ncols` columns count (default: all); `labels` [n]:
    class ids on the device (int32 / int64) or on the host, -1 where none is known (log probability 0); `mask`: uint8 or bool
    on the device, 0 where a class may not be chosen, [ncols] for all rows or [n, ncols]; a score of -infinity is a class that
    may not be chosen either.  `temperature`: between 1e-30 and 1e30.  `k` <= 16 alternatives, padded with (-1, -inf).  A row that allows nothing has entropy 0 and
    log probability -inf; one that allows a NaN or +inf is NaN throughout, with indices -1.  A label on the device outside
    [-1, ncols) gives NaN and is reported by the next Context.sync / download.  `out`: a LogProbabilities whose members are
    filled; only those it has are computed.  All arrays may be this library's or another one's (`_hip.array_view`: used in the
    order of `ctx`'s stream, which their owners have to respect)."""
    args, keep = _score_arguments(ctx, scores, labels, mask, ncols, temperature)
    rows = args[1]
    k = int(k)
    if not 0 <= k <= MAX_ALTERNATIVES:
        raise ValueError(f"k: {k} alternatives (0 to {MAX_ALTERNATIVES})")
    if out is None:
        out = LogProbabilities(ctx.empty(rows, np.float32) if labels is not None else None, ctx.empty(rows, np.float32), ctx.empty((rows, 2), np.float32),
                               ctx.empty((rows, k), np.int32) if k else None, ctx.empty((rows, k), np.float32) if k else None)
    if out.logp is not None and labels is None:
        raise ValueError("labels: log probabilities need them")
    if not k and (out.top_index is not None or out.top_logp is not None):
        raise ValueError("k: the alternatives' arrays are given, but k is 0")
    f32 = ("<f4",)
    ctx.call("skm_log_probabilities", *args, k, float(temperature), _packed(ctx, out.logp, "logp", (rows,), f32, True),
             _packed(ctx, out.entropy, "entropy", (rows,), f32, True), _packed(ctx, out.stats, "stats", (rows, 2), f32, True),
             _packed(ctx, out.top_index, "top_index", (rows, k), ("<i4",), True), _packed(ctx, out.top_logp, "top_logp", (rows, k), f32, True))
    return out


def log_probabilities_backward(ctx, scores, labels, forward: LogProbabilities, d_logp=None, d_entropy=None, temperature: float = 1.0, mask=None,
                               ncols: Optional[int] = None, out=None):
    """Gradient of ``(d_logp * logp + d_entropy * entropy).sum()`` with respect to the scores, in their type
    (skm_log_probabilities_backward).  `forward`: what `log_probabilities` left for the same scores, labels, mask and
    temperature (`stats`, and `entropy` if `d_entropy` is given).  Classes that may not be chosen get 0; columns of `out`
    behind `ncols` are left as they are.  `out` may be `scores` itself.  Alternatives carry no gradient.  Other libraries' arrays as in
    `log_probabilities`."""
    args, keep = _score_arguments(ctx, scores, labels, mask, ncols, temperature)
    code, rows, cols = args[:3]
    if d_logp is None and d_entropy is None:
        raise ValueError("d_logp, d_entropy: one of them is needed")
    if d_logp is not None and labels is None:
        raise ValueError("labels: the gradient of the log probabilities needs them")
    if forward.stats is None or (d_entropy is not None and forward.entropy is None):
        raise ValueError("forward: stats (and entropy, for d_entropy) are needed")
    f32 = ("<f4",)
    if out is None:
        out = ctx.empty((rows, cols), _hip.float_dtype(code))
    gp, gs, ldg, _ = _hip.array_view(ctx, out, "out", 2, tuple(t for t, c in _hip.FLOAT_TYPES.items() if c == code), writable=True)
    if gs[0] != rows or gs[1] < cols or (ncols is None and gs[1] != cols):
        raise ValueError(f"out: shape {tuple(gs)}, want {(rows, cols)}")
    ctx.call("skm_log_probabilities_backward", *args, float(temperature), _packed(ctx, forward.stats, "stats", (rows, 2), f32),
             _packed(ctx, forward.entropy, "entropy", (rows,), f32), _packed(ctx, d_logp, "d_logp", (rows,), f32),
             _packed(ctx, d_entropy, "d_entropy", (rows,), f32), gp, ldg)
    return out


def confidence_lookup(delta: np.ndarray, table) -> np.ndarray:
    """``vals["delta"].map(global_confidence_scores)`` of rules/apply.smk:325-326: the confidence of
    every (already rounded) delta from the global confidence table, NaN where the table has no such
    key.  `table` is a mapping or a pandas Series {delta value -> confidence}; keys match by float
    equality, exactly as ``Series.map`` does."""
    if hasattr(table, "to_dict"):
        table = table.to_dict()
    keys = {float(k): float(v) for k, v in dict(table).items()}
    return np.asarray([keys.get(float(d), np.nan) for d in np.asarray(delta, dtype=np.float64)], dtype=np.float64)


def predict(ctx, csr: engine.CountsCSR, ncols: int, totals: engine.CountsCSR, labels: Optional[Sequence] = None,
            confidence=None):
    """rules/apply.smk:312-328 for a batch: Prediction (label of the best family), Score (its cosine),
    delta = round(top1 - top2, 2) and, given the global confidence table, Confidence."""
    idx, score, dot = apply_top2(ctx, csr, ncols, totals)
    top, second = score[:, 0], score[:, 1]
    delta = np.round(top - second, 2)
    out = {"top2_index": idx, "top2_score": score, "top2_dot": dot, "Score": top, "delta": delta}
    if labels is not None:
        lab = np.asarray(labels, dtype=object)
        out["Prediction"] = np.asarray([str(lab[i]) for i in idx[:, 0]], dtype=object)
    if confidence is not None:
        out["Confidence"] = confidence_lookup(delta, confidence)
    return out


def learn_apply(ctx, csr: engine.CountsCSR, ncols: int, groups: Sequence[int], ngroups: int, materialize: bool = False, basis=None,
                alternatives: Optional[int] = None, temperature: float = 1.0):
    """Self-evaluation chain of rules/learn.smk: totals per annotation, cosine of every sequence
    against every annotation, top-2 and delta (rounded to 2 decimals as learn.smk:842/apply.smk:325).
    The N x A score block is only produced when `materialize` is set (the save_apply_associations
    branch of apply.smk:298-301 writes it out).  With `alternatives` (0 to 16; needs the block) the block is also read as a
    distribution over the annotations: out["log_probabilities"] is `log_probabilities` of every sequence's own annotation
    with that many best alternatives at `temperature`."""
    if alternatives is not None and not materialize:
        raise ValueError("alternatives: only read from the materialised block (materialize=True)")
    totals = group_sum(ctx, csr, groups, ngroups, basis=basis, ncols=ncols)
    # rows of one annotation next to each other: they share their family's k-mers (see apply_top2)
    idx, score, dot = apply_top2(ctx, csr, ncols, totals, order=np.argsort(np.asarray(groups), kind="stable"))
    out = {"totals": totals, "top2_index": idx, "top2_score": score, "top2_dot": dot,
           "delta": np.round(score[:, 0] - score[:, 1], 2)}
    if materialize:
        out["scores"], out["ld"] = cosine_rows_vs_totals(ctx, csr, ncols, totals)
        if alternatives is not None:
            out["log_probabilities"] = log_probabilities(ctx, out["scores"], groups, k=alternatives, temperature=temperature, ncols=ngroups)
    return out
