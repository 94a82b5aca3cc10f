"""The measured cases of the scoring operators: the matrix product with its epilogue (engine.linear and its backward pass) and
the log probabilities of given labels with entropy and best alternatives (apply.log_probabilities and its backward pass).

A case is a dict of plain values; `prepare` makes its inputs, `run` makes one pass: with `own` false in elementary torch
operations in 32 bits, with `own` true through the framework's entry points."""
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZES = {"f32": 4, "f16": 2, "bf16": 2}
ACTIVATIONS = ("none", "relu", "gelu", "gelu_tanh", "silu", "sigmoid")
_contexts = {}


def _logp(name, rows, cols, dtype, k, kind, mask="none", temperature=1.0, pad=0):
    return {"name": name, "op": "logp", "rows": rows, "cols": cols, "dtype": dtype, "k": k, "kind": kind, "mask": mask,
            "temperature": temperature, "pad": pad}


def _logp_grad(name, rows, cols, dtype, kind, mask="none", temperature=1.0, pad=0):
    return {"name": name, "op": "logp_grad", "rows": rows, "cols": cols, "dtype": dtype, "kind": kind, "mask": mask,
            "temperature": temperature, "pad": pad}


def _linear(name, m, k, n, dtype, kind, activation="none", residual=False, preact=False, pad=0):
    return {"name": name, "op": "linear", "m": m, "k": k, "n": n, "dtype": dtype, "kind": kind, "activation": activation,
            "residual": residual, "preact": preact, "pad": pad}


def _linear_grad(name, m, k, n, dtype, kind, activation="none", pad=0):
    return {"name": name, "op": "linear_grad", "m": m, "k": k, "n": n, "dtype": dtype, "kind": kind, "activation": activation, "pad": pad}


def listed():
    return [
        # one sequence against 1 000 annotations, as a service answers it: latency
        _logp("logp one query", 1, 1000, "f32", 5, "cosine", temperature=0.05),
        # the materialised score block of the learn / apply chain: 100 000 queries against 1 000 annotation totals
        _logp("logp apply block", 100000, 1000, "f32", 10, "cosine", temperature=0.05),
        # few queries against very many classes, a mask a row (classes that the query may not take), rows of odd length
        _logp("logp long masked rows", 129, 200003, "bf16", 16, "normal", mask="rows"),
        # the gradient of the same block, for fitting a temperature or a head in front of it
        _logp_grad("grad apply block", 100000, 1000, "f32", "cosine", temperature=0.05),
        # a training step's scores over many classes, some of them switched off for every row
        _logp_grad("grad many classes", 2047, 50001, "bf16", "normal", mask="shared"),
        # one query's features through a scoring head: latency and the weights' bandwidth
        _linear("linear one query", 1, 4096, 1000, "bf16", "normal"),
        # a proteome's k-mer counts (3 383 proteins, solvacc k=8: 3^8 columns) against 1 000 annotations
        _linear("linear proteome counts", 3383, 6561, 1000, "bf16", "counts"),
        # a large batch over the whole hydro k=14 basis (2^14 columns)
        _linear("linear whole basis", 32768, 16384, 1000, "bf16", "counts", activation="sigmoid"),
        # a hidden layer as training runs it: activation, residual, the pre-activation kept for the backward pass
        _linear("linear hidden layer", 8192, 4096, 4096, "bf16", "normal", activation="silu", residual=True, preact=True),
        # the same head on 32-bit features
        _linear("linear f32 counts", 10000, 6561, 1000, "f32", "counts", activation="relu"),
        # the hidden layer's backward pass
        _linear_grad("lgrad hidden layer", 8192, 4096, 4096, "bf16", "normal", activation="silu"),
        # the backward pass of the head over the proteome's counts
        _linear_grad("lgrad proteome counts", 3383, 6561, 1000, "f16", "counts"),
    ]


def _spread(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(("logp", "logp_grad", "linear", "linear", "linear_grad"))
    dtype = rng.choice(("f32", "f16", "bf16", "bf16"))
    pad = rng.choice((0, 0, 1, 3, 8))
    if op in ("logp", "logp_grad"):
        cols = _spread(rng, 2, 200000)
        rows = _spread(rng, 1, max(1, min(100000, 50000000 // cols)))
        c = {"op": op, "rows": rows, "cols": cols, "dtype": dtype, "kind": rng.choice(("cosine", "normal")),
             "mask": rng.choice(("none", "none", "shared", "rows")), "temperature": round(rng.uniform(0.05, 2.0), 3), "pad": pad}
        if op == "logp":
            c["k"] = rng.choice((0, 1, 2, 5, 10, 16))
        return c
    m, k, n = _spread(rng, 1, 20000), _spread(rng, 16, 12000), _spread(rng, 1, 4096)
    while m * k * n > 1 << 36:
        m = m // 2 + 1
    c = {"op": op, "m": m, "k": k, "n": n, "dtype": dtype, "kind": rng.choice(("counts", "normal")), "activation": rng.choice(ACTIVATIONS), "pad": pad}
    if op == "linear":
        c["residual"], c["preact"] = rng.random() < 0.5, rng.random() < 0.5
    return c


# ---------------------------------------------------------------------------- inputs
def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _matrix(rows, cols, pad, dtype, fill):
    """[rows, cols] inside rows of cols + pad values; what lies behind a row's end is not the operator's to read."""
    whole = torch.empty(rows, cols + pad, dtype=dtype, device="cuda")
    whole[:, :cols] = fill
    if pad:
        whole[:, cols:] = math.nan
    return whole[:, :cols]


def _scores(case, g):
    rows, cols = case["rows"], case["cols"]
    if case["kind"] == "cosine":  # most families share no k-mer with a query: exact zeros, some weak scores, a few strong ones
        u = torch.rand(rows, cols, generator=g, device="cuda")
        v = torch.rand(rows, cols, generator=g, device="cuda")
        s = torch.where(u < 0.9, torch.zeros_like(v), torch.where(u < 0.99, 0.1 * v, v))
    else:
        s = 3.0 * torch.randn(rows, cols, generator=g, device="cuda")
    return _matrix(rows, cols, case["pad"], DTYPES[case["dtype"]], s)


def _prepare_scores(case, g):
    rows, cols = case["rows"], case["cols"]
    state = {"case": case, "scores": _scores(case, g)}
    labels = torch.randint(0, cols, (rows,), generator=g, device="cuda", dtype=torch.int32)
    labels[rows // 2 + 1 :: 97] = -1  # sequences without a known annotation
    state["labels"] = labels
    state["mask"] = None
    if case["mask"] != "none":
        shape = (cols,) if case["mask"] == "shared" else (rows, cols)
        mask = (torch.rand(shape, generator=g, device="cuda") < 0.8).to(torch.uint8)
        if case["mask"] == "rows":
            mask[rows // 3 + 1 :: 61] = 0  # rows whose mask leaves nothing
        state["mask"] = mask
    return state


def _prepare_features(case, g):
    m, k, n, dtype = case["m"], case["k"], case["n"], DTYPES[case["dtype"]]
    if case["kind"] == "counts":  # k-mer counts: small whole numbers, most of them zero
        x = torch.floor(-1.2 * torch.log(torch.rand(m, k, generator=g, device="cuda").clamp_min(1e-7)) * (torch.rand(m, k, generator=g, device="cuda") < 0.3))
    else:
        x = torch.randn(m, k, generator=g, device="cuda")
    state = {"case": case, "x": _matrix(m, k, case["pad"], dtype, x)}
    state["w"] = (torch.randn(n, k, generator=g, device="cuda") / math.sqrt(k)).to(dtype)
    state["bias"] = (0.5 * torch.randn(n, generator=g, device="cuda")).to(dtype)
    return state


def prepare(case, seed):
    g = _generator(seed)
    if case["op"] == "logp":
        state = _prepare_scores(case, g)
        rows, k = case["rows"], case["k"]
        state["out"] = {name: torch.empty(shape, dtype=t, device="cuda") for name, shape, t in (
            ("logp", (rows,), torch.float32), ("entropy", (rows,), torch.float32), ("stats", (rows, 2), torch.float32),
            ("top_index", (rows, k), torch.int32), ("top_logp", (rows, k), torch.float32)) if k or not name.startswith("top")}
        return state
    if case["op"] == "logp_grad":
        state = _prepare_scores(case, g)
        z, m, ls = _log_softmax(state, torch.float64)  # what the forward pass left
        state["stats"] = torch.stack([m, ls], dim=1).float()
        state["entropy"] = _entropy(z).float()
        state["d_logp"] = torch.randn(case["rows"], generator=g, device="cuda")
        state["d_entropy"] = 0.1 * torch.randn(case["rows"], generator=g, device="cuda")
        state["out"] = torch.empty(case["rows"], case["cols"], dtype=DTYPES[case["dtype"]], device="cuda")
        return state
    state = _prepare_features(case, g)
    m, k, n, dtype = case["m"], case["k"], case["n"], DTYPES[case["dtype"]]
    if case["op"] == "linear":
        state["residual"] = torch.randn(m, n, generator=g, device="cuda").to(dtype) if case["residual"] else None
        state["out"] = torch.empty(m, n, dtype=dtype, device="cuda")
        state["preact"] = torch.empty(m, n, dtype=dtype, device="cuda") if case["preact"] else None
        return state
    state["preact"] = torch.randn(m, n, generator=g, device="cuda").to(dtype) if case["activation"] != "none" else None
    state["dy"] = torch.randn(m, n, generator=g, device="cuda").to(dtype)
    state["dx"] = torch.empty(m, k, dtype=dtype, device="cuda")
    state["dw"] = torch.empty(n, k, dtype=dtype, device="cuda")
    state["dbias"] = torch.empty(n, dtype=dtype, device="cuda")
    return state


# ---------------------------------------------------------------------------- plain forms
def _log_softmax(state, kind):
    """(log probabilities, row maxima, logs of the sums of exp((s - max) / T)) of the classes that the mask leaves."""
    s = state["scores"].to(kind)
    if state["mask"] is not None:
        s = torch.where(state["mask"].bool(), s, -math.inf)
    m = s.amax(dim=1)
    d = (s - torch.where(m > -math.inf, m, 0.0)[:, None]) / state["case"]["temperature"]
    ties = (d == 0.0).sum(dim=1)  # the largest entries count one each: log1p keeps what a sum next to 1 would lose
    ls = torch.log1p(torch.where(d < 0.0, torch.exp(d), 0.0).sum(dim=1) + (ties - 1))
    z = torch.where(d > -math.inf, d - torch.where(ls > -math.inf, ls, 0.0)[:, None], -math.inf)
    return z, m, ls


def _entropy(z):
    return -torch.where(z > -math.inf, torch.exp(z) * z, 0.0).sum(dim=1)


def _plain_logp(state):
    case, labels = state["case"], state["labels"].long()
    z, m, ls = _log_softmax(state, torch.float32)
    logp = z.gather(1, labels.clamp_min(0)[:, None])[:, 0]
    out = {"logp": torch.where(labels < 0, 0.0, logp), "entropy": _entropy(z), "stats": torch.stack([m, ls], dim=1)}
    k = case["k"]
    if k:
        s = state["scores"].float()
        if state["mask"] is not None:
            s = torch.where(state["mask"].bool(), s, -math.inf)
        value, index = torch.sort(s, dim=1, descending=True, stable=True)  # ties go to the lowest class
        value, index = value[:, :k], index[:, :k]
        gone = k - value.shape[1]
        if gone > 0:
            value = torch.nn.functional.pad(value, (0, gone), value=-math.inf)
            index = torch.nn.functional.pad(index, (0, gone))
        there = value > -math.inf
        out["top_index"] = torch.where(there, index, -1).to(torch.int32)
        out["top_logp"] = torch.where(there, z.gather(1, index), -math.inf)
    return out


def _plain_logp_grad(state):
    case, labels = state["case"], state["labels"].long()
    s, stats, t = state["scores"].float(), state["stats"], case["temperature"]
    z = (s - stats[:, :1]) / t - stats[:, 1:]
    p = torch.exp(z)
    gl = torch.where(labels < 0, 0.0, state["d_logp"])[:, None]
    d = -gl * p - state["d_entropy"][:, None] * p * (z + state["entropy"][:, None])
    at = labels.clamp_min(0)[:, None]
    d.scatter_add_(1, at, gl * torch.where(labels[:, None] < 0, 0.0, p.gather(1, at) - torch.expm1(z.gather(1, at))))
    if state["mask"] is not None:
        d = torch.where(state["mask"].bool(), d, 0.0)
    return (d / t).to(s.dtype if case["dtype"] == "f32" else DTYPES[case["dtype"]])


def _act(name, z):
    if name == "relu":
        return z.clamp_min(0.0)
    if name == "gelu":
        return 0.5 * z * (1.0 + torch.erf(z * math.sqrt(0.5)))
    if name == "gelu_tanh":
        return 0.5 * z * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (z + 0.044715 * z * z * z)))
    if name == "silu":
        return z / (1.0 + torch.exp(-z))
    if name == "sigmoid":
        return 1.0 / (1.0 + torch.exp(-z))
    return z


def _act_slope(name, z):
    if name == "relu":
        return (z > 0.0).to(z.dtype)
    if name == "gelu":
        return 0.5 * (1.0 + torch.erf(z * math.sqrt(0.5))) + z * torch.exp(-0.5 * z * z) * (1.0 / math.sqrt(2.0 * math.pi))
    if name == "gelu_tanh":
        c = math.sqrt(2.0 / math.pi)
        t = torch.tanh(c * (z + 0.044715 * z * z * z))
        return 0.5 * (1.0 + t) + 0.5 * z * (1.0 - t * t) * c * (1.0 + 3.0 * 0.044715 * z * z)
    if name == "silu":
        g = 1.0 / (1.0 + torch.exp(-z))
        return g * (1.0 + z * (1.0 - g))
    if name == "sigmoid":
        g = 1.0 / (1.0 + torch.exp(-z))
        return g * (1.0 - g)
    return torch.ones_like(z)


def _plain_linear(state, kind=torch.float32):
    case = state["case"]
    dtype = DTYPES[case["dtype"]] if kind == torch.float32 else kind
    z = state["x"].to(kind) @ state["w"].to(kind).t() + state["bias"].to(kind)
    y = _act(case["activation"], z)
    if state["residual"] is not None:
        y = y + state["residual"].to(kind)
    return {"y": y.to(dtype), "preact": z.to(dtype)} if case["preact"] else {"y": y.to(dtype)}


def _plain_linear_grad(state, kind=torch.float32):
    case = state["case"]
    dtype = DTYPES[case["dtype"]] if kind == torch.float32 else kind
    dz = state["dy"].to(kind)
    if state["preact"] is not None:
        dz = dz * _act_slope(case["activation"], state["preact"].to(kind))
    return {"dx": (dz @ state["w"].to(kind)).to(dtype), "dw": (dz.t() @ state["x"].to(kind)).to(dtype), "dbias": dz.sum(dim=0).to(dtype)}


# ---------------------------------------------------------------------------- one pass
def _own_run(state):
    """The framework's calls, on a context over torch's current stream, into the caller's arrays."""
    from snekmer_amd import _hip, apply, engine

    device = torch.cuda.current_device()
    where = device, torch._C._cuda_getCurrentRawStream(device)  # (torch.cuda.current_stream().cuda_stream: 2.8 us instead of 0.1)
    context = _contexts.get(where)
    if context is None:
        context = _contexts[where] = _hip.Context(where[0], stream=where[1])
    case = state["case"]
    if case["op"] == "logp":
        out = apply.LogProbabilities(**state["out"])
        apply.log_probabilities(context, state["scores"], state["labels"], k=case["k"], temperature=case["temperature"], mask=state["mask"], out=out)
        return state["out"]
    if case["op"] == "logp_grad":
        forward = apply.LogProbabilities(stats=state["stats"], entropy=state["entropy"])
        apply.log_probabilities_backward(context, state["scores"], state["labels"], forward, d_logp=state["d_logp"], d_entropy=state["d_entropy"],
                                         temperature=case["temperature"], mask=state["mask"], out=state["out"])
        return state["out"]
    if case["op"] == "linear":
        engine.linear(context, state["x"], state["w"], bias=state["bias"], activation=case["activation"], residual=state["residual"],
                      preact=state["preact"], out=state["out"])
        return {"y": state["out"], "preact": state["preact"]} if case["preact"] else {"y": state["out"]}
    engine.linear_backward(context, state["dy"], state["x"], state["w"], activation=case["activation"], preact=state["preact"],
                           dx=state["dx"], dw=state["dw"], dbias=state["dbias"])
    return {"dx": state["dx"], "dw": state["dw"], "dbias": state["dbias"]}


def run(state):
    if own:
        return _own_run(state)
    return {"logp": _plain_logp, "logp_grad": _plain_logp_grad, "linear": _plain_linear, "linear_grad": _plain_linear_grad}[state["case"]["op"]](state)


# ---------------------------------------------------------------------------- the definition in 64 bits
def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] in ("linear", "linear_grad"):
        return (_plain_linear if case["op"] == "linear" else _plain_linear_grad)(state, torch.float64)
    s = state["scores"].double()
    if state["mask"] is not None:
        s = s.masked_fill(state["mask"] == 0, -math.inf)
    t, labels = case["temperature"], state["labels"].long()
    empty = (s == -math.inf).all(dim=1)
    z = torch.log_softmax(s / t, dim=1)
    z[empty] = -math.inf
    p = torch.softmax(s / t, dim=1)
    p[empty] = 0.0
    entropy = torch.special.entr(p).sum(dim=1)
    known = labels >= 0
    at = labels.clamp_min(0)[:, None]
    if case["op"] == "logp":
        top = s.amax(dim=1)
        out = {"logp": torch.where(known, z.gather(1, at)[:, 0], 0.0), "entropy": entropy,
               "stats": torch.stack([top, torch.where(empty, -math.inf, torch.logsumexp(s / t, dim=1) - top / t)], dim=1)}
        if case["k"]:
            best = torch.topk(z, min(case["k"], case["cols"]), dim=1).values
            out["top_index"] = None
            out["top_logp"] = torch.nn.functional.pad(best, (0, case["k"] - best.shape[1]), value=-math.inf)
        return out
    picked = torch.zeros_like(p).scatter_(1, at, known.double()[:, None])
    gl = torch.where(known, state["d_logp"].double(), 0.0)[:, None]
    ge = state["d_entropy"].double()[:, None]
    logs = torch.where(p > 0, z, 0.0)
    d = gl * (picked - p) - ge * p * (logs + entropy[:, None])
    return d.masked_fill(s == -math.inf, 0.0) / t


# ---------------------------------------------------------------------------- what a pass cannot do without
def work(case):
    e = SIZES[case["dtype"]]
    if case["op"] in ("logp", "logp_grad"):
        cells = case["rows"] * case["cols"]
        masks = {"none": 0, "shared": case["cols"], "rows": cells}[case["mask"]]
        if case["op"] == "logp":
            return {"bytes": cells * e + masks + case["rows"] * (4 + 16 + 8 * case["k"]), "flops": 8.0 * cells}
        return {"bytes": 2 * cells * e + masks + case["rows"] * 24, "flops": 9.0 * cells}
    m, k, n = case["m"], case["k"], case["n"]
    if case["op"] == "linear":
        return {"bytes": e * (m * k + n * k + n + m * n * (1 + case["residual"] + case["preact"])), "flops": 2.0 * m * n * k}
    return {"bytes": e * (2 * m * k + 2 * n * k + n + m * n * (1 + (case["activation"] != "none"))), "flops": 4.0 * m * n * k}
