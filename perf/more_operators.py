"""Performance cases of gated feed-forward blocks, the norms and gates between blocks, and log probabilities of
given classes, as a program that uses this framework calls them.

A case is a dict of

  op       "gated"  y = D^T (act(G^T x + g0) * (U^T x + u0)) + d0 over columns x [n_in, batch]; the products take
                    operands of the model's type, so what one product hands to the next is rounded to it
           "norm"   state = residual + scale * gate * after(x) and before(state): what stands between two blocks
           "logp"   the log probability of each column's given class from logits [classes, batch], the entropy,
                    the logarithm of the normaliser, and the top_k classes with their log probabilities
  train    the gradients of all inputs and parameters too
  dtype    "f32", "f16", "bf16": type of the arrays; norms' weights, a gate of one value per feature and log
           probabilities are 32 bits
  batch    columns
  widths   gated: "n_in-hidden-n_out"; act; bias: with biases
  n        norm: features; after, before: "none", "rms" or "layer"; gate: "none", "feature" or "full";
           residual; scale
  classes, top_k, masked    logp: share of the logits that are -inf

`run` computes an operator in its plain form (elementary torch operations in 32 bits), or where `own` is
true through the framework's entry points.
"""
from __future__ import annotations

import math

import torch

own = False

TORCH = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"f32": 4, "f16": 2, "bf16": 2}
EPS = 1e-5
IGNORED = -1  # the class of a column that has none


def listed():
    return [
        # Serving one sample: the block's weights from memory, and the launches.
        {"name": "gated_one", "op": "gated", "train": False, "dtype": "bf16", "widths": "1024-4096-1024", "act": "silu",
         "bias": False, "batch": 1},
        # Serving a handful of samples together.
        {"name": "gated_few", "op": "gated", "train": False, "dtype": "f16", "widths": "2048-4096-2048", "act": "gelu",
         "bias": False, "batch": 20},
        # Training an fp32 emulator of odd widths, with biases, on an odd number of columns.
        {"name": "gated_train_odd", "op": "gated", "train": True, "dtype": "f32", "widths": "333-1001-77", "act": "tanh",
         "bias": True, "batch": 5_003},
        # A training step's block: three products forward, six backward.
        {"name": "gated_train", "op": "gated", "train": True, "dtype": "bf16", "widths": "1024-4096-1024", "act": "silu",
         "bias": False, "batch": 16_384},
        # A large batch through a wide block: matrix cores.
        {"name": "gated_wide", "op": "gated", "train": False, "dtype": "f16", "widths": "2048-8192-2048", "act": "silu",
         "bias": False, "batch": 32_768},
        # Between two blocks while one sample is served: latency counts.
        {"name": "norm_one", "op": "norm", "train": False, "dtype": "bf16", "n": 4096, "after": "rms", "before": "rms",
         "gate": "none", "residual": True, "scale": 1.0, "batch": 1},
        # Between two blocks of a large batch, a learnt gate for each feature.
        {"name": "norm_batch", "op": "norm", "train": False, "dtype": "bf16", "n": 1024, "after": "rms", "before": "rms",
         "gate": "feature", "residual": True, "scale": 0.5, "batch": 65_536},
        # Training with a gate for each feature of each column (a conditioned network), odd sizes, fp32.
        {"name": "norm_train_odd", "op": "norm", "train": True, "dtype": "f32", "n": 333, "after": "layer",
         "before": "layer", "gate": "full", "residual": True, "scale": 0.7, "batch": 40_003},
        # Training wide blocks: only the norm before the next block.
        {"name": "norm_train_wide", "op": "norm", "train": True, "dtype": "f16", "n": 4096, "after": "none",
         "before": "rms", "gate": "none", "residual": True, "scale": 1.0, "batch": 16_384},
        # One sample's log probabilities over a large set of classes, with alternatives.
        {"name": "logp_one", "op": "logp", "train": False, "dtype": "bf16", "classes": 131_072, "top_k": 8,
         "masked": 0.0, "batch": 1},
        # The ten classes of the benchmark's branched classifier over its whole batch.
        {"name": "logp_cells", "op": "logp", "train": False, "dtype": "f32", "classes": 10, "top_k": 3, "masked": 0.1,
         "batch": 4_194_304},
        # The loss of a training step and its gradient over many classes.
        {"name": "logp_train", "op": "logp", "train": True, "dtype": "bf16", "classes": 65_536, "top_k": 0,
         "masked": 0.02, "batch": 4_096},
    ]


ACTS = ("relu", "leaky_relu", "silu", "gelu", "tanh", "sigmoid")


def draw(rng):
    """A case of one of the listed kinds with other sizes and types."""

    def log_int(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(max(hi, lo))))))

    case = {"op": rng.choice(("gated", "gated", "norm", "logp")), "train": rng.random() < 0.4,
            "dtype": rng.choice(("f32", "f16", "bf16"))}
    if case["op"] == "gated":
        case["widths"] = f"{log_int(16, 4096)}-{log_int(16, 8192)}-{log_int(16, 4096)}"
        case["act"], case["bias"] = rng.choice(ACTS), rng.random() < 0.5
        # Batches within the largest listed case's cost: products and the states between them.
        products = (2e12 if case["train"] else 3e12) / (10 if case["dtype"] == "f32" else 1)
        case["batch"] = log_int(1, max(2, min(1_000_000, products / _gated_flops(case), 6e8 / sum(_widths(case)))))
    elif case["op"] == "norm":
        case["n"] = log_int(16, 8192)  # (of fewer, what a layer norm leaves of a gradient is its roundings)
        case["after"], case["before"] = rng.choice(("none", "rms", "layer")), rng.choice(("none", "rms", "rms", "layer"))
        case["gate"], case["residual"] = rng.choice(("none", "feature", "full")), rng.random() < 0.8
        case["scale"] = rng.choice((1.0, 0.5, 1.7))
        case["batch"] = log_int(1, max(2, min(1_000_000, 1e8 / case["n"])))
    else:
        case["classes"] = log_int(1, 200_000)
        case["top_k"] = rng.randint(0, min(8, case["classes"]))
        case["masked"] = rng.choice((0.0, 0.02, 0.5))
        case["batch"] = log_int(1, max(2, min(4_000_000, 2e8 / case["classes"])))
    return case


# -- inputs ------------------------------------------------------------------------------------


def _widths(case):
    return [int(w) for w in case["widths"].split("-")]


def _gated_flops(case):
    """Of one column."""
    i, h, o = _widths(case)
    return 2.0 * (2 * i + o) * h * (3 if case["train"] else 1)


def _inputs(case, seed):
    g = torch.Generator(device="cuda").manual_seed(1 + seed)
    t, b = TORCH[case["dtype"]], case["batch"]

    def normal(*shape):
        return torch.randn(shape, device="cuda", generator=g)

    s = {}
    if case["op"] == "gated":
        i, h, o = _widths(case)

        def weights(n_in, n_out):  # Glorot-uniform
            return ((torch.rand((n_in, n_out), device="cuda", generator=g) * 2 - 1) * math.sqrt(6 / (n_in + n_out))).to(t)

        s["gate"], s["up"], s["down"] = weights(i, h), weights(i, h), weights(h, o)
        s["biases"] = [(0.1 * normal(n)).to(t) for n in (h, h, o)] if case["bias"] else [None] * 3
        s["x"] = normal(i, b).to(t)
        if case["train"]:
            s["dy"] = normal(o, b).to(t)
    elif case["op"] == "norm":
        n = case["n"]
        for k in ("after", "before"):
            s[k] = None if case[k] == "none" else (1 + 0.2 * normal(n), 0.1 * normal(n) if case[k] == "layer" else None)
        # Features of different sizes, columns off centre.
        s["x"] = (normal(n, b) * torch.exp(0.5 * normal(n, 1)) + 0.3 * normal(1, b)).to(t)
        s["residual"] = (normal(n, b) * 2 + 0.5).to(t) if case["residual"] else None
        s["gate"] = {"none": None, "feature": 0.1 * normal(n) + 0.5}.get(case["gate"]) if case["gate"] != "full" else \
            (0.3 * normal(n, b)).to(t)
        if case["train"]:
            s["d_state"] = normal(n, b).to(t)
            s["d_normed"] = None if case["before"] == "none" else normal(n, b).to(t)
    else:
        c = case["classes"]
        x = 2 * normal(c, b) + normal(c, 1)
        s["targets"] = torch.randint(0, c, (b,), device="cuda", generator=g, dtype=torch.int32)
        if case["masked"]:
            off = torch.rand((c, b), device="cuda", generator=g) < case["masked"]
            off.scatter_(0, s["targets"][None].long(), False)  # a given class is allowed
            x = x.masked_fill(off, -math.inf)
        s["logits"] = x.to(t)
        if b > 3:  # columns without a class, as padding has
            s["targets"][torch.rand(b, device="cuda", generator=g) < 0.1] = IGNORED
        if case["train"]:
            s["d_log_probs"], s["d_entropy"], s["d_log_normalizer"] = -1 + 0.1 * normal(b), 0.01 * normal(b), 0.001 * normal(b)
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    s["case"] = case
    if own and case["op"] != "logp":
        s["model"] = _model(case, s)
    return s


def _model(case, s):
    import ponni_amd as P

    if case["op"] == "norm":
        def norm(k):
            return None if s[k] is None else P.BlockNorm(case[k], *s[k], eps=EPS)

        return P.create_residual_norm(case["n"], after=norm("after"), before=norm("before"), scale=case["scale"],
                                      dtype=case["dtype"])
    h = _widths(case)[1]
    act = {"relu": P.Relu, "leaky_relu": lambda n: P.LeakyRelu(n, 0.1), "tanh": P.Tanh, "sigmoid": P.Sigmoid,
           "silu": P.Silu, "gelu": lambda n: P.Gelu(n, True)}[case["act"]](h)
    g0, u0, d0 = s["biases"]
    return P.create_gated_model(s["gate"], s["up"], s["down"], act, gate_bias=g0, up_bias=u0, down_bias=d0)


# -- one pass ------------------------------------------------------------------------------------


def run(state):
    case = state["case"]
    if own:
        return _run_own(case, state)
    return {"gated": _gated, "norm": _norm, "logp": _logp}[case["op"]](case, state)


def _run_own(case, s):
    import ponni_amd as P

    if case["op"] == "gated":
        if not case["train"]:
            return {"y": s["model"].forward_batch_parallel(s["x"])}
        y, states = s["model"].forward_with_states(s["x"])
        d = s["model"].backward(s["x"], states, s["dy"])
        return _present(y=y, d_x=d.x, d_gate=d.gate, d_up=d.up, d_down=d.down, d_gate_bias=d.gate_bias,
                        d_up_bias=d.up_bias, d_down_bias=d.down_bias)
    if case["op"] == "norm":
        if not case["train"]:
            state, normed = s["model"].forward_batch_parallel(s["x"], s["residual"], s["gate"])
            return _present(state=state, normed=normed)
        state, normed, statistics = s["model"].forward_with_statistics(s["x"], s["residual"], s["gate"])
        d = s["model"].backward(s["x"], s["residual"], s["gate"], statistics, s["d_state"], s["d_normed"])
        return _present(state=state, normed=normed, d_x=d.x, d_residual=d.residual, d_gate=d.gate,
                        d_after_weight=d.after_weight, d_after_bias=d.after_bias, d_before_weight=d.before_weight,
                        d_before_bias=d.before_bias)
    r = P.log_probabilities(s["logits"], s["targets"], top_k=case["top_k"])
    out = _present(log_probs=r.log_probs, entropy=r.entropy, log_normalizer=r.log_normalizer,
                   top_classes=r.top_classes, top_log_probs=r.top_log_probs)
    if case["train"]:
        out["d_logits"] = r.backward(s["d_log_probs"], s["d_entropy"], s["d_log_normalizer"])
    return out


def _present(**outputs):
    return {k: v for k, v in outputs.items() if v is not None}


def _act(name, v):
    """The activation and its derivative."""
    if name == "relu":
        return v * (v > 0), (v > 0).to(v.dtype)
    if name == "leaky_relu":
        return torch.where(v > 0, v, 0.1 * v), torch.where(v > 0, 1.0, 0.1)
    if name == "tanh":
        t = torch.tanh(v)
        return t, 1 - t * t
    if name == "sigmoid":
        p = torch.sigmoid(v)
        return p, p * (1 - p)
    if name == "silu":
        p = torch.sigmoid(v)
        return v * p, p * (1 + v * (1 - p))
    c = math.sqrt(2 / math.pi)
    t = torch.tanh(c * (v + 0.044715 * v * v * v))
    return 0.5 * v * (1 + t), 0.5 * (1 + t) + 0.5 * v * (1 - t * t) * c * (1 + 3 * 0.044715 * v * v)


def _gated(case, s):
    t = TORCH[case["dtype"]]
    x, wg, wu, wd = (s[k].float() for k in ("x", "gate", "up", "down"))
    g, u = wg.T @ x, wu.T @ x
    g0, u0, d0 = s["biases"]
    if g0 is not None:
        g, u = g + g0.float()[:, None], u + u0.float()[:, None]
    h = (_act(case["act"], g)[0] * u).to(t).float()
    y = wd.T @ h
    if d0 is not None:
        y = y + d0.float()[:, None]
    out = {"y": y.to(t)}
    if not case["train"]:
        return out
    dy = s["dy"].float()
    dh = wd @ dy
    g, u = g.to(t).float(), u.to(t).float()  # as they are kept for the backward pass
    a, slope = _act(case["act"], g)
    dg, du = (dh * u * slope).to(t).float(), (dh * a).to(t).float()
    out.update(d_x=(wg @ dg + wu @ du).to(t), d_gate=(x @ dg.T).to(t), d_up=(x @ du.T).to(t), d_down=(h @ dy.T).to(t))
    if g0 is not None:
        out.update(d_gate_bias=dg.sum(1).to(t), d_up_bias=du.sum(1).to(t), d_down_bias=dy.sum(1).to(t))
    return out


def _normalise(kind, v, weight, bias):
    """The norm of each column, and what its gradient needs."""
    mean = v.mean(0) if kind == "layer" else torch.zeros_like(v[0])
    centred = v - mean
    r = 1 / torch.sqrt((centred * centred).mean(0) + EPS)
    unit = centred * r
    return unit * weight[:, None] + (0 if bias is None else bias[:, None]), unit, r


def _normalise_backward(kind, d, unit, r, weight):
    e = d * weight[:, None]
    d_in = e - unit * (e * unit).mean(0)
    if kind == "layer":
        d_in = d_in - e.mean(0)
    return d_in * r, (d * unit).sum(1), d.sum(1) if kind == "layer" else None


def _norm(case, s):
    t, scale = TORCH[case["dtype"]], case["scale"]
    x = s["x"].float()
    v = x
    if s["after"] is not None:
        v, unit1, r1 = _normalise(case["after"], x, *s["after"])
    gate = None if s["gate"] is None else s["gate"].float() if case["gate"] == "full" else s["gate"][:, None]
    state = scale * v if gate is None else scale * gate * v
    if s["residual"] is not None:
        state = s["residual"].float() + state
    out = {"state": state.to(t)}
    if s["before"] is not None:
        normed, unit2, r2 = _normalise(case["before"], state, *s["before"])
        out["normed"] = normed.to(t)
    if not case["train"]:
        return out
    d = s["d_state"].float()
    if s["before"] is not None:
        d2, w, b = _normalise_backward(case["before"], s["d_normed"].float(), unit2, r2, s["before"][0])
        d = d + d2
        out["d_before_weight"] = w
        if b is not None:
            out["d_before_bias"] = b
    if s["residual"] is not None:
        out["d_residual"] = d.to(t)
    dv = scale * d
    if gate is not None:
        out["d_gate"] = (dv * v).to(t) if case["gate"] == "full" else (dv * v).sum(1)
        dv = dv * gate
    if s["after"] is not None:
        dv, w, b = _normalise_backward(case["after"], dv, unit1, r1, s["after"][0])
        out["d_after_weight"] = w
        if b is not None:
            out["d_after_bias"] = b
    out["d_x"] = dv.to(t)
    return out


def _logp(case, s):
    x, targets = s["logits"].float(), s["targets"].long()
    c, b = x.shape
    top = x.amax(0)
    none = top == -math.inf  # every class is ruled out
    shift = torch.where(none, 0.0, top)
    e = torch.exp(x - shift)
    total = e.sum(0)
    normalizer = shift + torch.log(total)  # -inf where there is no class
    moment = torch.where(e > 0, e * (x - shift), 0.0).sum(0)
    p = torch.where(none, 0.0, moment / total)
    entropy = torch.where(none, 0.0, torch.log(total) - p)
    given = (targets >= 0) & (targets < c)
    logit = x.gather(0, targets.clamp(0, c - 1)[None])[0]
    out = {"log_probs": torch.where(given, torch.where(logit == -math.inf, logit, logit - normalizer), 0.0),
           "entropy": entropy, "log_normalizer": normalizer}
    if case["top_k"]:
        index = torch.arange(c, device=x.device, dtype=torch.int32)[:, None]
        left, classes, values = x.clone(), [], []
        for _ in range(case["top_k"]):
            most = left.amax(0)
            at = torch.where(left == most, index, c).amin(0)  # ties: the lowest index
            left.scatter_(0, at[None].long(), -math.inf)
            ruled_out = most == -math.inf
            classes.append(torch.where(ruled_out, -1, at))
            values.append(torch.where(ruled_out, most, most - normalizer))
        out["top_classes"], out["top_log_probs"] = torch.stack(classes).int(), torch.stack(values)
    if case["train"]:
        log_p = x - torch.where(none, 0.0, normalizer)
        p = torch.exp(log_p)
        d_logp = torch.where(given, s["d_log_probs"], 0.0)
        d = p * (s["d_log_normalizer"] - d_logp) - s["d_entropy"] * torch.where(p > 0, p * (log_p + entropy), 0.0)
        at = targets.clamp(0, c - 1)[None]
        d.scatter_add_(0, at, d_logp[None])
        out["d_logits"] = torch.where(none, 0.0, d).to(TORCH[case["dtype"]])
    return out


# -- what a pass cannot do without -----------------------------------------------------------------


def work(case):
    b, es = case["batch"], BYTES[case["dtype"]]
    if case["op"] == "gated":
        i, h, o = _widths(case)
        weights = es * ((2 * i + o) * h + (2 * h + o if case["bias"] else 0))
        data = es * (i + o) * b
        return {"bytes": float((weights + data) * (2 if case["train"] else 1)), "flops": _gated_flops(case) * b}
    if case["op"] == "norm":
        n, full, vector = case["n"], case["gate"] == "full", case["gate"] == "feature"
        arrays = 2 + case["residual"] + full + (case["before"] != "none")
        vectors = sum({"none": 0, "rms": 1, "layer": 2}[case[k]] for k in ("after", "before")) + vector
        flops = 20.0
        if case["train"]:
            # the gradients of what came out are read, those of what went in are written
            arrays += 2 + case["residual"] + full + (case["before"] != "none")
            vectors, flops = 2 * vectors, 60.0
        return {"bytes": float(arrays * n * b * es + 4 * vectors * n), "flops": flops * n * b}
    c, k = case["classes"], case["top_k"]
    data = (2 if case["train"] else 1) * c * b * es + (16 + 8 * k + (12 if case["train"] else 0)) * b
    return {"bytes": float(data), "flops": (12.0 if case["train"] else 6.0) * c * b}


# -- the same in 64 bits ---------------------------------------------------------------------------


def exact(case, seed):
    s = _inputs(case, seed)
    return {"gated": _exact_gated, "norm": _exact_norm, "logp": _exact_logp}[case["op"]](case, s)


EXACT_ACTS = {
    "relu": lambda v: v.clamp(min=0),
    "leaky_relu": lambda v: torch.maximum(v, 0.1 * v),
    "tanh": torch.tanh,
    "sigmoid": lambda v: 1 / (1 + torch.exp(-v)),
    "silu": lambda v: v / (1 + torch.exp(-v)),
    "gelu": lambda v: v / (1 + torch.exp(-2 * math.sqrt(2 / math.pi) * (v + 0.044715 * v ** 3))),
}


def _exact_gated(case, s):
    """Columns in pieces; the activation differentiated by torch."""
    t, f = TORCH[case["dtype"]], EXACT_ACTS[case["act"]]
    wg, wu, wd = (s[k].double() for k in ("gate", "up", "down"))
    g0, u0, d0 = (0.0 if v is None else v.double()[:, None] for v in s["biases"])
    out = {k: [] for k in (("y", "d_x") if case["train"] else ("y",))}
    sums = {}

    def add(name, v):
        sums[name] = sums[name] + v if name in sums else v

    step = max(1, int(2e8 / max(_widths(case))))
    for c in range(0, case["batch"], step):
        x = s["x"][:, c:c + step].double()
        g, u = torch.matmul(wg.T, x) + g0, torch.matmul(wu.T, x) + u0
        h = (f(g) * u).to(t).double()
        out["y"].append(torch.matmul(wd.T, h) + d0)
        if not case["train"]:
            continue
        dy = s["dy"][:, c:c + step].double()
        dh = torch.matmul(wd, dy)
        u = u.to(t).double()
        g = g.to(t).double().requires_grad_()
        with torch.enable_grad():
            a = f(g)
            slope, = torch.autograd.grad(a.sum(), g)
        du, dg = (dh * a.detach()).to(t).double(), (dh * u * slope).to(t).double()
        out["d_x"].append(torch.cat([wg, wu], 1) @ torch.cat([dg, du]))
        add("d_gate", x @ dg.T)
        add("d_up", x @ du.T)
        add("d_down", h @ dy.T)
        if case["bias"]:
            for k, v in (("d_gate_bias", dg), ("d_up_bias", du), ("d_down_bias", dy)):
                add(k, v.sum(1))
    return {**{k: torch.cat(v, 1) for k, v in out.items()}, **sums}


def _exact_norm(case, s):
    """Differentiated by torch."""
    leaves = {k: s[k].double().requires_grad_() for k in ("x", "residual", "gate") if s[k] is not None}
    for k in ("after", "before"):
        if s[k] is not None:
            leaves[k + "_weight"] = s[k][0].double().requires_grad_()
            if s[k][1] is not None:
                leaves[k + "_bias"] = s[k][1].double().requires_grad_()

    def norm(k, v):
        if s[k] is None:
            return v
        if case[k] == "layer":
            v = v - v.mean(0, keepdim=True)
        v = v * ((v ** 2).mean(0, keepdim=True) + EPS) ** -0.5 * leaves[k + "_weight"].unsqueeze(1)
        return v + leaves[k + "_bias"].unsqueeze(1) if k + "_bias" in leaves else v

    with torch.enable_grad():
        branch = norm("after", leaves["x"]) * case["scale"]
        if s["gate"] is not None:
            branch = branch * (leaves["gate"] if case["gate"] == "full" else leaves["gate"].unsqueeze(1))
        state = branch + leaves["residual"] if s["residual"] is not None else branch
        out = {"state": state}
        if s["before"] is not None:
            out["normed"] = norm("before", state)
        if case["train"]:
            loss = (state * s["d_state"].double()).sum()
            if s["before"] is not None:
                loss = loss + (out["normed"] * s["d_normed"].double()).sum()
            grads = torch.autograd.grad(loss, list(leaves.values()))
            out.update({"d_" + k: g for k, g in zip(leaves, grads)})
    return {k: v.detach() for k, v in out.items()}


def _exact_logp(case, s):
    """Columns in pieces, from log_softmax and a stable sort."""
    c, b, k = case["classes"], case["batch"], case["top_k"]
    parts = []
    step = max(1, int(1e8 / c))
    for at in range(0, b, step):
        x = s["logits"][:, at:at + step].double()
        t = s["targets"][at:at + step].long()
        none = torch.isinf(x).all(0)
        lp = torch.log_softmax(torch.where(none, 0.0, x), 0)
        p = torch.exp(lp)
        given = t >= 0
        one = torch.nn.functional.one_hot(t.clamp(min=0), c).T if c * x.shape[1] <= 4e6 else None
        mine = lp.gather(0, t.clamp(min=0)[None])[0] if one is None else torch.where(one == 1, lp, 0.0).sum(0)
        o = {"log_probs": torch.where(given, torch.where(none, -math.inf, mine), 0.0),
             "entropy": torch.where(none, 0.0, -torch.where(p > 0, p * lp, 0.0).sum(0)),
             "log_normalizer": torch.logsumexp(x, 0)}
        if k:
            values, order = torch.sort(x, dim=0, descending=True, stable=True)
            out = values[:k] == -math.inf
            o["top_classes"] = torch.where(out, -1, order[:k]).int()
            o["top_log_probs"] = torch.where(out, -math.inf, lp.gather(0, order[:k]))
        if case["train"]:
            d_logp = torch.where(given, s["d_log_probs"][at:at + step].double(), 0.0)
            d = s["d_log_normalizer"][at:at + step].double() * p - d_logp * p
            d -= s["d_entropy"][at:at + step].double() * torch.where(p > 0, p * (lp + o["entropy"]), 0.0)
            d[t.clamp(min=0), torch.arange(x.shape[1], device=x.device)] += d_logp
            o["d_logits"] = torch.where(none, 0.0, d)
        parts.append(o)
    return {name: torch.cat([o[name] for o in parts], -1) for name in parts[0]}
