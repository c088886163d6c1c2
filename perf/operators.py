"""Performance cases of the expert and 4-bit operators, as a program that uses this framework calls them.

A case is a dict of

  op       "route"    scores [experts, batch] -> top-k experts, weights and the samples sorted by expert
           "experts"  a chain of Matvec, Bias and activation per expert over columns sorted by expert;
                      the products take operands of the model's type, so states between layers are rounded to it
           "mixture"  scores -> route -> gather -> the chosen experts' chains -> weighted sum
           "mx4"      quantisation of x to microscaled 4-bit floating point, and back
  dtype    "f32", "f16", "bf16": type of the scores (route) or of x and y
  weights  "same" (the type of x) or "mx4" (weights and every layer's input in 4 bits)
  experts, top_k, batch (samples, or sorted columns), widths joined by "-", act after every layer but the last
  masked   route: share of the scores that are -inf
  normalize  route: weights of the softmax over the "chosen" scores or over "all"

`run` computes an operator in its plain form (elementary torch operations in 32 bits), or where `own` is
true through the framework's entry points.
"""
from __future__ import annotations

import math

import torch

own = False

TORCH = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"f32": 4, "f16": 2, "bf16": 2}
BLOCK = 32  # features that share a scale


def listed():
    return [
        # The router of a few regimes over one small domain's columns: latency counts.
        {"name": "route_few", "op": "route", "dtype": "f32", "experts": 8, "top_k": 2, "batch": 96,
         "masked": 0.0, "normalize": "chosen"},
        # Many experts over an odd million of cells, a tenth of them ruled out, bf16 scores full of ties.
        {"name": "route_cells", "op": "route", "dtype": "bf16", "experts": 64, "top_k": 4, "batch": 1_000_003,
         "masked": 0.1, "normalize": "all"},
        # Five regimes' fp32 emulators with odd widths, ragged groups.
        {"name": "experts_f32_odd", "op": "experts", "dtype": "f32", "weights": "same", "experts": 5,
         "widths": "33-200-17", "act": "tanh", "batch": 40_003},
        # The benchmark's fp16 tanh network as eight experts over a million sorted columns.
        {"name": "experts_tanh_f16", "op": "experts", "dtype": "f16", "weights": "same", "experts": 8,
         "widths": "64-256-256-256-64", "act": "tanh", "batch": 1_000_000},
        # One wide grouped product: matrix cores.
        {"name": "experts_wide_bf16", "op": "experts", "dtype": "bf16", "weights": "same", "experts": 16,
         "widths": "1024-1024", "act": "none", "batch": 65_536},
        # Serving single samples: the chosen experts' weights from memory, and the launches.
        {"name": "mixture_few_bf16", "op": "mixture", "dtype": "bf16", "weights": "same", "experts": 8, "top_k": 2,
         "widths": "1024-2048-1024", "act": "silu", "batch": 3},
        # A whole batch through a mixture of thirty-two experts.
        {"name": "mixture_f16", "op": "mixture", "dtype": "f16", "weights": "same", "experts": 32, "top_k": 4,
         "widths": "512-1024-512", "act": "gelu", "batch": 65_536},
        # Quantisation of an odd number of features of a small batch.
        {"name": "mx4_odd_f32", "op": "mx4", "dtype": "f32", "widths": "100", "batch": 1_003},
        # Quantisation of wide activations over a large batch.
        {"name": "mx4_wide_bf16", "op": "mx4", "dtype": "bf16", "widths": "1024", "batch": 262_144},
        # One dense layer with 4-bit weights on eight samples: the weights from memory.
        {"name": "mx4_product_few", "op": "experts", "dtype": "f16", "weights": "mx4", "experts": 1,
         "widths": "2048-2048", "act": "none", "batch": 8},
        # The largest 4-bit product: matrix cores.
        {"name": "mx4_product_wide", "op": "experts", "dtype": "bf16", "weights": "mx4", "experts": 1,
         "widths": "4096-4096", "act": "none", "batch": 16_384},
        # A mixture whose experts hold 4-bit weights.
        {"name": "mx4_mixture", "op": "mixture", "dtype": "bf16", "weights": "mx4", "experts": 16, "top_k": 2,
         "widths": "1024-2048-1024", "act": "silu", "batch": 16_384},
    ]


ACTS = ("relu", "leaky_relu", "silu", "gelu", "tanh", "sigmoid")


def draw(rng):
    """A case of one of the listed kinds with other sizes and types."""

    def log_int(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    kind = rng.choice(("route", "experts", "experts", "mixture", "mixture", "mx4", "product"))
    if kind == "route":
        e = log_int(2, 512)
        return {"op": "route", "dtype": rng.choice(("f32", "f16", "bf16")), "experts": e,
                "top_k": rng.randint(1, min(8, e)), "batch": log_int(1, min(1_000_000, 60_000_000 // e)),
                "masked": rng.choice((0.0, 0.1, 0.5)), "normalize": rng.choice(("chosen", "all"))}
    if kind == "mx4":
        k = log_int(1, 4096)
        return {"op": "mx4", "dtype": rng.choice(("f32", "f16", "bf16")), "widths": str(k),
                "batch": log_int(1, min(1_000_000, 120_000_000 // k))}
    case = {"op": "mixture" if kind == "mixture" else "experts"}
    case["weights"] = "mx4" if kind == "product" else rng.choice(("same", "same", "mx4"))
    case["dtype"] = rng.choice(("f16", "bf16") if case["weights"] == "mx4" else ("f32", "f16", "bf16"))
    case["experts"] = 1 if kind == "product" else log_int(2, 64)
    layers = 1 if kind == "product" else rng.randint(1, 3)
    case["widths"] = "-".join(str(log_int(8, 2048)) for _ in range(layers + 1))
    case["act"] = rng.choice(ACTS) if layers > 1 else "none"
    if kind == "mixture":
        case["top_k"] = rng.randint(1, min(4, case["experts"]))
    # Batches within the largest listed case's cost.
    macs = _macs(case) * case.get("top_k", 1)
    case["batch"] = log_int(1, max(2, min(1_000_000, 6e10 / macs, 2e8 / sum(_widths(case)) / case.get("top_k", 1))))
    return case


# -- inputs ------------------------------------------------------------------------------------


def _widths(case):
    return [int(w) for w in case["widths"].split("-")]


def _macs(case):
    w = _widths(case)
    return sum(a * b for a, b in zip(w, w[1:]))


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(1 + seed)


def _scores(case, g):
    """Router outputs: some experts are popular; a few samples are ruled out altogether."""
    e, b = case["experts"], case["batch"]
    s = torch.randn((e, b), device="cuda", generator=g) + 0.5 * torch.randn((e, 1), device="cuda", generator=g)
    if case.get("masked", 0.0):
        off = torch.rand((e, b), device="cuda", generator=g) < case["masked"]
        off |= torch.rand((1, b), device="cuda", generator=g) < 0.01
        s = s.masked_fill(off, -math.inf)
    return s.to(TORCH[case["dtype"]]) if case["op"] == "route" else s


def _parameters(case, g):
    """W [experts, n_in, n_out] Glorot-uniform and small biases, per layer, as the model's type holds them."""
    w, e, t = _widths(case), case["experts"], TORCH[case["dtype"]]
    out = []
    for a, b in zip(w, w[1:]):
        lim = math.sqrt(6.0 / (a + b))
        out.append((((torch.rand((e, a, b), device="cuda", generator=g) * 2 - 1) * lim).to(t),
                    torch.rand((e, b), device="cuda", generator=g) * 0.2 - 0.1))
    return out


def _inputs(case, seed):
    g = _generator(seed)
    s = {}
    if case["op"] == "route":
        s["scores"] = _scores(case, g)
        return s
    k, b = _widths(case)[0], case["batch"]
    x = torch.randn((k, b), device="cuda", generator=g)
    if case["op"] == "mx4":
        x = x * torch.exp(2.0 * torch.randn((k, 1), device="cuda", generator=g))  # features of different sizes
    s["x"] = x.to(TORCH[case["dtype"]])
    if case["op"] == "mx4":
        return s
    s["params"] = _parameters(case, g)
    if case["op"] == "mixture":
        s["scores"] = _scores(case, g)
        return s
    # Sorted columns: group sizes as a popularity gives them, one group empty where there are several.
    e = case["experts"]
    p = torch.softmax(0.7 * torch.randn(e, device="cuda", generator=g), 0)
    if e >= 4:
        p[e // 2] = 0.0
    counts = (p / p.sum() * b).long()
    counts[0] += b - counts.sum()
    s["offsets"] = torch.cat([counts.new_zeros(1), counts.cumsum(0)]).to(torch.int32)
    s["counts"] = counts.tolist()
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    s["case"] = case
    if "params" in s:
        # The plain form's weights laid out once, as a program keeps them: [experts, n_out, n_in] in 32 bits.
        s["plain"] = [((_mx4_values(w.float()) if case["weights"] == "mx4" else w.float()).transpose(1, 2).contiguous(),
                       b[:, :, None]) for w, b in s["params"]]
        if own:
            s["model"] = _model(case, s["params"])
        del s["params"]
    return s


def _model(case, params):
    import ponni_amd as P

    act = {"relu": P.Relu, "leaky_relu": lambda n: P.LeakyRelu(n, 0.1), "tanh": P.Tanh, "sigmoid": P.Sigmoid,
           "silu": P.Silu, "gelu": lambda n: P.Gelu(n, True)}
    layers = []
    for i, (w, b) in enumerate(params):
        layers += [P.ExpertMatvec(w), P.ExpertBias(b)]
        if i < len(params) - 1:
            layers.append(act[case["act"]](w.shape[2]))
    return P.create_expert_model(*layers, dtype=case["dtype"], weights=case["weights"])


# -- one pass ------------------------------------------------------------------------------------


def run(state):
    case = state["case"]
    if own:
        return _run_own(case, state)
    if case["op"] == "route":
        return _route(state["scores"], case["top_k"], case["normalize"])
    x = state["x"].float()
    if case["op"] == "mx4":
        v, scales = _mx4(x, 0)
        return {"values": v.to(state["x"].dtype), "scales": _scale_rows(scales)}
    if case["op"] == "experts":
        y = _grouped(case, state["plain"], x, state["offsets"], state["counts"])
        return y.to(state["x"].dtype)
    r = _route(state["scores"], case["top_k"], "chosen")
    counts = (r["offsets"][1:] - r["offsets"][:-1]).tolist()
    total = sum(counts)
    y = _grouped(case, state["plain"], x[:, r["source"][:total].long()], r["offsets"], counts)
    y = y[:, r["slots"].long().clamp(min=0)]  # [n_out, top_k, batch]
    return (y * r["weights"]).sum(1).to(state["x"].dtype)


def _run_own(case, state):
    import ponni_amd as P

    if case["op"] == "route":
        r = P.route_experts(state["scores"], case["top_k"], case["normalize"])
        return {"experts": r.experts, "weights": r.weights, "slots": r.slots, "source": r.source,
                "offsets": r.offsets}
    if case["op"] == "mx4":
        q = P.quantize_mx4(state["x"])
        return {"values": q.dequantize(state["x"].dtype), "scales": q.scales}
    if case["op"] == "experts":
        return state["model"].forward_batch_parallel(state["x"], state["offsets"])
    r = P.route_experts(state["scores"], case["top_k"], "chosen")
    return state["model"].forward_mixture(state["x"], r)


def _route(scores, top_k, normalize):
    s = scores.float()
    e, b = s.shape
    index = torch.arange(e, device=s.device)[:, None]
    left, experts, values = s.clone(), [], []
    for _ in range(top_k):
        top = left.amax(0)
        at = torch.where(left == top, index, e).amin(0)  # ties: the lowest index
        left.scatter_(0, at[None], -math.inf)
        experts.append(at)
        values.append(top)
    experts, values = torch.stack(experts), torch.stack(values)
    valid = values > -math.inf
    largest = torch.where(valid[0], values[0], 0.0)
    w = torch.exp(values - largest)
    total = (w if normalize == "chosen" else torch.exp(s - largest)).sum(0)
    w = torch.where(valid, w / total, 0.0)
    taken = torch.zeros((e, b), dtype=torch.int32, device=s.device)
    taken.scatter_(0, experts, valid.int())
    offsets = torch.cat([torch.zeros(1, dtype=torch.int64, device=s.device), taken.sum(1).cumsum(0)])
    rank = taken.cumsum(1).gather(0, experts) - 1
    slots = torch.where(valid, offsets[experts] + rank, -1)
    source = torch.full((top_k * b + 1,), -1, dtype=torch.int64, device=s.device)
    sample = torch.arange(b, device=s.device).expand(top_k, b)
    source.scatter_(0, torch.where(valid, slots, top_k * b).reshape(-1), sample.reshape(-1))
    return {"experts": torch.where(valid, experts, -1).int(), "weights": w, "slots": slots.int(),
            "source": source[:-1].int(), "offsets": offsets.int()}


def _grouped(case, weights, x, offsets, counts):
    """The chains over sorted columns: groups padded to the largest one, one batched product a layer."""
    e, cap, total = len(counts), max(max(counts), 1), x.shape[1]
    at = offsets[:-1, None].long() + torch.arange(cap, device=x.device)
    h = x if e == 1 else x[:, at.clamp(max=total - 1)].movedim(1, 0)  # [experts, n_in, cap]
    h = h.reshape(e, x.shape[0], cap)
    for i, (w, b) in enumerate(weights):
        if case["weights"] == "mx4":
            h = _mx4_values(h)
        h = torch.matmul(w, h.contiguous()) + b
        if i < len(weights) - 1:
            h = _activation(case["act"], h)
            if case["weights"] == "same":
                h = h.to(TORCH[case["dtype"]]).float()
    if e == 1:
        return h[0]
    group = torch.bucketize(torch.arange(total, device=x.device, dtype=torch.int32), offsets[1:], right=True)
    column = torch.arange(total, device=x.device) - offsets[group].long()
    return h.movedim(0, 1).reshape(-1, e * cap)[:, group * cap + column]


def _activation(name, v):
    if name == "relu":
        return v * (v > 0)
    if name == "leaky_relu":
        return torch.where(v > 0, v, 0.1 * v)
    if name == "tanh":
        return torch.tanh(v)
    if name == "sigmoid":
        return torch.sigmoid(v)
    if name == "silu":
        return v * torch.sigmoid(v)
    return 0.5 * v * (1 + torch.tanh(math.sqrt(2 / math.pi) * (v + 0.044715 * v * v * v)))


def _mx4(x, dim):
    """x as blocks of 32 along `dim` hold it, and the blocks' scale exponents (biased by 127)."""
    n = x.shape[dim]
    blocks = -(-n // BLOCK)
    v = x.movedim(dim, -1)
    v = torch.nn.functional.pad(v, (0, blocks * BLOCK - n)).unflatten(-1, (blocks, BLOCK))
    largest = v.abs().amax(-1, keepdim=True)
    exponent = torch.where(largest > 0, torch.frexp(largest)[1] - 3, -127).clamp(min=-127)
    v = torch.ldexp(v, -exponent)
    size = v.abs()
    step = torch.where(size < 2, 0.5, torch.where(size < 4, 1.0, 2.0))
    v = torch.round(v / step) * step
    v = torch.ldexp(v.clamp(-6, 6), exponent).flatten(-2)[..., :n].movedim(-1, dim)
    return v, (exponent[..., 0] + 127).to(torch.uint8)


def _mx4_values(x):
    return _mx4(x, 1)[0]


def _scale_rows(scales):
    """The scales as the framework's rows hold them: whole words of four."""
    return torch.nn.functional.pad(scales, (0, -scales.shape[1] % 4))


# -- what a pass cannot do without -----------------------------------------------------------------


def work(case):
    b, es = case["batch"], BYTES[case["dtype"]]
    if case["op"] == "route":
        e, k = case["experts"], case["top_k"]
        return {"bytes": float(e * b * es + 16 * k * b + 4 * (e + 1)), "flops": 3.0 * e * b}
    w = _widths(case)
    if case["op"] == "mx4":
        blocks = -(-w[0] // BLOCK)
        # x read, codes and scales written and read again, the values written
        return {"bytes": float(2 * w[0] * b * es + 2 * 17 * blocks * b), "flops": 4.0 * w[0] * b}
    k = case.get("top_k", 1)
    used = case["experts"] if case["op"] == "experts" else min(case["experts"], k * b)
    per = 17 / 32 if case["weights"] == "mx4" else es
    data = (w[0] + w[-1]) * b * es + used * (_macs(case) * per + 4 * sum(w[1:]))
    if case["op"] == "mixture":
        data += 4 * case["experts"] * b
    return {"bytes": float(data), "flops": 2.0 * k * b * _macs(case)}


# -- the same in 64 bits ---------------------------------------------------------------------------


def exact(case, seed):
    s = _inputs(case, seed)
    if case["op"] == "route":
        return _exact_route(s["scores"].double(), case["top_k"], case["normalize"])
    x = s["x"].double()
    if case["op"] == "mx4":
        return {"values": _exact_mx4(x), "scales": None}
    params = [(w.double(), b.double()) for w, b in s["params"]]
    if case["weights"] == "mx4":
        params = [(torch.stack([_exact_mx4(m) for m in w]), b) for w, b in params]

    def chain(e, h):
        for i, (w, b) in enumerate(params):
            if case["weights"] == "mx4":
                h = _exact_mx4(h)
            h = w[e].T.contiguous() @ h + b[e][:, None]
            if i < len(params) - 1:
                h = EXACT_ACTS[case["act"]](h)
                if case["weights"] == "same":
                    h = h.to(TORCH[case["dtype"]]).double()
        return h

    y = torch.zeros((_widths(case)[-1], case["batch"]), dtype=torch.float64, device="cuda")
    if case["op"] == "experts":
        first = 0
        for e, n in enumerate(s["counts"]):
            for c in range(first, first + n, 1 << 17):
                d = min(first + n, c + (1 << 17))
                y[:, c:d] = chain(e, x[:, c:d])
            first += n
        return y
    r = _exact_route(s["scores"].double(), case["top_k"], "chosen")
    for e in range(case["experts"]):
        j, b = torch.nonzero(r["experts"] == e, as_tuple=True)
        if len(b):
            y[:, b] += chain(e, x[:, b]) * r["weights"][j, b]
    return y


EXACT_ACTS = {
    "relu": lambda v: v.clamp(min=0),
    "leaky_relu": lambda v: torch.maximum(v, 0.1 * v),
    "tanh": torch.tanh,
    "sigmoid": lambda v: 1 / (1 + torch.exp(-v)),
    "silu": lambda v: v / (1 + torch.exp(-v)),
    "gelu": lambda v: v / (1 + torch.exp(-2 * math.sqrt(2 / math.pi) * (v + 0.044715 * v ** 3))),
}


def _exact_route(s, top_k, normalize):
    """From one stable sort of each sample's scores, and one of the assignments."""
    e, b = s.shape
    if e * b > 100_000_000:
        return None
    values, order = torch.sort(s, dim=0, descending=True, stable=True)
    values, order = values[:top_k], order[:top_k]
    none = values == -math.inf
    p = torch.softmax(values if normalize == "chosen" else s, 0)
    w = p if normalize == "chosen" else p.gather(0, order)
    group = torch.where(none, e, order).T.reshape(-1)  # sample by sample
    by_group = torch.sort(group, stable=True)[1]
    slots = torch.empty_like(by_group)
    slots[by_group] = torch.arange(len(by_group), device=s.device)
    total = int((~none).sum())
    source = by_group // top_k
    source[total:] = -1
    counts = torch.bincount(group, minlength=e + 1)[:e]
    return {"experts": torch.where(none, -1, order).int(), "weights": torch.where(none, 0.0, w),
            "slots": torch.where(none, -1, slots.reshape(b, top_k).T).int(), "source": source.int(),
            "offsets": torch.nn.functional.pad(counts.cumsum(0), (1, 0)).int()}


def _exact_mx4(x):
    """x [features, columns] through e2m1 codes and power-of-two scales, found by comparisons."""
    k, n = x.shape
    y = torch.zeros((-(-k // BLOCK) * BLOCK, n), dtype=torch.float64, device=x.device)
    y[:k] = x
    y = y.reshape(-1, BLOCK, n)
    largest = y.abs().amax(1, keepdim=True)
    scale = torch.exp2((torch.floor(torch.log2(largest.clamp(min=2.0 ** -200))) - 2).clamp(min=-127))
    size = y.abs() / scale
    level = sum(size >= t if even else size > t for t, even in
                ((0.25, 0), (0.75, 1), (1.25, 0), (1.75, 1), (2.5, 0), (3.5, 1), (5.0, 0)))
    table = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64, device=x.device)
    return (torch.sign(y) * table[level.long()] * scale).reshape(-1, n)[:k]
