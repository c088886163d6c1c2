"""Gated blocks, norms between blocks and log probabilities in 64 bits, each with a bound of how far a
computation in the kernels' precisions may be off, element by element.

The bounds add up rounding errors to first order: a sum of n products in fp32, in any order, is off by at most
(n + 2) 2^-24 times the sum of the products' magnitudes, a rounding to the model's type by U of the value (and half
of the least subnormal), an activation or exponential by 8 units of fp32; what later steps make of an error is its
factor in them.  `SLACK` covers second-order terms."""
import numpy as np

E = 2.0 ** -24
U = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}
TINY = {"f32": 2.0 ** -126, "f16": 2.0 ** -25, "bf16": 2.0 ** -126}
SLACK = 1.25


def half(a, dtype):
    """a rounded to the type, as float64."""
    import torch

    t = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[dtype]
    return torch.from_numpy(np.ascontiguousarray(a)).to(t).double().numpy()


def rounding(v, dtype):
    return U[dtype] * np.abs(v) + TINY[dtype]


# -- activations: value, slope, and the largest magnitude of slope and second derivative -------------

_erf = np.vectorize(__import__("math").erf, otypes=[float])


def activation(name, v):
    if name == "relu":
        return np.where(v > 0, v, 0.0), (v > 0).astype(float)
    if name == "leaky_relu":
        return np.where(v > 0, v, 0.1 * v), np.where(v > 0, 1.0, 0.1)
    if name == "tanh":
        t = np.tanh(v)
        return t, 1 - t * t
    if name == "gelu_erf":
        p = 0.5 * (1 + _erf(v / np.sqrt(2)))
        return v * p, p + v * np.exp(-0.5 * v * v) / np.sqrt(2 * np.pi)
    if name == "sigmoid":
        p = 1 / (1 + np.exp(-v))
        return p, p * (1 - p)
    if name == "silu":
        p = 1 / (1 + np.exp(-v))
        return v * p, p * (1 + v * (1 - p))
    c = np.sqrt(2 / np.pi)
    p = 1 / (1 + np.exp(-2 * c * (v + 0.044715 * v ** 3)))
    return v * p, p + v * p * (1 - p) * 2 * c * (1 + 3 * 0.044715 * v * v)


ACTS = ("relu", "leaky_relu", "silu", "gelu", "gelu_erf", "tanh", "sigmoid")


# -- gated blocks ----------------------------------------------------------------------


def gated(w, x, act, dtype, biases=(None, None, None)):
    """(g, u, h, y) of float64 arrays of the type's values, and their bounds."""
    G, U_, D = w
    b = [0.0 if v is None else v[:, None] for v in biases]
    n, nh = G.shape[0], G.shape[1]
    g, u = G.T @ x + b[0], U_.T @ x + b[1]
    eg = (n + 2) * E * (np.abs(G).T @ np.abs(x) + np.abs(b[0]))
    eu = (n + 2) * E * (np.abs(U_).T @ np.abs(x) + np.abs(b[1]))
    a, slope = activation(act, g)
    # (1.2: a slope's largest magnitude, of GELU and SiLU 1.13; where Relu bends, an error of g passes as it is)
    ea = 1.2 * eg + 8 * E * (np.abs(a) + np.abs(g))
    if dtype != "f32":  # the hardware's forms of tanh and the sigmoid: an ulp of one near zero, |v| / 2 ulp far off
        ea = ea + 16 * E * (1 + np.abs(g)) * np.minimum(1.0, np.abs(g) + (act == "sigmoid"))
    h64 = a * u
    h = half(h64, dtype)
    eh = np.abs(a) * eu + np.abs(u) * ea + 2 * rounding(h64, dtype)  # (either side of a rounding)
    y = D.T @ h + b[2]
    ey = np.abs(D).T @ eh + (nh + 2) * E * (np.abs(D).T @ np.abs(h) + np.abs(b[2]))
    return [(g, SLACK * (eg + rounding(g, dtype))), (u, SLACK * (eu + rounding(u, dtype))),
            (h64, SLACK * eh), (y, SLACK * (ey + rounding(y, dtype)))]


def gated_backward(w, x, states, dy, act, dtype):
    """Gradients from the states as they were kept: name -> (value, bound)."""
    G, U_, D = w
    nh, no, c = G.shape[1], D.shape[1], x.shape[1]
    g, u, h = states
    dh = D @ dy
    edh = (no + 2) * E * (np.abs(D) @ np.abs(dy))
    a, slope = activation(act, g)
    es = 16 * E * (1 + np.abs(g))  # of the slope, and of the value
    if dtype != "f32":
        es = 2 * es
    dg64, du64 = dh * u * slope, dh * a
    edg = np.abs(u * slope) * edh + np.abs(dh * u) * es + 2 * rounding(dg64, dtype) + 4 * E * np.abs(dg64)
    edu = np.abs(a) * edh + np.abs(dh) * es + 2 * rounding(du64, dtype) + 4 * E * np.abs(du64)
    dg, du = half(dg64, dtype), half(du64, dtype)
    out = {}

    def put(name, value, bound):
        out[name] = (value, SLACK * (bound + rounding(value, dtype)))

    put("x", G @ dg + U_ @ du, np.abs(G) @ edg + np.abs(U_) @ edu
        + (2 * nh + 2) * E * (np.abs(G) @ np.abs(dg) + np.abs(U_) @ np.abs(du)))
    for name, d, e in (("gate", dg, edg), ("up", du, edu)):
        put(name, x @ d.T, np.abs(x) @ e.T + (c + 2) * E * (np.abs(x) @ np.abs(d).T))
        put(name + "_bias", d.sum(1), e.sum(1) + (c + 2) * E * np.abs(d).sum(1))
    put("down", h @ dy.T, (c + 2) * E * (np.abs(h) @ np.abs(dy).T))
    put("down_bias", dy.sum(1), (c + 2) * E * np.abs(dy).sum(1))
    return out


# -- norms between blocks ------------------------------------------------------------------


def norm_forward(x, residual, gate, after, before, scale, eps, dtype):
    """after, before: (kind, weight, bias) or None; gate [n], [n, columns] or None.  Values, bounds, and what the
    backward pass needs."""
    n = x.shape[0]
    k = (n + 16) * E  # of a sum over features and the steps around it
    f = scale * (1.0 if gate is None else gate[:, None] if gate.ndim == 1 else gate) * np.ones_like(x)

    def normalise(kind, v, ev):
        """unit, r, the bound of unit, and its magnitude before anything cancels."""
        m = v.mean(0) if kind == "layer" else 0.0 * v[0]
        em = ev.mean(0) + k * np.abs(v).mean(0) if kind == "layer" else 0.0
        d = v - m
        ed = ev + em + E * np.abs(d)
        var = (d * d).mean(0)
        r = 1 / np.sqrt(var + eps)
        # r's relative error is half of the mean square's
        er = 0.5 * r * r * ((2 * np.abs(d) * ed).mean(0) + k * var) + 4 * E
        unit = d * r
        return m, r, unit, r * ed + np.abs(unit) * (er + 2 * E)

    s = {"f": f, "x": x}
    zero = np.zeros_like(x)
    if after is None:
        v, ev = x, zero
        s.update(m1=zero[0], r1=zero[0] + 1, u1=x, eu1=zero, w1=zero[:, :1] + 1)
    else:
        kind, w, b = after
        w, b = np.ones(n) if w is None else w, np.zeros(n) if b is None else b
        m, r, unit, eu = normalise(kind, x, zero)
        v = unit * w[:, None] + b[:, None]
        ev = eu * np.abs(w[:, None]) + 2 * E * (np.abs(unit * w[:, None]) + np.abs(b[:, None]))
        s.update(m1=m, r1=r, u1=unit, eu1=eu, w1=w[:, None])
    base = 0.0 if residual is None else residual
    state = base + f * v
    est = np.abs(f) * ev + 3 * E * (np.abs(f * v) + np.abs(base))
    s.update(v=v, ev=ev, state=state, est=est)
    out = {"state": (state, SLACK * (est + rounding(state, dtype)))}
    if before is not None:
        kind, w, b = before
        w, b = np.ones(n) if w is None else w, np.zeros(n) if b is None else b
        m, r, unit, eu = normalise(kind, state, est)
        y = unit * w[:, None] + b[:, None]
        ey = eu * np.abs(w[:, None]) + 2 * E * (np.abs(unit * w[:, None]) + np.abs(b[:, None]))
        s.update(m2=m, r2=r, u2=unit, eu2=eu, w2=w[:, None])
        out["normed"] = (y, SLACK * (ey + rounding(y, dtype)))
    return out, s


def norm_backward(s, after, before, d_state, d_normed, scale, gate, dtype):
    """name -> (value, bound), from norm_forward's state."""
    x = s["x"]
    n, c = x.shape
    k, kc = (n + 16) * E, (c + 16) * E

    def through(kind, e, ee, unit, eu, r):
        """A norm's gradient of e (off by ee), before the weight."""
        mean_eu, mean_e = (e * unit).mean(0), e.mean(0) if kind == "layer" else 0.0
        emeu = (np.abs(unit) * ee + np.abs(e) * eu).mean(0) + k * np.abs(e * unit).mean(0)
        eme = ee.mean(0) + k * np.abs(e).mean(0) if kind == "layer" else 0.0
        d = r * (e - mean_e - unit * mean_eu)
        # r is off by the same share as unit at most, where unit is 1
        er = eu.max(0) / np.maximum(np.abs(unit).max(0), 1e-30) + 8 * E
        big = r * (np.abs(e) + np.abs(mean_e) + np.abs(unit * mean_eu))
        return d, r * (ee + eme + np.abs(unit) * emeu + np.abs(mean_eu) * eu) + big * (er + 4 * E)

    out = {}
    D = np.zeros_like(x) if d_state is None else d_state
    eD = E * np.abs(D)
    if before is not None and d_normed is not None:
        e = d_normed * s["w2"]
        d, ed = through(before[0], e, E * np.abs(e), s["u2"], s["eu2"], s["r2"])
        D, eD = D + d, eD + ed + E * np.abs(d)
        terms = np.abs(d_normed * s["u2"])
        out["before_weight"] = ((d_normed * s["u2"]).sum(1), (np.abs(d_normed) * s["eu2"]).sum(1) + kc * terms.sum(1))
        out["before_bias"] = (d_normed.sum(1), kc * np.abs(d_normed).sum(1))
    out["residual"] = (D, eD + rounding(D, dtype))
    dv = s["f"] * D
    edv = np.abs(s["f"]) * eD + 3 * E * np.abs(dv)
    dgate = scale * D * s["v"]
    edgate = abs(scale) * (eD * np.abs(s["v"]) + np.abs(D) * s["ev"]) + 3 * E * np.abs(dgate)
    if gate is not None:
        out["gate"] = (dgate.sum(1), edgate.sum(1) + kc * np.abs(dgate).sum(1)) if gate.ndim == 1 else \
            (dgate, edgate + rounding(dgate, dtype))
    if after is None:
        out["x"] = (dv, edv + rounding(dv, dtype))
    else:
        e = dv * s["w1"]
        d, ed = through(after[0], e, np.abs(s["w1"]) * edv + E * np.abs(e), s["u1"], s["eu1"], s["r1"])
        out["x"] = (d, ed + rounding(d, dtype))
        out["after_weight"] = ((dv * s["u1"]).sum(1), (edv * np.abs(s["u1"]) + np.abs(dv) * s["eu1"]).sum(1)
                               + kc * np.abs(dv * s["u1"]).sum(1))
        out["after_bias"] = (dv.sum(1), edv.sum(1) + kc * np.abs(dv).sum(1))
    return {name: (v, SLACK * e + 2.0 ** -126) for name, (v, e) in out.items()}


# -- log probabilities ------------------------------------------------------------------------


def log_probs(x, targets, top_k):
    """Values and bounds; classes of -inf are ruled out."""
    c, b = x.shape
    none = np.isneginf(x).all(0)
    finite = np.where(np.isneginf(x), np.nan, x)
    size = np.where(none, 0.0, np.nanmax(np.where(none, 0.0, np.abs(finite)), axis=0))
    top = np.where(none, 0.0, np.where(none, 0.0, x).max(0))
    e = np.exp(x - top)
    total = e.sum(0)
    with np.errstate(divide="ignore"):
        normalizer = top + np.log(total)
    log_p = np.where(np.isneginf(x), -np.inf, x - np.where(none, 0.0, normalizer))
    p = np.where(none, 0.0, np.exp(log_p))
    entropy = -np.where(p > 0, p * np.where(p > 0, log_p, 0.0), 0.0).sum(0)
    # Sums of positive terms by lanes, then joined; an exponent's error is its rounding and the constant's.
    depth = (64 + c / 32) * E
    e_n = depth + E * (16 + 8 * size + 4 * np.abs(np.where(none, 0.0, normalizer)))
    e_h = (2 * depth + E * (32 + 16 * size)) * (2 + np.log(c))
    given = np.zeros(b, bool) if targets is None else (targets >= 0) & (targets < c)
    at = np.where(given, targets, 0) if targets is not None else np.zeros(b, int)
    with np.errstate(invalid="ignore"):
        mine = log_p[at, np.arange(b)]
    mine = np.where(given, np.where(none, -np.inf, mine), 0.0)
    out = {"log_normalizer": (np.where(none, -np.inf, normalizer), SLACK * e_n), "entropy": (entropy, SLACK * e_h),
           "log_probs": (mine, SLACK * (e_n + E * np.abs(np.where(np.isfinite(mine), mine, 0.0))))}
    if top_k:
        order = np.argsort(-x, axis=0, kind="stable")[:top_k]
        v = np.take_along_axis(x, order, 0)
        out["top_classes"] = np.where(np.isneginf(v), -1, order)
        lp = np.where(np.isneginf(v), -np.inf, v - np.where(none, 0.0, normalizer))
        out["top_log_probs"] = (lp, SLACK * (e_n + E * np.abs(np.where(np.isfinite(lp), lp, 0.0))))
    out["_"] = (none, log_p, p, entropy, e_n, e_h, size, given, at)
    return out


def log_probs_backward(r, g_p, g_h, g_n, dtype):
    none, log_p, p, entropy, e_n, e_h, size, given, at = r["_"]
    b = p.shape[1]
    gl = np.where(given & ~none, 0.0 if g_p is None else g_p, 0.0)
    gh = np.zeros(b) if g_h is None else g_h
    gz = np.zeros(b) if g_n is None else g_n
    lp = np.where(p > 0, np.maximum(log_p, -700.0), 0.0)
    d = p * (gz - gl) - gh * p * (lp + entropy)
    big = p * (np.abs(gz) + np.abs(gl) + np.abs(gh) * (np.abs(lp) + entropy))
    # p's relative error: that of its exponent; in 16 bits by the hardware's 2^x of a rounded product
    rel = e_n + E * (16 + 4 * np.abs(lp) + 2 * size)
    bound = big * (rel + 8 * E) + p * np.abs(gh) * (e_h + e_n)
    d[at, np.arange(b)] += gl
    bound[at, np.arange(b)] += 2 * E * np.abs(gl)
    return np.where(none, 0.0, d), SLACK * (np.where(none, 0.0, bound) + rounding(np.where(none, 0.0, d), dtype))
