"""Routing, expert chains and 4-bit blocks in 64 bits, with the distance that
an evaluation in the operators' types can have from them, element by element."""
import numpy as np

EPS = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}  # half a step, relative
TINY = {"f32": 2.0 ** -149, "f16": 2.0 ** -25, "bf16": 2.0 ** -133}  # half the smallest step


def route(scores, top_k, normalize):
    """scores [E, B] float64: experts, weights, slots, source, offsets."""
    E, B = scores.shape
    s = np.where(np.isnan(scores), -np.inf, scores)
    order = np.argsort(-s, axis=0, kind="stable")[:top_k]
    v = np.take_along_axis(s, order, 0)
    none = np.isneginf(v)
    top = np.where(none[0], 0.0, v[0])

    def term(a):
        with np.errstate(invalid="ignore"):
            return np.where(np.isneginf(a), 0.0, np.where(a == top, 1.0, np.exp(a - top)))

    w = term(v)
    total = w.sum(0) if normalize == "chosen" else term(s).sum(0)
    w = np.where(none, 0.0, w / np.where(total == 0, 1.0, total))
    experts = np.where(none, -1, order)
    slots = np.full((top_k, B), -1)
    source = np.full(top_k * B, -1)
    offsets = np.zeros(E + 1, dtype=np.int64)
    at = 0
    for e in range(E):
        hit = experts == e
        for b in np.nonzero(hit.any(0))[0]:
            slots[np.nonzero(hit[:, b])[0][0], b] = at
            source[at] = b
            at += 1
        offsets[e + 1] = at
    return experts, w, slots, source, offsets


LEVELS = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6])


def mx4_scale(amax):
    """Exponent of a block's scale from its largest magnitude."""
    with np.errstate(divide="ignore"):
        return np.where(amax > 0, np.maximum(np.frexp(amax)[1] - 3, -127), -127)


def mx4_round(v):
    """v / scale to the nearest value, ties to the even code, at most 6."""
    s = np.abs(v)
    code = np.minimum(np.abs(s[..., None] - LEVELS).argmin(-1), 7)  # (a tie: the lower one)
    up = np.minimum(code + 1, 7)
    tie = np.abs(s - LEVELS[code]) == np.abs(LEVELS[up] - s)
    code = np.where(tie & (code % 2 == 1) & (up > code), up, code)
    return np.copysign(LEVELS[code], v)


def mx4(x):
    """x [features, columns]: the values its blocks of 32 features stand for, and the scales' exponents."""
    k, n = x.shape
    pad = -k % 32
    v = np.concatenate([x, np.zeros((pad, n))]).reshape(-1, 32, n)
    bad = ~np.isfinite(v).all(1, keepdims=True)
    exponent = mx4_scale(np.where(bad, 0.0, np.abs(np.where(np.isfinite(v), v, 0)).max(1, keepdims=True)))
    q = np.ldexp(mx4_round(np.ldexp(np.where(np.isfinite(v), v, 0), -exponent)), exponent)
    q = np.where(bad, np.nan, q).reshape(-1, n)[:k]
    return q, np.where(bad[:, 0], 255, exponent[:, 0] + 127)


def mx4_bounded(x, err):
    """The same of values known to `err`: the values of x, and how far those of any x' within err can be."""
    q, _ = mx4(x)
    far = np.zeros_like(x)
    k, n = x.shape
    pad = -k % 32
    hi = np.concatenate([np.abs(x) + err, np.zeros((pad, n))]).reshape(-1, 32, n).max(1, keepdims=True)
    lo = np.concatenate([np.maximum(np.abs(x) - err, 0), np.zeros((pad, n))]).reshape(-1, 32, n).max(1, keepdims=True)
    for amax in (lo, hi):
        e = np.broadcast_to(mx4_scale(amax), (amax.shape[0], 32, n)).reshape(-1, n)[:k]
        for v in (x - err, x, x + err):
            far = np.maximum(far, np.abs(np.ldexp(mx4_round(np.ldexp(v, -e)), e) - q))
    return q, far


ACTS = {
    "none": lambda v: v,
    "relu": lambda v: np.maximum(v, 0),
    "leaky_relu": lambda v: np.where(v > 0, v, 0.1 * v),
    "tanh": np.tanh,
    "sigmoid": lambda v: 1 / (1 + np.exp(-v)),
    "silu": lambda v: v / (1 + np.exp(-v)),
    "gelu": lambda v: v / (1 + np.exp(-2 * np.sqrt(2 / np.pi) * (v + 0.044715 * v ** 3))),
    "gelu_erf": None,
}


def _gelu_erf(v):
    from scipy.special import erf

    return 0.5 * v * (1 + erf(v / np.sqrt(2)))


ACTS["gelu_erf"] = _gelu_erf


def chain(layers, x, dtype, weights="same"):
    """x [n_in, columns] through (W [n_in, n_out], b or None, activation)...: the
    values before the last rounding to dtype, and a bound of an evaluation with
    operands in dtype (or 4 bits), fp32 sums and fp32 activations.

    One product's sum of n terms is off by at most n + 1 roundings of partial sums that
    |W|^T |x| + |b| bounds.  The activations' slopes are at most 1.13 (GELU, SiLU 1.1); their
    fp32 evaluation is off by 2^-20 (1 + |v|) at most: a rounded argument of 2^x, |x| < 64,
    is off by 2^-19 / 2 relative, which the logistic's slope of a quarter scales, and a few ulp."""
    h, err = np.asarray(x, dtype=np.float64), np.zeros(np.shape(x))
    for i, (w, b, act) in enumerate(layers):
        if weights == "mx4":
            h, err = mx4_bounded(h, err) if i else (mx4(h)[0], err)
            w = mx4(w)[0]
        elif i:
            err = err + EPS[dtype] * (np.abs(h) + err) + TINY[dtype]
        a = np.abs(w).T
        size = a @ (np.abs(h) + err)
        v = w.T @ h
        if b is not None:
            v = v + b[:, None]
            size = size + np.abs(b)[:, None]
        err = a @ err + (w.shape[0] + 2) * 2.0 ** -24 * size
        h = ACTS[act](v)
        if act != "none":
            err = 1.13 * err + 2.0 ** -20 * (1 + np.abs(v))
    return h, err
