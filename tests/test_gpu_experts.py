"""Routing, expert networks and 4-bit rows on the GPU against numpy in 64 bits
(numpy_experts.py, which bounds every element's distance): ties, scores that
rule experts out, samples without experts, empty groups, odd widths and columns,
strides and alignments, non-finite inputs, columns in no group, streams, graphs."""
import numpy as np
import pytest

import ponni_amd as P
from ponni_amd import _abi as A
from tests import numpy_experts as N

pytestmark = pytest.mark.gpu

DTYPES = ["f32", "f16", "bf16"]


def torch_dtype(name):
    import torch

    return {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[name]


def tensor(a, dtype, device, pad=0, shift=0):
    """a [rows, columns] on the GPU in a wider array, `shift` columns in."""
    import torch

    t = torch.full((a.shape[0], a.shape[1] + pad + shift), 7.0, dtype=torch_dtype(dtype), device=device)
    v = t[:, shift:shift + a.shape[1]]
    v.copy_(torch.from_numpy(np.ascontiguousarray(a)).to(device))
    return v


def host(t):
    return t.double().cpu().numpy()


# -- routing ---------------------------------------------------------------------------


def check_routing(r, scores, top_k, normalize):
    """Everything but the weights has to be equal; they are off by the roundings of
    the argument, exp, E sums and one quotient."""
    experts, w, slots, source, offsets = N.route(scores, top_k, normalize)
    assert np.array_equal(r.experts.cpu().numpy(), experts)
    assert np.array_equal(r.slots.cpu().numpy(), slots)
    assert np.array_equal(r.source.cpu().numpy(), source)
    assert np.array_equal(r.offsets.cpu().numpy(), offsets)
    finite = np.where(np.isfinite(scores), scores, 0.0)
    spread = np.abs(finite).max() * 2
    assert np.all(np.abs(host(r.weights) - w) <= w * (scores.shape[0] + spread + 8) * 2.0 ** -23 + 2.0 ** -126)


@pytest.mark.parametrize("normalize", ["chosen", "all"])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("E,k,B", [(1, 1, 1), (2, 2, 3), (5, 1, 255), (8, 2, 1000), (64, 4, 257), (65, 3, 513),
                                   (256, 8, 300), (1000, 16, 70), (1024, 5, 2), (6, 2, 4097), (5, 3, 70_001),
                                   (3, 2, 131_073)])
def test_routing(cuda, E, k, B, dtype, normalize):
    print(f"routing: E={E} k={k} B={B} {dtype} {normalize}", flush=True)
    r = np.random.default_rng(E * 1000 + B)
    s = r.integers(-6, 7, (E, B)) * 0.25 if dtype == "bf16" else r.standard_normal((E, B)) * 2  # (many ties)
    if B > 2:
        s[r.random((E, B)) < 0.3] = -np.inf
        s[:, r.integers(0, B, 2)] = -np.inf  # samples without an expert
        s[r.integers(0, E), r.integers(0, B)] = np.nan
    t = tensor(s, dtype, cuda, pad=B % 3, shift=B % 2)
    check_routing(P.route_experts(t, k, normalize), host(t), k, normalize)


def test_routing_of_infinities_and_equal_scores(cuda):
    s = np.zeros((6, 5))
    s[[1, 4], 1] = np.inf
    s[:, 2] = -np.inf
    s[3, 3] = 3e38
    s[0, 3] = -3e38
    for normalize in ("chosen", "all"):
        t = tensor(s, "f32", cuda)
        got = P.route_experts(t, 3, normalize)
        experts, w, *_ = N.route(host(t), 3, normalize)
        assert np.array_equal(got.experts.cpu().numpy(), experts)
        assert np.allclose(host(got.weights), w, rtol=2.0 ** -20)


# -- 4-bit rows ------------------------------------------------------------------------


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("K,C", [(1, 1), (31, 5), (32, 64), (33, 65), (100, 1003), (128, 7), (129, 200), (1000, 33)])
def test_mx4_rows(cuda, K, C, dtype):
    print(f"mx4: K={K} C={C} {dtype}", flush=True)
    r = np.random.default_rng(K + C)
    x = r.standard_normal((K, C)) * np.exp2(r.integers(-30 if dtype != "f16" else -8, 9, (K, 1)))
    x[r.random((K, C)) < 0.2] = 0.0
    x[:, :C // 4] = np.round(x[:, :C // 4] * 4) / 4  # (ties)
    t = tensor(x, dtype, cuda, pad=C % 3, shift=C % 2)
    q = P.quantize_mx4(t)
    want, scales = N.mx4(host(t))
    assert np.array_equal(q.scales.cpu().numpy()[:, :scales.shape[0]], scales.T)
    assert not q.scales[:, scales.shape[0]:].any()
    import torch

    assert np.array_equal(host(q.dequantize(torch.float32)), want)
    back = q.dequantize(t.dtype)
    assert torch.equal(back, torch.from_numpy(want).to(cuda).to(t.dtype))
    # what 4 bits hold is held exactly
    again = P.quantize_mx4(torch.from_numpy(want).float().to(cuda))
    assert np.array_equal(host(again.dequantize()), want)


def test_mx4_extremes(cuda):
    """Subnormal blocks, the largest floats, blocks with NaN and infinities, and every rounding border."""
    import torch

    x = np.zeros((64, 8), dtype=np.float32)
    x[0, 0], x[1, 0] = 2.0 ** -149, 2.0 ** -130
    x[0, 1], x[1, 1] = 3.4028234e38, -1.0e38
    x[3, 2], x[40, 2] = np.nan, 5.0
    x[3, 3], x[40, 3] = -np.inf, 5.0
    x[:16, 4] = [4, .25, .75, 1.25, 1.75, 2.5, 3.5, 5, 6, 7, -.25, -.75, -1.25, -2.5, -3.5, -7.9]
    x[:3, 5] = [2.0 ** -126, 2.0 ** -127, -2.0 ** -128]
    x[:2, 6] = [-0.0, 0.0]
    t = torch.from_numpy(x).to(cuda)
    q = P.quantize_mx4(t)
    want, scales = N.mx4(x.astype(np.float64))
    assert np.array_equal(q.scales.cpu().numpy()[:, :2], scales.T)
    assert np.array_equal(host(q.dequantize()), want, equal_nan=True)


# -- expert networks ---------------------------------------------------------------------

ACT = {"relu": P.Relu, "leaky_relu": lambda n: P.LeakyRelu(n, 0.1), "tanh": P.Tanh, "sigmoid": P.Sigmoid,
       "silu": P.Silu, "gelu": lambda n: P.Gelu(n, True), "gelu_erf": P.Gelu}


def networks(r, experts, widths, acts, dtype, weights="same", bias=True):
    """A model, and per expert its (W, b, activation)s as the model holds them."""
    import torch

    layers, params = [], []
    for a, b, act in zip(widths, widths[1:], acts):
        w = torch.from_numpy(r.uniform(-1, 1, (experts, a, b)) * np.sqrt(6.0 / (a + b))).to(torch_dtype(dtype))
        v = r.uniform(-0.2, 0.2, (experts, b)).astype(np.float32)
        layers.append(P.ExpertMatvec(w))
        if bias:
            layers.append(P.ExpertBias(v))
        if act != "none":
            layers.append(ACT[act](b))
        params.append((w.double().numpy(), v.astype(np.float64) if bias else None, act))
    model = P.create_expert_model(*layers, dtype=dtype, weights=weights)
    return model, [[(w[e], None if v is None else v[e], act) for w, v, act in params] for e in range(experts)]


def group_sizes(r, experts, columns):
    """Offsets of groups, some empty, that end before the last column."""
    cuts = np.sort(r.integers(0, columns + 1, experts - 1)) if experts > 1 else np.array([], dtype=np.int64)
    end = columns - min(3, columns - 1)
    offsets = np.minimum(np.concatenate([[0], cuts, [columns]]), end)
    if experts > 3:
        offsets[2] = offsets[1]
    return offsets.astype(np.int32)


def close(got, want, err, dtype):
    """Within the bound and one rounding to dtype."""
    tol = err + N.EPS[dtype] * (np.abs(want) + err) + N.TINY[dtype]
    bad = ~(np.abs(got - want) <= tol)
    assert not bad.any(), (int(bad.sum()), float((np.abs(got - want) / tol).max()))


SHAPES = [
    # experts, widths, activations, columns
    (1, (1, 1), ("none",), 1),
    (3, (5, 7), ("tanh",), 2),
    (4, (33, 64), ("none",), 17),
    (5, (33, 200, 17), ("tanh", "none"), 403),
    (8, (64, 65, 63, 130), ("relu", "silu", "gelu"), 1000),
    (70, (40, 24), ("sigmoid",), 500),
    (2, (129, 300, 1), ("leaky_relu", "gelu_erf"), 3001),
    (6, (16, 513), ("none",), 5),
]


@pytest.mark.parametrize("dtype,weights", [("f32", "same"), ("f16", "same"), ("bf16", "same"), ("f16", "mx4"),
                                           ("bf16", "mx4")])
@pytest.mark.parametrize("E,widths,acts,C", SHAPES)
def test_grouped_columns(cuda, E, widths, acts, C, dtype, weights):
    import torch

    print(f"experts: E={E} {widths} {acts} C={C} {dtype} {weights}", flush=True)
    r = np.random.default_rng(C)
    model, params = networks(r, E, widths, acts, dtype, weights, bias=C % 2 == 1)
    offsets = group_sizes(r, E, C)
    x = tensor(r.standard_normal((widths[0], C)), dtype, cuda, pad=C % 4, shift=C % 3)
    y = tensor(np.full((widths[-1], C), 7.0), dtype, cuda, pad=C % 5, shift=C % 2)
    whole = y._base
    model.forward_batch_parallel(x, torch.from_numpy(offsets).to(cuda), y)
    got, xs = host(y), host(x)
    for e in range(E):
        a, b = offsets[e], offsets[e + 1]
        if a < b:
            want, err = N.chain(params[e], xs[:, a:b], dtype, weights)
            close(got[:, a:b], want, err, dtype)
    assert np.all(got[:, offsets[-1]:] == 7.0)  # columns in no group
    if whole is not None:
        y.fill_(7.0)
        assert bool((whole == 7.0).all())  # and everything around them


@pytest.mark.parametrize("dtype,weights", [("f32", "same"), ("bf16", "same"), ("f16", "mx4")])
@pytest.mark.parametrize("E,k,widths,acts,B", [(1, 1, (3, 4), ("none",), 1), (4, 2, (33, 70, 20), ("silu", "none"), 3),
                                               (8, 3, (64, 128), ("none",), 130),
                                               (16, 4, (100, 257, 65), ("tanh", "relu"), 700)])
def test_mixture(cuda, E, k, widths, acts, B, dtype, weights):
    print(f"mixture: E={E} k={k} {widths} B={B} {dtype} {weights}", flush=True)
    r = np.random.default_rng(B)
    model, params = networks(r, E, widths, acts, dtype, weights)
    s = r.standard_normal((E, B))
    if B > 2:
        s[r.random((E, B)) < 0.3] = -np.inf
        s[:, 1] = -np.inf
    routing = P.route_experts(tensor(s, "f32", cuda), k)
    x = tensor(r.standard_normal((widths[0], B)), dtype, cuda, pad=B % 4, shift=B % 3)
    y = model.forward_mixture(x, routing)
    xs, experts, w = host(x), routing.experts.cpu().numpy(), host(routing.weights)
    want, err = np.zeros(y.shape), np.zeros(y.shape)
    for e in range(E):
        j, b = np.nonzero(experts == e)
        if len(b):
            v, d = N.chain(params[e], xs[:, b], dtype, weights)
            d = d + N.EPS[dtype] * (np.abs(v) + d) + N.TINY[dtype]  # the chain's output in the model's type
            want[:, b] += w[j, b] * v
            err[:, b] += w[j, b] * (d + (k + 1) * 2.0 ** -24 * (np.abs(v) + d))
    close(host(y), want, err, dtype)
    if B > 2:
        assert np.all(host(y)[:, 1] == 0.0)
