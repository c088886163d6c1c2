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


# The kernels that SHAPES leaves out: 256 x 256 tiles, 4-bit states between layers of
# more features than a chain's kernel takes, its tiles of 128 columns.  A few hundred columns are checked.
LARGE = [
    # experts, widths, activations, columns, (dtype, weights)
    (3, (330, 1100), ("none",), 70_001, ("bf16", "same")),
    (3, (130, 1100), ("silu",), 70_001, ("f32", "same")),
    (3, (700, 1030), ("none",), 70_001, ("f16", "mx4")),
    (4, (129, 700, 600), ("tanh", "none"), 3001, ("bf16", "mx4")),
    (4, (129, 700, 600), ("gelu_erf", "none"), 3001, ("f16", "same")),
    (2, (100, 400, 500), ("sigmoid", "none"), 70_003, ("bf16", "same")),
    (2, (100, 400, 500), ("sigmoid", "none"), 70_003, ("f16", "mx4")),
    (2, (200, 256, 255), ("tanh", "none"), 40_003, ("f32", "same")),
    (9, (1000, 200), ("none",), 120, ("f16", "same")),
    (3, (1000, 200), ("none",), 90, ("bf16", "mx4")),
]


@pytest.mark.parametrize("E,widths,acts,C,types", LARGE)
def test_grouped_columns_large(cuda, E, widths, acts, C, types):
    import torch

    dtype, weights = types
    print(f"experts: E={E} {widths} {acts} C={C} {dtype} {weights}", flush=True)
    r = np.random.default_rng(C)
    model, params = networks(r, E, widths, acts, dtype, weights)
    offsets = group_sizes(r, E, C)
    x = torch.randn((widths[0], C), device=cuda, generator=torch.Generator(cuda).manual_seed(C)).to(torch_dtype(dtype))
    y = torch.full((widths[-1], C), 7.0, dtype=x.dtype, device=cuda)
    model.forward_batch_parallel(x, torch.from_numpy(offsets).to(cuda), y)
    for e in range(E):
        a, b = offsets[e], offsets[e + 1]
        if a < b:
            # the group's ends and some columns between
            cols = np.unique(np.concatenate([[a, b - 1], r.integers(a, b, 60)]))
            at = torch.from_numpy(cols).to(cuda)
            want, err = N.chain(params[e], host(x[:, at]), dtype, weights)
            close(host(y[:, at]), want, err, dtype)
    assert bool((y[:, offsets[-1]:] == 7.0).all())


@pytest.mark.parametrize("dtype,weights", [("f16", "same"), ("bf16", "same"), ("f16", "mx4"), ("bf16", "mx4")])
@pytest.mark.parametrize("E,widths,C", [(3, (130, 1100), 20_001), (11, (600, 650), 1701)])
@pytest.mark.parametrize("shift", [0, 1, 6])
def test_grouped_columns_in_aligned_rows(cuda, E, widths, C, shift, dtype, weights):
    """Rows a multiple of 16 bytes long hold the same bits as others, and the columns around the groups stay."""
    import torch

    r = np.random.default_rng(C + shift)
    model, params = networks(r, E, widths, ("none",), dtype, weights)
    offsets = group_sizes(r, E, C)
    at = torch.from_numpy(offsets).to(cuda)
    x = torch.randn((widths[0], C), device=cuda, generator=torch.Generator(cuda).manual_seed(C)).to(torch_dtype(dtype))
    results = []
    for pitch in ((C + 15) // 8 * 8, (C + 15) // 8 * 8 + 1):
        whole = torch.full((widths[-1], pitch), 7.0, dtype=x.dtype, device=cuda)
        y = whole[:, shift:shift + C]
        model.forward_batch_parallel(x, at, y)
        results.append(y.clone())
        y[:, :offsets[-1]] = 7.0
        assert bool((whole == 7.0).all())
    assert torch.equal(*results)
    for e in range(E):
        a, b = offsets[e], offsets[e + 1]
        if a < b:
            cols = np.unique(np.concatenate([np.arange(a, min(a + 9, b)), np.arange(max(b - 9, a), b), r.integers(a, b, 20)]))
            want, err = N.chain(params[e], host(x[:, torch.from_numpy(cols).to(cuda)]), dtype, weights)
            close(host(results[0][:, torch.from_numpy(cols).to(cuda)]), want, err, dtype)


def test_rows_beyond_four_gigabytes(cuda):
    """Byte offsets past 2^32 in the input, its rows and the output."""
    import torch

    r = np.random.default_rng(5)
    C, K, n = 2_200_000, 1024, 1040
    model, params = networks(r, 2, (K, n), ("none",), "bf16")
    x = torch.zeros((K, C), dtype=torch.bfloat16, device=cuda)
    cols = [0, 1, 1_099_999, 1_100_000, 2_097_152, C - 1]
    for c in cols:
        x[:, c] = torch.from_numpy(r.standard_normal(K)).to(cuda).to(x.dtype)
    offsets = torch.tensor([0, 1_100_000, C], dtype=torch.int32, device=cuda)
    y = model.forward_batch_parallel(x, offsets)
    for c in cols:
        want, err = N.chain(params[int(c >= 1_100_000)], host(x[:, c:c + 1]), "bf16")
        close(host(y[:, c:c + 1]), want, err, "bf16")
    # a column of zeros gives its expert's biases
    want, err = N.chain(params[1], np.zeros((K, 1)), "bf16")
    close(host(y[:, 2_000_000:2_000_001]), want, err, "bf16")


@pytest.mark.parametrize("dtype,weights", [("f32", "same"), ("bf16", "same"), ("f16", "mx4")])
@pytest.mark.parametrize("widths,C", [((37, 50), 20), ((37, 50, 41), 300), ((600, 700), 300)])
def test_non_finite_columns(cuda, dtype, weights, widths, C):
    """NaN and infinities stay in their columns, and meet no padding (37 features end inside a step)."""
    import torch

    r = np.random.default_rng(C)
    # (Relu, x > 0 ? x : 0, ends a NaN)
    model, params = networks(r, 2, widths, ("leaky_relu", "none")[-len(widths) + 1:], dtype, weights)
    x = r.standard_normal((widths[0], C))
    x[3, 1], x[widths[0] - 1, 2], x[0, C - 1] = np.nan, np.inf, -np.inf
    offsets = torch.tensor([0, C // 2, C], dtype=torch.int32, device=cuda)
    xt = tensor(x, dtype, cuda)
    got = host(model.forward_batch_parallel(xt, offsets))
    bad = [1, 2, C - 1]
    assert not np.isfinite(got[:, bad]).all(0).any()
    if weights == "same" and len(widths) == 2:
        w = params[0][0][0]
        assert np.array_equal(got[:, 2], np.where(w[-1] > 0, np.inf, -np.inf))  # inf * w and finite terms
    good = [c for c in range(C) if c not in bad]
    for e in range(2):
        cols = [c for c in good if (c >= C // 2) == bool(e)]
        want, err = N.chain(params[e], host(xt)[:, cols], dtype, weights)
        close(got[:, cols], want, err, dtype)


def test_empty_groups(cuda):
    import torch

    r = np.random.default_rng(1)
    for widths in ((20, 30), (20, 30, 10), (600, 700)):
        model, params = networks(r, 4, widths, ("none", "none")[-len(widths) + 1:], "f16")
        for C in (5, 400):
            x = tensor(r.standard_normal((widths[0], C)), "f16", cuda)
            y = torch.full((widths[-1], C), 7.0, dtype=torch.float16, device=cuda)
            model.forward_batch_parallel(x, torch.zeros(5, dtype=torch.int32, device=cuda), y)
            assert bool((y == 7.0).all())
            model.forward_batch_parallel(x, torch.tensor([0, 0, 0, C, C], dtype=torch.int32, device=cuda), y)
            want, err = N.chain(params[2], host(x), "f16")
            close(host(y), want, err, "f16")


def test_parameters_from_host_and_device(cuda):
    """The same model from numpy and torch arrays of any type, and new parameters after the first."""
    import torch

    r = np.random.default_rng(3)
    w, b = r.uniform(-1, 1, (3, 40, 50)).astype(np.float16), r.uniform(-1, 1, (3, 50)).astype(np.float16)
    x = tensor(r.standard_normal((40, 77)), "f16", cuda)
    offsets = torch.tensor([0, 30, 30, 77], dtype=torch.int32, device=cuda)
    want = None
    for make in (lambda a: a, lambda a: a.astype(np.float32), lambda a: a.astype(np.float64), torch.from_numpy,
                 lambda a: torch.from_numpy(a).to(cuda), lambda a: torch.from_numpy(a).double().to(cuda)):
        model = P.create_expert_model(P.ExpertMatvec(make(w)), P.ExpertBias(make(b)), dtype="f16")
        y = model.forward_batch_parallel(x, offsets)
        want = y if want is None else want
        assert torch.equal(y, want)
    model.set_layer_params(0, -w)
    model.set_layer_params(1, torch.from_numpy(-b).to(cuda))
    assert torch.equal(model.forward_batch_parallel(x, offsets), -want)


def test_4_bit_rows_as_input(cuda):
    """4-bit rows made beforehand give what the model makes of x itself."""
    import torch

    r = np.random.default_rng(8)
    for widths, C in (((100, 80), 12), ((100, 80, 30), 500), ((900, 700), 700), ((1100, 1100), 40_000)):
        model, _ = networks(r, 2, widths, ("relu", "none")[-len(widths) + 1:], "bf16", "mx4")
        x = torch.randn((widths[0], C), device=cuda).bfloat16()
        offsets = torch.tensor([0, C // 3, C], dtype=torch.int32, device=cuda)
        assert torch.equal(model.forward_batch_parallel(P.quantize_mx4(x), offsets),
                           model.forward_batch_parallel(x, offsets))


def test_dense_4_bit_layer(cuda):
    """One expert, no offsets: a plain dense product."""
    r = np.random.default_rng(9)
    for C in (1, 33, 200):
        model, params = networks(r, 1, (150, 90), ("none",), "f16", "mx4")
        x = tensor(r.standard_normal((150, C)), "f16", cuda)
        want, err = N.chain(params[0], host(x), "f16", "mx4")
        close(host(model.forward_batch_parallel(x)), want, err, "f16")


def test_own_routing(cuda):
    """A routing that a program made itself: an expert chosen twice by one sample, unsorted samples, unequal weights."""
    import torch

    r = np.random.default_rng(11)
    model, params = networks(r, 3, (30, 20), ("none",), "f32")
    x = tensor(r.standard_normal((30, 4)), "f32", cuda)
    i32 = dict(dtype=torch.int32, device=cuda)
    # expert 0: samples 3, 1, 1; expert 2: samples 0, 3; sample 2 has none
    routing = P.Routing(torch.tensor([[2, 0, -1, 0], [-1, 0, -1, 2]], **i32),
                        torch.tensor([[0.5, 2.0, 9.0, -1.0], [9.0, 0.25, 9.0, 3.0]], device=cuda),
                        torch.tensor([[3, 1, -1, 0], [-1, 2, -1, 4]], **i32),
                        torch.tensor([3, 1, 1, 0, 3, -1, -1, -1], **i32), torch.tensor([0, 3, 3, 5], **i32))
    got, xs = host(model.forward_mixture(x, routing)), host(x)
    f = [lambda c, e=e: N.chain(params[e], xs[:, c:c + 1], "f32")[0][:, 0] for e in range(3)]
    want = np.stack([0.5 * f[2](0), 2.25 * f[0](1), 0 * f[0](2), -f[0](3) + 3 * f[2](3)], 1)
    assert np.abs(got - want).max() <= 40 * 2.0 ** -24 * 4 * np.abs(xs).sum(0).max()
    with pytest.raises(ValueError):
        model.forward_mixture(x, P.Routing(routing.experts, routing.weights.double(), routing.slots, routing.source,
                                           routing.offsets))
    with pytest.raises(ValueError):
        model.forward_mixture(x, P.Routing(routing.experts, routing.weights, routing.slots, routing.source[:5],
                                           routing.offsets))


def mixture_model(r, dtype="bf16", weights="same"):
    experts, params = networks(r, 8, (64, 130, 48), ("silu", "none"), dtype, weights)
    w = r.uniform(-0.5, 0.5, (64, 8))
    return P.MixtureOfExperts(P.create_inference_model(P.Matvec(w), dtype=dtype), experts, top_k=2), params


@pytest.mark.parametrize("B", [1, 50, 3000])
def test_mixture_of_experts_model(cuda, B):
    """Router, routing, expert networks and the weighted sum together."""
    r = np.random.default_rng(B)
    model, params = mixture_model(r)
    x = tensor(r.standard_normal((64, B)), "bf16", cuda)
    y = model.forward_batch_parallel(x)
    scores = host(model.router.forward_batch_parallel(x))
    experts, w, *_ = N.route(scores, 2, "chosen")
    want, err = np.zeros(y.shape), np.zeros(y.shape)
    for e in range(8):
        j, b = np.nonzero(experts == e)
        if len(b):
            v, d = N.chain(params[e], host(x)[:, b], "bf16")
            want[:, b] += w[j, b] * v
            err[:, b] += w[j, b] * (d + 2.0 ** -8 * np.abs(v)) + 2.0 ** -20 * np.abs(v)
    close(host(y), want, err, "bf16")


@pytest.mark.parametrize("weights", ["same", "mx4"])
@pytest.mark.parametrize("B,hidden", [(3, 130), (700, 130), (700, 500), (700, 600)])
def test_graph_replays(cuda, B, hidden, weights):
    """Routing and a mixture captured in one graph, replayed with new inputs between
    the program's own work; two graphs of one model; the eager result each time."""
    import torch

    r = np.random.default_rng(B)
    experts, _ = networks(r, 8, (64, hidden, 48), ("silu", "none"), "bf16", weights)
    x = torch.empty((64, B), dtype=torch.bfloat16, device=cuda)
    s = torch.empty((8, B), device=cuda)

    def step():
        return experts.forward_mixture(x, P.route_experts(s, 2, "all"))

    def fill(seed):
        g = torch.Generator(cuda).manual_seed(seed)
        x.copy_(torch.randn(x.shape, device=cuda, generator=g))
        s.copy_(torch.randn(s.shape, device=cuda, generator=g))

    fill(0)
    step()
    torch.cuda.synchronize()
    graphs, outs = [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(step())
        graphs.append(g)
    for seed in range(1, 5):
        fill(seed)
        for g in graphs:
            g.replay()
        want = step()
        torch.cuda.synchronize()
        for out in outs:
            assert torch.equal(out, want)


def test_streams_and_dirty_workspaces(cuda):
    """Calls of one model on two streams at once, and work buffers full of NaN: the same results."""
    import ctypes
    import torch

    r = np.random.default_rng(4)
    for widths, dtype, weights in (((600, 700, 40), "bf16", "same"), ((64, 100, 40), "f16", "mx4"),
                                   ((700, 600, 64), "f16", "mx4")):
        model, _ = networks(r, 4, widths, ("tanh", "none"), dtype, weights)
        L, C = A.lib(), 2000
        offsets = torch.tensor([0, 300, 301, 1500, C], dtype=torch.int32, device=cuda)
        xs = [torch.randn((widths[0], C), device=cuda).to(torch_dtype(dtype)) for _ in range(2)]
        want = [model.forward_batch_parallel(x, offsets) for x in xs]
        torch.cuda.synchronize()
        streams = [torch.cuda.Stream() for _ in xs]
        for _ in range(5):
            got = []
            for x, stream in zip(xs, streams):
                with torch.cuda.stream(stream):
                    got.append(model.forward_batch_parallel(x, offsets))
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(got, want))
        need = L.ponni_experts_workspace_bytes(model._experts, C)
        work = torch.full((need + 64,), 255, dtype=torch.uint8, device=cuda)
        y = torch.empty_like(want[0])
        A.check(L.ponni_experts_forward(model._experts, xs[0].data_ptr(), C, offsets.data_ptr(), y.data_ptr(), C, C,
                                        work.data_ptr(), need, torch.cuda.current_stream().cuda_stream))
        torch.cuda.synchronize()
        assert torch.equal(y, want[0]) and bool((work[need:] == 255).all())
        routing = P.route_experts(torch.randn((4, C), device=cuda), 2)
        want = model.forward_mixture(xs[0], routing)
        need = L.ponni_experts_mixture_workspace_bytes(model._experts, 2, C)
        work = torch.full((need + 64,), 255, dtype=torch.uint8, device=cuda)
        arrays = routing.arrays()
        A.check(L.ponni_experts_forward_mixture(model._experts, xs[0].data_ptr(), C, ctypes.byref(arrays), y.data_ptr(),
                                                C, work.data_ptr(), need, torch.cuda.current_stream().cuda_stream))
        torch.cuda.synchronize()
        assert torch.equal(y, want) and bool((work[need:] == 255).all())


def test_refusals_of_tensors(cuda):
    """What the Python calls refuse before anything is launched."""
    import torch

    r = np.random.default_rng(2)
    model, _ = networks(r, 3, (20, 30), ("none",), "f16")
    x = torch.zeros((20, 8), dtype=torch.float16, device=cuda)
    offsets = torch.tensor([0, 2, 4, 8], dtype=torch.int32, device=cuda)
    bad = [
        lambda: model.forward_batch_parallel(x.float(), offsets),
        lambda: model.forward_batch_parallel(x[:19], offsets),
        lambda: model.forward_batch_parallel(x.cpu(), offsets),
        lambda: model.forward_batch_parallel(x.t().contiguous().t(), offsets),
        lambda: model.forward_batch_parallel(x, offsets.long()),
        lambda: model.forward_batch_parallel(x, offsets[:3]),
        lambda: model.forward_batch_parallel(x, offsets.cpu()),
        lambda: model.forward_batch_parallel(x, offsets, torch.empty((30, 7), dtype=x.dtype, device=cuda)),
        lambda: model.forward_batch_parallel(x, offsets, torch.empty((30, 8), device=cuda)),
        lambda: P.route_experts(torch.zeros((4, 4), device=cuda), 1, "some"),
        lambda: P.quantize_mx4(torch.zeros((4, 4), device=cuda, dtype=torch.int32)),
        lambda: P.Mx4(torch.zeros((2, 64), dtype=torch.uint8, device=cuda), torch.zeros((2, 3), dtype=torch.uint8,
                                                                                       device=cuda), 20).dequantize(),
    ]
    for call in bad:
        with pytest.raises(ValueError):
            call()
    refused = [
        (A.PONNI_ERR_INVALID_ARGUMENT, lambda: model.forward_batch_parallel(x)),  # three experts, no offsets
        (A.PONNI_ERR_SHAPE, lambda: model.forward_batch_parallel(x[:, :0], offsets)),
        (A.PONNI_ERR_UNSUPPORTED, lambda: model.forward_batch_parallel(P.quantize_mx4(x), offsets)),
        (A.PONNI_ERR_SHAPE, lambda: model.forward_batch_parallel(x[:1, :1].expand(20, 1), offsets)),  # stride 0
        (A.PONNI_ERR_UNSUPPORTED, lambda: P.route_experts(torch.zeros((4, 4), device=cuda, dtype=torch.float64), 1)),
        (A.PONNI_ERR_UNSUPPORTED, lambda: P.quantize_mx4(x).dequantize(torch.float64)),
        (A.PONNI_ERR_INVALID_ARGUMENT, lambda: P.route_experts(torch.zeros((4, 4), device=cuda), 5)),
        (A.PONNI_ERR_INVALID_ARGUMENT, lambda: P.route_experts(torch.zeros((4, 4), device=cuda), 0)),
        (A.PONNI_ERR_SHAPE, lambda: model.forward_mixture(x, P.route_experts(torch.zeros((4, 8), device=cuda), 1))),
    ]
    for status, call in refused:
        with pytest.raises(P.PonniError) as e:
            call()
        assert e.value.status == status
    wide = torch.zeros((50, 8), dtype=torch.float16, device=cuda)
    with pytest.raises(P.PonniError) as e:  # x and y share memory
        model.forward_batch_parallel(wide[:20], offsets, wide[19:49])
    assert e.value.status == A.PONNI_ERR_INVALID_ARGUMENT


# -- mixtures of many columns ------------------------------------------------------------

# Outputs of more than 64 MiB in 32 bits, held so all the same: no rounding between the chains and the weighted sum.
MIXTURES = [
    # experts, top_k, widths, activations, samples
    (2, 2, (40, 1001), ("none",), 9001),  # tiles of 128 columns
    (2, 2, (40, 70, 500), ("silu", "none"), 17_001),  # one kernel
    (5, 3, (130, 1100, 1030), ("tanh", "none"), 9334),  # tiles of 256 columns, gathered and between the layers
]


def check_mixture(model, params, x, routing, y, dtype, weights, samples):
    """The weighted sums of `samples` from the chains' values in 32 bits: those of N.chain, k products and sums,
    and the one rounding to dtype."""
    xs, experts, w = host(x[:, samples]), host(routing.experts[:, samples]).astype(int), host(routing.weights[:, samples])
    want, err = np.zeros((y.shape[0], len(samples))), np.zeros((y.shape[0], len(samples)))
    for e, p in enumerate(params):
        j, b = np.nonzero(experts == e)
        if len(b):
            v, d = N.chain(p, xs[:, b], dtype, weights)
            want[:, b] += w[j, b] * v
            err[:, b] += w[j, b] * (d + (routing.top_k + 1) * 2.0 ** -24 * (np.abs(v) + d))
    close(host(y[:, samples]), want, err, dtype)


@pytest.mark.parametrize("dtype,weights", [("f32", "same"), ("f16", "same"), ("bf16", "same"), ("f16", "mx4"),
                                           ("bf16", "mx4")])
@pytest.mark.parametrize("E,k,widths,acts,B", MIXTURES)
def test_large_mixture(cuda, E, k, widths, acts, B, dtype, weights):
    import torch

    print(f"mixture: E={E} k={k} {widths} B={B} {dtype} {weights}", flush=True)
    r = np.random.default_rng(B)
    model, params = networks(r, E, widths, acts, dtype, weights)
    g = torch.Generator(cuda).manual_seed(B)
    routing = P.route_experts(torch.randn((E, B), device=cuda, generator=g), k)
    x = torch.randn((widths[0], B), device=cuda, generator=g).to(torch_dtype(dtype))
    y = model.forward_mixture(x, routing)
    check_mixture(model, params, x, routing, y, dtype, weights,
                  torch.from_numpy(np.concatenate([[0, B - 1], r.integers(0, B, 150)])).to(cuda))


@pytest.mark.parametrize("dtype,weights", [("f16", "same"), ("bf16", "same"), ("f16", "mx4")])
@pytest.mark.parametrize("widths,B", [((40, 60), 50), ((40, 1001), 9001), ((40, 500), 17_001)])
def test_mixture_of_experts_that_cancel(cuda, widths, B, dtype, weights):
    """Two experts' outputs far above their weighted sum, in fp16 above the type's largest number: in a small batch
    and in one of more than 64 MiB of them."""
    import torch

    r = np.random.default_rng(B)
    size = 1e5 if dtype == "f16" else 100.0
    model, params = networks(r, 2, widths, ("none",), dtype, weights)
    bias = np.stack([np.full(widths[1], size), np.full(widths[1], -size)])
    model.set_layer_params(1, bias)
    params = [[(p[0][0], bias[e], "none")] for e, p in enumerate(params)]
    g = torch.Generator(cuda).manual_seed(B)
    scores = 0.2 * torch.randn((1, B), device=cuda, generator=g)
    routing = P.route_experts(torch.cat([scores, -scores]), 2)
    x = torch.randn((widths[0], B), device=cuda, generator=g).to(torch_dtype(dtype))
    y = model.forward_mixture(x, routing)
    # (the weights differ by tanh of the score: 0.2 * 4 gives 0.664, and 1e5 times that is beyond fp16's 65504)
    within = (routing.weights[0] - routing.weights[1]).abs() * size < 65000
    assert bool(torch.isfinite(y[:, within]).all())
    samples = torch.from_numpy(r.integers(0, B, 100)).to(cuda)
    check_mixture(model, params, x, routing, y, dtype, weights, samples[within[samples]])


# -- activations ---------------------------------------------------------------------------


def activation_error(act, v, dtype):
    """How far an activation's fp32 value may be, relative to it near zero and in the tails as elsewhere.

    A power 2^t is off by the rounding of t and an ulp (2^-23) of its own: |t| ln 2 times two roundings of t.
    fp32 models carry the rounding of t along (tanh: t <= 2.9 |x| only matters while 1 - |tanh| does, a
    relative 2^-21 at |x| = 0.55, where the form changes), then sum, reciprocal and quotient are a rounding or an ulp
    each: 2^-21, twice that for tanh.  GELU's argument is four roundings of 2u.  16-bit models round t
    (|t| ln 2 <= |x|), and tanh is x below 2^-7 (off by x^2 / 3 <= 2^-15), above that off by 2^-21 of one.
    A reciprocal below the normal range may be zero: 2^-126."""
    a = np.abs(v)
    two_u = 2 * np.sqrt(2 / np.pi) * (a + 0.044715 * a ** 3)
    if dtype == "f32":
        relative = {"tanh": 2.0 ** -20, "sigmoid": 2.0 ** -21, "silu": 2.0 ** -21,
                    "gelu": 2.0 ** -21 + two_u * 2.0 ** -22}[act]
    else:
        relative = {"tanh": 2.0 ** -14, "sigmoid": (a + 4) * 2.0 ** -23, "silu": (a + 4) * 2.0 ** -23,
                    "gelu": (two_u + 2) * 2.0 ** -22}[act]
    return relative * np.abs(N.ACTS[act](v)) + 2.0 ** -126 * (1 + a)


@pytest.mark.parametrize("dtype,weights", [("f32", "same"), ("f16", "same"), ("bf16", "same"), ("f16", "mx4"),
                                           ("bf16", "mx4")])
@pytest.mark.parametrize("act", ["tanh", "sigmoid", "silu", "gelu"])
@pytest.mark.parametrize("kernel,n_out,C", [("few columns", 1, 30), ("one kernel", 1, 400), ("tiles", 600, 400)])
def test_activations_of_every_kernel(cuda, kernel, n_out, C, act, dtype, weights):
    """Inputs from 1e-8 to 40 through weights of one: every size of batch and layer gives the activation that the
    type resolves."""
    import torch

    print(f"activation: {kernel} {act} {dtype} {weights}", flush=True)
    model = P.create_expert_model(P.ExpertMatvec(np.ones((1, 1, n_out))), ACT[act](n_out), dtype=dtype, weights=weights)
    v = np.geomspace(1e-8, 40, C // 2)
    x = tensor(np.concatenate([v, -v])[None], dtype, cuda)
    got = host(model.forward_batch_parallel(x))
    v = N.mx4(host(x))[0] if weights == "mx4" else host(x)
    with np.errstate(over="ignore"):
        want, err = N.ACTS[act](v), activation_error(act, v, dtype)
    close(got, np.broadcast_to(want, got.shape), err, dtype)


# -- parameters ----------------------------------------------------------------------------


@pytest.mark.parametrize("on_device", [False, True])
def test_new_parameters_wait_for_calls_in_flight(cuda, on_device):
    """A call that another stream has not run yet reads the parameters it was made with."""
    import torch

    r = np.random.default_rng(6)
    model, _ = networks(r, 2, (64, 600), ("none",), "f32")
    x = torch.randn((64, 300), device=cuda)
    offsets = torch.tensor([0, 100, 300], dtype=torch.int32, device=cuda)
    want = model.forward_batch_parallel(x, offsets)
    w = torch.from_numpy(r.standard_normal((2, 64, 600)))
    w = w.to(cuda) if on_device else w
    a = torch.randn((8192, 8192), device=cuda)
    torch.cuda.synchronize()
    with torch.cuda.stream(torch.cuda.Stream()):
        for _ in range(20):  # some 100 ms of work before the call
            a = a @ a
            a = a / a.abs().amax()
        got = model.forward_batch_parallel(x, offsets)
    model.set_layer_params(0, w)
    torch.cuda.synchronize()
    assert torch.equal(got, want)
    assert not torch.equal(model.forward_batch_parallel(x, offsets), want)


def test_parameters_beyond_a_launch_of_one_dimension(cuda):
    """More than 2^32 threads' worth of packed pieces: 1024 experts of 4096-4100."""
    import torch

    if torch.cuda.mem_get_info(cuda)[0] < 120 << 30:
        pytest.skip("needs 120 GiB of GPU memory")
    E, K, n = 1024, 4096, 4100
    w = torch.zeros((E, K, n), dtype=torch.float16, device=cuda)
    w[0, 0, 0], w[511, 17, 4099], w[E - 1, K - 1, n - 1] = 1.0, 2.0, 3.0
    model = P.create_expert_model(P.ExpertMatvec(w), dtype="f32")
    del w
    torch.cuda.empty_cache()
    x = torch.ones((K, 3), device=cuda)
    offsets = torch.zeros(E + 1, dtype=torch.int32, device=cuda)
    offsets[1:], offsets[512:], offsets[E:] = 1, 2, 3
    y = model.forward_batch_parallel(x, offsets)
    want = torch.zeros_like(y)
    want[0, 0], want[4099, 1], want[n - 1, 2] = 1.0, 2.0, 3.0
    assert torch.equal(y, want)


@pytest.mark.parametrize("on_device", [False, True])
@pytest.mark.parametrize("dtype,weights", [("f16", "same"), ("bf16", "same"), ("f16", "mx4"), ("f32", "same")])
def test_fp64_weights_are_rounded_once(cuda, dtype, weights, on_device):
    """fp64 weights next to the middle of two values of the operands' type, by less than fp32 resolves."""
    import torch

    # (4 bits: a scale of one from the first row, and values about 1.25)
    half, base = (0.25, 1.0) if weights == "mx4" else (N.EPS[dtype], 1.0)
    tiny = 2.0 ** -52
    w = np.zeros((1, 2, 6))
    w[0, 0] = 4.0
    w[0, 1] = [base + half - tiny, base + half, base + half + tiny, base - half / 2, -(base + half + tiny), 0.0]
    step = 2 * half
    want = np.array([base, base, base + step, base, -(base + step), 0.0])
    v = torch.from_numpy(w)
    model = P.create_expert_model(P.ExpertMatvec(v.to(cuda) if on_device else v), dtype=dtype, weights=weights)
    x = tensor(np.array([[0.0], [1.0]]), dtype, cuda)
    assert np.array_equal(host(model.forward_batch_parallel(x))[:, 0], want)
    if weights == "mx4":  # out of fp32's range: a block of NaN
        model.set_layer_params(0, w * 1e300)
        assert np.isnan(host(model.forward_batch_parallel(x))).all()


def test_new_parameters_in_one_dimension(cuda):
    r = np.random.default_rng(7)
    w, b = r.standard_normal((3, 20, 30)), r.standard_normal((3, 30))
    x = tensor(r.standard_normal((20, 9)), "f32", cuda)
    import torch

    offsets = torch.tensor([0, 2, 5, 9], dtype=torch.int32, device=cuda)
    want = P.create_expert_model(P.ExpertMatvec(w), P.ExpertBias(b)).forward_batch_parallel(x, offsets)
    model = P.create_expert_model(P.ExpertMatvec(np.zeros_like(w)), P.ExpertBias(np.zeros_like(b)))
    model.set_layer_params(0, w.reshape(-1))
    model.set_layer_params(1, torch.from_numpy(b).to(cuda).reshape(-1))
    assert torch.equal(model.forward_batch_parallel(x, offsets), want)


# Kernels that the shapes above leave out.
VARIANTS = [
    # experts, widths, activations, columns
    (64, (40, 1024), ("none",), 128),  # few columns, whole blocks of features: read in place
    (64, (40, 1024, 1030), ("tanh", "none"), 128),  # and rows between the layers
    (16, (300, 200, 130), ("silu", "none"), 400),  # few columns, tiles of 32 of them
    (40, (300, 900, 500), ("relu", "none"), 1000),  # both
    (8, (200, 500, 450), ("gelu", "none"), 100),  # few columns, whole blocks, of every type
    (3, (1100, 250, 60), ("silu", "none"), 1500),  # more input than one kernel takes for a chain
]


@pytest.mark.parametrize("dtype,weights", [("f32", "same"), ("f16", "same"), ("bf16", "same"), ("f16", "mx4"),
                                           ("bf16", "mx4")])
@pytest.mark.parametrize("E,widths,acts,C", VARIANTS)
def test_grouped_few_columns(cuda, E, widths, acts, C, dtype, weights):
    test_grouped_columns(cuda, E, widths, acts, C, dtype, weights)


@pytest.mark.parametrize("dtype,weights", [("f32", "same"), ("f16", "same"), ("bf16", "same"), ("f16", "mx4"),
                                           ("bf16", "mx4")])
@pytest.mark.parametrize("E,k,widths,acts,B", [(64, 2, (40, 1024, 1030), ("tanh", "none"), 64),
                                               (40, 2, (300, 900, 500), ("relu", "none"), 500),
                                               (16, 2, (300, 200, 130), ("silu", "none"), 200),
                                               (8, 2, (200, 500, 450), ("gelu", "none"), 50)])
def test_mixture_of_few_columns(cuda, E, k, widths, acts, B, dtype, weights):
    import torch

    print(f"mixture: E={E} k={k} {widths} B={B} {dtype} {weights}", flush=True)
    r = np.random.default_rng(B)
    model, params = networks(r, E, widths, acts, dtype, weights)
    g = torch.Generator(cuda).manual_seed(B)
    routing = P.route_experts(torch.randn((E, B), device=cuda, generator=g), k)
    x = torch.randn((widths[0], B), device=cuda, generator=g).to(torch_dtype(dtype))
    check_mixture(model, params, x, routing, model.forward_mixture(x, routing), dtype, weights,
                  torch.arange(B, device=cuda))


@pytest.mark.parametrize("E,widths,acts,C,types", [
    (3, (330, 1100, 1030), ("relu", "none"), 70_001, ("bf16", "same")),  # 256 x 256 tiles, rows between the layers
    (3, (330, 1100, 1030), ("relu", "none"), 70_001, ("f16", "same")),
    (3, (130, 1100, 1030), ("silu", "none"), 70_001, ("f32", "same")),
    (3, (700, 1100, 1030), ("silu", "none"), 70_001, ("f16", "mx4")),  # and 4-bit ones
    (3, (700, 1100, 1030), ("silu", "none"), 70_001, ("bf16", "mx4")),
])
def test_grouped_columns_large_states(cuda, E, widths, acts, C, types):
    test_grouped_columns_large(cuda, E, widths, acts, C, types)


# -- borders of the rules that choose kernels --------------------------------------------------


@pytest.mark.parametrize("normalize", ["chosen", "all"])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("E,k,B", [(128, 8, 64), (128, 8, 65), (128, 16, 256), (129, 8, 64), (129, 8, 65), (1024, 16, 256),
                                   (64, 4, 4096), (9, 2, 131_072)])
def test_routing_at_the_borders(cuda, E, k, B, dtype, normalize):
    test_routing(cuda, E, k, B, dtype, normalize)


@pytest.mark.parametrize("types", [("f16", "same"), ("bf16", "same"), ("f16", "mx4"), ("bf16", "mx4")])
def test_grouped_columns_in_wide_chain_tiles(cuda, types):
    """Tiles of 128 columns."""
    test_grouped_columns_large(cuda, 2, (100, 400, 500), ("tanh", "none"), 262_147, types)
