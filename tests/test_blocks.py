"""Gated blocks, norms between blocks and log probabilities without a GPU: what the C ABI refuses before it touches a
device, sizes, and the formulas that the GPU tests compare with."""
import ctypes

import numpy as np
import pytest

import ponni_amd as P
from ponni_amd import _abi as A
from tests import numpy_blocks as N

FAKE = 1 << 40  # addresses that nothing reads: every call below is refused first
STEP = 1 << 32


def fake(k):
    return FAKE + k * STEP


def block(n_in=8, n_hidden=12, n_out=6, dtype=A.F32, act=None, **kw):
    act = act or P.Silu(n_hidden)
    b = A.Gated(n_in, n_hidden, n_out, dtype, act.desc(), fake(1), fake(2), fake(3), n_hidden, n_hidden, n_out, None, None, None)
    for k, v in kw.items():
        setattr(b, k, v)
    return b


def gated_forward(b, x=fake(4), ld_x=10, y=fake(5), ld_y=10, states=None, ld_states=10, columns=10, work=fake(6), size=1 << 30):
    return A.lib().ponni_gated_forward(ctypes.byref(b), x, ld_x, y, ld_y, states, ld_states, columns, work, size, None)


def error():
    return A.lib().ponni_last_error().decode()


@pytest.mark.parametrize("status,kw", [
    (A.PONNI_ERR_INVALID_MODEL, {"n_in": 0}), (A.PONNI_ERR_INVALID_MODEL, {"n_out": 65537}),
    (A.PONNI_ERR_UNSUPPORTED, {"dtype": A.F64}), (A.PONNI_ERR_UNSUPPORTED, {"act": P.Softmax(12)}),
    (A.PONNI_ERR_UNSUPPORTED, {"act": P.Elu(12)}), (A.PONNI_ERR_INVALID_MODEL, {"act": P.Relu(11)}),
    (A.PONNI_ERR_INVALID_ARGUMENT, {"up": None}), (A.PONNI_ERR_SHAPE, {"ld_gate": 11}),
    (A.PONNI_ERR_SHAPE, {"ld_down": A.GATED_MAX_COLUMNS + 1}), (A.PONNI_ERR_INVALID_ARGUMENT, {"gate_bias": fake(5)}),
])
def test_refused_blocks(status, kw):
    assert gated_forward(block(**kw)) == status and error()


@pytest.mark.parametrize("status,kw", [
    (A.PONNI_ERR_SHAPE, {"columns": 0}), (A.PONNI_ERR_SHAPE, {"columns": A.GATED_MAX_COLUMNS + 1}),
    (A.PONNI_ERR_INVALID_ARGUMENT, {"x": None}), (A.PONNI_ERR_INVALID_ARGUMENT, {"y": None}),
    (A.PONNI_ERR_SHAPE, {"ld_x": 9}), (A.PONNI_ERR_SHAPE, {"ld_y": 9}), (A.PONNI_ERR_SHAPE, {"states": fake(7), "ld_states": 9}),
    (A.PONNI_ERR_INVALID_ARGUMENT, {"work": None}), (A.PONNI_ERR_INVALID_ARGUMENT, {"work": fake(6) + 8}),
    (A.PONNI_ERR_SHAPE, {"size": 3}), (A.PONNI_ERR_INVALID_ARGUMENT, {"y": fake(4)}),
    (A.PONNI_ERR_INVALID_ARGUMENT, {"y": fake(4) + 40}), (A.PONNI_ERR_INVALID_ARGUMENT, {"work": fake(4)}),
    (A.PONNI_ERR_INVALID_ARGUMENT, {"states": fake(5) + 16}), (A.PONNI_ERR_INVALID_ARGUMENT, {"y": fake(3)}),
])
def test_refused_gated_calls(status, kw):
    assert gated_forward(block(), **kw) == status and error()


def test_refused_gated_gradients():
    L, b = A.lib(), block()

    def call(x=fake(4), ld_x=10, states=fake(5), ld_s=10, dy=fake(6), ld_dy=10, columns=10, g=None, size=1 << 30, **kw):
        g = A.GatedGradientArrays(fake(7), 10, fake(8), fake(9), fake(10), 12, 12, 6, None, None, None) if g is None else g
        for k, v in kw.items():
            setattr(g, k, v)
        return L.ponni_gated_backward(ctypes.byref(b), x, ld_x, states, ld_s, dy, ld_dy, columns, ctypes.byref(g), fake(11), size, None)

    assert call(columns=-1) == A.PONNI_ERR_SHAPE
    assert call(dy=None) == A.PONNI_ERR_INVALID_ARGUMENT and call(states=None) == A.PONNI_ERR_INVALID_ARGUMENT
    assert call(ld_gate=5) == A.PONNI_ERR_SHAPE and call(ld_s=5) == A.PONNI_ERR_SHAPE
    assert call(gate=fake(9)) == A.PONNI_ERR_INVALID_ARGUMENT and call(x=fake(7)) == A.PONNI_ERR_INVALID_ARGUMENT
    assert call(size=10) == A.PONNI_ERR_SHAPE
    assert L.ponni_gated_backward(ctypes.byref(b), fake(4), 10, fake(5), 10, fake(6), 10, 10, None, fake(11), 1 << 30, None) \
        == A.PONNI_ERR_INVALID_ARGUMENT
    assert L.ponni_gated_forward(None, fake(4), 10, fake(5), 10, None, 0, 10, fake(6), 1, None) == A.PONNI_ERR_INVALID_ARGUMENT
    assert L.ponni_gated_workspace_bytes(None, 10) == -1


@pytest.mark.parametrize("dtype", [A.F32, A.F16, A.BF16])
def test_gated_work_buffers_serve_fewer_columns(dtype):
    L = A.lib()
    for sizes in ((8, 12, 6), (333, 1001, 77), (1024, 4096, 1024)):
        b = block(*sizes, dtype=dtype, act=P.Relu(sizes[1]), ld_gate=sizes[1], ld_up=sizes[1], ld_down=sizes[2])
        for size in (L.ponni_gated_workspace_bytes, L.ponni_gated_backward_workspace_bytes):
            most = 0
            for columns in [*range(1, 300), 511, 512, 1000, 4000, 4097, 16_384, 70_001, 1_000_000]:
                need = size(ctypes.byref(b), columns)
                assert need >= most >= 0
                most = need
        assert L.ponni_gated_workspace_bytes(ctypes.byref(b), 0) == -1


def gated_needs(b, columns, es, states=True, backward=True, odd=()):
    """What a call needs: those arrays of `odd` have rows that do not all begin at multiples of 4 bytes."""
    ld = {k: columns + columns % 2 + (k in odd) for k in ("x", "states", "dy")}
    at = {"x": fake(4), "states": fake(5) if states else None, "dy": fake(6) if backward else None}
    return A.lib().ponni_gated_call_workspace_bytes(ctypes.byref(b), *(v for k in ("x", "states", "dy") for v in (at[k], ld[k])), columns)


@pytest.mark.parametrize("dtype,es", [(A.F32, 4), (A.F16, 2), (A.BF16, 2)])
def test_gated_work_buffers_hold_what_is_used(dtype, es):
    """Copies are counted where they are made: of 16-bit arrays at odd places, of pairs of other strides; room for h where
    there are no states."""
    L, columns = A.lib(), 32_768
    i, h, o = 2048, 8192, 1024
    b = block(i, h, o, dtype=dtype, act=P.Silu(h), ld_gate=h, ld_up=h, ld_down=o)
    sums = 2 * 64 << 20  # most of a product's parts, both of a pair
    forward, backward = h * columns * es, 2 * h * columns * es
    assert gated_needs(b, columns, es, states=False, backward=False) <= forward + sums
    assert gated_needs(b, columns, es, backward=False) <= sums
    assert gated_needs(b, columns, es) <= backward + sums
    for odd, rows in (("x", i), ("states", h), ("dy", o)):
        more = gated_needs(b, columns, es, odd=(odd,)) - gated_needs(b, columns, es)
        assert more == (0 if es == 4 else rows * columns * es)
    # any call: of 16 bits with copies of all three
    copies = 0 if es == 4 else (i + h + o) * columns * es
    assert L.ponni_gated_backward_workspace_bytes(ctypes.byref(b), columns) == gated_needs(b, columns, es) + copies
    # the weights: a 16-bit one at an odd place, and a pair of two strides, which is read at one
    down = block(i, h, o, dtype=dtype, act=P.Silu(h), ld_gate=h, ld_up=h, ld_down=o + 1)
    assert gated_needs(down, columns, es) - gated_needs(b, columns, es) == (0 if es == 4 else h * o * es)
    pair = block(i, h, o, dtype=dtype, act=P.Silu(h), ld_gate=h, ld_up=h + 2, ld_down=o)
    assert gated_needs(pair, columns, es) - gated_needs(b, columns, es) == 2 * i * h * es


@pytest.mark.parametrize("dtype,es", [(A.F32, 4), (A.F16, 2), (A.BF16, 2)])
def test_gated_work_buffers_of_calls(dtype, es):
    """No call needs more than its number of columns says, and one of few columns needs no room of the weights' size."""
    L = A.lib()
    for sizes in ((8, 12, 6), (333, 1001, 77), (1024, 4096, 1024), (20, 19, 33)):
        b = block(*sizes, dtype=dtype, act=P.Relu(sizes[1]), ld_gate=sizes[1], ld_up=sizes[1], ld_down=sizes[2])
        for columns in (1, 8, 9, 32, 33, 200, 512, 513, 4097, 70_001, 1_000_000):
            any_forward, any_backward = (size(ctypes.byref(b), columns) for size in
                                         (L.ponni_gated_workspace_bytes, L.ponni_gated_backward_workspace_bytes))
            for odd in ((), ("x",), ("x", "states"), ("x", "states", "dy")):
                for states in (False, True):
                    assert 0 <= gated_needs(b, columns, es, states, False, odd) <= any_forward
                assert 0 <= gated_needs(b, columns, es, odd=odd) <= any_backward
    b = block(1024, 4096, 1024, dtype=dtype, act=P.Relu(4096), ld_gate=4096, ld_up=4096, ld_down=1024)
    assert gated_needs(b, 1, es, states=False, backward=False) < 3 << 20
    assert gated_needs(b, 0, es) == -1


def residual_norm(n=8, columns=10, dtype=A.F32, after=A.NORM_RMS, before=A.NORM_LAYER, **kw):
    r = A.ResidualNormArrays(n, dtype, columns, A.Norm(after, 1e-5), A.Norm(before, 1e-5), 1.0, fake(1), columns, fake(2),
                             columns, None, None, columns, fake(3), columns, fake(4), columns, fake(5))
    for k, v in kw.items():
        setattr(r, k, v)
    return r


@pytest.mark.parametrize("status,kw", [
    (A.PONNI_ERR_SHAPE, {"n": 0}), (A.PONNI_ERR_SHAPE, {"n": 65537}), (A.PONNI_ERR_SHAPE, {"columns": 0}),
    (A.PONNI_ERR_SHAPE, {"columns": A.MAX_COLUMNS + 1}), (A.PONNI_ERR_UNSUPPORTED, {"dtype": A.F64}),
    (A.PONNI_ERR_INVALID_ARGUMENT, {"after": 3}), (A.PONNI_ERR_INVALID_ARGUMENT, {"before": A.NORM_NONE}),
    (A.PONNI_ERR_INVALID_ARGUMENT, {"x": None}), (A.PONNI_ERR_SHAPE, {"ld_x": 9}), (A.PONNI_ERR_SHAPE, {"ld_normed": 9}),
    (A.PONNI_ERR_INVALID_ARGUMENT, {"state": None, "normed": None}), (A.PONNI_ERR_INVALID_ARGUMENT, {"state": fake(1)}),
    (A.PONNI_ERR_INVALID_ARGUMENT, {"normed": fake(3) + 36}), (A.PONNI_ERR_INVALID_ARGUMENT, {"statistics": fake(4)}),
    (A.PONNI_ERR_INVALID_ARGUMENT, {"gate": fake(6), "feature_gate": fake(7)}),
    (A.PONNI_ERR_INVALID_ARGUMENT, {"feature_gate": fake(3) + 4}),
])
def test_refused_norms(status, kw):
    r = residual_norm(**kw)
    assert A.lib().ponni_residual_norm_forward(ctypes.byref(r), None) == status and error()


def test_refused_norm_parameters_and_gradients():
    L = A.lib()
    r = residual_norm()
    r.after.eps = -1.0
    assert L.ponni_residual_norm_forward(ctypes.byref(r), None) == A.PONNI_ERR_INVALID_ARGUMENT
    r.after.eps = float("nan")
    assert L.ponni_residual_norm_forward(ctypes.byref(r), None) == A.PONNI_ERR_INVALID_ARGUMENT
    r = residual_norm(after=A.NORM_NONE)
    r.after.weight = fake(9)
    assert L.ponni_residual_norm_forward(ctypes.byref(r), None) == A.PONNI_ERR_INVALID_ARGUMENT
    assert L.ponni_residual_norm_forward(None, None) == A.PONNI_ERR_INVALID_ARGUMENT

    def backward(r, size=1 << 30, **kw):
        g = A.ResidualNormGradientArrays(fake(20), 10, fake(21), 10, fake(22), 10, fake(23), 10)
        for k, v in kw.items():
            setattr(g, k, v)
        return L.ponni_residual_norm_backward(ctypes.byref(r), ctypes.byref(g), fake(30), size, None)

    assert backward(residual_norm(statistics=None)) == A.PONNI_ERR_INVALID_ARGUMENT
    assert backward(residual_norm(), size=0) == A.PONNI_ERR_SHAPE
    assert backward(residual_norm(), d_gate=fake(24), ld_d_gate=10) == A.PONNI_ERR_INVALID_ARGUMENT
    assert backward(residual_norm(before=A.NORM_NONE, normed=None)) == A.PONNI_ERR_INVALID_ARGUMENT
    assert backward(residual_norm(), d_x=fake(20)) == A.PONNI_ERR_INVALID_ARGUMENT
    assert backward(residual_norm(), ld_d_x=9) == A.PONNI_ERR_SHAPE
    assert L.ponni_residual_norm_workspace_bytes(0, A.F32, 5) == -1
    sizes = [L.ponni_residual_norm_workspace_bytes(100, A.F16, c) for c in (1, 2, 500, 10_000, 10 ** 9)]
    assert sizes == sorted(sizes) and sizes[0] > 0


@pytest.mark.parametrize("what", ["d_after_weight", "d_after_bias", "d_before_weight", "d_before_bias", "d_feature_gate"])
def test_refused_gradients_of_what_is_not_there(what):
    """A norm that the call has not, or one value per feature of a gate of every element: no gradient, so no array."""
    L = A.lib()

    def backward(r):
        g = A.ResidualNormGradientArrays(fake(20), 10, None, 0, fake(22), 10, fake(23), 10)
        setattr(g, what, fake(25))
        return L.ponni_residual_norm_backward(ctypes.byref(r), ctypes.byref(g), fake(30), 0, None)

    # what the call has passes, up to the work buffer that is missing
    there = {"gate": None, "feature_gate": fake(7)}
    assert backward(residual_norm(**there)) == A.PONNI_ERR_SHAPE and "workspace" in error()
    missing = {"gate": fake(6)} if what == "d_feature_gate" else \
        {"after": A.NORM_NONE} if "after" in what else {"before": A.NORM_NONE, "normed": None}
    assert backward(residual_norm(**missing)) == A.PONNI_ERR_INVALID_ARGUMENT and what in error()


def log_probs(classes=20, columns=10, dtype=A.F32, top_k=2, **kw):
    p = A.LogProbsArrays(classes, columns, fake(1), columns, dtype, top_k, *(fake(k) for k in range(2, 8)))
    for k, v in kw.items():
        setattr(p, k, v)
    return p


@pytest.mark.parametrize("status,kw", [
    (A.PONNI_ERR_SHAPE, {"classes": 0}), (A.PONNI_ERR_SHAPE, {"columns": 0}), (A.PONNI_ERR_UNSUPPORTED, {"dtype": A.F64}),
    (A.PONNI_ERR_SHAPE, {"classes": A.MAX_COLUMNS + 1}), (A.PONNI_ERR_INVALID_ARGUMENT, {"top_k": 17}),
    (A.PONNI_ERR_INVALID_ARGUMENT, {"top_k": -1}), (A.PONNI_ERR_INVALID_ARGUMENT, {"classes": 1}),
    (A.PONNI_ERR_INVALID_ARGUMENT, {"logits": None}), (A.PONNI_ERR_INVALID_ARGUMENT, {"entropy": None}),
    (A.PONNI_ERR_INVALID_ARGUMENT, {"targets": None}), (A.PONNI_ERR_INVALID_ARGUMENT, {"log_probs": None}),
    (A.PONNI_ERR_INVALID_ARGUMENT, {"top_classes": None}), (A.PONNI_ERR_SHAPE, {"ld": 9}),
    (A.PONNI_ERR_INVALID_ARGUMENT, {"entropy": fake(1)}), (A.PONNI_ERR_INVALID_ARGUMENT, {"top_classes": fake(7) + 4}),
])
def test_refused_log_probs(status, kw):
    p = log_probs(**kw)
    assert A.lib().ponni_log_probs_forward(ctypes.byref(p), fake(9), 1 << 30, None) == status and error()


def test_refused_log_prob_gradients_and_buffers():
    L = A.lib()

    def backward(p, g=fake(10), d=fake(11), ld=10):
        return L.ponni_log_probs_backward(ctypes.byref(p), g, None, None, d, ld, None)

    assert backward(log_probs(targets=None)) == A.PONNI_ERR_INVALID_ARGUMENT
    assert backward(log_probs(), d=None) == A.PONNI_ERR_INVALID_ARGUMENT
    assert backward(log_probs(), ld=9) == A.PONNI_ERR_SHAPE
    assert backward(log_probs(), d=fake(1) + 4) == A.PONNI_ERR_INVALID_ARGUMENT  # the logits, but not in their place
    assert backward(log_probs(), d=fake(1), ld=12) == A.PONNI_ERR_INVALID_ARGUMENT
    assert L.ponni_log_probs_forward(None, fake(9), 0, None) == A.PONNI_ERR_INVALID_ARGUMENT
    p = log_probs(classes=100_000, columns=1)
    assert L.ponni_log_probs_forward(ctypes.byref(p), fake(9), 16, None) == A.PONNI_ERR_SHAPE
    assert L.ponni_log_probs_forward(ctypes.byref(p), fake(9) + 4, 1 << 30, None) == A.PONNI_ERR_INVALID_ARGUMENT
    assert L.ponni_log_probs_workspace_bytes(10, 5, 11) == -1
    for classes in (100, 5000, 131_072):
        sizes = [L.ponni_log_probs_workspace_bytes(classes, c, 3) for c in (1, 2, 7, 64, 100, 5000, 10 ** 6)]
        assert sizes == sorted(sizes) and sizes[0] >= 0


def test_column_ranges_of_one_array_do_not_overlap():
    """They pass the checks of overlap, and what is refused is the work buffer that is missing."""
    b = block()
    assert gated_forward(b, x=fake(4), ld_x=64, y=fake(4) + 40, ld_y=64, size=0) == A.PONNI_ERR_SHAPE and "workspace" in error()
    r = A.lib().ponni_gated_forward(ctypes.byref(b), fake(4), 64, fake(4) + 36, 64, None, 0, 10, fake(6), 1 << 30, None)
    assert r == A.PONNI_ERR_INVALID_ARGUMENT and "overlaps" in error()


def test_python_refusals():
    import torch

    with pytest.raises(ValueError):
        P.BlockNorm("batch")
    with pytest.raises(ValueError):
        P.create_residual_norm(4, dtype="f64")
    with pytest.raises(P.PonniError):
        P.create_residual_norm(0)
    with pytest.raises(ValueError):
        P.log_probabilities(torch.zeros(3, 4))  # not on a GPU
    with pytest.raises(ValueError):
        P.create_gated_model(torch.zeros(3, 4), torch.zeros(3, 4), torch.zeros(4, 2), P.Silu(4))
    with pytest.raises(ValueError, match="act must be"):
        P.create_gated_model(torch.zeros(3, 4), torch.zeros(3, 4), torch.zeros(4, 2), "silu")


# -- the oracle's formulas by differences ---------------------------------------------------------


@pytest.mark.parametrize("act", N.ACTS)
def test_slopes(act):
    v = np.linspace(-4, 4, 801) + 0.0037
    d = (N.activation(act, v + 1e-6)[0] - N.activation(act, v - 1e-6)[0]) / 2e-6
    assert np.abs(d - N.activation(act, v)[1]).max() < 1e-8


@pytest.mark.parametrize("after,before,gate", [("rms", "layer", "full"), ("layer", "rms", "feature"), (None, "layer", None),
                                               ("layer", None, "full")])
def test_norm_gradients(after, before, gate):
    r = np.random.default_rng(1)
    n, b = 7, 3
    x, res = r.standard_normal((n, b)), r.standard_normal((n, b))
    g = None if gate is None else r.standard_normal((n, b) if gate == "full" else n)
    norms = [None if k is None else [k, r.standard_normal(n), r.standard_normal(n)] for k in (after, before)]
    ds, dn = r.standard_normal((n, b)), r.standard_normal((n, b)) if before else None

    def value(x, res, g, norms):
        out, _ = N.norm_forward(x, res, g, *norms, 0.7, 1e-5, "f32")
        return (ds * out["state"][0]).sum() + (0.0 if before is None else (dn * out["normed"][0]).sum())

    _, s = N.norm_forward(x, res, g, *norms, 0.7, 1e-5, "f32")
    got = N.norm_backward(s, *norms, ds, dn, 0.7, g, "f32")

    def moved(name, e):
        args = {"x": x, "residual": res, "gate": g}
        m = [None if k is None else list(k) for k in norms]
        if name in args:
            args[name] = args[name] + e
        else:
            k = m[name.startswith("before")]
            k[1 + name.endswith("bias")] = k[1 + name.endswith("bias")] + e
        return value(args["x"], args["residual"], args["gate"], m)

    for name, (v, _) in got.items():
        e = r.standard_normal(v.shape)
        d = (moved(name, 1e-6 * e) - moved(name, -1e-6 * e)) / 2e-6
        assert abs(d - (v * e).sum()) < 1e-6 * (1 + abs(d)), name
