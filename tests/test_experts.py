"""Routing, expert networks and 4-bit rows without a GPU: the chains that a model
takes, the arguments that the C ABI refuses before it touches a device, sizes, and
the definitions that the GPU tests compare with."""
import ctypes

import numpy as np
import pytest

import ponni_amd as P
from ponni_amd import _abi as A
from tests import numpy_experts as N

FAKE = 1 << 40  # an address that nothing reads: every call below is refused first


def descs(*layers):
    return (A.LayerDesc * len(layers))(*[l.desc() for l in layers])


def create(layers, experts=2, dtype=A.F16, weights=A.WEIGHTS_SAME):
    e = ctypes.c_void_p()
    status = A.lib().ponni_experts_create(descs(*layers), len(layers), experts, dtype, weights, ctypes.byref(e))
    return status, e


def matvec(a, b):
    return P.Matvec(np.zeros((a, b)))


@pytest.mark.parametrize("layers", [
    [matvec(3, 4)],
    [matvec(3, 4), P.Bias(np.zeros(4)), P.Relu(4), matvec(4, 2), P.LeakyRelu(2, 0.1)],
    [matvec(3, 4), P.Gelu(4), matvec(4, 5), P.Bias(np.zeros(5)), P.Gelu(5, True), matvec(5, 5), P.Silu(5), matvec(5, 1),
     P.Sigmoid(1)],
])
def test_chains(layers):
    for dtype, weights in ((A.F32, 0), (A.F16, 0), (A.BF16, 0), (A.F16, 1), (A.BF16, 1)):
        status, e = create(layers, 3, dtype, weights)
        assert status == A.PONNI_OK
        L = A.lib()
        for i, l in enumerate(layers):
            assert L.ponni_experts_layer_param_count(e, i) == 3 * l.params.size
        assert L.ponni_experts_layer_param_count(e, len(layers)) == -1
        assert L.ponni_experts_workspace_bytes(e, 0) == -1
        assert L.ponni_experts_mixture_workspace_bytes(e, 4, 10) == -1  # more than the experts
        assert L.ponni_experts_workspace_bytes(e, 10) >= 0
        assert L.ponni_experts_mixture_workspace_bytes(e, 2, 10) > 0
        L.ponni_experts_destroy(e)


@pytest.mark.parametrize("status,layers,kw", [
    (A.PONNI_ERR_INVALID_MODEL, [P.Bias(np.zeros(3))], {}),
    (A.PONNI_ERR_INVALID_MODEL, [P.Relu(3), matvec(3, 3)], {}),
    (A.PONNI_ERR_INVALID_MODEL, [matvec(3, 4), P.Relu(5)], {}),
    (A.PONNI_ERR_INVALID_MODEL, [matvec(3, 4), matvec(5, 4)], {}),
    (A.PONNI_ERR_UNSUPPORTED, [matvec(3, 4), P.Relu(4), P.Tanh(4)], {}),
    (A.PONNI_ERR_UNSUPPORTED, [matvec(3, 4), P.Relu(4), P.Bias(np.zeros(4))], {}),
    (A.PONNI_ERR_UNSUPPORTED, [matvec(3, 4), P.Bias(np.zeros(4)), P.Bias(np.zeros(4))], {}),
    (A.PONNI_ERR_UNSUPPORTED, [matvec(3, 4), P.Softmax(4)], {}),
    (A.PONNI_ERR_UNSUPPORTED, [matvec(3, 4), P.Elu(4)], {}),
    (A.PONNI_ERR_UNSUPPORTED, [matvec(3, 4), P.LayerNorm(4)], {}),
    (A.PONNI_ERR_UNSUPPORTED, [matvec(3, 4)], {"dtype": A.F64}),
    (A.PONNI_ERR_UNSUPPORTED, [matvec(3, 4)], {"dtype": A.F32, "weights": 1}),
    (A.PONNI_ERR_INVALID_ARGUMENT, [matvec(3, 4)], {"weights": 2}),
    (A.PONNI_ERR_INVALID_ARGUMENT, [matvec(3, 4)], {"experts": 0}),
    (A.PONNI_ERR_INVALID_ARGUMENT, [matvec(3, 4)], {"experts": A.MAX_EXPERTS + 1}),
    (A.PONNI_ERR_INVALID_MODEL, [P.Layer(A.LAYER_MATVEC, 0, 4)], {}),
    (A.PONNI_ERR_INVALID_MODEL, [P.Layer(A.LAYER_MATVEC, 4, 65537)], {}),
])
def test_refused_chains(status, layers, kw):
    got, e = create(layers, **kw)
    assert got == status and not e.value and A.lib().ponni_last_error()


def test_null_arguments_of_create():
    L = A.lib()
    d = descs(matvec(2, 2))
    assert L.ponni_experts_create(d, 1, 1, A.F32, 0, None) == A.PONNI_ERR_INVALID_ARGUMENT
    e = ctypes.c_void_p()
    assert L.ponni_experts_create(None, 1, 1, A.F32, 0, ctypes.byref(e)) == A.PONNI_ERR_INVALID_ARGUMENT
    assert L.ponni_experts_create(d, 0, 1, A.F32, 0, ctypes.byref(e)) == A.PONNI_ERR_INVALID_ARGUMENT
    L.ponni_experts_destroy(None)
    assert L.ponni_experts_layer_param_count(None, 0) == -1
    assert L.ponni_experts_workspace_bytes(None, 5) == -1


def test_refused_forward_arguments():
    L = A.lib()
    _, e = create([matvec(4, 6)], 3, A.F16)
    _, q = create([matvec(4, 6)], 1, A.F16, 1)
    inv, shape, uns = A.PONNI_ERR_INVALID_ARGUMENT, A.PONNI_ERR_SHAPE, A.PONNI_ERR_UNSUPPORTED

    def fwd(e, x=FAKE, ld=8, off=FAKE, y=2 * FAKE, ldy=8, n=8, ws=3 * FAKE, size=1 << 20):
        return L.ponni_experts_forward(e, x, ld, off, y, ldy, n, ws, size, None)

    assert fwd(None) == inv
    assert fwd(e, n=0) == shape and fwd(e, n=-1) == shape and fwd(e, n=1_000_000_001, ld=1 << 31, ldy=1 << 31) == shape
    assert fwd(e, x=None) == inv and fwd(e, y=None) == inv
    assert fwd(e, off=None) == inv
    assert fwd(e, ld=7) == shape and fwd(e, ldy=7) == shape
    assert fwd(e) == inv and b"never set" in L.ponni_last_error()

    def fwd4(e, codes=FAKE, scales=2 * FAKE, y=3 * FAKE, n=8):
        return L.ponni_experts_forward_mx4(e, codes, scales, None, y, 8, n, 4 * FAKE, 1 << 20, None)

    assert fwd4(e) == uns
    assert fwd4(q, codes=None) == inv and fwd4(q, scales=None) == inv and fwd4(q, codes=FAKE + 8) == inv
    assert fwd4(q, n=0) == shape and fwd4(q) == inv

    def mix(e, k=2, b=8, experts=3, x=FAKE, y=2 * FAKE, ld=8, **arrays):
        r = A.RoutingArrays(experts, k, b, 0, arrays.get("weights", FAKE), arrays.get("slots", FAKE),
                            arrays.get("source", FAKE), arrays.get("offsets", FAKE))
        return L.ponni_experts_forward_mixture(e, x, ld, ctypes.byref(r), y, 8, 3 * FAKE, 1 << 20, None)

    assert mix(None) == inv and L.ponni_experts_forward_mixture(e, FAKE, 8, None, FAKE, 8, FAKE, 0, None) == inv
    assert mix(e, k=0) == inv and mix(e, k=4) == inv and mix(e, experts=0) == inv
    assert mix(e, b=0) == shape and mix(e, b=500_000_001, ld=1 << 30) == shape and mix(e, experts=4) == shape
    assert mix(e, x=None) == inv and mix(e, y=None) == inv and mix(e, ld=7) == shape
    for name in ("weights", "slots", "source", "offsets"):
        assert mix(e, **{name: None}) == inv
    assert mix(e) == inv and b"never set" in L.ponni_last_error()

    def put(layer=0, values=FAKE, dtype=A.F32, n=72):
        return L.ponni_experts_set_layer_params(e, layer, values, dtype, n, 1, None)

    assert L.ponni_experts_set_layer_params(None, 0, FAKE, A.F32, 72, 1, None) == inv
    assert put(layer=1) == inv and put(layer=-1) == inv and put(values=None) == inv and put(dtype=9) == inv
    assert put(n=71) == shape
    _, r = create([matvec(4, 6), P.Relu(6)])
    assert L.ponni_experts_set_layer_params(r, 1, FAKE, A.F32, 6, 1, None) == inv  # no parameters
    for h in (e, q, r):
        L.ponni_experts_destroy(h)


def test_refused_routing_arguments():
    L = A.lib()
    inv, shape, uns = A.PONNI_ERR_INVALID_ARGUMENT, A.PONNI_ERR_SHAPE, A.PONNI_ERR_UNSUPPORTED
    assert L.ponni_route_workspace_bytes(8, 2, 100) >= 0 and L.ponni_route_workspace_bytes(8, 2, 100_000) > 0
    for bad in ((0, 1, 5), (1025, 1, 5), (8, 0, 5), (8, 9, 5), (64, 17, 5), (8, 2, 0), (8, 2, 1 << 31)):
        assert L.ponni_route_workspace_bytes(*bad) == -1

    def route(E=8, k=2, b=1000, scores=FAKE, ld=1000, dtype=A.F32, norm=0, ws=FAKE, size=1 << 20, **arrays):
        names = ("experts", "weights", "slots", "source", "offsets")
        r = A.RoutingArrays(E, k, b, *[arrays.get(n, FAKE) for n in names])
        return L.ponni_route(scores, ld, dtype, norm, ctypes.byref(r), ws, size, None)

    assert L.ponni_route(FAKE, 8, A.F32, 0, None, FAKE, 1 << 20, None) == inv
    assert route(E=0) == inv and route(k=9) == inv and route(k=0) == inv and route(b=0) == shape
    assert route(scores=None) == inv and route(dtype=A.F64) == uns and route(norm=2) == inv and route(ld=999) == shape
    for name in ("experts", "weights", "slots", "source", "offsets"):
        assert route(**{name: None}) == inv
    assert route(ws=None) == inv and route(ws=FAKE + 4) == inv and route(size=10) == shape


def test_refused_mx4_arguments():
    L = A.lib()
    inv, shape, uns = A.PONNI_ERR_INVALID_ARGUMENT, A.PONNI_ERR_SHAPE, A.PONNI_ERR_UNSUPPORTED
    assert [L.ponni_mx4_code_bytes(k) for k in (1, 128, 129, 1000)] == [64, 64, 128, 512]
    assert [L.ponni_mx4_scale_bytes(k) for k in (1, 128, 129, 1000)] == [4, 4, 8, 32]
    assert L.ponni_mx4_code_bytes(0) == -1 and L.ponni_mx4_scale_bytes(-3) == -1

    def quantize(x=FAKE, ld=9, dtype=A.F32, k=40, n=9, codes=2 * FAKE, scales=3 * FAKE):
        return L.ponni_mx4_quantize(x, ld, dtype, k, n, codes, scales, None)

    assert quantize(x=None) == inv and quantize(codes=None) == inv and quantize(scales=None) == inv
    assert quantize(codes=2 * FAKE + 4) == inv and quantize(scales=3 * FAKE + 4) == inv
    assert quantize(k=0) == shape and quantize(k=65537) == shape and quantize(n=0) == shape and quantize(ld=8) == shape
    assert quantize(dtype=A.F64) == uns and quantize(codes=FAKE + 64) == inv and quantize(scales=2 * FAKE + 64) == inv
    assert L.ponni_mx4_dequantize(FAKE, 2 * FAKE, 40, 9, None, 9, A.F32, None) == inv
    assert L.ponni_mx4_dequantize(FAKE, 2 * FAKE, 40, 9, 3 * FAKE, 8, A.F32, None) == shape
    assert L.ponni_mx4_dequantize(FAKE, 2 * FAKE, 40, 9, 3 * FAKE, 9, A.F64, None) == uns


def test_refused_layers_in_python():
    with pytest.raises(ValueError):
        P.ExpertMatvec(np.zeros((3, 4)))
    with pytest.raises(ValueError):
        P.ExpertBias(np.zeros(4))
    with pytest.raises(ValueError):
        P.create_expert_model(P.ExpertMatvec(np.zeros((2, 3, 4))), weights="int4")
    with pytest.raises(P.PonniError):
        P.create_expert_model(P.Relu(3))
    with pytest.raises(P.PonniError):
        P.create_expert_model(P.ExpertMatvec(np.zeros((2, 3, 4))), P.ExpertBias(np.zeros((3, 4))))
    with pytest.raises(P.PonniError):
        P.create_expert_model(P.ExpertMatvec(np.zeros((2, 3, 4))), P.Relu(4), P.Elu(4))
    experts = P.create_expert_model(P.ExpertMatvec(np.zeros((2, 3, 4))))
    with pytest.raises(P.PonniError):
        P.MixtureOfExperts(P.create_inference_model(P.Matvec(np.zeros((3, 4)))), experts, 1)
    with pytest.raises(P.PonniError):
        P.MixtureOfExperts(P.create_inference_model(P.Matvec(np.zeros((5, 2)))), experts, 1)
    with pytest.raises(P.PonniError):
        P.MixtureOfExperts(P.create_inference_model(P.Matvec(np.zeros((3, 2))), dtype="bf16"), experts, 1)


def test_definition_of_4_bit_blocks():
    x = np.zeros((32, 1))
    x[:16, 0] = [4, .25, .75, 1.25, 1.75, 2.5, 3.5, 5, 6, 7, -.25, -.75, -1.25, -2.5, -3.5, -7.9]
    q, scale = N.mx4(x)
    assert scale[0, 0] == 127
    assert q[:16, 0].tolist() == [4, 0, 1, 1, 2, 2, 4, 4, 6, 6, 0, -1, -1, -2, -4, -6]
    for v in (1e-40, 1.0, 3.3e38):
        q, scale = N.mx4(np.full((5, 1), v))
        assert scale[0, 0] == max(0, int(np.floor(np.log2(v))) - 2 + 127)


def test_definition_of_routing():
    s = np.array([[1.0, -np.inf, 0.0], [2.0, -np.inf, 0.0], [1.0, -np.inf, np.nan]])
    experts, w, slots, source, offsets = N.route(s, 2, "chosen")
    assert experts.tolist() == [[1, -1, 0], [0, -1, 1]]
    assert np.allclose(w[:, 0], np.exp([0, -1]) / (1 + np.exp(-1))) and w[:, 2].tolist() == [0.5, 0.5]
    assert offsets.tolist() == [0, 2, 4, 4] and source.tolist() == [0, 2, 0, 2, -1, -1]
    assert slots.tolist() == [[2, -1, 1], [0, -1, 3]]


def test_layers_of_one_network_are_refused():
    """Their parameters belong to no expert: they would be left out."""
    w, b = np.ones((2, 3, 4)), np.full(4, 5.0)
    for layers in ([P.ExpertMatvec(w), P.Bias(b), P.Relu(4)], [P.Matvec(w[0]), P.ExpertBias(np.zeros((2, 4)))],
                   [P.ExpertMatvec(w), P.Relu(4), P.Matvec(np.zeros((4, 4)))]):
        with pytest.raises(P.PonniError) as e:
            P.create_expert_model(*layers)
        assert e.value.status == A.PONNI_ERR_INVALID_MODEL
    P.create_expert_model(P.ExpertMatvec(w), P.ExpertBias(np.zeros((2, 4))), P.Relu(4))


def test_overlapping_arrays_are_refused():
    """An output or work buffer on top of what a call reads, or of another output, by their last and first elements."""
    L = A.lib()
    names = ("experts", "weights", "slots", "source", "offsets")
    E, k, b = 8, 2, 1000
    size = {n: 4 * k * b for n in names} | {"offsets": 4 * (E + 1), "scores": 4 * E * b,
                                             "work": L.ponni_route_workspace_bytes(E, k, b)}

    def route(at):
        r = A.RoutingArrays(E, k, b, *[at[n] for n in names])
        return L.ponni_route(at["scores"], b, A.F32, 0, ctypes.byref(r), at["work"], size["work"], None)

    apart = {n: FAKE * (i + 1) for i, n in enumerate(size)}
    for one in size:
        for other in size:
            at = dict(apart)
            at[one] = apart[other] + (size[other] - 1) // 16 * 16
            if one != other:
                assert route(at) == A.PONNI_ERR_INVALID_ARGUMENT and b"overlap" in L.ponni_last_error(), (one, other)

    _, e = create([matvec(4, 6), P.Relu(6), matvec(6, 5)], 3, A.F16)
    read = {"x": 2 * 4 * 8, "weights": 64, "slots": 64, "source": 64, "offsets": 16}
    need = L.ponni_experts_mixture_workspace_bytes(e, 2, 8)
    assert need > 0

    def mix(at):
        r = A.RoutingArrays(3, 2, 8, 0, at["weights"], at["slots"], at["source"], at["offsets"])
        return L.ponni_experts_forward_mixture(e, at["x"], 8, ctypes.byref(r), at["y"], 8, at["work"], need, None)

    apart = {n: FAKE * (i + 1) for i, n in enumerate([*read, "y", "work"])}
    assert mix(apart) == A.PONNI_ERR_INVALID_ARGUMENT and b"never set" in L.ponni_last_error()
    for n, bytes_ in [*read.items(), ("y", 80)]:
        for written in ("y", "work"):
            if n != written:
                at = dict(apart)
                at[written] = apart[n] + (bytes_ - 1) // 16 * 16
                assert mix(at) == A.PONNI_ERR_INVALID_ARGUMENT and b"overlap" in L.ponni_last_error(), (n, written)
    need = L.ponni_experts_workspace_bytes(e, 8)
    for y, work in ((FAKE, 3 * FAKE), (2 * FAKE, FAKE)):
        status = L.ponni_experts_forward(e, 4 * FAKE, 8, FAKE, y, 8, 8, work, need, None)
        assert status == A.PONNI_ERR_INVALID_ARGUMENT and b"overlap" in L.ponni_last_error()
    L.ponni_experts_destroy(e)


def test_a_work_buffer_serves_smaller_batches():
    """The bytes of the largest batch that a program makes are enough for every smaller one."""
    L = A.lib()
    counts = sorted({int(round(1.3 ** i)) for i in range(50)} | {16, 17, 32, 33, 256, 257, 8192, 8193, 131072, 131073})

    for E, widths, weights in ((1, (500, 500), 0), (8, (500, 500, 500), 0), (8, (500, 500, 500), 1), (64, (40, 600), 0),
                               (64, (40, 2048, 30), 0), (4, (700, 900, 100), 1), (300, (16, 16, 16), 0)):
        _, e = create([matvec(a, b) for a, b in zip(widths, widths[1:])], E, A.BF16, weights)
        k = min(2, E)
        sizes, mixture_sizes = ([f(n) for n in counts] for f in (
            lambda n: L.ponni_experts_workspace_bytes(e, n), lambda n: L.ponni_experts_mixture_workspace_bytes(e, k, n)))
        assert sizes == sorted(sizes) and mixture_sizes == sorted(mixture_sizes)
        for i, n in enumerate(counts):  # the size as this batch's, and as a larger one's
            for size, mixture_size in ((sizes[i], mixture_sizes[i]), (sizes[-1], mixture_sizes[-1])):
                assert L.ponni_experts_forward(e, FAKE, n, 2 * FAKE, 3 * FAKE, n, n, 4 * FAKE, size, None) == \
                    A.PONNI_ERR_INVALID_ARGUMENT and b"never set" in L.ponni_last_error(), (E, widths, n, size)
                r = A.RoutingArrays(E, k, n, 0, 5 * FAKE, 6 * FAKE, 7 * FAKE, 8 * FAKE)
                assert L.ponni_experts_forward_mixture(e, FAKE, n, ctypes.byref(r), 3 * FAKE, n, 4 * FAKE, mixture_size,
                                                       None) == A.PONNI_ERR_INVALID_ARGUMENT
                assert b"never set" in L.ponni_last_error(), (E, widths, n, mixture_size)
        L.ponni_experts_destroy(e)
    sizes = [L.ponni_route_workspace_bytes(64, 2, n) for n in counts]
    assert sizes == sorted(sizes)


def test_new_parameters_of_another_shape_are_refused():
    """As many numbers in another order would be taken for weights of the layer's shape."""
    model = P.create_expert_model(P.ExpertMatvec(np.zeros((2, 3, 4))), P.ExpertBias(np.zeros((2, 4))))
    for i, shape in ((0, (2, 4, 3)), (0, (4, 3, 2)), (0, (6, 4)), (1, (4, 2)), (1, (2, 2, 2))):
        with pytest.raises(ValueError):
            model.set_layer_params(i, np.zeros(shape))
