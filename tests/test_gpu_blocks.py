"""Gated blocks, norms between blocks and log probabilities on the GPU against numpy in 64 bits
(numpy_blocks.py, which bounds every element's distance), and their gradients against differences."""
import numpy as np
import pytest

import ponni_amd as P
from ponni_amd import _abi as A
from tests import numpy_blocks as N

pytestmark = pytest.mark.gpu

DTYPES = ["f32", "f16", "bf16"]


def torch_dtype(name):
    import torch

    return {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[name]


def tensor(a, dtype, device, pad=0, shift=0):
    """a [rows, columns] on the GPU in a wider array of NaN, `shift` columns in."""
    import torch

    t = torch.full((a.shape[0], a.shape[1] + pad + shift), float("nan"), dtype=torch_dtype(dtype), device=device)
    v = t[:, shift:shift + a.shape[1]]
    v.copy_(torch.from_numpy(np.ascontiguousarray(a)).to(device))
    return v


def vector(a, device, dtype="f32"):
    import torch

    return None if a is None else torch.from_numpy(np.ascontiguousarray(a)).to(device).to(torch_dtype(dtype))


def host(t):
    return None if t is None else t.double().cpu().numpy()


def close(got, want, bound, what):
    got = host(got) if not isinstance(got, np.ndarray) else got
    assert got.shape == want.shape, what
    same = (got == want) | (np.isnan(got) & np.isnan(want))
    with np.errstate(invalid="ignore"):
        off = np.where(same, 0.0, np.abs(got - want))
    worst = np.nanmax(np.where(same, 0.0, off / bound)) if off.size else 0.0
    assert np.all(same | (off <= bound)), f"{what}: {worst:.3g} of its bound"


# -- log probabilities ---------------------------------------------------------------------


def logits_of(r, c, b, masked, dtype):
    x = r.standard_normal((c, b)) * 3
    if dtype == "bf16":
        x = np.round(x * 4) / 4  # (many ties)
    if masked:
        x[r.random((c, b)) < masked] = -np.inf
        if b > 2:
            x[:, r.integers(0, b, 2)] = -np.inf  # columns without a class
    return x


def check_logp(cuda, c, b, k, dtype, masked=0.3, pad=0, shift=0, seed=0, targets=True):
    r = np.random.default_rng(seed + c * 31 + b)
    x = tensor(logits_of(r, c, b, masked, dtype), dtype, cuda, pad, shift)
    t = r.integers(-1, c + 1, b) if targets else None
    got = P.log_probabilities(x, None if t is None else vector(t, cuda).int(), top_k=k)
    want = N.log_probs(host(x), t, k)
    for name in ("log_normalizer", "entropy", "log_probs", "top_log_probs"):
        if getattr(got, name) is not None:
            close(getattr(got, name), *want[name], name)
    if k:
        assert np.array_equal(got.top_classes.cpu().numpy(), want["top_classes"])
    assert (got.log_probs is None) == (t is None) and (got.top_classes is None) == (k == 0)
    g = [r.standard_normal(b).astype(np.float32) for _ in range(3)]
    for use in ((1, 1, 1), (1, 0, 0), (0, 1, 0), (0, 0, 1)):
        if t is None and use[0]:
            continue
        gs = [v if u else None for u, v in zip(use, g)]
        d = got.backward(*(vector(v, cuda) for v in gs))
        close(d, *N.log_probs_backward(want, *(None if v is None else v.astype(float) for v in gs), dtype), f"d_logits {use}")
    return got, x


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("c,b,k", [(1, 1, 1), (1, 9, 0), (2, 3, 2), (10, 5000, 3), (64, 1030, 4), (65, 1, 16), (100, 7, 0),
                                   (257, 33, 5), (1000, 64, 8), (1263, 516, 3), (5003, 3, 16), (5003, 1, 8), (20_011, 70, 0),
                                   (300, 70_003, 0), (33, 100_001, 16), (130_001, 2, 4)])
def test_log_probabilities(cuda, c, b, k, dtype):
    print(f"log probabilities: {c} classes {b} columns top {k} {dtype}", flush=True)
    check_logp(cuda, c, b, k, dtype, pad=b % 3, shift=b % 2)


def test_log_probabilities_without_targets_or_masks(cuda):
    check_logp(cuda, 1000, 130, 0, "bf16", masked=0.0, targets=False)
    check_logp(cuda, 100, 1, 2, "f32", masked=0.0, targets=False)


def test_log_probabilities_hold_no_work_buffer(cuda):
    """What the results keep allocated is their own size (up to the allocator's blocks of 512 bytes)."""
    import torch

    for c, b, k in ((131_072, 1, 8), (65_536, 256, 0), (20_000, 40, 16)):
        x = torch.randn((c, b), device=cuda).bfloat16()
        targets = torch.zeros(b, dtype=torch.int32, device=cuda)
        P.log_probabilities(x, targets, k)
        torch.cuda.synchronize()
        before = torch.cuda.memory_allocated(cuda)
        r = P.log_probabilities(x, targets, k)
        assert torch.cuda.memory_allocated(cuda) - before <= 4 * b * (3 + 2 * k) + 512
        assert r.log_probs.shape == (b,)


def test_equal_logits(cuda):
    """Ties go to the lower class across lanes, waves and workgroups."""
    import torch

    for c, b in ((40_000, 1), (40_000, 3), (3000, 40), (50, 300)):
        x = torch.zeros((c, b), device=cuda)
        r = P.log_probabilities(x, None, 16)
        assert torch.equal(r.top_classes.cpu(), torch.arange(16, dtype=torch.int32)[:, None].expand(16, b))
        x[c // 2:] = 1.0
        r = P.log_probabilities(x.bfloat16(), None, 5)
        assert torch.equal(r.top_classes.cpu(), (c // 2 + torch.arange(5, dtype=torch.int32))[:, None].expand(5, b))
        # an early class is overtaken and stays before its equals
        x[7] = 1.0
        r = P.log_probabilities(x, None, 4)
        assert r.top_classes[:, 0].tolist() == [7, c // 2, c // 2 + 1, c // 2 + 2]
        x[c - 1] = 2.0
        r = P.log_probabilities(x, None, 4)
        assert r.top_classes[:, 0].tolist() == [c - 1, 7, c // 2, c // 2 + 1]


@pytest.mark.parametrize("c,b", [(50, 300), (5000, 4), (3000, 70)])
def test_non_finite_logits(cuda, c, b):
    """NaN and +inf stay in their column; the lowest finite value is no mask."""
    import torch

    r = np.random.default_rng(c)
    x = r.standard_normal((c, b))
    x[3, 0], x[c - 1, 1] = np.nan, np.inf
    x[:, 2] = -np.finfo(np.float32).max
    x[5, 2] = -np.inf
    t = torch.full((b,), 4, dtype=torch.int32, device=cuda)
    got = P.log_probabilities(tensor(x, "f32", cuda), t, 2)
    assert torch.isnan(got.log_normalizer[:2]).all() and torch.isnan(got.entropy[:2]).all()
    assert torch.isnan(got.log_probs[:2]).all() and torch.isnan(got.top_log_probs[:, :2]).all()
    assert int(got.top_classes[0, 1]) == c - 1 and int(got.top_classes[0, 0]) not in (3, -1)
    # equal classes of the lowest value: c - 1 of them
    assert abs(float(got.entropy[2]) - np.log(c - 1)) < 1e-5 * np.log(c)
    assert got.top_classes[:, 2].tolist() == [0, 1]
    want = N.log_probs(x[:, 3:].astype(np.float32).astype(float), np.full(b - 3, 4), 2)
    for name in ("log_normalizer", "entropy", "log_probs", "top_log_probs"):
        close(getattr(got, name)[..., 3:].contiguous(), *want[name], name)
    ones = torch.ones(b, device=cuda)
    d = got.backward(ones, ones, ones)
    assert torch.isnan(d[:, :2]).all() and not torch.isnan(d[:, 2:]).any()
    # the lowest float as a mask: its classes have no probability, whatever is left
    y = torch.full((c, 2), torch.finfo(torch.float32).min, device=cuda)
    y[9] = 0.0
    got = P.log_probabilities(y, t[:2], 1)
    assert torch.equal(got.log_normalizer, torch.zeros(2, device=cuda)) and torch.equal(got.entropy, torch.zeros(2, device=cuda))
    assert got.top_classes[0].tolist() == [9, 9]
    assert not torch.isnan(got.backward(ones[:2], ones[:2], ones[:2])).any()


def test_gradient_of_log_probabilities_in_place(cuda):
    """Into the logits' own array, into a column range of a wider one, which keeps its other columns."""
    import torch

    for dtype in DTYPES:
        got, x = check_logp(cuda, 700, 83, 0, dtype, seed=5)
        g = torch.randn(83, device=cuda)
        want = got.backward(g)
        wide = torch.full((700, 99), 7.0, dtype=x.dtype, device=cuda)
        got.backward(g, out=wide[:, 5:88])
        assert torch.equal(wide[:, 5:88], want)
        assert bool((wide[:, :5] == 7).all()) and bool((wide[:, 88:] == 7).all())
        assert got.backward(g, out=x) is x
        assert torch.equal(x, want)


@pytest.mark.parametrize("dtype", DTYPES)
def test_log_probabilities_of_column_ranges(cuda, dtype):
    """Logits and their gradients in wider arrays, at odd and even places: neighbours neither enter nor change."""
    import torch

    t = torch_dtype(dtype)
    for c, b, left, right in ((50, 300, 1, 6), (5000, 4, 3, 2), (700, 131, 8, 5)):
        a = torch.full((c, left + b + right), float("inf"), dtype=t, device=cuda)
        x = a[:, left:left + b]
        x.copy_(torch.randn((c, b), device=cuda) * 2)
        near = x.contiguous()
        targets = torch.randint(0, c, (b,), dtype=torch.int32, device=cuda)
        got, want = P.log_probabilities(x, targets, 3), P.log_probabilities(near, targets, 3)
        for name in ("log_probs", "entropy", "log_normalizer", "top_classes", "top_log_probs"):
            assert torch.equal(getattr(got, name), getattr(want, name)), name
        g = torch.randn(b, device=cuda)
        d = want.backward(g, g, g)
        assert got.backward(g, g, g, out=x) is x
        assert torch.equal(x, d)
        assert bool(torch.isinf(a[:, :left]).all()) and bool(torch.isinf(a[:, left + b:]).all())


def test_logits_beyond_four_gigabytes(cuda):
    """Columns of an array of 2.4e9 elements: offsets past 2^31 elements and 2^32 bytes."""
    import torch

    c, ld = 40_000, 60_000
    wide = torch.zeros((c, ld), dtype=torch.bfloat16, device=cuda)
    for b in (1, 100):
        x = wide[:, ld - b:]
        x.copy_(torch.randn((c, b), device=cuda))
        near = x.contiguous()
        targets = torch.arange(c - b, c, dtype=torch.int32, device=cuda)
        got, want = P.log_probabilities(x, targets, 5), P.log_probabilities(near, targets, 5)
        for name in ("log_probs", "entropy", "log_normalizer", "top_classes", "top_log_probs"):
            assert torch.equal(getattr(got, name), getattr(want, name)), name
        g = torch.randn(b, device=cuda)
        d = want.backward(g, g)
        assert torch.equal(got.backward(g, g, out=x), d)
    assert not wide[:, :ld - 100].any()


def test_log_probabilities_of_more_columns_than_a_launch_has(cuda):
    """Tiles of 32 fp32 columns by 256 threads, 2^32 threads a launch (65 classes: fewer take other tiles); the gradient into
    the logits' place."""
    import torch

    c, b = 65, 536_900_005
    torch.cuda.empty_cache()
    if torch.cuda.mem_get_info(cuda)[0] < 170e9:
        pytest.skip("150 GB of logits and results")
    x = torch.empty((c, b), device=cuda).normal_()
    targets = torch.randint(-1, c, (b,), dtype=torch.int32, device=cuda)
    g = torch.empty(b, device=cuda).normal_()
    border = (2 ** 32 // 256 - 1) * 32
    pieces = [slice(k, k + 1021) for k in (0, 2 ** 28, border - 512, b - 1021)]
    near = [(x[:, k].contiguous(), targets[k].contiguous(), g[k].contiguous()) for k in pieces]
    got = P.log_probabilities(x, targets)
    d = got.backward(g, out=x)
    for k, (x2, t2, g2) in zip(pieces, near):
        want = P.log_probabilities(x2, t2)
        for name in ("log_probs", "entropy", "log_normalizer"):
            # (sums in another order: a batch of few columns has tiles of its own)
            close(getattr(got, name)[k], *N.log_probs(host(x2), host(t2).astype(int), 0)[name], name)
            close(getattr(want, name), *N.log_probs(host(x2), host(t2).astype(int), 0)[name], name)
        close(d[:, k], *N.log_probs_backward(N.log_probs(host(x2), host(t2).astype(int), 0), host(g2), None, None, "f32"), "d_logits")
    del got, d, x
    torch.cuda.empty_cache()


def test_gradient_of_log_probabilities_by_differences(cuda):
    import torch

    r = np.random.default_rng(2)
    x = r.standard_normal((30, 6))
    t = vector(np.array([3, 0, 29, -1, 7, 8]), cuda).int()
    g = [r.standard_normal(6) for _ in range(3)]

    def value(v):
        want = N.log_probs(v, t.cpu().numpy(), 0)
        return sum((a * want[n][0]).sum() for a, n in zip(g, ("log_probs", "entropy", "log_normalizer")))

    got = host(P.log_probabilities(vector(x, cuda), t).backward(*(vector(v, cuda) for v in g)))
    for i, c in ((0, 0), (3, 0), (29, 2), (5, 3), (7, 4), (1, 5)):
        e = np.zeros_like(x)
        e[i, c] = 1e-5
        # (differences of second order: 1e-10 of third derivatives; fp32's roundings beside them)
        assert abs((value(x + e) - value(x - e)) / 2e-5 - got[i, c]) < 1e-5


# -- norms between blocks ----------------------------------------------------------------------


def check_norm(cuda, n, b, after, before, gate, residual, dtype, scale=0.7, eps=1e-5, pad=0, shift=0, seed=0, bias=True,
               weight=True):
    r = np.random.default_rng(seed + 7 * n + b)
    x = tensor(r.standard_normal((n, b)) * np.exp(0.5 * r.standard_normal((n, 1))) + 0.3, dtype, cuda, pad, shift)
    res = tensor(2 * r.standard_normal((n, b)) + 0.5, dtype, cuda, shift, pad) if residual else None
    gt = vector(r.standard_normal(n), cuda) if gate == "feature" else tensor(r.standard_normal((n, b)), dtype, cuda, pad) \
        if gate == "full" else None
    specs, norms = [], []
    for kind in (after, before):
        w = (1 + 0.3 * r.standard_normal(n)).astype(np.float32) if weight else None
        c = (0.2 * r.standard_normal(n)).astype(np.float32) if bias else None
        norms.append(None if kind is None else (kind, None if w is None else w.astype(float), None if c is None else c.astype(float)))
        specs.append(None if kind is None else P.BlockNorm(kind, vector(w, cuda), vector(c, cuda), eps))
    model = P.create_residual_norm(n, after=specs[0], before=specs[1], scale=scale, dtype=dtype)
    f = np.float32(scale).astype(float)
    want, s = N.norm_forward(host(x), host(res), host(gt), norms[0], norms[1], f, float(np.float32(eps)), dtype)
    state, normed, statistics = model.forward_with_statistics(x, res, gt)
    close(state, *want["state"], "state")
    assert (normed is None) == (before is None)
    if before is not None:
        close(normed, *want["normed"], "normed")
    again = model.forward_batch_parallel(x, res, gt)
    import torch

    assert torch.equal(again[0], state) and (normed is None or torch.equal(again[1], normed))
    ds, dn = tensor(r.standard_normal((n, b)), dtype, cuda, pad), tensor(r.standard_normal((n, b)), dtype, cuda, pad, shift)
    for d_state, d_normed in ((ds, dn), (None, dn), (ds, None)):
        if before is None and d_normed is not None:
            if d_state is None:
                continue
            d_normed = None
        d = model.backward(x, res, gt, statistics, d_state, d_normed)
        wanted = N.norm_backward(s, norms[0], norms[1], host(d_state), host(d_normed), f, host(gt), dtype)
        for name in ("x", "residual", "gate", "after_weight", "after_bias", "before_weight", "before_bias"):
            got = getattr(d, name)
            if got is None:
                continue
            if name not in wanted:  # no gradient comes this way
                assert not got.any()
                continue
            close(got, *wanted[name], f"d_{name} {d_state is not None} {d_normed is not None}")
    return model


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,b,after,before,gate,residual", [
    (1, 1, "rms", "rms", None, True), (1, 300, None, "rms", "feature", True), (5, 3, "layer", "layer", "full", True),
    (64, 1000, "rms", "rms", "feature", True), (100, 33, "layer", "rms", None, False), (333, 515, "layer", "layer", "full", True),
    (511, 8, None, "layer", "full", False), (1024, 2051, "rms", None, "feature", True), (1000, 9000, "rms", "layer", None, True),
    (4096, 1, "rms", "rms", None, True), (4096, 37, None, "rms", None, True), (4097, 19, "layer", "rms", "full", True),
    (20_000, 2, "rms", "layer", "feature", True), (9000, 40, "layer", "layer", None, True), (700, 4, None, None, "full", True),
    (2048, 20, "rms", "rms", "full", False)])
def test_norms(cuda, n, b, after, before, gate, residual, dtype):
    print(f"norms: n={n} b={b} {after} {before} {gate} {residual} {dtype}", flush=True)
    check_norm(cuda, n, b, after, before, gate, residual, dtype, pad=b % 3, shift=b % 2)


@pytest.mark.parametrize("n,b,after,before,gate,residual,dtype", [
    # 16 bits: tiles of 64 columns, 516 of them; at most 8 rows of 64 threads' (4 beside a full gate or two layer norms) held
    (500, 33_003, "rms", "rms", None, True, "bf16"), (300, 33_003, "layer", "layer", None, True, "f16"),
    (250, 33_003, "layer", "rms", "full", True, "bf16"), (530, 33_003, None, "rms", "feature", True, "f16"),
    (270, 33_003, "rms", "layer", "full", False, "f16"),
    # fp32: tiles of 32 columns, 532 and more; held up to 512 rows at 128 bytes, read again from 1025 (2049 with a norm after)
    (500, 17_003, "rms", "layer", "full", True, "f32"), (1030, 17_003, None, "layer", "feature", True, "f32"),
    (2060, 16_390, "rms", "rms", None, True, "f32")])
def test_norms_of_more_tiles_than_workgroups(cuda, n, b, after, before, gate, residual, dtype):
    """The gradients' 512 workgroups add weights' gradients over several tiles, in registers and where columns are read
    again, 128 bytes of a row across, with a last tile that is not whole.  (In pieces of columns: a term of a sum passes
    fewer additions here, 16 in a lane, 6 across lanes and 48 behind the workgroups, than the pieces' bounds count.)"""
    import torch

    print(f"norms: n={n} b={b} {after} {before} {gate} {residual} {dtype}", flush=True)
    assert b > 512 * (32 if dtype == "f32" else 64)
    torch.manual_seed(n)
    t = torch_dtype(dtype)

    def normal(*shape, scale=1.0, shift=0.0):
        return (torch.randn(shape, device=cuda) * scale + shift)

    x, ds, dn = (normal(n, b).to(t) for _ in range(3))
    res = normal(n, b, scale=2.0, shift=0.5).to(t) if residual else None
    g = {"full": normal(n, b).to(t), "feature": normal(n), None: None}[gate]
    w = [None if k is None else (k, normal(n, scale=0.3, shift=1.0), normal(n, scale=0.2)) for k in (after, before)]
    model = P.create_residual_norm(n, *(None if k is None else P.BlockNorm(*k) for k in w), scale=0.7, dtype=dtype)
    state, normed, statistics = model.forward_with_statistics(x, res, g)
    d = model.backward(x, res, g, statistics, ds, dn)
    norms = [None if k is None else (k[0], host(k[1]), host(k[2])) for k in w]
    f, eps = float(np.float32(0.7)), float(np.float32(1e-5))
    sums, step = {}, 509
    for c in range(0, b, step):
        at = slice(c, c + step)
        px, pr, pds, pdn = (None if v is None else host(v[:, at]) for v in (x, res, ds, dn))
        pg = host(g[:, at]) if gate == "full" else host(g)
        want, s = N.norm_forward(px, pr, pg, *norms, f, eps, dtype)
        close(state[:, at], *want["state"], "state")
        close(normed[:, at], *want["normed"], "normed")
        wanted = N.norm_backward(s, *norms, pds, pdn, f, pg, dtype)
        for name, (v, e) in wanted.items():
            got = getattr(d, name)
            if got is not None and got.dim() == 2:
                close(got[:, at], v, e, f"d_{name}")
            elif got is not None:
                total = sums.setdefault(name, [0.0, 0.0])
                total[0], total[1] = total[0] + v, total[1] + e
    assert len(sums) == 2 * sum(k is not None for k in w) + (gate == "feature")
    for name, (v, e) in sums.items():
        close(getattr(d, name), v, e, f"d_{name}")


def test_gradients_of_weights_that_are_ones(cuda):
    """A norm without a weight or bias has their gradients all the same, at ones and zeros; and a gate of ones."""
    import ctypes

    import torch

    n, b = 77, 300
    x, ds, dn = (torch.randn((n, b), device=cuda) for _ in range(3))
    ones, zeros = torch.ones(n, device=cuda), torch.zeros(n, device=cuda)
    given = P.create_residual_norm(n, P.BlockNorm("layer", ones, zeros), P.BlockNorm("rms", ones, zeros))
    bare = P.create_residual_norm(n, P.BlockNorm("layer"), P.BlockNorm("rms"))
    _, _, statistics = given.forward_with_statistics(x, x, ones)
    want = given.backward(x, x, ones, statistics, ds, dn)
    r = bare._arrays(x, x, None)
    r.statistics = statistics.data_ptr()
    out = {k: torch.empty(n, device=cuda) for k in ("feature_gate", "after_weight", "after_bias", "before_weight", "before_bias")}
    g = A.ResidualNormGradientArrays(ds.data_ptr(), b, dn.data_ptr(), b)
    for k, v in out.items():
        setattr(g, "d_" + k, v.data_ptr())
    need = A.lib().ponni_residual_norm_workspace_bytes(n, r.dtype, b)
    work = torch.full((need,), 255, dtype=torch.uint8, device=cuda)  # (NaN)
    assert A.lib().ponni_residual_norm_backward(ctypes.byref(r), ctypes.byref(g), work.data_ptr(), need,
                                                torch.cuda.current_stream().cuda_stream) == 0
    for k, v in out.items():
        assert torch.equal(v, getattr(want, "gate" if k == "feature_gate" else k)), k


def test_norms_without_weights(cuda):
    check_norm(cuda, 120, 50, "rms", "layer", None, True, "f16", weight=False, bias=False)
    check_norm(cuda, 120, 50, "layer", "rms", "full", False, "f32", weight=True, bias=False, scale=-1.0)


@pytest.mark.parametrize("dtype", DTYPES)
def test_norms_of_the_most_features(cuda, dtype):
    for b in (1, 3, 20):
        check_norm(cuda, 65536, b, "layer", "rms", "full", True, dtype)


def test_norm_of_constant_columns(cuda):
    """Nothing is left to normalise: a layer norm gives its bias, zeros under eps."""
    import torch

    n, b = 96, 11
    x = torch.full((n, b), 3.0, device=cuda)
    bias = torch.randn(n, device=cuda)
    model = P.create_residual_norm(n, before=P.BlockNorm("layer", None, bias))
    _, normed, statistics = model.forward_with_statistics(x)
    assert torch.equal(normed, bias[:, None].expand(n, b))
    zero = P.create_residual_norm(n, before=P.BlockNorm("rms")).forward_batch_parallel(torch.zeros_like(x))[1]
    assert not zero.any()
    d = model.backward(x, None, None, statistics, None, torch.randn_like(x))
    assert torch.isfinite(d.x).all()


def test_non_finite_columns_of_norms(cuda):
    import torch

    for n, b in ((64, 40), (5000, 24), (300, 3)):
        x = torch.randn((n, b), device=cuda)
        model = P.create_residual_norm(n, after=P.BlockNorm("rms"), before=P.BlockNorm("layer"))
        want = model.forward_batch_parallel(x, x)
        x2 = x.clone()
        x2[1, 1], x2[2, 2] = float("nan"), float("inf")
        got = model.forward_batch_parallel(x2, x)
        for g, w in zip(got, want):
            assert torch.equal(g[:, [0, *range(3, b)]], w[:, [0, *range(3, b)]])
        assert torch.isnan(got[1][:, 1]).all() and torch.isnan(got[1][:, 2]).any()


def test_norm_rows_beyond_four_gigabytes(cuda):
    """Byte offsets past 2^32."""
    import torch

    n, b = 1100, 2_200_000
    x = torch.zeros((n, b), dtype=torch.bfloat16, device=cuda)
    cols = [0, 1_500_000, b - 1]
    x[:, cols] = torch.randn((n, 3), device=cuda).bfloat16()
    model = P.create_residual_norm(n, before=P.BlockNorm("rms"), dtype="bf16")
    state, normed = model.forward_batch_parallel(x)
    want = model.forward_batch_parallel(x[:, cols].contiguous())
    assert torch.equal(state[:, cols], want[0]) and torch.equal(normed[:, cols], want[1])


@pytest.mark.parametrize("dtype,b", [("f32", 268_500_003), ("bf16", 536_900_005)])
def test_norms_of_more_columns_than_a_launch_has(cuda, dtype, b):
    """Tiles of 32 columns (16 bits: 64) by 512 threads, 2^32 threads a launch: a column's results are those of the column
    among few, on either side of the border and at the end."""
    import torch

    t, n = torch_dtype(dtype), 2
    x, res = (torch.empty((n, b), dtype=t, device=cuda).normal_() for _ in range(2))
    model = P.create_residual_norm(n, after=P.BlockNorm("layer"), before=P.BlockNorm("rms"), scale=0.5, dtype=dtype)
    state, normed, statistics = model.forward_with_statistics(x, res)
    d = model.backward(x, res, None, statistics, None, normed)
    border = (2 ** 32 // 512 - 1) * (32 if dtype == "f32" else 64)
    for c in (0, 2 ** 27, border - 512, b - 1021):
        near = x[:, c:c + 1021].contiguous(), res[:, c:c + 1021].contiguous()
        want = model.forward_with_statistics(*near)
        for got, w in zip((state, normed, statistics), want):
            assert torch.equal(got[:, c:c + 1021], w)
        wanted = model.backward(*near, None, want[2], None, want[1])
        assert torch.equal(d.x[:, c:c + 1021], wanted.x) and torch.equal(d.residual[:, c:c + 1021], wanted.residual)
    assert not torch.equal(state[:, border - 512:border], state[:, border:border + 512])


def test_norm_results_leave_their_neighbours(cuda):
    """Column ranges of wider arrays for every result."""
    import ctypes

    import torch

    for dtype in DTYPES:
        t = torch_dtype(dtype)
        for n, b, left, right in ((33, 5, 3, 4), (70, 131, 8, 3), (5000, 41, 1, 7)):
            w = [1 + torch.randn(n, device=cuda) / 4 for _ in range(2)]
            model = P.create_residual_norm(n, after=P.BlockNorm("rms", w[0]), before=P.BlockNorm("layer", w[1]), scale=0.5,
                                           dtype=dtype)
            x, res, gate, ds, dn = (torch.randn((n, b), device=cuda).to(t) for _ in range(5))
            want = model.forward_with_statistics(x, res, gate)
            wanted = model.backward(x, res, gate, want[2], ds, dn)

            def wide():
                a = torch.full((n + 1, left + b + right), 7.0, dtype=t, device=cuda)
                return a, a[:n, left:left + b]

            def same(a, v, want):
                rest = torch.ones_like(a, dtype=torch.bool)
                rest[:n, left:left + b] = False
                return torch.equal(v, want) and bool((a[rest] == 7.0).all())

            r = model._arrays(x, res, gate)
            (sa, sv), (na, nv) = wide(), wide()
            statistics = torch.empty((4, b), device=cuda)
            r.state, r.normed, r.statistics = sv.data_ptr(), nv.data_ptr(), statistics.data_ptr()
            r.ld_state = r.ld_normed = left + b + right
            stream = torch.cuda.current_stream().cuda_stream
            L = A.lib()
            assert L.ponni_residual_norm_forward(ctypes.byref(r), stream) == 0
            assert same(sa, sv, want[0]) and same(na, nv, want[1]) and torch.equal(statistics, want[2])
            r = model._arrays(x, res, gate)
            r.statistics = statistics.data_ptr()
            g = A.ResidualNormGradientArrays()
            g.d_state, g.ld_d_state, g.d_normed, g.ld_d_normed = ds.data_ptr(), b, dn.data_ptr(), b
            out = [wide() for _ in range(3)]
            for name, (a, v) in zip(("d_x", "d_residual", "d_gate"), out):
                setattr(g, name, v.data_ptr())
                setattr(g, "ld_" + name, a.stride(0))
            need = L.ponni_residual_norm_workspace_bytes(n, r.dtype, b)
            work = torch.full((need + 64,), 255, dtype=torch.uint8, device=cuda)  # (NaN)
            work[need:] = 7
            assert L.ponni_residual_norm_backward(ctypes.byref(r), ctypes.byref(g), work.data_ptr(), need, stream) == 0
            for (a, v), v2 in zip(out, (wanted.x, wanted.residual, wanted.gate)):
                assert same(a, v, v2)
            assert bool((work[need:] == 7).all())


# -- gated blocks -------------------------------------------------------------------------


def act_layer(name, n):
    return {"relu": P.Relu, "leaky_relu": lambda n: P.LeakyRelu(n, 0.1), "silu": P.Silu, "gelu": lambda n: P.Gelu(n, True),
            "gelu_erf": P.Gelu, "tanh": P.Tanh, "sigmoid": P.Sigmoid}[name](n)


def check_gated(cuda, sizes, b, act, dtype, bias=False, pad=0, shift=0, seed=0, backward=True, wpad=0):
    i, h, o = sizes
    r = np.random.default_rng(seed + i + h + o + b)
    ws = [tensor(r.uniform(-1, 1, s) * np.sqrt(6 / sum(s)), dtype, cuda, wpad, wpad % 2) for s in ((i, h), (i, h), (h, o))]
    bs = [vector(0.3 * r.standard_normal(n), cuda, dtype) if bias else None for n in (h, h, o)]
    x = tensor(r.standard_normal((i, b)), dtype, cuda, pad, shift)
    model = P.create_gated_model(*ws, act_layer(act, h), *bs)
    w, hb = [host(t) for t in ws], [host(t) for t in bs]
    want = N.gated(w, host(x), act, dtype, hb)
    y = model.forward_batch_parallel(x)
    close(y, *want[3], "y")
    if not backward:
        return model, x, y
    y2, states = model.forward_with_states(x)
    close(y2, *want[3], "y with states")
    kept = np.split(host(states), 3)
    for name, got, (v, e) in zip("guh", kept, want):
        close(got, v, e, name)
    dy = tensor(r.standard_normal((o, b)), dtype, cuda, shift, pad)
    d = model.backward(x, states, dy)
    wanted = N.gated_backward(w, host(x), kept, host(dy), act, dtype)
    for name, (v, e) in wanted.items():
        got = getattr(d, name)
        if got is not None:
            close(got, v, e, f"d_{name}")
    assert bias == (d.gate_bias is not None)
    return model, x, y


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("sizes,b", [((1, 1, 1), 1), ((3, 5, 2), 4), ((16, 16, 16), 16), ((64, 256, 64), 1), ((64, 256, 64), 20),
                                     ((130, 70, 33), 65), ((333, 101, 77), 503), ((256, 300, 200), 1025), ((40, 640, 40), 3),
                                     ((200, 513, 129), 33), ((96, 128, 64), 3000), ((520, 264, 136), 257)])
def test_gated(cuda, sizes, b, dtype):
    print(f"gated: {sizes} b={b} {dtype}", flush=True)
    check_gated(cuda, sizes, b, "silu", dtype, bias=b % 2 == 1, pad=b % 5, shift=b % 2)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("act", N.ACTS)
def test_gated_activations(cuda, act, dtype):
    for b in (2, 40, 300):
        check_gated(cuda, (48, 80, 56), b, act, dtype, bias=True)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("act", N.ACTS)
def test_slopes_of_large_values(cuda, act, dtype):
    """Far from zero a slope is 0, 1 or LeakyRelu's: no infinity meets a zero on the way, up to the largest floats.  (The
    block hands out dg and du as they are: one input and one column of ones, D dy of ones.)"""
    import torch

    v = np.array([1e4, 6e4] if dtype == "f16" else [1e4, 1e8, 1e12, 1e13, 3e13, 1e19, 1e26, 3e38])
    g = N.half(np.tile(np.concatenate([v, -v]), 5), dtype)
    h = g.size
    with np.errstate(over="ignore"):
        a, slope = N.activation(act, g)
    for o in (1, 4099):  # the product D dy in one piece, and cut along k
        down = torch.zeros((h, o), dtype=torch_dtype(dtype), device=cuda)
        down[:, 0] = 1
        ones = torch.ones((o, 1), dtype=torch_dtype(dtype), device=cuda)
        model = P.create_gated_model(*(torch.ones((1, h), dtype=ones.dtype, device=cuda) for _ in range(2)), down, act_layer(act, h))
        states = vector(np.concatenate([g, np.ones(h), g])[:, None], cuda, dtype)
        d = model.backward(ones[:1], states, ones)
        # one product, 0.1 in fp32 and a rounding
        for got, want in ((d.gate, slope), (d.up, a)):
            close(got[0], want, 2 * N.E * np.abs(want) + N.rounding(want, dtype), f"{act} {o}")


@pytest.mark.parametrize("dtype", DTYPES)
def test_gated_strides(cuda, dtype):
    """Weights, inputs and gradients as column ranges of wider arrays, at odd and even places."""
    for pad, shift, wpad in ((8, 0, 8), (3, 1, 0), (16, 8, 3), (0, 0, 1), (64, 2, 2)):
        for b in (1, 24, 190):
            check_gated(cuda, (72, 136, 88), b, "silu", dtype, bias=True, pad=pad, shift=shift, wpad=wpad)


@pytest.mark.parametrize("dtype", DTYPES)
def test_gated_non_finite_columns(cuda, dtype):
    """NaN and infinities stay in their columns, and meet no padding."""
    import torch

    for b in (7, 90, 300):
        r = np.random.default_rng(b)
        i, h, o = 37, 70, 41
        ws = [tensor(r.uniform(-1, 1, s) * 0.3, dtype, cuda) for s in ((i, h), (i, h), (h, o))]
        model = P.create_gated_model(*ws, P.LeakyRelu(h, 0.1))
        x = tensor(r.standard_normal((i, b)), dtype, cuda)
        x2 = x.clone()
        x2[3, 1], x2[i - 1, 2], x2[0, b - 1] = float("nan"), float("inf"), -float("inf")
        good = [c for c in range(b) if c not in (1, 2, b - 1)]
        for forward in (model.forward_batch_parallel, lambda v: model.forward_with_states(v)[0]):
            want, got = forward(x), forward(x2)
            assert torch.equal(got[:, good], want[:, good])
            assert not torch.isfinite(got[:, [1, 2, b - 1]]).any()


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("sizes,b", [((103, 30, 1186), 6774), ((2205, 31, 35), 3647), ((37, 997, 36), 8387),
                                     ((1959, 2170, 121), 310), ((134, 1717, 177), 8561), ((2157, 387, 193), 4897)])
def test_gated_large_tiles(cuda, sizes, b, dtype):
    """Products large enough for the wider tiles, whole and cut along k, with ragged edges on every side."""
    print(f"gated: {sizes} b={b} {dtype}", flush=True)
    check_gated(cuda, sizes, b, "silu", dtype, bias=b % 2 == 1, pad=b % 5, shift=b % 2)


@pytest.mark.parametrize("sizes,b", [((300, 400, 260), 17_003), ((20, 19, 18), 40_003), ((48, 38, 131), 30_011), ((700, 33, 57), 9_001),
                                     ((64, 64, 64), 33_333)])
def test_gated_fp32_of_many_tiles(cuda, sizes, b):
    """More tiles than run at once, and narrow blocks over many columns."""
    print(f"gated: {sizes} b={b}", flush=True)
    check_gated(cuda, sizes, b, "silu", "f32", bias=b % 2 == 1, pad=b % 5, shift=b % 2)


@pytest.mark.parametrize("sizes", [(40, 31, 33), (300, 32, 64), (333, 33, 65), (77, 64, 20), (900, 65, 5), (2100, 30, 127)])
def test_gated_fp32_narrow_tiles(cuda, sizes):
    """Tiles of 64 rows (of a pair 32 of each) by 256 columns: either side of their borders, in one piece and cut along k."""
    for b in (255, 256, 257, 700, 3001):
        for act in ("tanh", "gelu"):
            check_gated(cuda, sizes, b, act, "f32", bias=b % 2 == 1, pad=b % 4, shift=b % 3, seed=b, wpad=b % 3)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("sizes,b", [((20, 19, 18), 60_001), ((130, 40, 70), 30_002)])
def test_gated_narrow_weights_over_many_columns(cuda, sizes, b, dtype):
    """Weights' gradients in as many parts as there are workgroups to share them."""
    print(f"gated: {sizes} b={b} {dtype}", flush=True)
    check_gated(cuda, sizes, b, "tanh", dtype, bias=True, pad=b % 3, shift=b % 2)


def test_gated_gradients_keep_to_their_work_buffer(cuda):
    """What is needed for the columns of a call, and no byte behind it."""
    import ctypes

    import torch

    i, h, o = 20, 19, 33
    for dtype in DTYPES:
        t = torch_dtype(dtype)
        ws = [(torch.randn(s, device=cuda) / 4).to(t) for s in ((i, h), (i, h), (h, o))]
        model = P.create_gated_model(*ws, P.Silu(h))
        L = A.lib()
        for b in (1, 7, 300, 4001, 20_000, 70_003):
            x, dy = torch.randn((i, b), device=cuda).to(t), torch.randn((o, b), device=cuda).to(t)
            _, states = model.forward_with_states(x)
            want = model.backward(x, states, dy)
            need = L.ponni_gated_backward_workspace_bytes(model._ref, b)
            work = torch.full((need + 4096,), 255, dtype=torch.uint8, device=cuda)  # (NaN)
            work[need:] = 7
            out = [torch.empty_like(v) for v in (want.x, want.gate, want.up, want.down)]
            g = A.GatedGradientArrays(out[0].data_ptr(), b, *(v.data_ptr() for v in out[1:]), h, h, o)
            assert L.ponni_gated_backward(model._ref, x.data_ptr(), b, states.data_ptr(), states.stride(0), dy.data_ptr(), b, b,
                                          ctypes.byref(g), work.data_ptr(), need, torch.cuda.current_stream().cuda_stream) == 0
            assert bool((work[need:] == 7).all())
            for v, w in zip(out, (want.x, want.gate, want.up, want.down)):
                assert torch.equal(v, w)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("sizes,b", [((4099, 70, 40), 130), ((40, 70, 4099), 61), ((3001, 45, 2003), 35)])
def test_gated_long_sums_of_few_tiles(cuda, sizes, b, dtype):
    """Every product cut along k, both first ones and that of D dy among them."""
    check_gated(cuda, sizes, b, "silu", dtype, bias=True, pad=3, shift=1)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("sizes", [(64, 256, 64), (1000, 600, 700), (130, 70, 33), (7, 1031, 5)])
def test_gated_few_columns(cuda, sizes, dtype):
    """Either side of the numbers of columns where kernels change; a column's result is that of the column alone, but
    for the order of sums."""
    for b in (1, 7, 8, 9, 15, 16, 17, 31, 32, 33, *((64, 65, 257, 511, 512, 513) if dtype == "f32" else ())):
        check_gated(cuda, sizes, b, "gelu", dtype, bias=b % 2 == 0, pad=b % 3, backward=False, seed=b, wpad=b % 4)


@pytest.mark.parametrize("dtype", DTYPES)
def test_gated_widest(cuda, dtype):
    """The largest widths, one at a time, and (16 bits) the most columns."""
    for sizes in ((2, 65536, 1), (65536, 3, 2), (5, 2, 65536)):
        for b in (1, 40):
            check_gated(cuda, sizes, b, "relu", dtype, bias=True)
    if dtype == "bf16":
        check_gated(cuda, (2, 3, 1), A.GATED_MAX_COLUMNS, "relu", dtype)


@pytest.mark.parametrize("dtype", DTYPES)
def test_gated_results_leave_their_neighbours(cuda, dtype):
    """Results that are column ranges of wider arrays: what lies beside them stays, with and without states, and of
    every gradient."""
    import ctypes

    import torch

    t = torch_dtype(dtype)
    r = np.random.default_rng(5)
    for (i, h, o), b, left, right in (((37, 70, 41), 5, 3, 4), ((37, 70, 41), 61, 8, 3), ((300, 300, 290), 517, 1, 7)):
        ws = [tensor(r.uniform(-1, 1, s) * 0.3, dtype, cuda) for s in ((i, h), (i, h), (h, o))]
        bs = [vector(r.standard_normal(n), cuda, dtype) for n in (h, h, o)]
        model = P.create_gated_model(*ws, P.Tanh(h), *bs)
        x, dy = tensor(r.standard_normal((i, b)), dtype, cuda), tensor(r.standard_normal((o, b)), dtype, cuda)

        def wide(rows, columns):
            a = torch.full((rows + 1, left + columns + right), 7.0, dtype=t, device=cuda)
            return a, a[:rows, left:left + columns]

        def untouched(a, v):
            rest = torch.ones_like(a, dtype=torch.bool)
            rest[:v.shape[0], left:left + v.shape[1]] = False
            return bool((a[rest] == 7.0).all())

        a, y = wide(o, b)
        assert model.forward_batch_parallel(x, y) is y
        assert untouched(a, y) and torch.equal(y, model.forward_batch_parallel(x))
        y2, states = model.forward_with_states(x)
        a, y = wide(o, b)
        sa, sv = wide(3 * h, b)
        L = A.lib()
        need = L.ponni_gated_backward_workspace_bytes(model._ref, b)
        work = torch.full((need,), 255, dtype=torch.uint8, device=cuda)  # (NaN)
        stream = torch.cuda.current_stream().cuda_stream
        assert L.ponni_gated_forward(model._ref, x.data_ptr(), b, y.data_ptr(), a.stride(0), sv.data_ptr(), sa.stride(0), b,
                                     work.data_ptr(), L.ponni_gated_workspace_bytes(model._ref, b), stream) == 0
        assert untouched(a, y) and untouched(sa, sv) and torch.equal(y, y2) and torch.equal(sv, states)
        want = model.backward(x, states, dy)
        got = [wide(*s) for s in ((i, b), (i, h), (i, h), (h, o))]
        biases = [torch.empty(n, dtype=t, device=cuda) for n in (h, h, o)]
        g = A.GatedGradientArrays(got[0][1].data_ptr(), got[0][0].stride(0), *(v.data_ptr() for _, v in got[1:]),
                                  *(w.stride(0) for w, _ in got[1:]), *(v.data_ptr() for v in biases))
        assert L.ponni_gated_backward(model._ref, x.data_ptr(), b, sv.data_ptr(), sa.stride(0), dy.data_ptr(), b, b,
                                      ctypes.byref(g), work.data_ptr(), need, stream) == 0
        for (a, v), w in zip(got, (want.x, want.gate, want.up, want.down)):
            assert untouched(a, v) and torch.equal(v, w)
        for v, w in zip(biases, (want.gate_bias, want.up_bias, want.down_bias)):
            assert torch.equal(v, w)


def test_gated_gradients_that_are_asked_for(cuda):
    """Each gradient by itself has the bits that it has among all."""
    import ctypes

    import torch

    i, h, o, b = 70, 150, 90, 333
    for dtype in DTYPES:
        t = torch_dtype(dtype)
        ws = [(torch.randn(s, device=cuda) / 8).to(t) for s in ((i, h), (i, h), (h, o))]
        bs = [torch.randn(n, device=cuda).to(t) for n in (h, h, o)]
        model = P.create_gated_model(*ws, P.Sigmoid(h), *bs)
        x, dy = torch.randn((i, b), device=cuda).to(t), torch.randn((o, b), device=cuda).to(t)
        _, states = model.forward_with_states(x)
        want = model.backward(x, states, dy)
        only = model.backward(x, states, dy, need_parameters=False)
        assert torch.equal(only.x, want.x) and only.gate is None and only.down_bias is None
        rest = model.backward(x, states, dy, need_x=False)
        assert rest.x is None and torch.equal(rest.up, want.up) and torch.equal(rest.gate_bias, want.gate_bias)
        L = A.lib()
        need = L.ponni_gated_backward_workspace_bytes(model._ref, b)
        work = torch.full((need,), 255, dtype=torch.uint8, device=cuda)  # (NaN)
        for name, ld in (("gate", h), ("up", h), ("down", o), ("gate_bias", 0), ("up_bias", 0), ("down_bias", 0)):
            v = torch.empty_like(getattr(want, name))
            g = A.GatedGradientArrays()
            setattr(g, name, v.data_ptr())
            if ld:
                setattr(g, "ld_" + name, ld)
            assert L.ponni_gated_backward(model._ref, x.data_ptr(), b, states.data_ptr(), states.stride(0), dy.data_ptr(), b, b,
                                          ctypes.byref(g), work.data_ptr(), need, torch.cuda.current_stream().cuda_stream) == 0
            if name not in ("gate", "up"):
                assert torch.equal(v, getattr(want, name)), name
                continue
            # One of the two products of x may be cut along k otherwise than both: b terms in another order, and a
            # rounding to either side.
            gv, uv = states[:h].double(), states[h:2 * h].double()
            p, dh = torch.sigmoid(gv), ws[2].double() @ dy.double()
            dv = dh * uv * p * (1 - p) if name == "gate" else dh * p
            bound = 1.1 * (2 * b * 2.0 ** -24 * (x.double().abs() @ dv.abs().T)
                           + torch.finfo(t).eps * getattr(want, name).double().abs())
            assert bool(((v.double() - getattr(want, name).double()).abs() <= bound).all()), name


def test_gated_inputs_beyond_four_gigabytes(cuda):
    """Columns of an array whose rows lie 4 MB apart: byte offsets past 2^32 in every operand with columns."""
    import torch

    i, ld, b = 1100, 2_000_000, 150
    wide = torch.zeros((i, ld), dtype=torch.bfloat16, device=cuda)
    x = wide[:, ld - b:]
    x.copy_(torch.randn((i, b), device=cuda))
    ws = [(torch.randn(s, device=cuda) / 16).bfloat16() for s in ((i, 96), (i, 96), (96, i))]
    model = P.create_gated_model(*ws, P.Silu(96))
    near = x.contiguous()
    for n in (b, 20):
        want = model.forward_batch_parallel(near[:, :n])
        assert torch.equal(model.forward_batch_parallel(x[:, :n]), want)
    y, states = model.forward_with_states(near)
    want = model.backward(near, states, near)
    got = model.backward(x, states, x)
    for name in ("x", "gate", "up", "down"):
        assert torch.equal(getattr(got, name), getattr(want, name)), name
    assert torch.equal(model.forward_batch_parallel(near, x), y) and torch.equal(x, y)
    assert not wide[:, :ld - b].any()


def test_gated_work_buffer_of_more_columns(cuda):
    """One buffer, of the most columns, for calls of fewer."""
    import torch

    i, h, o, most = 200, 900, 150, 3000
    for dtype in DTYPES:
        t = torch_dtype(dtype)
        ws = [(torch.randn(s, device=cuda) / 16).to(t) for s in ((i, h), (i, h), (h, o))]
        model = P.create_gated_model(*ws, P.Silu(h))
        L = A.lib()
        need = L.ponni_gated_workspace_bytes(model._ref, most)
        work = torch.full((need + 64,), 255, dtype=torch.uint8, device=cuda)  # (NaN)
        work[need:] = 7
        for b in (1, 8, 9, 32, 33, 200, 512, 513, 1000, most):
            x = torch.randn((i, b), device=cuda).to(t)
            y = torch.empty((o, b), dtype=t, device=cuda)
            assert L.ponni_gated_forward(model._ref, x.data_ptr(), b, y.data_ptr(), b, None, 0, b, work.data_ptr(), need,
                                         torch.cuda.current_stream().cuda_stream) == 0
            assert torch.equal(y, model.forward_batch_parallel(x))
        assert bool((work[need:] == 7).all())


@pytest.mark.parametrize("dtype", DTYPES)
def test_gated_calls_keep_to_what_they_ask_for(cuda, dtype):
    """The work buffer of a call with these arrays, whichever of them has to be copied first: enough, and no byte behind it
    is written."""
    import ctypes

    import torch

    t, L = torch_dtype(dtype), A.lib()
    stream = torch.cuda.current_stream().cuda_stream
    for (i, h, o), wpad in (((37, 70, 41), 1), ((300, 260, 50), 0), ((64, 33, 20), 3)):
        ws = [tensor(np.random.default_rng(h).uniform(-0.3, 0.3, s), dtype, cuda, wpad) for s in ((i, h), (i, h), (h, o))]
        model = P.create_gated_model(*ws, P.Gelu(h, True))
        for b in (1, 20, 130, 1501):
            for odd in ((), ("x",), ("states",), ("dy",), ("x", "states", "dy")):
                def array(name, rows):
                    return tensor(torch.randn((rows, b)).numpy(), dtype, cuda, b % 2, 1) if name in odd else \
                        tensor(torch.randn((rows, b)).numpy(), dtype, cuda, b % 2, 0)

                x, dy, states = array("x", i), array("dy", o), array("states", 3 * h)
                y = torch.empty((o, b), dtype=t, device=cuda)

                def call(fn, s, d, *args):
                    need = L.ponni_gated_call_workspace_bytes(model._ref, x.data_ptr(), x.stride(0), s, states.stride(0), d,
                                                              dy.stride(0), b)
                    work = torch.full((need + 4096,), 255, dtype=torch.uint8, device=cuda)  # (NaN)
                    work[need:] = 7
                    assert fn(model._ref, x.data_ptr(), x.stride(0), *args, b, *rest, work.data_ptr(), need, stream) == 0
                    assert bool((work[need:] == 7).all())

                rest = ()
                call(L.ponni_gated_forward, None, None, y.data_ptr(), b, None, 0)
                assert torch.equal(y, model.forward_batch_parallel(x))
                call(L.ponni_gated_forward, states.data_ptr(), None, y.data_ptr(), b, states.data_ptr(), states.stride(0))
                y2, states2 = model.forward_with_states(x)
                assert torch.equal(y, y2) and torch.equal(states, states2)
                want = model.backward(x, states2, dy)
                out = [torch.empty_like(v) for v in (want.x, want.gate, want.up, want.down)]
                g = A.GatedGradientArrays(out[0].data_ptr(), b, *(v.data_ptr() for v in out[1:]), h, h, o)
                rest = (ctypes.byref(g),)
                call(L.ponni_gated_backward, states.data_ptr(), dy.data_ptr(), states.data_ptr(), states.stride(0), dy.data_ptr(),
                     dy.stride(0))
                for v, w in zip(out, (want.x, want.gate, want.up, want.down)):
                    assert torch.equal(v, w)


def test_gated_gradient_by_differences(cuda):
    r = np.random.default_rng(9)
    i, h, o, b = 6, 9, 5, 4
    w = [r.standard_normal(s) for s in ((i, h), (i, h), (h, o))]
    bs = [r.standard_normal(n) for n in (h, h, o)]
    x, dy = r.standard_normal((i, b)), r.standard_normal((o, b))
    for act in ("silu", "gelu", "gelu_erf", "tanh", "sigmoid"):
        model = P.create_gated_model(*(vector(v, cuda) for v in w), act_layer(act, h), *(vector(v, cuda) for v in bs))
        _, states = model.forward_with_states(vector(x, cuda))
        d = model.backward(vector(x, cuda), states, vector(dy, cuda))

        def value(w, bs, x):
            a = N.activation(act, w[0].T @ x + bs[0][:, None])[0]
            return (dy * (w[2].T @ (a * (w[1].T @ x + bs[1][:, None])) + bs[2][:, None])).sum()

        leaves = [*w, *bs, x]
        grads = [d.gate, d.up, d.down, d.gate_bias, d.up_bias, d.down_bias, d.x]
        for k, g in enumerate(grads):
            direction = r.standard_normal(leaves[k].shape)

            def at(e):
                v = [a + e * direction if j == k else a for j, a in enumerate(leaves)]
                return value(v[:3], v[3:6], v[6])

            # fp32's roundings of some 300 terms of size up to 10, and the differences' third order
            want = (at(1e-4) - at(-1e-4)) / 2e-4
            assert abs((host(g) * direction).sum() - want) < 2e-4 * max(1.0, abs(want))


# -- together ---------------------------------------------------------------------------------


def test_a_block_with_its_head(cuda):
    """norm -> gated block -> residual, gate and norms -> head -> log probabilities and back, in fp32 against torch's
    gradients in 64 bits."""
    import torch

    torch.manual_seed(3)
    n, h, c, b = 48, 120, 211, 77
    w = {k: torch.randn(s, dtype=torch.float64) / s[0] ** 0.5 for k, s in
         (("G", (n, h)), ("U", (n, h)), ("D", (h, n)), ("R", (n, c)))}
    v = {k: 1 + 0.2 * torch.randn(n, dtype=torch.float64) for k in ("w1", "w2", "w3", "gate")}
    x = torch.randn((n, b), dtype=torch.float64)
    t = torch.randint(0, c, (b,))
    leaves = {k: p.to(torch.float32).double().requires_grad_() for k, p in {**w, **v, "x": x}.items()}

    def rms(y, weight):
        return y * (y.pow(2).mean(0, keepdim=True) + 1e-5).rsqrt() * weight[:, None]

    L = leaves
    hidden = rms(L["x"], L["w1"])
    y = L["D"].T @ (torch.nn.functional.silu(L["G"].T @ hidden) * (L["U"].T @ hidden))
    state = L["x"] + 0.5 * L["gate"][:, None] * rms(y, L["w2"])
    lp = torch.log_softmax(L["R"].T @ rms(state, L["w3"]), 0)
    entropy = -(lp.exp() * lp).sum(0)
    loss = -lp[t, torch.arange(b)].mean() + 0.1 * entropy.mean()
    loss.backward()

    g = {k: p.detach().float().to(cuda) for k, p in leaves.items()}
    first = P.create_residual_norm(n, before=P.BlockNorm("rms", g["w1"]))
    block = P.create_gated_model(g["G"], g["U"], g["D"], P.Silu(h))
    last = P.create_residual_norm(n, after=P.BlockNorm("rms", g["w2"]), before=P.BlockNorm("rms", g["w3"]), scale=0.5)
    head = P.create_inference_model(P.Matvec(g["R"].cpu().numpy()))
    back = P.create_inference_model(P.Matvec(g["R"].T.contiguous().cpu().numpy()))
    _, normed, s1 = first.forward_with_statistics(g["x"])
    out, states = block.forward_with_states(normed)
    new, final, s2 = last.forward_with_statistics(out, g["x"], g["gate"])
    r = P.log_probabilities(head.forward_batch_parallel(final), t.int().to(cuda), 3)
    got = -r.log_probs.mean() + 0.1 * r.entropy.mean()
    assert abs(float(got) - float(loss)) < 1e-5
    d_logits = r.backward(torch.full((b,), -1.0 / b, device=cuda), torch.full((b,), 0.1 / b, device=cuda))
    d_final = back.forward_batch_parallel(d_logits)
    d2 = last.backward(out, g["x"], g["gate"], s2, None, d_final)
    db = block.backward(normed, states, d2.x)
    d1 = first.backward(g["x"], None, None, s1, d2.residual, db.x)
    for name, value in (("G", db.gate), ("U", db.up), ("D", db.down), ("w1", d1.before_weight), ("w2", d2.after_weight),
                        ("w3", d2.before_weight), ("gate", d2.gate), ("x", d1.x)):
        want = leaves[name].grad
        # some 500 roundings of 2^-24 along the way
        assert float((value.double().cpu() - want).norm() / want.norm()) < 500 * 2.0 ** -24, name


def test_block_operators_on_streams_and_in_graphs(cuda):
    """Captured once, replayed with new inputs between eager calls; the same bits every time."""
    import torch

    n, h, c = 72, 200, 300
    for dtype, b in (("bf16", 3), ("f16", 200), ("f32", 70)):
        t = torch_dtype(dtype)
        ws = [(torch.randn(s, device=cuda) / 8).to(t) for s in ((n, h), (n, h), (h, c))]
        block = P.create_gated_model(*ws, P.Gelu(h, True))
        norm = P.create_residual_norm(n, after=P.BlockNorm("rms", torch.randn(n, device=cuda)),
                                      before=P.BlockNorm("layer", torch.randn(n, device=cuda), torch.randn(n, device=cuda)),
                                      dtype=dtype)
        x, res = torch.randn((n, b), device=cuda).to(t), torch.randn((n, b), device=cuda).to(t)
        gate = torch.randn(n, device=cuda)
        targets = torch.randint(0, c, (b,), dtype=torch.int32, device=cuda)
        g = torch.randn(b, device=cuda)

        def step():
            state, normed, s = norm.forward_with_statistics(x, res, gate)
            y, states = block.forward_with_states(normed)
            r = P.log_probabilities(y, targets, 2)
            dy = r.backward(g, g)
            d = block.backward(normed, states, dy)
            e = norm.backward(x, res, gate, s, state, d.x)
            return [state, normed, y, r.log_probs, r.entropy, r.top_classes, r.top_log_probs, dy, d.x, d.gate, d.up, d.down,
                    e.x, e.residual, e.gate, e.after_weight, e.before_weight, e.before_bias]

        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            warm = step()
        torch.cuda.current_stream().wait_stream(side)
        assert all(torch.equal(a, e) for a, e in zip(warm, step()))
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = step()
        for seed in range(3):
            torch.manual_seed(seed)
            x.copy_(torch.randn((n, b), device=cuda))
            ws[0].copy_(torch.randn((n, h), device=cuda) / 8)
            graph.replay()
            want = step()
            torch.cuda.synchronize()
            assert all(torch.equal(a, e) for a, e in zip(outs, want))


def test_graphs_of_block_operators_side_by_side(cuda):
    """Two captured programs, of other sizes, replayed in turn: neither disturbs the other's buffers."""
    import torch

    programs = []
    for n, h, c, b in ((72, 900, 300, 3), (160, 700, 1200, 90)):
        ws = [(torch.randn(s, device=cuda) / 16).bfloat16() for s in ((n, h), (n, h), (h, c))]
        block = P.create_gated_model(*ws, P.Silu(h))
        x = torch.randn((n, b), device=cuda).bfloat16()
        targets = torch.randint(0, c, (b,), dtype=torch.int32, device=cuda)
        g = torch.randn(b, device=cuda)

        def step(block=block, x=x, targets=targets, g=g):
            y = block.forward_batch_parallel(x)
            y2, states = block.forward_with_states(x)
            r = P.log_probabilities(y, targets, 4)
            d = block.backward(x, states, r.backward(g))
            return [y, y2, r.log_probs, r.top_classes, r.top_log_probs, d.x, d.gate, d.up, d.down]

        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step()
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = step()
        programs.append((graph, outs, step, x))
    for seed in range(3):
        torch.manual_seed(seed)
        for _, _, _, x in programs:
            x.copy_(torch.randn(x.shape, device=cuda))
        for graph, _, _, _ in programs:
            graph.replay()
        for graph, outs, step, _ in programs[::-1]:
            want = step()
            torch.cuda.synchronize()
            assert all(torch.equal(a, e) for a, e in zip(outs, want))
