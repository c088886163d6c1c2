"""Gated feed-forward blocks, the norms and gates between blocks, and log
probabilities of given classes, with their gradients, over libponni_hip.

    boundary = create_residual_norm(n, after=BlockNorm("rms", w1), before=BlockNorm("rms", w2))
    block = create_gated_model(G, U, D, Silu(hidden))      # G, U [n, hidden], D [hidden, n] on the GPU
    y = block.forward_batch_parallel(normed)               # normed [n, columns]
    state, normed = boundary.forward_batch_parallel(y, state)   # state + after(y), and its norm for the next block
    r = log_probabilities(logits, targets, top_k=5)        # logits [classes, columns], targets int32 [columns]
    d_logits = r.backward(d_log_probs)

GPU tensors are [features, columns] with contiguous rows, as for
Inference.forward_batch_parallel.  Parameters are the caller's tensors, read
where they are at every call: a program that trains changes them in place.
Gradients are explicit calls (these operators are no torch.autograd functions).
Work buffers are allocated by torch for each call, on the current stream.
"""
from __future__ import annotations

import ctypes
from dataclasses import dataclass

from . import _abi as A
from .experts import _call, _rows, _same_device, _types
from .model import _DTYPES, Layer


def _empty(like, *shape, dtype=None):
    return like.new_empty(shape) if dtype is None else like.new_empty(shape, dtype=dtype)


def _work(like, need: int):
    """A work buffer, or none: its address and what keeps it."""
    if need < 0:
        raise A.PonniError(A.PONNI_ERR_INVALID_ARGUMENT, A.lib().ponni_last_error().decode())
    if need == 0:
        return 0, None
    import torch

    t = torch.empty(need, dtype=torch.uint8, device=like.device)
    return t.data_ptr(), t


def _array(t, what: str, like, rows: int, columns: int) -> int:
    """Checks that t is [rows, columns] of the type and device of `like`; its row stride."""
    ld = _rows(t, what, rows, columns)
    if t.dtype != like.dtype:
        raise ValueError(f"{what} is {t.dtype}, not {like.dtype}")
    _same_device(t, like, what)
    return ld


def _vector(t, what: str, n: int, dtype, device_of=None):
    if tuple(t.shape) != (n,) or t.dtype != dtype or not t.is_cuda or (n > 1 and t.stride(0) != 1):
        raise ValueError(f"{what} must be a contiguous {dtype} GPU tensor of shape ({n},)")
    if device_of is not None:
        _same_device(t, device_of, what)


# -- gated feed-forward blocks -------------------------------------------------------------


@dataclass
class GatedGradients:
    """Gradients of a gated block's input and parameters, each in the shape and type of what it belongs to
    (None where they were not asked for)."""

    x: "object" = None
    gate: "object" = None
    up: "object" = None
    down: "object" = None
    gate_bias: "object" = None
    up_bias: "object" = None
    down_bias: "object" = None


class GatedInference:
    """y = D^T (act(G^T x + g0) * (U^T x + u0)) + d0 (ponni_gated).  G, U [n_in, n_hidden] and D [n_hidden, n_out]
    are GPU tensors of one type, f32, f16 or bf16, with contiguous rows, biases vectors of the same type; act is a
    pointwise layer: Relu, LeakyRelu, Gelu, Silu, Sigmoid or Tanh of n_hidden features."""

    def __init__(self, gate, up, down, act: Layer, gate_bias=None, up_bias=None, down_bias=None):
        if not isinstance(act, Layer):
            raise ValueError(f"act must be a pointwise layer such as Silu(n_hidden), not {act!r}")
        _rows(gate, "gate")
        self.n_in, self.n_hidden = gate.shape
        _array(up, "up", gate, self.n_in, self.n_hidden)
        _rows(down, "down", self.n_hidden)
        self.n_out = down.shape[1]
        _array(down, "down", gate, self.n_hidden, self.n_out)
        if gate.dtype not in _types()[1]:
            raise ValueError(f"weights of type {gate.dtype}")
        for t, n, what in ((gate_bias, self.n_hidden, "gate_bias"), (up_bias, self.n_hidden, "up_bias"),
                           (down_bias, self.n_out, "down_bias")):
            if t is not None:
                _vector(t, what, n, gate.dtype, gate)
        self.act = act
        self._weights, self._biases = (gate.detach(), up.detach(), down.detach()), tuple(
            None if t is None else t.detach() for t in (gate_bias, up_bias, down_bias))
        self._block = A.Gated(self.n_in, self.n_hidden, self.n_out, _types()[1][gate.dtype], act.desc(),
                              *(t.data_ptr() for t in self._weights), *(_rows(t, "weights") for t in self._weights),
                              *(None if t is None else t.data_ptr() for t in self._biases))
        self._ref = ctypes.byref(self._block)
        if A.lib().ponni_gated_workspace_bytes(self._ref, 1) < 0:
            raise A.PonniError(A.PONNI_ERR_INVALID_MODEL, A.lib().ponni_last_error().decode())

    gate = property(lambda self: self._weights[0])
    up = property(lambda self: self._weights[1])
    down = property(lambda self: self._weights[2])
    gate_bias = property(lambda self: self._biases[0])
    up_bias = property(lambda self: self._biases[1])
    down_bias = property(lambda self: self._biases[2])

    def get_num_inputs(self) -> int:
        return self.n_in

    def get_num_outputs(self) -> int:
        return self.n_out

    def _forward(self, x, y, states):
        ld_x = _rows(x, "x", self.n_in)
        w = self._weights[0]
        if x.dtype != w.dtype:
            raise ValueError(f"x is {x.dtype}, the block {w.dtype}")
        _same_device(x, w, "x")
        columns = x.shape[1]
        if y is None:
            y = _empty(x, self.n_out, columns)
            ld_y = columns
        else:
            ld_y = _array(y, "y", x, self.n_out, columns)
        L = A.lib()
        at, ld_s = (None, 0) if states is None else (states.data_ptr(), states.stride(0))
        need = L.ponni_gated_call_workspace_bytes(self._ref, x.data_ptr(), ld_x, at, ld_s, None, 0, columns)
        work, kept = _work(x, need)
        _call(x, L.ponni_gated_forward, self._ref, x.data_ptr(), ld_x, y.data_ptr(), ld_y, at, ld_s, columns, work, need)
        return y

    def forward_batch_parallel(self, x, y=None):
        """x [n_in, columns] of the block's type; y [n_out, columns]."""
        return self._forward(x, y, None)

    def forward_with_states(self, x, y=None):
        """y, and what the backward pass reads beside x: g, u and h, [3 n_hidden, columns]."""
        ld = -(-x.shape[1] // 64) * 64 if x.dim() == 2 else 0  # (rows at whole lines)
        states = _empty(x, 3 * self.n_hidden, ld)[:, :x.shape[1]] if ld else None
        return self._forward(x, y, states), states

    def backward(self, x, states, dy, need_x: bool = True, need_parameters: bool = True) -> GatedGradients:
        """Gradients from dy [n_out, columns], x and the states that forward_with_states left."""
        columns = dy.shape[1] if dy.dim() == 2 else 0
        ld_dy = _rows(dy, "dy", self.n_out)
        w = self._weights[0]
        if dy.dtype != w.dtype:
            raise ValueError(f"dy is {dy.dtype}, the block {w.dtype}")
        _same_device(dy, w, "dy")
        ld_x, ld_s = _array(x, "x", dy, self.n_in, columns), _array(states, "states", dy, 3 * self.n_hidden, columns)
        d = GatedGradients()
        if need_x:
            d.x = _empty(dy, self.n_in, columns)
        if need_parameters:
            d.gate, d.up = _empty(dy, self.n_in, self.n_hidden), _empty(dy, self.n_in, self.n_hidden)
            d.down = _empty(dy, self.n_hidden, self.n_out)
            for name, t in zip(("gate_bias", "up_bias", "down_bias"), self._biases):
                if t is not None:
                    setattr(d, name, _empty(dy, t.shape[0]))
        at = [None if t is None else t.data_ptr() for t in (d.x, d.gate, d.up, d.down, d.gate_bias, d.up_bias, d.down_bias)]
        g = A.GatedGradientArrays(at[0], columns, *at[1:4], self.n_hidden, self.n_hidden, self.n_out, *at[4:])
        L = A.lib()
        need = L.ponni_gated_call_workspace_bytes(self._ref, x.data_ptr(), ld_x, states.data_ptr(), ld_s, dy.data_ptr(), ld_dy,
                                                  columns)
        work, kept = _work(dy, need)
        _call(dy, L.ponni_gated_backward, self._ref, x.data_ptr(), ld_x, states.data_ptr(), ld_s, dy.data_ptr(), ld_dy,
              columns, ctypes.byref(g), work, need)
        return d


def create_gated_model(gate, up, down, act: Layer, gate_bias=None, up_bias=None, down_bias=None) -> GatedInference:
    """A gated feed-forward block of the caller's tensors (GatedInference)."""
    return GatedInference(gate, up, down, act, gate_bias, up_bias, down_bias)


# -- norms and gates between blocks ------------------------------------------------------------

_KINDS = {"rms": A.NORM_RMS, "layer": A.NORM_LAYER}


class BlockNorm:
    """A norm of each column's features: kind "rms" (v / sqrt(mean(v^2) + eps)) or "layer" (of v - mean(v)), times
    weight plus bias, float32 GPU tensors [n] or None."""

    __slots__ = ("kind", "weight", "bias", "eps")

    def __init__(self, kind: str, weight=None, bias=None, eps: float = 1e-5):
        if kind not in _KINDS:
            raise ValueError(f"kind must be 'rms' or 'layer', not {kind!r}")
        self.kind, self.eps = kind, eps
        self.weight, self.bias = (None if t is None else t.detach() for t in (weight, bias))

    def _struct(self, n: int, what: str):
        import torch

        for t, name in ((self.weight, "weight"), (self.bias, "bias")):
            if t is not None:
                _vector(t, f"the {name} {what}", n, torch.float32)
        return A.Norm(_KINDS[self.kind], self.eps, None if self.weight is None else self.weight.data_ptr(),
                      None if self.bias is None else self.bias.data_ptr())


@dataclass
class ResidualNormGradients:
    """Gradients of ResidualNorm's inputs, each in the shape and type of what it belongs to (None where there is no
    such input), and of its parameters, float32 [n]."""

    x: "object" = None
    residual: "object" = None
    gate: "object" = None
    after_weight: "object" = None
    after_bias: "object" = None
    before_weight: "object" = None
    before_bias: "object" = None


class ResidualNorm:
    """What stands between two blocks (ponni_residual_norm):
    state = residual + scale * gate * after(x), normed = before(state), over columns of n features."""

    def __init__(self, n: int, after: BlockNorm | None = None, before: BlockNorm | None = None, scale: float = 1.0,
                 dtype: str = "f32"):
        self.n, self.after, self.before, self.scale, self.dtype = n, after, before, scale, dtype
        if dtype not in _types()[0]:
            raise ValueError(f"norms between blocks are f32, f16 or bf16, not {dtype!r}")
        self._type = _types()[0][dtype]
        if A.lib().ponni_residual_norm_workspace_bytes(n, _DTYPES[dtype], 1) < 0:
            raise A.PonniError(A.PONNI_ERR_SHAPE, A.lib().ponni_last_error().decode())
        self._base = A.ResidualNormArrays(n, _DTYPES[dtype], 0, A.Norm() if after is None else after._struct(n, "after"),
                                          A.Norm() if before is None else before._struct(n, "before"), scale)
        self._parameters = [t for norm in (after, before) if norm is not None for t in (norm.weight, norm.bias)
                            if t is not None]

    def _arrays(self, x, residual, gate):
        import torch

        r = A.ResidualNormArrays.from_buffer_copy(self._base)
        r.ld_x = _rows(x, "x", self.n)
        if x.dtype != self._type:
            raise ValueError(f"x is {x.dtype}, the norms' type {self._type}")
        r.columns, r.x = x.shape[1], x.data_ptr()
        for t in self._parameters:
            _same_device(t, x, "a norm's parameter")
        if residual is not None:
            r.ld_residual, r.residual = _array(residual, "residual", x, self.n, x.shape[1]), residual.data_ptr()
        if gate is not None and gate.dim() == 1:
            _vector(gate, "gate", self.n, torch.float32, x)
            r.feature_gate = gate.data_ptr()
        elif gate is not None:
            r.ld_gate, r.gate = _array(gate, "gate", x, self.n, x.shape[1]), gate.data_ptr()
        return r

    def _forward(self, x, residual, gate, statistics):
        r = self._arrays(x, residual, gate)
        columns = r.columns
        state, normed = _empty(x, self.n, columns), None
        r.state, r.ld_state = state.data_ptr(), columns
        if self.before is not None:
            normed = _empty(x, self.n, columns)
            r.normed, r.ld_normed = normed.data_ptr(), columns
        if statistics is not None:
            r.statistics = statistics.data_ptr()
        _call(x, A.lib().ponni_residual_norm_forward, ctypes.byref(r))
        return state, normed

    def forward_batch_parallel(self, x, residual=None, gate=None):
        """x, residual [n, columns], gate float32 [n] or [n, columns]: state and normed (None without a norm before)."""
        return self._forward(x, residual, gate, None)

    def forward_with_statistics(self, x, residual=None, gate=None):
        """state, normed, and the norms' statistics for the backward pass, float32 [4, columns]."""
        import torch

        statistics = _empty(x, 4, x.shape[-1], dtype=torch.float32)
        return (*self._forward(x, residual, gate, statistics), statistics)

    def backward(self, x, residual, gate, statistics, d_state=None, d_normed=None) -> ResidualNormGradients:
        """Gradients from those of state and normed (None: zero), the inputs of the forward pass and its statistics."""
        import torch

        r = self._arrays(x, residual, gate)
        columns = r.columns
        if tuple(statistics.shape) != (4, columns) or statistics.dtype != torch.float32 or not statistics.is_contiguous():
            raise ValueError(f"statistics must be a contiguous float32 tensor of shape (4, {columns})")
        _same_device(statistics, x, "statistics")
        r.statistics = statistics.data_ptr()
        g = A.ResidualNormGradientArrays()
        if d_state is not None:
            g.ld_d_state, g.d_state = _array(d_state, "d_state", x, self.n, columns), d_state.data_ptr()
        if d_normed is not None:
            g.ld_d_normed, g.d_normed = _array(d_normed, "d_normed", x, self.n, columns), d_normed.data_ptr()
        d = ResidualNormGradients(x=_empty(x, self.n, columns))
        g.d_x, g.ld_d_x = d.x.data_ptr(), columns
        if residual is not None:
            d.residual = _empty(x, self.n, columns)
            g.d_residual, g.ld_d_residual = d.residual.data_ptr(), columns
        if gate is not None and gate.dim() == 1:
            d.gate = _empty(x, self.n, dtype=torch.float32)
            g.d_feature_gate = d.gate.data_ptr()
        elif gate is not None:
            d.gate = _empty(x, self.n, columns)
            g.d_gate, g.ld_d_gate = d.gate.data_ptr(), columns
        for norm, which in ((self.after, "after"), (self.before, "before")):
            for name in ("weight", "bias"):
                if norm is not None and getattr(norm, name) is not None:
                    t = _empty(x, self.n, dtype=torch.float32)
                    setattr(d, f"{which}_{name}", t)
                    setattr(g, f"d_{which}_{name}", t.data_ptr())
        L = A.lib()
        need = L.ponni_residual_norm_workspace_bytes(self.n, r.dtype, columns)
        work, kept = _work(x, need)
        _call(x, L.ponni_residual_norm_backward, ctypes.byref(r), ctypes.byref(g), work, need)
        return d


def create_residual_norm(n: int, after: BlockNorm | None = None, before: BlockNorm | None = None, scale: float = 1.0,
                         dtype: str = "f32") -> ResidualNorm:
    """The norm after a block, the gate and residual, and the norm before the next block (ResidualNorm)."""
    return ResidualNorm(n, after, before, scale, dtype)


# -- log probabilities ---------------------------------------------------------------------------


class LogProbabilities:
    """What log_probabilities found: log_probs (None without targets), entropy and log_normalizer float32 [columns],
    top_classes (int32) and top_log_probs (float32) [top_k, columns] (None with top_k = 0)."""

    __slots__ = ("logits", "targets", "log_probs", "entropy", "log_normalizer", "top_classes", "top_log_probs", "_p")

    def backward(self, d_log_probs=None, d_entropy=None, d_log_normalizer=None, out=None):
        """The gradient of the logits from those of log_probs, entropy and log_normalizer (float32 [columns], None:
        zero); out: a tensor for it, of the logits' shape and type, or the logits themselves, which every gradient reads:
        then it is the last one."""
        import torch

        classes, columns = self.logits.shape
        at = []
        for t, what in ((d_log_probs, "d_log_probs"), (d_entropy, "d_entropy"), (d_log_normalizer, "d_log_normalizer")):
            if t is not None:
                _vector(t, what, columns, torch.float32, self.logits)
            at.append(None if t is None else t.data_ptr())
        if out is None:
            out, ld = _empty(self.logits, classes, columns), columns
        else:
            ld = _array(out, "out", self.logits, classes, columns)
        _call(self.logits, A.lib().ponni_log_probs_backward, ctypes.byref(self._p), *at, out.data_ptr(), ld)
        return out


def log_probabilities(logits, targets=None, top_k: int = 0) -> LogProbabilities:
    """Log probabilities of the classes `targets` (int32 [columns]; -1 or any that is no class: none) of logits
    [classes, columns] (f32, f16 or bf16), the entropies, the logarithms of the normalisers and the top_k classes
    (ponni_log_probs)."""
    import torch

    codes = _types()[1]
    ld = _rows(logits, "logits")
    if logits.dtype not in codes:
        raise ValueError(f"logits of type {logits.dtype}")
    classes, columns = logits.shape
    if targets is not None:
        _vector(targets, "targets", columns, torch.int32, logits)
    L = A.lib()
    need = L.ponni_log_probs_workspace_bytes(classes, columns, top_k)
    work, kept = _work(logits, need)  # (of its own: the results outlive it)
    r = LogProbabilities()
    r.logits, r.targets = logits.detach(), targets
    rows = torch.empty((2 + (targets is not None) + 2 * top_k, columns), dtype=torch.float32, device=logits.device)
    r.entropy, r.log_normalizer = rows[0], rows[1]
    r.log_probs = rows[2] if targets is not None else None
    first = 2 + (targets is not None)
    r.top_log_probs = rows[first:first + top_k] if top_k else None
    r.top_classes = rows[first + top_k:].view(torch.int32) if top_k else None
    at = rows.data_ptr()
    of = lambda row: at + 4 * columns * row  # noqa: E731
    r._p = A.LogProbsArrays(classes, columns, logits.data_ptr(), ld, codes[logits.dtype], top_k,
                            None if targets is None else targets.data_ptr(), None if targets is None else of(2), of(0), of(1),
                            of(first + top_k) if top_k else None, of(first) if top_k else None)
    _call(logits, L.ponni_log_probs_forward, ctypes.byref(r._p), work, need)
    return r
