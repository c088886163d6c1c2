"""Routing, expert networks and 4-bit rows over libponni_hip.

    model = create_expert_model(ExpertMatvec(W1), ExpertBias(b1), Silu(n), ExpertMatvec(W2), ExpertBias(b2),
                                dtype="bf16")              # W [experts, n_in, n_out], b [experts, n_out]
    y = model.forward_batch_parallel(x, offsets)           # x [n_in, columns], columns sorted by expert
    routing = route_experts(scores, top_k=2)               # scores [experts, B], e.g. of an Inference model
    y = model.forward_mixture(x, routing)                  # x [n_in, B]

GPU tensors are [features, columns] with contiguous rows, as for
Inference.forward_batch_parallel.  Work buffers are allocated by torch for
each call, on the current stream.
"""
from __future__ import annotations

import ctypes
from dataclasses import dataclass
from typing import Sequence

import numpy as np

from . import _abi as A
from .model import _DTYPES, Inference, Layer, _current_stream

_torch = None  # (dtype name -> torch dtype, torch dtype -> ABI code), filled on first use


def _types():
    global _torch
    if _torch is None:
        import torch

        _torch = ({"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16},
                  {torch.float32: A.F32, torch.float16: A.F16, torch.bfloat16: A.BF16, torch.float64: A.F64})
    return _torch


_current_device = None  # () -> the current device's index


def _call(like, fn, *args) -> None:
    """fn(*args, current stream) with the tensor's device as the current one."""
    global _current_device
    if _current_device is None:
        import torch

        _current_device = getattr(torch._C, "_cuda_getDevice", None) or torch.cuda.current_device
    index = like.get_device()
    if _current_device() == index:
        status = fn(*args, _current_stream(like))
    else:
        import torch

        with torch.cuda.device(index):
            status = fn(*args, _current_stream(like))
    if status != A.PONNI_OK:
        A.check(status)


def _rows(t, what: str, rows: int | None = None, columns: int | None = None):
    """Checks a [features, columns] GPU tensor with contiguous rows; its row stride."""
    shape = t.shape
    if len(shape) != 2 or not t.is_cuda:
        raise ValueError(f"{what} must be a two-dimensional GPU tensor [features, columns]")
    if (rows is not None and shape[0] != rows) or (columns is not None and shape[1] != columns):
        raise ValueError(f"{what} has shape {tuple(shape)}, expected "
                         f"({'any' if rows is None else rows}, {'any' if columns is None else columns})")
    if shape[0] == 0 or shape[1] == 0:
        raise A.PonniError(A.PONNI_ERR_SHAPE, f"{what} of shape {tuple(shape)} is empty")
    stride = t.stride()
    if shape[1] > 1 and stride[1] != 1:
        raise ValueError(f"{what} needs contiguous rows")
    return stride[0] if shape[0] > 1 else shape[1]


def _same_device(t, other, what: str):
    if t.device != other.device:
        raise ValueError(f"{what} is on {t.device}, the input on {other.device}")


def _int_array(t, shape, other, what: str):
    import torch

    if t.dtype != torch.int32 or tuple(t.shape) != tuple(shape) or not t.is_contiguous():
        raise ValueError(f"{what} must be a contiguous int32 tensor of shape {tuple(shape)}")
    _same_device(t, other, what)


# -- routing ---------------------------------------------------------------------------


class Routing:
    """Where the samples of a batch go (ponni_routing): experts (int32), weights
    (float32) and slots (int32) [top_k, batch], source [top_k * batch] and offsets
    [num_experts + 1] (int32), on the GPU.  From route_experts, or a program's own."""

    __slots__ = ("num_experts", "top_k", "batch", "device", "_arrays", "_tensors", "_buffer")

    def __init__(self, experts, weights, slots, source, offsets):
        import torch

        if slots.dim() != 2 or offsets.dim() != 1 or not slots.is_cuda:
            raise ValueError("slots must be a GPU tensor [top_k, batch], offsets [num_experts + 1]")
        self.top_k, self.batch = slots.shape
        self.num_experts, self.device = offsets.shape[0] - 1, slots.get_device()
        _int_array(slots, slots.shape, slots, "slots")
        _int_array(experts, slots.shape, slots, "experts")
        _int_array(source, (self.top_k * self.batch,), slots, "source")
        _int_array(offsets, offsets.shape, slots, "offsets")
        if weights.dtype != torch.float32 or weights.shape != slots.shape or not weights.is_contiguous():
            raise ValueError(f"weights must be a contiguous float32 tensor of shape {tuple(slots.shape)}")
        _same_device(weights, slots, "weights")
        self._tensors = [experts, weights, slots, source, offsets]
        self._arrays = A.RoutingArrays(self.num_experts, self.top_k, self.batch, *[t.data_ptr() for t in self._tensors])

    @classmethod
    def _made(cls, like, num_experts: int, top_k: int, batch: int, work_bytes: int):
        """Arrays to be filled, in one allocation with a work buffer behind them; its address."""
        import torch

        r = cls.__new__(cls)
        r.num_experts, r.top_k, r.batch, r.device, r._tensors = num_experts, top_k, batch, like.get_device(), [None] * 5
        n = top_k * batch
        work = (4 * n + num_experts + 4) // 4 * 4  # (16-byte aligned)
        r._buffer = torch.empty(work + work_bytes // 4, dtype=torch.int32, device=like.device)
        at = r._buffer.data_ptr()
        r._arrays = A.RoutingArrays(num_experts, top_k, batch, at, at + 4 * n, at + 8 * n, at + 12 * n, at + 16 * n)
        return r, at + 4 * work

    def _tensor(self, i: int):
        t = self._tensors[i]
        if t is None:  # a view of the buffer, made when it is asked for
            k, b = self.top_k, self.batch
            if i < 3:
                t = self._buffer.as_strided((k, b), (b, 1), i * k * b)
                if i == 1:
                    import torch

                    t = t.view(torch.float32)
            else:
                t = self._buffer.as_strided((k * b if i == 3 else self.num_experts + 1,), (1,), i * k * b)
            self._tensors[i] = t
        return t

    experts = property(lambda self: self._tensor(0))
    weights = property(lambda self: self._tensor(1))
    slots = property(lambda self: self._tensor(2))
    source = property(lambda self: self._tensor(3))
    offsets = property(lambda self: self._tensor(4))

    def arrays(self) -> A.RoutingArrays:
        return self._arrays


def route_experts(scores, top_k: int, normalize: str = "chosen") -> Routing:
    """The top_k experts of each sample from scores [num_experts, batch] (f32, f16
    or bf16), and the samples sorted by expert (ponni_route).  normalize: the
    weights are softmax values over the sample's "chosen" experts or over "all"."""
    codes = _types()[1]
    ld = _rows(scores, "scores")
    if scores.dtype not in codes:
        raise ValueError(f"scores of type {scores.dtype}")
    if normalize not in ("chosen", "all"):
        raise ValueError(f"normalize must be 'chosen' or 'all', not {normalize!r}")
    e, b = scores.shape
    L = A.lib()
    need = L.ponni_route_workspace_bytes(e, top_k, b)
    if need < 0:
        raise A.PonniError(A.PONNI_ERR_INVALID_ARGUMENT, L.ponni_last_error().decode())
    r, work = Routing._made(scores, e, top_k, b, need)
    _call(scores, L.ponni_route, scores.data_ptr(), ld, codes[scores.dtype], A.ROUTE_ALL if normalize == "all" else
          A.ROUTE_CHOSEN, ctypes.byref(r._arrays), work, need)
    return r


# -- 4-bit rows ------------------------------------------------------------------------


def _mx4_bytes(features: int):
    """Bytes of a row's codes and of its scales (ponni_mx4_code_bytes, ponni_mx4_scale_bytes)."""
    steps = -(-features // 128)
    return 64 * steps, 4 * steps


class Mx4:
    """Samples as microscaled 4-bit rows (ponni_mx4_quantize): codes [columns,
    code bytes] and scales [columns, scale bytes], uint8."""

    __slots__ = ("codes", "scales", "features", "columns")

    def __init__(self, codes, scales, features: int):
        import torch

        for t, n, what in zip((codes, scales), _mx4_bytes(features), ("codes", "scales")):
            if t.dtype != torch.uint8 or tuple(t.shape) != (codes.shape[0], n) or not t.is_contiguous() or not t.is_cuda:
                raise ValueError(f"{what} must be a contiguous uint8 GPU tensor of shape ({codes.shape[0]}, {n})")
        _same_device(scales, codes, "scales")
        self._set(codes, scales, features)

    def _set(self, codes, scales, features: int):
        self.codes, self.scales, self.features, self.columns = codes, scales, features, codes.shape[0]
        return self

    def dequantize(self, dtype=None):
        """The values as a [features, columns] tensor (float32, float16 or bfloat16)."""
        import torch

        y = torch.empty((self.features, self.columns), dtype=dtype or torch.float32, device=self.codes.device)
        if y.dtype not in _types()[1]:
            raise ValueError(f"values of type {y.dtype}")
        _call(y, A.lib().ponni_mx4_dequantize, self.codes.data_ptr(), self.scales.data_ptr(), self.features, self.columns,
              y.data_ptr(), self.columns, _types()[1][y.dtype])
        return y


def quantize_mx4(x) -> Mx4:
    """x [features, columns] (f32, f16 or bf16) in microscaled 4-bit floating
    point: blocks of 32 features of a sample share a power-of-two scale."""
    import torch

    ld = _rows(x, "x")
    if x.dtype not in _types()[1]:
        raise ValueError(f"x of type {x.dtype}")
    k, n = x.shape
    L = A.lib()
    code_bytes, scale_bytes = _mx4_bytes(k)
    q = Mx4.__new__(Mx4)._set(torch.empty((n, code_bytes), dtype=torch.uint8, device=x.device),
                              torch.empty((n, scale_bytes), dtype=torch.uint8, device=x.device), k)
    _call(x, L.ponni_mx4_quantize, x.data_ptr(), ld, _types()[1][x.dtype], k, n, q.codes.data_ptr(), q.scales.data_ptr())
    return q


# -- expert networks ---------------------------------------------------------------------


def _host_or_device(values, dims: int, what: str):
    """A contiguous numpy array or torch tensor of `dims` dimensions."""
    if hasattr(values, "data_ptr"):
        values = values.detach()
        v = values.contiguous() if values.dtype in _types()[1] else values.double().contiguous()
    else:
        v = np.ascontiguousarray(values)
        if v.dtype not in (np.float32, np.float64, np.float16):
            v = v.astype(np.float64)
    if len(v.shape) != dims:
        raise ValueError(f"{what} must have {dims} dimensions, got shape {tuple(v.shape)}")
    return v


@dataclass
class ExpertLayer(Layer):
    """A layer with parameters of every expert: `values`, a numpy array or torch tensor."""

    values: "object" = None


def ExpertMatvec(weights) -> ExpertLayer:
    """One Matvec per expert: weights [experts, n_in, n_out] (numpy or torch, host or GPU)."""
    w = _host_or_device(weights, 3, "ExpertMatvec weights")
    return ExpertLayer(A.LAYER_MATVEC, w.shape[1], w.shape[2], label="Matvec", values=w)


def ExpertBias(bias) -> ExpertLayer:
    """One Bias per expert: bias [experts, n]."""
    b = _host_or_device(bias, 2, "ExpertBias values")
    return ExpertLayer(A.LAYER_BIAS, b.shape[1], b.shape[1], label="Bias", values=b)


class ExpertInference:
    """Networks of one architecture, one per expert (ponni_experts).  The layers'
    arrays are read by the constructor and not kept."""

    def __init__(self, layers: Sequence[Layer], dtype: str = "f32", weights: str = "same"):
        if weights not in ("same", "mx4"):
            raise ValueError(f"weights must be 'same' or 'mx4', not {weights!r}")
        held = [l for l in layers if getattr(l, "values", None) is not None]
        if any(l.kind in (A.LAYER_MATVEC, A.LAYER_BIAS) and getattr(l, "values", None) is None for l in layers):
            # (its parameters would reach no expert)
            raise A.PonniError(A.PONNI_ERR_INVALID_MODEL, "a Matvec or Bias of one network: use ExpertMatvec or ExpertBias")
        if not held:
            raise A.PonniError(A.PONNI_ERR_INVALID_MODEL, "the chain must begin with a Matvec")
        self.num_experts = int(held[0].values.shape[0])
        if any(l.values.shape[0] != self.num_experts for l in held):
            raise A.PonniError(A.PONNI_ERR_INVALID_MODEL, "the layers hold parameters of different numbers of experts")
        self.dtype, self.weights = dtype, weights
        self.n_in, self.n_out = layers[0].n_in, layers[-1].n_out
        descs = (A.LayerDesc * len(layers))(*[l.desc() for l in layers])
        self._shapes = {i: tuple(l.values.shape) for i, l in enumerate(layers) if getattr(l, "values", None) is not None}
        self._experts = ctypes.c_void_p()
        A.check(A.lib().ponni_experts_create(descs, len(layers), self.num_experts, _DTYPES[dtype],
                                             A.WEIGHTS_MX4 if weights == "mx4" else A.WEIGHTS_SAME,
                                             ctypes.byref(self._experts)))
        params = [(i, l.values) for i, l in enumerate(layers) if getattr(l, "values", None) is not None]
        import torch

        # On the GPU of the first array that is on one, or the current one.
        self.device = next((v.get_device() for _, v in params if hasattr(v, "data_ptr") and v.is_cuda), None)
        if self.device is None and torch.cuda.is_available():
            self.device = torch.cuda.current_device()
        if self.device is not None:
            for i, v in params:
                self.set_layer_params(i, v)

    def __del__(self):
        e = getattr(self, "_experts", None)
        if e is not None and e.value:
            try:
                A.lib().ponni_experts_destroy(e)
            except (AttributeError, TypeError):  # interpreter shutdown: the module is gone
                pass
            self._experts = None

    def set_layer_params(self, i: int, values) -> None:
        """All experts' parameters of layer i (numpy or torch, host or any GPU), in the
        layer's shape or as one dimension.  Waits for the device: calls made before, on
        any stream, read the old ones."""
        import torch

        shape = tuple(values.shape if hasattr(values, "shape") else np.shape(values))
        if len(shape) > 1 and shape != self._shapes.get(i, shape):
            raise ValueError(f"layer {i} holds parameters of shape {self._shapes[i]}, got {shape}")
        if hasattr(values, "data_ptr"):
            v = values.detach()
            if v.is_cuda and v.get_device() != self.device:
                v = v.to(f"cuda:{self.device}")
            v = v.contiguous() if v.dtype in _types()[1] else v.double().contiguous()
            code, ptr, n, on_device = _types()[1][v.dtype], v.data_ptr(), v.numel(), int(v.is_cuda)
        else:
            v = np.ascontiguousarray(values)
            v = v if v.dtype in (np.float32, np.float64, np.float16) else v.astype(np.float64)
            code = {np.dtype(np.float32): A.F32, np.dtype(np.float64): A.F64, np.dtype(np.float16): A.F16}[v.dtype]
            ptr, n, on_device = v.ctypes.data, v.size, 0
        with torch.cuda.device(self.device):
            stream = torch.cuda.current_stream().cuda_stream
            A.check(A.lib().ponni_experts_set_layer_params(self._experts, i, ptr, code, n, on_device, stream))

    def get_num_inputs(self) -> int:
        return self.n_in

    def get_num_outputs(self) -> int:
        return self.n_out

    def _buffers(self, like, columns, y):
        import torch

        dtype = _types()[0][self.dtype]
        if y is None:
            return torch.empty((self.n_out, columns), dtype=dtype, device=like.device), columns
        ld = _rows(y, "y", self.n_out, columns)
        if y.dtype != dtype:
            raise ValueError(f"y is {y.dtype}, the model {dtype}")
        _same_device(y, like, "y")
        return y, ld

    def forward_batch_parallel(self, x, offsets=None, y=None):
        """x [n_in, columns] of the model's type, or Mx4 rows (4-bit weights), columns
        sorted by expert; offsets int32 [num_experts + 1] on the GPU (None with one
        expert: all columns).  Returns y [n_out, columns]; columns in no group are
        left as they were (undefined in a new y)."""
        import torch

        L = A.lib()
        rows = isinstance(x, Mx4)
        if rows:
            like, columns = x.codes, x.columns
            if x.features != self.n_in:
                raise ValueError(f"x has {x.features} features, the model {self.n_in} inputs")
        else:
            like, columns = x, x.shape[1] if x.dim() == 2 else 0
            ld_in = _rows(x, "x", self.n_in)
            if x.dtype != _types()[0][self.dtype]:
                raise ValueError(f"x is {x.dtype}, the model {_types()[0][self.dtype]}")
        if offsets is not None:
            _int_array(offsets, (self.num_experts + 1,), like, "offsets")
        y, ld = self._buffers(like, columns, y)
        need = L.ponni_experts_workspace_bytes(self._experts, columns)
        work = torch.empty(max(need, 1), dtype=torch.uint8, device=like.device)
        at = 0 if offsets is None else offsets.data_ptr()
        if rows:
            _call(like, L.ponni_experts_forward_mx4, self._experts, x.codes.data_ptr(), x.scales.data_ptr(), at,
                  y.data_ptr(), ld, columns, work.data_ptr(), need)
        else:
            _call(like, L.ponni_experts_forward, self._experts, x.data_ptr(), ld_in, at, y.data_ptr(), ld, columns,
                  work.data_ptr(), need)
        return y

    def forward_mixture(self, x, routing: Routing, y=None):
        """x [n_in, batch]: the weighted sum of each sample's experts (ponni_experts_forward_mixture)."""
        import torch

        L = A.lib()
        ld_in = _rows(x, "x", self.n_in, routing.batch)
        if x.dtype != _types()[0][self.dtype]:
            raise ValueError(f"x is {x.dtype}, the model {_types()[0][self.dtype]}")
        if routing.device != x.get_device():
            raise ValueError(f"routing is on GPU {routing.device}, the input on {x.device}")
        y, ld = self._buffers(x, routing.batch, y)
        need = L.ponni_experts_mixture_workspace_bytes(self._experts, routing.top_k, routing.batch)
        work = torch.empty(max(need, 1), dtype=torch.uint8, device=x.device)
        _call(x, L.ponni_experts_forward_mixture, self._experts, x.data_ptr(), ld_in, ctypes.byref(routing._arrays),
              y.data_ptr(), ld, work.data_ptr(), need)
        return y


def create_expert_model(*layers: Layer, dtype: str = "f32", weights: str = "same") -> ExpertInference:
    """ExpertMatvec, each followed by an optional ExpertBias and an optional
    activation (no Matvec or Bias of one network).  dtype "f32", "f16" or "bf16"; weights "same" (as dtype) or "mx4"
    (weights and every layer's input in 4 bits)."""
    return ExpertInference(layers, dtype=dtype, weights=weights)


class MixtureOfExperts:
    """A router (an Inference model of num_experts outputs), and the experts it chooses among.

        model = MixtureOfExperts(create_inference_model(Matvec(R), dtype="bf16"), experts, top_k=2)
        y = model.forward_batch_parallel(x)
    """

    def __init__(self, router: Inference, experts: ExpertInference, top_k: int, normalize: str = "chosen"):
        if router.get_num_outputs() != experts.num_experts:
            raise A.PonniError(A.PONNI_ERR_INVALID_MODEL, "the router's outputs are not the experts")
        if router.get_num_inputs() != experts.get_num_inputs() or router.dtype != experts.dtype:
            raise A.PonniError(A.PONNI_ERR_INVALID_MODEL, "router and experts take different inputs")
        self.router, self.experts, self.top_k, self.normalize = router, experts, top_k, normalize

    def forward_batch_parallel(self, x, y=None):
        routing = route_experts(self.router.forward_batch_parallel(x), self.top_k, self.normalize)
        return self.experts.forward_mixture(x, routing, y)
