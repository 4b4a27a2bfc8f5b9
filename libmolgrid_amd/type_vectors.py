"""Learned type vectors: from type indices to the vectors that vector-typed gridding takes, and back.

The reference's type vectors are one-hot rows (``CoordinateSet.make_vector_types``) or come from a
typer; its gridding gives gradients of them (python/torch_bindings.py:44-100) that nothing there
learns from.  The functions below look vectors up in a table by type index, norm them and drop parts
of them out, each with its gradients; ``TypeEncoder`` does the three in one pass and plugs into
``Coords2Grid(gmaker, center, type_encoder=...)``, whose grids are then differentiable in the table.

    embed_types / embed_types_backward        rows of a table, scaled; gradients of table and scale
    layer_norm / layer_norm_backward          layer norm over the channels
    dropout                                   counter-based: the mask is a function of seed, offset
                                              and position, the gradient the same call on it
    encode_types / encode_types_backward      dropout(layer_norm(scale * table[type_index]))

These functions compute and return tensors; the modules ``TypeEmbedding``, ``TypeNorm``,
``TypeDropout`` and ``TypeEncoder`` (and the ``...Function`` classes under them) are what autograd
differentiates.  Vectors, tables and gradients are float32, float16 or bfloat16, contiguous, on the
current device; host tensors and numpy arrays are staged through the device and come back as host
tensors.  Type indices are float32 (as coordinate sets keep them: the whole number below counts),
int32 or int64 of any shape; an index that names no row gives a row of zeros and no gradient.
Everything runs on torch's current stream, nothing synchronises.
"""
import functools
import math
import threading

import numpy as np
import torch
from torch.autograd.function import once_differentiable

from . import _capi
from . import gridding as _gr

_DTYPES = {torch.float32: _capi.MG_FLOAT32, torch.float16: _capi.MG_FLOAT16,
           torch.bfloat16: _capi.MG_BFLOAT16}
_INDICES = {torch.float32: _capi.MG_INDEX_FLOAT32, torch.int32: _capi.MG_INDEX_INT32,
            torch.int64: _capi.MG_INDEX_INT64}


# --------------------------------------------------------------------------- #
# arguments
# --------------------------------------------------------------------------- #
def _is_array(x):
    return isinstance(x, (torch.Tensor, np.ndarray))


def _staged(fn):
    """Grid views and managed grids stand for their tensors; where every array is a host array the
    call runs on copies on the device and its tensors come back to the host."""
    @functools.wraps(fn)
    def wrapper(*args, **kw):
        first = args[0] if args else None
        if isinstance(first, torch.Tensor) and first.is_cuda:
            return fn(*args, **kw)
        args = [_gr._unwrap(a) for a in args]
        kw = {k: _gr._unwrap(v) for k, v in kw.items()}
        arrays = [a for a in list(args) + list(kw.values()) if _is_array(a)]
        if any(isinstance(a, torch.Tensor) and a.is_cuda for a in arrays):
            return fn(*args, **kw)

        def there(a):
            return torch.as_tensor(a).detach().to(device=_gr._device()) if _is_array(a) else a

        def back(r):
            if isinstance(r, tuple):
                return tuple(back(x) for x in r)
            return r.cpu() if isinstance(r, torch.Tensor) else r
        return back(fn(*[there(a) for a in args], **{k: there(v) for k, v in kw.items()}))
    return wrapper


def _tensor(x, name, dtypes):
    """The checks of gridding's device arrays (python/bindings_grids.cpp:91-137): a contiguous
    tensor of a supported type on the current device."""
    if not isinstance(x, torch.Tensor):
        x = _gr._unwrap(x)
        if not isinstance(x, torch.Tensor):
            raise ValueError("%s: expected a tensor" % name)
    if x.dtype in dtypes and x.is_cuda and x.get_device() == torch.cuda.current_device() and x.is_contiguous():
        return x
    if x.dtype not in dtypes:
        raise ValueError("%s: %s is not supported here" % (name, x.dtype))
    if not x.is_cuda:
        raise ValueError("%s: tensor is on the host, others are on the device" % name)
    if x.get_device() != torch.cuda.current_device():
        raise ValueError("%s: tensor is on device %d but the current device is %d"
                         % (name, x.get_device(), torch.cuda.current_device()))
    raise ValueError("%s: tensor is not contiguous" % name)


def _ptr(x):
    return None if x is None else x.data_ptr()


def _empty(shape, like, dtype=None):
    return like.new_empty(shape) if dtype is None else like.new_empty(shape, dtype=dtype)


def _workspace(size, like):
    """Device memory of one call: the allocator hands it to later work of this stream only, and a
    captured graph's calls get theirs from that graph's pool."""
    return like.new_empty(size, dtype=torch.uint8) if size else None


# bytes of workspace by sizes (a call into the library costs as much as four tensor attributes)
@functools.lru_cache(maxsize=256)
def _workspace_size(entry, *sizes):
    return getattr(_capi.lib, entry + "_workspace_size")(*sizes)


def _count(n, name):
    if n >= 2 ** 31:
        raise ValueError("%s: sizes of 2^31 and more are not supported" % name)
    return n


def _table_args(type_index, table):
    index = _tensor(type_index, "type_index", _INDICES)
    table = _tensor(table, "table", _DTYPES)
    if table.dim() != 2:
        raise ValueError("table: expected 2 dimensions, got %d" % table.dim())
    return index, table, (_count(index.numel(), "type_index"), _count(table.shape[0], "table"),
                          _count(table.shape[1], "table"))


def _scale_args(scale, index):
    """(number, per-token tensor or None)"""
    scale = _gr._unwrap(scale)
    if _is_array(scale):
        scale = _tensor(scale, "scale", (torch.float32,))
        if scale.shape != index.shape:
            raise ValueError("scale: expected the shape of type_index, %s, got %s"
                             % (tuple(index.shape), tuple(scale.shape)))
        return 1.0, scale
    return float(scale), None


def _param(x, name, channels, dtype, like=None):
    if x is None:
        return None
    x = _tensor(x, name, _DTYPES)
    if x.shape != (channels,):
        raise ValueError("%s: expected shape (%d,), got %s" % (name, channels, tuple(x.shape)))
    if x.dtype not in (torch.float32, dtype) or (like is not None and x.dtype != like.dtype):
        raise ValueError("%s: parameters are float32 or of the vectors' type, and alike" % name)
    return x


def _param_gradients(weight, channels, like):
    first = torch.empty_like(weight) if weight is not None else _empty((channels,), like, torch.float32)
    return first, torch.empty_like(first)


def _like(grad, name, shape, dtype):
    grad = _tensor(grad, name, (dtype,))
    if grad.shape != shape:
        raise ValueError("%s: expected shape %s, got %s" % (name, tuple(shape), tuple(grad.shape)))
    return grad


def _number(x, name):
    if _is_array(_gr._unwrap(x)):
        raise ValueError("%s: expected a number" % name)
    return float(x)


def _eps(eps):
    eps = float(eps)
    if not (eps >= 0 and math.isfinite(eps)):
        raise ValueError("eps: expected a finite number of at least 0, got %r" % eps)
    return eps


def _drop_args(p, seed, offset, state):
    p = float(p)
    if not 0 <= p <= 1:
        raise ValueError("p: expected a probability, got %r" % p)
    if state is not None:
        state = _tensor(state, "state", (torch.int64,))
        if tuple(state.shape) != (2,):
            raise ValueError("state: expected two numbers, seed and offset")
    seed, offset = int(seed), int(offset)
    if not (0 <= seed < 2 ** 64 and 0 <= offset < 2 ** 64):
        raise ValueError("seed and offset: expected numbers of 64 bits")
    return p, seed, offset, _ptr(state)


# --------------------------------------------------------------------------- #
# the operators
# --------------------------------------------------------------------------- #
@_staged
def embed_types(type_index, table, scale=1.0):
    """Rows of ``table`` (types, channels) by type index, times ``scale``: a number, or a float32
    tensor with one factor for each index.  Result: the shape of type_index, then channels."""
    index, table, (n, rows, channels) = _table_args(type_index, table)
    number, scales = _scale_args(scale, index)
    out = _empty(tuple(index.shape) + (channels,), table)
    _capi.check(_capi.lib.mg_embed_types(
        n, rows, channels, _DTYPES[table.dtype], _INDICES[index.dtype], _ptr(index), _ptr(table),
        number, _ptr(scales), _ptr(out), _gr._stream()), "embed_types")
    return out


@_staged
def embed_types_backward(grad, type_index, table, scale=1.0, table_gradient=True,
                         scale_gradient=True):
    """Gradients of ``embed_types`` for the upstream gradient ``grad``: (of the table, of the scale).
    The second is None for a scale that is a number; both can be left out.  The table's gradient is
    summed in float32 in a fixed order and rounded once."""
    index, table, (n, rows, channels) = _table_args(type_index, table)
    number, scales = _scale_args(scale, index)
    grad = _like(grad, "grad", tuple(index.shape) + (channels,), table.dtype)
    to_table = torch.empty_like(table) if table_gradient else None
    to_scale = _empty(index.shape, table, torch.float32) if scale_gradient and scales is not None \
        else None
    size = _workspace_size("mg_embed_types_backward", n, rows, channels) if table_gradient else 0
    workspace = _workspace(size, table)
    _capi.check(_capi.lib.mg_embed_types_backward(
        n, rows, channels, _DTYPES[table.dtype], _INDICES[index.dtype], _ptr(index), _ptr(grad),
        _ptr(table), number, _ptr(scales), _ptr(to_table), _ptr(to_scale), _ptr(workspace), size,
        _gr._stream()), "embed_types_backward")
    return to_table, to_scale


def _norm_sizes(x):
    x = _tensor(x, "x", _DTYPES)
    if x.dim() < 1:
        raise ValueError("x: expected at least one dimension")
    channels = _count(x.shape[-1], "x")
    return x, _count(x.numel() // channels if channels else 0, "x"), channels


@_staged
def layer_norm(x, weight=None, bias=None, eps=1e-5):
    """Layer norm over the last dimension: (result, mean, rstd).  The last two are float32, one
    number a row, for ``layer_norm_backward``."""
    x, rows, channels = _norm_sizes(x)
    weight = _param(weight, "weight", channels, x.dtype)
    bias = _param(bias, "bias", channels, x.dtype, weight)
    params = weight if weight is not None else bias
    out = torch.empty_like(x)
    mean = _empty(x.shape[:-1], x, torch.float32)
    rstd = torch.empty_like(mean)
    if channels == 0:
        mean.zero_(), rstd.zero_()
    _capi.check(_capi.lib.mg_layer_norm(
        rows, channels, _DTYPES[x.dtype], _DTYPES[params.dtype if params is not None else torch.float32],
        _ptr(x), _ptr(weight), _ptr(bias), _eps(eps), _ptr(out), _ptr(mean), _ptr(rstd),
        _gr._stream()), "layer_norm")
    return out, mean, rstd


@_staged
def layer_norm_backward(grad, x, mean, rstd, weight=None, input_gradient=True,
                        param_gradients=True):
    """Gradients of ``layer_norm`` for the upstream gradient ``grad``: (of x, of weight, of bias).
    Those of the parameters have weight's type (float32 without one); what is not asked for is
    None."""
    x, rows, channels = _norm_sizes(x)
    grad = _like(grad, "grad", x.shape, x.dtype)
    rows_shape = x.shape[:-1]
    mean = _like(mean, "mean", rows_shape, torch.float32)
    rstd = _like(rstd, "rstd", rows_shape, torch.float32)
    weight = _param(weight, "weight", channels, x.dtype)
    params = weight.dtype if weight is not None else torch.float32
    to_x = torch.empty_like(x) if input_gradient else None
    to_weight, to_bias = _param_gradients(weight, channels, x) if param_gradients else (None, None)
    size = _workspace_size("mg_layer_norm_backward", rows, channels) if param_gradients else 0
    workspace = _workspace(size, x)
    _capi.check(_capi.lib.mg_layer_norm_backward(
        rows, channels, _DTYPES[x.dtype], _DTYPES[params], _ptr(grad), _ptr(x), _ptr(mean),
        _ptr(rstd), _ptr(weight), _ptr(to_x), _ptr(to_weight), _ptr(to_bias), _ptr(workspace), size,
        _gr._stream()), "layer_norm_backward")
    return to_x, to_weight, to_bias


@_staged
def dropout(x, p, seed=0, offset=0, state=None):
    """``x`` with each element dropped (set to zero) with probability p and the others scaled up so
    that the expectation stays; p counts in steps of 2^-16.  Which elements are kept is a function
    of (seed, offset) and their position in the flattened tensor: other calls take another seed or
    offset (numbers of 64 bits), the backward pass the same ones on the gradient.  ``state``, an
    int64 tensor of two numbers on the device, is added to seed and offset (modulo 2^64), so that a
    captured graph can be replayed with other numbers."""
    x = _tensor(x, "x", _DTYPES)
    p, seed, offset, state_ptr = _drop_args(p, seed, offset, state)
    out = torch.empty_like(x)
    _capi.check(_capi.lib.mg_dropout(x.numel(), _DTYPES[x.dtype], _ptr(x), p, seed, offset, state_ptr,
                                     _ptr(out), _gr._stream()), "dropout")
    return out


@_staged
def encode_types(type_index, table, weight=None, bias=None, scale=1.0, eps=1e-5, p=0.0, seed=0,
                 offset=0, state=None):
    """``dropout(layer_norm(scale * table[type_index], weight, bias, eps), p, seed, offset)`` in one
    pass, rounded once; ``scale`` is a number.  An index that names no row gives zeros."""
    index, table, (n, rows, channels) = _table_args(type_index, table)
    weight = _param(weight, "weight", channels, table.dtype)
    bias = _param(bias, "bias", channels, table.dtype, weight)
    params = weight if weight is not None else bias
    p, seed, offset, state_ptr = _drop_args(p, seed, offset, state)
    out = _empty(tuple(index.shape) + (channels,), table)
    _capi.check(_capi.lib.mg_encode_types(
        n, rows, channels, _DTYPES[table.dtype],
        _DTYPES[params.dtype if params is not None else torch.float32], _INDICES[index.dtype],
        _ptr(index), _ptr(table), _number(scale, "scale"), _ptr(weight), _ptr(bias), _eps(eps), p, seed, offset,
        state_ptr, _ptr(out), _gr._stream()), "encode_types")
    return out


@_staged
def encode_types_backward(grad, type_index, table, weight=None, scale=1.0, eps=1e-5, p=0.0, seed=0,
                          offset=0, state=None, table_gradient=True, param_gradients=True):
    """Gradients of ``encode_types`` for the upstream gradient ``grad`` and the same numbers:
    (of the table, of weight, of bias); what is not asked for is None."""
    index, table, (n, rows, channels) = _table_args(type_index, table)
    grad = _like(grad, "grad", tuple(index.shape) + (channels,), table.dtype)
    weight = _param(weight, "weight", channels, table.dtype)
    params = weight.dtype if weight is not None else torch.float32
    p, seed, offset, state_ptr = _drop_args(p, seed, offset, state)
    to_table = torch.empty_like(table) if table_gradient else None
    to_weight, to_bias = _param_gradients(weight, channels, table) if param_gradients else (None, None)
    size = _workspace_size("mg_encode_types_backward", n, rows, channels)
    workspace = _workspace(size, table)
    _capi.check(_capi.lib.mg_encode_types_backward(
        n, rows, channels, _DTYPES[table.dtype], _DTYPES[params], _INDICES[index.dtype], _ptr(index),
        _ptr(grad), _ptr(table), _number(scale, "scale"), _ptr(weight), _eps(eps), p, seed, offset, state_ptr,
        _ptr(to_table), _ptr(to_weight), _ptr(to_bias), _ptr(workspace), size, _gr._stream()),
        "encode_types_backward")
    return to_table, to_weight, to_bias


# --------------------------------------------------------------------------- #
# autograd
# --------------------------------------------------------------------------- #
class TypeEmbeddingFunction(torch.autograd.Function):
    """type indices, table (T,C), scale (a number or one per index) -> type vectors."""

    @staticmethod
    def forward(ctx, type_index, table, scale):
        per_token = _is_array(scale)
        ctx.save_for_backward(type_index, table, scale if per_token else None)
        ctx.scale = None if per_token else float(scale)
        return embed_types(type_index, table, scale)

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        type_index, table, scale = ctx.saved_tensors
        to_table, to_scale = embed_types_backward(
            grad.contiguous(), type_index, table, ctx.scale if scale is None else scale,
            ctx.needs_input_grad[1], ctx.needs_input_grad[2])
        return None, to_table, to_scale


class TypeNormFunction(torch.autograd.Function):
    """vectors (..., C), weight (C) or None, bias (C) or None, eps -> normed vectors."""

    @staticmethod
    def forward(ctx, x, weight, bias, eps):
        out, mean, rstd = layer_norm(x, weight, bias, eps)
        ctx.save_for_backward(x, weight, mean, rstd)
        ctx.bias_dtype = bias.dtype if bias is not None else None
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        x, weight, mean, rstd = ctx.saved_tensors
        to_x, to_weight, to_bias = layer_norm_backward(
            grad.contiguous(), x, mean, rstd, weight, ctx.needs_input_grad[0],
            ctx.needs_input_grad[1] or ctx.needs_input_grad[2])
        return (to_x, to_weight if ctx.needs_input_grad[1] else None,
                to_bias.to(ctx.bias_dtype) if ctx.needs_input_grad[2] else None, None)


class TypeDropoutFunction(torch.autograd.Function):
    """vectors, p, seed, offset, state (or None) -> vectors with dropped elements."""

    @staticmethod
    def forward(ctx, x, p, seed, offset, state):
        # (autograd refuses the backward pass if state was changed in between)
        ctx.save_for_backward(state)
        ctx.numbers = p, seed, offset
        return dropout(x, p, seed, offset, state)

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        return (dropout(grad.contiguous(), *ctx.numbers, ctx.saved_tensors[0]), None, None, None,
                None)


class TypeEncoderFunction(torch.autograd.Function):
    """type indices, table (T,C), weight (C), bias (C), scale, eps, p, seed, offset, state -> vectors."""

    @staticmethod
    def forward(ctx, type_index, table, weight, bias, scale, eps, p, seed, offset, state):
        ctx.save_for_backward(type_index, table, weight, state)
        ctx.numbers = scale, eps, p, seed, offset
        ctx.bias_dtype = bias.dtype if bias is not None else None
        return encode_types(type_index, table, weight, bias, *ctx.numbers, state)

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        type_index, table, weight, state = ctx.saved_tensors
        need = ctx.needs_input_grad
        to_table, to_weight, to_bias = encode_types_backward(
            grad.contiguous(), type_index, table, weight, *ctx.numbers, state, need[1],
            need[2] or need[3])
        return (None, to_table, to_weight if need[2] else None,
                to_bias.to(ctx.bias_dtype) if need[3] else None) + (None,) * 6


def _new_seed():
    """From the package's random source (set_random_seed makes it repeatable)."""
    return int(_gr._rng.integers(0, 2 ** 63))


class _Calls(object):
    """Number of a module's calls so far.  Replicas of the module (nn.DataParallel makes new ones for every
    step) go on with the same one, copies with one of their own."""

    def __init__(self, made=0):
        self.made = made
        self.lock = threading.Lock()

    def __reduce__(self):
        return _Calls, (self.made,)

    def take(self):
        with self.lock:
            self.made += 1
            return self.made - 1


class _Drawing(torch.nn.Module):
    """Seed and offsets of a module that drops.

    With a seed, call k while training has offset k.  Without one the seed comes from the package's
    random source and every call draws its offset from torch's generator of the host, which
    activation checkpointing restores before it runs a call again (unless told not to,
    ``preserve_rng_state``): the repeated call drops the same elements.  A count cannot know of the
    repetition, so a module with a seed refuses calls during a backward pass; a call that is given
    its ``offset`` takes that one in any case.  Seed and count are part of the module's state_dict.

    ``state``, an int64 tensor of two numbers on the device, is added to the seed and to an offset of 0
    (or the one that the call is given), for calls that are captured into a graph; whoever replays the
    graph changes it between the replays (or inside it, behind the backward pass).  Modules that share
    a state drop other elements by their seeds; several calls of one module under the same numbers are
    given an offset each."""

    def _open(self, p, seed, state):
        if not 0 <= float(p) <= 1:
            raise ValueError("p: expected a probability, got %r" % p)
        self.p = float(p)
        self._counts = seed is not None
        self.seed = _new_seed() if seed is None else int(seed)
        if not 0 <= self.seed < 2 ** 64:
            raise ValueError("seed: expected a number of 64 bits")
        self._calls = _Calls()
        self.state = state

    @property
    def offset(self):
        """Calls so far of a module with a seed: the offset of the next one"""
        return self._calls.made

    @offset.setter
    def offset(self, value):
        self._calls.made = int(value)

    def _next_offset(self):
        if not self._counts:
            return int(torch.randint(2 ** 63 - 1, (), dtype=torch.int64, device="cpu"))
        if torch._C._current_graph_task_id() != -1:
            raise RuntimeError("a call during a backward pass, which may repeat an earlier one: give "
                               "the call its offset, or the module no seed")
        return self._calls.take()

    def _numbers(self, on_device, offset):
        """(p, seed, offset, state) of the next call"""
        if not self.training or self.p == 0:
            return 0.0, 0, 0, None
        if self.state is not None:
            return self.p, self.seed, 0 if offset is None else int(offset), self.state
        if on_device and torch.cuda.is_current_stream_capturing():
            raise RuntimeError("a captured graph would drop the same elements in every replay: "
                               "give the module a state tensor")
        return self.p, self.seed, self._next_offset() if offset is None else int(offset), None

    def get_extra_state(self):
        """(seed, calls so far), 64 bits each"""
        seed = self.seed - 2 ** 64 if self.seed >= 2 ** 63 else self.seed
        return torch.tensor([seed, self._calls.made], dtype=torch.int64, device="cpu")

    def set_extra_state(self, state):
        seed, made = (int(n) for n in state)
        self.seed, self._calls.made = seed % 2 ** 64, made

    def _load_from_state_dict(self, state_dict, prefix, local_metadata, strict, missing_keys, *others):
        super()._load_from_state_dict(state_dict, prefix, local_metadata, strict, missing_keys, *others)
        key = prefix + "_extra_state"
        if key in missing_keys:     # (of a module that kept no numbers: those here stay)
            missing_keys.remove(key)


class TypeEmbedding(torch.nn.Module):
    """Layer turning type indices into rows of a learned table times ``scale``; a second argument of
    the call gives a factor for each index instead."""

    def __init__(self, ntypes, channels, scale=1.0, dtype=None, device=None):
        super().__init__()
        self.weight = torch.nn.Parameter(torch.empty((ntypes, channels), dtype=dtype, device=device))
        self.scale = float(scale)
        torch.nn.init.normal_(self.weight)

    def forward(self, type_index, scale=None):
        scale = self.scale if scale is None else scale
        if _is_array(scale):
            scale = scale.contiguous()
        return TypeEmbeddingFunction.apply(type_index.contiguous(), self.weight.contiguous(), scale)

    def extra_repr(self):
        return "%d types, %d channels" % tuple(self.weight.shape)


class TypeNorm(torch.nn.Module):
    """Layer norm over the channels of type vectors, with a learned weight and bias."""

    def __init__(self, channels, eps=1e-5, dtype=None, device=None):
        super().__init__()
        self.weight = torch.nn.Parameter(torch.ones(channels, dtype=dtype, device=device))
        self.bias = torch.nn.Parameter(torch.zeros(channels, dtype=dtype, device=device))
        self.eps = _eps(eps)

    def forward(self, x):
        return TypeNormFunction.apply(x.contiguous(), self.weight, self.bias, self.eps)

    def extra_repr(self):
        return "%d channels, eps %g" % (self.weight.shape[0], self.eps)


class TypeDropout(_Drawing):
    """Drops elements of type vectors while training (see ``dropout``); every call takes other
    random numbers: a count with a seed, torch's generator without one."""

    def __init__(self, p=0.1, seed=None, state=None):
        super().__init__()
        self._open(p, seed, state)

    def forward(self, x, offset=None):
        p, seed, offset, state = self._numbers(x.is_cuda, offset)
        return x if p == 0 else TypeDropoutFunction.apply(x.contiguous(), p, seed, offset, state)

    def extra_repr(self):
        return "p %g" % self.p


class TypeEncoder(_Drawing):
    """Layer turning type indices into normed vectors of a learned table, in one pass:
    ``dropout(layer_norm(scale * weight[type_index]))``, the embedding of a language model's input.
    ``Coords2Grid(gmaker, center, type_encoder=TypeEncoder(...))`` grids them."""

    def __init__(self, ntypes, channels, scale=1.0, eps=1e-5, p=0.0, seed=None, state=None,
                 dtype=None, device=None, norm_dtype=None):
        super().__init__()
        self._open(p, seed, state)
        norm_dtype = dtype if norm_dtype is None else norm_dtype
        self.weight = torch.nn.Parameter(torch.empty((ntypes, channels), dtype=dtype, device=device))
        self.norm_weight = torch.nn.Parameter(torch.ones(channels, dtype=norm_dtype, device=device))
        self.norm_bias = torch.nn.Parameter(torch.zeros(channels, dtype=norm_dtype, device=device))
        self.scale, self.eps = float(scale), _eps(eps)
        torch.nn.init.normal_(self.weight)

    def forward(self, type_index, offset=None):
        p, seed, offset, state = self._numbers(self.weight.is_cuda, offset)
        return TypeEncoderFunction.apply(type_index.contiguous(), self.weight.contiguous(),
                                         self.norm_weight, self.norm_bias, self.scale, self.eps, p,
                                         seed, offset, state)

    def extra_repr(self):
        return "%d types, %d channels, p %g" % (tuple(self.weight.shape) + (self.p,))
